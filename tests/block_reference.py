"""The operators around a block's experts in 64 bits, with a bound on what 32-bit arithmetic may add to them.

A `Bound` holds a value and how far a 32-bit evaluation of the same expression may be from it: every product, sum and function adds half a unit in the last place of its own result
(u = 2^-24 relative; expf, division and square root a little more) to what its operands bring along.  A sum of n terms in chains of `depth` additions adds depth * u
times the sum of the terms' magnitudes.  Tolerances come out of the arithmetic, not out of what a run showed."""
import torch

U = 2.0 ** -24


class Bound:
    def __init__(self, v, e=None):
        self.v = v
        self.e = torch.zeros_like(v) if e is None else e

    def __mul__(self, o):
        if not isinstance(o, Bound):
            return Bound(self.v * o, self.e * abs(o) + U * (self.v * o).abs())
        v = self.v * o.v
        return Bound(v, self.v.abs() * o.e + o.v.abs() * self.e + self.e * o.e + U * v.abs())

    def __add__(self, o):
        v = self.v + o.v
        return Bound(v, self.e + o.e + U * (v.abs() + self.e + o.e))

    def __neg__(self):
        return Bound(-self.v, self.e)

    def __sub__(self, o):
        return self + (-o)

    def sum(self, dim, depth, keepdim=False):
        return Bound(self.v.sum(dim, keepdim=keepdim), self.e.sum(dim, keepdim=keepdim) + depth * U * (self.v.abs() + self.e).sum(dim, keepdim=keepdim))

    def rsqrt(self):
        """1 / sqrt(v), v > 0: relative error halved, one rounding each of the root and the quotient."""
        v = self.v.rsqrt()
        return Bound(v, v * (0.5 * self.e / (self.v - self.e).clamp(min=1e-300) + 3 * U))

    def sigmoid(self):
        """1 / (1 + exp(-v)) of an exact argument: expf within 2 units, a sum and a quotient."""
        v = torch.sigmoid(self.v)
        return Bound(v, 6 * U * v)

    def sigmoid_slope(self):
        v = torch.sigmoid(self.v) * torch.sigmoid(-self.v)
        return Bound(v, 10 * U * v)

    def limit(self, dtype):
        """How far the value rounded to dtype may be from the exact one (half a step, and half the smallest subnormal)."""
        f = torch.finfo(dtype)
        return self.e + (f.eps / 2) * (self.v.abs() + self.e) + f.smallest_normal * f.eps


def check(got, want, name, dtype=None):
    dtype = got.dtype if dtype is None else dtype
    assert got.dtype == dtype and got.shape == want.v.shape, f"{name}: {got.dtype} {list(got.shape)}"
    off = (got.to(want.v.device, torch.float64) - want.v).abs()
    bad = ~(off <= want.limit(dtype))
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / want.limit(dtype)).max()):.2f} times the bound"


def chain(k):
    """Longest chain of additions in a row sum: 8 elements a piece, pieces a thread (of 64 at least), 6 steps of a wave, up to 16 waves."""
    return 8 * -(-k // 512) + 8 + 6 + 16


def mean(b, k):
    return b.sum(1, chain(k), keepdim=True) * (1.0 / k)


def rms(b, k, eps):
    m = mean(b * b, k)
    return Bound(m.v + eps, m.e + U * (m.v + eps) + 2.0 ** -24 * eps).rsqrt()


def exact(x):
    return None if x is None else Bound(x.detach().double())


def norm(x, weight, eps):
    x, w, k = exact(x), exact(weight), x.shape[1]
    y = x * rms(x, k, eps)
    return y if w is None else y * w


def _residual(x, z, gate, gate_act, scale, w1, eps):
    k, t = x.shape[1], x.shape[0]
    x, z = exact(x), exact(z)
    r_z = rms(z, k, eps) if w1 is not None else Bound(torch.ones_like(z.v[:, :1]))
    zh = z * r_z
    s = scale if isinstance(scale, (float, int)) else (1.0 if scale is None else exact(scale))
    # (the kernels multiply in one order or another: three roundings either way)
    sn = (zh if w1 is None else zh * exact(w1)) * s
    g = None if gate is None else Bound(gate.detach().double().reshape(t, -1))
    a = Bound(torch.ones_like(z.v[:, :1])) if g is None else (g.sigmoid() if gate_act else g)
    slope = None if g is None else (g.sigmoid_slope() if gate_act else Bound(torch.ones_like(g.v)))
    return x + sn * a, zh, r_z, sn, a, slope, s


def residual(x, z, gate=None, gate_act=None, scale=None, norm_weight=None, next_weight=None, eps=1e-6):
    h = _residual(x, z, gate, gate_act, scale, norm_weight, eps)[0]
    return h, None if next_weight is None else h * rms(h, x.shape[1], eps) * exact(next_weight)


def norm_backward(grad_y, x, weight, eps, grad_residual=None):
    k, t = x.shape[1], x.shape[0]
    xb, dy = exact(x), exact(grad_y)
    d = dy if weight is None else dy * exact(weight)
    r = rms(xb, k, eps)
    dx = r * d - xb * (r * r * r * mean(d * xb, k))
    if grad_residual is not None:
        dx = dx + exact(grad_residual)
    return dx, None if weight is None else (dy * (xb * r)).sum(0, t + 20)


def residual_backward(grad_h, grad_y, x, z, gate=None, gate_act=None, scale=None, norm_weight=None, next_weight=None, eps=1e-6):
    """(grad_x, grad_z, grad_gate, grad_scale, grad_norm_weight, grad_next_weight)."""
    k, t = x.shape[1], x.shape[0]
    h, zh, r_z, sn, a, slope, s = _residual(x, z, gate, gate_act, scale, norm_weight, eps)
    zero = Bound(torch.zeros_like(h.v))
    gh = zero if grad_h is None else exact(grad_h)
    D, grad_w2 = gh, None
    v = sn if gate is not None and a.v.shape[1] == 1 else sn * a
    inner = gh * v
    if grad_y is not None:
        dy = exact(grad_y)
        d = dy * exact(next_weight)
        r = rms(h, k, eps)
        c1 = r * r * r * mean(d * h, k)
        D = gh + r * d - h * c1
        grad_w2 = (dy * (h * r)).sum(0, t + 20)
        # (the row's sum of D v is taken as three sums: their errors add up)
        c2 = inner.sum(1, chain(k), keepdim=True) + r * (d * v).sum(1, chain(k), keepdim=True) - c1 * (h * v).sum(1, chain(k), keepdim=True)
    else:
        c2 = inner.sum(1, chain(k), keepdim=True)
        if next_weight is not None:
            grad_w2 = Bound(torch.zeros_like(next_weight, dtype=torch.float64))
    grad_gate = None
    if gate is not None:
        grad_gate = c2 * slope if a.v.shape[1] == 1 else D * sn * slope
        grad_gate = Bound(grad_gate.v.view(gate.shape), grad_gate.e.view(gate.shape))
    Da = D * a
    q = (Da * zh).sum(0, t + 20)
    w1 = exact(norm_weight)
    grad_w1 = None if w1 is None else q * s
    grad_scale = None if not isinstance(scale, torch.Tensor) else (q if w1 is None else q * w1)
    dz = Da * s
    if w1 is not None:
        c = c2 * a if gate is not None and a.v.shape[1] == 1 else c2
        dz = r_z * (dz * w1 - zh * (c * (1.0 / k)))
    return D, dz, grad_gate, grad_scale, grad_w1, grad_w2


# ---- permutation ----

def sorted_rows(ids, experts):
    """(row_of_slot, token of every row or -1 behind the routed ones, counts), by counting expert after expert."""
    t, k = ids.shape
    flat = ids.reshape(-1).tolist()
    order = [i for e in range(experts) for i in range(t * k) if flat[i] == e] if t * k * experts < 200000 else None
    if order is None:
        lists = {}
        for i, e in enumerate(flat):
            if 0 <= e < experts:
                lists.setdefault(e, []).append(i)
        order = [i for e in sorted(lists) for i in lists[e]]
    routed = len(order)
    row = [0] * (t * k)
    for r, i in enumerate(order):
        row[i] = r
    for n, i in enumerate(i for i, e in enumerate(flat) if not 0 <= e < experts):
        row[i] = -2 - (routed + n)
    counts = [0] * experts
    for e in flat:
        if 0 <= e < experts:
            counts[e] += 1
    token = [i // k for i in order] + [-1] * (t * k - routed)
    return torch.tensor(row, dtype=torch.int32).view(t, k), torch.tensor(token), torch.tensor(counts)


def unpermute(rows, m, weights, shared):
    t, k = m.shape
    valid = (m >= 0)[..., None]
    x = torch.where(valid, rows.double()[m.clamp(min=0).long()], torch.zeros((), dtype=torch.float64, device=rows.device))
    x = Bound(x) if weights is None else Bound(x) * Bound(weights.double()[..., None])
    out = x.sum(1, k + 1)
    return out if shared is None else out + exact(shared)


def unpermute_backward(grad_out, rows, m, weights):
    t, k = m.shape
    g = exact(grad_out)
    n = rows.shape[0]
    grad_rows = Bound(torch.zeros_like(rows, dtype=torch.float64))
    wg = Bound(weights.double()[..., None]) * Bound(g.v[:, None]) if weights is not None else Bound(g.v[:, None].expand(t, k, -1))
    valid = m >= 0
    grad_rows.v[m[valid].long()] = wg.v[valid]
    grad_rows.e[m[valid].long()] = wg.e[valid]
    if weights is None:
        return grad_rows, None
    x = rows.double()[m.clamp(min=0).long()] * valid[..., None]
    assert n
    return grad_rows, (Bound(x) * Bound(g.v[:, None])).sum(2, chain(rows.shape[1]))


def route_backward(grad_weights, logits, ids, renormalise):
    e = logits.shape[1]
    x = logits.double()
    valid = (ids >= 0) & (ids < e)
    at = ids.long().clamp(0, e - 1)
    dw = Bound(grad_weights.double() * valid)
    if renormalise:
        picked = torch.where(valid, x.gather(1, at), torch.full((), float("-inf"), dtype=torch.float64, device=x.device))
        p = torch.nan_to_num(torch.softmax(picked, 1))
    else:
        p = torch.softmax(x, 1).gather(1, at) * valid
    # expf within 2 units of an argument rounded once (|x - max| <= 100 of them), a sum of up to e terms, a quotient
    span = (x.max(1, keepdim=True).values - x.min(1, keepdim=True).values).clamp(min=1.0)
    rel = (e + 10) * U + 2 * span * U
    p = Bound(p, p * rel)
    inner = (dw * p).sum(1, ids.shape[1] + 8, keepdim=True)
    hit = (at[:, :, None] == torch.arange(e, device=x.device)) & valid[:, :, None]
    d = Bound((dw.v[:, :, None] * hit).sum(1), ids.shape[1] * U * (dw.v.abs()[:, :, None] * hit).sum(1))
    if renormalise:
        pe = torch.where(hit.any(1), (p.v[:, :, None] * hit).amax(1), torch.zeros((), dtype=torch.float64, device=x.device))
        pe = Bound(pe, pe * rel)
    else:
        pe = torch.softmax(x, 1)
        pe = Bound(pe, pe * rel)
    # (renormalised: every slot that chose the expert brings its own share of the inner product)
    out = pe * (d - inner * Bound(hit.sum(1).double())) if renormalise else pe * (d - inner)
    out.e += 1e-44  # (probabilities below the smallest fp32 number)
    return out
