"""The operators around a block's experts without a GPU: the reference formulas of their gradients against differences, what the entry points refuse, sizes of workspaces."""
import ctypes as C

import pytest
import torch

import block_reference as R


def _differences(f, inputs, seeds):
    """d <f, seeds> / d inputs by central differences in 64 bits."""
    out = []
    for x in inputs:
        g = torch.zeros_like(x)
        flat, gf = x.view(-1), g.view(-1)
        for i in range(flat.numel()):
            old, step = float(flat[i]), 1e-5
            vals = []
            for s in (step, -step):
                flat[i] = old + s
                vals.append(sum((o * w).sum() for o, w in zip(f(), seeds)))
            flat[i] = old
            gf[i] = (vals[0] - vals[1]) / (2 * step)
        out.append(g)
    return out


def _close(got, want, name):
    # central differences of a function of size 1: step^2 from the third derivative, 1e-16 / step from rounding
    assert (got - want).abs().max() < 1e-7 * max(1.0, float(want.abs().max())), name


@pytest.mark.parametrize("gate", [None, "token", "element"])
@pytest.mark.parametrize("act", [None, "sigmoid"])
@pytest.mark.parametrize("scale", [0.7, "channel"])
@pytest.mark.parametrize("w1,w2", [(True, True), (False, True), (True, False)])
def test_residual_gradients_against_differences(gate, act, scale, w1, w2):
    g = torch.Generator().manual_seed(5)
    t, k = 3, 5
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, z = rnd(t, k), rnd(t, k)
    gt = {None: None, "token": rnd(t), "element": rnd(t, k)}[gate]
    sc = rnd(k) if scale == "channel" else scale
    a, b = rnd(k) if w1 else None, rnd(k) if w2 else None
    gh, gy = rnd(t, k), rnd(t, k) if w2 else None
    kw = dict(gate=gt, gate_act=act, scale=sc, norm_weight=a, next_weight=b, eps=1e-3)
    want = R.residual_backward(gh, gy, x, z, **kw)
    leaves = [(x, want[0], "x"), (z, want[1], "z"), (gt, want[2], "gate"), (sc if scale == "channel" else None, want[3], "scale"), (a, want[4], "w1"), (b, want[5], "w2")]
    leaves = [v for v in leaves if v[0] is not None]
    f = lambda: [o.v for o in R.residual(x, z, **kw) if o is not None]  # noqa: E731
    got = _differences(f, [v[0] for v in leaves], [gh] + ([gy] if w2 else []))
    for d, (_, w, name) in zip(got, leaves):
        _close(w.v, d, name)


def test_norm_gradients_against_differences():
    g = torch.Generator().manual_seed(6)
    x, w, gy, gr = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((3, 4), (4,), (3, 4), (3, 4)))
    dx, dw = R.norm_backward(gy, x, w, 1e-3, gr)
    got = _differences(lambda: [R.norm(x, w, 1e-3).v, x], [x, w], [gy, gr])
    _close(dx.v, got[0], "x")
    _close(dw.v, got[1], "w")


@pytest.mark.parametrize("renormalise", [False, True])
def test_routing_gradients_against_differences(renormalise):
    g = torch.Generator().manual_seed(7)
    logits = torch.randn(3, 6, generator=g, dtype=torch.float64)
    ids = torch.tensor([[0, 3], [5, 1], [2, 2]], dtype=torch.int32)      # (the last token names an expert twice)
    dw = torch.randn(3, 2, generator=g, dtype=torch.float64)

    def f():
        p = torch.softmax(logits, 1).gather(1, ids.long())
        return [p / p.sum(1, keepdim=True) if renormalise else p]

    _close(R.route_backward(dw, logits, ids, renormalise).v, _differences(f, [logits], [dw])[0], "logits")


def test_permutation_reference_on_a_hand_written_batch():
    ids = torch.tensor([[2, 0], [-1, 2], [0, 0]])
    m, token, counts = R.sorted_rows(ids, 3)
    assert m.tolist() == [[3, 0], [-2 - 5, 4], [1, 2]] and token.tolist() == [0, 2, 2, 0, 1, -1] and counts.tolist() == [3, 0, 2]


# ---- refusals of the C entry points: decided before anything touches a GPU ----

def _buffer():
    b = (C.c_int64 * 64)()
    return b, (C.addressof(b) + 15) & ~15


def test_permute_tokens_refuses(lib):
    keep, p = _buffer()

    def call(ld=8, dtype=0, ids_bytes=4, t=2, k=2, e=4, K=8, hidden=p, ids=p, rows=p, m=p, recv=p, ws=p):
        return lib.mxmoe_permute_tokens(hidden, ld, dtype, ids, ids_bytes, t, k, e, K, rows, 0, m, recv, None, ws, None)

    for bad in (dict(t=-1), dict(k=0), dict(k=65), dict(e=0), dict(e=4097), dict(K=0), dict(t=1 << 29, k=4), dict(dtype=3), dict(dtype=-1), dict(ids_bytes=2), dict(ld=-1),
                dict(t=5000, ws=p + 4)):
        assert call(**bad) == 3, bad
        assert lib.mxmoe_last_error()
    for bad in (dict(hidden=None), dict(ids=None), dict(rows=None), dict(m=None), dict(recv=None), dict(t=5000, ws=None)):
        assert call(**bad) == 5, bad
    # no scratch up to 4096 slots; beyond, a row of counts per expert and one for ids out of range, a count per 1024 slots (in whole 16 bytes) and a total
    assert lib.mxmoe_permute_tokens_workspace_bytes(2048, 2, 60) == 0
    assert lib.mxmoe_permute_tokens_workspace_bytes(4097, 1, 60) == 61 * (8 + 1) * 4
    assert lib.mxmoe_permute_tokens_workspace_bytes(0, 2, 60) == 0 and lib.mxmoe_permute_tokens_workspace_bytes(8192, 4, 0) == 0


def test_unpermute_tokens_refuses(lib):
    keep, p = _buffer()

    def fwd(rows=p, ld=8, n=4, m=p, w=p, sh=None, lds=0, dtype=0, t=2, k=2, K=8, out=p):
        return lib.mxmoe_unpermute_tokens(rows, ld, n, m, w, sh, lds, dtype, t, k, K, out, None)

    def bwd(g=p, ldg=8, rows=p, ld=8, n=4, m=p, w=p, dtype=0, t=2, k=2, K=8, gr=p, gw=p):
        return lib.mxmoe_unpermute_tokens_backward(g, ldg, rows, ld, n, m, w, dtype, t, k, K, gr, 0, gw, None)

    for bad in (dict(t=-1), dict(k=0), dict(k=65), dict(K=0), dict(n=-1), dict(dtype=3), dict(ld=-1)):
        assert fwd(**bad) == 3 and bwd(**bad) == 3, bad
    assert fwd(lds=-1) == 3 and bwd(ldg=-1) == 3
    for bad in (dict(rows=None), dict(m=None), dict(out=None)):
        assert fwd(**bad) == 5, bad
    for bad in (dict(g=None), dict(m=None), dict(gr=None), dict(rows=None)):
        assert bwd(**bad) == 5, bad
    assert fwd(t=0, rows=None, m=None, out=None) == 0 and bwd(t=0, n=0, g=None, m=None, gr=None) == 0 and bwd(t=0, gr=None) == 5


def test_route_topk_backward_refuses(lib):
    keep, p = _buffer()

    def call(g=p, x=p, dtype=1, ids=p, t=2, e=4, k=2, out=p):
        return lib.mxmoe_route_topk_backward(g, x, dtype, ids, t, e, k, 0, out, None)

    for bad in (dict(t=-1), dict(e=0), dict(e=4097), dict(k=0), dict(k=5), dict(e=100, k=65), dict(dtype=3)):
        assert call(**bad) == 3, bad
    for bad in (dict(g=None), dict(x=None), dict(ids=None), dict(out=None)):
        assert call(**bad) == 5, bad
    assert call(t=0, g=None, x=None, ids=None, out=None) == 0


def test_block_norms_refuse(lib):
    keep, p = _buffer()

    def norm(x=p, ldx=8, xt=0, w=p, wt=0, t=2, K=8, y=p, yt=0):
        return lib.mxmoe_block_norm(x, ldx, xt, w, wt, 1e-6, t, K, y, yt, None)

    def res(x=p, ldx=8, xt=0, z=p, ldz=8, zt=0, kind=0, gate=None, ldg=0, gt=1, t=2, K=8, h=p, wt=1):
        return lib.mxmoe_block_residual(x, ldx, xt, z, ldz, zt, kind, gate, ldg, gt, 0, 1.0, None, None, None, wt, 1e-6, t, K, h, None, None)

    def bwd(gh=p, gy=p, x=p, z=p, kind=0, gate=None, zt=0, gt=1, scale=None, w1=None, w2=p, t=2, K=8, gx=p, gz=p, gg=None, gs=None, g1=None, g2=p, ws=p):
        return lib.mxmoe_block_residual_backward(gh, 8, gy, 8, x, 8, 0, z, 8, zt, kind, gate, 8, gt, 0, 1.0, scale, w1, w2, 1, 1e-6, t, K, gx, gz, gg, gs, g1, g2, ws, None)

    def nbwd(gy=p, x=p, w=p, t=2, K=8, gx=p, gw=p, ws=p):
        return lib.mxmoe_block_norm_backward(gy, 8, 0, x, 8, 0, w, 1, None, 0, 1e-6, t, K, gx, gw, ws, None)

    for bad in (dict(t=-1), dict(K=0), dict(K=32769)):
        assert norm(**bad) == 3 and res(**bad) == 3 and bwd(**bad) == 3 and nbwd(**bad) == 3, bad
    for bad in (dict(ldx=-1), dict(xt=3), dict(wt=-1)):
        assert norm(**bad) == 3 and res(**bad) == 3, bad
    assert norm(yt=3) == 3 and res(zt=3) == 3 and res(kind=3) == 3 and res(kind=2, gate=p, gt=2) == 3 and res(ldz=-1) == 3 and bwd(kind=2, gate=p, gt=2) == 3
    for bad in (dict(x=None), dict(y=None)):
        assert norm(**bad) == 5, bad
    for bad in (dict(x=None), dict(z=None), dict(h=None), dict(kind=1)):
        assert res(**bad) == 5, bad
    for bad in (dict(gh=None, gy=None), dict(x=None), dict(z=None), dict(gx=None), dict(gz=None), dict(g2=None), dict(ws=None, t=5), dict(kind=1, gate=p), dict(scale=p), dict(w1=p)):
        assert bwd(**bad) == 5, bad
    for bad in (dict(gy=None), dict(x=None), dict(gx=None), dict(gw=None), dict(ws=None, t=5)):
        assert nbwd(**bad) == 5, bad
    assert norm(t=0, x=None, y=None) == 0 and res(t=0, x=None, z=None, h=None) == 0
    assert lib.mxmoe_block_backward_workspace_bytes(0, 64) == 0 and lib.mxmoe_block_backward_workspace_bytes(7, 64) == 2 * 2 * 64 * 4
    assert lib.mxmoe_block_backward_workspace_bytes(3, 32769) == 0


def test_operators_take_no_host_tensors_and_say_what_they_expect():
    from mxmoe_amd import ops

    x, ids, m = torch.zeros(3, 8), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32)
    calls = [lambda: ops.permute_tokens(x, ids, 4), lambda: ops.unpermute_tokens(x, m), lambda: ops.permute_tokens_backward(x, m), lambda: ops.unpermute_tokens_backward(x, x, m),
             lambda: ops.block_norm(x), lambda: ops.block_norm_backward(x, x), lambda: ops.block_residual(x, x), lambda: ops.block_residual_backward(x, None, x, x),
             lambda: ops.route_topk_backward(torch.zeros(3, 2), x, ids)]
    for call in calls:
        with pytest.raises(ValueError, match="a GPU expected"):
            call()
    with pytest.raises(ValueError, match="rows expected"):
        ops.block_norm(torch.zeros(3))
    with pytest.raises(ValueError, match="fp16, fp32 or bf16"):
        ops.block_norm(torch.zeros(3, 8, dtype=torch.float64))
