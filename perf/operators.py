"""The operators around the experts' products of one MoE block, as cases that can be timed: one pass of one operator, forward or backward.

  permute    tokens sorted by expert, from the routing's ids; backward: the rows' gradients summed back into the tokens
  unpermute  the experts' rows back in token order, weighted, with a shared expert's rows; backward: gradients of rows and weights
  route      backward of softmax + top-k (+ renormalisation): the weights' gradient to the router's logits
  norm       RMS norm in front of a block; backward: with the residual stream's own gradient added
  residual   a block's output normed, gated and scaled onto the residual stream, and the next block's norm of it; backward: all gradients

`run` computes them in plain 32-bit torch operations, or through `mxmoe_amd.ops` where `own` is set.  Sizes are those of the layers of
`mxmoe_amd.synth.CONFIGS` (60 experts top-4 and 64 experts top-6 with rows of 2048, 8 experts top-2 with rows of 4096).
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
QWEN = dict(experts=60, topk=4, hidden=2048)
DS2 = dict(experts=64, topk=6, hidden=2048)
MIXTRAL = dict(experts=8, topk=2, hidden=4096)


def _permute(direction, tokens, dtype, padded=0, skewed=False, ids="int32", **sizes):
    return dict(op="permute", direction=direction, tokens=tokens, padded=padded, skewed=skewed, ids=ids, dtype=dtype, **sizes)


def _unpermute(direction, tokens, dtype, padded=0, skewed=False, shared=False, **sizes):
    return dict(op="unpermute", direction=direction, tokens=tokens, padded=padded, skewed=skewed, shared=shared, dtype=dtype, **sizes)


def _route(tokens, dtype, experts, topk, renormalise):
    return dict(op="route", direction="backward", tokens=tokens, dtype=dtype, experts=experts, topk=topk, renormalise=renormalise)


def _norm(direction, tokens, hidden, x, y, weights):
    return dict(op="norm", direction=direction, tokens=tokens, hidden=hidden, x=x, y=y, weights=weights)


def _residual(direction, tokens, hidden, x, z, weights, gate, scale, norm, next):
    return dict(op="residual", direction=direction, tokens=tokens, hidden=hidden, x=x, z=z, weights=weights, gate=gate, scale=scale, norm=norm, next=next)


def listed():
    return [
        # one sequence decoding: a token copied to its six experts' rows; latency alone
        dict(name="permute decode 1", **_permute("forward", 1, "fp16", **DS2)),
        # a full prefill batch in front of experts of skewed popularity: 134 MB of rows written
        dict(name="permute prefill 8192", **_permute("forward", 8192, "bf16", skewed=True, **QWEN)),
        # a training step's odd batch in 32 bits with padding tokens, whose ids (torch.topk's 64-bit ones) name no expert
        dict(name="permute backward 2049 padded", **_permute("backward", 2049, "fp32", padded=137, ids="int64", **DS2)),
        # a decode batch on its way back, with the shared expert's rows
        dict(name="unpermute decode 32", **_unpermute("forward", 32, "fp16", shared=True, **DS2)),
        # a full prefill batch on its way back, long rows
        dict(name="unpermute prefill 8192 large", **_unpermute("forward", 8192, "bf16", **MIXTRAL)),
        # a training step: gradients of the rows and of the routing weights
        dict(name="unpermute backward 4096", **_unpermute("backward", 4096, "bf16", skewed=True, **QWEN)),
        # a small fine-tuning batch's router, renormalised weights
        dict(name="route backward 201", **_route(201, "fp32", 8, 2, True)),
        # a full batch's router, plain probabilities
        dict(name="route backward 8192", **_route(8192, "bf16", 64, 6, False)),
        # one token's norm on its way from a bfloat16 residual stream into the fp16 layer
        dict(name="norm decode 1", **_norm("forward", 1, 4096, "bf16", "fp16", "bf16")),
        # a training step's norm with the gradient that bypasses the block added
        dict(name="norm backward 8192", **_norm("backward", 8192, 2048, "bf16", "bf16", "bf16")),
        # a decode batch after the block: a sigmoid gate per token, and the next block's norm in the same pass
        dict(name="residual decode 32", **_residual("forward", 32, 2048, "fp16", "fp16", "fp16", "token", False, False, True)),
        # a training step after the block: norms on both sides, a gate per element, a learned scale per channel
        dict(name="residual backward 8192 large", **_residual("backward", 8192, 4096, "bf16", "bf16", "fp32", "element", True, True, True)),
    ]


def _between(rng, low, high):
    """A whole number in [low, high], even over its logarithm."""
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    most = max(work(c)["bytes"] for c in listed())
    while True:
        op = rng.choice(["permute", "permute", "unpermute", "unpermute", "route", "norm", "residual", "residual"])
        direction = rng.choice(["forward", "backward"])
        tokens = _between(rng, 1, 8192)
        # rows of whole 16-byte pieces, as models have them, and now and then any length
        hidden = _between(rng, 16, 1024) * 8 if rng.random() < 0.85 else _between(rng, 33, 8191)
        dtype = rng.choice(["fp16", "bf16", "bf16", "fp32"])
        experts = _between(rng, 2, 256)
        topk = rng.randint(1, min(8, experts))
        padded = rng.choice([0, 0, tokens // 10])
        sizes = dict(experts=experts, topk=topk, hidden=hidden)
        if op == "permute":
            case = _permute(direction, tokens, dtype, padded, rng.random() < 0.5, rng.choice(["int32", "int64"]), **sizes)
        elif op == "unpermute":
            case = _unpermute(direction, tokens, dtype, padded, rng.random() < 0.5, direction == "forward" and rng.random() < 0.5, **sizes)
        elif op == "route":
            case = _route(tokens, dtype, experts, topk, rng.random() < 0.5)
        elif op == "norm":
            case = _norm(direction, tokens, hidden, rng.choice(["bf16", "fp32", dtype]), dtype, rng.choice([dtype, "fp32"]))
        else:
            case = _residual(direction, tokens, hidden, rng.choice([dtype, dtype, "fp32"]), dtype, rng.choice([dtype, "fp32"]), rng.choice(["none", "token", "element"]),
                             rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.7)
        if work(case)["bytes"] <= most:
            return case


def _size(name):
    return TYPES[name].itemsize


def work(case):
    t, op, forward = case["tokens"], case["op"], case["direction"] == "forward"
    if op == "route":
        # logits in (renormalised weights need those of the chosen experts alone), their gradients out; ids and the weights' gradients in
        e, k, b = case["experts"], case["topk"], _size(case["dtype"])
        return dict(bytes=t * (b * ((k if case["renormalise"] else e) + e) + 8 * k), flops=t * (6 * (k if case["renormalise"] else e)))
    w = case["hidden"]
    if op in ("permute", "unpermute"):
        k, b = case["topk"], _size(case["dtype"])
        rows, routed = t * k, (t - case["padded"]) * k
        if op == "permute" and forward:
            return dict(bytes=b * w * (t + rows) + (4 if case["ids"] == "int32" else 8) * rows + 4 * rows + 8 * case["experts"], flops=0)
        if op == "permute":
            return dict(bytes=b * w * (routed + t) + 4 * rows, flops=routed * w)
        if forward:
            return dict(bytes=b * w * (routed + t + (t if case["shared"] else 0)) + 8 * rows, flops=2 * routed * w)
        return dict(bytes=b * w * (t + routed + rows) + 12 * rows, flops=3 * routed * w)
    if op == "norm":
        bx, by, bw = _size(case["x"]), _size(case["y"]), _size(case["weights"])
        if forward:
            return dict(bytes=t * w * (bx + by) + bw * w, flops=4 * t * w)
        return dict(bytes=t * w * (by + 3 * bx) + 2 * bw * w, flops=10 * t * w)
    bx, bz, bw = _size(case["x"]), _size(case["z"]), _size(case["weights"])
    gate = {"none": 0, "token": bz * t, "element": bz * t * w}[case["gate"]]
    vectors = bw * w * (case["scale"] + case["norm"] + case["next"])
    if forward:
        return dict(bytes=t * w * (2 * bx + bz + (bz if case["next"] else 0)) + gate + vectors, flops=t * w * (3 + 4 * case["norm"] + 4 * case["next"]))
    return dict(bytes=t * w * (2 * bx + bz + (bz if case["next"] else 0) + bx + bz) + 2 * gate + 2 * vectors, flops=t * w * (6 + 10 * case["norm"] + 10 * case["next"]))


# ---- inputs ----

class _Inputs:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, dtype="fp32", scale=1.0, mean=0.0):
        x = torch.empty(shape, dtype=torch.float32, device="cuda").normal_(mean, scale, generator=self.g)
        return x.to(TYPES[dtype])

    def routing(self, case):
        """(ids [T, k], weights fp32 [T, k]) of a router whose experts are equally or unequally (rank ^ -1.2) popular."""
        t, e, k = case["tokens"], case["experts"], case["topk"]
        logits = self.normal(t, e)
        if case.get("skewed"):
            u = torch.rand((t, e), generator=self.g, device="cuda").clamp_(1e-20, 1 - 1e-7)
            logits = -1.2 * torch.arange(1, e + 1, device="cuda").log() - (-u.log()).log()
        weights, ids = torch.softmax(logits, dim=1).topk(k, dim=1)
        return ids, weights

    def padding(self, case, ids):
        """Padding tokens all over the batch, as the ends of its sequences: their ids name no expert."""
        if case["padded"]:
            where = torch.randperm(case["tokens"], generator=self.g, device="cuda")[:case["padded"]]
            ids = ids.index_fill(0, where, -1)
        return ids


def _sorted_rows(ids, experts):
    """Row of every (token, slot) among all of them sorted by expert, stable; -2 - row where the id names no expert (those come last)."""
    flat = ids.reshape(-1).long()
    valid = (flat >= 0) & (flat < experts)
    order = torch.sort(torch.where(valid, flat, experts), stable=True).indices
    row = torch.empty_like(order)
    row[order] = torch.arange(flat.numel(), device=flat.device)
    counts = (flat[:, None] == torch.arange(experts, device=flat.device)).sum(0) if flat.numel() * experts < 1 << 24 else torch.bincount(flat[valid], minlength=experts)
    return torch.where(valid, row, -2 - row).to(torch.int32).view(ids.shape), order, counts


def prepare(case, seed):
    g, t, s = _Inputs(seed), case["tokens"], {"case": case}
    op, forward = case["op"], case["direction"] == "forward"
    if own:
        from mxmoe_amd import ops

        s["ops"] = ops
    if op in ("permute", "unpermute"):
        ids, weights = g.routing(case)
        ids = g.padding(case, ids)
        rows = ids.numel()
        w, dtype = case["hidden"], case["dtype"]
        if op == "permute" and forward:
            s["ids"] = ids.to(torch.int32) if case["ids"] == "int32" else ids
            s["hidden"] = g.normal(t, w, dtype=dtype)
            return s
        s["row_of_slot"] = _sorted_rows(ids, case["experts"])[0]
        if op == "permute":
            s["grad_rows"] = g.normal(rows, w, dtype=dtype, scale=0.02)
            return s
        s["weights"] = weights
        s["rows"] = g.normal(rows, w, dtype=dtype)
        if forward:
            s["shared"] = g.normal(t, w, dtype=dtype) if case["shared"] else None
        else:
            s["grad_out"] = g.normal(t, w, dtype=dtype, scale=0.02)
        return s
    if op == "route":
        s["logits"] = g.normal(t, case["experts"], dtype=case["dtype"], scale=2.0)
        s["ids"] = torch.topk(s["logits"].float(), case["topk"], dim=1).indices.to(torch.int32)
        s["grad_weights"] = g.normal(t, case["topk"], scale=0.05)
        return s
    w = case["hidden"]
    s["x"] = g.normal(t, w, dtype=case["x"], scale=3.0)
    if op == "norm":
        s["weight"] = g.normal(w, dtype=case["weights"], scale=0.1, mean=1.0)
        if not forward:
            s["grad_y"] = g.normal(t, w, dtype=case["y"], scale=0.02)
            s["grad_residual"] = g.normal(t, w, dtype=case["x"], scale=0.02)
        return s
    s["z"] = g.normal(t, w, dtype=case["z"])
    s["gate"] = {"none": lambda: None, "token": lambda: g.normal(t, dtype=case["z"], scale=1.5), "element": lambda: g.normal(t, w, dtype=case["z"], scale=1.5)}[case["gate"]]()
    s["scale"] = g.normal(w, dtype=case["weights"], scale=0.1, mean=0.5) if case["scale"] else None
    s["norm_weight"] = g.normal(w, dtype=case["weights"], scale=0.1, mean=1.0) if case["norm"] else None
    s["next_weight"] = g.normal(w, dtype=case["weights"], scale=0.1, mean=1.0) if case["next"] else None
    if not forward:
        s["grad_h"] = g.normal(t, w, dtype=case["x"], scale=0.02)
        s["grad_y"] = g.normal(t, w, dtype=case["z"], scale=0.02) if case["next"] else None
    return s


EPS = 1e-6


def run(s):
    case = s["case"]
    if own:
        return _run_own(s, s["ops"], case)
    return _PLAIN[case["op"], case["direction"]](s, case)


def _run_own(s, ops, case):
    op = case["op"]
    if case["direction"] == "forward":
        if op == "permute":
            return ops.permute_tokens(s["hidden"], s["ids"], case["experts"])
        if op == "unpermute":
            return ops.unpermute_tokens(s["rows"], s["row_of_slot"], s["weights"], shared=s["shared"])
        if op == "norm":
            return ops.block_norm(s["x"], s["weight"], EPS, out_dtype=TYPES[case["y"]])
        return ops.block_residual(s["x"], s["z"], gate=s["gate"], gate_act="sigmoid", scale=s["scale"], norm_weight=s["norm_weight"], next_weight=s["next_weight"], eps=EPS)
    if op == "permute":
        return ops.permute_tokens_backward(s["grad_rows"], s["row_of_slot"])
    if op == "unpermute":
        return ops.unpermute_tokens_backward(s["grad_out"], s["rows"], s["row_of_slot"], s["weights"])
    if op == "route":
        return ops.route_topk_backward(s["grad_weights"], s["logits"], s["ids"], renormalise=case["renormalise"])
    if op == "norm":
        return ops.block_norm_backward(s["grad_y"], s["x"], s["weight"], EPS, grad_residual=s["grad_residual"])
    grads = ops.block_residual_backward(s["grad_h"], s["grad_y"], s["x"], s["z"], gate=s["gate"], gate_act="sigmoid", scale=s["scale"], norm_weight=s["norm_weight"],
                                        next_weight=s["next_weight"], eps=EPS)
    return [g for g in grads if g is not None]


# ---- the plain forms: 32 bits, rounded once ----

def _plain_permute(s, case):
    row_of_slot, order, counts = _sorted_rows(s["ids"], case["experts"])
    rows = s["hidden"][order // case["topk"]]
    routed = (row_of_slot.reshape(-1)[order] >= 0)[:, None]
    return torch.where(routed, rows, torch.zeros((), dtype=rows.dtype, device=rows.device)), row_of_slot, counts


def _picked(rows, row_of_slot):
    """The sorted rows in (token, slot) order in 32 bits, zeros where a slot was dropped."""
    valid = (row_of_slot >= 0)[..., None]
    return torch.where(valid, rows[row_of_slot.clamp(min=0).long()].float(), 0.0)


def _plain_permute_backward(s, case):
    return _picked(s["grad_rows"], s["row_of_slot"]).sum(1).to(s["grad_rows"].dtype)


def _plain_unpermute(s, case):
    out = (_picked(s["rows"], s["row_of_slot"]) * s["weights"][..., None]).sum(1)
    if s["shared"] is not None:
        out = out + s["shared"].float()
    return out.to(s["rows"].dtype)


def _plain_unpermute_backward(s, case):
    m = s["row_of_slot"]
    valid, g = m >= 0, s["grad_out"].float()
    grad_weights = (_picked(s["rows"], m) * g[:, None]).sum(2)
    at = torch.where(valid, m, -2 - m).long().reshape(-1)
    grads = torch.where(valid[..., None], s["weights"][..., None] * g[:, None], 0.0).to(s["rows"].dtype)
    grad_rows = torch.empty_like(s["rows"])
    grad_rows[at] = grads.view(-1, grads.shape[-1])
    return grad_rows, grad_weights


def _plain_route_backward(s, case):
    logits, ids, dw = s["logits"].float(), s["ids"].long(), s["grad_weights"]
    x = logits.gather(1, ids) if case["renormalise"] else logits
    e = (x - x.max(1, keepdim=True).values).exp()
    p = e / e.sum(1, keepdim=True)
    if case["renormalise"]:
        grad = torch.zeros_like(logits).scatter_(1, ids, p * (dw - (p * dw).sum(1, keepdim=True)))
    else:
        d = torch.zeros_like(logits).scatter_(1, ids, dw)
        grad = p * (d - (p * d).sum(1, keepdim=True))
    return grad.to(s["logits"].dtype)


def _rms(x):
    return (x.square().mean(1, keepdim=True) + EPS).rsqrt()


def _plain_norm(s, case):
    x = s["x"].float()
    return (x * _rms(x) * s["weight"].float()).to(TYPES[case["y"]])


def _norm_gradient(dy, x, weight):
    """(gradient of x, gradient of the weight) of y = x rms(x) weight, 32 bits."""
    r = _rms(x)
    xh, d = x * r, dy * weight
    return r * (d - xh * (d * xh).mean(1, keepdim=True)), (dy * xh).sum(0)


def _plain_norm_backward(s, case):
    dx, dw = _norm_gradient(s["grad_y"].float(), s["x"].float(), s["weight"].float())
    return (dx + s["grad_residual"].float()).to(s["x"].dtype), dw.to(s["weight"].dtype)


def _plain_h(s, case):
    """(x + scale a n, n, a, scale) in 32 bits."""
    z = s["z"].float()
    n = z * _rms(z) * s["norm_weight"].float() if case["norm"] else z
    a = torch.ones((), device=z.device)
    if case["gate"] != "none":
        a = 1 / (1 + (-s["gate"].float()).exp())
        a = a[:, None] if case["gate"] == "token" else a
    scale = s["scale"].float() if case["scale"] else torch.ones((), device=z.device)
    return s["x"].float() + scale * a * n, n, a, scale


def _plain_residual(s, case):
    h = _plain_h(s, case)[0]
    out = h.to(s["x"].dtype)
    if not case["next"]:
        return out
    return out, (h * _rms(h) * s["next_weight"].float()).to(s["z"].dtype)


def _plain_residual_backward(s, case):
    h, n, a, scale = _plain_h(s, case)
    d = s["grad_h"].float()
    grad_next = None
    if case["next"]:
        dh, grad_next = _norm_gradient(s["grad_y"].float(), h, s["next_weight"].float())
        d, grad_next = d + dh, grad_next.to(s["next_weight"].dtype)
    grad_gate = None
    if case["gate"] != "none":
        grad_gate = d * scale * n
        if case["gate"] == "token":
            grad_gate = grad_gate.sum(1, keepdim=True)
        grad_gate = (grad_gate * a * (1 - a)).to(s["gate"].dtype).view(s["gate"].shape)
    grad_scale = (d * a * n).sum(0).to(s["scale"].dtype) if case["scale"] else None
    dn, grad_norm = d * scale * a, None
    if case["norm"]:
        dn, grad_norm = _norm_gradient(dn, s["z"].float(), s["norm_weight"].float())
        grad_norm = grad_norm.to(s["norm_weight"].dtype)
    grads = d.to(s["x"].dtype), dn.to(s["z"].dtype), grad_gate, grad_scale, grad_norm, grad_next
    return [g for g in grads if g is not None]


_PLAIN = {("permute", "forward"): _plain_permute, ("permute", "backward"): _plain_permute_backward, ("unpermute", "forward"): _plain_unpermute,
          ("unpermute", "backward"): _plain_unpermute_backward, ("route", "backward"): _plain_route_backward, ("norm", "forward"): _plain_norm,
          ("norm", "backward"): _plain_norm_backward, ("residual", "forward"): _plain_residual, ("residual", "backward"): _plain_residual_backward}


# ---- the definitions in 64 bits: sums by expert or by token, gradients by differentiation ----

def exact(case, seed):
    s = prepare(case, seed)
    t, op, forward = case["tokens"], case["op"], case["direction"] == "forward"
    if op == "permute" and forward:
        # expert after expert, the (token, slot) pairs that name it in order; then those that name none
        flat, k, n = s["ids"].reshape(-1), case["topk"], 0
        hidden = s["hidden"].double()
        rows = torch.zeros((flat.numel(), case["hidden"]), dtype=torch.float64, device=hidden.device)
        where = torch.zeros(flat.numel(), dtype=torch.int64, device=hidden.device)
        counts = []
        for e in range(case["experts"]):
            mine = (flat == e).nonzero().view(-1)
            m = mine.numel()
            rows[n:n + m] = hidden[mine // k]
            where[mine] = torch.arange(n, n + m, device=flat.device)
            counts.append(m)
            n += m
        rest = ((flat < 0) | (flat >= case["experts"])).nonzero().view(-1)
        where[rest] = -2 - torch.arange(n, n + rest.numel(), device=flat.device)
        return rows, where.view(t, k), torch.tensor(counts, device=flat.device)
    if op in ("permute", "unpermute"):
        m = s["row_of_slot"]
        if forward:
            rows, w = s["rows"].double(), s["weights"].double()
            out = torch.zeros((t, case["hidden"]), dtype=torch.float64, device=rows.device)
            for k in range(case["topk"]):
                have = (m[:, k] >= 0).nonzero().view(-1)
                out[have] += w[have, k, None] * rows[m[have, k].long()]
            return out + s["shared"].double() if s["shared"] is not None else out
        if op == "permute":
            out = torch.zeros((t, case["hidden"]), dtype=torch.float64, device=m.device)
            for k in range(case["topk"]):
                have = (m[:, k] >= 0).nonzero().view(-1)
                out[have] += s["grad_rows"][m[have, k].long()].double()
            return out
        grad_rows = torch.zeros(s["rows"].shape, dtype=torch.float64, device=m.device)
        grad_weights = torch.zeros(m.shape, dtype=torch.float64, device=m.device)
        for k in range(case["topk"]):
            have = (m[:, k] >= 0).nonzero().view(-1)
            row, d = m[have, k].long(), s["grad_out"][have].double()
            grad_rows[row] = s["weights"][have, k, None].double() * d
            grad_weights[have, k] = (d * s["rows"][row].double()).sum(1)
        return grad_rows, grad_weights
    if op == "route":
        logits = s["logits"].double().requires_grad_()
        p = torch.softmax(logits, 1).gather(1, s["ids"].long())
        w = p / p.sum(1, keepdim=True) if case["renormalise"] else p
        return torch.autograd.grad(w, logits, s["grad_weights"].double())[0]

    def norm(v, weight):
        return v / torch.sqrt((v * v).sum(1, keepdim=True) / v.shape[1] + EPS) * weight

    def leaf(name):
        return None if s[name] is None else s[name].double().requires_grad_(not forward)

    if op == "norm":
        x, weight = leaf("x"), leaf("weight")
        y = norm(x, weight)
        if forward:
            return y
        return torch.autograd.grad([y, x * 1], [x, weight], [s["grad_y"].double(), s["grad_residual"].double()])
    leaves = [leaf(name) for name in ("x", "z", "gate", "scale", "norm_weight", "next_weight")]
    x, z, gate, scale, norm_weight, next_weight = leaves
    block = z if norm_weight is None else norm(z, norm_weight)
    if gate is not None:
        block = block * torch.sigmoid(gate.view(t, -1))
    h = x + (block if scale is None else block * scale)
    y = None if next_weight is None else norm(h, next_weight)
    if forward:
        return h if y is None else (h, y)
    outs, seeds = ([h], [s["grad_h"].double()]) if y is None else ([h, y], [s["grad_h"].double(), s["grad_y"].double()])
    return list(torch.autograd.grad(outs, [v for v in leaves if v is not None], seeds))
