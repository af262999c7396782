"""The operators around a block's experts on the GPU against plain 64-bit arithmetic (block_reference.py), at the sizes, strides and masks where they can go wrong."""
import pytest
import torch

import block_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _rnd(*shape, dtype=F32, seed=0, scale=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + mean).to(dtype).to(DEV)


def _ids(t, k, e, seed=0, dropped=0.0, dtype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, e, (t, k), generator=g)
    if dropped:
        ids = torch.where(torch.rand(t, k, generator=g) < dropped, torch.tensor([-1, e, -7])[torch.randint(0, 3, (t, k), generator=g)], ids)
    return ids.to(dtype).to(DEV)


def _view(x, pad=3, offset=1):
    """The same values as rows of a wider buffer that starts in the middle of its storage: unaligned rows, a row stride of its own."""
    buf = torch.full((x.shape[0], x.shape[1] + pad), float("nan"), dtype=x.dtype, device=x.device)
    v = buf[:, offset:offset + x.shape[1]]
    v.copy_(x)
    return v


# ---- permutation ----

def _check_permute(hidden, ids, e, out=None):
    from mxmoe_amd import ops

    t, k = ids.shape
    rows, m, recv = ops.permute_tokens(hidden, ids, e, out=out)
    want_m, token, counts = R.sorted_rows(ids.cpu(), e)
    assert torch.equal(m.cpu(), want_m) and torch.equal(recv.cpu(), counts) and recv.dtype == torch.int64
    routed = int(counts.sum())
    token = token.to(hidden.device)
    assert torch.equal(rows[:routed], hidden[token[:routed]])
    if out is None:
        assert not rows[routed:].any()
    return rows, m, routed


@pytest.mark.parametrize("t,k,e", [(1, 1, 1), (1, 6, 64), (3, 64, 5), (7, 2, 4096), (63, 4, 60), (512, 8, 60), (513, 8, 3), (4096, 1, 64), (4097, 1, 64), (1025, 6, 64), (9001, 5, 256)])
@pytest.mark.parametrize("dropped", [0.0, 0.3])
@pytest.mark.parametrize("id_type", [torch.int32, torch.int64])
def test_permute_tokens(t, k, e, dropped, id_type):
    _check_permute(_rnd(t, 24, dtype=F16, seed=t), _ids(t, k, e, t + k, dropped, id_type), e)


@pytest.mark.parametrize("width", [1, 2, 7, 8, 9, 129, 2048, 2049, 8200])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_permute_tokens_row_lengths_and_views(width, dtype):
    x, ids = _rnd(37, width, dtype=dtype, seed=width), _ids(37, 3, 5, width, 0.2)
    rows, m, _ = _check_permute(x, ids, 5)
    assert torch.equal(_check_permute(_view(x), ids, 5)[0], rows)
    assert torch.equal(_check_permute(x[:1].expand(37, width), ids, 5)[0][0], x[0])          # (a row stride of 0)
    assert torch.equal(_check_permute(x.t().contiguous().t(), ids, 5)[0], rows)              # (elements not side by side: copied)
    assert torch.equal(_check_permute(x, ids.t().contiguous().t(), 5)[1], m)


def test_permute_tokens_ids_that_name_no_expert():
    from mxmoe_amd import ops

    x = _rnd(5, 16, dtype=BF16)
    _check_permute(x, torch.full((5, 2), -1, dtype=torch.int32, device=DEV), 3)
    # 64-bit ids whose low half would name an expert
    ids = torch.tensor([[0, 2 ** 32 + 1], [1, -2 ** 32], [2 ** 40 + 2, 2], [2 ** 63 - 1, 0], [-2 ** 63, 1]], device=DEV)
    _check_permute(x, ids, 3)
    # every token twice to the same expert
    _check_permute(x, torch.full((5, 2), 1, dtype=torch.int32, device=DEV), 3)
    # rows behind the last routed one are the caller's
    for t, k in ((40, 3), (3000, 2)):
        x, ids = _rnd(t, 40, dtype=F16, seed=1), _ids(t, k, 6, 9, 0.5)
        out = torch.full((t * k, 40), 7.0, dtype=F16, device=DEV)
        rows, _, routed = _check_permute(x, ids, 6, out=out)
        assert rows is out and 0 < routed < t * k and (out[routed:] == 7).all()
    rows, m, recv = ops.permute_tokens(x[:0], ids[:0], 6)
    assert rows.shape == (0, 40) and m.shape == (0, 2) and recv.tolist() == [0] * 6


def test_gg_permute_inp_gives_what_the_sort_and_the_copy_give():
    from mxmoe_amd import ops

    for t, k, e, dropped in ((33, 4, 8, 0.0), (33, 4, 8, 0.4), (3000, 3, 60, 0.1)):
        x, ids = _rnd(t, 48, dtype=F16, seed=t), _ids(t, k, e, t, dropped)
        problems, rows, perm, recv = ops.gg_permute_inp(x, ids, e)
        dst, want_perm, _slot, want_recv = ops.build_permutation(ids, e)
        routed = int(want_recv.sum())
        assert torch.equal(recv, want_recv.cpu()) and problems == int((want_recv != 0).sum()) and recv.device.type == "cpu"
        assert torch.equal(perm[:routed], want_perm[:routed]) and torch.equal(rows, x.index_select(0, want_perm[:routed]))
    x = x.clone().requires_grad_()
    rows = ops.gg_permute_inp(x, ids, e)[1]
    rows.backward(torch.ones_like(rows))
    assert torch.equal(x.grad[:, 0].float(), ((ids >= 0) & (ids < e)).sum(1).float())


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("t,k,e,width", [(1, 1, 1, 1), (1, 6, 64, 2048), (33, 6, 64, 520), (50, 9, 4, 129), (17, 20, 30, 1025), (300, 4, 60, 2048), (5, 2, 8, 8200)])
@pytest.mark.parametrize("dropped", [0.0, 0.4])
def test_unpermute_tokens_and_gradients(dtype, t, k, e, width, dropped):
    from mxmoe_amd import ops

    ids = _ids(t, k, e, t, dropped)
    x = _rnd(t, width, dtype=dtype, seed=3)
    rows, m, recv = ops.permute_tokens(x, ids, e)
    y = _rnd(t * k, width, dtype=dtype, seed=4)
    w, sh, g = _rnd(t, k, seed=5), _rnd(t, width, dtype=dtype, seed=6), _rnd(t, width, dtype=dtype, seed=7)
    y[int(recv.sum()):] = float("nan")                                                        # (rows of dropped slots are not read)
    for weights, shared in ((w, sh), (w, None), (None, None), (None, sh)):
        R.check(ops.unpermute_tokens(y, m, weights, shared), R.unpermute(y, m, weights, shared), "out")
    R.check(ops.permute_tokens_backward(y, m), R.unpermute(y, m, None, None), "grad_hidden")
    if dtype == F16 and width % 8 == 0:
        want = ops.gg_unpermute_out(torch.cat([y[:int(recv.sum())].reshape(-1), sh.reshape(-1), y.new_zeros((t * k) * width)]), ids, w, e, width, 1)
        assert torch.equal(ops.unpermute_tokens(y, m, w, sh), want)
    got, want = ops.unpermute_tokens_backward(g, y, m, w), R.unpermute_backward(g, torch.nan_to_num(y), m, w)
    R.check(got[0], want[0], "grad_rows")
    R.check(got[1], want[1], "grad_weights")
    assert not got[1][m < 0].any() and not got[0][int(recv.sum()):].any()
    for a, b in zip(ops.unpermute_tokens_backward(_view(g), _view(y), m, w), got):
        assert torch.equal(a, b)
    assert torch.equal(ops.unpermute_tokens(_view(y), m, w, _view(sh, 5, 2)), ops.unpermute_tokens(y, m, w, sh))
    # without weights: the copies; without rows: no gradient of the weights
    plain, none = ops.unpermute_tokens_backward(g, None, m)
    assert none is None and torch.equal(plain, ops.permute_tokens(g, ids, e)[0])
    only, none = ops.unpermute_tokens_backward(g, None, m, w)
    assert none is None and torch.equal(only, got[0])
    # rows behind the last routed one are the caller's
    out = torch.full_like(y, 3.0)
    ops.unpermute_tokens_backward(g, y, m, w, out=out)
    assert torch.equal(out[:int(recv.sum())], got[0][:int(recv.sum())]) and (out[int(recv.sum()):] == 3).all()


def test_unpermute_tokens_maps_of_the_other_permutation_and_bad_ones():
    from mxmoe_amd import ops

    ids = _ids(20, 3, 6, 1, 0.4)
    y, w, g = _rnd(60, 64, dtype=F16, seed=2), _rnd(20, 3, seed=3), _rnd(20, 64, dtype=F16, seed=4)
    m = ops.permute_tokens(g, ids, 6)[1]
    other = ops.build_permutation(ids, 6, with_inverse=True)[4].view(20, 3)                    # (-1 for every dropped slot)
    assert torch.equal(other, m.clamp(min=-1))
    assert torch.equal(ops.unpermute_tokens(y, other, w), ops.unpermute_tokens(y, m, w))
    routed = int((m >= 0).sum())
    a, b = ops.unpermute_tokens_backward(g, y, other, w), ops.unpermute_tokens_backward(g, y, m, w)
    assert torch.equal(a[0], b[0]) and not a[0][routed:].any() and torch.equal(a[1], b[1])
    assert torch.equal(ops.unpermute_tokens_backward(g, y[:routed], other, w)[0], b[0][:routed])
    leaf = y.clone().requires_grad_()
    ops.unpermute_tokens(leaf, other, w).backward(g)
    assert torch.equal(leaf.grad, b[0])
    more = torch.cat([y, y[:5]])                                                               # (rows that no slot can name)
    c = ops.unpermute_tokens_backward(g, more, m, w)
    assert torch.equal(c[0][:60], b[0]) and not c[0][60:].any() and torch.equal(c[1], b[1])
    # entries past the rows that there are name nothing, in either sign
    bad = m.clone()
    bad[0] = torch.tensor([60, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    out = ops.unpermute_tokens(y, bad, w)
    assert not out[0].any() and torch.equal(out[1:], ops.unpermute_tokens(y, m, w)[1:])
    _, gw = ops.unpermute_tokens_backward(g, y, bad, w)
    assert not gw[0].any() and torch.equal(gw[1:], b[1][1:])
    # a token without rows, no rows at all, no tokens
    assert not ops.unpermute_tokens(y, torch.full((4, 2), -1, dtype=torch.int32, device=DEV)).any()
    assert not ops.unpermute_tokens(y[:0], torch.full((4, 2), -1, dtype=torch.int32, device=DEV)).any()
    assert ops.unpermute_tokens(y, m[:0]).shape == (0, 64) and ops.unpermute_tokens_backward(g[:0], y[:0], m[:0], w[:0])[0].shape == (0, 64)
    nothing = ops.unpermute_tokens_backward(g[:0], y, m[:0], w[:0])
    assert nothing[0].shape == (60, 64) and not nothing[0].any() and nothing[1].shape == (0, 3)
    # many dropped slots of -1
    ids = _ids(3000, 4, 9, 5, 0.9)
    g, w = _rnd(3000, 40, dtype=F16, seed=6), _rnd(3000, 4, seed=7)
    m, other = ops.permute_tokens(g, ids, 9)[1], ops.build_permutation(ids, 9, with_inverse=True)[4].view(3000, 4)
    assert torch.equal(ops.unpermute_tokens_backward(g, None, other, w)[0], ops.unpermute_tokens_backward(g, None, m, w)[0])


def test_infinities_stay_in_their_rows():
    from mxmoe_amd import ops

    y, m = _rnd(4, 40, dtype=BF16), torch.tensor([[0, 2], [-3, 1], [-2, -1]], dtype=torch.int32, device=DEV)
    y[3] = float("inf")                                                                        # (no slot names it)
    y[1, 5] = float("nan")
    out = ops.unpermute_tokens(y, m, torch.full((3, 2), float("inf"), device=DEV).index_fill(0, torch.tensor([0, 1], device=DEV), 1.0))
    assert torch.isfinite(out[0]).all() and out[1].isnan().sum() == 1 and not out[2].any()


def test_permutation_past_32_bit_offsets():
    """More than 2^32 bytes of rows."""
    from mxmoe_amd import ops

    t, width, e = 540_000, 4096, 7
    x = torch.arange(t, device=DEV, dtype=torch.int32).bitwise_and(1023).to(BF16)[:, None].expand(t, width)
    ids = torch.arange(t, device=DEV, dtype=torch.int32).remainder(e)[:, None]
    rows, m, recv = ops.permute_tokens(x, ids, e)
    order = torch.sort(ids[:, 0], stable=True).indices
    assert torch.equal(rows[:, 0], x[order, 0]) and torch.equal(rows[-3:], x[order[-3:]]) and torch.equal(m[order, 0].long(), torch.arange(t, device=DEV))
    back = ops.unpermute_tokens(rows, m)
    assert torch.equal(back[:, 4095], x[:, 0]) and torch.equal(back[-3:], x[-3:])
    grad = ops.unpermute_tokens_backward(back, None, m)[0]
    assert torch.equal(grad[:, 4095], rows[:, 0])
    assert torch.equal(ops.block_norm(grad)[-1], ops.block_norm(grad[-1:])[0])
    z = torch.ones((), dtype=BF16, device=DEV).expand(t, width)
    h, y = ops.block_residual(grad, z, next_weight=torch.ones(width, device=DEV))
    assert torch.equal(h[-1], grad[-1] + 1) and torch.equal(y[-1], ops.block_norm(h[-1:])[0])


def test_more_rows_than_a_grid_holds_threads():
    """2^26 rows and some: a wave each would be 2^32 threads."""
    from mxmoe_amd import ops

    t = (1 << 26) + 77
    x = torch.arange(t, device=DEV, dtype=torch.int32).bitwise_and(255).to(BF16)[:, None].expand(t, 8)
    y = ops.block_norm(x, None, 1.0)
    one = ops.block_norm(x[:256].contiguous(), None, 1.0)
    assert torch.equal(y[-333:], one.repeat(3, 1)[(t - 333) % 256:][:333]) and torch.equal(y[::1001], one[(torch.arange(0, t, 1001, device=DEV)) % 256])
    del y
    m = torch.arange(t, device=DEV, dtype=torch.int32).bitwise_and(255)[:, None]
    g = ops.unpermute_tokens_backward(x, x[:256].contiguous(), m, torch.ones(t, 1, device=DEV))[1]   # a wave a token
    assert torch.equal(g[:, 0], 8 * m[:, 0].float() ** 2)
    del g
    ids = torch.ones(t, 1, device=DEV, dtype=torch.int32)
    logits = torch.tensor([0.0, 1.0] + [-1.0] * 62, dtype=BF16, device=DEV).expand(t, 64).contiguous()
    d = ops.route_topk_backward(torch.ones(t, 1, device=DEV), logits, ids)
    assert torch.equal(d, d[:1].expand(t, 64)) and torch.equal(d[:1], ops.route_topk_backward(torch.ones(1, 1, device=DEV), logits[:1], ids[:1]))


@pytest.mark.parametrize("width", [1, 5, 8, 12, 130, 515, 2055, 4100, 8200])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_nothing_is_written_past_the_rows(width, dtype):
    from mxmoe_amd import ops

    t = 5

    def guarded(rows, k, dt=dtype):
        buf = torch.full((rows * k + 64,), 7.0, dtype=dt, device=DEV)
        return buf, buf[32:32 + rows * k].view(rows, k)

    def untouched(*bufs):
        return all((b[:32] == 7).all() and (b[-32:] == 7).all() for b in bufs)

    x, ids, w = _rnd(t, width, dtype=dtype, seed=1), _ids(t, 2, 3, 1), _rnd(t, 2, seed=2)
    bufs, outs = zip(guarded(t * 2, width), guarded(t, width), guarded(t * 2, width), guarded(t, width), guarded(t, width))
    rows, m, _ = ops.permute_tokens(x, ids, 3, out=outs[0])
    ops.unpermute_tokens(rows, m, w, x, out=outs[1])
    ops.unpermute_tokens_backward(x, rows, m, w, out=outs[2])
    ops.block_norm(x, out=outs[3])
    ops.block_residual(x, x, next_weight=x[0], out=outs[4])
    assert untouched(*bufs)
    # gradients, whose buffers the operators take themselves: the entry points with guarded ones
    lib, s = _lib(), torch.cuda.current_stream().cuda_stream
    code, f = {F16: 0, F32: 1}[dtype], torch.ones(width, dtype=dtype, device=DEV)
    bufs, outs = zip(*(guarded(t, width) for _ in range(3)), *(guarded(1, width) for _ in range(3)), guarded(1, lib.mxmoe_block_backward_workspace_bytes(t, width) // 4, F32))
    p = [o.data_ptr() for o in outs]
    for tokens in (t, 3):
        rc = lib.mxmoe_block_residual_backward(x.data_ptr(), width, x.data_ptr(), width, x.data_ptr(), width, code, x.data_ptr(), width, code, 2, x.data_ptr(), width, code, 1, 1.0,
                                               f.data_ptr(), f.data_ptr(), f.data_ptr(), code, 1e-6, tokens, width, *p, s)
        torch.cuda.synchronize()
        assert rc == 0 and untouched(*bufs)


def _lib():
    from mxmoe_amd import _lib as L

    return L.load()


# ---- routing ----

@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (201, 8, 2), (33, 3, 3), (65, 60, 4), (130, 64, 6), (9, 65, 8), (21, 256, 8), (3, 4096, 64), (5, 100, 64)])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("renormalise", [False, True])
def test_route_topk_backward(t, e, k, dtype, renormalise):
    from mxmoe_amd import ops

    logits, dw = _rnd(t, e, dtype=dtype, seed=e, scale=2.0), _rnd(t, k, seed=k)
    ids, _ = ops.route_topk(logits, k, renormalise)
    got = ops.route_topk_backward(dw, logits, ids, renormalise)
    R.check(got, R.route_backward(dw, logits, ids, renormalise), "grad_logits")
    assert torch.equal(ops.route_topk_backward(dw, _view(logits), ids.long(), renormalise), got)
    # ids that a caller changed: twice the same expert, or none
    ids = ids.clone()
    ids[0] = ids[0, 0].clone()
    ids[-1, -1] = -1
    R.check(ops.route_topk_backward(dw, logits, ids, renormalise), R.route_backward(dw, logits, ids, renormalise), "grad_logits of edited ids")
    ids[-1] = e
    got = ops.route_topk_backward(dw, logits, ids.long() + 2 ** 33 * (ids == e), renormalise)
    assert not got[-1].any()


@pytest.mark.parametrize("masked", [float("-inf"), torch.finfo(F16).min])
@pytest.mark.parametrize("renormalise", [False, True])
def test_route_topk_backward_of_masked_experts(masked, renormalise):
    """Experts switched off by their logit: no gradient of their own, and that of the others as if they were not there."""
    from mxmoe_amd import ops

    logits, dw = _rnd(40, 24, dtype=F16, seed=1), _rnd(40, 3, seed=2)
    live = torch.arange(0, 24, 3, device=DEV)                                                  # (8 experts)
    few = logits[:, live].contiguous()
    full = torch.full_like(logits, masked).index_copy(1, live, few)
    ids = ops.route_topk(few, 3, renormalise)[0]
    want = R.route_backward(dw, few, ids, renormalise)
    got = ops.route_topk_backward(dw, full, live[ids.long()], renormalise)
    R.check(got[:, live], want, "grad of the live experts")
    rest = torch.ones(24, dtype=torch.bool, device=DEV).index_fill(0, live, False)
    assert not got[:, rest].any()
    # a masked expert among the chosen ones has probability 0
    ids = live[ids.long()]
    ids[:, 2] = 1
    got = ops.route_topk_backward(dw, full, ids, renormalise)
    assert torch.isfinite(got).all() and not got[:, rest].any() and got[:, live].abs().sum() > 0


def test_what_stands_in_masked_places_is_not_read():
    from mxmoe_amd import ops

    x, g = _rnd(6, 72, dtype=BF16, seed=1), _rnd(6, 72, dtype=BF16, seed=2)
    ids = _ids(6, 2, 4, 3)
    ids[[1, 4]] = -1                                                                           # (padding tokens)
    x[[1, 4]], g[[1, 4]] = float("nan"), float("inf")
    rows, m, recv = ops.permute_tokens(x, ids, 4)
    assert torch.isfinite(rows).all() and not rows[8:].any()
    w = _rnd(6, 2, seed=4)
    w[[1, 4]] = float("nan")
    out = ops.unpermute_tokens(rows, m, w)
    assert torch.isfinite(out).all() and not out[[1, 4]].any()
    gr, gw = ops.unpermute_tokens_backward(g, rows, m, w)
    assert torch.isfinite(gr).all() and not gr[8:].any() and torch.isfinite(gw).all() and not gw[[1, 4]].any()


def test_outputs_that_share_memory_with_inputs():
    from mxmoe_amd import ops

    x, ids = _rnd(6, 64, dtype=F16, seed=1), torch.tensor([[2], [0], [1], [0], [2], [1]], dtype=torch.int32, device=DEV)
    rows, m, _ = ops.permute_tokens(x, ids, 3)
    buf = torch.zeros(7, 64, dtype=F16, device=DEV)
    bad = [lambda: ops.permute_tokens(x, ids, 3, out=x), lambda: ops.unpermute_tokens(rows, m, out=rows), lambda: ops.unpermute_tokens_backward(x, None, m, out=x),
           lambda: ops.block_norm(buf[:6], out=buf[1:]), lambda: ops.block_residual(buf[:6], x, out=buf[1:]), lambda: ops.block_residual(x, buf[:6], out=buf[1:]),
           lambda: ops.unpermute_tokens(rows, m, shared=buf[:6], out=buf[1:])]
    for call in bad:
        with pytest.raises(ValueError, match="shares memory"):
            call()
    # the same tensor where a row's elements are read before they are written
    for width in (64, 61, 515, 2055):
        x, z, gate, w, r, sh = (_rnd(6, width, dtype=F16, seed=i) for i in range(6))
        tw = _rnd(6, 1, seed=7)
        calls = [(x, lambda t, o: ops.block_norm(t, out=o)), (x, lambda t, o: ops.block_residual(t, z, gate=gate, norm_weight=w[0], out=o)),
                 (z, lambda t, o: ops.block_residual(x, t, gate=gate, norm_weight=w[0], out=o)), (gate, lambda t, o: ops.block_residual(x, z, gate=t, norm_weight=w[0], out=o)),
                 (sh, lambda t, o: ops.unpermute_tokens(r, m, shared=t, out=o)), (r, lambda t, o: ops.unpermute_tokens_backward(x, t, m, tw, out=o)[0])]
        for tensor, call in calls:
            want, mine = call(tensor, None), tensor.clone()
            assert call(mine, mine) is mine and torch.equal(mine, want)


def test_route_topk_records_its_gradient():
    from mxmoe_amd import ops

    logits = _rnd(50, 12, seed=1)
    for renormalise in (False, True):
        leaf = logits.clone().requires_grad_()
        ids, w = ops.route_topk(leaf, 3, renormalise)
        plain = ops.route_topk(logits, 3, renormalise)
        assert torch.equal(ids, plain[0]) and torch.equal(w.detach(), plain[1]) and not ids.requires_grad
        g = _rnd(50, 3, seed=2)
        w.backward(g)
        assert torch.equal(leaf.grad, ops.route_topk_backward(g, logits, ids, renormalise))


# ---- norms ----

WIDTHS = [33, 512, 520, 1024, 1031, 2048, 2056, 4096, 4099, 4104, 8192, 8200, 8203, 16392, 20001, 32768]
TYPES = [(F16, F16), (BF16, BF16), (F32, F32), (F32, BF16), (BF16, F16), (F16, F32)]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("xt,yt", TYPES)
def test_block_norm_and_gradients(width, xt, yt):
    from mxmoe_amd import ops

    t = 3
    x, gy, gr = _rnd(t, width, dtype=xt, seed=1, scale=3), _rnd(t, width, dtype=yt, seed=2), _rnd(t, width, dtype=xt, seed=3)
    for wt in (None, F32, xt):
        w = None if wt is None else _rnd(width, dtype=wt, seed=4, scale=0.1, mean=1)
        y = ops.block_norm(x, w, 1e-5, out_dtype=yt)
        R.check(y, R.norm(x, w, 1e-5), "y", yt)
        assert torch.equal(ops.block_norm(_view(x), w, 1e-5, out_dtype=yt), y)
        for res in (None, gr):
            got, want = ops.block_norm_backward(gy, x, w, 1e-5, grad_residual=res), R.norm_backward(gy, x, w, 1e-5, res)
            R.check(got[0], want[0], "grad_x", xt)
            assert (got[1] is None) == (w is None)
            if w is not None:
                R.check(got[1], want[1], "grad_weight", w.dtype)
    again = ops.block_norm_backward(_view(gy), _view(x, 1, 0), w, 1e-5, grad_residual=_view(gr))
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


@pytest.mark.parametrize("width", [1, 2, 7, 8])
def test_block_norm_of_short_rows(width):
    from mxmoe_amd import ops

    x, w, g = _rnd(5, width, seed=1, scale=3), _rnd(width, seed=2), _rnd(5, width, seed=3)
    R.check(ops.block_norm(x, w, 1e-3), R.norm(x, w, 1e-3), "y")
    got, want = ops.block_norm_backward(g, x, w, 1e-3), R.norm_backward(g, x, w, 1e-3)
    R.check(got[0], want[0], "grad_x")
    R.check(got[1], want[1], "grad_weight")


@pytest.mark.parametrize("tokens", [1, 2, 255, 257, 600, 1023, 2500])
@pytest.mark.parametrize("width", [96, 515, 2048, 4100, 7168])
def test_gradient_sums_over_many_tokens(tokens, width):
    """Every number of tokens a workgroup works off, the last of them short."""
    from mxmoe_amd import ops

    x, z, w, gy = (_rnd(*s, seed=i) for i, s in enumerate(((tokens, width), (tokens, width), (width,), (tokens, width))))
    got, want = ops.block_norm_backward(gy, x, w), R.norm_backward(gy, x, w, 1e-6)
    R.check(got[0], want[0], "grad_x")
    R.check(got[1], want[1], "grad_weight")
    kw = dict(gate=x[:, 0], gate_act="sigmoid", norm_weight=w, scale=w, next_weight=w)
    for a, b, name in zip(ops.block_residual_backward(None, gy, x, z, **kw), R.residual_backward(None, gy, x, z, **kw), ("x", "z", "gate", "scale", "norm", "next")):
        R.check(a, b, name)


def _residual_case(t, width, xt, zt, wt, gate, scale, w1, w2, seed=0):
    kw = dict(gate={None: None, "token": _rnd(t, dtype=zt, seed=seed + 1, scale=1.5), "column": _rnd(t, 1, dtype=F32, seed=seed + 1), "element": _rnd(t, width, dtype=zt, seed=seed + 1, scale=1.5)}[gate],
              scale=_rnd(width, dtype=wt, seed=seed + 2, mean=0.5, scale=0.2) if scale == "channel" else scale,
              norm_weight=_rnd(width, dtype=wt, seed=seed + 3, mean=1, scale=0.1) if w1 else None, next_weight=_rnd(width, dtype=wt, seed=seed + 4, mean=1, scale=0.1) if w2 else None, eps=1e-5)
    return _rnd(t, width, dtype=xt, seed=seed + 5, scale=3), _rnd(t, width, dtype=zt, seed=seed + 6), kw


def _check_residual(x, z, kw, backward=True):
    from mxmoe_amd import ops

    t, width = x.shape
    got, want = ops.block_residual(x, z, **kw), R.residual(x, z, **kw)
    got = (got, None) if kw["next_weight"] is None else got
    R.check(got[0], want[0], "h", x.dtype)
    if want[1] is not None:
        R.check(got[1], want[1], "y", z.dtype)
    if not backward:
        return
    gh, gy = _rnd(t, width, dtype=x.dtype, seed=20), _rnd(t, width, dtype=z.dtype, seed=21) if kw["next_weight"] is not None else None
    for a, b in ((gh, gy), (None, gy), (gh, None)):
        if a is None and b is None:
            continue
        grads = ops.block_residual_backward(a, b, x, z, **kw)
        for g, want, name, like in zip(grads, R.residual_backward(a, b, x, z, **kw), ("x", "z", "gate", "scale", "norm_weight", "next_weight"),
                                       (x, z, kw["gate"], kw["scale"], kw["norm_weight"], kw["next_weight"])):
            assert (g is None) == (want is None)
            if g is not None:
                R.check(g, want, "grad of " + name, like.dtype)


@pytest.mark.parametrize("gate", [None, "token", "column", "element"])
@pytest.mark.parametrize("act", [None, "sigmoid"])
@pytest.mark.parametrize("scale", [None, 0.25, "channel"])
@pytest.mark.parametrize("w1,w2", [(False, False), (True, False), (False, True), (True, True)])
def test_block_residual_options(gate, act, scale, w1, w2):
    x, z, kw = _residual_case(5, 200, F32, F32, F32, gate, scale, w1, w2)
    _check_residual(x, z, dict(kw, gate_act=act))


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("xt,zt", TYPES)
def test_block_residual_sizes_and_types(width, xt, zt):
    for gate, wt in (("element", F32), ("token", zt)):
        x, z, kw = _residual_case(3, width, xt, zt, wt, gate, "channel", True, True)
        _check_residual(x, z, dict(kw, gate_act="sigmoid"))


def test_block_residual_views_and_in_place():
    from mxmoe_amd import ops

    x, z, kw = _residual_case(9, 264, BF16, BF16, BF16, "element", "channel", True, True)
    h, y = ops.block_residual(x, z, **kw)
    grads = ops.block_residual_backward(h, y, x, z, **kw)
    wide = dict(kw, gate=_view(kw["gate"], 5, 3))
    for a, b in zip(ops.block_residual(_view(x), _view(z), **wide), (h, y)):
        assert torch.equal(a, b)
    for a, b in zip(ops.block_residual_backward(_view(h), _view(y), _view(x), _view(z), **wide), grads):
        assert torch.equal(a, b)
    # a gate per channel, as one row for all tokens; a gate per token as a column of a matrix
    row = kw["gate"][:1].expand(9, 264)
    assert torch.equal(ops.block_residual(x, z, gate=row), ops.block_residual(x, z, gate=row.contiguous()))
    column = kw["gate"][:, 7]
    assert torch.equal(ops.block_residual(x, z, gate=column), ops.block_residual(x, z, gate=column.contiguous()))
    a, b = ops.block_residual_backward(h, None, x, z, gate=column), ops.block_residual_backward(h, None, x, z, gate=column.contiguous())
    assert torch.equal(a[2], b[2]) and torch.equal(a[0], b[0])
    # onto the residual stream itself
    kept = x.clone()
    got = ops.block_residual(x, z, out=x, **kw)
    assert got[0] is x and torch.equal(x, h) and torch.equal(got[1], y)
    with pytest.raises(ValueError, match="side by side"):
        turned = kept.t().contiguous().t()
        ops.block_residual(turned, z, out=turned)
    # no tokens: gradients of the vectors are zero
    none = ops.block_residual_backward(h[:0], y[:0], kept[:0], z[:0], **dict(kw, gate=kw["gate"][:0]))
    assert none[0].shape == (0, 264) and all(not g.any() and g.shape == (264,) for g in none[3:])
    assert ops.block_norm(kept[:0]).shape == (0, 264)


def test_norms_of_zeros_infinities_and_large_values():
    from mxmoe_amd import ops

    x = torch.zeros(4, 72, device=DEV, dtype=F16)
    x[1] = 65504.0
    x[2, 3] = float("inf")
    x[3] = 6e-8
    y = ops.block_norm(x, None, 1e-6)
    assert not y[0].any() and (y[1] == 1).all() and torch.isnan(y[2, 3]) and not y[2, :3].any()
    R.check(y[3:], R.norm(x[3:], None, 1e-6), "subnormal")
    # gradients of rows so small that 1 / rms^3 is past fp32's range
    x, g, w = _rnd(3, 72, seed=8, scale=1e-14), _rnd(3, 72, seed=9, scale=1e-3), _rnd(72, seed=10)
    got, want = ops.block_norm_backward(g, x, w, 0.0), R.norm_backward(g, x, w, 0.0)
    R.check(got[0], want[0], "grad_x of tiny rows")
    R.check(got[1], want[1], "grad_weight of tiny rows")
    # a row's values never reach another row, whatever they are
    z = _rnd(4, 72, dtype=F16)
    z[2] = float("nan")
    h, n = ops.block_residual(_rnd(4, 72, dtype=F16, seed=3), z, norm_weight=torch.ones(72, device=DEV), next_weight=torch.ones(72, device=DEV))
    assert torch.isfinite(h[[0, 1, 3]]).all() and torch.isfinite(n[[0, 1, 3]]).all() and torch.isnan(h[2]).all()
    # gates far out: exact ends, and slopes that do not vanish before their time
    gate = torch.tensor([-200.0, -80.0, 20.0, 200.0], device=DEV)
    x = _rnd(4, 72, seed=4)
    h = ops.block_residual(x, x, gate=gate, gate_act="sigmoid")
    assert torch.equal(h[0], x[0]) and torch.equal(h[3], x[3] + x[3])
    kw = dict(gate=gate, gate_act="sigmoid")
    g = ops.block_residual_backward(x, None, x, x, **kw)[2]
    want = (x.double() ** 2).sum(1) * torch.sigmoid(gate.double()) * torch.sigmoid(-gate.double())
    assert ((g.double() - want).abs() <= 1e-5 * want + 1e-38).all() and g[2] > 0


# ---- autograd ----

def test_recorded_calls_give_the_gradients_of_the_backward_calls():
    from mxmoe_amd import ops

    x, z, kw = _residual_case(7, 136, BF16, BF16, F32, "element", "channel", True, True)
    leaves = [v.clone().requires_grad_() for v in (x, z, kw["gate"], kw["scale"], kw["norm_weight"], kw["next_weight"])]
    h, y = ops.block_residual(leaves[0], leaves[1], gate=leaves[2], gate_act="sigmoid", scale=leaves[3], norm_weight=leaves[4], next_weight=leaves[5], eps=1e-5)
    gh, gy = _rnd(7, 136, dtype=BF16, seed=30), _rnd(7, 136, dtype=BF16, seed=31)
    torch.autograd.backward([h, y], [gh, gy])
    for leaf, want in zip(leaves, ops.block_residual_backward(gh, gy, x, z, **dict(kw, gate_act="sigmoid"))):
        assert torch.equal(leaf.grad, want)
    # only one of the outputs used; a gradient whose elements are one broadcast number
    for leaf in leaves:
        leaf.grad = None
    h, y = ops.block_residual(leaves[0], leaves[1], scale=0.5, next_weight=leaves[5])
    y.sum().backward()
    want = ops.block_residual_backward(None, torch.ones_like(y), x, z, scale=0.5, next_weight=kw["next_weight"])
    assert torch.equal(leaves[0].grad, want[0]) and torch.equal(leaves[5].grad, want[5]) and leaves[3].grad is None
    # one vector in two places, a gate broadcast over the tokens
    w, g = _rnd(136, seed=40).requires_grad_(), _rnd(1, 136, dtype=BF16, seed=41).requires_grad_()
    h, y = ops.block_residual(x, z, gate=g.expand(7, 136), norm_weight=w, next_weight=w, scale=w)
    torch.autograd.backward([h, y], [gh, gy])
    want = ops.block_residual_backward(gh, gy, x, z, gate=g.detach().expand(7, 136), norm_weight=w.detach(), next_weight=w.detach(), scale=w.detach())
    ref = R.residual_backward(gh, gy, x, z, gate=g.detach().expand(7, 136), norm_weight=w.detach(), next_weight=w.detach(), scale=w.detach())
    three = R.Bound(sum(b.v for b in ref[3:]), sum(b.e + 3 * R.U * b.v.abs() for b in ref[3:]))
    R.check(w.grad, three, "shared weight")
    assert torch.allclose(g.grad.float(), want[2].float().sum(0, keepdim=True), rtol=2 ** -8, atol=2 ** -8 * float(want[2].abs().sum(0).max()))  # (bf16 sum of 7 terms by torch)
    # a norm in front of a block whose residual goes past it
    leaf, wl = x.clone().requires_grad_(), kw["norm_weight"].clone().requires_grad_()
    ops.block_norm(leaf, wl, 1e-5).backward(gy)
    want = ops.block_norm_backward(gy, x, kw["norm_weight"], 1e-5)
    assert torch.equal(leaf.grad, want[0]) and torch.equal(wl.grad, want[1])
    # permutation
    ids = _ids(7, 3, 5, 1, 0.3)
    leaf = x.clone().requires_grad_()
    rows, m, recv = ops.permute_tokens(leaf, ids, 5)
    assert rows.requires_grad and not m.requires_grad and not recv.requires_grad
    gr = _rnd(21, 136, dtype=BF16, seed=50)
    rows.backward(gr)
    assert torch.equal(leaf.grad, ops.permute_tokens_backward(gr, m))
    r, w, sh = (v.requires_grad_() for v in (_rnd(21, 136, dtype=BF16, seed=51), _rnd(7, 3, dtype=BF16, seed=52), _rnd(7, 136, dtype=BF16, seed=53)))
    ops.unpermute_tokens(r, m, w, sh).backward(gh)
    want = ops.unpermute_tokens_backward(gh, r.detach(), m, w.detach())
    assert torch.equal(r.grad, want[0]) and torch.equal(w.grad, want[1].to(BF16)) and torch.equal(sh.grad, gh)
    r.grad = None
    ops.unpermute_tokens(r, m, w.detach()).sum().backward()
    assert torch.equal(r.grad, ops.unpermute_tokens_backward(torch.ones_like(gh), None, m, w.detach())[0])


def test_a_block_of_experts_trained_through():
    """Norm, router, permutation, the experts' products, the way back and the next norm as one graph, against the same in 64 bits."""
    from mxmoe_amd import ops

    t, width, e, k, inter = 70, 64, 6, 2, 48
    x, w1, w2, rw = _rnd(t, width, seed=1, scale=2), _rnd(width, seed=2, mean=1, scale=0.1), _rnd(width, seed=3, mean=1, scale=0.1), _rnd(e, width, seed=4, scale=0.2)
    up, down, gw = _rnd(e, inter, width, seed=5, scale=0.2), _rnd(e, width, inter, seed=6, scale=0.2), _rnd(width, seed=7, scale=0.2)
    pad = torch.zeros(t, dtype=torch.bool, device=DEV)
    pad[[3, 40, 69]] = True
    gh, gy = _rnd(t, width, seed=8), _rnd(t, width, seed=9)

    def grads(dtype, ids=None):
        leaves = [v.to(dtype).requires_grad_() for v in (x, w1, w2, rw, up, down, gw)]
        lx, l1, l2, lr, lu, ld, lg = leaves
        if dtype == F32:
            y = ops.block_norm(lx, l1)
            ids, weights = ops.route_topk(y @ lr.T, k, True)
            routed = ids.masked_fill(pad[:, None], -1)
            rows, m, recv = ops.permute_tokens(y, routed, e)
            parts = rows.split([*recv.tolist(), t * k - int(recv.sum())])
            z = ops.unpermute_tokens(torch.cat([torch.tanh(p @ lu[i].T) @ ld[i].T for i, p in enumerate(parts[:e])] + [parts[e]]), m, weights)
            h, n = ops.block_residual(lx, z, gate=y @ lg, gate_act="sigmoid", scale=0.5, norm_weight=l1, next_weight=l2)
        else:
            nrm = lambda v, w: v * (v.square().mean(1, keepdim=True) + 1e-6).rsqrt() * w  # noqa: E731
            y = nrm(lx, l1)
            p = torch.softmax(y @ lr.T, 1).gather(1, ids.long())
            p = p / p.sum(1, keepdim=True)
            p = p.masked_fill(pad[:, None], 0)
            z = sum(p[:, i, None] * torch.stack([torch.tanh(y[j] @ lu[a].T) @ ld[a].T for j, a in enumerate(ids[:, i].tolist())]) for i in range(k))
            h = lx + 0.5 * torch.sigmoid(y @ lg)[:, None] * nrm(z, l1)
            n = nrm(h, l2)
        return ids, torch.autograd.grad([h, n], leaves, [gh.to(dtype), gy.to(dtype)])

    ids, got = grads(F32)
    _, want = grads(torch.float64, ids)
    for a, b, name in zip(got, want, ("x", "norm", "next", "router", "up", "down", "gate")):
        # a padding token's z is zero: 1 / sqrt(eps) = 1000 stands before its gradient; otherwise some dozen roundings of 2^-24 and sums of up to 140 terms
        assert (a.double() - b).norm() <= 2 ** -24 * 2000 * b.norm(), name


def test_calls_in_python_and_in_the_extension_are_the_same(monkeypatch):
    """Every operator once with its host side in the extension and once in Python, with numbers of either kind for the residual scale."""
    from mxmoe_amd import block, ops

    class Nothing:
        def __getattr__(self, name):
            return lambda *a: None

    taken = []

    class Counted:
        def __getattr__(self, name):
            def call(*a):
                got = getattr(native, name)(*a)
                taken.append((name, got is not None))
                return got

            return call

    ops.block_norm(_rnd(1, 8))
    native = block._fast
    s = _state(3)
    monkeypatch.setattr(block, "_fast", Counted())
    want = _all_operators(s)
    scaled = [ops.block_residual(s["x"], s["x"], scale=c) for c in (2.0, 2, None)]
    assert len({name for name, ok in taken if ok}) == 8 and [ok for name, ok in taken if name == "block_residual"] == [True, True, False, True]
    monkeypatch.setattr(block, "_fast", Nothing())
    for a, b in zip(_all_operators(s), want):
        assert torch.equal(a, b) and a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride()
    for c, b in zip((2.0, 2, None), scaled):
        assert torch.equal(ops.block_residual(s["x"], s["x"], scale=c), b)
        assert torch.equal(ops.block_residual(s["x"].clone().requires_grad_(), s["x"], scale=c).detach(), b)


def test_calls_with_another_device_current(monkeypatch):
    """What a call does whose tensors are not on the current device (here: a current device that claims to be another)."""
    from mxmoe_amd import _lib as L
    from mxmoe_amd import block

    s = _state(4)
    want = _all_operators(s)
    raw = torch._C._cuda_getCurrentRawStream
    block._fast.bind(*block_addresses(), lambda: 7, raw)                                       # the extension leaves such calls to Python
    monkeypatch.setattr(L, "current_device", lambda: 7)
    try:
        got = _all_operators(s)
    finally:
        block._fast.bind(*block_addresses(), torch._C._cuda_getDevice, raw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def block_addresses():
    import ctypes as C

    from mxmoe_amd import _lib as L

    return [C.cast(getattr(L.load(), name), C.c_void_p).value for name in L._CALLS]


# ---- streams, graphs, refusals ----

def _all_operators(s):
    from mxmoe_amd import ops

    rows, m, recv = ops.permute_tokens(s["x"], s["ids"], s["e"])
    big_rows, big_m, big_recv = ops.permute_tokens(s["big"], s["big_ids"], s["e"])
    out = ops.unpermute_tokens(rows, m, s["w"], s["x"])
    gr, gw = ops.unpermute_tokens_backward(out, rows, m, s["w"])
    gx = ops.permute_tokens_backward(gr, m)
    gl = ops.route_topk_backward(gw, s["logits"], s["ids"])
    y = ops.block_norm(gx, s["v"])
    h, n = ops.block_residual(s["x"], y, gate=s["x"], gate_act="sigmoid", scale=s["v"], norm_weight=s["v"], next_weight=s["v"])
    return [rows, m, recv, big_rows, big_m, big_recv, out, gr, gw, gx, gl, y, h, n, *ops.block_norm_backward(n, h, s["v"], grad_residual=h),
            *ops.block_residual_backward(h, n, s["x"], y, gate=s["x"], gate_act="sigmoid", scale=s["v"], norm_weight=s["v"], next_weight=s["v"])]


def _state(seed):
    t, e, k = 90, 8, 3
    return dict(x=_rnd(t, 520, dtype=F16, seed=seed), ids=_ids(t, k, e, seed, 0.1), e=e, w=_rnd(t, k, seed=seed + 1), logits=_rnd(t, e, seed=seed + 2), v=_rnd(520, dtype=F16, seed=seed + 3),
                big=_rnd(2500, 24, dtype=F16, seed=seed + 4), big_ids=_ids(2500, 2, e, seed + 5, 0.1))


def test_operators_in_graphs_and_on_another_stream():
    """Two captures replayed in turn, with eager calls and new inputs between the replays: every replay gives the eager results."""
    side = torch.cuda.Stream()
    states, graphs, outs = [_state(1), _state(2)], [], []
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in states:
            _all_operators(s)
    torch.cuda.current_stream().wait_stream(side)
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(_all_operators(s))
        graphs.append(g)
    for replay in range(4):
        for i, s in enumerate(states):
            for key, v in _state(10 * replay + i).items():
                if isinstance(v, torch.Tensor):
                    s[key].copy_(v)
        wants = [[o.clone() for o in _all_operators(s)] for s in states]
        for o in outs[0] + outs[1]:
            o.fill_(3)
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, wants):
            for n, (a, b) in enumerate(zip(got, want)):
                assert torch.equal(a, b), f"output {n}, replay {replay}"
    with torch.cuda.stream(side):
        again = _all_operators(states[1])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, wants[1]))


def test_two_threads_on_two_streams():
    import threading

    states, wants, gots = [_state(5), _state(6)], [], [None, None]
    for s in states:
        wants.append([o.clone() for o in _all_operators(s)])
    torch.cuda.synchronize()

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                gots[i] = _all_operators(states[i])
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for got, want in zip(gots, wants):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_recorded_call_under_capture_is_refused():
    from mxmoe_amd import ops

    x = _rnd(4, 32).requires_grad_()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        for call in (lambda: ops.block_norm(x), lambda: ops.permute_tokens(x, torch.zeros(4, 1, dtype=torch.int32, device=DEV), 2), lambda: ops.block_residual(x, x),
                     lambda: ops.route_topk(x, 2)):
            with pytest.raises(RuntimeError, match="captured"):
                call()
        with torch.no_grad():
            y = ops.block_norm(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, ops.block_norm(x.detach()))


def test_refusals():
    from mxmoe_amd import ops

    x, ids, v = _rnd(4, 32, dtype=F16), _ids(4, 2, 3), _rnd(32)
    m = ops.permute_tokens(x, ids, 3)[1]
    bad = [lambda: ops.permute_tokens(x, ids[:3], 3), lambda: ops.permute_tokens(x, ids.float(), 3), lambda: ops.permute_tokens(x, ids.cpu(), 3), lambda: ops.permute_tokens(x.double(), ids, 3),
           lambda: ops.permute_tokens(x, ids, 3, out=x), lambda: ops.unpermute_tokens(x, m.long()), lambda: ops.unpermute_tokens(x, m, v), lambda: ops.unpermute_tokens(x, m, shared=x[:3]),
           lambda: ops.unpermute_tokens(x, m, shared=x.float()), lambda: ops.unpermute_tokens_backward(x, x[:, :8], m), lambda: ops.unpermute_tokens_backward(x[:3], x, m),
           lambda: ops.block_norm(x, v[:8]), lambda: ops.block_norm(x, v, out_dtype=torch.float64), lambda: ops.block_norm(x, out=x[:2]), lambda: ops.block_norm_backward(x[:2], x),
           lambda: ops.block_norm_backward(x, x, grad_residual=x.float()), lambda: ops.block_residual(x, x[:3]), lambda: ops.block_residual(x, x, gate=v),
           lambda: ops.block_residual(x, x, gate=x.float()), lambda: ops.block_residual(x, x, gate_act="tanh"), lambda: ops.block_residual(x, x, scale=v, norm_weight=v.half()),
           lambda: ops.block_residual(x, x, scale=v[:3]), lambda: ops.block_residual_backward(None, None, x, x), lambda: ops.block_residual_backward(x, x, x, x),
           lambda: ops.block_residual_backward(x.float(), None, x, x), lambda: ops.route_topk_backward(v, x, ids), lambda: ops.route_topk_backward(ids.float(), x, ids.float())]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f"call {i} was not refused")
    with pytest.raises(RuntimeError):
        ops.permute_tokens(x, ids, 0)
    with pytest.raises(RuntimeError):
        ops.block_norm(torch.zeros(1, 40000, device=DEV))
    with pytest.raises(ValueError, match="without gradients"):
        ops.block_norm(x.clone().requires_grad_(), out=torch.empty_like(x))


# ---- the layer's block ----

@pytest.mark.parametrize("stream_type", [F16, BF16, F32])
def test_forward_block_is_its_operators_in_sequence(stream_type):
    from mxmoe_amd import ops, synth
    from mxmoe_amd.layer import MxMoELayer

    t = 24
    cfg = synth.MoEConfig("block", "test", 8, 2, 512, 256, t, num_shared=1, rotate=1)
    layer = MxMoELayer(cfg, formats=[(synth.W4A4, synth.W8A8), (synth.W8A8, synth.W4A4)] * 4 + [(synth.W8A8, synth.W8A8)])
    x, rw = _rnd(t, 512, dtype=stream_type, seed=1, scale=2), _rnd(8, 512, dtype=F16, seed=2, scale=0.1)
    w1, w2, w3, gate = _rnd(512, seed=3, mean=1, scale=0.1), _rnd(512, seed=4, mean=1, scale=0.1), _rnd(512, seed=5, mean=1, scale=0.1), _rnd(t, seed=6)
    y = ops.block_norm(x, w1, out_dtype=F16)
    z = layer.forward_from_logits(y, torch.nn.functional.linear(y, rw), renormalise=True).clone()
    want = ops.block_residual(x, z, gate=gate, gate_act="sigmoid", scale=0.5, norm_weight=w2, next_weight=w3)
    kw = dict(renormalise=True, gate=gate, gate_act="sigmoid", scale=0.5, post_weight=w2, next_weight=w3)
    for got in (layer.forward_block(x, rw, w1, **kw), layer.forward_block(x, rw, normed=y, **kw)):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[1].dtype == F16 and got[0].dtype == stream_type
    # two blocks after each other in one graph: the second takes the first one's normed output
    def two():
        h, n = layer.forward_block(x, rw, w1, **kw)
        return layer.forward_block(h, rw, normed=n, renormalise=True)

    eager = two().clone()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        two()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph, stream=side):
        out = two()
    for _ in range(3):
        out.fill_(float("nan"))
        layer.forward_block(x, rw, w1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
    with pytest.raises(ValueError, match="one of"):
        layer.forward_block(x, rw)
