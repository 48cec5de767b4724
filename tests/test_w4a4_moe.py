"""The 4-bit operators as a MoE runs them: router logits -> top-k with groups -> expert order -> gather and
quantise -> w13 product with the gated activation -> quantise -> w2 product -> weighted sum over the slots."""
import pytest
import torch

import fp4_plain as P
from shard_b200 import formats as F
from shard_b200 import fp4, route

E, K, H, I = 16, 4, 256, 160


def _moe(x, logits, bias, w13, w2, fmt):
    w, ids = route.topk(logits, K, bias=bias, n_group=4, topk_group=2, group_score="top2")
    o = route.expert_order(ids, E)
    h = fp4.grouped_gemm(fp4.quant(x, fmt, rows=o.tokens, offsets=o.offsets), w13)
    y = fp4.grouped_gemm(fp4.quant(h, fmt, offsets=o.offsets), w2, out_dtype=torch.float32)
    return (y[o.places.long()] * w[..., None]).sum(1), ids, h, o


def _setup(fmt, t):
    g = torch.Generator().manual_seed(t)
    c13, s13, t13, v13 = P.weights(fmt, 2 * I, H, seed=1, mats=E, halves=2)
    c2, s2, t2, v2 = P.weights(fmt, H, I, seed=2, mats=E)
    # sizes that a layer has: outputs of the order of one
    w13 = fp4.pack(fmt, c13.cuda(), s13.cuda(), None if t13 is None else t13.cuda(), kind=fp4.W13)
    w2 = fp4.pack(fmt, c2.cuda(), s2.cuda(), None if t2 is None else t2.cuda())
    x = (0.05 * torch.randn(t, H, generator=g)).to(torch.bfloat16)
    return x, torch.randn(t, E, generator=g), 0.1 * torch.randn(E, generator=g), w13, w2, v13, v2


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [F.FMT_NVFP4, F.FMT_MXFP4])
@pytest.mark.parametrize("t", [1, 5, 130, 1000])
def test_moe_of_the_operators(fmt, t):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    x, logits, bias, w13, w2, v13, v2 = _setup(fmt, t)
    y, ids, h, o = _moe(x.cuda(), logits.cuda(), bias.cuda(), w13, w2, fmt)
    rw, rids = P.route(logits, K, bias, n_group=4, topk_group=2, group_score="top2")
    assert torch.equal(ids.cpu(), rids)
    off = o.offsets.tolist()
    tok = o.tokens.cpu().long()
    xv = P.values(*P.quant(x, fmt)[:2], fmt, P.quant(x, fmt)[2])[:, :H]
    # w13: bf16 rounding (2^-9), and sums that are far closer
    for e in range(E):
        r = xv[tok[off[e]:off[e + 1]]] @ v13[e].T
        want = r[:, :I] / (1 + torch.exp(-r[:, :I])) * r[:, I:]
        got = h[off[e]:off[e + 1]].cpu().double()
        assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 1e-4 * want.abs().max()).all()) if r.shape[0] else True
    # from h on, exactly the operand that the kernel made of h
    hc = h.cpu()
    c, s, ts = P.quant(hc, fmt)
    hv = P.values(c, s, fmt, ts)[:, :I]
    out = torch.empty(tok.numel(), H, dtype=torch.float64)
    tol = torch.empty_like(out)
    for e in range(E):
        a = hv[off[e]:off[e + 1]]
        out[off[e]:off[e + 1]] = a @ v2[e].T
        tol[off[e]:off[e + 1]] = (I / 64 + 2) * 2.0 ** -22 * (a.abs() @ v2[e].abs().T) + 2.0 ** -22 * (a @ v2[e].T).abs()
    pl = o.places.cpu().long()
    want = (out[pl] * rw[..., None]).sum(1)
    lim = ((tol[pl] + 2.0 ** -19 * out[pl].abs()) * rw[..., None]).sum(1)   # weights and the sum: fp32 roundings
    assert bool(((y.cpu().double() - want).abs() <= lim).all())
    assert fp4.device_error() == 0


@pytest.mark.gpu
def test_moe_captured_on_another_stream():
    """Captured once, replayed on new inputs: the eager results, bit for bit; twice in a row without a wait."""
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    x, logits, bias, w13, w2, _, _ = _setup(F.FMT_NVFP4, 64)
    xs, ls, bs = x.cuda(), logits.cuda(), bias.cuda()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        _moe(xs, ls, bs, w13, w2, F.FMT_NVFP4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        out = _moe(xs, ls, bs, w13, w2, F.FMT_NVFP4)[0]
    for seed in (1, 2, 3):
        g = torch.Generator().manual_seed(seed)
        xs.copy_((0.05 * torch.randn(64, H, generator=g)).to(torch.bfloat16))
        ls.copy_(torch.randn(64, E, generator=g))
        torch.cuda.synchronize()
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        want = _moe(xs, ls, bs, w13, w2, F.FMT_NVFP4)[0]
        assert torch.equal(out, want)


@pytest.mark.gpu
def test_a_given_stream_orders_the_call():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    x, logits, bias, w13, w2, _, _ = _setup(F.FMT_NVFP4, 200)
    xs, ls, bs = x.cuda(), logits.cuda(), bias.cuda()
    want = _moe(xs, ls, bs, w13, w2, F.FMT_NVFP4)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    _, ids = route.topk(ls, K, bias=bs, n_group=4, topk_group=2, group_score="top2", stream=st)
    o = route.expert_order(ids, E, stream=st)
    a = fp4.quant(xs, "nvfp4", rows=o.tokens, offsets=o.offsets, stream=st)
    h = fp4.grouped_gemm(a, w13, stream=st)
    st.synchronize()
    assert torch.equal(h, want[2]) and torch.equal(ids, want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [F.FMT_NVFP4, F.FMT_MXFP4])
def test_moe_with_dropped_pairs(fmt):
    """Ids outside the experts (dropped tokens, padding) add nothing, whatever the rows that no expert wrote hold."""
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    x, logits, bias, w13, w2, _, _ = _setup(fmt, 40)
    x, logits, bias = x.cuda(), logits.cuda(), bias.cuda()
    w, ids = route.topk(logits, K, bias=bias, n_group=4, topk_group=2, group_score="top2")

    def run(ids, w):
        o = route.expert_order(ids, E)
        h = fp4.grouped_gemm(fp4.quant(x, fmt, rows=o.tokens, offsets=o.offsets), w13)
        out = torch.full((ids.numel(), H), float("nan"), device="cuda")
        fp4.grouped_gemm(fp4.quant(h, fmt, offsets=o.offsets), w2, out_dtype=torch.float32, out=out)
        at = o.places.long()[..., None]
        return torch.where(at >= 0, out[at[..., 0]] * w[..., None], 0).sum(1)

    whole = run(ids, w)
    drop = torch.zeros(40, K, dtype=torch.bool, device="cuda")
    drop[3], drop[7, 1], drop[20:24, 2:], drop[39, 3] = True, True, True, True
    part = run(torch.where(drop, -1, ids), w)
    kept = run(ids, w * ~drop)
    assert torch.equal(part, kept) and bool((part[3] == 0).all()) and torch.equal(part[0], whole[0])
