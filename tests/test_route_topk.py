"""shard_b200.route against a plain 64-bit router. Ids and the order are compared exactly; a weight is a few
fp32 roundings from exact: the exponential's argument (|l - max| 2^-24 of the score), its value, the sums,
the division, the scale, together below (16 + |l - max|) 2^-23 of the weight."""
import math

import pytest
import torch

import fp4_plain as P
from shard_b200 import route

gpu = pytest.mark.gpu


def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _check(logits, k, bias=None, **kw):
    w, ids = route.topk(logits.cuda(), k, bias=None if bias is None else bias.cuda(), **kw)
    rw, rids = P.route(logits.cpu(), k, bias, **kw)
    assert torch.equal(ids.cpu(), rids)
    fin = logits.float().cpu()
    fin = fin[torch.isfinite(fin) & (fin.abs() < 1e30)]
    spread = float(fin.max() - fin.min()) if fin.numel() else 0.0
    assert bool(((w.cpu().double() - rw).abs() <= (16 + spread) * 2.0 ** -23 * rw + 1e-37).all())


GROUPS = [(1, 1, 1, 1), (5, 7, 3, 1), (16, 64, 6, 1), (33, 256, 8, 8), (130, 384, 8, 1), (9, 96, 4, 8), (6, 160, 8, 32),
          (4, 1024, 16, 16), (3, 60, 5, 4), (2, 31, 16, 1), (7, 100, 8, 4), (3, 1000, 8, 8)]


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid", "sqrtsoftplus"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,e,k,g", GROUPS)
def test_topk(score, dtype, t, e, k, g):
    _need_gpu()
    gen = torch.Generator().manual_seed(t * e + k)
    logits = (2 * torch.randn(t, e, generator=gen)).to(dtype)
    bias = 0.2 * torch.randn(e, generator=gen)
    kept = max(1, g // 2, -(-k * g // e))
    for b in (None, bias):
        for gs in ("max", "top2") if g > 1 else ("max",):
            _check(logits, k, b, score=score, n_group=g, topk_group=kept, group_score=gs, renormalize=score != "softmax",
                   scale=1.5)


@gpu
@pytest.mark.parametrize("bias", [None, "zero", "steps"])
def test_topk_ties_go_to_the_lower_id(bias):
    """Few distinct logits; biases that make the sums of unequal scores nearly or exactly equal."""
    _need_gpu()
    gen = torch.Generator().manual_seed(3)
    logits = torch.randint(-2, 3, (64, 256), generator=gen).float()
    b = None
    if bias == "zero":
        b = torch.zeros(256)
    if bias == "steps":     # bias = 0.5 - sigmoid(l) rounded to fp32: the sums differ in the 8th digit only
        logits = (0.5 * torch.arange(256).float() % 7 - 3).expand(64, 256).contiguous()
        b = (0.5 - torch.sigmoid(logits[0].double())).float()
    for g in (1, 8):
        for gs in ("max", "top2"):
            _check(logits, 8, b, score="sigmoid", n_group=g, topk_group=4 if g > 1 else 1, group_score=gs)
            _check(logits.to(torch.bfloat16), 8, b, score="sigmoid", n_group=g, topk_group=4 if g > 1 else 1, group_score=gs)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid", "sqrtsoftplus"])
def test_topk_masks(dtype, score):
    """Rows masked in part and whole by -inf, NaN and the type's lowest value; +inf counts as the largest."""
    _need_gpu()
    gen = torch.Generator().manual_seed(5)
    logits = torch.randn(12, 64, generator=gen).to(dtype)
    low = torch.finfo(dtype).min
    logits[0] = -math.inf
    logits[1] = low
    logits[2] = math.nan
    logits[3, :62] = -math.inf
    logits[4, ::2] = low
    logits[5, 8:] = math.nan
    logits[6, 7] = math.inf if score != "sqrtsoftplus" else 3.0
    logits[7, :32] = -math.inf
    logits[8] = 0
    for b in (None, 0.1 * torch.randn(64, generator=gen)):
        for g, kept in ((1, 1), (8, 3)):
            for gs in ("max", "top2"):
                _check(logits, 6, b, score=score, n_group=g, topk_group=kept, group_score=gs)


@gpu
def test_topk_biases_without_end():
    """-inf keeps experts (whole groups too) behind the others, +inf puts one first; weights are the scores all the same."""
    _need_gpu()
    gen = torch.Generator().manual_seed(8)
    logits = torch.randn(40, 64, generator=gen)
    bias = 0.2 * torch.randn(64, generator=gen)
    bias[::3] = -math.inf
    bias[16:24] = -math.inf
    for g, kept in ((1, 1), (8, 3)):
        for gs in ("max", "top2"):
            _check(logits, 6, bias, n_group=g, topk_group=kept, group_score=gs)
    bias[5] = math.inf
    _check(logits, 6, bias)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("e,g", [(64, 8), (96, 8), (60, 4), (1024, 16)])
def test_topk_groups_with_several_biases_of_inf(e, g, group_score, dtype):
    """Two of a group's experts at +inf, all of them, and several such groups, which come before every other; groups of
    whole lanes and groups that share them."""
    _need_gpu()
    gen = torch.Generator().manual_seed(e)
    s = e // g
    logits = torch.randn(20, e, generator=gen).to(dtype)
    for forced in ([2 * s, 2 * s + 3], list(range(2 * s, 3 * s)), [s, s + 1, 3 * s + 2, 3 * s + 4], [0, 3 * s, 3 * s + 1],
                   list(range(e))):
        bias = 0.2 * torch.randn(e, generator=gen)
        bias[forced] = math.inf
        for kept in (1, 3):
            _check(logits, 4, bias, n_group=g, topk_group=kept, group_score=group_score)


@gpu
@pytest.mark.parametrize("above", [False, True])
def test_topk_softmax_sums_that_lose_their_small_terms(above):
    """Two experts of 1 in lanes whose 31 others, just below 2^-24, are lost in the lane's fp32 sum: the group's score is 1.8e-6
    above the real one, further than one rounding of each value explains. The other group lies between the two, or above."""
    _need_gpu()
    e, g = 1024, 16
    logits = torch.full((1, e), -math.inf)
    logits[0, :64] = math.log(5.9e-8)
    logits[0, 0] = logits[0, 32] = 0.0
    logits[0, 64:128] = -30.0
    bias = torch.zeros(e)
    bias[64] = bias[65] = 0.5 + (1e-7 if above else -0.75e-6)
    _check(logits, 2, bias, score="softmax", n_group=g, topk_group=1, group_score="top2")


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid", "sqrtsoftplus"])
@pytest.mark.parametrize("e,g", [(64, 8), (60, 4), (256, 8), (1024, 16)])
def test_topk_finite_masks_and_large_biases(score, e, g):
    """Biases of -1e9 and fp32's lowest value, on some experts and whole groups, and of 1e9 and 1e30 on a few."""
    _need_gpu()
    gen = torch.Generator().manual_seed(e)
    s = e // g
    logits = 1.5 * torch.randn(16, e, generator=gen)
    for low in (-1e9, torch.finfo(torch.float32).min):
        bias = 0.2 * torch.randn(e, generator=gen)
        bias[::5] = low
        bias[s:2 * s] = low
        for high in (0.1, 1e9, 1e30):
            bias[2 * s + 1] = bias[3 * s + 2] = high
            _check(logits, 6, bias, score=score)
            for gs in ("max", "top2"):
                for kept in (2, g - 1):
                    _check(logits, 6, bias, score=score, n_group=g, topk_group=kept, group_score=gs)


@gpu
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("lo,hi", [(-120, -100), (-160, -80), (-100, 3)])
def test_topk_sqrtsoftplus_of_far_logits(lo, hi, renormalize):
    """e^l is subnormal or 0 where the score, its root, is a plain number."""
    _need_gpu()
    gen = torch.Generator().manual_seed(-lo)
    l = lo + (hi - lo) * torch.rand(9, 64, generator=gen)
    for scale in (1.0, 1e20):
        _check(l, 6, score="sqrtsoftplus", renormalize=renormalize, scale=scale)
        _check(l, 6, (l.mean() / 2).exp() * torch.rand(64, generator=gen), score="sqrtsoftplus", renormalize=renormalize, scale=scale)


@gpu
def test_topk_sigmoids_near_the_end_of_the_range():
    """Scores on both sides of 2^-126, with biases of their size: the selection is still that of the real sums."""
    _need_gpu()
    gen = torch.Generator().manual_seed(1)
    l = -87 - 2 * torch.rand(40, 64, generator=gen)
    _check(l, 6, 1e-38 * torch.rand(64, generator=gen), renormalize=False)
    _check(l, 6, 1e-38 * torch.rand(64, generator=gen), n_group=8, topk_group=3, group_score="top2", renormalize=False)
    l = -75 - 20 * torch.rand(40, 64, generator=gen)
    w, ids = route.topk(l.cuda(), 6, renormalize=False)
    want = 1 / (1 + torch.exp(-l.double().gather(1, ids.cpu())))
    assert bool(((w.cpu().double() - want).abs() <= 16 * 2.0 ** -23 * want + 2.0 ** -149).all())


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid", "sqrtsoftplus"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lo,hi", [(-98, -92), (-300, -90), (-110, 5), (-400, -60)])
def test_topk_renormalised_weights_of_far_logits(score, dtype, lo, hi):
    """Rows whose chosen scores are all subnormal or 0 in fp32 have weights that sum to one all the same; so do the experts
    far below one that a bias of -inf, or its group, leaves out."""
    _need_gpu()
    gen = torch.Generator().manual_seed(-lo)
    l = (lo + (hi - lo) * torch.rand(12, 64, generator=gen)).to(dtype)
    l[1::3, 5] = 12
    l[2, :] = -math.inf
    l[3, 7:] = -math.inf
    l[6, 3:] = -math.inf
    b = torch.zeros(64)
    b[5] = -math.inf
    for bias in (None, b, b + 0.1 * torch.rand(64, generator=gen)):
        _check(l, 6, bias, score=score, scale=2.5)
        _check(l, 6, bias, score=score, n_group=8, topk_group=3, group_score="top2")
    w, _ = route.topk(l.cuda(), 6, bias=b.cuda(), score=score)
    total = w.double().sum(1).cpu()
    assert bool(((total - 1).abs() <= 6 * 2.0 ** -23)[[i for i in range(12) if i != 2]].all()) and float(total[2]) == 0


@gpu
@pytest.mark.parametrize("copies", [1, 2, 3, 17, 40])
@pytest.mark.parametrize("k", [1, 2, 5, 16])
def test_topk_equal_experts_before_a_better_one(copies, k):
    """Experts of one logit and bias, whose fp32 sums are also that of experts behind them that are a little better: the equal
    ones are in order among themselves, and still behind those."""
    _need_gpu()
    logits = torch.full((1, 128), -2.0)
    bias = torch.zeros(128)
    logits[0, :copies], bias[:copies] = -0.25, 0.562176525592804            # 1.0000000247
    logits[0, 60:63], bias[60:63] = 0.5, 0.3775407075881958                 # 1.0000000388
    logits[0, 100:100 + copies // 3], bias[100:100 + copies // 3] = -0.25, 0.562176525592804
    for g, kept in ((1, 1), (8, 8)):
        _check(logits, k, bias, n_group=g, topk_group=kept)


@gpu
@pytest.mark.parametrize("e,g", [(64, 8), (60, 4), (16, 8)])
def test_topk_group_sums_below_the_range(e, g):
    """Groups whose two best have a bias of fp32's lowest value come behind the others and before masked ones, in the order of
    their real sums."""
    _need_gpu()
    gen = torch.Generator().manual_seed(e)
    s = e // g
    logits = torch.randn(12, e, generator=gen)
    low = torch.finfo(torch.float32).min
    bias = torch.full((e,), low)
    for own, factor in ((0, 1.0), (1, 1.0), (1, 0.75), (2, 0.75)):
        b = bias.clone()
        b[:own * s] = 0.1 * torch.randn(own * s, generator=gen)
        b[s * (g - 1):] = low * factor
        l = logits.clone()
        l[3:6, s:2 * s] = -math.inf
        l[6:9, s + 1:2 * s] = -math.inf
        l[9:, : s * (g - 1)] = -math.inf
        for kept in range(1, g):
            _check(l, min(6, kept * s), b, n_group=g, topk_group=kept, group_score="top2")


@gpu
def test_topk_strides_and_large_batches():
    _need_gpu()
    gen = torch.Generator().manual_seed(6)
    base = torch.randn(40, 300, generator=gen)
    _check(base[::2, :256], 8)
    _check(base[:, 1:257], 8)
    _check(base[:1].expand(5, 300), 4, score="softmax")
    _check(base.t()[:64].contiguous().t()[:8], 4)
    logits = torch.randn(20000, 64, generator=gen)
    bias = torch.randn(64, generator=gen)
    w, ids = route.topk(logits.cuda(), 6, bias=bias.cuda())
    pick = torch.sigmoid(logits.double()) + bias.double()
    want = torch.sort(pick, dim=1, descending=True, stable=True).indices[:, :6]
    assert torch.equal(ids.cpu(), want)
    assert route.topk(logits[:0].cuda(), 6)[1].shape == (0, 6)


@gpu
@pytest.mark.parametrize("t,k,e", [(0, 2, 4), (1, 1, 1), (3, 4, 16), (256, 8, 256), (257, 8, 7), (700, 8, 1024), (1024, 8, 256), (1025, 8, 256), (2048, 8, 64), (2049, 8, 64),
                                   (5000, 3, 100), (9000, 8, 1024), (16384, 8, 60), (16385, 8, 60), (40000, 9, 1), (50001, 16, 1001)])
def test_expert_order(t, k, e):
    _need_gpu()
    gen = torch.Generator().manual_seed(t + e)
    ids = (torch.rand(t, k, generator=gen) ** 2 * e).long()
    if t > 2:
        ids[1] = -1
        ids[2, 0] = e
        ids[0] = ids[0, 0]      # the same expert in every slot
    o = route.expert_order(ids.cuda(), e)
    offsets, tokens, places = P.order(ids, e) if t * k * e < 3_000_000 else _order_fast(ids, e)
    assert o.offsets.tolist() == offsets
    assert o.tokens.tolist() == tokens
    assert o.places.reshape(-1).tolist() == places


@gpu
def test_expert_order_of_many_pairs():
    """30 M pairs: the counts of 14649 blocks."""
    _need_gpu()
    gen = torch.Generator(device="cuda").manual_seed(3)
    ids = torch.randint(-1, 256, (3_000_000, 10), generator=gen, device="cuda")
    o = route.expert_order(ids, 256)
    flat = ids.reshape(-1)
    counts = torch.bincount(flat[flat >= 0], minlength=256)
    assert torch.equal(o.offsets[1:].long(), counts.cumsum(0)) and int(o.offsets[0]) == 0
    at = torch.sort(torch.where(flat >= 0, flat, 256), stable=True).indices
    n = int(counts.sum())
    assert torch.equal(o.tokens[:n].long(), at[:n] // 10) and bool((o.tokens[n:] == -1).all())
    places = torch.full_like(flat, -1)
    places[at[:n]] = torch.arange(n, device="cuda")
    assert torch.equal(o.places.reshape(-1).long(), places)


def _order_fast(ids, e):
    flat = ids.reshape(-1)
    good = (flat >= 0) & (flat < e)
    at = torch.sort(torch.where(good, flat, e), stable=True).indices
    n = int(good.sum())
    places = torch.full_like(flat, -1)
    places[at[:n]] = torch.arange(n)
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), torch.bincount(flat[good], minlength=e).cumsum(0)])
    return offsets.tolist(), (at[:n] // ids.shape[1]).tolist() + [-1] * (flat.numel() - n), places.tolist()


def test_refusals_of_the_python_calls():
    l = torch.zeros(2, 8)
    for call in (lambda: route.topk(l, 2), lambda: route.topk(l, 2, score="relu"), lambda: route.topk(l, 2, group_score="mean"),
                 lambda: route.expert_order(torch.zeros(2, 2, dtype=torch.int64), 4)):
        with pytest.raises(ValueError):
            call()


@gpu
def test_refusals_of_tensors():
    _need_gpu()
    l = torch.zeros(2, 8, device="cuda")
    for kw in (dict(bias=torch.zeros(7, device="cuda")), dict(bias=torch.zeros(8)), dict(bias=torch.zeros(8, device="cuda").half())):
        with pytest.raises(ValueError):
            route.topk(l, 2, **kw)
    for kw in (dict(n_group=3), dict(n_group=4, topk_group=5), dict(n_group=4, topk_group=0)):
        with pytest.raises(Exception, match="n_group"):
            route.topk(l, 2, **kw)
    for k in (0, 17, 9):
        with pytest.raises(Exception, match="topk"):
            route.topk(l, k)
    with pytest.raises(Exception, match="topk"):
        route.topk(l, 3, n_group=4, topk_group=1)
    with pytest.raises(Exception, match="1024"):
        route.topk(torch.zeros(1, 1025, device="cuda"), 2)
    with pytest.raises(ValueError):
        route.expert_order(torch.zeros(2, 2, dtype=torch.int32, device="cuda"), 4)
    with pytest.raises(Exception, match="1024"):
        route.expert_order(torch.zeros(2, 2, dtype=torch.int64, device="cuda"), 1025)
    for k in (2 ** 32 + 1, -2 ** 40):       # not cut to 32 bits, and nothing of that size is allocated
        with pytest.raises(Exception, match="topk"):
            route.topk(l, k)
    with pytest.raises(Exception, match="n_group"):
        route.topk(l, 2, n_group=2 ** 32 + 1)
    with pytest.raises(Exception, match="1024"):
        route.expert_order(torch.zeros(2, 2, dtype=torch.int64, device="cuda"), 2 ** 40)
