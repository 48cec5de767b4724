"""shard_b200.fp4 (W4A4) against plain 64-bit forms.

Quantisation and its inverse are compared exactly. The products' tolerance, with S = sum_k |a_k w_k|: the
tensor core adds K / 64 partial sums in fp32, each with an error of at most 2^-22 of the sums involved
(<= S); the epilogue rounds twice in fp32 and once to the output type:

    |y - exact| <= (K / 64 + 2) 2^-22 S + (eps_out / 2 + 2^-23) |exact|
"""
import math
import types

import pytest
import torch

import fp4_plain as P
from shard_b200 import formats as F
from shard_b200 import fp4, route

NV, MX = F.FMT_NVFP4, F.FMT_MXFP4
gpu = pytest.mark.gpu


def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _acts(m, k, dtype, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, k, generator=g) * torch.exp(spread * torch.randn(m, 1, generator=g))).to(dtype)


def _check_quant(x, q, fmt, ts=None):
    codes, sb, t = P.quant(x, fmt, ts)
    assert torch.equal(q.canonical_scales().cpu(), sb), "block scales"
    if t is not None:
        assert torch.equal(q.ts.cpu(), t), "row scales"
    got = P.unpack(q.codes)
    # a zero's sign is not part of its value
    zero = (codes & 7) == 0
    assert torch.equal(torch.where(zero, 0, got & 7), torch.where(zero, 0, codes & 7)) and \
        torch.equal(torch.where(zero, 0, got), torch.where(zero, 0, codes)), "codes"
    return codes, sb, t


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 17), (5, 32), (2, 100), (130, 96), (33, 1056), (3, 7168), (1, 65536)])
def test_quant_and_dequant_are_exact(fmt, dtype, m, k):
    _need_gpu()
    x = _acts(m, k, dtype, seed=m + k)
    q = fp4.quant(x.cuda(), fmt)
    codes, sb, t = _check_quant(x, q, fmt)
    v = P.values(codes, sb, fmt, t)[:, :k]
    y = fp4.dequant(q, torch.float32).cpu()
    assert torch.equal(y, v.float())          # code * scale is exact, times ts rounds once
    for out in (torch.bfloat16, torch.float16):
        # fp32 first, then the output type: at most one step apart from rounding once, half a step off
        d = (fp4.dequant(q, out).cpu().double() - v).abs()
        lim = v.abs() * (torch.finfo(out).eps / 2 + 2.0 ** -24) + torch.finfo(out).smallest_normal * torch.finfo(out).eps
        assert bool((d <= lim)[v.abs() < torch.finfo(out).max].all())


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k", [(3, 16), (5, 48), (40, 1040), (700, 4112)])
def test_rows_that_end_inside_a_block_of_32(fmt, dtype, m, k):
    """K = 16 more than a multiple of 32, loads of 16 bytes; the last half block is the largest, or not finite."""
    _need_gpu()
    x = _acts(m, k, dtype, seed=k)
    x[1, -16:] *= 64
    x[2, -1] = math.inf
    _check_quant(x, fp4.quant(x.cuda(), fmt), fmt)
    rows = torch.tensor([0, m, 2, -1, 1], dtype=torch.int32)
    q = fp4.quant(x.cuda(), fmt, rows=rows.cuda())
    z = torch.cat([x, x.new_zeros(1, k)])[[0, m, 2, m, 1]]
    _check_quant(z, q, fmt)
    w = fp4.quant(_acts(24, k, dtype, seed=1).cuda(), fmt)
    y = fp4.gemm(q, w, out_dtype=torch.float32)
    assert bool((y[[1, 3]] == 0).all()) and bool(y[2].isnan().all()) and bool(y[[0, 4]].isfinite().all())


@gpu
@pytest.mark.parametrize("ts", [1.0, 0.0148810, 2.0 ** -10, 3.4e-38, 1e-42, 1e30])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quant_with_a_calibrated_scale(ts, dtype):
    """Powers of two put many values exactly on a border; tiny and huge scales leave fp32's range."""
    _need_gpu()
    x = _acts(37, 256, dtype, seed=7, spread=1.0)
    if ts < 1e-30 or ts > 1e20:
        x = (x.double() * ts * 100).to(dtype)
    t = torch.tensor([ts], dtype=torch.float32)
    q = fp4.quant(x.cuda(), NV, tensor_scale=t.cuda())
    _check_quant(x, q, NV, t)


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
def test_quant_borders(fmt):
    """Values on the borders between codes and one fp32 step to either side, under scales that divide
    them exactly and scales that do not."""
    _need_gpu()
    rows = []
    for s in (1.0, 0.75, 1 / 3, 1.1, 2.0 ** -20, 7e4):
        mids = torch.tensor(F.E2M1_MID, dtype=torch.float64) * s
        r = [torch.tensor([6.0 * s], dtype=torch.float64), mids, -mids]
        f = torch.cat(r).float()
        up, dn = torch.nextafter(f, torch.tensor(math.inf)), torch.nextafter(f, torch.tensor(-math.inf))
        for v in (f, up, dn):
            v = v.clone()
            v[0] = f[0]
            rows.append(torch.cat([v, f[:1]]))
    x = torch.stack(rows)                       # [18, 16]
    x = torch.cat([x, x.flip(1)], 1)
    ts = torch.tensor([0.4], dtype=torch.float32)
    _check_quant(x, fp4.quant(x.cuda(), fmt), fmt)
    if fmt == NV:
        _check_quant(x, fp4.quant(x.cuda(), fmt, tensor_scale=ts.cuda()), fmt, ts)


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
def test_quant_of_empty_tiny_and_non_finite(fmt):
    _need_gpu()
    x = _acts(9, 128, torch.float32, seed=3)
    x[0] = 0
    x[1, 40] = math.nan
    x[2, 0], x[2, 127] = math.inf, -math.inf
    x[3] = 1e-45
    x[4] = torch.finfo(torch.float32).max
    x[5] = torch.finfo(torch.float32).min
    x[6, 16:] = 0
    x[7] = math.nan
    x[8] = 2.0 ** -126
    q = fp4.quant(x.cuda(), fmt)
    codes, sb, t = _check_quant(x, q, fmt)
    y = fp4.dequant(q, torch.float32).cpu()
    g = 16 if fmt == NV else 32
    bad = (~torch.isfinite(x)).view(9, -1, g).any(-1).repeat_interleave(g, 1)
    assert torch.equal(torch.isnan(y), bad)
    assert bool((y[0] == 0).all())
    b = x[:3].to(torch.bfloat16)
    _check_quant(b, fp4.quant(b.cuda(), fmt), fmt)
    assert fp4.quant(torch.empty(0, 64, device="cuda", dtype=torch.bfloat16), fmt).rows == 0


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
def test_quant_strides_gather_and_shape(fmt):
    _need_gpu()
    base = _acts(40, 333, torch.bfloat16, seed=5).cuda()
    for x in (base[::3], base[:, 1:], base[:, 8:264], base[:1].expand(6, 333), base.t()[:64], base[5:6]):
        _check_quant(x.cpu(), fp4.quant(x, fmt), fmt)
    x3 = base[:, :320].reshape(4, 10, 320)
    q = fp4.quant(x3, fmt)
    assert q.shape == (4, 10) and fp4.dequant(q).shape == (4, 10, 320)
    rows = torch.tensor([3, 3, 39, -1, 0, 40, 17], dtype=torch.int32)
    want = torch.stack([base[r].cpu() if 0 <= r < 40 else torch.zeros(333, dtype=torch.bfloat16) for r in rows.tolist()])
    _check_quant(want, fp4.quant(base, fmt, rows=rows.cuda()), fmt)
    wide = base[:, :320].contiguous()         # rows of whole 16-byte vectors, and sources of NaN beside a missing row
    wide[0] = math.nan
    want = torch.stack([wide[r].cpu() if 0 <= r < 40 else torch.zeros(320, dtype=torch.bfloat16) for r in rows.tolist()])
    _check_quant(want, fp4.quant(wide, fmt, rows=rows.cuda()), fmt)
    none = fp4.quant(wide[:0], fmt, rows=rows.cuda())      # no row exists
    assert bool((fp4.dequant(none) == 0).all())


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
@pytest.mark.parametrize("k,n", [(33, 300), (33, 70000), (160, 27000), (320, 14000), (2080, 2100)])
@pytest.mark.parametrize("calibrated", [False, True])
def test_quant_of_rows_taken_often(fmt, k, n, calibrated):
    """Source rows taken several times (many values: quantised once and copied): with groups, missing rows and rows
    behind the last group, the operand is the one of the rows gathered first."""
    _need_gpu()
    if calibrated and fmt == MX:
        return                                  # MXFP4 has no tensor scale
    x = _acts(7, k, torch.bfloat16, seed=k).cuda()
    g = torch.Generator().manual_seed(k)
    rows = torch.randint(-1, 8, (n,), generator=g).to(torch.int32)
    ts = torch.tensor([0.01], device="cuda") if calibrated else None
    src = torch.cat([x.cpu(), torch.zeros(2, k, dtype=torch.bfloat16)])      # rows 7 and -1 (8) are missing ones
    want = src[rows.long()]
    _check_quant(want, fp4.quant(x, fmt, tensor_scale=ts, rows=rows.cuda()), fmt, None if ts is None else ts.cpu())
    off = torch.tensor([0, 5, 5, 140, n - 2], dtype=torch.int32, device="cuda")
    a = fp4.quant(x, fmt, tensor_scale=ts, rows=rows.cuda(), offsets=off)
    b = fp4.quant(want.cuda(), fmt, tensor_scale=ts, offsets=off)
    codes, s, t, _ = P.weights(fmt, 96, -(-k // 32) * 32, seed=1, mats=4)
    bank = fp4.pack(fmt, codes.cuda(), s.cuda(), None if t is None else t.cuda())
    bank.k = k
    assert torch.equal(fp4.grouped_gemm(a, bank)[:n - 2], fp4.grouped_gemm(b, bank)[:n - 2])


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
def test_quant_rows_do_not_depend_on_the_batch(fmt):
    _need_gpu()
    x = _acts(300, 2080, torch.bfloat16, seed=9).cuda()
    whole = fp4.dequant(fp4.quant(x, fmt), torch.float32)
    for r in (0, 129, 299):
        assert torch.equal(fp4.dequant(fp4.quant(x[r:r + 1], fmt), torch.float32)[0], whole[r])


def _tol(av, wv, exact, k, out):
    s = av.abs() @ wv.abs().T
    return (k / 64 + 2) * 2.0 ** -22 * s + (torch.finfo(out).eps / 2 + 2.0 ** -23) * exact.abs()


def _values(q):
    return P.values(P.unpack(q.codes), q.canonical_scales().cpu(), q.fmt, q.ts)


SHAPES = [(1, 1, 32), (1, 300, 4096), (7, 31, 64), (8, 128, 96), (9, 129, 1056), (64, 257, 256), (65, 64, 288),
          (129, 256, 160), (192, 130, 512), (193, 128, 320), (257, 384, 64), (400, 100, 2048), (1025, 72, 128)]


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gemm(fmt, m, n, k):
    _need_gpu()
    codes, s, ts, wv = P.weights(fmt, n, k, seed=n + k)
    w = fp4.pack(fmt, codes[0].cuda(), s[0].cuda(), None if ts is None else ts[0].cuda())
    a = fp4.quant(_acts(m, k, torch.bfloat16, seed=m).cuda(), fmt)
    av = _values(a)
    exact = av @ wv[0].T
    for out in (torch.float32, torch.bfloat16):
        y = fp4.gemm(a, w, out_dtype=out).cpu().double()
        assert bool(((y - exact).abs() <= _tol(av, wv[0], exact, k, out)).all())
    # fp16's range ends early: a tensor scale that keeps the outputs inside it
    y = fp4.gemm(a, w, out_dtype=torch.float16).cpu().double()
    fits = exact.abs() < 6e4
    lim = _tol(av, wv[0], exact, k, torch.float16) + 2.0 ** -25
    assert bool(((y - exact).abs() <= lim)[fits].all())
    assert fp4.device_error() == 0


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
@pytest.mark.parametrize("m,n,k", [(150, 19000, 64), (300, 12808, 96), (513, 8200, 160), (3000, 1300, 544), (1000, 5000, 2080),
                                   (1500, 8196, 288), (2000, 4096, 4096)])
def test_gemm_of_many_tiles(fmt, m, n, k):
    """Tiles for more than one round of the SMs: pairs of CTAs, one to several tiles each, token tiles of 129 to 256."""
    _need_gpu()
    w = fp4.quant(_acts(n, k, torch.bfloat16, seed=n, spread=0.5).cuda(), fmt)
    a = fp4.quant(_acts(m, k, torch.bfloat16, seed=m).cuda(), fmt)
    av, wv = _values(a).cuda(), _values(w).cuda()
    exact = av @ wv.T
    for out in (torch.float32, torch.bfloat16):
        buf = torch.full((m + 1, n + 8), 3.0, dtype=out, device="cuda")
        y = fp4.gemm(a, w, out_dtype=out, out=buf[:m, :n])
        assert bool(((y.double() - exact).abs() <= _tol(av, wv, exact, k, out)).all())
        assert bool((buf[m:] == 3).all()) and bool((buf[:, n:] == 3).all())
    assert fp4.device_error() == 0


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
@pytest.mark.parametrize("w13", [False, True])
@pytest.mark.parametrize("counts,n,k", [([300, 0, 513, 190, 64, 1000, 1, 257], 2064, 160), ([256, 512, 768, 255, 257], 2048, 1024),
                                        ([0, 0, 0, 900], 6160, 96)])
def test_grouped_gemm_of_many_tiles(fmt, w13, counts, n, k):
    """Pairs of CTAs on groups of every width of tile; errors of the gated form as in test_grouped_gemm."""
    _need_gpu()
    e, p = len(counts), sum(counts)
    codes, s, ts, wv = P.weights(fmt, n, k, seed=k, mats=e, halves=2 if w13 else 1)
    bank = fp4.pack(fmt, codes.cuda(), s.cuda(), None if ts is None else ts.cuda(), kind=fp4.W13 if w13 else fp4.PLAIN)
    off = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    x = (_acts(p, k, torch.bfloat16, seed=p, spread=0.3) * 0.02).to(torch.bfloat16)
    a = fp4.quant(x.cuda(), fmt, offsets=off.cuda())
    c, sb, t = P.quant(x, fmt)
    av = P.values(c, sb, fmt, t).cuda()
    limit = 2.5 if w13 else 0.0
    for out in (torch.float32, torch.bfloat16):
        y = fp4.grouped_gemm(a, bank, out_dtype=out, limit=limit).double()
        for i in range(e):
            lo, hi = int(off[i]), int(off[i + 1])
            w = wv[i].cuda()
            r = av[lo:hi] @ w.T
            tol = _tol(av[lo:hi], w, r, k, torch.float32 if w13 else out)
            if w13:
                g, u = r[:, :n // 2].clamp_max(limit), r[:, n // 2:].clamp(-limit, limit)
                dg, du = tol[:, :n // 2], tol[:, n // 2:]
                silu = g / (1 + torch.exp(-g))
                r = silu * u
                # (g below -64: silu's own size bounds what the fast exponential can add)
                tol = 1.1 * dg * u.abs() + silu.abs() * du + (2.0 ** -19 + torch.finfo(out).eps / 2) * r.abs() * (g > -64) + \
                    1.01 * r.abs() * (g <= -64) + 1e-26
            assert bool(((y[lo:hi] - r).abs() <= tol).all())
    assert fp4.device_error() == 0


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
@pytest.mark.parametrize("calibrated", [False, True])
def test_gemm_of_two_quantised_matrices(fmt, calibrated):
    """K 100: both operands are padded to 128 with zero codes. Tensor scales: one, or one per row of either."""
    _need_gpu()
    x, wx = _acts(20, 100, torch.bfloat16, seed=1, spread=0.5), _acts(150, 100, torch.float32, seed=2, spread=0.5)
    ts = torch.tensor([0.02], device="cuda") if fmt == NV and calibrated else None
    a, w = fp4.quant(x.cuda(), fmt, tensor_scale=ts), fp4.quant(wx.cuda(), fmt, tensor_scale=ts)
    av, wv = _values(a), _values(w)
    exact = av @ wv.T
    y = fp4.gemm(a, w, out_dtype=torch.float32).cpu().double()
    assert bool(((y - exact).abs() <= _tol(av, wv, exact, 128, torch.float32)).all())
    one = fp4.gemm(fp4.quant(x[0].cuda(), fmt, tensor_scale=ts), w)      # a vector
    assert one.shape == (150,) and torch.equal(one, fp4.gemm(a, w)[0])


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
def test_gemm_output_rows_and_non_finite_blocks(fmt):
    _need_gpu()
    codes, s, ts, wv = P.weights(fmt, 136, 256, seed=4)
    w = fp4.pack(fmt, codes[0].cuda(), s[0].cuda(), None if ts is None else ts[0].cuda())
    x = _acts(21, 256, torch.bfloat16, seed=4)
    clean = fp4.gemm(fp4.quant(x.cuda(), fmt), w)
    x[5, 77] = math.inf
    a = fp4.quant(x.cuda(), fmt)
    buf = torch.full((21, 200), 7.0, dtype=torch.bfloat16, device="cuda")
    y = fp4.gemm(a, w, out=buf[:, 3:139])
    assert y.data_ptr() == buf[:, 3:139].data_ptr()
    assert bool((buf[:, :3] == 7).all()) and bool((buf[:, 139:] == 7).all())
    assert bool(torch.isnan(y[5]).all()), "the row that held an infinity is NaN"
    keep = [i for i in range(21) if i != 5]
    assert torch.equal(y[keep], clean[keep]), "and no other row is touched"


@gpu
def test_gemm_rows_do_not_depend_on_the_batch():
    _need_gpu()
    codes, s, ts, _ = P.weights(NV, 256, 1024, seed=8)
    w = fp4.pack(NV, codes[0].cuda(), s[0].cuda(), ts[0].cuda())
    x = _acts(17, 1024, torch.bfloat16, seed=8).cuda()
    whole = fp4.gemm(fp4.quant(x, NV), w)
    for r in (0, 9, 16):
        assert torch.equal(fp4.gemm(fp4.quant(x[r:r + 1], NV), w)[0], whole[r])


COUNTS = [[5], [0, 3, 0, 0, 1], [127, 128, 129, 1, 0, 64], [300, 0, 193], [0, 0], [1] * 40, [700, 5, 0, 260]]


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
@pytest.mark.parametrize("w13", [False, True])
@pytest.mark.parametrize("counts", COUNTS)
def test_grouped_gemm(fmt, w13, counts):
    """Rows in groups of any size, two rows behind the last group, with weights and a clamp for w13 banks.
    silu(g) u of values with errors dg, du: off by 1.1 dg |u| + |silu(g)| du, and 2^-19 of the result for
    the fast exponential and division at |g| <= 64."""
    _need_gpu()
    e, n, k = len(counts), 144, 224
    codes, s, ts, wv = P.weights(fmt, n, k, seed=e, mats=e, halves=2 if w13 else 1)
    bank = fp4.pack(fmt, codes.cuda(), s.cuda(), None if ts is None else ts.cuda(), kind=fp4.W13 if w13 else fp4.PLAIN)
    p = sum(counts) + 2
    off = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    x = _acts(p, k, torch.bfloat16, seed=p, spread=0.3) * 0.05
    x = x.to(torch.bfloat16)
    a = fp4.quant(x.cuda(), fmt, offsets=off.cuda())
    c, sb, t = P.quant(x, fmt)
    assert torch.equal(P.unpack(a.codes)[:p - 2] & 7, c[:p - 2] & 7)
    av = P.values(c, sb, fmt, t)
    rw = torch.rand(p, generator=torch.Generator().manual_seed(1)) + 0.5
    width = n // 2 if w13 else n
    out = torch.full((p, width + 5), 3.0, device="cuda")
    limit = 2.5 if w13 else 0.0
    y = fp4.grouped_gemm(a, bank, out_dtype=torch.float32, row_weight=rw.cuda(), limit=limit, out=out[:, :width])
    y = y.cpu().double()
    assert bool((out[p - 2:] == 3).all()) and bool((out[:, width:] == 3).all()), "rows behind the last group stay"
    for i in range(e):
        lo, hi = int(off[i]), int(off[i + 1])
        if lo == hi:
            continue
        r = av[lo:hi] @ wv[i].T
        tol = _tol(av[lo:hi], wv[i], r, k, torch.float32)
        if w13:
            g, u = r[:, :n // 2], r[:, n // 2:]
            dg, du = tol[:, :n // 2], tol[:, n // 2:]
            g, u = g.clamp_max(limit), u.clamp(-limit, limit)
            silu = g / (1 + torch.exp(-g))
            assert float(g.abs().max()) < 64
            r, tol = silu * u, 1.1 * dg * u.abs() + silu.abs() * du + 2.0 ** -19 * (silu * u).abs() + 1e-30
        r, tol = r * rw[lo:hi, None].double(), tol * rw[lo:hi, None].double() + 2.0 ** -22 * r.abs()
        assert bool(((y[lo:hi] - r).abs() <= tol).all()), f"expert {i}"
    assert fp4.device_error() == 0


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
def test_groups_that_begin_late(fmt):
    """Offsets of some of the experts of an order: rows before the first group and behind the last are left alone."""
    _need_gpu()
    codes, s, ts, _ = P.weights(fmt, 64, 128, seed=6, mats=6)
    one = lambda lo, hi: fp4.pack(fmt, codes[lo:hi].cuda(), s[lo:hi].cuda(), None if ts is None else ts[lo:hi].cuda())  # noqa: E731
    x = _acts(400, 128, torch.bfloat16, seed=6).cuda()
    off = torch.tensor([0, 130, 131, 131, 290, 300, 400], dtype=torch.int32, device="cuda")
    whole = fp4.grouped_gemm(fp4.quant(x, fmt, offsets=off), one(0, 6))
    part = off[1:5].contiguous()
    out = torch.full((400, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    fp4.grouped_gemm(fp4.quant(x, fmt, offsets=part), one(1, 4), out=out)
    assert torch.equal(out[130:290], whole[130:290])
    assert bool((out[:130] == 5).all()) and bool((out[290:] == 5).all())


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
def test_pack_reads_the_canonical_form(fmt):
    """Tiling and back; a plain product equals one with the operand that quant makes of the same values."""
    _need_gpu()
    codes, s, ts, _ = P.weights(fmt, 300, 160, seed=2, mats=3)
    w = fp4.pack(fmt, codes.cuda(), s.cuda(), None if ts is None else ts.cuda())
    assert torch.equal(w.canonical_scales().cpu(), s.view(900, -1)) and w.codes.data_ptr() != 0
    v = fp4.pack(fmt, codes.cuda(), s.cuda(), kind=fp4.W13)
    inter = torch.stack([s[:, :150], s[:, 150:]], 2).reshape(900, -1)
    assert torch.equal(v.canonical_scales().cpu(), inter)


@gpu
@pytest.mark.parametrize("m,n,k", [(5, 256, 64), (5, 256, 4096), (300, 256, 1024), (1024, 8192, 256)])
def test_products_whose_waits_run_out(m, n, k):
    """A consumer's wait that gives up at its first probe (one CTA a tile, K over a cluster, several tiles, CTA pairs):
    the call ends, the error word says so, and the next call is whole again."""
    _need_gpu()
    from shard_b200 import _lib
    L = _lib.lib()
    codes, s, ts, _ = P.weights(NV, n, k, seed=1)
    w = fp4.pack(NV, codes[0].cuda(), s[0].cuda(), ts[0].cuda())
    a = fp4.quant(_acts(m, k, torch.bfloat16).cuda(), NV)
    want = fp4.gemm(a, w)
    assert fp4.device_error() == 0
    try:
        assert L.sb_debug_set_wait_limit(1) == 0
        fp4.gemm(a, w)
        torch.cuda.synchronize()
    finally:
        assert L.sb_debug_set_wait_limit(0) == 0
    assert fp4.device_error() == 1 and fp4.device_error() == 0
    assert torch.equal(fp4.gemm(a, w), want)
    assert fp4.device_error() == 0


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
def test_pack_and_dequant_of_a_weight(fmt):
    _need_gpu()
    codes, s, ts, v = P.weights(fmt, 70, 96, seed=3)
    w = fp4.pack(fmt, codes[0].cuda(), s[0].cuda(), None if ts is None else ts[0].cuda())
    y = fp4.dequant(w, torch.float32).cpu()
    # P.weights applies the tensor scale in 64 bits: the kernel rounds that product once
    assert torch.equal(y, v[0].float())


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
def test_a_bank_of_one_matrix(fmt):
    _need_gpu()
    codes, s, ts, _ = P.weights(fmt, 80, 96, seed=4, mats=1)
    bank = fp4.pack(fmt, codes.cuda(), s.cuda(), None if ts is None else ts.cuda())
    x = _acts(70, 96, torch.bfloat16, seed=4).cuda()
    plain = fp4.gemm(fp4.quant(x, fmt), bank)
    off = torch.tensor([0, 70], dtype=torch.int32, device="cuda")
    assert torch.equal(fp4.grouped_gemm(fp4.quant(x, fmt, offsets=off), bank), plain)


@gpu
def test_calls_on_two_streams_at_once():
    """Products of all three forms and a large order, in flight on two streams: each gives what it gives alone."""
    _need_gpu()
    x = _acts(2048, 4096, torch.bfloat16, seed=2).cuda()
    w = fp4.quant(_acts(4096, 4096, torch.bfloat16, seed=3).cuda())
    ids = torch.randint(0, 256, (40000, 8), device="cuda")
    off = torch.tensor([0, 700, 701, 2048], dtype=torch.int32, device="cuda")
    bank = fp4.pack(NV, w.codes.view(1, 4096, -1).repeat(3, 1, 1), w.canonical_scales().view(1, 4096, -1).repeat(3, 1, 1))

    def work():
        return [fp4.gemm(fp4.quant(x[:m]), w) for m in (1, 40, 2048)] + \
            [fp4.grouped_gemm(fp4.quant(x, offsets=off), bank), *route.expert_order(ids, 256)]

    want = work()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for st, g in zip(streams, got):
            with torch.cuda.stream(st):
                g.append(work())
    torch.cuda.synchronize()
    assert fp4.device_error() == 0
    for g in got:
        for outs in g:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


@gpu
def test_gated_rows_of_nan_stay_nan():
    """A clamp does not hide a NaN, and only its row has it."""
    _need_gpu()
    codes, s, ts, _ = P.weights(NV, 64, 64, seed=1, mats=2, halves=2)
    bank = fp4.pack(NV, codes.cuda(), s.cuda(), ts.cuda(), kind=fp4.W13)
    off = torch.tensor([0, 3, 9], dtype=torch.int32, device="cuda")
    x = _acts(9, 64, torch.bfloat16, spread=0.1)
    x[4, 20] = math.nan
    for limit in (0.0, 1.5):
        y = fp4.grouped_gemm(fp4.quant(x.cuda(), NV, offsets=off), bank, limit=limit).cpu()
        assert torch.isnan(y).all(1).tolist() == [i == 4 for i in range(9)]
        assert not bool(torch.isnan(y[[0, 1, 2, 3, 5, 6, 7, 8]]).any())


def test_refusals_of_the_python_calls():
    """Arguments that no kernel may see are refused before the library is touched (no GPU needed)."""
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        fp4.quant(x)                                        # not on a CUDA device
    with pytest.raises(ValueError):
        fp4.quant(x, "fp8")
    with pytest.raises(ValueError):
        fp4.pack("nvfp4", torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8))

    def t(fmt=NV, mats=1, rows=4, k=64, ts=None, offsets=None, kind=fp4.PLAIN):
        z = torch.zeros(1, dtype=torch.uint8)
        return fp4.Fp4Tensor(fmt, mats, rows, k, z, z, ts, offsets, kind, (rows,))

    off = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: fp4.gemm(t(), t(fmt=MX)), lambda: fp4.gemm(t(), t(k=96)), lambda: fp4.gemm(t(), t(mats=2)),
                 lambda: fp4.gemm(t(offsets=off), t()), lambda: fp4.gemm(t(), t(kind=fp4.W13)),
                 lambda: fp4.gemm(t(mats=2), t()), lambda: fp4.gemm(t(), t(), out_dtype=torch.float64),
                 lambda: fp4.grouped_gemm(t(), t(mats=2)), lambda: fp4.grouped_gemm(t(offsets=off), t(mats=3)),
                 lambda: fp4.grouped_gemm(t(offsets=off), t(mats=2), limit=-1.0),
                 lambda: fp4.grouped_gemm(t(offsets=off), t(mats=2), limit=math.nan),
                 lambda: fp4.grouped_gemm(t(offsets=off), t(mats=2), row_weight=torch.ones(3)),
                 lambda: fp4.dequant(t(offsets=off)), lambda: fp4.dequant(t(), torch.float64),
                 lambda: t(offsets=off).canonical_scales()):
        with pytest.raises(ValueError):
            call()


@gpu
def test_refusals_of_tensors():
    _need_gpu()
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    i = torch.zeros(4, dtype=torch.int64, device="cuda")
    for kw in (dict(rows=i), dict(offsets=i), dict(offsets=i[:1].int()), dict(tensor_scale=torch.zeros(2, device="cuda")),
               dict(tensor_scale=torch.zeros(1)), dict(fmt=MX, tensor_scale=torch.ones(1, device="cuda")),
               dict(rows=torch.zeros(4, dtype=torch.int32))):
        with pytest.raises(ValueError):
            fp4.quant(x, **kw)
    with pytest.raises(Exception, match="65536"):
        fp4.quant(torch.zeros(1, 65537, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError):
        fp4.quant(x.double())
    a = fp4.quant(x)
    with pytest.raises(ValueError):
        fp4.gemm(a, a, out=torch.zeros(4, 5, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError):
        fp4.gemm(a, a, out=torch.zeros(4, 4, dtype=torch.bfloat16, device="cuda").t()[:, :])
    other = types.SimpleNamespace(device=torch.device("cuda", 7 if x.device.index != 7 else 0))
    for call in (lambda: fp4.quant(x, stream=other), lambda: fp4.gemm(a, a, stream=other), lambda: fp4.dequant(a, stream=other)):
        with pytest.raises(ValueError, match="stream"):
            call()


def _rows_of_all_sizes(rows, k, lo, hi, seed):
    """Rows from 10^lo to 10^hi, in no order of size."""
    g = torch.Generator().manual_seed(seed)
    size = torch.pow(10.0, torch.linspace(lo, hi, rows, dtype=torch.float64))[torch.randperm(rows, generator=g)]
    return (torch.randn(rows, k, generator=g).clamp(-3, 3) * size[:, None]).float()


# of the output type, behind its fp32 rounding: half a step of its smallest values
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133}


@gpu
@pytest.mark.parametrize("m,n,k", [(1, 64, 64), (5, 256, 4096), (300, 256, 1024), (1024, 8192, 256)])
@pytest.mark.parametrize("ts", [None, 4e-5, 1e-30, 1e28])
def test_gemm_of_tiny_and_huge_rows(m, n, k, ts):
    """The two tensor scales' own product leaves fp32's range where the output does not: rows of either operand near both
    ends of it (or one scale ts of the weights), one of zeros, in every form of the kernel, within _tol."""
    _need_gpu()
    x = _rows_of_all_sizes(m, k, -37.5, 37.5, m) if m > 1 else _rows_of_all_sizes(1, k, -34, -34, 1)
    if m > 3:
        x[2] = 0
    a = fp4.quant(x.cuda(), NV)
    if ts is None:
        wx = _rows_of_all_sizes(n, k, -33, 33, n)
        wx[n // 3] = 0
        w = fp4.quant(wx.cuda(), NV)
        wv = _values(w).cuda()
    else:
        codes, s, _, _ = P.weights(NV, n, k, seed=n + k)
        t = torch.tensor([ts])
        w = fp4.pack(NV, codes[0].cuda(), s[0].cuda(), t.cuda())
        wv = P.values(P.unpack(codes[0]), s[0], NV, t).cuda()
    av = _values(a).cuda()
    exact = av @ wv.T
    for out in (torch.float32, torch.bfloat16):
        tol = _tol(av, wv, exact, k, out) + TINY[out]
        y = fp4.gemm(a, w, out_dtype=out).double()
        fits = exact.abs() + tol < torch.finfo(out).max
        assert float(fits.double().mean()) > 0.3
        assert bool(((y - exact).abs() <= tol)[fits].all())
    assert fp4.device_error() == 0


@gpu
@pytest.mark.parametrize("counts,n,k", [([5, 0, 40, 130], 272, 96), ([513, 256, 0, 600], 2176, 64)])
@pytest.mark.parametrize("w13", [False, True])
def test_grouped_gemm_of_tiny_and_huge_rows(counts, n, k, w13):
    """The same with expert groups, with weights of the rows (0 among them) far from one. Gated rows: the exponential's argument
    is |g| 2^-23 of itself off, it, the division and the products 2^-20; below -87 its reciprocal may count as 0."""
    _need_gpu()
    e, p = len(counts), sum(counts)
    codes, s, _, _ = P.weights(NV, n, k, seed=k, mats=e)
    ts = torch.tensor([[1e-5, 1e30], [1e25, 1e-5], [1.0, 1.0], [1e-30, 1e-20]]) if w13 else torch.tensor([[1e-5], [1e25], [1.0], [1e-30]])
    bank = fp4.pack(NV, codes.cuda(), s.cuda(), ts.cuda(), kind=fp4.W13 if w13 else fp4.PLAIN)
    off = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    x = _rows_of_all_sizes(p, k, -37.5, 37.5, p)
    x[7] = 0
    a = fp4.quant(x.cuda(), NV, offsets=off.cuda())
    c, sb, t = P.quant(x, NV)
    av = P.values(c, sb, NV, t).cuda()
    rw = torch.pow(10.0, torch.linspace(-25, 25, p, dtype=torch.float64))[torch.randperm(p, generator=torch.Generator().manual_seed(1))].float()
    rw[::9] = 0
    rw[1::3] = 0.25
    for out in (torch.float32, torch.bfloat16):
        y = fp4.grouped_gemm(a, bank, out_dtype=out, row_weight=rw.cuda()).double()
        for i in range(e):
            lo, hi = int(off[i]), int(off[i + 1])
            if lo == hi:
                continue
            h = ts.shape[1]
            w = (P.values(P.unpack(codes[i]), s[i], NV).view(h, n // h, k) * ts[i].double().view(h, 1, 1)).view(n, k).cuda()
            f = rw[lo:hi, None].double().cuda()
            r = av[lo:hi] @ w.T
            if w13:
                d = _tol(av[lo:hi], w, r, k, torch.float32) + 2.0 ** -149
                fits = (r.abs() + d < 3e38).view(hi - lo, 2, -1).all(1)
                g, u = r[:, :n // 2], r[:, n // 2:]
                silu = g / (1 + torch.exp(-g))
                q = silu * u
                tol = 1.1 * d[:, :n // 2] * u.abs() + silu.abs() * d[:, n // 2:] + \
                    torch.where(g > -87, (g.abs() * 2.0 ** -23).clamp_max(2.0 ** -16) + 2.0 ** -20, 1.01) * q.abs() + 2.0 ** -149
                fits &= q.abs() < 3e38
            else:
                q, tol = r, _tol(av[lo:hi], w, r, k, torch.float32)
                fits = r.abs() + tol < 3e38
            r, tol = q * f, tol * f + (2.0 ** -23 + torch.finfo(out).eps / 2) * (q * f).abs() + TINY[out]
            fits &= r.abs() + tol < 3e38
            assert float(fits.double().mean()) > 0.1
            assert bool(((y[lo:hi] - r).abs() <= tol)[fits].all()), f"expert {i}"
    assert fp4.device_error() == 0


def test_pack_is_on_its_stream_before_it_touches_a_tensor(monkeypatch):
    """Conversions of the scales belong to the given stream, as the products behind them do (no GPU needed)."""
    class Reached(Exception):
        pass

    class Tensor:
        is_cuda, device = True, torch.device("cuda", 0)

        def dim(self):
            return 2

        def get_device(self):
            return 0

    def elsewhere(device, stream):
        raise Reached

    monkeypatch.setattr(fp4, "_elsewhere", elsewhere)
    with pytest.raises(Reached):
        fp4.pack(NV, Tensor(), Tensor(), Tensor(), stream=object())


@gpu
@pytest.mark.parametrize("kind", [fp4.PLAIN, fp4.W13])
def test_pack_on_a_stream(kind):
    """Tensor scales that have to be converted (64 bits, not contiguous), while the current stream is busy."""
    _need_gpu()
    codes, s, ts, _ = P.weights(NV, 64, 128, seed=3, mats=4, halves=2 if kind == fp4.W13 else 1)
    off = torch.tensor([0, 3, 3, 8, 9], dtype=torch.int32, device="cuda")
    c, sc = codes.cuda(), s.cuda()
    wide = ts.double().repeat(1, 2).cuda()[:, ::2] if kind == fp4.PLAIN else ts.double().t().contiguous().cuda().t()
    a = fp4.quant(_acts(9, 128, torch.bfloat16).cuda(), NV, offsets=off)
    want = fp4.grouped_gemm(a, fp4.pack(NV, c, sc, ts.cuda(), kind=kind))
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    fp4.pack(NV, c, sc, wide, kind=kind, stream=st)      # (what is loaded or allocated at the first call waits for the device)
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)          # about 0.1 s
    got = fp4.grouped_gemm(a, fp4.pack(NV, c, sc, wide, kind=kind, stream=st), stream=st)
    st.synchronize()
    assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
@pytest.mark.parametrize("m,n,k", [(1, 300, 65536), (3, 19000, 16384), (64, 19000, 8224)])
def test_gemm_of_long_rows(fmt, m, n, k):
    """Few tokens against weights that outgrow L2, and the longest K."""
    _need_gpu()
    w = fp4.quant(torch.randn(n, k, generator=torch.Generator("cuda").manual_seed(n), device="cuda", dtype=torch.bfloat16), fmt)
    a = fp4.quant(_acts(m, k, torch.bfloat16, seed=m).cuda(), fmt)
    y = fp4.gemm(a, w, out_dtype=torch.float32).double()
    at = torch.cat([torch.arange(0, n, 97), torch.arange(n - 130, n)])
    wv, av = fp4.dequant(w, torch.float32)[at].double(), fp4.dequant(a, torch.float32).double()
    exact = av @ wv.T
    # (values of 32 bits: each 2^-24 off, two in a product)
    tol = _tol(av, wv, exact, k, torch.float32) + 2.0 ** -22 * (av.abs() @ wv.abs().T)
    assert bool(((y[:, at] - exact).abs() <= tol).all())
    assert fp4.device_error() == 0


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
@pytest.mark.parametrize("k", [33, 64, 4096])
def test_operands_of_no_rows(fmt, k):
    """A batch of no tokens through every call, and its parts' shapes."""
    _need_gpu()
    x = torch.empty(2, 0, k, device="cuda", dtype=torch.bfloat16)
    q = fp4.quant(x, fmt)
    kp = -(-k // 32) * 32
    assert q.codes.shape == (0, kp // 2) and q.canonical_scales().shape == (0, kp // (16 if fmt == NV else 32))
    assert q.ts is None if fmt == MX else q.ts.shape == (0,)
    assert fp4.dequant(q).shape == (2, 0, k)
    w = fp4.quant(_acts(24, k, torch.bfloat16).cuda(), fmt)
    assert fp4.gemm(q, w).shape == (2, 0, 24)
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    codes, s, ts, _ = P.weights(fmt, 24, kp, seed=1, mats=3)
    bank = fp4.pack(fmt, codes.cuda(), s.cuda(), None if ts is None else ts.cuda())
    bank.k = k
    assert fp4.grouped_gemm(fp4.quant(x[0], fmt, offsets=off), bank).shape == (0, 24)
    torch.cuda.synchronize()


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
def test_a_gather_of_no_rows(fmt):
    _need_gpu()
    x = _acts(3, 64, torch.bfloat16).cuda()
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    q = fp4.quant(x, fmt, rows=none)
    assert q.rows == 0 and fp4.dequant(q).shape == (0, 64) and q.codes.shape == (0, 32)
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    codes, s, ts, _ = P.weights(fmt, 24, 64, seed=1, mats=3)
    bank = fp4.pack(fmt, codes.cuda(), s.cuda(), None if ts is None else ts.cuda())
    assert fp4.grouped_gemm(fp4.quant(x, fmt, rows=none, offsets=off), bank).shape == (0, 24)
    o = route.expert_order(torch.empty(0, 2, dtype=torch.int64, device="cuda"), 3)
    assert fp4.grouped_gemm(fp4.quant(x[:0], fmt, rows=o.tokens, offsets=o.offsets), bank).shape == (0, 24)
    torch.cuda.synchronize()


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
def test_pack_of_views(fmt):
    """Codes and scales inside larger buffers: at odd addresses, and every other matrix of a bank."""
    _need_gpu()
    codes, s, ts, _ = P.weights(fmt, 40, 96, seed=5, mats=4)
    t = None if ts is None else ts.cuda()
    off = torch.tensor([0, 3, 3, 8, 9], dtype=torch.int32, device="cuda")
    a = fp4.quant(_acts(9, 96, torch.bfloat16).cuda(), fmt, offsets=off)
    want = fp4.grouped_gemm(a, fp4.pack(fmt, codes.cuda(), s.cuda(), t))

    def inside(v, at):
        b = torch.empty(v.numel() + at, dtype=torch.uint8, device="cuda")
        w = b[at:].view(v.shape)
        w.copy_(v)
        return w

    for at in (1, 8, 16):
        assert torch.equal(fp4.grouped_gemm(a, fp4.pack(fmt, inside(codes, at), inside(s, at), t)), want)
    apart = lambda v: torch.stack([v, v], 1).cuda()[:, 1]  # noqa: E731
    assert torch.equal(fp4.grouped_gemm(a, fp4.pack(fmt, apart(codes), apart(s), t)), want)
    c = codes.cuda()
    assert fp4.pack(fmt, c, s.cuda(), t).codes.data_ptr() == c.data_ptr()


@gpu
@pytest.mark.parametrize("n", [8, 1 << 17])
@pytest.mark.parametrize("ts", [math.nan, 0.0, -1.0, math.inf])
def test_rows_under_a_tensor_scale_that_is_none(ts, n):
    """NaN, in a small gather and in one that quantises its source rows once; missing rows and rows of zeros too."""
    _need_gpu()
    x = _acts(7, 80, torch.bfloat16).cuda()
    x[1] = 0
    rows = torch.arange(n) % 8
    rows = torch.where(rows == 7, -1, rows).to(torch.int32).cuda()
    q = fp4.quant(x, NV, tensor_scale=torch.tensor([ts], device="cuda"), rows=rows)
    assert bool((q.canonical_scales()[:, :5] == 0x7F).all()) and bool(fp4.dequant(q).isnan().all())


@gpu
@pytest.mark.parametrize("offsets", [[0, 5, 3, 9], [9, 0, 9, 0], [0, 9, 9, -4], [0, 2 ** 31 - 1, -2 ** 31, 9]])
def test_offsets_that_descend(offsets):
    """They name rows more than once: nothing is written, and the error word says so. Ends outside the rows are cut."""
    _need_gpu()
    codes, s, ts, _ = P.weights(NV, 40, 64, seed=5, mats=3)
    bank = fp4.pack(NV, codes.cuda(), s.cuda(), ts.cuda())
    x = _acts(9, 64, torch.bfloat16).cuda()
    assert fp4.device_error() == 0
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    out = torch.full((9, 40), 3.0, dtype=torch.bfloat16, device="cuda")
    fp4.grouped_gemm(fp4.quant(x, NV, offsets=off), bank, out=out)
    assert bool((out == 3).all()) and fp4.device_error() == 1 and fp4.device_error() == 0
    good = torch.tensor([0, 4, 9, 9], dtype=torch.int32, device="cuda")
    a = fp4.quant(x, NV, offsets=good)
    want = fp4.grouped_gemm(a, bank)
    a.offsets = torch.tensor([0, 4, 12, 15], dtype=torch.int32, device="cuda")
    assert torch.equal(fp4.grouped_gemm(a, bank)[:9], want) and fp4.device_error() == 0


@gpu
@pytest.mark.parametrize("fmt", [NV, MX])
@pytest.mark.parametrize("e,t,k,n,kind", [(256, 16, 1024, 512, fp4.W13), (384, 16, 512, 256, fp4.PLAIN), (384, 700, 512, 256, fp4.W13),
                                          (1024, 300, 64, 64, fp4.PLAIN)])
def test_banks_of_many_experts(fmt, e, t, k, n, kind):
    """Verify chunks and larger ones over banks of as many experts as layers have, through the order of their routed pairs."""
    _need_gpu()
    h = 2 if kind == fp4.W13 else 1
    codes, s, ts, _ = P.weights(fmt, n, k, seed=e, mats=e, halves=h)
    codes, s, ts = codes.cuda(), s.cuda(), None if ts is None else ts.cuda()
    g = torch.Generator().manual_seed(e + t)
    ids = torch.stack([torch.randperm(e, generator=g)[:8] for _ in range(t)]).cuda()
    o = route.expert_order(ids, e)
    x = (_acts(t, k, torch.bfloat16, seed=t, spread=0.3) * 0.02).to(torch.bfloat16).cuda()
    a = fp4.quant(x, fmt, rows=o.tokens, offsets=o.offsets)
    y = fp4.grouped_gemm(a, fp4.pack(fmt, codes, s, ts, kind=kind), out_dtype=torch.float32).double()
    av = fp4.dequant(fp4.quant(x, fmt), torch.float32).double()[o.tokens.long()]
    off = o.offsets.tolist()
    for i in range(e):
        lo, hi = off[i], off[i + 1]
        if lo == hi:
            continue
        half = lambda v, j: v[i, j * (n // h):(j + 1) * (n // h)]  # noqa: E731
        w = torch.cat([fp4.dequant(fp4.pack(fmt, half(codes, j), half(s, j), None if ts is None else ts[i, j:j + 1]), torch.float32)
                       for j in range(h)]).double()
        r = av[lo:hi] @ w.T
        # (values of 32 bits: each 2^-24 off, two in a product)
        tol = _tol(av[lo:hi], w, r, k, torch.float32) + 2.0 ** -22 * (av[lo:hi].abs() @ w.abs().T)
        if h == 2:
            gate, up, dg, du = r[:, :n // 2], r[:, n // 2:], tol[:, :n // 2], tol[:, n // 2:]
            silu = gate / (1 + torch.exp(-gate))
            r = silu * up
            tol = 1.1 * dg * up.abs() + silu.abs() * du + \
                torch.where(gate > -87, gate.abs() * 2.0 ** -23 + 2.0 ** -20, 1.01) * r.abs() + 2.0 ** -149
        assert bool(((y[lo:hi] - r).abs() <= tol).all()), f"expert {i}"
    assert fp4.device_error() == 0


@gpu
@pytest.mark.parametrize("k", [16, 48, 4112])
def test_pack_of_nvfp4_rows_that_end_inside_a_block_of_32(k):
    """K = 16 more than a multiple of 32: the operand, its values, and products with activations of that K."""
    _need_gpu()
    codes, s, ts, wv = P.weights(NV, 72, k, seed=k, mats=3, halves=2)
    c, sc, t = codes.cuda(), s.cuda(), ts.cuda()
    one = fp4.pack(NV, c[0, :36], sc[0, :36], t[0, :1])
    assert one.k == k and torch.equal(fp4.dequant(one, torch.float32).cpu(), wv[0, :36].float())
    x = (_acts(40, k, torch.bfloat16, seed=k, spread=0.3) * 0.05).to(torch.bfloat16)
    a = fp4.quant(x.cuda(), NV)
    av = _values(a)[:, :k]
    exact = av @ wv[0, :36].T
    assert bool(((fp4.gemm(a, one, out_dtype=torch.float32).cpu().double() - exact).abs()
                 <= _tol(av, wv[0, :36], exact, k, torch.float32)).all())
    off = torch.tensor([0, 7, 7, 40], dtype=torch.int32, device="cuda")
    y = fp4.grouped_gemm(fp4.quant(x.cuda(), NV, offsets=off), fp4.pack(NV, c, sc, t, kind=fp4.W13), out_dtype=torch.float32)
    for i, (lo, hi) in enumerate(((0, 7), (7, 7), (7, 40))):
        r = av[lo:hi] @ wv[i].T
        d = _tol(av[lo:hi], wv[i], r, k, torch.float32)
        gate, up, dg, du = r[:, :36], r[:, 36:], d[:, :36], d[:, 36:]
        silu = gate / (1 + torch.exp(-gate))
        tol = 1.1 * dg * up.abs() + silu.abs() * du + \
            torch.where(gate > -87, gate.abs() * 2.0 ** -23 + 2.0 ** -20, 1.01) * (silu * up).abs() + 2.0 ** -149
        assert bool(((y[lo:hi].cpu().double() - silu * up).abs() <= tol).all())
    with pytest.raises(ValueError, match="32"):
        fp4.pack(MX, c[0], torch.zeros(72, k // 32 + 1, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="16"):
        fp4.pack(NV, c[0, :, :4].contiguous(), sc[0, :, :0].contiguous())
