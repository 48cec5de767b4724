"""C-ABI validation of the fp4 and routing entry points: every refusal comes before any launch, so these run
without a GPU."""
import ctypes

from shard_b200 import _lib
from shard_b200 import formats as F

FAKE = ctypes.c_void_p(1 << 12)   # an aligned address that these calls never dereference
ODD = ctypes.c_void_p((1 << 12) + 8)
NV, MX, FP8 = F.FMT_NVFP4, F.FMT_MXFP4, F.FMT_FP8


def test_scale_bytes():
    f = _lib.lib().sb_fp4_scale_bytes
    assert f(NV, 1, 1, 32, 0) == 512 and f(MX, 1, 1, 32, 0) == 512
    assert f(NV, 1, 129, 4096, 0) == 2 * 64 * 512 and f(MX, 1, 129, 4096, 0) == 2 * 32 * 512
    assert f(NV, 3, 130, 64, 0) == 3 * 2 * 512
    assert f(NV, 1, 300, 64, 7) == (300 // 128 + 7) * 512
    assert f(NV, 1, 1, 33, 0) == 512 and f(MX, 1, 1, 129, 0) == 2 * 512
    for bad in ((FP8, 1, 1, 64, 0), (NV, 0, 1, 64, 0), (NV, 1, -1, 64, 0), (NV, 1, 1, 0, 0), (NV, 1, 1, 65537, 0),
                (NV, 1, 1, 64, 1025), (NV, 2, 1, 64, 3), (NV, 1, 1 << 31, 64, 0)):
        assert f(*bad) == 0


def _quant(fmt=NV, x=FAKE, dtype=0, src=4, k=64, stride=64, rows_in=None, rows=4, ts=None, off=None, groups=0, codes=FAKE,
           scales=FAKE, rs=FAKE, ws=None, n=0):
    return _lib.lib().sb_fp4_quant(fmt, x, dtype, src, k, stride, rows_in, rows, ts, off, groups, codes, scales, rs, ws, n, None)


def test_quant_refusals():
    assert _quant(fmt=FP8) == -3
    assert _quant(dtype=3) == -1
    for kw in (dict(k=0), dict(k=65537), dict(rows=-1), dict(rows=(1 << 30) + 1), dict(src=-1), dict(stride=-1), dict(src=5)):
        assert _quant(**kw) == -2, kw
    for kw in (dict(x=None), dict(codes=None), dict(scales=None), dict(rs=None), dict(codes=ODD), dict(scales=ODD),
               dict(x=ctypes.c_void_p(4097)), dict(off=FAKE), dict(groups=2), dict(off=FAKE, groups=1025),
               dict(fmt=MX, ts=FAKE)):
        assert _quant(**kw) == -1, kw
    assert _quant(rows=0, src=0, x=None, codes=None, scales=None) == 0
    need = _lib.lib().sb_fp4_quant_workspace_bytes
    p = 1 << 16                     # from 2^22 values on, each source row taken twice or more
    assert need(NV, 4, p, 64) == 4 * (32 + 4 + 4) and need(MX, 4, p, 129) == 4 * (80 + 8 + 4) and need(NV, p // 2, p, 64) > 0
    assert need(NV, 4, p - 1, 64) == 0 and need(NV, p // 2 + 1, p, 64) == 0
    assert need(FP8, 4, p, 64) == 0 and need(NV, 0, p, 64) == 0 and need(NV, 4, p, 0) == 0
    assert _quant(rows_in=FAKE, rows=p, ws=FAKE, n=4 * 40 - 1) == -4
    assert _quant(rows_in=FAKE, rows=p, ws=ODD, n=1 << 20) == -1


def test_dequant_and_tile_refusals():
    L = _lib.lib()
    d = lambda fmt=NV, c=FAKE, s=FAKE, ts=None, rows=4, k=64, y=FAKE, dt=0: L.sb_fp4_dequant(  # noqa: E731
        fmt, c, s, ts, 0, rows, k, y, dt, None)
    assert d(fmt=FP8) == -3 and d(dt=7) == -1 and d(k=0) == -2
    assert d(c=None) == -1 and d(s=ODD) == -1 and d(y=ctypes.c_void_p(4097)) == -1 and d(fmt=MX, ts=FAKE) == -1
    assert d(rows=0, c=None) == 0
    t = lambda fmt=NV, s=FAKE, o=FAKE, m=1, n=4, k=64: L.sb_fp4_tile_scales(fmt, s, o, m, n, k, None)  # noqa: E731
    assert t(fmt=FP8) == -3 and t(k=48) == -2 and t(m=0) == -2 and t(n=0) == -2 and t(m=1 << 20, n=1 << 20) == -2
    assert t(s=None) == -1 and t(o=ODD) == -1


def test_product_refusals():
    L = _lib.lib()

    def g(fmt=NV, a=FAKE, s=FAKE, m=4, w=FAKE, ws=FAKE, wts=None, n=8, k=64, y=FAKE, dt=0, ld=8):
        return L.sb_fp4_gemm(fmt, a, s, None, 0, m, w, ws, wts, 0, n, k, y, dt, ld, None)

    assert g(fmt=FP8) == -3 and g(dt=3) == -1
    for kw in (dict(n=0), dict(k=0), dict(k=65537), dict(m=-1), dict(ld=7), dict(m=1 << 30, n=1 << 20, ld=1 << 20)):
        assert g(**kw) == -2, kw
    for kw in (dict(a=None), dict(s=ODD), dict(w=ODD), dict(ws=None), dict(y=None), dict(fmt=MX, wts=FAKE)):
        assert g(**kw) == -1, kw
    assert g(m=0, a=None, y=None) == 0

    def gg(off=FAKE, wtsn=1, wts=None, e=4, n=8, sw=0, lim=0.0, m=4, ld=8):
        return L.sb_fp4_grouped_gemm(NV, FAKE, FAKE, None, 0, m, off, FAKE, FAKE, wts, wtsn, e, n, 64, sw, lim, None, FAKE, 0,
                                     ld, None)

    assert gg(off=None) == -1 and gg(wts=FAKE, wtsn=3) == -1 and gg(lim=-1.0) == -1 and gg(lim=float("nan")) == -1
    assert gg(e=0) == -2 and gg(e=1025) == -2 and gg(sw=1, n=7) == -2 and gg(e=1024, n=1 << 21) == -2 and gg(sw=1, ld=3) == -2
    assert gg(m=0) == 0
    assert L.sb_fp4_error(None, None) == -1


def test_route_refusals():
    L = _lib.lib()

    def r(l=FAKE, dt=2, t=2, e=16, st=16, k=4, sc=1, g=1, kg=1, gs=0, w=FAKE, i=FAKE):
        return L.sb_route_topk(l, dt, t, e, st, None, k, sc, g, kg, gs, 1, 1.0, w, i, None)

    for kw in (dict(dt=3), dict(sc=3), dict(gs=2), dict(l=None), dict(w=None), dict(i=None), dict(l=ctypes.c_void_p(4098))):
        assert r(**kw) == -1, kw
    for kw in (dict(t=-1), dict(e=0), dict(e=1025), dict(st=-1), dict(g=0), dict(g=3), dict(g=64, e=64), dict(g=4, kg=5),
               dict(g=4, kg=0), dict(k=0), dict(k=17), dict(k=5, g=4, kg=1)):
        assert r(**kw) == -2, kw
    assert r(t=0, l=None) == 0
    assert L.sb_expert_order_workspace_bytes(16384, 256) == 0 and L.sb_expert_order_workspace_bytes(16385, 256) == 9 * 256 * 4

    def o(ids=FAKE, t=4, k=2, e=8, off=FAKE, tok=FAKE, pl=FAKE, ws=None, n=0):
        return L.sb_expert_order(ids, t, k, e, off, tok, pl, ws, n, None)

    assert o(t=-1) == -2 and o(k=0) == -2 and o(e=1025) == -2 and o(t=1 << 30, k=4) == -2
    assert o(ids=None) == -1 and o(off=None) == -1 and o(tok=None) == -1 and o(pl=None) == -1
    assert o(t=16384, ws=None) == -4 and o(t=16384, ws=FAKE, n=16 * 8 * 4 - 1) == -4
    assert o(t=16384, ws=ctypes.c_void_p(4097), n=1 << 20) == -1


def test_misaligned_pointers_are_refused():
    L = _lib.lib()
    at = lambda n: ctypes.c_void_p((1 << 12) + n)  # noqa: E731
    for kw in (dict(rows_in=at(2)), dict(ts=at(2)), dict(off=at(1), groups=2), dict(rs=at(2)), dict(x=at(2), dtype=2)):
        assert _quant(**kw) == -1, kw
    assert L.sb_fp4_dequant(NV, FAKE, FAKE, at(2), 0, 4, 64, FAKE, 0, None) == -1
    for ats, wts, y, dt in ((at(2), None, FAKE, 0), (None, at(1), FAKE, 0), (None, None, at(1), 0), (None, None, at(2), 2)):
        assert L.sb_fp4_gemm(NV, FAKE, FAKE, ats, 1, 4, FAKE, FAKE, wts, 0, 8, 64, y, dt, 8, None) == -1
    for off, rw in ((at(2), None), (FAKE, at(2))):
        assert L.sb_fp4_grouped_gemm(NV, FAKE, FAKE, None, 0, 4, off, FAKE, FAKE, None, 1, 2, 8, 64, 0, 0.0, rw, FAKE, 0, 8, None) == -1
    for bias, w, i in ((at(2), FAKE, FAKE), (None, at(2), FAKE), (None, FAKE, at(4))):
        assert L.sb_route_topk(FAKE, 2, 2, 16, 16, bias, 4, 1, 1, 1, 0, 1, 1.0, w, i, None) == -1
    for ids, off, tok, pl in ((at(4), FAKE, FAKE, FAKE), (FAKE, at(2), FAKE, FAKE), (FAKE, FAKE, at(1), FAKE), (FAKE, FAKE, FAKE, at(2))):
        assert L.sb_expert_order(ids, 4, 2, 8, off, tok, pl, None, 0, None) == -1


def test_expert_order_workspace_holds_the_counts_and_their_totals():
    f = _lib.lib().sb_expert_order_workspace_bytes
    assert f(64 * 2048, 256) == 64 * 256 * 4 and f(64 * 2048 + 1, 256) == 66 * 256 * 4
    assert f(2 ** 31 - 1, 1024) == (2 ** 20 + 1) * 1024 * 4


def test_sizes_whose_products_leave_64_bits_are_refused():
    L = _lib.lib()
    for n_mat, n in ((1 << 34, 1 << 30), (1 << 60, 16), ((1 << 62) + 1, 4), ((1 << 63) - 1, 2)):
        assert L.sb_fp4_tile_scales(NV, FAKE, FAKE, n_mat, n, 64, None) == -2, (n_mat, n)
    f = L.sb_fp4_scale_bytes
    assert f(NV, 1 << 30, 1 << 30, 64, 0) == 0 and f(NV, 1 << 20, (1 << 10) + 1, 64, 0) == 0 and f(NV, 1 << 34, 1 << 30, 64, 0) == 0
    assert f(NV, 1 << 20, 1 << 10, 64, 0) == (1 << 20) * 8 * 512 and f(MX, 1 << 30, 1, 65536, 0) == (1 << 30) * 512 * 512

    def gg(e, n, m=4, ld=None):
        return L.sb_fp4_grouped_gemm(NV, FAKE, FAKE, None, 0, m, FAKE, FAKE, FAKE, None, 1, e, n, 64, 0, 0.0, None, FAKE, 0,
                                     n if ld is None else ld, None)

    for e, n, m in ((4, 1 << 62, 508 * 128), (1024, 1 << 54, 4), (1, (1 << 63) - 1, 4), (2, 1 << 62, 4)):
        assert gg(e, n, m) == -2, (e, n)
        assert L.sb_fp4_gemm(NV, FAKE, FAKE, None, 0, m, FAKE, FAKE, None, 0, n, 64, FAKE, 0, n, None) == -2
