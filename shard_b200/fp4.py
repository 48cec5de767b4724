"""Microscaled 4-bit operands on both sides (W4A4): quantisation of activations and their products with
NVFP4 / MXFP4 weights, on the block-scaled tensor-core MMA.

The kernel seam's `ops.fp4_gemm` multiplies 4-bit weights with e4m3 activations, the arithmetic of the
V4 engine. NVFP4 checkpoints (the M2.5 engine's FusedMoE experts, engines/minimax_m25/m25_stage.py:288-311)
are calibrated for 4-bit activations too, and the reference's `fp4_act_quant` (kernel.py:128-200)
quantises activations to MXFP4: these are the operators of that form.

    quant(x, fmt)                    activations -> Fp4Tensor (codes, block scales, tensor scale per row)
    dequant(q)                       its values
    pack(fmt, codes, scales, ts)     canonical checkpoint weights -> Fp4Tensor, once at load time
    gemm(a, w)                       y = A W^T
    grouped_gemm(a, bank)            the same per expert, rows sorted by expert; w13 banks give
                                     silu(gate) * up

    a = quant(x, "nvfp4", rows=order.tokens, offsets=order.offsets)     # route.expert_order
    h = grouped_gemm(a, w13)                                            # [pairs, I] bf16
    o = grouped_gemm(quant(h, "nvfp4", offsets=order.offsets), w2)      # [pairs, H] bf16

NVFP4: q = e2m1(x / (s t)), s = e4m3(amax / (6 t)) per 16 values, t = max(2^-126, amax_row / 2688) per row (a row
then does not depend on its batch) or the caller's calibrated `tensor_scale`. MXFP4: one power of two
per 32 values, the smallest with amax <= 6 s. Roundings are to nearest, ties to even; a block with a
non-finite value comes back as NaN, and a row of zeros as zeros.

Every call runs on the tensors' device, on its current stream or on `stream`, allocates its outputs
through torch and does not synchronise; it can be captured into a CUDA graph. CUDA tensors only.
"""
from __future__ import annotations

import contextlib
import ctypes
from typing import Optional, Union

import torch

from . import _lib
from . import formats as F
from ._lib import check, lib, ptr

PLAIN, W13 = _lib.MAT_PLAIN, _lib.MAT_W13
DTYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.float32: _lib.F32}
_FMT = {"nvfp4": F.FMT_NVFP4, "mxfp4": F.FMT_MXFP4, F.FMT_NVFP4: F.FMT_NVFP4, F.FMT_MXFP4: F.FMT_MXFP4}

# A decoded token's call is bound by its host side: these run once per call, without lookups by name.
_current_device = torch._C._cuda_getDevice
_current_stream = torch._C._cuda_getCurrentRawStream
_empty = torch.empty


def _fmt(fmt: Union[int, str]) -> int:
    f = _FMT.get(fmt)
    if f is None:
        raise ValueError(f"format {fmt!r} is not nvfp4 or mxfp4")
    return f


@contextlib.contextmanager
def _elsewhere(device, stream):
    """`device` made current, and `stream` when one is given (also for the allocations of the call)."""
    with torch.cuda.device(device):
        if stream is None:
            yield
        else:
            with torch.cuda.stream(stream):
                yield


def _same_device(what, ref, *tensors):
    for t in tensors:
        if t is not None and t.device != ref.device:
            raise ValueError(f"{what}: tensors on {t.device} and {ref.device}")


def _index(what, name, t, n=None):
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() or (n is not None and t.shape[0] != n):
        raise ValueError(f"{what}: {name} must be a contiguous int32 vector" + ("" if n is None else f" of {n}"))


def _float_vec(what, name, t, n=None):
    if t.dtype != torch.float32 or not t.is_contiguous() or (n is not None and t.numel() != n):
        raise ValueError(f"{what}: {name} must be contiguous fp32" + ("" if n is None else f" with {n} values"))


class Fp4Tensor:
    """A 4-bit operand on the device: `mats` matrices of `rows` rows of `k` values (activations: one).

    codes   uint8 [mats * rows, kp / 2], kp = k rounded up to 32; low nibble first
    scales  uint8, the atoms of 128 rows x 4 scales that the products read
    ts      NVFP4: fp32 tensor scale, [1] or one per row (activations), [mats, 1 or 2] (weights), or None
    offsets int32 [groups + 1]: the rows' expert groups (activations of grouped_gemm), else None
    """
    __slots__ = ("fmt", "mats", "rows", "k", "kind", "shape", "offsets", "per_row", "_buf", "_parts", "_codes", "_scales",
                 "_ts", "codes_ptr", "scales_ptr", "ts_ptr")

    def __init__(self, fmt, mats, rows, k, codes, scales, ts=None, offsets=None, kind=PLAIN, shape=()):
        self.fmt, self.mats, self.rows, self.k, self.kind, self.shape, self.offsets = fmt, mats, rows, k, kind, shape, offsets
        self._buf, self._codes, self._scales, self._ts = codes, codes, scales, ts
        self._parts = None
        self.per_row = False
        self.codes_ptr, self.scales_ptr, self.ts_ptr = codes.data_ptr(), scales.data_ptr(), ptr(ts)

    @property
    def device(self):
        return self._buf.device

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            self._codes = self._buf[:self._parts[0]].view(self.rows, -1)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._scales = self._buf[self._parts[0]:self._parts[1]]
        return self._scales

    @property
    def ts(self) -> Optional[torch.Tensor]:
        if self._ts is None and self.per_row:
            self._ts = self._buf[self._parts[1]:].view(torch.float32)
        return self._ts

    def canonical_scales(self) -> torch.Tensor:
        """uint8 [mats * rows, K / 16 or K / 32]: the scales row by row (no expert groups)."""
        if self.offsets is not None:
            raise ValueError("canonical_scales: rows in expert groups")
        nb = self.codes.shape[1] // (8 if self.fmt == F.FMT_NVFP4 else 16)
        s = self.scales.view(self.mats, -(-self.rows // 128), -1, 32, 4, 4)     # mat, block, atom, lane, quarter, byte
        s = s.permute(0, 1, 4, 3, 2, 5).reshape(self.mats, -1, s.shape[2] * 4)
        return s[:, :self.rows, :nb].reshape(self.mats * self.rows, nb).contiguous()


def quant(x: torch.Tensor, fmt: Union[int, str] = F.FMT_NVFP4, tensor_scale: Optional[torch.Tensor] = None,
          rows: Optional[torch.Tensor] = None, offsets: Optional[torch.Tensor] = None, stream=None) -> Fp4Tensor:
    """x [..., K] (bf16, fp16 or fp32, any row stride, 1 <= K <= 65536) -> Fp4Tensor of its rows.

    tensor_scale  NVFP4: calibrated fp32 scale (one value) in place of the rows' own
    rows          int32 [P]: operand row p is x's row rows[p] (a gather in the same pass); outside x: zeros
    offsets       int32 [E + 1]: expert e's rows are offsets[e] .. offsets[e + 1] - 1 (for grouped_gemm);
                  rows behind offsets[E] are left as they are"""
    f = _FMT.get(fmt)
    if f is None:
        _fmt(fmt)
    dt = DTYPES.get(x.dtype)
    if dt is None or not x.is_cuda or x.dim() < 1:
        raise ValueError("quant: x must be a CUDA tensor of bf16, fp16 or fp32")
    dev = x.get_device()
    if stream is not None or dev != _current_device():
        with _elsewhere(x.device, stream):
            return quant(x, fmt, tensor_scale, rows, offsets)
    shape = x.shape
    k = shape[-1]
    z = x if x.dim() == 2 else x.reshape(-1, k)
    m = z.shape[0]
    stride, inner = z.stride()
    if inner != 1 and k > 1:
        z = z.contiguous()
        stride = k
    p, groups, po, pr, pt = m, 0, None, None, None
    if rows is not None:
        _index("quant", "rows", rows)
        _same_device("quant", x, rows)
        p, pr = rows.shape[0], rows.data_ptr()
    if offsets is not None:
        _index("quant", "offsets", offsets)
        _same_device("quant", x, offsets)
        groups, po = offsets.shape[0] - 1, offsets.data_ptr()
        if groups < 1:
            raise ValueError("quant: offsets must hold at least two values")
    if tensor_scale is not None:
        if f != F.FMT_NVFP4:
            raise ValueError("quant: MXFP4 has no tensor scale")
        _float_vec("quant", "tensor_scale", tensor_scale, 1)
        _same_device("quant", x, tensor_scale)
        pt = tensor_scale.data_ptr()
    # one allocation: codes, scale atoms (sb_fp4_scale_bytes), the rows' tensor scales
    kp = (k + 31) >> 5
    blocks = (p >> 7) + groups if groups else (p + 127) >> 7
    end = p * kp * 16
    per_row = f == F.FMT_NVFP4 and pt is None
    atoms_end = end + blocks * ((kp + 1) >> 1 if f == F.FMT_NVFP4 else (kp + 3) >> 2) * 512
    buf = _empty(atoms_end + 4 * p if per_row else atoms_end, dtype=torch.uint8, device=x.device)
    base = buf.data_ptr()
    q = Fp4Tensor.__new__(Fp4Tensor)
    q.fmt, q.mats, q.rows, q.k, q.kind, q.offsets, q.per_row = f, 1, p, k, PLAIN, offsets, per_row
    q.shape = shape[:-1] if rows is None else (p,)
    q._buf, q._parts, q._codes, q._scales, q._ts = buf, (end, atoms_end), None, None, tensor_scale
    q.codes_ptr, q.scales_ptr = base, base + end
    q.ts_ptr = base + atoms_end if per_row else pt
    rc = lib().sb_fp4_quant(f, z.data_ptr(), dt, m, k, stride if m > 1 else k, pr, p, pt, po, groups, base, base + end,
                            q.ts_ptr if per_row else None, _current_stream(dev))
    if rc:
        check(rc, "sb_fp4_quant")
    return q


def dequant(q: Fp4Tensor, dtype: torch.dtype = torch.bfloat16, stream=None) -> torch.Tensor:
    """The operand's values [..., K]: code * scale * tensor scale, rounded to `dtype`. Activations without
    expert groups."""
    if q.offsets is not None or q.mats != 1 or q.kind != PLAIN:
        raise ValueError("dequant: a plain operand of one matrix, without expert groups")
    dt = DTYPES.get(dtype)
    if dt is None:
        raise ValueError(f"dequant: dtype {dtype}")
    buf = q._buf
    dev = buf.get_device()
    if stream is not None or dev != _current_device():
        with _elsewhere(buf.device, stream):
            return dequant(q, dtype)
    y = _empty((*q.shape, q.k), dtype=dtype, device=buf.device)
    rc = lib().sb_fp4_dequant(q.fmt, q.codes_ptr, q.scales_ptr, q.ts_ptr, q.per_row, q.rows, q.k, y.data_ptr(), dt,
                              _current_stream(dev))
    if rc:
        check(rc, "sb_fp4_dequant")
    return y


def pack(fmt: Union[int, str], codes: torch.Tensor, scales: torch.Tensor, ts: Optional[torch.Tensor] = None,
         kind: int = PLAIN, stream=None) -> Fp4Tensor:
    """Canonical weights -> operand, once at load time. codes uint8 [N, K/2] or [E, N, K/2], scales as bytes or
    in their own type [.., K/16] (NVFP4) / [.., K/32] (MXFP4), ts fp32: one per matrix, or for w13 banks
    [E, 2] (w1, w3). K % 32 == 0. kind W13: the rows are w1's, then w3's; they are interleaved, so that one
    pass of grouped_gemm forms silu(w1 x) * (w3 x). PLAIN operands share the codes given."""
    f = _fmt(fmt)
    if not codes.is_cuda or codes.dim() not in (2, 3):
        raise ValueError("pack: codes must be a CUDA tensor [N, K/2] or [E, N, K/2]")
    c, s = codes.view(torch.uint8), scales.view(torch.uint8)
    _same_device("pack", codes, scales, ts)
    mats, n, k = (1 if c.dim() == 2 else c.shape[0]), c.shape[-2], 2 * c.shape[-1]
    nb = k // (16 if f == F.FMT_NVFP4 else 32)
    if k % 32 or tuple(s.shape) != (*c.shape[:-1], nb):
        raise ValueError(f"pack: scales {tuple(s.shape)} for codes {tuple(c.shape)} (K % 32 == 0 is needed)")
    if ts is not None:
        if f != F.FMT_NVFP4:
            raise ValueError("pack: MXFP4 has no tensor scale")
        ts = ts.to(torch.float32).reshape(mats, -1).contiguous()
        if ts.shape[1] not in ((1, 2) if kind == W13 else (1,)):
            raise ValueError(f"pack: {ts.shape[1]} tensor scales a matrix")
    if kind not in (PLAIN, W13) or (kind == W13 and n % 2):
        raise ValueError("pack: kind is PLAIN, or W13 with an even number of rows")
    if stream is not None or codes.get_device() != _current_device():
        with _elsewhere(codes.device, stream):
            return pack(fmt, codes, scales, ts, kind)
    c, s = c.reshape(mats, n, k // 2), s.reshape(mats, n, nb)
    if kind == W13:
        c, s = (t.view(mats, 2, n // 2, -1).transpose(1, 2).reshape(mats, n, -1) for t in (c, s))
    c, s = c.contiguous().view(mats * n, k // 2), s.contiguous()
    L = lib()
    out = torch.empty(L.sb_fp4_scale_bytes(f, mats, n, k, 0), dtype=torch.uint8, device=c.device)
    check(L.sb_fp4_tile_scales(f, s.data_ptr(), out.data_ptr(), mats, n, k, _current_stream(c.get_device())),
          "sb_fp4_tile_scales")
    return Fp4Tensor(f, mats, n, k, c, out, ts, None, kind, tuple(codes.shape[:-1]))


def _operands(what, a, w, out_dtype):
    """Checks shared by the products; the output type's code."""
    if a.fmt != w.fmt:
        raise ValueError(f"{what}: operands of two formats")
    if a.k != w.k:
        raise ValueError(f"{what}: K {a.k} and {w.k}")
    if a.mats != 1 or a.kind != PLAIN:
        raise ValueError(f"{what}: the first operand is one matrix of rows")
    dt = DTYPES.get(out_dtype)
    if dt is None:
        raise ValueError(f"{what}: out_dtype {out_dtype}")
    if w._buf.get_device() != a._buf.get_device():
        raise ValueError(f"{what}: operands on {a.device} and {w.device}")
    return dt


def _check_out(what, out, shape, dtype, like):
    if tuple(out.shape) != shape or out.dtype != dtype or out.device != like.device or \
            (out.numel() and shape[1] > 1 and out.stride(-1) != 1) or (shape[0] > 1 and out.stride(0) < shape[1]):
        raise ValueError(f"{what}: out must be {shape} {dtype} on {like.device}, with contiguous rows that do not overlap")


def gemm(a: Fp4Tensor, w: Fp4Tensor, out_dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None,
         stream=None) -> torch.Tensor:
    """y [..., N] = A [..., K] W [N, K]^T, summed in fp32 and rounded once. `out` [M, N] may have any row stride.
    The tensor scale of `w` is one value or none (one per row, as quant makes them, multiplies its outputs)."""
    dt = _operands("gemm", a, w, out_dtype)
    if a.offsets is not None or w.offsets is not None or w.mats != 1 or w.kind != PLAIN:
        raise ValueError("gemm: plain operands of one matrix (grouped_gemm takes banks and expert groups)")
    buf = a._buf
    dev = buf.get_device()
    if stream is not None or dev != _current_device():
        with _elsewhere(buf.device, stream):
            return gemm(a, w, out_dtype, out)
    m, n = a.rows, w.rows
    ld = n
    if out is None:
        out = _empty((*a.shape, n), dtype=out_dtype, device=buf.device)
    else:
        _check_out("gemm", out, (m, n), out_dtype, buf)
        if m > 1:
            ld = out.stride(0)
    rc = lib().sb_fp4_gemm(a.fmt, a.codes_ptr, a.scales_ptr, a.ts_ptr, a.per_row, m, w.codes_ptr, w.scales_ptr, w.ts_ptr,
                           w.per_row, n, a.k, out.data_ptr(), dt, ld, _current_stream(dev))
    if rc:
        check(rc, "sb_fp4_gemm")
    return out


def grouped_gemm(a: Fp4Tensor, w: Fp4Tensor, out_dtype: torch.dtype = torch.bfloat16,
                 row_weight: Optional[torch.Tensor] = None, limit: float = 0.0, out: Optional[torch.Tensor] = None,
                 stream=None) -> torch.Tensor:
    """Row p of expert e (offsets[e] <= p < offsets[e+1]) against W_e of the bank: y [P, N], or for a W13 bank
    y [P, N/2] = silu(min(g, limit)) * clip(u, -limit, limit) (limit 0: no clamp). row_weight fp32 [P]
    multiplies the output rows. Rows behind offsets[E] are left as they are."""
    dt = _operands("grouped_gemm", a, w, out_dtype)
    off = a.offsets
    if off is None or off.shape[0] != w.mats + 1 or w.per_row or w.offsets is not None:
        raise ValueError(f"grouped_gemm: rows with offsets [{w.mats + 1}] (quant(..., offsets=)) and a bank (pack)")
    if not limit >= 0.0:
        raise ValueError("grouped_gemm: limit must be >= 0")
    buf = a._buf
    p = a.rows
    pw = None
    if row_weight is not None:
        _float_vec("grouped_gemm", "row_weight", row_weight, p)
        _same_device("grouped_gemm", buf, row_weight)
        pw = row_weight.data_ptr()
    dev = buf.get_device()
    if stream is not None or dev != _current_device():
        with _elsewhere(buf.device, stream):
            return grouped_gemm(a, w, out_dtype, row_weight, limit, out)
    swiglu = w.kind == W13
    n = w.rows
    width = n >> 1 if swiglu else n
    ld = width
    if out is None:
        out = _empty((p, width), dtype=out_dtype, device=buf.device)
    else:
        _check_out("grouped_gemm", out, (p, width), out_dtype, buf)
        if p > 1:
            ld = out.stride(0)
    rc = lib().sb_fp4_grouped_gemm(a.fmt, a.codes_ptr, a.scales_ptr, a.ts_ptr, a.per_row, p, off.data_ptr(), w.codes_ptr,
                                   w.scales_ptr, w.ts_ptr, 1 if w._ts is None else w._ts.shape[1], w.mats, n, a.k, swiglu,
                                   limit, pw, out.data_ptr(), dt, ld, _current_stream(dev))
    if rc:
        check(rc, "sb_fp4_grouped_gemm")
    return out


def device_error(device=None) -> int:
    """1 if a product's kernel gave up a bounded wait on the device since the last call, else 0. Synchronises."""
    with torch.cuda.device(device):
        v = ctypes.c_int(0)
        check(lib().sb_fp4_error(ctypes.byref(v), torch.cuda.current_stream().cuda_stream), "sb_fp4_error")
    return v.value
