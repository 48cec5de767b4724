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
through torch and does not synchronise; it can be captured into a CUDA graph. CUDA tensors only. As with
torch's own operators, the caller orders streams and keeps inputs of another stream until the call has run.
"""
from __future__ import annotations

import contextlib
import ctypes
from typing import Optional, Union

import torch

from . import _lib
from . import formats as F
from ._lib import ShardB200Error, check, lib, ptr

PLAIN, W13 = _lib.MAT_PLAIN, _lib.MAT_W13
DTYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.float32: _lib.F32}
_FMT = {"nvfp4": F.FMT_NVFP4, "mxfp4": F.FMT_MXFP4, F.FMT_NVFP4: F.FMT_NVFP4, F.FMT_MXFP4: F.FMT_MXFP4}

_current_device = torch._C._cuda_getDevice
_new = object.__new__
_HOST = None


def host():
    """The extension module that checks, allocates and launches (csrc/sb_host.cpp). Like the library it has no
    substitute: a missing one raises."""
    global _HOST
    if _HOST is None:
        lib()
        try:
            from . import _host
        except ImportError as e:
            raise ShardB200Error(f"shard_b200/_host.so cannot be loaded ({e}); build it with `python -m shard_b200.build`")
        _HOST = _host
    return _HOST


def _fmt(fmt: Union[int, str]) -> int:
    f = _FMT.get(fmt)
    if f is None:
        raise ValueError(f"format {fmt!r} is not nvfp4 or mxfp4")
    return f


def _away(what: str, t: torch.Tensor, stream) -> bool:
    """Whether a call on `t` has to make another device or stream current first."""
    dev = t.get_device()
    if dev < 0:
        raise ValueError(f"{what}: the tensors must be on a CUDA device")
    return stream is not None or dev != _current_device()


@contextlib.contextmanager
def _elsewhere(device, stream):
    """`device` made current, and `stream` when one is given (also for the allocations of the call)."""
    if stream is not None and stream.device != device:
        raise ValueError(f"a stream of {stream.device} for tensors on {device}")
    with torch.cuda.device(device):
        if stream is None:
            yield
        else:
            with torch.cuda.stream(stream):
                yield


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
            self._codes = self._buf[:self._parts[0]].view(self.rows, -(-self.k // 32) * 16)
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
        """uint8 [mats * rows, kp / 16 or kp / 32]: the scales row by row (no expert groups)."""
        if self.offsets is not None:
            raise ValueError("canonical_scales: rows in expert groups")
        nb = self.codes.shape[1] // (8 if self.fmt == F.FMT_NVFP4 else 16)
        blocks, atoms = -(-self.rows // 128), -(-nb // 4)
        s = self.scales.view(self.mats, blocks, atoms, 32, 4, 4)                # mat, block, atom, lane, quarter, byte
        s = s.permute(0, 1, 4, 3, 2, 5).reshape(self.mats, blocks * 128, atoms * 4)
        return s[:, :self.rows, :nb].reshape(self.mats * self.rows, nb).contiguous()


def quant(x: torch.Tensor, fmt: Union[int, str] = F.FMT_NVFP4, tensor_scale: Optional[torch.Tensor] = None,
          rows: Optional[torch.Tensor] = None, offsets: Optional[torch.Tensor] = None, stream=None) -> Fp4Tensor:
    """x [..., K] (bf16, fp16 or fp32, any row stride, 1 <= K <= 65536) -> Fp4Tensor of its rows.

    tensor_scale  NVFP4: calibrated fp32 scale (one value) in place of the rows' own
    rows          int32 [P]: operand row p is x's row rows[p] (a gather in the same pass); outside x: zeros
    offsets       int32 [E + 1]: expert e's rows are offsets[e] .. offsets[e + 1] - 1 (for grouped_gemm);
                  rows of no expert are left as they are"""
    f = _FMT.get(fmt)
    if f is None:
        f = _fmt(fmt)
    if _away("quant", x, stream):
        with _elsewhere(x.device, stream):
            return quant(x, f, tensor_scale, rows, offsets)
    r = (_HOST or host()).quant(x, f, tensor_scale, rows, offsets)
    if type(r) is int:
        check(r, "sb_fp4_quant")
    q = _new(Fp4Tensor)
    q._buf, q.rows, q.k, q.per_row, end, atoms_end, base, q.shape = r
    q.fmt, q.mats, q.kind, q.offsets = f, 1, PLAIN, offsets
    q._parts, q._codes, q._scales, q._ts = (end, atoms_end), None, None, tensor_scale
    q.codes_ptr, q.scales_ptr = base, base + end
    q.ts_ptr = base + atoms_end if q.per_row else ptr(tensor_scale)
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
    if _away("dequant", buf, stream):
        with _elsewhere(buf.device, stream):
            return dequant(q, dtype)
    y = (_HOST or host()).dequant(buf, q.fmt, q.codes_ptr, q.scales_ptr, q.ts_ptr, q.per_row, q.rows, q.k, q.shape, dt)
    if type(y) is int:
        check(y, "sb_fp4_dequant")
    return y


def pack(fmt: Union[int, str], codes: torch.Tensor, scales: torch.Tensor, ts: Optional[torch.Tensor] = None,
         kind: int = PLAIN, stream=None) -> Fp4Tensor:
    """Canonical weights -> operand, once at load time. codes uint8 [N, K/2] or [E, N, K/2], scales as bytes or
    in their own type [.., K/16] (NVFP4) / [.., K/32] (MXFP4), ts fp32: one per matrix, or for w13 banks
    [E, 2] (w1, w3). K is whole blocks of scales (16 or 32; rows are padded to 32 with zeros). kind W13: the rows
    are w1's, then w3's; they are interleaved, so that one pass of grouped_gemm forms silu(w1 x) * (w3 x). PLAIN
    operands share the codes given, if these are contiguous, 16-byte aligned and not padded."""
    f = _fmt(fmt)
    if not codes.is_cuda or codes.dim() not in (2, 3):
        raise ValueError("pack: codes must be a CUDA tensor [N, K/2] or [E, N, K/2]")
    if _away("pack", codes, stream):      # before any conversion: those run there, too
        with _elsewhere(codes.device, stream):
            return pack(fmt, codes, scales, ts, kind)
    c, s = codes.view(torch.uint8), scales.view(torch.uint8)
    for t in (scales, ts):
        if t is not None and t.device != codes.device:
            raise ValueError(f"pack: tensors on {t.device} and {codes.device}")
    mats, n, k = (1 if c.dim() == 2 else c.shape[0]), c.shape[-2], 2 * c.shape[-1]
    block = 16 if f == F.FMT_NVFP4 else 32
    nb = k // block
    if k % block or tuple(s.shape) != (*c.shape[:-1], nb):
        raise ValueError(f"pack: scales {tuple(s.shape)} for codes {tuple(c.shape)} (K % {block} == 0 is needed)")
    if ts is not None:
        if f != F.FMT_NVFP4:
            raise ValueError("pack: MXFP4 has no tensor scale")
        ts = ts.to(torch.float32).reshape(mats, -1).contiguous()
        if ts.shape[1] not in ((1, 2) if kind == W13 else (1,)):
            raise ValueError(f"pack: {ts.shape[1]} tensor scales a matrix")
    if kind not in (PLAIN, W13) or (kind == W13 and n % 2):
        raise ValueError("pack: kind is PLAIN, or W13 with an even number of rows")
    kp = -(-k // 32) * 32
    if kp != k:
        c, s = torch.nn.functional.pad(c, (0, (kp - k) // 2)), torch.nn.functional.pad(s, (0, (kp - k) // block))
    c, s = c.reshape(mats, n, kp // 2), s.reshape(mats, n, kp // block)
    if kind == W13:
        c, s = (t.view(mats, 2, n // 2, -1).transpose(1, 2).reshape(mats, n, -1) for t in (c, s))
    c, s = c.contiguous().view(mats * n, kp // 2), s.contiguous()
    if c.data_ptr() % 16:                 # (a view into a larger buffer: the products copy from 16-byte addresses)
        c = c.clone()
    L = lib()
    out = torch.empty(L.sb_fp4_scale_bytes(f, mats, n, kp, 0), dtype=torch.uint8, device=c.device)
    check(L.sb_fp4_tile_scales(f, s.data_ptr(), out.data_ptr(), mats, n, kp, torch.cuda.current_stream().cuda_stream),
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


def gemm(a: Fp4Tensor, w: Fp4Tensor, out_dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None,
         stream=None) -> torch.Tensor:
    """y [..., N] = A [..., K] W [N, K]^T, summed in fp32 and rounded once. `out` [M, N] may have any row stride.
    The tensor scale of `w` is one value or none (one per row, as quant makes them, multiplies its outputs)."""
    dt = _operands("gemm", a, w, out_dtype)
    if a.offsets is not None or w.offsets is not None or w.mats != 1 or w.kind != PLAIN:
        raise ValueError("gemm: plain operands of one matrix (grouped_gemm takes banks and expert groups)")
    buf = a._buf
    if _away("gemm", buf, stream):
        with _elsewhere(buf.device, stream):
            return gemm(a, w, out_dtype, out)
    y = (_HOST or host()).gemm(buf, a.fmt, a.codes_ptr, a.scales_ptr, a.ts_ptr, a.per_row, a.rows, a.shape, a.k, w.codes_ptr,
                               w.scales_ptr, w.ts_ptr, w.per_row, w.rows, dt, out)
    if type(y) is int:
        check(y, "sb_fp4_gemm")
    return y


def grouped_gemm(a: Fp4Tensor, w: Fp4Tensor, out_dtype: torch.dtype = torch.bfloat16,
                 row_weight: Optional[torch.Tensor] = None, limit: float = 0.0, out: Optional[torch.Tensor] = None,
                 stream=None) -> torch.Tensor:
    """Row p of expert e (offsets[e] <= p < offsets[e+1]) against W_e of the bank: y [P, N], or for a W13 bank
    y [P, N/2] = silu(min(g, limit)) * clip(u, -limit, limit) (limit 0: no clamp). row_weight fp32 [P]
    multiplies the output rows. Rows of no expert are left as they are."""
    dt = _operands("grouped_gemm", a, w, out_dtype)
    off = a.offsets
    if off is None or off.shape[0] != w.mats + 1 or w.per_row or w.offsets is not None:
        raise ValueError(f"grouped_gemm: rows with offsets [{w.mats + 1}] (quant(..., offsets=)) and a bank (pack)")
    if not limit >= 0.0:
        raise ValueError("grouped_gemm: limit must be >= 0")
    buf = a._buf
    if _away("grouped_gemm", buf, stream):
        with _elsewhere(buf.device, stream):
            return grouped_gemm(a, w, out_dtype, row_weight, limit, out)
    y = (_HOST or host()).grouped_gemm(buf, a.fmt, a.codes_ptr, a.scales_ptr, a.ts_ptr, a.per_row, a.rows, a.k, off, w.codes_ptr,
                                       w.scales_ptr, w.ts_ptr, 1 if w._ts is None else w._ts.shape[1], w.mats, w.rows,
                                       w.kind == W13, limit, row_weight, dt, out)
    if type(y) is int:
        check(y, "sb_fp4_grouped_gemm")
    return y


def device_error(device=None) -> int:
    """1 if a product's kernel gave up a bounded wait on the device since the last call, or found offsets that descend
    (it then writes nothing), else 0. Synchronises."""
    with torch.cuda.device(device):
        v = ctypes.c_int(0)
        check(lib().sb_fp4_error(ctypes.byref(v), torch.cuda.current_stream().cuda_stream), "sb_fp4_error")
    return v.value
