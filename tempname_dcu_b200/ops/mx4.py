"""Microscaled 4-bit floating point ("MXFP4"): quantizer, its inverse and
products of two quantized operands (``csrc/mx4.cu``).

Format: e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6, signed), one power-of-two
scale (ue8m0 byte ``e + 127``) per 32 consecutive K values of a row.  The
scale of a block with absolute maximum ``a`` is the smallest ``2^e`` (e >= -127)
with ``a / 2^e <= 6``, so nothing saturates; values round to nearest even.  A
block with an infinity or NaN decodes as NaN.  Two values share a byte (even K
index low); scales are stored in 512-byte atoms as the tensor cores read them
and are opaque to callers (``dequantize`` is the way back).

Rows may be any number, K a multiple of 32 up to 2^26 - 1024, N of the products
a multiple of 8.
``offsets`` (int32 [groups + 1], on the device) are those of ``ops.grouped``:
an operand quantized with offsets goes into ``grouped_linear`` with the same
offsets.  Weights are quantized once, [N, K] or [groups, N, K].

``tile`` asks for a tile shape (0: by the sizes), for measurements.

Against ``ops.mx`` (8-bit values): half the bytes and twice the tensor-core
rate, at 2 significant bits per value.
"""
from __future__ import annotations

import ctypes

import torch

from . import native

V, I, I64, LL = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_longlong

native.register("tdb_mx4_scale_bytes", [LL, LL, LL, I], restype=LL)
native.register("tdb_mx4_quantize", [V, I64, I64, I64, I64, V, I, V, V, V])
native.register("tdb_mx4_dequantize", [V, V, I64, I64, I64, V, I, V, I64, V])
native.register("tdb_mx4_pick_tile", [LL, I, I])
native.register("tdb_mx4_gemm", [V, V, V, V, V, I, V, I64, I, I, I, V, I, V])

E2M1_MAX = 6.0
MAX_GROUPS = 1024
MAX_K = 2 ** 26 - 1024


def _groups(offsets, device):
    if offsets is None:
        return 0
    if not (offsets.dtype is torch.int32 and offsets.dim() == 1 and offsets.is_contiguous() and
            offsets.get_device() == device):
        raise ValueError("offsets must be a contiguous int32 vector on the operands' device")
    groups = offsets.numel() - 1
    if not (1 <= groups <= MAX_GROUPS):
        raise ValueError(f"the number of groups must be 1..{MAX_GROUPS}")
    return groups


def scale_bytes(rows: int, k: int, groups: int = 0, matrices: int = 1) -> int:
    """Bytes of the scales of ``matrices`` [rows, k] operands, or of one whose
    rows lie in ``groups`` groups (as ``tdb_mx4_scale_bytes``, without the call)."""
    if groups > 0:
        blocks = rows // (32 if rows <= groups * 32 else 128) + min(rows, groups)
    else:
        blocks = matrices * -(-rows // 128)
    return blocks * -(-k // 256) * 1024


def _operand(q, sf, groups, device, what):
    """(matrices, rows, K) of a quantized operand."""
    if not (q.dtype is torch.uint8 and q.dim() in (2, 3) and q.is_contiguous() and q.get_device() == device):
        raise ValueError(f"{what} must be contiguous uint8 [..., K/2] as written by quantize, on the operands' "
                         f"device")
    shape = q.shape
    matrices = shape[0] if len(shape) == 3 else 1
    rows, K = shape[-2], 2 * shape[-1]
    if not (0 < K <= MAX_K and K % 32 == 0 and rows < 2 ** 31):
        raise ValueError(f"{what}: K must be a positive multiple of 32 up to {MAX_K}, and rows fewer than 2^31")
    if not (sf.dtype is torch.uint8 and sf.is_contiguous() and sf.get_device() == device and
            sf.numel() >= scale_bytes(rows, K, groups, matrices)):
        raise ValueError(f"the scales of {what} must be the uint8 buffer that quantize wrote for these rows (and "
                         f"offsets)")
    return matrices, rows, K


@native.on_tensor_device
def quantize(x, offsets=None, q=None, sf=None):
    """bf16 ``x`` [rows, K] or [matrices, rows, K] -> (q uint8 [..., K/2], sf
    uint8).  With ``offsets``, rows outside every group are not written."""
    if x.dtype is not torch.bfloat16:
        raise TypeError("quantize expects bf16")
    dims = x.dim()
    if not (x.is_cuda and dims in (2, 3)):
        raise ValueError("x must be [rows, K] or [matrices, rows, K] on a CUDA device")
    shape, stride = x.shape, x.stride()
    rows, K = shape[-2:]
    if not (0 < K <= MAX_K and K % 32 == 0 and stride[-1] == 1):
        raise ValueError(f"K must be a positive multiple of 32 up to {MAX_K}, the last dimension contiguous")
    index = x.get_device()
    groups = _groups(offsets, index)
    matrices, ld = 1, stride[0] if rows > 1 else K
    if dims == 3:
        if not (x.is_contiguous() and offsets is None and shape[0] > 0):
            raise ValueError("a [matrices, rows, K] operand must be contiguous and takes no offsets")
        matrices, ld = shape[0], K
    if not (ld >= K):
        raise ValueError("x: rows must not overlap")
    need = scale_bytes(rows, K, groups, matrices)
    packed = shape[:-1] + (K // 2,)
    if q is None:
        q = x.new_empty(packed, dtype=torch.uint8)
    else:
        if not (q.dtype is torch.uint8 and q.shape == packed and q.is_contiguous() and q.get_device() == index):
            raise ValueError("q must be contiguous uint8 [..., K/2] on x's device")
    if sf is None:
        sf = x.new_empty(need, dtype=torch.uint8)
    else:
        if not (sf.dtype is torch.uint8 and sf.numel() >= need and sf.is_contiguous() and sf.get_device() == index):
            raise ValueError(f"sf must be a contiguous uint8 buffer of at least {need} bytes on x's device")
    native.check(native.lib().tdb_mx4_quantize(x.data_ptr(), ld, matrices, rows, K,
                                               None if offsets is None else offsets.data_ptr(), groups, q.data_ptr(),
                                               sf.data_ptr(), native.current_stream(index)), "mx4 quantize")
    return q, sf


@native.on_tensor_device
def dequantize(q, sf, offsets=None, out=None):
    """The bf16 values of an operand produced by ``quantize`` with the same
    ``offsets``: exact, but for a value of 2^128, which reads as an infinity."""
    if not (q.is_cuda):
        raise ValueError("q must be on a CUDA device")
    index = q.get_device()
    groups = _groups(offsets, index)
    matrices, rows, K = _operand(q, sf, groups, index, "q")
    if not (offsets is None or q.dim() == 2):
        raise ValueError("a [matrices, rows, K] operand takes no offsets")
    shape = q.shape[:-1] + (K,)
    if out is None:
        out = q.new_empty(shape, dtype=torch.bfloat16)
    if not (out.dtype is torch.bfloat16 and out.shape == shape and out.get_device() == index and
            out.stride(-1) == 1 and (out.is_contiguous() or (out.dim() == 2 and out.stride(0) >= K))):
        raise ValueError("out must be bf16 [..., K] with contiguous rows that do not overlap, on q's device")
    ld = out.stride(0) if out.dim() == 2 and rows > 1 else K
    native.check(native.lib().tdb_mx4_dequantize(q.data_ptr(), sf.data_ptr(), matrices, rows, K,
                                                 None if offsets is None else offsets.data_ptr(), groups,
                                                 out.data_ptr(), ld, native.current_stream(index)), "mx4 dequantize")
    return out


def _product(qx, sfx, qw, sfw, offsets, bias, out, tile):
    if not (qx.is_cuda and qx.dim() == 2):
        raise ValueError("qx must be a quantized [rows, K] operand on a CUDA device")
    index = qx.get_device()
    groups = _groups(offsets, index)
    _, rows, K = _operand(qx, sfx, groups, index, "qx")
    matrices, N, Kw = _operand(qw, sfw, 0, index, "qw")
    if not (K == Kw):
        raise ValueError(f"the K extents differ: {K} and {Kw}")
    if not (matrices == max(groups, 1)):
        raise ValueError("qw must hold one matrix per group")
    if not (N > 0 and N % 8 == 0):
        raise ValueError("N must be a positive multiple of 8")
    if bias is not None:
        if not (bias.dtype is torch.bfloat16 and bias.numel() == matrices * N and bias.shape[-1] == N and
                bias.is_contiguous() and bias.get_device() == index):
            raise ValueError("bias must be contiguous bf16 [N] or [groups, N]")
    if out is None:
        out, ld = qx.new_empty((rows, N), dtype=torch.bfloat16), N
    else:
        ld, step = out.stride() if out.dim() == 2 else (0, 0)
        if rows <= 1:
            ld = N
        if not (out.dtype is torch.bfloat16 and out.shape == (rows, N) and step == 1 and ld >= N and
                out.get_device() == index):
            raise ValueError(f"out must be bf16 [{rows}, {N}] with contiguous rows that do not overlap, on the "
                             f"operands' device")
    native.check(native.lib().tdb_mx4_gemm(
        qx.data_ptr(), sfx.data_ptr(), qw.data_ptr(), sfw.data_ptr(), None if offsets is None else offsets.data_ptr(),
        matrices, out.data_ptr(), ld, rows, N, K, None if bias is None else bias.data_ptr(), tile,
        native.current_stream(index)), "mx4 product")
    return out


@native.on_tensor_device
def linear(qx, sfx, qw, sfw, bias=None, out=None, tile=0):
    """``values(qx) @ values(qw)^T (+ bias)`` in bf16 with fp32 accumulation;
    qx [M, K], qw [N, K] from ``quantize``."""
    if not (qw.dim() == 2):
        raise ValueError("qw must be a quantized [N, K] matrix")
    return _product(qx, sfx, qw, sfw, None, bias, out, tile)


@native.on_tensor_device
def grouped_linear(qx, sfx, qw, sfw, offsets, bias=None, out=None, tile=0):
    """``values(qx)[r] @ values(qw)[g]^T (+ bias[g])`` for the rows r of group
    g; qx [R, K] quantized with these ``offsets``, qw [groups, N, K], bias
    [groups, N].  Rows outside every group keep their contents."""
    if not (offsets is not None and qw.dim() == 3):
        raise ValueError("grouped_linear needs offsets and a quantized [groups, N, K] operand")
    return _product(qx, sfx, qw, sfw, offsets, bias, out, tile)
