"""Matrix products grouped by expert, with ragged group sizes
(``csrc/grouped.cuh`` + ``csrc/grouped.cu``).

``offsets`` (int32 [groups + 1], on the device) gives group g the rows
[offsets[g], offsets[g + 1]) of the row operands; ``w`` [groups, N, K] holds one
matrix per group.  Groups may be empty; rows outside every group are neither
used nor written.  The sizes stay on the device: no call synchronises.

* forward        ``y[r] = x[r] @ w[g]^T (+ bias[g])``   ``linear``, ``linear_gelu``
* data gradient  ``dx[r] = dy[r] @ w[g]``               ``matmul_nt``
* weight grad    ``dw[g] (+)= dy_g^T @ x_g``            ``weight_grad``
* bias grad      ``db[g] (+)= sum of dy_g``             ``bias_grad``

Operands are bf16 with 16-byte aligned rows (N, K and row strides multiples of
8), sums fp32, outputs bf16 (gradients of parameters fp32).  Offsets that
decrease or leave the rows are found on the device: the call computes nothing
and ``native.raise_on_status`` raises.  Calls run on the current stream of the
tensors' device and are deterministic.
"""
from __future__ import annotations

import ctypes

from . import native
from .gemm import BIAS, BIAS_GELU, GELU_BWD, STORE

V, I, I64, LL = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_longlong

native.register("tdb_grouped_pick_tile", [I, LL, I, I, I])
native.register("tdb_grouped_gemm", [V, I64, V, I, V, I, V, I64, I, I, I, I, V, V, I64, V, I, V])
native.register("tdb_grouped_weight_grad", [V, I64, V, I64, V, I, V, I, I, I, I, I, V])
native.register("tdb_grouped_bias_grad", [V, I64, V, I, V, I, I, I, V])

MAX_GROUPS = 1024


def _need(cond, msg):
    if not cond:
        raise ValueError(msg)


def _rows(t, rows, cols, device, what):
    """Row stride of a bf16 [rows, cols] matrix with contiguous rows."""
    import torch
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{what} must be bf16")
    _need(t.dim() == 2 and tuple(t.shape) == (rows, cols) and t.stride(1) == 1 and t.device == device,
          f"{what} must be [{rows}, {cols}] with a contiguous last dimension on the operands' device")
    _need(rows <= 1 or t.stride(0) >= cols, f"{what}: rows must not overlap")
    return t.stride(0) if rows > 1 else cols


def _offsets(offsets, groups, device):
    import torch
    _need(offsets.dtype == torch.int32 and offsets.dim() == 1 and offsets.is_contiguous() and
          offsets.device == device, "offsets must be a contiguous int32 vector on the operands' device")
    _need(offsets.numel() == groups + 1, f"offsets must have groups + 1 = {groups + 1} entries")
    _need(1 <= groups <= MAX_GROUPS, f"the number of groups must be 1..{MAX_GROUPS}")


def _operands(a, w, what):
    import torch
    _need(a.dim() == 2 and a.is_cuda, f"{what} must be a matrix on a CUDA device")
    if w.dtype != torch.bfloat16:
        raise TypeError("w must be bf16")
    _need(w.dim() == 3 and w.is_contiguous() and w.device == a.device,
          "w must be a contiguous [groups, N, K] tensor on the operands' device")


def _gemm(a, w, offsets, data_grad, mode, out, bias=None, aux=None, aux_out=None, tile=0):
    import torch
    groups = w.shape[0]
    K, N = (w.shape[1], w.shape[2]) if data_grad else (w.shape[2], w.shape[1])
    dev = a.device
    rows = a.shape[0]
    _need(N > 0 and K > 0 and N % 8 == 0 and K % 8 == 0, "N and K must be positive multiples of 8")
    lda = _rows(a, rows, K, dev, "dy" if data_grad else "x")
    _offsets(offsets, groups, dev)
    if bias is not None:
        _need(bias.dtype == torch.bfloat16 and tuple(bias.shape) == (groups, N) and bias.is_contiguous() and
              bias.device == dev, f"bias must be contiguous bf16 [{groups}, {N}] on the operands' device")
    with native.on_device(dev):
        out = torch.empty((rows, N), dtype=torch.bfloat16, device=dev) if out is None else out
        ldc = _rows(out, rows, N, dev, "out")
        pre = aux_out if aux_out is not None else aux
        ld_aux = 0 if pre is None else _rows(pre, rows, N, dev, "the pre-activation")
        native.check(native.lib().tdb_grouped_gemm(
            a.data_ptr(), lda, w.data_ptr(), int(data_grad), offsets.data_ptr(), groups, out.data_ptr(), ldc, rows, N, K,
            mode, 0 if bias is None else bias.data_ptr(), 0 if aux is None else aux.data_ptr(), ld_aux,
            0 if aux_out is None else aux_out.data_ptr(), tile, native.stream_ptr()), "grouped gemm")
    return out


def linear(x, w, offsets, bias=None, out=None, tile=0):
    """``x[r] @ w[g]^T (+ bias[g])`` for the rows r of group g; x [R, K],
    w [groups, N, K], bias [groups, N] -> [R, N]."""
    _operands(x, w, "x")
    return _gemm(x, w, offsets, False, STORE if bias is None else BIAS, out, bias=bias, tile=tile)


def linear_gelu(x, w, offsets, bias=None, pre_out=None, out=None, tile=0):
    """Returns (gelu(z), z) with z = x[r] @ w[g]^T (+ bias[g]) from one kernel.
    The activation is taken of the fp32 sum; z is its bf16 rounding."""
    import torch
    _operands(x, w, "x")
    if pre_out is None:
        pre_out = torch.empty((x.shape[0], w.shape[1]), dtype=torch.bfloat16, device=x.device)
    y = _gemm(x, w, offsets, False, BIAS_GELU, out, bias=bias, aux_out=pre_out, tile=tile)
    return y, pre_out


def matmul_nt(dy, w, offsets, out=None, gelu_pre=None, tile=0):
    """``dy[r] @ w[g]`` (optionally times gelu'(gelu_pre)); dy [R, N],
    w [groups, N, K] -> [R, K]."""
    _operands(dy, w, "dy")
    return _gemm(dy, w, offsets, True, STORE if gelu_pre is None else GELU_BWD, out, aux=gelu_pre, tile=tile)


def weight_grad(dy, x, offsets, out_f32=None, accumulate=True, tile=0):
    """``out_f32[g] (+)= dy_g^T @ x_g`` in fp32, [groups, N, K]; an empty group
    adds nothing (or gets zeros without ``accumulate``)."""
    import torch
    _need(dy.dim() == 2 and x.dim() == 2 and dy.is_cuda, "dy and x must be matrices on a CUDA device")
    dev, rows = dy.device, dy.shape[0]
    N, K = dy.shape[1], x.shape[1]
    groups = offsets.numel() - 1
    _offsets(offsets, groups, dev)
    _need(N > 0 and K > 0 and N % 8 == 0 and K % 8 == 0, "N and K must be positive multiples of 8")
    ldy = _rows(dy, rows, N, dev, "dy")
    ldx = _rows(x, rows, K, dev, "x")
    with native.on_device(dev):
        if out_f32 is None:
            out_f32 = torch.empty((groups, N, K), dtype=torch.float32, device=dev)
            accumulate = False
        if out_f32.dtype != torch.float32:
            raise TypeError("the weight gradient is fp32")
        _need(tuple(out_f32.shape) == (groups, N, K) and out_f32.is_contiguous() and out_f32.device == dev,
              f"out_f32 must be contiguous [{groups}, {N}, {K}] on the operands' device")
        native.check(native.lib().tdb_grouped_weight_grad(
            dy.data_ptr(), ldy, x.data_ptr(), ldx, offsets.data_ptr(), groups, out_f32.data_ptr(), rows, N, K,
            int(bool(accumulate)), tile, native.stream_ptr()), "grouped weight gradient")
    return out_f32


def bias_grad(dy, offsets, out_f32=None, accumulate=True):
    """``out_f32[g] (+)= `` the sum of dy's rows of group g, fp32 [groups, N]."""
    import torch
    _need(dy.dim() == 2 and dy.is_cuda, "dy must be a matrix on a CUDA device")
    dev, (rows, N) = dy.device, dy.shape
    groups = offsets.numel() - 1
    _offsets(offsets, groups, dev)
    _need(N > 0 and N % 8 == 0, "N must be a positive multiple of 8")
    ldy = _rows(dy, rows, N, dev, "dy")
    with native.on_device(dev):
        if out_f32 is None:
            out_f32 = torch.empty((groups, N), dtype=torch.float32, device=dev)
            accumulate = False
        if out_f32.dtype != torch.float32:
            raise TypeError("the bias gradient is fp32")
        _need(tuple(out_f32.shape) == (groups, N) and out_f32.is_contiguous() and out_f32.device == dev,
              f"out_f32 must be contiguous [{groups}, {N}] on the operands' device")
        native.check(native.lib().tdb_grouped_bias_grad(dy.data_ptr(), ldy, offsets.data_ptr(), groups,
                                                        out_f32.data_ptr(), rows, N, int(bool(accumulate)),
                                                        native.stream_ptr()), "grouped bias gradient")
    return out_f32
