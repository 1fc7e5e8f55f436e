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
tensors' device and are deterministic: equal calls give equal bits (a different
``tile`` or ``native.grid_limit`` may add in another order).  ``tile`` asks for a tile shape (0: by
the sizes; see ``pick_tile`` in csrc/grouped.cu), for measurements.
"""
from __future__ import annotations

import ctypes

import torch

from . import native
from .gemm import BIAS, BIAS_GELU, GELU_BWD, STORE

V, I, I64, LL = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_longlong

native.register("tdb_grouped_pick_tile", [I, LL, I, I, I])
native.register("tdb_grouped_gemm", [V, I64, V, I, V, I, V, I64, I, I, I, I, V, V, I64, V, I, V])
native.register("tdb_grouped_weight_grad", [V, I64, V, I64, V, I, V, I, I, I, I, I, V])
native.register("tdb_grouped_bias_grad", [V, I64, V, I, V, I, I, I, V])

MAX_GROUPS = 1024


def _rows(t, rows, cols, device, what):
    """Row stride of a bf16 [rows, cols] matrix with contiguous rows."""
    if t.dtype is not torch.bfloat16:
        raise TypeError(f"{what} must be bf16")
    ld, step = t.stride() if t.dim() == 2 else (0, 0)
    if rows <= 1:
        ld = cols
    if not (rows < 2 ** 31 and cols < 2 ** 31):
        raise ValueError(f"{what} must have fewer than 2^31 rows and columns")
    if not (t.shape == (rows, cols) and step == 1 and ld >= cols and t.get_device() == device):
        raise ValueError(f"{what} must be [{rows}, {cols}] with contiguous rows that do not overlap, on the "
                         f"operands' device")
    return ld


def _offsets(offsets, groups, device):
    if not (offsets.dtype is torch.int32 and offsets.dim() == 1 and offsets.is_contiguous() and
            offsets.get_device() == device):
        raise ValueError("offsets must be a contiguous int32 vector on the operands' device")
    if not (offsets.numel() == groups + 1):
        raise ValueError(f"offsets must have groups + 1 = {groups + 1} entries")
    if not (1 <= groups <= MAX_GROUPS):
        raise ValueError(f"the number of groups must be 1..{MAX_GROUPS}")


def _fp32(out, shape, device, what):
    if out.dtype is not torch.float32:
        raise TypeError(f"{what} is fp32")
    if not (out.shape == shape and out.is_contiguous() and out.get_device() == device):
        raise ValueError(f"out_f32 must be contiguous {list(shape)} on the operands' device")


def _gemm(a, w, offsets, data_grad, mode, out, bias, aux, aux_out, tile):
    if not (a.dim() == 2 and a.is_cuda):
        raise ValueError("the row operand must be a matrix on a CUDA device")
    index = a.get_device()
    if w.dtype is not torch.bfloat16:
        raise TypeError("w must be bf16")
    if not (w.dim() == 3 and w.is_contiguous() and w.get_device() == index):
        raise ValueError("w must be a contiguous [groups, N, K] tensor on the operands' device")
    groups, N, K = w.shape
    if data_grad:
        N, K = K, N
    rows = a.shape[0]
    if not (N > 0 and K > 0 and N % 8 == 0 and K % 8 == 0):
        raise ValueError("N and K must be positive multiples of 8")
    lda = _rows(a, rows, K, index, "dy" if data_grad else "x")
    _offsets(offsets, groups, index)
    if bias is not None:
        if not (bias.dtype is torch.bfloat16 and bias.shape == (groups, N) and bias.is_contiguous() and
                bias.get_device() == index):
            raise ValueError(f"bias must be contiguous bf16 [{groups}, {N}] on the operands' device")
    if out is None:
        out, ldc = a.new_empty((rows, N)), N
    else:
        ldc = _rows(out, rows, N, index, "out")
    pre = aux_out if aux_out is not None else aux
    ld_aux = 0 if pre is None else _rows(pre, rows, N, index, "the pre-activation")
    native.check(native.lib().tdb_grouped_gemm(
        a.data_ptr(), lda, w.data_ptr(), data_grad, offsets.data_ptr(), groups, out.data_ptr(), ldc, rows, N, K, mode,
        None if bias is None else bias.data_ptr(), None if aux is None else aux.data_ptr(), ld_aux,
        None if aux_out is None else aux_out.data_ptr(), tile, native.current_stream(index)), "grouped gemm")
    return out


@native.on_tensor_device
def linear(x, w, offsets, bias=None, out=None, tile=0):
    """``x[r] @ w[g]^T (+ bias[g])`` for the rows r of group g; x [R, K],
    w [groups, N, K], bias [groups, N] -> [R, N]."""
    return _gemm(x, w, offsets, 0, STORE if bias is None else BIAS, out, bias, None, None, tile)


@native.on_tensor_device
def linear_gelu(x, w, offsets, bias=None, pre_out=None, out=None, tile=0):
    """Returns (gelu(z), z) with z = x[r] @ w[g]^T (+ bias[g]) from one kernel.
    The activation is taken of the fp32 sum; z is its bf16 rounding."""
    if not (x.dim() == 2 and w.dim() == 3):
        raise ValueError("x must be [R, K] and w [groups, N, K]")
    if pre_out is None:
        pre_out = x.new_empty((x.shape[0], w.shape[1]))
    return _gemm(x, w, offsets, 0, BIAS_GELU, out, bias, None, pre_out, tile), pre_out


@native.on_tensor_device
def matmul_nt(dy, w, offsets, out=None, gelu_pre=None, tile=0):
    """``dy[r] @ w[g]`` (optionally times gelu'(gelu_pre)); dy [R, N],
    w [groups, N, K] -> [R, K]."""
    return _gemm(dy, w, offsets, 1, STORE if gelu_pre is None else GELU_BWD, out, None, gelu_pre, None, tile)


@native.on_tensor_device
def weight_grad(dy, x, offsets, out_f32=None, accumulate=True, tile=0):
    """``out_f32[g] (+)= dy_g^T @ x_g`` in fp32, [groups, N, K]; an empty group
    adds nothing (or gets zeros without ``accumulate``)."""
    if not (dy.dim() == 2 and x.dim() == 2 and dy.is_cuda):
        raise ValueError("dy and x must be matrices on a CUDA device")
    index = dy.get_device()
    rows, N = dy.shape
    K = x.shape[1]
    groups = offsets.numel() - 1
    _offsets(offsets, groups, index)
    if not (N > 0 and K > 0 and N % 8 == 0 and K % 8 == 0):
        raise ValueError("N and K must be positive multiples of 8")
    ldy = _rows(dy, rows, N, index, "dy")
    ldx = _rows(x, rows, K, index, "x")
    if out_f32 is None:
        out_f32 = torch.empty((groups, N, K), dtype=torch.float32, device=dy.device)
        accumulate = False
    else:
        _fp32(out_f32, (groups, N, K), index, "the weight gradient")
    native.check(native.lib().tdb_grouped_weight_grad(
        dy.data_ptr(), ldy, x.data_ptr(), ldx, offsets.data_ptr(), groups, out_f32.data_ptr(), rows, N, K,
        bool(accumulate), tile, native.current_stream(index)), "grouped weight gradient")
    return out_f32


@native.on_tensor_device
def bias_grad(dy, offsets, out_f32=None, accumulate=True):
    """``out_f32[g] (+)= `` the sum of dy's rows of group g, fp32 [groups, N]."""
    if not (dy.dim() == 2 and dy.is_cuda):
        raise ValueError("dy must be a matrix on a CUDA device")
    index = dy.get_device()
    rows, N = dy.shape
    groups = offsets.numel() - 1
    _offsets(offsets, groups, index)
    if not (N > 0 and N % 8 == 0):
        raise ValueError("N must be a positive multiple of 8")
    ldy = _rows(dy, rows, N, index, "dy")
    if out_f32 is None:
        out_f32 = torch.empty((groups, N), dtype=torch.float32, device=dy.device)
        accumulate = False
    else:
        _fp32(out_f32, (groups, N), index, "the bias gradient")
    native.check(native.lib().tdb_grouped_bias_grad(dy.data_ptr(), ldy, offsets.data_ptr(), groups, out_f32.data_ptr(),
                                                    rows, N, bool(accumulate), native.current_stream(index)),
                 "grouped bias gradient")
    return out_f32
