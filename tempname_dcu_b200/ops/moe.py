"""Mixture-of-experts routing and row exchange (``csrc/moe.cu``).

``route`` picks the ``top_k`` experts of every token and groups the choices by
expert; ``dispatch`` copies the token rows into that order, where the products
of ``ops.grouped`` take them, and ``combine`` brings the experts' rows back as
a weighted sum::

    r   = moe.route(logits, top_k=2)
    xs  = moe.dispatch(x, r)                                   # [tokens*k, H]
    h,z = grouped.linear_gelu(xs, w1, r.offsets, b1)
    ys  = grouped.linear(h, w2, r.offsets, b2)
    out = moe.combine(ys, r, residual=x)

    dys, dweights = moe.combine_bwd(dout, ys, r)
    ...                                                        # products' gradients
    dx      = moe.dispatch_bwd(dxs, r)
    dlogits = moe.route_bwd(logits, r, dweights)

A choice is (token t, j-th expert), numbered t * k + j.  Rows move as bf16,
weights and their gradients are fp32, sums are fp32 with one rounding.  A
logit of -inf closes an expert to a token (weight 0; a row of them routes to
the lowest indices with weight 0 and gets no gradient).  Everything is
deterministic.  Calls run on the current stream of the tensors' device.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Any

import torch

from . import native

V, I, I64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64

native.register("tdb_moe_route_scratch_ints", [I, I], restype=ctypes.c_longlong)
native.register("tdb_moe_route", [V, I, I64, I, I, I, I, V, V, V, V, V, V, V])
native.register("tdb_moe_route_bwd", [V, I, I64, I, I, I, I, V, V, V, V, I, I64, V])
native.register("tdb_moe_dispatch", [V, I64, I, I, I, V, V, I64, V])
native.register("tdb_moe_combine", [V, I64, I, I, I, V, V, V, I64, V, I64, V])
native.register("tdb_moe_combine_bwd", [V, I64, V, I64, I, I, I, V, V, V, I64, V, V])

MAX_EXPERTS = 512
MAX_TOP_K = 16


@dataclass(frozen=True, eq=False)
class Routing:
    """A batch's choices of experts, grouped.

    ids      int32 [tokens, k]    chosen experts, largest logit first
    weights  fp32  [tokens, k]    their weights
    offsets  int32 [experts + 1]  expert e holds grouped rows [offsets[e], offsets[e + 1])
    order    int32 [tokens * k]   grouped row -> choice (t * k + j); stable within an expert
    slots    int32 [tokens * k]   choice -> grouped row

    Checked when it is made; a slot outside the grouped rows is found by the
    kernels that use it and reported through the status word.
    """
    ids: Any
    weights: Any
    offsets: Any
    order: Any
    slots: Any
    normalize: bool = True

    def __post_init__(self):
        ids, weights, index = self.ids, self.weights, self.ids.get_device()
        if not (ids.dim() == 2 and ids.dtype is torch.int32 and ids.is_contiguous()):
            raise ValueError("ids must be contiguous int32 [tokens, k]")
        if not (weights.shape == ids.shape and weights.dtype is torch.float32 and weights.is_contiguous()):
            raise ValueError("weights must be contiguous fp32 [tokens, k]")
        for t in (self.offsets, self.order, self.slots):
            if not (t.dtype is torch.int32 and t.dim() == 1 and t.is_contiguous()):
                raise ValueError("offsets, order and slots must be contiguous int32 vectors")
            if not (t.get_device() == index):
                raise ValueError("the tensors must be on one device")
        if not (weights.get_device() == index):
            raise ValueError("the tensors must be on one device")
        if not (ids.shape[1] >= 1 and ids.shape[1] <= MAX_TOP_K and ids.numel() < 2 ** 31):
            raise ValueError(f"1..{MAX_TOP_K} choices per token, fewer than 2^31 in all")
        if not (self.slots.numel() == ids.numel() and self.order.numel() == ids.numel() and self.offsets.numel() > 1):
            raise ValueError("order and slots must have tokens * k entries, offsets experts + 1")

    @property
    def tokens(self):
        return self.ids.shape[0]

    @property
    def top_k(self):
        return self.ids.shape[1]

    @property
    def experts(self):
        return self.offsets.numel() - 1


def _routing(ids, weights, offsets, order, slots, normalize):
    """A Routing of tensors that ``route`` has just made itself."""
    r = object.__new__(Routing)
    r.__dict__.update(ids=ids, weights=weights, offsets=offsets, order=order, slots=slots, normalize=normalize)
    return r


def _check_routing(r, device):
    """(tokens, k) of a routing on the device of a call's tensors."""
    ids = r.ids
    if not (ids.get_device() == device):
        raise ValueError("the routing must be on the tensors' device")
    return ids.shape


def _rows(t, rows, cols, device, what):
    """Row stride of a bf16 [rows, cols] matrix with contiguous rows."""
    ld, step = t.stride() if t.dim() == 2 else (0, 0)
    if rows <= 1:
        ld = cols
    if not (t.dtype is torch.bfloat16 and t.shape == (rows, cols) and step == 1 and ld >= cols and
            t.get_device() == device):
        raise ValueError(f"{what} must be bf16 [{rows}, {cols}] with contiguous rows that do not overlap, on the "
                         f"tensors' device")
    return ld


def _columns(t, what):
    """(rows, columns, device) of a row operand."""
    if not (t.dim() == 2 and t.is_cuda):
        raise ValueError(f"{what} must be a matrix on a CUDA device")
    rows, cols = t.shape
    if not (cols > 0 and cols % 8 == 0 and cols < 2 ** 31 and rows < 2 ** 31):
        raise ValueError(f"{what} needs a multiple of 8 columns, and fewer than 2^31 rows and columns")
    return rows, cols, t.get_device()


def _logits(logits, what="logits"):
    """(tokens, experts, row stride, is bf16, device)."""
    if not (logits.dim() == 2 and logits.is_cuda):
        raise ValueError(f"{what} must be a [tokens, experts] matrix on a CUDA device")
    bf16 = logits.dtype is torch.bfloat16
    if not (bf16 or logits.dtype is torch.float32):
        raise ValueError(f"{what} must be fp32 or bf16")
    tokens, experts = logits.shape
    if not (1 <= experts <= MAX_EXPERTS):
        raise ValueError(f"the number of experts must be 1..{MAX_EXPERTS}")
    if not (tokens < 2 ** 31 // MAX_TOP_K):
        raise ValueError("at most 2^27 tokens")
    ld, step = logits.stride()
    if tokens <= 1:
        ld = experts
    if not ((step == 1 or experts == 1) and ld >= experts):
        raise ValueError(f"{what} needs contiguous rows that do not overlap")
    return tokens, experts, ld, int(bf16), logits.get_device()


@native.on_tensor_device
def route(logits, top_k, normalize=True):
    """Top-k experts of each token -> ``Routing``.

    The experts of the ``top_k`` largest logits (equal logits: the lower
    index first; NaN counts as the largest) with softmax weights over the
    chosen ones (``normalize``) or over all experts."""
    tokens, experts, ld, bf16, index = _logits(logits)
    if not (type(top_k) is int and 1 <= top_k <= min(experts, MAX_TOP_K)):
        raise ValueError(f"top_k must be 1..{MAX_TOP_K} and at most the number of experts")
    normalize = bool(normalize)
    dev = logits.device
    weights = torch.empty((tokens, top_k), dtype=torch.float32, device=dev)
    order = torch.empty(tokens * top_k, dtype=torch.int32, device=dev)
    slots = torch.empty_like(order)
    ids = torch.empty_like(weights, dtype=torch.int32)
    offsets = torch.empty(experts + 1, dtype=torch.int32, device=dev)
    lib = native.lib()
    ints = lib.tdb_moe_route_scratch_ints(tokens, experts)
    scratch = torch.empty(ints, dtype=torch.int32, device=dev) if ints else None
    native.check(lib.tdb_moe_route(logits.data_ptr(), bf16, ld, tokens, experts, top_k, normalize, ids.data_ptr(),
                                   weights.data_ptr(), offsets.data_ptr(), order.data_ptr(), slots.data_ptr(),
                                   None if scratch is None else scratch.data_ptr(), native.current_stream(index)),
                 "moe route")
    return _routing(ids, weights, offsets, order, slots, normalize)


@native.on_tensor_device
def route_bwd(logits, routing, dweights, out=None):
    """Gradient of ``route``'s weights with respect to the logits.  ``out``
    (fp32 or bf16 [tokens, experts], default: the logits' type) is written
    whole: 0 for experts that were not chosen when the weights are
    normalised."""
    tokens, experts, ld, bf16, index = _logits(logits)
    shape = _check_routing(routing, index)
    if not (shape[0] == tokens and routing.experts == experts):
        raise ValueError("routing and logits have different sizes")
    if not (dweights.shape == shape and dweights.dtype is torch.float32 and dweights.is_contiguous() and
            dweights.get_device() == index):
        raise ValueError("dweights must be contiguous fp32 [tokens, k] on the logits' device")
    if out is None:
        out, ld_out, out_bf16 = torch.empty_like(logits, memory_format=torch.contiguous_format), experts, bf16
    else:
        if not (out.shape == (tokens, experts)):
            raise ValueError("out must be [tokens, experts]")
        _, _, ld_out, out_bf16, out_index = _logits(out, "out")
        if not (out_index == index):
            raise ValueError("out must be on the logits' device")
    native.check(native.lib().tdb_moe_route_bwd(logits.data_ptr(), bf16, ld, tokens, experts, shape[1],
                                                bool(routing.normalize), routing.ids.data_ptr(),
                                                routing.weights.data_ptr(), dweights.data_ptr(), out.data_ptr(),
                                                out_bf16, ld_out, native.current_stream(index)), "moe route backward")
    return out


@native.on_tensor_device
def dispatch(x, routing, out=None):
    """Rows grouped by expert: ``out[slots[t*k + j]] = x[t]``, [tokens*k, H]."""
    tokens, H, index = _columns(x, "x")
    shape = _check_routing(routing, index)
    if not (shape[0] == tokens):
        raise ValueError("routing and x have different numbers of tokens")
    k = shape[1]
    ldx = _rows(x, tokens, H, index, "x")
    if out is None:
        out, ldo = x.new_empty((tokens * k, H)), H
    else:
        ldo = _rows(out, tokens * k, H, index, "out")
    native.check(native.lib().tdb_moe_dispatch(x.data_ptr(), ldx, tokens, k, H, routing.slots.data_ptr(),
                                               out.data_ptr(), ldo, native.current_stream(index)), "moe dispatch")
    return out


def _combine(y, routing, weighted, residual, out, what):
    rows, H, index = _columns(y, "the grouped rows")
    tokens, k = _check_routing(routing, index)
    ldy = _rows(y, tokens * k, H, index, "the grouped rows")
    ldr = 0 if residual is None else _rows(residual, tokens, H, index, "residual")
    if out is None:
        out, ldo = y.new_empty((tokens, H)), H
    else:
        ldo = _rows(out, tokens, H, index, "out")
    native.check(native.lib().tdb_moe_combine(y.data_ptr(), ldy, tokens, k, H, routing.slots.data_ptr(),
                                              routing.weights.data_ptr() if weighted else None,
                                              None if residual is None else residual.data_ptr(), ldr, out.data_ptr(),
                                              ldo, native.current_stream(index)), what)
    return out


@native.on_tensor_device
def dispatch_bwd(dxs, routing, residual=None, out=None):
    """Gradient of ``dispatch``: ``out[t] = (residual[t] +) sum_j dxs[slots[t*k + j]]``."""
    return _combine(dxs, routing, False, residual, out, "moe dispatch backward")


@native.on_tensor_device
def combine(ys, routing, residual=None, out=None):
    """``out[t] = (residual[t] +) sum_j weights[t, j] * ys[slots[t*k + j]]``, [tokens, H]."""
    return _combine(ys, routing, True, residual, out, "moe combine")


@native.on_tensor_device
def combine_bwd(dout, ys, routing, out=None):
    """Gradients of ``combine``: (dys [tokens*k, H] bf16, dweights [tokens, k]
    fp32).  The residual's gradient is ``dout`` itself."""
    tokens, H, index = _columns(dout, "dout")
    shape = _check_routing(routing, index)
    if not (shape[0] == tokens):
        raise ValueError("routing and dout have different numbers of tokens")
    k = shape[1]
    ldd = _rows(dout, tokens, H, index, "dout")
    ldy = _rows(ys, tokens * k, H, index, "ys")
    if out is None:
        out, ldo = dout.new_empty((tokens * k, H)), H
    else:
        ldo = _rows(out, tokens * k, H, index, "out")
    dweights = torch.empty_like(routing.weights)
    native.check(native.lib().tdb_moe_combine_bwd(dout.data_ptr(), ldd, ys.data_ptr(), ldy, tokens, k, H,
                                                  routing.slots.data_ptr(), routing.weights.data_ptr(),
                                                  out.data_ptr(), ldo, dweights.data_ptr(),
                                                  native.current_stream(index)), "moe combine backward")
    return out, dweights
