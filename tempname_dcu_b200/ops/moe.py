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


@dataclass
class Routing:
    """A batch's choices of experts, grouped.

    ids      int32 [tokens, k]    chosen experts, largest logit first
    weights  fp32  [tokens, k]    their weights
    offsets  int32 [experts + 1]  expert e holds grouped rows [offsets[e], offsets[e + 1])
    order    int32 [tokens * k]   grouped row -> choice (t * k + j); stable within an expert
    slots    int32 [tokens * k]   choice -> grouped row
    """
    ids: Any
    weights: Any
    offsets: Any
    order: Any
    slots: Any
    normalize: bool = True

    @property
    def tokens(self):
        return self.ids.shape[0]

    @property
    def top_k(self):
        return self.ids.shape[1]

    @property
    def experts(self):
        return self.offsets.numel() - 1


def _need(cond, msg):
    if not cond:
        raise ValueError(msg)


def _check_routing(r, device):
    import torch
    _need(r.ids.dim() == 2 and r.ids.dtype == torch.int32 and r.ids.is_contiguous() and r.ids.device == device,
          "routing ids must be contiguous int32 [tokens, k] on the tensors' device")
    _need(r.weights.shape == r.ids.shape and r.weights.dtype == torch.float32 and r.weights.is_contiguous() and
          r.weights.device == device, "routing weights must be contiguous fp32 [tokens, k] on the tensors' device")
    _need(r.slots.numel() == r.ids.numel() and r.slots.dtype == torch.int32 and r.slots.is_contiguous() and
          r.slots.device == device, "routing slots must be contiguous int32 [tokens * k] on the tensors' device")


def _rows(t, rows, cols, device, what):
    import torch
    _need(t.dim() == 2 and t.dtype == torch.bfloat16 and tuple(t.shape) == (rows, cols) and
          (t.stride(1) == 1 or cols == 1) and t.device == device,
          f"{what} must be bf16 [{rows}, {cols}] with a contiguous last dimension on the tensors' device")
    _need(rows <= 1 or t.stride(0) >= cols, f"{what}: rows must not overlap")
    return t.stride(0) if rows > 1 else cols


def _logits(logits):
    import torch
    _need(logits.dim() == 2 and logits.is_cuda and logits.dtype in (torch.float32, torch.bfloat16),
          "logits must be an fp32 or bf16 [tokens, experts] matrix on a CUDA device")
    tokens, experts = logits.shape
    _need(1 <= experts <= MAX_EXPERTS, f"the number of experts must be 1..{MAX_EXPERTS}")
    _need(logits.stride(1) == 1 or experts == 1, "logits need a contiguous last dimension")
    _need(tokens <= 1 or logits.stride(0) >= experts, "logits: rows must not overlap")
    return tokens, experts, logits.stride(0) if tokens > 1 else experts


def route(logits, top_k, normalize=True):
    """Top-k experts of each token -> ``Routing``.

    The experts of the ``top_k`` largest logits (equal logits: the lower
    index first; NaN counts as the largest) with softmax weights over the
    chosen ones (``normalize``) or over all experts."""
    import torch
    tokens, experts, ld = _logits(logits)
    _need(type(top_k) is int and 1 <= top_k <= min(experts, MAX_TOP_K),
          f"top_k must be 1..{MAX_TOP_K} and at most the number of experts")
    dev = logits.device
    lib = native.lib()
    with native.on_device(dev):
        ids = torch.empty((tokens, top_k), dtype=torch.int32, device=dev)
        weights = torch.empty((tokens, top_k), dtype=torch.float32, device=dev)
        offsets = torch.empty(experts + 1, dtype=torch.int32, device=dev)
        order = torch.empty(tokens * top_k, dtype=torch.int32, device=dev)
        slots = torch.empty(tokens * top_k, dtype=torch.int32, device=dev)
        ints = int(lib.tdb_moe_route_scratch_ints(tokens, experts))
        scratch = torch.empty(ints, dtype=torch.int32, device=dev) if ints else None
        native.check(lib.tdb_moe_route(logits.data_ptr(), int(logits.dtype == torch.bfloat16), ld, tokens, experts,
                                       top_k, int(bool(normalize)), ids.data_ptr(), weights.data_ptr(),
                                       offsets.data_ptr(), order.data_ptr(), slots.data_ptr(),
                                       0 if scratch is None else scratch.data_ptr(), native.stream_ptr()),
                     "moe route")
    return Routing(ids=ids, weights=weights, offsets=offsets, order=order, slots=slots, normalize=bool(normalize))


def route_bwd(logits, routing, dweights, out=None):
    """Gradient of ``route``'s weights with respect to the logits.  ``out``
    (fp32 or bf16 [tokens, experts], default: the logits' type) is written
    whole: 0 for experts that were not chosen when the weights are
    normalised."""
    import torch
    tokens, experts, ld = _logits(logits)
    dev = logits.device
    _check_routing(routing, dev)
    top_k = routing.top_k
    _need(routing.tokens == tokens and routing.experts == experts, "routing and logits have different sizes")
    _need(dweights.shape == routing.ids.shape and dweights.dtype == torch.float32 and dweights.is_contiguous() and
          dweights.device == dev, "dweights must be contiguous fp32 [tokens, k] on the logits' device")
    with native.on_device(dev):
        out = torch.empty((tokens, experts), dtype=logits.dtype, device=dev) if out is None else out
        _need(out.dtype in (torch.float32, torch.bfloat16) and tuple(out.shape) == (tokens, experts) and
              (out.stride(1) == 1 or experts == 1) and (tokens <= 1 or out.stride(0) >= experts) and
              out.device == dev, "out must be fp32 or bf16 [tokens, experts] with a contiguous last dimension")
        native.check(native.lib().tdb_moe_route_bwd(logits.data_ptr(), int(logits.dtype == torch.bfloat16), ld, tokens,
                                                    experts, top_k, int(routing.normalize), routing.ids.data_ptr(),
                                                    routing.weights.data_ptr(), dweights.data_ptr(), out.data_ptr(),
                                                    int(out.dtype == torch.bfloat16),
                                                    out.stride(0) if tokens > 1 else experts,
                                                    native.stream_ptr()), "moe route backward")
    return out


def dispatch(x, routing, out=None):
    """Rows grouped by expert: ``out[slots[t*k + j]] = x[t]``, [tokens*k, H]."""
    import torch
    _need(x.dim() == 2 and x.is_cuda and x.shape[1] % 8 == 0 and x.shape[1] > 0,
          "x must be [tokens, H] on a CUDA device with H a multiple of 8")
    tokens, H = x.shape
    dev = x.device
    _check_routing(routing, dev)
    k = routing.top_k
    _need(routing.tokens == tokens, "routing and x have different numbers of tokens")
    ldx = _rows(x, tokens, H, dev, "x")
    with native.on_device(dev):
        out = torch.empty((tokens * k, H), dtype=torch.bfloat16, device=dev) if out is None else out
        ldo = _rows(out, tokens * k, H, dev, "out")
        native.check(native.lib().tdb_moe_dispatch(x.data_ptr(), ldx, tokens, k, H, routing.slots.data_ptr(),
                                                   out.data_ptr(), ldo, native.stream_ptr()), "moe dispatch")
    return out


def _combine(y, routing, weighted, residual, out, what):
    import torch
    _need(y.dim() == 2 and y.is_cuda and y.shape[1] % 8 == 0 and y.shape[1] > 0,
          "the grouped rows must be [tokens*k, H] on a CUDA device with H a multiple of 8")
    dev = y.device
    _check_routing(routing, dev)
    tokens, k, H = routing.tokens, routing.top_k, y.shape[1]
    ldy = _rows(y, tokens * k, H, dev, "the grouped rows")
    ldr = 0 if residual is None else _rows(residual, tokens, H, dev, "residual")
    with native.on_device(dev):
        out = torch.empty((tokens, H), dtype=torch.bfloat16, device=dev) if out is None else out
        ldo = _rows(out, tokens, H, dev, "out")
        native.check(native.lib().tdb_moe_combine(y.data_ptr(), ldy, tokens, k, H, routing.slots.data_ptr(),
                                                  routing.weights.data_ptr() if weighted else 0,
                                                  0 if residual is None else residual.data_ptr(), ldr, out.data_ptr(),
                                                  ldo, native.stream_ptr()), what)
    return out


def dispatch_bwd(dxs, routing, residual=None, out=None):
    """Gradient of ``dispatch``: ``out[t] = (residual[t] +) sum_j dxs[slots[t*k + j]]``."""
    return _combine(dxs, routing, False, residual, out, "moe dispatch backward")


def combine(ys, routing, residual=None, out=None):
    """``out[t] = (residual[t] +) sum_j weights[t, j] * ys[slots[t*k + j]]``, [tokens, H]."""
    return _combine(ys, routing, True, residual, out, "moe combine")


def combine_bwd(dout, ys, routing, out=None):
    """Gradients of ``combine``: (dys [tokens*k, H] bf16, dweights [tokens, k]
    fp32).  The residual's gradient is ``dout`` itself."""
    import torch
    _need(dout.dim() == 2 and dout.is_cuda and dout.shape[1] % 8 == 0 and dout.shape[1] > 0,
          "dout must be [tokens, H] on a CUDA device with H a multiple of 8")
    tokens, H = dout.shape
    dev = dout.device
    _check_routing(routing, dev)
    k = routing.top_k
    _need(routing.tokens == tokens, "routing and dout have different numbers of tokens")
    ldd = _rows(dout, tokens, H, dev, "dout")
    ldy = _rows(ys, tokens * k, H, dev, "ys")
    with native.on_device(dev):
        out = torch.empty((tokens * k, H), dtype=torch.bfloat16, device=dev) if out is None else out
        ldo = _rows(out, tokens * k, H, dev, "out")
        dweights = torch.empty((tokens, k), dtype=torch.float32, device=dev)
        native.check(native.lib().tdb_moe_combine_bwd(dout.data_ptr(), ldd, ys.data_ptr(), ldy, tokens, k, H,
                                                      routing.slots.data_ptr(), routing.weights.data_ptr(),
                                                      out.data_ptr(), ldo, dweights.data_ptr(), native.stream_ptr()),
                     "moe combine backward")
    return out, dweights
