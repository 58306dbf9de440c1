"""Layer normalisation of a transformer block: autograd Functions over the sm_100a kernels.

* ``cuda_layer_norm(x, weight, bias, eps)``: ``nn.LayerNorm`` over the last axis
  (the ``ln1`` / ``ln2`` / ``ln_f`` and ``norm`` layers of the reference models,
  ``src/isa/language/models.py:81-177``, ``src/isa/vision/models.py:93-250``).
* ``cuda_add_layer_norm(x, delta, weight, bias, eps)``: the residual sum in front
  of it as well, ``h = x + delta; y = LN(h)``, in one pass; returns ``(y, h)``.

Inputs are fp32, bf16 or fp16 with rows of contiguous elements (any row stride;
other layouts are copied).  Statistics and sums are fp32, results are rounded
once.  ``out_dtype`` is the type of ``y``: fp32 streams may hand out any of the
three, 16-bit streams their own type or fp32.  The backward is one pass over the
rows and a fixed-order reduction for the weight gradients, so it gives the same
bits every time; it cannot be differentiated again.

A backward captured into a CUDA graph follows torch's rule: no eager graph of the
same leaf parameters may be alive during the capture (``del`` the warm-up's
outputs and losses first).
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from isa_b200 import _lib

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check_inputs(x: torch.Tensor, delta: Optional[torch.Tensor], weight: Optional[torch.Tensor],
                  bias: Optional[torch.Tensor], eps: float, out_dtype: torch.dtype) -> None:
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor: the layer norm kernels have no CPU implementation")
    if x.dim() < 1:
        raise RuntimeError("x must have at least one axis")
    if x.dtype not in _TYPES:
        raise RuntimeError(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    cols = x.shape[-1]
    if not 1 <= cols <= _lib.LAYER_NORM_MAX_COLS:
        raise RuntimeError(f"layer norm takes 1 to {_lib.LAYER_NORM_MAX_COLS} columns, got {cols}")
    if not eps >= 0.0:
        raise RuntimeError(f"eps must be >= 0, got {eps}")
    if out_dtype not in _TYPES or (x.dtype != torch.float32 and out_dtype not in (x.dtype, torch.float32)):
        raise RuntimeError(f"out_dtype {out_dtype} is not available for {x.dtype} inputs")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        if t.device != x.device:
            raise RuntimeError(f"{name} must be on the device of x")
        if t.dtype not in _TYPES:
            raise RuntimeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
        if t.shape != (cols,):
            raise RuntimeError(f"{name} must have shape ({cols},), got {tuple(t.shape)}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError("weight and bias must have one type")
    if delta is not None:
        if delta.device != x.device:
            raise RuntimeError("delta must be on the device of x")
        if delta.shape != x.shape:
            raise RuntimeError(f"delta must have the shape of x: {tuple(delta.shape)}, {tuple(x.shape)}")
        if delta.dtype not in _TYPES or (x.dtype != torch.float32 and delta.dtype != x.dtype):
            raise RuntimeError(f"delta {delta.dtype} is not available for {x.dtype} streams")


def _rows(t: torch.Tensor, cols: int) -> Tuple[torch.Tensor, int]:
    """``t`` as rows of contiguous elements, and their stride."""
    if t.is_contiguous():
        return t, cols
    r = t if t.dim() == 2 else t.reshape(-1, cols)
    if cols > 1 and r.stride(1) != 1:
        r = r.contiguous()
    return r, (r.stride(0) if r.shape[0] > 1 else cols)


def _forward(x, delta, weight, bias, eps, out_dtype, keep):
    """Returns (y, h or None, [mean, rstd] or None, weight as read)."""
    cols = x.shape[-1]
    rows = x.numel() // cols
    x2, x_stride = _rows(x, cols)
    d2, d_stride = (None, 0) if delta is None else _rows(delta, cols)
    w = None if weight is None else weight.contiguous()
    b = None if bias is None else bias.contiguous()
    y = x.new_empty(x.shape, dtype=out_dtype)
    h = None if delta is None else x.new_empty(x.shape)
    stats = x.new_empty((2, rows), dtype=torch.float32) if keep else None
    with _lib.on_device(x.device):
        _lib.layer_norm_forward(x2, x_stride, d2, d_stride, w, b, rows, cols, eps, h, y, stats)
    return y, h, stats, w


def _backward(ctx, dy, dh):
    """Gradients (dx, d delta, dw, db) as far as they are needed."""
    src, weight, stats = ctx.saved_tensors
    need_x, need_d, need_w, need_b = ctx.need
    shape, d_dtype, w_dtype = ctx.meta
    cols = shape[-1]
    if dy is None:  # only the sum was used
        zero = [torch.zeros(cols, dtype=w_dtype, device=src.device) if n else None for n in (need_w, need_b)]
        return dh if need_x else None, dh.to(d_dtype) if need_d else None, *zero
    g2, g_stride = _rows(dy, cols)
    s2, s_stride = _rows(dh, cols) if dh is not None else (None, 0)
    h2, h_stride = _rows(src, cols)
    # one gradient for both where stream and branch have one type
    shared = need_d and d_dtype == src.dtype
    dx = src.new_empty(shape) if need_x or shared else None
    dd = src.new_empty(shape, dtype=d_dtype) if need_d and not shared else None
    dw = src.new_empty(cols, dtype=w_dtype) if need_w else None
    db = src.new_empty(cols, dtype=w_dtype) if need_b else None
    with _lib.on_device(src.device):
        _lib.layer_norm_backward(g2, g_stride, s2, s_stride, h2, h_stride, weight, w_dtype, stats,
                                 src.numel() // cols, cols, dx, dd, dw, db)
    return dx if need_x else None, dx if shared else dd, dw, db


class LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype):
        ctx.need = (ctx.needs_input_grad[0], False, ctx.needs_input_grad[1], ctx.needs_input_grad[2])
        y, _, stats, w = _forward(x, None, weight, bias, eps, out_dtype, True)
        ctx.save_for_backward(x, w, stats)
        ctx.meta = (x.shape, None, _affine_dtype(weight, bias))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dx, _, dw, db = _backward(ctx, dy, None)
        return dx, dw, db, None, None


class AddLayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, weight, bias, eps, out_dtype):
        ctx.need = tuple(ctx.needs_input_grad[:4])
        y, h, stats, w = _forward(x, delta, weight, bias, eps, out_dtype, True)
        ctx.save_for_backward(h, w, stats)
        ctx.meta = (x.shape, delta.dtype, _affine_dtype(weight, bias))
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        if dy is None and dh is None:
            return (None,) * 6
        return *_backward(ctx, dy, dh), None, None


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _affine_dtype(weight, bias):
    t = weight if weight is not None else bias
    return None if t is None else t.dtype


def cuda_layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                    eps: float = 1e-5, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Layer norm over the last axis of ``x``; ``y`` in ``out_dtype`` (default: the type of ``x``)."""
    out_dtype = x.dtype if out_dtype is None else out_dtype
    _check_inputs(x, None, weight, bias, eps, out_dtype)
    if not _wants_grad(x, weight, bias):
        return _forward(x, None, weight, bias, eps, out_dtype, False)[0]
    return LayerNormFn.apply(x, weight, bias, eps, out_dtype)


def cuda_add_layer_norm(x: torch.Tensor, delta: torch.Tensor, weight: Optional[torch.Tensor] = None,
                        bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
                        out_dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``h = x + delta`` in the type of ``x`` and ``y = LN(h)`` in ``out_dtype``; returns ``(y, h)``.

    The branch ``delta`` of an fp32 stream may be any of the three types (the
    bf16 output of an autocast projection); a 16-bit stream takes its own type.
    """
    out_dtype = x.dtype if out_dtype is None else out_dtype
    _check_inputs(x, delta, weight, bias, eps, out_dtype)
    if not _wants_grad(x, delta, weight, bias):
        return _forward(x, delta, weight, bias, eps, out_dtype, False)[:2]
    return AddLayerNormFn.apply(x, delta, weight, bias, eps, out_dtype)
