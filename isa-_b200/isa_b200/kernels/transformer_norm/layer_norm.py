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
    r = t if t.dim() == 2 else t.reshape(-1, cols)
    if cols > 1 and r.stride(1) != 1:
        r = r.contiguous()
    return r, (r.stride(0) if r.shape[0] > 1 else cols)


class _on_device:
    """Makes ``device`` current for a launch; free where it is already."""

    def __init__(self, device: torch.device):
        self.to = device.index
        self.back = None

    def __enter__(self):
        if torch.cuda.current_device() != self.to:
            self.back = torch.cuda.device(self.to)
            self.back.__enter__()

    def __exit__(self, *exc):
        if self.back is not None:
            self.back.__exit__(*exc)


def _forward(x, delta, weight, bias, eps, out_dtype, stats):
    """Returns (y, h or None, mean, rstd, h as rows, its stride)."""
    cols = x.shape[-1]
    x2, x_stride = _rows(x.detach(), cols)
    rows = x2.shape[0]
    d2, d_stride = (None, 0) if delta is None else _rows(delta.detach(), cols)
    w = None if weight is None else weight.detach().contiguous()
    b = None if bias is None else bias.detach().contiguous()
    y = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    h = None if delta is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = torch.empty(rows, dtype=torch.float32, device=x.device) if stats else None
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if stats else None
    with _on_device(x.device):
        _lib.layer_norm_forward(x2, x_stride, d2, d_stride, w, b, rows, cols, float(eps), h, y, mean, rstd)
    return y, h, mean, rstd, w


def _backward(ctx, dy, dh):
    """Gradients (dx, d delta, dw, db) as far as they are needed."""
    src, weight, mean, rstd = ctx.saved_tensors
    need_x, need_d, need_w, need_b = ctx.need
    shape, x_dtype, d_dtype, w_dtype = ctx.meta
    cols = shape[-1]
    if dy is None:  # only the sum was used
        one = dh
        zero = [torch.zeros(cols, dtype=w_dtype, device=src.device) if n else None for n in (need_w, need_b)]
        return one if need_x else None, one.to(d_dtype) if need_d else None, *zero
    g2, g_stride = _rows(dy, cols)
    s2, s_stride = _rows(dh, cols) if dh is not None else (None, 0)
    h2, h_stride = _rows(src, cols)
    # one gradient for both where stream and branch have one type
    shared = need_d and d_dtype == x_dtype
    dx = torch.empty(shape, dtype=x_dtype, device=src.device) if need_x or shared else None
    dd = torch.empty(shape, dtype=d_dtype, device=src.device) if need_d and not shared else None
    dw = torch.empty(cols, dtype=w_dtype, device=src.device) if need_w else None
    db = torch.empty(cols, dtype=w_dtype, device=src.device) if need_b else None
    with _on_device(src.device):
        _lib.layer_norm_backward(g2, g_stride, s2, s_stride, h2, h_stride, weight, w_dtype, mean, rstd, h2.shape[0],
                                 cols, dx, dd, dw, db)
    return dx if need_x else None, dx if shared else dd, dw, db


class LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype):
        ctx.need = (ctx.needs_input_grad[0], False, ctx.needs_input_grad[1], ctx.needs_input_grad[2])
        y, _, mean, rstd, w = _forward(x, None, weight, bias, eps, out_dtype, any(ctx.need))
        ctx.save_for_backward(x, w, mean, rstd)
        ctx.meta = (x.shape, x.dtype, None, _affine_dtype(weight, bias))
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
        y, h, mean, rstd, w = _forward(x, delta, weight, bias, eps, out_dtype, any(ctx.need))
        ctx.save_for_backward(h, w, mean, rstd)
        ctx.meta = (x.shape, x.dtype, delta.dtype, _affine_dtype(weight, bias))
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
