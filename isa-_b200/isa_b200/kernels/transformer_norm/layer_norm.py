"""Layer normalisation of a transformer block over the sm_100a kernels.

* ``cuda_layer_norm(x, weight, bias, eps)``: ``nn.LayerNorm`` over the last axis
  (the ``ln1`` / ``ln2`` / ``ln_f`` and ``norm`` layers of the reference models,
  ``src/isa/language/models.py:81-177``, ``src/isa/vision/models.py:93-250``).
* ``cuda_add_layer_norm(x, delta, weight, bias, eps)``: the residual sum in front
  of it as well, ``h = x + delta; y = LN(h)``, in one pass; returns ``(y, h)``.

Inputs are fp32, bf16 or fp16 with rows of contiguous elements (any row stride;
other layouts are copied).  Statistics and sums are fp32, results are rounded
once; a row whose sum or sum of squared deviations passes fp32 (means beyond 1e34,
deviations beyond 1e17 at the widest) overflows.  ``out_dtype`` is the type of ``y``: fp32 streams may hand out any of the
three, 16-bit streams their own type or fp32.  The backward is one pass over the
rows and a fixed-order reduction for the weight gradients, so it gives the same
bits every time; it cannot be differentiated again.  There is no forward-mode
derivative, and a trace (``torch.jit.trace``, ``make_fx``) would miss the kernels:
both are refused, with and without gradients recorded.

A backward captured into a CUDA graph follows torch's rule: no eager graph of the
same leaf parameters, made on the default stream, may be alive during the capture
(``del`` the warm-up's outputs and losses first).  Such a capture raises.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from isa_b200 import _lib


def cuda_layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                    eps: float = 1e-5, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Layer norm over the last axis of ``x``; ``y`` in ``out_dtype`` (default: the type of ``x``)."""
    return _lib.binding().layer_norm(x, weight, bias, eps, out_dtype)


def cuda_add_layer_norm(x: torch.Tensor, delta: torch.Tensor, weight: Optional[torch.Tensor] = None,
                        bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
                        out_dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``h = x + delta`` in the type of ``x`` and ``y = LN(h)`` in ``out_dtype``; returns ``(y, h)``.

    The branch ``delta`` of an fp32 stream may be any of the three types (the
    bf16 output of an autocast projection); a 16-bit stream takes its own type.
    """
    return _lib.binding().add_layer_norm(x, delta, weight, bias, eps, out_dtype)
