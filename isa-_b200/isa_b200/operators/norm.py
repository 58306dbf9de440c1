"""Layer norm of the digital part of a block, on the sm_100a kernels."""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
import torch.nn as nn

from isa_b200.kernels.transformer_norm import cuda_add_layer_norm, cuda_layer_norm


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over the last axis: same constructor, parameters and state
    dict, CUDA inputs only.  Forward-mode tangents and traces, which ``nn.LayerNorm``
    takes, raise.

    ``out_dtype`` is the type handed out.  None keeps ``nn.LayerNorm``'s own: the
    input's, or fp32 under CUDA autocast.  A norm that feeds an autocast
    projection can hand out the autocast type directly (what the projection would
    round to), which saves a pass over the tensor.
    """

    def __init__(self, normalized_shape, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True,
                 device=None, dtype=None):
        super().__init__(normalized_shape, eps, elementwise_affine, bias, device, dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError(f"LayerNorm normalises the last axis only, got normalized_shape {self.normalized_shape}")

    def _dtype(self, x: torch.Tensor, out_dtype: Optional[torch.dtype]) -> torch.dtype:
        if out_dtype is not None:
            return out_dtype
        return torch.float32 if torch.is_autocast_enabled("cuda") else x.dtype

    def _check(self, x: torch.Tensor) -> None:
        if x.dim() < 1 or x.shape[-1] != self.normalized_shape[0]:
            raise RuntimeError(f"expected {self.normalized_shape[0]} features in the last axis, got shape {tuple(x.shape)}")

    def forward(self, x: torch.Tensor, out_dtype: Optional[torch.dtype] = None,
                delta: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
        """``norm(x)``, or with a branch ``delta`` what :meth:`add` returns."""
        self._check(x)
        if delta is None:
            return cuda_layer_norm(x, self.weight, self.bias, self.eps, self._dtype(x, out_dtype))
        if delta.dtype != x.dtype and x.dtype != torch.float32:  # as torch's sum: the wider type holds it
            x = x.to(torch.promote_types(x.dtype, delta.dtype))
        return cuda_add_layer_norm(x, delta, self.weight, self.bias, self.eps, self._dtype(x, out_dtype))

    def add(self, x: torch.Tensor, delta: torch.Tensor,
            out_dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """``(norm(x + delta), x + delta)`` in one pass: the residual sum in front of the norm.  A call of the module,
        hooks included."""
        return self(x, out_dtype, delta)
