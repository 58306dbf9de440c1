"""Newton-Schulz orthogonalisation and the Muon step over the sm_100a kernels.

* ``cuda_orthogonalize(g)``: the matrices ``g[..., rows, cols]`` with their
  singular values moved close to 1 by ``steps`` Newton-Schulz products.
* ``cuda_muon_step(params, grads, momenta, lr=...)``: momentum, Nesterov,
  orthogonalisation, weight decay and update of a list of parameters, in place
  (K. Jordan et al., "Muon: an optimizer for hidden layers in neural networks",
  2024).

The reference trains with AdamW (``src/isa/language/train.py:717-764``); these
serve the digital matrices around the CIM layers (attention and output
projections), whose gradients are matrices in the sense of that method.
Threshold voltages are device parameters and stay with AdamW.

Matrices are fp32, bf16 or fp16; momenta are fp32.  Products run on the tensor
cores with operands of 22 bits and fp32 sums, so results are about as close
to the exact iteration as with fp32 products (fp32 results 0.35 to 1.2 times their error).  Results are the same bits every time.
"""

from __future__ import annotations

from typing import List, Sequence, Union

import torch

from isa_b200 import _lib

# Coefficients of the quintic step s -> s (a + b s^2 + c s^4) in the paper above.
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def cuda_orthogonalize(g: torch.Tensor, steps: int = 5, coefficients: Sequence[float] = NS_COEFFICIENTS,
                       eps: float = 1e-7) -> torch.Tensor:
    """Newton-Schulz steps on each matrix of ``g[..., rows, cols]``, after
    division by ``max(|g|_F, eps)`` (``eps`` at least 1e-30); a new tensor in the type of ``g``.  There is
    no gradient: the result is part of an optimiser's step."""
    return _lib.binding().orthogonalize(g, steps, coefficients, eps)


def cuda_muon_step(params: List[torch.Tensor], grads: List[torch.Tensor], momenta: List[torch.Tensor], *,
                   lr: Union[float, torch.Tensor], momentum: float = 0.95, nesterov: bool = True,
                   weight_decay: float = 0.1, steps: int = 5, coefficients: Sequence[float] = NS_COEFFICIENTS,
                   eps: float = 1e-7, adjust_lr: str = "original") -> None:
    """One Muon step on every ``params[i][..., rows, cols]`` (leading axes count
    matrices: a fused query / key / value projection is passed as ``view(3, d, d)``),
    updating ``params`` and ``momenta`` in place:

        m <- momentum m + (1 - momentum) g;  u = momentum m + (1 - momentum) g (nesterov) or m
        p <- p (1 - lr weight_decay) - lr s NS(u)

    with ``s = sqrt(max(1, rows / cols))`` for ``adjust_lr="original"`` (the spectral
    size of tall matrices is kept) or ``0.2 sqrt(max(rows, cols))`` for
    ``"match_rms_adamw"`` (all shapes move by AdamW's typical RMS).

    ``lr`` may be a one-element fp32 CUDA tensor, which a captured graph reads at
    each replay.  Matrices of one shape and type run together, small ones of several
    shapes side by side; parameters and momenta must not overlap.
    """
    if adjust_lr not in ("original", "match_rms_adamw"):
        raise ValueError(f"unknown adjust_lr {adjust_lr!r}")
    lr_tensor = lr if isinstance(lr, torch.Tensor) else None
    _lib.binding().muon_step(params, grads, momenta, 0.0 if lr_tensor is not None else lr, lr_tensor, momentum, nesterov,
                             weight_decay, steps, coefficients, eps, adjust_lr == "match_rms_adamw")
