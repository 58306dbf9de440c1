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
cores with operands of 22 bits and fp32 sums, so results are as close to the
exact iteration as fp32 products are.  Results are the same bits every time.
"""

from __future__ import annotations

import math
from typing import Dict, List, Sequence, Tuple, Union

import torch

from isa_b200 import _lib

# Coefficients of the quintic step s -> s (a + b s^2 + c s^4) in the paper above.
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check_matrix(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor: the Newton-Schulz kernels have no CPU implementation")
    if t.dtype not in _TYPES:
        raise RuntimeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if t.dim() < 2:
        raise RuntimeError(f"{name} must have at least two axes, got shape {tuple(t.shape)}")


def _coefficients(coefficients) -> Tuple[float, float, float]:
    a, b, c = (float(v) for v in coefficients)
    return a, b, c


@torch.no_grad()
def cuda_orthogonalize(g: torch.Tensor, steps: int = 5, coefficients: Sequence[float] = NS_COEFFICIENTS,
                       eps: float = 1e-7) -> torch.Tensor:
    """Newton-Schulz steps on each matrix of ``g[..., rows, cols]``, after
    division by ``max(|g|_F, eps)``; a new tensor in the type of ``g``.  There is
    no gradient: the result is part of an optimiser's step."""
    _check_matrix(g, "g")
    coefficients = _coefficients(coefficients)
    rows, cols = g.shape[-2:]
    if g.numel() == 0:
        return torch.empty_like(g)
    g3 = g if g.dim() == 3 else g.reshape(-1, rows, cols)
    if (cols > 1 and g3.stride(2) != 1) or g3.stride(1) < 0:
        g3 = g3.contiguous()
    out = g.new_empty(g.shape)
    batch = g3.shape[0]
    with _lib.on_device(g.device):
        ws = g.new_empty(max(_lib.orthogonalize_workspace_bytes(batch, rows, cols), 1), dtype=torch.uint8)
        _lib.orthogonalize(g3, g3.stride(0), g3.stride(1), batch, rows, cols, int(steps), coefficients, float(eps), out,
                           ws)
    return out


def update_scale(rows: int, cols: int, adjust_lr: str) -> float:
    """Factor on the orthogonalised update: "original" keeps the spectral size
    of tall matrices, "match_rms_adamw" gives all shapes AdamW's typical RMS."""
    if adjust_lr == "original":
        return math.sqrt(max(1.0, rows / cols))
    if adjust_lr == "match_rms_adamw":
        return 0.2 * math.sqrt(max(rows, cols))
    raise ValueError(f"unknown adjust_lr {adjust_lr!r}")


@torch.no_grad()
def cuda_muon_step(params: List[torch.Tensor], grads: List[torch.Tensor], momenta: List[torch.Tensor], *,
                   lr: Union[float, torch.Tensor], momentum: float = 0.95, nesterov: bool = True,
                   weight_decay: float = 0.1, steps: int = 5, coefficients: Sequence[float] = NS_COEFFICIENTS,
                   eps: float = 1e-7, adjust_lr: str = "original") -> None:
    """One Muon step on every ``params[i][..., rows, cols]`` (leading axes count
    matrices: a fused query / key / value projection is passed as ``view(3, d, d)``),
    updating ``params`` and ``momenta`` in place:

        m <- momentum m + (1 - momentum) g;  u = momentum m + (1 - momentum) g (nesterov) or m
        p <- p (1 - lr weight_decay) - lr s NS(u),  s = ``update_scale(rows, cols, adjust_lr)``

    ``lr`` may be a one-element fp32 CUDA tensor, which a captured graph reads at
    each replay.  Matrices of one shape and type run together.
    """
    if not len(params) == len(grads) == len(momenta):
        raise RuntimeError(f"expected as many gradients and momenta as parameters, got {len(params)}, {len(grads)}, "
                           f"{len(momenta)}")
    coefficients = _coefficients(coefficients)
    groups: Dict[tuple, Tuple[list, list, list]] = {}
    keep = []  # contiguous copies of gradients, alive until the launches
    for p, g, m in zip(params, grads, momenta):
        _check_matrix(p, "parameter")
        if g.shape != p.shape or m.shape != p.shape:
            raise RuntimeError(f"shape mismatch: parameter {tuple(p.shape)}, gradient {tuple(g.shape)}, momentum "
                               f"{tuple(m.shape)}")
        if g.device != p.device or m.device != p.device or p.device != params[0].device:
            raise RuntimeError("parameters, gradients and momenta must be on one device")
        if g.dtype not in _TYPES:
            raise RuntimeError(f"gradient must be float32, bfloat16 or float16, got {g.dtype}")
        if m.dtype != torch.float32:
            raise RuntimeError(f"momentum must be float32, got {m.dtype}")
        if not (p.is_contiguous() and m.is_contiguous()):
            raise RuntimeError("parameters and momenta are updated in place and must be contiguous")
        if p.numel() == 0:
            continue
        if not g.is_contiguous():
            g = g.contiguous()
            keep.append(g)
        rows, cols = p.shape[-2:]
        each = rows * cols
        ps, gs, ms = groups.setdefault((rows, cols, p.dtype, g.dtype), ([], [], []))
        pa, ga, ma = p.data_ptr(), g.data_ptr(), m.data_ptr()
        pe, ge = each * p.element_size(), each * g.element_size()
        for i in range(p.numel() // each):
            ps.append(pa + i * pe)
            gs.append(ga + i * ge)
            ms.append(ma + i * each * 4)
    lr_tensor = None
    if isinstance(lr, torch.Tensor):
        if lr.numel() != 1 or lr.dtype != torch.float32 or not params or lr.device != params[0].device:
            raise RuntimeError("lr must be a float or a one-element float32 tensor on the parameters' device")
        lr_tensor, lr = lr, 0.0
    if not groups:
        return
    most = _lib.MUON_MAX_MATRICES
    with _lib.on_device(params[0].device):
        size = max(_lib.orthogonalize_workspace_bytes(min(len(v[0]), most), *k[:2]) for k, v in groups.items())
        ws = params[0].new_empty(max(size, 1), dtype=torch.uint8)
        for (rows, cols, p_dtype, g_dtype), (ps, gs, ms) in groups.items():
            scale = update_scale(rows, cols, adjust_lr)
            for i in range(0, len(ps), most):
                _lib.muon_step(ps[i:i + most], gs[i:i + most], ms[i:i + most], p_dtype, g_dtype, rows, cols, float(lr),
                               lr_tensor, float(momentum), nesterov, float(weight_decay), scale, int(steps),
                               coefficients, float(eps), ws)
    torch.autograd.graph.increment_version(params)
    torch.autograd.graph.increment_version(momenta)
