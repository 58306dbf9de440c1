"""Muon for the digital matrices of a model, on the sm_100a kernels.

The reference trains everything with AdamW (``src/isa/language/train.py:717-764``).
Here the weights that act as matrices (attention and digital FFN projections) may
take Muon's step instead; threshold voltages, embeddings, norms and gains stay
with AdamW (``GPT2Model.configure_muon_groups`` makes the two sets).
"""

from __future__ import annotations

from typing import Sequence

import torch

from isa_b200.kernels.muon import NS_COEFFICIENTS, cuda_muon_step


class Muon(torch.optim.Optimizer):
    """Momentum, Newton-Schulz orthogonalisation and decoupled weight decay
    (``cuda_muon_step``) on parameters of two or more axes.

    A group's ``matrices`` is the number of matrices stacked along a parameter's
    rows: 3 for a fused query / key / value projection, whose three parts are
    orthogonalised separately.  ``lr`` may be a one-element fp32 CUDA tensor, which
    a captured step reads at each replay; the first step, which makes the momenta,
    cannot be captured.  Momenta are fp32.
    """

    def __init__(self, params, lr=1e-3, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.1,
                 steps: int = 5, coefficients: Sequence[float] = NS_COEFFICIENTS, eps: float = 1e-7,
                 adjust_lr: str = "original", matrices: int = 1):
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError(f"invalid learning rate {lr}")
        if not 0.0 <= momentum <= 1.0:
            raise ValueError(f"invalid momentum {momentum}")
        if not weight_decay >= 0.0:
            raise ValueError(f"invalid weight_decay {weight_decay}")
        if adjust_lr not in ("original", "match_rms_adamw"):
            raise ValueError(f"unknown adjust_lr {adjust_lr!r}")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=tuple(coefficients), eps=eps, adjust_lr=adjust_lr, matrices=matrices))

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        for p in group["params"]:
            if p.dim() < 2 or group["matrices"] < 1 or p.shape[-2] % group["matrices"]:
                del self.param_groups[-1]
                raise ValueError(f"a parameter of shape {tuple(p.shape)} is not {group['matrices']} stacked matrices")

    def load_state_dict(self, state_dict) -> None:
        super().load_state_dict(state_dict)
        # the base class casts state to the parameter's type; momenta stay fp32
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        for i, p in zip(ids, params):
            saved = state_dict["state"].get(i, {}).get("momentum_buffer")
            if saved is not None:
                self.state[p]["momentum_buffer"] = saved.detach().to(p.device, torch.float32, copy=True).contiguous()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # groups of one device that differ in `matrices` alone make one call, so that their shapes run side by side
        calls = {}
        for group in self.param_groups:
            options = {k: group[k] for k in ("lr", "momentum", "nesterov", "weight_decay", "steps", "coefficients", "eps",
                                             "adjust_lr")}
            k = group["matrices"]
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("Muon does not take sparse gradients")
                state = self.state[p]
                if "momentum_buffer" not in state:
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():  # every replay would begin with zeros
                        raise RuntimeError("Muon's first step cannot be captured: take one step before the capture")
                    state["momentum_buffer"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format)
                shape = (*p.shape[:-2], k, p.shape[-2] // k, p.shape[-1]) if k > 1 else p.shape
                key = (p.device, *(id(v) if isinstance(v, torch.Tensor) else repr(v) for v in options.values()))
                params, grads, momenta, _ = calls.setdefault(key, ([], [], [], options))
                params.append(p.view(shape))
                grads.append(p.grad.reshape(shape))
                momenta.append(state["momentum_buffer"].view(shape))
        for params, grads, momenta, options in calls.values():
            cuda_muon_step(params, grads, momenta, **options)
        return loss
