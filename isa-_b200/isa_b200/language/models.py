"""GPT-2 models whose FFN is the CIM operator: the callers of the hot path on the
language side.

Drop-in for ``src/isa/language/models.py`` and ``language/config.py`` of the
reference at the level of module names, constructor arguments and state-dict
keys, so a reference checkpoint loads unchanged:

* ``HybridFFN`` (``models.py:48-63``): VoltageMapping -> ``cim1`` (CIMLinear,
  up projection) -> ``fc2`` (digital nn.Linear) -> per-channel ADC affine ->
  dropout.  This is the GPT-side hybrid block; the operator-level
  ``isa_b200.operators.cim.HybridFFN`` (fc1/fc2, no affine) is a different
  module, as in the reference.
* ``GPT2PhysicalFFN`` (``models.py:66-74``): ``cim_ffn`` = the operator-level
  PhysicalFFN (VoltageMapping -> CIMLinear -> CIMLinear -> ADC affine), then
  dropout.
* ``GPT2Block`` / ``GPT2Model`` (``models.py:81-177``): pre-LayerNorm blocks,
  causal scaled-dot-product attention over the weights of an
  ``nn.MultiheadAttention`` (used as the parameter container, keys
  ``attn.in_proj_weight`` / ``attn.out_proj.*``), token + position embeddings,
  tied LM head.

The CIM layers run on this package's sm_100a kernels; everything else is
plain PyTorch, or with ``ModelConfig.fused_norm`` has its layer norms, joined with
the residual sums in front of them, on them as well.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from isa_b200.device_models.config import make_flash_transistor_ekv_config
from isa_b200.operators.cim import CIMLinear, PhysicalFFN, VoltageMapping
from isa_b200.operators.norm import LayerNorm

# The language experiments pin the table size to 4096 (reference config.py:13;
# EKV_LUT_SIZE in the environment still overrides it).
PHYSICAL_CONFIG = make_flash_transistor_ekv_config(default_lut_size=4096)

# Model size presets (reference config.py:16-38): embed dim, FFN dim, heads, depth.
SIZE_PRESETS: Dict[str, Dict] = {
    "tiny": dict(embed_dim=192, ffn_dim=768, num_heads=3, depth=12, dropout=0.0),
    "mid": dict(embed_dim=384, ffn_dim=1536, num_heads=6, depth=12, dropout=0.0),
    "small": dict(embed_dim=768, ffn_dim=3072, num_heads=12, depth=12, dropout=0.0),
}


@dataclass
class ModelConfig:
    """Architecture of a GPT-2 model (field names of the reference ModelConfig)."""

    size: str = "tiny"
    model_type: str = "standard"  # "standard" | "hybrid" | "physical"
    vocab_size: int = 50257
    max_seq_len: int = 128
    embed_dim: int = 192
    ffn_dim: int = 768
    num_heads: int = 3
    depth: int = 12
    dropout: float = 0.0
    voltage_max: float = 4.0
    affine_scope: str = "final"
    output_chunk_size: int = 16
    # layer norms and residual sums on this package's kernels (no counterpart there).  A block then hands on its stream and
    # its FFN output as a pair, whose sum the next norm takes, and a norm with a branch (result, sum): hooks see these.
    fused_norm: bool = False

    @classmethod
    def from_preset(cls, size: str, model_type: str, **kwargs) -> "ModelConfig":
        return cls(size=size, model_type=model_type, **SIZE_PRESETS[size], **kwargs)


class StandardFFN(nn.Module):
    """Digital FFN (Linear -> GELU -> Linear), the baseline the CIM variants replace."""

    def __init__(self, embed_dim: int, ffn_dim: int, dropout: float = 0.0):
        super().__init__()
        self.fc1 = nn.Linear(embed_dim, ffn_dim)
        self.fc2 = nn.Linear(ffn_dim, embed_dim)
        self.dropout = nn.Dropout(dropout)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.fc2(self.dropout(F.gelu(self.fc1(x))))


class HybridFFN(nn.Module):
    """CIM up projection, digital down projection, ADC affine."""

    def __init__(self, embed_dim: int, ffn_dim: int, voltage_max: float = 4.0, dropout: float = 0.0):
        super().__init__()
        self.input_mapping = VoltageMapping(voltage_max=voltage_max)
        self.cim1 = CIMLinear(embed_dim, ffn_dim)
        self.fc2 = nn.Linear(ffn_dim, embed_dim)
        self.adc_affine_scale = nn.Parameter(torch.ones(embed_dim))
        self.adc_affine_shift = nn.Parameter(torch.zeros(embed_dim))
        self.dropout = nn.Dropout(dropout)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        h = self.fc2(self.cim1(self.input_mapping(x)))
        return self.dropout(h * self.adc_affine_scale + self.adc_affine_shift)


class GPT2PhysicalFFN(nn.Module):
    """Both projections on the CIM operator (the operator-level PhysicalFFN)."""

    def __init__(self, embed_dim: int, ffn_dim: int, voltage_max: float = 4.0, dropout: float = 0.0,
                 physical_config: Optional[Dict] = None):
        super().__init__()
        self.cim_ffn = PhysicalFFN(embed_dim, ffn_dim, physical_config or PHYSICAL_CONFIG, voltage_max)
        self.dropout = nn.Dropout(dropout)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.dropout(self.cim_ffn(x))


class GPT2Block(nn.Module):
    """Pre-LayerNorm transformer block: causal attention, then the FFN variant."""

    def __init__(self, embed_dim: int, ffn_dim: int, num_heads: int, model_type: str, voltage_max: float = 4.0,
                 dropout: float = 0.0, physical_config: Optional[Dict] = None, fused_norm: bool = False):
        super().__init__()
        if embed_dim % num_heads:
            raise ValueError(f"embed_dim={embed_dim} must be divisible by num_heads={num_heads}")
        self.num_heads = num_heads
        self.head_dim = embed_dim // num_heads
        norm = LayerNorm if fused_norm else nn.LayerNorm
        self.ln1 = norm(embed_dim)
        # parameter container only (in_proj_weight/bias, out_proj); the forward
        # calls scaled_dot_product_attention on these weights directly
        self.attn = nn.MultiheadAttention(embed_dim, num_heads, dropout=dropout, batch_first=True)
        self.ln2 = norm(embed_dim)
        self.digital_ffn = model_type == "standard"
        if model_type == "standard":
            self.ffn = StandardFFN(embed_dim, ffn_dim, dropout)
        elif model_type == "hybrid":
            self.ffn = HybridFFN(embed_dim, ffn_dim, voltage_max, dropout)
        elif model_type == "physical":
            self.ffn = GPT2PhysicalFFN(embed_dim, ffn_dim, voltage_max, dropout, physical_config)
        else:
            raise ValueError(f"Unknown model_type: {model_type}")

    def attention(self, x: torch.Tensor) -> torch.Tensor:
        return self._attend(self.ln1(x))

    def _attend(self, normed: torch.Tensor) -> torch.Tensor:
        b, t, d = normed.shape
        qkv = F.linear(normed, self.attn.in_proj_weight, self.attn.in_proj_bias)
        q, k, v = (h.transpose(1, 2) for h in qkv.view(b, t, 3, self.num_heads, self.head_dim).unbind(2))
        p = float(self.attn.dropout) if self.training else 0.0
        y = F.scaled_dot_product_attention(q, k, v, dropout_p=p, is_causal=True)
        return F.linear(y.transpose(1, 2).reshape(b, t, d), self.attn.out_proj.weight, self.attn.out_proj.bias)

    def forward(self, x: torch.Tensor, need_intermediate: bool = False, delta: Optional[torch.Tensor] = None,
                carry: bool = False):
        """``carry`` (blocks with ``fused_norm``): the pair of :meth:`forward_fused` instead of the stream."""
        if carry:
            return self.forward_fused(x, delta)
        x = x + self.attention(x)
        ffn_out = self.ffn(self.ln2(x))
        out = x + ffn_out
        if need_intermediate:
            return out, {"ffn_output": ffn_out, "block_output": out}
        return out


    def forward_fused(self, x: torch.Tensor, delta: Optional[torch.Tensor]):
        """The block on ``x + delta`` (delta: the FFN output of the block before),
        with both residual sums inside the norms that follow them.  Returns the
        stream before this block's own FFN output, and that output."""
        digital = _projection_dtype(x)  # what a norm that feeds a projection hands out
        if delta is None:
            normed = self.ln1(x, digital)
        else:
            normed, x = self.ln1.add(x, delta, digital)
        normed, x = self.ln2.add(x, self._attend(normed), digital if self.digital_ffn else None)
        return x, self.ffn(normed)


def _projection_dtype(x: torch.Tensor) -> Optional[torch.dtype]:
    """The autocast type, where one is on and the stream can hand it out."""
    if not torch.is_autocast_enabled("cuda"):
        return None
    dtype = torch.get_autocast_dtype("cuda")
    return dtype if x.dtype in (torch.float32, dtype) else None


class GPT2Model(nn.Module):
    """GPT-2 with the FFN variant of ``cfg.model_type`` in every block."""

    def __init__(self, cfg: ModelConfig, physical_config: Optional[Dict] = None):
        super().__init__()
        self.cfg = cfg
        self.token_embedding = nn.Embedding(cfg.vocab_size, cfg.embed_dim)
        self.pos_embedding = nn.Embedding(cfg.max_seq_len, cfg.embed_dim)
        self.drop = nn.Dropout(cfg.dropout)
        self.blocks = nn.ModuleList(
            GPT2Block(cfg.embed_dim, cfg.ffn_dim, cfg.num_heads, cfg.model_type, cfg.voltage_max, cfg.dropout,
                      physical_config, cfg.fused_norm)
            for _ in range(cfg.depth))
        self.ln_f = (LayerNorm if cfg.fused_norm else nn.LayerNorm)(cfg.embed_dim)
        self.lm_head = nn.Linear(cfg.embed_dim, cfg.vocab_size, bias=False)
        self.lm_head.weight = self.token_embedding.weight
        self.register_buffer("pos_ids", torch.arange(cfg.max_seq_len).unsqueeze(0), persistent=False)

    def forward(self, input_ids: torch.Tensor, need_intermediate: bool = False):
        b, t = input_ids.shape
        x = self.drop(self.token_embedding(input_ids) + self.pos_embedding(self.pos_ids[:, :t].expand(b, -1)))
        if self.cfg.fused_norm and not need_intermediate:
            delta = None
            for blk in self.blocks:
                x, delta = blk(x, False, delta, True)
            dtype = _projection_dtype(x)
            normed = self.ln_f(x, dtype) if delta is None else self.ln_f.add(x, delta, dtype)[0]
            return self.lm_head(normed)
        inter: List[Dict[str, torch.Tensor]] = []
        for blk in self.blocks:
            if need_intermediate:
                x, info = blk(x, need_intermediate=True)
                inter.append(info)
            else:
                x = blk(x)
        logits = self.lm_head(self.ln_f(x))
        return (logits, inter) if need_intermediate else logits

    def cim_layers(self) -> List[CIMLinear]:
        return [m for m in self.modules() if isinstance(m, CIMLinear)]

    def configure_optimizer_groups(self, weight_decay: float, lr: float, ffn_only: bool = False):
        """AdamW groups: thresholds, TIA gains, embeddings / LM head and 1-D
        parameters take no weight decay (reference models.py:179-201)."""
        decay, no_decay = [], []
        for name, p in self.named_parameters():
            if not p.requires_grad or (ffn_only and ".ffn." not in name):
                continue
            exempt = name.startswith(("lm_head", "token_embedding")) or "vth_" in name or "r_tia" in name
            (no_decay if exempt or p.dim() < 2 else decay).append(p)
        return [{"params": decay, "weight_decay": weight_decay, "lr": lr},
                {"params": no_decay, "weight_decay": 0.0, "lr": lr}]


    def configure_muon_groups(self, weight_decay: float, lr: float, muon_weight_decay: float, muon_lr: float):
        """(groups for ``isa_b200.optim.Muon``, AdamW groups for the rest).  Muon
        takes the digital matrices of the blocks: attention projections, the fused
        query / key / value one as three, and the linear layers of a standard or
        hybrid FFN.  Threshold voltages are device parameters in a narrow window and
        stay with AdamW, as do embeddings, norms, gains and biases."""
        fused, single = [], []
        for blk in self.blocks:
            fused.append(blk.attn.in_proj_weight)
            single.append(blk.attn.out_proj.weight)
            single += [m.weight for m in blk.ffn.modules() if isinstance(m, nn.Linear)]
        both = dict(weight_decay=muon_weight_decay, lr=muon_lr)
        muon = [{"params": [p for p in ps if p.requires_grad], "matrices": k, **both} for ps, k in ((fused, 3), (single, 1))]
        taken = {id(p) for g in muon for p in g["params"]}
        rest = self.configure_optimizer_groups(weight_decay, lr)
        for g in rest:
            g["params"] = [p for p in g["params"] if id(p) not in taken]
        return [g for g in muon if g["params"]], [g for g in rest if g["params"]]


def create_model(cfg: ModelConfig, physical_config: Optional[Dict] = None) -> GPT2Model:
    return GPT2Model(cfg, physical_config)
