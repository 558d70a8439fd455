"""GPT-2 shaped decoder used as the data-parallel workload.

The reference has no model code; this is the synthetic workload the DDP
configuration names: 24 layers, d_model 1024, 16 heads, vocabulary 50257,
sequence 1024, bf16 weights, random initialisation.  The output projection and
the loss run on this library's kernels (ops/lm_loss.py), the rest of the compute
on PyTorch's; the gradient AllReduce goes through mini_nccl_b200.parallel.ddp.

``GPT2Config(linear="fp8")`` runs the linear layers of the blocks in 8 bits (ops/fp8.py; parameters keep their
type and names), and ``forward(ids, teacher=(top_ids, top_logits, temperature))`` trains against a teacher's top
logits instead of targets (ops/distill.py): a decoder that is brought to 8 bits and recovered from the original.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops.distill import lm_head_distillation
from ..ops.fp8 import linear_fp8
from ..ops.lm_loss import lm_head_cross_entropy


@dataclass
class GPT2Config:
    n_layer: int = 24
    d_model: int = 1024
    n_head: int = 16
    vocab_size: int = 50257
    seq_len: int = 1024
    dtype: torch.dtype = torch.bfloat16
    linear: str = "plain"   # of the blocks: "plain" or "fp8"

    @staticmethod
    def medium() -> "GPT2Config":
        return GPT2Config()

    @staticmethod
    def tiny() -> "GPT2Config":
        return GPT2Config(n_layer=2, d_model=128, n_head=4, vocab_size=512, seq_len=64)


class Fp8Linear(nn.Linear):
    """``nn.Linear`` whose products, forward and backward, run in 8 bits."""

    def forward(self, x):
        return linear_fp8(x, self.weight, self.bias)


_LINEAR = {"plain": nn.Linear, "fp8": Fp8Linear}


class Block(nn.Module):
    def __init__(self, cfg: GPT2Config):
        super().__init__()
        d = cfg.d_model
        if cfg.linear not in _LINEAR:
            raise ValueError(f"linear must be one of {tuple(_LINEAR)}, not {cfg.linear!r}")
        linear = _LINEAR[cfg.linear]
        self.n_head = cfg.n_head
        self.ln1 = nn.LayerNorm(d)
        self.qkv = linear(d, 3 * d)
        self.proj = linear(d, d)
        self.ln2 = nn.LayerNorm(d)
        self.fc = linear(d, 4 * d)
        self.out = linear(4 * d, d)

    def forward(self, x):
        b, s, d = x.shape
        q, k, v = self.qkv(self.ln1(x)).view(b, s, 3, self.n_head, d // self.n_head).permute(2, 0, 3, 1, 4)
        a = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        x = x + self.proj(a.transpose(1, 2).reshape(b, s, d))
        return x + self.out(F.gelu(self.fc(self.ln2(x)), approximate="tanh"))


class GPT2Model(nn.Module):
    def __init__(self, cfg: GPT2Config):
        super().__init__()
        self.cfg = cfg
        self.wte = nn.Embedding(cfg.vocab_size, cfg.d_model)
        self.wpe = nn.Embedding(cfg.seq_len, cfg.d_model)
        self.blocks = nn.ModuleList([Block(cfg) for _ in range(cfg.n_layer)])
        self.ln_f = nn.LayerNorm(cfg.d_model)
        self.apply(self._init)

    @staticmethod
    def _init(m):
        if isinstance(m, (nn.Linear, nn.Embedding)):
            nn.init.normal_(m.weight, std=0.02)
        if isinstance(m, nn.Linear) and m.bias is not None:
            nn.init.zeros_(m.bias)

    def forward(self, ids, targets=None, teacher=None):
        """Logits; with ``targets`` their mean cross-entropy; with ``teacher = (top_ids [b, s, K], top_logits [b, s, K][, temperature])``
        the distillation loss."""
        if targets is not None and teacher is not None:
            raise ValueError("targets or a teacher, not both")
        b, s = ids.shape
        pos = torch.arange(s, device=ids.device)
        x = self.wte(ids) + self.wpe(pos)
        for blk in self.blocks:
            x = blk(x)
        x = self.ln_f(x)
        if teacher is not None:
            return lm_head_distillation(x, self.wte.weight, *teacher)
        if targets is None:
            return F.linear(x, self.wte.weight)  # tied output embedding
        return lm_head_cross_entropy(x, self.wte.weight, targets)

    def num_params(self) -> int:
        return sum(p.numel() for p in self.parameters())
