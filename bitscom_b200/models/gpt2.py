"""GPT-2 (decoder-only transformer) for the sharded data-parallel benchmark.

Architecture of GPT-2: learned token + position embeddings, pre-LayerNorm
blocks (causal multi-head attention, 4x GELU MLP), final LayerNorm, LM head
tied to the token embedding.  Attention uses
``F.scaled_dot_product_attention`` (flash kernels under bf16).  The reference
used Hugging Face's GPT2LMHeadModel with a 4-layer/256-wide config (reference
benchmarks/multimodel_stochastic_e2e_curve.py:62-74); :func:`gpt2_medium` is
the 24-layer / 1024-wide / 16-head model of the sharded benchmark config.

Options beyond GPT-2, off by default (:class:`GPT2Config`): queries and keys
normalised for each head and rotated by position in place of the learned
position table, capped attention scores, a distance bias; and, as arguments of
``forward``, rows of packed documents and prefixes.  With any of them attention
runs through :func:`bitscom_b200.ops.attention`.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops.attention import attention, attention_mask
from ..ops.rotary import qk_norm_rotary, rotary_frequencies


@dataclass
class GPT2Config:
    vocab_size: int = 50257
    n_positions: int = 1024
    n_embd: int = 1024
    n_layer: int = 24
    n_head: int = 16
    dropout: float = 0.0
    rotary: bool = False  # norm of queries and keys per head + rotation, no position table
    softcap: float | None = None  # cap of the attention scores
    distance_bias: bool = False  # slope 2^(-8 h / n_head) times the distance off head h's scores


class _Attention(nn.Module):
    def __init__(self, cfg: GPT2Config):
        super().__init__()
        self.n_head = cfg.n_head
        self.qkv = nn.Linear(cfg.n_embd, 3 * cfg.n_embd)
        self.proj = nn.Linear(cfg.n_embd, cfg.n_embd)
        self.softcap = cfg.softcap
        self.rotary, self.distance_bias = cfg.rotary, cfg.distance_bias
        if cfg.rotary:
            self.q_gain = nn.Parameter(torch.ones(cfg.n_embd // cfg.n_head))
            self.k_gain = nn.Parameter(torch.ones(cfg.n_embd // cfg.n_head))
        # Constants, kept out of the buffers: a cast of the module must not round the float64 frequencies.
        self._constants = {}

    def _constant(self, name: str, device: torch.device) -> torch.Tensor:
        if (name, device) not in self._constants:
            # Kept for later calls, training among them, which an inference tensor could not serve.
            with torch.inference_mode(False):
                if name == "frequencies":
                    d = self.qkv.in_features // self.n_head
                    value = rotary_frequencies(d - d % 2)
                else:
                    value = 2.0 ** (-8.0 * torch.arange(1, self.n_head + 1, dtype=torch.float32) / self.n_head)
                self._constants[name, device] = value.to(device)
        return self._constants[name, device]

    def forward(self, x, mask=None):
        b, t, c = x.shape
        q, k, v = (z.view(b, t, self.n_head, c // self.n_head) for z in self.qkv(x).split(c, dim=2))
        if self.rotary:
            q, k = qk_norm_rotary(q, k, self._constant("frequencies", x.device), q_weight=self.q_gain,
                                  k_weight=self.k_gain)
        q, k, v = (z.transpose(1, 2) for z in (q, k, v))
        if mask is None and self.softcap is None and not self.distance_bias:
            y = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        else:
            slopes = self._constant("slopes", x.device) if self.distance_bias else None
            y = attention(q, k, v, mask=mask, softcap=self.softcap, slopes=slopes)
        return self.proj(y.transpose(1, 2).reshape(b, t, c))


class _Block(nn.Module):
    def __init__(self, cfg: GPT2Config):
        super().__init__()
        self.ln1 = nn.LayerNorm(cfg.n_embd)
        self.attn = _Attention(cfg)
        self.ln2 = nn.LayerNorm(cfg.n_embd)
        self.fc = nn.Linear(cfg.n_embd, 4 * cfg.n_embd)
        self.out = nn.Linear(4 * cfg.n_embd, cfg.n_embd)

    def forward(self, x, mask=None):
        x = x + self.attn(self.ln1(x), mask)
        return x + self.out(F.gelu(self.fc(self.ln2(x)), approximate="tanh"))


class GPT2(nn.Module):
    def __init__(self, cfg: GPT2Config):
        super().__init__()
        self.cfg = cfg
        self.wte = nn.Embedding(cfg.vocab_size, cfg.n_embd)
        self.wpe = None if cfg.rotary else nn.Embedding(cfg.n_positions, cfg.n_embd)
        self.blocks = nn.ModuleList([_Block(cfg) for _ in range(cfg.n_layer)])
        self.ln_f = nn.LayerNorm(cfg.n_embd)
        self.apply(self._init)
        for name, p in self.named_parameters():
            if name.endswith("proj.weight") or name.endswith("out.weight"):
                nn.init.normal_(p, 0.0, 0.02 / math.sqrt(2 * cfg.n_layer))

    @staticmethod
    def _init(m):
        if isinstance(m, nn.Linear):
            nn.init.normal_(m.weight, 0.0, 0.02)
            if m.bias is not None:
                nn.init.zeros_(m.bias)
        elif isinstance(m, nn.Embedding):
            nn.init.normal_(m.weight, 0.0, 0.02)

    def forward(
        self,
        idx: torch.Tensor,
        targets: torch.Tensor | None = None,
        documents: torch.Tensor | None = None,
        prefix: torch.Tensor | None = None,
    ):
        """Logits, or ``(logits, mean loss)`` with targets (-100: not counted).

        ``documents`` [batch, length]: ids of documents packed into the rows
        (tokens see their own one, positions restart with each; negative:
        padding).  ``prefix`` [batch]: leading tokens that all see each other.
        """
        t = idx.shape[1]
        mask = None if documents is None and prefix is None else attention_mask(documents, prefix, q_len=t, k_len=t)
        x = self.wte(idx)
        if self.wpe is not None:
            pos = torch.arange(t, device=idx.device)
            if documents is not None:
                starts = torch.ones_like(documents, dtype=torch.bool)
                starts[:, 1:] = documents[:, 1:] != documents[:, :-1]
                pos = pos - torch.where(starts, pos, 0).cummax(dim=1).values
            x = x + self.wpe(pos)
        for blk in self.blocks:
            x = blk(x, mask)
        logits = F.linear(self.ln_f(x), self.wte.weight)
        if targets is None:
            return logits
        loss = F.cross_entropy(logits.float().reshape(-1, logits.size(-1)), targets.reshape(-1))
        return logits, loss


def gpt2_medium(**overrides) -> GPT2:
    return GPT2(GPT2Config(**overrides))


def gpt2_small_test(**overrides) -> GPT2:
    """4-layer, 256-wide GPT-2 (the reference's benchmark size)."""
    cfg = dict(n_embd=256, n_layer=4, n_head=4, n_positions=512)
    cfg.update(overrides)
    return GPT2(GPT2Config(**cfg))
