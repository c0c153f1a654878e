"""Workload models for the benchmark configurations (random init, synthetic data).

These are the callers of the hot path, not part of it: an MLP, a GPT-2 with
nn.Linear projections, tied lm_head and per-sample position ids (configs[2] GPT-2-small,
configs[3] GPT-2-medium shape), and a rotary GPT-NeoX-style model (configs[4] Pythia-1B
shape).  Embeddings listed in ``ghost_embeddings`` receive the dummy bias of the engine's
forward swapper, which keeps the autograd graph alive when every weight is frozen.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch
import torch.nn.functional as F
from torch import nn

from .lm_layers import (HeadCrossEntropy, QKNormRotary, RMSNorm, ScaledEmbedding,
                        distillation_loss)


class MLP(nn.Module):
    """Linear 512 -> 1024 -> ReLU -> 1024 -> ReLU -> 10."""

    def __init__(self, dims=(512, 1024, 1024, 10)):
        super().__init__()
        layers = []
        for i in range(len(dims) - 1):
            layers.append(nn.Linear(dims[i], dims[i + 1]))
            if i < len(dims) - 2:
                layers.append(nn.ReLU())
        self.net = nn.Sequential(*layers)

    def forward(self, x):
        return self.net(x)


@dataclass
class LMConfig:
    n_layer: int = 12
    n_head: int = 12
    d_model: int = 768
    d_mlp: int = 3072
    vocab: int = 50257
    n_ctx: int = 1024
    rotary: bool = False
    tied: bool = True
    rotary_pct: float = 0.25
    # Queries and keys normed per head, with the rotation in the same pass (QKNormRotary).
    qk_norm: bool = False
    # Token embeddings times this (ScaledEmbedding); None: a plain embedding.
    embed_scale: Optional[float] = None
    # 'layer' (LayerNorm) or 'rms': RMSNorm, each with the addition to the residual stream before it.
    norm: str = "layer"
    # The labels' loss straight from the last hidden rows, without logits (HeadCrossEntropy).
    head_loss: bool = False


GPT2_SMALL = LMConfig()
GPT2_MEDIUM = LMConfig(n_layer=24, n_head=16, d_model=1024, d_mlp=4096)
PYTHIA_1B = LMConfig(n_layer=16, n_head=8, d_model=2048, d_mlp=8192, vocab=50304, n_ctx=2048,
                     rotary=True, tied=False)


def _attention(q, k, v):
    """Causal attention through the fused flash / memory-efficient SDPA kernels only."""
    from torch.nn.attention import SDPBackend, sdpa_kernel
    if q.is_cuda:
        with sdpa_kernel([SDPBackend.FLASH_ATTENTION, SDPBackend.EFFICIENT_ATTENTION]):
            return F.scaled_dot_product_attention(q, k, v, is_causal=True)
    return F.scaled_dot_product_attention(q.float(), k.float(), v.float(),
                                          is_causal=True).to(q.dtype)


def _rotary(x, cos, sin, n_rot):
    xr, xp = x[..., :n_rot], x[..., n_rot:]
    x1, x2 = xr[..., : n_rot // 2], xr[..., n_rot // 2:]
    rot = torch.cat((-x2, x1), dim=-1)
    return torch.cat((xr * cos + rot * sin, xp), dim=-1)


def _norm(cfg: "LMConfig") -> nn.Module:
    if cfg.norm not in ("layer", "rms"):
        raise ValueError(f"norm {cfg.norm!r}: 'layer' or 'rms'")
    return RMSNorm(cfg.d_model) if cfg.norm == "rms" else nn.LayerNorm(cfg.d_model)


class Block(nn.Module):
    def __init__(self, cfg: LMConfig):
        super().__init__()
        self.cfg = cfg
        d = cfg.d_model
        self.ln_1 = _norm(cfg)
        self.qkv = nn.Linear(d, 3 * d)
        self.proj = nn.Linear(d, d)
        if cfg.qk_norm:
            hd = d // cfg.n_head
            self.qk = QKNormRotary(cfg.n_head, cfg.n_head, hd, n_positions=cfg.n_ctx,
                                   n_rot=int(hd * cfg.rotary_pct) if cfg.rotary else 0)
        self.ln_2 = _norm(cfg)
        self.fc = nn.Linear(d, cfg.d_mlp)
        self.fc_out = nn.Linear(cfg.d_mlp, d)

    def forward(self, x, rope=None, stream=None):
        """With cfg.norm 'layer' x is the residual stream, and so is the result.  With 'rms' the stream
        comes beside x, which is still to be added to it (None: x is the stream): (what is to be added,
        stream)."""
        if self.cfg.norm == "rms":
            u, stream = (self.ln_1(x), x) if stream is None else self.ln_1(x, stream)
            u, stream = self.ln_2(self._attend(u, rope), stream)
            return self._mlp(u), stream
        x = x + self._attend(self.ln_1(x), rope)
        return x + self._mlp(self.ln_2(x))

    def _mlp(self, u):
        return self.fc_out(F.gelu(self.fc(u), approximate="tanh"))

    def _attend(self, u, rope):
        B, T, d = u.shape
        H = self.cfg.n_head
        qkv = self.qkv(u)
        if self.cfg.qk_norm:
            q, k, v = self.qk(qkv)
        else:
            q, k, v = qkv.split(d, dim=-1)
            q = q.view(B, T, H, d // H).transpose(1, 2)
            k = k.view(B, T, H, d // H).transpose(1, 2)
            v = v.view(B, T, H, d // H).transpose(1, 2)
            if rope is not None:
                cos, sin, n_rot = rope
                q = _rotary(q, cos, sin, n_rot)
                k = _rotary(k, cos, sin, n_rot)
        y = _attention(q.contiguous(), k.contiguous(), v.contiguous())
        return self.proj(y.transpose(1, 2).reshape(B, T, d))


class CausalLM(nn.Module):
    """GPT-2 (learned positions, tied lm_head) or rotary GPT-NeoX-style (untied embed_out)."""

    def __init__(self, cfg: LMConfig):
        super().__init__()
        self.cfg = cfg
        self.wte = nn.Embedding(cfg.vocab, cfg.d_model) if cfg.embed_scale is None else \
            ScaledEmbedding(cfg.vocab, cfg.d_model, cfg.embed_scale)
        if not cfg.rotary:
            self.wpe = nn.Embedding(cfg.n_ctx, cfg.d_model)
        self.h = nn.ModuleList([Block(cfg) for _ in range(cfg.n_layer)])
        self.ln_f = _norm(cfg)
        self.lm_head = HeadCrossEntropy(cfg.d_model, cfg.vocab) if cfg.head_loss else \
            nn.Linear(cfg.d_model, cfg.vocab, bias=False)
        if cfg.tied:
            self.lm_head.weight = self.wte.weight
        self.ghost_embeddings = ("wte",) if cfg.rotary else ("wte", "wpe")
        self.apply(self._init)

    @staticmethod
    def _init(m):
        if isinstance(m, (nn.Linear, nn.Embedding)):
            nn.init.normal_(m.weight, mean=0.0, std=0.02)
        if isinstance(m, nn.Linear) and m.bias is not None:
            nn.init.zeros_(m.bias)

    def _rope(self, T, device, dtype):
        hd = self.cfg.d_model // self.cfg.n_head
        n_rot = int(hd * self.cfg.rotary_pct)
        inv = 1.0 / (10000 ** (torch.arange(0, n_rot, 2, device=device).float() / n_rot))
        t = torch.arange(T, device=device).float()
        fr = torch.outer(t, inv)
        emb = torch.cat((fr, fr), dim=-1)
        return emb.cos().to(dtype), emb.sin().to(dtype), n_rot

    def forward(self, input_ids, labels=None, teacher=None, temperature=1.0, alpha=0.5):
        """Logits; with labels the mean cross entropy; with `teacher`, a pair of the teacher's top
        ids and logits [B, T, K], the distillation loss (labels: its hard-label part, weighted
        1 - alpha; without labels the teacher alone)."""
        B, T = input_ids.shape
        x = self.wte(input_ids)
        rope = None
        if self.cfg.rotary and not self.cfg.qk_norm:
            rope = self._rope(T, input_ids.device, x.dtype)
        elif not self.cfg.rotary:
            # per-sample position ids so the position embedding's hook sees [B, T]
            pos = torch.arange(T, device=input_ids.device).unsqueeze(0).repeat(B, 1)
            x = x + self.wpe(pos)
        if self.cfg.norm == "rms":
            stream = None
            for blk in self.h:
                x, stream = blk(x, rope, stream)
            x = self.ln_f(x) if stream is None else self.ln_f(x, stream)[0]
        else:
            for blk in self.h:
                x = blk(x, rope)
            x = self.ln_f(x)
        if self.cfg.head_loss and labels is not None and teacher is None:
            return self.lm_head(x, labels)
        logits = self.lm_head(x)
        if teacher is not None:
            return distillation_loss(logits, *teacher, labels, temperature=temperature,
                                     alpha=1.0 if labels is None else alpha)
        if labels is None:
            return logits
        return F.cross_entropy(logits.float().view(-1, logits.shape[-1]), labels.reshape(-1))


def synthetic_tokens(n_rows: int, T: int, vocab: int, seed: int, device="cpu"):
    """Uniform token ids and next-token labels (ids shifted by one, last label random)."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, vocab, (n_rows, T + 1), generator=g)
    return ids[:, :T].contiguous().to(device), ids[:, 1:].contiguous().to(device)


def lm_flops_per_step(cfg: LMConfig, n_rows: int, T: int) -> float:
    """6 * params * tokens + attention (fwd+bwd), the plain-backprop work of one step."""
    d, L = cfg.d_model, cfg.n_layer
    params = L * (4 * d * d + 2 * d * cfg.d_mlp) + cfg.vocab * d
    attn = L * 2 * 2 * T * T * d * 3  # QK^T and PV, fwd + 2x bwd
    return 6.0 * params * n_rows * T + attn * n_rows
