"""Layers and a loss of a language model's training step, on the gfx950 kernels.

  - ``embedding_lookup`` / ``ScaledEmbedding``: rows of an embedding table times a scale, and the
    table's gradient.
  - ``qkv_norm_rotary`` / ``qk_norm_rotary`` / ``QKNormRotary``: each head's root-mean-square
    norm of the queries and keys, their rotation by position, and the heads-first layout
    attention takes, in one pass forward and one backward.
  - ``distillation_loss``: the loss of logits against a teacher's top logits, alone or beside the
    labels' cross entropy, with its gradient.
  - ``head_cross_entropy`` / ``HeadCrossEntropy``: the output projection with its softmax cross
    entropy, in pieces of the vocabulary, without keeping the logits.
  - ``rms_norm`` / ``add_rms_norm`` / ``RMSNorm``: the root-mean-square norm of a residual stream,
    with the residual's addition.

All are differentiable (once), run on the current stream and take bf16 or fp32 tensors on a ROCm
GPU; anything else raises ``GhostHipError``, as do forward-mode differentiation, function
transforms (``torch.func``) and ``torch.jit`` tracing.  The layers are ones that the engines know:
``GradDotProdEngine`` gives their weights gradient dot products and train gradients,
``GradProjLoraEngine`` projects a ``ScaledEmbedding`` and a ``HeadCrossEntropy``.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch import nn

from ._native import GhostHipError, ops

__all__ = ["embedding_lookup", "ScaledEmbedding", "rotary_table", "qkv_norm_rotary",
           "qk_norm_rotary", "QKNormRotary", "distillation_loss", "head_cross_entropy",
           "HeadCrossEntropy", "rms_norm", "add_rms_norm", "RMSNorm"]


# Embedding lookup ###########################################################################

def embedding_lookup(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
                     padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[ids]``, [*ids.shape, d] in weight's dtype (fp32 product, one rounding).

    ids: int32 or int64 of any shape; one outside [0, len(weight)) gives a row of zeros and no
    gradient.  weight: [vocab, d].  padding_idx: the id whose row gets no gradient (negative:
    counted from the end).  The gradient sums each id's rows in fp32 in a fixed order."""
    if padding_idx is not None:
        if not -weight.shape[0] <= padding_idx < weight.shape[0]:
            raise GhostHipError(f"padding_idx {padding_idx} outside the table of "
                                f"{weight.shape[0]} rows")
        padding_idx %= weight.shape[0]
    return ops().embedding_lookup(ids, weight, float(scale), padding_idx)


class ScaledEmbedding(nn.Embedding):
    """An ``nn.Embedding`` whose rows are multiplied by ``scale`` (default: the square root of
    the embedding's width).  The options that change the weight or its gradient elsewhere
    (``max_norm``, ``scale_grad_by_freq``, ``sparse``) are not taken."""

    def __init__(self, num_embeddings: int, embedding_dim: int, scale: Optional[float] = None,
                 padding_idx: Optional[int] = None, device=None, dtype=None):
        super().__init__(num_embeddings, embedding_dim, padding_idx=padding_idx, device=device,
                         dtype=dtype)
        self.scale = math.sqrt(embedding_dim) if scale is None else float(scale)

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        return embedding_lookup(input, self.weight, self.scale, self.padding_idx)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, scale={self.scale:g}"


# Norms of queries and keys with their rotation ###############################################

def rotary_table(n_positions: int, n_rot: int, base: float = 10000.0, device=None
                 ) -> torch.Tensor:
    """[n_positions, 2, n_rot / 2] fp32: the cosines, then the sines, of each position's angles
    ``position * base^(-2 i / n_rot)``, formed in float64."""
    if n_positions <= 0 or n_rot < 0 or n_rot % 2:
        raise GhostHipError(f"rotary_table: {n_positions} positions, {n_rot} rotated features "
                            "(an even number)")
    i = torch.arange(n_rot // 2, device=device, dtype=torch.float64)
    inv = torch.pow(float(base), -2.0 * i / max(n_rot, 1))
    a = torch.arange(n_positions, device=device, dtype=torch.float64)[:, None] * inv
    return torch.stack((a.cos(), a.sin()), dim=1).float()


def _check_norm(norm, q_weight, k_weight) -> None:
    if not norm and (q_weight is not None or k_weight is not None):
        raise GhostHipError("norm weights without the norm")


def qkv_norm_rotary(qkv: torch.Tensor, n_head: int, n_kv_head: int, table: torch.Tensor,
                    positions: Optional[torch.Tensor] = None,
                    q_weight: Optional[torch.Tensor] = None,
                    k_weight: Optional[torch.Tensor] = None, *, norm: bool = True,
                    eps: float = 1e-6, interleaved: bool = False
                    ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Queries [B, n_head, T, D], keys and values [B, n_kv_head, T, D] from a fused projection.

    qkv: [B, T, (n_head + 2 n_kv_head) D] or [B, T, n_head + 2 n_kv_head, D], queries first, then
    keys, then values; any strides over contiguous features.  Each query and key row is divided by
    its root mean square (with ``norm``) and multiplied by q_weight / k_weight ([D], or None), then
    its first n_rot features are rotated: ``table`` is ``rotary_table``'s [positions, 2, n_rot / 2]
    (n_rot 0: no rotation), the pairs n_rot / 2 apart, or neighbours with ``interleaved``.
    positions: None (0, 1, ... in each sample; the table has to hold them) or integers [T] or
    [B, T]; one of those outside the table makes the rotated features NaN.  Formed in fp32,
    rounded once; D up to 512."""
    _check_norm(norm, q_weight, k_weight)
    q, k, v = ops().qk_norm_rotary(qkv, None, (n_head, n_kv_head, n_kv_head), table, positions,
                                   q_weight, k_weight, bool(norm), float(eps), bool(interleaved))
    return q, k, v


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, table: torch.Tensor,
                   positions: Optional[torch.Tensor] = None,
                   q_weight: Optional[torch.Tensor] = None,
                   k_weight: Optional[torch.Tensor] = None, *, norm: bool = True,
                   eps: float = 1e-6, interleaved: bool = False
                   ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``qkv_norm_rotary`` for queries [B, T, n_head, D] and keys [B, T, n_kv_head, D] of
    projections of their own: ([B, n_head, T, D], [B, n_kv_head, T, D])."""
    if q.dim() != 4 or k.dim() != 4:
        raise GhostHipError(f"expected queries and keys [B, T, heads, D], got {tuple(q.shape)} "
                            f"and {tuple(k.shape)}")
    _check_norm(norm, q_weight, k_weight)
    q, k = ops().qk_norm_rotary(q, k, (q.shape[2], k.shape[2], 0), table, positions, q_weight,
                                k_weight, bool(norm), float(eps), bool(interleaved))
    return q, k


class QKNormRotary(nn.Module):
    """``qkv_norm_rotary`` as a layer: ``layer(qkv, positions=None)`` gives (q, k, v).

    ``q_weight`` and ``k_weight`` ([head_dim], ones) are its parameters with ``norm`` (None
    without); ``table`` holds the angles of n_positions positions in fp32, whatever dtype the
    module is cast to.  n_rot: rotated features of a head (default all of them)."""

    def __init__(self, n_head: int, n_kv_head: int, head_dim: int, n_rot: Optional[int] = None,
                 n_positions: int = 2048, base: float = 10000.0, eps: float = 1e-6,
                 norm: bool = True, interleaved: bool = False, device=None, dtype=None):
        super().__init__()
        self.n_head, self.n_kv_head, self.head_dim = n_head, n_kv_head, head_dim
        self.n_rot = head_dim - head_dim % 2 if n_rot is None else n_rot
        if not 0 <= self.n_rot <= head_dim:
            raise GhostHipError(f"{self.n_rot} rotated features of {head_dim}")
        self.n_positions, self.base = n_positions, float(base)
        self.eps, self.norm, self.interleaved = float(eps), bool(norm), bool(interleaved)
        for name in ("q_weight", "k_weight"):
            w = nn.Parameter(torch.ones(head_dim, device=device, dtype=dtype)) if norm else None
            self.register_parameter(name, w)
        self.table = rotary_table(n_positions, self.n_rot, base, device)

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        # Not a buffer: a cast of the module would round the angles.
        device = fn(torch.empty(0, device=self.table.device)).device
        if device != self.table.device:
            self.table = rotary_table(self.n_positions, self.n_rot, self.base, device)
        return self

    def forward(self, qkv: torch.Tensor, positions: Optional[torch.Tensor] = None):
        sample_grads = None
        if self.norm and self._backward_hooks and hasattr(self.q_weight, "initially_requires_grad"):
            # An engine's backward hook reads these: the positions, and each sample's gradients of
            # the weights, which the backward pass forms on its way (it runs before the hook when
            # the input has a gradient).  A forward whose tensor no hook has taken yet leaves it to
            # the next one of the model's step: activation checkpointing runs the forward again within
            # the backward pass of the first run's nodes, which write the tensor they were given.
            d = self.__dict__
            if torch.is_grad_enabled() and qkv.requires_grad:
                shape = (2, qkv.shape[0], self.head_dim)
                sample_grads = d.get("_gs_sample_grads")
                if sample_grads is None or sample_grads.shape != shape or \
                        sample_grads.device != qkv.device:
                    sample_grads = torch.empty(shape, device=qkv.device, dtype=torch.float32)
                d["_gs_sample_version"] = sample_grads._version   # a backward pass counts it up
            d["_gs_positions"] = positions
            d["_gs_sample_grads"] = sample_grads
        q, k, v = ops().qk_norm_rotary(
            qkv, None, (self.n_head, self.n_kv_head, self.n_kv_head), self.table, positions,
            self.q_weight, self.k_weight, self.norm, self.eps, self.interleaved, sample_grads)
        return q, k, v

    def extra_repr(self) -> str:
        return (f"{self.n_head}, {self.n_kv_head}, {self.head_dim}, n_rot={self.n_rot}, "
                f"eps={self.eps:g}, norm={self.norm}, interleaved={self.interleaved}")


# Loss against a teacher's top logits #########################################################

def distillation_loss(logits: torch.Tensor, teacher_ids: torch.Tensor,
                      teacher_logits: torch.Tensor, labels: Optional[torch.Tensor] = None, *,
                      temperature: float = 1.0, alpha: float = 1.0, ignore_index: int = -100,
                      reduction: str = "mean") -> torch.Tensor:
    """The loss of student logits [..., V] against a teacher's top logits.

    Per row, with p the softmax of teacher_logits / temperature over the row's teacher entries and
    q the student's softmax of logits / temperature over the whole vocabulary:

        alpha temperature^2 sum_k p_k (log p_k - log q[id_k]) + (1 - alpha) cross entropy(label)

    teacher_ids, teacher_logits: [..., K], K up to 1024.  An entry whose id is outside [0, V) or
    whose logit is -inf takes no part; a row with none left has no first term; an id that stands
    twice counts twice.  labels: [...]; rows whose label is ignore_index count for nothing, their
    gradient is zero; may be None with alpha = 1.  Another label outside [0, V) makes its row NaN
    (alpha < 1).  temperature: positive, its square and 1.45 times its inverse within fp32.
    reduction: 'mean' (over the rows not ignored; NaN when there are none), 'sum', or 'none' ([...]).
    The loss is fp32; no gradient reaches the teacher.

    With 'mean' and 'sum' the loss's pass also writes the logits' gradient for an upstream gradient
    of one.  Any other, of a loss that is scaled or weighted, has the backward pass form it again:
    951 us instead of 432 for 8192 x 50257 bf16 logits, loss and gradient.  'none' with the weights
    as the rows' upstream gradients takes 583 us whatever they are."""
    _check_reduction(reduction)
    if labels is None and alpha != 1.0:
        raise GhostHipError("labels are needed unless alpha is 1")
    return ops().distillation_loss(logits, teacher_ids, teacher_logits, labels, float(temperature),
                                   float(alpha), int(ignore_index), reduction)


def _autocast() -> bool:
    return torch.is_autocast_enabled("cuda")


# Output projection with its cross entropy ####################################################

def _check_reduction(reduction) -> None:
    if reduction not in ("mean", "sum", "none"):
        raise GhostHipError(f"reduction {reduction!r}: 'mean', 'sum' or 'none'")


def head_cross_entropy(x: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, *,
                       ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """``cross_entropy(x @ weight.T, labels)`` without the logits.

    x: [..., d] hidden rows, weight: [vocab, d], of one type (bf16 or fp32); labels: [...] integers.
    The logits are formed in fp32 a piece of the vocabulary at a time, once in the forward pass and
    again in the backward pass, and never stored; the gradient of a piece is (in up to 1 GiB, but at
    least 256 entries), before it is multiplied into the gradients of x and weight: rounded once to
    bf16 in a bf16 model, for up to 32 rows in two bf16 parts.
    Rows whose label is ignore_index take no part and are not read; their loss and gradient are zero.
    Another label outside [0, vocab) makes its row's loss and gradient NaN.
    reduction: 'mean' (over the rows not ignored; NaN when there are none), 'sum', or 'none' ([...]).
    The loss is fp32.  Under autocast x and weight are cast to its type, as an ``nn.Linear``'s."""
    _check_reduction(reduction)
    x, weight = _head_operands(x, weight)
    return ops().head_cross_entropy(x, weight, labels, int(ignore_index), reduction)


def _head_operands(x: torch.Tensor, weight: torch.Tensor):
    if not _autocast():
        return x, weight
    dtype = torch.get_autocast_dtype("cuda")
    return x.to(dtype), weight.to(dtype)


class HeadCrossEntropy(nn.Linear):
    """An output projection without a bias that can end in its loss: ``layer(x)`` gives the logits as
    an ``nn.Linear`` does, ``layer(x, labels)`` the loss of ``head_cross_entropy``."""

    def __init__(self, in_features: int, out_features: int, ignore_index: int = -100,
                 reduction: str = "mean", device=None, dtype=None):
        super().__init__(in_features, out_features, bias=False, device=device, dtype=dtype)
        _check_reduction(reduction)
        self.ignore_index, self.reduction = int(ignore_index), reduction

    def forward(self, input: torch.Tensor, labels: Optional[torch.Tensor] = None) -> torch.Tensor:
        d, lse = self.__dict__, None
        d.pop("_gs_head", None)
        if labels is None:
            return super().forward(input)
        x, weight = _head_operands(input, self.weight)
        if self._backward_hooks and torch.is_grad_enabled():
            # An engine's backward hook forms the gradient of the logits from these.
            lse = torch.empty((*labels.shape, 2), device=labels.device, dtype=torch.float32)
            d["_gs_head"] = (x.detach(), labels, lse)
        return ops().head_cross_entropy(x, weight, labels, self.ignore_index, self.reduction, lse)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, reduction={self.reduction}"


PIECE_BYTES = 512 << 20   # of a piece of the logits' gradient under an engine, but for one of 256 entries


def head_gradient_pieces(layer: HeadCrossEntropy, x: torch.Tensor, labels: torch.Tensor,
                         lse: torch.Tensor, grad: torch.Tensor):
    """(first entry, entries, gradient of those logits [*labels.shape, entries up to a multiple of 8])
    of a HeadCrossEntropy's loss, piece by piece of the vocabulary, in up to PIECE_BYTES each (but at
    least 256 entries).  x: the rows as the loss took them."""
    weight = layer.weight.detach().to(x.dtype)
    vocab = weight.shape[0]
    each = max(256, PIECE_BYTES // max(1, labels.numel() * x.element_size()) // 256 * 256)
    each = -(-vocab // (-(-vocab // each)))               # pieces of a size
    each = -(-each // 256) * 256
    for v0 in range(0, vocab, each):
        n = min(each, vocab - v0)
        yield v0, n, ops().head_logit_grad(x, weight, labels, lse, grad, v0, n, layer.ignore_index,
                                           layer.reduction)


# Root-mean-square norm of a residual stream ##################################################

def _norm_operands(*tensors: torch.Tensor):
    """Tensors of several types: under autocast all in fp32, as torch's norms take them there."""
    return tuple(t.float() for t in tensors) if _autocast() else tensors


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6) -> torch.Tensor:
    """``weight * x / sqrt(mean(x^2) + eps)`` over the last dimension, in fp32, rounded once.
    x: [..., d], weight: [d], of one type; of several under autocast, which gives fp32."""
    if x.dtype != weight.dtype:
        x, weight = _norm_operands(x, weight)
    return ops().rms_norm(x, None, weight, float(eps))[0]


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, *,
                 eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """(``rms_norm(h, weight)``, h) with h = x + residual (one rounding), in one pass; x and residual
    of one shape, all of one type (under autocast as ``rms_norm``)."""
    if not x.dtype == residual.dtype == weight.dtype:
        x, residual, weight = _norm_operands(x, residual, weight)
    y, h = ops().rms_norm(x, residual, weight, float(eps))
    return y, h


class RMSNorm(nn.Module):
    """``rms_norm`` as a layer: ``layer(x)`` gives the normed rows, ``layer(x, residual)`` those of
    x + residual and that sum (``add_rms_norm``)."""

    def __init__(self, dim: int, eps: float = 1e-6, device=None, dtype=None):
        super().__init__()
        self.dim, self.eps = dim, float(eps)
        self.weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype))

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        if residual is None:
            return rms_norm(x, self.weight, eps=self.eps)
        return add_rms_norm(x, residual, self.weight, eps=self.eps)

    def extra_repr(self) -> str:
        return f"{self.dim}, eps={self.eps:g}"
