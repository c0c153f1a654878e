"""Float64 forms of the language-model operators, and a stand-in kernel layer made of them.

Everything is computed on the CPU in float64 from the definitions; the gradients are automatic
differentiation of the forward forms (which ``tests/test_lm_layers.py`` holds against differences).
"""
import math

import torch

from ghostsuite_amd import lm_layers
from tests.oracle_backend import OracleOps

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}   # of a rounding, relative
U = 2.0 ** -24                                                  # of one fp32 operation


def f64(x):
    return None if x is None else x.detach().cpu().double()


# ------------------------------------------------------------------------------ embedding
def lookup(ids, weight, scale):
    """weight float64; zero rows for ids outside the table."""
    inside = (ids >= 0) & (ids < weight.shape[0])
    rows = weight[ids.long().clamp(0, weight.shape[0] - 1)]
    return torch.where(inside[..., None], rows * scale, 0.0)


def lookup_grad(ids, g, vocab, scale, padding_idx=None):
    """(gradient, sum of the addends' magnitudes, addends per row)."""
    ids, g = ids.reshape(-1).long(), g.reshape(ids.numel(), -1)
    keep = (ids >= 0) & (ids < vocab)
    if padding_idx is not None:
        keep &= ids != padding_idx % vocab
    z = torch.zeros(vocab, g.shape[1], dtype=torch.float64)
    n = torch.zeros(vocab, dtype=torch.float64)
    k, r = ids[keep], g[keep]
    return (z.index_add(0, k, r) * scale, z.index_add(0, k, r.abs()) * abs(scale),
            n.index_add(0, k, torch.ones_like(k, dtype=torch.float64)))


# ------------------------------------------------- norms of queries and keys, rotation
def _turn(x, cos, sin, interleaved):
    """x [B, T, H, D]; cos, sin [B, T, 1, n_rot / 2]."""
    n = cos.shape[-1]
    r, rest = x[..., :2 * n], x[..., 2 * n:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = r[..., :n], r[..., n:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, rest), -1)


def angles(table, positions, B, T):
    """cos, sin [B, T, 1, n_rot / 2] float64 of a table's positions (NaN outside it)."""
    table = f64(table)
    pos = torch.arange(T) if positions is None else positions.detach().cpu().long()
    pos = pos.expand(B, T)
    inside = (pos >= 0) & (pos < table.shape[0])
    at = table[pos.clamp(0, table.shape[0] - 1)]
    at = torch.where(inside[..., None, None], at, math.nan)
    return at[..., 0, :].unsqueeze(-2), at[..., 1, :].unsqueeze(-2)


def qk_forward(x, w, cos, sin, norm, eps, interleaved):
    """One part [B, T, H, D] float64, heads first; w None: values, copied."""
    if w is not None:
        if norm:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
        if cos.shape[-1]:
            x = _turn(x, cos, sin, interleaved)
    return x.transpose(1, 2)


def split_heads(plan, parts):
    """The three parts [B, T, H, D] (None where there are none) of packed or separate inputs."""
    heads = plan["heads"]
    if len(parts) == 1:
        x = parts[0]
        x = x.reshape(x.shape[0], x.shape[1], sum(heads), -1)
        return list(x.split(list(heads), 2))
    return [*parts, None]


def qk_all(plan, parts, qw, kw):
    """Forward of every part from float64 inputs (differentiable)."""
    xs = split_heads(plan, parts)
    B, T, _, D = xs[0].shape
    cos, sin = angles(plan["table"], plan["positions"], B, T)
    ones = torch.ones(D, dtype=torch.float64)
    ws = (ones if qw is None else qw, ones if kw is None else kw, None)
    return [qk_forward(x, w, cos, sin, plan["norm"], plan["eps"], plan["interleaved"])
            for x, w in zip(xs, ws) if x is not None]


@torch.enable_grad()
def qk_grads(plan, parts, qw, kw, grads, per_sample=False):
    """([gradients of parts], dqw, dkw) in float64; per_sample: the weights' of each sample."""
    parts = [f64(p).requires_grad_() for p in parts]
    B, D = parts[0].shape[0], grads_dim(plan, parts)
    w = [torch.ones(D, dtype=torch.float64) if x is None else f64(x) for x in (qw, kw)]
    w = [x.expand(B, D).clone().requires_grad_() for x in w]
    out = qk_all(plan, parts, w[0][:, None, None], w[1][:, None, None])
    pairs = [(o, f64(g)) for o, g in zip(out, grads) if g is not None]
    got = torch.autograd.grad([o for o, _ in pairs], [*parts, *w], [g for _, g in pairs],
                              allow_unused=True)
    got = [torch.zeros_like(x) if g is None else g for g, x in zip(got, [*parts, *w])]
    dq, dk = got[-2:]
    return got[:-2], (dq if per_sample else dq.sum(0)), (dk if per_sample else dk.sum(0))


def grads_dim(plan, parts):
    x = parts[0]
    return x.shape[3] if x.dim() == 4 else x.shape[2] // sum(plan["heads"])


# ----------------------------------------------------------------------------- distillation
def distill_rows(z, ids, t, labels, tau, alpha, ignore=-100):
    """Row losses [N] of float64 logits [N, V] (differentiable), and which rows count."""
    N, V = z.shape
    use = (ids >= 0) & (ids < V) & (t != -math.inf)
    kept = torch.ones(N, dtype=torch.bool) if labels is None else labels != ignore
    rows = []
    for n in range(N):
        if not kept[n]:
            rows.append(z.new_zeros(()))
            continue
        loss = z.new_zeros(())
        if alpha != 0 and use[n].any():
            lp = torch.log_softmax(t[n][use[n]] / tau, 0)
            lq = torch.log_softmax(z[n] / tau, 0)[ids[n][use[n]]]
            p = lp.exp()
            term = torch.where(p > 0, p * (lp - lq), 0.0)
            loss = loss + alpha * tau ** 2 * term.sum()
        if alpha != 1:
            y = int(labels[n])
            loss = loss + (1 - alpha) * (-torch.log_softmax(z[n], 0)[y] if 0 <= y < V
                                         else z[n].sum() * math.nan)
        rows.append(loss)
    return torch.stack(rows), kept


def reduced(rows, kept, reduction):
    if reduction == "none":
        return rows
    return rows.sum() / (kept.sum() if reduction == "mean" else 1)


# -------------------------------------------------------------- the stand-in kernel layer
class LmOracleOps(OracleOps):
    """OracleOps with the language-model operators, for engine tests without a GPU."""

    # ids outside the table take no part: their rows count as zeros of id 0
    @staticmethod
    def _inside(ids, G):
        G3 = G.reshape(*ids.shape, -1)
        return ids.clamp(min=0), torch.where((ids < 0)[..., None], torch.zeros_like(G3), G3)

    def embedding_dot(self, ids, G, *args, **kw):
        return super().embedding_dot(*self._inside(ids, G), *args, **kw)

    def embedding_train_grad(self, ids, G, *args, **kw):
        return super().embedding_train_grad(*self._inside(ids, G), *args, **kw)

    def embedding_layer_pass(self, ids, G, *args, **kw):
        return super().embedding_layer_pass(*self._inside(ids, G), *args, **kw)

    # (differentiable as they stand: autograd records the float64 forms)
    def embedding_lookup(self, ids, weight, scale, padding_idx=None):
        w = weight.double()
        if padding_idx is not None:
            w = torch.where((torch.arange(len(w)) == padding_idx)[:, None], w.detach(), w)
        return lookup(ids, w, scale).to(weight.dtype)

    def qk_norm_rotary(self, q, k, heads, table, positions, qw, kw, norm, eps, interleaved,
                       sample_grads=None):
        parts = [p.double() for p in (q, k) if p is not None]
        if sample_grads is not None:   # weights of each sample, whose gradients a hook keeps
            B, D = sample_grads.shape[1:]
            w = [x.detach().double().expand(B, D).clone().requires_grad_() for x in (qw, kw)]
            for i in range(2):
                w[i].register_hook(lambda g, i=i: sample_grads[i].copy_(g) * 0 + g)
            out = qk_all(plan(heads, table, positions, norm, eps, interleaved), parts,
                         w[0][:, None, None], w[1][:, None, None])
            return [y.to(q.dtype).contiguous() for y in out]
        w = [None if x is None else x.double() for x in (qw, kw)]
        return [y.to(q.dtype).contiguous()
                for y in qk_all(plan(heads, table, positions, norm, eps, interleaved), parts, *w)]

    def qk_norm_rotary_dots(self, q, k, heads, table, positions, qw, kw, eps, interleaved, grads,
                            n_val, *, val_start=None, grad_scale=None):
        self.calls.append(("qk_norm_rotary_dots", tuple(q.shape)))
        parts = [p for p in (q, k) if p is not None]
        _, dq, dk = qk_grads(plan(heads, table, positions, True, eps, interleaved), parts, qw, kw,
                             grads, per_sample=True)
        B = dq.shape[0]
        vs = B - n_val if val_start is None else val_start
        val = torch.zeros(B, dtype=torch.bool)
        val[vs:vs + n_val] = True
        out = [(s[~val] @ s[val].sum(0)).float() for s in (dq, dk)]
        for s, w in ((dq, qw), (dk, kw)):
            out.append(None if grad_scale is None else (s[~val].sum(0) * grad_scale).to(w.dtype))
        return out

    def qk_sample_dots(self, sample_grads, qw, kw, n_val, *, val_start=None, grad_scale=None):
        self.calls.append(("qk_sample_dots", tuple(sample_grads.shape)))
        B = sample_grads.shape[1]
        vs = B - n_val if val_start is None else val_start
        val = torch.zeros(B, dtype=torch.bool)
        val[vs:vs + n_val] = True
        out = [(s[~val] @ s[val].sum(0)).float() for s in sample_grads]
        for s, w in zip(sample_grads, (qw, kw)):
            out.append(None if grad_scale is None else (s[~val].sum(0) * grad_scale).to(w.dtype))
        return out

    def distillation_loss(self, logits, ids, t, labels, temperature, alpha, ignore_index, reduction):
        V, K = logits.shape[-1], ids.shape[-1]
        rows, kept = distill_rows(logits.double().reshape(-1, V), ids.reshape(-1, K),
                                  f64(t).reshape(-1, K),
                                  None if labels is None else labels.reshape(-1), temperature, alpha,
                                  ignore_index)
        loss = reduced(rows, kept, reduction).float()
        return loss.reshape(logits.shape[:-1] if reduction == "none" else ())


def plan(heads, table, positions=None, norm=True, eps=1e-6, interleaved=False):
    return {"heads": heads, "table": table, "positions": positions, "norm": norm, "eps": eps,
            "interleaved": interleaved}


def table64(n_positions, n_rot, base=10000.0):
    return lm_layers.rotary_table(n_positions, n_rot, base)
