"""Float64 forms of the output projection with its cross entropy, the root-mean-square norm and AdamW,
their error bounds, and a stand-in kernel layer made of them.

Gradients are automatic differentiation of the forward forms (which ``tests/test_lm_train.py`` holds
against differences).  Bounds count, elementwise, U = 2^-24 for an fp32 operation and HALF[t] for the
rounding to type t.
"""
import math

import torch

from tests.lm_forms import HALF, U, LmOracleOps, f64


# ------------------------------------------------------- output projection, cross entropy
def head_rows(x, w, labels, ignore=-100):
    """(row losses of float64 x [N, d], w [V, d]; which rows count).  Rows that do not are not read."""
    V, kept = w.shape[0], labels != ignore
    rows = []
    for n in range(x.shape[0]):
        if not kept[n]:
            rows.append(x.new_zeros(()))
            continue
        z, y = w @ x[n], int(labels[n])
        rows.append(-torch.log_softmax(z, 0)[y] if 0 <= y < V else z.sum() * math.nan)
    return torch.stack(rows) if rows else x.new_zeros(0), kept


def head_loss(x, w, labels, reduction, ignore=-100):
    rows, kept = head_rows(x, w, labels, ignore)
    if reduction == "none":
        return rows
    return rows.sum() / (kept.sum() if reduction == "mean" else 1)


def head_all(x, w, labels, up, reduction, dtype, ignore=-100):
    """Loss, dx, dw of inputs of `dtype` in float64, and a bound of each one's error: {name: (value,
    bound)}.

    Logits: sums of d products, of 6 d products of parts with fp32 operands, whose parts leave out at most
    4 U of a product (2^-24 of each operand by the last part's rounding, and the products m l and l m, 2^-24
    each): off by ez = (6 d + 16) U sum |x w| at most.  The row's log of the sum of exponentials is off
    by the mean of ez under the softmax, by the rounding of z log2(e) and of the exponential and its
    argument (8 U (1 + |z|) each, as a share of its exponential), and by the sum's at most 64 + V / 128 + 40
    additions.  dz then is off by that share of p; between the products it is held in bf16 (HALF of its
    size with bf16 operands), and every sum adds its number of terms, times three for the parts."""
    N, (V, d) = x.shape[0], w.shape
    x, w, keep = f64(x), f64(w), labels != ignore
    y = labels.clamp(0, V - 1)
    fp32 = dtype == torch.float32
    half = U if fp32 else HALF[dtype]
    xs = torch.where(keep[:, None], x, 0.0)
    z = xs @ w.t()
    lp = torch.log_softmax(z, 1)
    p = lp.exp()
    ez = (6 * d + 16) * U * (xs.abs() @ w.abs().t()) + 8 * U * (1 + z.abs())
    el = (p * ez).sum(1) + (64 + V / 128 + 40) * U + 8 * U * torch.logsumexp(z, 1).abs()
    bad = keep & ((labels < 0) | (labels >= V))
    at = torch.arange(N)
    rows = torch.where(keep, -lp[at, y], 0.0)
    rows[bad] = math.nan
    erows = torch.where(keep, el + ez[at, y] + 8 * U * (z[at, y].abs() + rows.nan_to_num(0.0)), 0.0)
    count = max(1, int(keep.sum()))
    weight = up.double().expand(N) if reduction == "none" else \
        up.double().expand(N) / (count if reduction == "mean" else 1)
    dz = p - torch.nn.functional.one_hot(y, V)
    edz = p * (ez + el[:, None] + 16 * U) + half * dz.abs() * (1 + 2 * U) + 2 * U
    dz, edz = (t * torch.where(keep, weight if t is dz else weight.abs(), 0.0)[:, None]
               for t in (dz, edz))
    edz = edz + 4 * U * dz.abs()
    dz[bad] = math.nan
    terms = 3 * 6 if fp32 else 3
    out = {}
    loss = rows if reduction == "none" else rows.sum() / (count if reduction == "mean" else 1)
    eloss = erows if reduction == "none" else \
        (erows.sum() + (N / 64 + 20) * U * rows.abs().sum()) / (count if reduction == "mean" else 1) + \
        4 * U * loss.abs()
    if reduction == "mean" and not keep.any():
        loss = torch.tensor(math.nan, dtype=torch.float64)
    out["loss"] = loss, eloss
    for name, a, e, b in (("dx", dz, edz, w), ("dw", dz.t(), edz.t(), xs)):
        value = a @ b
        bound = e.abs() @ b.abs() + (terms * a.shape[1] + 64) * U * (a.abs() @ b.abs())
        if name == "dx":
            value[~keep], bound[~keep] = 0.0, 0.0
        out[name] = value, bound + value.abs() * (HALF[dtype] + 8 * U)
    return out


def head_dz(x, w, labels, grad, v0, n, reduction, ignore=-100):
    """The gradient of the logits [v0, v0 + n) of float64 rows, zeros where a row does not count."""
    kept = labels != ignore
    z = x @ w.t()
    dz = torch.softmax(z, 1) - torch.nn.functional.one_hot(labels.clamp(0, len(w) - 1), len(w))
    weight = grad.double() if reduction == "none" else \
        grad.double() / (kept.sum() if reduction == "mean" else 1)
    return torch.where(kept[:, None], dz * weight.reshape(-1, 1), 0.0)[:, v0:v0 + n]


# --------------------------------------------------------------------- root-mean-square norm
def norm_form(h, w, eps):
    return w * (h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps))


def norm_all(h, w, gy, gh, eps, dtype):
    """{name: (value, bound)} of y, dh, dw from the rows h as the norm took them.

    The mean of squares is off by (F + 8) U of itself at most (no sum has more additions), r by half of that;
    the gradient's mean likewise over the sizes of its addends; dw's sums over M rows by (M + 40) U of theirs."""
    h, w, gy, gh = (f64(t) for t in (h, w, gy, gh))
    F = h.shape[-1]
    er = (F / 2 + 8) * U
    r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    n = h * r
    y = w * n
    out = {"y": (y, y.abs() * (er + 6 * U + HALF[dtype]))}
    g = torch.zeros_like(h) if gy is None else gy
    mean, size = (g * w * n).mean(-1, keepdim=True), (g * w * n).abs().mean(-1, keepdim=True)
    dh = r * (w * g - n * mean)
    bound = r * ((w * g).abs() * (er + 8 * U) + n.abs() * (2 * er + 8 * U) * mean.abs() +
                 n.abs() * (F + 8) * U * size) + dh.abs() * 4 * U
    if gh is not None:
        dh = dh + gh
        bound = bound + gh.abs() * U
    out["dh"] = dh, bound + dh.abs() * (HALF[dtype] + U)
    a = (g * n).reshape(-1, F)
    dw = a.sum(0)
    out["dw"] = dw, a.abs().sum(0) * (er + (a.shape[0] + 40) * U) + dw.abs() * HALF[dtype]
    return out


# ---------------------------------------------------------------------------------- AdamW
TOP, BLOCK, M32 = 448.0, 256, 0xFFFFFFFF


def chances(n, step, seed):
    """The two numbers of [0, 1) of each of a tensor's n elements."""
    i = torch.arange(n, dtype=torch.int64)
    x = (i + step * 0x9E3779B9 + seed * 0x6A09E667) & M32
    x = (x * 0x9E3779B9) & M32
    x = ((x ^ (x >> 15)) * 0xBB67AE85) & M32
    x = x ^ (x >> 13)
    return ((x & 0xFFFF).double() + 0.5) / 65536, ((x >> 16).double() + 0.5) / 65536


def grid_step(a):
    """The distance of the 8-bit values at a: 2^-9 below 2^-6, then an eighth of each power of two."""
    return torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)


def averages(state, shape, bits):
    """m and the root of v in float64, flat."""
    if bits == 32:
        return f64(state["exp_avg"]).reshape(-1), f64(state["exp_avg_sq"]).reshape(-1).sqrt()
    out = []
    for name in ("exp_avg", "root_avg_sq"):
        q, s = state[name].detach().cpu().float().double().reshape(-1), f64(state[name + "_scale"])
        out.append(q * s.repeat_interleave(BLOCK)[:q.numel()])
    return out


def adamw_form(p, g, m, root, lr, betas, eps, decay, step):
    """(p, m, v, root) in float64 after the step."""
    b1, b2 = betas
    m = b1 * m + (1 - b1) * g
    v = b2 * root ** 2 + (1 - b2) * g ** 2
    root = v.sqrt()
    p = (1 - lr * decay) * p - lr / (1 - b1 ** step) * m / (root / math.sqrt(1 - b2 ** step) + eps)
    return p, m, v, root


def held(a, u):
    return torch.floor(a / grid_step(a) + u) * grid_step(a)


def blocks_max(x):
    pad = torch.zeros(-x.numel() % BLOCK, dtype=x.dtype)
    return torch.cat((x, pad)).view(-1, BLOCK).abs().amax(1)


# -------------------------------------------------------------- the stand-in kernel layer
class TrainOracleOps(LmOracleOps):
    """LmOracleOps with these operators, for host-logic tests without a GPU."""

    def head_cross_entropy(self, x, weight, labels, ignore_index, reduction, lse=None):
        self.calls.append(("head_cross_entropy", tuple(x.shape)))
        w = weight.double()
        rows, y = x.double().reshape(-1, w.shape[1]), labels.reshape(-1)
        if lse is not None:
            with torch.no_grad():
                z = rows @ w.t()
                top = z.amax(1, keepdim=True)
                lse.copy_(torch.cat((top / math.log(2), (z - top).exp().sum(1, keepdim=True)), 1)
                          .reshape(lse.shape))
        loss = head_loss(rows, w, y, reduction, ignore_index).float()
        return loss.reshape(labels.shape if reduction == "none" else ())

    def head_logit_grad(self, x, weight, labels, lse, grad, v0, n, ignore_index, reduction):
        self.calls.append(("head_logit_grad", (v0, n)))
        w = weight.double()
        rows = x.double().reshape(-1, w.shape[1])
        want = torch.logsumexp(rows @ w.t(), 1) / math.log(2)
        kept = labels.reshape(-1) != ignore_index
        ref, s = lse.reshape(-1, 2).double().unbind(1)
        assert torch.allclose((ref + s.log2())[kept], want[kept], atol=1e-4)
        dz = head_dz(rows, w, labels.reshape(-1), grad.reshape(-1), v0, n, reduction, ignore_index)
        out = torch.zeros(len(rows), -(-n // 8) * 8, dtype=x.dtype)
        out[:, :n] = dz.to(x.dtype)
        return out.reshape(*labels.shape, -1)

    def rms_norm(self, x, residual, weight, eps):
        h = x if residual is None else x + residual
        y = norm_form(h.double(), weight.double(), eps).to(x.dtype)
        return [y] if residual is None else [y, h]

    def rms_norm_dot(self, h, grad, weight, eps, n_val, *, val_start=None, grad_scale=None):
        self.calls.append(("rms_norm_dot", tuple(h.shape)))
        B, F = h.shape[0], h.shape[-1]
        x = h.double()
        n = (grad.double() * x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)).reshape(B, -1, F).sum(1)
        vs = B - n_val if val_start is None else val_start
        val = torch.zeros(B, dtype=torch.bool)
        val[vs:vs + n_val] = True
        dw = None if grad_scale is None else (n[~val].sum(0) * grad_scale).to(weight.dtype)
        return [(n[~val] @ n[val].sum(0)).float(), dw]

    def adamw(self, params, states, bits, lr, beta1, beta2, eps, weight_decay, step, seed):
        self.calls.append(("adamw", (len(params), step)))
        for p, state in zip(params, states):
            n = p.numel()
            m, root = averages(state, p.shape, bits)
            new, m, v, root = adamw_form(f64(p).reshape(-1), f64(p.grad).reshape(-1), m, root, lr,
                                         (beta1, beta2), eps, weight_decay, step)
            p.copy_(new.reshape(p.shape).to(p.dtype))
            if bits == 32:
                state["exp_avg"].copy_(m.reshape(p.shape))
                state["exp_avg_sq"].copy_(v.reshape(p.shape))
                continue
            for name, x, u in zip(("exp_avg", "root_avg_sq"), (m, root), chances(n, step, seed)):
                scale = blocks_max(x) / TOP
                a = x.abs() / scale.clamp(min=1e-300).repeat_interleave(BLOCK)[:n]
                q = held(a.clamp(max=TOP), u).clamp(max=TOP)
                if name == "root_avg_sq":
                    q = torch.where(x > 0, q.clamp(min=2.0 ** -9), 0.0)
                state[name].copy_((q * x.sign()).float().to(torch.float8_e4m3fn).reshape(p.shape))
                state[name + "_scale"].copy_(scale)
