"""Three operators of a language model's training step, as cases that can be timed one by one.

- ``embed``: rows of an embedding table times a scale, and the table's gradient by tokens.
- ``qk``: each head's root-mean-square norm of the queries and keys, their rotation by position
  and the heads-first layout of queries, keys and values in one pass; its backward; and (``dots``)
  the gradient dot products and train gradients of the two norm weights under the engine.
- ``distill``: the loss against a teacher's top logits (and the labels), and its gradient.

``run`` computes them with elementary torch operations in 32 bits, or, with ``own``, through the
package.  ``exact`` forms the same results in float64 from the definitions.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------ the cases
def _embed(n, T, vocab, d, dtype, pass_, pad=0.0):
    """n rows of T tokens; pad: the share of tokens that are the padding id 0 (none: no
    padding id)."""
    return {"op": "embed", "n": n, "T": T, "vocab": vocab, "d": d, "dtype": dtype, "pass": pass_,
            "pad": pad}


def _qk(n, T, heads, kv_heads, d, rot, dtype, pass_, interleaved=False, span=0, n_val=0):
    """span: positions start anywhere below it, per row (0: at zero)."""
    return {"op": "qk", "n": n, "T": T, "heads": heads, "kv_heads": kv_heads, "d": d, "rot": rot,
            "dtype": dtype, "pass": pass_, "interleaved": interleaved, "span": span,
            "n_val": n_val}


def _distill(n, vocab, k, dtype, pass_, tau, alpha, reduction="mean", ignored=0.1):
    return {"op": "distill", "n": n, "vocab": vocab, "k": k, "dtype": dtype, "pass": pass_,
            "tau": tau, "alpha": alpha, "reduction": reduction, "ignored": ignored}


def listed():
    return [
        # the next token of eight sequences, looked up while a model answers
        {"name": "embed next tokens", **_embed(8, 1, 50257, 768, "bf16", "forward")},
        # a GPT-2-small training batch's token embedding
        {"name": "embed GPT-2 batch", **_embed(16, 1024, 50257, 768, "bf16", "train")},
        # a padded batch of short texts, features of an odd count, 32-bit weights
        {"name": "embed padded odd", **_embed(48, 509, 30011, 515, "fp32", "train", 0.7)},
        # the next token of eight sequences at their own positions, four queries to a key
        {"name": "qk next tokens", **_qk(8, 1, 16, 4, 128, 128, "bf16", "forward", span=32000)},
        # the attention prologue of a GPT-2-small step, heads of 64
        {"name": "qk GPT-2 batch", **_qk(20, 1024, 12, 12, 64, 64, "bf16", "train")},
        # Pythia-1B's heads: 256 wide, the first quarter rotated
        {"name": "qk Pythia heads", **_qk(8, 2048, 8, 8, 256, 64, "bf16", "train")},
        # odd everything: one key head, neighbouring features rotated together, 32 bits
        {"name": "qk one key odd", **_qk(5, 333, 7, 1, 80, 20, "fp32", "train", True, 32000)},
        # the layer under the engine: dots and train gradients of both norm weights
        {"name": "qk engine dots", **_qk(20, 512, 16, 4, 128, 128, "bf16", "dots", n_val=4)},
        # a few rows: a short answer scored against the teacher, GPT-2's vocabulary
        {"name": "distill few rows", **_distill(8, 50257, 20, "bf16", "train", 2.0, 1.0)},
        # a training batch: both losses, GPT-2's vocabulary, some labels ignored
        {"name": "distill GPT-2 batch", **_distill(8192, 50257, 64, "bf16", "train", 2.0, 0.5)},
        # 32-bit logits at temperature one, a ragged vocabulary and many teacher entries
        {"name": "distill fp32 ragged", **_distill(2031, 32003, 100, "fp32", "train", 1.0, 0.7)},
        # validation: each row's loss, no gradient (Pythia's vocabulary)
        {"name": "distill rows' losses", **_distill(1500, 50304, 8, "bf16", "forward", 1.5, 0.9,
                                                    "none")},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "qk", "qk", "distill"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "embed":
        n, T = _spread(rng, 1, 32), _spread(rng, 1, 1024)
        d = rng.choice([64 * rng.randint(2, 16), rng.randint(33, 1024)])
        return _embed(n, T, _spread(rng, 1000, 60000), d, dtype,
                      rng.choice(["forward", "train", "train"]), rng.choice([0.0, 0.5, 0.9]))
    if op == "qk":
        kv = rng.choice([1, 2, 4, 8])
        d = rng.choice([64, 128, 256, rng.randint(32, 192)])
        rot = 2 * rng.choice([d // 2, d // 8, rng.randint(1, d // 2)])
        n, T = _spread(rng, 2, 20), _spread(rng, 1, 1024)
        pass_ = rng.choice(["forward", "train", "train", "dots"])
        return _qk(n, T, kv * rng.choice([1, 2, 3]), kv, d, rot, dtype, pass_,
                   rng.random() < 0.3, rng.choice([0, 32000]),
                   rng.randint(1, n - 1) if pass_ == "dots" else 0)
    n, vocab = _spread(rng, 1, 4000), _spread(rng, 500, 60000)
    return _distill(n, vocab, _spread(rng, 1, 200), dtype, rng.choice(["forward", "train", "train"]),
                    rng.choice([1.0, 2.0, round(rng.uniform(0.5, 4.0), 2)]),
                    rng.choice([1.0, 0.5, round(rng.random(), 2)]),
                    rng.choice(["mean", "mean", "sum", "none"]), rng.choice([0.0, 0.3]))


def work(case):
    """Each input read once, each output written once."""
    c, e = SimpleNamespace(**case), {"bf16": 2, "fp32": 4}[case["dtype"]]
    train = case["pass"] == "train"
    if c.op == "embed":
        M = c.n * c.T
        rows, out, table = min(M, c.vocab) * c.d * e, M * c.d * e, c.vocab * c.d * e
        return {"bytes": 8 * M + rows + out + (out + table if train else 0),
                "flops": M * c.d * (2 if train else 1)}
    if c.op == "qk":
        size = c.n * c.T * (c.heads + 2 * c.kv_heads) * c.d
        passes = 2 if case["pass"] == "forward" else 4
        return {"bytes": passes * size * e + 8 * c.n * c.T,
                "flops": size * (8 if passes == 2 else 30)}
    size = c.n * c.vocab
    return {"bytes": (2 if train else 1) * size * e + 12 * c.n * c.k + 8 * c.n,
            "flops": size * (14 if train else 8)}


# -------------------------------------------------------------------------------- inputs
EPS = 1e-6
BASE = 10000.0


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _embed_inputs(c, seed):
    g, dt = _gen(seed), DTYPES[c.dtype]
    u = torch.rand(c.n, c.T, generator=g, device="cuda")
    ids = (u ** 3 * c.vocab).long().clamp_(max=c.vocab - 1)   # low ids are the frequent ones
    if c.pad:
        ids[torch.rand(c.n, c.T, generator=g, device="cuda") < c.pad] = 0
    weight = (_randn(g, c.vocab, c.d) * 0.02).to(dt)
    return SimpleNamespace(ids=ids, weight=weight, grad=_randn(g, c.n, c.T, c.d).to(dt),
                           scale=math.sqrt(c.d), padding=0 if c.pad else None)


def _qk_inputs(c, seed):
    g, dt = _gen(seed), DTYPES[c.dtype]
    H = c.heads + 2 * c.kv_heads
    s = SimpleNamespace(positions=None, n_pos=c.T + c.span)
    s.qkv = (_randn(g, c.n, c.T, H * c.d) * (0.5 + torch.rand(c.n, c.T, 1, generator=g,
                                                              device="cuda"))).to(dt)
    s.qw = (1 + 0.1 * _randn(g, c.d)).to(dt)
    s.kw = (1 + 0.1 * _randn(g, c.d)).to(dt)
    if c.span:
        start = torch.randint(0, c.span, (c.n, 1), generator=g, device="cuda")
        s.positions = start + torch.arange(c.T, device="cuda")
    s.grads = [_randn(g, c.n, h, c.T, c.d).to(dt) for h in (c.heads, c.kv_heads, c.kv_heads)]
    return s


def _distill_inputs(c, seed):
    g, dt = _gen(seed), DTYPES[c.dtype]
    # k different ids a row: a start and steps whose sum stays below the vocabulary
    step = torch.randint(1, max(2, c.vocab // c.k), (c.n, c.k), generator=g, device="cuda")
    k = min(c.k, c.vocab)
    ids = (torch.randint(0, c.vocab, (c.n, 1), generator=g, device="cuda") +
           step[:, :k].cumsum(1)) % c.vocab
    t = (3 * _randn(g, c.n, k)).sort(dim=1, descending=True).values
    z = _randn(g, c.n, c.vocab).mul_(2)
    z.scatter_add_(1, ids, 4 + t)
    # every 16th row has half its entries only, every 64th none (its text ended before)
    row = torch.arange(c.n, device="cuda")[:, None]
    col = torch.arange(k, device="cuda")[None]
    ids = torch.where(((row % 16 == 5) & (col >= (k + 1) // 2)) | (row % 64 == 9), -1, ids)
    labels = torch.randint(0, c.vocab, (c.n,), generator=g, device="cuda")
    labels[1:][torch.rand(c.n, generator=g, device="cuda")[1:] < c.ignored] = -100
    return SimpleNamespace(logits=z.to(dt), ids=ids, teacher=t.to(dt), labels=labels,
                           grad=torch.rand(c.n, generator=g, device="cuda"))


def _angles(positions, rot):
    """cos and sin of position * base^(-2 i / rot), [..., rot / 2] each, from float64 angles."""
    i = torch.arange(rot // 2, device=positions.device, dtype=torch.float64)
    a = positions[..., None].double() * torch.exp(-(2 * i / rot) * math.log(BASE))
    return a.cos(), a.sin()


def prepare(case, seed):
    c = SimpleNamespace(**case)
    if c.op == "embed":
        s = _embed_inputs(c, seed)
        if own and case["pass"] == "train":
            s.weight.requires_grad_()
    elif c.op == "qk":
        s = _qk_inputs(c, seed)
        # the angles of every position, kept by a model: [positions, 2, rot / 2]
        s.table = torch.stack(_angles(torch.arange(s.n_pos, device="cuda"), c.rot), 1).float()
        if own and case["pass"] == "train":
            for x in (s.qkv, s.qw, s.kw):
                x.requires_grad_()
        if own and case["pass"] == "dots":
            _prepare_engine(s, c)
    else:
        s = _distill_inputs(c, seed)
        if own and case["pass"] == "train":
            s.logits.requires_grad_()
    s.c, s.way = c, case["pass"]
    return s


def _prepare_engine(s, c):
    from ghostsuite_amd import GradDotProdEngine, QKNormRotary
    with torch.device("cuda"):
        s.layer = QKNormRotary(c.heads, c.kv_heads, c.d, n_rot=c.rot, n_positions=s.n_pos,
                               base=BASE, eps=EPS, interleaved=c.interleaved)
    s.layer.to(s.qkv.dtype)
    with torch.no_grad():
        s.layer.q_weight.copy_(s.qw)
        s.layer.k_weight.copy_(s.kw)
    s.engine = GradDotProdEngine(s.layer, val_batch_size=c.n_val, use_dummy_bias=True)
    s.engine.attach(torch.optim.SGD(s.layer.parameters(), lr=0.0))
    s.qkv.requires_grad_()


# ------------------------------------------------------------------- through the package
def _run_own(s):
    import ghostsuite_amd as gs
    c = s.c
    if c.op == "embed":
        y = gs.embedding_lookup(s.ids, s.weight, scale=s.scale, padding_idx=s.padding)
        if s.way == "forward":
            return y
        return y.detach(), torch.autograd.grad(y, s.weight, s.grad)[0]
    if c.op == "qk":
        if s.way == "dots":
            y = s.layer(s.qkv, s.positions)
            torch.autograd.backward(y, s.grads)
            out = [x.detach() for x in y] + [s.qkv.grad]
            for w in (s.layer.q_weight, s.layer.k_weight):
                out += [w.grad_dot_prod, w.train_grad]
                del w.grad_dot_prod, w.train_grad
            s.qkv.grad = None
            return out
        y = gs.qkv_norm_rotary(s.qkv, c.heads, c.kv_heads, s.table, s.positions, s.qw, s.kw,
                               eps=EPS, interleaved=c.interleaved)
        if s.way == "forward":
            return list(y)
        return [x.detach() for x in y] + list(torch.autograd.grad(y, (s.qkv, s.qw, s.kw),
                                                                  s.grads))
    loss = gs.distillation_loss(s.logits, s.ids, s.teacher, s.labels, temperature=c.tau,
                                alpha=c.alpha, reduction=c.reduction)
    if s.way == "forward":
        return loss
    up = s.grad if c.reduction == "none" else None
    return loss.detach(), torch.autograd.grad(loss, s.logits, up)[0]


# --------------------------------------------------------------------------- plain forms
def _embed_plain(s):
    c, dt = s.c, s.weight.dtype
    y = (s.weight[s.ids].float() * s.scale).to(dt)
    if s.way == "forward":
        return y
    g = s.grad.float()
    if s.padding is not None:
        g = g * (s.ids != s.padding)[..., None]
    dw = torch.zeros(c.vocab, c.d, device="cuda").index_add_(0, s.ids.reshape(-1),
                                                             g.reshape(-1, c.d))
    return y, (dw * s.scale).to(dt)


def _pairs(x, c):
    """The two features of each rotated pair, and the features that are not rotated."""
    r = x[..., :c.rot]
    if c.interleaved:
        return r[..., 0::2], r[..., 1::2], x[..., c.rot:]
    return r[..., :c.rot // 2], r[..., c.rot // 2:], x[..., c.rot:]


def _joined(a, b, rest, c):
    r = torch.stack((a, b), -1).flatten(-2) if c.interleaved else torch.cat((a, b), -1)
    return torch.cat((r, rest), -1)


def _rotate(x, cos, sin, c):
    a, b, rest = _pairs(x, c)
    return _joined(a * cos - b * sin, b * cos + a * sin, rest, c)


def _qk_plain(s):
    c, dt = s.c, s.qkv.dtype
    x = s.qkv.float().reshape(c.n, c.T, -1, c.d)
    parts = x.split([c.heads, c.kv_heads, c.kv_heads], dim=2)
    at = s.table[torch.arange(c.T, device="cuda") if s.positions is None else s.positions]
    cos, sin = at[..., 0, :].unsqueeze(-2), at[..., 1, :].unsqueeze(-2)
    out, dx, dw = [], [], []
    for k, (u, w) in enumerate(zip(parts, (s.qw, s.kw, None))):
        g = None if s.way == "forward" else s.grads[k].float().transpose(1, 2)
        if w is None:
            out.append(u)
            dx.append(g)
            continue
        w = w.float()
        r = torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS)
        xn = u * r
        out.append(_rotate(xn * w, cos, sin, c))
        if g is not None:
            h = _rotate(g, cos, -sin, c)
            dw.append((h * xn).sum((1, 2)))                  # of each row
            h = h * w
            dx.append(r * (h - xn * (h * xn).mean(-1, keepdim=True)))
    y = [o.transpose(1, 2).contiguous().to(dt) for o in out]
    if s.way == "forward":
        return y
    dqkv = torch.cat(dx, 2).reshape(c.n, c.T, -1).to(dt)
    if s.way == "train":
        return y + [dqkv] + [w.sum(0).to(dt) for w in dw]
    n_t = c.n - c.n_val
    y.append(dqkv)
    for w in dw:
        y += [w[:n_t] @ w[n_t:].sum(0), (w[:n_t].sum(0) * (c.n / n_t)).to(dt)]
    return y


def _distill_plain(s):
    c = s.c
    z = s.logits.float()
    use = s.ids >= 0
    at = s.ids.clamp(min=0)
    t = torch.where(use, s.teacher.float() / c.tau, float("-inf"))
    top = t.max(1, keepdim=True).values
    top = torch.where(torch.isinf(top), 0.0, top)
    e = torch.exp(t - top)
    total = e.sum(1, keepdim=True)
    some = total > 0
    total = torch.where(some, total, 1.0)
    p = e / total
    log_p = torch.where(use, t - top, 0.0) - torch.log(total)
    m = z.max(1, keepdim=True).values
    keep = s.labels >= 0
    y = s.labels.clamp(min=0)[:, None]

    def row_softmax(tau):
        ez = torch.exp((z - m) / tau)
        n = ez.sum(1, keepdim=True)
        return ez, n

    ez, n = row_softmax(c.tau)
    log_q = (z.gather(1, at) - m) / c.tau - torch.log(n)
    kl = (p * (log_p - log_q)).sum(1)
    loss = c.alpha * c.tau ** 2 * kl
    if c.alpha != 1.0:
        e1, n1 = row_softmax(1.0)
        loss = loss + (1 - c.alpha) * (m + torch.log(n1) - z.gather(1, y))[:, 0]
    loss = torch.where(keep, loss, 0.0)
    w = keep.float()
    if c.reduction == "mean":
        w = w / keep.sum()
        value = loss.sum() / keep.sum()
    else:
        value = loss.sum() if c.reduction == "sum" else loss
    if s.way == "forward":
        return value
    if c.reduction == "none":
        w = w * s.grad
    dz = (c.alpha * c.tau) * (ez / n) * some
    dz.scatter_add_(1, at, -c.alpha * c.tau * p)
    if c.alpha != 1.0:
        dz += (1 - c.alpha) * (e1 / n1)
        dz.scatter_add_(1, y, torch.full_like(y, c.alpha - 1, dtype=torch.float32))
    return value, (dz * w[:, None]).to(s.logits.dtype)


def run(state):
    if own:
        return _run_own(state)
    return {"embed": _embed_plain, "qk": _qk_plain, "distill": _distill_plain}[state.c.op](state)


# -------------------------------------------------------------------------- float64 forms
def _embed_exact(c, way, s):
    y = torch.nn.functional.embedding(s.ids, s.weight.double()) * s.scale
    if way == "forward":
        return y
    # tokens in the order of their ids, each id's rows by the differences of the running sums
    ids, order = s.ids.reshape(-1).sort(stable=True)
    rows = s.grad.reshape(-1, c.d).double()[order]
    if s.padding is not None:
        rows[ids == s.padding] = 0.0
    sums = torch.cat((rows.new_zeros(1, c.d), rows.cumsum(0)))
    v = torch.arange(c.vocab, device="cuda")
    return y, (sums[torch.searchsorted(ids, v, right=True)] -
               sums[torch.searchsorted(ids, v)]) * s.scale


def _qk_exact(c, way, s):
    """Forward in float64; the gradients by automatic differentiation, a row's weights apart
    from the others' for the dots."""
    qkv = s.qkv.double().requires_grad_()
    qw, kw = (w.double().expand(c.n, c.d).clone().requires_grad_() for w in (s.qw, s.kw))
    pos = torch.arange(c.T, device="cuda").expand(c.n, c.T) if s.positions is None else s.positions
    i = torch.arange(c.rot // 2, device="cuda", dtype=torch.float64)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       pos.double()[..., None] * BASE ** (-2 * i / c.rot))[:, None]
    x = qkv.view(c.n, c.T, -1, c.d).transpose(1, 2)
    out = []
    for u, w in zip(x.split([c.heads, c.kv_heads, c.kv_heads], 1), (qw, kw, None)):
        if w is not None:
            u = u / (u.square().mean(-1, keepdim=True) + EPS).sqrt() * w[:, None, None]
            r, rest = u[..., :c.rot], u[..., c.rot:]
            shape = (c.rot // 2, 2) if c.interleaved else (2, c.rot // 2)
            dim = -1 if c.interleaved else -2
            a, b = r.unflatten(-1, shape).unbind(dim)
            z = torch.complex(a, b) * turn
            u = torch.cat((torch.stack((z.real, z.imag), dim).flatten(-2), rest), -1)
        out.append(u)
    if way == "forward":
        return [o.detach() for o in out]
    dx, dq, dk = torch.autograd.grad(out, (qkv, qw, kw), [g.double() for g in s.grads])
    out = [o.detach() for o in out] + [dx]
    if way == "train":
        return out + [dq.sum(0), dk.sum(0)]
    n_t = c.n - c.n_val
    for w in (dq, dk):
        out += [(w[:n_t] * w[n_t:].sum(0)).sum(1), w[:n_t].sum(0) * (c.n / n_t)]
    return out


def _distill_exact(c, way, s):
    keep = s.labels != -100
    count = int(keep.sum())
    losses, grads = [], []
    for r in range(0, c.n, 512):                    # some rows at a time: float64 logits are wide
        part = slice(r, r + 512)
        z = s.logits[part].double().requires_grad_(way == "train")
        use = s.ids[part] >= 0
        t = (s.teacher[part].double() / c.tau).masked_fill(~use, -1e300)
        p = torch.softmax(t, 1).masked_fill(~use, 0.0)
        log_q = torch.log_softmax(z / c.tau, 1).gather(1, s.ids[part].clamp(min=0))
        row = c.alpha * c.tau ** 2 * (torch.special.xlogy(p, p) - p * log_q).sum(1)
        row = row + (1 - c.alpha) * torch.nn.functional.cross_entropy(
            z, s.labels[part].clamp(min=0), reduction="none")
        row = torch.where(keep[part], row, 0.0)
        losses.append(row.detach())
        if way == "train":
            w = s.grad[part].double() if c.reduction == "none" else \
                torch.full_like(row, 1.0 / count if c.reduction == "mean" else 1.0)
            grads.append(torch.autograd.grad(row, z, w)[0])
    loss = torch.cat(losses)
    if c.reduction != "none":
        loss = loss.sum() / (count if c.reduction == "mean" else 1)
    return (loss, torch.cat(grads)) if way == "train" else loss


def exact(case, seed):
    c = SimpleNamespace(**case)
    s = {"embed": _embed_inputs, "qk": _qk_inputs, "distill": _distill_inputs}[c.op](c, seed)
    form = {"embed": _embed_exact, "qk": _qk_exact, "distill": _distill_exact}[c.op]
    return form(c, case["pass"], s)
