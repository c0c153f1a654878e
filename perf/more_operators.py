"""Three more operators of a language model's training step, as cases that can be timed one by one.

- ``head``: the output projection with its softmax cross entropy, in pieces of the vocabulary, and
  the gradients of the hidden rows and of the projection's weight.
- ``norm``: the root-mean-square norm of a residual stream, with the residual's addition; its
  backward; and (``dots``) the gradient dot products and train gradients of the norm's weight under
  the engine.
- ``adamw``: one step of AdamW over all tensors of a model, its averages held in 32 or in 8 bits.

``run`` computes them with elementary torch operations in 32 bits, or, with ``own``, through the
package.  ``exact`` forms the same results in float64 from the definitions.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp32": 4}


# ------------------------------------------------------------------------------ the cases
def _head(n, vocab, d, dtype, pass_, reduction="mean", ignored=0.1):
    """n hidden rows; ignored: the share of them without a label."""
    return {"op": "head", "n": n, "vocab": vocab, "d": d, "dtype": dtype, "pass": pass_,
            "reduction": reduction, "ignored": ignored}


def _norm(n, T, d, dtype, pass_, residual=True, n_val=0):
    return {"op": "norm", "n": n, "T": T, "d": d, "dtype": dtype, "pass": pass_,
            "residual": residual, "n_val": n_val}


def _adamw(kind, layers, d, vocab, dtype, bits):
    """kind: the tensors of an 'lm' or an 'mlp', or 'odd' ones (``_shapes``)."""
    return {"op": "adamw", "kind": kind, "layers": layers, "d": d, "vocab": vocab, "dtype": dtype,
            "bits": bits}


def listed():
    return [
        # a short answer's eight tokens, GPT-2's vocabulary
        {"name": "head few tokens", **_head(8, 50257, 768, "bf16", "train")},
        # a GPT-2-small training batch with its validation rows
        {"name": "head GPT-2 batch", **_head(20480, 50257, 768, "bf16", "train")},
        # 32 bits, an odd width and vocabulary, a batch that is half padding
        {"name": "head fp32 ragged", **_head(2031, 32003, 515, "fp32", "train", "none", 0.5)},
        # validation: each token's loss, no gradient, Pythia's vocabulary and width
        {"name": "head rows' losses", **_head(4096, 50304, 2048, "bf16", "forward", "none", 0.0)},
        # the next token of eight sequences
        {"name": "norm next tokens", **_norm(8, 1, 768, "bf16", "forward")},
        # a block's norm in a Pythia-1B step
        {"name": "norm Pythia batch", **_norm(8, 2048, 2048, "bf16", "train")},
        # 32 bits, rows off 16-byte boundaries, no residual
        {"name": "norm fp32 odd", **_norm(7, 333, 1023, "fp32", "train", False)},
        # the layer under the engine: dots and train gradient of its weight, GPT-2-medium's width
        {"name": "norm engine dots", **_norm(20, 512, 1024, "bf16", "dots", True, 4)},
        # the MLP of the smallest configuration: what a step costs when the tensors are small
        {"name": "adamw MLP", **_adamw("mlp", 2, 1024, 10, "fp32", 32)},
        # GPT-2-small in bf16, averages in 32 bits
        {"name": "adamw GPT-2", **_adamw("lm", 12, 768, 50257, "bf16", 32)},
        # the same with averages in 8 bits
        {"name": "adamw GPT-2 8 bits", **_adamw("lm", 12, 768, 50257, "bf16", 8)},
        # many tensors of odd sizes, 32-bit weights, averages in 8 bits
        {"name": "adamw odd 8 bits", **_adamw("odd", 97, 200003, 0, "fp32", 8)},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["head", "head", "norm", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "head":
        d = rng.choice([64 * rng.randint(1, 16), rng.randint(33, 1024)])
        n = _spread(rng, 1, 8000 if dtype == "bf16" else 2000)
        return _head(n, _spread(rng, 500, 60000), d, dtype, rng.choice(["forward", "train", "train"]),
                     rng.choice(["mean", "mean", "sum", "none"]), rng.choice([0.0, 0.3, 0.7]))
    if op == "norm":
        n, T = _spread(rng, 2, 20), _spread(rng, 1, 1024)
        d = rng.choice([64 * rng.randint(1, 32), rng.randint(17, 2500)])
        pass_ = rng.choice(["forward", "train", "train", "dots"])
        return _norm(n, T, d, dtype, pass_, rng.random() < 0.7,
                     rng.randint(1, n - 1) if pass_ == "dots" else 0)
    bits = rng.choice([8, 32])
    if rng.random() < 0.5:
        return _adamw("odd", rng.randint(1, 200), _spread(rng, 5, 300000), 0, dtype, bits)
    return _adamw("lm", rng.randint(1, 8), 8 * rng.randint(8, 96), _spread(rng, 500, 40000), dtype,
                  bits)


def _shapes(c):
    d = c.d
    if c.kind == "odd":
        return [(1 + 7919 * (i + 1) * (i + 3) % d,) for i in range(c.layers)]
    if c.kind == "mlp":
        dims = [d // 2] + [d] * c.layers + [c.vocab]
        return [s for i in range(len(dims) - 1) for s in ((dims[i + 1], dims[i]), (dims[i + 1],))]
    block = [(d,), (d,), (3 * d, d), (3 * d,), (d, d), (d,), (d,), (d,), (4 * d, d), (4 * d,),
             (d, 4 * d), (d,)]
    return [(c.vocab, d), (1024, d)] + block * c.layers + [(d,), (d,)]


def work(case):
    """Each input read once, each output written once."""
    c, e = SimpleNamespace(**case), BYTES[case["dtype"]]
    train = case["pass"] == "train" if "pass" in case else False
    if c.op == "head":
        x, w = c.n * c.d * e, c.vocab * c.d * e
        kept = max(1, round(c.n * (1 - c.ignored)))
        return {"bytes": (2 if train else 1) * (x + w) + 8 * c.n,
                "flops": (3 if train else 1) * 2 * kept * c.vocab * c.d}
    if c.op == "norm":
        size = c.n * c.T * c.d
        parts = 2 + 2 * c.residual                   # in, and out
        if case["pass"] != "forward":
            parts += 2 + c.residual                  # output gradients in, input gradient out
        return {"bytes": parts * size * e + c.d * e, "flops": size * (4 if parts < 5 else 14)}
    n = sum(math.prod(s) for s in _shapes(c))
    state = 8 if c.bits == 32 else 2 + 8 / 256
    return {"bytes": n * (3 * e + 2 * state), "flops": 16 * n}


# -------------------------------------------------------------------------------- inputs
EPS = 1e-6
LR, BETA1, BETA2, ADAM_EPS, DECAY = 3e-4, 0.9, 0.95, 1e-8, 0.1
STEPS, SEED = 41, 7          # the steps taken before; the seed of the 8-bit averages' rounding
BLOCK, TOP = 256, 448.0      # elements that share a scale; the largest 8-bit value


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _head_inputs(c, seed):
    g, dt = _gen(seed), DTYPES[c.dtype]
    w = _randn(g, c.vocab, c.d) * (2.0 / math.sqrt(c.d))
    labels = torch.randint(0, c.vocab, (c.n,), generator=g, device="cuda")
    # hidden rows that lean towards their label's row, some more than others
    lean = 4 * torch.rand(c.n, 1, generator=g, device="cuda")
    x = _randn(g, c.n, c.d) + lean * w[labels]
    labels[1:][torch.rand(c.n, generator=g, device="cuda")[1:] < c.ignored] = -100
    return SimpleNamespace(x=x.to(dt), w=w.to(dt), labels=labels,
                           grad=torch.rand(c.n, generator=g, device="cuda"))


def _norm_inputs(c, seed):
    g, dt = _gen(seed), DTYPES[c.dtype]
    shape = (c.n, c.T, c.d)
    size = 0.5 + torch.rand(c.n, c.T, 1, generator=g, device="cuda")
    s = SimpleNamespace(residual=None, grads=[_randn(g, *shape).to(dt)])
    s.x = (_randn(g, *shape) * size).to(dt)
    s.w = (1 + 0.1 * _randn(g, c.d)).to(dt)
    if c.residual:
        s.residual = (2 * _randn(g, *shape)).to(dt)
        s.grads.append(_randn(g, *shape).to(dt))
    return s


def _adamw_inputs(c, seed):
    """Every tensor in one array, each from a multiple of 256 elements on; zeros in between."""
    g, dt = _gen(seed), DTYPES[c.dtype]
    s = SimpleNamespace(shapes=_shapes(c), steps=STEPS)
    sizes = [math.prod(x) for x in s.shapes]
    blocks = [-(-n // BLOCK) for n in sizes]
    s.at = (BLOCK * torch.tensor([0] + blocks[:-1]).cumsum(0)).tolist()
    total = BLOCK * sum(blocks)
    # of each block: its place in its own tensor, and how many of its elements are the tensor's
    count, ends = torch.tensor(blocks), torch.tensor(sizes)
    place = torch.arange(sum(blocks)) - (count.cumsum(0) - count).repeat_interleave(count)
    live = (ends.repeat_interleave(count) - BLOCK * place).clamp(max=BLOCK).cuda()[:, None]
    s.index = (BLOCK * place).cuda()[:, None] + torch.arange(BLOCK, device="cuda")
    mask = torch.arange(BLOCK, device="cuda") < live
    # gradients whose size differs from block to block, and averages that they may have left
    size = torch.exp(2 * _randn(g, sum(blocks), 1)) * 1e-4
    s.p = (_randn(g, sum(blocks), BLOCK) * 0.02 * mask).reshape(total).to(dt)
    s.g = (_randn(g, sum(blocks), BLOCK) * size * mask).reshape(total).to(dt)
    m = _randn(g, sum(blocks), BLOCK) * size * 0.3 * mask
    r = (0.3 + torch.rand(sum(blocks), BLOCK, generator=g, device="cuda")) * size * mask
    if c.bits == 32:
        s.m, s.v = m.reshape(total), (r * r).reshape(total)
    else:
        s.m_scale, s.r_scale = m.abs().amax(1) / TOP, r.amax(1) / TOP
        s.m, s.r = ((x / y[:, None].clamp(min=1e-38)).to(torch.float8_e4m3fn).reshape(total)
                    for x, y in ((m, s.m_scale), (r, s.r_scale)))
    return s


def _prepare_adamw(s, c):
    from ghostsuite_amd import AdamW
    params = []
    for at, shape in zip(s.at, s.shapes):
        n = math.prod(shape)
        p = torch.nn.Parameter(s.p[at:at + n].view(shape))
        p.grad = s.g[at:at + n].view(shape)
        params.append(p)
    s.opt = AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=DECAY,
                  state_bits=c.bits, seed=SEED)
    for p, at, shape in zip(params, s.at, s.shapes):
        n, b, k = math.prod(shape), at // BLOCK, -(-math.prod(shape) // BLOCK)
        state = {"step": s.steps, "exp_avg": s.m[at:at + n].view(shape)}
        if c.bits == 32:
            state["exp_avg_sq"] = s.v[at:at + n].view(shape)
        else:
            state["exp_avg_scale"] = s.m_scale[b:b + k]
            state["root_avg_sq"] = s.r[at:at + n].view(shape)
            state["root_avg_sq_scale"] = s.r_scale[b:b + k]
        s.opt.state[p] = state


def _prepare_engine(s, c):
    from ghostsuite_amd import GradDotProdEngine, RMSNorm
    with torch.device("cuda"):
        s.layer = RMSNorm(c.d, eps=EPS)
    s.layer.to(s.x.dtype)
    with torch.no_grad():
        s.layer.weight.copy_(s.w)
    s.engine = GradDotProdEngine(s.layer, val_batch_size=c.n_val, use_dummy_bias=True)
    s.engine.attach(torch.optim.SGD(s.layer.parameters(), lr=0.0))


def prepare(case, seed):
    c = SimpleNamespace(**case)
    if c.op == "head":
        s = _head_inputs(c, seed)
        leaves = (s.x, s.w)
    elif c.op == "norm":
        s = _norm_inputs(c, seed)
        leaves = [t for t in (s.x, s.residual, s.w) if t is not None]
        if own and case["pass"] == "dots":
            _prepare_engine(s, c)
            leaves = leaves[:-1]
    else:
        s = _adamw_inputs(c, seed)
        leaves = ()
        if own:
            _prepare_adamw(s, c)
    s.c, s.way = c, case.get("pass", "step")
    if own and s.way != "forward":
        for t in leaves:
            t.requires_grad_()
    return s


# ------------------------------------------------------------------- through the package
def _run_own(s):
    import ghostsuite_amd as gs
    c = s.c
    if c.op == "head":
        loss = gs.head_cross_entropy(s.x, s.w, s.labels, reduction=c.reduction)
        if s.way == "forward":
            return loss
        up = s.grad if c.reduction == "none" else None
        return [loss.detach(), *torch.autograd.grad(loss, (s.x, s.w), up)]
    if c.op == "norm":
        if s.way == "dots":
            y = s.layer(s.x, s.residual) if c.residual else (s.layer(s.x),)
            torch.autograd.backward(y, s.grads)
            w = s.layer.weight
            out = [t.detach() for t in y] + [s.x.grad, w.grad_dot_prod, w.train_grad]
            del w.grad_dot_prod, w.train_grad
            s.x.grad = None
            if c.residual:
                s.residual.grad = None
            return out
        y = gs.add_rms_norm(s.x, s.residual, s.w, eps=EPS) if c.residual else \
            (gs.rms_norm(s.x, s.w, eps=EPS),)
        if s.way == "forward":
            return list(y)
        return [t.detach() for t in y] + list(torch.autograd.grad(y, (s.x, s.w), s.grads))
    s.opt.step()
    return _adamw_outputs(s)


def _adamw_outputs(s):
    if s.c.bits == 32:
        return [s.p, s.m, s.v]
    return [s.p, s.m, s.m_scale, s.r, s.r_scale]


# --------------------------------------------------------------------------- plain forms
def _head_plain(s):
    c = s.c
    x, w = s.x.float(), s.w.float()
    z = x @ w.t()
    keep = s.labels >= 0
    y = s.labels.clamp(min=0)[:, None]
    top = z.max(1, keepdim=True).values
    label = z.gather(1, y)
    e = z.sub_(top).exp_()
    total = e.sum(1, keepdim=True)
    loss = torch.where(keep, (top + torch.log(total) - label)[:, 0], 0.0)
    weight = keep.float()
    value = loss
    if c.reduction == "mean":
        weight = weight / keep.sum()
        value = loss.sum() / keep.sum()
    elif c.reduction == "sum":
        value = loss.sum()
    if s.way == "forward":
        return value
    if c.reduction == "none":
        weight = weight * s.grad
    dz = e.mul_((weight / total[:, 0])[:, None])
    dz.scatter_add_(1, y, -weight[:, None])
    return [value, (dz @ w).to(s.x.dtype), (dz.t() @ x).to(s.w.dtype)]


def _norm_plain(s):
    c, dt = s.c, s.x.dtype
    h = s.x if s.residual is None else (s.x.float() + s.residual.float()).to(dt)
    u, w = h.float(), s.w.float()
    r = torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS)
    xn = u * r
    out = [(xn * w).to(dt)] + ([h] if c.residual else [])
    if s.way == "forward":
        return out
    g = s.grads[0].float()
    gw = g * w
    dx = r * (gw - xn * (gw * xn).mean(-1, keepdim=True))
    if c.residual:
        dx = dx + s.grads[1].float()
    out.append(dx.to(dt))
    dw = (g * xn).sum(1)                             # of each row
    if s.way == "train":
        return out + [dw.sum(0).to(dt)]
    n_t = c.n - c.n_val
    return out + [dw[:n_t] @ dw[n_t:].sum(0), (dw[:n_t].sum(0) * (c.n / n_t)).to(dt)]


def _dither(index, step):
    """Two numbers of [0, 1) for each element, from its place in its tensor, the step and the seed."""
    key = (step * 0x9E3779B9 + SEED * 0x6A09E667) & 0xFFFFFFFF
    x = ((index + key) & 0xFFFFFFFF) * 0x9E3779B9 & 0xFFFFFFFF
    x = (x ^ x >> 15) * 0xBB67AE85 & 0xFFFFFFFF
    x = x ^ x >> 13
    return ((x & 0xFFFF) + 0.5) * 2.0 ** -16, ((x >> 16) + 0.5) * 2.0 ** -16


def _eighth(a, u):
    """a of [0, 448] on the grid of the 8-bit values, up or down by u."""
    exponent = torch.frexp(a).exponent.clamp(min=-5) - 4
    return torch.ldexp(torch.floor(torch.ldexp(a, -exponent) + u), exponent).clamp(max=TOP)


def _adamw_plain(s):
    c = s.c
    s.steps += 1
    p, g = s.p.float(), s.g.float()
    wide = (-1, BLOCK)
    if c.bits == 32:
        m, v = s.m, s.v
    else:
        m = (s.m.float().view(wide) * s.m_scale[:, None]).view(-1)
        v = (s.r.float().view(wide) * s.r_scale[:, None]).view(-1).square()
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + g * g * (1 - BETA2)
    root = v.sqrt()
    step = LR / (1 - BETA1 ** s.steps)
    p = p * (1 - LR * DECAY) - step * m / (root / math.sqrt(1 - BETA2 ** s.steps) + ADAM_EPS)
    s.p.copy_(p)
    if c.bits == 32:
        s.m.copy_(m)
        s.v.copy_(v)
        return _adamw_outputs(s)
    m, root = m.view(wide), root.view(wide)
    um, ur = _dither(s.index, s.steps)
    top_m, top_r = m.abs().amax(1, keepdim=True), root.amax(1, keepdim=True)
    some_m, some_r = (torch.where(t > 0, t, 1.0) for t in (top_m, top_r))
    q = torch.copysign(_eighth(m.abs() * (TOP / some_m), um), m)
    s.m.copy_(q.view(-1).to(torch.float8_e4m3fn))
    s.r.copy_(_eighth(root * (TOP / some_r), ur).view(-1).to(torch.float8_e4m3fn))
    s.m_scale.copy_(top_m[:, 0] / TOP)
    s.r_scale.copy_(top_r[:, 0] / TOP)
    return _adamw_outputs(s)


def run(state):
    if own:
        return _run_own(state)
    return {"head": _head_plain, "norm": _norm_plain, "adamw": _adamw_plain}[state.c.op](state)


# -------------------------------------------------------------------------- float64 forms
def _head_exact(c, way, s):
    keep = s.labels != -100
    w = s.w.double()
    count = int(keep.sum())
    losses, dx, dw = [], [], torch.zeros_like(w)
    for r in range(0, c.n, 1024):                    # some rows at a time: float64 logits are wide
        part = slice(r, r + 1024)
        x, labels = s.x[part].double(), s.labels[part].clamp(min=0)
        log_p = torch.log_softmax(x @ w.t(), 1)
        losses.append(torch.where(keep[part], -log_p.gather(1, labels[:, None])[:, 0], 0.0))
        if way == "forward":
            continue
        up = s.grad[part].double() if c.reduction == "none" else \
            torch.full_like(losses[-1], 1.0 / count if c.reduction == "mean" else 1.0)
        dz = log_p.exp_() - torch.nn.functional.one_hot(labels, c.vocab)
        dz *= torch.where(keep[part], up, 0.0)[:, None]
        dx.append(dz @ w)
        dw += dz.t() @ x
    loss = torch.cat(losses)
    if c.reduction != "none":
        loss = loss.sum() / (count if c.reduction == "mean" else 1)
    return loss if way == "forward" else [loss, torch.cat(dx), dw]


def _norm_exact(c, way, s):
    """Forward in float64; the gradients by automatic differentiation, a row's weight apart from the
    others' for the dots."""
    w = s.w.double().expand(c.n, c.d).clone().requires_grad_()
    h = s.x.double()
    if c.residual:                                   # as the stream holds it
        h = (h + s.residual.double()).to(s.x.dtype).double()
    h.requires_grad_()
    y = h / (h.square().mean(-1, keepdim=True) + EPS).sqrt() * w[:, None]
    out = [y.detach()] + ([h.detach()] if c.residual else [])
    if way == "forward":
        return out
    dx, dw = torch.autograd.grad(y, (h, w), s.grads[0].double())
    out.append(dx + s.grads[1].double() if c.residual else dx)
    if way == "train":
        return out + [dw.sum(0)]
    n_t = c.n - c.n_val
    return out + [(dw[:n_t] * dw[n_t:].sum(0)).sum(1), dw[:n_t].sum(0) * (c.n / n_t)]


def _adamw_exact(c, s):
    t = s.steps + 1
    p, g = s.p.double(), s.g.double()
    if c.bits == 32:
        m, v = s.m.double(), s.v.double()
    else:
        m, r = ((q.double().view(-1, BLOCK) * k.double()[:, None]).view(-1)
                for q, k in ((s.m, s.m_scale), (s.r, s.r_scale)))
        v = r ** 2
    m = torch.lerp(g, m, BETA1)
    v = torch.lerp(g ** 2, v, BETA2)
    m_hat, v_hat = m / (1 - BETA1 ** t), v / (1 - BETA2 ** t)
    p = p - LR * (m_hat / (v_hat.sqrt() + ADAM_EPS) + DECAY * p)
    if c.bits == 32:
        return [p, m, v]
    out = [p]
    for x, u in zip((m, v.sqrt()), _dither(s.index, t)):
        x = x.view(-1, BLOCK)
        scale = x.abs().amax(1) / TOP
        a = (x.abs() / scale.clamp(min=1e-300)[:, None]).clamp(max=TOP)
        # the grid's steps: 2^-9 below 2^-6, then an eighth of each power of two
        step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
        out += [(torch.sign(x) * (torch.floor(a / step + u) * step).clamp(max=TOP)).view(-1), scale]
    return out


def exact(case, seed):
    c = SimpleNamespace(**case)
    if c.op == "adamw":
        return _adamw_exact(c, _adamw_inputs(c, seed))
    inputs, form = {"head": (_head_inputs, _head_exact), "norm": (_norm_inputs, _norm_exact)}[c.op]
    return form(c, case["pass"], inputs(c, seed))
