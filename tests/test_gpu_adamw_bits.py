"""AdamW's averages in 8 bits on the GPU, bit for bit, against its arithmetic written out in elementary fp32
operations on the CPU, over several steps of each side's own state."""
import math

import pytest
import torch
from torch import nn

from ghostsuite_amd import AdamW
from tests.helpers import gen, randn
from tests.train_forms import BLOCK, TOP, chances

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


def blocks(x):
    return torch.cat((x, torch.zeros(-x.numel() % BLOCK))).view(-1, BLOCK)


def held(a, u):
    """floor(a / step + u) step, the sum rounded to fp32; step: the 8-bit values' distance at a."""
    exponent = torch.frexp(a).exponent.clamp(min=-5) - 4
    return torch.ldexp(torch.floor(torch.ldexp(a, -exponent) + u), exponent).clamp(max=TOP)


class Elementary:
    """One parameter's steps; every product, sum, root and quotient rounded to fp32 by itself."""

    def __init__(self, p):
        n = p.numel()
        self.p, self.t = p.clone(), 0
        self.m = self.r = torch.zeros(n)                                  # the 8-bit values
        self.m_scale = self.r_scale = torch.zeros(-(-n // BLOCK))

    def step(self, g, lr, betas, eps, decay, seed):
        f = lambda x: torch.tensor(x, dtype=torch.float32)   # noqa: E731
        n, (b1, b2) = g.numel(), betas
        self.t += 1
        p, g = self.p.float(), g.float()
        m = f(b1) * (blocks(self.m) * self.m_scale[:, None]).view(-1)[:n] + f(1 - b1) * g
        old = (blocks(self.r) * self.r_scale[:, None]).view(-1)[:n]
        # (torch's own fp32 root on the CPU is a unit off now and then; of a float64 root, rounded, no bit is)
        root = (f(b2) * (old * old) + f(1 - b2) * (g * g)).double().sqrt().float()
        den = root * f(1 / math.sqrt(1 - b2 ** self.t)) + f(eps)
        p = f(1 - lr * decay) * p - f(lr / (1 - b1 ** self.t)) * m / den
        self.p = p.to(self.p.dtype)
        out = []
        for x, u in zip((m, root), chances(n, self.t, seed)):
            top = blocks(x).abs().amax(1)
            top = torch.where(top >= 2.0 ** -100, top, 0.0)
            share = torch.where(top > 0, torch.ones(()) / top * f(TOP), f(0.0))
            a = (blocks(x).abs() * share[:, None]).view(-1)[:n]
            out += [held(a, u.float()), top * (f(1.0) / f(TOP))]
        q, self.m_scale, r, self.r_scale = out
        self.m = torch.copysign(q, m)
        some = self.r_scale.repeat_interleave(BLOCK)[:n] > 0
        self.r = torch.where((root > 0) & some, r.clamp(min=2.0 ** -9), 0.0)

    def same_as(self, p, state):
        for name, mine, theirs in (("p", self.p, p), ("m", self.m, state["exp_avg"]),
                                   ("m's scales", self.m_scale, state["exp_avg_scale"]),
                                   ("root", self.r, state["root_avg_sq"]),
                                   ("root's scales", self.r_scale, state["root_avg_sq_scale"])):
            mine, theirs = mine.float(), theirs.detach().cpu().float().reshape(-1)
            bad = ((mine != theirs) & ~(mine.isnan() & theirs.isnan())).nonzero().reshape(-1)
            assert bad.numel() == 0, (f"{name} after step {self.t}: {bad.numel()} of {mine.numel()}, the first at "
                                      f"{bad[0].item()}: {theirs[bad[0]].item()} for {mine[bad[0]].item()}")


def gradients(n, seed, spread):
    """Blocks of different sizes; with `spread`, of elements down to 10^-7 of their block's largest too."""
    size = torch.exp(2 * randn((-(-n // BLOCK),), seed, 1.0)) * 1e-4
    g = randn((n,), seed + 1, 1.0) * size.repeat_interleave(BLOCK)[:n]
    if spread:
        g = g * torch.pow(10.0, -7 * torch.rand(n, generator=gen(seed + 2)) ** 2)
    return g


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("betas,spread", [((0.9, 0.999), False), ((0.9, 0.999), True), ((0.5, 0.95), True)])
def test_steps_are_the_elementary_ones(gpu, dtype, betas, spread):
    """Some ten of ten steps' ten million chances lie within a unit of their line, so a single product that is
    not rounded where it is stated shows."""
    sizes = (1 << 20, 65537, 255, 1)
    start = [randn((n,), n, 0.02, dtype) for n in sizes]
    params = [nn.Parameter(p.to(gpu)) for p in start]
    plain = [Elementary(p) for p in start]
    opt = AdamW(params, lr=1e-3, betas=betas, weight_decay=0.1, state_bits=8, seed=5)
    for step in range(10):
        for k, p in enumerate(params):
            p.grad = gradients(p.numel(), 100 * step + 10 * k, spread).to(dtype).to(gpu)
        opt.step()
        for p, e in zip(params, plain):
            e.step(p.grad.cpu(), 1e-3, betas, 1e-8, 0.1, 5)
            e.same_as(p, opt.state[p])


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("largest", [2.0 ** -98, 1e-36, 1e-38, 1e-44])
def test_blocks_of_next_to_nothing(gpu, dtype, largest):
    """Averages that have fallen for hundreds of steps without a gradient, zeros among them: the zeros stay zeros,
    and elements without a root never move, also with eps = 0."""
    n = 4 * BLOCK
    some = torch.arange(n) % 3 == 0                      # a third ever had a gradient
    some[BLOCK:2 * BLOCK] = False
    p = nn.Parameter(randn((n,), 1, 1.0, dtype).to(gpu))
    plain = Elementary(p.detach().cpu())
    opt = AdamW([p], lr=1e-3, eps=0.0, weight_decay=0.0, state_bits=8, seed=5)
    p.grad = torch.zeros(n, dtype=dtype, device=gpu)
    opt.step()
    state = opt.state[p]
    m, r = (torch.where(some, randn((n,), k, 100.0).abs().clamp(2.0, 448.0), 0.0).to(torch.float8_e4m3fn).float()
            for k in (2, 3))
    m_scale, r_scale = torch.full((4,), largest / 448), torch.full((4,), 1e-9)
    for name, t in (("exp_avg", m), ("root_avg_sq", r), ("exp_avg_scale", m_scale), ("root_avg_sq_scale", r_scale)):
        state[name].copy_(t)
    plain.t, plain.m, plain.r, plain.m_scale, plain.r_scale = state["step"], m, r, m_scale, r_scale
    before = p.detach().cpu()
    for _ in range(25):
        opt.step()
        assert (state["exp_avg"].cpu().float()[~some] == 0).all()
        assert torch.equal(p.detach().cpu()[~some], before[~some])
        plain.step(p.grad.cpu(), 1e-3, (0.9, 0.999), 0.0, 0.0, 5)
        plain.p = torch.where(some, plain.p, before)     # 0 / 0
        plain.same_as(p, state)
    assert (state["exp_avg_scale"] == 0).all() or largest > 2.0 ** -99


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("eps", [1e-8, 0.0])
def test_finite_gradients_whose_squares_are_not(gpu, dtype, eps):
    """A gradient of 2e19, whose square is beyond fp32: no move on its own step (m over an infinite root), then NaN,
    never a number without meaning; so with a root that a loaded state holds as NaN.  The others are untouched."""
    n = 2 * BLOCK
    g = randn((n,), 1, 1.0, dtype).to(gpu)
    start = randn((n,), 2, 1.0, dtype).to(gpu)
    p = nn.Parameter(start.clone())
    opt = AdamW([p], lr=1e-3, eps=eps, weight_decay=0.0, state_bits=8)
    big = torch.zeros(n, dtype=torch.bool, device=gpu)
    big[[3, 300]] = True
    for step in range(3):
        p.grad = torch.where(big & (step == 0), torch.tensor(2e19, dtype=dtype, device=gpu), g)
        opt.step()
        assert torch.equal(p.detach().isnan(), big & (step > 0)), step
        assert p.detach()[~big].isfinite().all() and ((p.detach() - start).abs()[~big] < 0.1).all()
        if step == 0:
            assert torch.equal(p.detach()[big], start[big])
    assert torch.equal(opt.state[p]["root_avg_sq"].float().isnan(), big)
    opt.state[p]["root_avg_sq"].copy_(torch.where(torch.arange(n, device=gpu) == 7, math.nan, 1.0))
    opt.step()
    assert p.detach()[7].isnan()
    # where neither a gradient nor eps is there, nothing moves
    z = nn.Parameter(start.clone())
    opt = AdamW([z], lr=1e-3, eps=eps, weight_decay=0.0, state_bits=8)
    for step in range(2):
        z.grad = torch.zeros_like(z)
        opt.step()
        assert torch.equal(z.detach(), start)
