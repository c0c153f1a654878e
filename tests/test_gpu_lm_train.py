"""The output projection with its cross entropy, the root-mean-square norm and AdamW on the GPU against
their float64 forms, within the bounds counted in tests/train_forms.py."""
import math

import pytest
import torch
from torch import nn

import ghostsuite_amd as gs
from ghostsuite_amd import AdamW, GradDotProdEngine, _native
from ghostsuite_amd.workloads import CausalLM, LMConfig
from tests import train_forms as L
from tests.helpers import BF16_TOL, assert_close, gen, randn
from tests.lm_bounds import within
from tests.lm_forms import HALF, U, f64

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


# ------------------------------------------------------------- output projection, cross entropy
def head_inputs(N, V, d, dtype, seed, ignored=0.2):
    w = randn((V, d), seed, 2.0 / math.sqrt(d))
    labels = torch.randint(0, V, (N,), generator=gen(seed + 1))
    x = randn((N, d), seed + 2) + 3 * torch.rand(N, 1, generator=gen(seed + 3)) * w[labels]
    labels[torch.rand(N, generator=gen(seed + 4)) < ignored] = -100
    return x.to(dtype), w.to(dtype), labels


def check_head(x, w, labels, reduction, gpu, seed=9, ignore=-100):
    xg, wg = (t.detach().to(gpu).requires_grad_() for t in (x, w))
    loss = gs.head_cross_entropy(xg, wg, labels.to(gpu), reduction=reduction, ignore_index=ignore)
    up = torch.rand(loss.shape, generator=gen(seed)) + 0.5
    dx, dw = torch.autograd.grad(loss, (xg, wg), up.to(gpu))
    assert loss.dtype == FP32 and dx.dtype == dw.dtype == x.dtype
    want = L.head_all(x.reshape(-1, w.shape[1]), w, labels.reshape(-1), up.reshape(-1) if up.dim() else up,
                      reduction, x.dtype, ignore)
    within(loss.reshape(want["loss"][0].shape), *want["loss"], "loss")
    within(dx.reshape(want["dx"][0].shape), *want["dx"], "dx")
    within(dw, *want["dw"], "dw")
    with torch.no_grad():
        again = gs.head_cross_entropy(xg, wg, labels.to(gpu), reduction=reduction, ignore_index=ignore)
    assert torch.equal(again.nan_to_num(7.0), loss.detach().nan_to_num(7.0))
    return loss.detach(), dx, dw


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("N,V,d", [
    (1, 1, 1), (1, 257, 8), (2, 128, 64), (7, 130, 72), (31, 1000, 33), (32, 513, 128), (33, 256, 65),
    (40, 77, 200), (255, 300, 64), (256, 256, 8), (257, 1025, 96), (300, 2049, 130), (1025, 33, 16),
    (5, 5000, 300), (600, 12, 520)])
def test_head_sizes(gpu, dtype, N, V, d):
    for k, reduction in enumerate(("mean", "none", "sum")):
        check_head(*head_inputs(N, V, d, dtype, N + V + d + k), reduction, gpu)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("N", [20, 300, 3000])
def test_head_rows_that_do_not_count(gpu, dtype, N):
    """All of them, all but one, the first and last, and what they hold: infinities and NaN are not read."""
    V, d = 200, 40
    x, w, _ = head_inputs(N, V, d, dtype, N)
    y = torch.randint(0, V, (N,), generator=gen(1))
    for ignored in (range(N), range(N - 1), range(1, N), (0, N - 1), range(0, N, 2)):
        labels = y.clone()
        labels[list(ignored)] = -100
        dirty = x.clone()
        dirty[labels == -100] = torch.tensor([math.nan, math.inf, -math.inf, 3e38]).repeat(d // 4).to(dtype)
        for reduction in ("mean", "none"):
            loss, dx, dw = check_head(dirty, w, labels, reduction, gpu)
            assert (dx[labels == -100] == 0).all() and dw.isfinite().all()
            if reduction == "none":
                assert (loss[labels == -100] == 0).all()
            elif len(ignored) == N:
                assert loss.isnan() and (dw == 0).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("N", [9, 290])
def test_head_labels_outside_and_other_ignore_index(gpu, dtype, N):
    x, w, labels = head_inputs(N, 70, 24, dtype, 3, 0.0)
    labels[1], labels[2], labels[3] = 70, -1, 2 ** 40
    loss, dx, dw = check_head(x, w, labels, "none", gpu)
    assert loss[1:4].isnan().all() and dx[1:4].isnan().all() and loss[4:].isfinite().all()
    assert gs.head_cross_entropy(x.to(gpu), w.to(gpu), labels.to(gpu)).isnan()
    labels[1:4] = 5
    check_head(x, w, labels, "mean", gpu, ignore=5)
    check_head(x, w, labels.clamp(max=3), "sum", gpu, ignore=2)
    for t in (torch.int32, torch.int16, torch.uint8):
        got = gs.head_cross_entropy(x.to(gpu), w.to(gpu), labels.to(t).to(gpu))
        assert torch.equal(got, gs.head_cross_entropy(x.to(gpu), w.to(gpu), labels.to(gpu)))


@pytest.mark.parametrize("N", [6, 280])
def test_head_extreme_logits(gpu, N):
    """Logits of thousands, all equal ones, a row of infinities and one NaN: as log_softmax has them."""
    V, d = 300, 16
    x, w, labels = head_inputs(N, V, d, FP32, 3, 0.0)
    x[0] *= 1000
    x[1] = 0
    check_head(x, w, labels, "none", gpu)
    x[2, 3] = math.inf
    x[3, 3] = math.nan
    loss = gs.head_cross_entropy(x.to(gpu), w.to(gpu), labels.to(gpu), reduction="none").cpu()
    assert loss[2].isnan() and loss[3].isnan() and loss[4:].isfinite().all()
    # an entry of the vocabulary at minus infinity for every row has no share
    x, w, labels = head_inputs(N, V, d, FP32, 3, 0.0)
    x, w = x.abs() + 0.1, w.clone()
    w[7] = -1e38
    labels[labels == 7] = 8
    keep = torch.arange(V) != 7
    want = -torch.log_softmax((f64(x) @ f64(w)[keep].t()), 1)
    at = labels - (labels > 7).long()
    got = gs.head_cross_entropy(x.to(gpu), w.to(gpu), labels.to(gpu), reduction="none")
    assert_close(got, want[torch.arange(N), at], 1e-5)


@pytest.mark.parametrize("N", [4, 260])
def test_head_labels_with_most_of_the_mass(gpu, N):
    """Logits of a hundred, all but a ten thousandth of the mass on the label: the loss and the label's
    gradient keep what one rounding of the sum of exponentials (at least 1) and of p leaves them."""
    V, d = 300, 8
    w = torch.zeros(V, d)
    w[:, 0] = 100.0                                # the same for all
    w[:, 1] = torch.linspace(0, 1, V)
    w[7, 2] = 1.0
    x = torch.zeros(N, d)
    x[:, 0], x[:, 1], x[:, 2] = 1.0, 0.25, 15.0    # exact products
    labels = torch.full((N,), 7)
    xg, wg = x.to(gpu).requires_grad_(), w.to(gpu).requires_grad_()
    loss = gs.head_cross_entropy(xg, wg, labels.to(gpu), reduction="none")
    lp = torch.log_softmax(f64(x) @ f64(w).t(), 1)
    rest = -torch.expm1(lp[:, 7])                  # 1 - p
    assert 5e-5 < rest[0] < 2e-4
    # z: sums of three products, fp32 (three of its roundings at 100, of which the masses move by as much).
    # The sum of exponentials: a lane adds up to 64 to the label's 1, each sum rounded there (U), then sixteen
    # roundings at most of exponentials, joins, logarithm and quotient: the small ones lie below U's
    # multiples, so the roundings all go one way.
    share, sums = 3 * 128 * U, (64 + 16) * U
    assert ((loss.detach().cpu().double() + lp[:, 7]).abs() <= share * -lp[:, 7] * 4 + sums).all()
    dx, = torch.autograd.grad(loss, xg, torch.ones_like(loss))
    want = (lp.exp() - torch.nn.functional.one_hot(labels, V)) @ f64(w)
    assert ((dx.cpu().double() - want)[:, 2].abs() <= share * rest * 4 + sums).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_head_strides_alignment_and_shapes(gpu, dtype):
    """Rows apart, overlapping or reversed, off 16-byte boundaries, transposed weights, more dimensions."""
    V, d = 90, 24
    for N in (12, 270):
        x, w, labels = head_inputs(N, V, d, dtype, N)
        big = torch.zeros(N, d + 9, dtype=dtype, device=gpu)
        for off in (0, 1, 3, 8):
            rows = big[:, off:off + d]
            rows.copy_(x)
            flat = torch.zeros(V * d + 16, dtype=dtype, device=gpu)
            wt = flat[off:off + V * d].view(V, d)
            wt.copy_(w)
            base = gs.head_cross_entropy(x.to(gpu), w.to(gpu), labels.to(gpu), reduction="none")
            assert torch.equal(gs.head_cross_entropy(rows, wt, labels.to(gpu), reduction="none"), base)
            a, b = rows.detach().requires_grad_(), wt.detach().requires_grad_()
            g = torch.autograd.grad(gs.head_cross_entropy(a, b, labels.to(gpu)), (a, b))
            c, e = x.to(gpu).requires_grad_(), w.to(gpu).requires_grad_()
            h = torch.autograd.grad(gs.head_cross_entropy(c, e, labels.to(gpu)), (c, e))
            assert all(torch.equal(p, q) for p, q in zip(g, h))
        wt = w.t().contiguous().to(gpu).t()
        assert torch.equal(gs.head_cross_entropy(x.to(gpu), wt, labels.to(gpu), reduction="none"), base)
        x3, y3 = x.to(gpu).view(2, N // 2, d), labels.to(gpu).view(2, N // 2)
        got = gs.head_cross_entropy(x3.transpose(0, 1), w.to(gpu), y3.t(), reduction="none")
        assert got.shape == (N // 2, 2) and torch.equal(got, base.view(2, -1).t())
        same = x[:1].to(gpu).expand(N, d)
        got = gs.head_cross_entropy(same, w.to(gpu), labels.to(gpu).clamp(min=0), reduction="none")
        assert torch.equal(got, gs.head_cross_entropy(same.contiguous(), w.to(gpu),
                                                      labels.to(gpu).clamp(min=0), reduction="none"))
    one = gs.head_cross_entropy(x[0].to(gpu), w.to(gpu), labels[1].to(gpu).clamp(min=0), reduction="none")
    assert one.shape == ()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("d", [2, 7, 12, 34, 68, 101])
def test_head_operands_among_nan(gpu, dtype, d):
    """What lies around the rows and the weight takes no part, however a row's length divides."""
    V = 150
    for N in (3, 32, 70):
        x, w, labels = head_inputs(N, V, d, dtype, N + d, 0.3)
        rows = torch.full((N + 2, d + 3), math.nan, dtype=dtype, device=gpu)[1:-1, 2:2 + d]
        rows.copy_(x)
        for off in (0, 2, 9):
            flat = torch.full((V * d + 32,), math.nan, dtype=dtype, device=gpu)
            wt = flat[off:off + V * d].view(V, d)
            wt.copy_(w)
            for reduction in ("mean", "none"):
                got = []
                for a, b in ((rows, wt), (x.to(gpu), w.to(gpu))):
                    a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
                    loss = gs.head_cross_entropy(a, b, labels.to(gpu), reduction=reduction)
                    got.append((loss, *torch.autograd.grad(loss, (a, b), torch.ones_like(loss))))
                assert all(p.isfinite().all() and torch.equal(p, q) for p, q in zip(*got))
    check_head(x, w, labels, "mean", gpu)


def test_head_of_no_rows(gpu):
    w = randn((9, 8), 1).to(gpu).requires_grad_()
    x = torch.zeros(2, 0, 8, device=gpu, requires_grad=True)
    y = torch.zeros(2, 0, dtype=torch.long, device=gpu)
    for reduction in ("mean", "sum", "none"):
        loss = gs.head_cross_entropy(x, w, y, reduction=reduction)
        dx, dw = torch.autograd.grad(loss, (x, w), torch.ones_like(loss))
        assert dx.shape == x.shape and (dw == 0).all()
        assert loss.isnan() if reduction == "mean" else (loss == 0).all()


@pytest.mark.parametrize("N,dtype", [(4, BF16), (300, BF16), (700, FP32)])
def test_head_in_pieces(gpu, N, dtype, monkeypatch):
    """A vocabulary of several pieces (as many rows make) gives what one piece does; the gradient of the
    logits for a caller, piece by piece, multiplied up, gives the same again."""
    V, d = 1500, 48
    x, w, labels = head_inputs(N, V, d, dtype, 5)
    xg, wg, yg = x.to(gpu).requires_grad_(), w.to(gpu).requires_grad_(), labels.to(gpu)
    up = torch.tensor(0.7, device=gpu)
    loss = gs.head_cross_entropy(xg, wg, yg)
    lse = torch.empty(N, 2, device=gpu)
    _native.ops().head_cross_entropy(xg.detach(), wg.detach(), yg, -100, "mean", lse)
    want = L.head_all(x, w, labels, up.cpu(), "mean", dtype)
    whole = torch.cat([_native.ops().head_logit_grad(xg.detach(), wg.detach(), yg, lse, up, v0,
                                                     min(700, V - v0), -100, "mean")[:, :min(700, V - v0)]
                       for v0 in range(0, V, 700)], 1)
    exact = L.head_dz(f64(x), f64(w), labels, up.cpu(), 0, V, "mean")
    zeros = labels == -100
    assert (whole.cpu()[zeros] == 0).all()
    # a logit's error is far below the probability's rounding here: 1e-4 of it, and of its type
    within(whole, exact, exact.abs() * (1e-4 + HALF[dtype]) + 1e-6 * exact.abs().max(), "dz")
    for piece in (1, 700, 9):
        part = _native.ops().head_logit_grad(xg.detach(), wg.detach(), yg, lse, up, 3, piece, -100, "mean")
        assert part.shape == (N, -(-piece // 8) * 8)
        assert torch.equal(part[:, :piece], whole[:, 3:3 + piece]) and (part[:, piece:] == 0).all()
    dx, dw = torch.autograd.grad(loss, (xg, wg), up)
    within(dx, *want["dx"], "dx")
    within(dw, *want["dw"], "dw")


def test_head_of_many_rows_in_pieces(gpu):
    """Enough rows that the vocabulary takes several pieces: each row alone is in the bound, and the
    gradients are those of a product of the logits' gradient in one piece."""
    N, V, d = 150000, 4000, 16
    x, w, labels = head_inputs(N, V, d, BF16, 5)
    xg, wg, yg = x.to(gpu).requires_grad_(), w.to(gpu).requires_grad_(), labels.to(gpu)
    loss = gs.head_cross_entropy(xg, wg, yg, reduction="none")
    part = torch.randperm(N, generator=gen(1))[:300]
    want = L.head_all(x[part], w, labels[part], torch.ones(300), "none", BF16)
    within(loss[part.to(gpu)], *want["loss"], "loss")
    dx, dw = torch.autograd.grad(loss, (xg, wg), torch.ones_like(loss))
    within(dx[part.to(gpu)], *want["dx"], "dx")
    lse = torch.empty(N, 2, device=gpu)
    _native.ops().head_cross_entropy(xg.detach(), wg.detach(), yg, -100, "none", lse)
    for v0 in range(0, V, 1000):
        dz = _native.ops().head_logit_grad(xg.detach(), wg.detach(), yg, lse, torch.ones(N, device=gpu), v0,
                                           1000, -100, "none")
        ref = dz.double().t() @ xg.detach().double()
        # the same rounded dz on both sides: the sums' terms and the output's rounding
        size = dz.double().abs().t() @ xg.detach().double().abs()
        within(dw[v0:v0 + 1000], ref.cpu(), (ref.abs() * HALF[BF16] + (N + 64) * U * size).cpu(), "dw")


@pytest.mark.parametrize("ignored", [0.0, 0.7])
def test_head_weight_gradient_in_whole_rounds_and_shares(gpu, ignored):
    """A few tiles of dW more than compute units: the rest is a product of its own, over shares of the rows
    that count."""
    N, V, d = 4096, 65536 + 264, 256
    x, w, labels = head_inputs(N, V, d, BF16, 6, ignored)
    xg, wg, yg = x.to(gpu).requires_grad_(), w.to(gpu).requires_grad_(), labels.to(gpu)
    dw, = torch.autograd.grad(gs.head_cross_entropy(xg, wg, yg, reduction="none"), wg,
                              torch.ones(N, device=gpu))
    lse = torch.empty(N, 2, device=gpu)
    _native.ops().head_cross_entropy(xg.detach(), wg.detach(), yg, -100, "none", lse)
    for v0 in (0, 32000, 65536 - 300, V - 300):
        dz = _native.ops().head_logit_grad(xg.detach(), wg.detach(), yg, lse, torch.ones(N, device=gpu), v0,
                                           300, -100, "none")[:, :300]
        ref = dz.double().t() @ xg.detach().double()
        size = dz.double().abs().t() @ xg.detach().double().abs()
        within(dw[v0:v0 + 300], ref.cpu(), (ref.abs() * HALF[BF16] + (N + 64) * U * size).cpu(), "dw")


def test_head_gradients_by_differences(gpu):
    x, w, labels = head_inputs(40, 60, 12, FP32, 8)
    x, w, labels = x.to(gpu).requires_grad_(), w.to(gpu).requires_grad_(), labels.to(gpu)
    dx, dw = torch.autograd.grad(gs.head_cross_entropy(x, w, labels, reduction="sum"), (x, w))
    for leaf, grad in ((x, dx), (w, dw)):
        e = randn(leaf.shape, 4).to(gpu)
        e /= e.norm()
        step = 1e-2
        with torch.no_grad():
            at = [gs.head_cross_entropy(*(t + s * step * e if t is leaf else t for t in (x, w)), labels,
                                        reduction="none").double().sum() for s in (1, -1)]
        # central difference: its error is the third derivative's step^2, and the losses' roundings
        assert abs((at[0] - at[1]) / (2 * step) - (grad.double() * e).sum()) < 2e-3


def test_head_refusals(gpu):
    x, w, y = randn((4, 8), 1).to(gpu), randn((9, 8), 2).to(gpu), torch.zeros(4, dtype=torch.long, device=gpu)
    for bad in (dict(x=x.half()), dict(w=w.half()), dict(w=w.bfloat16()), dict(w=w[:, :4]), dict(w=w[0]),
                dict(w=w[:0]), dict(y=y[:3]), dict(y=y.float()), dict(y=y.bool()), dict(y=y.cpu()),
                dict(x=x[:, :0], w=w[:, :0])):
        a = {"x": x, "w": w, "y": y, **bad}
        with pytest.raises(_native.GhostHipError):
            gs.head_cross_entropy(a["x"], a["w"], a["y"])
    xg = x.detach().requires_grad_()
    g, = torch.autograd.grad(gs.head_cross_entropy(xg, w, y), xg, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
    loss = gs.head_cross_entropy(xg, w, y)
    w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


# ------------------------------------------------------------------ root-mean-square norm
def check_norm(x, res, w, eps, gpu, seed=3, unused=None):
    xg, rg, wg = (None if t is None else t.detach().to(gpu).requires_grad_() for t in (x, res, w))
    out = (gs.rms_norm(xg, wg, eps=eps),) if res is None else gs.add_rms_norm(xg, rg, wg, eps=eps)
    h = x if res is None else (x.float() + res.float()).to(x.dtype)
    if res is not None:
        assert torch.equal(out[1].cpu(), h)
    grads = [randn(x.shape, seed + k, 1.0, x.dtype) for k in range(len(out))]
    used = [k for k in range(len(out)) if k != unused]
    leaves = [t for t in (xg, rg, wg) if t is not None]
    got = torch.autograd.grad([out[k] for k in used], leaves, [grads[k].to(gpu) for k in used])
    gy = None if unused == 0 else grads[0]
    gh = grads[1] if len(out) > 1 and unused != 1 else None
    want = L.norm_all(h, w, gy, gh, eps, x.dtype)
    within(out[0], *want["y"], "y")
    within(got[0], *want["dh"], "dx")
    within(got[-1], *want["dw"], "dw")
    if res is not None:
        assert torch.equal(got[0], got[1])
    for k, t in enumerate(gs.add_rms_norm(xg.detach(), rg.detach(), wg.detach(), eps=eps) if res is not None
                          else (gs.rms_norm(xg.detach(), wg.detach(), eps=eps),)):
        assert torch.equal(t, out[k])


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("F", [1, 2, 7, 8, 31, 33, 64, 96, 100, 255, 256, 257, 520, 768, 769, 1023, 1024,
                               1500, 2048, 2049, 2560, 4096, 4100, 8191, 8192, 8193, 12000])
def test_norm_widths(gpu, dtype, F):
    for rows, eps in ((1, 1e-6), (37, 1e-2)):
        x, r = randn((rows, F), 1, 1.0, dtype), randn((rows, F), 2, 2.0, dtype)
        w = (1 + 0.2 * randn((F,), 3)).to(dtype)
        check_norm(x, r, w, eps, gpu)
        check_norm(x, None, w, eps, gpu)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape", [(3, 5, 64), (2, 3, 4, 24), (5000, 40), (9, 1000, 96), (1030, 9000), (16,)])
def test_norm_shapes_and_unused_outputs(gpu, dtype, shape):
    x, r = randn(shape, 1, 1.0, dtype), randn(shape, 2, 1.0, dtype)
    w = (1 + 0.2 * randn((shape[-1],), 3)).to(dtype)
    for unused in (None, 0, 1):
        check_norm(x, r, w, 1e-6, gpu, unused=unused)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_norm_strides_alignment_zeros_and_no_rows(gpu, dtype):
    F = 48
    w = (1 + 0.2 * randn((F,), 3)).to(dtype).to(gpu)
    big = randn((7, 3, F + 16), 1, 1.0, dtype).to(gpu)
    for x in (big[..., 3:3 + F], big[:, ::2, :F], big[..., :F].transpose(0, 1), big[:, :1, :F].expand(7, 5, F)):
        y, h = gs.add_rms_norm(x, x, w)
        a, b = gs.add_rms_norm(x.contiguous(), x.contiguous(), w)
        assert torch.equal(y, a) and torch.equal(h, b) and y.is_contiguous()
        x1 = x.detach().requires_grad_()
        g, = torch.autograd.grad(gs.rms_norm(x1, w).sum(), x1)      # an expanded output gradient
        x2 = x.detach().contiguous().requires_grad_()
        assert torch.equal(g, torch.autograd.grad(gs.rms_norm(x2, w), x2, torch.ones_like(x2))[0])
    flat = torch.zeros(5 * F + 8, dtype=dtype, device=gpu)
    for off in (1, 2, 4):
        x = flat[off:off + 5 * F].view(5, F).copy_(big[:5, 0, :F])
        # lanes hold other elements then, and the squares add up in another order: (F + 8) U of their sum
        # at most either way, which is what norm_all counts
        within(gs.rms_norm(x, w), *L.norm_all(big[:5, 0, :F], w, None, None, 1e-6, dtype)["y"])
    zero = torch.zeros(4, F, dtype=dtype, device=gpu, requires_grad=True)
    y = gs.rms_norm(zero, w, eps=0.25)
    assert (y == 0).all()
    g, = torch.autograd.grad(y.sum(), zero)
    assert torch.equal(g, (2 * w.float()).to(dtype).expand(4, F))
    none = torch.zeros(0, 3, F, dtype=dtype, device=gpu, requires_grad=True)
    wg = w.detach().requires_grad_()
    y, h = gs.add_rms_norm(none, none, wg)
    gx, gw = torch.autograd.grad((y, h), (none, wg), (torch.zeros_like(y), torch.zeros_like(h)))
    assert y.shape == h.shape == gx.shape == (0, 3, F) and (gw == 0).all()


def test_norm_rows_stay_apart(gpu):
    """An infinity or a NaN in one row leaves the others, forward and backward."""
    for F in (64, 700, 3001, 9000):
        x = randn((9, F), 1)
        x[2, 5], x[4, 0] = math.inf, math.nan
        w = torch.ones(F)
        clean = torch.arange(9) != 2
        clean[4] = False
        xg = x.to(gpu).requires_grad_()
        y = gs.rms_norm(xg, w.to(gpu))
        g, = torch.autograd.grad(y, xg, torch.ones_like(y))
        assert y.cpu()[clean].isfinite().all() and g.cpu()[clean].isfinite().all()
        assert y.cpu()[4].isnan().all()
        want = L.norm_all(x[clean], w, torch.ones(7, F), None, 1e-6, FP32)
        within(y[clean.to(gpu)], *want["y"], "y")
        within(g[clean.to(gpu)], *want["dh"], "dx")


def test_norm_of_more_rows_than_a_launch(gpu):
    rows = (1 << 25) + 5
    x = torch.randn(rows, 1, device=gpu, dtype=BF16)
    res = torch.randn(rows, 1, device=gpu, dtype=BF16)
    w = torch.full((1,), 1.5, device=gpu, dtype=BF16)
    y, h = gs.add_rms_norm(x, res, w)
    alone = gs.rms_norm(h, w)
    assert torch.equal(h, x + res) and torch.equal(alone, y)
    for at in (0, (1 << 25) - 500, rows - 1000):
        part = slice(at, at + 1000)
        some, _ = gs.add_rms_norm(x[part], res[part], w)
        assert torch.equal(some, y[part])


def test_norm_refusals(gpu):
    x, w = randn((4, 8), 1).to(gpu), torch.ones(8, device=gpu)
    for bad in (lambda: gs.rms_norm(x.half(), w.half()), lambda: gs.rms_norm(x, w[:4]),
                lambda: gs.rms_norm(x, w.bfloat16()), lambda: gs.add_rms_norm(x, x[:2], w),
                lambda: gs.add_rms_norm(x, x.bfloat16(), w), lambda: gs.add_rms_norm(x, x.cpu(), w),
                lambda: gs.rms_norm(x, w[None]), lambda: gs.rms_norm(x[:, :0], w[:0])):
        with pytest.raises(_native.GhostHipError):
            bad()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("N,T,F,n_val", [(5, 1, 8, 1), (7, 65, 96, 3), (4, 130, 1023, 2), (6, 33, 2500, 5),
                                         (20, 64, 768, 4)])
def test_norm_dots(gpu, dtype, N, T, F, n_val):
    """Dots and train gradient against float64: sums over T tokens, then over samples and features."""
    h, g = randn((N, T, F), 1, 1.0, dtype), randn((N, T, F), 2, 1.0, dtype)
    w = torch.ones(F, dtype=dtype)
    for start in (None, 0, 1):
        dots, dw = _native.ops().rms_norm_dot(h.to(gpu), g.to(gpu), w.to(gpu), 1e-6, n_val, val_start=start,
                                              grad_scale=0.3)
        x = f64(h)
        a = f64(g) * x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        vs = N - n_val if start is None else start
        val = torch.zeros(N, dtype=torch.bool)
        val[vs:vs + n_val] = True
        s, size = a.sum(1), a.abs().sum(1)
        e = ((F / 2 + 8) + T + 80) * U * size
        sv, ev = s[val].sum(0), e[val].sum(0) + n_val * U * size[val].sum(0)
        want = s[~val] @ sv
        within(dots, want, e[~val] @ sv.abs() + s[~val].abs() @ ev + (F + 64) * U * (s[~val].abs() @ sv.abs()),
               "dots")
        grad = s[~val].sum(0) * 0.3
        within(dw, grad, 0.3 * (e[~val].sum(0) + N * U * size.sum(0)) + grad.abs() * HALF[dtype], "gradient")


# ---------------------------------------------------------------------------------- AdamW
def check_adamw_step(opt, params, before, group):
    """The step just made against float64, from the state before it: (p, m, root) of each."""
    lr, betas, eps, decay = group["lr"], group["betas"], group["eps"], group["weight_decay"]
    bits = group["state_bits"]
    for p, (p0, g, m0, r0) in zip(params, before):
        state, n = opt.state[p], p.numel()
        step = state["step"]
        want, m, v, root = L.adamw_form(p0, g, m0, r0, lr, betas, eps, decay, step)
        em = 4 * U * (betas[0] * m0.abs() + (1 - betas[0]) * g.abs())
        ev = 8 * U * v
        er = 6 * U * root
        bc1, bc2 = 1 - betas[0] ** step, 1 - betas[1] ** step
        den = root / math.sqrt(bc2) + eps
        move = lr / bc1 * m.abs() / den
        bound = move * 24 * U + lr / bc1 * em / den + 4 * U * p0.abs() + 4 * U * move
        within(p.reshape(-1), want, bound + want.abs() * HALF[p.dtype], "p")
        if bits == 32:
            within(state["exp_avg"].reshape(-1), m, em, "m")
            within(state["exp_avg_sq"].reshape(-1), v, ev, "v")
            continue
        for name, x, u, e in zip(("exp_avg", "root_avg_sq"), (m, root),
                                 L.chances(n, step, group["seed"]), (em, er)):
            scale = f64(state[name + "_scale"])
            top = L.blocks_max(x)
            within(scale, top / L.TOP, top / L.TOP * 12 * U, name + " scale")
            share = (L.TOP / top.clamp(min=1e-300)).repeat_interleave(L.BLOCK)[:n]
            q = state[name].detach().cpu().float().double().reshape(-1)
            a, ea = x.abs() * share, e * share + 448 * 16 * U
            lo, hi = L.held((a - ea).clamp(min=0), u - 4 * U), L.held(a + ea, u + 4 * U).clamp(max=448)
            if name == "root_avg_sq":
                lo, hi = (torch.where(x > 0, t.clamp(min=2.0 ** -9), 0.0) for t in (lo, hi))
            assert ((q.abs() >= lo) & (q.abs() <= hi)).all(), name
            assert ((q * x.sign() >= 0) | (x == 0)).all(), name


def state_of(opt, p, bits):
    m, r = L.averages(opt.state[p], p.shape, bits) if p in opt.state else (torch.zeros(p.numel()).double(),) * 2
    return f64(p).reshape(-1), f64(p.grad).reshape(-1), m, r


SHAPES = [(1,), (3,), (255,), (256,), (257,), (8, 33), (512, 16), (8191,), (8192,), (8193,), (0,), (), (4, 0),
          (100, 331), (2, 3, 5, 7)]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("how", [dict(), dict(lr=0.3, betas=(0.0, 0.0), eps=1e-3, weight_decay=0.5),
                                 dict(betas=(0.5, 0.999), weight_decay=0.0, seed=-5)])
def test_adamw_steps(gpu, dtype, bits, how):
    params = [nn.Parameter(randn(s, k, 1.0, dtype).to(gpu)) for k, s in enumerate(SHAPES)]
    opt = AdamW(params, state_bits=bits, **how)
    for step in range(3):
        for k, p in enumerate(params):
            p.grad = (randn(p.shape, 100 * step + k, 10.0 ** (k % 5 - 3))).to(dtype).to(gpu)
        before = [state_of(opt, p, bits) for p in params]
        version = params[0]._version
        opt.step()
        assert params[0]._version > version
        check_adamw_step(opt, params, before, opt.param_groups[0])


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_memory_orders(gpu, bits):
    """Tensors off 16-byte boundaries, in other orders of memory than their indices', and gradients in
    others than their parameter's."""
    flat = torch.zeros(4000, device=gpu)
    a = nn.Parameter(flat[1:1001].view(10, 100))
    b = nn.Parameter(randn((6, 4, 5, 5), 1).to(gpu).to(memory_format=torch.channels_last))
    c = nn.Parameter(randn((30, 20), 2).to(gpu).t())
    d = nn.Parameter(randn((30, 20), 3).to(gpu))
    plain = [nn.Parameter(p.detach().clone(memory_format=torch.contiguous_format)) for p in (a, d)]
    opt, ref = AdamW([a, b, c, d], state_bits=bits), AdamW(plain, state_bits=bits)
    for step in range(2):
        for k, p in enumerate((a, b, c, d)):
            g = randn(p.shape, 10 * step + k).to(gpu)
            p.grad = torch.empty(4001, device=gpu)[1:1001].view(10, 100).copy_(g) if p is a else g
        d.grad = d.grad.t().contiguous().t()
        for p, q in zip((a, d), plain):
            q.grad = p.grad.contiguous()
        before = [state_of(opt, p, bits) for p in (a, d)]
        kept = {p: (f64(p), f64(p.grad)) for p in (b, c)}
        opt.step()
        ref.step()
        check_adamw_step(opt, [a, d], before, opt.param_groups[0])
        for p in (b, c):      # the first step of Adam moves by lr whatever the order
            p0, g = kept[p]
            if step == 0:
                want = p0 * (1 - 1e-5) - 1e-3 * g / (g.abs() + 1e-8)
                within(p, want, want.abs() * 8 * U + 1e-3 * 40 * U, "p")
            assert opt.state[p]["exp_avg"].stride() == p.stride()
    for p, q in zip((a, d), plain):
        assert torch.equal(p, q)
    assert (flat[0] == 0) and (flat[1001:] == 0).all()
    for view in (torch.zeros(4, 6, device=gpu)[:, :3], torch.zeros(1, 6, device=gpu).expand(4, 6)):
        p = nn.Parameter(view)
        p.grad = torch.zeros(view.shape, device=gpu)
        with pytest.raises(_native.GhostHipError, match="fill their memory"):
            AdamW([p], state_bits=bits).step()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_adamw_of_many_and_mixed_tensors(gpu, dtype):
    """More tensors than a launch takes, both types in one group, and the same bits on every run."""
    runs = []
    for _ in range(2):
        params = [nn.Parameter(randn((1 + 97 * k % 700,), k, 1.0, dtype if k % 3 else FP32).to(gpu))
                  for k in range(150)]
        opt = AdamW(params, state_bits=8, seed=1)
        for step in range(2):
            for k, p in enumerate(params):
                p.grad = randn(p.shape, 1000 * step + k, 1.0, p.dtype).to(gpu)
            before = [state_of(opt, p, 8) for p in params]
            opt.step()
            check_adamw_step(opt, params, before, opt.param_groups[0])
        runs.append([t for p in params for t in (p.detach(), opt.state[p]["exp_avg"].view(torch.uint8),
                                                 opt.state[p]["root_avg_sq"].view(torch.uint8))])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_adamw_beyond_32_bits(gpu):
    """A tensor of more than 2^32 bytes and 2^31 elements, bf16 with averages in 8 bits; its last block."""
    n = (1 << 31) + 300
    p = nn.Parameter(torch.ones(n, dtype=BF16, device=gpu))
    p.grad = torch.ones(n, dtype=BF16, device=gpu)
    opt = AdamW([p], lr=0.5, weight_decay=0.0, state_bits=8)
    opt.step()
    assert (p == 0.5).all()
    assert (opt.state[p]["exp_avg"].float()[-300:] == 448).all()
    assert_close(opt.state[p]["exp_avg_scale"][-2:], torch.full((2,), 0.1 / 448), 1e-6)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_adamw_8_bits_that_are_not_finite_or_stop(gpu, dtype):
    """NaN and infinite gradients stay in their element; an element whose gradient stops, beside one of a
    far larger gradient, is never divided by eps alone."""
    p = nn.Parameter(torch.zeros(700, dtype=dtype, device=gpu))
    opt = AdamW([p], lr=1e-3, weight_decay=0.0, state_bits=8)
    g = torch.full((700,), 0.5, dtype=dtype, device=gpu)
    g[3], g[300] = math.nan, math.inf
    p.grad = g
    opt.step()
    p.grad = torch.full_like(g, 0.5)
    opt.step()
    bad = torch.zeros(700, dtype=torch.bool)
    bad[[3, 300]] = True
    for t in (p, opt.state[p]["exp_avg"].float(), opt.state[p]["root_avg_sq"].float()):
        assert torch.equal(t.detach().isnan().cpu(), bad)
    assert opt.state[p]["exp_avg_scale"].isfinite().all()

    p = nn.Parameter(torch.zeros(256, dtype=dtype, device=gpu))
    opt = AdamW([p], lr=1e-3, weight_decay=0.0, state_bits=8)
    size = torch.logspace(-9, 2, 256).to(dtype).to(gpu)
    for step in range(12):
        p.grad = size * (1.0 if step < 3 else 0.0)
        old = p.detach().clone()
        opt.step()
        # |m| is at most its share of the largest m's step of 2^-9 / 448 above itself, the root at least
        # half of itself: a move of Adam's is lr m / root <= lr sqrt(1000) / 10, and twice that
        assert ((p - old).abs().float() <= 1e-3 * 2 * 4).all(), step
    assert (opt.state[p]["root_avg_sq"].float() > 0).all()


def test_adamw_refusals_leave_everything(gpu):
    good, bad = nn.Parameter(torch.ones(5, device=gpu)), nn.Parameter(torch.ones(5, device=gpu).half())
    good.grad, bad.grad = torch.ones_like(good), torch.ones_like(bad)
    opt = AdamW([good, bad])
    with pytest.raises(_native.GhostHipError, match="bf16 or fp32"):
        opt.step()
    assert (good == 1).all() and opt.state[good]["step"] == 0
    for name, value in (("exp_avg", torch.zeros(5, device=gpu).bfloat16()), ("exp_avg", torch.zeros(4, device=gpu)),
                        ("exp_avg_sq", torch.zeros(5))):
        opt = AdamW([good])
        opt.step()
        opt.state[good][name] = value
        with pytest.raises(_native.GhostHipError, match=name):
            opt.step()
    opt = AdamW([good])
    opt.step()
    del opt.state[good]["exp_avg_sq"]
    with pytest.raises(_native.GhostHipError, match="exp_avg_sq"):
        opt.step()
    graph = torch.cuda.CUDAGraph()
    opt = AdamW([good])
    opt.step()
    at = good.detach().clone()
    torch.cuda.synchronize()
    with pytest.raises(_native.GhostHipError, match="captured"):
        with torch.cuda.graph(graph):
            opt.step()
    torch.cuda.synchronize()
    assert torch.equal(good, at)


# ------------------------------------------------------- streams, graphs, and all of them together
def test_streams_and_two_calls_at_once(gpu):
    """Each call runs on the current stream; two on different streams do not share anything."""
    x, w, labels = head_inputs(400, 3000, 64, BF16, 5)
    x, w, labels = x.to(gpu), w.to(gpu), labels.to(gpu)
    nw = torch.ones(64, dtype=BF16, device=gpu)

    def work(x):
        a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
        n = nw.detach().requires_grad_()
        y, h = gs.add_rms_norm(a, a, n)
        loss = gs.head_cross_entropy(y, b, labels) + h.float().sum() * 1e-3
        return [loss.detach(), *torch.autograd.grad(loss, (a, b, n))]
    want = [work(x), work(-x)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for s, v in zip(streams, (x, -x)):
        with torch.cuda.stream(s):
            got.append([work(v) for _ in range(3)])
    torch.cuda.synchronize()
    for g, t in zip(got, want):
        for again in g:
            assert all(torch.equal(p, q) for p, q in zip(again, t))


@pytest.mark.parametrize("N,dtype", [(8, BF16), (300, BF16), (40, FP32)])
def test_captured_and_replayed(gpu, N, dtype):
    """Forward and backward of norm and head in a graph: every replay against the eager result, with eager
    work in between, other inputs, and another number of rows that count."""
    V, d = 700, 56
    x, w, labels = (t.to(gpu) for t in head_inputs(N, V, d, dtype, 5))
    nw = torch.ones(d, dtype=dtype, device=gpu)

    def work():
        a, b, n = (t.detach().requires_grad_() for t in (x, w, nw))
        y, h = gs.add_rms_norm(a, a, n)
        loss = gs.head_cross_entropy(y + h, b, labels)
        return [loss.detach(), *torch.autograd.grad(loss, (a, b, n))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for k in range(4):
        other = head_inputs(N, V, d, dtype, 50 + k, ignored=0.3 * k)
        for t, o in zip((x, w, labels), other):
            t.copy_(o)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = work()
        torch.cuda.synchronize()
        # (a mean over no rows is NaN)
        assert all(torch.equal(p.nan_to_num(7.0), q.nan_to_num(7.0)) for p, q in zip(out, eager)), k


def _model(dtype, gpu, **how):
    torch.manual_seed(0)
    cfg = LMConfig(n_layer=2, n_head=2, d_model=64, d_mlp=96, vocab=501, n_ctx=32, **how)
    return CausalLM(cfg).to(gpu, dtype)


@pytest.mark.parametrize("tied", [True, False])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_engine_step_of_a_model(gpu, tied, dtype):
    """A model with the norm and the head's loss under the engine and the optimizer: dots and train
    gradients as those of the same model whose logits go into torch's loss; then a step."""
    n, n_val, T = 6, 2, 32
    ids = torch.randint(0, 501, (n, T), generator=gen(1)).to(gpu)
    labels = torch.randint(0, 501, (n, T), generator=gen(2)).to(gpu)
    labels[0, :5] = -100
    got = []
    for head in (True, False):
        model = _model(dtype, gpu, tied=tied, norm="rms", head_loss=head)
        opt = AdamW(model.parameters(), lr=1e-3, state_bits=8)
        # ('reference' rounds the operands of most dots to bf16 in fp32 models too)
        eng = GradDotProdEngine(model, val_batch_size=n_val, use_dummy_bias=True,
                                precision="fp32" if dtype == FP32 else "reference")
        eng.attach(opt)
        eng.attach_train_batch(ids[:4], labels[:4], 0, 0)
        loss = model(ids, labels)
        loss.backward()
        dots = {k: p.grad_dot_prod.float().clone() for k, p in model.named_parameters()
                if hasattr(p, "grad_dot_prod")}
        eng.prepare_gradients()
        grads = {k: p.grad.clone() for k, p in model.named_parameters() if p.grad is not None}
        before = [p.detach().clone() for p in model.parameters()]
        opt.step()
        eng.aggregate_and_log()
        eng.clear_gradients()
        assert any(not torch.equal(p, q) for p, q in zip(model.parameters(), before))
        assert eng.dot_product_log[-1]["dot_product"].isfinite().all()
        got.append((loss.detach(), dots, grads))
        eng.detach()
    tol = BF16_TOL if dtype == BF16 else 1e-4
    assert_close(got[0][0], got[1][0], tol, "loss")
    assert got[0][1].keys() == got[1][1].keys() and got[0][2].keys() == got[1][2].keys()
    for k in got[0][1]:
        assert_close(got[0][1][k], got[1][1][k], 2 * tol, f"dot {k}")
    if dtype == FP32:
        for k in got[0][2]:
            assert_close(got[0][2][k], got[1][2][k], 2 * tol, f"gradient {k}")
        return
    # In bf16 the two round differently on the way (the logits' model rounds each logit, 2^-8 of it, its
    # loss's gradient and that of the logits; the head only the last), and an element of a gradient is a sum
    # of hundreds of such errors against terms that cancel: no bound relative to the element holds.  The
    # errors' 2-norms do compare: each gradient has at least 64 elements and thousands of independent
    # roundings, of which the head's are a part of the other's, so that its error against the fp32 model of
    # the same weights is at most the other's but for chance, which twice covers (the root of the mean of
    # 64 squares is off by a ninth, its deviation).
    model = _model(dtype, gpu, tied=tied, norm="rms", head_loss=False).float()
    loss = nn.functional.cross_entropy(model(ids).flatten(0, 1)[:(n - n_val) * T],
                                       labels[:n - n_val].flatten(), reduction="sum") * \
        n / (n - n_val) / int((labels != -100).sum())
    names = [k for k, _ in model.named_parameters()]
    ref = dict(zip(names, torch.autograd.grad(loss, list(model.parameters()))))
    for k, want in ref.items():
        ours, theirs = ((g[2][k].float() - want).norm() for g in got)
        assert ours <= 2 * theirs, f"gradient {k}: off by {ours:.3g}, from logits {theirs:.3g}"


def test_engine_head_large_pieces(gpu):
    """The head alone under the engine, bf16, its vocabulary in pieces, T a multiple of 64 and not: dots of
    the pairwise branch within bf16's tolerance of float64's."""
    for n, n_val, T in ((6, 2, 64), (7, 1, 50)):
        V, d = 3000, 128
        x, w, labels = head_inputs(n * T, V, d, BF16, 7, 0.0)
        layer = gs.HeadCrossEntropy(d, V).to(gpu, BF16)
        with torch.no_grad():
            layer.weight.copy_(w)
        eng = GradDotProdEngine(layer, val_batch_size=n_val, use_dummy_bias=True)
        eng.attach(torch.optim.SGD(layer.parameters(), lr=0.0))
        xg = x.view(n, T, d).to(gpu).requires_grad_()
        layer(xg, labels.view(n, T).to(gpu)).backward()
        dz = L.head_dz(f64(x), f64(w), labels, torch.tensor(1.0), 0, V, "mean").view(n, T, V)
        grads = torch.stack([dz[i].t() @ f64(x).view(n, T, d)[i] for i in range(n)])
        train, val = grads[:n - n_val], grads[n - n_val:]
        assert_close(layer.weight.grad_dot_prod, (train * val.sum(0)).sum((1, 2)), BF16_TOL, "dots")
        # the train gradient is the train rows' mean; the kernels round dz (here with every factor) and the
        # result once each, as the loss's own backward pass does
        mine = labels.clone()
        mine[(n - n_val) * T:] = -100
        one = torch.tensor(1.0)
        within(layer.weight.train_grad, *L.head_all(x, w, mine, one, "mean", BF16)["dw"], "gradient")
        within(xg.grad.view(-1, d), *L.head_all(x, w, labels, one, "mean", BF16)["dx"], "dx")
        eng.detach()
