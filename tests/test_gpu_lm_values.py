"""The language-model operators on the GPU at infinities, NaN and the ends of their ranges."""
import math

import pytest
import torch

import ghostsuite_amd as gs
from tests import lm_forms as L
from tests.helpers import gen, randn

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


def same(got, want, what):
    """The same values, NaN in the same places."""
    torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True, msg=lambda m: f"{what}: {m}")


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("D,n_rot", [(64, 32), (64, 16), (80, 20), (33, 10), (33, 32), (256, 64),
                                     (66, 2), (100, 6), (64, 2), (24, 0)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_qk_features_past_the_rotated_ones_stay_by_themselves(gpu, dtype, interleaved, norm, D,
                                                              n_rot, bad):
    """An infinity or NaN in one of them, or in its output gradient, reaches no other feature but
    through the row's norm.  Token t has it at feature n_rot + t, of the last query head for even
    tokens, of the key head for odd ones."""
    B, T, heads = 2, D - n_rot, (2, 1, 1)
    table = gs.rotary_table(T, n_rot, device=gpu)
    x = randn((B, T, sum(heads), D), 1).to(dtype).to(gpu)
    grads = [randn((B, h, T, D), 2 + i, 1.0, dtype).to(gpu) for i, h in enumerate(heads)]
    w = [(1 + 0.2 * randn((D,), 5 + i)).to(dtype).to(gpu).requires_grad_() for i in range(2)] \
        if norm else [None, None]

    def run(x, grads):
        x = x.clone().requires_grad_()
        y = gs.qkv_norm_rotary(x, 2, 1, table, None, *w, norm=norm, interleaved=interleaved)
        got = torch.autograd.grad(y, [x] + (w if norm else []), grads)
        return torch.cat([o.detach() for o in y], 1).transpose(1, 2), got[0], got[1:]

    y, dx, dw = run(x, grads)
    t = torch.arange(T, device=gpu)
    head, f = 1 + t % 2, n_rot + t
    at = (1, t, head, f)                           # sample 1 alone
    xb = x.clone()
    xb[at] = bad
    got, got_dx, _ = run(xb, grads)
    row = torch.zeros(B, T, sum(heads), dtype=torch.bool, device=gpu)
    row[1, t, head] = True
    want = y.clone()
    if norm:                                       # an infinite row length
        want[row] = math.nan if math.isnan(bad) else 0.0
        want[at] = math.nan
    else:
        want[at] = bad
    same(got, want, "forward")
    if not norm:
        same(got_dx, dx, "gradient of a row that was not read")
    else:
        same(got_dx[~row], dx[~row], "gradient of other rows")
    gb = [g.clone() for g in grads]
    gb[0][1, 1, t[::2], f[::2]] = bad
    gb[1][1, 0, t[1::2], f[1::2]] = bad
    got, got_dx, got_dw = run(x, gb)
    same(got, y, "forward of the same")
    if norm:
        same(got_dx[~row], dx[~row], "gradient of other rows")
        assert not got_dx[row].isfinite().any()
        for part in range(2):
            hit = torch.zeros(D, dtype=torch.bool, device=gpu)
            hit[f[part::2]] = True
            assert not got_dw[part][hit].isfinite().any()
            same(got_dw[part][~hit], dw[part][~hit], "gradient of other weights")
    else:
        want = dx.clone()
        want[at] = bad
        same(got_dx, want, "gradient")


@pytest.mark.parametrize("n_rot", [0, 16, 48])
def test_qk_rotated_features_of_a_bad_row_alone(gpu, n_rot):
    """A position outside the table: NaN in the rotated features, the others as at any position."""
    D, x = 48, randn((1, 3, 3 * 48), 1).to(gpu)
    table = gs.rotary_table(4, n_rot, device=gpu)
    for interleaved in (False, True):
        y = [gs.qkv_norm_rotary(x, 1, 1, table, torch.tensor(p, device=gpu), interleaved=interleaved)
             for p in ([0, 1, 2], [0, 9, 2])]
        for a, b in zip(y[0][:2], y[1][:2]):
            assert b[:, :, 1, :n_rot].isnan().all()
            same(b[:, :, 1, n_rot:], a[:, :, 1, n_rot:], "not rotated")
            same(b[:, :, ::2], a[:, :, ::2], "other tokens")


def _calls(gpu):
    """(outputs, inputs) of each operator."""
    w = randn((9, 8), 1).to(gpu).requires_grad_()
    yield [gs.embedding_lookup(torch.arange(5, device=gpu), w, 2.0)], [w]
    big = torch.arange(600, device=gpu) % 9        # more tokens than one launch sums
    yield [gs.embedding_lookup(big, w, 2.0)], [w]
    x = randn((2, 3, 4 * 16), 2).to(gpu).requires_grad_()
    q = torch.ones(16, device=gpu, requires_grad=True)
    yield list(gs.qkv_norm_rotary(x, 2, 1, gs.rotary_table(3, 16, device=gpu), None, q, q)), [x, q]
    z = randn((4, 31), 3).to(gpu).requires_grad_()
    ids, t = torch.arange(8, device=gpu).view(4, 2), randn((4, 2), 4).to(gpu)
    for reduction in ("none", "mean"):
        yield [gs.distillation_loss(z, ids, t, temperature=2.0, reduction=reduction)], [z]


def test_output_gradients_that_are_not_their_memory(gpu):
    """Zeros that are only marked, and signs that are only marked, as complex torch code gives them."""
    for outs, inputs in _calls(gpu):
        g = [torch.randn_like(o) for o in outs]
        for marked in ([torch._efficientzerotensor(o.shape, device=gpu) for o in outs],
                       [torch.complex(x, x).conj().imag for x in g]):
            written = [m.clone().resolve_neg() + 0.0 if m.is_neg() else torch.zeros(m.shape, device=gpu)
                       for m in marked]
            got = torch.autograd.grad(outs, inputs, marked, retain_graph=True)
            want = torch.autograd.grad(outs, inputs, written, retain_graph=True)
            for a, b in zip(got, want):
                same(a, b, "gradient")
    x = randn((2, 3, 4 * 16), 2).to(gpu).requires_grad_()
    y = gs.qkv_norm_rotary(x, 2, 1, gs.rotary_table(3, 16, device=gpu))[0]
    c = torch.randn(2, 2, 3, 16, dtype=torch.complex64, device=gpu)
    got, = torch.autograd.grad(torch.view_as_real(torch.complex(y, y).conj() * c).sum(), x)
    y = gs.qkv_norm_rotary(x, 2, 1, gs.rotary_table(3, 16, device=gpu))[0]
    z = torch.complex(y, -y) * c
    want, = torch.autograd.grad(z.real.sum() + z.imag.sum(), x)
    torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-6)


def _loss64(z, ids, t, labels, tau, alpha):
    z, t = z.double().cpu().requires_grad_(), t.double().cpu()
    rows, _ = L.distill_rows(z, ids.cpu(), t, labels.cpu(), tau, alpha)
    return rows.detach(), torch.autograd.grad(rows.sum(), z)[0]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("tau", [0.25, 0.4, 0.5, 1.0, 3.0])
@pytest.mark.parametrize("V", [29, 5000, 50257])
def test_distill_teacher_entries_at_masked_logits(gpu, dtype, tau, V):
    """The student's logits at some or all of the teacher's ids are the type's lowest value: losses of
    the order of that value, finite where they are in the type."""
    N, K = 6, 4
    z, t = randn((N, V), 1, 2.0, dtype), randn((N, K), 2, 2.0, dtype)
    ids = torch.stack([torch.randperm(V, generator=gen(n))[:K] for n in range(N)])
    low = torch.finfo(dtype).min
    z[0, ids[0, 0]] = low
    z[1, ids[1]] = low
    z[2] = low
    z[2, 3] = 1.0
    z[3, ids[3, 1:]] = low / 64
    z[4] = low / 64
    z[4, ids[4, 0]] = 0.0
    labels = ids[:, 0].contiguous()
    for alpha in (1.0, 0.25):
        zg = z.to(gpu).requires_grad_()
        loss = gs.distillation_loss(zg, ids.to(gpu), t.to(gpu), labels.to(gpu), temperature=tau,
                                    alpha=alpha, reduction="none")
        g, = torch.autograd.grad(loss, zg, torch.ones_like(loss))
        want, dwant = _loss64(z, ids, t, labels, tau, alpha)
        # within the comparison's 1e-5 of the largest number either side of it is right
        top = torch.finfo(FP32).max
        fits = want < top * (1 - 1e-5)
        assert fits[0] and fits[5]
        # a loss is K shares times differences of logits, all positive: some tens of roundings each
        off = (loss.double().cpu() - want).abs()
        assert (off <= 1e-5 * want.abs() + 1e-5)[fits].all(), (off, want)
        assert loss.cpu()[want > top * (1 + 1e-5)].isinf().all() and not loss.isnan().any()
        # shares and their differences from sums of exponentials: see the bound's smallest terms
        assert ((g.double().cpu() - dwant).abs() <= dwant.abs() * 2 ** -8 * (dtype == BF16) +
                2e-5).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("tau", [1e-37, 1e-30, 1e-23, 1e-20, 1e-12, 1e-6, 1e3, 1e9])
def test_distill_far_temperatures(gpu, dtype, tau):
    """Close to zero the shares are one and zero, the loss tau times a difference of logits."""
    N, V, K = 5, 301, 6
    z, t = randn((N, V), 3, 2.0, dtype), randn((N, K), 4, 2.0, dtype)
    ids = torch.stack([torch.randperm(V, generator=gen(n))[:K] for n in range(N)])
    labels = ids[:, 0].contiguous()
    zg = z.to(gpu).requires_grad_()
    loss = gs.distillation_loss(zg, ids.to(gpu), t.to(gpu), labels.to(gpu), temperature=tau,
                                reduction="none")
    g, = torch.autograd.grad(loss, zg, torch.ones_like(loss))
    tau32 = float(torch.tensor(tau, dtype=FP32))
    want, dwant = _loss64(z, ids, t, labels, tau32, 1.0)
    # tau^2 log(V / K) and above; a logarithm's rounding counts tau^2 times, a difference's tau times
    off = (loss.double().cpu() - want).abs()
    assert (off <= 1e-5 * (want.abs() + tau32 ** 2)).all(), (off, want)
    # an element is tau times a difference of shares up to one
    assert ((g.double().cpu() - dwant).abs() <= tau32 * (2 ** -8 * (dtype == BF16) + 2e-5)).all()


@pytest.mark.parametrize("index", [(slice(None), -1), (slice(None), slice(3, None, 100)),
                                   (slice(None, None, 8), slice(5, 9))])
def test_distill_of_few_rows_of_large_logits(gpu, index):
    """The last positions of a batch, every hundredth, a few of some samples: scratch and gradient of the
    size of the rows, not of what lies between them; as for a copy of the rows."""
    whole = torch.zeros(32, 400, 8192, dtype=BF16, device=gpu)
    z = whole[index]
    z.copy_(randn(z.shape, 1, 2.0, BF16))
    ids = torch.randint(0, 8192, (*z.shape[:-1], 5), generator=gen(2)).to(gpu)
    t = randn(ids.shape, 3).to(gpu)
    labels = torch.randint(0, 8192, z.shape[:-1], generator=gen(4)).to(gpu)

    def run(z):
        z = z.detach().requires_grad_()
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        loss = gs.distillation_loss(z, ids, t, labels, temperature=2.0, alpha=0.5)
        got = torch.autograd.grad(loss, z, retain_graph=True)[0]
        again = torch.autograd.grad(loss, z, torch.tensor(0.5, device=gpu))[0]
        return loss.detach(), got, again, torch.cuda.max_memory_allocated() - before

    loss, got, again, peak = run(z)
    assert peak < 8 * z.numel() * 2 + (1 << 22)     # a few copies of the rows
    want = run(z.clone().contiguous())
    same(loss, want[0], "loss")
    same(got, want[1], "gradient")
    same(again, want[2], "gradient of half the loss")
