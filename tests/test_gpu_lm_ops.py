"""The language-model operators on the GPU against float64 forms (tests/lm_forms.py).

Tolerances are error bounds of the arithmetic, elementwise: an output rounded to type t is off by
at most HALF[t] of its value; a sum of n fp32 terms by at most n U of the sum of their magnitudes
(U = 2^-24); the rest is counted where it stands.
"""
import math

import pytest
import torch

import ghostsuite_amd as gs
from ghostsuite_amd import GradDotProdEngine, _native
from ghostsuite_amd.workloads import CausalLM, LMConfig
from tests import lm_forms as L
from tests.helpers import gen, randn
from tests.lm_forms import HALF, U, f64

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


def within(got, want, bound, what=""):
    """|got - want| <= bound elementwise; NaN and infinities in the same places."""
    got, bound = f64(got), bound.expand_as(want)
    fine = want.isfinite()
    assert torch.equal(fine, got.isfinite()), f"{what}: not finite in other places"
    assert torch.equal(want.isnan(), got.isnan()), f"{what}: NaN in other places"
    off = (got - want).abs()[fine]
    over = off > bound[fine]
    assert not over.any(), (f"{what}: {int(over.sum())} of {over.numel()} over the bound, worst "
                            f"{(off / bound[fine].clamp(min=1e-300)).max():.3g} of it")


# ------------------------------------------------------------------------------- embedding
def check_lookup(ids, weight, scale, padding_idx, gpu, seed):
    w = weight.to(gpu).requires_grad_()
    y = gs.embedding_lookup(ids.to(gpu), w, scale, padding_idx)
    want = L.lookup(ids, f64(weight), scale)
    t = weight.dtype
    # the fp32 product, then the output's rounding
    within(y, want, want.abs() * (HALF[t] + 2 * U) * (1 + 1e-3), "rows")
    assert torch.equal(gs.embedding_lookup(ids.to(gpu), w.detach(), scale, padding_idx), y)
    g = randn(y.shape, seed + 1, 1.0, t)
    got, = torch.autograd.grad(y, w, g.to(gpu))
    assert got.dtype == t and got.shape == weight.shape
    want, mag, n = L.lookup_grad(ids, f64(g), weight.shape[0], scale, padding_idx)
    within(got, want, want.abs() * HALF[t] * (1 + 1e-3) + (n[:, None] + 4) * U * mag, "gradient")
    return y, got


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape,vocab,d", [
    ((1,), 1, 1), ((3,), 7, 8), ((2, 5), 11, 64), ((4, 33), 100, 40), ((2, 3, 7), 50, 515),
    ((1, 1025), 300, 96), ((8, 1), 50257, 768), ((5, 129), 2000, 1030), ((700,), 5, 33)])
def test_lookup_and_gradient(gpu, dtype, shape, vocab, d):
    ids = torch.randint(0, vocab, shape, generator=gen(d))
    check_lookup(ids, randn((vocab, d), 1, 1.0, dtype), math.sqrt(d), None, gpu, 5)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("d", [1, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33, 100, 257])
@pytest.mark.parametrize("off", [0, 1, 2, 4])
def test_lookup_rows_off_16_byte_boundaries(gpu, dtype, d, off):
    """Every width around a piece, the table at other places than allocations start at."""
    w = randn((off + 19 * d,), d, 1.0, dtype).to(gpu)[off:].view(19, d)
    for n in (1, 2, 37, 700):
        ids = torch.randint(-1, 20, (n,), generator=gen(n))
        y = gs.embedding_lookup(ids.to(gpu), w, 1.5)
        want = torch.where(((ids >= 0) & (ids < 19))[:, None], f64(w)[ids.clamp(0, 18)] * 1.5, 0.0)
        within(y, want, want.abs() * (HALF[dtype] + U), "rows")


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n", [2, 63, 65, 255, 256, 257])
@pytest.mark.parametrize("d", [3, 64, 333, 1100])
@pytest.mark.parametrize("ids", ["all", "one", "few", "outside"])
def test_lookup_gradient_around_its_two_ways(gpu, dtype, n, d, ids):
    """Up to 256 tokens are summed without a sort: ids spread, all the same, a dozen, or extreme."""
    vocab = 1003
    x = {"all": torch.randint(0, vocab, (n,), generator=gen(n)), "one": torch.full((n,), vocab - 1),
         "few": torch.randint(0, 12, (n,), generator=gen(n)) * 90,
         "outside": torch.tensor([0, -1, vocab, 2 ** 63 - 1, -2 ** 63, 7, 2 ** 32 + 7]).repeat(
             n // 7 + 1)[:n]}[ids]
    check_lookup(x, randn((vocab, d), 1, 1.0, dtype), 1.7, None, gpu, n + d)


@pytest.mark.parametrize("id_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("padding_idx", [None, 0, 3, -1])
def test_lookup_padding_strides_and_ids_outside(gpu, id_dtype, padding_idx):
    ids = torch.randint(-3, 23, (6, 70), generator=gen(1)).to(id_dtype)
    ids[0, :4] = torch.tensor([0, 3, 19, -100])
    if id_dtype == torch.int64:
        ids[1, 0], ids[1, 1] = 2 ** 40, -2 ** 40
    for view in (ids, ids.t(), ids[:, ::3]):
        check_lookup(view, randn((20, 24), 1, 1.0, BF16), 0.37, padding_idx, gpu, 7)
    with pytest.raises(_native.GhostHipError, match="padding_idx"):
        gs.embedding_lookup(ids.to(gpu), randn((20, 24), 1).to(gpu), 1.0, 20)


def test_lookup_empty_strided_and_refused(gpu):
    w = randn((9, 8), 1).to(gpu).requires_grad_()
    y = gs.embedding_lookup(torch.empty((2, 0), dtype=torch.int64, device=gpu), w, 2.0)
    assert y.shape == (2, 0, 8)
    assert (torch.autograd.grad(y, w, torch.empty_like(y))[0] == 0).all()
    # a transposed table and a broadcast gradient
    wt = randn((8, 9), 2).to(gpu).t().requires_grad_()
    ids = torch.tensor([0, 5, 5], device=gpu)
    y = gs.embedding_lookup(ids, wt, 2.0)
    assert torch.equal(y, 2.0 * wt[ids])
    got, = torch.autograd.grad(y.sum(), wt)
    assert got[5].tolist() == [4.0] * 8 and got[0].tolist() == [2.0] * 8 and (got[1] == 0).all()
    for bad in (dict(weight=w.half()), dict(weight=w[0]), dict(ids=ids.float()),
                dict(ids=ids.cpu())):
        with pytest.raises(_native.GhostHipError):
            gs.embedding_lookup(**{"ids": ids, "weight": w, **bad})


def test_lookup_beyond_32_bit_offsets(gpu):
    """Rows past 2^31 elements of the table, and an output of more than 2^31 elements."""
    vocab, d = (1 << 21) + 3, 1032
    w = torch.zeros(vocab, d, dtype=BF16, device=gpu)
    w[-1], w[-2] = 3.0, 5.0
    ids = torch.full((vocab,), vocab - 2, device=gpu)
    ids[-1] = vocab - 1
    y = gs.embedding_lookup(ids, w, 2.0)
    assert y.numel() > 2 ** 31
    assert (y[-1] == 6.0).all() and (y[-2] == 10.0).all() and (y[0] == 10.0).all()


def test_lookup_of_more_pieces_than_a_launch_has_threads(gpu):
    """Rows shorter than 16 bytes: 2^33 single elements and more, in several launches."""
    d, n = 7, (1 << 33) // 7 + 5
    w = randn((3, d), 1, 1.0, BF16).to(gpu)
    ids = torch.arange(n, dtype=torch.int32, device=gpu) % 4     # 3: outside
    y = gs.embedding_lookup(ids, w, 1.0)
    assert y.numel() > 1 << 33
    rows = torch.cat((w, torch.zeros_like(w[:1])))
    for i in [*range(0, n, n // 9), n - 1000]:
        assert torch.equal(y[i:i + 1000], rows[ids[i:i + 1000].long()])


# ------------------------------------------------------------ norms, rotation, heads first
def qk_bounds(plan, parts, qw, kw, grads):
    """Error bounds (of y per part, dx per part, and of dq, dk the magnitude of their addends).

    r's relative error: D + 2 additions and products of the mean square, halved by the root, and
    its own rounding: (D / 2 + 4) U; with the weight, the table's rounding, the two products and
    the sum of a rotation: (D / 2 + 12) U of |u_a c| + |u_b s| <= |u_a| + |u_b|.  The gradient's
    mean(w h x r) is another sum of D products: (D + 24) U more of its own magnitude."""
    xs = L.split_heads(plan, [f64(p) for p in parts])
    B, T, _, D = xs[0].shape
    ones = torch.ones(D, dtype=torch.float64)
    ws = [ones if w is None else f64(w) for w in (qw, kw)]
    n = plan["table"].shape[-1]

    def mixed(a):   # |a| + |its pair's| on the rotated features
        a = a.abs().nan_to_num(0.0)
        r, rest = a[..., :2 * n], a[..., 2 * n:]
        if plan["interleaved"]:
            p = r.unflatten(-1, (n, 2)).flip(-1).flatten(-2)
        else:
            p = r.roll(n, -1)
        return torch.cat((r + p, rest), -1)

    fwd, bwd, addends = [], [], []
    for i, x in enumerate(xs):
        if x is None:
            continue
        g = None if grads is None or grads[i] is None else f64(grads[i]).transpose(1, 2)
        if i == 2:
            fwd.append(torch.zeros_like(x).transpose(1, 2))
            bwd.append(None if g is None else torch.zeros_like(x))
            continue
        r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + plan["eps"]) if plan["norm"] else 1.0
        fwd.append((mixed(x * r * ws[i]) * (D / 2 + 12) * U).transpose(1, 2))
        if g is None:
            bwd.append(None), addends.append(None)
            continue
        h = mixed(g)
        if plan["norm"]:
            xn = (x * r).abs()
            m = (ws[i].abs() * h * xn).mean(-1, keepdim=True)
            bwd.append(r * (ws[i].abs() * h * (D / 2 + 16) + xn * m * (2.5 * D + 40)) * U)
            addends.append((h * xn).sum((0, 1, 2)))
        else:
            bwd.append(h * 8 * U)
    return fwd, bwd, addends


def check_qk(gpu, plan, parts, qw, kw, grads=None, weights=True):
    """Forward, and with grads ([None or heads-first gradients], GPU tensors) backward."""
    call = dict(norm=plan["norm"], eps=plan["eps"], interleaved=plan["interleaved"])
    heads, t = plan["heads"], parts[0].dtype
    args = (plan["table"], plan["positions"], qw, kw)
    if len(parts) == 1:
        y = gs.qkv_norm_rotary(parts[0], heads[0], heads[1], *args, **call)
    else:
        y = gs.qk_norm_rotary(*parts, *args, **call)
    want = L.qk_all(plan, [f64(p) for p in parts], f64(qw), f64(kw))
    fwd, bwd, addends = qk_bounds(plan, parts, qw, kw, grads)
    for o, w, b in zip(y, want, fwd):
        assert o.dtype == t and o.is_contiguous()
        within(o, w, b + w.abs().nan_to_num(0.0) * HALF[t], "forward")
    if grads is None:
        return y
    inputs = [*parts] + ([qw, kw] if weights and qw is not None else [])
    pairs = [(o, g) for o, g in zip(y, grads) if g is not None]
    got = torch.autograd.grad([o for o, _ in pairs], inputs, [g for _, g in pairs])
    dx, dq, dk = L.qk_grads(plan, parts, qw, kw, grads)
    for got_x, want_x, part in zip(L.split_heads(plan, got[:len(parts)]),
                                   L.split_heads(plan, dx), range(3)):
        if got_x is None:
            continue
        b = bwd[part] if bwd[part] is not None else torch.zeros_like(want_x)
        within(got_x, want_x, b + want_x.abs().nan_to_num(0.0) * HALF[t], f"dx of part {part}")
    if len(inputs) > len(parts):
        rows = parts[0].shape[0] * parts[0].shape[1]
        for g, w, a, w64, h in zip(got[-2:], (qw, kw), addends, (dq, dk), heads):
            assert g.dtype == w.dtype
            D = w.numel()
            a = torch.zeros(D, dtype=torch.float64) if a is None else a
            within(g, w64, (rows * h + D / 2 + 24) * U * a + w64.abs() * HALF[w.dtype],
                   "weight gradient")
    return y


def qk_inputs(gpu, B, T, heads, D, dtype, seed, w_dtype=None):
    x = (randn((B, T, sum(heads) * D), seed) * (0.2 + torch.rand(B, T, 1, generator=gen(seed)))
         ).to(dtype).to(gpu).requires_grad_()
    qw, kw = ((1 + 0.2 * randn((D,), seed + k)).to(w_dtype or dtype).to(gpu).requires_grad_()
              for k in (1, 2))
    grads = [randn((B, h, T, D), seed + 3 + i, 1.0, dtype).to(gpu) for i, h in enumerate(heads)]
    return x, qw, kw, grads


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,heads,D,n_rot", [
    (1, 1, (1, 1, 1), 64, 64), (2, 5, (3, 1, 1), 64, 64), (1, 70, (4, 2, 2), 128, 128),
    (3, 17, (2, 2, 2), 256, 64), (2, 9, (5, 1, 1), 80, 20), (2, 33, (1, 1, 1), 33, 32),
    (1, 3, (2, 1, 1), 1, 0), (2, 4, (2, 1, 1), 2, 2), (2, 7, (3, 3, 3), 48, 0),
    (1, 300, (2, 1, 1), 20, 6), (2, 5, (2, 1, 1), 512, 512), (1, 4, (2, 1, 1), 511, 302),
    (1, 6, (2, 1, 1), 100, 50), (4, 260, (12, 12, 12), 64, 64), (2, 40, (9, 3, 3), 96, 94),
    (1, 20011, (3, 1, 1), 64, 32), (2, 9001, (2, 7, 7), 128, 128)])
def test_qkv_shapes(gpu, dtype, interleaved, B, T, heads, D, n_rot):
    plan = L.plan(heads, gs.rotary_table(T + 3, n_rot, device=gpu), interleaved=interleaved)
    x, qw, kw, grads = qk_inputs(gpu, B, T, heads, D, dtype, 11)
    check_qk(gpu, plan, (x,), qw, kw, grads)


@pytest.mark.parametrize("dtype,w_dtype", [(BF16, FP32), (FP32, BF16)])
def test_qk_weights_of_another_dtype_and_none(gpu, dtype, w_dtype):
    heads = (4, 2, 2)
    plan = L.plan(heads, gs.rotary_table(20, 32, device=gpu))
    x, qw, kw, grads = qk_inputs(gpu, 2, 13, heads, 64, dtype, 3, w_dtype)
    check_qk(gpu, plan, (x,), qw, kw, grads)
    check_qk(gpu, plan, (x,), None, None, grads)
    check_qk(gpu, dict(plan, norm=False), (x,), None, None, grads)
    y = gs.qkv_norm_rotary(x, 4, 2, plan["table"], None, qw, None)   # one weight only
    got = torch.autograd.grad(y, (x, qw), grads)
    assert all(g.isfinite().all() for g in got)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("off", [1, 2, 3, 4, 8])
def test_qk_table_and_weights_off_16_byte_boundaries(gpu, dtype, interleaved, off):
    def moved(t):
        return torch.cat((t.new_zeros(off), t.detach().flatten()))[off:].view(t.shape)

    heads = (2, 1, 1)
    x, qw, kw, grads = qk_inputs(gpu, 2, 5, heads, 64, dtype, 31)
    plan = L.plan(heads, moved(gs.rotary_table(9, 64, device=gpu)), interleaved=interleaved)
    check_qk(gpu, plan, (x,), qw, kw, grads)
    plan = L.plan(heads, gs.rotary_table(9, 64, device=gpu), interleaved=interleaved)
    check_qk(gpu, plan, (x,), moved(qw).requires_grad_(), moved(kw).requires_grad_(), grads)


@pytest.mark.parametrize("pos_dtype", [torch.int32, torch.int64])
def test_qk_positions(gpu, pos_dtype):
    heads, B, T, D = (3, 1, 1), 4, 9, 64
    table = gs.rotary_table(32768, 40, device=gpu)
    x, qw, kw, grads = qk_inputs(gpu, B, T, heads, D, FP32, 5)
    far = torch.randint(0, 32768, (B, T), generator=gen(1)).to(pos_dtype).to(gpu)
    for pos in (far, far[0], far[:1], far[1].expand(B, T), far.t().contiguous().t(),
                torch.stack((far, far), -1)[..., 1]):
        check_qk(gpu, L.plan(heads, table, pos), (x,), qw, kw, grads)
    edge = far.clone()
    edge[0, 0], edge[1, 1], edge[2, 2] = 32768, -1, 32767
    y = gs.qkv_norm_rotary(x, 3, 1, table, edge, qw, kw)
    want = L.qk_all(L.plan(heads, table, edge), (f64(x),), f64(qw), f64(kw))
    for o, w in zip(y, want):
        assert torch.equal(f64(o).isnan(), w.isnan())
    assert y[0][0, :, 0, :40].isnan().all() and y[0][0, :, 0, 40:].isfinite().all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_qk_strides_and_separate_tensors(gpu, dtype):
    """Slices of wider tensors, heads before tokens, odd offsets, and gradients in the layouts
    attention gives: every one against the contiguous form."""
    B, T, D = 2, 11, 64
    heads = (4, 2, 2)
    table = gs.rotary_table(16, 64, device=gpu)
    plan = L.plan(heads, table)
    x, qw, kw, grads = qk_inputs(gpu, B, T, heads, D, dtype, 21)
    wide = torch.randn(B, T, 8 * D + 24, generator=gen(2)).to(dtype).to(gpu)
    odd = torch.randn(B * T * 8 * D + 1, generator=gen(3)).to(dtype).to(gpu)
    views = [wide[..., 8:8 + 8 * D], wide[..., 3:3 + 8 * D], odd[1:].view(B, T, 8 * D),
             x.detach().transpose(0, 1).contiguous().transpose(0, 1),
             x.detach().view(B, T, 8, D).transpose(1, 2).contiguous().transpose(1, 2),
             x.detach().view(B, T, 8, D).transpose(2, 3).contiguous().transpose(2, 3)]
    tfirst = [g.transpose(1, 2).contiguous().transpose(1, 2) for g in grads]
    spread = [torch.stack((g, g), -1)[..., 0] for g in grads]       # features apart
    for v in views:
        for gr in (grads, tfirst, spread):
            check_qk(gpu, plan, (v.requires_grad_(),), qw, kw, gr)
    q, k = (wide[..., :4 * D].unflatten(-1, (4, D)).detach().requires_grad_(),
            wide[..., 4 * D + 5:6 * D + 5].unflatten(-1, (2, D)).detach().requires_grad_())
    two = L.plan((4, 2, 0), table)
    check_qk(gpu, two, (q, k), qw, kw, grads[:2])
    check_qk(gpu, two, (q, k), qw, kw, [grads[0], None], weights=False)


def test_qk_missing_and_broadcast_gradients(gpu):
    heads = (3, 1, 1)
    plan = L.plan(heads, gs.rotary_table(8, 16, device=gpu))
    x, qw, kw, grads = qk_inputs(gpu, 2, 6, heads, 32, FP32, 31)
    for keep in ((0,), (1,), (2,), (0, 2)):
        check_qk(gpu, plan, (x,), qw, kw, [g if i in keep else None for i, g in enumerate(grads)],
                 weights=False)
    one = [torch.full((), 0.5, device=gpu).expand(2, h, 6, 32) for h in heads]
    check_qk(gpu, plan, (x,), qw, kw, one)


def test_qk_zero_rows_infinities_and_empty(gpu):
    heads = (2, 1, 1)
    table = gs.rotary_table(8, 16, device=gpu)
    plan = L.plan(heads, table)
    x, qw, kw, grads = qk_inputs(gpu, 1, 5, heads, 32, FP32, 41)
    with torch.no_grad():
        x[0, 0, :32] = 0.0               # a row of zeros: eps alone
        x[0, 1, 40] = math.nan           # one row of NaN
        x[0, 2, 100] = math.inf          # a value's infinity is copied
    check_qk(gpu, plan, (x,), qw, kw, [None, None, grads[2]], weights=False)
    y = gs.qkv_norm_rotary(x, 2, 1, table, None, qw, kw)
    got, = torch.autograd.grad(y, x, grads)
    bad = got.view(5, 4, 32).isnan().any(-1)
    assert bad.nonzero().tolist() == [[1, 1]]
    for B, T in ((0, 5), (2, 0)):
        e = torch.empty(B, T, 4 * 32, device=gpu, requires_grad=True)
        y = gs.qkv_norm_rotary(e, 2, 1, table, None, qw, kw)
        assert [o.shape for o in y] == [(B, 2, T, 32), (B, 1, T, 32), (B, 1, T, 32)]
        de, dq = torch.autograd.grad(y, (e, qw), [torch.empty_like(o) for o in y])
        assert de.shape == e.shape and (dq == 0).all()


def test_qk_gradient_against_differences(gpu):
    heads = (2, 1, 1)
    plan = L.plan(heads, gs.rotary_table(16, 8, device=gpu), interleaved=True)
    x, qw, kw, grads = qk_inputs(gpu, 2, 5, heads, 12, FP32, 51)
    y = gs.qkv_norm_rotary(x, 2, 1, plan["table"], None, qw, kw, interleaved=True)
    got = [f64(g) for g in torch.autograd.grad(y, (x, qw, kw), grads)]
    at = [f64(v) for v in (x, qw, kw)]

    def value(v):
        return sum((o * f64(g)).sum() for o, g in zip(L.qk_all(plan, (v[0],), v[1], v[2]), grads))
    for i in range(3):
        d = randn(at[i].shape, 60 + i).double()
        lo, hi = ([a + s * 1e-6 * d if j == i else a for j, a in enumerate(at)] for s in (-1, 1))
        want = (value(hi) - value(lo)) / 2e-6
        # fp32 gradients: 64 U of every product's magnitude
        assert abs((got[i] * d).sum() - want) <= 64 * U * (got[i] * d).abs().sum() + 1e-7


def test_qk_refusals(gpu):
    table = gs.rotary_table(8, 16, device=gpu)
    x = torch.zeros(2, 5, 4 * 32, device=gpu)
    ok = dict(qkv=x, n_head=2, n_kv_head=1, table=table)
    for bad in (dict(qkv=x.half()), dict(qkv=x[..., :-1]), dict(qkv=x.view(2, 5, 2, 64)),
                dict(n_head=0), dict(n_kv_head=0), dict(table=table.to(BF16)),
                dict(table=gs.rotary_table(8, 34, device=gpu)), dict(table=table[:, :1]),
                dict(table=table.transpose(0, 1)), dict(table=table.cpu()),
                dict(q_weight=torch.ones(31, device=gpu)),
                dict(q_weight=torch.ones(32, device=gpu).half()),
                dict(q_weight=torch.ones(32)), dict(eps=-1.0), dict(eps=math.nan),
                dict(positions=torch.arange(4, device=gpu)),
                dict(positions=torch.arange(5, device=gpu).float()),
                dict(positions=torch.zeros(3, 5, dtype=torch.int64, device=gpu)),
                dict(positions=torch.arange(5)),
                dict(qkv=torch.zeros(1, 2, 4 * 513, device=gpu))):
        with pytest.raises(_native.GhostHipError):
            gs.qkv_norm_rotary(**{**ok, **bad})
    q = torch.zeros(2, 5, 2, 32, device=gpu)
    for k in (q[:1], q[..., :16], q.to(BF16)):
        with pytest.raises(_native.GhostHipError):
            gs.qk_norm_rotary(q, k, table)


def test_qk_beyond_32_bit_offsets(gpu):
    """A batch of more than 2^31 elements: its first and last tokens as alone."""
    B, T, heads, D = 3, 349526, (14, 1, 1), 128
    assert B * T * sum(heads) * D > 2 ** 31
    table = gs.rotary_table(T, D, device=gpu)
    x = torch.zeros(B, T, sum(heads) * D, dtype=BF16, device=gpu)
    for b, t in ((0, 0), (2, T - 1)):
        x[b, t] = randn((sum(heads) * D,), b + 1).to(BF16).to(gpu)
    q, k, v = gs.qkv_norm_rotary(x, 14, 1, table)
    for b, t in ((0, 0), (2, T - 1)):
        alone = gs.qkv_norm_rotary(x[b:b + 1, t:t + 1], 14, 1, table,
                                   torch.tensor([t], device=gpu))
        for o, a in zip((q, k, v), alone):
            assert torch.equal(o[b, :, t], a[0, :, 0])


# ----------------------------------------------------------- the norm weights' dot products
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("B,n_val,T,heads,D,n_rot,val_start", [
    (2, 1, 1, (1, 1, 1), 64, 64, None), (5, 2, 33, (4, 1, 1), 128, 64, None),
    (7, 3, 300, (2, 2, 2), 80, 20, 0), (6, 1, 9, (3, 3, 3), 33, 10, 2),
    (40, 30, 3, (2, 1, 1), 48, 48, 5), (3, 1, 7001, (5, 1, 1), 64, 32, None),
    (65533, 2, 1, (260, 1, 1), 2, 2, None), (128, 100, 2, (2, 1, 1), 70, 70, 20),
    (129, 3, 2, (2, 1, 1), 130, 8, 64)])
def test_qk_dots(gpu, dtype, B, n_val, T, heads, D, n_rot, val_start):
    plan = L.plan(heads, gs.rotary_table(T, n_rot, device=gpu))
    x, qw, kw, grads = qk_inputs(gpu, B, T, heads, D, dtype, 71)
    x = x.detach()
    got = _native.ops().qk_norm_rotary_dots(x, None, heads, plan["table"], None, qw.detach(),
                                            kw.detach(), 1e-6, False, grads, n_val,
                                            val_start=val_start, grad_scale=0.25)
    check_dots(got, plan, x, qw, kw, grads, n_val, val_start)
    # the same from the sums that a layer's backward pass leaves
    samples = torch.full((2, B, D), math.nan, device=gpu)
    y = _native.ops().qk_norm_rotary(x.requires_grad_(), None, heads, plan["table"], None, qw, kw,
                                     True, 1e-6, False, samples)
    dx, dqw, dkw = torch.autograd.grad(y, (x, qw, kw), grads)
    got = _native.ops().qk_sample_dots(samples, qw.detach(), kw.detach(), n_val,
                                       val_start=val_start, grad_scale=0.25)
    check_dots(got, plan, x, qw, kw, grads, n_val, val_start)
    plain = gs.qkv_norm_rotary(x, heads[0], heads[1], plan["table"], None, qw, kw)
    assert torch.equal(dx, torch.autograd.grad(plain, x, grads)[0])
    _, dq, dk = L.qk_grads(plan, (x,), qw, kw, grads)
    addends = qk_bounds(plan, (x,), qw, kw, grads)[2]
    for g, want, mag, h in zip((dqw, dkw), (dq, dk), addends, heads):
        within(g, want, (B * T * h + D / 2 + 24) * U * mag + want.abs() * HALF[dtype], "total")


def check_dots(got, plan, x, qw, kw, grads, n_val, val_start):
    heads, (B, T) = plan["heads"], x.shape[:2]
    D, n_rot = L.grads_dim(plan, (x,)), 2 * plan["table"].shape[-1]
    _, dq, dk = L.qk_grads(plan, (x,), qw, kw, grads, per_sample=True)
    xs = L.split_heads(plan, (f64(x),))
    vs = B - n_val if val_start is None else val_start
    val = torch.zeros(B, dtype=torch.bool)
    val[vs:vs + n_val] = True
    for i, (s, w) in enumerate(((dq, qw), (dk, kw))):
        # addends' magnitudes per sample: |h| |x r| summed (the bound of |h|: both of a pair)
        h = f64(grads[i]).abs().transpose(1, 2)
        r = h[..., :n_rot]
        h = torch.cat((r + r.roll(n_rot // 2, -1), h[..., n_rot:]), -1)
        xn = (xs[i] / torch.sqrt((xs[i] ** 2).mean(-1, keepdim=True) + 1e-6)).abs()
        mag = (h * xn).sum((1, 2))
        err = (T * heads[i] + D / 2 + 24) * U * mag
        sv, ev, mv = s[val].sum(0), err[val].sum(0), mag[val].sum(0)
        bound = (err[~val] @ sv.abs() + mag[~val] @ ev +
                 (n_val + D) * U * (mag[~val] @ mv))
        within(got[i], s[~val] @ sv, bound, "dots")
        want = s[~val].sum(0) * 0.25
        within(got[2 + i], want, 0.25 * (err[~val].sum(0) + B * U * mag[~val].sum(0)) +
               want.abs() * HALF[w.dtype] * (1 + 1e-3), "train gradient")


# ------------------------------------------------------------------------------ distillation
def distill_inputs(N, V, K, seed, dtype, spread=3.0):
    g = gen(seed)
    z = (torch.randn(N, V, generator=g) * spread).to(dtype)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(N)])
    t = (torch.randn(N, K, generator=g) * 3).to(dtype)
    labels = torch.randint(0, V, (N,), generator=g)
    return z, ids, t, labels


def distill_bounds(z, ids, t, labels, tau, alpha):
    """Error bounds of each row's loss and of each element of the rows' gradients.

    An exponential's argument x (|x| <= R, the row's range over the temperature) is formed with
    two roundings and a constant's: 3 R U; the exponential itself 2 U; a sum of V of them adds a
    thread's own (at most 128 here) and about 20 more levels.  delta covers one such sum or
    quotient; a loss is made of logarithms of sums, of differences up to R, and of K products."""
    N, V = z.shape
    rows, grads = [], []
    for n in range(N):
        v, use = z[n], (ids[n] >= 0) & (ids[n] < V) & (t[n] != -math.inf)
        fin = v[v.isfinite()]
        R = (fin.max() - fin.min()) / min(tau, 1.0) if fin.numel() else 0.0
        tk = t[n][use] / tau
        tk = tk[tk.isfinite()]
        Rt = tk.max() - tk.min() if tk.numel() else 0.0
        delta = (3 * max(R, Rt) + 160) * U
        q, s = torch.softmax(v / tau, 0), torch.softmax(v, 0)
        P = torch.zeros(V, dtype=torch.float64)
        loss = 0.0
        if use.any():
            lp = torch.log_softmax(t[n][use] / tau, 0)
            p = lp.exp()
            P.index_add_(0, ids[n][use], p)
            lq = torch.log_softmax(v / tau, 0)[ids[n][use]]
            size = torch.where(p > 0, p * (lp.abs() + lq.abs() + R + Rt + math.log(V) + 2), 0.0)
            loss += alpha * tau ** 2 * size.sum() * (delta + (ids.shape[1] + 8) * U)
        else:
            q = q * 0
        if alpha != 1 and 0 <= int(labels[n]) < V:
            loss += (1 - alpha) * (R + math.log(V) + 2) * delta
        rows.append(torch.as_tensor(loss, dtype=torch.float64))
        one = torch.zeros(V, dtype=torch.float64)
        if alpha != 1 and 0 <= int(labels[n]) < V:
            one[int(labels[n])] = 1.0
        grads.append((alpha * tau * (q + P) + (1 - alpha) * (s + one)) *
                     (2 * delta + (ids.shape[1] + 16) * U))
    return torch.stack(rows), torch.stack(grads)


def check_distill(gpu, z, ids, t, labels, tau=1.0, alpha=1.0, reduction="mean", upstream=None,
                  ignore=-100, view=None):
    """Loss and gradient of [N, V] CPU logits (or of `view`, their GPU form of another shape)."""
    N, V = z.shape
    zg = z.to(gpu) if view is None else view
    zg = zg.detach().requires_grad_()
    lead = zg.shape[:-1]
    args = [ids.to(gpu).reshape(*lead, -1), t.to(gpu).reshape(*lead, -1),
            None if labels is None else labels.to(gpu).reshape(lead)]
    how = dict(temperature=tau, alpha=alpha, reduction=reduction, ignore_index=ignore)
    loss = gs.distillation_loss(zg, *args, **how)
    assert loss.dtype == FP32 and loss.shape == (lead if reduction == "none" else ())
    z64 = f64(z).requires_grad_()
    rows, kept = L.distill_rows(z64, ids, f64(t), labels, tau, alpha, ignore)
    want = L.reduced(rows, kept, reduction)
    b_rows, b_grad = distill_bounds(f64(z), ids, f64(t), labels, tau, alpha)
    b_rows = torch.where(kept, b_rows, 0.0) + rows.detach().abs().nan_to_num(0.0) * 4 * U
    n = int(kept.sum()) if reduction == "mean" else 1
    total = b_rows if reduction == "none" else \
        (b_rows.sum() + (N / 1024 + 24) * U * rows.detach().abs().nan_to_num(0.0).sum()) / max(n, 1)
    within(loss.reshape(want.shape), want.detach(), total, "loss")
    with torch.no_grad():   # without a gradient: the same values
        assert torch.equal(gs.distillation_loss(zg, *args, **how).nan_to_num(1e30),
                           loss.detach().nan_to_num(1e30))
    up = torch.ones(want.shape, dtype=torch.float64) if upstream is None else \
        torch.as_tensor(upstream, dtype=torch.float64).expand(want.shape)
    got, = torch.autograd.grad(loss, zg, up.float().to(gpu).reshape(loss.shape))
    assert got.dtype == z.dtype and got.shape == zg.shape
    dz, = torch.autograd.grad(want, z64, up)
    dz = torch.where(kept[:, None], dz, 0.0)
    per = up.abs() if reduction == "none" else (up.abs() / max(n, 1)).expand(N)
    b = torch.where(kept[:, None], b_grad * per[:, None], 0.0)
    within(got.reshape(N, V), dz, b.nan_to_num(0.0) + dz.abs().nan_to_num(0.0) * HALF[z.dtype] *
           (1 + 1e-3) + 2.0 ** -126, "gradient")
    assert (got.reshape(N, V)[~kept.to(gpu)] == 0).all()
    return loss, got


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("N,V,K", [
    (1, 1, 1), (3, 2, 2), (5, 7, 3), (4, 63, 5), (2, 64, 64), (3, 65, 7), (3, 1000, 1000),
    (7, 2051, 33), (2, 8193, 300), (3, 16385, 16), (2, 32767, 9), (3, 50257, 64), (2, 65537, 5),
    (2, 131073, 40), (1, 262147, 1024)])
def test_distill_sizes(gpu, dtype, N, V, K):
    z, ids, t, labels = distill_inputs(N, V, K, V + K, dtype)
    check_distill(gpu, z, ids, t, labels, 2.0, 0.5)
    check_distill(gpu, z, ids, t, labels, 1.0, 0.3, "sum", 0.37)


@pytest.mark.parametrize("tau", [1.0, 0.5, 3.7])
@pytest.mark.parametrize("alpha", [0.0, 0.25, 1.0])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("upstream", [None, 3.25])
def test_distill_options(gpu, tau, alpha, reduction, upstream):
    z, ids, t, labels = distill_inputs(9, 1003, 12, 5, BF16)
    labels[2] = labels[7] = -100
    check_distill(gpu, z, ids, t, labels, tau, alpha, reduction, upstream)
    if alpha == 1.0:
        check_distill(gpu, z, ids, t, None, tau, alpha, reduction, upstream)


@pytest.mark.parametrize("N", [63, 64, 65, 256, 257, 600])
@pytest.mark.parametrize("upstream", [None, -0.5])
def test_distill_mean_over_the_rows_that_count(gpu, N, upstream):
    """The rows are counted in two ways, by their number; from none ignored to all but one."""
    z, ids, t, labels = distill_inputs(N, 37, 3, N, FP32)
    for kept in (N, N // 2, 1):
        labels[kept:] = -100
        order = torch.randperm(N, generator=gen(kept))
        check_distill(gpu, z, ids, t, labels[order], 2.0, 0.5, "mean", upstream)


def test_distill_per_row_upstream_and_other_ignore_index(gpu):
    z, ids, t, labels = distill_inputs(6, 301, 4, 6, FP32)
    labels[1] = 7
    check_distill(gpu, z, ids, t, labels, 2.0, 0.5, "none",
                  torch.tensor([1.0, 2.0, 0.0, -3.0, 1e-3, 5.0]), ignore=7)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("V", [41, 301, 9000, 83001])
def test_distill_rows_with_little_or_nothing_left(gpu, dtype, V):
    """Teacher entries masked by id or by -inf, ids that stand several times (the label's among
    them), masked student logits, the lowest finite values, and NaN where nothing reads."""
    z, ids, t, labels = distill_inputs(15, V, 8, 7, dtype)
    ids[0] = -1                                   # no teacher, by id
    t[1] = -math.inf                              # no teacher, by logit
    t[2] = torch.finfo(dtype).min                 # all at the lowest value: even shares
    ids[3, 2:] = V                                # ids past the end
    ids[4] = 17                                   # one id for all
    ids[5, ::2], labels[5] = 40, 40               # half of them the label
    t[6, 0], ids[6, 0] = math.nan, -5             # NaN in a masked entry
    z[7] = -math.inf
    z[7, ids[7]] = 1.0                            # only the teacher's ids left
    labels[7] = ids[7, 0]
    z[8, :V // 2] = -math.inf
    z[8, ids[8, 0]], z[8, labels[8]] = 1.0, 2.0
    t[8, 1:] = -math.inf
    z[9], labels[9] = math.nan, -100              # an ignored row of NaN
    z[10] = -math.inf
    labels[10] = -100                             # an ignored row of nothing
    z[11] = torch.finfo(dtype).min                # a flat row
    t[12, 1:] = torch.finfo(dtype).min            # one entry takes all
    ids[13, 1] = 2 ** 40                          # far outside
    z[14] -= 400                                  # far below zero, masked from the first id on
    z[14, :V // 2] = -math.inf
    ids[14], labels[14] = torch.arange(V - 8, V), V - 1
    for tau, alpha in ((2.0, 0.5), (1.0, 1.0), (1.0, 0.5), (3.0, 0.0)):
        check_distill(gpu, z, ids, t, labels, tau, alpha)
        check_distill(gpu, z, ids, t, labels, tau, alpha, "none", 0.5)


def test_distill_infinities_where_they_count(gpu):
    """A teacher id whose student logit is -inf: an infinite loss, a finite gradient; a label
    outside the vocabulary, a NaN logit: NaN for that row alone; no row kept: NaN, no gradient."""
    z, ids, t, labels = distill_inputs(5, 77, 3, 8, FP32)
    z[0, ids[0, 1]] = -math.inf
    labels[0] = ids[0, 0]
    z[1, 5] = math.nan
    labels[2] = 77
    labels[3] = -1
    zg = z.to(gpu).requires_grad_()
    loss = gs.distillation_loss(zg, ids.to(gpu), t.to(gpu), labels.to(gpu), temperature=2.0,
                                alpha=0.5, reduction="none")
    assert loss[0] == math.inf and loss[1:4].isnan().all() and loss[4].isfinite()
    g, = torch.autograd.grad(loss, zg, torch.ones_like(loss))
    assert g[0].isfinite().all() and g[1:4].isnan().all() and g[4].isfinite().all()
    t[4, 1] = math.nan                            # a teacher entry that counts
    loss = gs.distillation_loss(zg, ids.to(gpu), t.to(gpu), labels.to(gpu), temperature=2.0,
                                alpha=0.5, reduction="none")
    g, = torch.autograd.grad(loss, zg, torch.ones_like(loss))
    assert loss[4].isnan() and g[4].isnan().all() and loss[0] == math.inf
    none = torch.full_like(labels, -100).to(gpu)
    loss = gs.distillation_loss(zg, ids.to(gpu), t.to(gpu), none)
    assert loss.isnan() and (torch.autograd.grad(loss, zg)[0] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_distill_strides_and_offsets(gpu, dtype):
    """Shifted, padded, transposed and odd-offset logits: as their contiguous copies."""
    B, T, V, K = 3, 5, 213, 6
    z, ids, t, labels = distill_inputs(B * T, V, K, 9, dtype)
    z3 = z.view(B, T, V).to(gpu)

    def place(shape, index):
        whole = torch.full(shape, math.nan, dtype=dtype, device=gpu)
        view = whole[index]
        view.copy_(z3.reshape(view.shape))
        return view
    s = slice
    views = [place((B, T + 1, V), (s(None), s(0, T))), place((B, T + 1, V), (s(None), s(1, None))),
             place((B, T, V + 11), (s(None), s(None), s(0, V))),
             place((B, T, V + 11), (s(None), s(None), s(3, V + 3))),
             place((B * T, V + 1), (s(None), s(1, None))),
             place((B, 2 * T, V), (s(None), s(None, None, 2))),
             z3.transpose(0, 1).contiguous().transpose(0, 1),
             z3.transpose(1, 2).contiguous().transpose(1, 2), z3.view(B, 1, T, V)]
    base = check_distill(gpu, z, ids, t, labels, 2.0, 0.4)
    for v in views:
        got = check_distill(gpu, z, ids, t, labels, 2.0, 0.4, view=v)
        # another split of the row into pieces adds in another order
        assert torch.allclose(got[0], base[0], rtol=1e-5)
        check_distill(gpu, z, ids, t, labels, 2.0, 0.4, "mean", 0.5, view=v)
    one = z[0].to(gpu)
    check_distill(gpu, z[:1], ids[:1], t[:1], labels[:1], 2.0, 0.4, view=one)
    check_distill(gpu, z[:1], ids[:1], t[:1], labels[:1], 2.0, 0.4,
                  view=torch.stack((one, one), -1)[:, 0])
    rows = z[:1].expand(4, V).to(gpu)[:1].expand(4, V)      # one row, broadcast
    check_distill(gpu, z[:1].expand(4, V), ids[:4], t[:4], labels[:4], 2.0, 0.4, view=rows)


def test_distill_types_of_teacher_and_ids(gpu):
    z, ids, t, labels = distill_inputs(4, 99, 5, 10, BF16)
    want = check_distill(gpu, z, ids, t, labels, 2.0, 0.5)[0]
    zg, lg = z.to(gpu), labels.to(gpu)
    for tt in (t.float(), t.double(), t.float().half().float()):
        got = gs.distillation_loss(zg, ids.int().to(gpu), tt.to(gpu), lg.int(), temperature=2.0,
                                   alpha=0.5)
        # (fp16 holds these bf16 values within 2^-11 of them)
        assert abs(got - want) <= 1e-2 * abs(want)
    assert gs.distillation_loss(zg, ids.to(gpu), t.float().to(gpu), lg, temperature=2.0,
                                alpha=0.5) == want


def test_distill_empty_and_refused(gpu):
    z = torch.zeros(4, 9, device=gpu, requires_grad=True)
    ids, t = torch.zeros(4, 2, dtype=torch.int64, device=gpu), torch.zeros(4, 2, device=gpu)
    y = torch.zeros(4, dtype=torch.int64, device=gpu)
    e = torch.zeros(0, 9, device=gpu, requires_grad=True)
    for reduction, want in (("mean", math.nan), ("sum", 0.0)):
        loss = gs.distillation_loss(e, ids[:0], t[:0], y[:0], reduction=reduction)
        assert loss.isnan() if math.isnan(want) else loss == want
        assert torch.autograd.grad(loss, e)[0].shape == (0, 9)
    assert gs.distillation_loss(e, ids[:0], t[:0], y[:0], reduction="none").shape == (0,)
    ok = dict(logits=z, teacher_ids=ids, teacher_logits=t, labels=y)
    for bad in (dict(logits=z.half()), dict(logits=z.double()), dict(teacher_ids=ids[:3]),
                dict(teacher_logits=t[:, :1]), dict(labels=y[:3]), dict(teacher_ids=ids.float()),
                dict(labels=y.float()), dict(temperature=0.0), dict(temperature=-1.0),
                dict(alpha=1.5), dict(labels=y.cpu()), dict(teacher_ids=ids[:, :0],
                                                            teacher_logits=t[:, :0])):
        with pytest.raises(_native.GhostHipError):
            gs.distillation_loss(**{**ok, **bad})
    wide = torch.zeros(1, 1025, dtype=torch.int64, device=gpu)
    with pytest.raises(_native.GhostHipError, match="1024"):
        gs.distillation_loss(torch.zeros(1, 2000, device=gpu), wide, wide.float())


def test_distill_beyond_32_bit_offsets(gpu):
    """More than 2^31 logits: the last rows as alone."""
    N, V = 43000, 50257
    z = torch.empty(N, V, dtype=BF16, device=gpu).fill_(0.25)
    z[-2:] = randn((2, V), 1, 2.0, BF16).to(gpu)
    ids = torch.arange(4, device=gpu).expand(N, 4) * 1000
    t = randn((N, 4), 2).to(gpu)
    z.requires_grad_()
    loss = gs.distillation_loss(z, ids, t, temperature=2.0, reduction="sum")
    g, = torch.autograd.grad(loss, z)
    zl = z.detach()[-2:].clone().requires_grad_()
    alone, = torch.autograd.grad(gs.distillation_loss(zl, ids[-2:], t[-2:], temperature=2.0,
                                                      reduction="sum"), zl)
    # another offset from a 16-byte boundary adds in another order: one rounding step of bf16
    off = (f64(g[-2:]) - f64(alone)).abs()
    assert (off <= f64(alone).abs() * 2 * HALF[BF16] + 1e-9).all()


def test_distill_more_rows_than_a_launch_has_workgroups(gpu):
    """2^21 workgroups take the rows in turn: the same rows again have the same bits."""
    N, V, part = (1 << 21) + 3, 5, 1000
    z, ids, t, labels = distill_inputs(part, V, 2, 3, FP32)
    z, ids, t, labels = (x.to(gpu).repeat(N // part + 1, *[1] * (x.dim() - 1))[:N].contiguous()
                         for x in (z, ids, t, labels))
    z.requires_grad_()
    how = dict(temperature=2.0, alpha=0.5, reduction="none")
    loss = gs.distillation_loss(z, ids, t, labels, **how)
    g, = torch.autograd.grad(loss, z, torch.ones_like(loss))
    few = [x[:part].detach() for x in (z, ids, t, labels)]
    few[0].requires_grad_()
    want = gs.distillation_loss(*few, **how)
    dwant, = torch.autograd.grad(want, few[0], torch.ones_like(want))
    # rows of 20 bytes start at other places of a 16-byte piece every four rows; 1000 is their multiple
    for i in (0, 5 * part, N // part * part):
        k = min(part, N - i)
        torch.testing.assert_close(loss[i:i + k], want[:k], rtol=0, atol=0, equal_nan=True)
        torch.testing.assert_close(g[i:i + k], dwant[:k], rtol=0, atol=0, equal_nan=True)


# ---------------------------------------------------------- together, graphs, streams, reuse
def test_backward_twice_and_results_owned_by_the_caller(gpu):
    z, ids, t, labels = (x.to(gpu) for x in distill_inputs(8, 501, 5, 11, BF16))
    z.requires_grad_()
    loss = gs.distillation_loss(z, ids, t, labels, temperature=2.0, alpha=0.5)
    first, = torch.autograd.grad(loss, z, retain_graph=True)
    want = first.clone()
    first.zero_()                                      # the caller's own
    again, = torch.autograd.grad(loss, z, retain_graph=True)
    assert torch.equal(again, want)
    half, = torch.autograd.grad(loss, z, torch.tensor(0.5, device=gpu), retain_graph=True)
    assert torch.equal(half, want * 0.5)               # a power of two: exact
    with torch.no_grad():
        z.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(loss, z)


def _three(gpu, seed, B=3, T=40, V=997, d=64):
    """One pass of the three operators as a model runs them, and its gradients."""
    w = (randn((V, d), seed) * 0.1).to(gpu).requires_grad_()
    proj = (randn((4 * 32, d), seed + 1) * 0.1).to(gpu).requires_grad_()
    out = (randn((V, 64), seed + 2) * 0.1).to(gpu).requires_grad_()
    qw, kw = (torch.ones(32, device=gpu, requires_grad=True) for _ in range(2))
    table = gs.rotary_table(T, 32, device=gpu)
    ids = torch.randint(0, V, (B, T), generator=gen(seed)).to(gpu)
    t_ids = torch.randint(0, V, (B, T, 6), generator=gen(seed + 3)).to(gpu)
    t = randn((B, T, 6), seed + 4).to(gpu)

    def step():
        x = gs.embedding_lookup(ids, w, 8.0, padding_idx=0)
        q, k, v = gs.qkv_norm_rotary(x @ proj.t(), 2, 1, table, None, qw, kw)
        y = ((q * k).sum(-1, keepdim=True) * v).transpose(1, 2).flatten(2)
        loss = gs.distillation_loss(y @ out.t(), t_ids, t, ids, temperature=2.0, alpha=0.5)
        return [loss, *torch.autograd.grad(loss, (w, proj, out, qw, kw))]
    return step, ids, (w, proj, out, qw, kw, table, t_ids, t)


def test_together_against_float64(gpu):
    step, ids, (w, proj, out, qw, kw, table, t_ids, t) = _three(gpu, 1)
    got = step()
    W, P, O, Q, K = (f64(x).requires_grad_() for x in (w, proj, out, qw, kw))
    i = ids.cpu()
    x = torch.where((i == 0)[..., None], W.detach()[i], W[i]) * 8.0
    q, k, v = L.qk_all(L.plan((2, 1, 1), table), (x @ P.t(),), Q, K)
    y = ((q * k).sum(-1, keepdim=True) * v).transpose(1, 2).flatten(2)
    z = (y @ O.t()).flatten(0, 1)
    rows, kept = L.distill_rows(z, t_ids.cpu().flatten(0, 1), f64(t).flatten(0, 1), i.flatten(),
                                2.0, 0.5)
    loss = L.reduced(rows, kept, "mean")
    want = [loss, *torch.autograd.grad(loss, (W, P, O, Q, K))]
    for a, b in zip(got, want):
        # fp32 throughout: normwise, a few hundred roundings of a chain of sums
        assert (f64(a) - b).norm() <= 2e-5 * b.norm() + 1e-12


def test_same_bits_on_every_run_and_on_another_stream(gpu):
    step, *_ = _three(gpu, 2)
    want = step()
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(want, step(), other):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_two_captured_graphs_and_eager_work_between(gpu):
    steps = [_three(gpu, 3), _three(gpu, 4, B=2, T=33, V=800)]
    side = torch.cuda.Stream(gpu)
    graphs, outs, want = [], [], []
    for step, *_ in steps:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                want_i = [x.clone() for x in step()]
        torch.cuda.current_stream().wait_stream(side)
        want.append(want_i)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append(g), outs.append(out)
    for _ in range(3):
        for g, out, w in zip(graphs, outs, want):
            for x in out:
                x.fill_(math.nan)
            g.replay()
            steps[0][0]()                              # eager work of the program's own
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, w))
    # new ids: the replay follows them
    ids = steps[0][1]
    ids.copy_(ids.roll(1))
    graphs[0].replay()
    for a, b in zip(outs[0], steps[0][0]()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rotary", [False, True])
def test_engine_step_of_a_model_with_all_three(gpu, rotary):
    """GradDotProd over the CausalLM with scaled embeddings, normed heads and the distillation
    loss: dots and train gradients against a float64 run of the same samples, one at a time."""
    torch.manual_seed(0)
    cfg = LMConfig(n_layer=2, n_head=2, d_model=32, d_mlp=64, vocab=61, n_ctx=16, rotary=rotary,
                   rotary_pct=0.5, tied=not rotary, qk_norm=True, embed_scale=3.0)
    lm = CausalLM(cfg).to(gpu)
    with torch.no_grad():
        for b in lm.h:
            b.qk.q_weight.uniform_(0.5, 1.5)
            b.qk.k_weight.uniform_(0.5, 1.5)
    n, n_val, T = 6, 2, 16
    ids = torch.randint(0, 61, (n, T), generator=gen(1))
    Y = torch.randint(0, 61, (n, T), generator=gen(2))
    teacher = (torch.randint(0, 61, (n, T, 4), generator=gen(3)), randn((n, T, 4), 4))
    names = [k for k, _ in lm.named_parameters()]
    opt = torch.optim.SGD(lm.parameters(), lr=0.0)
    # per-sample gradients by autograd through the same operators, a sample at a time
    per = {k: [] for k in names}
    for i in range(n):
        s = slice(i, i + 1)
        loss = lm(ids[s].to(gpu), Y[s].to(gpu), tuple(x[s].to(gpu) for x in teacher),
                  temperature=2.0, alpha=0.5) / n
        lm.zero_grad()
        loss.backward()
        for k, p in lm.named_parameters():
            per[k].append(f64(p.grad))
    lm.zero_grad(set_to_none=True)
    eng = GradDotProdEngine(lm, val_batch_size=n_val, use_dummy_bias=True, precision="fp32")
    eng.attach(opt)
    eng.attach_train_batch(ids[:-n_val], Y[:-n_val], 0, 0)
    lm(ids.to(gpu), Y.to(gpu), tuple(x.to(gpu) for x in teacher), temperature=2.0,
       alpha=0.5).backward()
    torch.cuda.synchronize()
    params = dict(lm.named_parameters())
    for k in names:
        G = torch.stack(per[k])
        want = G[:-n_val].sum(0) * n / (n - n_val)
        got = f64(params[k].train_grad)
        assert (got - want).norm() <= 1e-4 * G.norm(), k
        if k.endswith(("q_weight", "k_weight")) or (rotary and k == "wte.weight"):
            want = (G[:-n_val].flatten(1) @ G[-n_val:].sum(0).flatten())
            got = f64(params[k].grad_dot_prod)
            size = G[:-n_val].flatten(1).norm(dim=1) * G[-n_val:].sum(0).norm()
            assert ((got - want).abs() <= 1e-4 * size).all(), k
    eng.prepare_gradients()
    eng.aggregate_and_log()
    assert eng.dot_product_log[-1]["dot_product"].isfinite().all()
    eng.detach()


def test_gradients_are_not_differentiable_again(gpu):
    w = randn((9, 8), 1).to(gpu).requires_grad_()
    ids = torch.tensor([1, 2, 2], device=gpu)
    table = gs.rotary_table(4, 8, device=gpu)
    x = randn((1, 2, 32), 2).to(gpu).requires_grad_()
    z, t_ids, t, y = (v.to(gpu) for v in distill_inputs(3, 11, 2, 3, FP32))
    z.requires_grad_()
    outs = [(gs.embedding_lookup(ids, w, 2.0), w), (gs.qkv_norm_rotary(x, 2, 1, table)[0], x),
            (gs.distillation_loss(z, t_ids, t, y, alpha=0.5), z)]
    for out, inp in outs:
        want, = torch.autograd.grad(out.sum(), inp, retain_graph=True)
        got, = torch.autograd.grad(out.sum(), inp, create_graph=True)   # allowed: once
        assert torch.equal(got, want)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            got.sum().backward()


def test_saved_tensors_that_moved(gpu):
    """What autograd saved may come back elsewhere (offloaded to host memory meanwhile): an odd
    offset of the logits is gone then, and the gradient is formed again for the new place."""
    step, *_ = _three(gpu, 6)
    with torch.autograd.graph.save_on_cpu():
        got = step()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)
    z, t_ids, t, y = (v.to(gpu) for v in distill_inputs(5, 103, 4, 3, BF16))
    odd = torch.empty(5 * 103 + 1, dtype=BF16, device=gpu)[1:].view(5, 103)
    odd.copy_(z)
    odd.requires_grad_()
    want, = torch.autograd.grad(gs.distillation_loss(odd, t_ids, t, y, alpha=0.5), odd)
    with torch.autograd.graph.save_on_cpu():
        loss = gs.distillation_loss(odd, t_ids, t, y, alpha=0.5)
    got, = torch.autograd.grad(loss, odd)
    # another split of the row into pieces: another order of its sums, one rounding step of bf16
    assert ((f64(got) - f64(want)).abs() <= f64(want).abs() * 2 * HALF[BF16] + 1e-9).all()


def test_only_what_is_asked_for(gpu):
    """Gradients of some inputs alone, inputs that need none, and what a loss does not reach."""
    table = gs.rotary_table(8, 16, device=gpu)
    x, qw, kw, grads = qk_inputs(gpu, 2, 6, (3, 1, 1), 32, FP32, 91)
    y = gs.qkv_norm_rotary(x, 3, 1, table, None, qw, kw)
    dx, dq, dk = torch.autograd.grad(y, (x, qw, kw), grads, retain_graph=True)
    for inputs, want in (((x,), (dx,)), ((qw,), (dq,)), ((kw,), (dk,)), ((qw, kw), (dq, dk))):
        got = torch.autograd.grad(y, inputs, grads, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    frozen = gs.qkv_norm_rotary(x, 3, 1, table, None, qw.detach(), kw.detach())
    assert torch.equal(torch.autograd.grad(frozen, x, grads)[0], dx)
    weights = gs.qkv_norm_rotary(x.detach(), 3, 1, table, None, qw, kw)
    assert torch.equal(torch.autograd.grad(weights, qw, grads)[0], dq)
    q = x.detach()[..., :96].unflatten(-1, (3, 32)).clone().requires_grad_()
    k = x.detach()[..., 96:128].unflatten(-1, (1, 32)).clone().requires_grad_()
    rq, rk = gs.qk_norm_rotary(q, k, table, None, qw, kw)
    got, = torch.autograd.grad(rk, k, grads[1], retain_graph=True)
    assert torch.equal(got.flatten(2), dx[..., 96:128])
    assert torch.autograd.grad(rk, q, grads[1], allow_unused=True)[0].eq(0).all()
