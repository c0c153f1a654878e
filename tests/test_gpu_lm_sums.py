"""The norm weights' sums on the GPU within the bounds of tests/lm_bounds.py, gradients past 32-bit
offsets, and the projection of a scaled embedding."""
import pytest
import torch

import ghostsuite_amd as gs
from ghostsuite_amd import _native
from oracle import ghost_ref as R
from tests import lm_bounds as S
from tests import lm_forms as L
from tests.helpers import gen, randn
from tests.lm_forms import HALF, U, f64
from tests.test_lm_bounds import SHAPES, inputs

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("positions", [None, "row", "batch"])
@pytest.mark.parametrize("B,n_val,T,heads,D,n_rot", SHAPES + [
    (1, 0, 9001, (2, 7, 7), 128, 128), (2, 0, 3000, (7, 1, 1), 81, 20), (3, 1, 900, (1, 1, 1), 512, 512),
    (1000, 7, 5, (2, 1, 1), 16, 16)])
def test_norm_weights_sums(gpu, dtype, interleaved, positions, B, n_val, T, heads, D, n_rot):
    table = gs.rotary_table(T + 50, n_rot, device=gpu)
    pos = {None: None, "row": torch.randperm(T + 50, generator=gen(1))[:T].to(gpu),
           "batch": torch.randint(0, T + 50, (B, T), generator=gen(2)).to(gpu)}[positions]
    plan = L.plan(heads, table, pos, interleaved=interleaved)
    x, qw, kw, grads = inputs(B, T, heads, D, dtype, 71)
    sums = S.sample_sums(plan, x, qw, kw, grads)
    x, qw, kw, *grads = (t.to(gpu) for t in (x, qw, kw, *grads))
    leaves = [t.clone().requires_grad_() for t in (x, qw, kw)]
    y = gs.qkv_norm_rotary(leaves[0], heads[0], heads[1], table, pos, *leaves[1:],
                           interleaved=interleaved)
    S.check_total(torch.autograd.grad(y, leaves, grads)[1:], sums, plan, x)
    if n_val == 0:
        return
    ops = _native.ops()
    samples = torch.full((2, B, D), float("nan"), device=gpu)
    y = ops.qk_norm_rotary(leaves[0], None, heads, table, pos, *leaves[1:], True, 1e-6, interleaved,
                           samples)
    S.check_total(torch.autograd.grad(y, leaves, grads)[1:], sums, plan, x, "with samples: ")
    for start in (None, 0, (B - n_val) // 2):
        how = dict(val_start=start, grad_scale=0.25)
        got = ops.qk_norm_rotary_dots(x, None, heads, table, pos, qw, kw, 1e-6, interleaved, grads,
                                      n_val, **how)
        S.check_dots(got, sums, plan, x, n_val, start, what="own pass: ")
        S.check_dots(ops.qk_sample_dots(samples, qw, kw, n_val, **how), sums, plan, x, n_val, start,
                     what="samples: ")


def test_qk_gradients_beyond_32_bit_offsets(gpu):
    """More than 2^31 elements of input, gradients and input gradient: the first and the last token as
    alone, zeros between."""
    B, T, heads, D = 3, 349526, (14, 1, 1), 128
    assert B * T * sum(heads) * D > 2 ** 31
    table = gs.rotary_table(T, D, device=gpu)
    ends = ((0, 0), (B - 1, T - 1))
    x = torch.zeros(B, T, sum(heads) * D, dtype=BF16, device=gpu)
    grads = [torch.zeros(B, h, T, D, dtype=BF16, device=gpu) for h in heads]
    for b, t in ends:
        x[b, t] = randn((sum(heads) * D,), b + 1, 1.0, BF16).to(gpu)
        for i, g in enumerate(grads):
            g[b, :, t] = randn(g[b, :, t].shape, 5 + b + i, 1.0, BF16).to(gpu)
    w = [(1 + 0.2 * randn((D,), 9 + i)).to(gpu).requires_grad_() for i in range(2)]

    def run(x, grads, pos=None):
        x = x.requires_grad_()
        y = gs.qkv_norm_rotary(x, 14, 1, table, pos, *w)
        return torch.autograd.grad(y, (x, *w), grads)

    dx, dq, dk = run(x, grads)
    alone = [run(x.detach()[b:b + 1, t:t + 1], [g[b:b + 1, :, t:t + 1] for g in grads],
                 torch.tensor([t], device=gpu)) for b, t in ends]
    for (b, t), a in zip(ends, alone):
        assert torch.equal(dx[b, t], a[0][0, 0])
        dx[b, t] = 0
    assert not dx.any()
    for got, k in ((dq, 1), (dk, 2)):       # fp32 sums over at most 14 heads, twice
        size = sum(f64(a[k]).abs() for a in alone)
        S.within(got, sum(f64(a[k]) for a in alone), 64 * U * (size + 14.0), "weights")


@pytest.mark.parametrize("n", [5, 300])
def test_lookup_gradient_beyond_32_bit_offsets(gpu, n):
    """A table of more than 2^31 elements, for both ways of its gradient."""
    vocab, d = (1 << 21) + 3, 1032
    assert vocab * d > 2 ** 31
    w = torch.empty(vocab, d, dtype=BF16, device=gpu).requires_grad_()
    last = torch.tensor([vocab - 1, 0, vocab - 2, vocab - 1, 2 ** 31 // d + 1], device=gpu)
    ids = last.repeat(n // 5)
    g = randn((n, d), n, 1.0, BF16).to(gpu)
    got, = torch.autograd.grad(gs.embedding_lookup(ids, w, 2.0), w, g)
    rows = [0, 2 ** 31 // d + 1, vocab - 2, vocab - 1]
    want, mag, count = L.lookup_grad(torch.tensor([[3, 0, 2, 3, 1]]).repeat(n // 5, 1), f64(g), 4, 2.0)
    S.within(got[rows], want, want.abs() * HALF[BF16] * (1 + 1e-3) + (count[:, None] + 4) * U * mag,
             "rows")
    got[rows] = 0
    assert not got.any()


def test_lookup_gradient_of_many_rows_beyond_32_bit_offsets(gpu):
    """Output gradients of more than 2^31 elements, a table likewise."""
    n, d = (1 << 21) + 3, 1032
    w = torch.empty(n, d, dtype=BF16, device=gpu).requires_grad_()
    ids = torch.arange(n, device=gpu).flip(0)
    g = torch.zeros(n, d, dtype=BF16, device=gpu)
    for i in (0, n - 1):
        g[i] = randn((d,), 1 + i % 7, 1.0, BF16).to(gpu)
    got, = torch.autograd.grad(gs.embedding_lookup(ids, w, 2.0), w, g)
    for i in (0, n - 1):
        assert torch.equal(got[n - 1 - i], g[i] * 2)
        got[n - 1 - i] = 0
    assert not got.any()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("B,T,V,d,k_i,k_o", [(3, 7, 30, 24, 4, 6), (4, 130, 50257, 768, 16, 16),
                                             (2, 40, 3000, 96, 100, 5), (2, 70, 500, 100, 8, 128)])
def test_projection_of_a_scaled_embedding(gpu, dtype, B, T, V, d, k_i, k_o):
    """ScaledEmbedding under the projection hooks: its scale, and a padding id without a part."""
    from ghostsuite_amd.gradProjection.autograd_gradproj import create_projection_hooks
    pad, scale = 3, 1.75
    ids = torch.randint(0, V, (B, T), generator=gen(T))
    ids[0, :3], ids[1, ::2] = ids[0, 0], pad
    G = randn((B, T, d), 32 + T, 1.0, dtype)
    P_i, P_o = randn((k_i, V), 33, 1.0 / k_i ** 0.5), randn((k_o, d), 34, 1.0 / k_o ** 0.5)
    emb = gs.ScaledEmbedding(V, d, scale, padding_idx=pad, device=gpu, dtype=dtype)
    hooks = create_projection_hooks(emb, "emb", P_i.to(gpu), P_o.to(gpu))
    hooks._compute_embedding_proj(emb, ids.to(gpu), G.to(gpu))
    torch.cuda.synchronize()
    Gm = torch.where((ids == pad)[..., None], 0.0, G.double()) * scale
    want = R.kron_embed_proj_exact(ids, Gm, P_i.to(dtype).double(), P_o.to(dtype).double())
    got = f64(emb._ghost_grad_proj).reshape(want.shape)
    # products P_o g and their sum over tokens: fp32 sums of d and T terms, the bf16 operands exact
    lhs = P_o.to(dtype).double().abs() @ Gm.abs().transpose(1, 2)          # [B, k_o, T]
    rhs = P_i.to(dtype).double().abs().t()[ids]                            # [B, T, k_i]
    S.within(got, want.double(), (d + T + 16) * U * (lhs @ rhs), "projection")
