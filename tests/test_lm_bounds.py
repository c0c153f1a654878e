"""The bounds of the norm weights' sums reject what they are there for: results of a wrong size or
sign, and sums that lose some of their tokens.  Planted in float64 results, without a GPU."""
import pytest
import torch

import ghostsuite_amd as gs
from tests import lm_bounds as S
from tests import lm_forms as L
from tests.helpers import gen, randn

SHAPES = [  # B, n_val, T, heads, D, n_rot
    (2, 1, 1, (1, 1, 1), 64, 64), (5, 2, 33, (4, 1, 1), 128, 64), (7, 3, 300, (2, 2, 2), 80, 20),
    (6, 1, 9, (3, 3, 3), 33, 10), (40, 30, 3, (2, 1, 1), 48, 48), (3, 1, 7001, (5, 1, 1), 64, 32),
    (130, 3, 2, (2, 1, 1), 130, 8), (2, 1, 20011, (3, 1, 1), 64, 32), (400, 100, 40, (3, 1, 1), 32, 8)]


def inputs(B, T, heads, D, dtype, seed):
    x = (randn((B, T, sum(heads) * D), seed) * (0.2 + torch.rand(B, T, 1, generator=gen(seed)))
         ).to(dtype)
    qw, kw = (1 + 0.2 * randn((D,), seed + k) for k in (1, 2))
    return x, qw.to(dtype), kw.to(dtype), [randn((B, h, T, D), seed + 3 + i, 1.0, dtype)
                                           for i, h in enumerate(heads)]


def results(sums, n_val):
    """What a kernel would return: the float64 sums, rounded to fp32."""
    B = sums[0][0].shape[0]
    dots = [(s[:B - n_val] @ s[B - n_val:].sum(0)).float() for s, _ in sums]
    return dots + [(s[:B - n_val].sum(0) * 0.25).float() for s, _ in sums], \
        [s.sum(0).float() for s, _ in sums]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,n_val,T,heads,D,n_rot", SHAPES)
def test_wrong_sums_are_rejected(B, n_val, T, heads, D, n_rot, interleaved):
    plan = L.plan(heads, gs.rotary_table(T, n_rot), interleaved=interleaved)
    x, qw, kw, grads = inputs(B, T, heads, D, torch.float32, 71)
    sums = S.sample_sums(plan, x, qw, kw, grads)
    dots, total = results(sums, n_val)
    S.check_dots(dots, sums, plan, x, n_val)
    S.check_total(total, sums, plan, x)
    long = T > 1000                           # the features of a dot cancel: its bound is wider there
    for tokens in (max(1, T // 20), T // 20 if long else 1):       # the last 5%, the last one
        lost = [g.clone() for g in grads]
        for g in lost:
            g[:, :, T - tokens:] = 0
        part = results(S.sample_sums(plan, x, qw, kw, lost), n_val)
        for k in range(2):
            wrong = [dots[:k] + part[0][k:k + 1] + dots[k + 1:],
                     dots[:2 + k] + part[0][2 + k:3 + k] + dots[3 + k:]]
            for w in wrong:
                with pytest.raises(AssertionError, match="over the bound"):
                    S.check_dots(w, sums, plan, x, n_val)
            with pytest.raises(AssertionError, match="over the bound"):
                S.check_total(total[:k] + part[1][k:k + 1] + total[k + 1:], sums, plan, x)
    for k in range(4):
        for w in (dots[k] * 0, -dots[k], 2 * dots[k], dots[k] * (1.5 if long else 1 + 2 ** -6)):
            with pytest.raises(AssertionError, match="over the bound"):
                S.check_dots(dots[:k] + [w] + dots[k + 1:], sums, plan, x, n_val)
    for k in range(2):
        for w in (total[k] * 0, -total[k], 2 * total[k], total[k] * (1 + 2 ** -6)):
            with pytest.raises(AssertionError, match="over the bound"):
                S.check_total(total[:k] + [w] + total[k + 1:], sums, plan, x)


def test_infinities_of_the_other_sign_are_rejected():
    want, bound = torch.tensor([1.0, float("inf"), float("nan")]).double(), torch.zeros(3).double()
    S.within(want, want, bound)
    for wrong in ([1.0, float("-inf"), float("nan")], [1.0, float("nan"), float("inf")],
                  [float("inf"), float("inf"), float("nan")]):
        with pytest.raises(AssertionError):
            S.within(torch.tensor(wrong), want, bound)
