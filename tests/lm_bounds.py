"""Error bounds of the norm weights' sums (gradients, dots), tight enough to miss nothing that counts.

A weight's gradient at feature f is the sum over n tokens and heads of addends h x r.  With U = 2^-24:

  - an addend: h is two products, their sum and the table's rounding, r the root of a mean of D squares,
    then two products more: (D / 2 + 24) U of its size, where |h| counts both features of a pair;
  - the sum: no addend passes more than depth() additions, each of at most U of the addends' sizes.
    Workgroups take up to 6 heads of a part, so H heads make at most H / per + 3 head groups, and at least
    384 workgroups (half of 768, by rounding down) share M tokens and the head groups, each with S lane
    groups for a token each: a lane adds at most 6 + M (H + 18) / (384 S) addends.  A row of D features
    has at most D / 4 + 4 lanes of 64, so S is at least 1024 / (D + 16), and 4.  Fewer than 44 more
    additions follow: the lanes and waves of a workgroup (10), the second launch over up to 768
    workgroups' rows (13) or, over all samples' rows, one for every 128 of those.

Sums over samples and features count their own terms.
"""
import torch

from tests import lm_forms as L
from tests.lm_forms import HALF, U, f64


def within(got, want, bound, what=""):
    """|got - want| <= bound elementwise; NaN in the same places, infinities equal."""
    got, bound = f64(got), bound.expand_as(want)
    fine = want.isfinite()
    assert torch.equal(fine, got.isfinite()), f"{what}: not finite in other places"
    assert torch.equal(want[~fine].nan_to_num(nan=0.5), got[~fine].nan_to_num(nan=0.5)), \
        f"{what}: other infinities"
    over = (got - want).abs()[fine] > bound[fine]
    assert not over.any(), (
        f"{what}: {int(over.sum())} of {over.numel()} over the bound, worst "
        f"{((got - want).abs()[fine] / bound[fine].clamp(min=1e-300)).max():.3g} of it")


def depth(plan, x, D):
    B, T = x.shape[:2]
    H = sum(plan["heads"])
    return 50 + B * T * (H + 18) / (384 * max(4, 1024 // (D + 16))) + B * H / 128


def sample_sums(plan, x, qw, kw, grads):
    """[(s, size)] of both weights in float64: each sample's gradient [B, D], its addends' sizes."""
    _, dq, dk = L.qk_grads(plan, (x,), qw, kw, grads, per_sample=True)
    out = []
    for s, part, g in zip((dq, dk), L.split_heads(plan, (f64(x),)), grads):
        h = f64(g).abs().transpose(1, 2)
        n = plan["table"].shape[-1]
        r, rest = h[..., :2 * n], h[..., 2 * n:]
        other = r.unflatten(-1, (n, 2)).flip(-1).flatten(-2) if plan["interleaved"] else r.roll(n, -1)
        h = torch.cat((r + other, rest), -1)
        xn = (part / torch.sqrt((part ** 2).mean(-1, keepdim=True) + plan["eps"])).abs()
        out.append((s, (h * xn).sum((1, 2))))
    return out


def check_total(got, sums, plan, x, what=""):
    """The gradients of both weights over all samples."""
    for i, (g, (s, size)) in enumerate(zip(got, sums)):
        D, want = s.shape[1], s.sum(0)
        within(g, want, (depth(plan, x, D) + D / 2 + 24) * U * size.sum(0) + want.abs() * HALF[g.dtype],
               f"{what}gradient {i}")


def check_dots(got, sums, plan, x, n_val, val_start=None, scale=0.25, what=""):
    """[dot_q, dot_k, train gradient of q's weight, of k's]."""
    B = x.shape[0]
    vs = B - n_val if val_start is None else val_start
    val = torch.zeros(B, dtype=torch.bool)
    val[vs:vs + n_val] = True
    for i, (s, size) in enumerate(sums):
        D = s.shape[1]
        err = (depth(plan, x, D) + D / 2 + 24) * U * size
        st, et, sv = s[~val], err[~val], s[val].sum(0)
        ev = err[val].sum(0) + n_val * U * (s[val].abs() + err[val]).sum(0)
        bound = et @ sv.abs() + st.abs() @ ev + et @ ev + (D / 64 + 10) * U * (st.abs() @ sv.abs())
        within(got[i], st @ sv, bound, f"{what}dots {i}")
        want, t = st.sum(0) * scale, got[2 + i].dtype
        within(got[2 + i], want, scale * (et.sum(0) + len(st) * U * (st.abs() + et).sum(0)) +
               want.abs() * HALF[t] * (1 + 1e-3), f"{what}train gradient {i}")
