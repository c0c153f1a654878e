"""The output projection's loss and the norm on the GPU, under both engines and in calls with more than one piece
of the vocabulary."""
import pytest
import torch
from torch import nn

import ghostsuite_amd as gs
from ghostsuite_amd import GradProjLoraEngine, _native
from tests import train_forms as L
from tests.helpers import BF16_TOL, assert_close, gen, randn
from tests.lm_bounds import within
from tests.lm_forms import HALF, U

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


class Shifting(nn.Module):
    """Copies its labels within its forward, as models that shift them do: the head's are the only reference."""

    def __init__(self, V, d, dtype, gpu):
        super().__init__()
        self.body = nn.Linear(d, d).to(gpu, dtype)
        self.head = gs.HeadCrossEntropy(d, V).to(gpu, dtype)

    def forward(self, x, labels):
        labels = torch.cat((labels[:, 1:], torch.full_like(labels[:, :1], -100)), 1)
        return self.head(self.body(x), labels)


def projection(net, tmp_path):
    eng = GradProjLoraEngine(net, proj_layers="head", proj_rank_total=16, proj_rank_min=4, proj_seed=1,
                             proj_dtype="float32", proj_dir=str(tmp_path), proj_save_interval=100,
                             include_embeddings=False)
    eng.attach()
    return eng


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_projection_of_a_head_with_copied_labels(gpu, tmp_path, dtype):
    """GradProjLoraEngine on a HeadCrossEntropy against the projection of float64 gradients, with memory handed out
    and overwritten between and within the backward passes."""
    n, T, V, d = 5, 60, 1500, 64
    net = Shifting(V, d, dtype, gpu)
    x = randn((n, T, d), 1, 1.0, dtype).to(gpu)
    labels = torch.randint(0, V, (n, T), generator=gen(2)).to(gpu)
    eng = projection(net, tmp_path)
    P_i, P_o = (p.double().cpu() for p in eng.projection_matrices["head"])
    rows = net.body(x).detach().double().cpu()
    z = rows @ net.head.weight.detach().double().cpu().t()
    y = torch.cat((labels[:, 1:].cpu(), torch.full((n, 1), -100)), 1)
    dz = torch.softmax(z, -1) - nn.functional.one_hot(y.clamp(min=0), V)
    dz[y < 0] = 0
    dz /= int((y >= 0).sum())
    # the gradient of the mean loss, times the samples, as a Linear's
    want = n * torch.stack([P_o @ dz[b].t() @ rows[b] @ P_i.t() for b in range(n)])

    def junk(*_):
        for k in (n * T, 2 * n * T, 4 * n * T):
            for _ in range(4):
                torch.full((k,), 7, device=gpu, dtype=torch.int64)
                torch.full((2 * k,), float("nan"), device=gpu)
    net.body.register_full_backward_hook(lambda *a: junk())
    for _ in range(3):
        junk()
        loss = net(x, labels)
        loss.backward()
        del loss
        junk()
        torch.cuda.synchronize()
        got = net.head._ghost_grad_proj
        assert_close(got.reshape(want.shape).cpu(), want, BF16_TOL if dtype == BF16 else 1e-4, "projection")
    eng.detach()


# ------------------------------------------------------------------------ sizes
def test_head_of_more_than_2_31_features_of_rows(gpu):
    """262184 rows of 8192 features, 2^31 elements: each of some rows in its bound, the weight's gradient that of
    the logits' gradient."""
    N, V, d = 262184, 12, 8192
    g = torch.Generator(device=gpu).manual_seed(1)
    x = torch.empty(N, d, dtype=BF16, device=gpu)
    for at in range(0, N, 32773):
        x[at:at + 32773] = torch.randn(min(32773, N - at), d, generator=g, device=gpu)
    w = randn((V, d), 2, 2.0 / d ** 0.5, BF16)
    labels = torch.randint(0, V, (N,), generator=gen(3))
    labels[::7] = -100
    x.requires_grad_()
    wg, yg = w.to(gpu).requires_grad_(), labels.to(gpu)
    loss = gs.head_cross_entropy(x, wg, yg, reduction="none")
    dx, dw = torch.autograd.grad(loss, (x, wg), torch.ones_like(loss))
    part = torch.cat((torch.arange(50), torch.arange(N - 50, N), torch.randperm(N, generator=gen(4))[:100]))
    want = L.head_all(x.detach()[part.to(gpu)], w, labels[part], torch.ones(200), "none", BF16)
    within(loss[part.to(gpu)], *want["loss"], "loss")
    within(dx[part.to(gpu)], *want["dx"], "dx")
    lse = torch.empty(N, 2, device=gpu)
    _native.ops().head_cross_entropy(x.detach(), wg.detach(), yg, -100, "none", lse)
    dz = _native.ops().head_logit_grad(x.detach(), wg.detach(), yg, lse, torch.ones(N, device=gpu), 0, V, -100,
                                       "none")[:, :V].double()
    ref = size = 0
    for at in range(0, N, 32773):
        rows, a = x.detach()[at:at + 32773].double(), dz[at:at + 32773].t().contiguous()
        ref, size = ref + a @ rows, size + a.abs() @ rows.abs()
    # the same rounded dz on both sides: the sums' terms and the output's rounding
    within(dw, ref.cpu(), (ref.abs() * HALF[BF16] + (N + 64) * U * size).cpu(), "dw")


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_head_of_more_than_2_25_entries(gpu, dtype):
    N, V, d = 2, 2 ** 25 + 1000, 2
    x, w = randn((N, d), 1, 1.0, dtype), randn((V, d), 2, 1.0, dtype)
    labels = torch.tensor([V - 1, 5])
    xg, wg = x.to(gpu).requires_grad_(), w.to(gpu).requires_grad_()
    loss = gs.head_cross_entropy(xg, wg, labels.to(gpu))
    dx, dw = torch.autograd.grad(loss, (xg, wg))
    want = L.head_all(x, w, labels, torch.tensor(1.0), "mean", dtype)
    within(loss, *want["loss"], "loss")
    within(dx, *want["dx"], "dx")
    within(dw, *want["dw"], "dw")
