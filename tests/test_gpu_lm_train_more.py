"""The output projection's loss and the norm on the GPU, under both engines and in calls with more than one piece
of the vocabulary."""
import pytest
import torch
from torch import nn

import ghostsuite_amd as gs
from ghostsuite_amd import GradProjLoraEngine
from tests.helpers import BF16_TOL, assert_close, gen, randn

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
