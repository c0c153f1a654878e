"""The language-model layers under the engines on the GPU, where a program does more than a plain
step."""
import pytest
import torch
from torch import nn

from ghostsuite_amd import GradDotProdEngine
from tests.helpers import assert_close
from tests.test_lm_engine import _Recomputed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", ["reentrant", "not reentrant"])
def test_engine_dots_of_recomputed_layers(gpu, how):
    torch.manual_seed(3)
    n, n_val, T = 6, 2, 5
    nets = [_Recomputed(None).to(gpu), _Recomputed(how).to(gpu)]
    nets[1].load_state_dict(nets[0].state_dict())
    ids, Y = torch.randint(0, 13, (n, T), device=gpu), torch.randint(0, 13, (n, T), device=gpu)
    got = []
    for net in nets:
        net.positions = torch.arange(T, device=gpu) + 7
        eng = GradDotProdEngine(net, val_batch_size=n_val, use_dummy_bias=False, precision="fp32")
        eng.attach(torch.optim.SGD(net.parameters(), lr=0.0))
        for _ in range(2):
            # memory as it may come: the caching allocator hands these out again
            junk = [torch.full((k,), float("nan"), device=gpu) for k in range(1, 4097, 64)]
            del junk
            nn.functional.cross_entropy(net(ids).flatten(0, 1), Y.flatten()).backward()
            torch.cuda.synchronize()
            got.append({k: (p.grad_dot_prod.clone(), p.train_grad.clone())
                        for k, p in net.named_parameters()})
            for p in net.parameters():
                del p.grad_dot_prod, p.train_grad
        eng.detach()
    for other in got[1:]:
        for k, (dot, grad) in got[0].items():
            assert_close(other[k][0].cpu(), dot.cpu(), 1e-6, k)
            assert_close(other[k][1].cpu(), grad.cpu(), 1e-6, k)
