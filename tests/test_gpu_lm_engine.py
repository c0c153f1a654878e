"""The language-model layers under the engines on the GPU, where a program does more than a plain
step."""
import pytest
import torch
import torch.utils.checkpoint
from torch import nn

import ghostsuite_amd as gs
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


@pytest.mark.parametrize("early_stop", [True, False])
def test_operators_alone_under_checkpointing(gpu, early_stop):
    """Without re-entry the recomputation ends, by an exception through the operator, as soon as its
    saved tensors are there."""
    ids = torch.randint(0, 13, (4, 5), device=gpu)
    w = torch.randn(13, 24, device=gpu, requires_grad=True)
    x = torch.randn(4, 5, 24, device=gpu, requires_grad=True)
    qw = torch.rand(6, device=gpu, requires_grad=True)
    table = gs.rotary_table(5, 6, device=gpu)
    z = torch.randn(4, 5, 13, device=gpu, requires_grad=True)
    t = torch.randn(4, 5, 3, device=gpu)
    calls = [(lambda w: gs.embedding_lookup(ids, w, 2.0), (w,)),
             (lambda x, v: torch.cat(gs.qkv_norm_rotary(x, 2, 1, table, None, v, v), 1), (x, qw)),
             (lambda z: gs.distillation_loss(z, ids[..., None].expand(4, 5, 3), t, ids, alpha=0.5,
                                             temperature=2.0), (z,))]
    with torch.utils.checkpoint.set_checkpoint_early_stop(early_stop):
        for f, inputs in calls:
            y = f(*inputs)
            g = torch.randn_like(y)
            want = torch.autograd.grad(y, inputs, g)
            y = torch.utils.checkpoint.checkpoint(f, *inputs, use_reentrant=False)
            for a, b in zip(torch.autograd.grad(y, inputs, g), want):
                assert torch.equal(a, b)


def test_autograd_exceptions_keep_their_type(gpu):
    """What a saved-tensor hook raises comes through the operators as it is."""
    class Mine(Exception):
        pass

    def pack(t):
        raise Mine("stop")
    w = torch.randn(13, 24, device=gpu, requires_grad=True)
    x = torch.randn(4, 5, 24, device=gpu, requires_grad=True)
    ids = torch.zeros(4, 5, dtype=torch.int64, device=gpu)
    for f in (lambda: gs.embedding_lookup(ids, w), lambda: gs.qkv_norm_rotary(
            x, 2, 1, gs.rotary_table(5, 6, device=gpu)), lambda: gs.distillation_loss(
            x, ids[..., None], torch.zeros(4, 5, 1, device=gpu))):
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t), pytest.raises(Mine):
            f()
