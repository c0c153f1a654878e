"""The language-model layers under the engines where a program does more than a plain step, through
the stand-in kernel layer."""
import math

import pytest
import torch
import torch.utils.checkpoint
from torch import nn

import ghostsuite_amd as gs
from ghostsuite_amd import GradDotProdEngine
from tests.helpers import assert_close
from tests.test_lm_layers import _Net, oracle_ops  # noqa: F401  (the fixture)


class _Recomputed(_Net):
    """The net with projection, heads and a second layer of them under activation checkpointing."""

    def __init__(self, how):
        super().__init__()
        self.qkv2 = nn.Linear(2 * 6, (2 + 2 * 1) * 6)
        self.qk2 = gs.QKNormRotary(2, 1, 6, n_rot=4, n_positions=32)
        self.how = how

    def body(self, x):
        for qkv, qk in ((self.qkv, self.qk), (self.qkv2, self.qk2)):
            q, k, v = qk(qkv(x), self.positions)
            x = ((q * k).sum(-1, keepdim=True) * v).transpose(1, 2).flatten(2)
        return x

    def forward(self, ids):
        x = self.emb(ids)
        x = self.body(x) if self.how is None else \
            torch.utils.checkpoint.checkpoint(self.body, x, use_reentrant=self.how == "reentrant")
        return self.out(x)


def _memory_as_found(monkeypatch):
    """torch.empty as it may come: full of NaN."""
    empty = torch.empty

    def found(*args, **kw):
        t = empty(*args, **kw)
        with torch.no_grad():
            return t.fill_(math.nan) if t.is_floating_point() else t
    monkeypatch.setattr(torch, "empty", found)


@pytest.mark.parametrize("how", ["reentrant", "not reentrant"])
def test_engine_dots_of_recomputed_layers(oracle_ops, monkeypatch, how):
    """Checkpointing runs a layer's forward again during the backward pass, of which without
    re-entry the first forward's nodes are a part: the sample gradients are the ones they wrote."""
    torch.manual_seed(3)
    n, n_val, T = 6, 2, 5
    nets = [_Recomputed(None), _Recomputed(how)]
    nets[1].load_state_dict(nets[0].state_dict())
    ids, Y = torch.randint(0, 13, (n, T)), torch.randint(0, 13, (n, T))
    _memory_as_found(monkeypatch)
    got = []
    for net in nets:
        net.positions = torch.arange(T) + 7
        eng = GradDotProdEngine(net, val_batch_size=n_val, use_dummy_bias=False, precision="fp32")
        eng.attach(torch.optim.SGD(net.parameters(), lr=0.0))
        for _ in range(2):      # a second step as the first
            oracle_ops.calls.clear()
            nn.functional.cross_entropy(net(ids).flatten(0, 1), Y.flatten()).backward()
            got.append({k: (p.grad_dot_prod.clone(), p.train_grad.clone())
                        for k, p in net.named_parameters()})
            for p in net.parameters():
                del p.grad_dot_prod, p.train_grad
            assert [c[0] for c in oracle_ops.calls if c[0].startswith("qk_")] == \
                2 * ["qk_sample_dots"]
        assert all(m.__dict__.get("_gs_sample_grads") is None for m in net.modules())
        eng.detach()
    for other in got[1:]:
        for k, (dot, grad) in got[0].items():
            assert_close(other[k][0], dot, 1e-6, k)
            assert_close(other[k][1], grad, 1e-6, k)


def test_engine_dots_without_what_a_backward_pass_left(oracle_ops, monkeypatch):
    """Sample gradients that the pass under way did not write are not read: the hook makes its own
    pass over the activations."""
    torch.manual_seed(4)
    layer = gs.QKNormRotary(2, 1, 6, n_positions=16)
    x = torch.randn(5, 4, 24, requires_grad=True)
    eng = GradDotProdEngine(layer, val_batch_size=2, precision="fp32")
    eng.attach(torch.optim.SGD(layer.parameters(), lr=0.0))
    _memory_as_found(monkeypatch)

    def results():
        return [t.clone() for w in (layer.q_weight, layer.k_weight)
                for t in (w.grad_dot_prod, w.train_grad)]

    def clear():
        for w in (layer.q_weight, layer.k_weight):
            del w.grad_dot_prod, w.train_grad
    torch.autograd.backward(layer(x)[:2], [torch.ones(5, h, 4, 6) for h in (2, 1)])
    want = results()
    clear()
    oracle_ops.calls.clear()
    y = layer(x)                                   # its buffer, then one for two samples
    layer(x[:2])
    layer.__dict__["activations"] = x.detach()
    torch.autograd.backward(y[:2], [torch.ones(5, h, 4, 6) for h in (2, 1)])
    assert [c[0] for c in oracle_ops.calls] == ["qk_norm_rotary_dots"]
    for a, b in zip(results(), want):
        assert_close(a, b, 1e-6)
    eng.detach()


def test_sample_gradients_of_an_earlier_step_are_not_used_again(oracle_ops):
    """A step without a backward pass leaves nothing that a later one, which may be captured into a
    graph, would write."""
    net = _Net()
    eng = GradDotProdEngine(net, val_batch_size=2, use_dummy_bias=False, precision="fp32")
    eng.attach(torch.optim.SGD(net.parameters(), lr=0.0))
    ids = torch.randint(0, 13, (5, 4))
    net(ids)
    first = net.qk._gs_sample_grads
    loss = net(ids).sum()
    assert first is not None and net.qk._gs_sample_grads is not first
    loss.backward()
    assert net.qk.__dict__.get("_gs_sample_grads") is None and first._version == 0
    eng.detach()
