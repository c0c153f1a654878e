"""The output projection's loss, the norm and the optimizer without a GPU: what the engines keep, mark and split
on the way, and what the entry points take."""
import copy
import ctypes

import pytest
import torch

from ghostsuite_amd import AdamW, GradDotProdEngine, GradProjLoraEngine, _native, lm_layers
from ghostsuite_amd.gradProjection import autograd_gradproj
from tests.helpers import assert_close
from tests.test_lm_train import P16, _Net, _head, oracle_ops   # noqa: F401  (a fixture)


def _projection(net, tmp_path, **how):
    eng = GradProjLoraEngine(net, proj_layers="head", proj_rank_total=8, proj_rank_min=2, proj_seed=1,
                             proj_dtype="float32", proj_dir=str(tmp_path), proj_save_interval=100,
                             include_embeddings=False, **how)
    eng.attach()
    return eng


def test_projection_marks_what_the_side_stream_reads(oracle_ops, monkeypatch, tmp_path):   # noqa: F811
    """Labels and sums of the head's loss, whose last reference may die within the backward pass, are handed to
    the side stream with the activations, or the allocator gives their memory to the other stream too early."""
    marked = []
    real = autograd_gradproj._overlap.on_side_stream

    def on_side_stream(*tensors):
        marked.extend(tensors)
        return real(*tensors)
    monkeypatch.setattr(autograd_gradproj._overlap, "on_side_stream", on_side_stream)
    torch.manual_seed(3)
    net = _Net()
    _projection(net, tmp_path)
    ids, labels = torch.randint(0, 13, (5, 4)), torch.randint(0, 13, (5, 4))
    loss = net(ids, labels.clone())
    kept = net.head.__dict__["_gs_head"]
    assert any(torch.equal(t, labels) for t in kept)
    loss.backward()
    assert all(any(t is k for t in marked) for k in kept)
    assert "_gs_head" not in net.head.__dict__ and net.head._ghost_grad_proj is not None


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("first", ["dots", "projection"])
def test_both_engines_at_once_on_a_heads_loss(oracle_ops, tmp_path, reduction, first):   # noqa: F811
    """Either engine's hook may come first, as on an nn.Linear; each gives what it gives alone, step after step, with
    a call without labels in between."""
    torch.manual_seed(4)
    net = _Net(reduction=reduction)
    ids, labels = torch.randint(0, 13, (5, 4)), torch.randint(0, 13, (5, 4))

    def dots(m):
        eng = GradDotProdEngine(m, val_batch_size=2, use_dummy_bias=False, precision="fp32")
        eng.attach(torch.optim.SGD(m.parameters(), lr=0.0))

    def projection(m):
        _projection(m, tmp_path)

    def run(*engines):
        m = copy.deepcopy(net)
        for e in engines:
            e(m)
        for step in range(2):
            m(ids, labels).sum().backward()
            w = m.head.weight
            got = [getattr(w, "grad_dot_prod", None), getattr(w, "train_grad", None),
                   getattr(m.head, "_ghost_grad_proj", None)]
            assert not any(k in m.head.__dict__ for k in ("_gs_head", "_gs_dot_head", "_ghost_head"))
            for p in m.parameters():
                p.__dict__.pop("train_grad", None)
            with torch.no_grad():
                m(ids)
        return got
    order = (dots, projection) if first == "dots" else (projection, dots)
    both, alone, other = run(*order), run(dots), run(projection)
    for a, b in zip(both, (*alone[:2], other[2])):
        assert_close(a, b, 1e-6)


@pytest.mark.parametrize("vocab,pieces", [(256, 1), (257, 2), (700, 3)])
@pytest.mark.parametrize("T", [3, 40])
def test_engines_sum_over_the_vocabularys_pieces(oracle_ops, monkeypatch, tmp_path, vocab, pieces, T):   # noqa: F811
    """Dots, train gradient and projection of pieces of 256 entries, a shorter last one among them, are those of
    the whole vocabulary; both branches of the dots (2 T^2 against the weights)."""
    torch.manual_seed(3)
    net = _Net(vocab=vocab)
    ids, labels = torch.randint(0, vocab, (5, T)), torch.randint(0, vocab, (5, T))
    labels[0, 0] = -100
    got = []
    for limit in (1 << 30, 1):
        monkeypatch.setattr(lm_layers, "PIECE_BYTES", limit)
        for make in (lambda m: GradDotProdEngine(m, val_batch_size=2, use_dummy_bias=False, precision="fp32"), None):
            m = copy.deepcopy(net)
            if make is None:
                eng = _projection(m, tmp_path)
            else:
                eng = make(m)
                eng.attach(torch.optim.SGD(m.parameters(), lr=0.0))
            del oracle_ops.calls[:]
            m(ids, labels).backward()
            made = [c[1] for c in oracle_ops.calls if c[0] == "head_logit_grad"]
            assert made == ([(0, vocab)] if limit > 1 else
                            [(v, min(256, vocab - v)) for v in range(0, vocab, 256)])
            assert len(made) == (1 if limit > 1 else pieces)
            w = m.head.weight
            got.append([m.head._ghost_grad_proj] if make is None else [w.grad_dot_prod, w.train_grad])
    for whole, split in zip(got[:2], got[2:]):
        for a, b in zip(whole, split):
            assert_close(b, a, 1e-5)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("N,V,d", [(100, 2 ** 20, 4096), (524300, 50257, 4096), (262144, 300, 8192),
                                   (2, 2 ** 26, 16), (1, 2 ** 30, 2), (2 ** 24, 9, 64), (40, 70, 2 ** 20)])
def test_head_takes_every_shape_whose_grids_fit(N, V, d, dtype):
    """Past the check of the grids the missing workspace is what is refused."""
    lib = _native.load_library()
    ref = ctypes.byref(_head(N=N, V=V, d=d, x_stride=d, dtype=dtype))
    assert 0 < lib.gs_head_loss_workspace(ref) and 0 < lib.gs_head_grad_workspace(ref)
    assert lib.gs_head_loss(ref, P16, P16, None, 0, None) == -3
    assert lib.gs_head_grad(ref, P16, None, P16, P16, None, 0, None) == -3
    assert lib.gs_head_logit_grad(ref, P16, None, 0, 8, P16, 8, None, 0, None) == -3


@pytest.mark.parametrize("N,V,d,status", [(2 ** 27 + 1, 8, 8, -5), (2 ** 30, 2 ** 30, 8, -5), (2 ** 27, 8, 8, -3),
                                          (2 ** 25, 8, 1024, -5)])
def test_head_refuses_grids_beyond_a_launch(N, V, d, status):
    """2^31 threads: 16 to a row, 64 to a row of the logits' gradient, and one to four features of dx."""
    lib = _native.load_library()
    ref = ctypes.byref(_head(N=N, V=V, d=d, x_stride=d))
    assert lib.gs_head_grad(ref, P16, None, P16, P16, None, 0, None) == status
    assert lib.gs_head_grad(ref, P16, None, None, P16, None, 0, None) == (-3 if N == 2 ** 25 else status)
    assert lib.gs_head_loss(ref, P16, P16, None, 0, None) == (-3 if N == 2 ** 25 else status)
    assert lib.gs_head_logit_grad(ref, P16, None, 0, 8, P16, 8, None, 0, None) == (-3 if N == 2 ** 25 else -5)


def test_head_logit_grad_refuses_a_copy_of_the_weight_beyond_a_launch():
    """64 threads to an entry, of weights whose rows are copied; others have no copy."""
    lib = _native.load_library()
    for d, N, n, status in ((7, 40, 2 ** 25, -3), (7, 40, 2 ** 25 + 8, -5), (8, 40, 2 ** 25 + 8, -3),
                            (7, 1, 2 ** 25 + 8, -5), (6, 1, 2 ** 25 + 8, -3)):
        ref = ctypes.byref(_head(N=N, V=2 ** 28, d=d, x_stride=d))
        assert lib.gs_head_logit_grad(ref, P16, None, 0, n, P16, n, None, 0, None) == status, (d, N, n)


def test_adamw_refuses_a_state_of_adam():
    """torch.optim.Adam adds its weight decay to the gradients; without weight decay the two are one."""
    p, q = (torch.nn.Parameter(torch.ones(3)) for _ in range(2))
    p.grad = torch.ones(3)
    for decay in (0.1, 0.0):
        adam = torch.optim.Adam([p], lr=0.02, weight_decay=decay)
        adam.step()
        opt = AdamW([q], lr=7.0)
        if decay:
            with pytest.raises(_native.GhostHipError, match="state of Adam"):
                opt.load_state_dict(adam.state_dict())
            assert opt.param_groups[0]["lr"] == 7.0 and not opt.state
        else:
            opt.load_state_dict(adam.state_dict())
            assert opt.param_groups[0]["lr"] == 0.02 and opt.state[q]["step"] == 1
