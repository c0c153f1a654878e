"""The output projection's loss, the norm and the optimizer without a GPU: what the engines keep, mark and split
on the way, and what the entry points take."""
import pytest
import torch
from torch import nn

import ghostsuite_amd as gs
from ghostsuite_amd import GradProjLoraEngine
from ghostsuite_amd.gradProjection import autograd_gradproj
from tests.test_lm_train import _Net, oracle_ops   # noqa: F401  (a fixture)


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
    kept, lse = net.head.__dict__["_gs_head"]
    loss.backward()
    assert any(t is kept for t in marked) and any(t is lse for t in marked)
    assert "_gs_head" not in net.head.__dict__ and net.head._ghost_grad_proj is not None
