"""Calls that the language-model operators refuse whatever device their tensors are on: what torch does
around operators of its dispatcher would pass them by."""
import pytest
import torch

import ghostsuite_amd as gs
from ghostsuite_amd import _native

IDS = torch.tensor([0, 2])
TABLE = gs.rotary_table(8, 4)


def _lookup(w):
    return gs.embedding_lookup(IDS, w)


def _packed(x):
    return gs.qkv_norm_rotary(x.view(1, 2, 12), 1, 1, TABLE)[0]


def _separate(x):
    return gs.qk_norm_rotary(x.view(1, 2, 3, 4), torch.zeros(1, 2, 1, 4), TABLE)[1]


def _weight(w):
    return gs.qkv_norm_rotary(torch.zeros(1, 2, 12), 1, 1, TABLE, None, w, w)[0]


def _loss(z):
    return gs.distillation_loss(z, IDS[:, None], torch.zeros(2, 1))


def _teacher(t):
    return gs.distillation_loss(torch.zeros(2, 5), IDS[:, None], t)


OPERATORS = [(_lookup, (4, 6)), (_packed, (24,)), (_separate, (24,)), (_weight, (4,)), (_loss, (2, 5)),
             (_teacher, (2, 1))]


@pytest.fixture(autouse=True)
def kernels():
    saved = _native._backend
    _native._install_backend(_native.HipOps())
    yield
    _native._install_backend(saved)


def refused(what, f, *args):
    with pytest.raises(_native.GhostHipError, match=what):
        f(*args)


@pytest.mark.parametrize("op,shape", OPERATORS)
@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode(op, shape, requires_grad):
    x = torch.randn(shape, requires_grad=requires_grad)
    refused("ROCm GPU", op, x)                       # plain tensors get as far as the device
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones(shape))
        refused("forward-mode", op, dual)
    refused("transforms", torch.func.jvp, op, (x.detach(),), (torch.ones(shape),))


@pytest.mark.parametrize("op,shape", OPERATORS)
def test_function_transforms(op, shape):
    refused("transforms", torch.func.vmap(op), torch.randn(3, *shape))
    refused("transforms", torch.func.grad(lambda x: op(x).sum()), torch.randn(shape))
    refused("transforms", torch.func.functionalize(op), torch.randn(shape))


@pytest.mark.parametrize("op,shape", OPERATORS)
def test_tracing(op, shape):
    refused("traced", torch.jit.trace, op, (torch.randn(shape),))


@pytest.mark.parametrize("op,shape", OPERATORS)
def test_tensors_that_are_not_their_memory(op, shape):
    x = torch.randn(shape)
    marked = torch.complex(x, x).conj().imag         # -x, by a mark on the view
    assert marked.is_neg()
    refused("plain strided", op, marked)
    refused("plain strided", op, torch._efficientzerotensor(shape))
    from torch._subclasses import FakeTensorMode
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        refused("plain strided", op, mode.from_tensor(x))


def test_sparse_and_nested_tensors():
    refused("plain strided", _lookup, torch.eye(4).to_sparse())
    refused("plain strided", _loss, torch.randn(2, 5).to_sparse_csr())
    refused("plain strided", _loss, torch.nested.nested_tensor([torch.randn(5), torch.randn(3)]))


def test_dots_of_the_norm_weights():
    ops, w = _native.ops(), torch.ones(4)
    marked = torch.complex(w, w).conj().imag
    x, samples = torch.zeros(2, 2, 12), torch.zeros(2, 2, 4)
    refused("plain strided", ops.qk_norm_rotary_dots, x, None, (1, 1, 1), TABLE, None, marked, w, 1e-6,
            False, (None, None, None), 1)
    refused("plain strided", ops.qk_sample_dots, samples, w, marked, 1)
    refused("plain strided", ops.qk_norm_rotary, x, None, (1, 1, 1), TABLE, None, w, w, True, 1e-6,
            False, samples.to_sparse())


def test_temperatures_whose_inverse_overflows():
    import ctypes
    from tests.test_lm_layers import P16, _distill
    lib = _native.load_library()
    for tau, status in ((3e-39, -1), (4.2e-39, -1), (4.3e-39, -3), (1e-30, -3), (1.8e19, -3),
                        (1.9e19, -1)):           # -3: as far as the workspace
        ref = ctypes.byref(_distill(temperature=tau))
        assert lib.gs_distill_loss(ref, P16, None, None, 0, None) == status, tau
        assert lib.gs_distill_grad(ref, P16, 0, P16, None, 0, None) == status, tau
