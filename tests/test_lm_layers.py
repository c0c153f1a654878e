"""Host logic of the language-model operators without a GPU: refusals, the float64 forms against
differences, and the layers under both engines through the stand-in kernel layer."""
import ctypes
import math

import pytest
import torch
from torch import nn

import ghostsuite_amd as gs
from ghostsuite_amd import GradDotProdEngine, _native
from ghostsuite_amd.workloads import CausalLM, LMConfig
from oracle import brute
from tests import lm_forms as L
from tests.helpers import assert_close, randn


@pytest.fixture
def oracle_ops():
    saved = _native._backend
    ops = L.LmOracleOps()
    _native._install_backend(ops)
    yield ops
    _native._install_backend(saved)


# ------------------------------------------------------------------------------- refusals
def test_cpu_tensors_are_rejected_loudly():
    ops = _native.HipOps()
    table = gs.rotary_table(8, 4)
    with pytest.raises(_native.GhostHipError, match="ROCm GPU"):
        ops.embedding_lookup(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8), 1.0)
    with pytest.raises(_native.GhostHipError, match="ROCm GPU"):
        ops.qk_norm_rotary(torch.zeros(1, 2, 12), None, (1, 1, 1), table, None, None, None, True,
                           1e-6, False)
    with pytest.raises(_native.GhostHipError, match="ROCm GPU"):
        gs.distillation_loss(torch.zeros(2, 5), torch.zeros(2, 1, dtype=torch.int64),
                             torch.zeros(2, 1))


def test_python_refusals_before_any_device():
    w = torch.zeros(4, 8)
    with pytest.raises(_native.GhostHipError, match="padding_idx"):
        gs.embedding_lookup(torch.zeros(3, dtype=torch.int64), w, padding_idx=4)
    with pytest.raises(_native.GhostHipError, match="labels"):
        gs.distillation_loss(w, torch.zeros(4, 1, dtype=torch.int64), torch.zeros(4, 1), alpha=0.5)
    with pytest.raises(_native.GhostHipError, match="reduction"):
        gs.distillation_loss(w, torch.zeros(4, 1, dtype=torch.int64), torch.zeros(4, 1),
                             reduction="batchmean")
    with pytest.raises(_native.GhostHipError, match="even"):
        gs.rotary_table(8, 3)
    with pytest.raises(_native.GhostHipError, match="without the norm"):
        gs.qkv_norm_rotary(torch.zeros(1, 2, 12), 1, 1, gs.rotary_table(8, 4),
                           q_weight=torch.ones(4), norm=False)
    with pytest.raises(_native.GhostHipError, match="heads"):
        gs.qk_norm_rotary(torch.zeros(1, 2, 12), torch.zeros(1, 2, 12), gs.rotary_table(8, 4))
    with pytest.raises(_native.GhostHipError, match="rotated"):
        gs.QKNormRotary(1, 1, 8, n_rot=10)


class _QKShape(ctypes.Structure):   # gs_qk_shape
    _fields_ = [("dtype", ctypes.c_int), ("B", ctypes.c_int64), ("T", ctypes.c_int64),
                ("D", ctypes.c_int64), ("n_rot", ctypes.c_int64), ("heads", ctypes.c_int32 * 3),
                ("norm", ctypes.c_int), ("interleaved", ctypes.c_int), ("eps", ctypes.c_float),
                ("weight", ctypes.c_void_p * 2), ("weight_dtype", ctypes.c_int * 2),
                ("table", ctypes.c_void_p), ("n_positions", ctypes.c_int64),
                ("positions", ctypes.c_void_p), ("position_bits", ctypes.c_int),
                ("position_stride_b", ctypes.c_int64), ("position_stride_t", ctypes.c_int64)]


class _Distill(ctypes.Structure):   # gs_distill
    _fields_ = [("Z", ctypes.c_void_p), ("dtype", ctypes.c_int), ("N", ctypes.c_int64),
                ("V", ctypes.c_int64), ("inner", ctypes.c_int64), ("stride_outer", ctypes.c_int64),
                ("stride_inner", ctypes.c_int64), ("teacher_ids", ctypes.c_void_p),
                ("teacher", ctypes.c_void_p), ("teacher_dtype", ctypes.c_int), ("K", ctypes.c_int64),
                ("labels", ctypes.c_void_p), ("ignore_index", ctypes.c_int64),
                ("temperature", ctypes.c_float), ("alpha", ctypes.c_float),
                ("reduction", ctypes.c_int)]


P16 = 1 << 20   # an address that is never followed: the checks come first


def _qk_shape(**changes):
    s = _QKShape()
    s.dtype, s.B, s.T, s.D, s.n_rot, s.norm, s.eps = 0, 2, 3, 64, 64, 1, 1e-6
    s.heads[:] = (2, 1, 1)
    s.table, s.n_positions = P16, 16
    s.weight[:] = (P16, P16)
    for k, v in changes.items():
        if k == "heads":
            s.heads[:] = v
        else:
            setattr(s, k, v)
    return s


def _qk_rows(n=3):
    return (ctypes.c_int64 * 12)(*(n * [P16, 1024, 256, 64] + (3 - n) * [0, 0, 0, 0]))


@pytest.mark.parametrize("changes,status", [
    (dict(dtype=2), -2), (dict(dtype=9), -2), (dict(B=0), -1), (dict(T=0), -1), (dict(D=0), -1),
    (dict(n_rot=63), -1), (dict(n_rot=66), -1), (dict(n_rot=-2), -1), (dict(heads=(0, 0, 0)), -1),
    (dict(heads=(-1, 1, 1)), -1), (dict(table=None), -1), (dict(n_positions=0), -1),
    (dict(positions=P16, position_bits=16), -1), (dict(eps=-1.0), -1), (dict(eps=math.nan), -1),
    (dict(T=17), -1), (dict(heads=(0x7fffffff, 0x7fffffff, 2)), -5),
    (dict(D=513, n_rot=0), -5), (dict(heads=(65535, 1, 0)), -5),
    (dict(B=1 << 20, T=1 << 12), -5)])
def test_qk_arguments_are_checked_on_the_host(changes, status):
    lib = _native.load_library()
    s = _qk_shape(**changes)
    ref = ctypes.byref(s)
    rows = _qk_rows()
    assert lib.gs_qk_rotary(ref, rows, rows, None) == status
    assert lib.gs_qk_rotary_grad(ref, rows, rows, rows, P16, P16, None, None, 0, None) == status
    assert lib.gs_qk_rotary_grad(ref, rows, rows, rows, None, None, P16, None, 0, None) == status
    assert lib.gs_qk_rotary_dots(ref, rows, rows, 1, 1, P16, P16, P16, P16, 1.0, None, 0,
                                 None) == status
    assert lib.gs_qk_rotary_grad_workspace(ref, 0) == 0
    assert lib.gs_qk_rotary_grad_workspace(ref, 1) == 0
    assert lib.gs_qk_rotary_dots_workspace(ref) == 0
    assert b"gs_qk_rotary" in lib.gs_last_error()


def test_qk_pointers_and_workspaces_are_checked_on_the_host():
    lib = _native.load_library()
    ref, rows, none = ctypes.byref(_qk_shape()), _qk_rows(), _qk_rows(0)
    assert lib.gs_qk_rotary(None, rows, rows, None) == -1
    assert lib.gs_qk_rotary(ref, None, rows, None) == -1
    assert lib.gs_qk_rotary(ref, rows, none, None) == -1
    assert lib.gs_qk_rotary_grad(ref, rows, rows, None, None, None, None, None, 0, None) == -1
    assert lib.gs_qk_rotary_grad(ref, none, rows, rows, None, None, None, None, 0, None) == -1
    assert lib.gs_qk_rotary_grad(ref, rows, rows, rows, P16, None, None, None, 0, None) == -3
    assert lib.gs_qk_rotary_grad(ref, rows, rows, rows, None, None, P16, None, 0, None) == -3
    many = ctypes.byref(_qk_shape(B=65534, T=1))
    assert lib.gs_qk_rotary_grad(many, rows, rows, rows, None, None, P16, P16, 1 << 40, None) == -5
    need = lib.gs_qk_rotary_grad_workspace(ref, 0)
    assert need > 0
    unweighted = _qk_shape()
    unweighted.weight[:] = (None, None)
    assert lib.gs_qk_rotary_grad(ctypes.byref(unweighted), rows, rows, rows, P16, None, None, P16,
                                 need, None) == -1
    assert lib.gs_qk_rotary_grad(ctypes.byref(_qk_shape(norm=0)), rows, rows, rows, None, None, P16,
                                 P16, need, None) == -1          # sums of weights without the norm
    assert lib.gs_qk_rotary_dots(ref, rows, rows, 2, 0, P16, P16, P16, P16, 1.0, P16, 1 << 20,
                                 None) == -1                     # no train sample
    assert lib.gs_qk_rotary_dots(ref, rows, rows, 1, 2, P16, P16, P16, P16, 1.0, P16, 1 << 20,
                                 None) == -1                     # val block past the end
    assert lib.gs_qk_rotary_dots(ref, rows, rows, 1, 1, P16, P16, P16, P16, 1.0, None, 0,
                                 None) == -3
    assert lib.gs_qk_rotary_dots(ctypes.byref(_qk_shape(norm=0)), rows, rows, 1, 1, P16, P16, P16,
                                 P16, 1.0, P16, 1 << 20, None) == -1


def test_qk_sample_dots_arguments_are_checked_on_the_host():
    f = _native.load_library().gs_qk_sample_dots
    need = _native.load_library().gs_qk_sample_dots_workspace(129, 64)
    assert need > 0 == _native.load_library().gs_qk_sample_dots_workspace(128, 64)
    ok = [P16, 129, 64, 2, 127, P16, P16, P16, 0, P16, 1, 1.0, P16, need, None]
    for change, status in (({0: None}, -1), ({1: 0}, -1), ({2: 0}, -1), ({3: 0}, -1), ({3: 129}, -1),
                           ({4: 128}, -1), ({4: -1}, -1), ({8: 2}, -2), ({10: 7}, -2),
                           ({1: 65534}, -5), ({2: 513, 13: 1 << 20}, -5), ({12: None}, -3),
                           ({13: need - 1}, -3)):
        args = [change.get(i, v) for i, v in enumerate(ok)]
        assert f(*args) == status, change


def _distill(**changes):
    d = _Distill()
    d.Z, d.dtype, d.N, d.V, d.inner, d.stride_outer, d.stride_inner = P16, 0, 6, 100, 6, 0, 100
    d.teacher_ids = d.teacher = d.labels = P16
    d.teacher_dtype, d.K, d.ignore_index = 0, 4, -100
    d.temperature, d.alpha, d.reduction = 2.0, 0.5, 2
    for k, v in changes.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("changes,status", [
    (dict(dtype=2), -2), (dict(teacher_dtype=2), -2), (dict(Z=None), -1),
    (dict(teacher_ids=None), -1), (dict(teacher=None), -1), (dict(N=0), -1), (dict(V=0), -1),
    (dict(K=0), -1), (dict(inner=4), -1), (dict(inner=0), -1), (dict(stride_inner=99), -1),
    (dict(inner=3, stride_outer=99), -1), (dict(temperature=0.0), -1),
    (dict(temperature=math.inf), -1), (dict(temperature=math.nan), -1),
    (dict(temperature=1e-39), -1), (dict(temperature=1e30), -1), (dict(alpha=-0.1), -1),
    (dict(alpha=1.1), -1), (dict(alpha=math.nan), -1), (dict(labels=None), -1),
    (dict(reduction=3), -1), (dict(Z=P16 + 1), -1), (dict(K=1025), -5), (dict(N=1 << 31,
                                                                             inner=1 << 31), -5)])
def test_distill_arguments_are_checked_on_the_host(changes, status):
    lib = _native.load_library()
    d = _distill(**changes)
    ref = ctypes.byref(d)
    assert lib.gs_distill_loss(ref, P16, None, P16, 1 << 20, None) == status
    assert lib.gs_distill_grad(ref, P16, 0, P16, P16, 1 << 20, None) == status
    assert lib.gs_distill_workspace(ref) == 0


def test_distill_pointers_and_workspaces_are_checked_on_the_host():
    lib = _native.load_library()
    ref = ctypes.byref(_distill())
    assert lib.gs_distill_workspace(ref) > 0
    assert lib.gs_distill_loss(None, P16, None, P16, 1 << 20, None) == -1
    assert lib.gs_distill_loss(ref, None, None, P16, 1 << 20, None) == -1
    assert lib.gs_distill_loss(ref, P16, None, None, 0, None) == -3
    assert lib.gs_distill_loss(ref, P16, P16 + 2, P16, 1 << 20, None) == -1   # grad's alignment
    assert lib.gs_distill_grad(ref, P16, 0, None, P16, 1 << 20, None) == -1
    assert lib.gs_distill_grad(ref, None, 1, P16, P16, 1 << 20, None) == -1
    assert lib.gs_distill_grad(ref, P16, 0, P16, None, 0, None) == -3


def test_lookup_arguments_are_checked_on_the_host():
    f = _native.load_library().gs_embedding_lookup
    assert f(P16, 64, 4, P16, 2, 10, 8, 1.0, -1, P16, None, None) == -2
    for bad in ((None, 64, 4, P16, 0, 10, 8), (P16, 16, 4, P16, 0, 10, 8),
                (P16, 64, 0, P16, 0, 10, 8), (P16, 64, 4, None, 0, 10, 8),
                (P16, 64, 4, P16, 0, 0, 8), (P16, 64, 4, P16, 0, 10, 0)):
        assert f(*bad, 1.0, -1, P16, None, None) == -1
    assert f(P16, 64, 4, P16, 0, 10, 1 << 30, 1.0, -1, P16, None, None) == -5
    assert f(P16, 64, 1 << 40, P16, 0, 10, 8, 1.0, -1, P16, None, None) == -5


def test_lookup_gradient_arguments_are_checked_on_the_host():
    lib = _native.load_library()
    f, size = lib.gs_embedding_lookup_grad, lib.gs_embedding_lookup_grad_workspace
    assert size(256, 50257, 768) == 0 < size(257, 50257, 768)
    assert f(P16, P16, 2, 4, 10, 8, 1.0, P16, None, 0, None) == -2
    for bad in ((None, P16, 0, 4, 10, 8), (P16, None, 0, 4, 10, 8), (P16, P16, 0, 0, 10, 8),
                (P16, P16, 0, 4, 0, 8), (P16, P16, 0, 4, 10, 0)):
        assert f(*bad, 1.0, P16, None, 0, None) == -1
    assert f(P16, P16, 0, 4, 10, 8, 1.0, None, None, 0, None) == -1
    assert f(P16, P16, 0, 257, 10, 8, 1.0, P16, None, 0, None) == -3


# ---------------------------------------------------------------- the forms, by differences
def _difference(f, x, d, h=1e-6):
    return (f(x + h * d) - f(x - h * d)) / (2 * h)


@pytest.mark.parametrize("interleaved", [False, True])
def test_qk_form_against_differences(interleaved):
    heads, D, n_rot = (3, 2, 2), 10, 6
    plan = L.plan(heads, gs.rotary_table(40, n_rot), torch.tensor([[3, 30, 7], [0, 1, 39]]),
                  interleaved=interleaved)
    x = randn((2, 3, sum(heads) * D), 1).double()
    qw, kw = 1 + randn((D,), 2).double(), 1 + randn((D,), 3).double()
    grads = [randn((2, h, 3, D), 4 + h).double() for h in heads]
    (dx,), dq, dk = L.qk_grads(plan, (x,), qw, kw, grads)
    for what, at, got, f in (
            ("x", x, dx, lambda v: L.qk_all(plan, (v,), qw, kw)),
            ("q", qw, dq, lambda v: L.qk_all(plan, (x,), v, kw)),
            ("k", kw, dk, lambda v: L.qk_all(plan, (x,), qw, v))):
        d = randn(at.shape, 9).double()
        want = _difference(lambda v: sum((y * g).sum() for y, g in zip(f(v), grads)), at, d)
        assert abs((got * d).sum() - want) <= 1e-7 * (1 + abs(want)), what


def test_distill_form_against_differences_and_cross_entropy():
    N, V, K = 5, 17, 4
    z = randn((N, V), 1, 2.0).double()
    ids = torch.stack([torch.randperm(V)[:K] for _ in range(N)])
    ids[1] = -1                 # no teacher
    ids[2, 3] = ids[2, 0]       # an id twice
    t = randn((N, K), 2, 3.0).double()
    labels = torch.tensor([3, 4, 0, -100, 16])
    for tau, alpha in ((1.0, 1.0), (2.0, 0.3), (0.7, 0.0)):
        def loss(v):
            return L.reduced(*L.distill_rows(v, ids, t, labels, tau, alpha), "mean")
        zz = z.clone().requires_grad_()
        g, = torch.autograd.grad(loss(zz), zz)
        d = randn(z.shape, 3).double()
        assert abs((g * d).sum() - _difference(loss, z, d)) <= 1e-7
        assert (g[3] == 0).all()
    assert abs(loss(z) - nn.functional.cross_entropy(z, labels)) < 1e-12
    # the formula of the gradient, with the doubled id
    tau, alpha, n = 2.0, 1.0, 2
    zz = z.clone().requires_grad_()
    g, = torch.autograd.grad(L.distill_rows(zz, ids, t, None, tau, alpha)[0].sum(), zz)
    P = torch.zeros(V, dtype=torch.float64).index_add(0, ids[n], torch.softmax(t[n] / tau, 0))
    assert torch.allclose(g[n], tau * (torch.softmax(z[n] / tau, 0) - P), atol=1e-12)


# ------------------------------------------------------------------------------ the layers
def test_rotary_table_is_float64_rounded_once():
    t = gs.rotary_table(70000, 6, 500.0)
    a = torch.arange(70000, dtype=torch.float64)[:, None] * \
        500.0 ** (-torch.arange(3, dtype=torch.float64) / 3)
    assert t.shape == (70000, 2, 3) and t.dtype == torch.float32
    # an angle's own rounding (float64: 70000 2^-53), then one rounding of its cosine
    assert (t[:, 0].double() - a.cos()).abs().max() <= 2 ** -25 + 1e-10
    assert (t[:, 1].double() - a.sin()).abs().max() <= 2 ** -25 + 1e-10
    assert gs.rotary_table(3, 0).shape == (3, 2, 0)


def test_qk_layer_keeps_its_table_in_fp32_when_cast():
    layer = gs.QKNormRotary(2, 1, 8, n_positions=16).to(torch.bfloat16)
    assert layer.q_weight.dtype == torch.bfloat16 and layer.table.dtype == torch.float32
    assert torch.equal(layer.table, gs.rotary_table(16, 8))
    assert set(layer.state_dict()) == {"q_weight", "k_weight"}
    assert gs.QKNormRotary(2, 1, 9, norm=False).n_rot == 8
    assert list(gs.QKNormRotary(2, 1, 8, norm=False).parameters()) == []
    meta = gs.QKNormRotary(2, 1, 8, n_positions=16, device="meta")
    assert meta.table.is_meta
    assert torch.equal(meta.to_empty(device="cpu").table, layer.table)


def test_layers_have_forward_and_gradients(oracle_ops):
    emb = gs.ScaledEmbedding(11, 6, padding_idx=-2)
    assert emb.padding_idx == 9 and emb.scale == math.sqrt(6)
    ids = torch.tensor([[1, 9, 3], [3, 3, 0]], dtype=torch.int32)
    y = emb(ids)
    assert torch.allclose(y, emb.weight[ids.long()] * emb.scale)
    g = randn(y.shape, 1)
    got, = torch.autograd.grad(y, emb.weight, g)
    want = L.lookup_grad(ids, g.double(), 11, emb.scale, 9)[0]
    assert_close(got, want, 1e-6)
    assert (got[9] == 0).all()
    layer = gs.QKNormRotary(3, 1, 4, n_positions=8)
    x = randn((2, 5, 20), 2).requires_grad_()
    q, k, v = layer(x, torch.arange(5))
    assert q.shape == (2, 3, 5, 4) and k.shape == v.shape == (2, 1, 5, 4)
    dx, = torch.autograd.grad(k.sum(), x, retain_graph=True)   # queries and values unused
    assert (dx.view(2, 5, 5, 4)[:, :, [0, 1, 2, 4]] == 0).all() and (dx != 0).any()
    with torch.no_grad():
        assert not layer(x)[0].requires_grad


# ------------------------------------------------------------------------- under the engines
class _Net(nn.Module):
    """Scaled embedding, projection, rotated heads mixed per head, and a head of classes."""

    def __init__(self, padding_idx=None):
        super().__init__()
        self.emb = gs.ScaledEmbedding(13, 8, 1.7, padding_idx=padding_idx)
        self.qkv = nn.Linear(8, (2 + 2 * 1) * 6)
        self.qk = gs.QKNormRotary(2, 1, 6, n_rot=4, n_positions=32)
        self.out = nn.Linear(2 * 6, 13)
        self.positions = None

    def forward(self, ids):
        q, k, v = self.qk(self.qkv(self.emb(ids)), self.positions)
        y = (q * k).sum(-1, keepdim=True) * v          # [B, 2, T, 6]
        return self.out(y.transpose(1, 2).flatten(2))


class _Plain(_Net):
    """The same net of plain torch operations, in float64, for per-sample gradients."""

    def forward(self, ids):
        emb, qk = self.emb, self.qk
        w = emb.weight
        if emb.padding_idx is not None:
            w = torch.where((torch.arange(13) == emb.padding_idx)[:, None], w.detach(), w)
        x = self.qkv(w[ids] * emb.scale)
        q, k, v = L.qk_all(L.plan((2, 1, 1), qk.table, self.positions, eps=qk.eps), (x,),
                           qk.q_weight, qk.k_weight)
        y = (q * k).sum(-1, keepdim=True) * v
        return self.out(y.transpose(1, 2).flatten(2))


def _per_row_loss(m, x, y):
    return nn.functional.cross_entropy(m(x).flatten(0, 1), y.flatten(), reduction="sum")


@pytest.mark.parametrize("positions", [None, "row", "batch"])
@pytest.mark.parametrize("padding_idx", [None, 4])
@pytest.mark.parametrize("dummy_bias", [False, True])
def test_engine_dots_and_train_gradients(oracle_ops, positions, padding_idx, dummy_bias):
    torch.manual_seed(0)
    n, n_val, T = 7, 3, 5
    net, plain = _Net(padding_idx), _Plain(padding_idx)
    if dummy_bias:
        net.ghost_embeddings = ("emb",)
    plain.load_state_dict(net.state_dict())
    plain.double()
    ids = torch.randint(0, 13, (n, T))
    ids[0, 1] = ids[5, 2] = 4
    Y = torch.randint(0, 13, (n, T))
    if positions == "row":
        net.positions = torch.arange(T) + 9
    elif positions == "batch":
        net.positions = torch.randint(0, 32, (n, T))
    eng = GradDotProdEngine(net, val_batch_size=n_val, use_dummy_bias=dummy_bias, precision="fp32")
    eng.attach(torch.optim.SGD(net.parameters(), lr=0.0))
    nn.functional.cross_entropy(net(ids).flatten(0, 1), Y.flatten()).backward()
    names = [k for k, _ in plain.named_parameters()]
    params = dict(net.named_parameters())
    dots = {k: params[k].grad_dot_prod for k in names}
    grads = {k: params[k].train_grad for k in names}
    eng.detach()
    # a frozen or a trained embedding: the layer's input has a gradient, its backward pass the sums
    assert [c[0] for c in oracle_ops.calls if c[0].startswith("qk_")] == ["qk_sample_dots"]
    per = {k: [] for k in names}
    for i in range(n):
        if net.positions is not None:
            plain.positions = net.positions if positions == "row" else net.positions[i:i + 1]
        plain.zero_grad()
        _per_row_loss(plain, ids[i:i + 1], Y[i:i + 1]).backward()
        for k, p in plain.named_parameters():
            per[k].append(torch.zeros_like(p) if p.grad is None else p.grad.clone())
    for k in names:
        G = torch.stack(per[k]) / (n * T)
        want = brute.pairwise_dots(G, n_val) if k != "qkv.weight" and k != "out.weight" else None
        if want is not None:
            assert_close(dots[k], want, 1e-4, k)
        # the engine averages the N-scaled train rows
        assert_close(grads[k], G[:n - n_val].sum(0) * n / (n - n_val), 1e-4, k)


def test_engine_dots_of_a_layer_without_input_gradient(oracle_ops):
    """Nothing before the layer has a gradient: the hook runs first and makes its own pass."""
    torch.manual_seed(2)
    layer = gs.QKNormRotary(2, 1, 6, n_positions=16)
    x = torch.randn(5, 4, 24)
    grads = [torch.randn(5, h, 4, 6) for h in (2, 1, 1)]
    eng = GradDotProdEngine(layer, val_batch_size=2, precision="fp32")
    eng.attach(torch.optim.SGD(layer.parameters(), lr=0.0))
    torch.autograd.backward(layer(x, torch.arange(4) + 3)[:2], grads[:2])
    grads[2] = None
    assert [c[0] for c in oracle_ops.calls] == ["qk_norm_rotary_dots"]
    got = [(w.grad_dot_prod, w.train_grad) for w in (layer.q_weight, layer.k_weight)]
    eng.detach()
    plan = L.plan((2, 1, 1), layer.table, torch.arange(4) + 3)
    _, dq, dk = L.qk_grads(plan, (x,), layer.q_weight, layer.k_weight, grads, per_sample=True)
    for (dot, grad), s in zip(got, (dq, dk)):
        assert_close(dot, s[:3] @ s[3:].sum(0), 1e-5)
        assert_close(grad, s[:3].sum(0) * 5 / 3, 1e-5)


def test_sample_gradients_are_kept_in_fp32_and_only_under_an_engine(oracle_ops):
    layer = gs.QKNormRotary(2, 1, 6, n_positions=16)
    x = torch.randn(5, 4, 24, requires_grad=True)
    eng = GradDotProdEngine(layer, val_batch_size=2, precision="fp32")
    eng.attach(torch.optim.SGD(layer.parameters(), lr=0.0))
    torch.set_default_dtype(torch.float64)
    try:
        y = layer(x)
    finally:
        torch.set_default_dtype(torch.float32)
    assert layer._gs_sample_grads.dtype == torch.float32
    sum(t.sum() for t in y).backward()
    assert layer.q_weight.grad_dot_prod.dtype == torch.float32
    eng.detach()
    layer(x)
    assert "_gs_sample_grads" not in layer.__dict__


def test_tied_scaled_embedding_keeps_both_parts(oracle_ops):
    """A tied head under a scaled embedding: the head's train gradient and the embedding's add."""
    torch.manual_seed(1)
    emb = gs.ScaledEmbedding(9, 4, 3.0)
    head = nn.Linear(4, 9, bias=False)
    head.weight = emb.weight
    net = nn.Sequential(emb, head)
    ids, Y = torch.randint(0, 9, (5, 3)), torch.randint(0, 9, (5, 3))
    eng = GradDotProdEngine(net, val_batch_size=2, precision="fp32")
    eng.attach(torch.optim.SGD(net.parameters(), lr=0.0))
    nn.functional.cross_entropy(net(ids).flatten(0, 1), Y.flatten()).backward()
    got = emb.weight.train_grad
    eng.detach()
    w = emb.weight.detach().double().requires_grad_()
    z = (w[ids[:3]] * 3.0) @ w.t()
    want, = torch.autograd.grad(nn.functional.cross_entropy(z.flatten(0, 1), Y[:3].flatten(),
                                                            reduction="sum") / 15 * 5 / 3, w)
    assert_close(got, want, 1e-5)


def test_projection_engine_takes_the_scale(oracle_ops, monkeypatch):
    from ghostsuite_amd.gradProjection.autograd_gradproj import create_projection_hooks
    seen = []
    monkeypatch.setattr(oracle_ops, "kron_embed_proj",
                        lambda ids, g, P_iT, P_o, scale=1.0, **kw: seen.append((ids, scale)),
                        raising=False)
    emb = gs.ScaledEmbedding(9, 4, 3.0, padding_idx=2)
    hooks = create_projection_hooks(emb, "emb", torch.randn(2, 9), torch.randn(3, 4))
    ids = torch.tensor([[1, 2], [2, 8]])
    hooks._compute_embedding_proj(emb, ids, torch.randn(2, 2, 4))
    assert seen[0][1] == 3.0 and seen[0][0].tolist() == [[1, -1], [-1, 8]]
    plain = nn.Embedding(9, 4, padding_idx=2)
    hooks = create_projection_hooks(plain, "emb", torch.randn(2, 9), torch.randn(3, 4))
    hooks._compute_embedding_proj(plain, ids, torch.randn(2, 2, 4))
    assert seen[1][1] == 1.0 and seen[1][0] is ids


def test_causal_lm_options_and_unchanged_default(oracle_ops):
    plain = CausalLM(LMConfig(n_layer=1, n_head=2, d_model=16, d_mlp=32, vocab=31, n_ctx=8))
    assert type(plain.wte) is nn.Embedding and not hasattr(plain.h[0], "qk")
    for rotary in (False, True):
        cfg = LMConfig(n_layer=2, n_head=2, d_model=16, d_mlp=32, vocab=31, n_ctx=8, rotary=rotary,
                       rotary_pct=0.5, tied=not rotary, qk_norm=True, embed_scale=4.0)
        lm = CausalLM(cfg)
        assert lm.h[0].qk.n_rot == (4 if rotary else 0)
        ids = torch.randint(0, 31, (3, 8))
        teacher = (torch.randint(0, 31, (3, 8, 5)), torch.randn(3, 8, 5))
        loss = lm(ids, ids, teacher, temperature=2.0, alpha=0.3)
        loss.backward()
        assert all(p.grad is not None and p.grad.isfinite().all() for p in lm.parameters())
        assert lm(ids, None, teacher).isfinite()
