"""The output projection with its cross entropy, the root-mean-square norm and AdamW without a GPU: the
float64 forms against differences and against torch, the layers under the engines, the optimizer's host
side, and what the C entry points refuse."""
import copy
import ctypes
import math
import warnings

import pytest
import torch
from torch import nn

import ghostsuite_amd as gs
from ghostsuite_amd import AdamW, GradDotProdEngine, GradProjLoraEngine, _native
from ghostsuite_amd import supported_layers_grad_samplers_dotprod as samplers
from ghostsuite_amd.workloads import CausalLM, LMConfig
from oracle import brute
from tests import train_forms as L
from tests.helpers import assert_close, gen, randn


@pytest.fixture
def oracle_ops():
    saved = _native._backend
    ops = L.TrainOracleOps()
    _native._install_backend(ops)
    yield ops
    _native._install_backend(saved)


# ------------------------------------------------------------------------------- the forms
def test_forms_against_differences():
    x, w = (randn(s, k).double().requires_grad_() for s, k in (((4, 3), 1), ((5, 3), 2)))
    labels = torch.tensor([2, -100, 0, 4])
    for reduction in ("mean", "sum", "none"):
        torch.autograd.gradcheck(lambda a, b: L.head_loss(a, b, labels, reduction), (x, w))
        ref = nn.functional.cross_entropy(x @ w.t(), labels, reduction=reduction)
        assert torch.allclose(L.head_loss(x, w, labels, reduction), ref)
    torch.autograd.gradcheck(lambda a, b: L.norm_form(a, b, 1e-6), (x, w[0].detach().requires_grad_()))


def test_gradients_of_the_bounds_are_the_forms():
    """head_all's and norm_all's closed gradients are the forms' automatic ones."""
    x, w = randn((6, 5), 1).double().requires_grad_(), randn((9, 5), 2).double().requires_grad_()
    labels = torch.tensor([2, -100, 0, 8, -100, 5])
    for reduction in ("mean", "sum", "none"):
        up = torch.rand(6 if reduction == "none" else (), generator=gen(3))
        got = L.head_all(x, w, labels, up, reduction, torch.float32)
        loss = L.head_loss(x, w, labels, reduction)
        dx, dw = torch.autograd.grad(loss, (x, w), up.double())
        for name, value in (("loss", loss.detach()), ("dx", dx), ("dw", dw)):
            assert torch.allclose(got[name][0], value, atol=1e-12), (reduction, name)
        dz = L.head_dz(x.detach(), w.detach(), labels, up, 0, 9, reduction)
        assert torch.allclose(dz @ w, dx)
    gy, gh = randn((6, 5), 4).double(), randn((6, 5), 5).double()
    got = L.norm_all(x, w[0], gy, gh, 1e-6, torch.float32)
    w0 = w[0].detach().requires_grad_()
    dx, dw = torch.autograd.grad(L.norm_form(x, w0, 1e-6), (x, w0), gy)
    assert torch.allclose(got["dh"][0], dx + gh) and torch.allclose(got["dw"][0], dw)


def test_adamw_form_is_torchs():
    p = randn((7, 3), 1).double()
    ours, theirs = p.clone(), nn.Parameter(p.clone())
    opt = torch.optim.AdamW([theirs], lr=0.01, betas=(0.8, 0.9), eps=1e-6, weight_decay=0.3)
    m = root = torch.zeros_like(p)
    for step in range(1, 5):
        g = randn((7, 3), 10 + step).double()
        ours, m, _, root = L.adamw_form(ours, g, m, root, 0.01, (0.8, 0.9), 1e-6, 0.3, step)
        theirs.grad = g
        opt.step()
    assert torch.allclose(ours, theirs.detach(), rtol=1e-12)


def test_chances_are_spread():
    """Means and neighbours of the hashed numbers: within six deviations of even, independent ones."""
    n = 1 << 16
    for step, seed in ((1, 0), (2, 0), (1000, 7)):
        u = L.chances(n, step, seed)
        for x in u:
            assert abs(x.mean() - 0.5) < 6 * math.sqrt(1 / 12 / n)
            assert abs(((x[1:] - 0.5) * (x[:-1] - 0.5)).mean()) < 6 / 12 / math.sqrt(n)
        assert abs(((u[0] - 0.5) * (u[1] - 0.5)).mean()) < 6 / 12 / math.sqrt(n)
        other = L.chances(n, step + 1, seed)[0]
        assert abs(((u[0] - 0.5) * (other - 0.5)).mean()) < 6 / 12 / math.sqrt(n)


def test_held_values_are_8_bit_values():
    a = torch.cat((torch.linspace(0, 448, 4001), torch.logspace(-6, 2.6, 4001))).double()
    for u in (0.0, 0.5, 0.999):
        q = L.held(a, torch.full_like(a, u)).clamp(max=448.0)
        assert torch.equal(q.float().to(torch.float8_e4m3fn).float().double(), q)
        assert ((q - a).abs() <= L.grid_step(a)).all()


# ------------------------------------------------------------------- layers under the engines
class _Net(nn.Module):
    """Embedding, norms with and without a residual, and the head (tied to the embedding or not)."""

    def __init__(self, tied=False, vocab=13, d=6, reduction="mean"):
        super().__init__()
        self.emb = nn.Embedding(vocab, d)
        self.n1, self.n2 = gs.RMSNorm(d), gs.RMSNorm(d, eps=1e-3)
        self.fc = nn.Linear(d, d)
        self.head = gs.HeadCrossEntropy(d, vocab, reduction=reduction)
        if tied:
            self.head.weight = self.emb.weight
        with torch.no_grad():
            for n in (self.n1, self.n2):
                n.weight.copy_(1 + 0.3 * randn((d,), 5))

    def hidden(self, ids):
        x = self.emb(ids)
        y, h = self.n2(self.fc(self.n1(x)), x)
        return y + 0.5 * h

    def forward(self, ids, labels=None):
        return self.head(self.hidden(ids), labels)


def _plain_loss(net, ids, labels):
    """The same model from elementary operations."""
    def norm(n, h):
        return n.weight * h / torch.sqrt((h * h).mean(-1, keepdim=True) + n.eps)
    x = net.emb.weight[ids]
    h = net.fc(norm(net.n1, x)) + x
    z = (norm(net.n2, h) + 0.5 * h) @ net.head.weight.t()
    return z


@pytest.mark.parametrize("T", [1, 4, 9])
@pytest.mark.parametrize("few_entries", [False, True])
def test_engine_dots_and_gradients(oracle_ops, monkeypatch, T, few_entries):
    """Both branches of the switch (2 T^2 against 78 weights), the vocabulary whole and in pieces."""
    if few_entries:
        real = gs.lm_layers.head_gradient_pieces

        def pieces(layer, x, labels, lse, grad):
            for v0 in range(0, 13, 5):
                n = min(5, 13 - v0)
                yield v0, n, _native.ops().head_logit_grad(x, layer.weight.detach(), labels, lse, grad, v0,
                                                           n, layer.ignore_index, layer.reduction)
        assert real is samplers.head_gradient_pieces
        monkeypatch.setattr(samplers, "head_gradient_pieces", pieces)
    torch.manual_seed(1)
    n, n_val = 6, 2
    net = _Net()
    ids = torch.randint(0, 13, (n, T))
    labels = torch.randint(0, 13, (n, T))
    labels[0, 0] = -100
    ref = copy.deepcopy(net).double()
    eng = GradDotProdEngine(net, val_batch_size=n_val, use_dummy_bias=False, precision="fp32")
    eng.attach(torch.optim.SGD(net.parameters(), lr=0.0))
    net(ids, labels).backward()
    kept = int((labels != -100).sum())
    per_sample = brute.per_sample_grads(
        ref, ids, labels,
        lambda m, x, y: nn.functional.cross_entropy(_plain_loss(m, x, y).flatten(0, -2), y.flatten(),
                                                    reduction="sum"), 1.0 / kept)
    for name, p in net.named_parameters():
        g = per_sample[name].double()
        if name in ("emb.weight",):
            continue
        train, val = g[:n - n_val].flatten(1), g[n - n_val:].flatten(1)
        if name == "fc.weight" or (name == "head.weight" and not 2 * T * T <= p.numel()):
            continue   # summed over the val samples before the product: another quantity
        assert_close(p.grad_dot_prod, train @ val.sum(0), 1e-4, name)
    for name, p in net.named_parameters():
        want = per_sample[name].double()[:n - n_val].sum(0) * n / (n - n_val)
        assert_close(p.train_grad, want, 1e-4, name)
    assert "_gs_head" not in net.head.__dict__
    eng.detach()


def test_engine_head_is_a_linear_of_its_logits(oracle_ops):
    """Dots and train gradient equal those of an nn.Linear whose logits go into torch's loss, on both
    branches, tied (the dot left to the embedding) and untied, and without labels."""
    for tied in (False, True):
        for T in (3, 9):
            torch.manual_seed(2)
            a = _Net(tied)
            b = copy.deepcopy(a)
            ids, labels = torch.randint(0, 13, (5, T)), torch.randint(0, 13, (5, T))
            got = []
            for net, loss in ((a, lambda m: m(ids, labels)),
                              (b, lambda m: nn.functional.cross_entropy(m(ids).flatten(0, 1),
                                                                        labels.flatten()))):
                eng = GradDotProdEngine(net, val_batch_size=2, use_dummy_bias=False, precision="fp32")
                eng.attach(torch.optim.SGD(net.parameters(), lr=0.0))
                loss(net).backward()
                got.append({k: (p.grad_dot_prod.clone(), p.train_grad.clone())
                            for k, p in net.named_parameters()})
                eng.detach()
            for k in got[0]:
                assert_close(got[0][k][0], got[1][k][0], 1e-5, k)
                assert_close(got[0][k][1], got[1][k][1], 1e-5, k)


@pytest.mark.parametrize("reduction", ["sum", "none"])
@pytest.mark.parametrize("again", [False, True])
def test_engine_head_with_weighted_losses_and_recomputation(oracle_ops, reduction, again):
    """The rows' losses weighted outside the layer, the forward pass run again within the backward one:
    still a Linear of its logits."""
    from torch.utils.checkpoint import checkpoint
    torch.manual_seed(2)
    a = _Net()
    a.head.reduction = reduction
    b = copy.deepcopy(a)
    ids, labels = torch.randint(0, 13, (5, 3)), torch.randint(0, 13, (5, 3))
    labels[1, 1] = -100
    weights = torch.rand(5, 3) + 0.5 if reduction == "none" else torch.tensor(0.3)

    def theirs(net):
        loss = nn.functional.cross_entropy(net(ids).flatten(0, 1), labels.flatten(), reduction=reduction)
        return (loss * weights.reshape(loss.shape)).sum()

    def ours(net):
        loss = checkpoint(net, ids, labels, use_reentrant=False) if again else net(ids, labels)
        return (loss * weights).sum()
    got = []
    for net, loss in ((a, ours), (b, theirs)):
        eng = GradDotProdEngine(net, val_batch_size=2, use_dummy_bias=False, precision="fp32")
        eng.attach(torch.optim.SGD(net.parameters(), lr=0.0))
        loss(net).backward()
        got.append({k: (p.grad_dot_prod.clone(), p.train_grad.clone()) for k, p in net.named_parameters()})
        eng.detach()
    for k in got[0]:
        assert_close(got[0][k][0], got[1][k][0], 1e-5, k)
        assert_close(got[0][k][1], got[1][k][1], 1e-5, k)


def test_engine_with_an_unused_norm_output(oracle_ops):
    """A norm of whose outputs only the stream is used has dots and a gradient of zero."""
    net = nn.ModuleDict({"n": gs.RMSNorm(4)})
    net.forward = lambda x, r: net["n"](x, r)[1]
    eng = GradDotProdEngine(net, val_batch_size=1, use_dummy_bias=False)
    eng.attach(torch.optim.SGD(net.parameters(), lr=0.0))
    x = randn((3, 2, 4), 1).requires_grad_()
    net["n"](x, randn((3, 2, 4), 2))[1].sum().backward()
    w = net["n"].weight
    assert (w.grad_dot_prod == 0).all() and (w.train_grad == 0).all()
    eng.detach()


def test_projection_of_the_head(oracle_ops, tmp_path):
    """GradProjLoraEngine projects a head that ended in its loss as a Linear of its logits."""
    torch.manual_seed(3)
    a = _Net()
    b = copy.deepcopy(a)
    ids, labels = torch.randint(0, 13, (5, 4)), torch.randint(0, 13, (5, 4))
    got = []
    for net, loss in ((a, lambda m: m(ids, labels)),
                      (b, lambda m: nn.functional.cross_entropy(m(ids).flatten(0, 1), labels.flatten()))):
        eng = GradProjLoraEngine(net, proj_layers="head", proj_rank_total=8, proj_rank_min=2, proj_seed=1,
                                 proj_dtype="float32", proj_dir=str(tmp_path), proj_save_interval=100,
                                 include_embeddings=False)
        eng.attach()
        loss(net).backward()
        got.append(net.head._ghost_grad_proj.clone())
    assert_close(got[0], got[1], 1e-5)


@pytest.mark.parametrize("rotary", [False, True])
def test_causal_lm_takes_them(oracle_ops, rotary):
    """The model with the norm and the loss is the one from elementary operations, with and without
    labels; the defaults are as before."""
    cfg = LMConfig(n_layer=2, n_head=2, d_model=16, d_mlp=24, vocab=31, n_ctx=8, rotary=rotary,
                   tied=not rotary, norm="rms", head_loss=True)
    torch.manual_seed(0)
    model = CausalLM(cfg)
    plain = CausalLM(LMConfig(**{**cfg.__dict__, "head_loss": False}))
    plain.load_state_dict(model.state_dict())
    ids = torch.randint(0, 31, (3, 8))
    labels = torch.randint(0, 31, (3, 8))
    labels[1, 3:] = -100
    assert torch.equal(model(ids), plain(ids))
    a, b = model(ids, labels), plain(ids, labels)
    assert torch.allclose(a, b, rtol=1e-5)
    ga = torch.autograd.grad(a, list(model.parameters()))
    gb = torch.autograd.grad(b, list(plain.parameters()))
    for x, y in zip(ga, gb):
        assert torch.allclose(x, y, atol=1e-6)

    # the residual stream by hand
    def norm(n, h):
        return n.weight * h / torch.sqrt((h * h).mean(-1, keepdim=True) + n.eps)
    x = model.wte(ids)
    if not rotary:
        x = x + model.wpe(torch.arange(8).expand(3, 8))
    rope = model._rope(8, x.device, x.dtype) if rotary else None
    for blk in model.h:
        x = x + blk._attend(norm(blk.ln_1, x), rope)
        x = x + blk._mlp(norm(blk.ln_2, x))
    assert torch.allclose(norm(model.ln_f, x) @ model.lm_head.weight.t(), model(ids), atol=1e-5)
    with pytest.raises(ValueError, match="norm"):
        CausalLM(LMConfig(n_layer=1, d_model=8, n_head=1, vocab=5, norm="batch"))


def test_step_of_the_whole_set(oracle_ops):
    """Model, engine and optimizer together: the parameters after two steps are those of elementary
    operations on the train rows' gradients."""
    torch.manual_seed(4)
    net = _Net()
    ref = copy.deepcopy(net).double()
    opt = AdamW(net.parameters(), lr=0.01, betas=(0.8, 0.9), weight_decay=0.1)
    ropt = torch.optim.AdamW(ref.parameters(), lr=0.01, betas=(0.8, 0.9), weight_decay=0.1)
    eng = GradDotProdEngine(net, val_batch_size=2, use_dummy_bias=False, precision="fp32")
    eng.attach(opt)
    for step in range(2):
        ids, labels = torch.randint(0, 13, (6, 4)), torch.randint(0, 13, (6, 4))
        eng.attach_train_batch(ids[:4], labels[:4], step, 0)
        net(ids, labels).backward()
        eng.prepare_gradients()
        opt.step()
        eng.aggregate_and_log()
        eng.clear_gradients()
        opt.zero_grad(set_to_none=True)
        nn.functional.cross_entropy(_plain_loss(ref, ids[:4], None).flatten(0, 1),
                                    labels[:4].flatten()).backward()
        ropt.step()
        ropt.zero_grad()
    for (name, p), q in zip(net.named_parameters(), ref.parameters()):
        assert_close(p, q.detach(), 1e-4, name)
    assert len(eng.dot_product_log) == 2
    eng.detach()


# --------------------------------------------------------------------- the optimizer's host side
@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_state_and_reload(oracle_ops, bits):
    def params():
        return [nn.Parameter(randn(s, k, 1.0, t)) for k, (s, t) in enumerate(
            [((5, 3), torch.float32), ((300,), torch.bfloat16), ((0,), torch.float32), ((), torch.float32)])]

    def grads(ps, seed):
        for k, p in enumerate(ps):
            p.grad = randn(p.shape, seed + k, 1.0, p.dtype)
    a, b = params(), params()
    oa = AdamW(a, state_bits=bits, seed=3)
    ob = AdamW(b, lr=7.0, state_bits=32)
    for step in range(3):
        grads(a, 10 * step)
        oa.step()
    saved = copy.deepcopy(oa.state_dict())
    with torch.no_grad():
        for p, q in zip(a, b):
            q.copy_(p)
    ob.load_state_dict(saved)
    for p, q in zip(a, b):
        for name, value in oa.state[p].items():
            mine = ob.state[q][name]
            if not isinstance(value, torch.Tensor):
                assert mine == value == 3
                continue
            assert mine.dtype == value.dtype and mine.data_ptr() != value.data_ptr() or not value.numel()
            assert torch.equal(mine.float(), value.float())
            assert value.dtype == (torch.float32 if bits == 32 or "scale" in name
                                   else torch.float8_e4m3fn)
    grads(a, 99)
    grads(b, 99)
    oa.step()
    ob.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_adamw_steps_apart_and_missing_gradients(oracle_ops):
    """Parameters that got a gradient at other steps count their own; those without one stay."""
    a, b, c = (nn.Parameter(torch.ones(4)) for _ in range(3))
    opt = AdamW([a, b, c], lr=0.1)
    a.grad = torch.ones(4)
    opt.step()
    b.grad = torch.ones(4)
    opt.step()
    assert opt.state[a]["step"] == 2 and opt.state[b]["step"] == 1 and c not in opt.state
    assert [x[1] for x in oracle_ops.calls] == [(1, 1), (1, 2), (1, 1)]
    assert torch.equal(c, torch.ones(4))
    assert opt.step(lambda: torch.tensor(3.0)) == 3.0


@pytest.mark.parametrize("bad", [dict(lr=-1.0), dict(lr=math.nan), dict(lr=torch.tensor(0.1)),
                                 dict(eps=-1e-8), dict(weight_decay=math.inf), dict(betas=(1.0, 0.9)),
                                 dict(betas=(0.9, -0.1)), dict(betas=(0.9,)), dict(state_bits=16)])
def test_adamw_refuses(bad):
    with pytest.raises(_native.GhostHipError):
        AdamW([nn.Parameter(torch.zeros(2))], **bad)
    opt = AdamW([nn.Parameter(torch.zeros(2))])
    with pytest.raises(_native.GhostHipError):
        opt.add_param_group({"params": [nn.Parameter(torch.zeros(2))], **bad})
    assert len(opt.param_groups) == 1


def test_adamw_refuses_a_parameter_twice():
    p, q = (nn.Parameter(torch.zeros(2)) for _ in range(2))
    opt = AdamW([q])
    with pytest.raises(_native.GhostHipError, match="twice"), warnings.catch_warnings():
        warnings.simplefilter("ignore")   # torch's own
        AdamW([("a", p), ("b", p)])
    for params in ([p, p], iter([p, p])):
        with pytest.raises(_native.GhostHipError, match="twice"), warnings.catch_warnings():
            warnings.simplefilter("ignore")
            opt.add_param_group({"params": params})
        assert len(opt.param_groups) == 1


def test_adamw_goes_on_from_torchs_state(oracle_ops):
    """Of fp32 parameters: the same next step, within an fp32 rounding of each of its seven operations."""
    a, b = (nn.Parameter(randn((40, 7), 1)) for _ in range(2))
    ta = torch.optim.AdamW([a], lr=0.02, betas=(0.8, 0.95), weight_decay=0.3)
    for k in range(3):
        a.grad = randn((40, 7), 5 + k)
        ta.step()
    ob = AdamW([b])
    with torch.no_grad():
        b.copy_(a)
    ob.load_state_dict(copy.deepcopy(ta.state_dict()))
    assert ob.state[b]["step"] == 3 and isinstance(ob.state[b]["step"], int)
    a.grad = b.grad = randn((40, 7), 9)
    ta.step()
    ob.step()
    assert (a - b).abs().max() <= 7 * 2 ** -24 * 4   # |p| and the steps of it below 4
    for how in ("amsgrad", "maximize"):
        other = torch.optim.AdamW([a], **{how: True})
        with pytest.raises(_native.GhostHipError, match=how):
            ob.load_state_dict(other.state_dict())


def test_averages_in_8_bits_come_out_right_on_average(oracle_ops):
    """Steady noisy gradients: with b2 = 0.999 a nearest rounding would leave v where it started.

    2048 elements, each with a size of its own, 400 steps.  m and the root are unbiased; v's bias is the
    rounding's variance, at most 1/16 of the moves of v against its drift: under a tenth here.  The mean
    over the elements of v / (size^2 (1 - b2^t)) has a deviation of sqrt(2 (1 - b2) / 2) / sqrt(2048) and
    of the rounding's walk, together below 0.01: within 0.15 of one, and well off the start."""
    size = torch.exp(randn((2048,), 1) * 0.5)
    p = nn.Parameter(torch.zeros(2048))
    opt = AdamW([p], lr=0.0, betas=(0.9, 0.999), weight_decay=0.0, state_bits=8)
    for step in range(400):
        p.grad = size * randn((2048,), 100 + step)
        opt.step()
    _, root = L.averages(opt.state[p], p.shape, 8)
    share = (root ** 2 / (size.double() ** 2 * (1 - 0.999 ** 400))).mean()
    assert abs(share - 1) < 0.15, share


# ------------------------------------------------------------------------------- refusals
class HeadStruct(ctypes.Structure):
    _fields_ = [("X", ctypes.c_void_p), ("x_stride", ctypes.c_int64), ("W", ctypes.c_void_p),
                ("dtype", ctypes.c_int), ("N", ctypes.c_int64), ("V", ctypes.c_int64),
                ("d", ctypes.c_int64), ("labels", ctypes.c_void_p), ("ignore_index", ctypes.c_int64),
                ("reduction", ctypes.c_int)]


class TensorStruct(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("p", "g", "m", "v", "m_scale", "v_scale")] + \
        [("n", ctypes.c_int64)]


P16 = ctypes.c_void_p(0x10000)


def _head(**kw):
    base = dict(X=P16, x_stride=8, W=P16, dtype=0, N=4, V=100, d=8, labels=P16, ignore_index=-100,
                reduction=2)
    return HeadStruct(**{**base, **kw})


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=2), -2), (dict(N=0), -1), (dict(V=0), -1), (dict(d=0), -1), (dict(X=None), -1),
    (dict(W=None), -1), (dict(labels=None), -1), (dict(x_stride=7), -1), (dict(reduction=3), -1),
    (dict(N=2 ** 31), -5), (dict(V=2 ** 31), -5), (dict(d=2 ** 21, x_stride=2 ** 21), -5), (dict(), -3)])
def test_head_entry_points_refuse(bad, status):
    lib = _native.load_library()
    ref = ctypes.byref(_head(**bad))
    if bad:
        assert lib.gs_head_loss_workspace(ref) == 0 and lib.gs_head_grad_workspace(ref) == 0
        assert lib.gs_head_logit_grad_workspace(ref, 0, 8) == 0
    assert lib.gs_head_loss(ref, P16, P16, None, 0, None) == status
    assert lib.gs_head_grad(ref, P16, None, P16, P16, None, 0, None) == status
    assert lib.gs_head_logit_grad(ref, P16, None, 0, 8, P16, 8, None, 0, None) == status
    assert lib.gs_last_error()


def test_head_entry_points_refuse_their_own_arguments():
    lib, ref = _native.load_library(), ctypes.byref(_head())
    assert lib.gs_head_loss(ref, None, P16, P16, 1 << 30, None) == -1
    assert lib.gs_head_loss(ref, P16, None, P16, 1 << 30, None) == -1
    assert lib.gs_head_grad(ref, None, None, P16, P16, P16, 1 << 30, None) == -1
    assert lib.gs_head_loss(None, P16, P16, P16, 1 << 30, None) == -1
    for v0, n, stride in ((-1, 8, 8), (0, 0, 0), (96, 8, 8), (0, 8, 16), (0, 9, 9)):
        assert lib.gs_head_logit_grad(ref, P16, None, v0, n, P16, stride, P16, 1 << 30, None) == -1
    assert lib.gs_head_logit_grad(ref, P16, None, 0, 8, ctypes.c_void_p(0x10008), 8, P16, 1 << 30,
                                  None) == -1
    need = lib.gs_head_grad_workspace(ref)
    assert need > 0
    assert lib.gs_head_grad(ref, P16, None, P16, P16, P16, 1000, None) == -3


def test_norm_entry_points_refuse():
    lib = _native.load_library()
    good = [P16, None, P16, 0, 4, 8, 1e-6, P16, None, None]
    for at, value, status in ((0, None, -1), (2, None, -1), (3, 2, -2), (4, 0, -1), (5, 0, -1),
                              (7, None, -1), (8, P16, -1), (1, P16, -1), (4, 2 ** 32, -5),
                              (5, 2 ** 41, -5)):
        args = list(good)
        args[at] = value
        assert lib.gs_rms_norm(*args) == status, (at, value)
    good = [P16, P16, P16, None, 0, 4, 8, 1e-6, P16, P16, None, 0, None]
    for at, value, status in ((0, None, -1), (1, None, -1), (4, 2, -2), (5, 0, -1), (6, 0, -1), (4, 0, -3)):
        args = list(good)
        args[at] = value
        assert lib.gs_rms_norm_grad(*args) == status, (at, value)
    good = [P16, P16, 0, 4, 1, 3, 2, 8, 1e-6, P16, None, 0, 1.0, None, 0, None]
    for at, value, status in ((0, None, -1), (1, None, -1), (2, 2, -2), (11, 2, -2), (4, 0, -1), (4, 4, -1),
                              (5, 4, -1), (6, 0, -1), (7, 0, -1), (2, 0, -3)):
        args = list(good)
        args[at] = value
        assert lib.gs_rms_norm_dot(*args) == status, (at, value)


def test_adamw_entry_point_refuses():
    lib = _native.load_library()
    t = TensorStruct(P16, P16, P16, P16, P16, P16, 8)

    def call(tensor=t, count=1, dtype=0, bits=32, b1=0.9, b2=0.9, eps=1e-8, step=1):
        return lib.gs_adamw(ctypes.byref(tensor) if tensor is not None else None, count, dtype, bits, 0.1,
                            b1, b2, eps, 0.0, step, 0, None)
    assert call(dtype=2) == -2
    for bad in (dict(tensor=None), dict(count=-1), dict(bits=16), dict(b1=1.0), dict(b2=-0.1),
                dict(eps=-1.0), dict(eps=math.nan), dict(b1=math.nan), dict(step=0)):
        assert call(**bad) == -1, bad
    for k in ("p", "g", "m", "v"):
        broken = TensorStruct(P16, P16, P16, P16, P16, P16, 8)
        setattr(broken, k, None)
        assert call(tensor=broken) == -1
    assert call(tensor=TensorStruct(P16, P16, P16, P16, None, P16, 8), bits=8) == -1
    assert call(tensor=TensorStruct(P16, P16, P16, P16, P16, P16, -1)) == -1
    assert call(tensor=TensorStruct(P16, P16, P16, P16, P16, P16, 2 ** 43)) == -5
    assert call(tensor=TensorStruct(P16, P16, P16, P16, P16, P16, 2 ** 34 + 1)) == -5
    assert call(tensor=None, count=0) == 0
    assert call(tensor=TensorStruct(None, None, None, None, None, None, 0)) == 0


X, W, Y = torch.zeros(2, 4), torch.zeros(5, 4), torch.tensor([0, 3])
OPERATORS = [(lambda x: gs.head_cross_entropy(x, W, Y), (2, 4)),
             (lambda w: gs.head_cross_entropy(X, w, Y), (5, 4)),
             (lambda x: gs.rms_norm(x, W[0]), (2, 4)), (lambda w: gs.rms_norm(X, w), (4,)),
             (lambda r: gs.add_rms_norm(X, r, W[0])[0], (2, 4))]


@pytest.fixture
def kernels():
    saved = _native._backend
    _native._install_backend(_native.HipOps())
    yield
    _native._install_backend(saved)


def refused(what, f, *args):
    with pytest.raises(_native.GhostHipError, match=what):
        f(*args)


@pytest.mark.parametrize("op,shape", OPERATORS)
def test_what_torch_does_around_its_operators_is_refused(kernels, op, shape):
    x = torch.randn(shape)
    refused("ROCm GPU", op, x)
    with torch.autograd.forward_ad.dual_level():
        refused("forward-mode", op, torch.autograd.forward_ad.make_dual(x, torch.ones(shape)))
    refused("transforms", torch.func.vmap(op), torch.randn(3, *shape))
    refused("transforms", torch.func.grad(lambda t: op(t).sum()), x)
    refused("traced", torch.jit.trace, op, (x,))
    refused("plain strided", op, torch.complex(x, x).conj().imag)
    refused("plain strided", op, torch._efficientzerotensor(shape))


def test_reductions_and_optimizers_on_the_cpu_are_refused(kernels):
    refused("reduction", lambda: gs.head_cross_entropy(X, W, Y, reduction="max"))
    refused("reduction", lambda: gs.HeadCrossEntropy(4, 5, reduction="max"))
    p = nn.Parameter(torch.zeros(3))
    p.grad = torch.zeros(3)
    refused("ROCm GPU", AdamW([p]).step)
    p.grad = torch.zeros(3).to_sparse()
    refused("plain strided", AdamW([p]).step)
