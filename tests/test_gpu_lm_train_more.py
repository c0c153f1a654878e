"""The output projection's loss and the norm on the GPU, under both engines and in calls with more than one piece
of the vocabulary."""
import ctypes

import pytest
import torch
from torch import nn

import ghostsuite_amd as gs
from ghostsuite_amd import GradDotProdEngine, GradProjLoraEngine, _native, lm_layers
from tests import train_forms as L
from tests.helpers import BF16_TOL, assert_close, gen, randn
from tests.lm_bounds import within
from tests.lm_forms import HALF, U, f64
from tests.test_gpu_lm_train import _model, head_inputs
from tests.test_lm_train import _head

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


# ------------------------------------------------------------- pieces of the vocabulary
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n,T,n_val", [(6, 64, 2), (5, 50, 1), (4, 256, 2), (9, 1, 3)])
@pytest.mark.parametrize("V", [512, 700])
def test_engines_over_the_vocabularys_pieces(gpu, monkeypatch, tmp_path, dtype, n, T, n_val, V):
    """Under both engines, in pieces of 256 entries and in one: dots, train gradient and projection of either
    within the type's tolerance of the other's and of float64's."""
    d = 128
    x, w, labels = head_inputs(n * T, V, d, dtype, 7)
    got, made = [], []
    real = _native.ops().head_logit_grad

    def counted(*args):
        made.append(args[5:7])
        return real(*args)
    monkeypatch.setattr(_native.ops(), "head_logit_grad", counted)
    for limit in (1 << 30, 1):
        monkeypatch.setattr(lm_layers, "PIECE_BYTES", limit)
        net = nn.Sequential()
        net.add_module("head", gs.HeadCrossEntropy(d, V).to(gpu, dtype))
        layer = net.head
        with torch.no_grad():
            layer.weight.copy_(w)
        net.forward = layer.forward
        for which in ("dots", "projection"):
            del made[:]
            if which == "dots":
                eng = GradDotProdEngine(net, val_batch_size=n_val, use_dummy_bias=True,
                                        precision="fp32" if dtype == FP32 else "reference")
                eng.attach(torch.optim.SGD(layer.parameters(), lr=0.0))
            else:
                eng = projection(net, tmp_path)
                P_i, P_o = (p.double().cpu() for p in eng.projection_matrices["head"])
            xg = x.view(n, T, d).to(gpu).requires_grad_()
            layer(xg, labels.view(n, T).to(gpu)).backward()
            torch.cuda.synchronize()
            assert made == ([(0, V)] if limit > 1 else [(v, min(256, V - v)) for v in range(0, V, 256)])
            got += [layer.weight.grad_dot_prod.double().cpu(), layer.weight.train_grad.clone()] if which == "dots" \
                else [layer._ghost_grad_proj.double().cpu().clone()]
            eng.detach()
    tol = BF16_TOL if dtype == BF16 else 1e-4
    dz = L.head_dz(f64(x), f64(w), labels, torch.tensor(1.0), 0, V, "mean").view(n, T, V)
    grads = torch.stack([dz[i].t() @ f64(x).view(n, T, d)[i] for i in range(n)])
    # A dot of one branch is a sum over pairs of tokens of (dz_s dz_t)(x_s x_t), whose addends cancel.  With bf16
    # operands each dz is rounded once (two HALF), and each of the two products once more (two HALF) before their
    # product; dz itself is off by 10^-4 of itself at most (its logits' sums), so a dot by (4 HALF + 3e-4) of its
    # addends' sizes, second-order terms in the rest; fp32 likewise with U.
    sizes = torch.stack([dz[i].abs().t() @ f64(x).view(n, T, d)[i].abs() for i in range(n)])
    exact, bound = ((t[:n - n_val] * t[n - n_val:].sum(0)).sum((1, 2)) for t in (grads, sizes))
    bound = bound * (4 * HALF[dtype] + 3e-4)
    mine = labels.clone()
    mine[(n - n_val) * T:] = -100
    # the train rows' part of the whole batch's mean, times samples over train samples
    share = torch.tensor(float((mine != -100).sum()) / float((labels != -100).sum()) * n / (n - n_val))
    for dots, train, proj in (got[:3], got[3:]):
        if 2 * T * T <= V * d:   # the other branch sums the val samples' rows first: another quantity
            within(dots, exact, bound, "dots")
        within(train, *L.head_all(x, w, mine, share, "mean", dtype)["dw"], "train gradient")
        want = n * torch.stack([P_o @ g @ P_i.t() for g in grads])
        assert_close(proj.reshape(want.shape), want, tol, "projection")
    if 2 * T * T > V * d:
        assert_close(got[3], got[0], tol, "dots of the pieces")


def test_head_fp32_gradients_of_several_pieces(gpu):
    """fp32 rows whose pieces of 1 GiB of the logits' gradient are three: the weight is split into its parts a piece
    at a time, dx added up over them, and the last one is shorter."""
    N, V, d = 21000, 20000, 40
    x, w, labels = head_inputs(N, V, d, FP32, 5)
    up = torch.rand(N, generator=gen(6)) + 0.5
    xg, wg, yg = x.to(gpu).requires_grad_(), w.to(gpu).requires_grad_(), labels.to(gpu)
    need = _native.load_library().gs_head_grad_workspace(
        ctypes.byref(_head(N=N, V=V, d=d, x_stride=d, dtype=1, reduction=0)))
    assert 0 < need < 6 * N * V / 2   # less than half of the whole in three parts of 2 bytes
    loss = gs.head_cross_entropy(xg, wg, yg, reduction="none")
    dx, dw = torch.autograd.grad(loss, (xg, wg), up.to(gpu))
    part = torch.randperm(N, generator=gen(1))[:200]
    want = L.head_all(x[part], w, labels[part], up[part], "none", FP32)
    within(loss[part.to(gpu)], *want["loss"], "loss")
    within(dx[part.to(gpu)], *want["dx"], "dx")
    lse = torch.empty(N, 2, device=gpu)
    _native.ops().head_cross_entropy(xg.detach(), wg.detach(), yg, -100, "none", lse)
    for v0 in (0, 8448 - 300, 2 * 8448 - 300, V - 300):
        dz = _native.ops().head_logit_grad(xg.detach(), wg.detach(), yg, lse, up.to(gpu), v0, 300, -100,
                                           "none")[:, :300].double().t().contiguous()
        rows = xg.detach().double()
        ref, size = dz @ rows, dz.abs() @ rows.abs()
        # dz within U of either side's, six products of parts, the sums' terms and the output's rounding
        within(dw[v0:v0 + 300], ref.cpu(), (ref.abs() * U + (18 * N + 64) * U * size).cpu(), "dw")


# --------------------------------------------------------------------------- autocast
def test_norm_under_autocast(gpu):
    """fp32 weights with bf16 rows, fp32 rows or both: in fp32, as torch's norms; operands of one type as they are."""
    with torch.autocast("cuda", dtype=torch.bfloat16):
        for dtypes in ((BF16, BF16), (BF16, FP32), (FP32, BF16), (FP32, FP32)):
            x, res = (randn((5, 7, 96), k, 1.0, t).to(gpu).requires_grad_() for k, t in enumerate(dtypes))
            norm = gs.RMSNorm(96).to(gpu)
            with torch.no_grad():
                norm.weight.copy_(1 + 0.3 * randn((96,), 9))
            y, h = norm(x, res)
            alone = norm(x)
            assert y.dtype == h.dtype == alone.dtype == FP32
            gy, gh = randn(y.shape, 3).to(gpu), randn(y.shape, 4).to(gpu)
            dx, dres, dw = torch.autograd.grad((y, h), (x, res, norm.weight), (gy, gh))
            assert (dx.dtype, dres.dtype, dw.dtype) == (*dtypes, FP32)
            rows = x.detach().float() + res.detach().float()
            assert torch.equal(h, rows)
            want = L.norm_all(rows, norm.weight, gy, gh, 1e-6, FP32)
            within(y, *want["y"], "y")
            within(dw, *want["dw"], "dw")
            for g, t in ((dx, dtypes[0]), (dres, dtypes[1])):
                v, b = want["dh"]
                within(g, v, b + v.abs() * HALF[t], "dx")
            within(alone, *L.norm_all(x.detach().float(), norm.weight, None, None, 1e-6, FP32)["y"], "y alone")
        half = gs.RMSNorm(96).to(gpu, BF16)
        assert half(x.detach().bfloat16()).dtype == BF16
    with pytest.raises(_native.GhostHipError):
        norm(x.detach().bfloat16())


@pytest.mark.parametrize("N", [20, 300])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_head_under_autocast(gpu, dtype, N):
    """fp32 weights and rows of either type: the loss and gradients of the operands cast to bf16, the gradients in
    the operands' own types."""
    V, d = 700, 96
    x, w, labels = head_inputs(N, V, d, BF16, 3)
    xg = x.to(dtype).to(gpu).requires_grad_()
    layer = gs.HeadCrossEntropy(d, V).to(gpu)
    with torch.no_grad():
        layer.weight.copy_(w.float() + 1e-5 * randn((V, d), 4))
    with pytest.raises(_native.GhostHipError):
        layer(x.to(gpu), labels.to(gpu))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = layer(xg, labels.to(gpu))
        assert layer(xg).dtype == BF16
    dx, dw = torch.autograd.grad(loss, (xg, layer.weight))
    assert loss.dtype == FP32 and dx.dtype == dtype and dw.dtype == FP32
    want = L.head_all(x, layer.weight.detach().bfloat16().cpu(), labels, torch.tensor(1.0), "mean", BF16)
    for got, name in ((loss, "loss"), (dx, "dx"), (dw, "dw")):
        within(got, *want[name], name)


@pytest.mark.parametrize("tied", [True, False])
def test_engine_step_of_a_model_under_autocast(gpu, tied):
    """fp32 parameters under bf16 autocast: a model with the norm and the head's loss, its dots and train gradients
    beside those of the model whose logits go into torch's loss."""
    n, n_val, T = 6, 2, 32
    ids = torch.randint(0, 501, (n, T), generator=gen(1)).to(gpu)
    labels = torch.randint(0, 501, (n, T), generator=gen(2)).to(gpu)
    labels[0, :5] = -100
    got = []
    for head, cast in ((True, True), (False, True), (False, False)):
        model = _model(FP32, gpu, tied=tied, norm="rms", head_loss=head)
        eng = GradDotProdEngine(model, val_batch_size=n_val, use_dummy_bias=True,
                                precision="reference" if cast else "fp32")
        opt = gs.AdamW(model.parameters(), lr=1e-3, state_bits=8)
        eng.attach(opt)
        eng.attach_train_batch(ids[:4], labels[:4], 0, 0)
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=cast):
            loss = model(ids, labels)
        loss.backward()
        dots = {k: p.grad_dot_prod.double() for k, p in model.named_parameters() if hasattr(p, "grad_dot_prod")}
        eng.prepare_gradients()
        assert all(p.grad.dtype == FP32 for p in model.parameters() if p.grad is not None)
        grads = {k: p.grad.double() for k, p in model.named_parameters() if p.grad is not None}
        opt.step()
        eng.aggregate_and_log()
        eng.clear_gradients()
        eng.detach()
        got.append((loss.detach(), dots, grads))
    ref = got.pop()
    assert_close(got[0][0], got[1][0], BF16_TOL, "loss")
    # Both casted models round on the way, and their sums' addends cancel, so no bound relative to an element holds;
    # but the head's roundings are a part of the other's (no logits and no loss's gradient in bf16), so the 2-norm
    # of its error against the fp32 model is at most the other's but for chance, which twice covers for 64 elements
    # or more: a gradient's, and all dots together, each layer's as shares of their norm.
    assert got[0][1].keys() == got[1][1].keys() == ref[1].keys() and got[0][2].keys() == got[1][2].keys()
    ours, theirs = (torch.cat([(g[1][k] - v) / v.norm() for k, v in ref[1].items()]).norm() for g in got)
    assert ref[1] and sum(v.numel() for v in ref[1].values()) >= 64
    assert ours <= 2 * theirs, f"dots off by {ours:.3g}, from logits {theirs:.3g}"
    for k, want in ref[2].items():
        ours, theirs = ((g[2][k] - want).norm() for g in got)
        assert ours <= 2 * theirs, f"gradient {k}: off by {ours:.3g}, from logits {theirs:.3g}"


def test_projection_of_a_head_under_autocast(gpu, tmp_path):
    n, T, V, d = 5, 60, 900, 64
    net = Shifting(V, d, FP32, gpu)
    x = randn((n, T, d), 1).to(gpu)
    labels = torch.randint(0, V, (n, T), generator=gen(2)).to(gpu)
    eng = projection(net, tmp_path)
    got = []
    for cast in (True, False):
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=cast):
            loss = net(x, labels)
        loss.backward()
        got.append(net.head._ghost_grad_proj.clone())
    assert_close(got[0], got[1], BF16_TOL, "projection")
    eng.detach()
