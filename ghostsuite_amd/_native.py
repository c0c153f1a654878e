"""ctypes binding of libghost_hip.so (include/ghost_hip.h) and torch-tensor wrappers.

Every wrapper takes device tensors, checks shapes on the host, sizes and allocates the
workspace from torch's caching allocator, and launches on torch's current stream; no call
synchronises.  There is no CPU path: a tensor that is not on a ROCm device, or a missing
library, raises.

Host-logic tests swap the kernel layer for a checker through ``_install_backend`` (the
samplers call ``ops()``); product code never does.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import math
import threading
from typing import Optional, Tuple

import torch

from . import build as _build

# gs_dtype / gs_semantics / gs_algo / gs_rounding / gs_proj_layout / gs_reduction (include/ghost_hip.h)
DTYPE_BF16, DTYPE_F32, DTYPE_F16 = 0, 1, 2
SEM_PAIRWISE_SUM, SEM_PRESUM = 0, 1
ALGO_AUTO, ALGO_GHOST, ALGO_VALGRAD = 0, 1, 2
ROUND_FP32, ROUND_REF_BF16 = 0, 1
PROJ_KO_KI, PROJ_KI_KO = 0, 1
REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
ERR_UNSUPPORTED = -5  # gs_status GS_ERR_UNSUPPORTED: a valid request outside the kernels' limits
ABI_VERSION = 2

_TORCH_TO_GS = {torch.bfloat16: DTYPE_BF16, torch.float32: DTYPE_F32, torch.float16: DTYPE_F16}
ALGO_NAMES = {ALGO_AUTO: "auto", ALGO_GHOST: "ghost", ALGO_VALGRAD: "valgrad"}


class GhostHipError(RuntimeError):
    """A libghost_hip.so entry point returned an error status."""


_lock = threading.Lock()
_lib: Optional[ctypes.CDLL] = None

_I64 = ctypes.c_int64
_P = ctypes.c_void_p
_I = ctypes.c_int
_F = ctypes.c_float
_SZ = ctypes.c_size_t

_SIGNATURES = {
    "gs_abi_version": (_I, []),
    "gs_last_error": (ctypes.c_char_p, []),
    "gs_linear_dot_workspace": (_SZ, [_I, _I64, _I64, _I64, _I64, _I64, _I, _I, _I]),
    "gs_linear_dot_algo": (_I, [_I, _I64, _I64, _I64, _I64, _I64, _I, _I, _I]),
    "gs_linear_dot": (_I, [_P, _P, _I, _I64, _I64, _I64, _I64, _I64, _I64, _I, _I, _I,
                           _P, _P, _P, _SZ, _P]),
    "gs_linear_dot_noalloc_bytes": (_SZ, [_P, _P, _I, _I64, _I64, _I64, _I64, _I64, _I, _I,
                                         _I]),
    "gs_linear_dot_noalloc": (_I, [_P, _P, _I, _I64, _I64, _I64, _I64, _I64, _I64, _I, _I,
                                   _I, _P, _P, _P]),
    "gs_bias_dot_workspace": (_SZ, [_I64, _I64, _I64]),
    "gs_bias_dot": (_I, [_P, _I, _I64, _I64, _I64, _I64, _I64, _P, _P, _I, _F, _P, _SZ, _P]),
    "gs_embedding_dot_workspace": (_SZ, [_I64, _I64, _I64, _I64, _I64]),
    "gs_embedding_dot": (_I, [_P, _P, _I, _I64, _I64, _I64, _I64, _I64, _I64, _P, _P, _SZ,
                              _P]),
    "gs_embedding_train_grad_workspace": (_SZ, [_I64, _I64, _I64, _I64, _I64]),
    "gs_embedding_layer_pass_workspace": (_SZ, [_I64, _I64, _I64, _I64, _I64]),
    "gs_embedding_layer_pass": (_I, [_P, _P, _I, _I64, _I64, _I64, _I64, _I64, _I64, _P, _F, _P,
                                     _I, _I, _P, _SZ, _P]),
    "gs_embedding_train_grad": (_I, [_P, _P, _I, _I64, _I64, _I64, _I64, _I64, _I64, _F, _P,
                                     _I, _I, _P, _SZ, _P]),
    "gs_layernorm_dot_workspace": (_SZ, [_I64, _I64, _I64]),
    "gs_layernorm_dot": (_I, [_P, _P, _I, _I64, _I64, _I64, _I64, _I64, _F, _P, _P, _P, _P,
                              _I, _F, _P, _SZ, _P]),
    "gs_kron_proj_workspace": (_SZ, [_I64, _I64, _I64, _I64]),
    "gs_kron_proj": (_I, [_P, _P, _I, _I64, _I64, _I64, _I64, _P, _P, _I, _I64, _I64, _I, _F,
                          _P, _I, _P, _SZ, _P]),
    "gs_kron_embed_proj": (_I, [_P, _P, _I, _I64, _I64, _I64, _P, _P, _I, _I64, _I64, _I64, _F,
                                _P, _I, _P, _SZ, _P]),
    "gs_linear_rowdot_workspace": (_SZ, [_I, _I64, _I64, _I64, _I64, _I64]),
    "gs_linear_val_gradient_workspace": (_SZ, [_I, _I64, _I64, _I64, _I64, _I64, _I]),
    "gs_linear_val_gradient": (_I, [_P, _P, _I, _I64, _I64, _I64, _I64, _I64, _I64, _I, _P,
                                    _P, _SZ, _P]),
    "gs_linear_dot_train_grad_workspace": (_SZ, [_I, _I64, _I64, _I64, _I64, _I64, _I, _I]),
    "gs_linear_dot_train_grad": (_I, [_P, _P, _I, _I64, _I64, _I64, _I64, _I64, _I64, _I, _P,
                                      _P, _I, _F, _P, _P, _I, _F, _P, _SZ, _P]),
    "gs_conv1d_dot_train_grad_workspace": (_SZ, [_I, _I64, _I64, _I64, _I64, _I64, _I, _I]),
    "gs_conv1d_dot_train_grad": (_I, [_P, _P, _I, _I64, _I64, _I64, _I64, _I64, _I64, _I, _P,
                                      _P, _I, _F, _P, _P, _I, _F, _P, _SZ, _P]),
    "gs_linear_layer_pass_workspace": (_SZ, [_I, _I64, _I64, _I64, _I64, _I64, _I, _I, _I, _I,
                                             _I]),
    "gs_linear_layer_pass": (_I, [_P, _P, _I, _I64, _I64, _I64, _I64, _I64, _I64, _I, _I, _P, _I,
                                  _P, _I, _F, _P, _I, _P, _I, _F, _P, _SZ, _P]),
    "gs_linear_train_grad_workspace": (_SZ, [_I, _I64, _I64, _I64, _I64, _I64]),
    "gs_linear_train_grad": (_I, [_P, _P, _I, _I64, _I64, _I64, _I64, _I64, _I64, _F, _P, _I,
                                  _I, _P, _SZ, _P]),
    "gs_linear_rowdot_bias_workspace": (_SZ, [_I, _I64, _I64, _I64, _I64, _I64]),
    "gs_linear_rowdot_bias": (_I, [_P, _P, _P, _I, _I64, _I64, _I64, _I64, _I64, _I64, _P, _P,
                                   _P, _I, _F, _P, _SZ, _P]),
    "gs_linear_rowdot": (_I, [_P, _P, _P, _I, _I64, _I64, _I64, _I64, _I64, _I64, _P, _P, _SZ,
                              _P]),
    "gs_linear_bias_dot_workspace": (_SZ, [_I, _I64, _I64, _I64, _I64, _I64, _I]),
    "gs_linear_bias_dot": (_I, [_P, _P, _I, _I64, _I64, _I64, _I64, _I64, _I64, _I, _P, _P, _P,
                                _I, _F, _P, _SZ, _P]),
    "gs_ordered_sum": (_I, [_P, _P, _I, _I64, _P, _I, _P]),
    "gs_embedding_lookup": (_I, [_P, _I, _I64, _P, _I, _I64, _I64, _F, _I64, _P, _P, _P]),
    "gs_qk_rotary": (_I, [_P, _P, _P, _P]),
    "gs_qk_rotary_grad_workspace": (_SZ, [_P]),
    "gs_qk_rotary_grad": (_I, [_P, _P, _P, _P, _P, _P, _P, _SZ, _P]),
    "gs_qk_rotary_dots_workspace": (_SZ, [_P]),
    "gs_qk_rotary_dots": (_I, [_P, _P, _P, _I64, _I64, _P, _P, _P, _P, _F, _P, _SZ, _P]),
    "gs_distill_workspace": (_SZ, [_P]),
    "gs_distill_loss": (_I, [_P, _P, _P, _P, _SZ, _P]),
    "gs_distill_grad": (_I, [_P, _P, _I, _P, _P, _SZ, _P]),
}


class _QKShape(ctypes.Structure):   # gs_qk_shape
    _fields_ = [("dtype", _I), ("B", _I64), ("T", _I64), ("D", _I64), ("n_rot", _I64),
                ("heads", ctypes.c_int32 * 3), ("norm", _I), ("interleaved", _I), ("eps", _F),
                ("weight", _P * 2), ("weight_dtype", _I * 2), ("table", _P),
                ("n_positions", _I64), ("positions", _P), ("position_bits", _I),
                ("position_stride_b", _I64), ("position_stride_t", _I64)]


# gs_qk_rows[3]: (data, stride_b, stride_t, stride_h) of each part, eight bytes each.
_QKRows3 = _I64 * 12


class _Distill(ctypes.Structure):   # gs_distill
    _fields_ = [("Z", _P), ("dtype", _I), ("N", _I64), ("V", _I64), ("inner", _I64),
                ("stride_outer", _I64), ("stride_inner", _I64), ("teacher_ids", _P),
                ("teacher", _P), ("teacher_dtype", _I), ("K", _I64), ("labels", _P),
                ("ignore_index", _I64), ("temperature", _F), ("alpha", _F), ("reduction", _I)]


def load_library() -> ctypes.CDLL:
    """Loads libghost_hip.so (built in-tree by ghostsuite_amd.build) once per process."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        path = _build.library_path()
        if not path.exists():
            raise GhostHipError(
                f"{path} is not built: run `python -c 'import __graft_entry__ as g; g.build()'` "
                "or `python ghostsuite_amd/build.py` first")
        lib = ctypes.CDLL(str(path))
        for name, (res, args) in _SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        ver = lib.gs_abi_version()
        if ver != ABI_VERSION:
            raise GhostHipError(f"libghost_hip ABI {ver}, expected {ABI_VERSION}")
        _lib = lib
        return lib


def exported_symbols() -> list:
    return list(_SIGNATURES)


def _check(rc: int, what: str) -> None:
    if rc != 0:
        msg = load_library().gs_last_error().decode(errors="replace")
        raise GhostHipError(f"{what} failed ({rc}): {msg}")


def _gs_dtype(t: torch.Tensor) -> int:
    try:
        return _TORCH_TO_GS[t.dtype]
    except KeyError:
        raise GhostHipError(f"unsupported dtype {t.dtype}") from None


def _require_device(*ts: torch.Tensor) -> torch.device:
    dev = None
    for t in ts:
        if t is None:
            continue
        if t.device.type != "cuda":
            raise GhostHipError(
                "ghostsuite_amd kernels need tensors on a ROCm GPU device; got a tensor on "
                f"{t.device} (there is no CPU path)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise GhostHipError(f"tensors on different devices: {dev} and {t.device}")
    return dev


def _stream(dev: torch.device) -> int:
    """The current stream's handle (without the stream object torch.cuda.current_stream makes)."""
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    return torch._C._cuda_getCurrentRawStream(idx)


@functools.lru_cache(maxsize=4096)
def _size(query: str, *args: int) -> int:
    """A workspace query's answer: the host plan of the call, which depends on its sizes alone."""
    return getattr(load_library(), query)(*args)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _workspace(nbytes: int, dev: torch.device) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=dev)


def _tokens(x: torch.Tensor, n: int, feat: int) -> int:
    if x.dim() < 2 or x.shape[0] != n:
        raise GhostHipError(f"expected a [N, ..., F] tensor with N={n}, got {tuple(x.shape)}")
    return x.numel() // (n * feat) if n * feat > 0 else 0


def _on(dev: torch.device):
    """Kernels launch on the current device: makes `dev` that one for the body."""
    if dev.index is None or dev.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(dev)


def _kernel_dtype(t: torch.Tensor, what: str) -> int:
    if t.dtype not in (torch.bfloat16, torch.float32):
        raise GhostHipError(f"{what}: bf16 or fp32, got {t.dtype}")
    return _TORCH_TO_GS[t.dtype]


def _features_contiguous(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


class _QKCall:
    """The arguments of a gs_qk_rotary* call from a plan (the keywords of
    lm_layers.qkv_norm_rotary) and its input rows: one packed tensor, or queries and keys."""

    __slots__ = ("dev", "heads", "B", "T", "D", "dtype", "dt", "parts", "keep", "shape")

    def __init__(self, plan, parts, qw, kw):
        heads, table, positions = plan["heads"], plan["table"], plan["positions"]
        self.dev = _require_device(*parts, qw, kw, table, positions)
        self.parts = parts = [_features_contiguous(p) for p in parts]
        self.heads = heads
        x, total = parts[0], sum(heads)
        if min(heads[0], heads[1]) <= 0:
            raise GhostHipError(f"{heads[0]} query and {heads[1]} key heads")
        size = x.shape
        if len(parts) == 1 and not (len(size) == 3 and size[2] % total == 0) and \
                not (len(size) == 4 and size[2] == total):
            raise GhostHipError(f"qkv {tuple(size)} does not hold {total} heads")
        self.B, self.T = B, T = size[0], size[1]
        self.D = D = size[2] // total if len(size) == 3 else size[3]
        if D <= 0:
            raise GhostHipError("heads without features")
        self.dtype = x.dtype
        self.dt = dt = _kernel_dtype(x, "queries and keys")
        for p in parts[1:]:
            if p.shape[:2] != size[:2] or p.shape[3] != D or p.dtype != x.dtype:
                raise GhostHipError(f"queries {tuple(size)} {x.dtype} and keys "
                                    f"{tuple(p.shape)} {p.dtype} disagree")
        if table.dim() != 3 or table.shape[1] != 2 or table.dtype != torch.float32 or \
                not table.is_contiguous() or 2 * table.shape[2] > D:
            raise GhostHipError(f"table {tuple(table.shape)} {table.dtype}: contiguous fp32 "
                                f"[positions, 2, n_rot / 2] with n_rot up to {D} expected")
        n_rot = 2 * table.shape[2]
        w_ptr, w_dt = [None, None], [dt, dt]
        self.keep = [table, positions]   # alive until the call is enqueued
        for i, w in enumerate((qw, kw)):
            if w is None:
                continue
            if w.shape != (D,):
                raise GhostHipError(f"norm weight {tuple(w.shape)}: [{D}] expected")
            w_dt[i] = _kernel_dtype(w, "norm weights")
            if not w.is_contiguous():
                w = w.contiguous()
                self.keep.append(w)
            w_ptr[i] = w.data_ptr()
        pos, bits, p_sb, p_st = None, 0, 0, 0
        if positions is not None and n_rot:
            if positions.dtype not in (torch.int32, torch.int64) or \
                    tuple(positions.shape) not in ((T,), (1, T), (B, T)):
                raise GhostHipError(f"positions {tuple(positions.shape)} {positions.dtype}: int32 "
                                    f"or int64 [{T}] or [{B}, {T}] expected")
            pos, bits = positions.data_ptr(), 32 if positions.dtype == torch.int32 else 64
            p_st = positions.stride(-1)
            if positions.dim() == 2 and positions.shape[0] == B:
                p_sb = positions.stride(0)
        self.shape = _QKShape(dt, B, T, D, n_rot, heads, plan["norm"], plan["interleaved"],
                              plan["eps"], tuple(w_ptr), tuple(w_dt),
                              table.data_ptr() if n_rot else None, table.shape[0], pos, bits, p_sb,
                              p_st)

    def rows(self, parts):
        """gs_qk_rows[3] of input-shaped tensors ([B, T, heads, D] each, or one packed)."""
        out, D, (hq, hk, hv) = [], self.D, self.heads
        if len(parts) == 1:
            x, = parts
            st = x.stride()
            sh = st[2] if len(st) == 4 else D
            p, step = x.data_ptr(), sh * x.element_size()
            return _QKRows3(p, st[0], st[1], sh, p + hq * step, st[0], st[1], sh,
                            p + (hq + hk) * step if hv else 0, st[0], st[1], sh)
        for x in parts:
            out += [x.data_ptr(), *x.stride()[:3]]
        return _QKRows3(*out)

    @staticmethod
    def heads_first(tensors):
        """gs_qk_rows[3] of [B, heads, T, D] tensors (None: data NULL)."""
        out = []
        for t in tensors:
            if t is None:
                out += (0, 0, 0, 0)
            else:
                st = t.stride()
                out += (t.data_ptr(), st[0], st[2], st[1])
        return _QKRows3(*out)

    def gradients(self, grads):
        """The output gradients as the kernels take them (features contiguous)."""
        out = []
        for h, g in zip(self.heads, grads):
            if g is not None:
                if g.shape != (self.B, h, self.T, self.D) or g.dtype != self.dtype:
                    raise GhostHipError(f"output gradient {tuple(g.shape)} {g.dtype}")
                if g.device != self.dev:
                    raise GhostHipError(f"tensors on different devices: {self.dev} and {g.device}")
                g = _features_contiguous(g)
            out.append(g)
        return out

    def workspace(self, query: str) -> int:
        """The bytes a query answers: they follow from the sizes alone."""
        s = self.shape
        return _qk_size(query, self.dt, self.B, self.T, self.D, s.n_rot, self.heads,
                        s.interleaved)


@functools.lru_cache(maxsize=4096)
def _qk_size(query, dt, B, T, D, n_rot, heads, interleaved) -> int:
    # (any table: nothing of it is read)
    shape = _QKShape(dt, B, T, D, n_rot, heads, 1, interleaved, 0.0, (None, None), (dt, dt), 256,
                     1, None, 0, 0, 0)
    return getattr(load_library(), query)(ctypes.byref(shape))


class HipOps:
    """The kernel layer the samplers call: one C-ABI call per op, async on the current stream."""

    name = "hip"

    def linear_algo(self, dtype: torch.dtype, N: int, n_val: int, T: int, d_in: int, d_out: int,
                    semantics: int, algo: int, want_pair: bool) -> int:
        lib = load_library()
        rc = lib.gs_linear_dot_algo(_TORCH_TO_GS[dtype], N, n_val, T, d_in, d_out, semantics,
                                    algo, int(want_pair))
        _check(rc if rc < 0 else 0, "gs_linear_dot_algo")
        return rc

    def linear_dot(self, A: torch.Tensor, G: torch.Tensor, n_val: int, *, val_start=None,
                   semantics: int = SEM_PAIRWISE_SUM, algo: int = ALGO_AUTO,
                   rounding: int = ROUND_FP32, want_pair: bool = False
                   ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        dev = _require_device(A, G)
        if A.dtype != G.dtype:
            raise GhostHipError(f"A and G dtypes differ: {A.dtype} vs {G.dtype}")
        A = A.contiguous()
        G = G.contiguous()
        N = A.shape[0]
        d_in, d_out = A.shape[-1], G.shape[-1]
        T = _tokens(A, N, d_in)
        if _tokens(G, N, d_out) != T:
            raise GhostHipError(f"A {tuple(A.shape)} and G {tuple(G.shape)} token counts differ")
        vs = N - n_val if val_start is None else int(val_start)
        n_t = N - n_val
        dt = _gs_dtype(A)
        lib = load_library()
        ws_bytes = lib.gs_linear_dot_workspace(dt, N, n_val, T, d_in, d_out, semantics, algo,
                                               int(want_pair))
        if ws_bytes == 0:
            raise GhostHipError(
                f"gs_linear_dot: invalid arguments N={N} n_val={n_val} T={T} d_in={d_in} "
                f"d_out={d_out} semantics={semantics} algo={algo} pair={want_pair}")
        ws = _workspace(ws_bytes, dev)
        out = torch.empty(n_t, dtype=torch.float32, device=dev)
        pair = torch.empty((n_val, n_t), dtype=torch.float32, device=dev) if want_pair else None
        rc = lib.gs_linear_dot(A.data_ptr(), G.data_ptr(), dt, N, n_val, vs, T, d_in, d_out,
                               semantics, algo, rounding, out.data_ptr(), _ptr(pair),
                               ws.data_ptr(), ws_bytes, _stream(dev))
        _check(rc, "gs_linear_dot")
        return out, pair

    def linear_dot_noalloc(self, A: torch.Tensor, G: torch.Tensor, n_val: int,
                           out: torch.Tensor, pair: Optional[torch.Tensor] = None, *,
                           val_start=None, semantics: int = SEM_PAIRWISE_SUM,
                           algo: int = ALGO_AUTO, rounding: int = ROUND_FP32) -> None:
        """gs_linear_dot_noalloc into caller-given outputs (out [n_train], pair [n_val,
        n_train] or None); nothing is allocated (A and G must be contiguous)."""
        _require_device(A, G, out, pair)
        if not (A.is_contiguous() and G.is_contiguous() and out.is_contiguous()):
            raise GhostHipError("linear_dot_noalloc: A, G and out must be contiguous")
        if A.dtype != G.dtype:
            raise GhostHipError(f"A and G dtypes differ: {A.dtype} vs {G.dtype}")
        N = A.shape[0]
        d_in, d_out = A.shape[-1], G.shape[-1]
        T = _tokens(A, N, d_in)
        if _tokens(G, N, d_out) != T:
            raise GhostHipError(f"A {tuple(A.shape)} and G {tuple(G.shape)} token counts differ")
        n_t = N - n_val
        if out.dtype != torch.float32 or out.numel() != n_t or \
                (pair is not None and (pair.dtype != torch.float32 or
                                       pair.numel() != n_val * n_t)):
            raise GhostHipError("linear_dot_noalloc: outputs must be fp32 [n_train] and "
                                "[n_val, n_train]")
        vs = N - n_val if val_start is None else int(val_start)
        rc = load_library().gs_linear_dot_noalloc(
            A.data_ptr(), G.data_ptr(), _gs_dtype(A), N, n_val, vs, T, d_in, d_out, semantics,
            algo, rounding, out.data_ptr(), _ptr(pair), _stream(A.device))
        _check(rc, "gs_linear_dot_noalloc")

    def linear_val_gradient(self, A: torch.Tensor, G: torch.Tensor, n_val: int, *,
                            val_start=None, semantics: int = SEM_PAIRWISE_SUM) -> torch.Tensor:
        """The val term V [d_out, d_in] of the val-gradient algorithm (gs_linear_val_gradient):
        sum over the val rows of g a^T, or with SEM_PRESUM the product of the val rows
        presummed per token position."""
        dev = _require_device(A, G)
        if A.dtype != G.dtype:
            raise GhostHipError(f"A and G dtypes differ: {A.dtype} vs {G.dtype}")
        A = A.contiguous()
        G = G.contiguous()
        N = A.shape[0]
        d_in, d_out = A.shape[-1], G.shape[-1]
        T = _tokens(A, N, d_in)
        if _tokens(G, N, d_out) != T:
            raise GhostHipError(f"A {tuple(A.shape)} and G {tuple(G.shape)} token counts differ")
        vs = N - n_val if val_start is None else int(val_start)
        dt = _gs_dtype(A)
        lib = load_library()
        ws_bytes = lib.gs_linear_val_gradient_workspace(dt, N, n_val, T, d_in, d_out, semantics)
        if ws_bytes == 0:
            raise GhostHipError(f"gs_linear_val_gradient: invalid arguments N={N} n_val={n_val} "
                                f"T={T} d_in={d_in} d_out={d_out} semantics={semantics}")
        ws = _workspace(ws_bytes, dev)
        V = torch.empty((d_out, d_in), dtype=A.dtype, device=dev)
        rc = lib.gs_linear_val_gradient(A.data_ptr(), G.data_ptr(), dt, N, n_val, vs, T, d_in,
                                        d_out, semantics, V.data_ptr(), ws.data_ptr(), ws_bytes,
                                        _stream(dev))
        _check(rc, "gs_linear_val_gradient")
        return V

    def linear_dot_train_grad(self, A: torch.Tensor, G: torch.Tensor, n_val: int, *,
                              val_start=None, semantics: int = SEM_PAIRWISE_SUM,
                              grad_scale: Optional[float] = None,
                              grad_dtype: Optional[torch.dtype] = None, bias: bool = False,
                              bias_grad_scale: Optional[float] = None,
                              bias_grad_dtype: Optional[torch.dtype] = None,
                              conv1d: bool = False):
        """Weight dots and weight train gradient in one pass over the train rows
        (gs_linear_dot_train_grad), with the bias dots and bias train gradient when `bias`;
        with conv1d the HF Conv1D form (gs_conv1d_dot_train_grad: train gradient [d_in, d_out]).
        Returns (dot, grad, bias_dot, bias_grad), entries not asked for None; None for the
        cases the kernels do not take (non-bf16, unaligned, T not a multiple of 64, feature
        counts not multiples of 8)."""
        dev = _require_device(A, G)
        if A.dtype != G.dtype:
            raise GhostHipError(f"A and G dtypes differ: {A.dtype} vs {G.dtype}")
        A = A.contiguous()
        G = G.contiguous()
        N = A.shape[0]
        d_in, d_out = A.shape[-1], G.shape[-1]
        T = _tokens(A, N, d_in)
        if _tokens(G, N, d_out) != T:
            raise GhostHipError(f"A {tuple(A.shape)} and G {tuple(G.shape)} token counts differ")
        vs = N - n_val if val_start is None else int(val_start)
        dt = _gs_dtype(A)
        lib = load_library()
        name = "gs_conv1d_dot_train_grad" if conv1d else "gs_linear_dot_train_grad"
        ws_bytes = getattr(lib, name + "_workspace")(dt, N, n_val, T, d_in, d_out, semantics,
                                                     1 if bias else 0)
        if ws_bytes == 0:
            return None
        ws = _workspace(ws_bytes, dev)
        n_t = N - n_val
        dot = torch.empty(n_t, dtype=torch.float32, device=dev)
        grad = None
        if grad_scale is not None:
            grad = torch.empty((d_in, d_out) if conv1d else (d_out, d_in),
                               dtype=grad_dtype or A.dtype, device=dev)
        bdot = torch.empty(n_t, dtype=torch.float32, device=dev) if bias else None
        bgrad = None
        if bias and bias_grad_scale is not None:
            bgrad = torch.empty(d_out, dtype=bias_grad_dtype or A.dtype, device=dev)
        rc = getattr(lib, name)(
            A.data_ptr(), G.data_ptr(), dt, N, n_val, vs, T, d_in, d_out, semantics,
            dot.data_ptr(), _ptr(grad), _gs_dtype(grad) if grad is not None else DTYPE_BF16,
            float(grad_scale or 0.0), _ptr(bdot), _ptr(bgrad),
            _gs_dtype(bgrad) if bgrad is not None else DTYPE_BF16, float(bias_grad_scale or 0.0),
            ws.data_ptr(), ws_bytes, _stream(dev))
        if rc == ERR_UNSUPPORTED:
            return None
        _check(rc, name)
        return dot, grad, bdot, bgrad

    def linear_layer_pass(self, A: torch.Tensor, G: torch.Tensor, n_val: int, *, semantics: int,
                          algo: int, rounding: int, conv1d: bool, grad_scale: float,
                          grad_dtype: torch.dtype, dot_dtype: torch.dtype,
                          bias_grad_dtype: Optional[torch.dtype] = None,
                          bias_dot_dtype: Optional[torch.dtype] = None, val_start=None):
        """A Linear / Conv1D layer's dots and train gradients in one pass (gs_linear_layer_pass):
        any T, the dots in the dtypes asked for; the bias terms when bias_grad_dtype is given.
        Returns (dot, grad, bias_dot, bias_grad), or None where the separate passes must run or
        are faster for `algo`."""
        dev = _require_device(A, G)
        if A.dtype != G.dtype:
            raise GhostHipError(f"A and G dtypes differ: {A.dtype} vs {G.dtype}")
        A = A.contiguous()
        G = G.contiguous()
        N = A.shape[0]
        d_in, d_out = A.shape[-1], G.shape[-1]
        T = _tokens(A, N, d_in)
        if _tokens(G, N, d_out) != T:
            raise GhostHipError(f"A {tuple(A.shape)} and G {tuple(G.shape)} token counts differ")
        n_t = N - n_val
        vs = n_t if val_start is None else int(val_start)
        bias = bias_grad_dtype is not None
        dt = _gs_dtype(A)
        lib = load_library()
        ws_bytes = _size("gs_linear_layer_pass_workspace", dt, N, n_val, T, d_in, d_out,
                         semantics, int(conv1d), int(bias), algo, rounding)
        if ws_bytes == 0:
            return None
        ws = _workspace(ws_bytes, dev)
        dot = torch.empty(n_t, dtype=dot_dtype, device=dev)
        grad = torch.empty((d_in, d_out) if conv1d else (d_out, d_in), dtype=grad_dtype,
                           device=dev)
        bdot = bgrad = None
        if bias:
            bdot = torch.empty(n_t, dtype=bias_dot_dtype, device=dev)
            bgrad = torch.empty(d_out, dtype=bias_grad_dtype, device=dev)
        rc = lib.gs_linear_layer_pass(
            A.data_ptr(), G.data_ptr(), dt, N, n_val, vs, T, d_in, d_out, semantics, int(conv1d),
            dot.data_ptr(), _gs_dtype(dot), grad.data_ptr(), _gs_dtype(grad), float(grad_scale),
            _ptr(bdot), _gs_dtype(bdot) if bias else DTYPE_F32, _ptr(bgrad),
            _gs_dtype(bgrad) if bias else DTYPE_F32, float(grad_scale), ws.data_ptr(), ws_bytes,
            _stream(dev))
        if rc == ERR_UNSUPPORTED:
            return None
        _check(rc, "gs_linear_layer_pass")
        return dot, grad, bdot, bgrad

    def linear_train_grad(self, A: torch.Tensor, G: torch.Tensor, n_val: int, scale: float, *,
                          val_start=None, out_dtype: Optional[torch.dtype] = None,
                          conv1d: bool = False) -> Optional[torch.Tensor]:
        """scale * sum over the train rows of g a^T as [d_out, d_in] (Linear weight), or
        a g^T as [d_in, d_out] with conv1d (gs_linear_train_grad); None for the cases the
        kernel does not take (non-bf16 operands, unaligned rows, feature counts not multiples
        of 8, operands past 2 GiB)."""
        dev = _require_device(A, G)
        if A.dtype != G.dtype:
            raise GhostHipError(f"A and G dtypes differ: {A.dtype} vs {G.dtype}")
        A = A.contiguous()
        G = G.contiguous()
        N = A.shape[0]
        d_in, d_out = A.shape[-1], G.shape[-1]
        T = _tokens(A, N, d_in)
        if _tokens(G, N, d_out) != T:
            raise GhostHipError(f"A {tuple(A.shape)} and G {tuple(G.shape)} token counts differ")
        vs = N - n_val if val_start is None else int(val_start)
        dt = _gs_dtype(A)
        lib = load_library()
        ws_bytes = lib.gs_linear_train_grad_workspace(dt, N, n_val, T, d_in, d_out)
        if ws_bytes == 0:
            return None
        odt = out_dtype or A.dtype
        shape = (d_in, d_out) if conv1d else (d_out, d_in)
        out = torch.empty(shape, dtype=odt, device=dev)
        ws = _workspace(ws_bytes, dev)
        rc = lib.gs_linear_train_grad(A.data_ptr(), G.data_ptr(), dt, N, n_val, vs, T, d_in,
                                      d_out, float(scale), out.data_ptr(), _gs_dtype(out),
                                      1 if conv1d else 0, ws.data_ptr(), ws_bytes, _stream(dev))
        if rc == ERR_UNSUPPORTED:
            return None
        _check(rc, "gs_linear_train_grad")
        return out

    def linear_bias_dot(self, A: torch.Tensor, G: torch.Tensor, n_val: int, *, val_start=None,
                        semantics: int = SEM_PAIRWISE_SUM, algo: int = ALGO_AUTO,
                        rounding: int = ROUND_FP32, grad_scale: Optional[float] = None,
                        grad_dtype: Optional[torch.dtype] = None):
        """Weight and bias dots of a Linear layer (and the bias train gradient when
        grad_scale is given) in one pass over the train rows when the shape allows it (the
        val-gradient algorithm through gs_linear_bias_dot).  Otherwise None (the caller then
        uses linear_dot and bias_dot).  The val rows are [val_start, val_start + n_val)
        (default: the last n_val rows).  Returns (dot, bias_dot, bias_grad)."""
        dev = _require_device(A, G)
        if A.dtype != G.dtype or A.dtype != torch.bfloat16 or \
                semantics not in (SEM_PAIRWISE_SUM, SEM_PRESUM) or \
                (grad_dtype or G.dtype) not in (torch.bfloat16, torch.float32):
            return None
        N = A.shape[0]
        d_in, d_out = A.shape[-1], G.shape[-1]
        T = _tokens(A, N, d_in)
        n_t = N - n_val
        vs = N - n_val if val_start is None else int(val_start)
        if n_t <= 0 or _tokens(G, N, d_out) != T or not 0 <= vs <= N - n_val:
            return None
        dt = _gs_dtype(A)
        lib = load_library()
        if lib.gs_linear_dot_algo(dt, N, n_val, T, d_in, d_out, semantics, algo,
                                  0) != ALGO_VALGRAD:
            return None
        ws_bytes = lib.gs_linear_bias_dot_workspace(dt, N, n_val, T, d_in, d_out, semantics)
        if ws_bytes == 0:
            return None
        A = A.contiguous()
        G = G.contiguous()
        ws = _workspace(ws_bytes, dev)
        out = torch.empty(n_t, dtype=torch.float32, device=dev)
        bout = torch.empty(n_t, dtype=torch.float32, device=dev)
        gdt = grad_dtype or G.dtype
        grad = torch.empty(d_out, dtype=gdt, device=dev) if grad_scale is not None else None
        rc = lib.gs_linear_bias_dot(A.data_ptr(), G.data_ptr(), dt, N, n_val, vs, T, d_in,
                                    d_out, semantics, out.data_ptr(), bout.data_ptr(),
                                    _ptr(grad), _TORCH_TO_GS[gdt], float(grad_scale or 0.0),
                                    ws.data_ptr(), ws_bytes, _stream(dev))
        _check(rc, "gs_linear_bias_dot")
        return out, bout, grad

    def linear_rowdot_bias(self, A: torch.Tensor, G: torch.Tensor, V: torch.Tensor, n_val: int,
                           *, val_start=None, grad_scale: Optional[float] = None,
                           grad_dtype: Optional[torch.dtype] = None):
        """gs_linear_rowdot_bias with a caller-formed V [d_out, d_in] (bf16): the weight dot
        sum_t g^T V a, the bias dot and (with grad_scale) the bias train gradient of the train
        rows in one pass.  None when the shape is outside the fused pass's limits.  Returns
        (dot, bias_dot, bias_grad)."""
        dev = _require_device(A, G, V)
        if not (A.dtype == G.dtype == V.dtype == torch.bfloat16):
            return None
        A = A.contiguous()
        G = G.contiguous()
        V = V.contiguous()
        N = A.shape[0]
        d_in, d_out = A.shape[-1], G.shape[-1]
        T = _tokens(A, N, d_in)
        if _tokens(G, N, d_out) != T or tuple(V.shape) != (d_out, d_in):
            raise GhostHipError(f"shapes disagree: A {tuple(A.shape)} G {tuple(G.shape)} "
                                f"V {tuple(V.shape)}")
        vs = N - n_val if val_start is None else int(val_start)
        lib = load_library()
        ws_bytes = lib.gs_linear_rowdot_bias_workspace(DTYPE_BF16, N, n_val, T, d_in, d_out)
        if ws_bytes == 0:
            return None
        ws = _workspace(ws_bytes, dev)
        n_t = N - n_val
        out = torch.empty(n_t, dtype=torch.float32, device=dev)
        bout = torch.empty(n_t, dtype=torch.float32, device=dev)
        gdt = grad_dtype or G.dtype
        grad = torch.empty(d_out, dtype=gdt, device=dev) if grad_scale is not None else None
        rc = lib.gs_linear_rowdot_bias(A.data_ptr(), G.data_ptr(), V.data_ptr(), DTYPE_BF16, N,
                                       n_val, vs, T, d_in, d_out, out.data_ptr(), bout.data_ptr(),
                                       _ptr(grad), _TORCH_TO_GS[gdt], float(grad_scale or 0.0),
                                       ws.data_ptr(), ws_bytes, _stream(dev))
        _check(rc, "gs_linear_rowdot_bias")
        return out, bout, grad

    def linear_rowdot(self, A: torch.Tensor, G: torch.Tensor, V: torch.Tensor, n_val: int, *,
                      val_start=None) -> torch.Tensor:
        """dot_i = sum_t g_it^T V a_it over the train rows, V: [d_out, d_in]."""
        dev = _require_device(A, G, V)
        if not (A.dtype == G.dtype == V.dtype):
            raise GhostHipError(f"A, G, V dtypes differ: {A.dtype} {G.dtype} {V.dtype}")
        A = A.contiguous()
        G = G.contiguous()
        V = V.contiguous()
        N = A.shape[0]
        d_in, d_out = A.shape[-1], G.shape[-1]
        T = _tokens(A, N, d_in)
        if _tokens(G, N, d_out) != T or tuple(V.shape) != (d_out, d_in):
            raise GhostHipError(f"shapes disagree: A {tuple(A.shape)} G {tuple(G.shape)} "
                                f"V {tuple(V.shape)}")
        vs = N - n_val if val_start is None else int(val_start)
        dt = _gs_dtype(A)
        lib = load_library()
        ws_bytes = lib.gs_linear_rowdot_workspace(dt, N, n_val, T, d_in, d_out)
        if ws_bytes == 0:
            raise GhostHipError(f"gs_linear_rowdot: invalid arguments N={N} n_val={n_val} T={T}")
        ws = _workspace(ws_bytes, dev)
        out = torch.empty(N - n_val, dtype=torch.float32, device=dev)
        rc = lib.gs_linear_rowdot(A.data_ptr(), G.data_ptr(), V.data_ptr(), dt, N, n_val, vs, T,
                                  d_in, d_out, out.data_ptr(), ws.data_ptr(), ws_bytes,
                                  _stream(dev))
        _check(rc, "gs_linear_rowdot")
        return out

    def bias_dot(self, G: torch.Tensor, n_val: int, *, val_start=None,
                 grad_scale: Optional[float] = None, grad_dtype: Optional[torch.dtype] = None
                 ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        dev = _require_device(G)
        G = G.contiguous()
        N, d = G.shape[0], G.shape[-1]
        T = _tokens(G, N, d)
        vs = N - n_val if val_start is None else int(val_start)
        lib = load_library()
        ws_bytes = _size("gs_bias_dot_workspace", N, T, d)
        ws = _workspace(ws_bytes, dev)
        out = torch.empty(N - n_val, dtype=torch.float32, device=dev)
        grad = None
        if grad_scale is not None:
            grad = torch.empty(d, dtype=grad_dtype or G.dtype, device=dev)
        gdt = _gs_dtype(grad) if grad is not None else DTYPE_F32
        rc = lib.gs_bias_dot(G.data_ptr(), _gs_dtype(G), N, n_val, vs, T, d, out.data_ptr(),
                             _ptr(grad), gdt, float(grad_scale or 0.0), ws.data_ptr(), ws_bytes,
                             _stream(dev))
        _check(rc, "gs_bias_dot")
        return out, grad

    def embedding_dot(self, ids: torch.Tensor, G: torch.Tensor, n_val: int, vocab: int, *,
                      val_start=None) -> torch.Tensor:
        dev = _require_device(ids, G)
        ids = ids.to(torch.int64).contiguous()
        G = G.contiguous()
        N, d = G.shape[0], G.shape[-1]
        T = ids.numel() // N
        if _tokens(G, N, d) != T:
            raise GhostHipError(f"ids {tuple(ids.shape)} and G {tuple(G.shape)} disagree")
        vs = N - n_val if val_start is None else int(val_start)
        lib = load_library()
        ws_bytes = _size("gs_embedding_dot_workspace", N, n_val, T, d, vocab)
        if ws_bytes == 0:
            raise GhostHipError(f"gs_embedding_dot: invalid arguments N={N} n_val={n_val}")
        ws = _workspace(ws_bytes, dev)
        out = torch.empty(N - n_val, dtype=torch.float32, device=dev)
        rc = lib.gs_embedding_dot(ids.data_ptr(), G.data_ptr(), _gs_dtype(G), N, n_val, vs, T, d,
                                  vocab, out.data_ptr(), ws.data_ptr(), ws_bytes, _stream(dev))
        _check(rc, "gs_embedding_dot")
        return out

    def embedding_train_grad(self, ids: torch.Tensor, G: torch.Tensor, n_val: int,
                             scale: float, out: torch.Tensor, *, accumulate: bool = False,
                             val_start=None) -> None:
        """out[v] (+)= scale * sum of the train rows of G whose token id is v
        (gs_embedding_train_grad); out: [vocab, d] bf16 or fp32, written in place."""
        dev = _require_device(ids, G, out)
        ids = ids.to(torch.int64).contiguous()
        G = G.contiguous()
        N, d = G.shape[0], G.shape[-1]
        T = ids.numel() // N
        if _tokens(G, N, d) != T or out.dim() != 2 or out.shape[1] != d or \
                not out.is_contiguous():
            raise GhostHipError(f"embedding_train_grad: ids {tuple(ids.shape)}, G "
                                f"{tuple(G.shape)} and out {tuple(out.shape)} disagree")
        vocab = out.shape[0]
        vs = N - n_val if val_start is None else int(val_start)
        lib = load_library()
        ws_bytes = _size("gs_embedding_train_grad_workspace", N, n_val, T, d, vocab)
        if ws_bytes == 0:
            raise GhostHipError(f"gs_embedding_train_grad: invalid arguments N={N} n_val={n_val}")
        ws = _workspace(ws_bytes, dev)
        rc = lib.gs_embedding_train_grad(ids.data_ptr(), G.data_ptr(), _gs_dtype(G), N, n_val,
                                         vs, T, d, vocab, float(scale), out.data_ptr(),
                                         _gs_dtype(out), int(accumulate), ws.data_ptr(),
                                         ws_bytes, _stream(dev))
        _check(rc, "gs_embedding_train_grad")

    def embedding_layer_pass(self, ids: torch.Tensor, G: torch.Tensor, n_val: int, scale: float,
                             out: torch.Tensor, *, accumulate: bool = False,
                             val_start=None) -> Optional[torch.Tensor]:
        """embedding_dot and embedding_train_grad (into out) of one layer in shared launches
        (gs_embedding_layer_pass): the dots, or None, with nothing done, for sizes it leaves to
        the two calls."""
        dev = _require_device(ids, G, out)
        ids = ids.to(torch.int64).contiguous()
        G = G.contiguous()
        N, d = G.shape[0], G.shape[-1]
        T = ids.numel() // N
        if _tokens(G, N, d) != T or out.dim() != 2 or out.shape[1] != d or \
                not out.is_contiguous():
            raise GhostHipError(f"embedding_layer_pass: ids {tuple(ids.shape)}, G "
                                f"{tuple(G.shape)} and out {tuple(out.shape)} disagree")
        vocab = out.shape[0]
        vs = N - n_val if val_start is None else int(val_start)
        lib = load_library()
        ws_bytes = _size("gs_embedding_layer_pass_workspace", N, n_val, T, d, vocab)
        if ws_bytes == 0:
            return None
        ws = _workspace(ws_bytes, dev)
        dot = torch.empty(N - n_val, dtype=torch.float32, device=dev)
        rc = lib.gs_embedding_layer_pass(ids.data_ptr(), G.data_ptr(), _gs_dtype(G), N, n_val, vs,
                                         T, d, vocab, dot.data_ptr(), float(scale),
                                         out.data_ptr(), _gs_dtype(out), int(accumulate),
                                         ws.data_ptr(), ws_bytes, _stream(dev))
        _check(rc, "gs_embedding_layer_pass")
        return dot

    def layernorm_dot(self, X: torch.Tensor, G: torch.Tensor, n_val: int, eps: float, *,
                      val_start=None, want_dot: bool = True, want_bias: bool = True,
                      grad_scale: Optional[float] = None,
                      grad_dtype: Optional[torch.dtype] = None):
        """Returns (dot_w, dot_b, grad_w, grad_b); entries not asked for are None."""
        dev = _require_device(X, G)
        if X.dtype != G.dtype:
            raise GhostHipError(f"X and G dtypes differ: {X.dtype} vs {G.dtype}")
        X = X.contiguous()
        G = G.contiguous()
        N, F = X.shape[0], X.shape[-1]
        T = _tokens(X, N, F)
        vs = N - n_val if val_start is None else int(val_start)
        lib = load_library()
        ws_bytes = _size("gs_layernorm_dot_workspace", N, T, F)
        ws = _workspace(ws_bytes, dev)
        n_t = N - n_val
        dw = torch.empty(n_t, dtype=torch.float32, device=dev) if want_dot else None
        db = torch.empty(n_t, dtype=torch.float32, device=dev) if (want_dot and want_bias) else None
        gw = gb = None
        gdt = grad_dtype or X.dtype
        if grad_scale is not None:
            gw = torch.empty(F, dtype=gdt, device=dev)
            gb = torch.empty(F, dtype=gdt, device=dev) if want_bias else None
        rc = lib.gs_layernorm_dot(X.data_ptr(), G.data_ptr(), _gs_dtype(X), N, n_val, vs, T, F,
                                  float(eps), _ptr(dw), _ptr(db), _ptr(gw), _ptr(gb),
                                  _TORCH_TO_GS[gdt], float(grad_scale or 0.0), ws.data_ptr(),
                                  ws_bytes, _stream(dev))
        _check(rc, "gs_layernorm_dot")
        return dw, db, gw, gb

    def kron_proj(self, A: torch.Tensor, G: torch.Tensor, P_i: torch.Tensor, P_o: torch.Tensor,
                  scale: float, *, layout: int = PROJ_KO_KI,
                  out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
        dev = _require_device(A, G, P_i, P_o)
        if A.dtype != G.dtype:
            raise GhostHipError(f"A and G dtypes differ: {A.dtype} vs {G.dtype}")
        A = A.contiguous()
        G = G.contiguous()
        P_i = P_i.to(A.dtype).contiguous()
        P_o = P_o.to(A.dtype).contiguous()
        B = A.shape[0]
        n_a, n_g = A.shape[-1], G.shape[-1]
        T = A.numel() // (B * n_a)
        if G.numel() // (B * n_g) != T:
            raise GhostHipError(f"A {tuple(A.shape)} and G {tuple(G.shape)} token counts differ")
        k_i, k_o = P_i.shape[0], P_o.shape[0]
        if layout == PROJ_KO_KI:
            if P_i.shape[1] != n_a or P_o.shape[1] != n_g:
                raise GhostHipError("projection widths do not match the layer")
            shape = (B, k_o, k_i)
        else:
            if P_i.shape[1] != n_g or P_o.shape[1] != n_a:
                raise GhostHipError("projection widths do not match the layer (Conv1D roles)")
            shape = (B, k_i, k_o)
        lib = load_library()
        ws_bytes = _size("gs_kron_proj_workspace", B, T, k_i, k_o)
        ws = _workspace(ws_bytes, dev)
        out = torch.empty(shape, dtype=out_dtype, device=dev)
        rc = lib.gs_kron_proj(A.data_ptr(), G.data_ptr(), _gs_dtype(A), B, T, n_a, n_g,
                              P_i.data_ptr(), P_o.data_ptr(), _gs_dtype(P_i), k_i, k_o, layout,
                              float(scale), out.data_ptr(), _TORCH_TO_GS[out_dtype],
                              ws.data_ptr(), ws_bytes, _stream(dev))
        _check(rc, "gs_kron_proj")
        return out

    def kron_embed_proj(self, ids: torch.Tensor, G: torch.Tensor, P_iT: torch.Tensor,
                        P_o: torch.Tensor, scale: float = 1.0, *,
                        out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """out[b] = scale * sum_t (P_o g_bt)(P_iT[ids_bt])^T, [B, k_o, k_i]."""
        dev = _require_device(ids, G, P_iT, P_o)
        B = ids.shape[0]
        ids = ids.reshape(B, -1).long().contiguous()
        T = ids.shape[1]
        n_g = G.shape[-1]
        if G.numel() != B * T * n_g:
            raise GhostHipError(f"ids {tuple(ids.shape)} and G {tuple(G.shape)} disagree")
        G = G.contiguous()
        P_iT = P_iT.to(G.dtype).contiguous()
        P_o = P_o.to(G.dtype).contiguous()
        vocab, k_i = P_iT.shape
        k_o = P_o.shape[0]
        if P_o.shape[1] != n_g:
            raise GhostHipError("P_o width does not match the embedding dimension")
        lib = load_library()
        ws_bytes = lib.gs_kron_proj_workspace(B, T, k_i, k_o)
        ws = _workspace(ws_bytes, dev)
        out = torch.empty((B, k_o, k_i), dtype=out_dtype, device=dev)
        rc = lib.gs_kron_embed_proj(ids.data_ptr(), G.data_ptr(), _gs_dtype(G), B, T, n_g,
                                    P_iT.data_ptr(), P_o.data_ptr(), _gs_dtype(P_iT), vocab, k_i,
                                    k_o, float(scale), out.data_ptr(), _TORCH_TO_GS[out_dtype],
                                    ws.data_ptr(), ws_bytes, _stream(dev))
        _check(rc, "gs_kron_embed_proj")
        return out


    def ordered_sum_(self, tensors) -> torch.Tensor:
        """tensors[0] += tensors[1], then += tensors[2], ... in order, in place, in one launch
        per 48 tensors: fp32 arithmetic, each partial sum rounded to tensors[0]'s dtype (the
        in-place adds' own rounding).  Every tensor: contiguous, bf16 or fp32, the same
        number of elements, on one device.  Returns tensors[0]."""
        total = tensors[0]
        dev = _require_device(*tensors)
        n = total.numel()
        for t in tensors:
            if t.numel() != n or not t.is_contiguous() or \
                    t.dtype not in (torch.bfloat16, torch.float32):
                raise GhostHipError("ordered_sum_: contiguous bf16 / fp32 tensors of one size")
        k = len(tensors)
        ptrs = (ctypes.c_void_p * k)(*[t.data_ptr() for t in tensors])
        dts = (ctypes.c_int * k)(*[_TORCH_TO_GS[t.dtype] for t in tensors])
        rc = load_library().gs_ordered_sum(ptrs, dts, k, n, total.data_ptr(),
                                           _TORCH_TO_GS[total.dtype], _stream(dev))
        _check(rc, "gs_ordered_sum")
        return total

    # ---- embedding lookup, query / key norms with rotation, distillation (lm_layers) ----

    def embedding_lookup(self, ids: torch.Tensor, weight: torch.Tensor, scale: float,
                         padding_idx: Optional[int] = None, want_grad_ids: bool = False):
        """(scale * weight[ids], ids for embedding_grad or None): gs_embedding_lookup."""
        dev = _require_device(ids, weight)
        dt = _kernel_dtype(weight, "embedding weight")
        if ids.dtype not in (torch.int32, torch.int64):
            raise GhostHipError(f"token ids of dtype {ids.dtype}: int32 or int64 expected")
        if weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] == 0:
            raise GhostHipError(f"embedding weight {tuple(weight.shape)}: [vocab, d] expected")
        ids, weight = ids.contiguous(), weight.contiguous()
        vocab, d = weight.shape
        out = torch.empty((*ids.shape, d), dtype=weight.dtype, device=dev)
        grad_ids = None
        if want_grad_ids:
            same = padding_idx is None and ids.dtype == torch.int64
            grad_ids = ids if same else torch.empty(ids.shape, dtype=torch.int64, device=dev)
        if ids.numel():
            with _on(dev):
                rc = load_library().gs_embedding_lookup(
                    ids.data_ptr(), 32 if ids.dtype == torch.int32 else 64, ids.numel(),
                    weight.data_ptr(), dt, vocab, d, scale,
                    -1 if padding_idx is None else padding_idx, out.data_ptr(),
                    None if grad_ids is ids else _ptr(grad_ids), _stream(dev))
            _check(rc, "gs_embedding_lookup")
        return out, grad_ids

    def embedding_grad(self, ids: torch.Tensor, G: torch.Tensor, shape, dtype: torch.dtype,
                       scale: float) -> torch.Tensor:
        """scale * the rows of G added up by id, [vocab, d]: gs_embedding_train_grad over one
        sample of all the tokens."""
        dev = _require_device(ids, G)
        if not ids.numel():
            return torch.zeros(shape, dtype=dtype, device=dev)
        out = torch.empty(shape, dtype=dtype, device=dev)
        G, n, (vocab, d) = G.contiguous(), ids.numel(), shape
        ws_bytes = _size("gs_embedding_train_grad_workspace", 1, 0, n, d, vocab)
        ws = _workspace(ws_bytes, dev)
        with _on(dev):
            rc = load_library().gs_embedding_train_grad(
                ids.data_ptr(), G.data_ptr(), _kernel_dtype(G, "output gradient"), 1, 0, 1, n, d,
                vocab, scale, out.data_ptr(), _TORCH_TO_GS[dtype], 0, ws.data_ptr(), ws_bytes,
                _stream(dev))
        _check(rc, "gs_embedding_train_grad")
        return out

    def qk_norm_rotary(self, plan, parts, qw, kw):
        """Rotated queries and keys (and values), heads first: gs_qk_rotary.  plan: heads, table,
        positions, norm, eps, interleaved; parts: (qkv,) or (q, k)."""
        c = _QKCall(plan, parts, qw, kw)
        out = [torch.empty((c.B, h, c.T, c.D), dtype=c.dtype, device=c.dev)
               for h in c.heads if h]
        if c.B and c.T:
            with _on(c.dev):
                rc = load_library().gs_qk_rotary(ctypes.byref(c.shape), c.rows(c.parts),
                                                 c.heads_first(out), _stream(c.dev))
            _check(rc, "gs_qk_rotary")
        return out

    def qk_norm_rotary_grad(self, plan, parts, qw, kw, grads, *, want_x: bool, want_qw: bool,
                            want_kw: bool):
        """([input gradients] as parts or Nones, q weight gradient, k weight gradient):
        gs_qk_rotary_grad; grads: the outputs' gradients, None for zeros."""
        c = _QKCall(plan, parts, qw, kw)
        grads = c.gradients(grads)
        dparts = [torch.empty(p.shape, dtype=c.dtype, device=c.dev) if want_x else None
                  for p in parts]
        make = torch.empty if c.B and c.T else torch.zeros
        dqw = make(c.D, dtype=qw.dtype, device=c.dev) if want_qw else None
        dkw = make(c.D, dtype=kw.dtype, device=c.dev) if want_kw else None
        if c.B and c.T and (want_x or want_qw or want_kw):
            nbytes, ws = 0, None
            if want_qw or want_kw:
                nbytes = c.workspace("gs_qk_rotary_grad_workspace")
                ws = _workspace(nbytes, c.dev)
            with _on(c.dev):
                rc = load_library().gs_qk_rotary_grad(
                    ctypes.byref(c.shape), c.rows(c.parts), c.heads_first(grads),
                    c.rows(dparts) if want_x else None, _ptr(dqw), _ptr(dkw), _ptr(ws), nbytes,
                    _stream(c.dev))
            _check(rc, "gs_qk_rotary_grad")
        return dparts, dqw, dkw

    def qk_norm_rotary_dots(self, plan, parts, qw, kw, grads, n_val: int, *, val_start=None,
                            grad_scale: Optional[float] = None):
        """(dot_q, dot_k, grad_q, grad_k) of the norm weights: gs_qk_rotary_dots; the train
        gradients None without grad_scale."""
        c = _QKCall(plan, parts, qw, kw)
        if not (c.B and c.T):
            raise GhostHipError("qk_norm_rotary_dots: no tokens")
        grads = c.gradients(grads)
        n_t = c.B - n_val
        vs = n_t if val_start is None else int(val_start)
        dots = [torch.empty(max(n_t, 0), dtype=torch.float32, device=c.dev) for _ in range(2)]
        gw = [None, None]
        if grad_scale is not None:
            gw = [torch.empty(c.D, dtype=c.dtype if w is None else w.dtype, device=c.dev)
                  for w in (qw, kw)]
        nbytes = c.workspace("gs_qk_rotary_dots_workspace")
        ws = _workspace(nbytes, c.dev)
        with _on(c.dev):
            rc = load_library().gs_qk_rotary_dots(
                ctypes.byref(c.shape), c.rows(c.parts), c.heads_first(grads), n_val, vs,
                dots[0].data_ptr(), dots[1].data_ptr(), _ptr(gw[0]), _ptr(gw[1]),
                float(grad_scale or 0.0), ws.data_ptr(), nbytes, _stream(c.dev))
        _check(rc, "gs_qk_rotary_dots")
        return dots[0], dots[1], gw[0], gw[1]

    def distill_loss(self, logits, teacher_ids, teacher_logits, labels, *, temperature: float,
                     alpha: float, ignore_index: int, reduction: str, want_grad: bool = False):
        """(loss, None), or with want_grad (loss, a _DistillCall that holds the gradient for an
        upstream of one): gs_distill_loss."""
        c = _DistillCall(logits, teacher_ids, teacher_logits, labels, temperature, alpha,
                         ignore_index, reduction)
        shape = logits.shape[:-1] if reduction == "none" else ()
        if c.d.N == 0:
            c.grad = torch.empty_like(logits)
            return (torch.full(shape, math.nan if reduction == "mean" else 0.0, device=c.dev),
                    c if want_grad else None)
        loss = torch.empty(shape, dtype=torch.float32, device=c.dev)
        c.allocate(want_grad)
        with _on(c.dev):
            rc = load_library().gs_distill_loss(ctypes.byref(c.d), loss.data_ptr(), _ptr(c.grad),
                                                c.ws.data_ptr(), c.ws.numel(), _stream(c.dev))
        _check(rc, "gs_distill_loss")
        return loss, c if want_grad else None

    def distill_grad(self, logits, teacher_ids, teacher_logits, labels, *, temperature: float,
                     alpha: float, ignore_index: int, reduction: str, upstream: torch.Tensor,
                     unit: Optional["_DistillCall"] = None) -> torch.Tensor:
        """The logits' gradient for a loss gradient `upstream`: gs_distill_grad.  unit: what
        distill_loss gave for these tensors, used up by this call."""
        c = unit
        if c is None or not c.reads(logits, teacher_ids, teacher_logits, labels):
            c = _DistillCall(logits, teacher_ids, teacher_logits, labels, temperature, alpha,
                             ignore_index, reduction)
        if c.d.N == 0:
            return torch.empty_like(logits)
        filled = c.grad is not None
        if not filled:
            c.allocate(True)
        if upstream.dtype != torch.float32 or not upstream.is_contiguous():
            upstream = upstream.to(torch.float32).contiguous()
        with _on(c.dev):
            rc = load_library().gs_distill_grad(ctypes.byref(c.d), upstream.data_ptr(),
                                                int(filled), c.grad.data_ptr(), c.ws.data_ptr(),
                                                c.ws.numel(), _stream(c.dev))
        _check(rc, "gs_distill_grad")
        return c.grad if c.grad.shape == logits.shape else c.grad.view(logits.shape)


class _DistillCall:
    """The arguments of a gs_distill_* call, the tensors they point to, its scratch memory and
    the gradient it fills."""

    __slots__ = ("dev", "d", "given", "held", "ws", "grad")

    def __init__(self, logits, teacher_ids, teacher, labels, temperature, alpha, ignore_index,
                 reduction):
        self.dev = _require_device(logits, teacher_ids, teacher, labels)
        lead = logits.shape[:-1]
        if logits.dim() < 1 or logits.shape[-1] == 0 or teacher.shape != teacher_ids.shape or \
                teacher.dim() != logits.dim() or teacher.shape[:-1] != lead or \
                teacher.shape[-1] == 0 or (labels is not None and labels.shape != lead):
            raise GhostHipError(
                f"logits {tuple(logits.shape)}, teacher ids {tuple(teacher_ids.shape)}, teacher "
                f"logits {tuple(teacher.shape)}, labels "
                f"{None if labels is None else tuple(labels.shape)}: [..., V], [..., K] twice and "
                "[...] expected")
        if labels is not None and labels.is_floating_point() or teacher_ids.is_floating_point():
            raise GhostHipError("teacher ids and labels have to be integers")
        self.given = tuple(None if t is None else (t.data_ptr(), t.stride())
                           for t in (logits, teacher_ids, teacher, labels))
        dtype = _kernel_dtype(logits, "logits")
        if teacher.dtype not in (torch.bfloat16, torch.float32):
            teacher = teacher.float()
        teacher, teacher_ids = teacher.contiguous(), teacher_ids.to(torch.int64).contiguous()
        labels = None if labels is None else labels.to(torch.int64).contiguous()
        z = _rows_of_logits(logits)
        N, V = math.prod(lead), z.shape[-1]
        inner, outer, row = N, 0, z.stride(-2)
        if z.dim() == 3:
            inner, outer = z.shape[1], z.stride(0)
        elif N == 1:
            row = V
        self.held = (z, teacher_ids, teacher, labels)
        self.d = _Distill(z.data_ptr(), dtype, N, V, inner, outer, row, teacher_ids.data_ptr(),
                          teacher.data_ptr(), _TORCH_TO_GS[teacher.dtype], teacher.shape[-1],
                          _ptr(labels), ignore_index, temperature, alpha, REDUCTIONS[reduction])
        self.ws = self.grad = None

    def reads(self, *tensors) -> bool:
        """Whether these are the tensors it was made from (autograd may have moved what it saved)."""
        return self.given == tuple(None if t is None else (t.data_ptr(), t.stride())
                                   for t in tensors)

    def allocate(self, want_grad: bool) -> None:
        if self.ws is None:
            nbytes = load_library().gs_distill_workspace(ctypes.byref(self.d))
            self.ws = _workspace(nbytes, self.dev)
        if want_grad:
            self.grad = _empty_as(self.held[0])


def _rows_of_logits(z: torch.Tensor) -> torch.Tensor:
    """z as [N, V] or [B, T, V] with contiguous, non-overlapping rows; a copy where its strides
    do not allow that."""
    V = z.shape[-1]
    if z.dim() != 3:
        z = z.reshape(-1, V)
    T = z.shape[-2]
    ok = (V == 1 or z.stride(-1) == 1) and (T == 1 or z.stride(-2) >= V)
    if z.dim() == 3 and z.shape[0] > 1:
        ok = ok and z.stride(0) >= (T - 1) * z.stride(1) + V
    return z if ok else z.contiguous()


def _empty_as(z: torch.Tensor) -> torch.Tensor:
    """An uninitialised tensor of z's shape and strides at z's offset from a 16-byte boundary (the
    kernels read and write the same 16-byte pieces of both)."""
    off = z.data_ptr() % 16 // z.element_size()
    if off == 0 and z.is_contiguous():
        return torch.empty(z.shape, dtype=z.dtype, device=z.device)
    span = 1 + sum((n - 1) * s for n, s in zip(z.shape, z.stride()))
    base = torch.empty(off + span, dtype=z.dtype, device=z.device)
    return base.as_strided(z.shape, z.stride(), off)


_backend = None


def ops():
    """The active kernel layer (the HIP library unless a test installed a checker)."""
    global _backend
    if _backend is None:
        _backend = HipOps()
    return _backend


def _install_backend(backend) -> None:
    """Test seam: replace the kernel layer (host-logic tests on machines without a GPU)."""
    global _backend
    _backend = backend
