"""AdamW over all of a model's tensors in a few launches, its averages held in 32 or in 8 bits.

The optimizer of a training step with or without the engines: it takes ``.grad`` as it finds it
(``GradDotProdEngine.prepare_gradients`` puts the train gradients there) and runs on the current
stream, without a synchronisation.
"""
from __future__ import annotations

import itertools

import torch

from ._native import GhostHipError, ops

__all__ = ["AdamW"]

BLOCK = 256   # consecutive elements that share a scale in 8 bits (GS_ADAMW_BLOCK)


class AdamW(torch.optim.Optimizer):
    """Adam with decoupled weight decay.  Per element, in fp32, the parameter rounded once:

        m = beta1 m + (1 - beta1) g,   v = beta2 v + (1 - beta2) g^2
        p = (1 - lr weight_decay) p - lr / (1 - beta1^t) m / (sqrt(v / (1 - beta2^t)) + eps)

    Parameters: bf16 or fp32 on a ROCm GPU, dense in their memory.  ``state[p]`` holds ``step`` (the
    steps taken, a number) and, laid out like p:

      - state_bits=32: ``exp_avg`` and ``exp_avg_sq``, m and v in fp32 (also for bf16 parameters);
      - state_bits=8: ``exp_avg`` and ``root_avg_sq`` (float8_e4m3fn) with ``exp_avg_scale`` and
        ``root_avg_sq_scale`` (fp32, one for each 256 consecutive elements): their products are m
        and the root of v.  2.03 bytes an element instead of 8.  Each is rounded up or down by
        chance, with odds that keep it right on average; the chances come from ``seed``, the step and
        the element's place, so a run repeats bit for bit.  (v, the root's square, comes out a few
        hundredths high.)  An average that is not finite is held as NaN.

    A step cannot be captured into a graph: it counts on the host."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, seed: int = 0):
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits, seed=seed))

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        try:
            _check(self.param_groups[-1])
            params = self.param_groups[-1]["params"]
            if len(set(params)) < len(params):   # each would be written twice at once
                raise GhostHipError("AdamW: a parameter is in its group twice")
        except Exception:
            del self.param_groups[-1]
            raise

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise GhostHipError("an AdamW step cannot be captured into a graph: the step is counted on "
                                "the host")
        for group in self.param_groups:
            _check(group)
            bits = group["state_bits"]
            params = [p for p in group["params"] if p.grad is not None]
            states = [self.state[p] for p in params]
            for p, state in zip(params, states):
                if not state:
                    state.update(_new_state(p, bits))
            beta1, beta2 = group["betas"]
            taken = [state["step"] for state in states]
            counts = dict.fromkeys(taken)   # as a rule one number
            for before in counts:
                at = [i for i, t in enumerate(taken) if t == before] if len(counts) > 1 else None
                some_p, some_s = (params, states) if at is None else \
                    ([params[i] for i in at], [states[i] for i in at])
                ops().adamw(some_p, some_s, bits, group["lr"], beta1, beta2, group["eps"],
                            group["weight_decay"], before + 1, group["seed"] & 0xFFFFFFFF)
                for state in some_s:
                    state["step"] = before + 1
        return loss

    def load_state_dict(self, state_dict) -> None:
        """A state of this class, or one of ``torch.optim.AdamW`` for fp32 parameters (32 bits)."""
        for group in state_dict["param_groups"]:
            if group.get("amsgrad") or group.get("maximize"):
                raise GhostHipError("AdamW: a state with amsgrad or maximize")
            if not group.get("decoupled_weight_decay", True) and group["weight_decay"]:
                raise GhostHipError("AdamW: a state of Adam, whose weight decay is in its gradients")
        super().load_state_dict(state_dict)
        for group in self.param_groups:
            group.setdefault("state_bits", 32)
            group.setdefault("seed", 0)
        # The averages keep their types: the base class casts them to their parameters'.
        given = itertools.chain.from_iterable(g["params"] for g in state_dict["param_groups"])
        mine = itertools.chain.from_iterable(g["params"] for g in self.param_groups)
        for key, p in zip(given, mine):
            for name, value in state_dict["state"].get(key, {}).items():
                if name == "step":
                    self.state[p][name] = int(value)
                elif isinstance(value, torch.Tensor):
                    self.state[p][name] = value.detach().to(p.device, copy=True)


def _check(group) -> None:
    betas = group["betas"]
    for name, value in (("lr", group["lr"]), ("eps", group["eps"]),
                        ("weight_decay", group["weight_decay"])):
        if isinstance(value, torch.Tensor) or not 0.0 <= value < float("inf"):
            raise GhostHipError(f"AdamW: {name} {value}: a number of at least zero expected")
    if len(betas) != 2 or not all(not isinstance(b, torch.Tensor) and 0.0 <= b < 1.0 for b in betas):
        raise GhostHipError(f"AdamW: betas {betas}: two numbers of [0, 1) expected")
    if group["state_bits"] not in (8, 32):
        raise GhostHipError(f"AdamW: averages of {group['state_bits']} bits: 8 or 32")


def _new_state(p: torch.Tensor, bits: int) -> dict:
    if bits == 32:
        return {"step": 0, "exp_avg": torch.zeros_like(p, dtype=torch.float32),
                "exp_avg_sq": torch.zeros_like(p, dtype=torch.float32)}
    blocks = -(-p.numel() // BLOCK)
    state = {"step": 0}
    for name in ("exp_avg", "root_avg_sq"):
        state[name] = torch.zeros_like(p, dtype=torch.uint8).view(torch.float8_e4m3fn)
        state[name + "_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
    return state
