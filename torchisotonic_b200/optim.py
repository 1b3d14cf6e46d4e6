"""AdamW over many tensors in one launch, with its moments in 32 bits or in 8 (the update that
follows the losses of ``losses.py``; the reference has no counterpart).

With 8-bit states a parameter element costs 2 bytes of optimizer state instead of 8: the running
mean of the gradient and the square root of the running mean of its square are float8 (e4m3)
numbers, every 256 elements sharing a power of two (a float32), rounded to one of the two
neighbouring numbers at random, so that the means of the first moment and of the root's square stay
right (rounded to nearest, a second moment that moves by a thousandth a step would stay where it
is). The random bits are a function of ``seed``, the step and the element, so a run can be
repeated.
"""

from __future__ import annotations

from collections.abc import Iterable, Sequence
from itertools import chain
from typing import Any

import torch
from torch import Tensor

from torchisotonic_b200 import _ext

BLOCK = 256  # elements that share a scale


def adamw_step(
    params: Sequence[Tensor],
    grads: Sequence[Tensor],
    exp_avgs: Sequence[Tensor],
    exp_avg_sqs: Sequence[Tensor],
    *,
    step: int,
    lr: float = 1e-3,
    betas: tuple[float, float] = (0.9, 0.999),
    eps: float = 1e-8,
    weight_decay: float = 0.01,
    scales: tuple[Sequence[Tensor], Sequence[Tensor]] | None = None,
    seed: int = 0,
    indices: Sequence[int] | None = None,
) -> None:
    """One AdamW step (decoupled weight decay) over all of ``params``, in place:

    ``m = b1 m + (1 - b1) g``, ``v = b2 v + (1 - b2) g^2``, ``p = p (1 - lr weight_decay) - lr / (1 -
    b1^step) m / (sqrt(v) / sqrt(1 - b2^step) + eps)``, computed in float32.

    All tensors are contiguous and on one CUDA device. ``params``: float32, bfloat16 or float16
    (rounded to nearest after the step); ``grads``: like their parameter, or float32.
    ``exp_avgs`` and ``exp_avg_sqs``: float32 (m and v), shaped like the parameters; or
    float8_e4m3fn, with ``scales = (exp_avg_scales, exp_avg_sq_scales)``, a float32 tensor of
    ceil(n / 256) numbers for every state: a state's number times its block's scale is then m, and
    the square root of v. ``step`` counts from 1; ``seed`` enters the rounding of 8-bit states. Both
    are numbers of this call: captured in a CUDA graph, a replay repeats them. ``indices``: where a
    step takes several calls, each tensor's place among all of the step's (an integer for every
    parameter; its place in the list if None), so that no two are rounded by the same random bits.
    """
    if scales is not None and len(scales) != 2:
        raise ValueError("scales must be a pair of sequences")
    if step < 1:
        raise ValueError("step must be at least 1")
    if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
        raise ValueError("betas must be in [0, 1)")
    if not (lr >= 0 and eps >= 0 and weight_decay >= 0):
        raise ValueError("lr, eps and weight_decay must not be negative")
    if indices is not None and len(indices) != len(params):
        raise ValueError("indices must be as many as params")
    # the lists are checked there: hundreds of tensors a call
    _ext.native().adamw([params, grads, exp_avgs, exp_avg_sqs, *(scales or ())], step, lr, betas[0],
                        betas[1], eps, weight_decay, seed & 0xFFFFFFFF,
                        () if indices is None else indices)


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW``'s update through ``adamw_step``: every parameter group in one launch
    for each pair of parameter and gradient types (480 tensors a launch).

    ``state_bits``: 32, or 8 for float8 moments (see the module). ``seed``: of their rounding.
    Learning rate, betas, eps and weight decay are per group. A parameter that is not contiguous is
    stepped as a contiguous copy, written back. ``state_dict`` and
    ``load_state_dict`` keep the states' types, so a run resumes exactly. A step counts on the host:
    capturing one in a CUDA graph raises.
    """

    def __init__(self, params: Iterable[Any], lr: float = 1e-3,
                 betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, *, state_bits: int = 32, seed: int = 0) -> None:
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        if not (lr >= 0 and eps >= 0 and weight_decay >= 0):
            raise ValueError("lr, eps and weight_decay must not be negative")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError("betas must be in [0, 1)")
        super().__init__(params, {"lr": lr, "betas": betas, "eps": eps,
                                  "weight_decay": weight_decay, "state_bits": state_bits,
                                  "seed": seed})

    def _init_state(self, p: Tensor, bits: int) -> dict[str, Any]:
        state: dict[str, Any] = {"step": 0}
        for name in ("exp_avg", "exp_avg_sq"):
            if bits == 32:
                state[name] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            else:
                state[name] = torch.zeros(p.shape, dtype=torch.uint8,
                                          device=p.device).view(torch.float8_e4m3fn)
                state[name + "_scale"] = torch.zeros(-(-p.numel() // BLOCK), dtype=torch.float32,
                                                     device=p.device)
        return state

    @torch.no_grad()
    def step(self, closure: Any = None) -> Any:
        if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(
                "AdamW.step cannot be captured in a CUDA graph: a replay would repeat this step's "
                "number, bias corrections and random rounding"
            )
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        first = 0  # of the group's parameters among all
        for group in self.param_groups:
            bits = group["state_bits"]
            # parameters that joined later, or had no gradient in some steps, are at another step
            at_step: dict[tuple[int, torch.device], list[tuple[int, Tensor]]] = {}
            for index, p in enumerate(group["params"], first):
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW does not support sparse gradients")
                state = self.state[p]
                if not state:
                    state.update(self._init_state(p, bits))
                at_step.setdefault((state["step"] + 1, p.device), []).append((index, p))
            first += len(group["params"])
            for (step, _), stepped in at_step.items():
                indices, params = zip(*stepped)
                states = [self.state[p] for p in params]
                scales = None
                if bits == 8:
                    scales = tuple([s[name] for s in states]
                                   for name in ("exp_avg_scale", "exp_avg_sq_scale"))
                values = [p if p.is_contiguous() else p.contiguous() for p in params]
                adamw_step(values, [p.grad.contiguous() for p in params],
                           [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
                           step=step, lr=float(group["lr"]), betas=group["betas"],
                           eps=group["eps"], weight_decay=group["weight_decay"], scales=scales,
                           seed=group["seed"], indices=indices if bits == 8 else None)
                for p, state, value in zip(params, states, values):
                    state["step"] = step  # a step that is refused does not count
                    if value is not p:
                        p.copy_(value)
        return loss

    def __setstate__(self, state: dict[str, Any]) -> None:
        super().__setstate__(state)
        for group in self.param_groups:
            group.setdefault("state_bits", 32)
            group.setdefault("seed", 0)

    @torch.no_grad()
    def load_state_dict(self, state_dict: dict[str, Any]) -> None:
        """As torch's, but for the states' types: torch casts them to their parameter's. Also takes
        a state of ``torch.optim.AdamW`` (the moments become float32), without its ``amsgrad`` and
        ``maximize``."""
        if any(g.get("amsgrad") or g.get("maximize") for g in state_dict["param_groups"]):
            raise ValueError("AdamW has no amsgrad and no maximize")
        super().load_state_dict(state_dict)
        saved = chain.from_iterable(g["params"] for g in state_dict["param_groups"])
        params = chain.from_iterable(g["params"] for g in self.param_groups)
        for index, p in zip(saved, params):
            for name, value in state_dict["state"].get(index, {}).items():
                if name == "step":
                    self.state[p][name] = int(value)
                elif isinstance(value, Tensor):
                    kept = value.dtype in (torch.float32, torch.float8_e4m3fn)
                    self.state[p][name] = value.to(
                        p.device, value.dtype if kept else torch.float32, copy=True,
                        memory_format=torch.contiguous_format)
