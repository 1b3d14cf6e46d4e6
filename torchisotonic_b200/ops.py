"""The operator layer as torch custom operators (torch.library), over the C ABI of libtiso.so.

Two operators keep the reference's schemas (src/torchisotonic/csrc/ops.cpp:47-50), so that code
calling ``torch.ops.torchisotonic.isotonic_tiles`` / ``isotonic_grad`` can call
``torch.ops.torchisotonic_b200.*`` with the same arguments:

* ``isotonic_tiles(Tensor y, Tensor? w, bool increasing, bool exact=True, bool with_starts=False)
  -> Tensor[]``: ``[out, starts]``, starts empty unless ``with_starts``;
* ``isotonic_grad(Tensor out, Tensor starts, Tensor g, Tensor? w, Tensor? y) -> Tensor[]``:
  ``[grad_y, grad_w]``, grad_w empty when y is None. ``out`` is not read: the kernel recomputes
  each block's mean from y and w where d/dw needs it.

Two more carry what this library folds into its kernels, and are what ``isotonic()`` runs:

* ``fit(Tensor y, Tensor? w, bool increasing, bool exact, bool with_starts, float? y_min,
  float? y_max) -> (Tensor, Tensor)``: the clipped fit in y's dtype (float16 and bfloat16 read
  as they are) and its block starts; raises ValueError when a weight is not positive (one pass
  over the weights ahead of the fit; its flag is read inside the operator);
* ``fit_grad(Tensor starts, Tensor g, Tensor? w, Tensor? y, bool want_y, bool want_w,
  float? y_min, float? y_max) -> (Tensor, Tensor)``: d/dy and d/dw (empty when not wanted),
  the clamp's inclusive mask applied.

The losses of ``losses.py`` have theirs, which the public functions run under ``torch.compile``:
``token_logprobs``, ``token_scores``, ``preference``, ``policy`` and ``distillation``, each with its
``_grad``. (``policy`` and ``distillation`` leave the gradient to their ``_grad``, which reads the
logits again; the eager functions write it with the loss.)

``fit`` has its autograd registered (the reference's _Isotonic, src/torchisotonic/_api.py:73-97)
and every operator a fake (meta) implementation, so ``torch.compile`` traces through them
without a graph break. There is no CPU kernel: CUDA tensors only.
"""

from __future__ import annotations

import torch
from torch import Tensor

from torchisotonic_b200 import _ext

_NS = "torchisotonic_b200"


def _acc(dtype: torch.dtype) -> torch.dtype:
    return _ext.acc_dtype(dtype)


# ---------------------------------------------------------------------------------------------
# The reference's schemas


@torch.library.custom_op(
    f"{_NS}::isotonic_tiles", mutates_args=(),
    schema="(Tensor y, Tensor? w, bool increasing, bool exact=True, bool with_starts=False)"
           " -> Tensor[]")
def isotonic_tiles(y: Tensor, w: Tensor | None, increasing: bool, exact: bool = True,
                   with_starts: bool = False) -> list[Tensor]:
    out, starts = _ext.isotonic_tiles(y, w, increasing, exact, with_starts)
    return [out, starts]


@isotonic_tiles.register_fake
def _(y, w, increasing, exact=True, with_starts=False):
    starts = y.new_empty(y.shape if with_starts else (0,), dtype=torch.bool)
    return [torch.empty_like(y), starts]


@torch.library.custom_op(
    f"{_NS}::isotonic_grad", mutates_args=(),
    schema="(Tensor out, Tensor starts, Tensor g, Tensor? w, Tensor? y) -> Tensor[]")
def isotonic_grad(out: Tensor, starts: Tensor, g: Tensor, w: Tensor | None,
                  y: Tensor | None) -> list[Tensor]:
    want_w = y is not None and w is not None
    gy, gw = _ext.isotonic_grad(starts, g.contiguous(), w, y if want_w else None, True, want_w)
    if gw is None:
        gw = g.new_empty((0,), dtype=_acc(g.dtype))
    return [gy, gw]


@isotonic_grad.register_fake
def _(out, starts, g, w, y):
    gw = (torch.empty(g.shape, dtype=_acc(g.dtype), device=g.device)
          if (y is not None and w is not None) else g.new_empty((0,), dtype=_acc(g.dtype)))
    return [torch.empty_like(g), gw]


# ---------------------------------------------------------------------------------------------
# The fused operators behind isotonic()


@torch.library.custom_op(f"{_NS}::fit", mutates_args=())
def fit(y: Tensor, w: Tensor | None, increasing: bool, exact: bool, with_starts: bool,
        y_min: float | None, y_max: float | None) -> tuple[Tensor, Tensor]:
    check = None if w is None else _ext.WeightCheck(w)
    out, starts = _ext.isotonic_tiles(y, w, increasing, exact, with_starts, y_min, y_max,
                                      check and check.fused_flag)
    if check is not None and check.failed():
        raise ValueError("weight must be strictly positive")
    return out, starts


@fit.register_fake
def _(y, w, increasing, exact, with_starts, y_min, y_max):
    return torch.empty_like(y), y.new_empty(y.shape if with_starts else (0,), dtype=torch.bool)


@torch.library.custom_op(f"{_NS}::fit_grad", mutates_args=())
def fit_grad(starts: Tensor, g: Tensor, w: Tensor | None, y: Tensor | None, want_y: bool,
             want_w: bool, y_min: float | None, y_max: float | None) -> tuple[Tensor, Tensor]:
    gy, gw = _ext.isotonic_grad(starts, g.contiguous(), w, y, want_y, want_w, y_min, y_max)
    if gy is None:
        gy = g.new_empty((0,))
    if gw is None:
        gw = g.new_empty((0,), dtype=_acc(g.dtype))
    return gy, gw


@fit_grad.register_fake
def _(starts, g, w, y, want_y, want_w, y_min, y_max):
    gy = torch.empty_like(g) if want_y else g.new_empty((0,))
    gw = (torch.empty(g.shape, dtype=_acc(g.dtype), device=g.device) if want_w
          else g.new_empty((0,), dtype=_acc(g.dtype)))
    return gy, gw


def _fit_setup(ctx, inputs, output) -> None:
    y, w, _increasing, _exact, _with_starts, y_min, y_max = inputs
    _, starts = output
    ctx.save_for_backward(y, w, starts)
    ctx.clip = (y_min, y_max)


def _fit_backward(ctx, grad_out: Tensor, _grad_starts: Tensor):
    y, w, starts = ctx.saved_tensors
    want_y, want_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
    y_min, y_max = ctx.clip
    need_y = want_w or y_min is not None or y_max is not None
    gy, gw = fit_grad(starts, grad_out, w, y if need_y else None, want_y, want_w, y_min, y_max)
    return (gy if want_y else None, gw if want_w else None, None, None, None, None, None)


torch.library.register_autograd(f"{_NS}::fit", _fit_backward, setup_context=_fit_setup)


# ---------------------------------------------------------------------------------------------
# The losses (sizes, types and devices are checked in csrc/native.cpp)


def _dense(t: Tensor | None) -> Tensor | None:
    return None if t is None else t.contiguous()


@torch.library.custom_op(f"{_NS}::token_logprobs", mutates_args=())
def token_logprobs(logits: Tensor, targets: Tensor, temperature: float,
                   ignore_index: int) -> tuple[Tensor, Tensor]:
    return _ext.native().logprobs(logits, targets.contiguous(), temperature, ignore_index)


@token_logprobs.register_fake
def _(logits, targets, temperature, ignore_index):
    acc = _acc(logits.dtype)
    return (logits.new_empty(targets.shape, dtype=acc),
            logits.new_empty((2 * targets.numel(),), dtype=acc))


@torch.library.custom_op(f"{_NS}::token_logprobs_grad", mutates_args=())
def token_logprobs_grad(logits: Tensor, targets: Tensor, temperature: float, stats: Tensor,
                        coef: Tensor) -> Tensor:
    return _ext.native().logprobs_grad(logits, targets.contiguous(), temperature, _dense(stats),
                                       coef.contiguous())


@token_logprobs_grad.register_fake
def _(logits, targets, temperature, stats, coef):
    return torch.empty_like(logits, memory_format=torch.contiguous_format)


def _token_logprobs_setup(ctx, inputs, output) -> None:
    logits, targets, ctx.temperature, _ = inputs
    ctx.save_for_backward(logits, targets, output[1])


def _token_logprobs_backward(ctx, grad: Tensor, _grad_stats: Tensor):
    logits, targets, stats = ctx.saved_tensors
    return (token_logprobs_grad(logits, targets, ctx.temperature, stats, grad), None, None, None)


torch.library.register_autograd(f"{_NS}::token_logprobs", _token_logprobs_backward,
                                setup_context=_token_logprobs_setup)


@torch.library.custom_op(f"{_NS}::preference", mutates_args=())
def preference(logps: Tensor, refs: Tensor | None, mask: Tensor | None, offsets: Tensor, kind: int,
               average: bool, beta: float, label_smoothing: float,
               margin: float) -> tuple[Tensor, Tensor, Tensor]:
    loss, rewards, coef = _ext.native().preference(_dense(logps), _dense(refs), _dense(mask),
                                                   _dense(offsets), kind, average, beta,
                                                   label_smoothing, margin)
    return loss, rewards, coef[:rewards.numel()].clone()


@preference.register_fake
def _(logps, refs, mask, offsets, kind, average, beta, label_smoothing, margin):
    pairs = (offsets.numel() - 1) // 2
    return (logps.new_empty(()), logps.new_empty((2, pairs)), logps.new_empty((2 * pairs,)))


@torch.library.custom_op(f"{_NS}::preference_grad", mutates_args=())
def preference_grad(logps: Tensor, mask: Tensor | None, offsets: Tensor, coef: Tensor,
                    upstream: Tensor) -> Tensor:
    return _ext.native().preference_grad(_dense(logps), _dense(mask), _dense(offsets), _dense(coef),
                                         upstream)


@preference_grad.register_fake
def _(logps, mask, offsets, coef, upstream):
    return torch.empty_like(logps, memory_format=torch.contiguous_format)


def _preference_setup(ctx, inputs, output) -> None:
    logps, _, mask, offsets = inputs[:4]
    ctx.save_for_backward(logps, mask, offsets, output[2])


def _preference_backward(ctx, grad: Tensor, _grad_rewards: Tensor, _grad_coef: Tensor):
    logps, mask, offsets, coef = ctx.saved_tensors
    g = preference_grad(logps, mask, offsets, coef, grad)
    want, want_ref = ctx.needs_input_grad[:2]
    return (g if want else None, -g if want_ref else None, *(None,) * 7)


torch.library.register_autograd(f"{_NS}::preference", _preference_backward,
                                setup_context=_preference_setup)


def _kept(logits: Tensor, targets: Tensor) -> int:
    """float64 numbers of what policy_grad needs: a coefficient, a maximum and a sum for each token
    (the last two in the accumulation dtype)."""
    return targets.numel() * (3 if _acc(logits.dtype) == torch.float64 else 2)


@torch.library.custom_op(f"{_NS}::policy", mutates_args=())
def policy(logits: Tensor, targets: Tensor, ignore_index: int, temperature: float,
           old_logps: Tensor, advantages: Tensor, ref_logps: Tensor | None, weight: Tensor | None,
           clip_low: float, clip_high: float, kl_coef: float) -> tuple[Tensor, Tensor, Tensor]:
    out, logps, kept = _ext.native().policy(logits, _dense(targets), ignore_index, temperature,
                                            _dense(old_logps), _dense(advantages),
                                            _dense(ref_logps), _dense(weight), clip_low, clip_high,
                                            kl_coef)
    return out, logps, kept[:_kept(logits, targets)].clone()


@policy.register_fake
def _(logits, targets, ignore_index, temperature, old_logps, advantages, ref_logps, weight,
      clip_low, clip_high, kl_coef):
    acc = _acc(logits.dtype)
    return (logits.new_empty((3,), dtype=acc), logits.new_empty(targets.shape, dtype=acc),
            logits.new_empty((_kept(logits, targets),), dtype=torch.float64))


@torch.library.custom_op(f"{_NS}::policy_grad", mutates_args=())
def policy_grad(logits: Tensor, targets: Tensor, temperature: float, kept: Tensor,
                upstream: Tensor) -> Tensor:
    return _ext.native().policy_grad(logits, _dense(targets), temperature, _dense(kept), upstream)


@policy_grad.register_fake
def _(logits, targets, temperature, kept, upstream):
    return torch.empty_like(logits, memory_format=torch.contiguous_format)


def _policy_setup(ctx, inputs, output) -> None:
    logits, targets, _, ctx.temperature = inputs[:4]
    ctx.save_for_backward(logits, targets, output[2])


def _policy_backward(ctx, grad: Tensor, _grad_logps: Tensor, _grad_kept: Tensor):
    logits, targets, kept = ctx.saved_tensors
    return (policy_grad(logits, targets, ctx.temperature, kept, grad[0]), *(None,) * 10)


torch.library.register_autograd(f"{_NS}::policy", _policy_backward, setup_context=_policy_setup)


@torch.library.custom_op(f"{_NS}::token_scores", mutates_args=())
def token_scores(logits: Tensor, targets: Tensor | None, top: int, temperature: float,
                 ignore_index: int) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    return _ext.native().scores(logits, _dense(targets), top, temperature, ignore_index)


@token_scores.register_fake
def _(logits, targets, top, temperature, ignore_index):
    acc, shape = _acc(logits.dtype), logits.shape[:-1]
    return (logits.new_empty((0,) if targets is None else shape, dtype=acc),
            logits.new_empty(shape, dtype=acc), logits.new_empty((*shape, top), dtype=acc),
            logits.new_empty((*shape, top), dtype=torch.int64),
            logits.new_empty((3 * (logits.numel() // logits.shape[-1]),), dtype=acc))


@torch.library.custom_op(f"{_NS}::token_scores_grad", mutates_args=())
def token_scores_grad(logits: Tensor, targets: Tensor | None, temperature: float, stats: Tensor,
                      coef_logp: Tensor | None, coef_entropy: Tensor) -> Tensor:
    return _ext.native().scores_grad(logits, _dense(targets), temperature, _dense(stats),
                                     _dense(coef_logp), _dense(coef_entropy))


@token_scores_grad.register_fake
def _(logits, targets, temperature, stats, coef_logp, coef_entropy):
    return torch.empty_like(logits, memory_format=torch.contiguous_format)


def _token_scores_setup(ctx, inputs, output) -> None:
    logits, targets, _, ctx.temperature, _ = inputs
    ctx.save_for_backward(logits, targets, output[4])
    ctx.mark_non_differentiable(output[2], output[3])


def _token_scores_backward(ctx, grad: Tensor, grad_entropy: Tensor, *_):
    logits, targets, stats = ctx.saved_tensors
    return (token_scores_grad(logits, targets, ctx.temperature, stats,
                              None if targets is None else grad, grad_entropy), *(None,) * 4)


torch.library.register_autograd(f"{_NS}::token_scores", _token_scores_backward,
                                setup_context=_token_scores_setup)


def _kept_of_lists(logits: Tensor, ids: Tensor) -> int:
    """float64 numbers of what distillation_grad needs: for each token a coefficient, two numbers
    and one for each entry (in the accumulation dtype)."""
    n, numbers = logits.numel() // logits.shape[-1], 2 + ids.shape[-1]
    return n * (1 + numbers) if _acc(logits.dtype) == torch.float64 else n + (n * numbers + 1) // 2


@torch.library.custom_op(f"{_NS}::distillation", mutates_args=())
def distillation(logits: Tensor, teacher_ids: Tensor, teacher_logps: Tensor, weight: Tensor | None,
                 kind: int, drop: bool, mix: float, temperature: float,
                 ignore_index: int) -> tuple[Tensor, Tensor, Tensor]:
    loss, divergence, kept = _ext.native().distill(
        logits, _dense(teacher_ids), _dense(teacher_logps), _dense(weight), kind, drop, mix,
        temperature, ignore_index)
    return loss, divergence, kept[:_kept_of_lists(logits, teacher_ids)].clone()


@distillation.register_fake
def _(logits, teacher_ids, teacher_logps, weight, kind, drop, mix, temperature, ignore_index):
    acc = _acc(logits.dtype)
    return (logits.new_empty((), dtype=acc), logits.new_empty(logits.shape[:-1], dtype=acc),
            logits.new_empty((_kept_of_lists(logits, teacher_ids),), dtype=torch.float64))


@torch.library.custom_op(f"{_NS}::distillation_grad", mutates_args=())
def distillation_grad(logits: Tensor, teacher_ids: Tensor, temperature: float, ignore_index: int,
                      kept: Tensor, upstream: Tensor) -> Tensor:
    return _ext.native().distill_grad(logits, _dense(teacher_ids), temperature, ignore_index,
                                      _dense(kept), upstream)


@distillation_grad.register_fake
def _(logits, teacher_ids, temperature, ignore_index, kept, upstream):
    return torch.empty_like(logits, memory_format=torch.contiguous_format)


def _distillation_setup(ctx, inputs, output) -> None:
    logits, ids, *_, ctx.temperature, ctx.ignore_index = inputs
    ctx.save_for_backward(logits, ids, output[2])
    ctx.mark_non_differentiable(output[1], output[2])


def _distillation_backward(ctx, grad: Tensor, *_):
    logits, ids, kept = ctx.saved_tensors
    return (distillation_grad(logits, ids, ctx.temperature, ctx.ignore_index, kept, grad),
            *(None,) * 8)


torch.library.register_autograd(f"{_NS}::distillation", _distillation_backward,
                                setup_context=_distillation_setup)
