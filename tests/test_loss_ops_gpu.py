"""The losses as torch.library operators: opcheck, torch.compile(fullgraph=True) against the eager
functions (the same kernels: the same bits, but for the policy's gradient, which the compiled
function has from another kernel that writes the same bits too), and the training example."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch

import torchisotonic_b200 as ti
from torchisotonic_b200 import ops

pytestmark = pytest.mark.gpu


def inputs(dtype=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(0)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    x = normal(6, 10, 501).to(dtype)
    y = torch.randint(0, 501, (6, 10), generator=gen, device="cuda")
    return x, y, normal(6, 10) * 0.2 - 6.0, normal(6, 10), normal(6, 10) * 0.2 - 6.0


def offsets():
    return torch.tensor([0, 10, 20, 30, 40, 50, 60], device="cuda")


def test_opcheck() -> None:
    x, y, old, adv, ref = inputs()
    leaf = x.clone().requires_grad_()
    torch.library.opcheck(ops.token_logprobs, (leaf, y, 0.9, -100))
    lp = old.flatten().clone().requires_grad_()
    mask = adv.flatten() > -1
    torch.library.opcheck(ops.preference, (lp, ref.flatten(), mask, offsets()[:5], 0, True, 0.1, 0.1,
                                           0.0))
    torch.library.opcheck(ops.policy, (leaf, y, -100, 0.9, old, adv, ref, None, 0.2, 0.2, 0.1))


def good():
    """Arguments that every operator takes."""
    x, y, old, adv, ref = inputs()
    stats = ops.token_logprobs(x, y, 1.0, -100)[1]
    kept = ops.policy(x, y, -100, 1.0, old, adv, None, None, 0.2, 0.2, 0.0)[2]
    lp, off, one = old.flatten(), offsets()[:5], torch.ones((), device="cuda")
    coef = ops.preference(lp, None, None, off, 0, False, 0.1, 0.0, 0.0)[2]
    return {
        ops.token_logprobs: [x, y, 0.9, -100],
        ops.token_logprobs_grad: [x, y, 0.9, stats, adv],
        ops.preference: [lp, ref.flatten(), lp > -6, off, 0, True, 0.1, 0.1, 0.0],
        ops.preference_grad: [lp, lp > -6, off, coef, one],
        ops.policy: [x, y, -100, 0.9, old, adv, ref, adv.abs(), 0.2, 0.2, 0.1],
        ops.policy_grad: [x, y, 0.9, kept, one],
    }


def test_operators_take_strided_tensors() -> None:
    for op, args in good().items():
        want = op(*args)
        spread = [torch.stack([a, a], -1)[..., 0] if isinstance(a, torch.Tensor) and a.dim() else a
                  for a in args]
        got = op(*spread)
        for a, b in zip(got, want) if isinstance(want, tuple) else [(got, want)]:
            assert torch.equal(a, b)


def test_operators_refuse_what_they_would_misread() -> None:
    def short(t):
        return t[..., :-1] if t.dim() else torch.ones(2, device="cuda", dtype=t.dtype)

    def longer(t):
        return torch.cat([t, t], -1) if t.dim() else torch.ones(2, device="cuda", dtype=t.dtype)

    def other_type(t):
        if t.dtype == torch.float32:
            return t.half() if t.shape != (6, 10, 501) else t.int()
        return t.float() if t.dtype in (torch.int64, torch.float64) else t.to(torch.uint8)

    for op, args in good().items():
        op(*args)
        first_is_logits = args[0].dim() == 3
        for i, a in enumerate(args):
            if not isinstance(a, torch.Tensor):
                continue
            bad = [(other_type(a), TypeError), (a.cpu(), (ValueError, RuntimeError))]
            if not (i == 0 and first_is_logits):  # another vocabulary is another call
                bad += [(short(a), ValueError), (longer(a), ValueError)]
            for b, error in bad:
                with pytest.raises(error):
                    op(*args[:i], b, *args[i + 1:])
        if first_is_logits:
            for x in (args[0][..., :0], args[0][0], args[0][0, 0, 0]):
                with pytest.raises(ValueError):
                    op(x, *args[1:])
    # settings
    x, y, old, adv, _ = inputs()
    with pytest.raises(RuntimeError, match="temperature"):
        ops.token_logprobs(x, y, 0.0, -100)
    with pytest.raises(RuntimeError, match="clip_low"):
        ops.policy(x, y, -100, 1.0, old, adv, None, None, -0.1, 0.2, 0.0)
    for kind, beta, smoothing in ((3, 0.1, 0.0), (0, 0.0, 0.0), (0, 0.1, 0.5)):
        with pytest.raises(RuntimeError, match="kind|beta|label_smoothing"):
            ops.preference(old.flatten(), None, None, offsets(), kind, False, beta, smoothing, 0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_compile_fullgraph(dtype: torch.dtype) -> None:
    torch._dynamo.reset()
    x, y, old, adv, ref = inputs(dtype)

    def dpo(x):
        lp = ti.token_logprobs(x, y, temperature=0.9)
        loss, rewards = ti.preference_loss(lp.flatten(), ref.flatten(), offsets()[:5],
                                           label_smoothing=0.1, mask=adv.flatten() > -1)
        return loss * 2, rewards

    def grpo(x):
        got = ti.policy_loss(x, y, old, adv, ref_logps=ref, kl_coef=0.1, weight=adv > -1)
        return got.loss * 3, got.logps, got.kl, got.clip_fraction

    for f in (dpo, grpo):
        a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
        eager, compiled = f(a), torch.compile(f, fullgraph=True)(b)
        eager[0].backward()
        compiled[0].backward()
        for u, v in zip(eager, compiled):
            assert torch.equal(u, v)
        assert torch.equal(a.grad, b.grad)
        with torch.no_grad():
            for u, v in zip(f(x), torch.compile(f, fullgraph=True)(x)):
                assert torch.equal(u, v)


def test_compiled_losses_change_in_place() -> None:
    torch._dynamo.reset()
    x, y, old, adv, _ = inputs()

    def policy(x):
        return ti.policy_loss(x, y, old, adv).loss

    def preference(x):
        return ti.preference_loss(ti.token_logprobs(x, y).flatten(), None, offsets()[:5])[0]

    for f in (policy, preference):
        for g in (f, torch.compile(f, fullgraph=True)):
            a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
            loss = g(a)
            loss /= 4
            loss.backward()
            (f(b) / 4).backward()
            assert torch.equal(a.grad, b.grad)


def test_training_example() -> None:
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import preference_training

    got = preference_training.main(["--steps", "60", "--pairs", "64"])
    assert got["loss"][-1] < 0.8 * got["loss"][0]        # the preference is learned
    assert got["accuracy"] > 0.8                          # on held-out pairs
    assert got["reward"][-1] > got["reward"][0]           # the policy improves on its reward
    curve = got["curve"]
    assert (curve[1:] >= curve[:-1]).all() and 0 <= curve[0] and curve[-1] <= 1
