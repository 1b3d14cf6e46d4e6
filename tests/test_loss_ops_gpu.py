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


def test_training_example() -> None:
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import preference_training

    got = preference_training.main(["--steps", "60", "--pairs", "64"])
    assert got["loss"][-1] < 0.8 * got["loss"][0]        # the preference is learned
    assert got["accuracy"] > 0.8                          # on held-out pairs
    assert got["reward"][-1] > got["reward"][0]           # the policy improves on its reward
    curve = got["curve"]
    assert (curve[1:] >= curve[:-1]).all() and 0 <= curve[0] and curve[-1] <= 1
