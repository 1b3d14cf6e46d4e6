"""The forward divergence's gradient for a student near its teacher: differences of nearly equal numbers,
``p_v sum Q - q_v`` for a listed token and ``(P_rest sum Q - Q_rest) / n`` for each of n others that
share a logit, relative to themselves.

The rows are such that float32 sums are exact: the others' logits are the row's same number, their
exponentials 1 each, and n < 2^24. What is left of float32 is the output's own rounding (u = 2^-24; one
more for a factor or an entry that is kept in float32): ``4 u`` of the gradient. In float64 the terms are off
by some hundred roundings at most (128 entries, exponents of up to 40): ``2^-44`` of the larger one.
"""

from __future__ import annotations

import math

import pytest
import torch

import torchisotonic_b200 as ti


def rows_near_teacher(rows, vocab, top, near, temperature, seed):
    """Logits, and a teacher's lists from logits that are `near` the student's."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float64)

    level = normal(rows, 1).float()
    x = level.expand(rows, vocab).clone()
    ids = torch.rand(rows, vocab, generator=gen, device="cuda").topk(top, 1)[1]
    x.scatter_(1, ids, (level + 4 + 3 * normal(rows, top)).float())
    z = x.double() / temperature
    z.scatter_add_(1, ids, near * normal(rows, top))
    logps = torch.log_softmax(z, 1).gather(1, ids)
    return x, ids, logps.float()


def gradient(x, ids, logps, rest, weight, temperature):
    """In float64 from the definition, and the larger one of each difference's terms."""
    rows, vocab = x.shape
    z = x.double() / temperature
    m = z.amax(1, keepdim=True)
    e = (z - m).exp()
    listed = torch.zeros_like(x, dtype=torch.bool).scatter_(1, ids, True)
    n = vocab - ids.shape[1]
    s = e.sum(1, keepdim=True)
    p, p_rest = e / s, torch.where(listed, 0.0, e).sum(1, keepdim=True) / s
    q = logps.double().exp()
    if rest == "drop":
        q, q_rest = q / q.sum(1, keepdim=True), torch.zeros_like(s)
    else:
        q_rest = (1 - q.sum(1, keepdim=True)).clamp(min=0) if n else torch.zeros_like(s)
    whole = q.sum(1, keepdim=True) + q_rest
    c = (weight / weight.sum()).double()[:, None] / temperature
    q = torch.zeros_like(e).scatter_(1, ids, q)
    if n:
        g = torch.where(listed, p * whole - q, (p_rest * whole - q_rest) / n)
        terms = torch.where(listed, torch.maximum(p * whole, q), torch.maximum(p_rest * whole, q_rest) / n)
    else:
        g, terms = p * whole - q, torch.maximum(p * whole, q)
    return c * g, c * terms


@pytest.mark.gpu
@pytest.mark.parametrize("rest", ["bucket", "drop"])
@pytest.mark.parametrize("rows,vocab,top", [(7, 128, 128), (3, 33, 33), (9, 300, 1), (2500, 1003, 20),
                                            (5, 2047, 64), (401, 20011, 128), (2, 131075, 40)])
def test_forward_gradient_near_the_teacher(rows: int, vocab: int, top: int, rest: str) -> None:
    gen = torch.Generator(device="cuda").manual_seed(5)
    weight = torch.rand(rows, generator=gen, device="cuda") + 0.5
    for near, temperature in ((0.01, 1.0), (1e-4, 1.0), (1e-3, 2.0)):
        x, ids, logps = rows_near_teacher(rows, vocab, top, near, temperature, rows + vocab)
        want, terms = gradient(x, ids, logps, rest, weight, temperature)
        leaf = x.requires_grad_()
        loss = ti.distillation_loss(leaf, ids, logps, rest=rest, weight=weight,
                                    temperature=temperature).loss
        # written with the loss, and by the pass for another upstream gradient (a power of 2)
        for upstream in (1.0, 0.25):
            (got,) = torch.autograd.grad(loss * upstream, leaf, retain_graph=True)
            off = (got.double() / upstream - want).abs()
            allowed = 4 * 2.0**-24 * want.abs() + 2.0**-44 * terms + math.ldexp(1.0, -149)
            worst = float((off / allowed).max())
            assert worst <= 1, f"off by {worst:.3g} times the allowed (near {near}, upstream {upstream})"
