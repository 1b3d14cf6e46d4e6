"""The losses that write their gradient with the loss, backward captured in a CUDA graph: each replay
writes the gradient, also where the capture did not hold the forward."""

from __future__ import annotations

import pytest
import torch

import torchisotonic_b200 as ti


def policy(leaf):
    n = len(leaf)
    y = torch.arange(n, device="cuda") % leaf.shape[1]
    old = ti.token_logprobs(leaf.detach() * 0.9, y)
    advantages = torch.linspace(-1, 1, n, device="cuda")
    return lambda: ti.policy_loss(leaf, y, old, advantages).loss


def distillation(leaf):
    lists = ti.token_scores(leaf.detach() * 0.9, top=6)
    return lambda: ti.distillation_loss(leaf, lists.top_ids, lists.top_logps).loss


def logits(seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(48, 3001, generator=gen, device="cuda").requires_grad_()


@pytest.mark.gpu
@pytest.mark.parametrize("of", [policy, distillation])
def test_backward_of_an_eager_forward(of) -> None:
    leaf = logits()
    call = of(leaf)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        (want,) = torch.autograd.grad(call(), leaf)
        want = want.clone()
        loss, one = call(), torch.ones((), device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        (got,) = torch.autograd.grad(loss, leaf, one, retain_graph=True)
    for upstream in (1.0, 1.0, -2.0, 1.0):
        one.fill_(upstream)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want * upstream)
        got.mul_(0)  # as a program that clears or scales its gradients in place


@pytest.mark.gpu
@pytest.mark.parametrize("of", [policy, distillation])
def test_forward_and_backward_in_graphs_of_their_own(of) -> None:
    leaf = logits()
    call = of(leaf)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(2):
            (want,) = torch.autograd.grad(call(), leaf)
        want = want.clone()
        one = torch.ones((), device="cuda")
    torch.cuda.synchronize()
    forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(forward, stream=stream):
        loss = call()
    with torch.cuda.graph(backward, pool=forward.pool(), stream=stream):
        (got,) = torch.autograd.grad(loss, leaf, one, retain_graph=True)
    for _ in range(2):
        forward.replay()
        for _ in range(2):
            backward.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
            got.mul_(0)


@pytest.mark.gpu
@pytest.mark.parametrize("of", [policy, distillation])
def test_forward_and_backward_in_one_graph(of) -> None:
    leaf = logits()
    call = of(leaf)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        (want,) = torch.autograd.grad(call(), leaf)
        want = want.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        (got,) = torch.autograd.grad(call(), leaf)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        got.mul_(0)


@pytest.mark.gpu
@pytest.mark.parametrize("of", [policy, distillation])
def test_eager_backward_of_a_captured_forward(of) -> None:
    leaf = logits()
    call = of(leaf)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        (want,) = torch.autograd.grad(call(), leaf)
        want = want.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        loss = call()
    graph.replay()
    (got,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    with torch.no_grad():
        leaf.mul_(0.5)
    graph.replay()  # which leaves the gradient of the replay before alone
    torch.cuda.synchronize()
    assert torch.equal(got, want)
