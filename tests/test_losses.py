"""Token log-probabilities, the preference loss and the clipped policy loss, against their
definitions in float64 (plain torch below, gradients by automatic differentiation of it) and
against differences.

Tolerances, float32 arithmetic: a sum of V exponentials that 256 threads or more share has a
relative error of at most 2^-24 (V / 256 additions in a row + 64), the 64 for the exponentials
(2 units in the last place, and the rounding of their argument weighted by their size) and the
joins; so have the log-probability (absolutely) and, times its coefficient, a gradient. On top
come the roundings of the outputs to their types. float64: the same with 2^-53.
"""

from __future__ import annotations

import math
import re
from pathlib import Path

import pytest
import torch

import torchisotonic_b200 as ti
from torchisotonic_b200 import _ext, ops

HALF_ULP = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24,
            torch.float64: 2.0**-53}
LEAST = {torch.float16: 2.0**-24, torch.bfloat16: 0.0, torch.float32: 0.0, torch.float64: 0.0}
ALL = [torch.bfloat16, torch.float16, torch.float32, torch.float64]


def unit(dtype: torch.dtype) -> float:
    return 2.0**-53 if dtype == torch.float64 else 2.0**-24


def lp_atol(dtype: torch.dtype, vocab: int) -> float:
    return unit(dtype) * (64 + vocab / 256)


def check(got, want, atol: float, rtol: float) -> None:
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape
    torch.testing.assert_close(got, want, atol=atol, rtol=rtol, equal_nan=True)


def logits_of(shape, dtype, seed=0, scale=3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float64) * scale
    y = torch.randint(0, shape[-1], shape[:-1], generator=gen, device="cuda")
    g = torch.randn(shape[:-1], generator=gen, device="cuda", dtype=torch.float64)
    return x.to(dtype), y, g.to(_ext.acc_dtype(dtype))


def plain_logprobs(x, y, temperature=1.0, ignore=-100):
    lp = torch.log_softmax(x.double() / temperature, -1)
    used = y != ignore
    got = lp.gather(-1, torch.where(used, y, torch.zeros_like(y))[..., None])[..., 0]
    return torch.where(used, got, torch.zeros_like(got))


def check_logprobs(x, y, g, temperature=1.0, ignore=-100):
    """Values and gradient of one call against float64; returns the gradient."""
    vocab, dtype = x.shape[-1], x.dtype
    leaf = x.detach().requires_grad_()
    lp = ti.token_logprobs(leaf, y, temperature=temperature, ignore_index=ignore)
    assert lp.dtype == _ext.acc_dtype(dtype) and lp.shape == y.shape
    (gx,) = torch.autograd.grad(lp, leaf, g)
    assert gx.dtype == dtype and gx.shape == x.shape and gx.is_contiguous()
    with torch.no_grad():
        torch.testing.assert_close(ti.token_logprobs(x, y, temperature=temperature,
                                                     ignore_index=ignore), lp.detach(),
                                   rtol=0, atol=0, equal_nan=True)
    # the rows that are left out may hold anything: zeros for the float64 side
    seen = torch.where((y == ignore)[..., None], torch.zeros_like(x), x)
    wide = seen.double().requires_grad_()
    want = plain_logprobs(wide, y, temperature, ignore)
    (gw,) = torch.autograd.grad(want, wide, torch.where(y == ignore, torch.zeros_like(g), g).double())
    check(lp, want, lp_atol(dtype, vocab), 2 * unit(dtype))
    top = float(g.abs().max()) / temperature if g.numel() else 0.0
    check(gx, gw, top * unit(dtype) * (80 + vocab / 256) + LEAST[dtype], HALF_ULP[dtype] * 1.01)
    return gx


VOCABS = [1, 2, 7, 8, 31, 33, 257, 1000, 1024, 2047, 4099, 8192, 32001, 50021, 131072, 200003]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", VOCABS)
def test_logprobs_vocabularies(vocab: int, dtype: torch.dtype) -> None:
    for rows in (1, 5):
        x, y, g = logits_of((rows, vocab), dtype, seed=vocab + rows)
        check_logprobs(x, y, g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 70000), (2, 300), (37, 9001), (149, 777), (300, 5000),
                                        (600, 20000), (5000, 40), (3001, 1027)])
def test_logprobs_rows(rows: int, vocab: int, dtype: torch.dtype) -> None:
    x, y, g = logits_of((rows, vocab), dtype, seed=rows)
    y[torch.rand(rows, device="cuda") < 0.3] = -100
    check_logprobs(x, y, g, temperature=0.7)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", [5, 130, 1001, 4097, 33001])
def test_logprobs_layouts(vocab: int, dtype: torch.dtype) -> None:
    x, y, g = logits_of((3, 9, vocab), dtype, seed=vocab)
    check_logprobs(x[:, :-1], y[:, 1:], g[:, 1:])                   # cut along the length
    check_logprobs(x[:, 1:], y[:, 1:], g[:, 1:])                    # and at its start
    check_logprobs(x[..., :vocab - 1], y % (vocab - 1), g)          # a padded vocabulary
    check_logprobs(x[..., 1:], y % (vocab - 1), g)                  # rows off alignment
    check_logprobs(x[0], y[0], g[0])
    check_logprobs(x[0, 0], y[0, 0], g[0, 0])                       # one row, no leading dimension
    check_logprobs(x[:1].expand(3, 9, vocab), y, g)                 # a broadcast input
    check_logprobs(x.transpose(0, 1), y.t(), g.t())                 # two strides, in another order
    check_logprobs(x.transpose(1, 2), y[:, :1].expand(3, vocab) % 9,
                   g[:, :1].expand(3, vocab))                       # the vocabulary not contiguous
    check_logprobs(x.reshape(3, 3, 3, vocab)[:, :2, 1:], y.reshape(3, 3, 3)[:, :2, 1:],
                   g.reshape(3, 3, 3)[:, :2, 1:])                   # three strides: copied
    check_logprobs(x, y.to(torch.int32).long(), g.expand(3, 9))
    torch.testing.assert_close(ti.token_logprobs(x, y.to(torch.int32)), ti.token_logprobs(x, y),
                               rtol=0, atol=0)


@pytest.mark.gpu
def test_logprobs_broadcast_gradient() -> None:
    # one row of logits read by many tokens: their gradients add up in the row
    x, y, g = logits_of((1, 1203), torch.float32)
    y = torch.arange(40, device="cuda")
    leaf = x.clone().requires_grad_()
    ti.token_logprobs(leaf.expand(40, 1203), y).sum().backward()
    wide = x.double().requires_grad_()
    plain_logprobs(wide.expand(40, 1203), y).sum().backward()
    check(leaf.grad, wide.grad, 40 * 2.0**-24 * (80 + 1203 / 256 + 40), 2.0**-23)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 5), (2, 0, 5), (0, 40000)])
def test_logprobs_no_rows(shape) -> None:
    x = torch.zeros(shape, device="cuda", requires_grad=True)
    lp = ti.token_logprobs(x, torch.zeros(shape[:-1], dtype=torch.int64, device="cuda"))
    assert lp.shape == shape[:-1]
    lp.sum().backward()
    assert x.grad is not None and x.grad.shape == shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", [40, 2500, 40007])
def test_logprobs_masked_vocabulary(vocab: int, dtype: torch.dtype) -> None:
    least = torch.finfo(dtype).min
    x, y, g = logits_of((8, vocab), dtype, seed=vocab)
    hidden = torch.rand(8, vocab, device="cuda") < 0.7
    hidden.scatter_(1, y[:, None], False)
    for fill in (-math.inf, least):
        z = torch.where(hidden, torch.full_like(x, fill), x)
        check_logprobs(z, y, g)
    # all but the target hidden: log-probability 0, gradient 0
    only = torch.full_like(x, -math.inf).scatter_(1, y[:, None], 2.0)
    leaf = only.requires_grad_()
    lp = ti.token_logprobs(leaf, y)
    assert (lp == 0).all()
    (gx,) = torch.autograd.grad(lp, leaf, g)
    assert (gx == 0).all()
    # every logit the type's lowest: uniform
    lp = ti.token_logprobs(torch.full_like(x, least), y)
    check(lp, torch.full_like(lp, -math.log(vocab)).double(), lp_atol(dtype, vocab), 2 * unit(dtype))
    # the target itself hidden: minus infinity
    z = x.detach().clone().scatter_(1, y[:, None], -math.inf)
    assert (ti.token_logprobs(z, y) == -math.inf).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", [40, 2500, 40007])
def test_logprobs_not_finite(vocab: int, dtype: torch.dtype) -> None:
    # nothing but -inf, a +inf or a NaN anywhere: NaN for that row alone, as in log_softmax
    x, y, g = logits_of((6, vocab), dtype, seed=vocab)
    x[1] = -math.inf
    x[3, vocab // 2] = math.inf
    x[4, vocab - 1] = math.nan
    leaf = x.requires_grad_()
    lp = ti.token_logprobs(leaf, y)
    (gx,) = torch.autograd.grad(lp, leaf, g)
    bad = torch.tensor([False, True, False, True, True, False], device="cuda")
    assert torch.equal(lp.isnan(), bad)
    assert gx[1].isnan().all() and gx[4].isnan().all()
    assert not gx[~bad].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [40, 2500, 40007])
def test_logprobs_targets(vocab: int) -> None:
    x, y, g = logits_of((6, vocab), torch.float32, seed=vocab)
    x[2] = math.nan  # left out: not read
    y[2] = -100
    check_logprobs(x, y, g)
    y[y == 7] = 8
    y[2] = 7
    check_logprobs(x, y, g, ignore=7)
    # out of range: NaN, for that row alone
    y[2] = -100
    for wrong in (vocab, -1, 2**40):
        z = y.clone()
        z[4] = wrong
        leaf = x.detach().requires_grad_()
        lp = ti.token_logprobs(leaf, z)
        (gx,) = torch.autograd.grad(lp, leaf, g)
        assert lp.isnan().tolist() == [False] * 4 + [True, False]
        assert gx[4].isnan().all() and not gx[[0, 1, 2, 3, 5]].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [0.05, 0.7, 1.0, 30.0])
@pytest.mark.parametrize("vocab", [777, 32000])
def test_logprobs_temperature(vocab: int, temperature: float) -> None:
    # the argument of an exponential, (x - max) / t, is rounded to float: its error times the
    # size of the exponential is at most 2^-23 max(u exp(-u)) < 2^-24, inside the 64 of lp_atol.
    # The log-probability itself is rounded relative to its size.
    x, y, g = logits_of((9, vocab), torch.float32, seed=3)
    check_logprobs(x, y, g, temperature=temperature)


@pytest.mark.gpu
def test_logprobs_large_offsets() -> None:
    # more than 2^31 logits: the last rows lie past 32-bit offsets
    rows, vocab = 16500, 131072
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    x[-2:] = torch.randn(2, vocab, generator=gen, device="cuda") * 3
    y = torch.full((rows,), vocab - 1, device="cuda")
    leaf = x.requires_grad_()
    lp = ti.token_logprobs(leaf, y)
    want = plain_logprobs(x.detach()[-2:], y[-2:])
    check(lp[-2:], want, lp_atol(x.dtype, vocab), 2.0**-23)
    check(lp[:-2], torch.full((rows - 2,), -math.log(vocab)).double(), lp_atol(x.dtype, vocab), 2.0**-23)
    (gx,) = torch.autograd.grad(lp.sum(), leaf)
    p = torch.softmax(x.detach()[-2:].double(), 1)
    want = -p
    want[:, -1] += 1
    check(gx[-2:], want, 2.0**-24 * (80 + vocab / 256), HALF_ULP[x.dtype] * 1.01)
    assert (gx[:-2, :-1] == gx[0, 0]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 11), (2, 1100)])
def test_logprobs_gradcheck(shape) -> None:
    x, y, _ = logits_of(shape, torch.float64, scale=1.0)
    assert torch.autograd.gradcheck(lambda t: ti.token_logprobs(t, y, temperature=1.3),
                                    (x.requires_grad_(),))


@pytest.mark.gpu
def test_logprobs_on_another_stream() -> None:
    x, y, g = logits_of((64, 30011), torch.bfloat16)
    want = ti.token_logprobs(x, y)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = ti.token_logprobs(x, y)
        got = got * 1.0
    stream.synchronize()
    torch.testing.assert_close(got, want, rtol=0, atol=0)


# ---------------------------------------------------------------------------------------------
# Preference loss


def plain_preference(logps, refs, offsets, *, beta=0.1, kind="logistic", label_smoothing=0.0,
                     margin=0.0, mask=None, average=False):
    """The definition in float64, on the CPU, sequence by sequence."""
    d = logps.double() if refs is None else logps.double() - refs.double()
    edges = offsets.tolist()
    s = []
    for a, b in zip(edges[:-1], edges[1:]):
        part = d[a:b] if mask is None else d[a:b][mask[a:b]]
        total = part.sum()
        s.append(total / max(1, part.numel()) if average else total)
    s = torch.stack(s)
    pairs = len(s) // 2
    u = beta * (s[:pairs] - s[pairs:]) - margin
    if kind == "logistic":
        sp = torch.nn.functional.softplus
        losses = (1 - label_smoothing) * sp(-u, threshold=800) + label_smoothing * sp(u, threshold=800)
    elif kind == "hinge":
        losses = torch.relu(1 - u)
    else:
        losses = (u - 0.5) ** 2 / beta**2
    return losses.mean(), (beta * s).view(2, pairs)


def sequences(lengths, dtype=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed)
    n = sum(lengths)
    logps = -torch.rand(n, generator=gen, dtype=torch.float64).mul(3)
    refs = logps + 0.3 * torch.randn(n, generator=gen, dtype=torch.float64)
    mask = torch.rand(n, generator=gen) < 0.7
    offsets = torch.tensor([0, *lengths]).cumsum(0)
    return logps.to(dtype), refs.to(dtype), mask, offsets


def check_preference(logps, refs, mask, offsets, upstream=1.0, **settings):
    dtype = _ext.acc_dtype(logps.dtype)
    a = logps.cuda().requires_grad_()
    b = None if refs is None else refs.cuda().requires_grad_()
    loss, rewards = ti.preference_loss(a, b, offsets.cuda(),
                                       mask=None if mask is None else mask.cuda(), **settings)
    assert loss.dtype == rewards.dtype == dtype and loss.shape == () and not rewards.requires_grad
    wa = logps.double().requires_grad_()
    wb = None if refs is None else refs.double().requires_grad_()
    want, want_r = plain_preference(wa, wb, offsets, mask=mask, **settings)
    # sums in double: only the results are rounded
    u = unit(dtype)
    check(loss, want, 1e-12, 2 * u)
    check(rewards, want_r, 1e-12, 2 * u)
    got = torch.autograd.grad(loss * upstream, [a] if b is None else [a, b])
    wants = torch.autograd.grad(want * upstream, [wa] if wb is None else [wa, wb])
    for x, y in zip(got, wants):
        check(x, y, 1e-12, 4 * u + (HALF_ULP[logps.dtype] if logps.dtype != dtype else 0))
    return loss


LENGTHS = [[1, 1], [0, 3], [0, 0], [5, 0, 1, 4], [300, 2, 1, 700], [4097, 1023],
           [7, 9, 33, 64, 65, 128, 255, 256, 257, 1]]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["logistic", "hinge", "square"])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_preference_kinds(lengths, kind: str) -> None:
    logps, refs, mask, offsets = sequences(lengths, seed=len(lengths))
    for average in (False, True):
        check_preference(logps, refs, mask, offsets, kind=kind, average=average, beta=0.3)
        check_preference(logps, refs, None, offsets, kind=kind, average=average, margin=0.2,
                         label_smoothing=0.1)
        check_preference(logps, None, mask, offsets, kind=kind, average=average, upstream=-2.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
def test_preference_types(dtype: torch.dtype) -> None:
    gen = torch.Generator().manual_seed(2)
    lengths = torch.randint(0, 500, (60,), generator=gen).tolist()
    logps, refs, mask, offsets = sequences(lengths, dtype)
    check_preference(logps, refs, mask, offsets.int())


@pytest.mark.gpu
def test_preference_many_pairs_and_long_answers() -> None:
    gen = torch.Generator().manual_seed(4)
    check_preference(*sequences(torch.randint(0, 9, (6002,), generator=gen).tolist()))
    check_preference(*sequences([100_003, 70_001, 5, 200_000]), average=True, beta=2.0)


@pytest.mark.gpu
def test_preference_masked_tokens_may_hold_anything() -> None:
    logps, refs, mask, offsets = sequences([40, 50, 60, 70])
    want = check_preference(logps, refs, mask, offsets)
    logps[~mask], refs[~mask] = math.nan, math.inf
    a = logps.cuda().requires_grad_()
    loss, _ = ti.preference_loss(a, refs.cuda(), offsets.cuda(), mask=mask.cuda())
    assert loss == want
    (g,) = torch.autograd.grad(loss, a)
    assert (g[~mask.cuda()] == 0).all() and not g.isnan().any()
    # nothing counts: both answers' sums are 0
    none = torch.zeros_like(mask)
    check(ti.preference_loss(a, None, offsets.cuda(), mask=none.cuda(), average=True)[0],
          torch.tensor(math.log(2.0)), 0.0, 2.0**-23)


@pytest.mark.gpu
def test_preference_extremes() -> None:
    # margins far out: no overflow in either direction; -inf and NaN stay in their pair's loss
    off = torch.tensor([0, 1, 2], device="cuda")
    for a, b in ((-1e4, 0.0), (0.0, -1e4), (-1e30, -1.0)):
        x = torch.tensor([a, b], device="cuda", requires_grad=True)
        loss, _ = ti.preference_loss(x, None, off, beta=1.0)
        (g,) = torch.autograd.grad(loss, x)
        want = max(b - a, 0.0)
        check(loss, torch.tensor(want), 1e-30, 2.0**-22)
        slope = -1.0 if b > a else 0.0
        check(g, torch.tensor([slope, -slope]), 1e-30, 2.0**-22)
    x = torch.tensor([-math.inf, -1.0], device="cuda")
    assert ti.preference_loss(x, None, off)[0] == math.inf
    x = torch.tensor([-1.0, -math.inf], device="cuda")
    assert ti.preference_loss(x, None, off)[0] == 0
    for kind in ("logistic", "hinge", "square"):
        x = torch.tensor([math.nan, -1.0], device="cuda")
        assert ti.preference_loss(x, None, off, kind=kind)[0].isnan()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("u", [-40.0, -25.0, 0.0, 3.0, 20.0, 30.0, 40.0, 80.0])
def test_preference_slope_far_from_the_decision(u: float, dtype: torch.dtype) -> None:
    # -1 / (1 + exp(u)), to the type's precision however small: a dozen roundings in double, then one
    off = torch.tensor([0, 1, 2], device="cuda")
    x = torch.tensor([u, 0.0], device="cuda", dtype=dtype, requires_grad=True)
    for e in (0.0, 0.125):
        loss, _ = ti.preference_loss(x, None, off, beta=1.0, label_smoothing=e)
        (g,) = torch.autograd.grad(loss, x)
        slope = e / (1 + math.exp(-u)) - (1 - e) / (1 + math.exp(u))
        want = torch.tensor([slope, -slope], dtype=torch.float64)
        check(g, want, 0.0, unit(dtype) + 12 * 2.0**-53)


@pytest.mark.gpu
def test_preference_tokens_of_no_answer() -> None:
    # offsets that start late and end early: the tokens outside get no gradient
    logps, refs, _, _ = sequences([100])
    offsets = torch.tensor([10, 30, 30, 60, 90])
    a = logps.cuda().requires_grad_()
    loss, _ = ti.preference_loss(a, refs.cuda(), offsets.cuda())
    w = logps.double().requires_grad_()
    want, _ = plain_preference(w, refs, offsets)
    check(loss, want, 1e-12, 2.0**-23)
    (g,), (gw,) = torch.autograd.grad(loss, a), torch.autograd.grad(want, w)
    check(g, gw, 1e-12, 2.0**-22)
    # offsets past the tokens are cut to them
    ti.preference_loss(a, None, torch.tensor([0, 50, 1000], device="cuda"))[0].backward()
    assert not a.grad.isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["logistic", "hinge", "square"])
def test_preference_gradcheck(kind: str) -> None:
    logps, refs, mask, offsets = sequences([5, 3, 8, 2], torch.float64)
    assert torch.autograd.gradcheck(
        lambda a, b: ti.preference_loss(a, b, offsets.cuda(), kind=kind, mask=mask.cuda(),
                                        label_smoothing=0.1, margin=0.05, beta=0.4)[0],
        (logps.cuda().requires_grad_(), refs.cuda().requires_grad_()))


@pytest.mark.gpu
def test_preference_strided_and_shared() -> None:
    logps, refs, mask, offsets = sequences([40, 50, 60, 70])
    wide = torch.stack([logps, logps], 1).cuda()
    got, _ = ti.preference_loss(wide[:, 0], refs.cuda(), offsets.cuda())
    want, _ = ti.preference_loss(logps.cuda(), refs.cuda(), offsets.cuda())
    assert got == want
    # every token the same number, broadcast: its gradient is the sum
    one = torch.tensor(-0.7, device="cuda", requires_grad=True)
    loss, _ = ti.preference_loss(one.expand(220), None, offsets.cuda(), beta=0.01)
    (g,) = torch.autograd.grad(loss, one)
    w = torch.tensor(-0.7, dtype=torch.float64, requires_grad=True)
    (gw,) = torch.autograd.grad(plain_preference(w.expand(220), None, offsets, beta=0.01)[0], w)
    check(g, gw, 0.0, 220 * 2.0**-22)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[400_000, 0], [1, 400_000], [0, 1, 300_000, 0],
                                     [90_001, 1, 0, 5, 70_000, 2048]], ids=str)
def test_preference_long_answers_beside_short_ones(lengths) -> None:
    # several CTAs to an answer, of which most have no token where the answer is short
    for average in (False, True):
        check_preference(*sequences(lengths, seed=len(lengths)), average=average, beta=0.01)


def test_remote_shared_memory_is_written_after_its_cluster_has_started() -> None:
    # a CTA that has not started has no shared memory to write to
    sources = sorted((Path(_ext.__file__).parent / "csrc").glob("*.cu*"))
    found = 0
    for source in sources:
        for body in re.split(r"\n}\n", source.read_text()):  # a function each
            write = body.find("map_shared_rank")
            if write < 0:
                continue
            found += 1
            assert 0 <= body.find("wait_for_start()") < write, source.name
    assert found == 3


# ---------------------------------------------------------------------------------------------
# Policy loss


def plain_policy(x, y, old, adv, *, ref_logps=None, weight=None, clip_low=0.2, clip_high=0.2,
                 kl_coef=0.0, temperature=1.0, ignore=-100):
    w = torch.ones(y.shape, dtype=torch.float64, device=x.device) if weight is None \
        else weight.double()
    w = torch.where(y == ignore, torch.zeros_like(w), w)
    y = torch.where(w == 0, torch.zeros_like(y), y)
    x = torch.where((w == 0)[..., None], torch.zeros_like(x), x)
    lp = torch.log_softmax(x.double() / temperature, -1).gather(-1, y[..., None])[..., 0]
    zero = torch.zeros_like(lp)

    def kept(t):
        return torch.where(w == 0, zero, t.double())

    ratio = torch.exp(lp - kept(old))
    a = kept(adv)
    free, held = ratio * a, ratio.clamp(1 - clip_low, 1 + clip_high) * a
    l, kl = -torch.where(free <= held, free, held), zero
    if ref_logps is not None:
        d = kept(ref_logps) - lp
        kl = torch.expm1(d) - d
        l = l + kl_coef * kl
    total = w.sum()
    if total == 0:
        return 0 * lp.sum(), zero, zero.sum(), zero.sum()
    return ((w * l).sum() / total, torch.where(w == 0, zero, lp), (w * kl).sum() / total,
            (w * (free > held)).sum() / total)


def tokens_of(x, y, seed, temperature=1.0):
    """Old and reference log-probabilities around the policy's, advantages; no ratio within 1e-3
    of an edge of the clip, where float32 rounding decides."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal():
        return torch.randn(y.shape, generator=gen, device="cuda", dtype=torch.float64)

    lp = plain_logprobs(x, torch.where(y < 0, torch.zeros_like(y), y), temperature)
    moved = 0.3 * normal()
    for edge in (math.log(0.8), math.log(1.2), math.log(1.28)):
        moved = torch.where((moved - edge).abs() < 1e-3, moved + 3e-3, moved)
    acc = _ext.acc_dtype(x.dtype)
    return ((lp - moved).to(acc), (normal() + 0.3).to(acc), (lp + 0.3 * normal()).to(acc))


def check_policy(x, y, old, adv, upstream=1.0, **settings):
    vocab, dtype = x.shape[-1], x.dtype
    acc = _ext.acc_dtype(dtype)
    leaf = x.detach().requires_grad_()
    got = ti.policy_loss(leaf, y, old, adv, **settings)
    assert not (got.logps.requires_grad or got.kl.requires_grad or got.clip_fraction.requires_grad)
    assert all(t.dtype == acc for t in got)
    wide = torch.nan_to_num(x.detach().double(), nan=0.0).requires_grad_()
    plain = {("ignore" if k == "ignore_index" else k): v for k, v in settings.items()}
    want = plain_policy(wide, y, old, adv, **plain)
    t = settings.get("temperature", 1.0)
    e = lp_atol(dtype, vocab)
    live = want[1] != 0
    # a token's loss and slope move by rho |A| (and kl_coef exp(d)) times its log-probability's
    # error, all below 40 here
    check(got.logps, want[1], e, 2 * unit(dtype))
    for a, b in ((got.loss, want[0]), (got.kl, want[2])):
        check(a, b, 40 * e, 8 * unit(dtype))
    check(got.clip_fraction, want[3], 0.0, 8 * unit(dtype))
    (gx,) = torch.autograd.grad(got.loss * upstream, leaf)
    (gw,) = torch.autograd.grad(want[0] * upstream, wide)
    assert gx.dtype == dtype and gx.shape == x.shape and gx.is_contiguous()
    n = max(1, int(live.sum()))
    check(gx, gw, 80 * abs(upstream) / t / n * (e + unit(dtype) * (80 + vocab / 256)) + LEAST[dtype],
          HALF_ULP[dtype] * 1.01)
    with torch.no_grad():
        again = ti.policy_loss(x, y, old, adv, **settings)
    for a, b in zip(again, got):
        torch.testing.assert_close(a, b.detach(), rtol=0, atol=0)
    return gx


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", VOCABS)
def test_policy_vocabularies(vocab: int, dtype: torch.dtype) -> None:
    x, y, _ = logits_of((6, vocab), dtype, seed=vocab)
    old, adv, ref = tokens_of(x, y, vocab)
    check_policy(x, y, old, adv, ref_logps=ref, kl_coef=0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 70000), (37, 9001), (149, 777), (300, 5000),
                                        (600, 20000), (5000, 40), (1501, 1027)])
def test_policy_rows(rows: int, vocab: int, dtype: torch.dtype) -> None:
    x, y, _ = logits_of((rows, vocab), dtype, seed=rows)
    old, adv, ref = tokens_of(x, y, rows, 0.8)
    mask = torch.rand(rows, device="cuda") < 0.6
    mask[0] = True
    x[~mask], old[~mask], adv[~mask], ref[~mask], y[~mask] = math.nan, math.nan, math.inf, math.nan, -100
    gx = check_policy(x, y, old, adv, ref_logps=ref, kl_coef=0.2, weight=mask, temperature=0.8,
                      upstream=-3.0)
    assert (gx[~mask] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 40), (torch.float64, 2100)])
def test_policy_many_rows(vocab: int, dtype: torch.dtype) -> None:
    # enough of them that a cluster sums their weights
    x, y, _ = logits_of((8200 + vocab, vocab), dtype, seed=vocab)
    old, adv, ref = tokens_of(x, y, vocab)
    w = torch.rand(x.shape[0], device="cuda", dtype=dtype)
    w[w < 0.4] = 0.0
    check_policy(x, y, old, adv, ref_logps=ref, weight=w, kl_coef=0.1)


@pytest.mark.gpu
def test_policy_settings() -> None:
    x, y, _ = logits_of((4, 50, 301), torch.float32)
    old, adv, ref = tokens_of(x, y, 1)
    w = torch.rand(4, 50, device="cuda")
    w[w < 0.3] = 0.0
    check_policy(x, y, old, adv)
    check_policy(x, y, old, adv, weight=w, clip_high=0.28)
    check_policy(x, y, old, adv, ref_logps=ref, weight=w, kl_coef=0.0)
    check_policy(x, y, old, adv, ref_logps=ref, kl_coef=1.0, clip_low=1.0, clip_high=1e9)
    # a cut tensor, its tokens' inputs strided and of other types
    old1, adv1, _ = tokens_of(x[:, :-1], y[:, 1:], 2)
    wide = torch.stack([old1.double(), adv1.double()], -1)
    check_policy(x[:, :-1], y[:, 1:], wide[..., 0], wide[..., 1], weight=w[:, 1:])
    z = y.clone()
    z[1, :20] = 5
    check_policy(x, z, old, adv, ignore_index=5)
    # not clipped at a ratio of exactly 1: the slope is the unclipped side's
    lp = ti.token_logprobs(x, y)
    got = ti.policy_loss(x, y, lp, adv)
    assert got.clip_fraction == 0


@pytest.mark.gpu
def test_policy_nothing_left() -> None:
    # all weights 0, no rows, or every target ignored: loss 0 and gradients 0, whatever is there
    x = torch.full((5, 3000), math.nan, device="cuda", requires_grad=True)
    y = torch.zeros(5, dtype=torch.int64, device="cuda")
    t = torch.full((5,), math.nan, device="cuda")
    for weight, target in ((torch.zeros(5, device="cuda"), y), (torch.zeros(5, device="cuda").bool(), y),
                           (None, y - 100)):
        got = ti.policy_loss(x, target, t, t, ref_logps=t, weight=weight, kl_coef=0.1)
        assert [float(v) for v in (got.loss, got.kl, got.clip_fraction)] == [0, 0, 0]
        assert (got.logps == 0).all()
        (g,) = torch.autograd.grad(got.loss, x)
        assert (g == 0).all()
    e = torch.zeros(0, 40, device="cuda", requires_grad=True)
    got = ti.policy_loss(e, y[:0], t[:0], t[:0])
    assert got.loss == 0
    got.loss.backward()
    assert e.grad.shape == (0, 40)


@pytest.mark.gpu
def test_policy_backward_twice() -> None:
    # the gradient written with the loss is handed out once; later calls write their own
    x, y, _ = logits_of((40, 2003), torch.float32)
    old, adv, _ = tokens_of(x, y, 1)
    leaf = x.requires_grad_()
    loss = ti.policy_loss(leaf, y, old, adv).loss
    (a,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    kept = a.clone()
    (b,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    (c,) = torch.autograd.grad(loss, leaf, torch.tensor(2.0, device="cuda"), retain_graph=True)
    torch.testing.assert_close(a, kept, rtol=0, atol=0)
    check(b, kept, 1e-9, 2.0**-22)
    check(c, 2 * kept, 1e-9, 2.0**-22)
    assert a.data_ptr() not in (b.data_ptr(), c.data_ptr())
    loss.backward()
    loss2 = ti.policy_loss(leaf, y, old, adv).loss
    loss2.backward()
    check(leaf.grad, 2 * kept, 1e-9, 2.0**-22)


@pytest.mark.gpu
def test_policy_not_finite() -> None:
    x, y, _ = logits_of((6, 2003), torch.float32)
    old, adv, _ = tokens_of(x, y, 1)
    x[2, 7] = math.nan
    leaf = x.requires_grad_()
    got = ti.policy_loss(leaf, y, old, adv)
    (g,) = torch.autograd.grad(got.loss, leaf)
    assert got.loss.isnan() and g[2].isnan().all() and not g[[0, 1, 3, 4, 5]].isnan().any()
    assert got.logps.isnan().tolist() == [False, False, True, False, False, False]
    y[2] = 2003  # out of range
    got = ti.policy_loss(torch.nan_to_num(x.detach()).requires_grad_(), y, old, adv)
    assert got.loss.isnan() and got.logps.isnan().tolist() == [False, False, True] + [False] * 3


FAR = [95.0, 1e4, math.inf]  # beyond float's exponential (88.7), double's (709.8), and any


def far_tokens(vocab, dtype):
    """Six rows; the third is the one whose old or reference log-probability a test moves."""
    x, y, _ = logits_of((6, vocab), dtype, seed=vocab)
    old, adv, ref = tokens_of(x, y, vocab)
    lp = plain_logprobs(x, y).to(old.dtype)
    others = torch.arange(6, device="cuda") != 2
    return x, y, old, adv, ref, lp, others


@pytest.mark.gpu
@pytest.mark.parametrize("far", FAR)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float64])
@pytest.mark.parametrize("vocab", [40, 5000, 70001])
def test_policy_ratio_of_any_size(vocab: int, dtype: torch.dtype, far: float) -> None:
    # A token that the old policy all but excluded. With a positive advantage the clip holds: the
    # loss is -(1 + clip_high) A, the slope 0. With a negative one nothing does: the loss is rho |A|,
    # infinite where its type has no room for it; the other rows' gradients are not touched.
    x, y, old, adv, _, lp, others = far_tokens(vocab, dtype)
    acc, e = old.dtype, lp_atol(dtype, vocab)
    old[2] = lp[2] - far
    for a in (1.5, -1.5):
        adv[2] = a
        leaf = x.detach().requires_grad_()
        got = ti.policy_loss(leaf, y, old, adv)
        (gx,) = torch.autograd.grad(got.loss, leaf)
        p = torch.softmax(x.double(), -1)
        rho = torch.exp(plain_logprobs(x, y) - old.double())
        free, held = rho * adv.double(), rho.clamp(0.8, 1.2) * adv.double()
        slope = torch.where(free > held, torch.zeros_like(rho), -free) / 6
        want = -torch.minimum(free, held).mean()
        gw = slope[:, None] * (torch.nn.functional.one_hot(y, vocab) - p)
        check(got.logps, plain_logprobs(x, y), e, 2 * unit(dtype))
        check(got.clip_fraction, (free > held).double().mean(), 0.0, 8 * unit(dtype))
        rows = others if a < 0 else slice(None)
        if not torch.isfinite(gw[2].to(acc)).all():
            assert gx[2, y[2]] == math.inf
        check(gx[rows], gw[rows], 80 / 6 * (e + unit(dtype) * (80 + vocab / 256)),
              HALF_ULP[dtype] * 1.01)
        # rho |A| is off by its exponent's error, which is that of lp
        check(got.loss, want.to(acc), 40 * e, (2 * e + 8 * unit(dtype)) if a < 0 else 8 * unit(dtype))
        if a > 0:
            assert (gx[2] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("far", FAR)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float64])
@pytest.mark.parametrize("vocab", [40, 5000, 70001])
def test_policy_reference_of_any_size(vocab: int, dtype: torch.dtype, far: float) -> None:
    # a token that the reference all but excludes costs its distance, one that only the policy
    # excludes has no bound: infinite, not NaN, and not in the other rows
    x, y, old, adv, ref, lp, others = far_tokens(vocab, dtype)
    acc, e = old.dtype, lp_atol(dtype, vocab)
    plain = plain_logprobs(x, y)
    p = torch.softmax(x.double(), -1)
    rho = torch.exp(plain - old.double())
    free, held = rho * adv.double(), rho.clamp(0.8, 1.2) * adv.double()
    for moved in (-far, far if far < math.inf else 1e300):
        if moved > torch.finfo(acc).max:
            continue
        ref[2] = lp[2] + moved
        leaf = x.detach().requires_grad_()
        got = ti.policy_loss(leaf, y, old, adv, ref_logps=ref, kl_coef=0.1)
        (gx,) = torch.autograd.grad(got.loss, leaf)
        d = ref.double() - plain
        kl = torch.expm1(d) - d
        slope = (torch.where(free > held, torch.zeros_like(rho), -free) - 0.1 * torch.expm1(d)) / 6
        gw = slope[:, None] * (torch.nn.functional.one_hot(y, vocab) - p)
        rows = others if moved > 0 else slice(None)
        if not torch.isfinite(gw[2].to(acc)).all():
            assert gx[2, y[2]] == -math.inf
        check(gx[rows], gw[rows], 80 / 6 * (e + unit(dtype) * (80 + vocab / 256)),
              HALF_ULP[dtype] * 1.01)
        rtol = 2 * e + 8 * unit(dtype)
        check(got.kl, kl.mean().to(acc), 40 * e, rtol)
        check(got.loss, (0.1 * kl - torch.minimum(free, held)).mean().to(acc), 40 * e, rtol)
        check(got.logps, plain, e, 2 * unit(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("far", FAR)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float64])
@pytest.mark.parametrize("vocab", [40, 5000, 70001])
def test_policy_terms_with_a_factor_of_zero(vocab: int, dtype: torch.dtype, far: float) -> None:
    x, y, old, adv, ref, lp, others = far_tokens(vocab, dtype)
    e = lp_atol(dtype, vocab)

    def run(old, adv, x=x, **settings):
        leaf = x.detach().requires_grad_()
        got = ti.policy_loss(leaf, y, old, adv, **settings)
        return (got, *torch.autograd.grad(got.loss, leaf))

    # no advantage: neither loss nor gradient, however large the ratio
    far_old, no_adv = old.clone(), adv.clone()
    far_old[2], no_adv[2] = lp[2] - far, 0.0
    got, gx = run(far_old, no_adv)
    want, gw = run(old, no_adv)
    assert torch.equal(got.loss, want.loss) and torch.equal(got.clip_fraction, want.clip_fraction)
    assert torch.equal(gx, gw) and (gx[2] == 0).all()
    # the KL term only watched: it is not in the loss, however large
    want, gw = run(old, adv)
    far_ref = ref.clone()
    far_ref[2] = lp[2] + min(far, 1e30)
    got, gx = run(old, adv, ref_logps=far_ref)
    assert torch.equal(got.loss, want.loss) and torch.equal(gx, gw)
    d = far_ref.double() - plain_logprobs(x, y)
    check(got.kl, (torch.expm1(d) - d).mean().to(old.dtype), 40 * e, 2 * e + 8 * unit(dtype))
    # a target that the policy excludes: its ratio is 0, its distance to the reference infinite
    masked = x.clone()
    masked[2, y[2]] = -math.inf
    want, gw = run(old, adv, masked)
    got, gx = run(old, adv, masked, ref_logps=ref)
    assert torch.isfinite(got.loss) and torch.equal(got.loss, want.loss) and torch.equal(gx, gw)
    assert got.kl == math.inf


@pytest.mark.gpu
def test_policy_loss_changes_in_place() -> None:
    # as a training loop does: divided by the accumulated steps, another term added
    x, y, _ = logits_of((40, 2003), torch.float32)
    old, adv, ref = tokens_of(x, y, 1)
    leaf = x.requires_grad_()

    def grad(change):
        got = ti.policy_loss(leaf, y, old, adv, ref_logps=ref, kl_coef=0.1)
        was = [t.detach().clone() for t in got]
        loss = change(got.loss)
        for a, b in zip(got[1:], was[1:]):
            assert torch.equal(a, b)  # the other results stay as they were
        return loss.detach(), *torch.autograd.grad(loss, leaf)

    def divided(loss):
        loss /= 4
        return loss

    def added(loss):
        loss += leaf.square().mean()
        return loss

    for a, b in ((divided, lambda loss: loss / 4), (added, lambda loss: loss + leaf.square().mean())):
        for u, v in zip(grad(a), grad(b)):
            assert torch.equal(u, v)
    with torch.no_grad():
        got = ti.policy_loss(x, y, old, adv)
    want = got.loss.clone() * 2
    got.loss.mul_(2)
    got.kl.add_(1)
    assert got.loss == want and got.clip_fraction <= 1


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(4, 9), (3, 1100)])
def test_policy_gradcheck(shape) -> None:
    x, y, _ = logits_of(shape, torch.float64, scale=1.0)
    old, adv, ref = tokens_of(x, y, 2)
    w = torch.rand(shape[0], device="cuda", dtype=torch.float64) + 0.1
    assert torch.autograd.gradcheck(
        lambda t: ti.policy_loss(t, y, old, adv, ref_logps=ref, weight=w, kl_coef=0.3).loss,
        (x.requires_grad_(),))


@pytest.mark.gpu
def test_losses_repeat_exactly() -> None:
    x, y, g = logits_of((700, 30011), torch.bfloat16)
    old, adv, ref = tokens_of(x, y, 1)

    def once():
        leaf = x.detach().requires_grad_()
        got = ti.policy_loss(leaf, y, old, adv, ref_logps=ref, kl_coef=0.1)
        lp = ti.token_logprobs(leaf, y)
        loss, _ = ti.preference_loss(lp, None, torch.arange(0, 701, 100, device="cuda")[:7])
        return [*got, *torch.autograd.grad(got.loss, leaf), loss, *torch.autograd.grad(loss, leaf)]

    for a, b in zip(once(), once()):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------
# Refusals


def test_refusals_without_a_gpu() -> None:
    x, y = torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64)
    for bad in ("x", [1.0]):
        with pytest.raises(TypeError, match="torch.Tensors"):
            ti.token_logprobs(bad, y)  # type: ignore[arg-type]
    with pytest.raises(TypeError, match="float16"):
        ti.token_logprobs(y[:, None], y)
    with pytest.raises(TypeError, match="integer"):
        ti.token_logprobs(x, x[:, 0])
    with pytest.raises(ValueError, match="do not fit"):
        ti.token_logprobs(x, y[:2])
    with pytest.raises(ValueError, match="at least one element"):
        ti.token_logprobs(x[:, :0], y)
    for t in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            ti.token_logprobs(x, y, temperature=t)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ti.token_logprobs(x, y)
    with pytest.raises(ValueError, match="clip_low"):
        ti.policy_loss(x, y, x[:, 0], x[:, 0], clip_low=-0.1)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ti.policy_loss(x, y, x[:, 0], x[:, 0])
    lp, off = torch.zeros(6), torch.tensor([0, 2, 6])
    with pytest.raises(TypeError, match="floating-point"):
        ti.preference_loss(off, None, off)
    with pytest.raises(TypeError, match="integer"):
        ti.preference_loss(lp, None, lp)
    with pytest.raises(ValueError, match="1-D"):
        ti.preference_loss(lp[None], None, off)
    for bad_off in (off[:2], off[:1], torch.tensor([0, 1, 2, 6]), off[None]):
        with pytest.raises(ValueError, match="2 \\* pairs"):
            ti.preference_loss(lp, None, bad_off)
    with pytest.raises(ValueError, match="kind"):
        ti.preference_loss(lp, None, off, kind="other")
    with pytest.raises(ValueError, match="beta"):
        ti.preference_loss(lp, None, off, beta=0.0)
    with pytest.raises(ValueError, match="label_smoothing"):
        ti.preference_loss(lp, None, off, label_smoothing=0.5)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ti.preference_loss(lp, None, off)


@pytest.mark.gpu
def test_refusals() -> None:
    x, y = torch.zeros(3, 5, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    t = x[:, 0].contiguous()
    with pytest.raises(ValueError, match="device"):
        ti.token_logprobs(x, y.cpu())
    with pytest.raises(ValueError, match="clip_low"):
        ti.policy_loss(x, y, t, t, clip_high=-1.0)
    with pytest.raises(TypeError, match="advantages"):
        ti.policy_loss(x, y, t, None)  # type: ignore[arg-type]
    with pytest.raises(ValueError, match="old_logps must be shaped"):
        ti.policy_loss(x, y, t[:2], t)
    with pytest.raises(ValueError, match="ref_logps is a constant"):
        ti.policy_loss(x, y, t, t, ref_logps=t.clone().requires_grad_())
    off = torch.tensor([0, 1, 3], device="cuda")
    with pytest.raises(ValueError, match="ref_logps must be shaped"):
        ti.preference_loss(t, t[:2], off)
    with pytest.raises(TypeError, match="mask"):
        ti.preference_loss(t, None, off, mask=t)
    with pytest.raises(ValueError, match="mask must be shaped"):
        ti.preference_loss(t, None, off, mask=t[:2] > 0)
    with pytest.raises(ValueError, match="offsets must be on"):
        ti.preference_loss(t, None, off.cpu())
    leaf = x.requires_grad_()
    (g,) = torch.autograd.grad(ti.token_logprobs(leaf, y).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):  # differentiable once
        g.sum().backward()


@pytest.mark.gpu
def test_forward_mode_is_refused() -> None:
    # a tangent would be lost; also where an argument is converted first, and by the operators
    fw = torch.autograd.forward_ad
    x, y, _ = logits_of((4, 33), torch.float32)
    old, adv, ref = tokens_of(x, y, 1)
    off = torch.tensor([0, 2, 4], device="cuda")
    with fw.dual_level():
        def dual(t):
            return fw.make_dual(t.clone(), torch.ones_like(t))

        calls = [
            lambda: ti.token_logprobs(dual(x), y),
            lambda: ti.token_logprobs(dual(x), y.int()),
            lambda: ti.preference_loss(dual(old), None, off),
            lambda: ti.preference_loss(old, dual(ref), off),
            lambda: ti.preference_loss(dual(old.half()), None, off),
            lambda: ti.policy_loss(dual(x), y, old, adv),
            lambda: ti.policy_loss(x, y, dual(old), adv),
            lambda: ti.policy_loss(x, y, old, dual(adv.double())),
            lambda: ti.policy_loss(x, y, old, adv, ref_logps=dual(ref)),
            lambda: ti.policy_loss(x, y, old, adv, weight=dual(ref)),
            lambda: ops.token_logprobs(dual(x), y, 1.0, -100),
            lambda: ops.preference(dual(old), None, None, off, 0, False, 0.1, 0.0, 0.0),
            lambda: ops.policy(x, y, -100, 1.0, old, dual(adv), None, None, 0.2, 0.2, 0.0),
        ]
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ti.token_logprobs(fw.make_dual(x.clone().requires_grad_(), torch.ones_like(x)), y)
        ti.token_logprobs(x, y)  # one that has none passes



def test_operator_refusals_without_a_gpu() -> None:
    x, y, t = torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64), torch.zeros(3)
    off = torch.tensor([0, 1, 3])
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.token_logprobs(x, y, 1.0, -100)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.token_logprobs_grad(x, y, 1.0, torch.zeros(6), t)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.policy(x, y, -100, 1.0, t, t, None, None, 0.2, 0.2, 0.0)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.policy_grad(x, y, 1.0, torch.zeros(6, dtype=torch.float64), t[0])
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.preference(t, None, None, off, 0, False, 0.1, 0.0, 0.0)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.preference_grad(t, None, off, t[:2], t[0])


def test_abi_refusals() -> None:
    import ctypes

    so = _ext.lib()
    p = ctypes.c_void_p(16)
    rows = _ext.Rows(16, 4, 4, 0, 8, 8)
    assert so.tiso_logprobs(9, rows, p, -100, 1.0, p, None, None) == 1
    assert b"dtype" in so.tiso_last_error()
    assert so.tiso_logprobs(2, None, p, -100, 1.0, p, None, None) == 1
    assert so.tiso_logprobs(2, rows, p, -100, 0.0, p, None, None) == 1
    assert b"temperature" in so.tiso_last_error()
    assert so.tiso_logprobs(2, rows, None, -100, 1.0, p, None, None) == 1
    assert so.tiso_logprobs(2, _ext.Rows(16, 4, 4, 0, 8, 0), p, -100, 1.0, p, None, None) == 1
    assert so.tiso_logprobs(2, _ext.Rows(16, 4, 4, 0, -8, 8), p, -100, 1.0, p, None, None) == 1
    assert so.tiso_logprobs(2, _ext.Rows(None, 0, 1, 0, 8, 8), None, -100, 1.0, None, None, None) == 0
    assert so.tiso_logprobs_grad(2, rows, p, 1.0, None, 2, p, None, p, None) == 1
    assert so.tiso_logprobs_grad(3, rows, p, 1.0, p, 2, p, None, p, None) == 1
    assert so.tiso_logprobs_grad(2, rows, p, 1.0, p, 2, p, None, ctypes.c_void_p(18), None) == 1
    assert b"aligned" in so.tiso_last_error()
    args = _ext.PolicyArgs(16, None, 16, None, 0, 0.2, 0.2, 0.0)
    size = ctypes.c_size_t()
    assert so.tiso_policy_workspace_size(2, 4, ctypes.byref(size)) == 0 and size.value > 0
    assert so.tiso_policy(2, rows, p, -100, 1.0, args, p, p, p, p, None, None, 0, None) == 2
    assert so.tiso_policy(2, rows, p, -100, 1.0, args, p, p, p, p, None, p, size.value - 1, None) == 2
    assert so.tiso_policy(2, rows, p, -100, 1.0, None, p, p, p, p, None, p, size.value, None) == 1
    args = _ext.PreferenceArgs(16, None, None, 16, 10, 0, 0, 0, 0.1, 0.0, 0.0)
    assert so.tiso_preference(2, args, p, p, p, p, 1 << 20, None) == 1
    assert b"pairs" in so.tiso_last_error()
    args = _ext.PreferenceArgs(16, None, None, 16, 10, 2, 0, 0, 0.1, 0.0, 0.0)
    assert so.tiso_preference(0, args, p, p, p, p, 1 << 20, None) == 1
    assert so.tiso_preference(2, args, p, p, p, p, 8, None) == 2
    assert so.tiso_preference_grad(2, args, p, None, p, None, None) == 1
