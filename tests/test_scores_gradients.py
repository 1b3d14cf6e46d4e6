"""Gradients of a token's scores and of the distillation, element by element: each within a bound that has the
element's own probability as a factor, so that one that is zero, wrong or not written fails in the largest
vocabulary too; and the pass for another upstream gradient than the named one, where it has more
tiles than the GPU takes at once.

Bounds, u = 2^-24 (float64: 2^-53), z a logit over the temperature from its row's maximum, e = u (64 + V / 256) a sum of
V exponentials, relative to itself:

* An exponential is off by ``3 u |z|`` (the difference, the factor and the product of its argument) and its own
  ``4 u``; a probability by that, e and some roundings: together ``e + (8 + 3 |z|) u``.
* Scores: ``p_v (G + H (z_v - mean))`` with the mean of z, off by ``2 e E|z| + 4 u E[z^2]``, and two roundings each of
  the terms ``G``, ``H mean`` and ``H z_v``.
* Forward divergence: the terms ``p_v sum Q``, ``q_v`` and ``p_v / P_rest Q_rest`` are off by a probability's bound,
  the last by that of two.
* The other divergences: ``p_v (f - sum P f)``; f, a logarithm of a quotient, is off by e for each probability (of
  the rest: of two sums), the mean by that times ``1 + sum P |f|``: together ``4 e (1 + sum P |f|)``.
* The teacher's rest ``Q_rest = 1 - sum Q`` of a list of k entries is taken in float64 on either side: each
  exponential is off by at most ``2^-52 Q`` (one unit in its last place), each of the k additions by
  ``2^-53`` (partial sums are at most 1), the difference by ``2^-54``: together at most ``2^-52 + k 2^-53 +
  2^-54`` on each side, so the two differ by less than ``(k + 4) 2^-52``. Where Q_rest is small that is many
  units of a float64 gradient: f of the rest moves by ``df / dQ_rest`` times it.

On top come a gradient's rounding to its type and, where an exponential is below the type's least
normal number, that one.
"""

from __future__ import annotations

import math

import pytest
import torch

import torchisotonic_b200 as ti
from torchisotonic_b200 import _ext

HALF_STEP = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24, torch.float64: 2.0**-53}
ALL = [torch.bfloat16, torch.float16, torch.float32, torch.float64]
IGNORE = -100
LEAST_REST = 2.0**-24
KINDS = [("forward", "bucket"), ("forward", "drop"), ("reverse", "bucket"), ("jensen", "bucket"), ("jensen", "drop")]


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(shape, seed):
    return torch.randn(shape, generator=generator(seed), device="cuda", dtype=torch.float64)


def units(dtype, vocab):
    u = 2.0**-53 if dtype == torch.float64 else 2.0**-24
    return u, u * (64 + vocab / 256)


def outside(got, want, allowed):
    """Which elements are off by more than allowed; infinities have to be met."""
    got, want, allowed = got.detach().double(), want.double(), allowed.expand(want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    return ~(same | (want.isfinite() & ((got - want).abs() <= allowed)))


def rounded(bound, want, dtype, scale):
    """A bound with the output's rounding; scale: what a probability is multiplied with, at most."""
    least = torch.finfo(dtype).smallest_normal
    subnormal = least * HALF_STEP[dtype] * 2 if dtype == torch.float16 else 0.0
    return bound + HALF_STEP[dtype] * 1.01 * want.abs() + subnormal + scale * torch.finfo(
        torch.float64 if dtype == torch.float64 else torch.float32).smallest_normal


# ---------------------------------------------------------------------------------------------
# Scores


def scores_gradient(x, y, g, h, t):
    """In float64, and its bound."""
    vocab = x.shape[-1]
    u, e = units(x.dtype, vocab)
    used = (y != IGNORE)[..., None]
    z = torch.where(used, x, torch.zeros_like(x)).double()
    z = (z - z.amax(-1, keepdim=True)) / t
    s = z.exp().sum(-1, keepdim=True)
    p = z.exp() / s
    size = torch.where(p > 0, z, 0.0).abs()
    first, second = (p * size).sum(-1, keepdim=True), (p * size * size).sum(-1, keepdim=True)
    c, k = (torch.where(used, v.double()[..., None] / t, 0.0) for v in (g, h))
    slope = c + k * (torch.where(p > 0, z, 0.0) + first)
    want = -p * slope
    want.scatter_add_(-1, torch.where(used, y[..., None], 0), c)
    bound = p * ((e + (8 + 3 * size) * u) * slope.abs() + k.abs() * (2 * e * first + 4 * u * second)
                 + 4 * u * (c.abs() + k.abs() * (size + first)))
    return want, rounded(bound, want, x.dtype, c.abs() + k.abs() * 2000)


def check_scores(x, y, t=1.0, seed=0):
    g, h = (normal(y.shape, seed + i).to(_ext.acc_dtype(x.dtype)) for i in range(2))
    leaf = x.detach().requires_grad_()
    got = ti.token_scores(leaf, y, temperature=t)
    (gx,) = torch.autograd.grad((got.logps, got.entropy), leaf, (g, h))
    want, allowed = scores_gradient(x.detach(), y, g, h, t)
    bad = outside(gx, want, allowed)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off"
    return want, allowed


VOCABS = [7, 33, 257, 1000, 2047, 8192, 32001, 50021, 131072, 200003]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", VOCABS)
def test_scores_gradient(vocab: int, dtype: torch.dtype) -> None:
    x = (normal((2, 3, vocab), vocab) * 3).to(dtype)
    y = torch.randint(0, vocab, (2, 3), generator=generator(vocab), device="cuda")
    y[0, 1] = IGNORE
    check_scores(x, y)
    check_scores(x, y, t=0.6)
    check_scores(x[:, :, :-1], y.clamp(max=vocab - 2))
    check_scores(x[:, 1:], y[:, 1:].contiguous(), t=1.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(2500, 300), (2500, 5000), (700, 32003)])
def test_scores_gradient_of_many_rows(rows: int, vocab: int, dtype: torch.dtype) -> None:
    x = (normal((rows, vocab), rows) * 3).to(dtype)
    y = torch.randint(0, vocab, (rows,), generator=generator(rows), device="cuda")
    y[torch.rand(rows, generator=generator(1), device="cuda") < 0.3] = IGNORE
    check_scores(x, y)


# ---------------------------------------------------------------------------------------------
# Distillation


def near_lists(x, top, seed=0, t=1.0, noise=1.0):
    z = (x.double() + noise * normal(x.shape, seed + 77)) / t
    logps, ids = torch.log_softmax(z, -1).topk(top, -1)
    return ids, logps.to(_ext.acc_dtype(x.dtype))


def ragged(ids, seed=0):
    """Lists that end after 1 to all of their entries."""
    n = ids.shape[-1]
    ends = torch.randint(1, n + 1, ids.shape[:-1], generator=generator(seed + 5), device="cuda")
    return torch.where(torch.arange(n, device="cuda") < ends[..., None], ids, IGNORE)


def distill_gradient(x, ids, logps, kind, rest, mix, w, t, upstream):
    """In float64, and its bound (no token twice in a list)."""
    vocab = x.shape[-1]
    u, e = units(x.dtype, vocab)
    x, ids, logps = x.reshape(-1, vocab), ids.reshape(-1, ids.shape[-1]), logps.reshape(-1, ids.shape[-1])
    there = ids != IGNORE
    w = torch.ones(len(x), device="cuda", dtype=torch.float64) if w is None else w.reshape(-1).double()
    w = w * there[:, 0]
    z = torch.where((w != 0)[:, None], x, torch.zeros_like(x)).double()
    z = (z - z.amax(1, keepdim=True)) / t
    lp = torch.log_softmax(z, 1)
    p = lp.exp()
    row, col = there.nonzero(as_tuple=True)
    listed = torch.zeros_like(p, dtype=torch.bool)
    listed[row, ids[row, col]] = True
    q = torch.zeros_like(p)
    q[row, ids[row, col]] = logps[row, col].double().exp()
    lp_rest = torch.logsumexp(lp.masked_fill(listed, -math.inf), 1, keepdim=True)
    p_rest = lp_rest.exp()
    q_rest = (1 - q.sum(1, keepdim=True)).clamp(min=LEAST_REST if kind == "reverse" else 0.0)
    q_rest = torch.where(listed.all(1, keepdim=True), 0.0, q_rest)
    if rest == "drop":
        q, q_rest = q / q.sum(1, keepdim=True), torch.zeros_like(q_rest)
    of_rest = torch.where(lp_rest > -math.inf, (lp - lp_rest).exp(), 0.0)  # of a token of the rest, within it
    relative = e + (8 + 3 * z.abs()) * u
    slack = (ids.shape[1] + 4) * 2.0**-52
    if kind == "forward":
        whole = q.sum(1, keepdim=True) + q_rest
        teacher = torch.where(listed, q, of_rest * q_rest)
        want, bound = p * whole - teacher, (p * whole + teacher) * (relative + e)
        bound = bound + slack * (p + torch.where(listed, 0.0, of_rest))
    else:
        def slopes(lp, p, q):
            if kind == "reverse":
                return lp - q.log()
            return (1 - mix) * (lp - (mix * q + (1 - mix) * p).log())

        f_listed, f_rest = slopes(lp, p, q), torch.where(p_rest > 0, slopes(lp_rest, p_rest, q_rest), 0.0)
        mean = torch.where(listed, p * f_listed, 0.0).sum(1, keepdim=True) + p_rest * f_rest
        spread = torch.where(listed, p * f_listed.abs(), 0.0).sum(1, keepdim=True) + p_rest * f_rest.abs()
        f = torch.where(listed, f_listed, f_rest)
        want = p * (f - mean)
        bound = p * (relative * (f - mean).abs() + 4 * e * (1 + spread))
        step = 1 / q_rest if kind == "reverse" else mix * (1 - mix) / (mix * q_rest + (1 - mix) * p_rest)
        step = torch.where(p_rest > 0, step * slack, 0.0)
        bound = bound + p * step * (torch.where(listed, 0.0, 1.0) + p_rest)
    c = (w / w.sum() / t * upstream)[:, None]
    return c * want, rounded(c.abs() * bound, c * want, x.dtype, c.abs() * 2000)


def check_distill(x, ids, logps, kind="forward", rest="bucket", mix=0.5, w=None, t=1.0, upstream=1.0, expected=1.0):
    leaf = x.detach().requires_grad_()
    loss = ti.distillation_loss(leaf, ids, logps, kind=kind, rest=rest, mix=mix, weight=w, temperature=t,
                                upstream=expected).loss
    (gx,) = torch.autograd.grad(loss * upstream, leaf)
    want, allowed = distill_gradient(x.detach(), ids, logps, kind, rest, mix, w, t, upstream)
    bad = outside(gx.reshape(want.shape), want, allowed)
    assert gx.shape == x.shape and not bad.any(), f"{int(bad.sum())} of {bad.numel()} off"
    return want, allowed


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", VOCABS)
def test_distill_gradient(vocab: int, dtype: torch.dtype) -> None:
    x = (normal((2, 3, vocab), vocab) * 3).to(dtype)
    for n, (kind, rest) in enumerate(KINDS):
        top = min(vocab, (1, 5, 33, 128, 64)[(n + vocab) % 5])
        ids, logps = near_lists(x, top, n)
        check_distill(x, ids, logps, kind, rest)
        check_distill(x, ragged(ids), logps, kind, rest, mix=0.2, t=1.3, upstream=4.0)
        cut = x[:, :, :vocab - 1]
        check_distill(cut, *near_lists(cut, min(top, vocab - 1)), kind, rest, expected=4.0, upstream=4.0)
        check_distill(x[:, 1:], ids[:, 1:], logps[:, 1:], kind, rest)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(2500, 300), (2500, 5000), (700, 32003)])
def test_distill_gradient_of_many_rows(rows: int, vocab: int, dtype: torch.dtype) -> None:
    x = (normal((rows, vocab), rows) * 3).to(dtype)
    ids, logps = near_lists(x, 20)
    w = (torch.rand(rows, generator=generator(1), device="cuda") < 0.7).float() * 0.5
    for kind, rest in KINDS:
        check_distill(x, ragged(ids), logps, kind, rest, w=w)


@pytest.mark.gpu
def test_the_bounds_see_one_element() -> None:
    # a gradient of 0 at the row's last elements, at its first, and throughout
    for vocab in (1000, 50021, 131072, 200003):
        for dtype in ALL:
            x = (normal((2, vocab), vocab) * 3).to(dtype)
            y = torch.zeros(2, dtype=torch.int64, device="cuda")
            for want, allowed in (check_scores(x, y), check_distill(x, *near_lists(x, 8)),
                                  check_distill(x, *near_lists(x, 8), "jensen")):
                want, allowed = want.cpu(), allowed.cpu()
                seen = want.abs() > 2 * torch.finfo(dtype).smallest_normal
                share = (outside(torch.zeros_like(want), want, allowed) & seen).sum() / seen.sum()
                assert share > 0.99
                tail = want.clone()
                tail[:, -1] = 0
                if seen[:, -1].any():
                    assert outside(tail, want, allowed).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
def test_distill_where_the_vocabulary_is_not_contiguous(dtype: torch.dtype) -> None:
    x = (normal((3, 41, 7), 3) * 3).to(dtype)
    for z in (x.transpose(1, 2), x.permute(2, 0, 1)[..., :30], x[:, ::2].transpose(1, 2)):
        assert z.stride(-1) != 1
        for kind, rest in KINDS:
            ids, logps = near_lists(z, 4)
            check_distill(z, ids, logps, kind, rest)
            check_distill(z, ids, logps, kind, rest, upstream=0.25)


@pytest.mark.gpu
@pytest.mark.parametrize("cut", [0, 1])
@pytest.mark.parametrize("rows,vocab,dtype", [(700, 32003, torch.bfloat16), (2500, 5000, torch.bfloat16),
                                              (40000, 40, torch.float32), (1300, 9001, torch.float32),
                                              (2600, 1001, torch.float64)])
def test_distill_another_upstream(rows: int, vocab: int, dtype: torch.dtype, cut: int) -> None:
    # more tiles than are resident, rows left out between others, ragged lists, tokens twice: the bits of the
    # gradient that is written with the loss for that upstream gradient
    x = (normal((rows, vocab), vocab) * 3).to(dtype)[:, :vocab - cut]
    ids, logps = near_lists(x, 12)
    ids = ragged(ids)
    ids[::3, 1] = torch.where(ids[::3, 1] == IGNORE, IGNORE, ids[::3, 0])
    w = torch.rand(rows, generator=generator(1), device="cuda").to(_ext.acc_dtype(dtype))
    w[torch.rand(rows, generator=generator(2), device="cuda") < 0.33] = 0
    for kind, rest in KINDS:
        grads = []
        for expected in (-3.0, 1.0):
            leaf = x.detach().requires_grad_()
            loss = ti.distillation_loss(leaf, ids, logps, kind=kind, rest=rest, weight=w, upstream=expected).loss
            up = torch.tensor(-3.0, device="cuda", dtype=loss.dtype)
            grads.append(torch.autograd.grad(loss, leaf, up, retain_graph=True)[0])
            grads.append(torch.autograd.grad(loss, leaf, up)[0])
        assert (grads[0][w == 0] == 0).all() and grads[0].isfinite().all()
        for other in grads[1:]:
            assert torch.equal(grads[0], other)


@pytest.mark.gpu
def test_distill_another_upstream_of_large_offsets() -> None:
    rows, vocab = 16500, 131072  # 2^31 elements and more
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    x[-2:] = normal((2, vocab), 1) * 3
    ids = torch.arange(3, device="cuda").expand(rows, 3).contiguous()
    ids[-2:] = torch.tensor([[5, vocab - 1, 70000], [1, 2, vocab - 2]], device="cuda")
    logps = torch.full((rows, 3), math.log(0.2), device="cuda")
    grads = []
    for expected in (2.0 * rows, 1.0):
        leaf = x.requires_grad_()
        loss = ti.distillation_loss(leaf, ids, logps, upstream=expected).loss
        grads.append(torch.autograd.grad(loss, leaf, torch.tensor(2.0 * rows, device="cuda"))[0])
    assert torch.equal(*grads)
    want, allowed = distill_gradient(x.detach()[-2:], ids[-2:], logps[-2:], "forward", "bucket", 0.5, None, 1.0, 4.0)
    assert not outside(grads[1][-2:], want, allowed).any()


# ---------------------------------------------------------------------------------------------
# Infinite results


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", [40, 2500, 40007])
def test_infinite_results(vocab: int, dtype: torch.dtype) -> None:
    # hidden tokens among the alternatives and as targets: -inf and nothing else
    x = torch.full((3, vocab), -math.inf, device="cuda", dtype=dtype)
    x[:, ::vocab // 9] = (normal((3, len(range(0, vocab, vocab // 9))), 1)).to(dtype)
    y = torch.tensor([1, 0, 2], device="cuda")
    got = ti.token_scores(x, y, top=20)
    want = torch.log_softmax(x.double(), -1)
    u, e = units(dtype, vocab)
    tops = want.gather(-1, got.top_ids)
    assert (tops == -math.inf).any()
    assert not outside(got.top_logps, tops, e + 2 * u * tops.abs()).any()
    chosen = want.gather(-1, y[:, None])[:, 0]
    assert (chosen == -math.inf).sum() == 2
    assert not outside(got.logps, chosen, e + 2 * u * chosen.abs()).any()
    # a teacher's token that the student hides; a student's that the teacher has at 0
    ids = torch.tensor([[0, 1], [0, 1], [0, 1]], device="cuda")
    logps = torch.full((3, 2), math.log(0.3), device="cuda", dtype=_ext.acc_dtype(dtype))
    got = ti.distillation_loss(x, ids, logps)
    assert (got.divergence == math.inf).all() and got.loss == math.inf
    logps[:, 0] = -math.inf
    got = ti.distillation_loss(x, ids, logps, kind="reverse")
    assert (got.divergence == math.inf).all() and got.loss == math.inf
    assert ti.distillation_loss(x, ids, logps, kind="jensen").divergence.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", [40, 2500, 40007])
def test_lists_at_the_lowest_value(vocab: int, dtype: torch.dtype) -> None:
    # a student that hides the listed tokens with its type's lowest value: their probability is 0, and as where it is
    # -inf only the others count; and one that hides all but one, or has the largest value outside the list
    least = torch.finfo(dtype).min
    x = (normal((4, vocab), 1) * 3).to(dtype)
    ids, logps = near_lists(x, 6)
    rows = torch.arange(4, device="cuda")[:, None]
    x[rows[1:], ids[1:]] = least
    x[2] = least
    x[2, ids[2, 0].item() - 1] = 0
    x[3, (ids[3] + 1) % vocab] = -least
    hidden = x.clone()
    hidden[1:][hidden[1:] == least] = -math.inf
    hidden[3][hidden[3] != -least] = -math.inf
    for kind, rest in (("reverse", "bucket"), ("jensen", "bucket"), ("jensen", "drop")):
        got, want = [], []
        for z, out in ((x, got), (hidden, want)):
            leaf = z.detach().requires_grad_()
            loss = ti.distillation_loss(leaf, ids, logps, kind=kind, rest=rest)
            out += [loss.loss.detach(), loss.divergence, *torch.autograd.grad(loss.loss, leaf)]
        for a, b in zip(got, want):
            assert b.isfinite().all() and torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", [40, 2500, 40007])
def test_nothing_to_compare_with_and_not_finite(vocab: int, dtype: torch.dtype) -> None:
    # a renormalised list of probability 0 leaves 0; of a row that is not finite NaN, as any other list
    x = (normal((5, vocab), 1) * 3).to(dtype)
    ids, logps = near_lists(x, 5)
    logps[:4] = -math.inf
    x[1, vocab - 1] = math.nan
    x[2] = -math.inf
    x[3, ids[3, 0]] = math.inf
    bad = torch.tensor([False, True, True, True, False], device="cuda")
    for kind in ("forward", "jensen"):
        leaf = x.detach().requires_grad_()
        got = ti.distillation_loss(leaf, ids, logps, kind=kind, rest="drop")
        assert torch.equal(got.divergence.isnan(), bad) and got.divergence[0] == 0
        (gx,) = torch.autograd.grad(got.loss, leaf)
        assert gx[bad].isnan().all() and (gx[0] == 0).all() and gx[4].isfinite().all()
