"""A token's scores (log-probability, entropy, top alternatives) and the distillation from a teacher's
top lists, against their definitions in float64 (plain torch below, gradients by automatic
differentiation of it) and against differences.

Tolerances, float32 arithmetic (float64: the same with 2^-53): as for the log-probabilities, a row's
sum of V exponentials has a relative error of at most ``e = 2^-24 (64 + V / 256)``.

* Entropy ``log s - u / s``, u the sum of ``exp(z) z``: e from the logarithm, ``2 e E|z|`` from the
  quotient, and from the rounding of z, relative to its size, in the exponential and beside it ``4
  2^-24 E[z^2]`` (E over the row's distribution, z relative to its maximum).
* A divergence D: the logarithms of the student's probabilities are off by e each (of the rest by 2 e),
  ``dD / d log P_b = P_b f_b`` (f without its mean), so D by at most ``3 e (1 + sum P |f|)``; so is,
  times its coefficient, a gradient.

On top come the roundings of the outputs to their types.
"""

from __future__ import annotations

import math

import pytest
import torch

import torchisotonic_b200 as ti
from torchisotonic_b200 import _ext, ops

HALF_ULP = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24,
            torch.float64: 2.0**-53}
LEAST = {torch.float16: 2.0**-24, torch.bfloat16: 0.0, torch.float32: 0.0, torch.float64: 0.0}
ALL = [torch.bfloat16, torch.float16, torch.float32, torch.float64]
IGNORE = -100


def unit(dtype: torch.dtype) -> float:
    return 2.0**-53 if dtype == torch.float64 else 2.0**-24


def sum_error(dtype: torch.dtype, vocab: int) -> float:
    return unit(dtype) * (64 + vocab / 256)


def close(got, want, atol, rtol: float = 0.0) -> None:
    """atol: a number, or a tensor that broadcasts against the results."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape
    same = (got == want) | (got.isnan() & want.isnan())
    allowed = torch.as_tensor(atol, dtype=torch.float64).cpu() + rtol * want.abs()
    off = torch.where(same, torch.zeros_like(got), (got - want).abs())
    bad = ~(off <= allowed)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, by up to "
                           f"{float((off / allowed.clamp(min=1e-300)).max()):.3g} times the allowed")


def generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def logits_of(shape, dtype, seed=0, scale=3.0):
    gen = generator(seed)
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float64) * scale
    y = torch.randint(0, shape[-1], shape[:-1], generator=gen, device="cuda")
    return x.to(dtype), y


def upstream_of(shape, dtype, seed=0):
    gen = generator(seed + 1000)
    acc = _ext.acc_dtype(dtype)
    return [torch.randn(shape, generator=gen, device="cuda", dtype=torch.float64).to(acc)
            for _ in range(2)]


# ---------------------------------------------------------------------------------------------
# Scores


def ranked(x, top):
    """Ids of the largest, of equal ones the first; NaN with -inf."""
    x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x)
    return torch.sort(x, dim=-1, descending=True, stable=True)[1][..., :top]


def plain_scores(x, y, top, temperature=1.0, ignore=IGNORE):
    """In float64, differentiable in x: logps (or None), entropy, top_logps, top_ids, and of each row
    E|z| and E[z^2]."""
    lp = torch.log_softmax(x.double() / temperature, -1)
    p = lp.exp()
    finite = torch.where(p > 0, lp, torch.zeros_like(lp))
    entropy = -(p * finite).sum(-1)
    ids = ranked(x.detach(), top)
    tops = lp.detach().gather(-1, ids)
    z = torch.where(p > 0, lp - lp.amax(-1, keepdim=True), torch.zeros_like(lp)).detach()
    first, second = (p.detach() * z.abs()).sum(-1), (p.detach() * z * z).sum(-1)
    logps = None
    if y is not None:
        used = y != ignore
        logps = lp.gather(-1, torch.where(used, y, torch.zeros_like(y))[..., None])[..., 0]
        logps, entropy = (torch.where(used, t, torch.zeros_like(t)) for t in (logps, entropy))
        tops = torch.where(used[..., None], tops, torch.zeros_like(tops))
        ids = torch.where(used[..., None], ids, torch.full_like(ids, ignore))
    return logps, entropy, tops, ids, first, second


def check_scores(x, y, top, temperature=1.0, ignore=IGNORE, grads=True):
    vocab, dtype = x.shape[-1], x.dtype
    acc, e, u = _ext.acc_dtype(dtype), sum_error(dtype, vocab), unit(dtype)
    leaf = x.detach().requires_grad_()
    got = ti.token_scores(leaf, y, top=top, temperature=temperature, ignore_index=ignore)
    assert got.entropy.dtype == got.top_logps.dtype == acc and got.top_ids.dtype == torch.int64
    assert not got.top_logps.requires_grad and got.entropy.shape == x.shape[:-1]
    assert got.top_ids.shape == got.top_logps.shape == (*x.shape[:-1], top)
    # rows that are left out may hold anything: zeros for the float64 side
    seen = x.detach() if y is None else torch.where((y == ignore)[..., None], torch.zeros_like(x), x)
    wide = seen.double().requires_grad_()
    logps, entropy, tops, ids, first, second = plain_scores(wide, y, top, temperature, ignore)
    assert torch.equal(got.top_ids, ids)
    close(got.top_logps, tops, e, 2 * u)
    off = e * (1 + 2 * first) + 4 * u * second
    close(got.entropy, entropy, off, 2 * u)
    if y is None:
        assert got.logps is None
    else:
        assert got.logps.dtype == acc
        close(got.logps, logps, e, 2 * u)
    with torch.no_grad():  # the same without a gradient
        again = ti.token_scores(x, y, top=top, temperature=temperature, ignore_index=ignore)
    for a, b in zip(again, got):
        assert (a is None and b is None) or torch.equal(a, b.detach())
    if not grads:
        return got
    g, h = upstream_of(x.shape[:-1], dtype, vocab)
    outs, ups = [got.entropy], [h]
    wants, wups = [entropy], [h.double()]
    if y is not None:
        outs, ups = [got.logps, *outs], [g, *ups]
        wants, wups = [logps, *wants], [g.double(), *wups]
    (gx,) = torch.autograd.grad(outs, leaf, ups, retain_graph=True)
    assert gx.dtype == dtype and gx.shape == x.shape and gx.is_contiguous()
    (gw,) = torch.autograd.grad(wants, wide, wups)
    # exp(z) (alpha + beta z) / s: the sum's error, that of the mean of z, and the exponential's argument
    # (max p z^2 <= 4 / e^2 of the entropy's part)
    part = (e + 16 * u) * (g.abs() * (y is not None) + h.abs() * (1 + first + entropy.detach()))
    close(gx, gw, ((part + h.abs() * (off + 8 * u)) / temperature)[..., None] + LEAST[dtype],
          HALF_ULP[dtype] * 1.01)
    if y is not None:  # either one alone
        (ga,) = torch.autograd.grad(got.logps, leaf, g, retain_graph=True)
        (gb,) = torch.autograd.grad(got.entropy, leaf, h)
        both = 2 * (part + h.abs() * (off + 8 * u)) / temperature
        ends = (HALF_ULP[dtype] * (ga.double().abs() + gb.double().abs() + gw.abs()) * 1.01
                + 3 * LEAST[dtype])
        close(ga.double() + gb.double(), gw, both[..., None] + ends)
    return got


VOCABS = [1, 2, 7, 8, 31, 33, 257, 1000, 1024, 2047, 4099, 8192, 32001, 50021, 131072, 200003]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", VOCABS)
def test_scores_vocabularies(vocab: int, dtype: torch.dtype) -> None:
    for rows in (1, 5):
        x, y = logits_of((rows, vocab), dtype, seed=vocab + rows)
        for top in sorted({min(vocab, k) for k in (0, 1, 5, 64, 128)}):
            check_scores(x, y, top, grads=top in (0, 5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 70000), (2, 300), (37, 9001), (149, 777), (300, 5000),
                                        (600, 20000), (5000, 40), (3001, 1027), (2500, 9000)])
def test_scores_rows(rows: int, vocab: int, dtype: torch.dtype) -> None:
    x, y = logits_of((rows, vocab), dtype, seed=rows)
    y[torch.rand(rows, device="cuda", generator=generator(7)) < 0.3] = IGNORE
    check_scores(x, y, 20, temperature=0.7)
    check_scores(x, None, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", [5, 130, 1001, 4097, 33001])
def test_scores_layouts(vocab: int, dtype: torch.dtype) -> None:
    x, y = logits_of((3, 9, vocab), dtype, seed=vocab)
    top = min(vocab - 1, 7)
    check_scores(x[:, :-1], y[:, 1:], top)                   # cut along the length
    check_scores(x[:, 1:], y[:, 1:], top)
    check_scores(x[..., :vocab - 1], y % (vocab - 1), top)   # a padded vocabulary
    check_scores(x[..., 1:], y % (vocab - 1), top)           # rows off alignment
    check_scores(x[0, 0], y[0, 0], top)                      # one row, no leading dimension
    check_scores(x[:1].expand(3, 9, vocab), y, top)          # a broadcast input
    check_scores(x.transpose(0, 1), y.t(), top)              # two strides, in another order
    check_scores(x.transpose(1, 2), y[:, :1].expand(3, vocab) % 9, 2)  # the vocabulary not contiguous
    check_scores(x.reshape(3, 3, 3, vocab)[:, :2, 1:], y.reshape(3, 3, 3)[:, :2, 1:], top)
    for a, b in zip(ti.token_scores(x, y.int(), top=top), ti.token_scores(x, y, top=top)):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", [40, 300, 2500, 8000, 40007, 131072])
def test_scores_ties_and_orders(vocab: int, dtype: torch.dtype) -> None:
    at = torch.arange(vocab, device="cuda", dtype=torch.float64)
    gen = generator(vocab)
    few = torch.randint(0, 3, (vocab,), generator=gen, device="cuda").double()
    dense = torch.full((vocab,), -9.0, device="cuda", dtype=torch.float64)
    dense[vocab // 3:vocab // 3 + 300] = 2.0           # all of the largest side by side
    strided = torch.where(at % 256 == 3, 1.0, 0.0)     # all of them with one thread
    signs = torch.where(at % 2 == 0, 0.0, -0.0)
    rows = [torch.ones_like(at), few, at / vocab, -at / vocab, dense, strided, signs, (at * 7) % 13]
    x = torch.stack(rows).to(dtype)
    y = torch.randint(0, vocab, (len(rows),), generator=gen, device="cuda")
    for top in (1, 4, 40, 128):
        if top <= vocab:
            check_scores(x, y, top, grads=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(2500, 300), (2500, 2000), (2500, 9000), (2500, 20000), (300, 70001)])
def test_scores_alternatives_of_many_rows(rows: int, vocab: int, dtype: torch.dtype) -> None:
    # as many as a warp, a small and a large CTA and a cluster choose from, also where many are equal
    x, _ = logits_of((rows, vocab), dtype, seed=rows + vocab)
    flat = (x * 0.5).round()
    offset = x + 200  # what is left of the differences is below the upper 16 bits of a float
    for z in (x, flat, offset):
        want = ranked(z, 128)
        lp = torch.log_softmax(z.double(), -1).gather(-1, want)
        for top in (1, 16, 17, 33, 64, 65, 128):
            got = ti.token_scores(z, None, top=top)
            assert torch.equal(got.top_ids, want[:, :top])
            close(got.top_logps, lp[:, :top], sum_error(dtype, vocab), 2 * unit(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", [40, 2500, 40007])
def test_scores_masked_vocabulary(vocab: int, dtype: torch.dtype) -> None:
    least = torch.finfo(dtype).min
    x, y = logits_of((8, vocab), dtype, seed=vocab)
    hidden = torch.rand(8, vocab, device="cuda", generator=generator(1)) < 0.7
    hidden.scatter_(1, y[:, None], False)
    for fill in (-math.inf, least):
        check_scores(torch.where(hidden, torch.full_like(x, fill), x), y, 8)
    # fewer tokens left than alternatives asked for: the hidden ones follow, by their id
    few = torch.full_like(x, -math.inf)
    few[:, [3, vocab // 2, vocab - 1]] = x[:, :3]
    got = check_scores(few, y * 0 + 3, 20)
    assert (got.top_logps[:, 3:] == -math.inf).all()
    # all but the target hidden: nothing uncertain, no gradient
    only = torch.full_like(x, -math.inf).scatter_(1, y[:, None], 2.0).requires_grad_()
    got = ti.token_scores(only, y, top=2)
    assert (got.logps == 0).all() and (got.entropy == 0).all() and (got.top_ids[:, 0] == y).all()
    (gx,) = torch.autograd.grad((got.logps.sum() + got.entropy.sum()), only)
    assert (gx == 0).all()
    # every logit the type's lowest: uniform
    got = ti.token_scores(torch.full_like(x, least), y, top=5)
    close(got.entropy, torch.full_like(got.entropy, math.log(vocab)), sum_error(dtype, vocab),
          2 * unit(dtype))
    assert torch.equal(got.top_ids, torch.arange(5, device="cuda").expand(8, 5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", [40, 2500, 40007])
def test_scores_not_finite(vocab: int, dtype: torch.dtype) -> None:
    # nothing but -inf, a +inf or a NaN anywhere: NaN for that row alone
    x, y = logits_of((7, vocab), dtype, seed=vocab)
    x[1] = -math.inf
    x[3, vocab // 2] = math.inf
    x[4, vocab - 1] = math.nan
    x[5] = math.nan
    leaf = x.requires_grad_()
    got = ti.token_scores(leaf, y, top=6)
    assert torch.equal(got.top_ids, ranked(x.detach(), 6))
    bad = torch.tensor([False, True, False, True, True, True, False], device="cuda")
    assert torch.equal(got.logps.isnan(), bad) and torch.equal(got.entropy.isnan(), bad)
    assert torch.equal(got.top_logps.isnan().all(1), bad) and torch.equal(got.top_logps.isnan().any(1), bad)
    (gx,) = torch.autograd.grad(got.logps.sum() + got.entropy.sum(), leaf)
    assert gx[1].isnan().all() and gx[4].isnan().all() and not gx[~bad].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [40, 2500, 40007])
def test_scores_targets(vocab: int) -> None:
    x, y = logits_of((6, vocab), torch.float32, seed=vocab)
    x[2] = math.nan  # left out: not read
    y[2] = IGNORE
    check_scores(x, y, 4)
    y[y == 7] = 8
    y[2] = 7
    check_scores(x, y, 4, ignore=7)
    # out of range: a NaN log-probability and gradient, for that row alone
    y[2] = IGNORE
    for wrong in (vocab, -1, 2**40):
        z = y.clone()
        z[4] = wrong
        leaf = x.detach().requires_grad_()
        got = ti.token_scores(leaf, z, top=4)
        assert got.logps.isnan().tolist() == [False] * 4 + [True, False]
        assert not got.entropy.isnan().any() and not got.top_logps.isnan().any()
        (gx,) = torch.autograd.grad(got.logps.sum() + got.entropy.sum(), leaf)
        assert gx[4].isnan().all() and not gx[[0, 1, 2, 3, 5]].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [0.05, 0.7, 30.0])
@pytest.mark.parametrize("vocab", [777, 32000])
def test_scores_temperature(vocab: int, temperature: float) -> None:
    x, y = logits_of((9, vocab), torch.float32, seed=3)
    check_scores(x, y, 11, temperature=temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 5), (2, 0, 5), (0, 40000)])
def test_scores_no_rows(shape) -> None:
    x = torch.zeros(shape, device="cuda", requires_grad=True)
    got = ti.token_scores(x, torch.zeros(shape[:-1], dtype=torch.int64, device="cuda"), top=3)
    assert got.top_ids.shape == (*shape[:-1], 3)
    (got.logps.sum() + got.entropy.sum()).backward()
    assert x.grad is not None and x.grad.shape == shape


@pytest.mark.gpu
def test_scores_large_offsets() -> None:
    # more than 2^31 logits: the last rows lie past 32-bit offsets
    rows, vocab = 16500, 131072
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    x[-2:] = torch.randn(2, vocab, generator=generator(1), device="cuda") * 3
    y = torch.full((rows,), vocab - 1, device="cuda")
    leaf = x.requires_grad_()
    got = ti.token_scores(leaf, y, top=4)
    logps, entropy, tops, ids, first, second = plain_scores(x.detach()[-2:], y[-2:], 4)
    e, u = sum_error(x.dtype, vocab), unit(x.dtype)
    assert torch.equal(got.top_ids[-2:], ids)
    assert torch.equal(got.top_ids[:-2], torch.arange(4, device="cuda").expand(rows - 2, 4))
    close(got.logps[-2:], logps, e, 2 * u)
    close(got.entropy[-2:], entropy, e * (1 + 2 * first) + 4 * u * second, 2 * u)
    (gx,) = torch.autograd.grad(got.entropy.sum(), leaf)
    lp = torch.log_softmax(x.detach()[-2:].double(), 1)
    want = -lp.exp() * (lp + entropy[:, None])
    close(gx[-2:], want, (e + 16 * u) * 40, HALF_ULP[x.dtype] * 1.01)
    # uniform rows: log p + entropy is the rounding of two numbers of the size of log V
    assert gx[:-2].abs().max() <= (2 * e + 40 * u) / vocab * 12


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 11), (2, 1100)])
def test_scores_gradcheck(shape) -> None:
    x, y = logits_of(shape, torch.float64, scale=1.0)

    def f(t):
        got = ti.token_scores(t, y, top=2, temperature=1.3)
        return got.logps, got.entropy

    assert torch.autograd.gradcheck(f, (x.requires_grad_(),))
    assert torch.autograd.gradcheck(lambda t: ti.token_scores(t, None).entropy, (x,))


@pytest.mark.gpu
def test_scores_broadcast_gradient() -> None:
    # one row of logits read by many tokens: their gradients add up in the row
    x, _ = logits_of((1, 1203), torch.float64)
    y = torch.arange(40, device="cuda")
    leaf, wide = x.clone().requires_grad_(), x.clone().requires_grad_()
    got = ti.token_scores(leaf.expand(40, 1203), y, top=1)
    (got.logps.sum() - 0.5 * got.entropy.sum()).backward()
    logps, entropy, *_ = plain_scores(wide.expand(40, 1203), y, 1)
    (logps.sum() - 0.5 * entropy.sum()).backward()
    close(leaf.grad, wide.grad, 40 * 2.0**-53 * (64 + 1203 / 256 + 200))


# ---------------------------------------------------------------------------------------------
# Distillation


LEAST_REST = 2.0**-24


def plain_divergence(z, ids, logps, kind, rest, mix, ignore):
    """One row's divergence from its definition, in float64 on the CPU, differentiable in z (logits /
    temperature); also sum P |f|."""
    vocab = z.numel()
    q: dict[int, float] = {}
    for i, lp in zip(ids.tolist(), logps.tolist()):
        if i != ignore:
            q[i] = q.get(i, 0.0) + math.exp(lp)
    names = sorted(q)
    lp_all = torch.log_softmax(z, 0)
    others = torch.ones(vocab, dtype=torch.bool)
    others[names] = False
    rest_lp = (torch.logsumexp(lp_all[others], 0) if others.any()
               else torch.tensor(-math.inf, dtype=torch.float64))
    lp = torch.cat([lp_all[names], rest_lp[None]])
    total = math.fsum(q.values())
    if rest == "drop":
        if total == 0:
            return z.sum() * 0.0, 0.0
        values = [v / total for v in q.values()]
        values = [q[n] / total for n in names] + [0.0]
    else:
        left = max(0.0, 1.0 - total) if len(names) < vocab else 0.0
        if kind == "reverse" and len(names) < vocab:
            left = max(left, LEAST_REST)
        values = [q[n] for n in names] + [left]
    qs = torch.tensor(values, dtype=torch.float64)
    lq = qs.log()
    zero = torch.zeros_like(lp)
    p = lp.exp()
    if kind == "forward":
        d = torch.where(qs > 0, qs * (lq - lp), zero).sum()
        spread = float(qs.sum())
    elif kind == "reverse":
        f = torch.where(p > 0, lp, zero) - torch.where(p > 0, lq, zero)
        d = (p * f).sum()
        spread = float((p * f.abs()).sum().detach())
    else:
        lm = torch.logaddexp(lq + math.log(mix), lp + math.log1p(-mix))
        safe_lp, safe_lm = torch.where(p > 0, lp, zero), torch.where(p > 0, lm, zero)
        d = (mix * torch.where(qs > 0, qs * (lq - lm), zero).sum()
             + (1 - mix) * (p * (safe_lp - safe_lm)).sum())
        spread = float((p * (safe_lp - safe_lm).abs()).sum().detach())
    return d, spread


def lists_of(x, top, dtype=None, seed=0, temperature=1.0, noise=1.0):
    """A teacher near the student: ids and log-probabilities of its top."""
    gen = generator(seed + 77)
    z = x.double() + noise * torch.randn(x.shape, generator=gen, device="cuda", dtype=torch.float64)
    lp = torch.log_softmax(z / temperature, -1)
    logps, ids = lp.topk(top, -1)
    return ids, logps.to(dtype or _ext.acc_dtype(x.dtype))


def check_distill(x, ids, logps, *, kind="forward", rest="bucket", mix=0.5, weight=None,
                  temperature=1.0, ignore=IGNORE, upstream=1.0, expected=None):
    """One call's values and gradient against the definition, row by row."""
    vocab, dtype = x.shape[-1], x.dtype
    acc, e, u = _ext.acc_dtype(dtype), sum_error(dtype, vocab), unit(dtype)
    settings = dict(kind=kind, rest=rest, mix=mix, weight=weight, temperature=temperature,
                    ignore_index=ignore)
    leaf = x.detach().requires_grad_()
    got = ti.distillation_loss(leaf, ids, logps, upstream=upstream if expected is None else expected,
                               **settings)
    assert got.loss.dtype == got.divergence.dtype == acc and got.loss.shape == ()
    assert got.divergence.shape == x.shape[:-1] and not got.divergence.requires_grad
    with torch.no_grad():
        again = ti.distillation_loss(x, ids, logps, **settings)
    assert torch.equal(again.loss, got.loss.detach()) or got.loss.isnan()
    assert torch.equal(again.divergence.nan_to_num(), got.divergence.nan_to_num())
    (gx,) = torch.autograd.grad(got.loss * upstream, leaf)
    assert gx.dtype == dtype and gx.shape == x.shape and gx.is_contiguous()
    flat = x.detach().reshape(-1, vocab).double().cpu()
    ids_, lps_ = ids.reshape(-1, ids.shape[-1]).cpu(), logps.reshape(-1, ids.shape[-1]).double().cpu()
    lps_ = lps_.to(acc).double()
    w = torch.ones(len(flat), dtype=torch.float64) if weight is None else weight.reshape(-1).double().cpu()
    w = w * (ids_[:, 0] != ignore)
    total = float(w.sum())
    ds, gs, offs = [], [], []
    for r in range(len(flat)):
        if w[r] == 0:
            ds.append(0.0)
            gs.append(torch.zeros(vocab, dtype=torch.float64))
            offs.append(0.0)
            continue
        row = flat[r].requires_grad_()
        d, spread = plain_divergence(row / temperature, ids_[r], lps_[r], kind, rest, mix, ignore)
        (g,) = torch.autograd.grad(d, row)
        # tokens of -inf that are not listed have no gradient
        hidden = row.detach() == -math.inf
        hidden[ids_[r][(ids_[r] != ignore)]] = False
        ds.append(float(d.detach()))
        gs.append(torch.where(hidden, torch.zeros_like(g), g) * w[r] / total)
        offs.append(3 * e * (1 + spread))
    ds, offs = torch.tensor(ds, dtype=torch.float64), torch.tensor(offs, dtype=torch.float64)
    gs = torch.stack(gs) if gs else torch.zeros(0, vocab, dtype=torch.float64)
    close(got.divergence.reshape(-1), ds, offs, 2 * u)
    want = float((w * ds).sum()) / total if total else 0.0
    # w D is rounded once for each row, the sum is in double
    close(got.loss, torch.tensor(want, dtype=torch.float64), float((w * (offs + 4 * u * ds.abs())).sum() / total) if total else 0.0,
          2 * u)
    c = (w.abs() / total / temperature * abs(upstream))[:, None] if total else torch.zeros(len(w), 1)
    close(gx.reshape(-1, vocab), gs * upstream, c * (offs[:, None] + 8 * u) + LEAST[dtype],
          HALF_ULP[dtype] * 1.01 + 4 * u)
    return got


KINDS = [("forward", "bucket"), ("forward", "drop"), ("reverse", "bucket"), ("jensen", "bucket"),
         ("jensen", "drop")]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", VOCABS)
def test_distill_vocabularies(vocab: int, dtype: torch.dtype) -> None:
    x, _ = logits_of((5, vocab), dtype, seed=vocab)
    for n, (kind, rest) in enumerate(KINDS):
        top = min(vocab, (1, 5, 33, 128, 64)[(n + vocab) % 5])
        check_distill(x, *lists_of(x, top, seed=n), kind=kind, rest=rest)
    check_distill(x[:1], *lists_of(x[:1], min(vocab, 20)), upstream=-2.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 70000), (2, 300), (37, 9001), (149, 777), (700, 40),
                                        (400, 1027), (310, 9000)])
def test_distill_rows(rows: int, vocab: int, dtype: torch.dtype) -> None:
    x, _ = logits_of((rows, vocab), dtype, seed=rows)
    ids, logps = lists_of(x, 17, temperature=1.7)
    gen = generator(rows)
    numbers = torch.rand(rows, generator=gen, device="cuda")
    numbers[torch.rand(rows, generator=gen, device="cuda") < 0.3] = 0.0
    numbers[0] = 0.5
    check_distill(x, ids, logps, weight=numbers, temperature=1.7)
    check_distill(x, ids, logps, kind="jensen", mix=0.2, weight=numbers > 0.2, temperature=1.7,
                  upstream=3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(2500, 300), (2500, 5000), (2500, 9000), (700, 32003)])
def test_distill_many_rows(rows: int, vocab: int) -> None:
    # more rows than fit the GPU at once, against the same rows a few at a time
    x, _ = logits_of((rows, vocab), torch.bfloat16, seed=rows)
    ids, logps = lists_of(x, 9)
    leaf = x.requires_grad_()
    got = ti.distillation_loss(leaf, ids, logps, upstream=float(rows))
    (gx,) = torch.autograd.grad(got.loss * rows, leaf)
    e, u = sum_error(x.dtype, vocab), unit(x.dtype)
    for a in (0, rows // 2, rows - 40):
        part = x.detach()[a:a + 40].requires_grad_()
        few = ti.distillation_loss(part, ids[a:a + 40], logps[a:a + 40], upstream=40.0)
        (gp,) = torch.autograd.grad(few.loss * 40, part)
        close(few.divergence, got.divergence[a:a + 40], 12 * e, 4 * u)
        close(gp, gx[a:a + 40].double(), 12 * e, HALF_ULP[x.dtype] * 2.02)
    close(got.loss, got.divergence.double().mean(), 0.0, 4 * u)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", [6, 130, 1001, 4097, 33001])
def test_distill_layouts(vocab: int, dtype: torch.dtype) -> None:
    x, _ = logits_of((3, 5, vocab), dtype, seed=vocab)
    top = min(vocab - 1, 7)
    for z in (x[:, :-1], x[:, 1:], x[..., :vocab - 1], x[..., 1:], x[0, 0], x[:1].expand(3, 5, vocab),
              x.transpose(0, 1), x.transpose(1, 2)[..., :top + 1] if vocab > 9 and top < 5 else x):
        check_distill(z, *lists_of(z, min(top, z.shape[-1])), kind="jensen")
    ids, logps = lists_of(x, top)
    want = ti.distillation_loss(x, ids, logps)
    spread = torch.stack([logps, logps], -1)[..., 0]  # converted, strided
    for got in (ti.distillation_loss(x, ids.int(), logps), ti.distillation_loss(x, ids, spread),
                ti.distillation_loss(x, ids, logps, weight=torch.ones(3, 5, device="cuda", dtype=torch.int32))):
        assert torch.equal(got.loss, want.loss) and torch.equal(got.divergence, want.divergence)
    half = logps.bfloat16()
    check_distill(x, ids, half)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,rest", KINDS)
@pytest.mark.parametrize("vocab", [9, 300, 8001])
def test_distill_lists(vocab: int, kind: str, rest: str) -> None:
    for dtype in (torch.float32, torch.bfloat16):
        x, _ = logits_of((6, vocab), dtype, seed=vocab)
        top = min(vocab - 1, 40)
        ids, logps = lists_of(x, top)
        # entries left out, in the middle and at the end; they may hold anything
        cut, cut_logps = ids.clone(), logps.clone()
        cut[1, 1::2] = IGNORE
        cut[2, 3:] = IGNORE
        cut_logps[cut == IGNORE] = math.nan
        check_distill(x, cut, cut_logps, kind=kind, rest=rest)
        # nothing but entries left out: the token is
        cut[4] = IGNORE
        got = check_distill(x, cut, cut_logps, kind=kind, rest=rest)
        assert got.divergence[4] == 0
        # any order, a token more than once: its probabilities are added
        again = torch.cat([ids.flip(-1), ids[:, :3], ids[:, :1]], -1)
        twice = torch.cat([logps.flip(-1), logps[:, :3], logps[:, :1]], -1) - math.log(2.0)
        check_distill(x, again, twice, kind=kind, rest=rest)
        assert torch.equal(again[0, :top].sort()[0], ids[0].sort()[0])
        # another mark
        other = torch.where(cut == IGNORE, vocab + 5, cut)
        check_distill(x, other, cut_logps, kind=kind, rest=rest, ignore=vocab + 5)
        # probabilities of 0 in the list (the reverse divergence is infinite there)
        if kind != "reverse":
            none = logps.clone()
            none[:, 1] = -math.inf
            check_distill(x, ids, none, kind=kind, rest=rest)
            if rest == "drop":
                none[3] = -math.inf  # nothing to compare with
                assert check_distill(x, ids, none, kind=kind, rest=rest).divergence[3] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(2, 131075), (400, 20011), (2500, 1003)])
def test_distill_lists_in_one_place(rows: int, vocab: int) -> None:
    # tokens 2048 apart (one thread has them all), side by side at either end of the row, and all of them
    # listed twice
    x, _ = logits_of((rows, vocab), torch.bfloat16, seed=vocab)
    apart = torch.arange(5, vocab, 2048, device="cuda")[:64]
    ends = torch.cat([torch.arange(20, device="cuda"), torch.arange(vocab - 20, vocab, device="cuda")])
    few = slice(0, 3)
    for ids in (apart, ends, torch.cat([apart, apart.flip(0)]), torch.cat([ends, ends])):
        lists = ids.expand(rows, len(ids)).contiguous()
        logps = torch.full(lists.shape, -math.log(len(ids) + 3.0), device="cuda")
        leaf = x.detach().requires_grad_()
        got = ti.distillation_loss(leaf, lists, logps, upstream=float(rows))
        (gx,) = torch.autograd.grad(got.loss * rows, leaf)
        part = check_distill(x[few], lists[few], logps[few])
        close(got.divergence[few], part.divergence, 12 * sum_error(x.dtype, vocab), 2.0**-22)
        leaf = x[few].detach().requires_grad_()
        n = len(leaf)
        (gp,) = torch.autograd.grad(ti.distillation_loss(leaf, lists[few], logps[few],
                                                         upstream=float(n)).loss * n, leaf)
        close(gx[few], gp.double(), 12 * sum_error(x.dtype, vocab), HALF_ULP[x.dtype] * 2.02)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,rest", KINDS)
@pytest.mark.parametrize("vocab", [1, 2, 30, 128])
def test_distill_whole_vocabulary(vocab: int, kind: str, rest: str) -> None:
    # no rest: the divergence of the two distributions, and no loss from the rounding of their sum
    for dtype in (torch.float32, torch.float64):
        x, _ = logits_of((4, vocab), dtype, seed=vocab)
        ids, logps = lists_of(x, vocab)
        got = check_distill(x, ids, logps, kind=kind, rest=rest)
        assert got.loss.isfinite()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float64])
@pytest.mark.parametrize("vocab", [40, 5000, 70001])
def test_distill_sure_student(vocab: int, dtype: torch.dtype) -> None:
    # the rest's probability far below the row's own: neither cancelled nor underflown
    x, _ = logits_of((5, vocab), dtype, seed=vocab)
    x[:, 3] = torch.tensor([20.0, 60.0, 120.0, 400.0, 3000.0], device="cuda").to(dtype)
    ids = torch.tensor([3, 7, 11], device="cuda").expand(5, 3).contiguous()
    logps = torch.tensor([0.5, 0.2, 0.1], device="cuda", dtype=_ext.acc_dtype(dtype)).log().expand(5, 3).contiguous()
    for kind, rest in KINDS:
        check_distill(x, ids, logps, kind=kind, rest=rest)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", [40, 2500, 40007])
def test_distill_masked_vocabulary(vocab: int, dtype: torch.dtype) -> None:
    x, _ = logits_of((6, vocab), dtype, seed=vocab)
    ids, logps = lists_of(x, 8)
    hidden = torch.rand(6, vocab, device="cuda", generator=generator(2)) < 0.6
    hidden.scatter_(1, ids, False)
    least = torch.finfo(dtype).min
    for fill in (-math.inf, least):
        z = torch.where(hidden, torch.full_like(x, fill), x)
        for kind, rest in KINDS:
            check_distill(z, ids, logps, kind=kind, rest=rest)
    # a listed token hidden: infinite in "forward", not in the others; its gradient is -Q
    z = x.clone()
    z[2, ids[2, 1]] = -math.inf
    leaf = z.requires_grad_()
    got = ti.distillation_loss(leaf, ids, logps)
    (gx,) = torch.autograd.grad(got.loss, leaf)
    assert got.divergence[2] == math.inf and got.divergence[[0, 1, 3, 4, 5]].isfinite().all()
    close(gx[2, ids[2, 1]], -logps[2, 1].double().exp() / 6, LEAST[dtype], HALF_ULP[dtype] * 1.01 + 4 * unit(dtype))
    assert gx.isfinite().all()
    for kind in ("reverse", "jensen"):
        check_distill(z.detach(), ids, logps, kind=kind)
    # all but the list hidden: the rest has no probability, and no gradient
    z = torch.full_like(x, -math.inf).scatter_(1, ids, x.gather(1, ids))
    for kind, rest in KINDS:
        leaf = z.detach().requires_grad_()
        got = ti.distillation_loss(leaf, ids, logps, kind=kind, rest=rest)
        (gx,) = torch.autograd.grad(got.loss, leaf)
        assert (got.loss == math.inf) == ((kind, rest) == ("forward", "bucket"))
        assert gx.isfinite().all() and (gx.scatter(1, ids, 0.0) == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", [40, 2500, 40007])
def test_distill_not_finite(vocab: int, dtype: torch.dtype) -> None:
    x, _ = logits_of((8, vocab), dtype, seed=vocab)
    ids, logps = lists_of(x, 5)
    x[1] = -math.inf
    x[2, ids[2, 0]] = math.inf
    x[3, ids[3, 1]] = math.nan
    x[4] = math.nan
    ids[5, 2] = vocab
    logps[6, 3] = math.nan
    bad = torch.tensor([False, True, True, True, True, True, True, False], device="cuda")
    for kind, rest in KINDS:
        leaf = x.detach().requires_grad_()
        got = ti.distillation_loss(leaf, ids, logps, kind=kind, rest=rest)
        assert torch.equal(got.divergence.isnan(), bad) and got.loss.isnan()
        (gx,) = torch.autograd.grad(got.loss, leaf)
        assert not gx[~bad].isnan().any()
        assert gx[1].isnan().all() and gx[4].isnan().all() and gx[5].isnan().all()
        # left out, they are not read
        w = ~bad
        leaf = x.detach().requires_grad_()
        got = ti.distillation_loss(leaf, ids, logps, kind=kind, rest=rest, weight=w)
        (gx,) = torch.autograd.grad(got.loss, leaf)
        assert got.loss.isfinite() and (got.divergence[bad] == 0).all() and (gx[bad] == 0).all()


@pytest.mark.gpu
def test_distill_nothing_left() -> None:
    x, _ = logits_of((4, 700), torch.float32)
    ids, logps = lists_of(x, 5)
    for weight in (torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda", dtype=torch.bool)):
        got = check_distill(x, ids, logps, weight=weight)
        assert got.loss == 0
    got = check_distill(x, torch.full_like(ids, IGNORE), logps)
    assert got.loss == 0
    for shape in ((0, 9), (2, 0, 9), (0, 40000)):
        z = torch.zeros(shape, device="cuda", requires_grad=True)
        got = ti.distillation_loss(z, torch.zeros((*shape[:-1], 3), device="cuda", dtype=torch.int64),
                                   torch.zeros((*shape[:-1], 3), device="cuda"))
        assert got.loss == 0
        got.loss.backward()
        assert z.grad.shape == shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("vocab", [50, 3001, 40007])
def test_distill_upstream(vocab: int, dtype: torch.dtype) -> None:
    # the expected upstream gradient, another one, and the backward a second time
    x, _ = logits_of((6, vocab), dtype, seed=vocab)
    ids, logps = lists_of(x, 12)
    ids[1, 5] = ids[1, 2]  # also where a token is listed twice
    ids[2, 7:] = IGNORE
    w = torch.tensor([1.0, 2.0, 0.0, 0.5, 1.0, 1.0], device="cuda")
    check_distill(x, ids, logps, weight=w, upstream=0.1, expected=0.1)
    check_distill(x, ids, logps, weight=w, upstream=1024.0, expected=0.1)
    leaf = x.requires_grad_()
    loss = ti.distillation_loss(leaf, ids, logps, weight=w, upstream=0.1).loss
    tenth = torch.tensor(0.1, device="cuda", dtype=loss.dtype)
    got = [torch.autograd.grad(loss, leaf, g, retain_graph=True)[0] for g in (tenth, tenth, tenth * 4)]
    assert torch.equal(got[0], got[1]) and got[0].data_ptr() != got[1].data_ptr()
    close(got[2], 4 * got[0].double(), 8 * LEAST[dtype], HALF_ULP[dtype] * 2.02)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,rest", KINDS)
@pytest.mark.parametrize("shape", [(4, 9), (3, 1100)])
def test_distill_gradcheck(shape, kind: str, rest: str) -> None:
    x, _ = logits_of(shape, torch.float64, scale=1.0)
    ids, logps = lists_of(x, 4)
    w = torch.rand(shape[0], device="cuda", dtype=torch.float64, generator=generator(3)) + 0.1
    assert torch.autograd.gradcheck(
        lambda t: ti.distillation_loss(t, ids, logps, kind=kind, rest=rest, mix=0.3, weight=w,
                                       temperature=1.4).loss, (x.requires_grad_(),))


@pytest.mark.gpu
def test_distill_large_offsets() -> None:
    rows, vocab = 16500, 131072
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    x[-2:] = torch.randn(2, vocab, generator=generator(1), device="cuda") * 3
    ids = torch.arange(3, device="cuda").expand(rows, 3).contiguous()
    ids[-2:] = torch.tensor([[5, vocab - 1, 70000], [1, 2, vocab - 2]], device="cuda")
    logps = torch.full((rows, 3), math.log(0.2), device="cuda")
    leaf = x.requires_grad_()
    got = ti.distillation_loss(leaf, ids, logps, upstream=float(rows))
    (gx,) = torch.autograd.grad(got.loss * rows, leaf)
    tail = x.detach()[-2:]
    part = tail.clone().requires_grad_()
    few = check_distill(part, ids[-2:], logps[-2:])
    (gp,) = torch.autograd.grad(ti.distillation_loss(part, ids[-2:], logps[-2:], upstream=2.0).loss * 2, part)
    e = sum_error(x.dtype, vocab)
    close(got.divergence[-2:], few.divergence, 12 * e, 2.0**-22)
    close(gx[-2:], gp.double(), 12 * e, HALF_ULP[x.dtype] * 2.02)
    assert (gx[:-2] == gx[0]).all()


# ---------------------------------------------------------------------------------------------
# Together, and around both


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_teacher_to_student(dtype: torch.dtype) -> None:
    # a teacher's lists as they come, prompt tokens ignored, a student's step, a calibration curve
    teacher, y = logits_of((3, 7, 1300), dtype, seed=1)
    student, _ = logits_of((3, 7, 1300), dtype, seed=2)
    y[:, :2] = IGNORE
    lists = ti.token_scores(teacher, y, top=24, temperature=2.0)
    got = check_distill(student, lists.top_ids, lists.top_logps, temperature=2.0)
    assert (got.divergence[:, :2] == 0).all() and (got.divergence[:, 2:] > 0).all()
    # of the teacher from itself nothing is to learn
    same = check_distill(teacher, lists.top_ids, lists.top_logps, temperature=2.0)
    assert same.loss.abs() <= 40 * sum_error(dtype, 1300)
    p = torch.nn.Parameter(student.float())
    opt = ti.AdamW([p], lr=0.05)
    losses = []
    for _ in range(3):
        loss = ti.distillation_loss(p, lists.top_ids, lists.top_logps, temperature=2.0).loss
        loss.backward()
        opt.step()
        opt.zero_grad()
        losses.append(float(loss.detach()))
    assert all(math.isfinite(v) for v in losses)
    best = ti.token_scores(p.detach(), None, top=1)
    right = (best.top_ids[..., 0] == lists.top_ids[..., 0])[:, 2:].flatten().float()
    xs, curve = ti.fit_calibration(best.top_logps[:, 2:, 0].exp().flatten(), right)
    assert (curve[1:] >= curve[:-1]).all() and len(xs) == len(curve)


@pytest.mark.gpu
def test_scores_and_distillation_repeat_exactly() -> None:
    for shape in ((700, 30011), (4000, 900), (3, 131072)):
        x, y = logits_of(shape, torch.bfloat16)
        ids, logps = lists_of(x, 30)

        def once():
            leaf = x.detach().requires_grad_()
            a = ti.token_scores(leaf, y, top=30)
            b = ti.distillation_loss(leaf, ids, logps, kind="jensen")
            return [*a, *b, *torch.autograd.grad(a.logps.sum() + a.entropy.sum(), leaf),
                    *torch.autograd.grad(b.loss, leaf)]

        for a, b in zip(once(), once()):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_scores_and_distillation_on_other_streams() -> None:
    # two streams at once, each with inputs and workspaces of its own
    x, y = logits_of((64, 30011), torch.bfloat16)
    ids, logps = lists_of(x, 10)

    def both(z):
        leaf = z.detach().requires_grad_()
        a, b = ti.token_scores(leaf, y, top=10), ti.distillation_loss(leaf, ids, logps)
        return [*a, *b, *torch.autograd.grad(b.loss, leaf)]

    inputs = [x, x.flip(0).contiguous()]
    want = [both(z) for z in inputs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = both(inputs[i])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for u, v in zip(a, b):
            assert torch.equal(u.detach(), v.detach())


@pytest.mark.gpu
def test_scores_and_distillation_in_cuda_graphs() -> None:
    # two captured graphs, replayed in turn on new inputs, forward and backward
    x, y = logits_of((32, 9001), torch.bfloat16)
    ids, logps = lists_of(x, 10)

    def both(leaf):
        a, b = ti.token_scores(leaf, y, top=10), ti.distillation_loss(leaf, ids, logps)
        (g,) = torch.autograd.grad(b.loss + a.entropy.mean(), leaf)
        return [*(t.detach() for t in (*a, *b)), g]

    held = [x.clone().requires_grad_(), x.clone().requires_grad_()]
    for leaf in held:
        both(leaf)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph, leaf in zip(graphs, held):
        with torch.cuda.graph(graph):
            outs.append(both(leaf))
    for shift in (0.5, 1.0):
        new = [(x.float() * shift).bfloat16(), (x.float() - shift * x.float().flip(0)).bfloat16()]
        with torch.no_grad():
            for leaf, z in zip(held, new):
                leaf.copy_(z)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out, z in zip(outs, new):
            want = both(z.detach().requires_grad_())
            for u, v in zip(out, want):
                assert torch.equal(u, v)


# ---------------------------------------------------------------------------------------------
# torch.library operators


def test_operators_refuse_without_a_gpu() -> None:
    x, y = torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64)
    ids, logps = torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2)
    for call in (lambda: ops.token_scores(x, y, 2, 1.0, IGNORE),
                 lambda: ops.token_scores_grad(x, y, 1.0, torch.zeros(9), logps[:, 0], logps[:, 0]),
                 lambda: ops.distillation(x, ids, logps, None, 0, False, 0.5, 1.0, IGNORE),
                 lambda: ops.distillation_grad(x, ids, 1.0, IGNORE, torch.zeros(9, dtype=torch.float64), logps[0, 0])):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


@pytest.mark.gpu
def test_opcheck() -> None:
    x, y = logits_of((6, 10, 501), torch.float32)
    ids, logps = lists_of(x, 7)
    leaf = x.requires_grad_()
    torch.library.opcheck(ops.token_scores, (leaf, y, 3, 0.9, IGNORE))
    torch.library.opcheck(ops.token_scores, (leaf, None, 0, 0.9, IGNORE))
    torch.library.opcheck(ops.distillation, (leaf, ids, logps, None, 2, False, 0.5, 1.1, IGNORE))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_compile_fullgraph(dtype: torch.dtype) -> None:
    torch._dynamo.reset()
    x, y = logits_of((6, 10, 501), dtype)
    ids, logps = lists_of(x, 7)
    weight = logps[..., 0] > -2

    def scores(x):
        got = ti.token_scores(x, y, top=3, temperature=0.9)
        return got.logps.sum() - 0.1 * got.entropy.sum(), got.top_ids, got.top_logps

    def entropy(x):
        return (ti.token_scores(x).entropy.sum(),)

    def distill(x):
        got = ti.distillation_loss(x, ids, logps, kind="jensen", weight=weight)
        return got.loss * 3, got.divergence

    for f in (scores, entropy, distill):
        a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
        eager, compiled = f(a), torch.compile(f, fullgraph=True)(b)
        eager[0].backward()
        compiled[0].backward()
        close(compiled[0], eager[0], 0.0, 16 * 2.0**-24)  # the sums are torch's, fused
        for u, v in zip(eager[1:], compiled[1:]):
            assert torch.equal(u, v)
        assert torch.equal(a.grad, b.grad)


@pytest.mark.gpu
def test_operators_refuse_what_they_would_misread() -> None:
    x, y = logits_of((6, 10, 501), torch.float32)
    ids, logps = lists_of(x, 7)
    one = torch.ones((), device="cuda")
    stats = ops.token_scores(x, y, 1, 1.0, IGNORE)[4]
    kept = ops.distillation(x, ids, logps, None, 0, False, 0.5, 1.0, IGNORE)[2]
    lead = logps[..., 0].contiguous()
    good = {ops.token_scores: [x, y, 3, 0.9, IGNORE],
            ops.token_scores_grad: [x, y, 0.9, stats, lead, lead],
            ops.distillation: [x, ids, logps, lead.exp(), 0, False, 0.5, 1.0, IGNORE],
            ops.distillation_grad: [x, ids, 1.0, IGNORE, kept, one]}

    def other_type(t):
        if t.dtype == torch.float32:
            return t.int() if t is x else t.half()
        return t.float()

    for op, args in good.items():
        op(*args)
        for i, a in enumerate(args):
            if not isinstance(a, torch.Tensor):
                continue
            bad = [(other_type(a), TypeError), (a.cpu(), (ValueError, RuntimeError))]
            if a is not x and a is not ids:
                bad.append((torch.cat([a, a], -1) if a.dim() else torch.ones(2, device="cuda"), ValueError))
            for b, error in bad:
                with pytest.raises(error):
                    op(*args[:i], b, *args[i + 1:])
        for z in (x[..., :0], x[0], x[0, 0, 0]):
            with pytest.raises(ValueError):
                op(z, *args[1:])
    for bad, match in ([x, y, 129, 1.0, IGNORE], "top"), ([x, y, -1, 1.0, IGNORE], "top|negative"), \
            ([x, y, 3, 0.0, IGNORE], "temperature"):
        with pytest.raises(RuntimeError, match=match):
            ops.token_scores(*bad)
    for bad, match in (([ids[..., :0], logps[..., :0], None, 0, False, 0.5, 1.0], "entries"),
                       ([ids, logps, None, 3, False, 0.5, 1.0], "kind"),
                       ([ids, logps, None, 1, True, 0.5, 1.0], "rest"),
                       ([ids, logps, None, 2, False, 1.0, 1.0], "mix"),
                       ([ids, logps, None, 0, False, 0.5, -1.0], "temperature")):
        with pytest.raises(RuntimeError, match=match):
            ops.distillation(x, *bad, IGNORE)


# ---------------------------------------------------------------------------------------------
# Refusals


def test_refusals_without_a_gpu() -> None:
    x, y = torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64)
    ids, logps = torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2)
    with pytest.raises(TypeError, match="torch.Tensor"):
        ti.token_scores([1.0])  # type: ignore[arg-type]
    with pytest.raises(TypeError, match="float16"):
        ti.token_scores(y[:, None])
    with pytest.raises(ValueError, match="at least one element"):
        ti.token_scores(x[:, :0])
    for top in (-1, 6, 129, 2**40):
        with pytest.raises(ValueError, match="top"):
            ti.token_scores(x, y, top=top)
    for top in (1.0, True, None):
        with pytest.raises(TypeError, match="top"):
            ti.token_scores(x, y, top=top)  # type: ignore[arg-type]
    for t in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            ti.token_scores(x, y, temperature=t)
        with pytest.raises(ValueError, match="temperature"):
            ti.distillation_loss(x, ids, logps, temperature=t)
    with pytest.raises(TypeError, match="integer"):
        ti.token_scores(x, x[:, 0])
    with pytest.raises(ValueError, match="do not fit"):
        ti.token_scores(x, y[:2])
    for targets in (y, None):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            ti.token_scores(x, targets, top=2)
    with pytest.raises(ValueError, match="kind"):
        ti.distillation_loss(x, ids, logps, kind="other")
    with pytest.raises(ValueError, match="rest must be"):
        ti.distillation_loss(x, ids, logps, rest="other")
    with pytest.raises(ValueError, match="reverse"):
        ti.distillation_loss(x, ids, logps, kind="reverse", rest="drop")
    for mix in (0.0, 1.0, -1.0, math.nan):
        with pytest.raises(ValueError, match="mix"):
            ti.distillation_loss(x, ids, logps, kind="jensen", mix=mix)
    with pytest.raises(TypeError, match="torch.Tensors"):
        ti.distillation_loss(x, ids, None)  # type: ignore[arg-type]
    with pytest.raises(TypeError, match="integer"):
        ti.distillation_loss(x, logps, logps)
    with pytest.raises(TypeError, match="floating-point"):
        ti.distillation_loss(x, ids, ids)
    for bad in (ids[:2], ids[0], ids[None]):
        with pytest.raises(ValueError, match="do not fit"):
            ti.distillation_loss(x, bad, logps)
    for n in (0, 129):
        with pytest.raises(ValueError, match="entries"):
            ti.distillation_loss(x, torch.zeros(3, n, dtype=torch.int64), torch.zeros(3, n))
    with pytest.raises(ValueError, match="shaped like teacher_ids"):
        ti.distillation_loss(x, ids, logps[:, :1])
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ti.distillation_loss(x, ids, logps)


@pytest.mark.gpu
def test_refusals() -> None:
    x, y = logits_of((3, 50), torch.float32)
    ids, logps = lists_of(x, 4)
    with pytest.raises(ValueError, match="device"):
        ti.token_scores(x, y.cpu())
    for bad in ((ids.cpu(), logps), (ids, logps.cpu())):
        with pytest.raises(ValueError, match="device"):
            ti.distillation_loss(x, *bad)
    with pytest.raises(TypeError, match="weight"):
        ti.distillation_loss(x, ids, logps, weight=1.0)  # type: ignore[arg-type]
    with pytest.raises(ValueError, match="weight"):
        ti.distillation_loss(x, ids, logps, weight=torch.ones(2, device="cuda"))
    with pytest.raises(ValueError, match="teacher_logps is a constant"):
        ti.distillation_loss(x, ids, logps.clone().requires_grad_())
    with pytest.raises(ValueError, match="weight is a constant"):
        ti.distillation_loss(x, ids, logps, weight=torch.ones(3, device="cuda", requires_grad=True))
    leaf = x.requires_grad_()
    for f in (lambda: ti.token_scores(leaf, y).entropy.sum(), lambda: ti.distillation_loss(leaf, ids, logps).loss):
        (g,) = torch.autograd.grad(f(), leaf, create_graph=True)
        with pytest.raises(RuntimeError):  # differentiable once
            g.sum().backward()


@pytest.mark.gpu
def test_forward_mode_is_refused() -> None:
    fw = torch.autograd.forward_ad
    x, y = logits_of((4, 33), torch.float32)
    ids, logps = lists_of(x, 4)
    with fw.dual_level():
        def dual(t):
            return fw.make_dual(t.clone(), torch.ones_like(t))

        for call in (lambda: ti.token_scores(dual(x), y), lambda: ti.token_scores(dual(x)),
                     lambda: ti.distillation_loss(dual(x), ids, logps),
                     lambda: ti.distillation_loss(x, ids, dual(logps)),
                     lambda: ti.distillation_loss(x, ids, logps, weight=dual(logps[:, 0].contiguous())),
                     lambda: ops.token_scores(dual(x), y, 1, 1.0, IGNORE),
                     lambda: ops.distillation(dual(x), ids, logps, None, 0, False, 0.5, 1.0, IGNORE)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_abi_refusals() -> None:
    import ctypes

    so, p, none = _ext.lib(), ctypes.c_void_p(16), None
    rows = _ext.Rows(16, 4, 4, 0, 8, 8)

    def scores(dtype=2, rows=rows, targets=p, temperature=1.0, top=2, logps=p, entropy=p, tops=p, ids=p):
        return so.tiso_scores(dtype, rows, targets, IGNORE, temperature, top, logps, entropy, tops, ids,
                              none, none)

    for bad in (dict(dtype=9), dict(rows=none), dict(temperature=0.0), dict(top=-1), dict(top=9),
                dict(top=129), dict(logps=none), dict(entropy=none), dict(tops=none), dict(ids=none),
                dict(rows=_ext.Rows(16, 4, 4, 0, -8, 8)), dict(rows=_ext.Rows(17, 4, 4, 0, 8, 8))):
        assert scores(**bad) == 1, bad
    assert scores(rows=_ext.Rows(none, 0, 1, 0, 8, 8), logps=none, entropy=none, tops=none, ids=none) == 0
    huge = _ext.Rows(16, 1, 1, 0, 1 << 28, 1 << 28)
    assert scores(dtype=1, rows=huge, top=5) == 1 and b"vocabulary" in so.tiso_last_error()
    assert so.tiso_scores_grad(2, rows, p, 1.0, none, p, p, p, none) == 1
    assert so.tiso_scores_grad(2, rows, none, 1.0, p, p, p, p, none) == 1
    assert b"targets" in so.tiso_last_error()
    assert so.tiso_scores_grad(2, rows, p, 1.0, p, p, p, ctypes.c_void_p(18), none) == 1
    size = ctypes.c_size_t()
    assert so.tiso_distill_workspace_size(2, 4, ctypes.byref(size)) == 0 and size.value > 0
    assert so.tiso_distill_workspace_size(9, 4, ctypes.byref(size)) == 1
    assert so.tiso_distill_workspace_size(2, 4, ctypes.byref(size)) == 0

    def distill(args=(16, 16, none, 3, 0, 0, 0, 0.5, 1.0), temperature=1.0, out=p, divergence=p, kept=p,
                workspace=p, size=size.value):
        return so.tiso_distill(2, rows, IGNORE, temperature,
                               none if args is none else _ext.DistillArgs(*args), divergence, kept, p, p,
                               out, none, workspace, size, none)

    for bad in (dict(args=none), dict(temperature=0.0), dict(out=none), dict(divergence=none), dict(kept=none),
                dict(args=(none, 16, none, 3, 0, 0, 0, 0.5, 1.0)), dict(args=(16, none, none, 3, 0, 0, 0, 0.5, 1.0)),
                dict(args=(16, 16, none, 0, 0, 0, 0, 0.5, 1.0)), dict(args=(16, 16, none, 129, 0, 0, 0, 0.5, 1.0)),
                dict(args=(16, 16, none, 3, 0, 3, 0, 0.5, 1.0)), dict(args=(16, 16, none, 3, 0, 1, 1, 0.5, 1.0)),
                dict(args=(16, 16, none, 3, 0, 2, 0, 1.0, 1.0))):
        assert distill(**bad) == 1, bad
    assert distill(workspace=none) == 2 and distill(size=size.value - 1) == 2
    assert so.tiso_distill_grad(2, rows, IGNORE, 1.0, p, 3, p, p, none, 1.0, p, p, none) == 1
    assert so.tiso_distill_grad(2, rows, IGNORE, 1.0, p, 0, p, p, p, 1.0, p, p, none) == 1
