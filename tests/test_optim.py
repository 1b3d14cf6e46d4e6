"""The AdamW step over many tensors, 32-bit and 8-bit states: against its formula in float64, and
bit for bit against the same formula in float32 written one torch operation at a time.

Tolerances in float64: a step is a dozen float32 operations on numbers of one sign or on a sum whose
parts are bounded by the larger, so m, v and the update are within 2^-20 of their largest part. A
random rounding to 8 bits differs from float64's only where the float32 error moves a number
across the threshold: for an error of 4 units in the last place and at most 16 units of e4m3 that
is a chance of 2^-24 4 16 = 4e-6 an element, and then by one unit.
"""

from __future__ import annotations

import copy
import math

import pytest
import torch

import torchisotonic_b200 as ti
from torchisotonic_b200 import _ext

BLOCK = 256
WORD = 0xFFFFFFFF
SETTINGS = {"lr": 1e-2, "betas": (0.9, 0.99), "eps": 1e-6, "weight_decay": 0.1}


def mix(x):
    x = ((x ^ (x >> 16)) * 0x45D9F3B5) & WORD
    x = ((x ^ (x >> 15)) * 0x2C1B3C6D) & WORD
    return x ^ (x >> 16)


def words(n, seed, step, tensor):
    """The 32 random bits of every element of a tensor."""
    key = int(mix((mix((tensor + 0x9E3779B1 * step) & WORD) + seed) & WORD))
    at = torch.arange(n, device="cuda")
    return mix(((at & WORD) * 0x9E3779B1 + mix(key ^ (at >> 32))) & WORD)


def blocks_of(x):
    """[blocks, 256], the last one filled with zeros."""
    pad = -x.numel() % BLOCK
    return torch.cat([x.reshape(-1), x.new_zeros(pad)]).view(-1, BLOCK)


def two_to(power, dtype):
    return ((power.int() + 127) << 23).view(torch.float32).to(dtype)


def to_e4m3(x, bits, square):
    """x as e4m3 values and scales, rounded by 16 random bits an element; in x's precision."""
    n = x.numel()
    y, r = blocks_of(x), blocks_of(bits)
    fine = torch.isfinite(y)
    size = torch.where(fine, y.abs(), torch.zeros_like(y))
    top = size.amax(1, keepdim=True)
    some = top >= 1e-30
    part, power = torch.frexp(top)
    power = torch.where(part > 0.875, power - 8, power - 9)
    zero = torch.zeros_like(top)
    a = size * torch.where(some, two_to(-power, x.dtype), zero)
    unit = two_to(torch.frexp(a)[1].clamp(min=-5) - 4, x.dtype)
    low = (a / unit).floor() * unit
    u = r.to(x.dtype) * 2.0**-16 * unit
    up = (a - low) * (a + low) > u * (2.0 * low + unit) if square else a - low > u
    q = torch.where(up, low + unit, low).clamp(max=448.0)
    if square:
        q = torch.where(a > 0, q.clamp(min=2.0**-9), q)
    q = torch.where(fine, torch.copysign(q, y), torch.full_like(y, math.nan))
    return q.view(-1)[:n].view(x.shape), torch.where(some, two_to(power, x.dtype), zero)[:, 0]


def from_e4m3(q, scale):
    n = q.numel()
    return (blocks_of(q.reshape(-1)) * scale[:, None]).view(-1)[:n].view(q.shape)


def plain_step(p, g, m, v, step, tensor, seed, dtype, scales, *, lr, betas, eps, weight_decay):
    """(p, m, v[, m_scale, v_scale]) after the step, in ``dtype``; 8-bit states as values."""
    b1, b2 = betas
    p, g, m, v = (t.to(torch.float32).to(dtype) for t in (p, g, m, v))
    if scales is not None:
        m = from_e4m3(m, scales[0].to(dtype))
        v = from_e4m3(v, scales[1].to(dtype))
        v = v * v
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    root = v.sqrt()
    update = m / (root * (1 / math.sqrt(1 - b2**step)) + eps)
    p = p * (1 - lr * weight_decay) - update * (lr / (1 - b1**step))
    if scales is None:
        return p, m, v
    r = words(p.numel(), seed, step, tensor).view(p.shape)
    mq, ms = to_e4m3(m, r & 0xFFFF, False)
    vq, vs = to_e4m3(root, r >> 16, True)
    return p, mq, vq, ms, vs


def tensors(shapes, dtype, grad_dtype, bits, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape):
        return torch.randn(shape, generator=gen, device="cuda")

    params = [normal(s).to(dtype) for s in shapes]
    grads = [(normal(s) * 0.1 * torch.exp(2 * normal(s))).to(grad_dtype) for s in shapes]
    ms, vs, scales = [], [], ([], [])
    for k, s in enumerate(shapes):
        m, root = normal(s) * 0.05, normal(s).abs() * 0.1 + 0.01
        if bits == 32:
            ms.append(m)
            vs.append(root.square())
        else:
            r = words(m.numel(), 3, 1, k).view(m.shape)
            for x, keep, codes, part, where in ((m, False, ms, r & 0xFFFF, 0), (root, True, vs, r >> 16, 1)):
                q, scale = to_e4m3(x, part, keep)
                codes.append(q.to(torch.float8_e4m3fn))
                scales[where].append(scale)
    return params, grads, ms, vs, (scales if bits == 8 else None)


def check_step(shapes, dtype, grad_dtype, bits, step=7, seed=11, offset=0):
    params, grads, ms, vs, scales = tensors(shapes, dtype, grad_dtype, bits)
    if offset:  # views that start off every alignment
        def shift(x):
            base = torch.zeros(x.numel() + offset, dtype=torch.uint8 if x.dtype.itemsize == 1 else x.dtype,
                               device="cuda").view(x.dtype)
            base.view(torch.uint8)[offset * x.element_size():] = x.reshape(-1).view(torch.uint8)
            return base[offset:].view(x.shape)

        params, grads, ms, vs = ([shift(t) for t in x] for x in (params, grads, ms, vs))
    wants = {}
    for kind in (torch.float32, torch.float64):
        wants[kind] = [plain_step(p, g, m, v, step, k, seed, kind,
                                  None if scales is None else (scales[0][k], scales[1][k]), **SETTINGS)
                       for k, (p, g, m, v) in enumerate(zip(params, grads, ms, vs))]
    ti.adamw_step(params, grads, ms, vs, step=step, seed=seed, scales=scales, **SETTINGS)
    flips = total = 0
    for k, (same, wide) in enumerate(zip(wants[torch.float32], wants[torch.float64])):
        got = [params[k], ms[k], vs[k]] + ([] if scales is None else [scales[0][k], scales[1][k]])
        # bit for bit, every operation rounded once
        for x, y in zip(got, same):
            assert torch.equal(x.float(), y.to(x.dtype).float())
        half = {torch.float32: 0.0, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}[dtype]
        torch.testing.assert_close(got[0].double(), wide[0], atol=2.0**-20 * 10, rtol=half * 1.01)
        if scales is None:
            torch.testing.assert_close(got[1].double(), wide[1], atol=2.0**-20, rtol=2.0**-20)
            torch.testing.assert_close(got[2].double(), wide[2], atol=0, rtol=2.0**-20)
            continue
        for x, y, sx, sy in ((got[1], wide[1], got[3], wide[3]), (got[2], wide[2], got[4], wide[4])):
            torch.testing.assert_close(sx.double(), sy, atol=0, rtol=2.0**-20)
            d = (x.float().double() - y).abs()
            assert (d <= torch.maximum(y.abs() / 8, torch.full_like(y, 2.0**-9))).all()
            flips += int((d != 0).sum())
            total += d.numel()
    assert flips <= 5 + 2e-5 * total


SHAPES = [(1,), (2,), (0,), (255,), (256,), (257,), (7, 11), (64, 100), (3, 5, 17), (4099,), (),
          (100_003,)]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,grad_dtype", [
    (torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
    (torch.float16, torch.float16), (torch.bfloat16, torch.float32),
    (torch.float16, torch.float32)])
def test_step(dtype, grad_dtype, bits: int) -> None:
    check_step(SHAPES, dtype, grad_dtype, bits)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [1, 2, 4])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step_off_alignment(dtype, offset: int, bits: int) -> None:
    check_step([(300,), (256,), (7, 101), (5000,)], dtype, dtype, bits, offset=offset)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [47, 49, 479, 480, 481, 1100])
def test_many_tensors(count: int, bits: int) -> None:
    shapes = [((37 * k) % 1500 + 1,) for k in range(count)]
    check_step(shapes, torch.float32, torch.float32, bits, step=1)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_mixed_types_in_one_call(bits: int) -> None:
    a = tensors([(300,), (5,)], torch.float32, torch.float32, bits)
    b = tensors([(70, 9)], torch.bfloat16, torch.bfloat16, bits, seed=1)
    c = tensors([(2000,)], torch.bfloat16, torch.float32, bits, seed=2)
    joined = [x + y + z for x, y, z in zip(a[:4], b[:4], c[:4])]
    scales = None if bits == 32 else tuple(x + y + z for x, y, z in zip(a[4], b[4], c[4]))
    want = [plain_step(*(x[k] for x in joined), 3, k, 5, torch.float32,
                       None if scales is None else (scales[0][k], scales[1][k]), **SETTINGS)
            for k in range(4)]
    ti.adamw_step(*joined, step=3, seed=5, scales=scales, **SETTINGS)
    for k in range(4):
        for x, y in zip((joined[0][k], joined[2][k], joined[3][k]), want[k]):
            assert torch.equal(x.float(), y.to(x.dtype).float())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_zeros_and_numbers_that_are_not_finite(bits: int) -> None:
    params, grads, ms, vs, scales = tensors([(1000,)], torch.float32, torch.float32, bits)
    for x in (grads, ms, vs):
        x[0].view(torch.uint8)[:1024 * x[0].element_size() // 2] = 0
    grads[0][600] = math.inf
    grads[0][700] = math.nan
    before = params[0].clone()
    ti.adamw_step(params, grads, ms, vs, step=2, scales=scales, lr=0.5, weight_decay=0.0)
    assert torch.equal(params[0][:256], before[:256])  # no gradient, no moments: no change
    bad = torch.zeros(1000, dtype=torch.bool, device="cuda")
    bad[[600, 700]] = True
    assert torch.equal(params[0].isnan(), bad)
    if bits == 8:  # their blocks' scales, and so their neighbours, are as without them
        for x, s in zip((ms, vs), scales):
            assert torch.equal(x[0].float().isnan(), bad) and torch.isfinite(s[0]).all()


@pytest.mark.gpu
def test_second_moment_follows_in_eight_bits() -> None:
    # The gradient's size falls by 30: the mean square, held in 8 bits, follows the float32 one
    # down, where rounding to nearest would leave it at the top. A step of rounding has the
    # variance (unit of v) |change of v| <= (v / 4) (0.01 v), 50 steps are remembered: a spread of
    # 0.36 v at most, so the mean over 4096 elements is within 0.03 = 5 standard errors.
    n = 4096
    gen = torch.Generator(device="cuda").manual_seed(0)
    p = [torch.zeros(n, device="cuda")]
    v32, m32 = [torch.zeros(n, device="cuda")], [torch.zeros(n, device="cuda")]
    m8, v8 = ([torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)] for _ in range(2))
    scales = ([torch.zeros(n // BLOCK, device="cuda")], [torch.zeros(n // BLOCK, device="cuda")])
    q = [torch.zeros(n, device="cuda")]
    for step in range(1, 1501):
        g = [torch.randn(n, generator=gen, device="cuda") * (1.0 if step <= 200 else 1 / 30)]
        ti.adamw_step(p, g, m32, v32, step=step, betas=(0.9, 0.99))
        ti.adamw_step(q, g, m8, v8, step=step, betas=(0.9, 0.99), scales=scales, seed=1)
    held = from_e4m3(v8[0].float(), scales[1][0])
    assert float(held.square().mean() / v32[0].mean()) == pytest.approx(1.0, abs=0.03)
    assert float((held / v32[0].sqrt()).max()) < 3.0


@pytest.mark.gpu
def test_random_rounding_has_no_bias() -> None:
    # one number in many elements: the mean of its roundings is m, that of their squares v, within 5
    # standard errors of a choice between two neighbours (spread at most half their distance)
    n = 1 << 20
    x = torch.full((n,), 0.3, device="cuda")
    x[::BLOCK] = 1.0  # the blocks' largest
    m, v = ([torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)] for _ in range(2))
    scales = tuple([torch.zeros(n // BLOCK, device="cuda")] for _ in range(2))
    ti.adamw_step([torch.zeros(n, device="cuda")], [x], m, v, step=1, betas=(0.5, 0.5), scales=scales,
                  seed=9)
    for codes, scale, want, power in ((m, scales[0], 0.15, 1), (v, scales[1], 0.5 * 0.3**2, 2)):
        got = from_e4m3(codes[0].float(), scale[0]).view(-1, BLOCK)[:, 1:].double() ** power
        low, high = float(got.min()), float(got.max())
        assert got.unique().numel() == 2 and low < want < high
        off = 5 * 0.5 * (high - low) / math.sqrt(got.numel()) + 2e-5 * (high - low)
        assert float(got.mean()) == pytest.approx(want, abs=off)


# ---------------------------------------------------------------------------------------------
# The optimizer class


def model(seed=0, dtype=torch.float32):
    torch.manual_seed(seed)
    net = torch.nn.Sequential(torch.nn.Linear(20, 50), torch.nn.Tanh(), torch.nn.Linear(50, 3))
    return net.to(device="cuda", dtype=dtype)


def train(net, opt, steps, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = next(net.parameters()).dtype
    for _ in range(steps):
        x = torch.randn(16, 20, generator=gen, device="cuda").to(dtype)
        opt.zero_grad()
        (net(x).float() - x[:, :3].float()).square().mean().backward()
        opt.step()


@pytest.mark.gpu
def test_optimizer_matches_torch() -> None:
    # 20 steps of two float32 programs of one formula that round differently: each step's update
    # is within 2^-18 of lr; they drift by no more than 20 steps of a hundred times that
    ours, theirs = model(), model()
    a = ti.AdamW(ours.parameters(), lr=1e-3, weight_decay=0.1)
    b = torch.optim.AdamW(theirs.parameters(), lr=1e-3, weight_decay=0.1, foreach=False)
    train(ours, a, 20)
    train(theirs, b, 20)
    for p, q in zip(ours.parameters(), theirs.parameters()):
        torch.testing.assert_close(p, q, atol=20 * 100 * 1e-3 * 2.0**-18, rtol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_optimizer_resumes_exactly(bits: int, dtype: torch.dtype) -> None:
    net = model(dtype=dtype)
    opt = ti.AdamW(net.parameters(), lr=1e-2, state_bits=bits, seed=4)
    train(net, opt, 5)
    saved, weights = copy.deepcopy(opt.state_dict()), copy.deepcopy(net.state_dict())
    train(net, opt, 5, seed=1)
    again = model(seed=9, dtype=dtype)
    again.load_state_dict(weights)
    opt2 = ti.AdamW(again.parameters(), lr=1.0, state_bits=bits)
    opt2.load_state_dict(saved)
    for s in opt2.state.values():
        assert s["exp_avg"].dtype == (torch.float32 if bits == 32 else torch.float8_e4m3fn)
    train(again, opt2, 5, seed=1)
    for p, q in zip(net.parameters(), again.parameters()):
        assert torch.equal(p, q)


@pytest.mark.gpu
def test_optimizer_groups_and_missing_gradients() -> None:
    a = torch.nn.Parameter(torch.ones(300, device="cuda"))
    b = torch.nn.Parameter(torch.ones(10, device="cuda", dtype=torch.bfloat16))
    c = torch.nn.Parameter(torch.ones(4, 4, device="cuda"))
    opt = ti.AdamW([{"params": [a, c], "lr": 0.1}, {"params": [b], "weight_decay": 0.0}], lr=0.01)
    a.grad = torch.ones_like(a)
    opt.step()
    assert float(a[0]) == pytest.approx(1 - 0.1 * 0.01 - 0.1, abs=1e-6) and (c == 1).all() and (b == 1).all()
    c.grad = torch.ones(4, 4, device="cuda").t()
    b.grad = torch.ones_like(b)
    opt.step(lambda: None)
    assert opt.state[a]["step"] == 2 and opt.state[c]["step"] == 1
    assert float(c[0, 0]) == pytest.approx(1 - 0.1 * 0.01 - 0.1, abs=1e-6)
    assert (b < 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_parameters_in_other_layouts(bits: int) -> None:
    # stepped as their contiguous copies would be, bit for bit; what lies between is not touched
    torch.manual_seed(0)
    held = torch.randn(40, 1000, device="cuda")
    before = held.clone()
    params = [held.t()[:, :17], held[20:, 1::3], torch.randn(3, 5, device="cuda").expand(1, 3, 5)]
    params = [p.detach().requires_grad_() for p in params]
    copies = [p.detach().contiguous().clone().requires_grad_() for p in params]
    a, b = (ti.AdamW(ps, lr=0.1, state_bits=bits) for ps in (params, copies))
    for _ in range(3):
        for p, c in zip(params, copies):
            c.grad = torch.randn_like(c)
            p.grad = c.grad.clone()
        a.step()
        b.step()
    for p, c in zip(params, copies):
        assert torch.equal(p, c)
    assert torch.equal(held[17:20], before[17:20])
    assert torch.equal(held[20:, ::3], before[20:, ::3])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_optimizer_takes_over_a_state_of_torch(dtype: torch.dtype) -> None:
    p = torch.randn(300, device="cuda", dtype=dtype).requires_grad_()
    theirs = torch.optim.AdamW([p], lr=0.01)
    for _ in range(3):
        p.grad = torch.randn_like(p)
        theirs.step()
    ours = ti.AdamW([p], lr=0.5)
    ours.load_state_dict(theirs.state_dict())
    state, was = ours.state[p], theirs.state[p]
    assert state["step"] == 3 and ours.param_groups[0]["lr"] == 0.01
    for name in ("exp_avg", "exp_avg_sq"):
        assert state[name].dtype == torch.float32
        assert torch.equal(state[name], was[name].float())
    want = [p.detach().clone()], [state["exp_avg"].clone()], [state["exp_avg_sq"].clone()]
    p.grad = torch.randn_like(p)
    ti.adamw_step(want[0], [p.grad], want[1], want[2], step=4, lr=0.01)
    ours.step()
    assert torch.equal(p, want[0][0])
    bad = theirs.state_dict()
    bad["param_groups"][0]["amsgrad"] = True
    with pytest.raises(ValueError, match="amsgrad"):
        ours.load_state_dict(bad)


@pytest.mark.gpu
def test_a_step_counts_as_a_change_in_place() -> None:
    p = torch.nn.Parameter(torch.ones(5, device="cuda"))
    q = (p * p).sum()  # keeps p for its gradient
    version = p._version
    ti.adamw_step([p], [torch.ones_like(p)], [torch.zeros_like(p)], [torch.zeros_like(p)], step=1)
    assert p._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        q.backward()


@pytest.mark.gpu
def test_step_on_another_stream() -> None:
    a = tensors([(5000,)], torch.float32, torch.float32, 32)
    b = copy.deepcopy(a)
    torch.cuda.synchronize()
    ti.adamw_step(*a[:4], step=1)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ti.adamw_step(*b[:4], step=1)
    stream.synchronize()
    assert torch.equal(a[0][0], b[0][0])


@pytest.mark.gpu
def test_no_two_parameters_are_rounded_alike() -> None:
    # equal parameters with equal gradients, a group each: other random bits, so of 4096 numbers
    # between two neighbours many go the other way. A parameter's own do not depend on whether
    # another one has a gradient.
    grad = torch.randn(4096, generator=torch.Generator().manual_seed(0)).cuda()

    def codes(groups, without=()):
        params = [torch.nn.Parameter(torch.zeros(4096, device="cuda")) for _ in range(3)]
        opt = ti.AdamW([{"params": [params[k] for k in g]} for g in groups], state_bits=8, seed=3)
        for k, p in enumerate(params):
            p.grad = None if k in without else grad.clone()
        opt.step()
        return {k: opt.state[p]["exp_avg"].view(torch.uint8).clone() for k, p in enumerate(params)
                if k not in without}

    together = codes([[0, 1, 2]])
    apart = codes([[0], [1], [2]])
    for a, b in ((0, 1), (0, 2), (1, 2)):
        assert int((apart[a] != apart[b]).sum()) > 500
    for k in range(3):  # the place over all groups counts
        assert torch.equal(apart[k], together[k])
    for groups in ([[0, 1, 2]], [[0], [1, 2]]):
        some = codes(groups, without=(0, 1))
        assert torch.equal(some[2], together[2])


@pytest.mark.gpu
def test_indices_enter_the_rounding() -> None:
    params, grads, ms, vs, scales = tensors([(300,), (1000,)], torch.float32, torch.float32, 8)
    want = [plain_step(params[k], grads[k], ms[k], vs[k], 3, place, 5, torch.float32,
                       (scales[0][k], scales[1][k]), **SETTINGS) for k, place in enumerate((9, 2))]
    ti.adamw_step(params, grads, ms, vs, step=3, seed=5, scales=scales, indices=[9, 2], **SETTINGS)
    for k in range(2):
        for x, y in zip((params[k], ms[k], vs[k]), want[k]):
            assert torch.equal(x.float(), y.to(x.dtype).float())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_capture_of_a_step_is_refused(bits: int) -> None:
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    opt = ti.AdamW([p], lr=0.1, weight_decay=0.0, state_bits=bits)
    p.grad = torch.ones_like(p)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured in a CUDA graph"):
        with torch.cuda.graph(graph):
            opt.step()
    assert not opt.state and (p == 1).all()
    opt.step()  # the next one is the first
    assert opt.state[p]["step"] == 1
    torch.testing.assert_close(p.detach(), torch.full_like(p, 0.9), rtol=1e-5, atol=0)


def test_capture_of_a_step_is_refused_without_a_gpu(monkeypatch) -> None:
    p = torch.nn.Parameter(torch.ones(3))
    p.grad = torch.ones(3)
    opt = ti.AdamW([p])
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captured in a CUDA graph"):
        opt.step(lambda: pytest.fail("nothing of a refused step runs"))
    assert not opt.state


# ---------------------------------------------------------------------------------------------
# Refusals


def test_refusals_without_a_gpu() -> None:
    x = [torch.zeros(4)]
    for bad in ({"step": 0}, {"betas": (1.0, 0.9)}, {"lr": -1.0}, {"eps": math.nan}, {"weight_decay": -1.0}):
        with pytest.raises(ValueError):
            ti.adamw_step(x, x, x, x, **{"step": 1, **bad})
    with pytest.raises(ValueError, match="one length"):
        ti.adamw_step(x, x, x, [], step=1)
    with pytest.raises(TypeError, match="torch.Tensors"):
        ti.adamw_step(x, [None], x, x, step=1)  # type: ignore[list-item]
    with pytest.raises(ValueError, match="contiguous"):
        ti.adamw_step(x, [torch.zeros(8)[::2]], x, x, step=1)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ti.adamw_step(x, x, x, x, step=1)
    ti.adamw_step([], [], [], [], step=1)
    with pytest.raises(ValueError, match="state_bits"):
        ti.AdamW([torch.nn.Parameter(torch.zeros(3))], state_bits=16)
    with pytest.raises(ValueError, match="lr"):
        ti.AdamW([torch.nn.Parameter(torch.zeros(3))], lr=-1.0)
    with pytest.raises(ValueError, match="betas"):
        ti.AdamW([torch.nn.Parameter(torch.zeros(3))], betas=(0.9, 1.0))


@pytest.mark.gpu
def test_refusals() -> None:
    x, h = [torch.zeros(4, device="cuda")], [torch.zeros(4, device="cuda", dtype=torch.bfloat16)]
    with pytest.raises(ValueError, match="one device"):
        ti.adamw_step(x, x, [torch.zeros(4)], x, step=1)
    with pytest.raises(ValueError, match="shaped like"):
        ti.adamw_step(x, [torch.zeros(5, device="cuda")], x, x, step=1)
    with pytest.raises(TypeError, match="states must be float32"):
        ti.adamw_step(x, x, h, h, step=1)
    with pytest.raises(TypeError, match="grads like"):
        ti.adamw_step(x, h, x, x, step=1)
    d = [torch.zeros(4, device="cuda", dtype=torch.float64)]
    with pytest.raises(TypeError, match="params must be"):
        ti.adamw_step(d, d, x, x, step=1)
    q = [torch.zeros(4, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)]
    s = [torch.zeros(1, device="cuda")]
    with pytest.raises(ValueError, match="scales go with"):
        ti.adamw_step(x, x, q, q, step=1)
    with pytest.raises(ValueError, match="scales go with"):
        ti.adamw_step(x, x, x, x, step=1, scales=(s, s))
    with pytest.raises(ValueError, match="ceil"):
        ti.adamw_step(x, x, q, q, step=1, scales=(s, x))
    with pytest.raises(TypeError, match="one dtype"):
        ti.adamw_step(x, x, q, x, step=1, scales=(s, s))


def test_abi_refusals() -> None:
    import ctypes

    so = _ext.lib()
    table = (ctypes.c_int64 * 8)(16, 16, 16, 16, 0, 0, 4, 0)
    at = ctypes.addressof(table)
    good = _ext.AdamwArgs(1e-3, 0.9, 0.999, 1e-8, 0.01, 1, 0)
    assert so.tiso_adamw(3, 3, 32, 1, at, good, None) == 1
    assert so.tiso_adamw(2, 1, 32, 1, at, good, None) == 1
    assert so.tiso_adamw(2, 2, 16, 1, at, good, None) == 1
    assert so.tiso_adamw(2, 2, 8, 1, at, good, None) == 1  # no scales
    assert so.tiso_adamw(2, 2, 32, -1, at, good, None) == 1
    assert so.tiso_adamw(2, 2, 32, 1, None, good, None) == 1
    assert so.tiso_adamw(2, 2, 32, 1, at, _ext.AdamwArgs(1e-3, 0.9, 0.999, 1e-8, 0.01, 0, 0), None) == 1
    assert b"step" in so.tiso_last_error()
    off = (ctypes.c_int64 * 8)(18, 16, 16, 16, 0, 0, 4, 0)
    assert so.tiso_adamw(2, 2, 32, 1, ctypes.addressof(off), good, None) == 1
    assert b"aligned" in so.tiso_last_error()
    assert so.tiso_adamw(2, 2, 32, 0, None, good, None) == 0
    empty = (ctypes.c_int64 * 8)(0, 0, 0, 0, 0, 0, 0, 0)
    assert so.tiso_adamw(2, 2, 32, 1, ctypes.addressof(empty), good, None) == 0


def test_indices_go_with_params() -> None:
    x = [torch.zeros(4)]
    for bad in ([1, 2], [0, 1, 2]):
        with pytest.raises(ValueError, match="as many as params"):
            ti.adamw_step(x, x, x, x, step=1, indices=bad)
    with pytest.raises(TypeError):
        ti.adamw_step(x, x, x, x, step=1, indices=["a"])  # type: ignore[list-item]
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ti.adamw_step(x, x, x, x, step=1, indices=[5])


def test_a_refused_step_does_not_count() -> None:
    # a caller that catches the error goes on at the step's right number
    p = torch.nn.Parameter(torch.ones(3))
    p.grad = torch.ones(3)
    opt = ti.AdamW([p])
    for _ in range(2):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            opt.step()
        assert opt.state[p]["step"] == 0


@pytest.mark.gpu
def test_a_refused_step_does_not_count_in_its_group_alone() -> None:
    a = torch.nn.Parameter(torch.ones(3, device="cuda"))
    b = torch.nn.Parameter(torch.ones(3, device="cuda", dtype=torch.float64))
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    opt = ti.AdamW([{"params": [a]}, {"params": [b]}], lr=0.1, weight_decay=0.0)
    with pytest.raises(TypeError, match="params must be"):
        opt.step()
    assert opt.state[a]["step"] == 1 and opt.state[b]["step"] == 0
    assert (a < 1).all() and (b == 1).all()


def test_no_indices_for_some_params_are_refused() -> None:
    x = [torch.zeros(4)]
    with pytest.raises(ValueError, match="as many as params"):
        ti.adamw_step(x, x, x, x, step=1, indices=[])
    ti.adamw_step([], [], [], [], step=1, indices=[])
