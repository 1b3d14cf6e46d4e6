"""The language-model operators of this package as a user's program calls them, and in plain torch.

Four operators: token log-probabilities, the preference loss on them, the clipped policy loss straight
from logits, and the AdamW step. ``listed()`` has fixed cases, ``draw()`` more of the same ranges;
``run()`` makes one pass through a case's operator: elementary torch operations in float32 while
``own`` is false, this package's kernels where it is true. ``exact()`` has the definitions in float64.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
IGNORE = -100
BLOCK = 256  # elements that share one scale of an 8-bit optimizer state
WORD = 0xFFFFFFFF


# ---------------------------------------------------------------------------------------------
# Cases


def listed():
    return [
        # the log-probabilities of the tokens just sampled for a few requests: one decoding step
        {"name": "logprobs decode", "op": "logprobs", "batch": 4, "rows": 1, "vocab": 32000,
         "dtype": "bf16", "grad": False, "shift": False, "ignored": 0.0, "temperature": 0.7},
        # a reference model's scores of a batch of answers: forward only
        {"name": "logprobs scoring", "op": "logprobs", "batch": 4, "rows": 1024, "vocab": 131072,
         "dtype": "bf16", "grad": False, "shift": False, "ignored": 0.1, "temperature": 1.0},
        # training on the next token: logits[:, :-1] of an odd vocabulary, the prompt ignored
        {"name": "logprobs training", "op": "logprobs", "batch": 4, "rows": 1023, "vocab": 50021,
         "dtype": "bf16", "grad": True, "shift": True, "ignored": 0.3, "temperature": 1.0},
        # a small model trained in float32 over bytes and a few hundred merges
        {"name": "logprobs small vocabulary", "op": "logprobs", "batch": 16, "rows": 511,
         "vocab": 777, "dtype": "f32", "grad": True, "shift": True, "ignored": 0.0,
         "temperature": 1.0},
        # preference pairs of one micro-batch
        {"name": "preference micro-batch", "op": "preference", "pairs": 4, "longest": 100,
         "kind": "logistic", "reference": True, "masked": 0.4, "average": False,
         "smoothing": 0.0, "margin": 0.0, "beta": 0.1},
        # a batch of ragged answers with their prompts masked, labels smoothed
        {"name": "preference batch", "op": "preference", "pairs": 64, "longest": 2048,
         "kind": "logistic", "reference": True, "masked": 0.4, "average": False,
         "smoothing": 0.1, "margin": 0.0, "beta": 0.1},
        # long answers, averaged over their tokens, without a reference model
        {"name": "preference long answers", "op": "preference", "pairs": 256, "longest": 8191,
         "kind": "hinge", "reference": False, "masked": 0.1, "average": True,
         "smoothing": 0.0, "margin": 0.5, "beta": 2.0},
        # a policy update on a handful of tokens
        {"name": "policy micro-batch", "op": "policy", "rows": 64, "vocab": 32000,
         "dtype": "bf16", "reference": True, "masked": 0.2, "temperature": 1.0},
        # an odd vocabulary in float32, no reference model
        {"name": "policy odd vocabulary", "op": "policy", "rows": 1999, "vocab": 50021,
         "dtype": "f32", "reference": False, "masked": 0.4, "temperature": 0.9},
        # a full batch of a large vocabulary, with the reference's KL term
        {"name": "policy batch", "op": "policy", "rows": 8192, "vocab": 131072,
         "dtype": "bf16", "reference": True, "masked": 0.1, "temperature": 1.0},
        # the update of a small head
        {"name": "adamw head", "op": "adamw", "tensors": 12, "elements": 300_000,
         "dtype": "f32", "bits": 32},
        # a model's update with 8-bit states
        {"name": "adamw 8 bits", "op": "adamw", "tensors": 100, "elements": 250_000_000,
         "dtype": "bf16", "bits": 8},
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _rows_and_vocab(rng, most):
    vocab = _log(rng, 256, 131072)
    return _log(rng, 1, max(1, min(8192, most // vocab))), vocab


def draw(rng):
    op = rng.choice(["logprobs", "preference", "policy", "adamw"])
    if op == "logprobs":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        rows, vocab = _rows_and_vocab(rng, 1 << 28 if dtype == "f32" else 1 << 29)
        batch = rng.choice([1, 2, 4]) if rows >= 8 else 1
        grad = rng.random() < 0.6
        return {"op": op, "batch": batch, "rows": max(1, rows // batch), "vocab": vocab,
                "dtype": dtype, "grad": grad, "shift": grad and rng.random() < 0.5,
                "ignored": rng.choice([0.0, 0.1, 0.5]),
                "temperature": rng.choice([1.0, 1.0, 0.7, 1.5])}
    if op == "preference":
        longest, reference = _log(rng, 8, 8192), rng.random() < 0.7
        return {"op": op, "pairs": _log(rng, 1, min(512, (1 << 22) // (2 * longest))),
                "longest": longest, "kind": rng.choice(["logistic", "hinge", "square"]),
                "reference": reference, "masked": rng.choice([0.0, 0.2, 0.5]),
                "average": not reference or rng.random() < 0.2, "smoothing": rng.choice([0.0, 0.1]),
                "margin": rng.choice([0.0, 0.3]), "beta": rng.choice([0.05, 0.1, 0.5])}
    if op == "policy":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        rows, vocab = _rows_and_vocab(rng, 1 << 29 if dtype == "f32" else 1 << 30)
        return {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype,
                "reference": rng.random() < 0.6, "masked": rng.choice([0.0, 0.2, 0.5]),
                "temperature": rng.choice([1.0, 0.9, 1.2])}
    tensors = _log(rng, 1, 160)
    return {"op": op, "tensors": tensors,
            "elements": _log(rng, max(20_000, 700 * tensors), 200_000_000),
            "dtype": rng.choice(["bf16", "bf16", "f32"]), "bits": rng.choice([8, 32])}


def _sizes(case):
    """The tensors' sizes: a third of them vectors (norms, biases), the rest matrices of sizes that
    differ by up to a factor of ten, odd ones among them."""
    n, total = case["tensors"], case["elements"]
    rng = random.Random("%d of %d" % (n, total))
    vectors = [rng.randint(1, max(2, min(8192, total // (8 * n)))) for _ in range(n // 3)]
    shares = [math.exp(rng.uniform(0.0, math.log(10.0))) for _ in range(n - len(vectors))]
    rest = total - sum(vectors)
    sizes = vectors + [max(1, int(rest * s / sum(shares))) for s in shares]
    rng.shuffle(sizes)
    return sizes


def _lengths(case):
    """Lengths of the chosen and then the rejected answers, 1 to the longest, one of them the longest."""
    rng = random.Random("%d up to %d" % (case["pairs"], case["longest"]))
    got = [rng.randint(1, case["longest"]) for _ in range(2 * case["pairs"])]
    got[rng.randrange(len(got))] = case["longest"]
    return got


def work(case):
    if case["op"] == "logprobs":
        rows, size = case["batch"] * case["rows"], DTYPES[case["dtype"]].itemsize
        logits = rows * case["vocab"] * size * (1 - case["ignored"])
        if not case["grad"]:
            return {"bytes": logits + rows * 12, "flops": rows * case["vocab"] * 4}
        return {"bytes": logits + rows * (case["vocab"] * size + 16),
                "flops": rows * case["vocab"] * 8}
    if case["op"] == "preference":
        tokens = sum(_lengths(case))
        each = 4 + 4 * case["reference"] + (case["masked"] > 0) + 4
        return {"bytes": tokens * each + case["pairs"] * 24, "flops": tokens * 4}
    if case["op"] == "policy":
        rows, size = case["rows"], DTYPES[case["dtype"]].itemsize
        row = case["vocab"] * size
        return {"bytes": rows * (row * (1 - case["masked"]) + row + 28 + 4 * case["reference"]),
                "flops": rows * case["vocab"] * 8}
    n, size = sum(_sizes(case)), DTYPES[case["dtype"]].itemsize
    states = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": n * (3 * size + states), "flops": n * 14}


# ---------------------------------------------------------------------------------------------
# Inputs


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _logits_and_targets(rows, vocab, dtype, temperature, gen):
    """A trained model's logits (a few tokens well above the rest) and tokens sampled from them."""
    logits = torch.empty(rows, vocab, dtype=dtype, device=DEVICE)
    targets = torch.empty(rows, dtype=torch.int64, device=DEVICE)
    step = max(1, (1 << 27) // vocab)
    for at in range(0, rows, step):
        k = min(step, rows - at)
        x = torch.randn(k, vocab, generator=gen, device=DEVICE).mul_(2.0)
        likely = torch.randint(0, vocab, (k, 8), generator=gen, device=DEVICE)
        x.scatter_add_(1, likely, 10.0 + torch.randn(k, 8, generator=gen, device=DEVICE))
        logits[at:at + k] = x
        noise = torch.empty_like(x).exponential_(generator=gen).log_().neg_()  # Gumbel
        targets[at:at + k] = (logits[at:at + k].float() / temperature + noise).argmax(1)
    return logits, targets


def _sampled_logprobs(logits, targets, temperature):
    got = torch.empty(len(targets), dtype=torch.float64, device=DEVICE)
    step = max(1, (1 << 27) // logits.shape[1])
    for at in range(0, len(targets), step):
        z = logits[at:at + step].float() / temperature
        got[at:at + step] = (z.gather(1, targets[at:at + step, None])[:, 0].double()
                             - torch.logsumexp(z, 1).double())
    return got


def prepare(case, seed):
    gen = _generator(seed)
    state = {"case": dict(case)}
    if case["op"] == "logprobs":
        batch, rows, vocab = case["batch"], case["rows"], case["vocab"]
        whole = rows + 1 if case["shift"] else rows
        logits, targets = _logits_and_targets(batch * whole, vocab, DTYPES[case["dtype"]],
                                              case["temperature"], gen)
        targets[torch.rand(batch * whole, generator=gen, device=DEVICE) < case["ignored"]] = IGNORE
        state["logits"] = logits.view(batch, whole, vocab)[:, :rows]
        state["targets"] = targets.view(batch, whole)[:, :rows].contiguous()
        if case["grad"]:
            state["upstream"] = torch.randn(batch, rows, generator=gen, device=DEVICE) - 1.0
        return state
    if case["op"] == "preference":
        lengths = torch.tensor(_lengths(case), dtype=torch.int64, device=DEVICE)
        offsets = torch.zeros(len(lengths) + 1, dtype=torch.int64, device=DEVICE)
        offsets[1:] = lengths.cumsum(0)
        tokens = sum(_lengths(case))
        logps = torch.randn(tokens, generator=gen, device=DEVICE).exp_().mul_(-0.8)
        state.update(logps=logps, offsets=offsets, ref=None, mask=None)
        if case["reference"]:
            state["ref"] = logps + 0.1 * torch.randn(tokens, generator=gen, device=DEVICE)
        if case["masked"]:
            state["mask"] = (torch.rand(tokens, generator=gen, device=DEVICE) >= case["masked"])
        return state
    if case["op"] == "policy":
        rows, t = case["rows"], case["temperature"]
        logits, targets = _logits_and_targets(rows, case["vocab"], DTYPES[case["dtype"]], t, gen)
        lp = _sampled_logprobs(logits, targets, t)
        # the policy has moved a little since it sampled: most ratios are close to 1, a few are
        # clipped. None lies within a thousandth of the clip's edge, where float32 rounding
        # decides which of two gradients, both right, a token gets.
        moved = 0.12 * torch.randn(rows, generator=gen, device=DEVICE, dtype=torch.float64)
        for edge in (math.log(0.8), math.log(1.2)):
            moved = torch.where((moved - edge).abs() < 1e-3, torch.full_like(moved, edge + 2e-3),
                                moved)
        state.update(logits=logits, targets=targets, old=(lp - moved).float(), ref=None,
                     advantages=torch.randn(rows, generator=gen, device=DEVICE) + 0.5,
                     weight=(torch.rand(rows, generator=gen, device=DEVICE)
                             >= case["masked"]).float())
        state["weight"][0] = 1.0
        if case["reference"]:
            state["ref"] = (lp + 0.2 * torch.randn(rows, generator=gen, device=DEVICE,
                                                   dtype=torch.float64)).float()
        return state
    # adamw, some steps into a run: parameters, gradients and states lie in flat buffers, each
    # tensor a view that starts on a multiple of 256 elements (the gaps between them are zero)
    sizes = _sizes(case)
    blocks = [-(-n // BLOCK) for n in sizes]
    total = BLOCK * sum(blocks)
    starts = [BLOCK * sum(blocks[:k]) for k in range(len(blocks))]
    inside = torch.zeros(total, dtype=torch.bool, device=DEVICE)
    for at, n in zip(starts, sizes):
        inside[at:at + n] = True
    dtype = DTYPES[case["dtype"]]

    def normal():
        return torch.randn(total, generator=gen, device=DEVICE).mul_(inside)

    # gradients of unlike sizes, and rows of an embedding that no token has touched yet
    size = torch.exp(2.0 * torch.randn(total // BLOCK, 1, generator=gen, device=DEVICE) - 6.0)
    size *= torch.rand(total // BLOCK, 1, generator=gen, device=DEVICE) > 0.02
    flat = {"param": normal().mul_(0.02).to(dtype),
            "grad": (normal().view(-1, BLOCK) * size).view(-1).to(dtype)}
    m = (normal().view(-1, BLOCK).mul_(0.3) * size).view(-1)
    root = (normal().abs_().add_(0.5).mul_(inside).view(-1, BLOCK) * size).view(-1)
    if case["bits"] == 32:
        flat.update(m=m, v=root.square_())
    else:
        for name, x in (("m", m), ("v", root)):
            x = x.view(-1, BLOCK)
            top = x.abs().amax(1).double().clamp(min=1e-30)
            scale = torch.exp2(torch.ceil(torch.log2(top / 448.0))).float()
            scale *= x.abs().amax(1) > 0
            codes = torch.where(scale[:, None] > 0, x / scale[:, None], torch.zeros_like(x))
            flat[name] = codes.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(-1)
            flat[name + "_scale"] = scale
    state.update(flat=flat, step=100, blocks=blocks, settings={
        "lr": 1e-4, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01})
    for name in ("param", "grad", "m", "v"):
        state[name + "s"] = [flat[name][at:at + n] for at, n in zip(starts, sizes)]
    if case["bits"] == 8:
        state["scales"] = tuple([flat[k][at // BLOCK:at // BLOCK + b]
                                 for at, b in zip(starts, blocks)] for k in ("m_scale", "v_scale"))
    return state


# ---------------------------------------------------------------------------------------------
# One pass


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    import torchisotonic_b200 as ti

    case = state["case"]
    if case["op"] == "logprobs":
        x = state["logits"]
        if not case["grad"]:
            return ti.token_logprobs(x, state["targets"], temperature=case["temperature"])
        x = x.detach().requires_grad_()
        lp = ti.token_logprobs(x, state["targets"], temperature=case["temperature"])
        (gx,) = torch.autograd.grad(lp, x, state["upstream"])
        return {"logps": lp.detach(), "grad": gx}
    if case["op"] == "preference":
        x = state["logps"].detach().requires_grad_()
        loss, rewards = ti.preference_loss(
            x, state["ref"], state["offsets"], beta=case["beta"], kind=case["kind"],
            label_smoothing=case["smoothing"], margin=case["margin"], mask=state["mask"],
            average=case["average"])
        (gx,) = torch.autograd.grad(loss, x)
        return {"loss": loss.detach(), "rewards": rewards, "grad": gx}
    if case["op"] == "policy":
        x = state["logits"].detach().requires_grad_()
        got = ti.policy_loss(x, state["targets"], state["old"], state["advantages"],
                             ref_logps=state["ref"], weight=state["weight"], kl_coef=0.05,
                             temperature=case["temperature"])
        (gx,) = torch.autograd.grad(got.loss, x)
        return {"loss": got.loss.detach(), "logps": got.logps, "kl": got.kl,
                "clipped": got.clip_fraction, "grad": gx}
    state["step"] += 1
    ti.adamw_step(state["params"], state["grads"], state["ms"], state["vs"], step=state["step"],
                  scales=state.get("scales"), seed=7, **state["settings"])
    return {k: x for k, x in state["flat"].items() if k != "grad"}


def _run_plain(state):
    return {"logprobs": _plain_logprobs, "preference": _plain_preference,
            "policy": _plain_policy, "adamw": _plain_adamw}[state["case"]["op"]](state)


def _softmax_parts(x, targets, temperature):
    """(z at the target - log sum exp z, exp(z - max), their sum) of every row."""
    z = x.float() / temperature
    top = z.amax(1, keepdim=True)
    at = z.gather(1, targets[:, None])
    e = (z - top).exp_()
    s = e.sum(1, keepdim=True)
    return (at - top - s.log())[:, 0], e, s


def _plain_logprobs(state):
    case = state["case"]
    x, y = state["logits"], state["targets"].reshape(-1)
    used = y != IGNORE
    y = torch.where(used, y, torch.zeros_like(y))
    lp, e, s = _softmax_parts(x.reshape(-1, x.shape[-1]), y, case["temperature"])
    lp = torch.where(used, lp, torch.zeros_like(lp)).view(x.shape[:-1])
    if not case["grad"]:
        return lp
    g = torch.where(used, state["upstream"].reshape(-1) / case["temperature"], torch.zeros_like(s[:, 0]))
    grad = e.mul_(-g[:, None] / s)
    grad.scatter_add_(1, y[:, None], g[:, None])
    return {"logps": lp, "grad": grad.to(x.dtype).view(x.shape)}


def _plain_preference(state):
    case, x, offsets = state["case"], state["logps"], state["offsets"]
    pairs, beta = case["pairs"], case["beta"]
    lengths = offsets[1:] - offsets[:-1]
    seq = torch.repeat_interleave(torch.arange(2 * pairs, device=x.device), lengths,
                                  output_size=len(x))
    d = x if state["ref"] is None else x - state["ref"]
    used = torch.ones_like(x) if state["mask"] is None else state["mask"].float()
    d = torch.where(used > 0, d, torch.zeros_like(d))
    s = torch.zeros(2 * pairs, device=x.device).index_add_(0, seq, d)
    count = torch.zeros_like(s).index_add_(0, seq, used).clamp_(min=1.0)
    each = 1.0 / count if case["average"] else torch.ones_like(s)
    s = s * each
    margin = beta * (s[:pairs] - s[pairs:]) - case["margin"]
    eps = case["smoothing"]
    if case["kind"] == "logistic":
        # log(1 + exp(-|u|)) + max(u, 0): softplus without overflow
        tail = (-margin.abs()).exp().log1p()
        losses = ((1 - eps) * (tail + (-margin).clamp(min=0)) + eps * (tail + margin.clamp(min=0)))
        slope = 1.0 / (1.0 + (-margin).exp()) - (1 - eps)
    elif case["kind"] == "hinge":
        losses = (1 - margin).clamp(min=0)
        slope = -(margin < 1).float()
    else:
        losses = (margin - 0.5).square() / beta**2
        slope = 2 * (margin - 0.5) / beta**2
    slope = slope * (beta / pairs)
    grad = (torch.cat([slope, -slope]) * each)[seq] * used
    return {"loss": losses.mean(), "rewards": (beta * s).view(2, pairs), "grad": grad}


def _plain_policy(state):
    case, x, y, w = state["case"], state["logits"], state["targets"], state["weight"]
    t, adv = case["temperature"], state["advantages"]
    lp, e, s = _softmax_parts(x, y, t)
    ratio = (lp - state["old"]).exp()
    free, held = ratio * adv, ratio.clamp(1 - 0.2, 1 + 0.2) * adv
    losses = -torch.minimum(free, held)
    slope = torch.where(free <= held, -free, torch.zeros_like(free))
    kl = torch.zeros_like(lp)
    if state["ref"] is not None:
        d = state["ref"] - lp
        kl = torch.expm1(d) - d
        losses = losses + 0.05 * kl
        slope = slope - 0.05 * torch.expm1(d)
    total = w.sum()
    g = slope * w / (total * t)
    grad = e.mul_(-g[:, None] / s)
    grad.scatter_add_(1, y[:, None], g[:, None])
    grad = torch.where(w[:, None] != 0, grad, torch.zeros_like(grad)).to(x.dtype)
    return {"loss": (w * losses).sum() / total, "logps": torch.where(w != 0, lp, torch.zeros_like(lp)),
            "kl": (w * kl).sum() / total, "clipped": (w * (free > held)).sum() / total, "grad": grad}


def _mix(x):
    """A 32-bit multiply-xorshift mix of every value (held in 64-bit integers)."""
    x = ((x ^ (x >> 16)) * 0x45D9F3B5) & WORD
    x = ((x ^ (x >> 15)) * 0x2C1B3C6D) & WORD
    return x ^ (x >> 16)


def _random_words(blocks, seed, step):
    """32 random bits for every element, [blocks, 256]: a mix of the seed, the step, the tensor's
    place in the list and the element's place in the tensor."""
    n = torch.tensor(blocks, device=DEVICE)
    tensor = torch.repeat_interleave(torch.arange(len(blocks), device=DEVICE), n,
                                     output_size=sum(blocks))
    first = (n.cumsum(0) - n)[tensor]
    key = _mix((_mix((tensor + 0x9E3779B1 * step) & WORD) + seed) & WORD)
    at = (torch.arange(sum(blocks), device=DEVICE) - first)[:, None] * BLOCK \
        + torch.arange(BLOCK, device=DEVICE)
    return _mix(((at & WORD) * 0x9E3779B1 + _mix(key[:, None] ^ (at >> 32))) & WORD)


def _two_to(power):
    return ((power + 127) << 23).view(torch.float32)


def _plain_e4m3(x, bits, square):
    """x ([blocks, 256]) as e4m3 numbers and a power of two for each block, rounded to one of the two
    neighbours at random by 16 ``bits``: so that the mean is x, or with ``square`` that the mean of
    the square is x's (and what is not zero stays so)."""
    fine = torch.isfinite(x)
    size = torch.where(fine, x.abs(), torch.zeros_like(x))
    top = size.amax(1, keepdim=True)
    some = top >= 1e-30
    part, power = torch.frexp(top)  # top <= 448 scale, 448 = 0.875 2^9
    power = torch.where(part > 0.875, power - 8, power - 9)
    a = size * torch.where(some, _two_to(-power), torch.zeros_like(top))
    unit = _two_to(torch.frexp(a)[1].clamp(min=-5) - 4)
    low = (a / unit).floor() * unit
    u = bits.float() * 2.0**-16 * unit
    up = (a - low) * (a + low) > u * (2.0 * low + unit) if square else a - low > u
    q = torch.where(up, low + unit, low).clamp(max=448.0)
    if square:
        q = torch.where(a > 0, q.clamp(min=2.0**-9), q)
    q = torch.where(fine, torch.copysign(q, x), torch.full_like(x, math.nan))
    scale = torch.where(some, _two_to(power), torch.zeros_like(top))
    return q.to(torch.float8_e4m3fn), scale[:, 0]


def _plain_adamw(state):
    flat, s = state["flat"], state["settings"]
    state["step"] += 1
    b1, b2 = s["betas"]
    first, second = 1 - b1 ** state["step"], 1 - b2 ** state["step"]
    g = flat["grad"].float()
    if state["case"]["bits"] == 8:
        m = flat["m"].view(-1, BLOCK).float() * flat["m_scale"][:, None]
        v = (flat["v"].view(-1, BLOCK).float() * flat["v_scale"][:, None]).square_()
        m, v = m.view(-1), v.view(-1)
    else:
        m, v = flat["m"], flat["v"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    root = v.sqrt()
    update = m / (root * (1 / math.sqrt(second)) + s["eps"])
    p = flat["param"].float() * (1 - s["lr"] * s["weight_decay"]) - update * (s["lr"] / first)
    flat["param"].copy_(p)
    if state["case"]["bits"] == 8:
        bits = _random_words(state["blocks"], 7, state["step"])
        for name, x, part in (("m", m, bits & 0xFFFF), ("v", root, bits >> 16)):
            codes, scale = _plain_e4m3(x.view(-1, BLOCK), part, name == "v")
            flat[name].copy_(codes.view(-1))
            flat[name + "_scale"].copy_(scale)
    else:
        flat["m"].copy_(m)
        flat["v"].copy_(v)
    return {k: x for k, x in flat.items() if k != "grad"}


# ---------------------------------------------------------------------------------------------
# The definitions in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    return {"logprobs": _exact_logprobs, "preference": _exact_preference,
            "policy": _exact_policy, "adamw": _exact_adamw}[case["op"]](state)


def _each_step(rows, vocab):
    step = max(1, (1 << 26) // vocab)
    return ((at, min(rows, at + step)) for at in range(0, rows, step))


def _exact_gradient(x, y, g, temperature):
    """g_t / temperature (1[v = y] - softmax), zero rows where g is zero."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for a, b in _each_step(*x.shape):
        hit = torch.zeros(b - a, x.shape[1], dtype=torch.float64, device=x.device)
        hit[torch.arange(b - a, device=x.device), y[a:b]] = 1.0
        hit -= torch.softmax(x[a:b].double() / temperature, 1)
        out[a:b] = hit * (g[a:b, None] / temperature)
    return out


def _exact_lp(x, y, temperature):
    out = torch.empty(len(y), dtype=torch.float64, device=x.device)
    for a, b in _each_step(*x.shape):
        out[a:b] = torch.log_softmax(x[a:b].double() / temperature, 1).gather(1, y[a:b, None])[:, 0]
    return out


def _exact_logprobs(state):
    case = state["case"]
    shape = state["logits"].shape
    x, y = state["logits"].reshape(-1, shape[-1]), state["targets"].reshape(-1)
    y0 = y.clamp(min=0)
    lp = _exact_lp(x, y0, case["temperature"])
    lp[y == IGNORE] = 0.0
    if not case["grad"]:
        return lp.view(shape[:-1])
    g = state["upstream"].reshape(-1).double()
    g[y == IGNORE] = 0.0
    return {"logps": lp.view(shape[:-1]),
            "grad": _exact_gradient(x, y0, g, case["temperature"]).view(shape)}


def _exact_preference(state):
    """By automatic differentiation of the loss, in float64."""
    case, pairs = state["case"], state["case"]["pairs"]
    x = state["logps"].double().requires_grad_()
    d = x if state["ref"] is None else x - state["ref"].double()
    used = torch.ones_like(d).detach() if state["mask"] is None else state["mask"].double()
    edges = state["offsets"].tolist()
    ends = list(zip(edges[:-1], edges[1:]))
    s = torch.stack([(d[a:b] * used[a:b]).sum() for a, b in ends])
    if case["average"]:
        s = s / torch.stack([used[a:b].sum() for a, b in ends]).clamp(min=1.0)
    u = case["beta"] * (s[:pairs] - s[pairs:]) - case["margin"]
    eps = case["smoothing"]
    if case["kind"] == "logistic":
        losses = -(1 - eps) * torch.nn.functional.logsigmoid(u) - eps * torch.nn.functional.logsigmoid(-u)
    elif case["kind"] == "hinge":
        losses = torch.relu(1 - u)
    else:
        losses = (u - 0.5) ** 2 / case["beta"] ** 2
    loss = losses.mean()
    (grad,) = torch.autograd.grad(loss, x)
    return {"loss": loss.detach(), "rewards": (case["beta"] * s.detach()).view(2, pairs), "grad": grad}


def _exact_policy(state):
    case, x, y = state["case"], state["logits"], state["targets"]
    w = state["weight"].double()
    lp = _exact_lp(x, y, case["temperature"]).requires_grad_()
    adv = state["advantages"].double()
    ratio = torch.exp(lp - state["old"].double())
    free, held = ratio * adv, torch.clamp(ratio, 0.8, 1.2) * adv
    losses, kl = -torch.min(free, held), torch.zeros_like(free)
    if state["ref"] is not None:
        d = state["ref"].double() - lp
        kl = torch.exp(d) - d - 1
        losses = losses + 0.05 * kl
    loss = (w * losses).sum() / w.sum()
    # inside the clip's range the two sides of the minimum are equal and the gradient is split
    # between them, so it is the same there; where only the clipped side is smaller it is zero
    (g,) = torch.autograd.grad(loss, lp)
    lp = lp.detach()
    return {"loss": loss.detach(), "logps": torch.where(w != 0, lp, torch.zeros_like(lp)),
            "kl": ((w * kl).sum() / w.sum()).detach(),
            "clipped": ((w * (free > held)).sum() / w.sum()).detach(),
            "grad": _exact_gradient(x, y, g, case["temperature"])}


def _exact_e4m3(x, u, square):
    x = x.view(-1, BLOCK)
    size = x.abs()
    top = size.amax(1, keepdim=True)
    scale = torch.where(top > 0, torch.exp2(torch.ceil(torch.log2(top / 448.0))), torch.zeros_like(top))
    a = torch.where(top > 0, size / scale, torch.zeros_like(x))
    unit = torch.exp2(torch.floor(torch.log2(a)).clamp(min=-6.0) - 3.0)
    low = torch.floor(a / unit) * unit
    chance = (a**2 - low**2) / ((low + unit) ** 2 - low**2) if square else (a - low) / unit
    q = torch.where(u < chance, low + unit, low).clamp(max=448.0)
    if square:
        q = torch.where(a > 0, q.clamp(min=2.0**-9), q)
    return (torch.sign(x) * q).view(-1), scale[:, 0]


def _exact_adamw(state):
    flat, s, bits = state["flat"], state["settings"], state["case"]["bits"]
    step = state["step"] + 1
    b1, b2 = s["betas"]
    g = flat["grad"].double()
    if bits == 8:
        m = (flat["m"].float().double().view(-1, BLOCK) * flat["m_scale"].double()[:, None]).view(-1)
        v = (flat["v"].float().double().view(-1, BLOCK) * flat["v_scale"].double()[:, None]).view(-1) ** 2
    else:
        m, v = flat["m"].double(), flat["v"].double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g**2
    hat_m, hat_v = m / (1 - b1**step), v / (1 - b2**step)
    p = flat["param"].double()
    p = p - s["lr"] * s["weight_decay"] * p - s["lr"] * hat_m / (hat_v.sqrt() + s["eps"])
    out = {"param": p, "m": m, "v": v}
    if bits == 8:
        words = _random_words(state["blocks"], 7, step)
        out["m"], out["m_scale"] = _exact_e4m3(m, (words & 0xFFFF).double() / 65536, False)
        out["v"], out["v_scale"] = _exact_e4m3(v.sqrt(), (words >> 16).double() / 65536, True)
    return out
