"""A token's scores and the distillation from a teacher's top lists, as a user's program calls them, and
in plain torch.

Two operators: ``token_scores`` (log-probability of a given token, entropy, top alternatives, from
logits) and ``distillation_loss`` (a student's logits against a teacher's top lists). ``listed()`` has
fixed cases, ``draw()`` more of the same ranges; ``run()`` makes one pass through a case's operator:
elementary torch operations (in float32, what cancels in float64) while ``own`` is false, this package's
kernels where it is true. ``exact()`` has the definitions in float64.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
IGNORE = -100
LEAST_REST = 2.0**-24  # of the teacher's probability outside its list, where it is divided by


# ---------------------------------------------------------------------------------------------
# Cases


def listed():
    return [
        # the tokens just sampled for a few requests, with their five likeliest alternatives
        {"name": "scores decode", "op": "scores", "batch": 4, "rows": 1, "vocab": 32000,
         "dtype": "bf16", "target": True, "top": 5, "grad": False, "shift": False, "ignored": 0.0,
         "hidden": 0.0, "temperature": 0.7},
        # one step of a server's full batch, a third of a large vocabulary hidden by a grammar
        {"name": "scores serving", "op": "scores", "batch": 256, "rows": 1, "vocab": 131072,
         "dtype": "bf16", "target": True, "top": 20, "grad": False, "shift": False, "ignored": 0.0,
         "hidden": 0.3, "temperature": 1.0},
        # a teacher's lists for a batch of texts: nothing but the top alternatives is asked for
        {"name": "scores teacher", "op": "scores", "batch": 4, "rows": 1024, "vocab": 131072,
         "dtype": "bf16", "target": False, "top": 64, "grad": False, "shift": False, "ignored": 0.0,
         "hidden": 0.0, "temperature": 1.0},
        # log-probabilities and an entropy bonus in training: logits[:, :-1] of an odd vocabulary, the
        # prompt ignored
        {"name": "scores entropy", "op": "scores", "batch": 4, "rows": 1023, "vocab": 50021,
         "dtype": "bf16", "target": True, "top": 0, "grad": True, "shift": True, "ignored": 0.3,
         "hidden": 0.0, "temperature": 1.0},
        # a small model in float32, with the best alternative, whose probability is calibrated
        {"name": "scores small vocabulary", "op": "scores", "batch": 16, "rows": 511, "vocab": 777,
         "dtype": "f32", "target": True, "top": 1, "grad": True, "shift": True, "ignored": 0.1,
         "hidden": 0.0, "temperature": 1.0},
        # a micro-batch against short lists
        {"name": "distill micro-batch", "op": "distill", "rows": 64, "vocab": 32000, "dtype": "bf16",
         "top": 8, "kind": "forward", "rest": "bucket", "ragged": False, "masked": 0.0,
         "temperature": 1.0, "scale": 1.0},
        # a small model in float32 that is to put its mass where the teacher has it
        {"name": "distill small vocabulary", "op": "distill", "rows": 8176, "vocab": 777,
         "dtype": "f32", "top": 16, "kind": "reverse", "rest": "bucket", "ragged": False,
         "masked": 0.1, "temperature": 1.0, "scale": 1.0},
        # lists cut at a probability (ragged) in an odd vocabulary, float32, softened
        {"name": "distill odd vocabulary", "op": "distill", "rows": 1999, "vocab": 50021,
         "dtype": "f32", "top": 20, "kind": "jensen", "rest": "bucket", "ragged": True,
         "masked": 0.4, "temperature": 2.0, "scale": 1.0},
        # the longest lists, renormalised; float16, so the loss is scaled
        {"name": "distill long lists", "op": "distill", "rows": 4096, "vocab": 32000,
         "dtype": "f16", "top": 128, "kind": "forward", "rest": "drop", "ragged": False,
         "masked": 0.0, "temperature": 1.0, "scale": 1024.0},
        # a full batch of a large vocabulary
        {"name": "distill batch", "op": "distill", "rows": 8192, "vocab": 131072, "dtype": "bf16",
         "top": 64, "kind": "forward", "rest": "bucket", "ragged": False, "masked": 0.1,
         "temperature": 1.0, "scale": 1.0},
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["scores", "distill"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    vocab = _log(rng, 256, 131072)
    most = (1 << 30 if op == "distill" else 1 << 29) >> (dtype == "f32")
    rows = _log(rng, 1, max(1, min(8192, most // vocab)))
    if op == "scores":
        batch = rng.choice([1, 2, 4]) if rows >= 8 else 1
        grad = rng.random() < 0.4
        return {"op": op, "batch": batch, "rows": rows // batch, "vocab": vocab, "dtype": dtype,
                "target": grad or rng.random() < 0.7, "top": rng.choice([0, 1, 5, 20, 64, 128]),
                "grad": grad, "shift": grad and rng.random() < 0.5,
                "ignored": rng.choice([0.0, 0.1, 0.5]),
                "hidden": 0.0 if grad else rng.choice([0.0, 0.0, 0.3]),
                "temperature": rng.choice([1.0, 1.0, 0.7, 1.5])}
    kind = rng.choice(["forward", "forward", "reverse", "jensen"])
    rest = "bucket" if kind == "reverse" else rng.choice(["bucket", "bucket", "drop"])
    return {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype,
            "top": rng.choice([1, 8, 20, 50, 64, 128]), "kind": kind, "rest": rest,
            "ragged": rng.random() < 0.3, "masked": rng.choice([0.0, 0.2, 0.5]),
            "temperature": rng.choice([1.0, 1.0, 2.0]),
            "scale": 1024.0 if dtype == "f16" else rng.choice([1.0, 1.0, 0.125])}


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    vocab, top = case["vocab"], case["top"]
    if case["op"] == "scores":
        rows = case["batch"] * case["rows"]
        used = rows * (1 - case["ignored"] * case["target"])
        tokens = rows * (4 + 12 * top + 12 * case["target"] + 8 * case["grad"])
        return {"bytes": used * vocab * size + rows * vocab * size * case["grad"] + tokens,
                "flops": used * vocab * (6 + 8 * case["grad"])}
    rows, used = case["rows"], case["rows"] * (1 - case["masked"])
    return {"bytes": used * (vocab * size + 12 * top) + rows * (vocab * size + 8),
            "flops": used * vocab * 8}


# ---------------------------------------------------------------------------------------------
# Inputs


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _model_logits(rows, vocab, dtype, gen):
    """A trained model's logits: a few tokens well above the rest."""
    logits = torch.empty(rows, vocab, dtype=dtype, device=DEVICE)
    step = max(1, (1 << 27) // vocab)
    for at in range(0, rows, step):
        k = min(step, rows - at)
        x = torch.randn(k, vocab, generator=gen, device=DEVICE).mul_(2.0)
        likely = torch.randint(0, vocab, (k, 8), generator=gen, device=DEVICE)
        x.scatter_add_(1, likely, 10.0 + torch.randn(k, 8, generator=gen, device=DEVICE))
        logits[at:at + k] = x
    return logits


def _sampled(logits, temperature, gen):
    out = torch.empty(len(logits), dtype=torch.int64, device=DEVICE)
    step = max(1, (1 << 27) // logits.shape[1])
    for at in range(0, len(logits), step):
        z = logits[at:at + step].float() / temperature
        noise = torch.empty_like(z).exponential_(generator=gen).log_().neg_()  # Gumbel
        out[at:at + step] = (z + noise).argmax(1)
    return out


def _teacher_lists(logits, top, temperature, gen):
    """The top of a teacher that agrees with the student in most: ids and log-probabilities."""
    ids = torch.empty(len(logits), top, dtype=torch.int64, device=DEVICE)
    logps = torch.empty(len(logits), top, device=DEVICE)
    step = max(1, (1 << 27) // logits.shape[1])
    for at in range(0, len(logits), step):
        z = logits[at:at + step].float()
        z = (z + torch.randn(z.shape, generator=gen, device=DEVICE)).div_(temperature)
        best, ids[at:at + step] = z.topk(top, 1)
        logps[at:at + step] = best - torch.logsumexp(z, 1, keepdim=True)
    return ids, logps


def prepare(case, seed):
    gen = _generator(seed)
    state = {"case": dict(case)}
    vocab, dtype, t = case["vocab"], DTYPES[case["dtype"]], case["temperature"]
    if case["op"] == "scores":
        batch, rows = case["batch"], case["rows"]
        whole = rows + 1 if case["shift"] else rows
        logits = _model_logits(batch * whole, vocab, dtype, gen)
        if case["hidden"]:
            step = max(1, (1 << 28) // vocab)
            for at in range(0, len(logits), step):
                part = logits[at:at + step]
                part.masked_fill_(torch.rand(part.shape, generator=gen, device=DEVICE)
                                  < case["hidden"], -math.inf)
        state["logits"] = logits.view(batch, whole, vocab)[:, :rows]
        state["targets"] = None
        if case["target"]:
            y = _sampled(logits, t, gen)
            y[torch.rand(batch * whole, generator=gen, device=DEVICE) < case["ignored"]] = IGNORE
            state["targets"] = y.view(batch, whole)[:, :rows].contiguous()
        if case["grad"]:
            state["upstream"] = (torch.randn(batch, rows, generator=gen, device=DEVICE) - 1.0,
                                 torch.full((batch, rows), 0.01, device=DEVICE))
        return state
    rows, top = case["rows"], case["top"]
    logits = _model_logits(rows, vocab, dtype, gen)
    ids, logps = _teacher_lists(logits, top, t, gen)
    if case["ragged"]:
        # each list ends where it has its own share of the teacher's probability
        share = 0.5 + 0.5 * torch.rand(rows, 1, generator=gen, device=DEVICE)
        before = logps.exp().cumsum(1) - logps.exp()
        left_out = before >= share
        ids, logps = ids.masked_fill(left_out, IGNORE), logps.masked_fill(left_out, 0.0)
    weight = None
    if case["masked"]:
        weight = torch.rand(rows, generator=gen, device=DEVICE) >= case["masked"]
        weight[0] = True
    state.update(logits=logits, ids=ids, logps=logps, weight=weight)
    return state


# ---------------------------------------------------------------------------------------------
# One pass


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    import torchisotonic_b200 as ti

    case, x = state["case"], state["logits"]
    if case["op"] == "scores":
        if case["grad"]:
            x = x.detach().requires_grad_()
        got = ti.token_scores(x, state["targets"], top=case["top"], temperature=case["temperature"])
        out = {"entropy": got.entropy.detach(), "top_logps": got.top_logps, "top_ids": got.top_ids}
        if case["target"]:
            out["logps"] = got.logps.detach()
        if case["grad"]:
            (out["grad"],) = torch.autograd.grad((got.logps, got.entropy), x, state["upstream"])
        return out
    x = x.detach().requires_grad_()
    got = ti.distillation_loss(x, state["ids"], state["logps"], kind=case["kind"],
                               rest=case["rest"], weight=state["weight"],
                               temperature=case["temperature"], upstream=case["scale"])
    loss = got.loss if case["scale"] == 1.0 else got.loss * case["scale"]
    (gx,) = torch.autograd.grad(loss, x)
    return {"loss": got.loss.detach(), "divergence": got.divergence, "grad": gx}


def _run_plain(state):
    return _plain_scores(state) if state["case"]["op"] == "scores" else _plain_distill(state)


def _ordered(x):
    """Integers in the order of x's numbers (-0 beside 0), made unique by their place in the row: of
    equal ones the first is the largest."""
    bits = (x.float() + 0.0).view(torch.int32)
    keys = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32
    return keys + torch.arange(x.shape[-1] - 1, -1, -1, device=x.device)


def _plain_scores(state):
    case, shape = state["case"], state["logits"].shape
    t, x = case["temperature"], state["logits"].reshape(-1, shape[-1])
    z = x.float() / t
    a = z - z.amax(1, keepdim=True)
    e = a.exp()
    s = e.sum(1, keepdim=True)
    lse = s.log()
    # of a probability of 0 the logarithm is not taken: 0 log 0 = 0
    entropy = lse[:, 0] - (e * torch.where(e > 0, a, torch.zeros_like(a))).sum(1) / s[:, 0]
    ids = _ordered(x).topk(case["top"], 1)[1]
    top_logps = a.gather(1, ids) - lse
    if not case["target"]:
        return {"entropy": entropy.view(shape[:-1]),
                "top_logps": top_logps.view(*shape[:-1], -1), "top_ids": ids.view(*shape[:-1], -1)}
    y = state["targets"].reshape(-1)
    used = y != IGNORE
    y = torch.where(used, y, torch.zeros_like(y))
    lp = a.gather(1, y[:, None])[:, 0] - lse[:, 0]
    zero = torch.zeros_like(lp)
    out = {"entropy": torch.where(used, entropy, zero).view(shape[:-1]),
           "top_logps": torch.where(used[:, None], top_logps, zero[:, None]).view(*shape[:-1], -1),
           "top_ids": ids.masked_fill(~used[:, None], IGNORE).view(*shape[:-1], -1),
           "logps": torch.where(used, lp, zero).view(shape[:-1])}
    if case["grad"]:
        up, up_h = (torch.where(used, u.reshape(-1) / t, zero)[:, None] for u in state["upstream"])
        grad = e.div_(s).mul_(-(a.sub_(lse).add_(entropy[:, None]).mul_(up_h).add_(up)))
        grad.scatter_add_(1, y[:, None], up)
        out["grad"] = grad.to(x.dtype).view(shape)
    return out


def _xlogy(x, y):
    """x log y, 0 where x is 0."""
    return torch.where(x > 0, x * y.log(), torch.zeros_like(x))


def _plain_distill(state):
    case, x, kind, t = state["case"], state["logits"], state["case"]["kind"], state["case"]["temperature"]
    ids, w = state["ids"], state["weight"]
    there = ids != IGNORE
    at = torch.where(there, ids, torch.zeros_like(ids))
    w = torch.ones(len(x), device=x.device) if w is None else w.float()
    w = torch.where(there[:, 0], w, torch.zeros_like(w))
    # the teacher's buckets: 1 - the list's sum cancels
    q = torch.where(there, state["logps"].double().exp(), torch.zeros((), dtype=torch.float64, device=x.device))
    q_rest = (1.0 - q.sum(1)).clamp(min=0.0)
    if case["rest"] == "drop":
        q = q / q.sum(1, keepdim=True)
        q_rest = torch.zeros_like(q_rest)
    elif kind == "reverse":
        q_rest = q_rest.clamp(min=LEAST_REST)
    # the student's: the rest summed from its own exponentials
    z = x.float() / t
    listed_z = z.gather(1, at)
    top = z.amax(1, keepdim=True)
    e = z.sub_(top).exp_()
    rest = e.scatter(1, torch.where(there, ids, ids[:, :1]), 0.0).sum(1).double()
    listed_e = torch.where(there, (listed_z.double() - top).exp(), torch.zeros_like(q))
    s = rest + listed_e.sum(1)
    p, p_rest = listed_e / s[:, None], rest / s
    # f = d divergence / d p of the buckets; an entry that is left out has q = p = 0
    if kind == "forward":
        d = (_xlogy(q, q) - _xlogy(q, p)).sum(1) + _xlogy(q_rest, q_rest) - _xlogy(q_rest, p_rest)
        mean = -(q.sum(1) + q_rest)
        listed_g = -q - p * mean[:, None]
        rest_g = -q_rest / p_rest - mean
    else:
        a = 0.0 if kind == "reverse" else 0.5
        m, m_rest = (q, q_rest) if a == 0 else (a * q + (1 - a) * p, a * q_rest + (1 - a) * p_rest)
        f = torch.where(p > 0, (1 - a) * (p / m).log(), torch.zeros_like(p))
        f_rest = (1 - a) * (p_rest / m_rest).log()
        mean = (p * f).sum(1) + p_rest * f_rest
        d = mean
        if a:
            d = d + a * ((_xlogy(q, q) - _xlogy(q, m)).sum(1) + _xlogy(q_rest, q_rest)
                         - _xlogy(q_rest, m_rest))
        listed_g = p * (f - mean[:, None])
        rest_g = f_rest - mean
    total = w.double().sum()
    c = (case["scale"] * w / (total * t))[:, None]
    grad = e.mul_((c * rest_g[:, None] / s[:, None]).float())
    # entries left out stand behind their list's first, whose value they repeat
    value = (c * listed_g).float()
    grad.scatter_(1, torch.where(there, ids, at[:, :1]), torch.where(there, value, value[:, :1]))
    used = w != 0
    grad = torch.where(used[:, None], grad, torch.zeros_like(grad)).to(x.dtype)
    d = torch.where(used, d, torch.zeros_like(d))
    return {"loss": ((w * d).sum() / total).float(), "divergence": d.float(), "grad": grad}


# ---------------------------------------------------------------------------------------------
# The definitions in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_scores(state) if case["op"] == "scores" else _exact_distill(state)


def _each_step(rows, vocab):
    step = max(1, (1 << 26) // vocab)
    return ((at, min(rows, at + step)) for at in range(0, rows, step))


def _exact_scores(state):
    """By sorting, and automatic differentiation."""
    case, shape, t = state["case"], state["logits"].shape, state["case"]["temperature"]
    x, y = state["logits"].reshape(-1, shape[-1]), state["targets"]
    y = None if y is None else y.reshape(-1)
    up = [u.reshape(-1).double() for u in state["upstream"]] if case["grad"] else None
    parts = []
    for a, b in _each_step(*x.shape):
        wide = x[a:b].double().requires_grad_()
        used = torch.ones(b - a, dtype=torch.bool, device=x.device) if y is None else y[a:b] != IGNORE
        logp = torch.log_softmax(wide / t, 1)
        p = logp.exp()
        h = -(p * logp.clamp(min=-1e300)).sum(1) * used
        order = torch.sort(x[a:b], dim=1, descending=True, stable=True)[1][:, :case["top"]]
        part = {"entropy": h.detach(),
                "top_logps": torch.where(used[:, None], logp.detach().gather(1, order), 0.0),
                "top_ids": torch.where(used[:, None], order, IGNORE)}
        if y is not None:
            lp = torch.where(used, logp.gather(1, y[a:b].clamp(min=0)[:, None])[:, 0], 0.0)
            part["logps"] = lp.detach()
        if case["grad"]:
            (part["grad"],) = torch.autograd.grad((lp, h), wide, (up[0][a:b], up[1][a:b]))
        parts.append(part)
    out = {k: torch.cat([part[k] for part in parts]) for k in parts[0]}
    return {k: v.view(*shape[:-1], -1) if k.startswith("top") else v.view(shape if k == "grad" else shape[:-1])
            for k, v in out.items()}


def _exact_distill(state):
    """By automatic differentiation over the buckets' logarithms."""
    case, x, t = state["case"], state["logits"], state["case"]["temperature"]
    there = state["ids"] != IGNORE
    w = torch.ones(len(x), device=x.device) if state["weight"] is None else state["weight"]
    w = w.double() * there[:, 0]
    total, parts = w.sum(), []
    for a, b in _each_step(*x.shape):
        on = there[a:b]
        wide = x[a:b].double().requires_grad_()
        logp = torch.log_softmax(wide / t, 1)
        named = torch.zeros(wide.shape, dtype=torch.bool, device=x.device)
        row, col = on.nonzero(as_tuple=True)
        named[row, state["ids"][a:b][row, col]] = True
        rest = torch.logsumexp(logp.masked_fill(named, -math.inf), 1)
        lp = torch.cat([logp.gather(1, state["ids"][a:b].clamp(min=0)), rest[:, None]], 1)
        q = torch.where(on, state["logps"][a:b].double().exp(), 0.0)
        if case["rest"] == "drop":
            q = torch.cat([q / q.sum(1, keepdim=True), torch.zeros_like(q[:, :1])], 1)
        else:
            least = LEAST_REST if case["kind"] == "reverse" else 0.0
            q = torch.cat([q, (1 - q.sum(1, keepdim=True)).clamp(min=least)], 1)
        on = torch.cat([on, torch.ones_like(on[:, :1])], 1)
        lq = q.log()
        if case["kind"] == "forward":
            terms = torch.where(q > 0, q * (lq - lp), 0.0)
        elif case["kind"] == "reverse":
            terms = lp.exp() * (torch.where(on, lp, 0.0) - torch.where(on, lq, 0.0))
        else:
            lm = torch.logaddexp(lq, lp) - math.log(2.0)
            terms = 0.5 * torch.where(q > 0, q * (lq - lm), 0.0) + 0.5 * lp.exp() * (lp - lm)
        d = torch.where(on, terms, 0.0).sum(1)
        part_w = w[a:b]
        (grad,) = torch.autograd.grad((part_w * d).sum() / total * case["scale"], wide)
        parts.append((torch.where(part_w != 0, d.detach(), 0.0),
                      torch.where(part_w[:, None] != 0, grad, 0.0)))
    d = torch.cat([part[0] for part in parts])
    return {"loss": (w * d).sum() / total, "divergence": d,
            "grad": torch.cat([part[1] for part in parts])}
