"""Workloads of the distillation operators: the teacher's top logits, the distillation loss through a
frozen head with its gradient, and the verification of drafted tokens.

``listed()`` names the standing cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes
what a training or serving program holds before the call, ``run`` makes one pass (the plain torch form
below, or with ``own`` this package's kernels), ``exact`` gives the same outputs in 64 bits.
"""

import math

import torch

own = False

FLOATS = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}

# The largest listed cases bound what a drawn case may cost.
MOST_FLOPS = 6 * 8192 * 3584 * 151936
MOST_LOGITS = 3300 * 151936
MOST_PROBS = 256 * 6 * 151936


def listed():
    return [
        # ---- the teacher's top logits and log-sum-exp
        # One position of a teacher that answers while the student trains: latency.
        {"name": "top one token", "op": "top", "rows": 1, "vocab": 151936, "k": 64, "dtype": "fp16",
         "temperature": 1.0, "pad": 0},
        # A short generated answer, an odd vocabulary whose rows start anywhere, a long list.
        {"name": "top short odd", "op": "top", "rows": 37, "vocab": 32001, "k": 200, "dtype": "bf16",
         "temperature": 1.0, "pad": 0},
        # A packed training batch of the 151936-token vocabulary.
        {"name": "top packed batch", "op": "top", "rows": 3300, "vocab": 151936, "k": 64, "dtype": "fp16",
         "temperature": 2.0, "pad": 0},
        # A teacher that keeps fp32 logits in a padded buffer.
        {"name": "top fp32 padded", "op": "top", "rows": 1000, "vocab": 151936, "k": 100, "dtype": "fp32",
         "temperature": 1.5, "pad": 64},
        # ---- distillation through the frozen head
        # A few generated tokens: one read of the head is what counts.
        {"name": "distill few tokens", "op": "distill", "rows": 48, "hidden": 1536, "vocab": 151936, "k": 32,
         "dtype": "fp16", "temperature": 1.0, "tail": True, "labelled": 1.0, "train": True},
        # Validation on a packed batch: the loss alone.
        {"name": "distill evaluation", "op": "distill", "rows": 3300, "hidden": 1536, "vocab": 151936, "k": 64,
         "dtype": "fp16", "temperature": 1.0, "tail": True, "labelled": 1.0, "train": False},
        # The packed training batch with 37 % of the positions answered by the teacher.
        {"name": "distill packed batch", "op": "distill", "rows": 3300, "hidden": 1536, "vocab": 151936, "k": 64,
         "dtype": "fp16", "temperature": 2.0, "tail": True, "labelled": 0.37, "train": True},
        # A small bf16 student with an odd vocabulary; the teacher sent its list without a tail.
        {"name": "distill odd bf16", "op": "distill", "rows": 1001, "hidden": 896, "vocab": 32001, "k": 20,
         "dtype": "bf16", "temperature": 1.0, "tail": False, "labelled": 1.0, "train": True},
        # The wide model on a long packed batch, every position answered.
        {"name": "distill long wide", "op": "distill", "rows": 8192, "hidden": 3584, "vocab": 151936, "k": 100,
         "dtype": "bf16", "temperature": 1.0, "tail": True, "labelled": 1.0, "train": True},
        # ---- verification of drafted tokens
        # One sequence, four drafts: latency between two target steps.
        {"name": "verify one sequence", "op": "verify", "batch": 1, "drafts": 4, "vocab": 151936, "dtype": "fp32",
         "sampled": True, "ragged": False},
        # An odd batch of drafts looked up in the prompt (no draft distribution), some sequences without any.
        {"name": "verify looked up", "op": "verify", "batch": 33, "drafts": 7, "vocab": 32001, "dtype": "bf16",
         "sampled": False, "ragged": True},
        # A full serving batch.
        {"name": "verify full batch", "op": "verify", "batch": 256, "drafts": 5, "vocab": 151936, "dtype": "fp32",
         "sampled": True, "ragged": False},
    ]


def _spread(rng, low, high):
    """A whole number spread evenly over the logarithm of [low, high]."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["top", "distill", "verify"])
    vocab = _spread(rng, 1000, 152064)
    if op == "top":
        rows = min(_spread(rng, 1, 4096), MOST_LOGITS // vocab)
        return {"op": op, "rows": rows, "vocab": vocab, "k": _spread(rng, 1, 256),
                "dtype": rng.choice(["fp16", "bf16", "fp32"]), "temperature": rng.choice([0.7, 1.0, 2.0]),
                "pad": rng.choice([0, 0, 3, 64])}
    if op == "distill":
        hidden = 8 * _spread(rng, 16, 448) - rng.choice([0, 0, 0, 3])
        rows = min(_spread(rng, 1, 8192), MOST_FLOPS // (6 * hidden * vocab))
        return {"op": op, "rows": rows, "hidden": hidden, "vocab": vocab, "k": _spread(rng, 1, 128),
                "dtype": rng.choice(["fp16", "bf16"]), "temperature": rng.choice([0.7, 1.0, 2.0]),
                "tail": rng.random() < 0.6, "labelled": rng.choice([1.0, 0.37]), "train": rng.random() < 0.75}
    drafts = rng.randint(1, 8)
    batch = min(_spread(rng, 1, 512), MOST_PROBS // ((drafts + 1) * vocab))
    return {"op": op, "batch": max(1, batch), "drafts": drafts, "vocab": vocab,
            "dtype": rng.choice(["fp32", "fp32", "fp16", "bf16"]), "sampled": rng.random() < 0.7,
            "ragged": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs
def _head_and_hidden(rows, hidden, vocab, gen, peak):
    """A head ~N(0, 0.02) and hidden states whose logits are N(0, 1) with a few raised tokens, as a
    trained model's are: one token by about `peak` nats, two more by somewhat less."""
    dev = "cuda"
    weight = torch.randn((vocab, hidden), device=dev, generator=gen) * 0.02
    x = torch.randn((rows, hidden), device=dev, generator=gen) / (0.02 * math.sqrt(hidden))
    for drop in (0.0, 2.0, 4.0):
        token = torch.randint(vocab, (rows,), device=dev, generator=gen)
        lift = torch.rand(rows, device=dev, generator=gen) * 8 + (peak - 4 - drop)
        x += weight[token] * (lift / (0.02 ** 2 * hidden))[:, None]
    return weight, x


def _prepare_top(case, gen):
    """Logits of a trained model: a normal body and, as in language, few tokens far above it."""
    rows, vocab, pad = case["rows"], case["vocab"], case["pad"]
    dtype = FLOATS[case["dtype"]]
    buf = torch.empty((rows, vocab + pad), device="cuda", dtype=dtype)
    buf.normal_(0.0, 2.0, generator=gen)
    raised = torch.randint(vocab, (rows, 40), device="cuda", generator=gen)
    lift = -torch.log(torch.rand((rows, 40), device="cuda", generator=gen)) * 3 + 6
    buf.scatter_reduce_(1, raised, lift.to(dtype), "amax")
    return {"case": case, "logits": buf[:, :vocab]}


def _prepare_distill(case, gen):
    rows, hidden, vocab, k = case["rows"], case["hidden"], case["vocab"], case["k"]
    dtype, tau = FLOATS[case["dtype"]], case["temperature"]
    peak = math.log(vocab)
    weight, x = _head_and_hidden(rows, hidden, vocab, gen, peak)
    weight = weight.to(dtype)
    # The teacher saw the same text with another network: the same raised tokens, other noise.
    seen = x + 0.6 * torch.randn(x.shape, device="cuda", generator=gen) / (0.02 * math.sqrt(hidden))
    teacher = seen.to(dtype) @ weight.t()
    logits, indices = torch.topk(teacher.float(), min(k, vocab), dim=1)
    lse = torch.logsumexp(teacher.float() / tau, dim=1) if case["tail"] else None
    del teacher, seen
    if case["labelled"] < 1.0:
        prompt = torch.rand(rows, device="cuda", generator=gen) >= case["labelled"]
        indices[prompt] = -1
    # Upstream gradients: the mean over the batch, with fp16 training's loss scale.
    scale = (65536.0 if case["dtype"] == "fp16" else 1.0) / rows
    upstream = scale * (0.5 + torch.rand(rows, device="cuda", generator=gen))
    return {"case": case, "hidden": x.to(dtype).requires_grad_(case["train"]), "weight": weight,
            "indices": indices, "logits": logits, "lse": lse, "upstream": upstream}


def _prepare_verify(case, gen):
    batch, drafts, vocab = case["batch"], case["drafts"], case["vocab"]
    dtype = FLOATS[case["dtype"]]
    base = torch.randn((batch, drafts + 1, vocab), device="cuda", generator=gen).mul_(1.5)
    raised = torch.randint(vocab, (batch, drafts + 1, 20), device="cuda", generator=gen)
    base.scatter_reduce_(2, raised, torch.rand(raised.shape, device="cuda", generator=gen) * 8 + 6, "amax")
    # The draft model's logits follow the target's with noise.
    near = base[:, :drafts] + 0.7 * torch.randn((batch, drafts, vocab), device="cuda", generator=gen)
    draft = torch.softmax(near, -1)
    del near
    noise = torch.empty((batch, drafts, vocab), device="cuda").exponential_(generator=gen)
    tokens = (draft / noise.clamp_min_(1e-30)).argmax(-1)
    del noise
    state = {"case": case, "target": torch.softmax(base, -1).to(dtype),
             "draft": draft.to(dtype) if case["sampled"] else None, "tokens": tokens,
             "uniforms": torch.rand((batch, drafts), device="cuda", generator=gen),
             "noise": torch.empty((batch, vocab), device="cuda").exponential_(generator=gen).clamp_min_(1e-30),
             "lens": None}
    if case["ragged"]:
        state["lens"] = torch.randint(drafts + 1, (batch,), device="cuda", generator=gen)
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"top": _prepare_top, "distill": _prepare_distill, "verify": _prepare_verify}[case["op"]](case, gen)


# ------------------------------------------------------------------ the plain forms
def plain_top(logits, k, temperature):
    """The k largest logits of each row in falling order (ties: the lowest index first) and
    log sum exp(logits / temperature)."""
    z = logits.float()
    bits = z.view(torch.int32).to(torch.int64)
    bits = torch.where(z == 0, torch.zeros_like(bits), bits)
    rising = torch.where(bits < 0, -(bits & 0x7FFFFFFF) - 1, bits)
    columns = torch.arange(z.shape[1], device=z.device)
    keys = rising * (1 << 32) + ((1 << 32) - 1 - columns)
    best = torch.topk(keys, k, dim=1).values
    indices = (1 << 32) - 1 - (best & ((1 << 32) - 1))
    x = z / temperature
    top = x.amax(1, keepdim=True)
    lse = top[:, 0] + (x - top).exp().sum(1).log()
    return logits.gather(1, indices), indices, lse


def _gap(p, logp, q, logq):
    """p log(p / q) - p + q: the terms of a KL divergence of two distributions, each at least zero, so that
    their sum does not cancel where the two are close."""
    r = logp - logq
    return torch.where(p > 0, q * (r * r.exp() - r.expm1()), q)


def plain_distill(hidden, weight, indices, logits, lse, temperature, upstream):
    """KL(teacher || student) on the listed tokens and, where the teacher's log-sum-exp is given, one
    bucket of all others; the student's probability of the listed tokens; the gradient for `hidden`."""
    vocab = weight.shape[0]
    z = hidden.float() @ weight.float().t() / temperature
    used = indices >= 0
    some = used.any(1)
    t = torch.where(used, logits.float() / temperature, -math.inf)
    if lse is None:
        top = torch.where(some, t.amax(1), 0.0)
        norm = top + torch.where(some, (t - top[:, None]).exp().sum(1), 1.0).log()
    else:
        norm = lse
    logp = t - norm[:, None]
    p = logp.exp()
    rest = torch.zeros_like(norm) if lse is None else torch.where(some, (1 - p.sum(1)).clamp_min(0.0), 0.0)
    listed_ = torch.zeros((z.shape[0], vocab + 1), device=z.device, dtype=torch.bool)
    listed_.scatter_(1, torch.where(used, indices, vocab), True)
    listed_ = listed_[:, :vocab]
    m = z.amax(1)
    e = (z - m[:, None]).exp()
    total = e.sum(1)
    q_rest = torch.where(listed_, 0.0, e).sum(1) / total
    mass = torch.where(some, torch.where(listed_, e, 0.0).sum(1) / total, 0.0)
    spot = torch.where(used, indices, 0)
    logq = z.gather(1, spot) - (m + total.log())[:, None]
    loss = torch.where(used, _gap(p, logp, logq.exp(), logq), 0.0).sum(1)
    loss = loss + _gap(rest, rest.log(), q_rest, q_rest.log())
    loss = torch.where(some, loss, 0.0)
    if upstream is None:
        return loss, mass
    q = e / total[:, None]
    share = 1 - rest / torch.where(q_rest > 0, q_rest, 1.0)
    dz = torch.where(listed_, q, q * share[:, None])
    dz.scatter_add_(1, spot, torch.where(used, -p, 0.0))
    dz = dz * torch.where(some, upstream / temperature, 0.0)[:, None]
    return loss, mass, (dz @ weight.float()).to(hidden.dtype)


def plain_verify(target, tokens, uniforms, noise, draft, lens):
    """Accept draft s while u_s q_s(x_s) < p_s(x_s); then one token from the residual max(p - q, 0) of
    the first rejected place, or from the target after the last draft: the argmax of residual / noise."""
    batch, drafts = tokens.shape
    vocab = target.shape[2]
    place = torch.arange(drafts, device=target.device)
    lens = torch.full((batch,), drafts, device=target.device) if lens is None else lens
    p_tok = target[:, :drafts].float().gather(2, tokens[:, :, None])[:, :, 0]
    q_tok = torch.ones_like(p_tok) if draft is None else draft.float().gather(2, tokens[:, :, None])[:, :, 0]
    ok = (uniforms * q_tok < p_tok) & (place < lens[:, None])
    accepted = ok.to(torch.int64).cumprod(1).sum(1)
    row = torch.arange(batch, device=target.device)
    p = target[row, accepted].float()
    at = accepted.clamp_max(drafts - 1)
    if draft is None:
        q = torch.zeros_like(p).scatter_(1, tokens[row, at][:, None], 1.0)
        residual = torch.where(q > 0, 0.0, p)
    else:
        residual = (p - draft[row, at].float()).clamp_min(0.0)
    residual = torch.where((accepted < lens)[:, None], residual, p)
    residual = torch.where(residual.amax(1, keepdim=True) > 0, residual, p)
    score = residual / noise
    token = torch.where(score.amax(1) > 0, score.argmax(1), -1)
    out = torch.where(place < accepted[:, None], tokens, -1)
    out = torch.cat([out, torch.full((batch, 1), -1, device=out.device, dtype=out.dtype)], 1)
    return accepted, out.scatter(1, accepted[:, None], token[:, None])


def run(state):
    case = state["case"]
    if case["op"] == "top":
        if own:
            from soupsuck_b200.kernels import top_logits
            return top_logits(state["logits"], case["k"], temperature=case["temperature"])
        return plain_top(state["logits"], case["k"], case["temperature"])
    if case["op"] == "distill":
        upstream = state["upstream"] if case["train"] else None
        if own:
            from soupsuck_b200.kernels import fused_linear_distillation
            loss, mass = fused_linear_distillation(state["hidden"], state["weight"], state["indices"],
                                                   state["logits"], state["lse"],
                                                   temperature=case["temperature"], validate=False)
            if upstream is None:
                return loss, mass
            return loss.detach(), mass, torch.autograd.grad(loss, state["hidden"], upstream)[0]
        with torch.no_grad():
            return plain_distill(state["hidden"], state["weight"], state["indices"], state["logits"],
                                 state["lse"], case["temperature"], upstream)
    if own:
        from soupsuck_b200.kernels import verify_drafts
        return verify_drafts(state["target"], state["tokens"], state["uniforms"], state["noise"],
                             state["draft"], draft_lens=state["lens"])
    return plain_verify(state["target"], state["tokens"], state["uniforms"], state["noise"], state["draft"],
                        state["lens"])


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "top":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * BYTES[case["dtype"]] + case["rows"] * (case["k"] * (8 + BYTES[case["dtype"]]) + 4),
                "flops": 4 * n}
    if case["op"] == "distill":
        t, h, v, k = case["rows"], case["hidden"], case["vocab"], case["k"]
        answered = max(1, round(t * case["labelled"]))
        # Logits and, in training, the product of their gradient with the head, for the answered rows.
        flops = (4 if case["train"] else 2) * answered * h * v
        moved = v * h * 2 + answered * h * 2 + t * k * 12 + t * 8 + (t * h * 2 + t * 4 if case["train"] else 0)
        return {"bytes": moved, "flops": flops}
    b, s, v, e = case["batch"], case["drafts"], case["vocab"], BYTES[case["dtype"]]
    rows = 2 if case["sampled"] else 1
    return {"bytes": b * v * (rows * e + 4) + b * s * (2 * e + 12) + b * (s + 2) * 8, "flops": 3 * b * v}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_distill(state):
    case = state["case"]
    tau, vocab = case["temperature"], case["vocab"]
    weight = state["weight"].double()
    loss, mass, grad = [], [], []
    step = max(1, (1 << 28) // vocab)
    for a in range(0, case["rows"], step):
        x = state["hidden"][a:a + step].detach().double()
        index, t = state["indices"][a:a + step], state["logits"][a:a + step].double() / tau
        used = index >= 0
        alive = used.any(1).double()
        t = t.masked_fill(~used, -math.inf)
        if state["lse"] is None:
            p = torch.softmax(t, 1).nan_to_num(0.0)
            rest = torch.zeros_like(alive)
        else:
            p = torch.exp(t - state["lse"][a:a + step].double()[:, None])
            rest = (1.0 - p.sum(1)).clamp_min(0.0) * alive
        logq = torch.log_softmax(x @ weight.t() / tau, 1)
        column = torch.where(used, index, torch.zeros_like(index))
        logq_j = logq.gather(1, column)
        dense_p = torch.zeros_like(logq)
        member = torch.zeros_like(logq)
        row = torch.arange(len(x), device=x.device)[:, None].expand_as(index)
        dense_p.index_put_((row[used], index[used]), p[used], accumulate=True)
        member.index_put_((row[used], index[used]), torch.ones_like(p[used]))
        others = logq.masked_fill(member > 0, -math.inf)
        log_rest = torch.logsumexp(others, 1)
        kl = (torch.special.xlogy(p, p) - torch.where(p > 0, p * logq_j, 0.0)).sum(1)
        kl = kl + torch.where(rest > 0, torch.special.xlogy(rest, rest) - rest * log_rest, 0.0)
        loss.append(kl * alive)
        mass.append((logq.exp() * member).sum(1) * alive)
        if case["train"]:
            # d loss / d z = q - p on the list; q - rest * q / q_rest elsewhere.
            dz = logq.exp() - dense_p - rest[:, None] * torch.exp(others - log_rest[:, None])
            dz *= (state["upstream"][a:a + step].double() * alive / tau)[:, None]
            grad.append(dz @ weight)
    if case["train"]:
        return torch.cat(loss), torch.cat(mass), torch.cat(grad)
    return torch.cat(loss), torch.cat(mass)


def exact(case, seed):
    if case["op"] == "verify":
        return None  # whole numbers
    state = prepare(case, seed)
    if case["op"] == "distill":
        return _exact_distill(state)
    z = state["logits"].double()
    values = torch.topk(z, case["k"], dim=1).values
    return values, None, torch.logsumexp(z / case["temperature"], 1)
