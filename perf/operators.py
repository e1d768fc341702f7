"""Performance cases of the operators on language-model logits.

``token_logprob_fwd`` gives the log-probabilities of given tokens, the row's
entropy and its most likely alternatives, ``token_logprob_bwd`` the gradient;
``topk_distill_fwd`` the divergence of a student's logits from a teacher's top
entries, ``topk_distill_bwd`` its gradient.  All of ``credit_amd.hip_lib``.

The listed cases span the range in use: the decode step of one sequence and of
a batch, scoring and training rows of full vocabularies, odd vocabularies, both
types and each direction.  ``draw`` gives more of the same ranges.

``run`` makes the package's calls where ``own`` is true and computes the same in
elementary torch operations where it is not; ``exact`` computes it in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

F32, F64, I64 = torch.float32, torch.float64, torch.int64
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}

# Most bytes of logits of a drawn case (the largest listed ones have as many),
# its widest row and its most rows.
MOST_BYTES = 1 << 29
WIDEST, MOST_ROWS = 262144, 4096


def _logprob(name, dtype, rows, cols, tokens=1, top=0, entropy=True, temperature=1.0,
             masked=False):
    return {"name": name, "op": "logprob_fwd", "dtype": dtype, "rows": rows, "cols": cols,
            "tokens": tokens, "top": top, "entropy": entropy, "temperature": temperature,
            "masked": masked}


def _logprob_grad(name, dtype, rows, cols, tokens=1, entropy=True, temperature=1.0, padded=False):
    return {"name": name, "op": "logprob_bwd", "dtype": dtype, "rows": rows, "cols": cols,
            "tokens": tokens, "entropy": entropy, "temperature": temperature, "padded": padded}


def _distill(name, op, dtype, rows, cols, top, tail, temperature=1.0, padded=False):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "cols": cols, "top": top,
            "tail": tail, "temperature": temperature, "padded": padded}


def listed() -> list[dict]:
    return [
        # One sequence's decode step: the sampled token's log-probability and
        # the alternatives a client asks for.
        _logprob("decode_one", "f32", 1, 32768, top=8, entropy=False),
        # The same for a batch of sequences, with the entropy a monitor reads.
        _logprob("decode_batch", "bf16", 64, 131072, top=20),
        # Scoring the tokens of a prompt over an odd vocabulary whose last
        # columns are masked.
        _logprob("score_ragged", "bf16", 700, 50001, top=5, entropy=False, masked=True),
        # Ranking four candidate tokens of each position, full-width fp32 logits.
        _logprob("score_wide", "f32", 512, 262144, tokens=4),
        # A teacher's pass: what a distillation set keeps of every position.
        _logprob("teacher_top", "bf16", 2048, 131072, top=64, temperature=2.0),
        # The gradient of a policy loss with an entropy bonus.
        _logprob_grad("policy_grad", "bf16", 2048, 131072),
        # The gradient of a likelihood over an odd vocabulary, padded batch.
        _logprob_grad("likelihood_grad_ragged", "f32", 1000, 40003, entropy=False, padded=True),
        # A student's loss against the kept top entries and their tail.
        _distill("distill_tail", "distill_fwd", "bf16", 2048, 131072, 64, True, temperature=2.0),
        # The same over the top entries alone, on a few rows.
        _distill("distill_few", "distill_fwd", "f32", 16, 65536, 20, False),
        # The student's gradients: with the tail, over an odd vocabulary with a
        # padded batch, and full-width in fp32.
        _distill("distill_tail_grad", "distill_bwd", "bf16", 2048, 131072, 64, True,
                 temperature=2.0),
        _distill("distill_ragged_grad", "distill_bwd", "bf16", 500, 100003, 32, False,
                 padded=True),
        _distill("distill_wide_grad", "distill_bwd", "f32", 512, 262144, 128, True),
    ]


def _log_int(rng, low: int, high: int) -> int:
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng) -> dict:
    dtype = rng.choice(("f32", "bf16"))
    cols = _log_int(rng, 4096, WIDEST)
    if rng.random() < 0.5:  # vocabularies padded to a multiple of 64 are common
        cols -= cols % 64
    rows = _log_int(rng, 1, min(MOST_ROWS, MOST_BYTES // (cols * SIZE[dtype])))
    temperature = rng.choice((1.0, 1.0, 0.7, 2.0))
    op = rng.choice(("logprob_fwd", "logprob_fwd", "logprob_bwd", "distill_fwd", "distill_bwd"))
    if op == "logprob_fwd":
        case = _logprob("", dtype, rows, cols, rng.choice((1, 1, 4)),
                        rng.choice((0, _log_int(rng, 1, 64))), rng.random() < 0.5, temperature,
                        rng.random() < 0.25)
    elif op == "logprob_bwd":
        case = _logprob_grad("", dtype, rows, cols, rng.choice((1, 1, 4)), rng.random() < 0.5,
                             temperature, rng.random() < 0.25)
    else:
        case = _distill("", op, dtype, rows, cols, _log_int(rng, 4, 128), rng.random() < 0.5,
                        temperature, rng.random() < 0.25)
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs --


def _logits(g, case):
    """A few dozen likely tokens above a broad floor, as trained models give."""
    rows, cols = case["rows"], case["cols"]
    z = torch.randn((rows, cols), generator=g, device="cuda").mul_(2.0)
    u = torch.rand((rows, cols), generator=g, device="cuda")
    z += u.sub_(1.0 - 24.0 / cols).clamp_(min=0.0).mul_(12.0 * cols / 24.0)
    del u
    if case.get("masked"):
        z[:, cols - cols // 64:] = -math.inf
    return z


def _live_rows(case) -> int:
    """Rows in use: of a padded batch the last eighth are not."""
    return case["rows"] - (case["rows"] // 8 if case["padded"] else 0)


def _likely(g, z, n):
    """n tokens a row, drawn from the row's distribution."""
    noise = torch.empty(z.shape, device="cuda").exponential_(generator=g).log_()
    return (z - noise).topk(n, dim=1).indices if n > 1 else (z - noise).argmax(1, keepdim=True)


def _sums(z, temperature):
    """Row maximum and sum of exp((z - max) / temperature)."""
    m = z.amax(1, keepdim=True)
    return m, ((z - m) / temperature).exp().sum(1, keepdim=True)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rows, cols, temperature = case["rows"], case["cols"], case["temperature"]
    z = _logits(g, case)
    s = {"case": case, "logits": z.to(DTYPES[case["dtype"]])}
    f32 = dict(device="cuda", dtype=F32)
    if case["op"].startswith("logprob"):
        s["tokens"] = _likely(g, z, case["tokens"])
    else:
        # The teacher agrees with the student on most of what is likely.
        t = torch.randn(z.shape, generator=g, device="cuda").mul_(0.7).add_(z)
        values, s["ids"] = t.topk(case["top"], dim=1)
        if case["tail"]:
            m, total = _sums(t, temperature)
            values = (values - m) / temperature - total.log()
        s["teacher"] = values.contiguous()
        del t
    if case["op"] == "logprob_fwd":
        s["logp"] = torch.empty((rows, case["tokens"]), **f32)
        s["stats"] = torch.empty((rows, 2), **f32)
        s["entropy"] = torch.empty(rows, **f32) if case["entropy"] else None
        s["top_logp"] = torch.empty((rows, case["top"]), **f32) if case["top"] else None
        s["top_ids"] = (torch.empty((rows, case["top"]), device="cuda", dtype=I64)
                        if case["top"] else None)
        return s
    if case["op"] == "distill_fwd":
        s["loss"] = torch.empty(rows, **f32)
        s["stats"] = torch.empty((rows, 8), **f32)
    if case["padded"]:
        s["tokens" if case["op"] == "logprob_bwd" else "ids"][_live_rows(case):] = -1
    if case["op"] == "distill_fwd":
        return s
    # What the forward left.
    del z
    s["dlogits"] = torch.empty_like(s["logits"])
    if case["op"] == "logprob_bwd":
        logp, s["stats"], entropy, _, _ = _plain_logprob(s["logits"], s["tokens"], 0, True,
                                                         temperature)
        s["dlogp"] = torch.randn(s["tokens"].shape, generator=g, **f32) / rows
        s["entropy"] = entropy if case["entropy"] else None
        s["dentropy"] = (torch.randn(rows, generator=g, **f32) * (0.1 / rows)
                         if case["entropy"] else None)
        if case["entropy"]:
            s["dentropy"][_live_rows(case):] = 0.0
    else:
        _, s["stats"] = _plain_distill(s["logits"], s["ids"], s["teacher"], case["tail"],
                                       temperature)
        s["dloss"] = torch.rand(rows, generator=g, **f32) / rows
    return s


# -------------------------------------------------------------- plain form --


def _plain_logprob(logits, tokens, top, entropy, temperature):
    """logp [rows, tokens], stats (max, sum), entropy, top log-probabilities
    and columns."""
    z = logits.float()
    m, total = _sums(z, temperature)
    log_total = total.log()
    x = (z - m) / temperature - log_total
    logp = torch.where(tokens < 0, 0.0, x.gather(1, tokens.clamp(min=0)))
    h = None
    if entropy:
        p = x.exp()
        h = -torch.where(p == 0.0, 0.0, p * x).sum(1)
    values = ids = None
    if top:
        values, ids = _top(z, top)
        values = (values - m) / temperature - log_total
    return logp, torch.cat((m, total), 1), h, values, ids


def _top(z, top):
    """The largest of each row, equal ones by column."""
    values, ids = z.sort(dim=1, descending=True, stable=True)
    return values[:, :top].contiguous(), ids[:, :top].contiguous()


def _plain_logprob_grad(logits, tokens, stats, entropy, dlogp, dentropy, temperature):
    z = logits.float()
    live = tokens >= 0
    g = torch.where(live, dlogp, 0.0)
    x = (z - stats[:, :1]) / temperature - stats[:, 1:].log()
    weight = g.sum(1, keepdim=True)
    if dentropy is not None:
        weight = weight + dentropy[:, None] * (x + entropy[:, None])
    p = x.exp()
    d = torch.where(p == 0.0, 0.0, -p * weight)
    d.scatter_add_(1, tokens.clamp(min=0), g)
    return (d / temperature).to(logits.dtype)


def _teacher(ids, teacher, tail, temperature):
    """Probabilities of the live entries (0 elsewhere), of the tail, the whole
    mass, and the log-sum that normalised them."""
    live = ids >= 0
    if tail:
        q = torch.where(live, teacher.double().exp(), 0.0)
        rest = (1.0 - q.sum(1, keepdim=True)).clamp(min=0.0)
        log_sum = torch.zeros_like(rest)
    else:
        t = torch.where(live, teacher.double() / temperature, -math.inf)
        m = torch.where(live.any(1, keepdim=True), t.amax(1, keepdim=True), 0.0)
        total = (t - m).exp().sum(1, keepdim=True)
        log_sum = torch.where(total > 0.0, m + total.log(), 0.0)
        q = (t - log_sum).exp()
        rest = torch.zeros_like(log_sum)
    return q, rest, q.sum(1, keepdim=True) + rest, log_sum


def _plain_distill(logits, ids, teacher, tail, temperature):
    """loss [rows] and the stats [rows, 8] its backward takes: maximum, sum,
    maximum and sum of the tail, teacher mass, the tail's gradient, the teacher's
    log-sum, 0.  In 64 bits: the terms nearly cancel where the two agree."""
    z = logits.double()
    m, total = _sums(z, temperature)
    at = ids.clamp(min=0)
    live = ids >= 0
    q, rest, mass, log_sum = _teacher(ids, teacher, tail, temperature)
    log_p = (z.gather(1, at) - m) / temperature - total.log()
    loss = torch.where(q > 0.0, q * (q.clamp(min=1e-300).log() - log_p), 0.0).sum(1, keepdim=True)
    tail_m, tail_total, tail_grad = (torch.zeros_like(m) for _ in range(3))
    if tail:
        z = z.scatter(1, at, torch.where(live, -math.inf, z.gather(1, at)))
        tail_m, tail_total = _sums(z, temperature)
        log_tail = (tail_m - m) / temperature + tail_total.log() - total.log()
        loss = loss + torch.where(rest > 0.0, rest * (rest.clamp(min=1e-300).log() - log_tail),
                                  0.0)
        tail_grad = mass * log_tail.exp() - rest
    used = live.any(1, keepdim=True)
    stats = torch.cat((m, total, tail_m, tail_total, mass, tail_grad, log_sum,
                       torch.zeros_like(m)), 1)
    return torch.where(used, loss, 0.0)[:, 0].float(), torch.where(used, stats, 0.0).float()


def _plain_distill_grad(logits, ids, teacher, stats, dloss, tail, temperature):
    z = logits.float()
    live = ids >= 0
    q = torch.where(live, _teacher(ids, teacher, tail, temperature)[0].float(), 0.0)
    m, total, tail_m, tail_total, mass, tail_grad, _, _ = stats.split(1, 1)
    at = ids.clamp(min=0)
    p = ((z.gather(1, at) - m) / temperature).exp() / total
    if tail:
        d = ((z - tail_m) / temperature).exp() * (tail_grad / tail_total)
    else:
        d = ((z - m) / temperature).exp() * (mass / total)
    # A row's entries name different columns and are all there or all absent.
    d.scatter_(1, at, torch.where(live, p * mass - q, d.gather(1, at)))
    d = torch.where(live.any(1, keepdim=True), d * (dloss[:, None] / temperature), 0.0)
    return d.to(logits.dtype)


def run(s: dict):
    case, temperature = s["case"], s["case"]["temperature"]
    op = case["op"]
    if own:
        from credit_amd import hip_lib

        if op == "logprob_fwd":
            hip_lib.token_logprob_fwd(s["logits"], s["tokens"], s["logp"], s["stats"],
                                      entropy=s["entropy"], top_logp=s["top_logp"],
                                      top_ids=s["top_ids"], temperature=temperature)
            return s["logp"], s["stats"], s["entropy"], s["top_logp"], s["top_ids"]
        if op == "logprob_bwd":
            hip_lib.token_logprob_bwd(s["logits"], s["tokens"], s["stats"], s["dlogp"],
                                      s["dlogits"], entropy=s["entropy"],
                                      dentropy=s["dentropy"], temperature=temperature)
            return s["dlogits"]
        if op == "distill_fwd":
            hip_lib.topk_distill_fwd(s["logits"], s["ids"], s["teacher"], s["loss"], s["stats"],
                                     tail=case["tail"], temperature=temperature)
            return s["loss"], s["stats"]
        hip_lib.topk_distill_bwd(s["logits"], s["ids"], s["teacher"], s["stats"], s["dloss"],
                                 s["dlogits"], tail=case["tail"], temperature=temperature)
        return s["dlogits"]
    if op == "logprob_fwd":
        return _plain_logprob(s["logits"], s["tokens"], case["top"], case["entropy"], temperature)
    if op == "logprob_bwd":
        return _plain_logprob_grad(s["logits"], s["tokens"], s["stats"], s["entropy"], s["dlogp"],
                                   s["dentropy"], temperature)
    if op == "distill_fwd":
        return _plain_distill(s["logits"], s["ids"], s["teacher"], case["tail"], temperature)
    return _plain_distill_grad(s["logits"], s["ids"], s["teacher"], s["stats"], s["dloss"],
                               case["tail"], temperature)


def work(case: dict) -> dict:
    rows, cols = case["rows"], case["cols"]
    logits = rows * cols * SIZE[case["dtype"]]
    if case["op"] == "logprob_fwd":
        row = case["tokens"] * 12 + 8 + 4 * case["entropy"] + 12 * case["top"]
        return {"bytes": logits + rows * row, "flops": rows * cols * (6 if case["entropy"] else 4)}
    live = _live_rows(case)
    share = live / rows
    if case["op"] == "logprob_bwd":
        row = case["tokens"] * 12 + 8 + 8 * case["entropy"]
        return {"bytes": logits * (1 + share) + rows * row,
                "flops": live * cols * (6 if case["entropy"] else 4)}
    row = 12 * case["top"] + 36
    if case["op"] == "distill_fwd":
        return {"bytes": logits * share + rows * row, "flops": live * cols * 4}
    return {"bytes": logits * (1 + share) + rows * row, "flops": live * cols * 4}


# ------------------------------------------------------------------- exact --


def _by_rows(fn, *tensors):
    """fn over blocks of rows (None stays None), its results joined."""
    rows, cols = tensors[0].shape
    step = max(1, (1 << 27) // cols)
    parts = [fn(*(None if t is None else t[i:i + step] for t in tensors))
             for i in range(0, rows, step)]
    if isinstance(parts[0], torch.Tensor):
        return torch.cat(parts)
    return tuple(None if p[0] is None else torch.cat(p) for p in zip(*parts))


def _exact_logprob(case, z, tokens):
    z = z.double()
    lp = torch.log_softmax(z / case["temperature"], dim=1)
    m = z.amax(1, keepdim=True)
    stats = torch.cat((m, (torch.logsumexp(z / case["temperature"], 1, keepdim=True)
                           - m / case["temperature"]).exp()), 1)
    h = torch.special.entr(lp.exp()).sum(1) if case["entropy"] else None
    top = lp.topk(case["top"], dim=1).values if case["top"] else None
    return lp.gather(1, tokens), stats, h, top


def _exact_grad(z, tokens, dlogp, dentropy, temperature):
    """The gradient of sum_t dlogp_t logp_t + dentropy H by the chain rule
    through log_softmax: with u the gradient for lp, u - p sum(u)."""
    lp = torch.log_softmax(z.double() / temperature, dim=1)
    p = lp.exp()
    u = torch.zeros_like(lp)
    u.scatter_add_(1, tokens.clamp(min=0), dlogp.double() * (tokens >= 0))
    if dentropy is not None:
        u -= dentropy.double()[:, None] * p * (lp + 1.0)
    return (u - p * u.sum(1, keepdim=True)) / temperature


def _exact_q(case, ids, teacher):
    t = teacher.double()
    if case["tail"]:
        q = t.exp() * (ids >= 0)
        return q, (1.0 - q.sum(1)).clamp(min=0.0)
    t = (t / case["temperature"]).masked_fill(ids < 0, -math.inf)
    return torch.nan_to_num(torch.softmax(t, dim=1)), torch.zeros_like(t[:, 0])


def _exact_distill(case, z, ids, teacher):
    z = z.double() / case["temperature"]
    lse = z.logsumexp(1)
    q, rest = _exact_q(case, ids, teacher)
    at = ids.clamp(min=0)
    loss = (torch.xlogy(q, q) - q * (z.gather(1, at) - lse[:, None])).sum(1)
    if case["tail"]:
        outside = z.scatter(1, at, z.gather(1, at).masked_fill(ids >= 0, -math.inf))
        loss += torch.xlogy(rest, rest) - rest * (outside.logsumexp(1) - lse)
    return loss * (ids >= 0).any(1)


def _exact_distill_grad(case, z, ids, teacher, dloss):
    z = z.double() / case["temperature"]
    q, rest = _exact_q(case, ids, teacher)
    target = torch.zeros_like(z).scatter_add_(1, ids.clamp(min=0), q)
    if case["tail"]:
        at = ids.clamp(min=0)
        outside = z.scatter(1, at, z.gather(1, at).masked_fill(ids >= 0, -math.inf))
        target += rest[:, None] * torch.softmax(outside, dim=1)
    d = torch.softmax(z, dim=1) * target.sum(1, keepdim=True) - target
    used = (ids >= 0).any(1, keepdim=True)
    return d * used * (dloss.double()[:, None] / case["temperature"])


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    op, temperature = case["op"], case["temperature"]
    if op == "logprob_fwd":
        logp, stats, h, top = _by_rows(lambda z, t: _exact_logprob(case, z, t), s["logits"],
                                       s["tokens"])
        return logp, stats, h, top, None
    if op == "logprob_bwd":
        return _by_rows(lambda z, t, g, h: _exact_grad(z, t, g, h, temperature), s["logits"],
                        s["tokens"], s["dlogp"], s["dentropy"])
    if op == "distill_fwd":
        return _by_rows(lambda z, i, t: _exact_distill(case, z, i, t), s["logits"], s["ids"],
                        s["teacher"]), None
    return _by_rows(lambda z, i, t, g: _exact_distill_grad(case, z, i, t, g), s["logits"],
                    s["ids"], s["teacher"], s["dloss"])
