"""The logit operators, as cases to measure: what scores a model's tokens and
what distils one model into another.

* ``scores``: log probabilities of given tokens, entropy and the top
  alternatives of every row of logits; ``scores_grad`` its gradient;
  ``scores_step`` both in one call.
* ``distill``: the divergence of a student's distribution from a teacher's top
  logits; ``distill_grad`` its gradient; ``distill_step`` both in one call.

Rows of logits may be f32, f16 or bf16 and lie further apart than the
vocabulary is long; -inf masks an entry out.  A negative token is ignored, as
is a teacher entry with a negative id.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
INF = float("inf")


def case(op, n, vocab, dtype, name=None, pad=0, masked=False, top=0, entropy=False, temperature=1.0, ids="int32"):
    c = {"op": op, "n": n, "vocab": vocab, "dtype": dtype, "pad": pad, "masked": masked}
    if op == "scores":
        c["top"] = top
    elif op.startswith("scores"):
        c["entropy"] = entropy
    else:
        c["top"], c["temperature"] = top, temperature
    c["ids"] = ids
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one position of a decode loop: what its token cost and what else was likely
        case("scores", 1, 32000, "f32", "score one position", top=5, ids="int64"),
        # a codec chunk of 1,024 positions: code lengths, and the lists a student is distilled from
        case("scores", 1024, 128256, "f32", "score a chunk", top=20, ids="int64"),
        # a few rows under a grammar's mask, in a padded batch of half logits
        case("scores_grad", 24, 10003, "f16", "gradient of masked rows", pad=5, masked=True, ids="int64"),
        # policy training: log probabilities weighted by advantages, and an entropy bonus
        case("scores_grad", 1024, 32000, "bf16", "policy gradient", entropy=True, ids="int64"),
        # fine-tuning on the data to compress, a small ragged batch: the code length and its gradient
        case("scores_step", 317, 10003, "f32", "code length step, odd", masked=True, ids="int64"),
        # the same at a large batch and vocabulary
        case("scores_step", 4096, 128256, "bf16", "code length step", ids="int64"),
        # how far a quantised model is from its source on a short text
        case("distill", 16, 151936, "f32", "divergence, short", top=20),
        # and on a codec chunk
        case("distill", 1024, 128256, "f32", "divergence, chunk", top=50),
        # gradients of an odd batch under a raised temperature, as after a checkpointed forward
        case("distill_grad", 511, 10003, "bf16", "distillation gradient, odd", top=8, temperature=2.0, ids="int64"),
        case("distill_grad", 1024, 151936, "bf16", "distillation gradient", top=20),
        # a training step's smallest batch
        case("distill_step", 8, 32000, "f32", "distillation step, small", top=64),
        # and its largest
        case("distill_step", 4096, 151936, "bf16", "distillation step", top=50, temperature=2.0),
    ]


def draw(rng):
    op = rng.choice(["scores", "scores", "scores_grad", "scores_step", "distill", "distill_grad", "distill_step"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if rng.random() < 0.3:
        vocab = rng.choice([1024, 10003, 32000, 128256, 151936])
    else:
        vocab = round(math.exp(rng.uniform(math.log(300), math.log(160000))))
    most = min(4096, 500_000_000 // (SIZE[dtype] * vocab))
    n = round(math.exp(rng.uniform(0.0, math.log(most))))
    pad = rng.choice([0, 0, 1, 3, 8, 61])
    masked = rng.random() < 0.3
    ids = rng.choice(["int32", "int64"])
    if op == "scores":
        return case(op, n, vocab, dtype, pad=pad, masked=masked, top=rng.choice([0, 1, 5, rng.randint(2, 40), rng.randint(2, 128)]), ids=ids)
    if op.startswith("scores"):
        return case(op, n, vocab, dtype, pad=pad, masked=masked, entropy=rng.random() < 0.5, ids=ids)
    return case(op, n, vocab, dtype, pad=pad, masked=masked, top=rng.choice([1, 8, rng.randint(2, 64), rng.randint(2, 128)]),
                temperature=rng.choice([1.0, 1.0, 0.7, 2.0, 4.0]), ids=ids)


# ---- inputs --------------------------------------------------------------------


def _logits(n, vocab, gen):
    """Rows as a trained model gives them: a broad bell, with a few tokens far
    above it (more of them, and less far, where the model is unsure)."""
    x = torch.randn(n, vocab, generator=gen, device="cuda")
    x.mul_(2.2)
    sure = torch.rand(n, 1, generator=gen, device="cuda") * 9.0
    at = torch.randint(0, vocab, (n, 12), generator=gen, device="cuda")
    lift = sure * torch.rand(n, 12, generator=gen, device="cuda") + 4.0
    x.scatter_add_(1, at, lift)
    return x


def prepare(c, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    n, vocab = c["n"], c["vocab"]
    state = {"case": c}
    x = _logits(n, vocab, gen)
    store = torch.zeros(n, vocab + c["pad"], dtype=DTYPES[c["dtype"]], device="cuda")
    logits = store[:, :vocab]
    logits.copy_(x)
    if c["masked"]:
        logits.masked_fill_(torch.rand(n, vocab, generator=gen, device="cuda") < 0.4, -INF)
        if n > 2:
            logits[n // 3] = -INF  # nothing is left
            logits[n // 2, 3:] = -INF  # next to nothing is
    state["logits"] = logits
    idtype = torch.int64 if c["ids"] == "int64" else torch.int32
    if c["op"].startswith("scores"):
        tokens = torch.multinomial(torch.softmax(x[:, : min(vocab, 1 << 18)], 1), 1, generator=gen)[:, 0]
        if n > 4:
            tokens[torch.rand(n, generator=gen, device="cuda") < 0.05] = -100  # padding of the batch
        state["tokens"] = tokens.to(idtype)
        if c["op"] != "scores":
            state["grad_logprob"] = torch.randn(n, generator=gen, device="cuda") / n
            state["grad_entropy"] = torch.full((n,), 0.01 / n, device="cuda") if c["entropy"] else None
    else:
        k = c["top"]
        # the teacher agrees with the student up to some noise
        x.mul_(0.9).add_(torch.randn(n, vocab, generator=gen, device="cuda"))
        teacher, ids = torch.topk(x, k, dim=1)
        if k > 3:  # lists of different lengths
            ids[(torch.rand(n, 1, generator=gen, device="cuda") < 0.2) & (torch.arange(k, device="cuda") >= k // 2)] = -1
        if n > 4:
            ids[n // 4] = -1  # a row of padding
        state["ids"], state["teacher"] = ids.to(idtype), teacher
        if c["op"] != "distill":
            state["grad_loss"] = torch.rand(n, generator=gen, device="cuda") / n
    del x
    if c["op"].endswith("_grad"):  # what the forward left
        state["stats"] = _stats(logits.float(), c.get("temperature", 1.0))
    return state


# ---- the plain forms -------------------------------------------------------------


def _stats(x, temperature):
    """Of each row: its maximum, the sum of exp((x - maximum) / T), that sum
    weighted by (x - maximum) / T, and the logarithm of the first sum."""
    m = x.amax(dim=1)
    d = (x - torch.where(m == -INF, 0.0, m)[:, None]) / temperature
    e = torch.exp(d)
    s = e.sum(dim=1)
    s1 = (e * torch.where(d == -INF, 0.0, d)).sum(dim=1)
    return torch.stack([m, s, s1, torch.log(s)], dim=1)


def _probabilities(x, stats, temperature):
    """p and log p; an empty row has none of either."""
    m, s, log_s = stats[:, 0], stats[:, 1], stats[:, 3]
    full = m != -INF
    d = (x - torch.where(full, m, 0.0)[:, None]) / temperature
    p = torch.where(full[:, None], torch.exp(d) / torch.where(full, s, 1.0)[:, None], 0.0)
    return p, d - log_s[:, None]


def _top(x, k):
    """The k largest of each row, equal values in the order of their index."""
    bits = (x + 0.0).view(torch.int32).to(torch.int64)
    order = torch.where(bits >= 0, bits, -2147483648 - bits)
    index = torch.arange(x.shape[1], device=x.device)
    best = torch.topk(order * (1 << 20) + ((1 << 20) - 1 - index), k, dim=1).values
    return (1 << 20) - 1 - (best & ((1 << 20) - 1))


def _scores(x, tokens, top, stats):
    m, s, s1, log_s = stats.unbind(1)
    full = m != -INF
    token = tokens.to(torch.int64).clamp(min=0)
    logprob = x.gather(1, token[:, None])[:, 0] - m - log_s
    logprob = torch.where(tokens < 0, 0.0, torch.where(full, logprob, -INF))
    entropy = torch.where(full, log_s - s1 / torch.where(full, s, 1.0), 0.0)
    out = {"logprob": logprob, "entropy": entropy, "stats": stats}
    if top:
        ids = _top(x, top)
        values = x.gather(1, ids)
        out["top_ids"] = ids.to(torch.int32)
        out["top_logprobs"] = torch.where(full[:, None], values - m[:, None] - log_s[:, None], -INF)
    return out


def _scores_grad(x, tokens, stats, grad_logprob, grad_entropy):
    m, s, s1, log_s = stats.unbind(1)
    full = m != -INF
    p, log_p = _probabilities(x, stats, 1.0)
    g = torch.where(full & (tokens >= 0), grad_logprob, 0.0)
    grad = -g[:, None] * p
    if grad_entropy is not None:
        entropy = log_s - s1 / torch.where(full, s, 1.0)
        grad = grad - torch.where(p > 0, grad_entropy[:, None] * p * (log_p + entropy[:, None]), 0.0)
    return grad.scatter_add(1, tokens.to(torch.int64).clamp(min=0)[:, None], g[:, None])


def _teacher(ids, teacher, temperature):
    valid = (ids >= 0) & (teacher > -INF)
    u = torch.where(valid, teacher.float() / temperature, -INF)
    some = valid.any(dim=1)
    top = torch.where(some, u.amax(dim=1), 0.0)
    e = torch.exp(u - top[:, None])
    s = torch.where(some, e.sum(dim=1), 1.0)
    return e / s[:, None], u - top[:, None] - torch.log(s)[:, None], some


def _distill(x, ids, teacher, temperature, stats):
    q, log_q, some = _teacher(ids, teacher, temperature)
    m, log_s = stats[:, 0], stats[:, 3]
    full = m != -INF
    z = x.gather(1, ids.to(torch.int64).clamp(min=0))
    log_p = (z - torch.where(full, m, 0.0)[:, None]) / temperature - torch.where(full, log_s, 0.0)[:, None]
    loss = torch.where(q > 0, q * (log_q - log_p), 0.0).sum(dim=1)
    return {"loss": torch.where(some, loss, 0.0), "stats": stats}


def _distill_grad(x, ids, teacher, stats, grad_loss, temperature):
    q, _, some = _teacher(ids, teacher, temperature)
    live = some & (stats[:, 0] != -INF)
    g = torch.where(live, grad_loss / temperature, 0.0)
    p, _ = _probabilities(x, stats, temperature)
    return (g[:, None] * p).scatter_add(1, ids.to(torch.int64).clamp(min=0), -g[:, None] * q)


def run(state):
    c, logits = state["case"], state["logits"]
    op = c["op"]
    if own:
        from detllm_b200 import scoring

        if op == "scores":
            r = scoring.token_scores(logits, state["tokens"], top=c["top"])
            out = {"logprob": r.logprob, "entropy": r.entropy, "stats": r.stats}
            if c["top"]:
                out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
            return out
        if op == "scores_grad":
            return {"grad": scoring.token_scores_grad(logits, state["tokens"], state["stats"], state["grad_logprob"],
                                                      state["grad_entropy"])}
        if op == "scores_step":
            r, grad = scoring.token_scores_step(logits, state["tokens"], state["grad_logprob"], state["grad_entropy"])
            return {"logprob": r.logprob, "entropy": r.entropy, "stats": r.stats, "grad": grad}
        if op == "distill":
            r = scoring.distill_loss(logits, state["ids"], state["teacher"], c["temperature"])
            return {"loss": r.loss, "stats": r.stats}
        if op == "distill_grad":
            return {"grad": scoring.distill_grad(logits, state["ids"], state["teacher"], state["stats"],
                                                 state["grad_loss"], c["temperature"])}
        r, grad = scoring.distill_step(logits, state["ids"], state["teacher"], state["grad_loss"], c["temperature"])
        return {"loss": r.loss, "stats": r.stats, "grad": grad}
    x = logits.float()
    if op == "scores":
        return _scores(x, state["tokens"], c["top"], _stats(x, 1.0))
    if op == "scores_grad":
        return {"grad": _scores_grad(x, state["tokens"], state["stats"], state["grad_logprob"],
                                     state["grad_entropy"]).to(logits.dtype)}
    if op == "scores_step":
        out = _scores(x, state["tokens"], 0, _stats(x, 1.0))
        grad = _scores_grad(x, state["tokens"], out["stats"], state["grad_logprob"], state["grad_entropy"])
        return {**out, "grad": grad.to(logits.dtype)}
    if op == "distill":
        return _distill(x, state["ids"], state["teacher"], c["temperature"], _stats(x, c["temperature"]))
    if op == "distill_grad":
        return {"grad": _distill_grad(x, state["ids"], state["teacher"], state["stats"], state["grad_loss"],
                                      c["temperature"]).to(logits.dtype)}
    out = _distill(x, state["ids"], state["teacher"], c["temperature"], _stats(x, c["temperature"]))
    grad = _distill_grad(x, state["ids"], state["teacher"], out["stats"], state["grad_loss"], c["temperature"])
    return {**out, "grad": grad.to(logits.dtype)}


def work(c):
    n, vocab, size = c["n"], c["vocab"], SIZE[c["dtype"]]
    idsize = 8 if c["ids"] == "int64" else 4
    logits = n * vocab * size
    if c["op"] == "scores":
        return {"bytes": logits + n * (idsize + 24 + 8 * c["top"]), "flops": 6 * n * vocab}
    if c["op"] == "scores_grad":
        return {"bytes": 2 * logits + n * (idsize + 24), "flops": 4 * n * vocab}
    if c["op"] == "scores_step":
        return {"bytes": 2 * logits + n * (idsize + 32), "flops": 8 * n * vocab}
    lists = n * c["top"] * (idsize + 4)
    if c["op"] == "distill":
        return {"bytes": logits + lists + n * 20, "flops": 6 * n * vocab}
    if c["op"] == "distill_grad":
        return {"bytes": 2 * logits + lists + n * 20, "flops": 4 * n * vocab}
    return {"bytes": 2 * logits + lists + n * 24, "flops": 8 * n * vocab}


# ---- the definitions in 64 bits ----------------------------------------------------


def _exact_rows(c, z, s, rows):
    """exact() for some rows: z their logits in 64 bits, s the state."""
    op, temperature = c["op"], c.get("temperature", 1.0)
    z = z / temperature
    empty = torch.isneginf(z).all(dim=1, keepdim=True)
    logp = torch.log_softmax(z.masked_fill(empty, 0.0), dim=1).masked_fill(empty, -INF)
    p = logp.exp()
    plogp = (p * logp).nan_to_num(nan=0.0)  # 0 log 0 = 0
    high = (z * temperature).max(dim=1, keepdim=True).values
    weights = torch.exp((z - high / temperature).masked_fill(empty, -INF))
    total = weights.sum(dim=1)
    first = (weights * (z - high / temperature).masked_fill(weights == 0, 0.0)).sum(dim=1)
    stats = torch.stack([high[:, 0], total, first, total.log()], dim=1)
    if op.startswith("scores"):
        tok = s["tokens"][rows].long()
        seen = tok >= 0
        entropy = -plogp.sum(dim=1)
        hit = torch.zeros_like(p).scatter_(1, tok.clamp(min=0)[:, None], 1.0)
        if op != "scores":
            g = (s["grad_logprob"][rows].double() * seen)[:, None].masked_fill(empty, 0.0)
            grad = g * (hit - p)
            if s["grad_entropy"] is not None:
                grad -= s["grad_entropy"][rows].double()[:, None] * (plogp + p * entropy[:, None])
            if op == "scores_grad":
                return {"grad": grad}
        own_logp = logp.gather(1, tok.clamp(min=0)[:, None])[:, 0].masked_fill(~seen, 0.0)
        out = {"logprob": own_logp, "entropy": entropy, "stats": stats}
        if op == "scores_step":
            return {**out, "grad": grad}
        if c["top"]:
            out["top_logprobs"] = logp.sort(dim=1, descending=True).values[:, : c["top"]]
        return out
    ids = s["ids"][rows].long()
    valid = ids >= 0
    u = (s["teacher"][rows].double() / temperature).masked_fill(~valid, -INF)
    blank = ~valid.any(dim=1, keepdim=True)
    logq = torch.log_softmax(u.masked_fill(blank, 0.0), dim=1).masked_fill(~valid, -INF)
    q = logq.exp()
    if op != "distill":
        g = (s["grad_loss"][rows].double() / temperature)[:, None].masked_fill(blank | empty, 0.0)
        grad = g * (p - torch.zeros_like(p).scatter_add_(1, ids.clamp(min=0), q))
        if op == "distill_grad":
            return {"grad": grad}
    each = (q * (logq - logp.gather(1, ids.clamp(min=0)).masked_fill(~valid, 0.0))).masked_fill(~valid, 0.0)
    out = {"loss": each.sum(dim=1), "stats": stats}
    return out if op == "distill" else {**out, "grad": grad}


def exact(c, seed):
    s = prepare(c, seed)
    rows = max(1, 64_000_000 // c["vocab"])
    parts = []
    for at in range(0, c["n"], rows):
        part = slice(at, min(c["n"], at + rows))
        parts.append(_exact_rows(c, s["logits"][part].double(), s, part))
    out = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    if c["op"] == "scores" and c["top"]:
        out["top_ids"] = None
    return out
