"""The operators over rows of logits, as they are measured: plain forms, cases and exact values.

Four calls of the package, each on rows of V logits (bf16, fp16 or fp32):

* ``logits.top_logprobs``: a teacher's k largest log-probabilities per row, with their token ids;
* ``distill.top_logprob_loss``: the distillation loss of a student's logits against such a record, and
  its gradient through autograd;
* ``distill.top_logprob_loss_and_grad``: loss and gradient of the same in one call;
* ``logits.sample``: one token per row from given uniform numbers, with temperature, top-k, top-p and min-p.

``own`` selects between the plain forms (False) and the package's calls (True).
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
MAX_K = 256


def listed():
    return [
        # The serving teacher answers one request with a token's alternatives.
        {"name": "top_one_token", "op": "top", "rows": 1, "vocab": 32000, "dtype": "bf16", "k": 20, "pad": 0, "temperature": 1.0},
        # One decoding step of a full serving batch, every request with 64 alternatives.
        {"name": "top_decode_batch", "op": "top", "rows": 64, "vocab": 128256, "dtype": "bf16", "k": 64, "pad": 0, "temperature": 1.0},
        # A short prompt scored from fp32 logits whose vocabulary is odd and padded in memory.
        {"name": "top_fp32_ragged", "op": "top", "rows": 301, "vocab": 100003, "dtype": "fp32", "k": 256, "pad": 61, "temperature": 2.0},
        # A batch of training sequences scored by a teacher.
        {"name": "top_corpus", "op": "top", "rows": 2048, "vocab": 128256, "dtype": "bf16", "k": 64, "pad": 0, "temperature": 1.0},
        # A student's small batch, loss and gradient through autograd.
        {"name": "loss_small", "op": "loss", "rows": 16, "vocab": 32000, "dtype": "bf16", "k": 8, "pad": 0, "temperature": 1.0, "tail": "drop"},
        # fp32 logits of an odd vocabulary at temperature 2, the longest teacher record, padded rows.
        {"name": "loss_fp32_odd", "op": "loss", "rows": 333, "vocab": 50001, "dtype": "fp32", "k": 256, "pad": 0, "temperature": 2.0, "tail": "renormalize"},
        # A training micro-batch of 4096 tokens through autograd: the largest case.
        {"name": "loss_training", "op": "loss", "rows": 4096, "vocab": 151936, "dtype": "bf16", "k": 32, "pad": 0, "temperature": 1.0, "tail": "renormalize"},
        # A training micro-batch of 2048 tokens, loss and gradient in one call.
        {"name": "step_training", "op": "step", "rows": 2048, "vocab": 128256, "dtype": "bf16", "k": 64, "pad": 0, "temperature": 1.0, "tail": "drop"},
        # One request decoding alone.
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": 128256, "dtype": "bf16", "pad": 0, "params": "nucleus"},
        # A decoding step of a batch whose requests all have settings of their own (greedy ones among them).
        {"name": "sample_mixed_batch", "op": "sample", "rows": 128, "vocab": 128256, "dtype": "bf16", "pad": 0, "params": "mixed"},
        # Rollouts of a student: no truncation, fp32 logits.
        {"name": "sample_rollout", "op": "sample", "rows": 256, "vocab": 151936, "dtype": "fp32", "pad": 0, "params": "free"},
        # Rollouts with top-k and top-p over an odd vocabulary in fp16.
        {"name": "sample_topk_large", "op": "sample", "rows": 1024, "vocab": 100003, "dtype": "fp16", "pad": 0, "params": "topk"},
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["top", "top", "loss", "loss", "step", "sample", "sample"])
    vocab = _log_uniform(rng, 1000, 160000)
    most = {"top": 2048 * 128256, "loss": 4096 * 128256, "step": 2048 * 128256, "sample": 1024 * 100003}[op]
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    case = {"op": op, "rows": _log_uniform(rng, 1, min(4096, most * 2 // SIZE[dtype] // (vocab + 64))), "vocab": vocab,
            "dtype": dtype, "pad": rng.choice([0, 0, rng.randint(1, 64)])}
    if op == "sample":
        case["params"] = rng.choice(["nucleus", "mixed", "free", "topk", "minp"])
    else:
        case["k"] = _log_uniform(rng, 1, MAX_K)
        case["temperature"] = rng.choice([1.0, round(rng.uniform(0.5, 4.0), 3)])
    if op in ("loss", "step"):
        case["tail"] = rng.choice(["drop", "renormalize"])
    return case


def _rows(case, gen, seed_peaks=(13.0, 24.0), peaks=64):
    """Rows of logits as a language model gives them: noise over the whole vocabulary, and some tokens that stand out, more
    in one row than in another."""
    rows, vocab, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    buffer = torch.empty(rows, vocab + case["pad"], dtype=dtype, device="cuda")
    step = max(1, (1 << 26) // buffer.shape[1])
    for at in range(0, rows, step):  # in pieces: the fp32 noise of the largest case would not be small
        part = buffer[at : at + step]
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda") * 1.5)
    logits = buffer[:, :vocab]
    count = min(peaks, vocab)
    ids = _distinct(rows, count, vocab, gen)
    low, high = seed_peaks
    heights = low + (high - low) * torch.rand(rows, 1, generator=gen, device="cuda")
    falls = torch.cumsum(torch.rand(rows, count, generator=gen, device="cuda") * 0.5, 1)
    logits.scatter_(1, ids, (heights - falls).to(dtype))
    return logits, ids


def _distinct(rows, count, vocab, gen):
    """`count` different token ids for each row."""
    start = torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda")
    stride = torch.randint(1, vocab // count + 1, (rows, 1), generator=gen, device="cuda")
    return (start + stride * torch.arange(count, device="cuda")) % vocab


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 1_000_003 + 17)
    op, rows, vocab = case["op"], case["rows"], case["vocab"]
    state = {"case": dict(case)}
    if op == "top":
        state["logits"], _ = _rows(case, gen)
    elif op in ("loss", "step"):
        k = min(case["k"], vocab)
        # The student knows some of the teacher's tokens already.
        state["logits"], known = _rows(case, gen, peaks=max(1, k // 2))
        ids = _distinct(rows, k, vocab, gen)
        agree = torch.rand(rows, 1, generator=gen, device="cuda") < 0.5
        first = torch.where(agree, known, ids[:, : known.shape[1]])
        rest = ids[:, known.shape[1] :]
        state["ids"] = torch.cat([first, rest], 1).contiguous()  # a token may come twice in a row
        score = torch.randn(rows, k, generator=gen, device="cuda") * 2 - 0.1 * torch.arange(k, device="cuda")
        mass = 0.8 + 0.199 * torch.rand(rows, 1, generator=gen, device="cuda")
        logprobs = torch.log_softmax(score, 1) + mass.log()
        # Some rows have fewer than k alternatives on record.
        kept = torch.randint(max(1, k // 2), 2 * k + 1, (rows, 1), generator=gen, device="cuda")
        gone = torch.arange(k, device="cuda") >= kept
        state["ids"][gone] = -1
        state["logprobs"] = logprobs.masked_fill(gone, -math.inf).contiguous()
        # A tenth of the rows is padding behind the sequences' ends.
        alive = torch.rand(rows, generator=gen, device="cuda") < 0.9
        alive[0] = True
        state["weights"] = alive.float() / rows
        state["grad_out"] = 0.5 + torch.rand(rows, generator=gen, device="cuda")
        if op == "loss":
            state["logits"].requires_grad_(True)
    else:
        state["logits"], _ = _rows(case, gen)
        state["uniform"] = torch.rand(rows, generator=gen, device="cuda")
        state["params"] = _params(case, gen)
    return state


def _params(case, gen):
    """Sampling settings: plain numbers for all rows, or a tensor with one value for each row."""
    kind, rows = case["params"], case["rows"]
    if kind == "free":
        return {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
    if kind == "nucleus":
        return {"temperature": 0.7, "top_k": 0, "top_p": 0.9, "min_p": 0.0}
    if kind == "topk":
        return {"temperature": 1.0, "top_k": 50, "top_p": 0.95, "min_p": 0.0}
    if kind == "minp":
        return {"temperature": 1.2, "top_k": 0, "top_p": 1.0, "min_p": 0.05}

    def pick(values, dtype):
        at = torch.randint(0, len(values), (rows,), generator=gen, device="cuda")
        return torch.tensor(values, dtype=dtype, device="cuda")[at]

    return {
        "temperature": pick([0.0, 0.3, 0.7, 1.0, 1.0, 1.3], torch.float32),
        "top_k": pick([0, 0, 1, 20, 50, 1000], torch.int32),
        "top_p": pick([1.0, 1.0, 0.5, 0.9, 0.95], torch.float32),
        "min_p": pick([0.0, 0.0, 0.0, 0.05, 0.1], torch.float32),
    }


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        from warpshift_b200 import distill, logits

        if op == "top":
            top = logits.top_logprobs(state["logits"], min(case["k"], case["vocab"]), temperature=case["temperature"])
            return {"ids": top.ids, "logprobs": top.logprobs}
        if op == "loss":
            loss = distill.top_logprob_loss(state["logits"], state["ids"], state["logprobs"], weights=state["weights"],
                                            temperature=case["temperature"], tail=case["tail"])
            (grad,) = torch.autograd.grad(loss, state["logits"], state["grad_out"])
            return {"loss": loss, "grad": grad}
        if op == "step":
            loss, grad = distill.top_logprob_loss_and_grad(state["logits"], state["ids"], state["logprobs"], weights=state["weights"],
                                                           temperature=case["temperature"], tail=case["tail"])
            return {"loss": loss, "grad": grad}
        drawn = logits.sample(state["logits"], state["uniform"], **state["params"])
        return {"tokens": drawn.tokens, "logprobs": drawn.logprobs}
    if op == "top":
        return _plain_top(state)
    if op == "sample":
        return _plain_sample(state)
    return _plain_loss(state)


def _plain_top(state):
    case = state["case"]
    x = state["logits"].float()
    k = min(case["k"], case["vocab"])
    # A stable sort: among equal logits the lowest token id comes first.
    values, ids = torch.sort(x, dim=1, descending=True, stable=True)
    values = values[:, :k]
    top = values[:, :1]
    total = torch.exp((x - top) / case["temperature"]).sum(1, keepdim=True)
    return {"ids": ids[:, :k].contiguous(), "logprobs": (values - top) / case["temperature"] - total.log()}


def _plain_loss(state):
    case = state["case"]
    logits = state["logits"].detach()
    x = logits.float() / case["temperature"]
    top = x.max(1, keepdim=True).values
    weight = torch.exp(x - top)
    total = weight.sum(1, keepdim=True)
    ids, logprobs = state["ids"], state["logprobs"]
    there = (ids >= 0) & (logprobs > -math.inf)
    at = torch.where(there, ids, 0)
    q = torch.where(there, logprobs.exp(), 0.0)
    if case["tail"] == "renormalize":
        q = q / q.sum(1, keepdim=True)
    mass = q.sum(1, keepdim=True)
    log_q = torch.where(there, q, 1.0).log()
    w = state["weights"]
    loss = w * (q * (log_q - (x.gather(1, at) - top) + total.log())).sum(1)
    scale = w / case["temperature"]
    if case["op"] == "loss":
        scale = scale * state["grad_out"]
    scale = scale[:, None]
    grad = weight * (scale * mass / total)
    grad.scatter_add_(1, at, -scale * q)
    return {"loss": loss, "grad": grad.to(logits.dtype)}


def _plain_sample(state):
    # In 64 bits: a token changes where a cumulative sum over the vocabulary passes a border.
    x = state["logits"].double()
    rows, vocab = x.shape

    def each(name, dtype):
        v = state["params"][name]
        v = v if isinstance(v, torch.Tensor) else torch.full((rows,), v, dtype=dtype, device="cuda")
        return v[:, None]

    t, top_k = each("temperature", torch.float32).double(), each("top_k", torch.int32).long()
    top_p, min_p = each("top_p", torch.float32).double(), each("min_p", torch.float32).double()
    greedy = t <= 0
    t = torch.where(greedy, 1.0, t)
    ordered, ids = torch.sort(x, dim=1, descending=True, stable=True)
    weight = torch.exp((ordered - ordered[:, :1]) / t)
    total = weight.sum(1)
    place = torch.arange(vocab, device="cuda")
    keep = (place < torch.where(top_k > 0, top_k, vocab)) & ((place < 1) | ~greedy)
    before = torch.cumsum(weight, 1) - weight
    reach = torch.where(keep, weight, 0.0).sum(1, keepdim=True)
    keep &= (before < top_p * reach) | (top_p >= 1) | (place < 1)
    keep &= (weight >= min_p) | (place < 1)
    # Back in the order of the token ids; the first whose cumulative weight is above u times the total.
    kept = torch.zeros_like(x).scatter_(1, ids, torch.where(keep, weight, 0.0))
    cumulative = torch.cumsum(kept, 1)
    tokens = torch.searchsorted(cumulative, state["uniform"].double()[:, None] * cumulative[:, -1:], right=True)
    chosen = x.gather(1, tokens)
    return {"tokens": tokens[:, 0], "logprobs": (((chosen - ordered[:, :1]) / t)[:, 0] - total.log()).float()}


def work(case):
    rows, vocab, size = case["rows"], case["vocab"], SIZE[case["dtype"]]
    row = vocab * size
    if case["op"] == "top":
        k = min(case["k"], vocab)
        return {"bytes": rows * (row + 12 * k), "flops": 4 * rows * vocab}
    if case["op"] == "sample":
        return {"bytes": rows * (row + 16), "flops": 4 * rows * vocab}
    # The logits are read once and the gradient is written once; the record (id and log-probability), the weights and the loss.
    return {"bytes": rows * (2 * row + 12 * min(case["k"], vocab) + 12), "flops": 8 * rows * vocab}


def exact(case, seed):
    state = prepare(case, seed)
    op, rows, vocab = case["op"], case["rows"], case["vocab"]
    logits = state["logits"].detach()
    if op == "sample" and rows > 1100:
        return None
    step = max(1, (1 << 25) // vocab)
    pieces = []
    for at in range(0, rows, step):
        part = slice(at, min(rows, at + step))
        x = logits[part].to(torch.float64)
        if op == "top":
            logp = torch.log_softmax(x / case["temperature"], 1)
            pieces.append((logp.topk(min(case["k"], vocab), dim=1).values,))
        elif op == "sample":
            pieces.append((torch.stack([_exact_sample(x[r], {n: float(v[at + r]) if isinstance(v, torch.Tensor) else v
                                                              for n, v in state["params"].items()},
                                                      float(state["uniform"][at + r])) for r in range(x.shape[0])]),))
        else:
            pieces.append(_exact_loss(case, x, state, part))
    out = [torch.cat(p) for p in zip(*pieces)]
    if op == "top":
        return {"ids": None, "logprobs": out[0]}
    if op == "sample":
        return {"tokens": None, "logprobs": out[0]}
    return {"loss": out[0], "grad": out[1]}


def _exact_loss(case, x, state, part):
    """Sum over the record of q (log q - log p), by autograd in 64 bits."""
    x = x.clone().requires_grad_(True)
    logp = torch.log_softmax(x / case["temperature"], 1)
    ids, lp = state["ids"][part], state["logprobs"][part].double()
    lp = lp.masked_fill(ids < 0, -math.inf)
    if case["tail"] == "renormalize":
        lp = lp - torch.logsumexp(lp, 1, keepdim=True)
    q = lp.exp()
    terms = q * (lp.nan_to_num(neginf=0.0) - logp.gather(1, ids.clamp(min=0)))
    loss = state["weights"][part].double() * terms.sum(1)
    out = state["grad_out"][part].double() if case["op"] == "loss" else torch.ones_like(loss)
    (grad,) = torch.autograd.grad(loss, x, out)
    return loss.detach(), grad


def _exact_sample(row, params, u):
    """One row by thresholds in place of a sort of the kept tokens: the drawn token's log-probability."""
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731
    t, top_p, min_p, top_k = f32(params["temperature"]), f32(params["top_p"]), f32(params["min_p"]), int(params["top_k"])
    if t <= 0:
        return torch.log_softmax(row, 0).max()
    z = row / t
    p = torch.softmax(z, 0)
    keep = torch.ones_like(p, dtype=torch.bool)
    if 0 < top_k < row.numel():
        edge = row.topk(top_k).values[-1]
        above, level = row > edge, row == edge
        keep = above | (level & (torch.cumsum(level, 0) <= top_k - above.sum()))
    if top_p < 1:
        values, counts = torch.unique(row[keep], return_counts=True)  # ascending
        mass = (torch.exp((values - row.max()) / t) * counts).flip(0)
        level = int(torch.searchsorted(torch.cumsum(mass, 0), top_p * mass.sum()))
        edge = values.flip(0)[level]
        one = torch.exp((edge - row.max()) / t)
        left = top_p * mass.sum() - mass[:level].sum()
        count = max(1, int(torch.ceil(left / one)))
        ties = keep & (row == edge)
        keep = (keep & (row > edge)) | (ties & (torch.cumsum(ties, 0) <= count))
    if min_p > 0:
        keep = keep & (p >= min(min_p, 1.0) * p.max())
    w = torch.where(keep, torch.exp(z - z.max()), 0.0)
    c = torch.cumsum(w, 0)
    token = int((c > u * c[-1]).int().argmax())
    return torch.log_softmax(z, 0)[token]
