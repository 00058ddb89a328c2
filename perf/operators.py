"""The serving side of the vocabulary head: cases of its operators, their plain forms and the calls a user makes.

  linear   int8_linear: hidden states quantised per token, times int8 weights with a scale per vocabulary row -> logits
  score    int8_ce_entropy: the same product reduced to cross-entropy, entropy and log-probability per row
  verify   verify_drafts: drafted tokens against the target's probabilities, from given random numbers
"""

import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # One token of one request through a small head: latency.
        _linear("linear_one_token_small", 1, 1024, 32000, "bf16", "bf16"),
        # One token through a large head: the weight is streamed once.
        _linear("linear_one_token", 1, 4096, 128256, "bf16", "fp32"),
        # A decode batch, the sampler reads bf16 logits.
        _linear("linear_decode_batch", 64, 4096, 128256, "bf16", "bf16"),
        # Odd sizes everywhere, a bias, fp16 hidden states.
        _linear("linear_odd", 37, 1000, 3001, "fp16", "fp32", bias=True),
        # Prompt tokens, logits of all of them.
        _linear("linear_prompt", 4096, 4096, 32768, "bf16", "bf16"),
        # Scoring a small model's batch.
        _score("score_small_head", 1024, 1024, 32000, "bf16"),
        # Odd sizes, a bias, ignored rows, fp16.
        _score("score_odd", 427, 1000, 3001, "fp16", bias=True, ignored=True),
        # One chunk of the large head: per-token log-probabilities of a rollout.
        _score("score_rollout", 4096, 4096, 128256, "bf16"),
        # One request, four drafted tokens.
        _verify("verify_one_request", 1, 4, False, 32000, "bf16", "fp32"),
        # A serving batch whose requests drafted zero to seven tokens each.
        _verify("verify_batch", 64, 7, True, 128256, "bf16", "fp32"),
        # Many requests, fp32 logits, bf16 draft probabilities.
        _verify("verify_many_requests", 256, 4, False, 32000, "fp32", "bf16"),
        # Drafts without probabilities (looked up in the prompt), greedy requests among the sampled ones, odd vocabulary.
        _verify("verify_lookup", 33, 5, True, 3001, "fp16", "none"),
    ]


def _linear(name, tokens, hidden, vocab, dtype, out, bias=False):
    return {"name": name, "op": "linear", "tokens": tokens, "hidden": hidden, "vocab": vocab, "dtype": dtype,
            "out": out, "bias": bias}


def _score(name, tokens, hidden, vocab, dtype, bias=False, ignored=False):
    return {"name": name, "op": "score", "tokens": tokens, "hidden": hidden, "vocab": vocab, "dtype": dtype,
            "bias": bias, "ignored": ignored}


def _verify(name, requests, drafts, ragged, vocab, dtype, probs):
    return {"name": name, "op": "verify", "requests": requests, "drafts": drafts, "ragged": ragged, "vocab": vocab,
            "dtype": dtype, "probs": probs}


def _log_range(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "score", "verify"])
    if op == "verify":
        vocab = _log_range(rng, 1000, 131072)
        drafts = rng.randint(1, 8)
        requests = _log_range(rng, 1, max(2, min(256, 40_000_000 // (vocab * (drafts + 1)))))
        case = _verify("", requests, drafts, rng.random() < 0.6, vocab, rng.choice(["bf16", "fp16", "fp32"]),
                       rng.choice(["fp32", "bf16", "none"]))
    else:
        hidden = _log_range(rng, 100, 4608)
        if rng.random() < 0.5:
            hidden = max(128, hidden // 128 * 128)
        vocab = _log_range(rng, 1000, 131072)
        tokens = _log_range(rng, 1, max(2, min(4096, 4096 * 4096 * 32768 // (hidden * vocab))))
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        if op == "linear":
            case = _linear("", tokens, hidden, vocab, dtype, rng.choice(["bf16", "fp16", "fp32"]), rng.random() < 0.3)
        else:
            case = _score("", tokens, hidden, vocab, dtype, rng.random() < 0.3, rng.random() < 0.5)
    del case["name"]
    return case


def _draft_counts(case):
    """Drafted tokens of each request: all of them, or 0 .. drafts in a fixed mix."""
    k = case["drafts"]
    return [(5 * b + 3) % (k + 1) if case["ragged"] else k for b in range(case["requests"])]


def work(case):
    if case["op"] == "verify":
        rows = sum(_draft_counts(case)) + case["requests"]
        v = case["vocab"]
        size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
        q = {"none": 0, "bf16": 2, "fp32": 4}[case["probs"]]
        # every row of logits once, one row of draft probabilities for each request
        return {"bytes": rows * v * size + case["requests"] * v * q + rows * (8 + 4 + 8 + 4),
                "flops": 4 * rows * v + 4 * case["requests"] * v}
    m, k, n = case["tokens"], case["hidden"], case["vocab"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    n_bytes = m * k * size[case["dtype"]] + n * k + 4 * n + (n * size[case["dtype"]] if case["bias"] else 0)
    n_bytes += m * n * size[case["out"]] if case["op"] == "linear" else m * (8 + 12)
    return {"bytes": n_bytes, "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    return _prepare_verify(case, dev, g) if case["op"] == "verify" else _prepare_head(case, dev, g)


def _prepare_head(case, dev, g):
    m, k, n = case["tokens"], case["hidden"], case["vocab"]
    dtype = DTYPES[case["dtype"]]
    x = torch.randn(m, k, device=dev, generator=g)
    # hidden states have a few channels that are larger than the rest
    x *= 1 + 7 * (torch.rand(k, device=dev, generator=g) < 0.01).float()
    w = torch.randn(n, k, device=dev, generator=g) / math.sqrt(k)
    codes, scale = _quantize(w)
    # rows of codes start on 16-byte boundaries, as the framework's own quantisation lays a weight out
    stored = torch.zeros(n, (k + 15) // 16 * 16, device=dev, dtype=torch.int8)[:, :k]
    stored.copy_(codes)
    state = {"case": case, "x": x.to(dtype), "codes": stored, "scale": scale, "bias": None}
    if case["bias"]:
        state["bias"] = (0.5 * torch.randn(n, device=dev, generator=g)).to(dtype)
    if case["op"] == "score":
        t = torch.randint(0, n, (m,), device=dev, generator=g)
        if case["ignored"]:
            t[torch.rand(m, device=dev, generator=g) < 0.05] = -100
        state["target"] = t
    return state


def _prepare_verify(case, dev, g):
    v, counts = case["vocab"], _draft_counts(case)
    n, b = sum(counts), len(counts)
    rows = n + b
    cu = torch.tensor([0] + counts, dtype=torch.int64).cumsum(0).to(dev)
    # a peaked row over a long tail, as a language model's logits are
    z = 2.0 * torch.randn(rows, v, device=dev, generator=g)
    hot = torch.randint(0, v, (rows, 16), device=dev, generator=g)
    z.scatter_add_(1, hot, 4 + 10 * torch.rand(rows, 16, device=dev, generator=g))
    temperature = torch.tensor([0.0, 0.6, 0.8, 1.0], device=dev)[torch.randint(0, 4, (b,), device=dev, generator=g)]
    if b == 1:
        temperature.fill_(0.8)
    counts_d = torch.tensor(counts, device=dev)
    owner = torch.repeat_interleave(torch.arange(b, device=dev), counts_d)
    draft_rows = torch.arange(n, device=dev) + owner
    # the draft model: the target's logits, off by some noise
    zd = z[draft_rows] + 0.7 * torch.randn(n, v, device=dev, generator=g)
    t = temperature[owner].clamp(min=0.3)[:, None]
    q = torch.softmax(zd / t, -1)
    if case["probs"] == "none":
        d = zd.argmax(-1) if n else torch.zeros(0, dtype=torch.int64, device=dev)
        q = None
    else:
        d = torch.multinomial(q, 1, generator=g)[:, 0] if n else torch.zeros(0, dtype=torch.int64, device=dev)
        q = q.to(DTYPES[case["probs"]])
    return {"case": case, "logits": z.to(DTYPES[case["dtype"]]), "drafts": d, "cu": cu,
            "u": torch.rand(n, device=dev, generator=g), "r": torch.rand(b, device=dev, generator=g), "q": q,
            "temperature": temperature}


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "verify":
        return _verify_plain(state)
    z = _logits_plain(state)
    if op == "linear":
        return z.to(DTYPES[state["case"]["out"]])
    t = state["target"]
    d = z - z.amax(-1, keepdim=True)
    e = d.exp()
    s = e.sum(-1)
    entropy = s.log() - (d * e).sum(-1) / s
    ce = s.log() - d.gather(1, t.clamp(min=0)[:, None])[:, 0]
    ce = torch.where(t == -100, 0.0, ce)
    return ce, entropy, -ce


def _run_own(state):
    package = os.path.join(os.getcwd(), "fast-reduction_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import fast_reduction as fr

    op = state["case"]["op"]
    if op == "verify":
        return fr.verify_drafts(state["logits"], state["drafts"], state["cu"], state["u"], state["r"],
                                draft_probs=state["q"], temperature=state["temperature"])
    if op == "linear":
        return fr.int8_linear(state["x"], state["codes"], state["scale"], bias=state["bias"],
                              out_dtype=DTYPES[state["case"]["out"]])
    return fr.int8_ce_entropy(state["x"], state["codes"], state["scale"], state["target"], bias=state["bias"])


def _quantize(x):
    """Codes of each row (as float32 whole numbers) and the row's float32 scale: max |x| / 127, the codes the whole
    numbers nearest to x / scale. The quotient is formed in 64 bits, since a rounded one can fall on a half."""
    x = x.float()
    scale = x.abs().amax(-1)
    scale = scale / torch.full_like(scale, 127.0)  # a division, not a product with a rounded 1 / 127
    wide = scale.double()[..., None]
    codes = torch.round(x.double() / torch.where(wide > 0, wide, 1.0)).float()
    return codes, scale


def _logits_plain(state):
    codes, scale = _quantize(state["x"])
    z = (codes @ state["codes"].float().t()) * scale[:, None] * state["scale"][None, :]
    return z if state["bias"] is None else z + state["bias"].float()


def _verify_plain(state):
    """In 64 bits: an accepted token or the place where a running sum passes a number is a comparison."""
    z, d, cu, q = state["logits"], state["drafts"], state["cu"], state["q"]
    rows, v = z.shape
    b, n = cu.numel() - 1, d.numel()
    dev = z.device
    first = cu[:-1] + torch.arange(b, device=dev)  # first row of each request
    count = cu[1:] - cu[:-1]
    row_owner = torch.bucketize(torch.arange(rows, device=dev), first, right=True) - 1
    owner = torch.bucketize(torch.arange(n, device=dev), cu[1:], right=True)
    greedy = state["temperature"] < 1e-6
    t = torch.where(greedy, 1.0, state["temperature"]).double()
    z = z.double()
    top = z.amax(-1, keepdim=True)
    best = torch.where(z == top, torch.arange(v, device=dev), v).amin(-1)
    x = (z - top) / t[row_owner][:, None]
    e = x.exp()
    s = e.sum(-1, keepdim=True)
    p = e / s
    logp = x - s.log()
    # which drafts pass, and how many of a request's pass in a row
    draft_row = torch.arange(n, device=dev) + owner
    qd = torch.ones(n, device=dev, dtype=torch.float64) if q is None else q.gather(1, d[:, None])[:, 0].double()
    passes = state["u"].double() * qd < p[draft_row, d]
    passes = torch.where(greedy[owner], d == best[draft_row], passes)
    place = torch.arange(n, device=dev) - cu[:-1][owner]
    accepted = count.scatter_reduce(0, owner, torch.where(passes, count[owner], place), "amin")
    # the next token of each request: from what the rejected draft leaves, or from the last row
    row = first + accepted
    w = p[row]
    rejected = accepted < count
    if n:
        at = (cu[:-1] + accepted).clamp(max=n - 1)
        if q is None:
            left = w.scatter(1, d[at][:, None], 0.0)
        else:
            left = (w - q[at].double()).clamp(min=0)
        left = torch.where(left.sum(-1, keepdim=True) > 0, left, w)
        w = torch.where(rejected[:, None], left, w)
    c = w.cumsum(-1)
    past = (c > state["r"].double()[:, None] * c[:, -1:]) & (w > 0)
    token = torch.where(past, torch.arange(v, device=dev), v).amin(-1)
    token = torch.where(greedy, best[row], token)
    # what is emitted: the accepted drafts, then that token
    i = torch.arange(rows, device=dev) - first[row_owner]
    a = accepted[row_owner]
    tokens = torch.full((rows,), -1, device=dev)
    if n:
        drafted = d[(torch.arange(rows, device=dev) - row_owner).clamp(max=n - 1)]
        tokens = torch.where(i < a, drafted, tokens)
    tokens = torch.where(i == a, token[row_owner], tokens)
    emitted = logp.gather(1, tokens.clamp(min=0)[:, None])[:, 0]
    return accepted, tokens, torch.where(tokens >= 0, emitted, 0.0).float()


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "verify":
        return _verify_exact(state)
    x = state["x"].double()
    scale = (x.abs().max(-1).values.cpu().numpy().astype(np.float32) / np.float32(127)).astype(np.float64)
    scale = torch.from_numpy(scale).to(x.device)
    ratio = x / scale[:, None]
    low = ratio.floor()
    rest = ratio - low
    codes = low + ((rest > 0.5) | ((rest == 0.5) & (low % 2 != 0))).double()
    z = torch.mm(codes, state["codes"].double().t())
    z.mul_(scale[:, None]).mul_(state["scale"].double())
    if state["bias"] is not None:
        z.add_(state["bias"].double())
    if case["op"] == "linear":
        return z
    target = state["target"]
    lse = z.logsumexp(-1)
    rows = torch.arange(z.shape[0], device=z.device)
    ce = (lse - z[rows, target.clamp(min=0)]) * (target >= 0)
    logp = z.sub_(lse[:, None])
    entropy = -(logp * logp.exp()).sum(-1)
    return ce, entropy, -ce


def _verify_exact(state):
    """Request by request, on the host."""
    z, d, cu, u, r = (state[k].cpu().double().numpy() if k in ("logits", "u", "r") else state[k].cpu().numpy()
                      for k in ("logits", "drafts", "cu", "u", "r"))
    q = None if state["q"] is None else state["q"].cpu().double().numpy()
    temperature = state["temperature"].cpu().numpy().astype(np.float64)
    accepted = np.zeros(len(cu) - 1, np.int64)
    tokens = np.full(len(z), -1, np.int64)
    logps = np.zeros(len(z), np.float64)
    for b in range(len(cu) - 1):
        t = temperature[b]
        for i in range(int(cu[b + 1] - cu[b]) + 1):
            row, at = int(cu[b]) + b + i, int(cu[b]) + i
            scaled = z[row] if t < 1e-6 else z[row] / t
            logp = scaled - scaled.max()
            logp = logp - np.log(np.sum(np.exp(logp)))
            p = np.exp(logp)
            drafted = i < cu[b + 1] - cu[b]
            if t < 1e-6:
                token = int(np.argmax(z[row]))
                passed = drafted and token == d[at]
            else:
                passed = drafted and u[at] * (1.0 if q is None else q[at][d[at]]) < p[d[at]]
                if passed:
                    token = int(d[at])
                else:
                    w = p.copy()
                    if drafted and q is None:
                        w[d[at]] = 0
                    elif drafted:
                        w = np.maximum(p - q[at], 0)
                    w = w if w.sum() > 0 else p
                    c = np.cumsum(w)
                    past = np.nonzero((c > r[b] * c[-1]) & (w > 0))[0]
                    token = int(past[0])
            tokens[row], logps[row] = token, logp[token]
            if not passed:
                break
            accepted[b] += 1
    return accepted, tokens, logps
