"""The operators of a decode step around the coded projections, with the sizes they are measured at.

Three operators, each as elementary torch operations in fp32 (the plain form) and through the package's entry points:

  adapters   vllm_espalier_b200.adapters.Adapters: low-rank adapters of many requests beside a shared projection,
             out[t] = y[t] + scale[a] (x[t] A[a, s]^T) B[a, s]^T with a = ids[t], for every matrix s of the layer
  norm       vllm_espalier_b200.norms.BlockNorm: the norm after a block, its gate, the scaled residual add and the
             norm before the next block
  verify     vllm_espalier_b200.speculative.verify: drafted tokens against the target's probabilities, and the token
             after the last accepted one, from given random numbers

Shapes are those of the decoder the package's benchmark runs (hidden size 2048, a fused q/k/v projection of
4096 + 512 + 512 columns, an output projection 4096 -> 2048, a vocabulary of 248320, three drafted tokens a request)
and ordinary serving batches around them.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
HIDDEN, QKV, O_IN, VOCAB = 2048, (4096, 512, 512), 4096, 248320
EPS = 1e-6
ACCEPTED = 0.6      # about the share of drafted tokens that the verification inputs below accept


def listed():
    adapters = {"op": "adapters", "dtype": "bf16", "k": HIDDEN, "q": 4096, "kv": 512}
    norm = {"op": "norm", "kind": "rms", "dtype": "bf16", "residual": "bf16", "d": HIDDEN, "two": False, "post": False,
            "gate": "none", "act": "none"}
    verify = {"op": "verify", "dtype": "bf16", "vocab": VOCAB, "drafts": 3, "probs": "none", "padding": 0}
    return [
        # one request decoding alone: the latency of the q/k/v adapter beside one token's projection
        {"name": "adapters 1 token", **adapters, "tokens": 1, "slots": 4, "rank": 16, "order": "requests",
         "requests": 1},
        # a decode batch in which nearly every row has an adapter of its own
        {"name": "adapters 48 tokens mixed", **adapters, "tokens": 48, "slots": 64, "rank": 32, "order": "mixed",
         "requests": 48},
        # a drafted batch on the output projection, fp16, an odd number of rows in no order
        {"name": "adapters 333 tokens o", **adapters, "dtype": "f16", "k": O_IN, "q": HIDDEN, "kv": 0, "tokens": 333,
         "slots": 24, "rank": 16, "order": "mixed", "requests": 333},
        # a prefill step of a dozen prompts
        {"name": "adapters prefill rank 16", **adapters, "tokens": 8192, "slots": 16, "rank": 16, "order": "requests",
         "requests": 12},
        # a shorter ragged prefill step with wide adapters
        {"name": "adapters prefill rank 64", **adapters, "tokens": 3001, "slots": 8, "rank": 64, "order": "requests",
         "requests": 5},
        # one token's norm between two blocks
        {"name": "norm 1 row", **norm, "rows": 1},
        # the norm after the experts' two outputs, a verification batch of eight requests
        {"name": "norm 32 rows experts", **norm, "rows": 32, "two": True, "post": True, "gate": "channel"},
        # an odd width that no vector load fits, a gate an element, layer norm
        {"name": "norm 1023 rows odd", **norm, "rows": 1023, "d": 2047, "kind": "layer", "dtype": "f16",
         "residual": "f16", "post": True, "gate": "element", "act": "sigmoid"},
        # a prefill step with the residual stream kept in fp32
        {"name": "norm 16384 rows", **norm, "rows": 16384, "residual": "f32", "two": True, "post": True, "gate": "row",
         "act": "tanh"},
        # one request's three drafted tokens from a greedy drafter
        {"name": "verify 1 request", **verify, "requests": 1},
        # a batch whose drafter gives its probabilities, a vocabulary cut short of the head's padded columns
        {"name": "verify 13 requests ragged", **verify, "requests": 13, "drafts": 5, "vocab": 150001, "probs": "f32",
         "padding": 19, "dtype": "f32"},
        # a full batch
        {"name": "verify 96 requests", **verify, "requests": 96, "probs": "bf16"},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(("adapters", "norm", "verify"))
    if op == "adapters":
        k, q, kv = rng.choice(((HIDDEN, 4096, 512), (O_IN, HIDDEN, 0), (1032, 1400, 136)))
        tokens = _spread(rng, 1, 8192)
        order = "mixed" if tokens <= 512 and rng.random() < 0.6 else "requests"
        return {"op": op, "dtype": rng.choice(("bf16", "f16")), "k": k, "q": q, "kv": kv, "tokens": tokens,
                "slots": _spread(rng, 1, 64), "rank": rng.choice((8, 16, 16, 32, 64)) if tokens <= 3001 else 16,
                "order": order, "requests": tokens if order == "mixed" else _spread(rng, 1, min(tokens, 40))}
    if op == "norm":
        d = rng.choice((HIDDEN, 4096, 1408, _spread(rng, 33, 8191) | 1))
        rows = _spread(rng, 1, 12000 * HIDDEN // max(d, HIDDEN))
        dtype = rng.choice(("bf16", "f16"))
        return {"op": op, "kind": rng.choice(("rms", "layer")), "dtype": dtype, "residual": rng.choice((dtype, "f32")),
                "d": d, "rows": rows, "two": rng.random() < 0.5, "post": rng.random() < 0.5,
                "gate": rng.choice(("none", "channel", "row", "element")),
                "act": rng.choice(("none", "sigmoid", "tanh"))}
    vocab = rng.choice((VOCAB, _spread(rng, 999, VOCAB)))
    drafts = rng.randint(0, 6)
    return {"op": op, "dtype": rng.choice(("bf16", "f16", "f32")), "vocab": vocab, "drafts": drafts,
            "probs": rng.choice(("none", "f32", "bf16")), "padding": rng.choice((0, 0, 1, 64)),
            "requests": _spread(rng, 1, 192 // (drafts + 1))}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _widths(case):
    return [w for w in (case["q"], case["kv"], case["kv"]) if w]


def _ranks(case):
    """The ranks of the loaded adapters: most of the full rank, some of half of it, in steps of 8."""
    r = case["rank"]
    return [r if s % 3 else max(8, r // 2 // 8 * 8) for s in range(case["slots"])]


def _prepare_adapters(case, gen):
    dev, dt = gen.device, DTYPES[case["dtype"]]
    T, K, S, r = case["tokens"], case["k"], case["slots"], case["rank"]
    widths = _widths(case)
    N = sum(widths)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, device=dev, generator=gen) * std).to(dt)

    if case["order"] == "mixed":        # a row in ten has no adapter
        ids = torch.randint(0, S, (T,), device=dev, generator=gen)
        ids = torch.where(torch.rand(T, device=dev, generator=gen) < 0.1, -1, ids)
    else:                               # prompts one after another, of unequal lengths
        n = case["requests"]
        cuts = torch.sort(torch.rand(n - 1, device=dev, generator=gen) * T).values
        request = torch.searchsorted(cuts, torch.arange(T, device=dev, dtype=torch.float32), right=True)
        ids = (request + torch.randint(0, S, (1,), device=dev, generator=gen)) % S
    s = {"x": normal(T, K), "y": normal(T, N), "ids": ids.to(torch.int32), "widths": widths,
         "a": normal(S, len(widths), r, K, std=K ** -0.5), "b": normal(S, N, r, std=0.5 * r ** -0.5),
         "ranks": torch.tensor(_ranks(case), dtype=torch.int32, device=dev),
         "scales": 0.5 + 1.5 * torch.rand(S, device=dev, generator=gen)}
    if own:
        from vllm_espalier_b200 import adapters
        s["adapters"] = adapters.Adapters(s["a"], s["b"], widths, ranks=s["ranks"], scales=s["scales"])
    return s


def _prepare_norm(case, gen):
    dev, dt, rt = gen.device, DTYPES[case["dtype"]], DTYPES[case["residual"]]
    R, D = case["rows"], case["d"]

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        return (torch.randn(*shape, device=dev, generator=gen) * std + mean).to(dtype)

    layer = case["kind"] == "layer"
    s = {"x": normal(R, D), "x2": normal(R, D, std=0.5) if case["two"] else None,
         "residual": normal(R, D, std=4.0, dtype=rt),
         "post": normal(D, std=0.1, mean=1.0) if case["post"] else None,
         "post_bias": normal(D, std=0.1) if case["post"] and layer else None,
         "pre": normal(D, std=0.1, mean=1.0), "pre_bias": normal(D, std=0.1) if layer else None,
         "gate": {"none": None, "channel": (D,), "row": (R, 1), "element": (R, D)}[case["gate"]],
         "act": case["act"], "kind": case["kind"], "residual_scale": 0.9, "block_scale": 1.25}
    if s["gate"] is not None:
        s["gate"] = normal(*s["gate"], mean=0.5)
    if own:
        from vllm_espalier_b200 import norms
        s["norm"] = norms.BlockNorm(D, post=s["post"], post_bias=s["post_bias"], pre=s["pre"],
                                    pre_bias=s["pre_bias"], kind=case["kind"], eps=EPS, gate_act=case["act"],
                                    residual_scale=s["residual_scale"], block_scale=s["block_scale"])
    return s


def _draft_counts(case):
    """The drafted tokens of each request: all of one count, or ragged from none to the most."""
    k, n = case["drafts"], case["requests"]
    return [k if k <= 3 else (3 * b + k) % (k + 1) for b in range(n)]


def _prepare_verify(case, gen):
    dev, V, B = gen.device, case["vocab"], case["requests"]
    counts = torch.tensor(_draft_counts(case))
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])
    n, rows = int(starts[-1]), int(starts[-1]) + B
    buffer = torch.randn(rows, V + case["padding"], device=dev, generator=gen).mul_(2.0)
    logits = buffer[:, :V]
    # a trained model's rows: a few likely tokens that hold most of a row's probability
    top = torch.randint(0, V // 8, (rows, 8), device=dev, generator=gen) + torch.arange(8, device=dev) * (V // 8)
    logits.scatter_add_(1, top, math.log(V) - 2.5 + 3.0 * torch.rand(rows, 8, device=dev, generator=gen))
    # every fourth request has its unlikely tokens masked out, as a top-k filter does
    row_of = torch.arange(B).repeat_interleave(counts + 1).to(dev)
    cut = torch.where(row_of % 4 == 3, logits.amax(1) - 12.0, -math.inf)
    logits.masked_fill_(logits < cut[:, None], -math.inf)
    buffer = buffer.to(DTYPES[case["dtype"]])
    logits = buffer[:, :V]
    # every fifth request is greedy
    b = torch.arange(B)
    temperature = torch.where(b % 5 == 4, torch.tensor(0.0), 0.7 + 0.1 * (b % 7))
    # the drafter: the target's distribution blurred, a token drawn from it (or its likeliest)
    target_row = (torch.arange(n) + torch.arange(B).repeat_interleave(counts)).to(dev)
    blurred = logits[target_row].float()
    blurred += 0.5 * torch.randn(blurred.shape, device=dev, generator=gen)
    if case["probs"] == "none":
        probs, drafts = None, blurred.argmax(1) if n else torch.zeros(0, device=dev)
    else:
        q = torch.softmax(blurred, dim=1)
        drafts = (q / torch.empty_like(q).exponential_(generator=gen)).argmax(1) if n else torch.zeros(0, device=dev)
        probs = q.to(DTYPES[case["probs"]])
    del blurred
    return {"logits": logits, "starts": starts.to(dev, torch.int32), "drafts": drafts.to(torch.int32),
            "uniform": torch.rand(n, device=dev, generator=gen),
            "noise": torch.empty(B, V, device=dev).exponential_(generator=gen).clamp_(min=1e-30),
            "temperature": temperature.to(dev), "probs": probs, "most": case["drafts"]}


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    make = {"adapters": _prepare_adapters, "norm": _prepare_norm, "verify": _prepare_verify}[case["op"]]
    return {"op": case["op"], **make(case, gen)}


# ---------------------------------------------------------------------------------------------------------------
# the plain forms: fp32, rounded once at the end
# ---------------------------------------------------------------------------------------------------------------
def _plain_adapters(s):
    """Every row against every adapter, the products with the other adapters (and the columns past an adapter's rank)
    masked out before the second product."""
    x, a, b, ids = s["x"].float(), s["a"].float(), s["b"].float(), s["ids"]
    S, M, r, K = a.shape
    slot, col = torch.arange(S, device=x.device), torch.arange(r, device=x.device)
    keep = (ids[:, None] == slot)[:, :, None] & (col < s["ranks"][:, None])[None]          # [T, S, r]
    weight = torch.where(keep, s["scales"][None, :, None], torch.zeros((), device=x.device))

    def matrix(m, columns):
        u = (x @ a[:, m].reshape(S * r, K).T).reshape(-1, S, r) * weight
        return u.reshape(-1, S * r) @ columns.permute(0, 2, 1).reshape(S * r, -1)

    parts = [matrix(m, columns) for m, columns in enumerate(torch.split(b, s["widths"], dim=1))]
    return (s["y"].float() + torch.cat(parts, dim=1)).to(s["y"].dtype)


def _normed(v, weight, bias, kind):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    if weight is not None:
        v = v * weight.float()
    return v if bias is None else v + bias.float()


def _plain_norm(s):
    v = s["x"].float() if s["x2"] is None else s["x"].float() + s["x2"].float()
    if s["post"] is not None:
        v = _normed(v, s["post"], s["post_bias"], s["kind"])
    if s["gate"] is not None:
        g = s["gate"].float()
        v = v * (torch.sigmoid(g) if s["act"] == "sigmoid" else torch.tanh(g) if s["act"] == "tanh" else g)
    r = s["residual_scale"] * s["residual"].float() + s["block_scale"] * v
    return r.to(s["residual"].dtype), _normed(r, s["pre"], s["pre_bias"], s["kind"]).to(s["x"].dtype)


def _plain_verify(s):
    logits, starts, most, probs = s["logits"].float(), s["starts"].long(), s["most"], s["probs"]
    dev, B = logits.device, starts.shape[0] - 1
    b, place = torch.arange(B, device=dev), torch.arange(most + 1, device=dev)
    count, first = starts[1:] - starts[:-1], starts[:-1] + b            # drafts, first row of each request
    request = torch.searchsorted(first, torch.arange(logits.shape[0], device=dev), right=True) - 1
    greedy = s["temperature"] == 0
    z = logits / torch.where(greedy, 1.0, s["temperature"])[request, None]
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    p, likeliest = e / total, logits.argmax(1)
    n = torch.zeros(B, dtype=torch.int64, device=dev)
    draft = torch.full((B, most + 1), -1, dtype=torch.int64, device=dev)
    if s["drafts"].shape[0]:
        drafted = place[None, :most] < count[:, None]
        at = (starts[:-1, None] + place[None, :most]).clamp(max=s["drafts"].shape[0] - 1)
        row = torch.minimum(first[:, None] + place[None, :most], (first + count)[:, None])
        d = s["drafts"].long()[at]
        qd = torch.ones((), device=dev) if probs is None else probs[at, d].float()
        ok = torch.where(greedy[:, None], d == likeliest[row], s["uniform"][at] * qd < p[row, d]) & drafted
        n = ok.long().cumprod(1).sum(1)
        draft[:, :most] = d
    row = first + n
    w, best, rejected = p[row], likeliest[row], n < count
    if probs is None:
        w = torch.where((torch.arange(w.shape[1], device=dev) == draft[b, n][:, None]) & rejected[:, None], 0.0, w)
    elif s["drafts"].shape[0]:
        q = probs[(starts[:-1] + n).clamp(max=probs.shape[0] - 1)].float()
        w = torch.where(rejected[:, None], (w - q).clamp(min=0), w)
    drawn = torch.where((w > 0).any(1) & ~greedy, (w / s["noise"]).argmax(1), best)
    tokens = torch.where(place < n[:, None], draft, torch.where(place == n[:, None], drawn[:, None], -1))
    row = torch.minimum(first[:, None] + place, row[:, None])
    probability = torch.where(tokens >= 0, p[row, tokens.clamp(min=0)], 0.0)
    return tokens.to(torch.int32), n.to(torch.int32), probability


def run(state):
    op = state["op"]
    if not own:
        return {"adapters": _plain_adapters, "norm": _plain_norm, "verify": _plain_verify}[op](state)
    if op == "adapters":
        return state["adapters"].forward(state["x"], state["y"], state["ids"])
    if op == "norm":
        return state["norm"].forward(state["x"], state["residual"], x2=state["x2"], gate=state["gate"])
    from vllm_espalier_b200 import speculative
    return speculative.verify(state["logits"], state["starts"], state["drafts"], state["uniform"], state["noise"],
                              max_drafts=state["most"], temperature=state["temperature"], draft_probs=state["probs"])


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "adapters":
        T, K, N, slots, ranks = case["tokens"], case["k"], sum(_widths(case)), case["slots"], _ranks(case)
        rank = sum(ranks) / slots
        if case["order"] == "mixed":        # rows with an adapter, and the adapters that they use
            rows, used = 0.9 * T, slots * (1 - (1 - 1 / slots) ** (0.9 * T))
        else:
            rows, used = T, min(case["requests"], slots)
        columns = rank * (len(_widths(case)) * K + N)
        return {"bytes": e * (rows * K + 2 * T * N + used * columns) + 4 * T, "flops": 2 * rows * columns}
    if case["op"] == "norm":
        R, D = case["rows"], case["d"]
        gate = {"none": 0, "channel": D, "row": R, "element": R * D}[case["gate"]]
        weights = D * (1 + case["post"]) * (1 + (case["kind"] == "layer"))
        values = R * D * (2 + case["two"]) + gate + weights          # x, x2, h, the gate and the weights
        return {"bytes": e * values + 2 * R * D * SIZE[case["residual"]], "flops": 10 * R * D}
    V, counts = case["vocab"], _draft_counts(case)
    rows = sum((1 - ACCEPTED ** (k + 1)) / (1 - ACCEPTED) for k in counts)      # up to the first rejected one
    drawn = sum(1 for b in range(case["requests"]) if b % 5 != 4)
    rejected = 0 if case["probs"] == "none" else sum(1 - ACCEPTED ** k for k in counts) * drawn / case["requests"]
    q = rejected * SIZE[case["probs"]] if case["probs"] != "none" else 0
    return {"bytes": V * (rows * e + 4 * drawn + q), "flops": V * (4 * rows + 4 * drawn)}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def _exact_adapters(s):
    out = s["y"].double()
    for slot in sorted(set(s["ids"].tolist()) - {-1}):
        rows, r = (s["ids"] == slot).nonzero()[:, 0], int(s["ranks"][slot])
        x, col = s["x"][rows].double(), 0
        for m, width in enumerate(s["widths"]):
            u = x @ s["a"][slot, m, :r].double().T
            delta = u @ s["b"][slot, col:col + width, :r].double().T
            out[rows, col:col + width] += float(s["scales"][slot]) * delta
            col += width
    return out


def _exact_norm(s):
    def norm(v, weight, bias):
        if s["kind"] == "layer":
            v = v - v.sum(1, keepdim=True) / v.shape[1]
        v = v / (v.pow(2).sum(1, keepdim=True) / v.shape[1] + EPS).sqrt()
        v = v if weight is None else v * weight.double()
        return v if bias is None else v + bias.double()

    v = s["x"].double() + (0 if s["x2"] is None else s["x2"].double())
    if s["post"] is not None:
        v = norm(v, s["post"], s["post_bias"])
    if s["gate"] is not None:
        g = s["gate"].double()
        v = v * {"none": lambda t: t, "sigmoid": lambda t: 1 / (1 + (-t).exp()), "tanh": torch.tanh}[s["act"]](g)
    r = s["residual"].double() * s["residual_scale"] + v * s["block_scale"]
    return r, norm(r, s["pre"], s["pre_bias"])


def _exact_verify(s):
    """Request by request, row by row, as the definition reads."""
    starts, drafts, uniform = s["starts"].tolist(), s["drafts"].tolist(), s["uniform"].double().tolist()
    B, most = len(starts) - 1, s["most"]
    tokens = torch.full((B, most + 1), -1, dtype=torch.int32)
    counts, probability = torch.zeros(B, dtype=torch.int32), torch.zeros(B, most + 1, dtype=torch.float64)
    for b in range(B):
        t = float(s["temperature"][b])
        for i in range(starts[b + 1] - starts[b] + 1):
            logits = s["logits"][starts[b] + b + i].double()
            target = torch.softmax(logits / (t or 1.0), dim=0)
            p, at, last = target.clone(), starts[b] + i, starts[b] + i == starts[b + 1]
            best = int((logits == logits.max()).nonzero()[0])
            if not last:
                d = drafts[at]
                q = None if s["probs"] is None else s["probs"][at].double()
                if d == best if t == 0 else uniform[at] * (1.0 if q is None else float(q[d])) < float(p[d]):
                    tokens[b, i], probability[b, i] = d, target[d]
                    continue
                if q is None:
                    p[d] = 0
                else:
                    p = (p - q).clamp(min=0)
            token = best if t == 0 or not bool((p > 0).any()) else int((p / s["noise"][b].double()).argmax())
            tokens[b, i], probability[b, i], counts[b] = token, target[token], i
            break
    return tokens, counts, probability


def exact(case, seed):
    s = prepare(case, seed)
    return {"adapters": _exact_adapters, "norm": _exact_norm, "verify": _exact_verify}[s["op"]](s)
