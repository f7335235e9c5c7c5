"""speculative.verify against its definition in 64 bits, and the values where it can go wrong: rows with nothing left,
NaN and infinities, ties, drafted ids outside the vocabulary, starts that do not fit, odd strides.

Tokens and counts are whole numbers and have to be equal. The probabilities are fp32: a softmax's sum over at most
2^18 terms in a tree of sums of at most 2^11 sequential ones, each exp within 2 units and its argument within one of at
most 2^7, so 2^-24 x (2^11 worst, far less than that on average: 64 taken) x the value, and 2^7 x 2^-24 for the argument:
a relative 256 x 2^-24.
"""
from __future__ import annotations

import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from vllm_espalier_b200 import _lib
from vllm_espalier_b200 import speculative

REL = 256 * 2.0 ** -24
INF, NAN = math.inf, math.nan


def reference(logits, starts, drafts, uniform, noise, max_drafts, temperature=None, draft_probs=None):
    """The definition, one request and one row after another, fp64 on the CPU."""
    logits, noise = logits.double().cpu(), noise.double().cpu()
    logits = torch.where(logits.isnan(), -INF, logits)
    starts, drafts, uniform = starts.tolist(), drafts.tolist(), uniform.double().tolist()
    B, V = len(starts) - 1, logits.shape[1]
    tokens = torch.full((B, max_drafts + 1), -1, dtype=torch.int32)
    accepted = torch.zeros(B, dtype=torch.int32)
    probs = torch.zeros(B, max_drafts + 1, dtype=torch.float64)
    for b in range(B):
        t = 1.0 if temperature is None else float(temperature[b])
        greedy = not t > 0
        at, k = starts[b], starts[b + 1] - starts[b]
        if at < 0 or k < 0 or at + k > len(drafts) or at + b + k >= logits.shape[0]:
            continue
        k = min(k, max_drafts)
        for i in range(k + 1):
            row = logits[at + b + i]
            accepted[b] = i
            m = row.max()
            if m == -INF:
                break
            e = torch.where(row == m, 1.0, ((row - m) / (1.0 if greedy else t)).exp())
            e = torch.where(row == -INF, 0.0, e)
            p = e / e.sum()
            best = int((row == m).nonzero()[0])
            d = drafts[at + i] if i < k else -1
            valid = 0 <= d < V
            if valid:
                q = 1.0 if draft_probs is None else float(draft_probs[at + i, d])
                if d == best if greedy else uniform[at + i] * q < float(p[d]):
                    tokens[b, i], probs[b, i] = d, p[d]
                    continue
            token = best
            if not greedy:
                w = p.clone()
                if i < k:
                    if draft_probs is not None:
                        w = (p - draft_probs[at + i].double().cpu()).clamp(min=0)
                    elif valid:
                        w[d] = 0
                if (w > 0).any():
                    token = int(torch.where(w > 0, w / noise[b], -1.0).argmax())
            tokens[b, i], probs[b, i] = token, p[token]
            break
    return tokens, accepted, probs


def compare(got, want):
    tokens, accepted, probs = (t.cpu() for t in got)
    assert torch.equal(tokens, want[0]), (tokens, want[0])
    assert torch.equal(accepted, want[1])
    assert ((probs.double() - want[2]).abs() <= REL * want[2] + 1e-37).all()


def batch(dev, counts, V, dtype, probs, seed, peak=0.0, pad=0, temperatures=(1.0,)):
    g = torch.Generator(device=dev).manual_seed(seed)
    B, n = len(counts), sum(counts)
    starts = torch.tensor([sum(counts[:i]) for i in range(B + 1)], dtype=torch.int32, device=dev)
    logits = torch.randn(n + B, V + pad, device=dev, generator=g) * 2
    logits[torch.arange(n + B, device=dev), torch.randint(0, V, (n + B,), device=dev, generator=g)] += peak
    logits = logits.to(dtype)[:, :V]
    rows = torch.tensor([i + b for b, k in enumerate(counts) for i in range(sum(counts[:b]), sum(counts[:b]) + k)],
                        dtype=torch.long, device=dev)
    blurred = logits[rows].float() + 0.5 * torch.randn(n, V, device=dev, generator=g)
    q = torch.softmax(blurred, 1)
    if probs is None:
        drafts, q = (blurred.argmax(1) if n else torch.zeros(0, device=dev)), None
    else:
        e = torch.empty_like(q).exponential_(generator=g)
        drafts, q = ((q / e).argmax(1) if n else torch.zeros(0, device=dev)), q.to(probs)
    t = torch.tensor([temperatures[b % len(temperatures)] for b in range(B)], device=dev, dtype=torch.float32)
    return dict(logits=logits, starts=starts, drafts=drafts.to(torch.int32),
                uniform=torch.rand(n, device=dev, generator=g),
                noise=torch.empty(B, V, device=dev).exponential_(generator=g).clamp_(min=1e-30),
                max_drafts=max(counts, default=0), temperature=t, draft_probs=q)


def run_and_check(**kw):
    compare(speculative.verify(**kw), reference(**kw))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1, 2, 31, 128, 1000, 8191, 32000, 65537, 248320])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("probs", [None, torch.float32, torch.bfloat16])
def test_sizes(dev, V, dtype, probs):
    run_and_check(**batch(dev, [3, 0, 1, 4], V, dtype, probs, seed=V, peak=math.log(V) + 2, pad=V % 3,
                          temperatures=(1.0, 0.7, 0.0, 1.9)))


@pytest.mark.gpu
@pytest.mark.parametrize("requests", [1, 2, 17, 150, 600])
def test_requests(dev, requests):
    counts = [(5 * b + 2) % 4 for b in range(requests)]
    run_and_check(**batch(dev, counts, 1537, torch.bfloat16, torch.float32, seed=requests, peak=8.0,
                          temperatures=(0.9, 0.0, 1.0)))


@pytest.mark.gpu
@pytest.mark.parametrize("k", [0, 1, 16])
@pytest.mark.parametrize("probs", [None, torch.float16])
def test_long_drafts(dev, k, probs):
    run_and_check(**batch(dev, [k, k], 5000, torch.float32, probs, seed=k, peak=14.0))


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [1, 2, 3, 5, 7])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_no_vector_load_fits(dev, pad, dtype):
    kw = batch(dev, [2, 3, 0], 4099, dtype, torch.bfloat16, seed=pad, peak=9.0, pad=pad)
    wide = torch.empty(3, 4099 + pad, device=dev)
    wide[:, pad:] = kw["noise"]
    kw["noise"] = wide[:, pad:]
    q = torch.empty(5, 4099 + pad, device=dev, dtype=torch.bfloat16)
    q[:, pad:] = kw["draft_probs"]
    kw["draft_probs"] = q[:, pad:]
    run_and_check(**kw)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [40, 20000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_logits(dev, V, dtype):
    """Tokens ruled out by -inf, NaN or the type's lowest value; rows with one token left, with none; +inf logits."""
    kw = batch(dev, [3] * 8, V, dtype, torch.float32, seed=2, peak=4.0, temperatures=(1.0, 0.5, 0.0, INF, 1e-38))
    low = torch.finfo(dtype).min
    x = kw["logits"].clone()
    x[0:4, ::2] = -INF
    x[4:8, 1::2] = NAN
    x[8:12, : V - 3] = low
    x[12] = -INF
    x[17] = NAN
    x[21] = -INF
    x[21, 7] = 1.0
    x[24:28, 5] = INF
    x[25, 9] = INF
    x[28] = low
    run_and_check(**dict(kw, logits=x))
    one_hot = batch(dev, [3] * 8, V, dtype, None, seed=3, peak=4.0)
    run_and_check(**dict(one_hot, logits=x))


@pytest.mark.gpu
def test_ties_go_to_the_lowest_id(dev):
    V = 3001
    x = torch.zeros(4, V, device=dev)
    x[:, [700, 2999, 1500]] = 5.0
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev)
    drafts = torch.tensor([700, 1500], dtype=torch.int32, device=dev)
    kw = dict(logits=x, starts=starts, drafts=drafts, uniform=torch.rand(2, device=dev),
              noise=torch.ones(2, V, device=dev), max_drafts=1, temperature=torch.zeros(2, device=dev))
    tokens, accepted, _ = speculative.verify(**kw)
    assert tokens.tolist() == [[700, 700], [700, -1]] and accepted.tolist() == [1, 0]
    kw["temperature"] = torch.ones(2, device=dev)
    kw["uniform"] = torch.full((2,), 1 - 2.0 ** -24, device=dev)
    tokens, accepted, _ = speculative.verify(**kw)      # equal scores: the first of the likeliest that is left
    assert tokens.tolist() == [[1500, -1], [700, -1]] and accepted.tolist() == [0, 0]


@pytest.mark.gpu
def test_residual_of_nothing(dev):
    """The drafter's distribution is the target's and the drafted token impossible: the target's likeliest token."""
    x = torch.full((2, 64), -INF, device=dev)
    x[:, 10], x[:, 20] = 0.0, 0.0
    q = torch.zeros(1, 64, device=dev)
    q[0, 10] = q[0, 20] = 0.5
    tokens, accepted, probs = speculative.verify(
        x, torch.tensor([0, 1], dtype=torch.int32, device=dev), torch.tensor([5], dtype=torch.int32, device=dev),
        torch.zeros(1, device=dev), torch.ones(1, 64, device=dev), 1, draft_probs=q)
    assert tokens.tolist() == [[10, -1]] and accepted.tolist() == [0] and probs.tolist() == [[0.5, 0.0]]


@pytest.mark.gpu
def test_drafts_and_starts_out_of_range(dev):
    kw = batch(dev, [2, 3, 1], 500, torch.bfloat16, torch.float32, seed=6, peak=9.0)
    bad = kw["drafts"].clone()
    bad[0], bad[3], bad[5] = -1, 500, 2 ** 31 - 1
    run_and_check(**dict(kw, drafts=bad))
    run_and_check(**dict(kw, max_drafts=1))
    run_and_check(**dict(kw, max_drafts=0))
    for starts in ([0, 2, 5, 7], [-1, 2, 5, 6], [0, 3, 1, 6], [2 ** 31 - 1, 0, 0, 0], [0, 2 ** 31 - 1, 3, 9]):
        run_and_check(**dict(kw, starts=torch.tensor(starts, dtype=torch.int32, device=dev)))


@pytest.mark.gpu
@pytest.mark.parametrize("drafter", ["probs", "token"])
def test_first_token_is_distributed_as_the_target(dev, drafter):
    """20,000 requests of one drafted token over 8 tokens: whatever the drafter, the first emitted token follows p. Each
    count is binomial: within 5 standard deviations of its mean (a chance of 10^-5 that a right kernel fails)."""
    B, V = 20000, 8
    g = torch.Generator(device=dev).manual_seed(11)
    row = torch.tensor([1.0, 0.0, -1.0, 2.0, 0.5, -INF, 1.5, -2.0], device=dev)
    q = torch.softmax(torch.tensor([0.0, 2.0, 1.0, -1.0, 0.0, 1.0, 0.0, 0.0], device=dev), 0)
    drafts = (q / torch.empty(B, V, device=dev).exponential_(generator=g)).argmax(1).to(torch.int32)
    tokens, _, _ = speculative.verify(
        row.expand(2 * B, V).contiguous(), torch.arange(B + 1, dtype=torch.int32, device=dev),
        drafts if drafter == "probs" else torch.full_like(drafts, 3), torch.rand(B, device=dev, generator=g),
        torch.empty(B, V, device=dev).exponential_(generator=g).clamp_(min=1e-30), 1,
        draft_probs=q.expand(B, V) if drafter == "probs" else None)
    p = torch.softmax(row.double(), 0).cpu()
    got = torch.bincount(tokens[:, 0].cpu().long(), minlength=V).double()
    assert ((got - B * p).abs() <= 5 * (B * p * (1 - p)).sqrt()).all(), (got, B * p)


@pytest.mark.gpu
def test_same_inputs_same_outputs_on_any_stream_and_in_a_graph(dev):
    kw = batch(dev, [3] * 40, 50000, torch.bfloat16, torch.float32, seed=1, peak=12.0)
    want = speculative.verify(**kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = speculative.verify(**kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = speculative.verify(**kw)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, other, captured):
        assert torch.equal(a, b) and torch.equal(a, c)
    alone = {k: v for k, v in kw.items()}
    b = 7       # a request alone gives what it gives among the others
    alone.update(logits=kw["logits"][4 * b:4 * b + 4], drafts=kw["drafts"][3 * b:3 * b + 3],
                 uniform=kw["uniform"][3 * b:3 * b + 3], noise=kw["noise"][b:b + 1],
                 temperature=kw["temperature"][b:b + 1], draft_probs=kw["draft_probs"][3 * b:3 * b + 3],
                 starts=torch.tensor([0, 3], dtype=torch.int32, device=dev))
    for a, c in zip(want, speculative.verify(**alone)):
        assert torch.equal(a[b:b + 1], c)


@pytest.mark.gpu
def test_empty_batch_and_refusals(dev):
    kw = batch(dev, [2, 1], 100, torch.bfloat16, torch.float32, seed=0)
    e = torch.empty(0, device=dev)
    out = speculative.verify(e.view(0, 100), torch.zeros(1, dtype=torch.int32, device=dev), e.int(), e, e.view(0, 100),
                             2)
    assert [t.shape for t in out] == [(0, 3), (0,), (0, 3)]
    bad = [dict(logits=kw["logits"].cpu()), dict(logits=kw["logits"].int()), dict(logits=kw["logits"][0]),
           dict(logits=kw["logits"][:1]), dict(starts=kw["starts"].long()), dict(starts=kw["starts"][:0]),
           dict(drafts=kw["drafts"][:-1]), dict(drafts=kw["drafts"].long()), dict(uniform=kw["uniform"].double()),
           dict(noise=kw["noise"][:1]), dict(noise=kw["noise"].half()), dict(temperature=kw["temperature"][:1]),
           dict(draft_probs=kw["draft_probs"][:2]), dict(draft_probs=kw["draft_probs"].int()), dict(max_drafts=-1)]
    for change in bad:
        with pytest.raises(ValueError):
            speculative.verify(**dict(kw, **change))


def test_library_refusals():
    lib = _lib.lib()
    base = dict(logits=16, dtype=1, stride=8, rows=2, vocab=8, starts=16, requests=1, drafts=16, uniform=16, n_drafts=1,
                draft_probs=None, probs_dtype=2, probs_stride=8, noise=16, noise_stride=8, temperature=None,
                max_drafts=1, tokens=16, accepted=16, probs=16, stream=None)
    for change in (dict(logits=None), dict(dtype=5), dict(vocab=0), dict(requests=-1), dict(starts=None),
                   dict(drafts=None), dict(uniform=None), dict(draft_probs=16, probs_dtype=4), dict(noise=None),
                   dict(max_drafts=-1), dict(tokens=None), dict(accepted=None), dict(probs=None), dict(rows=-1)):
        assert lib.esp_verify(*dict(base, **change).values()) == _lib.ESP_ERR_INVALID, change
        assert lib.esp_last_error()
    assert lib.esp_verify(*dict(base, requests=0).values()) == _lib.ESP_OK


def test_sizes_past_the_calls_integers_are_refused(monkeypatch):
    """No GPU and no memory needed: shapes without storage."""
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    with FakeTensorMode():
        i, f = (lambda n: torch.empty(n, dtype=torch.int32, device="cuda:0")), (lambda *n: torch.empty(*n, device="cuda:0"))
        for B, V, drafts in ((1, 2 ** 32 + 5, 1), (1, 2 ** 30 + 1, 1), (1, 8, 2 ** 32 + 1), (1, 8, 2 ** 31 - 1),
                             (2 ** 32 + 1, 8, 1)):
            with pytest.raises(ValueError, match="up to"):
                speculative.verify(f(B, V), i(B + 1), i(0), f(0), f(B, V), drafts)
    for vocab, drafts in ((2 ** 31 - 1, 1), (2 ** 30 + 1, 1), (8, 2 ** 31 - 1)):
        assert _lib.lib().esp_verify(16, 1, 8, 2, vocab, 16, 1, 16, 16, 1, None, 2, 8, 16, 8, None, drafts, 16, 16, 16,
                                     None) == _lib.ESP_ERR_INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("V", [3, 1003, 20000])
@pytest.mark.parametrize("probs", [None, torch.float32])
@pytest.mark.parametrize("low,high", [(-149, -126), (-149, 3), (126, 128), (-126, 128)])
def test_noise_over_the_types_whole_range(dev, V, probs, low, high):
    """Noise that is subnormal, or whose reciprocal is: still argmax of weight / noise."""
    kw = batch(dev, [2, 0, 3, 1, 0], V, torch.float32, probs, seed=V, peak=2.0, temperatures=(1.0, 0.7))
    g = torch.Generator().manual_seed(V)
    noise = torch.exp2(torch.rand(5, V, generator=g, dtype=torch.float64) * (high - low) + low).clamp(2.0 ** -149, 3.4e38)
    kw["noise"] = noise.float().to(dev)
    assert (kw["noise"] > 0).all() and kw["noise"].isfinite().all()
    run_and_check(**kw)
