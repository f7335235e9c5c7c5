"""The example's decode step: the operators around the coded projections run together as a serving loop uses them, against
the same coded kernels with the norms, adapters and verification as plain torch operations; and their torch operators."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

from vllm_espalier_b200 import adapters, norms, ops, speculative

ROOT = Path(__file__).resolve().parent.parent


def example():
    spec = importlib.util.spec_from_file_location("decode_step", ROOT / "examples" / "decode_step.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def plain_norm(self, x, residual=None, x2=None, gate=None, **_):
    v = x.float() + (0 if x2 is None else x2.float())
    if residual is not None:
        v = residual.float() + 0.5 * v
    h = v * torch.rsqrt(v.pow(2).mean(1, keepdim=True) + 1e-6) * self.tensors["pre_w"].float()
    return v.to(torch.bfloat16), h.to(torch.bfloat16)


def plain_adapters(self, x, y, ids, out=None):
    d = y.float()
    for s in range(self.slots):
        at, col = (ids == s).nonzero()[:, 0], 0
        for m, w in enumerate(self.widths):
            u = x[at].float() @ self.a[s, m].float().T
            d[at, col:col + w] += self.scales[s] * (u @ self.b[s, col:col + w].float().T)
            col += w
    return y.copy_(d.to(y.dtype)) if out is not None else d.to(y.dtype)


@pytest.mark.gpu
def test_step_equals_the_plain_composition(dev, monkeypatch):
    """Every operator rounds once where the plain form does, so a step's logits differ by what a last bit of bf16 grows to
    over two layers (the decoder's own tolerance, 2e-2 of the largest logit, on its 2 layers)."""
    ex = example()
    model = ex.Decoder(dev)
    g = torch.Generator(device=dev).manual_seed(3)
    tokens = torch.randint(0, model.vocab, (24,), device=dev, generator=g)
    ids = (torch.arange(24, device=dev) % 5 - 1).to(torch.int32)
    got = model.logits(tokens, ids)
    without = model.logits(tokens, torch.full_like(ids, -1))
    with monkeypatch.context() as m:
        m.setattr(norms.BlockNorm, "__call__", plain_norm)
        m.setattr(adapters.Adapters, "forward", plain_adapters)
        want = model.logits(tokens, ids)
    assert ((got.float() - want.float()).abs().max() / want.float().abs().max()).item() < 2e-2
    assert torch.equal(got[ids < 0], without[ids < 0]) and not torch.equal(got[ids >= 0], without[ids >= 0])


@pytest.mark.gpu
def test_loop_emits_valid_tokens(dev):
    ex = example()
    batch = ex.Batch(ex.Decoder(dev), requests=6, drafts=3)
    total = 0
    for _ in range(4):
        tokens, accepted, probs = batch.step()
        at = torch.arange(4, device=dev)
        assert torch.equal(tokens >= 0, at[None] <= accepted[:, None])
        assert (tokens < batch.model.vocab).all() and (probs[tokens >= 0] > 0).all() and (probs[tokens < 0] == 0).all()
        total += int(accepted.sum())
    assert total > 0         # the drafter repeats the target's likeliest token most of the time
    with pytest.raises(ValueError):
        ex.Batch(batch.model, requests=9, drafts=3)


@pytest.mark.gpu
def test_torch_operators(dev):
    """espalier::adapt, espalier::block_norm and espalier::verify give what the classes and the function give."""
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(9, 128, device=dev, generator=g).to(torch.bfloat16)
    ad = adapters.Adapters(torch.randn(3, 2, 8, 128, device=dev, generator=g).to(torch.bfloat16),
                           torch.randn(3, 48, 8, device=dev, generator=g).to(torch.bfloat16), [32, 16])
    y = torch.randn(9, 48, device=dev, generator=g).to(torch.bfloat16)
    ids = (torch.arange(9, device=dev) % 4 - 1).to(torch.int32)
    assert torch.equal(ops.adapt(x, y, ids, ops.register(ad)), ad(x, y, ids))
    norm = norms.BlockNorm(128, pre=x[0].contiguous(), post=True, gate_act="sigmoid")
    key = ops.register(norm)
    for a, b in zip(ops.block_norm(x, x * 2, x * 3, x[:, :1], key), norm(x, x * 3, x2=x * 2, gate=x[:, :1])):
        assert torch.equal(a, b)
    logits = torch.randn(7, 50, device=dev, generator=g)
    args = (logits, torch.tensor([0, 2, 5], dtype=torch.int32, device=dev),
            torch.randint(0, 50, (5,), device=dev, generator=g).to(torch.int32), torch.rand(5, device=dev, generator=g),
            torch.empty(2, 50, device=dev).exponential_(generator=g), 3)
    for a, b in zip(ops.verify(*args), speculative.verify(*args)):
        assert torch.equal(a, b)
    with pytest.raises(KeyError):
        ops.adapt(x, y, ids, 10 ** 9)
    with pytest.raises(TypeError):
        ops.adapt(x, y, ids, key)


def test_operator_shapes():
    """The operators' shapes for a compiled graph, without a GPU."""
    with torch._subclasses.fake_tensor.FakeTensorMode():
        x, y = torch.empty(5, 64, dtype=torch.bfloat16), torch.empty(5, 96, dtype=torch.bfloat16)
        out = torch.ops.espalier.adapt(x, y, torch.empty(5, dtype=torch.int32), 0)
        assert out.shape == y.shape and out.dtype == y.dtype
        r, h = torch.ops.espalier.block_norm(x, None, x.float(), None, 0)
        assert r.shape == h.shape == x.shape and r.dtype == torch.float32 and h.dtype == x.dtype
        tokens, accepted, probs = torch.ops.espalier.verify(
            torch.empty(7, 50), torch.empty(4, dtype=torch.int32), torch.empty(4, dtype=torch.int32), torch.empty(4),
            torch.empty(3, 50), 2, None, None)
        assert tokens.shape == probs.shape == (3, 3) and accepted.shape == (3,) and tokens.dtype == torch.int32
