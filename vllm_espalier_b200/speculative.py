"""Verification of drafted tokens: which of a drafter's tokens the target model would have drawn, and the token after
the last of them, for every request of a batch in one launch.

Request b has k_b drafted tokens and k_b + 1 rows of target logits (the decode step over its drafted tokens). With
p_i = softmax(logits_i / temperature) and q_i the drafter's probabilities, drafted token d_i stands iff all before it
do and uniform_i q_i(d_i) < p_i(d_i); the first that falls is replaced by a draw from the residual max(p_i - q_i, 0), and
if all stand one more token is drawn from the last row. Draws are argmax_v w(v) / noise(v) with independent exponential
noise, so the emitted tokens are distributed as the target's own. All random numbers are inputs: the same inputs give
the same tokens. The kernel is esp_verify (csrc/verify.cu); it allocates nothing but its outputs.
"""
from __future__ import annotations

import torch

from ._lib import DTYPE, check, lib, stream_ptr


def _flat(t: torch.Tensor, n: int, dtype: torch.dtype, name: str, dev) -> int:
    if t.shape != (n,) or t.dtype != dtype or t.device != dev:
        raise ValueError(f"{name} must be {dtype} [{n}] on {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def verify(logits: torch.Tensor, starts: torch.Tensor, drafts: torch.Tensor, uniform: torch.Tensor,
           noise: torch.Tensor, max_drafts: int, temperature: torch.Tensor | None = None,
           draft_probs: torch.Tensor | None = None):
    """logits [n + B, vocab] fp16/bf16/fp32 (a slice of wider rows is fine: a head's padded columns are left out by
    logits[:, :vocab]), request b's rows starting at starts[b] + b; starts int32 [B + 1], the drafted tokens before each
    request; drafts int32 [n]; uniform fp32 [n] in [0, 1); noise fp32 [B, vocab], independent exponential numbers (above
    0); max_drafts: the most drafted tokens a request has; temperature fp32 [B] (0: greedy; None: 1); draft_probs
    [n, vocab], or None for a drafter that chose its token outright.

    Returns (tokens int32 [B, max_drafts + 1], accepted int32 [B], probs fp32 [B, max_drafts + 1]): the drafted tokens
    that stand and the drawn one, then -1; how many stand; the target's probability of each token (0 at -1)."""
    if logits.dim() != 2 or not logits.is_cuda or logits.dtype not in DTYPE:
        raise ValueError(f"logits must be a CUDA fp16/bf16/fp32 [rows, vocab] tensor, got {logits.dtype} "
                         f"{tuple(logits.shape)}")
    dev, (rows, vocab) = logits.device, logits.shape
    if starts.dim() != 1 or starts.shape[0] < 1:
        raise ValueError(f"starts must be int32 [requests + 1], got {tuple(starts.shape)}")
    B = starts.shape[0] - 1
    n = rows - B
    if n < 0 or (B == 0 and n > 0):
        raise ValueError(f"{rows} rows of logits for {B} requests: every request has a row for each drafted token "
                         "and one more")
    if vocab < 1 or max_drafts < 0:
        raise ValueError(f"a vocabulary of {vocab} and at most {max_drafts} drafted tokens")
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    at = [_flat(starts, B + 1, torch.int32, "starts", dev), _flat(drafts, n, torch.int32, "drafts", dev),
          _flat(uniform, n, torch.float32, "uniform", dev)]
    if noise.shape != (B, vocab) or noise.dtype != torch.float32 or noise.device != dev:
        raise ValueError(f"noise must be fp32 [{B}, {vocab}] on {dev}, got {noise.dtype} {tuple(noise.shape)} on "
                         f"{noise.device}")
    if noise.stride(1) != 1:
        noise = noise.contiguous()
    t_ptr = q_ptr = q_stride = q_dtype = 0
    if temperature is not None:
        t_ptr = _flat(temperature, B, torch.float32, "temperature", dev)
    if draft_probs is not None:
        if draft_probs.shape != (n, vocab) or draft_probs.dtype not in DTYPE or draft_probs.device != dev:
            raise ValueError(f"draft_probs must be fp16/bf16/fp32 [{n}, {vocab}] on {dev}, got {draft_probs.dtype} "
                             f"{tuple(draft_probs.shape)} on {draft_probs.device}")
        if draft_probs.stride(1) != 1:
            draft_probs = draft_probs.contiguous()
        q_ptr, q_stride, q_dtype = draft_probs.data_ptr(), draft_probs.stride(0), DTYPE[draft_probs.dtype]
    tokens = torch.empty((B, max_drafts + 1), dtype=torch.int32, device=dev)
    accepted = torch.empty(B, dtype=torch.int32, device=dev)
    probs = torch.empty((B, max_drafts + 1), dtype=torch.float32, device=dev)
    if B:
        check(lib().esp_verify(logits.data_ptr(), DTYPE[logits.dtype], logits.stride(0), rows, vocab, at[0], B, at[1],
                               at[2], n, q_ptr, q_dtype, q_stride, noise.data_ptr(), noise.stride(0), t_ptr,
                               int(max_drafts), tokens.data_ptr(), accepted.data_ptr(), probs.data_ptr(),
                               stream_ptr(dev)))
    return tokens, accepted, probs
