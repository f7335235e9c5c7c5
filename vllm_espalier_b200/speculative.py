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

from ._lib import DTYPE, launch, lib

MAX_COUNT = 1 << 30           # requests, ids of the vocabulary, drafted tokens of a request


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
    code = DTYPE.get(logits.dtype)
    if code is None or logits.dim() != 2 or not logits.is_cuda:
        raise ValueError(f"logits must be a CUDA fp16/bf16/fp32 [rows, vocab] tensor, got {logits.dtype} "
                         f"{tuple(logits.shape)}")
    dev, (rows, vocab) = logits.device, logits.shape
    if starts.dim() != 1 or starts.numel() < 1:
        raise ValueError(f"starts must be int32 [requests + 1], got {tuple(starts.shape)}")
    B = starts.numel() - 1
    n = rows - B
    if n < 0 or (B == 0 and n > 0):
        raise ValueError(f"{rows} rows of logits for {B} requests: every request has a row for each drafted token "
                         "and one more")
    if not (B <= MAX_COUNT and 1 <= vocab <= MAX_COUNT and 0 <= max_drafts <= MAX_COUNT):
        raise ValueError(f"{B} requests, a vocabulary of {vocab} and at most {max_drafts} drafted tokens (each up to "
                         f"{MAX_COUNT})")
    flat = [("starts", starts, B + 1, torch.int32), ("drafts", drafts, n, torch.int32),
            ("uniform", uniform, n, torch.float32)]
    if temperature is not None:
        flat.append(("temperature", temperature, B, torch.float32))
    at = []
    for name, t, size, dtype in flat:
        if t.dtype != dtype or t.dim() != 1 or t.numel() != size or t.device != dev or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous {dtype} [{size}] on {dev}, got {t.dtype} {tuple(t.shape)} on "
                             f"{t.device}")
        at.append(t.data_ptr())
    if noise.dtype != torch.float32 or noise.shape != (B, vocab) or noise.device != dev:
        raise ValueError(f"noise must be fp32 [{B}, {vocab}] on {dev}, got {noise.dtype} {tuple(noise.shape)} on "
                         f"{noise.device}")
    (stride, step), (noise_stride, noise_step) = logits.stride(), noise.stride()
    if step != 1:
        logits, stride = logits.contiguous(), vocab
    if noise_step != 1:
        noise, noise_stride = noise.contiguous(), vocab
    q_ptr = q_stride = q_code = 0
    if draft_probs is not None:
        q_code = DTYPE.get(draft_probs.dtype)
        if q_code is None or draft_probs.shape != (n, vocab) or draft_probs.device != dev:
            raise ValueError(f"draft_probs must be fp16/bf16/fp32 [{n}, {vocab}] on {dev}, got {draft_probs.dtype} "
                             f"{tuple(draft_probs.shape)} on {draft_probs.device}")
        if draft_probs.stride(1) != 1:
            draft_probs = draft_probs.contiguous()
        q_ptr, q_stride = draft_probs.data_ptr(), draft_probs.stride(0)
    tokens = starts.new_empty((B, max_drafts + 1))      # int32; new_empty parses no options
    accepted, probs = starts.new_empty(B), noise.new_empty((B, max_drafts + 1))
    if B:
        launch(dev, lib().esp_verify, logits.data_ptr(), code, stride, rows, vocab, at[0], B, at[1], at[2], n, q_ptr, q_code,
               q_stride, noise.data_ptr(), noise_stride, at[3] if len(at) > 3 else 0, max_drafts, tokens.data_ptr(),
               accepted.data_ptr(), probs.data_ptr())
    return tokens, accepted, probs
