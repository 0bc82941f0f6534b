"""What a serving program reports of its logits besides the token it picked: the
log probability of a given token per row, the entropy of the row's distribution and
the most likely alternatives, in one pass over the logits. Kernel:
se12_step_logprobs (include/se12_step.h). No counterpart in the reference, whose
runtime leaves sampling to the framework."""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as nat
from .paged import _on, _stream, check_softcap

MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor      # FP32 [rows]
    entropy: torch.Tensor       # FP32 [rows], in nats
    top_logprobs: torch.Tensor  # FP32 [rows, top], from the most likely
    top_ids: torch.Tensor       # int64 [rows, top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0, softcap: float = 0.0) -> TokenLogprobs:
    """Log probabilities of `tokens` int64 [rows] under softmax(z) of every row of `logits` [rows, vocab] (BF16 or FP32;
    rows may be strided), z = softcap tanh(logits / softcap) where softcap > 0 (2^-60 to 1024; a Gemma LM head's raw product),
    else the logits; the entropy; and the `top` (0 to 32) most likely tokens, ordered by logit, equal ones by the lower index.

    A token outside [0, vocab) has log probability -inf. Logits of -inf (tokens that are not allowed) have no part in the
    sums where there is no cap; under one, -inf counts as -softcap. A row of nothing else has log probabilities of -inf
    and entropy 0; a row with a NaN, or +inf without a cap, has NaN throughout, in its alternatives NaN comes last. Runs
    on the current stream of the logits' device and never waits for it; no gradients."""
    if not isinstance(logits, torch.Tensor) or logits.dim() != 2 or logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("logits must be a bfloat16 or float32 [rows, vocab] tensor")
    rows, vocab = logits.shape
    if not 1 <= vocab <= 2 ** 30 or rows >= 2 ** 31:
        raise ValueError(f"logits must have 1 to 2^30 columns and below 2^31 rows, got {list(logits.shape)}")
    if not logits.is_cuda:
        raise ValueError("expected a tensor on a HIP device")
    dev = logits.device
    if not isinstance(tokens, torch.Tensor) or tokens.dtype != torch.int64 or tuple(tokens.shape) != (rows,) or tokens.device != dev:
        raise ValueError(f"tokens must be an int64 [{rows}] tensor on {dev}")
    if int(top) != top or not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top must be 0 to {min(MAX_TOP, vocab)}, got {top}")
    check_softcap(softcap)
    if (logits.stride(1) != 1 and vocab > 1) or (logits.stride(0) < vocab and rows > 1):
        logits = logits.contiguous()
    tokens = tokens.contiguous()
    stride = max(logits.stride(0), vocab)
    with _on(dev):
        logprobs, entropy = torch.empty((2, rows), dtype=torch.float32, device=dev).unbind()
        top_logprobs = torch.empty((rows, top), dtype=torch.float32, device=dev)
        top_ids = torch.empty((rows, top), dtype=torch.int64, device=dev)
        if rows:
            lib = nat.lib()
            n = lib.se12_step_logprobs_workspace(rows, vocab, top)
            if n < 0:
                nat.step_check(n)
            ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
            nat.step_check(lib.se12_step_logprobs(
                logits.data_ptr(), nat.STEP_F32 if logits.dtype == torch.float32 else nat.STEP_BF16, stride, rows, vocab, float(softcap),
                tokens.data_ptr(), int(top), logprobs.data_ptr(), entropy.data_ptr(), top_logprobs.data_ptr(), top_ids.data_ptr(),
                ws.data_ptr() if n else None, n, _stream(dev)))
    return TokenLogprobs(logprobs, entropy, top_logprobs, top_ids)
