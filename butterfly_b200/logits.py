"""Log probabilities of given tokens, entropies and likeliest alternatives, from logits.

What a server returns beside its tokens, and what ``integrations.quality_smoke`` can score a prompt with under stock and compressed
attention: one pass over the logits, which are read once and never copied to fp32.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib


class TokenLogprobs(NamedTuple):
    """What ``token_logprobs`` returns, on the device (leading shape: the rows of the logits)."""
    logprobs: Optional[torch.Tensor]  # [...] fp32 of the given tokens, None without tokens
    entropy: torch.Tensor             # [...] fp32, in nats
    top_ids: torch.Tensor             # [..., top_k] int64, likeliest first
    top_logprobs: torch.Tensor        # [..., top_k] fp32


_native = None


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, *, top_k: int = 0) -> TokenLogprobs:
    """Log softmax of ``logits`` [..., V] (bf16, fp16 or fp32; V contiguous, the leading dims at any two strides) at
    ``tokens`` [...] (int64 or int32), the entropy of each row's distribution, and its ``top_k`` (at most 64) likeliest
    entries, of equal ones the lowest index first.

    A negative token is padding: its log probability is 0, so that it drops out of sums.  One that is not below V has -inf.
    Entries of -inf are masked; a row of nothing else has log probabilities -inf and entropy 0.  A row
    with a NaN or +inf gives NaN for both (its ids are in range, NaN ordered as -inf).  fp32 sums; the
    results carry no gradient, and share one allocation, which each keeps alive (``clone`` one that is to outlive the others)."""
    global _native
    if _native is None:
        _native = _lib.native()
    r = _native.logprobs(logits, tokens, top_k, _lib.raw_stream(logits))
    if r.__class__ is int:
        _lib.check(r)
    return TokenLogprobs(*r)


__all__ = ["TokenLogprobs", "token_logprobs"]
