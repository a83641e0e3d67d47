"""Log probabilities of given tokens, entropy and the most likely
alternatives of each row of logits (GPU kernels: csrc/logprobs.hip)."""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import reference as ref
from .interface import get_ext, use_hip


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor       # [...] fp32
    entropy: torch.Tensor        # [...] fp32
    top_logprobs: torch.Tensor   # [..., top_k] fp32
    top_ids: torch.Tensor        # [..., top_k] int64


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_k: int = 0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """logits [..., V] (bf16, fp16 or fp32), tokens [...] int64 or int32.

    logprobs: log softmax(logits) at the token; 0 where the token is
    ignore_index, NaN where it is outside the vocabulary. entropy: of the row's
    distribution, in nats. top_logprobs, top_ids: the top_k (at most 64) most
    likely tokens in falling order, ties to the lowest index, NaN first. All
    sums in fp32. -inf logits are tokens of probability 0; a row of nothing
    else has no distribution and gives NaN.

    logprobs and entropy have a gradient with respect to logits (taken
    once, on the GPU); the alternatives have none."""
    shape = tokens.shape
    if logits.shape[:-1] != shape:
        raise ValueError(f"tokens {tuple(shape)} do not match logits "
                         f"{tuple(logits.shape)}")
    if use_hip(logits):
        x, t = logits, tokens
        if x.dim() != 2:
            x = x.reshape(-1, x.shape[-1]) if x.numel() else \
                x.reshape(t.numel(), x.shape[-1])
            t = t.reshape(-1)
        if x.stride(1) != 1:
            x = x.contiguous()
        if not t.is_contiguous():
            t = t.contiguous()
        lp, ent, tl, ti = get_ext().token_logprobs(x, t, top_k, ignore_index)
    else:
        lp, ent, tl, ti = ref.token_logprobs(
            logits.reshape(tokens.numel(), logits.shape[-1]),
            tokens.reshape(-1), top_k, ignore_index)
    if logits.dim() != 2:
        lp, ent = lp.view(shape), ent.view(shape)
        tl, ti = tl.view(*shape, top_k), ti.view(*shape, top_k)
    return TokenLogprobs(lp, ent, tl, ti)
