"""Causal attention over packed sequences of different lengths.

`cu_seqlens` (int32, on the tensors' device) holds the sequences' borders:
sequence b is the tokens cu_seqlens[b] .. cu_seqlens[b + 1]; it starts at 0 and
never falls. It is not read by the host, so a captured graph may be replayed
with other borders. GPU kernels: csrc/packed_attention.hip. CPU:
ops/reference.py.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import reference as ref
from .interface import get_ext, use_hip


def flash_attention_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                           cu_seqlens: torch.Tensor,
                           scale: Optional[float] = None) -> torch.Tensor:
    """Causal GQA attention inside each packed sequence.

    q [T, H, D], k and v [T, kv_heads, D] (bf16 on the GPU, D <= 192, any
    strides), H a multiple of kv_heads, and at most 65536 sequences. Returns
    [T, H, D]. `scale` (positive) defaults to D ** -0.5. Rows behind the last
    sequence give zeros and get zero gradients. The gradient can be taken once
    (on the GPU) and has one order of summation, so it is the same each time; its
    probabilities are rounded to bf16, in calls of up to T * H = 8192 to 16 bits.
    The CPU refuses borders that fall or pass T; the GPU, which does not read
    them, cuts them to T and computes nothing outside the tensors, and what such
    borders give is not defined.

    A query whose scores are all -inf has no softmax and gives NaN. Values that
    are not finite may reach every query and gradient of their sequence, and no
    other."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if use_hip(q):
        return get_ext().packed_attn(q, k, v, cu_seqlens, scale)
    return ref.flash_attention_packed(q, k, v, cu_seqlens, scale)


def packed_positions(cu_seqlens: torch.Tensor, total: int) -> torch.Tensor:
    """Position of each of `total` packed tokens inside its sequence, int32 [1,
    total] as `rope` takes it; rows behind the last sequence count on."""
    tok = torch.arange(total, dtype=torch.int32, device=cu_seqlens.device)
    seq = torch.searchsorted(cu_seqlens[1:].contiguous(), tok, right=True)
    start = cu_seqlens[seq.clamp(max=cu_seqlens.shape[0] - 1)]
    # wrong borders must not index outside a rope table
    return (tok - start).clamp(0, total - 1).view(1, total)
