"""Paged key/value cache operators.

A pool holds pages `[pages, kv_heads, page, width]`: `page` tokens (a power of
two from 16) of `width` channels, which is head_dim rounded up to a multiple of
8. A sequence owns a row of page numbers (int32 `block_table[b]`) and a length
(int32 `seq_lens[b]`); token t of it lies in page `block_table[b, t // page]`,
row `t % page`. Lengths and tables stay on the device and are not read by the
host, so a captured graph may replay these calls with new contents:

- a length below zero counts as zero, one past the table's row is cut to it;
- the tokens of a page number outside the pool are left out of the attention,
  and are not written by `paged_kv_append`.

GPU kernels: csrc/paged.hip. CPU: ops/reference.py.
"""

from __future__ import annotations

from typing import List, Optional, Sequence

import torch

from . import reference as ref
from .interface import get_ext, use_hip


def page_width(head_dim: int) -> int:
    """Channels of a page's row: head_dim in whole 16-byte pieces of bf16."""
    return (head_dim + 7) // 8 * 8


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor,
                    v_pages: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor,
                    scale: Optional[float] = None) -> torch.Tensor:
    """Attention of one new token per sequence over its pages.

    q [B, H, D] (bf16 on the GPU, D <= 192), pages as above with H a multiple
    of kv_heads, block_table [B, M] int32, seq_lens [B] int32 (the new token
    included); a table's row has room for fewer than 2^29 tokens, all together
    for 2^31. Returns [B, H, D] in q's type; a sequence of length 0 gives
    zeros. `scale` defaults to D ** -0.5. There is no gradient. Nothing behind
    a sequence's end is read. A live token with a score of -inf has no weight; a
    sequence of nothing else has no softmax and gives NaN, as do other scores
    that are not finite."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if use_hip(q):
        return get_ext().paged_attn(q, k_pages, v_pages, block_table, seq_lens,
                                    scale)
    return ref.paged_attention(q, k_pages, v_pages, block_table, seq_lens,
                               scale)


def paged_kv_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor,
                    v_pages: torch.Tensor, block_table: torch.Tensor,
                    positions: torch.Tensor,
                    seq_ids: Optional[torch.Tensor] = None) -> None:
    """Writes new keys and values [T, kv_heads, D] into their pages, in place.

    Token t goes to position `positions[t]` of sequence `seq_ids[t]` (int32;
    without seq_ids, token t belongs to sequence t). Channels past D in a page's
    row become zero. A token without a place is not written: a negative
    position (padding), one past the table, or a sequence or page that does not
    exist. Two tokens for one place leave one of them there, it is not said
    which. Nothing flows back through the pool."""
    if use_hip(k):
        get_ext().paged_append(k, v, k_pages, v_pages, block_table, positions,
                               seq_ids)
        return
    ref.paged_kv_append(k.detach(), v.detach(), k_pages, v_pages, block_table,
                        positions, seq_ids)


def copy_pages(pools: Sequence[torch.Tensor], src: List[int],
               dst: List[int]) -> None:
    """pool[:, dst[i]] = pool[:, src[i]] for pools [layers, pages, ...], in
    place: a fork's last page, a shared page that is about to be written, or the
    moves of a compaction. `src` and `dst` are lists of ints, since tables are
    kept on the host too; nothing is copied to the device for them. A page is
    written once at most and is not both read and written."""
    if len(pools) and use_hip(pools[0]):
        get_ext().copy_pages(list(pools), src, dst)
        return
    ref.copy_pages(pools, src, dst)
