"""Fused op layer: hand-written CDNA4 (gfx950) HIP kernels with autograd,
plus pure-PyTorch CPU reference implementations."""

from . import reference
from .interface import (
    adamw_step,
    can_flash_attention,
    flash_attention,
    fused_cross_entropy,
    get_ext,
    has_ext,
    l2norm_sq,
    rmsnorm,
    rope,
    swiglu, swiglu_fused,
)
from .logprobs import TokenLogprobs, token_logprobs
from .packed import flash_attention_packed, packed_positions
from .paged import (
    copy_pages,
    page_width,
    paged_attention,
    paged_kv_append,
)
from .reference import rope_cache

__all__ = [
    "TokenLogprobs", "adamw_step", "can_flash_attention", "copy_pages",
    "flash_attention", "flash_attention_packed", "fused_cross_entropy",
    "get_ext", "has_ext", "l2norm_sq", "packed_positions", "page_width",
    "paged_attention", "paged_kv_append",
    "reference", "rmsnorm", "rope", "rope_cache", "swiglu", "swiglu_fused",
    "token_logprobs",
]
