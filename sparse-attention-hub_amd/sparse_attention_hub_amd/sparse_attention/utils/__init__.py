"""Mask type, masked-softmax attention and GQA helpers of the ResearchAttention path; the paged cache and token sampling of serving."""
from .kv_utils import _get_num_key_value_groups, repeat_kv
from .mask import Mask
from .mask_attention_utils import (
    apply_inv_mask_sum,
    get_masked_attention_output,
    get_true_attention_output,
)
from .paged_cache import PageAssignment, PagedKVCache, assign_pages, paged_attention, release_pages, store_paged
from .token_sampling import sample_tokens

__all__ = [
    "Mask",
    "repeat_kv",
    "_get_num_key_value_groups",
    "apply_inv_mask_sum",
    "get_masked_attention_output",
    "get_true_attention_output",
    "PageAssignment",
    "PagedKVCache",
    "assign_pages",
    "release_pages",
    "store_paged",
    "paged_attention",
    "sample_tokens",
]
