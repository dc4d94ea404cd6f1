"""B200 (sm_100a) implementation of SpargeAttn's training-free sparse attention hot path.

The reference package's five names (spas_sage_attn/__init__.py:1-7), and what a model needs beside them: rotary positions and
a paged key/value cache with the attention over it."""
from .core import (
    spas_sage2_attn_meansim_cuda,
    spas_sage2_attn_meansim_topk_cuda,
    block_sparse_sage2_attn_cuda,
    spas_sage_attn_meansim_cuda,
    spas_sage_attn_meansim_topk_cuda,
)
from .paged import (
    allocate_pages,
    append_kv,
    compact_pages,
    copy_pages,
    fork_sequences,
    free_sequences,
    paged_attention,
)
from .rotary import apply_rotary, rotary_frequencies

__all__ = [
    "spas_sage2_attn_meansim_cuda",
    "spas_sage2_attn_meansim_topk_cuda",
    "block_sparse_sage2_attn_cuda",
    "spas_sage_attn_meansim_cuda",
    "spas_sage_attn_meansim_topk_cuda",
    "apply_rotary",
    "rotary_frequencies",
    "append_kv",
    "paged_attention",
    "allocate_pages",
    "free_sequences",
    "fork_sequences",
    "compact_pages",
    "copy_pages",
]
