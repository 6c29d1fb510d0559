"""Sparse MLA (examples/sparse_attention in the reference) on MI355X, with the rotation and the append that fill its
caches, the dense attention over a latent cache, the append to a cache held in 8 bits, and the upkeep of pages."""

from .attention import sparse_mla, sparse_mla_planned
from .cache import append_paged_kv
from .gather import sparse_mla_gather
from .indexer import sparse_topk_indices
from .latent import latent_attention
from .ops import sparse_flash_mla
from .pages import compact_pages, copy_pages, fork_pages
from .quantized import append_quantized_kv
from .rotary import apply_rotary, rotary_frequencies, rotary_magnitude

__all__ = ["sparse_mla", "sparse_mla_planned", "sparse_mla_gather", "sparse_flash_mla", "sparse_topk_indices",
           "apply_rotary", "rotary_frequencies", "rotary_magnitude", "append_paged_kv", "latent_attention",
           "append_quantized_kv", "copy_pages", "fork_pages", "compact_pages"]
