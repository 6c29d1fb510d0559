"""Sparse MLA (examples/sparse_attention in the reference) on MI355X, with the rotation and the append that fill its
caches and the dense attention over a latent cache."""

from .attention import sparse_mla, sparse_mla_planned
from .cache import append_paged_kv
from .gather import sparse_mla_gather
from .indexer import sparse_topk_indices
from .latent import latent_attention
from .ops import sparse_flash_mla
from .rotary import apply_rotary, rotary_frequencies, rotary_magnitude

__all__ = ["sparse_mla", "sparse_mla_planned", "sparse_mla_gather", "sparse_flash_mla", "sparse_topk_indices",
           "apply_rotary", "rotary_frequencies", "rotary_magnitude", "append_paged_kv", "latent_attention"]
