"""Flash attention and the teaching attention (examples/flash_attention in the reference), and the prompt attention of
latent models."""

from .attention import attention_target, causal_policy
from .expanded import latent_attention_expanded
from .simple import simple_attention

__all__ = ["attention_target", "causal_policy", "latent_attention_expanded", "simple_attention"]
