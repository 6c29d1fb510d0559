"""Flash attention and the teaching attention (examples/flash_attention in the reference), the prompt attention of
latent models, and attention over a paged cache held in 8 bits."""

from .attention import attention_target, causal_policy
from .expanded import latent_attention_expanded
from .quantized import quantized_attention
from .simple import simple_attention

__all__ = ["attention_target", "causal_policy", "latent_attention_expanded", "quantized_attention", "simple_attention"]
