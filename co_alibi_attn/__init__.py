"""MI355X-native Co-ALiBi attention (drop-in for Nathancgy/Co-ALIBI's co_alibi_attn)."""
from .co_alibi_attn import co_alibi_attention, co_alibi_decode
from .serving import co_alibi_cache_append, co_alibi_decode_tree, co_alibi_sample  # noqa: F401

# What a star import takes: the reference's name and the decode.  The serving step is imported by name.
__all__ = ["co_alibi_attention", "co_alibi_decode"]
