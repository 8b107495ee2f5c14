"""``flag_attn.rotary`` -- rotary positions of one or several axes: ``embedding`` turns q and k,
``cache_kv`` turns q and writes the turned k and v into the paged cache.  Implemented in
``flagattention_amd.rotary``."""
from flagattention_amd.rotary import rotary_cache_kv as cache_kv  # noqa: F401
from flagattention_amd.rotary import rotary_embedding as embedding  # noqa: F401

__all__ = ["embedding", "cache_kv"]
