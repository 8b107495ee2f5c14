"""``flag_attn.mxfp4`` -- the paged K/V cache in 4 bits: ``cache_kv`` writes new tokens, ``gather_kv``
reads contexts back, ``attention`` is one-token decode over it.  Implemented in
``flagattention_amd.mxfp4``."""
from flagattention_amd.mxfp4 import cache_kv_mxfp4 as cache_kv  # noqa: F401
from flagattention_amd.mxfp4 import gather_kv_mxfp4 as gather_kv  # noqa: F401
from flagattention_amd.mxfp4 import paged_attention_mxfp4 as attention  # noqa: F401

__all__ = ["attention", "cache_kv", "gather_kv"]
