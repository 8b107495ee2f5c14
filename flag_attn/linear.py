"""``flag_attn.linear`` -- linear attention with a decay per head: ``attention`` over packed sequences,
``decode`` for one token per sequence.  Implemented in ``flagattention_amd.linear``."""
from flagattention_amd.linear import linear_attention_decode as decode  # noqa: F401
from flagattention_amd.linear import linear_attention_varlen as attention  # noqa: F401

__all__ = ["attention", "decode"]
