"""``flag_attn.varlen`` -- ``attention`` is prompt attention over packed sequences of different
lengths, implemented in ``flagattention_amd.varlen.flash_attention_varlen``."""
from flagattention_amd.varlen import flash_attention_varlen as attention  # noqa: F401

__all__ = ["attention"]
