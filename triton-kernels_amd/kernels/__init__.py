"""MI355X-native attention kernels: drop-in for the attention entry points of
harsh-vsingh/triton-kernels ``kernels/__init__.py`` (flash_attention_v1/v2
from ``kernels.attention``, ``decode_attention`` from ``kernels.decode``,
``speculative_decode_attention`` from ``kernels.speculative_decode``), and the
operators around them: query/key norms with rotation, the paged cache in 4 bits
and decode attention over it."""

from .attention import flash_attention_v1, flash_attention_v2
from .decode import decode_attention
from .decode_fp4 import decode_attention_fp4, speculative_decode_attention_fp4
from .fp4_cache import Fp4Cache, allocate_fp4_cache, paged_kv_append_fp4, paged_kv_gather_fp4
from .norm_rope import build_rope_table, qk_norm_rope
from .speculative_decode import speculative_decode_attention

__all__ = [
    "flash_attention_v1",
    "flash_attention_v2",
    "speculative_decode_attention",
    "decode_attention",
    "decode_attention_fp4",
    "speculative_decode_attention_fp4",
    "Fp4Cache",
    "allocate_fp4_cache",
    "paged_kv_append_fp4",
    "paged_kv_gather_fp4",
    "build_rope_table",
    "qk_norm_rope",
]
