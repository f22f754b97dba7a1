"""MI355X-native fused 2D axial RoPE + FlashAttention-style SDPA (fwd + bwd).

Drop-in for the public API of v1kstrand/triton_fused_rope_flash_attn
("fa_rope_full .py"): ``CosSinTable``, ``build_axial_rope_pairs``,
``sdpa_triton_fa_rope`` and ``TritonAttention``, backed by hand-written
gfx950 HIP kernels in libfarope.so (C ABI: include/farope.h), and
``RoPEAttention``, the ViT attention sub-layer that calls it; and the same rotary
attention for models that read or write tokens in order: ``sdpa_rope_varlen``
(packed sequences), ``rope_cache_append``, ``sdpa_rope_decode`` and ``sdpa_rope_tree`` (a paged cache),
``rope_cache_accept`` and ``rope_cache_fork`` (its rows and pages).
"""
from .rope import CosSinTable, build_axial_rope_pairs, pack_rope_tables
from .attention import TritonAttention, _sdpa_comp_dtype, sdpa_triton_fa_rope
from .block import RoPEAttention
from .pages import rope_cache_accept, rope_cache_fork
from .sequences import rope_cache_append, sdpa_rope_decode, sdpa_rope_tree, sdpa_rope_varlen

__all__ = [
    "CosSinTable",
    "build_axial_rope_pairs",
    "pack_rope_tables",
    "sdpa_triton_fa_rope",
    "TritonAttention",
    "RoPEAttention",
    "sdpa_rope_varlen",
    "rope_cache_append",
    "sdpa_rope_decode",
    "sdpa_rope_tree",
    "rope_cache_accept",
    "rope_cache_fork",
]
