"""MI355X-native block-sparse attention hot path of EchoSparse / VSA (reference package `echosparse`).

Public surface (mirrors the reference's):
  EchoSparseAttention       LSE-guided block-sparse self-attention (attention.py)
  enable, PRESETS           route a diffusers pipeline's self-attention through it (models/)
  backends                  device -> kernel set resolution ("auto" / "mi355x")
  packed_attention, relative_buckets, shared_prefix_attention
                            attention over packed sequences, its position bias, and over a shared prefix (packed.py)
  norm_rotate, rotary_table norms of queries and keys for each head with their position rotation (rotary.py)
  PagedCache, paged_cache, append_paged, paged_attention, paged_rows
                            paged caches of keys and values in 16 or 4 bits and attention over them (paged.py)
  kernels.gfx950            the kernel set (plugin interface), HIP kernels behind libechosparse_hip.so
"""
from .attention import EchoSparseAttention
from .models import PRESETS, enable
from .packed import packed_attention, relative_buckets, shared_prefix_attention
from .paged import PagedCache, append_paged, paged_attention, paged_cache, paged_rows
from .rotary import norm_rotate, rotary_table

__all__ = ["EchoSparseAttention", "PRESETS", "PagedCache", "append_paged", "enable", "norm_rotate", "packed_attention",
           "paged_attention", "paged_cache", "paged_rows", "relative_buckets", "rotary_table", "shared_prefix_attention"]
__version__ = "0.1.0"
