"""MI355X-native block-sparse attention hot path of EchoSparse / VSA (reference package `echosparse`).

Public surface (mirrors the reference's):
  EchoSparseAttention       LSE-guided block-sparse self-attention (attention.py)
  enable, PRESETS           route a diffusers pipeline's self-attention through it (models/)
  backends                  device -> kernel set resolution ("auto" / "mi355x")
  packed_attention, relative_buckets, shared_prefix_attention
                            attention over packed sequences, its position bias, and over a shared prefix (packed.py)
  kernels.gfx950            the kernel set (plugin interface), HIP kernels behind libechosparse_hip.so
"""
from .attention import EchoSparseAttention
from .models import PRESETS, enable
from .packed import packed_attention, relative_buckets, shared_prefix_attention

__all__ = ["EchoSparseAttention", "PRESETS", "enable", "packed_attention", "relative_buckets",
           "shared_prefix_attention"]
__version__ = "0.1.0"
