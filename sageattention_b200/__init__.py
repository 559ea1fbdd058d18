"""B200-native NVFP4 attention (SageAttention3 path): thin PyTorch front end over ``libsage3_b200.so``."""
from .api import (sageattn, sageattn3_blackwell, sageattn4_blackwell, pack_kv, sageattn_varlen, sageattn_from_host, quantize_qkv, fp4_attention,
                  QuantizedQKV, buffer_sizes)
from .kv_cache import (FP4KVCache, BlockTables, build_block_tables, qk_norm_rope, qk_norm_rope_append, sageattn_kvcache)

__all__ = ["sageattn", "sageattn3_blackwell", "sageattn4_blackwell", "pack_kv", "sageattn_varlen", "sageattn_from_host", "quantize_qkv", "fp4_attention",
           "QuantizedQKV", "buffer_sizes", "FP4KVCache", "BlockTables", "build_block_tables", "qk_norm_rope", "qk_norm_rope_append",
           "sageattn_kvcache"]
