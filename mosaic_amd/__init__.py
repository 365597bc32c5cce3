"""mosaic_amd: Mosaic's block-sparse attention on the HEALPix mesh, as HIP kernels for MI355X.

Drop-in Python surface of the reference op (primitives.py / ops.py):
``mosaic_attn_func``, ``block_attention``, ``attn_topk``, ``mosaic_sparse_attn``,
``MosaicAttnFunction``, ``RoPE``, ``MosaicAttention``; ``mosaic_attn_func_rope`` runs the op
with the input side's RoPE fused into its pooling pass.  For query tokens that are not the mesh
itself: ``query_topk`` and ``query_sparse_attn`` (together ``mosaic_query_attn``), each token's own key
blocks and the attention over them; ``rope_axes`` and ``qk_norm_rope``, rotary positions with several
axes and the norm of query and key heads.  For states that stay on the card: ``KVCache``, keys and values
in 8 bits, ``kv_cache_write`` and ``kv_cache_read``, and the attention over them, ``cache_attn`` and
``cache_query_attn``.  All compute runs in libmosaic_bsa.so
(built with ``python -m mosaic_amd.build``) through its C ABI (include/mosaic_bsa.h).
"""

from .ops import MosaicAttnFunction, mosaic_attn_bwd, mosaic_attn_fwd, mosaic_sparse_attn
from .primitives import (
    MosaicAttention,
    RoPE,
    attn_topk,
    block_attention,
    dense_attention,
    mosaic_attn_func,
    mosaic_attn_func_rope,
    mosaic_attn_proj,
    pool_mean,
    stack_projection_weight,
)
from .kvcache import KVCache, cache_attn, cache_query_attn, kv_cache_read, kv_cache_write
from .query import mosaic_query_attn, query_sparse_attn, query_topk
from .rotary import qk_norm_rope, rope_axes
from .healpix import get_healpix_grid, pix2ang_nest

__all__ = [
    "MosaicAttnFunction", "mosaic_attn_bwd", "mosaic_attn_fwd", "mosaic_sparse_attn", "MosaicAttention", "RoPE",
    "attn_topk", "block_attention", "dense_attention", "mosaic_attn_func", "mosaic_attn_func_rope", "mosaic_attn_proj",
    "stack_projection_weight", "pool_mean",
    "query_topk", "query_sparse_attn", "mosaic_query_attn", "rope_axes", "qk_norm_rope",
    "KVCache", "kv_cache_write", "kv_cache_read", "cache_attn", "cache_query_attn",
    "get_healpix_grid", "pix2ang_nest",
]
