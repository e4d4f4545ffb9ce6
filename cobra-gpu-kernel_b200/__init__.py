"""cobra-gpu-kernel_b200: the reference's single transformer-layer forward on B200.

Public API (mirrors dalberrt/COBRA-GPU-Kernel's drop-in module):
    TransformerConfig, B200TransformerLayer, SelfAttentionWeights
    ShardedLayer / sharded_forward: the layer split by batch over one process per GPU
    HeadShardedLayer / head_sharded_forward: split by head, for batches smaller than the GPU count
    B200Transformer (= UserOptimizedTransformer): the full stack, blocks with the GELU FFN
    kv_plan / kv_append / kv_read / kv_attention: a paged 8-bit key/value cache
        (KVCache, KVPool, new_kv_cache) and attention of new tokens over it;
        forward_cached of the layer and the stack run a step on them
Native boundary: ``include/cobra_b200.h`` (ctypes binding in ``_lib``).
"""

from .layer import B200TransformerLayer, SelfAttentionWeights, TransformerConfig  # noqa: F401
from . import _lib  # noqa: F401
from .sharding import ShardedLayer, batch_shards, sharded_forward  # noqa: F401
from .headshard import HeadShardedLayer, head_sharded_forward, head_shards  # noqa: F401
from .kvcache import (KVCache, KVPlan, KVPool, kv_append, kv_attention, kv_check_status, kv_plan, kv_read,  # noqa: F401
                      new_kv_cache, padded_head_dim)
from .model import B200Transformer, B200TransformerBlock, UserOptimizedTransformer  # noqa: F401

__all__ = ["B200TransformerLayer", "SelfAttentionWeights", "TransformerConfig",
           "ShardedLayer", "batch_shards", "sharded_forward",
           "HeadShardedLayer", "head_sharded_forward", "head_shards",
           "KVCache", "KVPlan", "KVPool", "kv_plan", "kv_append", "kv_read", "kv_attention", "kv_check_status",
           "new_kv_cache", "padded_head_dim",
           "B200Transformer", "B200TransformerBlock", "UserOptimizedTransformer"]
