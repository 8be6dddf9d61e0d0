"""mitten_amd — MI355X-native paged-KV hot path of the mitten inference engine.

Device side (libmitten_kv.so, hand-written gfx950 HIP):
    DeviceKvPool      the device KV pool and its operations (append, gather,
                      copy_blocks, decode_attention, extend_attention, and
                      qk_norm_rope_append, the fused norm + RoPE + append
                      step before attention)
    DeviceStatePool   the states of linear-attention layers (linear_extend,
                      linear_step, copy_states), beside add_rms_norm, the
                      residual + norm between layers
    DeviceKv8Pool     the K/V pool in 8 bits: e4m3 tiles with a power-of-two
                      scale per block and head, the steps that write it
                      (append, qk_norm_rope_append), gather, copy_blocks and
                      attention over it (decode_step, extend_attention)
Host side (libmitten_kvhost.so, C++):
    KvCachePool, PageTable, RadixCache, BlockManager
                      the engine's page allocator, radix prefix cache and
                      block-table bookkeeping (inference-engine/src/*.rs)
"""
from .device_pool import (  # noqa: F401
    BackendError,
    DeviceIndexError,
    DeviceKvPool,
    EngineError,
    OutOfKvPages,
    PoolDesc,
    required_bytes,
    rope_inv_freq,
    validate_block_tables,
    validate_copy_pairs,
    validate_slots,
)
from .kv8_pool import (  # noqa: F401
    KV8_MIN_EXP,
    DeviceKv8Pool,
    kv8_required_bytes,
    rope_scaled_inv_freq,
)
from .state_pool import (  # noqa: F401
    STATE_NONE,
    DeviceStatePool,
    StateDesc,
    add_rms_norm,
    state_required_bytes,
)

__version__ = "0.1.0"
