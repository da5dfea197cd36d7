"""MI355X (gfx950) paged-KV decode path for InferKernelLab.

Hand-written HIP kernels (KV append, fused RoPE + append with and without
norms of the heads, paged decode attention with split partitions, paged
prefill attention, page copies, token sampling, linear layers over 4-bit weights
and rows in 8 bits) behind the C ABI of include/ikl_paged.h, with the reference's
operator surface (ops), the drawing of tokens (sampling), the quantised layers'
operators (quantized), paged cache (cache), scheduler and runtime hooks, and
the decode runners that call them (decode: synthetic decoder; llama: Llama
over the paged cache).
"""

from .cache import BlockAllocator, CacheLayout, PagedKVCache
from .ops import (
    append_kv_hip,
    append_kv_triton,
    copy_blocks_hip,
    hip_append_available,
    hip_available,
    paged_decode_attention_hip,
    paged_decode_attention_hip_grouped,
    paged_decode_attention_triton,
    paged_decode_attention_triton_grouped,
    paged_decode_autotune_config,
    paged_decode_grouped_autotune_config,
    paged_decode_grouped_dot_autotune_config,
    paged_decode_grouped_path,
    paged_decode_step_hip,
    paged_prefill_attention_hip,
    paged_prefill_path,
    PreparedAppend,
    PreparedDecodeStep,
    PreparedPagedAttention,
    PreparedPagedPrefill,
    PreparedQKNormRopeAppend,
    qk_norm_rope_append_kv_hip,
    rope_append_kv_hip,
    triton_append_available,
    triton_available,
)
from .quantized import (
    add_rms_norm_int8_hip,
    int4_linear_hip,
    Int4Weight,
    Int8Rows,
    pack_int4_weight,
    PreparedAddRMSNormInt8,
    PreparedInt4Linear,
    PreparedQuantizeRowsInt8,
    PreparedSiluMulInt8,
    quantize_int4_weight,
    quantize_rows_int8_hip,
    silu_mul_int8_hip,
)
from .runtime import InferenceRuntime, RuntimeStats
from .sampling import PreparedSampler, sample_tokens_hip
from .scheduler import InferenceRequest, ScheduleBatch, TokenBudgetScheduler

__all__ = [
    "BlockAllocator",
    "CacheLayout",
    "PagedKVCache",
    "InferenceRequest",
    "ScheduleBatch",
    "TokenBudgetScheduler",
    "InferenceRuntime",
    "RuntimeStats",
    "append_kv_hip",
    "append_kv_triton",
    "hip_available",
    "hip_append_available",
    "paged_decode_attention_hip",
    "paged_decode_attention_hip_grouped",
    "paged_decode_attention_triton",
    "paged_decode_attention_triton_grouped",
    "paged_decode_grouped_path",
    "paged_decode_step_hip",
    "PreparedAppend",
    "PreparedDecodeStep",
    "PreparedPagedAttention",
    "paged_prefill_attention_hip",
    "paged_prefill_path",
    "PreparedPagedPrefill",
    "rope_append_kv_hip",
    "copy_blocks_hip",
    "qk_norm_rope_append_kv_hip",
    "PreparedQKNormRopeAppend",
    "Int4Weight",
    "Int8Rows",
    "pack_int4_weight",
    "quantize_int4_weight",
    "int4_linear_hip",
    "quantize_rows_int8_hip",
    "add_rms_norm_int8_hip",
    "silu_mul_int8_hip",
    "PreparedInt4Linear",
    "PreparedQuantizeRowsInt8",
    "PreparedAddRMSNormInt8",
    "PreparedSiluMulInt8",
    "sample_tokens_hip",
    "PreparedSampler",
    "paged_decode_autotune_config",
    "paged_decode_grouped_autotune_config",
    "paged_decode_grouped_dot_autotune_config",
    "triton_available",
    "triton_append_available",
]
