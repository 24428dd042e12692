"""uocr_moe: the DeepSeek-V2 routed-expert MoE block of unlimited-ocr-max on MI355X (gfx950).

The product is the HIP library ``libuocr_moe.so`` behind a C ABI
(``include/uocr_moe.h``); this package is its Python host side, mirroring the
reference's op names (:mod:`uocr_moe.ops`) and MoE module (:mod:`uocr_moe.moe`),
plus the ops either side of the block on the decode path (RMSNorm, RoPE, the
paged attention of a decode step and of a chunk of new tokens, the page pool's
copies, forks and compaction, an int8 pool, trees of drafted tokens, the dense
projections and lm_head GEMV, the n-gram guard, beams) and the decode step they make up (:mod:`uocr_moe.decoder`).
"""

from ._lib import LIB_PATH, UocrError
from .checkpoint import WeightMappingError, load_safetensors, moe_from_checkpoint, moe_layer_weights
from .decoder import Decoder, DecoderConfig, DecoderLayer, rope_tables
from .moe import MoE, MoeConfig, decode_stack, fused_status, gate
from .ops import (
    Beams,
    PagedChunk,
    PagedKv,
    accept_drafts,
    beam_select,
    compact_pages,
    copy_pages,
    custom,
    dense_bf16_qmv,
    dequantize_pages,
    draft_masks,
    fork_pages,
    int8_dequant_expert,
    int8_kv_blocks,
    kblocked,
    moe_bf16_qmv,
    moe_int8_qmv,
    ngram_block,
    paged_chunk_attention,
    paged_chunk_attention_qkv,
    paged_decode_attention,
    paged_decode_attention_qkv,
    quantize_pages,
    quantize_per_group,
    resize_pages,
    rms_norm,
    rms_norm_dense_bf16_qmv,
    rope,
    swiglu,
)

__all__ = [
    "Beams",
    "Decoder",
    "DecoderConfig",
    "DecoderLayer",
    "LIB_PATH",
    "MoE",
    "MoeConfig",
    "PagedChunk",
    "PagedKv",
    "UocrError",
    "WeightMappingError",
    "accept_drafts",
    "beam_select",
    "compact_pages",
    "copy_pages",
    "custom",
    "decode_stack",
    "dense_bf16_qmv",
    "dequantize_pages",
    "draft_masks",
    "fork_pages",
    "fused_status",
    "gate",
    "int8_dequant_expert",
    "int8_kv_blocks",
    "kblocked",
    "load_safetensors",
    "moe_bf16_qmv",
    "moe_from_checkpoint",
    "moe_int8_qmv",
    "moe_layer_weights",
    "ngram_block",
    "paged_chunk_attention",
    "paged_chunk_attention_qkv",
    "paged_decode_attention",
    "paged_decode_attention_qkv",
    "quantize_pages",
    "quantize_per_group",
    "resize_pages",
    "rms_norm",
    "rms_norm_dense_bf16_qmv",
    "rope",
    "rope_tables",
    "swiglu",
]
