"""openasr_b200 -- B200-native (sm_100a) backend for OpenASR's inference hot
path: quantized GGML_OP_MUL_MAT and f16-KV GGML_OP_FLASH_ATTN_EXT behind a C
ABI (include/oasr_b200.h), with a Python host mirror in `backend`; drafted trees
over a paged K/V cache beside it."""
from .backend import (  # noqa: F401
    F16, F32, I32, I64, OP_ARGMAX_FIRST, OP_ATTN_WEIGHTS, OP_FLASH_ATTN_EXT, OP_FLASH_ATTN_TREE, OP_KV_EVICT,
    OP_KV_PAGES_COPY, OP_MUL_MAT, OP_QK_NORM_ROPE, OP_SET_ROWS, OP_TREE_COMMIT, OP_TREE_SAMPLE, PREC_DEFAULT,
    PREC_F32, Q4_0, Q4_K, Q8_0, Backend, GgmlBackendError, KvPool, Weight, describe, device_count, lib, quantize, row_size, synth_normal, tree_mask,
)
