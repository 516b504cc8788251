"""ctypes binding of ``libtorchtune_amd.so`` (the C ABI declared in ``include/torchtune_amd.h``).

The library is the only compute path of this package: if it cannot be loaded, every op raises.  There is no
eager-PyTorch or CPU substitute behind it.
"""
from __future__ import annotations

import ctypes
import os
import threading
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "lib" / "libtorchtune_amd.so"
ABI_VERSION = 1

TTAMD_BF16 = 0
TTAMD_F32 = 1
TTAMD_MXFP4 = 4
TTAMD_MXFP8 = 8

_c_void_p = ctypes.c_void_p
_i64 = ctypes.c_int64
_u32 = ctypes.c_uint32
_int = ctypes.c_int
_f32 = ctypes.c_float
_size = ctypes.c_size_t

# name -> (restype, argtypes); one entry per symbol declared in include/torchtune_amd.h
SIGNATURES = {
    "ttamd_version": (_int, []),
    "ttamd_last_error": (ctypes.c_char_p, []),
    "ttamd_nf4_quantize_workspace_bytes": (_size, [_i64, _int]),
    "ttamd_nf4_quantize_with_codes": (
        _int,
        [_c_void_p, _int, _i64, _int, _int, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _size, _c_void_p],
    ),
    "ttamd_nf4_quantize": (
        _int,
        [_c_void_p, _int, _i64, _int, _int, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _size, _c_void_p],
    ),
    "ttamd_nf4_dequantize": (
        _int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _int, _i64, _int, _int, _c_void_p, _c_void_p],
    ),
    "ttamd_nf4_block_scalers": (_int, [_c_void_p, _c_void_p, _c_void_p, _int, _i64, _int, _c_void_p, _c_void_p]),
    "ttamd_nf4_dequantize_merge_bf16": (_int, [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _int, _f32, _c_void_p, _i64, _i64, _c_void_p]),
    "ttamd_lora_fwd_workspace_bytes": (_size, [_i64, _i64, _int]),
    "ttamd_lora_hidden_bf16": (_int, [_c_void_p, _c_void_p, _c_void_p, _i64, _i64, _int, _c_void_p, _size, _c_void_p]),
    "ttamd_lora_hidden_static_max_bytes": (_size, []),
    "ttamd_lora_hidden_static_init": (_int, []),
    "ttamd_lora_hidden_static_bf16": (_int, [_c_void_p, _c_void_p, _c_void_p, _i64, _i64, _int, _c_void_p]),
    "ttamd_nf4_lora_linear_fwd_bf16": (
        _int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _int, _f32, _c_void_p, _c_void_p, _i64, _i64, _i64,
         _c_void_p],
    ),
    "ttamd_dora_weight_norm_workspace_bytes": (_size, [_i64, _i64]),
    "ttamd_nf4_dora_weight_norm_bf16": (
        _int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _int, _f32, _c_void_p, _c_void_p, _c_void_p, _i64, _i64, _c_void_p, _size,
         _c_void_p],
    ),
    "ttamd_nf4_dora_linear_fwd_bf16": (
        _int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _int, _f32, _c_void_p, _c_void_p, _c_void_p, _i64, _i64,
         _i64, _c_void_p],
    ),
    "ttamd_dora_bwd_workspace_bytes": (_size, [_i64]),
    "ttamd_dora_bwd_prologue_bf16": (
        _int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _i64, _i64, _c_void_p, _size, _c_void_p],
    ),
    "ttamd_nf4_transpose_for_backward": (_int, [_c_void_p, _c_void_p, _i64, _i64, _c_void_p, _c_void_p, _c_void_p]),
    "ttamd_nf4_linear_bwd_dx_bf16": (
        _int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _int, _c_void_p, _i64, _i64, _i64,
         _c_void_p],
    ),
    "ttamd_nf4_gemm_workspace_bytes": (_size, [_i64, _i64, _i64]),
    "ttamd_nf4_gemm_expands_weight": (_int, [_i64, _i64, _i64]),
    "ttamd_nf4_lora_linear_fwd_ws_bf16": (
        _int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _int, _f32, _c_void_p, _c_void_p, _c_void_p, _i64, _i64,
         _i64, _c_void_p, _size, _c_void_p],
    ),
    "ttamd_nf4_linear_bwd_dx_ws_bf16": (
        _int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _int, _c_void_p, _i64, _i64, _i64,
         _c_void_p, _size, _c_void_p],
    ),
    "ttamd_nf4_linear_bwd_dx_swiglu_ws_bf16": (
        _int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _int, _c_void_p, _c_void_p, _c_void_p,
         _c_void_p, _i64, _i64, _i64, _c_void_p, _size, _c_void_p],
    ),
    "ttamd_lora_bwd_workspace_bytes": (_size, [_i64, _i64, _i64, _int]),
    "ttamd_lora_bwd_bf16": (
        _int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _f32, _c_void_p, _c_void_p, _c_void_p, _i64, _i64, _i64, _int,
         _c_void_p, _size, _c_void_p],
    ),
    "ttamd_qlora_linear_fwd_workspace_bytes": (_size, [_i64, _i64, _i64, _int]),
    "ttamd_qlora_linear_fwd_bf16": (
        _int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _int, _f32, _c_void_p, _c_void_p, _c_void_p, _i64, _i64,
         _i64, _c_void_p, _size, _c_void_p],
    ),
    "ttamd_qlora_linear_bwd_workspace_bytes": (_size, [_i64, _i64, _i64, _int]),
    "ttamd_qlora_linear_bwd_bf16": (
        _int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _int, _f32,
         _c_void_p, _c_void_p, _c_void_p, _i64, _i64, _i64, _c_void_p, _size, _c_void_p],
    ),
    "ttamd_lora_group_hidden_workspace_bytes": (_size, [_c_void_p, _int, _i64, _i64]),
    "ttamd_lora_group_hidden_bf16": (_int, [_c_void_p, _c_void_p, _int, _c_void_p, _i64, _i64, _c_void_p, _size, _c_void_p]),
    "ttamd_lora_group_fwd_workspace_bytes": (_size, [_c_void_p, _int, _i64, _i64]),
    "ttamd_nf4_lora_group_fwd_bf16": (_int, [_c_void_p, _c_void_p, _int, _c_void_p, _i64, _i64, _c_void_p, _size, _c_void_p]),
    "ttamd_lora_few_fwd_applies": (_int, [_c_void_p, _int, _i64, _i64, _int]),
    "ttamd_lora_few_fwd_bf16": (_int, [_c_void_p, _c_void_p, _int, _c_void_p, _c_void_p, _i64, _i64, _c_void_p]),
    "ttamd_nf4_lora_group_swiglu_fwd_bf16": (_int, [_c_void_p, _c_void_p, _int, _c_void_p, _c_void_p, _i64, _i64, _c_void_p, _size,
                                                    _c_void_p]),
    "ttamd_lora_group_bwd_workspace_bytes": (_size, [_c_void_p, _int, _i64, _i64]),
    "ttamd_lora_group_bwd_bf16": (_int, [_c_void_p, _c_void_p, _c_void_p, _int, _c_void_p, _i64, _i64, _c_void_p, _size, _c_void_p]),
    "ttamd_lora_group_swiglu_bwd_bf16": (_int, [_c_void_p, _c_void_p, _c_void_p, _int, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _i64, _i64, _c_void_p, _size, _c_void_p]),
    "ttamd_nf4_group_bwd_dx_bf16": (_int, [_c_void_p, _int, _c_void_p, _c_void_p, _i64, _i64, _c_void_p]),
    "ttamd_nf4_group_bwd_dx_workspace_bytes": (_size, [_c_void_p, _int, _i64, _i64]),
    "ttamd_nf4_group_bwd_dx_ws_bf16": (_int, [_c_void_p, _int, _c_void_p, _c_void_p, _i64, _i64, _c_void_p, _size, _c_void_p]),
    "ttamd_nf4_group_fwd_leaves_tiles": (_int, [_c_void_p, _int, _i64, _i64, _int]),
    "ttamd_nf4_group_bwd_dx_tiles_bf16": (_int, [_c_void_p, _int, _c_void_p, _c_void_p, _i64, _i64, _c_void_p, _int, _c_void_p]),
    "ttamd_nf4_lora_group_fwd_tiles_bf16": (_int, [_c_void_p, _c_void_p, _int, _c_void_p, _c_void_p, _i64, _i64, _c_void_p, _int, _c_void_p]),
    "ttamd_tiled_weight_bytes": (_size, [_i64, _i64]),
    "ttamd_gemm_tn_applies": (_int, [_i64, _i64, _i64]),
    "ttamd_gemm_tn_bf16": (_int, [_c_void_p, _c_void_p, _c_void_p, _i64, _i64, _i64, _c_void_p]),
    "ttamd_gemm_tn_group_bf16": (_int, [_c_void_p, _c_void_p, _c_void_p, _int, _i64, _c_void_p, _i64, _c_void_p]),
    "ttamd_gemm_tn_workspace_bytes": (_size, [_i64, _i64, _i64]),
    "ttamd_gemm_tn_ws_bf16": (_int, [_c_void_p, _c_void_p, _c_void_p, _i64, _i64, _i64, _c_void_p, _size, _c_void_p]),
    "ttamd_gemm_tn_group_ws_bf16": (_int, [_c_void_p, _c_void_p, _c_void_p, _int, _i64, _c_void_p, _i64, _c_void_p, _size, _c_void_p]),
    "ttamd_fq_per_group_int4_sym_tiled_bf16": (_int, [_c_void_p, _i64, _i64, _int, _int, _f32, _c_void_p, _c_void_p, _c_void_p, _c_void_p]),
    "ttamd_tiled_linear_bf16": (_int, [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _i64, _i64, _i64, _c_void_p]),
    "ttamd_tiled_lora_linear_bf16": (_int, [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _int, _int, _f32, _c_void_p, _c_void_p, _i64, _i64,
                                            _i64, _c_void_p]),
    "ttamd_fq_per_group_int4_sym_tiled_at_bf16": (_int, [_c_void_p, _i64, _i64, _int, _int, _f32, _c_void_p, _int, _c_void_p, _i64, _i64,
                                                         _c_void_p, _c_void_p]),
    "ttamd_tiled_linear_group_fwd_bf16": (_int, [_c_void_p, _c_void_p, _int, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _i64, _i64,
                                                 _c_void_p]),
    "ttamd_tiled_linear_group_dx_bf16": (_int, [_c_void_p, _c_void_p, _int, _c_void_p, _c_void_p, _i64, _i64, _c_void_p]),
    "ttamd_tiled_linear_dx_bf16": (_int, [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _int, _c_void_p, _i64, _i64, _i64, _c_void_p]),
    "ttamd_fq_per_token_int8_asym": (_int, [_c_void_p, _int, _i64, _i64, _int, _c_void_p, _c_void_p, _c_void_p, _c_void_p]),
    "ttamd_fq_per_group_int4_sym": (_int, [_c_void_p, _int, _i64, _i64, _int, _int, _c_void_p, _c_void_p, _c_void_p]),
    "ttamd_quantize_per_group_int4": (
        _int,
        [_c_void_p, _int, _i64, _i64, _int, _int, _c_void_p, _c_void_p, _c_void_p, _c_void_p],
    ),
    "ttamd_dequantize_per_group_int4": (_int, [_c_void_p, _c_void_p, _c_void_p, _int, _i64, _i64, _int, _c_void_p, _c_void_p]),
    "ttamd_fq_per_group_uint4_asym": (
        _int, [_c_void_p, _int, _i64, _i64, _int, _int, _c_void_p, _c_void_p, _c_void_p, _c_void_p]),
    "ttamd_quantize_per_group_uint4": (
        _int, [_c_void_p, _int, _i64, _i64, _int, _int, _c_void_p, _c_void_p, _c_void_p, _c_void_p]),
    "ttamd_dequantize_per_group_uint4": (_int, [_c_void_p, _c_void_p, _c_void_p, _int, _i64, _i64, _int, _c_void_p, _c_void_p]),
    "ttamd_gemm_mid_workspace_bytes": (_size, [_i64, _i64, _i64]),
    "ttamd_nf4_gemm_plan": (_int, [_i64, _i64, _i64, _int, _int, _int, _c_void_p, _c_void_p, _c_void_p]),
    "ttamd_gemm_mid_plan": (_int, [_int, _int, _i64, _i64, _i64, _c_void_p, _c_void_p, _c_void_p]),
    "ttamd_gemm_mid_bf16": (_int, [_int, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _i64, _i64, _i64, _c_void_p, _size, _c_void_p]),
    "ttamd_int4_linear_applies": (_int, [_i64, _i64, _i64, _int]),
    "ttamd_int4_linear_workspace_bytes": (_size, [_i64, _i64, _i64]),
    "ttamd_int8_group_linear_bf16": (
        _int, [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _int, _int, _c_void_p, _c_void_p, _i64, _i64, _i64, _c_void_p, _size, _c_void_p]),
    "ttamd_int8_dynamic_linear_workspace_bytes": (_size, [_i64, _i64, _i64]),
    "ttamd_int8_dynamic_linear_bf16": (
        _int, [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _int, _int, _c_void_p, _c_void_p, _i64, _i64, _i64, _c_void_p, _size, _c_void_p]),
    "ttamd_uint4_group_linear_bf16": (
        _int, [_c_void_p, _c_void_p, _c_void_p, _int, _c_void_p, _c_void_p, _i64, _i64, _i64, _c_void_p, _size, _c_void_p]),
    "ttamd_fq_per_token_int8_asym_conv": (
        _int, [_c_void_p, _int, _i64, _i64, _int, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p]),
    "ttamd_fq_per_group_int4_sym_conv": (
        _int, [_c_void_p, _int, _i64, _i64, _int, _int, _c_void_p, _c_void_p, _c_void_p, _c_void_p]),
    "ttamd_quantize_per_group_int4_conv": (
        _int, [_c_void_p, _int, _i64, _i64, _int, _int, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p]),
    "ttamd_fq_per_group_uint4_asym_conv": (
        _int, [_c_void_p, _int, _i64, _i64, _int, _int, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p]),
    "ttamd_quantize_per_group_uint4_conv": (
        _int, [_c_void_p, _int, _i64, _i64, _int, _int, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p]),
    "ttamd_rms_norm_fwd_bf16": (_int, [_c_void_p, _c_void_p, _f32, _c_void_p, _c_void_p, _i64, _i64, _c_void_p]),
    "ttamd_rms_norm_bwd_workspace_bytes": (_size, [_i64]),
    "ttamd_rms_norm_bwd_bf16": (
        _int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _i64, _i64, _c_void_p, _size, _c_void_p],
    ),
    "ttamd_add_rms_norm_fwd_bf16": (_int, [_c_void_p, _c_void_p, _c_void_p, _f32, _c_void_p, _c_void_p, _c_void_p, _i64, _i64, _c_void_p]),
    "ttamd_rms_norm_bwd_add_bf16": (
        _int,
        [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _i64, _i64, _c_void_p, _size, _c_void_p],
    ),
    "ttamd_rope_bf16": (_int, [_c_void_p, _c_void_p, _c_void_p, _i64, _i64, _i64, _i64, _int, _c_void_p]),
    "ttamd_repeat_kv_bf16": (_int, [_c_void_p, _c_void_p, _i64, _i64, _i64, _i64, _c_void_p]),
    "ttamd_repeat_kv_bwd_bf16": (_int, [_c_void_p, _c_void_p, _i64, _i64, _i64, _i64, _c_void_p]),
    "ttamd_qkv_rope_repeat_bf16": (_int, [_c_void_p] * 7 + [_i64] * 5 + [_c_void_p]),
    "ttamd_qkv_rope_repeat_bwd_bf16": (_int, [_c_void_p] * 7 + [_i64] * 5 + [_c_void_p]),
    "ttamd_swiglu_fwd_bf16": (_int, [_c_void_p, _c_void_p, _c_void_p, _i64, _c_void_p]),
    "ttamd_cross_entropy_fwd_bwd_bf16": (_int, [_c_void_p, _c_void_p, _i64, _f32, _c_void_p, _c_void_p, _i64, _i64, _c_void_p]),
    "ttamd_mx_quantize": (_int, [_c_void_p, _int, _i64, _i64, _int, _c_void_p, _c_void_p, _c_void_p]),
    "ttamd_mx_dequantize": (_int, [_c_void_p, _c_void_p, _int, _i64, _i64, _int, _c_void_p, _c_void_p]),
    "ttamd_mx_linear_workspace_bytes": (_size, [_i64, _i64, _i64, _int]),
    "ttamd_mx_linear_bf16": (
        _int, [_c_void_p, _int, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _i64, _i64, _i64, _c_void_p, _size, _c_void_p]),
    "ttamd_mx_linear_dx_workspace_bytes": (_size, [_i64, _i64, _i64]),
    "ttamd_mx_linear_dx_bf16": (_int, [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _i64, _i64, _i64, _c_void_p, _size, _c_void_p]),
    "ttamd_mx_kept_codes_bytes": (_size, [_i64, _i64]),
    "ttamd_mx_kept_scales_bytes": (_size, [_i64, _i64]),
    "ttamd_mx_lora_fwd_workspace_bytes": (_size, [_c_void_p, _int, _i64, _i64]),
    "ttamd_mx_lora_fwd_bf16": (
        _int, [_c_void_p, _c_void_p, _int, _c_void_p, _c_void_p, _c_void_p, _i64, _i64, _c_void_p, _size, _c_void_p]),
    "ttamd_mx_lora_bwd_workspace_bytes": (_size, [_c_void_p, _int, _i64, _i64]),
    "ttamd_mx_lora_bwd_bf16": (
        _int, [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _int, _c_void_p, _c_void_p, _i64, _i64, _c_void_p, _size, _c_void_p]),
    "ttamd_column_sum_workspace_bytes": (_size, [_i64, _i64]),
    "ttamd_column_sum_bf16": (_int, [_c_void_p, _c_void_p, _i64, _i64, _c_void_p, _size, _c_void_p]),
    "ttamd_qk_norm_rope_fwd": (_int, [_c_void_p, _c_void_p, _int, _f32, _i64, _i64, _i64, _c_void_p]),
    "ttamd_qk_norm_rope_bwd_workspace_bytes": (_size, [_i64]),
    "ttamd_qk_norm_rope_bwd": (_int, [_c_void_p, _c_void_p, _int, _f32, _i64, _i64, _i64, _c_void_p, _size, _c_void_p]),
    "ttamd_token_logprobs_workspace_bytes": (_size, [_i64, _i64, _int]),
    "ttamd_token_logprobs_fwd": (
        _int, [_c_void_p, _c_void_p, _i64, _i64, _f32, _c_void_p, _c_void_p, _int, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _size, _c_void_p]),
    "ttamd_token_logprobs_bwd": (
        _int, [_c_void_p, _c_void_p, _i64, _i64, _f32, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p]),
    "ttamd_adamw_key": (_u32, [_i64, _i64, _u32]),
    "ttamd_adamw_number": (_u32, [_u32, _i64]),
    "ttamd_adamw_step": (_int, [_c_void_p, _int, _int, _c_void_p, _u32, _u32, _u32, _c_void_p, _c_void_p]),
    "ttamd_adamw_moments_bf16": (_int, [_c_void_p, _u32, _c_void_p, _c_void_p, _c_void_p]),
    "ttamd_swiglu_bwd_bf16": (_int, [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _i64, _c_void_p]),
}

class FqConventions(ctypes.Structure):
    """``ttamd_fq_conventions`` of the header: the version-dependent constants of the fake-quant schemes."""

    _fields_ = [("eps_per_token", ctypes.c_float), ("eps_per_group_sym", ctypes.c_float), ("min_scale_uint4", ctypes.c_float),
                ("uint4_clamp_range_first", ctypes.c_int)]


GROUP_MAX = 4


class LoraGroupMember(ctypes.Structure):
    """``ttamd_lora_group_member`` of the header: one linear of a group that shares its input."""

    _fields_ = [("quantized_data", _c_void_p), ("block_scalers", _c_void_p), ("block_scalers_t", _c_void_p),
                ("quantized_data_t", _c_void_p), ("lora_a", _c_void_p), ("lora_b", _c_void_p), ("bias", _c_void_p),
                ("y", _c_void_p), ("grad_lora_a", _c_void_p), ("grad_lora_b", _c_void_p), ("N", _i64), ("rank", _int),
                ("scale", _f32)]


class MxLoraMember(ctypes.Structure):
    """``ttamd_mx_lora_member`` of the header: one adapter linear over an mxfp4 weight."""

    _fields_ = [("codes", _c_void_p), ("scales", _c_void_p), ("lora_a", _c_void_p), ("lora_b", _c_void_p), ("bias", _c_void_p),
                ("y", _c_void_p), ("grad_lora_a", _c_void_p), ("grad_lora_b", _c_void_p), ("N", _i64), ("rank", _int), ("scale", _f32)]


class RopeHeads(ctypes.Structure):
    """``ttamd_rope_heads`` of the header: the query heads, or the key heads."""

    _fields_ = [("x", _c_void_p), ("scale", _c_void_p), ("gy", _c_void_p), ("out", _c_void_p), ("gscale", _c_void_p), ("heads", _i64),
                ("x_stride", _i64 * 3), ("gy_stride", _i64 * 3)]


class RopePositions(ctypes.Structure):
    """``ttamd_rope_positions`` of the header: the table of angles and which of its rows each token follows."""

    _fields_ = [("cache", _c_void_p), ("cache_rows", _i64), ("positions", _c_void_p), ("stride", _i64 * 3), ("n_axes", _int),
                ("section", _int * 4), ("interleaved", _int)]


class Logits(ctypes.Structure):
    """``ttamd_logits`` of the header: rows of logits at two nested strides."""

    _fields_ = [("data", _c_void_p), ("dtype", _int), ("rows", _i64), ("V", _i64), ("n_inner", _i64), ("stride_outer", _i64), ("stride_inner", _i64)]


class AdamWStates(ctypes.Structure):
    """``ttamd_adamw_states`` of the header: where the moments of many tensors lie."""

    _fields_ = [("chunks", _c_void_p), ("exp_avg", _c_void_p), ("exp_avg_sq", _c_void_p),
                ("exp_avg_exponent", _c_void_p), ("exp_avg_sq_exponent", _c_void_p), ("state_bits", _int)]


class AdamWScalars(ctypes.Structure):
    """``ttamd_adamw_scalars`` of the header."""

    _fields_ = [("lr", ctypes.c_double), ("beta1", ctypes.c_double), ("beta2", ctypes.c_double), ("eps", ctypes.c_double),
                ("weight_decay", ctypes.c_double), ("step", _i64), ("seed", _i64), ("stochastic", _int)]


_lock = threading.Lock()
_lib = None


class LibraryNotBuiltError(RuntimeError):
    pass


def load() -> ctypes.CDLL:
    """Load the shared library (once) and attach the prototypes.  Raises if it is missing or stale."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not LIB_PATH.exists():
            raise LibraryNotBuiltError(
                f"{LIB_PATH} is missing: torchtune_amd has no compute path without its HIP library. "
                "Build it with `python -m torchtune_amd.build` (needs hipcc)."
            )
        lib = ctypes.CDLL(os.fspath(LIB_PATH))
        for name, (restype, argtypes) in SIGNATURES.items():
            try:
                fn = getattr(lib, name)
            except AttributeError as err:
                raise LibraryNotBuiltError(f"{LIB_PATH} does not export {name}; rebuild it") from err
            fn.restype = restype
            fn.argtypes = argtypes
        if lib.ttamd_version() != ABI_VERSION:
            raise LibraryNotBuiltError(
                f"{LIB_PATH} has ABI version {lib.ttamd_version()}, this package needs {ABI_VERSION}; rebuild it"
            )
        _lib = lib
    return _lib


def check(rc: int, what: str) -> None:
    """Turn a negative C-ABI return code into the matching Python exception."""
    if rc == 0:
        return
    msg = load().ttamd_last_error().decode("utf-8", "replace")
    if rc == -1:
        raise ValueError(f"{what}: {msg}")
    raise RuntimeError(f"{what} failed (code {rc}): {msg}")
