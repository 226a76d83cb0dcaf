"""ctypes declarations of include/nnops_amd.h and include/nnops_amd_ops.h."""
from __future__ import annotations

import ctypes as C
import os

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libnnops_amd.so")
DIAG_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libnnops_amd_diag.so")

OK, INVALID_ARGUMENT, UNSUPPORTED, NOT_INITIALIZED, OUT_OF_MEMORY, INTERNAL = range(6)
OUT_S32, OUT_S8, OUT_U8, OUT_F32, OUT_F16 = range(5)
(ACT_NONE, ACT_RELU, ACT_GELU, ACT_SIGMOID, ACT_TANH, ACT_LEAKY_RELU, ACT_SILU, ACT_HARDSWISH, ACT_ELU,
 ACT_RELU6) = range(10)
DT_F32, DT_F16, DT_BF16, DT_S8, DT_U8, DT_S32 = 0, 1, 2, 3, 4, 5
DT_Q4_1 = 11
LAYOUT_DENSE, LAYOUT_PACKED_B_HIP = 12, 18
BACKEND_CPU, BACKEND_CUDA, BACKEND_HIP = 0, 1, 4
# EpilogueActivateType / EpilogueQuantType values
EP_NONE, EP_RELU, EP_GELU, EP_SIGMOID, EP_TANH = 0, 1, 2, 3, 4
EP_LEAKY_RELU, EP_SILU, EP_HARDSWISH, EP_ELU, EP_RELU6 = 5, 6, 7, 8, 9
EQ_NONE, EQ_REQUANTIZE, EQ_DEQUANTIZE = 0, 1, 2


class GemmI8Args(C.Structure):
    _fields_ = [
        ("a", C.c_void_p), ("b", C.c_void_p), ("bias", C.c_void_p), ("c", C.c_void_p),
        ("m", C.c_int64), ("n", C.c_int64), ("k", C.c_int64),
        ("lda", C.c_int64), ("ldb", C.c_int64), ("ldc", C.c_int64),
        ("trans_a", C.c_int32), ("trans_b", C.c_int32), ("a_u8", C.c_int32),
        ("s_a", C.c_void_p), ("s_a_scalar", C.c_float), ("zp_a", C.c_void_p), ("zp_a_scalar", C.c_int32),
        ("s_b", C.c_void_p), ("s_b_scalar", C.c_float), ("zp_b", C.c_void_p), ("zp_b_scalar", C.c_int32),
        ("s_out_rows", C.c_void_p), ("zp_out_rows", C.c_void_p), ("s_out", C.c_float), ("zp_out", C.c_int32),
        ("out_kind", C.c_int32), ("act", C.c_int32), ("round_even", C.c_int32),
        ("float_ep", C.c_int32), ("min_clip", C.c_float), ("max_clip", C.c_float),
        ("add_to", C.c_int32), ("residual_pre", C.c_int32),
        ("bias_fp", C.c_void_p), ("act_alpha", C.c_float), ("act_beta", C.c_float),
        ("b_col_sums", C.c_void_p),
    ]


class QdqArgs(C.Structure):
    _fields_ = [
        ("x", C.c_void_p), ("y", C.c_void_p),
        ("rows", C.c_int64), ("cols", C.c_int64), ("ld_x", C.c_int64), ("ld_y", C.c_int64),
        ("x_kind", C.c_int32), ("y_kind", C.c_int32), ("zp_kind", C.c_int32),
        ("scale", C.c_void_p), ("zero_point", C.c_void_p), ("scale_scalar", C.c_float),
        ("zp_scalar", C.c_int32), ("inner", C.c_int64), ("dim", C.c_int64), ("segment", C.c_int64),
    ]


class GemmQ41Args(C.Structure):
    _fields_ = [
        ("a", C.c_void_p), ("b", C.c_void_p), ("c", C.c_void_p),
        ("m", C.c_int64), ("n", C.c_int64), ("k", C.c_int64),
        ("lda", C.c_int64), ("ldc", C.c_int64), ("ldb_bytes", C.c_int64),
        ("trans_b", C.c_int32), ("a_f16", C.c_int32), ("out_kind", C.c_int32),
        ("b_soa", C.c_int32), ("b_dm", C.c_void_p), ("ldb_dm", C.c_int64),
    ]


class GemmFpArgs(C.Structure):
    _fields_ = [
        ("a", C.c_void_p), ("b", C.c_void_p), ("c", C.c_void_p),
        ("m", C.c_int64), ("n", C.c_int64), ("k", C.c_int64),
        ("lda", C.c_int64), ("ldb", C.c_int64), ("ldc", C.c_int64),
        ("trans_b", C.c_int32), ("in_f16", C.c_int32), ("out_f16", C.c_int32), ("alpha", C.c_float),
    ]


class RmsNormArgs(C.Structure):
    _fields_ = [
        ("x", C.c_void_p), ("weight", C.c_void_p), ("residual", C.c_void_p),
        ("y", C.c_void_p), ("scale", C.c_void_p), ("sum", C.c_void_p),
        ("rows", C.c_int64), ("cols", C.c_int64),
        ("ld_x", C.c_int64), ("ld_residual", C.c_int64), ("ld_y", C.c_int64), ("ld_sum", C.c_int64),
        ("in_f16", C.c_int32), ("out_kind", C.c_int32), ("epsilon", C.c_float),
    ]


class RotaryArgs(C.Structure):
    _fields_ = [
        ("x", C.c_void_p), ("y", C.c_void_p), ("positions", C.c_void_p), ("table", C.c_void_p),
        ("tokens", C.c_int64), ("heads", C.c_int64), ("head_dim", C.c_int64), ("rotary_dim", C.c_int64),
        ("max_pos", C.c_int64), ("ld_x", C.c_int64), ("ld_y", C.c_int64), ("ld_table", C.c_int64),
        ("in_f16", C.c_int32), ("interleaved", C.c_int32),
    ]


class RotaryTableArgs(C.Structure):
    _fields_ = [
        ("table", C.c_void_p), ("max_pos", C.c_int64), ("rotary_dim", C.c_int64), ("ld_table", C.c_int64),
        ("base", C.c_double), ("factor", C.c_double), ("original_context", C.c_double),
        ("low_turns", C.c_double), ("high_turns", C.c_double), ("attention_factor", C.c_double),
    ]


class KvPages(C.Structure):
    _fields_ = [
        ("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
        ("pages", C.c_int64), ("heads", C.c_int64), ("page_tokens", C.c_int64), ("head_dim", C.c_int64),
        ("page_table", C.c_void_p), ("sequences", C.c_int64), ("table_pages", C.c_int64), ("ld_table", C.c_int64),
        ("lengths", C.c_void_p), ("row_starts", C.c_void_p),
    ]


class KvRowsArgs(C.Structure):
    _fields_ = [
        ("cache", KvPages), ("k_rows", C.c_void_p), ("v_rows", C.c_void_p),
        ("rows", C.c_int64), ("ld_k", C.c_int64), ("ld_v", C.c_int64), ("f16", C.c_int32),
    ]


class CacheAttentionArgs(C.Structure):
    _fields_ = [
        ("cache", KvPages), ("q", C.c_void_p), ("out", C.c_void_p),
        ("rows", C.c_int64), ("q_heads", C.c_int64), ("ld_q", C.c_int64), ("ld_out", C.c_int64),
        ("f16", C.c_int32), ("scale", C.c_float), ("window", C.c_int64), ("sinks", C.c_int64),
    ]


class PrefixAttentionArgs(C.Structure):
    _fields_ = [
        ("cache", KvPages), ("q", C.c_void_p), ("out", C.c_void_p),
        ("rows", C.c_int64), ("q_heads", C.c_int64), ("ld_q", C.c_int64), ("ld_out", C.c_int64),
        ("f16", C.c_int32), ("scale", C.c_float),
        ("groups", C.c_int64), ("group_starts", C.c_void_p), ("shared", C.c_void_p),
    ]


class KvForkArgs(C.Structure):
    _fields_ = [
        ("page_table", C.c_void_p), ("sequences", C.c_int64), ("table_pages", C.c_int64), ("ld_table", C.c_int64),
        ("lengths", C.c_void_p), ("refs", C.c_void_p), ("pages", C.c_int64), ("page_tokens", C.c_int64),
        ("parents", C.c_void_p), ("new_tokens", C.c_void_p), ("children", C.c_int64),
        ("new_table", C.c_void_p), ("new_table_pages", C.c_int64), ("ld_new_table", C.c_int64),
        ("new_lengths", C.c_void_p), ("new_refs", C.c_void_p), ("copies", C.c_void_p), ("counts", C.c_void_p),
    ]


class KvCompactArgs(C.Structure):
    _fields_ = [
        ("page_table", C.c_void_p), ("sequences", C.c_int64), ("table_pages", C.c_int64), ("ld_table", C.c_int64),
        ("lengths", C.c_void_p), ("refs", C.c_void_p), ("pages", C.c_int64), ("page_tokens", C.c_int64),
        ("new_table", C.c_void_p), ("ld_new_table", C.c_int64), ("new_refs", C.c_void_p), ("copies", C.c_void_p),
        ("moved", C.c_void_p), ("counts", C.c_void_p),
    ]


class KvCopyArgs(C.Structure):
    _fields_ = [
        ("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
        ("pages", C.c_int64), ("heads", C.c_int64), ("page_tokens", C.c_int64), ("head_dim", C.c_int64),
        ("copies", C.c_void_p), ("count", C.c_int64),
    ]


class TokenLogProbsArgs(C.Structure):
    _fields_ = [
        ("logits", C.c_void_p), ("rows", C.c_int64), ("vocab", C.c_int64), ("ld_logits", C.c_int64),
        ("f16", C.c_int32), ("top", C.c_int32),
        ("tokens", C.c_void_p), ("per_row", C.c_int64), ("ld_tokens", C.c_int64),
        ("log_probs", C.c_void_p), ("ld_log_probs", C.c_int64), ("entropy", C.c_void_p),
        ("top_tokens", C.c_void_p), ("top_log_probs", C.c_void_p),
        ("ld_top_tokens", C.c_int64), ("ld_top_log_probs", C.c_int64),
    ]


class Tensor(C.Structure):
    _fields_ = [
        ("rank", C.c_int64), ("dims", C.c_int64 * 8), ("dtype", C.c_int32),
        ("data", C.c_void_p), ("pitch", C.c_int64),
        ("granularity", C.c_int32), ("scale", C.c_float), ("zero_point", C.c_int32),
        ("scale_data", C.c_void_p), ("zero_point_data", C.c_void_p), ("num_scales", C.c_int64),
        ("layout", C.c_int32),
    ]


class Epilogue(C.Structure):
    _fields_ = [
        ("type", C.c_int32), ("alpha", C.c_float), ("beta", C.c_float),
        ("min_clip", C.c_float), ("max_clip", C.c_float),
        ("quant", C.c_int32), ("quant_scales", C.c_void_p), ("quant_zero_points", C.c_void_p),
        ("quant_param_count", C.c_int64),
    ]


class MatMulAttrs(C.Structure):
    _fields_ = [
        ("transpose_a", C.c_int32), ("transpose_b", C.c_int32),
        ("alpha", C.c_float), ("beta", C.c_float),
        ("residual_pre_activation", C.c_int32), ("output_dtype", C.c_int32),
        ("epilogue", Epilogue),
        ("requant_round_even", C.c_int32), ("float_epilogue", C.c_int32),
        ("act_quant_dtype", C.c_int32),
    ]


class QuantLinearAttrs(C.Structure):
    _fields_ = [("axis", C.c_int64), ("output_dtype", C.c_int32)]


class LinearAttrs(C.Structure):
    _fields_ = [
        ("epilogue", Epilogue),
        ("add_to", C.c_int32), ("residual_pre_activation", C.c_int32),
        ("output_dtype", C.c_int32), ("gated", C.c_int32),
        ("requant_round_even", C.c_int32), ("float_epilogue", C.c_int32),
        ("gate_activation", C.c_int32), ("gate_alpha", C.c_float), ("gate_beta", C.c_float),
        ("gate_limit", C.c_float),
        ("matmul_order", C.c_int32), ("alpha", C.c_float), ("beta", C.c_float),
    ]


class RmsNormAttrs(C.Structure):
    _fields_ = [("epsilon", C.c_float), ("output_dtype", C.c_int32)]


class RotaryAttrs(C.Structure):
    _fields_ = [("head_dim", C.c_int64), ("rotary_dim", C.c_int64), ("interleaved", C.c_int32)]


class CacheAttentionAttrs(C.Structure):
    _fields_ = [("scale", C.c_float), ("window", C.c_int64), ("sinks", C.c_int64)]


class PrefixAttentionAttrs(C.Structure):
    _fields_ = [("scale", C.c_float)]


class KvCachePagesAttrs(C.Structure):
    _fields_ = [("page_tokens", C.c_int64)]


class TokenLogProbsAttrs(C.Structure):
    _fields_ = [("top", C.c_int64)]


class FpOutArgs(C.Structure):
    _fields_ = [
        ("src", C.c_void_p), ("ld_src", C.c_int64), ("out", C.c_void_p), ("ld_out", C.c_int64),
        ("rows", C.c_int64), ("n", C.c_int64), ("out_f16", C.c_int32), ("bias", C.c_void_p),
        ("act", C.c_int32), ("act_alpha", C.c_float), ("act_beta", C.c_float),
        ("min_clip", C.c_float), ("max_clip", C.c_float),
        ("add_to", C.c_int32), ("residual_pre", C.c_int32), ("gated", C.c_int32),
        ("gate_act", C.c_int32), ("gate_alpha", C.c_float), ("gate_beta", C.c_float), ("gate_limit", C.c_float),
        ("matmul_order", C.c_int32), ("alpha", C.c_float), ("beta", C.c_float),
    ]


class GemmPlan(C.Structure):
    _fields_ = [("tile_m", C.c_int32), ("tile_n", C.c_int32), ("splits", C.c_int32), ("fused", C.c_int32),
                ("short_stage", C.c_int32), ("in_place", C.c_int32), ("workspace_bytes", C.c_size_t)]


class CacheAttentionPlan(C.Structure):
    _fields_ = [("tile_rows", C.c_int32), ("one_page", C.c_int32), ("splits", C.c_int32), ("split_tokens", C.c_int32),
                ("join", C.c_int32), ("workspace_bytes", C.c_size_t)]


class PrefixAttentionPlan(C.Structure):
    _fields_ = [("shared_rows", C.c_int32), ("shared_splits", C.c_int32), ("own_rows", C.c_int32),
                ("own_splits", C.c_int32), ("launches", C.c_int32), ("join", C.c_int32), ("workspace_bytes", C.c_size_t)]


PLAN_NO_PASS, PLAN_PASS, PLAN_GATED_PASS = range(3)


# Every symbol the two headers declare, with its ctypes signature.
SIGNATURES = {
    "nnops_hip_gemm_i8_workspace_size": (C.c_size_t, [C.POINTER(GemmI8Args)]),
    "nnops_hip_gemm_i8": (C.c_int, [C.POINTER(GemmI8Args), C.c_void_p, C.c_size_t, C.c_void_p]),
    "nnops_hip_gemm_i8_noalloc": (C.c_int, [C.POINTER(GemmI8Args), C.c_void_p]),
    "nnops_hip_gemm_q4_1_workspace_size": (C.c_size_t, [C.POINTER(GemmQ41Args)]),
    "nnops_hip_gemm_q4_1": (C.c_int, [C.POINTER(GemmQ41Args), C.c_void_p, C.c_size_t, C.c_void_p]),
    "nnops_hip_gemm_i8_plan": (C.c_int, [C.POINTER(GemmI8Args), C.c_size_t, C.POINTER(GemmPlan)]),
    "nnops_hip_gemm_fp_plan": (C.c_int, [C.POINTER(GemmFpArgs), C.c_size_t, C.POINTER(GemmPlan)]),
    "nnops_hip_gemm_q4_1_plan": (C.c_int, [C.POINTER(GemmQ41Args), C.c_int32, C.c_size_t, C.POINTER(GemmPlan)]),
    "nnops_hip_gemm_fp_workspace_size": (C.c_size_t, [C.POINTER(GemmFpArgs)]),
    "nnops_hip_gemm_fp": (C.c_int, [C.POINTER(GemmFpArgs), C.c_void_p, C.c_size_t, C.c_void_p]),
    "nnops_hip_fp_output_pass": (C.c_int, [C.POINTER(FpOutArgs), C.c_void_p]),
    "nnops_hip_gemm_q4_1_fused": (C.c_int, [C.POINTER(GemmQ41Args), C.POINTER(FpOutArgs), C.c_void_p]),
    "nnops_hip_build_info": (C.c_char_p, []),
    "nnops_hip_time_next_launch": (C.c_int, [C.c_void_p, C.c_void_p]),
    "nnops_hip_prepack_i8_bytes": (C.c_size_t, [C.c_int64, C.c_int64]),
    "nnops_hip_prepack_q4_1_bytes": (C.c_size_t, [C.c_int64, C.c_int64]),
    "nnops_hip_prepack_q4_1": (C.c_int, [C.c_void_p, C.c_int64, C.c_int64, C.c_int64, C.c_int32, C.c_void_p,
                                         C.c_void_p]),
    "nnops_hip_prepack_i8": (C.c_int, [C.c_void_p, C.c_int64, C.c_int64, C.c_int64, C.c_int32, C.c_void_p,
                                       C.c_void_p]),
    "nnops_hip_q4_1_quantize": (C.c_int, [C.c_void_p, C.c_int32, C.c_int64, C.c_int64, C.c_int64, C.c_void_p,
                                          C.c_int64, C.c_void_p]),
    "nnops_hip_q4_1_dequantize": (C.c_int, [C.c_void_p, C.c_int64, C.c_int64, C.c_int64, C.c_void_p, C.c_int32,
                                            C.c_int64, C.c_void_p]),
    "nnops_hip_quantize_linear": (C.c_int, [C.POINTER(QdqArgs), C.c_void_p]),
    "nnops_hip_dequantize_linear": (C.c_int, [C.POINTER(QdqArgs), C.c_void_p]),
    "nnops_hip_rms_norm": (C.c_int, [C.POINTER(RmsNormArgs), C.c_void_p]),
    "nnops_hip_rotary": (C.c_int, [C.POINTER(RotaryArgs), C.c_void_p]),
    "nnops_hip_rotary_table": (C.c_int, [C.POINTER(RotaryTableArgs), C.c_void_p]),
    "nnops_hip_kv_cache_write": (C.c_int, [C.POINTER(KvRowsArgs), C.c_void_p]),
    "nnops_hip_kv_cache_read": (C.c_int, [C.POINTER(KvRowsArgs), C.c_void_p]),
    "nnops_hip_cache_attention_workspace_size": (C.c_size_t, [C.POINTER(CacheAttentionArgs)]),
    "nnops_hip_cache_attention_plan": (C.c_int, [C.POINTER(CacheAttentionArgs), C.POINTER(CacheAttentionPlan)]),
    "nnops_hip_cache_attention": (C.c_int, [C.POINTER(CacheAttentionArgs), C.c_void_p, C.c_size_t, C.c_void_p]),
    "nnops_hip_prefix_attention_workspace_size": (C.c_size_t, [C.POINTER(PrefixAttentionArgs)]),
    "nnops_hip_prefix_attention": (C.c_int, [C.POINTER(PrefixAttentionArgs), C.c_void_p, C.c_size_t, C.c_void_p]),
    "nnops_hip_prefix_attention_plan": (C.c_int, [C.POINTER(PrefixAttentionArgs), C.POINTER(PrefixAttentionPlan)]),
    "nnops_hip_kv_cache_fork_workspace_size": (C.c_size_t, [C.POINTER(KvForkArgs)]),
    "nnops_hip_kv_cache_fork": (C.c_int, [C.POINTER(KvForkArgs), C.c_void_p, C.c_size_t, C.c_void_p]),
    "nnops_hip_kv_cache_compact_workspace_size": (C.c_size_t, [C.POINTER(KvCompactArgs)]),
    "nnops_hip_kv_cache_compact": (C.c_int, [C.POINTER(KvCompactArgs), C.c_void_p, C.c_size_t, C.c_void_p]),
    "nnops_hip_kv_cache_copy": (C.c_int, [C.POINTER(KvCopyArgs), C.c_void_p]),
    "nnops_hip_token_log_probs_workspace_size": (C.c_size_t, [C.POINTER(TokenLogProbsArgs)]),
    "nnops_hip_token_log_probs": (C.c_int, [C.POINTER(TokenLogProbsArgs), C.c_void_p, C.c_size_t, C.c_void_p]),
    "nnops_matmul_attrs_init": (None, [C.POINTER(MatMulAttrs)]),
    "nnops_linear_attrs_init": (None, [C.POINTER(LinearAttrs)]),
    "nnops_matmul_create": (C.c_void_p, [C.POINTER(MatMulAttrs), C.c_int32]),
    "nnops_linear_create": (C.c_void_p, [C.POINTER(LinearAttrs), C.c_int32]),
    "nnops_quant_linear_attrs_init": (None, [C.POINTER(QuantLinearAttrs)]),
    "nnops_quantize_linear_create": (C.c_void_p, [C.POINTER(QuantLinearAttrs), C.c_int32]),
    "nnops_dequantize_linear_create": (C.c_void_p, [C.POINTER(QuantLinearAttrs), C.c_int32]),
    "nnops_rms_norm_attrs_init": (None, [C.POINTER(RmsNormAttrs)]),
    "nnops_rms_norm_create": (C.c_void_p, [C.POINTER(RmsNormAttrs), C.c_int32]),
    "nnops_rotary_attrs_init": (None, [C.POINTER(RotaryAttrs)]),
    "nnops_rotary_create": (C.c_void_p, [C.POINTER(RotaryAttrs), C.c_int32]),
    "nnops_kv_cache_write_create": (C.c_void_p, [C.c_int32]),
    "nnops_kv_cache_read_create": (C.c_void_p, [C.c_int32, C.c_int32]),
    "nnops_cache_attention_attrs_init": (None, [C.POINTER(CacheAttentionAttrs)]),
    "nnops_cache_attention_create": (C.c_void_p, [C.POINTER(CacheAttentionAttrs), C.c_int32]),
    "nnops_prefix_attention_attrs_init": (None, [C.POINTER(PrefixAttentionAttrs)]),
    "nnops_prefix_attention_create": (C.c_void_p, [C.POINTER(PrefixAttentionAttrs), C.c_int32]),
    "nnops_kv_cache_pages_attrs_init": (None, [C.POINTER(KvCachePagesAttrs)]),
    "nnops_kv_cache_fork_create": (C.c_void_p, [C.POINTER(KvCachePagesAttrs), C.c_int32]),
    "nnops_kv_cache_compact_create": (C.c_void_p, [C.POINTER(KvCachePagesAttrs), C.c_int32]),
    "nnops_kv_cache_copy_create": (C.c_void_p, [C.c_int32]),
    "nnops_token_log_probs_attrs_init": (None, [C.POINTER(TokenLogProbsAttrs)]),
    "nnops_token_log_probs_create": (C.c_void_p, [C.POINTER(TokenLogProbsAttrs), C.c_int32]),
    "nnops_op_destroy": (None, [C.c_void_p]),
    "nnops_op_prepack_weights": (C.c_int, [C.c_void_p, C.POINTER(Tensor), C.c_int32, C.POINTER(Tensor), C.c_int32,
                                           C.c_void_p]),
    "nnops_op_output_desc": (C.c_int, [C.c_void_p, C.POINTER(Tensor), C.c_int32, C.POINTER(Tensor)]),
    "nnops_op_output_descs": (C.c_int, [C.c_void_p, C.POINTER(Tensor), C.c_int32, C.POINTER(Tensor), C.c_int32]),
    "nnops_op_validate": (C.c_int, [C.c_void_p, C.POINTER(Tensor), C.c_int32, C.POINTER(Tensor), C.c_int32]),
    "nnops_op_workspace_size": (C.c_size_t, [C.c_void_p, C.POINTER(Tensor), C.c_int32,
                                             C.POINTER(Tensor), C.c_int32]),
    "nnops_op_compute": (C.c_int, [C.c_void_p, C.POINTER(Tensor), C.c_int32, C.POINTER(Tensor),
                                   C.c_int32, C.c_void_p, C.c_void_p]),
}

_lib = None


def load(path: str = LIB_PATH):
    """Load the library (raises if it was not built: there is no fallback)."""
    global _lib
    if _lib is None:
        if not os.path.exists(path):
            raise RuntimeError(
                f"nnops_amd native library missing: {path}; build it with `python -m nnops_amd.build`")
        # One HIP runtime per process: torch ships its own libamdhip64 (same
        # soname as ROCm's). Loaded after torch, this library binds to that
        # copy; loaded first, it would bring in ROCm's and torch would then add
        # its own beside it, so device pointers from one runtime would be
        # unknown to the other. Import torch first when it is installed.
        try:
            import torch  # noqa: F401
        except ImportError:
            pass
        lib_ = C.CDLL(path)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib_, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib_
    return _lib


def lib():
    return load()


# include/nnops_amd_diag.h: measurement probes in their own library (bench only)
DIAG_SIGNATURES = {
    "nnops_hip_diag_mfma_i8": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_void_p]),
    "nnops_hip_diag_stream_read": (C.c_int, [C.c_void_p, C.c_int64, C.c_void_p, C.c_int, C.c_void_p]),
    "nnops_hip_diag_empty": (C.c_int, [C.c_void_p, C.c_void_p]),
}
_diag = None


def diag_lib():
    """The probe library (libnnops_amd_diag.so), loaded after the product one."""
    global _diag
    if _diag is None:
        load()
        if not os.path.exists(DIAG_PATH):
            raise RuntimeError(f"probe library missing: {DIAG_PATH}; build it with `python -m nnops_amd.build`")
        d = C.CDLL(DIAG_PATH)
        for name, (res, args) in DIAG_SIGNATURES.items():
            fn = getattr(d, name)
            fn.restype = res
            fn.argtypes = args
        _diag = d
    return _diag
