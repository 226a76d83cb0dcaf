/* nnops_amd.h -- C ABI of the MI355X (gfx950) quantized-matmul path.
 *
 * This is the drop-in boundary below nnops' operator front end. In nnops the
 * CPU and CUDA backends are bound to `MatMul` / `Linear` through one kernel
 * function pointer per op, `Status fn(attrs, TensorView& out, span<const
 * TensorView> in, const ComputeContext&, void* workspace)`
 * (src/ops/dispatch.hpp:42-43, 62-96); the CUDA side of the integer route
 * flattens the views into a POD parameter block and launches on
 * `ctx.cuda_stream` (src/backend/cuda/matmul/matmul.cu:34-98,
 * src/backend/cuda/matmul/matmul_i8_common.cuh). The entry points below are
 * that launch boundary for a `Backend::HIP`: plain device pointers, element
 * strides taken from `TensorView::row_stride_elems()`, scalars, a
 * caller-provided device workspace and an opaque `hipStream_t`.
 *
 * Contract (all entry points):
 *   - every pointer in an args block is a DEVICE pointer (the C++ front end
 *     stages host QuantParams tables into the workspace);
 *   - nothing is allocated and nothing synchronises the host: work is enqueued
 *     on `stream` and the call returns;
 *   - `workspace` must hold at least the matching *_workspace_size() bytes
 *     (NNOPS_NOT_INITIALIZED otherwise, but where an entry point says what
 *     it does with less) and must not be shared by calls that may run
 *     concurrently; its contents on entry are irrelevant;
 *   - a rejected call returns a non-zero status and enqueues nothing.
 */
#ifndef NNOPS_AMD_H
#define NNOPS_AMD_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes: nnops::Status values (include/nnops/core/status.hpp:19-33). */
enum {
    NNOPS_OK = 0,
    NNOPS_INVALID_ARGUMENT = 1,
    NNOPS_UNSUPPORTED = 2,
    NNOPS_NOT_INITIALIZED = 3,
    NNOPS_OUT_OF_MEMORY = 4,
    NNOPS_INTERNAL = 5,
};

/* Destination element types (nnops' s32/s8/u8 integer destinations,
 * MatMulAttributes::output_dtype, include/nnops/ops/matmul.hpp:53-60; f32/f16
 * for the Q4_1 route and the int8 route's dequantizing destinations). */
enum {
    NNOPS_OUT_S32 = 0,
    NNOPS_OUT_S8 = 1,
    NNOPS_OUT_U8 = 2,
    NNOPS_OUT_F32 = 3,
    NNOPS_OUT_F16 = 4,
};

/* Activations the output pass applies: EpilogueActivateType's values
 * (include/nnops/core/epilogue.hpp:25-36). The requantizing integer pass of
 * nnops honours only Relu (matmul_tile_impl.h:411); the float epilogue of an
 * s8/u8 destination takes None/Relu/Gelu; the dequantizing f32/f16
 * destinations take all of them. */
enum {
    NNOPS_ACT_NONE = 0,
    NNOPS_ACT_RELU = 1,
    NNOPS_ACT_GELU = 2,
    NNOPS_ACT_SIGMOID = 3,
    NNOPS_ACT_TANH = 4,
    NNOPS_ACT_LEAKY_RELU = 5,
    NNOPS_ACT_SILU = 6,
    NNOPS_ACT_HARDSWISH = 7,
    NNOPS_ACT_ELU = 8,
    NNOPS_ACT_RELU6 = 9,
};

/* Integer GEMM  C[M,N] = epilogue(A[M,K] x B[K,N]).
 * Replaces the integer route of nnops' matmul_cuda / linear_cuda
 * (src/backend/cuda/matmul/matmul.cu:34-98, GemmI8Params) and of matmul_cpu's
 * I8Route (src/backend/cpu/matmul/matmul_i8.cpp:55-159).
 *
 * A is s8 or u8 (a_u8), [M,K] row-major with row stride lda, or [K,M] with
 * trans_a. B is s8, [K,N] (ldb) or [N,K] with trans_b (Linear's weight).
 * Quantization tables override their scalars when non-null: s_a/zp_a per row
 * of A (PerToken), s_b/zp_b per output column (PerChannel), s_out_rows/
 * zp_out_rows per output row (Epilogue Requantize table).
 *
 * Output pass, per element, nnops order (simd_epilogue.hpp:341-467):
 *   v = sum (a - zp_a)(b - zp_b) + bias[n];  Relu;  for s8/u8:
 *   q = sat(round(clamp(float(v) * ((s_a / s_out) * s_b), lo - zp, hi - zp)) + zp)
 * with round = half away from zero (round_even = 0, nnops) or half to even.
 *
 * float_ep (extension, no nnops counterpart): the s8/u8 destination is
 * produced through the f32 epilogue instead:
 *   f = float(v) * (s_a * s_b);  r = float(C_old - zp_out) * s_out (add_to);
 *   y = act(clamp(f [+ r if residual_pre])) [+ r otherwise];
 *   q = sat(round(clamp(y / s_out, lo - zp, hi - zp)) + zp)
 * which is how an s8 add_to residual and a GELU on an integer destination are
 * defined here (nnops rejects both: linear.cpp:226).
 *
 * f32/f16 destinations (nnops' dequantizing route, DqRoute, matmul_i8.cpp:
 * 161-211; tests/reference/matmul_dq_ref.cpp:178-190):
 *   f = float(v) * (s_a * s_b) [+ bias_fp[n]] [+ C_old if add_to];
 *   y = act(clamp(f, min_clip, max_clip)), stored as f32 or f16 (nearest even);
 * `bias` must be NULL there (the fp bias is `bias_fp`, in C's type). */
typedef struct NnopsGemmI8Args {
    const void* a;
    const int8_t* b;
    const int32_t* bias;        /* [N] int32, or NULL */
    void* c;
    int64_t m, n, k;
    int64_t lda, ldb, ldc;      /* row strides in elements */
    int32_t trans_a, trans_b, a_u8;
    const float* s_a; float s_a_scalar; const int32_t* zp_a; int32_t zp_a_scalar;
    const float* s_b; float s_b_scalar; const int32_t* zp_b; int32_t zp_b_scalar;
    const float* s_out_rows; const int32_t* zp_out_rows; float s_out; int32_t zp_out;
    int32_t out_kind;           /* NNOPS_OUT_S32 / S8 / U8 */
    int32_t act;                /* NNOPS_ACT_* (integer route: NONE or RELU) */
    int32_t round_even;
    int32_t float_ep;
    float min_clip, max_clip;   /* float epilogue and f32/f16 destinations */
    int32_t add_to, residual_pre; /* float epilogue and f32/f16 destinations */
    const void* bias_fp;        /* [N] f32 or f16 (C's type), f32/f16 destinations only */
    float act_alpha, act_beta;  /* LeakyRelu / Elu alpha, HardSwish beta */
    const int32_t* b_col_sums;  /* [N] sum over k of B[k,n] (a prepacked B carries them), or
                                   NULL: computed into the workspace when the A zero point
                                   or a u8 A needs them */
} NnopsGemmI8Args;

/* The workspace of a call. With less, a call of fewer than 64 rows, of K % 64 !=
 * 0 or of N % 4 != 0 splits K less or runs without its ring kernel, and others
 * split K less as long as the buffer holds the splits that their rows' tile
 * asks for; below that NNOPS_NOT_INITIALIZED. */
size_t nnops_hip_gemm_i8_workspace_size(const NnopsGemmI8Args* args);
int nnops_hip_gemm_i8(const NnopsGemmI8Args* args, void* workspace, size_t workspace_bytes,
                      void* stream);

/* No counterpart in nnops. nnops_hip_gemm_i8 for callers that cannot allocate
 * (code under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc): the same kernels and results, with the workspace taken from a
 * fixed device array of NNOPS_HIP_NOALLOC_SCRATCH_BYTES that the library
 * holds on each GPU it runs on until the process ends. A call that needs more
 * even with its K split no further than its row count's tile asks for (e.g. a
 * raw [K,N] B of 64 MiB that is staged transposed) returns NNOPS_OUT_OF_MEMORY
 * and enqueues nothing; any other takes as many K splits as the array holds. Calls on one GPU share the array: calls that may overlap on one
 * GPU (two streams, two threads) race. `stream` must belong to the current
 * device. Nothing is allocated, no host sync. */
#define NNOPS_HIP_NOALLOC_SCRATCH_BYTES (64u << 20)
int nnops_hip_gemm_i8_noalloc(const NnopsGemmI8Args* args, void* stream);

/* Prepacked s8 B for the HIP kernels (nnops' MatMul::prepackWeights,
 * src/ops/matmul.cpp:96-141, with a gfx950 layout in place of the CPU
 * panels). From B [K,N] (trans_b = 0) or [N,K] (trans_b = 1), row stride ldb,
 * it writes:
 *   rows   [N][kp] k-contiguous, kp = K rounded up to 128, zero padded;
 *   sums   int32 [N] = sum over k of B[k,n], at byte offset
 *          align_up(N * kp, 256).
 * A call then passes b = out, ldb = kp, trans_b = 1, b_col_sums = out + that
 * offset: every route reads the weight k-contiguous and 16-byte aligned (no
 * per-call transpose, no column-sum pass). `out` must be 256-byte aligned and
 * hold nnops_hip_prepack_i8_bytes(k, n) bytes. Stream-ordered, no allocation. */
size_t nnops_hip_prepack_i8_bytes(int64_t k, int64_t n);
int nnops_hip_prepack_i8(const int8_t* b, int64_t k, int64_t n, int64_t ldb, int32_t trans_b, void* out,
                         void* stream);

/* Prepacked Q4_1 B with blocks along N (nnops' MatMul::prepackWeights,
 * src/ops/matmul.cpp:96-141; the CPU path packs no Q4_1 form,
 * matmul_helper.cpp:695-723, this is the gfx950 one). From B [K][ceil(N/32)]
 * blocks (trans_b = 0), row pitch ldb_bytes, it writes the same blocks as
 * two planes, structure of arrays, one block column (32 columns) after
 * another:
 *   nibbles  k-blocked: block column j is kg * 128 bytes (kg = ceil(K/8)),
 *            per group of 8 rows, per nibble dword d, the 8 rows' dwords:
 *            dword d of row k, block j at byte
 *            (j * kg + k / 8) * 128 + 32 d + 4 (k % 8) (rows past K zero);
 *   d|m      block column j is kdm u32 (kdm = K rounded up to 64), row k's
 *            (f16 d low, f16 m high) at j * kdm + k (rows past K zero), the
 *            plane at byte offset align_up(nbn * kg * 128, 256);
 * nbn = ceil(N / 32). A call then passes b = out, ldb_bytes = kg * 128,
 * b_soa = 1, b_dm = out + that offset, ldb_dm = kdm: a block column's bytes
 * are two contiguous runs over the whole of K, so the GEMV streams each as
 * whole lines with no K split, and the GEMM's lane loads are contiguous 4-
 * and 16-byte runs instead of 20-byte strides. Blocks along K (trans_b = 1)
 * already stream as whole rows and have no packed form (NNOPS_UNSUPPORTED). `out` must be 256-byte aligned and hold
 * nnops_hip_prepack_q4_1_bytes(k, n) bytes. Stream-ordered, no allocation. */
size_t nnops_hip_prepack_q4_1_bytes(int64_t k, int64_t n);
int nnops_hip_prepack_q4_1(const uint8_t* b, int64_t k, int64_t n, int64_t ldb_bytes, int32_t trans_b, void* out,
                           void* stream);

/* Q4_1 codec over rows x cols values (each row its own run of blocks; a
 * partial last block takes d and m from the values that exist and leaves the
 * missing nibbles zero).
 * nnops_hip_q4_1_quantize replaces quantize_q4 (include/nnops/detail/q4_1.hpp:
 *   92-149, llama.cpp's quantize_row_q4_1_ref): src f32 (src_f16 = 0) or f16,
 *   row stride ld_src elements -> dst rows of ceil(cols / 32) 20-byte blocks,
 *   ld_dst_bytes apart (a multiple of 4, 4-byte-aligned dst). Byte-identical to
 *   the reference: d = (max - min) / 15, m = min (f16, nearest even),
 *   q = min(trunc((x - min) * (1 / d) + 0.5), 15).
 * nnops_hip_q4_1_dequantize replaces pack_q4 (q4_1.hpp:155-183): blocks ->
 *   f32 / f16 (dst_f16) rows, ld_dst elements apart; y = d * q + m in f32, f16
 *   rounded to nearest even.
 * Stream-ordered, no allocation, no workspace. */
int nnops_hip_q4_1_quantize(const void* src, int32_t src_f16, int64_t rows, int64_t cols, int64_t ld_src,
                            void* dst, int64_t ld_dst_bytes, void* stream);
int nnops_hip_q4_1_dequantize(const void* src, int64_t ld_src_bytes, int64_t rows, int64_t cols, void* dst,
                              int32_t dst_f16, int64_t ld_dst, void* stream);

/* Q4_1-weight GEMM  C[M,N] = A[M,K] x dequant(B).
 * Replaces nnops' fp x q4_1 route: matmul_qblock_fused (small M,
 * src/backend/cpu/matmul/matmul_qblock_fused.cpp:174-197) and FpRoute with
 * the Q4_1 RHS pack (matmul_helper.cpp:408-497). B is a stream of llama.cpp
 * Q4_1 blocks (20 bytes: f16 d, f16 m, 16 nibble bytes, value = d*q + m;
 * include/nnops/detail/q4_1.hpp:5-18):
 *   trans_b = 1: [N] rows of ceil(K/32) blocks along K (Linear / GGUF form),
 *   trans_b = 0: [K] rows of ceil(N/32) blocks along N,
 * consecutive rows ldb_bytes apart. A is f16 or f32 (a_f16), C is f32 or f16
 * (out_kind NNOPS_OUT_F32 / NNOPS_OUT_F16). Accumulation is f32. */
typedef struct NnopsGemmQ41Args {
    const void* a;
    const uint8_t* b;
    void* c;
    int64_t m, n, k;
    int64_t lda, ldc;           /* elements */
    int64_t ldb_bytes;
    int32_t trans_b, a_f16;
    int32_t out_kind;           /* NNOPS_OUT_F32 / NNOPS_OUT_F16 */
    /* b_soa = 1: B is the prepacked blocks-along-N form (trans_b = 0) of
     * nnops_hip_prepack_q4_1: b = the k-blocked nibble plane (ldb_bytes =
     * its block-column pitch, exactly ceil(K/8) * 128), b_dm = the d|m plane
     * (ldb_dm = its block-column pitch in u32, exactly K rounded up to 64). */
    int32_t b_soa;
    const uint32_t* b_dm;
    int64_t ldb_dm;
} NnopsGemmQ41Args;

/* The workspace of a call. Where it is room for K splits only (f16 A, blocks
 * along K), a call given less runs unsplit. */
size_t nnops_hip_gemm_q4_1_workspace_size(const NnopsGemmQ41Args* args);
int nnops_hip_gemm_q4_1(const NnopsGemmQ41Args* args, void* workspace, size_t workspace_bytes,
                        void* stream);

/* Dense fp product of nnops' float MatMul / Linear routes: C = alpha (A B)
 * for f32 x f32 or f16 x f16 (in_f16), accumulated in f32 and rounded once
 * to C's type (f32, or f16 with out_f16). Replaces the product of nnops'
 * matmul_small_fp / FpRoute<T> over dense operands
 * (src/backend/cpu/matmul/matmul_small.cpp:325-360, matmul.cpp:57-198),
 * whose f16 form keeps its accumulator in C between 128-deep k blocks; the
 * bias, beta, residual and epilogue are the output pass below.
 * A [M][lda], B [N][ldb] (trans_b) or [K][ldb], C [M][ldc]; pitches in
 * elements. The workspace holds K-split partials (small M, [K][N] B), a
 * transposed [K][N] f16 B and the ring GEMM's split partials (f16):
 * nnops_hip_gemm_fp_workspace_size bytes, 16-byte aligned. With less, f16 calls
 * do as the int8 ones above (fewer than 64 rows, K % 32 != 0 or N % 4 != 0: none
 * is needed). */
typedef struct NnopsGemmFpArgs {
    const void* a;
    const void* b;
    void* c;
    int64_t m, n, k;
    int64_t lda, ldb, ldc;      /* elements */
    int32_t trans_b;
    int32_t in_f16;             /* A and B f16 (else f32) */
    int32_t out_f16;            /* C f16 (else f32) */
    float alpha;
} NnopsGemmFpArgs;

size_t nnops_hip_gemm_fp_workspace_size(const NnopsGemmFpArgs* args);
int nnops_hip_gemm_fp(const NnopsGemmFpArgs* args, void* workspace, size_t workspace_bytes, void* stream);

/* Output pass of the fp x q4_1 routes over the GEMM's f32 results:
 * bias, the residual (add_to) and the epilogue (clip, activation), and the
 * gated combine of Linear's gated form. Replaces the fp epilogue of nnops'
 * FpRoute / matmul_qblock_fused output (apply_epilogue,
 * src/backend/cpu/simd_kernel/simd_epilogue.hpp:56-90; Linear's residual
 * order, src/backend/cpu/matmul/linear.cpp:276-301) and linear_gated_impl +
 * gated_combine_act (src/backend/cpu/matmul/linear.cpp:84-170, the combine
 * of src/backend/cpu/common/gate_combine.hpp:47-85).
 *   not gated:  f = src[r][c] + bias[c] (+ old if residual_pre);
 *               f = act(clip(f)); out = f (+ old, after the output type's
 *               rounding of f, if add_to and not residual_pre)
 *   matmul_order (MatMul's C = act(clip(alpha P + bias + beta C_old)),
 *               include/nnops/ops/matmul.hpp:5-11, with the accumulator
 *               init of matmul_qblock_fused.cpp:106-142): b = residual_pre
 *               ? 1 : beta; init = T(b old + bias) with a bias, else
 *               T(b old) (old itself when b = 1, 0 when b = 0), T the
 *               output type; out = act(clip(alpha src + init)). add_to is
 *               not read in this order.
 *   gated:      src holds 2n columns, gate [0, n) and value [n, 2n):
 *               g = T(src[r][c] + bias[c]), v = T(src[r][n + c] + bias[n + c])
 *               (T the output type: the reference's GEMM tile is of X's
 *               type), both clamped to +-gate_limit when finite;
 *               y = act(clip(gate_act(g) * (v + gate_beta))), out = y (+ old
 *               if add_to, after y's rounding to the output type); gate_act:
 *               Silu g / (1 + exp(-gate_alpha g)), Gelu
 *               (tanh form), Relu, Sigmoid, Tanh, None.
 * bias is in the output's type (f32 or f16), or NULL. Stream-ordered, no
 * allocation. */
typedef struct NnopsFpOutArgs {
    const float* src;           /* [rows][ld_src] f32 */
    int64_t ld_src;             /* elements */
    void* out;                  /* [rows][ld_out] f32 or f16 (out_f16) */
    int64_t ld_out;             /* elements */
    int64_t rows, n;            /* output columns n (gated: src has 2n) */
    int32_t out_f16;
    const void* bias;           /* [n], gated [2n], or NULL */
    int32_t act;                /* NNOPS_ACT_* */
    float act_alpha, act_beta, min_clip, max_clip;
    int32_t add_to, residual_pre;
    int32_t gated;
    int32_t gate_act;           /* NNOPS_ACT_NONE/RELU/GELU/SIGMOID/TANH/SILU */
    float gate_alpha, gate_beta, gate_limit;
    int32_t matmul_order;       /* 0: the orders above; 1: MatMul's (alpha, beta) */
    float alpha, beta;          /* read only when matmul_order */
} NnopsFpOutArgs;

int nnops_hip_fp_output_pass(const NnopsFpOutArgs* args, void* stream);

/* The Q4_1 GEMM with its output pass fused into the write-back: the product
 * of `g` (its c, ldc and out_kind unused) goes through `pass` (src and
 * ld_src unused; rows = g->m, n = g->n, or g->n / 2 for the gated form, whose
 * weight holds the gate rows and then the value rows) straight to pass->out,
 * with the same operations and rounding as nnops_hip_gemm_q4_1 into f32
 * followed by nnops_hip_fp_output_pass (nnops' Linear write-back,
 * src/backend/cpu/matmul/linear.cpp:74-170,233-282). Taken by the gated
 * form on the blocks-along-K ring route (trans_b, f16 A, K % 32 == 0,
 * 16-byte A rows, M past the GEMV and skinny shapes), where it saves the
 * f32 staging of both halves; NNOPS_UNSUPPORTED otherwise (the plain pass
 * included: in the write-back it costs more than its staging), with nothing
 * launched, and the caller runs the two-step form. No workspace. */
int nnops_hip_gemm_q4_1_fused(const NnopsGemmQ41Args* g, const NnopsFpOutArgs* pass, void* stream);

/* QuantizeLinear / DequantizeLinear over a rows x cols view (row strides in
 * elements), and the activation quantization of the fp-activation int8 MatMul.
 * Replaces nnops' quantize_linear_impl / dequantize_linear_impl
 * (src/backend/cpu/quant_linear.cpp:77-331) and quantize_activation in
 * matmul_dq (src/backend/cpu/matmul/matmul_i8.cpp:400-446).
 *
 * Parameter of flat element i = r * cols + c: entry (i / inner) % dim of
 * `scale` (f32) / `zero_point` (s8, u8 or s32 per zp_kind); dim <= 1 uses
 * entry 0 (NULL tables: the scalars). PerTensor: dim = 1; PerToken:
 * inner = cols, dim = rows; PerChannel(axis): inner = prod(shape[axis+1:]),
 * dim = shape[axis] (include/nnops/ops/quant_linear.hpp resolve rules).
 *   quantize    x f32/f16 -> y s8/u8:  clamp(rint(fma(x, 1/s, zp))), ties even;
 *               NaN / |v| >= 2^31 -> qmin (the x86 integer indefinite);
 *   dequantize  x s8/u8 -> y f32/f16:  fma(q, s, -zp*s) on each segment's whole
 *               16-element blocks, (q - zp) * s on its last segment % 16
 *               elements, as nnops' vector body and scalar tail
 *               (src/backend/cpu/x86_64/quant.hpp:298-340); `segment` is the
 *               reference's row: numel, cols or inner for the three modes. */
typedef struct NnopsQdqArgs {
    const void* x;
    void* y;
    int64_t rows, cols;
    int64_t ld_x, ld_y;         /* elements */
    int32_t x_kind, y_kind;     /* NNOPS_OUT_F32 / F16 / S8 / U8 */
    int32_t zp_kind;            /* NNOPS_OUT_S8 / U8 / S32: zero_point's element type */
    const float* scale;
    const void* zero_point;
    float scale_scalar;
    int32_t zp_scalar;
    int64_t inner, dim;
    int64_t segment;            /* dequantize only */
} NnopsQdqArgs;

int nnops_hip_quantize_linear(const NnopsQdqArgs* args, void* stream);
int nnops_hip_dequantize_linear(const NnopsQdqArgs* args, void* stream);

/* Root-mean-square norm with the residual's addition, and its output as s8
 * codes with one scale per row: the step between two int8 products of a
 * decoder layer (no counterpart in nnops). Per row, in f32:
 *   h = x + residual;  sum = h in x's type;
 *   rstd = 1 / sqrt(mean(h^2) + epsilon);  u = h * weight;
 *   f16 / f32 (x's type):  y = u * rstd;
 *   s8:  a = max |u|,  q = rint(u * (127 / a)),  scale = a * rstd / 127,
 * so that q * scale is u * rstd within half a step (rstd cancels in q: the
 * codes do not depend on the order in which the squares are summed). A row
 * with a < 2^-119 has codes 0; a row with an infinity or a NaN in u has codes
 * 0 and the scale NaN. A row of zeros is 0 (codes, scale 0) whatever epsilon
 * is; f32 rows whose squares would leave f32's range are normed as multiples of
 * a power of two. The codes and scales are what nnops_hip_gemm_i8 takes
 * as A and s_a.
 * sum may be x's or residual's buffer, y (f16 / f32) x's or residual's where
 * that is not sum's, with the same row pitch; otherwise no output may overlap
 * another buffer.
 * Stream-ordered, no allocation, no workspace. */
typedef struct NnopsRmsNormArgs {
    const void* x;              /* [rows][ld_x] f16 (in_f16) or f32 */
    const void* weight;         /* [cols], x's type */
    const void* residual;       /* [rows][ld_residual], x's type, or NULL */
    void* y;                    /* [rows][ld_y] */
    float* scale;               /* [rows], s8 only */
    void* sum;                  /* [rows][ld_sum], x's type: with a residual only */
    int64_t rows, cols;
    int64_t ld_x, ld_residual, ld_y, ld_sum; /* elements */
    int32_t in_f16;
    int32_t out_kind;           /* NNOPS_OUT_S8, or x's type */
    float epsilon;              /* >= 0 */
} NnopsRmsNormArgs;

int nnops_hip_rms_norm(const NnopsRmsNormArgs* args, void* stream);

/* Rotary positions (no counterpart in nnops). Each row of x holds `heads`
 * heads of head_dim values; the first rotary_dim values of each head are
 * rotated in pairs by the row's position, the others are copied:
 *   (y_a, y_b) = (x_a c - x_b s, x_b c + x_a s)
 * with (a, b) = (i, i + rotary_dim / 2), or (2 i, 2 i + 1) when interleaved,
 * and c, s = table[position][i], table[position][rotary_dim / 2 + i], each
 * product and sum rounded in f32, y to x's type. A position outside [0,
 * max_pos) gives NaN in the rotated values. y may be x (in place); otherwise
 * they may not overlap. */
typedef struct NnopsRotaryArgs {
    const void* x;              /* [tokens][ld_x] f16 (in_f16) or f32 */
    void* y;                    /* [tokens][ld_y], x's type */
    const int32_t* positions;   /* [tokens] */
    const float* table;         /* [max_pos][ld_table]: cosines, then sines */
    int64_t tokens, heads, head_dim, rotary_dim, max_pos;
    int64_t ld_x, ld_y, ld_table; /* elements */
    int32_t in_f16, interleaved;
} NnopsRotaryArgs;

int nnops_hip_rotary(const NnopsRotaryArgs* args, void* stream);

/* Fills a rotary table: row p, column i: cos(p f_i) * attention_factor, column
 * rotary_dim / 2 + i the sine, with f_i = base^(-2 i / rotary_dim), angles in
 * f64. Scaled for long contexts: with factor != 1 a frequency becomes
 *   g f + (1 - g) f / factor,
 * g = 0 everywhere when original_context is 0 (every position divided by
 * factor); otherwise g = clamp((t - low_turns) / (high_turns - low_turns), 0,
 * 1) of the turns t = original_context f / (2 pi) that the pair made over the
 * context that the model was trained on: fast pairs keep their frequency, slow
 * ones are stretched. */
typedef struct NnopsRotaryTableArgs {
    float* table;
    int64_t max_pos, rotary_dim, ld_table; /* ld_table: elements */
    double base, factor, original_context, low_turns, high_turns, attention_factor;
} NnopsRotaryTableArgs;

int nnops_hip_rotary_table(const NnopsRotaryTableArgs* args, void* stream);

/* A key / value cache held in 8 bits, in pages (no counterpart in nnops).
 * A page holds page_tokens consecutive tokens of one sequence, for every KV
 * head head_dim codes of the key and of the value per token, with one scale
 * per page and head on each side (value = code * scale):
 *   k        [pages][heads][page_tokens][head_dim]
 *   v        [pages][heads][head_dim][page_tokens]   (a channel's tokens side
 *            by side: what the product with the probabilities reads)
 *   k_scale, v_scale   [pages][heads], finite and >= 0
 * Token p of sequence b lies in slot p % page_tokens of page
 * page_table[b][p / page_tokens].
 * A call's rows are the LAST tokens of each sequence: sequence b has rows
 * row_starts[b] .. row_starts[b + 1] - 1 (row_starts NULL: rows / sequences
 * each, which has to be whole), its last row stands for token lengths[b] - 1.
 * page_tokens: 16, 32, 64, 128 or 256; head_dim: a multiple of 16 up to 256;
 * k and v 16-byte aligned, dense.
 * The tables are device memory that the host does not see. What they should
 * not hold does not fault: lengths are taken into [0, table_pages *
 * page_tokens] and row_starts into [0, rows]; a row that would stand for a
 * token before the first is not written, reads as 0 and attends to nothing; a
 * page number outside [0, pages) is not written and reads as NaN. */
typedef struct NnopsKvPages {
    int8_t* k;
    int8_t* v;
    float* k_scale;
    float* v_scale;
    int64_t pages, heads, page_tokens, head_dim;
    const int32_t* page_table;  /* [sequences][ld_table], table_pages columns */
    int64_t sequences, table_pages, ld_table; /* ld_table: elements */
    const int32_t* lengths;     /* [sequences] */
    const int32_t* row_starts;  /* [sequences + 1], or NULL */
} NnopsKvPages;

/* Key and value rows of a call, `heads` * head_dim values each. */
typedef struct NnopsKvRowsArgs {
    NnopsKvPages cache;
    void* k_rows;               /* [rows][ld_k] f16 (f16) or f32; write: only read */
    void* v_rows;               /* [rows][ld_v] */
    int64_t rows, ld_k, ld_v;   /* elements */
    int32_t f16;
} NnopsKvRowsArgs;

/* Write: the rows become codes in the sequences' pages. For each page and head
 * that gets rows, with a the largest magnitude among them:
 *   scale = max(old scale, a / 127, 2^-100)   (the old one only if the page
 *           holds tokens of the sequence before the call's first),
 *   new code = rint(x / scale) (as x * (1 / scale)),
 *   code of an older token = rint(code * (old scale / scale)) where it grew.
 * An infinity or a NaN among them makes the page's scale NaN (until the page
 * is begun anew), so that whatever reads the page shows it. No atomics, no
 * order: the same inputs give the same bits. Pages that get rows may not be
 * shared between sequences.
 * Read: the rows' codes times their scales, in f32, rounded to the rows' type.
 * Stream-ordered, no allocation, no workspace. */
int nnops_hip_kv_cache_write(const NnopsKvRowsArgs* args, void* stream);
int nnops_hip_kv_cache_read(const NnopsKvRowsArgs* args, void* stream);

/* Causal attention of query rows over that cache (no counterpart in nnops).
 * Row r of q holds q_heads heads of head_dim values, head m attends to KV head
 * m / (q_heads / heads). For a query at position p:
 *   out = sum_j softmax_j(scale * q . k_j) v_j over the tokens
 *   j <= p  and  (window == 0  or  p - j < window  or  j < sinks),
 * 0 where there are none. (The call's own rows are in the cache already.)
 * Scores, softmax statistics and sums are f32. f16: q and the codes enter the
 * matrix products exactly, the probabilities as the sum of two f16 (22 bits),
 * in calls whose rows share their tiles (nnops_hip_cache_attention_plan) as one
 * f16 (11 bits, of 14 bits more range); f32: both exactly, as three bf16 parts.
 * nnops_hip_cache_attention_workspace_size bytes of workspace (16-byte
 * aligned) hold the partial results of long sequences that are split over the
 * chip; the size goes by the sizes in args alone (no pointer is followed), and
 * is 0 for a call that is refused. */
typedef struct NnopsCacheAttentionArgs {
    NnopsKvPages cache;
    const void* q;              /* [rows][ld_q] f16 (f16) or f32 */
    void* out;                  /* [rows][ld_out], q's type */
    int64_t rows, q_heads, ld_q, ld_out; /* ld: elements */
    int32_t f16;
    float scale;                /* 0: 1 / sqrt(head_dim) */
    int64_t window, sinks;      /* >= 0 */
} NnopsCacheAttentionArgs;

size_t nnops_hip_cache_attention_workspace_size(const NnopsCacheAttentionArgs* args);
int nnops_hip_cache_attention(const NnopsCacheAttentionArgs* args, void* workspace, size_t workspace_bytes,
                              void* stream);

/* Attention for sequences that share their first tokens (no counterpart in
 * nnops): the same results as nnops_hip_cache_attention without a window, up to
 * the order of the sums, with the tokens that a group of sequences shares read
 * once for the group. (Probabilities of f16 rows have as many bits in the second
 * product as there, or more: two f16 where it gives a workgroup 16 rows, at least
 * one where more.) Group g is the sequences group_starts[g] ..
 * group_starts[g + 1] - 1, whose page tables hold the same pages for the first
 * shared[g] tokens, as far as these fill whole pages (which the caller sees to;
 * a sequence may be shorter, and may bring no rows). Read as shared: the whole
 * pages and whole tiles of 64 tokens that every row of the group sees. Sequences
 * in no group share nothing.
 * group_starts and shared are device memory that the host does not see; starts
 * are taken into [0, sequences], no group begins before the last one's end, and
 * what is shared beyond the first sequence's tokens is not.
 * Where the page table has room for so few tokens that reading them once saves
 * nothing, or a call is larger than the launches for shared tokens can be, every
 * sequence is looked at by itself. The workspace holds
 * the parts of all rows: nnops_hip_prefix_attention_workspace_size bytes, 16-byte
 * aligned, which need no initialization (0: none is needed). */
typedef struct NnopsPrefixAttentionArgs {
    NnopsKvPages cache;
    const void* q;              /* [rows][ld_q] f16 (f16) or f32 */
    void* out;                  /* [rows][ld_out], q's type */
    int64_t rows, q_heads, ld_q, ld_out; /* ld: elements */
    int32_t f16;
    float scale;                /* 0: 1 / sqrt(head_dim) */
    int64_t groups;
    const int32_t* group_starts; /* [groups + 1] */
    const int32_t* shared;      /* [groups] */
} NnopsPrefixAttentionArgs;

size_t nnops_hip_prefix_attention_workspace_size(const NnopsPrefixAttentionArgs* args);
int nnops_hip_prefix_attention(const NnopsPrefixAttentionArgs* args, void* workspace, size_t workspace_bytes,
                               void* stream);

/* Page tables of a batch's continuations (no counterpart in nnops). A sequence
 * of `lengths` tokens holds the pages in the first ceil(length / page_tokens)
 * cells of its row of the table; refs[p] counts who holds page p (sequences of
 * the table, and whoever else the caller counts), 0: free.
 * Fork: all `sequences` are given up, and `children` take their place. Child i
 * goes on from sequence parents[i] (outside [0, sequences): from nothing), L
 * tokens, and has room for new_tokens[i] more (fewer, where negative):
 *   new_lengths[i] = L' = L + new_tokens[i], taken into [0, new_table_pages *
 *   page_tokens]; kept tokens K = min(L, L')
 * Its first ceil(K / page_tokens) pages are the parent's. Where it grows past a
 * page that K tokens fill in part, it will write into that page: if the page's
 * only holders are children of this call that will, the first of them keeps it;
 * the others take a fresh page each, and copies[i] = {old page, fresh page} says
 * what nnops_hip_kv_cache_copy has to copy, for each layer's cache, before that
 * (rows without: {-1, -1}). Pages up to ceil(L' / page_tokens) are fresh. Fresh
 * pages are those whose count is 0 after the above, in ascending order, given out
 * child by child, cell by cell; where there is none left, the cell is -1 (nothing
 * is written there, and it reads as NaN). Cells past a child's pages are -1.
 * new_refs: the counts after the call; may be refs. counts: {pages that are free
 * now, cells that got none}. No other two arrays may overlap (from their first to their
 * last element: tables may not lie between each other's rows either).
 * The contents of the arrays are not seen by the host; a page number outside
 * [0, pages) is no page, lengths are taken into what the table has room for.
 * page_tokens: a power of two from 16 to 256. children, sequences <= 16384; cells
 * of the new table < 2^30. */
typedef struct NnopsKvForkArgs {
    const int32_t* page_table;  /* [sequences][ld_table], table_pages columns */
    int64_t sequences, table_pages, ld_table; /* ld: elements */
    const int32_t* lengths;     /* [sequences] */
    const int32_t* refs;        /* [pages] */
    int64_t pages, page_tokens;
    const int32_t* parents;     /* [children] */
    const int32_t* new_tokens;  /* [children] */
    int64_t children;
    int32_t* new_table;         /* [children][ld_new_table], new_table_pages columns */
    int64_t new_table_pages, ld_new_table;
    int32_t* new_lengths;       /* [children] */
    int32_t* new_refs;          /* [pages] */
    int32_t* copies;            /* [children][2] */
    int32_t* counts;            /* [2] */
} NnopsKvForkArgs;

size_t nnops_hip_kv_cache_fork_workspace_size(const NnopsKvForkArgs* args);
int nnops_hip_kv_cache_fork(const NnopsKvForkArgs* args, void* workspace, size_t workspace_bytes, void* stream);

/* Compact: the pages that are held (refs != 0), U of them, moved to the numbers
 * below U: the i-th that lies at U or above goes to the i-th free number below U,
 * both ascending; copies[i] = {old, new} for nnops_hip_kv_cache_copy, {-1, -1}
 * behind them. moved[p]: page p's new number, -1 for a free page (for tables that
 * others keep). new_table: the table with the new numbers, -1 past a sequence's
 * pages; new_refs: the counts, by new numbers. counts: {U, pages that move}.
 * new_table may be page_table (with the same ld) and new_refs refs; no other two
 * arrays may overlap (as of fork). */
typedef struct NnopsKvCompactArgs {
    const int32_t* page_table;  /* [sequences][ld_table], table_pages columns */
    int64_t sequences, table_pages, ld_table; /* ld: elements */
    const int32_t* lengths;     /* [sequences] */
    const int32_t* refs;        /* [pages] */
    int64_t pages, page_tokens;
    int32_t* new_table;         /* [sequences][ld_new_table] */
    int64_t ld_new_table;
    int32_t* new_refs;          /* [pages] */
    int32_t* copies;            /* [pages / 2][2] */
    int32_t* moved;             /* [pages] */
    int32_t* counts;            /* [2] */
} NnopsKvCompactArgs;

size_t nnops_hip_kv_cache_compact_workspace_size(const NnopsKvCompactArgs* args);
int nnops_hip_kv_cache_compact(const NnopsKvCompactArgs* args, void* workspace, size_t workspace_bytes,
                               void* stream);

/* Copy: pages of a cache (codes and scales, all heads) copied to others of it,
 * copies[i] = {from, to}; a row with a number outside [0, pages) is skipped. No
 * page may be copied to twice, or both from and to. Sizes as of NnopsKvPages. */
typedef struct NnopsKvCopyArgs {
    int8_t* k;
    int8_t* v;
    float* k_scale;
    float* v_scale;
    int64_t pages, heads, page_tokens, head_dim;
    const int32_t* copies;      /* [count][2] */
    int64_t count;
} NnopsKvCopyArgs;

int nnops_hip_kv_cache_copy(const NnopsKvCopyArgs* args, void* stream);

/* Log probabilities of given tokens, the entropy of the distribution and its
 * most probable tokens (no counterpart in nnops). Of row r of the logits x:
 *   log p_j = x_j - m - log s,  m = max x,  s = sum_j exp(x_j - m)
 *   log_probs[r][i] = log p of tokens[r][i]; 0 where that is negative (no token),
 *                     NaN where it is vocab or more
 *   entropy[r] = - sum_j p_j log p_j
 *   top_tokens[r], top_log_probs[r]: the `top` largest, in descending order, of
 *                     equal logits the lower token first
 * A logit of -inf has probability 0. A row of nothing else: every log probability
 * -inf, the entropy 0. A row that holds a NaN or +inf: NaN, top_tokens -1.
 * Sums are f32. vocab: up to 2^21. top: 0 to 32, at most vocab (0: top_tokens and
 * top_log_probs are not looked at). rows: up to 2^22, and parts of 32768 logits fewer
 * than 2^23. Rows are split over the chip where there are few of them: their parts
 * are in the workspace, nnops_hip_token_log_probs_workspace_size bytes, 16-byte
 * aligned, which need no initialization. */
typedef struct NnopsTokenLogProbsArgs {
    const void* logits;         /* [rows][ld_logits] f16 (f16) or f32, vocab columns */
    int64_t rows, vocab, ld_logits; /* ld: elements */
    int32_t f16, top;
    const int32_t* tokens;      /* [rows][ld_tokens], per_row columns */
    int64_t per_row, ld_tokens;
    float* log_probs;           /* [rows][ld_log_probs] */
    int64_t ld_log_probs;
    float* entropy;             /* [rows] */
    int32_t* top_tokens;        /* [rows][ld_top_tokens] */
    float* top_log_probs;       /* [rows][ld_top_log_probs] */
    int64_t ld_top_tokens, ld_top_log_probs;
} NnopsTokenLogProbsArgs;

size_t nnops_hip_token_log_probs_workspace_size(const NnopsTokenLogProbsArgs* args);
int nnops_hip_token_log_probs(const NnopsTokenLogProbsArgs* args, void* workspace, size_t workspace_bytes,
                              void* stream);

/* What the kernel selection of a call comes to (no counterpart in nnops; for
 * tests and for callers that tune shapes). Host code: the arguments' pointers
 * are looked at for their alignment only, and nothing is launched. */
typedef struct NnopsGemmPlan {
    int32_t tile_m, tile_n;     /* output tile of the LDS-ring GEMM; 0: another kernel takes the call */
    int32_t splits;             /* K splits (0: the other kernel's own) */
    int32_t fused;              /* the GEMM writes the destination itself (else partials and a pass) */
    int32_t short_stage;        /* K ends in a stage shorter than the ring's */
    int32_t in_place;           /* int8: a [K,N] B read where it lies */
    size_t workspace_bytes;     /* what it uses of the workspace */
} NnopsGemmPlan;

/* Q4_1's pass: the product alone, or a product whose output pass follows (Linear:
 * plain or gated). */
#define NNOPS_PLAN_NO_PASS 0
#define NNOPS_PLAN_PASS 1
#define NNOPS_PLAN_GATED_PASS 2
int nnops_hip_gemm_i8_plan(const NnopsGemmI8Args* args, size_t workspace_bytes, NnopsGemmPlan* plan);
int nnops_hip_gemm_fp_plan(const NnopsGemmFpArgs* args, size_t workspace_bytes, NnopsGemmPlan* plan);
int nnops_hip_gemm_q4_1_plan(const NnopsGemmQ41Args* args, int32_t pass, size_t workspace_bytes,
                             NnopsGemmPlan* plan);

typedef struct NnopsCacheAttentionPlan {
    int32_t tile_rows;          /* rows (tokens x heads of a group) of a workgroup: 128 or 256 that share their
                                   tiles of tokens, 16 otherwise */
    int32_t one_page;           /* of those: a tile of 64 tokens lies in one page */
    int32_t splits;             /* of the longest sequence that the page table has room for */
    int32_t split_tokens;       /* tokens of a split where it fills the table (fewer otherwise) */
    int32_t join;               /* of the splits: 0 none, 1 four channels a lane, 2 a workgroup a row */
    size_t workspace_bytes;
} NnopsCacheAttentionPlan;

typedef struct NnopsPrefixAttentionPlan {
    int32_t shared_rows;        /* rows of a workgroup over the shared tokens: 16, 128 or 256; 0: the table has so
                                   little room that every sequence is looked at by itself */
    int32_t shared_splits;      /* of these tokens, at most */
    int32_t own_rows;           /* and over each sequence's own tokens */
    int32_t own_splits;
    int32_t launches;           /* of kernels */
    int32_t join;               /* parts joined: 0 where own tokens are looked at, 1 by a kernel of their own */
    size_t workspace_bytes;
} NnopsPrefixAttentionPlan;

int nnops_hip_prefix_attention_plan(const NnopsPrefixAttentionArgs* args, NnopsPrefixAttentionPlan* plan);

/* OK, or what the call itself would say of the sizes. */
int nnops_hip_cache_attention_plan(const NnopsCacheAttentionArgs* args, NnopsCacheAttentionPlan* plan);

/* Library version and build target, for the caller's diagnostics. */
const char* nnops_hip_build_info(void);

/* Kernel timing for benchmarks (no counterpart in nnops; for callers that
 * measure the library, such as bench.py). Arms the calling thread's next
 * kernel launch by this library: that one launch carries `start` and `stop`
 * (hipEvent_t, created with timing enabled) on its own dispatch packet, so
 * hipEventElapsedTime(start, stop) is the kernel's execution alone, without
 * the dispatch gap an event pair recorded around the call would include.
 * One-shot: the next launch disarms it. A call that launches several kernels
 * times its first. Returns NNOPS_OK; NNOPS_INVALID_ARGUMENT if exactly one of
 * the two events is null; (null, null) disarms. */
int nnops_hip_time_next_launch(void* start_event, void* stop_event);


#ifdef __cplusplus
}
#endif

#endif /* NNOPS_AMD_H */
