// Root-mean-square norm with the residual's addition, its output in the input's
// type or as s8 codes with one scale per row. Per row, in f32:
//   h = x + residual;  rstd = 1 / sqrt(mean(h^2) + eps);  u = h w;
//   y = u rstd,  or  a = max |u|, q = rint(u (127 / a)), scale = a rstd / 127.
// The code needs no rstd: u rstd / (a rstd / 127) = 127 u / a, so codes depend
// on a maximum only, which no order of evaluation changes.
//
// Bound: HBM; x and the residual are read once, the sum and the codes written
// once. A row stays in its threads' registers between the two sums and the
// output: lane l of a row's RW waves holds the NC chunks of 8 elements l, l +
// 64 RW, ..; chunks are 16-byte loads (two for f32) from any alignment, the
// last chunk of a row whose width is no multiple of 8 goes element by element.
// Rows wider than 16 waves x 2 chunks (16384) are read twice.
// Measured: 4096 rows of 4096 with residual and codes, 117 MB: 27 us, 4.3 TB/s; 777
// rows of 5001, f16 to f16, 15.6 MB: 6.9 us a call (7.8 alone under the profiler),
// most of it one load and store latency behind a launch; 8 rows of 4096: 4.4 us;
// rows read twice, 512 of 20000, f16 to f16, 41 MB: 12.1 us a call, with residual
// and codes, 72 MB: 17.7.
// Without a branch per element of a ragged last chunk (clamped loads, selected
// after) the compiler flattened whole chunks too: 777 x 5001 took 9.2 us.
#include "common.hpp"

namespace nnops_amd {
namespace {

struct NormKern {
    const void* x;
    const void* w;
    const void* r;
    void* y;
    float* scale;
    void* sum;
    int64_t rows, cols, ld_x, ld_r, ld_y, ld_sum;
    float eps;            // no less than the smallest positive f32
    float eps_given;
};

// |v|'s bits order like |v|, infinities and NaNs above every finite value, so
// an integer maximum keeps them where fmaxf would drop a NaN.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8])
{
    T t[8];
    __builtin_memcpy(t, p, sizeof t);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        f[e] = (float)t[e];
    }
}

template <typename T>
__device__ __forceinline__ void load_upto(const T* p, int n, float (&f)[8])
{
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        f[e] = e < n ? (float)p[e] : 0.0f;
    }
}

template <typename T>
__device__ __forceinline__ void store_upto(T* p, int n, const float (&f)[8])
{
    T t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        t[e] = (T)f[e];
    }
    if (n >= 8) {
        __builtin_memcpy(p, t, sizeof t);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if (e < n) {
            p[e] = t[e];
        }
    }
}

__device__ __forceinline__ void store_codes(int8_t* p, int n, const float (&u)[8], float inv)
{
    uint32_t d[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        // |u inv| <= 127 (1 + 2^-22): the rounding ends at +-127
        const int q = (int)__builtin_rintf(__fmul_rn(u[e], inv));
        d[e / 4] |= ((uint32_t)q & 0xffu) << (8 * (e % 4));
    }
    if (n >= 8) {
        __builtin_memcpy(p, d, 8);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if (e < n) {
            p[e] = (int8_t)(d[e / 4] >> (8 * (e % 4)));
        }
    }
}

// Sum and maximum over a row's RW waves, the same value in each of its lanes.
template <int RW>
__device__ __forceinline__ void row_reduce(float& ss, uint32_t& a)
{
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        ss += __shfl_xor(ss, m);
        a = max(a, (uint32_t)__shfl_xor((int)a, m));
    }
    if constexpr (RW > 1) {
        __shared__ float s_ss[RW];
        __shared__ uint32_t s_a[RW];
        const int wave = threadIdx.x / 64;
        if (threadIdx.x % 64 == 0) {
            s_ss[wave] = ss;
            s_a[wave] = a;
        }
        __syncthreads();
        ss = s_ss[0];
        a = s_a[0];
#pragma unroll
        for (int i = 1; i < RW; ++i) {
            ss += s_ss[i];
            a = max(a, s_a[i]);
        }
    }
}

// The factor of u in the codes; 0 gives codes 0 (rows of next to nothing, and
// rows that hold an infinity or a NaN, whose scale then says so).
__device__ __forceinline__ float code_factor(uint32_t a)
{
    constexpr uint32_t kLeast = (127 - 119) << 23, kInf = 0x7f800000u;
    return a >= kLeast && a < kInf ? __fmul_rn(__fdiv_rn(1.0f, __uint_as_float(a)), 127.0f) : 0.0f;
}

__device__ __forceinline__ float row_scale(uint32_t a, float rstd)
{
    return a < 0x7f800000u ? __fmul_rn(__fmul_rn(__uint_as_float(a), rstd), 1.0f / 127.0f) : __uint_as_float(0x7fc00000u);
}

__device__ __forceinline__ float row_rstd(float ss, float cols, float eps)
{
    return __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, cols) + eps));
}

// f32 rows whose squares leave f32's range: past 2^127 their sum is infinite and
// the factor 0, below 2^-126 they lose their bits or are 0 (which shows where
// epsilon is next to nothing). Such a row is normed as h times a power of two,
// epsilon times its square: the same result. 1 where a row needs none, as every
// row of f16 does (its squares are 0 or 2^-48 to 2^34).
template <typename T>
constexpr bool kRescales = sizeof(T) == 4;

__device__ __forceinline__ float row_rescale(float ss, float cols, float eps)
{
    const float m = __fdiv_rn(ss, cols) + eps;
    return m < 0x1p-100f ? 0x1p90f : m < __builtin_inff() ? 1.0f : 0x1p-80f;   // (a NaN stays one)
}

__device__ __forceinline__ float scaled_eps(const NormKern& p, float f)
{
    return fmaxf(__fmul_rn(__fmul_rn(p.eps_given, f), f), 0x1p-149f);
}

// A row's chunks as they lie in memory.
template <typename T, int NC>
struct RowChunks {
    T v[NC][8];
};

template <typename T, int RW, int NC>
__device__ __forceinline__ void load_row(RowChunks<T, NC>& c, const T* row, int lane, int cols)
{
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int at = (lane + i * 64 * RW) * 8, n = cols - at;
        if (n >= 8) {
            __builtin_memcpy(c.v[i], row + at, sizeof c.v[i]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                c.v[i][e] = e < n ? row[at + e] : (T)0.0f;
            }
        }
    }
}

// Each unit of RW waves takes every gridDim-th row, the next one's chunks in
// flight while it sums and writes this one's; the weight stays in registers.
template <typename T, int RW, int NC, bool S8, bool RES>
__global__ __launch_bounds__(64 * (RW > 4 ? RW : 4)) void rms_norm_kernel(const NormKern p)
{
    constexpr int kRows = RW >= 4 ? 1 : 4 / RW;   // rows of a workgroup
    static_assert(RW == 1 || RW >= 4, "a row has one wave, or the workgroup");
    const int lane = kRows == 1 ? threadIdx.x : threadIdx.x % 64;
    const int64_t step = (int64_t)gridDim.x * kRows;
    int64_t row = kRows == 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * kRows + threadIdx.x / 64;
    if (row >= p.rows) {
        return;                                    // one wave per row: no barrier below
    }
    const int cols = (int)p.cols;
    const T* x = static_cast<const T*>(p.x);
    const T* r = static_cast<const T*>(p.r);
    RowChunks<T, NC> xs, rs, ws;
    load_row<T, RW, NC>(xs, x + row * p.ld_x, lane, cols);
    if constexpr (RES) {
        load_row<T, RW, NC>(rs, r + row * p.ld_r, lane, cols);
    }
    load_row<T, RW, NC>(ws, static_cast<const T*>(p.w), lane, cols);
    for (;;) {
        float h[NC][8];
        float ss = 0.0f;
        uint32_t a = 0;
        T* sum = RES ? static_cast<T*>(p.sum) + row * p.ld_sum : nullptr;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                h[c][e] = RES ? __fadd_rn((float)xs.v[c][e], (float)rs.v[c][e]) : (float)xs.v[c][e];
            }
        }
        const int64_t next = row + step;
        if (next < p.rows) {
            load_row<T, RW, NC>(xs, x + next * p.ld_x, lane, cols);
            if constexpr (RES) {
                load_row<T, RW, NC>(rs, r + next * p.ld_r, lane, cols);
            }
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if constexpr (RES) {
                const int at = (lane + c * 64 * RW) * 8;
                store_upto(sum + at, cols - at, h[c]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                ss = __builtin_fmaf(h[c][e], h[c][e], ss);
                const float u = __fmul_rn(h[c][e], (float)ws.v[c][e]);
                if constexpr (S8) {
                    a = max(a, magnitude(u));
                }
                h[c][e] = kRescales<T> ? h[c][e] : u;
            }
        }
        row_reduce<RW>(ss, a);
        float eps = p.eps;
        if constexpr (kRescales<T>) {
            const float f = row_rescale(ss, (float)cols, eps);
            if (f != 1.0f) {                       // (the same in the whole row)
                if constexpr (RW > 1) {
                    __syncthreads();               // row_reduce's words are read
                }
                ss = 0.0f;
                a = 0;
#pragma unroll
                for (int c = 0; c < NC; ++c) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        h[c][e] = __fmul_rn(h[c][e], f);
                        ss = __builtin_fmaf(h[c][e], h[c][e], ss);
                        a = max(a, magnitude(__fmul_rn(h[c][e], (float)ws.v[c][e])));
                    }
                }
                row_reduce<RW>(ss, a);
                eps = scaled_eps(p, f);
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    h[c][e] = __fmul_rn(h[c][e], (float)ws.v[c][e]);
                }
            }
        }
        const float rstd = row_rstd(ss, (float)cols, eps);
        if constexpr (S8) {
            const float inv = code_factor(a);
            int8_t* y = static_cast<int8_t*>(p.y) + row * p.ld_y;
            if (lane == 0) {
                p.scale[row] = row_scale(a, rstd);
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int at = (lane + c * 64 * RW) * 8;
                if (inv == 0.0f) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        h[c][e] = 0.0f;            // inf * 0 is no 0
                    }
                }
                store_codes(y + at, cols - at, h[c], inv);
            }
        } else {
            T* y = static_cast<T*>(p.y) + row * p.ld_y;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int at = (lane + c * 64 * RW) * 8;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    h[c][e] = __fmul_rn(h[c][e], rstd);
                }
                store_upto(y + at, cols - at, h[c]);
            }
        }
        if (next >= p.rows) {
            return;
        }
        row = next;
        if constexpr (RW > 1) {
            __syncthreads();                       // row_reduce's words are read
        }
    }
}

// Rows of any width: one pass for the sum and the maximum, one for the output.
// Nothing is written before the last, so that sum may lie over x or the residual.
template <typename T, bool S8, bool RES>
__global__ __launch_bounds__(1024) void rms_norm_wide(const NormKern p)
{
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.ld_x;
    const T* r = RES ? static_cast<const T*>(p.r) + row * p.ld_r : nullptr;
    const T* w = static_cast<const T*>(p.w);
    auto chunk = [&](int64_t at, int n, float (&h)[8], float (&u)[8]) {
        float f[8];
        if (n >= 8) {
            load8(x + at, h);
            load8(w + at, u);
            if constexpr (RES) {
                load8(r + at, f);
            }
        } else {
            load_upto(x + at, n, h);
            load_upto(w + at, n, u);
            if constexpr (RES) {
                load_upto(r + at, n, f);
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (RES) {
                h[e] = __fadd_rn(h[e], f[e]);
            }
            u[e] = __fmul_rn(h[e], u[e]);
        }
    };
    float ss = 0.0f;
    uint32_t a = 0;
    for (int64_t at = (int64_t)threadIdx.x * 8; at < p.cols; at += 8192) {
        float h[8], u[8];
        chunk(at, (int)min((int64_t)8, p.cols - at), h, u);
        float part = 0.0f;                         // a sum of sums: no long chain of one rounding each
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            part = __builtin_fmaf(h[e], h[e], part);
            a = max(a, magnitude(u[e]));
        }
        ss += part;
    }
    row_reduce<16>(ss, a);
    float eps = p.eps, factor = 1.0f;              // of h (row_rescale)
    if constexpr (kRescales<T>) {
        factor = row_rescale(ss, (float)p.cols, eps);
        if (factor != 1.0f) {                      // (the same in the whole workgroup)
            __syncthreads();                       // row_reduce's words are read
            ss = 0.0f;
            a = 0;
            for (int64_t at = (int64_t)threadIdx.x * 8; at < p.cols; at += 8192) {
                float part = 0.0f;
                for (int64_t i = at; i < min(at + 8, p.cols); ++i) {
                    const float h = __fmul_rn(RES ? __fadd_rn((float)x[i], (float)r[i]) : (float)x[i], factor);
                    part = __builtin_fmaf(h, h, part);
                    a = max(a, magnitude(__fmul_rn(h, (float)w[i])));
                }
                ss += part;
            }
            row_reduce<16>(ss, a);
            eps = scaled_eps(p, factor);
        }
    }
    const float rstd = row_rstd(ss, (float)p.cols, eps);
    const float inv = code_factor(a);
    if (S8 && threadIdx.x == 0) {
        p.scale[row] = row_scale(a, rstd);
    }
    for (int64_t at = (int64_t)threadIdx.x * 8; at < p.cols; at += 8192) {
        const int n = (int)min((int64_t)8, p.cols - at);
        float h[8], u[8];
        chunk(at, n, h, u);
        if constexpr (kRescales<T>) {
            if (factor != 1.0f) {                  // (past f32's range u may be infinite before)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    u[e] = e < n ? __fmul_rn(__fmul_rn(h[e], factor), (float)w[at + e]) : 0.0f;
                }
            }
        }
        if constexpr (RES) {
            store_upto(static_cast<T*>(p.sum) + row * p.ld_sum + at, n, h);
        }
        if constexpr (S8) {
            if (inv == 0.0f) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    u[e] = 0.0f;
                }
            }
            store_codes(static_cast<int8_t*>(p.y) + row * p.ld_y + at, n, u, inv);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                u[e] = __fmul_rn(u[e], rstd);
            }
            store_upto(static_cast<T*>(p.y) + row * p.ld_y + at, n, u);
        }
    }
}

// 4 workgroups of 256 threads per CU (4096 x 4096 and its dequantization, us: 35.7
// with 2, 31.6 with 4, 33.6 with 8, 35.2 with a workgroup per row).
template <typename T, int RW, int NC, bool S8, bool RES>
void launch_rows(const NormKern& k, hipStream_t s)
{
    constexpr int kRows = RW >= 4 ? 1 : 4 / RW, kThreads = 64 * (RW > 4 ? RW : 4);
    const int64_t all = (k.rows + kRows - 1) / kRows, most = 4 * 256 * 256 / kThreads;
    NNOPS_LAUNCH((rms_norm_kernel<T, RW, NC, S8, RES>), dim3((unsigned)(all < most ? all : most)), dim3(kThreads), 0, s, k);
}

template <typename T, bool S8, bool RES>
void launch_norm(const NormKern& k, hipStream_t s)
{
    const int64_t chunks = (k.cols + 7) / 8;
    if (chunks <= 64) {
        launch_rows<T, 1, 1, S8, RES>(k, s);
    } else if (chunks <= 128) {
        launch_rows<T, 1, 2, S8, RES>(k, s);
    } else if (chunks <= 256) {
        launch_rows<T, 4, 1, S8, RES>(k, s);
    } else if (chunks <= 512) {
        launch_rows<T, 4, 2, S8, RES>(k, s);
    } else if (chunks <= 768) {
        launch_rows<T, 4, 3, S8, RES>(k, s);
    } else if (chunks <= 1024) {
        launch_rows<T, 8, 2, S8, RES>(k, s);
    } else if (chunks <= 2048) {
        launch_rows<T, 16, 2, S8, RES>(k, s);
    } else {
        // a launch has fewer than 2^32 threads: 2^22 workgroups of these are too many
        constexpr int64_t kSlab = 1 << 20;
        for (int64_t r0 = 0; r0 < k.rows; r0 += kSlab) {
            NormKern part = k;
            part.rows = k.rows - r0 < kSlab ? k.rows - r0 : kSlab;
            part.x = static_cast<const T*>(k.x) + r0 * k.ld_x;
            part.y = S8 ? (void*)(static_cast<int8_t*>(k.y) + r0 * k.ld_y) : (void*)(static_cast<T*>(k.y) + r0 * k.ld_y);
            if constexpr (S8) {
                part.scale = k.scale + r0;
            }
            if constexpr (RES) {
                part.r = static_cast<const T*>(k.r) + r0 * k.ld_r;
                part.sum = static_cast<T*>(k.sum) + r0 * k.ld_sum;
            }
            NNOPS_LAUNCH((rms_norm_wide<T, S8, RES>), dim3((unsigned)part.rows), dim3(1024), 0, s, part);
        }
    }
}

}  // namespace
}  // namespace nnops_amd

using namespace nnops_amd;

extern "C" int nnops_hip_rms_norm(const NnopsRmsNormArgs* g, void* stream)
{
    const TimingDisarm disarm;
    if (g == nullptr || g->rows < 0 || g->cols < 0) {
        return NNOPS_INVALID_ARGUMENT;
    }
    if (g->rows == 0 || g->cols == 0) {
        return NNOPS_OK;
    }
    const bool s8 = g->out_kind == NNOPS_OUT_S8;
    if (!s8 && g->out_kind != (g->in_f16 ? NNOPS_OUT_F16 : NNOPS_OUT_F32)) {
        return NNOPS_UNSUPPORTED;
    }
    if (g->rows > INT32_MAX || g->cols > INT32_MAX) {
        return NNOPS_UNSUPPORTED;
    }
    const bool res = g->residual != nullptr;
    if (g->x == nullptr || g->weight == nullptr || g->y == nullptr || g->ld_x < g->cols || g->ld_y < g->cols ||
        (s8 != (g->scale != nullptr)) || (res != (g->sum != nullptr)) ||
        (res && (g->ld_residual < g->cols || g->ld_sum < g->cols)) || !(g->epsilon >= 0.0f)) {
        return NNOPS_INVALID_ARGUMENT;
    }
    // an output over an input: rows at the same places, or a row would be written
    // that another has not read yet
    const auto over = [&](const void* in, int64_t ld_in, const void* out, int64_t ld_out) {
        return out == in && g->rows > 1 && ld_out != ld_in;
    };
    if (over(g->x, g->ld_x, g->y, g->ld_y) ||
        (res && (over(g->residual, g->ld_residual, g->y, g->ld_y) || over(g->x, g->ld_x, g->sum, g->ld_sum) ||
                 over(g->residual, g->ld_residual, g->sum, g->ld_sum) || g->y == g->sum)) ||
        (s8 && (g->y == g->x || (res && g->y == g->residual)))) {
        return NNOPS_INVALID_ARGUMENT;
    }
    // (no epsilon: the least that keeps the factor of a row of zeros finite, so that
    // the row is zeros. Testing for it in the kernel took 3 % of 512 x 16384.)
    const float eps = g->epsilon > 0.0f ? g->epsilon : 0x1p-149f;
    const NormKern k{g->x,    g->weight, g->residual,    g->y,    g->scale,  g->sum,    g->rows,
                     g->cols, g->ld_x,   g->ld_residual, g->ld_y, g->ld_sum, eps,
                     g->epsilon};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (g->in_f16) {
        s8 ? (res ? launch_norm<_Float16, true, true>(k, s) : launch_norm<_Float16, true, false>(k, s))
           : (res ? launch_norm<_Float16, false, true>(k, s) : launch_norm<_Float16, false, false>(k, s));
    } else {
        s8 ? (res ? launch_norm<float, true, true>(k, s) : launch_norm<float, true, false>(k, s))
           : (res ? launch_norm<float, false, true>(k, s) : launch_norm<float, false, false>(k, s));
    }
    return hipGetLastError() == hipSuccess ? NNOPS_OK : NNOPS_INTERNAL;
}
