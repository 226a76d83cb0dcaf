// Rotary positions over the heads of each row, and the table of cosines and
// sines they take.
//   (y_a, y_b) = (x_a c - x_b s, x_b c + x_a s),  products and sums rounded in
//   f32 one by one, pairs (i, i + rot / 2) or (2 i, 2 i + 1)
// Bound: HBM (x in, y out); the table's row is shared by a token's heads and
// comes from the caches. A thread takes 2 V values of a head: the V of each
// half (16 bytes each), or 2 V adjacent ones, or 2 V of the copied tail; V is
// 8 (f16) or 4 (f32) where the halves and the tail hold whole ones, else 4, else
// 1. A pair is read before either of its values is written, by one thread, which
// is what lets y be x. Measured: 2049 tokens x 40 heads of 128, 64 of them rotated,
// f32, 84 MB: 16.7 us, 5.06 TB/s; 32 tokens, f16: 5.9 us a call, 3.0 alone.
#include "common.hpp"

namespace nnops_amd {
namespace {

struct RotaryKern {
    const void* x;
    void* y;
    const int32_t* positions;
    const float* table;
    int64_t ld_x, ld_y, ld_table, max_pos;
    uint32_t units, per_token, per_head, rot_units;   // units of this launch; of a token; of a head; rotated ones
    int head_dim, rot;
};

template <typename T, int V, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryKern p)
{
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= p.units) {
        return;
    }
    const uint32_t token = i / p.per_token, rest = i - token * p.per_token;
    const uint32_t head = rest / p.per_head, unit = rest - head * p.per_head;
    const T* x = static_cast<const T*>(p.x) + (int64_t)token * p.ld_x + (int64_t)head * p.head_dim;
    T* y = static_cast<T*>(p.y) + (int64_t)token * p.ld_y + (int64_t)head * p.head_dim;
    if (unit >= p.rot_units) {                     // the copied tail
        if (x == y) {
            return;
        }
        const int at = p.rot + (int)(unit - p.rot_units) * 2 * V;
        const int n = min(2 * V, p.head_dim - at);
        T t[V];
        __builtin_memcpy(t, x + at, sizeof t);
        __builtin_memcpy(y + at, t, sizeof t);
        if (n > V) {
            __builtin_memcpy(t, x + at + V, sizeof t);
            __builtin_memcpy(y + at + V, t, sizeof t);
        }
        return;
    }
    const int half = p.rot / 2, pair = (int)unit * V;
    const int64_t pos = p.positions[token];
    float c[V], s[V];
    if (pos >= 0 && pos < p.max_pos) {
        const float* row = p.table + pos * p.ld_table + pair;
        __builtin_memcpy(c, row, sizeof c);
        __builtin_memcpy(s, row + half, sizeof s);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            c[e] = s[e] = __uint_as_float(0x7fc00000u);
        }
    }
    T t[2 * V];
    const int at_a = INTER ? 2 * pair : pair, at_b = INTER ? 2 * pair + V : pair + half;
    __builtin_memcpy(t, x + at_a, sizeof(T) * V);
    __builtin_memcpy(t + V, x + at_b, sizeof(T) * V);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int ia = INTER ? 2 * e : e, ib = INTER ? 2 * e + 1 : V + e;
        const float a = (float)t[ia], b = (float)t[ib];
        t[ia] = (T)__fsub_rn(__fmul_rn(a, c[e]), __fmul_rn(b, s[e]));
        t[ib] = (T)__fadd_rn(__fmul_rn(b, c[e]), __fmul_rn(a, s[e]));
    }
    __builtin_memcpy(y + at_a, t, sizeof(T) * V);
    __builtin_memcpy(y + at_b, t + V, sizeof(T) * V);
}

struct TableKern {
    float* table;
    int64_t max_pos, ld;
    int half;
    double base, factor, original, low, high, scale;
};

// One thread per (position, pair). The frequency is the same for every
// position: recomputed rather than stored, since a table is filled once.
__global__ __launch_bounds__(256) void rotary_table_kernel(const TableKern p)
{
    constexpr double kTwoPi = 6.283185307179586476925286766559;
    const int i = blockIdx.y * 256 + threadIdx.x;
    if (i >= p.half) {
        return;
    }
    double f = exp2(-(double)i / (double)p.half * log2(p.base));
    if (p.factor != 1.0) {
        double keep = 0.0;
        if (p.original > 0.0) {
            keep = (p.original * f / kTwoPi - p.low) / (p.high - p.low);
            keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
        }
        f = keep * f + (1.0 - keep) * f / p.factor;
    }
    for (int64_t pos = blockIdx.x; pos < p.max_pos; pos += gridDim.x) {
        double s, c;
        sincos((double)pos * f, &s, &c);
        p.table[pos * p.ld + i] = (float)(c * p.scale);
        p.table[pos * p.ld + p.half + i] = (float)(s * p.scale);
    }
}

template <typename T, int V>
void launch_rotary(const RotaryKern& k, bool inter, hipStream_t s)
{
    const dim3 grid((k.units + 255) / 256);
    if (inter) {
        NNOPS_LAUNCH((rotary_kernel<T, V, true>), grid, dim3(256), 0, s, k);
    } else {
        NNOPS_LAUNCH((rotary_kernel<T, V, false>), grid, dim3(256), 0, s, k);
    }
}

}  // namespace
}  // namespace nnops_amd

using namespace nnops_amd;

extern "C" int nnops_hip_rotary(const NnopsRotaryArgs* g, void* stream)
{
    const TimingDisarm disarm;
    if (g == nullptr || g->tokens < 0 || g->heads < 0) {
        return NNOPS_INVALID_ARGUMENT;
    }
    if (g->head_dim <= 0 || g->rotary_dim <= 0 || g->rotary_dim % 2 != 0 || g->rotary_dim > g->head_dim ||
        g->max_pos <= 0) {
        return NNOPS_INVALID_ARGUMENT;
    }
    if (g->tokens == 0 || g->heads == 0) {
        return NNOPS_OK;
    }
    if (g->head_dim > (1 << 20) || g->heads > (1 << 20) || g->heads * g->head_dim > INT32_MAX ||
        g->tokens > INT32_MAX) {
        return NNOPS_UNSUPPORTED;
    }
    const int64_t width = g->heads * g->head_dim;
    if (g->x == nullptr || g->y == nullptr || g->positions == nullptr || g->table == nullptr || g->ld_x < width ||
        g->ld_y < width || g->ld_table < g->rotary_dim || (g->x == g->y && g->ld_x != g->ld_y)) {
        return NNOPS_INVALID_ARGUMENT;
    }
    const int64_t half = g->rotary_dim / 2, tail = g->head_dim - g->rotary_dim;
    const int most = g->in_f16 ? 8 : 4;
    const int v = half % most == 0 && tail % most == 0 ? most : half % 4 == 0 && tail % 4 == 0 ? 4 : 1;
    RotaryKern k{};
    k.ld_x = g->ld_x;
    k.ld_y = g->ld_y;
    k.ld_table = g->ld_table;
    k.max_pos = g->max_pos;
    k.table = g->table;
    k.head_dim = (int)g->head_dim;
    k.rot = (int)g->rotary_dim;
    k.rot_units = (uint32_t)(half / v);
    k.per_head = k.rot_units + (uint32_t)((tail + 2 * v - 1) / (2 * v));
    k.per_token = k.per_head * (uint32_t)g->heads;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const size_t e = g->in_f16 ? 2 : 4;
    // launches of fewer than 2^31 units: 32-bit unit numbers
    const int64_t slab = INT32_MAX / (int64_t)k.per_token;
    for (int64_t t0 = 0; t0 < g->tokens; t0 += slab) {
        const int64_t n = g->tokens - t0 < slab ? g->tokens - t0 : slab;
        k.x = static_cast<const char*>(g->x) + (size_t)t0 * g->ld_x * e;
        k.y = static_cast<char*>(g->y) + (size_t)t0 * g->ld_y * e;
        k.positions = g->positions + t0;
        k.units = (uint32_t)(n * k.per_token);
        const bool inter = g->interleaved != 0;
        if (g->in_f16) {
            v == 8 ? launch_rotary<_Float16, 8>(k, inter, s)
                   : v == 4 ? launch_rotary<_Float16, 4>(k, inter, s) : launch_rotary<_Float16, 1>(k, inter, s);
        } else {
            v == 4 ? launch_rotary<float, 4>(k, inter, s) : launch_rotary<float, 1>(k, inter, s);
        }
    }
    return hipGetLastError() == hipSuccess ? NNOPS_OK : NNOPS_INTERNAL;
}

extern "C" int nnops_hip_rotary_table(const NnopsRotaryTableArgs* g, void* stream)
{
    const TimingDisarm disarm;
    if (g == nullptr || g->max_pos < 0 || g->rotary_dim <= 0 || g->rotary_dim % 2 != 0) {
        return NNOPS_INVALID_ARGUMENT;
    }
    if (g->max_pos == 0) {
        return NNOPS_OK;
    }
    if (g->rotary_dim > (1 << 20) || g->max_pos > INT32_MAX) {
        return NNOPS_UNSUPPORTED;
    }
    if (g->table == nullptr || g->ld_table < g->rotary_dim || !(g->base > 0.0) || !(g->factor > 0.0) ||
        !(g->original_context >= 0.0) || (g->original_context > 0.0 && !(g->high_turns > g->low_turns)) ||
        !(g->attention_factor > 0.0)) {
        return NNOPS_INVALID_ARGUMENT;
    }
    const TableKern k{g->table,  g->max_pos,          g->ld_table,  (int)(g->rotary_dim / 2), g->base,
                      g->factor, g->original_context, g->low_turns, g->high_turns,            g->attention_factor};
    const unsigned gx = (unsigned)(g->max_pos < 16384 ? g->max_pos : 16384);
    NNOPS_LAUNCH(rotary_table_kernel, dim3(gx, (unsigned)((k.half + 255) / 256)), dim3(256), 0,
                 static_cast<hipStream_t>(stream), k);
    return hipGetLastError() == hipSuccess ? NNOPS_OK : NNOPS_INTERNAL;
}
