// The 8-bit key / value cache: rows quantized into pages as they are written,
// and read back. A page has one scale per KV head and side (keys, values):
//   scale = max(old scale, max |new| / 127, 2^-100)
//   new code = rint(x (1 / scale)),  older code = rint(code (old / scale))
// so a page whose scale grows is rewritten; it can grow only as long as the
// page fills.
//
// Bound: HBM: the new rows and their codes; reading back, the codes and the
// values; for few tokens the chain of loads (lengths, page table, codes). One
// unit of waves owns one page of a sequence, one head and one side, so that a
// page's maximum needs no atomics and every run gives the same bits: a single
// wave where a page and head hold at most 4096 values, a workgroup of 4 waves
// else. Rows stay in registers between the maximum and the codes.
// Values lie transposed in a page (a channel's tokens side by side): writing, a
// thread takes 4 tokens by 8 channels, whole 16-byte loads, and stores a dword
// of 4 tokens per channel (two channels by 16 tokens, 4-byte loads and 16-byte
// stores, ran 11.1 us where keys take 6.2: a prompt of 4096, pages of 16);
// reading, two channels by 16 tokens, so that its lanes write whole rows.
// Measured, 8 heads of 128, f16: a prompt of 4096 tokens, pages of 16, 25 MB each
// way: written in 10.6 us, read in 8.8; 32 sequences of 1000, pages of 64: read in
// 20.6 us (98 MB, 4.8 TB/s), a token appended to each in 5.1, in 6.6 where every
// page's scale grows (pages of 16: 4.9 and 5.9, of 128: 5.1 and 8.3). All waves of
// the prompt's write are resident at once: it is one chain (lengths, table, rows,
// the page's maximum, codes) long, in which 8 vector instructions a value counted
// (now 4: 11.6 -> 10.6 us); asking for the rows before the page number is looked at
// did not.
#include "paged.hpp"

namespace nnops_amd {

int check_page_shapes(const NnopsKvPages& c, int64_t rows)
{
    if (rows < 0 || c.sequences < 0 || c.pages < 0 || c.heads < 0 || c.table_pages < 0) {
        return NNOPS_INVALID_ARGUMENT;
    }
    const int64_t t = c.page_tokens, d = c.head_dim;
    if (t != 16 && t != 32 && t != 64 && t != 128 && t != 256) {
        return NNOPS_UNSUPPORTED;
    }
    if (d < 16 || d > 256 || d % 16 != 0) {
        return NNOPS_UNSUPPORTED;
    }
    if (rows == 0 || c.heads == 0) {
        return NNOPS_OK;
    }
    if (rows > INT32_MAX / 2 || c.sequences > INT32_MAX / 2 || c.pages > INT32_MAX || c.heads > (1 << 16) ||
        c.table_pages > INT32_MAX / t || c.heads * t * d > INT32_MAX) {
        return NNOPS_UNSUPPORTED;
    }
    if (c.sequences == 0 || (c.row_starts == nullptr && rows % c.sequences != 0)) {
        return NNOPS_INVALID_ARGUMENT;
    }
    return -1;
}

int check_page_memory(const NnopsKvPages& c)
{
    if (c.page_table == nullptr || c.lengths == nullptr || c.ld_table < c.table_pages) {
        return NNOPS_INVALID_ARGUMENT;
    }
    if (c.pages > 0 && (c.k == nullptr || c.v == nullptr || c.k_scale == nullptr || c.v_scale == nullptr ||
                        (uintptr_t)c.k % 16 != 0 || (uintptr_t)c.v % 16 != 0)) {
        return NNOPS_INVALID_ARGUMENT;
    }
    return -1;
}

Paged paged(const NnopsKvPages& c, int64_t rows)
{
    Paged p{};
    p.k = c.k;
    p.v = c.v;
    p.k_scale = c.k_scale;
    p.v_scale = c.v_scale;
    p.table = c.page_table;
    p.lengths = c.lengths;
    p.row_starts = c.row_starts;
    p.ld_table = c.ld_table;
    p.pages = (int32_t)c.pages;
    p.heads = (int32_t)c.heads;
    p.page = (int32_t)c.page_tokens;
    p.page_log2 = __builtin_ctzll((unsigned long long)c.page_tokens);
    p.d = (int32_t)c.head_dim;
    p.seqs = (int32_t)c.sequences;
    p.table_pages = (int32_t)c.table_pages;
    p.rows = (int32_t)rows;
    p.uniform = (int32_t)(rows / c.sequences);
    return p;
}

namespace {

struct RowsKern {
    Paged c;
    void* k;
    void* v;
    int64_t ld_k, ld_v;
    int32_t per_seq;      // items of a sequence, equal rows each (0: found by search)
    int32_t head_groups;  // groups of heads of an item, a workgroup (and side) each
    int32_t group_heads;  // heads of a group
    uint32_t row_magic;   // ceil(2^32 / x), x the 16-byte pieces of group_heads heads' values: to divide by x
};

// Items of a sequence: the pages that its rows of the call fall in; one, of no
// slots, where it has rows but holds no tokens.
__device__ __forceinline__ int touched(const Paged& p, const SeqRows& s)
{
    const int first = max(s.len - s.n, 0);
    return s.n <= 0 ? 0 : s.len <= first ? 1 : ((s.len - 1) >> p.page_log2) - (first >> p.page_log2) + 1;
}

// The part of a page that a workgroup has: slots [from, to) are rows of the
// call, row `row` + slot - from; slots before `from` are older tokens. `absent`
// rows before it (of a sequence's first item) stand for no token.
struct PagePart {
    int id, from, to, absent;
    int64_t row;
};

__device__ __forceinline__ bool page_part(const RowsKern& p, uint32_t item, PagePart& t)
{
    int b, j;
    SeqRows s;
    if (p.per_seq > 0) {
        b = (int)(item / (uint32_t)p.per_seq);
        j = (int)(item - (uint32_t)b * p.per_seq);
        s = seq_rows(p.c, b);
        if (j >= touched(p.c, s)) {
            return false;
        }
    } else if (!find_item(p.c, item, [&](const SeqRows& q) { return touched(p.c, q); }, b, j, s)) {
        return false;
    }
    const int first = max(s.len - s.n, 0);
    const int page = (first >> p.c.page_log2) + j, base = page << p.c.page_log2;
    t.from = max(first - base, 0);
    t.to = min(s.len - base, p.c.page);
    t.id = t.to > t.from ? page_of(p.c, b, page) : -1;
    t.absent = j == 0 ? max(s.n - s.len, 0) : 0;
    t.row = (int64_t)s.start + (base + t.from) - (s.len - s.n);
    return true;
}

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t code_byte(float x, float inv)
{
    const int q = (int)__builtin_rintf(__fmul_rn(x, inv));
    return (uint32_t)min(max(q, -127), 127) & 0xffu;
}

// The codes of four new values. Their magnitudes are a page's largest at most,
// so that x inv is 127 (1 + 2^-22) at most and needs no clamp, and adding 1.5 2^23
// leaves its nearest integer (ties to even) in the sum's lowest byte.
template <typename T>
__device__ __forceinline__ uint32_t new_codes(T x0, T x1, T x2, T x3, float inv)
{
    const float magic = 12582912.0f;
    const uint32_t u0 = __float_as_uint(__fadd_rn(__fmul_rn((float)x0, inv), magic));
    const uint32_t u1 = __float_as_uint(__fadd_rn(__fmul_rn((float)x1, inv), magic));
    const uint32_t u2 = __float_as_uint(__fadd_rn(__fmul_rn((float)x2, inv), magic));
    const uint32_t u3 = __float_as_uint(__fadd_rn(__fmul_rn((float)x3, inv), magic));
    return __builtin_amdgcn_perm(u1, u0, 0x0c0c0400u) | __builtin_amdgcn_perm(u3, u2, 0x04000c0cu);
}

// The largest magnitude of N values, as the bits of an f32 (NaNs above all).
template <int N>
__device__ __forceinline__ uint32_t largest(const float (&x)[N])
{
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        m = max(m, magnitude(x[e]));
    }
    return m;
}

template <int N>
__device__ __forceinline__ uint32_t largest(const _Float16 (&x)[N])
{
    typedef uint16_t v2u16 __attribute__((ext_vector_type(2)));
    v2u16 m{0, 0}, w[N / 2];
    __builtin_memcpy(w, x, sizeof w);
#pragma unroll
    for (int e = 0; e < N / 2; ++e) {
        m = __builtin_elementwise_max(m, w[e] & v2u16{0x7fff, 0x7fff});
    }
    return magnitude((float)__builtin_bit_cast(_Float16, max(m[0], m[1])));
}

// Byte e of a dword as a signed code, scaled to the grown step.
__device__ __forceinline__ uint32_t rescaled(uint32_t d, float ratio)
{
    uint32_t o = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        o |= code_byte((float)(int8_t)(d >> (8 * e)), ratio) << (8 * e);
    }
    return o;
}

// blockIdx.x: item, group of heads; blockIdx.y: keys or values. A unit of WAVES
// waves has a head: 4 heads a workgroup, or one.
template <typename T, int WAVES>
__global__ __launch_bounds__(256) void kv_write_kernel(const RowsKern p)
{
    constexpr int kLanes = 64 * WAVES;
    constexpr int kHeldK = 4, kHeldV = 2;          // pieces of a thread that stay in registers
    __shared__ uint32_t s_max[4];
    const Paged& c = p.c;
    const uint32_t item = blockIdx.x / (uint32_t)p.head_groups;
    const int group = (int)(blockIdx.x - item * p.head_groups);
    const bool values = blockIdx.y != 0;
    PagePart t;
    if (!page_part(p, item, t) || t.id < 0) {
        return;                                    // the whole workgroup
    }
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int head = WAVES == 1 ? group * 4 + wave : group;
    if (head >= c.heads) {
        return;                                    // (WAVES == 1: no barrier below)
    }
    const int lane = WAVES == 1 ? threadIdx.x % 64 : threadIdx.x;
    const int d = c.d, n = t.to - t.from;
    const int64_t ld = values ? p.ld_v : p.ld_k;
    const T* rows = static_cast<const T*>(values ? p.v : p.k) + t.row * ld + (int64_t)head * d;
    float* scale = (values ? c.v_scale : c.k_scale) + (int64_t)t.id * c.heads + head;
    int8_t* page = (values ? c.v : c.k) + ((int64_t)t.id * c.heads + head) * ((int64_t)c.page * d);
    const float old = t.from > 0 ? *scale : 0.0f;

    // pieces: keys, 16 channels of a row; values, 8 channels of 4 slots
    const uint32_t per_row = d / 16, eighths = d / 8;
    const int q0 = t.from / 4, quads = (t.to + 3) / 4 - q0;
    const int pieces = values ? quads * (int)eighths : n * (int)per_row;
    const auto load_k = [&](int i, T (&x)[16]) {
        const uint32_t r = (uint32_t)i / per_row, at = ((uint32_t)i - r * per_row) * 16;
        __builtin_memcpy(x, rows + (int64_t)r * ld + at, sizeof x);
    };
    const auto load_v = [&](int i, T (&x)[4][8]) {
        const uint32_t q = (uint32_t)i / eighths, ch = ((uint32_t)i - q * eighths) * 8;
        const int slot0 = (q0 + (int)q) * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int slot = slot0 + e;
            if (slot >= t.from && slot < t.to) {
                __builtin_memcpy(x[e], rows + (int64_t)(slot - t.from) * ld + ch, sizeof x[e]);
            } else {
#pragma unroll
                for (int h = 0; h < 8; ++h) {
                    x[e][h] = (T)0.0f;
                }
            }
        }
    };
    const auto most = [&](const T (&x)[4][8]) {
        return max(max(largest(x[0]), largest(x[1])), max(largest(x[2]), largest(x[3])));
    };
    T held_k[kHeldK][16], held_v[kHeldV][4][8];
    uint32_t a = 0;
    if (!values) {
#pragma unroll
        for (int h = 0; h < kHeldK; ++h) {
            if (lane + h * kLanes < pieces) {
                load_k(lane + h * kLanes, held_k[h]);
                a = max(a, largest(held_k[h]));
            }
        }
        for (int i = lane + kHeldK * kLanes; i < pieces; i += kLanes) {
            T x[16];
            load_k(i, x);
            a = max(a, largest(x));
        }
    } else {
#pragma unroll
        for (int h = 0; h < kHeldV; ++h) {
            if (lane + h * kLanes < pieces) {
                load_v(lane + h * kLanes, held_v[h]);
                a = max(a, most(held_v[h]));
            }
        }
        for (int i = lane + kHeldV * kLanes; i < pieces; i += kLanes) {
            T x[4][8];
            load_v(i, x);
            a = max(a, most(x));
        }
    }
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        a = max(a, (uint32_t)__shfl_xor((int)a, m));
    }
    if constexpr (WAVES > 1) {
        if (threadIdx.x % 64 == 0) {
            s_max[wave] = a;
        }
        __syncthreads();                           // (every thread has read the old scale, too)
        a = max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3]));
    }
    // a NaN (of the rows or of the page before) stays one; fmaxf would drop it
    const bool bad = a >= 0x7f800000u || !(old == old);
    const float s = bad ? __uint_as_float(0x7fc00000u)
                        : fmaxf(fmaxf(old, __fmul_rn(__uint_as_float(a), 1.0f / 127.0f)), kLeastScale);
    const float inv = bad ? 0.0f : __fdiv_rn(1.0f, s);
    const uint32_t good = bad ? 0u : ~0u;          // codes of such pages are 0
    const bool grew = !bad && t.from > 0 && s > old;
    const float ratio = grew ? __fdiv_rn(old, s) : 1.0f;
    if (lane == 0) {
        *scale = s;
    }

    if (!values) {
        const auto write = [&](int i, const T (&x)[16]) {
            const uint32_t r = (uint32_t)i / per_row, at = ((uint32_t)i - r * per_row) * 16;
            uint32_t o[4] = {0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                o[e] = good & new_codes(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3], inv);
            }
            *reinterpret_cast<v4i*>(page + (t.from + r) * d + at) = v4i{(int)o[0], (int)o[1], (int)o[2], (int)o[3]};
        };
#pragma unroll
        for (int h = 0; h < kHeldK; ++h) {
            if (lane + h * kLanes < pieces) {
                write(lane + h * kLanes, held_k[h]);
            }
        }
        for (int i = lane + kHeldK * kLanes; i < pieces; i += kLanes) {
            T x[16];
            load_k(i, x);
            write(i, x);
        }
        if (grew) {
            for (int i = lane; i < t.from * (int)per_row; i += kLanes) {
                v4i* at = reinterpret_cast<v4i*>(page) + i;            // rows of a page are dense
                const v4i w = *at;
                *at = v4i{(int)rescaled((uint32_t)w.x, ratio), (int)rescaled((uint32_t)w.y, ratio),
                          (int)rescaled((uint32_t)w.z, ratio), (int)rescaled((uint32_t)w.w, ratio)};
            }
        }
        return;
    }
    // a dword that holds older tokens as well keeps those, brought to the scale
    // where it grew
    const auto write = [&](int i, const T (&x)[4][8]) {
        const uint32_t q = (uint32_t)i / eighths, ch = ((uint32_t)i - q * eighths) * 8;
        const int slot0 = (q0 + (int)q) * 4;
        uint32_t mine = 0;                         // the bytes of new tokens
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            mine |= slot0 + e >= t.from && slot0 + e < t.to ? 0xffu << (8 * e) : 0u;
        }
        uint32_t* dst = reinterpret_cast<uint32_t*>(page + ch * c.page + slot0);
        uint32_t old_dword[8] = {};
        if (mine != ~0u) {
#pragma unroll
            for (int h = 0; h < 8; ++h) {
                old_dword[h] = dst[h * (c.page / 4)];
            }
        }
#pragma unroll
        for (int h = 0; h < 8; ++h) {
            uint32_t o = good & new_codes(x[0][h], x[1][h], x[2][h], x[3][h], inv);
            if (mine != ~0u) {
                o = (o & mine) | ((grew ? rescaled(old_dword[h], ratio) : old_dword[h]) & ~mine);
            }
            dst[h * (c.page / 4)] = o;
        }
    };
#pragma unroll
    for (int h = 0; h < kHeldV; ++h) {
        if (lane + h * kLanes < pieces) {
            write(lane + h * kLanes, held_v[h]);
        }
    }
    for (int i = lane + kHeldV * kLanes; i < pieces; i += kLanes) {
        T x[4][8];
        load_v(i, x);
        write(i, x);
    }
    if (grew) {                                    // older tokens only: 16 at a time, and the dwords left
        const int whole = t.from / 16, left = q0 - 4 * whole;
        for (int i = lane; i < whole * d; i += kLanes) {
            const uint32_t ch = (uint32_t)i / (uint32_t)whole, g = (uint32_t)i - ch * whole;
            v4i* at = reinterpret_cast<v4i*>(page + ch * c.page) + g;
            const v4i w = *at;
            *at = v4i{(int)rescaled((uint32_t)w.x, ratio), (int)rescaled((uint32_t)w.y, ratio),
                      (int)rescaled((uint32_t)w.z, ratio), (int)rescaled((uint32_t)w.w, ratio)};
        }
        for (int i = lane; i < left * d; i += kLanes) {
            const uint32_t ch = (uint32_t)i / (uint32_t)left, q = (uint32_t)i - ch * left;
            uint32_t* at = reinterpret_cast<uint32_t*>(page + ch * c.page) + 4 * whole + q;
            *at = rescaled(*at, ratio);
        }
    }
}

// Values that the kernel does not read again, stored past the caches as far as
// they let it, whatever the row's alignment (32 sequences of 1000, 65 MB read back,
// of six caches in turn: 28.9 us, 35.5 with plain stores; f32 35.5 and 52.1. Such
// stores have to fill whole lines: 32 or 64 bytes a lane took 99 us).
template <typename T, int N>
__device__ __forceinline__ void put_once(T* to, const T (&y)[N])
{
    typedef int Word __attribute__((ext_vector_type(sizeof(T) * N / 4), aligned(sizeof(T))));
    Word w;
    __builtin_memcpy(&w, y, sizeof w);
    __builtin_nontemporal_store(w, reinterpret_cast<Word*>(to));
}

// A workgroup reads one page of a group of heads, one side; the heads' pieces
// side by side in a row, so that what it writes of a row is contiguous.
template <typename T>
__global__ __launch_bounds__(256) void kv_read_kernel(const RowsKern p)
{
    const Paged& c = p.c;
    const uint32_t item = blockIdx.x / (uint32_t)p.head_groups;
    const int head0 = (int)(blockIdx.x - item * p.head_groups) * p.group_heads;
    const int heads = min(p.group_heads, c.heads - head0);
    const bool values = blockIdx.y != 0;
    PagePart t;
    if (!page_part(p, item, t)) {
        return;
    }
    const int d = c.d;
    const int64_t ld = values ? p.ld_v : p.ld_k;
    T* rows = static_cast<T*>(values ? p.v : p.k) + t.row * ld + (int64_t)head0 * d;
    const int width = heads * d;
    for (int64_t i = threadIdx.x; i < (int64_t)t.absent * width; i += 256) {
        const int64_t r = i / width;
        rows[(r - t.absent) * ld + (i - r * width)] = (T)0.0f;
    }
    const bool there = t.id >= 0;
    const int64_t at_page = there ? (int64_t)t.id * c.heads + head0 : 0;
    const float* scales = (values ? c.v_scale : c.k_scale) + at_page;
    const uint32_t bytes = (uint32_t)c.page * d;
    const int8_t* page = (values ? c.v : c.k) + at_page * (int64_t)bytes;
    const float nan = __uint_as_float(0x7fc00000u);
    if (!values) {
        // 16 bytes of a row a thread: side by side in a wave, whole lines
        constexpr int kP = 16 / sizeof(T);
        const uint32_t per_tok = d / kP, per_row = per_tok * p.group_heads;
        const int n = (t.to - t.from) * (int)per_row;
#pragma unroll 4
        for (int i = threadIdx.x; i < n; i += 256) {
            const uint32_t r = __umulhi((uint32_t)i, p.row_magic), in = (uint32_t)i - r * per_row;
            const uint32_t h = in / per_tok, at = (in - h * per_tok) * kP;
            if ((int)h >= heads) {
                continue;
            }
            uint32_t wd[kP / 4] = {};
            if (there) {
                __builtin_memcpy(wd, __builtin_assume_aligned(page + h * bytes + (t.from + r) * d + at, kP), kP);
            }
            const float s = there ? scales[h] : nan;
            T y[kP];
#pragma unroll
            for (int e = 0; e < kP; ++e) {
                y[e] = (T)__fmul_rn((float)(int8_t)(wd[e / 4] >> (8 * (e % 4))), s);
            }
            put_once(rows + (int64_t)r * ld + h * d + at, y);
        }
        return;
    }
    const int g0 = t.from / 16, groups = (t.to + 15) / 16 - g0;
    const uint32_t pairs = d / 2, all = pairs * heads;
    for (int i = threadIdx.x; i < groups * (int)all; i += 256) {
        const uint32_t g = (uint32_t)i / all, in = (uint32_t)i - g * all, h = in / pairs, ch = (in - h * pairs) * 2;
        const int slot0 = (g0 + (int)g) * 16;
        uint32_t wd[2][4];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const v4i w = there ? *reinterpret_cast<const v4i*>(page + h * bytes + (ch + q) * c.page + slot0) : v4i{0, 0, 0, 0};
            wd[q][0] = (uint32_t)w.x, wd[q][1] = (uint32_t)w.y, wd[q][2] = (uint32_t)w.z, wd[q][3] = (uint32_t)w.w;
        }
        const float s = there ? scales[h] : nan;
        T* dst = rows + (int64_t)(slot0 - t.from) * ld + (h * d + ch);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int slot = slot0 + e;
            if (slot >= t.from && slot < t.to) {
                T y[2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    y[q] = (T)__fmul_rn((float)(int8_t)(wd[q][e / 4] >> (8 * (e % 4))), s);
                }
                put_once(dst + e * ld, y);
            }
        }
    }
}

// Workgroups along x: pages that the rows can fall in, by heads.
int64_t items(const NnopsKvRowsArgs* g, int32_t& per_seq)
{
    const int64_t t = g->cache.page_tokens, b = g->cache.sequences;
    if (g->cache.row_starts == nullptr) {
        const int64_t n = g->rows / b;
        per_seq = (int32_t)((n + t - 2) / t + 1);
        const int64_t held = g->cache.table_pages > 0 ? g->cache.table_pages : 1;
        per_seq = (int32_t)(per_seq < held ? per_seq : held);
        return b * per_seq;
    }
    per_seq = 0;
    // sum over the sequences that have rows of (n + t - 2) / t + 1
    const int64_t most = g->rows / t + 2 * (b < g->rows ? b : g->rows);
    return most;
}

int check_rows(const NnopsKvRowsArgs* g)
{
    if (g == nullptr) {
        return NNOPS_INVALID_ARGUMENT;
    }
    if (const int rc = check_page_shapes(g->cache, g->rows); rc >= 0) {
        return rc;
    }
    if (const int rc = check_page_memory(g->cache); rc >= 0) {
        return rc;
    }
    const int64_t width = g->cache.heads * g->cache.head_dim;
    if (g->k_rows == nullptr || g->v_rows == nullptr || g->ld_k < width || g->ld_v < width) {
        return NNOPS_INVALID_ARGUMENT;
    }
    return -1;
}

RowsKern rows_kern(const NnopsKvRowsArgs* g, int32_t per_seq, int32_t group_heads)
{
    RowsKern k{};
    k.c = paged(g->cache, g->rows);
    k.k = g->k_rows;
    k.v = g->v_rows;
    k.ld_k = g->ld_k;
    k.ld_v = g->ld_v;
    k.per_seq = per_seq;
    k.group_heads = group_heads;
    k.head_groups = (k.c.heads + group_heads - 1) / group_heads;
    const uint32_t per_row = (uint32_t)(group_heads * (k.c.d / (g->f16 ? 8 : 4)));
    k.row_magic = (uint32_t)(((1ull << 32) + per_row - 1) / per_row);
    return k;
}

}  // namespace
}  // namespace nnops_amd

using namespace nnops_amd;

extern "C" int nnops_hip_kv_cache_write(const NnopsKvRowsArgs* g, void* stream)
{
    const TimingDisarm disarm;
    const int rc = check_rows(g);
    if (rc >= 0) {
        return rc;
    }
    int32_t per_seq = 0;
    const int64_t n = items(g, per_seq);
    if (n == 0 || g->cache.pages == 0) {
        return NNOPS_OK;                          // no page to write to
    }
    // (written and read, us: 4096 tokens, pages of 16 x 128: a wave 17.2, four 22.6; of
    // 64 x 128: a wave 22.4, four 16.6)
    const bool small = g->cache.page_tokens * g->cache.head_dim <= 4096;
    const RowsKern k = rows_kern(g, per_seq, small ? 4 : 1);
    if (n * k.head_groups > INT32_MAX / 256) {
        return NNOPS_UNSUPPORTED;
    }
    const dim3 grid((unsigned)(n * k.head_groups), 2);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (g->f16) {
        if (small) {
            NNOPS_LAUNCH((kv_write_kernel<_Float16, 1>), grid, dim3(256), 0, s, k);
        } else {
            NNOPS_LAUNCH((kv_write_kernel<_Float16, 4>), grid, dim3(256), 0, s, k);
        }
    } else if (small) {
        NNOPS_LAUNCH((kv_write_kernel<float, 1>), grid, dim3(256), 0, s, k);
    } else {
        NNOPS_LAUNCH((kv_write_kernel<float, 4>), grid, dim3(256), 0, s, k);
    }
    return hipGetLastError() == hipSuccess ? NNOPS_OK : NNOPS_INTERNAL;
}

extern "C" int nnops_hip_kv_cache_read(const NnopsKvRowsArgs* g, void* stream)
{
    const TimingDisarm disarm;
    const int rc = check_rows(g);
    if (rc >= 0) {
        return rc;
    }
    int32_t per_seq = 0;
    const int64_t n = items(g, per_seq);
    // heads of a workgroup: 8192 codes, as long as there are workgroups to fill
    // the chip (32 sequences of 1000, plain stores: 26.1 us, 28.0 with 16384, 32.3
    // with 32768)
    int32_t group = (int32_t)(8192 / (g->cache.page_tokens * g->cache.head_dim));
    group = group < 1 ? 1 : group > g->cache.heads ? (int32_t)g->cache.heads : group;
    while (group > 1 && n * 2 * ((g->cache.heads + group - 1) / group) < 2048) {
        group /= 2;
    }
    const RowsKern k = rows_kern(g, per_seq, group);
    if (n * k.head_groups > INT32_MAX / 256) {
        return NNOPS_UNSUPPORTED;
    }
    const dim3 grid((unsigned)(n * k.head_groups), 2);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (g->f16) {
        NNOPS_LAUNCH(kv_read_kernel<_Float16>, grid, dim3(256), 0, s, k);
    } else {
        NNOPS_LAUNCH(kv_read_kernel<float>, grid, dim3(256), 0, s, k);
    }
    return hipGetLastError() == hipSuccess ? NNOPS_OK : NNOPS_INTERNAL;
}
