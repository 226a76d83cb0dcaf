// What the kernels of attention over the paged cache share: their parameters,
// which tokens a tile of rows looks at, and the operands of the two products.
#pragma once

#include <limits>
#include <type_traits>

#include "paged.hpp"

namespace nnops_amd {

constexpr int kTile = 64;           // tokens of a step

// Weights are 2^(x - M + kLift) for a reference M that is the running maximum,
// or up to kLazy below it: O and l are brought to a new reference only when the
// maximum has passed the old one by more, which is rare after the first tiles.
// The largest weight is then 2^14, and f16's range ends 2^-30 below the maximum.
constexpr float kLift = 6.0f, kLazy = 8.0f;
constexpr float kDrop = 0x1p-6f;    // 2^-kLift

constexpr float kNone = -std::numeric_limits<float>::infinity();

// What a launch looks at: sequences as they are; the tokens that groups of
// sequences share, as one sequence each of all their rows, which see them all; or
// what the sequences have behind those. (The last two leave all rows in parts.)
enum AttnMode { kWhole, kShared, kOwn };

// How a call with shared tokens is laid out (found on the device).
struct PrefixPlan {
    int32_t shared_chunk, own_chunk;   // tiles of a split
};
struct GroupPlan {
    int32_t start, rows, tokens, table;   // rows of the call, tokens that all share, whose page table
};
struct MemberPlan {
    int32_t group, skip;  // of a sequence: its group or -1, tiles that are the group's
};

struct AttnKern {
    Paged c;
    const void* q;
    void* out;
    int64_t ld_q, ld_out;
    float* part;          // partial O [splits][rows][q_heads][d]
    float* part_ml;       // their M and l [splits][rows][q_heads][2]
    float scale_log2;
    int32_t q_heads, group, window, sinks;
    int32_t tile_rows;    // rows (tokens x heads of a group) of a workgroup
    int32_t per_seq;      // row tiles of a sequence, equal rows each (0: found by search)
    int32_t splits;       // at most, of a tile of rows
    uint32_t by_splits;   // ceil(2^32 / splits): to divide by it
    int32_t tiles;        // of 64 tokens that the page table, or the window, has room for
    int32_t whole;        // tiles of the longest sequence up to which none is split
    int32_t chunk;        // tiles of a split where that sequence fills the table
};

// Of kShared and kOwn.
struct PartKern : AttnKern {
    PrefixPlan* plan;     // workspace, as are the next two: written before these launches, or
    GroupPlan* group_plan;   // (`few`) found by each wave, and written by one for the join
    MemberPlan* members;
    const int32_t* group_starts;
    const int32_t* shared;
    int32_t groups, first_part, few;
    int32_t join_here;    // kOwn, unsplit: joins the shared tokens' parts itself
    int32_t shared_splits;       // as splits and by_splits, of the tokens that groups share
    uint32_t shared_unit;        // tiles that a split of them is a multiple of: 4 where waves take every 4th
    uint32_t by_shared_splits;
};

template <AttnMode M>
using KernOf = std::conditional_t<M == kWhole, AttnKern, PartKern>;

// Where a launch's parts begin among a row's.
template <AttnMode M>
__device__ __forceinline__ int first_part(const KernOf<M>& p)
{
    if constexpr (M == kWhole) {
        return 0;
    } else {
        return p.first_part;
    }
}

// The tiles of 64 tokens that rows at positions pmin .. pmax look at: the
// first `sink_tiles`, then those from `first` on, `tiles` in all.
struct Span {
    int sink_tiles, first, tiles;
};

__host__ __device__ __forceinline__ Span span_of(int pmin, int pmax, int window, int sinks)
{
    Span s{0, 0, pmax < 0 ? 0 : pmax / kTile + 1};
    if (window > 0 && pmax >= 0) {
        const int lo = (pmin > window - 1 ? pmin - window + 1 : 0) / kTile;
        const int kept = sinks < pmax + 1 ? sinks : pmax + 1;
        const int st = (kept + kTile - 1) / kTile;
        if (st < lo) {
            s.sink_tiles = st;
            s.first = lo;
            s.tiles += st - lo;
        }
    }
    return s;
}

__device__ __forceinline__ int tile_base(const Span& s, int v)
{
    return kTile * (v < s.sink_tiles ? v : s.first + v - s.sink_tiles);
}

// A tile of rows of one sequence: row r is head r % group of token r / group
// among the sequence's rows.
struct RowTile {
    int b;
    SeqRows seq;
    int row0, rows;           // first row; rows of the sequence (entry: rows x heads fit 31 bits)
    int pmin, pmax;           // positions of the first and the last row
    Span span;
    int chunk;                // tiles of tokens that a split takes
    bool split;               // it has more than one
    int table;                // kShared: the sequence whose pages they are
    int shared_parts;         // kOwn: parts of the tokens that its group shares
};

// The largest of a wave's values, all 0 or more, as a scalar: along rows of 16
// lanes, then from row to row, the last lane has it.
__device__ __forceinline__ int wave_max(int v)
{
#if __HIP_DEVICE_COMPILE__
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true));   // row_shr:1, 2, 4, 8
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, true));   // row_bcast:15, to rows 1 and 3
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, true));   // row_bcast:31, to rows 2 and 3
    return __builtin_amdgcn_readlane(v, 63);
#else
    return v;
#endif
}

// Tiles of a split where the longest sequence (of shared tokens, or of what is behind
// them) has so many: see chunk_of.
__device__ __forceinline__ int chunk_for(int tiles, int splits, uint32_t by_splits, int whole, uint32_t unit = 4)
{
    if (splits == 1) {
        return std::numeric_limits<int>::max();
    }
    const uint32_t share = __umulhi((uint32_t)(tiles + splits - 1), by_splits);
    return tiles <= whole ? whole : max((int)((share + unit - 1) & ~(unit - 1)), 4);
}

// Tiles of tokens that a split takes: the longest sequence that has rows is
// divided among the splits, whatever the page table has room for (one as wide as
// a model's context, as a captured graph needs: one token over 2048, 64 splits of
// 32 tiles each 19.0 us, by the sequence 10.1; equal shares of each tile of rows
// instead fill a second round where few are longer: f32 1 x 384 of 4000 94 -> 119).
// Whole waves call it; the same in
// all of them. (The product rounds up past the quotient at most: no more splits
// than there are.)
//   own: any sequence (in flight, beside the others). `longest`, of a lane: among
// the sequences before the from-th, which were looked at already.
__device__ __forceinline__ int chunk_of(const AttnKern& p, const SeqRows& own, int longest = 0, int from = 0)
{
    if (p.splits == 1) {
        return std::numeric_limits<int>::max();
    }
    const Paged& c = p.c;
    if (c.seqs == 1) {
        longest = __builtin_amdgcn_readfirstlane(own.len);   // (scalar: loops over the tiles hang on it)
    } else {
        const int lane = threadIdx.x % 64;
        if (from == 0) {                           // (no branch per lane: beside the loads of its own sequence)
            const SeqRows s = seq_rows(c, min(lane, c.seqs - 1));
            longest = s.n > 0 ? s.len : 0;
            from = 64;
        }
        for (int b = from + lane; b < c.seqs; b += 64) {
            const SeqRows s = seq_rows(c, b);
            longest = s.n > 0 ? max(longest, s.len) : longest;
        }
        longest = wave_max(longest);
    }
    const int tiles = min((int)(((uint32_t)longest + kTile - 1) / kTile), p.tiles);
    const uint32_t share = __umulhi((uint32_t)(tiles + p.splits - 1), p.by_splits);
    return tiles <= p.whole ? p.whole : max((int)((share + 3u) & ~3u), 4);
}

template <AttnMode M>
__device__ __forceinline__ void place_tile(const AttnKern& p, int rt, int chunk, RowTile& t, int skip = 0)
{
    const uint32_t group = p.group;
    t.row0 = rt * p.tile_rows;
    t.rows = t.seq.n * p.group;
    const uint32_t last = min(t.row0 + p.tile_rows, t.rows) - 1;
    t.pmin = t.seq.len - t.seq.n + (int)((uint32_t)t.row0 / group);
    t.pmax = t.seq.len - t.seq.n + (int)(last / group);
    t.span = span_of(t.pmin, t.pmax, p.window, p.sinks);
    if constexpr (M == kShared) {
        const int tokens = t.seq.len;              // a multiple of the tile's
        t.pmin = t.pmax = tokens - 1;
        t.span = Span{0, 0, tokens / kTile};
    } else if constexpr (M == kOwn) {
        t.span = Span{0, skip, max(t.span.tiles - skip, 0)};   // (no row's position lies before)
    }
    t.chunk = chunk;
    t.split = t.span.tiles > chunk;
}

// The plan of a call of up to 64 sequences and 8 groups, as every wave finds it: lane
// g has group g, lane b sequence b.
constexpr int kFewGroups = 8;
struct FewPlan {
    SeqRows seq;
    GroupPlan of_group;
    MemberPlan member;
    int shared_chunk, own_chunk;
};

// What a group shares: whole tiles and whole pages that its first sequence has and
// every row sees.
__device__ __forceinline__ int shared_tokens(const Paged& c, int shared, int len, int least)
{
    return max(min(min(shared, len), least), 0) & ~(max(c.page, kTile) - 1);
}

__device__ __forceinline__ FewPlan few_plan(const PartKern& p)
{
    const Paged& c = p.c;
    const int lane = threadIdx.x % 64;
    constexpr int kBig = std::numeric_limits<int>::max();
    FewPlan f{};
    if (lane < c.seqs) {
        f.seq = seq_rows(c, lane);
    }
    int starts = min(max(p.group_starts[min(lane, p.groups)], 0), c.seqs);
    const int shared = lane < p.groups ? p.shared[lane] : 0;
#pragma unroll
    for (int m = 1; m <= kFewGroups; m *= 2) {     // (starts do not go back)
        const int before = __shfl_up(starts, m);
        starts = lane >= m ? max(starts, before) : starts;
    }
    f.member = MemberPlan{-1, 0};
    int longest = 0;
    for (int g = 0; g < p.groups; ++g) {
        const int b0 = __builtin_amdgcn_readlane(starts, g), b1 = __builtin_amdgcn_readlane(starts, g + 1);
        const bool in = lane >= b0 && lane < b1;
        const uint64_t rows = __ballot(in && f.seq.n > 0);
        GroupPlan plan{0, 0, 0, b0};
        if (rows != 0) {
            const int first = __builtin_ctzll(rows), last = 63 - __builtin_clzll(rows);
            const int sees = max(f.seq.len - f.seq.n + 1, 0);
            const int least = kBig - wave_max(in && f.seq.n > 0 ? kBig - sees : 0);
            plan.start = __builtin_amdgcn_readlane(f.seq.start, first);
            plan.rows = max(__builtin_amdgcn_readlane(f.seq.start + f.seq.n, last) - plan.start, 0);
            plan.tokens = shared_tokens(c, __builtin_amdgcn_readlane(shared, g),
                                        __builtin_amdgcn_readlane(f.seq.len, b0), least);
        }
        longest = max(longest, plan.tokens);
        if (lane == g) {
            f.of_group = plan;
        }
        if (in) {
            f.member = MemberPlan{g, plan.tokens / kTile};
        }
    }
    const int own = wave_max(f.seq.n > 0 ? f.seq.len - kTile * f.member.skip : 0);
    f.shared_chunk = chunk_for(longest / kTile, p.shared_splits, p.by_shared_splits, 4, p.shared_unit);
    f.own_chunk = chunk_for(min((own + kTile - 1) / kTile, p.tiles), p.splits, p.by_splits, p.whole);
    return f;
}

// The item-th tile. Later tiles of a sequence look at more tokens: `from_last`
// numbers them from the last, so that the longest work begins first.
template <AttnMode M>
__device__ __forceinline__ bool find_tile(const KernOf<M>& p, uint32_t item, bool from_last, RowTile& t)
{
    int rt, chunk = 0, seqs = p.c.seqs;
    FewPlan few{};
    if constexpr (M != kWhole) {
        seqs = M == kShared ? p.groups : seqs;
        if (p.few) {
            few = few_plan(p);
            if (M == kOwn && item == 0 && blockIdx.y == 0 && threadIdx.x < 64 && (int)threadIdx.x < p.c.seqs) {
                // (what the join needs; by the first workgroup of each KV head, all the same)
                p.members[threadIdx.x] = few.member;
                *p.plan = PrefixPlan{few.shared_chunk, few.own_chunk};
            }
        }
    }
    const auto at = [&](int b) {
        if constexpr (M == kShared) {
            GroupPlan g = few.of_group;            // (few: asked by lane b)
            if (!p.few) {
                g = p.group_plan[b];
            }
            return SeqRows{g.start, g.tokens > 0 ? g.rows : 0, g.tokens};
        } else {
            return seq_rows(p.c, b);
        }
    };
    if (p.per_seq > 0) {
        if (from_last) {
            const uint32_t back = item / (uint32_t)seqs;
            t.b = (int)(item - back * seqs);
            rt = p.per_seq - 1 - (int)back;
        } else {
            t.b = (int)(item / (uint32_t)p.per_seq);
            rt = (int)(item - (uint32_t)t.b * p.per_seq);
        }
        t.seq = at(t.b);
        if constexpr (M == kShared) {              // one group, which may have fewer rows than the call
            t.seq.start = __builtin_amdgcn_readfirstlane(t.seq.start);
            t.seq.n = __builtin_amdgcn_readfirstlane(t.seq.n);
            t.seq.len = __builtin_amdgcn_readfirstlane(t.seq.len);
            if (rt * p.tile_rows >= t.seq.n * p.group) {
                return false;
            }
        }
        if constexpr (M == kWhole) {
            chunk = chunk_of(p, t.seq);
        }
    } else {
        int longest = 0;
        const auto count = [&](const SeqRows& s) {
            longest = s.n > 0 ? max(longest, s.len) : longest;
            return (int)((uint32_t)(s.n * p.group + p.tile_rows - 1) / (uint32_t)p.tile_rows);
        };
        if (!find_item(seqs, item, at, count, t.b, rt, t.seq)) {
            return false;
        }
        if constexpr (M == kWhole) {
            chunk = chunk_of(p, t.seq, longest, (t.b / 64 + 1) * 64);
        }
        rt = from_last ? count(t.seq) - 1 - rt : rt;
    }
    int skip = 0;
    if constexpr (M == kShared) {
        chunk = few.shared_chunk;
        t.table = __builtin_amdgcn_readlane(few.of_group.table, t.b);
        if (!p.few) {
            chunk = p.plan->shared_chunk;
            t.table = p.group_plan[t.b].table;
        }
    } else if constexpr (M == kOwn) {
        chunk = few.own_chunk;
        skip = __builtin_amdgcn_readlane(few.member.skip, t.b);
        uint32_t shared_chunk = (uint32_t)few.shared_chunk;
        if (!p.few) {
            chunk = p.plan->own_chunk;
            skip = p.members[t.b].skip;
            shared_chunk = (uint32_t)p.plan->shared_chunk;
        }
        t.shared_parts = (int)(((uint32_t)skip + shared_chunk - 1) / shared_chunk);
    }
    place_tile<M>(p, rt, chunk, t, skip);
    return true;
}

// A page's scales as they lie in memory, and as the softmax takes them: x = s
// mul + add, l += w inv. (Loaded with the codes, turned where they are used:
// turning them at once would wait for the codes in flight.)
struct PageScales {
    float k, v, off;      // off: NaN where the page does not exist, else 0
};
struct Scales {
    float mul, add, inv;
};

// The page to read for a page number of the table: the first one's codes stand
// in for those of a page that does not exist, under scales that are NaN.
__device__ __forceinline__ bool exists(const Paged& c, int page) { return (uint32_t)page < (uint32_t)c.pages; }
__device__ __forceinline__ int64_t readable(const Paged& c, int page) { return exists(c, page) ? page : 0; }

__device__ __forceinline__ PageScales page_scales(const Paged& c, int page, int kvh)
{
    const int64_t at = readable(c, page) * c.heads + kvh;
    return PageScales{c.k_scale[at], c.v_scale[at], exists(c, page) ? 0.0f : __uint_as_float(0x7fc00000u)};
}

__device__ __forceinline__ Scales softmax_scales(const AttnKern& p, PageScales s)
{
    // (codes of a page whose scale is less count for nothing beside any other)
    const float v = (s.v < kLeastScale ? kLeastScale : s.v) + s.off;
    return Scales{p.scale_log2 * s.k + s.off, __builtin_amdgcn_logf(v), kDrop * __builtin_amdgcn_rcpf(v)};
}

// The operands of the two products, by the rows' type.
//   f16: the rows as they are, codes as f16, the probabilities rounded to f16
//        where many rows share their tiles, as the sum of two f16 (22 bits) where
//        few rows have a workgroup. HBM bounds few rows: the second part costs 1
//        to 5 % (us: one token over 777 9.1 -> 9.25, over 126976 55.4 -> 56.1, of 64
//        sequences of up to 4096 66.4 -> 68.3, heads of 64 36.9 -> 38.6, of 256 49.5
//        -> 50.5). The matrix cores bound many: a prompt of 4096 would take 196
//        instead of 152, for an error that the output's own rounding to f16 exceeds
//        (against 64 bits 2.6e-4 of the result, 2.1e-4 with that rounding alone).
//        Tiles over tokens that sequences share keep what their rows have by
//        themselves: two where these are few.
//   f32: each value as three bf16 parts that hold it exactly (8 bits each, by
//        truncation, the last difference having no more), codes as bf16 (7 bits
//        and a sign: exact), three products into one f32 accumulator. Two f16
//        parts would be one product fewer, but their range ends 2^-38 below the
//        largest probability.
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

template <typename T>
struct Operand {
    static constexpr int kParts = 1;
    typedef v8h Vec;
    static __device__ __forceinline__ Vec codes(uint32_t a, uint32_t b)
    {
        // a byte u of 0x64uu is 1024 + u; u = code ^ 0x80 is code + 128
        a ^= 0x80808080u;
        b ^= 0x80808080u;
        const v4u w{__builtin_amdgcn_perm(0x64646464u, a, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u),
                    __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)};
        Vec h;
        __builtin_memcpy(&h, &w, 16);
        return h - (_Float16)1152.0f;
    }
    template <typename S>
    static __device__ __forceinline__ void split(const S (&x)[8], Vec (&v)[1])
    {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[0][e] = (_Float16)x[e];   // (in pairs: v_cvt_pk_f16_f32, to nearest)
        }
    }
    static __device__ __forceinline__ void split(const float (&x)[8], Vec (&v)[2])
    {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[0][e] = (_Float16)x[e];
            v[1][e] = (_Float16)__fsub_rn(x[e], (float)v[0][e]);
        }
    }
    // The same values by 4 instructions a pair instead of 8 (v_fma_mix_f32 takes f16 as they
    // lie in a register), for tiles of many rows, which vector instructions bound as well.
    // minus_one: -1 that the compiler does not know, or it makes them two steps again.
    static __device__ __forceinline__ void split_in_pairs(const float (&x)[8], Vec (&v)[2], float minus_one)
    {
#if __HIP_DEVICE_COMPILE__
        typedef _Float16 v2h __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            v2h h{(_Float16)x[e], (_Float16)x[e + 1]};
            asm("" : "+v"(h));                     // (one conversion for both parts)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                v[0][e + i] = h[i];
                v[1][e + i] = (_Float16)__builtin_fmaf((float)h[i], minus_one, x[e + i]);   // (exact before its rounding)
            }
        }
#else
        (void)x, (void)v, (void)minus_one;
#endif
    }
    static __device__ __forceinline__ v4f mfma(Vec a, Vec b, v4f c)
    {
#if __HIP_DEVICE_COMPILE__
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
#else
        (void)a, (void)b;
        return c;
#endif
    }
    static __device__ __forceinline__ v16f mfma(Vec a, Vec b, v16f c)
    {
#if __HIP_DEVICE_COMPILE__
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
#else
        (void)a, (void)b;
        return c;
#endif
    }
};

template <>
struct Operand<float> {
    static constexpr int kParts = 3;
    typedef v8b Vec;
    // the upper halves of two f32
    static __device__ __forceinline__ uint32_t uppers(float lo, float hi)
    {
        return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
    }
    static __device__ __forceinline__ Vec codes(uint32_t a, uint32_t b)
    {
        // (a signed byte to f32: one instruction that picks it. Unsigned bytes less
        // 128 took two and more: vector instructions bound f32 rows, 7 ragged
        // sequences of up to 2500, 16 heads of 64, window 1024: 31.6 -> 26.2 us)
        const uint32_t d[2] = {a, b};
        v4u w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = d[i / 2] >> (16 * (i % 2));
            w[i] = uppers((float)(int8_t)u, (float)(int8_t)(u >> 8));
        }
        Vec h;
        __builtin_memcpy(&h, &w, 16);
        return h;
    }
    static __device__ __forceinline__ void split(const float (&x)[8], Vec (&v)[3])
    {
        float r[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            r[e] = x[e];
        }
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const v4u w{uppers(r[0], r[1]), uppers(r[2], r[3]), uppers(r[4], r[5]), uppers(r[6], r[7])};
            __builtin_memcpy(&v[i], &w, 16);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                r[e] = __fsub_rn(r[e], __uint_as_float(__float_as_uint(r[e]) & 0xffff0000u));
            }
        }
    }
    static __device__ __forceinline__ v4f mfma(Vec a, Vec b, v4f c)
    {
#if __HIP_DEVICE_COMPILE__
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
#else
        (void)a, (void)b;
        return c;
#endif
    }
    static __device__ __forceinline__ v16f mfma(Vec a, Vec b, v16f c)
    {
#if __HIP_DEVICE_COMPILE__
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
#else
        (void)a, (void)b;
        return c;
#endif
    }
};

// c + a (b's parts)
template <typename T, int N, typename Acc>
__device__ __forceinline__ Acc product(typename Operand<T>::Vec a, const typename Operand<T>::Vec (&b)[N], Acc c)
{
#pragma unroll
    for (int i = 0; i < N; ++i) {
        c = Operand<T>::mfma(a, b[i], c);
    }
    return c;
}

// Lanes that join a row's parts, 4 channels each.
__host__ __device__ __forceinline__ int join_lanes(int d) { return d <= 64 ? 16 : d <= 128 ? 32 : 64; }

struct AttnPlan {
    int64_t items;        // row tiles, all KV heads
    int32_t tile_rows, per_seq, chunk, splits, tiles, whole;
    bool tiled;           // attention_rows_tiled, else attention_rows16
    bool join_few;        // attention_join_few joins the splits, else attention_join
    size_t workspace;
};

// The choice for a call whose sizes check_attention_shapes lets pass (-1), and whether
// a launch holds it.
int check_attention_shapes(const NnopsCacheAttentionArgs* g);
AttnPlan attn_plan(const NnopsCacheAttentionArgs* g);
inline bool launch_holds(const AttnPlan& a)
{
    return a.items <= std::numeric_limits<int32_t>::max() / 512 && a.splits <= 65535;
}

// attention_rows_tiled's launch (cache_attention_tiled.hip): d, type and rows
// of a workgroup that it has a kernel for.
int tiled_rows(int64_t d, bool f16, int64_t page, int64_t rows);
// Its form for tiles that lie in one page (wider heads come with such pages only).
inline bool tiled_one_page(int64_t d, int64_t page) { return d > 128 || page >= kTile; }
void launch_tiled(const AttnKern& k, const dim3& grid, bool f16, hipStream_t s);

}  // namespace nnops_amd
