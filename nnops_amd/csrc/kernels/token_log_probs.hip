// Log probabilities of given tokens, the entropy and the most probable tokens of
// rows of logits, in one pass over them.
//
// With a reference r for a row (its largest logit so far) and y_j = (x_j - r)
// log2(e):
//   s = sum 2^y_j,  t = sum y_j 2^y_j
//   log p_j = ln 2 (y_j - log2 s),  entropy = ln 2 (log2 s - t / s)
// and s, t are brought to a new reference when the maximum grows (by d = y of the
// old one: s' = 2^d s, t' = 2^d (t + d s)), which a row's first tiles do and later
// ones hardly. f16 rows: y = fma(x, log2(e), -r log2(e)): the rounding of the
// second product is the same for all, and drops out. f32 rows: (x - r) log2(e),
// which masks of the type's lowest value do not take out of f32's range.
//
// The most probable: keys of 64 bits, the logit's bits in an order that whole
// numbers have, then the token's complement, so that no two are equal. A wave
// keeps those above a threshold (the top-th of what it has seen, as far as it
// knows) in LDS and drops all but the top when there is no room: after the first
// tile about top ln(n / 512) of n logits come that far.
//
// Bound: HBM, the logits read once.
#include <limits>

#include "common.hpp"

namespace nnops_amd {
namespace {

constexpr int kTile = 512;          // logits of a wave's step, 8 a lane
constexpr int kCap = 1024;          // keys that a wave has room for
constexpr int kMostTop = 32;
constexpr int kMostSplits = 64;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNone = -std::numeric_limits<float>::infinity();

struct LogProbsKern {
    const void* x;
    const int32_t* tokens;
    float* log_probs;
    float* entropy;
    int32_t* top_tokens;
    float* top_log_probs;
    int64_t ld_x, ld_tokens, ld_log_probs, ld_top_tokens, ld_top_log_probs;
    int32_t vocab, per_row, top, splits, part;   // part: logits of a split
    float* stats;         // workspace: reference, s, t of [rows][splits]
    uint64_t* keys;       //   keys of [rows][splits][top]
};

// The reference that goes with a maximum, y against it, and y of an old one.
template <typename T>
struct Reference;
template <>
struct Reference<_Float16> {
    static constexpr float kLeast = -1e38f;        // (its product is finite)
    static __device__ __forceinline__ float of(float m) { return m * kLog2e; }
    static __device__ __forceinline__ float y(float x, float r) { return __builtin_fmaf(x, kLog2e, -r); }
    static __device__ __forceinline__ float step(float old, float r) { return old - r; }
    static __device__ __forceinline__ float log_p(float x, float r, float s)
    {
        return (y(x, r) - log2f(s)) * kLn2;
    }
};
template <>
struct Reference<float> {
    static constexpr float kLeast = -std::numeric_limits<float>::max();
    static __device__ __forceinline__ float of(float m) { return m; }
    static __device__ __forceinline__ float y(float x, float r) { return (x - r) * kLog2e; }
    static __device__ __forceinline__ float step(float old, float r) { return (old - r) * kLog2e; }
    static __device__ __forceinline__ float log_p(float x, float r, float s) { return (x - r) - logf(s); }
};

__device__ __forceinline__ uint64_t key_of(float x, int token)
{
    const uint32_t b = __float_as_uint(x + 0.0f);  // (-0 and 0 are equal)
    const uint32_t order = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return (uint64_t)order << 32 | ~(uint32_t)token;
}
__device__ __forceinline__ float logit_of(uint64_t key)
{
    const uint32_t order = (uint32_t)(key >> 32);
    return __uint_as_float(order ^ (order & 0x80000000u ? 0x80000000u : ~0u));
}
__device__ __forceinline__ int token_of(uint64_t key) { return (int)~(uint32_t)key; }

// What a wave's lanes put into LDS is there for the others.
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ uint64_t lane_key(uint64_t key, int lane)
{
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(key >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)key, lane);
}

__device__ __forceinline__ int lanes_below(uint64_t mask)
{
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// The `top` largest of buf[0 .. n), in descending order at its begin; returns how
// many. Whole waves. As long as there are many: those that are at least the top-th
// of the lanes' largest stay (the lanes below it lose all of theirs, half and more).
__device__ __forceinline__ int keep_top(uint64_t* buf, int n, int top)
{
    const int lane = threadIdx.x % 64;
    wave_sync();
    while (n > 128) {
        uint64_t mine[kCap / 64], best = 0;
#pragma unroll
        for (int j = 0; j < kCap / 64; ++j) {
            mine[j] = 64 * j + lane < n ? buf[64 * j + lane] : 0;
            best = mine[j] > best ? mine[j] : best;
        }
        int rank = 0;
        for (int l = 0; l < 64; ++l) {
            rank += lane_key(best, l) > best;
        }
        const uint64_t least = lane_key(best, __builtin_ctzll(__ballot(rank == top - 1)));
        wave_sync();
        n = 0;
#pragma unroll
        for (int j = 0; j < kCap / 64; ++j) {
            const bool stays = mine[j] >= least;
            const uint64_t mask = __ballot(stays);
            if (stays) {
                buf[n + lanes_below(mask)] = mine[j];
            }
            n += __popcll(mask);
        }
        wave_sync();
    }
    const uint64_t a = lane < n ? buf[lane] : 0, b = 64 + lane < n ? buf[64 + lane] : 0;
    int rank_a = 0, rank_b = 0;
    for (int i = 0; i < n; ++i) {
        const uint64_t other = buf[i];
        rank_a += other > a;
        rank_b += other > b;
    }
    wave_sync();
    if (lane < n && rank_a < top) {
        buf[rank_a] = a;
    }
    if (64 + lane < n && rank_b < top) {
        buf[rank_b] = b;
    }
    wave_sync();
    return min(n, top);
}

struct Stats {
    float r, s, t;
};

template <typename T>
__device__ __forceinline__ Stats join(const Stats& a, const Stats& b)
{
    typedef Reference<T> Ref;
    const float r = fmaxf(a.r, b.r);
    Stats j{r, 0.0f, 0.0f};
    for (const Stats& x : {a, b}) {
        if (x.s != 0.0f) {                         // (NaN: joins)
            const float d = Ref::step(x.r, r), f = exp2f(d);
            j.s += x.s * f;
            j.t += f != 0.0f ? f * __builtin_fmaf(d, x.s, x.t) : 0.0f;
        }
    }
    return j;
}

// What a workgroup writes of a whole row.
template <typename T>
__device__ __forceinline__ void write_row(const LogProbsKern& p, int64_t row, const Stats& w, const uint64_t* best)
{
    typedef Reference<T> Ref;
    const int tid = threadIdx.x;
    const float nan = __uint_as_float(0x7fc00000u);
    const bool bad = !(w.s < std::numeric_limits<float>::infinity()), none = w.s == 0.0f;
    const auto log_p = [&](float x) { return bad ? nan : none ? kNone : Ref::log_p(x, w.r, w.s); };
    if (tid < p.top) {
        const uint64_t key = best[tid];
        p.top_tokens[row * p.ld_top_tokens + tid] = bad ? -1 : token_of(key);
        p.top_log_probs[row * p.ld_top_log_probs + tid] = log_p(logit_of(key));
    }
    if (tid == 0) {
        p.entropy[row] = bad ? nan : none ? 0.0f : fmaxf((log2f(w.s) - w.t / w.s) * kLn2, 0.0f);
    }
    const T* x = static_cast<const T*>(p.x) + row * p.ld_x;
    for (int i = tid; i < p.per_row; i += 256) {
        const int token = p.tokens[row * p.ld_tokens + i];
        const float lp = token < 0 ? 0.0f : token < p.vocab ? log_p((float)x[token]) : nan;
        p.log_probs[row * p.ld_log_probs + i] = lp;
    }
}

// The waves' stats and keys (each wave's at buf + kCap wave, `n` of them) as a
// workgroup's: in every thread, and in s_best.
template <typename T>
__device__ __forceinline__ Stats join_waves(const Stats& mine, int n, int top, uint64_t* bufs, uint64_t* s_best,
                                            Stats* s_stats, int* s_n)
{
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    if (lane == 0) {
        s_stats[wave] = mine;
        s_n[wave] = n;
    }
    __syncthreads();
    if (top > 0 && wave == 0) {
        // key i of wave w is slot 32 w + i
        uint64_t key[2];
        int rank[2] = {0, 0};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int w = 2 * h + lane / 32, i = lane % 32;
            key[h] = i < s_n[w] ? bufs[w * kCap + i] : 0;
        }
        for (int l = 0; l < 64; ++l) {
            const uint64_t a = lane_key(key[0], l), b = lane_key(key[1], l);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                rank[h] += (a > key[h]) + (b > key[h]);
            }
        }
        // (absent ones come last: there are `top` others, but in rows that are not finite)
        if (lane < top) {
            s_best[lane] = 0;
        }
        wave_sync();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (key[h] != 0 && rank[h] < top) {
                s_best[rank[h]] = key[h];
            }
        }
    }
    Stats w = join<T>(join<T>(s_stats[0], s_stats[1]), join<T>(s_stats[2], s_stats[3]));
    __syncthreads();
    return w;
}

template <typename T, bool kTop>
__global__ __launch_bounds__(256) void log_probs(const LogProbsKern p)
{
    typedef Reference<T> Ref;
    __shared__ uint64_t s_buf[kTop ? 4 * kCap : 1];
    __shared__ uint64_t s_best[kMostTop];
    __shared__ Stats s_stats[4];
    __shared__ int s_n[4];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int64_t row = blockIdx.x / (uint32_t)p.splits;
    const int split = (int)(blockIdx.x - (uint32_t)row * p.splits);
    const T* x = static_cast<const T*>(p.x) + row * p.ld_x;
    const int begin = split * p.part, end = (int)min((int64_t)begin + p.part, (int64_t)p.vocab);
    uint64_t* buf = s_buf + (kTop ? wave * kCap : 0);
    int n = 0;
    bool full = false;                             // at least top keys above the threshold, or at it
    float least = kNone;
    float m = Ref::kLeast, r = Ref::of(m), s = 0.0f, t = 0.0f;

    const auto load = [&](int at, T (&v)[8]) {
        const int i = at + 8 * lane;
        if (at + kTile <= end) {
            __builtin_memcpy(v, x + i, sizeof v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = i + e < end ? x[i + e] : (T)kNone;
            }
        }
    };
    const auto take = [&](int at, const T (&raw)[8]) {
        float v[8], high = kNone;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = (float)raw[e];
            high = fmaxf(high, v[e]);
        }
        if (__any(high > m)) {
            float top = high;
#pragma unroll
            for (int i = 1; i < 64; i *= 2) {
                top = fmaxf(top, __shfl_xor(top, i));
            }
            m = top;
            const float old = r;
            r = Ref::of(m);
            const float d = fmaxf(Ref::step(old, r), -1e30f), f = exp2f(d);   // (s and t are 0 at first)
            t = f * __builtin_fmaf(d, s, t);
            s *= f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float y = Ref::y(v[e], r), w = __builtin_amdgcn_exp2f(y);
            s += w;
            t = __builtin_fmaf(w, fmaxf(y, -256.0f), t);   // (0 times -inf)
        }
        if constexpr (kTop) {
            if (full && !__any(high > least)) {
                return;
            }
            if (n + kTile > kCap) {
                n = keep_top(buf, n, p.top);
                least = logit_of(buf[p.top - 1]);
            }
            bool equal = false;
            if (!full && at + kTile <= end) {
                // the top-th of the lanes' largest: as many are at least that
                int rank = 0;
                for (int l = 0; l < 64; ++l) {
                    const float other = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(high), l));
                    rank += other > high || (other == high && l < lane);
                }
                const int at_lane = __builtin_ctzll(__ballot(rank == p.top - 1));
                least = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(high), at_lane));
                equal = true;
                full = true;
            }
            const bool all = !full;                // (less than a tile: it is the wave's last)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int token = at + 8 * lane + e;
                const bool in = token < end && (all || v[e] > least || (equal && v[e] == least));
                const uint64_t mask = __ballot(in);
                if (in) {
                    buf[n + lanes_below(mask)] = key_of(v[e], token);
                }
                n += __popcll(mask);
            }
        }
    };
    int at = begin + kTile * wave;
    if (at < end) {
        T v[3][8];
        load(at, v[0]);
        if (at + 4 * kTile < end) {
            load(at + 4 * kTile, v[1]);
        }
        for (; at < end; at += 12 * kTile) {
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                if (at + 4 * kTile * i < end) {
                    if (at + 4 * kTile * (i + 2) < end) {
                        load(at + 4 * kTile * (i + 2), v[(i + 2) % 3]);
                    }
                    take(at + 4 * kTile * i, v[i]);
                }
            }
        }
    }
    if constexpr (kTop) {
        n = keep_top(buf, n, p.top);
    }
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
        s += __shfl_xor(s, i);
        t += __shfl_xor(t, i);
    }
    const Stats w = join_waves<T>(Stats{r, s, t}, n, kTop ? p.top : 0, s_buf, s_best, s_stats, s_n);
    if (p.splits == 1) {
        write_row<T>(p, row, w, s_best);
        return;
    }
    if (threadIdx.x == 0) {
        float* to = p.stats + 3 * (int64_t)blockIdx.x;
        to[0] = w.r;
        to[1] = w.s;
        to[2] = w.t;
    }
    if (kTop && (int)threadIdx.x < p.top) {
        p.keys[(int64_t)blockIdx.x * p.top + threadIdx.x] = s_best[threadIdx.x];
    }
}

// The splits of a row: at most 64, whose keys fit the waves' room.
template <typename T>
__global__ __launch_bounds__(256) void log_probs_join(const LogProbsKern p)
{
    __shared__ uint64_t s_buf[4 * kCap];
    __shared__ uint64_t s_best[kMostTop];
    __shared__ Stats s_stats[4];
    __shared__ int s_n[4];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int64_t row = blockIdx.x;
    Stats mine{Reference<T>::kLeast, 0.0f, 0.0f};
    mine.r = Reference<T>::of(mine.r);
    if (wave == 0 && lane < p.splits) {
        const float* from = p.stats + 3 * (row * p.splits + lane);
        mine = Stats{from[0], from[1], from[2]};
    }
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
        mine = join<T>(mine, Stats{__shfl_xor(mine.r, i), __shfl_xor(mine.s, i), __shfl_xor(mine.t, i)});
    }
    uint64_t* buf = s_buf + wave * kCap;
    int n = 0;
    if (p.top > 0) {
        const int all = p.splits * p.top, share = (all + 3) / 4;   // at most 512
        const uint64_t* keys = p.keys + row * all;
        const int first = wave * share, mine_n = max(min(share, all - first), 0);
        for (int i = 0; i < mine_n; i += 64) {     // (a split of fewer than top logits has 0 behind them)
            const uint64_t key = i + lane < mine_n ? keys[first + i + lane] : 0;
            const uint64_t mask = __ballot(key != 0);
            if (key != 0) {
                buf[n + lanes_below(mask)] = key;
            }
            n += __popcll(mask);
        }
        n = keep_top(buf, n, p.top);
    }
    write_row<T>(p, row, join_waves<T>(mine, n, p.top, s_buf, s_best, s_stats, s_n), s_best);
}

struct LogProbsPlan {
    int32_t splits, part;
    size_t stats, workspace;
};

// Splits of a row: as many workgroups as the chip holds, each with 2048 logits (a
// tile for each wave) or more.
LogProbsPlan log_probs_plan(const NnopsTokenLogProbsArgs* g)
{
    LogProbsPlan a{};
    const int64_t most = (g->vocab + 4 * kTile - 1) / (4 * kTile);
    int64_t splits = (1024 + g->rows - 1) / g->rows;
    splits = splits < most ? splits : most;
    splits = splits < kMostSplits ? splits : kMostSplits;
    const int64_t part = ((g->vocab + splits - 1) / splits + 4 * kTile - 1) / (4 * kTile) * (4 * kTile);
    a.part = (int32_t)(part < INT32_MAX ? part : INT32_MAX);
    a.splits = (int32_t)((g->vocab + part - 1) / part);
    if (a.splits > 1) {
        a.stats = ((size_t)12 * g->rows * a.splits + 15) / 16 * 16;
        a.workspace = a.stats + (size_t)8 * g->rows * a.splits * g->top;
    }
    return a;
}

int check_log_probs(const NnopsTokenLogProbsArgs* g)
{
    if (g == nullptr || g->rows < 0 || g->vocab < 0 || g->per_row < 0 || g->top < 0 || g->top > g->vocab) {
        return NNOPS_INVALID_ARGUMENT;
    }
    if (g->top > kMostTop) {
        return NNOPS_UNSUPPORTED;
    }
    if (g->rows == 0) {
        return NNOPS_OK;
    }
    if (g->vocab == 0) {
        return NNOPS_INVALID_ARGUMENT;
    }
    if (g->rows > (1 << 22) || g->vocab > INT32_MAX / 2 || g->per_row > INT32_MAX / 2) {
        return NNOPS_UNSUPPORTED;
    }
    return -1;
}

template <typename T>
void launch_log_probs(const LogProbsKern& k, int64_t rows, hipStream_t s)
{
    const dim3 grid((unsigned)(rows * k.splits));
    if (k.top > 0) {
        NNOPS_LAUNCH((log_probs<T, true>), grid, dim3(256), 0, s, k);
    } else {
        NNOPS_LAUNCH((log_probs<T, false>), grid, dim3(256), 0, s, k);
    }
    if (k.splits > 1) {
        NNOPS_LAUNCH(log_probs_join<T>, dim3((unsigned)rows), dim3(256), 0, s, k);
    }
}

}  // namespace
}  // namespace nnops_amd

using namespace nnops_amd;

extern "C" size_t nnops_hip_token_log_probs_workspace_size(const NnopsTokenLogProbsArgs* g)
{
    return check_log_probs(g) >= 0 ? 0 : log_probs_plan(g).workspace;
}

extern "C" int nnops_hip_token_log_probs(const NnopsTokenLogProbsArgs* g, void* workspace, size_t workspace_bytes,
                                         void* stream)
{
    const TimingDisarm disarm;
    if (const int rc = check_log_probs(g); rc >= 0) {
        return rc;
    }
    if (g->logits == nullptr || g->ld_logits < g->vocab || g->entropy == nullptr ||
        (g->per_row > 0 && (g->tokens == nullptr || g->log_probs == nullptr || g->ld_tokens < g->per_row ||
                            g->ld_log_probs < g->per_row)) ||
        (g->top > 0 && (g->top_tokens == nullptr || g->top_log_probs == nullptr || g->ld_top_tokens < g->top ||
                        g->ld_top_log_probs < g->top))) {
        return NNOPS_INVALID_ARGUMENT;
    }
    const LogProbsPlan a = log_probs_plan(g);
    if (a.workspace > 0 && (workspace == nullptr || workspace_bytes < a.workspace || (uintptr_t)workspace % 16 != 0)) {
        return NNOPS_NOT_INITIALIZED;
    }
    LogProbsKern k{};
    k.x = g->logits;
    k.tokens = g->tokens;
    k.log_probs = g->log_probs;
    k.entropy = g->entropy;
    k.top_tokens = g->top_tokens;
    k.top_log_probs = g->top_log_probs;
    k.ld_x = g->ld_logits;
    k.ld_tokens = g->ld_tokens;
    k.ld_log_probs = g->ld_log_probs;
    k.ld_top_tokens = g->ld_top_tokens;
    k.ld_top_log_probs = g->ld_top_log_probs;
    k.vocab = (int32_t)g->vocab;
    k.per_row = (int32_t)g->per_row;
    k.top = g->top;
    k.splits = a.splits;
    k.part = a.part;
    k.stats = static_cast<float*>(workspace);
    k.keys = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + a.stats);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (g->f16) {
        launch_log_probs<_Float16>(k, g->rows, s);
    } else {
        launch_log_probs<float>(k, g->rows, s);
    }
    return hipGetLastError() == hipSuccess ? NNOPS_OK : NNOPS_INTERNAL;
}
