// Log probabilities of given tokens, the entropy and the most probable tokens of
// rows of logits, in one pass over them.
//
// A workgroup holds a row, or a part of a long one, in its registers (up to 64
// logits a thread, all of its loads in flight at once): the maximum first, then
// with a reference r and y_j = (x_j - r) log2(e)
//   s = sum 2^y_j,  t = sum y_j 2^y_j
//   log p_j = ln 2 (y_j - log2 s),  entropy = ln 2 (log2 s - t / s)
// A part's s and t are brought to another's reference by d, the y of its own: s' =
// 2^d s, t' = 2^d (t + d s). f16 rows: y = fma(x, log2(e), -R), R = r log2(e) rounded: one
// instruction, and what R's rounding brings in is the same for all y: the entropy has it
// in both terms, log p = (x - r) - (ln s - ln 2 (r log2(e) - R)), where x - r is nearly exact.
// f32 rows: (x - r) log2(e), which masks of the type's lowest value do not take out of
// f32's range.
//
// The most probable: the top-th largest of the maxima of 64 groups of 8 lanes is a
// logit that at least `top` reach, and few more do (of random ones 64 ln(64 / (64 -
// top)): 24 for 20, 44 for 32): those go into LDS as keys of 64 bits, the logit's bits
// in an order that whole numbers have, then the token's complement, so that no two
// are equal, and each counts the keys above it.
//
// Bound: HBM, the logits read once; few rows, the chain of a part and its join. f16,
// 4096 x 32000, 5 alternatives 53 to 54 us, 4.9 TB/s (none 46.6; 32 60.7); f32 88 us, 5.9
// TB/s; 64 x 151000, 20 alternatives 15.5 us; 1 x 131072, 8 alternatives 7.7 to 8.5 (two
// launches).
// A wave that read on and on, with a running maximum and a list of candidates, took
// 174 us for the first of these: a list is thinned where nothing else is in flight.
#include <limits>

#include "common.hpp"
#include "key_rooms.hpp"

namespace nnops_amd {
namespace {

constexpr int kThreads = 512;
constexpr int kSpan = 8 * kThreads; // logits that the threads have side by side, 8 each
constexpr int kMostChunks = 8;      // of those a part
constexpr int kWaves = kThreads / 64;
constexpr int kGroups = kThreads / 16;
constexpr int kMostTop = 32;
constexpr int kMostSplits = 64;
constexpr int kRoom = 2048;         // keys above a threshold, as many of each wave ...
constexpr int kAllKeys = kRoom + kSpan;   // ... and those of a span that are equal to it
constexpr int kWaveRoom = kRoom / kWaves;
static_assert(2 * kRoom <= kAllKeys && kWaveRoom <= kThreads);   // (the waves' rooms, behind the keys of all; a thread each)
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
    uint64_t* keys;       //   keys of [rows][splits][top], 0 where a split has fewer
};

// y against a reference (`base`: what its part of y is made of), y of an old one, log p.
template <typename T>
struct Reference;
template <>
struct Reference<_Float16> {
    static constexpr float kLeast = -1e38f;        // (its product is finite)
    static __device__ __forceinline__ float base(float r) { return __fmul_rn(r, kLog2e); }
    static __device__ __forceinline__ float y(float x, float base) { return __builtin_fmaf(x, kLog2e, -base); }
    static __device__ __forceinline__ float step(float old, float r) { return base(old) - base(r); }
    static __device__ __forceinline__ float log_p(float x, float r, float s)
    {
        return (x - r) - (logf(s) - y(r, base(r)) * kLn2);
    }
};
template <>
struct Reference<float> {
    static constexpr float kLeast = -std::numeric_limits<float>::max();
    static __device__ __forceinline__ float base(float r) { return r; }
    static __device__ __forceinline__ float y(float x, float base) { return (x - base) * kLog2e; }
    static __device__ __forceinline__ float step(float old, float r) { return (old - r) * kLog2e; }
    static __device__ __forceinline__ float log_p(float x, float r, float s) { return (x - r) - logf(s); }
};

// A lane's value from elsewhere in its 16: step 0 to 3 of a reduction over them.
template <int kStep>
__device__ __forceinline__ uint32_t from_row(uint32_t v)
{
#if __HIP_DEVICE_COMPILE__
    constexpr int kCtrl = kStep == 0 ? 0xb1 : kStep == 1 ? 0x4e : kStep == 2 ? 0x141 : 0x140;   // pairs, quads, mirrors
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, 0xf, 0xf, true);
#else
    return v;
#endif
}
template <int kStep = 0, int kSteps = 4>
__device__ __forceinline__ float row_max(float v)
{
    if constexpr (kStep < kSteps) {
        return row_max<kStep + 1, kSteps>(fmaxf(v, __uint_as_float(from_row<kStep>(__float_as_uint(v)))));
    }
    return v;
}
template <int kStep = 0>
__device__ __forceinline__ float row_sum(float v)
{
    if constexpr (kStep < 4) {
        return row_sum<kStep + 1>(v + __uint_as_float(from_row<kStep>(__float_as_uint(v))));
    }
    return v;
}
template <int kStep, int kSteps>
__device__ __forceinline__ uint32_t row_max(uint32_t v)
{
    if constexpr (kStep < kSteps) {
        return row_max<kStep + 1, kSteps>(max(v, from_row<kStep>(v)));
    }
    return v;
}
template <int kStep = 0>
__device__ __forceinline__ uint64_t row_max(uint64_t v)
{
    if constexpr (kStep < 4) {
        const uint64_t o = (uint64_t)from_row<kStep>((uint32_t)(v >> 32)) << 32 | from_row<kStep>((uint32_t)v);
        return row_max<kStep + 1>(o > v ? o : v);
    }
    return v;
}

// The largest of 8 logits; NaNs count for nothing.
__device__ __forceinline__ float max_of(const float (&v)[8])
{
    float m = fmaxf(v[0], v[1]);
#pragma unroll
    for (int e = 2; e < 8; ++e) {
        m = fmaxf(m, v[e]);
    }
    return m;
}
__device__ __forceinline__ float max_of(const _Float16 (&v)[8])
{
#if __HIP_DEVICE_COMPILE__
    uint32_t w[4], a, b;
    __builtin_memcpy(w, v, sizeof w);
    asm("v_pk_max_f16 %0, %1, %2" : "=v"(a) : "v"(w[0]), "v"(w[1]));   // (the builtin makes quiet NaNs first)
    asm("v_pk_max_f16 %0, %1, %2" : "=v"(b) : "v"(w[2]), "v"(w[3]));
    asm("v_pk_max_f16 %0, %0, %1" : "+v"(a) : "v"(b));
    _Float16 h[2];
    __builtin_memcpy(h, &a, sizeof h);
    return fmaxf((float)h[0], (float)h[1]);
#else
    return (float)v[0];
#endif
}

// A value of all lanes' largest, or sum, of those that are the same in 16 lanes.
__device__ __forceinline__ float lane_of(float v, int lane)
{
#if __HIP_DEVICE_COMPILE__
    return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), lane));
#else
    return v;
#endif
}

// Whole numbers in the order of the values.
__device__ __forceinline__ uint32_t order_of(float x)
{
    const uint32_t b = __float_as_uint(x + 0.0f);  // (-0 and 0 are equal)
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t order)
{
    return __uint_as_float(order ^ (order & 0x80000000u ? 0x80000000u : ~0u));
}

__device__ __forceinline__ uint64_t key_of(float x, int token)
{
    return (uint64_t)order_of(x) << 32 | ~(uint32_t)token;
}
__device__ __forceinline__ float logit_of(uint64_t key) { return value_of((uint32_t)(key >> 32)); }
__device__ __forceinline__ int token_of(uint64_t key) { return (int)~(uint32_t)key; }

// The top-th largest of the lanes' numbers, bit by bit down to `last`: the largest
// that as many reach.
template <int kLast>
__device__ __forceinline__ uint32_t top_of_lanes(uint32_t mine, int top)
{
    uint32_t least = 0;
#pragma unroll
    for (int bit = 31; bit >= kLast; --bit) {
        const uint32_t more = least | 1u << bit;
        least = __popcll(__ballot(mine >= more)) >= top ? more : least;
    }
    return least;
}

// Of their values. (f16 values as f32 end in 13 zeros, which order_of turns into ones
// below 0.)
template <typename T>
__device__ __forceinline__ float top_value(float v, int top)
{
    constexpr int kLast = sizeof(T) == 2 ? 13 : 0;
    uint32_t least = top_of_lanes<kLast>(order_of(v), top);
    if (kLast > 0 && (least & 0x80000000u) == 0) {
        least |= (1u << kLast) - 1;
    }
    return value_of(least);
}

// The top-th largest of the groups' keys.
__device__ __forceinline__ uint64_t top_of(const uint64_t (&group)[kGroups], int top)
{
    const int mine = threadIdx.x % kGroups;
    const uint64_t v = group[mine];
    int rank = 0;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        rank += group[i] > v || (group[i] == v && i < mine);
    }
    const int lane = __builtin_ctzll(__ballot(rank == top - 1));
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

template <int kKeys>
struct Shared {
    uint64_t key[kKeys];
    uint64_t key_group[kGroups];
    float group[2 * kGroups], s[kGroups], t[kGroups];
    uint32_t order_group[2 * kGroups];
    int count[kWaves];
    int keys, left;
};

// Of sh.key[0 .. n): one of this thread's and how many are above it; a thread without
// any has 0 and its own number. More keys than threads are thinned first: those that
// reach the top-th of the groups' largest stay, which is a single one of its group (of
// 16 and more; keys of 0 all go). Then once by their logits alone. Every thread calls
// it.
template <int kKeys>
__device__ __forceinline__ uint64_t rank_keys(Shared<kKeys>& sh, int n, int top, int& rank)
{
    const int tid = threadIdx.x;
    while (n > kThreads) {
        uint64_t best = 0;
        for (int i = tid; i < n; i += kThreads) {
            best = sh.key[i] > best ? sh.key[i] : best;
        }
        best = row_max(best);
        if (tid % 16 == 0) {
            sh.key_group[tid / 16] = best;
        }
        if (tid == 0) {
            sh.left = 0;
        }
        __syncthreads();
        uint64_t least = top_of(sh.key_group, top);
        least = least > 0 ? least : 1;             // (what is 0 is no key)
        for (int i = 0; i < n; i += kThreads) {
            const uint64_t mine = i + tid < n ? sh.key[i + tid] : 0;
            __syncthreads();                       // (what stays goes over keys that were looked at)
            if (mine >= least) {
                sh.key[atomicAdd(&sh.left, 1)] = mine;
            }
        }
        __syncthreads();
        n = sh.left;
        __syncthreads();
    }
    if (n > 64) {
        const uint64_t mine = tid < n ? sh.key[tid] : 0;
        const uint32_t order = (uint32_t)(mine >> 32), best = row_max<0, 3>(order);
        if (tid % 8 == 0) {
            sh.order_group[tid / 8] = best;
        }
        if (tid == 0) {
            sh.left = 0;
        }
        __syncthreads();
        const uint32_t least = top_of_lanes<0>(sh.order_group[tid % 64], top);
        if (tid < n && order >= least) {
            sh.key[atomicAdd(&sh.left, 1)] = mine;
        }
        __syncthreads();
        n = sh.left;
    }
    const uint64_t key = tid < n ? sh.key[tid] : 0;
    rank = 0;
    if (tid < n) {
#pragma unroll 8
        for (int i = 0; i < n; ++i) {
            rank += sh.key[i] > key;
        }
    } else {
        rank = tid;                                // (behind the last key: nothing)
    }
    return key;
}

struct Stats {
    float r, s, t;
};

// Another reference's s and t, added.
template <typename T>
__device__ __forceinline__ void join(Stats& a, const Stats& x)
{
    if (x.s != 0.0f) {                             // (NaN: joins)
        const float d = Reference<T>::step(x.r, a.r), f = exp2f(d);
        a.s += x.s * f;
        a.t += f != 0.0f ? f * __builtin_fmaf(d, x.s, x.t) : 0.0f;
    }
}

// A given token of a row, and its logit: asked for before the row is looked at.
template <typename T>
struct Given {
    int token;
    T logit;
};
template <typename T>
__device__ __forceinline__ Given<T> given(const LogProbsKern& p, int64_t row, int i)
{
    Given<T> g{-1, (T)0.0f};
    if (i < p.per_row) {
        g.token = p.tokens[row * p.ld_tokens + i];
        if ((uint32_t)g.token < (uint32_t)p.vocab) {
            g.logit = static_cast<const T*>(p.x)[row * p.ld_x + g.token];
        }
    }
    return g;
}

// What `threads` threads write of a whole row: each its key, where it is among the top,
// and given tokens (from the last thread on: the first have keys).
template <typename T>
__device__ __forceinline__ void write_row(const LogProbsKern& p, int64_t row, const Stats& w, uint64_t key, int rank,
                                          Given<T> g, int threads)
{
    typedef Reference<T> Ref;
    const int tid = threadIdx.x % (uint32_t)threads;
    const float nan = __uint_as_float(0x7fc00000u);
    const bool bad = !(w.s < std::numeric_limits<float>::infinity()), none = w.s == 0.0f;
    const auto log_p = [&](float x) { return bad ? nan : none ? kNone : Ref::log_p(x, w.r, w.s); };
    const int to = bad ? tid : rank;
    if (to < p.top) {
        p.top_tokens[row * p.ld_top_tokens + to] = bad ? -1 : token_of(key);
        p.top_log_probs[row * p.ld_top_log_probs + to] = log_p(logit_of(key));
    }
    if (tid == threads - 1) {
        p.entropy[row] = bad ? nan : none ? 0.0f : fmaxf((log2f(w.s) - w.t / w.s) * kLn2, 0.0f);
    }
    for (int i = threads - 1 - tid; i < p.per_row;) {
        p.log_probs[row * p.ld_log_probs + i] = g.token < 0 ? 0.0f : g.token < p.vocab ? log_p((float)g.logit) : nan;
        i += threads;
        g = given<T>(p, row, i);
    }
}

// The keys of a part x[0 .. n) whose logits reach `least` in more places than there is
// room for (equal ones: masks; a few groups that have nearly all that is large), read
// again: how many there are. At least the `top` largest are among them. Every thread
// calls it.
template <typename T>
__device__ __forceinline__ int many_keys(Shared<kAllKeys>& sh, const T* x, int begin, int n, float least, int top)
{
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid == 0) {
        sh.keys = 0;
    }
    __syncthreads();
    for (int at = tid; at < n; at += kThreads) {
        const float v = (float)x[at];
        if (v > least) {
            const int to = atomicAdd(&sh.keys, 1);
            if (to < kRoom) {
                sh.key[to] = key_of(v, begin + at);
            }
        }
    }
    __syncthreads();
    int keys = sh.keys;
    __syncthreads();
    if (keys <= kRoom) {
        // the equal ones in order, until there are enough
        for (int j = 0; j < n && keys < top; j += kSpan) {
            for (int at = j + tid; at < min(j + kSpan, n); at += kThreads) {
                const float v = (float)x[at];
                if (v == least) {
                    sh.key[atomicAdd(&sh.keys, 1)] = key_of(v, begin + at);
                }
            }
            __syncthreads();
            keys = sh.keys;
            __syncthreads();
        }
        return keys;
    }
    // one after another
    uint64_t above = ~0ull;
    for (int i = 0; i < top; ++i) {
        uint64_t next = 0;
        for (int at = tid; at < n; at += kThreads) {
            const uint64_t k = key_of((float)x[at], begin + at);
            next = k < above && k > next ? k : next;
        }
        next = row_max(next);
        if (tid % 16 == 0) {
            sh.key_group[tid / 16] = next;
        }
        __syncthreads();
        above = top_of(sh.key_group, 1);
        if (tid == 0) {
            sh.key[i] = above;
        }
        __syncthreads();
    }
    return top;
}

template <typename T, int kChunks, bool kTop>
__global__ __launch_bounds__(kThreads, 4) void log_probs(const LogProbsKern p)
{
    typedef Reference<T> Ref;
    __shared__ Shared<kTop ? kAllKeys : 1> sh;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x / (uint32_t)p.splits;
    const int split = (int)(blockIdx.x - (uint32_t)row * p.splits);
    const int begin = split * p.part, n = min(p.part, p.vocab - begin);
    const T* x = static_cast<const T*>(p.x) + row * p.ld_x + begin;
    const Given<T> g = p.splits == 1 ? given<T>(p, row, kThreads - 1 - tid) : Given<T>{};
    T v[kChunks][8];
    float high[kChunks], best = kNone;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        const int at = j * kSpan + 8 * tid;
        if (j * kSpan + kSpan <= n) {
            __builtin_memcpy(v[j], x + at, sizeof v[j]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[j][e] = (T)kNone;
            }
            if (at + 8 <= n) {
                __builtin_memcpy(v[j], x + at, sizeof v[j]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (at + e < n) {
                        v[j][e] = x[at + e];
                    }
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        high[j] = max_of(v[j]);
        best = fmaxf(best, high[j]);
    }
    best = row_max<0, 3>(best);
    if (tid % 8 == 0) {
        sh.group[tid / 8] = best;
    }
    __syncthreads();
    const float group = sh.group[tid % 64], high_row = row_max(group);
    const float m = fmaxf(fmaxf(lane_of(high_row, 0), lane_of(high_row, 16)),
                          fmaxf(lane_of(high_row, 32), lane_of(high_row, 48)));
    const float r = fmaxf(m, Ref::kLeast), y_base = Ref::base(r);
    // (each phase converts f16 logits anew: kept as f32 they would take the registers of
    // another workgroup)
    const auto forget = [&] {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                v4i w;
                __builtin_memcpy(&w, v[j], sizeof w);
                asm volatile("" : "+v"(w));
                __builtin_memcpy(v[j], &w, sizeof w);
            }
        }
    };
    forget();
    float least = kNone;
    if constexpr (kTop) {
        // (the top-th of the maxima of 64 groups of 8 lanes)
        least = top_value<T>(group, p.top);
        const T reach = (T)least;                  // (one of the logits: exact)
        uint64_t* const room = sh.key + kRoom + tid / 64 * kWaveRoom;
        int count = least > kNone ? 0 : kRoom;     // (-inf: what is behind the row reaches it too)
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            if (j * kSpan < n && least > kNone && __any(high[j] >= least)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool in = v[j][e] >= reach;
                    const uint64_t mask = __ballot(in);
                    if (mask != 0) {
                        const int to = count + (int)__builtin_amdgcn_mbcnt_hi(
                                                   (uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
                        if (in && to < kWaveRoom) {
                            room[to] = key_of((float)v[j][e], begin + j * kSpan + 8 * tid + e);
                        }
                        count += __popcll(mask);
                    }
                }
            }
        }
        if (tid % 64 == 0) {
            sh.count[tid / 64] = count;
        }
    }
    forget();
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        if (j * kSpan < n) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = Ref::y((float)v[j][e], y_base), w = __builtin_amdgcn_exp2f(y);
                s += w;
                t = __builtin_fmaf(w, fmaxf(y, -256.0f), t);   // (0 times -inf)
            }
        }
    }
    s = row_sum(s);
    t = row_sum(t);
    if (tid % 16 == 0) {
        sh.s[tid / 16] = s;
        sh.t[tid / 16] = t;
    }
    __syncthreads();
    s = row_sum(sh.s[tid % kGroups]);
    t = row_sum(sh.t[tid % kGroups]);
    const Stats w{r, lane_of(s, 0) + lane_of(s, 16), lane_of(t, 0) + lane_of(t, 16)};
    uint64_t key = 0;
    int rank = tid;
    if constexpr (kTop) {
        int count[kWaves], to[kWaves];
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            count[i] = sh.count[i];
        }
        int keys = gather_rooms(count, kWaveRoom, to);
        if (keys < 0) {                            // (the same in all threads)
            keys = many_keys(sh, x, begin, n, least, p.top);
        } else {
#pragma unroll
            for (int i = 0; i < kWaves; ++i) {
                if (tid < count[i]) {
                    sh.key[to[i] + tid] = sh.key[kRoom + i * kWaveRoom + tid];
                }
            }
            __syncthreads();
        }
        key = rank_keys(sh, keys, p.top, rank);
    }
    if (p.splits == 1) {
        write_row<T>(p, row, w, key, rank, g, kThreads);
        return;
    }
    if (tid == 0) {
        float* to = p.stats + 3 * (int64_t)blockIdx.x;
        to[0] = w.r;
        to[1] = w.s;
        to[2] = w.t;
    }
    if (kTop && rank < p.top) {
        p.keys[(int64_t)blockIdx.x * p.top + rank] = key;
    }
}

// The splits of a row, at most 64: a lane each.
template <typename T>
__device__ __forceinline__ Stats join_splits(const LogProbsKern& p, int64_t row)
{
    const int lane = threadIdx.x % 64;
    Stats w{Reference<T>::kLeast, 0.0f, 0.0f};
    if (lane < p.splits) {
        const float* from = p.stats + 3 * (row * p.splits + lane);
        w = Stats{from[0], from[1], from[2]};
    }
    const float r = row_max(w.r);
    Stats sum{fmaxf(fmaxf(lane_of(r, 0), lane_of(r, 16)), fmaxf(lane_of(r, 32), lane_of(r, 48))), 0.0f, 0.0f};
    join<T>(sum, w);
    const float s = row_sum(sum.s), t = row_sum(sum.t);
    sum.s = (lane_of(s, 0) + lane_of(s, 16)) + (lane_of(s, 32) + lane_of(s, 48));
    sum.t = (lane_of(t, 0) + lane_of(t, 16)) + (lane_of(t, 32) + lane_of(t, 48));
    return sum;
}

// (Without alternatives a wave has a row, and a workgroup eight.)
template <typename T, bool kTop>
__global__ __launch_bounds__(kThreads) void log_probs_join(const LogProbsKern p, int64_t rows)
{
    const int tid = threadIdx.x;
    if constexpr (kTop) {
        __shared__ Shared<kMostSplits * kMostTop> sh;
        const int64_t row = blockIdx.x;
        const Given<T> g = given<T>(p, row, kThreads - 1 - tid);
        const int all = p.splits * p.top;
        for (int i = tid; i < all; i += kThreads) {
            sh.key[i] = p.keys[row * all + i];
        }
        const Stats sum = join_splits<T>(p, row);
        __syncthreads();
        int rank;
        const uint64_t key = rank_keys(sh, all, p.top, rank);
        // (a row that is not bad has `top` keys that are not 0)
        write_row<T>(p, row, sum, key, key != 0 ? rank : kMostTop, g, kThreads);
    } else {
        const int64_t row = (int64_t)blockIdx.x * kWaves + tid / 64;
        if (row < rows) {
            const Given<T> g = given<T>(p, row, 63 - tid % 64);
            write_row<T>(p, row, join_splits<T>(p, row), 0, kMostTop, g, 64);
        }
    }
}

struct LogProbsPlan {
    int32_t splits, part, chunks;
    size_t stats, workspace;
};

// A row that a workgroup can hold is not split (one launch; us, split / not, 10
// alternatives: 1 x 32000 8.1 / 6.5, 64 x 32000 8.1 / 6.7, 200 x 32000 10.8 / 7.6). Longer
// ones: the largest parts that leave 256 workgroups (that / 512 / 1024: 1 x 131072 8.4
// / 8.2 / 8.2, 64 x 151000 13.3 / 14.0 / 15.0, 128 x 131072 14.8 / 14.9 / 16.8, 300 x
// 131072 22.1 / 22.1 / 22.0).
LogProbsPlan log_probs_plan(const NnopsTokenLogProbsArgs* g)
{
    LogProbsPlan a{};
    const auto parts = [&](int64_t chunks) { return (g->vocab + chunks * kSpan - 1) / (chunks * kSpan); };
    a.chunks = kMostChunks;
    while (a.chunks > 1 && (parts(a.chunks) == 1 ? parts(a.chunks / 2) == 1
                                                 : parts(a.chunks / 2) <= kMostSplits && g->rows * parts(a.chunks) < 256)) {
        a.chunks /= 2;
    }
    const int64_t splits = parts(a.chunks), part = ((g->vocab + splits - 1) / splits + 7) / 8 * 8;
    a.part = (int32_t)part;
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
    if (g->rows > (1 << 22) || g->vocab > (int64_t)kMostSplits * kMostChunks * kSpan || g->per_row > INT32_MAX / 2) {
        return NNOPS_UNSUPPORTED;
    }
    // (threads of a launch: fewer than 2^32)
    return g->rows * log_probs_plan(g).splits < (int64_t)1 << 23 ? -1 : NNOPS_UNSUPPORTED;
}

template <typename T, int kChunks>
void launch_chunks(const LogProbsKern& k, int64_t rows, hipStream_t s)
{
    const dim3 grid((unsigned)(rows * k.splits));
    if (k.top > 0) {
        NNOPS_LAUNCH((log_probs<T, kChunks, true>), grid, dim3(kThreads), 0, s, k);
    } else {
        NNOPS_LAUNCH((log_probs<T, kChunks, false>), grid, dim3(kThreads), 0, s, k);
    }
}

template <typename T>
void launch_log_probs(const LogProbsKern& k, int chunks, int64_t rows, hipStream_t s)
{
    chunks == 1   ? launch_chunks<T, 1>(k, rows, s)
    : chunks == 2 ? launch_chunks<T, 2>(k, rows, s)
    : chunks == 4 ? launch_chunks<T, 4>(k, rows, s)
                  : launch_chunks<T, 8>(k, rows, s);
    if (k.splits > 1) {
        if (k.top > 0) {
            NNOPS_LAUNCH((log_probs_join<T, true>), dim3((unsigned)rows), dim3(kThreads), 0, s, k, rows);
        } else {
            const unsigned blocks = (unsigned)((rows + kWaves - 1) / kWaves);
            NNOPS_LAUNCH((log_probs_join<T, false>), dim3(blocks), dim3(kThreads), 0, s, k, rows);
        }
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
        launch_log_probs<_Float16>(k, a.chunks, g->rows, s);
    } else {
        launch_log_probs<float>(k, a.chunks, g->rows, s);
    }
    return hipGetLastError() == hipSuccess ? NNOPS_OK : NNOPS_INTERNAL;
}
