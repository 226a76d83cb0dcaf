// Causal attention over the paged 8-bit cache, with an optional sliding window
// and first tokens that stay visible.
//
// Rows: the query heads that share a KV head attend to the same codes, so a
// tile's rows are (token, head of the group), row = token * group + head. A
// wave has 16 rows and walks tiles of 64 tokens:
//   S^T[64 x 16] = K Q^T      v_mfma_f32_16x16x32_f16, K's codes as f16 (exact)
//   online softmax over S^T   a lane holds 16 tokens of one row
//   O^T[d x 16] += V^T P^T    P straight from the registers of S^T
// Nothing crosses LDS until the end: which token a matrix row stands for is
// free, so row m of score tile t is token 16 (m / 4) + 4 t + m % 4, and a lane
// of group g = lane / 16 then holds tokens 16 g .. 16 g + 15: the very 16 bytes
// that it loads of a channel's tokens (values lie with a channel's tokens side
// by side). Likewise a lane's 16-byte piece of a key is 8 channels of each of
// two k steps. Pages hold whole groups of 16 tokens, so a lane has one page and
// one scale on each side per tile.
//
// Scales: with ks, vs the scales of a token's page,
//   x = scale log2(e) (q . code) ks + log2(vs),  M = running max of x,
//   P = 2^(x - M + 6),  O += P code,  l += P 2^-6 / vs,  out = 2^-6 O / l:
// the value scale rides in the exponent (one fma), and P's largest weight is
// the same whatever the scales are.
//
// Bound: HBM for few rows, the codes read once per KV head. Long sequences are
// split over workgroups (partial O, M, l in the workspace, joined by a second
// kernel); a workgroup's 4 waves take every fourth tile and join in LDS. A wave
// has a tile's 16 KB (d 128) of codes in flight and 168 registers, three waves a
// SIMD. No branch stands around a tile's loads (channels past d are loaded as
// channel 0's, the last tile is peeled off): the waits after one are for
// everything (74 us for the batch below, and 42 against 35 at d 64).
// One token of each of 64 sequences of up to 4096, 32 query and 8 KV heads, d 128:
// 68.2 us, 4.55 TB/s; of one sequence of 126976: 55.9 us, 4.65 TB/s; of one of
// 777: 9.2 us, two launches and the host's 5.
#include <type_traits>

#include "cache_attention.hpp"

namespace nnops_amd {
namespace {

constexpr int kRows = 16;           // rows of a wave

template <typename T, int DP>
__global__ __launch_bounds__(256, DP > 128 ? 1 : sizeof(T) == 2 ? 3 : 2) void attention_rows16(const AttnKern p)
{
    constexpr int kC = DP / 64;                    // 64-channel pieces of a key
    constexpr int kT = DP / 16;                    // 16-channel tiles of O
    typedef Operand<T> Op;
    constexpr int kWeights = Op::kParts == 1 ? 2 : Op::kParts;   // parts of a probability
    constexpr int kPitch = DP + 4;
    __shared__ float s_o[4][kRows][kPitch];
    __shared__ float s_m[4][kRows], s_l[4][kRows];
    const Paged& c = p.c;
    const uint32_t item = blockIdx.x / (uint32_t)c.heads;
    const int kvh = (int)(blockIdx.x - item * c.heads);
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int n = lane % 16, g = lane / 16;
    const int kb = n / 4;                          // the token group of a lane's keys
    // Without a window a wave's first tile is known before the lengths are, if
    // sequences are not split or the longest fills the page table: its page numbers
    // are asked for beside them. (Past the sequence's end they may be anything; what
    // is read through them is masked.)
    const bool early = p.window == 0 && p.per_seq > 0 && c.table_pages > 0;
    int kid = 0, vid = 0;
    if (early) {
        const int32_t* row = c.table + (int64_t)(item / (uint32_t)p.per_seq) * c.ld_table;
        const int base = kTile * ((int)blockIdx.y * p.chunk + wave), last = c.table_pages - 1;
        kid = row[min((base + 16 * kb) >> c.page_log2, last)];
        vid = row[min((base + 16 * g) >> c.page_log2, last)];
    }
    RowTile rt;
    if (!find_tile(p, item, false, rt)) {
        return;
    }
    const SeqRows& seq = rt.seq;
    const Span& span = rt.span;
    const int b = rt.b, pmin = rt.pmin, pmax = rt.pmax;
    const int row0 = rt.row0, rows = rt.rows;
    const int tok_last = pmax - (seq.len - seq.n);
    const int split = blockIdx.y;
    const int v0 = split * rt.chunk;
    if (split > 0 && v0 >= span.tiles) {
        return;
    }
    const int v1 = min(span.tiles, v0 + rt.chunk);

    const int row = row0 + n;
    const bool is_row = row < rows;
    const int tok = is_row ? (int)((uint32_t)row / (uint32_t)p.group) : tok_last;
    const int head = kvh * p.group + (is_row ? row - tok * p.group : 0);
    const int pos = seq.len - seq.n + tok;
    const int d = c.d;

    // Q's fragments: channels 64 i + 16 g + 8 h .. + 7 of a row are k step 2 i + h
    typename Op::Vec qf[DP / 32][Op::kParts];
    const T* qrow = static_cast<const T*>(p.q) + (int64_t)(seq.start + tok) * p.ld_q + (int64_t)head * d;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) {
        const int at = 64 * (i / 2) + 16 * g + 8 * (i % 2);
        T x[8] = {};
        if (is_row && at < d) {
            __builtin_memcpy(x, qrow + at, sizeof x);
        }
        Op::split(x, qf[i]);
    }

    v4f o[kT];
#pragma unroll
    for (int t = 0; t < kT; ++t) {
        o[t] = v4f{0, 0, 0, 0};
    }
    float m_run = kNone, l_run = 0.0f;
    const int64_t page_bytes = (int64_t)c.page * d;
    const int ktok = 16 * kb + n % 4;              // + 4 t: its token in the tile

    // The codes of a wave's next tile are in flight while it works on this one:
    // its keys from the scores on, its values from the second product on, its
    // page numbers a tile earlier still. (Loads come back in order: page numbers
    // asked for beside the keys they lead to would wait for this tile's values.)
    const int32_t* table = c.table + (int64_t)b * c.ld_table;
    const int64_t page_step = page_bytes * c.heads;
    const int8_t* k_at = c.k + kvh * page_bytes + 16 * g;
    const int8_t* v_at = c.v + kvh * page_bytes + n * c.page;
    v4i kr[4][kC], vr[kT];
    PageScales scale_next{0.0f, 0.0f, 0.0f};
    // (a group past the last position has the last page's codes: they are masked)
    // (page numbers as they lie in the table: looked at when they are used)
    const auto ids = [&](int v) {
        const int base = tile_base(span, v);
        kid = table[min(base + 16 * kb, pmax) >> c.page_log2];
        vid = table[min(base + 16 * g, pmax) >> c.page_log2];
    };
    int koff[kC];                                  // channels past d: channel 0's codes (q is 0 there)
#pragma unroll
    for (int i = 0; i < kC; ++i) {
        koff[i] = 64 * i + 16 * g < d ? 64 * i : -16 * g;
    }
    const auto load_k = [&](int v, int page_k, int page_v) {
        const int base = tile_base(span, v);
        const int8_t* at = k_at + readable(c, page_k) * page_step + ((base + ktok) & (c.page - 1)) * d;
        int kstep = 4 * d;
        if constexpr (DP <= 128) {
            // (its multiples are computed here, not kept over the loop: 168 registers
            // instead of 256 and spills)
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("" : "+s"(kstep));
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int i = 0; i < kC; ++i) {
                kr[t][i] = *reinterpret_cast<const v4i*>(at + koff[i] + (int64_t)(t * kstep));
            }
        }
        scale_next = page_scales(c, page_v, kvh);
    };
    const auto load_v = [&](int v, int page_v) {
        const int base = tile_base(span, v);
        const int8_t* at = v_at + readable(c, page_v) * page_step + ((base + 16 * g) & (c.page - 1));
        int vstep = 16 * c.page;
        if constexpr (DP <= 128) {
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("" : "+s"(vstep));
        }
#pragma unroll
        for (int t = 0; t < kT; ++t) {
            vr[t] = *reinterpret_cast<const v4i*>(at + (int64_t)((16 * t < d ? t : 0) * vstep));
        }
    };
    // (no branch around the loads of a tile: it would wait for all of them)
    const auto tile = [&](auto go_on, int v) {
        constexpr bool more = decltype(go_on)::value;
        const int next_v = vid;                    // the next tile's page
        const int base = tile_base(span, v), vt0 = base + 16 * g;
        const PageScales scale = scale_next;

        v4f s[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            s[t] = v4f{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < kC; ++i) {
                s[t] = product<T>(Op::codes((uint32_t)kr[t][i].x, (uint32_t)kr[t][i].y), qf[2 * i], s[t]);
                s[t] = product<T>(Op::codes((uint32_t)kr[t][i].z, (uint32_t)kr[t][i].w), qf[2 * i + 1], s[t]);
            }
        }

        const Scales sc = softmax_scales(p, scale);
        if constexpr (more) {
            const int next_k = kid;
            ids(min(v + 8, v1 - 1));
            load_k(v + 4, next_k, next_v);
        }

        float x[4][4];
        float top = kNone;
        const bool open = base + kTile - 1 <= pmin && (p.window == 0 || pmax - base < p.window);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float y = __builtin_fmaf(s[t][i], sc.mul, sc.add);
                if (!open) {
                    const int at = vt0 + 4 * t + i;
                    const bool seen = at <= pos && (p.window == 0 || pos - at < p.window || at < p.sinks);
                    y = seen ? y : kNone;
                }
                x[t][i] = y;
                top = fmaxf(top, y);
            }
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        if (__any(top > m_run + kLazy)) {
            // (0 where nothing was seen before)
            const float f = top > m_run ? __builtin_amdgcn_exp2f(m_run - top) : 1.0f;
            l_run *= f;
#pragma unroll
            for (int t = 0; t < kT; ++t) {
                o[t] *= f;
            }
            m_run = fmaxf(m_run, top);
        }
        const float shift = m_run > kNone ? kLift - m_run : 0.0f;
        float sum = 0.0f, w[2][8];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[t / 2][4 * (t % 2) + i] = __builtin_amdgcn_exp2f(x[t][i] + shift);
                sum += w[t / 2][4 * (t % 2) + i];
            }
        }
        // a page of which the row sees nothing adds nothing, whatever its scale
        l_run += sum != 0.0f ? sum * sc.inv : 0.0f;
        typename Op::Vec pf[2][kWeights];
        Op::split(w[0], pf[0]);
        Op::split(w[1], pf[1]);
#pragma unroll
        for (int t = 0; t < kT; ++t) {
            o[t] = product<T>(Op::codes((uint32_t)vr[t].x, (uint32_t)vr[t].y), pf[0], o[t]);
            o[t] = product<T>(Op::codes((uint32_t)vr[t].z, (uint32_t)vr[t].w), pf[1], o[t]);
        }
        if constexpr (more) {
            load_v(v + 4, next_v);
        }
    };
    if (v0 + wave < v1) {
        int v = v0 + wave;
        if (!early || v0 != split * p.chunk) {
            ids(v);
        }
        const int first_k = kid, first_v = vid;
        ids(min(v + 4, v1 - 1));
        load_k(v, first_k, first_v);
        load_v(v, first_v);
        for (; v + 4 < v1; v += 4) {
            tile(std::true_type{}, v);
        }
        tile(std::false_type{}, v);
    }

    // the waves' parts, brought to one maximum and summed
    l_run += __shfl_xor(l_run, 16);
    l_run += __shfl_xor(l_run, 32);
    if (g == 0) {
        s_m[wave][n] = m_run;
        s_l[wave][n] = l_run;
    }
#pragma unroll
    for (int t = 0; t < kT; ++t) {
        *reinterpret_cast<v4f*>(&s_o[wave][n][16 * t + 4 * g]) = o[t];
    }
    __syncthreads();
    // 16 threads a row, 4 channels each at a time
    const int r = threadIdx.x / 16, ch0 = threadIdx.x % 16 * 4;
    if (row0 + r >= rows) {
        return;
    }
    const float m = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
    float f[4], l = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        // a wave that saw nothing has m = -inf and nothing to add
        f[w] = s_m[w][r] < m ? __builtin_amdgcn_exp2f(s_m[w][r] - m) : 1.0f;
        l += f[w] * s_l[w][r];
    }
    const int rtok = (int)((uint32_t)(row0 + r) / (uint32_t)p.group);
    const int64_t token = seq.start + rtok;
    const int qh = kvh * p.group + (row0 + r - rtok * p.group);
    const int64_t at_part = ((int64_t)split * c.rows + token) * p.q_heads + qh;
    const float scale = rt.split ? 1.0f : l == 0.0f ? 0.0f : kDrop / l;
#pragma unroll
    for (int i = 0; i < DP / 64; ++i) {
        const int ch = ch0 + 64 * i;
        if (ch >= d) {
            break;
        }
        v4f sum = v4f{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            sum += f[w] * *reinterpret_cast<const v4f*>(&s_o[w][r][ch]);
        }
        if (rt.split) {
            *reinterpret_cast<v4f*>(&p.part[at_part * d + ch]) = sum;
        } else {
            T y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[e] = (T)(sum[e] * scale);
            }
            __builtin_memcpy(static_cast<T*>(p.out) + token * p.ld_out + (int64_t)qh * d + ch, y, sizeof y);
        }
    }
    if (rt.split && ch0 == 0) {
        p.part_ml[2 * at_part] = m;
        p.part_ml[2 * at_part + 1] = l;
    }
}

// The splits of a row that have something: 0 or 1 where there is nothing to
// join (or the row is no sequence's). Whole waves call it.
__device__ __forceinline__ int splits_of(const AttnKern& p, int token, int qh)
{
    const Paged& c = p.c;
    int b;
    if (c.row_starts == nullptr) {
        b = (int)((uint32_t)token / (uint32_t)c.uniform);
    } else {
        int lo = 0, hi = c.seqs;                   // the last sequence that starts at or before the row
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            (c.row_starts[mid] <= token ? lo : hi) = mid;
        }
        b = lo;
    }
    RowTile rt;
    rt.seq = seq_rows(c, b);
    const int chunk = chunk_of(p, rt.seq);
    const int tok = token - rt.seq.start;
    if (tok < 0 || tok >= rt.seq.n) {
        return 0;
    }
    const uint32_t row = (uint32_t)(tok * p.group) + (uint32_t)qh % (uint32_t)p.group;
    place_tile(p, (int)(row / (uint32_t)p.tile_rows), chunk, rt);
    return rt.split ? (int)((uint32_t)(rt.span.tiles + chunk - 1) / (uint32_t)chunk) : 1;
}

// Joins the splits of the rows that have more than one. Few splits: 4 channels
// of a row by a lane, as many rows a wave as that gives.
constexpr int kFewSplits = 8;

__host__ __device__ __forceinline__ int join_lanes(int d) { return d <= 64 ? 16 : d <= 128 ? 32 : 64; }

template <typename T>
__global__ __launch_bounds__(256) void attention_join_few(const AttnKern p)
{
    const int lanes = join_lanes(p.c.d);
    const uint32_t i = (blockIdx.x * 256 + threadIdx.x) / (uint32_t)lanes;
    const int token = (int)(i / (uint32_t)p.q_heads), qh = (int)(i - (uint32_t)token * p.q_heads);
    const int active = splits_of(p, min(token, p.c.rows - 1), qh);
    const int d = p.c.d, ch = threadIdx.x % (uint32_t)lanes * 4;
    if (token >= p.c.rows || active <= 1 || ch >= d) {
        return;
    }
    const int64_t rows = (int64_t)p.c.rows * p.q_heads, at = (int64_t)token * p.q_heads + qh;
    float ms[kFewSplits], ls[kFewSplits], m = kNone, l = 0.0f;
    v4f os[kFewSplits], o = v4f{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < kFewSplits; ++s) {
        if (s < active) {
            ms[s] = p.part_ml[2 * (s * rows + at)];
            ls[s] = p.part_ml[2 * (s * rows + at) + 1];
            os[s] = *reinterpret_cast<const v4f*>(p.part + (s * rows + at) * d + ch);
        }
    }
#pragma unroll
    for (int s = 0; s < kFewSplits; ++s) {
        m = s < active ? fmaxf(m, ms[s]) : m;
    }
#pragma unroll
    for (int s = 0; s < kFewSplits; ++s) {
        if (s < active) {
            const float w = ms[s] < m ? __builtin_amdgcn_exp2f(ms[s] - m) : 1.0f;
            l += w * ls[s];
            o += w * os[s];
        }
    }
    const float f = l == 0.0f ? 0.0f : kDrop / l;
    T y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        y[e] = (T)(o[e] * f);
    }
    __builtin_memcpy(static_cast<T*>(p.out) + token * p.ld_out + (int64_t)qh * d + ch, y, sizeof y);
}

// Many: a workgroup per row, its weights 2^(M - max) in LDS, every 8th split by
// 32 lanes of 4 channels.
constexpr int kMostSplits = 512;

template <typename T>
__global__ __launch_bounds__(256) void attention_join(const AttnKern p)
{
    __shared__ float s_w[kMostSplits];
    __shared__ float s_red[8];
    __shared__ __attribute__((aligned(16))) float s_o[8][256];
    const Paged& c = p.c;
    const int token = (int)(blockIdx.x / (uint32_t)p.q_heads), tid = threadIdx.x;
    const int qh = (int)(blockIdx.x - (uint32_t)token * p.q_heads);
    const int active = splits_of(p, token, qh);
    if (active <= 1) {
        return;
    }
    const int d = c.d;
    const int64_t rows = (int64_t)c.rows * p.q_heads, at = (int64_t)token * p.q_heads + qh;
    float m = kNone;
    for (int s = tid; s < active; s += 256) {
        s_w[s] = p.part_ml[2 * (s * rows + at)];
        m = fmaxf(m, s_w[s]);
    }
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
        m = fmaxf(m, __shfl_xor(m, i));
    }
    if (tid % 64 == 0) {
        s_red[tid / 64] = m;
    }
    __syncthreads();
    m = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    float l = 0.0f;
    for (int s = tid; s < active; s += 256) {
        const float w = s_w[s] < m ? __builtin_amdgcn_exp2f(s_w[s] - m) : 1.0f;
        s_w[s] = w;
        l += w * p.part_ml[2 * (s * rows + at) + 1];
    }
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
        l += __shfl_xor(l, i);
    }
    if (tid % 64 == 0) {
        s_red[4 + tid / 64] = l;
    }
    __syncthreads();
    l = (s_red[4] + s_red[5]) + (s_red[6] + s_red[7]);
    const int g = tid / 32, i = tid % 32;
    v4f o[2] = {v4f{0, 0, 0, 0}, v4f{0, 0, 0, 0}};
#pragma unroll 4
    for (int s = g; s < active; s += 8) {
        const float* src = p.part + (s * rows + at) * d;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (4 * i + 128 * h < d) {
                o[h] += s_w[s] * *reinterpret_cast<const v4f*>(src + 4 * i + 128 * h);
            }
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        *reinterpret_cast<v4f*>(&s_o[g][4 * i + 128 * h]) = o[h];
    }
    __syncthreads();
    if (tid < d) {
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            sum += s_o[e][tid];
        }
        static_cast<T*>(p.out)[token * p.ld_out + (int64_t)qh * d + tid] = (T)(l == 0.0f ? 0.0f : sum * kDrop / l);
    }
}

struct AttnPlan {
    int64_t items;        // row tiles, all KV heads
    int32_t tile_rows, per_seq, chunk, splits, tiles, whole;
    bool tiled;           // attention_rows_tiled, else attention_rows16
    bool join_few;        // attention_join_few joins the splits, else attention_join
    size_t workspace;
};

// The kernel: tiles of many rows that share their codes (attention_rows_tiled)
// where a sequence has rows to fill one and the tiles, or the tiles by the
// tokens they look at, fill the chip; 16 rows a workgroup, its waves sharing the
// tokens, otherwise. Measured both ways (us, tiled / 16 rows; 32 query heads, 8
// KV heads, d 128, but where said), where the rule takes the slower marked *:
//   f16  64 x 33 of 300   32.4 / 57.8     64 x 64 of 64    32.3 / 58.7
//        1 x 64 of 2500   26.3 / 20.9     1 x 64 of 8000   31.1 / 34.9
//        1 x 256 of 1000  29.3 / 18.1     1 x 256 of 8000  52.9 / 96.6
//        16 x 128 of 128  16.4 / 33.6     8 x 200 of 1200  44.0 / 93.8
//        4 x 32 of 2000  *26.8 / 23.5     16 x 32 of 1000  32.1 / 32.1
//   16 / 4 heads, d 64: 16 x 128 of 128 8.9 / 12.8, of 300 *20.6 / 17.9; 1 x 256 of
//        8000 38.3 / 38.0; 8 x 200 of 1200 *34.7 / 32.6
//   ragged, of 2500: 24 of 1 to 100 rows 85.2 / *125, of 1 to 300 141 / 275; d 64
//        64.4 / *73.1 and 112 / 157; 7 of 1 to 300 78.5 / 103, d 64 62.2 / 60.1
//   f32  64 x 33 of 300   87.8 / 86.7     64 x 64 of 64    54.9 / 110
//        1 x 64 of 8000   45.6 / 40.2     1 x 256 of 1000  33.7 / 21.5
//        1 x 200 of 4000  64.4 / 68.1     1 x 96 of 12000  77.0 / 93.3
//        4 x 32 of 2000   32.3 / 27.0     2 x 128 of 8000  112 / 117
//        2 x 256 of 1000 *45.9 / 38.6     8 x 200 of 1200  119 / 126
//        d 64: 2 x 256 of 1000 30.6 / 22.5; 1 x 200 of 4000 35.8 / 41.7; 1 x 96 of
//        12000 47.4 / 57.2; 16 / 4 heads 16 x 128 of 128 12.3 / 18.0, of 300 *24.9 / 23.0
//   ragged, of 2500: 24 of 1 to 100 205 / 164, of 1 to 200 *290 / 270, of 1 to 300 365 /
//        367; d 64 95.3 / 91.0, 151 / 150 and 170 / 202
// (ragged calls: by their mean.) Splits of the longest sequence that the page
// table has room for: as many workgroups as the chip holds at once (more of
// them were slower: one token over 126976, 58 us with 512, 67 with 768, 72 with
// 1024), no fewer than 4 tiles each, and none where a wave has no more than two
// tiles without (f16 rows; split / not, one token of each, us: 8 x 300 9.8 / 8.6,
// 32 x 300 11.6 / 8.9, 1 x 500 9.7 / 9.1, 1 x 777 9.8 / 11.6; f32 2 x 300 11.3 /
// 11.8). Joining in the same launch, by the workgroup that is last to finish,
// took as long as the second launch: its words go past the caches, one round
// trip after another (1 x 777 10.2 us, 64 x 4096 75.1, 1 x 126976 66.0).
AttnPlan attn_plan(const NnopsCacheAttentionArgs* g)
{
    AttnPlan a{};
    const int64_t heads = g->cache.heads, group = g->q_heads / heads, b = g->cache.sequences, d = g->cache.head_dim;
    const int64_t mean = (g->rows * group + b - 1) / b;
    const auto items_of = [&](int64_t tile_rows) {
        if (g->cache.row_starts == nullptr) {
            return b * ((g->rows / b * group + tile_rows - 1) / tile_rows) * heads;
        }
        return (g->rows * group / tile_rows + (b < g->rows ? b : g->rows)) * heads;
    };
    const auto tiles_of = [&](int64_t tile_rows) {
        const int64_t tiles = (g->cache.table_pages * g->cache.page_tokens + kTile - 1) / kTile;
        if (g->window <= 0) {
            return tiles;
        }
        // a tile's rows see the window, up to tile_rows - 1 tokens more, and the sinks
        const int64_t sinks = (g->sinks < INT32_MAX ? g->sinks : INT32_MAX) / kTile + 1;
        const int64_t seen = (g->window < INT32_MAX ? g->window : INT32_MAX) / kTile + tile_rows / kTile + 3 + sinks;
        return tiles < seen ? tiles : seen;
    };
    a.tile_rows = kRows;
    const bool ragged = g->cache.row_starts != nullptr;
    if (const int rows = mean > (ragged ? 256 : 96) ? tiled_rows(d, g->f16, g->cache.page_tokens, mean) : 0; rows > 0) {
        // (tiles that are sure to be full; heads of 64 channels and fewer gain less,
        // and so do wider f32 ones, whose four waves are in one phase)
        const int64_t items = ragged ? g->rows * group / rows * heads : items_of(rows);
        const int64_t least = d > 64 ? (g->f16 ? 7 << 14 : 9 << 15) : g->f16 || ragged ? 7 << 15 : 7 << 14;
        if (items >= 128 || items * tiles_of(rows) * d >= least) {
            a.tiled = true;
            a.tile_rows = rows;
        }
    }
    a.items = items_of(a.tile_rows);
    a.per_seq = g->cache.row_starts == nullptr ? (int32_t)(a.items / (b * heads)) : 0;
    const int64_t tiles = tiles_of(a.tile_rows);
    int64_t splits = ((a.tiled ? 256 : 512) + a.items - 1) / a.items;
    a.whole = g->f16 && d <= 128 && !a.tiled ? 8 : 4;
    const int64_t most = tiles <= a.whole ? 1 : (tiles + 3) / 4;
    splits = splits < most ? splits : most;
    splits = splits > 1 ? splits : 1;
    const int64_t chunk = ((tiles + splits - 1) / splits + 3) / 4 * 4;
    a.chunk = (int32_t)(chunk > 4 ? chunk : 4);
    a.splits = (int32_t)(tiles > 0 ? (tiles + a.chunk - 1) / a.chunk : 1);
    a.tiles = (int32_t)tiles;
    // (a wave per row where few rows and 4 splits leave it waiting: 8 x 1 of 1500
    // 13.8 us, 12.6 with a workgroup; 1 x 64 of 2000 16.9 and 19.5)
    a.join_few = a.splits <= kFewSplits && (a.splits <= 3 || g->rows * g->q_heads >= 1024);
    a.workspace = a.splits > 1 ? (size_t)a.splits * g->rows * g->q_heads * (g->cache.head_dim + 2) * 4 : 0;
    return a;
}

// The rules on sizes: what attn_plan and the launch assume. (In particular,
// rows that divide among the sequences: there is a tile of rows to plan for.)
int check_shapes(const NnopsCacheAttentionArgs* g)
{
    if (g == nullptr || g->q_heads < 0 || g->window < 0 || g->sinks < 0 || !(g->scale >= 0.0f)) {
        return NNOPS_INVALID_ARGUMENT;
    }
    if (const int rc = check_page_shapes(g->cache, g->rows); rc >= 0) {
        return rc;
    }
    if (g->q_heads == 0 || g->q_heads % g->cache.heads != 0 || g->cache.pages == 0) {
        return NNOPS_INVALID_ARGUMENT;
    }
    if (g->q_heads > (1 << 16) || g->rows * g->q_heads > INT32_MAX / 2) {
        return NNOPS_UNSUPPORTED;
    }
    return -1;
}

template <typename T>
void launch_attention(const AttnKern& k, const AttnPlan& a, hipStream_t s)
{
    const dim3 grid((unsigned)a.items, (unsigned)a.splits);
    if (a.tiled) {
        launch_tiled(k, grid, sizeof(T) == 2, s);
    } else if (k.c.d <= 64) {
        NNOPS_LAUNCH((attention_rows16<T, 64>), grid, dim3(256), 0, s, k);
    } else if (k.c.d <= 128) {
        NNOPS_LAUNCH((attention_rows16<T, 128>), grid, dim3(256), 0, s, k);
    } else {
        NNOPS_LAUNCH((attention_rows16<T, 256>), grid, dim3(256), 0, s, k);
    }
    if (a.splits > 1 && a.join_few) {
        const int rows = 256 / join_lanes(k.c.d);   // of a workgroup
        NNOPS_LAUNCH(attention_join_few<T>, dim3((unsigned)((k.c.rows * k.q_heads + rows - 1) / rows)), dim3(256), 0, s, k);
    } else if (a.splits > 1) {
        NNOPS_LAUNCH(attention_join<T>, dim3((unsigned)(k.c.rows * k.q_heads)), dim3(256), 0, s, k);
    }
}

}  // namespace
}  // namespace nnops_amd

using namespace nnops_amd;

extern "C" size_t nnops_hip_cache_attention_workspace_size(const NnopsCacheAttentionArgs* g)
{
    // (the tables' contents and the pointers play no part; a call that is refused,
    // or that has nothing to do, needs none)
    return check_shapes(g) >= 0 ? 0 : attn_plan(g).workspace;
}

extern "C" int nnops_hip_cache_attention_plan(const NnopsCacheAttentionArgs* g, NnopsCacheAttentionPlan* out)
{
    if (out == nullptr) {
        return NNOPS_INVALID_ARGUMENT;
    }
    *out = NnopsCacheAttentionPlan{};
    if (const int rc = check_shapes(g); rc >= 0) {
        return rc;
    }
    const AttnPlan a = attn_plan(g);
    out->tile_rows = a.tile_rows;
    out->one_page = a.tiled && tiled_one_page(g->cache.head_dim, g->cache.page_tokens);
    out->splits = a.splits;
    out->split_tokens = a.chunk * kTile;
    out->join = a.splits <= 1 ? 0 : a.join_few ? 1 : 2;
    out->workspace_bytes = a.workspace;
    return NNOPS_OK;
}

extern "C" int nnops_hip_cache_attention(const NnopsCacheAttentionArgs* g, void* workspace, size_t workspace_bytes,
                                         void* stream)
{
    const TimingDisarm disarm;
    if (const int rc = check_shapes(g); rc >= 0) {
        return rc;
    }
    if (const int rc = check_page_memory(g->cache); rc >= 0) {
        return rc;
    }
    const int64_t width = g->q_heads * g->cache.head_dim;
    if (g->q == nullptr || g->out == nullptr || g->ld_q < width || g->ld_out < width) {
        return NNOPS_INVALID_ARGUMENT;
    }
    const AttnPlan a = attn_plan(g);
    if (a.items > INT32_MAX / 512 || a.splits > 65535) {
        return NNOPS_UNSUPPORTED;
    }
    if (a.workspace > 0 && (workspace == nullptr || workspace_bytes < a.workspace || (uintptr_t)workspace % 16 != 0)) {
        return NNOPS_NOT_INITIALIZED;
    }
    AttnKern k{};
    k.c = paged(g->cache, g->rows);
    k.q = g->q;
    k.out = g->out;
    k.ld_q = g->ld_q;
    k.ld_out = g->ld_out;
    k.part = static_cast<float*>(workspace);
    k.part_ml = k.part + (size_t)a.splits * g->rows * g->q_heads * g->cache.head_dim;
    const float scale = g->scale > 0.0f ? g->scale : 1.0f / __builtin_sqrtf((float)g->cache.head_dim);
    k.scale_log2 = scale * 1.4426950408889634f;
    k.q_heads = (int32_t)g->q_heads;
    k.group = (int32_t)(g->q_heads / g->cache.heads);
    k.window = g->window > INT32_MAX ? 0 : (int32_t)g->window;   // longer than any sequence: none
    k.sinks = g->sinks > INT32_MAX ? INT32_MAX : (int32_t)g->sinks;
    k.tile_rows = a.tile_rows;
    k.per_seq = a.per_seq;
    k.splits = a.splits;
    k.by_splits = a.splits > 1 ? (uint32_t)(((1ull << 32) + a.splits - 1) / a.splits) : 0;
    k.tiles = a.tiles;
    k.whole = a.whole;
    k.chunk = a.chunk;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (g->f16) {
        launch_attention<_Float16>(k, a, s);
    } else {
        launch_attention<float>(k, a, s);
    }
    return hipGetLastError() == hipSuccess ? NNOPS_OK : NNOPS_INTERNAL;
}
