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
#pragma once

#include <type_traits>

#include "cache_attention.hpp"

namespace nnops_amd {
namespace {

constexpr int kRows = 16;           // rows of a wave

// What the waves of a workgroup join. (aligned: 16 bytes at once, which a reference
// alone does not let the compiler see; 16 x 4096 at d 256 53.9 -> 53.3 us)
template <int DP>
struct WaveParts {
    __attribute__((aligned(16))) float o[4][kRows][DP + 4];
    float m[4][kRows], l[4][kRows];
};

// What the lanes that share a row's parts join.
struct WayParts {
    __attribute__((aligned(16))) v4f o[256];
    float m[16], l[16];
};

// One part more: M and l of a row, 4 channels of its O.
__device__ __forceinline__ void join_part(float& m, float& l, v4f& o, float pm, float pl, const v4f& po)
{
    const float top = fmaxf(m, pm);
    // (a part that saw nothing has -inf and nothing to add)
    const float f = m < top ? __builtin_amdgcn_exp2f(m - top) : 1.0f;
    const float w = pm < top ? __builtin_amdgcn_exp2f(pm - top) : 1.0f;
    l = f * l + w * pl;
    o = f * o + w * po;
    m = top;
}

// Every step-th of the parts from first on, of n in all: number s is at part(s). Of
// kAtOnce rows side by side, their loads in flight together.
template <int kBatch, int kAtOnce, typename Part>
__device__ __forceinline__ void join_parts(const AttnKern& p, const int64_t (&at)[kAtOnce], int ch, int first, int step,
                                           int n, Part part, float (&m)[kAtOnce], float (&l)[kAtOnce], v4f (&o)[kAtOnce])
{
    const int64_t rows = (int64_t)p.c.rows * p.q_heads;
    for (int s = first; s < n; s += kBatch * step) {
        float ms[kAtOnce][kBatch], ls[kAtOnce][kBatch];
        v4f os[kAtOnce][kBatch];
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
            const int i = s + e * step;
#pragma unroll
            for (int a = 0; a < kAtOnce; ++a) {
                ms[a][e] = kNone;
                ls[a][e] = 0.0f;
                os[a][e] = v4f{0, 0, 0, 0};
            }
            if (i < n) {
#pragma unroll
                for (int a = 0; a < kAtOnce; ++a) {
                    const int64_t from = part(i) * rows + at[a];
                    ms[a][e] = p.part_ml[2 * from];
                    ls[a][e] = p.part_ml[2 * from + 1];
                    if (ch < p.c.d) {
                        os[a][e] = *reinterpret_cast<const v4f*>(p.part + from * p.c.d + ch);
                    }
                }
            }
        }
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
#pragma unroll
            for (int a = 0; a < kAtOnce; ++a) {
                join_part(m[a], l[a], o[a], ms[a][e], ls[a][e], os[a][e]);
            }
        }
    }
}

// The `ways` neighbouring slots of lanes that have parts of one row: the first of them
// gets the sum. Every thread of the workgroup calls it.
__device__ __forceinline__ void join_ways(WayParts& sh, int lanes, int ways, float& m, float& l, v4f& o)
{
    const int slot = threadIdx.x / (uint32_t)lanes;
    if (ways > 1) {
        sh.o[threadIdx.x] = o;
        if (threadIdx.x % (uint32_t)lanes == 0) {
            sh.m[slot] = m;
            sh.l[slot] = l;
        }
        __syncthreads();
        if (slot % ways == 0) {
            for (int w = 1; w < ways; ++w) {
                join_part(m, l, o, sh.m[slot + w], sh.l[slot + w], sh.o[threadIdx.x + w * lanes]);
            }
        }
    }
}

// 4 channels of a row's result.
template <typename T>
__device__ __forceinline__ void write_result(const AttnKern& p, int64_t token, int qh, int ch, float l, const v4f& o)
{
    const float f = l == 0.0f ? 0.0f : kDrop / l;
    T y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        y[e] = (T)(o[e] * f);
    }
    __builtin_memcpy(static_cast<T*>(p.out) + token * p.ld_out + (int64_t)qh * p.c.d + ch, y, sizeof y);
}

template <typename T, int DP, AttnMode M>
__device__ __forceinline__ void attend_rows16(const KernOf<M>& p, WaveParts<DP>& sh, uint32_t block, int split,
                                              WayParts* join = nullptr)
{
    constexpr int kC = DP / 64;                    // 64-channel pieces of a key
    constexpr int kT = DP / 16;                    // 16-channel tiles of O
    typedef Operand<T> Op;
    constexpr int kWeights = Op::kParts == 1 ? 2 : Op::kParts;   // parts of a probability
    const Paged& c = p.c;
    const uint32_t item = block / (uint32_t)c.heads;
    const int kvh = (int)(block - item * c.heads);
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int n = lane % 16, g = lane / 16;
    const int kb = n / 4;                          // the token group of a lane's keys
    // Without a window a wave's first tile is known before the lengths are, if
    // sequences are not split or the longest fills the page table: its page numbers
    // are asked for beside them. (Past the sequence's end they may be anything; what
    // is read through them is masked.)
    const bool early = M == kWhole && p.window == 0 && p.per_seq > 0 && c.table_pages > 0;
    int kid = 0, vid = 0;
    if (early) {
        const int32_t* row = c.table + (int64_t)(item / (uint32_t)p.per_seq) * c.ld_table;
        const int base = kTile * (split * p.chunk + wave), last = c.table_pages - 1;
        kid = row[min((base + 16 * kb) >> c.page_log2, last)];
        vid = row[min((base + 16 * g) >> c.page_log2, last)];
    }
    RowTile rt;
    if (!find_tile<M>(p, item, false, rt)) {
        return;
    }
    const SeqRows& seq = rt.seq;
    const Span& span = rt.span;
    const int b = rt.b, pmin = rt.pmin, pmax = rt.pmax;
    const int row0 = rt.row0, rows = rt.rows;
    const int tok_last = M == kShared ? (int)((uint32_t)(min(row0 + kRows, rows) - 1) / (uint32_t)p.group)
                                      : pmax - (seq.len - seq.n);
    const int v0 = split * rt.chunk;
    if (split > 0 && v0 >= span.tiles) {
        return;
    }
    const int v1 = min(span.tiles, v0 + rt.chunk);

    const int row = row0 + n;
    const bool is_row = row < rows;
    const int tok = is_row ? (int)((uint32_t)row / (uint32_t)p.group) : tok_last;
    const int head = kvh * p.group + (is_row ? row - tok * p.group : 0);
    const int pos = M == kShared ? pmax : seq.len - seq.n + tok;
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
    const int32_t* table = c.table + (int64_t)(M == kShared ? rt.table : b) * c.ld_table;
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
        const bool open =
            M == kShared || (base + kTile - 1 <= pmin && (p.window == 0 || pmax - base < p.window));
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
        sh.m[wave][n] = m_run;
        sh.l[wave][n] = l_run;
    }
#pragma unroll
    for (int t = 0; t < kT; ++t) {
        *reinterpret_cast<v4f*>(&sh.o[wave][n][16 * t + 4 * g]) = o[t];
    }
    __syncthreads();
    if constexpr (M == kOwn) {
        if (p.join_here) {
            // the waves' parts and those of the shared tokens, by as many lanes a row as
            // there are
            const int lanes = join_lanes(d), slots = 256 / lanes, slot = threadIdx.x / (uint32_t)lanes;
            const int here = min(kRows, rows - row0), ch = threadIdx.x % (uint32_t)lanes * 4;
            int ways = 1;
            while (2 * ways * here <= slots) {
                ways *= 2;
            }
            const int way = slot % ways, step = slots / ways;
            constexpr int kAtOnce = DP > 64 ? 2 : 1;            // (with one way)
            for (int r0 = 0; r0 < here; r0 += kAtOnce * step) {   // (once, if there is more than one way)
                int64_t at[kAtOnce];
                float m[kAtOnce], l[kAtOnce];
                v4f o4[kAtOnce];
#pragma unroll
                for (int a = 0; a < kAtOnce; ++a) {
                    const int row = min(row0 + r0 + a * step + slot / ways, rows - 1);
                    const int t = (int)((uint32_t)row / (uint32_t)p.group);
                    at[a] = (int64_t)(seq.start + t) * p.q_heads + kvh * p.group + (row - t * p.group);
                    m[a] = kNone;
                    l[a] = 0.0f;
                    o4[a] = v4f{0, 0, 0, 0};
                }
                const auto part = [](int s) { return s; };
                if (kAtOnce > 1 && r0 + step < here) {
                    join_parts<4>(p, at, ch, way, ways, rt.shared_parts, part, m, l, o4);
                } else {
                    const int64_t one[1] = {at[0]};
                    float m1[1] = {m[0]}, l1[1] = {l[0]};
                    v4f o1[1] = {o4[0]};
                    join_parts<8>(p, one, ch, way, ways, rt.shared_parts, part, m1, l1, o1);
                    m[0] = m1[0];
                    l[0] = l1[0];
                    o4[0] = o1[0];
                }
#pragma unroll
                for (int a = 0; a < kAtOnce; ++a) {
                    const int row = r0 + a * step + slot / ways;
                    if (row < here) {
                        for (int w = way; w < 4 && ch < d; w += ways) {
                            join_part(m[a], l[a], o4[a], sh.m[w][row], sh.l[w][row],
                                      *reinterpret_cast<const v4f*>(&sh.o[w][row][ch]));
                        }
                    }
                }
                join_ways(*join, lanes, ways, m[0], l[0], o4[0]);
#pragma unroll
                for (int a = 0; a < kAtOnce; ++a) {
                    if (r0 + a * step + slot / ways < here && way == 0 && ch < d) {
                        const int64_t token = at[a] / p.q_heads;
                        write_result<T>(p, token, (int)(at[a] - token * p.q_heads), ch, l[a], o4[a]);
                    }
                }
            }
            return;
        }
    }
    // 16 threads a row, 4 channels each at a time
    const int r = threadIdx.x / 16, ch0 = threadIdx.x % 16 * 4;
    if (row0 + r >= rows) {
        return;
    }
    const float m = fmaxf(fmaxf(sh.m[0][r], sh.m[1][r]), fmaxf(sh.m[2][r], sh.m[3][r]));
    float f[4], l = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        // a wave that saw nothing has m = -inf and nothing to add
        f[w] = sh.m[w][r] < m ? __builtin_amdgcn_exp2f(sh.m[w][r] - m) : 1.0f;
        l += f[w] * sh.l[w][r];
    }
    const int rtok = (int)((uint32_t)(row0 + r) / (uint32_t)p.group);
    const int64_t token = seq.start + rtok;
    const int qh = kvh * p.group + (row0 + r - rtok * p.group);
    const bool parts = M != kWhole || rt.split;
    const int64_t at_part = ((int64_t)(split + first_part<M>(p)) * c.rows + token) * p.q_heads + qh;
    const float scale = parts ? 1.0f : l == 0.0f ? 0.0f : kDrop / l;
#pragma unroll
    for (int i = 0; i < DP / 64; ++i) {
        const int ch = ch0 + 64 * i;
        if (ch >= d) {
            break;
        }
        v4f sum = v4f{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            sum += f[w] * *reinterpret_cast<const v4f*>(&sh.o[w][r][ch]);
        }
        if (parts) {
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
    if (parts && ch0 == 0) {
        p.part_ml[2 * at_part] = m;
        p.part_ml[2 * at_part + 1] = l;
    }
}

template <typename T, int DP, AttnMode M>
__global__ __launch_bounds__(256, DP > 128 ? 1 : sizeof(T) == 2 ? 3 : 2) void attention_rows16(const KernOf<M> p)
{
    __shared__ WaveParts<DP> sh;
    if constexpr (M == kOwn) {
        __shared__ WayParts join;
        attend_rows16<T, DP, M>(p, sh, blockIdx.x, blockIdx.y, &join);
    } else {
        attend_rows16<T, DP, M>(p, sh, blockIdx.x, blockIdx.y);
    }
}

}  // namespace
}  // namespace nnops_amd
