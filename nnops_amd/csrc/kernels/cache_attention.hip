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
// kernel); a workgroup's 4 waves take every fourth tile and join in LDS.
#include "cache_attention.hpp"

namespace nnops_amd {
namespace {

constexpr int kRows = 16;           // rows of a wave

template <typename T, int DP>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void attention_rows16(const AttnKern p)
{
    constexpr int kC = DP / 64;                    // 64-channel pieces of a key
    constexpr int kT = DP / 16;                    // 16-channel tiles of O
    typedef Operand<T> Op;
    constexpr int kPitch = DP + 4;
    __shared__ float s_o[4][kRows][kPitch];
    __shared__ float s_m[4][kRows], s_l[4][kRows];
    const Paged& c = p.c;
    const int64_t item = blockIdx.x / (unsigned)c.heads;
    const int kvh = (int)(blockIdx.x - item * c.heads);
    RowTile rt;
    if (!find_tile(p, item, false, rt)) {
        return;
    }
    const SeqRows& seq = rt.seq;
    const Span& span = rt.span;
    const int b = rt.b, pmin = rt.pmin, pmax = rt.pmax, active = rt.active;
    const int64_t row0 = rt.row0, rows = rt.rows;
    const int tok_last = pmax - (seq.len - seq.n);
    const int split = blockIdx.y;
    if (split > 0 && split >= active) {
        return;
    }
    const int v0 = split * p.chunk, v1 = min(span.tiles, v0 + p.chunk);

    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int n = lane % 16, g = lane / 16;
    const int64_t row = row0 + n;
    const bool is_row = row < rows;
    const int tok = is_row ? (int)(row / p.group) : tok_last;
    const int head = kvh * p.group + (is_row ? (int)(row - (int64_t)tok * p.group) : 0);
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
    const int kb = n / 4;                          // the token group of a lane's keys
    const int ktok = 16 * kb + n % 4;              // + 4 t: its token in the tile

    for (int v = v0 + wave; v < v1; v += 4) {
        const int base = tile_base(span, v);
        // pages of the lane's key group and value group; past the last
        // position there is none, any page's codes do (they are masked)
        const int kt0 = base + 16 * kb, vt0 = base + 16 * g;
        const int kid = kt0 <= pmax ? page_of(c, b, kt0 >> c.page_log2) : 0;
        const int vid = vt0 <= pmax ? page_of(c, b, vt0 >> c.page_log2) : 0;
        const int8_t* kp = c.k + ((int64_t)max(kid, 0) * c.heads + kvh) * page_bytes +
                           (int64_t)((base + ktok) & (c.page - 1)) * d + 16 * g;
        const int64_t vpage = (int64_t)max(vid, 0) * c.heads + kvh;
        const int8_t* vp = c.v + vpage * page_bytes + (int64_t)n * c.page + (vt0 & (c.page - 1));
        v4i kr[4][kC], vr[kT];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int i = 0; i < kC; ++i) {
                kr[t][i] = 64 * i + 16 * g < d ? *reinterpret_cast<const v4i*>(kp + 4 * t * d + 64 * i) : v4i{0, 0, 0, 0};
            }
        }
        const Scales sc = vt0 <= pmax ? scales_of(p, vid, vpage) : Scales{0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < kT; ++t) {
            vr[t] = 16 * t < d ? *reinterpret_cast<const v4i*>(vp + (int64_t)16 * t * c.page) : v4i{0, 0, 0, 0};
        }

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
        typename Op::Vec pf[2][Op::kParts];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[t / 2][4 * (t % 2) + i] = __builtin_amdgcn_exp2f(x[t][i] + shift);
                sum += w[t / 2][4 * (t % 2) + i];
            }
        }
        Op::split(w[0], pf[0]);
        Op::split(w[1], pf[1]);
        // a page of which the row sees nothing adds nothing, whatever its scale
        l_run += sum != 0.0f ? sum * sc.inv : 0.0f;
#pragma unroll
        for (int t = 0; t < kT; ++t) {
            if (16 * t < d) {
                o[t] = product<T>(Op::codes((uint32_t)vr[t].x, (uint32_t)vr[t].y), pf[0], o[t]);
                o[t] = product<T>(Op::codes((uint32_t)vr[t].z, (uint32_t)vr[t].w), pf[1], o[t]);
            }
        }
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
    for (int i = threadIdx.x; i < kRows * d; i += 256) {
        const int r = i / d, ch = i - r * d;
        if (row0 + r >= rows) {
            break;
        }
        const float m = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
        float sum = 0.0f, l = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            // a wave that saw nothing has m = -inf and nothing to add
            const float f = s_m[w][r] < m ? __builtin_amdgcn_exp2f(s_m[w][r] - m) : 1.0f;
            sum += f * s_o[w][r][ch];
            l += f * s_l[w][r];
        }
        const int64_t at = row0 + r;
        const int64_t token = seq.start + at / p.group;
        const int qh = kvh * p.group + (int)(at % p.group);
        if (active > 1) {
            float* dst = p.part + (((int64_t)split * c.rows + token) * p.q_heads + qh) * (d + 2);
            dst[ch] = sum;
            if (ch == 0) {
                dst[d] = m;
                dst[d + 1] = l;
            }
        } else {
            static_cast<T*>(p.out)[token * p.ld_out + (int64_t)qh * d + ch] =
                (T)(l == 0.0f ? 0.0f : sum * kDrop / l);
        }
    }
}

// Joins the splits of the rows that have more than one. A wave per row.
template <typename T>
__global__ __launch_bounds__(256) void attention_join(const AttnKern p)
{
    const Paged& c = p.c;
    const int64_t i = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
    const int64_t token = i / p.q_heads;
    if (token >= c.rows) {
        return;
    }
    const int qh = (int)(i - token * p.q_heads), lane = threadIdx.x % 64;
    int b;
    if (c.row_starts == nullptr) {
        b = (int)(token / c.uniform);
    } else {
        int lo = 0, hi = c.seqs;                   // the last sequence that starts at or before the row
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            (c.row_starts[mid] <= token ? lo : hi) = mid;
        }
        b = lo;
    }
    const SeqRows seq = seq_rows(c, b);
    const int tok = (int)(token - seq.start);
    if (tok < 0 || tok >= seq.n) {
        return;
    }
    RowTile rt;
    rt.seq = seq;
    place_tile(p, (int)(((int64_t)tok * p.group + qh % p.group) / p.tile_rows), rt);
    const int active = rt.active;
    if (active <= 1) {
        return;
    }
    const int d = c.d;
    const int64_t step = (int64_t)c.rows * p.q_heads * (d + 2);
    const float* part = p.part + (token * p.q_heads + qh) * (d + 2);
    float m = kNone;
    for (int s = 0; s < active; ++s) {
        m = fmaxf(m, part[s * step + d]);
    }
    float l = 0.0f, o[4] = {0, 0, 0, 0};
    for (int s = 0; s < active; ++s) {
        const float ms = part[s * step + d];
        const float f = ms < m ? __builtin_amdgcn_exp2f(ms - m) : 1.0f;
        l += f * part[s * step + d + 1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (lane + 64 * e < d) {
                o[e] += f * part[s * step + lane + 64 * e];
            }
        }
    }
    T* out = static_cast<T*>(p.out) + token * p.ld_out + (int64_t)qh * d;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (lane + 64 * e < d) {
            out[lane + 64 * e] = (T)(l == 0.0f ? 0.0f : o[e] * kDrop / l);
        }
    }
}

struct AttnPlan {
    int64_t items;        // row tiles, all KV heads
    int32_t tile_rows, per_seq, chunk, splits;
    bool tiled;           // attention_rows_tiled, else attention_rows16
    size_t workspace;
};

// Rows of a sequence past kRows go to the kernel whose waves share their tiles
// (ragged calls: by their mean). Splits of the longest sequence that the page
// table has room for: enough workgroups to fill the chip, no fewer than 4 tiles
// each.
AttnPlan attn_plan(const NnopsCacheAttentionArgs* g)
{
    AttnPlan a{};
    const int64_t group = g->q_heads / g->cache.heads, b = g->cache.sequences;
    const int64_t mean = (g->rows * group + b - 1) / b;
    const int tiled = mean > kRows ? tiled_rows(g->cache.head_dim, g->f16, mean) : 0;
    a.tiled = tiled > 0;
    a.tile_rows = a.tiled ? tiled : kRows;
    if (g->cache.row_starts == nullptr) {
        a.per_seq = (int32_t)((g->rows / b * group + a.tile_rows - 1) / a.tile_rows);
        a.items = b * a.per_seq * g->cache.heads;
    } else {
        a.items = (g->rows * group / a.tile_rows + (b < g->rows ? b : g->rows)) * g->cache.heads;
    }
    int64_t tiles = (g->cache.table_pages * g->cache.page_tokens + kTile - 1) / kTile;
    if (g->window > 0) {
        // a tile's rows see the window, up to tile_rows - 1 tokens more, and the sinks
        const int64_t seen = (g->window + a.tile_rows) / kTile + 2 + (g->sinks + kTile - 1) / kTile;
        tiles = tiles < seen ? tiles : seen;
    }
    const int64_t full = a.tiled ? 256 : 512;
    int64_t splits = (full + a.items - 1) / a.items;
    const int64_t most = (tiles + 3) / 4;
    splits = splits < most ? splits : most;
    splits = splits > 1 ? splits : 1;
    const int64_t chunk = ((tiles + splits - 1) / splits + 3) / 4 * 4;
    a.chunk = (int32_t)(chunk > 4 ? chunk : 4);
    a.splits = (int32_t)(tiles > 0 ? (tiles + a.chunk - 1) / a.chunk : 1);
    a.workspace = a.splits > 1 ? (size_t)a.splits * g->rows * g->q_heads * (g->cache.head_dim + 2) * 4 : 0;
    return a;
}

int check_attention(const NnopsCacheAttentionArgs* g)
{
    if (g == nullptr || g->q_heads < 0 || g->window < 0 || g->sinks < 0 || !(g->scale >= 0.0f)) {
        return NNOPS_INVALID_ARGUMENT;
    }
    const int rc = check_pages(g->cache, g->rows);
    if (rc >= 0) {
        return rc;
    }
    if (g->q_heads == 0 || g->q_heads % g->cache.heads != 0 || g->cache.pages == 0) {
        return NNOPS_INVALID_ARGUMENT;
    }
    if (g->q_heads > (1 << 16) || g->rows * g->q_heads > INT32_MAX) {
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
    if (a.splits > 1) {
        const int64_t rows = (int64_t)k.c.rows * k.q_heads;
        NNOPS_LAUNCH(attention_join<T>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, k);
    }
}

}  // namespace
}  // namespace nnops_amd

using namespace nnops_amd;

extern "C" size_t nnops_hip_cache_attention_workspace_size(const NnopsCacheAttentionArgs* g)
{
    // (the tables' contents and the pointers play no part)
    if (g == nullptr || g->rows <= 0 || g->q_heads <= 0 || g->cache.heads <= 0 || g->cache.sequences <= 0 ||
        g->cache.head_dim <= 0 || g->cache.page_tokens <= 0 || g->cache.table_pages < 0 ||
        g->q_heads % g->cache.heads != 0 || g->window < 0 || g->sinks < 0) {
        return 0;
    }
    return attn_plan(g).workspace;
}

extern "C" int nnops_hip_cache_attention(const NnopsCacheAttentionArgs* g, void* workspace, size_t workspace_bytes,
                                         void* stream)
{
    const TimingDisarm disarm;
    const int rc = check_attention(g);
    if (rc >= 0) {
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
    const float scale = g->scale > 0.0f ? g->scale : 1.0f / __builtin_sqrtf((float)g->cache.head_dim);
    k.scale_log2 = scale * 1.4426950408889634f;
    k.q_heads = (int32_t)g->q_heads;
    k.group = (int32_t)(g->q_heads / g->cache.heads);
    k.window = g->window > INT32_MAX ? 0 : (int32_t)g->window;   // longer than any sequence: none
    k.sinks = g->sinks > INT32_MAX ? INT32_MAX : (int32_t)g->sinks;
    k.tile_rows = a.tile_rows;
    k.per_seq = a.per_seq;
    k.chunk = a.chunk;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (g->f16) {
        launch_attention<_Float16>(k, a, s);
    } else {
        launch_attention<float>(k, a, s);
    }
    return hipGetLastError() == hipSuccess ? NNOPS_OK : NNOPS_INTERNAL;
}
