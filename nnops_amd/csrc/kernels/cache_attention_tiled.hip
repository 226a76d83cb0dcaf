// Attention over the paged 8-bit cache for many rows (prompts, chunks of
// prompts). A workgroup has NW x 32 rows (token x head of the group) of one KV
// head and walks tiles of 64 tokens that its waves share through LDS:
//   S^T[64 x 32] = K Q^T,  O^T[d x 32] += V^T P^T   v_mfma_f32_32x32x16
// The codes are turned into f16 (f32 rows: bf16) once per workgroup, on their
// way into LDS; a wave's rows stay in its registers as the products' second
// operand, P goes from S^T's registers straight into the second product: row m
// of a score tile of 32 tokens is token (m with bits 2 and 3 exchanged), so that
// registers 8 s .. 8 s + 7 of lane l are tokens 16 s + 8 (l / 32) + 0..7, the
// operand's k order.
//
// Bound: the matrix cores and, as long, the exponentials and the other steps of
// the softmax. A wave alternates between a matrix phase (the last tile's
// second product, the next tile's scores) and a vector phase (its softmax, its
// share of the coming tiles' codes into LDS); of the two waves of a SIMD one is
// a phase behind, so that one multiplies while the other computes weights. A
// barrier ends each phase. Waves 4 to 7 stage a tile further ahead, since their
// vector phase comes half a tile later: the keys of tile j + 1 and the values of
// tile j are written in phases 2 j (waves 4 to 7) and 2 j + 1 (waves 0 to 3),
// over those of j - 1 and j - 2, which phase 2 j - 1 read last. The global loads
// of a piece are issued a period before it is written, its page number one
// before that. Rows in LDS are 16 bytes longer than their data: 16 lanes' reads
// of one column meet 16 bank groups, at constant offsets.
#include <type_traits>

#include "cache_attention.hpp"

namespace nnops_amd {
namespace {

__device__ __forceinline__ float across(float x)   // the other half-wave's value
{
#if __HIP_DEVICE_COMPILE__
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(threadIdx.x & 32 ? r[0] : r[1]);
#else
    return x;
#endif
}

template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW) void attention_rows_tiled(const AttnKern p)
{
    typedef Operand<T> Op;
    typedef typename Op::Vec Vec;
    constexpr int kThreads = 64 * NW;
    constexpr int kPieces = kTile * DP / 16;                         // 16-code pieces of a tile's side
    constexpr int kPer = (kPieces + kThreads - 1) / kThreads;        // of a thread
    constexpr int kSteps = DP / 16;                                  // k steps of the scores
    constexpr int kOut = DP / 32;                                    // 32-channel tiles of O
    constexpr int kRowPieces = DP / 16;
    constexpr int kPitchK = DP + 8, kPitchV = kTile + 8;             // in 2-byte values
    constexpr bool kPair = NW == 8;                                  // two waves of a SIMD, a phase apart

    __shared__ __attribute__((aligned(16))) uint16_t s_k[2][kTile * kPitchK];
    __shared__ __attribute__((aligned(16))) uint16_t s_v[2][DP * kPitchV];
    __shared__ __attribute__((aligned(16))) float s_scale[4][3][4];  // mul, add, inv of the groups of 16 tokens

    const Paged& c = p.c;
    const int64_t item = blockIdx.x / (unsigned)c.heads;
    const int kvh = (int)(blockIdx.x - item * c.heads);
    RowTile rt;
    if (!find_tile(p, item, true, rt)) {
        return;
    }
    const SeqRows& seq = rt.seq;
    const int split = blockIdx.y;
    if (split > 0 && split >= rt.active) {
        return;
    }
    const int v0 = split * p.chunk, v1 = min(rt.span.tiles, v0 + p.chunk);
    const int tid = threadIdx.x, lane = tid % 64;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);       // uniform: what hangs on it are scalar branches
    const int n = lane % 32, hh = lane / 32;
    const int d = c.d;
    const int64_t page_bytes = (int64_t)c.page * d;

    // the wave's rows; a wave without any only helps to fill LDS
    const int64_t wrow = rt.row0 + 32 * wave;
    const bool wave_live = wrow < rt.rows;
    const int64_t wlast = min(wrow + 32, rt.rows) - 1;
    const int pos0 = seq.len - seq.n;
    const int wmin = wave_live ? pos0 + (int)(wrow / p.group) : 0, wmax = wave_live ? pos0 + (int)(wlast / p.group) : -1;
    const int64_t row = wrow + n;
    const bool is_row = row < rt.rows;
    const int tok = is_row ? (int)(row / p.group) : 0;
    const int head = kvh * p.group + (is_row ? (int)(row - (int64_t)tok * p.group) : 0);
    const int pos = is_row ? pos0 + tok : -1;

    // Q's fragments: channels 16 i + 8 hh .. + 7 of the lane's row are k step i
    Vec qf[kSteps][Op::kParts];
    {
        const T* q = static_cast<const T*>(p.q) + (int64_t)(seq.start + tok) * p.ld_q + (int64_t)head * d;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            T x[8] = {};
            if (is_row && 16 * i < d) {
                __builtin_memcpy(x, q + 16 * i + 8 * hh, sizeof x);
            }
            Op::split(x, qf[i]);
        }
    }

    // --- codes: page number -> registers -> LDS -----------------------------
    // (a page past the last position: any page's codes, they are masked)
    const int32_t* table = c.table + (int64_t)rt.b * c.ld_table;
    const auto page_at = [&](int token) {
        const int id = table[min(token, rt.pmax) >> c.page_log2];
        return id >= 0 && id < c.pages ? id : -1;
    };
    const int64_t page_step = page_bytes * c.heads;
    const int8_t *k_at = c.k + kvh * page_bytes, *v_at = c.v + kvh * page_bytes;
    v4i rk[kPer], rv[kPer];
    int kid[kPer], vid[kPer], sid = 0;
    Scales rs{0.0f, 0.0f, 0.0f};
    const auto ids_k = [&](int v) {
        const int base = tile_base(rt.span, v);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            kid[i] = page_at(base + (tid + i * kThreads) / kRowPieces);
        }
        if (tid < 4) {
            sid = page_at(base + 16 * tid);
        }
    };
    const auto ids_v = [&](int v) {
        const int base = tile_base(rt.span, v);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            vid[i] = page_at(base + (tid + i * kThreads) % 4 * 16);
        }
    };
    const auto load_k = [&](int v) {
        const int base = tile_base(rt.span, v);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int piece = tid + i * kThreads, slot = (base + piece / kRowPieces) & (c.page - 1);
            const int at = piece % kRowPieces * 16;
            rk[i] = v4i{0, 0, 0, 0};
            if ((kPieces % kThreads == 0 || piece < kPieces) && at < d) {
                rk[i] = *reinterpret_cast<const v4i*>(k_at + max(kid[i], 0) * page_step + (slot * d + at));
            }
        }
        if (tid < 4) {
            rs = Scales{0.0f, 0.0f, 0.0f};
            if (base + 16 * tid <= rt.pmax) {
                rs = scales_of(p, sid, (int64_t)max(sid, 0) * c.heads + kvh);
            }
        }
    };
    const auto load_v = [&](int v) {
        const int base = tile_base(rt.span, v);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int piece = tid + i * kThreads, ch = piece / 4, slot = (base + piece % 4 * 16) & (c.page - 1);
            rv[i] = v4i{0, 0, 0, 0};
            if ((kPieces % kThreads == 0 || piece < kPieces) && ch < d) {
                rv[i] = *reinterpret_cast<const v4i*>(v_at + max(vid[i], 0) * page_step + (ch * c.page + slot));
            }
        }
    };
    const auto put = [&](uint16_t* at, const v4i& w) {
        const Vec lo = Op::codes((uint32_t)w.x, (uint32_t)w.y), hi = Op::codes((uint32_t)w.z, (uint32_t)w.w);
        __builtin_memcpy(__builtin_assume_aligned(at, 16), &lo, 16);
        __builtin_memcpy(__builtin_assume_aligned(at + 8, 16), &hi, 16);
    };
    const auto store_k = [&](int v) {
        uint16_t* buf = s_k[v & 1];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int piece = tid + i * kThreads;
            if (kPieces % kThreads == 0 || piece < kPieces) {
                put(buf + piece / kRowPieces * kPitchK + piece % kRowPieces * 16, rk[i]);
            }
        }
        if (tid < 4) {
            s_scale[v & 3][0][tid] = rs.mul;
            s_scale[v & 3][1][tid] = rs.add;
            s_scale[v & 3][2][tid] = rs.inv;
        }
    };
    const auto store_v = [&](int v) {
        uint16_t* buf = s_v[v & 1];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int piece = tid + i * kThreads;
            if (kPieces % kThreads == 0 || piece < kPieces) {
                put(buf + piece / 4 * kPitchV + piece % 4 * 16, rv[i]);
            }
        }
    };

    // --- the two products and the softmax of a wave ------------------------
    v16f o[kOut];
#pragma unroll
    for (int t = 0; t < kOut; ++t) {
        o[t] = v16f{};
    }
    float m_run = kNone, l_run = 0.0f, fresh = 1.0f;
    bool renew = false;                            // uniform
    const int krow = (n & 0x13) | (n & 4) << 1 | (n & 8) >> 1;      // the token of score row n

    const auto lds_vec = [&](const uint16_t* at) {
        Vec a;
        __builtin_memcpy(&a, __builtin_assume_aligned(at, 16), 16);
        return a;
    };
    // LDS reads a few fragments ahead of the products, not all at once
    const auto pace = [](auto fragments) {
        constexpr int kN = decltype(fragments)::value, kAhead = kN < 6 ? kN : 6;
        __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
        for (int i = 0; i < kN - kAhead; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, Op::kParts, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, Op::kParts * kAhead, 0);
    };
    v16f s[2];
    Vec pf[4][Op::kParts];
    const auto scores = [&](int v) {
        const uint16_t* buf = s_k[v & 1] + krow * kPitchK + 8 * hh;
        s[0] = v16f{};
        s[1] = v16f{};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                s[u] = product<T>(lds_vec(buf + 32 * u * kPitchK + 16 * i), qf[i], s[u]);
            }
        }
        pace(std::integral_constant<int, 2 * kSteps>{});
    };
    const auto soft = [&](auto masked, int v, int base) {
        constexpr bool kMasked = decltype(masked)::value;
        float mul[4], add[4], inv[4];
        __builtin_memcpy(mul, s_scale[v & 3][0], 16);
        __builtin_memcpy(add, s_scale[v & 3][1], 16);
        __builtin_memcpy(inv, s_scale[v & 3][2], 16);
        // bit i: the row sees token base + 8 hh + i
        uint32_t bits[2] = {~0u, ~0u};
        if (kMasked) {
            const auto below = [](int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; };
            const int at = base + 8 * hh;
            uint64_t m = below(pos - at + 1);
            if (p.window > 0) {
                m &= ~below(pos - p.window + 1 - at) | below(p.sinks - at);
            }
            bits[0] = (uint32_t)m;
            bits[1] = (uint32_t)(m >> 32);
        }
        const auto seen = [&](int g, int e) {      // all ones or none
            return (uint32_t)((int32_t)(bits[g / 2] << (31 - 16 * (g % 2) - e)) >> 31);
        };
        float top = kNone;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float t = kNone;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float v = s[g / 2][8 * (g % 2) + e];
                if (kMasked) {
                    const uint32_t m = seen(g, e);
                    v = __uint_as_float((__float_as_uint(v) & m) | (0xff800000u & ~m));
                }
                t = fmaxf(t, v);
            }
            // (-inf times a scale of 0 or NaN is a NaN, which fmaxf drops)
            top = fmaxf(top, __builtin_fmaf(t, mul[g], add[g]));
        }
        top = fmaxf(top, across(top));
        if (__any(top > m_run + kLazy)) {
            // (0 where nothing was seen before; O is brought along in the matrix phase)
            fresh = top > m_run ? __builtin_amdgcn_exp2f(m_run - top) : 1.0f;
            l_run *= fresh;
            m_run = top > m_run ? top : m_run;
            renew = true;
        }
        const float shift = m_run > kNone ? kLift - m_run : 0.0f;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float w[8], sum = 0.0f;
            const float a = add[g] + shift;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[g / 2][8 * (g % 2) + e], mul[g], a));
                if (kMasked) {
                    w[e] = __uint_as_float(__float_as_uint(w[e]) & seen(g, e));
                }
                sum += w[e];
            }
            // a page of which the row sees nothing adds nothing, whatever its scale
            l_run += !kMasked || sum != 0.0f ? sum * inv[g] : 0.0f;
            Op::split(w, pf[g]);
        }
    };
    const auto accumulate = [&](int v) {
        if (renew) {
#pragma unroll
            for (int t = 0; t < kOut; ++t) {
                o[t] *= fresh;
            }
            renew = false;
        }
        const uint16_t* buf = s_v[v & 1] + n * kPitchV + 8 * hh;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
#pragma unroll
            for (int t = 0; t < kOut; ++t) {
                o[t] = product<T>(lds_vec(buf + 32 * t * kPitchV + 16 * g), pf[g], o[t]);
            }
        }
        pace(std::integral_constant<int, 4 * kOut>{});
    };
    const auto live = [&](int base) {
        return wave_live && base <= wmax && (p.window == 0 || wmin - (base + kTile - 1) < p.window || base < p.sinks);
    };
    const auto open = [&](int base) { return base + kTile - 1 <= wmin && (p.window == 0 || wmax - base < p.window); };

    // LDS only: what is in flight from global memory stays in flight
    const auto meet = [&] {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };

    // Tiles in terms of 0 .. nt - 1. The group that is a phase behind writes
    // what the other will in its next vector phase.
    const int nt = v1 - v0, behind = kPair ? wave / 4 : 0;
    if (nt > 0) {
        // written: keys 0, and by those behind keys 1 and values 0 (in phase 0);
        // in flight: the first pieces of the loop
        ids_k(v0);
        ids_v(v0);
        load_k(v0);
        store_k(0);
        if (nt > 1) {
            ids_k(v0 + 1);
            load_k(v0 + 1);
        }
        load_v(v0);
        if (nt > 2) {
            ids_k(v0 + 2);
        }
        if (nt > 1) {
            ids_v(v0 + 1);
        }
        meet();
        // a thread's pieces of the values of tile x and the keys of x + 1, and the loads after them
        const auto pieces = [&](int x) {
            if (x < nt) {
                store_v(x);
            }
            if (x + 1 < nt) {
                store_k(x + 1);
                load_v(v0 + x + 1);
            }
            if (x + 2 < nt) {
                load_k(v0 + x + 2);
                ids_v(v0 + x + 2);
            }
            if (x + 3 < nt) {
                ids_k(v0 + x + 3);
            }
        };
        if (behind) {
            pieces(0);
            meet();
        }
        bool was = false;                          // the last tile has weights to multiply
        for (int j = 0; j < nt; ++j) {
            const int base = tile_base(rt.span, v0 + j);
            const bool now = live(base);
            if (was) {
                accumulate(j - 1);
            }
            if (now) {
                scores(j);
            }
            meet();
            pieces(j + behind);
            if (now) {
                if (open(base)) {
                    soft(std::false_type{}, j, base);
                } else {
                    soft(std::true_type{}, j, base);
                }
            }
            was = now;
            meet();
        }
        if (was) {
            accumulate(nt - 1);
        }
        if (kPair && !behind) {
            meet();                                // as many as the others
        }
    }

    if (!is_row) {
        return;                                    // no barrier below
    }
    l_run += across(l_run);
    const int64_t token = seq.start + tok;
    if (rt.active > 1) {
        float* dst = p.part + (((int64_t)split * c.rows + token) * p.q_heads + head) * (d + 2);
#pragma unroll
        for (int t = 0; t < kOut; ++t) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int ch = 32 * t + 8 * (r / 4) + 4 * hh + r % 4;
                if (ch < d) {
                    dst[ch] = o[t][r];
                }
            }
        }
        if (hh == 0) {
            dst[d] = m_run;
            dst[d + 1] = l_run;
        }
        return;
    }
    T* dst = static_cast<T*>(p.out) + token * p.ld_out + (int64_t)head * d;
    const float f = l_run == 0.0f ? 0.0f : kDrop / l_run;
#pragma unroll
    for (int t = 0; t < kOut; ++t) {
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int ch = 32 * t + 8 * (r / 4) + 4 * hh;
            T y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[e] = (T)(o[t][r + e] * f);
            }
            if (ch < d) {                          // (head sizes are multiples of 16: all four or none)
                __builtin_memcpy(dst + ch, y, sizeof y);
            }
        }
    }
}

}  // namespace

int tiled_rows(int64_t d, bool f16, int64_t rows)
{
    if (d > 128 && !f16) {
        return 0;                                  // three parts of 256 channels: more registers than there are
    }
    if (d > 128 || !f16) {
        return 128;
    }
    return rows > 128 ? 256 : 128;
}

void launch_tiled(const AttnKern& k, const dim3& grid, bool f16, hipStream_t s)
{
    const int d = k.c.d, rows = k.tile_rows;
    if (f16 && rows == 256) {
        if (d <= 64) {
            NNOPS_LAUNCH((attention_rows_tiled<_Float16, 64, 8>), grid, dim3(512), 0, s, k);
        } else {
            NNOPS_LAUNCH((attention_rows_tiled<_Float16, 128, 8>), grid, dim3(512), 0, s, k);
        }
    } else if (f16) {
        if (d <= 64) {
            NNOPS_LAUNCH((attention_rows_tiled<_Float16, 64, 4>), grid, dim3(256), 0, s, k);
        } else if (d <= 128) {
            NNOPS_LAUNCH((attention_rows_tiled<_Float16, 128, 4>), grid, dim3(256), 0, s, k);
        } else {
            NNOPS_LAUNCH((attention_rows_tiled<_Float16, 256, 4>), grid, dim3(256), 0, s, k);
        }
    } else if (d <= 64) {
        NNOPS_LAUNCH((attention_rows_tiled<float, 64, 4>), grid, dim3(256), 0, s, k);
    } else {
        NNOPS_LAUNCH((attention_rows_tiled<float, 128, 4>), grid, dim3(256), 0, s, k);
    }
}

}  // namespace nnops_amd
