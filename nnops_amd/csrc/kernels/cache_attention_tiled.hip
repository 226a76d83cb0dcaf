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
// the softmax. A wave alternates between a matrix phase (the last tile's second
// product and the next tile's scores, with its share of the coming tiles' codes
// turned and put into LDS between them: vector instructions beside a matrix
// instruction are nearly free) and a vector phase (the softmax); of the two
// waves of a SIMD one is a phase behind, so that one multiplies while the other
// computes weights. A barrier ends each phase. The keys of tile j + 1 and the
// values of tile j are written in phases 2 j (waves 0 to 3) and 2 j + 1 (waves 4
// to 7), over those of j - 1 and j - 2, which phase 2 j - 1 read last. The loads
// of a piece are issued a tile before it is written, its page number one before
// that. Rows in LDS are 16 bytes longer than their data: 16 lanes' reads
// of one column meet 16 bank groups, at constant offsets.
// Measured: a prompt of 4096, 32 query and 8 KV heads of 128, f16, 137 GFLOP: 143 to
// 153 us, 900 to 960 TFLOP/s, where a large f16 product reaches 1156 on this card;
// with four waves (128 rows), none a phase behind, 249 us.
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

// Memory that no kernel of the call writes, for addresses that are the same in
// a whole wave: scalar loads, whatever barriers lie between.
template <typename V>
__device__ __forceinline__ V uniform_load(const V* p)
{
#if __HIP_DEVICE_COMPILE__
    return *(const __attribute__((address_space(4))) V*)(uintptr_t)p;
#else
    return *p;
#endif
}

// kOne: pages of 64 tokens and more, so that a tile lies in one: its number and
// scales are scalars, its codes at a scalar base and fixed offsets.
template <typename T, int DP, int NW, bool kOne>
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
    __shared__ __attribute__((aligned(16))) v4f s_scale[4][4];       // mul, add, inv of the groups of 16 tokens

    const Paged& c = p.c;
    const uint32_t item = blockIdx.x / (uint32_t)c.heads;
    const int kvh = (int)(blockIdx.x - item * c.heads);
    RowTile rt;
    if (!find_tile(p, item, true, rt)) {
        return;
    }
    const SeqRows& seq = rt.seq;
    const int split = blockIdx.y;
    const int v0 = split * rt.chunk;
    if (split > 0 && v0 >= rt.span.tiles) {
        return;
    }
    const int v1 = min(rt.span.tiles, v0 + rt.chunk);
    const int tid = threadIdx.x, lane = tid % 64;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);       // uniform: what hangs on it are scalar branches
    const int n = lane % 32, hh = lane / 32;
    const int d = c.d;

    // the wave's rows; a wave without any only helps to fill LDS
    const uint32_t group = p.group;
    const int wrow = rt.row0 + 32 * wave;
    const bool wave_live = wrow < rt.rows;
    const int wlast = min(wrow + 32, rt.rows) - 1;
    const int pos0 = seq.len - seq.n;
    const int wmin = wave_live ? pos0 + (int)((uint32_t)wrow / group) : 0;
    const int wmax = wave_live ? pos0 + (int)((uint32_t)wlast / group) : -1;
    const int row = wrow + n;
    const bool is_row = row < rt.rows;
    const int tok = is_row ? (int)((uint32_t)row / group) : 0;
    const int head = kvh * p.group + (is_row ? row - tok * p.group : 0);
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
    // Without a branch, so that what is in flight stays in flight: tiles past the
    // last one are the last again, tokens past the last position have its page
    // (they are masked), channels past d are channel 0's codes (q is 0 there, and
    // their output is not stored). Page numbers are looked at when they are used.
    const int32_t* table = c.table + (int64_t)rt.b * c.ld_table;
    const uint32_t page_step = (uint32_t)c.page * d * c.heads;      // (entry: fits 31 bits)
    const int8_t *k_at = c.k + (uint32_t)(kvh * c.page * d), *v_at = c.v + (uint32_t)(kvh * c.page * d);
    v4i rk[kPer], rv[kPer];
    int kid[kPer], vid, sid;
    PageScales rs;
    const auto base_of = [&](int v) { return tile_base(rt.span, min(v, v1 - 1)); };
    const auto page_at = [&](int token) { return table[min(token, rt.pmax) >> c.page_log2]; };
    const auto ids_k = [&](int v) {
        const int base = base_of(v);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            kid[i] = page_at(base + (tid + i * kThreads) / kRowPieces % kTile);
        }
    };
    // (pieces of the values and scales: the thread's group of 16 tokens)
    const auto id_v = [&](int v) { return page_at(base_of(v) + tid % 4 * 16); };
    uint32_t koff[kPer], voff[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int piece = tid + i * kThreads, at = piece % kRowPieces * 16, ch = piece / 4;
        koff[i] = (uint32_t)(piece / kRowPieces % kTile * d + (at < d ? at : 0));
        voff[i] = (uint32_t)((ch < d ? ch : 0) * c.page + tid % 4 * 16);
    }
    int one_v = 0, one_k = 0;                      // kOne: page of the next values, of the next keys
    float one_ks = 0.0f, one_vs = 0.0f;            //       scales of the next softmax
    const auto one_page = [&](int v) { return uniform_load(table + (min(base_of(v), rt.pmax) >> c.page_log2)); };
    const auto load_k = [&](int v) {
        const int base = base_of(v);
        if constexpr (kOne) {
            const int8_t* page = k_at + readable(c, one_k) * (uint64_t)page_step + (uint32_t)((base & (c.page - 1)) * d);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                rk[i] = *reinterpret_cast<const v4i*>(page + koff[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int piece = tid + i * kThreads, slot = (base + piece / kRowPieces % kTile) & (c.page - 1);
                const int at = piece % kRowPieces * 16;
                rk[i] = *reinterpret_cast<const v4i*>(k_at + readable(c, kid[i]) * (uint64_t)page_step +
                                                      (uint32_t)(slot * d + (at < d ? at : 0)));
            }
        }
    };
    const auto load_scales = [&](int page) { rs = page_scales(c, page, kvh); };
    const auto load_v = [&](int v) {
        const int base = base_of(v);
        if constexpr (kOne) {
            const int8_t* page = v_at + readable(c, one_v) * (uint64_t)page_step + (uint32_t)(base & (c.page - 1));
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                rv[i] = *reinterpret_cast<const v4i*>(page + voff[i]);
            }
        } else {
            const int slot = (base + tid % 4 * 16) & (c.page - 1);
            const int8_t* page = v_at + readable(c, vid) * (uint64_t)page_step + (uint32_t)slot;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int ch = (tid + i * kThreads) / 4;
                rv[i] = *reinterpret_cast<const v4i*>(page + (uint32_t)((ch < d ? ch : 0) * c.page));
            }
        }
    };
    // (8 codes: half a piece)
    const auto put = [&](uint16_t* at, const v4i& w, int half) {
        const Vec x = half ? Op::codes((uint32_t)w.z, (uint32_t)w.w) : Op::codes((uint32_t)w.x, (uint32_t)w.y);
        __builtin_memcpy(__builtin_assume_aligned(at + 8 * half, 16), &x, 16);
    };
    const auto store_k = [&](int v, int i, int half) {
        const int piece = tid + i * kThreads;
        if (kPieces % kThreads == 0 || piece < kPieces) {
            put(s_k[v & 1] + piece / kRowPieces * kPitchK + piece % kRowPieces * 16, rk[i], half);
        }
    };
    const auto store_v = [&](int v, int i, int half) {
        const int piece = tid + i * kThreads;
        if (kPieces % kThreads == 0 || piece < kPieces) {
            put(s_v[v & 1] + piece / 4 * kPitchV + piece % 4 * 16, rv[i], half);
        }
    };
    const auto store_scales = [&](int v) {
        const Scales sc = softmax_scales(p, rs);
        s_scale[v & 3][tid % 4] = v4f{sc.mul, sc.add, sc.inv, 0.0f};   // (the same from many threads)
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
    };
    const auto soft = [&](auto masked, int v, int base) {
        constexpr bool kMasked = decltype(masked)::value;
        constexpr int kGroups = kOne ? 1 : 4, kSize = 32 / kGroups;   // values of a lane under one scale
        float mul[kGroups], add[kGroups], inv[kGroups];
        if constexpr (kOne) {
            const Scales sc = softmax_scales(p, PageScales{one_ks, one_vs, 0.0f});
            mul[0] = sc.mul;
            add[0] = sc.add;
            inv[0] = sc.inv;
        } else {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const v4f sc = s_scale[v & 3][g];
                mul[g] = sc.x;
                add[g] = sc.y;
                inv[g] = sc.z;
            }
        }
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
        // value i of a lane: token 16 (i / 8) + i % 8 of those. All ones or none
        const auto seen = [&](int i) {
            return (uint32_t)((int32_t)(bits[i / 16] << (31 - 16 * (i / 8 % 2) - i % 8)) >> 31);
        };
        float top = kNone;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            float t = kNone;
#pragma unroll
            for (int i = kSize * g; i < kSize * g + kSize; ++i) {
                float x = s[i / 16][i % 16];
                if (kMasked) {
                    const uint32_t m = seen(i);
                    x = __uint_as_float((__float_as_uint(x) & m) | (0xff800000u & ~m));
                }
                t = fmaxf(t, x);
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
        for (int g = 0; g < kGroups; ++g) {
            const float a = add[g] + shift;
            float sum = 0.0f;
#pragma unroll
            for (int h = kSize / 8 * g; h < kSize / 8 * (g + 1); ++h) {
                float w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h / 2][8 * (h % 2) + e], mul[g], a));
                    if (kMasked) {
                        w[e] = __uint_as_float(__float_as_uint(w[e]) & seen(8 * h + e));
                    }
                    sum += w[e];
                }
                Op::split(w, pf[h]);
            }
            // a page of which the row sees nothing adds nothing, whatever its scale
            l_run += !kMasked || sum != 0.0f ? sum * inv[g] : 0.0f;
        }
    };
    const auto rescale = [&] {
        if (renew) {
#pragma unroll
            for (int t = 0; t < kOut; ++t) {
                o[t] *= fresh;
            }
            renew = false;
        }
    };
    const auto accumulate = [&](int v) {
        const uint16_t* buf = s_v[v & 1] + n * kPitchV + 8 * hh;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
#pragma unroll
            for (int t = 0; t < kOut; ++t) {
                o[t] = product<T>(lds_vec(buf + 32 * t * kPitchV + 16 * g), pf[g], o[t]);
            }
        }
    };
    // accumulate(v - 1) and scores(v), each fragment read kAhead products before
    // its own, other work in `parts` between them: the order of reads and products
    // is fixed, vector instructions may move across.
    const auto both = [&](int v, auto work, auto parts) {
        constexpr int kFirst = 4 * kOut, kN = kFirst + 2 * kSteps, kAhead = 6;
        constexpr int kEvery = kN / (decltype(parts)::value + 1) > 0 ? kN / (decltype(parts)::value + 1) : 1;
        const uint16_t* bv = s_v[(v - 1) & 1] + n * kPitchV + 8 * hh;
        const uint16_t* bk = s_k[v & 1] + krow * kPitchK + 8 * hh;
        const auto fragment = [&](int i) {
            return i < kFirst ? lds_vec(bv + 32 * (i % kOut) * kPitchV + 16 * (i / kOut))
                              : lds_vec(bk + 32 * ((i - kFirst) % 2) * kPitchK + 16 * ((i - kFirst) / 2));
        };
        Vec f[kN];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            f[i] = fragment(i);
        }
        s[0] = v16f{};
        s[1] = v16f{};
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            if (i + kAhead < kN) {
                f[i + kAhead] = fragment(i + kAhead);
            }
            if (i < kFirst) {
                o[i % kOut] = product<T>(f[i], pf[i / kOut], o[i % kOut]);
            } else {
                s[(i - kFirst) % 2] = product<T>(f[i], qf[(i - kFirst) / 2], s[(i - kFirst) % 2]);
            }
            // (loads stay where they are: above the last use of what they replace,
            // they would need other registers, and a copy that waits for them)
            __builtin_amdgcn_sched_barrier(0x2 | 0x4 | 0x200);
            if (i % kEvery == kEvery - 1 && i / kEvery < decltype(parts)::value) {
                work(i / kEvery);
            }
        }
#pragma unroll
        for (int i = kN / kEvery; i < decltype(parts)::value; ++i) {
            work(i);
        }
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

    // Tiles in terms of 0 .. nt - 1.
    const int nt = v1 - v0, behind = kPair ? wave / 4 : 0;
    if (nt > 0) {
        // Step x of a thread: its pieces of the values of tile x and the keys of x
        // + 1 go into LDS, the next ones are asked for, then the page numbers of
        // those after. (Scales go with the keys.)
        constexpr int kParts = 4 * kPer + (kOne ? 2 : 4);
        const auto part = [&](int x, int i) {
            if (i < 2 * kPer) {
                store_v(x, i / 2, i % 2);
            } else if (i < 4 * kPer) {
                store_k(x + 1, i / 2 - kPer, i % 2);
            } else if (i == 4 * kPer) {
                if constexpr (!kOne) {
                    store_scales(x + 1);
                }
                load_v(v0 + x + 1);
            } else if (i == 4 * kPer + 1) {
                load_k(v0 + x + 2);
            } else if (i == 4 * kPer + 2) {
                load_scales(sid);
                vid = id_v(v0 + x + 2);
                sid = id_v(v0 + x + 3);
            } else {
                ids_k(v0 + x + 3);
            }
        };
        // kOne, between steps x and x + 1 (in the vector phase, where no LDS read is
        // in flight beside the scalar loads): the scales of tile x + 1, page numbers
        const auto one_step = [&](int x) {
            if constexpr (kOne) {
                const float off = exists(c, one_v) ? 0.0f : __uint_as_float(0x7fc00000u);
                const int64_t at = readable(c, one_v) * c.heads + kvh;
                one_ks = uniform_load(c.k_scale + at) + off;
                one_vs = uniform_load(c.v_scale + at) + off;
                one_v = one_k;
                one_k = one_page(v0 + x + 3);
            }
        };
        const auto step = [&](int x) {
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                part(x, i);
            }
        };
        if constexpr (kOne) {
            one_k = one_v = one_page(v0);
        } else {
            ids_k(v0);
            load_scales(id_v(v0));
            vid = id_v(v0);
        }
        load_k(v0);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            store_k(0, i, 0);
            store_k(0, i, 1);
        }
        if constexpr (!kOne) {
            store_scales(0);
        }
        load_v(v0);
        if constexpr (kOne) {
            one_step(-1);                          // scales of tile 0
            one_v = one_k = one_page(v0 + 1);
            load_k(v0 + 1);
            one_k = one_page(v0 + 2);
        } else {
            ids_k(v0 + 1);
            load_k(v0 + 1);
            load_scales(id_v(v0 + 1));
            vid = id_v(v0 + 1);
            sid = id_v(v0 + 2);
            ids_k(v0 + 2);
        }
        meet();
        if (behind) {
            meet();
        }
        // A wave multiplies tiles that it does not look at too (the last ones of a
        // tile of rows, and whole tiles outside a window): their weights are 0.
        // Without a branch in the matrix phase, pieces in flight need no copies.
        const auto weigh = [&](int j) {
            const int base = tile_base(rt.span, v0 + j);
            if (!live(base)) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
#pragma unroll
                    for (int i = 0; i < Op::kParts; ++i) {
                        pf[g][i] = Vec{};
                    }
                }
            } else if (open(base)) {
                soft(std::false_type{}, j, base);
            } else {
                soft(std::true_type{}, j, base);
            }
        };
        scores(0);
        step(0);
        meet();
        for (int j = 1; j < nt; ++j) {
            weigh(j - 1);
            one_step(j - 1);
            meet();
            rescale();
            __builtin_amdgcn_s_setprio(2);         // before the other wave's vector phase: 168.7 -> 158.5 us (a prompt of 4096)
            both(j, [&](int i) { part(j, i); }, std::integral_constant<int, kParts>{});
            __builtin_amdgcn_s_setprio(0);
            meet();
        }
        weigh(nt - 1);
        meet();
        rescale();
        accumulate(nt - 1);
        if (kPair && !behind) {
            meet();                                // as many as the others
        }
    }

    if (!is_row) {
        return;                                    // no barrier below
    }
    l_run += across(l_run);
    const int64_t token = seq.start + tok;
    if (rt.split) {
        const int64_t at_part = ((int64_t)split * c.rows + token) * p.q_heads + head;
        float* dst = p.part + at_part * d;
#pragma unroll
        for (int t = 0; t < kOut; ++t) {
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int ch = 32 * t + 8 * (r / 4) + 4 * hh;
                if (ch < d) {
                    *reinterpret_cast<v4f*>(dst + ch) = v4f{o[t][r], o[t][r + 1], o[t][r + 2], o[t][r + 3]};
                }
            }
        }
        if (hh == 0) {
            p.part_ml[2 * at_part] = m_run;
            p.part_ml[2 * at_part + 1] = l_run;
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

// Eight waves where their registers allow it and the rows fill more than four's
// (us, eight / four waves, 32 query and 8 KV heads; a prompt of 4096, d 128 150.7 /
// 249, d 64 107 / 122; 64 x 33 rows of 300 29.5 / 50.0; 24 sequences of 1 to 300 rows
// of 2500 121 / 177, d 64 99.6 / 97.9; f32, d 64, 64 x 64 of 300 38.5 / 54.4).
int tiled_rows(int64_t d, bool f16, int64_t page, int64_t rows)
{
    if (d > 128 && (!f16 || page < kTile)) {
        return 0;                                  // three parts of 256 channels: more registers than there are
    }
    if (d > (f16 ? 128 : 64)) {
        return 128;
    }
    return rows > 128 ? 256 : 128;
}

namespace {

template <typename T, int DP, int NW>
void launch_one(const AttnKern& k, const dim3& grid, hipStream_t s)
{
    if (DP > 128 || tiled_one_page(k.c.d, k.c.page)) {
        NNOPS_LAUNCH((attention_rows_tiled<T, DP, NW, true>), grid, dim3(64 * NW), 0, s, k);
    } else if constexpr (DP <= 128) {
        NNOPS_LAUNCH((attention_rows_tiled<T, DP, NW, false>), grid, dim3(64 * NW), 0, s, k);
    }
}

}  // namespace

void launch_tiled(const AttnKern& k, const dim3& grid, bool f16, hipStream_t s)
{
    const int d = k.c.d;
    if (f16 && k.tile_rows == 256) {
        d <= 64 ? launch_one<_Float16, 64, 8>(k, grid, s) : launch_one<_Float16, 128, 8>(k, grid, s);
    } else if (f16) {
        d <= 64    ? launch_one<_Float16, 64, 4>(k, grid, s)
        : d <= 128 ? launch_one<_Float16, 128, 4>(k, grid, s)
                   : launch_one<_Float16, 256, 4>(k, grid, s);
    } else if (k.tile_rows == 256) {
        launch_one<float, 64, 8>(k, grid, s);
    } else {
        d <= 64 ? launch_one<float, 64, 4>(k, grid, s) : launch_one<float, 128, 4>(k, grid, s);
    }
}

}  // namespace nnops_amd
