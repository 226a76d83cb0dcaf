// Attention for groups of sequences that share their first tokens: the kernels of
// cache_attention over those tokens, with all rows of a group as one sequence's
// (without a mask: every row sees them all), then over what each sequence has
// behind them, and the parts of every row joined:
//   out = sum_i 2^(M_i - M) O_i / sum_i 2^(M_i - M) l_i,  M = max M_i
//
// Bound: the codes are read once per group and tile of rows. A batch's single
// tokens that would read a prompt once per sequence become a tile of up to 256
// rows that the matrix cores bound.
//
// Which tokens are shared is found on the device: whole tiles and whole pages that
// every row of the group sees. Rows then need no mask, and a sequence's own tokens
// begin at a tile. Every wave finds it for few sequences (a launch less: 4 sequences over
// 2000 shared tokens 16 -> 12 us), one workgroup before the others for more.
// Probabilities of f16 rows are held in as many parts as CacheAttention has for the same
// rows, two f16 where it gives them workgroups of 16 and one where tiles of many: results
// differ by the order of the sums alone. With one f16 in every tile the calls below took
// 69 and 116 us, and were off by 2.3e-4 and 2.4e-4 of the result instead of 2.1e-4, as its
// own rounding to f16 is.
// Measured, 32 query and 8 KV heads of 128, f16: 64 sequences of a token each, 32768
// shared and up to 400 of their own: 78 us (each sequence by itself: 406), of which the
// shared tokens 62 (34.4 GFLOP, and 17 for the second parts) and the rest with the join 17 to
// 22; 530 rows over 8000: 135 (289).
#include "cache_attention_rows.hpp"
#include "cache_attention_tiled.hpp"

namespace nnops_amd {
namespace {

constexpr int kPlanThreads = 1024;

struct PrefixKern {
    PartKern own;
    int32_t* starts;      // workspace: group_starts, in order and in range
    int32_t ways;         // of the join: parts of a row that are summed side by side
};

// The largest of a workgroup's values, all 0 or more.
__device__ __forceinline__ int group_max(int v, int* s_waves)
{
    v = wave_max(v);
    __syncthreads();
    if (threadIdx.x % 64 == 0) {
        s_waves[threadIdx.x / 64] = v;
    }
    __syncthreads();
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        v = max(v, s_waves[w]);
    }
    return v;
}

__global__ __launch_bounds__(kPlanThreads) void prefix_plan(const PrefixKern p)
{
    __shared__ int s_waves[kPlanThreads / 64];
    const PartKern& k = p.own;
    const Paged& c = k.c;
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    // starts that do not go back
    int so_far = 0;
    for (int base = 0; base <= k.groups; base += kPlanThreads) {
        const int g = base + tid;
        int v = g <= k.groups ? min(max(k.group_starts[g], 0), c.seqs) : 0;
#pragma unroll
        for (int m = 1; m < 64; m *= 2) {
            const int before = __shfl_up(v, m);    // (by all lanes: one that takes no part gives nothing)
            v = lane >= m ? max(v, before) : v;
        }
        __syncthreads();
        if (lane == 63) {
            s_waves[wave] = v;
        }
        __syncthreads();
        int before = so_far;
        for (int w = 0; w < kPlanThreads / 64; ++w) {
            before = max(before, w < wave ? s_waves[w] : 0);
            so_far = max(so_far, s_waves[w]);
        }
        if (g <= k.groups) {
            p.starts[g] = max(v, before);
        }
    }
    for (int b = tid; b < c.seqs; b += kPlanThreads) {
        k.members[b] = MemberPlan{-1, 0};
    }
    __syncthreads();
    int longest = 0;
    for (int g = wave; g < k.groups; g += kPlanThreads / 64) {
        const int b0 = p.starts[g], b1 = p.starts[g + 1];
        GroupPlan plan{0, 0, 0, b0};
        int least = std::numeric_limits<int>::max(), first = c.rows, last = 0, len = 0;
        for (int b = b0 + lane; b < b1; b += 64) {
            const SeqRows s = seq_rows(c, b);
            if (s.n > 0) {
                least = min(least, s.len - s.n + 1);
                first = min(first, s.start);
                last = max(last, s.start + s.n);
            }
            len = b == b0 ? s.len : len;
        }
#pragma unroll
        for (int m = 1; m < 64; m *= 2) {
            least = min(least, __shfl_xor(least, m));
            first = min(first, __shfl_xor(first, m));
            last = max(last, __shfl_xor(last, m));
            len = max(len, __shfl_xor(len, m));
        }
        if (first < last) {
            plan.start = first;
            plan.rows = last - first;
            plan.tokens = shared_tokens(c, k.shared[g], len, least);
        }
        longest = max(longest, plan.tokens);
        if (lane == 0) {
            k.group_plan[g] = plan;
        }
        for (int b = b0 + lane; b < b1; b += 64) {
            k.members[b] = MemberPlan{g, plan.tokens / kTile};
        }
    }
    __syncthreads();
    int own = 0;
    for (int b = tid; b < c.seqs; b += kPlanThreads) {
        const SeqRows s = seq_rows(c, b);
        own = s.n > 0 ? max(own, s.len - kTile * k.members[b].skip) : own;
    }
    longest = group_max(longest, s_waves);
    own = group_max(own, s_waves);
    if (tid == 0) {
        *k.plan = PrefixPlan{chunk_for(longest / kTile, k.shared_splits, k.by_shared_splits, 4, k.shared_unit),
                             chunk_for(min((own + kTile - 1) / kTile, k.tiles), k.splits, k.by_splits, k.whole)};
    }
}

// Joins the parts of every row: lanes of 4 channels, `ways` of them a row, each
// with every ways-th part.
template <typename T>
__global__ __launch_bounds__(256) void prefix_join(const PrefixKern p)
{
    __shared__ WayParts sh;
    const PartKern& k = p.own;
    const Paged& c = k.c;
    const int lanes = join_lanes(c.d), slot = threadIdx.x / (uint32_t)lanes, ways = p.ways;
    const int way = slot % ways, per_block = 256 / lanes / ways;
    const int64_t i = (int64_t)blockIdx.x * per_block + slot / ways;
    const int token = (int)min(i / k.q_heads, (int64_t)c.rows - 1), qh = (int)(i % k.q_heads);
    bool live = i < (int64_t)c.rows * k.q_heads;
    RowTile rt;
    if (c.row_starts == nullptr) {
        rt.b = (int)((uint32_t)token / (uint32_t)c.uniform);
    } else {
        int lo = 0, hi = c.seqs;                   // the last sequence that starts at or before the row
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            (c.row_starts[mid] <= token ? lo : hi) = mid;
        }
        rt.b = lo;
    }
    rt.seq = seq_rows(c, rt.b);
    const int tok = token - rt.seq.start;
    live = live && tok >= 0 && tok < rt.seq.n;
    int shared = 0, own = 0;
    if (live) {
        const uint32_t row = (uint32_t)(tok * k.group) + (uint32_t)qh % (uint32_t)k.group;
        const int own_chunk = k.plan->own_chunk, shared_chunk = k.plan->shared_chunk;
        const int skip = k.members[rt.b].skip;
        place_tile<kOwn>(k, (int)(row / (uint32_t)k.tile_rows), own_chunk, rt, skip);
        shared = (int)(((uint32_t)skip + (uint32_t)shared_chunk - 1) / (uint32_t)shared_chunk);
        own = (int)(((uint32_t)rt.span.tiles + (uint32_t)own_chunk - 1) / (uint32_t)own_chunk);
    }
    const int ch = threadIdx.x % (uint32_t)lanes * 4;
    const int64_t at[1] = {(int64_t)token * k.q_heads + qh};
    float m[1] = {kNone}, l[1] = {0.0f};
    v4f o[1] = {v4f{0, 0, 0, 0}};
    join_parts<4>(k, at, ch, way, ways, shared + own, [&](int s) { return s < shared ? s : k.first_part + s - shared; }, m,
                  l, o);
    join_ways(sh, lanes, ways, m[0], l[0], o[0]);
    if (live && way == 0 && ch < c.d) {
        write_result<T>(k, token, qh, ch, l[0], o[0]);
    }
}

struct SharedPlan {
    AttnPlan own;
    int64_t items;        // tiles of the groups' rows, all KV heads
    int32_t tile_rows, per_seq, splits, ways;
    bool share;           // else: as CacheAttention, every sequence by itself
    bool few;             // every wave finds the plan
    bool join_here;       // own tokens, 16 rows a workgroup and unsplit: they join the parts themselves
    size_t groups_at, members_at, starts_at, parts_at, workspace;
};

NnopsCacheAttentionArgs whole_args(const NnopsPrefixAttentionArgs& g)
{
    NnopsCacheAttentionArgs a{};
    a.cache = g.cache;
    a.q = g.q;
    a.out = g.out;
    a.rows = g.rows;
    a.q_heads = g.q_heads;
    a.ld_q = g.ld_q;
    a.ld_out = g.ld_out;
    a.f16 = g.f16;
    a.scale = g.scale;
    return a;
}

int check_prefix(const NnopsPrefixAttentionArgs* g)
{
    if (g == nullptr || g->groups < 0) {
        return NNOPS_INVALID_ARGUMENT;
    }
    const NnopsCacheAttentionArgs a = whole_args(*g);
    if (const int rc = check_attention_shapes(&a); rc >= 0) {
        return rc;
    }
    return g->groups > (1 << 24) || g->cache.sequences > (1 << 24) ? NNOPS_UNSUPPORTED : -1;
}

size_t up16(size_t n) { return (n + 15) / 16 * 16; }

// Whether what is shared is read once, or each sequence looked at by itself, which the
// tables allow. Both are taken to read as many tokens as the table has room for (the host
// sees no lengths: in a table far wider than what is in use, as a captured graph has, more
// is shared than pays: 16 x up to 97 below, of 500 tokens in a table for 2000), a tile of rows at
// a time, and full or not, a tile takes the same time: sharing pays where it fills tiles
// that a sequence's rows fill in part, or makes them larger, and costs the parts of every
// row. The rates are those of the kernels, of a row, token and channel (and 64 more for
// the softmax; shared tiles whose probabilities are two f16 run at five sixths of it,
// which changes none of the choices below). Measured, by itself / shared in us, what is taken
// marked *; n sequences of r tokens, 32 query and 8 KV heads of 128, 500, 2000 and 8000
// shared tokens:
//   f16, 4 x 1     *9.9 / 11.0     *12.4 / 11.6    17.1 / *16.5
//        16 x 1    *11.7 / 11.2    18.6 / *14.9    34.3 / *21.2
//        48 x 1    15.9 / *15.2    30.2 / *20.6    77.6 / *35.0
//        48 x 3    *17.4 / 19.9    *31.5 / 33.8    78.9 / *59.5
//        48 x 8    *17.7 / 30.9    43.1 / *43.7    140 / *90.0
//        48 x 33   *40.6 / 63.5    *114 / 112      402 / *303
//        48 x 97   *71.7 / 159     *200 / 303      *709 / 776
//        16 x up to 97 *32.4 / 54.3 88.2 / *74.6  311 / *176
//   f32, 48 x 1    19.3 / *19.3    35.6 / *24.6    91.9 / *38.1
//        48 x 33   *97.6 / 115     302 / *238      1101 / *648
// Over 179 calls of such sizes and of 8 and 2 heads of 64, what is taken is 1 % slower than the
// faster one in the mean, 13 % if it always were the one or the other.
bool sharing_pays(const NnopsPrefixAttentionArgs& g, const SharedPlan& a)
{
    const double d = (double)g.cache.head_dim, seqs = (double)g.cache.sequences, groups = (double)g.groups;
    const double rows = (double)g.rows * g.q_heads / g.cache.heads;
    const double work = (double)g.cache.heads * (d + 64) * g.cache.table_pages * g.cache.page_tokens;
    const auto rate = [&](int tile) { return tile == kRows ? g.f16 ? 1.0e8 : 1.1e8 : g.f16 ? 4.5e8 : 1.35e8; };   // a us
    // rows that tiles hold, `of` in equal shares or of unknown ones
    const auto held = [&](double of, double tile, bool equal) {
        const double share = rows / of;
        return of * (equal ? __builtin_ceil(share / tile) * tile : share + tile / 2 > tile ? share + tile / 2 : tile);
    };
    const double part = 0.85e-6 * 4 * g.rows * g.q_heads * d;             // us, written and read
    const double alone = held(seqs, a.own.tile_rows, g.cache.row_starts == nullptr) * work / rate(a.own.tile_rows) +
                         (a.own.splits > 1 ? a.own.splits * part : 0);
    const double shared = held(groups, a.tile_rows, g.groups == 1) * work / rate(a.tile_rows) +
                          (a.splits + (a.join_here ? 0 : a.own.splits)) * part + 1.2;
    return shared < alone;
}

// Workgroups of the join.
int64_t join_blocks(const NnopsPrefixAttentionArgs& g, const SharedPlan& a)
{
    const int64_t per_block = 256 / join_lanes((int)g.cache.head_dim) / a.ways;
    return (g.rows * g.q_heads + per_block - 1) / per_block;
}

// Whether its launches hold what is shared (fewer than 2^31 threads each): larger
// calls are left to the other way, whose launches are fewer.
bool shared_way_fits(const NnopsPrefixAttentionArgs& g, const SharedPlan& a)
{
    constexpr int64_t kMost = INT32_MAX / 512;
    return a.own.items * a.own.splits <= kMost && a.items * a.splits <= kMost && a.own.splits <= 65535 &&
           a.splits <= 65535 && (a.join_here || join_blocks(g, a) <= INT32_MAX / 256);
}

SharedPlan shared_plan(const NnopsPrefixAttentionArgs* g)
{
    SharedPlan a{};
    const NnopsCacheAttentionArgs whole = whole_args(*g);
    a.own = attn_plan(&whole);
    const int64_t heads = g->cache.heads, group = g->q_heads / heads, d = g->cache.head_dim;
    if (g->groups == 0) {
        a.workspace = a.own.workspace;
        return a;
    }
    const int64_t groups = g->groups;
    const int64_t mean = (g->rows * group + groups - 1) / groups;
    // Tiles of many rows where they fill more than a quarter and there is work enough for
    // their longer beginning and end; 16 rows a workgroup otherwise, in one launch with
    // the sequences' own tokens (us, tiled / 16 rows; n sequences of one token, 32 query
    // and 8 KV heads of 128, f16; shared tokens 4096 and 32768): 16 28.6 / 19.0 and 55.4 /
    // 39.9, 24 29.7 / 23.0 and 57.9 / 54.2, 32 31.4 / 23.3 and 60.3 / 64.5, 48 37.7 / 27.7 and
    // 74.9 / 94.7; over 8192, 32 of them, d 64 27.0 / 18.8, d 256 60.0 / 62.8, f32 41.1 / 34.4.
    const int64_t room = g->cache.table_pages * g->cache.page_tokens;
    const bool much = (double)g->rows * g->q_heads * d * room >= 0x1p31;
    const int rows = mean > 64 && much ? tiled_rows(d, g->f16, g->cache.page_tokens, mean) : 0;
    a.tile_rows = rows > 0 ? rows : kRows;
    if (groups == 1) {
        a.per_seq = (int32_t)((g->rows * group + a.tile_rows - 1) / a.tile_rows);
        a.items = a.per_seq * heads;
    } else {
        a.items = (g->rows * group / a.tile_rows + (groups < g->rows ? groups : g->rows)) * heads;
    }
    const int64_t tiles = room / kTile;
    // Splits by rounds of the chip's workgroups: a round takes its tiles of tokens and
    // about `extra` tiles' time to begin, and to write its parts.
    const int64_t chip = rows > 0 ? 256 : 512, extra = 5, fine = 64;
    const int64_t most = (tiles + 3) / 4 < 4 * chip / a.items + 1 ? (tiles + 3) / 4 : 4 * chip / a.items + 1;
    a.splits = 1;
    int64_t best = INT64_MAX;
    for (int64_t n = 1; n <= most; ++n) {
        const int64_t cost = (a.items * n + chip - 1) / chip * (fine * tiles / n + fine * extra);
        if (cost < best) {
            best = cost;
            a.splits = (int32_t)n;
        }
    }
    a.few = g->cache.sequences <= 64 && g->groups <= kFewGroups;
    a.join_here = a.tile_rows != kRows && a.own.tile_rows == kRows && a.own.splits == 1;
    const int64_t parts = a.splits + (a.join_here ? 0 : a.own.splits);
    // workgroups to fill the chip, as long as each lane has a batch of parts
    const int lanes = join_lanes((int)d);
    a.ways = 1;
    while (a.ways < 256 / lanes && 4 * a.ways < parts && g->rows * g->q_heads * a.ways * lanes < 2048 * 256) {
        a.ways *= 2;
    }
    a.share = shared_way_fits(*g, a) && sharing_pays(*g, a);
    if (!a.share) {
        a.workspace = a.own.workspace;
        return a;
    }
    a.groups_at = 16;
    a.members_at = a.groups_at + up16(sizeof(GroupPlan) * (size_t)groups);
    a.starts_at = a.members_at + up16(sizeof(MemberPlan) * (size_t)g->cache.sequences);
    a.parts_at = a.starts_at + up16(4 * (size_t)(groups + 1));
    a.workspace = a.parts_at + (size_t)parts * g->rows * g->q_heads * (d + 2) * 4;
    return a;
}

template <typename T, int DP, int NW, AttnMode M, bool kFine>
void launch_tiled_one(const PartKern& k, const dim3& grid, hipStream_t s)
{
    if (DP > 128 || tiled_one_page(k.c.d, k.c.page)) {
        NNOPS_LAUNCH((attention_rows_tiled<T, DP, NW, true, M, kFine>), grid, dim3(64 * NW), 0, s, k);
    } else if constexpr (DP <= 128) {
        NNOPS_LAUNCH((attention_rows_tiled<T, DP, NW, false, M, kFine>), grid, dim3(64 * NW), 0, s, k);
    }
}

// (the kernels that tiled_rows names)
template <typename T, AttnMode M, bool kFine>
void launch_tiles(const PartKern& k, const dim3& grid, hipStream_t s)
{
    const int d = k.c.d;
    if constexpr (sizeof(T) == 2) {
        if (k.tile_rows == 256) {
            d <= 64 ? launch_tiled_one<T, 64, 8, M, kFine>(k, grid, s) : launch_tiled_one<T, 128, 8, M, kFine>(k, grid, s);
        } else {
            d <= 64    ? launch_tiled_one<T, 64, 4, M, kFine>(k, grid, s)
            : d <= 128 ? launch_tiled_one<T, 128, 4, M, kFine>(k, grid, s)
                       : launch_tiled_one<T, 256, 4, M, kFine>(k, grid, s);
        }
    } else if (k.tile_rows == 256) {
        launch_tiled_one<T, 64, 8, M, kFine>(k, grid, s);
    } else {
        d <= 64 ? launch_tiled_one<T, 64, 4, M, kFine>(k, grid, s) : launch_tiled_one<T, 128, 4, M, kFine>(k, grid, s);
    }
}

template <typename T, AttnMode M>
void launch_part(const PartKern& k, bool fine, const dim3& grid, hipStream_t s)
{
    const int d = k.c.d;
    if (k.tile_rows == kRows) {
        if (d <= 64) {
            NNOPS_LAUNCH((attention_rows16<T, 64, M>), grid, dim3(256), 0, s, k);
        } else if (d <= 128) {
            NNOPS_LAUNCH((attention_rows16<T, 128, M>), grid, dim3(256), 0, s, k);
        } else {
            NNOPS_LAUNCH((attention_rows16<T, 256, M>), grid, dim3(256), 0, s, k);
        }
    } else if (M == kShared && sizeof(T) == 2 && fine) {
        launch_tiles<T, M, M == kShared && sizeof(T) == 2>(k, grid, s);
    } else {
        launch_tiles<T, M, false>(k, grid, s);
    }
}

uint32_t reciprocal(int n) { return n > 1 ? (uint32_t)(((1ull << 32) + n - 1) / n) : 0; }

// Shared and own tokens in one launch, where both take 16 rows a workgroup: the first
// `shared` workgroups, `items` a split, and those behind them.
template <typename T, int DP>
__global__ __launch_bounds__(256, DP > 128 ? 1 : sizeof(T) == 2 ? 3 : 2) void attention_both16(
    const PartKern s, const PartKern o, uint32_t items, uint32_t shared, uint32_t own_items)
{
    __shared__ WaveParts<DP> sh;
    if (blockIdx.x < shared) {
        const uint32_t split = blockIdx.x / items;
        attend_rows16<T, DP, kShared>(s, sh, blockIdx.x - split * items, (int)split);
    } else {
        const uint32_t block = blockIdx.x - shared, split = block / own_items;
        attend_rows16<T, DP, kOwn>(o, sh, block - split * own_items, (int)split);
    }
}

template <typename T>
void launch_prefix(const PrefixKern& p, const SharedPlan& a, int64_t blocks, hipStream_t s)
{
    if (!p.own.few) {
        NNOPS_LAUNCH(prefix_plan, dim3(1), dim3(kPlanThreads), 0, s, p);
    }
    PartKern k = p.own;
    k.tile_rows = a.tile_rows;
    k.per_seq = a.per_seq;
    k.first_part = 0;
    const uint32_t shared = (uint32_t)(a.items * a.splits), own = (uint32_t)(a.own.items * a.own.splits);
    if (a.tile_rows == kRows && p.own.tile_rows == kRows) {
        const dim3 grid(shared + own);
        const uint32_t items = (uint32_t)a.items, own_items = (uint32_t)a.own.items;
        if (k.c.d <= 64) {
            NNOPS_LAUNCH((attention_both16<T, 64>), grid, dim3(256), 0, s, k, p.own, items, shared, own_items);
        } else if (k.c.d <= 128) {
            NNOPS_LAUNCH((attention_both16<T, 128>), grid, dim3(256), 0, s, k, p.own, items, shared, own_items);
        } else {
            NNOPS_LAUNCH((attention_both16<T, 256>), grid, dim3(256), 0, s, k, p.own, items, shared, own_items);
        }
    } else {
        // (probabilities in as many parts as CacheAttention has them in for the same rows)
        launch_part<T, kShared>(k, a.own.tile_rows == kRows, dim3((unsigned)a.items, (unsigned)a.splits), s);
        launch_part<T, kOwn>(p.own, false, dim3((unsigned)a.own.items, (unsigned)a.own.splits), s);
        if (p.own.join_here) {
            return;
        }
    }
    NNOPS_LAUNCH(prefix_join<T>, dim3((unsigned)blocks), dim3(256), 0, s, p);
}

}  // namespace
}  // namespace nnops_amd

using namespace nnops_amd;

extern "C" size_t nnops_hip_prefix_attention_workspace_size(const NnopsPrefixAttentionArgs* g)
{
    if (check_prefix(g) >= 0) {
        return 0;
    }
    const SharedPlan a = shared_plan(g);
    return a.share || launch_holds(a.own) ? a.workspace : 0;
}

extern "C" int nnops_hip_prefix_attention_plan(const NnopsPrefixAttentionArgs* g, NnopsPrefixAttentionPlan* out)
{
    if (out == nullptr) {
        return NNOPS_INVALID_ARGUMENT;
    }
    *out = NnopsPrefixAttentionPlan{};
    if (const int rc = check_prefix(g); rc >= 0) {
        return rc;
    }
    const SharedPlan a = shared_plan(g);
    if (!a.share && !launch_holds(a.own)) {
        return NNOPS_UNSUPPORTED;
    }
    out->own_rows = a.own.tile_rows;
    out->own_splits = a.own.splits;
    out->workspace_bytes = a.workspace;
    if (!a.share) {
        out->launches = 1 + (a.own.splits > 1);
        out->join = a.own.splits > 1;
        return NNOPS_OK;
    }
    const bool both = a.tile_rows == kRows && a.own.tile_rows == kRows;
    out->shared_rows = a.tile_rows;
    out->shared_splits = a.splits;
    out->launches = !a.few + (both ? 1 : 2) + !a.join_here;
    out->join = !a.join_here;
    return NNOPS_OK;
}

extern "C" int nnops_hip_prefix_attention(const NnopsPrefixAttentionArgs* g, void* workspace, size_t workspace_bytes,
                                          void* stream)
{
    const TimingDisarm disarm;
    if (const int rc = check_prefix(g); rc >= 0) {
        return rc;
    }
    if (const int rc = check_page_memory(g->cache); rc >= 0) {
        return rc;
    }
    const int64_t width = g->q_heads * g->cache.head_dim;
    if (g->q == nullptr || g->out == nullptr || g->ld_q < width || g->ld_out < width ||
        (g->groups > 0 && (g->group_starts == nullptr || g->shared == nullptr))) {
        return NNOPS_INVALID_ARGUMENT;
    }
    const SharedPlan a = shared_plan(g);
    if (!a.share) {
        const NnopsCacheAttentionArgs whole = whole_args(*g);
        return nnops_hip_cache_attention(&whole, workspace, workspace_bytes, stream);
    }
    if (workspace == nullptr || workspace_bytes < a.workspace || (uintptr_t)workspace % 16 != 0) {
        return NNOPS_NOT_INITIALIZED;
    }
    char* at = static_cast<char*>(workspace);
    PrefixKern p{};
    p.starts = reinterpret_cast<int32_t*>(at + a.starts_at);
    p.ways = a.ways;
    PartKern& k = p.own;
    k.c = paged(g->cache, g->rows);
    k.q = g->q;
    k.out = g->out;
    k.ld_q = g->ld_q;
    k.ld_out = g->ld_out;
    k.part = reinterpret_cast<float*>(at + a.parts_at);
    k.part_ml = k.part + (size_t)(a.splits + (a.join_here ? 0 : a.own.splits)) * g->rows * g->q_heads * g->cache.head_dim;
    const float scale = g->scale > 0.0f ? g->scale : 1.0f / __builtin_sqrtf((float)g->cache.head_dim);
    k.scale_log2 = scale * 1.4426950408889634f;
    k.q_heads = (int32_t)g->q_heads;
    k.group = (int32_t)(g->q_heads / g->cache.heads);
    k.tile_rows = a.own.tile_rows;
    k.per_seq = a.own.per_seq;
    k.splits = a.own.splits;
    k.by_splits = reciprocal(a.own.splits);
    k.tiles = a.own.tiles;
    k.whole = a.own.whole;
    k.chunk = a.own.chunk;
    k.plan = reinterpret_cast<PrefixPlan*>(at);
    k.group_plan = reinterpret_cast<GroupPlan*>(at + a.groups_at);
    k.members = reinterpret_cast<MemberPlan*>(at + a.members_at);
    k.group_starts = g->group_starts;
    k.shared = g->shared;
    k.few = a.few;
    k.join_here = a.join_here;
    k.shared_splits = a.splits;
    k.shared_unit = a.tile_rows == kRows ? 4 : 1;
    k.by_shared_splits = reciprocal(a.splits);
    k.groups = (int32_t)g->groups;
    k.first_part = a.splits;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (g->f16) {
        launch_prefix<_Float16>(p, a, join_blocks(*g, a), s);
    } else {
        launch_prefix<float>(p, a, join_blocks(*g, a), s);
    }
    return hipGetLastError() == hipSuccess ? NNOPS_OK : NNOPS_INTERNAL;
}
