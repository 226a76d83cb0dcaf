// Page tables of a paged cache: continuations of sequences (fork), the pages in
// use moved together (compact), and the copying of pages that both ask for.
//
// Counts are whole numbers: they may be added in any order, and the same inputs
// give the same tables. What has an order (which child keeps a page, which free
// page goes to which cell) is taken from prefix sums.
//
// Bound: launches, and chains of loads and barriers; copying, HBM. One workgroup
// does all of a fork or compact whose counts fit in LDS and whose cells are few (us,
// with the copies' launch, one / several launches; n sequences in pages of 64: fork 64
// of 1500 11.9 / 16.0, 128 of 4000 17.4 / 16.2, 256 of 4000 27.1 / 15.8; compact 64 of
// 1500 11.7 / 16.3, 128 of 4000 19.4 / 17.2, 256 of 4000 33.0 / 21.4).
#include "common.hpp"
#include "paged.hpp"

namespace nnops_amd {
namespace {

constexpr int kPlan = 1024;         // threads of the workgroup that hands pages out
constexpr int kMostRows = 16384;    // children whose offsets lie in LDS

__device__ __forceinline__ int pages_of(int tokens, int page_log2)
{
    return (int)(((uint32_t)tokens + (1u << page_log2) - 1) >> page_log2);
}

// The sum of the lanes before, and of all in `total`.
__device__ __forceinline__ int wave_before(int v, int& total)
{
    const int lane = threadIdx.x % 64;
    int upto = v;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        const int other = __shfl_up(upto, m);
        upto += lane >= m ? other : 0;
    }
    total = __shfl(upto, 63);
    return upto - v;
}

__device__ __forceinline__ int wave_max(int v)
{
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        v = max(v, __shfl_xor(v, m));
    }
    return v;
}

// The same over a workgroup of kPlan threads; s_waves: one int a wave. Every
// thread calls it, with a barrier before the next call's.
__device__ __forceinline__ int group_before(int v, int* s_waves, int& total)
{
    const int wave = threadIdx.x / 64;
    int mine;
    int before = wave_before(v, mine);
    if (threadIdx.x % 64 == 0) {
        s_waves[wave] = mine;
    }
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < kPlan / 64; ++w) {
        before += w < wave ? s_waves[w] : 0;
        total += s_waves[w];
    }
    __syncthreads();
    return before;
}

// A bit for each of the 16 pages from `at` on that is held.
__device__ __forceinline__ uint32_t held_bits(const int32_t* refs, int at, int pages)
{
    int n[16] = {};
    if (at + 16 <= pages) {
        __builtin_memcpy(n, refs + at, sizeof n);
    } else {
        for (int e = 0; e < 16 && at + e < pages; ++e) {
            n[e] = refs[at + e];
        }
    }
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        bits |= (uint32_t)(n[e] != 0) << e;
    }
    return bits;
}

// --- fork ----------------------------------------------------------------------

// What a child takes: `fresh` pages from cell `kept` on; tail: the page before
// them that it will write into, kNoTail where it writes into none, kNoPage where
// the cell holds none (it gets a fresh one, nothing is copied).
constexpr int kNoTail = -1, kNoPage = -2;
struct Child {
    int kept, fresh, tail;
};

struct ForkKern {
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* refs;
    const int32_t* parents;
    const int32_t* new_tokens;
    int32_t* new_table;
    int32_t* new_lengths;
    int32_t* new_refs;
    int32_t* copies;
    int32_t* counts;
    int64_t ld_table, ld_new;
    int32_t seqs, table_pages, pages, page_log2, children, new_pages, chunks;
    int32_t* writers;     // workspace: children that will write into a page
    int32_t* first;       //   and the first of them
    int32_t* free;        //   free pages, as many as are asked for
    Child* child;
};

__device__ __forceinline__ int length_of(const ForkKern& p, int b)
{
    return (int)min((int64_t)max(p.lengths[b], 0), (int64_t)p.table_pages << p.page_log2);
}

// A child's parent (-1: none), the tokens that it keeps and those it has room for.
__device__ __forceinline__ void tokens_of(const ForkKern& p, int i, int& parent, int& kept, int& will)
{
    parent = p.parents[i];
    parent = (uint32_t)parent < (uint32_t)p.seqs ? parent : -1;
    const int had = parent >= 0 ? length_of(p, parent) : 0;
    const int64_t most = (int64_t)p.new_pages << p.page_log2;
    will = (int)min(max((int64_t)had + p.new_tokens[i], (int64_t)0), most);
    kept = min(had, will);
}

__global__ __launch_bounds__(256) void fork_clear(const ForkKern p)
{
    const int at = (int)(blockIdx.x * 256 + threadIdx.x);
    if (at < p.pages) {
        p.new_refs[at] = p.refs[at];              // (the same array, or another)
        p.writers[at] = 0;
        p.first[at] = p.children;
    }
}

// A wave has 256 cells of a row: of an old one, whose pages are given up, or of a
// child's, which holds the parent's from now on.
__global__ __launch_bounds__(256) void fork_hold(const ForkKern p)
{
    const int lane = threadIdx.x % 64;
    const uint32_t item = blockIdx.x * 4 + threadIdx.x / 64;
    const int row = (int)(item / (uint32_t)p.chunks), c0 = (int)(item - (uint32_t)row * p.chunks) * 256;
    if (row >= p.seqs + p.children) {
        return;
    }
    if (row < p.seqs) {
        const int held = pages_of(length_of(p, row), p.page_log2);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int c = c0 + 64 * e + lane;
            if (c < held) {
                const int id = p.table[row * p.ld_table + c];
                if ((uint32_t)id < (uint32_t)p.pages) {
                    atomicSub(&p.new_refs[id], 1);
                }
            }
        }
        return;
    }
    const int i = row - p.seqs;
    int parent, kept, will;
    tokens_of(p, i, parent, kept, will);
    const int shared = pages_of(kept, p.page_log2);
    const bool writes = will > kept && (kept & ((1 << p.page_log2) - 1)) != 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int c = c0 + 64 * e + lane;
        int id = -1;
        if (c < shared) {
            id = p.table[parent * p.ld_table + c];
            id = (uint32_t)id < (uint32_t)p.pages ? id : -1;
            if (id >= 0) {
                atomicAdd(&p.new_refs[id], 1);
            }
            if (writes && c == shared - 1) {
                if (id >= 0) {
                    atomicAdd(&p.writers[id], 1);
                    atomicMin(&p.first[id], i);
                }
                p.child[i].tail = id >= 0 ? id : kNoPage;
            }
        }
        if (c < p.new_pages) {
            p.new_table[i * p.ld_new + c] = id;
        }
    }
    if (c0 == 0 && lane == 0) {
        p.new_lengths[i] = will;
        p.child[i].kept = shared;
        p.child[i].fresh = pages_of(will, p.page_log2) - shared;
        if (!writes) {
            p.child[i].tail = kNoTail;
        }
        p.copies[2 * i] = -1;
        p.copies[2 * i + 1] = -1;
    }
}

// Hands out the free pages: one workgroup, whose threads take a child each, then
// 16 pages each (100000 pages are 7 steps), then a cell each. 500 sequences and 24000
// pages: 10 us (a lane's pages 64 apart and ballots, all loads in flight: 11.3; four cells'
// chains side by side: 13).
__global__ __launch_bounds__(kPlan) void fork_take(const ForkKern p)
{
    __shared__ int s_at[kMostRows + 1];            // a child's first in the list of free pages
    __shared__ uint8_t s_tail[kMostRows];          // 0: no page before its fresh ones, 1: copied, 2: fresh
    __shared__ int s_waves[kPlan / 64];
    const int tid = threadIdx.x;
    int want = 0;
    for (int base = 0; base < p.children; base += kPlan) {
        const int i = base + tid;
        int n = 0;
        if (i < p.children) {
            const Child c = p.child[i];
            int kind = c.tail == kNoPage ? 2 : 0;
            if (c.tail >= 0) {
                kind = p.new_refs[c.tail] <= p.writers[c.tail] && p.first[c.tail] == i ? 0 : 1;
            }
            n = c.fresh + (kind != 0);
            s_tail[i] = (uint8_t)kind;
        }
        int total;
        const int before = group_before(n, s_waves, total);
        if (i < p.children) {
            s_at[i] = want + before;
        }
        want += total;
    }
    int found = 0;
    for (int base = 0; base < p.pages; base += 16 * kPlan) {
        const int at = base + 16 * tid;
        const int there = min(max(p.pages - at, 0), 16);
        uint32_t zero = ~held_bits(p.new_refs, at, p.pages) & ((1u << there) - 1);
        int total;
        int rank = found + group_before(__popc(zero), s_waves, total);
        while (zero != 0 && rank < want) {
            p.free[rank++] = at + __ffs(zero) - 1;
            zero &= zero - 1;
        }
        found += total;
    }
    __syncthreads();                               // (the list, and all counts looked at before they change)
    const int got = min(want, found);
    for (int r = tid; r < want; r += kPlan) {
        int lo = 0, hi = p.children;               // the last child that begins at or before r
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            (s_at[mid] <= r ? lo : hi) = mid;
        }
        const Child c = p.child[lo];
        const int k = r - s_at[lo], kind = s_tail[lo];
        const int page = r < got ? p.free[r] : -1;
        p.new_table[lo * p.ld_new + c.kept + k - (kind != 0)] = page;
        if (page >= 0) {
            p.new_refs[page] = 1;
        }
        if (kind == 1 && k == 0) {
            atomicSub(&p.new_refs[c.tail], 1);
            p.copies[2 * lo] = page >= 0 ? c.tail : -1;
            p.copies[2 * lo + 1] = page;
        }
    }
    if (tid == 0) {
        p.counts[0] = found - got;
        p.counts[1] = want - got;
    }
}

// The same by one workgroup, counts and lists in LDS: four cells a thread and step
// (64 sequences of 1500: 6.6 us).
constexpr int kSmallPages = 12288, kSmallRows = 1024, kSmallCells = 12288;

__global__ __launch_bounds__(kPlan) void fork_small(const ForkKern p)
{
    __shared__ int s_refs[kSmallPages];
    __shared__ int s_list[kSmallPages];            // writers, then the first of them, then the free pages
    __shared__ int s_held[kSmallRows], s_parent[kSmallRows], s_shared[kSmallRows], s_fresh[kSmallRows];
    __shared__ int s_tail[kSmallRows], s_at[kSmallRows + 1];
    __shared__ uint8_t s_kind[kSmallRows], s_writes[kSmallRows];
    __shared__ int s_waves[kPlan / 64];
    const int tid = threadIdx.x;
    for (int i = tid; i < p.pages; i += kPlan) {
        s_refs[i] = p.refs[i];
        s_list[i] = 0;
    }
    int held = 0;
    if (tid < p.seqs) {
        held = pages_of(length_of(p, tid), p.page_log2);
        s_held[tid] = held;
    }
    if (tid < p.children) {
        int parent, kept, will;
        tokens_of(p, tid, parent, kept, will);
        const int shared = pages_of(kept, p.page_log2);
        s_parent[tid] = parent;
        s_shared[tid] = shared;
        s_fresh[tid] = pages_of(will, p.page_log2) - shared;
        s_writes[tid] = will > kept && (kept & ((1 << p.page_log2) - 1)) != 0;
        s_tail[tid] = kNoTail;
        p.new_lengths[tid] = will;
    }
    held = wave_max(held);
    if (tid % 64 == 0) {
        s_waves[tid / 64] = held;
    }
    __syncthreads();
    int most = 0;                                  // pages of the longest
    for (int w = 0; w < kPlan / 64; ++w) {
        most = max(most, s_waves[w]);
    }
    const uint32_t old_cells = (uint32_t)p.seqs * most, new_cells = (uint32_t)p.children * p.new_pages;
    for (uint32_t base = 0; base < old_cells + new_cells; base += 4 * kPlan) {
        int row[4], col[4], id[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t i = base + e * kPlan + tid;
            const bool old = i < old_cells;
            const uint32_t j = old ? i : i - old_cells, wide = old ? (uint32_t)most : (uint32_t)p.new_pages;
            row[e] = -1;
            id[e] = -1;
            if (i < old_cells + new_cells) {
                const int r = (int)(j / wide);
                col[e] = (int)(j - r * wide);
                row[e] = old ? r : p.seqs + r;
                const int from = old ? r : s_parent[r];
                if (col[e] < (old ? s_held[r] : s_shared[r])) {
                    id[e] = p.table[from * p.ld_table + col[e]];
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int page = (uint32_t)id[e] < (uint32_t)p.pages ? id[e] : -1;
            const int i = row[e] - p.seqs;
            if (row[e] >= 0 && i < 0) {
                if (page >= 0) {
                    atomicSub(&s_refs[page], 1);
                }
            } else if (i >= 0) {
                if (page >= 0) {
                    atomicAdd(&s_refs[page], 1);
                }
                if (s_writes[i] && col[e] == s_shared[i] - 1) {
                    s_tail[i] = page >= 0 ? page : kNoPage;
                    if (page >= 0) {
                        atomicAdd(&s_list[page], 1);
                    }
                }
                p.new_table[i * p.ld_new + col[e]] = page;
            }
        }
    }
    __syncthreads();
    const int tail = tid < p.children ? s_tail[tid] : kNoTail;
    const bool alone = tail >= 0 && s_refs[tail] <= s_list[tail];
    __syncthreads();
    if (tail >= 0) {
        s_list[tail] = p.children;
    }
    __syncthreads();
    if (tail >= 0) {
        atomicMin(&s_list[tail], tid);
    }
    __syncthreads();
    const int kind = tail == kNoPage ? 2 : tail >= 0 && !(alone && s_list[tail] == tid) ? 1 : 0;
    int want;
    const int at = group_before(tid < p.children ? s_fresh[tid] + (kind != 0) : 0, s_waves, want);
    if (tid < p.children) {
        s_at[tid] = at;
        s_kind[tid] = (uint8_t)kind;
        if (kind != 1) {                           // (else by the thread that has the fresh page)
            p.copies[2 * tid] = -1;
            p.copies[2 * tid + 1] = -1;
        }
    }
    const int share = (p.pages + kPlan - 1) / kPlan, first = min(share * tid, p.pages), end = min(first + share, p.pages);
    int free = 0;
    for (int i = first; i < end; ++i) {
        free += s_refs[i] == 0;
    }
    int found;
    int rank = group_before(free, s_waves, found);
    for (int i = first; i < end && rank < want; ++i) {
        if (s_refs[i] == 0) {
            s_list[rank++] = i;
        }
    }
    __syncthreads();
    const int got = min(want, found);
    for (int r = tid; r < want; r += kPlan) {
        int lo = 0, hi = p.children;               // the last child that begins at or before r
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            (s_at[mid] <= r ? lo : hi) = mid;
        }
        const int k = r - s_at[lo], page = r < got ? s_list[r] : -1;
        p.new_table[lo * p.ld_new + s_shared[lo] + k - (s_kind[lo] != 0)] = page;
        if (page >= 0) {
            s_refs[page] = 1;
        }
        if (s_kind[lo] == 1 && k == 0) {
            atomicSub(&s_refs[s_tail[lo]], 1);
            p.copies[2 * lo] = page >= 0 ? s_tail[lo] : -1;
            p.copies[2 * lo + 1] = page;
        }
    }
    __syncthreads();
    for (int i = tid; i < p.pages; i += kPlan) {
        p.new_refs[i] = s_refs[i];
    }
    if (tid == 0) {
        p.counts[0] = found - got;
        p.counts[1] = want - got;
    }
}

// --- compact ---------------------------------------------------------------------

constexpr int kBlock = 4096;        // pages of a workgroup, 16 a thread

struct CompactKern {
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* refs;
    int32_t* new_table;
    int32_t* new_refs;
    int32_t* copies;
    int32_t* moved;
    int32_t* counts;
    int64_t ld_table, ld_new;
    int32_t seqs, table_pages, pages, page_log2, blocks, chunks;
    int32_t* used;        // workspace: pages in use, by blocks
    int32_t* code;        //   of a page: itself where it stays, -1 if it is free, -2 - i for the i-th that moves
};

__global__ __launch_bounds__(256) void compact_count(const CompactKern p)
{
    __shared__ int s_waves[4];
    int total;
    wave_before(__popc(held_bits(p.refs, (int)blockIdx.x * kBlock + 16 * (int)threadIdx.x, p.pages)), total);
    if (threadIdx.x % 64 == 0) {
        s_waves[threadIdx.x / 64] = total;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        p.used[blockIdx.x] = (s_waves[0] + s_waves[1]) + (s_waves[2] + s_waves[3]);
    }
}

// Pages in use before a thread's 16, among the block's: every thread of the
// workgroup calls it.
__device__ __forceinline__ int used_before(uint32_t bits, int* s_waves)
{
    int total;
    int before = wave_before(__popc(bits), total);
    if (threadIdx.x % 64 == 0) {
        s_waves[threadIdx.x / 64] = total;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        before += w < (int)threadIdx.x / 64 ? s_waves[w] : 0;
    }
    return before;
}

// Who moves where, by ranks: a free page at j below U is number j - (used before
// j) of those, a used one at j from U on number (used before j) - (used below U).
__global__ __launch_bounds__(256) void compact_rank(const CompactKern p)
{
    __shared__ int s_waves[4];
    __shared__ int s_sums[4][3];
    const int tid = threadIdx.x, block = blockIdx.x;
    int all = 0, before = 0;
    for (int b = tid; b < p.blocks; b += 256) {
        const int n = p.used[b];
        all += n;
        before += b < block ? n : 0;
    }
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        all += __shfl_xor(all, m);
        before += __shfl_xor(before, m);
    }
    if (tid % 64 == 0) {
        s_sums[tid / 64][0] = all;
        s_sums[tid / 64][1] = before;
    }
    __syncthreads();
    const int u = (s_sums[0][0] + s_sums[1][0]) + (s_sums[2][0] + s_sums[3][0]);
    before = (s_sums[0][1] + s_sums[1][1]) + (s_sums[2][1] + s_sums[3][1]);
    // used pages below U: the blocks before U's, and those of its block
    const int edge = u / kBlock;
    int below = 0;
    for (int b = tid; b < min(edge, p.blocks); b += 256) {
        below += p.used[b];
    }
    const int at_edge = edge * kBlock + 16 * tid;
    const uint32_t edge_bits = held_bits(p.refs, at_edge, p.pages);
    const int take = min(max(u - at_edge, 0), 16);
    below += __popc(edge_bits & ((1u << take) - 1));
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        below += __shfl_xor(below, m);
    }
    if (tid % 64 == 0) {
        s_sums[tid / 64][2] = below;
    }
    __syncthreads();
    below = (s_sums[0][2] + s_sums[1][2]) + (s_sums[2][2] + s_sums[3][2]);
    const int moves = u - below;
    const int at = block * kBlock + 16 * tid;
    const uint32_t bits = held_bits(p.refs, at, p.pages);
    int rank = before + used_before(bits, s_waves);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int j = at + e;
        const bool is = (bits >> e & 1) != 0;
        if (j < p.pages) {
            if (is && j >= u) {
                p.copies[2 * (rank - below)] = j;
            } else if (!is && j < u) {
                p.copies[2 * (j - rank) + 1] = j;
            }
            p.code[j] = !is ? -1 : j < u ? j : -2 - (rank - below);
        }
        rank += is;
    }
    // the rows behind the moves
    for (int i = block * 256 + tid; i < p.pages / 2; i += 256 * p.blocks) {
        if (i >= moves) {
            p.copies[2 * i] = -1;
            p.copies[2 * i + 1] = -1;
        }
    }
    if (block == 0 && tid == 0) {
        p.counts[0] = u;
        p.counts[1] = moves;
    }
}

__device__ __forceinline__ int new_number(const CompactKern& p, int page)
{
    const int code = p.code[page];
    return code >= -1 ? code : p.copies[2 * (-2 - code) + 1];
}

__global__ __launch_bounds__(256) void compact_apply(const CompactKern p)
{
    const int lane = threadIdx.x % 64;
    const int page_blocks = (p.pages + 255) / 256;
    if ((int)blockIdx.x < page_blocks) {
        const int j = (int)blockIdx.x * 256 + (int)threadIdx.x;
        if (j < p.pages) {
            // (of one array in place: a page that moves is written by the thread that read
            // it, and nobody else touches the number that it goes to)
            const int u = p.counts[0], to = new_number(p, j), refs = p.refs[j];
            p.moved[j] = to;
            if (to >= 0) {
                p.new_refs[to] = refs;
            }
            if (j >= u) {
                p.new_refs[j] = 0;
            }
        }
        return;
    }
    const uint32_t item = (blockIdx.x - page_blocks) * 4 + threadIdx.x / 64;
    const int row = (int)(item / (uint32_t)p.chunks), c0 = (int)(item - (uint32_t)row * p.chunks) * 256;
    if (row >= p.seqs) {
        return;
    }
    const int64_t len = min((int64_t)max(p.lengths[row], 0), (int64_t)p.table_pages << p.page_log2);
    const int held = pages_of((int)len, p.page_log2);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int c = c0 + 64 * e + lane;
        if (c < p.table_pages) {
            const int id = c < held ? p.table[row * p.ld_table + c] : -1;
            p.new_table[row * p.ld_new + c] = (uint32_t)id < (uint32_t)p.pages ? new_number(p, id) : -1;
        }
    }
}

// The same by one workgroup: 16 pages a thread, their counts in its registers.
constexpr int kCompactPages = 16 * kPlan, kCompactCells = 6144;

__global__ __launch_bounds__(kPlan) void compact_small(const CompactKern p)
{
    __shared__ int s_code[kCompactPages];          // new numbers, -1 for a free page
    __shared__ int s_to[kCompactPages / 2];        // where the i-th page that moves goes
    __shared__ int s_waves[kPlan / 64];
    const int tid = threadIdx.x, at = 16 * tid;
    int refs[16];
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        refs[e] = 0;
    }
    if (at + 16 <= p.pages) {
        __builtin_memcpy(refs, p.refs + at, sizeof refs);
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            if (at + e < p.pages) {
                refs[e] = p.refs[at + e];
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        bits |= (uint32_t)(refs[e] != 0) << e;
    }
    int u, below;
    const int before = group_before(__popc(bits), s_waves, u);
    group_before(__popc(bits & ((1u << min(max(u - at, 0), 16)) - 1)), s_waves, below);
    const int moves = u - below;
    int rank = before;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int j = at + e;
        const bool is = (bits >> e & 1) != 0;
        if (!is && j < u) {
            s_to[j - rank] = j;
        }
        rank += is;
    }
    __syncthreads();
    rank = before;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int j = at + e;
        const bool is = (bits >> e & 1) != 0;
        if (j < p.pages) {
            int to = is ? j : -1;
            if (is && j >= u) {
                to = s_to[rank - below];
                p.copies[2 * (rank - below)] = j;
                p.copies[2 * (rank - below) + 1] = to;
            }
            s_code[j] = to;
            if (to >= 0) {
                p.new_refs[to] = refs[e];
            }
            if (j >= u) {
                p.new_refs[j] = 0;
            }
        }
        rank += is;
    }
    for (int i = moves + tid; i < p.pages / 2; i += kPlan) {
        p.copies[2 * i] = -1;
        p.copies[2 * i + 1] = -1;
    }
    if (tid == 0) {
        p.counts[0] = u;
        p.counts[1] = moves;
    }
    __syncthreads();
    for (int j = tid; j < p.pages; j += kPlan) {
        p.moved[j] = s_code[j];
    }
    const uint32_t cells = (uint32_t)p.seqs * p.table_pages;
    for (uint32_t base = 0; base < cells; base += 4 * kPlan) {
        int row[4], col[4], id[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t i = base + e * kPlan + tid;
            row[e] = -1;
            id[e] = -1;
            if (i < cells) {
                row[e] = (int)(i / (uint32_t)p.table_pages);
                col[e] = (int)(i - (uint32_t)row[e] * p.table_pages);
                const int64_t len = min((int64_t)max(p.lengths[row[e]], 0), (int64_t)p.table_pages << p.page_log2);
                if (col[e] < pages_of((int)len, p.page_log2)) {
                    id[e] = p.table[row[e] * p.ld_table + col[e]];
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (row[e] >= 0) {
                p.new_table[row[e] * p.ld_new + col[e]] = (uint32_t)id[e] < (uint32_t)p.pages ? s_code[id[e]] : -1;
            }
        }
    }
}

// --- copy ------------------------------------------------------------------------

constexpr int kPiece = 16384;       // bytes of a workgroup, four 16-byte loads a thread in flight

struct CopyKern {
    int8_t* k;
    int8_t* v;
    float* k_scale;
    float* v_scale;
    const int32_t* copies;
    int64_t page_bytes;   // of a side
    int32_t pages, heads, pieces;
};

// A workgroup copies a piece of a page's side, stored past the caches. Bound: HBM: 89
// MB of pages of 131 KB in 31 us, 5.8 TB/s both ways (38.8 with plain stores; pieces
// of 32 KB 54, of 8 KB the same, of 4 KB 34).
__global__ __launch_bounds__(256) void kv_copy(const CopyKern p)
{
    const int i = (int)(blockIdx.x / (uint32_t)(2 * p.pieces));
    const int piece = (int)(blockIdx.x - (uint32_t)i * (2 * p.pieces));
    const int from = p.copies[2 * i], to = p.copies[2 * i + 1];
    if ((uint32_t)from >= (uint32_t)p.pages || (uint32_t)to >= (uint32_t)p.pages || from == to) {
        return;
    }
    const bool values = piece >= p.pieces;
    const int64_t at = (int64_t)(piece - (values ? p.pieces : 0)) * kPiece;
    int8_t* side = values ? p.v : p.k;
    const v4i* src = reinterpret_cast<const v4i*>(side + from * p.page_bytes + at);
    v4i* dst = reinterpret_cast<v4i*>(side + to * p.page_bytes + at);
    const int n = (int)(min(p.page_bytes - at, (int64_t)kPiece) / 16);
    v4i x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int j = 256 * e + (int)threadIdx.x;
        if (j < n) {
            x[e] = src[j];
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int j = 256 * e + (int)threadIdx.x;
        if (j < n) {
            __builtin_nontemporal_store(x[e], dst + j);
        }
    }
    if (at == 0) {
        float* scale = values ? p.v_scale : p.k_scale;
        for (int h = threadIdx.x; h < p.heads; h += 256) {
            scale[(int64_t)to * p.heads + h] = scale[(int64_t)from * p.heads + h];
        }
    }
}

// --- the calls ---------------------------------------------------------------------

bool page_tokens_fit(int64_t t) { return t == 16 || t == 32 || t == 64 || t == 128 || t == 256; }

int check_fork(const NnopsKvForkArgs* g)
{
    if (g == nullptr || g->sequences < 0 || g->table_pages < 0 || g->pages < 0 || g->children < 0 ||
        g->new_table_pages < 0) {
        return NNOPS_INVALID_ARGUMENT;
    }
    if (!page_tokens_fit(g->page_tokens) || g->sequences > kMostRows || g->children > kMostRows ||
        g->pages > INT32_MAX / 4 || g->table_pages > INT32_MAX / g->page_tokens ||
        g->new_table_pages > INT32_MAX / g->page_tokens || g->children * g->new_table_pages > INT32_MAX / 2) {
        return NNOPS_UNSUPPORTED;                  // (what all ask for is an int)
    }
    return -1;
}

int check_compact(const NnopsKvCompactArgs* g)
{
    if (g == nullptr || g->sequences < 0 || g->table_pages < 0 || g->pages < 0) {
        return NNOPS_INVALID_ARGUMENT;
    }
    if (!page_tokens_fit(g->page_tokens) || g->sequences > INT32_MAX / 2 || g->pages > INT32_MAX / 4 ||
        g->table_pages > INT32_MAX / g->page_tokens) {
        return NNOPS_UNSUPPORTED;
    }
    return -1;
}

// Whether `rows` rows of `cols` 4-byte values, ld apart, share memory with others.
struct Range {
    uintptr_t begin, end;
};
Range range_of(const void* p, int64_t rows, int64_t cols, int64_t ld)
{
    const uintptr_t at = (uintptr_t)p;
    return rows > 0 && cols > 0 ? Range{at, at + 4 * (uintptr_t)((rows - 1) * ld + cols)} : Range{at, at};
}
bool overlap(const Range& a, const Range& b) { return a.begin < b.end && b.begin < a.end; }

// No output may lie over an input or another output, but for output `same_out[i]`
// over input `same_in[i]`, at the same place.
template <int kIn, int kOut, int kSame>
bool apart(const Range (&in)[kIn], const Range (&out)[kOut], const int (&same)[kSame][2])
{
    for (int o = 0; o < kOut; ++o) {
        for (int i = 0; i < kIn; ++i) {
            bool in_place = false;
            for (int s = 0; s < kSame; ++s) {
                in_place |= same[s][0] == i && same[s][1] == o && in[i].begin == out[o].begin;
            }
            if (!in_place && overlap(in[i], out[o])) {
                return false;
            }
        }
        for (int q = 0; q < o; ++q) {
            if (overlap(out[q], out[o])) {
                return false;
            }
        }
    }
    return true;
}

size_t align16(size_t n) { return (n + 15) / 16 * 16; }

// (cells: where both ways take as long)
bool fork_is_small(const NnopsKvForkArgs* g)
{
    return g->pages <= kSmallPages && g->sequences <= kSmallRows && g->children <= kSmallRows &&
           g->sequences * g->table_pages + g->children * g->new_table_pages <= kSmallCells;
}

size_t fork_workspace(const NnopsKvForkArgs* g)
{
    return fork_is_small(g) ? 0 : 3 * align16(4 * (size_t)g->pages) + align16(sizeof(Child) * (size_t)g->children);
}

bool compact_is_small(const NnopsKvCompactArgs* g)
{
    return g->pages <= kCompactPages && g->sequences * g->table_pages <= kCompactCells;
}

size_t compact_workspace(const NnopsKvCompactArgs* g)
{
    return compact_is_small(g) ? 0 : align16(4 * (size_t)((g->pages + kBlock - 1) / kBlock)) + align16(4 * (size_t)g->pages);
}

}  // namespace
}  // namespace nnops_amd

using namespace nnops_amd;

extern "C" size_t nnops_hip_kv_cache_fork_workspace_size(const NnopsKvForkArgs* g)
{
    return check_fork(g) >= 0 ? 0 : fork_workspace(g);
}

extern "C" int nnops_hip_kv_cache_fork(const NnopsKvForkArgs* g, void* workspace, size_t workspace_bytes, void* stream)
{
    const TimingDisarm disarm;
    if (const int rc = check_fork(g); rc >= 0) {
        return rc;
    }
    const int64_t b = g->sequences, n = g->children;
    if (g->counts == nullptr || (g->pages > 0 && (g->refs == nullptr || g->new_refs == nullptr)) ||
        (b > 0 && (g->lengths == nullptr || g->ld_table < g->table_pages ||
                   (g->table_pages > 0 && g->page_table == nullptr))) ||
        (n > 0 && (g->parents == nullptr || g->new_tokens == nullptr || g->new_lengths == nullptr ||
                   g->copies == nullptr || g->ld_new_table < g->new_table_pages ||
                   (g->new_table_pages > 0 && g->new_table == nullptr)))) {
        return NNOPS_INVALID_ARGUMENT;
    }
    const Range in[5] = {range_of(g->page_table, b, g->table_pages, g->ld_table), range_of(g->lengths, 1, b, b),
                         range_of(g->refs, 1, g->pages, g->pages), range_of(g->parents, 1, n, n),
                         range_of(g->new_tokens, 1, n, n)};
    const Range out[5] = {range_of(g->new_table, n, g->new_table_pages, g->ld_new_table),
                          range_of(g->new_lengths, 1, n, n), range_of(g->new_refs, 1, g->pages, g->pages),
                          range_of(g->copies, 1, 2 * n, 2 * n), range_of(g->counts, 1, 2, 2)};
    if (const int same[1][2] = {{2, 2}}; !apart(in, out, same)) {
        return NNOPS_INVALID_ARGUMENT;
    }
    const size_t need = fork_workspace(g);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || (uintptr_t)workspace % 16 != 0)) {
        return NNOPS_NOT_INITIALIZED;
    }
    ForkKern k{};
    k.table = g->page_table;
    k.lengths = g->lengths;
    k.refs = g->refs;
    k.parents = g->parents;
    k.new_tokens = g->new_tokens;
    k.new_table = g->new_table;
    k.new_lengths = g->new_lengths;
    k.new_refs = g->new_refs;
    k.copies = g->copies;
    k.counts = g->counts;
    k.ld_table = g->ld_table;
    k.ld_new = g->ld_new_table;
    k.seqs = (int32_t)b;
    k.table_pages = (int32_t)g->table_pages;
    k.pages = (int32_t)g->pages;
    k.page_log2 = __builtin_ctzll((unsigned long long)g->page_tokens);
    k.children = (int32_t)n;
    k.new_pages = (int32_t)g->new_table_pages;
    const int64_t wide = g->table_pages > g->new_table_pages ? g->table_pages : g->new_table_pages;
    k.chunks = (int32_t)((wide + 255) / 256 > 0 ? (wide + 255) / 256 : 1);
    char* at = static_cast<char*>(workspace);
    const size_t side = align16(4 * (size_t)g->pages);
    k.writers = reinterpret_cast<int32_t*>(at);
    k.first = reinterpret_cast<int32_t*>(at + side);
    k.free = reinterpret_cast<int32_t*>(at + 2 * side);
    k.child = reinterpret_cast<Child*>(at + 3 * side);
    const int64_t holds = ((b + n) * k.chunks + 3) / 4;
    if (holds > INT32_MAX / 256) {
        return NNOPS_UNSUPPORTED;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (fork_is_small(g)) {
        NNOPS_LAUNCH(fork_small, dim3(1), dim3(kPlan), 0, s, k);
        return hipGetLastError() == hipSuccess ? NNOPS_OK : NNOPS_INTERNAL;
    }
    if (g->pages > 0) {
        NNOPS_LAUNCH(fork_clear, dim3((unsigned)((g->pages + 255) / 256)), dim3(256), 0, s, k);
    }
    if (holds > 0) {
        NNOPS_LAUNCH(fork_hold, dim3((unsigned)holds), dim3(256), 0, s, k);
    }
    NNOPS_LAUNCH(fork_take, dim3(1), dim3(kPlan), 0, s, k);
    return hipGetLastError() == hipSuccess ? NNOPS_OK : NNOPS_INTERNAL;
}

extern "C" size_t nnops_hip_kv_cache_compact_workspace_size(const NnopsKvCompactArgs* g)
{
    return check_compact(g) >= 0 ? 0 : compact_workspace(g);
}

extern "C" int nnops_hip_kv_cache_compact(const NnopsKvCompactArgs* g, void* workspace, size_t workspace_bytes,
                                          void* stream)
{
    const TimingDisarm disarm;
    if (const int rc = check_compact(g); rc >= 0) {
        return rc;
    }
    const int64_t b = g->sequences;
    if (g->counts == nullptr ||
        (g->pages > 0 && (g->refs == nullptr || g->new_refs == nullptr || g->moved == nullptr)) ||
        (g->pages > 1 && g->copies == nullptr) ||
        (b > 0 && (g->lengths == nullptr || g->ld_table < g->table_pages || g->ld_new_table < g->table_pages ||
                   (g->table_pages > 0 && (g->page_table == nullptr || g->new_table == nullptr))))) {
        return NNOPS_INVALID_ARGUMENT;
    }
    if (b > 1 && g->page_table == g->new_table && g->ld_table != g->ld_new_table) {
        return NNOPS_INVALID_ARGUMENT;
    }
    const Range in[3] = {range_of(g->page_table, b, g->table_pages, g->ld_table), range_of(g->lengths, 1, b, b),
                         range_of(g->refs, 1, g->pages, g->pages)};
    const Range out[5] = {range_of(g->new_table, b, g->table_pages, g->ld_new_table),
                          range_of(g->new_refs, 1, g->pages, g->pages),
                          range_of(g->copies, 1, g->pages / 2 * 2, g->pages), range_of(g->moved, 1, g->pages, g->pages),
                          range_of(g->counts, 1, 2, 2)};
    if (const int same[2][2] = {{0, 0}, {2, 1}}; !apart(in, out, same)) {
        return NNOPS_INVALID_ARGUMENT;
    }
    const size_t need = compact_workspace(g);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || (uintptr_t)workspace % 16 != 0)) {
        return NNOPS_NOT_INITIALIZED;
    }
    CompactKern k{};
    k.table = g->page_table;
    k.lengths = g->lengths;
    k.refs = g->refs;
    k.new_table = g->new_table;
    k.new_refs = g->new_refs;
    k.copies = g->copies;
    k.moved = g->moved;
    k.counts = g->counts;
    k.ld_table = g->ld_table;
    k.ld_new = g->ld_new_table;
    k.seqs = (int32_t)b;
    k.table_pages = (int32_t)g->table_pages;
    k.pages = (int32_t)g->pages;
    k.page_log2 = __builtin_ctzll((unsigned long long)g->page_tokens);
    k.blocks = (int32_t)((g->pages + kBlock - 1) / kBlock);
    k.chunks = (int32_t)((g->table_pages + 255) / 256);
    k.used = static_cast<int32_t*>(workspace);
    k.code = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + align16(4 * (size_t)k.blocks));
    const int64_t groups = (g->pages + 255) / 256 + (b * k.chunks + 3) / 4;
    if (groups > INT32_MAX / 256) {
        return NNOPS_UNSUPPORTED;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (compact_is_small(g)) {
        NNOPS_LAUNCH(compact_small, dim3(1), dim3(kPlan), 0, s, k);
        return hipGetLastError() == hipSuccess ? NNOPS_OK : NNOPS_INTERNAL;
    }
    if (k.blocks > 0) {
        NNOPS_LAUNCH(compact_count, dim3((unsigned)k.blocks), dim3(256), 0, s, k);
    }
    // (without pages too: the counts, and a table of nothing)
    NNOPS_LAUNCH(compact_rank, dim3((unsigned)(k.blocks > 0 ? k.blocks : 1)), dim3(256), 0, s, k);
    if (groups > 0) {
        NNOPS_LAUNCH(compact_apply, dim3((unsigned)groups), dim3(256), 0, s, k);
    }
    return hipGetLastError() == hipSuccess ? NNOPS_OK : NNOPS_INTERNAL;
}

extern "C" int nnops_hip_kv_cache_copy(const NnopsKvCopyArgs* g, void* stream)
{
    const TimingDisarm disarm;
    if (g == nullptr || g->pages < 0 || g->heads < 0 || g->count < 0) {
        return NNOPS_INVALID_ARGUMENT;
    }
    if (!page_tokens_fit(g->page_tokens) || g->head_dim < 16 || g->head_dim > 256 || g->head_dim % 16 != 0) {
        return NNOPS_UNSUPPORTED;
    }
    if (g->count == 0 || g->pages == 0 || g->heads == 0) {
        return NNOPS_OK;
    }
    if (g->pages > INT32_MAX || g->heads > (1 << 16) || g->heads * g->page_tokens * g->head_dim > INT32_MAX) {
        return NNOPS_UNSUPPORTED;
    }
    if (g->copies == nullptr || g->k == nullptr || g->v == nullptr || g->k_scale == nullptr || g->v_scale == nullptr ||
        (uintptr_t)g->k % 16 != 0 || (uintptr_t)g->v % 16 != 0) {
        return NNOPS_INVALID_ARGUMENT;
    }
    CopyKern k{};
    k.k = g->k;
    k.v = g->v;
    k.k_scale = g->k_scale;
    k.v_scale = g->v_scale;
    k.copies = g->copies;
    k.page_bytes = g->heads * g->page_tokens * g->head_dim;
    k.pages = (int32_t)g->pages;
    k.heads = (int32_t)g->heads;
    k.pieces = (int32_t)((k.page_bytes + kPiece - 1) / kPiece);
    hipStream_t s = static_cast<hipStream_t>(stream);
    // launches of fewer than 2^23 workgroups
    const int64_t slab = (1 << 23) / (2 * (int64_t)k.pieces) > 0 ? (1 << 23) / (2 * (int64_t)k.pieces) : 1;
    for (int64_t i0 = 0; i0 < g->count; i0 += slab) {
        const int64_t n = g->count - i0 < slab ? g->count - i0 : slab;
        k.copies = g->copies + 2 * i0;
        NNOPS_LAUNCH(kv_copy, dim3((unsigned)(n * 2 * k.pieces)), dim3(256), 0, s, k);
    }
    return hipGetLastError() == hipSuccess ? NNOPS_OK : NNOPS_INTERNAL;
}
