// The paged 8-bit cache as its kernels see it: pages, the sequences' tables, and
// which rows, pages and tiles a workgroup has, found on the device from tables
// that the host does not read.
#pragma once

#include "common.hpp"

namespace nnops_amd {

// The smallest scale of a page that holds tokens: what divides by it stays finite.
constexpr float kLeastScale = 0x1p-100f;

struct Paged {
    int8_t* k;
    int8_t* v;
    float* k_scale;
    float* v_scale;
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* row_starts;   // or nullptr: each sequence has `uniform` rows
    int64_t ld_table;
    int32_t pages, heads, page, page_log2, d;
    int32_t seqs, table_pages, rows, uniform;
};

// A sequence's rows of this call and the tokens that it holds after it.
struct SeqRows {
    int32_t start, n, len;
};

__device__ __forceinline__ SeqRows seq_rows(const Paged& p, int b)
{
    SeqRows s;
    if (p.row_starts != nullptr) {
        s.start = min(max(p.row_starts[b], 0), p.rows);
        s.n = max(min(max(p.row_starts[b + 1], 0), p.rows) - s.start, 0);
    } else {
        s.start = b * p.uniform;
        s.n = p.uniform;
    }
    s.len = (int32_t)min((int64_t)max(p.lengths[b], 0), (int64_t)p.table_pages << p.page_log2);
    return s;
}

// Page number of a sequence's page, -1 if the table holds none that exists.
__device__ __forceinline__ int page_of(const Paged& p, int b, int page)
{
    const int id = p.table[(int64_t)b * p.ld_table + page];
    return id >= 0 && id < p.pages ? id : -1;
}

// Work item w of a launch that numbers count(sequence) items per sequence one
// after another (fewer than 2^31 in all): its sequence and its number there;
// false past the last. Whole waves call it (each wave searches for itself, 64
// sequences a step); w is the same in all lanes.
template <typename At, typename Count>
__device__ __forceinline__ bool find_item(int seqs, uint32_t w, At at, Count count, int& b, int& j, SeqRows& seq)
{
    const int lane = threadIdx.x % 64;
    uint32_t before = 0;
    for (int base = 0; base < seqs; base += 64) {
        SeqRows s{0, 0, 0};
        uint32_t c = 0;
        if (base + lane < seqs) {
            s = at(base + lane);
            c = (uint32_t)count(s);
        }
        uint32_t upto = c;
#pragma unroll
        for (int m = 1; m < 64; m *= 2) {
            const uint32_t other = (uint32_t)__shfl_up((int)upto, m);
            upto += lane >= m ? other : 0u;
        }
        const uint64_t hit = __ballot(before + upto > w);
        if (hit != 0) {
            const int l = __builtin_ctzll(hit);
            b = base + l;
            j = (int)(w - before) - __builtin_amdgcn_readlane((int)(upto - c), l);
            seq.start = __builtin_amdgcn_readlane(s.start, l);
            seq.n = __builtin_amdgcn_readlane(s.n, l);
            seq.len = __builtin_amdgcn_readlane(s.len, l);
            return true;
        }
        before += (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    }
    return false;
}

template <typename Count>
__device__ __forceinline__ bool find_item(const Paged& p, uint32_t w, Count count, int& b, int& j, SeqRows& seq)
{
    return find_item(p.seqs, w, [&](int i) { return seq_rows(p, i); }, count, b, j, seq);
}

// What every entry point checks of a cache: its sizes, then what it points to.
// They return -1 if the call is to run.
int check_page_shapes(const NnopsKvPages& c, int64_t rows);
int check_page_memory(const NnopsKvPages& c);
Paged paged(const NnopsKvPages& c, int64_t rows);

}  // namespace nnops_amd
