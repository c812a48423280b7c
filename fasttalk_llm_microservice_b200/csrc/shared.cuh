// Attention of one query token per sequence where groups of sequences have their first tokens in common: what its kernels share.
//
// Group g's queries are group_start[g] .. group_start[g + 1] - 1; each sees min(shared, ctx) keys on the pages of the group's first query's row of the page table and
// the rest of its ctx keys on its own.  Two kinds of work come of that:
//   shared part   a unit = one group, key head and tile of queries, all pages of the prefix (shared_prefix.cu, tcgen05): keys are read once for all of them;
//   own part      a unit = one sequence and key head, its own pages (shared_decode.cu); whoever ends it adds the shared part's results and writes the output.
// A group that does not pay (SharedPlan) has no shared part: its sequences read the first row's pages themselves, as steps ahead of their own.
#pragma once
#include "common.cuh"

namespace ft {

constexpr int kSharedGroup = 8;                  // query heads a key head at most
constexpr int kSharedRows = 128;                 // rows (query, head of the group) of a half of a tile
constexpr float kSharedLog2E = 1.4426950408889634f;
// Probabilities are formed 2^6 times their size, so that fp16's normal numbers reach down to 2^-20 of the largest; a running maximum may lag by 2^8
constexpr float kSharedTop = 6.f, kSharedGrow = 8.f;
constexpr int kSharedStart = 3;                  // what a unit of the shared part costs beyond its pages, in pages: it takes that much more of the list, behind its last step

// one sequence.  Steps: `lead` tiles of the first row's pages, then its own from token `begin` on, and one if there are none of either
struct SharedSeq { int ctx, begin, lead, group, row_lead, row_own, first, steps; };      // group: whose shared part it takes, or -1; first: steps of the sequences ahead
// one group's shared part.  base: where it begins in the list of steps; pages 0: none
struct SharedGroup { int base, seq0, size, tokens, pages, row, pad0, pad1; };

struct SharedHead {                              // of the plan
    int own_total, own_per, own_whole, prefix_total, prefix_per;
};

struct SharedArgs {
    const __half* q;
    const uint8_t* cache;
    const int *page_table, *req_slot, *ctx_lens, *group_start, *shared_lens;
    __nv_bfloat16 *out, *out_lo;
    SharedHead* head;
    SharedSeq* seqs;
    SharedGroup* groups;
    int *own_from, *prefix_from;                 // where each CTA begins: a sequence, a group
    int* counters;
    float *own_parts, *rows_o;
    float2* rows_ml;                             // prefix results: O [row + 256 CTA][D], (m, l)
    int B, n_groups, num_pages, table_rows, max_pages, nq, nkv, G, th;        // th: queries of a half
    int own_ctas, prefix_ctas;
    float scale_log2;
};

// steps of a tile of `tokens` queries over `pages` pages: where they fill one half only, each half takes every other page
__host__ __device__ __forceinline__ int shared_steps(int tokens, int th, int pages) { return tokens <= th ? (pages + 1) / 2 : pages; }
// of all tiles of one key head
__host__ __device__ __forceinline__ int shared_head_steps(int size, int th, int pages) {
    const int tiles = (size + 2 * th - 1) / (2 * th);
    return (tiles - 1) * (pages + kSharedStart) + shared_steps(size - (tiles - 1) * 2 * th, th, pages) + kSharedStart;
}
// where row 0 of (group, key head, query i of the group) lies among the prefix's results
__host__ __device__ __forceinline__ size_t shared_row(const SharedGroup& g, int h, int i, int nq, int G) { return (size_t)g.seq0 * nq + ((size_t)h * g.size + i) * G; }

int launch_shared_prefix(const SharedArgs& p, int d, cudaStream_t st);
int shared_prefix_waits(int* out);

}  // namespace ft
