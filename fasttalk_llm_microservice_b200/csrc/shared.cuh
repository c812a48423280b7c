// Attention of one query token per sequence where groups of sequences have their first tokens in common: the two lists of work that its kernel (shared.cu) walks.
//
// Group g's queries are group_start[g] .. group_start[g + 1] - 1; each sees min(shared, ctx) keys on the pages of the group's first query's row of the page table and
// the rest of its ctx keys on its own.  Two kinds of work come of that:
//   prefix   a unit = one group, key head and tile of queries; its steps are the pages of the prefix, read once for all queries of the tile
//   own      a unit = one sequence and key head; its steps are chunks of its own pages
// A group that does not pay has no prefix units: its sequences read the first row's pages themselves, as steps ahead of their own.  The prefix list is cut into equal shares,
// one for each SM, the own list into one for each warp that walks it.  Plain arithmetic, the same on the host.
#pragma once
#include "common.cuh"

namespace ft {

constexpr int kSharedGroup = 8;                  // query heads a key head at most
constexpr int kSharedRows = 128;                 // rows (query, head of the group) of a half of a tile
constexpr int kSharedStart = 3;                  // what a prefix unit costs beyond its pages, in pages: it takes that much more of the list, behind its last step

struct SharedArgs {
    const __half* q;
    const uint8_t* cache;
    const int *page_table, *req_slot, *ctx_lens, *group_start, *shared_lens;
    __nv_bfloat16 *out, *out_lo;
    int4 *own_units, *prefix_units;              // [B][nkv]: first and last warp that has a part, whether there is a prefix part;
                                                 //           first and last CTA that has a part, its row among the results
    float* own_parts;                            // [unit + warp][G][D], then (m, l)
    float* rows_o;                               // prefix results: O [D / 4][row + 256 CTA][4], (m, l)
    float2* rows_ml;
    int* gave_up_at;                             // [CTA]: 1 where a wait of this call ran out
    int B, n_groups, num_pages, table_rows, max_pages, nq, nkv, G, th;        // th: queries of a half
    int rows;                                    // of the prefix's results
    int chunk_log;                               // tokens of an own step: 2^6 or 2^4
    unsigned inv_g;                              // row / G = row * inv_g >> 16 for a half's rows
    float scale_log2;

    unsigned inv_tile;                           // 2^32 / (2 th), rounded up
    int least_size, least_pages;                 // sharing pays: queries of a group; pages that the call's groups save in all
    int give_up;                                 // 1: at the first wait that is not over yet
    int ctas;

    __host__ __device__ __forceinline__ int reach() const { return max_pages * kKvTile; }
    // tiles of 2 th queries: exact for any batch that fits (up to 2^32 / (2 th) queries)
    __host__ __device__ __forceinline__ int tiles(int size) const { return (int)((unsigned long long)(unsigned)(size + 2 * th - 1) * inv_tile >> 32); }
    __host__ __device__ __forceinline__ int row_of(int b) const {
        const int slot = req_slot ? req_slot[b] : b;
        return slot >= 0 && slot < table_rows ? slot : -1;
    }
};

// The groups, wherever the lists lie; n = 0: none.  share: their prefixes are read once
struct SharedGroups {
    const int *start, *lens;
    int n;
    bool share;
    __host__ __device__ __forceinline__ int tokens(const SharedArgs& p, int g) const { return max(0, min(lens[g], p.reach())); }
    // whether group g has a prefix part
    __host__ __device__ __forceinline__ bool pays(const SharedArgs& p, int g) const { return share && start[g + 1] - start[g] >= p.least_size && tokens(p, g) >= 2 * kKvTile; }
    // pages that sharing saves group g (up to a million), beyond what it costs
    __host__ __device__ __forceinline__ int saves(const SharedArgs& p, int g) const {
        const long long n = (long long)(start[g + 1] - start[g] - p.least_size + 1) * (tokens(p, g) / kKvTile);
        return !pays(p, g) ? 0 : n < 1 << 20 ? (int)n : 1 << 20;
    }
    // the last group that begins at or before b (those without queries begin where the next one does), or -1
    __host__ __device__ __forceinline__ int of(int b) const {
        int lo = -1, hi = n - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (start[mid] <= b) lo = mid; else hi = mid - 1;
        }
        return lo;
    }
};

// A group's prefix part; pages 0: none
struct SharedPrefix {
    int seq0, size, tokens, pages, tiles;
    __host__ __device__ __forceinline__ void load(const SharedArgs& p, const SharedGroups& gr, int g) {
        seq0 = gr.start[g];
        size = gr.start[g + 1] - seq0;
        tokens = gr.tokens(p, g);
        pages = gr.pays(p, g) ? (tokens + kKvTile - 1) / kKvTile : 0;
        tiles = pages ? p.tiles(size) : 0;
    }
    __host__ __device__ __forceinline__ int queries(const SharedArgs& p, int tile) const { return min(2 * p.th, size - tile * 2 * p.th); }
    // steps of a tile of n queries: where they fill one half only, each half takes every other page (40960 tokens, heads of 64, four to a key head: 32 queries in this way
    // 31.5 us, 33 in the other 46.5)
    __host__ __device__ __forceinline__ int steps(const SharedArgs& p, int n) const { return n <= p.th ? (pages + 1) / 2 : pages; }
    // what all tiles of one key head take of the list
    __host__ __device__ __forceinline__ int each(const SharedArgs& p) const { return (tiles - 1) * (pages + kSharedStart) + steps(p, queries(p, tiles - 1)) + kSharedStart; }
    __host__ __device__ __forceinline__ int all(const SharedArgs& p) const { return pages ? p.nkv * each(p) : 0; }
    // where row 0 of (key head, query i of the group) lies among the results
    __host__ __device__ __forceinline__ int row(const SharedArgs& p, int h, int i) const { return seq0 * p.nq + (h * size + i) * p.G; }
};

// A sequence: `lead` chunks of the first row's pages, then its own from token `begin` on, and one step if there are none of either
struct SharedSeq {
    int ctx, begin, lead, steps, first;          // first: the query whose row has the shared pages
    bool prefix;                                 // a prefix part is added
    __host__ __device__ __forceinline__ void load(const SharedArgs& p, const SharedGroups& gr, int b, int ctx_len) {
        const int up = (1 << p.chunk_log) - 1;
        ctx = max(0, min(ctx_len, p.reach()));
        begin = lead = 0;
        first = -1;
        prefix = false;
        const int g = gr.of(b);
        if (g >= 0 && b < gr.start[g + 1]) {
            begin = gr.tokens(p, g);
            first = gr.start[g];
            prefix = ctx >= begin && gr.pays(p, g);
            if (!prefix) lead = min(begin, ctx) + up >> p.chunk_log;
        }
        const int own = ctx > begin ? (ctx + up >> p.chunk_log) - (begin >> p.chunk_log) : 0;
        steps = max(1, lead + own);
    }
    // its steps where its group had no prefix part
    __host__ __device__ __forceinline__ int steps_alone(const SharedArgs& p) const { return prefix ? steps - (ctx == begin) + (begin + (1 << p.chunk_log) - 1 >> p.chunk_log) : steps; }
    // tokens lo .. hi - 1 that step t reads (none: lo >= hi); true: on the first row's pages
    __host__ __device__ __forceinline__ bool step(const SharedArgs& p, int t, int& lo, int& hi) const {
        const bool led = t < lead;
        const int at = (led ? t : (begin >> p.chunk_log) + t - lead) << p.chunk_log;
        lo = max(at, led ? 0 : begin);
        hi = min(at + (1 << p.chunk_log), led ? min(begin, ctx) : ctx);
        return led;
    }
};

// The own list's shares: `warps` of each CTA, the first `busy` CTAs (those with a share of the prefix list) shorter ones.  They follow one another CTA by CTA, then warp by
// warp, so that neighbouring ones are on different SMs; none is empty, but for those behind the list's end.
struct OwnShares {
    int ctas, busy, few, many;
    // as the prefix part takes the time of `cost` steps from each warp of its CTAs
    __host__ __device__ __forceinline__ void set(int total, int warps, int ctas_, int busy_, int cost) {
        ctas = ctas_;
        busy = busy_;
        const int each = (int)((unsigned)(total + warps - 1) / (unsigned)warps);         // steps of a round over all CTAs
        few = many = (int)((unsigned)(each + ctas - 1) / (unsigned)ctas);
        if (busy > 0 && busy < ctas) {
            few = max(1, (int)((unsigned)(each + busy * cost + ctas - 1) / (unsigned)ctas) - cost);
            many = max(1, (int)((unsigned)(max(0, each - busy * few) + ctas - busy - 1) / (unsigned)(ctas - busy)));
        }
    }
    __host__ __device__ __forceinline__ int round() const { return busy * few + (ctas - busy) * many; }
    __host__ __device__ __forceinline__ int size(int cta) const { return cta < busy ? few : many; }
    __host__ __device__ __forceinline__ int begin(int warp, int cta) const { return warp * round() + (cta < busy ? cta * few : busy * few + (cta - busy) * many); }
    // the share that step f lies in: warp * CTAs + CTA
    __host__ __device__ __forceinline__ int of(int f) const {
        const int warp = (int)((unsigned)f / (unsigned)round()), rest = f - warp * round(), far = rest - busy * few;
        return warp * ctas + (far < 0 ? (int)((unsigned)rest / (unsigned)few) : busy + (int)((unsigned)far / (unsigned)many));
    }
};

// A warp looks up 32 steps of the own list at once, a lane each: F, F + 1 .. among 32 sequences, the first of which holds step F.  Every sequence has a step at least, so that the 32 hold
// all of these; a sequence that is over by F would leave 31, which with one key head and a step each is one too few.  Which of them holds F; end_of(i): behind the last step of the i-th
template <class EndOf>
__host__ __device__ __forceinline__ int own_sequence(int F, EndOf&& end_of) {
    int l = 0;                                   // the first that ends behind F
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        if (end_of(l + o - 1) <= F) l += o;
    return l;
}

// Step F, in sequence `seq`, whose steps (so many for each key head) begin at `base`
struct OwnStep {
    int head, from, last;                        // the unit: its key head, its first and last step
    int next_seq, next_base;                     // the sequence that holds step F + 1, and where that begins
    __host__ __device__ __forceinline__ void set(const SharedArgs& p, int F, int seq, int base, int steps) {
        head = (int)((unsigned)(F - base) / (unsigned)steps);
        from = base + head * steps;
        last = from + steps - 1;
        const bool over = F == last && head == p.nkv - 1;
        next_seq = seq + over;
        next_base = over ? last + 1 : base;
    }
};

// n queries from q0 on, over pages p0 .. of the row of query seq0; row0: where the first one's results lie; last: the last share that the unit lies in
struct SharedStretch {
    int p0, pages, n, h, seq0, q0, row0, tokens, last;
    bool few;                                    // the queries fill one half only
    __host__ __device__ __forceinline__ int of_half(int half) const { return few ? (pages - half + 1) / 2 : pages; }      // its pages
};

// A CTA's share of the prefix list, walked stretch by stretch; a stretch = pages p0 .. p0 + pages - 1 of one unit
struct PrefixWalk {
    SharedPrefix w;
    int f, f_end, unit_f, g, h, tile, t;
    int n, steps;                                // queries and steps of the tile
    int p0, pages;
    bool few;                                    // the queries fill one half only
    __host__ __device__ __forceinline__ void unit(const SharedArgs& p) {
        n = w.queries(p, tile);
        few = n <= p.th;
        steps = w.steps(p, n);
    }
    // the share begins at f, in group g, which begins at base
    __host__ __device__ __forceinline__ void start(const SharedArgs& p, const SharedGroups& gr, int f_, int f_end_, int g_, int base) {
        f = f_;
        f_end = f_end_;
        if (f >= f_end) return;
        g = g_;
        w.load(p, gr, g);
        const int each = w.each(p), full = w.pages + kSharedStart;
        int rest = f - base;
        h = (int)((unsigned)rest / (unsigned)each);
        rest -= h * each;
        tile = min((int)((unsigned)rest / (unsigned)full), w.tiles - 1);
        t = rest - tile * full;
        unit(p);
    }
    __host__ __device__ __forceinline__ bool next(const SharedArgs& p, const SharedGroups& gr) {
#pragma unroll 1
        for (;;) {
            if (f >= f_end) return false;
            if (t >= steps + kSharedStart) {
                t = 0;
                if (++tile == w.tiles) {
                    tile = 0;
                    if (++h == p.nkv) {
                        h = 0;
#pragma unroll 1
                        do w.load(p, gr, ++g);
                        while (w.pages == 0);
                    }
                }
                unit(p);
            }
            const int take = min(f_end - f, steps + kSharedStart - t), t0 = min(t, steps), t1 = min(t + take, steps);
            unit_f = f - t;
            t += take;
            f += take;
            if (t1 > t0) {
                p0 = few ? 2 * t0 : t0;
                pages = (few ? min(2 * t1, w.pages) : t1) - p0;
                return true;
            }                                    // else all of it was behind the unit's last step
        }
    }
    // the stretch as the other warps get it; per: steps of a share
    __host__ __device__ __forceinline__ SharedStretch stretch(const SharedArgs& p, int per) const {
        SharedStretch s;
        s.p0 = p0, s.pages = pages, s.few = few, s.n = n, s.h = h;
        s.seq0 = w.seq0;
        s.q0 = w.seq0 + tile * 2 * p.th;
        s.row0 = w.row(p, h, tile * 2 * p.th);
        s.tokens = w.tokens;
        s.last = (int)((unsigned)(unit_f + steps - 1) / (unsigned)per);
        return s;
    }
};

}  // namespace ft
