// The walk over the units of work of the prompt attention (kv8_prefill.cu): plain arithmetic, the same on the host
#pragma once
#include "common.cuh"

namespace ft {

// a unit that begins in a share and goes on in the next ones: how many, its first row of q, its key head, its tokens (below zero: few, whose halves are parts)
struct Kv8Split { int parts, row0, head, tokens; };

struct Kv8Prompt {
    const __half* q;
    const uint8_t* cache;
    const int *page_table, *req_q_start, *req_slot, *req_pos0;
    __nv_bfloat16 *out, *out_lo;
    Kv8Split* split;
    float* parts;
    int num_pages, table_rows, max_pages, n_req, T, nq, nkv;
    int G, th;                                                       // query heads a key head, tokens of a half
    int few_pages;                                                   // pages of a step of a unit of few tokens
    int wait_limit;                                                  // tries of a wait
    unsigned inv_g;                                                  // row / G = row * inv_g >> 16
    float scale_log2;
};

// The flat list's length fits 31 bits (the host has seen to it), so do all sums and differences along it.
// sum over i < n of floor((a i + b) / 64): the lattice points below a line, by Euclid's steps.  Each term is a part of the result (or wraps and is multiplied by 0)
__host__ __device__ inline int floor_sum64(unsigned n, unsigned a, unsigned b) {
    unsigned m = 64, sum = 0;
#pragma unroll 1
    while (n > 0) {
        sum += (n & 1 ? (n - 1) / 2 * n : n / 2 * (n - 1)) * (a / m) + n * (b / m);
        a %= m;
        b %= m;
        const unsigned top = a * n + b;
        n = top / m;
        b = top % m;
        const unsigned t = a;
        a = m;
        m = t;
    }
    return (int)sum;
}

// What a unit costs beyond its pages, in pages: it takes that much more of the flat list, behind its last step
constexpr int kKv8Start = 3;

// one request: its rows of q, tiles of 2 th tokens, steps of its tiles.  at = the position of row0, which may lie ahead of the sequence: the list is made as if it were 0 then
struct Kv8Request {
    int row0, len, at, pos0, slot, tiles;
    __host__ __device__ __forceinline__ void load(const Kv8Prompt& p, int r) {
        row0 = max(0, min(p.req_q_start[r], p.T));
        len = max(0, min(p.req_q_start[r + 1], p.T) - row0);
        const long long first = (long long)p.req_pos0[r] + ((long long)row0 - p.req_q_start[r]), low = -p.T, high = p.max_pages * kKvTile;
        at = (int)(first < low ? low : first > high ? high : first);
        pos0 = max(0, at);
        slot = p.req_slot[r];
        tiles = (len + 2 * p.th - 1) / (2 * p.th);
    }
    __host__ __device__ __forceinline__ int tokens(const Kv8Prompt& p, int i) const { return min(2 * p.th, len - i * 2 * p.th); }
    __host__ __device__ __forceinline__ int pages(const Kv8Prompt& p, int i) const { return (pos0 + i * 2 * p.th + tokens(p, i) - 1) / kKvTile + 1; }
    __host__ __device__ __forceinline__ int steps(const Kv8Prompt& p, int i) const {
        const int n = pages(p, i);
        return tokens(p, i) <= p.th ? (n + p.few_pages - 1) / p.few_pages : n;
    }
    __host__ __device__ __forceinline__ int before(const Kv8Prompt& p, int i) const { return floor_sum64(i, 2 * p.th, pos0 + 2 * p.th - 1) + i * (1 + kKv8Start); }   // lengths of the full tiles 0 .. i - 1
    __host__ __device__ __forceinline__ int all(const Kv8Prompt& p) const { return tiles ? before(p, tiles - 1) + steps(p, tiles - 1) + kKv8Start : 0; }
};

// What a run of requests adds up to: steps and units of one key head, the longest unit's steps, and whether the list grows
struct Kv8Sums {
    int steps = 0, units = 0, most = 0;
    bool grows = true;
    __host__ __device__ __forceinline__ void add(const Kv8Prompt& p, int r) {
        Kv8Request q;
        q.load(p, r);
        grows = grows && p.req_q_start[r] <= p.req_q_start[r + 1];
        steps += q.all(p);
        units += q.tiles;
        if (q.tiles) most = max(most, max(q.steps(p, q.tiles - 1), q.tiles > 1 ? q.steps(p, q.tiles - 2) : 0));
    }
};

// A stretch of pages of one unit.  parts: 0 = it is the whole unit; else, where the unit begins, how many shares it lies in
struct Kv8Stretch { int page0, pages, few, row0, tokens, pos0, head, slot, begins, parts; };

// A CTA's share, walked stretch by stretch; a stretch = steps t0 .. t1 - 1 of one unit
struct Kv8Walk {
    Kv8Request q;
    int f, f_end, first;                                       // where it is in the flat list; where the unit begins
    int r, h, i, t, t0, t1, n_steps, n_pages, n_tok;
    bool few;
    __host__ __device__ __forceinline__ void unit(const Kv8Prompt& p) {
        n_tok = q.tokens(p, i);
        n_pages = q.pages(p, i);
        few = n_tok <= p.th;
        n_steps = few ? (n_pages + p.few_pages - 1) / p.few_pages : n_pages;
    }
    __host__ __device__ __forceinline__ bool next(const Kv8Prompt& p) {
#pragma unroll 1
        for (;;) {
            if (f >= f_end) return false;
            if (t >= n_steps + kKv8Start) {
                t = 0;
                if (++i == q.tiles) {
                    i = 0;
                    if (++h == p.nkv) {
                        h = 0;
#pragma unroll 1
                        do q.load(p, ++r);
                        while (q.len == 0);
                    }
                }
                unit(p);
            }
            const int take = min(f_end - f, n_steps + kKv8Start - t);
            first = f - t;
            t0 = min(t, n_steps);
            t1 = min(t + take, n_steps);
            t += take;
            f += take;
            if (t1 > t0) return true;                                // else all of it was behind the unit's last step
        }
    }
    // the share of CTA `cta` in a list of `len`, `each` of them a CTA.  true: there is something in it.  Where the requests' list does not grow there is not: its sums
    // could be any, and next() must find nothing to walk, since nothing else of the walk is set then
    __host__ __device__ __forceinline__ bool share(bool grows, int len, int each, int cta) {
        f = grows ? min(len, each * cta) : 0;
        f_end = grows ? min(len, f + each) : 0;
        return f < f_end;
    }
    // where step (or, where each CTA takes whole units, unit) `at` of the flat list lies; `before` of them belong to requests ahead of r0, and it is r0's or a later one's
    __host__ __device__ inline void seek(const Kv8Prompt& p, bool whole, int r0, int before, int at) {
#pragma unroll 1
        for (r = r0;; ++r) {
            q.load(p, r);
            const int n = whole ? q.tiles : q.all(p);
            if (at < (before + n) * p.nkv) {
                int rest = at - before * p.nkv;
                h = (int)((unsigned)rest / (unsigned)n);
                rest -= h * n;
                int lo = 0, hi = q.tiles - 1;                        // the last tile that begins at or before rest
#pragma unroll 1
                while (!whole && lo < hi) {
                    const int mid = (lo + hi + 1) >> 1;
                    if (q.before(p, mid) <= rest) lo = mid; else hi = mid - 1;
                }
                i = whole ? rest : lo;
                t = whole ? 0 : rest - q.before(p, lo);
                return;
            }
            before += n;
        }
    }
    // the stretch as the other warps get it; per: steps of a share
    __host__ __device__ inline Kv8Stretch stretch(const Kv8Prompt& p, int per, int share) const {
        Kv8Stretch s;
        s.page0 = page0(p.few_pages);
        s.pages = page1(p.few_pages) - s.page0;
        s.few = few;
        s.row0 = row0(p);
        s.tokens = n_tok;
        s.pos0 = position0(p);
        s.head = h;
        s.slot = q.slot;
        s.begins = t0 == 0;
        s.parts = t0 == 0 && t1 == n_steps ? 0 : t0 == 0 ? (int)((unsigned)(first + n_steps - 1) / (unsigned)per) - share + 1 : 1;
        return s;
    }
    // pages of the stretch, in the order in which they are asked for
    __host__ __device__ __forceinline__ int page0(int p_few) const { return few ? p_few * t0 : t0; }
    __host__ __device__ __forceinline__ int page1(int p_few) const { return few ? min(p_few * t1, n_pages) : t1; }
    __host__ __device__ __forceinline__ int row0(const Kv8Prompt& p) const { return q.row0 + i * 2 * p.th; }
    __host__ __device__ __forceinline__ int position0(const Kv8Prompt& p) const { return q.at + i * 2 * p.th; }
};

}  // namespace ft
