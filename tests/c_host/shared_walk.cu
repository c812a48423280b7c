// The lists of work of attention over shared prefixes on the host: every CTA's and warp's share, walked with the kernel's own arithmetic (csrc/shared.cuh).
#include <cstring>

#include "shared.cuh"

using namespace ft;

// own: stretches of all warps (`warps` in each of `shares` CTAs, of which `busy` lose `cost` steps), nine numbers each: warp, sequence, head, t0, t1, steps, prefix, first and last warp of the unit.
// else: of all CTAs: cta, group, head, tile, p0, pages, few, first and last CTA of the unit.  -> how many (at most `room` are written), or -1 - share where one is longer than `limit`
extern "C" int shared_stretches(int own, const int* ctx_lens, int B, const int* starts, const int* shared, int n_groups, int max_pages, int nkv, int G, int chunk, int shares,
                                int warps, int busy, int cost, int share, int unset, int limit, int* out, int room) {
    SharedArgs p{};
    p.ctx_lens = ctx_lens, p.group_start = starts, p.shared_lens = shared;
    p.B = B, p.n_groups = n_groups, p.max_pages = max_pages, p.table_rows = B, p.nkv = nkv, p.nq = nkv * G, p.G = G, p.th = kSharedRows / G, p.inv_tile = (unsigned)(((1ull << 32) + 2 * p.th - 1) / (2 * p.th)), p.chunk_log = chunk == 64 ? 6 : chunk == 32 ? 5 : 4;
    bool grows = true;
    for (int g = 0; g < n_groups; ++g) grows = grows && starts[g] >= 0 && starts[g] <= starts[g + 1] && starts[g + 1] <= B;
    const int groups = grows ? n_groups : 0;
    p.least_size = 2;
    const SharedGroups gr{starts, shared, grows ? n_groups : 0, share != 0};
    int total = 0, found = 0;
    for (int g = 0; !own && g < gr.n; ++g) {
        SharedPrefix w;
        w.load(p, gr, g);
        total += w.all(p);
    }
    for (int b = 0; own && b < B; ++b) {
        SharedSeq s;
        s.load(p, gr, b, ctx_lens[b]);
        total += s.steps * nkv;
        SharedSeq alone;
        alone.load(p, SharedGroups{starts, shared, grows ? n_groups : 0, false}, b, ctx_lens[b]);
        if (alone.steps != s.steps_alone(p)) return -1000000;
    }
    const int per = (int)((unsigned)(total + shares - 1) / (unsigned)shares);
    OwnShares of;
    of.set(total, warps, shares, busy, cost);
    auto tell = [&](const int* row) {
        if (found < room) memcpy(out + 9 * found, row, 9 * sizeof(int));
        ++found;
    };
    for (int x = 0; x < (own ? shares * warps : shares); ++x) {
        const int f = min(own ? of.begin(x / shares, x % shares) : per * x, total), end = min(f + (own ? of.size(x % shares) : per), total);
        int base = 0, at = 0;
        if (own) {                                   // step by step, told as stretches (how the kernel looks steps up: shared_windows.cu)
            SharedSeq s;
            for (; f < end; base += s.steps * nkv, ++at) {
                s.load(p, gr, at, ctx_lens[at]);
                if (f < base + s.steps * nkv) break;
            }
            for (int F = f; F < end;) {
                for (s.load(p, gr, at, ctx_lens[at]); F >= base + s.steps * nkv; s.load(p, gr, at, ctx_lens[at])) base += s.steps * nkv, ++at;
                const int rest = F - base, h = rest / s.steps, t = rest - h * s.steps, take = min(s.steps - t, end - F), from = F - t;
                const int row[9] = {x, at, h, t, t + take, s.steps, s.prefix, of.of(from), of.of(from + s.steps - 1)};
                tell(row);
                F += take;
            }
        } else {
            SharedPrefix s;
            for (; f < end; base += s.all(p), ++at) {
                s.load(p, gr, at);
                if (f < base + s.all(p)) break;
            }
            PrefixWalk w;
            memset((void*)&w, unset, sizeof(w));
            w.start(p, gr, f, end, at, base);
            for (int n = 0; w.next(p, gr); ++n) {
                if (n == limit) return -1 - x;
                const int row[9] = {x, w.g, w.h, w.tile, w.p0, w.pages, w.few, w.unit_f / per, (w.unit_f + w.steps - 1) / per};
                tell(row);
            }
        }
    }
    return found;
}

// What step x of a sequence reads: lo, hi, query
extern "C" void shared_step(const int* ctx_lens, int B, int b, const int* starts, const int* shared, int n_groups, int max_pages, int chunk, int share, int x, int* out) {
    SharedArgs p{};
    p.ctx_lens = ctx_lens, p.group_start = starts, p.shared_lens = shared;
    p.B = B, p.n_groups = n_groups, p.max_pages = max_pages, p.nkv = 1, p.nq = 1, p.G = 1, p.th = kSharedRows, p.inv_tile = (1u << 31) / kSharedRows, p.chunk_log = chunk == 64 ? 6 : chunk == 32 ? 5 : 4;
    SharedSeq s;
    p.least_size = 2;
    s.load(p, SharedGroups{starts, shared, n_groups, share != 0}, b, ctx_lens[b]);
    out[2] = s.step(p, x, out[0], out[1]) ? s.first : b;
}

// Where row 0 of (group, head, query i of the group) lies among the prefix's results
extern "C" int shared_row(const int* starts, const int* shared, int g, int h, int i, int max_pages, int nkv, int G) {
    SharedArgs p{};
    p.group_start = starts, p.shared_lens = shared, p.max_pages = max_pages, p.nkv = nkv, p.nq = nkv * G, p.G = G, p.th = kSharedRows / G, p.inv_tile = (unsigned)(((1ull << 32) + 2 * p.th - 1) / (2 * p.th));
    SharedPrefix w;
    w.load(p, SharedGroups{starts, shared, 1 << 30, true}, g);
    return w.row(p, h, i);
}

extern "C" int shared_tiles(int G, int size) {
    SharedArgs p{};
    p.th = kSharedRows / G, p.inv_tile = (unsigned)(((1ull << 32) + 2 * p.th - 1) / (2 * p.th));
    return p.tiles(size);
}
