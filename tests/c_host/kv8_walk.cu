// The plan of the 8-bit prompt attention on the host: what the warp that finds a CTA's work does, lane by lane, with the kernel's own arithmetic (csrc/kv8_walk.cuh).
#include <cstring>

#include "kv8_walk.cuh"

using namespace ft;

// Stretches of all CTAs, eleven numbers each: cta, row0, tokens, head, page0, pages, few, pos0, begins, parts, slot.  unset: what fields hold that nobody has written.
// -> how many (at most `room` are written), or -1 - cta where a CTA walks more than `limit`
extern "C" int kv8_stretches(const int* starts, const int* slots, const int* pos0, int n_req, int T, int max_pages, int nkv, int G, int few_pages, int ctas, int room_for_parts,
                             int whole_slack, int unset, int limit, int* out, int room) {
    Kv8Prompt p{};
    p.req_q_start = starts, p.req_slot = slots, p.req_pos0 = pos0;
    p.n_req = n_req, p.T = T, p.max_pages = max_pages, p.nkv = nkv, p.G = G, p.th = 128 / G, p.few_pages = few_pages;
    int found = 0;
    for (int cta = 0; cta < ctas; ++cta) {
        Kv8Sums lane[32];
        int steps = 0, units = 0, most = 0, r0[32], at_steps[32], at_units[32];
        bool grows = true;
        const int chunk = (n_req + 31) / 32;
        for (int i = 0; i < 32; ++i) {
            r0[i] = min(n_req, i * chunk);
            for (int r = r0[i]; r < min(n_req, r0[i] + chunk); ++r) lane[i].add(p, r);
            at_steps[i] = steps, at_units[i] = units;
            steps += lane[i].steps, units += lane[i].units, most = max(most, lane[i].most);
            grows = grows && lane[i].grows;
        }
        const int total = (int)((unsigned)steps * nkv), n_units = (int)((unsigned)units * nkv);
        const int per = (unsigned)(total + ctas - 1) / (unsigned)ctas;
        const bool whole = !room_for_parts || (n_units <= ctas && most + kKv8Start <= per + whole_slack);
        const int len = whole ? n_units : total, each = whole ? 1 : per;
        Kv8Walk w;
        memset((void*)&w, unset, sizeof(w));
        const bool work = w.share(grows, len, each, cta);
        for (int i = 0; work && i < 32; ++i) {
            const int at0 = whole ? at_units[i] : at_steps[i];
            if (!(at0 * nkv <= w.f && w.f < (at0 + (whole ? lane[i].units : lane[i].steps)) * nkv)) continue;
            w.seek(p, whole, r0[i], at0, w.f);
            w.unit(p);
            if (whole) w.f = 0, w.f_end = w.n_steps;
            break;
        }
        for (int n = 0; w.next(p); ++n) {
            if (n == limit) return -1 - cta;
            const Kv8Stretch s = w.stretch(p, per, cta);
            const int row[11] = {cta, s.row0, s.tokens, s.head, s.page0, s.pages, s.few, s.pos0, s.begins, s.parts, s.slot};
            if (found < room) memcpy(out + 11 * found, row, sizeof(row));
            ++found;
        }
    }
    return found;
}

extern "C" int kv8_floor_sum64(unsigned n, unsigned a, unsigned b) { return floor_sum64(n, a, b); }
