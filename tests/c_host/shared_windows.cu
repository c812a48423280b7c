// The own list of attention over shared prefixes as a warp looks it up, 32 steps at a time (csrc/shared.cuh: own_sequence, OwnStep), on the host: a lane is an index.
#include "shared.cuh"

using namespace ft;

// The share f0 .. f_end - 1 of a list whose sequence b has steps[b] steps for each of nkv key heads.  out: four numbers a step: sequence, key head, the unit's first and last step; -1 where a
// lane's search leaves the list.  -> windows that were looked up
extern "C" int shared_windows(const int* steps, int B, int nkv, int f0, int f_end, int* out) {
    SharedArgs p{};
    p.B = B, p.nkv = nkv;
    int b0 = 0, base = 0, windows = 0;
    while (base + steps[b0] * nkv <= f0) base += steps[b0++] * nkv;          // as the plan tells the warp
    for (int f = f0; f < f_end; f += 32, ++windows) {
        int begins[32], ends[32], at = base;
        for (int x = 0; x < 32; ++x) {
            begins[x] = at;
            at += b0 + x < B ? steps[b0 + x] * nkv : 0;
            ends[x] = at;
        }
        OwnStep s[32];
        for (int x = 0; x < 32; ++x) {
            const int F = f + x < f_end ? f + x : f_end - 1, l = own_sequence(F, [&](int i) { return ends[i]; }), b = b0 + l;
            int* const row = out + 4 * (F - f0);
            if (b >= B) {
                s[x] = OwnStep{};
                row[0] = row[1] = row[2] = row[3] = -1;
                continue;
            }
            s[x].set(p, F, b, begins[l], steps[b]);
            row[0] = b, row[1] = s[x].head, row[2] = s[x].from, row[3] = s[x].last;
        }
        b0 = s[31].next_seq;
        base = s[31].next_base;
    }
    return windows;
}
