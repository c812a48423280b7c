// Attention of one query token per sequence over common prefixes and own tails: out[b][h] = sum_j softmax_j(q . k_j / sqrt(D)) v_j, j < ctx_lens[b], with the first tokens of a
// group's sequences read once for all of them.  The lists of work are in shared.cuh.
//
// One CTA per SM does both kinds of work side by side, since one is bound by the tensor and exponential units and the other by memory:
//   prefix   tcgen05 / TMEM as in attention_tc.cu: a tile of up to 2 * (128 / G) queries in two halves of up to 128 rows (row = query * G + head of the group).  Per page and
//            half S = Q K^T (M128 N64 K=D, the cache's slab as it lies), one thread a row for the softmax, P to tensor memory over the scores that it came from,
//            O += P V (M128 N=D K64).  Queries that fill one half only go to both halves, which take every other page each.  All rows see all pages: the only
//            mask is the end of the last one.
//   own      a warp walks a share of its own: chunks of 16 or 8 KB by bulk copies that it asks for itself, two of them on their way while it multiplies (mma.sync, the
//            query heads of a key head in the columns).  No warp waits for another.
// Each share's results are O, maximum and sum of its rows; a second kernel puts them together in their order.
//
// Measured in a graph, us (launch included), what it has to read at 6.46 TB/s in brackets: 64 sequences behind one prefix of 2048 tokens, up to 600 own (329 on
// average), 32 heads of 64 over 8, 20.6 (7.4), a key head for each of 16 of 128 52.5 (29.4), 16 of 64 over 2 15.6 (1.9); 24 behind one of 16001, up to 300 own, 32 heads of 128 over 8,
// 25.5 (12.6); two behind 517, 10.0 (0.2).  What bounds it: 4.4 us from the launch to the first page asked for (the
// plan 2.0, what the shares begin with 1.4, a copy 1.3), then memory (74 MB in about 11 us) or, where all 256 rows of a tile are in use, the softmax (2000 clocks a page and
// half pair of which 1024 are exponentials), 1 to 2 us to write O, and the second kernel, 3.5 to 6 with its launch.
#include "common.cuh"
#include "ft_internal.h"
#include "shared.cuh"

namespace ft {

constexpr float kSharedLog2E = 1.4426950408889634f;
// Probabilities are formed 2^6 times their size, so that fp16's normal numbers reach down to 2^-20 of the largest; a running maximum may lag by 2^8
constexpr float kSharedTop = 6.f, kSharedGrow = 8.f;

// Groups of four warps: warp 0 copies the prefix's pages, 1 and 2 issue the halves' products, 3 owns tensor memory and walks the list; 4 .. 11 softmax (half = (warp - 4) / 4); 12 .. 15 own
constexpr int SH_THREADS = 512, SH_WARPS = SH_THREADS / 32;
constexpr int SH_REGS = 128, SH_REGS_ISSUE = 88, SH_REGS_SOFT = 144, SH_REGS_OWN = 136;
static_assert(SH_REGS_ISSUE + 2 * SH_REGS_SOFT + SH_REGS_OWN <= 4 * SH_REGS, "what the block is launched with");
constexpr int SH_SOFT = 256;
constexpr int SH_TOLD = 4, SH_LISTENERS = 11;    // stretches told ahead; warps that hear of them
constexpr int SH_STRETCH = 64;                   // times the limit, for what takes a whole stretch: it may be a million keys
// Steps of a share of the prefix at least: fewer CTAs have one, with fewer results, and the others more of the own list.  Per share 3 / 4 / 5 / 6 steps, us: 64 sequences behind 2048
// tokens 22.5 / 20.4 / 20.6 / 20.6, 128 behind two prefixes of 1500 22.3 / 22.4 / 22.6 / 22.8, 37 behind five of 4099 23.0 / 23.0 / 23.0 / 23.3
constexpr int SH_LEAST = 4;
constexpr int SH_COST = 2;                       // steps of the prefix that cost a warp on its SM one of its own (1 / 2 / 3 / none: the first of these 23.7 / 20.4 / 21.9 / 22.3)
constexpr int SH_LIST = 100;                     // groups whose lists are kept in shared memory
constexpr int SH_PIECE = kKvTile * 128;          // [64 tokens][64 dims] in fp16

__device__ int g_shared_waits;                   // 1: a wait ran out on this device (ft_attn_shared_waits)

template <int D>
struct Shared {
    static constexpr int KH = D / 64;
    static constexpr int TILE = 2 * KH * SH_PIECE;                           // K | V of a page
    // of the prefix.  Three at least: a half that has every other page asks for its scores two of its own pages ahead, whose stage must not wait for a product behind them
    static constexpr int STAGES = D == 64 ? 4 : 3, SLAB = TILE / 2, TOKENS = 16;
    static constexpr int AHEAD = 2;                                          // pages that keys are copied ahead of values
    static constexpr int QBLK = kSharedRows * 128;                           // [128 rows][64 dims]
    static constexpr int OWN_WARPS = 4, OWN_STAGES = 2;
    // tokens: what is left of shared memory, for four warps (at heads of 128 two warps with 32 tokens each: 128 sequences with 150 own 30.3 us, four with 16 24.5)
    static constexpr int CHUNK = D == 64 ? 64 : 16;
    static constexpr int CHUNK_BYTES = 2 * CHUNK * D * 2, HALF = CHUNK_BYTES / 2;        // keys | values; of each D / 64 pieces of [CHUNK][64 dims]
    static constexpr int KV = 2 * KH * QBLK, OWN = KV + STAGES * TILE, SMEM = 1024 + OWN + OWN_WARPS * OWN_STAGES * CHUNK_BYTES;
    // tensor memory: scores [half][2][64 columns] (probabilities, pairs of fp16, over the first 32 of them), O [half][D]
    static constexpr int COL_S = 0, COL_O = 256, COLS = 512;
    static_assert(COL_O + 2 * D <= COLS, "tensor memory");
    static_assert(SMEM <= 232448 - 2048, "shared memory (the rest is what the kernel declares)");
};

// A wait that ends, in a few instructions: calls of ten microseconds touch most of their code for the first time.  (With waits and loops unrolled and the walk in every role
// the two kernels were 126 KB and a call over 16001 tokens took 35.8 us; with a loop here and the walk in one warp, 78 KB, 31.)
// Who gives up touches none of the barriers again: what it skipped would make it take one phase for another.
__device__ __forceinline__ bool shared_wait(uint64_t* bar, uint32_t parity, volatile int* dead, int times = 1) {
#pragma unroll 1
    for (int i = 0; i < times * kWaitLimit; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*dead) return false;
    }
    *dead = 1;
    return false;
}

// Whether two of them are over already: tries that do not sleep, on their way together
__device__ __forceinline__ void shared_over(uint64_t* bar0, uint32_t parity0, uint64_t* bar1, uint32_t parity1, bool& over0, bool& over1) {
    uint32_t x, y;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%2], %3;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 q, [%4], %5;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "selp.u32 %1, 1, 0, q;\n\t}\n"
        : "=r"(x), "=r"(y)
        : "r"(smem_u32(bar0)), "r"(parity0), "r"(smem_u32(bar1)), "r"(parity1)
        : "memory");
    over0 = x, over1 = y;
}

// floats of an own part: O [G][D], (m, l) of the heads; on 16 bytes
__host__ __device__ __forceinline__ int shared_part(int G, int d) { return (G * (d + 2) + 3) / 4 * 4; }

// ------------------------------------------------------------------ own part
// A warp's state of one (sequence, key head): S[token][query] = K Q^T with 16 tokens in the rows of mma.sync; the probabilities, transposed 8 x 8 at a time, are the other
// operand of O^T[dim][query] = V^T P^T, where all 16 rows are dims.
template <int D>
struct SharedQuery {
    static constexpr int CHUNK = Shared<D>::CHUNK, TOGETHER = 128 / D;        // blocks of 16 tokens that are multiplied together
    uint32_t q[D / 16][2];
    float o[D / 16][4];                  // O^T: dims 16 i + g (+ 8), queries 2 tq (+ 1) at [i][2 * upper + (query & 1)]
    float m[2], l[2];                    // of queries 2 tq (+ 1): reference, this lane's tokens' sum

    static __device__ __forceinline__ int at(int t, int c) { return (c >> 3) * (CHUNK * 128) + t * 128 + (((c & 7) ^ (t & 7)) << 4); }       // 16-byte chunk c of token t

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
    }
    // tokens lo .. hi - 1 of the chunk at `tile` (an address in shared memory) as far as they are among the 16 * TOGETHER from t0 on; hidden values are zeros
    __device__ __forceinline__ void blocks(uint32_t tile, int t0, int lo, int hi, float scale_log2, int lane) {
        const int g = lane >> 2;
        float s[TOGETHER][4], most[2] = {-INFINITY, -INFINITY};
        // operands of several products are asked for ahead of the first (one by one, each waited for its own 33 clocks)
        uint32_t x[8][4];
#pragma unroll
        for (int i = 0; i < 8; ++i) ldmatrix_x4(tile + at(t0 + i / (D / 16) * 16 + (lane & 15), 2 * (i % (D / 16)) + (lane >> 4)), x[i][0], x[i][1], x[i][2], x[i][3]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int b = i / (D / 16), ks = i % (D / 16);
            if (ks == 0) s[b][0] = s[b][1] = s[b][2] = s[b][3] = 0.f;
            mma_f16_16816(s[b], x[i][0], x[i][1], x[i][2], x[i][3], q[ks][0], q[ks][1]);
        }
        if (lo > t0 || hi < t0 + 16 * TOGETHER) {
#pragma unroll
            for (int b = 0; b < TOGETHER; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int t = t0 + 16 * b + 8 * (e >> 1) + g;
                    s[b][e] = t >= lo && t < hi ? s[b][e] : -INFINITY;
                }
        }
#pragma unroll
        for (int b = 0; b < TOGETHER; ++b) {
            most[0] = fmaxf(most[0], fmaxf(s[b][0], s[b][2]));
            most[1] = fmaxf(most[1], fmaxf(s[b][1], s[b][3]));
        }
        most[0] *= scale_log2, most[1] *= scale_log2;
        if (__any_sync(0xffffffffu, most[0] > m[0] + kSharedGrow || most[1] > m[1] + kSharedGrow)) {     // after the first chunk rarely
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) most[e] = fmaxf(most[e], __shfl_xor_sync(0xffffffffu, most[e], x));
                const float m_new = fmaxf(m[e], most[e]);
                const float keep = m_new == -INFINITY ? 1.f : ex2_fast(m[e] - m_new);
                l[e] *= keep;
                m[e] = m_new;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) o[i][e] *= keep, o[i][2 + e] *= keep;
            }
        }
        const float r0 = kSharedTop - (m[0] == -INFINITY ? 0.f : m[0]), r1 = kSharedTop - (m[1] == -INFINITY ? 0.f : m[1]);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            ldmatrix_x4_trans(tile + Shared<D>::HALF + at(t0 + i / (D / 16) * 16 + (lane & 7) + (lane >> 4) * 8, 2 * (i % (D / 16)) + (lane >> 3 & 1)), x[i][0], x[i][1], x[i][2], x[i][3]);
#pragma unroll
        for (int b = 0; b < TOGETHER; ++b) {
            uint32_t pb[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float p0 = ex2_fast(fmaf(s[b][2 * h], scale_log2, r0)), p1 = ex2_fast(fmaf(s[b][2 * h + 1], scale_log2, r1));
                l[0] += p0;
                l[1] += p1;
                const __half2 t = __floats2half2_rn(p0, p1);
                asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(pb[h]) : "r"(*reinterpret_cast<const uint32_t*>(&t)));
            }
#pragma unroll
            for (int n = 0; n < D / 16; ++n) mma_f16_16816(o[n], x[b * (D / 16) + n][0], x[b * (D / 16) + n][1], x[b * (D / 16) + n][2], x[b * (D / 16) + n][3], pb[0], pb[1]);
        }
    }
    // sums over all lanes' tokens
    __device__ __forceinline__ void total(float* sum) const {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            sum[e] = l[e];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], x);
        }
    }
};

// The share f0 .. f_end - 1 of the own list; sequence b0 begins at `base` of it, and the share in b0.  Thirty-two steps at a time, a lane each, the warp finds out what they
// read; copies run ahead and results are written whichever sequences the steps belong to.
template <int D>
__device__ __forceinline__ void shared_own(const SharedArgs& p, const SharedGroups& gr, int f0, int f_end, int b0, int base, const OwnShares& shares, int warp, uint8_t* ring, uint64_t* full,
                                           volatile int* dead, int* err) {
    using C = Shared<D>;
    constexpr int S = C::OWN_STAGES, CH = C::CHUNK;
    const int lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3, G = p.G;
    if (f0 >= f_end) return;
    const uint64_t pol = policy_evict_first();                               // every byte is read once
    bool ok = true;
    int it = 0, asked = 0;                                                   // chunks of the share so far, with a page: a stage's phase follows from the count
    SharedQuery<D> a;
    uint32_t q_next[D / 16][2];                                              // the next unit's queries, on their way while this one's chunks are multiplied
    auto query_of = [&](int u) {
        const __half* row = p.q + ((size_t)u * G + g) * D + 2 * tq;          // (unit = sequence * key heads + key head)
        const bool on = g < G && u < p.B * p.nkv;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            q_next[ks][0] = on ? *reinterpret_cast<const uint32_t*>(row + ks * 16) : 0u;
            q_next[ks][1] = on ? *reinterpret_cast<const uint32_t*>(row + ks * 16 + 8) : 0u;
        }
    };
    // lane x: step x of the 32 at hand
    int unit_x = 0, from_x = 0, last_x = 0, seen_x = 0;                      // seen: of the chunk's tokens, first and behind the last one in bytes
    const uint8_t* src_x = nullptr;                                          // the chunk's first keys in the cache
    bool prefix_x = false;
    unsigned paged = 0, to_ask = 0;
    int unit = -1, from = 0, last = 0;                                       // the unit under way: where it begins in the list, its last step
    bool prefix = false;
#pragma unroll 1
    for (int f = f0;; ++f) {
        const int x = (f - f0) & 31;
        if (x == 0 && f < f_end) {
            // ---- the next 32 steps, in the 32 sequences from b0 on (own_sequence says why they are there)
            const int b = b0 + lane;
            SharedSeq s;
            int row = -1, led_row = -1;
            s.steps = 0;
            if (b < p.B) {
                row = p.row_of(b);
                s.load(p, gr, b, p.ctx_lens[b]);
                if (s.lead) led_row = p.row_of(s.first);
            }
            const int span = s.steps * p.nkv;
            int end = span;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, end, o);
                if (lane >= o) end += up;
            }
            end += base;
            const int F = min(f + lane, f_end - 1);
            const int l = own_sequence(F, [&](int i) { return __shfl_sync(0xffffffffu, end, i); });
            SharedSeq w;
            w.ctx = __shfl_sync(0xffffffffu, s.ctx, l);
            w.begin = __shfl_sync(0xffffffffu, s.begin, l);
            w.lead = __shfl_sync(0xffffffffu, s.lead, l);
            w.steps = __shfl_sync(0xffffffffu, s.steps, l);
            prefix_x = __shfl_sync(0xffffffffu, (int)s.prefix, l);
            const int base_l = __shfl_sync(0xffffffffu, end - span, l), r_own = __shfl_sync(0xffffffffu, row, l), r_led = __shfl_sync(0xffffffffu, led_row, l);
            OwnStep step;
            step.set(p, F, b0 + l, base_l, w.steps);
            from_x = step.from;
            last_x = step.last;
            unit_x = (b0 + l) * p.nkv + step.head;
            int lo, hi, page = -1;
            const int r = w.step(p, F - from_x, lo, hi) ? r_led : r_own, at = lo / CH * CH;
            if (f + lane < f_end && lo < hi && r >= 0) page = p.page_table[(size_t)r * p.max_pages + at / kKvTile];
            seen_x = lo - at | hi - at << 8;
            src_x = p.cache + ((size_t)page * p.nkv + step.head) * C::TILE + at % kKvTile * 128;
            b0 = __shfl_sync(0xffffffffu, step.next_seq, 31);
            base = __shfl_sync(0xffffffffu, step.next_base, 31);
            to_ask = paged = __ballot_sync(0xffffffffu, page >= 0 && page < p.num_pages);
            if (unit < 0) query_of(__shfl_sync(0xffffffffu, unit_x, 0));
        }
        // ---- copies run S chunks ahead
#pragma unroll 1
        while (ok && to_ask && asked < it + S) {
            const int y = __ffs(to_ask) - 1, stage = asked % S;
            uint8_t* dst = ring + stage * C::CHUNK_BYTES;
            const uint8_t* src = (const uint8_t*)__shfl_sync(0xffffffffu, (unsigned long long)src_x, y);
            if (elect_one()) {
                mbar_expect_tx(&full[stage], C::CHUNK_BYTES);
                if (CH == kKvTile) {
                    tma_bulk_g2s(dst, src, C::CHUNK_BYTES, &full[stage], pol);
                } else {                                                     // 2 D / 64 pieces
#pragma unroll
                    for (int j = 0; j < 2 * C::KH; ++j) tma_bulk_g2s(dst + j * (CH * 128), src + j * SH_PIECE, CH * 128, &full[stage], pol);
                }
            }
            to_ask &= to_ask - 1;
            ++asked;
        }
        const int u = f < f_end ? __shfl_sync(0xffffffffu, unit_x, x) : -1;
        if (u != unit) {
            if (unit >= 0) {
                // ---- what this warp has of the unit that ends here
                float sum[2];
                a.total(sum);
                if (!ok) {                                                   // NaN for all that this (sequence, head) says
                    *err = 1;
                    a.m[0] = a.m[1] = 0.f;
                    sum[0] = sum[1] = NAN;
                }
                if (lane == 0 && from >= f0) p.own_units[unit] = make_int4(warp, shares.of(last), prefix, 0);
                float* part = p.own_parts + (size_t)(unit + warp) * shared_part(G, D);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int head = 2 * tq + e;
                    if (head >= G) continue;
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        part[head * D + 16 * i + g] = a.o[i][e];
                        part[head * D + 16 * i + 8 + g] = a.o[i][2 + e];
                    }
                    if (g == 0) *reinterpret_cast<float2*>(part + G * D + 2 * head) = make_float2(a.m[e], sum[e]);
                }
            }
            if (u < 0) break;
            unit = u;
            from = __shfl_sync(0xffffffffu, from_x, x);
            last = __shfl_sync(0xffffffffu, last_x, x);
            prefix = __shfl_sync(0xffffffffu, (int)prefix_x, x);
            a.clear();
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) a.q[ks][0] = q_next[ks][0], a.q[ks][1] = q_next[ks][1];
            query_of(u + 1);
        }
        if (!ok || !(paged >> x & 1)) continue;
        const int stage = it % S;
        ok = __all_sync(0xffffffffu, shared_wait(&full[stage], it / S & 1, dead));
        if (!ok) continue;
        ++it;
        const int seen = __shfl_sync(0xffffffffu, seen_x, x), lo = seen & 255, hi = seen >> 8;
        uint8_t* tile = ring + stage * C::CHUNK_BYTES;
        constexpr int STEP = 16 * SharedQuery<D>::TOGETHER;                  // (steps that nothing sees are left out)
        if (lo > 0 || hi < CH) {                                             // hidden values may be anything: 0 * infinity is none
#pragma unroll 1
            for (int b = lo / STEP * STEP; b < (hi + STEP - 1) / STEP * STEP; b += 16) {
                const int from_t = lo - b, to_t = hi - b;
                if (from_t <= 0 && to_t >= 16) continue;
#pragma unroll
                for (int j = 0; j < D / 16; ++j) {
                    const int v = lane + 32 * j, k = v / (D / 8);
                    if (k < from_t || k >= to_t) *reinterpret_cast<uint4*>(tile + C::HALF + SharedQuery<D>::at(b + k, v % (D / 8))) = make_uint4(0u, 0u, 0u, 0u);
                }
            }
            fence_proxy_async();                                             // ahead of the next copy into this stage
            __syncwarp();
        }
        if constexpr (CH == STEP) {
            a.blocks(smem_u32(tile), 0, lo, hi, p.scale_log2, lane);
        } else {
#pragma unroll 1
            for (int t = lo / STEP * STEP; t < hi; t += STEP) a.blocks(smem_u32(tile), t, lo, hi, p.scale_log2, lane);
        }
        __syncwarp();                                                        // all lanes have read it: the next copy may come
    }
    if (lane == 0)
#pragma unroll 1
        for (int i = it; i < asked; ++i)                                     // nothing may still be on its way into this CTA's memory when it ends
#pragma unroll 1
            for (int k = 0; k < kWaitLimit && !mbar_try_wait(&full[i % S], i / S & 1); ++k) {}
}

// A page of the prefix that lands in a stage tells who waits for it by one of three barriers: of the pages that half 0 alone takes, of those of half 1, of those of both.  (With
// one barrier a half that takes every other page could see only every second phase of a stage, and a phase looks complete while the one before it is under way.)
// Each role keeps the phases of the barriers that it uses: one bit each, turned by every page.
struct SharedPhases {
    uint32_t bits = 0;
    int at;                              // the barrier of the last page asked for
    __device__ __forceinline__ uint32_t next(int stages, int stage, int set) {
        at = set * stages + stage;
        const uint32_t parity = bits >> at & 1;
        bits ^= 1u << at;
        return parity;
    }
};

// Exclusive sums of four numbers over the block's threads, and whether all say yes; `all` the sums of all
__device__ __forceinline__ bool shared_before(const int* mine, int (*warp_s)[4], int* before, int* all, bool yes) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = mine[k];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int up = __shfl_up_sync(0xffffffffu, x[k], o);
            if (lane >= o) x[k] += up;
        }
    if (lane == 31)
#pragma unroll
        for (int k = 0; k < 4; ++k) warp_s[warp][k] = x[k];
    yes = __syncthreads_and(yes);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        before[k] = x[k] - mine[k];
        all[k] = 0;
    }
#pragma unroll 4
    for (int w = 0; w < SH_WARPS; ++w) {                                     // (one 16-byte read a warp, the same for all lanes)
        const int4 v = *reinterpret_cast<const int4*>(warp_s[w]);
        const int s[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (w < warp) before[k] += s[k];
            all[k] += s[k];
        }
    }
    return yes;
}

template <int D>
__global__ void __launch_bounds__(SH_THREADS, 1)
shared_attn_kernel(const __grid_constant__ SharedArgs p) {
    using C = Shared<D>;
    constexpr int KH = C::KH;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t k_full[3 * C::STAGES], v_full[3 * C::STAGES], k_empty[C::STAGES], v_empty[C::STAGES];        // (full: see SharedPhases)
    __shared__ uint64_t own_full[C::OWN_WARPS * C::OWN_STAGES];
    __shared__ uint64_t q_full[2];                                           // the queries of a half
    __shared__ uint64_t s_full[2][2], p_full[2][2], pv_done[2][2];           // half, buffer: scores are in tensor memory; probabilities are; O += P V retired
    __shared__ uint64_t told_full[SH_TOLD], told_empty[SH_TOLD];             // a stretch has been told; all have done with it
    __shared__ SharedStretch told[SH_TOLD];
    __shared__ uint64_t met;                                                 // all softmax warps are here
    __shared__ uint64_t drained[2];                                          // all products of a half retired
    __shared__ int tokens_s[C::TOKENS];                                      // of the last pages copied; 0: the page is not there
    __shared__ __align__(16) int sums_s[SH_WARPS][4];
    __shared__ int start_s[SH_LIST + 1], lens_s[SH_LIST];
    __shared__ int2 prefix_at, own_at[C::OWN_WARPS];                         // the group (sequence) that a share begins in, and where that begins
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int dead;
    int* const err = &g_shared_waits;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < 3 * C::STAGES; ++s) mbar_init(&k_full[s], 1), mbar_init(&v_full[s], 1);
        for (int s = 0; s < C::STAGES; ++s) mbar_init(&k_empty[s], 2), mbar_init(&v_empty[s], 2);
        for (int s = 0; s < C::OWN_WARPS * C::OWN_STAGES; ++s) mbar_init(&own_full[s], 1);
        for (int s = 0; s < SH_TOLD; ++s) mbar_init(&told_full[s], 1), mbar_init(&told_empty[s], SH_LISTENERS);
        mbar_init(&met, SH_SOFT / 32);
        for (int h = 0; h < 2; ++h) {
            mbar_init(&q_full[h], kSharedRows / 32);
            mbar_init(&drained[h], 1);
            for (int s = 0; s < 2; ++s) mbar_init(&s_full[h][s], 1), mbar_init(&p_full[h][s], kSharedRows / 32), mbar_init(&pv_done[h][s], 1);
        }
        fence_mbar_init();
        dead = p.give_up;
    }
    if (warp == 3) {
        tmem_alloc(&tmem_slot, C::COLS);
        tmem_relinquish();
    }
    pdl_wait();

    // ---------------- the plan: every CTA adds up both lists, a run of groups and one of sequences a thread.  A list of groups that does not grow, or leaves the batch,
    // shares nothing
    SharedGroups gr{p.group_start, p.shared_lens, p.n_groups, true};
    int prefix_f, prefix_end, prefix_per, own_total;
    OwnShares shares;
    {
        // (groups from the last threads back, so that few of them and few sequences are different warps' work)
        const int gc = (p.n_groups + SH_THREADS - 1) / SH_THREADS, g0 = max(0, p.n_groups - (SH_THREADS - tid) * gc), g1 = max(0, p.n_groups - (SH_THREADS - 1 - tid) * gc);
        const int bc = (p.B + SH_THREADS - 1) / SH_THREADS, b0 = min(p.B, tid * bc), b1 = min(p.B, b0 + bc);
        const int ctx0 = b0 < b1 ? p.ctx_lens[b0] : 0;
        if (bc == 1 && b0 < b1 && p.req_slot) asm volatile("prefetch.global.L1 [%0];" ::"l"(p.req_slot + b0));       // the own warps look these up first
        // Groups that are looked for are kept in shared memory: two of them 22.5 us a call, not kept 23.3, five 23.1 and 24.0; for one alone the round through it
        // costs more than it saves (21.0 and 20.4)
        if (p.n_groups > 1 && p.n_groups <= SH_LIST) {
            if (tid <= p.n_groups) start_s[tid] = p.group_start[tid];
            if (tid < p.n_groups) lens_s[tid] = p.shared_lens[tid];
            gr.start = start_s;
            gr.lens = lens_s;
            __syncthreads();
        }
        bool grows = true;
        // prefix steps and own steps where prefixes are shared, own steps where they are not, pages saved
        int mine[4], before[4], all[4];
#pragma unroll 1
        for (int g = g0; g < g1; ++g) grows = grows && gr.start[g] >= 0 && gr.start[g] <= gr.start[g + 1] && gr.start[g + 1] <= p.B;
#pragma unroll 1
        for (;;) {
            mine[0] = mine[1] = mine[2] = mine[3] = 0;
#pragma unroll 1
            for (int g = g0; g < g1 && grows && gr.n; ++g) {
                SharedPrefix w;
                w.load(p, gr, g);
                mine[0] += w.all(p);
                mine[3] = min(mine[3] + gr.saves(p, g), 1 << 20);
            }
#pragma unroll 1
            for (int b = b0; b < b1; ++b) {
                SharedSeq s;
                s.load(p, gr, b, b == b0 ? ctx0 : p.ctx_lens[b]);
                mine[1] += s.steps;
                mine[2] += s.steps_alone(p);
            }
            if (shared_before(mine, sums_s, before, all, grows) || gr.n == 0) break;
            gr.n = 0;
            __syncthreads();
        }
        // Sharing costs a call about 2 us, and a step of the prefix more than an own one (least_size, least_pages: launch_shared)
        gr.share = all[3] >= p.least_pages;
        if (!gr.share) {
            mine[0] = all[0] = 0;
            mine[1] = mine[2];
            before[1] = before[2];
            all[1] = all[2];
        }
        own_total = all[1] * p.nkv;
        const int own_per = (int)((unsigned)(own_total + gridDim.x * C::OWN_WARPS - 1) / (gridDim.x * C::OWN_WARPS));
        // Prefix shares of four steps at least where the own ones are as long: half the results to put together
        prefix_per = max((int)((unsigned)(all[0] + gridDim.x - 1) / gridDim.x), min(SH_LEAST, own_per));
        shares.set(own_total, C::OWN_WARPS, gridDim.x, (int)((unsigned)(all[0] + prefix_per - 1) / (unsigned)prefix_per), prefix_per / SH_COST);
        prefix_f = min(prefix_per * (int)blockIdx.x, all[0]);
        prefix_end = min(prefix_f + prefix_per, all[0]);
        if (before[0] <= prefix_f && prefix_f < before[0] + mine[0]) {
            SharedPrefix w;
            int g = g0;
#pragma unroll 1
            for (;; ++g) {
                w.load(p, gr, g);
                const int n = w.all(p);
                if (before[0] + n > prefix_f) break;
                before[0] += n;
            }
            prefix_at = make_int2(g, before[0]);
        }
        const int from = before[1] * p.nkv, to = from + mine[1] * p.nkv;
#pragma unroll 1
        for (int w = 0; w < C::OWN_WARPS; ++w) {
            const int f = shares.begin(w, blockIdx.x);
            if (from <= f && f < to) {
                int b = b0, at = from;
                if (bc > 1)
#pragma unroll 1
                    for (;; ++b) {
                        SharedSeq s;
                        s.load(p, gr, b, p.ctx_lens[b]);
                        if (f < at + s.steps * p.nkv) break;
                        at += s.steps * p.nkv;
                    }
                own_at[w] = make_int2(b, at);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    uint32_t k_bits = 0, v_bits = 0;                                         // of the warp that copies: the phases of what it has asked for
    bool ok = true;                                                          // false: a wait ran out
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, shared_wait(bar, parity, &dead)); };
    // the n-th stretch of the prefix's share, or one without pages behind the last; and this warp's word that it has done with it
    auto hear = [&](int n) {
        ok = ok && __all_sync(0xffffffffu, shared_wait(&told_full[n % SH_TOLD], n / SH_TOLD & 1, &dead, SH_STRETCH));
        SharedStretch w = told[n % SH_TOLD];
        if (!ok) w.pages = 0;
        return w;
    };
    auto heard = [&](int n) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&told_empty[n % SH_TOLD]);
    };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(SH_REGS_ISSUE));
        if (warp == 3) {
            // ---------------- the walk
            if (lane == 0) {
                PrefixWalk w;
                w.start(p, gr, prefix_f, prefix_end, prefix_at.x, prefix_at.y);
#pragma unroll 1
                for (int n = 0, more = 1; more; ++n) {
                    more = w.next(p, gr);
                    if (!shared_wait(&told_empty[n % SH_TOLD], (n / SH_TOLD & 1) ^ 1, &dead, SH_STRETCH)) break;
                    SharedStretch s{};
                    if (more) s = w.stretch(p, prefix_per);
                    told[n % SH_TOLD] = s;
                    mbar_arrive(&told_full[n % SH_TOLD]);
                }
            }
            __syncwarp();
        } else if (warp == 0) {
            // ---------------- copies of the prefix: a page's keys, and the values of the page two ahead of it, which are needed that much later.  (Never a circle: keys wait for
            // products of keys STAGES pages back, which wait for products of values further back than those that are copied behind them.)
            // What a warp asks shared memory for comes back after some 200 clocks here, behind the exponentials of the same scheduler.  So both empty stages are asked for at once, and one
            // elected thread copies (with a lane picked by its number the compiler cannot know that it is alone): with one after the other a page took 1350 to 2050 clocks, whatever its
            // size, now 1000 (one prefix of 40960 tokens, heads of 64: for 8 queries 36.7 -> 29.8 us, for 65 123 -> 65.8).  A lane for each kind was slower (35.8, 116).
            const uint64_t pol = policy_evict_first();
            SharedPhases phases[2];                                          // keys, values
            int at[2] = {0, 0};                                              // the next stages
            uint32_t turn[2] = {1, 1};
            int n = 0, k = 0, k1 = 0, my_page = -1, row = -1;                // stretches heard; of the 32 pages at hand: the next, how many
            const uint8_t* from[C::AHEAD + 1];                               // the last pages (null: not there), the newest first, and their sets
            int set[C::AHEAD + 1], page = -1;
            SharedStretch w;
            w.pages = 0;
            int p0 = 0, p1 = 0;                                              // pages of the stretch that are not at hand yet
            bool more = true;
#pragma unroll 1
            for (int drain = 0, it = 0; drain < C::AHEAD; ++it) {
                if (more && k == k1) {
                    if (p0 == p1) {
                        if (n) heard(n - 1);
                        w = hear(n++);
                        more = w.pages != 0;
                        p0 = w.p0;
                        p1 = p0 + w.pages;
                        row = more ? p.row_of(w.seq0) : -1;
                    }
                    my_page = p0 + lane < p1 && row >= 0 ? p.page_table[(size_t)row * p.max_pages + p0 + lane] : -1;
                    if (my_page >= p.num_pages) my_page = -1;
                    k = 0;
                    k1 = min(32, p1 - p0);
                    p0 += k1;
                    page = __shfl_sync(0xffffffffu, my_page, 0);
                }
                if (!more) ++drain;
                const int tile = p0 - k1 + k, next_page = __shfl_sync(0xffffffffu, my_page, (k + 1) & 31);
#pragma unroll
                for (int i = C::AHEAD; i > 0; --i) from[i] = from[i - 1], set[i] = set[i - 1];
                from[0] = page >= 0 ? p.cache + ((size_t)page * p.nkv + w.h) * C::TILE : nullptr;
                set[0] = w.few ? (tile - w.p0) & 1 : 2;
                if (ok) {
                    bool over[2];
                    const uint8_t* const src[2] = {from[0], from[C::AHEAD]};
                    shared_over(&k_empty[at[0]], turn[0], &v_empty[at[1]], turn[1], over[0], over[1]);
#pragma unroll
                    for (int kind = 0; kind < 2; ++kind) {
                        if (!ok || (kind ? it < C::AHEAD : !more)) continue;
                        if (!__all_sync(0xffffffffu, over[kind])) ok = wait((kind ? v_empty : k_empty) + at[kind], turn[kind]);       // (one lane may have seen it later than another)
                        if (!ok) continue;
                        phases[kind].next(C::STAGES, at[kind], set[kind * C::AHEAD]);
                        uint64_t* const full = (kind ? v_full : k_full) + phases[kind].at;
                        if (elect_one()) {
                            // (keys are copied when those STAGES back have been multiplied, which is when the scores of eight back were read)
                            if (kind == 0) tokens_s[it % C::TOKENS] = page >= 0 ? min(kKvTile, w.tokens - tile * kKvTile) : 0;
                            if (src[kind]) {
                                mbar_expect_tx(full, C::SLAB);
                                tma_bulk_g2s(smem + C::KV + (kind * C::STAGES + at[kind]) * C::SLAB, src[kind] + kind * C::SLAB, C::SLAB, full, pol);
                            } else {
                                mbar_arrive(full);
                            }
                        }
                        if (++at[kind] == C::STAGES) at[kind] = 0, turn[kind] ^= 1;
                    }
                }
                page = next_page;
                if (more) ++k;
            }
            k_bits = phases[0].bits;
            v_bits = phases[1].bits;
            __syncwarp();
        } else {
            // ---------------- products, one warp a half
            constexpr uint32_t idesc_qk = umma_idesc_f16(kSharedRows, kKvTile, false), idesc_pv = umma_idesc_f16(kSharedRows, D, true);
            const int h = warp - 1;
            const bool lead = elect_one();
            {
                const uint64_t q_desc = umma_desc_k128(smem_u32(smem + h * KH * C::QBLK)), k_desc = umma_desc_k128(smem_u32(smem + C::KV)),
                               v_desc = umma_desc_mn128(smem_u32(smem + C::KV + C::STAGES * C::SLAB));
                const uint32_t s_at = tmem + C::COL_S + h * 128, o_at = tmem + C::COL_O + h * D;
                SharedPhases k_phases, v_phases;
                int base = 0, n_qk = 0, n_pv = 0, n_q = 0;                   // pages of the share, products of this half, stretches of this half so far
                struct Landing { uint64_t* bar; uint32_t parity; bool over; };
                auto landing = [&](SharedPhases& phases, uint64_t* full, int page, bool alone) {       // page: counted over the whole share; alone: the other half has no use for it
                    const uint32_t parity = phases.next(C::STAGES, page % C::STAGES, alone ? h : 2);
                    return Landing{full + phases.at, parity, false};
                };
                auto issue_qk = [&](int page, bool alone, const Landing& k_in) {
                    const int s = page % C::STAGES, buf = n_qk & 1;
                    ok = k_in.over || shared_wait(k_in.bar, k_in.parity, &dead);
                    if (!ok) return;
                    ++n_qk;
                    tc_fence_after();
                    const uint64_t b = k_desc + (uint64_t)(s * (C::SLAB >> 4));
#pragma unroll
                    for (int kh = 0; kh < KH; ++kh)
#pragma unroll
                        for (int k = 0; k < 4; ++k) umma_bf16(s_at + buf * 64, q_desc + kh * (C::QBLK >> 4) + 2 * k, b + kh * (SH_PIECE >> 4) + 2 * k, idesc_qk, (kh | k) != 0);
                    umma_commit(&s_full[h][buf]);
                    umma_commit(&k_empty[s]);
                    if (alone) umma_commit(&k_empty[s]);
                };
                auto issue_pv = [&](int page, bool first, bool alone, const Landing& v_in) {
                    const int s = page % C::STAGES, buf = n_pv & 1;
                    ok = shared_wait(&p_full[h][buf], n_pv >> 1 & 1, &dead) && (v_in.over || shared_wait(v_in.bar, v_in.parity, &dead));
                    if (!ok) return;
                    ++n_pv;
                    tc_fence_after();
                    const uint64_t b = v_desc + (uint64_t)(s * (C::SLAB >> 4));
#pragma unroll
                    for (int k = 0; k < kKvTile / 16; ++k) umma_f16_ts(o_at, s_at + buf * 64 + 8 * k, b + k * (2048 >> 4), idesc_pv, k != 0 || !first);
                    umma_commit(&pv_done[h][buf]);
                    umma_commit(&v_empty[s]);
                    if (alone) umma_commit(&v_empty[s]);
                };
#pragma unroll 1
                for (int n = 0;; ++n) {
                    const SharedStretch w = hear(n);
                    if (w.pages == 0) break;
                    const int mine = w.of_half(h);
                    auto page_of = [&](int i) { return base + (w.few ? h + 2 * i : i); };      // page i of this half
                    if (lead && ok && mine) {
                        ok = shared_wait(&q_full[h], n_q & 1, &dead);
                        tc_fence_after();
                        // Scores run two pages ahead, issued behind the product that reads the probabilities in their buffer
#pragma unroll 1
                        for (int i = -2; ok && i < mine; ++i) {
                            Landing v_in{v_full, 0, false}, k_in{k_full, 0, false};
                            if (i >= 0) v_in = landing(v_phases, v_full, page_of(i), w.few);
                            if (i + 2 < mine) k_in = landing(k_phases, k_full, page_of(i + 2), w.few);
                            shared_over(v_in.bar, v_in.parity, k_in.bar, k_in.parity, v_in.over, k_in.over);
                            if (i >= 0) issue_pv(page_of(i), i == 0, w.few, v_in);
                            if (ok && i + 2 < mine) issue_qk(page_of(i + 2), w.few, k_in);
                        }
                    }
                    if (mine) ++n_q;
                    base += w.pages;
                    ok = __all_sync(0xffffffffu, ok);
                    heard(n);
                }
                if (lead) {
                    umma_commit(&drained[h]);                                // nothing may still run in tensor memory when it is given back, whoever gave up
#pragma unroll 1
                    for (int k = 0; k < kWaitLimit && !mbar_try_wait(&drained[h], 0); ++k) {}
                }
            }
            __syncwarp();
        }
    } else if (warp < 12) {
        // ---------------- softmax: one thread a row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SH_REGS_SOFT));
        const int h = (warp - 4) >> 2;
        const int row = (tid - 128) & 127;                                   // lane of tensor memory: warp % 4 is the quarter that a warp may read
        const int tok = row * p.inv_g >> 16;
        const uint32_t lanes = tmem + ((uint32_t)(row & 96) << 16);
        const uint32_t s_at0 = lanes + C::COL_S + h * 128, o_at = lanes + C::COL_O + h * D;
        SharedPhases phases;
        int base = 0, cnt = 0;                                               // pages of the share, pages of this half so far
        // maxima and sums of a half, where its queries were: the products that read those have retired
        auto ml_of = [&](int half) { return reinterpret_cast<float2*>(smem + half * KH * C::QBLK); };
        int meetings = 0;
        auto meet = [&]() {
            tc_fence_before();
            __syncwarp();
            if (ok && lane == 0) mbar_arrive(&met);
            ok = ok && wait(&met, meetings++ & 1);
            tc_fence_after();
        };
#pragma unroll 1
        for (int seg = 0;; ++seg) {
            const SharedStretch w = hear(seg);
            if (w.pages == 0) break;
            const int mine = w.of_half(h);
            const int tok0 = w.few ? 0 : h * p.th;                           // of the tile
            const bool valid = tok < p.th && tok0 + tok < w.n;
            if (mine) {
                // the queries, 16 bytes at a time, zeros for rows without one (the products that read the last stretch's have retired: their scores were here)
                constexpr int CH = D / 8;
                const int c = row % CH;
#pragma unroll 4
                for (int r = row / CH; r < kSharedRows; r += kSharedRows / CH) {
                    const int tk = r * p.inv_g >> 16, head = r - tk * p.G;
                    const bool on = tk < p.th && tok0 + tk < w.n;
                    const __half* from = p.q + ((size_t)(w.q0 + tok0 + (on ? tk : 0)) * p.nq + (size_t)w.h * p.G + (on ? head : 0)) * D + c * 8;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem + (h * KH + (c >> 3)) * C::QBLK + r * 128 + ((c & 7) ^ (r & 7)) * 16)), "l"(from),
                                 "r"(on ? 16 : 0)
                                 : "memory");
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full[h]);
            }
            float m_ref = -INFINITY, l_run = 0.f;
#pragma unroll 1
            for (int i = 0; i < mine; ++i, ++cnt) {
                const int buf = cnt & 1, page = base + (w.few ? h + 2 * i : i), stage = page % C::STAGES;
                const uint32_t landed = phases.next(C::STAGES, stage, w.few ? h : 2);
                ok = ok && wait(&s_full[h][buf], cnt >> 1 & 1);
                if (!ok) break;
                tc_fence_after();
                uint32_t sr[64];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld16_nowait(s_at0 + buf * 64 + 16 * c, sr + 16 * c);
                const int seen = tokens_s[page % C::TOKENS];                 // (written ahead of the copy that the scores came of, and not again before they are read)
                tmem_arrived<64>(sr);
                if (seen < kKvTile) {
#pragma unroll
                    for (int c = 0; c < 64; ++c) sr[c] = c < seen ? sr[c] : 0xff800000u;
                    // values behind the end may be anything, and 0 * infinity is not 0.  (Both halves may write here: zeros.)
                    ok = wait(&v_full[phases.at], landed);
                    if (!ok) break;
                    uint8_t* v = smem + C::KV + (C::STAGES + stage) * C::SLAB;
#pragma unroll 1
                    for (int u = row; u < (kKvTile - seen) * 8 * KH; u += kSharedRows) {
                        const int kh = u / ((kKvTile - seen) * 8), x = u % ((kKvTile - seen) * 8);
                        *reinterpret_cast<uint4*>(v + kh * SH_PIECE + seen * 128 + x * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_proxy_async();
                }
                float t0 = max3(sr[0], sr[1], sr[2]), t1 = max3(sr[3], sr[4], sr[5]);
#pragma unroll
                for (int c = 6; c < 62; c += 4) t0 = max3(t0, sr[c], sr[c + 1]), t1 = max3(t1, sr[c + 2], sr[c + 3]);
                t0 = max3(t0, sr[62], sr[63]);
                const float m_new = fmaxf(m_ref, fmaxf(t0, t1) * p.scale_log2);
                if (i == 0) {
                    m_ref = m_new;
                } else if (__any_sync(0xffffffffu, valid && m_new > m_ref + kSharedGrow)) {        // tcgen05.ld / st are warp-wide: all 32 rows
                    ok = wait(&pv_done[h][buf ^ 1], (cnt - 1) >> 1 & 1);
                    if (!ok) break;
                    tc_fence_after();
                    const float alpha = m_new == -INFINITY ? 1.f : exp2f(m_ref - m_new);
                    l_run *= alpha;
                    m_ref = m_new;
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t o[16];
                        tmem_ld16_nowait(o_at + 16 * c, o);
                        tmem_arrived<16>(o);
#pragma unroll
                        for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
                        tmem_st16(o_at + 16 * c, o);
                    }
                }
                const float mu = kSharedTop - (m_ref == -INFINITY ? 0.f : m_ref);
                const f32x2 plus = pack2(mu, mu), scale = pack2(p.scale_log2, p.scale_log2);
                f32x2 sum[2] = {0, 0};                                       // pairs of fp32 zeros
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int c = half * 32 + 2 * e;
                        float p0, p1;
                        unpack2(fma2(pack2(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), scale, plus), p0, p1);
                        p0 = ex2_fast(p0), p1 = ex2_fast(p1);
                        sum[e & 1] = sum2(sum[e & 1], pack2(p0, p1));
                        const __half2 x = __floats2half2_rn(p0, p1);
                        pk[e] = *reinterpret_cast<const uint32_t*>(&x);
                    }
                    tmem_st16(s_at0 + buf * 64 + 16 * half, pk);             // over the scores that they came from (this row has read them)
                }
                tmem_st_wait();
                float a0, a1;
                unpack2(sum2(sum[0], sum[1]), a0, a1);
                l_run += a0 + a1;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[h][buf]);
            }
            if (ok && mine) ok = wait(&pv_done[h][(cnt - 1) & 1], (cnt - 1) >> 1 & 1);
            tc_fence_after();
            if (!ok) {                                                       // NaN for all that this unit says
                l_run = NAN;
                m_ref = 0.f;
            }
            const int row0 = w.row0 + tok0 * p.G;
            const size_t at = (size_t)row0 + (size_t)2 * kSharedRows * blockIdx.x + row;
            if (w.p0 == 0 && valid && row == tok * p.G && (!w.few || h == 0))        // the unit begins here: where each of its queries' results will be
                p.prefix_units[(size_t)(w.q0 + tok0 + tok) * p.nkv + w.h] = make_int4(blockIdx.x, w.last, row0 + row, 0);
            float z = 1.f, zo = 0.f, m = m_ref, l = l_run;
            if (w.few) {                                                     // the halves' results as one: each half puts half of the dims together
                ml_of(h)[row] = make_float2(m_ref, l_run);
                meet();
                const float2 other = ml_of(1 - h)[row];
                m = fmaxf(m_ref, other.x);
                z = m_ref == -INFINITY ? 0.f : exp2f(m_ref - m), zo = other.x == -INFINITY ? 0.f : exp2f(other.x - m);
                l = h == 0 ? l_run * z + other.y * zo : other.y * zo + l_run * z;
                if (!ok) l = NAN;
            }
            const int c0 = w.few ? h * (D / 32) : 0, c1 = w.few ? c0 + D / 32 : D / 16;
#pragma unroll 1
            for (int c = c0; c < c1; ++c) {
                uint32_t o[16];
                tmem_ld16_nowait(o_at + 16 * c, o);
                tmem_arrived<16>(o);
                if (w.few) {                                                 // a half without a page has nothing in tensor memory
                    uint32_t x[16];
                    tmem_ld16_nowait(lanes + C::COL_O + (1 - h) * D + 16 * c, x);
                    tmem_arrived<16>(x);
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float u = z == 0.f ? 0.f : __uint_as_float(o[k]) * z, v = zo == 0.f ? 0.f : __uint_as_float(x[k]) * zo;
                        o[k] = __float_as_uint(h == 0 ? u + v : v + u);
                    }
                }
                if (valid) {
                    float4* to = reinterpret_cast<float4*>(p.rows_o) + (size_t)(4 * c) * p.rows + at;       // a warp's lanes side by side
#pragma unroll
                    for (int k = 0; k < 4; ++k) to[(size_t)k * p.rows] = make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]), __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
                }
            }
            if (valid && (!w.few || h == 0)) p.rows_ml[at] = make_float2(m, l);
            if (w.few) {                                                     // the other half has read what the next products write over
                meet();
            }
            base += w.pages;
            heard(seg);
        }
        tmem_st_wait();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SH_REGS_OWN));
        const int mine = warp - 12;
        if (mine < C::OWN_WARPS) {
            const int f = min(shares.begin(mine, blockIdx.x), own_total);
            shared_own<D>(p, gr, f, min(f + shares.size(blockIdx.x), own_total), own_at[mine].x, own_at[mine].y, shares, mine * gridDim.x + blockIdx.x, smem + C::OWN + mine * (C::OWN_STAGES * C::CHUNK_BYTES), own_full + mine * C::OWN_STAGES, &dead, err);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0) p.gave_up_at[blockIdx.x] = dead;                           // every call writes all of them: the second kernel reads none of an earlier one's
    if (tid == 0 && dead) {
        *err = 1;
#pragma unroll 1
        for (int i = 0; i < 6 * C::STAGES; ++i) {                            // nothing may still be on its way into this CTA's memory when it ends: who gave up has not waited for it
            const int x = i % (3 * C::STAGES);
            uint64_t* const full = (i == x ? k_full : v_full) + x;
#pragma unroll 1
            for (int j = 0; j < kWaitLimit && !mbar_try_wait(full, ((i == x ? k_bits : v_bits) >> x & 1) ^ 1); ++j) {}
        }
    }
    if (warp == 3) {
        tc_fence_after();
        tmem_dealloc(tmem, C::COLS);
    }
}

// ------------------------------------------------------------------ all parts of a (sequence, key head) as one
// Parts that a thread asks for at once, threads.  64 sequences behind 2048 tokens: five parts cost 0.7 us more, 512 threads 2.9; one unit an SM (37 sequences, four key heads):
// 512 threads 0.2 us less.  The kernel takes 3.5 to 6 us, of which 1 is the launch and 3 are waits for what was written last
constexpr int SM_PARTS = 3, SM_THREADS = 256;
template <int D>
__global__ void __launch_bounds__(SM_THREADS, 1024 / SM_THREADS)
shared_merge_kernel(const __grid_constant__ SharedArgs p) {
    pdl_wait();
    __shared__ __align__(16) float acc_s[SM_THREADS * 4];
    __shared__ float2 ml_s[SM_THREADS];
    const int unit = blockIdx.x, G = p.G;
    const int4 own = p.own_units[unit];
    int4 pre = make_int4(0, -1, 0, 0);
    if (p.n_groups) pre = p.prefix_units[unit];
    // Where a wait ran out anywhere, parts of this call may be missing and those of an earlier one in their place: all that the call says is NaN
    int gave_up = (int)threadIdx.x < p.ctas ? __ldcg(p.gave_up_at + threadIdx.x) : 0;      // (no loop: it would wait for this ahead of the reads below, 0.2 us)
    // (nobody has written there without a prefix part, or where a wait ran out ahead of that: what is there then may be anything, and nothing is read by it)
    const bool there = own.z && pre.x >= 0 && pre.x <= pre.y && pre.y < p.ctas && pre.z >= 0 && pre.z < p.rows && pre.z + 2 * kSharedRows * pre.y + G <= p.rows;
    if (!there) pre = make_int4(0, -1, 0, 0);
    // a thread has four dims of a head (neighbours the same of neighbouring heads, as the prefix's results lie), and every `lanes`-th part
    const int mine = (int)((threadIdx.x / (D / 4)) * p.inv_g >> 16), e = threadIdx.x - mine * (G * D / 4), lanes = (int)((SM_THREADS / (D / 4)) * p.inv_g >> 16);
    const int quad = (int)(e * p.inv_g >> 16), hg = e - quad * G;
    const int n_own = own.y - own.x + 1, n = n_own + pre.y - pre.x + 1, record = shared_part(G, D);
    const float* const own0 = p.own_parts + (size_t)(unit + own.x) * record;
    const size_t pre0 = (size_t)pre.z + (size_t)(2 * kSharedRows) * (pre.x - n_own) + hg;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float M = -INFINITY, L = 0.f;
    if (mine < lanes) {
#pragma unroll 1
        for (int k0 = mine; k0 < n; k0 += SM_PARTS * lanes) {
            float4 o[SM_PARTS];
            float2 ml[SM_PARTS];
            float Mn = M;
#pragma unroll
            for (int u = 0; u < SM_PARTS; ++u) {                             // (behind the last part: it once more, with nothing to say)
                const int k = min(k0 + u * lanes, n - 1);
                const float* const part = own0 + (size_t)k * record;
                const size_t at = pre0 + (size_t)(2 * kSharedRows) * k;
                o[u] = __ldcg(k < n_own ? reinterpret_cast<const float4*>(part + hg * D + 4 * quad) : reinterpret_cast<const float4*>(p.rows_o) + (size_t)quad * p.rows + at);
                ml[u] = __ldcg(k < n_own ? reinterpret_cast<const float2*>(part + G * D + 2 * hg) : p.rows_ml + at);
            }
#pragma unroll
            for (int u = 0; u < SM_PARTS; ++u) {
                if (k0 + u * lanes >= n) ml[u].x = -INFINITY;
                Mn = fmaxf(Mn, ml[u].x);
            }
            const float keep = M == -INFINITY ? 0.f : ex2_fast(M - Mn);
            L *= keep;
            acc.x *= keep, acc.y *= keep, acc.z *= keep, acc.w *= keep;
#pragma unroll
            for (int u = 0; u < SM_PARTS; ++u) {
                const float z = ml[u].x == -INFINITY ? 0.f : ex2_fast(ml[u].x - Mn);
                L = fmaf(ml[u].y, z, L);
                acc = fma_f4(o[u], make_float4(z, z, z, z), acc);
            }
            M = Mn;
        }
        *reinterpret_cast<float4*>(acc_s + 4 * threadIdx.x) = acc;
        ml_s[threadIdx.x] = make_float2(M, L);
    }
    gave_up = __syncthreads_or(gave_up);
    if (mine) return;
#pragma unroll 1
    for (int x = 1; x < lanes; ++x) M = fmaxf(M, ml_s[x * (G * D / 4) + e].x);
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
    L = 0.f;
#pragma unroll 1
    for (int x = 0; x < lanes; ++x) {
        const float2 ml = ml_s[x * (G * D / 4) + e];
        const float z = ml.x == -INFINITY ? 0.f : ex2_fast(ml.x - M);
        L = fmaf(ml.y, z, L);
        acc = fma_f4(*reinterpret_cast<const float4*>(acc_s + 4 * (x * (G * D / 4) + e)), make_float4(z, z, z, z), acc);
    }
    if (gave_up) L = NAN;
    const float r = L == 0.f ? 0.f : 1.f / L;                                // a query without a visible key: zeros
    const float v[4] = {acc.x * r, acc.y * r, acc.z * r, acc.w * r};
    const size_t at = ((size_t)unit * G + hg) * D + 4 * quad;                // (unit = sequence * key heads + key head)
    const uint2 hi = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
    *reinterpret_cast<uint2*>(p.out + at) = hi;
    if (p.out_lo)
        *reinterpret_cast<uint2*>(p.out_lo + at) = make_uint2(pack_bf16(v[0] - bf16_lo(hi.x), v[1] - bf16_hi(hi.x)), pack_bf16(v[2] - bf16_lo(hi.y), v[3] - bf16_hi(hi.y)));
}

// ------------------------------------------------------------------ host
struct SharedLayout { size_t own_units, prefix_units, own_parts, rows_o, rows_ml, gave_up_at, rows, bytes; };
static SharedLayout shared_layout(int B, int n_groups, int nq, int nkv, int d) {
    const size_t sms = device_sms(), rows = (size_t)B * nq + 2 * kSharedRows * sms, units = (size_t)B * nkv;
    SharedLayout l;
    l.rows = rows;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 63) / 64 * 64;
        return here;
    };
    l.own_units = take(units * sizeof(int4));
    l.prefix_units = take(n_groups ? units * sizeof(int4) : 0);
    l.own_parts = take((units + 4 * sms) * shared_part(nq / nkv, d) * 4);
    l.rows_o = take(n_groups ? rows * d * 4 : 0);
    l.rows_ml = take(n_groups ? rows * 8 : 0);
    l.gave_up_at = take(sms * sizeof(int));
    l.bytes = at;
    return l;
}

// settings of the calling thread: another one's calls do not change with them
static thread_local long long g_shared_least = -1;
static thread_local int g_shared_give_up = 0;

template <int D>
static int launch_shared(SharedArgs& p, cudaStream_t st) {
    using C = Shared<D>;
    static PerDeviceFlag attr_set;
    if (!attr_set.done()) {
        FT_CHECK_CUDA(cudaFuncSetAttribute(shared_attn_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        cudaFuncAttributes a;
        FT_CHECK_CUDA(cudaFuncGetAttributes(&a, shared_attn_kernel<D>));
        FT_REQUIRE(a.numRegs >= SH_REGS, "ft_attn_decode_shared: built with %d registers a thread, its warps share out %d", a.numRegs, SH_REGS);
        attr_set.mark();
    }
    p.chunk_log = C::CHUNK == 64 ? 6 : 4;
    // What sharing has to save, measured with one group and 100 own tokens each, us shared / not: heads of 64 (32 over 8), two sequences of 8000 tokens 15.0 / 15.5, of 16000
    // 18.3 / 18.2, three of 2000 12.8 / 12.6, of 8000 15.1 / 16.8 (16 MB saved, from the third on), eight of 1000 12.1 / 11.8, of 2000 13.2 / 14.4 (24 MB), sixteen of 130 11.8 / 10.4,
    // of 517 11.9 / 13.4 (15 MB); heads of 128 (32 over 8), two of 1000 13.6 / 13.3, of 2000 15.3 / 15.3 (8 MB), of 8000 17.8 / 23.5, four of 517 12.8 / 13.0 (6 MB), eight of
    // 130 12.9 / 11.9, of 517 13.1 / 13.6; sixteen key heads, two of 1000 15.0 / 12.9, of 2000 16.2 / 15.8 (16 MB), four of 130 13.2 / 11.4, of 517 13.5 / 14.1 (13 MB).
    // The bytes that a call saves decide alone, not what its units cost: so two of 1000 at sixteen key heads are shared where that takes 2.1 us more, two of 2000 there 0.4 more, and
    // two of 8000 at heads of 64 are not where it would take 0.5 less.
    const long long least = g_shared_least, pages = (least < 0 ? (D == 64 ? 12 : 6) << 20 : least) / ((long long)C::TILE * p.nkv);
    p.least_size = D == 64 && least < 0 ? 3 : 2;
    p.least_pages = (int)(pages < INT32_MAX ? pages : INT32_MAX) + (least < 0);
    p.give_up = g_shared_give_up;
    p.ctas = device_sms();
    FT_REQUIRE(p.ctas <= SM_THREADS, "ft_attn_decode_shared: %d SMs (at most %d)", p.ctas, SM_THREADS);      // a thread of the second kernel for each
    FT_CHECK_CUDA(launch_after(shared_attn_kernel<D>, dim3(p.ctas), dim3(SH_THREADS), C::SMEM, st, (const SharedArgs&)p));
    FT_CHECK_CUDA(launch_after(shared_merge_kernel<D>, dim3(p.B * p.nkv), dim3(SM_THREADS), 0, st, (const SharedArgs&)p));
    return 0;
}

}  // namespace ft

extern "C" long long ft_attn_decode_shared_scratch_bytes(int B, int n_groups, int nq, int nkv, int d) {
    FT_REQUIRE(d == 64 || d == 128, "ft_attn_decode_shared_scratch_bytes: head_dim %d not supported (64 or 128)", d);
    FT_REQUIRE(nq >= 1 && nkv >= 1 && nq % nkv == 0 && nq / nkv <= ft::kSharedGroup, "ft_attn_decode_shared_scratch_bytes: GQA group %d/%d not supported", nq, nkv);
    FT_REQUIRE(B >= 0 && n_groups >= 0 && (double)B * nq * d <= INT32_MAX, "ft_attn_decode_shared_scratch_bytes: bad sizes B=%d nq=%d groups=%d", B, nq, n_groups);
    return (long long)ft::shared_layout(B, n_groups, nq, nkv, d).bytes;
}

extern "C" void ft_attn_shared_give_up(int on) { ft::g_shared_give_up = on != 0; }

extern "C" void ft_attn_shared_set_least(long long bytes) { ft::g_shared_least = bytes < 0 ? -1 : bytes; }

extern "C" int ft_attn_shared_waits(void) {
    int n = 0;
    FT_CHECK_CUDA(cudaDeviceSynchronize());                                  // the copy below waits for the default stream only
    FT_CHECK_CUDA(cudaMemcpyFromSymbol(&n, ft::g_shared_waits, sizeof(n)));
    return n;
}

extern "C" int ft_attn_decode_shared(const ft_attn_shared_args* args, void* stream) {
    using namespace ft;
    FT_REQUIRE(args, "ft_attn_decode_shared: null argument");
    const auto [q, kv_layer, page_table, req_slot, ctx_lens, group_start, shared_lens, out, out_lo, scratch, num_pages, table_rows, max_pages, n_groups, B, nq, nkv, d] = *args;
    FT_REQUIRE(d == 64 || d == 128, "ft_attn_decode_shared: head_dim %d not supported (64 or 128)", d);
    FT_REQUIRE(nq >= 1 && nkv >= 1 && nq % nkv == 0 && nq / nkv <= kSharedGroup, "ft_attn_decode_shared: GQA group %d/%d not supported", nq, nkv);
    const int G = nq / nkv, th = kSharedRows / G;
    FT_REQUIRE(B >= 0 && n_groups >= 0 && num_pages >= 0 && table_rows >= 0 && max_pages >= 0 && max_pages < INT32_MAX / kKvTile && (double)B * nq * d <= INT32_MAX,
               "ft_attn_decode_shared: bad sizes B=%d nq=%d groups=%d table %d x %d, %d pages", B, nq, n_groups, table_rows, max_pages, num_pages);
    // both lists: at most so many units of at most so many steps, and what the shares are rounded up by
    FT_REQUIRE(((double)B + 1) * nkv * (8.0 * max_pages + 8) + 65536 <= INT32_MAX && ((double)B / (2 * th) + n_groups) * nkv * (max_pages + kSharedStart + 1.0) + 65536 <= INT32_MAX,
               "ft_attn_decode_shared: %d sequences of %d pages in %d groups are more than one call takes", B, max_pages, n_groups);
    if (B == 0) return 0;
    FT_REQUIRE(q && ctx_lens && out && scratch && (n_groups == 0 || (group_start && shared_lens)) && (page_table || table_rows == 0 || max_pages == 0) && (kv_layer || num_pages == 0),
               "ft_attn_decode_shared: null argument");
    FT_REQUIRE(((uintptr_t)q | (uintptr_t)kv_layer | (uintptr_t)out | (uintptr_t)out_lo | (uintptr_t)scratch) % 16 == 0, "ft_attn_decode_shared: tensors on 16 bytes");
    const SharedLayout l = shared_layout(B, n_groups, nq, nkv, d);
    uint8_t* w = (uint8_t*)scratch;
    SharedArgs p{(const __half*)q, (const uint8_t*)kv_layer, page_table, req_slot, ctx_lens, group_start, shared_lens, (__nv_bfloat16*)out, (__nv_bfloat16*)out_lo,
                 (int4*)(w + l.own_units), (int4*)(w + l.prefix_units), (float*)(w + l.own_parts), (float*)(w + l.rows_o), (float2*)(w + l.rows_ml), (int*)(w + l.gave_up_at), B, n_groups, num_pages, table_rows,
                 max_pages, nq, nkv, G, th, (int)l.rows, 0, (65536u + G - 1) / G, kSharedLog2E / sqrtf((float)d), (unsigned)(((1ull << 32) + 2 * th - 1) / (2 * th)), 0, 0, 0, 0};
    return d == 64 ? launch_shared<64>(p, (cudaStream_t)stream) : launch_shared<128>(p, (cudaStream_t)stream);
}
