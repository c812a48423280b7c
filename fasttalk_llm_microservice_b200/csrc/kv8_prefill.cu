// Causal attention of prompt portions over the 8-bit KV cache (kv8.cuh) on tcgen05 / TMEM: request r owns rows req_q_start[r] .. req_q_start[r + 1] - 1 of q, its
// first query sits at position req_pos0[r], and out[t][h] = sum_j softmax_j(q . k_j / sqrt(D)) v_j over the keys j <= position of t.
//
// A unit of work is a tile of query tokens of one request and one key head: two halves of up to 128 rows (row = token * G + head of the group), so that every
// record that reaches an SM serves both.  Per page and half, as in attention_tc.cu:  S = Q K^T (M128 N64 K=D, both operands in shared memory), one thread a row
// for the softmax, P to tensor memory, O += P V (A from tensor memory, M128 N=D K64).  A unit whose tokens fill one half only gives both halves the same queries and
// every other page each.
//
// The tensor cores want fp16, so eight warps turn each record into the two operands, swizzled as the instructions read them: codes as they are, which fp16 holds exactly.
// The keys' scales go to the scores (one multiplication per 16 of them for the maximum, and the multiply-add's factor for the exponents), the values' to the probabilities.
// Such a weight is rounded to fp16, 2^-11 of it, relative to the largest weight that its own row has met (kKv8Top in kv8.cuh): nothing that a row does not see, and no large
// value without weight, takes bits from it.
//
// The flat list of all (request, key head, tile, page) is cut into equal shares, one for each SM: a causal list's units differ in length by any factor, and shares do
// not.  A unit that lies in several shares is put together by a second kernel, in the parts' order.  Where there is an SM for every unit and none is much longer than
// a share, each CTA takes a whole one.  (A unit's list is longer than its pages by what its start and end cost.  With one buffer of scores a half, at D = 128, the halves of a
// unit of few tokens gain nothing over one: a page counts as one there.)  One warp of each CTA finds its share from the lists on the device and tells the others stretch by stretch; nothing is planned
// ahead of the kernel.
//
// What bounds it: each half's chain of a page, scores out of tensor memory - exponentials - probabilities into it - products - next scores, and the instructions of
// eight softmax and eight converting warps around it: 1.2 us (2350 clocks) a page of both halves at heads of 64 and 1.24 at 128, by the time that more pages add to a unit on each
// SM, where the exponentials alone take 1024 clocks (the SFU's 16 a clock and SM).  A unit of one page on each SM takes 11 us from launch to launch, 15 at heads of 128, the second
// kernel with nothing to do included.  Four prompts of 2048 .. 1578 tokens, 32 heads over 8 of 64: 160 us, 353 TFLOP/s; six portions of 211 .. 153 tokens behind about 5000, heads
// of 128: 128 us, 655 TFLOP/s; five tokens behind 16001 on one rank's heads: 25 us.  The weights' multiplication is 5 % of the first: with the scales in the value operands,
// relative to the largest of a stretch, they took 152 / 122, but what a row did not see took its bits.
// Measured on the way, us for the first two: scales in the exponents' addends instead, and the sums of p by blocks, 163 / 130 (registers spill); shares of pages alone, without a
// unit's start and end, 175 / 176 (with them 153 / 126); the next page's scores read ahead of this
// page's exponentials 251 / 349 (with two buffers they are formed only behind the products that wait for this page's probabilities); copies and conversions that nap between
// their tries 223 / 339; longer waits written out in every role, 173 / 138 against 153 / 127 (instruction fetch).
#include "common.cuh"
#include "ft_internal.h"
#include "kv8.cuh"
#include "kv8_walk.cuh"

namespace ft {

// Groups of four warps: warp 0 copies records, 1 and 2 issue the halves' products, 3 finds the work, 4 .. 11 softmax (half = (warp - 4) / 4), 12 .. 19 convert.  The
// softmax threads hold a page's scores and take registers that the others give up: 64 + 2 x 144 + 2 x 64 = 5 x 96 a lane of the SM's quarter.
constexpr int K8P_THREADS = 640;
constexpr int K8P_REGS = 96, K8P_REGS_ISSUE = 64, K8P_REGS_SOFT = 144, K8P_REGS_CONV = 64;
static_assert(K8P_REGS_ISSUE + 2 * K8P_REGS_SOFT + 2 * K8P_REGS_CONV <= 5 * K8P_REGS, "what the block is launched with");
constexpr int K8P_SOFT = 256, K8P_CONV = 256;    // (256: four threads a row of a piece)
constexpr int K8P_LISTENERS = 19;                // warps that hear of a stretch: all but the one that tells
constexpr int K8P_ROWS = 128;                    // rows of a half
constexpr int K8P_GROUP = 8;                     // query heads a key head at most
constexpr int K8P_PIECE = kKvTile * 128;         // [64 tokens][64 dims] in fp16; 64 rows of a Q block
constexpr float K8P_LOG2E = 1.4426950408889634f;
// Pages that a share may be shorter than a whole unit for parts not to pay.  us with 5 / 7 / 10, heads of 128: four portions of 100 tokens behind 300 22.0 / 20.4 / 20.4, three of
// 150 behind 900 34.1 / 33.8 / 36.9, six of 100 behind 1000 38.8 / 37.0 / 37.0.  Heads of 64: four of 100 behind 300 18.1 / 17.0 / 17.1, 700 and 619 behind 333 with a key head
// each 28.0 / 28.1 / 31.8, six of 100 behind 1000 31.8 / 32.5 / 32.5
constexpr int K8P_WHOLE = 7;

template <int D>
struct K8Prefill {
    static constexpr int KH = D / 64;
    static constexpr int TILE = 2 * KH * K8P_PIECE;                  // K | V of a page in fp16
    static constexpr int S16 = D == 64 ? 6 : 3, S8 = D == 64 ? 6 : 3;
    static constexpr int NS = D == 64 ? 2 : 1;                       // score buffers of a half
    static constexpr int QBLK = K8P_ROWS * 128;                      // [128 rows][64 dims]
    static constexpr int Q_BYTES = 2 * KH * QBLK;
    static constexpr int KV = Q_BYTES, REC = KV + S16 * TILE, SMEM = 1024 + REC + S8 * Kv8<D>::REC;
    // tensor memory: scores [half][NS][64 columns], probabilities [half][2][32] (pairs of fp16), O [half][D]
    static constexpr int COL_S = 0, COL_P = 2 * NS * 64, COL_O = COL_P + 128, COLS = 512;
    static_assert(COL_O + 2 * D <= COLS, "tensor memory");
    static constexpr size_t PART = (size_t)2 * K8P_ROWS * (D + 2);   // floats of a part: O [D / 4][256 rows][4], then (m, l) [256]
};

// two fp32 sums in one instruction, and the largest of three
__device__ __forceinline__ f32x2 sum2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max3(uint32_t a, uint32_t b, uint32_t c) { return max3(__uint_as_float(a), __uint_as_float(b), __uint_as_float(c)); }
__device__ __forceinline__ float max3(float a, uint32_t b, uint32_t c) { return max3(a, __uint_as_float(b), __uint_as_float(c)); }

// Registers that tcgen05.ld fills are there after the wait only, which the compiler cannot see from its operands: nothing that reads them moves ahead of this
template <int N>
__device__ __forceinline__ void tmem_arrived(uint32_t* r) {
    tmem_ld_wait();
#pragma unroll
    for (int c = 0; c < N; c += 8)
        asm volatile("" : "+r"(r[c]), "+r"(r[c + 1]), "+r"(r[c + 2]), "+r"(r[c + 3]), "+r"(r[c + 4]), "+r"(r[c + 5]), "+r"(r[c + 6]), "+r"(r[c + 7]));
}
constexpr int kStretchWaits = 64;                // times the limit, for what takes a whole stretch: it may be a million keys
// A warp's wait (all lanes ask, so that the warp stays together)
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* dead, int limit) {
    return __all_sync(0xffffffffu, kv8_mbar_wait_limited(bar, parity, dead, limit));
}

__device__ int g_kv8_prefill_waits;              // 1: a wait ran out on this device (ft_kv8_waits)

// floats that the descriptions of split units take at the head of the work memory
static size_t kv8_prefill_splits(int ctas) { return (size_t)(ctas + 15) / 16 * 16 * (sizeof(Kv8Split) / 4); }

template <int D>
__global__ void __launch_bounds__(K8P_THREADS, 1)
kv8_prefill_kernel(const __grid_constant__ Kv8Prompt p) {
    using C = K8Prefill<D>;
    constexpr int KH = C::KH;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t rec_full[C::S8], rec_empty[C::S8];                   // a record is there
    __shared__ uint64_t kv_full[C::S16], kv_empty[C::S16];                   // a page's operands are
    __shared__ uint64_t q_full, q_empty;                                     // the queries of a stretch
    __shared__ uint64_t s_full[2][C::NS], s_free[2];                         // half, buffer: scores are in tensor memory; (NS = 1) and in registers
    __shared__ uint64_t p_full[2][2], pv_done[2][2];                         // probabilities are in tensor memory; O += P V retired
    __shared__ uint64_t seg_full[4], seg_empty[4];                           // a stretch has been told; all have done with it
    __shared__ uint64_t halves_met;                                          // all softmax warps are here
    __shared__ uint64_t drained[2];                                          // all products of a half retired
    __shared__ Kv8Stretch told[4];
    __shared__ __align__(16) float kscale_s[C::S16][4];                      // times scale_log2; the first below 0: the page is not there
    __shared__ __align__(16) float vscale_s[C::S16][4], vlog_s[C::S16][4];   // of the values; 0 for blocks behind the unit's last token.  And their log2
    __shared__ int blocks_s[C::S8];                                          // of 16 tokens, that some query of the unit sees; 0: none, or the page is not there
    __shared__ float2 ml_s[K8P_SOFT];
    __shared__ float size_s[K8P_SOFT];                                       // what a row's O is multiplied by to be in its own size
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int dead;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int* const err = &g_kv8_prefill_waits;
    if (tid == 0) {
        for (int s = 0; s < C::S16; ++s) mbar_init(&kv_full[s], K8P_CONV / 32), mbar_init(&kv_empty[s], 2);
        for (int s = 0; s < C::S8; ++s) mbar_init(&rec_full[s], 1), mbar_init(&rec_empty[s], K8P_CONV / 32);
        for (int s = 0; s < 4; ++s) mbar_init(&seg_full[s], 1), mbar_init(&seg_empty[s], K8P_LISTENERS);
        mbar_init(&q_full, K8P_CONV / 32);
        mbar_init(&q_empty, 2);
        mbar_init(&halves_met, K8P_SOFT / 32);
        for (int h = 0; h < 2; ++h) {
            for (int s = 0; s < C::NS; ++s) mbar_init(&s_full[h][s], 1);
            mbar_init(&s_free[h], K8P_ROWS / 32);
            for (int s = 0; s < 2; ++s) mbar_init(&p_full[h][s], K8P_ROWS / 32), mbar_init(&pv_done[h][s], 1);
            mbar_init(&drained[h], 1);
        }
        fence_mbar_init();
        dead = 0;
    }
    if (warp == 1) {
        tmem_alloc(&tmem_slot, C::COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_wait();
    bool ok = true;                                                          // false: a wait ran out
    // the n-th stretch of the share, or one without pages behind the last; and this warp's word that it has done with it
    auto hear = [&](int n) {
        ok = ok && warp_wait(&seg_full[n & 3], n >> 2 & 1, &dead, kStretchWaits * p.wait_limit);
        Kv8Stretch w = told[n & 3];
        if (!ok) w.pages = 0;
        return w;
    };
    auto done = [&](int n) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&seg_empty[n & 3]);
    };

    // (the register counts change inside the branches, where the compiler sees what they are for)
    if (warp < 4) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(K8P_REGS_ISSUE));
      if (warp == 3) {
        // ---------------- the plan: this CTA's share, stretch by stretch.  A lane adds up a run of requests
        const int chunk = (p.n_req + 31) / 32;
        const int r0 = min(p.n_req, lane * chunk), r1 = min(p.n_req, r0 + chunk);
        Kv8Walk w;
        Kv8Sums mine;
#pragma unroll 1
        for (int r = r0; r < r1; ++r) mine.add(p, r);
        int b_steps = mine.steps, b_units = mine.units;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, b_steps, o), y = __shfl_up_sync(0xffffffffu, b_units, o);
            if (lane >= o) b_steps += x, b_units += y;
        }
        const int most = __reduce_max_sync(0xffffffffu, mine.most);
        const int total = __shfl_sync(0xffffffffu, b_steps, 31) * p.nkv, n_units = __shfl_sync(0xffffffffu, b_units, 31) * p.nkv, ctas = gridDim.x;
        b_steps -= mine.steps;
        b_units -= mine.units;
        const int per = (unsigned)(total + ctas - 1) / (unsigned)ctas;
        const bool whole = p.split == nullptr || (n_units <= ctas && most + kKv8Start <= per + K8P_WHOLE);      // (no room for parts: the host knows that there are none)
        // the flat list is one of units or of steps
        const int len = whole ? n_units : total, each = whole ? 1 : per, at0 = whole ? b_units : b_steps;
        const bool work = w.share(__all_sync(0xffffffffu, mine.grows), len, each, blockIdx.x);
        if (work ? at0 * p.nkv <= w.f && w.f < (at0 + (whole ? mine.units : mine.steps)) * p.nkv : lane == 0) {      // one lane
            if (work) {
                w.seek(p, whole, r0, at0, w.f);
                w.unit(p);
                if (whole) w.f = 0, w.f_end = w.n_steps;
            }
#pragma unroll 1
            for (int n = 0, more = 1; more; ++n) {
                more = w.next(p);
                if (!kv8_mbar_wait_limited(&seg_empty[n & 3], (n >> 2 & 1) ^ 1, &dead, kStretchWaits * p.wait_limit)) break;
                if (more) told[n & 3] = w.stretch(p, per, blockIdx.x);
                else told[n & 3].pages = 0;
                mbar_arrive(&seg_full[n & 3]);
            }
        }
        __syncwarp();
      } else if (warp == 0) {
        // ---------------- copies: one record a page
        const uint64_t pol = policy_evict_last();                            // read again by other tiles
        int it = 0, asked = 0;
        bool go = true;
#pragma unroll 1
        for (int seg = 0;; ++seg) {
            const Kv8Stretch w = hear(seg);
            if (w.pages == 0) break;
            const int* pt = p.page_table + (size_t)w.slot * p.max_pages;
            const int most_here = w.slot >= 0 && w.slot < p.table_rows ? p.max_pages : 0;
            const int p1 = w.page0 + w.pages;
#pragma unroll 1
            for (int p0 = w.page0; p0 < p1; p0 += 32) {
                const int mine = p0 + lane;
                const int my_page = mine < p1 && mine < most_here ? pt[mine] : -1;
                const int n = min(32, p1 - p0);
#pragma unroll 1
                for (int k = 0; k < n; ++k, ++it) {
                    const int page = __shfl_sync(0xffffffffu, my_page, k);
                    if (lane == 0 && go) {
                        const int s = it % C::S8;
                        go = kv8_mbar_wait_limited(&rec_empty[s], (it / C::S8 & 1) ^ 1, &dead, p.wait_limit);
                        if (!go) continue;
                        asked = it + 1;
                        const bool there = page >= 0 && page < p.num_pages;
                        blocks_s[s] = there ? max(0, min(4, ((w.pos0 + w.tokens - 1 - (p0 + k) * kKvTile) >> 4) + 1)) : 0;
                        if (there) {
                            mbar_expect_tx(&rec_full[s], Kv8<D>::REC);
                            tma_bulk_g2s(smem + C::REC + s * Kv8<D>::REC, p.cache + ((size_t)page * p.nkv + w.head) * Kv8<D>::REC, Kv8<D>::REC, &rec_full[s], pol);
                        } else {
                            mbar_arrive(&rec_full[s]);
                        }
                    }
                }
            }
            done(seg);
        }
        if (lane == 0) kv8_copies_landed(rec_full, C::S8, asked);            // (those who read them may give up at any time)
      } else {
        // ---------------- products, one warp a half
        constexpr uint32_t idesc_qk = umma_idesc_f16(K8P_ROWS, kKvTile, false), idesc_pv = umma_idesc_f16(K8P_ROWS, D, true);
        const int h = warp - 1;
        const bool lead = elect_one();
        // operands' descriptors differ in their addresses alone, in units of 16 bytes
        const uint64_t q_desc = umma_desc_k128(smem_u32(smem)), k_desc = umma_desc_k128(smem_u32(smem + C::KV)), v_desc = umma_desc_mn128(smem_u32(smem + C::KV) + KH * K8P_PIECE);
        const uint32_t s_at = tmem + C::COL_S + h * C::NS * 64, p_at = tmem + C::COL_P + h * 64, o_at = tmem + C::COL_O + h * D;
        int base = 0, n_qk = 0, n_pv = 0;                                    // pages of the share, products of this half so far
        auto issue_qk = [&](int page, int qh) {                              // page: counted over the whole share
            const int s = page % C::S16, buf = n_qk % C::NS;
            if (C::NS == 1) ok = kv8_mbar_wait_limited(&s_free[h], (n_qk & 1) ^ 1, &dead, p.wait_limit);
            ok = ok && kv8_mbar_wait_limited(&kv_full[s], page / C::S16 & 1, &dead, p.wait_limit);
            if (!ok) return;
            ++n_qk;
            tc_fence_after();
            const uint64_t a = q_desc + (uint64_t)(qh * KH * (C::QBLK >> 4)), b = k_desc + (uint64_t)(s * (C::TILE >> 4));
#pragma unroll
            for (int kh = 0; kh < KH; ++kh)
#pragma unroll
                for (int k = 0; k < 4; ++k) umma_bf16(s_at + buf * 64, a + kh * (C::QBLK >> 4) + 2 * k, b + kh * (K8P_PIECE >> 4) + 2 * k, idesc_qk, (kh | k) != 0);
            umma_commit(&s_full[h][buf]);
        };
        auto issue_pv = [&](int page, bool first, bool alone) {
            const int s = page % C::S16, buf = n_pv & 1;
            ok = kv8_mbar_wait_limited(&p_full[h][buf], n_pv >> 1 & 1, &dead, p.wait_limit);
            if (!ok) return;
            ++n_pv;
            tc_fence_after();
            const uint64_t b = v_desc + (uint64_t)(s * (C::TILE >> 4));
#pragma unroll
            for (int k = 0; k < kKvTile / 16; ++k) umma_f16_ts(o_at, p_at + buf * 32 + 8 * k, b + k * (2048 >> 4), idesc_pv, k != 0 || !first);
            umma_commit(&pv_done[h][buf]);
            umma_commit(&kv_empty[s]);
            if (alone) umma_commit(&kv_empty[s]);                            // the other half has no use for this page
        };
#pragma unroll 1
        for (int seg = 0;; ++seg) {
            const Kv8Stretch w = hear(seg);
            if (w.pages == 0) break;
            const int mine_n = w.few ? (w.pages - h + 1) / 2 : w.pages;      // page i of this half is page j of the stretch
            auto page_of = [&](int i) { return base + (w.few ? h + 2 * i : i); };
            if (lead) {
                ok = kv8_mbar_wait_limited(&q_full, seg & 1, &dead, p.wait_limit);
                tc_fence_after();
                if (ok && mine_n == 0) umma_commit(&q_empty);
                // Scores run NS pages ahead.  With two buffers page i + 2's follow the product that reads page i's probabilities, which says that page i's scores
                // have been read; with one, page i + 1's follow the softmax's word that it has them in registers, ahead of that product.  Either way scores that are
                // there mean that the product before the last is done, and the probabilities' buffer with it.
#pragma unroll 1
                for (int i = -C::NS; ok && i < mine_n; ++i) {
                    if (C::NS == 2 && i >= 0) issue_pv(page_of(i), i == 0, w.few);
                    if (ok && i + C::NS < mine_n) issue_qk(page_of(i + C::NS), w.few ? 0 : h);
                    if (i + C::NS == mine_n - 1) umma_commit(&q_empty);
                    if (C::NS == 1 && ok && i >= 0) issue_pv(page_of(i), i == 0, w.few);
                }
            }
            base += w.pages;
            ok = __all_sync(0xffffffffu, ok);
            done(seg);
        }
        if (lead) {                                                          // nothing may still run in tensor memory when it is given back, whoever gave up
            umma_commit(&drained[h]);
#pragma unroll 1
            for (int k = 0; k < kWaitLimit && !mbar_try_wait(&drained[h], 0); ++k) {}
        }
        __syncwarp();
      }
    } else if (warp >= 12) {
        // ---------------- conversion: Q of each stretch, then its pages
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(K8P_REGS_CONV));
        const int ct = tid - 128 - K8P_SOFT;
        int it = 0;
#pragma unroll 1
        for (int seg = 0;; ++seg) {
            const Kv8Stretch w = hear(seg);
            if (w.pages == 0) break;
            // the queries, 16 bytes at a time and all on their way at once; zeros for rows without a token
            if (seg) ok = warp_wait(&q_empty, (seg - 1) & 1, &dead, p.wait_limit);
            if (ok) {
                constexpr int CH = D / 8;
#pragma unroll 4
                for (int k = ct; k < (w.few ? 1 : 2) * K8P_ROWS * CH; k += K8P_CONV) {
                    const int c = k % CH, rr = k / CH, h = rr >> 7, row = rr & 127;
                    const int tok = row * p.inv_g >> 16, head = row - tok * p.G;
                    const bool on = tok < p.th && h * p.th + tok < w.tokens;
                    const __half* from = p.q + ((size_t)(w.row0 + (on ? h * p.th + tok : 0)) * p.nq + (size_t)w.head * p.G + (on ? head : 0)) * D + c * 8;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem + (h * KH + (c >> 3)) * C::QBLK + row * 128 + ((c & 7) ^ (row & 7)) * 16)),
                                 "l"(from), "r"(on ? 16 : 0)
                                 : "memory");
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full);
            }
#pragma unroll 1
            for (int k = 0; ok && k < w.pages; ++k, ++it) {
                const int s8 = it % C::S8, s16 = it % C::S16;
                ok = warp_wait(&rec_full[s8], it / C::S8 & 1, &dead, p.wait_limit) && warp_wait(&kv_empty[s16], (it / C::S16 & 1) ^ 1, &dead, p.wait_limit);
                if (!ok) break;
                const uint8_t* rec = smem + C::REC + s8 * Kv8<D>::REC;
                uint8_t* dst = smem + C::KV + s16 * C::TILE;
                const int blocks = blocks_s[s8];
                const float* scales = reinterpret_cast<const float*>(rec + Kv8<D>::SCALES);
                // a block of zeros keeps a factor above 0, so that hidden scores stay minus infinity
                if (ct < 4) {
                    const float v = ct < blocks ? scales[4 + ct] : 0.f;      // of a block behind the last token, whatever its scale is, nothing comes
                    kscale_s[s16][ct] = blocks ? fmaxf(scales[ct] * p.scale_log2, 1e-37f) : -1.f;
                    vscale_s[s16][ct] = v;
                    vlog_s[s16][ct] = __log2f(fabsf(v));
                }
                if (blocks) {
#pragma unroll
                    for (int u = ct; u < kKvTile * D / 16; u += K8P_CONV) {  // keys: 16 codes, two chunks of the swizzled row
                        const int piece = u >> 8, t = u >> 2 & 63, c = u & 3;
                        const uint4 x = *reinterpret_cast<const uint4*>(rec + u * 16);
                        uint8_t* at = dst + piece * K8P_PIECE + t * 128;
                        *reinterpret_cast<uint4*>(at + ((2 * c) ^ (t & 7)) * 16) = make_uint4(kv8_lo(x.x), kv8_hi(x.x), kv8_lo(x.y), kv8_hi(x.y));
                        *reinterpret_cast<uint4*>(at + ((2 * c + 1) ^ (t & 7)) * 16) = make_uint4(kv8_lo(x.z), kv8_hi(x.z), kv8_lo(x.w), kv8_hi(x.w));
                    }
#pragma unroll
                    for (int u = ct; u < kKvTile * D / 16; u += K8P_CONV) {  // values, by where they lie
                        const int piece = u >> 8, slot = u >> 2 & 63, t = slot ^ (slot >> 1 & 1), c = (u & 3) ^ (t >> 1 & 2);
                        const uint4 x = *reinterpret_cast<const uint4*>(rec + Kv8<D>::SLAB + u * 16);
                        uint8_t* at = dst + (KH + piece) * K8P_PIECE + t * 128;
                        *reinterpret_cast<uint4*>(at + ((2 * c) ^ (t & 7)) * 16) = make_uint4(kv8_lo(x.x), kv8_hi(x.x), kv8_lo(x.y), kv8_hi(x.y));
                        *reinterpret_cast<uint4*>(at + ((2 * c + 1) ^ (t & 7)) * 16) = make_uint4(kv8_lo(x.z), kv8_hi(x.z), kv8_lo(x.w), kv8_hi(x.w));
                    }
                } else {                                                     // hidden probabilities are zeros, and so must be what they are multiplied by
#pragma unroll 1
                    for (int u = ct; u < C::TILE / 16; u += K8P_CONV) *reinterpret_cast<uint4*>(dst + u * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&kv_full[s16]), mbar_arrive(&rec_empty[s8]);
            }
            done(seg);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
        // ---------------- softmax: one thread a row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(K8P_REGS_SOFT));
        const int st = tid - 128, h = (warp - 4) >> 2;
        const int row = st & 127;                                            // lane of tensor memory: warp % 4 is the quarter that a warp may read
        const int tok = row * p.inv_g >> 16, head = row - tok * p.G;
        const uint32_t lanes = tmem + ((uint32_t)(row & 96) << 16);
        const uint32_t s_at = lanes + C::COL_S + h * C::NS * 64, p_at = lanes + C::COL_P + h * 64, o_at = lanes + C::COL_O + h * D;
        if (st == 0 && p.split) p.split[blockIdx.x].parts = 0;
        // rows that no request owns
        {
            const int a = p.n_req ? max(0, min(p.req_q_start[0], p.T)) : p.T, b = p.n_req ? max(a, min(p.req_q_start[p.n_req], p.T)) : p.T;
            const int n = a + p.T - b;
#pragma unroll 1
            for (int i = blockIdx.x; i < n; i += gridDim.x) {
                const size_t at = (size_t)(i < a ? i : b + i - a) * p.nq * D;
#pragma unroll 1
                for (int e = 8 * st; e < p.nq * D; e += 8 * K8P_SOFT) {
                    *reinterpret_cast<uint4*>(p.out + at + e) = make_uint4(0u, 0u, 0u, 0u);
                    if (p.out_lo) *reinterpret_cast<uint4*>(p.out_lo + at + e) = make_uint4(0u, 0u, 0u, 0u);
                }
            }
        }
        // the largest of a page's scores, and of score + log2(value scale), in log2 units
        auto largest = [](const uint32_t* sr, const float* ks, const float* vl, float& heavy) {
            float most = -INFINITY;
            heavy = -INFINITY;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const uint32_t* x = sr + 16 * b;
                float t0 = max3(x[0], x[1], x[2]), t1 = max3(x[3], x[4], x[5]);
                t0 = max3(t0, x[6], x[7]), t1 = max3(t1, x[8], x[9]);
                t0 = max3(t0, x[10], x[11]), t1 = max3(t1, x[12], x[13]);
                t0 = max3(t0, x[14], x[15]);
                const float t = fmaxf(t0, t1) * ks[b];
                most = fmaxf(most, t);
                heavy = fmaxf(heavy, t + vl[b]);
            }
            return most;
        };
        int base = 0, cnt = 0, met = 0;                                      // pages of the share, pages of this half so far; meetings of the halves
#pragma unroll 1
        for (int seg = 0;; ++seg) {
            const Kv8Stretch w = hear(seg);
            if (w.pages == 0) break;
            const int mine_n = w.few ? (w.pages - h + 1) / 2 : w.pages;      // pages of this half
            const int my_tok = w.few ? tok : h * p.th + tok;
            const bool valid = tok < p.th && my_tok < w.tokens;
            float m_ref = -INFINITY, h_ref = -INFINITY, r = 1.f, l_run = 0.f;        // r = 2^(m - h + 7): a weight is p * scale * r
            int it = base + (w.few ? h : 0), ahead = w.pos0 + my_tok - (w.page0 + (w.few ? h : 0)) * kKvTile;     // page of the share; the row's position from the page's first key on
#pragma unroll 1
            for (int i = 0; i < mine_n; ++i, ++cnt) {
                const int sb = cnt % C::NS, pb = cnt & 1;
                ok = ok && warp_wait(&s_full[h][sb], cnt / C::NS & 1, &dead, p.wait_limit);
                if (!ok) break;
                tc_fence_after();
                uint32_t sr[64];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld16_nowait(s_at + sb * 64 + 16 * c, sr + 16 * c);
                // (the page's scales are visible: they were written ahead of the operands that the product behind this barrier read)
                const float4 k4 = *reinterpret_cast<const float4*>(kscale_s[it % C::S16]);
                const float ks[4] = {fabsf(k4.x), fabsf(k4.y), fabsf(k4.z), fabsf(k4.w)};
                const float4 l4 = *reinterpret_cast<const float4*>(vlog_s[it % C::S16]);
                const float vl[4] = {l4.x, l4.y, l4.z, l4.w};
                const float* vs = vscale_s[it % C::S16];
                tmem_arrived<64>(sr);
                if constexpr (C::NS == 1) {                                  // the scores are in registers: the next ones may be formed
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_free[h]);
                }
                const int seen = k4.x < 0.f ? -1 : ahead;                    // the last key of the page that the row sees
                it += w.few ? 2 : 1;
                ahead -= w.few ? 2 * kKvTile : kKvTile;
                if (seen < kKvTile - 1) {
#pragma unroll
                    for (int c = 0; c < 64; ++c) sr[c] = c <= seen ? sr[c] : 0xff800000u;
                }
                const uint32_t at = p_at + pb * 32;
                // The exponentials are taken with the references of the pages before while this page's are found; where one has grown by too much they are taken again.
                // (The stretch's first page has nothing before it.)
                bool known = i == 0;
                if (known) {
                    m_ref = largest(sr, ks, vl, h_ref);
                    h_ref = fmaxf(h_ref, m_ref - kKv8Low);
                    r = m_ref == -INFINITY ? 1.f : exp2f(m_ref - h_ref + kKv8Top);
                }
                f32x2 sum[2];
#pragma unroll 1
                for (;;) {
                    const float mu = m_ref == -INFINITY ? 0.f : m_ref;
                    const f32x2 minus = pack2(-mu, -mu);
                    sum[0] = sum[1] = 0;                                     // pairs of fp32 zeros
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t pk[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int c = half * 32 + 2 * e;
                            const float f = ks[c >> 4], g = vs[c >> 4] * r;
                            float p0, p1;
                            unpack2(fma2(pack2(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), pack2(f, f), minus), p0, p1);
                            p0 = ex2_fast(p0), p1 = ex2_fast(p1);
                            const f32x2 both = pack2(p0, p1);
                            sum[e & 1] = sum2(sum[e & 1], both);
                            unpack2(mul2(both, pack2(g, g)), p0, p1);
                            const __half2 t = __floats2half2_rn(p0, p1);
                            pk[e] = *reinterpret_cast<const uint32_t*>(&t);
                        }
                        tmem_st16(at + 16 * half, pk);
                    }
                    if (known) break;
                    float h_new;
                    const float m_new = fmaxf(m_ref, largest(sr, ks, vl, h_new));
                    h_new = fmaxf(fmaxf(h_ref, h_new), m_new - kKv8Low);
                    // rows without a token say nothing: a row's rounding depends on its own request alone
                    if (!__any_sync(0xffffffffu, valid && (m_new > m_ref + kKv8GrowM || h_new > h_ref + kKv8GrowH))) break;
                    known = true;
                    ok = warp_wait(&pv_done[h][pb ^ 1], (cnt - 1) >> 1 & 1, &dead, p.wait_limit);
                    if (!ok) break;
                    tc_fence_after();
                    const float alpha = m_new == -INFINITY ? 1.f : exp2f(h_ref - h_new);
                    if (m_new != -INFINITY) l_run *= exp2f(m_ref - m_new), r = exp2f(m_new - h_new + kKv8Top);
                    m_ref = m_new;
                    h_ref = h_new;
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
                if (!ok) break;
                tmem_st_wait();
                float a0, a1;
                unpack2(sum2(sum[0], sum[1]), a0, a1);
                l_run += a0 + a1;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[h][pb]);
            }
            if (ok && mine_n) ok = warp_wait(&pv_done[h][(cnt - 1) & 1], (cnt - 1) >> 1 & 1, &dead, p.wait_limit);
            if (w.few && w.parts == 0) {                                     // the halves' maxima and sums; and a half without a page has waited for nothing yet
                ml_s[st] = make_float2(m_ref, l_run);
                size_s[st] = 1.f / r;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&halves_met);
                ok = ok && warp_wait(&halves_met, met++ & 1, &dead, p.wait_limit);
            }
            tc_fence_after();
            if (!ok) {                                                       // NaN for all that this unit says
                l_run = NAN;
                m_ref = 0.f;
            }
            const float size = 1.f / r;                                      // O times this is in its own size
            if (w.parts == 0) {
                float inv = l_run == 0.f ? 0.f : size / l_run, z = 1.f, zo = 0.f;        // a query without a visible key: zeros
                if (w.few && ok) {
                    const float2 other = ml_s[st ^ K8P_ROWS];
                    const float m = fmaxf(m_ref, other.x);
                    z = m_ref == -INFINITY ? 0.f : exp2f(m_ref - m), zo = other.x == -INFINITY ? 0.f : exp2f(other.x - m);
                    const float L = h == 0 ? l_run * z + other.y * zo : other.y * zo + l_run * z;
                    inv = L == 0.f ? 0.f : 1.f / L;
                    z *= size, zo *= size_s[st ^ K8P_ROWS];
                }
                const size_t off = ((size_t)(w.row0 + my_tok) * p.nq + (size_t)w.head * p.G + head) * D;
                const int c0 = w.few ? h * (D / 32) : 0, c1 = w.few ? c0 + D / 32 : D / 16;      // few: each half of the warps puts half of the dims together
#pragma unroll 1
                for (int c = c0; c < c1; ++c) {
                    uint32_t o[16], hi[8], lo[8];
                    tmem_ld16_nowait(o_at + 16 * c, o);
                    tmem_arrived<16>(o);
                    if (w.few) {                                             // a half without a page has nothing in tensor memory
                        uint32_t x[16];
                        tmem_ld16_nowait(lanes + C::COL_O + (1 - h) * D + 16 * c, x);
                        tmem_arrived<16>(x);
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const float u = z == 0.f ? 0.f : __uint_as_float(o[k]) * z, v = zo == 0.f ? 0.f : __uint_as_float(x[k]) * zo;
                            o[k] = __float_as_uint(h == 0 ? u + v : v + u);
                        }
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float x = __uint_as_float(o[2 * k]) * inv, y = __uint_as_float(o[2 * k + 1]) * inv;
                        hi[k] = pack_bf16(x, y);
                        lo[k] = pack_bf16(x - bf16_lo(hi[k]), y - bf16_hi(hi[k]));
                    }
                    if (valid) {
                        uint4* to = reinterpret_cast<uint4*>(p.out + off + 16 * c);
                        to[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        to[1] = make_uint4(hi[4], hi[5], hi[6], hi[7]);
                        if (p.out_lo) {
                            to = reinterpret_cast<uint4*>(p.out_lo + off + 16 * c);
                            to[0] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                            to[1] = make_uint4(lo[4], lo[5], lo[6], lo[7]);
                        }
                    }
                }
                if (w.few) {                                                 // the other half has read what the next products write over
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&halves_met);
                    ok = ok && warp_wait(&halves_met, met++ & 1, &dead, p.wait_limit);
                }
            } else {
                // a part: O in its own size, 16 bytes a row side by side, maximum and sum of each row; the halves of a unit of few tokens are two parts
                float4* part = reinterpret_cast<float4*>(p.parts + (2 * (size_t)blockIdx.x + w.begins) * C::PART);
                const float f = mine_n ? size : 0.f;
#pragma unroll 1
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t o[16];
                    tmem_ld16_nowait(o_at + 16 * c, o);
                    tmem_arrived<16>(o);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (valid)
                            part[(size_t)(4 * c + k) * (2 * K8P_ROWS) + st] =
                                mine_n ? make_float4(__uint_as_float(o[4 * k]) * f, __uint_as_float(o[4 * k + 1]) * f, __uint_as_float(o[4 * k + 2]) * f, __uint_as_float(o[4 * k + 3]) * f)
                                       : make_float4(0.f, 0.f, 0.f, 0.f);
                }
                if (valid) reinterpret_cast<float2*>(part + (size_t)(D / 4) * (2 * K8P_ROWS))[st] = make_float2(m_ref, l_run);
                if (st == 0 && w.begins)                                     // what the next kernel has to know of the unit
                    p.split[blockIdx.x] = Kv8Split{w.parts, w.row0, w.head, w.few ? -w.tokens : w.tokens};
            }
            base += w.pages;
            done(seg);
        }
        tmem_st_wait();
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && dead) *err = 1;
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, C::COLS);
    }
}

// Units that lie in several shares, out of their parts.  CTA (c, y) puts together dims 16 y .. 16 y + 15 of the unit that begins in share c and goes on in the next
// ones; a lane has a row, a warp 32 of them side by side.  Few parts: each warp has rows of its own; many (few tokens over a long history): all warps have the same rows
// and every eighth part each.
constexpr int K8P_MERGE_WARPS = 2 * K8P_ROWS / 32, K8P_FEW_PARTS = 8;
template <int D>
__global__ void __launch_bounds__(K8P_MERGE_WARPS * 32)
kv8_prefill_merge_kernel(const __grid_constant__ Kv8Prompt p) {
    pdl_wait();
    using C = K8Prefill<D>;
    __shared__ float acc_s[K8P_MERGE_WARPS][18][32];
    const Kv8Split u = p.split[blockIdx.x];
    if (u.parts == 0) return;
    const bool few = u.tokens < 0;
    const int n_tok = few ? -u.tokens : u.tokens, subs = few ? 2 : 1, np = u.parts * subs;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.y;
    const bool alone = np <= K8P_FEW_PARTS;
    for (int g = alone ? warp : 0; g < (few ? 1 : 2) * K8P_ROWS / 32; g += alone ? K8P_MERGE_WARPS : 1) {
        const int r = 32 * g + lane, row = r & 127, tok = row * p.inv_g >> 16, t = (r >> 7) * p.th + tok;
        const bool valid = tok < p.th && t < n_tok;
        if (!__any_sync(0xffffffffu, valid)) continue;               // the same for all warps of the CTA that are at g
        float M = -INFINITY, L = 0.f, acc[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) acc[k] = 0.f;
        const int first = alone ? 0 : warp, stride = alone ? 1 : K8P_MERGE_WARPS;
        for (int x0 = first; x0 < np; x0 += 4 * stride) {
            float2 ml[4];
            float4 o[4][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {                            // four parts asked for at once
                const int x = min(x0 + k * stride, np - 1);
                const float4* part = reinterpret_cast<const float4*>(p.parts + (2 * (size_t)(blockIdx.x + x / subs) + (x < subs)) * C::PART);
                const int rr = r + (x % subs) * K8P_ROWS;
                const bool on = valid && x0 + k * stride < np;
                ml[k] = make_float2(-INFINITY, 0.f);
                if (on) ml[k] = reinterpret_cast<const float2*>(part + (size_t)(D / 4) * (2 * K8P_ROWS))[rr];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[k][e] = on ? part[(size_t)(4 * c + e) * (2 * K8P_ROWS) + rr] : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            const float Mn = fmaxf(M, fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)));
            const float keep = M == -INFINITY ? 0.f : exp2f(M - Mn);
            L *= keep;
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[k] *= keep;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float z = ml[k].x == -INFINITY ? 0.f : exp2f(ml[k].x - Mn);
                L = fmaf(ml[k].y, z, L);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    acc[4 * e] = fmaf(o[k][e].x, z, acc[4 * e]);
                    acc[4 * e + 1] = fmaf(o[k][e].y, z, acc[4 * e + 1]);
                    acc[4 * e + 2] = fmaf(o[k][e].z, z, acc[4 * e + 2]);
                    acc[4 * e + 3] = fmaf(o[k][e].w, z, acc[4 * e + 3]);
                }
            }
            M = Mn;
        }
        if (!alone) {
#pragma unroll
            for (int k = 0; k < 16; ++k) acc_s[warp][k][lane] = acc[k];
            acc_s[warp][16][lane] = M;
            acc_s[warp][17][lane] = L;
            __syncthreads();
            if (warp == 0) {
                float Mn = M, Ls = 0.f;
                for (int x = 1; x < K8P_MERGE_WARPS; ++x) Mn = fmaxf(Mn, acc_s[x][16][lane]);
#pragma unroll
                for (int k = 0; k < 16; ++k) acc[k] = 0.f;
                for (int x = 0; x < K8P_MERGE_WARPS; ++x) {
                    const float z = acc_s[x][16][lane] == -INFINITY ? 0.f : exp2f(acc_s[x][16][lane] - Mn);
                    Ls = fmaf(acc_s[x][17][lane], z, Ls);
#pragma unroll
                    for (int k = 0; k < 16; ++k) acc[k] = fmaf(acc_s[x][k][lane], z, acc[k]);
                }
                L = Ls;
            }
            __syncthreads();
            if (warp) continue;
        }
        if (!valid) continue;
        const float inv = L == 0.f ? 0.f : 1.f / L;
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float x = acc[2 * k] * inv, y = acc[2 * k + 1] * inv;
            hi[k] = pack_bf16(x, y);
            lo[k] = pack_bf16(x - bf16_lo(hi[k]), y - bf16_hi(hi[k]));
        }
        const size_t off = ((size_t)(u.row0 + t) * p.nq + (size_t)u.head * p.G + (row - tok * p.G)) * D + 16 * c;
        uint4* to = reinterpret_cast<uint4*>(p.out + off);
        to[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        to[1] = make_uint4(hi[4], hi[5], hi[6], hi[7]);
        if (p.out_lo) {
            to = reinterpret_cast<uint4*>(p.out_lo + off);
            to[0] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            to[1] = make_uint4(lo[4], lo[5], lo[6], lo[7]);
        }
    }
}

template <int D>
static int launch_kv8_prefill(Kv8Prompt& p, void* scratch, cudaStream_t st) {
    using C = K8Prefill<D>;
    static_assert(C::SMEM <= 232448 - 4096 && C::REC % 16 == 0, "shared memory");
    static PerDeviceFlag attr_set;
    if (!attr_set.done()) {
        FT_CHECK_CUDA(cudaFuncSetAttribute(kv8_prefill_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        attr_set.mark();
    }
    const int ctas = device_sms();
    // parts only where a unit can be longer than a share by more than K8P_WHOLE, or there are more units than SMs
    const bool parts = ((long long)p.T / (2 * p.th) + p.n_req) * p.nkv > ctas || p.max_pages > K8P_WHOLE;
    FT_REQUIRE(!parts || scratch, "ft_attn_prefill_kv8: needs ft_attn_prefill_kv8_scratch_bytes of work memory");
    p.split = parts ? (Kv8Split*)scratch : nullptr;
    p.parts = (float*)scratch + kv8_prefill_splits(ctas);
    FT_CHECK_CUDA(launch_after(kv8_prefill_kernel<D>, dim3(ctas), dim3(K8P_THREADS), C::SMEM, st, (const Kv8Prompt&)p));
    if (parts) FT_CHECK_CUDA(launch_after(kv8_prefill_merge_kernel<D>, dim3(ctas, D / 16), dim3(K8P_MERGE_WARPS * 32), 0, st, (const Kv8Prompt&)p));
    return 0;
}

int kv8_prefill_waits(int* out) {
    FT_CHECK_CUDA(cudaMemcpyFromSymbol(out, g_kv8_prefill_waits, sizeof(*out)));
    return 0;
}

}  // namespace ft

extern "C" long long ft_attn_prefill_kv8_scratch_bytes(int d) {
    FT_REQUIRE(d == 64 || d == 128, "ft_attn_prefill_kv8_scratch_bytes: head_dim %d not supported (64 or 128)", d);
    const int ctas = ft::device_sms();
    return (long long)(ft::kv8_prefill_splits(ctas) + 2 * (size_t)ctas * (d == 64 ? ft::K8Prefill<64>::PART : ft::K8Prefill<128>::PART)) * 4;
}

extern "C" int ft_attn_prefill_kv8(const void* q, const void* kv8_layer, int num_pages, const int* page_table, int table_rows, int max_pages,
                                   const int* req_q_start, const int* req_slot, const int* req_pos0, int n_req, int T, void* out, void* out_lo, void* scratch,
                                   int nq, int nkv, int d, void* stream) {
    using namespace ft;
    FT_REQUIRE(d == 64 || d == 128, "ft_attn_prefill_kv8: head_dim %d not supported (64 or 128)", d);
    FT_REQUIRE(nq >= 1 && nkv >= 1 && nq % nkv == 0 && nq / nkv <= K8P_GROUP, "ft_attn_prefill_kv8: GQA group %d/%d not supported", nq, nkv);
    FT_REQUIRE(T >= 0 && n_req >= 0 && table_rows >= 0 && max_pages >= 0 && num_pages >= 0 && (long long)max_pages * kKvTile + T <= INT32_MAX - 64,
               "ft_attn_prefill_kv8: bad sizes T=%d n_req=%d nkv=%d table %d x %d, %d pages", T, n_req, nkv, table_rows, max_pages, num_pages);
    // the work's list: at most so many tiles of at most so many pages, and what the shares are rounded up by
    FT_REQUIRE(((double)T / (2 * (K8P_ROWS / (nq / nkv))) + n_req) * ((double)max_pages + T / kKvTile + 2 + kKv8Start) * nkv + 4096 <= INT32_MAX,
               "ft_attn_prefill_kv8: %d tokens of %d requests over %d pages are more than one call takes", T, n_req, max_pages);
    if (T == 0) return 0;
    FT_REQUIRE(q && out && (n_req == 0 || (req_q_start && req_slot && req_pos0 && kv8_there(page_table, table_rows, max_pages, kv8_layer, num_pages))), "ft_attn_prefill_kv8: null argument");
    FT_REQUIRE(((uintptr_t)q | (uintptr_t)kv8_layer | (uintptr_t)out | (uintptr_t)out_lo | (uintptr_t)scratch) % 16 == 0, "ft_attn_prefill_kv8: tensors on 16 bytes");
    const int G = nq / nkv;
    Kv8Prompt p{(const __half*)q, (const uint8_t*)kv8_layer, page_table, req_q_start, req_slot, req_pos0, (__nv_bfloat16*)out, (__nv_bfloat16*)out_lo, nullptr, nullptr,
                num_pages, table_rows, max_pages, n_req, T, nq, nkv, G, K8P_ROWS / G, d == 64 ? 2 : 1, ft::kv8_wait_limit(), (65536u + G - 1) / G, K8P_LOG2E / sqrtf((float)d)};
    return d == 64 ? launch_kv8_prefill<64>(p, scratch, (cudaStream_t)stream) : launch_kv8_prefill<128>(p, scratch, (cudaStream_t)stream);
}
