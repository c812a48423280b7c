// Causal attention of prompt portions over the 8-bit KV cache (kv8.cuh) on tcgen05 / TMEM: request r owns rows req_q_start[r] .. req_q_start[r + 1] - 1 of q, its
// first query sits at position req_pos0[r], and out[t][h] = sum_j softmax_j(q . k_j / sqrt(D)) v_j over the keys j <= position of t.
//
// A unit of work is a tile of query tokens of one request and one key head: two halves of up to 128 rows (row = token * G + head of the group), so that every
// record that reaches an SM serves both.  Per page and half, as in attention_tc.cu:  S = Q K^T (M128 N64 K=D, both operands in shared memory), one thread a row
// for the softmax, P to tensor memory over the scores it came from, O += P V (A from tensor memory, M128 N=D K64).  A unit whose tokens fill one half only gives
// both halves the same queries and every other page each.
//
// The tensor cores want fp16, so four warps turn each record into the two operands, swizzled as the instructions read them: key codes as they are (the blocks' scales
// go to the scores, one multiplication per 16 of them for the maximum and the multiply-add's factor for the exponents), value codes times their block's scale relative
// to the largest of the stretch of pages at hand, which the same warps look up ahead (vref; the output takes it back).  Both roundings are fp16's 2^-11 of a value.
//
// The flat list of all (request, key head, tile, page) is cut into equal shares, one for each SM: a causal list's units differ in length by any factor, and shares do
// not.  A unit that lies in several shares is put together by a second kernel, in the parts' order.  Where there is an SM for every unit and none is much longer than
// a share, each CTA takes a whole one.  Everything is found by each CTA from the lists on the device; nothing is planned ahead.
#include "common.cuh"
#include "ft_internal.h"
#include "kv8.cuh"
#include "kv8_walk.cuh"

namespace ft {

constexpr int K8P_THREADS = 448;                 // warp 0 copies records, 1 issues products, 2 .. 9 softmax (half = (warp - 2) / 4), 10 .. 13 convert
constexpr int K8P_SOFT = 256, K8P_CONV = 128;
constexpr int K8P_ROWS = 128;                    // rows of a half
constexpr int K8P_GROUP = 8;                     // query heads a key head at most
constexpr int K8P_PIECE = kKvTile * 128;         // [64 tokens][64 dims] in fp16; 64 rows of a Q block
constexpr float K8P_LOG2E = 1.4426950408889634f;
constexpr float K8P_GROW = 8.f;                  // O is rescaled when a row's maximum has grown by more than 2^8
constexpr int K8P_WHOLE = 5;                     // pages that a share may be shorter than a whole unit for parts not to pay

template <int D>
struct K8Prefill {
    static constexpr int KH = D / 64;
    static constexpr int TILE = 2 * KH * K8P_PIECE;                  // K | V of a page in fp16
    static constexpr int S16 = D == 64 ? 6 : 3, S8 = D == 64 ? 6 : 3;
    static constexpr int QBLK = K8P_ROWS * 128;                      // [128 rows][64 dims]
    static constexpr int Q_BYTES = 2 * KH * QBLK;
    static constexpr int KV = Q_BYTES, REC = KV + S16 * TILE, BARS = REC + S8 * Kv8<D>::REC;
    static constexpr int N_BARS = 2 * S16 + 2 * S8 + 2 + 12 + 2;              // an even number: 16-byte words behind them
    static constexpr int SMEM = 1024 + BARS + N_BARS * 8 + S16 * 16 + S8 * 4;
    static constexpr int COL_S = 0, COL_O = 256, COLS = 512;
    static constexpr size_t PART = (size_t)2 * K8P_ROWS * (D + 2);   // floats of a part: O [256][D], then (m, l) [256]
};

// floats that the descriptions of split units take at the head of the work memory
static size_t kv8_prefill_splits(int ctas) { return (size_t)(ctas + 15) / 16 * 16 * (sizeof(Kv8Split) / 4); }

template <int D>
__global__ void __launch_bounds__(K8P_THREADS, 1)
kv8_prefill_kernel(const __grid_constant__ Kv8Prompt p) {
    using C = K8Prefill<D>;
    constexpr int KH = C::KH;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* kv_full = reinterpret_cast<uint64_t*>(smem + C::BARS);         // [S16] a page's operands are there
    uint64_t* kv_empty = kv_full + C::S16;
    uint64_t* rec_full = kv_empty + C::S16;                                  // [S8] a record is there
    uint64_t* rec_empty = rec_full + C::S8;
    uint64_t* q_full = rec_empty + C::S8;
    uint64_t* q_empty = q_full + 1;
    uint64_t* s_full = q_empty + 1;                                          // [2][2] half, buffer: scores are in tensor memory
    uint64_t* p_full = s_full + 4;                                           // [2][2] probabilities are
    uint64_t* pv_done = p_full + 4;                                          // [2][2] O += P V retired
    uint64_t* drained = pv_done + 4;                                         // all products retired (after a wait that ran out)
    float* kscale_s = reinterpret_cast<float*>(kv_full + C::N_BARS);                 // [S16][4], times scale_log2; the first below 0: the page is not there
    int* there_s = reinterpret_cast<int*>(kscale_s + 4 * C::S16);            // [S8]
    __shared__ uint32_t tmem_slot;
    __shared__ long long s_sum[K8P_THREADS / 32], s_units[K8P_THREADS / 32];
    __shared__ int s_most[K8P_THREADS / 32], s_r, s_h, s_i, s_t;
    __shared__ float2 s_ml[K8P_SOFT];
    __shared__ float s_vref[4], s_vmax[K8P_CONV / 32];
    __shared__ volatile int dead;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < C::S16; ++s) mbar_init(&kv_full[s], K8P_CONV / 32), mbar_init(&kv_empty[s], 1);
        for (int s = 0; s < C::S8; ++s) mbar_init(&rec_full[s], 1), mbar_init(&rec_empty[s], K8P_CONV / 32);
        mbar_init(q_full, K8P_CONV / 32);
        mbar_init(q_empty, 1);
        for (int k = 0; k < 4; ++k) mbar_init(&s_full[k], 1), mbar_init(&p_full[k], K8P_ROWS / 32), mbar_init(&pv_done[k], 1);
        mbar_init(drained, 1);
        fence_mbar_init();
        dead = 0;
    }
    if (warp == 1) {
        tmem_alloc(&tmem_slot, C::COLS);
        tmem_relinquish();
    }

    // ---------------- the plan: this CTA's share
    const int chunk = (p.n_req + K8P_THREADS - 1) / K8P_THREADS;
    const int r0 = min(p.n_req, tid * chunk), r1 = min(p.n_req, r0 + chunk);
    Kv8Walk w;
    long long mine = 0, units = 0;
    int most = 0;
    for (int r = r0; r < r1; ++r) {
        w.q.load(p, r);
        mine += w.q.all(p);
        units += w.q.tiles;
        if (w.q.tiles) most = max(most, max(w.q.steps(p, w.q.tiles - 1), w.q.tiles > 1 ? w.q.steps(p, w.q.tiles - 2) : 0));
    }
    long long b_steps = mine, b_units = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, b_steps, o), y = __shfl_up_sync(0xffffffffu, b_units, o);
        if (lane >= o) b_steps += x, b_units += y;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 31) s_sum[warp] = b_steps, s_units[warp] = b_units, s_most[warp] = most;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    b_steps -= mine;
    b_units -= units;
    long long total = 0, n_units = 0;
    for (int k = 0; k < K8P_THREADS / 32; ++k) {
        if (k < warp) b_steps += s_sum[k], b_units += s_units[k];
        total += s_sum[k];
        n_units += s_units[k];
        most = max(most, s_most[k]);
    }
    total *= p.nkv;
    n_units *= p.nkv;
    const long long per = (total + gridDim.x - 1) / gridDim.x;
    const bool whole = p.split == nullptr || (n_units <= gridDim.x && most <= per + K8P_WHOLE);      // no room for parts: the host knows that there are none
    // the flat list is one of units or of steps
    const long long len = whole ? n_units : total, each = whole ? 1 : per;
    w.f = min(len, each * blockIdx.x);
    w.f_end = min(len, w.f + each);
    const bool work = w.f < w.f_end;
    const long long at0 = whole ? b_units : b_steps;
    if (work && at0 * p.nkv <= w.f && w.f < (at0 + (whole ? units : mine)) * p.nkv) {
        w.seek(p, whole, r0, at0, w.f);
        s_r = w.r; s_h = w.h; s_i = w.i; s_t = w.t;
    }
    __syncthreads();
    if (work) {
        w.r = s_r; w.h = s_h; w.i = s_i; w.t = s_t;
        w.q.load(p, w.r);
        w.unit(p);
        if (whole) w.f = 0, w.f_end = w.n_steps;
    }
    bool ok = true;                                                          // false: a wait ran out
    int* const err = p.err;

    if (warp == 0) {
        // ---------------- copies: one record a page
        const uint64_t pol = policy_evict_last();                            // read again by other tiles
        int it = 0, asked = 0;
        while (w.next(p)) {
            const int* pt = p.page_table + (size_t)w.q.slot * p.max_pages;
            const int most_here = w.q.slot >= 0 && w.q.slot < p.table_rows ? p.max_pages : 0;
            const int p1 = w.page1();
            for (int p0 = w.page0(); p0 < p1; p0 += 32) {
                const int mine_ = p0 + lane;
                const int my_page = mine_ < p1 && mine_ < most_here ? pt[mine_] : -1;
                const int n = min(32, p1 - p0);
                for (int k = 0; k < n; ++k, ++it) {
                    const int page = __shfl_sync(0xffffffffu, my_page, k);
                    if (lane == 0 && ok) {
                        const int s = it % C::S8;
                        ok = mbar_wait_limited(&rec_empty[s], (it / C::S8 & 1) ^ 1, &dead);
                        if (!ok) continue;
                        asked = it + 1;
                        const bool there = page >= 0 && page < p.num_pages;
                        there_s[s] = there;
                        if (there) {
                            mbar_expect_tx(&rec_full[s], Kv8<D>::REC);
                            tma_bulk_g2s(smem + C::REC + s * Kv8<D>::REC, p.cache + ((size_t)page * p.nkv + w.h) * Kv8<D>::REC, Kv8<D>::REC, &rec_full[s], pol);
                        } else {
                            mbar_arrive(&rec_full[s]);
                        }
                    }
                }
            }
        }
        if (lane == 0 && (!ok || dead)) {                                    // what is under way still lands in this CTA's memory
            *err = 1;
            for (int i = max(0, asked - C::S8); i < asked; ++i)
                for (int k = 0; k < kWaitLimit && !mbar_try_wait(&rec_full[i % C::S8], i / C::S8 & 1); ++k) {}
        }
    } else if (warp == 1) {
        // ---------------- products
        if (elect_one()) {
            constexpr uint32_t idesc_qk = umma_idesc_f16(K8P_ROWS, kKvTile, false), idesc_pv = umma_idesc_f16(K8P_ROWS, D, true);
            const uint32_t q_addr = smem_u32(smem), kv_addr = smem_u32(smem + C::KV);
            int base = 0, seg = 0;                                           // pages so far; stretches so far
            int n_qk[2] = {0, 0}, n_pv[2] = {0, 0};                          // products of each half so far
            auto issue_qk = [&](int h, int page, int qh) {                   // page: counted over the whole share
                const int s = page % C::S16;
                ok = ok && mbar_wait_limited(&kv_full[s], page / C::S16 & 1, &dead);
                if (!ok) return;
                tc_fence_after();
                const int buf = n_qk[h]++ & 1;
#pragma unroll
                for (int kh = 0; kh < KH; ++kh) {
                    const uint64_t a = umma_desc_k128(q_addr + (qh * KH + kh) * C::QBLK), b = umma_desc_k128(kv_addr + s * C::TILE + kh * K8P_PIECE);
#pragma unroll
                    for (int k = 0; k < 4; ++k) umma_bf16(tmem + C::COL_S + (2 * h + buf) * 64, a + 2 * k, b + 2 * k, idesc_qk, (kh | k) != 0);
                }
                umma_commit(&s_full[2 * h + buf]);
            };
            auto issue_pv = [&](int h, int page, bool first, bool last) {
                const int s = page % C::S16, buf = n_pv[h] & 1;
                ok = ok && mbar_wait_limited(&p_full[2 * h + buf], n_pv[h] >> 1 & 1, &dead);
                if (!ok) return;
                ++n_pv[h];
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < kKvTile / 16; ++k)
                    umma_f16_ts(tmem + C::COL_O + h * D, tmem + C::COL_S + (2 * h + buf) * 64 + 8 * k,
                                umma_desc_mn128(kv_addr + s * C::TILE + KH * K8P_PIECE + k * 2048), idesc_pv, k != 0 || !first);
                umma_commit(&pv_done[2 * h + buf]);
                if (last) umma_commit(&kv_empty[s]);
            };
            while (ok && w.next(p)) {
                ok = mbar_wait_limited(q_full, seg & 1, &dead);
                if (!ok) break;
                tc_fence_after();
                const int n = w.page1() - w.page0();
                if (w.few) {
                    // page j is half (j & 1)'s; scores run two pages ahead
                    for (int j = -2; ok && j < n; ++j) {
                        if (j >= 0) issue_pv(j & 1, base + j, j < 2, true);
                        if (j + 2 < n) issue_qk(j & 1, base + j + 2, 0);
                        if (j + 2 == n - 1) umma_commit(q_empty);
                    }
                } else {
                    for (int j = -2; ok && j < n; ++j)
                        for (int h = 0; h < 2; ++h) {
                            if (j >= 0) issue_pv(h, base + j, j == 0, h == 1);
                            if (j + 2 < n) issue_qk(h, base + j + 2, h);
                            if (j + 2 == n - 1 && h == 1) umma_commit(q_empty);
                        }
                }
                base += n;
                ++seg;
            }
            if (!ok) {                                                       // nothing may still run in tensor memory when it is given back
                *err = 1;
                umma_commit(drained);
                for (int k = 0; k < kWaitLimit && !mbar_try_wait(drained, 0); ++k) {}
            }
        }
        __syncwarp();
    } else if (warp >= 2 + K8P_SOFT / 32) {
        // ---------------- conversion: Q of each stretch, then its pages
        const int ct = tid - 64 - K8P_SOFT, cw = ct >> 5;
        int it = 0, seg = 0;
        while (w.next(p)) {                                                  // after a wait that ran out: only the barriers that the four warps share
            const int g0 = w.page0(), g1 = w.page1();
            // the largest scale of the stretch's values: its pages are asked for first, the answers are used after Q
            const int* pt = p.page_table + (size_t)w.q.slot * p.max_pages;
            const int most_here = w.q.slot >= 0 && w.q.slot < p.table_rows ? min(g1, p.max_pages) : 0;
            float vmax = 0.f;
            for (int k = g0 + ct; k < most_here; k += K8P_CONV) {
                const int page = pt[k];
                if (page < 0 || page >= p.num_pages) continue;
                const float4 v = *reinterpret_cast<const float4*>(p.cache + ((size_t)page * p.nkv + w.h) * Kv8<D>::REC + Kv8<D>::SCALES + 16);
                vmax = fmaxf(vmax, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
            }
            if (seg) ok = ok && mbar_wait_limited(q_empty, (seg - 1) & 1, &dead);
            ok = __all_sync(0xffffffffu, ok);
            const int halves = !ok ? 0 : w.few ? 1 : 2, row0 = w.row0(p);
            constexpr int CH = D / 8;
#pragma unroll 8
            for (int k = ct; k < halves * K8P_ROWS * CH; k += K8P_CONV) {    // 16 bytes each, all on their way at once; zeros for rows without a token
                const int c = k % CH, rr = k / CH, h = rr >> 7, row = rr & 127;
                const int tok = row * p.inv_g >> 16, head = row - tok * p.G;
                const bool on = tok < p.th && h * p.th + tok < w.n_tok;
                const __half* from = p.q + ((size_t)(row0 + (on ? h * p.th + tok : 0)) * p.nq + (size_t)w.h * p.G + (on ? head : 0)) * D + c * 8;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem + (h * KH + (c >> 3)) * C::QBLK + row * 128 + ((c & 7) ^ (row & 7)) * 16)),
                             "l"(from), "r"(on ? 16 : 0)
                             : "memory");
            }
            vmax = warp_max(vmax);
            if (lane == 0) s_vmax[cw] = vmax;
            asm volatile("bar.sync 2, %0;" ::"n"(K8P_CONV) : "memory");
            vmax = fmaxf(fmaxf(s_vmax[0], s_vmax[1]), fmaxf(s_vmax[2], s_vmax[3]));
            asm volatile("bar.sync 2, %0;" ::"n"(K8P_CONV) : "memory");
            if (ct == 0) s_vref[seg & 3] = vmax;                             // the softmax warps may still be at the end of the stretch before the last
            const float vinv = vmax > 0.f ? 1.f / vmax : 0.f;
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_proxy_async();
            __syncwarp();
            if (lane == 0 && ok) mbar_arrive(q_full);
            ++seg;
            for (int k = g0; ok && k < g1; ++k, ++it) {
                const int s8 = it % C::S8, s16 = it % C::S16;
                ok = mbar_wait_limited(&rec_full[s8], it / C::S8 & 1, &dead) && mbar_wait_limited(&kv_empty[s16], (it / C::S16 & 1) ^ 1, &dead);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const uint8_t* rec = smem + C::REC + s8 * Kv8<D>::REC;
                uint8_t* dst = smem + C::KV + s16 * C::TILE;
                const bool there = there_s[s8];
                const float* scales = reinterpret_cast<const float*>(rec + Kv8<D>::SCALES);
                // a block of zeros keeps a factor above 0, so that hidden scores stay minus infinity
                if (ct < 4) kscale_s[4 * s16 + ct] = there ? fmaxf(scales[ct] * p.scale_log2, 1e-37f) : -1.f;
#pragma unroll 4
                for (int u = ct; u < kKvTile * D / 16; u += K8P_CONV) {      // keys: 16 codes, two chunks of the swizzled row
                    const int piece = u >> 8, t = u >> 2 & 63, c = u & 3;
                    uint4 x = *reinterpret_cast<const uint4*>(rec + u * 16);
                    if (!there) x = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
                    uint8_t* at = dst + piece * K8P_PIECE + t * 128;
                    *reinterpret_cast<uint4*>(at + ((2 * c) ^ (t & 7)) * 16) = make_uint4(kv8_lo(x.x), kv8_hi(x.x), kv8_lo(x.y), kv8_hi(x.y));
                    *reinterpret_cast<uint4*>(at + ((2 * c + 1) ^ (t & 7)) * 16) = make_uint4(kv8_lo(x.z), kv8_hi(x.z), kv8_lo(x.w), kv8_hi(x.w));
                }
                dst += KH * K8P_PIECE;
#pragma unroll 4
                for (int u = ct; u < kKvTile * D / 16; u += K8P_CONV) {      // values, by where they lie
                    const int piece = u >> 8, slot = u >> 2 & 63, t = slot ^ (slot >> 1 & 1), c = (u & 3) ^ (t >> 1 & 2);
                    uint4 x = *reinterpret_cast<const uint4*>(rec + Kv8<D>::SLAB + u * 16);
                    if (!there) x = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
                    const __half2 f = __float2half2_rn(there ? scales[4 + (t >> 4)] * vinv : 0.f);
                    auto mul = [&](uint32_t y) {
                        const __half2 z = __hmul2(*reinterpret_cast<const __half2*>(&y), f);
                        return *reinterpret_cast<const uint32_t*>(&z);
                    };
                    uint8_t* at = dst + piece * K8P_PIECE + t * 128;
                    *reinterpret_cast<uint4*>(at + ((2 * c) ^ (t & 7)) * 16) = make_uint4(mul(kv8_lo(x.x)), mul(kv8_hi(x.x)), mul(kv8_lo(x.y)), mul(kv8_hi(x.y)));
                    *reinterpret_cast<uint4*>(at + ((2 * c + 1) ^ (t & 7)) * 16) = make_uint4(mul(kv8_lo(x.z)), mul(kv8_hi(x.z)), mul(kv8_lo(x.w)), mul(kv8_hi(x.w)));
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&kv_full[s16]), mbar_arrive(&rec_empty[s8]);
            }
        }
    } else {
        // ---------------- softmax: one thread a row
        const int st = tid - 64, h = (warp - 2) >> 2, quarter = warp & 3;
        const int row = quarter * 32 + lane;                                 // lane of tensor memory
        const int tok = row * p.inv_g >> 16, head = row - tok * p.G;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint32_t s_at = lanes + C::COL_S + 2 * h * 64, o_at = lanes + C::COL_O + h * D;
        if (st == 0 && p.split) p.split[blockIdx.x].parts = 0;
        // rows that no request owns
        {
            const int a = p.n_req ? max(0, min(p.req_q_start[0], p.T)) : p.T, b = p.n_req ? max(a, min(p.req_q_start[p.n_req], p.T)) : p.T;
            const int n = a + p.T - b;
            for (int i = blockIdx.x; i < n; i += gridDim.x) {
                const size_t at = (size_t)(i < a ? i : b + i - a) * p.nq * D;
                for (int e = 8 * st; e < p.nq * D; e += 8 * K8P_SOFT) {
                    *reinterpret_cast<uint4*>(p.out + at + e) = make_uint4(0u, 0u, 0u, 0u);
                    if (p.out_lo) *reinterpret_cast<uint4*>(p.out_lo + at + e) = make_uint4(0u, 0u, 0u, 0u);
                }
            }
        }
        int base = 0, seg = 0, cnt = 0;                                      // pages and stretches of the share, pages of this half so far
        while (w.next(p)) {
            const int g0 = w.page0(), n = w.page1() - g0;
            const int mine_n = w.few ? (n - h + 1) / 2 : n;                  // pages of this half
            const int my_tok = w.few ? tok : h * p.th + tok;
            const bool valid = tok < p.th && my_tok < w.n_tok;
            const int pos = w.position0(p) + my_tok;
            float m_ref = -INFINITY, l_run = 0.f;                            // in log2 units
            for (int i = 0; i < mine_n; ++i, ++cnt) {
                const int j = w.few ? h + 2 * i : i;                         // page of the stretch
                const int buf = cnt & 1, ph = cnt >> 1 & 1, it = base + j, s16 = it % C::S16;
                ok = ok && mbar_wait_limited(&s_full[2 * h + buf], ph, &dead) && mbar_wait_limited(&kv_full[s16], it / C::S16 & 1, &dead);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = s_at + buf * 64;
                uint32_t sr[64];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld16_nowait(at + 16 * c, sr + 16 * c);
                const float4 ks4 = *reinterpret_cast<const float4*>(kscale_s + 4 * s16);
                const float ks[4] = {ks4.x, ks4.y, ks4.z, ks4.w};
                tmem_ld_wait();
                const int seen = ks4.x < 0.f ? -1 : pos - (g0 + j) * kKvTile;         // the last key of the page that the row sees
                if (seen < kKvTile - 1) {
#pragma unroll
                    for (int c = 0; c < 64; ++c) sr[c] = c <= seen ? sr[c] : 0xff800000u;
                }
                float tmax = -INFINITY;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    float t2[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < 16; ++c) t2[c & 1] = fmaxf(t2[c & 1], __uint_as_float(sr[16 * b + c]));
                    tmax = fmaxf(tmax, fmaxf(t2[0], t2[1]) * fabsf(ks[b]));
                }
                const float m_new = fmaxf(m_ref, tmax);
                const bool grow = valid && m_new > m_ref + K8P_GROW;
                if (i == 0) {
                    m_ref = m_new;
                } else if (__any_sync(0xffffffffu, grow)) {
                    ok = mbar_wait_limited(&pv_done[2 * h + ((cnt - 1) & 1)], (cnt - 1) >> 1 & 1, &dead);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after();
                    const float alpha = m_new == -INFINITY ? 1.f : exp2f(m_ref - m_new);
                    l_run *= alpha;
                    m_ref = m_new;
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t o[16];
                        tmem_ld16_nowait(o_at + 16 * c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
                        tmem_st16(o_at + 16 * c, o);
                    }
                    tmem_st_wait();
                }
                const float mu = m_ref == -INFINITY ? 0.f : m_ref;
                float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c16 = 0; c16 < 2; ++c16) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float f = fabsf(ks[2 * c16 + (e >> 3)]);
                        const float p0 = ex2_fast(fmaf(__uint_as_float(sr[c16 * 32 + 2 * e]), f, -mu));
                        const float p1 = ex2_fast(fmaf(__uint_as_float(sr[c16 * 32 + 2 * e + 1]), f, -mu));
                        ps[(2 * e) & 3] += p0;
                        ps[(2 * e + 1) & 3] += p1;
                        const __half2 t = __floats2half2_rn(p0, p1);
                        pk[e] = *reinterpret_cast<const uint32_t*>(&t);
                    }
                    tmem_st16(at + 16 * c16, pk);
                }
                tmem_st_wait();
                l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[2 * h + buf]);
            }
            if (ok && mine_n) {
                ok = mbar_wait_limited(&pv_done[2 * h + ((cnt - 1) & 1)], (cnt - 1) >> 1 & 1, &dead);
                ok = __all_sync(0xffffffffu, ok);
            }
            tc_fence_after();
            if (!ok) {                                                       // NaN for all that this unit says
                *err = 1;
                l_run = NAN;
                m_ref = 0.f;
            }
            float vref = ok && mine_n ? s_vref[seg & 3] : 0.f;
            const bool all = w.t0 == 0 && w.t1 == w.n_steps;
            const size_t off = ((size_t)(w.row0(p) + my_tok) * p.nq + (size_t)w.h * p.G + head) * D;
            auto put = [&](int c, const uint32_t* o) {                       // 16 dims of the row
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float x = __uint_as_float(o[2 * k]), y = __uint_as_float(o[2 * k + 1]);
                    hi[k] = pack_bf16(x, y);
                    lo[k] = pack_bf16(x - bf16_lo(hi[k]), y - bf16_hi(hi[k]));
                }
                uint4* to = reinterpret_cast<uint4*>(p.out + off + 16 * c);
                to[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                to[1] = make_uint4(hi[4], hi[5], hi[6], hi[7]);
                if (p.out_lo) {
                    to = reinterpret_cast<uint4*>(p.out_lo + off + 16 * c);
                    to[0] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    to[1] = make_uint4(lo[4], lo[5], lo[6], lo[7]);
                }
            };
            if (all && !w.few) {
                const float inv = l_run == 0.f ? 0.f : vref / l_run;         // a query without a visible key: zeros
#pragma unroll 1
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t o[16];
                    tmem_ld16_nowait(o_at + 16 * c, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * inv);
                    if (valid) put(c, o);
                }
            } else if (all) {
                // two halves of the pages: each half of the warps puts half of the dims together
                s_ml[st] = make_float2(m_ref, l_run);
                tc_fence_before();
                asm volatile("bar.sync 1, %0;" ::"n"(K8P_SOFT) : "memory");
                tc_fence_after();
                if (ok) vref = s_vref[seg & 3];                              // a half without a page has waited for nothing before
                const float2 other = s_ml[st ^ K8P_ROWS];
                const float m = fmaxf(m_ref, other.x);
                const float z = m_ref == -INFINITY ? 0.f : exp2f(m_ref - m), zo = other.x == -INFINITY ? 0.f : exp2f(other.x - m);
                const float L = h == 0 ? l_run * z + other.y * zo : other.y * zo + l_run * z;
                const float inv = L == 0.f ? 0.f : vref / L;
#pragma unroll 1
                for (int c = h * (D / 32); c < (h + 1) * (D / 32); ++c) {
                    uint32_t o[16], x[16];
                    tmem_ld16_nowait(o_at + 16 * c, o);
                    tmem_ld16_nowait(lanes + C::COL_O + (1 - h) * D + 16 * c, x);
                    tmem_ld_wait();
#pragma unroll
                    for (int k = 0; k < 16; ++k) {                           // a half without a page has nothing in tensor memory
                        const float u = z == 0.f ? 0.f : __uint_as_float(o[k]) * z, v = zo == 0.f ? 0.f : __uint_as_float(x[k]) * zo;
                        o[k] = __float_as_uint((h == 0 ? u + v : v + u) * inv);
                    }
                    if (valid) put(c, o);
                }
                asm volatile("bar.sync 1, %0;" ::"n"(K8P_SOFT) : "memory");
            } else {
                // a part: O in its own size, maximum and sum of each row; the halves of a unit of few tokens are two parts
                float* part = p.parts + (2 * (size_t)blockIdx.x + (w.t0 == 0)) * C::PART;
                const int rr = h * K8P_ROWS + row;                           // (not st: a warp's rows are those lanes of tensor memory that it may read)
#pragma unroll 1
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t o[16];
                    tmem_ld16_nowait(o_at + 16 * c, o);
                    tmem_ld_wait();
                    float4* to = reinterpret_cast<float4*>(part + (size_t)rr * D + 16 * c);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (valid) to[k] = mine_n ? make_float4(__uint_as_float(o[4 * k]) * vref, __uint_as_float(o[4 * k + 1]) * vref, __uint_as_float(o[4 * k + 2]) * vref,
                                                     __uint_as_float(o[4 * k + 3]) * vref)
                                       : make_float4(0.f, 0.f, 0.f, 0.f);
                }
                if (valid) *reinterpret_cast<float2*>(part + (size_t)2 * K8P_ROWS * D + 2 * rr) = make_float2(m_ref, l_run);
                if (st == 0 && w.t0 == 0)                                    // the unit begins here: what the next kernel has to know of it
                    p.split[blockIdx.x] = Kv8Split{(int)((w.f - w.t1 + w.n_steps - 1) / per) - (int)blockIdx.x + 1, w.row0(p), w.h, w.few ? -w.n_tok : w.n_tok};
            }
            base += n;
            ++seg;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, C::COLS);
    }
}

// Units that lie in several shares, out of their parts.  CTA (c, y) takes rows of the unit that begins in share c and goes on in the next ones.  Few parts: a group of D / 4
// lanes takes a row; many (few tokens over a long history): all groups take one row, every eighth (sixteenth) part each.
constexpr int K8P_MERGE = 256, K8P_SLICES = 16, K8P_FEW_PARTS = 6;
template <int D>
__global__ void __launch_bounds__(K8P_MERGE)
kv8_prefill_merge_kernel(const __grid_constant__ Kv8Prompt p) {
    using C = K8Prefill<D>;
    constexpr int LR = D / 4, GROUPS = K8P_MERGE / LR;
    __shared__ float4 s_acc[GROUPS][LR];
    __shared__ float2 s_ml[GROUPS];
    pdl_wait();
    const Kv8Split u = p.split[blockIdx.x];
    if (u.parts == 0) return;
    const bool few = u.tokens < 0;
    const int n_tok = few ? -u.tokens : u.tokens, subs = few ? 2 : 1, np = u.parts * subs;
    const int group = threadIdx.x / LR, d4 = threadIdx.x % LR * 4;
    const bool alone = np <= K8P_FEW_PARTS;                          // a group has a row to itself
    const int step = alone ? K8P_SLICES * GROUPS : K8P_SLICES;
    for (int r = alone ? blockIdx.y * GROUPS + group : blockIdx.y; r < (few ? 1 : 2) * K8P_ROWS; r += step) {
        const int row = r & 127, tok = row * p.inv_g >> 16, t = (r >> 7) * p.th + tok;
        if (tok >= p.th || t >= n_tok) continue;                     // the same for all that take the row
        float M = -INFINITY, L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        const int first = alone ? 0 : group, stride = alone ? 1 : GROUPS;
        for (int x0 = first; x0 < np; x0 += 4 * stride) {
            float2 ml[4];
            float4 o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {                            // four parts asked for at once
                const int x = min(x0 + k * stride, np - 1), cta = blockIdx.x + x / subs, rec_row = r + (x % subs) * K8P_ROWS;
                const float* rec = p.parts + (2 * (size_t)cta + (x < subs)) * C::PART;
                ml[k] = *reinterpret_cast<const float2*>(rec + (size_t)2 * K8P_ROWS * D + 2 * rec_row);
                o[k] = *reinterpret_cast<const float4*>(rec + (size_t)rec_row * D + d4);
                if (x0 + k * stride >= np) ml[k] = make_float2(-INFINITY, 0.f);
            }
            const float Mn = fmaxf(M, fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)));
            const float keep = M == -INFINITY ? 0.f : exp2f(M - Mn);
            L *= keep; acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float z = ml[k].x == -INFINITY ? 0.f : exp2f(ml[k].x - Mn);
                L = fmaf(ml[k].y, z, L);
                acc = fma_f4(o[k], make_float4(z, z, z, z), acc);
            }
            M = Mn;
        }
        if (!alone) {
            s_acc[group][threadIdx.x % LR] = acc;
            if (d4 == 0) s_ml[group] = make_float2(M, L);
            __syncthreads();
            if (group == 0) {
                float Mn = M;
                for (int k = 1; k < GROUPS; ++k) Mn = fmaxf(Mn, s_ml[k].x);
                float Ls = 0.f;
                float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int k = 0; k < GROUPS; ++k) {
                    const float z = s_ml[k].x == -INFINITY ? 0.f : exp2f(s_ml[k].x - Mn);
                    Ls = fmaf(s_ml[k].y, z, Ls);
                    a = fma_f4(s_acc[k][threadIdx.x], make_float4(z, z, z, z), a);
                }
                L = Ls;
                acc = a;
            }
            __syncthreads();
            if (group) continue;
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const float y0 = acc.x * inv, y1 = acc.y * inv, y2 = acc.z * inv, y3 = acc.w * inv;
        const uint32_t h0 = pack_bf16(y0, y1), h1 = pack_bf16(y2, y3);
        const size_t to = ((size_t)(u.row0 + t) * p.nq + (size_t)u.head * p.G + (row - tok * p.G)) * D + d4;
        *reinterpret_cast<uint2*>(p.out + to) = make_uint2(h0, h1);
        if (p.out_lo)
            *reinterpret_cast<uint2*>(p.out_lo + to) = make_uint2(pack_bf16(y0 - bf16_lo(h0), y1 - bf16_hi(h0)), pack_bf16(y2 - bf16_lo(h1), y3 - bf16_hi(h1)));
    }
}

template <int D>
static int launch_kv8_prefill(Kv8Prompt& p, void* scratch, cudaStream_t st) {
    using C = K8Prefill<D>;
    static_assert(C::SMEM <= 232448 - 3072 && (C::BARS + C::N_BARS * 8) % 16 == 0 && C::REC % 16 == 0, "shared memory");
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
    if (int r = kv8_waits_address(&p.err)) return r;
    kv8_prefill_kernel<D><<<ctas, K8P_THREADS, C::SMEM, st>>>(p);
    FT_CHECK_CUDA(cudaGetLastError());
    if (parts) FT_CHECK_CUDA(launch_after(kv8_prefill_merge_kernel<D>, dim3(ctas, K8P_SLICES), dim3(K8P_MERGE), 0, st, (const Kv8Prompt&)p));
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
    if (T == 0) return 0;
    FT_REQUIRE(q && kv8_layer && out && (n_req == 0 || (page_table && req_q_start && req_slot && req_pos0)), "ft_attn_prefill_kv8: null argument");
    FT_REQUIRE(((uintptr_t)q | (uintptr_t)kv8_layer | (uintptr_t)out | (uintptr_t)out_lo | (uintptr_t)scratch) % 16 == 0, "ft_attn_prefill_kv8: tensors on 16 bytes");
    const int G = nq / nkv;
    Kv8Prompt p{(const __half*)q, (const uint8_t*)kv8_layer, page_table, req_q_start, req_slot, req_pos0, (__nv_bfloat16*)out, (__nv_bfloat16*)out_lo, nullptr, nullptr,
                nullptr, num_pages, table_rows, max_pages, n_req, T, nq, nkv, G, K8P_ROWS / G, (65536u + G - 1) / G, K8P_LOG2E / sqrtf((float)d)};
    return d == 64 ? launch_kv8_prefill<64>(p, scratch, (cudaStream_t)stream) : launch_kv8_prefill<128>(p, scratch, (cudaStream_t)stream);
}
