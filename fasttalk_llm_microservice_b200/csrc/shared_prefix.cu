// Shared part of attention over common prefixes (shared.cuh) on tcgen05 / TMEM: the first tokens of a group, read once for all its queries.
//
// A unit of work is a tile of up to 2 * (128 / G) queries of one group and one key head: two halves of up to 128 rows (row = query * G + head of the group), so that every
// page that reaches an SM serves both.  Per page and half, as in attention_tc.cu:  S = Q K^T (M128 N64 K=D, both operands in shared memory, the cache's slab as it lies),
// one thread a row for the softmax, P to tensor memory over the scores that it came from, O += P V (A from tensor memory, M128 N=D K64).  A unit whose queries fill
// one half only gives both halves the same queries and every other page each.
//
// The list of all (group, key head, tile, page) is cut into equal shares, one for each SM.  What a share has of a unit goes out as O, maximum and sum of each row; the own
// part's kernel puts these together with what a sequence has of its own.  All rows of a unit see all its pages, so the only mask is the end of the last one.
#include "common.cuh"
#include "ft_internal.h"
#include "shared.cuh"

namespace ft {

// warp 0 copies pages, 1 and 2 issue the halves' products, 3 owns tensor memory, 4 .. 11 softmax (half = (warp - 4) / 4)
constexpr int SX_THREADS = 384;
constexpr int SX_SOFT = 256;
constexpr int SX_PIECE = kKvTile * 128;          // [64 tokens][64 dims] in fp16

__device__ int g_shared_prefix_waits;            // 1: a wait ran out on this device (ft_attn_shared_waits)

template <int D>
struct SharedPrefix {
    static constexpr int KH = D / 64;
    static constexpr int TILE = 2 * KH * SX_PIECE;                           // K | V of a page
    static constexpr int STAGES = D == 64 ? 6 : 4;
    static constexpr int QBLK = kSharedRows * 128;                           // [128 rows][64 dims]
    static constexpr int Q_BYTES = 2 * KH * QBLK;
    static constexpr int KV = Q_BYTES, SMEM = 1024 + KV + STAGES * TILE;
    // tensor memory: scores [half][2][64 columns] (probabilities, pairs of fp16, over the first 32 of them), O [half][D]
    static constexpr int COL_S = 0, COL_O = 256, COLS = 512;
    static_assert(COL_O + 2 * D <= COLS, "tensor memory");
};

// A CTA's share, walked stretch by stretch; a stretch = pages p0 .. p1 - 1 of one unit.  Every warp walks for itself
struct PrefixWalk {
    SharedGroup w;
    int f, f_end, g, h, tile, t;
    int n, steps, tiles;                         // queries and steps of the tile, tiles of the group
    int p0, pages;
    bool few;
    __device__ __forceinline__ void unit(const SharedArgs& p) {
        n = min(2 * p.th, w.size - tile * 2 * p.th);
        few = n <= p.th;
        steps = shared_steps(n, p.th, w.pages);
    }
    __device__ __forceinline__ void start(const SharedArgs& p) {
        const int total = p.head->prefix_total, per = p.head->prefix_per;
        f = min(per * (int)blockIdx.x, total);
        f_end = min(f + per, total);
        if (f >= f_end) return;
        g = p.prefix_from[blockIdx.x];
        w = p.groups[g];
        const int each = shared_head_steps(w.size, p.th, w.pages), full = w.pages + kSharedStart;
        tiles = (w.size + 2 * p.th - 1) / (2 * p.th);
        int rest = f - w.base;
        h = (int)((unsigned)rest / (unsigned)each);
        rest -= h * each;
        tile = min((int)((unsigned)rest / (unsigned)full), tiles - 1);
        t = rest - tile * full;
        unit(p);
    }
    __device__ __forceinline__ bool next(const SharedArgs& p) {
#pragma unroll 1
        for (;;) {
            if (f >= f_end) return false;
            if (t >= steps + kSharedStart) {
                t = 0;
                if (++tile == tiles) {
                    tile = 0;
                    if (++h == p.nkv) {
                        h = 0;
#pragma unroll 1
                        do w = p.groups[++g];
                        while (w.pages == 0);
                        tiles = (w.size + 2 * p.th - 1) / (2 * p.th);
                    }
                }
                unit(p);
            }
            const int take = min(f_end - f, steps + kSharedStart - t), t0 = min(t, steps), t1 = min(t + take, steps);
            t += take;
            f += take;
            if (t1 > t0) {
                p0 = few ? 2 * t0 : t0;
                pages = (few ? min(2 * t1, w.pages) : t1) - p0;
                return true;
            }                                                                // else all of it was behind the unit's last step
        }
    }
    __device__ __forceinline__ int of_half(int half) const { return few ? (pages - half + 1) / 2 : pages; }      // its pages
};

template <int D>
__global__ void __launch_bounds__(SX_THREADS, 1)
shared_prefix_kernel(const __grid_constant__ SharedArgs p) {
    using C = SharedPrefix<D>;
    constexpr int KH = C::KH;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t kv_full[C::STAGES], kv_empty[C::STAGES];
    __shared__ uint64_t q_full[2];                                           // the queries of a half
    __shared__ uint64_t s_full[2][2], p_full[2][2], pv_done[2][2];           // half, buffer: scores are in tensor memory; probabilities are; O += P V retired
    __shared__ uint64_t drained[2];                                          // all products of a half retired
    __shared__ int tokens_s[C::STAGES];                                      // of the page in each stage; 0: the page is not there
    __shared__ float2 ml_s[SX_SOFT];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int dead;
    int* const err = &g_shared_prefix_waits;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < C::STAGES; ++s) mbar_init(&kv_full[s], 1), mbar_init(&kv_empty[s], 2);
        for (int h = 0; h < 2; ++h) {
            mbar_init(&q_full[h], kSharedRows / 32);
            mbar_init(&drained[h], 1);
            for (int s = 0; s < 2; ++s) mbar_init(&s_full[h][s], 1), mbar_init(&p_full[h][s], kSharedRows / 32), mbar_init(&pv_done[h][s], 1);
        }
        fence_mbar_init();
        dead = 0;
    }
    if (warp == 3) {
        tmem_alloc(&tmem_slot, C::COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_wait();
    bool ok = true;                                                          // false: a wait ran out
    PrefixWalk w;
    w.start(p);

    if (warp == 0) {
        // ---------------- copies: one page a time
        const uint64_t pol = policy_evict_first();
        int it = 0, asked = 0;
#pragma unroll 1
        while (w.next(p)) {
            const int p1 = w.p0 + w.pages;
#pragma unroll 1
            for (int p0 = w.p0; p0 < p1; p0 += 32) {
                const int tile = p0 + lane;
                int my_page = tile < p1 && w.w.row >= 0 ? p.page_table[(size_t)w.w.row * p.max_pages + tile] : -1;
                if (my_page >= p.num_pages) my_page = -1;
                const int n = min(32, p1 - p0);
#pragma unroll 1
                for (int k = 0; k < n; ++k, ++it) {
                    const int page = __shfl_sync(0xffffffffu, my_page, k);
                    if (lane == 0 && ok) {
                        const int s = it % C::STAGES;
                        ok = mbar_wait_limited(&kv_empty[s], (it / C::STAGES & 1) ^ 1, &dead);
                        if (!ok) continue;
                        asked = it + 1;
                        tokens_s[s] = page >= 0 ? min(kKvTile, w.w.tokens - (p0 + k) * kKvTile) : 0;
                        if (page >= 0) {
                            mbar_expect_tx(&kv_full[s], C::TILE);
                            tma_bulk_g2s(smem + C::KV + s * C::TILE, p.cache + ((size_t)page * p.nkv + w.h) * C::TILE, C::TILE, &kv_full[s], pol);
                        } else {
                            mbar_arrive(&kv_full[s]);
                        }
                    }
                }
            }
        }
        if (lane == 0)
            for (int i = max(0, asked - C::STAGES); i < asked; ++i)          // nothing may still be on its way into this CTA's memory when it ends
                for (int k = 0; k < kWaitLimit && !mbar_try_wait(&kv_full[i % C::STAGES], i / C::STAGES & 1); ++k) {}
        __syncwarp();
    } else if (warp < 3) {
        // ---------------- products, one warp a half
        constexpr uint32_t idesc_qk = umma_idesc_f16(kSharedRows, kKvTile, false), idesc_pv = umma_idesc_f16(kSharedRows, D, true);
        const int h = warp - 1;
        if (elect_one()) {
            const uint64_t q_desc = umma_desc_k128(smem_u32(smem + h * KH * C::QBLK)), k_desc = umma_desc_k128(smem_u32(smem + C::KV)),
                           v_desc = umma_desc_mn128(smem_u32(smem + C::KV) + KH * SX_PIECE);
            const uint32_t s_at = tmem + C::COL_S + h * 128, o_at = tmem + C::COL_O + h * D;
            int base = 0, n_qk = 0, n_pv = 0, n_q = 0;                       // pages of the share, products of this half, stretches of this half so far
            auto issue_qk = [&](int page) {                                  // page: counted over the whole share
                const int s = page % C::STAGES, buf = n_qk & 1;
                ok = mbar_wait_limited(&kv_full[s], page / C::STAGES & 1, &dead);
                if (!ok) return;
                ++n_qk;
                tc_fence_after();
                const uint64_t b = k_desc + (uint64_t)(s * (C::TILE >> 4));
#pragma unroll
                for (int kh = 0; kh < KH; ++kh)
#pragma unroll
                    for (int k = 0; k < 4; ++k) umma_bf16(s_at + buf * 64, q_desc + kh * (C::QBLK >> 4) + 2 * k, b + kh * (SX_PIECE >> 4) + 2 * k, idesc_qk, (kh | k) != 0);
                umma_commit(&s_full[h][buf]);
            };
            auto issue_pv = [&](int page, bool first, bool alone) {
                const int s = page % C::STAGES, buf = n_pv & 1;
                ok = mbar_wait_limited(&p_full[h][buf], n_pv >> 1 & 1, &dead);
                if (!ok) return;
                ++n_pv;
                tc_fence_after();
                const uint64_t b = v_desc + (uint64_t)(s * (C::TILE >> 4));
#pragma unroll
                for (int k = 0; k < kKvTile / 16; ++k) umma_f16_ts(o_at, s_at + buf * 64 + 8 * k, b + k * (2048 >> 4), idesc_pv, k != 0 || !first);
                umma_commit(&pv_done[h][buf]);
                umma_commit(&kv_empty[s]);
                if (alone) umma_commit(&kv_empty[s]);                        // the other half has no use for this page
            };
#pragma unroll 1
            while (w.next(p)) {
                const int mine = w.of_half(h);
                auto page_of = [&](int i) { return base + (w.few ? h + 2 * i : i); };      // page i of this half
                if (ok && mine) {
                    ok = mbar_wait_limited(&q_full[h], n_q++ & 1, &dead);
                    tc_fence_after();
                    // Scores run two pages ahead, issued behind the product that reads the probabilities in their buffer
#pragma unroll 1
                    for (int i = -2; ok && i < mine; ++i) {
                        if (i >= 0) issue_pv(page_of(i), i == 0, w.few);
                        if (ok && i + 2 < mine) issue_qk(page_of(i + 2));
                    }
                }
                base += w.pages;
            }
            umma_commit(&drained[h]);                                        // nothing may still run in tensor memory when it is given back, whoever gave up
#pragma unroll 1
            for (int k = 0; k < kWaitLimit && !mbar_try_wait(&drained[h], 0); ++k) {}
        }
        __syncwarp();
    } else if (warp >= 4) {
        // ---------------- softmax: one thread a row
        const int st = tid - 128, h = (warp - 4) >> 2;
        const int row = st & 127;                                            // lane of tensor memory: warp % 4 is the quarter that a warp may read
        const int tok = row / p.G;
        const uint32_t lanes = tmem + ((uint32_t)(row & 96) << 16);
        const uint32_t s_at0 = lanes + C::COL_S + h * 128, o_at = lanes + C::COL_O + h * D;
        int base = 0, cnt = 0;                                               // pages of the share, pages of this half so far
        auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_limited(bar, parity, &dead)); };
#pragma unroll 1
        while (w.next(p)) {
            const int mine = w.of_half(h);
            const int tok0 = w.few ? 0 : h * p.th;                           // of the tile
            const bool valid = tok < p.th && tok0 + tok < w.n;
            const int q0 = w.w.seq0 + w.tile * 2 * p.th + tok0;
            if (mine) {
                // the queries, 16 bytes at a time, zeros for rows without one (the products that read the last stretch's have retired: their scores were here)
                constexpr int CH = D / 8;
#pragma unroll 4
                for (int k = row; k < kSharedRows * CH; k += kSharedRows) {
                    const int c = k % CH, r = k / CH, tk = r / p.G, head = r - tk * p.G;
                    const bool on = tk < p.th && tok0 + tk < w.n;
                    const __half* from = p.q + ((size_t)(q0 + (on ? tk : 0)) * p.nq + (size_t)w.h * p.G + (on ? head : 0)) * D + c * 8;
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
                ok = ok && wait(&s_full[h][buf], cnt >> 1 & 1);
                if (!ok) break;
                tc_fence_after();
                uint32_t sr[64];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld16_nowait(s_at0 + buf * 64 + 16 * c, sr + 16 * c);
                const int seen = tokens_s[stage];                            // (written ahead of the copy that the scores came of)
                tmem_arrived<64>(sr);
                if (seen < kKvTile) {
#pragma unroll
                    for (int c = 0; c < 64; ++c) sr[c] = c < seen ? sr[c] : 0xff800000u;
                    // values behind the end may be anything, and 0 * infinity is not 0.  (Both halves may write here: zeros.)
                    ok = wait(&kv_full[stage], page / C::STAGES & 1);
                    if (!ok) break;
                    uint8_t* v = smem + C::KV + stage * C::TILE + KH * SX_PIECE;
#pragma unroll 1
                    for (int u = row; u < (kKvTile - seen) * 8 * KH; u += kSharedRows) {
                        const int kh = u / ((kKvTile - seen) * 8), x = u % ((kKvTile - seen) * 8);
                        *reinterpret_cast<uint4*>(v + kh * SX_PIECE + seen * 128 + x * 16) = make_uint4(0u, 0u, 0u, 0u);
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
            const size_t at = shared_row(w.w, w.h, w.tile * 2 * p.th + tok0, p.nq, p.G) + (size_t)2 * kSharedRows * blockIdx.x + row;
            float z = 1.f, zo = 0.f, m = m_ref, l = l_run;
            if (w.few) {                                                     // the halves' results as one: each half puts half of the dims together
                ml_s[st] = make_float2(m_ref, l_run);
                tc_fence_before();
                asm volatile("bar.sync 1, %0;" ::"n"(SX_SOFT) : "memory");
                tc_fence_after();
                const float2 other = ml_s[st ^ kSharedRows];
                m = fmaxf(m_ref, other.x);
                z = m_ref == -INFINITY ? 0.f : exp2f(m_ref - m), zo = other.x == -INFINITY ? 0.f : exp2f(other.x - m);
                l = h == 0 ? l_run * z + other.y * zo : other.y * zo + l_run * z;
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
                    float4* to = reinterpret_cast<float4*>(p.rows_o + at * D + 16 * c);
#pragma unroll
                    for (int k = 0; k < 4; ++k) to[k] = make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]), __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
                }
            }
            if (valid && (!w.few || h == 0)) p.rows_ml[at] = make_float2(m, l);
            if (w.few) {                                                     // the other half has read what the next products write over
                tc_fence_before();
                asm volatile("bar.sync 1, %0;" ::"n"(SX_SOFT) : "memory");
            }
            base += w.pages;
        }
        tmem_st_wait();
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && dead) *err = 1;
    if (warp == 3) {
        tc_fence_after();
        tmem_dealloc(tmem, C::COLS);
    }
}

template <int D>
static int launch_prefix(const SharedArgs& p, cudaStream_t st) {
    using C = SharedPrefix<D>;
    static_assert(C::SMEM <= 232448 - 4096, "shared memory");
    static PerDeviceFlag attr_set;
    if (!attr_set.done()) {
        FT_CHECK_CUDA(cudaFuncSetAttribute(shared_prefix_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        attr_set.mark();
    }
    FT_CHECK_CUDA(launch_after(shared_prefix_kernel<D>, dim3(p.prefix_ctas), dim3(SX_THREADS), C::SMEM, st, p));
    return 0;
}
int launch_shared_prefix(const SharedArgs& p, int d, cudaStream_t st) { return d == 64 ? launch_prefix<64>(p, st) : launch_prefix<128>(p, st); }

int shared_prefix_waits(int* out) {
    FT_CHECK_CUDA(cudaMemcpyFromSymbol(out, g_shared_prefix_waits, sizeof(*out)));
    return 0;
}

}  // namespace ft
