// Own part of attention over shared prefixes (shared.cuh), and the plan of both parts.
//
// What bounds the own part is the cache's bytes, so the list of all (sequence, key head, step) is cut into equal shares, one for each of two CTAs per SM.  In a CTA one
// warp copies pages (keys and values of a head lie side by side: one copy) into a ring of shared memory and the others take whole pages in turn.  A (sequence, head) that
// several CTAs have parts of is put together by the last of them to arrive, in the order of the parts, and with the prefix's results behind them.
#include "common.cuh"
#include "ft_internal.h"
#include "shared.cuh"

namespace ft {

__device__ int g_shared_decode_waits;            // 1: a wait ran out on this device (ft_attn_shared_waits)

// ------------------------------------------------------------------ plan
constexpr int SP_THREADS = 1024;

__device__ __forceinline__ int plan_before(int mine, int* warp_s, int& all) {          // exclusive sum over the block
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += up;
    }
    __syncthreads();
    if (lane == 31) warp_s[warp] = x;
    __syncthreads();
    int w = warp_s[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += up;
    }
    all = __shfl_sync(0xffffffffu, w, 31);
    const int ahead = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
    return x - mine + (warp ? ahead : 0);
}

__global__ void __launch_bounds__(SP_THREADS)
shared_plan_kernel(const __grid_constant__ SharedArgs p) {
    pdl_wait();
    __shared__ int warp_s[32];
    const int tid = threadIdx.x;
    const int reach = p.max_pages * kKvTile;
    auto row_of = [&](int b) {
        const int slot = p.req_slot ? p.req_slot[b] : b;
        return slot >= 0 && slot < p.table_rows ? slot : -1;
    };
    for (int i = tid; i < p.own_ctas; i += SP_THREADS) p.counters[i] = 0;

    // ---- groups.  A list that does not grow, or leaves the batch, shares nothing
    bool grows = true;
    for (int g = tid; g < p.n_groups; g += SP_THREADS) grows = grows && p.group_start[g] >= 0 && p.group_start[g] <= p.group_start[g + 1] && p.group_start[g + 1] <= p.B;
    grows = __syncthreads_and(grows);
    auto shared_of = [&](int g) { return max(0, min(p.shared_lens[g], reach)); };
    auto pays = [&](int g) { return p.group_start[g + 1] - p.group_start[g] >= 2 && shared_of(g) >= 2 * kKvTile; };
    {
        const int chunk = (p.n_groups + SP_THREADS - 1) / SP_THREADS, g0 = min(p.n_groups, tid * chunk), g1 = min(p.n_groups, g0 + chunk);
        int mine = 0, total;
        for (int g = g0; g < g1; ++g)
            if (grows && pays(g)) mine += p.nkv * shared_head_steps(p.group_start[g + 1] - p.group_start[g], p.th, (shared_of(g) + kKvTile - 1) / kKvTile);
        int base = plan_before(mine, warp_s, total);
        const int per = (int)((unsigned)(total + p.prefix_ctas - 1) / (unsigned)p.prefix_ctas);
        if (tid == 0) p.head->prefix_total = total, p.head->prefix_per = per;
        for (int g = g0; g < g1; ++g) {
            SharedGroup w{base, grows ? p.group_start[g] : 0, grows ? p.group_start[g + 1] - p.group_start[g] : 0, 0, 0, -1, 0, 0};
            if (grows && pays(g)) {
                w.tokens = shared_of(g);
                w.pages = (w.tokens + kKvTile - 1) / kKvTile;
                w.row = row_of(w.seq0);
                const int n = p.nkv * shared_head_steps(w.size, p.th, w.pages);
                for (int c = (int)((unsigned)(base + per - 1) / (unsigned)per); c < p.prefix_ctas && c * per < base + n; ++c) p.prefix_from[c] = g;
                base += n;
            }
            p.groups[g] = w;
        }
    }
    __syncthreads();

    // ---- sequences
    const int chunk = (p.B + SP_THREADS - 1) / SP_THREADS, b0 = min(p.B, tid * chunk), b1 = min(p.B, b0 + chunk);
    int mine = 0, most = 0, total;
    for (int b = b0; b < b1; ++b) {
        SharedSeq s{max(0, min(p.ctx_lens[b], reach)), 0, 0, -1, -1, row_of(b), 0, 0};
        if (grows && p.n_groups > 0) {
            int lo = 0, hi = p.n_groups - 1;                                // the last group that begins at or before b: those without queries begin where the next one does
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (p.group_start[mid] <= b) lo = mid; else hi = mid - 1;
            }
            const int start = p.group_start[lo];
            if (start <= b && b < p.group_start[lo + 1]) {
                s.begin = shared_of(lo);
                s.row_lead = row_of(start);
                if (p.groups[lo].pages > 0 && s.ctx >= s.begin) s.group = lo;
                else s.lead = (min(s.begin, s.ctx) + kKvTile - 1) / kKvTile;
            }
        }
        const int own = s.ctx > s.begin ? (s.ctx + kKvTile - 1) / kKvTile - s.begin / kKvTile : 0;
        s.steps = max(1, s.lead + own);
        mine += s.steps;
        most = max(most, s.steps);
        p.seqs[b] = s;
    }
    int first = plan_before(mine, warp_s, total);
    most = __reduce_max_sync(0xffffffffu, most);
    __syncthreads();
    if ((tid & 31) == 0) warp_s[tid >> 5] = most;
    __syncthreads();
    for (int w = 0; w < 32; ++w) most = max(most, warp_s[w]);
    total *= p.nkv;
    const int per = (int)((unsigned)(total + p.own_ctas - 1) / (unsigned)p.own_ctas);
    const int whole = 0;
    if (tid == 0) p.head->own_total = total, p.head->own_per = per, p.head->own_whole = whole;
    for (int b = b0; b < b1; ++b) {
        const int n = p.seqs[b].steps, at = first * p.nkv, end = (first + n) * p.nkv;
        p.seqs[b].first = first;
        for (int c = (int)((unsigned)(at + per - 1) / (unsigned)per); c < p.own_ctas && c * per < end; ++c) p.own_from[c] = b;
        first += n;
    }
}

// ------------------------------------------------------------------ own part
template <int D>
struct SharedDecode {
    static constexpr int WARPS = D == 64 ? 6 : 3;                            // that compute; one more copies
    static constexpr int STAGES = WARPS;                                     // (a stage is always the same warp's: another one's page in it would show it the wrong phase)
    static constexpr int THREADS = (WARPS + 1) * 32;
    static constexpr int SLAB = kKvTile * D * 2, TILE = 2 * SLAB;
    static constexpr int REC = D + 2;                                        // O[D], m, l
    static constexpr int BARS = STAGES * TILE;
    static constexpr int TOKENS = BARS + 2 * STAGES * 8;
    static constexpr int MERGE = (TOKENS + STAGES * 8 + 15) / 16 * 16;
    static constexpr int SMEM = MERGE + WARPS * kSharedGroup * REC * 4;
    static constexpr size_t PART = (size_t)kSharedGroup * REC;
    static_assert(PART % 4 == 0, "parts on 16 bytes");
};

// A warp's state of one (sequence, key head): S[token][query] = K Q^T with 16 tokens in the rows of mma.sync; the probabilities, transposed 8 x 8 at a time, are the other
// operand of O^T[dim][query] = V^T P^T, where all 16 rows are dims.
template <int D>
struct SharedQuery {
    uint32_t q[D / 16][2];
    float o[D / 16][4];                  // O^T: dims 16 i + g (+ 8), queries 2 tq (+ 1) at [i][2 * (upper) + (query & 1)]
    float m[2], l[2];                    // of queries 2 tq (+ 1): reference, this lane's tokens' sum

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
    }
    __device__ __forceinline__ void load_query(const __half* row, int tq) {  // row: query head g of the group, or null
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            q[ks][0] = row ? *reinterpret_cast<const uint32_t*>(row + ks * 16 + 2 * tq) : 0u;
            q[ks][1] = row ? *reinterpret_cast<const uint32_t*>(row + ks * 16 + 8 + 2 * tq) : 0u;
        }
    }
    // tokens lo .. hi - 1 of the page at `tile` (an address in shared memory); its hidden values are zeros
    __device__ __forceinline__ void page(uint32_t tile, int lo, int hi, float scale_log2, int lane) {
        const int g = lane >> 2;
        float s[4][4], most[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            s[b][0] = s[b][1] = s[b][2] = s[b][3] = 0.f;
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
                uint32_t a0, a1, a2, a3;
                ldmatrix_x4(tile + kv_swizzled_chunk<D>(16 * b + (lane & 15), 2 * ks + (lane >> 4)), a0, a1, a2, a3);
                mma_f16_16816(s[b], a0, a1, a2, a3, q[ks][0], q[ks][1]);
            }
        }
        if (lo > 0 || hi < kKvTile) {
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int t = 16 * b + 8 * (e >> 1) + g;
                    s[b][e] = t >= lo && t < hi ? s[b][e] : -INFINITY;
                }
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            most[0] = fmaxf(most[0], fmaxf(s[b][0], s[b][2]));
            most[1] = fmaxf(most[1], fmaxf(s[b][1], s[b][3]));
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) most[e] = fmaxf(most[e], __shfl_xor_sync(0xffffffffu, most[e], x));
            most[e] *= scale_log2;
        }
        if (__any_sync(0xffffffffu, most[0] > m[0] + kSharedGrow || most[1] > m[1] + kSharedGrow)) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
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
        for (int b = 0; b < 4; ++b) {
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
            for (int i = 0; i < D / 16; ++i) {
                uint32_t a0, a1, a2, a3;
                ldmatrix_x4_trans(tile + kKvTile * D * 2 + kv_swizzled_chunk<D>(16 * b + (lane & 7) + (lane >> 4) * 8, 2 * i + (lane >> 3 & 1)), a0, a1, a2, a3);
                mma_f16_16816(o[i], a0, a1, a2, a3, pb[0], pb[1]);
            }
        }
    }
    // the warp's state as a record of eight query heads: [query][D | m | l]
    __device__ __forceinline__ void store(float* rec, int lane) {
        const int g = lane >> 2, tq = lane & 3;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float sum = l[e];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            float* at = rec + (size_t)(2 * tq + e) * (D + 2);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) at[16 * i + g] = o[i][e], at[16 * i + 8 + g] = o[i][2 + e];
            if (g == 0) at[D] = m[e], at[D + 1] = sum;
        }
    }
};

template <int D>
__global__ void __launch_bounds__(SharedDecode<D>::THREADS, 2)
shared_decode_kernel(const __grid_constant__ SharedArgs p) {
    pdl_wait();
    using C = SharedDecode<D>;
    extern __shared__ __align__(128) uint8_t smem[];
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BARS);
    uint64_t* empty = full + C::STAGES;
    int2* tokens = reinterpret_cast<int2*>(smem + C::TOKENS);                // visible ones of the page in each stage; none: nothing was copied
    float* merge = reinterpret_cast<float*>(smem + C::MERGE);
    __shared__ int s_last;
    __shared__ volatile int dead;
    int* const err = &g_shared_decode_waits;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2;
    const int G = p.G;
    if (tid == 0) {
        for (int s = 0; s < C::STAGES; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
        fence_mbar_init();
        dead = 0;
    }
    __syncthreads();
    const int total = p.head->own_total, per = p.head->own_per;
    int f = min(per * (int)blockIdx.x, total);
    const int f_end = min(f + per, total);
    if (f >= f_end) return;
    int b = p.own_from[blockIdx.x];
    SharedSeq s = p.seqs[b];
    int h, t;
    {
        const unsigned rest = f - s.first * p.nkv;
        h = (int)(rest / (unsigned)s.steps);
        t = (int)(rest - (unsigned)h * s.steps);
    }
    // the next stretch of this share that lies in one (sequence, head): its steps t0 .. t1 - 1
    int t0, t1;
    auto next = [&]() {
        if (f >= f_end) return false;
        if (t >= s.steps) {
            t = 0;
            if (++h == p.nkv) {
                h = 0;
                s = p.seqs[++b];
            }
        }
        const int take = min(f_end - f, s.steps - t);
        t0 = t;
        t1 = t + take;
        t = t1;
        f += take;
        return true;
    };

    if (warp == C::WARPS) {
        // ---------------- copies: one page a step
        const uint64_t pol = policy_evict_first();                           // every byte is read once
        int it = 0, asked = 0;
        bool ok = true;
        while (next()) {
            for (int p0 = t0; p0 < t1; p0 += 32) {
                const int step = p0 + lane;
                const bool lead = step < s.lead;
                const int tile = lead ? step : s.begin / kKvTile + step - s.lead, row = lead ? s.row_lead : s.row_own;
                const int from = max(0, (lead ? 0 : s.begin) - tile * kKvTile), to = min(kKvTile, (lead ? min(s.begin, s.ctx) : s.ctx) - tile * kKvTile);
                int my_page = -1;
                if (step < t1 && from < to && row >= 0) my_page = p.page_table[(size_t)row * p.max_pages + tile];
                if (my_page >= p.num_pages) my_page = -1;
                const int n = min(32, t1 - p0);
                for (int i = 0; i < n; ++i, ++it) {
                    const int page = __shfl_sync(0xffffffffu, my_page, i);
                    const int2 seen = make_int2(__shfl_sync(0xffffffffu, from, i), __shfl_sync(0xffffffffu, to, i));
                    if (lane == 0 && ok) {
                        const int st = it % C::STAGES;
                        ok = mbar_wait_limited(&empty[st], (it / C::STAGES & 1) ^ 1, &dead);
                        if (!ok) continue;
                        asked = it + 1;
                        tokens[st] = page >= 0 ? seen : make_int2(0, 0);
                        if (page >= 0) {
                            mbar_expect_tx(&full[st], C::TILE);
                            tma_bulk_g2s(smem + st * C::TILE, p.cache + ((size_t)page * p.nkv + h) * C::TILE, C::TILE, &full[st], pol);
                        } else {
                            mbar_arrive(&full[st]);
                        }
                    }
                }
            }
        }
        if (lane == 0) {
            if (!ok) *err = 1;
            for (int i = max(0, asked - C::STAGES); i < asked; ++i)          // nothing may still be on its way into this CTA's memory when it ends
                for (int k = 0; k < kWaitLimit && !mbar_try_wait(&full[i % C::STAGES], i / C::STAGES & 1); ++k) {}
        }
        return;
    }

    // ---------------- the others: page it of the share is warp it % WARPS's
    int it = 0;
    bool ok = true;                                                          // false from the first wait on that ran out
    while (next()) {
        SharedQuery<D> a;
        a.clear();
        a.load_query(g < G ? p.q + ((size_t)b * p.nq + (size_t)h * G + g) * D : nullptr, lane & 3);
        for (int i = it + (warp - it % C::WARPS + C::WARPS) % C::WARPS; ok && i < it + t1 - t0; i += C::WARPS) {
            const int st = i % C::STAGES;
            ok = __all_sync(0xffffffffu, mbar_wait_limited(&full[st], i / C::STAGES & 1, &dead));
            if (!ok) break;
            const int2 seen = tokens[st];
            if (seen.x < seen.y) {
                uint8_t* tile = smem + st * C::TILE;
                if (seen.x > 0 || seen.y < kKvTile) {                        // hidden values may be anything: 0 * infinity is none
                    const int hidden = seen.x + kKvTile - seen.y;
                    for (int u = lane; u < hidden * (D / 8); u += 32) {
                        const int k = u / (D / 8), c = u % (D / 8), tok = k < seen.x ? k : seen.y + k - seen.x;
                        *reinterpret_cast<uint4*>(tile + C::SLAB + kv_swizzled_chunk<D>(tok, c)) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_proxy_async();                                     // ahead of the next copy into this stage
                    __syncwarp();
                }
                a.page(smem_u32(tile), seen.x, seen.y, p.scale_log2, lane);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
        }
        it += t1 - t0;
        if (!ok) {                                                           // NaN for all that this (sequence, head) says
            *err = 1;
            a.m[0] = a.m[1] = 0.f;
            a.l[0] = a.l[1] = NAN;
        }
        const bool all = t0 == 0 && t1 == s.steps;
        const int first = (s.first * p.nkv) + h * s.steps;                   // of the (sequence, head) in the list
        const int c0 = all ? 0 : (int)((unsigned)first / (unsigned)per), c1 = all ? 0 : (int)((unsigned)(first + s.steps - 1) / (unsigned)per);
        float* part = p.own_parts + (2 * (size_t)blockIdx.x + (t0 == 0)) * C::PART;          // [head][D], then (m, l) of the heads
        const size_t row = ((size_t)b * p.nq + (size_t)h * G) * D;
        a.store(merge + (size_t)warp * C::PART, lane);
        // the warps' records as one, to the output or to this CTA's part
        auto reduce = [&](bool final) {
            asm volatile("bar.sync 1, %0;" ::"n"(C::WARPS * 32) : "memory");
            for (int e = 2 * tid; e < G * D; e += 2 * C::WARPS * 32) {
                const int hg = e / D, dim = e % D;
                const float* rec = merge + (size_t)hg * C::REC;
                float m[C::WARPS], M = -INFINITY, L = 0.f, x = 0.f, y = 0.f;
#pragma unroll
                for (int w = 0; w < C::WARPS; ++w) m[w] = rec[w * C::PART + D], M = fmaxf(M, m[w]);
#pragma unroll
                for (int w = 0; w < C::WARPS; ++w) {
                    const float z = m[w] == -INFINITY ? 0.f : exp2f(m[w] - M);
                    const float2 o = *reinterpret_cast<const float2*>(rec + w * C::PART + dim);
                    L = fmaf(rec[w * C::PART + D + 1], z, L);
                    x = fmaf(o.x, z, x);
                    y = fmaf(o.y, z, y);
                }
                if (final) {                                                 // a query without a visible key: zeros
                    const float r = L == 0.f ? 0.f : 1.f / L;
                    x *= r, y *= r;
                    const uint32_t hi = pack_bf16(x, y);
                    *reinterpret_cast<uint32_t*>(p.out + row + e) = hi;
                    if (p.out_lo) *reinterpret_cast<uint32_t*>(p.out_lo + row + e) = pack_bf16(x - bf16_lo(hi), y - bf16_hi(hi));
                } else {
                    *reinterpret_cast<float2*>(part + e) = make_float2(x, y);
                    if (dim == 0) *reinterpret_cast<float2*>(part + kSharedGroup * D + 2 * hg) = make_float2(M, L);
                }
            }
            asm volatile("bar.sync 1, %0;" ::"n"(C::WARPS * 32) : "memory");
        };
        if (!all) {
            reduce(false);
            if (tid == 0) {
                __threadfence();
                s_last = atomicAdd(&p.counters[c0], 1) == c1 - c0;
            }
            asm volatile("bar.sync 1, %0;" ::"n"(C::WARPS * 32) : "memory");
            if (!s_last) continue;
            __threadfence();
        }
        if (!all || s.group >= 0) {
            // each warp takes every WARPS-th part, in their order, and of the prefix's results, and then they are records of the warps once more
            float* mine = merge + (size_t)warp * C::PART;
            int x0 = 0, x1 = -1;                                             // CTAs that have results of the prefix's unit
            size_t row0 = 0;
            if (s.group >= 0) {
                const SharedGroup w = p.groups[s.group];
                const int i = b - w.seq0, tile = i / (2 * p.th), n = min(2 * p.th, w.size - tile * 2 * p.th), per_x = p.head->prefix_per;
                const int from = w.base + h * shared_head_steps(w.size, p.th, w.pages) + tile * (w.pages + kSharedStart);
                x0 = (int)((unsigned)from / (unsigned)per_x);
                x1 = (int)((unsigned)(from + shared_steps(n, p.th, w.pages) - 1) / (unsigned)per_x);
                row0 = shared_row(w, h, i, p.nq, G);
            }
            __syncwarp();
#pragma unroll 1
            for (int eb = 0; eb < G * D; eb += 128) {
                const int e0 = min(eb + 4 * lane, G * D - 4), hg = e0 / D, dim = e0 % D;
                float* rec = mine + hg * C::REC;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                float M = -INFINITY, L = 0.f;
                auto add = [&](const float4& o, const float2& ml) {
                    const float Mn = fmaxf(M, ml.x);
                    const float keep = M == -INFINITY ? 0.f : exp2f(M - Mn), z = ml.x == -INFINITY ? 0.f : exp2f(ml.x - Mn);
                    L = fmaf(ml.y, z, L * keep);
                    acc = fma_f4(o, make_float4(z, z, z, z), make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep));
                    M = Mn;
                };
                if (all) {
                    add(make_float4(rec[dim], rec[dim + 1], rec[dim + 2], rec[dim + 3]), make_float2(rec[D], rec[D + 1]));
                } else {
#pragma unroll 2
                    for (int c = c0 + warp; c <= c1; c += C::WARPS) {
                        const float* part = p.own_parts + (2 * (size_t)c + (c == c0)) * C::PART;
                        add(__ldcg(reinterpret_cast<const float4*>(part + e0)), __ldcg(reinterpret_cast<const float2*>(part + kSharedGroup * D + 2 * hg)));
                    }
                }
#pragma unroll 2
                for (int c = x0 + warp; c <= x1; c += C::WARPS) {
                    const size_t at = row0 + (size_t)2 * kSharedRows * c + hg;
                    add(__ldcg(reinterpret_cast<const float4*>(p.rows_o + at * D + dim)), __ldcg(p.rows_ml + at));
                }
                __syncwarp();                                                // all have read what the first lane of a head writes over
                if (eb + 4 * lane < G * D) {
                    *reinterpret_cast<float2*>(rec + dim) = make_float2(acc.x, acc.y);
                    *reinterpret_cast<float2*>(rec + dim + 2) = make_float2(acc.z, acc.w);
                    if (dim == 0) *reinterpret_cast<float2*>(rec + D) = make_float2(M, L);
                }
            }
        }
        reduce(true);
    }
}

// ------------------------------------------------------------------ host
static size_t up64(size_t n) { return (n + 63) / 64 * 64; }
struct SharedLayout { size_t head, seqs, groups, own_from, prefix_from, counters, own_parts, rows_o, rows_ml, bytes; };
static SharedLayout shared_layout(int B, int n_groups, int nq, int d) {
    const size_t sms = device_sms(), rows = (size_t)B * nq + 2 * kSharedRows * sms;
    SharedLayout l;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += up64(bytes); return here; };
    l.head = take(sizeof(SharedHead));
    l.seqs = take(B * sizeof(SharedSeq));
    l.groups = take(n_groups * sizeof(SharedGroup));
    l.own_from = take(2 * sms * 4);
    l.prefix_from = take(sms * 4);
    l.counters = take(2 * sms * 4);
    l.own_parts = take(2 * 2 * sms * kSharedGroup * (d + 2) * 4);
    l.rows_o = take(n_groups ? rows * d * 4 : 0);
    l.rows_ml = take(n_groups ? rows * 8 : 0);
    l.bytes = at;
    return l;
}

template <int D>
static int launch_shared(const SharedArgs& p, cudaStream_t st) {
    using C = SharedDecode<D>;
    static PerDeviceFlag attr_set;
    if (!attr_set.done()) {
        FT_CHECK_CUDA(cudaFuncSetAttribute(shared_decode_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        attr_set.mark();
    }
    FT_CHECK_CUDA(launch_after(shared_plan_kernel, dim3(1), dim3(SP_THREADS), 0, st, p));
    if (p.n_groups)
        if (int r = launch_shared_prefix(p, D, st)) return r;
    FT_CHECK_CUDA(launch_after(shared_decode_kernel<D>, dim3(p.own_ctas), dim3(C::THREADS), C::SMEM, st, p));
    return 0;
}

}  // namespace ft

extern "C" long long ft_attn_decode_shared_scratch_bytes(int B, int n_groups, int nq, int d) {
    FT_REQUIRE(d == 64 || d == 128, "ft_attn_decode_shared_scratch_bytes: head_dim %d not supported (64 or 128)", d);
    FT_REQUIRE(B >= 0 && n_groups >= 0 && nq >= 1 && (double)B * nq * d <= INT32_MAX, "ft_attn_decode_shared_scratch_bytes: bad sizes B=%d nq=%d groups=%d", B, nq, n_groups);
    return (long long)ft::shared_layout(B, n_groups, nq, d).bytes;
}

extern "C" int ft_attn_shared_waits(void) {
    int n = 0, m = 0;
    FT_CHECK_CUDA(cudaDeviceSynchronize());                                  // the copies below wait for the default stream only
    FT_CHECK_CUDA(cudaMemcpyFromSymbol(&n, ft::g_shared_decode_waits, sizeof(n)));
    if (int r = ft::shared_prefix_waits(&m)) return r;
    return n | m;
}

extern "C" int ft_attn_decode_shared(const void* q, const void* kv_layer, int num_pages, const int* page_table, int table_rows, int max_pages, const int* req_slot,
                                     const int* ctx_lens, const int* group_start, const int* shared_lens, int n_groups, void* out, void* out_lo, void* scratch, int B, int nq,
                                     int nkv, int d, void* stream) {
    using namespace ft;
    FT_REQUIRE(d == 64 || d == 128, "ft_attn_decode_shared: head_dim %d not supported (64 or 128)", d);
    FT_REQUIRE(nq >= 1 && nkv >= 1 && nq % nkv == 0 && nq / nkv <= kSharedGroup, "ft_attn_decode_shared: GQA group %d/%d not supported", nq, nkv);
    const int G = nq / nkv, th = kSharedRows / G;
    FT_REQUIRE(B >= 0 && n_groups >= 0 && num_pages >= 0 && table_rows >= 0 && max_pages >= 0 && max_pages < INT32_MAX / kKvTile && (double)B * nq * d <= INT32_MAX,
               "ft_attn_decode_shared: bad sizes B=%d nq=%d groups=%d table %d x %d, %d pages", B, nq, n_groups, table_rows, max_pages, num_pages);
    // both lists: at most so many units of at most so many steps, and what the shares are rounded up by
    FT_REQUIRE(((double)B + 1) * nkv * (2.0 * max_pages + 2) + 4096 <= INT32_MAX && ((double)B / (2 * th) + n_groups) * nkv * (max_pages + kSharedStart + 1.0) + 4096 <= INT32_MAX,
               "ft_attn_decode_shared: %d sequences of %d pages in %d groups are more than one call takes", B, max_pages, n_groups);
    if (B == 0) return 0;
    FT_REQUIRE(q && ctx_lens && out && scratch && (n_groups == 0 || (group_start && shared_lens)) && (page_table || table_rows == 0 || max_pages == 0) && (kv_layer || num_pages == 0),
               "ft_attn_decode_shared: null argument");
    FT_REQUIRE(((uintptr_t)q | (uintptr_t)kv_layer | (uintptr_t)out | (uintptr_t)out_lo | (uintptr_t)scratch) % 16 == 0, "ft_attn_decode_shared: tensors on 16 bytes");
    const SharedLayout l = shared_layout(B, n_groups, nq, d);
    uint8_t* w = (uint8_t*)scratch;
    const int sms = device_sms();
    SharedArgs p{(const __half*)q, (const uint8_t*)kv_layer, page_table, req_slot, ctx_lens, group_start, shared_lens, (__nv_bfloat16*)out, (__nv_bfloat16*)out_lo,
                 (SharedHead*)(w + l.head), (SharedSeq*)(w + l.seqs), (SharedGroup*)(w + l.groups), (int*)(w + l.own_from), (int*)(w + l.prefix_from), (int*)(w + l.counters),
                 (float*)(w + l.own_parts), (float*)(w + l.rows_o), (float2*)(w + l.rows_ml), B, n_groups, num_pages, table_rows, max_pages, nq, nkv, G, th, 2 * sms, sms,
                 kSharedLog2E / sqrtf((float)d)};
    return d == 64 ? launch_shared<64>(p, (cudaStream_t)stream) : launch_shared<128>(p, (cudaStream_t)stream);
}
