// Attention of one query token per sequence over the 8-bit KV cache (kv8.cuh): out[b][h] = sum_j softmax_j(q . k_j / sqrt(D)) v_j, j < ctx_lens[b].
//
// What bounds it is the cache's bytes, so the list of all (sequence, key head, page) is cut into equal shares, one for each of two CTAs per SM, however ragged
// the batch is.  In a CTA one warp copies records (a page of a head: codes and scales in one piece) into a ring of shared memory, and the others take whole
// records in turn (Kv8Query in kv8.cuh).  A (sequence, head) that several CTAs have parts of is put together by the last of them to arrive, in the order of the
// parts.  Where there is a CTA for every (sequence, head) and none of them is long, each CTA takes a whole one instead: no parts, nothing to put together.
//
// Nothing is planned ahead of the kernel: every CTA adds up the sequences' pages itself (one read of ctx_lens).  What the arrival counters need, zeros, is
// written by a kernel of its own ahead of this one.
//
// 64 sequences of about 2000 keys, 32 heads over 8 of 64 (133 MB): 32.5 us, 4.1 TB/s.  Some 11 us of that are start (lengths, page number and record are read one after the other)
// and end (the parts): from 4096 to 8192 keys each, 539 MB in 93 us, more bytes stream at 6.6 TB/s (7.0 at heads of 128).  Three of 30011 .. 9377 keys, heads of 128: 28.7 us.  On the
// way, for the two: shares with the queries in the rows of the first product 36 / 38, the tokens in them 32 / 34, and then all warps putting parts together 32 / 30.
#include <atomic>

#include "common.cuh"
#include "ft_internal.h"
#include "kv8.cuh"

namespace ft {

constexpr int K8D_GROUP = 8;                     // query heads a key head at most
constexpr int K8D_WHOLE_PAGES = 16;              // with page tables no wider than this, and a CTA for each (sequence, head), there are never parts
                                                 // (32 sequences of 1000 keys, 8 heads of 128: 14.7 us whole, 20.0 in shares; 8 of 77, heads of 64, 4.5 / 7.7, counters' zeros included)
constexpr float K8D_LOG2E = 1.4426950408889634f;

__device__ int g_kv8_decode_waits;               // 1: a wait ran out on this device (ft_kv8_waits)

template <int D>
struct K8Decode {
    static constexpr int WARPS = D == 64 ? 6 : 5;                            // that compute; one more copies
    static constexpr int STAGES = D == 64 ? 12 : 5;                          // 99 / 82 KB on their way
    // A stage is always the same warp's: a warp that another one's page passes in the same stage would take the phase before its own for its own
    static_assert(STAGES % WARPS == 0, "a stage belongs to one warp");
    static constexpr int THREADS = (WARPS + 1) * 32;
    static constexpr int REC = D + 2;                                        // O[D], m, l
    static constexpr int BARS = STAGES * Kv8<D>::REC;                        // byte offsets in shared memory
    static constexpr int TOKENS = BARS + 2 * STAGES * 8;
    static constexpr int MERGE = (TOKENS + STAGES * 4 + 15) / 16 * 16;
    static constexpr int SMEM = MERGE + WARPS * K8D_GROUP * REC * 4;
    static constexpr size_t PART = (size_t)K8D_GROUP * REC;                  // floats of a record, and of a part
    static_assert(PART % 4 == 0, "parts on 16 bytes");
};

__global__ void kv8_decode_zero_kernel(int* counters, int n) {
    pdl_wait();
    for (int i = threadIdx.x; i < n; i += blockDim.x) counters[i] = 0;
}

template <int D>
__global__ void __launch_bounds__(K8Decode<D>::THREADS, 2)
kv8_decode_kernel(const __half* __restrict__ q, const uint8_t* __restrict__ cache, int num_pages, const int* __restrict__ page_table, int max_pages,
                  const int* __restrict__ ctx_lens, __nv_bfloat16* __restrict__ out, __nv_bfloat16* __restrict__ out_lo, int* counters, float* parts,
                  int B, int nq, int nkv, float scale_log2, int wait_limit) {
    pdl_wait();
    using C = K8Decode<D>;
    extern __shared__ __align__(128) uint8_t smem[];
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BARS);
    uint64_t* empty = full + C::STAGES;
    int* tokens = reinterpret_cast<int*>(smem + C::TOKENS);                  // of the page in each stage; 0: a page that is not there
    float* merge = reinterpret_cast<float*>(smem + C::MERGE);
    __shared__ int s_sum[C::WARPS + 1];
    __shared__ int s_most[C::WARPS + 1], s_b, s_last;
    __shared__ int s_base;
    __shared__ volatile int dead;
    int* const err = &g_kv8_decode_waits;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tq = lane & 3;
    const int G = nq / nkv;
    if (tid == 0) {
        for (int s = 0; s < C::STAGES; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
        fence_mbar_init();
        dead = 0;
    }
    auto ctx_of = [&](int b) { return max(0, min(ctx_lens[b], max_pages * kKvTile)); };
    auto pages_of = [&](int b) { return (ctx_of(b) + kKvTile - 1) / kKvTile; };

    // ---------------- the plan: this CTA's share of the flat list [sequence][head][page]
    const int chunk = (B + C::THREADS - 1) / C::THREADS;
    const int b0 = min(B, tid * chunk), b1 = min(B, b0 + chunk);
    int mine = 0;                                                            // (the host has seen that 32 bits hold the whole list)
    int most = 0;
    for (int b = b0; b < b1; ++b) {
        const int n = pages_of(b);
        mine += n;
        most = max(most, n);
    }
    int before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += up;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 31) s_sum[warp] = before, s_most[warp] = most;
    __syncthreads();
    int total = 0;
    before -= mine;
#pragma unroll
    for (int w = 0; w <= C::WARPS; ++w) {
        if (w < warp) before += s_sum[w];
        total += s_sum[w];
        most = max(most, s_most[w]);
    }
    total *= nkv;
    const int per = (int)((unsigned)(total + gridDim.x - 1) / gridDim.x);
    const bool each = B * nkv <= (int)gridDim.x;
    const bool whole = each && (parts == nullptr || (most + C::WARPS - 1) / C::WARPS <= (per + C::WARPS - 1) / C::WARPS + 1);
    int f = min(per * (int)blockIdx.x, total), f_end = min(f + per, total);
    int b, h, t;
    if (whole) {
        b = blockIdx.x / nkv;
        if (b >= B) return;
        h = blockIdx.x % nkv;
        t = 0;
        f = 0;
        f_end = pages_of(b);
    } else {
        if (before * nkv <= f && f < (before + mine) * nkv) {
            int x = b0;
            for (int n; (before + (n = pages_of(x))) * nkv <= f; ++x) before += n;
            s_b = x;
            s_base = before;
        }
        __syncthreads();
        if (f >= f_end) f_end = f;
        b = s_b;
        const unsigned rest = f - s_base * nkv;
        const int n = f < f_end ? pages_of(b) : 1;
        h = (int)(rest / (unsigned)n);
        t = (int)(rest - (unsigned)h * n);
    }
    // a sequence without keys has no page and so no share: zeros
    auto zeros = [&](int b_, int h0, int h1) {
        for (int e = tid; e < (h1 - h0) * G * D; e += C::THREADS) {
            const size_t at = ((size_t)b_ * nq + (size_t)h0 * G) * D + e;
            out[at] = __float2bfloat16(0.f);
            if (out_lo) out_lo[at] = __float2bfloat16(0.f);
        }
    };
    if (whole) {
        if (f_end == 0) zeros(b, h, h + 1);
    } else {
        for (int i = blockIdx.x; i < B; i += gridDim.x)
            if (pages_of(i) == 0) zeros(i, 0, nkv);
    }
    if (f >= f_end) {
        return;
    }

    int n_pages = pages_of(b);
    // the next stretch of this share that lies in one (sequence, head): pages t0 .. t1 - 1
    int seg_b, seg_h, t0, t1;
    auto next = [&]() {
        if (f >= f_end) return false;
        while (t >= n_pages) {
            t = 0;
            if (++h == nkv) {
                h = 0;
                do n_pages = pages_of(++b);
                while (n_pages == 0);
            }
        }
        const int take = min(f_end - f, n_pages - t);
        seg_b = b; seg_h = h; t0 = t; t1 = t + take;
        t = t1;
        f += take;
        return true;
    };

    if (warp == C::WARPS) {
        // ---------------- copies: one record a page
        const uint64_t pol = policy_evict_first();                           // every byte is read once
        int it = 0, asked = 0;
        bool ok = true;
        while (next()) {
            const int ctx = ctx_of(seg_b);
            const int* pt = page_table + (size_t)seg_b * max_pages;
            for (int p0 = t0; p0 < t1; p0 += 32) {
                const int my_page = p0 + lane < t1 ? pt[p0 + lane] : -1;
                const int n = min(32, t1 - p0);
                for (int i = 0; i < n; ++i, ++it) {
                    const int page = __shfl_sync(0xffffffffu, my_page, i);
                    if (lane == 0 && ok) {
                        const int s = it % C::STAGES;
                        ok = kv8_mbar_wait_limited(&empty[s], (it / C::STAGES & 1) ^ 1, &dead, wait_limit);
                        if (!ok) continue;
                        asked = it + 1;
                        const bool there = page >= 0 && page < num_pages;
                        tokens[s] = there ? min(kKvTile, ctx - (p0 + i) * kKvTile) : 0;
                        if (there) {
                            mbar_expect_tx(&full[s], Kv8<D>::REC);
                            tma_bulk_g2s(smem + s * Kv8<D>::REC, cache + ((size_t)page * nkv + seg_h) * Kv8<D>::REC, Kv8<D>::REC, &full[s], pol);
                        } else {
                            mbar_arrive(&full[s]);
                        }
                    }
                }
            }
        }
        if (lane == 0) {
            if (!ok) *err = 1;
            kv8_copies_landed(full, C::STAGES, asked);                       // (those who read them may give up at any time)
        }
        return;
    }

    // ---------------- the others: page it of the share is warp it % WARPS's
    int it = 0;
    bool ok = true;                                                          // false from the first wait on that ran out
    while (next()) {
        Kv8Query<D> a;
        a.clear();
        a.load_query(g < G ? q + ((size_t)seg_b * nq + (size_t)seg_h * G + g) * D : nullptr, tq);
        for (int i = it + (warp - it % C::WARPS + C::WARPS) % C::WARPS; ok && i < it + t1 - t0; i += C::WARPS) {
            const int s = i % C::STAGES;
            ok = __all_sync(0xffffffffu, kv8_mbar_wait_limited(&full[s], i / C::STAGES & 1, &dead, wait_limit));
            if (!ok) break;
            const int n = tokens[s];
            if (n) a.page(smem + s * Kv8<D>::REC, n, scale_log2, g, tq);
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[s]);
        }
        it += t1 - t0;
        if (!ok) {                                                           // NaN for all that this (sequence, head) says
            *err = 1;
            a.m[0] = a.m[1] = 0.f;
            a.l[0] = a.l[1] = NAN;
        }
        const bool all = t0 == 0 && t1 == n_pages;
        const int first = f - t1;                                            // of the (sequence, head) in the flat list (a whole one has no parts)
        const int c0 = all ? 0 : (int)((unsigned)first / (unsigned)per), c1 = all ? 0 : (int)((unsigned)(first + n_pages - 1) / (unsigned)per);
        float* part = parts + (2 * (size_t)blockIdx.x + (t0 == 0)) * C::PART;                // [head][D], then (m, l) of the heads
        const size_t row = ((size_t)seg_b * nq + (size_t)seg_h * G) * D;
        a.store(merge + (size_t)warp * C::PART, g, tq);
        for (bool final = all;; final = true) {
            // the warps' records as one: to the output, or to this CTA's part
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
                    *reinterpret_cast<uint32_t*>(out + row + e) = hi;
                    if (out_lo) *reinterpret_cast<uint32_t*>(out_lo + row + e) = pack_bf16(x - bf16_lo(hi), y - bf16_hi(hi));
                } else {
                    *reinterpret_cast<float2*>(part + e) = make_float2(x, y);
                    if (dim == 0) *reinterpret_cast<float2*>(part + K8D_GROUP * D + 2 * hg) = make_float2(M, L);
                }
            }
            if (final) break;
            // The last CTA to deliver a part puts all of them together: each warp takes every WARPS-th part, in their order, and then they are records of the
            // warps once more.  (All threads walking all parts one after the other: 12 us at the end of three sequences of 20000 keys, 19 parts each.)
            asm volatile("bar.sync 1, %0;" ::"n"(C::WARPS * 32) : "memory");
            if (tid == 0) {
                __threadfence();
                s_last = atomicAdd(&counters[c0], 1) == c1 - c0;
            }
            asm volatile("bar.sync 1, %0;" ::"n"(C::WARPS * 32) : "memory");
            if (!s_last) break;
            __threadfence();
            float* mine = merge + (size_t)warp * C::PART;
#pragma unroll 1
            for (int e0 = 4 * lane; e0 < G * D; e0 += 512) {
                float4 acc[4];                                               // four floats each 128 further on
                float M[4], L[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f), M[k] = -INFINITY, L[k] = 0.f;
#pragma unroll 2
                for (int c = c0 + warp; c <= c1; c += C::WARPS) {
                    const float* rec = parts + (2 * (size_t)c + (c == c0)) * C::PART;
                    float4 o[4];
                    float2 ml[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int e = min(e0 + 128 * k, G * D - 4);
                        o[k] = __ldcg(reinterpret_cast<const float4*>(rec + e));
                        ml[k] = __ldcg(reinterpret_cast<const float2*>(rec + K8D_GROUP * D + 2 * (e / D)));
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float Mn = fmaxf(M[k], ml[k].x);
                        const float keep = M[k] == -INFINITY ? 0.f : exp2f(M[k] - Mn), z = ml[k].x == -INFINITY ? 0.f : exp2f(ml[k].x - Mn);
                        L[k] = fmaf(ml[k].y, z, L[k] * keep);
                        acc[k] = fma_f4(o[k], make_float4(z, z, z, z), make_float4(acc[k].x * keep, acc[k].y * keep, acc[k].z * keep, acc[k].w * keep));
                        M[k] = Mn;
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int e = e0 + 128 * k, hg = e / D, dim = e % D;
                    if (e >= G * D) continue;
                    *reinterpret_cast<float2*>(mine + hg * C::REC + dim) = make_float2(acc[k].x, acc[k].y);
                    *reinterpret_cast<float2*>(mine + hg * C::REC + dim + 2) = make_float2(acc[k].z, acc[k].w);
                    if (dim == 0) *reinterpret_cast<float2*>(mine + hg * C::REC + D) = make_float2(M[k], L[k]);
                }
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(C::WARPS * 32) : "memory");
    }
}

static std::atomic<int> g_kv8_wait_limit{kWaitLimit};
int kv8_wait_limit() { return g_kv8_wait_limit.load(std::memory_order_relaxed); }

// counters (one for each CTA that a split (sequence, head) can begin in), then two parts a CTA: of the (sequence, head) it begins in the middle of, and of the one it ends in
static int kv8_decode_ctas() { return 2 * device_sms(); }
static size_t kv8_decode_counters(int ctas) { return (size_t)(ctas + 63) / 64 * 64; }

template <int D>
static int launch_kv8_decode(const void* q, const void* cache, int num_pages, const int* page_table, int max_pages, const int* ctx_lens, void* out, void* out_lo,
                             void* scratch, int B, int nq, int nkv, cudaStream_t st) {
    using C = K8Decode<D>;
    static PerDeviceFlag attr_set;
    if (!attr_set.done()) {
        FT_CHECK_CUDA(cudaFuncSetAttribute(kv8_decode_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        attr_set.mark();
    }
    const int ctas = kv8_decode_ctas();
    const bool whole = (long long)B * nkv <= ctas && max_pages <= K8D_WHOLE_PAGES;
    FT_REQUIRE(whole || scratch, "ft_attn_decode_kv8: needs ft_attn_decode_kv8_scratch_bytes of work memory");
    int* counters = whole ? nullptr : (int*)scratch;
    float* parts = whole ? nullptr : (float*)scratch + kv8_decode_counters(ctas);
    const float scale_log2 = K8D_LOG2E / sqrtf((float)D);
    if (whole) {
        FT_CHECK_CUDA(launch_after(kv8_decode_kernel<D>, dim3(B * nkv), dim3(C::THREADS), C::SMEM, st, (const __half*)q, (const uint8_t*)cache, num_pages, page_table,
                                   max_pages, ctx_lens, (__nv_bfloat16*)out, (__nv_bfloat16*)out_lo, counters, parts, B, nq, nkv, scale_log2, kv8_wait_limit()));
        return 0;
    }
    FT_CHECK_CUDA(launch_after(kv8_decode_zero_kernel, dim3(1), dim3(128), 0, st, counters, ctas));
    FT_CHECK_CUDA(launch_after(kv8_decode_kernel<D>, dim3(ctas), dim3(C::THREADS), C::SMEM, st, (const __half*)q, (const uint8_t*)cache, num_pages, page_table,
                               max_pages, ctx_lens, (__nv_bfloat16*)out, (__nv_bfloat16*)out_lo, counters, parts, B, nq, nkv, scale_log2, kv8_wait_limit()));
    return 0;
}

}  // namespace ft

extern "C" long long ft_attn_decode_kv8_scratch_bytes(int d) {
    FT_REQUIRE(d == 64 || d == 128, "ft_attn_decode_kv8_scratch_bytes: head_dim %d not supported (64 or 128)", d);
    const int ctas = ft::kv8_decode_ctas();
    return (long long)(ft::kv8_decode_counters(ctas) + 2 * (size_t)ctas * ft::K8D_GROUP * (d + 2)) * 4;
}

extern "C" void ft_kv8_set_wait_limit(int tries) { ft::g_kv8_wait_limit = tries < 0 || tries > ft::kWaitLimit ? ft::kWaitLimit : tries; }

extern "C" int ft_kv8_waits(void) {
    int n = 0, m = 0;
    FT_CHECK_CUDA(cudaDeviceSynchronize());                                  // the copies below wait for the default stream only
    FT_CHECK_CUDA(cudaMemcpyFromSymbol(&n, ft::g_kv8_decode_waits, sizeof(n)));
    if (int r = ft::kv8_prefill_waits(&m)) return r;
    return n | m;
}

extern "C" int ft_attn_decode_kv8(const void* q, const void* kv8_layer, int num_pages, const int* page_table, int max_pages, const int* ctx_lens, void* out,
                                  void* out_lo, void* scratch, int B, int nq, int nkv, int d, void* stream) {
    using namespace ft;
    FT_REQUIRE(d == 64 || d == 128, "ft_attn_decode_kv8: head_dim %d not supported (64 or 128)", d);
    FT_REQUIRE(nq >= 1 && nkv >= 1 && nq % nkv == 0 && nq / nkv <= K8D_GROUP, "ft_attn_decode_kv8: GQA group %d/%d not supported", nq, nkv);
    FT_REQUIRE(B >= 0 && max_pages >= 0 && num_pages >= 0 && max_pages <= INT32_MAX / kKvTile && ((double)B + 1) * nkv * (max_pages + 1) + 4096 <= INT32_MAX,
               "ft_attn_decode_kv8: bad sizes B=%d nkv=%d max_pages=%d num_pages=%d", B, nkv, max_pages, num_pages);
    if (B == 0) return 0;
    FT_REQUIRE(q && ctx_lens && out && kv8_there(page_table, B, max_pages, kv8_layer, num_pages), "ft_attn_decode_kv8: null argument");
    FT_REQUIRE(((uintptr_t)q | (uintptr_t)kv8_layer | (uintptr_t)out | (uintptr_t)out_lo | (uintptr_t)scratch) % 16 == 0, "ft_attn_decode_kv8: tensors on 16 bytes");
    return d == 64 ? launch_kv8_decode<64>(q, kv8_layer, num_pages, page_table, max_pages, ctx_lens, out, out_lo, scratch, B, nq, nkv, (cudaStream_t)stream)
                   : launch_kv8_decode<128>(q, kv8_layer, num_pages, page_table, max_pages, ctx_lens, out, out_lo, scratch, B, nq, nkv, (cudaStream_t)stream);
}
