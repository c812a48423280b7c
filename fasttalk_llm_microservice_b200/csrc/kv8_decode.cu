// Attention of one query token per sequence over the 8-bit KV cache (kv8.cuh): out[b][h] = sum_j softmax_j(q . k_j / sqrt(D)) v_j, j < ctx_lens[b].
//
// One CTA per (sequence, key head); its warps take the pages in turn and their results are put together at the end.
#include "common.cuh"
#include "ft_internal.h"
#include "kv8.cuh"

namespace ft {

constexpr int K8D_WARPS = 8, K8D_GROUP = 8;      // warps a CTA; query heads a key head at most
constexpr float K8D_LOG2E = 1.4426950408889634f;

template <int D>
__global__ void __launch_bounds__(K8D_WARPS * 32)
kv8_decode_kernel(const __half* __restrict__ q, const uint8_t* __restrict__ cache, int num_pages, const int* __restrict__ page_table, int max_pages,
                  const int* __restrict__ ctx_lens, __nv_bfloat16* __restrict__ out, __nv_bfloat16* __restrict__ out_lo, int nq, int nkv, float scale_log2) {
    __shared__ float rec_s[K8D_WARPS][K8D_GROUP][D + 2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
    const int b = blockIdx.x / nkv, kvh = blockIdx.x % nkv, G = nq / nkv;
    const int ctx = min(ctx_lens[b], max_pages * kKvTile);
    const int tiles = (max(ctx, 0) + kKvTile - 1) / kKvTile;
    Kv8Query<D> a;
    a.clear();
    a.load_query(g < G ? q + ((size_t)b * nq + (size_t)kvh * G + g) * D : nullptr, tq);
    for (int t = warp; t < tiles; t += K8D_WARPS) {
        const int page = page_table[(size_t)b * max_pages + t];
        if (page < 0 || page >= num_pages) continue;
        a.page(cache + ((size_t)page * nkv + kvh) * Kv8<D>::REC, min(ctx - t * kKvTile, kKvTile), scale_log2, g, tq);
    }
    a.store(&rec_s[warp][0][0], g, tq);
    __syncthreads();
    for (int e = threadIdx.x; e < G * D; e += K8D_WARPS * 32) {
        const int h = e / D, dim = e % D;
        float M = -INFINITY, L = 0.f, O = 0.f;
        for (int w = 0; w < K8D_WARPS; ++w) M = fmaxf(M, rec_s[w][h][D]);
        for (int w = 0; w < K8D_WARPS; ++w) {
            const float f = M == -INFINITY ? 0.f : exp2f(rec_s[w][h][D] - M);
            L += rec_s[w][h][D + 1] * f;
            O += rec_s[w][h][dim] * f;
        }
        const float r = L > 0.f ? O / L : 0.f;                       // a sequence without a visible key: zeros
        const size_t at = ((size_t)b * nq + (size_t)kvh * G) * D + e;
        const __nv_bfloat16 hb = __float2bfloat16(r);
        out[at] = hb;
        if (out_lo) out_lo[at] = __float2bfloat16(r - __bfloat162float(hb));
    }
}

}  // namespace ft

extern "C" int ft_attn_decode_kv8(const void* q, const void* kv8_layer, int num_pages, const int* page_table, int max_pages, const int* ctx_lens, void* out,
                                  void* out_lo, int B, int nq, int nkv, int d, void* stream) {
    using namespace ft;
    FT_REQUIRE(d == 64 || d == 128, "ft_attn_decode_kv8: head_dim %d not supported (64 or 128)", d);
    FT_REQUIRE(nq >= 1 && nkv >= 1 && nq % nkv == 0 && nq / nkv <= K8D_GROUP, "ft_attn_decode_kv8: GQA group %d/%d not supported", nq, nkv);
    FT_REQUIRE(B >= 0 && max_pages >= 0 && num_pages >= 0 && max_pages <= INT32_MAX / kKvTile && (long long)B * nkv <= INT32_MAX,
               "ft_attn_decode_kv8: bad sizes B=%d nkv=%d max_pages=%d num_pages=%d", B, nkv, max_pages, num_pages);
    if (B == 0) return 0;
    FT_REQUIRE(q && kv8_layer && page_table && ctx_lens && out, "ft_attn_decode_kv8: null argument");
    FT_REQUIRE(((uintptr_t)q | (uintptr_t)kv8_layer) % 16 == 0, "ft_attn_decode_kv8: tensors on 16 bytes");
    const float scale_log2 = K8D_LOG2E / sqrtf((float)d);
    auto go = [&](auto kernel) {
        kernel<<<B * nkv, K8D_WARPS * 32, 0, (cudaStream_t)stream>>>((const __half*)q, (const uint8_t*)kv8_layer, num_pages, page_table, max_pages, ctx_lens,
                                                                     (__nv_bfloat16*)out, (__nv_bfloat16*)out_lo, nq, nkv, scale_log2);
    };
    if (d == 64) go(kv8_decode_kernel<64>);
    else go(kv8_decode_kernel<128>);
    FT_CHECK_CUDA(cudaGetLastError());
    return 0;
}
