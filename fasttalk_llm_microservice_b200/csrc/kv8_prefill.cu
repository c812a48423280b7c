// Causal attention of prompt portions over the 8-bit KV cache (kv8.cuh): request r owns rows req_q_start[r] .. req_q_start[r + 1] - 1 of q, its first query
// sits at position req_pos0[r], and out[t][h] = sum_j softmax_j(q . k_j / sqrt(D)) v_j over the keys j <= position of t.
//
// A CTA takes a request's 64 query rows (row = token * G + head of the group) of one key head; each page is turned into fp16 in shared memory and multiplied
// there (mma.sync), one warp for 16 rows.
#include "common.cuh"
#include "ft_internal.h"
#include "kv8.cuh"

namespace ft {

constexpr int K8P_WARPS = 4, K8P_ROWS = 16 * K8P_WARPS, K8P_GROUP = 8;
constexpr float K8P_LOG2E = 1.4426950408889634f;

template <int D>
__global__ void __launch_bounds__(K8P_WARPS * 32)
kv8_prefill_kernel(const __half* __restrict__ q, const uint8_t* __restrict__ cache, int num_pages, const int* __restrict__ page_table, int table_rows,
                   int max_pages, const int* __restrict__ req_q_start, const int* __restrict__ req_slot, const int* __restrict__ req_pos0, int n_req, int T,
                   int tokens, __nv_bfloat16* __restrict__ out, __nv_bfloat16* __restrict__ out_lo, int nq, int nkv, float scale_log2) {
    constexpr int LD = D + 8;                                        // halves a row: 16 bytes more than the row, no bank twice in ldmatrix
    __shared__ __align__(16) __half kv_s[kKvTile * LD];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
    const int G = nq / nkv, kvh = blockIdx.y;
    // which request's which tile this CTA is
    int tile = blockIdx.x, req = 0, q0 = 0, len = 0;
    for (; req < n_req; ++req) {
        q0 = max(0, min(req_q_start[req], T));
        len = max(0, min(req_q_start[req + 1], T) - q0);
        const int n = (len + tokens - 1) / tokens;
        if (tile < n) break;
        tile -= n;
    }
    if (req >= n_req) return;
    const int t0 = tile * tokens, n_tok = min(tokens, len - t0);
    const int slot = req_slot[req];
    const int pos0 = max(0, req_pos0[req]) + t0;
    const int keys = slot < 0 || slot >= table_rows ? 0 : (int)min((long long)pos0 + n_tok, (long long)max_pages * kKvTile);
    uint32_t qa[D / 16][4];
    int row[2], pos[2];
    size_t at[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        row[e] = warp * 16 + g + 8 * e;
        const int tok = row[e] / G;
        pos[e] = tok < n_tok ? pos0 + tok : -1;
        at[e] = ((size_t)(q0 + t0 + tok) * nq + (size_t)kvh * G + row[e] % G) * D;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h) qa[k][e + 2 * h] = pos[e] >= 0 ? *reinterpret_cast<const uint32_t*>(q + at[e] + k * 16 + 8 * h + 2 * tq) : 0u;
    }
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, vref = 0.f;
    for (int tile_k = 0; tile_k * kKvTile < keys; ++tile_k) {
        const int page = page_table[(size_t)slot * max_pages + tile_k];
        if (page < 0 || page >= num_pages) continue;
        const uint8_t* rec = cache + ((size_t)page * nkv + kvh) * Kv8<D>::REC;
        const float4 ks = *reinterpret_cast<const float4*>(rec + Kv8<D>::SCALES), vs = *reinterpret_cast<const float4*>(rec + Kv8<D>::SCALES + 16);
        const float kscale[4] = {ks.x * scale_log2, ks.y * scale_log2, ks.z * scale_log2, ks.w * scale_log2};
        auto load = [&](bool values) {
            __syncthreads();
            for (int i = threadIdx.x; i < kKvTile * D / 16; i += K8P_WARPS * 32) {
                const int t = i / (D / 16), c = i % (D / 16);
                const uint4 w = *reinterpret_cast<const uint4*>(rec + (values ? kv8_value_chunk<D>(t, c) : kv8_key_chunk(t, c)));
                uint4* dst = reinterpret_cast<uint4*>(kv_s + t * LD + c * 16);
                dst[0] = make_uint4(kv8_lo(w.x), kv8_hi(w.x), kv8_lo(w.y), kv8_hi(w.y));
                dst[1] = make_uint4(kv8_lo(w.z), kv8_hi(w.z), kv8_lo(w.w), kv8_hi(w.w));
            }
            __syncthreads();
        };
        load(false);
        float s[8][4], most[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                const uint32_t* b = reinterpret_cast<const uint32_t*>(kv_s + (8 * j + g) * LD + k * 16 + 2 * tq);
                mma_f16_16816(s[j], qa[k][0], qa[k][1], qa[k][2], qa[k][3], b[0], b[4]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = tile_k * kKvTile + 8 * j + 2 * tq + (e & 1);
                s[j][e] = key <= pos[e >> 1] ? s[j][e] * kscale[j >> 1] : -INFINITY;
                most[e >> 1] = fmaxf(most[e >> 1], s[j][e]);
            }
        }
        load(true);
        const float v_new = fmaxf(vref, fmaxf(fmaxf(vs.x, vs.y), fmaxf(vs.z, vs.w)));
        const float v_inv = v_new > 0.f ? 1.f / v_new : 0.f;
        float keep[2], mu[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            most[e] = fmaxf(most[e], __shfl_xor_sync(0xffffffffu, most[e], 1));
            most[e] = fmaxf(most[e], __shfl_xor_sync(0xffffffffu, most[e], 2));
            const float m_new = fmaxf(m[e], most[e]);
            mu[e] = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = exp2f(m[e] - mu[e]);
            l[e] *= alpha;
            keep[e] = alpha * (vref * v_inv);
            m[e] = m_new;
        }
        vref = v_new;
        const float vscale[4] = {vs.x * v_inv, vs.y * v_inv, vs.z * v_inv, vs.w * v_inv};
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[i][0] *= keep[0], o[i][1] *= keep[0], o[i][2] *= keep[1], o[i][3] *= keep[1];
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            uint32_t pa[4];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float p0 = exp2f(s[2 * kk + h][2 * e] - mu[e]), p1 = exp2f(s[2 * kk + h][2 * e + 1] - mu[e]);
                    l[e] += p0 + p1;
                    const __half2 t = __floats2half2_rn(p0 * vscale[kk], p1 * vscale[kk]);
                    pa[2 * h + e] = *reinterpret_cast<const uint32_t*>(&t);
                }
            const int r = kk * 16 + (lane & 15);
#pragma unroll
            for (int np = 0; np < D / 16; ++np) {
                uint32_t b0, b1, b2, b3;
                ldmatrix_x4_trans(smem_u32(kv_s + r * LD + np * 16 + (lane >> 4) * 8), b0, b1, b2, b3);
                mma_f16_16816(o[2 * np], pa[0], pa[1], pa[2], pa[3], b0, b1);
                mma_f16_16816(o[2 * np + 1], pa[0], pa[1], pa[2], pa[3], b2, b3);
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
        if (pos[e] < 0) continue;
        const float f = l[e] > 0.f ? vref / l[e] : 0.f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            const float x = o[i][2 * e] * f, y = o[i][2 * e + 1] * f;
            const uint32_t h = pack_bf16(x, y);
            *reinterpret_cast<uint32_t*>(out + at[e] + 8 * i + 2 * tq) = h;
            if (out_lo) *reinterpret_cast<uint32_t*>(out_lo + at[e] + 8 * i + 2 * tq) = pack_bf16(x - bf16_lo(h), y - bf16_hi(h));
        }
    }
}

}  // namespace ft

extern "C" int ft_attn_prefill_kv8(const void* q, const void* kv8_layer, int num_pages, const int* page_table, int table_rows, int max_pages,
                                   const int* req_q_start, const int* req_slot, const int* req_pos0, int n_req, int T, void* out, void* out_lo, int nq, int nkv,
                                   int d, void* stream) {
    using namespace ft;
    FT_REQUIRE(d == 64 || d == 128, "ft_attn_prefill_kv8: head_dim %d not supported (64 or 128)", d);
    FT_REQUIRE(nq >= 1 && nkv >= 1 && nq % nkv == 0 && nq / nkv <= K8P_GROUP, "ft_attn_prefill_kv8: GQA group %d/%d not supported", nq, nkv);
    FT_REQUIRE(T >= 0 && n_req >= 0 && table_rows >= 0 && max_pages >= 0 && num_pages >= 0 && max_pages <= INT32_MAX / kKvTile && nkv <= 65535,
               "ft_attn_prefill_kv8: bad sizes T=%d n_req=%d nkv=%d table %d x %d, %d pages", T, n_req, nkv, table_rows, max_pages, num_pages);
    if (T == 0) return 0;
    FT_REQUIRE(q && kv8_layer && out && (n_req == 0 || (page_table && req_q_start && req_slot && req_pos0)), "ft_attn_prefill_kv8: null argument");
    FT_REQUIRE(((uintptr_t)q | (uintptr_t)kv8_layer) % 16 == 0, "ft_attn_prefill_kv8: tensors on 16 bytes");
    cudaStream_t st = (cudaStream_t)stream;
    FT_CHECK_CUDA(cudaMemsetAsync(out, 0, (size_t)T * nq * d * 2, st));      // rows that no request owns
    if (out_lo) FT_CHECK_CUDA(cudaMemsetAsync(out_lo, 0, (size_t)T * nq * d * 2, st));
    if (n_req == 0) return 0;
    const int tokens = K8P_ROWS / (nq / nkv);
    const dim3 grid(T / tokens + n_req, nkv);
    const float scale_log2 = K8P_LOG2E / sqrtf((float)d);
    auto go = [&](auto kernel) {
        kernel<<<grid, K8P_WARPS * 32, 0, st>>>((const __half*)q, (const uint8_t*)kv8_layer, num_pages, page_table, table_rows, max_pages, req_q_start, req_slot,
                                                req_pos0, n_req, T, tokens, (__nv_bfloat16*)out, (__nv_bfloat16*)out_lo, nq, nkv, scale_log2);
    };
    if (d == 64) go(kv8_prefill_kernel<64>);
    else go(kv8_prefill_kernel<128>);
    FT_CHECK_CUDA(cudaGetLastError());
    return 0;
}
