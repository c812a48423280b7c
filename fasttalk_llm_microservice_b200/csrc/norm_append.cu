// Keys and queries normed head by head, rotated and, with the values, put where they belong, in one pass over the projection's result:
//   y = x * rsqrt(mean(x^2) + eps) * gain   per head of d,   then pairs (a, b) -> (a cos - b sin, b cos + a sin);   q to q_out, k and v to the paged fp16 cache.
// Pairs are (i, i + rotated / 2) or neighbours (2 i, 2 i + 1); dims from `rotated` on stay as they are.
//
// A head belongs to D / (2 E) lanes (E numbers are 16 bytes of the input), each with two chunks of E, chosen so that both numbers of a pair lie in one lane: whatever
// `rotated` is, lane j's chunks are j and j + rotated / (2 E), and those behind `rotated` follow two by two.  So the only exchange is the sum of squares, and a chunk of
// eight fp16 results is one 16-byte store, a chunk of a row in the cache.
#include "common.cuh"
#include "ft_internal.h"

namespace ft {

constexpr int NA_WARPS = 4, NA_THREADS = NA_WARPS * 32;

template <class T> struct NaType;
template <> struct NaType<float> { static constexpr int E = 4; };
template <> struct NaType<__half> { static constexpr int E = 8; };
template <> struct NaType<__nv_bfloat16> { static constexpr int E = 8; };

struct NormAppend {
    const void* x;
    long long part_stride, row_stride;               // elements from part to part, token to token
    const float *cos_t, *sin_t, *q_gain, *k_gain;
    const int *positions, *kv_slots;
    __half* q_out;
    uint8_t* kv_layer;
    long long slots;                                 // pages * 64
    int parts, T, nq, nkv, n_angles, rotated, gain_q_stride, gain_k_stride;      // gain strides: 0 = one gain for all heads
    int passes, per, per_token;                      // passes of a token (a warp's heads each), of a warp; warps of a token
    int wide;                                        // 1: 16-byte loads
    float eps;
};

__device__ __forceinline__ float na_float(float v) { return v; }
__device__ __forceinline__ float na_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float na_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ void na_load(const T* p, float* v, bool wide) {
    constexpr int E = NaType<T>::E;
    alignas(16) T raw[E];
    if (wide) {
        *reinterpret_cast<uint4*>(raw) = __ldcg(reinterpret_cast<const uint4*>(p));
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) raw[e] = p[e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = na_float(raw[e]);
}
template <int E>
__device__ __forceinline__ void na_load_f32(const float* p, float* v) {
#pragma unroll
    for (int e = 0; e < E; e += 4) {
        const float4 w = *reinterpret_cast<const float4*>(p + e);
        v[e] = w.x; v[e + 1] = w.y; v[e + 2] = w.z; v[e + 3] = w.w;
    }
}
// within fp16's range, NaN as it is
__device__ __forceinline__ __half2 na_half2(float a, float b) {
    a = a != a ? a : fminf(fmaxf(a, -65504.f), 65504.f);
    b = b != b ? b : fminf(fmaxf(b, -65504.f), 65504.f);
    return __floats2half2_rn(a, b);
}

template <int D, class T, bool NEIGHBOURS>
__global__ void __launch_bounds__(NA_THREADS)
norm_append_kernel(const __grid_constant__ NormAppend p) {
    pdl_wait();
    constexpr int E = NaType<T>::E, LANES = D / (2 * E), HEADS = 32 / LANES;      // lanes of a head, heads of a pass
    const int warp = blockIdx.x * NA_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int t = warp / p.per_token;
    if (t >= p.T) return;
    const int heads = p.nq + 2 * p.nkv, sub = lane / LANES, j = lane % LANES;
    const int turned = p.rotated / (2 * E);          // lanes of a head that rotate
    // chunks of this lane; behind the rotated ones they follow two by two
    int c0, c1;
    if (NEIGHBOURS) c0 = 2 * j, c1 = 2 * j + 1;
    else if (j < turned) c0 = j, c1 = j + turned;
    else c0 = 2 * j, c1 = 2 * j + 1;
    const int pos = p.positions[t];
    const long long slot = p.kv_slots[t];
    const bool known = pos >= 0 && (p.rotated == 0 || pos < p.n_angles);
    const bool kept = known && slot >= 0 && slot < p.slots;
    float cs[E], sn[E];                              // halves: of chunk c0's numbers; neighbours: of c0's pairs, then of c1's
    const bool rotates = known && (NEIGHBOURS ? j * 2 * E < p.rotated : j < turned);
    if (rotates) {
        const float* at = p.cos_t + (size_t)pos * (p.rotated / 2) + j * E;
        na_load_f32<E>(at, cs);
        na_load_f32<E>(p.sin_t + (at - p.cos_t), sn);
    }
    const int p0 = (warp - t * p.per_token) * p.per, p1 = min(p0 + p.per, p.passes);
    for (int pass = p0; pass < p1; ++pass) {
        const int hd = pass * HEADS + sub;
        const bool on = hd < heads;
        float v[2][E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[0][e] = v[1][e] = 0.f;
        if (on) {
            const T* row = (const T*)p.x + (long long)t * p.row_stride + (long long)hd * D;
            na_load<T>(row + c0 * E, v[0], p.wide);
            na_load<T>(row + c1 * E, v[1], p.wide);
            for (int s = 1; s < p.parts; ++s) {
                float w[2][E];
                na_load<T>(row + s * p.part_stride + c0 * E, w[0], p.wide);
                na_load<T>(row + s * p.part_stride + c1 * E, w[1], p.wide);
#pragma unroll
                for (int e = 0; e < E; ++e) v[0][e] += w[0][e], v[1][e] += w[1][e];
            }
        }
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) ss = fmaf(v[0][e], v[0][e], fmaf(v[1][e], v[1][e], ss));
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (!on) continue;
        if (hd < p.nq + p.nkv) {
            const float r = rsqrtf(ss * (1.f / D) + p.eps);
            const float* gain = hd < p.nq ? p.q_gain : p.k_gain;
            if (gain) {
                gain += hd < p.nq ? hd * p.gain_q_stride : (hd - p.nq) * p.gain_k_stride;
                float g0[E], g1[E];
                na_load_f32<E>(gain + c0 * E, g0);
                na_load_f32<E>(gain + c1 * E, g1);
#pragma unroll
                for (int e = 0; e < E; ++e) v[0][e] *= r * g0[e], v[1][e] *= r * g1[e];
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) v[0][e] *= r, v[1][e] *= r;
            }
            if (rotates) {
                if (NEIGHBOURS) {
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int e = 0; e < E; e += 2) {
                            const float a = v[c][e], b = v[c][e + 1], co = cs[c * (E / 2) + e / 2], si = sn[c * (E / 2) + e / 2];
                            v[c][e] = a * co - b * si;
                            v[c][e + 1] = b * co + a * si;
                        }
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float a = v[0][e], b = v[1][e];
                        v[0][e] = a * cs[e] - b * sn[e];
                        v[1][e] = b * cs[e] + a * sn[e];
                    }
                }
            }
        }
        uint8_t *to0, *to1;
        if (hd < p.nq) {
            to0 = reinterpret_cast<uint8_t*>(p.q_out + ((size_t)t * p.nq + hd) * D);
            to1 = to0 + c1 * E * 2;
            to0 += c0 * E * 2;
            if (!known) {                            // a token without a position: zeros
#pragma unroll
                for (int e = 0; e < E; ++e) v[0][e] = v[1][e] = 0.f;
            }
        } else {
            if (!kept) continue;
            const bool is_v = hd >= p.nq + p.nkv;
            const int h = hd - p.nq - (is_v ? p.nkv : 0), r = (int)(slot % kKvTile);
            uint8_t* slab = p.kv_layer + (((size_t)(slot / kKvTile) * p.nkv + h) * 2 + is_v) * (size_t)(kKvTile * D * 2);
            to0 = slab + kv_swizzled_chunk<D>(r, c0 * E / 8) + c0 * E % 8 * 2;
            to1 = slab + kv_swizzled_chunk<D>(r, c1 * E / 8) + c1 * E % 8 * 2;
        }
        alignas(16) __half2 h[2][E / 2];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < E; e += 2) h[c][e / 2] = na_half2(v[c][e], v[c][e + 1]);
        if (E == 8) {
            *reinterpret_cast<uint4*>(to0) = *reinterpret_cast<const uint4*>(h[0]);
            *reinterpret_cast<uint4*>(to1) = *reinterpret_cast<const uint4*>(h[1]);
        } else {
            *reinterpret_cast<uint2*>(to0) = *reinterpret_cast<const uint2*>(h[0]);
            *reinterpret_cast<uint2*>(to1) = *reinterpret_cast<const uint2*>(h[1]);
        }
    }
}

template <int D, class T>
static int launch_norm_append(NormAppend& p, bool neighbours, cudaStream_t st) {
    constexpr int E = NaType<T>::E, HEADS = 32 * 2 * E / D;
    p.passes = (p.nq + 2 * p.nkv + HEADS - 1) / HEADS;
    p.per = 1;
    p.per_token = (p.passes + p.per - 1) / p.per;
    const long long warps = (long long)p.T * p.per_token;
    const dim3 grid((unsigned)((warps + NA_WARPS - 1) / NA_WARPS));
    if (neighbours) FT_CHECK_CUDA(launch_after(norm_append_kernel<D, T, true>, grid, dim3(NA_THREADS), 0, st, (const NormAppend&)p));
    else FT_CHECK_CUDA(launch_after(norm_append_kernel<D, T, false>, grid, dim3(NA_THREADS), 0, st, (const NormAppend&)p));
    return 0;
}

}  // namespace ft

extern "C" int ft_norm_rope_kv_append(const void* qkv, int type, int n_parts, long long part_stride, long long row_stride, const float* cos_t, const float* sin_t, int n_angles,
                                      int rotated, int neighbours, const float* q_gain, int q_gains, const float* k_gain, int k_gains, float eps, const int* positions,
                                      const int* kv_slots, void* q_out, void* kv_layer, int num_pages, int T, int nq, int nkv, int d, void* stream) {
    using namespace ft;
    FT_REQUIRE(d == 64 || d == 128, "ft_norm_rope_kv_append: head_dim %d not supported (64 or 128)", d);
    FT_REQUIRE(type >= FT_F32 && type <= FT_F16, "ft_norm_rope_kv_append: type %d (FT_F32, FT_BF16 or FT_F16)", type);
    FT_REQUIRE(nq >= 0 && nkv >= 0 && nq + 2LL * nkv >= 1 && (nq + 2LL * nkv) * d <= INT32_MAX && T >= 0 && n_parts >= 1 && num_pages >= 0 && num_pages <= INT32_MAX / kKvTile,
               "ft_norm_rope_kv_append: bad sizes T=%d nq=%d nkv=%d parts=%d pages=%d", T, nq, nkv, n_parts, num_pages);
    FT_REQUIRE(rotated >= 0 && rotated <= d && rotated % 16 == 0 && n_angles >= 0 && (rotated == 0 || n_angles == 0 || (cos_t && sin_t)),
               "ft_norm_rope_kv_append: %d dims rotated (a multiple of 16 up to %d, with tables)", rotated, d);
    FT_REQUIRE((!q_gain || q_gains == 1 || q_gains == nq) && (!k_gain || k_gains == 1 || k_gains == nkv), "ft_norm_rope_kv_append: a gain for all heads or one for each");
    FT_REQUIRE(n_parts == 1 || type == FT_F32, "ft_norm_rope_kv_append: parts are fp32");
    if (T == 0) return 0;
    FT_REQUIRE(qkv && positions && kv_slots && (q_out || nq == 0) && (kv_layer || num_pages == 0 || nkv == 0), "ft_norm_rope_kv_append: null argument");
    FT_REQUIRE(((uintptr_t)q_out | (uintptr_t)kv_layer | (uintptr_t)cos_t | (uintptr_t)sin_t | (uintptr_t)q_gain | (uintptr_t)k_gain) % 16 == 0,
               "ft_norm_rope_kv_append: q_out, the cache, the tables and the gains on 16 bytes");
    const int size = type == FT_F32 ? 4 : 2;
    FT_REQUIRE((uintptr_t)qkv % size == 0, "ft_norm_rope_kv_append: qkv on its own size");
    FT_REQUIRE((double)T * (nq + 2.0 * nkv) <= INT32_MAX, "ft_norm_rope_kv_append: %d tokens are more than one call takes", T);
    const bool wide = (uintptr_t)qkv % 16 == 0 && row_stride * size % 16 == 0 && (n_parts == 1 || part_stride * size % 16 == 0);
    NormAppend p{qkv, part_stride, row_stride, cos_t, sin_t, q_gain, k_gain, positions, kv_slots, (__half*)q_out, (uint8_t*)kv_layer, (long long)num_pages * kKvTile, n_parts, T,
                 nq, nkv, n_angles, rotated, q_gains > 1 ? d : 0, k_gains > 1 ? d : 0, 0, 0, 0, wide, eps};
    const cudaStream_t st = (cudaStream_t)stream;
#define FT_NA_CASE(D_, TYPE_, T_) \
    if (d == D_ && type == TYPE_) return launch_norm_append<D_, T_>(p, neighbours != 0, st);
    FT_NA_CASE(64, FT_F32, float)
    FT_NA_CASE(64, FT_BF16, __nv_bfloat16)
    FT_NA_CASE(64, FT_F16, __half)
    FT_NA_CASE(128, FT_F32, float)
    FT_NA_CASE(128, FT_BF16, __nv_bfloat16)
    FT_NA_CASE(128, FT_F16, __half)
#undef FT_NA_CASE
    return 0;
}
