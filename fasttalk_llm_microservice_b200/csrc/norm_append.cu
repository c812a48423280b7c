// Keys and queries normed head by head, rotated and, with the values, put where they belong, in one pass over the projection's result:
//   y = x * rsqrt(mean(x^2) + eps) * gain   per head of d,   then pairs (a, b) -> (a cos - b sin, b cos + a sin);   q to q_out, k and v to the paged fp16 cache.
// Pairs are (i, i + rotated / 2) or neighbours (2 i, 2 i + 1); dims from `rotated` on stay as they are.
//
// A head belongs to d / 8 lanes, each with two chunks of four numbers, chosen so that both numbers of a pair lie in one lane (lane j's chunks are j and j + rotated / 8, and
// those behind `rotated` are shared out the same way) and neighbouring lanes have neighbouring chunks.  So the only exchange is the sum of squares, and a load or store
// of the warp takes whole lines.  The factor rsqrt(..) is the same for a head, so it comes last: gain and rotation do not wait for the sum.
#include "common.cuh"
#include "ft_internal.h"

namespace ft {

constexpr int NA_WARPS = 4, NA_THREADS = NA_WARPS * 32;
constexpr int NA_AHEAD = 2;                          // passes whose reads are on their way together
constexpr int NA_FILL = 40;                          // warps per SM from which a warp takes more than one pass of a token
constexpr int NA_E = 4;
constexpr int NA_CTAS = 5;                           // per SM

struct NormAppend {
    const void* x;
    long long part_stride, row_stride;               // elements from part to part, token to token
    const float *cos_t, *sin_t, *q_gain, *k_gain;
    const int *positions, *kv_slots;
    __half* q_out;
    uint8_t* kv_layer;
    int slots;                                       // pages * 64
    int parts, T, nq, nkv, n_angles, rotated, gain_q_stride, gain_k_stride;      // gain strides: 0 = one gain for all heads
    int passes, per, per_token;                      // passes of a token (a warp's heads each), of a warp; warps of a token
    float eps;
};

__device__ __forceinline__ float na_float(float v) { return v; }
__device__ __forceinline__ float na_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float na_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// four numbers as they lie in memory
template <class T> struct NaRaw { typedef uint2 type; };
template <> struct NaRaw<float> { typedef uint4 type; };
template <class T, bool WIDE>
__device__ __forceinline__ typename NaRaw<T>::type na_load(const T* p) {     // WIDE: a chunk is one load
    typedef typename NaRaw<T>::type Raw;
    alignas(16) T raw[NA_E];
    if (WIDE) {
        *reinterpret_cast<Raw*>(raw) = __ldcs(reinterpret_cast<const Raw*>(p));      // read once
    } else {
#pragma unroll
        for (int e = 0; e < NA_E; ++e) raw[e] = p[e];
    }
    return *reinterpret_cast<const Raw*>(raw);
}
// within fp16's range, NaN as it is
__device__ __forceinline__ uint32_t na_half2(float a, float b) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

template <int D, class T, bool NEIGHBOURS, bool WIDE>
__global__ void __launch_bounds__(NA_THREADS, NA_CTAS)
norm_append_kernel(const __grid_constant__ NormAppend p) {
    pdl_wait();
    constexpr int E = NA_E, LANES = D / (2 * E), HEADS = 32 / LANES;         // lanes of a head, heads of a pass
    typedef typename NaRaw<T>::type Raw;
    const int warp = blockIdx.x * NA_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int t = warp / p.per_token;
    if (t >= p.T) return;
    const int heads = p.nq + 2 * p.nkv, sub = lane / LANES, j = lane % LANES;
    const int turned = p.rotated / (2 * E);          // lanes of a head that rotate, where pairs are halves
    const int c0 = !NEIGHBOURS && j >= turned ? turned + j : j, c1 = !NEIGHBOURS && j < turned ? j + turned : j + LANES;
    const int p0 = (warp - t * p.per_token) * p.per, p1 = min(p0 + p.per, p.passes);
    const T* const row = (const T*)p.x + (long long)t * p.row_stride + sub * D;
    Raw raw[NA_AHEAD][2];
    auto ask = [&](int u, int first, int s) {        // pass first + u, part s
        if (first + u < p1 && (first + u) * HEADS + sub < heads) {
            const T* from = row + s * p.part_stride + (long long)(first + u) * (HEADS * D);
            raw[u][0] = na_load<T, WIDE>(from + c0 * E);
            raw[u][1] = na_load<T, WIDE>(from + c1 * E);
        } else {
            raw[u][0] = raw[u][1] = Raw{};
        }
    };
#pragma unroll
    for (int u = 0; u < NA_AHEAD; ++u) ask(u, p0, 0);
    const int pos = p.positions[t], slot = p.kv_slots[t];
    const bool known = pos >= 0 && (p.rotated == 0 || pos < p.n_angles);
    const bool kept = known && slot >= 0 && slot < p.slots;
    // angles: halves, of chunk c0's numbers; neighbours, of c0's pairs and then of c1's.  Chunks that do not rotate: 1 and 0
    float cs[E] = {1.f, 1.f, 1.f, 1.f}, sn[E] = {0.f, 0.f, 0.f, 0.f};
    {
        const size_t at = (size_t)pos * (p.rotated / 2);
        if (NEIGHBOURS) {
            if (known && c0 * E < p.rotated) {
                *reinterpret_cast<float2*>(cs) = *reinterpret_cast<const float2*>(p.cos_t + at + c0 * (E / 2));
                *reinterpret_cast<float2*>(sn) = *reinterpret_cast<const float2*>(p.sin_t + at + c0 * (E / 2));
            }
            if (known && c1 * E < p.rotated) {
                *reinterpret_cast<float2*>(cs + 2) = *reinterpret_cast<const float2*>(p.cos_t + at + c1 * (E / 2));
                *reinterpret_cast<float2*>(sn + 2) = *reinterpret_cast<const float2*>(p.sin_t + at + c1 * (E / 2));
            }
        } else if (known && j < turned) {
            *reinterpret_cast<float4*>(cs) = load_f4(p.cos_t + at + c0 * E);
            *reinterpret_cast<float4*>(sn) = load_f4(p.sin_t + at + c0 * E);
        }
    }
    uint8_t* const cache = p.kv_layer + ((size_t)(slot / kKvTile) * p.nkv * 2) * (size_t)(kKvTile * D * 2);
    const int in0 = kv_swizzled_chunk<D>(slot % kKvTile, c0 / 2) + c0 % 2 * 8, in1 = kv_swizzled_chunk<D>(slot % kKvTile, c1 / 2) + c1 % 2 * 8;      // of a page's head
    const float* have = nullptr;                     // the gain that is in g
    float g[2][E];
#pragma unroll 1
    for (int first = p0; first < p1; first += NA_AHEAD) {
        float v[NA_AHEAD][2][E];
#pragma unroll
        for (int u = 0; u < NA_AHEAD; ++u)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < E; ++e) v[u][c][e] = na_float(reinterpret_cast<const T*>(&raw[u][c])[e]);
        if (sizeof(T) == 4)                          // parts are fp32
#pragma unroll 1
            for (int s = 1; s < p.parts; ++s) {
#pragma unroll
                for (int u = 0; u < NA_AHEAD; ++u) ask(u, first, s);
#pragma unroll
                for (int u = 0; u < NA_AHEAD; ++u)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int e = 0; e < E; ++e) v[u][c][e] += na_float(reinterpret_cast<const T*>(&raw[u][c])[e]);
            }
#pragma unroll
        for (int u = 0; u < NA_AHEAD; ++u) ask(u, first + NA_AHEAD, 0);      // the next passes are on their way meanwhile
#pragma unroll
        for (int u = 0; u < NA_AHEAD; ++u) {
            if (first + u >= p1) break;
            const int hd = (first + u) * HEADS + sub;
            float(&x)[2][E] = v[u];
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) ss = fmaf(x[0][e], x[0][e], fmaf(x[1][e], x[1][e], ss));
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (hd >= heads) continue;
            float r = 1.f;
            if (hd < p.nq + p.nkv) {
                const float* gain = hd < p.nq ? p.q_gain : p.k_gain;
                if (gain) {
                    gain += hd < p.nq ? hd * p.gain_q_stride : (hd - p.nq) * p.gain_k_stride;
                    if (gain != have) {
                        *reinterpret_cast<float4*>(g[0]) = load_f4(gain + c0 * E);
                        *reinterpret_cast<float4*>(g[1]) = load_f4(gain + c1 * E);
                        have = gain;
                    }
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int e = 0; e < E; ++e) x[c][e] *= g[c][e];
                }
                if (NEIGHBOURS) {
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int e = 0; e < E; e += 2) {
                            const float a = x[c][e], b = x[c][e + 1], co = cs[c * 2 + e / 2], si = sn[c * 2 + e / 2];
                            x[c][e] = a * co - b * si;
                            x[c][e + 1] = b * co + a * si;
                        }
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float a = x[0][e], b = x[1][e];
                        x[0][e] = a * cs[e] - b * sn[e];
                        x[1][e] = b * cs[e] + a * sn[e];
                    }
                }
                r = rsqrtf(ss * (1.f / D) + p.eps);
            }
            uint8_t *to0, *to1;
            if (hd < p.nq) {
                to0 = reinterpret_cast<uint8_t*>(p.q_out + ((size_t)t * p.nq + hd) * D);
                to1 = to0 + c1 * E * 2;
                to0 += c0 * E * 2;
            } else {
                if (!kept) continue;
                const bool is_v = hd >= p.nq + p.nkv;
                uint8_t* slab = cache + ((hd - p.nq - (is_v ? p.nkv : 0)) * 2 + is_v) * (kKvTile * D * 2);
                to0 = slab + in0;
                to1 = slab + in1;
            }
            uint2 h[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                h[c] = make_uint2(na_half2(x[c][0] * r, x[c][1] * r), na_half2(x[c][2] * r, x[c][3] * r));
                if (!known) h[c] = make_uint2(0u, 0u);       // q of a token without a position
            }
            *reinterpret_cast<uint2*>(to0) = h[0];
            *reinterpret_cast<uint2*>(to1) = h[1];
        }
    }
}

template <int D, class T>
static int launch_norm_append(NormAppend& p, bool neighbours, bool wide, cudaStream_t st) {
    constexpr int HEADS = 32 * 2 * NA_E / D;
    p.passes = (p.nq + 2 * p.nkv + HEADS - 1) / HEADS;
    // a warp takes as much of a token as leaves NA_FILL warps an SM: its angles and gains are read once
    const long long each = (long long)p.T * p.passes / ((long long)NA_FILL * device_sms());
    p.per = each < 1 ? 1 : each < p.passes ? (int)each : p.passes;
    p.per_token = (p.passes + p.per - 1) / p.per;
    const long long warps = (long long)p.T * p.per_token;
    const dim3 grid((unsigned)((warps + NA_WARPS - 1) / NA_WARPS));
    const auto kernel = neighbours ? (wide ? norm_append_kernel<D, T, true, true> : norm_append_kernel<D, T, true, false>)
                                   : (wide ? norm_append_kernel<D, T, false, true> : norm_append_kernel<D, T, false, false>);
    FT_CHECK_CUDA(launch_after(kernel, grid, dim3(NA_THREADS), 0, st, (const NormAppend&)p));
    return 0;
}

}  // namespace ft

extern "C" int ft_norm_rope_kv_append(const ft_norm_append_args* args, void* stream) {
    using namespace ft;
    FT_REQUIRE(args, "ft_norm_rope_kv_append: null argument");
    const auto [qkv, part_stride, row_stride, cos_t, sin_t, q_gain, k_gain, positions, kv_slots, q_out, kv_layer, type, n_parts, n_angles, rotated, neighbours, q_gains, k_gains,
                num_pages, T, nq, nkv, d, eps] = *args;
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
    const int chunk = size * NA_E;
    const bool wide = (uintptr_t)qkv % chunk == 0 && row_stride * size % chunk == 0 && (n_parts == 1 || part_stride * size % chunk == 0);
    NormAppend p{qkv, part_stride, row_stride, cos_t, sin_t, q_gain, k_gain, positions, kv_slots, (__half*)q_out, (uint8_t*)kv_layer, num_pages * kKvTile, n_parts, T,
                 nq, nkv, n_angles, rotated, q_gains > 1 ? d : 0, k_gains > 1 ? d : 0, 0, 0, 0, eps};
    const cudaStream_t st = (cudaStream_t)stream;
#define FT_NA_CASE(D_, TYPE_, T_) \
    if (d == D_ && type == TYPE_) return launch_norm_append<D_, T_>(p, neighbours != 0, wide, st);
    FT_NA_CASE(64, FT_F32, float)
    FT_NA_CASE(64, FT_BF16, __nv_bfloat16)
    FT_NA_CASE(64, FT_F16, __half)
    FT_NA_CASE(128, FT_F32, float)
    FT_NA_CASE(128, FT_BF16, __nv_bfloat16)
    FT_NA_CASE(128, FT_F16, __half)
#undef FT_NA_CASE
    return 0;
}
