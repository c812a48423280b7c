// Keys and queries normed head by head, rotated and, with the values, put where they belong, in one pass over the projection's result:
//   y = x * rsqrt(mean(x^2) + eps) * gain   per head of d,   then pairs (a, b) -> (a cos - b sin, b cos + a sin);   q to q_out, k and v to the paged fp16 cache.
// Pairs are (i, i + rotated / 2) or neighbours (2 i, 2 i + 1); dims from `rotated` on stay as they are.
//
// A head belongs to d / 8 lanes, each with two chunks of four numbers, chosen so that both numbers of a pair lie in one lane (lane j's chunks are j and j + rotated / 8, and
// those behind `rotated` are shared out the same way) and neighbouring lanes have neighbouring chunks.  So the only exchange is the sum of squares, and a load or store
// of the warp takes whole lines.  The factor rsqrt(..) is the same for a head, so it comes last: gain and rotation do not wait for the sum.
//
// Measured in a graph, us: one token of 48 heads of 64 1.9; 64 of 48 heads of 128 in two fp32 parts 2.5 (latency: a launch, two reads, a store).
// 7299 of 48 heads of 128 from bf16 (180 MB): neighbouring pairs 35.4 = 5.1 TB/s, 79 % of a copy; halves 41.8 = 4.3 TB/s.  From fp32 (270 MB): 55.1, and halves 48.2 = 5.6 TB/s.  With
// neighbouring pairs six of ten issue slots are in use, and a warp waits for its reads at the end of each token.  Registers, at heads of 128: 72 with neighbours and 83 in halves from
// 16 bits, 80 and 91 from 32, so seven, five, six and five CTAs fit an SM: 1825 CTAs are 1.8 rounds of them with neighbours from 16 bits and 2.5 in halves.
#include "common.cuh"
#include "ft_internal.h"

namespace ft {

constexpr int NA_WARPS = 4, NA_THREADS = NA_WARPS * 32;
// 7299 tokens of 48 heads of 128, neighbouring pairs, from bf16, us: passes whose reads are on their way together, 1 / 2 / 3: 47.9 / 35.6 / 45.8 (registers); numbers of a chunk, 4 / 8: 35.6 / 54
constexpr int NA_AHEAD = 2;
constexpr int NA_E = 4;
// Warps per SM from which a warp takes more than one pass of a token, 16 / 40 / 100: the same 35.4 / 35.4 / 37.5, and for 1861 tokens of 20 heads 8.7 / 8.7 / 12.1
constexpr int NA_FILL = 40;
constexpr int NA_CTAS = 5;                           // per SM at least (6 and 7 take as long)

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

// four numbers as two pairs of fp32
__device__ __forceinline__ void na_pairs(const uint4& raw, float, f32x2* v) {
    v[0] = pack2(__uint_as_float(raw.x), __uint_as_float(raw.y));
    v[1] = pack2(__uint_as_float(raw.z), __uint_as_float(raw.w));
}
__device__ __forceinline__ void na_pairs(const uint2& raw, __nv_bfloat16, f32x2* v) {
    v[0] = pack2(bf16_lo(raw.x), bf16_hi(raw.x));
    v[1] = pack2(bf16_lo(raw.y), bf16_hi(raw.y));
}
__device__ __forceinline__ void na_pairs(const uint2& raw, __half, f32x2* v) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&raw.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&raw.y));
    v[0] = pack2(a.x, a.y);
    v[1] = pack2(b.x, b.y);
}
__device__ __forceinline__ void na_pairs(const float* p, f32x2* v) {
    const float4 w = load_f4(p);
    v[0] = pack2(w.x, w.y);
    v[1] = pack2(w.z, w.w);
}

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
__device__ __forceinline__ uint32_t na_half2(f32x2 v) {
    uint32_t r;
    float a, b;
    unpack2(v, a, b);
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
    const int far = (c1 - c0) * E;
    const T* from = (const T*)p.x + (long long)t * p.row_stride + (p0 * HEADS + sub) * D + c0 * E;      // chunk c0 of the pass whose reads come next
    int next = p0;                                   // that pass
    Raw raw[NA_AHEAD][2];
    auto ask = [&](int u, const T* x) {              // pass next + u
        if (next + u < p1 && (next + u) * HEADS + sub < heads) {
            raw[u][0] = na_load<T, WIDE>(x + u * (HEADS * D));
            raw[u][1] = na_load<T, WIDE>(x + u * (HEADS * D) + far);
        } else {
            raw[u][0] = raw[u][1] = Raw{};
        }
    };
#pragma unroll
    for (int u = 0; u < NA_AHEAD; ++u) ask(u, from);
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
    f32x2 c2[2], s2[2], m2[2];                       // cosines, sines, minus sines
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        c2[e] = pack2(cs[2 * e], cs[2 * e + 1]);
        s2[e] = pack2(sn[2 * e], sn[2 * e + 1]);
        m2[e] = pack2(-sn[2 * e], -sn[2 * e + 1]);
    }
    uint8_t* to_q = reinterpret_cast<uint8_t*>(p.q_out + ((size_t)t * p.nq + p0 * HEADS + sub) * D + c0 * E);      // where the pass at hand goes, if it is queries
    constexpr int SLAB = kKvTile * D * 2;
    uint8_t* const cache = p.kv_layer + ((size_t)(slot / kKvTile) * p.nkv * 2) * (size_t)SLAB + kv_swizzled_chunk<D>(slot % kKvTile, c0 / 2) + c0 % 2 * 8;
    const int far_kv = kv_swizzled_chunk<D>(slot % kKvTile, c1 / 2) + c1 % 2 * 8 - (kv_swizzled_chunk<D>(slot % kKvTile, c0 / 2) + c0 % 2 * 8);
    const float* have = nullptr;                     // the gain that is in g
    f32x2 g[2][2];
    int hd = p0 * HEADS + sub;                       // the head of the pass at hand
#pragma unroll 1
    while (next < p1) {
        f32x2 v[NA_AHEAD][2][2];
#pragma unroll
        for (int u = 0; u < NA_AHEAD; ++u) na_pairs(raw[u][0], T(), v[u][0]), na_pairs(raw[u][1], T(), v[u][1]);
        if (sizeof(T) == 4) {                        // parts are fp32
            const T* part = from;
#pragma unroll 1
            for (int s = 1; s < p.parts; ++s) {
                part += p.part_stride;
#pragma unroll
                for (int u = 0; u < NA_AHEAD; ++u) ask(u, part);
#pragma unroll
                for (int u = 0; u < NA_AHEAD; ++u)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        f32x2 more[2];
                        na_pairs(raw[u][c], T(), more);
                        v[u][c][0] = sum2(v[u][c][0], more[0]);
                        v[u][c][1] = sum2(v[u][c][1], more[1]);
                    }
            }
        }
        const int here = p1 - next;
        next += NA_AHEAD;
        from += NA_AHEAD * HEADS * D;
#pragma unroll
        for (int u = 0; u < NA_AHEAD; ++u) ask(u, from);                     // the next passes are on their way meanwhile
#pragma unroll
        for (int u = 0; u < NA_AHEAD; ++u, hd += HEADS, to_q += HEADS * D * 2) {
            if (u >= here) break;
            f32x2(&x)[2][2] = v[u];
            f32x2 sq = mul2(x[0][0], x[0][0]);
            sq = fma2(x[0][1], x[0][1], sq);
            sq = fma2(x[1][0], x[1][0], sq);
            sq = fma2(x[1][1], x[1][1], sq);
            float ss, s1;
            unpack2(sq, ss, s1);
            ss += s1;
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (hd >= heads) continue;
            if (hd < p.nq + p.nkv) {
                const float* gain = hd < p.nq ? p.q_gain : p.k_gain;
                if (gain) {
                    gain += hd < p.nq ? hd * p.gain_q_stride : (hd - p.nq) * p.gain_k_stride;
                    if (gain != have) {
                        na_pairs(gain + c0 * E, g[0]);
                        na_pairs(gain + c1 * E, g[1]);
                        have = gain;
                    }
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int e = 0; e < 2; ++e) x[c][e] = mul2(x[c][e], g[c][e]);
                }
                if (NEIGHBOURS) {
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float a, b;
                            unpack2(x[c][e], a, b);
                            x[c][e] = pack2(a * cs[2 * c + e] - b * sn[2 * c + e], b * cs[2 * c + e] + a * sn[2 * c + e]);
                        }
                } else {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const f32x2 a = x[0][e], b = x[1][e];
                        x[0][e] = fma2(a, c2[e], mul2(b, m2[e]));
                        x[1][e] = fma2(b, c2[e], mul2(a, s2[e]));
                    }
                }
                const float r = rsqrtf(ss * (1.f / D) + p.eps);
                const f32x2 r2 = pack2(r, r);
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int e = 0; e < 2; ++e) x[c][e] = mul2(x[c][e], r2);
            }
            uint2 h0 = make_uint2(na_half2(x[0][0]), na_half2(x[0][1])), h1 = make_uint2(na_half2(x[1][0]), na_half2(x[1][1]));
            if (hd < p.nq) {
                if (!known) h0 = h1 = make_uint2(0u, 0u);                    // a token without a position
                *reinterpret_cast<uint2*>(to_q) = h0;
                *reinterpret_cast<uint2*>(to_q + far * 2) = h1;
            } else if (kept) {
                const int is_v = hd >= p.nq + p.nkv;
                uint8_t* to = cache + ((hd - p.nq - is_v * p.nkv) * 2 + is_v) * SLAB;
                *reinterpret_cast<uint2*>(to) = h0;
                *reinterpret_cast<uint2*>(to + far_kv) = h1;
            }
        }
    }
}

template <int D, class T>
static int launch_norm_append(NormAppend& p, bool neighbours, bool wide, cudaStream_t st) {
    constexpr int HEADS = 32 * 2 * NA_E / D;
    p.passes = (p.nq + 2 * p.nkv + HEADS - 1) / HEADS;
    // a warp takes as much of a token as leaves NA_FILL warps an SM: its angles and gains are read once
    const long long each = (long long)p.T * p.passes / ((long long)NA_FILL * device_sms());
    p.per_token = each < 1 ? p.passes : each < p.passes ? (int)((p.passes + each - 1) / each) : 1;
    p.per = (p.passes + p.per_token - 1) / p.per_token;
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
    // chunks that lie on their size are one load each (7299 tokens, neighbouring pairs, from bf16 35.4 us, with four loads 44.7; 64 single tokens 2.5 and 2.7)
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
