// The 8-bit KV cache: layout of a record and the conversions its kernels share.
//
// One layer is [page][kv_head][record], a page = 64 tokens.  A record holds the key codes and the value codes of the page's 64 tokens for one head, D bytes a
// token each, and behind them eight fp32 scales: keys' blocks 0..3, values' blocks 0..3, a block = 16 tokens.  A code c stands for (c - 128) * scale of its block.
// Codes and scales lie side by side so that an attention tile is ONE contiguous copy (8224 bytes at D = 64, 16416 at 128, both multiples of 32).
//
// Keys: D / 64 pieces of [64 tokens][64 bytes].  A lane of an mma.sync fragment takes 16 bytes of one token; eight lanes take two whole rows, 128 bytes.
// Values: the same pieces, but token t lies in row t ^ (t >> 1 & 1) and the two 32-byte halves of a row change places where t & 4: the lanes of a fragment
// take 8 bytes each of the tokens 0, 2, 4, 6 (or 1, 3, 5, 7) at once, which would be the same banks of shared memory four times over.
#pragma once
#include "common.cuh"

namespace ft {

constexpr int kKv8Block = 16;                 // tokens that share a scale
constexpr float kKv8Least = 7.888609052210118e-31f;      // 2^-100: a block with nothing larger is a block of zeros (its scale's reciprocal has to be a number)

template <int D>
struct Kv8 {
    static constexpr int SLAB = kKvTile * D;              // codes of the keys (or values) of one page and head
    static constexpr int SCALES = 2 * SLAB;               // where the eight scales begin
    static constexpr int REC = 2 * SLAB + 32;
};

// Byte of a record at which 16-byte chunk c of token t begins
__device__ __forceinline__ int kv8_key_chunk(int t, int c) { return (c >> 2) * (kKvTile * 64) + t * 64 + (c & 3) * 16; }
template <int D>
__device__ __forceinline__ int kv8_value_chunk(int t, int c) {
    return Kv8<D>::SLAB + (c >> 2) * (kKvTile * 64) + (t ^ (t >> 1 & 1)) * 64 + (((c & 3) ^ (t >> 1 & 2)) << 4);
}

// Two of the four codes of a word, chosen by sel (bytes 0, 1: 0x4140; 2, 3: 0x4342), as fp16 numbers -128 .. 127, exactly: 0x64 above a byte is 1024 + the byte
__device__ __forceinline__ uint32_t kv8_pair(uint32_t w, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0x64646464u), "r"(sel));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(r), "r"(0x64806480u));
    return r;
}
__device__ __forceinline__ uint32_t kv8_lo(uint32_t w) { return kv8_pair(w, 0x4140); }
__device__ __forceinline__ uint32_t kv8_hi(uint32_t w) { return kv8_pair(w, 0x4342); }
__device__ __forceinline__ uint32_t byte_perm(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}

// ------------------------------------------------------------------ one query token a sequence, up to eight query heads a key head (mma.sync m16n8k16)
// A warp takes whole pages.  S[query][token] = Q K^T with the query heads in the M rows (rows 8 .. 15 are zeros), so that a lane holds one query's scores of two
// neighbouring tokens: exactly what the second product wants as its B operand, O^T[dim][query] = V^T P^T, where all 16 rows are dims.  The order of the dims in the
// first product is the lanes' (16 bytes of a token a lane), that of the dims in the second theirs too (8 neighbouring dims of each 64 a lane).
// Codes are multiplied as they are; the keys' scale goes to the scores, the values' to the probabilities, relative to the largest values' scale that the warp has
// seen (vref), or small values would leave fp16's range.
template <int D>
struct Kv8Query {
    uint32_t q[D / 16][2];      // A operand, rows 0 .. 7
    float o[D / 16][4];         // O^T / vref: dims 64 sub + 8 g + 2 i (+ 1), queries 2 tq (+ 1), at [4 sub + i][2 * (dim & 1) + (query & 1)]
    float m, l, vref;           // of query g: maximum in log2 units, sum

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        m = -INFINITY;
        l = vref = 0.f;
    }
    // row: query head g of the group, or null
    __device__ __forceinline__ void load_query(const __half* row, int tq) {
#pragma unroll
        for (int sub = 0; sub < D / 64; ++sub) {
            uint4 a = make_uint4(0u, 0u, 0u, 0u), b = a;
            if (row) {
                a = *reinterpret_cast<const uint4*>(row + sub * 64 + tq * 16);
                b = *reinterpret_cast<const uint4*>(row + sub * 64 + tq * 16 + 8);
            }
            const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) q[sub * 4 + k][0] = w[2 * k], q[sub * 4 + k][1] = w[2 * k + 1];
        }
    }
    // the first n (1 .. 64) tokens of the page at rec
    __device__ __forceinline__ void page(const uint8_t* rec, int n, float scale_log2, int g, int tq) {
        const float4 ks = *reinterpret_cast<const float4*>(rec + Kv8<D>::SCALES), vs = *reinterpret_cast<const float4*>(rec + Kv8<D>::SCALES + 16);
        const float kscale[4] = {ks.x * scale_log2, ks.y * scale_log2, ks.z * scale_log2, ks.w * scale_log2};
        float p[8][2], most = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int sub = 0; sub < D / 64; ++sub) {
                const uint4 w = *reinterpret_cast<const uint4*>(rec + kv8_key_chunk(8 * j + g, sub * 4 + tq));
                const uint32_t c[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) mma_f16_16816(s, q[sub * 4 + k][0], 0u, q[sub * 4 + k][1], 0u, kv8_lo(c[k]), kv8_hi(c[k]));
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                p[j][e] = 8 * j + 2 * tq + e < n ? s[e] * kscale[j >> 1] : -INFINITY;
                most = fmaxf(most, p[j][e]);
            }
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const float m_new = fmaxf(m, most);                          // finite: a page has a token
        const float v_new = fmaxf(vref, fmaxf(fmaxf(vs.x, vs.y), fmaxf(vs.z, vs.w)));
        const float v_inv = v_new > 0.f ? __fdividef(1.f, v_new) : 0.f;
        if (__any_sync(0xffffffffu, m_new > m || v_new > vref)) {    // after the first few pages rarely
            const float alpha = ex2_fast(m - m_new);
            const float keep = alpha * (vref * v_inv);
            l *= alpha;
            m = m_new;
            vref = v_new;
            const float k0 = __shfl_sync(0xffffffffu, keep, 8 * tq), k1 = __shfl_sync(0xffffffffu, keep, 8 * tq + 4);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[i][0] *= k0, o[i][1] *= k1, o[i][2] *= k0, o[i][3] *= k1;
        }
        const float vscale[4] = {vs.x * v_inv, vs.y * v_inv, vs.z * v_inv, vs.w * v_inv};
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {                             // a block of 16 tokens
            uint32_t b[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float p0 = ex2_fast(p[2 * kk + h][0] - m), p1 = ex2_fast(p[2 * kk + h][1] - m);
                l += p0 + p1;
                const __half2 t = __floats2half2_rn(p0 * vscale[kk], p1 * vscale[kk]);
                b[h] = *reinterpret_cast<const uint32_t*>(&t);
            }
#pragma unroll
            for (int sub = 0; sub < D / 64; ++sub) {
                uint2 t[4];                                          // tokens 2 tq, + 1, + 8, + 9
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    t[e] = *reinterpret_cast<const uint2*>(rec + kv8_value_chunk<D>(16 * kk + 2 * tq + (e & 1) + (e >> 1) * 8, sub * 4 + (g >> 1)) + (g & 1) * 8);
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const uint32_t t0 = w ? t[0].y : t[0].x, t1 = w ? t[1].y : t[1].x, t2 = w ? t[2].y : t[2].x, t3 = w ? t[3].y : t[3].x;
                    const uint32_t x = byte_perm(t0, t1, 0x5140), y = byte_perm(t0, t1, 0x7362), u = byte_perm(t2, t3, 0x5140), v = byte_perm(t2, t3, 0x7362);
                    mma_f16_16816(o[sub * 4 + 2 * w], kv8_lo(x), kv8_hi(x), kv8_lo(u), kv8_hi(u), b[0], b[1]);
                    mma_f16_16816(o[sub * 4 + 2 * w + 1], kv8_lo(y), kv8_hi(y), kv8_lo(v), kv8_hi(v), b[0], b[1]);
                }
            }
        }
    }
    // the warp's state as a record of eight query heads, O in its own size: [query][D | m | l]
    __device__ __forceinline__ void store(float* rec, int g, int tq) {
        float sum = l + __shfl_xor_sync(0xffffffffu, l, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float* at = rec + (size_t)(2 * tq + e) * (D + 2) + (i >> 2) * 64 + 8 * g + 2 * (i & 3);
                *reinterpret_cast<float2*>(at) = make_float2(o[i][e] * vref, o[i][2 + e] * vref);
            }
        if (tq == 0) *reinterpret_cast<float2*>(rec + (size_t)g * (D + 2) + D) = make_float2(m, sum);
    }
};

}  // namespace ft
