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

// What both attention kernels keep of a query, in log2 units: m = a maximum of its scores, for the sum of probabilities in fp32; h = one of score + log2(value scale), for the
// weights p * scale in fp16.  These are formed 2^7 / 2^h of their size: below 2^15 until h has grown by 2^8, and fp16's normal numbers reach down to 2^-21 of the largest.
// m may lag by 2^30.  h is kept at or above m - 100, or a query whose weight lies on zeros would divide by nothing: values below 2^-100 of 1 count as zeros there.
constexpr float kKv8Top = 7.f, kKv8GrowH = 8.f, kKv8GrowM = 30.f, kKv8Low = 100.f;

template <int D>
struct Kv8 {
    static constexpr int SLAB = kKvTile * D;              // codes of the keys (or values) of one page and head
    static constexpr int SCALES = 2 * SLAB;               // where the eight scales begin
    static constexpr int REC = 2 * SLAB + 32;
};

// A page table without rows or pages, and a cache without pages, may be null: nothing is read there
inline bool kv8_there(const void* page_table, int table_rows, int max_pages, const void* layer, int num_pages) {
    return (page_table || table_rows == 0 || max_pages == 0) && (layer || num_pages == 0);
}

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

// Waits that end, as those of common.cuh do, with the number of tries as an argument (ft_kv8_set_wait_limit) and a few instructions each: the prompt kernel has some
// twenty of them among five kinds of warps, and its time hangs on what the instruction caches hold (unrolled, they and the rest were 104 KB, and 16 KB more or less of
// waits outside the loops over pages was 8 % of its time).  Who gives up touches none of the barriers again: what it skipped would make it take one phase for another.
__device__ __forceinline__ bool kv8_mbar_wait_limited(uint64_t* bar, uint32_t parity, volatile int* dead, int limit) {
#pragma unroll 1
    for (int i = 0; i < limit; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*dead) return false;
    }
    *dead = 1;
    return false;
}
// What must have ended before the memory that it writes is given back, however the CTA ends: the copies of a ring's last phases
__device__ __forceinline__ void kv8_copies_landed(uint64_t* full, int stages, int asked) {
#pragma unroll 1
    for (int i = max(0, asked - stages); i < asked; ++i)
#pragma unroll 1
        for (int k = 0; k < kWaitLimit && !mbar_try_wait(&full[i % stages], i / stages & 1); ++k) {}
}

// ------------------------------------------------------------------ one query token a sequence, up to eight query heads a key head (mma.sync m16n8k16)
// A warp takes whole pages.  S[token][query] = K Q^T with 16 tokens in the M rows: K is the A operand, 16 bytes of two tokens a lane, in whatever order of the dims the
// lanes have them (Q is loaded in the same).  The probabilities, transposed 8 x 8 at a time, are the B operand of O^T[dim][query] = V^T P^T, where all 16 rows are dims:
// 8 neighbouring ones of each 64 a lane.  (With the queries in the rows of the first product nothing is transposed, but half the rows are zeros: 32 products a page
// instead of 16 at D = 64, and their operands put together by 200 moves.)
// Codes are multiplied as they are; the keys' scale goes to the exponents, the values' to the probabilities.  Such a weight p * scale is rounded to fp16 relative to the
// largest of its query so far (kKv8Top above): neither a large value without weight nor a key without a value takes another's bits.
template <int D>
struct Kv8Query {
    uint32_t q[D / 16][2];      // B operand
    float o[D / 16][4];         // O^T times r: dims 64 sub + 8 g + 2 i (+ 1), queries 2 tq (+ 1), at [4 sub + i][2 * (dim & 1) + (query & 1)]
    float m[2], h[2], r[2], l[2];       // of queries 2 tq (+ 1): the references, 2^(m - h + 7), this lane's tokens' sum

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        m[0] = m[1] = h[0] = h[1] = -INFINITY;
        r[0] = r[1] = 1.f;
        l[0] = l[1] = 0.f;
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
        const float4 k4 = *reinterpret_cast<const float4*>(rec + Kv8<D>::SCALES);
        float4 vs = *reinterpret_cast<const float4*>(rec + Kv8<D>::SCALES + 16);
        const float ks[4] = {k4.x * scale_log2, k4.y * scale_log2, k4.z * scale_log2, k4.w * scale_log2};
        float s[4][4], most[2] = {-INFINITY, -INFINITY}, heavy[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int b = 0; b < 4; ++b) {                                // a block of 16 tokens
            s[b][0] = s[b][1] = s[b][2] = s[b][3] = 0.f;
#pragma unroll
            for (int sub = 0; sub < D / 64; ++sub) {
                const uint4 w0 = *reinterpret_cast<const uint4*>(rec + kv8_key_chunk(16 * b + g, sub * 4 + tq));
                const uint4 w1 = *reinterpret_cast<const uint4*>(rec + kv8_key_chunk(16 * b + 8 + g, sub * 4 + tq));
                const uint32_t c0[4] = {w0.x, w0.y, w0.z, w0.w}, c1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) mma_f16_16816(s[b], kv8_lo(c0[k]), kv8_lo(c1[k]), kv8_hi(c0[k]), kv8_hi(c1[k]), q[sub * 4 + k][0], q[sub * 4 + k][1]);
            }
        }
        if (n < kKvTile) {
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[b][e] = 16 * b + 8 * (e >> 1) + g < n ? s[b][e] : -INFINITY;
            // blocks behind the last token: whatever their scales are, nothing comes of it (the keys' meets minus infinity alone)
            if (n <= 16) vs.y = 0.f;
            if (n <= 32) vs.z = 0.f;
            if (n <= 48) vs.w = 0.f;
        }
        const float vscale[4] = {vs.x, vs.y, vs.z, vs.w}, vl[4] = {__log2f(fabsf(vs.x)), __log2f(fabsf(vs.y)), __log2f(fabsf(vs.z)), __log2f(fabsf(vs.w))};
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const float f = fmaxf(ks[b], 1e-37f);                    // a block of zeros: hidden scores stay minus infinity
            const float t0 = fmaxf(s[b][0], s[b][2]) * f, t1 = fmaxf(s[b][1], s[b][3]) * f;
            most[0] = fmaxf(most[0], t0);
            most[1] = fmaxf(most[1], t1);
            heavy[0] = fmaxf(heavy[0], t0 + vl[b]);
            heavy[1] = fmaxf(heavy[1], t1 + vl[b]);
        }
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                most[e] = fmaxf(most[e], __shfl_xor_sync(0xffffffffu, most[e], x));
                heavy[e] = fmaxf(heavy[e], __shfl_xor_sync(0xffffffffu, heavy[e], x));
            }
        }
        const bool grown = most[0] > m[0] + kKv8GrowM || most[1] > m[1] + kKv8GrowM || heavy[0] > h[0] + kKv8GrowH || heavy[1] > h[1] + kKv8GrowH;
        if (__any_sync(0xffffffffu, grown)) {                        // after the first few pages rarely
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float m_new = fmaxf(m[e], most[e]);            // finite: a page has a token
                const float h_new = fmaxf(fmaxf(h[e], heavy[e]), m_new - kKv8Low);
                const float keep = ex2_fast(h[e] - h_new);
                l[e] *= ex2_fast(m[e] - m_new);
                m[e] = m_new;
                h[e] = h_new;
                r[e] = ex2_fast(m_new - h_new + kKv8Top);
#pragma unroll
                for (int i = 0; i < D / 16; ++i) o[i][e] *= keep, o[i][2 + e] *= keep;
            }
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const float f = fmaxf(ks[b], 1e-37f);
            const float p0 = ex2_fast(fmaf(s[b][0], f, -m[0])), p1 = ex2_fast(fmaf(s[b][1], f, -m[1]));
            const float p2 = ex2_fast(fmaf(s[b][2], f, -m[0])), p3 = ex2_fast(fmaf(s[b][3], f, -m[1]));
            const float g0 = vscale[b] * r[0], g1 = vscale[b] * r[1];
            l[0] += p0 + p2;
            l[1] += p1 + p3;
            uint32_t pb[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const __half2 t = h ? __floats2half2_rn(p2 * g0, p3 * g1) : __floats2half2_rn(p0 * g0, p1 * g1);
                asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(pb[h]) : "r"(*reinterpret_cast<const uint32_t*>(&t)));
            }
#pragma unroll
            for (int sub = 0; sub < D / 64; ++sub) {
                uint2 t[4];                                          // tokens 2 tq, + 1, + 8, + 9
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    t[e] = *reinterpret_cast<const uint2*>(rec + kv8_value_chunk<D>(16 * b + 2 * tq + (e & 1) + (e >> 1) * 8, sub * 4 + (g >> 1)) + (g & 1) * 8);
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const uint32_t t0 = w ? t[0].y : t[0].x, t1 = w ? t[1].y : t[1].x, t2 = w ? t[2].y : t[2].x, t3 = w ? t[3].y : t[3].x;
                    const uint32_t x = byte_perm(t0, t1, 0x5140), y = byte_perm(t0, t1, 0x7362), u = byte_perm(t2, t3, 0x5140), v = byte_perm(t2, t3, 0x7362);
                    mma_f16_16816(o[sub * 4 + 2 * w], kv8_lo(x), kv8_hi(x), kv8_lo(u), kv8_hi(u), pb[0], pb[1]);
                    mma_f16_16816(o[sub * 4 + 2 * w + 1], kv8_lo(y), kv8_hi(y), kv8_lo(v), kv8_hi(v), pb[0], pb[1]);
                }
            }
        }
    }
    // the warp's state as a record of eight query heads, O in its own size: [query][D | m | l]
    __device__ __forceinline__ void store(float* rec, int g, int tq) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float sum = l[e];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            const float size = 1.f / r[e];
            float* at = rec + (size_t)(2 * tq + e) * (D + 2);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) *reinterpret_cast<float2*>(at + (i >> 2) * 64 + 8 * g + 2 * (i & 3)) = make_float2(o[i][e] * size, o[i][2 + e] * size);
            if (g == 0) *reinterpret_cast<float2*>(at + D) = make_float2(m[e], sum);
        }
    }
};

}  // namespace ft
