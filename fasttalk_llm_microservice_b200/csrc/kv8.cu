// Writing the 8-bit KV cache (kv8.cuh) as keys and values are formed, and reading it back.
//
// Append.  x = the sum of the projection's split-K parts, keys rotated; per block of 16 tokens, head and keys | values, with a = max |x| over the block's new
// rows and s_old the block's scale where it holds rows below the first new one (else 0):
//   s = max(s_old, a / 127);   rows below the first new one: c <- rint(c * (s_old / s));   new rows: c = rint(x / s)
// A token that fits under its block's scale is written as it is; one that does not rescales the at most 15 rows before it.  Each growth costs the older rows half
// a step more of rounding; a block written at once is rounded once.  NaN becomes 0 and what lies beyond fp16's range is cut to it, as far as the fp16 cache reaches.
//
// A warp takes the runs that begin among one (or four, where there are many tokens) of the list, for one head's keys or values; a run = neighbouring tokens that go
// to one block of one sequence.  Its rows stay in registers between the maximum and the rounding, so the projection is read once, all of it asked for before the
// first number is used: what bounds a prompt's portion is that reading.  1954 tokens of four sequences behind 1003 each, in two
// parts, 32 + 16 heads of 128 (116 MB): 24.8 us, 4.7 TB/s (with the rows read back 29, a row at a time 64); 64 single tokens, 32 + 16 heads of 64: 4.2 us, list, page and scale read one after the other.
#include <type_traits>

#include "common.cuh"
#include "ft_internal.h"
#include "kv8.cuh"

namespace ft {

constexpr int K8_WARPS = 8;
constexpr int K8_QHEADS = 8;                 // query heads a warp takes
constexpr int K8_MANY = 512;                 // tokens from which a warp looks at four of them: most of a prompt's begin no run, single ones all do.
                                             // Four against one, us, heads of 64: 1800 in portions of 300 10.7 / 15.6, 700 in one 6.5 / 8.6, 400 in portions of 100 6.2 / 7.2, 512 single 13.7 / 14.8, 64 single 10.9 / 4.1

struct Kv8Append {
    const float* qkv;
    size_t split_stride;
    const float *cos_t, *sin_t;
    const int *positions, *seq_rows, *page_table;
    __half* q_out;
    uint8_t* cache;
    int n_splits, T, table_rows, max_pages, num_pages, n_angles, nq, nkv, window;
};

__device__ __forceinline__ float kv8_in(float x) { return x != x ? 0.f : fminf(fmaxf(x, -65504.f), 65504.f); }

// N rows of the projection, their parts added up in order.  D / 4 lanes take a row, four neighbouring dims each; at(i) = where this lane's part of row i begins, null = no row
template <int N, class At>
__device__ __forceinline__ void kv8_rows(const Kv8Append& p, float4* x, At at) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < p.n_splits; ++s) {
        constexpr int M = N < 8 ? N : 8;     // asked for at once
#pragma unroll
        for (int b = 0; b < N; b += M) {
            float4 y[M];
#pragma unroll
            for (int i = 0; i < M; ++i) {
                const float* from = at(b + i);
                y[i] = from ? __ldcs(reinterpret_cast<const float4*>(from + s * p.split_stride)) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int i = 0; i < M; ++i) x[b + i].x += y[i].x, x[b + i].y += y[i].y, x[b + i].z += y[i].z, x[b + i].w += y[i].w;
        }
    }
}
// lo cos - hi sin | hi cos + lo sin; the partner of a rotated pair is half a row's lanes away.  c, s: of this lane's four pairs
template <int D>
__device__ __forceinline__ float4 kv8_rotate(float4 x, float4 c, float4 s, int sub) {
    constexpr int HL = D / 8;                // lanes of half a row
    float4 y;
    y.x = __shfl_xor_sync(0xffffffffu, x.x, HL);
    y.y = __shfl_xor_sync(0xffffffffu, x.y, HL);
    y.z = __shfl_xor_sync(0xffffffffu, x.z, HL);
    y.w = __shfl_xor_sync(0xffffffffu, x.w, HL);
    const float sign = sub < HL ? -1.f : 1.f;
    return make_float4(x.x * c.x + sign * y.x * s.x, x.y * c.y + sign * y.y * s.y, x.z * c.z + sign * y.z * s.z, x.w * c.w + sign * y.w * s.w);
}

template <int D>
__global__ void __launch_bounds__(K8_WARPS * 32, 2)
kv8_append_kernel(const Kv8Append p, int kv_rows, int kv_ctas) {
    pdl_wait();
    constexpr int LR = D / 4, RP = 32 / LR, N = kKv8Block / RP, HL = D / 8;      // lanes a row, rows a pass, passes; lanes of half a row
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sub = lane % LR, rsub = lane / LR;
    const size_t width = (size_t)(p.nq + 2 * p.nkv) * D;

    if ((int)blockIdx.x >= kv_ctas) {
        // ---------------- queries: rotated, to fp16.  A warp takes eight heads of a token
        const int groups = (p.nq + K8_QHEADS - 1) / K8_QHEADS;
        const unsigned task = (blockIdx.x - kv_ctas) * K8_WARPS + warp;
        const int t = (int)(task / groups), h0 = (int)(task % groups) * K8_QHEADS;
        if (t >= p.T) return;
        const int pos = p.positions[t];
        const bool on = pos >= 0 && pos < p.n_angles;
        const float4 c = load_f4(p.cos_t + (size_t)(on ? pos : 0) * (D / 2) + (sub % HL) * 4), s = load_f4(p.sin_t + (size_t)(on ? pos : 0) * (D / 2) + (sub % HL) * 4);
        const float* row = p.qkv + (size_t)t * width + sub * 4;
        float4 x[K8_QHEADS / RP];
        kv8_rows<K8_QHEADS / RP>(p, x, [&](int i) { return on && h0 + i * RP + rsub < p.nq ? row + (size_t)(h0 + i * RP + rsub) * D : nullptr; });
#pragma unroll
        for (int i = 0; i < K8_QHEADS / RP; ++i) {
            const int h = h0 + i * RP + rsub;
            const float4 y = kv8_rotate<D>(x[i], c, s, sub);
            if (h < p.nq)
                *reinterpret_cast<uint2*>(p.q_out + ((size_t)t * p.nq + h) * D + sub * 4) = make_uint2(pack_f16_sat(y.x, y.y), pack_f16_sat(y.z, y.w));
        }
        return;
    }

    const int task = (int)blockIdx.x % kv_rows * K8_WARPS + warp;    // head * 2 + (keys 0 | values 1)
    if (task >= 2 * p.nkv) return;
    const int kvh = task >> 1, is_v = task & 1, head = p.nq + (is_v ? p.nkv : 0) + kvh;
    // lane i: token t0 + i of the list, lane 31 the one before: which of the window's tokens begin a run?
    const int t0 = (int)blockIdx.x / kv_rows * p.window;
    int seq = -1, pos = -1;
    {
        const int u = lane == 31 ? t0 - 1 : t0 + lane;
        if (u >= 0 && u < p.T) seq = p.seq_rows[u], pos = p.positions[u];
    }
    const int blk = pos >> 4;
    const int before = (lane + 31) & 31;
    const int seq_before = __shfl_sync(0xffffffffu, seq, before), blk_before = __shfl_sync(0xffffffffu, blk, before);
    const bool begins = lane < p.window && t0 + lane < p.T && (t0 + lane == 0 || seq_before != seq || blk_before != blk);
    for (unsigned lead = __ballot_sync(0xffffffffu, begins); lead; lead &= lead - 1) {
        const int i0 = __ffs(lead) - 1;
        const int seq0 = __shfl_sync(0xffffffffu, seq, i0), blk0 = __shfl_sync(0xffffffffu, blk, i0);
        if (seq0 < 0 || seq0 >= p.table_rows || blk0 < 0 || blk0 >= p.max_pages * (kKvTile / kKv8Block)) continue;
        const int page = p.page_table[(size_t)seq0 * p.max_pages + (blk0 >> 2)];
        if (page < 0 || page >= p.num_pages) continue;
        uint8_t* rec = p.cache + ((size_t)page * p.nkv + kvh) * Kv8<D>::REC;
        float* scale = reinterpret_cast<float*>(rec + Kv8<D>::SCALES) + is_v * 4 + (blk0 & 3);
        const int row0 = (blk0 & 3) * kKv8Block;
        auto code_at = [&](int row) -> uint32_t* {                   // four codes of this lane
            const int at = is_v ? kv8_value_chunk<D>(row0 + row, sub >> 2) : kv8_key_chunk(row0 + row, sub >> 2);
            return reinterpret_cast<uint32_t*>(rec + at + (sub & 3) * 4);
        };
        unsigned held = 0;                                           // rows of the block that hold something
        // the run's positions, from lane `base` on; up to 16 at a time (a longer run names a row twice: the later token stands)
        int run_pos = pos, base = i0, first = t0 + i0;
        bool same = lane != 31 && t0 + lane < p.T && seq == seq0 && blk == blk0;
        for (;;) {
            const unsigned m = __ballot_sync(0xffffffffu, same) >> base;
            const int n = min(16, __ffs(~m) - 1);
            const float* row = p.qkv + (size_t)first * width + (size_t)head * D + sub * 4;
            float4 x[N];
            const float s_was = *scale;
            kv8_rows<N>(p, x, [&](int i) { return i * RP + rsub < n ? row + (size_t)(i * RP + rsub) * width : nullptr; });
            unsigned rows = 0, low = kKv8Block;
            float a = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = i * RP + rsub;
                const int ps = __shfl_sync(0xffffffffu, run_pos, base + r);
                const bool on = r < n && ps < p.n_angles;
                if (!is_v) {
                    const size_t at = (size_t)(on ? ps : 0) * (D / 2) + (sub % HL) * 4;
                    x[i] = kv8_rotate<D>(x[i], load_f4(p.cos_t + at), load_f4(p.sin_t + at), sub);
                }
                x[i] = make_float4(kv8_in(x[i].x), kv8_in(x[i].y), kv8_in(x[i].z), kv8_in(x[i].w));
                if (on) {
                    a = fmaxf(a, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
                    rows |= 1u << (ps & 15);
                    low = min(low, (unsigned)(ps & 15));
                }
            }
            a = warp_max(a);
            rows = __reduce_or_sync(0xffffffffu, rows);
            low = __reduce_min_sync(0xffffffffu, low);
            if (first == t0 + i0) held = (1u << low) - 1;
            if (__popc(rows) < n) {
                // a token whose row a later one of these 16 takes is not written: of two stores at once either could stand
                const unsigned like = __match_any_sync(0xffffffffu, lane >= base && lane < base + n ? run_pos : -1 - lane);
                if (like >> lane >> 1) run_pos = INT32_MAX;
            }
            if (rows) {
                const float s_old = held ? s_was : 0.f;
                const float s_new = a > kKv8Least ? a / 127.f : 0.f;
                const float s = fmaxf(s_old, s_new);
                const unsigned kept = held & ~rows;
                if (s > s_old && kept) {
                    const float f = s_old / s;
                    for (int r = rsub; r < kKv8Block; r += RP) {
                        if (!(kept >> r & 1)) continue;
                        uint32_t* at = code_at(r);
                        const uint32_t w = *at;
                        uint32_t y = 0;
#pragma unroll
                        for (int k = 0; k < 4; ++k) y |= (uint32_t)(__float2int_rn((float)((int)(w >> 8 * k & 255) - 128) * f) + 128) << 8 * k;
                        *at = y;
                    }
                }
                // rint(v / s) + 128 in the low byte: the product with the reciprocal, rounded to a whole number c by adding 1.5 * 2^23 (+ 128), is the quotient's own
                // unless that lies next to a border; then the remainder v - c s, which fp32 holds there, says on which side: |v - c s| > s / 2, or half
                // of it and c odd (numbers that are not negative order as their bits do).  A block of zeros may hold numbers below 2^-100: codes of 0.  A division for each
                // number was 1 us slower at 1954 tokens.
                const float inv = s > 0.f ? 1.f / s : 0.f, half = s > 0.f ? 0.5f * s : INFINITY;
                auto code = [&](float v) {
                    constexpr float shift = 12583040.f;
                    const float t = fmaf(v, inv, shift), rest = fmaf(shift - t, s, v);
                    return __float_as_uint(__float_as_uint(fabsf(rest)) + (__float_as_uint(t) & 1) > __float_as_uint(half) ? t + copysignf(1.f, rest) : t);
                };
                auto codes = [&](float4 v) { return byte_perm(byte_perm(code(v.x), code(v.y), 0x0040), byte_perm(code(v.z), code(v.w), 0x0040), 0x5410); };
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int r = i * RP + rsub;
                    const int ps = __shfl_sync(0xffffffffu, run_pos, base + r);
                    if (r < n && ps < p.n_angles) *code_at(ps & 15) = codes(x[i]);
                }
                __syncwarp();
                if (lane == 0) *scale = s;
                __syncwarp();
                held |= rows;
            }
            if (n < 16) break;
            first += 16;
            const int u = first + lane;
            base = 0;
            same = false;
            run_pos = -1;
            if (u < p.T) run_pos = p.positions[u], same = lane != 31 && p.seq_rows[u] == seq0 && (run_pos >> 4) == blk0;
            if (!__shfl_sync(0xffffffffu, (int)same, 0)) break;
        }
    }
}

// ------------------------------------------------------------------ reading back
// Row i of k and v: (c - 128) * s of the request that owns it, in fp16 (cut to its range); rows that no request owns, and rows whose page lies outside the
// cache, are zeros.  A CTA takes 16 rows of eight (sixteen) heads' keys or values: 16 bytes of codes a load, 32 bytes of fp16 a store, four loads on their way a
// thread.  Bound by memory (one byte in, two out): 16 sequences of 2048 .. 1987 tokens, 8 heads of 64 (99 MB): 16.8 us, 5.9 TB/s (the records partly out of L2, being the same each
// time); 5003 tokens of 8 heads of 128 (31 MB): 8.6 us, 3.6 TB/s, too short for more.  With one load at a time 23.7 (then 18.9) and 9.9 us.
constexpr int K8_READ_ROWS = 16, K8_READ_THREADS = 256, K8_READ_TASKS = 4;

template <int D>
__global__ void __launch_bounds__(K8_READ_THREADS)
kv8_read_kernel(const uint8_t* __restrict__ cache, const int* __restrict__ page_table, int table_rows, int max_pages, int num_pages,
                const int* __restrict__ req_start, const int* __restrict__ req_slot, const int* __restrict__ req_pos0, int n_req, int rows, int nkv,
                uint8_t* __restrict__ k_out, uint8_t* __restrict__ v_out) {
    pdl_wait();
    __shared__ int s_page[K8_READ_ROWS], s_tok[K8_READ_ROWS];
    const int row0 = blockIdx.x * K8_READ_ROWS;
    if (threadIdx.x < 32) {
        // lane i: row i; its request is the last that starts at or before it
        const int lane = threadIdx.x, row = row0 + lane;
        int r = -1;
        for (int b = 0; b < n_req; b += 32) {
            const int start = b + lane < n_req ? req_start[b + lane] : INT32_MAX;
#pragma unroll
            for (int i = 0; i < K8_READ_ROWS; ++i) {
                const int n = __popc(__ballot_sync(0xffffffffu, start <= row0 + i));
                if (lane == i) r += n;
            }
        }
        int page = -1, tok = 0;
        if (lane < K8_READ_ROWS && r >= 0 && row < rows) {
            const int start = req_start[r], end = req_start[r + 1], slot = req_slot[r];
            const long long pos = (long long)req_pos0[r] + row - start;
            if (row < end && pos >= 0 && pos < (long long)max_pages * kKvTile && slot >= 0 && slot < table_rows) {
                page = page_table[(size_t)slot * max_pages + (int)(pos / kKvTile)];
                if (page < 0 || page >= num_pages) page = -1;
                tok = (int)(pos % kKvTile);
            }
        }
        if (lane < K8_READ_ROWS) s_page[lane] = page, s_tok[lane] = tok;
    }
    __syncthreads();
    constexpr int CH = D / 16;                                       // chunks of a row
    uint4 w[K8_READ_TASKS];
    float s[K8_READ_TASKS];
    const int first = blockIdx.y * (K8_READ_TASKS * K8_READ_THREADS) + threadIdx.x;      // [head][keys | values][row][chunk]: neighbouring lanes read neighbouring rows of one record
#pragma unroll
    for (int k = 0; k < K8_READ_TASKS; ++k) {
        const int i = first + k * K8_READ_THREADS, c = i % CH, r = i / CH % K8_READ_ROWS, rest = i / (CH * K8_READ_ROWS), is_v = rest & 1, h = rest >> 1;
        const int page = s_page[r], t = s_tok[r];
        w[k] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
        s[k] = 0.f;
        if (page >= 0 && h < nkv) {
            const uint8_t* rec = cache + ((size_t)page * nkv + h) * Kv8<D>::REC;
            w[k] = __ldg(reinterpret_cast<const uint4*>(rec + (is_v ? kv8_value_chunk<D>(t, c) : kv8_key_chunk(t, c))));
            s[k] = __ldg(reinterpret_cast<const float*>(rec + Kv8<D>::SCALES) + is_v * 4 + (t >> 4));
        }
    }
#pragma unroll
    for (int k = 0; k < K8_READ_TASKS; ++k) {
        const int i = first + k * K8_READ_THREADS, c = i % CH, r = i / CH % K8_READ_ROWS, rest = i / (CH * K8_READ_ROWS), is_v = rest & 1, h = rest >> 1;
        if (h >= nkv || row0 + r >= rows) continue;
        uint32_t o[8];
        const uint32_t in[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            // a byte below 0x4b0000 is 2^23 and the byte: its code, exactly
            auto val = [&](uint32_t sel) { return (__uint_as_float(byte_perm(in[e], 0x4b000000u, sel)) - 8388736.f) * s[k]; };
            o[2 * e] = pack_f16_sat(val(0x7540), val(0x7541));
            o[2 * e + 1] = pack_f16_sat(val(0x7542), val(0x7543));
        }
        uint4* dst = reinterpret_cast<uint4*>((is_v ? v_out : k_out) + (((size_t)(row0 + r) * nkv + h) * D + c * 16) * 2);
        __stcs(dst, make_uint4(o[0], o[1], o[2], o[3]));
        __stcs(dst + 1, make_uint4(o[4], o[5], o[6], o[7]));
    }
}

static bool kv8_head_dim(int d) { return d == 64 || d == 128; }

}  // namespace ft

// ------------------------------------------------------------------ C ABI
extern "C" long long ft_kv8_record_bytes(int d) {
    FT_REQUIRE(ft::kv8_head_dim(d), "ft_kv8_record_bytes: head_dim %d not supported (64 or 128)", d);
    return 128LL * d + 32;
}

extern "C" int ft_rope_kv8_append(const float* qkv, int n_splits, long long split_stride, const float* cos_t, const float* sin_t, int n_angles,
                                  const int* positions, const int* seq_rows, const int* page_table, int table_rows, int max_pages, void* q_out,
                                  void* kv8_layer, int num_pages, int T, int nq, int nkv, int d, void* stream) {
    using namespace ft;
    FT_REQUIRE(kv8_head_dim(d), "ft_rope_kv8_append: head_dim %d not supported (64 or 128)", d);
    FT_REQUIRE(T >= 0 && nq >= 1 && nkv >= 1 && n_splits >= 1 && n_angles >= 0 && table_rows >= 0 && max_pages >= 0 && num_pages >= 0,
               "ft_rope_kv8_append: bad sizes T=%d nq=%d nkv=%d n_splits=%d n_angles=%d table %d x %d, %d pages", T, nq, nkv, n_splits, n_angles, table_rows,
               max_pages, num_pages);
    FT_REQUIRE(max_pages <= INT32_MAX / kKvTile - 1, "ft_rope_kv8_append: %d pages a sequence", max_pages);
    if (T == 0) return 0;
    FT_REQUIRE(qkv && cos_t && sin_t && positions && seq_rows && q_out && kv8_there(page_table, table_rows, max_pages, kv8_layer, num_pages), "ft_rope_kv8_append: null argument");
    FT_REQUIRE(n_angles >= 1, "ft_rope_kv8_append: no angles");
    FT_REQUIRE(((uintptr_t)qkv | (uintptr_t)cos_t | (uintptr_t)sin_t | (uintptr_t)q_out | (uintptr_t)kv8_layer) % 16 == 0 && split_stride % 4 == 0,
               "ft_rope_kv8_append: tensors on 16 bytes");
    const int window = T >= K8_MANY ? 4 : 1;
    Kv8Append p{qkv, (size_t)split_stride, cos_t, sin_t, positions, seq_rows, page_table, (__half*)q_out, (uint8_t*)kv8_layer, n_splits, T, table_rows, max_pages,
                num_pages, n_angles, nq, nkv, window};
    const long long kv_rows = (2LL * nkv + K8_WARPS - 1) / K8_WARPS, kv_ctas = (T + window - 1LL) / window * kv_rows;
    const long long q_tasks = (long long)T * ((nq + K8_QHEADS - 1) / K8_QHEADS), q_ctas = (q_tasks + K8_WARPS - 1) / K8_WARPS;
    FT_REQUIRE(q_tasks <= INT32_MAX && kv_ctas + q_ctas <= INT32_MAX, "ft_rope_kv8_append: %d tokens of %d + %d heads", T, nq, nkv);
    const int grid = (int)(kv_ctas + q_ctas);
    auto send = [&](auto head) {
        return launch_after(kv8_append_kernel<decltype(head)::value>, dim3(grid), dim3(K8_WARPS * 32), 0, (cudaStream_t)stream, p, (int)kv_rows, (int)kv_ctas);
    };
    FT_CHECK_CUDA(d == 64 ? send(std::integral_constant<int, 64>{}) : send(std::integral_constant<int, 128>{}));
    return 0;
}

extern "C" int ft_kv8_read(const void* kv8_layer, int num_pages, const int* page_table, int table_rows, int max_pages, const int* req_start,
                           const int* req_slot, const int* req_pos0, int n_req, int rows, void* k_out, void* v_out, int nkv, int d, void* stream) {
    using namespace ft;
    FT_REQUIRE(kv8_head_dim(d), "ft_kv8_read: head_dim %d not supported (64 or 128)", d);
    FT_REQUIRE(rows >= 0 && n_req >= 0 && nkv >= 1 && table_rows >= 0 && max_pages >= 0 && num_pages >= 0,
               "ft_kv8_read: bad sizes rows=%d n_req=%d nkv=%d table %d x %d, %d pages", rows, n_req, nkv, table_rows, max_pages, num_pages);
    if (rows == 0) return 0;
    FT_REQUIRE(k_out && v_out && (n_req == 0 || (req_start && req_slot && req_pos0 && kv8_there(page_table, table_rows, max_pages, kv8_layer, num_pages))), "ft_kv8_read: null argument");
    FT_REQUIRE(((uintptr_t)kv8_layer | (uintptr_t)k_out | (uintptr_t)v_out) % 16 == 0, "ft_kv8_read: tensors on 16 bytes");
    const long long tasks = (long long)nkv * 2 * K8_READ_ROWS * (d / 16), per = K8_READ_TASKS * K8_READ_THREADS;
    FT_REQUIRE((tasks + per - 1) / per <= 65535, "ft_kv8_read: %d heads", nkv);
    const dim3 grid((rows + K8_READ_ROWS - 1) / K8_READ_ROWS, (unsigned)((tasks + per - 1) / per));
    auto send = [&](auto head) {
        return launch_after(kv8_read_kernel<decltype(head)::value>, grid, dim3(K8_READ_THREADS), 0, (cudaStream_t)stream, (const uint8_t*)kv8_layer, page_table, table_rows,
                            max_pages, num_pages, req_start, req_slot, req_pos0, n_req, rows, nkv, (uint8_t*)k_out, (uint8_t*)v_out);
    };
    FT_CHECK_CUDA(d == 64 ? send(std::integral_constant<int, 64>{}) : send(std::integral_constant<int, 128>{}));
    return 0;
}
