// Writing the 8-bit KV cache (kv8.cuh) as keys and values are formed, and reading it back.
//
// Append.  x = the sum of the projection's split-K parts, keys rotated; per block of 16 tokens, head and keys | values, with a = max |x| over the block's new
// rows and s_old the block's scale where it holds rows below the first new one (else 0):
//   s = max(s_old, a / 127);   rows below the first new one: c <- rint(c * s_old / s);   new rows: c = rint(x / s)
// A token that fits under its block's scale is written as it is; one that does not rescales the at most 15 rows before it.  Each growth costs the older rows half
// a step more of rounding; a block written at once is rounded once.  NaN becomes 0 and what lies beyond fp16's range is cut to it, as far as the fp16 cache reaches.
//
// A warp takes one (run, head, keys | values); a run = neighbouring tokens of the list that go to one block of one sequence.  Its rows stay in registers between
// the maximum and the rounding, so the projection is read once.
#include "common.cuh"
#include "ft_internal.h"
#include "kv8.cuh"

namespace ft {

constexpr int K8_WARPS = 8;
constexpr int K8_QHEADS = 2;                 // query heads a warp takes

struct Kv8Append {
    const float* qkv;
    size_t split_stride;
    const float *cos_t, *sin_t;
    const int *positions, *seq_rows, *page_table;
    __half* q_out;
    uint8_t* cache;
    int n_splits, T, table_rows, max_pages, num_pages, n_angles, nq, nkv;
};

__device__ __forceinline__ float kv8_in(float x) { return x != x ? 0.f : fminf(fmaxf(x, -65504.f), 65504.f); }

// D / 4 lanes take a row, four neighbouring dims each; the partner of a rotated pair is half a row's lanes away
template <int D>
__device__ __forceinline__ float4 kv8_row(const Kv8Append& p, int t, int head, int sub) {
    const float* at = p.qkv + (size_t)t * (p.nq + 2 * p.nkv) * D + (size_t)head * D + sub * 4;
    float4 x = __ldcg(reinterpret_cast<const float4*>(at));
    for (int s = 1; s < p.n_splits; ++s) {
        const float4 y = __ldcg(reinterpret_cast<const float4*>(at + s * p.split_stride));
        x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
    }
    return x;
}
template <int D>
__device__ __forceinline__ float4 kv8_rotate(float4 x, const Kv8Append& p, int pos, int sub) {
    constexpr int HL = D / 8;                 // lanes of half a row
    const float4 c = load_f4(p.cos_t + (size_t)pos * (D / 2) + (sub % HL) * 4), s = load_f4(p.sin_t + (size_t)pos * (D / 2) + (sub % HL) * 4);
    float4 y;
    y.x = __shfl_xor_sync(0xffffffffu, x.x, HL);
    y.y = __shfl_xor_sync(0xffffffffu, x.y, HL);
    y.z = __shfl_xor_sync(0xffffffffu, x.z, HL);
    y.w = __shfl_xor_sync(0xffffffffu, x.w, HL);
    const float sign = sub < HL ? -1.f : 1.f;  // lo cos - hi sin | hi cos + lo sin
    return make_float4(x.x * c.x + sign * y.x * s.x, x.y * c.y + sign * y.y * s.y, x.z * c.z + sign * y.z * s.z, x.w * c.w + sign * y.w * s.w);
}

template <int D>
__global__ void __launch_bounds__(K8_WARPS * 32)
kv8_append_kernel(const Kv8Append p, int kv_rows) {
    constexpr int LR = D / 4, RP = 32 / LR, N = kKv8Block / RP;      // lanes a row, rows a pass, passes
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sub = lane % LR, rsub = lane / LR;
    const int angles = min(p.n_angles, p.max_pages * kKvTile);

    if ((int)blockIdx.y >= kv_rows) {
        // ---------------- queries: rotated, to fp16
        const int pos = p.positions[t];
        const int h0 = (((int)blockIdx.y - kv_rows) * K8_WARPS + warp) * K8_QHEADS;
#pragma unroll
        for (int i = 0; i < K8_QHEADS; i += RP) {
            const int h = h0 + i + rsub;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            const bool on = h < p.nq && pos >= 0 && pos < angles;
            if (on) x = kv8_row<D>(p, t, h, sub);
            x = kv8_rotate<D>(x, p, on ? pos : 0, sub);
            if (h < p.nq)
                *reinterpret_cast<uint2*>(p.q_out + ((size_t)t * p.nq + h) * D + sub * 4) = make_uint2(pack_f16_sat(x.x, x.y), pack_f16_sat(x.z, x.w));
        }
        return;
    }

    const int task = blockIdx.y * K8_WARPS + warp;                   // head * 2 + (keys 0 | values 1)
    if (task >= 2 * p.nkv) return;
    const int kvh = task >> 1, is_v = task & 1;
    // lane i: token t + i of the list; the lane before the run's first token says whether it is a run's first
    int u = t + lane, seq = -1, pos = -1;
    if (lane == 31) u = t - 1;
    if (u >= 0 && u < p.T) seq = p.seq_rows[u], pos = p.positions[u];
    const int seq0 = __shfl_sync(0xffffffffu, seq, 0), blk0 = __shfl_sync(0xffffffffu, pos, 0) >> 4;
    bool same = u >= 0 && u < p.T && seq == seq0 && (pos >> 4) == blk0;
    if (__ballot_sync(0xffffffffu, same) >> 31) return;              // the token before t goes to the same block: its warp takes this one too
    if (seq0 < 0 || seq0 >= p.table_rows || blk0 < 0 || blk0 >= p.max_pages * (kKvTile / kKv8Block)) return;
    const int page = p.page_table[(size_t)seq0 * p.max_pages + (blk0 >> 2)];
    if (page < 0 || page >= p.num_pages) return;
    uint8_t* rec = p.cache + ((size_t)page * p.nkv + kvh) * Kv8<D>::REC;
    float* scale = reinterpret_cast<float*>(rec + Kv8<D>::SCALES) + is_v * 4 + (blk0 & 3);
    const int head = p.nq + (is_v ? p.nkv : 0) + kvh;
    const int row0 = (blk0 & 3) * kKv8Block;
    auto code_at = [&](int row) -> uint32_t* {                       // four codes of this lane
        const int at = is_v ? kv8_value_chunk<D>(row0 + row, sub >> 2) : kv8_key_chunk(row0 + row, sub >> 2);
        return reinterpret_cast<uint32_t*>(rec + at + (sub & 3) * 4);
    };

    unsigned held = 0;                                               // rows of the block that hold something
    for (int first = t;;) {
        // up to 16 tokens of the run; a longer one names a row twice: the later token stands
        const unsigned m = __ballot_sync(0xffffffffu, lane < 16 && same);
        const int n = __ffs(~m) - 1;
        float4 x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = i * RP + rsub;
            x[i] = r < n ? kv8_row<D>(p, first + r, head, sub) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        unsigned rows = 0, low = kKv8Block;
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = i * RP + rsub;
            const int ps = __shfl_sync(0xffffffffu, pos, r);
            if (!is_v) x[i] = kv8_rotate<D>(x[i], p, r < n && ps < angles ? ps : 0, sub);
            x[i] = make_float4(kv8_in(x[i].x), kv8_in(x[i].y), kv8_in(x[i].z), kv8_in(x[i].w));
            if (r < n && ps < angles) {
                a = fmaxf(a, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
                rows |= 1u << (ps & 15);
                low = min(low, (unsigned)(ps & 15));
            }
        }
        a = warp_max(a);
        rows = __reduce_or_sync(0xffffffffu, rows);
        low = __reduce_min_sync(0xffffffffu, low);
        if (first == t) held = (1u << low) - 1;
        if (rows) {
            const float s_old = held ? *scale : 0.f;
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
                    for (int b = 0; b < 4; ++b) y |= (uint32_t)(__float2int_rn((float)((int)(w >> 8 * b & 255) - 128) * f) + 128) << 8 * b;
                    *at = y;
                }
            }
            const float inv = s > 0.f ? 1.f / s : 0.f;
            auto code = [&](float v) { return (uint32_t)(max(-127, min(127, __float2int_rn(v * inv))) + 128); };
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = i * RP + rsub;
                const int ps = __shfl_sync(0xffffffffu, pos, r);
                if (r < n && ps < angles) *code_at(ps & 15) = code(x[i].x) | code(x[i].y) << 8 | code(x[i].z) << 16 | code(x[i].w) << 24;
            }
            __syncwarp();
            if (lane == 0) *scale = s;
            __syncwarp();
            held |= rows;
        }
        // what the run has beyond these 16
        if (n < 16) return;
        first += 16;
        u = first + lane;
        same = lane < 16 && u < p.T;
        if (same) seq = p.seq_rows[u], pos = p.positions[u];
        same = same && seq == seq0 && (pos >> 4) == blk0;
        if (!__shfl_sync(0xffffffffu, (int)same, 0)) return;
    }
}

// ------------------------------------------------------------------ reading back
// Row i of k and v: (c - 128) * s of the request that owns it, in fp16 (cut to its range); rows that no request owns, and rows whose page lies outside the
// cache, are zeros.  A CTA takes 16 rows of all heads: 16 bytes of codes a load, 32 bytes of fp16 a store, bound by memory (one byte in, two out).
constexpr int K8_READ_ROWS = 16, K8_READ_THREADS = 256;

template <int D>
__global__ void __launch_bounds__(K8_READ_THREADS)
kv8_read_kernel(const uint8_t* __restrict__ cache, const int* __restrict__ page_table, int table_rows, int max_pages, int num_pages,
                const int* __restrict__ req_start, const int* __restrict__ req_slot, const int* __restrict__ req_pos0, int n_req, int rows, int nkv,
                uint8_t* __restrict__ k_out, uint8_t* __restrict__ v_out) {
    __shared__ int s_page[K8_READ_ROWS], s_tok[K8_READ_ROWS];
    const int row0 = blockIdx.x * K8_READ_ROWS;
    if (threadIdx.x < K8_READ_ROWS) {
        const int row = row0 + threadIdx.x;
        int page = -1, tok = 0;
        int lo = 0, hi = n_req;                                      // the last request that starts at or before this row
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (req_start[mid] <= row) lo = mid + 1; else hi = mid;
        }
        const int r = lo - 1;
        if (r >= 0 && row < req_start[r + 1] && row < rows) {
            const long long pos = (long long)req_pos0[r] + row - req_start[r];
            const int slot = req_slot[r];
            if (pos >= 0 && pos < (long long)max_pages * kKvTile && slot >= 0 && slot < table_rows) {
                page = page_table[(size_t)slot * max_pages + (int)(pos / kKvTile)];
                if (page < 0 || page >= num_pages) page = -1;
                tok = (int)(pos % kKvTile);
            }
        }
        s_page[threadIdx.x] = page;
        s_tok[threadIdx.x] = tok;
    }
    __syncthreads();
    constexpr int CH = D / 16;                                       // chunks of a row
    const int n = min(rows - row0, K8_READ_ROWS);
    const int tasks = n * nkv * 2 * CH;
    for (int i = threadIdx.x; i < tasks; i += K8_READ_THREADS) {
        // chunk fastest, then row, so that neighbouring lanes read neighbouring rows of one record
        const int c = i % CH, r = i / CH % n, rest = i / CH / n, is_v = rest & 1, h = rest >> 1;
        const int page = s_page[r], t = s_tok[r];
        uint4 w = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
        float s = 0.f;
        if (page >= 0) {
            const uint8_t* rec = cache + ((size_t)page * nkv + h) * Kv8<D>::REC;
            w = *reinterpret_cast<const uint4*>(rec + (is_v ? kv8_value_chunk<D>(t, c) : kv8_key_chunk(t, c)));
            s = reinterpret_cast<const float*>(rec + Kv8<D>::SCALES)[is_v * 4 + (t >> 4)];
        }
        uint32_t o[8];
        const uint32_t in[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            auto val = [&](int b) { return (float)((int)(in[k] >> 8 * b & 255) - 128) * s; };
            o[2 * k] = pack_f16_sat(val(0), val(1));
            o[2 * k + 1] = pack_f16_sat(val(2), val(3));
        }
        uint4* dst = reinterpret_cast<uint4*>((is_v ? v_out : k_out) + (((size_t)(row0 + r) * nkv + h) * D + c * 16) * 2);
        dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
        dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
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
    FT_REQUIRE(qkv && cos_t && sin_t && positions && seq_rows && page_table && q_out && kv8_layer, "ft_rope_kv8_append: null argument");
    FT_REQUIRE(n_angles >= 1, "ft_rope_kv8_append: no angles");
    FT_REQUIRE(((uintptr_t)qkv | (uintptr_t)cos_t | (uintptr_t)sin_t | (uintptr_t)q_out | (uintptr_t)kv8_layer) % 16 == 0 && split_stride % 4 == 0,
               "ft_rope_kv8_append: tensors on 16 bytes");
    Kv8Append p{qkv, (size_t)split_stride, cos_t, sin_t, positions, seq_rows, page_table, (__half*)q_out, (uint8_t*)kv8_layer, n_splits, T, table_rows, max_pages,
                num_pages, n_angles, nq, nkv};
    const int kv_rows = (2 * nkv + K8_WARPS - 1) / K8_WARPS, q_rows = (nq + K8_WARPS * K8_QHEADS - 1) / (K8_WARPS * K8_QHEADS);
    FT_REQUIRE(kv_rows + q_rows <= 65535, "ft_rope_kv8_append: %d + %d heads", nq, nkv);
    const dim3 grid(T, kv_rows + q_rows);
    if (d == 64) kv8_append_kernel<64><<<grid, K8_WARPS * 32, 0, (cudaStream_t)stream>>>(p, kv_rows);
    else kv8_append_kernel<128><<<grid, K8_WARPS * 32, 0, (cudaStream_t)stream>>>(p, kv_rows);
    FT_CHECK_CUDA(cudaGetLastError());
    return 0;
}

extern "C" int ft_kv8_read(const void* kv8_layer, int num_pages, const int* page_table, int table_rows, int max_pages, const int* req_start,
                           const int* req_slot, const int* req_pos0, int n_req, int rows, void* k_out, void* v_out, int nkv, int d, void* stream) {
    using namespace ft;
    FT_REQUIRE(kv8_head_dim(d), "ft_kv8_read: head_dim %d not supported (64 or 128)", d);
    FT_REQUIRE(rows >= 0 && n_req >= 0 && nkv >= 1 && table_rows >= 0 && max_pages >= 0 && num_pages >= 0,
               "ft_kv8_read: bad sizes rows=%d n_req=%d nkv=%d table %d x %d, %d pages", rows, n_req, nkv, table_rows, max_pages, num_pages);
    if (rows == 0) return 0;
    FT_REQUIRE(k_out && v_out && kv8_layer && (n_req == 0 || (req_start && req_slot && req_pos0 && page_table)), "ft_kv8_read: null argument");
    FT_REQUIRE(((uintptr_t)kv8_layer | (uintptr_t)k_out | (uintptr_t)v_out) % 16 == 0, "ft_kv8_read: tensors on 16 bytes");
    FT_REQUIRE((long long)nkv * d * 2 * K8_READ_ROWS / 16 <= INT32_MAX, "ft_kv8_read: %d heads", nkv);
    const int grid = (rows + K8_READ_ROWS - 1) / K8_READ_ROWS;
    auto go = [&](auto kernel) {
        kernel<<<grid, K8_READ_THREADS, 0, (cudaStream_t)stream>>>((const uint8_t*)kv8_layer, page_table, table_rows, max_pages, num_pages, req_start, req_slot, req_pos0,
                                                                   n_req, rows, nkv, (uint8_t*)k_out, (uint8_t*)v_out);
    };
    if (d == 64) go(kv8_read_kernel<64>);
    else go(kv8_read_kernel<128>);
    FT_CHECK_CUDA(cudaGetLastError());
    return 0;
}
