// The lists of one step, built on the GPU from the requests' lengths: in their order, request r with c_r tokens in the cache and n_r new ones takes
//   m_r = min(n_r, room in its row of the page table, tokens that its last page and the pool's pages that are left hold, tokens that the budget leaves),
// ceil((c_r + m_r) / 64) - ceil(c_r / 64) pages come from the pool, and every token gets its position, its row of the page table and its place in the cache.
//
// Taken one request after the other this is a chain, but both cuts have closed forms over two prefix sums.  Let w_r be the pages that r's tokens want (cut by its row
// alone) and P_r their sum over the requests ahead: the pool has max(0, F - P_r) pages left for r, since who is cut by the pool takes all that is left.  With the tokens
// cut so and S_r their sum ahead, the budget leaves max(0, budget - S_r), and nobody behind the one that it cuts gets any; so P_r is also where r's pages begin.
//
// What bounds it: latency alone (a launch, two rounds of reads, two scans, a search, a store).  Every CTA makes the scans for itself, one request a thread, which costs less
// than a kernel ahead of this one, and then looks up 512 tokens and writes its part of the table.  Measured in a graph: 64 requests of one token 4.5 us, 21 with 4419 tokens of a
// budget of 8192 4.4, 1021 with 28977 of one of 65536 6.4 (CTAs of 256: 4.5, 4.4, 8.3; of 1024: 5.9, 5.8, 7.2); a call after another takes 12, the host's time.
#include "common.cuh"
#include "ft_internal.h"

namespace ft {

constexpr int SL_THREADS = 512, SL_WARPS = SL_THREADS / 32;
constexpr int SL_MAX_REQUESTS = 8192;
constexpr int SL_NONE = -1;

struct StepRequest { int start, cached, slot, pages; };        // its first token of the step, its first page of those taken

// Exclusive sums over the block's threads; `all` is the sum of all
__device__ __forceinline__ long long block_before(long long mine, long long* warp_s, long long& all) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    long long x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += up;
    }
    __syncthreads();                                           // the last call's sums have been read
    if (lane == 31) warp_s[warp] = x;
    __syncthreads();
    long long w = lane < SL_WARPS ? warp_s[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += up;
    }
    all = __shfl_sync(0xffffffffu, w, 31);
    const long long ahead = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
    return x - mine + (warp ? ahead : 0);
}

__global__ void __launch_bounds__(SL_THREADS)
step_lists_kernel(const int* __restrict__ cached_lens, const int* __restrict__ new_lens, const int* __restrict__ req_slot, int R, int* page_table, int table_rows,
                  int max_pages, const int* __restrict__ free_pages, int n_free, const int* first_free, int budget, int hash, int* __restrict__ req_start,
                  int* __restrict__ ctx_lens, int* __restrict__ positions, int* __restrict__ seq_rows, int* __restrict__ kv_slots, int* taken) {
    pdl_wait();
    extern __shared__ __align__(16) uint8_t smem[];
    StepRequest* req = reinterpret_cast<StepRequest*>(smem);
    int* owner = reinterpret_cast<int*>(req + R);              // [hash]: the first request of each row of the table
    __shared__ long long warp_s[SL_WARPS];
    const int tid = threadIdx.x;
    const int chunk = (R + SL_THREADS - 1) / SL_THREADS, r0 = min(R, tid * chunk), r1 = min(R, r0 + chunk);
    const int reach = max_pages * kKvTile;                     // tokens that a row has room for (the host has seen that 32 bits hold them)
    const int first = first_free ? max(0, min(*first_free, n_free)) : 0, pool = n_free - first;

    // of several requests with the same row the first has it; the others get nothing
    for (int i = tid; i < hash; i += SL_THREADS) owner[i] = INT_MAX;
    for (int r = r0; r < r1; ++r) {
        const int slot = req_slot ? req_slot[r] : r;
        req[r].slot = slot >= 0 && slot < table_rows ? slot : SL_NONE;
        req[r].cached = max(0, min(cached_lens[r], reach));
    }
    __syncthreads();
    auto place = [&](int slot) { return (int)((unsigned)slot * 2654435761u >> 16) & (hash - 1); };
    if (req_slot) {
        for (int r = r0; r < r1; ++r) {
            const int slot = req[r].slot;
            if (slot == SL_NONE) continue;
            for (int h = place(slot);; h = (h + 1) & (hash - 1)) {        // (at most half of the places are taken)
                const int before = atomicCAS(&owner[h], INT_MAX, r);
                if (before == INT_MAX) break;
                if (req[before].slot == slot) {                           // (whoever of a row's requests is in a place, the row is the same)
                    atomicMin(&owner[h], r);
                    break;
                }
            }
        }
        __syncthreads();
    }
    auto wanted = [&](int r) {                                            // tokens that its row has room for
        const int slot = req[r].slot, c = req[r].cached;
        if (slot == SL_NONE) return 0;
        if (req_slot) {
            int h = place(slot);
            while (req[owner[h]].slot != slot) h = (h + 1) & (hash - 1);
            if (owner[h] != r) return 0;
        }
        return max(0, min(new_lens[r], reach - c));
    };
    auto pages_of = [](int tokens) { return (tokens + kKvTile - 1) / kKvTile; };

    long long want = 0, all, tokens = 0;
    for (int r = r0; r < r1; ++r) {
        const int n = wanted(r);
        req[r].start = n;                                                 // (until the sums are known)
        want += pages_of(req[r].cached + n) - pages_of(req[r].cached);
    }
    long long P = block_before(want, warp_s, all);
    for (int r = r0; r < r1; ++r) {
        const int c = req[r].cached, held = pages_of(c), n = req[r].start, w = pages_of(c + n) - held;
        const long long left = P < pool ? pool - P : 0;
        req[r].pages = (int)(P < pool ? P : pool);
        req[r].start = left >= w ? n : held * kKvTile - c + (int)left * kKvTile;
        P += w;
        tokens += req[r].start;
    }
    long long S = block_before(tokens, warp_s, all);
    const int total = (int)(all < budget ? all : budget);
    long long last = 0;                                                   // behind the last page that this thread's requests take
    for (int r = r0; r < r1; ++r) {
        const int c = req[r].cached, room = S < budget ? (int)(budget - S) : 0, n = min(req[r].start, room);
        const int takes = pages_of(c + n) - pages_of(c);
        if (takes) last = req[r].pages + takes;
        req[r].start = (int)(S < budget ? S : budget);
        S += n;
        if (blockIdx.x == 0) {
            req_start[r] = req[r].start;
            ctx_lens[r] = c + n;
        }
    }
    if (blockIdx.x == 0 && tid == 0) req_start[R] = total;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const long long x = __shfl_xor_sync(0xffffffffu, last, o);
        last = x > last ? x : last;
    }
    __syncthreads();                                                      // the sums have been read, and the requests are complete
    if ((tid & 31) == 0) warp_s[tid >> 5] = last;
    __syncthreads();
    int takes_all = 0;
    for (int w = 0; w < SL_WARPS; ++w) takes_all = max(takes_all, (int)warp_s[w]);
    if (blockIdx.x == 0 && tid == 0) *taken = first + takes_all;

    // The last request that begins at or before x; those without tokens (or pages) begin where the next one does
    auto owner_of = [&](int x, auto&& begin) {
        int lo = 0, hi = R - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (begin(mid) <= x) lo = mid; else hi = mid - 1;
        }
        return lo;
    };
    const int at = blockIdx.x * SL_THREADS + tid, step = gridDim.x * SL_THREADS;
    for (long long k = at; k < takes_all; k += step) {
        const StepRequest q = req[owner_of((int)k, [&](int r) { return req[r].pages; })];
        page_table[(size_t)q.slot * max_pages + pages_of(q.cached) + ((int)k - q.pages)] = free_pages[first + k];
    }
    for (long long i = at; i < budget; i += step) {
        int pos = -1, row = -1, where = -1;
        if (i < total) {
            const StepRequest q = req[owner_of((int)i, [&](int r) { return req[r].start; })];
            const int held = pages_of(q.cached);
            pos = q.cached + (int)i - q.start;
            row = q.slot;
            const int j = pos / kKvTile;
            // pages that this call hands out are read from the pool: other CTAs may not have written them into the table yet
            const int page = j < held ? page_table[(size_t)q.slot * max_pages + j] : free_pages[first + q.pages + j - held];
            if (page >= 0 && page < INT_MAX / kKvTile) where = page * kKvTile + pos % kKvTile;
        }
        positions[i] = pos;
        seq_rows[i] = row;
        kv_slots[i] = where;
    }
}

static int step_lists_hash(int R) {                            // places: a power of two, twice the requests at least
    int n = 64;
    while (n < 2 * R) n *= 2;
    return n;
}

}  // namespace ft

extern "C" int ft_step_lists(const ft_step_lists_args* args, void* stream) {
    using namespace ft;
    FT_REQUIRE(args, "ft_step_lists: null argument");
    const auto [cached_lens, new_lens, req_slot, page_table, free_pages, first_free, req_start, ctx_lens, positions, seq_rows, kv_slots, taken, R, table_rows, max_pages, n_free,
                max_tokens] = *args;
    FT_REQUIRE(R >= 0 && R <= SL_MAX_REQUESTS, "ft_step_lists: %d requests (at most %d)", R, SL_MAX_REQUESTS);
    FT_REQUIRE(max_tokens >= 0 && max_tokens <= 1 << 30 && table_rows >= 0 && n_free >= 0 && max_pages >= 0 && max_pages < INT32_MAX / kKvTile,
               "ft_step_lists: bad sizes max_tokens=%d table %d x %d, %d free pages", max_tokens, table_rows, max_pages, n_free);
    FT_REQUIRE(req_start && taken && (R == 0 || (cached_lens && new_lens && ctx_lens)) && (max_tokens == 0 || (positions && seq_rows && kv_slots)) &&
                   (page_table || table_rows == 0 || max_pages == 0) && (free_pages || n_free == 0),
               "ft_step_lists: null argument");
    FT_REQUIRE(taken != first_free, "ft_step_lists: taken at the address of first_free, which other CTAs may read later");
    // Every CTA makes the scans for itself, when it comes to run: what one writes must be nothing that another may still read (lengths advanced in place, say)
    const struct { const int* at; size_t n; } arrays[] = {
        {req_start, (size_t)R + 1}, {ctx_lens, (size_t)R}, {positions, (size_t)max_tokens}, {seq_rows, (size_t)max_tokens}, {kv_slots, (size_t)max_tokens}, {taken, 1},
        {page_table, (size_t)table_rows * max_pages}, {cached_lens, (size_t)R}, {new_lens, (size_t)R}, {req_slot, req_slot ? (size_t)R : 0}, {free_pages, (size_t)n_free},
        {first_free, first_free ? 1u : 0u}};
    constexpr int kWritten = 7;                                // the first of these
    for (int i = 0; i < kWritten; ++i)
        for (int j = i + 1; j < (int)(sizeof(arrays) / sizeof(arrays[0])); ++j)
            FT_REQUIRE(!arrays[i].n || !arrays[j].n || (uintptr_t)arrays[i].at + arrays[i].n * 4 <= (uintptr_t)arrays[j].at || (uintptr_t)arrays[j].at + arrays[j].n * 4 <= (uintptr_t)arrays[i].at,
                       "ft_step_lists: an array that it writes overlaps another one");
    static PerDeviceFlag attr_set;
    if (!attr_set.done()) {
        FT_CHECK_CUDA(cudaFuncSetAttribute(step_lists_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           SL_MAX_REQUESTS * (int)sizeof(StepRequest) + step_lists_hash(SL_MAX_REQUESTS) * 4));
        attr_set.mark();
    }
    const int hash = req_slot ? step_lists_hash(R) : 0, sms = device_sms();
    const int ctas = max_tokens <= SL_THREADS ? 1 : (max_tokens + SL_THREADS - 1) / SL_THREADS < sms ? (max_tokens + SL_THREADS - 1) / SL_THREADS : sms;
    FT_CHECK_CUDA(launch_after(step_lists_kernel, dim3(ctas), dim3(SL_THREADS), (size_t)R * sizeof(StepRequest) + (size_t)hash * 4, (cudaStream_t)stream, cached_lens, new_lens,
                               req_slot, R, page_table, table_rows, max_pages, free_pages, n_free, first_free, max_tokens, hash, req_start, ctx_lens, positions, seq_rows,
                               kv_slots, taken));
    return 0;
}
