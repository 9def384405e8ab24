// Pages of a pool handed to requests and taken back, and the slots of a packed batch of new tokens, on the GPU: a scheduler's turn without
// a copy to the host.
//
// With n the new tokens of a request, len what it holds and P the tokens of a page
//     ends = inclusive sum of n,   need = ceil((len + n) / P) - ceil(len / P),   upto = inclusive sum of need
// a request is served if its table and the batch have room and need = 0 or upto <= free pages; page j of it, the (upto - need + j - have)-th
// handed out, is taken from the end of the stack of free ones.  So everything is two sums over the requests, then independent per token.
//
// The sums are one CTA's, 1,024 requests at a time; what follows is its own too while it is little (one launch is the floor of a small turn),
// and a second kernel's beyond.  Nothing is chosen by an order of arrival, so results repeat.  Bound by latency and by
// the host: a turn of two calls takes 19 us for four requests, 23 for 1,024 with 99,000 tokens.
//
// Back go the entries of a request's table that are pages of the pool: the others (minus ones where another request owns the page) are counted
// out before the sum over the requests, since an id that no page has would be handed out again and its tokens stored nowhere.
#include <cuda_runtime.h>
#include <stdint.h>

#include "slotscan.h"
#include "slotscan_common.cuh"
#include "slotscan_launch.h"

namespace slotscan {

constexpr int PG_THREADS = 1024;
constexpr int PG_OWN_ROWS = 8192;                        // rows, or entries of tables, that the CTA of the sums sees to itself

struct PageArgs {
    int B, M, shift, pages, tokens;
    long long table_stride;
    int32_t *lengths, *tables, *free_pages, *n_free;
};
// What the sums leave for the rows: per request the tokens held before (minus one: not served) and the rank of its first page; once the
// free pages before.  Of requests that end: the entries of their table, the rank within their CTA's requests and how many go back, and per CTA
// how many in all.
constexpr int PG_CTAS = 148 * 8;
struct PagePlan {
    int32_t *held, *rank, *n_free, *back, *total;
    static size_t ints(int B) { return 3 * (size_t)B + 1 + PG_CTAS; }
    __host__ __device__ explicit PagePlan(int32_t* scratch, int B)
        : held(scratch), rank(scratch + B), n_free(scratch + 2 * (size_t)B), back(n_free + 1), total(back + B) {}
};

__device__ __forceinline__ long long pages_of(long long n, int shift) { return (n + (1 << shift) - 1) >> shift; }

// inclusive sum over the CTA on top of `carry`, which becomes the total; s_warp: 32 places that the call before this one did not have
__device__ __forceinline__ long long cta_sum(long long v, long long* s_warp, long long& carry) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
#pragma unroll
    for (int off = 1; off < 32; off *= 2) {
        const long long up = __shfl_up_sync(FULL, v, off);
        if (lane >= off) v += up;
    }
    if (lane == 31) s_warp[warp] = v;
    __syncthreads();
    long long w = s_warp[lane];                          // every warp sums the warps' totals for itself
#pragma unroll
    for (int off = 1; off < 32; off *= 2) {
        const long long up = __shfl_up_sync(FULL, w, off);
        if (lane >= off) w += up;
    }
    const long long before = __shfl_sync(FULL, w, (warp + 31) % 32), all = __shfl_sync(FULL, w, 31);
    v += carry + (warp > 0 ? before : 0);
    carry += all;
    return v;
}
__device__ __forceinline__ int free_before(const PageArgs& a) { return min(max(*a.n_free, 0), a.pages); }

// Slots and positions of packed rows, 32 to a warp, and the table's entries of pages that begin with them.  `i`: the lane's row.  The first
// row's request is found in steps of 32, so that few loads wait for one another, and the others' among the 32 that follow it.
__device__ __forceinline__ void place_rows(const PageArgs& a, const PagePlan& plan, const int32_t* starts, int32_t* slots, int32_t* pos, int i) {
    const int lane = threadIdx.x & 31, i0 = i - lane;
    int slot = -1, at = -1;
    if (i0 < starts[a.B]) {                              // the same in all lanes
        int lo = 0, n = a.B;                             // the first request that ends behind i0 is one of n from lo on
        while (n > 1) {
            const int step = (n + 31) / 32, mine = lo + min((lane + 1) * step, n);
            const int below = __popc(__ballot_sync(FULL, (lane + 1) * step < n && starts[mine] <= i0));
            lo += below * step;
            n = min(step, n - below * step);
        }
        int b = lo;
        for (int b0 = lo;; b0 += 32) {                   // those without rows among them
            const int end = b0 + lane < a.B ? starts[b0 + lane + 1] : BIGI;
            int behind = 0;                              // of the 32, how many end at or before i
#pragma unroll
            for (int step = 16; step > 0; step /= 2)
                if (__shfl_sync(FULL, end, behind + step - 1) <= i) behind += step;
            const int last = __shfl_sync(FULL, end, 31);
            if (behind == 31 && last <= i) behind = 32;
            if (b == b0) b += behind;
            if (!__any_sync(FULL, b == b0 + 32 && b < a.B)) break;
        }
        if (i < starts[a.B]) {
            const int held = plan.held[b];
            if (held >= 0) {
                at = held + i - starts[b];
                const int page = at >> a.shift, have = (int)pages_of(held, a.shift);
                int32_t* entry = a.tables + b * a.table_stride + page;
                const int id = page < have ? *entry : a.free_pages[*plan.n_free - 1 - (plan.rank[b] + page - have)];
                const int in_page = at & ((1 << a.shift) - 1);
                if (in_page == 0) *entry = id;
                const long long s = ((long long)id << a.shift) + in_page;
                slot = id >= 0 && s < BIGI ? (int)s : -1;                          // of a page of the pool it is one (slotscan_pages_check)
            }
        }
    }
    if (i < a.tokens) {
        slots[i] = slot;
        pos[i] = at;
    }
}

template <bool OWN>
__global__ void __launch_bounds__(PG_THREADS) extend_kernel(PageArgs a, const int32_t* fresh, int32_t* scratch, int32_t* slots, int32_t* pos, int32_t* starts,
                                                            int32_t* taken) {
    __shared__ long long s_warp[2][32];
    __shared__ int s_handed;
    const PagePlan plan(scratch, a.B);
    const int tid = threadIdx.x;
    if (tid == 0) { s_handed = 0; starts[0] = 0; }
    if (tid < 64) s_warp[tid / 32][tid % 32] = 0;        // of warps that the CTA does not have
    const int nf = free_before(a);
    long long tokens = 0, pages = 0;
    __syncthreads();
    for (int b0 = 0; b0 < a.B; b0 += blockDim.x) {
        const int b = b0 + tid;
        const bool in = b < a.B;
        const long long n = in ? max(fresh[b], 0) : 0, held = in ? max(a.lengths[b], 0) : 0;
        const long long ends = cta_sum(n, s_warp[0], tokens);
        const bool fits = in && held + n <= ((long long)a.M << a.shift) && ends <= a.tokens;
        const long long need = fits ? pages_of(held + n, a.shift) - pages_of(held, a.shift) : 0;
        const long long upto = cta_sum(need, s_warp[1], pages);
        const bool served = fits && (need == 0 || upto <= nf);
        if (in) {
            starts[b + 1] = (int)min(ends, (long long)a.tokens);
            taken[b] = served ? (int)n : 0;
            plan.held[b] = served ? (int)held : -1;
            plan.rank[b] = (int)min(upto - need, (long long)BIGI);
            if (served && n > 0) a.lengths[b] = (int)(held + n);
            if (served && need > 0) atomicMax(&s_handed, (int)upto);
        }
    }
    __syncthreads();
    if (tid == 0) {
        *plan.n_free = nf;
        *a.n_free = nf - s_handed;
    }
    if constexpr (OWN) {
        __syncthreads();
        for (int i = tid; i - (tid & 31) < a.tokens; i += blockDim.x) place_rows(a, plan, starts, slots, pos, i);
    }
}
__global__ void __launch_bounds__(256) place_kernel(PageArgs a, int32_t* scratch, const int32_t* starts, int32_t* slots, int32_t* pos) {
    cudaGridDependencySynchronize();
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i - (int)(threadIdx.x & 31) < a.tokens) place_rows(a, PagePlan(scratch, a.B), starts, slots, pos, i);
}

// how many of a table's first n entries are pages of the pool, as far as this thread sees them
__device__ __forceinline__ int pool_pages(const PageArgs& a, const int32_t* row, int n, int tid, int threads) {
    int mine = 0;
    for (int j = tid; j < n; j += threads) mine += row[j] >= 0 && row[j] < a.pages;
    return mine;
}
__device__ __forceinline__ int held_pages(const PageArgs& a, int b) { return (int)min(pages_of(max(a.lengths[b], 0), a.shift), (long long)a.M); }

// a request's pages onto the stack from place `to` on, in their order, and its table emptied
__device__ __forceinline__ void give_back(const PageArgs& a, const PagePlan& plan, int b, long long to, int tid, int threads) {
    const int n = plan.held[b];
    if (n < 0) return;
    int32_t* row = a.tables + b * a.table_stride;
    const bool all = plan.back[b] == n;
    if (!all && tid < 32) {                              // some are none: those before them are counted, 32 at a time
        for (int j0 = 0; j0 < n; j0 += 32) {
            const int id = j0 + tid < n ? row[j0 + tid] : -1;
            const bool page = id >= 0 && id < a.pages;
            const unsigned pages = __ballot_sync(FULL, page);
            const long long at = to + __popc(pages & ((1u << tid) - 1));
            if (page && at < a.pages) a.free_pages[at] = id;
            if (j0 + tid < n) row[j0 + tid] = -1;
            to += __popc(pages);
        }
    }
    for (int j = (all ? 0 : n) + tid; j < a.M; j += threads) {
        if (j < n && to + j < a.pages) a.free_pages[to + j] = row[j];
        row[j] = -1;
    }
}

// by one CTA: a warp to a request
__global__ void __launch_bounds__(PG_THREADS) release_kernel(PageArgs a, const uint8_t* done, int32_t* scratch) {
    __shared__ long long s_warp[2][32];
    const PagePlan plan(scratch, a.B);
    const int tid = threadIdx.x, lane = tid & 31;
    if (tid < 64) s_warp[tid / 32][tid % 32] = 0;
    const int nf = free_before(a);
    for (int b = tid / 32; b < a.B; b += blockDim.x / 32) {
        const int n = done[b] != 0 ? held_pages(a, b) : -1;
        const int pages = __reduce_add_sync(FULL, pool_pages(a, a.tables + b * a.table_stride, n, lane, 32));
        if (lane == 0) { plan.held[b] = n; plan.back[b] = pages; }
    }
    long long pages = 0;
    int turn = 0;
    __syncthreads();
    for (int b0 = 0; b0 < a.B; b0 += blockDim.x, turn ^= 1) {
        const int b = b0 + tid, n = b < a.B ? plan.back[b] : 0;
        const long long upto = cta_sum(n, s_warp[turn], pages);
        if (b < a.B) {
            plan.rank[b] = (int)min(upto - n, (long long)BIGI);
            if (plan.held[b] >= 0) a.lengths[b] = 0;
        }
    }
    if (tid == 0) *a.n_free = (int)min(nf + pages, (long long)a.pages);
    __syncthreads();
    for (int b = tid / 32; b < a.B; b += blockDim.x / 32) give_back(a, plan, b, (long long)nf + plan.rank[b], lane, 32);
}

// By many: a CTA counts a run of requests, one after the other, and another one like it, which knows the counts of those before it, gives
// their pages back.
struct Run { int b0, b1; };
__device__ __forceinline__ Run run_of(const PageArgs& a) {
    const int per = (a.B + gridDim.x - 1) / gridDim.x, b0 = min((int)blockIdx.x * per, a.B);
    return {b0, min(b0 + per, a.B)};
}
constexpr int PG_RUN_THREADS = 256;
__device__ __forceinline__ long long run_sum(long long v, long long* s_warp) {     // over the CTA; s_warp: a place to a warp
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(FULL, v, off);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x / 32] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < PG_RUN_THREADS / 32; i++) v += s_warp[i];
    return v;
}
__global__ void __launch_bounds__(PG_RUN_THREADS) count_back_kernel(PageArgs a, const uint8_t* done, int32_t* scratch) {
    __shared__ long long s_warp[PG_RUN_THREADS / 32];
    const PagePlan plan(scratch, a.B);
    const int tid = threadIdx.x;
    const Run r = run_of(a);
    if (blockIdx.x == 0 && tid == 0) *plan.n_free = free_before(a);
    long long sum = 0;
    for (int b = r.b0; b < r.b1; b++) {
        const bool ends = done[b] != 0;                  // the same in all threads
        const int n = ends ? held_pages(a, b) : -1;
        const int pages = ends ? (int)run_sum(pool_pages(a, a.tables + b * a.table_stride, n, tid, PG_RUN_THREADS), s_warp) : 0;
        if (tid == 0) {
            plan.held[b] = n;
            plan.back[b] = pages;
            plan.rank[b] = (int)min(sum, (long long)BIGI);
        }
        sum += pages;
    }
    if (tid == 0) plan.total[blockIdx.x] = (int)min(sum, (long long)BIGI);
}
__global__ void __launch_bounds__(PG_RUN_THREADS) give_back_kernel(PageArgs a, int32_t* scratch) {
    __shared__ long long s_warp[PG_RUN_THREADS / 32];
    const PagePlan plan(scratch, a.B);
    const int tid = threadIdx.x;
    cudaGridDependencySynchronize();
    const Run r = run_of(a);
    long long before = 0;
    for (int i = tid; i < blockIdx.x; i += PG_RUN_THREADS) before += plan.total[i];
    const long long to = *plan.n_free + run_sum(before, s_warp);
    for (int b = r.b0; b < r.b1; b++) {
        give_back(a, plan, b, to + plan.rank[b], tid, PG_RUN_THREADS);
        if (tid == 0 && plan.held[b] >= 0) a.lengths[b] = 0;
    }
    if (blockIdx.x == gridDim.x - 1 && tid == 0) *a.n_free = (int)min(to + plan.total[blockIdx.x], (long long)a.pages);
}

// threads of the sums' CTA: fewer where there are few requests and rows
static int sum_threads(long long most) { return most <= 256 ? 256 : PG_THREADS; }

static PageArgs page_args(const slotscan_pages_params& p, int32_t* lengths, int32_t* tables, int32_t* free_pages, int32_t* n_free) {
    PageArgs a;
    a.B = p.B; a.M = p.M; a.pages = p.pages; a.tokens = p.tokens;
    a.shift = 0;
    while ((1 << a.shift) < p.page) a.shift++;
    a.table_stride = p.table_stride;
    a.lengths = lengths; a.tables = tables; a.free_pages = free_pages; a.n_free = n_free;
    return a;
}

}  // namespace slotscan

using namespace slotscan;

extern "C" int slotscan_pages_check(const slotscan_pages_params* p) {
    if (p == nullptr) return SLOTSCAN_E_NULL;
    if (p->B < 0 || p->B > (1 << 24) || p->M < 1 || p->M > (1 << 26) || p->pages < 1 || p->tokens < 0 || p->tokens > (1 << 30) || p->page < 8 ||
        p->page > 1024 || (p->page & (p->page - 1)) || (int64_t)p->M * p->page > (1 << 29) || (int64_t)p->pages * p->page > BIGI || p->table_stride < p->M)
        return SLOTSCAN_E_SHAPE;
    return SLOTSCAN_OK;
}

extern "C" size_t slotscan_pages_scratch_bytes(const slotscan_pages_params* p) {
    return slotscan_pages_check(p) == SLOTSCAN_OK ? sizeof(int32_t) * PagePlan::ints(p->B) : 0;
}

extern "C" int slotscan_extend_pages(const slotscan_pages_params* p, const int32_t* fresh, int32_t* lengths, int32_t* tables, int32_t* free_pages,
                                     int32_t* n_free, int32_t* slots, int32_t* pos, int32_t* starts, int32_t* taken, void* scratch,
                                     size_t scratch_bytes, void* stream) {
    const int rc = slotscan_pages_check(p);
    if (rc != SLOTSCAN_OK) return rc;
    if (!starts || !n_free || !free_pages || (p->B && (!fresh || !lengths || !tables || !taken)) || (p->tokens && (!slots || !pos))) return SLOTSCAN_E_NULL;
    if (scratch == nullptr || scratch_bytes < slotscan_pages_scratch_bytes(p)) return SLOTSCAN_E_NULL;
    const PageArgs a = page_args(*p, lengths, tables, free_pages, n_free);
    cudaStream_t st = (cudaStream_t)stream;
    int32_t* s = (int32_t*)scratch;
    if (a.tokens <= PG_OWN_ROWS) {
        extend_kernel<true><<<1, sum_threads(a.tokens > a.B ? a.tokens : a.B), 0, st>>>(a, fresh, s, slots, pos, starts, taken);
        return (int)cudaGetLastError();
    }
    extend_kernel<false><<<1, sum_threads(a.B), 0, st>>>(a, fresh, s, slots, pos, starts, taken);
    return (int)launch_behind(place_kernel, dim3((a.tokens + 255) / 256), dim3(256), st, a, s, (const int32_t*)starts, slots, pos);
}

extern "C" int slotscan_release_pages(const slotscan_pages_params* p, const uint8_t* done, int32_t* lengths, int32_t* tables, int32_t* free_pages,
                                      int32_t* n_free, void* scratch, size_t scratch_bytes, void* stream) {
    const int rc = slotscan_pages_check(p);
    if (rc != SLOTSCAN_OK) return rc;
    if (p->B == 0) return SLOTSCAN_OK;
    if (!done || !lengths || !tables || !free_pages || !n_free) return SLOTSCAN_E_NULL;
    if (scratch == nullptr || scratch_bytes < slotscan_pages_scratch_bytes(p)) return SLOTSCAN_E_NULL;
    const PageArgs a = page_args(*p, lengths, tables, free_pages, n_free);
    cudaStream_t st = (cudaStream_t)stream;
    int32_t* s = (int32_t*)scratch;
    if ((int64_t)a.B * a.M <= PG_OWN_ROWS) {
        release_kernel<<<1, sum_threads((int64_t)a.B * a.M), 0, st>>>(a, done, s);
        return (int)cudaGetLastError();
    }
    const int ctas = a.B < PG_CTAS ? a.B : PG_CTAS;
    count_back_kernel<<<ctas, PG_RUN_THREADS, 0, st>>>(a, done, s);
    return (int)launch_behind(give_back_kernel, dim3(ctas), dim3(PG_RUN_THREADS), st, a, s);
}
