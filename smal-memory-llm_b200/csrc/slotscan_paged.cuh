// Attention over pages of a pool: what its kernels share.
#pragma once
#include <cfloat>

#include "slotscan_attn.cuh"

namespace slotscan {

struct PagedArgs {
    int N, B, H, KV, D;
    int pages, shift, M;                                 // pages of the pool, log2 of a page's tokens, pages of a request at most
    int window;                                          // 0: none
    int chunks;                                          // of the query heads of a key head
    float scale, cap;
    long long qs[2], ks[3], vs[3], table_stride;
    const int32_t *tables, *starts, *pos, *start;
    const float* slopes;
};

// keys that a query at position `at` sees, [lo, hi), of a request that sees from `first` on; empty where hi <= lo.  What a table does not reach
// is not seen.
__device__ __forceinline__ Span paged_keys_from(const PagedArgs& a, int first, int at) {
    const int hi = at < 0 ? 0 : min(at, (a.M << a.shift) - 1) + 1;
    return {a.window > 0 && at >= a.window ? max(first, at - a.window + 1) : first, hi};
}
__device__ __forceinline__ int first_key(const PagedArgs& a, int b) { return a.start != nullptr ? max(a.start[b], 0) : 0; }
__device__ __forceinline__ Span paged_keys(const PagedArgs& a, int b, int at) { return paged_keys_from(a, first_key(a, b), at); }
// id of the page of key j; minus one where it is not of the pool
__device__ __forceinline__ int page_of(const PagedArgs& a, int b, int j) {
    const int id = a.tables[b * a.table_stride + (j >> a.shift)];
    return id < a.pages ? id : -1;
}

__device__ __forceinline__ Score paged_score(const PagedArgs& a, int h) {
    AttnArgs s;
    s.scale = a.scale; s.cap = a.cap; s.slopes = a.slopes;
    return Score(s, min(h, a.H - 1));
}
// Packed rows of a request [begin, end), the position of the first (minus one: they see nothing) and the first key that they see
struct Request { int begin, end, at, first; };
__device__ __forceinline__ int rows_begin(const PagedArgs& a, int b) { return min(max(a.starts[b], 0), a.N); }
__device__ __forceinline__ int rows_end(const PagedArgs& a, int b) { return max(min(a.starts[b + 1], a.N), rows_begin(a, b)); }
// Position of a request's first row, minus one where its rows see nothing; so that those behind it, and the rows that a tile does not have, stay
// within an int
__device__ __forceinline__ int first_position(const PagedArgs& a, int begin, int end) { return min(max(a.pos[begin], -1), BIGI - 512 - (end - begin)); }
__device__ __forceinline__ Request request(const PagedArgs& a, int b) {
    Request r = {rows_begin(a, b), rows_end(a, b), -1, first_key(a, b)};
    if (r.end > r.begin) r.at = first_position(a, r.begin, r.end);
    return r;
}
// Rows of a tile: `heads` query heads (of the `chunks`-th part of a group) of `tokens` tokens, the heads of a token side by side
struct RowShape { int heads, tokens; };                  // of a tile, or of a half of it

// ---- a row at a time, by a warp, over the keys that it sees within [lo, hi): where hidden values have made a result not finite ----
template <typename T>
__device__ __forceinline__ void careful_row(const PagedArgs& a, const Score& sc, const T* q, const T* kp, const T* vp, int b, int hk, int at, int lo, int hi,
                                            float (&o)[4], float& m, float& l) {
    const int in_page = (1 << a.shift) - 1;
    careful_keys(sc, q, a.D, at, lo, hi,
                 [&](int j, const T*& key, const T*& value) {
                     const int id = page_of(a, b, j), row = j & in_page;
                     key = id >= 0 ? kp + id * a.ks[0] + row * a.ks[1] + hk * a.ks[2] : nullptr;
                     value = id >= 0 ? vp + id * a.vs[0] + row * a.vs[1] + hk * a.vs[2] : nullptr;
                 },
                 o, m, l);
}

static inline PagedArgs paged_args(const slotscan_paged_params& p, const int32_t* tables, const int32_t* starts, const int32_t* pos, const int32_t* start,
                                   const float* slopes) {
    PagedArgs a;
    a.N = p.N; a.B = p.B; a.H = p.H; a.KV = p.KV; a.D = p.D; a.pages = p.pages; a.M = p.M;
    a.window = p.window; a.chunks = 1;
    a.shift = 0;
    while ((1 << a.shift) < p.page) a.shift++;
    a.scale = p.scale; a.cap = p.cap;
    for (int i = 0; i < 2; i++) a.qs[i] = p.q_stride[i];
    for (int i = 0; i < 3; i++) { a.ks[i] = p.k_stride[i]; a.vs[i] = p.v_stride[i]; }
    a.table_stride = p.table_stride;
    a.tables = tables; a.starts = starts; a.pos = pos; a.start = start; a.slopes = slopes;
    return a;
}

// attention of packed rows, by type
size_t paged_attn_scratch_bf16(const PagedArgs& a);
size_t paged_attn_scratch_f32(const PagedArgs& a);
cudaError_t run_paged_attn_bf16(const PagedArgs& a, const void* q, const void* k, const void* v, void* o, void* scratch, cudaStream_t st);
cudaError_t run_paged_attn_f32(const PagedArgs& a, const void* q, const void* k, const void* v, void* o, void* scratch, cudaStream_t st);

}  // namespace slotscan
