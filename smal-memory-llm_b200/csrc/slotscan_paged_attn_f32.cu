// Attention of packed new tokens over pages on the CUDA cores: float32, whose products the tensor cores would round to 11 bits or fewer.
//
// A CTA holds 32 rows, (token, query head) pairs of one request and one key head, and passes over their keys 64 at a time with the running
// maximum and sum of each row's softmax.  Where the tiles of rows would leave SMs idle, their keys are split evenly among several CTAs, and
// a second kernel joins the parts in their order.  Bound by shared memory, as the attention over tokens in float32 is; small calls by
// their launches (two chunks of 40 tokens: 12 us with the host's side).
#include "slotscan_attn_cores.cuh"
#include "slotscan_launch.h"
#include "slotscan_paged.cuh"

namespace slotscan {

constexpr int PC_ROWS = 32, PC_THREADS = 4 * PC_ROWS;

// request and tile of the u-th tile of rows, by all threads of the CTA; false where there are not so many
__device__ __forceinline__ bool find_tile(const PagedArgs& a, const RowShape& rs, int u, int& b, int& tile) {
    __shared__ int s_sum[PC_THREADS], s_at[2];
    const int tid = threadIdx.x, per_b = (a.B + PC_THREADS - 1) / PC_THREADS, b0 = min(tid * per_b, a.B), b1 = min(b0 + per_b, a.B);
    auto tiles_of = [&](int x) { return (rows_end(a, x) - rows_begin(a, x) + rs.tokens - 1) / rs.tokens; };
    int n = 0;
    for (int x = b0; x < b1; x++) n = min(n + tiles_of(x), 1 << 30);
    s_sum[tid] = n;
    if (tid == 0) s_at[0] = -1;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < tid; i++) before = min(before + s_sum[i], 1 << 30);
    if (u >= before && u < before + n) {
        int x = b0, in = u - before;
        for (int k = tiles_of(x); in >= k; k = tiles_of(x)) { in -= k; x++; }
        s_at[0] = x;
        s_at[1] = in;
    }
    __syncthreads();
    b = s_at[0];
    tile = s_at[1];
    return b >= 0;
}

// parts: per tile, pair and split its rows' outputs, unscaled, and maximum and sum of each
template <int DP>
__global__ void __launch_bounds__(PC_THREADS, 3) paged_attn_cores_kernel(PagedArgs a, RowShape rs, int splits, const float* q, const float* k, const float* v, float* o,
                                                                         float* parts) {
    extern __shared__ float4 smem4[];
    float* Qs = reinterpret_cast<float*>(smem4);
    float* Ys = Qs + PC_ROWS * (DP + 4);                 // keys, then values
    float* Ps = Ys + SA_N * (DP + 4);
    __shared__ int s_red[2];
    const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16, group = a.H / a.KV, pairs = a.KV * a.chunks;
    const int pair = blockIdx.y / splits, split = blockIdx.y % splits, hk = pair / a.chunks, g0 = pair % a.chunks * rs.heads, heads = min(rs.heads, group - g0);
    if (blockIdx.y == 0) {                               // rows of no request
        const int r0 = a.B > 0 ? rows_begin(a, 0) : a.N, r1 = a.B > 0 ? max(rows_end(a, a.B - 1), r0) : a.N;
        const long long row = (long long)a.H * a.D, n = (r0 + a.N - r1) * row;
        for (long long i = (long long)blockIdx.x * PC_THREADS + tid; i < n; i += (long long)gridDim.x * PC_THREADS) o[i < r0 * row ? i : i + (r1 - r0) * row] = 0.f;
    }
    int b, tile;
    if (!find_tile(a, rs, blockIdx.x, b, tile)) return;
    const int begin = rows_begin(a, b), t0 = tile * rs.tokens, tokens = min(rs.tokens, rows_end(a, b) - begin - t0), row0 = begin + t0;
    const int at = first_position(a, begin, rows_end(a, b)), at0 = at < 0 ? -1 : at + t0;
    auto exists = [&](int r) { return r / rs.heads < tokens && r % rs.heads < heads; };
    auto span = [&](int r) { return exists(r) && at0 >= 0 ? paged_keys(a, b, at0 + r / rs.heads) : Span{0, 0}; };
    auto query = [&](int r) { return q + (long long)(row0 + r / rs.heads) * a.qs[0] + (long long)(hk * group + g0 + r % rs.heads) * a.qs[1]; };
    auto out = [&](int r) { return o + ((size_t)(row0 + r / rs.heads) * a.H + hk * group + g0 + r % rs.heads) * a.D; };
    for (int i = tid; i < PC_ROWS * (DP / 4); i += PC_THREADS) {
        const int r = i / (DP / 4), c = i % (DP / 4) * 4;
        st4(Qs + r * (DP + 4) + c, exists(r) && c < a.D ? ld4(query(r) + c) : make_float4(0.f, 0.f, 0.f, 0.f));
    }
    Span sp[4];
    Score sc[4] = {paged_score(a, 0), paged_score(a, 0), paged_score(a, 0), paged_score(a, 0)};
#pragma unroll
    for (int r = 0; r < 4; r++) {
        sp[r] = span(4 * ty + r);
        sc[r] = paged_score(a, hk * group + g0 + (4 * ty + r) % rs.heads);
    }
    const Span all = cta_span(tid < PC_ROWS ? span(tid) : Span{0, 0}, tid < PC_ROWS, s_red);
    // this split's share of the tile's keys, in tiles of them
    const int n_all = all.hi > all.lo ? (all.hi - all.lo + SA_N - 1) / SA_N : 0, per = (n_all + splits - 1) / splits;
    const int lo = all.lo + min(split * per, n_all) * SA_N, hi = min(all.hi, all.lo + min((split + 1) * per, n_all) * SA_N);
    float m[4], l[4], acc[4][DP / 16];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        m[r] = -INFINITY; l[r] = 0.f;
#pragma unroll
        for (int c = 0; c < DP / 16; c++) acc[r][c] = 0.f;
    }
    // a tile of keys or values, zeros where no row of the tile sees them or the page is none of the pool
    auto load = [&](const float* from, const long long (&s)[3], int j0) {
        for (int i = tid; i < SA_N * (DP / 4); i += PC_THREADS) {
            const int r = i / (DP / 4), c = i % (DP / 4) * 4, j = j0 + r;
            const int id = j < hi && c < a.D ? page_of(a, b, j) : -1;
            st4(Ys + r * (DP + 4) + c, id >= 0 ? ld4(from + id * s[0] + (j & ((1 << a.shift) - 1)) * s[1] + hk * s[2] + c) : make_float4(0.f, 0.f, 0.f, 0.f));
        }
    };
    for (int j0 = lo; j0 < hi; j0 += SA_N) {
        __syncthreads();
        load(k, a.ks, j0);
        __syncthreads();
        float s[4][4];
        dot_block<DP>(s, Qs, Ys, ty, tx);
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int here = at0 + (4 * ty + r) / rs.heads;
            float top = -INFINITY, unused;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int j = j0 + tx + 16 * c;
                s[r][c] = j >= sp[r].lo && j < min(sp[r].hi, hi) ? score2(sc[r], s[r][c], here - j, unused) : -INFINITY;
                top = fmaxf(top, s[r][c]);
            }
            top = fmaxf(m[r], max16(top));
            const float base = top == -INFINITY ? 0.f : top, shrink = exp2f(m[r] - base);
            m[r] = top;
            float sum = 0.f;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const float p = exp2f(s[r][c] - base);
                sum += p;
                Ps[(4 * ty + r) * SA_LDP + tx + 16 * c] = p;
            }
            l[r] = fmaf(l[r], shrink, group_sum<16>(sum));
#pragma unroll
            for (int c = 0; c < DP / 16; c++) acc[r][c] *= shrink;
        }
        __syncthreads();
        load(v, a.vs, j0);
        __syncthreads();
        product_block<DP>(acc, Ps, Ys, ty, tx);
    }
    float* part = parts + (((size_t)blockIdx.x * pairs + pair) * splits + split) * PC_ROWS * (a.D + 2);
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int row = 4 * ty + r;
        if (!exists(row)) continue;
        const bool empty = sp[r].hi <= sp[r].lo;
        const float inv = splits > 1 ? 1.f : empty ? 0.f : 1.f / l[r];
        float* to = splits > 1 ? part + row * a.D : out(row);
#pragma unroll
        for (int c = 0; c < DP / 64; c++) {
            const int d = tx * 4 + 64 * c;
            if (d < a.D) st4(to + d, make_float4(acc[r][4 * c] * inv, acc[r][4 * c + 1] * inv, acc[r][4 * c + 2] * inv, acc[r][4 * c + 3] * inv));
        }
        if (splits > 1 && tx == 0) *reinterpret_cast<float2*>(part + PC_ROWS * a.D + 2 * row) = make_float2(fmaxf(m[r], -FLT_MAX), l[r]);
    }
    // rows that hidden values have made not finite, a warp's eight rows one after the other
#pragma unroll
    for (int r = 0; r < 4; r++) {
        float w = 0.f;
#pragma unroll
        for (int c = 0; c < DP / 16; c++) watch(w, acc[r][c]);
        const unsigned hit = __ballot_sync(FULL, w != w && exists(4 * ty + r));
#pragma unroll
        for (int half = 0; half < 2; half++) {
            if (!(hit >> (16 * half) & 0xffffu)) continue;
            const int row = 4 * (2 * (tid / 32) + half) + r, lane = tid & 31;
            const Span x = span(row);
            float y[4], xm, xl;
            __syncwarp();
            careful_row(a, paged_score(a, hk * group + g0 + row % rs.heads), query(row), k, v, b, hk, at0 + row / rs.heads, max(x.lo, lo), min(x.hi, hi), y, xm, xl);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int d = lane + 32 * c;
                if (d < a.D) (splits > 1 ? part + row * a.D : out(row))[d] = splits > 1 ? y[c] : x.hi > x.lo ? y[c] / xl : 0.f;
            }
            if (splits > 1 && lane == 0) *reinterpret_cast<float2*>(part + PC_ROWS * a.D + 2 * row) = make_float2(fmaxf(xm, -FLT_MAX), xl);
        }
    }
}

// the splits of a tile of rows, in their order; a warp to a row
__global__ void __launch_bounds__(PC_THREADS) paged_cores_join_kernel(PagedArgs a, RowShape rs, int splits, const float* parts, float* o) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, group = a.H / a.KV, pairs = a.KV * a.chunks, pair = blockIdx.y;
    const int hk = pair / a.chunks, g0 = pair % a.chunks * rs.heads, heads = min(rs.heads, group - g0);
    int b, tile;
    if (!find_tile(a, rs, blockIdx.x, b, tile)) return;
    const int begin = rows_begin(a, b), t0 = tile * rs.tokens, tokens = min(rs.tokens, rows_end(a, b) - begin - t0);
    const int at = first_position(a, begin, rows_end(a, b)), at0 = at < 0 ? -1 : at + t0;
    const float* from = parts + ((size_t)blockIdx.x * pairs + pair) * splits * PC_ROWS * (a.D + 2);
    for (int r = warp; r < PC_ROWS; r += PC_THREADS / 32) {
        if (r / rs.heads >= tokens || r % rs.heads >= heads) continue;
        const Span sp = at0 >= 0 ? paged_keys(a, b, at0 + r / rs.heads) : Span{0, 0};
        float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < splits; s++) {
            const float* part = from + (size_t)s * PC_ROWS * (a.D + 2);
            const float2 ml = *reinterpret_cast<const float2*>(part + PC_ROWS * a.D + 2 * r);
            const float top = fmaxf(m, ml.x), f = exp2f(m - top), pf = exp2f(ml.x - top);
            l = l * f + ml.y * pf;
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (lane + 32 * c < a.D) acc[c] = acc[c] * f + part[r * a.D + lane + 32 * c] * pf;
            m = top;
        }
        float* to = o + ((size_t)(begin + t0 + r / rs.heads) * a.H + hk * group + g0 + r % rs.heads) * a.D;
#pragma unroll
        for (int c = 0; c < 4; c++)
            if (lane + 32 * c < a.D) to[lane + 32 * c] = sp.hi > sp.lo ? acc[c] / l : 0.f;
    }
}

struct CoresShape { RowShape rs; int chunks, splits; long long tiles; };
static CoresShape cores_shape(const PagedArgs& a) {
    const int group = a.H / a.KV, heads = group < PC_ROWS ? group : PC_ROWS;
    CoresShape c = {{heads, PC_ROWS / heads}, (group + heads - 1) / heads, 1, 0};
    c.tiles = a.N / c.rs.tokens + (long long)(a.B < a.N ? a.B : a.N);              // requests without rows have no tile
    if (c.tiles < 1) c.tiles = 1;                        // no request: zeros to write all the same
    // three CTAs to an SM; a split takes four tiles of keys at least
    const long long ctas = c.tiles * a.KV * c.chunks, want = 148 * 3 / ctas, most = (((long long)a.M << a.shift) + 4 * SA_N - 1) / (4 * SA_N);
    c.splits = (int)(want < 1 ? 1 : want > most ? most : want);
    return c;
}

size_t paged_attn_scratch_f32(const PagedArgs& a) {
    const CoresShape c = cores_shape(a);
    return c.splits == 1 ? 0 : sizeof(float) * (size_t)c.tiles * a.KV * c.chunks * c.splits * PC_ROWS * (a.D + 2);
}

template <int DP>
static cudaError_t launch_cores(const PagedArgs& a, const CoresShape& c, const void* q, const void* k, const void* v, void* o, float* parts, cudaStream_t st) {
    const size_t sm = sizeof(float) * (PC_ROWS * (DP + 4) + SA_N * (DP + 4) + PC_ROWS * SA_LDP);
    auto kern = paged_attn_cores_kernel<DP>;
    const cudaError_t e = opt_in_smem(kern, sm);
    if (e != cudaSuccess) return e;
    const long long pairs = (long long)a.KV * c.chunks;
    if (c.tiles > 0x7fffffffll || pairs * c.splits > 65535) return cudaErrorInvalidValue;
    kern<<<dim3((unsigned)c.tiles, (unsigned)(pairs * c.splits)), PC_THREADS, sm, st>>>(a, c.rs, c.splits, (const float*)q, (const float*)k, (const float*)v, (float*)o, parts);
    if (c.splits > 1) paged_cores_join_kernel<<<dim3((unsigned)c.tiles, (unsigned)pairs), PC_THREADS, 0, st>>>(a, c.rs, c.splits, parts, (float*)o);
    return cudaGetLastError();
}

cudaError_t run_paged_attn_f32(const PagedArgs& args, const void* q, const void* k, const void* v, void* o, void* scratch, cudaStream_t st) {
    PagedArgs a = args;
    const CoresShape c = cores_shape(a);
    a.chunks = c.chunks;
    return a.D <= 64 ? launch_cores<64>(a, c, q, k, v, o, (float*)scratch, st) : launch_cores<128>(a, c, q, k, v, o, (float*)scratch, st);
}

}  // namespace slotscan

using namespace slotscan;

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

extern "C" size_t slotscan_paged_attn_scratch_bytes(const slotscan_paged_params* p) {
    if (slotscan_paged_check(p) != SLOTSCAN_OK) return 0;
    const PagedArgs a = paged_args(*p, nullptr, nullptr, nullptr, nullptr, nullptr);
    return p->dtype == SLOTSCAN_BF16 ? paged_attn_scratch_bf16(a) : paged_attn_scratch_f32(a);
}

extern "C" int slotscan_paged_attn(const slotscan_paged_params* p, const void* q, const void* kp, const void* vp, const int32_t* tables, const int32_t* starts,
                                   const int32_t* pos, const int32_t* start, const float* slopes, void* o, void* scratch, size_t scratch_bytes, void* stream) {
    const int rc = slotscan_paged_check(p);
    if (rc != SLOTSCAN_OK) return rc;
    if (p->N == 0) return SLOTSCAN_OK;
    if (!q || !kp || !vp || !starts || !pos || !o || (p->B > 0 && !tables)) return SLOTSCAN_E_NULL;
    if (!aligned16(q) || !aligned16(kp) || !aligned16(vp) || !aligned16(o) || !aligned16(scratch)) return SLOTSCAN_E_ALIGN;
    const size_t need = slotscan_paged_attn_scratch_bytes(p);
    if (need && (scratch == nullptr || scratch_bytes < need)) return SLOTSCAN_E_NULL;
    const PagedArgs a = paged_args(*p, tables, starts, pos, start, slopes);
    return (int)(p->dtype == SLOTSCAN_BF16 ? run_paged_attn_bf16(a, q, kp, vp, o, scratch, (cudaStream_t)stream)
                                           : run_paged_attn_f32(a, q, kp, vp, o, scratch, (cudaStream_t)stream));
}
