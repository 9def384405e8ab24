// Attention of packed new tokens over pages on the tensor cores, bf16: chunks of prompts, drafted tokens and single ones in one batch.
//
// A row of a tile is a (token, query head) of one request and one key head, so that a key is read once for all heads that share it; a
// tile is two halves of 128 rows, each a thread's to a row.  Its keys come 128 at a time, page by page (a copy of up to 128 rows each), and
// the softmax runs along them as in the attention over tokens: scores and outputs in tensor memory, s = q k^T, p written over s, o += p v, the
// products of one half running while the other's weights are formed, outputs rescaled only when a maximum has grown by more than 2^8.
//
// Requests are of uneven lengths, and few new tokens see many keys: so the work is cut by tiles of keys, not by tiles of rows.  All (tile of
// rows, key head, tile of keys) stand in one line, which is shared out evenly among one CTA to an SM.  A CTA writes results where it has a tile
// of rows whole, else its part (at most two to a CTA), and a second kernel joins the parts of the tiles that were cut, in their order.
// p is rounded to bf16 for its product, as its operand type asks; the sum of the softmax takes it unrounded.
#include "slotscan_attn_scores.cuh"
#include "slotscan_launch.h"
#include "slotscan_paged.cuh"
#include "slotscan_tensor.cuh"

namespace slotscan {

static __device__ int g_paged_status = 0;                // a bounded wait gave up (slotscan_device_status)

constexpr float PA_GROWN = 8.f;                          // in powers of two
constexpr int PA_HALVES = 2, PA_KEYS = 128, PA_ROWS = PA_HALVES * 128;
constexpr int PA_THREADS = PA_ROWS + 128;
constexpr int PA_STAGES = 4;                             // tiles of the ring, keys and values in turn
template <int DP>
struct PagedShape {
    static constexpr int SUBS = DP / 64;                 // 64-column sub-tiles of a tile
    static constexpr int QTILE = 128 * DP * 2, KTILE = PA_KEYS * DP * 2;           // bytes
    static constexpr int SMEM = PA_HALVES * QTILE + PA_STAGES * KTILE + 1024;
};
struct PagedMaps { CUtensorMap q, k, v; };

// What the first CTA leaves for the join: of each tile of rows its place in the line and its request, and the length of a CTA's share
struct LinePlan {
    long long* before;                                   // most + 1
    long long* per;
    long long* tiles;
    int2* tile;                                          // request, tile of its rows
    float* parts;
    long long most;                                      // tiles that the scratch has room for: all, unless starts falls
    static size_t head_bytes(long long most) { return (sizeof(long long) * (most + 3) + sizeof(int2) * most + 15) / 16 * 16; }
    LinePlan(void* scratch, long long most_) : before((long long*)scratch), per(before + most_ + 1), tiles(per + 1), tile((int2*)(tiles + 1)),
                                               parts((float*)((char*)scratch + head_bytes(most_))), most(most_) {}
    // outputs, unscaled, then maximum and sum of each row
    __device__ __forceinline__ float* part(int cta, bool begun, int D) const { return parts + (2 * (size_t)cta + begun) * PA_ROWS * (D + 2); }
};

// A tile of rows of one request
struct RowTile {
    int row0, tokens, at0;                               // first packed row, its tokens, position of the first (minus one: they see nothing)
    int n0, n1;                                          // key tiles; one that nobody sees where there are none
};
__device__ __forceinline__ RowTile row_tile(const PagedArgs& a, const RowShape& rs, int b, int tile) {
    const int begin = rows_begin(a, b), most = PA_HALVES * rs.tokens;
    RowTile t;
    t.row0 = begin + tile * most;
    t.tokens = min(most, rows_end(a, b) - t.row0);
    const int at = a.pos[begin];
    t.at0 = at < 0 ? -1 : min(at, 1 << 30) + tile * most;
    t.n0 = 0;
    t.n1 = 1;
    if (at >= 0) {
        const int lo = paged_keys(a, b, t.at0).lo, hi = paged_keys(a, b, t.at0 + t.tokens - 1).hi;
        if (hi > lo) { t.n0 = lo / PA_KEYS; t.n1 = (hi + PA_KEYS - 1) / PA_KEYS; }
    }
    return t;
}
// key tiles [first, last) that a half of the tile sees within [n0, n1); first = last where it sees none
struct HalfRange { int first, last; };
__device__ __forceinline__ HalfRange half_range(const PagedArgs& a, const RowShape& rs, int b, const RowTile& t, int half, int n0, int n1) {
    const int from = half * rs.tokens, n = min(rs.tokens, t.tokens - from);
    if (n <= 0 || t.at0 < 0) return {n0, n0};
    const int lo = paged_keys(a, b, t.at0 + from).lo, hi = paged_keys(a, b, t.at0 + from + n - 1).hi;
    if (hi <= lo) return {n0, n0};
    const int first = max(lo / PA_KEYS, n0), last = min((hi + PA_KEYS - 1) / PA_KEYS, n1);
    return last > first ? HalfRange{first, last} : HalfRange{n0, n0};
}

// A place in the line, and what of it lies ahead
struct LineCursor {
    int b, tile, pair, n;                                // pair: key head and chunk of its query heads; n: key tiles of the tile passed
    long long left;
    RowTile t;
    __device__ __forceinline__ int steps() const { return t.n1 - t.n0; }
    // the piece of the current tile that is this CTA's
    __device__ __forceinline__ int piece() const { return (int)min((long long)(steps() - n), left); }
    __device__ __forceinline__ void next_tile(const PagedArgs& a, const RowShape& rs) {
        n = 0;
        if (++pair < a.KV * a.chunks) return;
        pair = 0;
        tile++;
        while (rows_begin(a, b) + (long long)tile * PA_HALVES * rs.tokens >= rows_end(a, b)) {
            tile = 0;
            if (++b >= a.B) return;
        }
        t = row_tile(a, rs, b, tile);
    }
    __device__ __forceinline__ void next_piece(const PagedArgs& a, const RowShape& rs) {
        const int p = piece();
        n += p;
        left -= p;
        if (left > 0 && n == steps()) next_tile(a, rs);
    }
};

__device__ __forceinline__ long long line_sum(long long v, long long* s_sum) {     // inclusive over the CTA's threads, kept in s_sum
    const int tid = threadIdx.x, lane = tid & 31;
#pragma unroll
    for (int off = 1; off < 32; off *= 2) {
        const long long up = __shfl_up_sync(FULL, v, off);
        if (lane >= off) v += up;
    }
    __syncthreads();
    s_sum[tid] = v;
    __syncthreads();
    long long base = 0;
    for (int i = 0; i < tid / 32; i++) base += s_sum[32 * i + 31];
    __syncthreads();
    s_sum[tid] = v + base;
    __syncthreads();
    return v + base;
}
__device__ __forceinline__ int first_above(const long long* s_sum, int threads, long long x) {      // first thread whose sum is greater
    int lo = 0, hi = threads - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (s_sum[mid] > x) hi = mid; else lo = mid + 1;
    }
    return lo;
}
// The CTA's share of the line, by all its threads
template <int THREADS>
__device__ __forceinline__ void line_share(const PagedArgs& a, const RowShape& rs, const LinePlan& plan, LineCursor* out) {
    __shared__ long long s_tiles[THREADS], s_steps[THREADS];
    const int tid = threadIdx.x, most = PA_HALVES * rs.tokens, pairs = a.KV * a.chunks;
    auto tiles_of = [&](int b) { return (rows_end(a, b) - rows_begin(a, b) + most - 1) / most; };
    const int per_b = (a.B + THREADS - 1) / THREADS, b0 = min(tid * per_b, a.B), b1 = min(b0 + per_b, a.B);
    long long v = 0;
    for (int b = b0; b < b1; b++) v += tiles_of(b);
    line_sum(v, s_tiles);
    const long long tiles = min(s_tiles[THREADS - 1], plan.most), per_u = (tiles + THREADS - 1) / THREADS;
    // request and tile of the u-th tile of rows
    auto find = [&](long long u, int& b, int& tile) {
        const int t = first_above(s_tiles, THREADS, u);
        b = t * per_b;
        long long in = u - (t > 0 ? s_tiles[t - 1] : 0);
        for (int n = tiles_of(b); in >= n; n = tiles_of(b)) { in -= n; b++; }
        tile = (int)in;
    };
    auto walk = [&](long long u0, long long u1, auto each) {
        if (u0 >= u1) return;
        int b, tile;
        find(u0, b, tile);
        for (long long u = u0; u < u1; u++) {
            const RowTile t = row_tile(a, rs, b, tile);
            if (!each(u, b, tile, t)) return;
            if (++tile >= tiles_of(b) && u + 1 < u1) { tile = 0; do b++; while (tiles_of(b) == 0); }
        }
    };
    const long long u0 = min(tid * per_u, tiles), u1 = min(u0 + per_u, tiles);
    v = 0;
    walk(u0, u1, [&](long long, int, int, const RowTile& t) { v += t.n1 - t.n0; return true; });
    const long long upto = line_sum(v, s_steps), total = s_steps[THREADS - 1] * pairs, per = (total + gridDim.x - 1) / gridDim.x;
    if (blockIdx.x == 0) {
        long long at = upto - v;
        walk(u0, u1, [&](long long u, int b, int tile, const RowTile& t) {
            plan.before[u] = at * pairs;
            plan.tile[u] = make_int2(b, tile);
            at += t.n1 - t.n0;
            return true;
        });
        if (tid == 0) { plan.before[tiles] = total; *plan.per = per; *plan.tiles = tiles; }
    }
    const long long x0 = blockIdx.x * per, x1 = min(x0 + per, total);
    if (tid == 0) {
        LineCursor c = {};
        c.left = max(x1 - x0, 0ll);
        if (c.left > 0) {
            const int t = first_above(s_steps, THREADS, x0 / pairs);
            long long at = t > 0 ? s_steps[t - 1] : 0;
            walk(t * per_u, tiles, [&](long long, int b, int tile, const RowTile& rt) {
                const int steps = rt.n1 - rt.n0;
                if ((at + steps) * pairs <= x0) { at += steps; return true; }
                c.b = b; c.tile = tile; c.t = rt;
                c.pair = (int)((x0 - at * pairs) / steps);
                c.n = (int)((x0 - at * pairs) % steps);
                return false;
            });
        }
        *out = c;
    }
    __syncthreads();
}

template <int DP, bool CAP, bool BIAS>
__global__ void __launch_bounds__(PA_THREADS, 1)
paged_attn_kernel(PagedArgs a, RowShape rs, LinePlan plan, const __grid_constant__ PagedMaps maps, const bf16* q, const bf16* kp, const bf16* vp, bf16* o) {
    typedef PagedShape<DP> Sh;
    extern __shared__ char smem_raw[];
    char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    char* Qs = smem;
    char* Ks = smem + PA_HALVES * Sh::QTILE;
    __shared__ uint64_t q_full, q_empty, s_full[PA_HALVES], p_full[PA_HALVES], o_full[PA_HALVES], full[PA_STAGES], empty[PA_STAGES];
    __shared__ uint32_t s_tmem;
    __shared__ int s_fail;
    __shared__ LineCursor s_at;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31, group = a.H / a.KV;
    if (tid == 0) {
        mbar_init(&q_full, 1); mbar_init(&q_empty, 1);
        for (int t = 0; t < PA_HALVES; t++) { mbar_init(&s_full[t], 1); mbar_init(&p_full[t], 4); mbar_init(&o_full[t], 1); }
        for (int s = 0; s < PA_STAGES; s++) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        mbar_fence_init();
        s_fail = 0;
    }
    if (warp == PA_HALVES * 4) tmem_alloc(&s_tmem, 512);
    line_share<PA_THREADS>(a, rs, plan, &s_at);
    {                                                    // rows of no request
        const int r0 = a.B > 0 ? rows_begin(a, 0) : a.N, r1 = a.B > 0 ? max(rows_end(a, a.B - 1), r0) : a.N;
        const long long pieces = (long long)a.H * a.D / 8, n = (long long)(r0 + a.N - r1) * pieces;
        for (long long i = (long long)blockIdx.x * PA_THREADS + tid; i < n; i += (long long)gridDim.x * PA_THREADS) {
            const long long row = i / pieces;
            *reinterpret_cast<uint4*>(o + (row < r0 ? row : row - r0 + r1) * a.H * a.D + i % pieces * 8) = make_uint4(0, 0, 0, 0);
        }
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    constexpr uint32_t tmem = 0;                         // all 512 columns are this CTA's, so they begin at the first
    LineCursor c = s_at;
    bool ok = true;
    // 3 x 128 threads x 168 registers at launch = 2 x 128 x 216 + 128 x 72; a row of 128 scores stays in registers
    if (warp < PA_HALVES * 4) {                          // ---- softmax of a half ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int half = tid / 128, r = tid % 128, token = r / rs.heads, g = r % rs.heads;
        const uint32_t lane_at = (uint32_t)((warp % 4) * 32) << 16;
        const uint32_t S = tmem + half * PA_KEYS + lane_at, O = tmem + PA_HALVES * PA_KEYS + half * DP + lane_at;
        unsigned done = 0, x0 = 0;                       // key tiles of this half so far; tiles of the ring before this piece
        const long long share = c.left;
        for (; c.left > 0 && ok; c.next_piece(a, rs)) {
            const int n0 = c.t.n0 + c.n, n1 = n0 + c.piece(), b = c.b, hk = c.pair / a.chunks, h = hk * group + c.pair % a.chunks * rs.heads + g;
            const bool cut = n0 > c.t.n0 || n1 < c.t.n1;
            const HalfRange hr = half_range(a, rs, b, c.t, half, n0, n1);
            const int tk = half * rs.tokens + token;     // of the tile
            const bool row = token < rs.tokens && tk < c.t.tokens && c.pair % a.chunks * rs.heads + g < group;
            const Span sp = row && c.t.at0 >= 0 ? paged_keys(a, b, c.t.at0 + tk) : Span{0, 0};
            const int all_lo = paged_keys(a, b, c.t.at0).lo, all_hi = paged_keys(a, b, c.t.at0 + c.t.tokens - 1).hi;
            const WarpSpan ws(sp);
            const Score sc = paged_score(a, h);
            float m = -INFINITY, l = 0.f;                // m in base-2 exponents
            const float at = (float)(c.t.at0 + tk);
            for (int n = hr.first; n < hr.last; n++, done++) {
                const int j0 = n * PA_KEYS;
                const bool masked = !ws.clear(j0, PA_KEYS);
                if (!(ok = wait_soon_warp(&s_full[half], done & 1))) break;
                tmem_fence_after();
                uint32_t raw[PA_KEYS / 32][32];
#pragma unroll
                for (int i = 0; i < PA_KEYS / 32; i++) tmem_ld(S + i * 32, raw[i]);
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < PA_KEYS / 32; i++) {
                    tmem_ld_wait(raw[i]);
                    float(&s)[32] = reinterpret_cast<float(&)[32]>(raw[i]);
                    scores32<CAP, BIAS>(s, sc, at - (float)(j0 + i * 32), masked, sp.lo - j0 - i * 32, sp.hi - j0 - i * 32);
                    float t0 = s[0], t1 = s[1], t2 = s[2], t3 = s[3];
#pragma unroll
                    for (int e = 4; e < 32; e += 4) { t0 = fmaxf(t0, s[e]); t1 = fmaxf(t1, s[e + 1]); t2 = fmaxf(t2, s[e + 2]); t3 = fmaxf(t3, s[e + 3]); }
                    top = fmaxf(top, fmaxf(fmaxf(t0, t1), fmaxf(t2, t3)));
                }
                if constexpr (!CAP && !BIAS) top *= sc.lin;
                const bool grown = top > m + PA_GROWN && m != -INFINITY;           // a row that has seen nothing so far has only zeros to rescale
                if (m == -INFINITY) m = top;
                if (__any_sync(FULL, grown)) {
                    const float to = fmaxf(m, top), f = to == -INFINITY ? 1.f : exp2_fast(m - to);
                    if (n > hr.first) {
                        if (!(ok = wait_soon_warp(&o_full[half], (done - 1) & 1))) break;
                        tmem_fence_after();
#pragma unroll
                        for (int i = 0; i < DP / 32; i++) {
                            uint32_t y[32];
                            tmem_ld(O + i * 32, y);
                            tmem_ld_wait(y);
#pragma unroll
                            for (int e = 0; e < 32; e++) y[e] = __float_as_uint(__uint_as_float(y[e]) * f);
                            tmem_st(O + i * 32, y);
                        }
                    }
                    m = to;
                    l *= f;
                }
                const float base = m == -INFINITY ? 0.f : m;
                f32x2 sum[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
                const f32x2 lin = pack2(sc.lin, sc.lin), back = pack2(-base, -base);
#pragma unroll
                for (int i = 0; i < PA_KEYS / 32; i++) {
                    uint32_t w[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const f32x2 y = pack2(__uint_as_float(raw[i][e]), __uint_as_float(raw[i][e + 1]));
                        const float2 z = unpack2(CAP || BIAS ? add2(y, back) : fma2(y, lin, back));
                        const float p0 = exp2_fast(z.x), p1 = exp2_fast(z.y);
                        sum[(e / 2) % 2] = add2(sum[(e / 2) % 2], pack2(p0, p1));
                        w[e / 2] = pack_bf16(p0, p1);
                    }
                    tmem_st(S + i * 16, w);
                }
                const float2 total = unpack2(add2(sum[0], sum[1]));
                l += total.x + total.y;
                if (j0 < all_lo || j0 + PA_KEYS > all_hi) {
                    // values that no row of the tile sees (the rest of a page, another request's) must not reach the product: zeros
                    const unsigned xv = x0 + 2 * (n - n0) + 1, s = xv % PA_STAGES;
                    if (!(ok = wait_soon_warp(&full[s], (xv / PA_STAGES) & 1))) break;
                    if (j0 + r < all_lo || j0 + r >= all_hi) {
#pragma unroll
                        for (int i = 0; i < DP / 8; i++)
                            *reinterpret_cast<uint4*>(Ks + s * Sh::KTILE + (i / 8) * PA_KEYS * 128 + r * 128 + (i % 8) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                }
                tmem_st_wait();
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) arrive(&p_full[half]);
            }
            if (ok && hr.last > hr.first) ok = wait_soon_warp(&o_full[half], (done - 1) & 1);
            if (!ok) break;
            tmem_fence_after();
            const bool none = sp.hi <= sp.lo;
            const float inv = none ? 0.f : 1.f / l;
            // at the share's first step a part continues what the CTA before has begun
            float* part = plan.part(blockIdx.x, c.left != share, a.D);
            const int pr = half * 128 + r;
            bf16* to = o + ((size_t)(c.t.row0 + tk) * a.H + h) * a.D;
            float seen = 0.f;
#pragma unroll
            for (int i = 0; i < DP / 32; i++) {
                uint32_t y[32];
#pragma unroll
                for (int e = 0; e < 32; e++) y[e] = 0u;
                if (hr.last > hr.first) { tmem_ld(O + i * 32, y); tmem_ld_wait(y); }
#pragma unroll
                for (int e = 0; e < 32; e++) watch(seen, __uint_as_float(y[e]));
                if (!row) continue;
                if (cut) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        if (i * 32 + e < a.D)
                            *reinterpret_cast<uint4*>(part + (size_t)pr * a.D + i * 32 + e) = make_uint4(y[e], y[e + 1], y[e + 2], y[e + 3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        uint32_t w[4];
#pragma unroll
                        for (int u = 0; u < 4; u++)
                            w[u] = none ? 0u : pack_bf16(__uint_as_float(y[e + 2 * u]) * inv, __uint_as_float(y[e + 2 * u + 1]) * inv);
                        if (i * 32 + e < a.D) *reinterpret_cast<uint4*>(to + i * 32 + e) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
            if (cut && row) *reinterpret_cast<float2*>(part + (size_t)PA_ROWS * a.D + 2 * pr) = make_float2(fmaxf(m, -FLT_MAX), l);
            for (unsigned bad = __ballot_sync(FULL, row && !none && (seen != seen)); bad != 0; bad &= bad - 1) {
                const int from = __ffs(bad) - 1;
                const int xr = __shfl_sync(FULL, r, from), xtk = __shfl_sync(FULL, tk, from), xh = __shfl_sync(FULL, h, from);
                const int lo = max(__shfl_sync(FULL, sp.lo, from), n0 * PA_KEYS), hi = min(__shfl_sync(FULL, sp.hi, from), n1 * PA_KEYS);
                float y[4], xm, xl;
                careful_row(a, paged_score(a, xh), q + (long long)(c.t.row0 + xtk) * a.qs[0] + xh * a.qs[1], kp, vp, b, hk, c.t.at0 + xtk, lo, hi, y, xm, xl);
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int d = lane + 32 * e;
                    if (d >= a.D) continue;
                    if (cut) part[(size_t)(half * 128 + xr) * a.D + d] = y[e];
                    else o[((size_t)(c.t.row0 + xtk) * a.H + xh) * a.D + d] = __float2bfloat16_rn(y[e] / xl);
                }
                if (cut && lane == 0) *reinterpret_cast<float2*>(part + (size_t)PA_ROWS * a.D + 2 * (half * 128 + xr)) = make_float2(fmaxf(xm, -FLT_MAX), xl);
            }
            x0 += 2 * (n1 - n0);
            tmem_fence_before();
            __syncwarp();
        }
        if (!ok) s_fail = 1;
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == PA_HALVES * 4 + 1) {                 // ---- copies ----
            unsigned x = 0, piece = 0;
            const int rows = min(1 << a.shift, PA_KEYS), boxes = PA_KEYS / rows;
            for (; c.left > 0 && ok; c.next_piece(a, rs), piece++) {
                const int n0 = c.t.n0 + c.n, n1 = n0 + c.piece(), hk = c.pair / a.chunks, h0 = hk * group + c.pair % a.chunks * rs.heads;
                if (piece > 0 && !(ok = wait_soon_warp(&q_empty, (piece - 1) & 1))) break;
                if (lane == 0) {
                    const int halves = c.t.tokens > rs.tokens ? 2 : 1;
                    mbar_arrive_expect_tx(&q_full, halves * Sh::SUBS * rs.heads * rs.tokens * 128);
                    for (int t = 0; t < halves; t++)
                        for (int s = 0; s < Sh::SUBS; s++)
                            box_g2s(Qs + t * Sh::QTILE + s * 128 * 128, &maps.q, s * 64, h0, c.t.row0 + t * rs.tokens, &q_full);
                }
                for (int n = n0; n < n1 && ok; n++) {
                    for (int w = 0; w < 2; w++, x++) {   // keys, values
                        const unsigned s = x % PA_STAGES, turn = x / PA_STAGES;
                        if (turn > 0 && !(ok = wait_soon_warp(&empty[s], (turn - 1) & 1))) break;
                        if (lane == 0) mbar_arrive_expect_tx(&full[s], Sh::KTILE);
                        __syncwarp();
                        for (int i = lane; i < boxes * Sh::SUBS; i += 32) {        // a page outside the pool, or beyond the table: zeros
                            const int sub = i / boxes, box = i % boxes, j = n * PA_KEYS + box * rows;
                            const int id = (j >> a.shift) < a.M ? page_of(a, c.b, j) : -1;
                            tile_g2s(Ks + s * Sh::KTILE + sub * PA_KEYS * 128 + box * rows * 128, w ? &maps.v : &maps.k, sub * 64, j & ((1 << a.shift) - 1), hk,
                                     max(id, -1), &full[s]);
                        }
                    }
                }
            }
            if (!ok && lane == 0) s_fail = 1;
        } else if (warp == PA_HALVES * 4) {              // ---- products ----
            const bool lead = elected();
            unsigned x = 0, piece = 0, done[PA_HALVES] = {0, 0};
            auto stage = [](unsigned i) { return i % PA_STAGES; };
            auto arrived = [&](unsigned i) { return wait_soon_warp(&full[stage(i)], (i / PA_STAGES) & 1); };
            auto scores = [&](int t, unsigned i) {       // s = q k^T
                const uint32_t qd = tile_desc(smem_u32(Qs + t * Sh::QTILE), 16), kd = tile_desc(smem_u32(Ks + stage(i) * Sh::KTILE), 16);
                if (lead) {
#pragma unroll
                    for (int k = 0; k < DP / 16; k++)
                        mma_ss(tmem + t * PA_KEYS, qd + ((k / 4) * 128 * 128 + (k % 4) * 32) / 16, kd + ((k / 4) * PA_KEYS * 128 + (k % 4) * 32) / 16,
                               mma_shape(PA_KEYS, false), k > 0);
                    mma_commit(&s_full[t]);
                }
                __syncwarp();
            };
            for (; c.left > 0 && ok; c.next_piece(a, rs), piece++) {
                const int n0 = c.t.n0 + c.n, n1 = n0 + c.piece();
                HalfRange hr[PA_HALVES];
#pragma unroll
                for (int t = 0; t < PA_HALVES; t++) hr[t] = half_range(a, rs, c.b, c.t, t, n0, n1);
                ok = wait_soon_warp(&q_full, piece & 1) && arrived(x);
#pragma unroll
                for (int t = 0; t < PA_HALVES; t++)
                    if (ok && hr[t].first == n0 && hr[t].last > hr[t].first) scores(t, x);
                if (lead) mma_commit(&empty[stage(x)]);
                __syncwarp();
                for (int n = n0; n < n1 && ok; n++, x += 2) {
                    ok = arrived(x + 1) && (n + 1 == n1 || arrived(x + 2));
                    const uint32_t vd = tile_desc(smem_u32(Ks + stage(x + 1) * Sh::KTILE), PA_KEYS * 128);
#pragma unroll
                    for (int t = 0; t < PA_HALVES; t++) {
                        if (!ok) break;
                        if (n >= hr[t].first && n < hr[t].last) {
                            ok = wait_soon_warp(&p_full[t], done[t] & 1);
                            done[t]++;
                            tmem_fence_after();
                            if (lead) {
#pragma unroll
                                for (int k = 0; k < PA_KEYS / 16; k++)
                                    mma_ts(tmem + PA_HALVES * PA_KEYS + t * DP, tmem + t * PA_KEYS + k * 8, vd + k * 2048 / 16, mma_shape(DP, true), n > hr[t].first || k > 0);
                                mma_commit(&o_full[t]);
                            }
                            __syncwarp();
                        }
                        if (n + 1 >= hr[t].first && n + 1 < hr[t].last) scores(t, x + 2);
                    }
                    if (lead) {
                        mma_commit(&empty[stage(x + 1)]);
                        if (n + 1 < n1) mma_commit(&empty[stage(x + 2)]);
                    }
                    __syncwarp();
                }
                if (lead) mma_commit(&q_empty);
                __syncwarp();
            }
            if (!ok) s_fail = 1;
        }
    }
    tmem_fence_before();
    __syncthreads();
    if (s_fail != 0) {                                   // report, and give copies and products in flight time to land
        if (tid == 0) atomicExch(&g_paged_status, 1);
        for (int i = 0; i < 1000; i++) __nanosleep(1000);
    }
    if (warp == PA_HALVES * 4) { tmem_fence_after(); tmem_free(s_tmem, 512); }
}

// The tile of rows that the end of a CTA's share cuts, joined in the order of its parts: blockIdx.x the share, the first that cuts it
// does; a warp to a row
constexpr int LJ_ROWS = 32;
__global__ void __launch_bounds__(256) line_join_kernel(PagedArgs a, RowShape rs, LinePlan plan, bf16* o) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, group = a.H / a.KV, pairs = a.KV * a.chunks;
    const long long tiles = *plan.tiles, per = *plan.per;
    const long long x = (blockIdx.x + 1ll) * per;        // the cut
    if (per == 0 || x >= plan.before[tiles]) return;
    long long lo = 0, hi = tiles - 1;                    // the tile that holds it
    while (lo < hi) {
        const long long mid = (lo + hi + 1) / 2;
        if (plan.before[mid] <= x) lo = mid; else hi = mid - 1;
    }
    const long long steps = (plan.before[lo + 1] - plan.before[lo]) / pairs, pair = (x - plan.before[lo]) / steps, x0 = plan.before[lo] + pair * steps;
    if (x == x0 || x - per > x0) return;                 // cuts nothing, or is not the first to cut it
    const int w0 = (int)(x0 / per), w1 = (int)((x0 + steps - 1) / per);
    const int2 at = plan.tile[lo];
    const RowTile t = row_tile(a, rs, at.x, at.y);
    for (int pr = blockIdx.y * LJ_ROWS + warp; pr < (blockIdx.y + 1) * LJ_ROWS; pr += 8) {
        const int half = pr / 128, r = pr % 128, token = r / rs.heads, g = (int)(pair % a.chunks) * rs.heads + r % rs.heads, tk = half * rs.tokens + token;
        if (token >= rs.tokens || tk >= t.tokens || g >= group) continue;
        const Span sp = t.at0 >= 0 ? paged_keys(a, at.x, t.at0 + tk) : Span{0, 0};
        float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (int w = w0; w <= w1; w++) {
            const float* part = plan.part(w, w * per < x0, a.D);
            const float2 ml = *reinterpret_cast<const float2*>(part + (size_t)PA_ROWS * a.D + 2 * pr);
            const float top = fmaxf(m, ml.x), f = exp2f(m - top), pf = exp2f(ml.x - top);
            l = l * f + ml.y * pf;
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (lane + 32 * c < a.D) acc[c] = acc[c] * f + part[(size_t)pr * a.D + lane + 32 * c] * pf;
            m = top;
        }
        bf16* to = o + ((size_t)(t.row0 + tk) * a.H + (pair / a.chunks) * group + g) * a.D;
#pragma unroll
        for (int c = 0; c < 4; c++)
            if (lane + 32 * c < a.D) to[lane + 32 * c] = __float2bfloat16_rn(sp.hi > sp.lo ? acc[c] / l : 0.f);
    }
}

static RowShape row_shape(const PagedArgs& a) {
    const int group = a.H / a.KV, heads = group < 128 ? group : 128;
    return {heads, 128 / heads};
}
static long long most_tiles(const PagedArgs& a) { return a.N / (PA_HALVES * row_shape(a).tokens) + (long long)a.B; }

size_t paged_attn_scratch_bf16(const PagedArgs& a) {
    return LinePlan::head_bytes(most_tiles(a)) + sizeof(float) * 148 * 2 * PA_ROWS * (size_t)(a.D + 2);
}

template <int DP, bool CAP, bool BIAS>
static cudaError_t paged_tensor(const PagedArgs& a, const void* q, const void* k, const void* v, void* o, void* scratch, cudaStream_t st) {
    typedef PagedShape<DP> Sh;
    auto kern = paged_attn_kernel<DP, CAP, BIAS>;
    const cudaError_t e = opt_in_smem(kern, Sh::SMEM);   // before the maps: a thread's first runtime call makes the context current for them
    if (e != cudaSuccess) return e;
    const RowShape rs = row_shape(a);
    PagedMaps maps;
    const int page = 1 << a.shift, rows = page < PA_KEYS ? page : PA_KEYS;
    if (!box_map(&maps.q, q, a.N, a.H, a.D, a.qs, rs.heads, rs.tokens) || !tile_map(&maps.k, k, a.pages, page, a.KV, a.D, a.ks, rows) || !tile_map(&maps.v, v, a.pages, page, a.KV, a.D, a.vs, rows))
        return cudaErrorInvalidValue;
    const LinePlan plan(scratch, most_tiles(a));
    kern<<<148, PA_THREADS, Sh::SMEM, st>>>(a, rs, plan, maps, (const bf16*)q, (const bf16*)k, (const bf16*)v, (bf16*)o);
    line_join_kernel<<<dim3(147, PA_ROWS / LJ_ROWS), 256, 0, st>>>(a, rs, plan, (bf16*)o);
    return cudaGetLastError();
}
template <int DP>
static cudaError_t paged_tensor_score(const PagedArgs& a, const void* q, const void* k, const void* v, void* o, void* scratch, cudaStream_t st) {
    if (a.cap > 0.f) return a.slopes != nullptr ? paged_tensor<DP, true, true>(a, q, k, v, o, scratch, st) : paged_tensor<DP, true, false>(a, q, k, v, o, scratch, st);
    return a.slopes != nullptr ? paged_tensor<DP, false, true>(a, q, k, v, o, scratch, st) : paged_tensor<DP, false, false>(a, q, k, v, o, scratch, st);
}

cudaError_t run_paged_attn_bf16(const PagedArgs& args, const void* q, const void* k, const void* v, void* o, void* scratch, cudaStream_t st) {
    PagedArgs a = args;
    const int heads = row_shape(a).heads;
    a.chunks = (a.H / a.KV + heads - 1) / heads;
    return a.D <= 64 ? paged_tensor_score<64>(a, q, k, v, o, scratch, st) : paged_tensor_score<128>(a, q, k, v, o, scratch, st);
}

int paged_attn_status() {
    int v = 0;
    const int z = 0;
    if (cudaMemcpyFromSymbol(&v, g_paged_status, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) cudaMemcpyToSymbol(g_paged_status, &z, sizeof(int));
    return v;
}

}  // namespace slotscan
