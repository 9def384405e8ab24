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
// p is rounded to bf16 for its product, as its operand type asks; the sum of the softmax takes it unrounded.  Results are off by 0.0023 of
// their norm so, 0.0017 of which is their own rounding.
//
// A chunk of 2,048 tokens of 12 heads over 65,536 keys of four: 826 us in a run of twenty (983 TFLOP/s), 930 in runs of seconds (873), in which
// the power cap holds the clock at 1,680 MHz of 1,965.  A key tile takes 3,770 cycles: a half's softmax 2,420 of them, its two products and
// their hand-overs 1,320, during which the other half's softmax runs.  A third of the special function unit's and half of the tensor cores'
// time is left.  Handing the weights over 64 keys at a time took 6 % more.  Few rows over many keys are bound by memory: 16 x 5 tokens over
// up to 32,768 keys 129 to 142 us, 5.4 to 4.9 TB/s.
#include "slotscan_attn_scores.cuh"
#include "slotscan_launch.h"
#include "slotscan_paged.cuh"
#include "slotscan_tensor.cuh"

namespace slotscan {

static __device__ int g_paged_status = 0;                // a bounded wait gave up (slotscan_device_status)

constexpr float PA_GROWN = 8.f;                          // in powers of two
constexpr int PA_HALVES = 2, PA_KEYS = 128, PA_ROWS = PA_HALVES * 128;
constexpr int PA_THREADS = PA_ROWS + 128;
constexpr int PA_OUT_ROW = 64 + 16, PA_OUT = 32 * PA_OUT_ROW;             // bytes of a warp's outputs on their way: 64 of a row, and what keeps banks apart
// Steps of the line, as their times are: of a tile of keys with rows in both halves, in one, and of a tile of rows itself (its queries and
// results)
constexpr int PA_TWO = 5, PA_ONE = 3, PA_TILE_COST = 9;
constexpr int PA_STAGES = 4;                             // tiles of the ring, keys and values in turn
template <int DP>
struct PagedShape {
    static constexpr int SUBS = DP / 64;                 // 64-column sub-tiles of a tile
    static constexpr int QTILE = 128 * DP * 2, KTILE = PA_KEYS * DP * 2;           // bytes
    static constexpr int SMEM = PA_HALVES * QTILE + PA_STAGES * KTILE + PA_HALVES * 4 * PA_OUT + 1024;
};
struct PagedMaps { CUtensorMap q, k, v; };

// What the CTAs leave for the join: each the tile of rows that its end is the first to cut (tokens 0: none), and its parts, at most two: of the
// tile that its share begins in, and of the one that it ends in
struct Cut {
    int row0, tokens, at0, first, h0, heads;
    int begun;                                           // the share that begins the tile begins with it
    int shares;                                          // CTAs that have a part of it
};
struct LinePlan {
    Cut* cuts;
    float* parts;
    long long most;                                      // tiles of rows, unless starts falls
    static size_t head_bytes() { return (sizeof(Cut) * 148 + 15) / 16 * 16; }
    LinePlan(void* scratch, long long most_) : cuts((Cut*)scratch), parts((float*)((char*)scratch + head_bytes())), most(most_) {}
    // outputs, unscaled, then maximum and sum of each row
    __device__ __forceinline__ float* part(int cta, bool begun, int D) const { return parts + (2 * (size_t)cta + !begun) * PA_ROWS * (D + 2); }
};

// A tile of rows of one request
struct RowTile {
    int row0, tokens, at0;                               // first packed row, its tokens, position of the first (minus one: they see nothing)
    int n0, n1;                                          // key tiles; one that nobody sees where there are none
};
__device__ __forceinline__ RowTile row_tile(const PagedArgs& a, const RowShape& rs, const Request& r, int tile) {
    const int most = PA_HALVES * rs.tokens;
    RowTile t;
    t.row0 = r.begin + tile * most;
    t.tokens = min(most, r.end - t.row0);
    t.at0 = r.at < 0 ? -1 : r.at + tile * most;
    t.n0 = 0;
    t.n1 = 1;
    if (r.at >= 0) {
        const int lo = paged_keys_from(a, r.first, t.at0).lo, hi = paged_keys_from(a, r.first, t.at0 + t.tokens - 1).hi;
        if (hi > lo) { t.n0 = lo / PA_KEYS; t.n1 = (hi + PA_KEYS - 1) / PA_KEYS; }
    }
    return t;
}
__device__ __forceinline__ int step_cost(const RowShape& rs, const RowTile& t) { return t.tokens > rs.tokens ? PA_TWO : PA_ONE; }
// The first requests, kept in shared memory: a CTA looks them up again and again while it finds its share
struct Requests {
    Request* kept;                                       // PA_THREADS
    __device__ __forceinline__ Request at(const PagedArgs& a, int b) const { return b < PA_THREADS ? kept[b] : request(a, b); }
};
// A place in the line, and what of it lies ahead.  A tile of rows takes PA_TILE_COST steps of the line, then its key tiles theirs; a key
// tile is the share's in which its last step lies.
struct LineCursor {
    int b, tile, pair, n;                                // pair: key head and chunk of its query heads; n: steps of the tile passed
    long long left;
    RowTile t;
    int each;                                            // steps of a key tile
    __device__ __forceinline__ int steps() const { return PA_TILE_COST + (t.n1 - t.n0) * each; }
    // the steps of the current tile that are this CTA's, and the key tiles whose last step is before the n-th
    __device__ __forceinline__ int piece() const { return (int)min((long long)(steps() - n), left); }
    __device__ __forceinline__ int key(int n) const { return t.n0 + max(n - PA_TILE_COST, 0) / each; }
    __device__ __forceinline__ void next_tile(const PagedArgs& a, const RowShape& rs, const Requests& all) {
        n = 0;
        if (++pair < a.KV * a.chunks) return;
        pair = 0;
        tile++;
        Request r = all.at(a, b);
        while (tile * PA_HALVES * rs.tokens >= r.end - r.begin) {
            tile = 0;
            if (++b >= a.B) return;
            r = all.at(a, b);
        }
        t = row_tile(a, rs, r, tile);
        each = step_cost(rs, t);
    }
    __device__ __forceinline__ void next_piece(const PagedArgs& a, const RowShape& rs, const Requests& all) {
        const int p = piece();
        n += p;
        left -= p;
        if (left > 0 && n == steps()) next_tile(a, rs, all);
    }
};

// inclusive over the CTA's threads, kept in s_sum; s_warp: a place for each warp, of this call alone
template <typename T>
__device__ __forceinline__ void line_sum(T v, T* s_sum, T* s_warp) {
    const int tid = threadIdx.x, lane = tid & 31;
#pragma unroll
    for (int off = 1; off < 32; off *= 2) {
        const T up = __shfl_up_sync(FULL, v, off);
        if (lane >= off) v += up;
    }
    if (lane == 31) s_warp[tid / 32] = v;
    __syncthreads();
    for (int i = 0; i < tid / 32; i++) v += s_warp[i];
    s_sum[tid] = v;
    __syncthreads();
}
template <typename T>
__device__ __forceinline__ int first_above(const T* s_sum, T x) {                  // first thread whose sum is greater
    int lo = 0, hi = PA_THREADS - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (s_sum[mid] > x) hi = mid; else lo = mid + 1;
    }
    return lo;
}
// The CTA's share of the line, by all its threads
__device__ __forceinline__ void line_share(const PagedArgs& a, const RowShape& rs, int most_tiles, const Requests& all, LineCursor* out, long long* out_per) {
    __shared__ int s_tiles[PA_THREADS], s_warp0[PA_THREADS / 32];
    __shared__ long long s_steps[PA_THREADS], s_warp1[PA_THREADS / 32];
    const int tid = threadIdx.x, most = PA_HALVES * rs.tokens, pairs = a.KV * a.chunks;
    if (tid < a.B) all.kept[tid] = request(a, tid);
    __syncthreads();
    auto tiles_of = [&](const Request& r) { return (r.end - r.begin + most - 1) / most; };
    const int per_b = (a.B + PA_THREADS - 1) / PA_THREADS, b0 = min(tid * per_b, a.B), b1 = min(b0 + per_b, a.B);
    int n = 0;
    for (int b = b0; b < b1; b++) n = min(n + tiles_of(all.at(a, b)), most_tiles);                   // more there are not, unless starts falls
    line_sum(n, s_tiles, s_warp0);
    const int tiles = min(s_tiles[PA_THREADS - 1], most_tiles), per_u = (tiles + PA_THREADS - 1) / PA_THREADS;
    auto walk = [&](int u0, int u1, auto each) {         // tiles of rows [u0, u1)
        if (u0 >= u1) return;
        const int t = first_above(s_tiles, u0);
        int b = t * per_b, tile = u0 - (t > 0 ? s_tiles[t - 1] : 0);
        Request r = all.at(a, b);
        for (int k = tiles_of(r); tile >= k; k = tiles_of(r)) { tile -= k; r = all.at(a, ++b); }
        for (int u = u0; u < u1; u++) {
            if (!each(b, tile, row_tile(a, rs, r, tile))) return;
            if (++tile >= tiles_of(r) && u + 1 < u1) {
                tile = 0;
                do r = all.at(a, ++b); while (r.end == r.begin);
            }
        }
    };
    long long v = 0;
    walk(min(tid * per_u, tiles), min((tid + 1) * per_u, tiles), [&](int, int, const RowTile& t) { v += PA_TILE_COST + (t.n1 - t.n0) * step_cost(rs, t); return true; });
    line_sum(v, s_steps, s_warp1);
    if (tid == 0) {
        const long long total = s_steps[PA_THREADS - 1] * pairs, per = max((total + gridDim.x - 1) / gridDim.x, (long long)PA_TWO), x0 = blockIdx.x * per;     // a key tile to each
        LineCursor c = {};
        c.left = max(min(per, total - x0), 0ll);
        if (c.left > 0) {
            const int t = first_above(s_steps, x0 / pairs);
            long long at = (t > 0 ? s_steps[t - 1] : 0) * pairs;
            walk(t * per_u, tiles, [&](int b, int tile, const RowTile& rt) {
                const int each = step_cost(rs, rt), steps = PA_TILE_COST + (rt.n1 - rt.n0) * each;
                if (at + (long long)steps * pairs <= x0) { at += (long long)steps * pairs; return true; }
                c.b = b; c.tile = tile; c.t = rt; c.each = each;
                c.pair = (int)((x0 - at) / steps);
                c.n = (int)(x0 - at - (long long)c.pair * steps);
                return false;
            });
        }
        *out = c;
        *out_per = per;
    }
    __syncthreads();
}

// A piece of a CTA's share: a tile of rows over some of its key tiles.  One warp writes them ahead of the others, whose addresses
// in global memory it thereby keeps out of their way.
struct Piece {
    int b, hk, h0, heads;                                // h0: its first query head
    int row0, tokens, at0, first;                        // first: where the request begins to see
    int n0, n1;                                          // key tiles
    int lo, hi;                                          // keys that some row of the tile sees
    int from[PA_HALVES], to[PA_HALVES];                  // key tiles of each half
    int cut, begun;                                      // it has not all key tiles of its tile; it begins the share
    int twin;                                            // rows for one half alone: both take them, each every other key tile
    int stop;                                            // nothing more
};
constexpr int PA_PIECES = 4;
// Tiles of a piece in the ring: keys and values in turn.  Of a twin the keys come one tile earlier, as they are used: k0 k1 v0 k2 v1 k3 ...
__device__ __forceinline__ unsigned twin_key(unsigned i) { return i < 2 ? i : 2 * i - 1; }
__device__ __forceinline__ unsigned twin_value(unsigned i, unsigned n) { return i + 1 == n ? 2 * n - 1 : 2 * i + 2; }
struct RingTile { int i; bool value; };                  // the inverse: what stands at a place
__device__ __forceinline__ RingTile ring_tile(bool twin, int place, int n) {
    if (!twin) return {place / 2, (place & 1) != 0};
    if (place < 2) return {place, false};
    if (place == 2 * n - 1) return {n - 1, true};
    return place & 1 ? RingTile{(place + 1) / 2, false} : RingTile{(place - 2) / 2, true};
}

__device__ __forceinline__ Piece make_piece(const PagedArgs& a, const RowShape& rs, const LineCursor& c, int first, bool begun) {
    Piece p;
    p.b = c.b;
    p.hk = c.pair / a.chunks;
    const int g0 = c.pair % a.chunks * rs.heads, group = a.H / a.KV;
    p.h0 = p.hk * group + g0;
    p.heads = min(rs.heads, group - g0);
    p.row0 = c.t.row0; p.tokens = c.t.tokens; p.at0 = c.t.at0;
    p.first = first;
    p.n0 = c.key(c.n);
    p.n1 = c.key(c.n + c.piece());
    p.lo = paged_keys_from(a, first, c.t.at0).lo;
    p.hi = paged_keys_from(a, first, c.t.at0 < 0 ? -1 : c.t.at0 + c.t.tokens - 1).hi;
    for (int t = 0; t < PA_HALVES; t++) {
        const int at = t * rs.tokens, n = min(rs.tokens, p.tokens - at);
        p.from[t] = p.to[t] = p.n0;
        if (n <= 0 || p.at0 < 0) continue;
        const int lo = paged_keys_from(a, first, p.at0 + at).lo, hi = paged_keys_from(a, first, p.at0 + at + n - 1).hi;
        const int from = max(lo / PA_KEYS, p.n0), to = min((hi + PA_KEYS - 1) / PA_KEYS, p.n1);
        if (hi > lo && to > from) { p.from[t] = from; p.to[t] = to; }
    }
    p.cut = p.n0 > c.t.n0 || p.n1 < c.t.n1;
    p.begun = begun;
    p.twin = p.tokens <= rs.tokens && p.to[0] - p.from[0] >= 2;
    p.stop = 0;
    return p;
}

// A wait for a piece or for the place of one, which may last as long as others' whole pieces (up to 4 million key tiles, 8 s) or the search for
// the next request that has rows.  It is given up where a warp has given up one of the other waits, each of which is for a tile's time
// and bounded, and is bounded itself.
__device__ __forceinline__ bool wait_piece(uint64_t* bar, unsigned parity, const int* fail) {
    bool ok = false;
    for (int it = 0; it < (1 << 28); it++) {
        if ((ok = mbar_try_wait(bar, parity))) break;
        if (it > (1 << 12)) {
            __nanosleep(100);
            if (*reinterpret_cast<const volatile int*>(fail) != 0) break;
        }
    }
    return __all_sync(FULL, ok);
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
    __shared__ uint64_t piece_full[PA_PIECES], piece_empty[PA_PIECES], merge_full, merge_empty;
    __shared__ Piece s_piece[PA_PIECES];
    __shared__ float2 s_merge[128];
    __shared__ uint32_t s_tmem;
    __shared__ int s_fail;
    __shared__ LineCursor s_at;
    __shared__ long long s_per;
    __shared__ Request s_request[PA_THREADS];
    const Requests all = {s_request};
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    if (tid == 0) {
        mbar_init(&q_full, 1); mbar_init(&q_empty, 1); mbar_init(&merge_full, 4); mbar_init(&merge_empty, 4);
        for (int t = 0; t < PA_HALVES; t++) { mbar_init(&s_full[t], 1); mbar_init(&p_full[t], 4); mbar_init(&o_full[t], 1); }
        for (int s = 0; s < PA_STAGES; s++) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int s = 0; s < PA_PIECES; s++) { mbar_init(&piece_full[s], 1); mbar_init(&piece_empty[s], PA_HALVES * 4 + 3); }
        mbar_fence_init();
        s_fail = 0;
    }
    if (warp == PA_HALVES * 4) tmem_alloc(&s_tmem, 512);
    if (tid == 32) {
        prefetch_map(&maps.q);
        prefetch_map(&maps.k);
        prefetch_map(&maps.v);
    }
    line_share(a, rs, (int)plan.most, all, &s_at, &s_per);
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
    bool failed = false;
    unsigned turn = 0;                                   // pieces so far
    auto next = [&]() -> const Piece& {                  // waits for the piece; `failed` where none came
        failed = failed || !wait_piece(&piece_full[turn % PA_PIECES], (turn / PA_PIECES) & 1, &s_fail);
        return s_piece[turn % PA_PIECES];
    };
    auto passed = [&] {                                  // by a whole warp that reads no more of it
        __syncwarp();
        if (lane == 0) arrive(&piece_empty[turn % PA_PIECES]);
        turn++;
    };
    // 3 x 128 threads x 168 registers at launch = 2 x 128 x 200 + 128 x 104 (with 72 the product warp spilled)
    if (warp < PA_HALVES * 4) {                          // ---- softmax of a half ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        const int half = tid / 128, r = tid % 128, token = r / rs.heads, g = r % rs.heads;
        const uint32_t lane_at = (uint32_t)((warp % 4) * 32) << 16;
        const uint32_t S = tmem + half * PA_KEYS + lane_at, O = tmem + PA_HALVES * PA_KEYS + half * DP + lane_at;
        unsigned done = 0, others = 0, x0 = 0, merges = 0;   // key tiles of this half and of the other so far; tiles of the ring before this piece
        while (true) {
            const Piece& p = next();
            if (failed || p.stop) break;
            const int tk = (p.twin ? 0 : half) * rs.tokens + token;                // of the tile
            const bool row = token < rs.tokens && tk < p.tokens && g < p.heads;
            const int where = p.at0 + tk;
            const Span sp = row && p.at0 >= 0 ? paged_keys_from(a, p.first, where) : Span{0, 0};
            const WarpSpan ws(row ? sp : Span{0, BIGI});  // rows that are none ask for no mask
            const Score sc = paged_score(a, p.h0 + g);
            const int by = p.twin ? 2 : 1, n_first = p.twin ? p.from[0] + half : p.from[half], n_last = p.twin ? p.to[0] : p.to[half];
            const int all_lo = p.lo, all_hi = p.hi, n_base = p.n0;
            float m = -INFINITY, l = 0.f;                // m in base-2 exponents
            const bool rows_here = __any_sync(FULL, row);                          // of this warp
            for (int n = n_first; n < n_last; n += by, done++) {
                const int j0 = n * PA_KEYS;
                const bool masked = !ws.clear(j0, PA_KEYS);
                const bool edge = j0 < all_lo || j0 + PA_KEYS > all_hi;
                if (!wait_soon_warp(&s_full[half], done & 1)) { failed = true; break; }
                if (!rows_here && !edge) {               // products of rows that are none: whatever stands there
                    if (lane == 0) arrive(&p_full[half]);
                    continue;
                }
                tmem_fence_after();
                // The weights are taken relative to the maximum so far, and the new one is found beside them; only where it has grown too
                // much (or the row begins) are they taken once more, out of the scores that still stand in tensor memory.
                uint32_t w[PA_KEYS / 2];
                float total;
                while (true) {
                    float top = -INFINITY;
                    const float base = m == -INFINITY ? 0.f : m;
                    f32x2 sum[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
                    const f32x2 lin = pack2(sc.lin, sc.lin), back = pack2(-base, -base);
                    uint32_t raw[2][32];
                    tmem_ld(S, raw[0]);
#pragma unroll
                    for (int i = 0; i < PA_KEYS / 32; i++) {
                        uint32_t(&x)[32] = raw[i % 2];
                        tmem_ld_wait(x);
                        if (i + 1 < PA_KEYS / 32) tmem_ld(S + (i + 1) * 32, raw[(i + 1) % 2]);
                        float(&s)[32] = reinterpret_cast<float(&)[32]>(x);
                        // the distance is taken between whole numbers: float32 does not hold the positions beyond 2^24
                        scores32<CAP, BIAS, true>(s, sc, (float)(where - j0 - i * 32), masked, sp.lo - j0 - i * 32, sp.hi - j0 - i * 32, row);
                        float t0 = s[0], t1 = s[1];
#pragma unroll
                        for (int e = 2; e < 32; e += 4) { t0 = fmaxf(fmaxf(t0, s[e]), s[e + 1]); if (e + 2 < 32) t1 = fmaxf(fmaxf(t1, s[e + 2]), s[e + 3]); }
                        top = fmaxf(top, fmaxf(t0, t1));
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const f32x2 y = pack2(s[e], s[e + 1]);
                            const float2 z = unpack2(CAP || BIAS ? add2(y, back) : fma2(y, lin, back));
                            const float p0 = exp2_fast(z.x), p1 = exp2_fast(z.y);
                            sum[(e / 2) % 2] = add2(sum[(e / 2) % 2], pack2(p0, p1));
                            w[i * 16 + e / 2] = pack_bf16(p0, p1);
                        }
                    }
                    if constexpr (!CAP && !BIAS) top *= sc.lin;
                    const float2 both = unpack2(add2(sum[0], sum[1]));
                    total = both.x + both.y;
                    const bool grown = row && top > m + PA_GROWN;                         // minus infinity: a row begins
                    if (!__any_sync(FULL, grown)) break;
                    const float to = fmaxf(m, top);
                    if (__any_sync(FULL, m != -INFINITY) && n > n_first) {         // a row that has seen nothing so far has only zeros to rescale
                        const float f = m == -INFINITY ? 1.f : exp2_fast(m - to);
                        if (!wait_soon_warp(&o_full[half], (done - 1) & 1)) { failed = true; break; }
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
                        l *= f;
                    }
                    m = to;
                }
                if (failed) break;
                l += total;
#pragma unroll
                for (int i = 0; i < PA_KEYS / 32; i++) tmem_st(S + i * 16, reinterpret_cast<const uint32_t(&)[16]>(w[16 * i]));
                if (edge) {
                    // values that no row of the tile sees (the rest of a page, another request's) must not reach the product: zeros
                    const unsigned xv = x0 + (p.twin ? twin_value(n - n_base, p.n1 - n_base) : 2 * (n - n_base) + 1), s = xv % PA_STAGES;
                    if (!wait_soon_warp(&full[s], (xv / PA_STAGES) & 1)) { failed = true; break; }
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
            if (failed) break;
            others += p.twin ? (p.to[0] - p.from[0] + half) / 2 : p.to[1 - half] - p.from[1 - half];
            if (n_last > n_first && !wait_soon_warp(&o_full[half], (done - 1) & 1)) { failed = true; break; }
            float f0 = 1.f, f1 = 0.f;                    // of a twin: what the halves' outputs count
            if (p.twin && half == 1) {                   // its rows are the other half's to finish
                s_merge[r] = make_float2(m, l);
                __syncwarp();
                if (lane == 0) arrive(&merge_full);
                if (!wait_soon_warp(&merge_empty, merges & 1)) { failed = true; break; }
            } else {
                if (p.twin) {
                    if (!wait_soon_warp(&merge_full, merges & 1) || !wait_soon_warp(&o_full[1], (others - 1) & 1)) { failed = true; break; }
                    const float2 other = s_merge[r];
                    const float top = fmaxf(m, other.x), base = top == -INFINITY ? 0.f : top;
                    f0 = exp2f(m - base);
                    f1 = exp2f(other.x - base);
                    l = l * f0 + other.y * f1;
                    m = top;
                }
                tmem_fence_after();
                const bool none = sp.hi <= sp.lo;
                const float inv = none ? 0.f : 1.f / l;
                float* part = plan.part(blockIdx.x, p.begun, a.D);
                const int pr = (p.twin ? 0 : half) * 128 + r;
                const unsigned rows = __ballot_sync(FULL, row);
                // rows of 64 bytes through shared memory, so that a store covers 8 of them and not 32
                const uint32_t out = smem_u32(smem + PA_HALVES * Sh::QTILE + PA_STAGES * Sh::KTILE) + warp * PA_OUT;
                size_t to[4];                            // where this lane's four rows of the warp go
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int x = r - lane + e * 8 + lane / 4, xt = x / rs.heads;
                    to[e] = p.cut ? (size_t)(pr - r + x) * a.D : ((size_t)(p.row0 + tk - token + xt) * a.H + p.h0 + x - xt * rs.heads) * a.D;
                }
                auto put = [&](const uint32_t (&w)[16], auto* base, int d) {       // channels from d on
                    typedef typename std::remove_reference<decltype(*base)>::type E;
#pragma unroll
                    for (int e = 0; e < 4; e++) st_shared16(out + lane * PA_OUT_ROW + e * 16, w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int x = e * 8 + lane / 4;  // row of the warp
                        const uint4 v = ld_shared16(out + x * PA_OUT_ROW + (lane % 4) * 16);
                        if ((rows >> x & 1) && d + (lane % 4) * (16 / (int)sizeof(E)) < a.D)
                            *reinterpret_cast<uint4*>(base + to[e] + d + (lane % 4) * (16 / (int)sizeof(E))) = v;
                    }
                    __syncwarp();
                };
                float seen = 0.f;
                // 16 or 32 columns at a time, in loops that are not unrolled: code that a CTA runs this seldom is fetched as it runs
                auto columns = [&](auto n, int first, auto& y) {
                    constexpr int N = decltype(n)::value;
#pragma unroll
                    for (int e = 0; e < N; e++) y[e] = 0u;
                    if (n_last > n_first) { tmem_ld(O + first, y); tmem_ld_wait(y); }
                    if (p.twin) {
                        uint32_t z[N];
                        tmem_ld(O + DP + first, z);
                        tmem_ld_wait(z);
#pragma unroll
                        for (int e = 0; e < N; e++) y[e] = __float_as_uint(fmaf(__uint_as_float(z[e]), f1, __uint_as_float(y[e]) * f0));
                    }
#pragma unroll
                    for (int e = 0; e < N; e++) watch(seen, __uint_as_float(y[e]));
                };
                if (p.cut) {
#pragma unroll 1
                    for (int d = 0; d < DP; d += 16) {
                        uint32_t y[16];
                        columns(std::integral_constant<int, 16>(), d, y);
                        put(y, part, d);
                    }
                } else {
#pragma unroll 1
                    for (int d = 0; d < DP; d += 32) {
                        uint32_t y[32], w[16];
                        columns(std::integral_constant<int, 32>(), d, y);
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            w[e] = none ? 0u : pack_bf16(__uint_as_float(y[2 * e]) * inv, __uint_as_float(y[2 * e + 1]) * inv);
                        put(w, o, d);
                    }
                }
                if (p.cut && row) *reinterpret_cast<float2*>(part + (size_t)PA_ROWS * a.D + 2 * pr) = make_float2(fmaxf(m, -FLT_MAX), l);
                for (unsigned bad = __ballot_sync(FULL, row && !none && (seen != seen)); bad != 0; bad &= bad - 1) {
                    const int from = __ffs(bad) - 1;
                    const int xpr = __shfl_sync(FULL, pr, from), xtk = __shfl_sync(FULL, tk, from), xh = p.h0 + __shfl_sync(FULL, g, from);
                    const int lo = max(__shfl_sync(FULL, sp.lo, from), p.n0 * PA_KEYS), hi = min(__shfl_sync(FULL, sp.hi, from), p.n1 * PA_KEYS);
                    float y[4], xm, xl;
                    careful_row(a, paged_score(a, xh), q + (long long)(p.row0 + xtk) * a.qs[0] + xh * a.qs[1], kp, vp, p.b, p.hk, p.at0 + xtk, lo, hi, y, xm, xl);
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int d = lane + 32 * e;
                        if (d >= a.D) continue;
                        if (p.cut) part[(size_t)xpr * a.D + d] = y[e];
                        else o[((size_t)(p.row0 + xtk) * a.H + xh) * a.D + d] = __float2bfloat16_rn(y[e] / xl);
                    }
                    if (p.cut && lane == 0) *reinterpret_cast<float2*>(part + (size_t)PA_ROWS * a.D + 2 * xpr) = make_float2(fmaxf(xm, -FLT_MAX), xl);
                }
                tmem_fence_before();
                __syncwarp();
                if (p.twin && lane == 0) arrive(&merge_empty);
            }
            merges += p.twin;
            x0 += 2 * (p.n1 - p.n0);
            passed();
        }
        if (failed) s_fail = 1;
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        if (warp == PA_HALVES * 4 + 2) {                 // ---- pieces ----
            LineCursor c = s_at;
            Cut cut = {};
            for (bool begun = true; !failed; begun = false) {
                Piece p;
                p.stop = c.left <= 0;
                if (!p.stop) {
                    p = make_piece(a, rs, c, all.at(a, c.b).first, begun);
                    const int left = c.steps() - c.n - c.piece();                  // of the tile, to the next shares
                    if (left > 0 && p.n0 == c.t.n0 && p.n1 > p.n0)
                        cut = {p.row0, p.tokens, p.at0, p.first, p.h0, p.heads, begun, 1 + (int)((left + s_per - 1) / s_per)};
                    c.next_piece(a, rs, all);
                    if (p.n1 == p.n0) continue;
                }
                const unsigned slot = turn % PA_PIECES;
                if (turn >= PA_PIECES && !wait_piece(&piece_empty[slot], (turn / PA_PIECES - 1) & 1, &s_fail)) { failed = true; break; }
                if (lane == 0) {
                    s_piece[slot] = p;
                    arrive(&piece_full[slot]);
                }
                __syncwarp();
                turn++;
                if (p.stop) break;
            }
            if (lane == 0) plan.cuts[blockIdx.x] = cut;
            if (failed && lane == 0) s_fail = 1;
        } else if (warp != PA_HALVES * 4) {              // ---- copies, by two warps ----
            // Pages of 8 to 32 rows make 32 to 8 boxes a tile, whose issue takes longer than their bytes: a warp issued one in 130 cycles with a
            // lane to each.  So two warps share them, and a box's coordinates are the same in all lanes, of which the elected one issues.
            unsigned x = 0;
            const bool lead = elected(), second = warp == PA_HALVES * 4 + 3;
            const int rows = min(1 << a.shift, PA_KEYS), boxes = PA_KEYS / rows;
            const int sub = Sh::SUBS == 2 && second, by = Sh::SUBS == 2 ? 1 : 2, mine = Sh::SUBS == 2 ? boxes : (boxes + !second) / 2;
            const int box = lane * by + (Sh::SUBS == 1 && second);                 // this lane fetches the id of its page, a tile ahead
            while (true) {
                const Piece& p = next();
                if (failed || p.stop) break;
                const int n = p.n1 - p.n0, hk = p.hk;
                const bool twin = p.twin != 0;
                auto id_of = [&](int place) {            // a page outside the pool, or beyond the table: zeros
                    const int j = (p.n0 + ring_tile(twin, place, n).i) * PA_KEYS + box * rows;
                    return lane < mine && place < 2 * n && (j >> a.shift) < a.M ? max(page_of(a, p.b, j), -1) : -1;
                };
                int id = id_of(0);
                auto queries = [&] {
                    if (second || !lead) return;
                    const int halves = p.tokens > rs.tokens ? 2 : 1;
                    mbar_arrive_expect_tx(&q_full, halves * Sh::SUBS * rs.heads * rs.tokens * 128);
                    for (int t = 0; t < halves; t++)
                        for (int s = 0; s < Sh::SUBS; s++)
                            box_g2s(Qs + t * Sh::QTILE + s * 128 * 128, &maps.q, s * 64, p.h0, p.row0 + t * rs.tokens, &q_full);
                };
                if (turn == 0) queries();
                for (int place = 0; place < 2 * n; place++, x++) {
                    const int then = id_of(place + 1);
                    const RingTile t = ring_tile(twin, place, n);
                    const unsigned s = x % PA_STAGES, round = x / PA_STAGES;
                    if (round > 0 && !wait_soon_warp(&empty[s], (round - 1) & 1)) { failed = true; break; }
                    if (!second && lead) mbar_arrive_expect_tx(&full[s], Sh::KTILE);
                    const int row = (p.n0 + t.i) * PA_KEYS & ((1 << a.shift) - 1);     // of pages of more than a tile
                    char* to = Ks + s * Sh::KTILE + sub * PA_KEYS * 128;
#pragma unroll 4
                    for (int i = 0; i < mine; i++) {
                        const int at = i * by + (Sh::SUBS == 1 && second), page = __shfl_sync(FULL, id, i);
                        if (lead) tile_g2s(to + at * rows * 128, t.value ? &maps.v : &maps.k, sub * 64, row, hk, page, &full[s]);
                    }
                    __syncwarp();
                    id = then;
                    if (place != 1 || turn == 0) continue;
                    // the queries, whose place is the last piece's until its scores are done, behind the first two tiles
                    if (!wait_soon_warp(&q_empty, (turn - 1) & 1)) { failed = true; break; }
                    queries();
                }
                if (failed) break;
                passed();
            }
            if (failed && lane == 0) s_fail = 1;
        } else if (warp == PA_HALVES * 4) {              // ---- products ----
            const bool lead = elected();
            unsigned x = 0, phase = 0;                       // phase: a bit to a half, the parity of its weights' next hand-over
            auto stage = [](unsigned i) { return i % PA_STAGES; };
            auto arrived = [&](unsigned i) { failed = failed || !wait_soon_warp(&full[stage(i)], (i / PA_STAGES) & 1); return !failed; };
            auto scores = [&](int t, int tile, unsigned i) {                       // s = q k^T of a half, with the queries of tile 0 or 1
                const uint32_t qd = tile_desc(smem_u32(Qs + tile * Sh::QTILE), 16), kd = tile_desc(smem_u32(Ks + stage(i) * Sh::KTILE), 16);
                if (lead) {
#pragma unroll
                    for (int k = 0; k < DP / 16; k++)
                        mma_ss(tmem + t * PA_KEYS, qd + ((k / 4) * 128 * 128 + (k % 4) * 32) / 16, kd + ((k / 4) * PA_KEYS * 128 + (k % 4) * 32) / 16,
                               mma_shape(PA_KEYS, false), k > 0);
                    mma_commit(&s_full[t]);
                }
                __syncwarp();
            };
            auto outputs = [&](int t, unsigned i, bool add) {                      // o += p v of a half
                failed = failed || !wait_soon_warp(&p_full[t], phase >> t & 1);
                if (failed) return;
                phase ^= 1u << t;
                tmem_fence_after();
                const uint32_t vd = tile_desc(smem_u32(Ks + stage(i) * Sh::KTILE), PA_KEYS * 128);
                if (lead) {
#pragma unroll
                    for (int k = 0; k < PA_KEYS / 16; k++)
                        mma_ts(tmem + PA_HALVES * PA_KEYS + t * DP, tmem + t * PA_KEYS + k * 8, vd + k * 2048 / 16, mma_shape(DP, true), add || k > 0);
                    mma_commit(&o_full[t]);
                }
                __syncwarp();
            };
            auto used = [&](unsigned i) {
                if (lead) mma_commit(&empty[stage(i)]);
                __syncwarp();
            };
            while (true) {
                const Piece& p = next();
                if (failed || p.stop) break;
                failed = !wait_soon_warp(&q_full, turn & 1);
                if (failed) break;
                const int n0 = p.n0, n1 = p.n1, from[PA_HALVES] = {p.from[0], p.from[1]}, to[PA_HALVES] = {p.to[0], p.to[1]};
                if (p.twin) {                            // p.from[0] is n0 and p.to[0] n1: all its key tiles are seen by some row
                    const unsigned n = n1 - n0;
                    for (unsigned i = 0; i < 2; i++)
                        if (arrived(x + i)) { scores(i, 0, x + i); used(x + i); }
                    if (n == 2 && lead) mma_commit(&q_empty);
                    for (unsigned i = 0; i < n; i++) {
                        const unsigned v = x + twin_value(i, n), k = x + twin_key(i + 2);
                        if (!arrived(v)) break;
                        outputs(i & 1, v, i >= 2);
                        used(v);
                        if (i + 2 < n && arrived(k)) { scores(i & 1, 0, k); used(k); }
                        if (i + 3 == n && lead) mma_commit(&q_empty);
                    }
                    x += 2 * n;
                } else {
                    arrived(x);
#pragma unroll
                    for (int t = 0; t < PA_HALVES; t++)
                        if (!failed && from[t] == n0 && to[t] > n0) scores(t, t, x);
                    used(x);
                    if (n0 + 1 == n1 && lead) mma_commit(&q_empty);
                    for (int n = n0; n < n1 && arrived(x + 1) && (n + 1 == n1 || arrived(x + 2)); n++, x += 2) {
#pragma unroll
                        for (int t = 0; t < PA_HALVES; t++) {
                            if (n >= from[t] && n < to[t]) outputs(t, x + 1, n > from[t]);
                            if (!failed && n + 1 >= from[t] && n + 1 < to[t]) scores(t, t, x + 2);
                        }
                        used(x + 1);
                        if (n + 1 < n1) used(x + 2);
                        if (n + 2 == n1 && lead) mma_commit(&q_empty);
                    }
                }
                if (failed) break;
                passed();
            }
            if (failed) s_fail = 1;
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

// The tile of rows that the end of a share is the first to cut, joined in the order of its parts; a warp to a row
constexpr int LJ_ROWS = 16;
__global__ void __launch_bounds__(256) line_join_kernel(PagedArgs a, RowShape rs, LinePlan plan, bf16* o) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    cudaGridDependencySynchronize();
    const Cut c = plan.cuts[blockIdx.x];
    for (int pr = blockIdx.y * LJ_ROWS + warp; pr < (blockIdx.y + 1) * LJ_ROWS; pr += 8) {
        const int half = pr / 128, r = pr % 128, token = r / rs.heads, g = r % rs.heads, tk = half * rs.tokens + token;
        if (token >= rs.tokens || tk >= c.tokens || g >= c.heads) continue;
        const Span sp = c.at0 >= 0 ? paged_keys_from(a, c.first, c.at0 + tk) : Span{0, 0};
        float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (int s0 = 0; s0 < c.shares; s0 += 32) {
            const int n = min(c.shares - s0, 32);
            float2 ml = make_float2(-INFINITY, 0.f);
            if (lane < n) ml = *reinterpret_cast<const float2*>(plan.part(blockIdx.x + s0 + lane, s0 + lane > 0 || c.begun, a.D) + (size_t)PA_ROWS * a.D + 2 * pr);
            float top = ml.x;
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, off));
            top = fmaxf(m, top);
            const float f = exp2f(m - top), weight = exp2f(ml.x - top);
            l = l * f + warp_sum(ml.y * weight);
            m = top;
#pragma unroll
            for (int e = 0; e < 4; e++) acc[e] *= f;
#pragma unroll 4
            for (int s = 0; s < n; s++) {
                const float* part = plan.part(blockIdx.x + s0 + s, s0 + s > 0 || c.begun, a.D) + (size_t)pr * a.D;
                const float w = __shfl_sync(FULL, weight, s);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (lane + 32 * e < a.D) acc[e] = fmaf(part[lane + 32 * e], w, acc[e]);
            }
        }
        bf16* to = o + ((size_t)(c.row0 + tk) * a.H + c.h0 + g) * a.D;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (lane + 32 * e < a.D) to[lane + 32 * e] = __float2bfloat16_rn(sp.hi > sp.lo ? acc[e] / l : 0.f);
    }
}

static RowShape row_shape(const PagedArgs& a) {
    const int group = a.H / a.KV, heads = group < 128 ? group : 128;
    return {heads, 128 / heads};
}
static long long most_tiles(const PagedArgs& a) { return a.N / (PA_HALVES * row_shape(a).tokens) + (long long)a.B; }

// one to an SM; fewer where the longest requests that the tables hold would not give each a tile of keys
static int line_ctas(const PagedArgs& a) {
    const int heads = row_shape(a).heads;
    const long long keys = (((long long)a.M << a.shift) + PA_KEYS - 1) / PA_KEYS, pairs = (long long)a.KV * ((a.H / a.KV + heads - 1) / heads);
    const long long tiles = most_tiles(a) < 148 ? most_tiles(a) : 148, most = (tiles * pairs * (PA_TILE_COST + PA_TWO * keys) + PA_TWO - 1) / PA_TWO;
    return (int)(most < 1 ? 1 : most < 148 ? most : 148);
}

size_t paged_attn_scratch_bf16(const PagedArgs& a) {
    return LinePlan::head_bytes() + sizeof(float) * line_ctas(a) * 2 * PA_ROWS * (size_t)(a.D + 2);
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
    const int ctas = line_ctas(a);
    kern<<<ctas, PA_THREADS, Sh::SMEM, st>>>(a, rs, plan, maps, (const bf16*)q, (const bf16*)k, (const bf16*)v, (bf16*)o);
    return ctas == 1 ? cudaGetLastError() : launch_behind(line_join_kernel, dim3(ctas - 1, PA_ROWS / LJ_ROWS), dim3(256), st, a, rs, plan, (bf16*)o);
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
