// Attention over tokens on the tensor cores, bf16: backward.
//
// The walk of the forward twice: with rows of queries (dq, and delta = <do, o>), then with rows of keys over the queries of all
// heads that share the key head (dk, dv).  Five products would do for both, with sums of dq by atomics; two walks take seven, have
// no atomics, and give the same bits from run to run.
//   rows X0, X1 / stream Y0, Y1:   queries: q, do / k, v      keys: k, v / q, do
//   s = X0 Y0^T, dp = X1 Y1^T, p = exp2(s - lse), ds = p (dp - delta) (1 - tanh^2),   out1 += ds Y0,  keys also out0 += p Y1
// A CTA holds 128 rows; the stream comes 128 at a time.  (With 64 at a time a product of 128 x 64 reads 6 KB of shared memory in 48
// cycles for 32 of sums, and the walk over keys took 720 us for one sequence of 16,384 with six heads of 128; it takes 638.)
//   copy warp     the tiles of the rows, then Y0 and Y1 through rings of their own: Y0 is needed first and let go last
//   product warp  between two steps' scores it runs the sums of the step before, so that it waits for weights only if they take longer
//                 than the products
//   16 warps      form the weights, a thread 32 columns of a row: p as soon as s is there, ds when dp is
// A barrier serves every step where its next round needs what the warp that waits on it does after the wait.  With rows of queries that
// does not hold for ds: both scores of a step are issued before the ds of the step before are waited for, so warps may hand over two
// steps' ds before the product warp looks at the first.  ds has two barriers in turn; the third step's needs the wait for the first.
// Tensor memory, 512 columns:  rows of queries:  s | dp | dq | 2 x ds;   rows of keys:  s, p written over it | dp, ds over it | dk | dv
// Weights are bf16 where the sums' products read them as their first operand; a group of 32 columns' weights lie where its scores
// lay, which its own threads have read.  One rounding of ds to bf16 costs dq and dk about as much as their own rounding; ds as a sum of
// two would take a fourth product of three, and a fifth of four.
#include <type_traits>

#include "slotscan_attn.cuh"
#include "slotscan_launch.h"
#include "slotscan_tensor.cuh"

namespace slotscan {

static __device__ int g_attn_bwd_status = 0;             // a bounded wait gave up (slotscan_device_status)

constexpr int AB_N = 128;                                // rows of a step of the stream
constexpr int AB_WARPS = 16;                             // that form weights: four groups of four, 32 columns to a group
constexpr int AB_R0 = 3, AB_R1 = 2;                      // tiles in the rings

template <int DP>
struct BwdShape {
    static constexpr int SUBS = DP / 64;
    static constexpr int TILE = 128 * DP * 2;            // bytes
    static constexpr int THREADS = AB_WARPS * 32 + 128;
    static constexpr int SMEM = (2 + AB_R0 + AB_R1) * TILE + 2 * AB_N * 8;          // 231,424 at DP 128
};
struct BwdMaps { CUtensorMap x0, x1, y0, y1, d0, d1; };

template <int DP, bool KEYS, bool CAP, bool BIAS>
__global__ void __launch_bounds__(AB_WARPS * 32 + 128, 1)
attn_bwd_tensor_kernel(AttnArgs a, RowInputs<bf16> in, const __grid_constant__ BwdMaps maps, const bf16* o, const bf16* rest, const float* lse, float* delta, int tiles,
                       int tile_major) {
    typedef BwdShape<DP> Sh;
    extern __shared__ __align__(1024) char smem[];
    char *X0 = smem, *X1 = smem + Sh::TILE, *Y0 = X1 + Sh::TILE, *Y1 = Y0 + AB_R0 * Sh::TILE;
    float* s_stat = reinterpret_cast<float*>(Y1 + AB_R1 * Sh::TILE);               // [2][2][128] -lse, -delta of the stream's queries
    __shared__ uint64_t x_full, done, s_full, d_full, s_read, d_read, p_full, ds_full[2], full0[AB_R0], full1[AB_R1], empty0[AB_R0], empty1[AB_R1];
    __shared__ uint32_t s_tmem;
    __shared__ int s_fail;
    __shared__ TileSpan s_span;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31, group = a.H / a.KV;
    const int heads = (KEYS ? a.KV : a.H) * a.B, rows = KEYS ? a.Tk : a.Tq, off = a.Tk - a.Tq;
    const int at_tile = (int)(tile_major ? blockIdx.x / heads : blockIdx.x % tiles), tile = KEYS ? at_tile : tiles - 1 - at_tile;   // long ones first
    const int hb = (int)(tile_major ? blockIdx.x % heads : blockIdx.x / tiles);
    const int hx = hb % (heads / a.B), b = hb / (heads / a.B), hk = KEYS ? hx : hx / group, x0 = tile * 128;
    if (tid == 0) {
        mbar_init(&x_full, 1); mbar_init(&done, 1); mbar_init(&s_full, 1); mbar_init(&d_full, 1);
        mbar_init(&s_read, AB_WARPS); mbar_init(&d_read, AB_WARPS); mbar_init(&p_full, AB_WARPS);
        for (int i = 0; i < 2; i++) mbar_init(&ds_full[i], AB_WARPS);
        for (int i = 0; i < AB_R0; i++) { mbar_init(&full0[i], 1); mbar_init(&empty0[i], 1); }
        for (int i = 0; i < AB_R1; i++) { mbar_init(&full1[i], 1); mbar_init(&empty1[i], 1); }
        mbar_fence_init();
        tile_span_reset(&s_span);
        s_fail = 0;
    }
    if (warp == AB_WARPS) tmem_alloc(&s_tmem, 512);
    __syncthreads();
    const int r = tid % 128, row = x0 + r;               // of the threads that form weights
    Span sp = {0, 0};
    if (warp < AB_WARPS) {
        if (row < rows) sp = KEYS ? queries_of(a, b, row) : keys_of(a, b, row);
        if (warp < 4) tile_span_add(&s_span, sp, row < rows);
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    constexpr uint32_t tmem = 0;                         // all 512 columns are this CTA's, so they begin at the first
    const TileSpan ts = s_span;
    const int y_first = ts.hi_max > 0 ? ts.lo_min / AB_N : 0, y_tiles = ts.hi_max > 0 ? (ts.hi_max + AB_N - 1) / AB_N - y_first : 0;
    const int steps = y_tiles * (KEYS ? group : 1);
    if (warp < AB_WARPS) {                               // ---- weights ----
        const int cg = warp / 4;                         // columns 32 cg ..
        const uint32_t lane_at = (uint32_t)((warp % 4) * 32) << 16;
        const uint32_t S = tmem + cg * 32 + lane_at;
        const int at = KEYS ? row - off : row + off;     // this row's place among the stream's
        bool ok = true;
        float my_lse = 0.f, my_delta = 0.f;              // negated
        if constexpr (!KEYS) {
            // delta of the row, a quarter of its channels to each group
            if (row < rows) my_lse = -lse[((size_t)b * a.H + hx) * a.Tq + row];
            uint4 ov[DP / 32], rv[DP / 32];
            const size_t at_o = (((size_t)b * a.Tq + row) * a.H + hx) * a.D + cg * (DP / 4);
#pragma unroll
            for (int i = 0; i < DP / 32; i++) {
                const bool in = row < rows && cg * (DP / 4) + i * 8 < a.D;
                ov[i] = in ? *reinterpret_cast<const uint4*>(o + at_o + i * 8) : make_uint4(0u, 0u, 0u, 0u);
                rv[i] = in ? *reinterpret_cast<const uint4*>(rest + at_o + i * 8) : make_uint4(0u, 0u, 0u, 0u);
            }
            float s = 0.f;
            if (steps > 0) {
                ok = wait_soon_warp(&x_full, 0);
#pragma unroll
                for (int i = 0; i < DP / 32; i++) {
                    const int d = cg * (DP / 4) + i * 8;
                    float x[8], y[8], z[8];
                    ld8(x, reinterpret_cast<const bf16*>(&ov[i]));
                    ld8(y, reinterpret_cast<const bf16*>(&rv[i]));
                    ld8(z, reinterpret_cast<const bf16*>(X1 + (d / 64) * 128 * 128 + swizzled(r, d % 64 / 8)));
#pragma unroll
                    for (int e = 0; e < 8; e++) s = fmaf(x[e] + y[e], z[e], s);
                }
            }
            float* ex = s_stat;
            ex[cg * 128 + r] = s;
            sync_group(1, AB_WARPS * 32);
            my_delta = (ex[r] + ex[128 + r]) + (ex[256 + r] + ex[384 + r]);
            if (warp < 4 && row < rows) delta[((size_t)b * a.H + hx) * a.Tq + row] = my_delta;
            my_delta = -my_delta;
        }
        // lse and delta of the step's queries: a thread of a group fetches one of its 32 columns' a step ahead
        int head = KEYS ? hk * group : hx, y_at = 0;     // of the step: head, tile of the stream
        float next = 0.f;
        auto fetch = [&] {
            const int i = (y_first + y_at) * AB_N + cg * 32 + r % 32;
            if (r < 64) next = i < a.Tq ? -(r < 32 ? lse : delta)[((size_t)b * a.H + head) * a.Tq + i] : 0.f;
        };
        if (KEYS && steps > 0) fetch();
        for (int s = 0; s < steps; s++) {
            const int y0 = (y_first + y_at) * AB_N + cg * 32;
            const float ahead = (float)(at - y0);        // float32 does not hold the places beyond 2^24
            const Score sc(a, head);
            const bool masked = y0 < ts.lo_max || y0 + 32 > ts.hi_min;
            float* stat = s_stat + (s & 1) * 2 * AB_N + cg * 32;
            if (++y_at == y_tiles) { y_at = 0; head++; }
            if constexpr (KEYS) {
                if (r < 64) stat[r / 32 * AB_N + r % 32] = next;
                if (s + 1 < steps) fetch();
                sync_group(2 + cg, 128);
            }
            const int lo = sp.lo - y0, hi = sp.hi - y0;
            uint32_t xs[32];                             // s, then p (1 - tanh^2)
            // a warp that has given up stays with its group's barrier, at which the others would wait for it without a limit
            if (!(ok = ok && wait_soon_warp(&s_full, s & 1))) continue;
            tmem_fence_after();
            tmem_ld(S, xs);
            tmem_ld_wait(xs);
            if constexpr (!KEYS) {
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) arrive(&s_read);
            }
            bool small = true;                           // the capped scores' polynomial serves this warp's block
            if constexpr (CAP) {
                float m0 = 0.f, m1 = 0.f;
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    m0 = fmaxf(m0, fabsf(__uint_as_float(xs[i])));
                    m1 = fmaxf(m1, fabsf(__uint_as_float(xs[i + 1])));
                }
                small = __all_sync(FULL, fmaxf(m0, m1) * sc.cap_in <= CAP_POLY_MOST);
            }
            auto weights = [&](auto poly, auto some) {   // some: of the block's scores are masked
                const CapPoly cp(sc);
                const f32x2 lin = pack2(sc.lin, sc.lin), steep = pack2(-sc.slope, -sc.slope), one = pack2(1.f, 1.f);
                const float in2 = -1.f / (sc.cap_out * sc.cap_out);
                [[maybe_unused]] uint32_t wp[16];
                [[maybe_unused]] float4 four;
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    float L[2] = {my_lse, my_lse};
                    if constexpr (KEYS) {                // four at a time: the products want the shared memory's cycles
                        if (i % 4 == 0) four = ld4(stat + i);
                        L[0] = i % 4 ? four.z : four.x; L[1] = i % 4 ? four.w : four.y;
                    }
                    const f32x2 x = pack2(__uint_as_float(xs[i]), __uint_as_float(xs[i + 1]));
                    f32x2 z, f = one;
                    if constexpr (CAP && decltype(poly)::value) {
                        const f32x2 y = mul2(x, cp.slope(x));
                        z = add2(y, pack2(L[0], L[1]));
                        f = fma2(mul2(y, y), pack2(in2, in2), one);
                    } else if constexpr (CAP) {          // tanh x = 1 - 2 r, 1 - tanh^2 = 4 r (1 - r),  r = 1 / (e^2x + 1)
                        float zz[2], ff[2];
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const float rr = rcp_fast(exp2_fast(__uint_as_float(xs[i + e]) * (2.f * LOG2E * sc.cap_in)) + 1.f);
                            zz[e] = fmaf(-2.f * sc.cap_out, rr, sc.cap_out) + L[e];
                            ff[e] = 4.f * fmaf(-rr, rr, rr);
                        }
                        z = pack2(zz[0], zz[1]);
                        f = pack2(ff[0], ff[1]);
                    } else z = fma2(x, lin, pack2(L[0], L[1]));
                    if constexpr (BIAS) z = fma2(pack2(fabsf(ahead - (float)i), fabsf(ahead - (float)(i + 1))), steep, z);
                    const float2 zf = unpack2(z);
                    float2 p = make_float2(exp2_fast(zf.x), exp2_fast(zf.y));
                    float2 pf = p;
                    if constexpr (CAP) pf = unpack2(mul2(pack2(p.x, p.y), f));
                    if constexpr (decltype(some)::value) {
                        // a query that sees one key alone has weight 1, and its scores no gradient
                        const bool in0 = i >= lo && i < hi, in1 = i + 1 >= lo && i + 1 < hi, alone0 = L[0] == -INFINITY, alone1 = L[1] == -INFINITY;
                        p = make_float2(in0 ? (alone0 ? 1.f : p.x) : 0.f, in1 ? (alone1 ? 1.f : p.y) : 0.f);
                        pf = make_float2(in0 && !alone0 ? pf.x : 0.f, in1 && !alone1 ? pf.y : 0.f);
                    }
                    if constexpr (KEYS) wp[i / 2] = pack_bf16(p.x, p.y);
                    xs[i] = __float_as_uint(pf.x);
                    xs[i + 1] = __float_as_uint(pf.y);
                }
                if constexpr (KEYS) tmem_st(S, wp);
            };
            if (small) {
                if (masked) weights(std::true_type{}, std::true_type{});
                else weights(std::true_type{}, std::false_type{});
            } else if constexpr (CAP) weights(std::false_type{}, std::true_type{});
            if constexpr (KEYS) {
                tmem_st_wait();
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) arrive(&p_full);
            }
            if (!(ok = wait_soon_warp(&d_full, s & 1))) continue;
            tmem_fence_after();
            uint32_t xd[32], wd[16];
            [[maybe_unused]] float4 four;
            tmem_ld(S + 128, xd);
            tmem_ld_wait(xd);
            if constexpr (!KEYS) {
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) arrive(&d_read);
            }
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
                float dl[2] = {my_delta, my_delta};
                if constexpr (KEYS) {
                    if (i % 4 == 0) four = ld4(stat + AB_N + i);
                    dl[0] = i % 4 ? four.z : four.x; dl[1] = i % 4 ? four.w : four.y;
                }
                float2 ds = unpack2(mul2(pack2(__uint_as_float(xs[i]), __uint_as_float(xs[i + 1])),
                                         add2(pack2(__uint_as_float(xd[i]), __uint_as_float(xd[i + 1])), pack2(dl[0], dl[1]))));
                if (masked) {                            // nothing of a hidden dp, infinities and NaN among them
                    if (xs[i] == 0u) ds.x = 0.f;
                    if (xs[i + 1] == 0u) ds.y = 0.f;
                }
                wd[i / 2] = pack_bf16(ds.x, ds.y);
            }
            tmem_st(KEYS ? S + 128 : tmem + 384 + (s & 1) * 64 + cg * 16 + lane_at, wd);
            tmem_st_wait();
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) arrive(&ds_full[s & 1]);
        }
        if (ok && steps > 0) ok = wait_soon(&done, 0);
        tmem_fence_after();
        if (!ok) s_fail = 1;
        // results through the tiles of the rows, whose products are done: two groups take a result each (keys) or half the columns each
        const bool mine = cg < 2 && (KEYS || DP == 128 || cg == 0);
        const int c0 = KEYS || DP == 64 ? 0 : cg, c1 = KEYS || DP == 64 ? Sh::SUBS : cg + 1;
        const uint32_t from = tmem + 256 + lane_at + (KEYS && cg == 0 ? DP : 0);
        const float mul = KEYS && cg == 0 ? 1.f : a.scale;
        char* out = KEYS && cg == 1 ? X1 : X0;
        if (mine) {
            float seen = 0.f;
            for (int c = c0 * 2; c < c1 * 2; c++) {
                uint32_t x[32];
                if (steps > 0) { tmem_ld(from + c * 32, x); tmem_ld_wait(x); }
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    uint32_t y[4];
                    if (steps > 0) {
#pragma unroll
                        for (int e = 0; e < 8; e++) watch(seen, __uint_as_float(x[i + e]));
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        y[e] = steps > 0 ? pack_bf16(__uint_as_float(x[i + 2 * e]) * mul, __uint_as_float(x[i + 2 * e + 1]) * mul) : 0u;
                    *reinterpret_cast<uint4*>(out + (c / 2) * 128 * 128 + swizzled(r, (c % 2) * 4 + i / 8)) = make_uint4(y[0], y[1], y[2], y[3]);
                }
            }
            for (unsigned bad = __ballot_sync(FULL, seen != seen && row < rows); bad != 0; bad &= bad - 1) {
                const int n = __ffs(bad) - 1, nr = r - lane + n;
                float x[4], y[4];
                if constexpr (KEYS) careful_dkv(a, in, lse, delta, b, hx, row - lane + n, x, y);
                else careful_dq(a, in, lse, delta, b, hx, row - lane + n, x);
#pragma unroll
                for (int c = 0; c < DP / 32; c++) {
                    const int d = lane + 32 * c;
                    if (d / 64 >= c0 && d / 64 < c1)
                        *reinterpret_cast<bf16*>(out + (d / 64) * 128 * 128 + swizzled(nr, d % 64 / 8) + d % 8 * 2) = __float2bfloat16_rn(KEYS && cg == 0 ? y[c] : x[c]);
                }
            }
            fence_proxy_async_smem();
            sync_group(2 + cg, 128);
            if (r == 0) {
                for (int c = c0; c < c1; c++) tile_s2g(KEYS && cg == 0 ? &maps.d0 : &maps.d1, c * 64, x0, hx, b, out + c * 128 * 128);
                bulk_commit();
                bulk_wait_read<0>();
            }
        }
    } else {
        if (warp == AB_WARPS + 1 && lane == 0 && steps > 0) {                      // ---- copies ----
            bool ok = true;
            auto tile_in = [&](char* to, const CUtensorMap* map, int y, int head, uint64_t* bar) {
                for (int c = 0; c < Sh::SUBS; c++) tile_g2s(to + c * 128 * 128, map, c * 64, y, head, b, bar);
            };
            mbar_arrive_expect_tx(&x_full, 2 * Sh::TILE);
            tile_in(X0, &maps.x0, x0, hx, &x_full);
            tile_in(X1, &maps.x1, x0, hx, &x_full);
            for (int s = 0, head = KEYS ? hk * group : hk, y_at = 0; s < steps; s++) {
                const int u = s % AB_R0, v = s % AB_R1, y0 = (y_first + y_at) * AB_N;
                if (s >= AB_R0 && !(ok = wait_soon(&empty0[u], (s / AB_R0 - 1) & 1))) break;
                mbar_arrive_expect_tx(&full0[u], Sh::TILE);
                tile_in(Y0 + u * Sh::TILE, &maps.y0, y0, head, &full0[u]);
                if (s >= AB_R1 && !(ok = wait_soon(&empty1[v], (s / AB_R1 - 1) & 1))) break;
                mbar_arrive_expect_tx(&full1[v], Sh::TILE);
                tile_in(Y1 + v * Sh::TILE, &maps.y1, y0, head, &full1[v]);
                if (++y_at == y_tiles) { y_at = 0; head++; }
            }
            if (!ok) s_fail = 1;
        } else if (warp == AB_WARPS && steps > 0) {      // ---- products ----
            const uint32_t x0d = tile_desc(smem_u32(X0), 16), x1d = tile_desc(smem_u32(X1), 16);
            const bool lead = elected();
            // s (x = 0) or dp of a step
            auto scores = [&](int s, int x) {
                const int u = x ? s % AB_R1 : s % AB_R0;
                if (!wait_soon_warp(x ? &full1[u] : &full0[u], (x ? s / AB_R1 : s / AB_R0) & 1)) return false;
                const uint32_t yd = tile_desc(smem_u32((x ? Y1 : Y0) + u * Sh::TILE), 16), xd = x ? x1d : x0d;
                if (lead) {
#pragma unroll
                    for (int k = 0; k < DP / 16; k++) {
                        const int step = ((k / 4) * 128 * 128 + (k % 4) * 32) / 16;
                        mma_ss(tmem + x * 128, xd + step, yd + step, mma_shape(AB_N, false), k > 0);
                    }
                    mma_commit(x ? &d_full : &s_full);
                    if (!KEYS && x) mma_commit(&empty1[u]);
                }
                __syncwarp();
                return true;
            };
            // out1 += ds Y0 (x = 0), out0 += p Y1
            auto sums = [&](int s, int x) {
                const uint32_t yd = tile_desc(smem_u32(x ? Y1 + s % AB_R1 * Sh::TILE : Y0 + s % AB_R0 * Sh::TILE), 128 * 128);
                const uint32_t w = KEYS ? tmem + (x ? 0 : 128) : tmem + 384 + (s & 1) * 64;
                if (lead) {
#pragma unroll
                    for (int k = 0; k < AB_N / 16; k++)
                        mma_ts(tmem + 256 + x * DP, w + (KEYS ? (k / 2) * 32 + (k % 2) * 8 : k * 8), yd + k * 2048 / 16, mma_shape(DP, true), s > 0 || k > 0);
                    mma_commit(x ? &empty1[s % AB_R1] : &empty0[s % AB_R0]);
                }
                __syncwarp();
            };
            bool ok = wait_soon_warp(&x_full, 0) && scores(0, 0) && scores(0, 1);
            for (int s = 0; s < steps && ok; s++) {
                const bool more = s + 1 < steps;
                if constexpr (KEYS) {
                    if (!(ok = wait_soon_warp(&p_full, s & 1))) break;
                    tmem_fence_after();
                    sums(s, 1);
                    if (more && !(ok = scores(s + 1, 0))) break;
                    if (!(ok = wait_soon_warp(&ds_full[s & 1], (s >> 1) & 1))) break;
                    tmem_fence_after();
                    sums(s, 0);
                    if (more && !(ok = scores(s + 1, 1))) break;
                } else {
                    if (more) {
                        if (!(ok = wait_soon_warp(&s_read, s & 1))) break;
                        tmem_fence_after();
                        if (!(ok = scores(s + 1, 0))) break;
                        if (!(ok = wait_soon_warp(&d_read, s & 1))) break;
                        tmem_fence_after();
                        if (!(ok = scores(s + 1, 1))) break;
                    }
                    if (!(ok = wait_soon_warp(&ds_full[s & 1], (s >> 1) & 1))) break;
                    tmem_fence_after();
                    sums(s, 0);
                }
            }
            if (lead) mma_commit(&done);
            __syncwarp();
            if (!ok) s_fail = 1;
        }
    }
    tmem_fence_before();
    __syncthreads();
    if (s_fail != 0) {                                   // report, and give copies and products in flight time to land
        if (tid == 0) atomicExch(&g_attn_bwd_status, 1);
        for (int i = 0; i < 1000; i++) __nanosleep(1000);
    }
    if (warp == AB_WARPS) { tmem_fence_after(); tmem_free(s_tmem, 512); }
}

template <int DP, bool CAP, bool BIAS>
static cudaError_t bwd_tensor(const AttnArgs& a, const void* q, const void* k, const void* v, const void* o, const void* rest, const float* lse,
                              const void* dout, float* delta, void* dq, void* dk, void* dv, cudaStream_t st) {
    typedef BwdShape<DP> Sh;
    auto rows_q = attn_bwd_tensor_kernel<DP, false, CAP, BIAS>;
    auto rows_k = attn_bwd_tensor_kernel<DP, true, CAP, BIAS>;
    cudaError_t e = opt_in_smem(rows_q, Sh::SMEM);       // before the maps: a thread's first runtime call makes the context current for them
    if (e == cudaSuccess) e = opt_in_smem(rows_k, Sh::SMEM);
    if (e != cudaSuccess) return e;
    const long long os[3] = {(long long)a.Tq * a.H * a.D, (long long)a.H * a.D, a.D}, gs[3] = {(long long)a.Tk * a.KV * a.D, (long long)a.KV * a.D, a.D};
    BwdMaps mq, mk;
    if (!tile_map(&mq.x0, q, a.B, a.Tq, a.H, a.D, a.qs, 128) || !tile_map(&mq.x1, dout, a.B, a.Tq, a.H, a.D, os, 128) ||
        !tile_map(&mq.y0, k, a.B, a.Tk, a.KV, a.D, a.ks, AB_N) || !tile_map(&mq.y1, v, a.B, a.Tk, a.KV, a.D, a.vs, AB_N) ||
        !tile_map(&mq.d1, dq, a.B, a.Tq, a.H, a.D, os, 128))
        return cudaErrorInvalidValue;
    mq.d0 = mq.d1;
    if (!tile_map(&mk.x0, k, a.B, a.Tk, a.KV, a.D, a.ks, 128) || !tile_map(&mk.x1, v, a.B, a.Tk, a.KV, a.D, a.vs, 128) ||
        !tile_map(&mk.y0, q, a.B, a.Tq, a.H, a.D, a.qs, AB_N) || !tile_map(&mk.y1, dout, a.B, a.Tq, a.H, a.D, os, AB_N) ||
        !tile_map(&mk.d0, dv, a.B, a.Tk, a.KV, a.D, gs, 128) || !tile_map(&mk.d1, dk, a.B, a.Tk, a.KV, a.D, gs, 128))
        return cudaErrorInvalidValue;
    const RowInputs<bf16> in = {(const bf16*)q, (const bf16*)k, (const bf16*)v, (const bf16*)dout};
    const int tq = (a.Tq + 127) / 128, tk = (a.Tk + 127) / 128;
    const long long cq = (long long)tq * a.H * a.B, ck = (long long)tk * a.KV * a.B;
    if (cq > 0x7fffffffll || ck > 0x7fffffffll) return cudaErrorInvalidValue;
    rows_q<<<(unsigned)cq, Sh::THREADS, Sh::SMEM, st>>>(a, in, mq, (const bf16*)o, (const bf16*)rest, lse, delta, tq, cq < 148 * 8);
    rows_k<<<(unsigned)ck, Sh::THREADS, Sh::SMEM, st>>>(a, in, mk, nullptr, nullptr, lse, delta, tk, ck < 148 * 8);
    return cudaGetLastError();
}
template <int DP>
static cudaError_t bwd_tensor_score(const AttnArgs& a, const void* q, const void* k, const void* v, const void* o, const void* rest, const float* lse,
                                    const void* dout, float* delta, void* dq, void* dk, void* dv, cudaStream_t st) {
    if (a.cap > 0.f)
        return a.slopes != nullptr ? bwd_tensor<DP, true, true>(a, q, k, v, o, rest, lse, dout, delta, dq, dk, dv, st)
                                   : bwd_tensor<DP, true, false>(a, q, k, v, o, rest, lse, dout, delta, dq, dk, dv, st);
    return a.slopes != nullptr ? bwd_tensor<DP, false, true>(a, q, k, v, o, rest, lse, dout, delta, dq, dk, dv, st)
                               : bwd_tensor<DP, false, false>(a, q, k, v, o, rest, lse, dout, delta, dq, dk, dv, st);
}

cudaError_t run_attn_bwd_bf16(const AttnArgs& a, const void* q, const void* k, const void* v, const void* o, const void* rest, const float* lse,
                              const void* dout, float* delta, void* dq, void* dk, void* dv, cudaStream_t st) {
    return a.D <= 64 ? bwd_tensor_score<64>(a, q, k, v, o, rest, lse, dout, delta, dq, dk, dv, st)
                     : bwd_tensor_score<128>(a, q, k, v, o, rest, lse, dout, delta, dq, dk, dv, st);
}

int attn_bwd_mma_status() {
    int v = 0;
    const int z = 0;
    if (cudaMemcpyFromSymbol(&v, g_attn_bwd_status, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) cudaMemcpyToSymbol(g_attn_bwd_status, &z, sizeof(int));
    return v;
}

}  // namespace slotscan
