// Attention over tokens on the tensor cores, bf16: backward.
//
// The walk of the forward twice: with rows of queries (dq, and delta = <do, o>), then with rows of keys over the queries of all
// heads that share the key head (dk, dv).  Five products would do for both, with sums of dq by atomics; two walks take seven, have
// no atomics, and give the same bits from run to run.
//   rows X0, X1 / stream Y0, Y1:   queries: q, do / k, v      keys: k, v / q, do
//   s = X0 Y0^T, dp = X1 Y1^T, p = exp2(s - lse), ds = p (dp - delta) (1 - tanh^2),   out1 += ds Y0,  keys also out0 += p Y1
// A CTA holds 128 rows; the stream comes 64 at a time.  Tensor memory holds one step's scores and dp, and two steps' weights: warps
// read s and dp into registers, whereupon the products of the next step's run while the weights p and ds are formed; these are
// written as bf16 where the sums' products read them as their first operand, and the next weights meanwhile go to the other
// place.  (With the weights written over the scores, the next scores wait for the sums: 2,290 cycles a step instead of @@STEP@@.)
// A product of 128 x 64 with both operands in shared memory is bound by reading them (6 KB, 48 cycles, for 32 cycles of sums).  With
// rows of queries there is room in tensor memory for the rows, so they are copied there once and only the stream is read; with
// rows of keys the two results fill it.
#include <type_traits>

#include "slotscan_attn.cuh"
#include "slotscan_launch.h"
#include "slotscan_tensor.cuh"

namespace slotscan {

static __device__ int g_attn_bwd_status = 0;             // a bounded wait gave up (slotscan_device_status)

constexpr int AB_N = 64;                                 // rows of a step of the stream
constexpr int AB_WARPS = 16;                             // that form weights
constexpr int AB_COLS = AB_N * 4 / AB_WARPS;             // of a step to a thread

template <int DP>
struct BwdShape {
    static constexpr int STAGES = 4;
    static constexpr int SUBS = DP / 64;
    static constexpr int XTILE = 128 * DP * 2, YTILE = AB_N * DP * 2;
    static constexpr int THREADS = AB_WARPS * 32 + 128;
    static constexpr int SMEM = 2 * XTILE + STAGES * 2 * YTILE + 1024;
};
struct BwdMaps { CUtensorMap x0, x1, y0, y1, d0, d1; };

template <int DP, bool KEYS, bool CAP, bool BIAS>
__global__ void __launch_bounds__(AB_WARPS * 32 + 128, 1)
attn_bwd_tensor_kernel(AttnArgs a, const __grid_constant__ BwdMaps maps, const bf16* o, const bf16* rest, const bf16* dout, const float* lse,
                       float* delta, int tiles, int tile_major) {
    typedef BwdShape<DP> Sh;
    extern __shared__ char smem_raw[];
    char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    char *X0 = smem, *X1 = smem + Sh::XTILE, *Ys = smem + 2 * Sh::XTILE;
    __shared__ uint64_t x_full, x_moved, done, s_full, s_read, p_full[2], full[Sh::STAGES], empty[Sh::STAGES];
    __shared__ uint32_t s_tmem;
    __shared__ int s_fail;
    __shared__ TileSpan s_span;
    __shared__ __align__(16) float s_stat[AB_WARPS][2][2][AB_COLS];    // warp, buffer, -lse / -delta
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31, group = a.H / a.KV;
    const int heads = (KEYS ? a.KV : a.H) * a.B, rows = KEYS ? a.Tk : a.Tq, off = a.Tk - a.Tq;
    const int at_tile = (int)(tile_major ? blockIdx.x / heads : blockIdx.x % tiles), tile = KEYS ? at_tile : tiles - 1 - at_tile;   // long ones first
    const int hb = (int)(tile_major ? blockIdx.x % heads : blockIdx.x / tiles);
    const int hx = hb % (heads / a.B), b = hb / (heads / a.B), hk = KEYS ? hx : hx / group, x0 = tile * 128;
    if (tid == 0) {
        mbar_init(&x_full, 1); mbar_init(&x_moved, 8); mbar_init(&done, 1);
        mbar_init(&s_full, 1); mbar_init(&s_read, AB_WARPS); mbar_init(&p_full[0], AB_WARPS); mbar_init(&p_full[1], AB_WARPS);
        for (int s = 0; s < Sh::STAGES; s++) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        mbar_fence_init();
        tile_span_reset(&s_span);
        s_fail = 0;
    }
    if (warp == AB_WARPS) tmem_alloc(&s_tmem, 512);
    __syncthreads();
    const int r = tid % 128, row = x0 + r;               // of the threads that form weights: groups of 128, some columns each
    Span sp = {0, 0};
    if (warp < AB_WARPS) {
        if (row < rows) sp = KEYS ? queries_of(a, b, row) : keys_of(a, b, row);
        if (warp < 4) tile_span_add(&s_span, sp, row < rows);
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = s_tmem;
    const TileSpan ts = s_span;
    const int y_first = ts.hi_max > 0 ? ts.lo_min / AB_N : 0, y_tiles = ts.hi_max > 0 ? (ts.hi_max + AB_N - 1) / AB_N - y_first : 0;
    const int steps = y_tiles * (KEYS ? group : 1);
    if (warp < AB_WARPS) {                               // ---- weights ----
        const int w = warp / 4;
        const uint32_t lane_at = (uint32_t)((warp % 4) * 32) << 16;
        const float at = (float)(KEYS ? row - off : row + off);                    // this row's place among the stream's
        bool ok = true;
        float my_lse = 0.f, my_delta = 0.f;
        if constexpr (!KEYS) {
            // delta of the row, half of its channels to each of two groups; the rows into tensor memory, q by one group and do by the other
            float* ex = &s_stat[0][0][0][0];             // used here only, before the first step
            if (row < rows) my_lse = lse[((size_t)b * a.H + hx) * a.Tq + row];
            if (w < 2) {
                uint4 ov[DP / 16], rv[DP / 16];
                const size_t at_o = (((size_t)b * a.Tq + row) * a.H + hx) * a.D + w * (DP / 2);
#pragma unroll
                for (int i = 0; i < DP / 16; i++) {
                    const bool in = row < rows && w * (DP / 2) + i * 8 < a.D;
                    ov[i] = in ? *reinterpret_cast<const uint4*>(o + at_o + i * 8) : make_uint4(0u, 0u, 0u, 0u);
                    rv[i] = in ? *reinterpret_cast<const uint4*>(rest + at_o + i * 8) : make_uint4(0u, 0u, 0u, 0u);
                }
                ok = wait_soon_warp(&x_full, 0);
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < DP / 16; i++) {
                    const int d = w * (DP / 2) + i * 8;
                    float x[8], y[8], z[8];
                    ld8(x, reinterpret_cast<const bf16*>(&ov[i]));
                    ld8(y, reinterpret_cast<const bf16*>(&rv[i]));
                    ld8(z, reinterpret_cast<const bf16*>(X1 + (d / 64) * 128 * 128 + swizzled(r, d % 64 / 8)));
#pragma unroll
                    for (int e = 0; e < 8; e++) s = fmaf(x[e] + y[e], z[e], s);
                }
                ex[w * 128 + r] = s;
                const char* x = w ? X1 : X0;
#pragma unroll
                for (int c = 0; c < DP / 32; c++) {
                    uint32_t y[16];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint4 u = *reinterpret_cast<const uint4*>(x + (c / 2) * 128 * 128 + swizzled(r, (c % 2) * 4 + i));
                        y[4 * i] = u.x; y[4 * i + 1] = u.y; y[4 * i + 2] = u.z; y[4 * i + 3] = u.w;
                    }
                    tmem_st(tmem + 384 + w * 64 + lane_at + c * 16, y);
                }
                tmem_st_wait();
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) arrive(&x_moved);
            }
            sync_group(3, AB_WARPS * 32);
            my_delta = ex[r] + ex[128 + r];
            if (w == 0 && row < rows) delta[((size_t)b * a.H + hx) * a.Tq + row] = my_delta;
            my_lse = -my_lse; my_delta = -my_delta;
        }
        // lse and delta of the step's queries that this thread's columns belong to: a lane fetches one of each, a step ahead
        int head = KEYS ? hk * group : hx, y_at = 0;     // of the step: head, tile of the stream
        float next_lse = 0.f, next_delta = 0.f;
        auto fetch = [&](int h, int y) {
            const int i = (y_first + y) * AB_N + w * AB_COLS + lane % AB_COLS;
            const size_t from = ((size_t)b * a.H + h) * a.Tq + i;
            next_lse = i < a.Tq ? -lse[from] : 0.f;
            next_delta = i < a.Tq ? -delta[from] : 0.f;
        };
        if (KEYS && steps > 0) fetch(head, 0);
        for (int s = 0; s < steps; s++) {
            const int buf = s & 1, y0 = (y_first + y_at) * AB_N + w * AB_COLS;
            const uint32_t S = tmem + w * AB_COLS + lane_at, P = tmem + 128 + buf * 64 + w * (AB_COLS / 2) + lane_at;
            const Score sc(a, head);
            const bool masked = y0 < ts.lo_max || y0 + AB_COLS > ts.hi_min;
            float* stat = &s_stat[warp][buf][0][0];
            if (++y_at == y_tiles) { y_at = 0; head++; }
            if constexpr (KEYS) {
                if (lane < AB_COLS) { stat[lane] = next_lse; stat[AB_COLS + lane] = next_delta; }
                __syncwarp();
                if (s + 1 < steps) fetch(head, y_at);
            }
            if (!(ok = __all_sync(FULL, ok && wait_soon(&s_full, s & 1)))) break;
            tmem_fence_after();
            uint32_t xs[AB_COLS], xd[AB_COLS], wp[AB_COLS / 2], wd[AB_COLS / 2];
            tmem_ld(S, xs);
            tmem_ld(S + 64, xd);
            tmem_ld_wait(xs);
            tmem_ld_wait(xd);
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) arrive(&s_read);
            const int lo = sp.lo - y0, hi = sp.hi - y0;
            const float ahead = at - (float)y0;
            bool small = true;                           // the capped scores' polynomial serves this warp's block
            if constexpr (CAP) {
                float m0 = 0.f, m1 = 0.f;
#pragma unroll
                for (int i = 0; i < AB_COLS; i += 2) {
                    m0 = fmaxf(m0, fabsf(__uint_as_float(xs[i])));
                    m1 = fmaxf(m1, fabsf(__uint_as_float(xs[i + 1])));
                }
                small = __all_sync(FULL, fmaxf(m0, m1) * sc.cap_in <= 1.f);
            }
            auto weights = [&](auto poly) {
                const CapPoly cp(sc);
                const f32x2 lin = pack2(sc.lin, sc.lin), steep = pack2(-sc.slope, -sc.slope), one = pack2(1.f, 1.f);
                const f32x2 k2 = pack2(-1.f / (sc.cap_out * sc.cap_out), -1.f / (sc.cap_out * sc.cap_out));
#pragma unroll
                for (int i = 0; i < AB_COLS; i += 2) {
                    float L[2] = {my_lse, my_lse}, dl[2] = {my_delta, my_delta};
                    if constexpr (KEYS) {
                        const float2 u = *reinterpret_cast<const float2*>(stat + i), v = *reinterpret_cast<const float2*>(stat + AB_COLS + i);
                        L[0] = u.x; L[1] = u.y; dl[0] = v.x; dl[1] = v.y;
                    }
                    const f32x2 x = pack2(__uint_as_float(xs[i]), __uint_as_float(xs[i + 1]));
                    f32x2 z, f = one;
                    if constexpr (CAP && decltype(poly)::value) {
                        const f32x2 y = mul2(x, cp.slope(x));
                        z = add2(y, pack2(L[0], L[1]));
                        f = fma2(mul2(y, y), k2, one);
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
                    f32x2 d = mul2(pack2(p.x, p.y), add2(pack2(__uint_as_float(xd[i]), __uint_as_float(xd[i + 1])), pack2(dl[0], dl[1])));
                    if constexpr (CAP) d = mul2(d, f);
                    float2 ds = unpack2(d);
                    if (masked) {
                        const bool in0 = i >= lo && i < hi, in1 = i + 1 >= lo && i + 1 < hi, alone0 = L[0] == -INFINITY, alone1 = L[1] == -INFINITY;
                        p = make_float2(in0 ? (alone0 ? 1.f : p.x) : 0.f, in1 ? (alone1 ? 1.f : p.y) : 0.f);
                        ds = make_float2(in0 && !alone0 ? ds.x : 0.f, in1 && !alone1 ? ds.y : 0.f);
                    }
                    wp[i / 2] = pack_bf16(p.x, p.y);
                    wd[i / 2] = pack_bf16(ds.x, ds.y);
                }
            };
            if (small) weights(std::true_type{});
            else if constexpr (CAP) weights(std::false_type{});
            if constexpr (KEYS) tmem_st(P, wp);
            tmem_st(P + 32, wd);
            tmem_st_wait();
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) arrive(&p_full[buf]);
        }
        if (ok && steps > 0) ok = wait_soon(&done, 0);
        tmem_fence_after();
        if (!ok) s_fail = 1;
        // results through the tiles of the rows, whose products are done: of keys, dv by one group and dk by the other; of queries half the
        // columns each, where there are two sub-tiles
        const bool mine = w < 2 && (KEYS || DP == 128 || w == 0);
        const int c0 = KEYS || DP == 64 ? 0 : w, c1 = KEYS || DP == 64 ? Sh::SUBS : w + 1;
        const uint32_t from = tmem + 256 + lane_at + (KEYS && w == 0 ? DP : 0);
        const float mul = KEYS && w == 0 ? 1.f : a.scale;
        char* out = KEYS && w == 1 ? X1 : X0;
        if (mine) {
            for (int c = c0 * 2; c < c1 * 2; c++) {
                uint32_t x[32];
                if (steps > 0) { tmem_ld(from + c * 32, x); tmem_ld_wait(x); }
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    uint32_t y[4];
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        y[e] = steps > 0 ? pack_bf16(__uint_as_float(x[i + 2 * e]) * mul, __uint_as_float(x[i + 2 * e + 1]) * mul) : 0u;
                    *reinterpret_cast<uint4*>(out + (c / 2) * 128 * 128 + swizzled(r, (c % 2) * 4 + i / 8)) = make_uint4(y[0], y[1], y[2], y[3]);
                }
            }
            fence_proxy_async_smem();
            sync_group(1 + w, 128);
            if (r == 0) {
                for (int c = c0; c < c1; c++) tile_s2g(KEYS && w == 0 ? &maps.d0 : &maps.d1, c * 64, x0, hx, b, out + c * 128 * 128);
                bulk_commit();
                bulk_wait_read<0>();
            }
        }
    } else if (warp == AB_WARPS + 1) {                   // ---- copies ----
        if (lane == 0 && steps > 0) {
            bool ok = true;
            mbar_arrive_expect_tx(&x_full, 2 * Sh::XTILE);
            for (int c = 0; c < Sh::SUBS; c++) {
                tile_g2s(X0 + c * 128 * 128, &maps.x0, c * 64, x0, hx, b, &x_full);
                tile_g2s(X1 + c * 128 * 128, &maps.x1, c * 64, x0, hx, b, &x_full);
            }
            for (int s = 0; s < steps; s++) {
                const int st = s % Sh::STAGES, turn = s / Sh::STAGES;
                if (turn > 0 && !(ok = wait_soon(&empty[st], (turn - 1) & 1))) break;
                const int head = KEYS ? hk * group + s / y_tiles : hk, y0 = (y_first + (KEYS ? s % y_tiles : s)) * AB_N;
                char* y = Ys + st * 2 * Sh::YTILE;
                mbar_arrive_expect_tx(&full[st], 2 * Sh::YTILE);
                for (int c = 0; c < Sh::SUBS; c++) {
                    tile_g2s(y + c * AB_N * 128, &maps.y0, c * 64, y0, head, b, &full[st]);
                    tile_g2s(y + Sh::YTILE + c * AB_N * 128, &maps.y1, c * 64, y0, head, b, &full[st]);
                }
            }
            if (!ok) s_fail = 1;
        }
    } else if (warp == AB_WARPS) {                       // ---- products ----
        if (steps > 0) {
            bool ok = wait_soon_warp(KEYS ? &x_full : &x_moved, 0);
            tmem_fence_after();
            const uint64_t x0d = tile_desc(smem_u32(X0), 16), x1d = tile_desc(smem_u32(X1), 16);
            auto scores = [&](int s) {                   // s and dp of a step
                const int st = s % Sh::STAGES;
                if (!wait_soon_warp(&full[st], (s / Sh::STAGES) & 1)) return false;
                const uint64_t yd = tile_desc(smem_u32(Ys + st * 2 * Sh::YTILE), 16);
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int k = 0; k < DP / 16; k++) {
                        const uint64_t y = yd + (x * Sh::YTILE + (k / 4) * AB_N * 128 + (k % 4) * 32) / 16;
                        if constexpr (KEYS) mma_ss(tmem + x * 64, (x ? x1d : x0d) + ((k / 4) * 128 * 128 + (k % 4) * 32) / 16, y, mma_shape(AB_N, false), k > 0);
                        else mma_ts(tmem + x * 64, tmem + 384 + x * 64 + k * 8, y, mma_shape(AB_N, false), k > 0);
                    }
                mma_commit(&s_full);
                return true;
            };
            ok = ok && scores(0);
            for (int s = 0; s < steps && ok; s++) {
                const int st = s % Sh::STAGES;
                if (s + 1 < steps) {
                    if (!(ok = wait_soon_warp(&s_read, s & 1))) break;
                    tmem_fence_after();
                    if (!(ok = scores(s + 1))) break;
                }
                if (!(ok = wait_soon_warp(&p_full[s & 1], (s / 2) & 1))) break;
                tmem_fence_after();
                const uint64_t yd = tile_desc(smem_u32(Ys + st * 2 * Sh::YTILE), AB_N * 128);
                const uint32_t p = tmem + 128 + (s & 1) * 64;
                if constexpr (KEYS) {
#pragma unroll
                    for (int k = 0; k < AB_N / 16; k++)
                        mma_ts(tmem + 256 + DP, p + k * 8, yd + (Sh::YTILE + k * 2048) / 16, mma_shape(DP, true), s > 0 || k > 0);
                }
#pragma unroll
                for (int k = 0; k < AB_N / 16; k++) mma_ts(tmem + 256, p + 32 + k * 8, yd + k * 2048 / 16, mma_shape(DP, true), s > 0 || k > 0);
                mma_commit(&empty[st]);
            }
            mma_commit(&done);
            if (!ok) s_fail = 1;
        }
    }
    tmem_fence_before();
    __syncthreads();
    if (s_fail != 0) {                                   // report, and give copies and products in flight time to land
        if (tid == 0) atomicExch(&g_attn_bwd_status, 1);
        for (int i = 0; i < 1000; i++) __nanosleep(1000);
    }
    if (warp == AB_WARPS) { tmem_fence_after(); tmem_free(tmem, 512); }
}

template <int DP, bool CAP, bool BIAS>
static cudaError_t bwd_tensor(const AttnArgs& a, const void* q, const void* k, const void* v, const void* o, const void* rest, const float* lse,
                              const void* dout, float* delta, void* dq, void* dk, void* dv, cudaStream_t st) {
    typedef BwdShape<DP> Sh;
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
    auto rows_q = attn_bwd_tensor_kernel<DP, false, CAP, BIAS>;
    auto rows_k = attn_bwd_tensor_kernel<DP, true, CAP, BIAS>;
    cudaError_t e = opt_in_smem(rows_q, Sh::SMEM);
    if (e == cudaSuccess) e = opt_in_smem(rows_k, Sh::SMEM);
    if (e != cudaSuccess) return e;
    const int tq = (a.Tq + 127) / 128, tk = (a.Tk + 127) / 128;
    const long long cq = (long long)tq * a.H * a.B, ck = (long long)tk * a.KV * a.B;
    if (cq > 0x7fffffffll || ck > 0x7fffffffll) return cudaErrorInvalidValue;
    rows_q<<<(unsigned)cq, Sh::THREADS, Sh::SMEM, st>>>(a, mq, (const bf16*)o, (const bf16*)rest, (const bf16*)dout, lse, delta, tq, cq < 148 * 8);
    rows_k<<<(unsigned)ck, Sh::THREADS, Sh::SMEM, st>>>(a, mk, nullptr, nullptr, nullptr, lse, delta, tk, ck < 148 * 8);
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
