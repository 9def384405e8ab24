// Attention over tokens on the tensor cores, bf16: forward.
//
// A CTA holds two tiles of 128 queries of a head, passes over their keys 128 at a time, and keeps scores and outputs in tensor
// memory (two of each fill its 512 columns).
//   copy warp    tiles of q once, then k, v, k, v, ... through a ring of stages
//   product warp s = q k^T into columns S, o += p v with p read from the same columns
//   128 threads to a query tile: a thread owns a row, so maximum and sum of its softmax need no other lane.  It reads its scores,
//                writes the weights p (bf16) over them, and hands them to the product warp
// The products of one tile run while the other tile's weights are formed.  (One tile to a CTA, two CTAs to an SM: 597 us against
// 375 for one sequence of 16,384, and no better for short ones.)  The outputs are rescaled in place, and only
// when a row's maximum has grown by more than 2^8: until then the weights are taken relative to the old one, which
// float32 sums and the relative precision of bf16 bear.
// p is rounded to bf16 for its product, as its operand type asks; the sum of the softmax takes it unrounded.
#include <type_traits>

#include "slotscan_attn.cuh"
#include "slotscan_launch.h"
#include "slotscan_tensor.cuh"

namespace slotscan {

static __device__ int g_attn_status = 0;                 // a bounded wait gave up (slotscan_device_status)

constexpr float GROWN = 8.f;                             // in powers of two
constexpr int NT = 2;                                    // tiles of 128 queries of a CTA
constexpr int KT = 128;                                  // keys of a tile

template <int DP>
struct FwdShape {
    static constexpr int STAGES = 4;                     // tiles of the ring, keys and values in turn
    static constexpr int SUBS = DP / 64;                 // 64-column sub-tiles of a tile
    static constexpr int QTILE = 128 * DP * 2, KTILE = KT * DP * 2;                // bytes
    static constexpr int THREADS = NT * 128 + 128;
    static constexpr int SMEM = NT * QTILE + STAGES * KTILE + 1024;
};
struct FwdMaps { CUtensorMap q, k, v, o, rest; };

// 32 scores of a row as base-2 exponents (CAP or BIAS: whole; else still without the factor `lin`), minus infinity where the row does
// not see them
template <bool CAP, bool BIAS>
__device__ __forceinline__ void scores32(float (&s)[32], const Score& sc, float ahead, bool masked, int lo, int hi) {
    bool small = true;                                   // the capped scores' polynomial serves this warp's block
    if constexpr (CAP) {
        float m0 = 0.f, m1 = 0.f;
#pragma unroll
        for (int i = 0; i < 32; i += 2) { m0 = fmaxf(m0, fabsf(s[i])); m1 = fmaxf(m1, fabsf(s[i + 1])); }
        small = __all_sync(FULL, fmaxf(m0, m1) * sc.cap_in <= CAP_POLY_MOST);
    }
    if constexpr (CAP || BIAS) {
        auto whole = [&](auto poly) {
            const CapPoly cp(sc);
            const f32x2 lin = pack2(sc.lin, sc.lin), steep = pack2(-sc.slope, -sc.slope);
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
                const f32x2 x = pack2(s[i], s[i + 1]);
                f32x2 z;
                if constexpr (CAP && decltype(poly)::value) z = mul2(x, cp.slope(x));
                else if constexpr (CAP) {                                                      // tanh x = 1 - 2 / (e^2x + 1)
                    const float in = 2.f * LOG2E * sc.cap_in;
                    z = pack2(fmaf(-2.f * sc.cap_out, rcp_fast(exp2_fast(s[i] * in) + 1.f), sc.cap_out),
                              fmaf(-2.f * sc.cap_out, rcp_fast(exp2_fast(s[i + 1] * in) + 1.f), sc.cap_out));
                } else z = mul2(x, lin);
                if constexpr (BIAS) z = fma2(pack2(fabsf(ahead - (float)i), fabsf(ahead - (float)(i + 1))), steep, z);
                const float2 u = unpack2(z);
                s[i] = u.x;
                s[i + 1] = u.y;
            }
        };
        if (small) whole(std::true_type{});
        else if constexpr (CAP) whole(std::false_type{});
    }
    if (masked) {
#pragma unroll
        for (int i = 0; i < 32; i++) s[i] = i >= lo && i < hi ? s[i] : -INFINITY;
    }
}

template <int DP, bool CAP, bool BIAS>
__global__ void __launch_bounds__(NT * 128 + 128, 1)
attn_fwd_tensor_kernel(AttnArgs a, RowInputs<bf16> in, const __grid_constant__ FwdMaps maps, float* lse, int tiles, int tile_major) {
    typedef FwdShape<DP> Sh;
    extern __shared__ char smem_raw[];
    char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    char* Qs = smem;
    char* Ks = smem + NT * Sh::QTILE;
    __shared__ uint64_t q_full[NT], s_full[NT], p_full[NT], o_full[NT], full[Sh::STAGES], empty[Sh::STAGES];
    __shared__ uint32_t s_tmem;
    __shared__ int s_fail;
    __shared__ TileSpan s_span[NT];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    // one dimension of CTAs: the long rows first, over all heads (tile_major), or head by head, whose keys then stay in the cache
    const int heads = a.H * a.B;
    const int tile = tiles - 1 - (int)(tile_major ? blockIdx.x / heads : blockIdx.x % tiles);
    const int hb = (int)(tile_major ? blockIdx.x % heads : blockIdx.x / tiles), h = hb % a.H, b = hb / a.H, hk = h / (a.H / a.KV);
    const int i0 = tile * NT * 128;
    if (tid == 0) {
        for (int t = 0; t < NT; t++) {
            mbar_init(&q_full[t], 1); mbar_init(&s_full[t], 1); mbar_init(&p_full[t], 4); mbar_init(&o_full[t], 1);
            tile_span_reset(&s_span[t]);
        }
        for (int s = 0; s < Sh::STAGES; s++) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        mbar_fence_init();
        s_fail = 0;
    }
    if (warp == NT * 4) tmem_alloc(&s_tmem, 512);
    __syncthreads();
    const int my_t = tid / 128, row = i0 + tid;          // of the softmax threads
    Span sp = {0, 0};
    if (warp < NT * 4) {
        if (row < a.Tq) sp = keys_of(a, b, row);
        tile_span_add(&s_span[my_t], sp, row < a.Tq);
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    constexpr uint32_t tmem = 0;                         // all 512 columns are this CTA's, so they begin at the first
    int first[NT], last[NT], n0 = BIGI, n1 = 0;          // key tiles of each query tile, and of all
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const TileSpan s = s_span[t];
        first[t] = s.hi_max > 0 ? s.lo_min / KT : 0;
        last[t] = s.hi_max > 0 ? (s.hi_max + KT - 1) / KT : 0;
        if (last[t] > first[t]) { n0 = min(n0, first[t]); n1 = max(n1, last[t]); }
    }
    // 3 x 128 threads x 168 registers at launch = 2 x 128 x 216 + 128 x 72; a row of 128 scores stays in registers
    if (warp < NT * 4) {                                 // ---- softmax of a tile ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int t = my_t;
        const int f0 = t == 0 ? first[0] : first[NT - 1], l0 = t == 0 ? last[0] : last[NT - 1];
        const WarpSpan ws(sp);
        const uint32_t lane_at = (uint32_t)((warp % 4) * 32) << 16;
        const uint32_t S = tmem + t * KT + lane_at, O = tmem + NT * KT + t * DP + lane_at;
        const Score sc(a, h);
        float m = -INFINITY, l = 0.f;                    // m in base-2 exponents
        const float at = (float)(row + a.Tk - a.Tq);
        bool ok = true;
        for (int n = f0; n < l0; n++) {
            const int j0 = n * KT;
            const bool masked = !ws.clear(j0, KT);
            if (!(ok = wait_soon_warp(&s_full[t], (n - f0) & 1))) break;
            tmem_fence_after();
            uint32_t raw[KT / 32][32];
#pragma unroll
            for (int c = 0; c < KT / 32; c++) tmem_ld(S + c * 32, raw[c]);
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < KT / 32; c++) {
                tmem_ld_wait(raw[c]);
                float(&s)[32] = reinterpret_cast<float(&)[32]>(raw[c]);
                scores32<CAP, BIAS>(s, sc, at - (float)(j0 + c * 32), masked, sp.lo - j0 - c * 32, sp.hi - j0 - c * 32);
                float t0 = s[0], t1 = s[1], t2 = s[2], t3 = s[3];
#pragma unroll
                for (int i = 4; i < 32; i += 4) { t0 = fmaxf(t0, s[i]); t1 = fmaxf(t1, s[i + 1]); t2 = fmaxf(t2, s[i + 2]); t3 = fmaxf(t3, s[i + 3]); }
                top = fmaxf(top, fmaxf(fmaxf(t0, t1), fmaxf(t2, t3)));
            }
            if constexpr (!CAP && !BIAS) top *= sc.lin;
            // a row that has seen nothing so far has only zeros to rescale
            const bool grown = top > m + GROWN && m != -INFINITY;
            if (m == -INFINITY) m = top;
            if (__any_sync(FULL, grown)) {
                const float to = fmaxf(m, top), f = to == -INFINITY ? 1.f : exp2_fast(m - to);
                if (n > f0) {
                    if (!(ok = wait_soon_warp(&o_full[t], (n - f0 - 1) & 1))) break;
                    tmem_fence_after();
#pragma unroll
                    for (int c = 0; c < DP / 32; c++) {
                        uint32_t o[32];
                        tmem_ld(O + c * 32, o);
                        tmem_ld_wait(o);
#pragma unroll
                        for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tmem_st(O + c * 32, o);
                    }
                }
                m = to;
                l *= f;
            }
            const float base = m == -INFINITY ? 0.f : m;
            f32x2 sum[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
            const f32x2 lin = pack2(sc.lin, sc.lin), back = pack2(-base, -base);
#pragma unroll
            for (int c = 0; c < KT / 32; c++) {
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const f32x2 x = pack2(__uint_as_float(raw[c][i]), __uint_as_float(raw[c][i + 1]));
                    const float2 z = unpack2(CAP || BIAS ? add2(x, back) : fma2(x, lin, back));
                    const float p0 = exp2_fast(z.x), p1 = exp2_fast(z.y);
                    sum[(i / 2) % 2] = add2(sum[(i / 2) % 2], pack2(p0, p1));
                    w[i / 2] = pack_bf16(p0, p1);
                }
                tmem_st(S + c * 16, w);
            }
            const float2 total = unpack2(add2(sum[0], sum[1]));
            l += total.x + total.y;
            tmem_st_wait();
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) arrive(&p_full[t]);
        }
        if (ok && l0 > f0) ok = wait_soon(&o_full[t], (l0 - f0 - 1) & 1);
        else if (ok && n0 < n1) ok = wait_soon(&q_full[t], 0);                     // a tile that sees nothing: its queries still come in where its outputs go
        tmem_fence_after();
        if (!ok) s_fail = 1;
        const bool none = sp.hi <= sp.lo;
        const float inv = none ? 0.f : 1.f / l;
        // the outputs through the tile of the queries, whose products are done; with lse also what their rounding left, for
        // the backward's <do, o>
        char* out = Qs + t * Sh::QTILE;
        const int r = tid % 128;
        for (int pass = 0; pass < (lse != nullptr ? 2 : 1); pass++) {
            if (pass) {
                if (r == 0) bulk_wait_read<0>();
                sync_group(1 + t, 128);
            }
            float seen = 0.f;
#pragma unroll
            for (int c = 0; c < DP / 32; c++) {
                uint32_t o[32];
                if (l0 > f0) { tmem_ld(O + c * 32, o); tmem_ld_wait(o); }
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float x = none ? 0.f : __uint_as_float(o[i + 2 * e]) * inv, y = none ? 0.f : __uint_as_float(o[i + 2 * e + 1]) * inv;
                        w[e] = pack_bf16(x, y);
                        watch(seen, x);
                        watch(seen, y);
                        if (pass) w[e] = pack_bf16(x - __uint_as_float(w[e] << 16), y - __uint_as_float(w[e] & 0xffff0000u));
                    }
                    *reinterpret_cast<uint4*>(out + (c / 2) * 128 * 128 + swizzled(r, (c % 2) * 4 + i / 8)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            for (unsigned bad = __ballot_sync(FULL, seen != seen && row < a.Tq); bad != 0; bad &= bad - 1) {
                const int x = __ffs(bad) - 1, xr = r - lane + x;
                float v[4], unused0, unused1;
                careful_query(a, in, b, h, row - lane + x, v, unused0, unused1);
#pragma unroll
                for (int c = 0; c < DP / 32; c++) {
                    const bf16 hi = __float2bfloat16_rn(v[c]);
                    const int d = lane + 32 * c;
                    *reinterpret_cast<bf16*>(out + (d / 64) * 128 * 128 + swizzled(xr, d % 64 / 8) + d % 8 * 2) = pass ? __float2bfloat16_rn(v[c] - __bfloat162float(hi)) : hi;
                }
            }
            fence_proxy_async_smem();
            sync_group(1 + t, 128);
            if (r == 0 && i0 + t * 128 < a.Tq) {
                for (int c = 0; c < Sh::SUBS; c++) tile_s2g(pass ? &maps.rest : &maps.o, c * 64, i0 + t * 128, h, b, out + c * 128 * 128);
                bulk_commit();
            }
        }
        if (lse != nullptr && row < a.Tq)
            lse[((size_t)b * a.H + h) * a.Tq + row] = none ? -INFINITY : sp.hi - sp.lo == 1 ? INFINITY : m + log2f(l);
        if (r == 0) bulk_wait_read<0>();
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == NT * 4 + 1) {                            // ---- copies ----
            if (lane == 0 && n0 < n1) {
                bool ok = true;
                for (int t = 0; t < NT; t++) {
                    mbar_arrive_expect_tx(&q_full[t], Sh::QTILE);
                    for (int c = 0; c < Sh::SUBS; c++) tile_g2s(Qs + t * Sh::QTILE + c * 128 * 128, &maps.q, c * 64, i0 + t * 128, h, b, &q_full[t]);
                }
                for (int n = n0, x = 0; n < n1 && ok; n++) {
                    for (int w = 0; w < 2; w++, x++) {       // keys, values
                        const int s = x % Sh::STAGES, turn = x / Sh::STAGES;
                        if (turn > 0 && !wait_soon(&empty[s], (turn - 1) & 1)) { ok = false; break; }
                        mbar_arrive_expect_tx(&full[s], Sh::KTILE);
                        for (int c = 0; c < Sh::SUBS; c++)
                            tile_g2s(Ks + s * Sh::KTILE + c * KT * 128, w ? &maps.v : &maps.k, c * 64, n * KT, hk, b, &full[s]);
                    }
                }
                if (!ok) s_fail = 1;
            }
        } else if (warp == NT * 4) {                         // ---- products ----
            if (n0 < n1) {
                bool ok = true;
                const bool lead = elected();
                auto stage = [](int x) { return x % Sh::STAGES; };
                auto arrived = [&](int x) { return wait_soon_warp(&full[stage(x)], (x / Sh::STAGES) & 1); };
                auto scores = [&](int t, int x) {            // s = q k^T
                    const uint32_t qd = tile_desc(smem_u32(Qs + t * Sh::QTILE), 16), kd = tile_desc(smem_u32(Ks + stage(x) * Sh::KTILE), 16);
                    if (lead) {
#pragma unroll
                        for (int k = 0; k < DP / 16; k++)
                            mma_ss(tmem + t * KT, qd + ((k / 4) * 128 * 128 + (k % 4) * 32) / 16, kd + ((k / 4) * KT * 128 + (k % 4) * 32) / 16, mma_shape(KT, false), k > 0);
                        mma_commit(&s_full[t]);
                    }
                    __syncwarp();
                };
                for (int t = 0; t < NT && ok; t++) ok = wait_soon_warp(&q_full[t], 0);
                ok = ok && arrived(0);
                for (int t = 0; t < NT && ok; t++)
                    if (first[t] == n0 && last[t] > first[t]) scores(t, 0);
                if (lead) mma_commit(&empty[0]);
                __syncwarp();
                for (int n = n0, x = 0; n < n1 && ok; n++, x += 2) {
                    ok = arrived(x + 1) && (n + 1 == n1 || arrived(x + 2));
                    const uint32_t vd = tile_desc(smem_u32(Ks + stage(x + 1) * Sh::KTILE), KT * 128);
                    for (int t = 0; t < NT && ok; t++) {
                        if (n >= first[t] && n < last[t]) {
                            ok = wait_soon_warp(&p_full[t], (n - first[t]) & 1);
                            tmem_fence_after();
                            if (lead) {
#pragma unroll
                                for (int k = 0; k < KT / 16; k++)
                                    mma_ts(tmem + NT * KT + t * DP, tmem + t * KT + k * 8, vd + k * 2048 / 16, mma_shape(DP, true), n > first[t] || k > 0);
                                mma_commit(&o_full[t]);
                            }
                            __syncwarp();
                        }
                        if (n + 1 >= first[t] && n + 1 < last[t]) scores(t, x + 2);
                    }
                    if (lead) {
                        mma_commit(&empty[stage(x + 1)]);
                        if (n + 1 < n1) mma_commit(&empty[stage(x + 2)]);
                    }
                    __syncwarp();
                }
                if (!ok) s_fail = 1;
            }
        }
    }
    tmem_fence_before();
    __syncthreads();
    if (s_fail != 0) {                                   // report, and give copies and products in flight time to land
        if (tid == 0) atomicExch(&g_attn_status, 1);
        for (int i = 0; i < 1000; i++) __nanosleep(1000);
    }
    if (warp == NT * 4) { tmem_fence_after(); tmem_free(s_tmem, 512); }
}

template <int DP, bool CAP, bool BIAS>
static cudaError_t fwd_tensor(const AttnArgs& a, const void* q, const void* k, const void* v, void* o, void* rest, float* lse, cudaStream_t st) {
    typedef FwdShape<DP> Sh;
    auto kern = attn_fwd_tensor_kernel<DP, CAP, BIAS>;
    const cudaError_t e = opt_in_smem(kern, Sh::SMEM);   // before the maps: a thread's first runtime call makes the context current for them
    if (e != cudaSuccess) return e;
    FwdMaps maps;
    const long long os[3] = {(long long)a.Tq * a.H * a.D, (long long)a.H * a.D, a.D};
    if (!tile_map(&maps.q, q, a.B, a.Tq, a.H, a.D, a.qs, 128) || !tile_map(&maps.k, k, a.B, a.Tk, a.KV, a.D, a.ks, KT) ||
        !tile_map(&maps.v, v, a.B, a.Tk, a.KV, a.D, a.vs, KT) || !tile_map(&maps.o, o, a.B, a.Tq, a.H, a.D, os, 128) ||
        !tile_map(&maps.rest, lse != nullptr ? rest : o, a.B, a.Tq, a.H, a.D, os, 128))
        return cudaErrorInvalidValue;
    const int tiles = (a.Tq + NT * 128 - 1) / (NT * 128);
    const long long ctas = (long long)tiles * a.H * a.B;
    if (ctas > 0x7fffffffll) return cudaErrorInvalidValue;
    kern<<<(unsigned)ctas, Sh::THREADS, Sh::SMEM, st>>>(a, RowInputs<bf16>{(const bf16*)q, (const bf16*)k, (const bf16*)v, nullptr}, maps, lse, tiles, ctas < 148 * 8);
    return cudaGetLastError();
}
template <int DP>
static cudaError_t fwd_tensor_score(const AttnArgs& a, const void* q, const void* k, const void* v, void* o, void* rest, float* lse, cudaStream_t st) {
    if (a.cap > 0.f) return a.slopes != nullptr ? fwd_tensor<DP, true, true>(a, q, k, v, o, rest, lse, st)
                                                : fwd_tensor<DP, true, false>(a, q, k, v, o, rest, lse, st);
    return a.slopes != nullptr ? fwd_tensor<DP, false, true>(a, q, k, v, o, rest, lse, st)
                               : fwd_tensor<DP, false, false>(a, q, k, v, o, rest, lse, st);
}

cudaError_t run_attn_fwd_bf16(const AttnArgs& a, const void* q, const void* k, const void* v, void* o, void* rest, float* lse, cudaStream_t st) {
    return a.D <= 64 ? fwd_tensor_score<64>(a, q, k, v, o, rest, lse, st) : fwd_tensor_score<128>(a, q, k, v, o, rest, lse, st);
}

int attn_mma_status() {
    int v = 0;
    const int z = 0;
    if (cudaMemcpyFromSymbol(&v, g_attn_status, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) cudaMemcpyToSymbol(g_attn_status, &z, sizeof(int));
    return v;
}

}  // namespace slotscan
