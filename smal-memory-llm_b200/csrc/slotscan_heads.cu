// Norms of queries and keys per head with the position rotation in the same pass, forward, backward and into ring caches.
//
// Per row x of D channels:  r = (mean x^2 + eps)^(-1/2),  y = x r w,  and the pairs (i, i + R/2) turned by the position's angle.
// Backward, with g the upstream gradient turned back by the same angle:  dw += g x r,  h = g w,
//     dx = r (h - x r mean(h x r))
// A row's two sums are its only reductions, so each element is read once and written once: two rows of traffic forward, three
// backward, and some ten operations an element.  Bandwidth bounds it.
//
// Layout: a group of LPG lanes (a power of two, 8 channels to a lane: one 16-byte load of bf16, two of float32) takes a token and walks
// over a slice of its heads, queries first, with the token's cosines and sines in registers: the table of a position has the bytes of
// two bf16 rows, and is read once for all its heads.  A pair's two channels lie R/16 lanes apart: one shuffle.  What hides a row's
// chain of load, two sums and store is the other warps: two rows in flight to a group and four CTAs to an SM took 101 us for
// 64 x 1,024 tokens of 6 + 6 heads of 128 (4.0 TB/s), six rows and three CTAs 113; the backward, with more to keep, 150 us (4.0 TB/s)
// with four rows and two CTAs, 164 with three, 186 with two, 256 with two rows and three CTAs.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "slotscan.h"
#include "slotscan_common.cuh"
#include "slotscan_launch.h"

namespace slotscan {

typedef __nv_bfloat16 bf16;
constexpr int NR_THREADS = 256;
constexpr int NR_FWD_CTAS = 4, NR_BWD_CTAS = 2;         // of an SM
constexpr int NR_MAX_CTAS = 148 * NR_BWD_CTAS;                     // of the backward, which sums the weights' gradients per CTA: those of one wave

struct NormArgs {
    int T, H, KV, D, R, table_len, slices, per_slice;    // per_slice heads (queries, keys, then values) to a group
    long long tokens;
    float eps;
    long long qs[3], ks[3];
    const float* table;
    const int32_t* pos;
    const float *qw, *kw;
};
struct AppendArgs {                                      // L 0: no caches
    int L;
    long long vs[3], kcs[3], vcs[3];
};

// 8 channels as they lie in memory: what a row in flight costs a thread in registers
template <typename T>
struct Raw8 { uint4 v[sizeof(T) / 2]; };
template <typename T>
__device__ __forceinline__ Raw8<T> raw8(const T* p, bool in) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) r.v[i] = in ? reinterpret_cast<const uint4*>(p)[i] : make_uint4(0u, 0u, 0u, 0u);
    return r;
}
template <typename T>
__device__ __forceinline__ void widen(float (&x)[8], const Raw8<T>& r) { ld8(x, reinterpret_cast<const T*>(&r)); }

// cosines and sines of this lane's 8 channels; NaN where the position lies outside the table
__device__ __forceinline__ void load_turn(const NormArgs& a, long long at, int half, int c, float (&cs)[8], float (&sn)[8]) {
    const bool in = at >= 0 && at < a.table_len;
    const float* t = a.table + ((size_t)(in ? at : 0) * (a.R / 2) + (c % half) * 8) * 2;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float4 u = ld4(t + 4 * i);
        cs[2 * i] = u.x; sn[2 * i] = u.y; cs[2 * i + 1] = u.z; sn[2 * i + 1] = u.w;
    }
    if (!in) {
#pragma unroll
        for (int i = 0; i < 8; i++) cs[i] = sn[i] = __int_as_float(0x7fffffff);
    }
}

// y turned by the angle (DIR 1) or back (DIR -1); lanes c < half hold the first of each pair, [half, 2 half) the second
template <int DIR>
__device__ __forceinline__ void turn(float (&y)[8], const float (&cs)[8], const float (&sn)[8], int half, int c, int LPG) {
    const int lane = threadIdx.x & 31;
    const bool first = c < half, rot = c < 2 * half;
    const int partner = rot ? (lane & ~(LPG - 1)) + (first ? c + half : c - half) : lane;
    const bool minus = first == (DIR > 0);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float o = __shfl_sync(FULL, y[i], partner);
        if (rot) y[i] = fmaf(y[i], cs[i], minus ? -o * sn[i] : o * sn[i]);
    }
}

// T: bf16 or float.  CACHE: the keys and the values go into the caches.
template <typename T, int LPG, bool CACHE>
__global__ void __launch_bounds__(NR_THREADS, CACHE ? 3 : NR_FWD_CTAS) norm_rope_kernel(NormArgs a, AppendArgs ap, const T* q, const T* k, const T* v, T* qo, T* ko,
                                                               T* kc, T* vc) {
    const int c = threadIdx.x % LPG;
    const unsigned unit = blockIdx.x * (NR_THREADS / LPG) + threadIdx.x / LPG, tok = unit / a.slices;            // fewer than 2^31
    const int h0 = (int)(unit % a.slices) * a.per_slice, all = a.H + a.KV + (CACHE ? a.KV : 0);
    const bool live = tok < a.tokens && c * 8 < a.D;
    const unsigned b = live ? tok / a.T : 0, t = live ? tok % a.T : 0;
    const long long at = CACHE ? (long long)a.pos[b] + t : a.pos != nullptr ? (long long)a.pos[live ? tok : 0] : t;
    const T* qt = q + b * a.qs[0] + t * a.qs[1] + c * 8;                           // of the token
    const T* kt = k + b * a.ks[0] + t * a.ks[1] + c * 8;
    const T* vt = CACHE ? v + b * ap.vs[0] + t * ap.vs[1] + c * 8 : nullptr;
    T* qot = qo + (size_t)tok * a.H * a.D + c * 8;
    const int half = a.R / 16;
    float cs[8], sn[8], w[8];
    if (half) load_turn(a, at, half, c, cs, sn);
    const long long row = CACHE && at >= 0 ? (unsigned)at % (unsigned)ap.L : 0;
    T* kot = CACHE ? kc + b * ap.kcs[0] + row * ap.kcs[1] + c * 8 : ko + (size_t)tok * a.KV * a.D + c * 8;
    T* vot = CACHE ? vc + b * ap.vcs[0] + row * ap.vcs[1] + c * 8 : nullptr;
    const long long kos = CACHE ? ap.kcs[2] : a.D;
    const float inv_d = 1.f / a.D;
    constexpr int U = 2;                                 // rows in flight to a group
    for (int u0 = 0; u0 < a.per_slice; u0 += U) {
        Raw8<T> in[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int h = h0 + u0 + u;
            const T* from = h < a.H ? qt + h * a.qs[2] : !CACHE || h < a.H + a.KV ? kt + (h - a.H) * a.ks[2] : vt + (h - a.H - a.KV) * ap.vs[2];
            in[u] = raw8(from, live && u0 + u < a.per_slice && h < all);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int h = h0 + u0 + u;
            if (u0 + u >= a.per_slice) break;            // the same in every lane of the CTA
            const bool is_v = CACHE && h >= a.H + a.KV, is_q = h < a.H;
            if (h == a.H || u0 + u == 0) {               // the queries' weights, then the keys'
                const float* from = is_q ? a.qw : a.kw;
#pragma unroll
                for (int i = 0; i < 8; i++) w[i] = 1.f;
                if (live && from != nullptr) ld8(w, from + c * 8);
            }
            float ss = 0.f, x[8], y[8];
            widen(x, in[u]);
#pragma unroll
            for (int i = 0; i < 8; i++) ss = fmaf(x[i], x[i], ss);
            const float r = rsqrtf(fmaf(group_sum<LPG>(ss), inv_d, a.eps));
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = x[i] * r * w[i];
            if (half) turn<1>(y, cs, sn, half, c, LPG);
            if (!live || h >= all) continue;
            if (is_q) st8(qot + h * a.D, y);
            else if (!CACHE || at >= 0) {
                if (!is_v) st8(kot + (h - a.H) * kos, y);
                else st8(vot + (h - a.H - a.KV) * ap.vcs[2], x);
            }
        }
    }
}

// grid-stride over (token, slice of heads); part: (CTAs, 2, D) sums of the weights' gradients, or NULL
template <typename T, int LPG>
__global__ void __launch_bounds__(NR_THREADS, NR_BWD_CTAS) norm_rope_bwd_kernel(NormArgs a, const T* q, const T* k, const T* gq, const T* gk, T* dq, T* dk,
                                                                   float* part) {
    constexpr int GROUPS = NR_THREADS / LPG;
    __shared__ float s_part[GROUPS][LPG * 8];
    const int c = threadIdx.x % LPG, grp = threadIdx.x / LPG;
    const int half = a.R / 16;
    const float inv_d = 1.f / a.D;
    float w[8], acc[2][8];
#pragma unroll
    for (int i = 0; i < 8; i++) acc[0][i] = acc[1][i] = 0.f;
    const unsigned units = (unsigned)a.tokens * a.slices;                          // fewer than 2^31
    for (unsigned u0 = blockIdx.x * GROUPS; u0 < units; u0 += gridDim.x * GROUPS) {
        const unsigned unit = u0 + grp, tok = unit / a.slices;
        const int h0 = (int)(unit % a.slices) * a.per_slice;
        const bool live = unit < units && c * 8 < a.D;
        const unsigned b = live ? tok / a.T : 0, t = live ? tok % a.T : 0;
        const T* qt = q + b * a.qs[0] + t * a.qs[1] + c * 8;                       // of the token
        const T* kt = k + b * a.ks[0] + t * a.ks[1] + c * 8;
        const size_t qo = (size_t)tok * a.H * a.D + c * 8, ko = (size_t)tok * a.KV * a.D + c * 8;
        float cs[8], sn[8];
        if (half) load_turn(a, a.pos != nullptr ? (long long)a.pos[live ? tok : 0] : t, half, c, cs, sn);
        constexpr int U = sizeof(T) == 2 ? 4 : 2;
        for (int v0 = 0; v0 < a.per_slice; v0 += U) {
            Raw8<T> in[U], up[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int h = h0 + v0 + u;
                const bool ok = live && v0 + u < a.per_slice && h < a.H + a.KV;
                in[u] = raw8(h < a.H ? qt + h * a.qs[2] : kt + (h - a.H) * a.ks[2], ok);
                up[u] = raw8(h < a.H ? gq + qo + h * a.D : gk + ko + (h - a.H) * a.D, ok);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int h = h0 + v0 + u;
                if (v0 + u >= a.per_slice) break;        // the same in every lane of the CTA
                const bool is_q = h < a.H;
                if (h == a.H || v0 + u == 0) {           // the queries' weights, then the keys'
                    const float* from = is_q ? a.qw : a.kw;
#pragma unroll
                    for (int i = 0; i < 8; i++) w[i] = 1.f;
                    if (c * 8 < a.D && from != nullptr) ld8(w, from + c * 8);
                }
                float x[8], g[8], s1 = 0.f, s2 = 0.f;
                widen(x, in[u]);
                widen(g, up[u]);
                if (half) turn<-1>(g, cs, sn, half, c, LPG);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    s1 = fmaf(x[i], x[i], s1);
                    s2 = fmaf(g[i] * w[i], x[i], s2);
                }
                const float r = rsqrtf(fmaf(group_sum<LPG>(s1), inv_d, a.eps));
                const float m = group_sum<LPG>(s2) * r * r * inv_d;
                if (!live || h >= a.H + a.KV) continue;
                float dx[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    dx[i] = r * fmaf(-x[i], m, g[i] * w[i]);
                    const float gx = g[i] * x[i] * r;
                    if (is_q) acc[0][i] += gx; else acc[1][i] += gx;
                }
                if (is_q) st8(dq + qo + h * a.D, dx);
                else st8(dk + ko + (h - a.H) * a.D, dx);
            }
        }
    }
    if (part == nullptr) return;
    for (int n = 0; n < 2; n++) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; i++) s_part[grp][c * 8 + i] = n ? acc[1][i] : acc[0][i];
        __syncthreads();
        for (int d = threadIdx.x; d < a.D; d += NR_THREADS) {
            float s = 0.f;
            for (int gI = 0; gI < GROUPS; gI++) s += s_part[gI][d];
            part[((size_t)blockIdx.x * 2 + n) * a.D + d] = s;
        }
    }
}

// dw[d] = sum over the CTAs, in their order; a warp to a channel
__global__ void norm_rope_weights_kernel(const float* part, int ctas, int D, float* dqw, float* dkw) {
    const int d = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32, lane = threadIdx.x & 31;
    if (d >= 2 * D) return;
    float s = 0.f;
    for (int i = lane; i < ctas; i += 32) s += part[(size_t)i * 2 * D + d];
    s = warp_sum(s);
    if (lane == 0) (d < D ? dqw : dkw)[d < D ? d : d - D] = s;
}

static int lanes_of(int D) { return D <= 64 ? 8 : D <= 128 ? 16 : 32; }
static NormArgs norm_args(const slotscan_norm_params& p, const float* table, const int32_t* pos, const float* qw, const float* kw, int heads) {
    NormArgs a;
    a.T = p.T; a.H = p.H; a.KV = p.KV; a.D = p.D; a.R = p.R; a.table_len = p.table_len;
    a.tokens = (long long)p.B * p.T;
    a.eps = p.eps;
    for (int i = 0; i < 3; i++) { a.qs[i] = p.q_stride[i]; a.ks[i] = p.k_stride[i]; }
    a.table = table; a.pos = pos; a.qw = qw; a.kw = kw;
    // fewer heads to a group while the groups would leave SMs idle (three CTAs each, two rounds); whole tokens beyond, whose table is
    // then read once
    const long long groups = 148ll * 6 * NR_THREADS / lanes_of(p.D), want = (a.tokens * heads + groups - 1) / groups;
    a.per_slice = (int)(want < 1 ? 1 : want > heads ? heads : want);
    a.slices = (heads + a.per_slice - 1) / a.per_slice;
    return a;
}
static int bwd_ctas(const NormArgs& a) {
    const long long want = (a.tokens * a.slices + NR_THREADS / lanes_of(a.D) - 1) / (NR_THREADS / lanes_of(a.D));
    return (int)(want < NR_MAX_CTAS ? want : NR_MAX_CTAS);
}

template <typename T, bool CACHE>
static cudaError_t launch_norm(const NormArgs& a, const AppendArgs& ap, const void* q, const void* k, const void* v, void* qo, void* ko, void* kc,
                               void* vc, cudaStream_t st) {
    const int groups = NR_THREADS / lanes_of(a.D);
    const unsigned grid = (unsigned)((a.tokens * a.slices + groups - 1) / groups);
    auto go = [&](auto kern) { kern<<<grid, NR_THREADS, 0, st>>>(a, ap, (const T*)q, (const T*)k, (const T*)v, (T*)qo, (T*)ko, (T*)kc, (T*)vc); };
    if (lanes_of(a.D) == 8) go(norm_rope_kernel<T, 8, CACHE>);
    else if (lanes_of(a.D) == 16) go(norm_rope_kernel<T, 16, CACHE>);
    else go(norm_rope_kernel<T, 32, CACHE>);
    return cudaGetLastError();
}
template <typename T>
static cudaError_t launch_norm_bwd(const NormArgs& a, const void* q, const void* k, const void* gq, const void* gk, void* dq, void* dk, float* dqw,
                                   float* dkw, float* part, cudaStream_t st) {
    const int grid = bwd_ctas(a);
    auto go = [&](auto kern) {
        kern<<<grid, NR_THREADS, 0, st>>>(a, (const T*)q, (const T*)k, (const T*)gq, (const T*)gk, (T*)dq, (T*)dk, part);
    };
    if (lanes_of(a.D) == 8) go(norm_rope_bwd_kernel<T, 8>);
    else if (lanes_of(a.D) == 16) go(norm_rope_bwd_kernel<T, 16>);
    else go(norm_rope_bwd_kernel<T, 32>);
    if (part != nullptr) norm_rope_weights_kernel<<<(2 * a.D + 7) / 8, 256, 0, st>>>(part, grid, a.D, dqw, dkw);
    return cudaGetLastError();
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
static bool strides16(const int64_t* s, int n, int dtype) {
    for (int i = 0; i < n; i++)
        if (s[i] * (dtype == SLOTSCAN_BF16 ? 2 : 4) % 16) return false;
    return true;
}

}  // namespace slotscan

using namespace slotscan;

extern "C" int slotscan_norm_rope_check(const slotscan_norm_params* p) {
    if (p == nullptr) return SLOTSCAN_E_NULL;
    if (p->dtype != SLOTSCAN_F32 && p->dtype != SLOTSCAN_BF16) return SLOTSCAN_E_DTYPE;
    if (p->B < 0 || p->T < 0 || p->H < 1 || p->KV < 1 || p->D < 8 || p->D > 256 || p->D % 8 || p->R < 0 || p->R > p->D || p->R % 16 ||
        (p->R && p->table_len < 1))
        return SLOTSCAN_E_SHAPE;
    if ((int64_t)p->B * p->T >= (1ll << 31) || (int64_t)p->B * p->T * ((int64_t)p->H + 2ll * p->KV) > (1ll << 33)) return SLOTSCAN_E_SHAPE;
    if (!strides16(p->q_stride, 3, p->dtype) || !strides16(p->k_stride, 3, p->dtype)) return SLOTSCAN_E_ALIGN;
    return SLOTSCAN_OK;
}

extern "C" int slotscan_norm_rope_fwd(const slotscan_norm_params* p, const void* q, const void* k, const float* table, const int32_t* pos,
                                      const float* qw, const float* kw, void* qo, void* ko, void* stream) {
    const int rc = slotscan_norm_rope_check(p);
    if (rc != SLOTSCAN_OK) return rc;
    if ((int64_t)p->B * p->T == 0) return SLOTSCAN_OK;
    if (!q || !k || !qo || !ko || (p->R && !table)) return SLOTSCAN_E_NULL;
    if (!aligned16(q) || !aligned16(k) || !aligned16(qo) || !aligned16(ko) || !aligned16(table) || !aligned16(qw) || !aligned16(kw)) return SLOTSCAN_E_ALIGN;
    const NormArgs a = norm_args(*p, table, pos, qw, kw, p->H + p->KV);
    const AppendArgs none = {};
    return (int)(p->dtype == SLOTSCAN_BF16 ? launch_norm<bf16, false>(a, none, q, k, nullptr, qo, ko, nullptr, nullptr, (cudaStream_t)stream)
                                           : launch_norm<float, false>(a, none, q, k, nullptr, qo, ko, nullptr, nullptr, (cudaStream_t)stream));
}

extern "C" size_t slotscan_norm_rope_bwd_scratch_bytes(const slotscan_norm_params* p) {
    if (slotscan_norm_rope_check(p) != SLOTSCAN_OK) return 0;
    return sizeof(float) * (size_t)bwd_ctas(norm_args(*p, nullptr, nullptr, nullptr, nullptr, p->H + p->KV)) * 2 * p->D;
}

extern "C" int slotscan_norm_rope_bwd(const slotscan_norm_params* p, const void* q, const void* k, const float* table, const int32_t* pos,
                                      const float* qw, const float* kw, const void* dqo, const void* dko, void* dq, void* dk, float* dqw, float* dkw,
                                      void* scratch, size_t scratch_bytes, void* stream) {
    const int rc = slotscan_norm_rope_check(p);
    if (rc != SLOTSCAN_OK) return rc;
    if ((dqw == nullptr) != (dkw == nullptr)) return SLOTSCAN_E_NULL;
    cudaStream_t st = (cudaStream_t)stream;
    if ((int64_t)p->B * p->T == 0) {
        cudaError_t e = cudaSuccess;
        if (dqw != nullptr) {
            e = cudaMemsetAsync(dqw, 0, sizeof(float) * p->D, st);
            if (e == cudaSuccess) e = cudaMemsetAsync(dkw, 0, sizeof(float) * p->D, st);
        }
        return (int)e;
    }
    if (!q || !k || !dqo || !dko || !dq || !dk || (p->R && !table)) return SLOTSCAN_E_NULL;
    if (dqw != nullptr && (scratch == nullptr || scratch_bytes < slotscan_norm_rope_bwd_scratch_bytes(p))) return SLOTSCAN_E_NULL;
    if (!aligned16(q) || !aligned16(k) || !aligned16(dqo) || !aligned16(dko) || !aligned16(dq) || !aligned16(dk) || !aligned16(table) ||
        !aligned16(qw) || !aligned16(kw))
        return SLOTSCAN_E_ALIGN;
    const NormArgs a = norm_args(*p, table, pos, qw, kw, p->H + p->KV);
    float* part = dqw != nullptr ? (float*)scratch : nullptr;
    return (int)(p->dtype == SLOTSCAN_BF16 ? launch_norm_bwd<bf16>(a, q, k, dqo, dko, dq, dk, dqw, dkw, part, st)
                                           : launch_norm_bwd<float>(a, q, k, dqo, dko, dq, dk, dqw, dkw, part, st));
}

extern "C" int slotscan_norm_rope_append(const slotscan_append_params* p, const void* q, const void* k, const void* v, const float* table,
                                         const int32_t* pos, const float* qw, const float* kw, void* qo, void* kc, void* vc, void* stream) {
    const int rc = slotscan_norm_rope_check(p == nullptr ? nullptr : &p->base);
    if (rc != SLOTSCAN_OK) return rc;
    const slotscan_norm_params& n = p->base;
    if (p->L < 1 || n.T > p->L) return SLOTSCAN_E_SHAPE;
    if (!strides16(p->v_stride, 3, n.dtype) || !strides16(p->kc_stride, 3, n.dtype) || !strides16(p->vc_stride, 3, n.dtype)) return SLOTSCAN_E_ALIGN;
    if ((int64_t)n.B * n.T == 0) return SLOTSCAN_OK;
    if (!q || !k || !v || !pos || !qo || !kc || !vc || (n.R && !table)) return SLOTSCAN_E_NULL;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(qo) || !aligned16(kc) || !aligned16(vc) || !aligned16(table) || !aligned16(qw) ||
        !aligned16(kw))
        return SLOTSCAN_E_ALIGN;
    const NormArgs a = norm_args(n, table, pos, qw, kw, n.H + 2 * n.KV);
    AppendArgs ap;
    ap.L = p->L;
    for (int i = 0; i < 3; i++) { ap.vs[i] = p->v_stride[i]; ap.kcs[i] = p->kc_stride[i]; ap.vcs[i] = p->vc_stride[i]; }
    return (int)(n.dtype == SLOTSCAN_BF16 ? launch_norm<bf16, true>(a, ap, q, k, v, qo, nullptr, kc, vc, (cudaStream_t)stream)
                                          : launch_norm<float, true>(a, ap, q, k, v, qo, nullptr, kc, vc, (cudaStream_t)stream));
}
