// Attention over tokens: what its kernels share.
//
// A query at position i sees, of the keys, one interval [lo, hi): its document's bounds, the window and the causal rule (or the prefix)
// are intervals each.  Read from a key's side, the queries that see it are one interval too.  So a tile of rows visits the tiles of
// the other side between the least lo and the greatest hi of its rows, and masks the ones that some row does not see whole.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "slotscan.h"
#include "slotscan_common.cuh"

namespace slotscan {

typedef __nv_bfloat16 bf16;
constexpr float LOG2E = 1.44269504088896f;

struct AttnArgs {
    int B, Tq, Tk, H, KV, D;
    int window;                                          // 1 .. Tk: |i - j| < window
    float scale, cap;                                    // cap 0: none
    long long qs[3], ks[3], vs[3];                       // elements from sequence to sequence, token to token, head to head
    const float* slopes;                                 // per query head, or NULL
    const int2* docs;                                    // (B, Tk) bounds, or NULL
    const int32_t* prefix;                               // (B), or NULL
};

struct Span { int lo, hi; };                             // empty where hi <= lo

// keys that query row i (of Tq) sees
__device__ __forceinline__ Span keys_of(const AttnArgs& a, int b, int i) {
    const int at = i + a.Tk - a.Tq;
    const int2 d = a.docs != nullptr ? a.docs[(size_t)b * a.Tk + at] : make_int2(0, a.Tk);
    const int reach = a.prefix != nullptr ? max(at + 1, a.prefix[b]) : at + 1;
    return {max(max(d.x, 0), at - a.window + 1), min(min(d.y, a.Tk), min(reach, at + a.window))};
}
// query rows that see key j
__device__ __forceinline__ Span queries_of(const AttnArgs& a, int b, int j) {
    const int off = a.Tk - a.Tq;
    const int2 d = a.docs != nullptr ? a.docs[(size_t)b * a.Tk + j] : make_int2(0, a.Tk);
    const int from = a.prefix != nullptr && j < a.prefix[b] ? 0 : j;
    return {max(max(max(d.x, from), j - a.window + 1) - off, 0), min(min(d.y, a.Tk), j + a.window) - off};
}

// spans of the 128 rows of a tile
struct TileSpan { int lo_min, lo_max, hi_min, hi_max; };
__device__ __forceinline__ void tile_span_reset(TileSpan* s) { *s = {BIGI, 0, BIGI, 0}; }
// by all 32 lanes; rows that do not exist do not count, and empty rows keep every tile masked
__device__ __forceinline__ void tile_span_add(TileSpan* s, Span r, bool counts) {
    const bool some = counts && r.hi > r.lo, none = counts && r.hi <= r.lo;
    const int a = __reduce_min_sync(FULL, some ? r.lo : BIGI), b = __reduce_max_sync(FULL, none ? BIGI : some ? r.lo : 0);
    const int c = __reduce_min_sync(FULL, none ? 0 : some ? r.hi : BIGI), d = __reduce_max_sync(FULL, some ? r.hi : 0);
    if ((threadIdx.x & 31) == 0) {
        atomicMin(&s->lo_min, a); atomicMax(&s->lo_max, b); atomicMin(&s->hi_min, c); atomicMax(&s->hi_max, d);
    }
}

// spans of the 32 rows of a warp: which of its blocks of 32 columns are hidden from all of them, and which are seen whole by all
struct WarpSpan {
    int lo_min, lo_max, hi_min, hi_max;
    __device__ __forceinline__ explicit WarpSpan(Span r) {
        const bool some = r.hi > r.lo;
        lo_min = __reduce_min_sync(FULL, some ? r.lo : BIGI);
        lo_max = __reduce_max_sync(FULL, some ? r.lo : BIGI);
        hi_min = __reduce_min_sync(FULL, some ? r.hi : 0);
        hi_max = __reduce_max_sync(FULL, some ? r.hi : 0);
    }
    __device__ __forceinline__ bool dead(int j) const { return j + 32 <= lo_min || j >= hi_max; }
    __device__ __forceinline__ bool clear(int j, int n = 32) const { return j >= lo_max && j + n <= hi_min; }
};

// a score as the base-2 exponent of its weight, before the softmax's shift.  Of the cap, t = tanh(scale <q, k> / cap), whose
// derivative is 1 - t^2.
struct Score {
    float lin, cap_in, cap_out, slope;                   // slope in base 2
    __device__ __forceinline__ Score(const AttnArgs& a, int h) {
        lin = a.scale * LOG2E;
        cap_in = a.cap > 0.f ? a.scale / a.cap : 0.f;
        cap_out = a.cap * LOG2E;
        slope = a.slopes != nullptr ? a.slopes[h] * LOG2E : 0.f;
    }
};

// base-2 exponent of a score, and 1 - tanh^2 of it
__device__ __forceinline__ float score2(const Score& sc, float s, int dist, float& slope_of_cap) {
    if (sc.cap_in != 0.f) {
        const float t = tanhf(s * sc.cap_in);
        slope_of_cap = 1.f - t * t;
        return fmaf(-sc.slope, (float)dist, sc.cap_out * t);
    }
    slope_of_cap = 1.f;
    return fmaf(-sc.slope, (float)dist, s * sc.lin);
}

// ---- A row at a time, by a warp, over the visible pairs alone ----
// The tiles' products take hidden keys with weight zero, and zero times infinity or NaN is NaN.  Where a row's result is not finite, it is
// done anew here: what a row does not see then cannot reach it, and what it sees does.  Costs nothing where all is finite, and
// much where it is not: one NaN in the padding of 8,192 tokens takes a forward of six heads from 0.18 to 135 ms.
// A lane holds channels lane + 32 c.
template <typename T>
struct RowInputs { const T *q, *k, *v, *dout; };         // dout (B,Tq,H,D) contiguous

template <typename T>
__device__ __forceinline__ void lane_row(float (&x)[4], const T* row, int D) {
#pragma unroll
    for (int c = 0; c < 4; c++) { const int d = (threadIdx.x & 31) + 32 * c; x[c] = d < D ? ld1(row + d) : 0.f; }
}
__device__ __forceinline__ float lane_dot(const float (&x)[4], const float (&y)[4]) {
    return warp_sum(fmaf(x[0], y[0], fmaf(x[1], y[1], fmaf(x[2], y[2], x[3] * y[3]))));
}
template <typename T>
__device__ __forceinline__ const T* query_row(const AttnArgs& a, const RowInputs<T>& in, int b, int h, int i) { return in.q + b * a.qs[0] + i * a.qs[1] + h * a.qs[2]; }
template <typename T>
__device__ __forceinline__ const T* key_row(const AttnArgs& a, const T* k, const long long (&s)[3], int b, int hk, int j) { return k + b * s[0] + j * s[1] + hk * s[2]; }
template <typename T>
__device__ __forceinline__ const T* dout_row(const AttnArgs& a, const RowInputs<T>& in, int b, int h, int i) {
    return in.dout + (((size_t)b * a.Tq + i) * a.H + h) * a.D;
}

// o of a query, and the base-2 logarithm of its sum; with `dout` also delta = sum p <do, v>
template <typename T>
__device__ __forceinline__ void careful_query(const AttnArgs& a, const RowInputs<T>& in, int b, int h, int i, float (&o)[4], float& lse, float& delta) {
    const Span sp = keys_of(a, b, i);
    const Score sc(a, h);
    const int hk = h / (a.H / a.KV), at = i + a.Tk - a.Tq;
    float q[4], g[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f, d = 0.f, unused;
    lane_row(q, query_row(a, in, b, h, i), a.D);
    if (in.dout != nullptr) lane_row(g, dout_row(a, in, b, h, i), a.D);
#pragma unroll
    for (int c = 0; c < 4; c++) o[c] = 0.f;
    for (int j = sp.lo; j < sp.hi; j++) {
        float x[4];
        lane_row(x, key_row(a, in.k, a.ks, b, hk, j), a.D);
        const float z = score2(sc, lane_dot(q, x), abs(at - j), unused);
        const float top = fmaxf(m, z), base = top == -INFINITY ? 0.f : top, f = exp2f(m - base), p = exp2f(z - base);
        lane_row(x, key_row(a, in.v, a.vs, b, hk, j), a.D);
        l = fmaf(l, f, p);
        d = d * f + (in.dout != nullptr && p != 0.f ? p * lane_dot(g, x) : 0.f);
        bool gone = true;                                // NaN stays NaN
#pragma unroll
        for (int c = 0; c < 4; c++) {
            o[c] = p != 0.f ? fmaf(p, x[c], o[c] * f) : o[c] * f;
            gone = gone && (isnan(o[c]) || (threadIdx.x & 31) + 32 * c >= a.D);
        }
        m = top;
        if (__all_sync(FULL, gone)) break;
    }
    const float inv = sp.hi > sp.lo ? 1.f / l : 0.f;
#pragma unroll
    for (int c = 0; c < 4; c++) o[c] = sp.hi > sp.lo ? o[c] * inv : 0.f;
    lse = sp.hi - sp.lo == 1 ? INFINITY : m + log2f(l);
    delta = d * inv;
}
// weight and scaled gradient of the score of a visible pair
__device__ __forceinline__ void careful_pair(const AttnArgs& a, const Score& sc, float s, float dp, int dist, float lse, float delta, float& p, float& ds) {
    float f;
    const float z = score2(sc, s, dist, f);
    const bool alone = lse == INFINITY;
    p = alone ? 1.f : exp2f(z - lse);
    ds = alone ? 0.f : p * (dp - delta) * f * a.scale;
}
// dq of a query.  lse, delta: of all queries (B,H,Tq), or NULL: formed anew
template <typename T>
__device__ __forceinline__ void careful_dq(const AttnArgs& a, const RowInputs<T>& in, const float* lse, const float* delta, int b, int h, int i, float (&dq)[4]) {
    const Span sp = keys_of(a, b, i);
    const Score sc(a, h);
    const int hk = h / (a.H / a.KV), at = i + a.Tk - a.Tq;
    const size_t row = ((size_t)b * a.H + h) * a.Tq + i;
    float q[4], g[4], o[4], L = 0.f, dl = 0.f;
    if (lse != nullptr) { L = lse[row]; dl = delta[row]; }
    else careful_query(a, in, b, h, i, o, L, dl);
    lane_row(q, query_row(a, in, b, h, i), a.D);
    lane_row(g, dout_row(a, in, b, h, i), a.D);
#pragma unroll
    for (int c = 0; c < 4; c++) dq[c] = 0.f;
    for (int j = sp.lo; j < sp.hi; j++) {
        float k[4], v[4], p, ds;
        lane_row(k, key_row(a, in.k, a.ks, b, hk, j), a.D);
        lane_row(v, key_row(a, in.v, a.vs, b, hk, j), a.D);
        careful_pair(a, sc, lane_dot(q, k), lane_dot(g, v), abs(at - j), L, dl, p, ds);
        bool gone = true;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            if (ds != 0.f) dq[c] = fmaf(ds, k[c], dq[c]);
            gone = gone && (isnan(dq[c]) || (threadIdx.x & 31) + 32 * c >= a.D);
        }
        if (__all_sync(FULL, gone)) break;
    }
}
// dk and dv of a key, over the queries of all heads that share it
template <typename T>
__device__ __forceinline__ void careful_dkv(const AttnArgs& a, const RowInputs<T>& in, const float* lse, const float* delta, int b, int hk, int j, float (&dk)[4],
                                         float (&dv)[4]) {
    const Span sp = queries_of(a, b, j);
    const int group = a.H / a.KV;
    float k[4], v[4];
    lane_row(k, key_row(a, in.k, a.ks, b, hk, j), a.D);
    lane_row(v, key_row(a, in.v, a.vs, b, hk, j), a.D);
#pragma unroll
    for (int c = 0; c < 4; c++) dk[c] = dv[c] = 0.f;
    for (int g = 0; g < group; g++) {
        const int h = hk * group + g;
        const Score sc(a, h);
        for (int i = sp.lo; i < sp.hi; i++) {
            const size_t row = ((size_t)b * a.H + h) * a.Tq + i;
            float q[4], x[4], o[4], L = 0.f, dl = 0.f, p, ds;
            if (lse != nullptr) { L = lse[row]; dl = delta[row]; }
            else careful_query(a, in, b, h, i, o, L, dl);
            lane_row(q, query_row(a, in, b, h, i), a.D);
            lane_row(x, dout_row(a, in, b, h, i), a.D);
            careful_pair(a, sc, lane_dot(q, k), lane_dot(x, v), abs(i + a.Tk - a.Tq - j), L, dl, p, ds);
            bool gone = true;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                if (ds != 0.f) dk[c] = fmaf(ds, q[c], dk[c]);
                if (p != 0.f) dv[c] = fmaf(p, x[c], dv[c]);
                gone = gone && ((isnan(dk[c]) && isnan(dv[c])) || (threadIdx.x & 31) + 32 * c >= a.D);
            }
            if (__all_sync(FULL, gone)) return;
        }
    }
}
// 0 while all values added are finite, NaN from the first that is not
__device__ __forceinline__ void watch(float& w, float x) { w = fmaf(x, 0.f, w); }

// The capped score as a polynomial, for |x| <= 0.6 (x = scale <q, k> / cap): tanh x = x sum_k a_k x^2k, the a_k fitted here for the
// least greatest error of tanh (iteratively reweighted least squares on Chebyshev nodes): 6e-7.  Two and a half instructions a score,
// two scores to an instruction, where the exponential form takes two of the special function unit's, eight cycles a warp each; a
// block of a warp with a larger score takes that form.  (Six terms for |x| <= 1 and its two registers a term: 626 + 1,575 us for one capped
// sequence of 16,384, forward + backward; 538 + 1,470 so.)  The coefficients carry cap and scale: base-2 exponent = s sum_k c_k s^2k.
constexpr float CAP_POLY_MOST = 0.6f;
struct CapPoly {
    f32x2 c[4];
    __device__ __forceinline__ explicit CapPoly(const Score& sc) {
        const float a[4] = {0.9999910176913201f, -0.33298974340939966f, 0.12974554465812582f, -0.03961128075861646f};
        float f = sc.cap_out * sc.cap_in;
#pragma unroll
        for (int k = 0; k < 4; k++) { c[k] = pack2(a[k] * f, a[k] * f); f *= sc.cap_in * sc.cap_in; }
    }
    // two scores without their last factor: exponents = s * slope(s)
    __device__ __forceinline__ f32x2 slope(f32x2 s) const {
        const f32x2 w = mul2(s, s);
        return fma2(w, fma2(w, fma2(w, c[3], c[2]), c[1]), c[0]);
    }
};

// the launches of the two families, float32 and bf16
cudaError_t run_attn_fwd_f32(const AttnArgs& a, const void* q, const void* k, const void* v, void* o, float* lse, cudaStream_t st);
cudaError_t run_attn_bwd_f32(const AttnArgs& a, const void* q, const void* k, const void* v, const void* o, const float* lse, const void* dout,
                             float* delta, void* dq, void* dk, void* dv, cudaStream_t st);
cudaError_t run_attn_fwd_bf16(const AttnArgs& a, const void* q, const void* k, const void* v, void* o, void* rest, float* lse, cudaStream_t st);
cudaError_t run_attn_bwd_bf16(const AttnArgs& a, const void* q, const void* k, const void* v, const void* o, const void* rest,
                              const float* lse, const void* dout, float* delta, void* dq, void* dk, void* dv, cudaStream_t st);

// bf16 with a window of up to NARROW_WINDOW tokens, as many queries as keys and no prefix: kernels of their own, whose backward needs
// nothing of the forward
constexpr int NARROW_WINDOW = 65;
bool attn_narrow(const AttnArgs& a);
cudaError_t run_attn_fwd_narrow(const AttnArgs& a, const void* q, const void* k, const void* v, void* o, void* rest, float* lse, cudaStream_t st);
cudaError_t run_attn_bwd_narrow(const AttnArgs& a, const void* q, const void* k, const void* v, const void* dout, void* dq, void* dk, void* dv,
                                cudaStream_t st);

}  // namespace slotscan
