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

// The capped score as a polynomial, for |x| <= 1 (x = scale <q, k> / cap): tanh x = x sum_k a_k x^2k, the a_k fitted here for the least
// greatest error of tanh (iteratively reweighted least squares on Chebyshev nodes): 2.4e-7.  Three and a half instructions a score,
// two scores to an instruction, where the exponential form takes two of the special function unit's, eight cycles a warp each; a
// block with a larger score takes that form.  The coefficients carry cap and scale: base-2 exponent = s sum_k c_k s^2k.
struct CapPoly {
    f32x2 c[6];
    float most;                                          // the greatest |s| it serves
    __device__ __forceinline__ explicit CapPoly(const Score& sc) {
        const float a[6] = {0.9999968538152487f, -0.333240039679371f, 0.13253525772679928f, -0.050972871352707325f, 0.016114187219736308f, -0.002839467407190691f};
        float f = sc.cap_out * sc.cap_in;
#pragma unroll
        for (int k = 0; k < 6; k++) { c[k] = pack2(a[k] * f, a[k] * f); f *= sc.cap_in * sc.cap_in; }
        most = 1.f / sc.cap_in;
    }
    // two scores without their last factor: exponents = s * slope(s)
    __device__ __forceinline__ f32x2 slope(f32x2 s) const {
        const f32x2 w = mul2(s, s);
        return fma2(w, fma2(w, fma2(w, fma2(w, fma2(w, c[5], c[4]), c[3]), c[2]), c[1]), c[0]);
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
cudaError_t run_attn_fwd_narrow(const AttnArgs& a, const void* q, const void* k, const void* v, void* o, cudaStream_t st);
cudaError_t run_attn_bwd_narrow(const AttnArgs& a, const void* q, const void* k, const void* v, const void* dout, void* dq, void* dk, void* dv,
                                cudaStream_t st);

}  // namespace slotscan
