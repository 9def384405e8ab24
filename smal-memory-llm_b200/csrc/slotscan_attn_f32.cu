// Attention over tokens on the CUDA cores: float32, whose products the tensor cores would round to 11 bits or fewer.
//
// Forward: a CTA holds 64 or 32 queries of a head and passes over their keys 64 at a time, with the running maximum and sum of each
// row's softmax.  Backward: the same walk twice, once with rows of queries (dq, and delta = <do, o> for the other), once with
// rows of keys over the queries of all heads that share the key head (dk, dv): one more pair of products than a single walk with
// atomic sums would take, and the same bits from run to run.
//   rows X0, X1 / stream Y0, Y1:   queries: q, do / k, v      keys: k, v / q, do
//   s = X0 Y0^T, dp = X1 Y1^T, p = exp(s - lse), ds = p (dp - delta) (1 - tanh^2),  out1 += ds Y0,  keys also out0 += p Y1
// Bound by shared memory and its latency: a thread's 4 x 4 block takes eight 16-byte reads for 32 paired multiply-adds, with 8 warps on
// an SM in the backward.  One sequence of 4,096 with six heads of 128: 33 TFLOP/s forward, 33 of its seven products backward.
// Blocks of 2 x 4 with twice the warps took 1.4 times as long, unpaired multiply-adds 1.1 times.
// All heads' long rows first: of the CTAs of one head after the other a third of the SMs' time was lost at the end.
#include "slotscan_attn.cuh"
#include "slotscan_launch.h"

namespace slotscan {

constexpr int SA_N = 64, SA_LDP = SA_N + 4;              // rows of a step of the stream
constexpr int SA_SMS = 148;

template <typename T>
__device__ __forceinline__ float4 ld4or0(const T* p, bool ok) { return ok ? ld4(p) : make_float4(0.f, 0.f, 0.f, 0.f); }

// rows [r0, r0 + N) of a strided matrix into shared memory, zeros beyond `rows` and beyond D channels
template <int DP, int N, int THREADS, typename T>
__device__ __forceinline__ void load_tile(float* dst, const T* src, long long stride, int r0, int rows, int D) {
    for (int i = threadIdx.x; i < N * (DP / 4); i += THREADS) {
        const int r = i / (DP / 4), c = i % (DP / 4) * 4;
        st4(dst + r * (DP + 4) + c, ld4or0(src + (long long)(r0 + r) * stride + c, r0 + r < rows && c < D));
    }
}
// C[r][c] = <A row 4 ty + r, B row tx + 16 c>
template <int DP>
__device__ __forceinline__ void dot_block(float (&C)[4][4], const float* A, const float* Bm, int ty, int tx) {
    f32x2 sum[4][4];                                     // of the even and of the odd channels
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
        for (int c = 0; c < 4; c++) sum[r][c] = pack2(0.f, 0.f);
#pragma unroll 4
    for (int d = 0; d < DP; d += 4) {
        f32x4 x[4], y[4];
#pragma unroll
        for (int r = 0; r < 4; r++) x[r] = pack4(ld4(A + (4 * ty + r) * (DP + 4) + d));
#pragma unroll
        for (int c = 0; c < 4; c++) y[c] = pack4(ld4(Bm + (tx + 16 * c) * (DP + 4) + d));
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int c = 0; c < 4; c++) sum[r][c] = fma2(x[r].b, y[c].b, fma2(x[r].a, y[c].a, sum[r][c]));
    }
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const float2 t = unpack2(sum[r][c]);
            C[r][c] = t.x + t.y;
        }
}
// acc[r][8 channels of tx] += sum_j P[4 ty + r][j] Y[j]
template <int DP>
__device__ __forceinline__ void product_block(float (&acc)[4][DP / 16], const float* P, const float* Y, int ty, int tx) {
    for (int j = 0; j < SA_N; j += 4) {
        float4 p[4];
#pragma unroll
        for (int r = 0; r < 4; r++) p[r] = ld4(P + (4 * ty + r) * SA_LDP + j);
#pragma unroll
        for (int jj = 0; jj < 4; jj++) {
#pragma unroll
            for (int c = 0; c < DP / 64; c++) {
                const f32x4 y = pack4(ld4(Y + (j + jj) * (DP + 4) + tx * 4 + 64 * c));
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float w = jj == 0 ? p[r].x : jj == 1 ? p[r].y : jj == 2 ? p[r].z : p[r].w;
                    const f32x2 w2 = pack2(w, w);
                    const float2 lo = unpack2(fma2(w2, y.a, pack2(acc[r][4 * c], acc[r][4 * c + 1])));
                    const float2 hi = unpack2(fma2(w2, y.b, pack2(acc[r][4 * c + 2], acc[r][4 * c + 3])));
                    acc[r][4 * c] = lo.x;
                    acc[r][4 * c + 1] = lo.y;
                    acc[r][4 * c + 2] = hi.x;
                    acc[r][4 * c + 3] = hi.y;
                }
            }
        }
    }
}
__device__ __forceinline__ float max16(float v) {        // over the 16 lanes of a row block
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(FULL, v, off));
    return v;
}
// least lo and greatest hi of the CTA's 64 rows (the rows that do not exist have an empty span)
__device__ __forceinline__ Span cta_span(Span mine, bool counts, int* s_red) {
    if (threadIdx.x == 0) { s_red[0] = BIGI; s_red[1] = 0; }
    __syncthreads();
    if (counts && mine.hi > mine.lo) { atomicMin(&s_red[0], mine.lo); atomicMax(&s_red[1], mine.hi); }
    __syncthreads();
    return {s_red[0], s_red[1]};
}

template <typename T>
__device__ __forceinline__ void put_lane_row(T* row, const float (&x)[4], int D) {
#pragma unroll
    for (int c = 0; c < 4; c++) { const int d = (threadIdx.x & 31) + 32 * c; if (d < D) st1(row + d, x[c]); }
}
// `again(r)`, by the whole warp, for each of its eight rows r of the CTA whose sums `bad` says not to be finite; after the rows are stored
template <int N, typename Bad, typename Again>
__device__ __forceinline__ void again_where_not_finite(const float (&acc)[4][N], Bad bad, Again again) {
    const int ty = threadIdx.x / 16, warp = threadIdx.x / 32;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        float w = 0.f;
#pragma unroll
        for (int c = 0; c < N; c++) watch(w, acc[r][c]);
        const unsigned hit = __ballot_sync(FULL, bad(4 * ty + r, w));
#pragma unroll
        for (int half = 0; half < 2; half++)
            if (hit >> (16 * half) & 0xffffu) { __syncwarp(); again(4 * (2 * warp + half) + r); }
    }
}

template <int DP, int M, typename T>
__global__ void __launch_bounds__(4 * M, M == 64 ? 2 : 3) attn_fwd_cores_kernel(AttnArgs a, const T* q, const T* k, const T* v, T* o, float* lse) {
    extern __shared__ float4 smem4[];
    float* Qs = reinterpret_cast<float*>(smem4);
    float* Ys = Qs + M * (DP + 4);                    // keys, then values
    float* Ps = Ys + SA_N * (DP + 4);
    __shared__ int s_red[2];
    const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
    const int heads = a.H * a.B, h = blockIdx.x % heads % a.H, b = blockIdx.x % heads / a.H, hk = h / (a.H / a.KV);
    const int i0 = ((a.Tq + M - 1) / M - 1 - (int)(blockIdx.x / heads)) * M;       // the long rows of all heads first
    const T* kb = k + b * a.ks[0] + hk * a.ks[2];
    const T* vb = v + b * a.vs[0] + hk * a.vs[2];
    load_tile<DP, M, 4 * M>(Qs, q + b * a.qs[0] + h * a.qs[2], a.qs[1], i0, a.Tq, a.D);
    Span sp[4];
#pragma unroll
    for (int r = 0; r < 4; r++) sp[r] = i0 + 4 * ty + r < a.Tq ? keys_of(a, b, i0 + 4 * ty + r) : Span{0, 0};
    const Span all = cta_span(i0 + tid < a.Tq && tid < M ? keys_of(a, b, i0 + tid) : Span{0, 0}, tid < M, s_red);
    const Score sc(a, h);
    float m[4], l[4], acc[4][DP / 16];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        m[r] = -INFINITY; l[r] = 0.f;
#pragma unroll
        for (int c = 0; c < DP / 16; c++) acc[r][c] = 0.f;
    }
    for (int j0 = all.lo; j0 < all.hi; j0 += SA_N) {
        __syncthreads();
        load_tile<DP, SA_N, 4 * M>(Ys, kb, a.ks[1], j0, a.Tk, a.D);
        __syncthreads();
        float s[4][4];
        dot_block<DP>(s, Qs, Ys, ty, tx);
        float shrink[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int at = i0 + 4 * ty + r + a.Tk - a.Tq;
            float top = -INFINITY, unused;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int j = j0 + tx + 16 * c;
                s[r][c] = j >= sp[r].lo && j < sp[r].hi ? score2(sc, s[r][c], abs(at - j), unused) : -INFINITY;
                top = fmaxf(top, s[r][c]);
            }
            top = fmaxf(m[r], max16(top));
            const float base = top == -INFINITY ? 0.f : top;
            shrink[r] = exp2f(m[r] - base);
            m[r] = top;
            float sum = 0.f;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const float p = exp2f(s[r][c] - base);
                sum += p;
                Ps[(4 * ty + r) * SA_LDP + tx + 16 * c] = p;
            }
            l[r] = fmaf(l[r], shrink[r], group_sum<16>(sum));
#pragma unroll
            for (int c = 0; c < DP / 16; c++) acc[r][c] *= shrink[r];
        }
        __syncthreads();
        load_tile<DP, SA_N, 4 * M>(Ys, vb, a.vs[1], j0, a.Tk, a.D);
        __syncthreads();
        product_block<DP>(acc, Ps, Ys, ty, tx);
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int i = i0 + 4 * ty + r;
        if (i >= a.Tq) continue;
        const bool empty = sp[r].hi <= sp[r].lo;
        const float inv = empty ? 0.f : 1.f / l[r];
#pragma unroll
        for (int c = 0; c < DP / 64; c++) {
            const int d = tx * 4 + 64 * c;
            if (d < a.D)
                st4(o + (((size_t)b * a.Tq + i) * a.H + h) * a.D + d,
                    make_float4(acc[r][4 * c] * inv, acc[r][4 * c + 1] * inv, acc[r][4 * c + 2] * inv, acc[r][4 * c + 3] * inv));
        }
        if (lse != nullptr && tx == 0)
            lse[((size_t)b * a.H + h) * a.Tq + i] = empty ? -INFINITY : sp[r].hi - sp[r].lo == 1 ? INFINITY : m[r] + log2f(l[r]);
    }
    again_where_not_finite(acc, [&](int r, float w) { return i0 + r < a.Tq && w != w; }, [&](int r) {
        float x[4], unused0, unused1;
        careful_query(a, RowInputs<T>{q, k, v, nullptr}, b, h, i0 + r, x, unused0, unused1);
        put_lane_row(o + (((size_t)b * a.Tq + i0 + r) * a.H + h) * a.D, x, a.D);
    });
}

// KEYS: rows of keys (dk, dv); else rows of queries (dq, and delta)
template <int DP, int M, bool KEYS, typename T>
__global__ void __launch_bounds__(4 * M, DP == 64 ? 2 : 1) attn_bwd_cores_kernel(AttnArgs a, const T* q, const T* k, const T* v, const T* o, const float* lse,
                                                                    const T* dout, float* delta, T* d0, T* d1) {
    extern __shared__ float4 smem4[];
    float* X0 = reinterpret_cast<float*>(smem4);
    float* X1 = X0 + M * (DP + 4);
    float* Y0 = X1 + M * (DP + 4);
    float* Y1 = Y0 + SA_N * (DP + 4);
    float* Ps = Y1 + SA_N * (DP + 4);
    float* Ds = Ps + M * SA_LDP;
    __shared__ int s_red[2];
    __shared__ float s_lse[64], s_delta[64];             // of the queries: this CTA's rows, or the stream's
    const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16, group = a.H / a.KV;
    const int hs = KEYS ? a.KV : a.H, heads = hs * a.B, hx = blockIdx.x % heads % hs, b = blockIdx.x % heads / hs;
    const int off = a.Tk - a.Tq, rows = KEYS ? a.Tk : a.Tq, cols = KEYS ? a.Tq : a.Tk, tile = (int)(blockIdx.x / heads);
    const int r0 = (KEYS ? tile : (a.Tq + M - 1) / M - 1 - tile) * M;              // the long rows of all heads first
    const int hk = KEYS ? hx : hx / group;
    const long long os = (long long)a.H * a.D;           // of o and dout: contiguous
    const T* kb = k + b * a.ks[0] + hk * a.ks[2];
    const T* vb = v + b * a.vs[0] + hk * a.vs[2];
    if constexpr (KEYS) {
        load_tile<DP, M, 4 * M>(X0, kb, a.ks[1], r0, rows, a.D);
        load_tile<DP, M, 4 * M>(X1, vb, a.vs[1], r0, rows, a.D);
    } else {
        load_tile<DP, M, 4 * M>(X0, q + b * a.qs[0] + hx * a.qs[2], a.qs[1], r0, rows, a.D);
        load_tile<DP, M, 4 * M>(X1, dout + (size_t)b * a.Tq * os + hx * a.D, os, r0, rows, a.D);
    }
    auto span = [&](int r) { return r >= rows ? Span{0, 0} : KEYS ? queries_of(a, b, r) : keys_of(a, b, r); };
    Span sp[4];
#pragma unroll
    for (int r = 0; r < 4; r++) sp[r] = span(r0 + 4 * ty + r);
    const Span all = cta_span(tid < M ? span(r0 + tid) : Span{0, 0}, tid < M, s_red);
    if constexpr (!KEYS) {
        // delta of a row by four lanes; the products of a row are a sum over its channels, so it needs no other row
        const int r = tid / 4, i = r0 + r;
        float s = 0.f;
        if (i < a.Tq) {
            const T* ob = o + (((size_t)b * a.Tq + i) * a.H + hx) * a.D;
            for (int d = (tid % 4) * 4; d < a.D; d += 16) s += dot4(ld4(ob + d), ld4(X1 + r * (DP + 4) + d));
        }
        s += __shfl_xor_sync(FULL, s, 1);
        s += __shfl_xor_sync(FULL, s, 2);
        if (tid % 4 == 0) {
            const size_t at = ((size_t)b * a.H + hx) * a.Tq + i;
            s_delta[r] = s;
            s_lse[r] = i < a.Tq ? lse[at] : 0.f;
            if (i < a.Tq) delta[at] = s;
        }
    }
    float acc0[4][DP / 16], acc1[4][DP / 16];
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
        for (int c = 0; c < DP / 16; c++) acc0[r][c] = acc1[r][c] = 0.f;
    for (int g = 0; g < (KEYS ? group : 1); g++) {
        const int h = KEYS ? hk * group + g : hx;
        const Score sc(a, h);
        for (int y0 = all.lo; y0 < all.hi; y0 += SA_N) {
            __syncthreads();
            if constexpr (KEYS) {
                load_tile<DP, SA_N, 4 * M>(Y0, q + b * a.qs[0] + h * a.qs[2], a.qs[1], y0, cols, a.D);
                load_tile<DP, SA_N, 4 * M>(Y1, dout + (size_t)b * a.Tq * os + h * a.D, os, y0, cols, a.D);
                if (tid < SA_N) {
                    const bool in = y0 + tid < a.Tq;
                    const size_t at = ((size_t)b * a.H + h) * a.Tq + y0 + tid;
                    s_lse[tid] = in ? lse[at] : 0.f;
                    s_delta[tid] = in ? delta[at] : 0.f;
                }
            } else {
                load_tile<DP, SA_N, 4 * M>(Y0, kb, a.ks[1], y0, cols, a.D);
                load_tile<DP, SA_N, 4 * M>(Y1, vb, a.vs[1], y0, cols, a.D);
            }
            __syncthreads();
            float s[4][4], dp[4][4];
            dot_block<DP>(s, X0, Y0, ty, tx);
            dot_block<DP>(dp, X1, Y1, ty, tx);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int x = r0 + 4 * ty + r;
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const int yl = tx + 16 * c, y = y0 + yl, ql = KEYS ? yl : 4 * ty + r;
                    float p = 0.f, ds = 0.f;
                    if (y >= sp[r].lo && y < sp[r].hi) {
                        float f;
                        const float z = score2(sc, s[r][c], KEYS ? abs(y + off - x) : abs(x + off - y), f);
                        const bool single = s_lse[ql] == INFINITY;
                        p = single ? 1.f : exp2f(z - s_lse[ql]);
                        ds = single ? 0.f : p * (dp[r][c] - s_delta[ql]) * f;
                    }
                    if constexpr (KEYS) Ps[(4 * ty + r) * SA_LDP + yl] = p;
                    Ds[(4 * ty + r) * SA_LDP + yl] = ds;
                }
            }
            __syncthreads();
            if constexpr (KEYS) product_block<DP>(acc0, Ps, Y1, ty, tx);
            product_block<DP>(acc1, Ds, Y0, ty, tx);
        }
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int x = r0 + 4 * ty + r;
        if (x >= rows) continue;
        const size_t at = (((size_t)b * rows + x) * (KEYS ? a.KV : a.H) + hx) * a.D;
#pragma unroll
        for (int c = 0; c < DP / 64; c++) {
            const int d = tx * 4 + 64 * c;
            if (d >= a.D) continue;
            if constexpr (KEYS) st4(d0 + at + d, make_float4(acc0[r][4 * c], acc0[r][4 * c + 1], acc0[r][4 * c + 2], acc0[r][4 * c + 3]));
            st4(d1 + at + d, make_float4(acc1[r][4 * c] * a.scale, acc1[r][4 * c + 1] * a.scale, acc1[r][4 * c + 2] * a.scale, acc1[r][4 * c + 3] * a.scale));
        }
    }
    auto again = [&](int r) {
        const RowInputs<T> in = {q, k, v, dout};
        const size_t at = (((size_t)b * rows + r0 + r) * (KEYS ? a.KV : a.H) + hx) * a.D;
        float x[4], y[4];
        if constexpr (KEYS) {
            careful_dkv(a, in, lse, delta, b, hx, r0 + r, x, y);
            put_lane_row(d0 + at, y, a.D);
        } else careful_dq(a, in, lse, delta, b, hx, r0 + r, x);
        put_lane_row(d1 + at, x, a.D);
    };
    auto bad = [&](int r, float w) { return r0 + r < rows && w != w; };
    if constexpr (KEYS) again_where_not_finite(acc0, bad, again);
    again_where_not_finite(acc1, bad, again);
}

template <int DP, int M>
static cudaError_t fwd_cores(const AttnArgs& a, const void* q, const void* k, const void* v, void* o, float* lse, cudaStream_t st) {
    const size_t sm = sizeof(float) * ((M + SA_N) * (DP + 4) + M * SA_LDP);
    auto kern = attn_fwd_cores_kernel<DP, M, float>;
    const cudaError_t e = opt_in_smem(kern, sm);
    if (e != cudaSuccess) return e;
    const long long ctas = (long long)((a.Tq + M - 1) / M) * a.H * a.B;
    if (ctas > 0x7fffffffll) return cudaErrorInvalidValue;
    kern<<<(unsigned)ctas, 4 * M, sm, st>>>(a, (const float*)q, (const float*)k, (const float*)v, (float*)o, lse);
    return cudaGetLastError();
}
template <int DP, int M, bool KEYS>
static cudaError_t bwd_cores(const AttnArgs& a, const void* q, const void* k, const void* v, const void* o, const float* lse, const void* dout,
                             float* delta, void* d0, void* d1, cudaStream_t st) {
    const size_t sm = sizeof(float) * (2 * (M + SA_N) * (DP + 4) + 2 * M * SA_LDP);
    auto kern = attn_bwd_cores_kernel<DP, M, KEYS, float>;
    const cudaError_t e = opt_in_smem(kern, sm);
    if (e != cudaSuccess) return e;
    const long long ctas = (long long)(((KEYS ? a.Tk : a.Tq) + M - 1) / M) * (KEYS ? a.KV : a.H) * a.B;
    if (ctas > 0x7fffffffll) return cudaErrorInvalidValue;
    kern<<<(unsigned)ctas, 4 * M, sm, st>>>(a, (const float*)q, (const float*)k, (const float*)v, (const float*)o, lse, (const float*)dout, delta,
                                            (float*)d0, (float*)d1);
    return cudaGetLastError();
}
// 32 rows to a CTA where 64 would leave SMs without one.  The forward and the walk over queries of 64 channels, of whose CTAs
// several fit an SM, take 32 up to three of 64 for each SM.  With 64 rows against 32, us, forward + queries + keys:
//   2 x 1,881 tokens, one head of 128    288 + 389 + 485     222 + 281 + 339
//   4 x 1,024 tokens, four heads of 64   128 + 168 + 365     105 + 127 + 315
//   1 x 4,096 tokens, six heads of 128   864 + 1,234 + 1,527     792 + 1,618 + 1,951
//   34 x 494 tokens, twelve heads of 128     853 + 1,663 + 1,835     941 + 2,657 + 2,815
static bool few(int rows, int heads, int B, int each) { return (long long)((rows + 63) / 64) * heads * B < each * SA_SMS; }

template <int DP>
static cudaError_t fwd_cores_rows(const AttnArgs& a, const void* q, const void* k, const void* v, void* o, float* lse, cudaStream_t st) {
    return few(a.Tq, a.H, a.B, 3) ? fwd_cores<DP, 32>(a, q, k, v, o, lse, st) : fwd_cores<DP, 64>(a, q, k, v, o, lse, st);
}
template <int DP>
static cudaError_t bwd_cores_rows(const AttnArgs& a, const void* q, const void* k, const void* v, const void* o, const float* lse, const void* dout,
                                  float* delta, void* dq, void* dk, void* dv, cudaStream_t st) {
    const cudaError_t e = few(a.Tq, a.H, a.B, DP == 64 ? 3 : 1) ? bwd_cores<DP, 32, false>(a, q, k, v, o, lse, dout, delta, nullptr, dq, st)
                                              : bwd_cores<DP, 64, false>(a, q, k, v, o, lse, dout, delta, nullptr, dq, st);
    if (e != cudaSuccess) return e;
    return few(a.Tk, a.KV, a.B, 1) ? bwd_cores<DP, 32, true>(a, q, k, v, o, lse, dout, delta, dv, dk, st)
                                : bwd_cores<DP, 64, true>(a, q, k, v, o, lse, dout, delta, dv, dk, st);
}

cudaError_t run_attn_fwd_f32(const AttnArgs& a, const void* q, const void* k, const void* v, void* o, float* lse, cudaStream_t st) {
    return a.D <= 64 ? fwd_cores_rows<64>(a, q, k, v, o, lse, st) : fwd_cores_rows<128>(a, q, k, v, o, lse, st);
}
cudaError_t run_attn_bwd_f32(const AttnArgs& a, const void* q, const void* k, const void* v, const void* o, const float* lse, const void* dout,
                             float* delta, void* dq, void* dk, void* dv, cudaStream_t st) {
    return a.D <= 64 ? bwd_cores_rows<64>(a, q, k, v, o, lse, dout, delta, dq, dk, dv, st)
                     : bwd_cores_rows<128>(a, q, k, v, o, lse, dout, delta, dq, dk, dv, st);
}
}  // namespace slotscan
