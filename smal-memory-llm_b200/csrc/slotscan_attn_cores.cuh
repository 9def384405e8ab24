// Products of attention on the CUDA cores, float32: tiles in shared memory, a thread's 4 x 4 block of scores and its slice of the outputs.
#pragma once
#include "slotscan_attn.cuh"

namespace slotscan {

constexpr int SA_N = 64, SA_LDP = SA_N + 4;              // rows of a step of the stream

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

}  // namespace slotscan
