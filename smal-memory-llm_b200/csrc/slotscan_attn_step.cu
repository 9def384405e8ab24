// Attention of one query for each sequence over ring caches: the step of a generation loop.
//
// Every visible key and value is read once, for all query heads that share it: bound by those bytes.  The visible positions of a
// (sequence, key head) are split evenly among S CTAs, whatever their number turns out to be on the device; with S > 1 a second kernel
// joins the splits.
//
// bf16: the heads of a group are the rows of m16n8k16 products (up to 16 of them, the others zero), the keys the columns.  The
// tensor cores idle most of the time all the same; what they save is instructions, which on the CUDA cores took longer than
// the bytes do (one key in 20 instructions a head; 32 sequences of 8,192, three heads to a key head: 233 us so, 79 now).  tcgen05
// would compute 128 rows for these few.  Each warp streams 16 keys and values a step through a ring of its own in shared memory, several
// steps ahead (cp.async, zero-filled beyond its span), with a maximum, a sum and an output of its own; the warps are joined at the end.
// p is split into two bf16 (p = hi + lo, off by 2^-17): the second product costs nothing here and keeps the float32 weights' precision.
//
// float32: the CUDA cores.  A row is read by LPG lanes, 8 channels each, and every group of lanes goes its own way through the split.
#include <cfloat>

#include "slotscan_attn.cuh"
#include "slotscan_launch.h"
#include "slotscan_tensor.cuh"

namespace slotscan {

constexpr int ST_THREADS = 128;
constexpr int ST_U = 2;                                  // rows a turn of a group of lanes, the next turn's in flight
constexpr int ST_MAX_SPLITS = 256;

struct StepArgs {
    int B, H, KV, D, L, window;                          // window 1 .. L
    int splits, chunks;                                  // chunks of query heads to a key head
    float scale, cap;
    long long qs[2], ks[3], vs[3];
    const int32_t *pos, *start;
    const float* slopes;
};

struct Softmax { float m, l; };                          // running maximum (base-2 exponent) and sum
// what a split hands to the join as its maximum: minus infinity says that the query sees nothing at all
__device__ __forceinline__ float split_max(int visible, float top) { return visible == 0 ? -INFINITY : fmaxf(top, -FLT_MAX); }

template <typename T, int LPG, int G>
__global__ void __launch_bounds__(ST_THREADS) attn_step_kernel(StepArgs a, const T* q, const T* k, const T* v, T* o, float* part) {
    constexpr int GROUPS = ST_THREADS / LPG, DP = LPG * 8;
    __shared__ float s_acc[GROUPS][G][DP];
    __shared__ Softmax s_sm[GROUPS][G];
    const int c = threadIdx.x % LPG, grp = threadIdx.x / LPG;
    const int split = blockIdx.x, hk = blockIdx.y / a.chunks, b = blockIdx.z, group = a.H / a.KV;
    const int g0 = (blockIdx.y % a.chunks) * G;          // first query head of this CTA within its group
    const bool live = c * 8 < a.D;
    const long long pos = a.pos[b];
    const long long first = max(max(pos - a.window + 1, a.start != nullptr ? (long long)a.start[b] : 0ll), 0ll);
    const int n = (int)max(pos - first + 1, 0ll), per = (n + a.splits - 1) / a.splits;
    const int lo = min(split * per, n), hi = min(lo + per, n);
    const int row0 = n > 0 ? (int)(first % a.L) : 0;
    float qr[G][8], acc[G][8], slope[G];
    Softmax sm[G];
#pragma unroll
    for (int g = 0; g < G; g++) {
        const int h = hk * group + min(g0 + g, group - 1);
#pragma unroll
        for (int i = 0; i < 8; i++) qr[g][i] = acc[g][i] = 0.f;
        if (live) ld8(qr[g], q + b * a.qs[0] + h * a.qs[1] + c * 8);
        const float in = a.cap > 0.f ? a.scale / a.cap : a.scale * LOG2E;
#pragma unroll
        for (int i = 0; i < 8; i++) qr[g][i] *= in;
        slope[g] = a.slopes != nullptr ? a.slopes[h] * LOG2E : 0.f;
        sm[g] = {-INFINITY, 0.f};
    }
    const T* kb = k + b * a.ks[0] + hk * a.ks[2] + c * 8;
    const T* vb = v + b * a.vs[0] + hk * a.vs[2] + c * 8;
    float kn[ST_U][8], vn[ST_U][8];
    auto load = [&](int j0) {                            // the rows of a turn; zeros beyond the split
#pragma unroll
        for (int u = 0; u < ST_U; u++) {
            const int j = j0 + u * GROUPS + grp;
#pragma unroll
            for (int i = 0; i < 8; i++) kn[u][i] = vn[u][i] = 0.f;
            if (j < hi && live) {
                const int r = row0 + j, row = r >= a.L ? r - a.L : r;              // j < n <= L
                ld8(kn[u], kb + row * a.ks[1]);
                ld8(vn[u], vb + row * a.vs[1]);
            }
        }
    };
    load(lo);
    for (int j0 = lo; j0 < hi; j0 += GROUPS * ST_U) {
        float kx[ST_U][8], vx[ST_U][8];
#pragma unroll
        for (int u = 0; u < ST_U; u++)
#pragma unroll
            for (int i = 0; i < 8; i++) { kx[u][i] = kn[u][i]; vx[u][i] = vn[u][i]; }
        load(j0 + GROUPS * ST_U);
#pragma unroll
        for (int g = 0; g < G; g++) {
            float z[ST_U], top = sm[g].m;
#pragma unroll
            for (int u = 0; u < ST_U; u++) {
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) s = fmaf(qr[g][i], kx[u][i], s);
                s = group_sum<LPG>(s);
                if (a.cap > 0.f) s = a.cap * LOG2E * tanhf(s);
                s = fmaf(-slope[g], (float)(n - 1 - (j0 + u * GROUPS + grp)), s);
                z[u] = j0 + u * GROUPS + grp < hi ? s : -INFINITY;
                top = fmaxf(top, z[u]);
            }
            const float base = top == -INFINITY ? 0.f : top;
            const float shrink = exp2f(sm[g].m - base);
            float p[ST_U], sum = 0.f;
#pragma unroll
            for (int u = 0; u < ST_U; u++) { p[u] = exp2f(z[u] - base); sum += p[u]; }
            sm[g].m = top;
            sm[g].l = fmaf(sm[g].l, shrink, sum);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float t = acc[g][i] * shrink;
#pragma unroll
                for (int u = 0; u < ST_U; u++) t = fmaf(p[u], vx[u][i], t);
                acc[g][i] = t;
            }
        }
    }
#pragma unroll
    for (int g = 0; g < G; g++) {
        st8(&s_acc[grp][g][c * 8], acc[g]);
        if (c == 0) s_sm[grp][g] = sm[g];
    }
    __syncthreads();
    for (int x = threadIdx.x; x < G * a.D; x += ST_THREADS) {
        const int g = x / a.D, d = x % a.D, h = hk * group + g0 + g;
        if (g0 + g >= group) continue;
        float top = -INFINITY, l = 0.f, s = 0.f;
        for (int i = 0; i < GROUPS; i++) top = fmaxf(top, s_sm[i][g].m);
        const float base = top == -INFINITY ? 0.f : top;
        for (int i = 0; i < GROUPS; i++) {
            const float f = exp2f(s_sm[i][g].m - base);
            l = fmaf(s_sm[i][g].l, f, l);
            s = fmaf(s_acc[i][g][d], f, s);
        }
        if (a.splits == 1) st1(o + ((size_t)b * a.H + h) * a.D + d, n == 0 ? 0.f : s / l);
        else {
            float* pp = part + (((size_t)b * a.H + h) * a.splits + split) * (a.D + 2);
            pp[d] = s;
            if (d == 0) { pp[a.D] = split_max(n, top); pp[a.D + 1] = l; }
        }
    }
}

// ---- bf16 ----
constexpr int SM_WARPS = 4, SM_KEYS = 16, SM_STAGES = 3;

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
}
// 16 bytes into shared memory, zeros unless `in`
__device__ __forceinline__ void cp_async16_or0(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}

// WIDE: 16 query heads to a CTA, else 8
template <int DP, bool WIDE>
__global__ void __launch_bounds__(SM_WARPS * 32) attn_step_mma_kernel(StepArgs a, const bf16* q, const bf16* k, const bf16* v, bf16* o, float* part) {
    constexpr int PIECES = DP / 8, PER_PASS = 32 / PIECES, ROW = DP * 2, TILE = SM_KEYS * ROW, R = WIDE ? 2 : 1, HEADS = 8 * R;
    extern __shared__ float4 smem4[];
    __shared__ Softmax s_sm[SM_WARPS][HEADS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const int split = blockIdx.x, hk = blockIdx.y / a.chunks, b = blockIdx.z, group = a.H / a.KV, g0 = (blockIdx.y % a.chunks) * HEADS;
    const long long pos = a.pos[b];
    const long long first = max(max(pos - a.window + 1, a.start != nullptr ? (long long)a.start[b] : 0ll), 0ll);
    const int n = (int)max(pos - first + 1, 0ll), per = (n + a.splits - 1) / a.splits;
    const int lo = min(split * per, n), hi = min(lo + per, n);
    const int row0 = n > 0 ? (int)(first % a.L) : 0;
    const uint32_t ring = smem_u32(smem4) + warp * SM_STAGES * 2 * TILE;
    const bf16* kb = k + b * a.ks[0] + hk * a.ks[2];
    const bf16* vb = v + b * a.vs[0] + hk * a.vs[2];
    const int piece = lane % PIECES, sub = lane / PIECES;
    auto load = [&](int step) {                          // 16 keys and values of this warp's step into its ring
        const int j0 = lo + (step * SM_WARPS + warp) * SM_KEYS;
        if (j0 < hi) {
            const uint32_t to = ring + (step % SM_STAGES) * 2 * TILE;
#pragma unroll
            for (int i = 0; i < SM_KEYS / PER_PASS; i++) {
                const int key = i * PER_PASS + sub, j = j0 + key, r = row0 + j, row = r >= a.L ? r - a.L : r;          // j < n <= L
                const bool in = j < hi && piece * 8 < a.D;
                const uint32_t at = to + key * ROW + (((piece & ~7) | ((piece ^ key) & 7)) << 4);
                cp_async16_or0(at, in ? kb + row * a.ks[1] + piece * 8 : kb, in);
                cp_async16_or0(at + TILE, in ? vb + row * a.vs[1] + piece * 8 : vb, in);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int s = 0; s < SM_STAGES - 1; s++) load(s);
    // the queries as A fragments: row = head; heads beyond the group repeat its last, and are not stored
    uint32_t qf[DP / 16][4];
    float slope[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int h = hk * group + min(g0 + lane / 4 + 8 * r, group - 1);
        const bf16* qh = q + b * a.qs[0] + h * a.qs[1];
        slope[r] = a.slopes != nullptr ? a.slopes[h] * LOG2E : 0.f;
#pragma unroll
        for (int kk = 0; kk < DP / 16; kk++)
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const int d = kk * 16 + half * 8 + (lane % 4) * 2;
                qf[kk][half * 2 + r] = d < a.D ? *reinterpret_cast<const uint32_t*>(qh + d) : 0u;
                if (!WIDE) qf[kk][half * 2 + 1] = 0u;
            }
    }
    const bool capped = a.cap > 0.f;
    const float lin = capped ? a.scale / a.cap * (2.f * LOG2E) : a.scale * LOG2E, cap2 = a.cap * LOG2E;
    float m[R], l[R], acc[DP / 8][4];
#pragma unroll
    for (int r = 0; r < R; r++) { m[r] = -INFINITY; l[r] = 0.f; }
#pragma unroll
    for (int c = 0; c < DP / 8; c++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[c][i] = 0.f;
    for (int step = 0;; step++) {
        const int j0 = lo + (step * SM_WARPS + warp) * SM_KEYS;
        if (j0 >= hi) break;                             // the same in all lanes of the warp
        asm volatile("cp.async.wait_group %0;" ::"n"(SM_STAGES - 2) : "memory");
        __syncwarp();
        const uint32_t ks = ring + (step % SM_STAGES) * 2 * TILE, vs = ks + TILE;
        float s[2][4];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[t][i] = 0.f;
#pragma unroll
        for (int kk = 0; kk < DP / 16; kk++) {
            uint32_t f[4];
            const int key = (lane / 16) * 8 + lane % 8, pc = kk * 2 + (lane / 8) % 2;
            ldsm4(f, ks + key * ROW + (((pc & ~7) | ((pc ^ key) & 7)) << 4));
            mma16(s[0], qf[kk], f[0], f[1]);
            mma16(s[1], qf[kk], f[2], f[3]);
        }
        uint32_t ph[4], pl[4];
        if (!WIDE) ph[1] = ph[3] = pl[1] = pl[3] = 0u;
#pragma unroll
        for (int r = 0; r < R; r++) {
            float z[4], top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int j = j0 + (i / 2) * 8 + (lane % 4) * 2 + i % 2;
                float x = s[i / 2][2 * r + i % 2] * lin;
                if (capped) x = fmaf(-2.f * cap2, __fdividef(1.f, exp2f(x) + 1.f), cap2);      // tanh x = 1 - 2 / (e^2x + 1)
                x = fmaf(-slope[r], (float)(n - 1 - j), x);
                z[i] = j < hi ? x : -INFINITY;
                top = fmaxf(top, z[i]);
            }
            top = fmaxf(top, __shfl_xor_sync(FULL, top, 1));
            top = fmaxf(top, __shfl_xor_sync(FULL, top, 2));
            top = fmaxf(top, m[r]);
            const float base = top == -INFINITY ? 0.f : top;
            if (__any_sync(FULL, top > m[r])) {
                const float shrink = exp2f(m[r] - base);
                l[r] *= shrink;
#pragma unroll
                for (int c = 0; c < DP / 8; c++) { acc[c][2 * r] *= shrink; acc[c][2 * r + 1] *= shrink; }
                m[r] = top;
            }
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; i++) { p[i] = exp2f(z[i] - base); l[r] += p[i]; }
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const uint32_t w = pack_bf16(p[2 * t], p[2 * t + 1]);
                ph[2 * t + r] = w;
                pl[2 * t + r] = pack_bf16(p[2 * t] - __uint_as_float(w << 16), p[2 * t + 1] - __uint_as_float(w & 0xffff0000u));
            }
        }
#pragma unroll
        for (int c = 0; c < DP / 8; c += 2) {
            uint32_t f[4];
            const int key = ((lane / 8) % 2) * 8 + lane % 8, pc = c + lane / 16;
            ldsm4_t(f, vs + key * ROW + (((pc & ~7) | ((pc ^ key) & 7)) << 4));
            mma16(acc[c], ph, f[0], f[1]);
            mma16(acc[c], pl, f[0], f[1]);
            mma16(acc[c + 1], ph, f[2], f[3]);
            mma16(acc[c + 1], pl, f[2], f[3]);
        }
        __syncwarp();
        load(step + SM_STAGES - 1);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();                                     // the ring becomes the warps' outputs
    float* s_acc = reinterpret_cast<float*>(smem4);      // [warp][head][DP]
#pragma unroll
    for (int r = 0; r < R; r++) {
        l[r] += __shfl_xor_sync(FULL, l[r], 1);
        l[r] += __shfl_xor_sync(FULL, l[r], 2);
        if (lane % 4 == 0) s_sm[warp][lane / 4 + 8 * r] = {m[r], l[r]};
#pragma unroll
        for (int c = 0; c < DP / 8; c++)
            *reinterpret_cast<float2*>(&s_acc[(warp * HEADS + lane / 4 + 8 * r) * DP + c * 8 + (lane % 4) * 2]) = make_float2(acc[c][2 * r], acc[c][2 * r + 1]);
    }
    __syncthreads();
    for (int x = threadIdx.x; x < min(HEADS, group - g0) * a.D; x += SM_WARPS * 32) {
        const int g = x / a.D, d = x % a.D, h = hk * group + g0 + g;
        float top = -INFINITY, ll = 0.f, sum = 0.f;
#pragma unroll
        for (int i = 0; i < SM_WARPS; i++) top = fmaxf(top, s_sm[i][g].m);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int i = 0; i < SM_WARPS; i++) {
            const float f = exp2f(s_sm[i][g].m - base);
            ll = fmaf(s_sm[i][g].l, f, ll);
            sum = fmaf(s_acc[(i * HEADS + g) * DP + d], f, sum);
        }
        if (a.splits == 1) o[((size_t)b * a.H + h) * a.D + d] = __float2bfloat16_rn(n == 0 ? 0.f : sum / ll);
        else {
            float* pp = part + (((size_t)b * a.H + h) * a.splits + split) * (a.D + 2);
            pp[d] = sum;
            if (d == 0) { pp[a.D] = split_max(n, top); pp[a.D + 1] = ll; }
        }
    }
}

// o = the splits' sums joined, a CTA to a (sequence, head)
template <typename T>
__global__ void __launch_bounds__(128) attn_step_join_kernel(const float* part, int splits, int D, T* o) {
    __shared__ float s_f[ST_MAX_SPLITS], s_red[2];
    const float* pp = part + (size_t)blockIdx.x * splits * (D + 2);
    const int tid = threadIdx.x;
    if (tid < 32) {
        float top = -INFINITY, l = 0.f;
        for (int i = tid; i < splits; i += 32) top = fmaxf(top, pp[(size_t)i * (D + 2) + D]);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, off));
        const float base = top == -INFINITY ? 0.f : top;
        for (int i = tid; i < splits; i += 32) {
            const float f = exp2f(pp[(size_t)i * (D + 2) + D] - base);
            s_f[i] = f;
            l = fmaf(pp[(size_t)i * (D + 2) + D + 1], f, l);
        }
        l = warp_sum(l);
        if (tid == 0) { s_red[0] = l; s_red[1] = top; }
    }
    __syncthreads();
    for (int d = tid; d < D; d += 128) {
        float s = 0.f;
        for (int i = 0; i < splits; i++) s = fmaf(pp[(size_t)i * (D + 2) + d], s_f[i], s);
        st1(o + (size_t)blockIdx.x * D + d, s_red[1] == -INFINITY ? 0.f : s / s_red[0]);
    }
}

static int heads_at_once(int group, int dtype) { return dtype == SLOTSCAN_BF16 ? (group > 8 ? 16 : 8) : group > 4 ? 8 : group; }

static StepArgs step_args(const slotscan_attn_step_params& p) {
    StepArgs a;
    a.B = p.B; a.H = p.H; a.KV = p.KV; a.D = p.D; a.L = p.L;
    a.window = p.window > 0 && p.window < p.L ? p.window : p.L;
    a.scale = p.scale; a.cap = p.cap;
    for (int i = 0; i < 2; i++) a.qs[i] = p.q_stride[i];
    for (int i = 0; i < 3; i++) { a.ks[i] = p.k_stride[i]; a.vs[i] = p.v_stride[i]; }
    const int group = p.H / p.KV, G = heads_at_once(group, p.dtype);
    a.chunks = (group + G - 1) / G;
    // 128 rows at least; bf16: two CTAs for each SM at a time (their rings), six rounds of them (8 x 131,072 rows: two rounds 384 us, four
    // 363, six 341, eight 351); float32: eight for each SM.  Rounded up: 32 sequences over four key heads take 14 splits, 1,792 CTAs, the last
    // 16 of them in a seventh round
    const long long ctas = (long long)p.B * p.KV * a.chunks, want = 148 * (p.dtype == SLOTSCAN_BF16 ? 12 : 8);
    long long s = (want + ctas - 1) / (ctas > 0 ? ctas : 1);
    if (s > (a.window + 127) / 128) s = (a.window + 127) / 128;
    a.splits = (int)(s < 1 ? 1 : s > ST_MAX_SPLITS ? ST_MAX_SPLITS : s);
    return a;
}

template <int LPG>
static cudaError_t launch_step_f32(const StepArgs& a, const void* q, const void* k, const void* v, void* o, float* part, cudaStream_t st) {
    const dim3 grid(a.splits, a.KV * a.chunks, a.B);
    auto go = [&](auto kern) { kern<<<grid, ST_THREADS, 0, st>>>(a, (const float*)q, (const float*)k, (const float*)v, (float*)o, part); };
    switch (heads_at_once(a.H / a.KV, SLOTSCAN_F32)) {
        case 1: go(attn_step_kernel<float, LPG, 1>); break;
        case 2: go(attn_step_kernel<float, LPG, 2>); break;
        case 3: go(attn_step_kernel<float, LPG, 3>); break;
        case 4: go(attn_step_kernel<float, LPG, 4>); break;
        default: go(attn_step_kernel<float, LPG, 8>); break;
    }
    if (a.splits > 1) attn_step_join_kernel<float><<<a.B * a.H, 128, 0, st>>>(part, a.splits, a.D, (float*)o);
    return cudaGetLastError();
}
template <int DP>
static cudaError_t launch_step_bf16(const StepArgs& a, const void* q, const void* k, const void* v, void* o, float* part, cudaStream_t st) {
    const size_t sm = (size_t)SM_WARPS * SM_STAGES * 2 * SM_KEYS * DP * 2;
    auto kern = heads_at_once(a.H / a.KV, SLOTSCAN_BF16) == 16 ? attn_step_mma_kernel<DP, true> : attn_step_mma_kernel<DP, false>;
    const cudaError_t e = opt_in_smem(kern, sm);
    if (e != cudaSuccess) return e;
    kern<<<dim3(a.splits, a.KV * a.chunks, a.B), SM_WARPS * 32, sm, st>>>(a, (const bf16*)q, (const bf16*)k, (const bf16*)v, (bf16*)o, part);
    if (a.splits > 1) attn_step_join_kernel<bf16><<<a.B * a.H, 128, 0, st>>>(part, a.splits, a.D, (bf16*)o);
    return cudaGetLastError();
}

}  // namespace slotscan

using namespace slotscan;

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

extern "C" int slotscan_attn_step_check(const slotscan_attn_step_params* p) {
    if (p == nullptr) return SLOTSCAN_E_NULL;
    if (p->dtype != SLOTSCAN_F32 && p->dtype != SLOTSCAN_BF16) return SLOTSCAN_E_DTYPE;
    if (p->B < 0 || p->B > 65535 || p->H < 1 || p->KV < 1 || p->H > 65535 || p->H % p->KV || p->D < 8 || p->D > 128 || p->D % 8 || p->L < 1 ||
        p->L > (1 << 29))
        return SLOTSCAN_E_SHAPE;
    if (p->window < 0 || !(p->cap >= 0.f) || !(p->cap < INFINITY) || !(p->scale > 0.f) || !(p->scale < INFINITY)) return SLOTSCAN_E_MODE;
    const int e = p->dtype == SLOTSCAN_BF16 ? 2 : 4;
    for (int i = 0; i < 3; i++)
        if ((i < 2 && p->q_stride[i] * e % 16) || p->k_stride[i] * e % 16 || p->v_stride[i] * e % 16) return SLOTSCAN_E_ALIGN;
    return SLOTSCAN_OK;
}

extern "C" size_t slotscan_attn_step_scratch_bytes(const slotscan_attn_step_params* p) {
    if (slotscan_attn_step_check(p) != SLOTSCAN_OK) return 0;
    const StepArgs a = step_args(*p);
    return a.splits == 1 ? 0 : sizeof(float) * (size_t)a.B * a.H * a.splits * (a.D + 2);
}

extern "C" int slotscan_attn_step(const slotscan_attn_step_params* p, const void* q, const void* k, const void* v, const int32_t* pos,
                                  const int32_t* start, const float* slopes, void* o, void* scratch, size_t scratch_bytes, void* stream) {
    const int rc = slotscan_attn_step_check(p);
    if (rc != SLOTSCAN_OK) return rc;
    if (p->B == 0) return SLOTSCAN_OK;
    if (!q || !k || !v || !pos || !o) return SLOTSCAN_E_NULL;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o)) return SLOTSCAN_E_ALIGN;
    StepArgs a = step_args(*p);
    const size_t need = slotscan_attn_step_scratch_bytes(p);
    if (need && (scratch == nullptr || scratch_bytes < need)) return SLOTSCAN_E_NULL;
    a.pos = pos; a.start = start; a.slopes = slopes;
    cudaStream_t st = (cudaStream_t)stream;
    if (p->dtype == SLOTSCAN_BF16) return (int)(p->D <= 64 ? launch_step_bf16<64>(a, q, k, v, o, (float*)scratch, st) : launch_step_bf16<128>(a, q, k, v, o, (float*)scratch, st));
    return (int)(p->D <= 64 ? launch_step_f32<8>(a, q, k, v, o, (float*)scratch, st) : launch_step_f32<16>(a, q, k, v, o, (float*)scratch, st));
}
