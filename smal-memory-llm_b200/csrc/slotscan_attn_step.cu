// Attention of one query for each sequence over ring caches: the step of a generation loop.
//
// Every visible key and value is read once, for all query heads that share it: bound by those bytes.  Some 20 operations a key and
// head on the CUDA cores hide behind them up to six heads to a key head; tensor cores would have 16 rows to fill with those heads.
//
// The visible positions of a (sequence, key head) are split evenly among S CTAs, whatever their number turns out to be on the device.
// In a CTA a row is read by LPG lanes, 8 channels each, and every group of lanes goes its own way through the split, U rows at a
// time with all their loads ahead, with a maximum, a sum and an output of its own.  The groups are joined at the end, in their
// order; with S > 1 a second kernel joins the splits.
#include "slotscan_attn.cuh"
#include "slotscan_launch.h"

namespace slotscan {

constexpr int ST_THREADS = 128;
constexpr int ST_U = 4;                                  // rows in flight to a group of lanes
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
    for (int j0 = lo; j0 < hi; j0 += GROUPS * ST_U) {
        float kx[ST_U][8], vx[ST_U][8];
        bool in[ST_U];
#pragma unroll
        for (int u = 0; u < ST_U; u++) {
            const int j = j0 + u * GROUPS + grp;
            in[u] = j < hi;
#pragma unroll
            for (int i = 0; i < 8; i++) kx[u][i] = vx[u][i] = 0.f;
            if (in[u] && live) {
                const int r = row0 + j, row = r >= a.L ? r - a.L : r;              // j < n <= L
                ld8(kx[u], kb + row * a.ks[1]);
                ld8(vx[u], vb + row * a.vs[1]);
            }
        }
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
                z[u] = in[u] ? s : -INFINITY;
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
            if (d == 0) { pp[a.D] = top; pp[a.D + 1] = l; }
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
        if (tid == 0) s_red[0] = l;
    }
    __syncthreads();
    for (int d = tid; d < D; d += 128) {
        float s = 0.f;
        for (int i = 0; i < splits; i++) s = fmaf(pp[(size_t)i * (D + 2) + d], s_f[i], s);
        st1(o + (size_t)blockIdx.x * D + d, s_red[0] == 0.f ? 0.f : s / s_red[0]);
    }
}

static int heads_at_once(int group) { return group >= 8 || group > 4 ? 8 : group; }

static StepArgs step_args(const slotscan_attn_step_params& p) {
    StepArgs a;
    a.B = p.B; a.H = p.H; a.KV = p.KV; a.D = p.D; a.L = p.L;
    a.window = p.window > 0 && p.window < p.L ? p.window : p.L;
    a.scale = p.scale; a.cap = p.cap;
    for (int i = 0; i < 2; i++) a.qs[i] = p.q_stride[i];
    for (int i = 0; i < 3; i++) { a.ks[i] = p.k_stride[i]; a.vs[i] = p.v_stride[i]; }
    const int group = p.H / p.KV, G = heads_at_once(group);
    a.chunks = (group + G - 1) / G;
    // eight CTAs for each SM, of 128 rows at least
    const long long ctas = (long long)p.B * p.KV * a.chunks;
    long long s = (148 * 8 + ctas - 1) / (ctas > 0 ? ctas : 1);
    if (s > (a.window + 127) / 128) s = (a.window + 127) / 128;
    a.splits = (int)(s < 1 ? 1 : s > ST_MAX_SPLITS ? ST_MAX_SPLITS : s);
    return a;
}

template <typename T, int LPG>
static cudaError_t launch_step(const StepArgs& a, const void* q, const void* k, const void* v, void* o, float* part, cudaStream_t st) {
    const dim3 grid(a.splits, a.KV * a.chunks, a.B);
    auto go = [&](auto kern) { kern<<<grid, ST_THREADS, 0, st>>>(a, (const T*)q, (const T*)k, (const T*)v, (T*)o, part); };
    switch (heads_at_once(a.H / a.KV)) {
        case 1: go(attn_step_kernel<T, LPG, 1>); break;
        case 2: go(attn_step_kernel<T, LPG, 2>); break;
        case 3: go(attn_step_kernel<T, LPG, 3>); break;
        case 4: go(attn_step_kernel<T, LPG, 4>); break;
        default: go(attn_step_kernel<T, LPG, 8>); break;
    }
    if (a.splits > 1) attn_step_join_kernel<T><<<a.B * a.H, 128, 0, st>>>(part, a.splits, a.D, (T*)o);
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
    const bool h = p->dtype == SLOTSCAN_BF16;
    if (p->D <= 64) return (int)(h ? launch_step<bf16, 8>(a, q, k, v, o, (float*)scratch, st) : launch_step<float, 8>(a, q, k, v, o, (float*)scratch, st));
    return (int)(h ? launch_step<bf16, 16>(a, q, k, v, o, (float*)scratch, st) : launch_step<float, 16>(a, q, k, v, o, (float*)scratch, st));
}
