// Attention of one query for each request over pages: the step of a server's loop.
//
// Every visible key and value is read once for all query heads that share it: bound by those bytes.  Requests are of uneven lengths, so the
// work is cut by keys and not by requests: all visible keys of all (request, key head) pairs, one behind the other, in steps of 16, are shared
// out evenly among the warps of one round of CTAs.  A warp goes through its steps with a ring of its own in shared memory (cp.async, zero-filled
// beyond what is seen), which it does not drain where one pair ends and the next begins.  It joins nothing with other warps: where it has
// all of a pair it writes the result, else its part, and a second kernel joins the parts of a pair in their order.
//
// bf16: the heads of a group are the rows of m16n8k16 products (up to 16 of them, the others zero), the keys the columns.  p is split into
// two bf16 (p = hi + lo, off by 2^-17): the second product costs nothing here and keeps the float32 weights' precision.
// float32: the CUDA cores.  A row is read by LPG lanes, 8 channels each.
// 8 requests of up to 131,072 tokens over six key heads (2.2 GB): 357 us, 6.1 TB/s, over inputs that change; 318 where the same are read again
// and again, part of them from the cache.  32 of up to 8,192 over four: 57, of which 5 for the join.  One round of warps: where one took
// 370 us, in an earlier form, two to six shorter ones took up to 393, for the ends of shares and the search for them.
#include "slotscan_async.cuh"
#include "slotscan_launch.h"
#include "slotscan_paged.cuh"
#include "slotscan_tensor.cuh"
#include "slotscan_warp_mma.cuh"

namespace slotscan {

constexpr int PS_WARPS = 4, PS_THREADS = PS_WARPS * 32, PS_KEYS = 16, PS_STAGES = 3;
constexpr int PS_LEAST = 4;                              // steps of a warp, at least: a part's own cost

// CTAs that an SM holds at a time, which the kernels are compiled for: as many are launched, one round.  bf16: by their rings beyond 64 channels,
// by registers below; float32: by the registers that its heads take.  Where more were launched than fit, 1.4 GB of keys and values took
// 291 us in place of 210 (bf16, 12 heads over four, 64 channels), 356 in place of 286 (16 heads over one), 314 in place of 230 (float32,
// three heads to a key head).
__host__ __device__ constexpr int step_ctas_per_sm(int dtype, int D, int heads) {
    return dtype == SLOTSCAN_BF16 ? (D > 64 ? 2 : 4) : heads == 1 ? 4 : heads <= 3 ? 3 : 2;
}

// What a request's query sees, in steps of 16 keys from a multiple of 16 on (so that no step but those of pages of 8 meets two pages)
struct Walk {
    int lo, hi, from, steps;
    __device__ __forceinline__ Walk() : lo(0), hi(0), from(0), steps(0) {}
    __device__ __forceinline__ Walk(const PagedArgs& a, int b) {
        const Span s = paged_keys(a, b, a.pos[b]);
        lo = s.lo; hi = s.hi;
        from = lo & ~(PS_KEYS - 1);
        steps = hi > lo ? (hi - from + PS_KEYS - 1) / PS_KEYS : 0;
    }
};
// The scratch: steps before each request (times the pairs of a request: before its first pair), steps of a warp, then the parts, two to a
// warp: of a pair that it takes up at its first step, and of one that it begins and leaves
struct StepPlan {
    long long* before;                                   // B + 1
    long long* per;
    float* parts;
    int heads;                                           // to a part
    static size_t head_bytes(int B) { return ((sizeof(long long) * (B + 2ll) + 15) / 16) * 16; }
    __host__ __device__ StepPlan(void* scratch, int B, int heads_, size_t head) : before((long long*)scratch), per(before + B + 1), parts((float*)((char*)scratch + head)), heads(heads_) {}
    __device__ __forceinline__ float* part(long long warp, bool begun, int g, int D) const { return parts + ((2 * warp + begun) * heads + g) * (D + 2); }
};

// A place in the line of steps
struct Cursor {
    int b, pair, s;                                      // pair: of key head and chunk of its query heads
    Walk w;
    __device__ __forceinline__ void next_request(const PagedArgs& a) {
        do { b++; w = b < a.B ? Walk(a, b) : Walk(); } while (w.steps == 0 && b < a.B);
    }
    __device__ __forceinline__ void next(const PagedArgs& a) {
        if (++s < w.steps) return;
        s = 0;
        if (++pair < a.KV * a.chunks) return;
        pair = 0;
        next_request(a);
    }
};

// This warp's range [x0, x1) of the line and the place where it begins.  By all threads of the CTA; the first CTA writes the plan.
__device__ __forceinline__ void step_range(const PagedArgs& a, const StepPlan& plan, long long& x0, long long& x1, Cursor& c) {
    __shared__ long long s_sum[PS_THREADS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32, pairs = a.KV * a.chunks;
    const int per_thread = (a.B + PS_THREADS - 1) / PS_THREADS, b0 = min(tid * per_thread, a.B), b1 = min(b0 + per_thread, a.B);
    long long mine = 0;
    for (int b = b0; b < b1; b++) mine += Walk(a, b).steps;
    long long v = mine;
#pragma unroll
    for (int off = 1; off < 32; off *= 2) {
        const long long up = __shfl_up_sync(FULL, v, off);
        if (lane >= off) v += up;
    }
    s_sum[tid] = v;
    __syncthreads();
    long long base = 0;
    for (int i = 0; i < warp; i++) base += s_sum[32 * i + 31];
    __syncthreads();
    s_sum[tid] = v + base;                               // up to and with this thread's requests
    __syncthreads();
    const long long total = s_sum[PS_THREADS - 1] * pairs, warps = (long long)gridDim.x * PS_WARPS;
    const long long per = max((total + warps - 1) / warps, (long long)PS_LEAST);
    if (blockIdx.x == 0) {
        long long at = v + base - mine;
        for (int b = b0; b < b1; b++) { plan.before[b] = at * pairs; at += Walk(a, b).steps; }
        if (tid == 0) { plan.before[a.B] = total; *plan.per = per; }
    }
    x0 = ((long long)warp * gridDim.x + blockIdx.x) * per;                         // few steps go to as many SMs as there are
    x1 = min(x0 + per, total);
    if (x0 >= x1) return;
    int t = 0;                                           // the thread whose requests hold x0
#pragma unroll
    for (int i = 0; i < PS_WARPS; i++) t += __popc(__ballot_sync(FULL, s_sum[32 * i + lane] * pairs <= x0));
    c.b = t * per_thread;
    long long at = t > 0 ? s_sum[t - 1] : 0;
    for (c.w = Walk(a, c.b); (at + c.w.steps) * pairs <= x0; c.w = Walk(a, c.b)) { at += c.w.steps; c.b++; }
    const long long in = x0 - at * pairs;
    c.pair = (int)(in / c.w.steps);
    c.s = (int)(in % c.w.steps);
}

// Page ids of 32 steps from `base` on, a lane to a step; of both halves of 8 keys
struct Ids {
    int base, lo, hi;
    __device__ __forceinline__ void fetch(const PagedArgs& a, const Cursor& c) {
        base = c.s;
        const int j = c.w.from + (c.s + (threadIdx.x & 31)) * PS_KEYS;
        lo = j < c.w.hi ? page_of(a, c.b, j) : -1;
        hi = j + 8 < c.w.hi ? page_of(a, c.b, j + 8) : -1;
    }
};

// WIDE: 16 query heads to a pair, else 8
template <int DP, bool WIDE>
__global__ void __launch_bounds__(PS_THREADS, step_ctas_per_sm(SLOTSCAN_BF16, DP, 0)) paged_step_mma_kernel(PagedArgs a, StepPlan plan, const bf16* q, const bf16* k, const bf16* v, bf16* o) {
    constexpr int PIECES = DP / 8, PER_PASS = 32 / PIECES, ROW = DP * 2, TILE = PS_KEYS * ROW, R = WIDE ? 2 : 1, HEADS = 8 * R;
    extern __shared__ float4 smem4[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, group = a.H / a.KV;
    const uint32_t ring = smem_u32(smem4) + warp * PS_STAGES * 2 * TILE;
    long long x0, x1;
    Cursor c;
    step_range(a, plan, x0, x1, c);
    if (x0 >= x1) return;
    Cursor ahead = c;
    Ids ids;
    ids.fetch(a, ahead);
    // A lane fetches piece `piece` of rows sub, sub + PER_PASS, ...  The instructions of a step are what bounds this kernel once its bytes come
    // fast enough (690 of them: 5.5 TB/s), so addresses are sums of what a lane knows beforehand, and a step that is seen whole asks for
    // no mask.
    const int piece = lane % PIECES, sub = lane / PIECES, in_page = (1 << a.shift) - 1;
    const bool live = piece * 8 < a.D;
    const uint32_t put_at = sub * ROW + (((piece & ~7) | ((piece ^ sub) & 7)) << 4);
    const bf16* kl = k + sub * a.ks[1] + (live ? piece * 8 : 0);
    const bf16* vl = v + sub * a.vs[1] + (live ? piece * 8 : 0);
    const long long k_pass = PER_PASS * a.ks[1], v_pass = PER_PASS * a.vs[1];
    long long fetched = x0;
    int put = 0, get = 0;
    auto fetch = [&] {                                   // the next step's 16 keys and values into the ring
        if (fetched < x1) {
            if (ahead.s < ids.base || ahead.s - ids.base >= 32) ids.fetch(a, ahead);
            const int id0 = __shfl_sync(FULL, ids.lo, ahead.s - ids.base), id1 = __shfl_sync(FULL, ids.hi, ahead.s - ids.base);
            const int j0 = ahead.w.from + ahead.s * PS_KEYS, hk = ahead.pair / a.chunks;
            const uint32_t to = ring + put * 2 * TILE;
            const bf16* kr = kl + max(id0, 0) * a.ks[0] + (j0 & in_page) * a.ks[1] + hk * a.ks[2];
            const bf16* vr = vl + max(id0, 0) * a.vs[0] + (j0 & in_page) * a.vs[1] + hk * a.vs[2];
            const bool whole = j0 >= ahead.w.lo && j0 + PS_KEYS <= ahead.w.hi && id0 >= 0 && id1 >= 0;
#pragma unroll
            for (int i = 0; i < PS_KEYS / PER_PASS; i++) {
                if (i * PER_PASS == 8 && a.shift < 4) {  // the second half lies in another page
                    kr = kl + max(id1, 0) * a.ks[0] + hk * a.ks[2];
                    vr = vl + max(id1, 0) * a.vs[0] + hk * a.vs[2];
                }
                bool in = live;
                if (!whole) {
                    const int j = j0 + i * PER_PASS + sub;
                    in = live && j >= ahead.w.lo && j < ahead.w.hi && (i * PER_PASS < 8 ? id0 : id1) >= 0;
                }
                const uint32_t at = to + (put_at ^ ((i * PER_PASS & 7) << 4)) + i * PER_PASS * ROW;
                cp_async16_or0(at, in ? kr : k, in);
                cp_async16_or0(at + TILE, in ? vr : v, in);
                kr += k_pass;
                vr += v_pass;
            }
            put = put + 1 == PS_STAGES ? 0 : put + 1;
            fetched++;
            const int b = ahead.b;
            ahead.next(a);
            if (ahead.b != b) ids.base = BIGI;           // another table
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int s = 0; s < PS_STAGES - 1; s++) fetch();
    const bool capped = a.cap > 0.f;
    const float lin = capped ? a.scale / a.cap * (2.f * LOG2E) : a.scale * LOG2E, cap2 = a.cap * LOG2E;
    const long long me = (long long)warp * gridDim.x + blockIdx.x;
    // of fewer than 9 heads rows 8 to 15 of the products take the lower parts of the weights, whose sums are added at the end
    uint32_t qf[DP / 16][4];
    float slope[R], m[R], l[R], acc[DP / 8][4];
    bool begins = true;                                  // a pair, at this step
    long long begun = x0;                                // the place of its first step here
    int pos = 0;
    for (long long x = x0; x < x1; x++) {
        const int hk = c.pair / a.chunks, g0 = c.pair % a.chunks * HEADS;
        if (begins) {                                    // the queries as A fragments: row = head; heads beyond the group repeat its last
            pos = a.pos[c.b];
            begun = x;
            begins = false;
#pragma unroll
            for (int r = 0; r < R; r++) {
                const int h = hk * group + min(g0 + lane / 4 + 8 * r, group - 1);
                const bf16* qh = q + c.b * a.qs[0] + h * a.qs[1];
                slope[r] = a.slopes != nullptr ? a.slopes[h] * LOG2E : 0.f;
                m[r] = -INFINITY;
                l[r] = 0.f;
#pragma unroll
                for (int kk = 0; kk < DP / 16; kk++)
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const int d = kk * 16 + half * 8 + (lane % 4) * 2;
                        qf[kk][half * 2 + r] = d < a.D ? *reinterpret_cast<const uint32_t*>(qh + d) : 0u;
                        if (!WIDE) qf[kk][half * 2 + 1] = 0u;
                    }
            }
#pragma unroll
            for (int i = 0; i < DP / 8; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][e] = 0.f;
        }
        const int j0 = c.w.from + c.s * PS_KEYS;
        asm volatile("cp.async.wait_group %0;" ::"n"(PS_STAGES - 2) : "memory");
        __syncwarp();
        const uint32_t ks = ring + get * 2 * TILE, vs = ks + TILE;
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
        const bool seen = j0 >= c.w.lo && j0 + PS_KEYS <= c.w.hi;                  // whole
#pragma unroll
        for (int r = 0; r < R; r++) {
            float z[4], top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; i++) z[i] = s[i / 2][2 * r + i % 2] * lin;
            if (capped) {                                // one form for a warp whose scores are all small: 57.3 us of 32 capped requests, both 60.5
                const bool small = fmaxf(fmaxf(fabsf(z[0]), fabsf(z[1])), fmaxf(fabsf(z[2]), fabsf(z[3]))) < CAP_SMALL;
                if (__all_sync(FULL, small)) {
#pragma unroll
                    for (int i = 0; i < 4; i++) z[i] = cap_small(z[i], cap2);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) z[i] = fabsf(z[i]) < CAP_SMALL ? cap_small(z[i], cap2) : cap_large(z[i], cap2);
                }
            }
            if (a.slopes != nullptr) {
                const float dist = (float)(pos - j0 - (lane % 4) * 2);
#pragma unroll
                for (int i = 0; i < 4; i++) z[i] = fmaf(-slope[r], dist - (float)((i / 2) * 8 + i % 2), z[i]);
            }
            if (!seen) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int j = j0 + (i / 2) * 8 + (lane % 4) * 2 + i % 2;
                    z[i] = j >= c.w.lo && j < c.w.hi ? z[i] : -INFINITY;
                }
            }
            top = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
            top = fmaxf(top, __shfl_xor_sync(FULL, top, 1));
            top = fmaxf(top, __shfl_xor_sync(FULL, top, 2));
            top = fmaxf(top, m[r]);
            const float base = top == -INFINITY ? 0.f : top;
            if (__any_sync(FULL, top > m[r])) {
                const float shrink = exp2f(m[r] - base);
                l[r] *= shrink;
#pragma unroll
                for (int i = 0; i < DP / 8; i++)
#pragma unroll
                    for (int e = 0; e < (WIDE ? 2 : 4); e++) acc[i][2 * r + e] *= shrink;
                m[r] = top;
            }
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; i++) { p[i] = exp2f(z[i] - base); l[r] += p[i]; }
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const uint32_t w = pack_bf16(p[2 * t], p[2 * t + 1]);
                ph[2 * t + r] = w;
                (WIDE ? pl : ph)[2 * t + (WIDE ? r : 1)] = pack_bf16(p[2 * t] - __uint_as_float(w << 16), p[2 * t + 1] - __uint_as_float(w & 0xffff0000u));
            }
        }
#pragma unroll
        for (int i = 0; i < DP / 8; i += 2) {
            uint32_t f[4];
            const int key = ((lane / 8) % 2) * 8 + lane % 8, pc = i + lane / 16;
            ldsm4_t(f, vs + key * ROW + (((pc & ~7) | ((pc ^ key) & 7)) << 4));
            mma16(acc[i], ph, f[0], f[1]);
            mma16(acc[i + 1], ph, f[2], f[3]);
            if (WIDE) {
                mma16(acc[i], pl, f[0], f[1]);
                mma16(acc[i + 1], pl, f[2], f[3]);
            }
        }
        __syncwarp();
        get = get + 1 == PS_STAGES ? 0 : get + 1;
        fetch();
        const bool ends = c.s + 1 == c.w.steps;
        if (ends || x + 1 == x1) {
            const bool whole = ends && x - begun + 1 == c.w.steps;
            if (!WIDE) {
#pragma unroll
                for (int i = 0; i < DP / 8; i++) { acc[i][0] += acc[i][2]; acc[i][1] += acc[i][3]; }
            }
#pragma unroll
            for (int r = 0; r < R; r++) {
                float sum = l[r];
                sum += __shfl_xor_sync(FULL, sum, 1);
                sum += __shfl_xor_sync(FULL, sum, 2);
                const int g = lane / 4 + 8 * r, h = hk * group + g0 + g;
                if (g0 + g >= group) continue;
                if (whole) {
                    bf16* to = o + ((size_t)c.b * a.H + h) * a.D;
                    const float inv = 1.f / sum;
#pragma unroll
                    for (int i = 0; i < DP / 8; i++) {
                        const int d = i * 8 + (lane % 4) * 2;
                        if (d < a.D) *reinterpret_cast<uint32_t*>(to + d) = pack_bf16(acc[i][2 * r] * inv, acc[i][2 * r + 1] * inv);
                    }
                } else {
                    float* to = plan.part(me, begun != x0, g, a.D);
#pragma unroll
                    for (int i = 0; i < DP / 8; i++) {
                        const int d = i * 8 + (lane % 4) * 2;
                        if (d < a.D) *reinterpret_cast<float2*>(to + d) = make_float2(acc[i][2 * r], acc[i][2 * r + 1]);
                    }
                    if (lane % 4 == 0) *reinterpret_cast<float2*>(to + a.D) = make_float2(fmaxf(m[r], -FLT_MAX), sum);
                }
            }
            // infinity times the lower part of a weight, which is zero or negative, is not what it is times the weight: such a row anew
#pragma unroll
            for (int r = 0; r < R; r++) {
                float seen_all = 0.f;
#pragma unroll
                for (int i = 0; i < DP / 8; i++) { watch(seen_all, acc[i][2 * r]); watch(seen_all, acc[i][2 * r + 1]); }
                for (unsigned bad = __ballot_sync(FULL, seen_all != seen_all && g0 + lane / 4 + 8 * r < group); bad != 0;) {
                    const int from = __ffs(bad) - 1, g = from / 4 + 8 * r, h = hk * group + g0 + g;
                    bad &= ~(15u << (from & ~3));        // a row's four lanes
                    const int first = max(c.w.lo, c.w.from + (c.s - (int)(x - begun)) * PS_KEYS), end = min(c.w.hi, c.w.from + (c.s + 1) * PS_KEYS);
                    float y[4], xm, xl;
                    careful_row(a, paged_score(a, h), q + c.b * a.qs[0] + h * a.qs[1], k, v, c.b, hk, pos, first, end, y, xm, xl);
                    __syncwarp();
                    float* part = plan.part(me, begun != x0, g, a.D);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int d = lane + 32 * e;
                        if (d >= a.D) continue;
                        if (whole) o[((size_t)c.b * a.H + h) * a.D + d] = __float2bfloat16_rn(y[e] / xl);
                        else part[d] = y[e];
                    }
                    if (!whole && lane == 0) *reinterpret_cast<float2*>(part + a.D) = make_float2(fmaxf(xm, -FLT_MAX), xl);
                }
            }
            begins = true;
        }
        c.next(a);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// LPG lanes to a row, G heads to a pair
template <int LPG, int G>
__global__ void __launch_bounds__(PS_THREADS, step_ctas_per_sm(SLOTSCAN_F32, LPG * 8, G)) paged_step_kernel(PagedArgs a, StepPlan plan, const float* q, const float* k, const float* v, float* o) {
    constexpr int GROUPS = 32 / LPG, U = 4;              // rows of a turn of a group of lanes
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, group = a.H / a.KV, ch = lane % LPG, grp = lane / LPG;
    const bool live = ch * 8 < a.D;
    long long x0, x1;
    Cursor c;
    step_range(a, plan, x0, x1, c);
    if (x0 >= x1) return;
    const long long me = (long long)warp * gridDim.x + blockIdx.x;
    Ids ids;
    ids.fetch(a, c);
    float qr[G][8], acc[G][8], m[G], l[G], slope[G];
    bool begins = true;
    long long begun = x0;
    int pos = 0;
    for (long long x = x0; x < x1; x++) {
        const int hk = c.pair / a.chunks, g0 = c.pair % a.chunks * G;
        if (c.s < ids.base || c.s - ids.base >= 32) ids.fetch(a, c);
        const int id_lo = __shfl_sync(FULL, ids.lo, c.s - ids.base), id_hi = __shfl_sync(FULL, ids.hi, c.s - ids.base);
        if (begins) {
            pos = a.pos[c.b];
            begun = x;
            begins = false;
            const float in = a.cap > 0.f ? a.scale / a.cap : a.scale * LOG2E;
#pragma unroll
            for (int g = 0; g < G; g++) {
                const int h = hk * group + min(g0 + g, group - 1);
#pragma unroll
                for (int i = 0; i < 8; i++) qr[g][i] = acc[g][i] = 0.f;
                if (live) ld8(qr[g], q + c.b * a.qs[0] + h * a.qs[1] + ch * 8);
#pragma unroll
                for (int i = 0; i < 8; i++) qr[g][i] *= in;
                slope[g] = a.slopes != nullptr ? a.slopes[h] * LOG2E : 0.f;
                m[g] = -INFINITY;
                l[g] = 0.f;
            }
        }
        const int j0 = c.w.from + c.s * PS_KEYS;
#pragma unroll
        for (int turn = 0; turn < PS_KEYS; turn += GROUPS * U) {
            float kx[U][8], vx[U][8];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int key = turn + u * GROUPS + grp, j = j0 + key, id = key < 8 ? id_lo : id_hi;
#pragma unroll
                for (int i = 0; i < 8; i++) kx[u][i] = vx[u][i] = 0.f;
                if (j >= c.w.lo && j < c.w.hi && id >= 0 && live) {
                    const long long row = j & ((1 << a.shift) - 1);
                    ld8(kx[u], k + id * a.ks[0] + row * a.ks[1] + hk * a.ks[2] + ch * 8);
                    ld8(vx[u], v + id * a.vs[0] + row * a.vs[1] + hk * a.vs[2] + ch * 8);
                }
            }
#pragma unroll
            for (int g = 0; g < G; g++) {
                float z[U], top = m[g];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int j = j0 + turn + u * GROUPS + grp;
                    float s = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; i++) s = fmaf(qr[g][i], kx[u][i], s);
                    s = group_sum<LPG>(s);
                    if (a.cap > 0.f) s = a.cap * LOG2E * tanhf(s);
                    s = fmaf(-slope[g], (float)(pos - j), s);
                    z[u] = j >= c.w.lo && j < c.w.hi ? s : -INFINITY;
                    top = fmaxf(top, z[u]);
                }
                const float base = top == -INFINITY ? 0.f : top, shrink = exp2f(m[g] - base);
                float p[U], sum = 0.f;
#pragma unroll
                for (int u = 0; u < U; u++) { p[u] = exp2f(z[u] - base); sum += p[u]; }
                m[g] = top;
                l[g] = fmaf(l[g], shrink, sum);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    float t = acc[g][i] * shrink;
#pragma unroll
                    for (int u = 0; u < U; u++) t = fmaf(p[u], vx[u][i], t);
                    acc[g][i] = t;
                }
            }
        }
        const bool ends = c.s + 1 == c.w.steps;
        if (ends || x + 1 == x1) {
            const bool whole = ends && x - begun + 1 == c.w.steps;
#pragma unroll
            for (int g = 0; g < G; g++) {
#pragma unroll
                for (int off = LPG; off < 32; off *= 2) {                          // the groups of lanes, pair by pair
                    const float om = __shfl_xor_sync(FULL, m[g], off), ol = __shfl_xor_sync(FULL, l[g], off);
                    const float top = fmaxf(m[g], om), base = top == -INFINITY ? 0.f : top, f = exp2f(m[g] - base), of = exp2f(om - base);
                    l[g] = l[g] * f + ol * of;
#pragma unroll
                    for (int i = 0; i < 8; i++) acc[g][i] = acc[g][i] * f + __shfl_xor_sync(FULL, acc[g][i], off) * of;
                    m[g] = top;
                }
                if (g0 + g >= group || grp != 0) continue;
                if (whole) {
#pragma unroll
                    for (int i = 0; i < 8; i++) acc[g][i] /= l[g];
                    if (live) st8(o + ((size_t)c.b * a.H + hk * group + g0 + g) * a.D + ch * 8, acc[g]);
                } else {
                    float* to = plan.part(me, begun != x0, g, a.D);
                    if (live) {
#pragma unroll
                        for (int i = 0; i < 8; i += 2) *reinterpret_cast<float2*>(to + ch * 8 + i) = make_float2(acc[g][i], acc[g][i + 1]);
                    }
                    if (ch == 0) *reinterpret_cast<float2*>(to + a.D) = make_float2(fmaxf(m[g], -FLT_MAX), l[g]);
                }
            }
            begins = true;
        }
        const int b = c.b;
        c.next(a);
        if (c.b != b) ids.base = BIGI;
    }
}

// o of a (request, head) whose pair several warps took, joined in their order; zeros where it sees nothing.  W warps to a (request, head):
// one where there are many of them, most of which have nothing to join.  That goes by their number alone, so a long request among many short
// ones is joined slowly: 131,072 tokens beside 63 requests of one token take 196 us, beside 40 of them, with a CTA to a head, 91.
constexpr int PJ_WARPS = 8;
template <typename T, int W>
__global__ void __launch_bounds__(PJ_WARPS * 32) paged_join_kernel(PagedArgs a, StepPlan plan, T* o) {
    __shared__ float s_acc[W > 1 ? W : 1][128], s_m[PJ_WARPS], s_l[PJ_WARPS];
    cudaGridDependencySynchronize();
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, x = blockIdx.x * (PJ_WARPS / W) + warp / W, mine = warp % W;
    if (x >= a.B * a.H) return;                          // W > 1: never, a CTA has one
    const int b = x / a.H, h = x % a.H, group = a.H / a.KV, hk = h / group, g = h % group, pair = hk * a.chunks + g / plan.heads, pairs = a.KV * a.chunks;
    const long long before = plan.before[b], steps = (plan.before[b + 1] - before) / pairs, per = *plan.per;
    T* to = o + (size_t)x * a.D;
    if (steps == 0) {
        for (int d = mine * 32 + lane; d < a.D; d += W * 32) st1(to + d, 0.f);
        return;
    }
    const long long x0 = before + pair * steps, w0 = x0 / per, w1 = (x0 + steps - 1) / per;
    if (w0 == w1) return;                                // one warp had it all
    float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (long long w = w0 + mine; w <= w1; w += W) {
        const float* from = plan.part(w, w * per < x0, g % plan.heads, a.D);
        const float2 ml = *reinterpret_cast<const float2*>(from + a.D);
        const float top = fmaxf(m, ml.x), f = exp2f(m - top), pf = exp2f(ml.x - top);
        l = l * f + ml.y * pf;
#pragma unroll
        for (int c = 0; c < 4; c++) acc[c] = acc[c] * f + (lane + 32 * c < a.D ? from[lane + 32 * c] : 0.f) * pf;
        m = top;
    }
    if constexpr (W == 1) {
#pragma unroll
        for (int c = 0; c < 4; c++)
            if (lane + 32 * c < a.D) st1(to + lane + 32 * c, acc[c] / l);
    } else {
#pragma unroll
        for (int c = 0; c < 4; c++) s_acc[warp][lane + 32 * c] = acc[c];
        if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
        __syncthreads();
        for (int d = threadIdx.x; d < a.D; d += PJ_WARPS * 32) {
            float top = -INFINITY, sum = 0.f, y = 0.f;
            for (int i = 0; i < W; i++) top = fmaxf(top, s_m[i]);
            for (int i = 0; i < W; i++) {
                const float f = exp2f(s_m[i] - top);
                sum = fmaf(s_l[i], f, sum);
                y = fmaf(s_acc[i][d], f, y);
            }
            st1(to + d, y / sum);
        }
    }
}
template <typename T>
static cudaError_t launch_join(const PagedArgs& a, const StepPlan& plan, void* o, cudaStream_t st) {
    const int n = a.B * a.H;
    return n < 148 * 4 ? launch_behind(paged_join_kernel<T, PJ_WARPS>, dim3(n), dim3(PJ_WARPS * 32), st, a, plan, (T*)o)
                       : launch_behind(paged_join_kernel<T, 1>, dim3((n + PJ_WARPS - 1) / PJ_WARPS), dim3(PJ_WARPS * 32), st, a, plan, (T*)o);
}

static int paged_heads(int group, int dtype) { return dtype == SLOTSCAN_BF16 ? (group > 8 ? 16 : 8) : group > 4 ? 8 : group; }
static int step_ctas(const PagedArgs& a, int dtype) {
    const int round = 148 * step_ctas_per_sm(dtype, a.D, paged_heads(a.H / a.KV, dtype));
    const long long steps = (long long)a.B * a.KV * a.chunks * (((long long)a.M << a.shift) / PS_KEYS + 1), want = (steps + PS_LEAST * PS_WARPS - 1) / (PS_LEAST * PS_WARPS);
    return (int)(want < round ? want : round);
}

template <int LPG>
static void launch_step_f32(const PagedArgs& a, const StepPlan& plan, int ctas, const void* q, const void* k, const void* v, void* o, cudaStream_t st) {
    auto go = [&](auto kern) { kern<<<ctas, PS_THREADS, 0, st>>>(a, plan, (const float*)q, (const float*)k, (const float*)v, (float*)o); };
    switch (paged_heads(a.H / a.KV, SLOTSCAN_F32)) {
        case 1: go(paged_step_kernel<LPG, 1>); break;
        case 2: go(paged_step_kernel<LPG, 2>); break;
        case 3: go(paged_step_kernel<LPG, 3>); break;
        case 4: go(paged_step_kernel<LPG, 4>); break;
        default: go(paged_step_kernel<LPG, 8>); break;
    }
}
template <int DP>
static cudaError_t launch_step_bf16(const PagedArgs& a, const StepPlan& plan, int ctas, const void* q, const void* k, const void* v, void* o, cudaStream_t st) {
    const size_t sm = (size_t)PS_WARPS * PS_STAGES * 2 * PS_KEYS * DP * 2;
    auto kern = paged_heads(a.H / a.KV, SLOTSCAN_BF16) == 16 ? paged_step_mma_kernel<DP, true> : paged_step_mma_kernel<DP, false>;
    const cudaError_t e = opt_in_smem(kern, sm);
    if (e != cudaSuccess) return e;
    kern<<<ctas, PS_THREADS, sm, st>>>(a, plan, (const bf16*)q, (const bf16*)k, (const bf16*)v, (bf16*)o);
    return cudaSuccess;
}

}  // namespace slotscan

using namespace slotscan;

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

extern "C" int slotscan_paged_check(const slotscan_paged_params* p) {
    if (p == nullptr) return SLOTSCAN_E_NULL;
    if (p->dtype != SLOTSCAN_F32 && p->dtype != SLOTSCAN_BF16) return SLOTSCAN_E_DTYPE;
    // rows times heads, rounded up to whole CTAs of the join, stay an int
    if (p->N < 0 || p->N > (1 << 28) || p->B < 0 || p->B > (1 << 24) || p->H < 1 || p->H > 65535 || p->KV < 1 || p->H % p->KV || (int64_t)p->N * p->H > 0x7ffffff8 ||
        p->D < 8 || p->D > 128 || p->D % 8 || p->pages < 1 || p->M < 1 || p->page < 8 || p->page > 1024 || (p->page & (p->page - 1)) ||
        (int64_t)p->M * p->page > (1 << 29) || p->table_stride < p->M)
        return SLOTSCAN_E_SHAPE;
    if (p->window < 0 || !(p->cap >= 0.f) || !(p->cap < INFINITY) || !(p->scale > 0.f) || !(p->scale < INFINITY)) return SLOTSCAN_E_MODE;
    const int e = p->dtype == SLOTSCAN_BF16 ? 2 : 4;
    for (int i = 0; i < 3; i++)
        if ((i < 2 && p->q_stride[i] * e % 16) || p->k_stride[i] * e % 16 || p->v_stride[i] * e % 16) return SLOTSCAN_E_ALIGN;
    return SLOTSCAN_OK;
}

static PagedArgs step_args(const slotscan_paged_params& p, const int32_t* tables, const int32_t* pos, const int32_t* start, const float* slopes, int& heads) {
    PagedArgs a = paged_args(p, tables, nullptr, pos, start, slopes);
    const int group = p.H / p.KV, most = paged_heads(group, p.dtype);
    a.chunks = (group + most - 1) / most;
    heads = group < most ? group : most;
    return a;
}

extern "C" size_t slotscan_paged_step_scratch_bytes(const slotscan_paged_params* p) {
    if (slotscan_paged_check(p) != SLOTSCAN_OK || p->N != p->B) return 0;
    int heads;
    const PagedArgs a = step_args(*p, nullptr, nullptr, nullptr, nullptr, heads);
    return StepPlan::head_bytes(a.B) + sizeof(float) * (size_t)step_ctas(a, p->dtype) * PS_WARPS * 2 * heads * (a.D + 2);
}

extern "C" int slotscan_paged_step(const slotscan_paged_params* p, const void* q, const void* kp, const void* vp, const int32_t* tables, const int32_t* pos,
                                   const int32_t* start, const float* slopes, void* o, void* scratch, size_t scratch_bytes, void* stream) {
    const int rc = slotscan_paged_check(p);
    if (rc != SLOTSCAN_OK) return rc;
    if (p->N != p->B) return SLOTSCAN_E_SHAPE;
    if (p->B == 0) return SLOTSCAN_OK;
    if (!q || !kp || !vp || !tables || !pos || !o) return SLOTSCAN_E_NULL;
    if (!aligned16(q) || !aligned16(kp) || !aligned16(vp) || !aligned16(o) || !aligned16(scratch)) return SLOTSCAN_E_ALIGN;
    if (scratch == nullptr || scratch_bytes < slotscan_paged_step_scratch_bytes(p)) return SLOTSCAN_E_NULL;
    int heads;
    const PagedArgs a = step_args(*p, tables, pos, start, slopes, heads);
    const StepPlan plan(scratch, a.B, heads, StepPlan::head_bytes(a.B));
    const int ctas = step_ctas(a, p->dtype);
    cudaStream_t st = (cudaStream_t)stream;
    if (p->dtype == SLOTSCAN_BF16) {
        const cudaError_t e = p->D <= 64 ? launch_step_bf16<64>(a, plan, ctas, q, kp, vp, o, st) : launch_step_bf16<128>(a, plan, ctas, q, kp, vp, o, st);
        if (e != cudaSuccess) return (int)e;
        return (int)launch_join<bf16>(a, plan, o, st);
    } else {
        if (p->D <= 64) launch_step_f32<8>(a, plan, ctas, q, kp, vp, o, st);
        else launch_step_f32<16>(a, plan, ctas, q, kp, vp, o, st);
        return (int)launch_join<float>(a, plan, o, st);
    }
}
