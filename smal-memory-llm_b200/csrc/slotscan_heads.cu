// Norms of queries and keys per head with the position rotation in the same pass, forward, backward, into ring caches and into pages.
//
// Per row x of D channels:  r = (mean x^2 + eps)^(-1/2),  y = x r w,  and the pairs (i, i + R/2) turned by the position's angle.
// Backward, with g the upstream gradient turned back by the same angle:  dw += g x r,  h = g w,
//     dx = r (h - x r mean(h x r))
// A row's two sums are its only reductions, so each element is read once and written once: two rows of traffic forward, three
// backward, and some ten operations an element.  Bandwidth bounds it.
//
// Layout: a group of LPG lanes (a power of two, 8 channels to a lane) takes a token and walks over a slice of its heads, queries first,
// with the token's cosines and sines in registers: the table of a position has the bytes of two bf16 rows, and is read once for all its
// heads.  A lane owns both sides of four pairs, so that a turn is its own.  Rows come ahead through shared memory, which takes no
// registers: 4 in flight to a group and four CTAs to an SM, backward 5 rows with their gradients and two CTAs.  64 x 1,024 tokens of
// 6 + 6 heads of 128, bf16: 76 us (5.3 TB/s), backward 120 us (5.0 TB/s).  Before: 101 and 150 us with rows in registers and a pair's
// sides 8 lanes apart; 80 and 129 with the ring alone.  Three, five or six CTAs: 78, 85, 84 us; backward three CTAs 129, four 204.
// Into pages: 6,456 packed tokens of 12 + 4 + 4 heads of 128 in 19 us, 49,000 in 100 (5.0 TB/s), four CTAs to an SM (three took as long).
// Now bound by the issue of instructions (84 % of the slots, backward 76 %); paired multiply-adds took 81 and 126: their operands
// have to be moved into pairs.  float32 is as fast either way (8 x 4,096 tokens of 12 + 4 heads of 64: 44 + 71 us, 6.1 TB/s).
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
// slots of a thread's ring, one more than the rows in flight
template <typename T> constexpr int NR_FWD_SLOTS = 5;
template <typename T> constexpr int NR_BWD_SLOTS = sizeof(T) == 2 ? 6 : 3;
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
// Where keys and values go: rows of their own, ring caches (row = position mod L), or slots in the pages of a pool
enum Dest { OUT, RING, PAGES };
struct AppendArgs {
    int L;                                               // of a ring
    int shift;                                           // of pages: log2 of their tokens
    long long slots;                                     // of pages: how many there are
    const int32_t* slot;                                 // of pages: of each token
    long long vs[3], kcs[3], vcs[3];
};

// The two pieces of four adjacent channels that a lane owns.  In the rotated part they are the two sides of four pairs, so that a turn
// needs no other lane; beyond it they lie side by side.
struct Pieces {
    int at[2];
    __device__ __forceinline__ Pieces(int c, int R) {
        const bool rot = c * 8 < R;
        at[0] = rot ? 4 * c : 8 * c;
        at[1] = rot ? R / 2 + 4 * c : 8 * c + 4;
    }
};
__device__ __forceinline__ void ld4x(float* x, const float* p) { const float4 v = ld4(p); x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; }
__device__ __forceinline__ void ld4x(float* x, const bf16* p) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xffff0000u); x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xffff0000u);
}
__device__ __forceinline__ void st4x(float* p, const float* x) { *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]); }
__device__ __forceinline__ void st4x(bf16* p, const float* x) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
template <typename T>
__device__ __forceinline__ void ld_pieces(float (&x)[8], const T* row, const Pieces& pc) { ld4x(x, row + pc.at[0]); ld4x(x + 4, row + pc.at[1]); }
template <typename T>
__device__ __forceinline__ void st_pieces(T* row, const float (&x)[8], const Pieces& pc) { st4x(row + pc.at[0], x); st4x(row + pc.at[1], x + 4); }

// Rows fetched ahead into S slots of shared memory, X of them to a slot, 16-byte pieces in their own order: a group's lanes read
// each other's.  A slot is fetched again only after the warp has met at the next one's arrival.
template <typename T, int LPG, int X, int S>
struct Ahead {
    static constexpr int P = sizeof(T) / 2, BYTES = S * X * P * NR_THREADS * 16;
    uint4* rows;                                         // the group's rows of the first slot
    int put, get;
    __device__ __forceinline__ explicit Ahead(uint4* ring) : rows(ring + threadIdx.x / LPG * LPG * P), put(0), get(0) {}
    __device__ __forceinline__ uint4* row(int slot, int x) const { return rows + (slot * X + x) * P * NR_THREADS; }
    // piece c of a row; zeros unless `in`; `from` (the row) is an address of the tensor all the same
    __device__ __forceinline__ void fetch(int x, const T* from, int c, bool in, int D) {
#pragma unroll
        for (int i = 0; i < P; i++) {
            const bool piece = in && (c + i * LPG) * 16 < D * (int)sizeof(T);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(row(put, x) + c + i * LPG)),
                         "l"(reinterpret_cast<const uint4*>(from) + (piece ? c + i * LPG : 0)), "r"(piece ? 16 : 0)
                         : "memory");
        }
    }
    __device__ __forceinline__ void fetched() {          // the slot is complete
        asm volatile("cp.async.commit_group;" ::: "memory");
        put = put + 1 == S ? 0 : put + 1;
    }
    __device__ __forceinline__ void arrived() {          // of S - 1 fetched, the oldest
        asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
        __syncwarp();
    }
    __device__ __forceinline__ void rest() {             // before the ring serves something else
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
    __device__ __forceinline__ void read(int x, float (&y)[8], const Pieces& pc) const { ld_pieces(y, reinterpret_cast<const T*>(row(get, x)), pc); }
    __device__ __forceinline__ void used() { get = get + 1 == S ? 0 : get + 1; }
};

// cosines and sines of this lane's four pairs; NaN where the position lies outside the table
__device__ __forceinline__ void load_turn(const NormArgs& a, long long at, int c, float (&cs)[4], float (&sn)[4]) {
    if (c * 8 >= a.R) return;
    const bool in = at >= 0 && at < a.table_len;
    const float* t = a.table + ((size_t)(in ? at : 0) * (a.R / 2) + c * 4) * 2;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const float4 u = ld4(t + 4 * i);
        cs[2 * i] = u.x; sn[2 * i] = u.y; cs[2 * i + 1] = u.z; sn[2 * i + 1] = u.w;
    }
    if (!in) {
#pragma unroll
        for (int i = 0; i < 4; i++) cs[i] = sn[i] = __int_as_float(0x7fffffff);
    }
}

// y turned by the angle (DIR 1) or back (DIR -1)
template <int DIR>
__device__ __forceinline__ void turn(float (&y)[8], const float (&cs)[4], const float (&sn)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float a = y[i], b = y[4 + i], s = DIR > 0 ? sn[i] : -sn[i];
        y[i] = fmaf(a, cs[i], -b * s);
        y[4 + i] = fmaf(b, cs[i], a * s);
    }
}

// T: bf16 or float
template <typename T, int LPG, Dest DEST>
__global__ void __launch_bounds__(NR_THREADS, DEST == RING ? 3 : NR_FWD_CTAS) norm_rope_kernel(NormArgs a, AppendArgs ap, const T* q, const T* k, const T* v, T* qo, T* ko,
                                                               T* kc, T* vc) {
    constexpr bool CACHE = DEST != OUT;
    constexpr int SLOTS = NR_FWD_SLOTS<T>;
    __shared__ uint4 ring[Ahead<T, LPG, 1, SLOTS>::BYTES / 16];
    Ahead<T, LPG, 1, SLOTS> rows(ring);
    const int c = threadIdx.x % LPG;
    const unsigned unit = blockIdx.x * (NR_THREADS / LPG) + threadIdx.x / LPG, tok = unit / a.slices;            // fewer than 2^31
    const int h0 = (int)(unit % a.slices) * a.per_slice, all = a.H + a.KV + (CACHE ? a.KV : 0);
    const bool token = tok < a.tokens, live = token && c * 8 < a.D;                // a lane without channels still fetches for the others
    const unsigned b = token ? tok / a.T : 0, t = token ? tok % a.T : 0;
    const long long at = DEST == RING ? (long long)a.pos[b] + t : a.pos != nullptr ? (long long)a.pos[token ? tok : 0] : t;
    const T* qt = q + b * a.qs[0] + t * a.qs[1];         // of the token
    const T* kt = k + b * a.ks[0] + t * a.ks[1];
    const T* vt = CACHE ? v + b * ap.vs[0] + t * ap.vs[1] : nullptr;
    // a row's 16-byte pieces are shared out over the lanes in order: in float32 lane c also takes piece LPG + c
    auto fetch = [&](int u) {
        const int h = h0 + u;
        const T* from = h < a.H ? qt + h * a.qs[2] : !CACHE || h < a.H + a.KV ? kt + (h - a.H) * a.ks[2] : vt + (h - a.H - a.KV) * ap.vs[2];
        const bool in = token && u < a.per_slice && h < all;
        rows.fetch(0, in ? from : q, c, in, a.D);
        rows.fetched();
    };
#pragma unroll
    for (int u = 0; u < SLOTS - 1; u++) fetch(u);
    const Pieces pc(c, a.R);
    T* qot = qo + (size_t)tok * a.H * a.D;
    const bool rot = c * 8 < a.R;
    float cs[4], sn[4], w[8];
    load_turn(a, at, c, cs, sn);
    long long outer = b, row = 0;                        // sequence and row of a ring, page and row within it
    bool stored = at >= 0;
    if constexpr (DEST == RING) row = stored ? (unsigned)at % (unsigned)ap.L : 0;
    if constexpr (DEST == PAGES) {
        const long long slot = token ? ap.slot[tok] : -1;
        stored = stored && slot >= 0 && slot < ap.slots;
        outer = stored ? slot >> ap.shift : 0;
        row = stored ? slot & ((1 << ap.shift) - 1) : 0;
    }
    T* kot = CACHE ? kc + outer * ap.kcs[0] + row * ap.kcs[1] : ko + (size_t)tok * a.KV * a.D;
    T* vot = CACHE ? vc + outer * ap.vcs[0] + row * ap.vcs[1] : nullptr;
    const long long kos = CACHE ? ap.kcs[2] : a.D;
    const float inv_d = 1.f / a.D;
    for (int u = 0; u < a.per_slice; u++) {
        const int h = h0 + u;
        const bool is_v = CACHE && h >= a.H + a.KV, is_q = h < a.H;
        rows.arrived();
        fetch(u + SLOTS - 1);
        if (h == a.H || u == 0) {                        // the queries' weights, then the keys'
            const float* from = is_q ? a.qw : a.kw;
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] = 1.f;
            if (live && from != nullptr) ld_pieces(w, from, pc);
        }
        float ss = 0.f, x[8], y[8];
        rows.read(0, x, pc);
        rows.used();
#pragma unroll
        for (int i = 0; i < 8; i++) ss = fmaf(x[i], x[i], ss);
        const float r = rsqrtf(fmaf(group_sum<LPG>(ss), inv_d, a.eps));
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = x[i] * r * w[i];
        if (rot) turn<1>(y, cs, sn);
        if (!live || h >= all) continue;
        if (DEST == PAGES && at < 0) {                   // a row of no token
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = 0.f;
        }
        if (is_q) st_pieces(qot + h * a.D, y, pc);
        else if (!CACHE || stored) {
            if (!is_v) st_pieces(kot + (h - a.H) * kos, y, pc);
            else st_pieces(vot + (h - a.H - a.KV) * ap.vcs[2], x, pc);
        }
    }
    rows.rest();
}

// grid-stride over (token, slice of heads); part: (CTAs, 2, D) sums of the weights' gradients, or NULL
template <typename T, int LPG>
__global__ void __launch_bounds__(NR_THREADS, NR_BWD_CTAS) norm_rope_bwd_kernel(NormArgs a, const T* q, const T* k, const T* gq, const T* gk, T* dq, T* dk,
                                                                   float* part) {
    constexpr int GROUPS = NR_THREADS / LPG, SLOTS = NR_BWD_SLOTS<T>;              // a slot: a row and its gradient
    __shared__ uint4 ring[Ahead<T, LPG, 2, SLOTS>::BYTES / 16];
    float(*s_part)[LPG * 8] = reinterpret_cast<float(*)[LPG * 8]>(ring);           // after the last row
    const int c = threadIdx.x % LPG, grp = threadIdx.x / LPG;
    const Pieces pc(c, a.R);
    const bool rot = c * 8 < a.R;
    const float inv_d = 1.f / a.D;
    float w[8], acc[2][8];
#pragma unroll
    for (int i = 0; i < 8; i++) acc[0][i] = acc[1][i] = 0.f;
    const unsigned units = (unsigned)a.tokens * a.slices, first = blockIdx.x * GROUPS + grp, stride = gridDim.x * GROUPS;      // fewer than 2^31
    const int rounds = (int)((units - blockIdx.x * GROUPS + stride - 1) / stride); // the same in all groups of the CTA
    struct Place { unsigned tok, b, t; int h0; bool live; };
    auto place = [&](int round) {
        const unsigned unit = first + round * stride, tok = unit / a.slices;
        const bool live = round < rounds && unit < units;
        return Place{tok, live ? tok / a.T : 0, live ? tok % a.T : 0, (int)(unit % a.slices) * a.per_slice, live};
    };
    Ahead<T, LPG, 2, SLOTS> rows(ring);
    Place pf = place(0);                                 // of the rows to fetch next
    const T *qt, *kt, *gqt, *gkt;
    auto bases = [&] {
        qt = q + pf.b * a.qs[0] + pf.t * a.qs[1];
        kt = k + pf.b * a.ks[0] + pf.t * a.ks[1];
        gqt = gq + (size_t)pf.tok * a.H * a.D;
        gkt = gk + (size_t)pf.tok * a.KV * a.D;
    };
    bases();
    int f_round = 0, f_u = 0;
    auto fetch = [&] {
        const int h = pf.h0 + f_u;
        const bool in = pf.live && h < a.H + a.KV;
        rows.fetch(0, !in ? q : h < a.H ? qt + h * a.qs[2] : kt + (h - a.H) * a.ks[2], c, in, a.D);
        rows.fetch(1, !in ? gq : h < a.H ? gqt + h * a.D : gkt + (h - a.H) * a.D, c, in, a.D);
        rows.fetched();
        if (++f_u == a.per_slice) { f_u = 0; pf = place(++f_round); bases(); }
    };
#pragma unroll
    for (int u = 0; u < SLOTS - 1; u++) fetch();
    for (int round = 0; round < rounds; round++) {
        const Place p = place(round);
        const bool live = p.live && c * 8 < a.D;
        const size_t qo = (size_t)p.tok * a.H * a.D, ko = (size_t)p.tok * a.KV * a.D;
        float cs[4], sn[4];
        load_turn(a, a.pos != nullptr ? (long long)a.pos[p.live ? p.tok : 0] : p.t, c, cs, sn);
        for (int u = 0; u < a.per_slice; u++) {
            const int h = p.h0 + u;
            const bool is_q = h < a.H;
            rows.arrived();
            fetch();
            if (h == a.H || u == 0) {                    // the queries' weights, then the keys'
                const float* from = is_q ? a.qw : a.kw;
#pragma unroll
                for (int i = 0; i < 8; i++) w[i] = 1.f;
                if (c * 8 < a.D && from != nullptr) ld_pieces(w, from, pc);
            }
            float x[8], g[8], s1 = 0.f, s2 = 0.f;
            rows.read(0, x, pc);
            rows.read(1, g, pc);
            rows.used();
            if (rot) turn<-1>(g, cs, sn);
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
            if (is_q) st_pieces(dq + qo + h * a.D, dx, pc);
            else st_pieces(dk + ko + (h - a.H) * a.D, dx, pc);
        }
    }
    rows.rest();
    if (part == nullptr) return;
    for (int n = 0; n < 2; n++) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; i++) s_part[grp][pc.at[i / 4] + i % 4] = n ? acc[1][i] : acc[0][i];
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
    // Fewer heads to a group while the groups would leave SMs idle; whole tokens beyond, whose table is then read once.  Aimed at 148 x 6
    // CTAs: two rounds of the append's three to an SM, one and a half of the forward's four, three of the backward's two.  Heads are
    // rounded up and the last slice may be short, so that is not met exactly: 8 x 512 tokens of 12 + 4 + 4 heads of 128 go in slices of
    // 6 + 6 + 6 + 2, 1,024 CTAs, 2.3 rounds (15.4 us)
    const long long groups = 148ll * 6 * NR_THREADS / lanes_of(p.D), want = (a.tokens * heads + groups - 1) / groups;
    a.per_slice = (int)(want < 1 ? 1 : want > heads ? heads : want);
    a.slices = (heads + a.per_slice - 1) / a.per_slice;
    return a;
}
// Slices of a token's heads for packed tokens, whose number is any: the ones of least time, which is rounds of four CTAs to an SM, each of its
// rows and of some six more until the first are there.  6,456 tokens of 12 + 4 + 4 heads: whole tokens, two thirds of a round, 19 us; two
// slices are 1.36 rounds, 23 us
static void slice_for_rounds(NormArgs& a, int heads, int lanes) {
    const long long round = 148ll * NR_FWD_CTAS * (NR_THREADS / lanes);
    long long best = 0;
    for (int s = 1; s <= heads && s <= 64; s++) {
        const int rows = (heads + s - 1) / s, slices = (heads + rows - 1) / rows;
        const long long time = (a.tokens * slices + round - 1) / round * (rows + 6);
        if (s == 1 || time < best) { best = time; a.per_slice = rows; a.slices = slices; }
    }
}
static int bwd_ctas(const NormArgs& a) {
    const long long want = (a.tokens * a.slices + NR_THREADS / lanes_of(a.D) - 1) / (NR_THREADS / lanes_of(a.D));
    return (int)(want < NR_MAX_CTAS ? want : NR_MAX_CTAS);
}

template <typename T, Dest DEST>
static cudaError_t launch_norm(const NormArgs& a, const AppendArgs& ap, const void* q, const void* k, const void* v, void* qo, void* ko, void* kc,
                               void* vc, cudaStream_t st) {
    const int groups = NR_THREADS / lanes_of(a.D);
    const unsigned grid = (unsigned)((a.tokens * a.slices + groups - 1) / groups);
    auto go = [&](auto kern) { kern<<<grid, NR_THREADS, 0, st>>>(a, ap, (const T*)q, (const T*)k, (const T*)v, (T*)qo, (T*)ko, (T*)kc, (T*)vc); };
    if (lanes_of(a.D) == 8) go(norm_rope_kernel<T, 8, DEST>);
    else if (lanes_of(a.D) == 16) go(norm_rope_kernel<T, 16, DEST>);
    else go(norm_rope_kernel<T, 32, DEST>);
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
    return (int)(p->dtype == SLOTSCAN_BF16 ? launch_norm<bf16, OUT>(a, none, q, k, nullptr, qo, ko, nullptr, nullptr, (cudaStream_t)stream)
                                           : launch_norm<float, OUT>(a, none, q, k, nullptr, qo, ko, nullptr, nullptr, (cudaStream_t)stream));
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
    AppendArgs ap = {};
    ap.L = p->L;
    for (int i = 0; i < 3; i++) { ap.vs[i] = p->v_stride[i]; ap.kcs[i] = p->kc_stride[i]; ap.vcs[i] = p->vc_stride[i]; }
    return (int)(n.dtype == SLOTSCAN_BF16 ? launch_norm<bf16, RING>(a, ap, q, k, v, qo, nullptr, kc, vc, (cudaStream_t)stream)
                                          : launch_norm<float, RING>(a, ap, q, k, v, qo, nullptr, kc, vc, (cudaStream_t)stream));
}

extern "C" int slotscan_norm_rope_pages(const slotscan_page_append_params* p, const void* q, const void* k, const void* v, const float* table,
                                        const int32_t* slots, const int32_t* pos, const float* qw, const float* kw, void* qo, void* kp, void* vp,
                                        void* stream) {
    const int rc = slotscan_norm_rope_check(p == nullptr ? nullptr : &p->base);
    if (rc != SLOTSCAN_OK) return rc;
    const slotscan_norm_params& n = p->base;
    if (n.B != 1 || p->pages < 1 || p->page < 8 || p->page > 1024 || (p->page & (p->page - 1)) || (int64_t)p->pages * p->page > BIGI) return SLOTSCAN_E_SHAPE;
    if (!strides16(p->v_stride, 3, n.dtype) || !strides16(p->kp_stride, 3, n.dtype) || !strides16(p->vp_stride, 3, n.dtype)) return SLOTSCAN_E_ALIGN;
    if (n.T == 0) return SLOTSCAN_OK;
    if (!q || !k || !v || !slots || !pos || !qo || !kp || !vp || (n.R && !table)) return SLOTSCAN_E_NULL;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(qo) || !aligned16(kp) || !aligned16(vp) || !aligned16(table) || !aligned16(qw) ||
        !aligned16(kw))
        return SLOTSCAN_E_ALIGN;
    NormArgs a = norm_args(n, table, pos, qw, kw, n.H + 2 * n.KV);
    slice_for_rounds(a, n.H + 2 * n.KV, lanes_of(n.D));
    AppendArgs ap = {};
    while ((1 << ap.shift) < p->page) ap.shift++;
    ap.slots = (long long)p->pages << ap.shift;
    ap.slot = slots;
    for (int i = 0; i < 3; i++) { ap.vs[i] = p->v_stride[i]; ap.kcs[i] = p->kp_stride[i]; ap.vcs[i] = p->vp_stride[i]; }
    return (int)(n.dtype == SLOTSCAN_BF16 ? launch_norm<bf16, PAGES>(a, ap, q, k, v, qo, nullptr, kp, vp, (cudaStream_t)stream)
                                          : launch_norm<float, PAGES>(a, ap, q, k, v, qo, nullptr, kp, vp, (cudaStream_t)stream));
}
