// Attention over tokens with a narrow causal window, bf16: the local window that the model reads beside its memory.
//
// A row sees a few keys around its own place, so nothing is worth handing from warp to warp and bytes bound: the products are
// m16n8k16, a warp's own from scores to output.  A warp takes 16 queries and the NB blocks of 16 keys that their windows touch; the whole
// softmax of a row is in its registers at once.  (On the tcgen05 kernels a tile of 128 rows costs 26,000 cycles of filling and handing
// over whatever it sees: 163 us for 64 x 1,024 tokens of six heads of 128, window 16, against 69 here; backward 567 against 167.)
//
// Forward: a CTA takes 64 queries and the 64 + 16 (NB - 1) keys before and among them.
// Backward: a CTA owns 64 keys and the 64 queries at their places.  It also takes the queries behind that see its keys, and the keys that
// those see, forms the softmax of each row anew and sums delta = sum p dp of the row itself, so nothing but q, k, v and do is
// read (the halo comes from the cache) and nothing is kept by the forward.  dq is done by the warp of its rows; p and ds go to
// shared memory, where the warp of 16 keys gathers dk and dv from the NB blocks of queries that see them: no atomics.
// p and ds are rounded once to bf16 for their products, as the operands' type asks: dq and dk are then off by about the root of two times
// what their own rounding costs.
#include "slotscan_attn.cuh"
#include "slotscan_launch.h"
#include "slotscan_tensor.cuh"

namespace slotscan {

static __device__ int g_narrow_status = 0;               // a bounded wait gave up (slotscan_device_status)

constexpr int NA_ROWS = 64;                              // queries (forward) or keys (backward) of a CTA

__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
}
// address of the 16-byte piece `piece` of row `row` of a tile of `rows` rows: sub-tiles of 64 columns, swizzled as the copies write them
__device__ __forceinline__ uint32_t piece_at(uint32_t tile, int rows, int row, int piece) {
    return tile + (piece / 8) * rows * 128 + swizzled(row, piece % 8);
}
// The fragments of 16 rows x 16 columns (columns 16 c ..) of a tile, by the lane's place
__device__ __forceinline__ void rows_as_a(uint32_t (&f)[4], uint32_t tile, int rows, int row0, int c, int lane) {        // rows x columns
    ldsm(f, piece_at(tile, rows, row0 + lane % 16, 2 * c + lane / 16));
}
__device__ __forceinline__ void rows_as_b(uint32_t (&f)[4], uint32_t tile, int rows, int row0, int c, int lane) {        // n = rows, k = columns: f[0..1], f[2..3]
    ldsm(f, piece_at(tile, rows, row0 + (lane / 16) * 8 + lane % 8, 2 * c + (lane / 8) % 2));
}
__device__ __forceinline__ void rows_as_bt(uint32_t (&f)[4], uint32_t tile, int rows, int row0, int c, int lane) {       // k = rows, n = columns
    ldsm_t(f, piece_at(tile, rows, row0 + ((lane / 8) % 2) * 8 + lane % 8, 2 * c + lane / 16));
}
// rows row0 .. of 16 x DP results of a warp into a tile
template <int DP>
__device__ __forceinline__ void put_rows(uint32_t tile, int rows, int row0, int c, int lane, uint32_t lo, uint32_t hi) {  // n-tile c of 8 columns
    const uint32_t at = (lane % 4) * 4;
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(piece_at(tile, rows, row0 + lane / 4, c) + at), "r"(lo) : "memory");
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(piece_at(tile, rows, row0 + lane / 4 + 8, c) + at), "r"(hi) : "memory");
}

// a row's channels lane + 32 c
__device__ __forceinline__ void put_lane_row(bf16* row, const float (&x)[4], int D) {
#pragma unroll
    for (int c = 0; c < 4; c++) { const int d = (threadIdx.x & 31) + 32 * c; if (d < D) row[d] = __float2bfloat16_rn(x[c]); }
}

// 16 x 16 NB scores of a warp's queries (rows `row0` of the tile Q, keys from `key0` of the tile K)
template <int DP, int NB>
__device__ __forceinline__ void band(float (&s)[2 * NB][4], uint32_t Q, int q_rows, int row0, uint32_t K, int k_rows, int key0, int lane) {
#pragma unroll
    for (int t = 0; t < 2 * NB; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[t][i] = 0.f;
#pragma unroll
    for (int c = 0; c < DP / 16; c++) {
        uint32_t x[4];
        rows_as_a(x, Q, q_rows, row0, c, lane);
#pragma unroll
        for (int n = 0; n < NB; n++) {
            uint32_t y[4];
            rows_as_b(y, K, k_rows, key0 + 16 * n, c, lane);
            mma(s[2 * n], x, y[0], y[1]);
            mma(s[2 * n + 1], x, y[2], y[3]);
        }
    }
}

// Scores to unnormalised weights exp2(z - max), in place, and the sum's reciprocal of the lane's two rows; F: also 1 - tanh^2 of each.
// key0: position of the first key; lse: the two rows' logarithms as slotscan_attn_fwd gives them, or NULL
template <int NB, bool F>
__device__ __forceinline__ void band_softmax(float (&s)[2 * NB][4], float (&f)[F ? 2 * NB : 1][4], float (&inv)[2], const Score& sc, const Span (&sp)[2],
                                             const int (&at)[2], int key0, int lane, float* lse = nullptr) {
    const bool capped = sc.cap_in != 0.f;
#pragma unroll
    for (int r = 0; r < 2; r++) {
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2 * NB; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int j = key0 + t * 8 + (lane % 4) * 2 + e;
                float z = s[t][2 * r + e];
                if constexpr (F) f[t][2 * r + e] = 1.f;
                if (capped) {                            // tanh x = 1 - 2 q, 1 - tanh^2 = 4 q (1 - q),  q = 1 / (e^2x + 1)
                    const float q = rcp_fast(exp2_fast(z * (2.f * LOG2E * sc.cap_in)) + 1.f);
                    z = fmaf(-2.f * sc.cap_out, q, sc.cap_out);
                    if constexpr (F) f[t][2 * r + e] = 4.f * fmaf(-q, q, q);
                } else z *= sc.lin;
                z = fmaf(-sc.slope, (float)abs(at[r] - j), z);
                z = j >= sp[r].lo && j < sp[r].hi ? z : -INFINITY;
                s[t][2 * r + e] = z;
                top = fmaxf(top, z);
            }
        top = fmaxf(top, __shfl_xor_sync(FULL, top, 1));
        top = fmaxf(top, __shfl_xor_sync(FULL, top, 2));
        const float base = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < 2 * NB; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float p = exp2_fast(s[t][2 * r + e] - base);
                s[t][2 * r + e] = p;
                sum += p;
            }
        sum += __shfl_xor_sync(FULL, sum, 1);
        sum += __shfl_xor_sync(FULL, sum, 2);
        const int n = sp[r].hi - sp[r].lo;
        inv[r] = n > 0 ? 1.f / sum : 0.f;
        if (lse != nullptr) lse[r] = n <= 0 ? -INFINITY : n == 1 ? INFINITY : base + log2f(sum);
    }
}

struct NarrowMaps { CUtensorMap q, k, v, o; };
struct NarrowBwdMaps { CUtensorMap q, k, v, d, dq, dk, dv; };

// a wait that all threads of a CTA stand at: false in all of them when it gave up in one
__device__ __forceinline__ bool all_arrived(uint64_t* bar, unsigned parity) {
    const bool ok = wait_soon(bar, parity);
    return __syncthreads_and(ok) != 0;
}
__device__ __forceinline__ void give_up() {              // report, and give the copies in flight time to land
    if (threadIdx.x == 0) atomicExch(&g_narrow_status, 1);
    for (int i = 0; i < 1000; i++) __nanosleep(1000);
}

// KEEP: with lse, and rest where it is given.  The backward of these windows reads neither, so only callers of the C ABI ask for
// them; a form of its own, since asking while running costs all others 5 us of 68 (64 x 1,024 tokens, window 16)
template <int DP, int NB, bool KEEP>
__global__ void __launch_bounds__(128) attn_fwd_narrow_kernel(AttnArgs a, RowInputs<bf16> in, bf16* out, bf16* rest, float* lse, const __grid_constant__ NarrowMaps maps) {
    constexpr int KEYS = NA_ROWS + 16 * (NB - 1), SUBS = DP / 64;
    extern __shared__ __align__(1024) char smem[];
    const uint32_t Q = smem_u32(smem), K = Q + NA_ROWS * DP * 2, V = K + KEYS * DP * 2;
    __shared__ uint64_t qk_full, v_full;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const int i0 = blockIdx.x * NA_ROWS, h = blockIdx.y, b = blockIdx.z, hk = h / (a.H / a.KV), j0 = i0 - 16 * (NB - 1);
    if (tid == 0) { mbar_init(&qk_full, 1); mbar_init(&v_full, 1); mbar_fence_init(); }
    __syncthreads();
    if (tid == 0) {
        mbar_arrive_expect_tx(&qk_full, (NA_ROWS + KEYS) * DP * 2);
        for (int c = 0; c < SUBS; c++) {
            tile_g2s(smem + c * NA_ROWS * 128, &maps.q, c * 64, i0, h, b, &qk_full);
            tile_g2s(smem + NA_ROWS * DP * 2 + c * KEYS * 128, &maps.k, c * 64, j0, hk, b, &qk_full);
        }
        mbar_arrive_expect_tx(&v_full, KEYS * DP * 2);
        for (int c = 0; c < SUBS; c++) tile_g2s(smem + (NA_ROWS + KEYS) * DP * 2 + c * KEYS * 128, &maps.v, c * 64, j0, hk, b, &v_full);
    }
    const Score sc(a, h);
    Span sp[2];
    int at[2];
#pragma unroll
    for (int r = 0; r < 2; r++) {
        at[r] = i0 + warp * 16 + lane / 4 + 8 * r;
        sp[r] = at[r] < a.Tq ? keys_of(a, b, at[r]) : Span{0, 0};
    }
    if (!all_arrived(&qk_full, 0)) { give_up(); return; }
    float s[2 * NB][4], none[1][4], inv[2];
    band<DP, NB>(s, Q, NA_ROWS, warp * 16, K, KEYS, warp * 16, lane);
    if constexpr (!KEEP) band_softmax<NB, false>(s, none, inv, sc, sp, at, j0 + warp * 16, lane);
    else {
        float x[2];
        band_softmax<NB, false>(s, none, inv, sc, sp, at, j0 + warp * 16, lane, x);
#pragma unroll
        for (int r = 0; r < 2; r++)
            if (lane % 4 == 0 && at[r] < a.Tq) lse[((size_t)b * a.H + h) * a.Tq + at[r]] = x[r];
    }
    if (!all_arrived(&v_full, 0)) { give_up(); return; }
    uint32_t p[NB][4];
#pragma unroll
    for (int n = 0; n < NB; n++) {
        p[n][0] = pack_bf16(s[2 * n][0], s[2 * n][1]);
        p[n][1] = pack_bf16(s[2 * n][2], s[2 * n][3]);
        p[n][2] = pack_bf16(s[2 * n + 1][0], s[2 * n + 1][1]);
        p[n][3] = pack_bf16(s[2 * n + 1][2], s[2 * n + 1][3]);
    }
    __syncwarp();                                        // the warp's queries are read: its outputs go over them
    float seen = 0.f;
#pragma unroll
    for (int c = 0; c < DP / 16; c++) {
        float o[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int n = 0; n < NB; n++) {
            uint32_t y[4];
            rows_as_bt(y, V, KEYS, warp * 16 + 16 * n, c, lane);
            mma(o[0], p[n], y[0], y[1]);
            mma(o[1], p[n], y[2], y[3]);
        }
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const uint32_t w[2] = {pack_bf16(o[t][0] * inv[0], o[t][1] * inv[0]), pack_bf16(o[t][2] * inv[1], o[t][3] * inv[1])};
            put_rows<DP>(Q, NA_ROWS, warp * 16, 2 * c + t, lane, w[0], w[1]);
#pragma unroll
            for (int i = 0; i < 4; i++) watch(seen, o[t][i]);
            if (KEEP && rest != nullptr) {
                const int d = c * 16 + t * 8 + (lane % 4) * 2;
#pragma unroll
                for (int r = 0; r < 2; r++)
                    if (d < a.D && at[r] < a.Tq)
                        *reinterpret_cast<uint32_t*>(rest + (((size_t)b * a.Tq + at[r]) * a.H + h) * a.D + d) =
                            pack_bf16(o[t][2 * r] * inv[r] - __uint_as_float(w[r] << 16), o[t][2 * r + 1] * inv[r] - __uint_as_float(w[r] & 0xffff0000u));
            }
        }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0 && i0 + warp * 16 < a.Tq) {
        for (int c = 0; c < SUBS; c++) tile_s2g(&maps.o, c * 64, i0 + warp * 16, h, b, smem + c * NA_ROWS * 128 + warp * 16 * 128);
        bulk_commit();
        bulk_wait_read<0>();
    }
    if (__any_sync(FULL, seen != seen)) {                // some row is not finite: the warp's rows anew, over what they see alone
        if (lane == 0) bulk_wait<0>();
        __syncwarp();
        for (int i = i0 + warp * 16; i < min(i0 + warp * 16 + 16, a.Tq); i++) {
            float x[4], l, unused;
            const size_t to = (((size_t)b * a.Tq + i) * a.H + h) * a.D;
            careful_query(a, in, b, h, i, x, l, unused);
            put_lane_row(out + to, x, a.D);
            if (KEEP && lane == 0) lse[((size_t)b * a.H + h) * a.Tq + i] = l;
            if (KEEP && rest != nullptr) {
#pragma unroll
                for (int c = 0; c < 4; c++) x[c] -= __bfloat162float(__float2bfloat16_rn(x[c]));
                put_lane_row(rest + to, x, a.D);
            }
        }
    }
}

template <int DP, int NB>
struct NarrowBwd {
    static constexpr int HB = NB - 1, WARPS = 4 + HB, QROWS = NA_ROWS + 16 * HB, KROWS = NA_ROWS + 32 * HB;
    static constexpr int PLD = NB * 32 + 16;             // bytes of a row of p or ds: no two rows of eight on the same banks
    static constexpr int QT = QROWS * DP * 2, KT = KROWS * DP * 2, PT = 16 * PLD;
    static constexpr int SMEM = 2 * QT + 2 * KT + WARPS * 2 * PT;
};

// GROUP: several query heads share a key head, whose dk and dv stay in registers over them; one CTA to an SM.  Without, dv is done before dk is
// begun, and two CTAs fit (286 against 158 us for 64 x 1,024 tokens, window 16).
template <int DP, int NB, bool GROUP>
__global__ void __launch_bounds__(NarrowBwd<DP, NB>::WARPS * 32, GROUP || NB > 3 ? 1 : 2) attn_bwd_narrow_kernel(AttnArgs a, RowInputs<bf16> in, bf16* dq_out, bf16* dk_out, bf16* dv_out, const __grid_constant__ NarrowBwdMaps maps) {
    typedef NarrowBwd<DP, NB> Sh;
    constexpr int HB = Sh::HB, SUBS = DP / 64;
    extern __shared__ __align__(1024) char smem[];
    const uint32_t Q = smem_u32(smem), G = Q + Sh::QT, K = G + Sh::QT, V = K + Sh::KT, Pm = V + Sh::KT;      // G: do
    __shared__ uint64_t kv_full, q_full;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31, group = a.H / a.KV;
    const int x0 = blockIdx.x * NA_ROWS, hk = blockIdx.y, b = blockIdx.z, j0 = x0 - 16 * HB;
    if (tid == 0) { mbar_init(&kv_full, 1); mbar_init(&q_full, 1); mbar_fence_init(); }
    __syncthreads();
    if (tid == 0) {
        mbar_arrive_expect_tx(&kv_full, 2 * Sh::KT);
        for (int c = 0; c < SUBS; c++) {
            tile_g2s(smem + 2 * Sh::QT + c * Sh::KROWS * 128, &maps.k, c * 64, j0, hk, b, &kv_full);
            tile_g2s(smem + 2 * Sh::QT + Sh::KT + c * Sh::KROWS * 128, &maps.v, c * 64, j0, hk, b, &kv_full);
        }
    }
    Span sp[2];
    int at[2];
#pragma unroll
    for (int r = 0; r < 2; r++) {
        at[r] = x0 + warp * 16 + lane / 4 + 8 * r;
        sp[r] = at[r] < a.Tq ? keys_of(a, b, at[r]) : Span{0, 0};
    }
    float sums[GROUP ? 2 : 1][DP / 8][4];                // of the warp's 16 keys: dv, dk
    auto clear = [](float (&x)[DP / 8][4]) {
#pragma unroll
        for (int c = 0; c < DP / 8; c++)
#pragma unroll
            for (int i = 0; i < 4; i++) x[c][i] = 0.f;
    };
    // += p^T do (which 0) or ds^T q: the queries of block warp + n see these keys in their block HB - n
    auto gather = [&](float (&x)[DP / 8][4], int which) {
#pragma unroll
        for (int n = 0; n < NB; n++) {
            uint32_t w[4];
            ldsm_t(w, Pm + ((warp + n) * 2 + which) * Sh::PT + ((lane / 16) * 8 + lane % 8) * Sh::PLD + (HB - n) * 32 + ((lane / 8) % 2) * 16);
#pragma unroll
            for (int c = 0; c < DP / 16; c++) {
                uint32_t y[4];
                rows_as_bt(y, which ? Q : G, Sh::QROWS, (warp + n) * 16, c, lane);
                mma(x[2 * c], w, y[0], y[1]);
                mma(x[2 * c + 1], w, y[2], y[3]);
            }
        }
    };
    float seen_keys = 0.f;                               // NaN where dk or dv is not finite
    unsigned bad_heads = 0;                              // of the group, whose dq is not: bit 31 for all from the 32nd on
    // dv over v, dk over k, which all have read
    auto put = [&](const float (&x)[DP / 8][4], int which) {
        const float mul = which ? a.scale : 1.f;
#pragma unroll
        for (int c = 0; c < DP / 8; c++) {
#pragma unroll
            for (int i = 0; i < 4; i++) watch(seen_keys, x[c][i]);
            put_rows<DP>(which ? K : V, Sh::KROWS, warp * 16, c, lane, pack_bf16(x[c][0] * mul, x[c][1] * mul), pack_bf16(x[c][2] * mul, x[c][3] * mul));
        }
    };
    if constexpr (GROUP) { clear(sums[0]); clear(sums[1]); }
    const uint32_t P = Pm + warp * 2 * Sh::PT, D = P + Sh::PT;
    for (int g = 0; g < (GROUP ? group : 1); g++) {
        const int h = hk * group + g;
        if (tid == 0) {
            mbar_arrive_expect_tx(&q_full, 2 * Sh::QT);
            for (int c = 0; c < SUBS; c++) {
                tile_g2s(smem + c * Sh::QROWS * 128, &maps.q, c * 64, x0, h, b, &q_full);
                tile_g2s(smem + Sh::QT + c * Sh::QROWS * 128, &maps.d, c * 64, x0, h, b, &q_full);
            }
        }
        if (g == 0 && !all_arrived(&kv_full, 0)) { give_up(); return; }
        if (!all_arrived(&q_full, g & 1)) { give_up(); return; }
        const Score sc(a, h);
        float s[2 * NB][4], f[2 * NB][4], dp[2 * NB][4], inv[2];
        band<DP, NB>(s, Q, Sh::QROWS, warp * 16, K, Sh::KROWS, warp * 16, lane);
        band_softmax<NB, true>(s, f, inv, sc, sp, at, j0 + warp * 16, lane);
        band<DP, NB>(dp, G, Sh::QROWS, warp * 16, V, Sh::KROWS, warp * 16, lane);
        uint32_t ds[NB][4];
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const bool alone = sp[r].hi - sp[r].lo <= 1; // the scores of a row that sees one key have no gradient
            float delta = 0.f;
#pragma unroll
            for (int t = 0; t < 2 * NB; t++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float& p = s[t][2 * r + e];
                    p *= inv[r];
                    if (p != 0.f) delta = fmaf(p, dp[t][2 * r + e], delta);
                }
            delta += __shfl_xor_sync(FULL, delta, 1);
            delta += __shfl_xor_sync(FULL, delta, 2);
#pragma unroll
            for (int t = 0; t < 2 * NB; t++) {
                float w[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float p = s[t][2 * r + e];
                    w[e] = p == 0.f || alone ? 0.f : p * (dp[t][2 * r + e] - delta) * f[t][2 * r + e];
                }
                const uint32_t pw = pack_bf16(s[t][2 * r], s[t][2 * r + 1]), dw = pack_bf16(w[0], w[1]);
                const uint32_t to = (lane / 4 + 8 * r) * Sh::PLD + t * 16 + (lane % 4) * 4;
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(P + to), "r"(pw) : "memory");
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(D + to), "r"(dw) : "memory");
                ds[t / 2][(t % 2) * 2 + r] = dw;
            }
        }
        // dq = scale ds k, kept packed until k and v are no longer needed as they are
        uint32_t dq[DP / 8][2];
        float seen = 0.f;
#pragma unroll
        for (int c = 0; c < DP / 16; c++) {
            float x[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int n = 0; n < NB; n++) {
                uint32_t y[4];
                rows_as_bt(y, K, Sh::KROWS, warp * 16 + 16 * n, c, lane);
                mma(x[0], ds[n], y[0], y[1]);
                mma(x[1], ds[n], y[2], y[3]);
            }
#pragma unroll
            for (int t = 0; t < 2; t++) {
#pragma unroll
                for (int i = 0; i < 4; i++) watch(seen, x[t][i]);
                dq[2 * c + t][0] = pack_bf16(x[t][0] * a.scale, x[t][1] * a.scale);
                dq[2 * c + t][1] = pack_bf16(x[t][2] * a.scale, x[t][3] * a.scale);
            }
        }
        if (__any_sync(FULL, seen != seen)) bad_heads |= 1u << min(g, 31);
        __syncthreads();                                 // p and ds of all queries are there
        if (warp < 4) {
#pragma unroll
            for (int which = 0; which < 2; which++) {
                if constexpr (GROUP) gather(sums[which], which);
                else {
                    clear(sums[0]);
                    gather(sums[0], which);
                    put(sums[0], which);
                }
            }
        }
        __syncthreads();                                 // q and do are read: dq goes over q's rows, which are dq's
        if (warp < 4) {
#pragma unroll
            for (int c = 0; c < DP / 8; c++) put_rows<DP>(Q, Sh::QROWS, warp * 16, c, lane, dq[c][0], dq[c][1]);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && x0 + warp * 16 < a.Tq) {
                for (int c = 0; c < SUBS; c++) tile_s2g(&maps.dq, c * 64, x0 + warp * 16, h, b, smem + c * Sh::QROWS * 128 + warp * 16 * 128);
                bulk_commit();
                bulk_wait_read<0>();
            }
        }
        if (GROUP && g + 1 < group) __syncthreads();     // before the next head's queries come in
    }
    if (warp < 4) {
        if constexpr (GROUP) { put(sums[0], 0); put(sums[1], 1); }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && x0 + warp * 16 < a.Tk) {
            for (int c = 0; c < SUBS; c++) {
                tile_s2g(&maps.dk, c * 64, x0 + warp * 16, hk, b, smem + 2 * Sh::QT + c * Sh::KROWS * 128 + warp * 16 * 128);
                tile_s2g(&maps.dv, c * 64, x0 + warp * 16, hk, b, smem + 2 * Sh::QT + Sh::KT + c * Sh::KROWS * 128 + warp * 16 * 128);
            }
            bulk_commit();
            bulk_wait_read<0>();
        }
        if (bad_heads != 0 || __any_sync(FULL, seen_keys != seen_keys)) {          // some row is not finite: anew, over what sees what alone
            const bool keys = __any_sync(FULL, seen_keys != seen_keys);
            if (lane == 0) bulk_wait<0>();
            __syncwarp();
            for (int x = x0 + warp * 16; x < min(x0 + warp * 16 + 16, a.Tk); x++) {
                float dk[4], dv[4];
                for (int g = 0; g < group; g++) {
                    if (!(bad_heads >> min(g, 31) & 1)) continue;
                    careful_dq(a, in, nullptr, nullptr, b, hk * group + g, x, dk);
                    put_lane_row(dq_out + (((size_t)b * a.Tq + x) * a.H + hk * group + g) * a.D, dk, a.D);
                }
                if (!keys) continue;
                careful_dkv(a, in, nullptr, nullptr, b, hk, x, dk, dv);
                put_lane_row(dk_out + (((size_t)b * a.Tk + x) * a.KV + hk) * a.D, dk, a.D);
                put_lane_row(dv_out + (((size_t)b * a.Tk + x) * a.KV + hk) * a.D, dv, a.D);
            }
        }
    }
}

template <int DP, int NB>
static cudaError_t fwd_narrow(const AttnArgs& a, const void* q, const void* k, const void* v, void* o, void* rest, float* lse, cudaStream_t st) {
    constexpr int KEYS = NA_ROWS + 16 * (NB - 1), SMEM = (NA_ROWS + 2 * KEYS) * DP * 2;
    const long long os[3] = {(long long)a.Tq * a.H * a.D, (long long)a.H * a.D, a.D};
    auto kern = lse != nullptr ? attn_fwd_narrow_kernel<DP, NB, true> : attn_fwd_narrow_kernel<DP, NB, false>;
    const cudaError_t e = opt_in_smem(kern, SMEM);       // before the maps: a thread's first runtime call makes the context current for them
    if (e != cudaSuccess) return e;
    NarrowMaps m;
    if (!tile_map(&m.q, q, a.B, a.Tq, a.H, a.D, a.qs, NA_ROWS) || !tile_map(&m.k, k, a.B, a.Tk, a.KV, a.D, a.ks, KEYS) ||
        !tile_map(&m.v, v, a.B, a.Tk, a.KV, a.D, a.vs, KEYS) || !tile_map(&m.o, o, a.B, a.Tq, a.H, a.D, os, 16))
        return cudaErrorInvalidValue;
    kern<<<dim3((a.Tq + NA_ROWS - 1) / NA_ROWS, a.H, a.B), 128, SMEM, st>>>(a, RowInputs<bf16>{(const bf16*)q, (const bf16*)k, (const bf16*)v, nullptr}, (bf16*)o, (bf16*)rest, lse, m);
    return cudaGetLastError();
}
template <int DP, int NB>
static cudaError_t bwd_narrow(const AttnArgs& a, const void* q, const void* k, const void* v, const void* dout, void* dq, void* dk, void* dv, cudaStream_t st) {
    typedef NarrowBwd<DP, NB> Sh;
    const long long os[3] = {(long long)a.Tq * a.H * a.D, (long long)a.H * a.D, a.D}, gs[3] = {(long long)a.Tk * a.KV * a.D, (long long)a.KV * a.D, a.D};
    auto kern = a.H > a.KV ? attn_bwd_narrow_kernel<DP, NB, true> : attn_bwd_narrow_kernel<DP, NB, false>;
    const cudaError_t e = opt_in_smem(kern, Sh::SMEM);      // before the maps
    if (e != cudaSuccess) return e;
    NarrowBwdMaps m;
    if (!tile_map(&m.q, q, a.B, a.Tq, a.H, a.D, a.qs, Sh::QROWS) || !tile_map(&m.d, dout, a.B, a.Tq, a.H, a.D, os, Sh::QROWS) ||
        !tile_map(&m.k, k, a.B, a.Tk, a.KV, a.D, a.ks, Sh::KROWS) || !tile_map(&m.v, v, a.B, a.Tk, a.KV, a.D, a.vs, Sh::KROWS) ||
        !tile_map(&m.dq, dq, a.B, a.Tq, a.H, a.D, os, 16) || !tile_map(&m.dk, dk, a.B, a.Tk, a.KV, a.D, gs, 16) ||
        !tile_map(&m.dv, dv, a.B, a.Tk, a.KV, a.D, gs, 16))
        return cudaErrorInvalidValue;
    kern<<<dim3((a.Tk + NA_ROWS - 1) / NA_ROWS, a.KV, a.B), Sh::WARPS * 32, Sh::SMEM, st>>>(a, RowInputs<bf16>{(const bf16*)q, (const bf16*)k, (const bf16*)v, (const bf16*)dout}, (bf16*)dq, (bf16*)dk, (bf16*)dv, m);
    return cudaGetLastError();
}

bool attn_narrow(const AttnArgs& a) { return a.prefix == nullptr && a.Tq == a.Tk && a.window <= NARROW_WINDOW; }

cudaError_t run_attn_fwd_narrow(const AttnArgs& a, const void* q, const void* k, const void* v, void* o, void* rest, float* lse, cudaStream_t st) {
    if (a.window <= 17) return a.D <= 64 ? fwd_narrow<64, 2>(a, q, k, v, o, rest, lse, st) : fwd_narrow<128, 2>(a, q, k, v, o, rest, lse, st);
    if (a.window <= 33) return a.D <= 64 ? fwd_narrow<64, 3>(a, q, k, v, o, rest, lse, st) : fwd_narrow<128, 3>(a, q, k, v, o, rest, lse, st);
    return a.D <= 64 ? fwd_narrow<64, 5>(a, q, k, v, o, rest, lse, st) : fwd_narrow<128, 5>(a, q, k, v, o, rest, lse, st);
}
cudaError_t run_attn_bwd_narrow(const AttnArgs& a, const void* q, const void* k, const void* v, const void* dout, void* dq, void* dk, void* dv,
                                cudaStream_t st) {
    if (a.window <= 17) return a.D <= 64 ? bwd_narrow<64, 2>(a, q, k, v, dout, dq, dk, dv, st) : bwd_narrow<128, 2>(a, q, k, v, dout, dq, dk, dv, st);
    if (a.window <= 33) return a.D <= 64 ? bwd_narrow<64, 3>(a, q, k, v, dout, dq, dk, dv, st) : bwd_narrow<128, 3>(a, q, k, v, dout, dq, dk, dv, st);
    return a.D <= 64 ? bwd_narrow<64, 5>(a, q, k, v, dout, dq, dk, dv, st) : bwd_narrow<128, 5>(a, q, k, v, dout, dq, dk, dv, st);
}

int attn_narrow_status() {
    int v = 0;
    const int z = 0;
    if (cudaMemcpyFromSymbol(&v, g_narrow_status, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) cudaMemcpyToSymbol(g_narrow_status, &z, sizeof(int));
    return v;
}

}  // namespace slotscan
