// Tensor cores of sm_100a: tensor memory, tcgen05 products, tiled bulk tensor copies.
//
// Tiles in shared memory are sub-tiles of 64 bf16 columns, rows of 128 bytes, 16-byte pieces swizzled by the row within eight
// (the 128-byte swizzle of the copies).  A tile is an operand of a product either way: with its columns along the sum
// (K-major: the eight-row groups 1,024 bytes apart, 32 bytes further per 16 columns), or with its rows along the sum (MN-major: the
// sub-tiles one stride apart, 2,048 bytes further per 16 rows).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "slotscan_async.cuh"

namespace slotscan {

// ---- tensor memory: 128 lanes x 512 columns of 32 bits; a warp reaches the 32 lanes of its place within four ----
// one whole warp; columns a power of two >= 32; waits while another CTA of the SM holds them
__device__ __forceinline__ void tmem_alloc(uint32_t* out, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(out)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// a lane's row, consecutive columns
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr));
}
// orders the loaded registers behind the loads of this warp
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :: "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
}
// orders the loaded registers behind the loads of this warp
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :: "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
                 ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
                 ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
                 : "memory");
}

__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};"
                 ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(addr)
                 : "memory");
}
// ---- products: D (128 x N, float32 in tensor memory) = A B^T (+ D), bf16 operands ----
// The warp runs to them as a whole, so that addresses are known to be the same in every lane, and its elected lane issues.
// The operands' descriptors are built from their lower halves, the upper one being a constant, so that a product takes
// few instructions: with 64-bit sums and an election each the issue was slower than the products.
// shared-memory operand with the 128-byte swizzle: lower half.  lead: bytes from sub-tile to sub-tile (used where rows run along
// the sum); add bytes / 16 to move on
__device__ __forceinline__ uint32_t tile_desc(uint32_t addr, uint32_t lead) { return ((addr >> 4) & 0x3fff) | ((lead >> 4) & 0x3fff) << 16; }
constexpr uint32_t TILE_DESC_HIGH = (1024 >> 4) | 1u << 14 | 2u << 29;              // eight rows 1,024 bytes apart, version, swizzle
// float32 sums of bf16 products, 128 x N; bT: B's rows run along the sum
__host__ __device__ constexpr uint32_t mma_shape(int n, bool bT) { return 1u << 4 | 1u << 7 | 1u << 10 | (bT ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (128u >> 4) << 24; }
__device__ __forceinline__ bool elected() {
    uint32_t e;
    asm volatile("{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\nselp.u32 %0, 1, 0, q;\n}\n" : "=r"(e));
    return e != 0;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t shape, bool add) {
    asm volatile("{\n.reg .pred p;\n.reg .b64 x, y;\nmov.b64 x, {%1, %5};\nmov.b64 y, {%2, %5};\nsetp.ne.u32 p, %4, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(shape), "r"((uint32_t)add), "r"(TILE_DESC_HIGH)
                 : "memory");
}
// A in tensor memory: two bf16 to a column
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t shape, bool add) {
    asm volatile("{\n.reg .pred p;\n.reg .b64 y;\nmov.b64 y, {%2, %5};\nsetp.ne.u32 p, %4, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(shape), "r"((uint32_t)add), "r"(TILE_DESC_HIGH)
                 : "memory");
}
// one arrival at `bar` when all products issued so far by the elected lane (the same each time) are done; called by that lane
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// ---- tiled copies of a (sequence, head, token, channel) tensor ----
__device__ __forceinline__ void tile_g2s(void* dst, const CUtensorMap* map, int col, int row, int head, int seq, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(col), "r"(row), "r"(head), "r"(seq), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tile_s2g(const CUtensorMap* map, int col, int row, int head, int seq, const void* src) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(col),
                 "r"(row), "r"(head), "r"(seq), "r"(smem_u32(src))
                 : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory"); }
// of a (row, head, channel) tensor
__device__ __forceinline__ void box_g2s(void* dst, const CUtensorMap* map, int col, int head, int row, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(col), "r"(head), "r"(row), "r"(smem_u32(bar))
                 : "memory");
}
// byte offset of the 16-byte piece `piece` (of 8) of row `row` in a sub-tile
__device__ __forceinline__ uint32_t swizzled(int row, int piece) { return row * 128 + ((piece ^ (row & 7)) << 4); }

__device__ __forceinline__ void arrive(uint64_t* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory"); }
// Bounded wait without a sleep in its first polls: the products hand over every microsecond.
__device__ __forceinline__ bool wait_soon(uint64_t* bar, unsigned parity) {
    for (int it = 0; it < (1 << 21); it++) {
        if (mbar_try_wait(bar, parity)) return true;
        if (it > (1 << 12)) __nanosleep(100);
    }
    return false;
}
__device__ __forceinline__ bool wait_soon_warp(uint64_t* bar, unsigned parity) { return __all_sync(0xffffffffu, wait_soon(bar, parity)); }
__device__ __forceinline__ void sync_group(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float rcp_fast(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// (sequence, head, token, channel) bf16 tensor, boxes of 64 channels x `rows` tokens of one head; zeros beyond the tensor's ends.
// strides in elements, of a sequence, a token and a head (any value where that dimension has one element).
typedef CUresult (*TileMapEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                    const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static inline TileMapEncodeFn tile_map_encoder() {
    static TileMapEncodeFn enc = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) f = nullptr;
        return (TileMapEncodeFn)f;
    }();
    return enc;
}
static inline bool tile_map(CUtensorMap* m, const void* base, int B, int T, int H, int D, const long long* stride, int rows) {
    const TileMapEncodeFn enc = tile_map_encoder();
    if (enc == nullptr) return false;
    auto bytes = [&](long long s, int n) { return (cuuint64_t)(n == 1 ? 2ll * D : 2ll * s); };
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)T, (cuuint64_t)H, (cuuint64_t)B};
    const cuuint64_t strides[3] = {bytes(stride[1], T), bytes(stride[2], H), bytes(stride[0], B)};
    const cuuint32_t box[4] = {64u, (cuuint32_t)rows, 1u, 1u}, es[4] = {1u, 1u, 1u, 1u};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// (row, head, channel) bf16 tensor, boxes of 64 channels x `heads` heads x `rows` rows, the heads of a row side by side; strides of a row and
// a head
static inline bool box_map(CUtensorMap* m, const void* base, int N, int H, int D, const long long* stride, int heads, int rows) {
    const TileMapEncodeFn enc = tile_map_encoder();
    if (enc == nullptr) return false;
    auto bytes = [&](long long s, int n) { return (cuuint64_t)(n == 1 ? 2ll * D : 2ll * s); };
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)N}, strides[2] = {bytes(stride[1], H), bytes(stride[0], N)};
    const cuuint32_t box[3] = {64u, (cuuint32_t)heads, (cuuint32_t)rows}, es[3] = {1u, 1u, 1u};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace slotscan
