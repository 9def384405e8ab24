// The scores of a thread's row, out of tensor memory: cap, bias and mask, of the forward kernels on the tensor cores.
#pragma once
#include <type_traits>

#include "slotscan_attn.cuh"
#include "slotscan_tensor.cuh"

namespace slotscan {

// 32 scores of a row as base-2 exponents (CAP or BIAS: whole; else still without the factor `lin`), minus infinity where the row does
// not see them.  A warp's block is capped by one of two forms, which are rounded differently, and by its greatest score: rows that do not count
// (whatever stands there) have no say in that, nor, with SEEN, have columns that a row does not see.
template <bool CAP, bool BIAS, bool SEEN = false>
__device__ __forceinline__ void scores32(float (&s)[32], const Score& sc, float ahead, bool masked, int lo, int hi, bool counts = true) {
    bool small = true;                                   // the capped scores' polynomial serves this warp's block
    if constexpr (CAP) {
        float m0 = 0.f, m1 = 0.f;
        if (SEEN && masked) {
#pragma unroll
            for (int i = 0; i < 32; i++) m0 = i >= lo && i < hi ? fmaxf(m0, fabsf(s[i])) : m0;
        } else {
#pragma unroll
            for (int i = 0; i < 32; i += 2) { m0 = fmaxf(m0, fabsf(s[i])); m1 = fmaxf(m1, fabsf(s[i + 1])); }
        }
        small = __all_sync(FULL, !counts || fmaxf(m0, m1) * sc.cap_in <= CAP_POLY_MOST);
    }
    if constexpr (CAP || BIAS) {
        auto whole = [&](auto poly) {
            const CapPoly cp(sc);
            const f32x2 lin = pack2(sc.lin, sc.lin), steep = pack2(-sc.slope, -sc.slope);
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
                const f32x2 x = pack2(s[i], s[i + 1]);
                f32x2 z;
                if constexpr (CAP && decltype(poly)::value) z = mul2(x, cp.slope(x));
                else if constexpr (CAP) {                                                      // tanh x = 1 - 2 / (e^2x + 1)
                    const float in = 2.f * LOG2E * sc.cap_in;
                    z = pack2(fmaf(-2.f * sc.cap_out, rcp_fast(exp2_fast(s[i] * in) + 1.f), sc.cap_out),
                              fmaf(-2.f * sc.cap_out, rcp_fast(exp2_fast(s[i + 1] * in) + 1.f), sc.cap_out));
                } else z = mul2(x, lin);
                if constexpr (BIAS) z = fma2(pack2(fabsf(ahead - (float)i), fabsf(ahead - (float)(i + 1))), steep, z);
                const float2 u = unpack2(z);
                s[i] = u.x;
                s[i + 1] = u.y;
            }
        };
        if (small) whole(std::true_type{});
        else if constexpr (CAP) whole(std::false_type{});
    }
    if (masked) {
#pragma unroll
        for (int i = 0; i < 32; i++) s[i] = i >= lo && i < hi ? s[i] : -INFINITY;
    }
}

}  // namespace slotscan
