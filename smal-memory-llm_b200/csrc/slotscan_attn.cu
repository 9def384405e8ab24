// C ABI of the attention over tokens: argument checks and the choice of the kernels by type.
#include "slotscan_attn.cuh"
#include "slotscan_launch.h"

using namespace slotscan;

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

extern "C" int slotscan_attn_check(const slotscan_attn_params* p) {
    if (p == nullptr) return SLOTSCAN_E_NULL;
    if (p->dtype != SLOTSCAN_F32 && p->dtype != SLOTSCAN_BF16) return SLOTSCAN_E_DTYPE;
    if (p->B < 0 || p->B > 65535 || p->Tq < 0 || p->Tk < p->Tq || p->Tk > (1 << 29) || p->H < 1 || p->H > 65535 || p->KV < 1 || p->H % p->KV ||
        p->D < 8 || p->D > 128 || p->D % 8)
        return SLOTSCAN_E_SHAPE;
    if (p->window < 0 || !(p->cap >= 0.f) || !(p->cap < INFINITY) || !(p->scale > 0.f) || !(p->scale < INFINITY)) return SLOTSCAN_E_MODE;
    const int e = p->dtype == SLOTSCAN_BF16 ? 2 : 4;
    for (int i = 0; i < 3; i++)
        if (p->q_stride[i] * e % 16 || p->k_stride[i] * e % 16 || p->v_stride[i] * e % 16) return SLOTSCAN_E_ALIGN;
    return SLOTSCAN_OK;
}

static AttnArgs attn_args(const slotscan_attn_params& p, const float* slopes, const int32_t* docs, const int32_t* prefix) {
    AttnArgs a;
    a.B = p.B; a.Tq = p.Tq; a.Tk = p.Tk; a.H = p.H; a.KV = p.KV; a.D = p.D;
    a.window = p.window > 0 && p.window < p.Tk ? p.window : p.Tk;
    a.scale = p.scale; a.cap = p.cap;
    for (int i = 0; i < 3; i++) { a.qs[i] = p.q_stride[i]; a.ks[i] = p.k_stride[i]; a.vs[i] = p.v_stride[i]; }
    a.slopes = slopes; a.docs = (const int2*)docs; a.prefix = prefix;
    return a;
}

extern "C" int slotscan_attn_keeps(const slotscan_attn_params* p, int with_prefix) {
    if (slotscan_attn_check(p) != SLOTSCAN_OK) return 0;
    const int32_t none = 0;
    return !(p->dtype == SLOTSCAN_BF16 && attn_narrow(attn_args(*p, nullptr, nullptr, with_prefix ? &none : nullptr)));
}

extern "C" int slotscan_attn_fwd(const slotscan_attn_params* p, const void* q, const void* k, const void* v, const float* slopes,
                                 const int32_t* docs, const int32_t* prefix, void* o, void* rest, float* lse, void* stream) {
    const int rc = slotscan_attn_check(p);
    if (rc != SLOTSCAN_OK) return rc;
    if ((int64_t)p->B * p->Tq == 0) return SLOTSCAN_OK;
    if (!q || !k || !v || !o) return SLOTSCAN_E_NULL;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || !aligned16(rest) || ((uintptr_t)docs & 7)) return SLOTSCAN_E_ALIGN;
    const AttnArgs a = attn_args(*p, slopes, docs, prefix);
    if (p->dtype == SLOTSCAN_BF16 && attn_narrow(a)) return (int)run_attn_fwd_narrow(a, q, k, v, o, lse ? rest : nullptr, lse, (cudaStream_t)stream);
    if (p->dtype == SLOTSCAN_BF16 && lse && !rest) return SLOTSCAN_E_NULL;
    return (int)(p->dtype == SLOTSCAN_BF16 ? run_attn_fwd_bf16(a, q, k, v, o, rest, lse, (cudaStream_t)stream)
                                           : run_attn_fwd_f32(a, q, k, v, o, lse, (cudaStream_t)stream));
}

extern "C" int slotscan_attn_bwd(const slotscan_attn_params* p, const void* q, const void* k, const void* v, const float* slopes,
                                 const int32_t* docs, const int32_t* prefix, const void* o, const void* rest, const float* lse, const void* dout,
                                 float* delta, void* dq, void* dk, void* dv, void* stream) {
    const int rc = slotscan_attn_check(p);
    if (rc != SLOTSCAN_OK) return rc;
    if ((int64_t)p->B * p->Tk == 0) return SLOTSCAN_OK;
    if (p->Tq == 0) {                                    // keys without a query
        const size_t n = (size_t)p->B * p->Tk * p->KV * p->D * (p->dtype == SLOTSCAN_BF16 ? 2 : 4);
        if (!dk || !dv) return SLOTSCAN_E_NULL;
        cudaError_t e = cudaMemsetAsync(dk, 0, n, (cudaStream_t)stream);
        if (e == cudaSuccess) e = cudaMemsetAsync(dv, 0, n, (cudaStream_t)stream);
        return (int)e;
    }
    if (!q || !k || !v || !dout || !dq || !dk || !dv) return SLOTSCAN_E_NULL;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || !aligned16(rest) || !aligned16(dout) || !aligned16(dq) || !aligned16(dk) ||
        !aligned16(dv) || ((uintptr_t)docs & 7))
        return SLOTSCAN_E_ALIGN;
    const AttnArgs a = attn_args(*p, slopes, docs, prefix);
    if (p->dtype == SLOTSCAN_BF16 && attn_narrow(a)) return (int)run_attn_bwd_narrow(a, q, k, v, dout, dq, dk, dv, (cudaStream_t)stream);
    if (!o || !lse || !delta || (p->dtype == SLOTSCAN_BF16 && !rest)) return SLOTSCAN_E_NULL;
    return (int)(p->dtype == SLOTSCAN_BF16 ? run_attn_bwd_bf16(a, q, k, v, o, rest, lse, dout, delta, dq, dk, dv, (cudaStream_t)stream)
                                           : run_attn_bwd_f32(a, q, k, v, o, lse, dout, delta, dq, dk, dv, (cudaStream_t)stream));
}
