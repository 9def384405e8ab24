// Host side of the token ops for ordinary eager calls: argument checks, outputs, launch and autograd in C++ over the C ABI.
//
// A small training call through a Python autograd.Function takes some 160 us of host time, most of it the engine's hand-over to a Python
// backward; its kernels take ten.  This module takes the calls that need no preparation: tensors of the expected types that the kernels
// can read in place.  Whatever else comes (another layout, a type to convert, an argument to refuse) it hands back as None, and
// tokens.py does it, with its errors.
#include <torch/extension.h>

#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cstdint>
#include <optional>
#include <stdexcept>
#include <string>

#include "slotscan.h"

namespace {

using at::Tensor;
typedef std::optional<Tensor> Maybe;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ---- what the kernels can take as it is ----
int code(const Tensor& t) { return t.scalar_type() == at::kFloat ? SLOTSCAN_F32 : t.scalar_type() == at::kBFloat16 ? SLOTSCAN_BF16 : -1; }
// adjacent channels, everything else on 16-byte boundaries, no dimension expanded; strides of a dimension of one element: 0
bool laid(const Tensor& t, int64_t* strides) {
    const int64_t n = t.dim(), size = t.element_size();
    if (t.stride(n - 1) != 1 || (uintptr_t)t.const_data_ptr() % 16) return false;
    for (int64_t i = 0; i + 1 < n; i++) {
        const int64_t s = t.stride(i);
        if (t.size(i) > 1 && (s == 0 || s * size % 16)) return false;
        strides[i] = t.size(i) == 1 ? 0 : s;
    }
    return true;
}
bool some(const Maybe& t) { return t.has_value() && t->defined(); }
// absent, or contiguous of this type and these sizes on this device
bool fits(const Maybe& t, at::ScalarType type, at::IntArrayRef sizes, const Tensor& like) {
    return !some(t) || (t->scalar_type() == type && t->sizes() == sizes && t->is_contiguous() && t->device() == like.device());
}
bool wants_grad(std::initializer_list<const Maybe*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Maybe* t : ts)
        if (some(*t) && (*t)->requires_grad()) return true;
    return false;
}
template <typename T>
const T* ptr(const Maybe& t) { return some(t) && t->numel() ? (const T*)t->const_data_ptr() : nullptr; }
const void* in(const Tensor& t) { return t.numel() ? t.const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() && t.numel() ? t.mutable_data_ptr() : nullptr; }
void* stream_of(const Tensor& t) { return (void*)c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
void check(int rc, const char* what) {
    if (rc < 0) throw std::invalid_argument(std::string(what) + " rejected the call (code " + std::to_string(rc) + ")");
    if (rc > 0) throw std::runtime_error(std::string(what) + ": CUDA error " + std::to_string(rc));
}
// An upstream gradient, contiguous and on a 16-byte boundary.
Tensor whole(const Tensor& g, at::ScalarType type) {
    Tensor t = g.scalar_type() == type ? g.contiguous() : g.to(type).contiguous();
    return (uintptr_t)t.const_data_ptr() % 16 ? t.clone() : t;
}
// Whether a backward may go round the registered op: ordinary gradients (of no mode, batch or subclass), and none of a higher order wanted
bool first_order(const variable_list& grads) {
    using K = c10::DispatchKey;
    static const c10::DispatchKeySet special({K::Python, K::PythonTLSSnapshot, K::Batched, K::BatchedNestedTensor, K::FuncTorchBatched, K::FuncTorchGradWrapper,
                                              K::FuncTorchDynamicLayerFrontMode, K::FuncTorchDynamicLayerBackMode, K::Functionalize, K::Negative, K::Conjugate,
                                              K::ZeroTensor, K::NestedTensor});
    if (at::GradMode::is_enabled() || c10::impl::TorchDispatchModeTLS::any_modes_set()) return false;
    if (c10::impl::tls_local_dispatch_key_set().included_.has_any(special)) return false;
    for (const Tensor& g : grads)
        if (g.defined() && (!g.is_cuda() || g.key_set().has_any(special))) return false;
    return true;
}
variable_list registered(const char* name, std::vector<c10::IValue> args) {
    const auto op = c10::Dispatcher::singleton().findSchemaOrThrow(name, "");
    torch::jit::Stack stack(std::move(args));
    op.callBoxed(&stack);
    variable_list r;
    for (const c10::IValue& v : stack) r.push_back(v.toTensor());
    return r;
}
c10::IValue or_none(const Tensor& t) { return t.defined() ? c10::IValue(t) : c10::IValue(); }
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
// Written in place, past the dispatcher: a backward that has saved `t` must find out (tensors of inference mode are not counted)
void changed(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// int64 as the kernels read integers; what 32 bits cannot hold becomes the nearest that they can: beyond every table, bound and length
Tensor in_32_bits(const Tensor& t) { return t.scalar_type() == at::kLong && t.is_cuda() ? t.clamp(INT32_MIN, INT32_MAX).to(at::kInt) : t; }
Maybe in_32_bits(const Maybe& t) { return some(t) ? Maybe(in_32_bits(*t)) : t; }

// ---- norms and rotation ----
bool norm_params(slotscan_norm_params& p, const Tensor& q, const Tensor& k, const Maybe& table, const Maybe& qw, const Maybe& kw, double eps) {
    if (q.dim() != 4 || k.dim() != 4 || code(q) < 0 || code(q) != code(k) || !q.is_cuda() || q.device() != k.device()) return false;
    const int64_t B = q.size(0), T = q.size(1), H = q.size(2), D = q.size(3);
    if (k.size(0) != B || k.size(1) != T || k.size(3) != D || std::max({B, T, H, k.size(2), D}) > 0x7fffffff) return false;
    if (some(table) && (table->dim() != 3 || !fits(table, at::kFloat, {table->size(0), table->size(1), 2}, q) || table->size(0) > 0x7fffffff ||
                        table->size(1) > D))
        return false;
    if (!fits(qw, at::kFloat, {D}, q) || !fits(kw, at::kFloat, {D}, q)) return false;
    p.B = (int32_t)B; p.T = (int32_t)T; p.H = (int32_t)H; p.KV = (int32_t)k.size(2); p.D = (int32_t)D;
    p.R = some(table) ? 2 * (int32_t)table->size(1) : 0;
    p.table_len = some(table) ? (int32_t)table->size(0) : 0;
    p.dtype = code(q);
    p.eps = (float)eps;
    return laid(q, p.q_stride) && laid(k, p.k_stride) && slotscan_norm_rope_check(&p) == SLOTSCAN_OK;
}

std::tuple<Tensor, Tensor> norm_fwd(const slotscan_norm_params& p, const Tensor& q, const Tensor& k, const Maybe& table, const Maybe& pos, const Maybe& qw,
                                    const Maybe& kw) {
    const c10::cuda::CUDAGuard here(q.device());
    Tensor qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), k.options());
    check(slotscan_norm_rope_fwd(&p, in(q), in(k), ptr<float>(table), ptr<int32_t>(pos), ptr<float>(qw), ptr<float>(kw), out(qo), out(ko), stream_of(q)),
          "slotscan_norm_rope_fwd");
    return {qo, ko};
}

struct NormRope : torch::autograd::Function<NormRope> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Maybe& table, const Maybe& pos, const Maybe& qw, const Maybe& kw,
                                 double eps) {
        slotscan_norm_params p;
        norm_params(p, q, k, table, qw, kw, eps);
        ctx->save_for_backward({q, k, table.value_or(Tensor()), pos.value_or(Tensor()), qw.value_or(Tensor()), kw.value_or(Tensor())});
        ctx->saved_data["eps"] = eps;
        auto [qo, ko] = norm_fwd(p, q, k, table, pos, qw, kw);
        return {qo, ko};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1];
        const double eps = ctx->saved_data["eps"].toDouble();
        if (!first_order(grads)) {
            variable_list r = registered("slotscan::norm_rope_bwd", {q, k, or_none(s[2]), or_none(s[3]), or_none(s[4]), or_none(s[5]), grads[0], grads[1], eps});
            return {r[0], r[1], Tensor(), Tensor(), s[4].defined() ? r[2] : Tensor(), s[5].defined() ? r[3] : Tensor(), Tensor()};
        }
        slotscan_norm_params p;
        const Maybe table = maybe(s[2]), pos = maybe(s[3]), qw = maybe(s[4]), kw = maybe(s[5]);
        TORCH_CHECK(norm_params(p, q, k, table, qw, kw, eps), "norm_rope: a tensor saved for the backward has been changed");
        const c10::cuda::CUDAGuard here(q.device());
        const Tensor gq = whole(grads[0], q.scalar_type()), gk = whole(grads[1], k.scalar_type());
        Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dqw, dkw, scratch;
        size_t bytes = 0;
        if (some(qw) || some(kw)) {
            bytes = slotscan_norm_rope_bwd_scratch_bytes(&p);
            const auto f32 = q.options().dtype(at::kFloat);
            dqw = at::empty({q.size(3)}, f32);
            dkw = at::empty({q.size(3)}, f32);
            scratch = at::empty({(int64_t)(bytes / sizeof(float))}, f32);
        }
        check(slotscan_norm_rope_bwd(&p, in(q), in(k), ptr<float>(table), ptr<int32_t>(pos), ptr<float>(qw), ptr<float>(kw), in(gq), in(gk), out(dq), out(dk),
                                     (float*)out(dqw), (float*)out(dkw), out(scratch), bytes, stream_of(q)),
              "slotscan_norm_rope_bwd");
        return {dq, dk, Tensor(), Tensor(), some(qw) ? dqw : Tensor(), some(kw) ? dkw : Tensor(), Tensor()};
    }
};

py::object norm_rope(const Tensor& q, const Tensor& k, const Maybe& table, const Maybe& qw, const Maybe& kw, const Maybe& any_pos, double eps) {
    slotscan_norm_params p;
    const Maybe pos = in_32_bits(any_pos);
    if (!norm_params(p, q, k, table, qw, kw, eps) || !fits(pos, at::kInt, {q.size(0), q.size(1)}, q)) return py::none();
    if (some(table) && !some(pos) && q.size(1) > table->size(0)) return py::none();
    if (some(table) && (uintptr_t)table->const_data_ptr() % 16) return py::none();
    if ((some(qw) && (uintptr_t)qw->const_data_ptr() % 16) || (some(kw) && (uintptr_t)kw->const_data_ptr() % 16)) return py::none();
    const Maybe mq(q), mk(k);
    if (wants_grad({&mq, &mk, &qw, &kw, &table})) {
        const variable_list r = NormRope::apply(q, k, table, pos, qw, kw, eps);
        return py::cast(std::make_tuple(r[0], r[1]));
    }
    return py::cast(norm_fwd(p, q, k, table, pos, qw, kw));
}

py::object norm_rope_append(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& kc, const Tensor& vc, const Tensor& any_pos, const Maybe& table,
                            const Maybe& qw, const Maybe& kw, double eps) {
    slotscan_append_params p;
    const Tensor pos = in_32_bits(any_pos);
    if (!norm_params(p.base, q, k, table, qw, kw, eps)) return py::none();
    const int64_t B = q.size(0), T = q.size(1), D = q.size(3), KV = k.size(2);
    if (v.sizes() != k.sizes() || v.scalar_type() != q.scalar_type() || v.device() != q.device() || kc.dim() != 4 || vc.sizes() != kc.sizes() ||
        kc.scalar_type() != q.scalar_type() || vc.scalar_type() != q.scalar_type() || kc.device() != q.device() || vc.device() != q.device())
        return py::none();
    const int64_t L = kc.size(1);
    if (kc.size(0) != B || kc.size(2) != KV || kc.size(3) != D || T > L || L > 0x7fffffff || !fits(pos, at::kInt, {B}, q)) return py::none();
    const Maybe ts[] = {q, k, v, kc, vc, pos};
    if (wants_grad({&ts[0], &ts[1], &ts[2], &ts[3], &ts[4], &ts[5], &table, &qw, &kw})) return py::none();
    if (!laid(v, p.v_stride) || !laid(kc, p.kc_stride) || !laid(vc, p.vc_stride)) return py::none();
    if ((some(table) && (uintptr_t)table->const_data_ptr() % 16) || (some(qw) && (uintptr_t)qw->const_data_ptr() % 16) ||
        (some(kw) && (uintptr_t)kw->const_data_ptr() % 16))
        return py::none();
    p.L = (int32_t)L;
    const c10::cuda::CUDAGuard here(q.device());
    Tensor qo = at::empty(q.sizes(), q.options());
    check(slotscan_norm_rope_append(&p, in(q), in(k), in(v), ptr<float>(table), ptr<int32_t>(pos), ptr<float>(qw), ptr<float>(kw), out(qo), out(kc), out(vc),
                                    stream_of(q)),
          "slotscan_norm_rope_append");
    changed(kc);
    changed(vc);
    return py::cast(qo);
}

// ---- attention ----
bool attn_params(slotscan_attn_params& p, const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& slopes, const Maybe& docs, const Maybe& prefix,
                 int64_t window, double cap, double scale) {
    if (q.dim() != 4 || k.dim() != 4 || code(q) < 0 || code(k) != code(q) || code(v) != code(q) || !q.is_cuda() || k.device() != q.device() ||
        v.device() != q.device() || v.sizes() != k.sizes())
        return false;
    const int64_t B = q.size(0), Tq = q.size(1), H = q.size(2), D = q.size(3), Tk = k.size(1), KV = k.size(2);
    if (k.size(0) != B || k.size(3) != D || KV == 0 || H % KV || Tq > Tk || std::max({B, Tk, H, D, window}) > 0x7fffffff) return false;
    if (!fits(slopes, at::kFloat, {H}, q) || !fits(docs, at::kInt, {B, Tk, 2}, q) || !fits(prefix, at::kInt, {B}, q)) return false;
    if (some(docs) && (uintptr_t)docs->const_data_ptr() % 8) return false;
    p.B = (int32_t)B; p.Tq = (int32_t)Tq; p.Tk = (int32_t)Tk; p.H = (int32_t)H; p.KV = (int32_t)KV; p.D = (int32_t)D;
    p.window = (int32_t)window;
    p.dtype = code(q);
    p.scale = (float)scale;
    p.cap = (float)cap;
    return laid(q, p.q_stride) && laid(k, p.k_stride) && laid(v, p.v_stride) && slotscan_attn_check(&p) == SLOTSCAN_OK;
}
// o, and with `keep` what the backward needs: lse, rest
variable_list attn_fwd(const slotscan_attn_params& p, const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& slopes, const Maybe& docs,
                       const Maybe& prefix, bool keep) {
    const c10::cuda::CUDAGuard here(q.device());
    Tensor o = at::empty(q.sizes(), q.options()), lse, rest;
    if (keep) {
        lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
        if (p.dtype == SLOTSCAN_BF16) rest = at::empty(q.sizes(), q.options());
    }
    check(slotscan_attn_fwd(&p, in(q), in(k), in(v), ptr<float>(slopes), ptr<int32_t>(docs), ptr<int32_t>(prefix), out(o), out(rest), (float*)out(lse),
                            stream_of(q)),
          "slotscan_attn_fwd");
    return {o, lse, rest};
}

struct TokenAttention : torch::autograd::Function<TokenAttention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& slopes, const Maybe& docs, const Maybe& prefix,
                          int64_t window, double cap, double scale) {
        slotscan_attn_params p;
        attn_params(p, q, k, v, slopes, docs, prefix, window, cap, scale);
        const bool keep = slotscan_attn_keeps(&p, some(prefix));
        const variable_list r = attn_fwd(p, q, k, v, slopes, docs, prefix, keep);
        ctx->save_for_backward({q, k, v, slopes.value_or(Tensor()), docs.value_or(Tensor()), prefix.value_or(Tensor()), keep ? r[0] : Tensor(), r[1], r[2]});
        ctx->saved_data["window"] = window;
        ctx->saved_data["cap"] = cap;
        ctx->saved_data["scale"] = scale;
        return r[0];
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2];
        const int64_t window = ctx->saved_data["window"].toInt();
        const double cap = ctx->saved_data["cap"].toDouble(), scale = ctx->saved_data["scale"].toDouble();
        const Tensor none;
        if (!first_order(grads)) {
            const auto or_empty = [&](const Tensor& t, at::ScalarType type) { return t.defined() ? t : at::empty({0}, q.options().dtype(type)); };
            variable_list r = registered("slotscan::attn_bwd", {q, k, v, or_none(s[3]), or_none(s[4]), or_none(s[5]), or_empty(s[6], q.scalar_type()),
                                                               or_empty(s[7], at::kFloat), or_empty(s[8], q.scalar_type()), grads[0], window, cap, scale});
            return {r[0], r[1], r[2], none, none, none, none, none, none};
        }
        slotscan_attn_params p;
        const Maybe slopes = maybe(s[3]), docs = maybe(s[4]), prefix = maybe(s[5]);
        TORCH_CHECK(attn_params(p, q, k, v, slopes, docs, prefix, window, cap, scale), "token_attention: a tensor saved for the backward has been changed");
        const c10::cuda::CUDAGuard here(q.device());
        const Tensor g = whole(grads[0], q.scalar_type());
        Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(k.sizes(), k.options()), delta;
        if (s[7].defined()) delta = at::empty(s[7].sizes(), s[7].options());
        check(slotscan_attn_bwd(&p, in(q), in(k), in(v), ptr<float>(slopes), ptr<int32_t>(docs), ptr<int32_t>(prefix), ptr<void>(maybe(s[6])),
                                ptr<void>(maybe(s[8])), ptr<float>(maybe(s[7])), in(g), (float*)out(delta), out(dq), out(dk), out(dv), stream_of(q)),
              "slotscan_attn_bwd");
        return {dq, dk, dv, none, none, none, none, none, none};
    }
};

py::object token_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& slopes, const Maybe& any_docs, const Maybe& any_prefix,
                           int64_t window, double cap, double scale) {
    slotscan_attn_params p;
    const Maybe docs = in_32_bits(any_docs), prefix = in_32_bits(any_prefix);
    if (!attn_params(p, q, k, v, slopes, docs, prefix, window, cap, scale)) return py::none();
    const Maybe ts[] = {q, k, v};
    if (wants_grad({&ts[0], &ts[1], &ts[2]})) return py::cast(TokenAttention::apply(q, k, v, slopes, docs, prefix, window, cap, scale));
    return py::cast(attn_fwd(p, q, k, v, slopes, docs, prefix, false)[0]);
}

py::object token_attention_step(const Tensor& q, const Tensor& kc, const Tensor& vc, const Tensor& any_pos, const Maybe& slopes, const Maybe& any_start,
                                int64_t window, double cap, double scale) {
    const Tensor pos = in_32_bits(any_pos);
    const Maybe start = in_32_bits(any_start);
    if (q.dim() != 4 || q.size(1) != 1 || kc.dim() != 4 || vc.sizes() != kc.sizes() || code(q) < 0 || code(kc) != code(q) || code(vc) != code(q) ||
        !q.is_cuda() || kc.device() != q.device() || vc.device() != q.device())
        return py::none();
    const int64_t B = q.size(0), H = q.size(2), D = q.size(3), L = kc.size(1), KV = kc.size(2);
    if (kc.size(0) != B || kc.size(3) != D || KV == 0 || H % KV || std::max({B, H, D, L, window}) > 0x7fffffff) return py::none();
    if (!fits(pos, at::kInt, {B}, q) || !fits(start, at::kInt, {B}, q) || !fits(slopes, at::kFloat, {H}, q)) return py::none();
    const Maybe ts[] = {q, kc, vc, pos};
    if (wants_grad({&ts[0], &ts[1], &ts[2], &ts[3], &slopes, &start})) return py::none();
    slotscan_attn_step_params p;
    int64_t qs[3];
    if (!laid(q, qs) || !laid(kc, p.k_stride) || !laid(vc, p.v_stride)) return py::none();
    p.B = (int32_t)B; p.H = (int32_t)H; p.KV = (int32_t)KV; p.D = (int32_t)D; p.L = (int32_t)L;
    p.window = (int32_t)window;
    p.dtype = code(q);
    p.scale = (float)scale;
    p.cap = (float)cap;
    p.q_stride[0] = qs[0];
    p.q_stride[1] = qs[2];
    if (slotscan_attn_step_check(&p) != SLOTSCAN_OK) return py::none();
    const c10::cuda::CUDAGuard here(q.device());
    Tensor o = at::empty(q.sizes(), q.options()), scratch;
    const size_t bytes = slotscan_attn_step_scratch_bytes(&p);
    if (bytes) scratch = at::empty({(int64_t)(bytes / sizeof(float))}, q.options().dtype(at::kFloat));
    check(slotscan_attn_step(&p, in(q), in(kc), in(vc), ptr<int32_t>(pos), ptr<int32_t>(start), ptr<float>(slopes), out(o), out(scratch), bytes, stream_of(q)),
          "slotscan_attn_step");
    return py::cast(o);
}

// ---- pages ----
// rows of integers side by side, in place
bool table_laid(const Tensor& t, const Tensor& like, int64_t B) {
    return t.dim() == 2 && t.scalar_type() == at::kInt && t.device() == like.device() && t.size(0) == B && t.size(1) > 0 && t.size(1) <= 0x7fffffff &&
           (t.size(1) == 1 || t.stride(1) == 1) && (B <= 1 || t.stride(0) >= t.size(1));
}
int64_t table_stride(const Tensor& t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }
bool ints(const Tensor& t, int64_t n, const Tensor& like) { return t.dim() == 1 && t.size(0) == n && fits(Maybe(t), at::kInt, {n}, like); }

// `n` elements of `t` from the `from`-th on, as a tensor of its own that shares the memory
Tensor part_of(const Tensor& t, int64_t from, int64_t n) {
    Tensor r = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(t.storage()), t.key_set(), t.dtype());
    r.unsafeGetTensorImpl()->set_storage_offset(from);
    r.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    return r;
}

bool pages_params(slotscan_pages_params& p, const Tensor& lengths, const Tensor& tables, const Tensor& free_pages, const Tensor& n_free, int64_t page, int64_t tokens) {
    if (!lengths.is_cuda() || lengths.dim() != 1 || free_pages.dim() != 1) return false;
    const int64_t B = lengths.size(0);
    if (!ints(lengths, B, lengths) || !ints(free_pages, free_pages.size(0), lengths) || !ints(n_free, 1, lengths) || !table_laid(tables, lengths, B)) return false;
    if (std::max({B, free_pages.size(0), page, tokens}) > 0x7fffffff || page < 0 || tokens < 0) return false;
    const Maybe ts[] = {lengths, tables, free_pages, n_free};
    if (wants_grad({&ts[0], &ts[1], &ts[2], &ts[3]})) return false;
    p.B = (int32_t)B; p.M = (int32_t)tables.size(1); p.page = (int32_t)page; p.pages = (int32_t)free_pages.size(0); p.tokens = (int32_t)tokens;
    p.table_stride = table_stride(tables);
    return slotscan_pages_check(&p) == SLOTSCAN_OK;
}

py::object extend_pages(const Tensor& any_new, const Tensor& lengths, const Tensor& tables, const Tensor& free_pages, const Tensor& n_free, int64_t page,
                        int64_t tokens) {
    slotscan_pages_params p;
    const Tensor fresh = in_32_bits(any_new);
    if (!pages_params(p, lengths, tables, free_pages, n_free, page, tokens) || !ints(fresh, p.B, lengths)) return py::none();
    const c10::cuda::CUDAGuard here(lengths.device());
    // the results and the scratch lie in one allocation: five of them were a third of a small call's host time
    const size_t bytes = slotscan_pages_scratch_bytes(&p);
    const int64_t sizes[] = {tokens, tokens, p.B + 1, p.B, (int64_t)(bytes / sizeof(int32_t))};
    int64_t at[6] = {0};
    for (int i = 0; i < 5; i++) at[i + 1] = at[i] + (sizes[i] + 3) / 4 * 4;        // each on 16 bytes
    const Tensor all = at::empty({at[5]}, lengths.options());
    const Tensor slots = part_of(all, at[0], sizes[0]), pos = part_of(all, at[1], sizes[1]), starts = part_of(all, at[2], sizes[2]),
                 taken = part_of(all, at[3], sizes[3]), scratch = part_of(all, at[4], sizes[4]);
    check(slotscan_extend_pages(&p, (const int32_t*)in(fresh), (int32_t*)out(lengths), (int32_t*)out(tables), (int32_t*)out(free_pages), (int32_t*)out(n_free),
                                (int32_t*)out(slots), (int32_t*)out(pos), (int32_t*)out(starts), (int32_t*)out(taken), out(scratch), bytes, stream_of(lengths)),
          "slotscan_extend_pages");
    for (const Tensor& t : {lengths, tables, free_pages, n_free}) changed(t);
    return py::cast(std::make_tuple(slots, pos, starts, taken));
}

bool release_pages(const Tensor& done, const Tensor& lengths, const Tensor& tables, const Tensor& free_pages, const Tensor& n_free, int64_t page) {
    slotscan_pages_params p;
    if (!pages_params(p, lengths, tables, free_pages, n_free, page, 0) || done.dim() != 1 || done.size(0) != p.B || done.device() != lengths.device() ||
        (done.scalar_type() != at::kBool && done.scalar_type() != at::kByte) || !done.is_contiguous())
        return false;
    const c10::cuda::CUDAGuard here(lengths.device());
    const size_t bytes = slotscan_pages_scratch_bytes(&p);
    Tensor scratch = at::empty({(int64_t)(bytes / sizeof(int32_t))}, lengths.options());
    check(slotscan_release_pages(&p, (const uint8_t*)in(done), (int32_t*)out(lengths), (int32_t*)out(tables), (int32_t*)out(free_pages), (int32_t*)out(n_free),
                                 out(scratch), bytes, stream_of(lengths)),
          "slotscan_release_pages");
    for (const Tensor& t : {lengths, tables, free_pages, n_free}) changed(t);
    return true;
}

py::object norm_rope_pages(const Tensor& q3, const Tensor& k3, const Tensor& v3, const Tensor& kp, const Tensor& vp, const Tensor& any_slots, const Tensor& any_pos,
                           const Maybe& table, const Maybe& qw, const Maybe& kw, double eps) {
    if (q3.dim() != 3 || k3.dim() != 3 || v3.dim() != 3) return py::none();
    slotscan_page_append_params p;
    const Tensor q = q3.unsqueeze(0), k = k3.unsqueeze(0), v = v3.unsqueeze(0), slots = in_32_bits(any_slots), pos = in_32_bits(any_pos);
    if (!norm_params(p.base, q, k, table, qw, kw, eps)) return py::none();
    const int64_t N = q.size(1), D = q.size(3), KV = k.size(2);
    if (v.sizes() != k.sizes() || code(v) != code(q) || v.device() != q.device() || kp.dim() != 4 || vp.sizes() != kp.sizes() || code(kp) != code(q) ||
        code(vp) != code(q) || kp.device() != q.device() || vp.device() != q.device() || kp.size(2) != KV || kp.size(3) != D ||
        std::max(kp.size(0), kp.size(1)) > 0x7fffffff || !ints(slots, N, q) || !ints(pos, N, q))
        return py::none();
    const Maybe ts[] = {q3, k3, v3, kp, vp};
    if (wants_grad({&ts[0], &ts[1], &ts[2], &ts[3], &ts[4], &table, &qw, &kw})) return py::none();
    if (!laid(v, p.v_stride) || !laid(kp, p.kp_stride) || !laid(vp, p.vp_stride)) return py::none();
    if ((some(table) && (uintptr_t)table->const_data_ptr() % 16) || (some(qw) && (uintptr_t)qw->const_data_ptr() % 16) ||
        (some(kw) && (uintptr_t)kw->const_data_ptr() % 16))
        return py::none();
    p.pages = (int32_t)kp.size(0);
    p.page = (int32_t)kp.size(1);
    if (p.pages < 1 || p.page < 8 || p.page > 1024 || (p.page & (p.page - 1)) || (int64_t)p.pages * p.page > INT32_MAX) return py::none();
    const c10::cuda::CUDAGuard here(q.device());
    Tensor qo = at::empty(q3.sizes(), q3.options());
    check(slotscan_norm_rope_pages(&p, in(q), in(k), in(v), ptr<float>(table), (const int32_t*)in(slots), (const int32_t*)in(pos), ptr<float>(qw), ptr<float>(kw),
                                   out(qo), out(kp), out(vp), stream_of(q)),
          "slotscan_norm_rope_pages");
    changed(kp);
    changed(vp);
    return py::cast(qo);
}

// q: (N, 1, H, D), a row for each request (starts absent), or (N, H, D)
py::object paged_attention(const Tensor& q, const Tensor& kp, const Tensor& vp, const Tensor& any_tables, const Maybe& any_starts, const Tensor& any_pos,
                           const Maybe& slopes, const Maybe& any_start, int64_t window, double cap, double scale) {
    const bool step = !some(any_starts);
    const Tensor tables = in_32_bits(any_tables), pos = in_32_bits(any_pos);
    const Maybe starts = in_32_bits(any_starts), start = in_32_bits(any_start);
    if (q.dim() != (step ? 4 : 3) || (step && q.size(1) != 1) || kp.dim() != 4 || vp.sizes() != kp.sizes() || code(q) < 0 || code(kp) != code(q) ||
        code(vp) != code(q) || !q.is_cuda() || kp.device() != q.device() || vp.device() != q.device())
        return py::none();
    const int64_t N = q.size(0), H = q.size(-2), D = q.size(-1), KV = kp.size(2), B = step ? N : starts->numel() - 1;
    if (kp.size(3) != D || KV == 0 || H % KV || std::max({N, H, D, kp.size(0), kp.size(1), window}) > 0x7fffffff || B < 0) return py::none();
    if (!table_laid(tables, q, B) || !ints(pos, N, q) || !fits(starts, at::kInt, {B + 1}, q) || !fits(start, at::kInt, {B}, q) || !fits(slopes, at::kFloat, {H}, q))
        return py::none();
    const Maybe ts[] = {q, kp, vp, tables, pos};
    if (wants_grad({&ts[0], &ts[1], &ts[2], &ts[3], &ts[4], &slopes, &start})) return py::none();
    slotscan_paged_params p;
    int64_t qs[3];
    if (!laid(q, qs) || !laid(kp, p.k_stride) || !laid(vp, p.v_stride)) return py::none();
    p.N = (int32_t)N; p.B = (int32_t)B; p.H = (int32_t)H; p.KV = (int32_t)KV; p.D = (int32_t)D;
    p.pages = (int32_t)kp.size(0); p.page = (int32_t)kp.size(1); p.M = (int32_t)tables.size(1);
    p.window = (int32_t)window;
    p.dtype = code(q);
    p.scale = (float)scale;
    p.cap = (float)cap;
    p.q_stride[0] = qs[0];
    p.q_stride[1] = qs[step ? 2 : 1];
    p.table_stride = table_stride(tables);
    if (slotscan_paged_check(&p) != SLOTSCAN_OK) return py::none();
    const c10::cuda::CUDAGuard here(q.device());
    Tensor o = at::empty(q.sizes(), q.options()), scratch;
    const size_t bytes = step ? slotscan_paged_step_scratch_bytes(&p) : slotscan_paged_attn_scratch_bytes(&p);
    if (bytes) scratch = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    if (step)
        check(slotscan_paged_step(&p, in(q), in(kp), in(vp), (const int32_t*)in(tables), (const int32_t*)in(pos), ptr<int32_t>(start), ptr<float>(slopes), out(o),
                                  out(scratch), bytes, stream_of(q)),
              "slotscan_paged_step");
    else
        check(slotscan_paged_attn(&p, in(q), in(kp), in(vp), (const int32_t*)in(tables), ptr<int32_t>(starts), (const int32_t*)in(pos), ptr<int32_t>(start),
                                  ptr<float>(slopes), out(o), out(scratch), bytes, stream_of(q)),
              "slotscan_paged_attn");
    return py::cast(o);
}

}  // namespace

PYBIND11_MODULE(_tokens_host, m) {
    m.def("norm_rope", &norm_rope);
    m.def("norm_rope_append", &norm_rope_append);
    m.def("token_attention", &token_attention);
    m.def("token_attention_step", &token_attention_step);
    m.def("extend_pages", &extend_pages);
    m.def("release_pages", &release_pages);
    m.def("norm_rope_pages", &norm_rope_pages);
    m.def("paged_attention", &paged_attention);
}
