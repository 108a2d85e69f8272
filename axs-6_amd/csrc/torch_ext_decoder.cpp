// The decoder's operators in the torch extension: rotary positions, attention,
// the 8-bit cache and the distillation loss, each as argument checks, outputs,
// workspaces and an autograd node over the C ABI (include/axs6.h).
//
// Tensors are float32, bfloat16 or float16 on one GPU; anything else raises.
// Views are taken as they are where a head's values are adjacent and the
// kernels' 16-byte accesses are aligned, else copied.
#include <cmath>
#include <optional>

#include "torch_ext_common.h"

namespace axs6_ext {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<at::Tensor>;

bool given(const OptTensor& t) { return t && t->defined(); }

// Whether a call on t goes through its autograd node: for a gradient, or for a forward-mode
// tangent, which the node refuses (there is no such derivative) and no call may drop.
bool records(const at::Tensor& t) {
    return t.defined() && ((at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined());
}

void check_dtype(const at::Tensor& t, const char* fn, const char* name) {
    TORCH_CHECK(dtype_code(t.scalar_type()) >= 0, fn, ": ", name, " has dtype ", t.scalar_type(),
                ", not float32, bfloat16 or float16");
}

// t: a tensor of `dims` dims on the device and of the dtype of `like`.
void check_like(const at::Tensor& t, const at::Tensor& like, int64_t dims, const char* fn, const char* name) {
    require_device(t, fn);
    TORCH_CHECK(t.dim() == dims, fn, ": ", name, " must have ", dims, " dims, got ", t.dim());
    TORCH_CHECK(t.device() == like.device(), fn, ": ", name, " is on ", t.device(), ", not ", like.device());
    TORCH_CHECK(t.scalar_type() == like.scalar_type(), fn, ": ", name, " has dtype ", t.scalar_type(), ", not ",
                like.scalar_type());
}

bool aligned(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// The last dim's values adjacent.
at::Tensor packed_last(const at::Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

// (B, T, H, D) with whole aligned 16-byte vectors: zeros after a D that is not.
at::Tensor vectors(const at::Tensor& t) {
    const int64_t v = vec_multiple(t.scalar_type()), d = t.size(3), pad = (v - d % v) % v;
    if (pad) return at::constant_pad_nd(t, {0, pad});
    if (t.numel() == 0) return t;
    // a dim of one element is never walked: its stride may be anything, and the kernels get d
    bool ok = t.stride(3) == 1, same = true;
    std::vector<int64_t> strides = t.strides().vec();
    for (int i = 0; i < 3; ++i) {
        if (t.size(i) == 1) {
            same = same && strides[i] % v == 0 && strides[i] < AXS6_ATTENTION_MAX_TOKEN_STRIDE;
            strides[i] = d;
        }
        ok = ok && strides[i] % v == 0;
    }
    if (!ok || strides[1] >= AXS6_ATTENTION_MAX_TOKEN_STRIDE) return t.contiguous();
    if (!aligned(t)) return t.clone(at::MemoryFormat::Contiguous);
    return same ? t : t.as_strided(t.sizes(), strides);
}

at::Tensor int64s(const at::Tensor& t, at::IntArrayRef shape, const at::Tensor& like, const char* fn, const char* name) {
    require_device(t, fn);
    TORCH_CHECK(t.device() == like.device() && t.sizes() == shape, fn, ": ", name, " must be of shape ", shape, " on ",
                like.device(), ", got ", t.sizes(), " on ", t.device());
    TORCH_CHECK(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, fn, ": ", name,
                " must be int64 or int32, got ", t.scalar_type());
    return t.to(at::kLong).contiguous();
}

// `bytes` of workspace beside `like`; undefined for 0.
at::Tensor workspace(int64_t bytes, const at::Tensor& like) {
    return bytes ? at::empty({bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}
void* data_of(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
int64_t size_of(const at::Tensor& t) { return t.defined() ? t.numel() : 0; }

// ---- rotary positions ---------------------------------------------------------------

struct Rotary {
    at::Tensor table, positions;
    bool interleaved;
};

// q, k: undefined, or (B, T, H, D).
std::pair<at::Tensor, at::Tensor> rotate(const at::Tensor& q, const at::Tensor& k, const Rotary& r, bool inverse) {
    const char* fn = "axs6_rotary";
    const at::Tensor& any = q.defined() ? q : k;
    c10::DeviceGuard guard(any.device());
    const at::Tensor qc = q.defined() ? packed_last(q) : q, kc = k.defined() ? packed_last(k) : k;
    at::Tensor qo, ko;
    if (q.defined()) qo = at::empty(q.sizes(), q.options());
    if (k.defined()) ko = at::empty(k.sizes(), k.options());
    const int64_t T = any.size(1);
    const at::Tensor& p = r.positions;
    check_rc(axs6_rotary(q.defined() ? qc.data_ptr() : nullptr, k.defined() ? kc.data_ptr() : nullptr,
                         q.defined() ? qo.data_ptr() : nullptr, k.defined() ? ko.data_ptr() : nullptr,
                         dtype_code(any.scalar_type()), any.size(0), T, q.defined() ? q.size(2) : 0,
                         k.defined() ? k.size(2) : 0, any.size(3), r.table.size(1),
                         q.defined() ? qc.strides().data() : nullptr, k.defined() ? kc.strides().data() : nullptr,
                         r.table.data_ptr<float>(), r.table.size(0), p.defined() ? p.data_ptr<int64_t>() : nullptr,
                         p.defined() && p.dim() == 2 && p.size(0) > 1 ? p.stride(0) : 0,
                         p.defined() ? p.stride(-1) : 0, r.interleaved, inverse, stream_of(any)),
             fn);
    return {qo, ko};
}

struct RotaryFunction : public torch::autograd::Function<RotaryFunction> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& table,
                                 const at::Tensor& positions, bool interleaved, bool has_k, bool has_p) {
        auto [qo, ko] = rotate(q, has_k ? k : at::Tensor(), {table, has_p ? positions : at::Tensor(), interleaved}, false);
        ctx->save_for_backward({table, has_p ? positions : at::Tensor()});
        ctx->saved_data["interleaved"] = interleaved;
        if (!has_k) return {qo};
        return {qo, ko};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const at::Tensor gq = ctx->needs_input_grad(0) ? grads[0] : at::Tensor();
        const at::Tensor gk = grads.size() > 1 && ctx->needs_input_grad(1) ? grads[1] : at::Tensor();
        variable_list out(7);
        if (gq.defined() || gk.defined()) {
            auto [dq, dk] = rotate(gq, gk, {saved[0], saved[1], ctx->saved_data["interleaved"].toBool()}, true);
            out[0] = dq;
            out[1] = dk;
        }
        return out;
    }
};

py::object rotary(const at::Tensor& q, const OptTensor& k, const at::Tensor& table, const OptTensor& positions,
                  bool interleaved) {
    const char* fn = "axs_rotary_unified";
    require_device(q, fn);
    check_dtype(q, fn, "q");
    TORCH_CHECK(q.dim() == 4, fn, ": q must be (B, T, heads, D), got ", q.dim(), " dims");
    const int64_t B = q.size(0), T = q.size(1), D = q.size(3);
    if (given(k)) {
        check_like(*k, q, 4, fn, "k");
        TORCH_CHECK(k->size(0) == B && k->size(1) == T && k->size(3) == D, fn, ": q is ", q.sizes(), " but k ",
                    k->sizes());
    }
    require_device(table, fn);
    TORCH_CHECK(table.dim() == 2 && table.scalar_type() == at::kFloat && table.device() == q.device(), fn,
                ": the table must be (positions, rotated values) float32 on q's device");
    TORCH_CHECK(table.size(1) % 2 == 0 && table.size(1) <= D, fn, ": the table's ", table.size(1),
                " values are not an even part of the head's ", D);
    TORCH_CHECK(!table.requires_grad(), fn, ": the table takes no gradient");
    const at::Tensor tab = table.contiguous();
    at::Tensor pos;
    if (given(positions)) {
        require_device(*positions, fn);
        TORCH_CHECK(positions->device() == q.device(), fn, ": positions are on ", positions->device());
        TORCH_CHECK(positions->scalar_type() == at::kLong || positions->scalar_type() == at::kInt, fn,
                    ": positions must be int64 or int32, got ", positions->scalar_type());
        TORCH_CHECK((positions->dim() == 1 && positions->size(0) == T) ||
                        (positions->dim() == 2 && positions->size(1) == T &&
                         (positions->size(0) == B || positions->size(0) == 1)),
                    fn, ": positions must be (T) or (B, T) for q ", q.sizes(), ", got ", positions->sizes());
        pos = positions->to(at::kLong);
    } else {
        TORCH_CHECK(T <= tab.size(0), fn, ": ", T, " tokens for a table of ", tab.size(0), " positions");
    }
    if (records(q) || (given(k) && records(*k))) {
        // absent tensors travel as empty ones: the node records every argument's device
        const at::Tensor none = at::empty({0}, q.options());
        variable_list r = RotaryFunction::apply(q, given(k) ? *k : none, tab, pos.defined() ? pos : none, interleaved,
                                                given(k), pos.defined());
        return given(k) ? py::cast(std::make_tuple(r[0], r[1])) : py::object(py::make_tuple(r[0], py::none()));
    }
    auto [qo, ko] = rotate(q, given(k) ? *k : at::Tensor(), {tab, pos, interleaved}, false);
    return given(k) ? py::cast(std::make_tuple(qo, ko)) : py::object(py::make_tuple(qo, py::none()));
}

// ---- attention ------------------------------------------------------------------------

struct Mask {
    at::Tensor t;
    int type = 0;
    int64_t strides[4] = {0, 0, 0, 0};
    const void* data() const { return t.defined() ? t.data_ptr() : nullptr; }
};

Mask mask_of(const at::Tensor& t, int64_t B, int64_t Hq, int64_t Tq, int64_t Tk) {
    Mask m;
    if (!t.defined()) return m;
    m.t = t;
    m.type = t.scalar_type() == at::kBool ? -1 : dtype_code(t.scalar_type());
    const int64_t want[4] = {B, Hq, Tq, Tk}, skip = 4 - t.dim();
    for (int64_t i = skip; i < 4; ++i) m.strides[i] = t.size(i - skip) == 1 && want[i] != 1 ? 0 : t.stride(i - skip);
    return m;
}

// The kernels' out and, for the backward, row statistics of operands of whole vectors.
std::pair<at::Tensor, at::Tensor> attention_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                const at::Tensor& mask, bool causal, double scale, bool stats) {
    const int64_t B = q.size(0), Tq = q.size(1), Hq = q.size(2), D = q.size(3), Tk = k.size(1), H = k.size(2);
    const Mask m = mask_of(mask, B, Hq, Tq, Tk);
    at::Tensor out = at::empty({B, Tq, Hq, D}, q.options());
    at::Tensor st = stats ? at::empty({B, Hq, Tq, 2}, q.options().dtype(at::kFloat)) : at::Tensor();
    const at::Tensor ws = workspace(axs6_attention_forward_workspace(B, Tq, Tk, Hq, D), q);
    check_rc(axs6_attention_forward(q.data_ptr(), k.data_ptr(), v.data_ptr(), dtype_code(q.scalar_type()), B, Tq, Tk, Hq,
                                    H, D, q.strides().data(), k.strides().data(), v.strides().data(), m.data(), m.type,
                                    m.strides, causal, (float)scale, out.data_ptr(),
                                    stats ? st.data_ptr<float>() : nullptr, data_of(ws), size_of(ws), stream_of(q)),
             "axs6_attention_forward");
    return {out, st};
}

struct AttentionFunction : public torch::autograd::Function<AttentionFunction> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                              const at::Tensor& mask, bool has_mask, bool causal, double scale) {
        c10::DeviceGuard guard(q.device());
        const at::Tensor qv = vectors(q), kv = vectors(k), vv = vectors(v), m = has_mask ? mask : at::Tensor();
        auto [out, stats] = attention_fwd(qv, kv, vv, m, causal, scale, true);
        ctx->save_for_backward({qv, kv, vv, out, stats, m});
        auto& d = ctx->saved_data;
        d["causal"] = causal;
        d["scale"] = scale;
        d["D"] = q.size(3);
        return out.size(3) == q.size(3) ? out : out.narrow(3, 0, q.size(3)).contiguous();
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list r(7);
        if (!grads[0].defined()) return r;
        const auto s = ctx->get_saved_variables();
        auto& d = ctx->saved_data;
        const at::Tensor &q = s[0], &k = s[1], &v = s[2], &out = s[3], &stats = s[4];
        const int64_t B = q.size(0), Tq = q.size(1), Hq = q.size(2), D = q.size(3), Tk = k.size(1), H = k.size(2);
        const int64_t D0 = d["D"].toInt();
        c10::DeviceGuard guard(q.device());
        const at::Tensor g = vectors(grads[0].to(q.scalar_type()));
        const Mask m = mask_of(s[5], B, Hq, Tq, Tk);
        at::Tensor dq = at::empty({B, Tq, Hq, D}, q.options()), dk = at::empty({B, Tk, H, D}, q.options());
        at::Tensor dv = at::empty({B, Tk, H, D}, q.options());
        const bool causal = d["causal"].toBool();
        // delta, then the workspace (whole 16 bytes each)
        const int64_t rows = (B * Hq * Tq + 3) / 4 * 4;
        const int64_t bytes = axs6_attention_backward_workspace(B, Tq, Tk, Hq, H, D, causal);
        const at::Tensor scratch = at::empty({rows + bytes / 4}, stats.options());
        float* delta = scratch.data_ptr<float>();
        check_rc(axs6_attention_backward(
                     g.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), stats.data_ptr<float>(),
                     dtype_code(q.scalar_type()), B, Tq, Tk, Hq, H, D, g.strides().data(), q.strides().data(),
                     k.strides().data(), v.strides().data(), m.data(), m.type, m.strides, causal,
                     (float)d["scale"].toDouble(), delta, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                     delta + rows, bytes, stream_of(q)),
                 "axs6_attention_backward");
        const at::Tensor got[3] = {dq, dk, dv};
        for (int i = 0; i < 3; ++i)
            if (ctx->needs_input_grad(i)) r[i] = D == D0 ? got[i] : got[i].narrow(3, 0, D0).contiguous();
        return r;
    }
};

at::Tensor attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const OptTensor& mask, bool causal,
                     std::optional<double> scale) {
    const char* fn = "axs_attention_unified";
    require_device(q, fn);
    check_dtype(q, fn, "q");
    TORCH_CHECK(q.dim() == 4, fn, ": q must be (B, Tq, heads, D), got ", q.dim(), " dims");
    check_like(k, q, 4, fn, "k");
    check_like(v, q, 4, fn, "v");
    const int64_t B = q.size(0), Tq = q.size(1), Hq = q.size(2), D = q.size(3), Tk = k.size(1), H = k.size(2);
    TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == B && k.size(3) == D, fn, ": q is ", q.sizes(), ", k ", k.sizes(),
                ", v ", v.sizes());
    TORCH_CHECK(H ? Hq % H == 0 : Hq == 0, fn, ": ", Hq, " query heads are not a multiple of ", H, " key heads");
    TORCH_CHECK(D >= 1 && D <= AXS6_ATTENTION_MAX_HEAD, fn, ": heads of 1 to ", AXS6_ATTENTION_MAX_HEAD,
                " values, got ", D);
    const double s = scale ? *scale : 1.0 / std::sqrt((double)D);
    TORCH_CHECK(s > 0.0 && std::isfinite((float)s) && (float)s > 0.0f, fn, ": the scale must be positive and finite, got ", s);
    if (given(mask)) {
        require_device(*mask, fn);
        TORCH_CHECK(mask->device() == q.device(), fn, ": the mask is on ", mask->device(), ", q on ", q.device());
        TORCH_CHECK(mask->scalar_type() == at::kBool || dtype_code(mask->scalar_type()) >= 0, fn,
                    ": the mask must be bool, float32, bfloat16 or float16, got ", mask->scalar_type());
        TORCH_CHECK(!mask->requires_grad(), fn, ": the mask takes no gradient");
        const int64_t want[4] = {B, Hq, Tq, Tk}, skip = 4 - mask->dim();
        bool ok = mask->dim() >= 1 && mask->dim() <= 4;
        for (int64_t i = skip; ok && i < 4; ++i) ok = mask->size(i - skip) == 1 || mask->size(i - skip) == want[i];
        TORCH_CHECK(ok, fn, ": a mask of shape ", mask->sizes(), " does not broadcast to (", B, ", ", Hq, ", ", Tq, ", ",
                    Tk, ")");
    }
    const at::Tensor m = given(mask) ? *mask : at::Tensor();
    if (records(q) || records(k) || records(v))
        return AttentionFunction::apply(q, k, v, m.defined() ? m : at::empty({0}, q.options()), m.defined(), causal, s);
    c10::DeviceGuard guard(q.device());
    at::Tensor out = attention_fwd(vectors(q), vectors(k), vectors(v), m, causal, s, false).first;
    return out.size(3) == D ? out : out.narrow(3, 0, D).contiguous();
}

// ---- the 8-bit cache ----------------------------------------------------------------------

struct Cache {
    const at::Tensor &kc, &ks, &vc, &vs, &kt, &vt;
    int64_t B, H, D, nb;
};

Cache cache_of(const at::Tensor& kc, const at::Tensor& ks, const at::Tensor& vc, const at::Tensor& vs,
               const at::Tensor& kt, const at::Tensor& vt, const char* fn) {
    require_device(kc, fn);
    TORCH_CHECK(kc.dim() == 5 && kc.size(3) == AXS6_KV_BLOCK, fn, ": k_codes must be (B, heads, blocks, ", AXS6_KV_BLOCK,
                ", D), got ", kc.sizes());
    const int64_t B = kc.size(0), H = kc.size(1), nb = kc.size(2), D = kc.size(4);
    TORCH_CHECK(D % 16 == 0 && D > 0 && D <= AXS6_KV_MAX_HEAD, fn, ": heads of a multiple of 16 values up to ",
                AXS6_KV_MAX_HEAD, ", got ", D);
    auto check = [&](const at::Tensor& t, const char* name, at::ScalarType dt, at::IntArrayRef shape) {
        TORCH_CHECK(t.sizes() == shape && t.scalar_type() == dt && t.device() == kc.device(), fn, ": ", name,
                    " must be ", dt, " ", shape, " on ", kc.device(), ", got ", t.scalar_type(), " ", t.sizes(), " on ",
                    t.device());
        TORCH_CHECK(t.is_contiguous() && aligned(t), fn, ": ", name, " must be contiguous and aligned to 16 bytes");
    };
    check(kc, "k_codes", at::kChar, {B, H, nb, AXS6_KV_BLOCK, D});
    check(vc, "v_codes", at::kChar, {B, H, nb, D, AXS6_KV_BLOCK});
    check(ks, "k_scales", at::kFloat, {B, H, nb});
    check(vs, "v_scales", at::kFloat, {B, H, nb});
    check_dtype(kt, fn, "k_tail");
    check(kt, "k_tail", kt.scalar_type(), {B, H, AXS6_KV_BLOCK, D});
    check(vt, "v_tail", kt.scalar_type(), {B, H, AXS6_KV_BLOCK, D});
    return {kc, ks, vc, vs, kt, vt, B, H, D, nb};
}

void kv_append(const at::Tensor& k_codes, const at::Tensor& k_scales, const at::Tensor& v_codes,
               const at::Tensor& v_scales, const at::Tensor& k_tail, const at::Tensor& v_tail, const at::Tensor& k,
               const at::Tensor& v, const at::Tensor& starts) {
    const char* fn = "axs_cache_append_unified";
    const Cache c = cache_of(k_codes, k_scales, v_codes, v_scales, k_tail, v_tail, fn);
    check_like(k, c.kt, 4, fn, "k");
    check_like(v, c.kt, 4, fn, "v");
    const int64_t n = k.size(1);
    TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == c.B && k.size(2) == c.H && k.size(3) == c.D, fn, ": k ", k.sizes(),
                " and v ", v.sizes(), " for a cache of ", c.B, " sequences, ", c.H, " heads of ", c.D);
    const at::Tensor s = int64s(starts, {c.B}, k, fn, "starts"), kp = packed_last(k), vp = packed_last(v);
    c10::DeviceGuard guard(k.device());
    check_rc(axs6_kv_append(kp.data_ptr(), vp.data_ptr(), dtype_code(k.scalar_type()), c.B, n, c.H, c.D,
                            kp.strides().data(), vp.strides().data(), s.data_ptr<int64_t>(), c.nb, c.kc.data_ptr(),
                            c.ks.data_ptr<float>(), c.vc.data_ptr(), c.vs.data_ptr<float>(), c.kt.data_ptr(),
                            c.vt.data_ptr(), stream_of(k)),
             "axs6_kv_append");
}

std::tuple<at::Tensor, at::Tensor> kv_read(const at::Tensor& k_codes, const at::Tensor& k_scales,
                                           const at::Tensor& v_codes, const at::Tensor& v_scales,
                                           const at::Tensor& k_tail, const at::Tensor& v_tail, const at::Tensor& first,
                                           int64_t count) {
    const char* fn = "axs_cache_read_unified";
    const Cache c = cache_of(k_codes, k_scales, v_codes, v_scales, k_tail, v_tail, fn);
    TORCH_CHECK(count >= 0, fn, ": count must not be negative, got ", count);
    const at::Tensor f = int64s(first, {c.B}, c.kc, fn, "first");
    c10::DeviceGuard guard(c.kc.device());
    at::Tensor k = at::empty({c.B, count, c.H, c.D}, c.ks.options()), v = at::empty_like(k);
    check_rc(axs6_kv_read(c.kc.data_ptr(), c.ks.data_ptr<float>(), c.vc.data_ptr(), c.vs.data_ptr<float>(), c.B, c.H, c.D,
                          c.nb, f.data_ptr<int64_t>(), count, k.data_ptr<float>(), v.data_ptr<float>(), stream_of(c.kc)),
             "axs6_kv_read");
    return {k, v};
}

at::Tensor kv_attention(const at::Tensor& q, const at::Tensor& k_codes, const at::Tensor& k_scales,
                        const at::Tensor& v_codes, const at::Tensor& v_scales, const at::Tensor& k_tail,
                        const at::Tensor& v_tail, const at::Tensor& lengths, std::optional<double> scale) {
    const char* fn = "axs_cache_attention_unified";
    const Cache c = cache_of(k_codes, k_scales, v_codes, v_scales, k_tail, v_tail, fn);
    check_like(q, c.kt, 4, fn, "q");
    const int64_t Tq = q.size(1), Hq = q.size(2);
    TORCH_CHECK(q.size(0) == c.B && q.size(3) == c.D && (c.H ? Hq % c.H == 0 : Hq == 0), fn, ": q ", q.sizes(),
                " for a cache of ", c.B, " sequences, ", c.H, " heads of ", c.D);
    const double s = scale ? *scale : 1.0 / std::sqrt((double)c.D);
    TORCH_CHECK(std::isfinite((float)s), fn, ": the scale must be finite, got ", s);
    const at::Tensor n = int64s(lengths, {c.B}, q, fn, "lengths"), qp = packed_last(q);
    c10::DeviceGuard guard(q.device());
    at::Tensor out = at::empty({c.B, Tq, Hq, c.D}, q.options());
    if (c.nb == 0) return out.zero_();
    const at::Tensor ws = workspace(axs6_kv_attention_workspace(c.B, Tq, Hq, c.H, c.D, c.nb), q);
    check_rc(axs6_kv_attention(qp.data_ptr(), dtype_code(q.scalar_type()), c.B, Tq, Hq, c.H, c.D, qp.strides().data(),
                               c.kc.data_ptr(), c.ks.data_ptr<float>(), c.vc.data_ptr(), c.vs.data_ptr<float>(), c.nb,
                               n.data_ptr<int64_t>(), (float)s, out.data_ptr(), data_of(ws), size_of(ws),
                               stream_of(q)),
             "axs6_kv_attention");
    return out;
}

// ---- distillation ---------------------------------------------------------------------------

// Reductions: 0 each row's loss, 1 the weighted mean, 2 the weighted sum.
struct DistillFunction : public torch::autograd::Function<DistillFunction> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& values,
                              const at::Tensor& indices, const at::Tensor& weights, bool has_weights, double T,
                              int64_t reduction) {
        const int64_t V = logits.size(-1), N = V ? logits.numel() / V : 0, K = values.size(-1);
        c10::DeviceGuard guard(logits.device());
        // rows one stride apart are taken as they are
        at::Tensor z = logits.dim() == 2 && (V <= 1 || logits.stride(1) == 1) && logits.stride(0) >= V
                           ? logits
                           : logits.reshape({N, V}).contiguous();
        const at::Tensor w = has_weights ? weights : at::Tensor();
        const auto f32 = logits.options().dtype(at::kFloat);
        at::Tensor rows = at::empty({N}, f32), stats = at::empty({N, 2}, f32);
        at::Tensor loss, norm;
        if (reduction) {
            loss = at::empty({}, f32);
            norm = at::empty({}, f32);   // the gradient's factor
        }
        check_rc(axs6_distill_forward(z.data_ptr(), dtype_code(z.scalar_type()), z.stride(0), N, V,
                                      values.data_ptr<float>(), indices.data_ptr<int64_t>(), K, (float)T,
                                      has_weights ? w.data_ptr<float>() : nullptr, reduction == 1,
                                      rows.data_ptr<float>(), stats.data_ptr<float>(),
                                      reduction ? loss.data_ptr<float>() : nullptr,
                                      reduction ? norm.data_ptr<float>() : nullptr, stream_of(z)),
                 "axs6_distill_forward");
        ctx->save_for_backward({z, values, indices, w, stats, norm});
        auto& d = ctx->saved_data;
        d["T"] = T;
        d["reduction"] = reduction;
        d["shape"] = logits.sizes().vec();
        if (reduction) return loss;
        if (has_weights) rows.mul_(w.view({N}));
        return rows.view(logits.sizes().slice(0, logits.dim() - 1));
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list r(7);
        if (!grads[0].defined() || !ctx->needs_input_grad(0)) return r;
        const auto s = ctx->get_saved_variables();
        auto& d = ctx->saved_data;
        const at::Tensor &z = s[0], &values = s[1], &indices = s[2], &w = s[3];
        const int64_t reduction = d["reduction"].toInt(), N = z.size(0), V = z.size(1);
        c10::DeviceGuard guard(z.device());
        const at::Tensor g = grads[0].to(at::kFloat).contiguous();
        at::Tensor dz = at::empty({N, V}, z.options());
        check_rc(axs6_distill_backward(z.data_ptr(), dtype_code(z.scalar_type()), z.stride(0), N, V,
                                       values.data_ptr<float>(), indices.data_ptr<int64_t>(), values.size(-1),
                                       (float)d["T"].toDouble(), w.defined() ? w.data_ptr<float>() : nullptr,
                                       s[4].data_ptr<float>(), g.data_ptr<float>(), reduction == 0,
                                       reduction ? s[5].data_ptr<float>() : nullptr, dz.data_ptr(), stream_of(z)),
                 "axs6_distill_backward");
        r[0] = dz.view(d["shape"].toIntVector());
        return r;
    }
};

at::Tensor distill(const at::Tensor& logits, const at::Tensor& values, const at::Tensor& indices, double T,
                   const OptTensor& weights, int64_t reduction) {
    const char* fn = "axs_distillation_loss_unified";
    require_device(logits, fn);
    check_dtype(logits, fn, "student_logits");
    TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) >= 1, fn, ": student_logits must be (*, classes), got ",
                logits.sizes());
    require_device(values, fn);
    TORCH_CHECK(values.device() == logits.device(), fn, ": teacher_values are on ", values.device());
    check_dtype(values, fn, "teacher_values");
    TORCH_CHECK(values.dim() == logits.dim() &&
                    values.sizes().slice(0, values.dim() - 1) == logits.sizes().slice(0, logits.dim() - 1),
                fn, ": teacher_values ", values.sizes(), " for student_logits ", logits.sizes());
    TORCH_CHECK(!values.requires_grad(), fn, ": the teacher takes no gradient; detach teacher_values");
    TORCH_CHECK(T > 0.0 && std::isfinite((float)T) && (float)T > 0.0f, fn,
                ": the temperature must be positive and finite, got ", T);
    TORCH_CHECK(reduction >= 0 && reduction <= 2, fn, ": unknown reduction");
    const at::Tensor idx = int64s(indices, values.sizes(), logits, fn, "teacher_indices");
    at::Tensor w;
    if (given(weights)) {
        w = *weights;
        require_device(w, fn);
        TORCH_CHECK(w.device() == logits.device() && w.sizes() == logits.sizes().slice(0, logits.dim() - 1), fn,
                    ": weights must be one value a row, ", logits.sizes().slice(0, logits.dim() - 1), ", got ", w.sizes());
        TORCH_CHECK(!w.requires_grad(), fn, ": the weights take no gradient");
        w = w.to(at::kFloat).contiguous();
    }
    return DistillFunction::apply(logits, values.to(at::kFloat).contiguous(), idx,
                                  w.defined() ? w : at::empty({0}, logits.options()), w.defined(), T, reduction);
}

}  // namespace

void register_decoder(py::module& m) {
    m.def("rotary", &rotary, "rotary positions of q and k (autograd node)", py::arg("q"), py::arg("k"), py::arg("table"),
          py::arg("positions"), py::arg("interleaved"));
    m.def("attention", &attention, "softmax(scale q k^T + mask) v of grouped heads (autograd node)", py::arg("q"),
          py::arg("k"), py::arg("v"), py::arg("mask"), py::arg("causal"), py::arg("scale"));
    m.def("kv_append", &kv_append, "new tokens into the 8-bit cache", py::arg("k_codes"), py::arg("k_scales"),
          py::arg("v_codes"), py::arg("v_scales"), py::arg("k_tail"), py::arg("v_tail"), py::arg("k"), py::arg("v"),
          py::arg("starts"));
    m.def("kv_read", &kv_read, "the values that the 8-bit cache stands for", py::arg("k_codes"), py::arg("k_scales"),
          py::arg("v_codes"), py::arg("v_scales"), py::arg("k_tail"), py::arg("v_tail"), py::arg("first"),
          py::arg("count"));
    m.def("kv_attention", &kv_attention, "attention of the newest tokens over the 8-bit cache", py::arg("q"),
          py::arg("k_codes"), py::arg("k_scales"), py::arg("v_codes"), py::arg("v_scales"), py::arg("k_tail"),
          py::arg("v_tail"), py::arg("lengths"), py::arg("scale"));
    m.def("distill", &distill, "distillation loss against a teacher's top logits (autograd node)", py::arg("logits"),
          py::arg("values"), py::arg("indices"), py::arg("temperature"), py::arg("weights"), py::arg("reduction"));
}

}  // namespace axs6_ext
