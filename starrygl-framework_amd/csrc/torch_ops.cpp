// Autograd side of the attention-layer operators: torch tensors in, calls of the C ABI (include/sgl_hot.h) out.
//
// Host code only; the kernels stay behind the C ABI, whose entry points are handed over as addresses when the module is
// initialised.  It exists because a training step on a mini-batch is shorter than what Python needs to issue it: with the
// graph's nodes in Python a rotary step over 120000 rows (52 us of kernels, forward and gradient) took 130 us of host time.
// Every function returns None for arguments that are not in the plain form it takes (the Python side then says what is
// wrong, or brings them into that form).
#include <torch/extension.h>

#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "../../include/sgl_hot.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

struct Entry {
    decltype(&sgl_last_error_string) error;
    decltype(&sgl_rotary) rotary;
    decltype(&sgl_qk_norm_rotary) norm;
    decltype(&sgl_qk_norm_rotary_backward_workspace_bytes) norm_backward_bytes;
    decltype(&sgl_qk_norm_rotary_backward) norm_backward;
    decltype(&sgl_diff_attn_workspace_bytes) attn_bytes;
    decltype(&sgl_diff_attn) attn;
    decltype(&sgl_diff_attn_backward_workspace_bytes) attn_backward_bytes;
    decltype(&sgl_diff_attn_backward) attn_backward;
} lib;

void init(const std::vector<uintptr_t>& at) {
    TORCH_CHECK(at.size() == sizeof(Entry) / sizeof(uintptr_t), "torch_ops: wrong number of entry points");
    memcpy(&lib, at.data(), sizeof(Entry));
}

void check(int32_t rc) {
    if (rc == SGL_OK) return;
    const std::string msg = "sgl status " + std::to_string(rc) + ": " + lib.error();
    TORCH_CHECK_VALUE(rc != SGL_EINVAL, msg);
    TORCH_CHECK(false, msg);
}

int32_t code_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return SGL_DT_F32;
        case at::kBFloat16: return SGL_DT_BF16;
        case at::kHalf: return SGL_DT_F16;
        default: return 0;
    }
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// [rows, heads, dim] on the GPU, the last axis contiguous
bool is_rows(const Tensor& t) { return t.is_cuda() && t.dim() == 3 && (t.stride(2) == 1 || t.size(2) == 1 || t.numel() == 0) && code_of(t); }
sgl_rows rows(const Tensor& t) { return sgl_rows{t.data_ptr(), t.stride(0), t.stride(1)}; }
Tensor inner(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 || t.numel() == 0 ? t : t.contiguous(); }

bool is_vector(const Tensor& t, const Tensor& like, at::ScalarType type, int64_t n) {
    return t.device() == like.device() && t.scalar_type() == type && t.dim() == 1 && t.size(0) == n && t.is_contiguous();
}
bool wants_grad(const Tensor& t) { return t.requires_grad(); }
bool wants_grad(const MaybeTensor& t) { return t.has_value() && t->requires_grad(); }

// A dual tensor asks for no gradient: without this its tangent would be dropped without a word.
void no_tangent(const char* what, std::initializer_list<MaybeTensor> inputs) {
    for (const MaybeTensor& t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t.has_value() || !t->defined() || !t->_fw_grad(0).defined(), what, ": forward-mode derivatives are not implemented");
}

// The gradients below are formed outside of autograd.  Under create_graph=True they are tied to a node that refuses to be
// differentiated, or a second derivative would silently miss them.
variable_list once(const char* what, variable_list got) {
    if (!at::GradMode::is_enabled()) return got;
    for (Tensor& t : got)
        if (t.defined()) {
            t = t.detach().requires_grad_();
            auto refuse = std::make_shared<torch::autograd::DelayedError>(std::string(what) + ": the gradient cannot be differentiated again", 1);
            t = (*refuse)({t})[0];
        }
    return got;
}

// ------------------------------------------------------------------------------------------------------------ rotary
bool params_fit(const Tensor& x, const Tensor& freq) {
    return freq.device() == x.device() && freq.scalar_type() == at::kDouble && freq.dim() == 1 && freq.is_contiguous() && 2 * freq.size(0) <= x.size(2);
}
sgl_rotary_params params_of(const Tensor& x, const MaybeTensor& freq, bool interleaved, double amplitude, bool inverse) {
    const int64_t half = freq.has_value() ? freq->size(0) : 0;
    return sgl_rotary_params{code_of(x), (int32_t)x.size(2), (int32_t)(2 * half), interleaved, inverse, 0, amplitude, half ? freq->data_ptr<double>() : nullptr};
}

Tensor rotary_call(const Tensor& x, const Tensor& pos, const Tensor& freq, bool interleaved, double amplitude, bool inverse) {
    Tensor out = at::empty(x.sizes(), x.options());
    const c10::DeviceGuard guard(x.device());
    const sgl_rotary_params p = params_of(x, freq, interleaved, amplitude, inverse);
    const sgl_rows from = rows(x), to = rows(out);
    check(lib.rotary(&p, (int32_t)x.size(1), &from, pos.data_ptr<int64_t>(), x.size(0), nullptr, &to, stream_of(x)));
    return out;
}

struct Rotary : public torch::autograd::Function<Rotary> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& pos, const Tensor& freq, bool interleaved, double amplitude) {
        ctx->save_for_backward({pos, freq});
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["amplitude"] = amplitude;
        return rotary_call(x, pos, freq, interleaved, amplitude, false);
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        no_tangent("rotary_encode", {grads[0]});
        return once("rotary_encode", gradients(ctx, grads[0]));
    }
    static variable_list gradients(AutogradContext* ctx, const Tensor& grad) {
        const at::AutoGradMode off(false);
        const variable_list saved = ctx->get_saved_variables();
        const bool interleaved = ctx->saved_data["interleaved"].toBool();
        const double amplitude = ctx->saved_data["amplitude"].toDouble();
        return {rotary_call(inner(grad), saved[0], saved[1], interleaved, amplitude, true), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

MaybeTensor rotary(const Tensor& x, const Tensor& pos, const Tensor& freq, bool interleaved, double amplitude) {
    if (!is_rows(x) || !params_fit(x, freq) || !is_vector(pos, x, at::kLong, x.size(0))) return std::nullopt;
    no_tangent("rotary_encode", {x, freq});
    if (x.requires_grad() && at::GradMode::is_enabled()) return Rotary::apply(x, pos, freq, interleaved, amplitude);
    return rotary_call(x, pos, freq, interleaved, amplitude, false);
}

// ------------------------------------------------------------------------------------------------------- norm + rotary
sgl_norm_side side_of(const Tensor& x, const MaybeTensor& pos, const MaybeTensor& w32) {
    sgl_norm_side s{};
    s.x = rows(x);
    s.pos = pos.has_value() ? pos->data_ptr<int64_t>() : nullptr;
    s.N_max = x.size(0);
    s.heads = (int32_t)x.size(1);
    if (w32.has_value()) {
        s.weight = w32->data_ptr<float>();
        s.weight_stride = w32->dim() == 2 ? x.size(2) : 0;
    }
    return s;
}
MaybeTensor as_f32(const MaybeTensor& w) {
    if (!w.has_value() || (w->scalar_type() == at::kFloat && w->is_contiguous())) return w;
    return w->detach().to(at::kFloat).contiguous();
}

std::tuple<Tensor, Tensor> norm_call(const Tensor& q, const Tensor& k, const MaybeTensor& pos_q, const MaybeTensor& pos_k, const MaybeTensor& wq, const MaybeTensor& wk,
                                     const MaybeTensor& freq, double eps, bool interleaved, double amplitude) {
    Tensor yq = at::empty(q.sizes(), q.options()), yk = at::empty(k.sizes(), k.options());
    const c10::DeviceGuard guard(q.device());
    const MaybeTensor wq32 = as_f32(wq), wk32 = as_f32(wk);
    const sgl_rotary_params p = params_of(q, freq, interleaved, amplitude, false);
    sgl_norm_side s[2] = {side_of(q, pos_q, wq32), side_of(k, pos_k, wk32)};
    s[0].y = rows(yq), s[1].y = rows(yk);
    check(lib.norm(&p, eps, 2, s, stream_of(q)));
    return {yq, yk};
}

struct Norm : public torch::autograd::Function<Norm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const MaybeTensor& pos_q, const MaybeTensor& pos_k, const MaybeTensor& wq,
                                 const MaybeTensor& wk, const MaybeTensor& freq, double eps, bool interleaved, double amplitude) {
        const auto some = [](const MaybeTensor& t) { return t.has_value() ? *t : Tensor(); };
        ctx->save_for_backward({q, k, some(pos_q), some(pos_k), some(wq), some(wk), some(freq)});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["amplitude"] = amplitude;
        ctx->set_materialize_grads(false);
        auto [yq, yk] = norm_call(q, k, pos_q, pos_k, wq, wk, freq, eps, interleaved, amplitude);
        return {yq, yk};
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        no_tangent("qk_norm_rotary", {grads[0], grads[1]});
        return once("qk_norm_rotary", gradients(ctx, grads));
    }
    static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
        const at::AutoGradMode off(false);
        const variable_list v = ctx->get_saved_variables();
        const auto some = [](const Tensor& t) { return t.defined() ? MaybeTensor(t) : std::nullopt; };
        variable_list got(10);
        size_t edge[6];                          // (the graph's edges count the tensors that are there)
        for (int i = 0, n = 0; i < 6; ++i) {
            edge[i] = n;
            n += v[i].defined();
        }
        sgl_norm_side s[2];
        MaybeTensor w32[2];
        Tensor g[2];
        int n = 0;
        bool sums = false;
        for (int i = 0; i < 2; ++i) {
            const bool want_w = v[4 + i].defined() && ctx->needs_input_grad(edge[4 + i]);
            if (!grads[i].defined() || !(ctx->needs_input_grad(edge[i]) || want_w)) continue;
            w32[i] = as_f32(some(v[4 + i]));
            g[i] = inner(grads[i]);
            Tensor dx = at::empty(v[i].sizes(), v[i].options());
            s[n] = side_of(v[i], some(v[2 + i]), w32[i]);
            s[n].y = rows(g[i]);
            s[n].dx = rows(dx);
            if (ctx->needs_input_grad(edge[i])) got[i] = dx;
            else got[7 + i] = dx;               // (kept until the call is issued)
            if (want_w) {
                got[4 + i] = at::empty(v[4 + i].sizes(), v[i].options().dtype(at::kFloat));
                s[n].dweight = got[4 + i].data_ptr<float>();
                sums = true;
            }
            ++n;
        }
        if (n > 0) {
            const Tensor& q = v[0];
            const c10::DeviceGuard guard(q.device());
            const sgl_rotary_params p = params_of(q, some(v[6]), ctx->saved_data["interleaved"].toBool(), ctx->saved_data["amplitude"].toDouble(), false);
            Tensor ws;
            size_t bytes = 0;
            if (sums) {
                bytes = lib.norm_backward_bytes(&p, n, s);
                ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
            }
            check(lib.norm_backward(&p, ctx->saved_data["eps"].toDouble(), n, s, sums ? ws.data_ptr() : nullptr, bytes, stream_of(q)));
        }
        got[7] = got[8] = Tensor();
        for (int i = 4; i < 6; ++i)
            if (got[i].defined() && got[i].scalar_type() != v[i].scalar_type()) got[i] = got[i].to(v[i].scalar_type());
        return got;
    }
};

std::optional<std::tuple<Tensor, Tensor>> norm(const Tensor& q, const Tensor& k, const MaybeTensor& pos_q, const MaybeTensor& pos_k, const MaybeTensor& wq,
                                               const MaybeTensor& wk, const MaybeTensor& freq, double eps, bool interleaved, double amplitude) {
    if (!is_rows(q) || !is_rows(k) || q.device() != k.device() || q.scalar_type() != k.scalar_type() || q.size(2) != k.size(2)) return std::nullopt;
    if (freq.has_value() && (!params_fit(q, *freq) || !pos_q.has_value() || !pos_k.has_value() || !is_vector(*pos_q, q, at::kLong, q.size(0)) ||
                             !is_vector(*pos_k, q, at::kLong, k.size(0))))
        return std::nullopt;
    const auto fits = [&](const MaybeTensor& w, const Tensor& x) {
        return !w.has_value() || (w->device() == x.device() && at::isFloatingType(w->scalar_type()) &&
                                  ((w->dim() == 1 && w->size(0) == x.size(2)) || (w->dim() == 2 && w->size(0) == x.size(1) && w->size(1) == x.size(2))));
    };
    if (!fits(wq, q) || !fits(wk, k)) return std::nullopt;
    no_tangent("qk_norm_rotary", {q, k, wq, wk, freq});
    const MaybeTensor pq = freq.has_value() ? pos_q : std::nullopt, pk = freq.has_value() ? pos_k : std::nullopt;
    if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(wq) || wants_grad(wk))) {
        const variable_list y = Norm::apply(q, k, pq, pk, wq, wk, freq, eps, interleaved, amplitude);
        return std::make_tuple(y[0], y[1]);
    }
    return norm_call(q, k, pq, pk, wq, wk, freq, eps, interleaved, amplitude);
}

// ------------------------------------------------------------------------------------------------------------ attention
// [rows, heads, 2, dim] whose halves lie like heads of their own
bool is_halves(const Tensor& t) {
    if (!t.is_cuda() || t.dim() != 4 || t.size(2) != 2 || !code_of(t)) return false;
    return t.numel() == 0 || ((t.stride(3) == 1 || t.size(3) == 1) && (t.size(1) == 1 || t.stride(1) == 2 * t.stride(2)));
}
sgl_rows halves(const Tensor& t) { return sgl_rows{t.data_ptr(), t.stride(0), t.stride(2)}; }

sgl_diff_attn_args attn_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, const Tensor& k_ptr, const MaybeTensor& q_ptr, double scale, bool causal,
                             int64_t window, const MaybeTensor& key_mask) {
    sgl_diff_attn_args a{};
    a.dtype = code_of(q);
    a.Hq = (int32_t)q.size(1), a.Hk = (int32_t)k.size(1), a.D = (int32_t)q.size(3), a.Dv = (int32_t)v.size(2);
    a.causal = causal;
    a.window = window;
    a.scale = scale;
    a.B = k_ptr.size(0) - 1, a.Tq = q.size(0), a.Tk = k.size(0);
    a.k_ptr = k_ptr.data_ptr<int64_t>();
    a.q_ptr = q_ptr.has_value() ? q_ptr->data_ptr<int64_t>() : nullptr;
    a.key_mask = key_mask.has_value() ? static_cast<const uint8_t*>(key_mask->data_ptr()) : nullptr;
    a.lam = lam.data_ptr<float>();
    a.q = halves(q), a.k = halves(k), a.v = rows(v);
    a.flags = SGL_ATTN_ZERO_REST;
    return a;
}

// What the backward takes its row sums from: in fp32 out and o2, whose roundings are those of a sum; in 16 bits both maps'
// results before they are rounded.
void set_kept(sgl_diff_attn_args& a, const Tensor& lse, const Tensor& kept) {
    if (a.Tq == 0) return;
    a.lse = lse.data_ptr<float>();
    if (kept.dim() == 3) a.o2 = rows(kept);
    else a.maps = kept.data_ptr<float>();
}

Tensor attn_forward(sgl_diff_attn_args& a, const Tensor& q, Tensor* lse, Tensor* kept) {
    Tensor out = at::empty({a.Tq, a.Hq, a.Dv}, q.options());
    a.out = rows(out);
    if (lse) {
        const auto f32 = q.options().dtype(at::kFloat);
        *lse = at::empty({a.Tq, a.Hq, 2}, f32);
        *kept = a.dtype == SGL_DT_F32 ? at::empty({a.Tq, a.Hq, a.Dv}, f32) : at::empty({a.Tq, a.Hq, 2, a.Dv}, f32);
        set_kept(a, *lse, *kept);
    }
    const c10::DeviceGuard guard(q.device());
    const size_t bytes = lib.attn_bytes(&a);
    Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    check(lib.attn(&a, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(q)));
    return out;
}

struct Attention : public torch::autograd::Function<Attention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, const Tensor& k_ptr, const MaybeTensor& q_ptr,
                          double scale, bool causal, int64_t window, const MaybeTensor& key_mask) {
        sgl_diff_attn_args a = attn_args(q, k, v, lam, k_ptr, q_ptr, scale, causal, window, key_mask);
        Tensor lse, kept;
        Tensor out = attn_forward(a, q, &lse, &kept);
        const auto some = [](const MaybeTensor& t) { return t.has_value() ? *t : Tensor(); };
        ctx->save_for_backward({q, k, v, lam, kept.dim() == 3 ? out : Tensor(), lse, kept, k_ptr, some(q_ptr), some(key_mask)});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["causal"] = causal;
        ctx->saved_data["window"] = window;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        no_tangent("diff_attention", {grads[0]});
        return once("diff_attention", gradients(ctx, grads[0]));
    }
    static variable_list gradients(AutogradContext* ctx, const Tensor& grad) {
        const at::AutoGradMode off(false);
        const variable_list t = ctx->get_saved_variables();
        const auto some = [](const Tensor& x) { return x.defined() ? MaybeTensor(x) : std::nullopt; };
        const Tensor &q = t[0], &k = t[1], &v = t[2], &lam = t[3], &out = t[4];
        sgl_diff_attn_args a = attn_args(q, k, v, lam, t[7], some(t[8]), ctx->saved_data["scale"].toDouble(), ctx->saved_data["causal"].toBool(),
                                         ctx->saved_data["window"].toInt(), some(t[9]));
        const Tensor g = inner(grad);
        Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options());
        Tensor dlam = at::empty({a.Hq}, lam.options());
        set_kept(a, t[5], t[6]);
        if (out.defined()) a.out = rows(out);
        a.d_out = rows(g);
        a.d_q = halves(dq), a.d_k = halves(dk), a.d_v = rows(dv);
        a.d_lam = dlam.data_ptr<float>();
        const c10::DeviceGuard guard(q.device());
        const size_t bytes = lib.attn_backward_bytes(&a);
        const Tensor ws = at::empty({(int64_t)std::max<size_t>(bytes, 16)}, q.options().dtype(at::kByte));
        check(lib.attn_backward(&a, ws.data_ptr(), bytes, stream_of(q)));
        return {dq, dk, dv, dlam, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

MaybeTensor attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, const Tensor& k_ptr, const MaybeTensor& q_ptr, std::optional<double> scale,
                      bool causal, std::optional<int64_t> window, const MaybeTensor& key_mask) {
    if (!is_halves(q) || !is_halves(k) || !is_rows(v) || k.device() != q.device() || v.device() != q.device() || k.scalar_type() != q.scalar_type() ||
        v.scalar_type() != q.scalar_type())
        return std::nullopt;
    const int64_t Hq = q.size(1), Hk = k.size(1), B = k_ptr.dim() == 1 ? k_ptr.size(0) - 1 : -1;
    if (Hk < 1 || Hq % Hk || v.size(1) != Hk || v.size(0) != k.size(0) || k.size(3) != q.size(3) || B < 0) return std::nullopt;
    if (!is_vector(lam, q, at::kFloat, Hq) || !is_vector(k_ptr, q, at::kLong, B + 1) || (q_ptr.has_value() && !is_vector(*q_ptr, q, at::kLong, B + 1)) ||
        (!q_ptr.has_value() && q.size(0) != B))
        return std::nullopt;
    if (key_mask.has_value() && !is_vector(*key_mask, q, at::kBool, k.size(0)) && !is_vector(*key_mask, q, at::kByte, k.size(0))) return std::nullopt;
    if (window.has_value() && (!causal || *window < 1)) return std::nullopt;
    no_tangent("diff_attention", {q, k, v, lam});
    const double c = scale.has_value() ? *scale : 1.0 / std::sqrt((double)q.size(3));
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() || lam.requires_grad()))
        return Attention::apply(q, k, v, lam, k_ptr, q_ptr, c, causal, window.value_or(0), key_mask);
    sgl_diff_attn_args a = attn_args(q, k, v, lam, k_ptr, q_ptr, c, causal, window.value_or(0), key_mask);
    return attn_forward(a, q, nullptr, nullptr);
}

}  // namespace

PYBIND11_MODULE(sgl_torch, m) {
    m.def("init", &init);
    m.def("rotary", &rotary, pybind11::call_guard<pybind11::gil_scoped_release>());
    m.def("norm", &norm, pybind11::call_guard<pybind11::gil_scoped_release>());
    m.def("attention", &attention, pybind11::call_guard<pybind11::gil_scoped_release>());
}
