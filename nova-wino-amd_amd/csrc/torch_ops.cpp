// Python binding of group norm and attention (module _nova_ops): argument
// checks, allocation, autograd. The work itself is the library's C entry points
// (include/nova_winograd.h); this file only calls them.
//
// It is native because a call's host part was several times its kernels' time:
// us a call from Python on MI355X, ctypes and a Python autograd function ->
// this: group norm 1x1280x8x8 14.7 -> 7.4, a training step of 3x960x33x47 137 -> 70.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/python.h>

#include <limits>

#include "../../include/nova_winograd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check(const char* where) {
    const int code = nova_get_last_error();
    TORCH_CHECK(code == 0, "nova_winograd ", where, ": ", nova_get_last_error_message(), " (code ",
                code, ")");
}

void require_gpu(const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), "nova_winograd: ", name, " is on ", t.device(),
                "; NOVA Winograd runs only on a ROCm GPU (no CPU fallback)");
}

void* stream_of(const Tensor& t) {
    return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

int dtype_code(at::ScalarType t) {
    return t == at::kHalf ? 0 : t == at::kBFloat16 ? 1 : t == at::kFloat ? 2 : -1;
}

// The C structures hold sizes as int.
void require_ints(const char* fn, const char* name, at::IntArrayRef sizes) {
    for (const int64_t n : sizes)
        TORCH_CHECK_VALUE(n <= std::numeric_limits<int>::max(), fn, ": ", name, " of ", sizes,
                          " exceeds launch limits");
}

// Scratch memory for one call from PyTorch's allocator: its owner may go when
// the call returns (the allocator hands it on in stream order only), and in a
// graph capture it comes from the graph's pool.
Tensor scratch(const Tensor& like, long long bytes, const char* where) {
    if (bytes < 0) check(where);
    return at::empty({bytes}, like.options().dtype(at::kByte));
}

const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

// An optional argument of an autograd function.
std::optional<Tensor> given(const Tensor& t) {
    return t.defined() ? std::optional<Tensor>(t) : std::nullopt;
}

// Whether a result takes part in a backward. Forward-mode derivatives are an
// error: outside of the autograd functions nothing else would stop a tangent
// from being dropped.
bool recorded(const char* fn, std::initializer_list<const Tensor*> in) {
    bool any = false;
    for (const Tensor* t : in) {
        if (!t->defined()) continue;
        TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), fn,
                                    ": forward-mode derivatives are not implemented");
        any |= t->requires_grad();
    }
    return any && at::GradMode::is_enabled();
}

// Gradients of a backward that runs with gradients enabled (create_graph): what
// the kernels wrote cannot be differentiated again, which is an error only if
// someone does.
variable_list once(variable_list grads, const char* what) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list in;
    for (const auto& g : grads) in.push_back(g.defined() ? g.detach().requires_grad_() : g);
    auto fn = std::make_shared<torch::autograd::DelayedError>(
        std::string(what) + " is not differentiable twice", (int)in.size());
    return (*fn)(std::move(in));
}

// ---- group norm ---------------------------------------------------------------

struct Norm {
    Tensor x, weight, bias;
    int64_t groups;
    double eps;
    bool silu;
    at::MemoryFormat format;

    nova_group_norm_t args() const {
        nova_group_norm_t a{};
        a.x = x.const_data_ptr();
        a.weight = ptr(weight);
        a.bias = ptr(bias);
        a.dtype = dtype_code(x.scalar_type());
        const Tensor& p = weight.defined() ? weight : bias;
        a.param_dtype = p.defined() ? dtype_code(p.scalar_type()) : 2;
        a.batch = (int)x.size(0);
        a.channels = (int)x.size(1);
        a.groups = (int)groups;
        a.channels_last = format == at::MemoryFormat::Contiguous ? 0 : 1;
        a.silu = silu;
        a.eps = (float)eps;
        a.pixels = 1;
        for (int64_t d = 2; d < x.dim(); d++) a.pixels *= x.size(d);
        return a;
    }
};

// x in a dense layout: channels-last where it is that and not also contiguous,
// else contiguous (copied if it is neither).
Norm norm_of(const Tensor& x, int64_t groups, const Tensor& weight, const Tensor& bias, double eps,
             bool silu) {
    Norm n{x, weight, bias, groups, eps, silu, at::MemoryFormat::Contiguous};
    if (!x.is_contiguous()) {
        if (x.dim() == 4 && x.is_contiguous(at::MemoryFormat::ChannelsLast))
            n.format = at::MemoryFormat::ChannelsLast;
        else if (x.dim() == 5 && x.is_contiguous(at::MemoryFormat::ChannelsLast3d))
            n.format = at::MemoryFormat::ChannelsLast3d;
        else
            n.x = x.contiguous();
    }
    return n;
}

// y. stats: gets mean and 1 / standard deviation, [2][B][G], for a backward; or
// null. The workspace lies behind them in one allocation: another one costs a
// training step about 1 us of host time (40 us against 39). But what a backward
// keeps of it is held to 1/16 of x (2/3 for 10240 channels of 9 pixels, NCHW).
Tensor norm_forward(const Norm& n, Tensor* stats) {
    const c10::DeviceGuard guard(n.x.device());
    const nova_group_norm_t a = n.args();
    const long long ws = nova_group_norm_workspace_bytes(&a, 0);
    if (ws < 0) check("group_norm");
    const int64_t count = (int64_t)a.batch * a.groups;
    const int64_t front = (2 * count + 3) / 4 * 4;  // the workspace starts on 16 bytes
    const bool apart = stats && ws > (long long)n.x.nbytes() / 16;
    const Tensor both = at::empty({front + (apart ? 0 : (ws + 3) / 4)},
                                  n.x.options().dtype(at::kFloat), at::MemoryFormat::Contiguous);
    Tensor work;
    if (apart) work = scratch(n.x, ws, "group_norm");
    if (stats) *stats = both;
    Tensor y = at::empty_like(n.x, n.x.options(), n.format);
    float* s = both.mutable_data_ptr<float>();
    void* w = work.defined() ? work.mutable_data_ptr() : s + front;
    nova_group_norm(&a, y.mutable_data_ptr(), s, s + count, w, ws, stream_of(n.x));
    check("group_norm");
    return y;
}

struct GroupNormFunction : torch::autograd::Function<GroupNormFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x,
                          const std::optional<Tensor>& weight_, const std::optional<Tensor>& bias_,
                          int64_t groups, double eps, bool silu) {
        const Tensor weight = weight_.value_or(Tensor()), bias = bias_.value_or(Tensor());
        const Norm n = norm_of(x, groups, weight, bias, eps, silu);
        Tensor stats;
        Tensor y = norm_forward(n, &stats);
        ctx->save_for_backward({n.x, weight, bias, stats});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["silu"] = silu;
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Norm n = norm_of(saved[0], ctx->saved_data["groups"].toInt(), saved[1], saved[2],
                               ctx->saved_data["eps"].toDouble(), ctx->saved_data["silu"].toBool());
        const Tensor stats = saved[3].detach();
        const c10::DeviceGuard guard(n.x.device());
        const Tensor gy = grads[0].detach().to(n.x.scalar_type()).contiguous(n.format);
        const nova_group_norm_t a = n.args();
        Tensor gx = at::empty_like(n.x.detach(), n.x.options(), n.format), gp;
        // absent parameters have no place among the inputs with gradients
        const bool params =
            (n.weight.defined() && ctx->needs_input_grad(1)) ||
            (n.bias.defined() && ctx->needs_input_grad(n.weight.defined() ? 2 : 1));
        if (params)
            gp = at::empty({2, n.x.size(1)},
                           (n.weight.defined() ? n.weight : n.bias).options());
        const Tensor ws = scratch(n.x, nova_group_norm_workspace_bytes(&a, 1), "group_norm backward");
        const int64_t count = (int64_t)a.batch * a.groups;
        const float* s = stats.const_data_ptr<float>();
        char* to = params ? static_cast<char*>(gp.mutable_data_ptr()) : nullptr;
        nova_group_norm_backward(&a, gy.const_data_ptr(), s, s + count, gx.mutable_data_ptr(), to,
                                 params ? to + gp.nbytes() / 2 : nullptr, ws.mutable_data_ptr(),
                                 ws.numel(), stream_of(n.x));
        check("group_norm backward");
        variable_list out(6);
        out[0] = gx;
        if (params && n.weight.defined()) out[1] = gp.select(0, 0);
        if (params && n.bias.defined()) out[2] = gp.select(0, 1);
        return once(std::move(out), "nova_group_norm");
    }
};

Tensor group_norm(const Tensor& x, int64_t groups, const std::optional<Tensor>& weight_,
                  const std::optional<Tensor>& bias_, double eps, bool silu) {
    require_gpu(x, "input");
    TORCH_CHECK_TYPE(dtype_code(x.scalar_type()) >= 0, "nova_group_norm: input is ",
                     x.scalar_type(), "; float16, bfloat16 and float32 are supported");
    TORCH_CHECK_VALUE(x.dim() >= 2, "nova_group_norm: input needs a batch and a channel axis");
    const int64_t C = x.size(1);
    require_ints("nova_group_norm", "input", x.sizes().slice(0, 2));
    TORCH_CHECK_VALUE(groups >= 1 && C >= 1 && C % groups == 0, "nova_group_norm: num_groups (",
                      groups, ") does not divide the ", C, " channels");
    Tensor p[2] = {weight_.value_or(Tensor()), bias_.value_or(Tensor())};
    for (int i = 0; i < 2; i++) {
        if (!p[i].defined()) continue;
        const char* name = i ? "bias" : "weight";
        require_gpu(p[i], name);
        TORCH_CHECK_TYPE(dtype_code(p[i].scalar_type()) >= 0, "nova_group_norm: ", name, " is ",
                         p[i].scalar_type());
        TORCH_CHECK_VALUE(p[i].dim() == 1 && p[i].size(0) == C && p[i].device() == x.device(),
                          "nova_group_norm: ", name, " has to hold ", C, " values on ", x.device());
        p[i] = p[i].contiguous();
    }
    if (p[0].defined() && p[1].defined()) p[1] = p[1].to(p[0].scalar_type());
    if (recorded("nova_group_norm", {&x, &p[0], &p[1]}))
        return GroupNormFunction::apply(x, given(p[0]), given(p[1]), groups, eps, silu);
    const at::AutoDispatchBelowADInplaceOrView below;
    return norm_forward(norm_of(x, groups, p[0], p[1], eps, silu), nullptr);
}

// ---- attention ----------------------------------------------------------------

nova_attention_t attention_args(const Tensor& q, const Tensor& k, const Tensor& v,
                                const Tensor& mask, double scale) {
    nova_attention_t a{};
    a.q = q.const_data_ptr();
    a.k = k.const_data_ptr();
    a.v = v.const_data_ptr();
    for (int i = 0; i < 3; i++) {
        a.q_strides[i] = q.stride(i);
        a.k_strides[i] = k.stride(i);
        a.v_strides[i] = v.stride(i);
    }
    if (mask.defined()) {
        a.key_mask = static_cast<const unsigned char*>(mask.const_data_ptr());
        a.mask_stride = mask.size(0) == 1 ? 0 : mask.stride(0);
    }
    a.dtype = dtype_code(q.scalar_type());
    a.batch = (int)q.size(0);
    a.kv_batch = (int)k.size(0);
    a.queries = (int)q.size(1);
    a.keys = (int)k.size(1);
    a.heads = (int)q.size(2);
    a.kv_heads = (int)k.size(2);
    a.head_dim = (int)q.size(3);
    a.scale = (float)scale;
    return a;
}

Tensor attention_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& mask,
                         double scale, Tensor* rest, Tensor* lse) {
    const c10::DeviceGuard guard(q.device());
    const nova_attention_t a = attention_args(q, k, v, mask, scale);
    Tensor out = at::empty(q.sizes(), q.options());
    const long long bytes = nova_cross_attention_workspace_bytes(&a, 0);
    Tensor ws;
    if (bytes != 0) ws = scratch(q, bytes, "cross_attention");
    if (lse) {
        *lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
        if (nova_cross_attention_uses_rest(&a)) *rest = at::empty(q.sizes(), q.options());
    }
    nova_cross_attention(&a, out.mutable_data_ptr(),
                         rest && rest->defined() ? rest->mutable_data_ptr() : nullptr,
                         lse ? lse->mutable_data_ptr<float>() : nullptr,
                         ws.defined() ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(q));
    check("cross_attention");
    return out;
}

struct AttentionFunction : torch::autograd::Function<AttentionFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                          const std::optional<Tensor>& mask_, double scale) {
        const Tensor mask = mask_.value_or(Tensor());
        Tensor rest, lse;
        Tensor out = attention_forward(q, k, v, mask, scale, &rest, &lse);
        ctx->save_for_backward({q, k, v, mask, out, rest, lse});
        ctx->saved_data["scale"] = scale;
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const Tensor q = s[0].detach(), k = s[1].detach(), v = s[2].detach(), &mask = s[3];
        const c10::DeviceGuard guard(q.device());
        const Tensor go = grads[0].detach().to(q.scalar_type()).contiguous();
        const nova_attention_t a =
            attention_args(q, k, v, mask, ctx->saved_data["scale"].toDouble());
        Tensor gq = at::empty(q.sizes(), q.options()), gk = at::empty(k.sizes(), k.options()),
               gv = at::empty(v.sizes(), v.options());
        const Tensor ws =
            scratch(q, nova_cross_attention_workspace_bytes(&a, 1), "cross_attention backward");
        nova_cross_attention_backward(&a, s[4].const_data_ptr(), ptr(s[5]),
                                      s[6].const_data_ptr<float>(), go.const_data_ptr(),
                                      gq.mutable_data_ptr(), gk.mutable_data_ptr(),
                                      gv.mutable_data_ptr(), ws.mutable_data_ptr(), ws.numel(),
                                      stream_of(q));
        check("cross_attention backward");
        return once({gq, gk, gv, Tensor(), Tensor()}, "nova_cross_attention");
    }
};

Tensor dense_rows(const Tensor& t) { return t.stride(3) == 1 ? t : t.contiguous(); }

Tensor cross_attention(const Tensor& query, const Tensor& key, const Tensor& value,
                       const std::optional<Tensor>& key_mask, std::optional<double> scale_) {
    const char* names[3] = {"query", "key", "value"};
    const Tensor* in[3] = {&query, &key, &value};
    for (int i = 0; i < 3; i++) {
        const Tensor& t = *in[i];
        require_gpu(t, names[i]);
        const int code = dtype_code(t.scalar_type());
        TORCH_CHECK_TYPE((code == 0 || code == 1) && t.scalar_type() == query.scalar_type(),
                         "nova_cross_attention: ", names[i], " is ", t.scalar_type(),
                         "; query, key and value have to be float16 or bfloat16, all the same");
        TORCH_CHECK_VALUE(t.dim() == 4 && t.device() == query.device(), "nova_cross_attention: ",
                          names[i], " has to be [batch, length, heads, channels] on ",
                          query.device(), ", got ", t.sizes(), " on ", t.device());
        require_ints("nova_cross_attention", names[i], t.sizes());
    }
    const int64_t B = query.size(0), H = query.size(2), D = query.size(3);
    TORCH_CHECK_VALUE(key.sizes() == value.sizes() && (key.size(0) == B || key.size(0) == 1) &&
                          key.size(3) == D,
                      "nova_cross_attention: shapes do not fit: query ", query.sizes(), ", key ",
                      key.sizes(), ", value ", value.sizes());
    TORCH_CHECK_VALUE(H >= 1 && key.size(2) >= 1 && H % key.size(2) == 0, "nova_cross_attention: ",
                      key.size(2), " key heads do not divide ", H, " query heads");
    TORCH_CHECK_VALUE(D >= 1 && D <= 256, "nova_cross_attention: head size ", D,
                      "; 1 to 256 are supported");
    Tensor mask = key_mask.value_or(Tensor());
    if (mask.defined()) {
        require_gpu(mask, "key_mask");
        TORCH_CHECK_TYPE(mask.scalar_type() == at::kBool, "nova_cross_attention: key_mask is ",
                         mask.scalar_type(), ", not bool");
        TORCH_CHECK_VALUE(mask.dim() == 2 && (mask.size(0) == B || mask.size(0) == 1) &&
                              mask.size(1) == key.size(1) && mask.device() == query.device(),
                          "nova_cross_attention: key_mask has to be [batch, keys] on the query's "
                          "device, got ",
                          mask.sizes());
        if (mask.stride(1) != 1) mask = mask.contiguous();
    }
    const double scale = scale_ ? *scale_ : 1.0 / std::sqrt((double)D);
    const Tensor q = dense_rows(query), k = dense_rows(key), v = dense_rows(value);
    if (recorded("nova_cross_attention", {&q, &k, &v}))
        return AttentionFunction::apply(q, k, v, given(mask), scale);
    const at::AutoDispatchBelowADInplaceOrView below;
    return attention_forward(q, k, v, mask, scale, nullptr, nullptr);
}

}  // namespace

PYBIND11_MODULE(_nova_ops, m) {
    m.def("group_norm", &group_norm);
    m.def("cross_attention", &cross_attention);
}
