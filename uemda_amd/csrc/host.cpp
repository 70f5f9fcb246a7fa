// The host side of layer norm, grouped products and gradient clipping: argument checks, allocations, autograd nodes and the launches through the
// C ABI, as a CPython extension (uemda_amd._host) on libtorch.  Its kernels often take 5 - 30 us; a forward and backward pass of a node written in
// Python took 110 us of host time (its backward runs in the engine's thread, where every attribute and call costs twice), one of these 40.
// The library's entry points arrive as addresses from uemda_amd._lib, which loads it (and honours UEM_LIB_PATH): there is one library in a process.
#include <torch/csrc/python_headers.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/InferenceMode.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <sstream>
#include <string>
#include <utility>
#include <vector>

#include "uemda_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

PyObject* g_error = nullptr;                      // uemda_amd.UemError

// raises UemError, from any thread
template <typename... A> [[noreturn]] void refuse(const A&... a) {
    std::ostringstream s;
    (s << ... << a);
    const PyGILState_STATE gil = PyGILState_Ensure();
    PyErr_SetString(g_error, s.str().c_str());
    python_error e;
    e.persist();
    PyGILState_Release(gil);
    throw e;
}

// ---- the C ABI --------------------------------------------------------------------------------------------------------------------------
#define UEM_HOST_FUNCTIONS(F) \
    F(uem_last_error) F(uem_layernorm_workspace_floats) F(uem_layernorm_fwd) F(uem_layernorm_bwd) F(uem_multi_norm_workspace_doubles) \
    F(uem_multi_norm) F(uem_multi_clip) F(uem_grouped_pad) F(uem_grouped_any_rows) F(uem_grouped_fwd) F(uem_grouped_dgrad) F(uem_grouped_wgrad_workspace_floats) \
    F(uem_grouped_wgrad) F(uem_cast_f32_bf16)
#define UEM_DECLARE(name) decltype(&::name) name##_ = nullptr;
UEM_HOST_FUNCTIONS(UEM_DECLARE)

template <typename F, typename... A> void call(const char* name, F f, A... a) {
    const int rc = f(a...);
    if (rc != UEM_OK) {
        const char* msg = uem_last_error_();
        refuse(name, " failed (code ", rc, "): ", msg ? msg : "?");
    }
}
#define CALL(name, ...) call(#name, name##_, __VA_ARGS__)

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
bool is16(const Tensor& t) { return t.defined() && t.scalar_type() == at::kBFloat16; }
bool is_real(const Tensor& t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16; }
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
void need_gpu(std::initializer_list<const Tensor*> list) {
    for (const Tensor* t : list)
        if (t->defined() && !t->is_cuda())
            refuse("uemda_amd: the HIP path needs tensors on the MI355X device (there is no CPU / PyTorch fallback)");
}
void no_second_derivative(const char* what) {
    // its kernels are nothing autograd can see through: under create_graph=True the result would silently count as a constant
    if (at::GradMode::is_enabled()) refuse(what, ": a gradient of the gradient is not offered (create_graph=True)");
}

// Forward-mode derivatives and traces would pass the kernels by as silently: a dual tensor's tangent counts as zero in the result, and a trace
// records the allocation of the output and no launch.  (A call without requires_grad never reaches the autograd node, which would refuse.)
void no_transforms(const char* what, std::initializer_list<const Tensor*> list) {
    if (torch::jit::tracer::isTracing()) refuse(what, ": its kernels cannot be traced (torch.jit.trace)");
    for (const Tensor* t : list)
        if (t->defined() && t->_fw_grad(0).defined()) refuse(what, ": a forward-mode derivative is not offered (a tensor of torch.autograd.forward_ad)");
}

// A graph of the same leaves that lives outside a capture holds the nodes that add up their gradients, on the stream they were made on; a
// backward pass captured on another stream would join that stream to the capture, inside the engine, which ends the process.
void no_outside_graph(const char* what, std::initializer_list<const Tensor*> list) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    for (const Tensor* t : list) {
        if (!wants_grad(*t) || !t->is_leaf()) continue;
        const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
        const auto st = node ? node->stream() : std::nullopt;
        if (st && st->id() != c10::hip::getCurrentHIPStream(t->get_device()).id())
            refuse(what, ": a graph of the same leaf, made outside this capture, is still alive (an output of an eager pass that somebody holds): "
                         "release it before capturing a pass that records gradients");
    }
}

// an argument that may be absent, as autograd takes it: absent ones have no edge in the graph
std::optional<Tensor> maybe(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// ---- layer norm ------------------------------------------------------------------------------------------------------------------------
// t as rows of c channels: itself where it is dense, or 2-d with a stride between its rows; a copy otherwise
Tensor norm_rows(const Tensor& t, int64_t c, int64_t& ld) {
    if (t.is_contiguous()) { ld = c; return t; }
    if (t.dim() == 2 && t.stride(1) == 1 && t.stride(0) >= c) { ld = t.stride(0); return t; }
    ld = c;
    return t.contiguous();
}
int norm_flags(const Tensor& x, bool param16) { return (is16(x) ? UEM_LN_BF16 : 0) | (param16 ? UEM_LN_PARAM_BF16 : 0); }
struct Normed { Tensor y, stats, x; };             // x: as the kernel reads it
Normed norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, bool save) {
    const c10::DeviceGuard guard(x.device());
    const int64_t c = x.size(-1), rows = x.numel() / c;
    Tensor y = at::empty(x.sizes(), x.options()), stats;
    if (save) stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
    if (rows == 0) return {y, stats, x};
    int64_t ld;
    const Tensor xr = norm_rows(x, c, ld);
    float* const mean = save ? stats.data_ptr<float>() : nullptr;
    CALL(uem_layernorm_fwd, ptr(xr), ld, ptr(w), ptr(b), mptr(y), mean, save ? mean + rows : nullptr, rows, (int)c, (float)eps,
         norm_flags(x, is16(w) || is16(b)), stream_of(x));
    return {y, stats, xr};
}
struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& w_, const std::optional<Tensor>& b_, double eps) {
        const Tensor w = w_.value_or(Tensor()), b = b_.value_or(Tensor());
        const Normed r = norm_forward(x, w, b, eps, true);
        ctx->save_for_backward({r.x, w, r.stats});
        ctx->saved_data["param16"] = is16(w) || is16(b);
        ctx->saved_data["bias"] = b.defined();
        return r.y;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        no_second_derivative("layer_norm");
        no_transforms("layer_norm", {&grads[0]});
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
        const c10::DeviceGuard guard(x.device());
        const bool p16 = ctx->saved_data["param16"].toBool();
        const int64_t c = x.size(-1), rows = x.numel() / c;
        const bool need_w = w.defined() && ctx->needs_input_grad(1), need_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(w.defined() ? 2 : 1);
        const auto popt = x.options().dtype(p16 ? at::kBFloat16 : at::kFloat);
        const Tensor dx = at::empty(x.sizes(), x.options());
        Tensor dw, db, ws;
        if (need_w) dw = at::empty({c}, popt);
        if (need_b) db = at::empty({c}, popt);
        if (rows == 0) {
            if (need_w) dw.zero_();
            if (need_b) db.zero_();
        } else {
            int64_t x_ld, dy_ld;
            const Tensor xr = norm_rows(x, c, x_ld), dyr = norm_rows(grads[0], c, dy_ld);
            if (need_w || need_b) ws = at::empty({uem_layernorm_workspace_floats_(rows, (int)c)}, x.options().dtype(at::kFloat));
            const float* const mean = stats.const_data_ptr<float>();
            CALL(uem_layernorm_bwd, ptr(xr), x_ld, ptr(dyr), dy_ld, ptr(w), mean, mean + rows, mptr(dx), mptr(dw), mptr(db), (float*)mptr(ws), rows, (int)c,
                 norm_flags(x, p16), stream_of(x));
        }
        return {ctx->needs_input_grad(0) ? dx : Tensor(), dw, db, Tensor()};
    }
};
Tensor layer_norm(const Tensor& x, const Tensor& w, const Tensor& b, double eps) {
    if (!is_real(x)) refuse("layer_norm: x must be a float32 or bfloat16 tensor, got ", x.scalar_type());
    no_transforms("layer_norm", {&x, &w, &b});
    need_gpu({&x, &w, &b});
    if (x.dim() == 0 || x.size(-1) == 0) refuse("layer_norm: x needs a last dimension of at least one channel, got shape ", x.sizes());
    if (x.size(-1) > (1 << 30)) refuse("layer_norm: at most 2^30 channels, got ", x.size(-1));
    if (!(eps >= 0) || std::isinf(eps)) refuse("layer_norm: eps must be finite and not negative, got ", eps);
    for (const auto& [name, p] : {std::pair<const char*, const Tensor*>{"weight", &w}, {"bias", &b}})
        if (p->defined() && (p->dim() != 1 || p->size(0) != x.size(-1) || !is_real(*p) || !p->is_contiguous() || p->device() != x.device()))
            refuse("layer_norm: ", name, " must be a contiguous float32 or bfloat16 vector of ", x.size(-1), " channels on ", x.device(), ", got ",
                   p->scalar_type(), " ", p->sizes(), " strides ", p->strides(), " on ", p->device());
    if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type())
        refuse("layer_norm: weight and bias must have one type, got ", w.scalar_type(), " and ", b.scalar_type());
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b))) {
        const c10::DeviceGuard guard(x.device());
        no_outside_graph("layer_norm", {&x, &w, &b});
        return LayerNormFn::apply(x, maybe(w), maybe(b), eps);
    }
    return norm_forward(x, w, b, eps, false).y;
}

// ---- grouped products -------------------------------------------------------------------------------------------------------------------
constexpr int64_t MOST_LD = 1 << 21;              // elements between rows that the kernels address
// 2-d t as rows that begin on 16-byte boundaries and end in zeros up to the next -- `any`: on any element -- t itself, or a copy
Tensor operand(Tensor t, int& ld, bool any = false) {
    const int64_t rows = t.size(0), cols = t.size(1), per = 16 / t.element_size();
    if ((cols > 1 && t.stride(1) != 1) || (rows > 1 && !(cols <= t.stride(0) && t.stride(0) <= MOST_LD))) t = t.contiguous();
    const int64_t have = rows > 1 ? t.stride(0) : cols;
    if (any || (cols % per == 0 && have % per == 0 && ((uintptr_t)t.const_data_ptr() & 15) == 0)) { ld = (int)have; return t; }
    ld = (int)((cols + per - 1) / per * per);
    const Tensor out = at::empty({rows, ld}, t.options());
    CALL(uem_grouped_pad, ptr(t), have, mptr(out), ld, (int)cols, rows, is16(t) ? UEM_GROUPED_BF16 : 0, stream_of(t));
    return out;
}
int grouped_flags(const Tensor& x, const Tensor& offsets) {
    return (is16(x) ? UEM_GROUPED_BF16 : 0) | (offsets.scalar_type() == at::kLong ? UEM_GROUPED_OFFSETS_64 : 0);
}
struct Grouped { Tensor y, x, w; };               // y, and the operands as the forward's kernel reads them
Grouped grouped_forward(const Tensor& x, const Tensor& weight, const Tensor& offsets, const Tensor& bias) {
    const c10::DeviceGuard guard(x.device());
    const int64_t T = x.size(0), K = x.size(1), G = weight.size(0), N = weight.size(1);
    Grouped r{at::empty({T, N}, x.options()), x, weight};
    if (T == 0) return r;
    Tensor w = weight.reshape({G * N, K});
    if (w.scalar_type() != x.scalar_type()) {                                  // fp32 master weights under bf16 rows
        w = w.contiguous();
        const Tensor w16 = at::empty({G * N, K}, x.options());
        CALL(uem_cast_f32_bf16, w.const_data_ptr<float>(), (uint16_t*)mptr(w16), w.numel(), stream_of(x));
        w = w16;
    }
    int x_ld, w_ld;
    const int flags = grouped_flags(x, offsets);
    const bool any = uem_grouped_any_rows_((int)T, (int)G, (int)K, (int)N, flags, 0) != 0;
    r.x = operand(x, x_ld, any);
    r.w = operand(w, w_ld, any);
    CALL(uem_grouped_fwd, ptr(r.x), x_ld, ptr(r.w), w_ld, ptr(bias), mptr(r.y), ptr(offsets), (int)T, (int)G, (int)K, (int)N,
         flags | (is16(bias) ? UEM_GROUPED_BIAS_BF16 : 0), stream_of(x));
    return r;
}
struct GroupedLinearFn : torch::autograd::Function<GroupedLinearFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& offsets, const std::optional<Tensor>& bias_) {
        const Tensor bias = bias_.value_or(Tensor());
        const Grouped r = grouped_forward(x, weight, offsets, bias);
        ctx->save_for_backward({r.x, r.w, offsets});
        ctx->saved_data["sizes"] = std::vector<int64_t>{x.size(0), weight.size(0), x.size(1), weight.size(1)};
        ctx->saved_data["w16"] = is16(weight);
        ctx->saved_data["b16"] = is16(bias);
        ctx->saved_data["bias"] = bias.defined();
        return r.y;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        no_second_derivative("grouped_linear");
        no_transforms("grouped_linear", {&grads[0]});
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &offsets = saved[2];
        const c10::DeviceGuard guard(x.device());
        const auto sizes = ctx->saved_data["sizes"].toIntVector();
        const int T = (int)sizes[0], G = (int)sizes[1], K = (int)sizes[2], N = (int)sizes[3];
        const bool w16 = ctx->saved_data["w16"].toBool(), b16 = ctx->saved_data["b16"].toBool();
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(3);
        Tensor dx, dw, db;
        if (need_x) dx = at::empty({T, K}, x.options());
        if (need_w || need_b) dw = at::empty({G, N, K}, x.options().dtype(w16 ? at::kBFloat16 : at::kFloat));      // db falls off its products
        if (need_b) db = at::empty({G, N}, x.options().dtype(b16 ? at::kBFloat16 : at::kFloat));
        if (T == 0) {
            if (need_w) dw.zero_();
            if (need_b) db.zero_();
        } else {
            const int flags = grouped_flags(x, offsets);
            const bool any = uem_grouped_any_rows_(T, G, K, N, flags, 1) != 0;
            int dy_ld, w_ld, x_ld;
            const Tensor dy = operand(grads[0], dy_ld, any && !need_w && !need_b);
            if (need_x) {
                const Tensor wr = operand(w, w_ld, any);
                CALL(uem_grouped_dgrad, ptr(dy), dy_ld, ptr(wr), w_ld, mptr(dx), ptr(offsets), T, G, K, N, flags, stream_of(x));
            }
            if (need_w || need_b) {
                const int64_t n = uem_grouped_wgrad_workspace_floats_(T, G, K, N, flags);
                Tensor ws;
                if (n > 0) ws = at::empty({n}, x.options().dtype(at::kFloat));
                const Tensor xr = operand(x, x_ld);
                CALL(uem_grouped_wgrad, ptr(dy), dy_ld, ptr(xr), x_ld, mptr(dw), mptr(db), (float*)mptr(ws), ptr(offsets), T, G, K, N,
                     flags | (w16 ? 0 : UEM_GROUPED_OUT_F32) | (b16 ? UEM_GROUPED_BIAS_BF16 : 0), stream_of(x));
            }
        }
        return {dx, need_w ? dw : Tensor(), Tensor(), db};
    }
};
Tensor grouped_linear(const Tensor& x, const Tensor& weight, const Tensor& offsets, const Tensor& bias) {
    if (x.dim() != 2 || weight.dim() != 3 || weight.size(2) != x.size(1) || weight.numel() == 0)
        refuse("grouped_linear: expected x (rows, in) and weight (groups, out, in), none of groups, out, in zero; got ", x.sizes(), " and ", weight.sizes());
    if (!is_real(x) || !(weight.scalar_type() == x.scalar_type() || (weight.scalar_type() == at::kFloat && is16(x))))
        refuse("grouped_linear: x and weight must be float32, bfloat16, or bfloat16 rows with float32 weights; got ", x.scalar_type(), " and ", weight.scalar_type());
    const int64_t T = x.size(0), G = weight.size(0), N = weight.size(1), K = weight.size(2);
    if (offsets.dim() != 1 || offsets.size(0) != G + 1 || (offsets.scalar_type() != at::kInt && offsets.scalar_type() != at::kLong))
        refuse("grouped_linear: offsets must be int32 or int64 of ", G + 1, " entries, got ", offsets.scalar_type(), " ", offsets.sizes());
    if (bias.defined() && (bias.dim() != 2 || bias.size(0) != G || bias.size(1) != N || !is_real(bias)))
        refuse("grouped_linear: bias must be float32 or bfloat16 of shape (", G, ", ", N, "), got ", bias.scalar_type(), " ", bias.sizes());
    no_transforms("grouped_linear", {&x, &weight, &bias});
    need_gpu({&x, &weight, &offsets, &bias});
    for (const auto& [name, t] : {std::pair<const char*, const Tensor*>{"weight", &weight}, {"offsets", &offsets}, {"bias", &bias}})
        if (t->defined() && t->device() != x.device()) refuse("grouped_linear: ", name, " is on ", t->device(), ", x on ", x.device());
    if (T >= (1 << 30) || G >= (1 << 16) || std::max(K, N) > (1 << 20))
        refuse("grouped_linear: fewer than 2^30 rows and 2^16 groups and at most 2^20 channels, got ", T, ", ", G, ", ", std::max(K, N));
    const Tensor off = offsets.contiguous(), b = bias.defined() ? bias.contiguous() : bias;
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(b))) {
        const c10::DeviceGuard guard(x.device());
        no_outside_graph("grouped_linear", {&x, &weight, &bias});
        return GroupedLinearFn::apply(x, weight, off, maybe(b));
    }
    return grouped_forward(x, weight, off, b).y;
}

// ---- the norm of many tensors ---------------------------------------------------------------------------------------------------------------
// `clip`: scale them in place
Tensor multi_norm(std::vector<Tensor> list, const std::string& what, int kind, bool clip, float max_norm) {
    const at::NoGradGuard no_grad;
    const c10::Device dev = list[0].device();
    const int n = (int)list.size();
    std::vector<uint64_t> ptrs(n);
    std::vector<int64_t> numels(n);
    std::vector<uint8_t> kinds(n);
    std::vector<std::pair<Tensor, Tensor>> copies;
    std::vector<std::pair<uint64_t, uint64_t>> spans;                         // of the gradients themselves
    for (int i = 0; i < n; ++i) {
        Tensor& t = list[i];
        no_transforms(what.c_str(), {&t});
        if (t.layout() != at::kStrided) refuse(what, ": gradients must be dense tensors, got ", t.layout());
        if (clip && t.is_inference() && !c10::InferenceMode::is_enabled()) refuse(what, ": a gradient is an inference tensor: it cannot be scaled in place");
        if (!is_real(t)) refuse(what, ": gradients must be float32 or bfloat16 tensors, got ", t.scalar_type());
        if (t.device() != dev || !t.is_cuda())
            refuse(what, ": all gradients must be on one MI355X device, got ", dev, " and ", t.device(), " (there is no CPU / PyTorch fallback)");
        if (clip && t.numel() > 0) {
            uint64_t last = 0;                                                 // from its first element
            for (int64_t d = 0; d < t.dim(); ++d) {
                if (t.stride(d) == 0 && t.size(d) > 1)
                    refuse(what, ": a gradient of shape ", t.sizes(), ", strides ", t.strides(), " repeats its elements: it cannot be scaled in place");
                last += (uint64_t)(t.size(d) - 1) * t.stride(d);
            }
            const uint64_t first = (uint64_t)t.const_data_ptr();
            spans.emplace_back(first, first + (last + 1) * t.element_size());
        }
        if (!t.is_non_overlapping_and_dense()) {                               // gaps between its elements: summed, and scaled, in a dense copy
            Tensor c = t.contiguous();
            if (clip) copies.emplace_back(t, c);
            t = c;
        }
        ptrs[i] = (uint64_t)t.const_data_ptr();
        numels[i] = t.numel();
        kinds[i] = is16(t) ? 1 : 0;
    }
    if (!copies.empty()) {                                                     // (the library sees the copies only)
        std::sort(spans.begin(), spans.end());
        for (size_t i = 1; i < spans.size(); ++i)
            if (spans[i].first < spans[i - 1].second) refuse(what, ": the memory of two gradients overlaps or interleaves: they cannot be scaled in place");
    }
    const c10::DeviceGuard guard(dev);
    const auto opt = list[0].options();
    const Tensor partial = at::empty({uem_multi_norm_workspace_doubles_(n)}, opt.dtype(at::kDouble)), norm = at::empty({}, opt.dtype(at::kFloat));
    if (clip) {
        CALL(uem_multi_clip, ptrs.data(), numels.data(), kinds.data(), n, kind, partial.data_ptr<double>(), norm.data_ptr<float>(), max_norm, stream_of(norm));
        for (const Tensor& t : list) torch::autograd::impl::bump_version(t);   // written through raw pointers: autograd must see the change
        for (const auto& [to, from] : copies) to.copy_(from);
    } else {
        CALL(uem_multi_norm, ptrs.data(), numels.data(), kinds.data(), n, kind, partial.data_ptr<double>(), norm.data_ptr<float>(), stream_of(norm));
    }
    return norm;
}

// ---- CPython ----------------------------------------------------------------------------------------------------------------------------------
Tensor tensor_arg(PyObject* o, const char* what, const char* name, bool optional = false) {
    if (optional && o == Py_None) return Tensor();
    if (!THPVariable_Check(o)) refuse(what, ": ", name, " must be a tensor, got ", Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}
double double_arg(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}
void count_args(const char* what, Py_ssize_t got, Py_ssize_t want) {
    if (uem_grouped_wgrad_ == nullptr) {
        PyErr_SetString(PyExc_RuntimeError, "uemda_amd._host is not bound to the library: uemda_amd._lib.host() does that");
        throw python_error();
    }
    if (got != want) refuse(what, ": ", want, " arguments expected, got ", got);
}
PyObject* py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count_args("layer_norm", n, 4);
    return THPVariable_Wrap(layer_norm(tensor_arg(a[0], "layer_norm", "x"), tensor_arg(a[1], "layer_norm", "weight", true),
                                       tensor_arg(a[2], "layer_norm", "bias", true), double_arg(a[3])));
    END_HANDLE_TH_ERRORS
}
PyObject* py_grouped_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count_args("grouped_linear", n, 4);
    return THPVariable_Wrap(grouped_linear(tensor_arg(a[0], "grouped_linear", "x"), tensor_arg(a[1], "grouped_linear", "weight"),
                                           tensor_arg(a[2], "grouped_linear", "offsets"), tensor_arg(a[3], "grouped_linear", "bias", true)));
    END_HANDLE_TH_ERRORS
}
// (list of tensors, what, kind, of gradients, max_norm or None) -> norm, or None for an empty list.  `of gradients`: the list holds parameters, their
// .grad is meant, those without one are skipped
PyObject* py_multi_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count_args("multi_norm", n, 5);
    const char* const what = PyUnicode_AsUTF8(a[1]);
    if (what == nullptr || !PyList_Check(a[0])) refuse("multi_norm: a list of tensors and its caller's name expected");
    const int kind = (int)double_arg(a[2]);
    const bool of_grads = PyObject_IsTrue(a[3]) == 1, clip = a[4] != Py_None;
    std::vector<Tensor> list;
    list.reserve(PyList_GET_SIZE(a[0]));
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(a[0]); ++i) {
        PyObject* const o = PyList_GET_ITEM(a[0], i);
        if (!THPVariable_Check(o)) refuse(what, ": expected tensors, got ", Py_TYPE(o)->tp_name);
        const Tensor& t = THPVariable_Unpack(o);
        if (!of_grads) list.push_back(t);
        else if (t.grad().defined()) list.push_back(t.grad());
    }
    if (list.empty()) Py_RETURN_NONE;
    return THPVariable_Wrap(multi_norm(std::move(list), what, kind, clip, clip ? (float)double_arg(a[4]) : 0.f));
    END_HANDLE_TH_ERRORS
}
// (UemError, {entry point: address})
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 2 || !PyDict_Check(a[1])) {
        PyErr_SetString(PyExc_TypeError, "bind(UemError, {entry point: address})");
        return nullptr;
    }
    Py_INCREF(a[0]);
    g_error = a[0];
    auto address = [&](const char* name) {
        PyObject* const v = PyDict_GetItemString(a[1], name);
        void* const p = v ? PyLong_AsVoidPtr(v) : nullptr;
        if (p == nullptr) refuse("_host.bind: no address of ", name);
        return p;
    };
#define UEM_BIND(name) name##_ = reinterpret_cast<decltype(name##_)>(address(#name));
    UEM_HOST_FUNCTIONS(UEM_BIND)
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}
PyObject* py_names(PyObject*, PyObject*) {
    PyObject* const list = PyList_New(0);
#define UEM_NAME(name)                                     \
    {                                                      \
        PyObject* const s = PyUnicode_FromString(#name);   \
        PyList_Append(list, s);                            \
        Py_DECREF(s);                                      \
    }
    UEM_HOST_FUNCTIONS(UEM_NAME)
    return list;
}
PyMethodDef methods[] = {{"bind", (PyCFunction)(void*)py_bind, METH_FASTCALL, nullptr},
                         {"names", py_names, METH_NOARGS, nullptr},
                         {"layer_norm", (PyCFunction)(void*)py_layer_norm, METH_FASTCALL, nullptr},
                         {"grouped_linear", (PyCFunction)(void*)py_grouped_linear, METH_FASTCALL, nullptr},
                         {"multi_norm", (PyCFunction)(void*)py_multi_norm, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
