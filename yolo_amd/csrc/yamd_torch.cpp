// torch binding of the token operators (yolo_amd.tokens): argument checks, allocation of results and workspaces, and the
// autograd nodes over the C ABI.  Host code only.  It exists because of what these operators cost when called from Python:
// a training step of layer norm through a Python autograd function and ctypes took 150 us of host time for 30 us of
// kernels, since the backward pass then has to hand the interpreter over to the autograd thread.
//
// Results and workspaces come from torch's allocator on the current stream of the tensors' device, so calls on different
// streams or inside different captured graphs share nothing.
#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <optional>
#include <sstream>
#include <stdexcept>
#include <string>
#include <unordered_set>
#include <vector>

#include "../../include/yolo_amd.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

struct Error : std::runtime_error {
    using std::runtime_error::runtime_error;
};

template <typename... A>
[[noreturn]] void fail(A &&...parts)
{
    std::ostringstream s;
    (s << ... << parts);
    throw Error(s.str());
}

void check(int rc, const char *what)
{
    if (rc != YAMD_OK) fail(what, " failed (", rc, "): ", yamd_last_error());
}

// The kernels work on a tensor's memory alone: a forward-mode tangent would be dropped, and a trace would hold the result as a
// constant.
void refuse_tangents(const char *what, std::initializer_list<const Tensor *> tensors)
{
    if (at::tracer::impl::is_dispatch_enabled()) fail(what, " cannot be recorded by torch.jit.trace");
    for (const Tensor *t : tensors)
        if (t->defined() && t->_fw_grad(0).defined()) fail(what, " has no forward-mode derivative (an argument carries a tangent)");
}

void require_gpu(const Tensor &t, const char *name, const at::Device *device = nullptr)
{
    if (!t.defined() || !t.is_cuda()) fail(name, " must live on the GPU: yolo_amd has no CPU path");
    if (device && t.device() != *device) fail(name, " is on ", t.device(), ", expected ", *device);
}

void *stream_of(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
int dtype_of(const Tensor &t) { return t.scalar_type() == at::kBFloat16 ? YAMD_BF16 : YAMD_F32; }
bool known_dtype(const Tensor &t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }
Tensor bytes(size_t n, const Tensor &like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }

bool wants_grad(std::initializer_list<const Tensor *> tensors)
{
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor *t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// absent tensors go through autograd as empty optionals
std::optional<Tensor> maybe(const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// the library's gradients carry no graph of their own
void once_only(const char *what)
{
    if (at::GradMode::is_enabled()) fail(what, " cannot be differentiated twice (create_graph=True)");
}

// A leaf has one accumulator for all live graphs that reach it, on the stream of the first.  If that was an eager graph on the
// default stream, autograd would make the default stream wait for a captured one on the way there, which breaks the capture
// and ends the process.  So a captured backward pass stops here when what it leads to holds a node of the default stream.
void refuse_eager_nodes(const char *what, std::initializer_list<const Tensor *> inputs, c10::DeviceIndex device)
{
    using torch::autograd::Node;
    const c10::hip::HIPStream none = c10::hip::getDefaultHIPStream(device);
    if (c10::hip::getCurrentHIPStream(device) == none || c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const auto *asked = torch::autograd::get_current_graph_task_exec_info();     // (empty: all that can be reached)
    std::vector<Node *> todo;
    std::unordered_set<Node *> seen;
    auto visit = [&](Node *n) {
        if (!n || !seen.insert(n).second) return;
        if (asked && !asked->empty()) {
            const auto it = asked->find(n);
            if (it == asked->end() || !it->second.should_execute()) return;
        }
        todo.push_back(n);
    };
    for (const Tensor *t : inputs) {
        if (!t->defined() || !t->requires_grad()) continue;
        visit(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t).get() : t->grad_fn().get());
        while (!todo.empty()) {
            Node *n = todo.back();
            todo.pop_back();
            // (by id: autograd's streams and HIPStream name one device by two types)
            const auto on = n->stream();
            if (on && on->device_index() == device && on->id() == none.id())
                fail(what, ": the backward pass is captured while an eager result of the same leaves is alive (delete it before the capture)");
            for (const auto &e : n->next_edges()) visit(e.function.get());
        }
    }
}

// ---- layer norm ---------------------------------------------------------------------------------------------------------
// row stride of (..., C) taken as evenly spaced rows
int64_t row_stride(const Tensor &t, const char *name)
{
    const int64_t c = t.size(-1);
    int64_t stride = c, span = 0;              // span: elements from one index of the dimension to the next, if rows are even
    if (t.numel() == 0) return c;
    if (c > 1 && t.stride(-1) != 1) fail(name, ": channels must be contiguous, got strides ", t.strides());
    for (int64_t d = t.dim() - 2; d >= 0; --d) {
        if (t.size(d) == 1) continue;
        if (span == 0) stride = t.stride(d);
        else if (t.stride(d) != span) fail(name, ": rows must be evenly spaced, got shape ", t.sizes(), " strides ", t.strides());
        if (stride < c) fail(name, ": rows must not overlap, got strides ", t.strides());
        span = t.stride(d) * t.size(d);
    }
    return stride;
}

struct NormOut {
    Tensor y, mean, rstd;
};

NormOut norm_forward(const Tensor &x, const Tensor &w, const Tensor &b, double eps, bool stats)
{
    const int64_t c = x.size(-1), n = x.numel() / c;
    const c10::DeviceGuard guard(x.device());
    NormOut o;
    o.y = at::empty(x.sizes(), x.options());
    if (stats) {
        o.mean = at::empty({n}, x.options().dtype(at::kFloat));
        o.rstd = at::empty({n}, x.options().dtype(at::kFloat));
    }
    const Tensor &p = w.defined() ? w : b;
    check(yamd_layer_norm(x.data_ptr(), row_stride(x, "x"), ptr(w), ptr(b), p.defined() ? dtype_of(p) : YAMD_F32, (float)eps, o.y.data_ptr(), c,
                          (float *)ptr(o.mean), (float *)ptr(o.rstd), n, (int)c, dtype_of(x), stream_of(x)),
          "layer_norm");
    return o;
}

struct LayerNorm : Function<LayerNorm> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const std::optional<Tensor> &weight, const std::optional<Tensor> &bias, double eps)
    {
        const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
        NormOut o = norm_forward(x, w, b, eps, true);
        ctx->save_for_backward({x, w, b, o.mean, o.rstd});
        return o.y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        once_only("layer_norm");
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &mean = saved[3], &rstd = saved[4];
        const int64_t c = x.size(-1), n = x.numel() / c;
        const c10::DeviceGuard guard(x.device());
        refuse_eager_nodes("layer_norm", {&x, &w, &b}, x.device().index());
        const Tensor dy = grads[0].contiguous();
        Tensor dx, dw, db, ws;
        if (ctx->needs_input_grad(0)) dx = at::empty(x.sizes(), x.options());
        // (absent tensors have no edge)
        if (w.defined() && ctx->needs_input_grad(1)) dw = at::empty_like(w);
        if (b.defined() && ctx->needs_input_grad(w.defined() ? 2 : 1)) db = at::empty_like(b);
        if (n == 0 && !dw.defined() && !db.defined()) return {dx, Tensor(), Tensor(), Tensor()};
        size_t nbytes = 0;
        if (dw.defined() || db.defined()) {
            nbytes = yamd_layer_norm_backward_workspace_bytes(n, (int)c);
            ws = bytes(nbytes, x);
        }
        const Tensor &p = w.defined() ? w : b;
        check(yamd_layer_norm_backward(dy.data_ptr(), c, x.data_ptr(), row_stride(x, "x"), ptr(w), p.defined() ? dtype_of(p) : YAMD_F32,
                                       (const float *)mean.data_ptr(), (const float *)rstd.data_ptr(), ptr(dx), c, ptr(dw), ptr(db), n, (int)c,
                                       dtype_of(x), ptr(ws), nbytes, stream_of(x)),
              "layer_norm_backward");
        return {dx, dw, db, Tensor()};
    }
};

Tensor layer_norm(const Tensor &x, const std::optional<Tensor> &weight, const std::optional<Tensor> &bias, double eps)
{
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    refuse_tangents("layer_norm", {&x, &w, &b});
    require_gpu(x, "x");
    if (!known_dtype(x)) fail("x must be bfloat16 or float32, got ", x.scalar_type());
    if (x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > 16384) fail("x must have 1 to 16384 channels, got shape ", x.sizes());
    const at::Device dev = x.device();
    for (const auto &[t, name] : {std::pair<const Tensor &, const char *>{w, "weight"}, {b, "bias"}}) {
        if (!t.defined()) continue;
        require_gpu(t, name, &dev);
        if (!known_dtype(t) || t.dim() != 1 || t.size(0) != x.size(-1) || !t.is_contiguous())
            fail(name, " must be contiguous (", x.size(-1), ",) bfloat16 or float32, got ", t.sizes(), " ", t.scalar_type());
    }
    if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type())
        fail("weight and bias must have one type, got ", w.scalar_type(), " and ", b.scalar_type());
    if (!(eps >= 0)) fail("eps must not be negative, got ", eps);
    row_stride(x, "x");
    if (wants_grad({&x, &w, &b})) return LayerNorm::apply(x, maybe(w), maybe(b), eps);
    return norm_forward(x, w, b, eps, false).y;
}

// ---- relative position bias ---------------------------------------------------------------------------------------------
Tensor bias_forward(const Tensor &table, const Tensor &bucket_of)
{
    const c10::DeviceGuard guard(table.device());
    const int64_t heads = table.size(1), n = bucket_of.numel();
    Tensor bias = at::empty({heads, n}, table.options().dtype(at::kFloat));
    check(yamd_relative_bias(table.data_ptr(), dtype_of(table), (const int32_t *)bucket_of.data_ptr(), (int)n, (int)heads, (int)table.size(0),
                             (float *)bias.data_ptr(), stream_of(table)),
          "relative_bias");
    return bias;
}

struct RelativeBias : Function<RelativeBias> {
    static Tensor forward(AutogradContext *ctx, const Tensor &table, const Tensor &bucket_of, const Tensor &order, const Tensor &start)
    {
        ctx->save_for_backward({order, start});
        ctx->saved_data["table"] = table;
        return bias_forward(table, bucket_of);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        once_only("relative_bias");
        const variable_list saved = ctx->get_saved_variables();
        const Tensor d = grads[0].contiguous();
        const c10::DeviceGuard guard(d.device());
        const Tensor table = ctx->saved_data["table"].toTensor();
        refuse_eager_nodes("relative_bias", {&table}, d.device().index());
        const int64_t rows = saved[1].numel() - 1, heads = d.size(0);
        Tensor dtable = at::empty({rows, heads}, d.options().dtype(table.scalar_type()));
        check(yamd_relative_bias_backward((const float *)d.data_ptr(), (const int32_t *)saved[0].data_ptr(), (const int32_t *)saved[1].data_ptr(),
                                          (int)d.size(1), (int)heads, (int)rows, dtable.data_ptr(), dtype_of(dtable), stream_of(d)),
              "relative_bias_backward");
        return {dtable, Tensor(), Tensor(), Tensor()};
    }
};

Tensor relative_bias(const Tensor &table, const Tensor &bucket_of, const Tensor &order, const Tensor &start)
{
    refuse_tangents("relative_bias", {&table});
    const at::Device dev = bucket_of.device();
    const int64_t rows = start.numel() - 1;
    require_gpu(bucket_of, "position");
    require_gpu(table, "table", &dev);
    if (!known_dtype(table) || table.dim() != 2 || table.size(0) != rows || table.size(1) < 1 || table.size(1) > 65535 || !table.is_contiguous())
        fail("table must be contiguous (", rows, ", heads) bfloat16 or float32, got ", table.sizes(), " ", table.scalar_type());
    if (wants_grad({&table})) return RelativeBias::apply(table, bucket_of, order, start);
    return bias_forward(table, bucket_of);
}

// ---- attention ----------------------------------------------------------------------------------------------------------
yamd_tokens tokens(const Tensor &t)
{
    // (the stride of a dimension of one element is never used; torch leaves any value there)
    return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}

yamd_attention_desc descriptor(const Tensor &q, const Tensor &k, double scale, int64_t h, int64_t w)
{
    yamd_attention_desc d;
    d.batch = (int)q.size(0);
    d.heads = (int)q.size(2);
    d.kv_heads = (int)k.size(2);
    d.head_dim = (int)q.size(3);
    d.q_len = (int)q.size(1);
    d.k_len = (int)k.size(1);
    d.map_h = (int)h;
    d.map_w = (int)w;
    d.scale = (float)scale;
    return d;
}

struct AttentionOut {
    Tensor o, lse, exact;
};

AttentionOut attention_forward(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &mask, const Tensor &bias, double scale, int64_t h,
                               int64_t w, bool stats)
{
    const c10::DeviceGuard guard(q.device());
    AttentionOut r;
    const bool nothing = q.numel() == 0 || k.numel() == 0;       // no query, or no key: rows left without keys are zero
    if (stats) {
        const auto opt = q.options().dtype(at::kFloat);
        r.lse = nothing ? at::full({q.size(0), q.size(2), q.size(1)}, -std::numeric_limits<float>::infinity(), opt)
                        : at::empty({q.size(0), q.size(2), q.size(1)}, opt);
    }
    if (nothing) {
        r.o = at::zeros(q.sizes(), q.options());
        return r;
    }
    r.o = at::empty(q.sizes(), q.options());
    if (stats)
        r.exact = at::empty({q.size(0), q.size(2), q.size(1), q.size(3)}, q.options().dtype(at::kFloat));
    const yamd_attention_desc d = descriptor(q, k, scale, h, w);
    const yamd_tokens tq = tokens(q), tk = tokens(k), tv = tokens(v), to = tokens(r.o);
    const size_t nbytes = yamd_attention_workspace_bytes(&d, bias.defined());
    Tensor ws;
    if (nbytes) ws = bytes(nbytes, q);
    check(yamd_attention(&d, &tq, &tk, &tv, (const uint8_t *)ptr(mask), mask.defined() ? mask.stride(0) : 0, (const float *)ptr(bias), &to,
                         (float *)ptr(r.exact), (float *)ptr(r.lse), ptr(ws), nbytes, stream_of(q)),
          "attention");
    return r;
}

struct Attention : Function<Attention> {
    static Tensor forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const std::optional<Tensor> &bias_,
                          const std::optional<Tensor> &mask_, double scale, int64_t h, int64_t w)
    {
        const Tensor bias = bias_.value_or(Tensor()), mask = mask_.value_or(Tensor());
        AttentionOut r = attention_forward(q, k, v, mask, bias, scale, h, w, true);
        // (not o: the caller may change it)
        ctx->save_for_backward({q, k, v, bias, mask, r.lse, r.exact});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["h"] = h;
        ctx->saved_data["w"] = w;
        return r.o;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        once_only("attention");
        const variable_list s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2], &bias = s[3], &mask = s[4], &lse = s[5], &exact = s[6];
        const c10::DeviceGuard guard(q.device());
        refuse_eager_nodes("attention", {&q, &k, &v, &bias}, q.device().index());
        const bool nothing = q.numel() == 0 || k.numel() == 0;
        auto result = [&](const Tensor &t) { return nothing ? at::zeros(t.sizes(), t.options()) : at::empty(t.sizes(), t.options()); };
        Tensor dq = result(q), dk = result(k), dv = result(v), dbias;
        if (bias.defined() && ctx->needs_input_grad(3)) dbias = result(bias);
        if (!nothing) {
            Tensor go = grads[0].contiguous();
            if (reinterpret_cast<uintptr_t>(go.data_ptr()) % 16) go = go.clone();      // (a piece of a longer vector)
            const yamd_attention_desc d = descriptor(q, k, ctx->saved_data["scale"].toDouble(), ctx->saved_data["h"].toInt(),
                                                     ctx->saved_data["w"].toInt());
            const yamd_tokens tq = tokens(q), tk = tokens(k), tv = tokens(v), tg = tokens(go), tdq = tokens(dq), tdk = tokens(dk), tdv = tokens(dv);
            const size_t nbytes = yamd_attention_backward_workspace_bytes(&d, dbias.defined());
            const Tensor ws = bytes(nbytes, q);
            check(yamd_attention_backward(&d, &tq, &tk, &tv, (const uint8_t *)ptr(mask), mask.defined() ? mask.stride(0) : 0,
                                          (const float *)ptr(bias), nullptr, (const float *)ptr(exact),
                                          (const float *)lse.data_ptr(), &tg, &tdq, &tdk, &tdv,
                                          (float *)ptr(dbias), ws.data_ptr(), nbytes, stream_of(q)),
                  "attention_backward");
        }
        return {dq, dk, dv, dbias, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

void check_tokens(const Tensor &t, const char *name, const at::Device &dev, at::IntArrayRef shape)
{
    require_gpu(t, name, &dev);
    if (t.scalar_type() != at::kBFloat16) fail(name, " must be bfloat16, got ", t.scalar_type());
    if (t.sizes() != shape) fail(name, " must be ", shape, ", got ", t.sizes());
    if (t.numel() == 0) return;
    bool ok = (t.stride(3) == 1) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int d = 0; d < 3; ++d) ok = ok && (t.size(d) == 1 || (t.stride(d) % 8 == 0 && t.stride(d) >= 8));
    if (!ok) fail(name, ": channels must be contiguous and tokens, heads and images start at multiples of 16 bytes (strides ", t.strides(), ")");
}

Tensor attention(const Tensor &q, const Tensor &k, const Tensor &v, std::optional<double> scale_, const std::optional<Tensor> &key_mask,
                 const std::optional<Tensor> &bias_, int64_t h, int64_t w)
{
    const Tensor mask = key_mask.value_or(Tensor()), bias = bias_.value_or(Tensor());
    refuse_tangents("attention", {&q, &k, &v, &bias});
    require_gpu(q, "q");
    if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4)
        fail("q must be (batch, tokens, heads, channels) and k, v (batch, tokens, kv_heads, channels)");
    const int64_t b = q.size(0), lq = q.size(1), heads = q.size(2), d = q.size(3), lk = k.size(1), kv_heads = k.size(2);
    if (heads < 1 || kv_heads < 1 || heads % kv_heads) fail(heads, " heads do not share ", kv_heads, " key heads evenly");
    if (d < 8 || d > 128 || d % 8) fail("channels per head must be a multiple of 8 up to 128, got ", d);
    if (std::max(lq, lk) > (1 << 24) || b > (1 << 20) || heads > (1 << 20)) fail("attention is too large: q ", q.sizes(), ", k ", k.sizes());
    const at::Device dev = q.device();
    check_tokens(q, "q", dev, {b, lq, heads, d});
    check_tokens(k, "k", dev, {b, lk, kv_heads, d});
    check_tokens(v, "v", dev, {b, lk, kv_heads, d});
    const double scale = scale_.value_or(1.0 / std::sqrt((double)d));
    if (!(scale >= 1e-20 && scale <= 1e20)) fail("scale must be between 1e-20 and 1e20, got ", scale);
    if (mask.defined()) {
        require_gpu(mask, "key_mask", &dev);
        if (mask.scalar_type() != at::kBool || mask.dim() != 2 || mask.size(0) != b || mask.size(1) != lk || (lk > 1 && mask.stride(1) != 1) ||
            (b > 1 && lk > 0 && mask.stride(0) < lk))
            fail("key_mask must be bool (", b, ", ", lk, ") with contiguous rows, got ", mask.sizes(), " ", mask.scalar_type());
    }
    if (bias.defined()) {
        require_gpu(bias, "bias", &dev);
        if (lq != lk || lq != h * w) fail("a position bias needs Lq == Lk == ", h, " * ", w, ", got ", lq, " and ", lk);
        if (bias.scalar_type() != at::kFloat || bias.dim() != 2 || bias.size(0) != heads || bias.size(1) != (2 * h - 1) * (2 * w - 1) ||
            !bias.is_contiguous())
            fail("bias must be contiguous float32 (", heads, ", ", (2 * h - 1) * (2 * w - 1), "), got ", bias.sizes(), " ", bias.scalar_type());
    }
    if (wants_grad({&q, &k, &v, &bias})) return Attention::apply(q, k, v, maybe(bias), maybe(mask), scale, h, w);
    return attention_forward(q, k, v, mask, bias, scale, h, w, false).o;
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m)
{
    // errors of this module are the package's own (kept for the life of the process)
    static PyObject *const yamd_error = py::object(py::module_::import("yolo_amd.lib").attr("YamdError")).release().ptr();
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Error &e) {
            PyErr_SetString(yamd_error, e.what());
        }
    });
    m.def("layer_norm", &layer_norm, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("eps"));
    m.def("relative_bias", &relative_bias, py::arg("table"), py::arg("bucket_of"), py::arg("order"), py::arg("start"));
    m.def("attention", &attention, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("scale"), py::arg("key_mask"), py::arg("bias"),
          py::arg("map_h"), py::arg("map_w"));
}
