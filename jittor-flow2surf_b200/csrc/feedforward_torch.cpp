// PyTorch binding of the 8-bit feed-forward operators (flow2surf_b200/
// feedforward.py documents them): checks of arguments, output tensors, streams
// and autograd around the C entries of libflow2surf_sm100.so. A decode step's
// norm or product takes 2 to 5 us on the device, less than Python needs to
// prepare one call through ctypes (13 to 20 us; a training step's backward
// through a Python autograd function 100 us), so these run natively.
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros_like.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <sstream>

#include "flow2surf_b200.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ValueError for what the caller can mend, RuntimeError otherwise, as _lib.check
// (whose subclass of it a backward, which runs without the interpreter's lock,
// cannot raise).
void check(int status) {
    if (status == F2S_OK) return;
    const std::string message = f2s_last_error();
    TORCH_CHECK_VALUE(status != F2S_ERR_INVALID_ARGUMENT && status != F2S_ERR_UNSUPPORTED, message);
    TORCH_CHECK(false, "[status ", status, "] ", message);
}

std::string shape_of(const Tensor& t) {
    std::ostringstream s;
    s << "(";
    for (int64_t i = 0; i < t.dim(); ++i) s << (i ? ", " : "") << t.size(i);
    s << (t.dim() == 1 ? ",)" : ")");
    return s.str();
}

int dtype_code(at::ScalarType type) {
    switch (type) {
        case at::kFloat: return F2S_DTYPE_F32;
        case at::kBFloat16: return F2S_DTYPE_BF16;
        case at::kHalf: return F2S_DTYPE_F16;
        default:
            TORCH_CHECK_VALUE(false, "expected float32, bfloat16 or float16, got ", c10::toString(type));
    }
}

void check_rows(const char* name, const Tensor& t) {
    TORCH_CHECK_VALUE(t.dim() >= 1 && t.size(-1) >= 1, name,
                      " must be (..., channels) with at least one channel, got ", shape_of(t));
    TORCH_CHECK_VALUE(t.size(-1) <= INT32_MAX, name, " has too many channels: ", shape_of(t));
}

void check_device(const Tensor& first, std::initializer_list<const Tensor*> others) {
    TORCH_CHECK_VALUE(first.is_cuda(), "flow2surf_b200 operators take CUDA tensors (no CPU path)");
    for (const Tensor* t : others) {
        if (!t || !t->defined()) continue;
        TORCH_CHECK_VALUE(t->is_cuda(), "flow2surf_b200 operators take CUDA tensors (no CPU path)");
        TORCH_CHECK_VALUE(t->device() == first.device(), "tensors lie on different devices: ", first.device(),
                          " and ", t->device());
    }
}

bool needs_grad(std::initializer_list<const Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t && t->defined() && t->requires_grad()) return true;
    return false;
}

// Tangents of forward-mode differentiation, which would be lost (and read as zeros):
// they come with or without requires_grad, and torch.no_grad() leaves them on.
void refuse_tangents(std::initializer_list<const Tensor*> tensors) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor* t : tensors)
        TORCH_CHECK_VALUE(!(t && t->defined() && t->_fw_grad(/*level=*/0).defined()),
                          "the 8-bit feed-forward operators have no forward-mode derivative");
}

// A (..., channels) tensor read as rows of one pitch: as it is where its last
// dimension has stride 1 and its rows lie evenly, else copied.
struct Rows {
    Tensor t;
    int64_t rows, pitch;
    explicit Rows(const Tensor& from) : t(from) {
        const int64_t width = t.size(-1), dims = t.dim();
        rows = t.numel() / width;
        pitch = width;
        if (t.is_contiguous()) return;
        bool even = dims >= 2 && t.stride(-1) == 1 && t.stride(-2) >= width;
        for (int64_t i = 0; even && i < dims - 2; ++i) even = t.stride(i) == t.stride(i + 1) * t.size(i + 1);
        if (even) pitch = t.stride(-2);
        else t = t.contiguous();
    }
    void* data() const { return t.data_ptr(); }
};

// The current stream of the tensors' device, which is made the current device.
struct Launch {
    c10::cuda::CUDAGuard guard;
    explicit Launch(const Tensor& t) : guard(t.device()) {}
    void* stream() const { return c10::cuda::getCurrentCUDAStream().stream(); }
};

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor contiguous_like(const Tensor& t) { return at::empty_like(t, {}, at::MemoryFormat::Contiguous); }

std::vector<int64_t> with_width(const Tensor& t, int64_t width) {
    std::vector<int64_t> shape = t.sizes().vec();
    shape.back() = width;
    return shape;
}

// ---- 8-bit rows ----

struct Eight {
    Tensor values, scale;
    int64_t pitch;
    int8_t* q() const { return static_cast<int8_t*>(values.data_ptr()); }
    float* s() const { return static_cast<float*>(scale.data_ptr()); }
    std::pair<Tensor, Tensor> both() const { return {values, scale}; }
};

// Unset rows with the leading shape of `like`, each from a multiple of 16 bytes.
Eight empty_eight(const Tensor& like, int64_t width) {
    const int64_t pitch = (width + 15) / 16 * 16;
    Tensor values = at::empty(with_width(like, pitch), like.options().dtype(at::kChar));
    if (pitch != width) values = values.narrow(-1, 0, width);
    return {values, at::empty(like.sizes().slice(0, like.dim() - 1), like.options().dtype(at::kFloat)), pitch};
}

void check_eight(const char* name, const Tensor& values, const Tensor& scale) {
    check_rows(name, values);
    TORCH_CHECK_VALUE(values.scalar_type() == at::kChar && scale.scalar_type() == at::kFloat, name,
                      " must hold int8 values and float32 scales, got ", c10::toString(values.scalar_type()), " and ",
                      c10::toString(scale.scalar_type()));
    TORCH_CHECK_VALUE(scale.sizes() == values.sizes().slice(0, values.dim() - 1), name, ": scales ", shape_of(scale),
                      " do not match values ", shape_of(values));
    check_device(values, {&scale});
    TORCH_CHECK_VALUE(!needs_grad({&scale}), name,
                      ": 8-bit rows have no gradient, their scales neither; call under torch.no_grad()");
}

std::pair<Tensor, Tensor> quantize_rows(const Tensor& x) {
    check_rows("x", x);
    const int code = dtype_code(x.scalar_type());
    refuse_tangents({&x});
    check_device(x, {});
    TORCH_CHECK_VALUE(!needs_grad({&x}), "8-bit rows have no gradient; call quantize_rows under torch.no_grad()");
    Eight out = empty_eight(x, x.size(-1));
    if (x.numel() == 0) return out.both();
    const Rows r(x);
    const Launch launch(x);
    check(f2s_quantize_rows(r.data(), r.pitch, code, r.rows, (int)x.size(-1), out.q(), out.pitch, out.s(),
                            launch.stream()));
    return out.both();
}

Tensor dequantize_rows(const Tensor& values, const Tensor& scale, at::ScalarType type) {
    const int code = dtype_code(type);
    refuse_tangents({&scale});
    check_eight("rows", values, scale);
    Tensor out = at::empty(values.sizes(), values.options().dtype(type));
    if (out.numel() == 0) return out;
    const Rows r(values);
    const Tensor s = scale.contiguous();
    const Launch launch(values);
    const int width = (int)values.size(-1);
    check(f2s_dequantize_rows(static_cast<const int8_t*>(r.data()), r.pitch, static_cast<const float*>(s.data_ptr()),
                              r.rows, width, out.data_ptr(), width, code, launch.stream()));
    return out;
}

Tensor linear_int8(const Tensor& xv, const Tensor& xs, const Tensor& wv, const Tensor& ws,
                   const optional<Tensor>& bias, at::ScalarType type) {
    const int code = dtype_code(type);
    refuse_tangents({&xs, &ws, bias ? &*bias : nullptr});
    check_eight("x", xv, xs);
    check_eight("weight", wv, ws);
    TORCH_CHECK_VALUE(wv.dim() == 2, "weight must be (cols, K), got ", shape_of(wv));
    const int64_t cols = wv.size(0), K = wv.size(1);
    TORCH_CHECK_VALUE(xv.size(-1) == K, "x has ", xv.size(-1), " channels, weight ", K);
    check_device(xv, {&wv, bias ? &*bias : nullptr});
    if (bias) {
        TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == cols && bias->scalar_type() == type, "bias must be (",
                          cols, ",) of ", c10::toString(type), ", got ", shape_of(*bias), " of ",
                          c10::toString(bias->scalar_type()));
        TORCH_CHECK_VALUE(!needs_grad({&*bias}),
                          "the 8-bit product has no gradient; call linear_int8 under torch.no_grad()");
    }
    Tensor out = at::empty(with_width(xv, cols), xv.options().dtype(type));
    if (out.numel() == 0) return out;
    const Rows x(xv), w(wv);
    TORCH_CHECK_VALUE(x.rows <= INT32_MAX - 255 && cols <= INT32_MAX - 255,
                      "linear_int8 takes at most 2^31 - 256 rows and columns");
    const Tensor xc = xs.contiguous(), wc = ws.contiguous(), b = bias ? bias->contiguous() : Tensor();
    const Launch launch(xv);
    check(f2s_linear_int8(static_cast<const int8_t*>(x.data()), x.pitch, static_cast<const float*>(xc.data_ptr()),
                          static_cast<const int8_t*>(w.data()), w.pitch, static_cast<const float*>(wc.data_ptr()),
                          data(b), out.data_ptr(), cols, code, (int)x.rows, (int)cols, (int)K, launch.stream()));
    return out;
}

// ---- RMS norm ----

int check_norm(const Tensor& x, const Tensor& weight, const Tensor& residual) {
    check_rows("x", x);
    const int code = dtype_code(x.scalar_type());
    TORCH_CHECK_VALUE(weight.dim() == 1 && weight.size(0) == x.size(-1) && weight.scalar_type() == x.scalar_type(),
                      "weight must be (", x.size(-1), ",) of ", c10::toString(x.scalar_type()), ", got ",
                      shape_of(weight), " of ", c10::toString(weight.scalar_type()));
    TORCH_CHECK_VALUE(!residual.defined() ||
                          (residual.sizes() == x.sizes() && residual.scalar_type() == x.scalar_type()),
                      "residual must be ", shape_of(x), " of ", c10::toString(x.scalar_type()), ", got ",
                      residual.defined() ? shape_of(residual) : "", " of ",
                      residual.defined() ? c10::toString(residual.scalar_type()) : "");
    refuse_tangents({&x, &weight, &residual});
    check_device(x, {&weight, &residual});
    return code;
}

// (normed, stream); the stream is x without a residual.
std::pair<Tensor, Tensor> norm_forward(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps,
                                       int code) {
    Tensor normed = contiguous_like(x);
    Tensor stream = residual.defined() ? contiguous_like(x) : x;
    if (x.numel() == 0) return {normed, stream};
    const Rows r(x);
    optional<Rows> added;
    if (residual.defined()) added.emplace(residual);
    const Tensor w = weight.contiguous();
    const Launch launch(x);
    check(f2s_add_rms_norm(r.data(), r.pitch, added ? added->data() : nullptr, added ? added->pitch : 0, w.data_ptr(),
                           code, r.rows, (int)x.size(-1), (float)eps, added ? stream.data_ptr() : nullptr,
                           normed.data_ptr(), launch.stream()));
    return {normed, stream};
}

// Gradients of a step that asks for a second derivative raise once one is taken.
variable_list once_differentiable(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    for (Tensor& g : grads)
        if (g.defined()) g = g.detach().set_requires_grad(true);
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "the 8-bit feed-forward operators have no second derivative", (int64_t)grads.size());
    return (*error)(std::move(grads));
}

// The backward reads the stream; the norm's reciprocal root is recomputed from
// it, so no statistics are kept.
struct AddRmsNorm : torch::autograd::Function<AddRmsNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                                 const optional<Tensor>& added, double eps, int64_t code) {
        const Tensor residual = added.value_or(Tensor());
        ctx->set_materialize_grads(false);
        auto [normed, stream] = norm_forward(x, weight, residual, eps, (int)code);
        ctx->save_for_backward({stream, weight});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["code"] = code;
        ctx->saved_data["added"] = residual.defined();
        if (residual.defined()) return {normed, stream};
        return {normed};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &stream = saved[0], &weight = saved[1], &dy = grads[0];
        const Tensor dstream = grads.size() > 1 ? grads[1] : Tensor();
        const bool need_x = ctx->needs_input_grad(0), need_weight = ctx->needs_input_grad(1),
                   need_residual = ctx->saved_data["added"].toBool() && ctx->needs_input_grad(2);
        Tensor dx, dweight;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            if (!dy.defined()) {  // only the stream was used
                dx = dstream;
                if (need_weight) dweight = at::zeros_like(weight);
            } else {
                dx = contiguous_like(stream);
                if (need_weight) dweight = at::empty(weight.sizes(), weight.options());
                if (stream.numel() == 0) {
                    if (need_weight) dweight.zero_();
                } else {
                    const Rows s(stream), d(dy);
                    optional<Rows> ds;
                    if (dstream.defined()) ds.emplace(dstream);
                    const Tensor w = weight.contiguous();
                    const int width = (int)stream.size(-1);
                    const Launch launch(stream);
                    size_t bytes = 0;
                    Tensor workspace;
                    if (need_weight) {
                        check(f2s_add_rms_norm_backward_workspace_bytes(s.rows, width, &bytes));
                        workspace = at::empty({(int64_t)bytes}, stream.options().dtype(at::kByte));
                    }
                    check(f2s_add_rms_norm_backward(s.data(), s.pitch, w.data_ptr(), (int)ctx->saved_data["code"].toInt(),
                                                    s.rows, width, (float)ctx->saved_data["eps"].toDouble(), d.data(),
                                                    d.pitch, ds ? ds->data() : nullptr, ds ? ds->pitch : 0,
                                                    dx.data_ptr(), data(dweight), data(workspace), bytes,
                                                    launch.stream()));
                }
            }
        }
        return once_differentiable({need_x ? dx : Tensor(), dweight, need_residual ? dx : Tensor(), Tensor(), Tensor()});
    }
};

std::pair<Tensor, Tensor> add_rms_norm(const Tensor& x, const Tensor& weight, const optional<Tensor>& residual,
                                       double eps) {
    const Tensor r = residual.value_or(Tensor());
    const int code = check_norm(x, weight, r);
    if (!needs_grad({&x, &weight, &r})) return norm_forward(x, weight, r, eps, code);
    variable_list out = AddRmsNorm::apply(x, weight, residual, eps, (int64_t)code);
    return {out[0], out.size() > 1 ? out[1] : x};
}

std::tuple<Tensor, Tensor, Tensor> add_rms_norm_int8(const Tensor& x, const Tensor& weight,
                                                     const optional<Tensor>& residual, double eps) {
    const Tensor r = residual.value_or(Tensor());
    const int code = check_norm(x, weight, r);
    TORCH_CHECK_VALUE(!needs_grad({&x, &weight, &r}),
                      "8-bit rows have no gradient; call add_rms_norm_int8 under torch.no_grad(), or add_rms_norm");
    Eight out = empty_eight(x, x.size(-1));
    Tensor stream = r.defined() ? contiguous_like(x) : x;
    if (x.numel() == 0) return {out.values, out.scale, stream};
    const Rows from(x);
    optional<Rows> added;
    if (r.defined()) added.emplace(r);
    const Tensor w = weight.contiguous();
    const Launch launch(x);
    check(f2s_add_rms_norm_int8(from.data(), from.pitch, added ? added->data() : nullptr, added ? added->pitch : 0,
                                w.data_ptr(), code, from.rows, (int)x.size(-1), (float)eps,
                                added ? stream.data_ptr() : nullptr, out.q(), out.pitch, out.s(), launch.stream()));
    return {out.values, out.scale, stream};
}

// ---- SwiGLU ----

int check_projected(const Tensor& p) {
    check_rows("projected", p);
    TORCH_CHECK_VALUE(p.size(-1) % 2 == 0, "projected must be (..., 2 H) = [gate | value], got ", shape_of(p));
    const int code = dtype_code(p.scalar_type());
    refuse_tangents({&p});
    check_device(p, {});
    return code;
}

Tensor swiglu_forward(const Tensor& projected, int code, const Tensor& kept, const Tensor& scales) {
    const int64_t hidden = projected.size(-1) / 2;
    Tensor out = at::empty(with_width(projected, hidden), projected.options());
    if (out.numel() == 0) return out;
    const Rows p(projected);
    const Launch launch(projected);
    check(f2s_swiglu(p.data(), p.pitch, code, p.rows, (int)hidden, out.data_ptr(), static_cast<int8_t*>(data(kept)),
                     static_cast<float*>(data(scales)), launch.stream()));
    return out;
}

struct SwiGlu : torch::autograd::Function<SwiGlu> {
    static Tensor forward(AutogradContext* ctx, const Tensor& projected, bool keep8, int64_t code) {
        const int64_t hidden = projected.size(-1) / 2;
        ctx->saved_data["code"] = code;
        ctx->saved_data["shape"] = projected.sizes();
        if (!keep8) {
            ctx->save_for_backward({projected});
            return swiglu_forward(projected, (int)code, Tensor(), Tensor());
        }
        const int64_t groups =
            projected.numel() / (2 * hidden) * ((hidden + F2S_SWIGLU_GROUP - 1) / F2S_SWIGLU_GROUP);
        Tensor kept = at::empty({groups * 2 * F2S_SWIGLU_GROUP}, projected.options().dtype(at::kChar));
        Tensor scales = at::empty({2 * groups}, projected.options().dtype(at::kFloat));
        ctx->save_for_backward({kept, scales});
        return swiglu_forward(projected, (int)code, kept, scales);
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
        const Tensor& dy = grads[0];
        Tensor grad;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            grad = at::empty(shape, dy.options());
            if (grad.numel()) {
                const Rows d(dy);
                const bool kept = saved.size() > 1;
                optional<Rows> p;
                if (!kept) p.emplace(saved[0]);
                const Launch launch(dy);
                check(f2s_swiglu_backward(p ? p->data() : nullptr, p ? p->pitch : 0,
                                          kept ? static_cast<const int8_t*>(saved[0].data_ptr()) : nullptr,
                                          kept ? static_cast<const float*>(saved[1].data_ptr()) : nullptr, d.data(),
                                          d.pitch, (int)ctx->saved_data["code"].toInt(), d.rows,
                                          (int)(shape.back() / 2), grad.data_ptr(), launch.stream()));
            }
        }
        return once_differentiable({grad, Tensor(), Tensor()});
    }
};

Tensor swiglu(const Tensor& projected, bool keep8) {
    const int code = check_projected(projected);
    if (needs_grad({&projected})) return SwiGlu::apply(projected, keep8, (int64_t)code);
    return swiglu_forward(projected, code, Tensor(), Tensor());
}

std::pair<Tensor, Tensor> swiglu_int8(const Tensor& projected) {
    const int code = check_projected(projected);
    TORCH_CHECK_VALUE(!needs_grad({&projected}),
                      "8-bit rows have no gradient; call swiglu_int8 under torch.no_grad(), or swiglu");
    const int64_t hidden = projected.size(-1) / 2;
    Eight out = empty_eight(projected, hidden);
    if (projected.numel() == 0) return out.both();
    const Rows p(projected);
    const Launch launch(projected);
    check(f2s_swiglu_int8(p.data(), p.pitch, code, p.rows, (int)hidden, out.q(), out.pitch, out.s(), launch.stream()));
    return out.both();
}

}  // namespace

PYBIND11_MODULE(_feedforward, m) {
    m.doc() = "Native side of flow2surf_b200.feedforward.";
    m.def("quantize_rows", &quantize_rows);
    m.def("dequantize_rows", &dequantize_rows);
    m.def("linear_int8", &linear_int8);
    m.def("add_rms_norm", &add_rms_norm);
    m.def("add_rms_norm_int8", &add_rms_norm_int8);
    m.def("swiglu", &swiglu);
    m.def("swiglu_int8", &swiglu_int8);
}
