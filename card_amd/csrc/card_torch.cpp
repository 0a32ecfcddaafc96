// card_torch.cpp - the layer operators as torch calls: argument checks, outputs from torch's allocator, the current stream,
// and the nodes of the autograd graph, over the C ABI of libcard_hip.so (whose functions Python hands over by address: this
// module links no HIP code and follows whichever library card_amd/_lib.py loaded).
//
// Why not ctypes, as for the sampler: these calls take 3 to 20 us on the device, and a Python call with its checks, outputs
// and launch took 7 to 12 us, one that goes through a Python autograd node 81 us forward and backward.
#include <torch/extension.h>
#include <ATen/TracerMode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "card_hip.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

struct CardErr : std::runtime_error {
    using std::runtime_error::runtime_error;
};
template <typename... Args> [[noreturn]] void refuse(const Args&... args) { throw CardErr(c10::str(args...)); }

struct {
    decltype(&card_last_error) last_error;
    decltype(&card_dropout) dropout;
    decltype(&card_dropout_backward) dropout_backward;
    decltype(&card_rms_norm) rms_norm;
    decltype(&card_rms_norm_backward) rms_norm_backward;
    decltype(&card_rms_norm_backward_workspace_bytes) rms_norm_backward_workspace_bytes;
    decltype(&card_linear4_forward) linear4_forward;
    decltype(&card_linear4_workspace_bytes) linear4_workspace_bytes;
} lib;
PyObject* card_error;

void check(int status, const char* what) {
    if (status != CARD_OK) refuse(what, " failed (", status, "): ", lib.last_error());
}

int dtype_of(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kFloat: return CARD_DTYPE_F32;
        case at::kBFloat16: return CARD_DTYPE_BF16;
        case at::kHalf: return CARD_DTYPE_F16;
        default: refuse(name, ": dtype ", t.scalar_type(), " is none of float32, bfloat16, float16");
    }
}
void on_gpu(const Tensor& t) {
    if (!t.is_cuda())
        refuse("card_amd runs on an AMD GPU only (the tensor is on '", t.device().str(), "'); there is no CPU fallback. Move the model and inputs to cuda.");
}
void same(const Tensor& t, const Tensor& like, at::IntArrayRef shape, const char* name) {
    if (t.sizes() != shape || t.scalar_type() != like.scalar_type() || t.device() != like.device())
        refuse(name, ": expected ", shape, " ", like.scalar_type(), " on ", like.device().str(), ", got ", t.sizes(), " ", t.scalar_type(), " on ", t.device().str());
}
Tensor dense(const OptTensor& t) { return t ? t->contiguous() : Tensor(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
// What would vanish without an error: a tangent (forward-mode derivative) of an input, and the kernels themselves in a trace, which
// sees torch's calls only and would keep the outputs as they were allocated.
template <typename... T> void check_mode(const char* what, const T&... inputs) {
    if (at::tracer::impl::is_dispatch_enabled()) refuse(what, ": torch.jit.trace does not see the kernels; call it outside the trace");
    const auto dual = [](const OptTensor& t) { return t && t->defined() && t->_fw_grad(0).defined(); };
    if ((dual(inputs) || ...)) refuse(what, " has no forward-mode derivative");
}
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool capturing(const c10::hip::HIPStream& s) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    return hipStreamIsCapturing(s.stream(), &status) == hipSuccess && status != hipStreamCaptureStatusNone;
}
// What a backward pass is refused for.  A leaf's gradient node remembers the stream it was made on, and lives as long as any
// graph of the leaf.  Into a capture that began after it, the engine would draw that stream with a wait that is not allowed
// there, and the process would not survive the capture's end.
void check_backward(const char* what, const torch::autograd::tensor_list& grads) {
    for (const Tensor& g : grads) check_mode(what, g);
    if (at::GradMode::is_enabled()) refuse(what, ": the backward pass is of first order only (create_graph=True asks for more)");
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    const auto current = c10::hip::getCurrentHIPStream();
    if (!capturing(current)) return;
    for (size_t i = 0; i < node->num_outputs(); ++i) {
        const auto& next = node->next_edge(i).function;
        if (!next || !node->task_should_compute_output(i)) continue;
        const auto stream = next->stream();
        if (!stream || (stream->id() == current.id() && stream->device_index() == current.device_index())) continue;
        const c10::hip::HIPStream other(c10::hip::HIPStream::UNCHECKED, c10::Stream(c10::Stream::UNSAFE, current.device(), stream->id()));
        if (stream->id() == 0 || !capturing(other))          // 0: the default stream, which is never captured
            refuse(what, ": this backward pass is being captured, but an input's gradient belongs to another stream: a graph of the same "
                   "tensors from before the capture is still alive. Drop its results first, or make them on the capture's stream");
    }
}

// ------------------------------------------------------------------------------------------------ dropout
struct DropCall {
    int dtype;
    int64_t rows, cols;
    int n_z;
    double p;
    uint64_t seed, elem_offset;
    int draw;
};
Tensor drop_forward(const Tensor& x, const Tensor& residual, const Tensor& state, const DropCall& c) {
    c10::DeviceGuard guard(x.device());
    Tensor y;
    if (c.n_z == 1) {
        y = at::empty_like(x, at::MemoryFormat::Contiguous);
    } else {
        auto shape = x.sizes().vec();
        shape.insert(shape.end() - 1, c.n_z);
        y = at::empty(shape, x.options());
    }
    check(lib.dropout(ptr(x), ptr(residual), ptr(y), c.dtype, c.rows, c.cols, c.n_z, c.p, c.seed, c.elem_offset, (const uint64_t*)ptr(state), c.draw, stream_of(x)),
          "card_dropout");
    return y;
}
struct Dropout : torch::autograd::Function<Dropout> {
    // x and residual as the caller has them: a copy made ahead of this node would be a node between it and the leaf (check_backward)
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& residual, const OptTensor& state, int64_t dtype,
                          int64_t rows, int64_t cols, int64_t n_z, double p, int64_t seed, int64_t elem_offset, int64_t draw) {
        auto& d = ctx->saved_data;
        d["call"] = std::vector<int64_t>{dtype, rows, cols, n_z, seed, elem_offset, draw, residual.has_value()};
        d["p"] = p;
        d["shape"] = x.sizes().vec();
        if (state) ctx->save_for_backward({*state});          // numbers written into it before the backward pass are noticed
        return drop_forward(x.contiguous(), dense(residual), dense(state), {(int)dtype, rows, cols, (int)n_z, p, (uint64_t)seed, (uint64_t)elem_offset, (int)draw});
    }
    static torch::autograd::tensor_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::tensor_list grads) {
        check_backward("dropout", grads);
        const auto c = ctx->saved_data["call"].toIntVector();
        const auto saved = ctx->get_saved_variables();
        torch::autograd::tensor_list out(11);
        if (ctx->needs_input_grad(0)) {
            const Tensor g = grads[0].contiguous();
            c10::DeviceGuard guard(g.device());
            out[0] = at::empty(ctx->saved_data["shape"].toIntVector(), g.options());
            check(lib.dropout_backward(ptr(g), ptr(out[0]), (int)c[0], c[1], c[2], (int)c[3], ctx->saved_data["p"].toDouble(), (uint64_t)c[4], (uint64_t)c[5],
                                       saved.empty() ? nullptr : (const uint64_t*)ptr(saved[0]), (int)c[6], stream_of(g)), "card_dropout_backward");
        }
        if (c[7] && ctx->needs_input_grad(1)) out[1] = grads[0];          // inputs that are not given have no number
        return out;
    }
};
Tensor dropout(const Tensor& x, double p, uint64_t seed, const OptTensor& state_, int64_t elem_offset, int64_t draw, int64_t n_z, const OptTensor& residual) {
    on_gpu(x);
    check_mode("dropout", x, residual);
    const int dtype = dtype_of(x, "dropout");
    if (x.dim() < 1) refuse("dropout: x is a scalar; expected (..., cols)");
    if (n_z < 1 || n_z > INT32_MAX || draw < 0 || draw > INT32_MAX || elem_offset < 0)
        refuse("dropout: n_z=", n_z, ", draw=", draw, " or elem_offset=", elem_offset, " out of range");
    if (state_) {
        const Tensor& state = *state_;
        if (state.scalar_type() != at::kLong || state.numel() != 2 || state.device() != x.device() || !state.is_contiguous())
            refuse("dropout: a seed tensor holds two int64 numbers on ", x.device().str(), ", got ", state.sizes(), " ", state.scalar_type(), " on ", state.device().str());
    }
    const int64_t cols = x.size(-1);
    if (residual) {
        auto shape = x.sizes().vec();
        if (n_z > 1) shape.insert(shape.end() - 1, n_z);
        same(*residual, x, shape, "dropout: residual");
    }
    const int64_t rows = cols ? x.numel() / cols : 0;
    if (at::GradMode::is_enabled() && (x.requires_grad() || (residual && residual->requires_grad())))
        return Dropout::apply(x, residual, state_, (int64_t)dtype, rows, cols, n_z, p, (int64_t)seed, elem_offset, draw);
    return drop_forward(x.contiguous(), dense(residual), dense(state_), {dtype, rows, cols, (int)n_z, p, seed, (uint64_t)elem_offset, (int)draw});
}

// ------------------------------------------------------------------------------------------------ norm
struct Normed {
    Tensor y, scale, h;
};
Normed norm_forward(const Tensor& x, const Tensor& residual, const Tensor& weight, double eps, bool e4m3) {
    c10::DeviceGuard guard(x.device());
    const int64_t cols = x.size(-1), rows = x.numel() / cols;
    const int dt = dtype_of(x, "rms_norm"), wt = weight.defined() ? dtype_of(weight, "rms_norm: weight") : dt;
    Normed n;
    if (residual.defined()) n.h = at::empty_like(x, at::MemoryFormat::Contiguous);
    if (e4m3) {
        n.y = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
        n.scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
    } else {
        n.y = at::empty_like(x, at::MemoryFormat::Contiguous);
    }
    check(lib.rms_norm(ptr(x), ptr(residual), ptr(weight), dt, wt, rows, cols, eps, ptr(n.h), ptr(n.y), e4m3 ? (int)CARD_DTYPE_E4M3 : dt,
                       (float*)ptr(n.scale), stream_of(x)), "card_rms_norm");
    return n;
}
struct RmsNorm : torch::autograd::Function<RmsNorm> {
    static torch::autograd::tensor_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& residual, const OptTensor& weight, double eps) {
        const Tensor xc = x.contiguous(), wc = dense(weight);          // the caller's tensors come in, as in Dropout
        const Normed n = norm_forward(xc, dense(residual), wc, eps, false);
        ctx->save_for_backward({n.h.defined() ? n.h : xc, wc});
        ctx->saved_data["eps"] = eps;
        ctx->set_materialize_grads(false);
        return n.h.defined() ? torch::autograd::tensor_list{n.y, n.h} : torch::autograd::tensor_list{n.y};
    }
    static torch::autograd::tensor_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::tensor_list grads) {
        check_backward("rms_norm", grads);
        const auto saved = ctx->get_saved_variables();
        const Tensor h = saved[0], weight = saved[1];
        const Tensor g = grads[0].defined() ? grads[0].contiguous() : Tensor();
        const Tensor gh = grads.size() > 1 && grads[1].defined() ? grads[1].contiguous() : Tensor();
        c10::DeviceGuard guard(h.device());
        const int64_t cols = h.size(-1), rows = h.numel() / cols;
        const int dt = dtype_of(h, "rms_norm"), wt = weight.defined() ? dtype_of(weight, "rms_norm: weight") : dt;
        const bool residual = grads.size() > 1;               // inputs that are not given have no number
        Tensor dx = at::empty_like(h), dw, ws;
        uint64_t bytes = 0;
        if (weight.defined() && ctx->needs_input_grad(residual ? 2 : 1)) {
            dw = at::empty_like(weight);
            check(lib.rms_norm_backward_workspace_bytes(dt, rows, cols, &bytes), "card_rms_norm_backward_workspace_bytes");
            ws = at::empty({(int64_t)bytes}, h.options().dtype(at::kByte));
        }
        check(lib.rms_norm_backward(ptr(h), ptr(weight), ptr(g), ptr(gh), dt, wt, rows, cols, ctx->saved_data["eps"].toDouble(), ptr(dx), ptr(dw), ptr(ws), bytes,
                                    stream_of(h)), "card_rms_norm_backward");
        return {ctx->needs_input_grad(0) ? dx : Tensor(), residual && ctx->needs_input_grad(1) ? dx : Tensor(), dw, Tensor()};
    }
};
// checks the arguments; whether a gradient is asked for
bool norm_args(const char* what, const Tensor& x, const OptTensor& weight_, const OptTensor& residual) {
    on_gpu(x);
    check_mode(what, x, weight_, residual);
    dtype_of(x, what);
    if (x.dim() < 1 || x.size(-1) < 1) refuse(what, ": x has shape ", x.sizes(), "; expected (..., cols) with cols >= 1");
    if (weight_) {
        const Tensor& weight = *weight_;
        if (weight.dim() != 1 || weight.size(0) != x.size(-1) || (weight.scalar_type() != at::kFloat && weight.scalar_type() != x.scalar_type()) ||
            weight.device() != x.device())
            refuse(what, ": weight: expected (", x.size(-1), ",) ", x.scalar_type(), " or float32 on ", x.device().str(), ", got ", weight.sizes(), " ",
                   weight.scalar_type(), " on ", weight.device().str());
    }
    if (residual) same(*residual, x, x.sizes(), c10::str(what, ": residual").c_str());
    return at::GradMode::is_enabled() && (x.requires_grad() || (weight_ && weight_->requires_grad()) || (residual && residual->requires_grad()));
}
std::vector<Tensor> rms_norm(const Tensor& x, const OptTensor& weight, const OptTensor& residual, double eps) {
    if (norm_args("rms_norm", x, weight, residual)) return RmsNorm::apply(x, residual, weight, eps);
    const Normed n = norm_forward(x.contiguous(), dense(residual), dense(weight), eps, false);
    return n.h.defined() ? std::vector<Tensor>{n.y, n.h} : std::vector<Tensor>{n.y};
}
std::vector<Tensor> rms_norm_e4m3(const Tensor& x, const OptTensor& weight, const OptTensor& residual, double eps) {
    if (norm_args("rms_norm_e4m3", x, weight, residual)) refuse("rms_norm_e4m3 has no backward pass; use rms_norm, or torch.no_grad()");
    const Normed n = norm_forward(x.contiguous(), dense(residual), dense(weight), eps, true);
    return n.h.defined() ? std::vector<Tensor>{n.y, n.scale, n.h} : std::vector<Tensor>{n.y, n.scale};
}

// ------------------------------------------------------------------------------------------------ 4-bit weights
Tensor linear4(uintptr_t handle, int64_t device, int64_t in, int64_t out, const Tensor& x, const OptTensor& x_scale_, const OptTensor& gamma_, double slope,
               const std::optional<at::ScalarType>& out_dtype) {
    on_gpu(x);
    check_mode("QuantLinear", x, x_scale_, gamma_);
    const at::Device dev = x.device();
    if (dev.index() != device) refuse("QuantLinear: x is on ", dev.str(), ", the weights are on cuda:", device);
    if (x.dim() < 1 || x.size(-1) != in) refuse("QuantLinear: x has shape ", x.sizes(), "; expected (..., ", in, ")");
    Tensor x_scale = x_scale_ ? *x_scale_ : Tensor(), gamma = gamma_ ? *gamma_ : Tensor();
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(x_scale) || wants_grad(gamma)))
        refuse("QuantLinear has no backward pass; call it under torch.no_grad() or detach its input");
    const bool e4m3 = x.scalar_type() == at::kFloat8_e4m3fn;
    const int xt = e4m3 ? (int)CARD_DTYPE_E4M3 : dtype_of(x, "QuantLinear");
    if (e4m3) {
        const auto lead = x.sizes().slice(0, x.dim() - 1);
        if (!x_scale.defined() || x_scale.sizes() != lead || x_scale.scalar_type() != at::kFloat || x_scale.device() != dev)
            refuse("QuantLinear: 8-bit rows come with x_scale ", lead, " float32 on ", dev.str());
        x_scale = x_scale.contiguous();
    } else if (x_scale.defined()) {
        refuse("QuantLinear: x_scale goes with float8_e4m3fn rows");
    }
    const at::ScalarType ot = out_dtype ? *out_dtype : e4m3 ? at::kBFloat16 : x.scalar_type();
    if (ot != at::kFloat && ot != at::kBFloat16 && ot != at::kHalf) refuse("QuantLinear: out_dtype ", ot, " is none of float32, bfloat16, float16");
    if (gamma.defined()) {
        if (gamma.dim() != 1 || gamma.size(0) != out || gamma.scalar_type() != at::kFloat || gamma.device() != dev)
            refuse("QuantLinear: gamma is (", out, ",) float32 on ", dev.str(), ", got ", gamma.sizes(), " ", gamma.scalar_type(), " on ", gamma.device().str());
        gamma = gamma.contiguous();
    }
    c10::DeviceGuard guard(dev);
    const Tensor xc = x.contiguous();
    auto shape = x.sizes().vec();
    shape.back() = out;
    Tensor y = at::empty(shape, x.options().dtype(ot));
    uint64_t bytes = 0;
    check(lib.linear4_workspace_bytes((const card_linear4*)handle, xt, xc.numel() / in, &bytes), "card_linear4_forward");
    const Tensor ws = bytes ? at::empty({(int64_t)bytes}, x.options().dtype(at::kByte)) : Tensor();
    check(lib.linear4_forward((const card_linear4*)handle, ptr(xc), xt, (const float*)ptr(x_scale), xc.numel() / in, (const float*)ptr(gamma), (float)slope, ptr(y),
                              ot == at::kFloat ? CARD_DTYPE_F32 : ot == at::kBFloat16 ? CARD_DTYPE_BF16 : CARD_DTYPE_F16, ptr(ws), bytes, stream_of(x)), "card_linear4_forward");
    return y;
}

void init(py::dict address, py::object error) {
#define CARD_TAKE(name) lib.name = reinterpret_cast<decltype(lib.name)>(address["card_" #name].cast<uintptr_t>())
    CARD_TAKE(last_error); CARD_TAKE(dropout); CARD_TAKE(dropout_backward); CARD_TAKE(rms_norm); CARD_TAKE(rms_norm_backward);
    CARD_TAKE(rms_norm_backward_workspace_bytes); CARD_TAKE(linear4_forward); CARD_TAKE(linear4_workspace_bytes);
#undef CARD_TAKE
    card_error = error.inc_ref().ptr();
}

}  // namespace

PYBIND11_MODULE(_card_torch, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const CardErr& e) {
            PyErr_SetString(card_error, e.what());
        }
    });
    const auto free = py::call_guard<py::gil_scoped_release>();
    m.def("init", &init);
    m.def("dropout", &dropout, free);
    m.def("rms_norm", &rms_norm, free);
    m.def("rms_norm_e4m3", &rms_norm_e4m3, free);
    m.def("linear4", &linear4, free);
}
