// The autograd nodes of the norm and dropout operators, in C++ (module transformer_vae_amd._host).
//
// What it saves is host time: at a few hundred rows the kernels take some microseconds, and a Python autograd.Function's
// backward pass has to take the interpreter lock in the autograd thread (layer norm of 40 x 512, forward and backward: 158 us
// of host time with Python nodes over ctypes).  The kernels are reached through the same C interface (include/tvae_hip.h).
//
// The operators are registered with torch's dispatcher (torch.ops.tvae): what records a program by its operators -- torch.jit.trace,
// make_fx, fake tensors -- sees one operator where a kernel launched beside the dispatcher would leave nothing but the
// allocation of its output.  Their kernels check everything they are given, since a recorded graph calls them directly.
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/library.h>

#include <dlfcn.h>

#include <array>
#include <cstdint>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "../../include/tvae_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;
using MaybeType = std::optional<at::ScalarType>;

// The library's entry points, of the one that the package has loaded: this module is not linked to it, so that there is one copy,
// whichever build of it that is.
struct Library {
    decltype(&tvae_last_error) last_error = nullptr;
    decltype(&tvae_dropout) dropout = nullptr;
    decltype(&tvae_norm_fwd) norm_fwd = nullptr;
    decltype(&tvae_norm_bwd) norm_bwd = nullptr;
    decltype(&tvae_norm_bwd_workspace_bytes) norm_bwd_workspace_bytes = nullptr;
} bound;
void bind(uintptr_t handle) {
    const auto find = [&](auto& entry, const char* name) {
        void* const at = dlsym(reinterpret_cast<void*>(handle), name);
        TORCH_CHECK(at, "the library has no ", name, ": it was not built from these sources");
        entry = reinterpret_cast<std::decay_t<decltype(entry)>>(at);
    };
    Library l;
    find(l.last_error, "tvae_last_error");
    find(l.dropout, "tvae_dropout");
    find(l.norm_fwd, "tvae_norm_fwd");
    find(l.norm_bwd, "tvae_norm_bwd");
    find(l.norm_bwd_workspace_bytes, "tvae_norm_bwd_workspace_bytes");
    bound = l;
}
const Library& library() {
    TORCH_CHECK(bound.dropout, "the operators' library has not been loaded (transformer_vae_amd loads it with the first call)");
    return bound;
}

void check(int status, const char* what) {
    TORCH_CHECK(status == 0, what, " failed (status ", status, "): ", library().last_error());
}

int code_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return TVAE_F32;
        case at::kBFloat16: return TVAE_BF16;
        case at::kHalf: return TVAE_F16;
        default: return -1;
    }
}

std::string name_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return "torch.float32";
        case at::kBFloat16: return "torch.bfloat16";
        case at::kHalf: return "torch.float16";
        case at::kDouble: return "torch.float64";
        case at::kInt: return "torch.int32";
        case at::kLong: return "torch.int64";
        default: return at::toString(t);
    }
}

const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out_ptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

const int64_t* rng_ptr(const MaybeTensor& rng) { return rng ? rng->const_data_ptr<int64_t>() : nullptr; }

// Row layout of tensors of one shape (..., d): element (i, c) of a tensor lies at (i / grp) * so + (i % grp) * si + c.  Dense tensors,
// 2-d ones and 3-d ones of any row strides are read where they lie (the first n tokens of longer sequences, an expanded
// batch); anything else is made dense first.
struct Row { Tensor t; int64_t so = 0, si = 0; };
struct Rows {
    std::vector<Row> r;
    int64_t grp = 1, rows = 1, d = 0;
    Rows(at::IntArrayRef shape, std::initializer_list<Tensor> tensors) {
        const size_t dims = shape.size();
        d = shape.back();
        for (size_t i = 0; i + 1 < dims; ++i) rows *= shape[i];
        bool dense = true;
        for (const Tensor& t : tensors) {
            Row row{t};
            if (t.defined() && !t.is_contiguous()) {
                if ((dims == 2 || dims == 3) && t.stride(-1) == 1) dense = false;
                else row.t = t.contiguous();
            }
            r.push_back(std::move(row));
        }
        if (!dense && dims == 3) grp = shape[1];
        for (Row& row : r) {
            if (!row.t.defined()) continue;
            row.so = dense ? d : row.t.stride(0);
            row.si = dense || dims != 3 ? 0 : row.t.stride(1);
        }
    }
};

void check_device(const char* what, const Tensor& x) {
    TORCH_CHECK(x.is_cuda(), what, ": tensor is on ", x.device(), "; the bottleneck kernels run on MI355X only (there is no CPU fallback)");
}
// The checks of the operators' arguments, beside the making of their outputs: in the kernels, and where shapes alone are made.
void check_rows(const char* what, const Tensor& x) {
    TORCH_CHECK_VALUE(x.dim() >= 1, what, " works on rows of the last axis, got a tensor without axes");
    TORCH_CHECK_TYPE(code_of(x.scalar_type()) >= 0, what, " takes float32, bfloat16 or float16, got ", name_of(x.scalar_type()));
}
void check_beside(const char* what, const char* name, const Tensor& x, const Tensor& t, bool row_shape) {
    if (!t.defined()) return;
    const auto want = row_shape ? x.sizes() : x.sizes().slice(x.dim() - 1);
    TORCH_CHECK_VALUE(t.sizes() == want, what, ": ", name, " must be ", want, ", got ", t.sizes());
    TORCH_CHECK_VALUE(t.device() == x.device(), what, ": ", name, " is on ", t.device(), ", x on ", x.device());
    TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat, what, ": ", name, " must be ",
                     name_of(x.scalar_type()), " or torch.float32, got ", name_of(t.scalar_type()));
}
void check_probability(const char* what, double p) {
    TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, what, ": p must be between 0 and 1, got ", p);
}
void check_dropout(const char* what, const Tensor& x, double p, const MaybeTensor& rng) {
    check_probability(what, p);
    if (!rng) return;
    TORCH_CHECK_VALUE(rng->scalar_type() == at::kLong && rng->dim() == 1 && rng->size(0) == 2 && rng->is_contiguous() && rng->device() == x.device(),
                      what, ": rng must be two contiguous int64 on ", x.device(), " (seed, offset), got ", rng->sizes(), " ",
                      name_of(rng->scalar_type()), " on ", rng->device());
}

// a dropout call's randomness: a device tensor {seed, offset}, or the two words themselves; drawn where dropout is on and none is given
struct Rng {
    MaybeTensor state;
    int64_t seed = 0, offset = 0;
};
Rng rng_of(const char* what, const Tensor& x, double p, const pybind11::object& rng) {
    check_probability(what, p);
    Rng r;
    if (p == 0.0) return r;
    if (rng.is_none()) {
        r.state = at::empty({2}, x.options().dtype(at::kLong)).random_();
    } else if (THPVariable_Check(rng.ptr())) {
        r.state = THPVariable_Unpack(rng.ptr()).detach();
    } else {
        const bool sequence = PySequence_Check(rng.ptr()) && !PyUnicode_Check(rng.ptr()) && !PyBytes_Check(rng.ptr());
        TORCH_CHECK_TYPE(sequence, what, ": rng must be a tensor or two ints (seed, offset), got ", Py_TYPE(rng.ptr())->tp_name);
        const auto words = pybind11::reinterpret_borrow<pybind11::sequence>(rng);
        TORCH_CHECK_VALUE(words.size() == 2, what, ": rng must be a tensor or two ints (seed, offset), got ", words.size(), " of them");
        const auto word = [&](const pybind11::object& o) {
            const auto index = pybind11::reinterpret_steal<pybind11::object>(PyNumber_Index(o.ptr()));
            if (!index) PyErr_Clear();
            TORCH_CHECK_TYPE(index, what, ": rng must be a tensor or two ints (seed, offset), got a ", Py_TYPE(o.ptr())->tp_name);
            const uint64_t v = PyLong_AsUnsignedLongLongMask(index.ptr());
            if (PyErr_Occurred()) throw pybind11::error_already_set();
            return (int64_t)v;
        };
        r.seed = word(words[0]);
        r.offset = word(words[1]);
    }
    return r;
}

// gradients that must not be differentiated again: an error node in their place where a graph of the backward pass is made
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)grads.size());
    variable_list marked;
    for (Tensor& g : grads) marked.push_back(g.defined() ? g.detach().requires_grad_(true) : g);
    return (*error)(std::move(marked));
}

// A gradient that is captured into a graph must not go to a node on the default stream, which may not join a capture.  The engine would
// have it wait there nonetheless and end the process.  A leaf's accumulation node belongs to the stream of the oldest graph
// of it that still lives: an eager one, kept alive by a loss, puts it on the default stream.
void refuse_default_stream(const char* what) {
    const auto node = torch::autograd::get_current_node();
    for (const torch::autograd::Edge& edge : node->next_edges()) {
        if (!edge.function) continue;
        const auto stream = edge.function->stream();
        if (!stream || *stream != c10::Stream(c10::Stream::DEFAULT, stream->device())) continue;
        const auto current = c10::hip::getCurrentHIPStream(stream->device_index());
        if (current.id() == stream->id()) continue;
        hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
        if (hipStreamIsCapturing(current.stream(), &capture) != hipSuccess) (void)hipGetLastError();
        TORCH_CHECK(capture == hipStreamCaptureStatusNone, what, ": the captured backward pass leads to ", edge.function->name(),
                    " on the default stream, which cannot be captured; release the eager results (a loss, an output) that keep "
                    "a graph of the same leaves alive, then capture again");
    }
}

// A node's inputs that may be missing go as optionals; the gradient edges are numbered over those that are there.
MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : std::nullopt; }
Tensor tensor_of(const MaybeTensor& t) { return t ? *t : Tensor(); }
bool wants_gradient(const MaybeTensor& t) { return t && t->requires_grad(); }
// there is no forward-mode derivative: an input that carries a tangent is refused, whether it requires a gradient or not
void refuse_tangents(const char* what, std::initializer_list<const MaybeTensor*> inputs) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const MaybeTensor* t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!*t || !(*t)->_fw_grad(0).defined(), what, ": forward-mode derivatives are not implemented");
}
template <typename Signature>
auto operator_handle(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}

// ---- dropout ---------------------------------------------------------------------------------------------------------------
Tensor dropout_out(const Tensor& x, const MaybeTensor& residual, double p, const MaybeTensor& rng, int64_t, int64_t, MaybeType type) {
    const char* what = residual ? "dropout_add" : "dropout";
    check_rows(what, x);
    check_beside(what, "residual", x, tensor_of(residual), true);
    check_dropout(what, x, p, rng);
    return at::empty(x.sizes(), x.options().dtype(residual ? residual->scalar_type() : type.value_or(x.scalar_type())));
}
Tensor dropout_cuda(const Tensor& x, const MaybeTensor& residual_, double p, const MaybeTensor& rng, int64_t seed, int64_t offset, MaybeType type) {
    const Tensor residual = tensor_of(residual_);
    check_device("dropout", x);
    const c10::DeviceGuard guard(x.device());
    const Tensor out = dropout_out(x, residual_, p, rng, seed, offset, type);
    const Rows l(x.sizes(), {x, residual});
    if (l.rows * l.d > 0)
        check(library().dropout(ptr(l.r[0].t), l.r[0].so, l.r[0].si, ptr(l.r[1].t), l.r[1].so, l.r[1].si, l.grp, out_ptr(out), l.rows, l.d, p,
                           rng_ptr(rng), (uint64_t)seed, (uint64_t)offset, code_of(x.scalar_type()), code_of(out.scalar_type()),
                           stream_of(x)), "tvae_dropout");
    return out;
}
const auto& dropout_op() {
    static const auto op = operator_handle<decltype(dropout_out)>("tvae::dropout");
    return op;
}

struct DropoutNode : torch::autograd::Function<DropoutNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& residual, double p, const MaybeTensor& rng, int64_t seed,
                          int64_t offset, MaybeType type) {
        ctx->saved_data["add"] = residual.has_value();
        ctx->save_for_backward({tensor_of(rng)});
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        ctx->saved_data["type"] = (int64_t)x.scalar_type();
        const at::AutoDispatchBelowADInplaceOrView below;
        return dropout_op().call(x, residual, p, rng, seed, offset, type);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        refuse_default_stream("dropout");
        const MaybeTensor rng = maybe(ctx->get_saved_variables()[0]);       // may run a checkpointed forward pass again: with autograd
        Tensor dx;
        if (ctx->needs_input_grad(0)) {
            const at::AutoDispatchBelowADInplaceOrView below;
            dx = dropout_op().call(grads[0], std::nullopt, ctx->saved_data["p"].toDouble(), rng, ctx->saved_data["seed"].toInt(),
                                   ctx->saved_data["offset"].toInt(), (at::ScalarType)ctx->saved_data["type"].toInt());
        }
        return once({dx, ctx->saved_data["add"].toBool() && ctx->needs_input_grad(1) ? grads[0] : Tensor(), {}, {}, {}, {}, {}});
    }
};

Tensor dropout_autograd(const Tensor& x, const MaybeTensor& residual, double p, const MaybeTensor& rng, int64_t seed, int64_t offset, MaybeType type) {
    const MaybeTensor input(x);
    refuse_tangents("dropout", {&input, &residual});
    if (at::GradMode::is_enabled() && (x.requires_grad() || wants_gradient(residual)))
        return DropoutNode::apply(x, residual, p, rng, seed, offset, type);
    const at::AutoDispatchBelowADInplaceOrView below;
    return dropout_op().call(x, residual, p, rng, seed, offset, type);
}

Tensor dropout(const Tensor& x, const MaybeTensor& residual, double p, const pybind11::object& rng_) {
    const char* what = residual ? "dropout_add" : "dropout";
    check_device(what, x);
    const Rng rng = rng_of(what, x, p, rng_);
    const pybind11::gil_scoped_release release;
    return dropout_op().call(x, residual, p, rng.state, rng.seed, rng.offset, std::nullopt);
}

// ---- norms -----------------------------------------------------------------------------------------------------------------

// {y}, then v where the sum is asked for, then rstd and (layer norm) the mean where the statistics are
std::vector<Tensor> norm_out(const Tensor& x, const MaybeTensor& residual, const MaybeTensor& weight, const MaybeTensor& bias, int64_t kind, double eps,
                             double p, const MaybeTensor& rng, int64_t, int64_t, bool return_sum, bool stats) {
    const char* names[2][2] = {{"layer_norm", "rms_norm"}, {"dropout_add_layer_norm", "dropout_add_rms_norm"}};
    const char* what = names[residual || p != 0.0 || return_sum][kind == TVAE_NORM_RMS];
    check_rows(what, x);
    check_beside(what, "residual", x, tensor_of(residual), true);
    check_beside(what, "weight", x, tensor_of(weight), false);
    check_beside(what, "bias", x, tensor_of(bias), false);
    TORCH_CHECK_VALUE(x.size(-1) > 0, what, ": the last axis is empty");
    if (weight && bias)
        TORCH_CHECK_TYPE(weight->scalar_type() == bias->scalar_type(), what,
                         ": weight and bias are of one type, got ", name_of(weight->scalar_type()), " and ", name_of(bias->scalar_type()));
    TORCH_CHECK_VALUE(eps >= 0.0 && eps < 1e30, what, ": eps must be a finite number >= 0, got ", eps);
    check_dropout(what, x, p, rng);
    std::vector<Tensor> out{at::empty(x.sizes(), x.options())};
    if (return_sum) out.push_back(at::empty(x.sizes(), x.options().dtype(residual ? residual->scalar_type() : x.scalar_type())));
    if (stats) {
        for (int i = 0; i < (kind == TVAE_NORM_RMS ? 1 : 2); ++i)
            out.push_back(at::empty({x.numel() / x.size(-1)}, x.options().dtype(at::kFloat)));
    }
    return out;
}
std::vector<Tensor> norm_cuda(const Tensor& x, const MaybeTensor& residual_, const MaybeTensor& weight_, const MaybeTensor& bias_, int64_t kind,
                              double eps, double p, const MaybeTensor& rng, int64_t seed, int64_t offset, bool return_sum, bool stats) {
    check_device("norm", x);
    const c10::DeviceGuard guard(x.device());
    const std::vector<Tensor> out = norm_out(x, residual_, weight_, bias_, kind, eps, p, rng, seed, offset, return_sum, stats);
    const Tensor residual = tensor_of(residual_);
    const Rows l(x.sizes(), {x, residual});
    const at::ScalarType r_type = residual.defined() ? residual.scalar_type() : x.scalar_type();
    const Tensor weight = weight_ ? weight_->contiguous() : Tensor(), bias = bias_ ? bias_->contiguous() : Tensor();
    const at::ScalarType w_type = weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : x.scalar_type();
    const size_t at_rstd = return_sum ? 2 : 1;
    if (l.rows > 0)
        check(library().norm_fwd((int)kind, ptr(l.r[0].t), l.r[0].so, l.r[0].si, ptr(l.r[1].t), l.r[1].so, l.r[1].si, l.grp, ptr(weight), ptr(bias), eps,
                            p, rng_ptr(rng), (uint64_t)seed, (uint64_t)offset, out_ptr(out[0]), return_sum ? out_ptr(out[1]) : nullptr,
                            stats && kind != TVAE_NORM_RMS ? (float*)out_ptr(out[at_rstd + 1]) : nullptr,
                            stats ? (float*)out_ptr(out[at_rstd]) : nullptr, l.rows, l.d, code_of(x.scalar_type()), code_of(w_type),
                            code_of(r_type), stream_of(x)), "tvae_norm_fwd");
    return out;
}
const auto& norm_op() {
    static const auto op = operator_handle<decltype(norm_out)>("tvae::norm");
    return op;
}

// those of dx, dresidual, dweight and dbias that are needed
std::vector<Tensor> norm_backward_out(const Tensor& dy, const MaybeTensor& dsum, const MaybeTensor& x, const MaybeTensor& residual,
                                      const MaybeTensor& weight, const MaybeTensor& mean, const Tensor& rstd, int64_t, double p,
                                      const MaybeTensor& rng, int64_t, int64_t, at::ScalarType w_type, std::array<bool, 4> need) {
    const char* what = "norm_backward";
    check_rows(what, dy);
    TORCH_CHECK_VALUE(dy.size(-1) > 0, what, ": the last axis is empty");
    const at::ScalarType r_type = residual ? residual->scalar_type() : dy.scalar_type();
    check_beside(what, "x", dy, tensor_of(x), true);
    check_beside(what, "residual", dy, tensor_of(residual), true);
    check_beside(what, "dsum", dy, tensor_of(dsum), true);
    check_beside(what, "weight", dy, tensor_of(weight), false);
    TORCH_CHECK_TYPE((!x || x->scalar_type() == dy.scalar_type()) && (!dsum || dsum->scalar_type() == r_type) && code_of(w_type) >= 0 &&
                     (!weight || weight->scalar_type() == w_type), what, ": the types are not those of a forward call");
    const int64_t rows = dy.numel() / dy.size(-1);
    for (const MaybeTensor& t : {mean, MaybeTensor(rstd)})
        TORCH_CHECK_VALUE(!t || (t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == rows && t->is_contiguous() && t->device() == dy.device()),
                          what, ": mean and rstd are ", rows, " contiguous float32 on ", dy.device());
    check_dropout(what, dy, p, rng);
    const at::ScalarType types[4] = {dy.scalar_type(), r_type, w_type, w_type};
    std::vector<Tensor> out;
    for (int i = 0; i < 4; ++i) {
        if (!need[i]) continue;
        const auto options = dy.options().dtype(types[i]);
        out.push_back(i < 2 ? at::empty(dy.sizes(), options) : at::empty({dy.size(-1)}, options));
    }
    return out;
}
std::vector<Tensor> norm_backward_cuda(const Tensor& dy, const MaybeTensor& dsum, const MaybeTensor& x, const MaybeTensor& residual,
                                       const MaybeTensor& weight_, const MaybeTensor& mean, const Tensor& rstd, int64_t kind, double p,
                                       const MaybeTensor& rng, int64_t seed, int64_t offset, at::ScalarType w_type, std::array<bool, 4> need) {
    check_device("norm_backward", dy);
    const c10::DeviceGuard guard(dy.device());
    const std::vector<Tensor> out = norm_backward_out(dy, dsum, x, residual, weight_, mean, rstd, kind, p, rng, seed, offset, w_type, need);
    Tensor grads[4];
    for (int i = 0, k = 0; i < 4; ++i)
        if (need[i]) grads[i] = out[k++];
    const Rows l(dy.sizes(), {dy, tensor_of(dsum), tensor_of(x), tensor_of(residual)});
    if (l.rows == 0) {
        for (int i = 2; i < 4; ++i)
            if (need[i]) grads[i].zero_();
        return out;
    }
    Tensor ws;
    const int64_t bytes = need[2] || need[3] ? library().norm_bwd_workspace_bytes(l.rows, l.d) : 0;
    if (bytes > 0) ws = at::empty({bytes}, dy.options().dtype(at::kByte));
    const Tensor weight = weight_ ? weight_->contiguous() : Tensor();
    const at::ScalarType r_type = residual ? residual->scalar_type() : dy.scalar_type();
    check(library().norm_bwd((int)kind, ptr(l.r[0].t), l.r[0].so, l.r[0].si, ptr(l.r[1].t), l.r[1].so, l.r[1].si, ptr(l.r[2].t), l.r[2].so, l.r[2].si,
                        ptr(l.r[3].t), l.r[3].so, l.r[3].si, l.grp, ptr(weight), mean ? (const float*)ptr(*mean) : nullptr,
                        (const float*)ptr(rstd), p, rng_ptr(rng), (uint64_t)seed, (uint64_t)offset, out_ptr(grads[0]), out_ptr(grads[1]),
                        out_ptr(grads[2]), out_ptr(grads[3]), l.rows, l.d, code_of(dy.scalar_type()), code_of(w_type), code_of(r_type),
                        out_ptr(ws), bytes, stream_of(dy)), "tvae_norm_bwd");
    return out;
}
const auto& norm_backward_op() {
    static const auto op = operator_handle<decltype(norm_backward_out)>("tvae::norm_backward");
    return op;
}

// {norm(v), v or nothing} with v = [residual +] dropout(x): one node for the sum, the dropout and the norm.  The statistics come out
// too where a recorded program asks for them, which holds the calls below autograd; they have no derivative.
struct NormNode : torch::autograd::Function<NormNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& residual, const MaybeTensor& weight,
                                 const MaybeTensor& bias, int64_t kind, double eps, double p, const MaybeTensor& rng, int64_t seed,
                                 int64_t offset, bool return_sum, bool stats) {
        ctx->set_materialize_grads(false);
        variable_list out;
        {
            const at::AutoDispatchBelowADInplaceOrView below;
            out = norm_op().call(x, residual, weight, bias, kind, eps, p, rng, seed, offset, return_sum, true);
        }
        const Tensor mean = kind == TVAE_NORM_RMS ? Tensor() : out.back(), rstd = out[return_sum ? 2 : 1];
        if (stats) ctx->mark_non_differentiable(variable_list(out.begin() + (return_sum ? 2 : 1), out.end()));
        else out.resize(return_sum ? 2 : 1);
        // The backward pass needs v in fp32: it forms it again from x and the residual, or reads the returned sum where that holds
        // v as it is (fp32: 4 bytes an element for the 4 + 2 or 4 + 4 of x and residual).  A 16-bit sum would put its rounding
        // into the weights' gradient.
        const bool kept = return_sum && out[1].scalar_type() == at::kFloat;
        ctx->save_for_backward({kept ? Tensor() : x, kept ? out[1] : tensor_of(residual), tensor_of(weight), mean, rstd, tensor_of(rng)});
        const auto type = [](const MaybeTensor& t) { return t ? (int64_t)t->scalar_type() : (int64_t)-1; };
        ctx->saved_data["meta"] = std::vector<int64_t>{type(x), type(residual), type(weight), type(bias), kind, seed, offset, return_sum};
        ctx->saved_data["p"] = p;
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        refuse_default_stream("norm");
        const auto saved = ctx->get_saved_variables();
        const auto meta = ctx->saved_data["meta"].toIntVector();
        const double p = ctx->saved_data["p"].toDouble();
        const at::ScalarType x_type = (at::ScalarType)meta[0], r_type = meta[1] < 0 ? x_type : (at::ScalarType)meta[1];
        const at::ScalarType w_type = meta[2] >= 0 ? (at::ScalarType)meta[2] : meta[3] >= 0 ? (at::ScalarType)meta[3] : x_type;
        const MaybeTensor rng = maybe(saved[5]);
        size_t edge = 0;
        std::array<bool, 4> need;
        for (int i = 0; i < 4; ++i) need[i] = meta[i] >= 0 && ctx->needs_input_grad(edge++);
        const Tensor dy = grads[0], ds = meta[7] ? grads[1] : Tensor();
        Tensor out[4];
        {
            const at::AutoDispatchBelowADInplaceOrView below;
            if (!dy.defined()) {                // only the sum was used: the norm has no part in the gradient
                if (ds.defined()) {
                    if (need[0]) out[0] = dropout_op().call(ds, std::nullopt, p, rng, meta[5], meta[6], x_type);
                    if (need[1]) out[1] = ds;
                }
            } else {
                // without dropout x and a residual of its type have one gradient
                const bool shared = need[0] && need[1] && p == 0.0 && r_type == x_type;
                if (shared) need[1] = false;
                const auto got = norm_backward_op().call(dy, maybe(ds), maybe(saved[0]), maybe(saved[1]), maybe(saved[2]), maybe(saved[3]), saved[4],
                                                         meta[4], p, rng, meta[5], meta[6], w_type, need);
                for (int i = 0, k = 0; i < 4; ++i)
                    if (need[i]) out[i] = got[k++];
                if (shared) out[1] = out[0];
            }
        }
        return once({out[0], out[1], out[2], out[3], {}, {}, {}, {}, {}, {}, {}, {}});
    }
};

std::vector<Tensor> norm_autograd(const Tensor& x, const MaybeTensor& residual, const MaybeTensor& weight, const MaybeTensor& bias, int64_t kind,
                                  double eps, double p, const MaybeTensor& rng, int64_t seed, int64_t offset, bool return_sum, bool stats) {
    const MaybeTensor input(x);
    refuse_tangents("norm", {&input, &residual, &weight, &bias});
    if (at::GradMode::is_enabled() && (x.requires_grad() || wants_gradient(residual) || wants_gradient(weight) || wants_gradient(bias)))
        return NormNode::apply(x, residual, weight, bias, kind, eps, p, rng, seed, offset, return_sum, stats);
    const at::AutoDispatchBelowADInplaceOrView below;
    return norm_op().call(x, residual, weight, bias, kind, eps, p, rng, seed, offset, return_sum, stats);
}

// a recorded backward pass: not to be differentiated again
std::vector<Tensor> norm_backward_autograd(const Tensor& dy, const MaybeTensor& dsum, const MaybeTensor& x, const MaybeTensor& residual,
                                           const MaybeTensor& weight, const MaybeTensor& mean, const Tensor& rstd, int64_t kind, double p,
                                           const MaybeTensor& rng, int64_t seed, int64_t offset, at::ScalarType w_type, std::array<bool, 4> need) {
    const MaybeTensor first(dy);
    refuse_tangents("norm_backward", {&first, &dsum, &x, &residual, &weight});
    std::vector<Tensor> out;
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        out = norm_backward_op().call(dy, dsum, x, residual, weight, mean, rstd, kind, p, rng, seed, offset, w_type, need);
    }
    const bool wanted = dy.requires_grad() || wants_gradient(dsum) || wants_gradient(x) || wants_gradient(residual) || wants_gradient(weight);
    return wanted ? once(std::move(out)) : out;
}

pybind11::object norm(const char* what, int64_t kind, const Tensor& x, const MaybeTensor& residual, const MaybeTensor& weight,
                      const MaybeTensor& bias, double eps, double p, const pybind11::object& rng_, bool return_sum) {
    check_device(what, x);
    const Rng rng = rng_of(what, x, p, rng_);
    variable_list out;
    {
        const pybind11::gil_scoped_release release;
        out = norm_op().call(x, residual, weight, bias, kind, eps, p, rng.state, rng.seed, rng.offset, return_sum, false);
    }
    if (return_sum) return pybind11::make_tuple(out[0], out[1]);
    return pybind11::cast(out[0]);
}

}  // namespace

TORCH_LIBRARY(tvae, m) {
    m.def("dropout(Tensor x, Tensor? residual, float p, Tensor? rng, int seed, int offset, ScalarType? dtype=None) -> Tensor");
    m.def("norm(Tensor x, Tensor? residual, Tensor? weight, Tensor? bias, int kind, float eps, float p, Tensor? rng, int seed, int offset, "
          "bool return_sum, bool stats=False) -> Tensor[]");
    m.def("norm_backward(Tensor dy, Tensor? dsum, Tensor? x, Tensor? residual, Tensor? weight, Tensor? mean, Tensor rstd, int kind, float p, "
          "Tensor? rng, int seed, int offset, ScalarType w_dtype, bool[4] need) -> Tensor[]");
}
TORCH_LIBRARY_IMPL(tvae, CUDA, m) {
    m.impl("dropout", &dropout_cuda);
    m.impl("norm", &norm_cuda);
    m.impl("norm_backward", &norm_backward_cuda);
}
TORCH_LIBRARY_IMPL(tvae, Meta, m) {
    m.impl("dropout", &dropout_out);
    m.impl("norm", &norm_out);
    m.impl("norm_backward", &norm_backward_out);
}
TORCH_LIBRARY_IMPL(tvae, Autograd, m) {
    m.impl("dropout", &dropout_autograd);
    m.impl("norm", &norm_autograd);
    m.impl("norm_backward", &norm_backward_autograd);
}

PYBIND11_MODULE(_host, m) {
    m.doc() = "autograd nodes of the norm and dropout operators";
    m.def("norm", &norm);
    m.def("dropout", &dropout);
    m.def("bind", &bind);
}
