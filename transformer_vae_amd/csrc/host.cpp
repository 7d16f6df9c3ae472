// The autograd nodes of the norm and dropout operators, in C++ (module transformer_vae_amd._host).
//
// What it saves is host time: at a few hundred rows the kernels take some microseconds, and a Python autograd.Function's
// backward pass has to take the interpreter lock in the autograd thread (layer norm of 40 x 512, forward and backward: 158 us
// of host time with Python nodes over ctypes).  The kernels are reached through the same C interface (include/tvae_hip.h).
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

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

void check(int status, const char* what) {
    TORCH_CHECK(status == 0, what, " failed (status ", status, "): ", tvae_last_error());
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

// a dropout call's randomness: a device tensor {seed, offset}, or the two words themselves
struct Rng {
    Tensor state;
    uint64_t seed = 0, offset = 0;
    const int64_t* device() const { return state.defined() ? state.const_data_ptr<int64_t>() : nullptr; }
};

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

void check_rows(const char* what, const Tensor& x) {
    TORCH_CHECK(x.is_cuda(), what, ": tensor is on ", x.device(), "; the bottleneck kernels run on MI355X only (there is no CPU fallback)");
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
// p and the randomness as the launches take them; draws where dropout is on and no state is given
Rng check_dropout(const char* what, const Tensor& x, double p, const pybind11::object& rng) {
    TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, what, ": p must be between 0 and 1, got ", p);
    Rng r;
    if (p == 0.0) return r;
    if (rng.is_none()) {
        r.state = at::empty({2}, x.options().dtype(at::kLong)).random_();
    } else if (THPVariable_Check(rng.ptr())) {
        r.state = THPVariable_Unpack(rng.ptr()).detach();
        TORCH_CHECK_VALUE(r.state.scalar_type() == at::kLong && r.state.dim() == 1 && r.state.size(0) == 2 && r.state.is_contiguous() &&
                          r.state.device() == x.device(), what, ": rng must be two contiguous int64 on ", x.device(), " (seed, offset), got ",
                          r.state.sizes(), " ", name_of(r.state.scalar_type()), " on ", r.state.device());
    } else {
        const auto words = pybind11::cast<pybind11::tuple>(rng);
        TORCH_CHECK_VALUE(words.size() == 2, what, ": rng is a tensor or two ints (seed, offset)");
        const auto word = [](const pybind11::object& o) {
            const uint64_t v = PyLong_AsUnsignedLongLongMask(pybind11::int_(o).ptr());
            if (PyErr_Occurred()) throw pybind11::error_already_set();
            return v;
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
using MaybeTensor = std::optional<Tensor>;
MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : std::nullopt; }
Tensor tensor_of(const MaybeTensor& t) { return t ? *t : Tensor(); }

// ---- dropout ---------------------------------------------------------------------------------------------------------------

Tensor dropout_launch(const Tensor& x, const Tensor& residual, double p, const Rng& rng, at::ScalarType out_type) {
    const c10::DeviceGuard guard(x.device());
    const Rows l(x.sizes(), {x, residual});
    Tensor out = at::empty(x.sizes(), x.options().dtype(out_type));
    if (l.rows * l.d > 0)
        check(tvae_dropout(ptr(l.r[0].t), l.r[0].so, l.r[0].si, ptr(l.r[1].t), l.r[1].so, l.r[1].si, l.grp, out_ptr(out), l.rows, l.d, p,
                           rng.device(), rng.seed, rng.offset, code_of(x.scalar_type()), code_of(out_type), stream_of(x)), "tvae_dropout");
    return out;
}

struct DropoutNode : torch::autograd::Function<DropoutNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& residual_, double p, const Rng& rng) {
        const Tensor residual = tensor_of(residual_);
        ctx->saved_data["add"] = residual.defined();
        ctx->save_for_backward({rng.state});
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = (int64_t)rng.seed;
        ctx->saved_data["offset"] = (int64_t)rng.offset;
        ctx->saved_data["type"] = (int64_t)x.scalar_type();
        return dropout_launch(x, residual, p, rng, residual.defined() ? residual.scalar_type() : x.scalar_type());
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        refuse_default_stream("dropout");
        const Rng rng{ctx->get_saved_variables()[0], (uint64_t)ctx->saved_data["seed"].toInt(), (uint64_t)ctx->saved_data["offset"].toInt()};
        Tensor dx;
        if (ctx->needs_input_grad(0)) {
            const at::AutoDispatchBelowADInplaceOrView below;
            dx = dropout_launch(grads[0], {}, ctx->saved_data["p"].toDouble(), rng, (at::ScalarType)ctx->saved_data["type"].toInt());
        }
        return once({dx, ctx->saved_data["add"].toBool() && ctx->needs_input_grad(1) ? grads[0] : Tensor(), {}, {}});
    }
};

Tensor dropout(const Tensor& x, const std::optional<Tensor>& residual_, double p, const pybind11::object& rng_) {
    const char* what = residual_ ? "dropout_add" : "dropout";
    const Tensor residual = residual_.value_or(Tensor());
    check_rows(what, x);
    check_beside(what, "residual", x, residual, true);
    const Rng rng = check_dropout(what, x, p, rng_);
    const pybind11::gil_scoped_release release;
    if (at::GradMode::is_enabled() && (x.requires_grad() || (residual.defined() && residual.requires_grad())))
        return DropoutNode::apply(x, maybe(residual), p, rng);
    const at::AutoDispatchBelowADInplaceOrView below;
    return dropout_launch(x, residual, p, rng, residual.defined() ? residual.scalar_type() : x.scalar_type());
}

// ---- norms -----------------------------------------------------------------------------------------------------------------

struct NormOut { Tensor y, sum, mean, rstd; };

NormOut norm_forward(const Tensor& x, const Tensor& residual, const Tensor& weight_, const Tensor& bias_, int64_t kind, double eps, double p,
                     const Rng& rng, bool return_sum, bool stats) {
    const c10::DeviceGuard guard(x.device());
    const Rows l(x.sizes(), {x, residual});
    const at::ScalarType r_type = residual.defined() ? residual.scalar_type() : x.scalar_type();
    const Tensor weight = weight_.defined() ? weight_.contiguous() : weight_, bias = bias_.defined() ? bias_.contiguous() : bias_;
    const at::ScalarType w_type = weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : x.scalar_type();
    NormOut o;
    o.y = at::empty(x.sizes(), x.options());
    if (return_sum) o.sum = at::empty(x.sizes(), x.options().dtype(r_type));
    if (stats) {
        o.rstd = at::empty({l.rows}, x.options().dtype(at::kFloat));
        if (kind == TVAE_NORM_LAYER) o.mean = at::empty({l.rows}, x.options().dtype(at::kFloat));
    }
    if (l.rows > 0)
        check(tvae_norm_fwd((int)kind, ptr(l.r[0].t), l.r[0].so, l.r[0].si, ptr(l.r[1].t), l.r[1].so, l.r[1].si, l.grp, ptr(weight), ptr(bias), eps,
                            p, rng.device(), rng.seed, rng.offset, out_ptr(o.y), out_ptr(o.sum), (float*)out_ptr(o.mean),
                            (float*)out_ptr(o.rstd), l.rows, l.d, code_of(x.scalar_type()), code_of(w_type), code_of(r_type), stream_of(x)),
              "tvae_norm_fwd");
    return o;
}

// {norm(v), v or nothing} with v = [residual +] dropout(x): one node for the sum, the dropout and the norm
struct NormNode : torch::autograd::Function<NormNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& residual_, const MaybeTensor& weight_,
                                 const MaybeTensor& bias_, int64_t kind, double eps, double p, const Rng& rng, bool return_sum) {
        const Tensor residual = tensor_of(residual_), weight = tensor_of(weight_), bias = tensor_of(bias_);
        ctx->set_materialize_grads(false);
        const NormOut o = norm_forward(x, residual, weight, bias, kind, eps, p, rng, return_sum, true);
        // The backward pass needs v in fp32: it forms it again from x and the residual, or reads the returned sum where that holds
        // v as it is (fp32: 4 bytes an element for the 4 + 2 or 4 + 4 of x and residual).  A 16-bit sum would put its rounding
        // into the weights' gradient.
        const bool kept = return_sum && o.sum.scalar_type() == at::kFloat;
        ctx->save_for_backward({kept ? Tensor() : x, kept ? o.sum : residual, weight, o.mean, o.rstd, rng.state});
        ctx->saved_data["shape"] = x.sizes().vec();
        const auto type = [](const Tensor& t) { return t.defined() ? (int64_t)t.scalar_type() : (int64_t)-1; };
        ctx->saved_data["meta"] = std::vector<int64_t>{type(x), type(residual), type(weight), type(bias), kind, (int64_t)rng.seed, (int64_t)rng.offset};
        ctx->saved_data["p"] = p;
        if (return_sum) return {o.y, o.sum};
        return {o.y};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        refuse_default_stream("norm");
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &residual = saved[1], &mean = saved[3], &rstd = saved[4];
        const auto meta = ctx->saved_data["meta"].toIntVector();
        const auto shape = ctx->saved_data["shape"].toIntVector();
        const double p = ctx->saved_data["p"].toDouble();
        const at::ScalarType x_type = (at::ScalarType)meta[0], r_type = meta[1] < 0 ? x_type : (at::ScalarType)meta[1];
        const at::ScalarType w_type = meta[2] >= 0 ? (at::ScalarType)meta[2] : meta[3] >= 0 ? (at::ScalarType)meta[3] : x_type;
        const Rng rng{saved[5], (uint64_t)meta[5], (uint64_t)meta[6]};
        size_t edge = 0;
        bool need[4];
        for (int i = 0; i < 4; ++i) need[i] = meta[i] >= 0 && ctx->needs_input_grad(edge++);
        const bool need_x = need[0], need_r = need[1], need_w = need[2], need_b = need[3];
        const Tensor dy = grads[0], ds = grads.size() > 1 ? grads[1] : Tensor();
        Tensor dx, dr, dw, db;
        {
            const at::AutoDispatchBelowADInplaceOrView below;
            if (!dy.defined()) {                // only the sum was used: the norm has no part in the gradient
                if (ds.defined()) {
                    if (need_x) dx = dropout_launch(ds, {}, p, rng, x_type);
                    if (need_r) dr = ds;
                }
            } else {
                const c10::DeviceGuard guard(dy.device());
                const Rows l(shape, {dy, ds, x, residual});
                // without dropout x and a residual of its type have one gradient
                const bool shared = need_x && need_r && p == 0.0 && r_type == x_type;
                if (need_x) dx = at::empty(shape, dy.options().dtype(x_type));
                if (need_r && !shared) dr = at::empty(shape, dy.options().dtype(r_type));
                if (need_w) dw = at::empty({l.d}, dy.options().dtype(w_type));
                if (need_b) db = at::empty({l.d}, dy.options().dtype(w_type));
                if (l.rows == 0) {
                    if (need_w) dw.zero_();
                    if (need_b) db.zero_();
                } else {
                    Tensor ws;
                    const int64_t bytes = need_w || need_b ? tvae_norm_bwd_workspace_bytes(l.rows, l.d) : 0;
                    if (bytes > 0) ws = at::empty({bytes}, dy.options().dtype(at::kByte));
                    const Tensor weight = saved[2].defined() ? saved[2].contiguous() : saved[2];
                    check(tvae_norm_bwd((int)meta[4], ptr(l.r[0].t), l.r[0].so, l.r[0].si, ptr(l.r[1].t), l.r[1].so, l.r[1].si, ptr(l.r[2].t),
                                        l.r[2].so, l.r[2].si, ptr(l.r[3].t), l.r[3].so, l.r[3].si, l.grp, ptr(weight), (const float*)ptr(mean),
                                        (const float*)ptr(rstd), p, rng.device(), rng.seed, rng.offset, out_ptr(dx), out_ptr(dr), out_ptr(dw),
                                        out_ptr(db), l.rows, l.d, code_of(x_type), code_of(w_type), code_of(r_type), out_ptr(ws), bytes,
                                        stream_of(dy)), "tvae_norm_bwd");
                }
                if (shared) dr = dx;
            }
        }
        return once({dx, dr, dw, db, {}, {}, {}, {}, {}});
    }
};

pybind11::object norm(const char* what, int64_t kind, const Tensor& x, const std::optional<Tensor>& residual_, const std::optional<Tensor>& weight_,
                      const std::optional<Tensor>& bias_, double eps, double p, const pybind11::object& rng_, bool return_sum) {
    const Tensor residual = residual_.value_or(Tensor()), weight = weight_.value_or(Tensor()), bias = bias_.value_or(Tensor());
    check_rows(what, x);
    check_beside(what, "residual", x, residual, true);
    check_beside(what, "weight", x, weight, false);
    check_beside(what, "bias", x, bias, false);
    TORCH_CHECK_VALUE(x.size(-1) > 0, what, ": the last axis is empty");
    if (weight.defined() && bias.defined())
        TORCH_CHECK_TYPE(weight.scalar_type() == bias.scalar_type(), what,
                         ": weight and bias are of one type, got ", name_of(weight.scalar_type()), " and ", name_of(bias.scalar_type()));
    TORCH_CHECK_VALUE(eps >= 0.0 && eps < 1e30, what, ": eps must be a finite number >= 0, got ", eps);
    const Rng rng = check_dropout(what, x, p, rng_);
    const auto wants = [](const Tensor& t) { return t.defined() && t.requires_grad(); };
    variable_list out;
    {
        const pybind11::gil_scoped_release release;
        if (at::GradMode::is_enabled() && (wants(x) || wants(residual) || wants(weight) || wants(bias))) {
            out = NormNode::apply(x, maybe(residual), maybe(weight), maybe(bias), kind, eps, p, rng, return_sum);
        } else {
            const at::AutoDispatchBelowADInplaceOrView below;
            NormOut o = norm_forward(x, residual, weight, bias, kind, eps, p, rng, return_sum, false);
            out = {o.y, o.sum};
        }
    }
    if (return_sum) return pybind11::make_tuple(out[0], out[1]);
    return pybind11::cast(out[0]);
}

}  // namespace

PYBIND11_MODULE(_host, m) {
    m.doc() = "autograd nodes of the norm and dropout operators";
    m.def("norm", &norm);
    m.def("dropout", &dropout);
}
