// The feature operators (embed, layer_norm, dropout) as differentiable torch functions: argument
// checks, output and workspace allocation, the autograd nodes, and the calls into libigs_b200.so.
//
// Why this is C++ while the splat's autograd Functions are Python: a splat takes hundreds of
// microseconds on the device, these operators on the features of one image a few, and a Python
// autograd Function with its ctypes call costs more than the kernels.  Forward and gradient of a
// 128 x 1024 layer norm, issued back to back: 131 us that way, 69 this way; torch's own negation of one
// such tensor and its gradient take 50 on the same host.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <optional>

#include "../../../include/igs_b200.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

struct Failure : std::runtime_error {
    std::string fn;
    int code;
    Failure(const char* f, int c)
        : std::runtime_error(std::string(f) + " failed with code " + std::to_string(c) + ": " + igs_strerror(c)),
          fn(f), code(c) {}
};

void check(const char* fn, int code) {
    if (code) throw Failure(fn, code);
}

int type_code(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return IGS_F32;
        case at::kBFloat16: return IGS_BF16;
        case at::kHalf: return IGS_F16;
        default: return -1;
    }
}

// These functions are not dispatched operators: torch would take their results for constants where it
// looks for a tangent or records a trace.
void refuse_forward_mode(const Tensor& t) {
    TORCH_CHECK(!torch::autograd::isFwGradDefined(t), "the feature operators of igs_b200 have no forward-mode derivative");
}
void refuse_tracing() {
    TORCH_CHECK(!torch::jit::tracer::isTracing(), "the feature operators of igs_b200 cannot be traced (torch.jit.trace)");
}

void require_features(const char* name, const Tensor& t) {
    TORCH_CHECK(t.is_cuda(), name, " is on ", t.device(), ": igs_b200 runs on CUDA devices only (no CPU path)");
    TORCH_CHECK_TYPE(type_code(t.scalar_type()) >= 0, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
    refuse_forward_mode(t);
}

void same_device(const char* name, const Tensor& t, const Tensor& first) {
    TORCH_CHECK(t.device() == first.device(), "all tensors must be on one device; got ", first.device(), " and ", name,
                " on ", t.device());
}

float finite(const char* name, double v) {
    const float f = static_cast<float>(v);
    TORCH_CHECK_VALUE(std::isfinite(f), name, " must be a finite 32-bit number, got ", v);
    return f;
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
int device_index(const Tensor& t) { return t.device().index(); }
void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// The tensor with its values in its memory: torch keeps the sign of some views beside it.
Tensor in_memory(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

Tensor workspace(size_t bytes, const Tensor& like) {
    return at::empty({static_cast<int64_t>(bytes < 256 ? 256 : bytes)}, like.options().dtype(at::kByte));
}

// A tensor that comes back in a backward pass: the upstream gradient, or one that a saved-tensor hook
// may have replaced (copied to another place, say).  Values are taken on trust, the layout is the
// tensor's own, and what the kernels' addresses go by is checked.
Tensor came_back(const char* name, Tensor t, at::IntArrayRef sizes, at::ScalarType type, at::Device device) {
    TORCH_CHECK(t.defined() && t.sizes() == sizes && t.scalar_type() == type && t.device() == device, name,
                " came back in the backward pass as another tensor than went in: expected ", type, " ", sizes, " on ", device,
                t.defined() ? c10::str(", got ", t.scalar_type(), " ", t.sizes(), " on ", t.device()) : ", got nothing");
    return in_memory(t);
}

// The upstream gradient of a node's only output, contiguous.
Tensor upstream(const torch::autograd::Node& node, const Tensor& grad) {
    const auto& out = node.input_metadata(0);
    refuse_forward_mode(grad);
    return came_back("the upstream gradient", grad, C10_AS_INTARRAYREF_SLOW(out.shape_as_dim_vector()),
                     c10::typeMetaToScalarType(out.dtype()), out.device()).contiguous();
}

// What a backward pass under create_graph hands on: gradients that raise when they are
// differentiated again, instead of passing for constants.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    for (auto& g : grads)
        if (g.defined()) g = g.detach().requires_grad_();
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "the feature operators of igs_b200 are differentiable once", static_cast<int64_t>(grads.size()));
    return (*error)(std::move(grads));
}

template <typename N>
std::shared_ptr<N> make_node() {
    return std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
}

// ---------------------------------------------------------------------------
// embedding lookup
// ---------------------------------------------------------------------------
struct EmbedCall {
    std::vector<int64_t> shape;  // of the tokens
    at::ScalarType index = at::kLong;
    int64_t rows = 0, width = 0;
    float scale = 1;
    int has_empty = 0;
    int64_t empty = 0;
};

struct EmbedBackward : torch::autograd::Node {
    SavedVariable tokens_;
    EmbedCall call;

    variable_list apply(variable_list&& grads) override {
        variable_list res(1);
        if (!grads[0].defined() || !task_should_compute_output(0)) return res;
        const Tensor dy = upstream(*this, grads[0]);
        const Tensor tokens = came_back("tokens", tokens_.unpack(), call.shape, call.index, dy.device()).contiguous();
        const int64_t n = tokens.numel();
        Tensor d_table = at::empty({call.rows, call.width}, dy.options());
        size_t bytes = 0;
        check("igs_embed_grad_workspace_bytes",
              igs_embed_grad_workspace_bytes(n, call.rows, call.width, type_code(dy.scalar_type()), device_index(dy), &bytes));
        Tensor ws = workspace(bytes, dy);
        check("igs_embed_grad",
              igs_embed_grad(tokens.data_ptr(), static_cast<int>(tokens.element_size()), n, dy.data_ptr(),
                             type_code(dy.scalar_type()), call.rows, call.width, call.scale, call.has_empty, call.empty,
                             d_table.data_ptr(), ws.data_ptr(), bytes, device_index(dy), stream_of(dy)));
        res[0] = d_table;
        return once(std::move(res));
    }
    std::string name() const override { return "igs_b200::EmbedBackward"; }
    void release_variables() override { tokens_.reset_data(); }
};

Tensor embed(const Tensor& tokens, const Tensor& table, double scale, std::optional<int64_t> empty) {
    refuse_tracing();
    require_features("table", table);
    TORCH_CHECK_TYPE(tokens.scalar_type() == at::kInt || tokens.scalar_type() == at::kLong,
                     "tokens must be int32 or int64, got ", tokens.scalar_type());
    same_device("tokens", tokens, table);
    TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) >= 1 && table.size(1) >= 1,
                      "table must be [rows,D] with at least one row and column, got ", table.sizes());
    EmbedCall c;
    c.rows = table.size(0);
    c.width = table.size(1);
    c.scale = finite("scale", scale);
    c.has_empty = empty.has_value();
    c.empty = empty.value_or(0);

    std::shared_ptr<EmbedBackward> node;
    const bool grad = torch::autograd::compute_requires_grad(table);
    Tensor out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor tok = in_memory(tokens).contiguous();
        Tensor tab = in_memory(table);
        if (tab.stride(1) != 1 && c.width != 1) tab = tab.contiguous();
        auto shape = tokens.sizes().vec();
        shape.push_back(c.width);
        out = at::empty(shape, table.options());
        check("igs_embed",
              igs_embed(tok.data_ptr(), static_cast<int>(tok.element_size()), tok.numel(), tab.data_ptr(),
                        type_code(tab.scalar_type()), c.rows, c.width, c.rows > 1 ? tab.stride(0) : c.width, c.scale,
                        c.has_empty, c.empty, out.data_ptr(), device_index(tab), stream_of(tab)));
        if (grad) {
            node = make_node<EmbedBackward>();
            c.shape = tok.sizes().vec();
            c.index = tok.scalar_type();
            node->call = std::move(c);
            node->tokens_ = SavedVariable(tok, false);
        }
    }
    if (grad) {
        node->set_next_edges(torch::autograd::collect_next_edges(table));
        torch::autograd::set_history(out, node);
    }
    return out;
}

// ---------------------------------------------------------------------------
// layer norm
// ---------------------------------------------------------------------------
struct Rows {
    int64_t count, width, stride;
};

// x as rows of its last dimension where they lie: false when its strides do not allow it
bool as_rows(const Tensor& x, Rows& r) {
    const auto sizes = x.sizes(), strides = x.strides();
    const int64_t last = x.dim() - 1;
    r.width = sizes[last];
    r.count = 1;
    r.stride = r.width;
    if (x.numel() == 0) {
        r.count = 0;
        return true;
    }
    if (strides[last] != 1 && r.width != 1) return false;
    for (int64_t d = last - 1; d >= 0; --d) {
        if (sizes[d] == 1) continue;
        if (r.count == 1) r.stride = strides[d];
        else if (strides[d] != r.stride * r.count) return false;
        r.count *= sizes[d];
    }
    return true;
}

struct NormBackward : torch::autograd::Node {
    SavedVariable x_, weight_;
    Tensor stats;  // [rows, 4]
    bool weighted;
    at::ScalarType wtype;

    variable_list apply(variable_list&& grads) override {
        variable_list res(3);
        if (!grads[0].defined()) return res;
        const Tensor dy = upstream(*this, grads[0]);
        Tensor x = came_back("x", x_.unpack(), dy.sizes(), dy.scalar_type(), dy.device()), weight = weight_.unpack();
        Rows rows;  // (of the tensor that came back)
        if (!as_rows(x, rows)) {
            x = x.contiguous();
            as_rows(x, rows);
        }
        if (weighted) weight = came_back("weight", weight, {rows.width}, wtype, dy.device()).contiguous();
        const bool want_w = task_should_compute_output(1), want_b = task_should_compute_output(2);
        if (task_should_compute_output(0)) res[0] = at::empty(x.sizes(), dy.options());
        if (want_w) res[1] = at::empty({rows.width}, dy.options().dtype(wtype));
        if (want_b) res[2] = at::empty({rows.width}, dy.options().dtype(wtype));
        Tensor ws;
        size_t bytes = 0;
        if (want_w || want_b) {
            bytes = igs_layer_norm_grad_workspace_bytes(rows.count, rows.width, device_index(dy));
            ws = workspace(bytes, dy);
        }
        check("igs_layer_norm_grad",
              igs_layer_norm_grad(dy.data_ptr(), x.data_ptr(), type_code(dy.scalar_type()), rows.count, rows.width,
                                  rows.stride, data(weight), type_code(wtype), stats.data_ptr<float>(), data(res[0]),
                                  data(res[1]), data(res[2]), data(ws), bytes, device_index(dy), stream_of(dy)));
        return once(std::move(res));
    }
    std::string name() const override { return "igs_b200::NormBackward"; }
    void release_variables() override {
        x_.reset_data();
        weight_.reset_data();
        stats.reset();
    }
};

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight_, const std::optional<Tensor>& bias_, double eps) {
    refuse_tracing();
    require_features("x", x);
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must be [...,D] with D >= 1, got ", x.sizes());
    const int64_t D = x.size(-1);
    at::ScalarType wtype = x.scalar_type();
    Tensor given[2] = {weight_.value_or(Tensor()), bias_.value_or(Tensor())};
    bool typed = false;
    for (int i = 0; i < 2; ++i) {
        const Tensor& t = given[i];
        const char* name = i ? "bias" : "weight";
        if (!t.defined()) continue;
        require_features(name, t);
        same_device(name, t, x);
        TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == D, name, " must be [D] = [", D, "], got ", t.sizes());
        TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat, name,
                         " must be of x's type (", x.scalar_type(), ") or float32, got ", t.scalar_type());
        TORCH_CHECK_TYPE(!typed || t.scalar_type() == wtype, "weight and bias must be of one type, got ", wtype, " and ",
                         t.scalar_type());
        wtype = t.scalar_type();
        typed = true;
    }
    const float e = finite("eps", eps);
    TORCH_CHECK_VALUE(e >= 0, "eps must not be negative, got ", eps);

    const bool grad = torch::autograd::compute_requires_grad(x, given[0], given[1]);
    std::shared_ptr<NormBackward> node;
    Tensor y;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        Rows r;
        Tensor src = in_memory(x);
        if (!as_rows(src, r)) {
            src = src.contiguous();
            as_rows(src, r);
        }
        const Tensor w = given[0].defined() ? in_memory(given[0]).contiguous() : Tensor();
        const Tensor b = given[1].defined() ? in_memory(given[1]).contiguous() : Tensor();
        y = at::empty(x.sizes(), x.options());
        Tensor stats;
        if (grad) stats = at::empty({r.count, 4}, x.options().dtype(at::kFloat));
        check("igs_layer_norm",
              igs_layer_norm(src.data_ptr(), type_code(x.scalar_type()), r.count, D, r.stride, data(w), data(b),
                             type_code(wtype), e, y.data_ptr(), grad ? stats.data_ptr<float>() : nullptr, device_index(x),
                             stream_of(x)));
        if (grad) {
            node = make_node<NormBackward>();
            node->x_ = SavedVariable(src, false);
            node->weight_ = SavedVariable(w, false);
            node->stats = stats;
            node->weighted = w.defined();
            node->wtype = wtype;
        }
    }
    if (grad) {
        node->set_next_edges(torch::autograd::collect_next_edges(x, given[0], given[1]));
        torch::autograd::set_history(y, node);
    }
    return y;
}

// ---------------------------------------------------------------------------
// dropout
// ---------------------------------------------------------------------------
struct DropoutCall {
    double p;
    uint64_t seed, offset;
};

Tensor run_dropout(const Tensor& x, const DropoutCall& c, const Tensor& state) {
    Tensor y = at::empty(x.sizes(), x.options());
    check("igs_dropout",
          igs_dropout(x.data_ptr(), type_code(x.scalar_type()), x.numel(), c.p, c.seed, c.offset,
                      state.defined() ? reinterpret_cast<const long long*>(state.data_ptr<int64_t>()) : nullptr,
                      y.data_ptr(), device_index(x), stream_of(x)));
    return y;
}

struct DropoutBackward : torch::autograd::Node {
    SavedVariable state_;
    DropoutCall call;
    bool stateful;

    variable_list apply(variable_list&& grads) override {
        variable_list res(1);
        if (!grads[0].defined() || !task_should_compute_output(0)) return res;
        const Tensor dy = upstream(*this, grads[0]);
        Tensor state = state_.unpack();
        if (stateful) state = came_back("seed", state, {2}, at::kLong, dy.device()).contiguous();
        res[0] = run_dropout(dy, call, state);
        return once(std::move(res));
    }
    std::string name() const override { return "igs_b200::DropoutBackward"; }
    void release_variables() override { state_.reset_data(); }
};

Tensor dropout(const Tensor& x, double p, uint64_t seed, uint64_t offset, const std::optional<Tensor>& state) {
    refuse_tracing();
    require_features("x", x);
    TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "p must be in 0 .. 1, got ", p);
    if (state) {
        TORCH_CHECK_VALUE(state->scalar_type() == at::kLong && state->dim() == 1 && state->size(0) == 2,
                          "seed must be a number or an int64 tensor of two values, got ", state->scalar_type(), " ",
                          state->sizes());
        same_device("seed", *state, x);
    }
    const DropoutCall call{p, seed, offset};
    const bool grad = torch::autograd::compute_requires_grad(x);
    std::shared_ptr<DropoutBackward> node;
    Tensor y;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor st = state ? in_memory(*state).contiguous() : Tensor();
        y = run_dropout(in_memory(x).contiguous(), call, st);
        if (grad) {
            node = make_node<DropoutBackward>();
            node->call = call;
            node->stateful = st.defined();
            node->state_ = SavedVariable(st, false);
        }
    }
    if (grad) {
        node->set_next_edges(torch::autograd::collect_next_edges(x));
        torch::autograd::set_history(y, node);
    }
    return y;
}

}  // namespace

PYBIND11_MODULE(_features, m) {
    // the package's own exception class, with its arguments (function, code, message)
    pybind11::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Failure& f) {
            const auto cls = pybind11::module_::import("igs_b200._lib").attr("IgsError");
            PyErr_SetObject(cls.ptr(), cls(f.fn, f.code, igs_strerror(f.code)).ptr());
        }
    });
    m.def("embed", &embed, pybind11::arg("tokens"), pybind11::arg("table"), pybind11::arg("scale"), pybind11::arg("empty"));
    m.def("layer_norm", &layer_norm, pybind11::arg("x"), pybind11::arg("weight"), pybind11::arg("bias"),
          pybind11::arg("eps"));
    m.def("dropout", &dropout, pybind11::arg("x"), pybind11::arg("p"), pybind11::arg("seed"), pybind11::arg("offset"),
          pybind11::arg("state"));
}
