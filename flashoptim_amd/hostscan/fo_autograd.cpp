// _fo_autograd: the calls of the norm, the embedding and the loss over tensor objects, and their nodes in the autograd graph.
//
// What such a call does on the host (argument checks, allocations, launches) and the way into and out of a Python autograd function cost more
// than the kernels take for small batches: 146 us for a norm with three gradients of 1003 rows whose kernels take 30.  Here the checks and
// allocations are C++ and the backward pass runs in the engine's thread without the interpreter.  It is host code only; the kernels are reached through the
// addresses of the C entry points that the Python binding hands over.  The package does the same in Python when the module has not been built
// (flashoptim_amd/norm.py, embed.py, loss.py), and for every call that is out of the ordinary: a function here gives None, and has done nothing, for
// operands that are not plain strided tensors of this device with adjacent values, and where torch's operations are recorded, of which a launch is none; the Python
// path checks, converts, records and raises.
//
// kinds                                                dict from the name of a C entry point to the types it was built to call it with, and of sizes
// bind(addresses)                                      dict from the name of a C entry point to its address
// rms_norm(x, weight, residual, eps)                   None | y | (y, stream)
// rms_norm_mxfp4(x, weight, residual, eps)             None | (codes, scales) | (codes, scales, stream)
// embedding(tokens, weight, scale, padding)            None | y
// linear_cross_entropy(x, weight, target, ignore, reduction, smoothing)     None | loss
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cmath>
#include <mutex>
#include <string>
#include <type_traits>

#include "../../include/flashoptim_hip.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

#define FO_ENTRIES(X)                                                                                                        \
    X(fo_last_error) X(fo_rms_norm) X(fo_rms_norm_mxfp4) X(fo_rms_norm_backward_workspace) X(fo_rms_norm_backward) X(fo_embedding) \
    X(fo_embedding_backward_workspace) X(fo_embedding_backward) X(fo_linear_cross_entropy_workspace) X(fo_linear_cross_entropy) \
    X(fo_linear_cross_entropy_backward_workspace) X(fo_linear_cross_entropy_backward)

struct Api {
#define FO_MEMBER(name) decltype(&::name) name = nullptr;
    FO_ENTRIES(FO_MEMBER)
#undef FO_MEMBER
    bool bound = false;
} api;

void check(int64_t rc, const char* what) { TORCH_CHECK(rc >= 0 && rc <= 0, what, " failed (code ", rc, "): ", api.fo_last_error()); }
void check_size(int64_t size, const char* what) {
    if (size < 0) check(size, what);
}

int code_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? FO_F32 : t.scalar_type() == at::kBFloat16 ? FO_BF16 : FO_F16; }
int index_bytes(const Tensor& t) { return t.scalar_type() == at::kLong ? 8 : 4; }
void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }

// Whether somebody may be looking at the operations that are called here.
bool watched() {
    return torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::any_modes_set() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch);
}

// An ordinary tensor on a GPU; null for any other object.
const Tensor* tensor_of(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.layout() != at::kStrided || !t.has_storage() || t._is_zerotensor() || t.is_neg() || t._fw_grad(0).defined()) return nullptr;
    return &t;
}
bool is_values(const Tensor& t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }
const Tensor* values_of(PyObject* o) {
    const Tensor* t = tensor_of(o);
    return t && is_values(*t) && t->dim() > 0 ? t : nullptr;
}
bool optional_values(PyObject* o, const Tensor*& t) {
    t = nullptr;
    if (o == Py_None) return true;
    return (t = values_of(o)) != nullptr;
}
// Rows of adjacent values, one distance apart: a matrix, or a contiguous tensor.
bool is_rows(const Tensor& t) {
    if (t.dim() == 2) return t.size(1) <= 1 || t.stride(1) == 1;
    return t.is_contiguous();
}
int64_t row_stride(const Tensor& t) { return t.dim() == 2 ? t.stride(0) : t.size(-1); }
Tensor as_rows(const Tensor& t) {
    const Tensor u = t.is_neg() ? t.resolve_neg() : t;
    return is_rows(u) ? u : u.contiguous();
}
int64_t leading(const Tensor& t) { return c10::multiply_integers(t.sizes().slice(0, t.dim() - 1)); }
bool records(std::initializer_list<const Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t && t->requires_grad()) return true;
    return false;
}

// A node's tensors are taken and released under its mutex_: backward passes of one graph may run in several threads.
typedef std::lock_guard<std::mutex> Lock;

// A tensor kept for the backward pass.  Hooks on saved tensors may lay it out anew, but not give back another one.
struct Kept {
    SavedVariable saved;
    c10::SmallVector<int64_t, 6> sizes;
    at::ScalarType type = at::kFloat;
    c10::Device device = c10::Device(at::kCPU);

    void keep(const Tensor& t, bool is_output = false) {
        saved = SavedVariable(t, is_output);
        sizes.assign(t.sizes().begin(), t.sizes().end());
        type = t.scalar_type();
        device = t.device();
    }
    void release() { saved.reset_data(); }
    // As the kernels read it.
    Tensor take(const char* what, std::shared_ptr<Node> owner = nullptr) const {
        const Tensor t = saved.unpack(std::move(owner));
        TORCH_CHECK(t.defined() && t.sizes() == at::IntArrayRef(sizes) && t.scalar_type() == type && t.device() == device && t.layout() == at::kStrided, what,
                    ": a hook on saved tensors gave back another tensor than the one it was given");
        at::NoGradGuard none;
        return as_rows(t);
    }
};

// Gradients have no derivative here: in a graph that records the backward pass they lead to an error.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    for (Tensor& g : grads) {
        if (!g.defined()) continue;
        auto error = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that has one derivative only", 1);
        g = (*error)({g.detach().requires_grad_()})[0];
    }
    return grads;
}

// ---------------------------------------------------------------------------------------------------- norm
struct NormNode : Node {
    Kept s, weight, inverse;
    bool has_weight = false, has_residual = false;
    at::ScalarType x_type;
    std::vector<int64_t> sizes;

    void release_variables() override {
        const Lock lock(mutex_);
        s.release();
        weight.release();
        inverse.release();
    }
    std::string name() const override { return "RMSNormBackward"; }

    variable_list apply(variable_list&& grads) override {
        variable_list out(3);    // x, weight, residual
        const bool with_stream = grads.size() > 1 && grads[1].defined();
        const bool need_dx = task_should_compute_output(0), need_dw = has_weight && task_should_compute_output(1), need_dresidual = has_residual && task_should_compute_output(2);
        if (!grads[0].defined()) {    // nothing comes from the norm, whatever stands in its rows
            if (!with_stream) return out;
            {
                at::NoGradGuard none;
                if (need_dx) out[0] = grads[1].to(x_type);
                if (need_dw) out[1] = at::zeros(weight.sizes, grads[1].options().dtype(weight.type));
                if (need_dresidual) out[2] = grads[1];
            }
            return once(std::move(out));
        }
        Tensor s, weight, inverse;
        {
            const Lock lock(mutex_);
            s = this->s.take("rms_norm", has_residual ? getptr() : nullptr);
            if (has_weight) weight = this->weight.take("rms_norm");
            inverse = this->inverse.take("rms_norm");
        }
        {
            at::NoGradGuard none;
            const c10::DeviceGuard guard(s.device());
            const int64_t width = s.size(-1), rows = inverse.numel();
            const bool same = s.scalar_type() == x_type;
            const Tensor dy = as_rows(grads[0]), dstream = with_stream ? as_rows(grads[1]) : Tensor();
            Tensor dx, dresidual, dw, workspace;
            if (need_dx || (need_dresidual && same)) dx = at::empty(sizes, s.options().dtype(x_type));
            if (need_dresidual && !same) dresidual = at::empty(sizes, s.options());
            int64_t size = 0;
            if (need_dw) {
                dw = rows ? at::empty(weight.sizes(), weight.options()) : at::zeros(weight.sizes(), weight.options());
                size = api.fo_rms_norm_backward_workspace(rows, width);
                check_size(size, "fo_rms_norm_backward");
                workspace = bytes(size, s);
            }
            check(api.fo_rms_norm_backward(s.data_ptr(), code_of(s), row_stride(s), ptr(weight), has_weight ? code_of(weight) : 0, (const float*)inverse.data_ptr(), dy.data_ptr(),
                                           code_of(dy), row_stride(dy), ptr(dstream), with_stream ? row_stride(dstream) : 0, rows, width, ptr(dx), ptr(dresidual), ptr(dw),
                                           ptr(workspace), size, stream_of(s)),
                  "fo_rms_norm_backward");
            if (need_dx) out[0] = dx;
            out[1] = dw;
            if (need_dresidual) out[2] = same ? dx : dresidual;
        }
        return once(std::move(out));
    }
};

PyObject* rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4 || !api.bound || watched()) Py_RETURN_NONE;
    const Tensor *x = values_of(args[0]), *weight, *residual;
    if (!x || !optional_values(args[1], weight) || !optional_values(args[2], residual)) Py_RETURN_NONE;
    const double eps = PyFloat_AsDouble(args[3]);
    if (PyErr_Occurred()) return nullptr;
    const int64_t width = x->size(-1), rows = leading(*x);
    if (!is_rows(*x) || !(eps >= 0.0 && eps < 1e30)) Py_RETURN_NONE;
    if (weight && (weight->dim() != 1 || weight->size(0) != width || weight->device() != x->device() || (width > 1 && weight->stride(0) != 1))) Py_RETURN_NONE;
    if (residual && (residual->sizes() != x->sizes() || residual->device() != x->device() || !is_rows(*residual) ||
                     (residual->scalar_type() != x->scalar_type() && residual->scalar_type() != at::kFloat)))
        Py_RETURN_NONE;
    Tensor y, stream;
    {
        const bool keep = records({x, weight, residual});
        std::shared_ptr<NormNode> node;
        if (keep) {
            node = std::shared_ptr<NormNode>(new NormNode(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(*x, weight ? *weight : Tensor(), residual ? *residual : Tensor()));
        }
        const c10::DeviceGuard guard(x->device());
        Tensor inverse;
        {
            at::NoGradGuard none;
            y = at::empty(x->sizes(), x->options());
            if (residual) stream = at::empty(x->sizes(), residual->options());
            if (keep) inverse = at::empty({rows}, x->options().dtype(at::kFloat));
            check(api.fo_rms_norm(x->data_ptr(), code_of(*x), rows, width, row_stride(*x), residual ? residual->data_ptr() : nullptr, residual ? code_of(*residual) : 0,
                                  residual ? row_stride(*residual) : 0, weight ? weight->data_ptr() : nullptr, weight ? code_of(*weight) : 0, (float)eps, ptr(stream), y.data_ptr(),
                                  (float*)ptr(inverse), stream_of(*x)),
                  "fo_rms_norm");
        }
        if (keep) {
            node->x_type = x->scalar_type();
            node->sizes = x->sizes().vec();
            node->has_weight = weight != nullptr;
            node->has_residual = residual != nullptr;
            torch::autograd::set_history(y, node);
            if (residual) torch::autograd::set_history(stream, node);
            node->s.keep(residual ? stream : *x, residual != nullptr);
            if (weight) node->weight.keep(*weight);
            node->inverse.keep(inverse);
        }
    }
    if (!residual) return THPVariable_Wrap(y);
    PyObject *first = THPVariable_Wrap(y), *second = THPVariable_Wrap(stream);
    PyObject* both = first && second ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return both;
    END_HANDLE_TH_ERRORS
}

PyObject* rms_norm_mxfp4(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4 || !api.bound || watched()) Py_RETURN_NONE;
    const Tensor *x = values_of(args[0]), *weight, *residual;
    if (!x || !optional_values(args[1], weight) || !optional_values(args[2], residual)) Py_RETURN_NONE;
    const double eps = PyFloat_AsDouble(args[3]);
    if (PyErr_Occurred()) return nullptr;
    if (x->dim() != 2 || !is_rows(*x) || !(eps >= 0.0 && eps < 1e30)) Py_RETURN_NONE;
    const int64_t rows = x->size(0), width = x->size(1), blocks = (width + 127) / 128;
    if (weight && (weight->dim() != 1 || weight->size(0) != width || weight->device() != x->device() || (width > 1 && weight->stride(0) != 1))) Py_RETURN_NONE;
    if (residual && (residual->sizes() != x->sizes() || residual->device() != x->device() || !is_rows(*residual) ||
                     (residual->scalar_type() != x->scalar_type() && residual->scalar_type() != at::kFloat)))
        Py_RETURN_NONE;
    Tensor codes, scales, stream;
    {
        at::NoGradGuard none;
        const c10::DeviceGuard guard(x->device());
        codes = at::empty({rows, blocks * 64}, x->options().dtype(at::kByte));
        scales = at::empty({rows, blocks * 4}, x->options().dtype(at::kByte));
        if (residual) stream = at::empty(x->sizes(), residual->options());
        check(api.fo_rms_norm_mxfp4(x->data_ptr(), code_of(*x), rows, width, row_stride(*x), residual ? residual->data_ptr() : nullptr, residual ? code_of(*residual) : 0,
                                    residual ? row_stride(*residual) : 0, weight ? weight->data_ptr() : nullptr, weight ? code_of(*weight) : 0, (float)eps, ptr(stream),
                                    codes.data_ptr(), scales.data_ptr(), stream_of(*x)),
              "fo_rms_norm_mxfp4");
    }
    PyObject *first = THPVariable_Wrap(codes), *second = THPVariable_Wrap(scales), *third = residual ? THPVariable_Wrap(stream) : nullptr;
    PyObject* all = !first || !second || (residual && !third) ? nullptr : residual ? PyTuple_Pack(3, first, second, third) : PyTuple_Pack(2, first, second);
    Py_XDECREF(first);
    Py_XDECREF(second);
    Py_XDECREF(third);
    return all;
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------------- embedding
struct EmbeddingNode : Node {
    Kept tokens;
    int64_t vocabulary = 0, width = 0, padding = -1;
    float scale = 1.0f;

    void release_variables() override {
        const Lock lock(mutex_);
        tokens.release();
    }
    std::string name() const override { return "EmbeddingBackward"; }

    variable_list apply(variable_list&& grads) override {
        variable_list out(1);
        if (!grads[0].defined()) return out;
        Tensor tokens;
        {
            const Lock lock(mutex_);
            tokens = this->tokens.take("embedding").contiguous();
        }
        {
            at::NoGradGuard none;
            const c10::DeviceGuard guard(tokens.device());
            const Tensor dy = as_rows(grads[0]);
            const int64_t size = api.fo_embedding_backward_workspace(tokens.numel(), vocabulary, width);
            check_size(size, "fo_embedding_backward");
            const Tensor workspace = bytes(size, tokens);
            out[0] = at::empty({vocabulary, width}, dy.options());
            check(api.fo_embedding_backward(tokens.data_ptr(), index_bytes(tokens), tokens.numel(), dy.data_ptr(), code_of(dy), row_stride(dy), vocabulary, width, scale, padding,
                                            out[0].data_ptr(), workspace.data_ptr(), size, stream_of(tokens)),
                  "fo_embedding_backward");
        }
        return once(std::move(out));
    }
};

PyObject* embedding(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4 || !api.bound || watched()) Py_RETURN_NONE;
    const Tensor *tokens = tensor_of(args[0]), *weight = values_of(args[1]);
    if (!tokens || !weight) Py_RETURN_NONE;
    const double scale = PyFloat_AsDouble(args[2]);
    const int64_t padding = PyLong_AsLongLong(args[3]);
    if (PyErr_Occurred()) return nullptr;
    if ((tokens->scalar_type() != at::kLong && tokens->scalar_type() != at::kInt) || !tokens->is_contiguous() || tokens->device() != weight->device() || weight->dim() != 2 ||
        !is_rows(*weight) || !std::isfinite(scale))
        Py_RETURN_NONE;
    const int64_t vocabulary = weight->size(0), width = weight->size(1);
    c10::SmallVector<int64_t, 6> sizes(tokens->sizes().begin(), tokens->sizes().end());
    sizes.push_back(width);
    Tensor y;
    {
        const c10::DeviceGuard guard(weight->device());
        {
            at::NoGradGuard none;
            y = at::empty(sizes, weight->options());
            check(api.fo_embedding(tokens->data_ptr(), index_bytes(*tokens), tokens->numel(), weight->data_ptr(), code_of(*weight), vocabulary, width, weight->stride(0), (float)scale,
                                   y.data_ptr(), stream_of(*weight)),
                  "fo_embedding");
        }
        if (records({weight})) {
            auto node = std::shared_ptr<EmbeddingNode>(new EmbeddingNode(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(*weight));
            node->tokens.keep(*tokens);
            node->vocabulary = vocabulary;
            node->width = width;
            node->padding = padding;
            node->scale = (float)scale;
            torch::autograd::set_history(y, node);
        }
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------------- loss
struct LossNode : Node {
    Kept x, weight, kept;
    int reduction = 0;
    float smoothing = 0.0f;

    void release_variables() override {
        const Lock lock(mutex_);
        x.release();
        weight.release();
        kept.release();
    }
    std::string name() const override { return "LinearCrossEntropyBackward"; }

    variable_list apply(variable_list&& grads) override {
        variable_list out(2);
        if (!grads[0].defined()) return out;
        Tensor x, weight, kept;
        {
            const Lock lock(mutex_);
            const char* what = "linear_cross_entropy";
            x = this->x.take(what);
            weight = this->weight.take(what);
            kept = this->kept.take(what);
        }
        const bool need_dx = task_should_compute_output(0), need_dw = task_should_compute_output(1);
        if (!need_dx && !need_dw) return out;
        {
            at::NoGradGuard none;
            const c10::DeviceGuard guard(x.device());
            const int64_t width = x.size(-1), tokens = leading(x), vocabulary = weight.size(0);
            Tensor upstream = grads[0].is_neg() ? grads[0].resolve_neg() : grads[0];
            if (upstream.dim() > 1) upstream = upstream.reshape({tokens});
            const int64_t size = api.fo_linear_cross_entropy_backward_workspace(x.data_ptr(), code_of(x), tokens, row_stride(x), weight.data_ptr(), weight.stride(0), vocabulary,
                                                                                width, need_dx, need_dw);
            check_size(size, "fo_linear_cross_entropy_backward");
            const Tensor workspace = bytes(size, x);
            if (need_dx) out[0] = at::empty(x.sizes(), x.options());
            if (need_dw) out[1] = at::empty({vocabulary, width}, weight.options());
            check(api.fo_linear_cross_entropy_backward(x.data_ptr(), code_of(x), tokens, row_stride(x), weight.data_ptr(), weight.stride(0), vocabulary, width, reduction,
                                                       smoothing, (const float*)kept.data_ptr(), (const float*)upstream.data_ptr(),
                                                       upstream.dim() ? upstream.stride(0) : 0, ptr(out[0]), ptr(out[1]), workspace.data_ptr(), size, stream_of(x)),
                  "fo_linear_cross_entropy_backward");
        }
        return once(std::move(out));
    }
};

PyObject* linear_cross_entropy(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6 || !api.bound || watched()) Py_RETURN_NONE;
    const Tensor *x = values_of(args[0]), *weight = values_of(args[1]), *target = tensor_of(args[2]);
    if (!x || !weight || !target) Py_RETURN_NONE;
    const int64_t ignore = PyLong_AsLongLong(args[3]), reduction = PyLong_AsLongLong(args[4]);
    const double smoothing = PyFloat_AsDouble(args[5]);
    if (PyErr_Occurred()) return nullptr;
    if (weight->dim() != 2 || weight->scalar_type() != x->scalar_type() || weight->device() != x->device() || target->device() != x->device() || !is_rows(*x) || !is_rows(*weight) ||
        (target->scalar_type() != at::kLong && target->scalar_type() != at::kInt) || !target->is_contiguous() ||
        target->sizes() != x->sizes().slice(0, x->dim() - 1) || weight->size(1) != x->size(-1) || x->numel() == 0 || weight->numel() == 0 || !(smoothing >= 0.0 && smoothing <= 1.0))
        Py_RETURN_NONE;
    const int64_t width = weight->size(1), vocabulary = weight->size(0), tokens = target->numel();
    Tensor loss, kept;
    {
        const c10::DeviceGuard guard(x->device());
        {
            at::NoGradGuard none;
            const auto numbers = x->options().dtype(at::kFloat);
            loss = reduction == FO_REDUCE_NONE ? at::empty(target->sizes(), numbers) : at::empty({}, numbers);
            // fp32 numbers and int32 labels.  Hooks on saved tensors may convert what is floating-point; these are bits.
            kept = at::empty({FO_LINEAR_CROSS_ENTROPY_KEPT(tokens)}, x->options().dtype(at::kInt));
            const int64_t size = api.fo_linear_cross_entropy_workspace(x->data_ptr(), code_of(*x), tokens, row_stride(*x), weight->data_ptr(), weight->stride(0), vocabulary, width,
                                                                       (float)smoothing);
            check_size(size, "fo_linear_cross_entropy");
            const Tensor workspace = bytes(size, *x);
            check(api.fo_linear_cross_entropy(x->data_ptr(), code_of(*x), tokens, row_stride(*x), weight->data_ptr(), weight->stride(0), vocabulary, width, target->data_ptr(),
                                              index_bytes(*target), ignore, (int)reduction, (float)smoothing, (float*)loss.data_ptr(), (float*)kept.data_ptr(), workspace.data_ptr(),
                                              size, stream_of(*x)),
                  "fo_linear_cross_entropy");
        }
        if (records({x, weight})) {
            auto node = std::shared_ptr<LossNode>(new LossNode(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(*x, *weight));
            node->x.keep(*x);
            node->weight.keep(*weight);
            node->kept.keep(kept);
            node->reduction = (int)reduction;
            node->smoothing = (float)smoothing;
            torch::autograd::set_history(loss, node);
        }
    }
    return THPVariable_Wrap(loss);
    END_HANDLE_TH_ERRORS
}

// The result's and the arguments' types, a letter each, as the struct module names them; P: a pointer.
template <class T> constexpr char kind_of() {
    if (std::is_pointer<T>::value) return 'P';
    if (std::is_same<T, float>::value) return 'f';
    if (std::is_same<T, double>::value) return 'd';
    return std::is_integral<T>::value && sizeof(T) == 8 ? 'q' : std::is_integral<T>::value && sizeof(T) == 4 ? 'i' : '?';
}
template <class R, class... A> std::string kinds_of(R (*)(A...)) { return {kind_of<R>(), kind_of<A>()...}; }

PyObject* all_kinds() {
    PyObject* kinds = PyDict_New();
#define FO_KINDS(name)                                                                              \
    {                                                                                               \
        PyObject* o = kinds ? PyUnicode_FromString(kinds_of(api.name).c_str()) : nullptr;           \
        if (!o || PyDict_SetItemString(kinds, #name, o) < 0) Py_CLEAR(kinds);                       \
        Py_XDECREF(o);                                                                              \
    }
    FO_ENTRIES(FO_KINDS)
#undef FO_KINDS
    PyObject* o = kinds ? PyUnicode_FromString(std::to_string(FO_LINEAR_CROSS_ENTROPY_KEPT(1)).c_str()) : nullptr;    // sizes that the two sides have to agree upon
    if (!o || PyDict_SetItemString(kinds, "FO_LINEAR_CROSS_ENTROPY_KEPT", o) < 0) Py_CLEAR(kinds);
    Py_XDECREF(o);
    return kinds;
}

PyObject* bind(PyObject*, PyObject* addresses) {
    if (!PyDict_Check(addresses)) return PyErr_Format(PyExc_TypeError, "bind takes a dict");
    if (api.bound) Py_RETURN_NONE;    // calls may be under way in other threads
#define FO_BIND(name)                                                                                         \
    {                                                                                                         \
        PyObject* o = PyDict_GetItemString(addresses, #name);                                                 \
        void* p = o ? PyLong_AsVoidPtr(o) : nullptr;                                                          \
        if (!p) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "no address of " #name);   \
        api.name = (decltype(api.name))p;                                                                     \
    }
    FO_ENTRIES(FO_BIND)
#undef FO_BIND
    api.bound = true;
    Py_RETURN_NONE;
}

#define FO_FAST(f) (PyCFunction)(void (*)(void)) f, METH_FASTCALL
PyMethodDef methods[] = {
    {"bind", bind, METH_O, "bind(addresses): the C entry points by name"},
    {"rms_norm", FO_FAST(rms_norm), "rms_norm(x, weight, residual, eps) -> None | y | (y, stream)"},
    {"rms_norm_mxfp4", FO_FAST(rms_norm_mxfp4), "rms_norm_mxfp4(x, weight, residual, eps) -> None | (codes, scales) | (codes, scales, stream)"},
    {"embedding", FO_FAST(embedding), "embedding(tokens, weight, scale, padding) -> None | y"},
    {"linear_cross_entropy", FO_FAST(linear_cross_entropy), "linear_cross_entropy(x, weight, target, ignore, reduction, smoothing) -> None | loss"},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fo_autograd", "calls and autograd nodes of the norm, the embedding and the loss", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fo_autograd(void) {
    PyObject *m = PyModule_Create(&module), *kinds = m ? all_kinds() : nullptr;
    if (kinds && PyModule_AddObject(m, "kinds", kinds) == 0) return m;
    Py_XDECREF(kinds);
    Py_XDECREF(m);
    return nullptr;
}
