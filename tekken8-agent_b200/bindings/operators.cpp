// The Python side of the operators: one call from tensors to the C entries of t8b.h. It checks
// the tensors, allocates the outputs and the workspace on torch's current stream, and queues the
// work there; t8b/ops.py documents each function and names its arguments. ctypes takes about as long
// for the twenty arguments of an entry as everything here.
//
// The module is bound to the library at run time (bind() takes the entries' addresses from the
// handle that t8b/_lib.py loaded), so there is one copy of the library whichever file it is.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstring>
#include <stdexcept>
#include <string>

#include "t8b.h"

namespace {

using at::Tensor;

struct Entries {
    decltype(&t8b_last_error) last_error;
    decltype(&t8b_layer_norm_forward) layer_norm_forward;
    decltype(&t8b_layer_norm_workspace) layer_norm_workspace;
    decltype(&t8b_layer_norm_backward) layer_norm_backward;
    decltype(&t8b_linear_workspace) linear_workspace;
    decltype(&t8b_linear_forward) linear_forward;
    decltype(&t8b_linear_backward) linear_backward;
    decltype(&t8b_gated_workspace) gated_workspace;
    decltype(&t8b_gated_forward) gated_forward;
    decltype(&t8b_gated_backward) gated_backward;
    decltype(&t8b_causal_conv_forward) causal_conv_forward;
    decltype(&t8b_causal_conv_workspace) causal_conv_workspace;
    decltype(&t8b_causal_conv_backward) causal_conv_backward;
    decltype(&t8b_causal_conv_step) causal_conv_step;
    decltype(&t8b_selective_scan_saved) selective_scan_saved;
    decltype(&t8b_selective_scan_workspace) selective_scan_workspace;
    decltype(&t8b_selective_scan_forward) selective_scan_forward;
    decltype(&t8b_selective_scan_backward) selective_scan_backward;
    decltype(&t8b_selective_scan_step) selective_scan_step;
    decltype(&t8b_policy_loss) policy_loss;
} entry{};
PyObject* library_error = nullptr;  // T8bError(status, message)
PyObject* memory_error = nullptr;   // torch.OutOfMemoryError

struct Refused : std::invalid_argument {
    using std::invalid_argument::invalid_argument;
};
struct Failed {
    int status;
};
struct Raised {};  // a Python exception that is set already
[[noreturn]] void refuse(const std::string& why) { throw Refused(why); }

std::string text(at::IntArrayRef shape) {
    std::string s = "(";
    for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
    return s + ")";
}

int type_of(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kFloat: return T8B_F32;
        case at::kBFloat16: return T8B_BF16;
        case at::kHalf: return T8B_F16;
        default: refuse(std::string(name) + " is " + c10::toString(t.scalar_type()) + ": fp32, bf16 or f16 is expected");
    }
}
at::ScalarType scalar(int type) { return type == T8B_F32 ? at::kFloat : type == T8B_BF16 ? at::kBFloat16 : at::kHalf; }

// A tensor of rows of `columns` elements, its leading axes a common row stride apart.
struct Rows {
    void* data = nullptr;
    int64_t rows = 0, stride = 0;
};
Rows rows_of(const Tensor& t, const char* name, int64_t columns, int device) {
    if (t.layout() != at::kStrided) refuse(std::string(name) + " must be a dense tensor");
    if (t.get_device() != device || !t.is_cuda()) refuse(std::string(name) + " is on another device");
    const auto shape = t.sizes();
    if (shape.empty() || shape.back() != columns) {
        refuse(std::string(name) + " has shape " + text(shape) + ", expected rows of " + std::to_string(columns));
    }
    const auto strides = t.strides();
    if (strides.back() != 1 && columns > 1) refuse(std::string(name) + ": the last axis must be contiguous");
    Rows r;
    r.data = t.data_ptr();
    r.rows = 1;
    r.stride = columns;
    bool first = true;
    for (int64_t i = static_cast<int64_t>(shape.size()) - 2; i >= 0; --i) {
        if (shape[i] == 1) continue;
        if (first) {
            r.stride = strides[i];
            first = false;
        } else if (shape[i] != 0 && r.rows != 0 && strides[i] != r.stride * r.rows) {
            refuse(std::string(name) + ": its leading axes have no common row stride");
        }
        r.rows *= shape[i];
    }
    if (r.rows <= 1) r.stride = columns;  // a stride that addresses nothing may be anything
    return r;
}

void* vector_of(const Tensor& t, const char* name, int64_t count, int device, int type) {
    if (!t.defined()) return nullptr;
    if (t.get_device() != device || !t.is_cuda()) refuse(std::string(name) + " is on another device");
    if (type_of(t, name) != type) refuse(std::string(name) + " is " + c10::toString(t.scalar_type()) + ", expected " + c10::toString(scalar(type)));
    if (t.dim() != 1 || t.size(0) != count || !t.is_contiguous()) {
        refuse(std::string(name) + " must be a contiguous vector of " + std::to_string(count));
    }
    return t.data_ptr();
}

// x's shape with another last axis.
struct Shape {
    c10::SmallVector<int64_t, 5> sizes;
    Shape(const Tensor& x, int64_t columns) : sizes(x.sizes().begin(), x.sizes().end()) { sizes.back() = columns; }
    operator at::IntArrayRef() const { return sizes; }
};
Tensor make(const Tensor& like, at::IntArrayRef shape, int type) { return at::empty(shape, like.options().dtype(scalar(type))); }
Tensor make_bytes(const Tensor& like, size_t bytes) {
    return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}
void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

void done(int status) {
    if (status == T8B_OK) return;
    if (status == T8B_EINVAL) refuse(entry.last_error());
    throw Failed{status};
}

// The call's device, current for its duration, and torch's stream there.
struct On {
    int device;
    c10::cuda::CUDAGuard guard;
    explicit On(const Tensor& t) : device(cuda_index(t)), guard(static_cast<c10::DeviceIndex>(device)) {}
    static int cuda_index(const Tensor& t) {
        if (!t.is_cuda()) refuse("expected CUDA tensors");
        return t.get_device();
    }
    void* stream() const { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream(); }
};

// ------------------------------------------------------------------ arguments
constexpr Py_ssize_t kMost = 15;
struct Arguments {
    PyObject* const* at;
    Arguments(PyObject* const* args, Py_ssize_t given, Py_ssize_t expected) : at(args) {
        if (given != expected || given > kMost) refuse("wrong number of arguments");
        if (entry.last_error == nullptr) refuse("the module is not bound to the library");
    }
    Tensor tensor(int i, const char* name) const {
        if (!THPVariable_Check(at[i])) refuse(std::string(name) + " must be a tensor");
        return THPVariable_Unpack(at[i]);
    }
    Tensor optional(int i, const char* name) const { return at[i] == Py_None ? Tensor() : tensor(i, name); }
    double number(int i) const {
        const double v = PyFloat_AsDouble(at[i]);
        if (v == -1.0 && PyErr_Occurred()) throw Raised();
        return v;
    }
    bool flag(int i) const {
        const int truth = PyObject_IsTrue(at[i]);
        if (truth < 0) throw Raised();
        return truth == 1;
    }
    // a torch.dtype as a T8B type; None: `missing`
    int type(int i, int missing) const {
        if (at[i] == Py_None) return missing;
        if (!THPDtype_Check(at[i])) refuse("out_dtype must be a torch.dtype");
        switch (reinterpret_cast<THPDtype*>(at[i])->scalar_type) {
            case at::kFloat: return T8B_F32;
            case at::kBFloat16: return T8B_BF16;
            case at::kHalf: return T8B_F16;
            default: refuse("out_dtype must be fp32, bf16 or f16");
        }
    }
    int activation(int i) const {
        const char* name = PyUnicode_Check(at[i]) ? PyUnicode_AsUTF8(at[i]) : "";
        const std::string s = name ? name : "";
        if (s == "none") return T8B_LINEAR;
        if (s == "relu") return T8B_RELU;
        if (s == "gelu") return T8B_GELU;
        if (s == "silu") return T8B_SILU;
        if (s == "tanh") return T8B_TANH;
        refuse("activation '" + s + "': one of none, relu, gelu, silu, tanh");
    }
};

PyObject* wrap(const Tensor& t) {
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}
template <typename... T>
PyObject* wrap_all(const T&... t) {
    PyObject* tuple = PyTuple_New(sizeof...(T));
    if (tuple == nullptr) return nullptr;
    Py_ssize_t i = 0;
    bool ok = true;
    for (PyObject* each : {wrap(t)...}) {
        ok = ok && each != nullptr;
        PyTuple_SET_ITEM(tuple, i++, each);
    }
    if (ok) return tuple;
    Py_DECREF(tuple);
    return nullptr;
}

// No exception leaves a function of the module but as a Python one.
template <typename Body>
PyObject* answer(Body&& body) {
    try {
        return body();
    } catch (const Refused& error) {
        PyErr_SetString(PyExc_ValueError, error.what());
    } catch (const Raised&) {
    } catch (const Failed& error) {
        PyObject* args = Py_BuildValue("(is)", error.status, entry.last_error());
        if (args != nullptr) {
            PyErr_SetObject(library_error ? library_error : PyExc_RuntimeError, args);
            Py_DECREF(args);
        }
    } catch (const c10::OutOfMemoryError& error) {
        PyErr_SetString(memory_error ? memory_error : PyExc_MemoryError, error.what_without_backtrace());
    } catch (const c10::Error& error) {
        PyErr_SetString(PyExc_RuntimeError, error.what_without_backtrace());
    } catch (const std::exception& error) {
        PyErr_SetString(PyExc_RuntimeError, error.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown failure");
    }
    return nullptr;
}

// ------------------------------------------------------------------ layer norm
int parameter_type(const Tensor& weight, const Tensor& bias) {
    if (weight.defined()) return type_of(weight, "weight");
    return bias.defined() ? type_of(bias, "bias") : T8B_F32;
}

// x, weight, bias, eps, out_dtype, save
PyObject* layer_norm(PyObject*, PyObject* const* args, Py_ssize_t given) {
    return answer([&]() -> PyObject* {
        const Arguments a(args, given, 6);
        const Tensor x = a.tensor(0, "x"), weight = a.optional(1, "weight"), bias = a.optional(2, "bias");
        const double eps = PyFloat_AsDouble(args[3]);
        if (eps == -1.0 && PyErr_Occurred()) throw Raised();
        const On on(x);
        const int x_type = type_of(x, "x"), y_type = a.type(4, x_type);
        const int64_t n = x.dim() ? x.size(-1) : 0;
        const Rows in = rows_of(x, "x", n, on.device);
        const int p = parameter_type(weight, bias);
        void *pw = vector_of(weight, "weight", n, on.device, p), *pb = vector_of(bias, "bias", n, on.device, p);
        const bool save = a.flag(5);
        const Tensor y = make(x, x.sizes(), y_type);
        Tensor mean, rstd;
        if (save) {
            mean = make(x, x.sizes().slice(0, x.dim() - 1), T8B_F32);
            rstd = make(x, x.sizes().slice(0, x.dim() - 1), T8B_F32);
        }
        done(entry.layer_norm_forward(in.data, x_type, in.stride, pw, pb, p, static_cast<float>(eps), in.rows, n, y.data_ptr(),
                                      y_type, n, static_cast<float*>(pointer(mean)), static_cast<float*>(pointer(rstd)), on.stream()));
        return save ? wrap_all(y, mean, rstd) : wrap(y);
    });
}

// dy, x, weight, bias, mean, rstd, residual_gradient
PyObject* layer_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t given) {
    return answer([&]() -> PyObject* {
        const Arguments a(args, given, 7);
        const Tensor dy = a.tensor(0, "dy"), x = a.tensor(1, "x"), weight = a.optional(2, "weight"), bias = a.optional(3, "bias");
        const Tensor mean = a.tensor(4, "mean"), rstd = a.tensor(5, "rstd"), residual = a.optional(6, "residual_gradient");
        const On on(x);
        const int x_type = type_of(x, "x"), y_type = type_of(dy, "dy");
        const int64_t n = x.dim() ? x.size(-1) : 0;
        const Rows in = rows_of(x, "x", n, on.device);
        if (dy.sizes() != x.sizes()) refuse("dy has shape " + text(dy.sizes()) + ", x " + text(x.sizes()));
        const Rows d = rows_of(dy, "dy", n, on.device);
        Rows r;
        if (residual.defined()) {
            if (residual.sizes() != x.sizes()) refuse("residual_gradient has shape " + text(residual.sizes()) + ", x " + text(x.sizes()));
            if (residual.scalar_type() != x.scalar_type()) refuse("residual_gradient must have x's type");
            r = rows_of(residual, "residual_gradient", n, on.device);
        }
        const int p = parameter_type(weight, bias);
        void* pw = vector_of(weight, "weight", n, on.device, p);
        vector_of(bias, "bias", n, on.device, p);
        for (const Tensor* t : {&mean, &rstd}) {
            if (t->numel() != in.rows || !t->is_contiguous() || t->scalar_type() != at::kFloat || !t->is_cuda() || t->get_device() != on.device) {
                refuse("mean and rstd must be contiguous fp32 tensors with one value a row");
            }
        }
        const Tensor dx = make(x, x.sizes(), x_type);
        Tensor dweight, dbias, workspace;
        if (weight.defined()) dweight = make(x, {n}, p);
        if (bias.defined()) dbias = make(x, {n}, p);
        const size_t size = weight.defined() || bias.defined() ? entry.layer_norm_workspace(in.rows, n) : 0;
        if (size) workspace = make_bytes(x, size);
        done(entry.layer_norm_backward(d.data, y_type, d.stride, in.data, x_type, in.stride, pw, p, mean.data_ptr<float>(),
                                       rstd.data_ptr<float>(), r.data, r.stride, in.rows, n, dx.data_ptr(), n, pointer(dweight),
                                       pointer(dbias), pointer(workspace), size, on.stream()));
        return wrap_all(dx, dweight, dbias);
    });
}

// ------------------------------------------------------------------ linear and gated
// What both directions of both operators check alike. parts: 1 linear, 2 gated.
struct Operands {
    const On on;
    int type;
    int64_t columns, in, out;
    Rows x, weight;
    Operands(const Tensor& tx, const Tensor& tw, int parts) : on(tx), type(type_of(tx, "x")) {
        if (type == T8B_F32) refuse("x is Float: matrix operands are bf16 or f16");
        if (tw.dim() != 2 || tw.size(0) % parts != 0) {
            refuse("weight has shape " + text(tw.sizes()) + ", expected [" + (parts == 2 ? "2 out" : "out") + "][in]");
        }
        if (tw.scalar_type() != tx.scalar_type()) refuse("weight must have x's type");
        columns = tw.size(0);
        in = tw.size(1);
        out = columns / parts;
        x = rows_of(tx, "x", in, on.device);
        weight = rows_of(tw, "weight", in, on.device);
    }
    int bias_type(const Tensor& bias) const {
        if (!bias.defined()) return T8B_F32;
        const int t = type_of(bias, "bias");
        if (t != T8B_F32 && t != type) refuse("bias must be fp32 or of x's type");
        vector_of(bias, "bias", columns, on.device, t);
        return t;
    }
    // the operands whose rows do not suit TMA, as the library's own rule has it
    static bool off(const Rows& r) {
        return (reinterpret_cast<uintptr_t>(r.data) & 15) != 0 || (r.rows > 1 && ((r.stride & 7) != 0 || r.stride >= (1ll << 39)));
    }
    int packed(bool of_x, bool of_weight) const {
        return (of_x && off(x) ? T8B_WORKSPACE_X : 0) | (of_weight && off(weight) ? T8B_WORKSPACE_WEIGHT : 0);
    }
    size_t room(decltype(&t8b_linear_workspace) query, int what) const { return what ? query(x.rows, in, out, what) : 0; }
};

// x, weight, bias, activation, residual, out_dtype, save
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t given) {
    return answer([&]() -> PyObject* {
        const Arguments a(args, given, 7);
        const Tensor x = a.tensor(0, "x"), weight = a.tensor(1, "weight"), bias = a.optional(2, "bias");
        const Tensor residual = a.optional(4, "residual");
        const int act = a.activation(3);
        const Operands o(x, weight, 1);
        const int y_type = a.type(5, o.type), b_type = o.bias_type(bias);
        if (y_type != o.type && y_type != T8B_F32) refuse("out_dtype: fp32 or x's type");
        const Shape shape(x, o.out);
        Rows r;
        if (residual.defined()) {
            if (residual.sizes() != at::IntArrayRef(shape)) refuse("residual has shape " + text(residual.sizes()) + ", expected " + text(shape));
            if (type_of(residual, "residual") != y_type) refuse("residual must have the output's type");
            r = rows_of(residual, "residual", o.out, o.on.device);
        }
        const bool save = a.flag(6);
        const Tensor y = make(x, shape, y_type);
        Tensor pre, workspace;
        if (save) pre = make(x, shape, o.type);
        const size_t size = o.room(entry.linear_workspace, o.packed(true, true));
        if (size) workspace = make_bytes(x, size);
        done(entry.linear_forward(o.type, o.x.data, o.x.stride, o.weight.data, o.weight.stride, pointer(bias), b_type, act, r.data,
                                  r.stride, o.x.rows, o.in, o.out, y.data_ptr(), y_type, o.out, pointer(pre), o.out,
                                  pointer(workspace), size, o.on.stream()));
        return save ? wrap_all(y, pre) : wrap(y);
    });
}

// x, weight, bias, activation, save
PyObject* gated(PyObject*, PyObject* const* args, Py_ssize_t given) {
    return answer([&]() -> PyObject* {
        const Arguments a(args, given, 5);
        const Tensor x = a.tensor(0, "x"), weight = a.tensor(1, "weight"), bias = a.optional(2, "bias");
        const int act = a.activation(3);
        const Operands o(x, weight, 2);
        const int b_type = o.bias_type(bias);
        const bool save = a.flag(4);
        const Tensor h = make(x, Shape(x, o.out), o.type);
        Tensor pre, workspace;
        if (save) pre = make(x, Shape(x, o.columns), o.type);
        const size_t size = o.room(entry.gated_workspace, o.packed(true, true));
        if (size) workspace = make_bytes(x, size);
        done(entry.gated_forward(o.type, o.x.data, o.x.stride, o.weight.data, o.weight.stride, pointer(bias), b_type, act, o.x.rows,
                                 o.in, o.out, h.data_ptr(), o.out, pointer(pre), o.columns, pointer(workspace), size, o.on.stream()));
        return save ? wrap_all(h, pre) : wrap(h);
    });
}

// dy, x, weight, bias, pre, activation, input_gradient
template <int PARTS>
PyObject* backward(PyObject*, PyObject* const* args, Py_ssize_t given) {
    return answer([&]() -> PyObject* {
        const Arguments a(args, given, 7);
        const Tensor dy = a.tensor(0, "the output's gradient"), x = a.tensor(1, "x"), weight = a.tensor(2, "weight");
        const Tensor bias = a.optional(3, "bias"), pre = a.optional(4, "pre");
        const int act = a.activation(5);
        const Operands o(x, weight, PARTS);
        const int b_type = o.bias_type(bias);
        if (dy.sizes() != at::IntArrayRef(Shape(x, o.out))) {
            refuse("the output's gradient has shape " + text(dy.sizes()) + ", expected " + text(Shape(x, o.out)));
        }
        if (dy.scalar_type() != x.scalar_type()) refuse("the output's gradient must have x's type");
        const Rows d = rows_of(dy, "the output's gradient", o.out, o.on.device);
        Rows z;
        if (PARTS == 2 || act != T8B_LINEAR) {
            if (!pre.defined()) refuse("pre (what the forward pass's `save` gave) is needed");
            if (pre.sizes() != at::IntArrayRef(Shape(x, o.columns))) {
                refuse("pre has shape " + text(pre.sizes()) + ", expected " + text(Shape(x, o.columns)));
            }
            if (pre.scalar_type() != x.scalar_type()) refuse("pre must have x's type");
            z = rows_of(pre, "pre", o.columns, o.on.device);
        }
        Tensor dx, dbias, workspace;
        if (a.flag(6)) dx = make(x, x.sizes(), o.type);
        const Tensor dweight = make(x, {o.columns, o.in}, o.type);
        if (bias.defined()) dbias = make(x, {o.columns}, b_type);
        int what = T8B_WORKSPACE_BACKWARD | o.packed(true, dx.defined());
        if (PARTS == 2 || act != T8B_LINEAR || Operands::off(d)) what |= T8B_WORKSPACE_DZ;
        const size_t size = o.room(PARTS == 2 ? entry.gated_workspace : entry.linear_workspace, what);
        if (size) workspace = make_bytes(x, size);
        done((PARTS == 2 ? entry.gated_backward : entry.linear_backward)(
            o.type, d.data, d.stride, o.x.data, o.x.stride, o.weight.data, o.weight.stride, z.data, z.stride, b_type, act, o.x.rows,
            o.in, o.out, pointer(dx), o.in, dweight.data_ptr(), o.in, pointer(dbias), pointer(workspace), size, o.on.stream()));
        return wrap_all(dx, dweight, dbias);
    });
}

// ------------------------------------------------------------------ sequences
// What the sequence operators share: [sequences][steps][...] tensors of any strides with a contiguous last axis
// (single steps: [sequences][...]), resets and lengths.
struct Tracks {
    const On on;
    const bool step;
    int type;
    t8b_sequences_t q{};
    bool by_step = false;  // whether x lies [step][sequence]: outputs do too
    Tracks(const Tensor& x, const char* name, bool step_) : on(x), step(step_), type(type_of(x, name)) {
        if (x.dim() != (step ? 2 : 3)) {
            refuse(std::string(name) + " has shape " + text(x.sizes()) + ", expected " + (step ? "[sequences][channels]" : "[sequences][steps][channels]"));
        }
        q.sequences = x.size(0);
        q.steps = step ? 1 : x.size(1);
        q.channels = x.size(-1);
        by_step = !step && q.sequences > 1 && q.steps > 1 && x.stride(0) < x.stride(1);
    }
    void place(const Tensor& t, const char* name) const {
        if (t.layout() != at::kStrided) refuse(std::string(name) + " must be a dense tensor");
        if (!t.is_cuda() || t.get_device() != on.device) refuse(std::string(name) + " is on another device");
    }
    void expect(const Tensor& t, const char* name, at::IntArrayRef shape, at::ScalarType scalar_type) const {
        place(t, name);
        if (t.sizes() != shape) refuse(std::string(name) + " has shape " + text(t.sizes()) + ", expected " + text(shape));
        if (t.scalar_type() != scalar_type) refuse(std::string(name) + " is " + c10::toString(t.scalar_type()) + ", expected " + c10::toString(scalar_type));
    }
    void* packed(const Tensor& t, const char* name, at::IntArrayRef shape, int element) const {
        if (!t.defined()) return nullptr;
        expect(t, name, shape, scalar(element));
        if (!t.is_contiguous()) refuse(std::string(name) + " must be contiguous");
        return t.data_ptr();
    }
    // a tensor of x's type and first axes
    t8b_track_t track(const Tensor& t, const char* name, int64_t width) const {
        if (!t.defined()) return {};
        if (step) {
            expect(t, name, {q.sequences, width}, scalar(type));
        } else {
            expect(t, name, {q.sequences, q.steps, width}, scalar(type));
        }
        if (width > 1 && t.stride(-1) != 1) refuse(std::string(name) + ": the last axis must be contiguous");
        return {t.data_ptr(), t.stride(0), step ? 0 : t.stride(1)};
    }
    void rounds(const Tensor& reset, const Tensor& lengths) {
        if (reset.defined()) {
            place(reset, "reset");
            const bool fits = step ? reset.dim() == 1 && reset.size(0) == q.sequences
                                   : reset.dim() == 2 && reset.size(0) == q.sequences && reset.size(1) == q.steps;
            if (!fits) refuse("reset has shape " + text(reset.sizes()) + ", expected " + (step ? "[sequences]" : "[sequences][steps]"));
            if (reset.scalar_type() != at::kBool && reset.scalar_type() != at::kByte) refuse("reset must be bool or uint8");
            q.reset = static_cast<const uint8_t*>(reset.data_ptr());
            q.reset_sequence = reset.stride(0);
            q.reset_step = step ? 0 : reset.stride(1);
        }
        if (lengths.defined()) {
            expect(lengths, "lengths", {q.sequences}, at::kInt);
            if (!lengths.is_contiguous()) refuse("lengths must be contiguous");
            q.lengths = lengths.data_ptr<int32_t>();
        }
    }
    // an output [sequences][steps][width...], in the order of x
    Tensor output(const Tensor& like, int64_t groups, int64_t width, bool grouped) const {
        const auto options = like.options().dtype(scalar(type));
        const int64_t row = groups * width;
        if (step) return at::empty({q.sequences, row}, options);
        const int64_t s = by_step ? row : q.steps * row, t = by_step ? q.sequences * row : row;
        if (grouped) return at::empty_strided({q.sequences, q.steps, groups, width}, {s, t, width, 1}, options);
        return at::empty_strided({q.sequences, q.steps, row}, {s, t, 1}, options);
    }
    t8b_track_t fresh(const Tensor& t) const { return t.defined() ? t8b_track_t{t.data_ptr(), t.stride(0), step ? 0 : t.stride(1)} : t8b_track_t{}; }
};

// ------------------------------------------------------------------ causal convolution
struct Filter {
    int width = 0, type = T8B_F32;
    void *weight = nullptr, *bias = nullptr;
    Filter(const Tracks& k, const Tensor& tw, const Tensor& tb) {
        type = type_of(tw, "weight");
        if (type != T8B_F32 && type != k.type) refuse("weight must be fp32 or of x's type");
        if (tw.dim() != 2) refuse("weight has shape " + text(tw.sizes()) + ", expected [channels][width]");
        width = static_cast<int>(std::min<int64_t>(tw.size(1), 1 << 20));
        weight = k.packed(tw, "weight", {k.q.channels, tw.size(1)}, type);
        bias = k.packed(tb, "bias", {k.q.channels}, type);
    }
};

// x, weight, bias, activation, state, reset, lengths, final
PyObject* causal_conv(PyObject*, PyObject* const* args, Py_ssize_t given) {
    return answer([&]() -> PyObject* {
        const Arguments a(args, given, 8);
        const Tensor x = a.tensor(0, "x"), weight = a.tensor(1, "weight"), bias = a.optional(2, "bias"), state = a.optional(4, "state");
        const Tensor reset = a.optional(5, "reset"), lengths = a.optional(6, "lengths");
        const int act = a.activation(3);
        Tracks k(x, "x", false);
        const t8b_track_t in = k.track(x, "x", k.q.channels);
        k.rounds(reset, lengths);
        const Filter f(k, weight, bias);
        const void* ps = k.packed(state, "state", {k.q.sequences, f.width - 1, k.q.channels}, k.type);
        const bool last = a.flag(7);
        if (f.width < 2 || f.width > 4) refuse("weight has shape " + text(weight.sizes()) + ": a width of 2 to 4");
        const Tensor y = k.output(x, 1, k.q.channels, false);
        Tensor end;
        if (last) end = make(x, {k.q.sequences, f.width - 1, k.q.channels}, k.type);
        done(entry.causal_conv_forward(&k.q, k.type, in, f.weight, f.bias, f.type, f.width, act, ps, k.fresh(y), pointer(end), k.on.stream()));
        return last ? wrap_all(y, end) : wrap(y);
    });
}

// dy, x, weight, bias, activation, state, reset, lengths, dfinal
PyObject* causal_conv_backward(PyObject*, PyObject* const* args, Py_ssize_t given) {
    return answer([&]() -> PyObject* {
        const Arguments a(args, given, 9);
        const Tensor dy = a.tensor(0, "dy"), x = a.tensor(1, "x"), weight = a.tensor(2, "weight"), bias = a.optional(3, "bias");
        const Tensor state = a.optional(5, "state"), reset = a.optional(6, "reset"), lengths = a.optional(7, "lengths"), dfinal = a.optional(8, "dfinal");
        const int act = a.activation(4);
        Tracks k(x, "x", false);
        const t8b_track_t in = k.track(x, "x", k.q.channels), d = k.track(dy, "dy", k.q.channels);
        k.rounds(reset, lengths);
        const Filter f(k, weight, bias);
        if (f.width < 2 || f.width > 4) refuse("weight has shape " + text(weight.sizes()) + ": a width of 2 to 4");
        const void* ps = k.packed(state, "state", {k.q.sequences, f.width - 1, k.q.channels}, k.type);
        const void* pf = k.packed(dfinal, "dfinal", {k.q.sequences, f.width - 1, k.q.channels}, k.type);
        const Tensor dx = k.output(x, 1, k.q.channels, false), dweight = make(x, weight.sizes(), f.type);
        Tensor dbias, dstate;
        if (bias.defined()) dbias = make(x, {k.q.channels}, f.type);
        if (state.defined()) dstate = make(x, state.sizes(), k.type);
        const size_t size = entry.causal_conv_workspace(&k.q, f.width);
        const Tensor workspace = make_bytes(x, size);
        done(entry.causal_conv_backward(&k.q, k.type, d, in, f.weight, f.bias, f.type, f.width, act, ps, pf, k.fresh(dx), dweight.data_ptr(),
                                        pointer(dbias), pointer(dstate), workspace.data_ptr(), size, k.on.stream()));
        return wrap_all(dx, dweight, dbias, dstate);
    });
}

// x, weight, bias, state, activation, reset
PyObject* causal_conv_step(PyObject*, PyObject* const* args, Py_ssize_t given) {
    return answer([&]() -> PyObject* {
        const Arguments a(args, given, 6);
        const Tensor x = a.tensor(0, "x"), weight = a.tensor(1, "weight"), bias = a.optional(2, "bias"), state = a.tensor(3, "state");
        const Tensor reset = a.optional(5, "reset");
        const int act = a.activation(4);
        Tracks k(x, "x", true);
        const t8b_track_t in = k.track(x, "x", k.q.channels);
        k.rounds(reset, Tensor());
        const Filter f(k, weight, bias);
        if (f.width < 2 || f.width > 4) refuse("weight has shape " + text(weight.sizes()) + ": a width of 2 to 4");
        void* ps = k.packed(state, "state", {k.q.sequences, f.width - 1, k.q.channels}, k.type);
        const Tensor y = k.output(x, 1, k.q.channels, false);
        done(entry.causal_conv_step(&k.q, k.type, in, f.weight, f.bias, f.type, f.width, act, ps, k.fresh(y), k.on.stream()));
        return wrap(y);
    });
}

// ------------------------------------------------------------------ selective scan
struct Scanned {
    t8b_scan_t scan{};
    bool grouped = false;  // b and c have an axis of groups
    Scanned(const Tracks& k, const Tensor& u, const Tensor& delta, const Tensor& a, const Tensor& b, const Tensor& c, const Tensor& d,
            const Tensor& z, const Tensor& delta_bias, bool softplus) {
        scan.type = k.type;
        scan.softplus = softplus;
        scan.u = k.track(u, "u", k.q.channels);
        scan.delta = k.track(delta, "delta", k.q.channels);
        scan.z = k.track(z, "z", k.q.channels);
        if (a.dim() != 2) refuse("a has shape " + text(a.sizes()) + ", expected [channels][states]");
        scan.states = a.size(1);
        if (scan.states < 1 || scan.states > 64) refuse("a has shape " + text(a.sizes()) + ": 1 to 64 states");
        scan.a = static_cast<const float*>(k.packed(a, "a", {k.q.channels, scan.states}, T8B_F32));
        scan.d = static_cast<const float*>(k.packed(d, "d", {k.q.channels}, T8B_F32));
        scan.delta_bias = static_cast<const float*>(k.packed(delta_bias, "delta_bias", {k.q.channels}, T8B_F32));
        const int plain = k.step ? 2 : 3;
        grouped = b.dim() == plain + 1;
        scan.groups = grouped ? b.size(plain - 1) : 1;
        if (scan.groups < 1 || k.q.channels % scan.groups != 0) refuse("b has shape " + text(b.sizes()) + ": its groups must divide the channels");
        scan.b = shared(k, b, "b", scan.b_group);
        scan.c = shared(k, c, "c", scan.c_group);
    }
    t8b_track_t shared(const Tracks& k, const Tensor& t, const char* name, int64_t& group) const {
        group = scan.states;
        if (!grouped) return k.track(t, name, scan.states);
        if (k.step) {
            k.expect(t, name, {k.q.sequences, scan.groups, scan.states}, scalar(k.type));
        } else {
            k.expect(t, name, {k.q.sequences, k.q.steps, scan.groups, scan.states}, scalar(k.type));
        }
        if (scan.states > 1 && t.stride(-1) != 1) refuse(std::string(name) + ": the last axis must be contiguous");
        if (scan.groups > 1) group = t.stride(-2);
        return {t.data_ptr(), t.stride(0), k.step ? 0 : t.stride(1)};
    }
};

// u, delta, a, b, c, d, z, delta_bias, softplus, state, reset, lengths, final, save
PyObject* selective_scan(PyObject*, PyObject* const* args, Py_ssize_t given) {
    return answer([&]() -> PyObject* {
        const Arguments a(args, given, 14);
        const Tensor u = a.tensor(0, "u"), delta = a.tensor(1, "delta"), ta = a.tensor(2, "a"), b = a.tensor(3, "b"), c = a.tensor(4, "c");
        const Tensor d = a.optional(5, "d"), z = a.optional(6, "z"), delta_bias = a.optional(7, "delta_bias"), state = a.optional(9, "state");
        const Tensor reset = a.optional(10, "reset"), lengths = a.optional(11, "lengths");
        Tracks k(u, "u", false);
        k.rounds(reset, lengths);
        Scanned s(k, u, delta, ta, b, c, d, z, delta_bias, a.flag(8));
        s.scan.state = static_cast<const float*>(k.packed(state, "state", {k.q.sequences, k.q.channels, s.scan.states}, T8B_F32));
        const bool last = a.flag(12), save = a.flag(13);
        const Tensor y = k.output(u, 1, k.q.channels, false);
        Tensor end, saved, workspace;
        if (last) end = make(u, {k.q.sequences, k.q.channels, s.scan.states}, T8B_F32);
        if (save) saved = make(u, {static_cast<int64_t>(entry.selective_scan_saved(&k.q, s.scan.groups, s.scan.states))}, T8B_F32);
        const size_t size = entry.selective_scan_workspace(&k.q, s.scan.groups, s.scan.states, 0);
        if (size) workspace = make_bytes(u, size);
        done(entry.selective_scan_forward(&k.q, &s.scan, k.fresh(y), static_cast<float*>(pointer(end)), static_cast<float*>(pointer(saved)),
                                          pointer(workspace), size, k.on.stream()));
        return last ? (save ? wrap_all(y, end, saved) : wrap_all(y, end)) : save ? wrap_all(y, saved) : wrap(y);
    });
}

// dy, u, delta, a, b, c, saved, d, z, delta_bias, softplus, state, reset, lengths, dfinal
PyObject* selective_scan_backward(PyObject*, PyObject* const* args, Py_ssize_t given) {
    return answer([&]() -> PyObject* {
        const Arguments a(args, given, 15);
        const Tensor dy = a.tensor(0, "dy"), u = a.tensor(1, "u"), delta = a.tensor(2, "delta"), ta = a.tensor(3, "a"), b = a.tensor(4, "b");
        const Tensor c = a.tensor(5, "c"), saved = a.tensor(6, "saved"), d = a.optional(7, "d"), z = a.optional(8, "z");
        const Tensor delta_bias = a.optional(9, "delta_bias"), state = a.optional(11, "state"), reset = a.optional(12, "reset");
        const Tensor lengths = a.optional(13, "lengths"), dfinal = a.optional(14, "dfinal");
        Tracks k(u, "u", false);
        k.rounds(reset, lengths);
        Scanned s(k, u, delta, ta, b, c, d, z, delta_bias, a.flag(10));
        const int64_t states = s.scan.states;
        s.scan.state = static_cast<const float*>(k.packed(state, "state", {k.q.sequences, k.q.channels, states}, T8B_F32));
        const void* pf = k.packed(dfinal, "dfinal", {k.q.sequences, k.q.channels, states}, T8B_F32);
        const void* ps = k.packed(saved, "saved", {static_cast<int64_t>(entry.selective_scan_saved(&k.q, s.scan.groups, states))}, T8B_F32);
        const t8b_track_t given_dy = k.track(dy, "dy", k.q.channels);
        const Tensor du = k.output(u, 1, k.q.channels, false), ddelta = k.output(u, 1, k.q.channels, false);
        const Tensor db = k.output(u, s.scan.groups, states, s.grouped), dc = k.output(u, s.scan.groups, states, s.grouped);
        const Tensor da = make(u, {k.q.channels, states}, T8B_F32);
        Tensor dz, dd, dbias, dstate;
        if (z.defined()) dz = k.output(u, 1, k.q.channels, false);
        if (d.defined()) dd = make(u, {k.q.channels}, T8B_F32);
        if (delta_bias.defined()) dbias = make(u, {k.q.channels}, T8B_F32);
        if (state.defined()) dstate = make(u, state.sizes(), T8B_F32);
        t8b_scan_gradients_t g{};
        g.du = k.fresh(du);
        g.ddelta = k.fresh(ddelta);
        g.dz = k.fresh(dz);
        g.db = k.fresh(db);
        g.dc = k.fresh(dc);
        g.db_group = g.dc_group = states;
        g.da = da.data_ptr<float>();
        g.dd = static_cast<float*>(pointer(dd));
        g.ddelta_bias = static_cast<float*>(pointer(dbias));
        g.dstate = static_cast<float*>(pointer(dstate));
        const size_t size = entry.selective_scan_workspace(&k.q, s.scan.groups, states, 1);
        const Tensor workspace = make_bytes(u, size);
        done(entry.selective_scan_backward(&k.q, &s.scan, given_dy, static_cast<const float*>(ps), static_cast<const float*>(pf), &g,
                                           workspace.data_ptr(), size, k.on.stream()));
        return wrap_all(du, ddelta, da, db, dc, dd, dz, dbias, dstate);
    });
}

// u, delta, a, b, c, state, d, z, delta_bias, softplus, reset
PyObject* selective_scan_step(PyObject*, PyObject* const* args, Py_ssize_t given) {
    return answer([&]() -> PyObject* {
        const Arguments a(args, given, 11);
        const Tensor u = a.tensor(0, "u"), delta = a.tensor(1, "delta"), ta = a.tensor(2, "a"), b = a.tensor(3, "b"), c = a.tensor(4, "c");
        const Tensor state = a.tensor(5, "state"), d = a.optional(6, "d"), z = a.optional(7, "z"), delta_bias = a.optional(8, "delta_bias");
        const Tensor reset = a.optional(10, "reset");
        Tracks k(u, "u", true);
        k.rounds(reset, Tensor());
        const Scanned s(k, u, delta, ta, b, c, d, z, delta_bias, a.flag(9));
        void* ps = k.packed(state, "state", {k.q.sequences, k.q.channels, s.scan.states}, T8B_F32);
        const Tensor y = k.output(u, 1, k.q.channels, false);
        done(entry.selective_scan_step(&k.q, &s.scan, static_cast<float*>(ps), k.fresh(y), k.on.stream()));
        return wrap(y);
    });
}

// ------------------------------------------------------------------ policy loss
// logits, actions, old_log_probabilities, advantages, mask, reference, weights, clip, clip_high, kl, entropy, gradient
PyObject* policy_loss(PyObject*, PyObject* const* args, Py_ssize_t given) {
    return answer([&]() -> PyObject* {
        const Arguments a(args, given, 12);
        const Tensor logits = a.tensor(0, "logits"), actions = a.tensor(1, "actions"), old = a.tensor(2, "old_log_probabilities");
        const Tensor advantages = a.tensor(3, "advantages"), mask = a.optional(4, "mask"), reference = a.optional(5, "reference");
        const Tensor weights = a.optional(6, "weights");
        const On on(logits);
        if (logits.dim() < 1) refuse("logits has shape (), expected [rows][logits]");
        t8b_policy_loss_t c{};
        c.type = type_of(logits, "logits");
        c.n = logits.size(-1);
        const Rows z = rows_of(logits, "logits", c.n, on.device);
        const auto lead = logits.sizes().slice(0, logits.dim() - 1);
        auto per_row = [&](const Tensor& t, const char* name, at::ScalarType type) -> const void* {
            if (!t.defined()) return nullptr;
            if (!t.is_cuda() || t.get_device() != on.device) refuse(std::string(name) + " is on another device");
            if (t.scalar_type() != type) refuse(std::string(name) + " is " + c10::toString(t.scalar_type()) + ", expected " + c10::toString(type));
            if (t.sizes() != lead) refuse(std::string(name) + " has shape " + text(t.sizes()) + ", expected one value a row, " + text(lead));
            if (!t.is_contiguous()) refuse(std::string(name) + " must be contiguous");
            return t.data_ptr();
        };
        c.rows = z.rows;
        c.logits = z.data;
        c.logits_stride = z.stride;
        c.actions = static_cast<const int64_t*>(per_row(actions, "actions", at::kLong));
        c.old_log_probabilities = static_cast<const float*>(per_row(old, "old_log_probabilities", at::kFloat));
        c.advantages = static_cast<const float*>(per_row(advantages, "advantages", at::kFloat));
        c.weights = static_cast<const float*>(per_row(weights, "weights", at::kFloat));
        if (mask.defined()) {
            const bool bits = mask.scalar_type() == at::kInt;
            if (!bits && mask.scalar_type() != at::kBool && mask.scalar_type() != at::kByte) {
                refuse("mask must be bool or uint8 (one value a logit) or int32 (one bit)");
            }
            if (mask.dim() < 1 || mask.sizes().slice(0, mask.dim() - 1) != lead) refuse("mask has shape " + text(mask.sizes()) + ", logits " + text(logits.sizes()));
            const Rows m = rows_of(mask, "mask", bits ? (c.n + 31) / 32 : c.n, on.device);
            c.mask_kind = bits ? T8B_MASK_BITS : T8B_MASK_BYTES;
            c.mask = m.data;
            c.mask_stride = m.stride;
        }
        if (reference.defined()) {
            if (reference.dim() == logits.dim()) {
                if (reference.sizes() != logits.sizes()) refuse("reference has shape " + text(reference.sizes()) + ", logits " + text(logits.sizes()));
                if (reference.scalar_type() != logits.scalar_type()) refuse("a reference's logits must have the logits' type");
                const Rows r = rows_of(reference, "reference", c.n, on.device);
                c.reference_kind = T8B_REFERENCE_LOGITS;
                c.reference = r.data;
                c.reference_stride = r.stride;
            } else {
                c.reference = per_row(reference, "reference", at::kFloat);
                c.reference_kind = T8B_REFERENCE_SAMPLED;
            }
        }
        c.clip_low = static_cast<float>(a.number(7));
        c.clip_high = args[8] == Py_None ? c.clip_low : static_cast<float>(a.number(8));
        c.kl = static_cast<float>(a.number(9));
        c.entropy = static_cast<float>(a.number(10));
        const bool gradient = a.flag(11);
        const Tensor loss = make(logits, lead, T8B_F32), lp = make(logits, lead, T8B_F32), entropies = make(logits, lead, T8B_F32);
        const Tensor divergences = make(logits, lead, T8B_F32);
        Tensor dlogits;
        int64_t stride = c.n;
        if (gradient) {  // rows start on 16 bytes, as the matrix products that read them like
            const int64_t pack = c.type == T8B_F32 ? 4 : 8;
            stride = (c.n + pack - 1) / pack * pack;
            dlogits = make(logits, Shape(logits, stride), c.type);
            if (stride != c.n) dlogits = dlogits.narrow(-1, 0, c.n);
        }
        done(entry.policy_loss(&c, loss.data_ptr<float>(), lp.data_ptr<float>(), entropies.data_ptr<float>(), divergences.data_ptr<float>(),
                               pointer(dlogits), stride, on.stream()));
        return gradient ? wrap_all(loss, lp, entropies, divergences, dlogits) : wrap_all(loss, lp, entropies, divergences);
    });
}

// bind(T8bError, torch.OutOfMemoryError, addresses of the entries in the order of Entries)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t given) {
    constexpr Py_ssize_t kEntries = sizeof(Entries) / sizeof(void*);
    if (given != kEntries + 2) {
        PyErr_SetString(PyExc_TypeError, "bind takes two error classes and every entry's address");
        return nullptr;
    }
    void* address[kEntries];
    for (Py_ssize_t i = 0; i < kEntries; ++i) {
        address[i] = PyLong_AsVoidPtr(args[i + 2]);
        if (address[i] == nullptr) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "a null entry");
            return nullptr;
        }
    }
    std::memcpy(&entry, address, sizeof(entry));
    Py_INCREF(args[0]);
    Py_INCREF(args[1]);
    Py_XDECREF(library_error);
    Py_XDECREF(memory_error);
    library_error = args[0];
    memory_error = args[1];
    Py_RETURN_NONE;
}

#define T8B_METHOD(name, function) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(function)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    T8B_METHOD("bind", bind),
    T8B_METHOD("layer_norm", layer_norm),
    T8B_METHOD("layer_norm_backward", layer_norm_backward),
    T8B_METHOD("linear", linear),
    T8B_METHOD("linear_backward", backward<1>),
    T8B_METHOD("gated", gated),
    T8B_METHOD("gated_backward", backward<2>),
    T8B_METHOD("causal_conv", causal_conv),
    T8B_METHOD("causal_conv_backward", causal_conv_backward),
    T8B_METHOD("causal_conv_step", causal_conv_step),
    T8B_METHOD("selective_scan", selective_scan),
    T8B_METHOD("selective_scan_backward", selective_scan_backward),
    T8B_METHOD("selective_scan_step", selective_scan_step),
    T8B_METHOD("policy_loss", policy_loss),
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_operators", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__operators() { return PyModule_Create(&module); }
