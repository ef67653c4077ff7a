// binding.cpp - the Python side of the 8-bit linear map, the residual-norm step and the beam search: checks of arguments,
// the output tensors, the descriptor and the C-ABI call, in one C++ function each (kea_kernels._binding; documented entry
// points in kea_kernels/lowbit.py). A decoding step issues these for a handful of rows, where a call lasts a few
// microseconds on the GPU and filling a descriptor through ctypes would take several times that on the host.
// The C-ABI functions are handed over by address at import (bind), so that one loaded library serves every caller.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <algorithm>
#include <cstring>
#include <limits>
#include <string>
#include <utility>
#include <vector>

#include "kea_lowbit.h"

namespace {

using at::Tensor;

struct Library {
    decltype(&kea_lowbit_int8_gemm) int8_gemm = nullptr;
    decltype(&kea_lowbit_residual_norm) residual_norm = nullptr;
    decltype(&kea_lowbit_beam_select) beam_select = nullptr;
    decltype(&kea_lowbit_beam_reorder) beam_reorder = nullptr;
    decltype(&kea_lowbit_status_string) status_string = nullptr;
    PyObject *layer_norm = nullptr, *rms_norm = nullptr;   // nn.LayerNorm, nn.RMSNorm
    PyObject *layer_forward = nullptr, *rms_forward = nullptr;
} lib;

[[noreturn]] void raise(PyObject *type, const std::string &text) {
    PyErr_SetString(type, text.c_str());
    throw python_error();
}
[[noreturn]] void refuse(const std::string &text) { raise(PyExc_ValueError, text); }

// ---- arguments -----------------------------------------------------------------------------------------------------
bool none(PyObject *o) { return o == Py_None; }

const Tensor &tensor(PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}
const Tensor &cuda_tensor(PyObject *o, const char *name) {
    const bool fine = THPVariable_Check(o) && THPVariable_Unpack(o).is_cuda();
    if (!fine) refuse(std::string(name) + " must be a CUDA tensor");
    return THPVariable_Unpack(o);
}
int64_t integer(PyObject *o, const char *name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    if (v < std::numeric_limits<int32_t>::min() || v > std::numeric_limits<int32_t>::max())
        refuse(std::string(name) + " is out of range");
    return v;
}
float number(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return (float)v;
}
bool truth(PyObject *o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v != 0;
}
at::ScalarType dtype(PyObject *o, const char *name) {
    if (!THPDtype_Check(o)) refuse(std::string(name) + " must be a torch.dtype");
    return reinterpret_cast<THPDtype *>(o)->scalar_type;
}

// ---- checks --------------------------------------------------------------------------------------------------------
int element_type(at::ScalarType t) {
    return t == at::kFloat ? KEA_TYPE_F32 : t == at::kHalf ? KEA_TYPE_F16 : t == at::kBFloat16 ? KEA_TYPE_BF16 : -1;
}
int value_type(at::ScalarType t, const char *name) {
    const int v = element_type(t);
    if (v < 0) refuse(std::string(name) + " must be FP32, FP16 or BF16, got " + c10::toString(t));
    return v;
}
void on(const Tensor &t, const char *name, const at::Device &device) {
    if (t.device() != device) refuse(std::string(name) + " must be on " + device.str());
}
int32_t small(int64_t v, const char *name) {
    if (v > std::numeric_limits<int32_t>::max()) refuse(std::string(name) + " has too many elements along one dimension");
    return (int32_t)v;
}

// The row stride of a matrix of unit column stride (a single row's stride says nothing: its width).
int64_t matrix(const Tensor &t, const char *name, const at::Device &device, int64_t rows, int64_t cols) {
    if (t.dim() != 2 || t.size(0) != rows || t.size(1) != cols)
        refuse(std::string(name) + " must be [" + std::to_string(rows) + ", " + std::to_string(cols) + "]");
    if (t.stride(1) != 1 && cols > 1) refuse(std::string(name) + " must have unit column stride");
    on(t, name, device);
    return rows > 1 ? t.stride(0) : cols;
}
const float *vector(const Tensor &t, int64_t n, const char *name, const at::Device &device) {
    if (t.scalar_type() != at::kFloat || t.dim() != 1 || t.size(0) != n || !t.is_contiguous() || t.device() != device)
        refuse(std::string(name) + " must be contiguous FP32 [" + std::to_string(n) + "] on " + device.str());
    return static_cast<const float *>(t.const_data_ptr());
}
// The one stride at which the rows of t [..., D] lie.
int64_t row_stride(const Tensor &t, const char *name) {
    const int64_t dims = t.dim(), d = t.size(-1);
    if (t.is_contiguous()) return d;
    if (t.stride(-1) != 1 && d > 1) refuse(std::string(name) + " must have unit stride along its last dimension");
    int64_t rows = 1, step = d;
    for (int64_t i = dims - 2; i >= 0; --i) {
        if (t.size(i) == 1) continue;
        if (rows == 1) step = t.stride(i);
        else if (t.stride(i) != step * rows) refuse(std::string(name) + "'s rows must lie at one stride");
        rows *= t.size(i);
    }
    return step;
}
uint32_t *error_word(PyObject *o, const at::Device &device) {
    if (none(o)) return nullptr;
    const Tensor &t = tensor(o, "error_word");
    if (t.scalar_type() != at::kInt || t.numel() != 1 || t.device() != device) refuse("error_word must be one int32 on " + device.str());
    return static_cast<uint32_t *>(t.data_ptr());
}

Tensor make(at::IntArrayRef shape, at::ScalarType type, const at::Device &device) {
    return at::empty(shape, at::TensorOptions().dtype(type).device(device));
}

template <typename Call>
void launch(const char *what, const at::Device &device, Call call) {
    if (!lib.status_string) raise(PyExc_RuntimeError, "kea_kernels._binding is not bound to the library");
    const c10::cuda::OptionalCUDAGuard guard(device);
    const int status = call(static_cast<void *>(c10::cuda::getCurrentCUDAStream(device.index()).stream()));
    if (status == KEA_OK) return;
    const std::string text = std::string(what) + ": " + lib.status_string(status);
    if ((status >= KEA_ERR_INVALID_VALUE && status <= KEA_ERR_INVALID_CODES) || status == KEA_ERR_SCRATCH_LIMIT) refuse(text);
    raise(PyExc_RuntimeError, text + " (status " + std::to_string(status) + ")");
}

void count(Py_ssize_t n, Py_ssize_t want) {
    if (n != want) raise(PyExc_TypeError, std::to_string(want) + " arguments expected, got " + std::to_string(n));
}

// ---- 8-bit linear map ----------------------------------------------------------------------------------------------
// (q, qs, weight, alpha, bias, out, k, dtype, silu, residual, residual_scale, acc, kernel, pdl, error_word) -> out
PyObject *int8_linear(PyObject *, PyObject *const *o, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    count(n_args, 15);
    const Tensor &q = cuda_tensor(o[0], "q"), &qs = tensor(o[1], "qs"), &w = tensor(o[2], "weight"), &alpha = tensor(o[3], "alpha");
    const at::Device device = q.device();
    if (q.scalar_type() != at::kChar || w.scalar_type() != at::kChar || q.dim() != 2 || w.dim() != 2)
        refuse("q and weight must be int8 [m, k] and [n, k]");
    const int64_t m = q.size(0), n = w.size(0);
    int64_t k = w.size(1);
    if (!none(o[6])) {
        k = integer(o[6], "k");
        if (k < 1 || k > q.size(1) || k > w.size(1))
            refuse("k must lie between 1 and the columns of q and weight, got " + std::to_string(k));
    } else if (q.size(1) != k) {
        refuse("q has " + std::to_string(q.size(1)) + " columns and weight " + std::to_string(k));
    }
    KeaInt8Desc d{};
    const int64_t ldq = matrix(q, "q", device, m, q.size(1)), ldw = matrix(w, "weight", device, n, w.size(1));
    d.ldq = m > 1 ? ldq : (k + 15) / 16 * 16;
    d.ldw = n > 1 ? ldw : (k + 15) / 16 * 16;
    d.qs = vector(qs, m, "qs", device);
    d.alpha = vector(alpha, n, "alpha", device);
    if (!none(o[4])) d.bias = vector(tensor(o[4], "bias"), n, "bias", device);
    Tensor out;
    if (none(o[5])) {
        const at::ScalarType type = dtype(o[7], "dtype");
        d.y_type = value_type(type, "the output");
        out = make({m, n}, type, device);
        d.ldy = n;
    } else {
        out = tensor(o[5], "out");
        d.y_type = value_type(out.scalar_type(), "the output");
        d.ldy = matrix(out, "out", device, m, n);
    }
    if (!none(o[9])) {
        const Tensor &r = tensor(o[9], "residual");
        if (r.scalar_type() != out.scalar_type()) refuse("residual must have the output's type");
        d.ld_residual = matrix(r, "residual", device, m, n);
        d.residual = r.const_data_ptr();
    }
    d.residual_scale = number(o[10]);
    if (!none(o[11])) {
        const Tensor &acc = tensor(o[11], "acc");
        if (acc.scalar_type() != at::kInt) refuse("acc must be int32");
        d.ld_acc = matrix(acc, "acc", device, m, n);
        d.acc = static_cast<int32_t *>(acc.data_ptr());
    }
    d.flags = (truth(o[8]) ? KEA_INT8_SILU : 0) | (truth(o[13]) ? KEA_INT8_PDL : 0);
    d.kernel = (int32_t)integer(o[12], "kernel");
    d.error_word = error_word(o[14], device);
    if (m > 0 && n > 0) {
        d.q = static_cast<const int8_t *>(q.const_data_ptr());
        d.w = static_cast<const int8_t *>(w.const_data_ptr());
        d.y = out.data_ptr();
        d.m = small(m, "q");
        d.n = small(n, "weight");
        d.k = small(k, "weight");
        launch("int8_linear", device, [&](void *stream) { return lib.int8_gemm(&d, stream); });
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// ---- residual norm -------------------------------------------------------------------------------------------------
struct Norm {
    int kind = KEA_NORM_NONE;
    float eps = 0.f;
    const float *weight = nullptr, *bias = nullptr;
};

// An nn.LayerNorm or nn.RMSNorm over the last dimension, or None. The module is read, not called, so one whose call would do
// something else - a class with a forward of its own, a forward or hooks of the module's - is refused.
Norm norm_of(PyObject *o, int64_t d, const at::Device &device, const char *name) {
    Norm r;
    if (none(o)) return r;
    const int layer = PyObject_IsInstance(o, lib.layer_norm);
    const int rms = layer == 1 ? 0 : PyObject_IsInstance(o, lib.rms_norm);
    if (layer < 0 || rms < 0) throw python_error();
    if (!layer && !rms) refuse(std::string(name) + " must be an nn.LayerNorm or an nn.RMSNorm");
    r.kind = layer ? KEA_NORM_LAYER : KEA_NORM_RMS;
    static PyObject *const s_parameters = PyUnicode_InternFromString("_parameters"), *const s_eps = PyUnicode_InternFromString("eps");
    static PyObject *const s_weight = PyUnicode_InternFromString("weight"), *const s_bias = PyUnicode_InternFromString("bias");
    static PyObject *const s_forward = PyUnicode_InternFromString("forward");
    static PyObject *const s_hooks[2] = {PyUnicode_InternFromString("_forward_hooks"), PyUnicode_InternFromString("_forward_pre_hooks")};
    PyObject *const type = reinterpret_cast<PyObject *>(Py_TYPE(o));
    if (type != (layer ? lib.layer_norm : lib.rms_norm)) {
        THPObjectPtr forward(PyObject_GetAttr(type, s_forward));
        if (!forward) throw python_error();
        if (forward.get() != (layer ? lib.layer_forward : lib.rms_forward)) refuse(std::string(name) + "'s class has a forward of its own");
    }
    THPObjectPtr own(PyObject_GenericGetDict(o, nullptr));
    if (!own) throw python_error();
    if (PyDict_GetItemWithError(own.get(), s_forward)) refuse(std::string(name) + " has a forward of its own");
    for (PyObject *s : s_hooks) {
        PyObject *hooks = PyDict_GetItemWithError(own.get(), s);   // borrowed
        if (hooks && PyDict_Check(hooks) && PyDict_Size(hooks) > 0) refuse(std::string(name) + " has forward hooks, which would not run");
    }
    if (PyErr_Occurred()) throw python_error();
    THPObjectPtr parameters(PyObject_GetAttr(o, s_parameters)), eps(PyObject_GetAttr(o, s_eps));
    if (!parameters || !eps) throw python_error();
    if (!PyDict_Check(parameters.get())) refuse(std::string(name) + " must be a module with parameters");
    PyObject *weight = PyDict_GetItemWithError(parameters.get(), s_weight);   // borrowed
    PyObject *bias = layer ? PyDict_GetItemWithError(parameters.get(), s_bias) : nullptr;
    if (PyErr_Occurred()) throw python_error();
    if (!weight || none(weight)) refuse(std::string(name) + " needs a weight");
    r.weight = vector(tensor(weight, name), d, name, device);
    if (bias && !none(bias)) r.bias = vector(tensor(bias, name), d, name, device);
    r.eps = none(eps.get()) ? std::numeric_limits<float>::epsilon() : number(eps.get());
    return r;
}

// Fills everything but h, q and qs; returns r. `rows` gets the number of rows (0: nothing to launch).
Tensor residual_arguments(PyObject *const *o, KeaResidualNormDesc &d, int64_t &rows) {
    const Tensor &x = cuda_tensor(o[0], "x"), &y = tensor(o[1], "y");
    const at::Device device = x.device();
    const int xt = element_type(x.scalar_type()), yt = element_type(y.scalar_type());
    if (x.dim() < 2 || y.sizes() != x.sizes() || xt < 0 || yt < 0)
        refuse("x and y must be FP32, FP16 or BF16 tensors [..., T, D] of one shape");
    on(y, "y", device);
    const int64_t width = x.size(-1), frames = x.size(-2);
    d.x_type = xt;
    d.y_type = yt;
    Tensor out;
    if (none(o[7])) {
        out = make(x.sizes(), x.scalar_type(), device);
    } else {
        out = tensor(o[7], "out");
        if (out.sizes() != x.sizes() || out.scalar_type() != x.scalar_type() || out.device() != device)
            refuse("out must have x's shape and type on " + device.str());
    }
    d.frames = small(std::max<int64_t>(frames, 1), "x");
    if (!none(o[3])) {
        const Tensor &g = tensor(o[3], "gate");
        if (g.dim() < 1 || g.scalar_type() != y.scalar_type() || g.device() != device || g.size(-1) != width ||
            (g.stride(-1) != 1 && width > 1))
            refuse("gate must be [..., " + std::to_string(width) + "] of y's type on " + device.str() +
                   " with unit stride along its last dimension");
        if (g.sizes() == x.sizes()) {
            d.gate_row_stride = row_stride(g, "gate");
            d.gate_clip_stride = frames * d.gate_row_stride;
        } else if (g.dim() == 2 && x.dim() == 3 && g.size(0) == x.size(0)) {
            d.gate_clip_stride = g.size(0) > 1 ? g.stride(0) : 0;
        } else if (g.dim() != 1) {
            refuse("gate must be one row [D], one row per clip [B, D] of x [B, T, D], or of x's shape");
        }
        d.gate = g.const_data_ptr();
    }
    const char *act = PyUnicode_Check(o[4]) ? PyUnicode_AsUTF8(o[4]) : nullptr;
    if (act && !strcmp(act, "none")) d.gate_act = KEA_GATE_NONE;
    else if (act && !strcmp(act, "sigmoid")) d.gate_act = KEA_GATE_SIGMOID;
    else refuse("gate_act must be \"none\" or \"sigmoid\"");
    d.scale = number(o[5]);
    const Norm post = norm_of(o[2], width, device, "post_norm"), pre = norm_of(o[6], width, device, "pre_norm");
    d.post = post.kind;
    d.post_eps = post.eps;
    d.post_weight = post.weight;
    d.post_bias = post.bias;
    d.pre = pre.kind;
    d.pre_eps = pre.eps;
    d.pre_weight = pre.weight;
    d.pre_bias = pre.bias;
    rows = width ? x.numel() / width : 0;
    if (rows) {
        d.x = x.const_data_ptr();
        d.y = y.const_data_ptr();
        d.r = out.data_ptr();
        d.ldx = row_stride(x, "x");
        d.ldy = row_stride(y, "y");
        d.ldr = row_stride(out, "out");
        d.m = small(rows, "x");
        d.d = small(width, "x");
    }
    d.flags = truth(o[8]) ? KEA_RNORM_PDL : 0;
    return out;
}

// (x, y, post_norm, gate, gate_act, scale, pre_norm, out, pdl, dtype or None) -> (r, h)
PyObject *residual_norm(PyObject *, PyObject *const *o, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    count(n_args, 10);
    KeaResidualNormDesc d{};
    int64_t rows = 0;
    Tensor r = residual_arguments(o, d, rows);
    const at::ScalarType type = none(o[9]) ? THPVariable_Unpack(o[1]).scalar_type() : dtype(o[9], "dtype");
    d.h_type = value_type(type, "h");
    Tensor h = make(r.sizes(), type, r.device());
    if (rows) {
        d.h = h.data_ptr();
        d.ldh = r.size(-1);
        launch("residual_norm", r.device(), [&](void *stream) { return lib.residual_norm(&d, stream); });
    }
    THPObjectPtr a(THPVariable_Wrap(std::move(r))), b(THPVariable_Wrap(std::move(h)));
    if (!a || !b) throw python_error();
    return PyTuple_Pack(2, a.get(), b.get());
    END_HANDLE_TH_ERRORS
}

// (x, y, post_norm, gate, gate_act, scale, pre_norm, out, pdl) -> (r, q, qs)
PyObject *residual_norm_quantized(PyObject *, PyObject *const *o, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    count(n_args, 9);
    KeaResidualNormDesc d{};
    int64_t rows = 0;
    Tensor r = residual_arguments(o, d, rows);
    const int64_t width = r.size(-1), ldq = (width + 15) / 16 * 16;
    Tensor q = make({rows, ldq}, at::kChar, r.device()), qs = make({rows}, at::kFloat, r.device());
    if (rows) {
        d.q = static_cast<int8_t *>(q.data_ptr());
        d.qs = static_cast<float *>(qs.data_ptr());
        d.ldq = small(ldq, "x");
        launch("residual_norm", r.device(), [&](void *stream) { return lib.residual_norm(&d, stream); });
    }
    if (ldq != width) q = q.narrow(1, 0, width);
    THPObjectPtr a(THPVariable_Wrap(std::move(r))), b(THPVariable_Wrap(std::move(q))), c(THPVariable_Wrap(std::move(qs)));
    if (!a || !b || !c) throw python_error();
    return PyTuple_Pack(3, a.get(), b.get(), c.get());
    END_HANDLE_TH_ERRORS
}

// ---- beam search ---------------------------------------------------------------------------------------------------
bool flags_like(const Tensor &t) { return t.scalar_type() == at::kBool || t.scalar_type() == at::kByte; }

// (logits, scores, width, end, ended, out or None, pdl) -> (scores, parents, tokens, ended)
PyObject *beam_select(PyObject *, PyObject *const *o, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    count(n_args, 7);
    const Tensor &x = cuda_tensor(o[0], "logits"), &s = tensor(o[1], "scores");
    const at::Device device = x.device();
    KeaBeamDesc d{};
    d.logits_type = element_type(x.scalar_type());
    if (x.dim() != 3 || d.logits_type < 0 || (x.stride(2) != 1 && x.size(2) > 1))
        refuse("logits must be FP32, FP16 or BF16 [clips, beams, vocab] with unit stride along the labels");
    const int64_t clips = x.size(0), beams = x.size(1), vocab = x.size(2), width = none(o[2]) ? beams : integer(o[2], "width");
    const std::string given = "[" + std::to_string(clips) + ", " + std::to_string(beams) + "] on " + device.str();
    const int64_t shape[2] = {clips, beams}, place[2] = {clips, width};
    const at::IntArrayRef in(shape, 2), to(place, 2);
    if (s.scalar_type() != at::kFloat || s.sizes() != in || s.device() != device || !s.is_contiguous())
        refuse("scores must be contiguous FP32 " + given);
    d.end = -1;
    if (!none(o[3])) {
        const int64_t end = integer(o[3], "end");
        if (end < 0 || end >= vocab) refuse("end must be a label below " + std::to_string(vocab) + ", got " + std::to_string(end));
        d.end = (int32_t)end;
    }
    if (!none(o[4])) {
        if (d.end < 0) refuse("ended hypotheses need the label `end`");
        const Tensor &e = tensor(o[4], "ended");
        if (!flags_like(e) || e.sizes() != in || e.device() != device || !e.is_contiguous()) refuse("ended must be contiguous bool " + given);
        d.ended = static_cast<const uint8_t *>(e.const_data_ptr());
    }
    if (width < 1 || width > beams * vocab) refuse("width must lie between 1 and beams * vocab, got " + std::to_string(width));
    Tensor out[4];
    if (none(o[5])) {
        out[0] = make(to, at::kFloat, device);
        out[1] = make(to, at::kInt, device);
        out[2] = make(to, at::kInt, device);
        if (d.end >= 0) out[3] = make(to, at::kBool, device);
    } else {
        if (!PyTuple_Check(o[5]) || PyTuple_GET_SIZE(o[5]) != 4) refuse("out must be a BeamStep");
        static const char *const names[4] = {"out.scores", "out.parents", "out.tokens", "out.ended"};
        for (int i = 0; i < 4; ++i) {
            PyObject *t = PyTuple_GET_ITEM(o[5], i);
            if (i == 3 && none(t)) continue;
            out[i] = tensor(t, names[i]);
            const bool type = i == 0 ? out[i].scalar_type() == at::kFloat : i < 3 ? out[i].scalar_type() == at::kInt : flags_like(out[i]);
            if (!type || out[i].sizes() != to || out[i].device() != device || !out[i].is_contiguous())
                refuse(std::string(names[i]) + " must be contiguous " + (i == 0 ? "FP32" : i < 3 ? "int32" : "bool") + " [" +
                       std::to_string(clips) + ", " + std::to_string(width) + "] on " + device.str());
        }
    }
    if (clips > 0) {
        d.logits = x.const_data_ptr();
        d.ld_clip = x.stride(0);
        d.ld_beam = x.stride(1);
        d.scores = static_cast<const float *>(s.const_data_ptr());
        d.out_scores = static_cast<float *>(out[0].data_ptr());
        d.parents = static_cast<int32_t *>(out[1].data_ptr());
        d.labels = static_cast<int32_t *>(out[2].data_ptr());
        d.out_ended = out[3].defined() ? static_cast<uint8_t *>(out[3].data_ptr()) : nullptr;
        d.clips = small(clips, "logits");
        d.beams = small(beams, "logits");
        d.vocab = small(vocab, "logits");
        d.width = (int32_t)width;
        d.flags = truth(o[6]) ? KEA_BEAM_PDL : 0;
        launch("beam_select", device, [&](void *stream) { return lib.beam_select(&d, stream); });
    }
    THPObjectPtr r[4];
    for (int i = 0; i < 4; ++i) {
        r[i] = out[i].defined() ? THPVariable_Wrap(std::move(out[i])) : Py_NewRef(Py_None);
        if (!r[i]) throw python_error();
    }
    return PyTuple_Pack(4, r[0].get(), r[1].get(), r[2].get(), r[3].get());
    END_HANDLE_TH_ERRORS
}

// A state's strides in bytes; what follows the hypotheses contiguous, the dimensions before the clips at one stride.
struct Layout {
    int64_t group = 0, clip, beam, row = 1, groups = 1;
};
Layout layout(const Tensor &t, int64_t batch, const char *what, Py_ssize_t index) {
    Layout r;
    const std::string name = std::string(what) + " " + std::to_string(index);
    const int64_t size = (int64_t)t.element_size();
    for (int64_t i = t.dim() - 1; i > batch + 1; --i) {
        if (t.size(i) > 1 && t.stride(i) != r.row) refuse(name + ": what follows the hypotheses must be contiguous");
        r.row *= t.size(i);
    }
    for (int64_t i = batch - 1; i >= 0; --i) {
        if (t.size(i) == 1) continue;
        if (r.groups == 1) r.group = t.stride(i);
        else if (t.stride(i) != r.group * r.groups) refuse(name + ": the dimensions before the clips must lie at one stride");
        r.groups *= t.size(i);
    }
    r.row *= size;
    r.group *= size;
    r.clip = t.stride(batch) * size;
    r.beam = t.stride(batch + 1) * size;
    return r;
}

// The bytes of a state or an output: rows at three strides.
struct Span {
    uintptr_t first, end;
    int64_t row, rows;
    int64_t count[3], step[3];
    Span(const void *p, const Layout &l, int64_t clips, int64_t beams)
        : first(reinterpret_cast<uintptr_t>(p)), end(first + l.row), row(l.row), rows(l.groups * clips * beams), count{l.groups, clips, beams},
          step{l.group, l.clip, l.beam} {
        for (int i = 0; i < 3; ++i) {
            if (count[i] == 1) step[i] = 0;
            end += (count[i] - 1) * step[i];
        }
    }
    // From the first byte to the last, modulo s: steps that are its multiples do not count.
    int64_t extent(int64_t s) const {
        int64_t n = row;
        for (int i = 0; i < 3; ++i)
            if (step[i] % s) n += (count[i] - 1) * step[i];
        return n;
    }
    void add(std::vector<std::pair<uintptr_t, uintptr_t>> &to) const {
        for (int64_t g = 0; g < count[0]; ++g)
            for (int64_t b = 0; b < count[1]; ++b)
                for (int64_t k = 0; k < count[2]; ++k) {
                    const uintptr_t at = first + g * step[0] + b * step[1] + k * step[2];
                    to.emplace_back(at, at + row);
                }
    }
};

// Whether no byte is in both: by their ends, by one of the steps (halves of a buffer that interleave), or row by row.
bool apart(const Span &a, const Span &b) {
    if (a.end <= b.first || b.end <= a.first) return true;
    for (const Span *of : {&a, &b})
        for (const int64_t s : of->step) {
            if (s == 0) continue;
            const int64_t from = ((int64_t)(b.first - a.first) % s + s) % s, ea = a.extent(s), eb = b.extent(s);
            if (from >= ea && from + eb <= s) return true;
        }
    if (a.rows + b.rows > (1 << 22)) return false;   // taken for an overlap
    std::vector<std::pair<uintptr_t, uintptr_t>> ra, rb;
    a.add(ra);
    b.add(rb);
    std::sort(ra.begin(), ra.end());
    std::sort(rb.begin(), rb.end());
    for (size_t i = 0, j = 0; i < ra.size() && j < rb.size();) {
        if (ra[i].second <= rb[j].first) ++i;
        else if (rb[j].second <= ra[i].first) ++j;
        else return false;
    }
    return true;
}

// (states, parents, batch_dim, out or None, pdl, error_word) -> list
PyObject *beam_reorder(PyObject *, PyObject *const *o, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    count(n_args, 6);
    const Tensor &parents = cuda_tensor(o[1], "parents");
    if (parents.scalar_type() != at::kInt || parents.dim() != 2 || !parents.is_contiguous())
        refuse("parents must be contiguous int32 [clips, width]");
    THPObjectPtr states(PySequence_Fast(o[0], "states must be a sequence of tensors"));
    if (!states) throw python_error();
    const Py_ssize_t total = PySequence_Fast_GET_SIZE(states.get());
    THPObjectPtr given;
    if (!none(o[3])) {
        given = PySequence_Fast(o[3], "out must be a sequence of tensors");
        if (!given) throw python_error();
        if (PySequence_Fast_GET_SIZE(given.get()) != total) refuse("one output per state");
    }
    const at::Device device = parents.device();
    const int64_t clips = parents.size(0), width = parents.size(1), batch = integer(o[2], "batch_dim");
    if (batch < 0) refuse("batch_dim must not be negative");
    KeaReorderDesc d{};
    d.parents = static_cast<const int32_t *>(parents.const_data_ptr());
    d.clips = small(clips, "parents");
    d.width = small(width, "parents");
    d.flags = truth(o[4]) ? KEA_BEAM_PDL : 0;
    d.error_word = error_word(o[5], device);
    THPObjectPtr results(PyList_New(total));
    if (!results) throw python_error();
    std::vector<KeaReorderItem> items;
    std::vector<Span> read, written;   // with outputs given
    items.reserve((size_t)total);
    int64_t beams = -1;
    for (Py_ssize_t i = 0; i < total; ++i) {
        const Tensor &s = tensor(PySequence_Fast_GET_ITEM(states.get(), i), "a state");
        if (s.dim() < batch + 2 || s.size(batch) != clips || s.device() != device)
            refuse("state " + std::to_string(i) + " must have " + std::to_string(clips) + " clips at dimension " +
                   std::to_string(batch) + " on " + device.str());
        if (beams < 0) beams = s.size(batch + 1);
        else if (s.size(batch + 1) != beams) refuse("every state must have the same number of hypotheses");
        at::DimVector want(s.sizes());
        want[(size_t)batch + 1] = width;
        Tensor r;
        if (!given) {
            r = make(want, s.scalar_type(), device);
        } else {
            r = tensor(PySequence_Fast_GET_ITEM(given.get(), i), "an output");
            if (r.sizes() != at::IntArrayRef(want) || r.scalar_type() != s.scalar_type() || r.device() != device)
                refuse("output " + std::to_string(i) + " must have its state's type and shape with " + std::to_string(width) + " places");
            if (at::has_internal_overlap(r) == at::MemOverlap::Yes) refuse("output " + std::to_string(i) + " overlaps itself");
        }
        if (r.numel()) {
            const Layout from = layout(s, batch, "state", i), into = layout(r, batch, "output", i);
            items.push_back(KeaReorderItem{s.const_data_ptr(), r.data_ptr(), from.group, from.clip, from.beam, into.group, into.clip,
                                           into.beam, from.row, small(from.groups, "a state")});
            if (given) {
                read.emplace_back(s.const_data_ptr(), from, clips, beams);
                written.emplace_back(r.data_ptr(), into, clips, width);
            }
        }
        PyObject *wrapped = given ? Py_NewRef(PySequence_Fast_GET_ITEM(given.get(), i)) : THPVariable_Wrap(std::move(r));
        if (!wrapped) throw python_error();
        PyList_SET_ITEM(results.get(), i, wrapped);
    }
    // every row moves in one launch, in any order
    if (!written.empty()) read.emplace_back(parents.const_data_ptr(), Layout{0, 0, 0, (int64_t)parents.nbytes(), 1}, 1, 1);
    for (size_t i = 0; i < written.size(); ++i) {
        for (const Span &from : read)
            if (!apart(written[i], from)) refuse("an output overlaps a state or the parents");
        for (size_t j = 0; j < i; ++j)
            if (!apart(written[i], written[j])) refuse("two outputs overlap");
    }
    d.beams = small(std::max<int64_t>(beams, 1), "a state");
    for (size_t first = 0; first < items.size(); first += KEA_REORDER_MAX) {
        d.count = (int32_t)std::min<size_t>(items.size() - first, KEA_REORDER_MAX);
        launch("beam_reorder", device, [&](void *stream) { return lib.beam_reorder(&d, items.data() + first, stream); });
    }
    return results.release();
    END_HANDLE_TH_ERRORS
}

// (int8_gemm, residual_norm, beam_select, beam_reorder, status_string: addresses; nn.LayerNorm, nn.RMSNorm)
PyObject *bind(PyObject *, PyObject *const *o, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    count(n_args, 7);
    void *address[5];
    for (int i = 0; i < 5; ++i) {
        address[i] = PyLong_AsVoidPtr(o[i]);
        if (!address[i]) refuse("bind needs the library's functions");
    }
    lib.int8_gemm = reinterpret_cast<decltype(lib.int8_gemm)>(address[0]);
    lib.residual_norm = reinterpret_cast<decltype(lib.residual_norm)>(address[1]);
    lib.beam_select = reinterpret_cast<decltype(lib.beam_select)>(address[2]);
    lib.beam_reorder = reinterpret_cast<decltype(lib.beam_reorder)>(address[3]);
    lib.status_string = reinterpret_cast<decltype(lib.status_string)>(address[4]);
    Py_XSETREF(lib.layer_norm, Py_NewRef(o[5]));
    Py_XSETREF(lib.rms_norm, Py_NewRef(o[6]));
    Py_XSETREF(lib.layer_forward, PyObject_GetAttrString(o[5], "forward"));
    Py_XSETREF(lib.rms_forward, PyObject_GetAttrString(o[6], "forward"));
    if (!lib.layer_forward || !lib.rms_forward) throw python_error();
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

#define KEA_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {KEA_METHOD(int8_linear), KEA_METHOD(residual_norm), KEA_METHOD(residual_norm_quantized),
                         KEA_METHOD(beam_select), KEA_METHOD(beam_reorder), KEA_METHOD(bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", "C++ entry points of kea_kernels.lowbit", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&module); }
