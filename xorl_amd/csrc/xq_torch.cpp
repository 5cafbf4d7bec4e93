// The host path of the modules as native code: a CPython extension over libxq_hip.so and torch's C++ API.
//
// A decode forward is one or two kernels of 5-20 us; read from Python (parameter look-ups, the weight descriptor and its
// checks, torch.empty, ctypes) the same call cost 22 us of host time for one linear, 50 for a SwiGLU MLP or three joint
// projections and 70 for a routed expert layer, so the GPU waited for the host.  Here the module's own dictionaries are read
// directly, outputs and workspaces come from torch's caching allocator without the dispatcher, and the backward is a C++
// autograd node that runs without the interpreter.
//
// Every entry point returns None where anything is out of the ordinary (tensor subclasses, sharded or CPU state, tangents of
// forward-mode differentiation, function transforms, a trace being recorded, quantization noise, an active rank below the
// stored one, unexpected dtypes or layouts, a module that defines for itself what is read or done here): the caller then takes its Python path, which also raises the argument errors.
// Nothing is remembered from one call to the next, and a backward takes the addresses of the packed weights anew from
// their tensors: storage may have been freed and filled again between the two.
#include <Python.h>

#include <ATen/TensorSubclassLikeUtils.h>
#include <ATen/TracerMode.h>
#include <ATen/core/Tensor.h>
#include <ATen/EmptyTensor.h>
#include <ATen/ops/_foreach_add.h>
#include <ATen/ops/zeros_like.h>
#include <ATen/hip/impl/HIPCachingAllocatorMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <string>
#include <vector>

#include "../../include/xq.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// ---- names and classes handed over by the Python side (init)
PyObject* g_error = nullptr;            // xorl_amd._C.XqError
PyObject* g_functional = nullptr;       // the dict of xorl_amd.functional: SKINNY_CHECK_EVERY, skinny_status

// a module class and the methods whose work is done here in their place, as the class defines them
struct Program {
    PyTypeObject* type = nullptr;
    std::vector<PyObject*> name, method;
};
constexpr int kFormats = XQ_FMT_NF4 + 1;
Program g_linear[kFormats], g_experts[kFormats];      // by format; no type: no such class

#define XQ_NAMES(F)                                                                                                       \
    F(_parameters) F(_buffers) F(lora_A) F(lora_B) F(bias) F(packed_weight_f32) F(weight_scales) F(weight_block_scales)   \
    F(weight_global_scale) F(_scale_dtypes) F(active_r) F(active_lora_alpha) F(enable_aqn) F(training) F(quant_format)    \
    F(quant_group_size) F(in_features) F(out_features) F(num_local_experts) F(num_experts) F(hidden_size)                 \
    F(intermediate_size) F(use_rslora) F(swiglu_limit) F(moe_implementation) F(gate) F(up) F(down) F(gate_packed)         \
    F(up_packed) F(down_packed) F(gate_block_scales) F(up_block_scales) F(down_block_scales) F(gate_scales) F(up_scales)  \
    F(down_scales) F(gate_global_scale) F(up_global_scale) F(down_global_scale) F(gate_proj_lora_A) F(gate_proj_lora_B)   \
    F(up_proj_lora_A) F(up_proj_lora_B) F(down_proj_lora_A) F(down_proj_lora_B) F(SKINNY_CHECK_EVERY) F(skinny_status)     \
    F(__getattr__) F(__getattribute__)
#define XQ_DECLARE(n) PyObject* s_##n;
struct Names { XQ_NAMES(XQ_DECLARE) } N;
#undef XQ_DECLARE

PyObject* get(PyObject* dict, PyObject* name) { return dict ? PyDict_GetItem(dict, name) : nullptr; }   // borrowed, no error set

PyObject* dict_of(PyObject* module) {
    PyObject** p = _PyObject_GetDictPtr(module);
    return p ? *p : nullptr;
}

// whether the methods of `p` are the ones that run on `module` (no subclass, instance attribute or patch replaces one) and, in
// a subclass, whether what is read from the module's dictionaries is what attribute access gives (no property, no __getattr__
// of its own).  The library's own classes: 4-6 look-ups in the type's method cache and as many in the instance's dictionary.
bool as_defined(PyObject* module, PyObject* dict, const Program& p) {
    if (!p.type || !PyObject_TypeCheck(module, p.type)) return false;
    PyTypeObject* type = Py_TYPE(module);
    for (size_t i = 0; i < p.name.size(); ++i)
        if (_PyType_Lookup(type, p.name[i]) != p.method[i] || get(dict, p.name[i])) return false;
    if (type == p.type) return true;
#define XQ_SAME(n) if (_PyType_Lookup(type, N.s_##n) != _PyType_Lookup(p.type, N.s_##n)) return false;
    XQ_NAMES(XQ_SAME)
#undef XQ_SAME
    return true;
}

bool get_int(PyObject* dict, PyObject* name, int64_t* out) {
    PyObject* o = get(dict, name);
    if (!o || !PyLong_Check(o)) return false;
    *out = PyLong_AsLongLong(o);
    if (*out == -1 && PyErr_Occurred()) { PyErr_Clear(); return false; }
    return true;
}

bool get_number(PyObject* dict, PyObject* name, double* out) {
    PyObject* o = get(dict, name);
    if (!o || !(PyFloat_Check(o) || PyLong_Check(o))) return false;
    *out = PyFloat_AsDouble(o);
    if (*out == -1.0 && PyErr_Occurred()) { PyErr_Clear(); return false; }
    return true;
}

// a plain torch tensor (or Parameter) on the GPU; subclasses, fakes, functorch wrappers and tensors that carry a tangent are
// left to the Python path (whose autograd functions refuse what they do not define)
const Tensor* plain(PyObject* o) {
    if (!o || !THPVariable_CheckExact(o)) return nullptr;
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || at::isTensorSubclassLike(t) || t._fw_grad(0).defined()) return nullptr;
    return &t;
}

// a recorded trace or a function transform sees the operators of the Python path only
bool under_transform() {
    return at::tracer::impl::is_dispatch_enabled() ||
           c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}

// library calls launch kernels and may wait for room in the queue: other Python threads go on meanwhile
struct ReleaseGil {
    PyThreadState* state = PyEval_SaveThread();
    ~ReleaseGil() { PyEval_RestoreThread(state); }
};

int scale_code(PyObject* dtype, int* bytes) {
    if (!dtype || !THPDtype_Check(dtype)) return -1;
    switch (((THPDtype*)dtype)->scalar_type) {
        case at::kFloat: *bytes = 4; return XQ_SCALE_F32;
        case at::kBFloat16: *bytes = 2; return XQ_SCALE_BF16;
        case at::kFloat8_e4m3fn: *bytes = 1; return XQ_SCALE_E4M3;
        default: return -1;
    }
}

int format_code(PyObject* name) {
    if (!name || !PyUnicode_Check(name)) return -1;
    if (PyUnicode_CompareWithASCIIString(name, "block_fp8") == 0) return XQ_FMT_FP8;
    if (PyUnicode_CompareWithASCIIString(name, "nvfp4") == 0) return XQ_FMT_NVFP4;
    if (PyUnicode_CompareWithASCIIString(name, "int4") == 0) return XQ_FMT_INT4;
    if (PyUnicode_CompareWithASCIIString(name, "nf4") == 0) return XQ_FMT_NF4;
    return -1;
}

int64_t nbytes(const Tensor& t) { return t.numel() * (int64_t)t.element_size(); }

// packed bytes, scales and (nvfp4) the global scale of a weight, checked for size as _C.make_weight does
struct Weight {
    xq_weight w{};
    Tensor packed, scales, global_scale;
    int64_t packed_bytes = 0, scale_bytes = 0;

    bool fill(int fmt, int layout, int64_t rows, int64_t cols, int64_t group, int64_t experts, PyObject* packed_o, PyObject* scales_o,
              PyObject* scale_dtype, PyObject* global_o, PyObject* global_dtype) {
        const Tensor *p = plain(packed_o), *s = plain(scales_o);
        int sb = 0;
        const int sd = scale_code(scale_dtype, &sb);
        if (!p || !s || sd < 0 || !p->is_contiguous() || !s->is_contiguous() || rows <= 0 || cols <= 0 || group <= 0) return false;
        if (nbytes(*p) != experts * (fmt == XQ_FMT_FP8 ? rows * cols : rows * cols / 2)) return false;
        if (fmt == XQ_FMT_FP8) {
            if (sd != XQ_SCALE_F32 || nbytes(*s) != experts * ((rows + 127) / 128) * ((cols + 127) / 128) * 4) return false;
        } else if (rows * cols % group || nbytes(*s) != experts * (rows * cols / group) * sb) {
            return false;
        }
        if (fmt == XQ_FMT_NVFP4) {
            const Tensor* g = plain(global_o);
            int gb = 0;
            if (!g || scale_code(global_dtype, &gb) != XQ_SCALE_F32 || !g->is_contiguous() || nbytes(*g) < 4 * experts) return false;
            if ((uintptr_t)g->data_ptr() % 4) return false;
            global_scale = *g;
            w.global_scale = (const float*)g->data_ptr();
        }
        packed = *p;
        scales = *s;
        w.format = fmt; w.layout = layout; w.scale_dtype = sd; w.group = (int32_t)group;
        w.rows = rows; w.cols = cols; w.num_experts = (int32_t)experts;
        w.packed = p->data_ptr(); w.scales = s->data_ptr();
        packed_bytes = nbytes(*p); scale_bytes = nbytes(*s);
        return true;
    }

    // the descriptor for a later call: addresses as they are now, and storage that still holds the bytes
    const xq_weight* now() {
        auto held = [](const Tensor& t, int64_t bytes) {
            return nbytes(t) == bytes && t.is_contiguous() &&
                   (int64_t)t.storage().nbytes() >= t.storage_offset() * (int64_t)t.element_size() + bytes;
        };
        TORCH_CHECK(held(packed, packed_bytes) && held(scales, scale_bytes) &&
                        (!global_scale.defined() || held(global_scale, nbytes(global_scale))),
                    "the packed weight of a QLoRA module was freed or resized between forward and backward");
        w.packed = packed.data_ptr();
        w.scales = scales.data_ptr();
        if (global_scale.defined()) w.global_scale = (const float*)global_scale.data_ptr();
        return &w;
    }
};

// a QLoRALinear as the kernels see it
struct Linear {
    Weight q;
    Tensor A, B, bias;      // bias undefined: none
    int r = 0;
    double scaling = 0;
    bool A_grad = false, B_grad = false, bias_grad = false;

    int lora_dtype() const { return A.scalar_type() == at::kFloat ? XQ_DT_F32 : XQ_DT_BF16; }
    bool wants_grad() const { return A_grad || B_grad || bias_grad; }
    const void* bias_ptr() const { return bias.defined() ? bias.data_ptr() : nullptr; }

    bool read(PyObject* module) {
        PyObject* d = dict_of(module);
        PyObject *params = get(d, N.s__parameters), *bufs = get(d, N.s__buffers), *sdt = get(d, N.s__scale_dtypes);
        if (!params || !bufs || !sdt || !PyDict_Check(sdt)) return false;
        PyObject* aqn = get(d, N.s_enable_aqn);
        if (aqn != Py_False && !(aqn == Py_True && get(d, N.s_training) == Py_False)) return false;
        const int fmt = format_code(get(d, N.s_quant_format));
        int64_t rank, group, n, k;
        double alpha;
        if (fmt < 0 || !as_defined(module, d, g_linear[fmt]) || !get_int(d, N.s_active_r, &rank) || !get_number(d, N.s_active_lora_alpha, &alpha) ||
            !get_int(d, N.s_quant_group_size, &group) || !get_int(d, N.s_out_features, &n) || !get_int(d, N.s_in_features, &k))
            return false;
        PyObject* packed_o = get(params, N.s_packed_weight_f32);
        const Tensor* packed = plain(packed_o);
        if (!packed || packed->scalar_type() != at::kFloat) return false;      // (bytes held as fp32: anything else has been cast)
        PyObject* sname = fmt == XQ_FMT_FP8 || fmt == XQ_FMT_NVFP4 ? N.s_weight_block_scales : N.s_weight_scales;
        if (!q.fill(fmt, XQ_LAYOUT_FLAT, n, k, group, 1, packed_o, get(bufs, sname), get(sdt, sname),
                    get(bufs, N.s_weight_global_scale), get(sdt, N.s_weight_global_scale)))
            return false;
        const Tensor *a = plain(get(params, N.s_lora_A)), *b = plain(get(params, N.s_lora_B));
        if (!a || !b || rank < 1 || rank > 64 || a->dim() != 2 || b->dim() != 2 || a->size(0) != rank || b->size(1) != rank || a->size(1) != k ||
            b->size(0) != n || !a->is_contiguous() || !b->is_contiguous() || a->scalar_type() != b->scalar_type() ||
            (a->scalar_type() != at::kFloat && a->scalar_type() != at::kBFloat16))
            return false;
        PyObject* bias_o = get(params, N.s_bias);
        if (bias_o && bias_o != Py_None) {
            const Tensor* bt = plain(bias_o);
            if (!bt || bt->numel() != n || !bt->data_ptr()) return false;        // (without memory it would count as absent)
            bias_grad = bt->requires_grad();
            bias = bt->scalar_type() == at::kBFloat16 && bt->is_contiguous() ? *bt : bt->detach().to(at::kBFloat16).contiguous();
        }
        A = *a;
        B = *b;
        A_grad = a->requires_grad();
        B_grad = b->requires_grad();
        r = (int)rank;
        scaling = alpha / (double)rank;
        return true;
    }
};

// activations as rows of `width`: the pointer and pitch the library takes.  Rows that lie a fixed pitch apart over all leading
// dimensions are read where they are (a slice of a wider last dimension, any number of dimensions); other layouts, and pitches
// or addresses that are no multiple of 16 bytes, take a packed copy.
struct Rows {
    Tensor keep;
    const void* ptr = nullptr;
    int64_t ld = 0, M = 0;

    static bool pitched(const Tensor& x, int64_t* pitch) {
        return (uintptr_t)x.data_ptr() % 16 == 0 && any_pitch(x, pitch) && (x.numel() == x.size(-1) || *pitch % 8 == 0);
    }
    static bool any_pitch(const Tensor& x, int64_t* pitch) {
        if (x.stride(-1) != 1) return false;
        int64_t rows = 1;                                          // of the dimensions looked at, the innermost first
        for (int64_t d = x.dim() - 2; d >= 0; --d) {
            if (x.size(d) == 1) continue;
            if (rows == 1) *pitch = x.stride(d);
            else if (x.stride(d) != *pitch * rows) return false;
            rows *= x.size(d);
        }
        return true;
    }

    Rows(const Tensor& x, int64_t width) {
        M = width ? x.numel() / width : 0;
        ld = width;
        keep = x;
        if (!x.is_contiguous() && !pitched(x, &ld)) {
            keep = x.contiguous();
            ld = width;
        }
        ptr = keep.data_ptr();
    }
};

// torch's caching allocator, in the form whose tensors are "cuda" tensors
c10::Allocator* allocator() {
    static c10::Allocator* a = c10::hip::HIPCachingAllocatorMasqueradingAsCUDA::get();
    return a;
}

Tensor empty(at::IntArrayRef size, at::ScalarType dt) {
    constexpr c10::DispatchKeySet ks(c10::DispatchKey::CUDA);
    return at::detail::empty_generic(size, allocator(), ks, dt, std::nullopt);
}
Tensor empty_bf(at::IntArrayRef size) { return empty(size, at::kBFloat16); }
Tensor empty_f32(at::IntArrayRef size) { return empty(size, at::kFloat); }

// scratch of one call: back with the allocator (in stream order) when the call returns
struct Scratch {
    c10::DataPtr p;
    int64_t bytes;
    explicit Scratch(int64_t n) : p(allocator()->allocate((size_t)(n > 0 ? n : 0))), bytes(n) {}
    void* get() const { return p.get(); }
};

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

struct ArgError : std::runtime_error { using std::runtime_error::runtime_error; };

void check(int rc) {
    if (rc == XQ_OK) return;
    if (rc == XQ_ERR_LAUNCH) throw std::runtime_error(xq_last_error());
    throw ArgError(xq_last_error());
}

std::vector<int64_t> with_last(const Tensor& x, int64_t last) {
    std::vector<int64_t> s(x.sizes().begin(), x.sizes().end());
    s.back() = last;
    return s;
}

int r_pad_of(int r) { return (r + 15) / 16 * 16; }

int shared_format(const xq_weight& a, const xq_weight& b, const xq_weight& c) { return a.format == b.format && a.format == c.format ? a.format : -1; }

// the report of the one-launch decode forwards is read after every functional.SKINNY_CHECK_EVERY forwards of up to 16 rows
bool note_decode_forward(const Tensor& x, int64_t M) {
    static int64_t calls = 0;       // (under the GIL)
    if (M > 16) return true;
    int64_t every;
    if (!get_int(g_functional, N.s_SKINNY_CHECK_EVERY, &every)) every = 1024;
    if (++calls < every) return true;
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing((hipStream_t)stream_of(x), &cap) != hipSuccess || cap != hipStreamCaptureStatusNone) return true;
    calls = 0;
    PyObject* fn = get(g_functional, N.s_skinny_status);
    PyObject* dev = THPDevice_New(x.device());
    PyObject* r = fn && dev ? PyObject_CallFunctionObjArgs(fn, dev, nullptr) : nullptr;
    Py_XDECREF(dev);
    Py_XDECREF(r);
    return r != nullptr;
}

// ---- backward nodes: edges in the order of the inputs named in each
Tensor cast_to(Tensor g, at::ScalarType dt) {
    if (g.is_neg()) g = g.resolve_neg();                 // (a view whose memory holds the other sign)
    return g.scalar_type() == dt ? g : g.to(dt);
}

struct QLoRALinearBackward : public Node {
    SavedVariable x_, su_, A_, B_;
    Weight q;
    int r = 0;
    double scaling = 0;
    at::ScalarType bias_dt = at::kBFloat16;

    std::string name() const override { return "QLoRALinearBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        x_.reset_data();
        su_.reset_data();
        A_.reset_data();
        B_.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(4);
        if (!grads[0].defined()) grads[0] = input_metadata(0).zeros_like();
        const Tensor x = x_.unpack(), A = A_.unpack(), B = B_.unpack(), su = su_.unpack(shared_from_this());
        const int64_t Nf = q.w.rows, K = q.w.cols;
        Tensor dy = cast_to(grads[0], at::kBFloat16);
        c10::DeviceGuard guard(x.device());
        const Rows dr(dy, Nf), xr(x, K);
        const int64_t M = dr.M;
        const bool need_dx = task_should_compute_output(0), need_dA = task_should_compute_output(1), need_dB = task_should_compute_output(2);
        if (need_dx) out[0] = empty_bf(x.sizes());
        if (need_dA) out[1] = empty_f32({r, K});
        if (need_dB) out[2] = empty_f32({Nf, r});
        Scratch ws(xq_linear_workspace_bytes_fmt(q.w.format, M, Nf, K, r));
        check(xq_linear_bwd(q.now(), xr.ptr, xr.ld, dr.ptr, dr.ld, M, A.data_ptr(), B.data_ptr(),
                            A.scalar_type() == at::kFloat ? XQ_DT_F32 : XQ_DT_BF16, r, (float)scaling, M ? su.data_ptr() : nullptr,
                            need_dx ? out[0].data_ptr() : nullptr, K, need_dA ? (float*)out[1].data_ptr() : nullptr,
                            need_dB ? (float*)out[2].data_ptr() : nullptr, ws.get(), ws.bytes, stream_of(x)));
        if (need_dA) out[1] = cast_to(out[1], A.scalar_type());
        if (need_dB) out[2] = cast_to(out[2], B.scalar_type());
        if (task_should_compute_output(3)) out[3] = cast_to(grads[0].reshape({-1, Nf}).sum(0), bias_dt);
        return out;
    }
};

void mlp_lora(xq_mlp_lora* L, const Tensor* A, const Tensor* B, int r, double scaling) {
    for (int p = 0; p < 3; ++p) {
        L->A[p] = A[p].data_ptr();
        L->B[p] = B[p].data_ptr();
        L->bias[p] = nullptr;
    }
    L->dtype = A[0].scalar_type() == at::kFloat ? XQ_DT_F32 : XQ_DT_BF16;
    L->r = r;
    L->scaling = (float)scaling;
    L->reserved = 0;
}

struct QLoRAMLPBackward : public Node {
    SavedVariable x_, kept_[4], A_[3], B_[3];     // kept: gate | up, h, su of gate and up, su of down
    Weight q[3];
    int r = 0, gate_up_fused = 0;
    double scaling = 0;

    std::string name() const override { return "QLoRAMLPBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        x_.reset_data();
        for (auto& v : kept_) v.reset_data();
        for (auto& v : A_) v.reset_data();
        for (auto& v : B_) v.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(7);                      // x, gate A, gate B, up A, up B, down A, down B
        if (!grads[0].defined()) grads[0] = input_metadata(0).zeros_like();
        const Tensor x = x_.unpack();
        Tensor kept[4], A[3], B[3];
        for (int i = 0; i < 4; ++i) kept[i] = kept_[i].unpack(shared_from_this());
        for (int p = 0; p < 3; ++p) { A[p] = A_[p].unpack(); B[p] = B_[p].unpack(); }
        const int64_t I = q[0].w.rows, H = q[0].w.cols;
        Tensor dy = cast_to(grads[0], at::kBFloat16);
        c10::DeviceGuard guard(x.device());
        const Rows dr(dy, H), xr(x, H);
        const bool need_dx = task_should_compute_output(0);
        if (need_dx) out[0] = empty_bf(x.sizes());
        xq_mlp_grads G;
        for (int p = 0; p < 3; ++p) {
            out[1 + 2 * p] = empty_f32(A[p].sizes());
            out[2 + 2 * p] = empty_f32(B[p].sizes());
            G.dA[p] = (float*)out[1 + 2 * p].data_ptr();
            G.dB[p] = (float*)out[2 + 2 * p].data_ptr();
        }
        xq_mlp_lora L;
        mlp_lora(&L, A, B, r, scaling);
        xq_mlp_saved S{kept[0].data_ptr(), kept[1].data_ptr(), kept[2].data_ptr(), kept[3].data_ptr(), gate_up_fused, 0};
        Scratch ws(xq_mlp_workspace_bytes_fmt(shared_format(q[0].w, q[1].w, q[2].w), dr.M, H, I, r, 1));
        check(xq_mlp_bwd(q[0].now(), q[1].now(), q[2].now(), &L, xr.ptr, xr.ld, dr.ptr, dr.ld, dr.M, &S, need_dx ? out[0].data_ptr() : nullptr, H, &G,
                         ws.get(), ws.bytes, stream_of(x)));
        for (int p = 0; p < 3; ++p) {
            out[1 + 2 * p] = cast_to(out[1 + 2 * p], A[p].scalar_type());
            out[2 + 2 * p] = cast_to(out[2 + 2 * p], B[p].scalar_type());
        }
        return out;
    }
};

// what a cross entropy over a head is about: tensors, checked, as the library takes them.  A head whose rows do not lie a multiple of 16 bytes
// apart is copied by the call, in the forward and in the backward again: kept in between it would be held twice
struct HeadLoss {
    xq_lce_problem q{};
    Tensor keep_w, keep_labels;
    Rows xr;

    HeadLoss(const Tensor& x, const Tensor& w, const Tensor& labels, int64_t ignore, int reduction, double scale) : xr(aligned(x), x.size(-1)) {
        keep_w = in_rows(w) ? w : aligned(w.contiguous());
        keep_labels = labels.is_contiguous() ? labels : labels.contiguous();
        q.x = xr.ptr; q.ldx = xr.ld; q.M = xr.M;
        q.w = keep_w.data_ptr(); q.V = w.size(0); q.H = w.size(1); q.ldw = q.V > 1 ? keep_w.stride(0) : q.H;
        q.labels = keep_labels.data_ptr(); q.label_bytes = (int32_t)keep_labels.element_size();
        q.ignore_index = ignore; q.reduction = reduction; q.logit_scale = (float)scale;
    }
    static bool takes(const Tensor& x, const Tensor& w, const Tensor& labels) {
        if (x.scalar_type() != at::kBFloat16 || w.scalar_type() != at::kBFloat16 || w.dim() != 2 || x.dim() < 1 || labels.dim() != x.dim() - 1) return false;
        if (labels.scalar_type() != at::kLong && labels.scalar_type() != at::kInt) return false;
        if (x.sizes().slice(0, x.dim() - 1) != labels.sizes() || x.size(-1) != w.size(1) || w.size(1) < 64 || w.size(1) % 64 || w.size(0) < 1) return false;
        if (x.device() != w.device() || x.device() != labels.device() || x.is_neg() || w.is_neg() || labels.is_neg()) return false;
        return true;
    }
    static bool in_rows(const Tensor& w) {
        return w.stride(1) == 1 && (w.size(0) == 1 || (w.stride(0) >= w.size(1) && w.stride(0) % 8 == 0)) && (uintptr_t)w.data_ptr() % 16 == 0;
    }
    static Tensor aligned(const Tensor& t) { return t.is_contiguous() && (uintptr_t)t.data_ptr() % 16 != 0 ? t.clone() : t; }
};

// whether a tensor's elements lie in its storage
bool in_storage(const Tensor& t) {
    if (t.numel() == 0) return true;
    int64_t last = t.storage_offset();
    for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    return (last + 1) * (int64_t)t.element_size() <= (int64_t)t.storage().nbytes();
}

// the tensors of a forward whose memory was freed or cut under them: a view into it has an address all the same
void check_held(const char* who, std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        if (t && !in_storage(*t)) throw ArgError(std::string(who) + ": a tensor has no memory of its own (any more): it was freed or resized");
}

// whether a stream of torch's is part of this capture (the default stream, which has id 0, never is, and may not be asked while one goes on)
bool in_capture(const c10::Stream& s, unsigned long long id) {
    if (s.id() == 0) return false;
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long other = 0;
    const hipStream_t h = c10::hip::HIPStreamMasqueradingAsCUDA(s).stream();
    return hipStreamGetCaptureInfo(h, &status, &other) == hipSuccess && status == hipStreamCaptureStatusActive && other == id;
}

// Gradients that go on to another stream make that stream wait for this one; under capture that ends the process, unless the stream is in the
// same capture.  A leaf's stream is that of the oldest graph which still holds it, so an eager result that lives is enough.
template <typename F>
void refuse_other_streams(const Node& node, const Tensor& on, F&& wanted, const char* who, const char* results, const char* input) {
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    unsigned long long capture_id = 0;
    if (hipStreamGetCaptureInfo((hipStream_t)stream_of(on), &capture, &capture_id) != hipSuccess || capture == hipStreamCaptureStatusNone) return;
    const c10::StreamId here = c10::hip::getCurrentHIPStream(on.device().index()).unwrap().id();
    for (uint32_t i = 0; i < node.num_outputs(); ++i) {
        const auto& edge = node.next_edge(i);
        const auto there = edge.function ? edge.function->stream() : std::nullopt;
        if (wanted(i) && there && there->id() != here && !in_capture(*there, capture_id))
            throw std::runtime_error(std::string(who) + ": a captured backward would hand its gradients to another stream; free the " + results +
                                     " that were made from the same tensors outside the capture, and make " + input + " inside it or let it be a leaf");
    }
}

// a graph of the backward is being recorded: what comes out of it cannot be differentiated, and says so if it is
void differentiable_once(variable_list& out, const char* who) {
    for (Tensor& t : out)
        if (t.defined()) {
            auto error = std::make_shared<torch::autograd::DelayedError>(std::string(who) + " is differentiable once", 1);
            t = (*error)({t.detach().requires_grad_(true)})[0];
        }
}

struct LinearCrossEntropyBackward : public Node {
    SavedVariable x_, w_, labels_, saved_;
    int64_t ignore = 0;
    int reduction = 0, keep = 0;
    double scale = 1;
    int64_t M = 0, V = 0, H = 0, saved_bytes = 0;            // of the forward: what was saved is as long as that

    std::string name() const override { return "LinearCrossEntropyBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        x_.reset_data();
        w_.reset_data();
        labels_.reset_data();
        saved_.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(2);
        if (!grads[0].defined()) grads[0] = input_metadata(0).zeros_like();
        const Tensor x = x_.unpack(), w = w_.unpack(), labels = labels_.unpack(), saved = saved_.unpack(shared_from_this());
        c10::DeviceGuard guard(x.device());
        const bool again = at::GradMode::is_enabled();
        refuse_other_streams(*this, x, [this](size_t i) { return task_should_compute_output(i); }, "linear_cross_entropy", "losses", "x");
        {
            at::NoGradGuard no_grad;
            const Tensor g = cast_to(grads[0], at::kFloat).contiguous();
            // (`.data` and the storage can be exchanged without a word to autograd)
            if (!in_storage(x) || !in_storage(w) || x.dim() < 1 || w.dim() != 2 || x.size(-1) != H || w.size(1) != H || w.size(0) != V || x.numel() != M * H)
                throw std::runtime_error("linear_cross_entropy: x or weight was freed or resized between forward and backward");
            if (!saved.is_cuda() || nbytes(saved) != saved_bytes || !saved.is_contiguous() || !in_storage(saved))
                throw std::runtime_error("linear_cross_entropy: hooks of saved tensors gave back something else than was saved");
            const HeadLoss h(x, w, labels, ignore, reduction, scale);
            const bool need_dx = task_should_compute_output(0), need_dw = task_should_compute_output(1);
            if (need_dx) out[0] = empty_bf(x.sizes());
            if (need_dw) out[1] = empty_bf(w.sizes());
            Scratch ws(need_dw ? xq_lce_workspace_bytes(h.q.M, h.q.V, h.q.H, XQ_LCE_KEEP_HEAD_BWD) : 0);
            check(xq_lce_bwd(&h.q, (const float*)g.data_ptr(), saved.data_ptr(), keep, need_dx ? out[0].data_ptr() : nullptr, h.q.H,
                             need_dw ? out[1].data_ptr() : nullptr, h.q.H, need_dw ? ws.get() : nullptr, ws.bytes, stream_of(x)));
        }
        if (again) differentiable_once(out, "linear_cross_entropy");
        return out;
    }
};

// ---- what a program picks by an index per token
// rows of any pitch and alignment, not overlapping; other layouts take a packed copy
struct AnyRows {
    Tensor keep;
    void* ptr = nullptr;
    int64_t ld = 0, M = 0;

    explicit AnyRows(const Tensor& x) : keep(x.is_neg() ? x.resolve_neg() : x), ld(x.size(-1)) {
        M = ld ? x.numel() / ld : 0;
        const int64_t width = ld;
        if (!keep.is_contiguous() && (!Rows::any_pitch(keep, &ld) || ld < width)) {
            keep = keep.contiguous();
            ld = width;
        }
        ptr = keep.data_ptr();
    }
};

// a tensor that a node kept, as it was: hooks of saved tensors may give back anything, and storage can be exchanged without a word to autograd
void check_kept(const char* who, const Tensor& t, const Tensor& on, at::ScalarType dt, int64_t numel) {
    if (!t.defined() || t.device() != on.device() || t.scalar_type() != dt || t.numel() != numel || !in_storage(t))
        throw std::runtime_error(std::string(who) + ": what the forward kept was freed, resized or exchanged before the backward");
}

bool route_keeps_logits(const xq_moe_route& q) { return q.scoring != XQ_ROUTE_SOFTMAX || !q.renormalize; }

struct MoeRouteBackward : public Node {
    SavedVariable z_, w_, ids_;
    xq_moe_route q{};                          // without addresses
    std::vector<int64_t> shape;                // of the logits

    std::string name() const override { return "MoeRouteBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        z_.reset_data();
        w_.reset_data();
        ids_.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(1);
        if (!task_should_compute_output(0)) return out;
        const Tensor w = w_.unpack(shared_from_this()), ids = ids_.unpack(shared_from_this());
        const at::ScalarType dt = q.dtype == XQ_DT_F32 ? at::kFloat : at::kBFloat16;
        const int64_t kept = q.n_tokens * q.top_k;
        if (!w.defined() || !w.is_cuda()) throw std::runtime_error("moe_route: what the forward kept was freed, resized or exchanged before the backward");
        c10::DeviceGuard guard(w.device());
        const bool again = at::GradMode::is_enabled();
        refuse_other_streams(*this, w, [](size_t) { return true; }, "moe_route", "weights", "the logits");
        {
            at::NoGradGuard no_grad;
            const Tensor g = grads[0].defined() ? cast_to(grads[0], at::kFloat).contiguous() : at::zeros_like(w, at::MemoryFormat::Contiguous);
            check_kept("moe_route", w, w, at::kFloat, kept);
            check_kept("moe_route", ids, w, at::kLong, kept);
            check_kept("moe_route", g, w, at::kFloat, kept);
            const Tensor wc = w.contiguous(), ic = ids.contiguous();
            xq_moe_route p = q;
            p.ld = p.num_experts;
            std::optional<AnyRows> rows;
            if (route_keeps_logits(q)) {
                const Tensor z = z_.unpack();
                check_kept("moe_route", z, w, dt, q.n_tokens * q.num_experts);
                rows.emplace(z.view(shape));
                p.logits = rows->ptr;
                p.ld = rows->ld;
            }
            out[0] = empty(shape, dt);
            check(xq_moe_route_bwd(&p, (const float*)wc.data_ptr(), (const int64_t*)ic.data_ptr(), (const float*)g.data_ptr(), out[0].data_ptr(), p.num_experts,
                                   stream_of(w)));
        }
        if (again) differentiable_once(out, "moe_route");
        return out;
    }
};

struct EmbeddingBackward : public Node {
    SavedVariable ids_;
    xq_embedding q{};                          // without addresses
    at::ScalarType id_dt = at::kLong;
    c10::Device device{c10::kCUDA, 0};

    std::string name() const override { return "EmbeddingBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        ids_.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(1);
        if (!task_should_compute_output(0)) return out;
        const Tensor ids = ids_.unpack();
        c10::DeviceGuard guard(device);
        if (!grads[0].defined()) grads[0] = input_metadata(0).zeros_like();
        const bool again = at::GradMode::is_enabled();
        refuse_other_streams(*this, grads[0], [](size_t) { return true; }, "embedding", "results", "the weight");
        {
            at::NoGradGuard no_grad;
            const at::ScalarType dt = q.dtype == XQ_DT_F32 ? at::kFloat : at::kBFloat16;
            const Tensor g = cast_to(grads[0], dt);
            check_kept("embedding", ids, g, id_dt, q.n_tokens);
            check_kept("embedding", g, g, dt, q.n_tokens * q.H);
            const AnyRows rows(g);
            const Tensor ic = ids.contiguous();
            xq_embedding p = q;
            p.ids = ic.data_ptr();
            out[0] = empty({q.V, q.H}, dt);
            Scratch ws(xq_embedding_workspace_bytes(q.n_tokens, q.V, q.H));
            check(xq_embedding_bwd(&p, rows.ptr, rows.ld, out[0].data_ptr(), q.H, ws.get(), ws.bytes, stream_of(g)));
        }
        if (again) differentiable_once(out, "embedding");
        return out;
    }
};

// the eleven buffers of xq_grouped_saved that a forward fills, in its order
constexpr int kGroupedKept = 11;
void grouped_saved(xq_grouped_saved* S, const Tensor* kept, const Rows* x) {
    auto p = [&](int i) { return kept[i].numel() ? kept[i].data_ptr() : nullptr; };
    *S = xq_grouped_saved{};
    S->xs = p(0); S->gate_up = p(1); S->h = p(2); S->w_row = (float*)p(3); S->su_gate = p(4); S->su_up = p(5); S->su_down = p(6);
    S->scatter_index = (int32_t*)p(7); S->offsets = (int32_t*)p(8); S->tile_offsets = (int32_t*)p(9); S->counts = (int32_t*)p(10);
    if (x && x->M) { S->x_tokens = const_cast<void*>(x->ptr); S->ld_x_tokens = x->ld; }
}

void grouped_lora(xq_grouped_lora* L, const Tensor* A, const Tensor* B, int r, double scaling, double limit) {
    for (int p = 0; p < 3; ++p) {
        L->A[p] = A[p].data_ptr();
        L->B[p] = B[p].data_ptr();
        L->A_experts[p] = (int32_t)A[p].size(0);
        L->B_experts[p] = (int32_t)B[p].size(0);
    }
    L->dtype = A[0].scalar_type() == at::kFloat ? XQ_DT_F32 : XQ_DT_BF16;
    L->r = r;
    L->scaling = (float)scaling;
    L->swiglu_limit = (float)limit;
}

struct QLoRAMoeBackward : public Node {
    SavedVariable x_, kept_[kGroupedKept], A_[3], B_[3];
    Weight q[3];
    int r = 0;
    int64_t T = 0, topk = 0;
    double scaling = 0, limit = 0;
    at::ScalarType rw_dt = at::kFloat;
    std::vector<int64_t> rw_shape;

    std::string name() const override { return "QLoRAMoeBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        x_.reset_data();
        for (auto& v : kept_) v.reset_data();
        for (auto& v : A_) v.reset_data();
        for (auto& v : B_) v.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(8);                      // x, routing weights, then the factors as above
        if (!grads[0].defined()) grads[0] = input_metadata(0).zeros_like();
        const Tensor x = x_.unpack();
        Tensor kept[kGroupedKept], A[3], B[3];
        for (int i = 0; i < kGroupedKept; ++i) kept[i] = kept_[i].unpack(shared_from_this());
        for (int p = 0; p < 3; ++p) { A[p] = A_[p].unpack(); B[p] = B_[p].unpack(); }
        const int64_t H = q[0].w.rows, I = q[0].w.cols, E = q[0].w.num_experts;
        Tensor dy = cast_to(grads[0], at::kBFloat16);
        c10::DeviceGuard guard(x.device());
        const Rows dr(dy, H), xr(x, H);
        const bool need_dx = task_should_compute_output(0), need_drw = task_should_compute_output(1);
        if (need_dx) out[0] = empty_bf(x.sizes());
        const at::ScalarType kernel_dt = rw_dt == at::kBFloat16 ? at::kBFloat16 : at::kFloat;
        if (need_drw) out[1] = empty(rw_shape, kernel_dt);
        xq_grouped_grads G;
        for (int p = 0; p < 3; ++p) {
            out[2 + 2 * p] = empty_f32(A[p].sizes());
            out[3 + 2 * p] = empty_f32(B[p].sizes());
            G.dA[p] = (float*)out[2 + 2 * p].data_ptr();
            G.dB[p] = (float*)out[3 + 2 * p].data_ptr();
        }
        xq_grouped_lora L;
        grouped_lora(&L, A, B, r, scaling, limit);
        xq_grouped_saved S;
        grouped_saved(&S, kept, &xr);
        Scratch ws(xq_grouped_workspace_bytes(T, (int32_t)topk, (int32_t)E, H, I, r, 1));
        check(xq_grouped_bwd(q[0].now(), q[1].now(), q[2].now(), &L, dr.ptr, dr.ld, T, (int32_t)topk, &S, need_dx ? out[0].data_ptr() : nullptr, H,
                             need_drw ? out[1].data_ptr() : nullptr, kernel_dt == at::kBFloat16 ? XQ_DT_BF16 : XQ_DT_F32, &G, ws.get(),
                             ws.bytes, stream_of(x)));
        if (need_drw) out[1] = cast_to(out[1], rw_dt);
        for (int p = 0; p < 3; ++p) {
            out[2 + 2 * p] = cast_to(out[2 + 2 * p], A[p].scalar_type());
            out[3 + 2 * p] = cast_to(out[3 + 2 * p], B[p].scalar_type());
        }
        return out;
    }
};

// ---- entry points
bool usable_input(const Tensor* x, const Linear& m) {
    return x && x->scalar_type() == at::kBFloat16 && x->dim() >= 1 && x->size(-1) == m.q.w.cols && x->device() == m.q.packed.device() &&
           x->device() == m.A.device();
}

template <typename F>
PyObject* guarded(F&& f) {
    try {
        return f();
    } catch (const ArgError& e) {
        PyErr_SetString(g_error, e.what());
    } catch (const python_error& e) {
        const_cast<python_error&>(e).restore();
    } catch (const std::exception& e) {
        torch::translate_exception_to_python(std::current_exception());
    }
    return nullptr;
}

#define XQ_NONE Py_RETURN_NONE

// linear(module, x)
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 2) { PyErr_SetString(PyExc_TypeError, "linear(module, x)"); return nullptr; }
        const Tensor* x = plain(args[1]);
        Linear m;
        if (under_transform() || !x || !m.read(args[0]) || !usable_input(x, m)) XQ_NONE;
        const int64_t Nf = m.q.w.rows, K = m.q.w.cols;
        const bool train = at::GradMode::is_enabled() && (x->requires_grad() || m.wants_grad());
        if (train && Nf % 64 != 0) XQ_NONE;
        c10::DeviceGuard guard(x->device());
        const Rows xr(*x, K);
        Tensor y = empty_bf(with_last(*x, Nf)), su;
        if (train) su = empty_bf({xr.M, r_pad_of(m.r)});
        Scratch ws(xq_linear_workspace_bytes_fmt(m.q.w.format, xr.M, Nf, K, m.r));
        {
            ReleaseGil nogil;
            check(xq_linear_fwd(&m.q.w, xr.ptr, xr.ld, xr.M, m.A.data_ptr(), m.B.data_ptr(), m.lora_dtype(), m.r, (float)m.scaling, m.bias_ptr(),
                  y.data_ptr(), Nf, train ? su.data_ptr() : nullptr, ws.get(), ws.bytes, stream_of(*x)));
        }
        if (!train) {
            if (!note_decode_forward(*x, xr.M)) return nullptr;
            return THPVariable_Wrap(std::move(y));
        }
        auto node = std::shared_ptr<QLoRALinearBackward>(new QLoRALinearBackward(), torch::autograd::deleteNode);
        const Tensor* bias = m.bias.defined() ? plain(get(get(dict_of(args[0]), N.s__parameters), N.s_bias)) : nullptr;
        node->set_next_edges(torch::autograd::collect_next_edges(*x, m.A, m.B, bias ? *bias : Tensor()));
        node->x_ = SavedVariable(*x, false);
        node->su_ = SavedVariable(su, false);
        node->A_ = SavedVariable(m.A, false);
        node->B_ = SavedVariable(m.B, false);
        if (bias) node->bias_dt = bias->scalar_type();
        node->q = m.q;
        node->r = m.r;
        node->scaling = m.scaling;
        torch::autograd::set_history(y, node);
        return THPVariable_Wrap(std::move(y));
    });
}

// linears(modules, x): up to XQ_LINEAR_MULTI_MAX forwards on one input, nothing differentiated
PyObject* linears(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 2 || !PyList_Check(args[0])) { PyErr_SetString(PyExc_TypeError, "linears([modules], x)"); return nullptr; }
        const Py_ssize_t cnt = PyList_GET_SIZE(args[0]);
        const Tensor* x = plain(args[1]);
        if (under_transform() || !x || cnt < 2 || cnt > XQ_LINEAR_MULTI_MAX) XQ_NONE;
        const bool grad = at::GradMode::is_enabled();
        if (grad && x->requires_grad()) XQ_NONE;
        Linear m[XQ_LINEAR_MULTI_MAX];
        for (Py_ssize_t i = 0; i < cnt; ++i) {
            if (!m[i].read(PyList_GET_ITEM(args[0], i)) || !usable_input(x, m[i]) || (grad && m[i].wants_grad())) XQ_NONE;
            if (m[i].lora_dtype() != m[0].lora_dtype()) XQ_NONE;
        }
        c10::DeviceGuard guard(x->device());
        const Rows xr(*x, m[0].q.w.cols);
        xq_linear_job jobs[XQ_LINEAR_MULTI_MAX];
        Tensor y[XQ_LINEAR_MULTI_MAX];
        for (Py_ssize_t i = 0; i < cnt; ++i) {
            y[i] = empty_bf(with_last(*x, m[i].q.w.rows));
            jobs[i] = xq_linear_job{&m[i].q.w, m[i].A.data_ptr(), m[i].B.data_ptr(), m[i].r, (float)m[i].scaling, m[i].bias_ptr(),
                                    y[i].data_ptr(), m[i].q.w.rows};
        }
        Scratch ws(xq_linear_fwd_multi_workspace_bytes(jobs, (int)cnt, xr.M));
        {
            ReleaseGil nogil;
            check(xq_linear_fwd_multi(jobs, (int)cnt, xr.ptr, xr.ld, xr.M, m[0].lora_dtype(), ws.get(), ws.bytes, stream_of(*x)));
        }
        if (!note_decode_forward(*x, xr.M)) return nullptr;
        PyObject* out = PyList_New(cnt);
        if (!out) return nullptr;
        for (Py_ssize_t i = 0; i < cnt; ++i) PyList_SET_ITEM(out, i, THPVariable_Wrap(std::move(y[i])));
        return out;
    });
}

// mlp(gate, up, down, x)
PyObject* mlp(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 4) { PyErr_SetString(PyExc_TypeError, "mlp(gate, up, down, x)"); return nullptr; }
        const Tensor* x = plain(args[3]);
        if (under_transform() || !x) XQ_NONE;
        Linear m[3];
        for (int p = 0; p < 3; ++p)
            if (!m[p].read(args[p])) XQ_NONE;
        const int64_t I = m[0].q.w.rows, H = m[0].q.w.cols;
        if (!usable_input(x, m[0]) || m[1].q.w.rows != I || m[1].q.w.cols != H || m[2].q.w.rows != H || m[2].q.w.cols != I || H % 64 || I % 64)
            XQ_NONE;
        for (int p = 0; p < 3; ++p)
            if (m[p].r != m[0].r || m[p].scaling != m[0].scaling || m[p].bias_grad || m[p].lora_dtype() != m[0].lora_dtype() ||
                m[p].q.packed.device() != x->device() || m[p].A.device() != x->device())
                XQ_NONE;
        const bool train = at::GradMode::is_enabled() && (x->requires_grad() || m[0].wants_grad() || m[1].wants_grad() || m[2].wants_grad());
        const int r = m[0].r, rp = r_pad_of(r), fmt = shared_format(m[0].q.w, m[1].q.w, m[2].q.w);
        c10::DeviceGuard guard(x->device());
        const Rows xr(*x, H);
        const int64_t M = xr.M;
        Tensor A[3] = {m[0].A, m[1].A, m[2].A}, B[3] = {m[0].B, m[1].B, m[2].B};
        xq_mlp_lora L;
        mlp_lora(&L, A, B, r, m[0].scaling);
        for (int p = 0; p < 3; ++p) L.bias[p] = m[p].bias_ptr();
        Tensor y = empty_bf(x->sizes());
        if (!train) {
            Scratch ws(xq_mlp_infer_workspace_bytes_fmt(fmt, M, H, I, r));
            {
                ReleaseGil nogil;
                check(xq_mlp_fwd_infer(&m[0].q.w, &m[1].q.w, &m[2].q.w, &L, xr.ptr, xr.ld, M, y.data_ptr(), H, ws.get(), ws.bytes, stream_of(*x)));
            }
            if (!note_decode_forward(*x, M)) return nullptr;
            return THPVariable_Wrap(std::move(y));
        }
        Tensor kept[4] = {empty_bf({M, 2 * I}), empty_bf({M, I}), empty_bf({M, 2 * rp}), empty_bf({M, rp})};
        // gate and up in one launch or two: settled once, for this forward and its backward
        const int gu = xq_get_mlp_gate_up_fused() && m[0].q.w.format == XQ_FMT_FP8 && m[1].q.w.format == XQ_FMT_FP8;
        xq_mlp_saved S{kept[0].data_ptr(), kept[1].data_ptr(), kept[2].data_ptr(), kept[3].data_ptr(), gu, 0};
        Scratch ws(xq_mlp_workspace_bytes_fmt(fmt, M, H, I, r, 0));
        {
            ReleaseGil nogil;
            check(xq_mlp_fwd(&m[0].q.w, &m[1].q.w, &m[2].q.w, &L, xr.ptr, xr.ld, M, y.data_ptr(), H, &S, ws.get(), ws.bytes, stream_of(*x)));
        }
        TORCH_CHECK(S.gate_up_fused == gu, "xq_mlp_fwd ran gate and up in form ", S.gate_up_fused, ", asked for ", gu);
        auto node = std::shared_ptr<QLoRAMLPBackward>(new QLoRAMLPBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(*x, A[0], B[0], A[1], B[1], A[2], B[2]));
        node->x_ = SavedVariable(*x, false);
        for (int i = 0; i < 4; ++i) node->kept_[i] = SavedVariable(kept[i], false);
        for (int p = 0; p < 3; ++p) {
            node->A_[p] = SavedVariable(A[p], false);
            node->B_[p] = SavedVariable(B[p], false);
            node->q[p] = m[p].q;
        }
        node->r = r;
        node->gate_up_fused = gu;
        node->scaling = m[0].scaling;
        torch::autograd::set_history(y, node);
        return THPVariable_Wrap(std::move(y));
    });
}

// moe(module, x, routing_weights, selected_experts, streaming): the routed forward; `streaming` asks for the weight-streaming
// form for a handful of tokens and nothing else (None where the call is differentiated or does not fit it)
PyObject* moe(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 5) { PyErr_SetString(PyExc_TypeError, "moe(module, x, routing_weights, selected_experts, streaming)"); return nullptr; }
        const bool streaming = args[4] == Py_True;
        const Tensor *x = plain(args[1]), *rw = plain(args[2]), *sel = plain(args[3]);
        if (under_transform() || !x || !rw || !sel) XQ_NONE;
        PyObject* d = dict_of(args[0]);
        PyObject *params = get(d, N.s__parameters), *bufs = get(d, N.s__buffers), *sdt = get(d, N.s__scale_dtypes);
        PyObject* impl = get(d, N.s_moe_implementation);
        const int fmt = format_code(get(d, N.s_quant_format));
        int64_t rank, group, E, local, H, I;
        double alpha, limit = 0;
        if (!params || !bufs || !sdt || !PyDict_Check(sdt) || fmt < 0 || !as_defined(args[0], d, g_experts[fmt]) || !impl || !PyUnicode_Check(impl) ||
            PyUnicode_CompareWithASCIIString(impl, "eager") == 0 || !get_int(d, N.s_active_r, &rank) ||
            !get_number(d, N.s_active_lora_alpha, &alpha) || !get_int(d, N.s_quant_group_size, &group) || !get_int(d, N.s_num_experts, &E) ||
            !get_int(d, N.s_num_local_experts, &local) || local != E || !get_int(d, N.s_hidden_size, &H) ||
            !get_int(d, N.s_intermediate_size, &I) || rank < 1 || rank > 64)
            XQ_NONE;
        if (!get_number(d, N.s_swiglu_limit, &limit)) XQ_NONE;
        PyObject* rs = get(d, N.s_use_rslora);
        if (rs != Py_True && rs != Py_False) XQ_NONE;
        const double scaling = rs == Py_True ? alpha / std::sqrt((double)rank) : alpha / (double)rank;
        if (limit < 0) limit = 0;

        PyObject* const proj[3] = {N.s_gate, N.s_up, N.s_down};
        PyObject* const packed[3] = {N.s_gate_packed, N.s_up_packed, N.s_down_packed};
        PyObject* const bscales[3] = {N.s_gate_block_scales, N.s_up_block_scales, N.s_down_block_scales};
        PyObject* const scales[3] = {N.s_gate_scales, N.s_up_scales, N.s_down_scales};
        PyObject* const gscale[3] = {N.s_gate_global_scale, N.s_up_global_scale, N.s_down_global_scale};
        PyObject* const fA[3] = {N.s_gate_proj_lora_A, N.s_up_proj_lora_A, N.s_down_proj_lora_A};
        PyObject* const fB[3] = {N.s_gate_proj_lora_B, N.s_up_proj_lora_B, N.s_down_proj_lora_B};
        Weight q[3];
        Tensor A[3], B[3];
        bool factor_grad = false;
        for (int p = 0; p < 3; ++p) {
            PyObject* dts = get(sdt, proj[p]);
            if (!dts || !PyDict_Check(dts)) XQ_NONE;
            const bool blocks = fmt == XQ_FMT_FP8 || fmt == XQ_FMT_NVFP4;
            const int64_t K = p == 2 ? I : H, Nf = p == 2 ? H : I;
            if (!q[p].fill(fmt, XQ_LAYOUT_GKN, K, Nf, group, E, get(bufs, packed[p]), get(bufs, blocks ? bscales[p] : scales[p]),
                           get(dts, blocks ? N.s_weight_block_scales : N.s_weight_scales), get(bufs, gscale[p]),
                           get(dts, N.s_weight_global_scale)))
                XQ_NONE;
            const Tensor *a = plain(get(params, fA[p])), *b = plain(get(params, fB[p]));
            if (!a) a = plain(get(bufs, fA[p]));           // a projection that is not a LoRA target holds frozen zero factors
            if (!b) b = plain(get(bufs, fB[p]));
            if (!a || !b || a->dim() != 3 || b->dim() != 3 || a->size(2) != rank || b->size(1) != rank || a->size(1) != K || b->size(2) != Nf ||
                !a->is_contiguous() || !b->is_contiguous() || (a->scalar_type() != at::kFloat && a->scalar_type() != at::kBFloat16) ||
                a->scalar_type() != b->scalar_type() || q[p].packed.device() != x->device() || a->device() != x->device())
                XQ_NONE;
            A[p] = *a;
            B[p] = *b;
            if (A[p].scalar_type() != A[0].scalar_type()) XQ_NONE;
            factor_grad = factor_grad || a->requires_grad() || b->requires_grad();
        }
        if (x->scalar_type() != at::kBFloat16 || x->dim() < 1 || x->size(-1) != H || sel->dim() < 1) XQ_NONE;
        const int64_t topk = sel->size(-1);
        if (rw->scalar_type() != at::kFloat && rw->scalar_type() != at::kBFloat16) XQ_NONE;
        if (sel->scalar_type() != at::kLong && sel->scalar_type() != at::kInt) XQ_NONE;
        c10::DeviceGuard guard(x->device());
        const Rows xr(*x, H);
        const int64_t T = xr.M;
        if (topk < 1 || T < 1 || sel->numel() != T * topk || rw->numel() != T * topk || (uintptr_t)xr.ptr % 16 ||
            rw->device() != x->device() || sel->device() != x->device())
            XQ_NONE;
        const int r = (int)rank, rp = r_pad_of(r);
        const bool train = at::GradMode::is_enabled() && (x->requires_grad() || rw->requires_grad() || factor_grad);
        if (streaming && (train || !xq_grouped_infer_supported(&q[0].w, &q[1].w, &q[2].w, T, (int32_t)topk, r) || !xq_grouped_infer_shorter(&q[0].w, T, (int32_t)topk)))
            XQ_NONE;
        Tensor ids = sel->is_contiguous() ? *sel : sel->detach().contiguous();       // 64-bit ids as they are: a conversion would be a launch
        const int id_bytes = (int)ids.element_size();
        Tensor w = rw->is_contiguous() ? *rw : rw->detach().contiguous();
        const int rw_code = w.scalar_type() == at::kFloat ? XQ_DT_F32 : XQ_DT_BF16;
        xq_grouped_lora L;
        grouped_lora(&L, A, B, r, scaling, limit);
        Tensor out = empty_bf(x->sizes());
        void* stream = stream_of(*x);
        if (streaming) {
            Scratch ws(xq_grouped_infer_workspace_bytes(T, (int32_t)topk, (int32_t)E, H, I, r));
            {
                ReleaseGil nogil;
                check(xq_grouped_fwd_infer_ids(&q[0].w, &q[1].w, &q[2].w, &L, xr.ptr, xr.ld, T, w.data_ptr(), rw_code, ids.data_ptr(), id_bytes,
                      (int32_t)topk, out.data_ptr(), H, ws.get(), ws.bytes, stream));
            }
            return THPVariable_Wrap(std::move(out));
        }
        const int64_t R = T * topk;
        // where the banks allow it the routed rows are read in place: no [R, H] copy is kept for the backward
        const bool in_place = xq_grouped_in_place(&q[0].w, &q[1].w, &q[2].w);
        auto i32 = [](int64_t c) { return empty({c}, at::kInt); };
        Tensor kept[kGroupedKept] = {in_place ? empty_bf({0, H}) : empty_bf({R, H}), empty_bf({R, 2 * I}), empty_bf({R, I}), empty_f32({R}),
                                     empty_bf({R, rp}), empty_bf({R, rp}), empty_bf({R, rp}), i32(R), i32(E + 1), i32(2 * (E + 1)), i32(E)};
        xq_grouped_saved S;
        grouped_saved(&S, kept, nullptr);
        Scratch ws(xq_grouped_workspace_bytes(T, (int32_t)topk, (int32_t)E, H, I, r, 0));
        {
            ReleaseGil nogil;
            check((train ? xq_grouped_fwd_ids : xq_grouped_fwd_eval_ids)(&q[0].w, &q[1].w, &q[2].w, &L, xr.ptr, xr.ld, T, w.data_ptr(), rw_code,
                  ids.data_ptr(), id_bytes, (int32_t)topk, out.data_ptr(), H, &S, ws.get(), ws.bytes, stream));
        }
        if (!train) return THPVariable_Wrap(std::move(out));
        auto node = std::shared_ptr<QLoRAMoeBackward>(new QLoRAMoeBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(*x, *rw, A[0], B[0], A[1], B[1], A[2], B[2]));
        node->x_ = SavedVariable(*x, false);
        for (int i = 0; i < kGroupedKept; ++i) node->kept_[i] = SavedVariable(kept[i], false);
        for (int p = 0; p < 3; ++p) {
            node->A_[p] = SavedVariable(A[p], false);
            node->B_[p] = SavedVariable(B[p], false);
            node->q[p] = q[p];
        }
        node->r = r;
        node->T = T;
        node->topk = topk;
        node->scaling = scaling;
        node->limit = limit;
        node->rw_dt = rw->scalar_type();
        node->rw_shape.assign(rw->sizes().begin(), rw->sizes().end());
        torch::autograd::set_history(out, node);
        return THPVariable_Wrap(std::move(out));
    });
}

// cross_entropy(x, weight, labels, ignore_index, reduction, logit_scale)
PyObject* cross_entropy(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 6) { PyErr_SetString(PyExc_TypeError, "cross_entropy(x, weight, labels, ignore_index, reduction, logit_scale)"); return nullptr; }
        // (numbers first: their conversion may run Python, and with it change the tensors)
        const int64_t ignore = PyLong_AsLongLong(args[3]);
        if (ignore == -1 && PyErr_Occurred()) { PyErr_Clear(); XQ_NONE; }
        const long reduction = PyLong_AsLong(args[4]);
        const double scale = PyFloat_AsDouble(args[5]);
        if (PyErr_Occurred()) { PyErr_Clear(); XQ_NONE; }
        const Tensor *x = plain(args[0]), *w = plain(args[1]), *labels = plain(args[2]);
        if (under_transform() || !x || !w || !labels || !HeadLoss::takes(*x, *w, *labels)) XQ_NONE;
        if (!(scale > 0.0) || !std::isfinite(scale)) XQ_NONE;
        const bool grad = at::GradMode::is_enabled(), want_x = grad && x->requires_grad(), want_w = grad && w->requires_grad();
        const int keep = want_x ? XQ_LCE_KEEP_DX : want_w ? XQ_LCE_KEEP_HEAD : XQ_LCE_KEEP_NONE;
        c10::DeviceGuard guard(x->device());
        Tensor loss, saved;
        {
            at::NoGradGuard no_grad;
            const HeadLoss h(*x, *w, *labels, ignore, (int)reduction, scale);
            loss = reduction == XQ_LCE_NONE ? empty_f32(labels->sizes()) : empty_f32({});
            saved = empty({xq_lce_saved_bytes(h.q.M, h.q.V, h.q.H, keep)}, at::kByte);
            Scratch ws(xq_lce_workspace_bytes(h.q.M, h.q.V, h.q.H, keep));
            void* stream = stream_of(*x);
            ReleaseGil nogil;
            check(xq_lce_fwd(&h.q, (float*)loss.data_ptr(), saved.data_ptr(), keep, ws.get(), ws.bytes, stream));
        }
        if (!keep) return THPVariable_Wrap(std::move(loss));
        auto node = std::shared_ptr<LinearCrossEntropyBackward>(new LinearCrossEntropyBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(*x, *w));
        node->x_ = SavedVariable(*x, false);
        node->w_ = SavedVariable(*w, false);
        node->labels_ = SavedVariable(*labels, false);
        node->saved_ = SavedVariable(saved, false);
        node->ignore = ignore;
        node->reduction = (int)reduction;
        node->keep = keep;
        node->scale = scale;
        node->saved_bytes = nbytes(saved); node->M = x->numel() / x->size(-1); node->V = w->size(0); node->H = w->size(1);
        torch::autograd::set_history(loss, node);
        return THPVariable_Wrap(std::move(loss));
    });
}

// the numbers of a call, which come before its tensors: their conversion may run Python, and with it change those
bool as_int(PyObject* o, int64_t* v) {
    if (!PyLong_Check(o)) return false;
    *v = PyLong_AsLongLong(o);
    if (*v == -1 && PyErr_Occurred()) { PyErr_Clear(); return false; }
    return true;
}
bool as_number(PyObject* o, double* v) {
    if (!PyFloat_Check(o) && !PyLong_Check(o)) return false;
    *v = PyFloat_AsDouble(o);
    if (*v == -1.0 && PyErr_Occurred()) { PyErr_Clear(); return false; }
    return true;
}

// moe_route(logits, bias or None, top_k, scoring, num_groups, top_groups, group_score, renormalize, scale)
PyObject* moe_route(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 9) { PyErr_SetString(PyExc_TypeError, "moe_route(9 arguments)"); return nullptr; }
        int64_t k, scoring, groups, top_groups, group_score;
        double scale;
        if (!as_int(args[2], &k) || !as_int(args[3], &scoring) || !as_int(args[4], &groups) || !as_int(args[5], &top_groups) || !as_int(args[6], &group_score) ||
            !as_number(args[8], &scale))
            XQ_NONE;
        const Tensor *z = plain(args[0]), *bias = args[1] == Py_None ? nullptr : plain(args[1]);
        if (under_transform() || !z || (args[1] != Py_None && !bias) || z->dim() < 1 || z->is_neg() || (z->scalar_type() != at::kFloat && z->scalar_type() != at::kBFloat16))
            XQ_NONE;
        const int64_t E = z->size(-1);
        if (E < 1 || E > 1024 || scoring < 0 || group_score < 0 || groups < 1 || groups > 64 || E % groups || top_groups < 1 || top_groups > groups || k < 1 || k > 32 ||
            k > E / groups * top_groups || !(scale >= 0x1p-60 && scale <= 0x1p60))
            XQ_NONE;
        if (bias && (bias->scalar_type() != at::kFloat || bias->dim() != 1 || bias->size(0) != E || bias->device() != z->device() || bias->is_neg())) XQ_NONE;
        check_held("moe_route", {z, bias});
        const bool grad = at::GradMode::is_enabled() && z->requires_grad();
        c10::DeviceGuard guard(z->device());
        Tensor weights, ids;
        xq_moe_route q{};
        q.dtype = z->scalar_type() == at::kFloat ? XQ_DT_F32 : XQ_DT_BF16;
        q.num_experts = (int32_t)E; q.top_k = (int32_t)k; q.scoring = (int32_t)scoring; q.num_groups = (int32_t)groups; q.top_groups = (int32_t)top_groups;
        q.group_score = (int32_t)group_score; q.renormalize = args[7] == Py_True; q.scale = (float)scale;
        {
            at::NoGradGuard no_grad;
            const AnyRows rows(*z);
            const Tensor b = bias ? bias->contiguous() : Tensor();
            weights = empty_f32(with_last(*z, k));
            ids = empty(with_last(*z, k), at::kLong);
            q.n_tokens = rows.M;
            xq_moe_route p = q;
            p.logits = rows.ptr; p.ld = rows.ld; p.bias = bias ? (const float*)b.data_ptr() : nullptr;
            void* stream = stream_of(*z);
            ReleaseGil nogil;
            check(xq_moe_route_fwd(&p, (float*)weights.data_ptr(), (int64_t*)ids.data_ptr(), stream));
        }
        if (grad) {
            auto node = std::shared_ptr<MoeRouteBackward>(new MoeRouteBackward(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(*z));
            if (route_keeps_logits(q)) node->z_ = SavedVariable(*z, false);
            node->ids_ = SavedVariable(ids, false);
            node->q = q;
            node->shape.assign(z->sizes().begin(), z->sizes().end());
            torch::autograd::set_history(weights, node);
            node->w_ = SavedVariable(weights, true);
        }
        PyObject *w = THPVariable_Wrap(std::move(weights)), *i = THPVariable_Wrap(std::move(ids));
        PyObject* out = w && i ? PyTuple_Pack(2, w, i) : nullptr;
        Py_XDECREF(w);
        Py_XDECREF(i);
        return out;
    });
}

// adapters(base, x, A, B, ids, scalings, in place)
PyObject* adapters(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 7) { PyErr_SetString(PyExc_TypeError, "adapters(base, x, A, B, ids, scalings, in_place)"); return nullptr; }
        const Tensor *base = plain(args[0]), *x = plain(args[1]), *A = plain(args[2]), *B = plain(args[3]), *ids = plain(args[4]), *s = plain(args[5]);
        if (under_transform() || !base || !x || !A || !B || !ids || !s) XQ_NONE;
        const bool in_place = args[6] == Py_True;
        for (const Tensor* t : {base, x, A, B, s})
            if ((at::GradMode::is_enabled() && t->requires_grad()) || t->is_neg()) XQ_NONE;
        if (base->scalar_type() != at::kBFloat16 || x->scalar_type() != at::kBFloat16 || A->scalar_type() != B->scalar_type() || s->scalar_type() != at::kFloat ||
            (A->scalar_type() != at::kFloat && A->scalar_type() != at::kBFloat16) || (ids->scalar_type() != at::kInt && ids->scalar_type() != at::kLong) || ids->is_neg())
            XQ_NONE;
        if (x->dim() < 1 || base->dim() != x->dim() || A->dim() != 3 || B->dim() != 3 || s->dim() != 1 || ids->dim() != x->dim() - 1) XQ_NONE;
        const int64_t K = x->size(-1), N = base->size(-1), a = A->size(0), r = A->size(1);
        if (K < 64 || K % 64 || N < 16 || N % 16 || r < 1 || r > 64 || A->size(2) != K || B->size(0) != a || B->size(1) != N || B->size(2) != r || s->size(0) != a ||
            a >= (1ll << 31))
            XQ_NONE;
        const auto lead = x->sizes().slice(0, x->dim() - 1);
        if (lead != base->sizes().slice(0, base->dim() - 1) || lead != ids->sizes()) XQ_NONE;
        for (const Tensor* t : {base, A, B, ids, s})
            if (t->device() != x->device()) XQ_NONE;
        check_held("lora_adapters", {base, x, A, B, ids, s});
        auto aligned = [](const Tensor& t) { return (uintptr_t)t.data_ptr() % 16 == 0; };
        // (rows and factors that have to be copied first, and a base that cannot be written, are the Python path's)
        int64_t ldx = K, ldb = N;
        if (!A->is_contiguous() || !B->is_contiguous() || !s->is_contiguous() || !ids->is_contiguous() || !aligned(*A) || !aligned(*B) || !aligned(*x) || !aligned(*base) ||
            (!x->is_contiguous() && (!Rows::pitched(*x, &ldx) || ldx < K)) || (!base->is_contiguous() && (!Rows::pitched(*base, &ldb) || ldb < N)))
            XQ_NONE;
        c10::DeviceGuard guard(x->device());
        xq_adapters q{};
        q.M = x->numel() / K; q.N = N; q.K = K;
        q.x = x->data_ptr(); q.ldx = ldx; q.base = base->data_ptr(); q.ld_base = ldb;
        q.A = A->data_ptr(); q.B = B->data_ptr(); q.scaling = (const float*)s->data_ptr(); q.ids = ids->data_ptr();
        q.n_adapters = (int32_t)a; q.r = (int32_t)r; q.factor_dtype = A->scalar_type() == at::kFloat ? XQ_DT_F32 : XQ_DT_BF16; q.id_bytes = (int32_t)ids->element_size();
        Tensor out = in_place ? *base : empty_bf(base->sizes());
        q.out = out.data_ptr(); q.ld_out = in_place ? ldb : N;
        if (in_place) {                                     // nothing else that is read may lie in what is written
            auto end = [](const Tensor& t) {
                int64_t last = 0;
                for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
                return (const char*)t.data_ptr() + (t.numel() ? (last + 1) * (int64_t)t.element_size() : 0);
            };
            for (const Tensor* t : {x, A, B, ids, s})
                if ((const char*)t->data_ptr() < end(out) && (const char*)out.data_ptr() < end(*t)) XQ_NONE;
        }
        Scratch ws(xq_adapters_workspace_bytes(q.M, N, K, (int)r));
        {
            void* stream = stream_of(*x);
            ReleaseGil nogil;
            check(xq_adapters_add(&q, ws.get(), ws.bytes, stream));
        }
        if (in_place && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
        return THPVariable_Wrap(std::move(out));
    });
}

// embedding(ids, weight, scale, padding_idx or None)
PyObject* embedding(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 4) { PyErr_SetString(PyExc_TypeError, "embedding(ids, weight, scale, padding_idx)"); return nullptr; }
        double scale;
        int64_t pad = -1;
        if (!as_number(args[2], &scale) || (args[3] != Py_None && !as_int(args[3], &pad))) XQ_NONE;
        const Tensor *ids = plain(args[0]), *w = plain(args[1]);
        if (under_transform() || !ids || !w || w->dim() != 2 || w->size(0) < 1 || w->size(1) < 1 || (w->scalar_type() != at::kFloat && w->scalar_type() != at::kBFloat16) ||
            (ids->scalar_type() != at::kInt && ids->scalar_type() != at::kLong) || ids->device() != w->device() || w->is_neg() || ids->is_neg())
            XQ_NONE;
        const int64_t V = w->size(0), H = w->size(1);
        if (args[3] != Py_None) {
            if (pad < -V || pad >= V) XQ_NONE;
            if (pad < 0) pad += V;
        }
        if (!(std::fabs(scale) <= 3.4e38)) XQ_NONE;
        check_held("embedding", {ids, w});
        const bool grad = at::GradMode::is_enabled() && w->requires_grad();
        c10::DeviceGuard guard(w->device());
        Tensor out;
        xq_embedding q{};
        q.n_tokens = ids->numel(); q.V = V; q.H = H; q.padding_idx = pad; q.scale = (float)scale;
        q.dtype = w->scalar_type() == at::kFloat ? XQ_DT_F32 : XQ_DT_BF16; q.id_bytes = (int32_t)ids->element_size();
        {
            at::NoGradGuard no_grad;
            const Tensor i = ids->contiguous();
            const AnyRows rows(*w);
            std::vector<int64_t> shape(ids->sizes().begin(), ids->sizes().end());
            shape.push_back(H);
            out = empty(shape, w->scalar_type());
            xq_embedding p = q;
            p.ids = i.data_ptr(); p.weight = rows.ptr; p.ldw = rows.ld;
            void* stream = stream_of(*w);
            ReleaseGil nogil;
            check(xq_embedding_fwd(&p, out.data_ptr(), H, stream));
        }
        if (grad) {
            auto node = std::shared_ptr<EmbeddingBackward>(new EmbeddingBackward(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(*w));
            node->ids_ = SavedVariable(*ids, false);
            node->q = q;
            node->id_dt = ids->scalar_type();
            node->device = w->device();
            torch::autograd::set_history(out, node);
        }
        return THPVariable_Wrap(std::move(out));
    });
}

// ---- the optimizer step: its arguments are hundreds of tensors, whose addresses and checks are a matter of tens of microseconds here
// (a tuple of its own: the caller's list may change while this call converts a number of a user's class or has let go of the GIL, and with it go
// the tensors)
struct TensorList {
    const char* name;
    PyObject* seq = nullptr;
    TensorList(const char* n, PyObject* o) : name(n) {
        if (o == Py_None) return;
        seq = PySequence_Tuple(o);
        if (!seq) { PyErr_Clear(); throw ArgError(std::string("adamw_step: ") + n + " must be a list of tensors"); }
    }
    ~TensorList() { Py_XDECREF(seq); }
    TensorList(const TensorList&) = delete;
    Py_ssize_t size() const { return PyTuple_GET_SIZE(seq); }
    std::string at(Py_ssize_t i) const { return std::string("adamw_step: ") + name + "[" + std::to_string(i) + "]"; }
    const Tensor& operator[](Py_ssize_t i) const {
        PyObject* o = PyTuple_GET_ITEM(seq, i);
        if (!THPVariable_Check(o)) throw ArgError(at(i) + " is not a tensor");
        const Tensor& t = THPVariable_Unpack(o);
        if (!t.defined() || t.layout() != at::kStrided || at::isTensorSubclassLike(t)) throw ArgError(at(i) + " is not a plain dense tensor");
        if (!t.is_cuda()) throw std::runtime_error(at(i) + ": xorl_amd kernels run on a HIP device only; got a tensor on " + t.device().str() + " (there is no CPU fallback)");
        return t;
    }
};

int float_code(const Tensor& t, const TensorList& l, Py_ssize_t i) {
    if (t.scalar_type() == at::kFloat) return XQ_DT_F32;
    if (t.scalar_type() == at::kBFloat16) return XQ_DT_BF16;
    throw ArgError(l.at(i) + " must be fp32 or bf16, got " + toString(t.scalar_type()));
}

// adamw(params, grads, exp_avgs, exp_avg_sqs, steps, exp_avg_scales or None, exp_avg_sq_scales or None, (lr, beta1, beta2, eps, weight_decay),
//       lr tensor or None, max_norm or None, norm or None) -> the norm, or None.  params None: the norm of grads alone.
PyObject* adamw(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        if (n_args != 11) { PyErr_SetString(PyExc_TypeError, "adamw(11 arguments)"); return nullptr; }
        const TensorList p("params", args[0]), g("grads", args[1]), m("exp_avgs", args[2]), v("exp_avg_sqs", args[3]), t("steps", args[4]),
            ms("exp_avg_scales", args[5]), vs("exp_avg_sq_scales", args[6]);
        const bool norm_only = !p.seq, eight = ms.seq || vs.seq;
        if (!g.seq) throw ArgError("adamw_step: grads must be a list of tensors");
        const Py_ssize_t n = g.size();
        if (!norm_only) {
            for (const TensorList* l : {&p, &m, &v, &t})
                if (!l->seq || l->size() != n) throw ArgError(std::string("adamw_step: ") + l->name + " and grads differ in length");
            if (eight && (!ms.seq || !vs.seq || ms.size() != n || vs.size() != n))
                throw ArgError("adamw_step: 8-bit states need exp_avg_scales and exp_avg_sq_scales, one for each tensor");
        }
        xq_adamw_options o{};
        if (!norm_only && !PyArg_ParseTuple(args[7], "ddddd", &o.lr, &o.beta1, &o.beta2, &o.eps, &o.weight_decay)) return nullptr;
        o.state_bits = eight ? 8 : 32;
        if (args[9] != Py_None) {          // (before an address is taken: this may run Python)
            o.max_norm = PyFloat_AsDouble(args[9]);
            if (o.max_norm == -1.0 && PyErr_Occurred()) return nullptr;
        }
        std::optional<at::Device> device;
        auto same_device = [&](const Tensor& a, auto&& what) {
            if (!device) device = a.device();
            else if (a.device() != *device) throw ArgError(what() + " is on " + a.device().str() + ", others on " + device->str());
        };
        std::vector<xq_adamw_tensor> q;
        std::vector<Tensor> keep, empty_steps;    // (step counts of tensors without elements, of which the kernels hear nothing)
        std::vector<at::TensorImpl*> written;     // (the tuples hold them)
        struct Span { const char *from, *to; bool write; };
        std::vector<Span> once;        // what the step writes and what it reads all along: written twice, or read where another block writes, the result would hang on the order
        auto note = [&](const Tensor& t, bool write = true) { once.push_back({(const char*)t.data_ptr(), (const char*)t.data_ptr() + nbytes(t), write}); };
        q.reserve(n);
        written.reserve(6 * n);
        once.reserve(7 * n);
        for (Py_ssize_t i = 0; i < n; ++i) {
            const Tensor& gr = g[i];
            xq_adamw_tensor a{};
            a.numel = gr.numel();
            a.grad_dtype = float_code(gr, g, i);
            same_device(gr, [&] { return g.at(i); });
            a.grad = gr.data_ptr();
            if (!gr.is_contiguous() || gr.is_neg()) {
                keep.push_back(gr.detach().resolve_neg().contiguous());
                a.grad = keep.back().data_ptr();
            }
            if (!norm_only) {
                const Tensor &pt = p[i], &mt = m[i], &vt = v[i], &st = t[i];
                a.param_dtype = float_code(pt, p, i);
                if (pt.sizes() != gr.sizes()) throw ArgError(g.at(i) + " has another shape than its parameter");
                struct { const Tensor& t; const TensorList& l; at::ScalarType dt; int64_t n; } all[] = {
                    {pt, p, pt.scalar_type(), a.numel}, {mt, m, eight ? at::kChar : at::kFloat, a.numel},
                    {vt, v, eight ? at::kByte : at::kFloat, a.numel}, {st, t, at::kFloat, 1}};
                for (const auto& c : all) {
                    same_device(c.t, [&] { return c.l.at(i); });
                    if (c.t.scalar_type() != c.dt) throw ArgError(c.l.at(i) + " must be " + toString(c.dt) + ", got " + toString(c.t.scalar_type()));
                    if (c.t.numel() != c.n) throw ArgError(c.l.at(i) + " holds " + std::to_string(c.t.numel()) + " elements, expected " + std::to_string(c.n));
                    if (!c.t.is_contiguous() || c.t.is_neg()) throw ArgError(c.l.at(i) + " must be contiguous");
                }
                a.param = pt.data_ptr(); a.exp_avg = mt.data_ptr(); a.exp_avg_sq = vt.data_ptr(); a.step = (float*)st.data_ptr();
                if (eight) {
                    float** to[] = {&a.exp_avg_scale, &a.exp_avg_sq_scale};
                    const TensorList* from[] = {&ms, &vs};
                    for (int k = 0; k < 2; ++k) {
                        const Tensor& sc = (*from[k])[i];
                        same_device(sc, [&] { return from[k]->at(i); });
                        if (sc.scalar_type() != at::kFloat || !sc.is_contiguous() || sc.numel() != (a.numel + 255) / 256)
                            throw ArgError(from[k]->at(i) + " must be contiguous fp32 with " + std::to_string((a.numel + 255) / 256) + " element(s)");
                        *to[k] = (float*)sc.data_ptr();
                        written.push_back(sc.unsafeGetTensorImpl());
                        if (a.numel) note(sc);
                    }
                }
                for (const Tensor* w : {&pt, &mt, &vt}) {
                    written.push_back(w->unsafeGetTensorImpl());
                    if (a.numel) note(*w);
                }
                written.push_back(st.unsafeGetTensorImpl());
                note(st);
                if (a.numel && a.grad == gr.data_ptr()) note(gr, false);
                if (!a.numel) empty_steps.push_back(st);
            }
            if (a.numel) q.push_back(a);
        }
        if (args[8] != Py_None) {
            const Tensor* lr = plain(args[8]);
            if (!lr || lr->scalar_type() != at::kFloat || lr->numel() != 1) throw ArgError("adamw_step: an lr tensor must be one fp32 element on the device");
            same_device(*lr, [] { return std::string("adamw_step: lr"); });
            o.lr_device = (const float*)lr->data_ptr();
            note(*lr, false);
        }
        Tensor norm;
        if (args[10] != Py_None) {
            const Tensor* given = plain(args[10]);
            if (!given || given->scalar_type() != at::kFloat || given->numel() != 1) throw ArgError("adamw_step: grad_norm must be one fp32 element on the device");
            same_device(*given, [] { return std::string("adamw_step: grad_norm"); });
            norm = *given;
            o.norm_given = 1;
            note(norm, false);
        }
        std::sort(once.begin(), once.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
        const char *read_to = nullptr, *written_to = nullptr;         // the ends of what came before
        for (const Span& a : once) {
            if (a.from < written_to || (a.write && a.from < read_to)) throw ArgError("adamw_step: two tensors share memory of a parameter, a state or a step count");
            const char*& to = a.write ? written_to : read_to;
            to = std::max(to, a.to);
        }
        if (args[9] == Py_None && o.norm_given) throw ArgError("adamw_step: grad_norm without max_norm");
        if (!device) {
            if (norm_only || args[9] != Py_None) throw ArgError("adamw_step: a norm over no gradients has no device");
            Py_RETURN_NONE;
        }
        c10::DeviceGuard guard(*device);
        if (!norm.defined() && (norm_only || args[9] != Py_None)) norm = empty_f32({});
        if (norm.defined()) o.norm = (float*)norm.data_ptr();
        void* stream = (void*)c10::hip::getCurrentHIPStream(device->index()).stream();
        Scratch ws(xq_adamw_workspace_bytes((int64_t)q.size()));
        {
            ReleaseGil nogil;
            check(norm_only ? xq_grad_norm(q.data(), (int64_t)q.size(), o.norm, ws.get(), ws.bytes, stream)
                            : xq_adamw_step(q.data(), (int64_t)q.size(), &o, ws.get(), ws.bytes, stream));
        }
        if (!empty_steps.empty()) {
            at::AutoDispatchBelowADInplaceOrView below;
            at::_foreach_add_(empty_steps, 1);
        }
        for (at::TensorImpl* w : written)
            if (!w->is_inference()) w->bump_version();
        if (!norm.defined()) Py_RETURN_NONE;
        return THPVariable_Wrap(std::move(norm));
    });
}

// {format: (class, ((method name, method), ...))} -> programs by format
bool fill_programs(PyObject* table, Program* out) {
    PyObject *key, *entry;
    for (Py_ssize_t at = 0; PyDict_Next(table, &at, &key, &entry);) {
        const int fmt = format_code(key);
        PyObject *type, *methods;
        if (fmt < 0 || !PyArg_ParseTuple(entry, "O!O!", &PyType_Type, &type, &PyTuple_Type, &methods)) return false;
        Program p;
        p.type = (PyTypeObject*)type;
        for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(methods); ++i) {
            PyObject *name, *method;
            if (!PyArg_ParseTuple(PyTuple_GET_ITEM(methods, i), "UO", &name, &method)) return false;
            Py_INCREF(name);
            PyUnicode_InternInPlace(&name);
            Py_INCREF(method);
            p.name.push_back(name);
            p.method.push_back(method);
        }
        Py_INCREF(type);
        out[fmt] = p;
    }
    return true;
}

// init(XqError, dict of xorl_amd.functional, programs of the linear modules, programs of the expert modules)
PyObject* init(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 4 || !PyDict_Check(args[1]) || !PyDict_Check(args[2]) || !PyDict_Check(args[3]) || !fill_programs(args[2], g_linear) ||
        !fill_programs(args[3], g_experts)) {
        PyErr_SetString(PyExc_TypeError, "init(error class, dict, linear programs, expert programs)");
        return nullptr;
    }
    for (Py_ssize_t i = 0; i < 2; ++i) Py_INCREF(args[i]);
    g_error = args[0];
    g_functional = args[1];
#define XQ_INTERN(m) N.s_##m = PyUnicode_InternFromString(#m);
    XQ_NAMES(XQ_INTERN)
#undef XQ_INTERN
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"init", (PyCFunction)(void (*)())init, METH_FASTCALL, nullptr},
    {"linear", (PyCFunction)(void (*)())linear, METH_FASTCALL, nullptr},
    {"linears", (PyCFunction)(void (*)())linears, METH_FASTCALL, nullptr},
    {"mlp", (PyCFunction)(void (*)())mlp, METH_FASTCALL, nullptr},
    {"moe", (PyCFunction)(void (*)())moe, METH_FASTCALL, nullptr},
    {"cross_entropy", (PyCFunction)(void (*)())cross_entropy, METH_FASTCALL, nullptr},
    {"moe_route", (PyCFunction)(void (*)())moe_route, METH_FASTCALL, nullptr},
    {"adapters", (PyCFunction)(void (*)())adapters, METH_FASTCALL, nullptr},
    {"embedding", (PyCFunction)(void (*)())embedding, METH_FASTCALL, nullptr},
    {"adamw", (PyCFunction)(void (*)())adamw, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "xq_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_xq_torch() { return PyModule_Create(&module_def); }
