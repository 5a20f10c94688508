// The window and cache calls in one step from Python to libkfa.so, for tensors that need nothing but the launch.
//
// A decoding step or a small training step lasts a few microseconds on the GPU and many times that in the interpreter:
// checks, records, allocations, and a Python function in the backward thread.  Each function here does what its public
// namesake does where the arguments are plain and already have the form the kernels address; for anything else, and for
// every error, it returns None having done nothing, and the Python code takes the call from the beginning (and raises, or
// copies, or pads).  The module is optional: without it (no torch headers at build time) Python serves every call.
//
//   bind(addresses, raise_error)   entry points of libkfa.so by name; raise_error(code) raises what a code means
//   allow(device index)            the device has been checked by the Python layer
//   window_attention(q, k, v, window, sinks, query_start, scale)      -> O, with a graph node in C++, or None
//   cache_write(cache, k, v, start, lengths)                          -> True or None
//   cache_read(cache, start, length)                                  -> (K, V) or None
//   cache_attention(q, cache, query_start, window, sinks, scale)      -> O or None
//   torch_version                  of the torch whose headers it was built with, the only one it may be used with
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TensorSubclassLikeUtils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <atomic>
#include <cfloat>
#include <cmath>
#include <cstring>
#include <initializer_list>
#include <memory>
#include <optional>
#include <vector>

#include "../../include/kfa.h"

namespace {

using at::Tensor;

decltype(&kfa_window_forward_workspace_bytes) window_forward_workspace_bytes;
decltype(&kfa_window_forward) window_forward;
decltype(&kfa_window_backward_workspace_bytes) window_backward_workspace_bytes;
decltype(&kfa_window_backward) window_backward;
decltype(&kfa_cache_write) cache_write;
decltype(&kfa_cache_read) cache_read;
decltype(&kfa_cache_attention_workspace_bytes) cache_attention_workspace_bytes;
decltype(&kfa_cache_attention) cache_attention;
PyObject* raise_error = nullptr;  // set last: the functions are there when it is
std::atomic<uint64_t> allowed{0};

struct Unserved {};  // the Python layer has to take this call

// ------------------------------------------------------------------ arguments
bool plain(const Tensor& t) {
    return t.is_cuda() && t.layout() == at::kStrided && !t.is_conj() && !t.is_neg() && !at::isTensorSubclassLike(t) &&
           !t._fw_grad(0).defined();  // (a forward-mode tangent, which Python refuses)
}

const Tensor& tensor(PyObject* o) {
    if (!THPVariable_CheckExact(o)) throw Unserved();
    const Tensor& t = THPVariable_Unpack(o);
    if (!plain(t)) throw Unserved();
    return t;
}

int64_t integer(PyObject* o) {
    if (!PyLong_CheckExact(o)) throw Unserved();  // (a bool is not)
    int overflow = 0;
    const int64_t x = PyLong_AsLongLongAndOverflow(o, &overflow);
    if (overflow) throw Unserved();
    return x;
}

int half_type(const Tensor& t) {
    if (t.scalar_type() == at::kHalf) return KFA_F16;
    if (t.scalar_type() == at::kBFloat16) return KFA_BF16;
    throw Unserved();
}

void on_allowed_device(const Tensor& t) {
    const int device = t.device().index();
    if (device < 0 || device > 63 || !(allowed.load(std::memory_order_relaxed) >> device & 1)) throw Unserved();
}

// Unit channel stride, 16-byte aligned base, other strides positive multiples of 8 elements of 16 bits.
bool addressable(const Tensor& t) {
    const auto sizes = t.sizes(), strides = t.strides();
    if (strides[3] != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
    for (int i = 0; i < 3; ++i)
        if (sizes[i] != 1 && (strides[i] <= 0 || strides[i] % 8)) return false;
    return true;
}

// Whether two elements may share memory: an axis whose stride does not clear what the axes of smaller strides reach.
bool may_overlap(const Tensor& t) {
    int64_t reach = 0, done = -1;
    for (int n = 0; n < t.dim(); ++n) {  // in the order of their strides, equal ones of two axes are an overlap
        int64_t next = INT64_MAX, size = 1;
        for (int i = 0; i < t.dim(); ++i) {
            if (t.size(i) == 1 || t.stride(i) > next || t.stride(i) <= done) continue;
            if (t.stride(i) == next) return true;
            next = t.stride(i);
            size = t.size(i);
        }
        if (size == 1) break;
        if (next <= reach) return true;
        reach += next * (size - 1);
        done = next;
    }
    return false;
}

bool differentiated(std::initializer_list<const Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t->requires_grad()) return true;
    return false;
}

// A position per sequence, or one for all of them.
struct Positions {
    std::optional<Tensor> each;
    int64_t all = 0;
};
Tensor per_sequence(PyObject* o, const Tensor& like) {
    const Tensor& t = tensor(o);
    if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != like.size(0) || t.device() != like.device() || !t.is_contiguous())
        throw Unserved();
    return t;
}
Positions positions(PyObject* o, const Tensor& like) {
    Positions p;
    if (PyLong_CheckExact(o)) {
        p.all = integer(o);
        if (p.all < 0 || p.all > INT32_MAX) throw Unserved();
    } else {
        p.each = per_sequence(o, like);
    }
    return p;
}

double scale_of(PyObject* o, int64_t channels) {
    if (o == Py_None) return std::pow((double)channels, -0.5);
    if (!PyFloat_CheckExact(o)) throw Unserved();
    const double x = PyFloat_AS_DOUBLE(o);
    if (!std::isfinite(x) || std::fabs(x) > FLT_MAX) throw Unserved();
    return x;
}

// ------------------------------------------------------------------ records and launches
kfa_tensor record(const Tensor& t, int type) {
    kfa_tensor r;
    std::memset(&r, 0, sizeof(r));
    r.data = t.data_ptr();
    r.dtype = type;
    r.ndim = (int32_t)t.dim();
    for (int i = 0; i < r.ndim; ++i) {
        r.sizes[i] = t.size(i);
        r.strides[i] = t.stride(i);
    }
    return r;
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

Tensor workspace_of(size_t bytes, const Tensor& like) {
    return at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(like.device()));
}

Tensor row_statistics(const Tensor& q) {
    return at::empty({q.size(0), q.size(1), q.size(2)}, at::TensorOptions().dtype(at::kFloat).device(q.device()));
}

// O (and its row statistics where asked for) of checked operands, or the library's code.
int run_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Positions& at, int64_t window, int64_t sinks,
                double scale, bool statistics, Tensor& out, Tensor& maximum, Tensor& logsum) {
    const c10::cuda::CUDAGuard guard(q.device());
    const int type = half_type(q);
    out = at::empty_like(q);
    const kfa_tensor rq = record(q, type), rk = record(k, type), rv = record(v, type);
    kfa_tensor ro = record(out, type), rs, rm, rl;
    if (at.each) rs = record(*at.each, KFA_I32);
    if (statistics) {
        maximum = row_statistics(q);
        logsum = row_statistics(q);
        rm = record(maximum, KFA_F32);
        rl = record(logsum, KFA_F32);
    }
    const size_t need = window_forward_workspace_bytes(&rq, &rk, window, sinks, statistics);
    Tensor workspace;
    if (need) workspace = workspace_of(need, q);
    return window_forward(&rq, &rk, &rv, at.each ? &rs : nullptr, &ro, statistics ? &rm : nullptr, statistics ? &rl : nullptr,
                          need ? workspace.data_ptr() : nullptr, need, at.all, window, sinks, (float)scale, stream_of(q));
}

struct WindowAttention : public torch::autograd::Function<WindowAttention> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, int64_t start,
                          int64_t window, int64_t sinks, double scale) {
        Positions at;
        at.all = start;
        Tensor out, maximum, logsum;
        if (run_forward(q, k, v, at, window, sinks, scale, true, out, maximum, logsum)) throw Unserved();
        ctx->save_for_backward({q, k, v, out, maximum, logsum});
        int64_t bits;
        std::memcpy(&bits, &scale, sizeof(bits));
        ctx->saved_data["call"] = std::vector<int64_t>{start, window, sinks, bits};
        return out;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &out = saved[3], &maximum = saved[4], &logsum = saved[5];
        const std::vector<int64_t> call = ctx->saved_data["call"].toIntVector();
        double scale;
        std::memcpy(&scale, &call[3], sizeof(scale));
        const c10::cuda::CUDAGuard guard(q.device());
        Tensor dout = grads[0].resolve_conj().resolve_neg();
        if (!addressable(dout)) dout = dout.clone(at::MemoryFormat::Contiguous);  // (contiguous() keeps an odd address)
        const int type = half_type(q);
        Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v);
        const kfa_tensor rq = record(q, type), rk = record(k, type), rv = record(v, type), ro = record(out, type),
                         rm = record(maximum, KFA_F32), rl = record(logsum, KFA_F32), rg = record(dout, type);
        kfa_tensor rdq = record(dq, type), rdk = record(dk, type), rdv = record(dv, type);
        const size_t need = window_backward_workspace_bytes(&rq, &rk, call[0], call[1], call[2]);
        const Tensor workspace = workspace_of(need, q);
        const int code = window_backward(&rq, &rk, &rv, &ro, &rm, &rl, &rg, &rdq, &rdk, &rdv, workspace.data_ptr(), need,
                                         call[0], call[1], call[2], (float)scale, stream_of(q));
        if (code) {
            const pybind11::gil_scoped_acquire gil;
            PyObject* nothing = PyObject_CallFunction(raise_error, "i", code);
            Py_XDECREF(nothing);
            python_error error;
            error.persist();
            throw python_error(std::move(error));
        }
        if (at::GradMode::is_enabled()) {
            // create_graph: gradients that raise when they are differentiated, not constants
            const auto twice = std::make_shared<torch::autograd::DelayedError>(
                "sliding_window_attention cannot be differentiated twice", 3);
            torch::autograd::variable_list results{dq, dk, dv};
            for (Tensor& t : results) t = t.detach().set_requires_grad(true);
            results = (*twice)(std::move(results));
            dq = results[0], dk = results[1], dv = results[2];
        }
        return {dq, dk, dv, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// ------------------------------------------------------------------ calls
// The four tensors of a cache, checked against one another; `channels` and `type` are the model's.
struct Cache {
    const Tensor *k_codes, *k_params, *v_codes, *v_params;
    int64_t channels;
    int type;
    kfa_tensor r[4];
    explicit Cache(PyObject* o) {
        if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) throw Unserved();
        const Tensor* t[4];
        for (int i = 0; i < 4; ++i) t[i] = &tensor(PyTuple_GET_ITEM(o, i));
        k_codes = t[0], k_params = t[1], v_codes = t[2], v_params = t[3];
        const Tensor &kc = *k_codes, &kp = *k_params;
        on_allowed_device(kc);
        type = half_type(kp);
        if (kc.scalar_type() != at::kByte || kc.dim() != 4 || kc.numel() == 0 || kc.size(3) % 32 || kc.size(3) > 256) throw Unserved();
        if (kp.dim() != 5 || kp.size(3) != kc.size(3) / 32 || kp.size(4) != 2) throw Unserved();
        for (int i = 0; i < 3; ++i)
            if (kp.size(i) != kc.size(i)) throw Unserved();
        if (v_codes->scalar_type() != at::kByte || v_codes->sizes() != kc.sizes() || v_params->scalar_type() != kp.scalar_type() ||
            v_params->sizes() != kp.sizes())
            throw Unserved();
        for (int i = 1; i < 4; ++i)
            if (t[i]->device() != kc.device()) throw Unserved();
        channels = 2 * kc.size(3);
        for (int i = 0; i < 4; ++i) r[i] = record(*t[i], i % 2 ? type : KFA_U8);
    }
};

// Runs a call: its result, None where Python has to take it, or NULL with the exception of a failed allocation.
template <typename Call>
PyObject* served(Call call) {
    HANDLE_TH_ERRORS
    try {
        if (raise_error) return call();
    } catch (const Unserved&) {
    }
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

template <typename Launch>
void launched(Launch launch) {
    int code;
    {
        const pybind11::gil_scoped_release others;  // as a ctypes call would
        code = launch();
    }
    if (code) throw Unserved();  // nothing was launched: Python repeats the call and raises
}

PyObject* py_window_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return served([&]() -> PyObject* {
        if (n != 7) throw Unserved();
        const Tensor &q = tensor(args[0]), k = tensor(args[1]), v = tensor(args[2]);
        const int64_t window = integer(args[3]), sinks = integer(args[4]);
        if (q.dim() != 4 || k.dim() != 4 || q.numel() == 0 || k.numel() == 0 || k.sizes() != v.sizes()) throw Unserved();
        const int64_t D = q.size(3);
        half_type(q);
        on_allowed_device(q);
        if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() || k.device() != q.device() ||
            v.device() != q.device() || k.size(0) != q.size(0) || k.size(3) != D || q.size(1) % k.size(1) || window < 1 || sinks < 0)
            throw Unserved();
        if (D > 128 ? D != 256 && D != 384 && D != 512 : D % 8 != 0) throw Unserved();
        if (!addressable(q) || !addressable(k) || !addressable(v)) throw Unserved();
        const Positions at = positions(args[5], q);
        const double scale = scale_of(args[6], D);
        const bool graph = differentiated({&q, &k, &v});
        if (graph && at.each) throw Unserved();
        Tensor out;
        // keys behind the last query's position are seen by nobody: leave them out (and their gradients zero)
        const int64_t end = at.each ? k.size(2) : std::min(k.size(2), at.all + q.size(2));
        const bool cut = end < k.size(2);
        const Tensor seen_k = cut ? k.narrow(2, 0, end) : k, seen_v = cut ? v.narrow(2, 0, end) : v;
        if (graph) {
            out = WindowAttention::apply(q, seen_k, seen_v, at.all, window, sinks, scale);
        } else {
            Tensor maximum, logsum;
            launched([&] { return run_forward(q, seen_k, seen_v, at, window, sinks, scale, false, out, maximum, logsum); });
        }
        return THPVariable_Wrap(out);
    });
}

PyObject* py_cache_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return served([&]() -> PyObject* {
        if (n != 5) throw Unserved();
        Cache cache(args[0]);
        const Tensor &k = tensor(args[1]), v = tensor(args[2]), kc = *cache.k_codes;
        if (k.dim() != 4 || k.numel() == 0 || k.sizes() != v.sizes() || k.device() != kc.device() || v.device() != kc.device() ||
            k.scalar_type() != cache.k_params->scalar_type() || v.scalar_type() != k.scalar_type() || k.size(0) != kc.size(0) ||
            k.size(1) != kc.size(1) || k.size(3) != cache.channels)
            throw Unserved();
        for (const Tensor* t : {cache.k_codes, cache.k_params, cache.v_codes, cache.v_params})
            if (!t->is_contiguous() && may_overlap(*t)) throw Unserved();
        if (differentiated({&k, &v, cache.k_params, cache.v_params}) || !addressable(k) || !addressable(v)) throw Unserved();
        const Positions at = positions(args[3], kc);
        if (!at.each && at.all + k.size(2) > kc.size(2)) throw Unserved();
        std::optional<Tensor> lengths;
        if (args[4] != Py_None) lengths = per_sequence(args[4], kc);
        const kfa_tensor rk = record(k, cache.type), rv = record(v, cache.type);
        kfa_tensor rs, rl;
        if (at.each) rs = record(*at.each, KFA_I32);
        if (lengths) rl = record(*lengths, KFA_I32);
        const c10::cuda::CUDAGuard guard(kc.device());
        launched([&] {
            return cache_write(&rk, &rv, &cache.r[0], &cache.r[1], &cache.r[2], &cache.r[3], at.each ? &rs : nullptr,
                               lengths ? &rl : nullptr, at.all, stream_of(kc));
        });
        for (const Tensor* t : {cache.k_codes, cache.k_params, cache.v_codes, cache.v_params})
            if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
        Py_RETURN_TRUE;
    });
}

PyObject* py_cache_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return served([&]() -> PyObject* {
        if (n != 3) throw Unserved();
        const Cache cache(args[0]);
        const Tensor& kc = *cache.k_codes;
        if (differentiated({cache.k_params, cache.v_params})) throw Unserved();
        const Positions at = positions(args[1], kc);
        if (args[2] == Py_None && at.each) throw Unserved();
        const int64_t length = args[2] == Py_None ? kc.size(2) - at.all : integer(args[2]);
        if (length < 1 || (!at.each && at.all + length > kc.size(2))) throw Unserved();
        const c10::cuda::CUDAGuard guard(kc.device());
        const auto options = at::TensorOptions().dtype(cache.k_params->scalar_type()).device(kc.device());
        const Tensor k = at::empty({kc.size(0), kc.size(1), length, cache.channels}, options), v = at::empty_like(k);
        kfa_tensor rk = record(k, cache.type), rv = record(v, cache.type), rs;
        if (at.each) rs = record(*at.each, KFA_I32);
        launched([&] {
            return cache_read(&cache.r[0], &cache.r[1], &cache.r[2], &cache.r[3], at.each ? &rs : nullptr, &rk, &rv, at.all,
                              stream_of(kc));
        });
        PyObject* pair = PyTuple_New(2);
        if (!pair) throw python_error();
        PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(k));
        PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(v));
        return pair;
    });
}

PyObject* py_cache_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return served([&]() -> PyObject* {
        if (n != 6) throw Unserved();
        const Tensor& q = tensor(args[0]);
        const Cache cache(args[1]);
        const Tensor& kc = *cache.k_codes;
        if (q.dim() != 4 || q.numel() == 0 || q.device() != kc.device() || q.scalar_type() != cache.k_params->scalar_type() ||
            q.size(0) != kc.size(0) || q.size(1) % kc.size(1) || q.size(3) != cache.channels)
            throw Unserved();
        const int64_t window = args[3] == Py_None ? 0 : integer(args[3]), sinks = integer(args[4]);
        if (args[3] == Py_None ? sinks != 0 : window < 1 || sinks < 0) throw Unserved();
        if (differentiated({&q, cache.k_params, cache.v_params}) || !addressable(q)) throw Unserved();
        const Positions at = positions(args[2], q);
        const double scale = scale_of(args[5], cache.channels);
        const c10::cuda::CUDAGuard guard(q.device());
        const Tensor out = at::empty_like(q);
        const kfa_tensor rq = record(q, cache.type);
        kfa_tensor ro = record(out, cache.type), rs;
        if (at.each) rs = record(*at.each, KFA_I32);
        const size_t need = cache_attention_workspace_bytes(&rq, &cache.r[0], window, sinks);
        if (need == 0) throw Unserved();
        const Tensor workspace = workspace_of(need, q);
        launched([&] {
            return cache_attention(&rq, &cache.r[0], &cache.r[1], &cache.r[2], &cache.r[3], at.each ? &rs : nullptr, &ro,
                                   workspace.data_ptr(), need, at.all, window, sinks, (float)scale, stream_of(q));
        });
        return THPVariable_Wrap(out);
    });
}

// ------------------------------------------------------------------ the module
template <typename F>
bool entry(PyObject* addresses, const char* name, F& function) {
    PyObject* address = PyDict_GetItemString(addresses, name);  // borrowed
    if (!address) {
        PyErr_Format(PyExc_KeyError, "no address for %s", name);
        return false;
    }
    function = reinterpret_cast<F>(PyLong_AsVoidPtr(address));
    return function && !PyErr_Occurred();
}

PyObject* py_bind(PyObject*, PyObject* args) {
    PyObject *addresses, *raiser;
    if (!PyArg_ParseTuple(args, "O!O", &PyDict_Type, &addresses, &raiser)) return nullptr;
    if (!entry(addresses, "kfa_window_forward_workspace_bytes", window_forward_workspace_bytes) ||
        !entry(addresses, "kfa_window_forward", window_forward) ||
        !entry(addresses, "kfa_window_backward_workspace_bytes", window_backward_workspace_bytes) ||
        !entry(addresses, "kfa_window_backward", window_backward) || !entry(addresses, "kfa_cache_write", cache_write) ||
        !entry(addresses, "kfa_cache_read", cache_read) ||
        !entry(addresses, "kfa_cache_attention_workspace_bytes", cache_attention_workspace_bytes) ||
        !entry(addresses, "kfa_cache_attention", cache_attention))
        return nullptr;
    Py_INCREF(raiser);
    Py_XDECREF(raise_error);
    raise_error = raiser;
    Py_RETURN_NONE;
}

PyObject* py_allow(PyObject*, PyObject* index) {
    const long device = PyLong_AsLong(index);
    if (device == -1 && PyErr_Occurred()) return nullptr;
    if (device >= 0 && device < 64) allowed.fetch_or(uint64_t(1) << device);
    Py_RETURN_NONE;
}

template <PyObject* (*function)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(function)); }

PyMethodDef methods[] = {
    {"bind", py_bind, METH_VARARGS, nullptr},
    {"allow", py_allow, METH_O, nullptr},
    {"window_attention", fast<py_window_attention>(), METH_FASTCALL, nullptr},
    {"cache_write", fast<py_cache_write>(), METH_FASTCALL, nullptr},
    {"cache_read", fast<py_cache_read>(), METH_FASTCALL, nullptr},
    {"cache_attention", fast<py_cache_attention>(), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fast_calls() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", KFA_TORCH_VERSION) < 0) Py_CLEAR(m);
    return m;
}
