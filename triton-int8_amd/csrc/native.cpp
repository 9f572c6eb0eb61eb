// The host side of a layer call (ops.linear_call) and of the calls on the 4-bit cache (cache4.py) as one Python call each: outputs, workspace and argument
// block, then the library's entry points.  It makes the same allocations and calls as the Python that it stands in for.  Calls with anything out of the ordinary
// (subclasses of Tensor, other dtypes, tensors that are not on a GPU) return None and take the Python way, which says what is wrong.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <cmath>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <ATen/detail/CUDAHooksInterface.h>
#include <ATen/ops/narrow.h>
#include <ATen/TracerMode.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

#include "../../include/ti8.h"

namespace {

// The library is the one that the binding has loaded: its entry points come from there
decltype(&ti8_linear) linear = nullptr;
decltype(&ti8_linear_quantise) linear_quantise = nullptr;
decltype(&ti8_gemm_i8_nt_multi) gemm_multi = nullptr;
decltype(&ti8_cache4_append) cache4_append_entry = nullptr;
decltype(&ti8_cache4_read) cache4_read_entry = nullptr;
decltype(&ti8_cache4_attention) cache4_attention_entry = nullptr;
decltype(&ti8_cache4_attention_workspace) cache4_attention_workspace = nullptr;
decltype(&ti8_cache4_evict) cache4_evict_entry = nullptr;
PyObject* parameter_class = nullptr;

// *out = the tensor behind `o` (undefined for None); false if it is not a plain tensor
bool plain(PyObject* o, at::Tensor* out) {
    if (o == Py_None) return true;
    if (Py_TYPE(o) != reinterpret_cast<PyTypeObject*>(THPVariableClass) && Py_TYPE(o) != reinterpret_cast<PyTypeObject*>(parameter_class)) return false;
    *out = THPVariable_Unpack(o);
    return true;
}

bool bf16_matrix(const at::Tensor& t) { return !t.defined() || (t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.dim() == 2); }

// The tensor itself where the library can read its rows in place, else a dense copy (ops.rows16)
at::Tensor rows16(const at::Tensor& t) {
    if (!t.defined()) return t;
    const int64_t row = t.stride(0);
    if (t.stride(1) == 1 && row % 8 == 0 && row >= t.size(1) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0) return t;
    return t.clone(at::MemoryFormat::Contiguous);
}

struct GilReleased {
    PyThreadState* const state = PyEval_SaveThread();
    ~GilReleased() { PyEval_RestoreThread(state); }
};

// Device memory that a call needs until its launches are queued, from the allocator that tensors come from at the time (a program may put its own in
// the place of torch's) but without making one
struct Workspace {
    c10::DataPtr plain;
    at::Tensor tensor;
    void* p;
    Workspace(int64_t bytes, const at::Device& dev, const at::TensorOptions& options) {
        if (c10::impl::getDeviceGuardImpl(c10::DeviceType::CUDA)->getDevice() == dev) {
            plain = at::detail::getCUDAHooks().getCUDADeviceAllocator()->allocate(bytes);
            p = plain.get();
        } else {
            tensor = at::empty({bytes}, options);
            p = tensor.data_ptr();
        }
    }
};

// Whether a tracer, a dispatch mode or a function transform looks at the operators of this thread
bool followed() {
    return at::tracer::impl::is_dispatch_enabled() || c10::impl::dispatch_mode_enabled() ||
           c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}

PyObject* wrap(const at::Tensor& t) {
    if (t.defined()) return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}

enum { PARTS, SCHEME, HADAMARD, TOKENS, K_, N_, GEMM_FLAGS, NEED, NEED_SAVED, APART, STREAM, SERVED, NUMBERS, TENSORS = 7 };

// linear_call(parts, scheme, hadamard, tokens, K, N, gemm_flags, workspace bytes, saved bytes, whether the GEMMs are a call of their
// own, stream, whether only Y is wanted, and of that the rows of tokens alone, X, W, dY, wq, ws, saved, bias) -> (Y, dX, dW, saved) or that Y,
// (name, status) of an entry point that failed, or None
PyObject* linear_call(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != NUMBERS + TENSORS) {
        PyErr_SetString(PyExc_TypeError, "linear_call takes 19 arguments");
        return nullptr;
    }
    at::Tensor X, W, dY, wq, ws, saved, bias;
    at::Tensor* const tensors[TENSORS] = {&X, &W, &dY, &wq, &ws, &saved, &bias};
    for (int i = 0; i < TENSORS; ++i)
        if (!plain(args[NUMBERS + i], tensors[i])) Py_RETURN_NONE;
    if (!bf16_matrix(X) || !bf16_matrix(W) || !bf16_matrix(dY) || (!X.defined() && !dY.defined())) Py_RETURN_NONE;
    int64_t v[NUMBERS];
    for (int i = 0; i < NUMBERS; ++i) {
        v[i] = PyLong_AsLongLong(args[i]);
        if (v[i] == -1 && PyErr_Occurred()) return nullptr;
    }
    at::Tensor Y, dX, dW;
    const char* name = "ti8_linear";
    int status;
    {
        const GilReleased released;      // the allocator and the library have locks of their own
        const int64_t tokens = v[TOKENS], K = v[K_], N = v[N_], T = (tokens + 127) / 128 * 128;
        const at::Device dev = X.defined() ? X.device() : dY.device();
        const auto bf16 = at::TensorOptions().dtype(at::kBFloat16).device(dev), bytes = at::TensorOptions().dtype(at::kByte).device(dev);
        X = rows16(X);
        W = rows16(W);
        dY = rows16(dY);
        if (v[PARTS] & TI8_PART_FORWARD) {
            Y = at::empty({T, N}, bf16);
            if (v[NEED_SAVED]) saved = at::empty({v[NEED_SAVED]}, bytes);
        }
        if (v[PARTS] & TI8_PART_BACKWARD) {
            dX = at::empty({T, K}, bf16);
            dW = at::empty({N, K}, bf16);
        }
        const Workspace workspace(v[NEED], dev, bytes);
        const auto ptr = [](const at::Tensor& t) -> void* { return t.defined() ? t.data_ptr() : nullptr; };
        const auto row = [](const at::Tensor& t) -> int64_t { return t.defined() ? t.stride(0) : 0; };
        ti8_linear_args a = {};
        a.X = ptr(X); a.ldx = row(X);
        a.W = ptr(W); a.ldw = row(W);
        a.dY = ptr(dY); a.lddy = row(dY);
        a.Y = ptr(Y); a.ldy = N;
        a.dX = ptr(dX); a.lddx = K;
        a.dW = ptr(dW); a.lddw = K;
        a.wq = static_cast<const int8_t*>(ptr(wq)); a.ws = static_cast<const float*>(ptr(ws));
        a.tokens = tokens; a.K = K; a.N = N;
        a.scheme = (int)v[SCHEME]; a.hadamard = (int)v[HADAMARD]; a.parts = (int)v[PARTS]; a.gemm_flags = (int)v[GEMM_FLAGS];
        a.workspace = workspace.p; a.workspace_bytes = v[NEED];      // (device allocations start on 512-byte boundaries)
        a.saved = ptr(saved); a.saved_bytes = v[NEED_SAVED];
        a.bias = ptr(bias);
        ti8_stream_t stream = reinterpret_cast<ti8_stream_t>(static_cast<uintptr_t>(v[STREAM]));
        if (v[APART]) {
            ti8_gemm_problem problems[3];
            int count = 0;
            name = "ti8_linear_quantise";
            status = linear_quantise(&a, problems, &count, stream);
            if (status == TI8_OK) {
                name = "ti8_gemm_i8_nt_multi";
                status = gemm_multi(problems, count, a.gemm_flags | TI8_GEMM_TOGETHER, stream);
            }
        } else {
            status = linear(&a, stream);
        }
    }
    if (status != TI8_OK) return Py_BuildValue("(si)", name, status);
    if (v[SERVED]) {
        // (in its own sizes, unless something follows what is made of Y operator by operator)
        if (followed()) Y = Y.narrow(0, 0, v[TOKENS]);
        else Y.unsafeGetTensorImpl()->set_sizes_contiguous({v[TOKENS], v[N_]});
        return wrap(Y);
    }
    return Py_BuildValue("(NNNN)", wrap(Y), wrap(dX), wrap(dW), wrap(saved));
    END_HANDLE_TH_ERRORS
}

// ---- the 4-bit cache: every function returns None for what cache4.py has to look at, else what its calls return, or (name, status) -------------------

c10::DeviceIndex current_device() { return c10::impl::getDeviceGuardImpl(c10::DeviceType::CUDA)->getDevice().index(); }

// Whether a gradient or a tangent is asked for
bool derived(const at::Tensor& t) { return (t.requires_grad() && at::GradMode::is_enabled()) || t._fw_grad(0).defined(); }

struct CacheCall {
    const c10::DeviceIndex device = current_device();
    ti8_cache4 c = {};

    bool here(const at::Tensor& t, at::ScalarType type, int64_t dim) const {
        return t.defined() && t.is_cuda() && t.get_device() == device && t.scalar_type() == type && t.dim() == dim;
    }
    // int32 [batch], or nothing where that is allowed
    bool ints(const at::Tensor& t, bool optional, const int32_t** p) const {
        if (!t.defined()) return optional;
        if (!here(t, at::kInt, 1) || t.size(0) != c.batch || !t.is_contiguous()) return false;
        *p = static_cast<const int32_t*>(t.data_ptr());
        return true;
    }
    bool rows_of(const at::Tensor& t, int64_t* pages, int64_t* stride) const {
        if (!here(t, at::kInt, 2) || t.size(0) != c.batch || t.size(1) == 0 || (t.size(1) > 1 && t.stride(1) != 1) || (c.batch > 1 && t.stride(0) < t.size(1))) return false;
        *pages = t.size(1);
        *stride = c.batch == 1 ? t.size(1) : t.stride(0);
        return true;
    }
    bool describe(const at::Tensor& pool, const at::Tensor& table, const at::Tensor& weights, int64_t head_dim, int64_t batch) {
        if (!here(pool, at::kByte, 3) || !pool.is_contiguous() || (head_dim != 64 && head_dim != 128)) return false;
        const int64_t entry = head_dim + head_dim / 16, page = pool.size(2) / entry;
        if (page * entry != pool.size(2) || (page != 16 && page != 32 && page != 64 && page != 128 && page != 256)) return false;
        c.batch = batch;
        if (!rows_of(table, &c.table_pages, &c.table_stride)) return false;
        if (weights.defined() && (!here(weights, at::kFloat, 3) || derived(weights) || !weights.is_contiguous() || weights.size(0) != pool.size(0) || weights.size(1) != pool.size(1) || weights.size(2) != page)) return false;
        c.pool = pool.data_ptr();
        c.table = static_cast<const int32_t*>(table.data_ptr());
        c.weights = weights.defined() ? static_cast<float*>(weights.data_ptr()) : nullptr;
        c.pages = pool.size(0);
        c.kv_heads = pool.size(1);
        c.page_size = page;
        c.head_dim = head_dim;
        return true;
    }
    // bf16 [batch][tokens][heads][head_dim] that is read in place; strides between batches, tokens and heads
    bool tokens_of(const at::Tensor& t, int64_t (&strides)[3]) const {
        if (!here(t, at::kBFloat16, 4) || t.numel() == 0 || derived(t)) return false;
        int64_t any = 0;
        for (int i = 0; i < 3; ++i) any |= strides[i] = t.size(i) == 1 ? 0 : t.stride(i);
        return t.stride(3) == 1 && !(any & 7) && !(reinterpret_cast<uintptr_t>(t.data_ptr()) & 15);
    }
};

bool tensors_of(PyObject* const* args, at::Tensor* const* tensors, int count) {
    for (int i = 0; i < count; ++i)
        if (!plain(args[i], tensors[i])) return false;
    return !followed();
}
bool number(PyObject* o, int64_t* v) {
    if (!PyLong_CheckExact(o)) return false;
    *v = PyLong_AsLongLong(o);
    if (*v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}
ti8_stream_t stream_of(int64_t v) { return reinterpret_cast<ti8_stream_t>(static_cast<uintptr_t>(v)); }

// cache4_append(pool, table, starts, k, v, counts, weights, stream) -> True
PyObject* cache4_append(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    at::Tensor pool, table, starts, k, v, counts, weights;
    at::Tensor* const tensors[] = {&pool, &table, &starts, &k, &v, &counts, &weights};
    int64_t stream, sk[3], sv[3];
    const int32_t *at_starts = nullptr, *at_counts = nullptr;
    if (nargs != 8 || !tensors_of(args, tensors, 7) || !number(args[7], &stream)) Py_RETURN_NONE;
    CacheCall call;
    if (!call.tokens_of(k, sk) || !call.tokens_of(v, sv) || k.sizes() != v.sizes() || !call.describe(pool, table, weights, k.size(3), k.size(0)) ||
        call.c.kv_heads != k.size(2) || !call.ints(starts, false, &at_starts) || !call.ints(counts, true, &at_counts))
        Py_RETURN_NONE;
    int status;
    {
        const GilReleased released;
        status = cache4_append_entry(&call.c, at_starts, at_counts, k.size(1), k.data_ptr(), sk[0], sk[1], sk[2], v.data_ptr(), sv[0], sv[1], sv[2], stream_of(stream));
    }
    if (status != TI8_OK) return Py_BuildValue("(si)", "ti8_cache4_append", status);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// cache4_read(pool, table, starts, counts, tokens, head_dim, stream) -> [k, v]
PyObject* cache4_read(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    at::Tensor pool, table, starts, counts, k, v;
    at::Tensor* const tensors[] = {&pool, &table, &starts, &counts};
    int64_t tokens, head_dim, stream;
    const int32_t *at_starts = nullptr, *at_counts = nullptr;
    if (nargs != 7 || !tensors_of(args, tensors, 4) || !number(args[4], &tokens) || !number(args[5], &head_dim) || !number(args[6], &stream)) Py_RETURN_NONE;
    CacheCall call;
    if (tokens <= 0 || !table.defined() || table.dim() != 2 || table.size(0) == 0 || !call.describe(pool, table, at::Tensor(), head_dim, table.size(0)) ||
        !call.ints(starts, false, &at_starts) || !call.ints(counts, true, &at_counts))
        Py_RETURN_NONE;
    int status;
    {
        const GilReleased released;
        const auto bf16 = at::TensorOptions().dtype(at::kBFloat16).device(pool.device());
        k = at::empty({call.c.batch, tokens, call.c.kv_heads, head_dim}, bf16);
        v = at::empty({call.c.batch, tokens, call.c.kv_heads, head_dim}, bf16);
        status = cache4_read_entry(&call.c, at_starts, at_counts, tokens, k.data_ptr(), v.data_ptr(), stream_of(stream));
    }
    if (status != TI8_OK) return Py_BuildValue("(si)", "ti8_cache4_read", status);
    return Py_BuildValue("[NN]", wrap(k), wrap(v));
    END_HANDLE_TH_ERRORS
}

// cache4_attention(pool, table, lengths, q, counts, weights, scale or None, stream) -> [out, lse]
PyObject* cache4_attention(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    at::Tensor pool, table, lengths, q, counts, weights, out, lse;
    at::Tensor* const tensors[] = {&pool, &table, &lengths, &q, &counts, &weights};
    int64_t stream, sq[3];
    const int32_t *at_lengths = nullptr, *at_counts = nullptr;
    if (nargs != 8 || !tensors_of(args, tensors, 6) || !number(args[7], &stream) || (args[6] != Py_None && !PyFloat_CheckExact(args[6]))) Py_RETURN_NONE;
    CacheCall call;
    if (!call.tokens_of(q, sq) || !call.describe(pool, table, weights, q.size(3), q.size(0)) || q.size(2) % call.c.kv_heads != 0 ||
        !call.ints(lengths, false, &at_lengths) || !call.ints(counts, true, &at_counts))
        Py_RETURN_NONE;
    const int64_t need = cache4_attention_workspace(&call.c, q.size(1), q.size(2));
    if (need < 0) Py_RETURN_NONE;
    const float scale = args[6] == Py_None ? (float)(1.0 / std::sqrt((double)q.size(3))) : (float)PyFloat_AS_DOUBLE(args[6]);
    if (!(std::fabs(scale) <= 0x1p127f)) Py_RETURN_NONE;
    int status;
    {
        const GilReleased released;
        const at::TensorOptions options = at::TensorOptions().device(q.device());
        out = at::empty(q.sizes(), options.dtype(at::kBFloat16));
        lse = at::empty({q.size(0), q.size(1), q.size(2)}, options.dtype(at::kFloat));
        const Workspace workspace(need, q.device(), options.dtype(at::kByte));
        status = cache4_attention_entry(&call.c, at_lengths, at_counts, q.size(1), q.size(2), q.data_ptr(), sq[0], sq[1], sq[2], scale, weights.defined(),
                                        out.data_ptr(), static_cast<float*>(lse.data_ptr()), workspace.p, need, stream_of(stream));
    }
    if (status != TI8_OK) return Py_BuildValue("(si)", "ti8_cache4_attention", status);
    return Py_BuildValue("[NN]", wrap(out), wrap(lse));
    END_HANDLE_TH_ERRORS
}

// cache4_evict(pool, table, lengths, weights, new_table, keep, recent, stream) -> [kept, new lengths]
PyObject* cache4_evict(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    at::Tensor pool, table, lengths, weights, new_table, kept, new_lengths;
    at::Tensor* const tensors[] = {&pool, &table, &lengths, &weights, &new_table};
    int64_t keep, recent, stream, pages, stride;
    const int32_t* at_lengths = nullptr;
    if (nargs != 8 || !tensors_of(args, tensors, 5) || !number(args[5], &keep) || !number(args[6], &recent) || !number(args[7], &stream)) Py_RETURN_NONE;
    CacheCall call;
    if (!table.defined() || table.dim() != 2 || table.size(0) == 0 || !pool.defined() || pool.dim() != 3 || !weights.defined() || weights.dim() != 3 || weights.size(2) == 0 ||
        !call.describe(pool, table, weights, pool.size(2) / weights.size(2) * 16 / 17, table.size(0)) || !call.ints(lengths, false, &at_lengths) ||
        !call.rows_of(new_table, &pages, &stride) || keep <= 0 || keep > pages * call.c.page_size || recent < 0 || recent > keep)
        Py_RETURN_NONE;
    int status;
    {
        const GilReleased released;
        const auto ints = at::TensorOptions().dtype(at::kInt).device(pool.device());
        kept = at::empty({call.c.batch, call.c.kv_heads, keep}, ints);
        new_lengths = at::empty({call.c.batch}, ints);
        status = cache4_evict_entry(&call.c, at_lengths, static_cast<const int32_t*>(new_table.data_ptr()), pages, stride, keep, recent,
                                    static_cast<int32_t*>(kept.data_ptr()), static_cast<int32_t*>(new_lengths.data_ptr()), stream_of(stream));
    }
    if (status != TI8_OK) return Py_BuildValue("(si)", "ti8_cache4_evict", status);
    return Py_BuildValue("[NN]", wrap(kept), wrap(new_lengths));
    END_HANDLE_TH_ERRORS
}

// set_up_cache4(addresses of ti8_cache4_append, _read, _attention, _attention_workspace, _evict)
PyObject* set_up_cache4(PyObject*, PyObject* args) {
    unsigned long long a, r, t, w, e;
    if (!PyArg_ParseTuple(args, "KKKKK", &a, &r, &t, &w, &e)) return nullptr;
    cache4_append_entry = reinterpret_cast<decltype(cache4_append_entry)>(a);
    cache4_read_entry = reinterpret_cast<decltype(cache4_read_entry)>(r);
    cache4_attention_entry = reinterpret_cast<decltype(cache4_attention_entry)>(t);
    cache4_attention_workspace = reinterpret_cast<decltype(cache4_attention_workspace)>(w);
    cache4_evict_entry = reinterpret_cast<decltype(cache4_evict_entry)>(e);
    Py_RETURN_NONE;
}

// set_up(addresses of ti8_linear, ti8_linear_quantise, ti8_gemm_i8_nt_multi; torch.nn.Parameter)
PyObject* set_up(PyObject*, PyObject* args) {
    unsigned long long l, q, g;
    PyObject* parameter;
    if (!PyArg_ParseTuple(args, "KKKO", &l, &q, &g, &parameter)) return nullptr;
    linear = reinterpret_cast<decltype(linear)>(l);
    linear_quantise = reinterpret_cast<decltype(linear_quantise)>(q);
    gemm_multi = reinterpret_cast<decltype(gemm_multi)>(g);
    Py_INCREF(parameter);
    Py_XSETREF(parameter_class, parameter);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"linear_call", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear_call)), METH_FASTCALL, nullptr},
    {"cache4_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cache4_append)), METH_FASTCALL, nullptr},
    {"cache4_read", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cache4_read)), METH_FASTCALL, nullptr},
    {"cache4_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cache4_attention)), METH_FASTCALL, nullptr},
    {"cache4_evict", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cache4_evict)), METH_FASTCALL, nullptr},
    {"set_up", set_up, METH_VARARGS, nullptr},
    {"set_up_cache4", set_up_cache4, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// built_for: what the code above was compiled against, for whoever loads it to compare (fields of torch's and Python's objects and of the
// library's argument blocks are read and written here without a call)
PyMODINIT_FUNC PyInit__native(void) {
    PyObject* const m = PyModule_Create(&module);
    PyObject* const built_for = Py_BuildValue("(s(ii)nnn)", TI8_BUILT_FOR_TORCH, PY_MAJOR_VERSION, PY_MINOR_VERSION, (Py_ssize_t)sizeof(ti8_linear_args), (Py_ssize_t)sizeof(ti8_gemm_problem),
                                              (Py_ssize_t)sizeof(ti8_cache4));
    if (m && (!built_for || PyModule_AddObject(m, "built_for", built_for) < 0)) {
        Py_XDECREF(built_for);
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
