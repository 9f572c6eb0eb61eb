// The host side of a layer call (ops.linear_call), of the calls on the 4-bit cache (cache4.py) and of those on tensors in 4 bits (mx4.py) as one Python call each: outputs, workspace and argument
// block, then the library's entry points.  It makes the same allocations and calls as the Python that it stands in for.  Calls with anything out of the ordinary
// (subclasses of Tensor, other dtypes, tensors that are not on a GPU) return None and take the Python way, which says what is wrong.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <cmath>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/EmptyTensor.h>
#include <ATen/ops/empty.h>
#include <c10/util/SmallVector.h>
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
decltype(&ti8_mx4_quant) mx4_quant_entry = nullptr;
decltype(&ti8_mx4_dequant) mx4_dequant_entry = nullptr;
decltype(&ti8_mx4_gemm_nt) mx4_gemm_entry = nullptr;
decltype(&ti8_mx4_gemm_nt_workspace) mx4_gemm_workspace = nullptr;
decltype(&ti8_mx4_gemm_nt_multi) mx4_multi_entry = nullptr;
decltype(&ti8_mx4_gemm_nt_multi_workspace) mx4_multi_workspace = nullptr;
decltype(&ti8_mx4_linear_fwd_bwd) mx4_step_entry = nullptr;
decltype(&ti8_mx4_linear_fwd_bwd_workspace) mx4_step_workspace = nullptr;
decltype(&ti8_rmsnorm_quant) rmsnorm_quant_entry = nullptr;
decltype(&ti8_dequant_row) dequant_row_entry = nullptr;
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
    return at::tracer::impl::is_dispatch_enabled() || c10::impl::dispatch_mode_enabled() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) ||
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

// ---- tensors in 4 bits: every function returns None for what mx4.py (ops.py) has to look at, else what its call returns, or (name, status) -------------

constexpr int64_t MX4_ROWS = 1 << 28, MX4_CONTRACTED = 1 << 22;

// (codes carry no tangent on)
bool on(const at::Tensor& t, at::ScalarType type, c10::DeviceIndex device) {
    return t.defined() && t.is_cuda() && t.get_device() == device && t.scalar_type() == type && t.numel() > 0 && !t._fw_grad(0).defined();
}
bool at_multiple(const at::Tensor& t, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0; }

// A new tensor on the current device, from the allocator that tensors come from (what at::empty comes down to; without the dispatcher, which takes as long)
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type) {
    return at::detail::empty_generic(sizes, at::detail::getCUDAHooks().getCUDADeviceAllocator(), c10::DispatchKeySet(c10::DispatchKey::CUDA), type, c10::nullopt);
}

// Room for the results of one call that die together.  Up to 4 MB in all they share a block of memory: asking for one and giving it back takes 0.4 us of a call
// that takes 5, and up to about there the kernel takes no longer than that.
class Room {
  public:
    explicit Room(int64_t bytes = INT64_MAX) {
        if (bytes <= 4 << 20) block_ = fresh({bytes}, at::kByte);
    }
    static int64_t of(int64_t bytes) { return (bytes + 255) / 256 * 256; }
    static int64_t of_mx4(int64_t rows, int64_t cols) { return of(rows * ((cols + 255) / 256) * 128) + of(rows * ((cols + 255) / 256) * 8); }
    at::Tensor operator()(at::IntArrayRef sizes, at::ScalarType type) {
        if (!block_.defined()) return fresh(sizes, type);
        at::Tensor t = at::detail::make_tensor<at::TensorImpl>(c10::Storage(block_.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA), c10::scalarTypeToTypeMeta(type));
        t.unsafeGetTensorImpl()->set_storage_offset(at_ / (int64_t)c10::elementSize(type));
        t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
        at_ += of(t.numel() * (int64_t)c10::elementSize(type));
        return t;
    }

  private:
    at::Tensor block_;
    int64_t at_ = 0;
};

// room for a tensor in 4 bits
struct Mx4Out {
    at::Tensor codes, scales;
    ti8_mx4 mx = {};
    Mx4Out() = default;
    Mx4Out(Room& room, at::IntArrayRef lead, int64_t rows, int64_t cols) {
        const int64_t tiles = (cols + 255) / 256;
        c10::SmallVector<int64_t, 4> sizes(lead.begin(), lead.end());
        sizes.push_back(tiles * 128);
        codes = room(sizes, at::kByte);
        scales = room({tiles, rows, 8}, at::kByte);
        mx = ti8_mx4{codes.data_ptr(), scales.data_ptr(), tiles * 128, rows * 8};
    }
};

// codes [rows][bytes] or [batch][rows][bytes] with their scales, where they are read in place
bool mx4_operand(const at::Tensor& codes, const at::Tensor& scales, c10::DeviceIndex device, ti8_mx4* mx) {
    if (!on(codes, at::kByte, device) || !on(scales, at::kByte, device) || (codes.dim() != 2 && codes.dim() != 3) || scales.dim() != 3) return false;
    const int64_t bytes = codes.size(-1), rows = codes.numel() / bytes, tiles = bytes / 128;
    if (bytes % 128 || scales.size(0) != tiles || scales.size(1) != rows || scales.size(2) != 8 || !at_multiple(codes, 16) || !at_multiple(scales, 8)) return false;
    int64_t ld = bytes, scale_ld = rows * 8;
    if (!codes.is_contiguous()) {
        if (codes.dim() != 2 || codes.stride(1) != 1 || codes.stride(0) % 16 || codes.stride(0) < bytes) return false;
        ld = codes.stride(0);
    }
    if (!scales.is_contiguous()) {
        if (scales.stride(2) != 1 || (rows > 1 && scales.stride(1) != 8) || (tiles > 1 && (scales.stride(0) % 8 || scales.stride(0) < rows * 8))) return false;
        if (tiles > 1) scale_ld = scales.stride(0);
    }
    *mx = ti8_mx4{codes.data_ptr(), scales.data_ptr(), ld, scale_ld};
    return true;
}

// mx4_quant(x [.., cols], by rows, by columns (x a matrix), stream) -> [codes, scales] or [codes, scales, codes, scales]
PyObject* mx4_quant(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    at::Tensor x;
    at::Tensor* const tensors[] = {&x};
    int64_t by_rows, by_columns, stream;
    if (nargs != 4 || !tensors_of(args, tensors, 1) || !number(args[1], &by_rows) || !number(args[2], &by_columns) || !number(args[3], &stream)) Py_RETURN_NONE;
    if (!on(x, at::kBFloat16, current_device()) || x.dim() < 1 || (x.dim() != 2 && (by_columns || !x.is_contiguous()))) Py_RETURN_NONE;
    const int64_t C = x.size(-1), R = x.numel() / C, ldx = x.dim() != 2 || R == 1 ? C : x.stride(0);
    if (x.stride(-1) != 1 || ldx < C || R > MX4_ROWS || C > MX4_ROWS) Py_RETURN_NONE;
    Mx4Out rows, cols;
    int status;
    {
        const GilReleased released;
        // (one view alone may be a weight's, kept and saved: two tensors of their own)
        Room room = by_rows && by_columns ? Room(Room::of_mx4(R, C) + Room::of_mx4(C, R)) : Room();
        if (by_rows) rows = Mx4Out(room, x.sizes().slice(0, x.dim() - 1), R, C);
        if (by_columns) cols = Mx4Out(room, {C}, C, R);
        const ti8_mx4_operand o = {x.data_ptr(), ldx, R, C, rows.mx, cols.mx};
        status = mx4_quant_entry(&o, 1, stream_of(stream));
    }
    if (status != TI8_OK) return Py_BuildValue("(si)", "ti8_mx4_quant", status);
    if (by_rows && by_columns) return Py_BuildValue("[NNNN]", wrap(rows.codes), wrap(rows.scales), wrap(cols.codes), wrap(cols.scales));
    const Mx4Out& made = by_rows ? rows : cols;
    return Py_BuildValue("[NN]", wrap(made.codes), wrap(made.scales));
    END_HANDLE_TH_ERRORS
}

// mx4_dequant(codes [rows, bytes], scales, cols, stream) -> y
PyObject* mx4_dequant(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    at::Tensor codes, scales, y;
    at::Tensor* const tensors[] = {&codes, &scales};
    int64_t cols, stream;
    ti8_mx4 mx;
    if (nargs != 4 || !tensors_of(args, tensors, 2) || !number(args[2], &cols) || !number(args[3], &stream) || !mx4_operand(codes, scales, current_device(), &mx)) Py_RETURN_NONE;
    const int64_t rows = codes.size(0);
    if (codes.dim() != 2 || cols <= 0 || codes.size(1) != (cols + 255) / 256 * 128 || rows > MX4_ROWS) Py_RETURN_NONE;
    int status;
    {
        const GilReleased released;
        y = fresh({rows, cols}, at::kBFloat16);
        status = mx4_dequant_entry(&mx, rows, cols, y.data_ptr(), cols, stream_of(stream));
    }
    if (status != TI8_OK) return Py_BuildValue("(si)", "ti8_mx4_dequant", status);
    return wrap(y);
    END_HANDLE_TH_ERRORS
}

// mx4_gemm_nt(A, scales of A, B, scales of B, whether in fp32, stream) -> C
PyObject* mx4_gemm_nt(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    at::Tensor A, sA, B, sB, out;
    at::Tensor* const tensors[] = {&A, &sA, &B, &sB};
    int64_t wide, stream;
    ti8_mx4 a, b;
    const c10::DeviceIndex device = current_device();
    if (nargs != 6 || !tensors_of(args, tensors, 4) || !number(args[4], &wide) || !number(args[5], &stream) || !mx4_operand(A, sA, device, &a) || !mx4_operand(B, sB, device, &b)) Py_RETURN_NONE;
    const int64_t K = A.size(-1) * 2, N = B.size(-2), rows = A.numel() / A.size(-1);
    if (B.size(-1) * 2 != K || (B.dim() == 3 && (A.dim() != 3 || A.size(0) != B.size(0)))) Py_RETURN_NONE;
    const int64_t batch = B.dim() == 3 ? B.size(0) : 1, M = rows / batch;      // (one weight for all batches: their rows are rows of one product)
    if (M > MX4_ROWS || N > MX4_ROWS || K > MX4_CONTRACTED || batch > 65535) Py_RETURN_NONE;
    int status;
    {
        const GilReleased released;
        const at::ScalarType type = wide ? at::kFloat : at::kBFloat16;
        out = A.dim() == 2 ? fresh({M, N}, type) : fresh({A.size(0), A.size(1), N}, type);
        const int64_t need = mx4_gemm_workspace(batch, M, N, K);
        c10::optional<Workspace> workspace;
        if (need > 0) workspace.emplace(need, A.device(), at::TensorOptions().dtype(at::kByte).device(A.device()));
        status = mx4_gemm_entry(&a, batch > 1 ? M : 0, &b, batch > 1 ? N : 0, out.data_ptr(), N, M * N, batch, M, N, K, wide ? 1 : 0, workspace ? workspace->p : nullptr, need,
                                stream_of(stream));
    }
    if (status != TI8_OK) return Py_BuildValue("(si)", "ti8_mx4_gemm_nt", status);
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// mx4_gemm_nt_multi(A, scales of A, B, scales of B, of the next product likewise .., stream) -> [C ..] in bf16
PyObject* mx4_gemm_nt_multi(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    const int count = (int)(nargs - 1) / 4;
    int64_t stream;
    if (count < 1 || count > 3 || nargs != 4 * count + 1 || !number(args[4 * count], &stream)) Py_RETURN_NONE;
    at::Tensor t[12], out[3];
    at::Tensor* tensors[12];
    for (int i = 0; i < 4 * count; ++i) tensors[i] = &t[i];
    if (!tensors_of(args, tensors, 4 * count)) Py_RETURN_NONE;
    ti8_mx4_gemm_problem p[3] = {};
    for (int i = 0; i < count; ++i) {
        const at::Tensor *A = &t[4 * i], *B = &t[4 * i + 2];
        if (!mx4_operand(A[0], A[1], current_device(), &p[i].a) || !mx4_operand(B[0], B[1], current_device(), &p[i].b) || A->dim() != 2 || B->dim() != 2 || A->size(1) != B->size(1)) Py_RETURN_NONE;
        p[i].M = A->size(0);
        p[i].N = p[i].ldc = B->size(0);
        p[i].K = A->size(1) * 2;
    }
    const int64_t need = mx4_multi_workspace(p, count);
    if (need < 0) Py_RETURN_NONE;
    int status;
    {
        const GilReleased released;
        c10::optional<Workspace> workspace;
        if (need > 0) workspace.emplace(need, t[0].device(), at::TensorOptions().dtype(at::kByte).device(t[0].device()));
        for (int i = 0; i < count; ++i) {
            out[i] = fresh({p[i].M, p[i].N}, at::kBFloat16);
            p[i].c = out[i].data_ptr();
        }
        status = mx4_multi_entry(p, count, workspace ? workspace->p : nullptr, need, stream_of(stream));
    }
    if (status != TI8_OK) return Py_BuildValue("(si)", "ti8_mx4_gemm_nt_multi", status);
    PyObject* const list = PyList_New(count);
    if (!list) return nullptr;
    for (int i = 0; i < count; ++i) PyList_SET_ITEM(list, i, wrap(out[i]));
    return list;
    END_HANDLE_TH_ERRORS
}

// mx4_linear_fwd_bwd(X [.., K], W, dY [.., N], stream) -> [Y, dX, dW]
PyObject* mx4_linear_fwd_bwd(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    at::Tensor X, W, dY, Y, dX, dW;
    at::Tensor* const tensors[] = {&X, &W, &dY};
    int64_t stream;
    if (nargs != 4 || !tensors_of(args, tensors, 3) || !number(args[3], &stream)) Py_RETURN_NONE;
    // rows apart, or in a tensor of other dimensions dense
    int64_t ld[3];
    for (int i = 0; i < 3; ++i) {
        const at::Tensor& t = *tensors[i];
        if (!on(t, at::kBFloat16, current_device()) || t.dim() < 1 || (t.dim() == 2 ? t.stride(1) != 1 || t.stride(0) < t.size(1) : !t.is_contiguous())) Py_RETURN_NONE;
        ld[i] = t.dim() == 2 ? t.stride(0) : t.size(-1);
    }
    if (W.dim() != 2 || dY.dim() != X.dim() || dY.sizes().slice(0, dY.dim() - 1) != X.sizes().slice(0, X.dim() - 1)) Py_RETURN_NONE;
    const int64_t K = X.size(-1), T = X.numel() / K, N = W.size(0);
    if (W.size(1) != K || dY.size(-1) != N) Py_RETURN_NONE;
    const int64_t need = mx4_step_workspace(T, K, N);
    if (need < 0) Py_RETURN_NONE;
    int status;
    {
        const GilReleased released;
        Y = fresh(dY.sizes(), at::kBFloat16);
        dX = fresh(X.sizes(), at::kBFloat16);
        dW = fresh({N, K}, at::kBFloat16);
        const Workspace workspace(need, X.device(), at::TensorOptions().dtype(at::kByte).device(X.device()));
        status = mx4_step_entry(X.data_ptr(), ld[0], W.data_ptr(), ld[1], dY.data_ptr(), ld[2], Y.data_ptr(), dX.data_ptr(), dW.data_ptr(), T, K, N,
                                workspace.p, need, stream_of(stream));
    }
    if (status != TI8_OK) return Py_BuildValue("(si)", "ti8_mx4_linear_fwd_bwd", status);
    return Py_BuildValue("[NNN]", wrap(Y), wrap(dX), wrap(dW));
    END_HANDLE_TH_ERRORS
}

// rmsnorm_quant(x, weight, residual, eps, whether in 4 bits, group, inv_mode, qflags, stream) -> [q, s, rstd] or [q, s, rstd, h]
PyObject* rmsnorm_quant(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    at::Tensor x, w, r, q, s, rstd, h;
    at::Tensor* const tensors[] = {&x, &w, &r};
    int64_t mx, group, inv_mode, qflags, stream;
    if (nargs != 9 || !tensors_of(args, tensors, 3) || !PyFloat_CheckExact(args[3]) || !number(args[4], &mx) || !number(args[5], &group) || !number(args[6], &inv_mode) ||
        !number(args[7], &qflags) || !number(args[8], &stream))
        Py_RETURN_NONE;
    const c10::DeviceIndex device = current_device();
    const auto dense = [&](const at::Tensor& t) { return on(t, at::kBFloat16, device) && t.is_contiguous() && at_multiple(t, 16) && !derived(t); };
    if (!dense(x) || !dense(w) || (r.defined() && (!dense(r) || r.sizes() != x.sizes())) || x.dim() < 1 || w.dim() != 1) Py_RETURN_NONE;
    const int64_t dim = x.size(-1), rows = x.numel() / dim;
    if (w.size(0) != dim || dim % (mx ? 8 : 128) || dim > 16384 || rows > (dim > 1024 ? (1 << 24) - 1 : (1 << 26) - 4) || (group != 0 && (group != 128 || mx))) Py_RETURN_NONE;
    int status;
    {
        const GilReleased released;
        const at::IntArrayRef lead = x.sizes().slice(0, x.dim() - 1);
        ti8_rmsnorm_quant_args a = {};
        Mx4Out out;
        Room room(Room::of(rows * 4) + (r.defined() ? Room::of(rows * dim * 2) : 0) + (mx ? Room::of_mx4(rows, dim) : Room::of(rows * dim) + Room::of(group ? rows * (dim / 128) * 4 : rows * 4)));
        rstd = room(lead, at::kFloat);
        if (r.defined()) h = room(x.sizes(), at::kBFloat16);
        if (mx) {
            out = Mx4Out(room, lead, rows, dim);
            q = out.codes;
            s = out.scales;
            a.mx4 = out.mx;
        } else {
            q = room(x.sizes(), at::kChar);
            c10::SmallVector<int64_t, 4> sizes(lead.begin(), lead.end());
            if (group) sizes.push_back(dim / 128);
            s = room(sizes, at::kFloat);
            a.q = static_cast<int8_t*>(q.data_ptr());
            a.ldq = dim;
            a.s = static_cast<float*>(s.data_ptr());
        }
        a.x = x.data_ptr(); a.ldx = dim;
        a.w = w.data_ptr();
        if (r.defined()) {
            a.residual = r.data_ptr(); a.ldr = dim;
            a.h = h.data_ptr(); a.ldh = dim;
        }
        a.rstd = static_cast<float*>(rstd.data_ptr());
        a.rows = rows; a.dim = dim; a.eps = PyFloat_AS_DOUBLE(args[3]);
        a.group = (int)group; a.qflags = (int)qflags; a.inv_mode = (int)inv_mode;
        status = rmsnorm_quant_entry(&a, stream_of(stream));
    }
    if (status != TI8_OK) return Py_BuildValue("(si)", "ti8_rmsnorm_quant", status);
    if (r.defined()) return Py_BuildValue("[NNNN]", wrap(q), wrap(s), wrap(rstd), wrap(h));
    return Py_BuildValue("[NNN]", wrap(q), wrap(s), wrap(rstd));
    END_HANDLE_TH_ERRORS
}

// dequant_row(q, s, stream) -> y
PyObject* dequant_row(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    at::Tensor q, s, y;
    at::Tensor* const tensors[] = {&q, &s};
    int64_t stream;
    if (nargs != 3 || !tensors_of(args, tensors, 2) || !number(args[2], &stream)) Py_RETURN_NONE;
    const c10::DeviceIndex device = current_device();
    if (!on(q, at::kChar, device) || !on(s, at::kFloat, device) || q.dim() < 1 || !q.is_contiguous() || !s.is_contiguous() || !at_multiple(q, 8)) Py_RETURN_NONE;
    const int64_t cols = q.size(-1), rows = q.numel() / cols;
    const at::IntArrayRef lead = q.sizes().slice(0, q.dim() - 1);
    const bool by_group = s.sizes() != lead;
    if (cols % 8 || rows > MX4_ROWS || cols > MX4_ROWS ||
        (by_group && (cols % 128 || s.dim() != q.dim() || s.sizes().slice(0, q.dim() - 1) != lead || s.size(-1) != cols / 128)))
        Py_RETURN_NONE;
    int status;
    {
        const GilReleased released;
        y = fresh(q.sizes(), at::kBFloat16);
        status = dequant_row_entry(static_cast<const int8_t*>(q.data_ptr()), cols, static_cast<const float*>(s.data_ptr()), rows, cols, by_group ? 128 : 0, y.data_ptr(), cols,
                                   stream_of(stream));
    }
    if (status != TI8_OK) return Py_BuildValue("(si)", "ti8_dequant_row", status);
    return wrap(y);
    END_HANDLE_TH_ERRORS
}

// set_up_mx4(addresses of ti8_mx4_quant, ti8_mx4_dequant, ti8_mx4_gemm_nt, ti8_mx4_gemm_nt_workspace, ti8_mx4_gemm_nt_multi, ti8_mx4_gemm_nt_multi_workspace, ti8_mx4_linear_fwd_bwd,
// ti8_mx4_linear_fwd_bwd_workspace, ti8_rmsnorm_quant, ti8_dequant_row)
PyObject* set_up_mx4(PyObject*, PyObject* args) {
    unsigned long long q, d, g, w, m, v, t, u, n, r;
    if (!PyArg_ParseTuple(args, "KKKKKKKKKK", &q, &d, &g, &w, &m, &v, &t, &u, &n, &r)) return nullptr;
    mx4_multi_entry = reinterpret_cast<decltype(mx4_multi_entry)>(m);
    mx4_multi_workspace = reinterpret_cast<decltype(mx4_multi_workspace)>(v);
    mx4_step_entry = reinterpret_cast<decltype(mx4_step_entry)>(t);
    mx4_step_workspace = reinterpret_cast<decltype(mx4_step_workspace)>(u);
    mx4_quant_entry = reinterpret_cast<decltype(mx4_quant_entry)>(q);
    mx4_dequant_entry = reinterpret_cast<decltype(mx4_dequant_entry)>(d);
    mx4_gemm_entry = reinterpret_cast<decltype(mx4_gemm_entry)>(g);
    mx4_gemm_workspace = reinterpret_cast<decltype(mx4_gemm_workspace)>(w);
    rmsnorm_quant_entry = reinterpret_cast<decltype(rmsnorm_quant_entry)>(n);
    dequant_row_entry = reinterpret_cast<decltype(dequant_row_entry)>(r);
    Py_RETURN_NONE;
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
    {"mx4_quant", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(mx4_quant)), METH_FASTCALL, nullptr},
    {"mx4_dequant", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(mx4_dequant)), METH_FASTCALL, nullptr},
    {"mx4_gemm_nt", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(mx4_gemm_nt)), METH_FASTCALL, nullptr},
    {"mx4_gemm_nt_multi", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(mx4_gemm_nt_multi)), METH_FASTCALL, nullptr},
    {"mx4_linear_fwd_bwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(mx4_linear_fwd_bwd)), METH_FASTCALL, nullptr},
    {"rmsnorm_quant", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rmsnorm_quant)), METH_FASTCALL, nullptr},
    {"dequant_row", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(dequant_row)), METH_FASTCALL, nullptr},
    {"set_up", set_up, METH_VARARGS, nullptr},
    {"set_up_cache4", set_up_cache4, METH_VARARGS, nullptr},
    {"set_up_mx4", set_up_mx4, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// built_for: what the code above was compiled against, for whoever loads it to compare (fields of torch's and Python's objects and of the
// library's argument blocks are read and written here without a call)
PyMODINIT_FUNC PyInit__native(void) {
    PyObject* const m = PyModule_Create(&module);
    PyObject* const built_for = Py_BuildValue("(s(ii)nnnnnn)", TI8_BUILT_FOR_TORCH, PY_MAJOR_VERSION, PY_MINOR_VERSION, (Py_ssize_t)sizeof(ti8_linear_args), (Py_ssize_t)sizeof(ti8_gemm_problem),
                                              (Py_ssize_t)sizeof(ti8_cache4), (Py_ssize_t)sizeof(ti8_mx4_operand), (Py_ssize_t)sizeof(ti8_mx4_gemm_problem), (Py_ssize_t)sizeof(ti8_rmsnorm_quant_args));
    if (m && (!built_for || PyModule_AddObject(m, "built_for", built_for) < 0)) {
        Py_XDECREF(built_for);
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
