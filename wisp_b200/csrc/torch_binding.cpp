// torch_binding.cpp -- the Python binding of the paged cache's calls (module _paged_torch).
//
// A decode step makes a few of these calls per layer on a few microseconds of GPU work each,
// so the tensors are checked and the argument structs built here instead of in Python.  (The
// same checks with ctypes took 20 to 25 us a call, this takes 3 to 5.)  The C ABI stays free of
// torch types: its functions are handed over by address, from the library that wisp_b200.lib
// loaded.

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <cstdio>
#include <new>
#include <vector>

#include "wisp_b200.h"

namespace {

decltype(&wisp_paged_attention_workspace_bytes) p_ws_bytes;
decltype(&wisp_paged_attention) p_attention;
decltype(&wisp_prefix_attention) p_prefix;
decltype(&wisp_rope_append) p_rope;
decltype(&wisp_pages_copy) p_copy;
PyObject* g_fail;  // Python callable that raises WispError(code, message, file, line)

PyObject* g_names[4];  // "q_start", "kv_len", "table", "max_q"

struct Refused {};  // a Python exception is set

[[noreturn]] void refuse(const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    PyErr_SetString(PyExc_ValueError, buf);
    throw Refused();
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s: a tensor is wanted, got %s", name, Py_TYPE(o)->tp_name);
        throw Refused();
    }
    return THPVariable_Unpack(o);
}

int dtype_of(const at::Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kFloat: return WISP_DTYPE_F32;
        case at::kHalf: return WISP_DTYPE_F16;
        case at::kBFloat16: return WISP_DTYPE_BF16;
        default: refuse("%s of %s (fp32, fp16 or bf16)", name, at::toString(t.scalar_type()));
    }
}


const int* ints(const at::Tensor& t, const char* name, int dim) {
    if (t.scalar_type() != at::kInt || t.dim() != dim || !t.is_cuda() || t.stride(dim - 1) != 1)
        refuse("%s: a contiguous int32 CUDA tensor of %d dimension(s) is wanted", name, dim);
    return static_cast<const int*>(t.data_ptr());
}

// These calls have no derivative, backward or forward.
void no_derivative(const at::Tensor& x, const char* name) {
    if (x.requires_grad() && c10::GradMode::is_enabled())
        refuse("%s asks for a gradient: these calls have none (use torch.no_grad())", name);
    if (x._fw_grad(/*level=*/0).defined())
        refuse("%s has a forward-mode tangent: these calls have none", name);
}

WispKvPages pages(const at::Tensor& k, const at::Tensor& v, int dim0) {
    if (k.dim() != dim0 || k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type() ||
        k.strides() != v.strides())
        refuse("k_pages and v_pages: two [%sn_pages, page_size, n_kv_heads, head_dim] tensors of one "
               "shape, layout and dtype are wanted", dim0 == 5 ? "n_layers, " : "");
    no_derivative(k, "k_pages");
    no_derivative(v, "v_pages");
    const int o = dim0 - 4;
    const int64_t n = k.size(o), page = k.size(o + 1), heads = k.size(o + 2), dim = k.size(o + 3);
    const bool one = page > 0 && heads > 0 && dim > 0;
    if (!one || (dim > 1 && k.stride(o + 3) != 1) || (heads > 1 && k.stride(o + 2) != dim) ||
        (page > 1 && k.stride(o + 1) != heads * dim))
        refuse("k_pages: a page's positions, heads and dims must be contiguous");
    if (!k.is_cuda() || v.device() != k.device())
        refuse("k_pages and v_pages must be on one CUDA device");
    const int dt = dtype_of(k, "k_pages");
    if (n > 0x7fffffff || page > 0x7fffffff || heads > 0x7fffffff || dim > 0x7fffffff)
        refuse("k_pages: a dimension passes 31 bits");
    WispKvPages P;
    P.k = k.data_ptr();
    P.v = v.data_ptr();
    P.page_stride = n > 1 ? k.stride(o) : page * heads * dim;
    P.n_pages = (int)n;
    P.page_size = (int)page;
    P.n_kv_heads = (int)heads;
    P.head_dim = (int)dim;
    P.dtype = dt;
    return P;
}

WispRows rows(const at::Tensor& x, const char* name, int64_t n, int64_t dim, const at::Device& dev) {
    if (x.dim() != 3 || x.size(0) != n || x.size(2) != dim)
        refuse("%s: [%lld, heads, %lld] is wanted", name, (long long)n, (long long)dim);
    const int64_t heads = x.size(1);
    if (x.stride(2) != 1 || (heads > 1 && x.stride(1) != dim))
        refuse("%s: a row's heads must be contiguous", name);
    if (x.device() != dev) refuse("%s is not on the pages' device", name);
    no_derivative(x, name);
    if (heads > 65535) refuse("%s: %lld heads", name, (long long)heads);
    WispRows R;
    R.base = x.data_ptr();
    R.stride = n > 1 ? x.stride(0) : heads * dim;
    R.n_heads = (int)heads;
    R.dtype = dtype_of(x, name);
    return R;
}

// q_start, kv_len, table, max_q
WispTokenBatch batch_parts(PyObject* const* a, int64_t n_tokens, at::Device* dev) {
    const at::Tensor &qs = tensor(a[0], "q_start"), &kl = tensor(a[1], "kv_len"),
                     &tb = tensor(a[2], "table");
    WispTokenBatch B{};
    B.q_start = ints(qs, "q_start", 1);
    B.kv_len = ints(kl, "kv_len", 1);
    B.table = ints(tb, "table", 2);
    const int64_t n = kl.size(0);
    if (qs.size(0) != n + 1 || tb.size(0) != n)
        refuse("%lld sequences: q_start has %lld entries, table %lld rows", (long long)n,
               (long long)qs.size(0), (long long)tb.size(0));
    if (qs.device() != kl.device() || tb.device() != kl.device())
        refuse("q_start, kv_len and table are on different devices");
    const long mq = PyLong_AsLong(a[3]);
    if (mq == -1 && PyErr_Occurred()) throw Refused();
    const int64_t stride = n > 1 ? tb.stride(0) : tb.size(1);
    if (mq < 0 || mq > 0x7fffffff || n >= 0x7fffffff || n_tokens > 0x7fffffff ||
        stride > 0x7fffffff || tb.size(1) > stride)
        refuse("a batch of %lld sequences, %lld tokens, max_q %ld, table rows %lld apart",
               (long long)n, (long long)n_tokens, mq, (long long)stride);
    B.n_seq = (int)n;
    B.n_tokens = (int)n_tokens;
    B.max_q = (int)mq;
    B.table_stride = (int)stride;
    B.table_width = (int)tb.size(1);
    *dev = kl.device();
    return B;
}

// The same from a TokenBatch (its attributes, as they are at the time of the call).
WispTokenBatch batch_of(PyObject* batch, int64_t n_tokens, at::Device* dev) {
    PyObject* a[4] = {};
    struct Held {
        PyObject** a;
        ~Held() {
            for (int i = 0; i < 4; ++i) Py_XDECREF(a[i]);
        }
    } held{a};
    for (int i = 0; i < 4; ++i)
        if (!(a[i] = PyObject_GetAttr(batch, g_names[i]))) throw Refused();
    return batch_parts(a, n_tokens, dev);
}

int* status_word(PyObject* o, const at::Device& dev) {
    if (o == Py_None) return nullptr;
    const at::Tensor& w = tensor(o, "status");
    const int* p = ints(w, "status", 1);
    if (w.size(0) != 1 || w.device() != dev)
        refuse("status: one int32 value on the pages' device is wanted");
    return const_cast<int*>(p);
}

cudaStream_t stream_on(const at::Device& dev) {
    if (c10::cuda::current_device() != dev.index())
        refuse("tensors on cuda:%d, but the current device is cuda:%d", dev.index(),
               c10::cuda::current_device());
    return c10::cuda::getCurrentCUDAStream().stream();
}

void checked(WispError rc, const WispErrCtx& err) {
    if (rc == WISP_OK) return;
    PyObject* r = PyObject_CallFunction(g_fail, "isyi", (int)rc, err.message,
                                        err.file ? err.file : "", err.line);
    Py_XDECREF(r);
    throw Refused();
}

int as_int(PyObject* o, const char* name) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused();
    if (v < -0x7fffffff || v > 0x7fffffff) refuse("%s: %ld", name, v);
    return (int)v;
}

template <typename F>
PyObject* guarded(F f) {
    try {
        return f();
    } catch (const Refused&) {
    } catch (const std::bad_alloc&) {
        PyErr_NoMemory();
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

#define WANT_ARGS(name, n)                                                             \
    if (nargs != (n)) {                                                                \
        PyErr_Format(PyExc_TypeError, name " takes %d arguments, got %zd", (n), nargs); \
        return nullptr;                                                                \
    }

// check_batch(q_start, kv_len, table, max_q)
PyObject* check_batch(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    WANT_ARGS("check_batch", 4)
    return guarded([&]() -> PyObject* {
        at::Device dev(at::kCUDA);
        batch_parts(a, 0, &dev);
        Py_RETURN_NONE;
    });
}

// workspace_bytes(q, k_pages, v_pages, batch, n_groups)
PyObject* workspace_bytes(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    WANT_ARGS("workspace_bytes", 5)
    return guarded([&]() -> PyObject* {
        const at::Tensor& q = tensor(a[0], "q");
        const WispKvPages P = pages(tensor(a[1], "k_pages"), tensor(a[2], "v_pages"), 4);
        const WispRows R = rows(q, "q", q.dim() ? q.size(0) : 0, P.head_dim,
                                tensor(a[1], "k_pages").device());
        at::Device dev(at::kCUDA);
        const WispTokenBatch B = batch_of(a[3], q.size(0), &dev);
        return PyLong_FromSize_t(p_ws_bytes(&P, &B, R.n_heads, R.dtype, as_int(a[4], "n_groups")));
    });
}

// attend(q, k_pages, v_pages, batch, groups, prefix_len, out, scale, window, sinks, return_lse,
//        workspace, status)
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    WANT_ARGS("attend", 13)
    return guarded([&]() -> PyObject* {
        const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k_pages"),
                         &v = tensor(a[2], "v_pages");
        const WispKvPages P = pages(k, v, 4);
        const at::Device dev = k.device();
        const int64_t T = q.dim() ? q.size(0) : 0;
        const WispRows rq = rows(q, "q", T, P.head_dim, dev);
        at::Device bdev(at::kCUDA);
        WispTokenBatch B = batch_of(a[3], T, &bdev);
        if (bdev != dev) refuse("the batch is not on the pages' device");
        B.status = status_word(a[12], dev);
        const cudaStream_t s = stream_on(dev);
        int n_groups = 0;
        const int *groups = nullptr, *prefix = nullptr;
        if (a[4] != Py_None) {
            const at::Tensor &g = tensor(a[4], "groups"), &p = tensor(a[5], "prefix_len");
            groups = ints(g, "groups", 1);
            prefix = ints(p, "prefix_len", 1);
            if (g.size(0) != p.size(0) + 1 || p.size(0) == 0 || g.device() != dev ||
                p.device() != dev || p.size(0) > 0x7ffffffe)
                refuse("groups of %lld entries, prefix_len of %lld (one more and at least one, on the "
                       "pages' device)", (long long)g.size(0), (long long)p.size(0));
            n_groups = (int)p.size(0);
        }
        const at::TensorOptions opt = q.options().requires_grad(false);
        at::Tensor out = a[6] == Py_None ? at::empty(q.sizes(), opt) : tensor(a[6], "out");
        const WispRows ro = rows(out, "out", T, P.head_dim, dev);
        float scale = 0.f;
        if (a[7] == Py_None) {
            scale = 1.f / sqrtf((float)P.head_dim);
        } else {
            const double x = PyFloat_AsDouble(a[7]);
            if (x == -1.0 && PyErr_Occurred()) throw Refused();
            scale = (float)x;
        }
        const int window = as_int(a[8], "window"), sinks = as_int(a[9], "sinks");
        const int want_lse = PyObject_IsTrue(a[10]);
        if (want_lse < 0) throw Refused();
        at::Tensor lse, ws;
        if (want_lse) lse = at::empty({T, (int64_t)rq.n_heads}, opt.dtype(at::kFloat));
        if (a[11] == Py_None) {
            ws = at::empty({(int64_t)p_ws_bytes(&P, &B, rq.n_heads, rq.dtype, n_groups)},
                           opt.dtype(at::kByte));
        } else {
            ws = tensor(a[11], "workspace");
            if (ws.scalar_type() != at::kByte || ws.device() != dev || !ws.is_contiguous())
                refuse("workspace: a contiguous uint8 tensor on the pages' device is wanted");
        }
        WispErrCtx err{};
        float* lp = want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
        const WispError rc =
            n_groups ? p_prefix(&rq, &ro, lp, &P, &B, groups, prefix, n_groups, scale, window, sinks,
                                ws.data_ptr(), ws.numel(), s, &err)
                     : p_attention(&rq, &ro, lp, &P, &B, scale, window, sinks, ws.data_ptr(),
                                   ws.numel(), s, &err);
        checked(rc, err);
        PyObject* o = THPVariable_Wrap(out);
        if (!want_lse || !o) return o;
        PyObject* z = THPVariable_Wrap(lse);
        if (!z) {
            Py_DECREF(o);
            return nullptr;
        }
        PyObject* both = PyTuple_Pack(2, o, z);
        Py_DECREF(o);
        Py_DECREF(z);
        return both;
    });
}

// rope_append(q, k, v, k_pages, v_pages, batch, inv_freq, q_out, offset, interleaved, gain,
//             positions, status)
PyObject* rope_append(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    WANT_ARGS("rope_append", 13)
    return guarded([&]() -> PyObject* {
        const at::Tensor &q = tensor(a[0], "q"), &kp = tensor(a[3], "k_pages");
        const WispKvPages P = pages(kp, tensor(a[4], "v_pages"), 4);
        const at::Device dev = kp.device();
        const int64_t T = q.dim() ? q.size(0) : 0;
        const WispRows rq = rows(q, "q", T, P.head_dim, dev);
        const WispRows rk = rows(tensor(a[1], "k"), "k", T, P.head_dim, dev);
        const WispRows rv = rows(tensor(a[2], "v"), "v", T, P.head_dim, dev);
        at::Device bdev(at::kCUDA);
        const WispTokenBatch B = batch_of(a[5], T, &bdev);
        if (bdev != dev) refuse("the batch is not on the pages' device");
        const cudaStream_t s = stream_on(dev);
        const at::Tensor& f = tensor(a[6], "inv_freq");
        if (f.scalar_type() != at::kDouble || f.dim() != 1 || f.device() != dev ||
            !f.is_contiguous() || f.size(0) > 4096)
            refuse("inv_freq: a contiguous float64 vector on the pages' device is wanted");
        at::Tensor out = a[7] == Py_None ? at::empty(q.sizes(), q.options().requires_grad(false))
                                          : tensor(a[7], "q_out");
        const WispRows ro = rows(out, "q_out", T, P.head_dim, dev);
        WispRope R{};
        R.inv_freq = static_cast<const double*>(f.data_ptr());
        R.dim = 2 * (int)f.size(0);
        R.offset = as_int(a[8], "offset");
        R.interleaved = PyObject_IsTrue(a[9]);
        const double gain = PyFloat_AsDouble(a[10]);
        if (R.interleaved < 0 || (gain == -1.0 && PyErr_Occurred())) throw Refused();
        R.gain = (float)gain;
        if (a[11] != Py_None) {
            const at::Tensor& p = tensor(a[11], "positions");
            R.positions = ints(p, "positions", 1);
            if (p.size(0) != T || p.device() != dev)
                refuse("positions: %lld int32 values on the pages' device are wanted", (long long)T);
        }
        int* status = status_word(a[12], dev);
        WispErrCtx err{};
        checked(p_rope(&rq, &rk, &rv, &ro, &P, &B, &R, status, s, &err), err);
        return THPVariable_Wrap(out);
    });
}

std::vector<int> int_list(PyObject* o, const char* name) {
    PyObject* seq = PySequence_Fast(o, "copy_pages: sequences of page numbers are wanted");
    if (!seq) throw Refused();
    std::vector<int> v;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
    bool ok = n <= 0x7fffffff;
    try {
        v.resize(ok ? n : 0);
    } catch (...) {
        Py_DECREF(seq);
        throw;
    }
    for (Py_ssize_t i = 0; ok && i < n; ++i) {
        const long x = PyLong_AsLong(PySequence_Fast_GET_ITEM(seq, i));
        if (x == -1 && PyErr_Occurred()) ok = false;
        v[i] = x < 0 || x > 0x7fffffff ? -1 : (int)x;
    }
    Py_DECREF(seq);
    if (PyErr_Occurred()) throw Refused();
    if (!ok) refuse("%s: too many pages", name);
    return v;
}

// copy_pages(k_pages, v_pages, src, dst)
PyObject* copy_pages(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    WANT_ARGS("copy_pages", 4)
    return guarded([&]() -> PyObject* {
        const at::Tensor &k = tensor(a[0], "k_pages"), &v = tensor(a[1], "v_pages");
        const int dim = k.dim() == 5 ? 5 : 4;
        const WispKvPages P = pages(k, v, dim);
        const int64_t layers = dim == 5 ? k.size(0) : 1;
        if (layers == 0 || layers > 32767) refuse("copy_pages: %lld layers", (long long)layers);
        const std::vector<int> s = int_list(a[2], "src"), d = int_list(a[3], "dst");
        if (s.size() != d.size())
            refuse("copy_pages: %zu sources, %zu destinations", s.size(), d.size());
        const cudaStream_t stream = stream_on(k.device());
        WispErrCtx err{};
        checked(p_copy(&P, (int)layers, layers > 1 ? k.stride(0) : 0, s.data(), d.data(),
                       (int)s.size(), stream, &err),
                err);
        Py_RETURN_NONE;
    });
}

// init(workspace_bytes, attention, prefix_attention, rope_append, pages_copy, fail)
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    WANT_ARGS("init", 6)
    void* p[5];
    for (int i = 0; i < 5; ++i) {
        p[i] = PyLong_AsVoidPtr(a[i]);
        if (PyErr_Occurred()) return nullptr;
    }
    p_ws_bytes = reinterpret_cast<decltype(p_ws_bytes)>(p[0]);
    p_attention = reinterpret_cast<decltype(p_attention)>(p[1]);
    p_prefix = reinterpret_cast<decltype(p_prefix)>(p[2]);
    p_rope = reinterpret_cast<decltype(p_rope)>(p[3]);
    p_copy = reinterpret_cast<decltype(p_copy)>(p[4]);
    Py_INCREF(a[5]);
    Py_XSETREF(g_fail, a[5]);
    Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"init", FAST(init)},
                         {"check_batch", FAST(check_batch)},
                         {"workspace_bytes", FAST(workspace_bytes)},
                         {"attend", FAST(attend)},
                         {"rope_append", FAST(rope_append)},
                         {"copy_pages", FAST(copy_pages)},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_torch", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" PyObject* PyInit__paged_torch(void) {
    const char* names[4] = {"q_start", "kv_len", "table", "max_q"};
    for (int i = 0; i < 4; ++i)
        if (!(g_names[i] = PyUnicode_InternFromString(names[i]))) return nullptr;
    return PyModule_Create(&module);
}
