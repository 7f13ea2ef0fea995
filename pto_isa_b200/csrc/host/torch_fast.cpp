// The serving operators' calls without the interpreter's share of them.
//
// pto_isa_b200/ops.py checks every argument and calls the C ABI through ctypes, which takes 15 to 30 us for a call with a
// cache: more than a decode step's kernels.  Each function here takes a call whose arguments are in order, makes its
// outputs and calls the same C entry point; for anything else (a wrong shape or type, a tensor on another device than the
// current one, an entry point that reports an error) it returns None and ops.py goes through its own checks, which name
// the fault or serve the unusual call.  It accepts nothing that ops.py refuses.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "../../../include/pto_b200.h"

namespace {

struct Unusual {}; // leave the call to ops.py

inline void need(bool ok)
{
    if (!ok) {
        throw Unusual{};
    }
}

inline const at::Tensor &tensor(PyObject *o, int device)
{
    need(THPVariable_Check(o));
    const at::Tensor &t = THPVariable_Unpack(o);
    need(t.layout() == at::kStrided && t.is_cuda() && t.get_device() == device);
    return t;
}

inline int dtype16(const at::Tensor &t)
{
    need(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16);
    return t.scalar_type() == at::kHalf ? PTO_B200_DTYPE_F16 : PTO_B200_DTYPE_BF16;
}

inline bool aligned16(const void *p)
{
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}

// the last dimension contiguous, the others' strides (0 where the extent is 1) multiples of 8 elements
inline void row_strides(const at::Tensor &t, int64_t *out)
{
    const int64_t n = t.dim();
    need((t.size(n - 1) <= 1 || t.stride(n - 1) == 1) && aligned16(t.data_ptr()));
    for (int64_t i = 0; i + 1 < n; ++i) {
        out[i] = t.size(i) > 1 ? t.stride(i) : 0;
        need((out[i] & 7) == 0);
    }
}

struct Cache {
    pto_b200_kv_cache c;
};

inline Cache cache(PyObject *o, int device)
{
    need(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 5);
    const long fmt = PyLong_AsLong(PyTuple_GET_ITEM(o, 4));
    need(fmt >= PTO_B200_KV_F16 && fmt <= PTO_B200_KV_MXFP4);
    const bool mx = fmt >= PTO_B200_KV_MXFP8;
    const at::Tensor &k = tensor(PyTuple_GET_ITEM(o, 0), device), &v = tensor(PyTuple_GET_ITEM(o, 1), device);
    need(k.dim() == 4 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() && k.is_contiguous() && v.is_contiguous());
    need(mx ? k.element_size() == 1 : k.scalar_type() == (fmt == PTO_B200_KV_F16 ? at::kHalf : at::kBFloat16));
    const int64_t d = fmt == PTO_B200_KV_MXFP4 ? 2 * k.size(3) : k.size(3);
    need((d == 64 || d == 128) && k.size(1) >= 1 && k.size(1) <= 0x7fffffff && k.size(2) <= 1024);
    Cache r;
    r.c = pto_b200_kv_cache{k.data_ptr(), v.data_ptr(), nullptr, nullptr, k.size(0), static_cast<int32_t>(fmt),
                            static_cast<int32_t>(k.size(1)), static_cast<int32_t>(k.size(2)), static_cast<int32_t>(d)};
    if (mx) {
        const at::Tensor &ks = tensor(PyTuple_GET_ITEM(o, 2), device), &vs = tensor(PyTuple_GET_ITEM(o, 3), device);
        for (const at::Tensor *s : {&ks, &vs}) {
            need(s->dim() == 4 && s->size(0) == k.size(0) && s->size(1) == k.size(1) && s->size(2) == k.size(2) &&
                 s->size(3) == d / 32 && s->element_size() == 1 && s->is_contiguous());
        }
        r.c.k_scale = static_cast<uint8_t *>(ks.data_ptr());
        r.c.v_scale = static_cast<uint8_t *>(vs.data_ptr());
    } else {
        need(PyTuple_GET_ITEM(o, 2) == Py_None && PyTuple_GET_ITEM(o, 3) == Py_None);
    }
    return r;
}

inline const at::Tensor &index_vector(PyObject *o, int device, int64_t n)
{
    const at::Tensor &t = tensor(o, device);
    need(t.scalar_type() == at::kInt && t.dim() == 1 && (n < 0 || t.size(0) == n) && t.is_contiguous());
    return t;
}

inline const at::Tensor &page_table(PyObject *o, int device, int64_t batch)
{
    const at::Tensor &t = tensor(o, device);
    need(t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == batch && (t.size(1) <= 1 || t.stride(1) == 1) &&
         t.size(1) <= 0x7fffffff);
    return t;
}

inline int64_t integer(PyObject *o)
{
    need(PyLong_Check(o));
    const long long v = PyLong_AsLongLong(o);
    need(!(v == -1 && PyErr_Occurred()));
    return v;
}

// a call's work, with every way out of it turned into None (ops.py takes over) but Python's own errors
template <class F>
PyObject *guarded(F &&f)
{
    try {
        return f();
    } catch (...) {
        PyErr_Clear();
    }
    Py_RETURN_NONE;
}

inline void *stream(int device)
{
    return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
}

// An output on the current device, and scratch memory for the current stream, from torch's allocator directly: 1 us each
// where a call through the dispatcher takes 2 (w4_matvec of 5 rows: 13 us of host time with at::empty, 6.7 so).
inline at::Tensor output(at::IntArrayRef size, at::ScalarType type, int device)
{
    return at::Tensor(at::detail::empty_cuda(size, type, at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(device)), std::nullopt));
}
inline c10::DataPtr scratch(int64_t bytes)
{
    return c10::cuda::CUDACachingAllocator::get()->allocate(static_cast<size_t>(bytes));
}

// (cache, k, v, slots) -> True
PyObject *fast_write(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded([&]() -> PyObject * {
        need(n == 4);
        const int device = c10::cuda::current_device();
        const Cache c = cache(args[0], device);
        const at::Tensor &k = tensor(args[1], device), &v = tensor(args[2], device);
        const int dtype = dtype16(k);
        need(k.dim() == 3 && k.sizes() == v.sizes() && v.scalar_type() == k.scalar_type() && k.size(1) == c.c.kv_heads && k.size(2) == c.c.head_dim);
        const at::Tensor &slots = index_vector(args[3], device, k.size(0));
        int64_t strides[4];
        row_strides(k, strides);
        row_strides(v, strides + 2);
        need(pto_b200_kv_cache_write(&c.c, k.data_ptr(), v.data_ptr(), dtype, slots.data_ptr<int32_t>(), k.size(0), strides, stream(device)) == 0);
        Py_RETURN_TRUE;
    });
}

// (cache, table, lens, max_len, bfloat16) -> (k, v)
PyObject *fast_read(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded([&]() -> PyObject * {
        need(n == 5);
        const int device = c10::cuda::current_device();
        const Cache c = cache(args[0], device);
        const at::Tensor &lens = index_vector(args[2], device, -1);
        const int64_t batch = lens.size(0), max_len = integer(args[3]);
        const at::Tensor &table = page_table(args[1], device, batch);
        need(max_len >= 0 && max_len <= 0x7fffffff && batch <= 0x7fffffff);
        const bool bf16 = args[4] == Py_True;
        const at::ScalarType type = bf16 ? at::kBFloat16 : at::kHalf;
        const int64_t size[4] = {batch, c.c.kv_heads, max_len, c.c.head_dim};
        at::Tensor k = output(size, type, device), v = output(size, type, device);
        need(pto_b200_kv_cache_read(&c.c, table.data_ptr<int32_t>(), batch > 1 ? table.stride(0) : 0, static_cast<int>(table.size(1)),
                                    lens.data_ptr<int32_t>(), static_cast<int>(batch), static_cast<int>(max_len), k.data_ptr(), v.data_ptr(),
                                    bf16 ? PTO_B200_DTYPE_BF16 : PTO_B200_DTYPE_F16, stream(device)) == 0);
        PyObject *r = PyTuple_New(2);
        PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(k)));
        PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(v)));
        return r;
    });
}

// (q, cache, prefix_pages, prefix_len, table, lens, scale or None, max_seq_len or None, return_lse) -> o or (o, lse)
PyObject *fast_attn(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded([&]() -> PyObject * {
        need(n == 9);
        const int device = c10::cuda::current_device();
        const at::Tensor &q = tensor(args[0], device);
        const Cache c = cache(args[1], device);
        const int dtype = dtype16(q);
        need((q.dim() == 3 || q.dim() == 4) && (c.c.format >= PTO_B200_KV_MXFP8 || c.c.format == (dtype == PTO_B200_DTYPE_F16 ? PTO_B200_KV_F16 : PTO_B200_KV_BF16)));
        int64_t s[3], strides[3];
        row_strides(q, s);
        const bool single = q.dim() == 3;
        strides[0] = s[0];
        strides[1] = single ? 0 : s[1];
        strides[2] = single ? s[1] : s[2];
        const int64_t batch = q.size(0), tokens = single ? 1 : q.size(1), heads = q.size(q.dim() - 2), d = q.size(q.dim() - 1);
        need(batch >= 1 && tokens >= 1 && heads >= 1 && d == c.c.head_dim && heads % c.c.kv_heads == 0 && batch <= (1 << 26) &&
             tokens <= (1 << 26) && heads <= (1 << 26));
        const at::Tensor &pages = index_vector(args[2], device, -1), &lens = index_vector(args[5], device, batch);
        const at::Tensor &table = page_table(args[4], device, batch);
        const int64_t prefix_len = integer(args[3]), covered = table.size(1) * c.c.page_size;
        const int64_t most = args[7] == Py_None ? covered : integer(args[7]);
        need(prefix_len >= 0 && prefix_len <= pages.size(0) * c.c.page_size && most >= 0 && most <= covered && prefix_len <= (1 << 30) && most <= (1 << 30));
        double scale = 1.0 / std::sqrt(static_cast<double>(d));
        if (args[6] != Py_None) {
            need(PyFloat_Check(args[6]));
            scale = PyFloat_AS_DOUBLE(args[6]);
        }
        const int64_t bytes = pto_b200_prefix_attn_workspace_bytes(static_cast<int>(batch), static_cast<int>(tokens), static_cast<int>(heads),
                                                                   c.c.kv_heads, static_cast<int>(d), static_cast<int>(prefix_len), static_cast<int>(most));
        at::Tensor o = output(q.sizes(), q.scalar_type(), device), lse;
        const c10::DataPtr workspace = scratch(bytes);
        const bool with_lse = args[8] == Py_True;
        if (with_lse) {
            lse = output(q.sizes().slice(0, q.dim() - 1), at::kFloat, device);
        }
        need(pto_b200_prefix_attn(&c.c, q.data_ptr(), dtype, strides, pages.data_ptr<int32_t>(), static_cast<int>(prefix_len), table.data_ptr<int32_t>(),
                                  batch > 1 ? table.stride(0) : 0, static_cast<int>(table.size(1)), lens.data_ptr<int32_t>(), static_cast<int>(most),
                                  static_cast<int>(batch), static_cast<int>(tokens), static_cast<int>(heads), static_cast<float>(scale), o.data_ptr(),
                                  with_lse ? lse.data_ptr<float>() : nullptr, workspace.get(), bytes, stream(device)) == 0);
        if (!with_lse) {
            return THPVariable_Wrap(std::move(o));
        }
        PyObject *r = PyTuple_New(2);
        PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(o)));
        PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(lse)));
        return r;
    });
}

// (x, w, scale, zero or None, out32) -> y
PyObject *fast_w4(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded([&]() -> PyObject * {
        need(n == 5);
        const int device = c10::cuda::current_device();
        const at::Tensor &x = tensor(args[0], device), &w = tensor(args[1], device), &scale = tensor(args[2], device);
        const int dtype = dtype16(x);
        need(x.dim() == 1 || x.dim() == 2);
        int64_t stride = 0;
        row_strides(x, &stride);
        const int64_t m = x.dim() == 1 ? 1 : x.size(0), k = x.size(x.dim() - 1), rows = w.size(0);
        need(w.dim() == 2 && w.element_size() == 1 && w.size(1) * 2 == k && w.is_contiguous() && scale.dim() == 2 && scale.size(0) == rows &&
             scale.size(1) >= 1 && k % scale.size(1) == 0 && scale.is_contiguous() && m <= 64 && rows <= 0x7fffffff && k <= 0x7fffffff);
        const int64_t group = k / scale.size(1);
        const bool mx = scale.element_size() == 1;
        need(mx ? group == 32 && args[3] == Py_None : scale.scalar_type() == x.scalar_type() && (group == 32 || group == 64 || group == 128));
        const void *zero = nullptr;
        if (args[3] != Py_None) {
            const at::Tensor &z = tensor(args[3], device);
            need(z.sizes() == scale.sizes() && z.scalar_type() == scale.scalar_type() && z.is_contiguous());
            zero = z.data_ptr();
        }
        const bool out32 = args[4] == Py_True;
        const int64_t size[2] = {m, rows};
        at::Tensor y = output(at::IntArrayRef(x.dim() == 1 ? size + 1 : size, size + 2), out32 ? at::kFloat : x.scalar_type(), device);
        const int64_t bytes = pto_b200_w4_matvec_workspace_bytes(static_cast<int>(m), static_cast<int>(k), mx ? PTO_B200_W4_MXFP4 : PTO_B200_W4_INT4);
        c10::DataPtr workspace;
        if (bytes > 0) {
            workspace = scratch(bytes);
        }
        need(pto_b200_w4_matvec(x.data_ptr(), stride, static_cast<const uint8_t *>(w.data_ptr()), scale.data_ptr(), zero, y.data_ptr(), static_cast<int>(m),
                                static_cast<int>(rows), static_cast<int>(k), static_cast<int>(group), mx ? PTO_B200_W4_MXFP4 : PTO_B200_W4_INT4, dtype,
                                out32 ? 1 : 0, workspace.get(), bytes, stream(device)) == 0);
        return THPVariable_Wrap(std::move(y));
    });
}

PyMethodDef methods[] = {
    {"kv_cache_write", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&fast_write)), METH_FASTCALL, nullptr},
    {"kv_cache_read", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&fast_read)), METH_FASTCALL, nullptr},
    {"prefix_attn", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&fast_attn)), METH_FASTCALL, nullptr},
    {"w4_matvec", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&fast_w4)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit__fast(void)
{
    return PyModule_Create(&module);
}
