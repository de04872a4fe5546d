// Minimal CPython binding of the per-call entry points: the launch path of
// FlashUlyssesContext.ulysses_qkv_forward passes 14 plain integers/floats per
// call, which ctypes converts in ~3 us and this METH_FASTCALL function in well
// under 1 us; the attention and cache calls pass up to 24.  Everything else
// (buffers, context creation, errors) stays on the ctypes binding of the same
// library.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cmath>
#include <cstdint>

#include "flash_ulysses_b200.h"

namespace {

inline void* as_ptr(PyObject* o) {
    return o == Py_None ? nullptr : PyLong_AsVoidPtr(o);
}

// forward(handle, x, w, positions, q_gamma, k_gamma, rope, local_tokens,
//         rope_rows, q_eps, k_eps, flags, stream, gemm_out) -> None
PyObject* forward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 14) {
        PyErr_SetString(PyExc_TypeError, "forward() takes 14 arguments");
        return nullptr;
    }
    fu_qkv_ctx* ctx = static_cast<fu_qkv_ctx*>(as_ptr(args[0]));
    const void* x = as_ptr(args[1]);
    const void* w = as_ptr(args[2]);
    const int64_t* pos = static_cast<const int64_t*>(as_ptr(args[3]));
    const float* qg = static_cast<const float*>(as_ptr(args[4]));
    const float* kg = static_cast<const float*>(as_ptr(args[5]));
    const float* rope = static_cast<const float*>(as_ptr(args[6]));
    const long long L = PyLong_AsLongLong(args[7]);
    const long long rows = PyLong_AsLongLong(args[8]);
    const double q_eps = PyFloat_AsDouble(args[9]);
    const double k_eps = PyFloat_AsDouble(args[10]);
    const unsigned long flags = PyLong_AsUnsignedLong(args[11]);
    void* stream = as_ptr(args[12]);
    void* gemm_out = as_ptr(args[13]);
    if (PyErr_Occurred()) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fu_qkv_forward(ctx, x, w, pos, qg, kg, rope, L, rows, q_eps, k_eps,
                        static_cast<uint32_t>(flags), stream, gemm_out);
    Py_END_ALLOW_THREADS
    if (rc != FU_OK) {
        PyErr_Format(PyExc_RuntimeError, "fu_qkv_forward failed (code %d): %s", rc,
                     fu_last_error());
        return nullptr;
    }
    Py_RETURN_NONE;
}

inline int64_t as_int(PyObject* o) { return PyLong_AsLongLong(o); }
inline int32_t as_i32(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v < INT32_MIN || v > INT32_MAX)
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_OverflowError, "argument exceeds 32 bits");
    return static_cast<int32_t>(v);
}
inline float as_float(PyObject* o) { return static_cast<float>(PyFloat_AsDouble(o)); }
inline const int32_t* as_ints(PyObject* o) { return static_cast<const int32_t*>(as_ptr(o)); }

PyObject* result(int rc, const char* what) {
    if (rc == FU_OK) Py_RETURN_NONE;
    PyErr_Format(PyExc_RuntimeError, "%s failed (code %d): %s", what, rc, fu_last_error());
    return nullptr;
}

// attention(device, q_heads, kv_heads, causal, tokens, q, k, v, out, q_stride,
//           k_stride, v_stride, out_stride, cu_seqlens, prefix_lens,
//           alibi_slopes, docs, scale, softcap, status, status_host,
//           timeout_ns, flags, stream) -> None
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    if (nargs != 24) {
        PyErr_SetString(PyExc_TypeError, "attention() takes 24 arguments");
        return nullptr;
    }
    fu_attention_args p = {};
    p.device = as_i32(a[0]);
    p.q_heads = as_i32(a[1]);
    p.kv_heads = as_i32(a[2]);
    p.causal = as_i32(a[3]);
    p.tokens = as_int(a[4]);
    p.q = as_ptr(a[5]);
    p.k = as_ptr(a[6]);
    p.v = as_ptr(a[7]);
    p.out = as_ptr(a[8]);
    p.q_stride = as_int(a[9]);
    p.k_stride = as_int(a[10]);
    p.v_stride = as_int(a[11]);
    p.out_stride = as_int(a[12]);
    p.cu_seqlens = as_ints(a[13]);
    p.prefix_lens = as_ints(a[14]);
    p.alibi_slopes = static_cast<const float*>(as_ptr(a[15]));
    p.docs = as_i32(a[16]);
    p.scale = as_float(a[17]);
    p.softcap = as_float(a[18]);
    p.status = static_cast<int32_t*>(as_ptr(a[19]));
    p.status_host = static_cast<int32_t*>(as_ptr(a[20]));
    p.timeout_ns = static_cast<uint64_t>(as_int(a[21]));
    const uint32_t flags = static_cast<uint32_t>(as_int(a[22]));
    void* stream = as_ptr(a[23]);
    if (PyErr_Occurred()) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fu_attention_forward(&p, flags, stream);
    Py_END_ALLOW_THREADS
    return result(rc, "fu_attention_forward");
}

// The arguments of fu_kvcache_append.
PyObject* kvcache_append(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    if (nargs != 14) {
        PyErr_SetString(PyExc_TypeError, "kvcache_append() takes 14 arguments");
        return nullptr;
    }
    const fu_kvcache* cache = static_cast<const fu_kvcache*>(as_ptr(a[0]));
    const void *k = as_ptr(a[1]), *v = as_ptr(a[2]);
    const int64_t k_stride = as_int(a[3]), v_stride = as_int(a[4]), tokens = as_int(a[5]);
    const int32_t *slots = as_ints(a[6]), *seq_lens = as_ints(a[7]), *cu = as_ints(a[8]);
    const int32_t seqs = as_i32(a[9]);
    int32_t* status = static_cast<int32_t*>(as_ptr(a[10]));
    int32_t* status_host = static_cast<int32_t*>(as_ptr(a[11]));
    const uint32_t flags = static_cast<uint32_t>(as_int(a[12]));
    void* stream = as_ptr(a[13]);
    if (PyErr_Occurred()) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fu_kvcache_append(cache, k, v, k_stride, v_stride, tokens, slots, seq_lens, cu, seqs,
                           status, status_host, flags, stream);
    Py_END_ALLOW_THREADS
    return result(rc, "fu_kvcache_append");
}

// The arguments of fu_kvcache_attention.
PyObject* kvcache_attention(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    if (nargs != 18) {
        PyErr_SetString(PyExc_TypeError, "kvcache_attention() takes 18 arguments");
        return nullptr;
    }
    const fu_kvcache* cache = static_cast<const fu_kvcache*>(as_ptr(a[0]));
    const void* q = as_ptr(a[1]);
    const int64_t q_stride = as_int(a[2]);
    void* out = as_ptr(a[3]);
    const int64_t out_stride = as_int(a[4]);
    const int32_t q_heads = as_i32(a[5]);
    const int32_t *slots = as_ints(a[6]), *seq_lens = as_ints(a[7]);
    const int32_t seqs = as_i32(a[8]);
    const float scale = as_float(a[9]), softcap = as_float(a[10]);
    const float* slopes = static_cast<const float*>(as_ptr(a[11]));
    void* workspace = as_ptr(a[12]);
    const int64_t bytes = as_int(a[13]);
    int32_t* status = static_cast<int32_t*>(as_ptr(a[14]));
    int32_t* status_host = static_cast<int32_t*>(as_ptr(a[15]));
    const uint32_t flags = static_cast<uint32_t>(as_int(a[16]));
    void* stream = as_ptr(a[17]);
    if (PyErr_Occurred()) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fu_kvcache_attention(cache, q, q_stride, out, out_stride, q_heads, slots, seq_lens, seqs,
                              scale, softcap, slopes, workspace, bytes, status, status_host, flags,
                              stream);
    Py_END_ALLOW_THREADS
    return result(rc, "fu_kvcache_attention");
}

// ------------------------------------------------------------ calls with tensors
// The attention and cache calls are a few microseconds on the GPU at decode sizes, as
// much as asking their tensors for shapes and strides in Python takes.  These functions
// read them through DLPack's C exchange API instead and make the call if everything
// fits.  They return False, having done nothing, for whatever does not: the caller then
// goes its ordinary way, which names the argument that is wrong.
//
// The structures are those of DLPack 1.x (dlpack.h), whose layout is stable.
struct DlTensor {
    void* data;
    int32_t device_type, device_id;
    int32_t ndim;
    uint8_t type_code, type_bits;
    uint16_t type_lanes;
    int64_t* shape;
    int64_t* strides;
    uint64_t byte_offset;
};
struct DlExchange {
    uint32_t major, minor;
    void* prev_api;
    void* allocator;
    void* from_py_object;
    void* to_py_object;
    int (*tensor_from_py_object)(void* object, DlTensor* out);
    int (*current_work_stream)(int device_type, int32_t device_id, void** stream);
};
enum : uint8_t { DL_INT = 0, DL_FLOAT = 2, DL_BFLOAT = 4 };
constexpr int32_t DL_CUDA = 2;

const DlExchange* exchange = nullptr;  // torch.Tensor's, set by use_exchange()
PyTypeObject* tensor_type = nullptr;

// use_exchange(torch.Tensor) -> bool
PyObject* use_exchange(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    if (nargs != 1 || !PyType_Check(a[0])) {
        PyErr_SetString(PyExc_TypeError, "use_exchange() takes the tensor type");
        return nullptr;
    }
    PyObject* capsule = PyObject_GetAttrString(a[0], "__dlpack_c_exchange_api__");
    if (capsule == nullptr) {
        PyErr_Clear();
        Py_RETURN_FALSE;
    }
    auto* api = static_cast<const DlExchange*>(PyCapsule_GetPointer(capsule, "dlpack_exchange_api"));
    Py_DECREF(capsule);                // (the type keeps it)
    if (api == nullptr) {
        PyErr_Clear();
        Py_RETURN_FALSE;
    }
    if (api->major != 1 || api->tensor_from_py_object == nullptr ||
        api->current_work_stream == nullptr)
        Py_RETURN_FALSE;
    Py_INCREF(a[0]);
    tensor_type = reinterpret_cast<PyTypeObject*>(a[0]);
    exchange = api;
    Py_RETURN_TRUE;
}

// A tensor of exactly the given type on the device; false also if it is none.
inline bool look(PyObject* o, int32_t device, DlTensor& t) {
    if (Py_TYPE(o) != tensor_type) return false;
    if (exchange->tensor_from_py_object(o, &t) != 0) {
        PyErr_Clear();
        return false;
    }
    return t.device_type == DL_CUDA && t.device_id == device && t.type_lanes == 1;
}

// BF16 [rows, width] with contiguous, 16-byte aligned rows.
struct RowsArg {
    char* ptr;
    int64_t rows, stride;
};
inline bool look_rows(PyObject* o, int32_t device, int64_t width, RowsArg& r) {
    DlTensor t;
    if (!look(o, device, t) || t.type_code != DL_BFLOAT || t.type_bits != 16 || t.ndim != 2 ||
        t.shape[1] != width || t.shape[0] < 1 || t.strides == nullptr)
        return false;
    r.ptr = static_cast<char*>(t.data) + t.byte_offset;
    r.rows = t.shape[0];
    r.stride = r.rows == 1 ? width : t.strides[0];
    return t.strides[1] == 1 && r.stride >= width && r.stride % 8 == 0 &&
           (reinterpret_cast<uintptr_t>(r.ptr) & 15) == 0;
}

// A contiguous vector; None is NULL with length 0.
inline bool look_vector(PyObject* o, int32_t device, uint8_t code, void*& ptr, int64_t& length) {
    ptr = nullptr;
    length = 0;
    if (o == Py_None) return true;
    DlTensor t;
    if (!look(o, device, t) || t.type_code != code || t.type_bits != 32 || t.ndim != 1 ||
        t.shape[0] < 1 || t.strides == nullptr || (t.shape[0] > 1 && t.strides[0] != 1))
        return false;
    ptr = static_cast<char*>(t.data) + t.byte_offset;
    length = t.shape[0];
    return true;
}

inline bool overlap(const RowsArg& a, int64_t a_width, const RowsArg& b, int64_t b_width) {
    return a.ptr < b.ptr + 2 * ((b.rows - 1) * b.stride + b_width) &&
           b.ptr < a.ptr + 2 * ((a.rows - 1) * a.stride + a_width);
}

inline bool as_number(PyObject* o, float& x) {
    const double d = PyFloat_AsDouble(o);
    if (d == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    x = static_cast<float>(d);
    return std::isfinite(d) && std::isfinite(x);
}

// True if launched; False for a refusal, which the ordinary way explains.
PyObject* launched(int rc, const char* what) {
    if (rc == FU_OK) Py_RETURN_TRUE;
    if (rc == FU_ERR_INVALID || rc == FU_ERR_DEVICE) Py_RETURN_FALSE;
    return result(rc, what);
}

// try_attention(device, q_heads, kv_heads, q, k, v, cu_seqlens, prefix_lens, alibi_slopes,
//               out, causal, scale, softcap, status, status_host) -> bool
PyObject* try_attention(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    if (nargs != 15) {
        PyErr_SetString(PyExc_TypeError, "try_attention() takes 15 arguments");
        return nullptr;
    }
    if (exchange == nullptr) Py_RETURN_FALSE;
    fu_attention_args p = {};
    p.device = as_i32(a[0]);
    p.q_heads = as_i32(a[1]);
    p.kv_heads = as_i32(a[2]);
    p.status = static_cast<int32_t*>(as_ptr(a[13]));
    p.status_host = static_cast<int32_t*>(as_ptr(a[14]));
    if (PyErr_Occurred()) return nullptr;
    const int64_t q_width = 128ll * p.q_heads, kv_width = 128ll * p.kv_heads;
    RowsArg q, k, v, out;
    void *cu, *prefix, *slopes, *stream;
    int64_t cu_length, prefix_length, slopes_length;
    const int causal = PyObject_IsTrue(a[10]);
    if (causal < 0) return nullptr;
    if (!look_rows(a[3], p.device, q_width, q) || !look_rows(a[4], p.device, kv_width, k) ||
        !look_rows(a[5], p.device, kv_width, v) || !look_rows(a[9], p.device, q_width, out) ||
        k.rows != q.rows || v.rows != q.rows || out.rows != q.rows || q.rows > (1 << 30) ||
        overlap(out, q_width, q, q_width) || overlap(out, q_width, k, kv_width) ||
        overlap(out, q_width, v, kv_width) ||
        !look_vector(a[6], p.device, DL_INT, cu, cu_length) ||
        !look_vector(a[7], p.device, DL_INT, prefix, prefix_length) ||
        !look_vector(a[8], p.device, DL_FLOAT, slopes, slopes_length) ||
        !as_number(a[11], p.scale) || !as_number(a[12], p.softcap) || p.softcap < 0.f)
        Py_RETURN_FALSE;
    const int64_t docs = cu != nullptr ? cu_length - 1 : 1;
    if (docs < 1 || docs > (1 << 30) || (prefix != nullptr && (!causal || prefix_length != docs)) ||
        (slopes != nullptr && slopes_length != p.q_heads) ||
        exchange->current_work_stream(DL_CUDA, p.device, &stream) != 0) {
        PyErr_Clear();
        Py_RETURN_FALSE;
    }
    p.causal = causal;
    p.tokens = q.rows;
    p.q = q.ptr;
    p.k = k.ptr;
    p.v = v.ptr;
    p.out = out.ptr;
    p.q_stride = q.stride;
    p.k_stride = k.stride;
    p.v_stride = v.stride;
    p.out_stride = out.stride;
    p.cu_seqlens = static_cast<const int32_t*>(cu);
    p.prefix_lens = static_cast<const int32_t*>(prefix);
    p.alibi_slopes = static_cast<const float*>(slopes);
    p.docs = static_cast<int32_t>(docs);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fu_attention_forward(&p, 0, stream);
    Py_END_ALLOW_THREADS
    return launched(rc, "fu_attention_forward");
}

// try_append(cache, k, v, slots, seq_lens, cu_seqlens, status, status_host) -> bool
PyObject* try_append(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    if (nargs != 8) {
        PyErr_SetString(PyExc_TypeError, "try_append() takes 8 arguments");
        return nullptr;
    }
    const fu_kvcache* cache = static_cast<const fu_kvcache*>(as_ptr(a[0]));
    int32_t* status = static_cast<int32_t*>(as_ptr(a[6]));
    int32_t* status_host = static_cast<int32_t*>(as_ptr(a[7]));
    if (PyErr_Occurred()) return nullptr;
    if (exchange == nullptr || cache == nullptr) Py_RETURN_FALSE;
    const int32_t device = cache->device;
    const int64_t width = 128ll * cache->kv_heads;
    RowsArg k, v;
    void *slots, *lens, *cu, *stream;
    int64_t count, lens_length, cu_length;
    if (!look_rows(a[1], device, width, k) || !look_rows(a[2], device, width, v) ||
        k.rows != v.rows || k.rows > (1 << 30) ||
        !look_vector(a[3], device, DL_INT, slots, count) ||
        !look_vector(a[4], device, DL_INT, lens, lens_length) ||
        !look_vector(a[5], device, DL_INT, cu, cu_length) || slots == nullptr || lens == nullptr ||
        lens_length != count || count > (1 << 24) ||
        (cu != nullptr ? cu_length != count + 1 : k.rows != count) ||
        exchange->current_work_stream(DL_CUDA, device, &stream) != 0) {
        PyErr_Clear();
        Py_RETURN_FALSE;
    }
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fu_kvcache_append(cache, k.ptr, v.ptr, k.stride, v.stride, k.rows,
                           static_cast<const int32_t*>(slots), static_cast<const int32_t*>(lens),
                           static_cast<const int32_t*>(cu), static_cast<int32_t>(count), status,
                           status_host, 0, stream);
    Py_END_ALLOW_THREADS
    return launched(rc, "fu_kvcache_append");
}

// try_decode(cache, q_heads, q, slots, seq_lens, alibi_slopes, out, work, scale, softcap,
//            status, status_host) -> bool; `work` is a contiguous BF16 vector
PyObject* try_decode(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    if (nargs != 12) {
        PyErr_SetString(PyExc_TypeError, "try_decode() takes 12 arguments");
        return nullptr;
    }
    const fu_kvcache* cache = static_cast<const fu_kvcache*>(as_ptr(a[0]));
    const int32_t q_heads = as_i32(a[1]);
    int32_t* status = static_cast<int32_t*>(as_ptr(a[10]));
    int32_t* status_host = static_cast<int32_t*>(as_ptr(a[11]));
    if (PyErr_Occurred()) return nullptr;
    if (exchange == nullptr || cache == nullptr) Py_RETURN_FALSE;
    const int32_t device = cache->device;
    const int64_t width = 128ll * q_heads;
    RowsArg q, out;
    DlTensor work;
    void *slots, *lens, *slopes, *stream;
    int64_t count, lens_length, slopes_length;
    float scale, softcap;
    if (!look_rows(a[2], device, width, q) || !look_rows(a[6], device, width, out) ||
        out.rows != q.rows || overlap(out, width, q, width) ||
        !look_vector(a[3], device, DL_INT, slots, count) ||
        !look_vector(a[4], device, DL_INT, lens, lens_length) ||
        !look_vector(a[5], device, DL_FLOAT, slopes, slopes_length) || slots == nullptr ||
        lens == nullptr || count != q.rows || lens_length != count || count > (1 << 24) ||
        (slopes != nullptr && slopes_length != q_heads) || !look(a[7], device, work) ||
        work.ndim != 1 || work.type_bits != 16 || !as_number(a[8], scale) ||
        !as_number(a[9], softcap) || softcap < 0.f ||
        exchange->current_work_stream(DL_CUDA, device, &stream) != 0) {
        PyErr_Clear();
        Py_RETURN_FALSE;
    }
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fu_kvcache_attention(cache, q.ptr, q.stride, out.ptr, out.stride, q_heads,
                              static_cast<const int32_t*>(slots),
                              static_cast<const int32_t*>(lens), static_cast<int32_t>(count), scale,
                              softcap, static_cast<const float*>(slopes),
                              static_cast<char*>(work.data) + work.byte_offset, work.shape[0] * 2,
                              status, status_host, 0, stream);
    Py_END_ALLOW_THREADS
    return launched(rc, "fu_kvcache_attention");
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name, const char* doc) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL,
            doc};
}

PyMethodDef methods[] = {
    method<attention>("attention", "fu_attention_forward with plain arguments"),
    method<kvcache_append>("kvcache_append", "fu_kvcache_append with plain arguments"),
    method<kvcache_attention>("kvcache_attention", "fu_kvcache_attention with plain arguments"),
    method<use_exchange>("use_exchange", "take the tensor type's DLPack exchange API"),
    method<try_attention>("try_attention", "fu_attention_forward on tensors, if they fit"),
    method<try_append>("try_append", "fu_kvcache_append on tensors, if they fit"),
    method<try_decode>("try_decode", "fu_kvcache_attention on tensors, if they fit"),
    {"forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(forward)),
     METH_FASTCALL, "fu_qkv_forward with plain integer/float arguments"},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fu_fast", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fu_fast(void) { return PyModule_Create(&module); }
