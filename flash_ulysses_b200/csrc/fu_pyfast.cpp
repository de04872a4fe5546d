// Minimal CPython binding of the per-call entry points: the launch path of
// FlashUlyssesContext.ulysses_qkv_forward passes 14 plain integers/floats per
// call, which ctypes converts in ~3 us and this METH_FASTCALL function in well
// under 1 us; the attention and cache calls pass up to 24.  Everything else
// (buffers, context creation, errors) stays on the ctypes binding of the same
// library.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

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

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name, const char* doc) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL,
            doc};
}

PyMethodDef methods[] = {
    method<attention>("attention", "fu_attention_forward with plain arguments"),
    method<kvcache_append>("kvcache_append", "fu_kvcache_append with plain arguments"),
    method<kvcache_attention>("kvcache_attention", "fu_kvcache_attention with plain arguments"),
    {"forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(forward)),
     METH_FASTCALL, "fu_qkv_forward with plain integer/float arguments"},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fu_fast", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fu_fast(void) { return PyModule_Create(&module); }
