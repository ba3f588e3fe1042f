// The calls of llama_cpp/device_ops.py on tensors: reads what a call needs of its tensors, checks it and calls the C entry point, for arguments that are all right.
// Anything else returns None, and the Python code, which makes the same checks, says what is wrong or goes its own way. (An extension module, g++ and Python's
// headers, no CUDA: with the checks in Python a call took 15 to 23 us of the host, more than most of them take on the device.)
#include <Python.h>
#include <math.h>
#include <stdint.h>

#include "../../include/b200_gguf.h"

namespace {

PyObject *s_shape, *s_stride, *s_dtype, *s_data_ptr, *s_get_device, *s_is_contiguous, *s_nbytes;

// dtype objects (one of each kind exists) and their type ids, entered by the Python side as it meets them
constexpr int MAX_TYPES = 32;
struct { PyObject* dtype; int code; } types[MAX_TYPES];
int n_types = 0;

struct Tensor {
    void* p;
    int64_t shape[4], stride[4];
    int type, device;
};

bool read_tuple(PyObject* t, int n, int64_t* out) {
    if (!t) return false;
    bool ok = PyTuple_Check(t) && PyTuple_GET_SIZE(t) == n;
    for (int i = 0; ok && i < n; i++) {
        out[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(t, i));
        ok = !(out[i] == -1 && PyErr_Occurred());
    }
    Py_DECREF(t);
    return ok;
}
bool read_int(PyObject* v, long long* out) {
    if (!v) return false;
    *out = PyLong_AsLongLong(v);
    Py_DECREF(v);
    return !(*out == -1 && PyErr_Occurred());
}
bool read_address(PyObject* v, void** out) {
    if (!v) return false;
    *out = PyLong_AsVoidPtr(v);
    Py_DECREF(v);
    return !(*out == nullptr && PyErr_Occurred());
}

// a tensor of n dimensions on the given device (-1: any CUDA device), of the given type (-1: any known one); dense: contiguous, else its last dimension is
bool read(PyObject* t, int n, int device, int type, bool dense, Tensor& o) {
    PyObject* dtype = PyObject_GetAttr(t, s_dtype);
    if (!dtype) return false;
    o.type = -1;
    for (int i = 0; i < n_types; i++) if (types[i].dtype == dtype) { o.type = types[i].code; break; }
    Py_DECREF(dtype);
    if (o.type < 0 || (type >= 0 && o.type != type)) return false;
    long long d;
    if (!read_int(PyObject_CallMethodNoArgs(t, s_get_device), &d) || d < 0 || (device >= 0 && d != device)) return false;
    o.device = (int)d;
    if (!read_tuple(PyObject_GetAttr(t, s_shape), n, o.shape)) return false;
    if (dense) {
        PyObject* c = PyObject_CallMethodNoArgs(t, s_is_contiguous);
        if (!c) return false;
        const bool yes = c == Py_True;
        Py_DECREF(c);
        if (!yes) return false;
    } else {
        if (!read_tuple(PyObject_CallMethodNoArgs(t, s_stride), n, o.stride)) return false;
        if (o.stride[n - 1] != 1 && o.shape[n - 1] > 1) return false;
    }
    return read_address(PyObject_CallMethodNoArgs(t, s_data_ptr), &o.p);
}

bool fits(int64_t v) { return v >= 0 && v <= INT32_MAX; }

// pools, tables and rows of a call. `codes`: pools in 4 bits, whose shape becomes [pages][KV heads][tokens of a page][head_dim]
bool read_where(PyObject* const* a, int64_t n_rows, int device, Tensor& k_pool, Tensor& v_pool, b2_ragged_pages& w, bool codes = false) {
    Tensor pages, start, held;
    if (!read(a[0], 4, device, codes ? B2_TYPE_U8 : -1, true, k_pool) || !read(a[1], 4, device, k_pool.type, true, v_pool) || !read(a[2], 2, device, B2_TYPE_I32, false, pages) ||
        !read(a[3], 1, device, B2_TYPE_I32, true, start) || !read(a[4], 1, device, B2_TYPE_I32, true, held)) return false;
    for (int i = 0; i < 4; i++) if (k_pool.shape[i] != v_pool.shape[i]) return false;
    const int64_t n = held.shape[0];
    if (codes) {
        if (k_pool.shape[3] != 9 * 64 && k_pool.shape[3] != 9 * 128) return false;
        k_pool.shape[2] *= 16; k_pool.shape[3] /= 9;
    }
    if ((!codes && k_pool.type != B2_TYPE_F16 && k_pool.type != B2_TYPE_BF16) || pages.shape[0] != n || start.shape[0] != n + 1 || !fits(n) || !fits(pages.shape[1]) || !fits(n_rows) ||
        !fits(k_pool.shape[1]) || !fits(k_pool.shape[2]) || !fits(k_pool.shape[3])) return false;
    w.row_start = (const int32_t*)start.p; w.lengths = (const int32_t*)held.p; w.pages = (const int32_t*)pages.p;
    w.table_stride = n > 1 ? pages.stride[0] : pages.shape[1];
    w.n_pages = k_pool.shape[0]; w.max_pages = (int32_t)pages.shape[1]; w.n_seqs = (int32_t)n; w.n_rows = (int32_t)n_rows; w.block_tokens = (int32_t)k_pool.shape[2];
    return true;
}

bool read_stream(PyObject* s, void** out) {
    if (s == Py_None) { *out = nullptr; return true; }
    *out = PyLong_AsVoidPtr(s);
    return !PyErr_Occurred();
}

// a contiguous tensor of any type on the device
bool read_workspace(PyObject* t, int device, void*& p, int64_t& bytes) {
    long long d, n;
    if (t == Py_None || !read_int(PyObject_CallMethodNoArgs(t, s_get_device), &d) || d != device || !read_int(PyObject_GetAttr(t, s_nbytes), &n)) return false;
    PyObject* c = PyObject_CallMethodNoArgs(t, s_is_contiguous);
    const bool dense = c == Py_True;
    Py_XDECREF(c);
    bytes = n;
    return dense && read_address(PyObject_CallMethodNoArgs(t, s_data_ptr), &p);
}

PyObject* not_ours() {
    PyErr_Clear();
    Py_RETURN_NONE;
}

bool is_rows(int type) { return type == B2_TYPE_F32 || type == B2_TYPE_F16 || type == B2_TYPE_BF16; }

// (entry point, k, v, k_pool, v_pool, pages, row_start, lengths, freqs, q, q_out, layout, first_pos, amplitude, stream) -> code, or None
PyObject* append(PyObject* const* a, Py_ssize_t n, bool codes) {
    if (n != 15) return not_ours();
    Tensor k, v, k_pool, v_pool, freqs, q, q_out;
    b2_ragged_pages w;
    b2_kv_append_args x = {};
    void *fn = PyLong_AsVoidPtr(a[0]), *stream;
    if (!fn || !read(a[1], 3, -1, -1, false, k) || !is_rows(k.type) || !read(a[2], 3, k.device, k.type, false, v) || !read_where(a + 3, k.shape[0], k.device, k_pool, v_pool, w, codes)) return not_ours();
    for (int i = 0; i < 3; i++) if (k.shape[i] != v.shape[i]) return not_ours();
    if (k.shape[1] != k_pool.shape[1] || k.shape[2] != k_pool.shape[3]) return not_ours();
    if (a[8] != Py_None) {
        if (!read(a[8], 1, k.device, B2_TYPE_F32, true, freqs) || freqs.shape[0] > 4096) return not_ours();
        x.freqs = (const float*)freqs.p; x.rot_dims = (int32_t)(2 * freqs.shape[0]);
    }
    if ((a[9] == Py_None) != (a[10] == Py_None)) return not_ours();
    x.cache_type = codes ? B2_TYPE_F16 : k_pool.type;
    if (a[9] != Py_None) {
        if (!read(a[9], 3, k.device, k.type, false, q) || !read(a[10], 3, k.device, codes ? -1 : k_pool.type, false, q_out)) return not_ours();
        if (codes) {
            if (q_out.type != B2_TYPE_F16 && q_out.type != B2_TYPE_BF16) return not_ours();
            x.cache_type = q_out.type;
        }
        for (int i = 0; i < 3; i++) if (q.shape[i] != q_out.shape[i]) return not_ours();
        if (q.shape[0] != k.shape[0] || q.shape[2] != k.shape[2] || !fits(q.shape[1])) return not_ours();
        x.q = q.p; x.q_row = q.stride[0]; x.q_head = q.stride[1]; x.q_out = q_out.p; x.q_out_row = q_out.stride[0]; x.q_out_head = q_out.stride[1];
        x.n_head = (int32_t)q.shape[1];
    }
    x.k = k.p; x.v = v.p; x.k_row = k.stride[0]; x.k_head = k.stride[1]; x.v_row = v.stride[0]; x.v_head = v.stride[1];
    x.k_pool = k_pool.p; x.v_pool = v_pool.p; x.in_type = k.type; x.n_kv = (int32_t)k.shape[1]; x.head_dim = (int32_t)k.shape[2];
    x.layout = (int32_t)PyLong_AsLong(a[11]); x.first_pos = PyLong_AsLongLong(a[12]); x.amplitude = (float)PyFloat_AsDouble(a[13]);
    if (!read_stream(a[14], &stream) || PyErr_Occurred()) return not_ours();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = ((decltype(&b2_kv_append))fn)(k.device, &w, &x, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

PyObject* kv_append(PyObject*, PyObject* const* a, Py_ssize_t n) { return append(a, n, false); }
PyObject* kv_append_4bit(PyObject*, PyObject* const* a, Py_ssize_t n) { return append(a, n, true); }

// (entry point, k_pool, v_pool, pages, row_start, lengths, k, v, stream) -> code, or None
PyObject* kv_read_4bit(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 9) return not_ours();
    Tensor k, v, k_pool, v_pool;
    b2_ragged_pages w;
    b2_kv_read_4bit_args x = {};
    void *fn = PyLong_AsVoidPtr(a[0]), *stream;
    const bool has_k = a[6] != Py_None, has_v = a[7] != Py_None;
    if (!fn || (!has_k && !has_v) || (has_k && !read(a[6], 3, -1, -1, false, k)) || (has_v && !read(a[7], 3, has_k ? k.device : -1, has_k ? k.type : -1, false, v))) return not_ours();
    const Tensor& t = has_k ? k : v;
    if (!is_rows(t.type) || !read_where(a + 1, t.shape[0], t.device, k_pool, v_pool, w, true)) return not_ours();
    for (int i = 0; has_k && has_v && i < 3; i++) if (k.shape[i] != v.shape[i]) return not_ours();
    if (t.shape[1] != k_pool.shape[1] || t.shape[2] != k_pool.shape[3]) return not_ours();
    x.k_pool = k_pool.p; x.v_pool = v_pool.p; x.n_kv = (int32_t)t.shape[1]; x.head_dim = (int32_t)t.shape[2]; x.out_type = t.type;
    if (has_k) { x.k = k.p; x.k_row = k.stride[0]; x.k_head = k.stride[1]; }
    if (has_v) { x.v = v.p; x.v_row = v.stride[0]; x.v_head = v.stride[1]; }
    if (!read_stream(a[8], &stream) || PyErr_Occurred()) return not_ours();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = ((decltype(&b2_kv_read_4bit))fn)(t.device, &w, &x, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

// (entry point, q, k_pool, v_pool, pages, row_start, lengths, out, workspace, max_rows, scale, stream) -> code, or None
PyObject* attention_4bit(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 12) return not_ours();
    Tensor q, out, k_pool, v_pool;
    b2_ragged_pages w;
    b2_attention_4bit_args x = {};
    void *fn = PyLong_AsVoidPtr(a[0]), *stream;
    if (!fn || !read(a[1], 3, -1, -1, false, q) || !read(a[7], 3, q.device, q.type, false, out) || !read_where(a + 2, q.shape[0], q.device, k_pool, v_pool, w, true)) return not_ours();
    for (int i = 0; i < 3; i++) if (q.shape[i] != out.shape[i]) return not_ours();
    if ((q.type != B2_TYPE_F16 && q.type != B2_TYPE_BF16) || q.shape[2] != k_pool.shape[3] || k_pool.shape[1] == 0 || !fits(q.shape[1]) || q.shape[1] % k_pool.shape[1]) return not_ours();
    const long long max_rows = a[9] == Py_None ? (q.shape[0] > 1 ? q.shape[0] : 1) : PyLong_AsLongLong(a[9]);
    if (PyErr_Occurred() || max_rows > INT32_MAX || max_rows < INT32_MIN || !read_workspace(a[8], q.device, x.workspace, x.workspace_bytes)) return not_ours();
    x.q = q.p; x.k_pool = k_pool.p; x.v_pool = v_pool.p; x.out = out.p; x.q_row = q.stride[0]; x.q_head = q.stride[1]; x.out_row = out.stride[0]; x.out_head = out.stride[1];
    x.max_rows = (int32_t)max_rows; x.n_head = (int32_t)q.shape[1]; x.n_kv = (int32_t)k_pool.shape[1]; x.head_dim = (int32_t)q.shape[2]; x.type = q.type;
    x.scale = (float)(a[10] == Py_None ? 1.0 / sqrt((double)q.shape[2]) : PyFloat_AsDouble(a[10]));
    if (!read_stream(a[11], &stream) || PyErr_Occurred()) return not_ours();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = ((decltype(&b2_attention_4bit))fn)(q.device, &w, &x, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

// (entry point, q, k_pool, v_pool, pages, row_start, lengths, prefix_pages, n_prefix, out, workspace, max_rows, scale, stream) -> code, or None
PyObject* attention_shared_prefix(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 14) return not_ours();
    Tensor q, out, k_pool, v_pool, prefix;
    b2_ragged_pages w;
    b2_shared_prefix_args x = {};
    void *fn = PyLong_AsVoidPtr(a[0]), *stream;
    if (!fn || !read(a[1], 3, -1, -1, false, q) || !read(a[9], 3, q.device, q.type, false, out) || !read_where(a + 2, q.shape[0], q.device, k_pool, v_pool, w)) return not_ours();
    for (int i = 0; i < 3; i++) if (q.shape[i] != out.shape[i]) return not_ours();
    if (q.type != k_pool.type || q.shape[2] != k_pool.shape[3] || k_pool.shape[1] == 0 || !fits(q.shape[1]) || q.shape[1] % k_pool.shape[1]) return not_ours();
    const long long n_prefix = PyLong_AsLongLong(a[8]), max_rows = a[11] == Py_None ? (q.shape[0] > 1 ? q.shape[0] : 1) : PyLong_AsLongLong(a[11]);
    if (PyErr_Occurred() || n_prefix < 0 || n_prefix > INT32_MAX || max_rows > INT32_MAX || max_rows < INT32_MIN) return not_ours();
    if (n_prefix) {
        if (!read(a[7], 1, q.device, B2_TYPE_I32, true, prefix) || n_prefix > prefix.shape[0] * k_pool.shape[2]) return not_ours();
        if (!read_workspace(a[10], q.device, x.workspace, x.workspace_bytes)) return not_ours();
        x.prefix_pages = (const int32_t*)prefix.p;
    }
    x.q = q.p; x.k_pool = k_pool.p; x.v_pool = v_pool.p; x.out = out.p; x.q_row = q.stride[0]; x.q_head = q.stride[1]; x.out_row = out.stride[0]; x.out_head = out.stride[1];
    x.n_prefix = (int32_t)n_prefix; x.max_rows = (int32_t)max_rows; x.n_head = (int32_t)q.shape[1]; x.n_kv = (int32_t)k_pool.shape[1]; x.head_dim = (int32_t)q.shape[2]; x.type = q.type;
    x.scale = (float)(a[12] == Py_None ? 1.0 / sqrt((double)q.shape[2]) : PyFloat_AsDouble(a[12]));
    if (!read_stream(a[13], &stream) || PyErr_Occurred()) return not_ours();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = ((decltype(&b2_attention_shared_prefix))fn)(q.device, &w, &x, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

// (entry point, logits, tokens, logprob, entropy, top_logprob, top_id, stream) -> code, or None
PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 8) return not_ours();
    Tensor x, t;
    void *fn = PyLong_AsVoidPtr(a[0]), *stream, *p[5] = {};
    if (!fn || !read(a[1], 2, -1, -1, false, x) || !is_rows(x.type) || !fits(x.shape[0]) || !fits(x.shape[1])) return not_ours();
    if ((a[2] == Py_None) != (a[3] == Py_None) || (a[5] == Py_None) != (a[6] == Py_None)) return not_ours();
    int64_t top = 0;
    for (int i = 0; i < 5; i++) {
        if (a[2 + i] == Py_None) continue;
        const int dims = i < 3 ? 1 : 2, type = i == 0 || i == 4 ? B2_TYPE_I32 : B2_TYPE_F32;
        if (!read(a[2 + i], dims, x.device, type, true, t) || t.shape[0] != x.shape[0]) return not_ours();
        if (i == 3) top = t.shape[1];
        if (i == 4 && t.shape[1] != top) return not_ours();
        p[i] = t.p;
    }
    if (!fits(top) || !read_stream(a[7], &stream)) return not_ours();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = ((decltype(&b2_token_logprobs))fn)(x.device, x.p, x.type, x.shape[0] > 1 ? x.stride[0] : x.shape[1], (int)x.shape[0], (int)x.shape[1], (const int32_t*)p[0], (float*)p[1], (float*)p[2],
                                            (int)top, (float*)p[3], (int32_t*)p[4], stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

// (dtype, type id)
PyObject* add_type(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n == 2 && n_types < MAX_TYPES) {
        const long code = PyLong_AsLong(a[1]);
        if (code == -1 && PyErr_Occurred()) return nullptr;
        types[n_types].dtype = Py_NewRef(a[0]);
        types[n_types++].code = (int)code;
    }
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"kv_append", (PyCFunction)(void (*)(void))kv_append, METH_FASTCALL, nullptr},
    {"kv_append_4bit", (PyCFunction)(void (*)(void))kv_append_4bit, METH_FASTCALL, nullptr},
    {"kv_read_4bit", (PyCFunction)(void (*)(void))kv_read_4bit, METH_FASTCALL, nullptr},
    {"attention_4bit", (PyCFunction)(void (*)(void))attention_4bit, METH_FASTCALL, nullptr},
    {"attention_shared_prefix", (PyCFunction)(void (*)(void))attention_shared_prefix, METH_FASTCALL, nullptr},
    {"token_logprobs", (PyCFunction)(void (*)(void))token_logprobs, METH_FASTCALL, nullptr},
    {"add_type", (PyCFunction)(void (*)(void))add_type, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "libb200_pylists", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// (the library of py_lists.cpp is this module: loaded once more by name, for calls that take no conversion of arguments)
PyMODINIT_FUNC PyInit_libb200_pylists(void) {
    s_shape = PyUnicode_InternFromString("shape"); s_stride = PyUnicode_InternFromString("stride"); s_dtype = PyUnicode_InternFromString("dtype");
    s_data_ptr = PyUnicode_InternFromString("data_ptr"); s_get_device = PyUnicode_InternFromString("get_device");
    s_is_contiguous = PyUnicode_InternFromString("is_contiguous"); s_nbytes = PyUnicode_InternFromString("nbytes");
    return PyModule_Create(&module);
}
