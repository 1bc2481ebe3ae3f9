// CPython extension `kvhip._step`: one call of a layer -- `attentionWithCacheUpdate`, with or without the rotary
// positions in front, a gated delta layer's convolution or update, or a beam search's selection -- from its tensors to the C entry point in one
// native call.  A short decode step takes the device less
// time than the interpreter took to look the tensors' shapes, types and addresses up and to convert twenty arguments
// (16 layers over 512 keys of one sequence: 149 us a pass, 130 from here).  Handles the ordinary form of the call; for
// everything else (other masks, arrays that are not contiguous, shapes or types that do not go together, numbers that are
// none) it returns None before anything is done, and the Python methods, which check and report, take the call.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <math.h>

#include "kvhip.h"

namespace {

PyObject *g_tensor_type, *g_rope_type;           // torch.Tensor, kvhip.RoPE
PyObject *g_dtypes[3], *g_device, *g_raw_stream, *g_int32;  // float16, bfloat16, float32; the current device and its stream; dtype=int32
PyObject *s_is_contiguous, *s_is_cuda, *s_dtype, *s_shape, *s_data_ptr, *s_new_empty, *s_dims, *s_traditional, *s_base, *s_scale, *s_freqs, *s_get_device,
    *s_stride;

struct Array {
    long long n[4];
    int dtype;  // kvhip_dtype
    void *p;
};

bool take_int(PyObject *o, long long &v) {
    v = PyLong_AsLongLong(o);
    return !(v == -1 && PyErr_Occurred());
}
bool is_true(PyObject *o) {  // steals o
    const bool t = o == Py_True;
    Py_XDECREF(o);
    return t;
}
// the tensor as the library reads it; false (perhaps with an exception set): not of the ordinary form
bool take(PyObject *t, Array &a) {
    if (reinterpret_cast<PyObject *>(Py_TYPE(t)) != g_tensor_type) return false;
    if (!is_true(PyObject_GetAttr(t, s_is_cuda)) || !is_true(PyObject_CallMethodNoArgs(t, s_is_contiguous))) return false;
    PyObject *dt = PyObject_GetAttr(t, s_dtype);
    a.dtype = -1;
    for (int i = 0; i < 3; ++i)
        if (dt == g_dtypes[i]) a.dtype = i;
    Py_XDECREF(dt);
    if (a.dtype < 0) return false;
    PyObject *shape = PyObject_GetAttr(t, s_shape);
    bool ok = shape && PyTuple_Check(shape) && PyTuple_GET_SIZE(shape) == 4;
    for (int i = 0; ok && i < 4; ++i) ok = take_int(PyTuple_GET_ITEM(shape, i), a.n[i]) && a.n[i] > 0 && a.n[i] <= INT32_MAX;
    Py_XDECREF(shape);
    if (!ok) return false;
    PyObject *ptr = PyObject_CallMethodNoArgs(t, s_data_ptr);
    a.p = ptr ? PyLong_AsVoidPtr(ptr) : nullptr;
    Py_XDECREF(ptr);
    return a.p != nullptr;
}
PyObject *none() {  // (an interrupt or an exit is not a form of the call)
    if (PyErr_Occurred()) {
        if (!PyErr_ExceptionMatches(PyExc_Exception)) return nullptr;
        PyErr_Clear();
    }
    Py_RETURN_NONE;
}

// attend(entry, handle, shape, q, k, v, scale, mask, rope, keep)
//   entry    address of kvhip_cache_update_attend, or of kvhip_cache_update_attend_rope if `rope` is not None
//   shape    (B, kv heads, key size, value size, dtype) of what the cache holds
//   mask     address of a kvhip_mask
//   keep     largest rotated queries, in bytes, for which the cache's own buffer is to be used
// Returns the output tensor, None (not handled, nothing done) or the status of a call that failed.
PyObject *attend(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    if (nargs != 10) {
        PyErr_SetString(PyExc_TypeError, "attend takes 10 arguments");
        return nullptr;
    }
    Array q, k, v;
    if (!take(args[3], q) || !take(args[4], k) || !take(args[5], v)) return none();
    const long long B = q.n[0], Hq = q.n[1], L = q.n[2], Dk = q.n[3], Hkv = k.n[1], Dv = v.n[3];
    if (k.n[0] != B || v.n[0] != B || k.n[2] != L || v.n[2] != L || k.n[3] != Dk || v.n[1] != Hkv || q.dtype != k.dtype || v.dtype != k.dtype) return none();
    PyObject *held = args[2];
    if (!PyTuple_Check(held) || PyTuple_GET_SIZE(held) != 5 || PyTuple_GET_ITEM(held, 4) != g_dtypes[k.dtype]) return none();
    const long long want[4] = {B, Hkv, Dk, Dv};
    for (int i = 0; i < 4; ++i) {
        long long n;
        if (!take_int(PyTuple_GET_ITEM(held, i), n) || n != want[i]) return none();
    }
    PyObject *rope = args[8];
    kvhip_rope r{};
    PyObject *freqs = nullptr;
    if (rope != Py_None) {
        long long keep;
        if (reinterpret_cast<PyObject *>(Py_TYPE(rope)) != g_rope_type) return none();
        if (!take_int(args[9], keep) || B * Hq * L * Dk * (k.dtype == KVHIP_F32 ? 4 : 2) > keep) return none();
        PyObject *dims = PyObject_GetAttr(rope, s_dims), *trad = PyObject_GetAttr(rope, s_traditional), *base = PyObject_GetAttr(rope, s_base),
                 *scale = PyObject_GetAttr(rope, s_scale);
        freqs = PyObject_GetAttr(rope, s_freqs);
        if (dims && trad && base && scale && freqs) {
            r.dims = (int32_t)PyLong_AsLong(dims);
            r.traditional = PyObject_IsTrue(trad) == 1;
            r.base = (float)PyFloat_AsDouble(base);
            r.scale = (float)PyFloat_AsDouble(scale);
            if (freqs != Py_None) {
                PyObject *ptr = PyObject_CallMethodNoArgs(freqs, s_data_ptr);
                r.freqs = ptr ? static_cast<const float *>(PyLong_AsVoidPtr(ptr)) : nullptr;
                Py_XDECREF(ptr);
            }
        }
        Py_XDECREF(dims);
        Py_XDECREF(trad);
        Py_XDECREF(base);
        Py_XDECREF(scale);
    }
    const float scale = (float)PyFloat_AsDouble(args[6]);
    auto *cache = static_cast<kvhip_cache *>(PyLong_AsVoidPtr(args[1]));
    const auto *mask = static_cast<const kvhip_mask *>(PyLong_AsVoidPtr(args[7]));
    void *entry = PyLong_AsVoidPtr(args[0]);
    if (PyErr_Occurred() || !cache || !mask || !entry) {
        Py_XDECREF(freqs);
        return none();
    }
    PyObject *size = Py_BuildValue("(LLLL)", B, Hq, L, Dv);
    PyObject *out = size ? PyObject_CallMethodOneArg(args[3], s_new_empty, size) : nullptr;
    Py_XDECREF(size);
    PyObject *device = out ? PyObject_CallNoArgs(g_device) : nullptr;
    PyObject *stream = device ? PyObject_CallOneArg(g_raw_stream, device) : nullptr;
    PyObject *ptr = stream ? PyObject_CallMethodNoArgs(out, s_data_ptr) : nullptr;
    void *dst = ptr ? PyLong_AsVoidPtr(ptr) : nullptr, *st = stream ? PyLong_AsVoidPtr(stream) : nullptr;
    Py_XDECREF(ptr);
    Py_XDECREF(device);
    Py_XDECREF(stream);
    if (PyErr_Occurred()) {
        Py_XDECREF(out);
        Py_XDECREF(freqs);
        return nullptr;
    }
    kvhip_status status;
    Py_BEGIN_ALLOW_THREADS
    if (rope == Py_None)
        status = reinterpret_cast<decltype(&kvhip_cache_update_attend)>(entry)(cache, q.p, k.p, v.p, (int32_t)B, (int32_t)Hq, (int32_t)Hkv, (int32_t)L,
                                                                               (int32_t)Dk, (int32_t)Dv, k.dtype, scale, mask, dst, st);
    else
        status = reinterpret_cast<decltype(&kvhip_cache_update_attend_rope)>(entry)(cache, &r, nullptr, q.p, k.p, v.p, (int32_t)B, (int32_t)Hq, (int32_t)Hkv,
                                                                                    (int32_t)L, (int32_t)Dk, (int32_t)Dv, k.dtype, scale, mask, nullptr, dst, st);
    Py_END_ALLOW_THREADS
    Py_XDECREF(freqs);
    if (status >= KVHIP_OK) return out;
    Py_DECREF(out);
    return PyLong_FromLong(status);
}

// A tensor of `nd` dimensions on device `dev`, whose last two (three dimensions: last) are dense.
struct Part {
    long long n[4], stride_b, stride_l;
    int dtype;
    void *p;
};
bool take_part(PyObject *t, int nd, long long dev, Part &a) {
    if (reinterpret_cast<PyObject *>(Py_TYPE(t)) != g_tensor_type) return false;
    long long n;
    PyObject *o = PyObject_CallMethodNoArgs(t, s_get_device);
    const bool here = o && take_int(o, n) && n == dev;
    Py_XDECREF(o);
    if (!here) return false;
    PyObject *dt = PyObject_GetAttr(t, s_dtype);
    a.dtype = -1;
    for (int i = 0; i < 3; ++i)
        if (dt == g_dtypes[i]) a.dtype = i;
    Py_XDECREF(dt);
    if (a.dtype < 0) return false;
    PyObject *shape = PyObject_GetAttr(t, s_shape), *stride = shape ? PyObject_CallMethodNoArgs(t, s_stride) : nullptr;
    bool ok = stride && PyTuple_Check(shape) && PyTuple_Check(stride) && PyTuple_GET_SIZE(shape) == nd && PyTuple_GET_SIZE(stride) == nd;
    long long st[4] = {0, 0, 0, 0}, dense = 1;
    for (int i = nd - 1; ok && i >= 0; --i) {
        ok = take_int(PyTuple_GET_ITEM(shape, i), a.n[i]) && take_int(PyTuple_GET_ITEM(stride, i), st[i]) && a.n[i] > 0 && a.n[i] <= INT32_MAX;
        if (ok && i > 1) ok = a.n[i] == 1 || st[i] == dense;
        dense *= a.n[i];
    }
    Py_XDECREF(stride);
    Py_XDECREF(shape);
    if (!ok) return false;
    a.stride_b = nd > 1 ? st[0] : 0;
    a.stride_l = nd > 1 ? st[1] : 0;
    if (nd == 1 && a.n[0] > 1 && st[0] != 1) return false;
    PyObject *ptr = PyObject_CallMethodNoArgs(t, s_data_ptr);
    a.p = ptr ? PyLong_AsVoidPtr(ptr) : nullptr;
    Py_XDECREF(ptr);
    return a.p != nullptr;
}

// delta(entry, workspace, q, k, v, a, b, a_log, dt_bias, state, scale, norm_eps)
//   entry, workspace   addresses of kvhip_gated_delta and kvhip_gated_delta_workspace
//   state              the cache's, dense float32, updated in place
// Handles calls without paddings whose gates come from a_log and dt_bias in float32 (scale None: Dk^-0.5); returns as attend does.
PyObject *delta(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    if (nargs != 12) {
        PyErr_SetString(PyExc_TypeError, "delta takes 12 arguments");
        return nullptr;
    }
    PyObject *device = PyObject_CallNoArgs(g_device);
    long long dev = -1;
    const bool known = device && take_int(device, dev);
    PyObject *stream = known ? PyObject_CallOneArg(g_raw_stream, device) : nullptr;
    void *st = stream ? PyLong_AsVoidPtr(stream) : nullptr;
    Py_XDECREF(device);
    Py_XDECREF(stream);
    Part q, k, v, a, b, log, bias, s;
    if (!stream || !take_part(args[2], 4, dev, q) || !take_part(args[3], 4, dev, k) || !take_part(args[4], 4, dev, v) || !take_part(args[5], 3, dev, a) ||
        !take_part(args[6], 3, dev, b) || !take_part(args[7], 1, dev, log) || !take_part(args[8], 1, dev, bias) || !take_part(args[9], 4, dev, s))
        return none();
    const long long B = v.n[0], L = v.n[1], Hv = v.n[2], Dv = v.n[3], Hk = k.n[2], Dk = k.n[3];
    const long long rows[3] = {B, L, Hv};
    for (int i = 0; i < 3; ++i)
        if (a.n[i] != rows[i] || b.n[i] != rows[i]) return none();
    if (q.n[0] != B || q.n[1] != L || q.n[2] != Hk || q.n[3] != Dk || k.n[0] != B || k.n[1] != L || log.n[0] != Hv || bias.n[0] != Hv) return none();
    if (s.n[0] != B || s.n[1] != Hv || s.n[2] != Dv || s.n[3] != Dk || s.stride_l != Dv * Dk || s.stride_b != Hv * Dv * Dk) return none();
    if (q.dtype != v.dtype || k.dtype != v.dtype || a.dtype != b.dtype || log.dtype != KVHIP_F32 || bias.dtype != KVHIP_F32 || s.dtype != KVHIP_F32) return none();
    kvhip_gated_delta_args x{};
    x.q = q.p, x.k = k.p, x.v = v.p, x.a = a.p, x.b = b.p;
    x.q_stride_b = q.stride_b, x.q_stride_l = q.stride_l, x.k_stride_b = k.stride_b, x.k_stride_l = k.stride_l;
    x.v_stride_b = v.stride_b, x.v_stride_l = v.stride_l, x.a_stride_b = a.stride_b, x.a_stride_l = a.stride_l;
    x.b_stride_b = b.stride_b, x.b_stride_l = b.stride_l;
    x.a_log = static_cast<const float *>(log.p), x.dt_bias = static_cast<const float *>(bias.p);
    x.state_in = static_cast<const float *>(s.p), x.state_out = static_cast<float *>(s.p);
    x.B = (int32_t)B, x.L = (int32_t)L, x.Hk = (int32_t)Hk, x.Hv = (int32_t)Hv, x.Dk = (int32_t)Dk, x.Dv = (int32_t)Dv;
    x.dtype = v.dtype, x.gate_dtype = a.dtype;
    x.scale = args[10] == Py_None ? (float)pow((double)Dk, -0.5) : (float)PyFloat_AsDouble(args[10]);
    x.norm_eps = (float)PyFloat_AsDouble(args[11]);
    void *entry = PyLong_AsVoidPtr(args[0]), *workspace = PyLong_AsVoidPtr(args[1]);
    if (PyErr_Occurred() || !entry || !workspace) return none();
    const size_t need = reinterpret_cast<decltype(&kvhip_gated_delta_workspace)>(workspace)(&x);
    auto empty = [&](PyObject *size) {  // (steals size)
        PyObject *t = size ? PyObject_CallMethodOneArg(args[9], s_new_empty, size) : nullptr;
        Py_XDECREF(size);
        return t;
    };
    auto address = [&](PyObject *t) {
        PyObject *ptr = t ? PyObject_CallMethodNoArgs(t, s_data_ptr) : nullptr;
        void *p = ptr ? PyLong_AsVoidPtr(ptr) : nullptr;
        Py_XDECREF(ptr);
        return p;
    };
    PyObject *size = Py_BuildValue("(LLLL)", B, L, Hv, Dv), *out = size ? PyObject_CallMethodOneArg(args[4], s_new_empty, size) : nullptr;
    Py_XDECREF(size);
    PyObject *scratch = need ? empty(Py_BuildValue("(L)", (long long)((need + 3) / 4))) : nullptr;
    x.out = address(out);
    void *at = address(scratch);
    if (PyErr_Occurred()) {
        Py_XDECREF(out);
        Py_XDECREF(scratch);
        return nullptr;
    }
    kvhip_status status;
    Py_BEGIN_ALLOW_THREADS
    status = reinterpret_cast<decltype(&kvhip_gated_delta)>(entry)(&x, at, need, st);
    Py_END_ALLOW_THREADS
    Py_XDECREF(scratch);
    if (status >= KVHIP_OK) return out;
    Py_DECREF(out);
    return PyLong_FromLong(status);
}

// convolve(entry, x, weight, bias or None, window, silu)
//   entry    address of kvhip_short_convolution
//   window   the cache's, dense, updated in place
// Handles calls without paddings; returns as attend does.
PyObject *convolve(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    if (nargs != 6) {
        PyErr_SetString(PyExc_TypeError, "convolve takes 6 arguments");
        return nullptr;
    }
    PyObject *device = PyObject_CallNoArgs(g_device);
    long long dev = -1;
    const bool known = device && take_int(device, dev);
    PyObject *stream = known ? PyObject_CallOneArg(g_raw_stream, device) : nullptr;
    void *st = stream ? PyLong_AsVoidPtr(stream) : nullptr;
    Py_XDECREF(device);
    Py_XDECREF(stream);
    Part x, w, bias{}, s;
    const bool biased = args[3] != Py_None;
    if (!stream || !take_part(args[1], 3, dev, x) || !take_part(args[2], 2, dev, w) || (biased && !take_part(args[3], 1, dev, bias)) ||
        !take_part(args[4], 3, dev, s))
        return none();
    const long long B = x.n[0], L = x.n[1], C = x.n[2], W = w.n[1];
    if (w.n[0] != C || (C > 1 && w.stride_b != W) || (W > 1 && w.stride_l != 1) || (biased && bias.n[0] != C)) return none();
    if (s.n[0] != B || s.n[1] != W - 1 || s.n[2] != C || (B > 1 && s.stride_b != (W - 1) * C) || (W > 2 && s.stride_l != C)) return none();
    if (w.dtype != x.dtype || s.dtype != x.dtype || (biased && bias.dtype != x.dtype)) return none();
    const int silu = PyObject_IsTrue(args[5]);
    void *entry = PyLong_AsVoidPtr(args[0]);
    if (PyErr_Occurred() || !entry) return none();
    PyObject *size = Py_BuildValue("(LLL)", B, L, C), *out = size ? PyObject_CallMethodOneArg(args[1], s_new_empty, size) : nullptr;
    Py_XDECREF(size);
    PyObject *ptr = out ? PyObject_CallMethodNoArgs(out, s_data_ptr) : nullptr;
    void *p = ptr ? PyLong_AsVoidPtr(ptr) : nullptr;
    Py_XDECREF(ptr);
    if (PyErr_Occurred()) {
        Py_XDECREF(out);
        return nullptr;
    }
    kvhip_status status;
    Py_BEGIN_ALLOW_THREADS
    status = reinterpret_cast<decltype(&kvhip_short_convolution)>(entry)(x.p, x.stride_b, x.stride_l, w.p, bias.p, (int32_t)B, (int32_t)L,
                                                                         (int32_t)C, (int32_t)W, x.dtype, silu, nullptr, nullptr, s.p, s.p, p, st);
    Py_END_ALLOW_THREADS
    if (status >= KVHIP_OK) return out;
    Py_DECREF(out);
    return PyLong_FromLong(status);
}

// select(entry, workspace, logits, scores, count, pad_token)
//   entry, workspace   addresses of kvhip_beam_select and kvhip_beam_select_workspace
// Handles dense [B, K, V] logits with dense float32 [B, K] scores and no beam done: (rows, tokens, scores), None or a status.
PyObject *select(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    if (nargs != 6) {
        PyErr_SetString(PyExc_TypeError, "select takes 6 arguments");
        return nullptr;
    }
    PyObject *device = PyObject_CallNoArgs(g_device);
    long long dev = -1, count, pad;
    const bool known = device && take_int(device, dev);
    PyObject *stream = known ? PyObject_CallOneArg(g_raw_stream, device) : nullptr;
    void *st = stream ? PyLong_AsVoidPtr(stream) : nullptr;
    Py_XDECREF(device);
    Py_XDECREF(stream);
    Part x, s;
    if (!g_int32 || !stream || !take_part(args[2], 3, dev, x) || !take_part(args[3], 2, dev, s) || !take_int(args[4], count) || !take_int(args[5], pad)) return none();
    const long long B = x.n[0], K = x.n[1], V = x.n[2];
    if (s.dtype != KVHIP_F32 || s.n[0] != B || s.n[1] != K || (B > 1 && s.stride_b != K) || (K > 1 && s.stride_l != 1)) return none();
    const long long pitch = K > 1 ? x.stride_l : x.stride_b;  // elements from a row to the next
    if ((B > 1 && x.stride_b != K * pitch) || count <= 0 || count > INT32_MAX || pad < INT32_MIN || pad > INT32_MAX) return none();
    void *entry = PyLong_AsVoidPtr(args[0]), *workspace = PyLong_AsVoidPtr(args[1]);
    if (PyErr_Occurred() || !entry || !workspace) return none();
    const size_t need = reinterpret_cast<decltype(&kvhip_beam_select_workspace)>(workspace)((int32_t)B, (int32_t)K, (int32_t)V, x.dtype, (int32_t)count);
    if (!need) return none();  // (refused: the general path says why)
    PyObject *t[4] = {nullptr, nullptr, nullptr, nullptr};  // rows, tokens, scores, scratch
    void *at[4] = {nullptr, nullptr, nullptr, nullptr};
    bool ok = true;
    for (int i = 0; ok && i < 4; ++i) {
        PyObject *size = i < 3 ? Py_BuildValue("((LL))", B, count) : Py_BuildValue("((L))", (long long)((need + 3) / 4));
        PyObject *method = size ? PyObject_GetAttr(args[3], s_new_empty) : nullptr;
        t[i] = method ? PyObject_Call(method, size, i < 2 ? g_int32 : nullptr) : nullptr;
        Py_XDECREF(method);
        Py_XDECREF(size);
        PyObject *ptr = t[i] ? PyObject_CallMethodNoArgs(t[i], s_data_ptr) : nullptr;
        at[i] = ptr ? PyLong_AsVoidPtr(ptr) : nullptr;
        Py_XDECREF(ptr);
        ok = at[i] != nullptr && !PyErr_Occurred();
    }
    kvhip_status status = KVHIP_OK;
    if (ok) {
        Py_BEGIN_ALLOW_THREADS
        status = reinterpret_cast<decltype(&kvhip_beam_select)>(entry)(x.p, pitch, (int32_t)B, (int32_t)K, (int32_t)V, x.dtype,
                                                                       static_cast<const float *>(s.p), nullptr, (int32_t)count, (int32_t)pad,
                                                                       static_cast<int32_t *>(at[0]), static_cast<int32_t *>(at[1]),
                                                                       static_cast<float *>(at[2]), at[3], need, st);
        Py_END_ALLOW_THREADS
    }
    PyObject *r = !ok ? nullptr : status >= KVHIP_OK ? PyTuple_Pack(3, t[0], t[1], t[2]) : PyLong_FromLong(status);
    for (PyObject *o : t) Py_XDECREF(o);
    return r;
}

// bind(Tensor, RoPE, (float16, bfloat16, float32), current device, its raw stream[, {"dtype": int32}: without it `select` takes no call])
PyObject *bind(PyObject *, PyObject *args) {
    PyObject *types;
    g_int32 = nullptr;
    if (!PyArg_ParseTuple(args, "OOO!OO|O!", &g_tensor_type, &g_rope_type, &PyTuple_Type, &types, &g_device, &g_raw_stream, &PyDict_Type, &g_int32)) return nullptr;
    if (PyTuple_GET_SIZE(types) != 3) {
        PyErr_SetString(PyExc_TypeError, "three dtypes");
        return nullptr;
    }
    Py_INCREF(g_tensor_type);
    Py_INCREF(g_rope_type);
    Py_INCREF(g_device);
    Py_INCREF(g_raw_stream);
    Py_XINCREF(g_int32);
    for (int i = 0; i < 3; ++i) {
        g_dtypes[i] = PyTuple_GET_ITEM(types, i);
        Py_INCREF(g_dtypes[i]);
    }
    Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {{"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(attend)), METH_FASTCALL, nullptr},
                           {"delta", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(delta)), METH_FASTCALL, nullptr},
                           {"convolve", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(convolve)), METH_FASTCALL, nullptr},
                           {"select", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(select)), METH_FASTCALL, nullptr},
                           {"bind", bind, METH_VARARGS, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_step", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__step() {
    const struct {
        PyObject **to;
        const char *name;
    } names[] = {{&s_is_contiguous, "is_contiguous"}, {&s_is_cuda, "is_cuda"}, {&s_dtype, "dtype"}, {&s_shape, "shape"}, {&s_data_ptr, "data_ptr"},
                 {&s_new_empty, "new_empty"}, {&s_dims, "dims"}, {&s_traditional, "traditional"}, {&s_base, "base"}, {&s_scale, "scale"}, {&s_freqs, "freqs"},
                 {&s_get_device, "get_device"}, {&s_stride, "stride"}};
    for (const auto &n : names)
        if (!(*n.to = PyUnicode_InternFromString(n.name))) return nullptr;
    return PyModule_Create(&g_module);
}
