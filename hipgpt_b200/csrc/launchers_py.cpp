// The Python mirror's hot calls (hipgpt_b200/launchers.py, training.py, serving.py) as a CPython extension: tensors are looked at and their addresses taken in C++.  Through
// attribute look-ups and ctypes a call of decode attention cost 3.4 us of the host beside the launch's own 2.6, more than the kernel takes
// (2.6 us at B=8 H=8 D=32 ctx=77): 6.2 -> 3.1 us per call, attention at B=2 H=8 S=64 D=32 5.6 -> 4.8 (the kernel 4.4).
// Every function returns the library's status; launchers.py raises.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "hipgpt_attn.h"

namespace {

// launchers._ptr and _ptr_bf16, for what is not exactly a tensor; _int, for what is not an int
PyObject *g_any_ptr = nullptr, *g_any_bf16 = nullptr, *g_any_int = nullptr;

// A contiguous CUDA tensor of `type` (for float32 also None or an address) -> its address; false with an exception set
bool address_of(PyObject *o, at::ScalarType type, void **out)
{
    if (o == Py_None && type == at::kFloat) { *out = nullptr; return true; }
    if (THPVariable_CheckExact(o)) {
        const at::Tensor &t = THPVariable_Unpack(o);
        if (!(t.is_cuda() && t.scalar_type() == type && t.is_contiguous())) {
            PyErr_Format(PyExc_ValueError, "expected a contiguous CUDA %s tensor", type == at::kFloat ? "float32" : "bfloat16");
            return false;
        }
        *out = t.data_ptr();
        return true;
    }
    PyObject *p = PyObject_CallOneArg(type == at::kFloat ? g_any_ptr : g_any_bf16, o);
    if (!p) return false;
    *out = reinterpret_cast<void *>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLongMask(p)));
    Py_DECREF(p);
    return !PyErr_Occurred();
}

bool ints(PyObject *const *args, int n, int *out)
{
    for (int i = 0; i < n; ++i) {
        if (PyLong_Check(args[i])) {
            out[i] = static_cast<int>(PyLong_AsUnsignedLongMask(args[i]));
            continue;
        }
        PyObject *x = PyObject_CallOneArg(g_any_int, args[i]);
        if (!x) return false;
        out[i] = static_cast<int>(PyLong_AsUnsignedLongMask(x));
        Py_DECREF(x);
    }
    return !PyErr_Occurred();
}

bool count(Py_ssize_t n, Py_ssize_t want)
{
    if (n != want) PyErr_Format(PyExc_TypeError, "%zd arguments expected, %zd given", want, n);
    return n == want;
}

// The call itself, without the interpreter's lock
template <typename F>
PyObject *status_of(F call)
{
    int rc;
    void *stream = c10::cuda::getCurrentCUDAStream().stream();
    Py_BEGIN_ALLOW_THREADS
    rc = call(stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

PyObject *attention(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    void *p[3];
    int i[5];
    if (!count(n, 8)) return nullptr;
    for (int x = 0; x < 3; ++x) if (!address_of(a[x], at::kFloat, &p[x])) return nullptr;
    if (!ints(a + 3, 5, i)) return nullptr;
    return status_of([&](void *st) {
        return hipgpt_mha_forward_planes(static_cast<const float *>(p[0]), static_cast<float *>(p[1]), static_cast<float *>(p[2]), i[0], i[1], i[2], i[3], i[4], st);
    });
    END_HANDLE_TH_ERRORS
}

PyObject *attention_bf16(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    void *p[2];
    int i[6];
    if (!count(n, 8)) return nullptr;
    for (int x = 0; x < 2; ++x) if (!address_of(a[x], at::kBFloat16, &p[x])) return nullptr;
    if (!ints(a + 2, 6, i)) return nullptr;
    const size_t plane = (size_t)i[0] * i[1] * i[2] * 2;         // bytes
    const char *q = static_cast<const char *>(p[0]);
    return status_of([&](void *st) { return hipgpt_mha_forward_bf16_ex(q, q + plane, q + 2 * plane, p[1], i[0], i[1], i[2], i[3], i[4], i[5], st); });
    END_HANDLE_TH_ERRORS
}

// q, key cache, value cache, out, scratch, bytes of scratch where it is not exactly a tensor, B, H, D, ctx, cap
PyObject *decode(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    void *p[5];
    int i[5];
    if (!count(n, 11)) return nullptr;
    for (int x = 0; x < 5; ++x) if (!address_of(a[x], at::kFloat, &p[x])) return nullptr;
    size_t bytes = 0;
    if (a[5] == Py_None) {
        if (THPVariable_CheckExact(a[4])) bytes = THPVariable_Unpack(a[4]).nbytes();
    } else {
        bytes = PyLong_AsSize_t(a[5]);
        if (PyErr_Occurred()) return nullptr;
    }
    if (!ints(a + 6, 5, i)) return nullptr;
    return status_of([&](void *st) {
        return hipgpt_mha_decode(static_cast<const float *>(p[0]), static_cast<const float *>(p[1]), static_cast<const float *>(p[2]), static_cast<float *>(p[3]),
                                 static_cast<float *>(p[4]), bytes, i[0], i[1], i[2], i[3], i[4], st);
    });
    END_HANDLE_TH_ERRORS
}

// ---- training.py ------------------------------------------------------------------------------------------------------

// Like ints, but what an int does not hold is refused (its low bits alone could pass for a size that the tensors have)
bool sizes(PyObject *const *args, int n, int *out)
{
    for (int i = 0; i < n; ++i) {
        PyObject *x = PyLong_Check(args[i]) ? Py_NewRef(args[i]) : PyObject_CallOneArg(g_any_int, args[i]);
        if (!x) return false;
        int over = 0;
        const long v = PyLong_AsLongAndOverflow(x, &over);
        Py_DECREF(x);
        if (v == -1 && PyErr_Occurred()) return false;
        out[i] = static_cast<int>(v);
        if (over || out[i] != v) {
            PyErr_Format(PyExc_ValueError, "%R is beyond one call", args[i]);
            return false;
        }
    }
    return true;
}

// The tensors of one call of training.py: contiguous, on the current device, of at least `count` values; None gives NULL.  Tables and weights of two or more dimensions: of rows of `row` values
// (weights by token given as [E][V], or the other way round, are no others than these to the count).  The first failure stands.
struct Tensors {
    PyObject *const *a;
    bool ok = true;

    void *at(int i, const char *name, at::ScalarType type, int64_t count, int64_t row = -1)
    {
        if (!ok || a[i] == Py_None) return nullptr;
        ok = false;
        if (!THPVariable_Check(a[i])) { PyErr_Format(PyExc_ValueError, "%s: expected a contiguous CUDA %s tensor", name, c10::toString(type)); return nullptr; }
        const at::Tensor &t = THPVariable_Unpack(a[i]);
        if (row >= 0 && t.dim() >= 2 && t.size(-1) != row) PyErr_Format(PyExc_ValueError, "%s has rows of %lld values, %lld are expected", name, (long long)t.size(-1), (long long)row);
        else if (!(t.is_cuda() && t.scalar_type() == type && t.is_contiguous())) PyErr_Format(PyExc_ValueError, "%s: expected a contiguous CUDA %s tensor", name, c10::toString(type));
        else if (t.get_device() != c10::cuda::current_device()) PyErr_Format(PyExc_ValueError, "%s is on cuda:%d, another is the current device", name, (int)t.get_device());
        else if (t.numel() < count) PyErr_Format(PyExc_ValueError, "%s holds %lld values, %lld are needed", name, (long long)t.numel(), (long long)count);
        else { ok = true; return t.data_ptr(); }
        return nullptr;
    }
    // float32 or bfloat16: the storage type that the call goes by
    at::ScalarType kind(int i, const char *name, int *type)
    {
        if (!ok) return at::kFloat;
        ok = false;
        if (!THPVariable_Check(a[i])) { PyErr_Format(PyExc_ValueError, "%s: expected a CUDA tensor", name); return at::kFloat; }
        const at::ScalarType t = THPVariable_Unpack(a[i]).scalar_type();
        ok = t == at::kFloat || t == at::kBFloat16;
        if (!ok) PyErr_Format(PyExc_ValueError, "expected float32 or bfloat16, not %s", c10::toString(t));
        *type = t == at::kFloat ? HIPGPT_TYPE_F32 : HIPGPT_TYPE_BF16;
        return t;
    }
};

// ids, tok, pos, out, scale, B, S, V, E
PyObject *embedding_scaled(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    int i[4], type = 0;
    if (!count(n, 9) || !sizes(a + 5, 4, i)) return nullptr;
    const double scale = PyFloat_AsDouble(a[4]);
    if (PyErr_Occurred()) return nullptr;
    const int64_t B = i[0], S = i[1], V = i[2], E = i[3];
    Tensors t{a};
    const at::ScalarType k = t.kind(3, "out", &type);
    const void *tok = t.at(1, "tok", k, V * E, E), *pos = t.at(2, "pos", k, S * E, E), *ids = t.at(0, "ids", at::kInt, B * S);
    void *out = t.at(3, "out", k, B * S * E);
    if (!t.ok) return nullptr;
    return status_of([&](void *st) { return hipgpt_embedding_scaled(static_cast<const int *>(ids), tok, pos, out, (float)scale, i[0], i[1], i[2], i[3], type, st); });
    END_HANDLE_TH_ERRORS
}

// grad_out, ids, grad_tok, grad_pos, scale, accumulate, B, S, V, E
PyObject *embedding_backward(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    int i[5], type = 0, grad_type = 0;
    if (!count(n, 10) || !sizes(a + 5, 5, i)) return nullptr;
    const double scale = PyFloat_AsDouble(a[4]);
    if (PyErr_Occurred()) return nullptr;
    const int64_t B = i[1], S = i[2], V = i[3], E = i[4];
    Tensors t{a};
    const at::ScalarType k = t.kind(0, "grad_out", &type), gk = t.kind(a[2] == Py_None ? 3 : 2, "grad_tok", &grad_type);
    void *tok = t.at(2, "grad_tok", gk, V * E, E), *pos = t.at(3, "grad_pos", gk, S * E, E);
    const void *g = t.at(0, "grad_out", k, B * S * E), *ids = t.at(1, "ids", at::kInt, B * S);
    if (!t.ok) return nullptr;
    return status_of([&](void *st) { return hipgpt_embedding_backward(g, static_cast<const int *>(ids), tok, pos, (float)scale, i[0], i[1], i[2], i[3], i[4], type, grad_type, st); });
    END_HANDLE_TH_ERRORS
}

// x, residual, out, counter, p, seed, offset
PyObject *dropout_counter(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    int type = 0;
    if (!count(n, 7)) return nullptr;
    const double p = PyFloat_AsDouble(a[4]);
    const unsigned long long seed = PyLong_AsUnsignedLongLongMask(a[5]), offset = PyLong_AsUnsignedLongLongMask(a[6]);
    if (PyErr_Occurred()) return nullptr;
    Tensors t{a};
    const at::ScalarType k = t.kind(2, "out", &type);
    if (!t.ok) return nullptr;
    const int64_t size = THPVariable_Unpack(a[2]).numel();
    const void *x = t.at(0, "x", k, size), *res = t.at(1, "residual", k, size), *counter = t.at(3, "counter", at::kLong, 1);
    void *out = t.at(2, "out", k, size);
    if (!t.ok) return nullptr;
    return status_of([&](void *st) { return hipgpt_dropout_counter(x, res, out, (float)p, seed, offset, static_cast<const unsigned long long *>(counter), size, type, st); });
    END_HANDLE_TH_ERRORS
}

// x, w, targets, loss, lse, N, E, V, layout
PyObject *linear_cross_entropy(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    int i[4], type = 0;
    if (!count(n, 9) || !sizes(a + 5, 4, i)) return nullptr;
    const int64_t N = i[0], E = i[1], V = i[2], row = i[3] == HIPGPT_WEIGHTS_EV ? V : E;
    Tensors t{a};
    const at::ScalarType k = t.kind(0, "x", &type);
    const void *w = t.at(1, "w", k, V * E, row), *x = t.at(0, "x", k, N * E), *targets = t.at(2, "targets", at::kInt, N);
    void *loss = t.at(3, "loss", at::kFloat, N), *lse = t.at(4, "lse", at::kFloat, N);
    if (!t.ok) return nullptr;
    return status_of([&](void *st) {
        return hipgpt_linear_cross_entropy(x, w, static_cast<const int *>(targets), static_cast<float *>(loss), static_cast<float *>(lse), i[0], i[1], i[2], i[3], type, st);
    });
    END_HANDLE_TH_ERRORS
}

// x, w, targets, lse, grad_loss, grad_x, grad_w, accumulate, N, E, V, layout
PyObject *linear_cross_entropy_backward(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    int i[5], type = 0;
    if (!count(n, 12) || !sizes(a + 7, 5, i)) return nullptr;
    const int64_t N = i[1], E = i[2], V = i[3], row = i[4] == HIPGPT_WEIGHTS_EV ? V : E;
    Tensors t{a};
    const at::ScalarType k = t.kind(0, "x", &type);
    const void *w = t.at(1, "w", k, V * E, row), *x = t.at(0, "x", k, N * E), *targets = t.at(2, "targets", at::kInt, N), *lse = t.at(3, "lse", at::kFloat, N), *g = t.at(4, "grad_loss", at::kFloat, N);
    void *gx = t.at(5, "grad_x", k, N * E), *gw = t.at(6, "grad_w", k, V * E, row);
    if (!t.ok) return nullptr;
    return status_of([&](void *st) {
        return hipgpt_linear_cross_entropy_backward(x, w, static_cast<const int *>(targets), static_cast<const float *>(lse), static_cast<const float *>(g), gx, gw, i[0], i[1], i[2], i[3], i[4], type, st);
    });
    END_HANDLE_TH_ERRORS
}

// ---- serving.py -------------------------------------------------------------------------------------------------------

// A tensor of T rows of H * D values, contiguous or its first dimension alone spread: its address, and the values between its rows
void *rows_at(Tensors &t, int i, const char *name, at::ScalarType type, int64_t T, int64_t H, int64_t D, long long *stride)
{
    if (!t.ok) return nullptr;
    t.ok = false;
    const char *kind = c10::toString(type);
    if (!THPVariable_Check(t.a[i])) { PyErr_Format(PyExc_ValueError, "%s: expected a CUDA %s tensor", name, kind); return nullptr; }
    const at::Tensor &x = THPVariable_Unpack(t.a[i]);
    const int64_t width = H * D;
    const bool whole = x.is_contiguous();
    int64_t inner = 1;
    bool rows = x.dim() >= 2 && x.size(0) > 0;
    for (int64_t d = x.dim() - 1; d >= 1; --d) {
        rows = rows && (x.size(d) == 1 || x.stride(d) == inner);
        inner *= x.size(d);
    }
    // rows as one, or with the tokens in more dimensions than one: [...][width], [...][H][D], or heads one behind the other [T * H][D]
    const bool heads = whole && x.dim() >= 2 && x.size(-1) == D && (x.dim() == 2 || x.size(-2) == H);
    if (x.dim() >= 2 && !(inner == width || heads || (whole && x.size(-1) == width))) PyErr_Format(PyExc_ValueError, "%s has rows of %lld values, %lld are expected", name, (long long)inner, (long long)width);
    else if (!(x.is_cuda() && x.scalar_type() == type && (whole || rows))) PyErr_Format(PyExc_ValueError, "%s: expected a CUDA %s tensor, contiguous but for its first dimension", name, kind);
    else if (x.get_device() != c10::cuda::current_device()) PyErr_Format(PyExc_ValueError, "%s is on cuda:%d, another is the current device", name, (int)x.get_device());
    else if (x.numel() < T * width) PyErr_Format(PyExc_ValueError, "%s holds %lld values, %lld are needed", name, (long long)x.numel(), (long long)(T * width));
    else { t.ok = true; *stride = whole ? width : x.stride(0); return x.data_ptr(); }
    return nullptr;
}

// x, positions, words, out, T, H, D, R, interleaved, inverse, magnitude
PyObject *rotary(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    int i[6], type = 0;
    if (!count(n, 11) || !sizes(a + 4, 6, i)) return nullptr;
    const double magnitude = PyFloat_AsDouble(a[10]);
    if (PyErr_Occurred()) return nullptr;
    const int64_t T = i[0], H = i[1], D = i[2], R = i[3];
    Tensors t{a};
    long long sx = 0, so = 0;
    const at::ScalarType k = t.kind(3, "out", &type);
    const void *x = rows_at(t, 0, "x", k, T, H, D, &sx);
    void *out = rows_at(t, 3, "out", k, T, H, D, &so);
    const void *positions = t.at(1, "positions", at::kInt, T), *words = t.at(2, "words", at::kLong, R / 2);
    if (!t.ok) return nullptr;
    return status_of([&](void *st) {
        return hipgpt_rotary(x, sx, static_cast<const int *>(positions), static_cast<const unsigned long long *>(words), out, so, (float)magnitude, i[4], i[5], i[0], i[1], i[2], i[3], type, st);
    });
    END_HANDLE_TH_ERRORS
}

// A cache's address and device, then (at 4) offsets, lengths, pages, T, B
const hipgpt_paged_cache *cache_at(PyObject *const *a)
{
    const auto *c = static_cast<const hipgpt_paged_cache *>(PyLong_AsVoidPtr(a[0]));
    const long device = PyLong_AsLong(a[1]);
    if (PyErr_Occurred()) return nullptr;
    if (device != c10::cuda::current_device()) { PyErr_Format(PyExc_ValueError, "the cache is on cuda:%ld, another is the current device", device); return nullptr; }
    return c;
}
bool batch_at(Tensors &t, int64_t T, int64_t B, hipgpt_paged_batch *out)
{
    if (!t.ok) return false;
    if (!THPVariable_Check(t.a[6]) || THPVariable_Unpack(t.a[6]).dim() != 2) { PyErr_SetString(PyExc_ValueError, "pages: expected a contiguous CUDA int32 tensor of two dimensions"); return t.ok = false; }
    const int64_t most = THPVariable_Unpack(t.a[6]).size(1);
    if (most > 2147483647LL) { PyErr_Format(PyExc_ValueError, "%lld is beyond one call", (long long)most); return t.ok = false; }
    *out = {static_cast<const int *>(t.at(4, "offsets", at::kInt, B + 1)), static_cast<const int *>(t.at(5, "lengths", at::kInt, B)), static_cast<const int *>(t.at(6, "pages", at::kInt, B * most)),
            (int)B, (int)T, (int)most};
    return t.ok;
}
at::ScalarType type_of(const hipgpt_paged_cache *c) { return c->type == HIPGPT_TYPE_F32 ? at::kFloat : at::kBFloat16; }

// cache, device, k, v, offsets, lengths, pages, T, B, write
PyObject *cache_move(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    int i[3];
    if (!count(n, 10) || !sizes(a + 7, 3, i)) return nullptr;
    Tensors t{a};
    const hipgpt_paged_cache *c = reinterpret_cast<const hipgpt_paged_cache *>(PyLong_AsVoidPtr(a[0]));
    if (PyErr_Occurred()) return nullptr;
    long long sk = 0, sv = 0;
    hipgpt_paged_batch batch;
    void *k = rows_at(t, 2, "k", type_of(c), i[0], c->heads, c->head_dim, &sk), *v = rows_at(t, 3, "v", type_of(c), i[0], c->heads, c->head_dim, &sv);
    if (!t.ok || !cache_at(a) || !batch_at(t, i[0], i[1], &batch)) return nullptr;
    return status_of([&](void *st) { return i[2] ? hipgpt_cache_write(c, &batch, k, sk, v, sv, st) : hipgpt_cache_read(c, &batch, k, sk, v, sv, st); });
    END_HANDLE_TH_ERRORS
}

// cache, device, q, out, offsets, lengths, pages, T, B, H, causal, scale
PyObject *paged_attention(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    int i[4];
    if (!count(n, 12) || !sizes(a + 7, 4, i)) return nullptr;
    const double scale = PyFloat_AsDouble(a[11]);
    if (PyErr_Occurred()) return nullptr;
    Tensors t{a};
    const hipgpt_paged_cache *c = reinterpret_cast<const hipgpt_paged_cache *>(PyLong_AsVoidPtr(a[0]));
    if (PyErr_Occurred()) return nullptr;
    long long sq = 0, so = 0;
    hipgpt_paged_batch batch;
    const void *q = rows_at(t, 2, "q", type_of(c), i[0], i[2], c->head_dim, &sq);
    void *out = rows_at(t, 3, "out", type_of(c), i[0], i[2], c->head_dim, &so);
    if (!t.ok || !cache_at(a) || !batch_at(t, i[0], i[1], &batch)) return nullptr;
    return status_of([&](void *st) { return hipgpt_paged_attention(c, &batch, q, sq, out, so, i[2], i[3], (float)scale, st); });
    END_HANDLE_TH_ERRORS
}

PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    if (!count(n, 3)) return nullptr;
    Py_XSETREF(g_any_int, Py_NewRef(a[2]));
    Py_XSETREF(g_any_ptr, Py_NewRef(a[0]));
    Py_XSETREF(g_any_bf16, Py_NewRef(a[1]));
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(attention)), METH_FASTCALL, nullptr},
                         {"attention_bf16", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(attention_bf16)), METH_FASTCALL, nullptr},
                         {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(decode)), METH_FASTCALL, nullptr},
                         {"embedding_scaled", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(embedding_scaled)), METH_FASTCALL, nullptr},
                         {"embedding_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(embedding_backward)), METH_FASTCALL, nullptr},
                         {"dropout_counter", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(dropout_counter)), METH_FASTCALL, nullptr},
                         {"linear_cross_entropy", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(linear_cross_entropy)), METH_FASTCALL, nullptr},
                         {"linear_cross_entropy_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(linear_cross_entropy_backward)), METH_FASTCALL, nullptr},
                         {"rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(rotary)), METH_FASTCALL, nullptr},
                         {"cache_move", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(cache_move)), METH_FASTCALL, nullptr},
                         {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(paged_attention)), METH_FASTCALL, nullptr},
                         {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(bind)), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "hipgpt_launch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_hipgpt_launch() { return PyModule_Create(&module); }
