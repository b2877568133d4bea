// Python module _torch_calls: the calls of capi.py that take torch tensors, with everything between the
// Python call and the C ABI in native code: the checks of the tensors, their addresses and sizes, the
// current stream and the device switch.  capi.py keeps the public functions (names, defaults,
// allocation of outputs that are not given) and hands the rest to this module.
//
// What bounds a small call is this host path: a 4096 x 4096 linear takes 4 us on the device, and with
// the same steps as Python statements around a ctypes call one call took 9.9 us (now 4.1).
//
// The library is not linked but bound: capi.py passes the addresses of the functions it has loaded,
// so the range-checked debug build is reached the same way as the normal one.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>

#include "../../../include/jq_b200.h"
#include "../../../include/jq_kv_cache.h"

namespace {

// ---- functions of the library, bound by capi.py -----------------------------------------------------
decltype(&jq_quantize_q8_1_device) f_quantize = nullptr;
decltype(&jq_mul_mat_q4_0_q8_1_device_ex) f_mul_mat = nullptr;
decltype(&jq_linear_q4_0_device) f_linear = nullptr;
decltype(&jq_linear_q4_0_multi_device) f_multi = nullptr;
decltype(&jq_rms_norm_q8_1_device) f_rms_norm = nullptr;
decltype(&jq_swiglu_q8_1_device) f_swiglu = nullptr;
decltype(&jq_rope_device) f_rope = nullptr;
decltype(&jq_rope_kv_append_device) f_rope_append = nullptr;
decltype(&jq_paged_attention_ws_bytes) f_attention_ws_bytes = nullptr;
decltype(&jq_paged_attention_q8_1_device) f_attention = nullptr;
decltype(&jq_kv_evict_device) f_evict = nullptr;

struct Binding {
    const char *name;
    void **slot;
};
const Binding bindings[] = {
    {"jq_quantize_q8_1_device", reinterpret_cast<void **>(&f_quantize)},
    {"jq_mul_mat_q4_0_q8_1_device_ex", reinterpret_cast<void **>(&f_mul_mat)},
    {"jq_linear_q4_0_device", reinterpret_cast<void **>(&f_linear)},
    {"jq_linear_q4_0_multi_device", reinterpret_cast<void **>(&f_multi)},
    {"jq_rms_norm_q8_1_device", reinterpret_cast<void **>(&f_rms_norm)},
    {"jq_swiglu_q8_1_device", reinterpret_cast<void **>(&f_swiglu)},
    {"jq_rope_device", reinterpret_cast<void **>(&f_rope)},
    {"jq_rope_kv_append_device", reinterpret_cast<void **>(&f_rope_append)},
    {"jq_paged_attention_ws_bytes", reinterpret_cast<void **>(&f_attention_ws_bytes)},
    {"jq_paged_attention_q8_1_device", reinterpret_cast<void **>(&f_attention)},
    {"jq_kv_evict_device", reinterpret_cast<void **>(&f_evict)},
};

PyObject *bind(PyObject *, PyObject *addresses) {
    for (const Binding &b : bindings) {
        PyObject *v = PyDict_GetItemString(addresses, b.name);
        if (v == nullptr && *b.slot != nullptr) continue;  // stays as it was bound before
        if (v == nullptr) {
            PyErr_Format(PyExc_KeyError, "no address given for %s", b.name);
            return nullptr;
        }
        *b.slot = PyLong_AsVoidPtr(v);
        if (PyErr_Occurred()) return nullptr;
    }
    Py_RETURN_NONE;
}

// a reference that is given back on every way out, an exception's included
struct Owned {
    PyObject *p = nullptr;
    ~Owned() { Py_XDECREF(p); }
};

// ---- arguments -------------------------------------------------------------------------------------
const char *dtype_text(at::ScalarType t) {
    return t == at::kFloat ? "torch.float32" : t == at::kInt ? "torch.int32" : t == at::kLong ? "torch.int64" : "torch.uint8";
}

// The tensor behind `o` when it is a contiguous CUDA tensor of this type, else nullptr with ValueError set.
const at::Tensor *tensor_arg(PyObject *o, at::ScalarType type, const char *name) {
    if (THPVariable_Check(o)) {
        const at::Tensor &t = THPVariable_Unpack(o);
        if (t.is_cuda() && t.scalar_type() == type && t.is_contiguous()) return &t;
    }
    PyErr_Format(PyExc_ValueError, "%s must be a contiguous CUDA tensor of dtype %s", name, dtype_text(type));
    return nullptr;
}
bool pointer_arg(PyObject *o, at::ScalarType type, const char *name, void **out) {
    const at::Tensor *t = tensor_arg(o, type, name);
    if (t == nullptr) return false;
    *out = t->data_ptr();
    return true;
}
bool optional_pointer_arg(PyObject *o, at::ScalarType type, const char *name, void **out) {
    *out = nullptr;
    return o == Py_None || pointer_arg(o, type, name, out);
}
// any tensor (its bytes are what counts) or None
bool optional_bytes_arg(PyObject *o, const char *name, void **out) {
    *out = nullptr;
    if (o == Py_None) return true;
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_ValueError, "%s must be a tensor", name);
        return false;
    }
    *out = THPVariable_Unpack(o).data_ptr();
    return true;
}
bool size_arg(PyObject *o, int64_t *out) {
    *out = PyLong_AsLongLong(o);
    return !(*out == -1 && PyErr_Occurred());
}
bool two_sizes(const at::Tensor &t, const char *name, int64_t *rows, int64_t *cols) {
    if (t.dim() != 2) {
        PyErr_Format(PyExc_ValueError, "%s must have two dimensions (has %d)", name, (int)t.dim());
        return false;
    }
    *rows = t.size(0);
    *cols = t.size(1);
    return true;
}
bool argument_count(Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", want, n);
    return false;
}

// The device of the call made current for its duration, and the stream that torch would use on it.
class OnDevice {
  public:
    explicit OnDevice(const at::Tensor &t) : want_(t.get_device()) {
        had_ = c10::cuda::current_device();
        if (had_ != want_) c10::cuda::set_device(want_);
    }
    ~OnDevice() {
        if (had_ != want_) (void)c10::cuda::SetDevice(had_);  // no exception from here: restore() has reported the error
    }
    void restore() {
        const c10::DeviceIndex back = had_;
        had_ = want_;
        if (back != want_) c10::cuda::set_device(back);
    }
    void *stream() const { return c10::cuda::getCurrentCUDAStream(want_).stream(); }

  private:
    c10::DeviceIndex want_, had_;
};

// Other Python threads run while this is in scope: no Python object and no tensor is touched meanwhile.
class WithoutGil {
  public:
    WithoutGil() : state_(PyEval_SaveThread()) {}
    ~WithoutGil() { PyEval_RestoreThread(state_); }

  private:
    PyThreadState *state_;
};

// Runs `call` (which returns a jq_status) and hands the status to Python.  A launch can wait: for room in the queue, for a
// kernel's module to be loaded on its first use.  So `call` has only plain values left to pass on, and runs without the GIL.
template <typename F>
PyObject *status_of(const at::Tensor &on, F &&call) {
    OnDevice device(on);
    void *const stream = device.stream();
    int status;
    {
        const WithoutGil released;
        status = call(stream);
    }
    device.restore();
    return PyLong_FromLong(status);
}

// What Python calls.  Almost everything of torch can throw, is_contiguous() and data_ptr() of a tensor without storage
// (under vmap, for instance) included, and no exception may leave a C function: each becomes the Python exception that
// torch's own functions raise for it.
template <PyObject *(*Call)(PyObject *const *, Py_ssize_t)>
PyObject *entry(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    return Call(a, n);
    END_HANDLE_TH_ERRORS
}

// ---- the calls: every one returns the library's status -------------------------------------------------
// (x, out, order, s_mode)
PyObject *quantize(PyObject *const *a, Py_ssize_t n) {
    int64_t M, K, order, s_mode;
    void *xp, *op;
    if (!argument_count(n, 4)) return nullptr;
    const at::Tensor *x = tensor_arg(a[0], at::kFloat, "x");
    if (x == nullptr || !two_sizes(*x, "x", &M, &K) || !pointer_arg(a[1], at::kByte, "out", &op) || !size_arg(a[2], &order) ||
        !size_arg(a[3], &s_mode))
        return nullptr;
    xp = x->data_ptr();
    return status_of(*x, [&](void *st) { return f_quantize(st, static_cast<const float *>(xp), op, K, M, (int)order, (int)s_mode); });
}

// (w, xq, out, K, N, M, order, kernel)
PyObject *mul_mat(PyObject *const *a, Py_ssize_t n) {
    int64_t K, N, M, order, kernel;
    void *xp, *yp;
    if (!argument_count(n, 8)) return nullptr;
    const at::Tensor *w = tensor_arg(a[0], at::kByte, "w");
    if (w == nullptr || !pointer_arg(a[1], at::kByte, "xq", &xp) || !pointer_arg(a[2], at::kFloat, "out", &yp) || !size_arg(a[3], &K) ||
        !size_arg(a[4], &N) || !size_arg(a[5], &M) || !size_arg(a[6], &order) || !size_arg(a[7], &kernel))
        return nullptr;
    const void *wp = w->data_ptr();
    return status_of(*w, [&](void *st) {
        return f_mul_mat(st, wp, xp, static_cast<float *>(yp), K, N, M, (int)order, (int)kernel);
    });
}

// (w, x, ws, out, N, s_mode)
PyObject *linear(PyObject *const *a, Py_ssize_t n) {
    int64_t K, N, M, s_mode;
    void *wp, *wsp, *yp;
    if (!argument_count(n, 6)) return nullptr;
    if (!pointer_arg(a[0], at::kByte, "w", &wp)) return nullptr;
    const at::Tensor *x = tensor_arg(a[1], at::kFloat, "x");
    if (x == nullptr || !two_sizes(*x, "x", &M, &K) || !pointer_arg(a[2], at::kByte, "ws", &wsp) ||
        !pointer_arg(a[3], at::kFloat, "out", &yp) || !size_arg(a[4], &N) || !size_arg(a[5], &s_mode))
        return nullptr;
    const void *xp = x->data_ptr();
    return status_of(*x, [&](void *st) {
        return f_linear(st, wp, static_cast<const float *>(xp), wsp, static_cast<float *>(yp), K, N, M, (int)s_mode);
    });
}

// (ws_list, N_list, outs, x or None, xq or None, ws or None, K, M, s_mode); the first three are sequences of one length
PyObject *multi(PyObject *const *a, Py_ssize_t n) {
    constexpr Py_ssize_t MOST = 16;  // the library says how many it takes; this only bounds the arrays here
    const void *w[MOST];
    float *y[MOST];
    int64_t rows[MOST];
    int64_t K, M, s_mode;
    void *xp, *xqp, *wsp;
    if (!argument_count(n, 9)) return nullptr;
    Owned seq[3];  // tuples of the call's own: converting a row count may run Python code that changes the caller's lists
    for (int i = 0; i < 3; ++i) {
        seq[i].p = PySequence_Tuple(a[i]);
        if (seq[i].p == nullptr) return nullptr;
    }
    const Py_ssize_t n_mats = PyTuple_GET_SIZE(seq[0].p);
    if (n_mats < 1 || n_mats > MOST || PyTuple_GET_SIZE(seq[1].p) != n_mats || PyTuple_GET_SIZE(seq[2].p) != n_mats) {
        PyErr_SetString(PyExc_ValueError, "weights, row counts and outputs must be sequences of one length (1 to 16)");
        return nullptr;
    }
    const at::Tensor *first = nullptr;
    for (Py_ssize_t i = 0; i < n_mats; ++i) {
        void *yp = nullptr;
        const at::Tensor *t = tensor_arg(PyTuple_GET_ITEM(seq[0].p, i), at::kByte, "w");
        if (t == nullptr || !pointer_arg(PyTuple_GET_ITEM(seq[2].p, i), at::kFloat, "out", &yp)) return nullptr;
        Owned r{PyNumber_Long(PyTuple_GET_ITEM(seq[1].p, i))};
        if (r.p == nullptr || !size_arg(r.p, &rows[i])) return nullptr;
        if (i == 0) first = t;
        w[i] = t->data_ptr();
        y[i] = static_cast<float *>(yp);
    }
    if (!optional_pointer_arg(a[3], at::kFloat, "x", &xp) || !optional_pointer_arg(a[4], at::kByte, "xq", &xqp) ||
        !optional_pointer_arg(a[5], at::kByte, "ws", &wsp) || !size_arg(a[6], &K) || !size_arg(a[7], &M) || !size_arg(a[8], &s_mode))
        return nullptr;
    return status_of(*first, [&](void *st) {
        return f_multi(st, (int)n_mats, w, rows, y, static_cast<const float *>(xp), xqp, wsp, K, M, (int)s_mode);
    });
}

// (x, weight, epsilon, residual or None, normed or None, xq or None, order, s_mode)
PyObject *rms_norm(PyObject *const *a, Py_ssize_t n) {
    int64_t T, H, order, s_mode;
    void *wp, *rp, *np, *qp;
    if (!argument_count(n, 8)) return nullptr;
    const at::Tensor *x = tensor_arg(a[0], at::kFloat, "x");
    if (x == nullptr || !two_sizes(*x, "x", &T, &H) || !pointer_arg(a[1], at::kFloat, "weight", &wp)) return nullptr;
    const double epsilon = PyFloat_AsDouble(a[2]);
    if (epsilon == -1.0 && PyErr_Occurred()) return nullptr;
    if (!optional_pointer_arg(a[3], at::kFloat, "residual", &rp) || !optional_pointer_arg(a[4], at::kFloat, "normed", &np) ||
        !optional_bytes_arg(a[5], "xq", &qp) || !size_arg(a[6], &order) || !size_arg(a[7], &s_mode))
        return nullptr;
    void *xp = x->data_ptr();
    return status_of(*x, [&](void *st) {
        return f_rms_norm(st, static_cast<float *>(xp), static_cast<float *>(rp), static_cast<const float *>(wp),
                          static_cast<float *>(np), qp, H, T, (float)epsilon, (int)order, (int)s_mode);
    });
}

// (gate, up, mid or None, xq or None, order, s_mode)
PyObject *swiglu(PyObject *const *a, Py_ssize_t n) {
    int64_t T, I, order, s_mode;
    void *up, *mp, *qp;
    if (!argument_count(n, 6)) return nullptr;
    const at::Tensor *g = tensor_arg(a[0], at::kFloat, "gate");
    if (g == nullptr || !two_sizes(*g, "gate", &T, &I) || !pointer_arg(a[1], at::kFloat, "up", &up) ||
        !optional_pointer_arg(a[2], at::kFloat, "mid", &mp) || !optional_bytes_arg(a[3], "xq", &qp) || !size_arg(a[4], &order) ||
        !size_arg(a[5], &s_mode))
        return nullptr;
    const void *gp = g->data_ptr();
    return status_of(*g, [&](void *st) {
        return f_swiglu(st, static_cast<const float *>(gp), static_cast<const float *>(up), static_cast<float *>(mp), qp, I, T,
                        (int)order, (int)s_mode);
    });
}

// ---- the paged cache and what reads and writes it: strided tensors, all on one device, sizes checked against one another --------------
// The tensor behind `o` when it is a CUDA tensor of this type with `dims` dimensions whose last one is contiguous, on the device of `like`
// (when given), else nullptr with ValueError set.
const at::Tensor *strided_arg(PyObject *o, at::ScalarType type, int64_t dims, const char *name, const at::Tensor *like) {
    if (THPVariable_Check(o)) {
        const at::Tensor &t = THPVariable_Unpack(o);
        if (t.is_cuda() && t.scalar_type() == type && t.dim() == dims && (t.size(dims - 1) <= 1 || t.stride(dims - 1) == 1)) {
            if (like == nullptr || t.get_device() == like->get_device()) return &t;
            PyErr_Format(PyExc_ValueError, "%s is on another device than the other tensors", name);
            return nullptr;
        }
    }
    PyErr_Format(PyExc_ValueError, "%s must be a CUDA tensor of dtype %s with %d dimensions, the last one contiguous", name, dtype_text(type), (int)dims);
    return nullptr;
}
bool size_is(int64_t got, int64_t want, const char *name, const char *what) {
    if (got == want) return true;
    PyErr_Format(PyExc_ValueError, "%s has %lld %s where %lld are expected", name, (long long)got, what, (long long)want);
    return false;
}
// A contiguous vector of `n` int32 on the device of `like`; None where that is allowed.
bool vector_arg(PyObject *o, int64_t n, const char *name, const at::Tensor &like, bool optional, const int32_t **out) {
    *out = nullptr;
    if (optional && o == Py_None) return true;
    const at::Tensor *t = strided_arg(o, at::kInt, 1, name, &like);
    if (t == nullptr || !size_is(t->size(0), n, name, "elements")) return false;
    *out = static_cast<const int32_t *>(t->data_ptr());
    return true;
}
bool double_arg(PyObject *o, double *out) {
    *out = PyFloat_AsDouble(o);
    return !(*out == -1.0 && PyErr_Occurred());
}
bool truth_arg(PyObject *o, int *out) {
    *out = PyObject_IsTrue(o);
    return *out >= 0;
}

// (k, v, page_table): k and v [pages, slot, head, element] of one type with the same sizes and strides.
bool cache_arg(PyObject *ko, PyObject *vo, PyObject *to, const at::Tensor *like, jq_kv_cache *c, const at::Tensor **k_out) {
    if (!THPVariable_Check(ko)) {
        PyErr_SetString(PyExc_ValueError, "k_cache must be a tensor");
        return false;
    }
    const at::ScalarType type = THPVariable_Unpack(ko).scalar_type();
    if (type == at::kHalf)
        c->type = JQ_KV_F16;
    else if (type == at::kBFloat16)
        c->type = JQ_KV_BF16;
    else if (type == at::kFloat8_e4m3fn)
        c->type = JQ_KV_E4M3;
    else {
        PyErr_SetString(PyExc_ValueError, "k_cache must have dtype torch.float16, torch.bfloat16 or torch.float8_e4m3fn");
        return false;
    }
    const at::Tensor *k = nullptr, *v = nullptr;
    for (PyObject *o : {ko, vo}) {
        const char *name = o == ko && k == nullptr ? "k_cache" : "v_cache";
        const at::Tensor *t = nullptr;
        if (THPVariable_Check(o)) t = &THPVariable_Unpack(o);
        if (t == nullptr || !t->is_cuda() || t->scalar_type() != type || t->dim() != 4 || t->stride(3) != 1) {
            PyErr_Format(PyExc_ValueError, "%s must be a CUDA tensor [pages, slots, heads, elements] of the cache's dtype, the last dimension contiguous", name);
            return false;
        }
        (k == nullptr ? k : v) = t;
    }
    const at::Tensor *table = strided_arg(to, at::kInt, 2, "page_table", k);
    if (table == nullptr) return false;
    if (v->get_device() != k->get_device() || (like != nullptr && like->get_device() != k->get_device())) {
        PyErr_SetString(PyExc_ValueError, "the cache is on another device than the other tensors");
        return false;
    }
    for (int i = 0; i < 4; ++i) {
        if (k->size(i) != v->size(i) || k->stride(i) != v->stride(i)) {
            PyErr_SetString(PyExc_ValueError, "k_cache and v_cache must have the same sizes and strides");
            return false;
        }
    }
    c->d_k = k->data_ptr();
    c->d_v = v->data_ptr();
    c->num_pages = k->size(0), c->page_size = k->size(1), c->num_kv_heads = k->size(2), c->head_dim = k->size(3);
    c->stride_page = k->stride(0), c->stride_slot = k->stride(1), c->stride_head = k->stride(2);
    c->k_scale = c->v_scale = 1.f;
    c->d_page_table = static_cast<const int32_t *>(table->data_ptr());
    c->num_seqs = table->size(0), c->max_pages = table->size(1);
    c->table_stride = table->size(0) > 1 ? table->stride(0) : table->size(1);
    *k_out = k;
    return true;
}

// (x, out, positions, table, interleaved, mscale)
PyObject *rope(PyObject *const *a, Py_ssize_t n) {
    const int32_t *positions;
    int interleaved;
    double mscale;
    if (!argument_count(n, 6)) return nullptr;
    const at::Tensor *x = strided_arg(a[0], at::kFloat, 3, "x", nullptr);
    if (x == nullptr) return nullptr;
    const at::Tensor *out = strided_arg(a[1], at::kFloat, 3, "out", x), *table = strided_arg(a[3], at::kLong, 1, "table", x);
    if (out == nullptr || table == nullptr || !vector_arg(a[2], x->size(0), "positions", *x, false, &positions) || !truth_arg(a[4], &interleaved) ||
        !double_arg(a[5], &mscale))
        return nullptr;
    for (int i = 0; i < 3; ++i) {
        if (!size_is(out->size(i), x->size(i), "out", "elements in a dimension")) return nullptr;
    }
    const float *xp = static_cast<const float *>(x->data_ptr());
    float *yp = static_cast<float *>(out->data_ptr());
    const uint64_t *tp = static_cast<const uint64_t *>(table->data_ptr());
    const int64_t T = x->size(0), H = x->size(1), D = x->size(2), R = 2 * table->size(0);
    const int64_t s[4] = {x->stride(0), x->stride(1), out->stride(0), out->stride(1)};
    return status_of(*x, [&](void *st) { return f_rope(st, xp, yp, positions, tp, T, H, D, R, s[0], s[1], s[2], s[3], interleaved, (float)mscale); });
}

// (qkv, q_out, positions, table, k, v, page_table, index, seqs or None, k_scale, v_scale, interleaved, mscale)
PyObject *rope_append(PyObject *const *a, Py_ssize_t n) {
    const int32_t *positions, *index, *seqs;
    int interleaved;
    double mscale, k_scale, v_scale;
    jq_kv_cache c = {};
    const at::Tensor *k = nullptr;
    if (!argument_count(n, 13)) return nullptr;
    const at::Tensor *x = strided_arg(a[0], at::kFloat, 2, "qkv", nullptr);
    if (x == nullptr) return nullptr;
    const int64_t T = x->size(0);
    const at::Tensor *q = strided_arg(a[1], at::kFloat, 3, "q_out", x), *table = strided_arg(a[3], at::kLong, 1, "table", x);
    if (q == nullptr || table == nullptr || !cache_arg(a[4], a[5], a[6], x, &c, &k) || !vector_arg(a[2], T, "positions", *x, false, &positions) ||
        !vector_arg(a[7], T, "index", *x, false, &index) || !vector_arg(a[8], T, "seqs", *x, true, &seqs) || !double_arg(a[9], &k_scale) ||
        !double_arg(a[10], &v_scale) || !truth_arg(a[11], &interleaved) || !double_arg(a[12], &mscale))
        return nullptr;
    const int64_t H = q->size(1);
    if (!size_is(q->size(0), T, "q_out", "rows") || !size_is(q->size(2), c.head_dim, "q_out", "elements in a head") ||
        !size_is(x->size(1), (H + 2 * c.num_kv_heads) * c.head_dim, "qkv", "columns"))
        return nullptr;
    c.k_scale = (float)k_scale, c.v_scale = (float)v_scale;
    const float *xp = static_cast<const float *>(x->data_ptr());
    float *qp = static_cast<float *>(q->data_ptr());
    const uint64_t *tp = static_cast<const uint64_t *>(table->data_ptr());
    const int64_t R = 2 * table->size(0), s[3] = {x->stride(0), q->stride(0), q->stride(1)};
    return status_of(*x, [&](void *st) {
        return f_rope_append(st, xp, s[0], qp, s[1], s[2], positions, index, seqs, tp, R, T, H, &c, interleaved, (float)mscale);
    });
}

// (q, k, page_table, weights) -> bytes; 0 after an error
PyObject *attention_ws_bytes(PyObject *const *a, Py_ssize_t n) {
    int weights;
    jq_kv_cache c = {};
    const at::Tensor *k = nullptr;
    if (!argument_count(n, 4)) return nullptr;
    const at::Tensor *q = strided_arg(a[0], at::kFloat, 3, "q", nullptr);
    if (q == nullptr || !cache_arg(a[1], a[1], a[2], q, &c, &k) || !truth_arg(a[3], &weights)) return nullptr;
    OnDevice device(*q);
    const size_t bytes = f_attention_ws_bytes(q->size(0), q->size(1), &c, weights);
    device.restore();
    return PyLong_FromSize_t(bytes);
}

// (q, k, v, page_table, lens, seqs or None, scale, window, k_scale, v_scale, out or None, xq or None, order, s_mode, weights or None, ws)
PyObject *attention(PyObject *const *a, Py_ssize_t n) {
    const int32_t *lens, *seqs;
    double scale, k_scale, v_scale;
    int64_t window, order, s_mode, weights_stride = 0, weights_len = 0;
    jq_kv_cache c = {};
    const at::Tensor *k = nullptr;
    if (!argument_count(n, 16)) return nullptr;
    const at::Tensor *q = strided_arg(a[0], at::kFloat, 3, "q", nullptr);
    if (q == nullptr) return nullptr;
    const int64_t T = q->size(0), H = q->size(1);
    if (!cache_arg(a[1], a[2], a[3], q, &c, &k) || !size_is(q->size(2), c.head_dim, "q", "elements in a head") ||
        !vector_arg(a[4], T, "lens", *q, false, &lens) || !vector_arg(a[5], T, "seqs", *q, true, &seqs) || !double_arg(a[6], &scale) ||
        !size_arg(a[7], &window) || !double_arg(a[8], &k_scale) || !double_arg(a[9], &v_scale) || !size_arg(a[12], &order) || !size_arg(a[13], &s_mode))
        return nullptr;
    c.k_scale = (float)k_scale, c.v_scale = (float)v_scale;
    float *out = nullptr, *weights = nullptr;
    void *xq = nullptr;
    if (a[10] != Py_None) {
        const at::Tensor *t = tensor_arg(a[10], at::kFloat, "out");
        if (t == nullptr || !size_is(t->numel(), q->numel(), "out", "elements")) return nullptr;
        if (t->get_device() != q->get_device()) {
            PyErr_SetString(PyExc_ValueError, "out is on another device than the other tensors");
            return nullptr;
        }
        out = static_cast<float *>(t->data_ptr());
    }
    if (a[11] != Py_None) {
        const at::Tensor *t = tensor_arg(a[11], at::kByte, "xq");
        if (t == nullptr) return nullptr;
        if (t->numel() < T * ((H * c.head_dim + 127) / 128) * 144 || t->get_device() != q->get_device()) {
            PyErr_SetString(PyExc_ValueError, "xq is too small for the Q8_1 blocks, or on another device");
            return nullptr;
        }
        xq = t->data_ptr();
    }
    if (a[14] != Py_None) {
        const at::Tensor *t = strided_arg(a[14], at::kFloat, 3, "weights", q);
        if (t == nullptr || !size_is(t->size(0), T, "weights", "rows") || !size_is(t->size(1), c.num_kv_heads, "weights", "heads")) return nullptr;
        weights_stride = c.num_kv_heads > 1 ? t->stride(1) : T > 1 ? t->stride(0) : t->size(2);
        if ((T > 1 && c.num_kv_heads > 1 && t->stride(0) != weights_stride * c.num_kv_heads)) {
            PyErr_SetString(PyExc_ValueError, "weights must have its rows and heads evenly spaced");
            return nullptr;
        }
        weights_len = t->size(2);
        weights = static_cast<float *>(t->data_ptr());
    }
    const at::Tensor *ws = tensor_arg(a[15], at::kByte, "ws");
    if (ws == nullptr) return nullptr;
    if (ws->get_device() != q->get_device()) {
        PyErr_SetString(PyExc_ValueError, "ws is on another device than the other tensors");
        return nullptr;
    }
    void *wp = ws->data_ptr();
    const size_t ws_bytes = (size_t)ws->numel();
    const float *qp = static_cast<const float *>(q->data_ptr());
    const int64_t s[2] = {q->stride(0), q->stride(1)};
    return status_of(*q, [&](void *st) {
        return f_attention(st, qp, s[0], s[1], T, H, &c, lens, seqs, (float)scale, window, out, xq, (int)order, (int)s_mode, weights, weights_stride, weights_len,
                           wp, ws_bytes);
    });
}

// (weights, lens, k, v, page_table, new_page_table or None, keep, recent, sinks, kept, new_lens, new_weights)
PyObject *evict(PyObject *const *a, Py_ssize_t n) {
    const int32_t *lens, *new_lens, *new_table = nullptr;
    int64_t keep, recent, sinks, new_pages = 0, new_stride = 0;
    jq_kv_cache c = {};
    const at::Tensor *k = nullptr;
    if (!argument_count(n, 12)) return nullptr;
    const at::Tensor *w = strided_arg(a[0], at::kFloat, 3, "weights", nullptr);
    if (w == nullptr || !cache_arg(a[2], a[3], a[4], w, &c, &k)) return nullptr;
    const int64_t B = c.num_seqs, H = c.num_kv_heads;
    if (!vector_arg(a[1], B, "lens", *w, false, &lens) || !size_arg(a[6], &keep) || !size_arg(a[7], &recent) || !size_arg(a[8], &sinks) ||
        !vector_arg(a[10], B, "new_lens", *w, false, &new_lens))
        return nullptr;
    const at::Tensor *nw = strided_arg(a[11], at::kFloat, 3, "new_weights", w), *kept = tensor_arg(a[9], at::kInt, "kept");
    if (nw == nullptr || kept == nullptr) return nullptr;
    if (kept->get_device() != w->get_device() || kept->numel() != B * H * keep) {
        PyErr_SetString(PyExc_ValueError, "kept must have [sequences, heads, keep] elements on the device of the other tensors");
        return nullptr;
    }
    int64_t stride[2];
    const at::Tensor *both[2] = {w, nw};
    for (int i = 0; i < 2; ++i) {
        const char *name = i == 0 ? "weights" : "new_weights";
        if (!size_is(both[i]->size(0), B, name, "rows") || !size_is(both[i]->size(1), H, name, "heads") || !size_is(both[i]->size(2), w->size(2), name, "tokens"))
            return nullptr;
        stride[i] = H > 1 ? both[i]->stride(1) : B > 1 ? both[i]->stride(0) : both[i]->size(2);
        if (B > 1 && H > 1 && both[i]->stride(0) != stride[i] * H) {
            PyErr_Format(PyExc_ValueError, "%s must have its rows and heads evenly spaced", name);
            return nullptr;
        }
    }
    if (a[5] != Py_None) {
        const at::Tensor *t = strided_arg(a[5], at::kInt, 2, "new_page_table", w);
        if (t == nullptr || !size_is(t->size(0), B, "new_page_table", "rows")) return nullptr;
        new_table = static_cast<const int32_t *>(t->data_ptr());
        new_pages = t->size(1);
        new_stride = B > 1 ? t->stride(0) : t->size(1);
    }
    const float *wp = static_cast<const float *>(w->data_ptr());
    float *nwp = static_cast<float *>(nw->data_ptr());
    int32_t *kp = static_cast<int32_t *>(kept->data_ptr());
    const int64_t S = w->size(2);
    return status_of(*w, [&](void *st) {
        return f_evict(st, &c, lens, wp, stride[0], S, keep, recent, sinks, new_table, new_pages, new_stride, kp, const_cast<int32_t *>(new_lens), nwp,
                       stride[1]);
    });
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(&entry<f>)), METH_FASTCALL
PyMethodDef methods[] = {
    {"bind", bind, METH_O, "Addresses of the library's functions, by name; the first time of all of them."},
    {"quantize", FAST(quantize), "(x, out, order, s_mode) -> status"},
    {"mul_mat", FAST(mul_mat), "(w, xq, out, K, N, M, order, kernel) -> status"},
    {"linear", FAST(linear), "(w, x, ws, out, N, s_mode) -> status"},
    {"multi", FAST(multi), "(ws_list, N_list, outs, x, xq, ws, K, M, s_mode) -> status"},
    {"rms_norm", FAST(rms_norm), "(x, weight, epsilon, residual, normed, xq, order, s_mode) -> status"},
    {"swiglu", FAST(swiglu), "(gate, up, mid, xq, order, s_mode) -> status"},
    {"rope", FAST(rope), "(x, out, positions, table, interleaved, mscale) -> status"},
    {"rope_append", FAST(rope_append),
     "(qkv, q_out, positions, table, k, v, page_table, index, seqs, k_scale, v_scale, interleaved, mscale) -> status"},
    {"attention_ws_bytes", FAST(attention_ws_bytes), "(q, k, page_table, weights) -> bytes"},
    {"attention", FAST(attention),
     "(q, k, v, page_table, lens, seqs, scale, window, k_scale, v_scale, out, xq, order, s_mode, weights, ws) -> status"},
    {"evict", FAST(evict), "(weights, lens, k, v, page_table, new_page_table, keep, recent, sinks, kept, new_lens, new_weights) -> status"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_calls", "Native part of capi.py's tensor calls.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__torch_calls(void) { return PyModule_Create(&module); }
