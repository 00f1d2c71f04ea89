// m27q_torch.cpp -- the token mixers' calls, and those of a batch's steps beside them, for Python, straight from tensors.
//
// A call costs the GPU as little as 4 us; reading shapes, strides and pointers of
// up to ten tensors through Python costs the host as much again.  This module
// reads them from the tensors themselves (0.4 us a call) and returns the
// library's status; shapes that the records cannot express are M27Q_ERR_SHAPE, and
// a call with a tensor that the current GPU cannot read is kNotHere.
#include <Python.h>

#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>

#include "../../include/m27q.h"

namespace {

struct Bad {
    int status;  // m27q_status, or kNotHere
};
constexpr int kNotHere = -1;

// The GPU that a call's tensors lie on.  A kernel that follows a pointer to pageable host
// memory or into another GPU faults, so such a call is refused.  The codes are those of the
// binding's records: a GPU's number, kHost, or kPinned, which every GPU reads.
constexpr int32_t kHost = -1, kPinned = -2;
thread_local int32_t place;
thread_local bool apart;

void note(int32_t at) {
    if (at == kPinned) return;
    if (place == kPinned) place = at;
    apart |= at == kHost || at != place;
}

const at::Tensor *tensor(PyObject *o, bool may_be_none = false) {
    if (may_be_none && o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) throw Bad{M27Q_ERR_NULL};
    return &THPVariable_Unpack(o);
}

uint32_t type_of(const at::Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return M27Q_TYPE_F32;
        case at::kHalf: return M27Q_TYPE_F16;
        case at::kBFloat16: return M27Q_TYPE_BF16;
        default: return 0xffffffffu;  // for the library to refuse
    }
}

void *data(const at::Tensor &t) {
    note(t.is_cuda() ? t.get_device() : t.is_pinned() ? kPinned : kHost);
    return t.mutable_data_ptr();
}

struct Scratch {
    void *ptr;
    size_t bytes;
    explicit Scratch(PyObject *o) {
        const at::Tensor &t = *tensor(o);
        if (!t.is_contiguous()) throw Bad{M27Q_ERR_LAYOUT};  // its elements need not be as many bytes of memory
        ptr = data(t);
        bytes = t.numel() * t.element_size();
    }
};

m27q_rows rows(PyObject *o, int64_t tokens) {
    const at::Tensor &t = *tensor(o);
    if (t.dim() != 3 || t.size(0) != tokens || (t.stride(2) != 1 && t.size(2) != 1) || t.size(1) > 0xffff || t.size(2) > 0xffff)
        throw Bad{M27Q_ERR_SHAPE};
    return {data(t), type_of(t), (uint32_t)t.size(1), (uint32_t)t.size(2), 0, t.stride(0), t.stride(1)};
}

// [tokens][dim] or [tokens][heads][dim] of a norm, which may be missing (no ptr).
m27q_rows norm_rows(PyObject *o, int64_t tokens) {
    const at::Tensor *t = tensor(o, true);
    if (!t) return {};
    const int64_t d = t->dim(), dim = d < 2 ? 0 : t->size(d - 1), heads = d == 3 ? t->size(1) : 1;
    if (d < 2 || d > 3 || t->size(0) != tokens || (t->stride(d - 1) != 1 && dim != 1) || heads > 0xffff || dim > 0x7fffffff)
        throw Bad{M27Q_ERR_SHAPE};
    return {data(*t), type_of(*t), (uint32_t)heads, (uint32_t)dim, 0, t->stride(0), d == 3 ? t->stride(1) : dim};
}

const int32_t *int32s(PyObject *o, int64_t n, bool may_be_none = false) {
    const at::Tensor *t = tensor(o, may_be_none);
    if (!t) return nullptr;
    if (t->scalar_type() != at::kInt || !t->is_contiguous()) throw Bad{M27Q_ERR_LAYOUT};
    if (n >= 0 && t->numel() != n) throw Bad{M27Q_ERR_SHAPE};
    return (const int32_t *)data(*t);
}

float *floats(PyObject *o, int64_t n, bool may_be_none = false) {
    const at::Tensor *t = tensor(o, may_be_none);
    if (!t) return nullptr;
    if (t->scalar_type() != at::kFloat || !t->is_contiguous() || t->numel() != n) throw Bad{M27Q_ERR_SHAPE};
    return (float *)data(*t);
}

// A record that the Python side packed when its object was made, and where its tensors lie.
template <typename T>
const T *record(PyObject *o) {
    int32_t at;
    if (!PyBytes_Check(o) || PyBytes_GET_SIZE(o) != sizeof(T) + sizeof at) throw Bad{M27Q_ERR_NULL};
    memcpy(&at, PyBytes_AS_STRING(o) + sizeof(T), sizeof at);
    note(at);
    return (const T *)PyBytes_AS_STRING(o);
}

PyObject *stream_of = nullptr;  // the binding's function from a stream argument (or None) to its handle

struct Args {
    PyObject *const *a;
    double real(int i) const {
        const double v = PyFloat_AsDouble(a[i]);
        if (v == -1.0 && PyErr_Occurred()) throw Bad{M27Q_ERR_RANGE};
        return v;
    }
    long long whole(int i) const {
        const long long v = PyLong_AsLongLong(a[i]);
        if (v == -1 && PyErr_Occurred()) throw Bad{M27Q_ERR_RANGE};
        return v;
    }
    uint32_t u32(int i) const {
        const long long v = whole(i);
        if (v < 0 || v > 0xffffffffll) throw Bad{M27Q_ERR_RANGE};
        return (uint32_t)v;
    }
    // Last, when all other arguments are known to fit: in a statement of its own, as a call's arguments are
    // evaluated in any order, and a tensor that is looked at later is not refused.
    hipStream_t stream(int i) const {
        if (apart || (place != kPinned && place != c10::impl::getDeviceGuardImpl(at::kCUDA)->getDevice().index()))
            throw Bad{kNotHere};
        PyObject *h = stream_of ? PyObject_CallOneArg(stream_of, a[i]) : nullptr;
        const unsigned long long v = h ? PyLong_AsUnsignedLongLong(h) : 0;
        Py_XDECREF(h);
        if (!h || PyErr_Occurred()) throw Bad{M27Q_ERR_NULL};
        return (hipStream_t)(uintptr_t)v;
    }
};

template <typename F>
PyObject *call(PyObject *const *a, Py_ssize_t n, Py_ssize_t want, F f) {
    if (n != want) {
        PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
        return nullptr;
    }
    place = kPinned;
    apart = false;
    try {
        return PyLong_FromLong((long)f(Args{a}));
    } catch (const Bad &b) {
        if (PyErr_Occurred()) return nullptr;  // the stream could not be had, or an argument is of another kind
        return PyLong_FromLong((long)b.status);
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// plan, pos, x, out, stream
PyObject *py_rope(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return call(a, n, 5, [](Args c) {
        const int64_t tokens = tensor(c.a[1])->numel();
        if (tokens > 0x7fffffff) throw Bad{M27Q_ERR_SHAPE};
        const int32_t *pos = int32s(c.a[1], tokens);
        const m27q_rows x = rows(c.a[2], tokens), out = rows(c.a[3], tokens);
        const m27q_rope_plan *plan = record<m27q_rope_plan>(c.a[0]);
        const hipStream_t stream = c.stream(4);
        return m27q_rope(plan, pos, (int)tokens, &x, &out, stream);
    });
}

// plan, pos, seqs, cache, q, q_out, k, v, stream
PyObject *py_rope_append(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return call(a, n, 9, [](Args c) {
        const m27q_seqs *s = record<m27q_seqs>(c.a[2]);
        const int64_t t = s->tokens;
        const int32_t *pos = int32s(c.a[1], t);
        const m27q_rows q = rows(c.a[4], t), q_out = rows(c.a[5], t), k = rows(c.a[6], t), v = rows(c.a[7], t);
        const m27q_rope_plan *plan = record<m27q_rope_plan>(c.a[0]);
        const m27q_cache *cache = record<m27q_cache>(c.a[3]);
        const hipStream_t stream = c.stream(8);
        return m27q_rope_append(plan, pos, s, cache, &q, &q_out, &k, &v, stream);
    });
}

// seqs, cache, q, out, scratch, scale, window, stream
PyObject *py_attn_paged(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return call(a, n, 8, [](Args c) {
        const m27q_seqs *s = record<m27q_seqs>(c.a[0]);
        const m27q_rows q = rows(c.a[2], s->tokens), out = rows(c.a[3], s->tokens);
        const m27q_cache *cache = record<m27q_cache>(c.a[1]);
        const Scratch scratch(c.a[4]);
        const float scale = (float)c.real(5);
        const long long window = c.whole(6);
        if (window > 0x7fffffff || window < 0) throw Bad{M27Q_ERR_RANGE};
        const hipStream_t stream = c.stream(7);
        return m27q_attn_paged(s, cache, &q, &out, scale, (int)window, scratch.ptr, scratch.bytes, stream);
    });
}

// seqs, prefixes, cache, q, out, scratch, scale, stream
PyObject *py_attn_shared(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return call(a, n, 8, [](Args c) {
        const m27q_seqs *s = record<m27q_seqs>(c.a[0]);
        const m27q_prefixes *x = record<m27q_prefixes>(c.a[1]);
        const m27q_rows q = rows(c.a[3], s->tokens), out = rows(c.a[4], s->tokens);
        const m27q_cache *cache = record<m27q_cache>(c.a[2]);
        const Scratch scratch(c.a[5]);
        const float scale = (float)c.real(6);
        const hipStream_t stream = c.stream(7);
        return m27q_attn_shared(s, x, cache, &q, &out, scale, scratch.ptr, scratch.bytes, stream);
    });
}

// x, add, weight, eps, sum, out, act's buffer, M, K, stream
PyObject *py_rms_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return call(a, n, 10, [](Args c) {
        const at::Tensor &t = *tensor(c.a[0]);
        if (t.dim() < 2 || t.size(0) > 0x7fffffff) throw Bad{M27Q_ERR_SHAPE};
        const int64_t tokens = t.size(0);
        const m27q_rows x = norm_rows(c.a[0], tokens), add = norm_rows(c.a[1], tokens), sum = norm_rows(c.a[4], tokens),
                        out = norm_rows(c.a[5], tokens);
        const float *weight = floats(c.a[2], x.dim, true);
        void *xq = nullptr;
        if (const at::Tensor *act = tensor(c.a[6], true)) {
            const long long M = c.whole(7), K = c.whole(8);
            if (!act->is_contiguous()) throw Bad{M27Q_ERR_LAYOUT};
            if (M != tokens || K != (long long)x.heads * x.dim || M > 0xffff + 1 || K > (1 << 20) ||
                (size_t)(act->numel() * act->element_size()) < m27q_act_bytes((int)M, (int)K))
                throw Bad{M27Q_ERR_SHAPE};
            xq = data(*act);
        }
        const float eps = (float)c.real(3);
        const hipStream_t stream = c.stream(9);
        return m27q_rms_norm(&x, add.ptr ? &add : nullptr, (int)tokens, weight, eps, sum.ptr ? &sum : nullptr,
                             out.ptr ? &out : nullptr, xq, stream);
    });
}

// logits, u, token, scratch, temperature, top_k, top_p, min_p, prob, stream
PyObject *py_sample_rows(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return call(a, n, 10, [](Args c) {
        const at::Tensor &t = *tensor(c.a[0]);
        if (t.dim() != 2 || t.size(0) > 0x7fffffff || t.size(1) > 0x7fffffff || (t.stride(1) != 1 && t.size(1) != 1))
            throw Bad{M27Q_ERR_SHAPE};
        const int64_t rows = t.size(0);
        m27q_sampling s{};
        s.logits = data(t);
        s.type = type_of(t);
        s.rows = (uint32_t)rows;
        s.n = (uint32_t)t.size(1);
        s.stride = rows == 1 ? t.size(1) : t.stride(0);
        s.u = floats(c.a[1], rows);
        s.token = const_cast<int32_t *>(int32s(c.a[2], rows));
        s.temperature = floats(c.a[4], rows, true);
        s.top_k = int32s(c.a[5], rows, true);
        s.top_p = floats(c.a[6], rows, true);
        s.min_p = floats(c.a[7], rows, true);
        s.prob = floats(c.a[8], rows, true);
        const Scratch scratch(c.a[3]);
        const hipStream_t stream = c.stream(9);
        return m27q_sample_rows(&s, scratch.ptr, scratch.bytes, stream);
    });
}

// start, q, k, v, g, beta, state, state_out, out, scratch, scale, max_len, slots, head_map, stream
PyObject *py_delta_rule(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return call(a, n, 15, [](Args c) {
        const at::Tensor &v = *tensor(c.a[3]), &start = *tensor(c.a[0]);
        if (v.dim() != 3 || start.numel() < 1 || start.numel() > 0x7fffffff) throw Bad{M27Q_ERR_SHAPE};
        const int64_t tokens = v.size(0);
        if (tokens > 0x7fffffff) throw Bad{M27Q_ERR_SHAPE};
        m27q_delta d{};
        d.q = rows(c.a[1], tokens);
        d.k = rows(c.a[2], tokens);
        d.v = rows(c.a[3], tokens);
        d.out = rows(c.a[8], tokens);
        d.start = int32s(c.a[0], -1);
        d.n = (uint32_t)(start.numel() - 1);
        d.slots = int32s(c.a[12], d.n, true);
        d.g = floats(c.a[4], tokens * d.v.heads);
        d.beta = floats(c.a[5], tokens * d.v.heads);
        const at::Tensor *held = tensor(c.a[6], true);
        if (!held) held = tensor(c.a[7], true);
        if (held) {
            if (held->dim() != 4 || held->size(0) > 0x7fffffff || held->size(1) != d.v.heads || held->size(2) != d.v.dim || held->size(3) != d.k.dim)
                throw Bad{M27Q_ERR_SHAPE};
            d.n_slots = (uint32_t)held->size(0);
            d.state_in = floats(c.a[6], held->numel(), true);
            d.state_out = floats(c.a[7], held->numel(), true);
        }
        d.tokens = (uint32_t)tokens;
        d.scale = (float)c.real(10);
        d.max_len = c.u32(11);
        d.head_map = c.u32(13);
        const Scratch scratch(c.a[9]);
        const hipStream_t stream = c.stream(14);
        return m27q_delta_rule(&d, scratch.ptr, scratch.bytes, stream);
    });
}

PyObject *py_streams(PyObject *, PyObject *f) {
    Py_INCREF(f);
    Py_XDECREF(stream_of);
    stream_of = f;
    Py_RETURN_NONE;
}

#define FAST(f) (PyCFunction)(void (*)(void)) f, METH_FASTCALL
PyMethodDef methods[] = {{"rope", FAST(py_rope), nullptr},
                         {"rope_append", FAST(py_rope_append), nullptr},
                         {"attn_paged", FAST(py_attn_paged), nullptr},
                         {"attn_shared", FAST(py_attn_shared), nullptr},
                         {"delta_rule", FAST(py_delta_rule), nullptr},
                         {"rms_norm", FAST(py_rms_norm), nullptr},
                         {"sample_rows", FAST(py_sample_rows), nullptr},
                         {"streams", py_streams, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "m27q_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_m27q_torch(void) { return PyModule_Create(&module); }
