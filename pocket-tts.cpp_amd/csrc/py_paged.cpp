// Python binding of the paged-cache operators (module _ptts_paged, used through pyhost/ptts_paged.py).
//
// A decode step makes a few of these calls per layer and each kernel takes a few microseconds, so the binding reads its arrays in C:
// torch tensors through the C exchange table that array libraries publish on their types (attribute __dlpack_c_exchange_api__, DLPack
// 1.2: the structures below restate its layout), other device memory as DeviceArray.  It links neither torch nor
// libpocket_tts.so: the entry points' addresses come from ptts_lib, which decides whose HIP runtime the library is bound to.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <exception>
#include <initializer_list>

#include "pocket_tts/pocket_tts_amd.h"
#include "rotary_frequencies.h"

namespace {

// ------------------------------------------------------------------ exchange table (DLPack 1.2)

struct DlDevice { int32_t type, id; };
struct DlType { uint8_t code, bits; uint16_t lanes; };
struct DlTensor { void* data; DlDevice device; int32_t ndim; DlType dtype; int64_t* shape; int64_t* strides; uint64_t byte_offset; };
struct DlApi {
    struct { uint32_t major, minor; void* prev; } header;
    void *allocate, *managed_from, *managed_to;
    int (*view)(void* object, DlTensor* out);
    int (*stream)(int32_t device_type, int32_t device, void** out);
};
constexpr int kCuda = 2, kRocm = 10;

// ------------------------------------------------------------------ state of the module

PyObject *g_error = nullptr;       // ptts_lib.PttsError
PyObject *g_bind = nullptr;        // callable(with_torch): loads the library and calls bind()
PyObject *g_allocate = nullptr;    // callable(device, bytes, stream or None): a torch tensor for the workspace
PyObject *g_records = nullptr;     // callable(): whether torch records gradients now
PyObject *g_needs_grad = nullptr;  // "requires_grad"
int g_runtime = 0;                 // 0: not bound, 1: the system's runtime, 2: torch's

struct Entries {
    int (*plan)(const PttsPagedPlan*, int, void*);
    int (*rotary)(const PttsRotaryAppend*, int, void*);
    long long (*workspace)(const PttsPagedAttention*, int);
    int (*attention)(const PttsPagedAttention*, int, void*);
    const char* (*last_error)();
} g_lib;

bool fail(const char* format, const char* name, const char* more = "") {
    PyErr_Format(g_error ? g_error : PyExc_RuntimeError, format, name, more);
    return false;
}

// ------------------------------------------------------------------ arrays

enum Kind { kF32, kBf16, kF16, kI32, kF64, kOther };          // the first three are PTTS_TYPE_*
const char* const kKindNames[] = {"float32", "bfloat16", "float16", "int32", "float64", "another type"};
const int kKindSizes[] = {4, 2, 2, 4, 8, 1};

struct DeviceArray {
    PyObject_HEAD
    unsigned long long ptr;
    int kind, device, ndim;
    long long shape[8], strides[8];
};
PyTypeObject* g_device_array = nullptr;

struct View {
    const char* name = "";
    void* ptr = nullptr;
    Kind kind = kOther;
    int device = -1, ndim = 0;
    bool torch = false, given = false;
    long long bytes = 0;
    long long shape[8], strides[8];
    const DlApi* api = nullptr;
    int dl_type = 0;
};

const DlApi* api_of(PyTypeObject* type) {
    static PyTypeObject* last = nullptr;
    static const DlApi* found = nullptr;
    if (type == last) return found;
    PyObject* capsule = PyObject_GetAttrString(reinterpret_cast<PyObject*>(type), "__dlpack_c_exchange_api__");
    if (!capsule) {
        PyErr_Clear();
        return nullptr;
    }
    auto* api = static_cast<const DlApi*>(PyCapsule_GetPointer(capsule, "dlpack_exchange_api"));
    Py_DECREF(capsule);
    if (!api || api->header.major != 1 || !api->view || !api->stream) {
        PyErr_Clear();
        return nullptr;
    }
    Py_INCREF(type);               // kept for the comparison above
    Py_XDECREF(last);
    last = type;
    found = api;
    return api;
}

// A tensor that requires gradients is refused while torch records them: these calls would drop them without a word.
bool no_gradient(PyObject* o, const char* name) {
    PyObject* needs = PyObject_GetAttr(o, g_needs_grad);
    if (!needs) {
        PyErr_Clear();
        return true;
    }
    const bool maybe = needs != Py_False;
    Py_DECREF(needs);
    if (!maybe) return true;
    PyObject* records = PyObject_CallNoArgs(g_records);
    if (!records) return false;
    const int on = PyObject_IsTrue(records);
    Py_DECREF(records);
    if (on < 0) return false;
    return !on || fail("%s: requires gradients, which these calls do not record: detach it, or call under torch.no_grad()%s", name);
}

// Any array; false with an exception set.
bool read(PyObject* o, const char* name, View& v) {
    v.name = name;
    v.given = true;
    if (Py_TYPE(o) == g_device_array) {
        const auto* d = reinterpret_cast<const DeviceArray*>(o);
        v.ptr = reinterpret_cast<void*>(d->ptr);
        v.kind = static_cast<Kind>(d->kind);
        v.device = d->device;
        v.ndim = d->ndim;
        std::memcpy(v.shape, d->shape, sizeof v.shape);
        std::memcpy(v.strides, d->strides, sizeof v.strides);
    } else {
        v.api = api_of(Py_TYPE(o));
        if (!v.api && PyObject_HasAttrString(o, "data_ptr"))
            return fail("%s: %s publishes no exchange table (__dlpack_c_exchange_api__, in PyTorch from 2.10 on): pass a DeviceArray", name, Py_TYPE(o)->tp_name);
        if (!v.api) return fail("%s: a torch tensor on the GPU or a DeviceArray is required, got %s", name, Py_TYPE(o)->tp_name);
        DlTensor t;
        if (v.api->view(o, &t) != 0) return false;
        if (t.dtype.code != 0 && !no_gradient(o, name)) return false;         // integers have none
        if (t.device.type != kCuda && t.device.type != kRocm) return fail("%s: the tensor is not on the GPU%s", name);
        if (t.ndim > 8) return fail("%s: too many axes%s", name);
        v.ptr = static_cast<char*>(t.data) + t.byte_offset;
        v.device = t.device.id;
        v.dl_type = t.device.type;
        v.ndim = t.ndim;
        v.torch = true;
        long long n = 1;
        for (int i = t.ndim - 1; i >= 0; --i) {
            v.shape[i] = t.shape[i];
            v.strides[i] = t.strides ? t.strides[i] : n;
            n *= t.shape[i];
        }
        const auto d = t.dtype;
        v.kind = d.lanes != 1 ? kOther : d.code == 2 && d.bits == 32 ? kF32 : d.code == 4 && d.bits == 16 ? kBf16 : d.code == 2 && d.bits == 16 ? kF16
                 : d.code == 0 && d.bits == 32 ? kI32 : d.code == 2 && d.bits == 64 ? kF64 : kOther;
        v.bytes = d.bits / 8;
    }
    if (!v.torch) v.bytes = kKindSizes[v.kind];
    long long count = 1;
    bool empty = false;
    for (int i = 0; i < v.ndim; ++i) {
        count *= v.shape[i];
        empty = empty || v.shape[i] == 0;
    }
    v.bytes *= count;
    if (empty) v.ptr = nullptr;
    return true;
}

constexpr unsigned kFloats = 1u << kF32 | 1u << kBf16 | 1u << kF16;

// An array of `rank` axes and one of the kinds, its last axis contiguous; the stride of an axis of one element says nothing and becomes 0.
bool read(PyObject* o, const char* name, int rank, unsigned kinds, View& v) {
    if (!read(o, name, v)) return false;
    if (v.ndim != rank) {
        PyErr_Format(g_error, "%s: %d axes are required, got %d", name, rank, v.ndim);
        return false;
    }
    if (!(kinds >> v.kind & 1)) {
        char want[64] = "";
        for (int k = 0; k < kOther; ++k)
            if (kinds >> k & 1) {
                if (*want) std::strcat(want, " or ");
                std::strcat(want, kKindNames[k]);
            }
        PyErr_Format(g_error, "%s: %s is required, got %s", name, want, kKindNames[v.kind]);
        return false;
    }
    if (rank > 0 && v.shape[rank - 1] > 1 && v.strides[rank - 1] != 1) return fail("%s: the last axis must be contiguous%s", name);
    for (int i = 0; i < rank; ++i) {
        if (v.shape[i] > 0x7fffffff) return fail("%s: an axis is too long%s", name);
        if (v.shape[i] <= 1) v.strides[i] = 0;
        else if (v.strides[i] <= 0) return fail("%s: strides must be positive (axes of one element repeated are not taken)%s", name);
    }
    return true;
}

bool has_shape(const View& v, std::initializer_list<long long> want) {       // -1: any
    int i = 0;
    for (long long n : want) {
        if (n >= 0 && v.shape[i] != n) {
            PyErr_Format(g_error, "%s: axis %d has %lld elements, shape needs %lld", v.name, i, v.shape[i], n);
            return false;
        }
        ++i;
    }
    return true;
}

// One device for all arrays of a call, and whether they are torch's; the library bound to the runtime that they need.
const View* same_device(std::initializer_list<const View*> views) {
    const View* first = nullptr;
    for (const View* v : views) {
        if (!v->given) continue;
        if (!first) first = v;
        if (v->device != first->device || v->torch != first->torch) {
            PyErr_SetString(g_error, "all arrays of a call must be on one device, and all torch tensors or all DeviceArray");
            return nullptr;
        }
    }
    if (g_runtime == 0 || (first->torch && g_runtime != 2)) {
        PyObject* r = PyObject_CallFunction(g_bind, "i", first->torch ? 1 : 0);
        if (!r) return nullptr;
        Py_DECREF(r);
    }
    return first;
}

// None: the current stream of the tensors' framework, or the default stream; else an integer handle or an object with cuda_stream.
bool stream_of(PyObject* o, const View& first, void** out) {
    *out = nullptr;
    if (!o || o == Py_None) return !first.torch || first.api->stream(first.dl_type, first.device, out) == 0;
    PyObject* h = PyObject_GetAttrString(o, "cuda_stream");
    if (!h) {
        PyErr_Clear();
        Py_INCREF(o);
        h = o;
    }
    const unsigned long long v = PyLong_AsUnsignedLongLong(h);
    Py_DECREF(h);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        return fail("%s: None, a stream or its handle is required%s", "stream");
    }
    *out = reinterpret_cast<void*>(v);
    return true;
}

// ------------------------------------------------------------------ arguments

struct Names {
    static constexpr int kMost = 24;
    const char* what;
    int count, positional, required;          // the first `positional` may come without a name, the bits of `required` have to come
    const char* text[kMost];
    PyObject* key[kMost];
};

bool parse(Names& n, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames, PyObject** out) {
    for (int i = 0; i < n.count; ++i) out[i] = nullptr;
    if (nargs > n.positional) {
        PyErr_Format(PyExc_TypeError, "%s() takes %d positional arguments, got %zd", n.what, n.positional, nargs);
        return false;
    }
    for (Py_ssize_t i = 0; i < nargs; ++i) out[i] = args[i];
    const Py_ssize_t kw = kwnames ? PyTuple_GET_SIZE(kwnames) : 0;
    for (Py_ssize_t i = 0; i < kw; ++i) {
        PyObject* key = PyTuple_GET_ITEM(kwnames, i);
        int at = -1;
        for (int j = 0; j < n.count && at < 0; ++j)
            if (n.key[j] == key) at = j;
        for (int j = 0; j < n.count && at < 0; ++j)
            if (PyUnicode_Compare(n.key[j], key) == 0) at = j;
        if (at < 0 || out[at]) {
            PyErr_Format(PyExc_TypeError, at < 0 ? "%s() has no argument %R" : "%s() got %R twice", n.what, key);
            return false;
        }
        out[at] = args[nargs + i];
    }
    for (int i = 0; i < n.count; ++i)
        if (!out[i] && (n.required >> i & 1)) {
            PyErr_Format(PyExc_TypeError, "%s() needs %s", n.what, n.text[i]);
            return false;
        }
    return true;
}
bool intern(Names& n) {
    for (int i = 0; i < n.count; ++i)
        if (!(n.key[i] = PyUnicode_InternFromString(n.text[i]))) return false;
    return true;
}

bool is_none(PyObject* o) { return !o || o == Py_None; }
bool int_of(PyObject* o, const char* name, int& out) {          // kept where absent
    if (!o) return true;
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) return false;
    if (v < -0x7fffffff || v > 0x7fffffff) return fail("%s: out of range%s", name);
    out = static_cast<int>(v);
    return true;
}
bool float_of(PyObject* o, float& out) {
    if (is_none(o)) return true;
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) return false;
    out = static_cast<float>(v);
    return true;
}

bool status_of(PyObject* o, View& v) {
    if (is_none(o)) return true;
    if (!read(o, "status", 1, 1u << kI32, v)) return false;
    return v.shape[0] >= 1 || fail("%s: one element is required%s", "status");
}

PyObject* ran(int rc) {
    if (rc < 0) {
        PyErr_SetString(g_error, g_lib.last_error());
        return nullptr;
    }
    Py_RETURN_NONE;
}

template <typename T> T* as(const View& v) { return static_cast<T*>(v.ptr); }

// ------------------------------------------------------------------ plan

Names g_plan_names = {"plan", 12, 5, 0x3ff, {"cached", "arriving", "free_pages", "block_table", "page_size", "slot_map", "positions", "cu_rows", "kv_len", "counts",
                                             "status", "stream"}, {}};

PyObject* plan(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
    PyObject* o[12];
    if (!parse(g_plan_names, args, nargs, kwnames, o)) return nullptr;
    View cached, arriving, free_pages, table, slots, positions, cu, kv_len, counts, status;
    constexpr unsigned I = 1u << kI32;
    if (!read(o[0], "cached", 1, I, cached) || !read(o[1], "arriving", 1, I, arriving) || !read(o[2], "free_pages", 1, I, free_pages) ||
        !read(o[3], "block_table", 2, I, table) || !read(o[5], "slot_map", 1, I, slots) || !read(o[6], "positions", 1, I, positions) ||
        !read(o[7], "cu_rows", 1, I, cu) || !read(o[8], "kv_len", 1, I, kv_len) || !read(o[9], "counts", 1, I, counts) || !status_of(o[10], status))
        return nullptr;
    const long long n = cached.shape[0], rows = slots.shape[0];
    if (!has_shape(arriving, {n}) || !has_shape(table, {n, -1}) || !has_shape(positions, {rows}) || !has_shape(cu, {n + 1}) || !has_shape(kv_len, {n}) ||
        !has_shape(counts, {4}))
        return nullptr;
    PttsPagedPlan p;
    std::memset(&p, 0, sizeof p);
    p.cached = as<int>(cached); p.arriving = as<int>(arriving); p.free_pages = as<int>(free_pages); p.block_table = as<int>(table);
    p.slot_map = as<int>(slots); p.positions = as<int>(positions); p.cu_rows = as<int>(cu); p.kv_len = as<int>(kv_len); p.counts = as<int>(counts);
    p.status = as<int>(status);
    p.table_stride = table.strides[0];
    p.requests = static_cast<int>(n); p.table_width = static_cast<int>(table.shape[1]); p.n_free = static_cast<int>(free_pages.shape[0]);
    p.rows = static_cast<int>(rows);
    if (!int_of(o[4], "page_size", p.page_size)) return nullptr;
    const View* first = same_device({&cached, &arriving, &free_pages, &table, &slots, &positions, &cu, &kv_len, &counts, &status});
    void* stream;
    if (!first || !stream_of(o[11], *first, &stream)) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = g_lib.plan(&p, first->device, stream);
    Py_END_ALLOW_THREADS return ran(rc);
}

// ------------------------------------------------------------------ pages

bool pages_of(PyObject* ko, PyObject* vo, long long heads, long long dim, View& k, View& v, PttsPages& p) {
    if (!read(ko, "k_pages", 4, kFloats, k) || !read(vo, "v_pages", 4, kFloats, v)) return false;
    if (!has_shape(v, {k.shape[0], k.shape[1], k.shape[2], k.shape[3]}) || !has_shape(k, {-1, -1, heads, dim})) return false;
    if (v.kind != k.kind || v.strides[0] != k.strides[0] || v.strides[1] != k.strides[1] || v.strides[2] != k.strides[2])
        return fail("%s: type and strides must be those of k_pages%s", "v_pages");
    p.k = k.ptr; p.v = v.ptr;
    p.page_stride = k.strides[0]; p.row_stride = k.strides[1]; p.head_stride = k.strides[2];
    p.type = k.kind;
    p.pages = static_cast<int>(k.shape[0]); p.page_size = static_cast<int>(k.shape[1]); p.kv_heads = static_cast<int>(k.shape[2]);
    p.head_dim = static_cast<int>(k.shape[3]);
    return true;
}

// ------------------------------------------------------------------ rotary append

Names g_rotary_names = {"rotary_append", 13, 5, 0x1f, {"q", "k", "v", "positions", "freq", "interleaved", "magnitude", "q_out", "slot_map", "k_pages", "v_pages",
                                                       "status", "stream"}, {}};

PyObject* rotary_append(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
    PyObject* o[13];
    if (!parse(g_rotary_names, args, nargs, kwnames, o)) return nullptr;
    View q, k, v, positions, freq, out, slots, kp, vp, status;
    PttsRotaryAppend p;
    std::memset(&p, 0, sizeof p);
    p.magnitude = 1.0f;
    if (!is_none(o[0])) {
        if (!read(o[0], "q", 3, kFloats, q) || !read(is_none(o[7]) ? o[0] : o[7], "q_out", 3, kFloats, out)) return nullptr;
        if (!has_shape(out, {q.shape[0], q.shape[1], q.shape[2]})) return nullptr;
        if (out.kind != q.kind) { fail("%s: must have q's type%s", "q_out"); return nullptr; }
        p.q = q.ptr; p.q_out = out.ptr;
        p.q_row_stride = q.strides[0]; p.q_head_stride = q.strides[1]; p.out_row_stride = out.strides[0]; p.out_head_stride = out.strides[1];
        p.q_heads = static_cast<int>(q.shape[1]);
    }
    const bool none = is_none(o[1]);
    if (none != is_none(o[2]) || none != is_none(o[8]) || none != is_none(o[9]) || none != is_none(o[10])) {
        PyErr_SetString(g_error, "k, v, slot_map, k_pages and v_pages come together");
        return nullptr;
    }
    if (!none) {
        if (!read(o[1], "k", 3, kFloats, k) || !read(o[2], "v", 3, kFloats, v) || !read(o[8], "slot_map", 1, 1u << kI32, slots)) return nullptr;
        if (!has_shape(v, {k.shape[0], k.shape[1], k.shape[2]}) || !has_shape(slots, {k.shape[0]})) return nullptr;
        if (v.kind != k.kind || (q.given && q.kind != k.kind)) { PyErr_SetString(g_error, "q, k and v must have one type"); return nullptr; }
        if (q.given && !has_shape(k, {q.shape[0], -1, q.shape[2]})) return nullptr;
        if (!pages_of(o[9], o[10], k.shape[1], k.shape[2], kp, vp, p.pages)) return nullptr;
        p.k = k.ptr; p.v = v.ptr; p.slot_map = as<int>(slots);
        p.k_row_stride = k.strides[0]; p.k_head_stride = k.strides[1]; p.v_row_stride = v.strides[0]; p.v_head_stride = v.strides[1];
    }
    const View& lead = q.given ? q : k;
    if (!lead.given) { PyErr_SetString(g_error, "nothing to rotate: q and k are both missing"); return nullptr; }
    if (none) p.pages.head_dim = static_cast<int>(lead.shape[2]);
    if (!read(o[3], "positions", 1, 1u << kI32, positions) || !read(o[4], "freq", 1, 1u << kF64, freq) || !has_shape(positions, {lead.shape[0]}) ||
        !status_of(o[11], status))
        return nullptr;
    p.positions = as<int>(positions); p.freq = as<double>(freq); p.status = as<int>(status);
    p.type = lead.kind;
    p.rows = static_cast<int>(lead.shape[0]);
    if (freq.shape[0] > 1 << 20) { fail("%s: too many frequencies%s", "freq"); return nullptr; }
    p.rot_dim = 2 * static_cast<int>(freq.shape[0]);
    if (o[5]) {
        const int t = PyObject_IsTrue(o[5]);
        if (t < 0) return nullptr;
        p.interleaved = t;
    }
    if (!float_of(o[6], p.magnitude)) return nullptr;
    const View* first = same_device({&q, &out, &k, &v, &slots, &kp, &vp, &positions, &freq, &status});
    void* stream;
    if (!first || !stream_of(o[12], *first, &stream)) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = g_lib.rotary(&p, first->device, stream);
    Py_END_ALLOW_THREADS return ran(rc);
}

// ------------------------------------------------------------------ attention

struct AttentionCall {
    View q, out, kp, vp, table, cu, kv_len, lse, status;
    PttsPagedAttention p;
    const View* first = nullptr;
};

// o: q, k_pages, v_pages, block_table, cu_rows, kv_len, out, lse, scale, window, sinks, max_rows, max_kv, status
bool attention_args(PyObject** o, AttentionCall& c) {
    constexpr unsigned I = 1u << kI32;
    if (!read(o[0], "q", 3, kFloats, c.q) || !read(o[6], "out", 3, kFloats, c.out)) return false;
    if (!has_shape(c.out, {c.q.shape[0], c.q.shape[1], c.q.shape[2]})) return false;
    if (c.out.kind != c.q.kind) return fail("%s: must have q's type%s", "out");
    PttsPagedAttention& p = c.p;
    std::memset(&p, 0, sizeof p);
    if (!pages_of(o[1], o[2], -1, c.q.shape[2], c.kp, c.vp, p.pages)) return false;
    if (!read(o[3], "block_table", 2, I, c.table) || !read(o[4], "cu_rows", 1, I, c.cu) || !read(o[5], "kv_len", 1, I, c.kv_len)) return false;
    const long long n = c.kv_len.shape[0];
    if (!has_shape(c.table, {n, -1}) || !has_shape(c.cu, {n + 1})) return false;
    if (!is_none(o[7]) && (!read(o[7], "lse", 2, 1u << kF32, c.lse) || !has_shape(c.lse, {c.q.shape[0], c.q.shape[1]}))) return false;
    if (!status_of(o[13], c.status)) return false;
    p.q = c.q.ptr; p.out = c.out.ptr; p.lse = as<float>(c.lse); p.cu_rows = as<int>(c.cu); p.kv_len = as<int>(c.kv_len); p.block_table = as<int>(c.table);
    p.status = as<int>(c.status);
    p.q_row_stride = c.q.strides[0]; p.q_head_stride = c.q.strides[1]; p.out_row_stride = c.out.strides[0]; p.out_head_stride = c.out.strides[1];
    p.lse_row_stride = c.lse.given ? c.lse.strides[0] : 0;
    p.table_stride = c.table.strides[0];
    p.scale = 1.0f / std::sqrt(static_cast<float>(c.q.shape[2]));
    p.q_type = c.q.kind;
    p.rows = static_cast<int>(c.q.shape[0]); p.requests = static_cast<int>(n); p.q_heads = static_cast<int>(c.q.shape[1]);
    p.table_width = static_cast<int>(c.table.shape[1]);
    if (!float_of(o[8], p.scale) || !int_of(o[9], "window", p.window) || !int_of(o[10], "sinks", p.sinks) || !int_of(o[11], "max_rows", p.max_rows) ||
        !int_of(o[12], "max_kv", p.max_kv))
        return false;
    c.first = same_device({&c.q, &c.out, &c.kp, &c.vp, &c.table, &c.cu, &c.kv_len, &c.lse, &c.status});
    return c.first != nullptr;
}

Names g_workspace_names = {"attention_workspace", 12, 6, 0x3f, {"q", "k_pages", "v_pages", "block_table", "cu_rows", "kv_len", "out", "scale", "window", "sinks",
                                                                "max_rows", "max_kv"}, {}};

PyObject* attention_workspace(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
    PyObject* o[12];
    if (!parse(g_workspace_names, args, nargs, kwnames, o)) return nullptr;
    PyObject* full[14] = {o[0], o[1], o[2], o[3], o[4], o[5], is_none(o[6]) ? o[0] : o[6], nullptr, o[7], o[8], o[9], o[10], o[11], nullptr};
    AttentionCall c;
    if (!attention_args(full, c)) return nullptr;
    if (is_none(o[6])) c.p.out = static_cast<char*>(c.p.out) + (c.p.out ? 16 : 0);      // stands for an out of its own, which is not looked at here
    const long long need = g_lib.workspace(&c.p, c.first->device);
    if (need < 0) return ran(-1);
    return PyLong_FromLongLong(need);
}

Names g_attention_names = {"attention", 16, 6, 0x7f, {"q", "k_pages", "v_pages", "block_table", "cu_rows", "kv_len", "out", "lse", "scale", "window", "sinks",
                                                      "max_rows", "max_kv", "status", "workspace", "stream"}, {}};

PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
    PyObject* o[16];
    if (!parse(g_attention_names, args, nargs, kwnames, o)) return nullptr;
    AttentionCall c;
    void* stream;
    if (!attention_args(o, c) || !stream_of(o[15], *c.first, &stream)) return nullptr;
    PyObject* own = nullptr;
    if (!is_none(o[14])) {
        View w;
        if (!read(o[14], "workspace", w)) return nullptr;
        long long n = 1;
        for (int i = w.ndim - 1; i >= 0; n *= w.shape[i], --i)
            if (w.shape[i] > 1 && w.strides[i] != n) { fail("%s: a contiguous array is required%s", "workspace"); return nullptr; }
        if (w.device != c.first->device) { fail("%s: must be on the arrays' device%s", "workspace"); return nullptr; }
        c.p.workspace = w.ptr;
        c.p.workspace_bytes = w.bytes;
    } else {
        const long long need = g_lib.workspace(&c.p, c.first->device);
        if (need < 0) return ran(-1);
        if (need > 0 && !c.first->torch) {
            PyErr_Format(g_error, "attention: a workspace of %lld bytes is required", need);
            return nullptr;
        }
        if (need > 0) {
            own = PyObject_CallFunction(g_allocate, "iLO", c.first->device, need, is_none(o[15]) ? Py_None : o[15]);
            View w;
            if (!own || !read(own, "workspace", w)) {
                Py_XDECREF(own);
                return nullptr;
            }
            c.p.workspace = w.ptr;
            c.p.workspace_bytes = w.bytes;
        }
    }
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = g_lib.attention(&c.p, c.first->device, stream);
    Py_END_ALLOW_THREADS Py_XDECREF(own);          // the allocator hands the memory to later work of the same stream only
    return ran(rc);
}

// ------------------------------------------------------------------ DeviceArray

int device_array_init(PyObject* self, PyObject* args, PyObject* kw) {
    auto* d = reinterpret_cast<DeviceArray*>(self);
    static const char* names[] = {"ptr", "shape", "dtype", "strides", "device", nullptr};
    PyObject *shape, *strides = Py_None;
    const char* dtype;
    d->device = 0;
    if (!PyArg_ParseTupleAndKeywords(args, kw, "KOs|Oi", const_cast<char**>(names), &d->ptr, &shape, &dtype, &strides, &d->device)) return -1;
    d->kind = -1;
    for (int k = 0; k < kOther; ++k)
        if (!std::strcmp(dtype, kKindNames[k])) d->kind = k;
    if (d->kind < 0) return fail("DeviceArray: unknown type %s%s", dtype), -1;
    auto take = [](PyObject* o, const char* what, long long* out, int want) {
        PyObject* f = PySequence_Fast(o, what);
        if (!f) return -1;
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(f);
        bool ok = n <= 8 && (want < 0 || n == want);
        for (Py_ssize_t i = 0; ok && i < n; ++i) {
            out[i] = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(f, i));
            if (out[i] < 0) ok = false;
        }
        Py_DECREF(f);
        if (PyErr_Occurred()) return -1;
        if (!ok) return fail("DeviceArray: %s: up to 8 numbers, none negative, are required%s", what), -1;
        return static_cast<int>(n);
    };
    d->ndim = take(shape, "shape", d->shape, -1);
    if (d->ndim < 0) return -1;
    if (strides != Py_None) return take(strides, "strides", d->strides, d->ndim) < 0 ? -1 : 0;
    long long n = 1;
    for (int i = d->ndim - 1; i >= 0; n *= d->shape[i], --i) d->strides[i] = n;
    return 0;
}

PyType_Slot g_device_array_slots[] = {
    {Py_tp_doc, const_cast<char*>("DeviceArray(ptr, shape, dtype, strides=None, device=0): a view of GPU memory that the caller owns.\n"
                                  "dtype: float32, bfloat16, float16, int32 or float64; strides count elements (default: contiguous).")},
    {Py_tp_init, reinterpret_cast<void*>(device_array_init)},
    {Py_tp_new, reinterpret_cast<void*>(PyType_GenericNew)},
    {0, nullptr}};
PyType_Spec g_device_array_spec = {"ptts_paged.DeviceArray", sizeof(DeviceArray), 0, Py_TPFLAGS_DEFAULT, g_device_array_slots};

// ------------------------------------------------------------------ module

// _frequencies(rot_dim, base, scaling, factor, trained, fast, slow, address of rot_dim / 2 doubles) -> magnitude
PyObject* frequencies(PyObject*, PyObject* args) {
    int rot_dim, scaling;
    double base, factor, trained, fast, slow;
    unsigned long long out;
    if (!PyArg_ParseTuple(args, "ididdddK", &rot_dim, &base, &scaling, &factor, &trained, &fast, &slow, &out)) return nullptr;
    try {
        float magnitude;
        ptts::rotary_frequencies(rot_dim, base, scaling, factor, trained, fast, slow, reinterpret_cast<double*>(out), &magnitude);
        return PyFloat_FromDouble(magnitude);
    } catch (const std::exception& e) {
        PyErr_SetString(g_error, e.what());
        return nullptr;
    }
}

PyObject* setup(PyObject*, PyObject* args) {
    PyObject *error, *bind, *allocate, *records;
    if (!PyArg_ParseTuple(args, "OOOO", &error, &bind, &allocate, &records)) return nullptr;
    Py_INCREF(error); Py_INCREF(bind); Py_INCREF(allocate); Py_INCREF(records);
    g_error = error; g_bind = bind; g_allocate = allocate; g_records = records;
    Py_RETURN_NONE;
}

PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long plan, rotary, workspace, attention, error;
    int with_torch;
    if (!PyArg_ParseTuple(args, "pKKKKK", &with_torch, &plan, &rotary, &workspace, &attention, &error)) return nullptr;
    g_lib.plan = reinterpret_cast<decltype(g_lib.plan)>(plan);
    g_lib.rotary = reinterpret_cast<decltype(g_lib.rotary)>(rotary);
    g_lib.workspace = reinterpret_cast<decltype(g_lib.workspace)>(workspace);
    g_lib.attention = reinterpret_cast<decltype(g_lib.attention)>(attention);
    g_lib.last_error = reinterpret_cast<decltype(g_lib.last_error)>(error);
    g_runtime = with_torch ? 2 : 1;
    Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL | METH_KEYWORDS
PyMethodDef g_methods[] = {
    {"plan", FAST(plan),
     "plan(cached, arriving, free_pages, block_table, page_size, *, slot_map, positions, cu_rows, kv_len, counts, status=None, stream=None)\n\n"
     "Block tables and slot maps from request lengths (ptts_paged_plan).  cached, arriving, kv_len: int32 [requests]; cu_rows\n"
     "[requests + 1]; free_pages [any]; block_table [requests][width], updated in place; slot_map, positions [rows]; counts [4];\n"
     "status [1] or None."},
    {"rotary_append", FAST(rotary_append),
     "rotary_append(q, k, v, positions, freq, *, interleaved=False, magnitude=1.0, q_out=None, slot_map=None, k_pages=None, v_pages=None,\n"
     "              status=None, stream=None)\n\n"
     "Rotates q [rows][q_heads][dim] into q_out (None: in place) and files k, v [rows][kv_heads][dim] into the pages\n"
     "[pages][page_size][kv_heads][dim] at slot_map [rows] (ptts_rotary_append).  positions: int32 [rows]; freq: float64 [rot_dim / 2].\n"
     "q, or k, v, slot_map and the pages, may be None."},
    {"attention_workspace", FAST(attention_workspace),
     "attention_workspace(q, k_pages, v_pages, block_table, cu_rows, kv_len, *, out=None, scale=None, window=0, sinks=0, max_rows=0, max_kv=0)\n\n"
     "Bytes of workspace that attention() needs for these arguments (ptts_paged_attention_workspace)."},
    {"attention", FAST(attention),
     "attention(q, k_pages, v_pages, block_table, cu_rows, kv_len, *, out, lse=None, scale=None, window=0, sinks=0, max_rows=0, max_kv=0,\n"
     "          status=None, workspace=None, stream=None)\n\n"
     "Attention of every request's new rows over its pages (ptts_paged_attention).  q, out [rows][heads][dim]; block_table int32\n"
     "[requests][width]; cu_rows [requests + 1]; kv_len [requests]; lse float32 [rows][heads] or None; scale: default dim ** -0.5.\n"
     "workspace: any contiguous array of at least attention_workspace() bytes; None: torch's allocator provides it (torch tensors only)."},
    {"setup", setup, METH_VARARGS, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {"_frequencies", frequencies, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_ptts_paged", "C side of ptts_paged", -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ptts_paged(void) {
    for (Names* n : {&g_plan_names, &g_rotary_names, &g_workspace_names, &g_attention_names})
        if (!intern(*n)) return nullptr;
    if (!(g_needs_grad = PyUnicode_InternFromString("requires_grad"))) return nullptr;
    PyObject* type = PyType_FromSpec(&g_device_array_spec);
    if (!type) return nullptr;
    g_device_array = reinterpret_cast<PyTypeObject*>(type);
    PyObject* m = PyModule_Create(&g_module);
    if (!m) return nullptr;
    Py_INCREF(type);
    if (PyModule_AddObject(m, "DeviceArray", type) < 0) return nullptr;
    return m;
}
