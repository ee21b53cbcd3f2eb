// Direct calls of the packed / paged attention, cache and verification entry points for torch tensors (module
// imagecaption_amd._calls).
//
// ops.py checks its arguments in Python and calls libcapdec.so through ctypes: 4 to 9 us of host time a call, next to 3 for
// the launch itself and 3 to 9 for the kernels of a decode step.  The functions here take the plain form of each call -- results
// allocated here, every row of a matrix in use -- check it and make it.  Whatever they do not take returns None: ops.py then goes
// its general way, which also words the errors, so nothing is refused or accepted here that is not there.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "../../include/capdec.h"

// the torch and the Python this was built for; build.py looks for it in the file before anything is loaded
extern "C" __attribute__((used, visibility("default"))) const char capdec_calls_stamp[] = CAPDEC_CALLS_STAMP;

namespace {

struct Entry {
    decltype(&capdec_attn_packed_fwd) packed_fwd;
    decltype(&capdec_attn_packed_scratch_bytes) packed_scratch;
    decltype(&capdec_attn_packed_bwd) packed_bwd;
    decltype(&capdec_kv_write) kv_write;
    decltype(&capdec_kv_read) kv_read;
    decltype(&capdec_attn_paged_workspace_bytes) paged_workspace;
    decltype(&capdec_attn_paged) paged;
    decltype(&capdec_draft_verify) verify;
} lib;

struct Matrix {
    void* at;
    int ld;
    int64_t rows;
};

const at::Tensor* tensor(PyObject* o, at::ScalarType type, int64_t dims, int64_t device) {
    if (!THPVariable_Check(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || t.scalar_type() != type || t.dim() != dims || !t.is_cuda() || t.get_device() != device || t.layout() != at::kStrided)
        return nullptr;
    return &t;
}

// [>= rows, width], 16-byte aligned, unit column stride, rows in whole 16-byte pieces
bool matrix(PyObject* o, at::ScalarType type, int64_t rows, int64_t width, int64_t device, Matrix* m) {
    const at::Tensor* t = tensor(o, type, 2, device);
    if (!t || t->size(1) != width || t->size(0) < rows) return false;
    m->at = t->data_ptr();
    m->rows = t->size(0);
    if ((uintptr_t)m->at & 15) return false;
    if (t->is_contiguous()) {
        m->ld = (int)width;
        return true;
    }
    const int64_t ld = t->stride(0);
    if (t->stride(1) != 1 || ld < width || ld >= (1ll << 31) || (ld * (int64_t)t->element_size()) & 15) return false;
    m->ld = (int)ld;
    return true;
}

bool vector(PyObject* o, at::ScalarType type, int64_t n, int64_t device, const void** at) {
    const at::Tensor* t = tensor(o, type, 1, device);
    if (!t || t->numel() != n || !t->is_contiguous()) return false;
    *at = t->data_ptr();
    return true;
}

struct Args {
    PyObject* const* a;
    bool ok = true;
    int64_t integer(int i) {
        const long long v = PyLong_AsLongLong(a[i]);
        if (v == -1 && PyErr_Occurred()) {
            PyErr_Clear();
            ok = false;
        }
        return v;
    }
    void* address(int i) { return (void*)(uintptr_t)integer(i); }
    float scale(int i, int dh) {
        if (a[i] == Py_None) return (float)(1.0 / std::sqrt((double)dh));
        const double v = PyFloat_AsDouble(a[i]);
        if (v == -1.0 && PyErr_Occurred()) {
            PyErr_Clear();
            ok = false;
        }
        return (float)v;
    }
};

at::Tensor new_like(const Matrix& m, int64_t width, const at::Tensor& like) { return at::empty({m.rows, width}, like.options()); }

PyObject* none() { Py_RETURN_NONE; }

// something was thrown (an unusual tensor, no memory) or raised: the general way meets and reports the same
PyObject* refused() {
    PyErr_Clear();
    return none();
}

// the results of a call whose return code was rc
template <typename... T>
PyObject* results(int rc, const T&... t) {
    if (rc != 0) return none();
    if constexpr (sizeof...(T) == 0) {
        Py_RETURN_TRUE;
    } else if constexpr (sizeof...(T) == 1) {
        return THPVariable_Wrap(t...);
    } else {
        PyObject* out = PyTuple_New(sizeof...(T));
        Py_ssize_t i = 0;
        (PyTuple_SET_ITEM(out, i++, t.defined() ? THPVariable_Wrap(t) : none()), ...);
        return out;
    }
}

// q, k, v of a packed call: arguments 1 to 5 are q, k, v, Hq, Hkv
struct Packed {
    Matrix q, k, v;
    const capdec_packed_seqs* seqs;
    int Hq, Hkv, dh, dtype;
    at::ScalarType type;
    int64_t device;
    bool read(Args& x, int64_t dev) {
        if (!THPVariable_Check(x.a[1])) return false;
        const at::Tensor& t = THPVariable_Unpack(x.a[1]);
        seqs = (const capdec_packed_seqs*)x.address(0);
        const int64_t hq = x.integer(4), hkv = x.integer(5);
        device = dev;
        if (!x.ok || t.dim() != 2 || hq <= 0 || hkv <= 0 || hq % hkv || hq > (1 << 17) || seqs->rows_q <= 0 || seqs->rows_k <= 0) return false;
        type = t.scalar_type();
        if ((type != at::kFloat && type != at::kBFloat16) || (t.size(1) != 64 * hq && t.size(1) != 128 * hq)) return false;
        Hq = (int)hq;
        Hkv = (int)hkv;
        dh = (int)(t.size(1) / hq);
        dtype = type == at::kFloat ? CAPDEC_F32 : CAPDEC_BF16S;
        return wide(x.a[1], &q) && narrow(x.a[2], &k) && narrow(x.a[3], &v);
    }
    // matrices without rows behind the last sequence
    bool wide(PyObject* o, Matrix* m) const { return matrix(o, type, seqs->rows_q, (int64_t)Hq * dh, device, m) && m->rows == seqs->rows_q; }
    bool narrow(PyObject* o, Matrix* m) const { return matrix(o, type, seqs->rows_k, (int64_t)Hkv * dh, device, m) && m->rows == seqs->rows_k; }
};

// (seqs, q, k, v, Hq, Hkv, save_lse, scale, device, stream) -> (o, lse or None)
PyObject* attn_packed_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) try {
    Args x{a};
    Packed p;
    if (n != 10 || !p.read(x, x.integer(8))) return none();
    const float scale = x.scale(7, p.dh);
    void* stream = x.address(9);
    const int save = PyObject_IsTrue(a[6]);
    if (save < 0) return refused();
    if (!x.ok) return none();
    const at::Tensor& q = THPVariable_Unpack(a[1]);
    at::Tensor o = new_like(p.q, p.Hq * p.dh, q), lse;
    if (save) lse = at::empty({p.Hq, p.q.rows}, q.options().dtype(at::kFloat));
    void *po = o.data_ptr(), *pl = save ? lse.data_ptr() : nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = lib.packed_fwd(p.seqs, p.q.at, p.q.ld, p.k.at, p.k.ld, p.v.at, p.v.ld, po, p.Hq * p.dh, pl, (size_t)p.q.rows, p.Hq, p.Hkv, p.dh, p.dtype,
                        scale, stream);
    Py_END_ALLOW_THREADS;
    return results(rc, o, lse);
} catch (...) {
    return refused();
}

// (seqs, q, k, v, Hq, Hkv, o, do, lse, scale, device, stream) -> (dq, dk, dv)
PyObject* attn_packed_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) try {
    Args x{a};
    Packed p;
    Matrix o, dout;
    if (n != 12 || !p.read(x, x.integer(10)) || !p.wide(a[6], &o) || !p.wide(a[7], &dout)) return none();
    const at::Tensor* lse = tensor(a[8], at::kFloat, 2, p.device);
    const float scale = x.scale(9, p.dh);
    void* stream = x.address(11);
    if (!x.ok || !lse || lse->size(0) != p.Hq || lse->size(1) < p.q.rows || !lse->is_contiguous()) return none();
    const size_t rows = (size_t)lse->size(1), need = lib.packed_scratch(p.seqs, rows, p.Hq, p.Hkv, p.dh, p.dtype);
    at::Tensor dq = new_like(p.q, p.Hq * p.dh, THPVariable_Unpack(a[1])), dk = new_like(p.k, p.Hkv * p.dh, THPVariable_Unpack(a[2])),
               dv = new_like(p.v, p.Hkv * p.dh, THPVariable_Unpack(a[3])), scratch;
    if (need) scratch = at::empty({(int64_t)need}, lse->options().dtype(at::kByte));
    void *pl = lse->data_ptr(), *ps = need ? scratch.data_ptr() : nullptr, *pq = dq.data_ptr(), *pk = dk.data_ptr(), *pv = dv.data_ptr();
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = lib.packed_bwd(p.seqs, p.q.at, p.q.ld, p.k.at, p.k.ld, p.v.at, p.v.ld, o.at, o.ld, dout.at, dout.ld, pl, rows, ps, need, pq, p.Hq * p.dh,
                        pk, p.Hkv * p.dh, pv, p.Hkv * p.dh, p.Hq, p.Hkv, p.dh, p.dtype, scale, stream);
    Py_END_ALLOW_THREADS;
    return results(rc, dq, dk, dv);
} catch (...) {
    return refused();
}

// (cache, k, v, slots, device, stream) -> True
PyObject* kv_cache_write(PyObject*, PyObject* const* a, Py_ssize_t n) try {
    Args x{a};
    if (n != 6 || !THPVariable_Check(a[1]) || !THPVariable_Check(a[3])) return none();
    const auto* cache = (const capdec_kv_cache*)x.address(0);
    const int64_t device = x.integer(4), rows = THPVariable_Unpack(a[3]).numel();
    void* stream = x.address(5);
    const at::ScalarType type = THPVariable_Unpack(a[1]).scalar_type();
    const void* slots;
    Matrix k, v;
    if (!x.ok || rows >= (1ll << 31) || (type != at::kFloat && type != at::kBFloat16)) return none();
    const int64_t width = (int64_t)cache->heads * cache->dh;
    if (!matrix(a[1], type, rows, width, device, &k) || !matrix(a[2], type, rows, width, device, &v) || !vector(a[3], at::kInt, rows, device, &slots))
        return none();
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = lib.kv_write(cache, k.at, k.ld, v.at, v.ld, type == at::kFloat ? CAPDEC_F32 : CAPDEC_BF16S, (const int*)slots, (int)rows, stream);
    Py_END_ALLOW_THREADS;
    return results(rc);
} catch (...) {
    return refused();
}

// (cache, slots, bf16, device, stream) -> (k, v)
PyObject* kv_cache_read(PyObject*, PyObject* const* a, Py_ssize_t n) try {
    Args x{a};
    if (n != 5 || !THPVariable_Check(a[1])) return none();
    const auto* cache = (const capdec_kv_cache*)x.address(0);
    const at::Tensor& s = THPVariable_Unpack(a[1]);
    const int64_t bf16 = x.integer(2), device = x.integer(3), rows = s.numel();
    void* stream = x.address(4);
    const void* slots;
    if (!x.ok || rows >= (1ll << 31) || !vector(a[1], at::kInt, rows, device, &slots)) return none();
    const int64_t width = (int64_t)cache->heads * cache->dh;
    const at::TensorOptions like = s.options().dtype(bf16 ? at::kBFloat16 : at::kFloat);
    at::Tensor k = at::empty({rows, width}, like), v = at::empty({rows, width}, like);
    void *pk = k.data_ptr(), *pv = v.data_ptr();
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = lib.kv_read(cache, (const int*)slots, (int)rows, pk, (int)width, pv, (int)width, bf16 ? CAPDEC_BF16S : CAPDEC_F32, stream);
    Py_END_ALLOW_THREADS;
    return results(rc, k, v);
} catch (...) {
    return refused();
}

// (cache, q, page_table, kv_lens, Hq, cu_q or None, max_q, scale, device, stream) -> o
PyObject* attn_paged(PyObject*, PyObject* const* a, Py_ssize_t n) try {
    Args x{a};
    if (n != 10 || !THPVariable_Check(a[3])) return none();
    const auto* cache = (const capdec_kv_cache*)x.address(0);
    const int64_t Hq = x.integer(4), max_q = x.integer(6), device = x.integer(8), seqs = THPVariable_Unpack(a[3]).numel();
    const float scale = x.scale(7, cache->dh);
    void* stream = x.address(9);
    if (!x.ok || Hq <= 0 || Hq > (1 << 17) || Hq % cache->heads || max_q <= 0 || max_q >= (1ll << 31) || seqs <= 0 || seqs >= (1ll << 31) - 1)
        return none();
    const int64_t width = Hq * cache->dh;
    const at::Tensor* table = tensor(a[2], at::kInt, 2, device);
    const void *lens, *cu = nullptr;
    Matrix q;
    if (!table || !vector(a[3], at::kInt, seqs, device, &lens) || (a[5] != Py_None && !vector(a[5], at::kInt, seqs + 1, device, &cu)) ||
        !matrix(a[1], at::kBFloat16, cu ? 1 : seqs, width, device, &q) || q.rows >= (1ll << 31))
        return none();
    const int64_t cols = table->size(1), ld = seqs > 1 ? table->stride(0) : cols;
    if (table->size(0) != seqs || cols == 0 || cols >= (1ll << 31) || table->stride(1) != 1 || ld < cols || ld >= (1ll << 31)) return none();
    at::Tensor o = new_like(q, width, THPVariable_Unpack(a[1])), ws;
    const size_t need = lib.paged_workspace(cache, (int)seqs, (int)q.rows, (int)max_q, (int)Hq, (int)cols);
    if (need) ws = at::empty({(int64_t)need}, o.options().dtype(at::kByte));
    void *po = o.data_ptr(), *pw = need ? ws.data_ptr() : nullptr, *pt = table->data_ptr();
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = lib.paged(cache, q.at, q.ld, (const int*)cu, (const int*)lens, (const int*)pt, (int)ld, (int)cols, (int)seqs, (int)q.rows, (int)max_q,
                   (int)Hq, scale, po, (int)width, 1, nullptr, pw, need, stream);
    Py_END_ALLOW_THREADS;
    return results(rc, o);
} catch (...) {
    return refused();
}

// (target, draft or None, tokens, u_accept, u_sample, num_draft or None, pad, device, stream) -> (out, accepted)
PyObject* draft_verify(PyObject*, PyObject* const* a, Py_ssize_t n) try {
    Args x{a};
    if (n != 9) return none();
    const int64_t pad = x.integer(6), device = x.integer(7);
    void* stream = x.address(8);
    if (!x.ok) return none();
    const at::Tensor *target = tensor(a[0], at::kFloat, 3, device), *draft = nullptr, *tokens = tensor(a[2], at::kLong, 2, device),
                     *u = tensor(a[3], at::kFloat, 2, device);
    if (!target || !tokens || !u) return none();
    const int64_t seqs = target->size(0), d = target->size(1) - 1, V = target->size(2);
    if (seqs <= 0 || seqs >= (1ll << 31) || d < 1 || d > 64 || V < 2 || V >= (1ll << 30)) return none();
    auto block = [&](const at::Tensor& t, int64_t rows, int64_t* row) {  // [seqs, rows, V]
        *row = rows > 1 ? t.stride(1) : V;
        return t.size(0) == seqs && t.size(1) == rows && t.size(2) == V && t.stride(2) == 1 && *row >= V && t.stride(0) >= 0;
    };
    auto small = [&](const at::Tensor& t, int64_t* ld) {  // [seqs, d]
        *ld = seqs > 1 ? t.stride(0) : d;
        return t.size(0) == seqs && t.size(1) == d && (d == 1 || t.stride(1) == 1) && *ld >= d && *ld < (1ll << 31);
    };
    int64_t target_row, draft_row = 0, ldt, ldu;
    if (!block(*target, d + 1, &target_row) || !small(*tokens, &ldt) || !small(*u, &ldu)) return none();
    if (a[1] != Py_None && (!(draft = tensor(a[1], at::kFloat, 3, device)) || !block(*draft, d, &draft_row))) return none();
    const void *us, *num = nullptr;
    if (!vector(a[4], at::kFloat, seqs, device, &us) || (a[5] != Py_None && !vector(a[5], at::kInt, seqs, device, &num))) return none();
    at::Tensor out = at::empty({seqs, d + 1}, tokens->options()), accepted = at::empty({seqs}, tokens->options().dtype(at::kInt));
    const void *pt = target->data_ptr(), *pd = draft ? draft->data_ptr() : nullptr, *pk = tokens->data_ptr(), *pu = u->data_ptr();
    const int64_t target_seq = target->stride(0), draft_seq = draft ? draft->stride(0) : 0;
    void *po = out.data_ptr(), *pa = accepted.data_ptr();
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = lib.verify(pt, target_seq, target_row, pd, draft_seq, draft_row, (const int64_t*)pk, (int)ldt, (const int*)num, pu, (int)ldu, us, (int)seqs,
                    (int)d, (int)V, pad, (int64_t*)po, (int*)pa, stream);
    Py_END_ALLOW_THREADS;
    return results(rc, out, accepted);
} catch (...) {
    return refused();
}

// (addresses of the entry points, in the order of Entry)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    void* at[sizeof(Entry) / sizeof(void*)];
    Args x{a};
    for (size_t i = 0; i < sizeof(at) / sizeof(at[0]); ++i) at[i] = (Py_ssize_t)i < n ? x.address((int)i) : nullptr;
    if (!x.ok || n != (Py_ssize_t)(sizeof(at) / sizeof(at[0]))) {
        PyErr_SetString(PyExc_TypeError, "bind: one address for each entry point");
        return nullptr;
    }
    static_assert(sizeof(Entry) == sizeof(at), "an entry is an address");
    memcpy(&lib, at, sizeof(at));
    return none();
}

#define CAPDEC_METHOD(name) {#name, (PyCFunction)(void (*)())name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {CAPDEC_METHOD(bind), CAPDEC_METHOD(attn_packed_fwd), CAPDEC_METHOD(attn_packed_bwd), CAPDEC_METHOD(kv_cache_write),
                         CAPDEC_METHOD(kv_cache_read), CAPDEC_METHOD(attn_paged), CAPDEC_METHOD(draft_verify), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
