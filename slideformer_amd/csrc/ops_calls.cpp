// slideformer_amd: the host side of the model operators' smallest calls, as a
// CPython module (plain C++17 against torch's headers, no HIP).
//
// The embedding or the norm of one token is over in 3 us on the device; in Python
// its checks, its allocations and ctypes' argument conversion took 8 to 13 us.
// The functions here do the same checks on the tensors themselves, allocate the
// outputs and call the library's C-ABI through the addresses of the library
// that slideformer_amd._ops_lib has loaded.
//
// Each handles the calls that pass every check on the current device, and
// returns None for any other, before anything has happened: the caller then
// takes its own path, which raises the errors, or serves another stream or
// device.  Otherwise it returns the outputs, or the library's code where that is
// not zero.  Nothing is kept from one call for the next.

#include <Python.h>

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>

#include <cmath>
#include <cstdint>
#include <exception>

#include "../../include/model_ops.h"

namespace {

decltype(&la_embedding) p_embedding = nullptr;
decltype(&la_embedding_grad_workspace) p_embedding_grad_workspace = nullptr;
decltype(&la_embedding_grad) p_embedding_grad = nullptr;
decltype(&la_rms_norm) p_rms_norm = nullptr;
decltype(&la_rms_norm_grad_workspace) p_rms_norm_grad_workspace = nullptr;
decltype(&la_rms_norm_grad) p_rms_norm_grad = nullptr;
decltype(&la_qk_norm_rotary) p_rotary = nullptr;
decltype(&la_qk_norm_rotary_grad_workspace) p_rotary_grad_workspace = nullptr;
decltype(&la_qk_norm_rotary_grad) p_rotary_grad = nullptr;
decltype(&la_attention_workspace) p_attention_workspace = nullptr;
decltype(&la_attention) p_attention = nullptr;
decltype(&la_attention_grad_workspace) p_attention_grad_workspace = nullptr;
decltype(&la_attention_grad) p_attention_grad = nullptr;

int code_of(at::ScalarType t)
{
    switch (t) {
    case at::kFloat: return LA_F32;
    case at::kBFloat16: return LA_BF16;
    case at::kHalf: return LA_F16;
    case at::kInt: return LA_I32;
    case at::kLong: return LA_I64;
    case at::kChar: return LA_I8;
    case at::kFloat8_e4m3fn: return LA_F8E4M3;
    default: return -1;
    }
}

// A plain tensor or Parameter with memory of its own on HIP device `dev`; null otherwise.
const at::Tensor* plain(PyObject* o, int64_t dev)
{
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || t.layout() != at::kStrided || !t.is_cuda() || t.get_device() != dev || !t.has_storage())
        return nullptr;
    return &t;
}

// A matrix of floats in contiguous rows that do not overlap, `stride` elements apart.
struct Matrix {
    const at::Tensor* t = nullptr;
    int64_t rows = 0, hidden = 0, stride = 0;
    int code = -1;
    void* data() const { return t ? t->data_ptr() : nullptr; }
};

bool matrix(PyObject* o, int64_t dev, Matrix& m)
{
    m.t = plain(o, dev);
    if (!m.t || m.t->dim() != 2) return false;
    m.code = code_of(m.t->scalar_type());
    m.rows = m.t->size(0);
    m.hidden = m.t->size(1);
    m.stride = m.rows > 1 ? m.t->stride(0) : m.hidden;
    return m.code >= 0 && m.code <= LA_F16 && m.rows > 0 && m.hidden > 0 && (m.hidden == 1 || m.t->stride(1) == 1) &&
           m.stride >= m.hidden;
}

bool same_shape(const Matrix& a, const Matrix& b)
{
    return a.rows == b.rows && a.hidden == b.hidden && a.code == b.code;
}

// None (then m.t stays null), or a matrix of a's shape and type.
bool optional(PyObject* o, int64_t dev, const Matrix& a, Matrix& m)
{
    m.stride = a.hidden;
    return o == Py_None || (matrix(o, dev, m) && same_shape(a, m));
}

const at::Tensor* vector(PyObject* o, int64_t dev, int64_t size)
{
    const at::Tensor* t = plain(o, dev);
    return t && t->numel() == size && t->is_contiguous() ? t : nullptr;
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, int64_t dev)
{
    return at::empty(shape, at::TensorOptions().dtype(type).device(at::kCUDA, static_cast<c10::DeviceIndex>(dev)));
}

PyObject* none()
{
    Py_RETURN_NONE;
}

// The Python error of the exception in flight, torch's own types among them (what an
// allocation raises where memory runs out).
PyObject* failed()
{
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
}

PyObject* code(int rc) { return PyLong_FromLong(rc); }

PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }

// A tuple of tensors, or of objects passed on.
PyObject* tuple(std::initializer_list<PyObject*> items)
{
    PyObject* t = PyTuple_New(static_cast<Py_ssize_t>(items.size()));
    Py_ssize_t k = 0;
    for (PyObject* o : items) {
        if (t && o) PyTuple_SET_ITEM(t, k, o);
        else {
            Py_XDECREF(t);
            t = nullptr;
            Py_XDECREF(o);
        }
        ++k;
    }
    return t;
}

PyObject* again(PyObject* o)
{
    Py_INCREF(o);
    return o;
}

// embedding(tokens, weight, scale, device, stream)
PyObject* embedding(PyObject*, PyObject* const* a, Py_ssize_t count)
try {
    if (count != 5) return none();
    const int64_t dev = PyLong_AsLongLong(a[3]);
    Matrix w;
    const at::Tensor* tokens = plain(a[0], dev);
    if (!tokens || !matrix(a[1], dev, w) || !tokens->is_contiguous() || tokens->numel() == 0) return none();
    const int token = code_of(tokens->scalar_type());
    const double scale = PyFloat_AsDouble(a[2]);
    void* stream = PyLong_AsVoidPtr(a[4]);
    if (PyErr_Occurred() || (token != LA_I32 && token != LA_I64)) {
        PyErr_Clear();
        return none();
    }
    c10::SmallVector<int64_t, 5> shape(tokens->sizes().begin(), tokens->sizes().end());
    shape.push_back(w.hidden);
    const at::Tensor out = empty(shape, w.t->scalar_type(), dev);
    const void* from = tokens->data_ptr();
    const uint64_t n = tokens->numel();
    void *data = w.data(), *to = out.data_ptr();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = p_embedding(token, from, n, w.code, data, w.rows, w.hidden, w.stride, static_cast<float>(scale), to, w.hidden,
                     stream);
    Py_END_ALLOW_THREADS
    return rc ? code(rc) : wrap(out);
} catch (const std::exception&) {
    return failed();
}

// embedding_grad(tokens, grad_out, grad_weight, scale, padding_idx, accumulate, device, stream)
PyObject* embedding_grad(PyObject*, PyObject* const* a, Py_ssize_t count)
try {
    if (count != 8) return none();
    const int64_t dev = PyLong_AsLongLong(a[6]);
    Matrix g, w;
    if (!matrix(a[1], dev, g) || !matrix(a[2], dev, w) || g.hidden != w.hidden ||
        (w.code != g.code && w.code != LA_F32))
        return none();
    const at::Tensor* tokens = vector(a[0], dev, g.rows);
    if (!tokens) return none();
    const int token = code_of(tokens->scalar_type());
    const double scale = PyFloat_AsDouble(a[3]);
    const int64_t padding = PyLong_AsLongLong(a[4]);
    const int accumulate = PyObject_IsTrue(a[5]);
    void* stream = PyLong_AsVoidPtr(a[7]);
    if (PyErr_Occurred() || (token != LA_I32 && token != LA_I64)) {
        PyErr_Clear();
        return none();
    }
    const uint64_t bytes = p_embedding_grad_workspace(g.rows, w.rows, w.hidden);
    const at::Tensor work = empty({static_cast<int64_t>(bytes) + 1}, at::kByte, dev);
    void *from = tokens->data_ptr(), *grad = g.data(), *to = w.data(), *ws = work.data_ptr();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = p_embedding_grad(token, from, g.rows, g.code, grad, g.stride, w.code, to, w.rows, w.hidden, w.stride,
                          static_cast<float>(scale), padding, accumulate, ws, bytes, stream);
    Py_END_ALLOW_THREADS
    return rc ? code(rc) : again(a[2]);
} catch (const std::exception&) {
    return failed();
}

// rms_norm(x, weight, eps, residual, device, stream) and
// rms_norm_8bit(x, weight, eps, residual, float8, device, stream)
PyObject* norm(PyObject* const* a, bool eight, bool float8, PyObject* device, PyObject* on)
{
    const int64_t dev = PyLong_AsLongLong(device);
    Matrix x, r;
    if (!matrix(a[0], dev, x) || !optional(a[3], dev, x, r)) return none();
    const at::Tensor* weight = vector(a[1], dev, x.hidden);
    const double eps = PyFloat_AsDouble(a[2]);
    void* stream = PyLong_AsVoidPtr(on);
    if (PyErr_Occurred() || !weight || weight->scalar_type() != x.t->scalar_type()) {
        PyErr_Clear();
        return none();
    }
    const at::ScalarType type = x.t->scalar_type();
    const at::Tensor out =
        empty({x.rows, x.hidden}, !eight ? type : float8 ? at::kFloat8_e4m3fn : at::kChar, dev);
    const at::Tensor per_row = empty({x.rows}, at::kFloat, dev);       // rstd, or the scales
    at::Tensor summed;
    if (r.t) summed = empty({x.rows, x.hidden}, type, dev);
    float* rows = static_cast<float*>(per_row.data_ptr());
    const int out_code = code_of(out.scalar_type());
    void *from = x.data(), *res = r.data(), *w = weight->data_ptr(), *sum = r.t ? summed.data_ptr() : nullptr,
         *to = out.data_ptr();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = p_rms_norm(x.code, from, x.stride, res, r.stride, w, x.rows, x.hidden, static_cast<float>(eps), sum, x.hidden,
                    out_code, to, x.hidden, eight ? rows : nullptr, eight ? nullptr : rows, stream);
    Py_END_ALLOW_THREADS
    if (rc) return code(rc);
    PyObject* z = r.t ? wrap(summed) : again(a[0]);
    return eight ? tuple({wrap(out), wrap(per_row), z}) : tuple({wrap(out), z, wrap(per_row)});
}

PyObject* rms_norm(PyObject*, PyObject* const* a, Py_ssize_t count)
try {
    return count == 6 ? norm(a, false, false, a[4], a[5]) : none();
} catch (const std::exception&) {
    return failed();
}

PyObject* rms_norm_8bit(PyObject*, PyObject* const* a, Py_ssize_t count)
try {
    return count == 7 ? norm(a, true, PyObject_IsTrue(a[4]), a[5], a[6]) : none();
} catch (const std::exception&) {
    return failed();
}

// rms_norm_grad(grad_out, summed, rstd, weight, grad_summed, grad_weight, accumulate, device, stream)
PyObject* rms_norm_grad(PyObject*, PyObject* const* a, Py_ssize_t count)
try {
    if (count != 9) return none();
    const int64_t dev = PyLong_AsLongLong(a[7]);
    Matrix g, z, past;
    if (!matrix(a[0], dev, g) || !matrix(a[1], dev, z) || !same_shape(g, z) || !optional(a[4], dev, g, past))
        return none();
    const at::Tensor* rstd = vector(a[2], dev, g.rows);
    const at::Tensor* weight = vector(a[3], dev, g.hidden);
    const bool fresh = a[5] == Py_None;
    const at::Tensor* given = fresh ? nullptr : vector(a[5], dev, g.hidden);
    const int accumulate = PyObject_IsTrue(a[6]);
    void* stream = PyLong_AsVoidPtr(a[8]);
    const at::ScalarType type = g.t->scalar_type();
    if (PyErr_Occurred() || !rstd || rstd->scalar_type() != at::kFloat || !weight || weight->scalar_type() != type ||
        (fresh ? accumulate != 0
               : !given || (given->scalar_type() != type && given->scalar_type() != at::kFloat))) {
        PyErr_Clear();
        return none();
    }
    const at::Tensor grad_x = empty({g.rows, g.hidden}, type, dev);
    const at::Tensor grad_weight = fresh ? empty({g.hidden}, type, dev) : *given;
    const uint64_t bytes = p_rms_norm_grad_workspace(g.rows, g.hidden);
    const at::Tensor work = empty({static_cast<int64_t>(bytes) + 1}, at::kByte, dev);
    const int w_code = code_of(grad_weight.scalar_type());
    const float* r = static_cast<const float*>(rstd->data_ptr());
    void *go = g.data(), *sum = z.data(), *w = weight->data_ptr(), *through = past.data(), *gx = grad_x.data_ptr(),
         *gw = grad_weight.data_ptr(), *ws = work.data_ptr();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = p_rms_norm_grad(g.code, go, g.stride, sum, z.stride, r, w, through, past.stride, g.rows, g.hidden, gx,
                         g.hidden, w_code, gw, accumulate, ws, bytes, stream);
    Py_END_ALLOW_THREADS
    if (rc) return code(rc);
    return tuple({wrap(grad_x), fresh ? wrap(grad_weight) : again(a[5])});
} catch (const std::exception&) {
    return failed();
}

// Heads [.., heads, dim] of `dims` dimensions with contiguous elements, none of them empty.
const at::Tensor* heads(PyObject* o, int64_t dev, int64_t dims, la_heads_t& h)
{
    const at::Tensor* t = plain(o, dev);
    if (!t || t->dim() != dims || t->numel() == 0 || (t->size(-1) > 1 && t->stride(-1) != 1)) return nullptr;
    h = {t->data_ptr(), dims == 4 ? static_cast<uint64_t>(t->stride(0)) : 0, static_cast<uint64_t>(t->stride(-3)),
         static_cast<uint64_t>(t->stride(-2))};
    return t;
}

const at::Tensor* heads_like(PyObject* o, int64_t dev, const at::Tensor& like, la_heads_t& h)
{
    const at::Tensor* t = heads(o, dev, like.dim(), h);
    return t && t->sizes() == like.sizes() && t->scalar_type() == like.scalar_type() ? t : nullptr;
}

la_heads_t fresh_heads(const at::Tensor& t)
{
    return {t.data_ptr(), t.dim() == 4 ? static_cast<uint64_t>(t.stride(0)) : 0, static_cast<uint64_t>(t.stride(-3)),
            static_cast<uint64_t>(t.stride(-2))};
}

// None, or a vector of `size` indices.
bool indices(PyObject* o, int64_t dev, int64_t size, const at::Tensor*& t)
{
    t = nullptr;
    if (o == Py_None) return true;
    t = vector(o, dev, size);
    return t && (t->scalar_type() == at::kInt || t->scalar_type() == at::kLong);
}

void* data_of(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }

// What both calls of the rotation check alike: tables, weights, positions; `of_q` and `of_k` have their sizes.
bool rotary_call(PyObject* const* a, int64_t dev, const at::Tensor& of_q, const at::Tensor& of_k, la_rotary_t& c)
{
    const at::Tensor *cos = plain(a[0], dev), *sin = plain(a[1], dev), *at = nullptr;
    c.dtype = code_of(of_q.scalar_type());
    c.n = of_q.size(0);
    c.heads = of_q.size(1);
    c.kv_heads = of_k.size(1);
    c.dim = of_q.size(2);
    if (c.dtype < 0 || c.dtype > LA_F16 || of_k.scalar_type() != of_q.scalar_type() || of_k.size(0) != of_q.size(0) ||
        of_k.size(2) != of_q.size(2) || c.dim > 256 || !cos || !sin || cos->dim() != 2 || sin->sizes() != cos->sizes() ||
        cos->scalar_type() != at::kFloat || sin->scalar_type() != at::kFloat || !cos->is_contiguous() ||
        !sin->is_contiguous() || 2 * cos->size(1) > of_q.size(2) || cos->numel() == 0 || !indices(a[4], dev, of_q.size(0), at))
        return false;
    const void** weights[] = {&c.q_weight, &c.k_weight};
    for (int k = 0; k < 2; ++k) {
        if (a[2 + k] == Py_None) continue;
        const at::Tensor* w = vector(a[2 + k], dev, of_q.size(2));
        if (!w || w->scalar_type() != of_q.scalar_type()) return false;
        *weights[k] = w->data_ptr();
    }
    c.cos = static_cast<const float*>(cos->data_ptr());
    c.sin = static_cast<const float*>(sin->data_ptr());
    c.rotated = 2 * cos->size(1);
    c.positions = cos->size(0);
    c.at = data_of(at);
    if (at) c.at_dtype = code_of(at->scalar_type());
    c.eps = static_cast<float>(PyFloat_AsDouble(a[5]));
    c.interleaved = PyObject_IsTrue(a[6]);
    return true;
}

// qk_norm_rotary(q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved, device, stream)
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t count)
try {
    if (count != 11) return none();
    const int64_t dev = PyLong_AsLongLong(a[9]);
    void* stream = PyLong_AsVoidPtr(a[10]);
    la_rotary_t c{};
    const at::Tensor *q = heads(a[0], dev, 3, c.q), *k = heads(a[1], dev, 3, c.k);
    if (!q || !k || !rotary_call(a + 2, dev, *q, *k, c) || PyErr_Occurred()) {
        PyErr_Clear();
        return none();
    }
    const at::Tensor q_out = empty(q->sizes(), q->scalar_type(), dev), k_out = empty(k->sizes(), k->scalar_type(), dev);
    c.q_out = fresh_heads(q_out);
    c.k_out = fresh_heads(k_out);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = p_rotary(&c, stream);
    Py_END_ALLOW_THREADS
    return rc ? code(rc) : tuple({wrap(q_out), wrap(k_out)});
} catch (const std::exception&) {
    return failed();
}

// qk_norm_rotary_grad(grad_q, grad_k, q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved, device, stream):
// the call whose results are all new, of heads that are both normed or both not
PyObject* rotary_grad(PyObject*, PyObject* const* a, Py_ssize_t count)
try {
    if (count != 13) return none();
    const int64_t dev = PyLong_AsLongLong(a[11]);
    void* stream = PyLong_AsVoidPtr(a[12]);
    la_rotary_t c{};
    const at::Tensor *gq = heads(a[0], dev, 3, c.grad_q), *gk = heads(a[1], dev, 3, c.grad_k);
    if (!gq || !gk || !rotary_call(a + 4, dev, *gq, *gk, c) || PyErr_Occurred() || !c.q_weight != !c.k_weight ||
        (c.q_weight && (!heads_like(a[2], dev, *gq, c.q) || !heads_like(a[3], dev, *gk, c.k)))) {
        PyErr_Clear();
        return none();
    }
    const at::ScalarType type = gq->scalar_type();
    const at::Tensor q_out = empty(gq->sizes(), type, dev), k_out = empty(gk->sizes(), type, dev);
    c.q_out = fresh_heads(q_out);
    c.k_out = fresh_heads(k_out);
    at::Tensor wq, wk, work;
    const uint64_t bytes = p_rotary_grad_workspace(&c);
    c.weight_grad_dtype = c.dtype;
    if (c.q_weight) {
        wq = empty({gq->size(2)}, type, dev);
        wk = empty({gq->size(2)}, type, dev);
        work = empty({static_cast<int64_t>(bytes)}, at::kByte, dev);
        c.grad_q_weight = wq.data_ptr();
        c.grad_k_weight = wk.data_ptr();
    }
    void* ws = c.q_weight ? work.data_ptr() : nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = p_rotary_grad(&c, ws, bytes, stream);
    Py_END_ALLOW_THREADS
    if (rc) return code(rc);
    return tuple({wrap(q_out), wrap(k_out), c.q_weight ? wrap(wq) : again(Py_None), c.q_weight ? wrap(wk) : again(Py_None)});
} catch (const std::exception&) {
    return failed();
}

// What both calls of attention check alike: (q, k, v), and from `a` on (causal, window or 0, scale or None, starts,
// key_starts, lengths, key_lengths).
bool attention_call(PyObject* const* qkv, PyObject* const* a, int64_t dev, la_attention_t& c, const at::Tensor* (&t)[3])
{
    const at::Tensor* of_q = plain(qkv[0], dev);
    if (!of_q || (of_q->dim() != 3 && of_q->dim() != 4)) return false;
    const int64_t dims = of_q->dim();
    t[0] = heads(qkv[0], dev, dims, c.q);
    t[1] = heads(qkv[1], dev, dims, c.k);
    if (!t[0] || !t[1]) return false;
    t[2] = heads_like(qkv[2], dev, *t[1], c.v);
    const at::Tensor &q = *t[0], &k = *t[1];
    if (!t[2] || k.scalar_type() != q.scalar_type()) return false;
    c.dtype = code_of(q.scalar_type());
    c.rows = q.size(-3);
    c.heads = q.size(-2);
    c.dim = q.size(-1);
    c.key_rows = k.size(-3);
    c.kv_heads = k.size(-2);
    c.causal = PyObject_IsTrue(a[0]);
    c.window = PyLong_AsUnsignedLongLong(a[1]);
    c.scale = static_cast<float>(a[2] == Py_None ? 1.0 / std::sqrt(static_cast<double>(c.dim)) : PyFloat_AsDouble(a[2]));
    if ((c.dtype != LA_BF16 && c.dtype != LA_F16) || k.size(-1) != q.size(-1) || c.dim > 128 || c.heads % c.kv_heads ||
        (c.window && !c.causal) || !(c.scale > 0.0f) || !std::isfinite(c.scale))
        return false;
    const at::Tensor *starts, *key_starts, *lengths, *key_lengths, *first;
    if (dims == 3) {
        const at::Tensor* given = plain(a[3], dev);
        if (!given || given->numel() < 2 || a[5] != Py_None || a[6] != Py_None ||
            !indices(a[3], dev, given->numel(), starts) || !indices(a[4], dev, given->numel(), key_starts) ||
            (!key_starts && c.rows != c.key_rows) || (key_starts && key_starts->scalar_type() != starts->scalar_type()))
            return false;
        c.batch = given->numel() - 1;
        c.starts = data_of(starts);
        c.key_starts = data_of(key_starts);
        first = starts;
    } else {
        if (a[3] != Py_None || a[4] != Py_None || k.size(0) != q.size(0) || !indices(a[5], dev, q.size(0), lengths) ||
            !indices(a[6], dev, q.size(0), key_lengths))
            return false;
        if (lengths && !key_lengths) {
            if (c.rows != c.key_rows) return false;
            key_lengths = lengths;
        }
        if (lengths && lengths->scalar_type() != key_lengths->scalar_type()) return false;
        c.batch = q.size(0);
        c.lengths = data_of(lengths);
        c.key_lengths = data_of(key_lengths);
        first = key_lengths;
    }
    if (first) c.index_dtype = code_of(first->scalar_type());
    return true;
}

// The values of one fp32 for each head.
bool row_values(PyObject* o, int64_t dev, const at::Tensor& q, la_heads_t& h)
{
    const at::Tensor* t = plain(o, dev);
    if (!t || t->dim() != q.dim() - 1 || t->sizes() != q.sizes().slice(0, q.dim() - 1) || t->scalar_type() != at::kFloat)
        return false;
    h = {t->data_ptr(), t->dim() == 3 ? static_cast<uint64_t>(t->stride(0)) : 0, static_cast<uint64_t>(t->stride(-2)),
         static_cast<uint64_t>(t->stride(-1))};
    return true;
}

// attention(q, k, v, causal, window, scale, starts, key_starts, lengths, key_lengths, device, stream)
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t count)
try {
    if (count != 12) return none();
    const int64_t dev = PyLong_AsLongLong(a[10]);
    void* stream = PyLong_AsVoidPtr(a[11]);
    la_attention_t c{};
    const at::Tensor* t[3];
    if (!attention_call(a, a + 3, dev, c, t) || PyErr_Occurred()) {
        PyErr_Clear();
        return none();
    }
    const at::Tensor& q = *t[0];
    const at::Tensor out = empty(q.sizes(), q.scalar_type(), dev);
    const at::Tensor lse = empty(q.sizes().slice(0, q.dim() - 1), at::kFloat, dev);
    c.out = fresh_heads(out);
    c.lse = {lse.data_ptr(), q.dim() == 4 ? c.rows * c.heads : 0, c.heads, 1};
    const uint64_t bytes = p_attention_workspace(&c);
    at::Tensor work;
    if (bytes) work = empty({static_cast<int64_t>(bytes)}, at::kByte, dev);
    void* ws = bytes ? work.data_ptr() : nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = p_attention(&c, ws, bytes, stream);
    Py_END_ALLOW_THREADS
    return rc ? code(rc) : tuple({wrap(out), wrap(lse)});
} catch (const std::exception&) {
    return failed();
}

// attention_grad(grad_out, q, k, v, out, lse, causal, window, scale, starts, key_starts, lengths, key_lengths, device,
// stream): the call whose results are new
PyObject* attention_grad(PyObject*, PyObject* const* a, Py_ssize_t count)
try {
    if (count != 15) return none();
    const int64_t dev = PyLong_AsLongLong(a[13]);
    void* stream = PyLong_AsVoidPtr(a[14]);
    la_attention_t c{};
    const at::Tensor* t[3];
    if (!attention_call(a + 1, a + 6, dev, c, t) || PyErr_Occurred() || !heads_like(a[0], dev, *t[0], c.grad_out) ||
        !heads_like(a[4], dev, *t[0], c.out) || !row_values(a[5], dev, *t[0], c.lse)) {
        PyErr_Clear();
        return none();
    }
    at::Tensor grads[3];
    for (int k = 0; k < 3; ++k) grads[k] = empty(t[k]->sizes(), t[k]->scalar_type(), dev);
    c.grad_q = fresh_heads(grads[0]);
    c.grad_k = fresh_heads(grads[1]);
    c.grad_v = fresh_heads(grads[2]);
    const uint64_t bytes = p_attention_grad_workspace(&c);
    const at::Tensor work = empty({static_cast<int64_t>(bytes) + 1}, at::kByte, dev);
    void* ws = work.data_ptr();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = p_attention_grad(&c, ws, bytes, stream);
    Py_END_ALLOW_THREADS
    return rc ? code(rc) : tuple({wrap(grads[0]), wrap(grads[1]), wrap(grads[2])});
} catch (const std::exception&) {
    return failed();
}

// bind(addresses of the functions above, in the order of their pointers)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t count)
{
    constexpr Py_ssize_t kCount = 13;
    if (count != kCount) {
        PyErr_SetString(PyExc_TypeError, "bind takes thirteen addresses");
        return nullptr;
    }
    void* at[kCount];
    for (Py_ssize_t k = 0; k < kCount; ++k) at[k] = PyLong_AsVoidPtr(a[k]);
    if (PyErr_Occurred()) return nullptr;
    p_embedding = reinterpret_cast<decltype(p_embedding)>(at[0]);
    p_embedding_grad_workspace = reinterpret_cast<decltype(p_embedding_grad_workspace)>(at[1]);
    p_embedding_grad = reinterpret_cast<decltype(p_embedding_grad)>(at[2]);
    p_rms_norm = reinterpret_cast<decltype(p_rms_norm)>(at[3]);
    p_rms_norm_grad_workspace = reinterpret_cast<decltype(p_rms_norm_grad_workspace)>(at[4]);
    p_rms_norm_grad = reinterpret_cast<decltype(p_rms_norm_grad)>(at[5]);
    p_rotary = reinterpret_cast<decltype(p_rotary)>(at[6]);
    p_rotary_grad_workspace = reinterpret_cast<decltype(p_rotary_grad_workspace)>(at[7]);
    p_rotary_grad = reinterpret_cast<decltype(p_rotary_grad)>(at[8]);
    p_attention_workspace = reinterpret_cast<decltype(p_attention_workspace)>(at[9]);
    p_attention = reinterpret_cast<decltype(p_attention)>(at[10]);
    p_attention_grad_workspace = reinterpret_cast<decltype(p_attention_grad_workspace)>(at[11]);
    p_attention_grad = reinterpret_cast<decltype(p_attention_grad)>(at[12]);
    Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL

PyMethodDef methods[] = {
    {"bind", FAST(bind), nullptr},
    {"embedding", FAST(embedding), nullptr},
    {"embedding_grad", FAST(embedding_grad), nullptr},
    {"rms_norm", FAST(rms_norm), nullptr},
    {"rms_norm_8bit", FAST(rms_norm_8bit), nullptr},
    {"rms_norm_grad", FAST(rms_norm_grad), nullptr},
    {"qk_norm_rotary", FAST(rotary), nullptr},
    {"qk_norm_rotary_grad", FAST(rotary_grad), nullptr},
    {"attention", FAST(attention), nullptr},
    {"attention_grad", FAST(attention_grad), nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__ops_calls(void) { return PyModule_Create(&module); }
