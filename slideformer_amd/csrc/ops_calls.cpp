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

// bind(addresses of the six functions above, in the order of their pointers)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t count)
{
    if (count != 6) {
        PyErr_SetString(PyExc_TypeError, "bind takes six addresses");
        return nullptr;
    }
    void* at[6];
    for (int k = 0; k < 6; ++k) at[k] = PyLong_AsVoidPtr(a[k]);
    if (PyErr_Occurred()) return nullptr;
    p_embedding = reinterpret_cast<decltype(p_embedding)>(at[0]);
    p_embedding_grad_workspace = reinterpret_cast<decltype(p_embedding_grad_workspace)>(at[1]);
    p_embedding_grad = reinterpret_cast<decltype(p_embedding_grad)>(at[2]);
    p_rms_norm = reinterpret_cast<decltype(p_rms_norm)>(at[3]);
    p_rms_norm_grad_workspace = reinterpret_cast<decltype(p_rms_norm_grad_workspace)>(at[4]);
    p_rms_norm_grad = reinterpret_cast<decltype(p_rms_norm_grad)>(at[5]);
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
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__ops_calls(void) { return PyModule_Create(&module); }
