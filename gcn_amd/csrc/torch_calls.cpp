// The host side of the scoring and optimiser calls on torch tensors: checks, results, the call of the C ABI.  A small
// call of these is bound by it - five tensors looked at and four made through Python take longer than the kernels.
//
// Every function takes the stream and the device it belongs to, and gives None where an argument is not what it
// has to be (ops.py then says what), the error code where the C ABI gives one, else its result.  The C ABI is
// called through the addresses that bind() gets: the library is loaded once, by lib.py.
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

#include "../../include/ccnn.h"

namespace {

decltype(&ccnn_log_probs_workspace_bytes) log_probs_bytes_fn;
decltype(&ccnn_log_probs) log_probs_fn;
decltype(&ccnn_log_probs_grad) log_probs_grad_fn;
decltype(&ccnn_grad_norm_workspace_bytes) grad_norm_bytes_fn;
decltype(&ccnn_grad_norm) grad_norm_fn;
decltype(&ccnn_adamw_step) adamw_step_fn;
decltype(&ccnn_adamw_moments) adamw_moments_fn;

int type_of(const at::Tensor &t)
{
    switch (t.scalar_type()) {
    case at::kFloat: return CCNN_TYPE_F32;
    case at::kDouble: return CCNN_TYPE_F64;
    case at::kBFloat16: return CCNN_TYPE_BF16;
    case at::kHalf: return CCNN_TYPE_F16;
    default: return 0;
    }
}

// The tensor behind a Python object if it is one, with memory on that GPU.
const at::Tensor *tensor(PyObject *o, long device)
{
    if (!THPVariable_Check(o)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    return t.is_cuda() && t.layout() == at::kStrided && t.get_device() == device ? &t : nullptr;
}

// The same for a contiguous one of n elements of a type; none stays none.
bool plain(PyObject *o, long device, at::ScalarType type, long n, void **at)
{
    *at = nullptr;
    if (o == Py_None) return true;
    const at::Tensor *t = tensor(o, device);
    if (!t || t->scalar_type() != type || t->numel() != n || !t->is_contiguous()) return false;
    *at = t->data_ptr();
    return true;
}

// A matrix whose rows are contiguous and do not overlap, and the elements from row to row.
bool rows_of(const at::Tensor *t, long *rows, long *classes, long *stride)
{
    if (!t || !type_of(*t) || t->dim() != 2 || t->size(1) < 1 || t->size(1) > CCNN_MAX_LOGITS) return false;
    *rows = t->size(0), *classes = t->size(1);
    if (*classes > 1 && t->stride(1) != 1) return false;
    *stride = *rows > 1 ? t->stride(0) : *classes;
    return *stride >= *classes;
}

// Bytes of a target, 0 if they are not one contiguous row of whole numbers.
int targets_of(const at::Tensor *t, long rows)
{
    if (!t || t->dim() != 1 || t->size(0) != rows || !t->is_contiguous()) return 0;
    return t->scalar_type() == at::kInt ? 4 : t->scalar_type() == at::kLong ? 8 : 0;
}

void *address(PyObject *o) { return PyLong_AsVoidPtr(o); }

PyObject *none() { Py_RETURN_NONE; }

template <typename F>
int unlocked(F call)
{
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = call();
    Py_END_ALLOW_THREADS return rc;
}

bool count_is(Py_ssize_t n, Py_ssize_t want)
{
    if (n != want) PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", want, n);
    return n == want;
}

// bind(seven addresses, in the order of their names above)
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    if (!count_is(n, 7)) return nullptr;
    log_probs_bytes_fn = (decltype(log_probs_bytes_fn))address(a[0]);
    log_probs_fn = (decltype(log_probs_fn))address(a[1]);
    log_probs_grad_fn = (decltype(log_probs_grad_fn))address(a[2]);
    grad_norm_bytes_fn = (decltype(grad_norm_bytes_fn))address(a[3]);
    grad_norm_fn = (decltype(grad_norm_fn))address(a[4]);
    adamw_step_fn = (decltype(adamw_step_fn))address(a[5]);
    adamw_moments_fn = (decltype(adamw_moments_fn))address(a[6]);
    return PyErr_Occurred() ? nullptr : none();
}

// log_probs(stream, device, logits, targets, top, want_entropy) -> (logp, entropy, top_logp, top_index, stats)
PyObject *log_probs(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    if (!count_is(n, 6)) return nullptr;
    void *stream = address(a[0]);
    const long device = PyLong_AsLong(a[1]), top = PyLong_AsLong(a[4]);
    const bool want_entropy = a[5] == Py_True;
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor *x = tensor(a[2], device), *y = tensor(a[3], device);
    long rows, classes, stride;
    if (!rows_of(x, &rows, &classes, &stride)) return none();
    const int target_bytes = targets_of(y, rows), type = type_of(*x);
    if (!target_bytes || top < 0 || top > CCNN_MAX_TOP || top > classes) return none();
    const auto wide = at::TensorOptions().device(x->device()).dtype(type == CCNN_TYPE_F64 ? at::kDouble : at::kFloat);
    const at::Tensor stats = at::empty({4, rows}, wide);
    at::Tensor top_logp, top_index, ws;
    if (top) {
        top_logp = at::empty({rows, top}, wide);
        top_index = at::empty({rows, top}, wide.dtype(at::kInt));
    }
    if (rows) {
        const size_t bytes = log_probs_bytes_fn(rows, (int)classes, (int)top, type);
        if (bytes) ws = at::empty({(long)bytes}, wide.dtype(at::kByte));
        const int rc = unlocked([&] {
            return log_probs_fn(x->const_data_ptr(), type, rows, (int)classes, stride, y->const_data_ptr(), target_bytes, (int)top,
                                want_entropy, stats.data_ptr(), top ? top_logp.data_ptr() : nullptr,
                                top ? top_index.data_ptr<int>() : nullptr, bytes ? ws.data_ptr() : nullptr, bytes, stream);
        });
        if (rc) return PyLong_FromLong(rc);
    }
    PyObject *out = PyTuple_New(5);
    if (!out) return nullptr;
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(stats.select(0, 0)));
    PyTuple_SET_ITEM(out, 1, want_entropy ? THPVariable_Wrap(stats.select(0, 1)) : none());
    PyTuple_SET_ITEM(out, 2, top ? THPVariable_Wrap(top_logp) : none());
    PyTuple_SET_ITEM(out, 3, top ? THPVariable_Wrap(top_index) : none());
    PyTuple_SET_ITEM(out, 4, THPVariable_Wrap(stats));
    return out;
    END_HANDLE_TH_ERRORS
}

// log_probs_grad(stream, device, logits, targets, stats, entropy, d_logp, d_entropy, out) -> out
PyObject *log_probs_grad(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    if (!count_is(n, 9)) return nullptr;
    void *stream = address(a[0]);
    const long device = PyLong_AsLong(a[1]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor *x = tensor(a[2], device), *y = tensor(a[3], device);
    long rows, classes, stride, out_rows, out_classes, out_stride;
    if (!rows_of(x, &rows, &classes, &stride)) return none();
    const int target_bytes = targets_of(y, rows), type = type_of(*x);
    const auto wide = type == CCNN_TYPE_F64 ? at::kDouble : at::kFloat;
    void *stats, *d_logp, *d_entropy;
    if (!target_bytes || !plain(a[4], device, wide, 4 * rows, &stats) || a[4] == Py_None
        || !plain(a[6], device, wide, rows, &d_logp) || !plain(a[7], device, wide, rows, &d_entropy))
        return none();
    if ((a[6] == Py_None && a[7] == Py_None) || (a[7] != Py_None && a[5] == Py_None)) return none();
    at::Tensor out;
    if (a[8] == Py_None) {
        out = at::empty({rows, classes}, at::TensorOptions().device(x->device()).dtype(x->scalar_type()));
        out_stride = classes;
    } else {
        const at::Tensor *o = tensor(a[8], device);
        if (!rows_of(o, &out_rows, &out_classes, &out_stride) || type_of(*o) != type || out_rows != rows || out_classes != classes)
            return none();
        const long size = x->element_size();
        const char *p = (const char *)x->const_data_ptr(), *q = (const char *)o->const_data_ptr();
        if (rows && !(p == q && stride == out_stride) && p < q + ((rows - 1) * out_stride + classes) * size
            && q < p + ((rows - 1) * stride + classes) * size)
            return none();
        out = *o;
    }
    if (rows) {
        const int rc = unlocked([&] {
            return log_probs_grad_fn(x->const_data_ptr(), type, rows, (int)classes, stride, y->const_data_ptr(), target_bytes, stats,
                                     d_logp, d_entropy, out.data_ptr(), out_stride, stream);
        });
        if (rc) return PyLong_FromLong(rc);
    }
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

struct List {
    std::vector<const void *> at;
    std::vector<long> n;
    std::vector<int> types;
};

// The contiguous tensors of a Python list.
bool list_of(PyObject *o, long device, List *l)
{
    if (!PyList_Check(o)) return false;
    const Py_ssize_t count = PyList_GET_SIZE(o);
    l->at.resize(count);
    l->n.resize(count);
    l->types.resize(count);
    for (Py_ssize_t i = 0; i < count; i++) {
        const at::Tensor *t = tensor(PyList_GET_ITEM(o, i), device);
        if (!t || !(l->types[i] = type_of(*t)) || !t->is_contiguous()) return false;
        l->at[i] = t->const_data_ptr();
        l->n[i] = t->numel();
    }
    return count > 0;
}

// grad_norm(stream, device, grads, max_norm) -> [2]
PyObject *grad_norm(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    if (!count_is(n, 4)) return nullptr;
    void *stream = address(a[0]);
    const long device = PyLong_AsLong(a[1]);
    const double max_norm = PyFloat_AsDouble(a[3]);
    if (PyErr_Occurred()) return nullptr;
    List l;
    if (!list_of(a[2], device, &l) || !(max_norm > 0)) return none();
    const int count = (int)l.n.size();
    const auto on = at::TensorOptions().device(at::Device(at::kCUDA, (c10::DeviceIndex)device));
    const at::Tensor out = at::empty({2}, on.dtype(at::kDouble));
    at::Tensor ws;
    const size_t bytes = grad_norm_bytes_fn(l.n.data(), count);
    if (bytes) ws = at::empty({(long)bytes}, on.dtype(at::kByte));
    const int rc = unlocked([&] {
        return grad_norm_fn(l.at.data(), l.n.data(), l.types.data(), count, max_norm, (double *)out.data_ptr(),
                            bytes ? ws.data_ptr() : nullptr, bytes, stream);
    });
    return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// The bytes of an object that has them (a ctypes array), none of any other.
struct Bytes {
    Py_buffer view = {};
    explicit Bytes(PyObject *o)
    {
        if (PyObject_CheckBuffer(o) && PyObject_GetBuffer(o, &view, PyBUF_SIMPLE)) PyErr_Clear(), view = {};
    }
    ~Bytes() { PyBuffer_Release(&view); }
    Bytes(const Bytes &) = delete;
};

// adamw_step(stream, device, params, grads, table, bits, m, v, m_scale, v_scale, master, clock, lr, beta1, beta2, eps, clip)
// -> 0.  table: an array of ccnn_adamw_tensor_t, one for each parameter, which is still what it says, with their places
// one after the other; the state's tensors hold what it counts.
PyObject *adamw_step(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    if (!count_is(n, 17)) return nullptr;
    void *stream = address(a[0]);
    const long device = PyLong_AsLong(a[1]);
    const long bits = PyLong_AsLong(a[5]);
    const double beta1 = PyFloat_AsDouble(a[13]), beta2 = PyFloat_AsDouble(a[14]), eps = PyFloat_AsDouble(a[15]);
    if (PyErr_Occurred()) return nullptr;
    const Bytes held(a[4]);
    const auto *table = (const ccnn_adamw_tensor_t *)held.view.buf;
    List g;
    if (!PyList_Check(a[2]) || !list_of(a[3], device, &g) || (Py_ssize_t)g.n.size() != PyList_GET_SIZE(a[2])) return none();
    const int count = (int)g.n.size();
    if (held.view.len != (Py_ssize_t)(count * sizeof *table)) return none();
    long elements = 0, blocks = 0;
    bool any_half = false;
    for (int i = 0; i < count; i++) {
        const at::Tensor *p = tensor(PyList_GET_ITEM(a[2], i), device);
        const ccnn_adamw_tensor_t &t = table[i];
        const bool half = t.type == CCNN_TYPE_BF16 || t.type == CCNN_TYPE_F16;
        if (!p || p->const_data_ptr() != t.param || p->numel() != t.n || type_of(*p) != t.type) return none();
        if (g.n[i] != t.n || (g.types[i] != t.type && !(half && g.types[i] == CCNN_TYPE_F32))) return none();
        elements += t.n;
        blocks += (t.n + CCNN_MOMENT_BLOCK - 1) / CCNN_MOMENT_BLOCK;
        any_half |= half;
    }
    const bool coded = bits == 8;
    const auto moments = coded ? at::kByte : table[0].type == CCNN_TYPE_F64 ? at::kDouble : at::kFloat;
    const long held_moments = coded ? blocks * CCNN_MOMENT_BLOCK : elements;
    void *state[6];
    if (!plain(a[6], device, moments, held_moments, &state[0]) || !plain(a[7], device, moments, held_moments, &state[1])
        || !plain(a[8], device, at::kFloat, blocks, &state[2]) || !plain(a[9], device, at::kFloat, blocks, &state[3])
        || !plain(a[10], device, at::kFloat, elements, &state[4]) || !plain(a[11], device, at::kDouble, CCNN_ADAMW_CLOCK, &state[5])
        || a[6] == Py_None || a[7] == Py_None || a[11] == Py_None || (a[8] == Py_None) == coded || (a[9] == Py_None) == coded
        || (a[10] == Py_None) == any_half)
        return none();
    double lr = 0;
    void *lr_device = nullptr, *clip;
    if (THPVariable_Check(a[12])) {
        if (!plain(a[12], device, at::kDouble, 1, &lr_device)) return none();
    } else {
        lr = PyFloat_AsDouble(a[12]);
        if (PyErr_Occurred()) return nullptr;
    }
    if (!plain(a[16], device, at::kDouble, 2, &clip)) return none();
    const int rc = unlocked([&] {
        return adamw_step_fn(table, g.at.data(), g.types.data(), count, (int)bits, state[0], state[1], (float *)state[2],
                             (float *)state[3], (float *)state[4], (double *)state[5], lr, (const double *)lr_device, beta1, beta2,
                             eps, (const double *)clip, stream);
    });
    return PyLong_FromLong(rc);
    END_HANDLE_TH_ERRORS
}

// adamw_moments(stream, device, table, m, v, m_scale, v_scale, master) -> (m, v) of 8-bit moments, as the values they stand for,
// of a state that is whole
PyObject *adamw_moments(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    if (!count_is(n, 8)) return nullptr;
    void *stream = address(a[0]);
    const long device = PyLong_AsLong(a[1]);
    if (PyErr_Occurred()) return nullptr;
    const Bytes held(a[2]);
    const auto *table = (const ccnn_adamw_tensor_t *)held.view.buf;
    const int count = (int)(held.view.len / (Py_ssize_t)sizeof *table);
    if (count == 0 || held.view.len != (Py_ssize_t)(count * sizeof *table)) return none();
    long elements = 0, blocks = 0;
    bool any_half = false;
    for (int i = 0; i < count; i++) {
        elements += table[i].n;
        blocks += (table[i].n + CCNN_MOMENT_BLOCK - 1) / CCNN_MOMENT_BLOCK;
        any_half |= table[i].type == CCNN_TYPE_BF16 || table[i].type == CCNN_TYPE_F16;
    }
    void *state[4], *master;
    if (!plain(a[7], device, at::kFloat, elements, &master) || (a[7] == Py_None) == any_half) return none();
    for (int i = 0; i < 4; i++)
        if (!plain(a[3 + i], device, i < 2 ? at::kByte : at::kFloat, i < 2 ? blocks * CCNN_MOMENT_BLOCK : blocks, &state[i])
            || a[3 + i] == Py_None)
            return none();
    const auto wide = at::TensorOptions().device(at::Device(at::kCUDA, (c10::DeviceIndex)device)).dtype(at::kFloat);
    const at::Tensor m = at::empty({elements}, wide), v = at::empty({elements}, wide);
    const int rc = unlocked([&] {
        return adamw_moments_fn(table, count, state[0], state[1], (const float *)state[2], (const float *)state[3],
                                (float *)m.data_ptr(), (float *)v.data_ptr(), stream);
    });
    if (rc) return PyLong_FromLong(rc);
    PyObject *out = PyTuple_New(2);
    if (!out) return nullptr;
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(m));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(v));
    return out;
    END_HANDLE_TH_ERRORS
}

#define CALL(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {CALL(bind), CALL(log_probs), CALL(log_probs_grad), CALL(grad_norm), CALL(adamw_step), CALL(adamw_moments),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "ccnn_torch_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_ccnn_torch_calls() { return PyModule_Create(&module); }
