// torch_ops.cpp -- what lightfm_amd.operators calls: checks torch tensors, allocates results and scratch memory with torch's
// allocator and hands device pointers and torch's current stream to liblfm_ops.so.  Native because a call of a few
// microseconds on the GPU is otherwise bound by the interpreter (the same work in Python with ctypes took 11 to 30 us a call,
// against 4 to 12 us here).
//
// Nothing throws through the C interface: torch's exceptions (out of memory) are caught and become Python exceptions.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

#include "../../include/lfm_ops.h"

namespace {

PyObject *backend_error = nullptr;  // lightfm_amd._native.HipBackendError

// An argument that the caller has to change: raised as TypeError / ValueError
struct Refused {};

template <typename... A>
[[noreturn]] void refuse(PyObject *type, const char *format, A... a)
{
    PyErr_Format(type, format, a...);
    throw Refused();
}

[[noreturn]] void raise_code(int rc)
{
    PyObject *type = rc == LFM_EINVAL ? PyExc_ValueError : rc == LFM_ENOMEM ? PyExc_MemoryError
                     : rc == LFM_EUNSUPPORTED ? PyExc_NotImplementedError : backend_error ? backend_error : PyExc_RuntimeError;
    refuse(type, "%s", lfm_ops_last_error());
}

void check(int rc)
{
    if (rc != LFM_OK) raise_code(rc);
}

int dtype_of(const at::Tensor &t)
{
    switch (t.scalar_type()) {
    case at::kFloat: return LFM_F32;
    case at::kBFloat16: return LFM_BF16;
    case at::kHalf: return LFM_F16;
    default: return -1;
    }
}

const char *type_name(const at::Tensor &t) { return c10::toString(t.scalar_type()); }

const at::Tensor &tensor(PyObject *o, const char *name)
{
    if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s must be a torch tensor", name);
    const at::Tensor &t = THPVariable_Unpack(o);
    // the caller's backward pass would end here without a word
    if (t.requires_grad() && c10::GradMode::is_enabled() &&
        PyErr_WarnFormat(PyExc_UserWarning, 2, "%s requires a gradient, which this operator does not record: call the gradient functions, "
                                               "and this one under torch.no_grad() or with %s.detach()", name, name) < 0)
        throw Refused();
    if (t.is_neg()) refuse(PyExc_ValueError, "%s is a lazily negated view: call resolve_neg() first", name);
    return t;
}

void shape(const at::Tensor &t, const char *name, int64_t dims)
{
    if (t.layout() != at::kStrided) refuse(PyExc_ValueError, "%s must be a dense tensor", name);
    if (t.dim() != dims) refuse(PyExc_ValueError, "%s has %lld dimensions, expected %lld", name, (long long)t.dim(), (long long)dims);
}

void on_gpu(const at::Tensor &t, const char *name, const at::Tensor *other)
{
    if (!t.is_cuda()) refuse(PyExc_ValueError, "%s is on the %s: the operators need a GPU tensor (there is no CPU fallback)", name, t.device().str().c_str());
    if (other && t.device() != other->device())
        refuse(PyExc_ValueError, "%s is on %s, expected %s", name, t.device().str().c_str(), other->device().str().c_str());
}

// A matrix of contiguous rows of a floating type (that of `like` where it is given); its row stride.
int64_t matrix(const at::Tensor &t, const char *name, const at::Tensor *like)
{
    if (dtype_of(t) < 0) refuse(PyExc_ValueError, "%s has dtype %s, expected float32, bfloat16 or float16", name, type_name(t));
    if (like && t.scalar_type() != like->scalar_type()) refuse(PyExc_ValueError, "%s has dtype %s, expected %s", name, type_name(t), type_name(*like));
    shape(t, name, 2);
    on_gpu(t, name, like);
    const int64_t rows = t.size(0), d = t.size(1);
    if (d < 1) refuse(PyExc_ValueError, "%s has no columns", name);
    if (d > 65536) refuse(PyExc_NotImplementedError, "%s has more than 65536 columns", name);
    if (rows > 0 && d > 1 && t.stride(1) != 1) refuse(PyExc_ValueError, "the elements of a row of %s are not contiguous", name);
    const int64_t stride = rows > 1 ? t.stride(0) : d;
    if (stride < d) refuse(PyExc_ValueError, "the rows of %s overlap", name);
    return stride;
}

// A dense vector; n < 0: any length
void vector(const at::Tensor &t, const char *name, int64_t n, const at::Tensor &like)
{
    shape(t, name, 1);
    on_gpu(t, name, &like);
    if (!t.is_contiguous()) refuse(PyExc_ValueError, "%s is not contiguous", name);
    if (n >= 0 && t.size(0) != n) refuse(PyExc_ValueError, "%s has %lld entries, expected %lld", name, (long long)t.size(0), (long long)n);
}

int id_bytes(const at::Tensor &t, const char *name)
{
    if (t.scalar_type() == at::kInt) return 4;
    if (t.scalar_type() == at::kLong) return 8;
    refuse(PyExc_ValueError, "%s has dtype %s, expected int32 or int64", name, type_name(t));
}

const float *floats(PyObject *o, const char *name, int64_t n, const at::Tensor &like)
{
    if (o == Py_None) return nullptr;
    const at::Tensor &t = tensor(o, name);
    if (t.scalar_type() != at::kFloat) refuse(PyExc_ValueError, "%s has dtype %s, expected float32", name, type_name(t));
    vector(t, name, n, like);
    return (const float *)t.const_data_ptr();
}

// The device of a call made current, its current stream, and memory from torch's allocator
struct On {
    c10::OptionalDeviceGuard guard;
    c10::Device device;
    explicit On(const at::Tensor &t) : device(t.device())
    {
        if (c10::hip::current_device() != device.index()) guard.reset_device(device);
    }
    void *stream() const { return (void *)c10::hip::getCurrentHIPStream(device.index()).stream(); }
    at::Tensor make(at::IntArrayRef sizes, at::ScalarType type) const { return at::empty(sizes, at::TensorOptions().dtype(type).device(device)); }
    at::Tensor scratch(int64_t bytes) const { return make({bytes}, at::kByte); }
};

// runs f and turns what it throws into a Python exception
template <typename F>
PyObject *guarded(F f)
{
    HANDLE_TH_ERRORS
    try {
        return f();
    } catch (const Refused &) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

bool arguments(const char *name, Py_ssize_t got, Py_ssize_t want)
{
    if (got == want) return true;
    PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", name, want, got);
    return false;
}

PyObject *tuple_of(std::initializer_list<at::Tensor> ts)
{
    PyObject *r = PyTuple_New((Py_ssize_t)ts.size());
    if (!r) return nullptr;
    Py_ssize_t i = 0;
    for (const at::Tensor &t : ts) {
        PyObject *o;
        if (t.defined()) o = THPVariable_Wrap(t);
        else {
            Py_INCREF(Py_None);
            o = Py_None;
        }
        if (!o) {
            Py_DECREF(r);
            return nullptr;
        }
        PyTuple_SET_ITEM(r, i++, o);
    }
    return r;
}

// softmax(hidden, table, targets, bias, weights, grad)
PyObject *softmax(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    if (!arguments("softmax", n, 6)) return nullptr;
    return guarded([&]() -> PyObject * {
        const at::Tensor &hidden = tensor(args[0], "hidden"), &table = tensor(args[1], "table"), &targets = tensor(args[2], "targets");
        const bool grad = args[5] == Py_True;
        lfm_softmax_args a = {};
        a.hidden_stride = matrix(hidden, "hidden", nullptr);
        a.table_stride = matrix(table, "table", &hidden);
        a.rows = hidden.size(0);
        a.vocab = table.size(0);
        if (table.size(1) != hidden.size(1))
            refuse(PyExc_ValueError, "hidden has %lld columns, table %lld", (long long)hidden.size(1), (long long)table.size(1));
        if (a.vocab < 1) refuse(PyExc_ValueError, "%s", "table has no rows");
        a.id_bytes = id_bytes(targets, "targets");
        vector(targets, "targets", a.rows, hidden);
        a.bias = floats(args[3], "bias", a.vocab, hidden);
        a.weights = floats(args[4], "weights", a.rows, hidden);
        a.hidden = hidden.const_data_ptr();
        a.table = table.const_data_ptr();
        a.targets = targets.const_data_ptr();
        a.d = (int32_t)hidden.size(1);
        a.dtype = dtype_of(hidden);
        int64_t need = 0;
        check(lfm_ops_softmax_workspace(a.rows, a.vocab, a.d, a.dtype, grad, &need));
        const On on(hidden);
        const at::Tensor loss = on.make({a.rows}, at::kFloat), lse = on.make({a.rows}, at::kFloat), ws = on.scratch(need);
        a.loss = (float *)loss.data_ptr();
        a.lse = (float *)lse.data_ptr();
        if (!grad) {
            check(lfm_ops_softmax_loss(&a, ws.data_ptr(), need, on.stream()));
            return tuple_of({loss, lse});
        }
        const at::Tensor dh = on.make({a.rows, a.d}, hidden.scalar_type()), dt = on.make({a.vocab, a.d}, hidden.scalar_type());
        at::Tensor db;
        if (a.bias) {
            db = on.make({a.vocab}, at::kFloat);
            a.d_bias = (float *)db.data_ptr();
        }
        a.d_hidden = dh.data_ptr();
        a.d_table = dt.data_ptr();
        check(lfm_ops_softmax_loss_grad(&a, ws.data_ptr(), need, on.stream()));
        return tuple_of({loss, lse, dh, dt, db});
    });
}

// lookup(table or d_out, ids, indptr, values, scale, n_rows): n_rows < 0 the lookup, else the gradient for so many rows
PyObject *lookup(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    if (!arguments("lookup", n, 6)) return nullptr;
    return guarded([&]() -> PyObject * {
        const long long n_rows = PyLong_AsLongLong(args[5]);
        const double scale = PyFloat_AsDouble(args[4]);
        if (PyErr_Occurred()) throw Refused();
        const bool grad = n_rows >= 0;
        const char *name = grad ? "d_out" : "table";
        const at::Tensor &m = tensor(args[0], name), &ids = tensor(args[1], "ids");
        const bool bags = args[2] != Py_None;
        lfm_lookup_args a = {};
        const int64_t stride = matrix(m, name, nullptr);
        a.id_bytes = id_bytes(ids, "ids");
        vector(ids, "ids", -1, m);
        a.nnz = ids.size(0);
        a.rows = a.nnz;
        if (bags) {
            const at::Tensor &indptr = tensor(args[2], "indptr");
            if (indptr.scalar_type() != ids.scalar_type()) refuse(PyExc_ValueError, "indptr has dtype %s, expected %s", type_name(indptr), type_name(ids));
            vector(indptr, "indptr", -1, m);
            if (indptr.size(0) < 1) refuse(PyExc_ValueError, "%s", "indptr is empty");
            a.rows = indptr.size(0) - 1;
            if (a.rows == 0 && a.nnz) refuse(PyExc_ValueError, "%s", "ids without a bag");
            a.indptr = indptr.const_data_ptr();
            a.values = floats(args[3], "values", a.nnz, m);
        } else if (args[3] != Py_None)
            refuse(PyExc_ValueError, "%s", "values need an indptr");
        a.ids = ids.const_data_ptr();
        a.d = (int32_t)m.size(1);
        a.dtype = dtype_of(m);
        a.scale = (float)scale;
        const On on(m);
        if (!grad) {
            a.vocab = m.size(0);
            if (a.vocab < 1) refuse(PyExc_ValueError, "%s", "table has no rows");
            a.table = m.const_data_ptr();
            a.table_stride = stride;
            const at::Tensor out = on.make({a.rows, a.d}, m.scalar_type());
            a.out = out.data_ptr();
            check(lfm_ops_embedding_lookup(&a, on.stream()));
            return THPVariable_Wrap(out);
        }
        if (m.size(0) != a.rows) refuse(PyExc_ValueError, "d_out has %lld rows, expected %lld", (long long)m.size(0), (long long)a.rows);
        if (n_rows < 1) refuse(PyExc_ValueError, "%s", "n_rows must be positive");
        a.vocab = n_rows;
        a.d_out = m.const_data_ptr();
        a.d_out_stride = stride;
        int64_t need = 0;
        check(lfm_ops_embedding_grad_workspace(a.rows, a.vocab, a.nnz, a.d, bags, &need));
        const at::Tensor out = on.make({a.vocab, a.d}, m.scalar_type()), ws = on.scratch(need);
        a.out = out.data_ptr();
        check(lfm_ops_embedding_lookup_grad(&a, ws.data_ptr(), need, on.stream()));
        return THPVariable_Wrap(out);
    });
}

// A list or tuple of tensors, all on one device
void tensors_of(PyObject *o, const char *name, std::vector<const at::Tensor *> &to)
{
    if (!PyList_Check(o) && !PyTuple_Check(o)) refuse(PyExc_TypeError, "%s must be a list or tuple of tensors", name);
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(o);
    to.reserve((size_t)n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        const at::Tensor &t = tensor(PySequence_Fast_GET_ITEM(o, i), name);
        if (dtype_of(t) < 0) refuse(PyExc_ValueError, "%s[%zd] has dtype %s, expected float32, bfloat16 or float16", name, i, type_name(t));
        on_gpu(t, name, to.empty() ? nullptr : to[0]);
        if (t.layout() != at::kStrided || !t.is_contiguous()) refuse(PyExc_ValueError, "%s[%zd] is not contiguous", name, i);
        to.push_back(&t);
    }
}

// clip(tensors, max_norm, out): out None the norm alone
PyObject *clip(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    if (!arguments("clip", n, 3)) return nullptr;
    return guarded([&]() -> PyObject * {
        const double top = PyFloat_AsDouble(args[1]);
        if (PyErr_Occurred()) throw Refused();
        std::vector<const at::Tensor *> xs, ys;
        tensors_of(args[0], "tensors", xs);
        if (xs.empty()) refuse(PyExc_ValueError, "%s", "no tensors");
        const bool scale = args[2] != Py_None;
        if (scale) {
            tensors_of(args[2], "out", ys);
            if (ys.size() != xs.size()) refuse(PyExc_ValueError, "%zd tensors, %zd outputs", (Py_ssize_t)xs.size(), (Py_ssize_t)ys.size());
        }
        std::vector<const void *> x(xs.size());
        std::vector<void *> y(ys.size());
        std::vector<int64_t> counts(xs.size());
        std::vector<int32_t> kinds(xs.size());
        for (size_t i = 0; i < xs.size(); ++i) {
            x[i] = xs[i]->const_data_ptr();
            counts[i] = xs[i]->numel();
            kinds[i] = dtype_of(*xs[i]);
            if (!scale) continue;
            if (ys[i]->scalar_type() != xs[i]->scalar_type()) refuse(PyExc_ValueError, "out[%zd] has dtype %s, expected %s", (Py_ssize_t)i, type_name(*ys[i]), type_name(*xs[i]));
            if (ys[i]->sizes() != xs[i]->sizes()) refuse(PyExc_ValueError, "out[%zd] has another shape than tensors[%zd]", (Py_ssize_t)i, (Py_ssize_t)i);
            if (ys[i]->device() != xs[0]->device()) refuse(PyExc_ValueError, "out[%zd] is on another device", (Py_ssize_t)i);
            y[i] = ys[i]->data_ptr();
        }
        int64_t need = 0;
        check(lfm_ops_clip_workspace((int64_t)xs.size(), counts.data(), &need));
        const On on(*xs[0]);
        const at::Tensor norm = on.make({}, at::kFloat), ws = on.scratch(need);
        check(lfm_ops_clip_global_norm((int64_t)xs.size(), x.data(), scale ? y.data() : nullptr, counts.data(), kinds.data(), top,
                                       (float *)norm.data_ptr(), ws.data_ptr(), need, on.stream()));
        for (const at::Tensor *t : ys)  // written in place: autograd has to notice
            if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
        return THPVariable_Wrap(norm);
    });
}

PyMethodDef methods[] = {
    {"softmax", (PyCFunction)(void (*)(void))softmax, METH_FASTCALL, nullptr},
    {"lookup", (PyCFunction)(void (*)(void))lookup, METH_FASTCALL, nullptr},
    {"clip", (PyCFunction)(void (*)(void))clip, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef definition = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops(void)
{
    if (PyObject *native = PyImport_ImportModule("lightfm_amd._native")) {
        backend_error = PyObject_GetAttrString(native, "HipBackendError");
        Py_DECREF(native);
    }
    if (!backend_error) return nullptr;
    return PyModule_Create(&definition);
}
