// What the optimizer's entry points have to know about a list of tensors, in one call: addresses, sizes, types, device, order
// in memory.  The seven attribute calls a tensor that this takes in Python cost 0.5 us, more than a whole elementwise pass over
// a small parameter.  A CPython module over torch's C++ tensors; it reads their metadata only and touches no GPU.
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <string>
#include <vector>

namespace {

// element type codes of include/ddcn_hip.h
int code_of(at::ScalarType t)
{
    return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1;
}

constexpr int kNone = -3, kMixed = -2;

template <class T> PyObject *bytes_of(const std::vector<T> &v)
{
    return PyBytes_FromStringAndSize((const char *)v.data(), (Py_ssize_t)(v.size() * sizeof(T)));
}

// The tensor of an item, or null with an error set
const at::Tensor *tensor_of(PyObject *o)
{
    if (THPVariable_Check(o)) return &THPVariable_Unpack(o);
    PyErr_Format(PyExc_TypeError, "a tensor was expected, got %s", Py_TYPE(o)->tp_name);
    return nullptr;
}

template <class F> PyObject *guarded(F f)
{
    try {
        return f();
    } catch (const c10::Error &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// describe(list) -> (addresses u64, sizes i64, types i32, device, type, contiguous, distinct, given).  None: address, size and
// type 0.  device: the common GPU, -1 if any tensor is elsewhere, -2 if there are several, -3 if there is no tensor; type: the
// common code, -1 if any is no supported type, -2 if there are several, -3 if there is no tensor; contiguous: all are;
// distinct: no address of a tensor with elements comes twice; given: the number of tensors.
PyObject *describe(PyObject *, PyObject *list)
{
    if (!PyList_Check(list)) {
        PyErr_SetString(PyExc_TypeError, "a list was expected");
        return nullptr;
    }
    return guarded([&]() -> PyObject * {
        const Py_ssize_t count = PyList_GET_SIZE(list);
        std::vector<uint64_t> pointers(count, 0), places;
        std::vector<int64_t> sizes(count, 0);
        std::vector<int32_t> types(count, 0);
        places.reserve(count);
        int device = kNone, type = kNone;
        long given = 0;
        bool contiguous = true;
        for (Py_ssize_t i = 0; i < count; ++i) {
            PyObject *o = PyList_GET_ITEM(list, i);
            if (o == Py_None) continue;
            const at::Tensor *t = tensor_of(o);
            if (!t) return nullptr;
            const int d = t->is_cuda() ? t->get_device() : -1, c = code_of(t->scalar_type());
            device = device == kNone ? d : device == -1 || d == -1 ? -1 : device == d ? d : kMixed;
            type = type == kNone ? c : type == -1 || c == -1 ? -1 : type == c ? c : kMixed;
            ++given;
            contiguous = contiguous && t->is_contiguous();
            pointers[i] = (uint64_t)t->data_ptr();
            sizes[i] = t->numel();
            types[i] = c;
            if (sizes[i]) places.push_back(pointers[i]);
        }
        std::sort(places.begin(), places.end());
        const bool distinct = std::adjacent_find(places.begin(), places.end()) == places.end();
        return Py_BuildValue("NNNiiOOl", bytes_of(pointers), bytes_of(sizes), bytes_of(types), device, type,
                             contiguous ? Py_True : Py_False, distinct ? Py_True : Py_False, given);
    });
}

// changed(tensors, beside=None): the versions that autograd compares, one on; where `beside` holds a None the tensor is left.
// Inference tensors keep no versions.
PyObject *changed(PyObject *, PyObject *args)
{
    PyObject *list, *beside = Py_None;
    if (!PyArg_ParseTuple(args, "O!|O", &PyList_Type, &list, &beside)) return nullptr;
    if (beside != Py_None && (!PyList_Check(beside) || PyList_GET_SIZE(beside) != PyList_GET_SIZE(list))) {
        PyErr_SetString(PyExc_TypeError, "two lists of one length were expected");
        return nullptr;
    }
    return guarded([&]() -> PyObject * {
        for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); ++i) {
            if (beside != Py_None && PyList_GET_ITEM(beside, i) == Py_None) continue;
            const at::Tensor *t = tensor_of(PyList_GET_ITEM(list, i));
            if (!t) return nullptr;
            if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
        }
        Py_RETURN_NONE;
    });
}

// alike(params, grads) -> 0, or what is wrong with a pair (a None among the gradients is none): 1, another shape or order in memory, or
// one that is neither contiguous nor channels-last; 2, another number of elements
PyObject *alike(PyObject *, PyObject *args)
{
    PyObject *params, *grads;
    if (!PyArg_ParseTuple(args, "O!O!", &PyList_Type, &params, &PyList_Type, &grads)) return nullptr;
    if (PyList_GET_SIZE(params) != PyList_GET_SIZE(grads)) {
        PyErr_SetString(PyExc_TypeError, "two lists of one length were expected");
        return nullptr;
    }
    return guarded([&]() -> PyObject * {
        long wrong = 0;
        for (Py_ssize_t i = 0; i < PyList_GET_SIZE(params) && !wrong; ++i) {
            if (PyList_GET_ITEM(grads, i) == Py_None) continue;
            const at::Tensor *p = tensor_of(PyList_GET_ITEM(params, i)), *g = p ? tensor_of(PyList_GET_ITEM(grads, i)) : nullptr;
            if (!g) return nullptr;
            if (!p->is_contiguous() || !g->is_contiguous())
                wrong = p->sizes() == g->sizes() && p->strides() == g->strides() &&
                        (p->is_contiguous() || p->is_contiguous(at::MemoryFormat::ChannelsLast) ||
                         p->is_contiguous(at::MemoryFormat::ChannelsLast3d)) ? 0 : 1;
            if (!wrong && p->numel() != g->numel()) wrong = 2;
        }
        return PyLong_FromLong(wrong);
    });
}

PyMethodDef methods[] = {{"describe", describe, METH_O, nullptr}, {"alike", alike, METH_VARARGS, nullptr},
                         {"changed", changed, METH_VARARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ddcn_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ddcn_tensors(void)
{
    return PyModule_Create(&module);
}
