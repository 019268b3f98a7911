// Calls of the operators on device pointers from Python: what each operand is, its address, and the call.  A call costs the host some 4 us with its
// launch, and some 1.5 of them are Python's, with the look at eight tensors that this file takes (in Python itself: 3.0; without a look 1.5).
// Only Python's own API is used: a tensor is asked through its attributes, so that any build of torch will do.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstdint>

namespace {

// What an operand has to hold where it is a tensor: values of a type of the library (0 .. 2), of the descriptor's own type field, of its cache's
// (its first field); and kStrided, where the descriptor has strides for all but the last dimension.
enum { kInts = 3, kBytes = 4, kAny = 5, kRows = 6, kCache = 7, kStrided = 8 };
const char* const kNames[] = {"float32", "float16", "bfloat16", "int32", "uint8 or bool", "any type"};
constexpr int kMost = 10;                    // operands

PyObject *tensor_type, *dtypes, *devices_differ, *current_stream, *other_address;     // (learn)
PyObject *s_dtype, *s_is_cuda, *s_is_contiguous, *s_stride, *s_data_ptr;

bool is_true(PyObject* x) {                  // takes the reference
    const bool yes = x == Py_True;
    Py_XDECREF(x);
    return yes;
}

// Whether the tensor is on the device, of that type and laid out as the library reads it; false with an error set: asking failed.
bool fits(PyObject* x, int kind, int type) {
    if (!is_true(PyObject_GetAttr(x, s_is_cuda))) return false;
    if (type != kAny) {
        PyObject* const dtype = PyObject_GetAttr(x, s_dtype);
        if (!dtype) return false;
        Py_DECREF(dtype);                    // (torch keeps its types)
        if (dtype != PyTuple_GET_ITEM(dtypes, type) && !(type == kBytes && dtype == PyTuple_GET_ITEM(dtypes, kBytes + 1))) return false;
    }
    if (!is_true(PyObject_CallMethodNoArgs(x, s_is_contiguous))) {
        if (PyErr_Occurred() || !(kind & kStrided)) return false;
        PyObject* const strides = PyObject_CallMethodNoArgs(x, s_stride);
        if (!strides) return false;
        const Py_ssize_t n = PyTuple_GET_SIZE(strides);
        const bool last = n && PyLong_AsLongLong(PyTuple_GET_ITEM(strides, n - 1)) == 1;
        Py_DECREF(strides);
        if (!last) return false;
    }
    if (devices_differ != Py_None) {         // several devices
        PyObject* const other = PyObject_CallOneArg(devices_differ, x);
        if (!other || is_true(other)) return false;
    }
    return true;
}

// call(operator, descriptor, bytes of the workspace or None, stream, *operands): the operator is (address, kinds, offset of the type field,
// bytes of the descriptor).
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
    PyObject* const op = args[0];
    const char* const kinds = PyBytes_AS_STRING(PyTuple_GET_ITEM(op, 1));
    const Py_ssize_t operands = n - 4;
    if (operands != PyBytes_GET_SIZE(PyTuple_GET_ITEM(op, 1)) || operands > kMost) return PyErr_Format(PyExc_TypeError, "%zd operands", operands);
    Py_buffer desc;
    if (PyObject_GetBuffer(args[1], &desc, PyBUF_SIMPLE)) return nullptr;
    struct Release {
        Py_buffer* b;
        ~Release() { PyBuffer_Release(b); }
    } release{&desc};
    const long type_at = PyLong_AsLong(PyTuple_GET_ITEM(op, 2)), size = PyLong_AsLong(PyTuple_GET_ITEM(op, 3));
    if (desc.len != size) return PyErr_Format(PyExc_TypeError, "a descriptor of %ld bytes is needed, not one of %zd", size, desc.len);
    const auto field = [&](long at) {
        const int32_t v = *(const int32_t*)((const char*)desc.buf + at);
        return v >= 0 && v <= 2 ? (int)v : (int)kAny;        // (types that there are not: the library refuses them)
    };
    void* p[kMost] = {};
    bool tensors = false;
    for (Py_ssize_t i = 0; i < operands; ++i) {
        PyObject* const x = args[4 + i];
        if (x == Py_None) continue;
        PyObject* address;
        if (tensor_type && ((PyObject*)Py_TYPE(x) == tensor_type || PyObject_IsInstance(x, tensor_type) == 1)) {
            int type = kinds[i] & 7;
            if (type == kRows) type = field(type_at);
            if (type == kCache) type = field(0);
            if (!fits(x, kinds[i], type)) {
                if (!PyErr_Occurred())
                    PyErr_Format(PyExc_TypeError, "operand %zd: a tensor on the current device, of %s, %s, is needed, not one of another device, type or layout (%.100s)", i,
                                 kNames[type], kinds[i] & kStrided ? "contiguous in its last dimension" : "contiguous", Py_TYPE(x)->tp_name);
                return nullptr;
            }
            tensors = true;
            address = PyObject_CallMethodNoArgs(x, s_data_ptr);
        } else if (PyLong_CheckExact(x)) {
            Py_INCREF(x);
            address = x;
        } else {
            address = PyObject_CallOneArg(other_address, x);     // (may find the first tensor: asked again)
            if (address == Py_None && tensor_type && PyObject_IsInstance(x, tensor_type) == 1) {
                Py_DECREF(address);
                --i;
                continue;
            }
        }
        if (!address) return nullptr;
        if (address != Py_None) p[i] = (void*)PyLong_AsUnsignedLongLongMask(address);
        Py_DECREF(address);
        if (PyErr_Occurred()) return nullptr;
    }
    void* stream = nullptr;
    if (args[3] != Py_None || tensors) {
        PyObject* const s = args[3] == Py_None ? PyObject_CallNoArgs(current_stream) : PyLong_CheckExact(args[3]) ? Py_NewRef(args[3]) : PyObject_CallOneArg(other_address, args[3]);
        if (!s) return nullptr;
        if (s != Py_None) stream = (void*)PyLong_AsUnsignedLongLongMask(s);
        Py_DECREF(s);
        if (PyErr_Occurred()) return nullptr;
    }
    const bool sized = args[2] != Py_None;
    const int64_t bytes = sized ? PyLong_AsLongLong(args[2]) : 0;
    void* const f = PyLong_AsVoidPtr(PyTuple_GET_ITEM(op, 0));
    if (PyErr_Occurred()) return nullptr;
    typedef void* P;
    const void* const d = desc.buf;
    int status = 1;
    bool known = true;
    Py_BEGIN_ALLOW_THREADS
    switch (operands * 2 + sized) {
        case 10: status = ((int (*)(const void*, P, P, P, P, P, P))f)(d, p[0], p[1], p[2], p[3], p[4], stream); break;
        case 13: status = ((int (*)(const void*, P, P, P, P, P, P, int64_t, P))f)(d, p[0], p[1], p[2], p[3], p[4], p[5], bytes, stream); break;
        case 15: status = ((int (*)(const void*, P, P, P, P, P, P, P, int64_t, P))f)(d, p[0], p[1], p[2], p[3], p[4], p[5], p[6], bytes, stream); break;
        case 16: status = ((int (*)(const void*, P, P, P, P, P, P, P, P, P))f)(d, p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], stream); break;
        case 17: status = ((int (*)(const void*, P, P, P, P, P, P, P, P, int64_t, P))f)(d, p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], bytes, stream); break;
        case 18: status = ((int (*)(const void*, P, P, P, P, P, P, P, P, P, P))f)(d, p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], p[8], stream); break;
        case 21:
            status = ((int (*)(const void*, P, P, P, P, P, P, P, P, P, P, int64_t, P))f)(d, p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], p[8], p[9], bytes, stream);
            break;
        default: known = false;
    }
    Py_END_ALLOW_THREADS
    return known ? PyLong_FromLong(status) : PyErr_Format(PyExc_TypeError, "%zd operands", operands);
}

// learn(other_address): asked for what is no tensor, address or None.
// learn(other_address, tensor type, types by their numbers, devices_differ(tensor) or None, current_stream()).
PyObject* learn(PyObject*, PyObject* args) {
    PyObject *other, *type = nullptr, *types = nullptr, *differ = nullptr, *stream = nullptr;
    if (!PyArg_ParseTuple(args, "O|OO!OO", &other, &type, &PyTuple_Type, &types, &differ, &stream)) return nullptr;
    Py_INCREF(other);
    Py_XSETREF(other_address, other);
    if (stream) {
        if (PyTuple_GET_SIZE(types) != kBytes + 2) return PyErr_Format(PyExc_ValueError, "%zd types", PyTuple_GET_SIZE(types));
        Py_INCREF(types);
        Py_XSETREF(dtypes, types);
        Py_INCREF(differ);
        Py_XSETREF(devices_differ, differ);
        Py_INCREF(stream);
        Py_XSETREF(current_stream, stream);
        Py_INCREF(type);
        Py_XSETREF(tensor_type, type);
    }
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"call", (PyCFunction)(void (*)())call, METH_FASTCALL, nullptr}, {"learn", learn, METH_VARARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "reef_operands", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_reef_operands() {
    s_dtype = PyUnicode_InternFromString("dtype");
    s_is_cuda = PyUnicode_InternFromString("is_cuda");
    s_is_contiguous = PyUnicode_InternFromString("is_contiguous");
    s_stride = PyUnicode_InternFromString("stride");
    s_data_ptr = PyUnicode_InternFromString("data_ptr");
    return PyModule_Create(&module);
}
