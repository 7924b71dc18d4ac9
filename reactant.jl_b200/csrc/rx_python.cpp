// The Python package's hot path as an extension module: buffer handles, the call of a single-device program, and the
// capsules of the array exchange.  Everything else goes through ctypes; these three run on every call, where ctypes alone
// costs more than the launch (a call with five results handed to another library: 33 us of the host's time with it).
// The library's entry points are handed in as addresses, so that the module follows whichever build was loaded.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <structmember.h>

#include <vector>

#include "../../include/rx_b200.h"
#include "rx_dlpack.h"

namespace {

struct Entry {
  decltype(&XLAExecuteSharded) execute;
  decltype(&RxLastErrorCode) error_code;
  decltype(&PjRtBufferFree) free_buffer;
  decltype(&RxBufferToDLPack) to_dlpack;
  decltype(&RxBufferFromDLPack) from_dlpack;
  PyObject* check;  // raises what the library reported
} lib = {};

PyObject *s_data, *s_handle, *s_shape, *s_dtype, *s_sharding, *s_replicated;

void raise_reported() {
  PyObject* r = PyObject_CallNoArgs(lib.check);
  if (r) {
    Py_DECREF(r);
    PyErr_SetString(PyExc_RuntimeError, "a call failed without a report");
  }
}

// ---- a buffer handle, freed with the object ----------------------------------------------------------------------
struct Buffer {
  PyObject_HEAD
  void* handle;
  PyObject* device;
};

PyObject* buffer_make(PyTypeObject* type, void* handle, PyObject* device) {
  Buffer* b = (Buffer*)type->tp_alloc(type, 0);
  if (!b) return nullptr;
  b->handle = handle;
  b->device = Py_NewRef(device);
  return (PyObject*)b;
}
PyObject* buffer_new(PyTypeObject* type, PyObject* args, PyObject*) {
  PyObject *handle, *device;
  if (!PyArg_ParseTuple(args, "OO", &handle, &device)) return nullptr;
  void* h = PyLong_AsVoidPtr(handle);
  if (!h && PyErr_Occurred()) return nullptr;
  return buffer_make(type, h, device);
}
void buffer_dealloc(PyObject* self) {
  Buffer* b = (Buffer*)self;
  if (b->handle) lib.free_buffer((RxBuffer*)b->handle);
  Py_XDECREF(b->device);
  Py_TYPE(self)->tp_free(self);
}
PyObject* buffer_handle(PyObject* self, void*) { return PyLong_FromVoidPtr(((Buffer*)self)->handle); }

PyGetSetDef buffer_getset[] = {{"handle", buffer_handle, nullptr, nullptr, nullptr}, {}};
PyMemberDef buffer_members[] = {{"device", T_OBJECT_EX, offsetof(Buffer, device), READONLY, nullptr}, {}};
PyTypeObject BufferType = {PyVarObject_HEAD_INIT(nullptr, 0)};

// ---- a program's call on one device, without waiting ---------------------------------------------------------------
struct Call {
  PyObject_HEAD
  void* exec;
  int n_args, n_results;
  PyObject* masks[2];     // bytes: which arguments are donated, without and with the caller's leave
  PyObject* buffer_type;  // of the results
  PyObject* device;       // where a program without arguments runs
  PyObject* results;      // None, or a tuple of (class, shape, dtype)
};

PyObject* call_new(PyTypeObject* type, PyObject* args, PyObject*) {
  PyObject *exec, *kept, *given, *buffer_type, *device;
  int n_args, n_results;
  if (!PyArg_ParseTuple(args, "OiiSSO!O", &exec, &n_args, &n_results, &kept, &given, &PyType_Type, &buffer_type, &device)) return nullptr;
  if (n_args < 0 || n_results < 0 || PyBytes_GET_SIZE(kept) < n_args || PyBytes_GET_SIZE(given) < n_args || !PyType_IsSubtype((PyTypeObject*)buffer_type, &BufferType)) {
    PyErr_SetString(PyExc_ValueError, "malformed call");
    return nullptr;
  }
  void* h = PyLong_AsVoidPtr(exec);
  if (!h && PyErr_Occurred()) return nullptr;
  Call* c = (Call*)type->tp_alloc(type, 0);
  if (!c) return nullptr;
  c->exec = h;
  c->n_args = n_args;
  c->n_results = n_results;
  c->masks[0] = Py_NewRef(kept);
  c->masks[1] = Py_NewRef(given);
  c->buffer_type = Py_NewRef(buffer_type);
  c->device = Py_NewRef(device);
  c->results = Py_NewRef(Py_None);
  return (PyObject*)c;
}
void call_dealloc(PyObject* self) {
  Call* c = (Call*)self;
  for (PyObject* o : {c->masks[0], c->masks[1], c->buffer_type, c->device, c->results}) Py_XDECREF(o);
  Py_TYPE(self)->tp_free(self);
}

struct Refs {  // references that end with the scope
  std::vector<PyObject*> at;
  ~Refs() {
    for (PyObject* o : at) Py_DECREF(o);
  }
};

// an array object around a buffer, with the attributes of one that is not sharded
PyObject* array_of(PyObject* info, PyObject* buffer) {
  PyObject *cls, *shape, *dtype;
  if (!PyArg_ParseTuple(info, "O!OO", &PyType_Type, &cls, &shape, &dtype)) return nullptr;
  PyObject* a = PyType_GenericAlloc((PyTypeObject*)cls, 0);
  PyObject* data = a ? PyList_New(1) : nullptr;
  if (data) {
    PyList_SET_ITEM(data, 0, Py_NewRef(buffer));
    if (PyObject_SetAttr(a, s_data, data) == 0 && PyObject_SetAttr(a, s_shape, shape) == 0 && PyObject_SetAttr(a, s_dtype, dtype) == 0 &&
        PyObject_SetAttr(a, s_sharding, Py_None) == 0 && PyObject_SetAttr(a, s_replicated, Py_False) == 0) {
      Py_DECREF(data);
      return a;
    }
    Py_DECREF(data);
  }
  Py_XDECREF(a);
  return nullptr;
}

// run(arguments, donate): the results' arrays -- one, or a tuple -- or, as long as `results` is None, a list of their buffers.
// None: an argument is not one buffer on one device, which is not this call's business.
PyObject* call_run(PyObject* self, PyObject* const* argv, Py_ssize_t n) {
  Call* c = (Call*)self;
  if (n != 2 || !PyTuple_Check(argv[0]) || PyTuple_GET_SIZE(argv[0]) != c->n_args) {
    PyErr_SetString(PyExc_TypeError, "run(tuple of the program's arguments, donate)");
    return nullptr;
  }
  const int donate = PyObject_IsTrue(argv[1]);
  if (donate < 0) return nullptr;
  Refs held;  // another thread may give an argument new buffers while this one is in the library
  std::vector<RxBuffer*> in((size_t)c->n_args + 1);
  PyObject* device = c->device;
  for (int k = 0; k < c->n_args; ++k) {
    PyObject* data = PyObject_GetAttr(PyTuple_GET_ITEM(argv[0], k), s_data);
    if (!data) return nullptr;
    PyObject* b = PyList_Check(data) && PyList_GET_SIZE(data) == 1 ? Py_NewRef(PyList_GET_ITEM(data, 0)) : nullptr;
    Py_DECREF(data);
    if (!b) Py_RETURN_NONE;
    held.at.push_back(b);
    if (!PyObject_TypeCheck(b, &BufferType)) Py_RETURN_NONE;
    in[k] = (RxBuffer*)((Buffer*)b)->handle;
    if (k == 0) device = ((Buffer*)b)->device;
  }
  PyObject* handle = PyObject_GetAttr(device, s_handle);
  if (!handle) return nullptr;
  held.at.push_back(handle);
  void* d = PyLong_AsVoidPtr(handle);
  if (!d && PyErr_Occurred()) return nullptr;
  std::vector<RxBuffer*> out((size_t)c->n_results + 1);
  uint8_t* mask = (uint8_t*)PyBytes_AS_STRING(c->masks[donate ? 1 : 0]);
  int failed;
  Py_BEGIN_ALLOW_THREADS;
  lib.execute((RxExecutable*)c->exec, c->n_args, in.data(), (RxDevice*)d, mask, c->n_results, out.data(), nullptr, nullptr);
  failed = lib.error_code();
  Py_END_ALLOW_THREADS;
  if (failed) {
    raise_reported();
    return nullptr;
  }
  Refs buffers;
  for (int k = 0; k < c->n_results; ++k) {
    PyObject* b = buffer_make((PyTypeObject*)c->buffer_type, out[k], device);
    if (!b) {
      for (; k < c->n_results; ++k) lib.free_buffer(out[k]);
      return nullptr;
    }
    buffers.at.push_back(b);
  }
  if (!PyTuple_Check(c->results)) {
    PyObject* list = PyList_New(c->n_results);
    for (int k = 0; list && k < c->n_results; ++k) PyList_SET_ITEM(list, k, Py_NewRef(buffers.at[k]));
    return list;
  }
  if (PyTuple_GET_SIZE(c->results) != c->n_results) {
    PyErr_SetString(PyExc_ValueError, "malformed call");
    return nullptr;
  }
  if (c->n_results == 1) return array_of(PyTuple_GET_ITEM(c->results, 0), buffers.at[0]);
  PyObject* tuple = PyTuple_New(c->n_results);
  for (int k = 0; tuple && k < c->n_results; ++k) {
    PyObject* a = array_of(PyTuple_GET_ITEM(c->results, k), buffers.at[k]);
    if (!a) Py_CLEAR(tuple);
    else PyTuple_SET_ITEM(tuple, k, a);
  }
  return tuple;
}

PyMethodDef call_methods[] = {{"run", (PyCFunction)(void (*)(void))call_run, METH_FASTCALL, nullptr}, {}};
PyMemberDef call_members[] = {{"results", T_OBJECT, offsetof(Call, results), 0, nullptr}, {}};
PyTypeObject CallType = {PyVarObject_HEAD_INIT(nullptr, 0)};

// ---- capsules (the names, and the rule that the consumer renames the capsule, are the specification's) ---------------
constexpr const char *kFresh = "dltensor", *kUsed = "used_dltensor";

void drop_unused(PyObject* capsule) {
  if (!PyCapsule_IsValid(capsule, kFresh)) return;
  auto* t = (rx::DLManagedTensor*)PyCapsule_GetPointer(capsule, kFresh);
  if (t->deleter) t->deleter(t);
}

PyObject* hand_out(PyObject*, PyObject* const* argv, Py_ssize_t n) {
  if (n != 2 || !PyObject_TypeCheck(argv[0], &BufferType)) {
    PyErr_SetString(PyExc_TypeError, "hand_out(buffer, the consumer's stream)");
    return nullptr;
  }
  void* stream = (void*)(intptr_t)PyLong_AsLongLong(argv[1]);
  if (PyErr_Occurred()) return nullptr;
  void* t;
  Py_BEGIN_ALLOW_THREADS;
  t = lib.to_dlpack((RxBuffer*)((Buffer*)argv[0])->handle, stream);
  Py_END_ALLOW_THREADS;
  if (!t) {
    raise_reported();
    return nullptr;
  }
  PyObject* capsule = PyCapsule_New(t, kFresh, drop_unused);
  if (!capsule) ((rx::DLManagedTensor*)t)->deleter((rx::DLManagedTensor*)t);
  return capsule;
}

PyObject* take_over(PyObject*, PyObject* const* argv, Py_ssize_t n) {
  if (n != 2) {
    PyErr_SetString(PyExc_TypeError, "take_over(device handle, capsule)");
    return nullptr;
  }
  void* device = PyLong_AsVoidPtr(argv[0]);
  if (!device && PyErr_Occurred()) return nullptr;
  void* t = PyCapsule_GetPointer(argv[1], kFresh);
  if (!t) return nullptr;
  RxBuffer* b;
  Py_BEGIN_ALLOW_THREADS;
  b = lib.from_dlpack((RxDevice*)device, t);
  Py_END_ALLOW_THREADS;
  if (!b) {
    raise_reported();
    return nullptr;
  }
  PyCapsule_SetName(argv[1], kUsed);
  return PyLong_FromVoidPtr(b);
}

PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long execute, error_code, free_buffer, to_dlpack, from_dlpack;
  PyObject* check;
  if (!PyArg_ParseTuple(args, "KKKKKO", &execute, &error_code, &free_buffer, &to_dlpack, &from_dlpack, &check)) return nullptr;
  lib.execute = (decltype(lib.execute))execute;
  lib.error_code = (decltype(lib.error_code))error_code;
  lib.free_buffer = (decltype(lib.free_buffer))free_buffer;
  lib.to_dlpack = (decltype(lib.to_dlpack))to_dlpack;
  lib.from_dlpack = (decltype(lib.from_dlpack))from_dlpack;
  Py_XSETREF(lib.check, Py_NewRef(check));
  Py_RETURN_NONE;
}

PyMethodDef functions[] = {{"bind", bind, METH_VARARGS, nullptr},
                           {"hand_out", (PyCFunction)(void (*)(void))hand_out, METH_FASTCALL, nullptr},
                           {"take_over", (PyCFunction)(void (*)(void))take_over, METH_FASTCALL, nullptr},
                           {}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_call", nullptr, -1, functions};

}  // namespace

PyMODINIT_FUNC PyInit__call() {
  BufferType.tp_name = "_call.Buffer";
  BufferType.tp_basicsize = sizeof(Buffer);
  BufferType.tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_BASETYPE;
  BufferType.tp_new = buffer_new;
  BufferType.tp_dealloc = buffer_dealloc;
  BufferType.tp_getset = buffer_getset;
  BufferType.tp_members = buffer_members;
  CallType.tp_name = "_call.Call";
  CallType.tp_basicsize = sizeof(Call);
  CallType.tp_flags = Py_TPFLAGS_DEFAULT;
  CallType.tp_new = call_new;
  CallType.tp_dealloc = call_dealloc;
  CallType.tp_methods = call_methods;
  CallType.tp_members = call_members;
  if (PyType_Ready(&BufferType) < 0 || PyType_Ready(&CallType) < 0) return nullptr;
  s_data = PyUnicode_InternFromString("data");
  s_handle = PyUnicode_InternFromString("handle");
  s_shape = PyUnicode_InternFromString("shape");
  s_dtype = PyUnicode_InternFromString("dtype");
  s_sharding = PyUnicode_InternFromString("sharding");
  s_replicated = PyUnicode_InternFromString("replicated");
  PyObject* m = PyModule_Create(&module);
  if (!m || PyModule_AddObjectRef(m, "Buffer", (PyObject*)&BufferType) < 0 || PyModule_AddObjectRef(m, "Call", (PyObject*)&CallType) < 0) return nullptr;
  return m;
}
