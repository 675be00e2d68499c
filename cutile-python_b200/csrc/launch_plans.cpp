// Checked calls of the library's entry points, remembered by the layouts of their tensors.
//
// A wrapper checks a call and fills in an argument struct once per combination of shapes, strides,
// types, devices and scalars; this module keeps the struct under that combination.  A later call
// with the same layouts makes its outputs and workspace, sets the pointers in a copy of the struct
// and calls the entry point.  Nothing is kept of an address (but whether it is a multiple of 16,
// which a kernel's vector loads depend on) or of contents.  It is the wrapper-side half of what
// the reference keeps per kernel in its launch path (hash lookup, then the launch,
// cext/tile_kernel.cpp:3816-3844).
//
// As Python it took 14 us per call, of which 10 were lookups of tensor attributes; on small problems
// the GPU waited for the host.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cstring>
#include <deque>
#include <memory>
#include <string>
#include <unordered_map>
#include <utility>
#include <vector>

namespace {

constexpr size_t kMaxPlans = 1024;        // beyond, a new one takes the oldest's place
constexpr Py_ssize_t kMaxTensors = 24;
constexpr size_t kMaxArgBytes = 1024;

using EntryPoint = int (*)(const void* args, void* stream);

struct Plan {
  std::string args;                                   // the struct, pointers not set
  std::vector<std::pair<int, int>> inputs;            // (offset, tensor)
  std::vector<std::pair<int, int>> outputs;           // (offset, tensor whose shape and type it has)
  int workspace_offset = -1;
  int64_t workspace_bytes = 0;
  std::vector<int> returns;                           // output i, or -1 - i for tensor i; kNone
  static constexpr int kNone = -1000;
};

// Plans by key, and the keys in the order they came; a full table drops its oldest.
struct Table {
  std::unordered_map<std::string, std::shared_ptr<const Plan>> plans;
  std::deque<const std::string*> order;               // (a map's keys stay where they are)

  void put(const std::string& key, std::shared_ptr<const Plan> plan) {
    const auto [at, added] = plans.insert_or_assign(key, std::move(plan));
    if (!added) return;
    order.push_back(&at->first);
    if (plans.size() <= kMaxPlans) return;
    plans.erase(plans.find(*order.front()));
    order.pop_front();
  }
};

struct Plans {
  PyObject_HEAD
  EntryPoint entry;
  PyObject* check;                                    // raises the error of a negative status
  Table* table;
};

struct Call {
  std::string key;
  const at::Tensor* tensor[kMaxTensors];
  Py_ssize_t count = 0;
};

template <typename T> void put(std::string& key, T v) { key.append(reinterpret_cast<const char*>(&v), sizeof(v)); }

// False where a call can have no plan (an argument that is no strided CUDA tensor or has a tangent, an
// odd scalar):
// the wrapper's checks say what is wrong with it.
bool read_call(PyObject* tensors, PyObject* scalars, Call& c) {
  if (!PyTuple_Check(tensors) || !PyTuple_Check(scalars) || PyTuple_GET_SIZE(tensors) > kMaxTensors) return false;
  c.count = PyTuple_GET_SIZE(tensors);
  c.key.reserve(768);
  for (Py_ssize_t i = 0; i < c.count; ++i) {
    PyObject* o = PyTuple_GET_ITEM(tensors, i);
    c.tensor[i] = nullptr;
    if (o == Py_None) {
      put<int8_t>(c.key, -1);
      continue;
    }
    if (!THPVariable_Check(o)) return false;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t._fw_grad(0).defined()) return false;
    c.tensor[i] = &t;
    put<int8_t>(c.key, static_cast<int8_t>(t.dim()));
    put<int8_t>(c.key, static_cast<int8_t>(t.scalar_type()));
    put<int8_t>(c.key, static_cast<int8_t>(t.device().index()));
    put<int8_t>(c.key, static_cast<int8_t>((t.requires_grad() ? 1 : 0) |
                                           ((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0 ? 2 : 0)));
    const auto sizes = t.sizes(), strides = t.strides();
    c.key.append(reinterpret_cast<const char*>(sizes.data()), sizes.size() * sizeof(int64_t));
    c.key.append(reinterpret_cast<const char*>(strides.data()), strides.size() * sizeof(int64_t));
  }
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(scalars); ++i) {
    PyObject* o = PyTuple_GET_ITEM(scalars, i);
    if (o == Py_None) {
      put<int8_t>(c.key, 0);
    } else if (o == Py_True || o == Py_False) {
      put<int8_t>(c.key, o == Py_True ? 2 : 1);
    } else if (PyFloat_Check(o)) {
      put<int8_t>(c.key, 3);
      put<double>(c.key, PyFloat_AS_DOUBLE(o));
    } else {
      return false;
    }
  }
  put<int8_t>(c.key, c10::GradMode::is_enabled() ? 1 : 0);
  return true;
}

int plans_init(PyObject* self_, PyObject* args, PyObject*) {
  auto* self = reinterpret_cast<Plans*>(self_);
  unsigned long long address;
  PyObject* check;
  if (!PyArg_ParseTuple(args, "KO", &address, &check)) return -1;
  self->entry = reinterpret_cast<EntryPoint>(static_cast<uintptr_t>(address));
  Py_INCREF(check);
  Py_XSETREF(self->check, check);
  if (self->table == nullptr) self->table = new Table();
  return 0;
}

void plans_dealloc(PyObject* self_) {
  auto* self = reinterpret_cast<Plans*>(self_);
  Py_XDECREF(self->check);
  delete self->table;
  PyTypeObject* type = Py_TYPE(self_);
  type->tp_free(self_);
  Py_DECREF(type);
}

bool read_pairs(PyObject* seq, Py_ssize_t tensors, size_t arg_bytes, std::vector<std::pair<int, int>>& out) {
  if (!PyTuple_Check(seq)) return false;
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(seq); ++i) {
    int offset, index;
    if (!PyArg_ParseTuple(PyTuple_GET_ITEM(seq, i), "ii", &offset, &index)) return false;
    if (offset < 0 || offset + sizeof(void*) > arg_bytes || index < 0 || index >= tensors) return false;
    out.emplace_back(offset, index);
  }
  return true;
}

// The interpreter's lock, released while this lives: taken back also where an exception leaves.
struct ReleasedLock {
  PyThreadState* const state = PyEval_SaveThread();
  ~ReleasedLock() { PyEval_RestoreThread(state); }
};

// Runs a plan: makes its outputs and workspace, sets the pointers in a copy of the struct, calls the
// entry point.  The caller holds `plan`: another thread may drop it from the table meanwhile.
PyObject* launch(const Plans* self, const Plan& plan, const Call& call, PyObject* tensors) {
  alignas(16) char args[kMaxArgBytes];
  std::memcpy(args, plan.args.data(), plan.args.size());
  const auto set = [&args](int offset, const void* pointer) { std::memcpy(args + offset, &pointer, sizeof(pointer)); };
  for (const auto& [offset, index] : plan.inputs) set(offset, call.tensor[index]->data_ptr());
  const at::Device device = call.tensor[0]->device();
  int code;
  std::vector<at::Tensor> outputs;
  {
    const c10::cuda::CUDAGuard guard(device);
    outputs.reserve(plan.outputs.size());
    for (const auto& [offset, index] : plan.outputs) {
      const at::Tensor& like = *call.tensor[index];
      outputs.push_back(at::empty(like.sizes(), at::TensorOptions().dtype(like.scalar_type()).device(device)));
      set(offset, outputs.back().data_ptr());
    }
    // made per call: calls on other streams and other captured graphs have their own
    at::Tensor workspace;
    if (plan.workspace_offset >= 0 && plan.workspace_bytes > 0) {
      workspace = at::empty({plan.workspace_bytes}, at::TensorOptions().dtype(at::kByte).device(device));
      set(plan.workspace_offset, workspace.data_ptr());
    }
    void* stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    const ReleasedLock released;
    code = self->entry(args, stream);
  }
  if (code < 0) {
    PyObject* raised = PyObject_CallFunction(self->check, "i", code);
    if (raised != nullptr) {
      Py_DECREF(raised);
      PyErr_Format(PyExc_RuntimeError, "entry point returned %d", code);
    }
    return nullptr;
  }
  const auto result = [&](int v) -> PyObject* {
    if (v == Plan::kNone) Py_RETURN_NONE;
    if (v >= 0) return THPVariable_Wrap(outputs[v]);
    return Py_NewRef(PyTuple_GET_ITEM(tensors, -1 - v));
  };
  if (plan.returns.size() == 1) return result(plan.returns[0]);
  PyObject* tuple = PyTuple_New(static_cast<Py_ssize_t>(plan.returns.size()));
  if (tuple == nullptr) return nullptr;
  for (size_t i = 0; i < plan.returns.size(); ++i) {
    PyObject* o = result(plan.returns[i]);
    if (o == nullptr) {
      Py_DECREF(tuple);
      return nullptr;
    }
    PyTuple_SET_ITEM(tuple, static_cast<Py_ssize_t>(i), o);
  }
  return tuple;
}

// The error that the C++ exception being handled becomes.
PyObject* raise_current() {
  try {
    throw;
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch == nullptr ? nullptr : PyObject_GetAttrString(torch, "OutOfMemoryError");
    Py_XDECREF(torch);
    if (type != nullptr) {
      PyErr_SetString(type, e.what());
      Py_DECREF(type);
    }
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

// add(tensors, scalars, args, inputs, outputs, workspace_offset, workspace_bytes, returns): remembers the
// call and makes it.  One step, so that no other thread's plans come between.
PyObject* plans_add(PyObject* self_, PyObject* args) try {
  auto* self = reinterpret_cast<Plans*>(self_);
  if (self->table == nullptr) {
    PyErr_SetString(PyExc_RuntimeError, "Plans without an entry point");
    return nullptr;
  }
  PyObject *tensors, *scalars, *inputs, *outputs, *returns;
  const char* bytes;
  Py_ssize_t size;
  Plan plan;
  long long workspace;
  if (!PyArg_ParseTuple(args, "OOy#OOiLO", &tensors, &scalars, &bytes, &size, &inputs, &outputs, &plan.workspace_offset,
                        &workspace, &returns))
    return nullptr;
  Call call;
  bool ok = read_call(tensors, scalars, call) && call.count > 0 && call.tensor[0] != nullptr && size > 0 &&
            static_cast<size_t>(size) <= kMaxArgBytes && read_pairs(inputs, call.count, size, plan.inputs) && read_pairs(outputs, call.count, size, plan.outputs) &&
            workspace >= 0 && (plan.workspace_offset < 0 || plan.workspace_offset + static_cast<Py_ssize_t>(sizeof(void*)) <= size) &&
            PyTuple_Check(returns);
  for (const auto& [offset, index] : plan.inputs) ok = ok && call.tensor[index] != nullptr;
  for (const auto& [offset, index] : plan.outputs) ok = ok && call.tensor[index] != nullptr;
  if (ok) {
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(returns); ++i) {
      PyObject* o = PyTuple_GET_ITEM(returns, i);
      const long v = o == Py_None ? Plan::kNone : PyLong_AsLong(o);
      ok = ok && !PyErr_Occurred() &&
           (v == Plan::kNone || (v >= 0 ? v < static_cast<long>(plan.outputs.size())
                                        : -1 - v < call.count && call.tensor[-1 - v] != nullptr));
      plan.returns.push_back(static_cast<int>(v));
    }
  }
  if (!ok) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "not a plan");
    return nullptr;
  }
  plan.args.assign(bytes, size);
  plan.workspace_bytes = workspace;
  const auto kept = std::make_shared<const Plan>(std::move(plan));
  self->table->put(call.key, kept);
  return launch(self, *kept, call, tensors);
} catch (...) {
  return raise_current();
}

// call(tensors, scalars): the outputs, or NotImplemented where these layouts have no plan
PyObject* plans_call(PyObject* self_, PyObject* const* argv, Py_ssize_t argc) try {
  auto* self = reinterpret_cast<Plans*>(self_);
  if (argc != 2 || self->table == nullptr) {
    PyErr_SetString(PyExc_TypeError, "call(tensors, scalars) of a Plans with an entry point");
    return nullptr;
  }
  Call call;
  if (!read_call(argv[0], argv[1], call)) Py_RETURN_NOTIMPLEMENTED;
  const auto found = self->table->plans.find(call.key);
  if (found == self->table->plans.end()) Py_RETURN_NOTIMPLEMENTED;
  const std::shared_ptr<const Plan> plan = found->second;
  return launch(self, *plan, call, argv[0]);
} catch (...) {
  return raise_current();
}

PyObject* plans_size(PyObject* self_, PyObject*) {
  const auto* table = reinterpret_cast<Plans*>(self_)->table;
  return PyLong_FromSize_t(table == nullptr ? 0 : table->plans.size());
}

PyMethodDef plans_methods[] = {
    {"add", plans_add, METH_VARARGS, "add(tensors, scalars, args, inputs, outputs, workspace_offset, workspace_bytes, returns): "
     "remembers the call and makes it"},
    {"call", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(plans_call)), METH_FASTCALL,
     "call(tensors, scalars): the call's results, NotImplemented for layouts without a plan"},
    {"size", plans_size, METH_NOARGS, "remembered plans"},
    {nullptr, nullptr, 0, nullptr}};

PyType_Slot plans_slots[] = {{Py_tp_init, reinterpret_cast<void*>(plans_init)},
                             {Py_tp_dealloc, reinterpret_cast<void*>(plans_dealloc)},
                             {Py_tp_methods, plans_methods},
                             {Py_tp_new, reinterpret_cast<void*>(PyType_GenericNew)},
                             {0, nullptr}};
PyType_Spec plans_spec = {"b200k._plans.Plans", sizeof(Plans), 0, Py_TPFLAGS_DEFAULT, plans_slots};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_plans", "launch plans remembered by tensor layouts", -1, nullptr,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__plans(void) {
  PyObject* m = PyModule_Create(&module);
  if (m == nullptr) return nullptr;
  PyObject* type = PyType_FromSpec(&plans_spec);
  if (type == nullptr || PyModule_AddObject(m, "Plans", type) < 0) {
    Py_XDECREF(type);
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
