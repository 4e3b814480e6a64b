// Host side of the decoder-layer operators: what a call costs before its kernels are enqueued.
//
// Checking operands and choosing a launch in Python takes longer than a small launch.  A call is answered from a plan
// here: shapes, strides, types, devices and alignments of the operands and the values of the other arguments
// make a key, and a Python function (kernels.py) makes the plan of a new key, which is where every check of the
// operands lives.  A plan says which results and workspaces to allocate and which kernels to enqueue on
// the current stream, with the constant part of their argument segments packed.  Nothing about contents, addresses beyond
// their alignment, or identity is kept.
//
// Window attention with gradients is an autograd function over the same calls, so that the engine's thread runs
// no Python between two launches: short training steps are bound by that thread.
//
// What rides on torch's dispatcher (a tracer, a dispatch mode, a functorch transform, a tensor subclass) would see nothing
// of such a call but its allocations.  Where one is there the call goes to the registered op instead, which reaches
// run() below when it is time for the kernels.
//
// Python's lock is held wherever plans are touched.
#define PY_SSIZE_T_CLEAN
#include <torch/csrc/python_headers.h>

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <memory>
#include <string>
#include <unordered_map>
#include <vector>

namespace {

using LaunchFn = int (*)(void*, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, void*, const void*, size_t);

constexpr size_t kMaxPlans = 4096;  // of an operator; a server with ever new shapes starts over then
constexpr int kMaxArgs = 12, kMaxTensors = 24;

struct Launch {
  void* function;
  uint32_t dims[7];  // grid, block, LDS bytes
  std::string constants, name;
  std::vector<int> pointers;  // into operands, then outputs; -1: null
};

struct Output {
  std::vector<int64_t> sizes, strides;
  at::ScalarType dtype;
  bool zero;
};

struct Plan {
  std::vector<Launch> launches;
  std::vector<Output> outputs;
  int returned;  // leading outputs that the caller gets, the others are workspaces
};

struct KeyHash {
  size_t operator()(const std::vector<int64_t>& key) const {
    uint64_t h = 0x9e3779b97f4a7c15ull;
    for (int64_t x : key) {
      h = (h ^ static_cast<uint64_t>(x)) * 0xff51afd7ed558ccdull;
      h ^= h >> 32;
    }
    return h;
  }
};

struct Operator {
  PyObject *maker, *registered;  // the latter takes a call's arguments to the dispatcher
  int operands;  // bit i: argument i may be a tensor
  std::unordered_map<std::vector<int64_t>, std::shared_ptr<const Plan>, KeyHash> plans;
};

// An argument: a tensor, or a value that is part of the key
struct Arg {
  enum Kind : int64_t { kNone, kTensor, kInt, kFloat, kInts } kind = kNone;
  const at::Tensor* tensor = nullptr;
  bool subclass = false;  // of torch.Tensor in Python
  int64_t i = 0;
  double d = 0;
  std::vector<int64_t> list;

  Arg() = default;
  explicit Arg(const at::Tensor& t) : kind(t.defined() ? kTensor : kNone), tensor(&t) {}
  explicit Arg(int64_t x) : kind(kInt), i(x) {}
  explicit Arg(double x) : kind(kFloat), d(x) {}
};

LaunchFn g_launch = nullptr;
PyObject *g_launch_failed = nullptr, *g_launcher_dict = nullptr, *g_log_name = nullptr;
std::vector<std::unique_ptr<Operator>>& operators() {
  static auto* all = new std::vector<std::unique_ptr<Operator>>();  // never destroyed: plans may outlive the interpreter's end
  return *all;
}

[[noreturn]] void fail() {  // with Python's error set
  python_error e;
  e.persist();
  throw std::move(e);
}
[[noreturn]] void fail(PyObject* type, const char* text) {
  PyErr_SetString(type, text);
  fail();
}

struct Ref {  // an owned Python object
  PyObject* p;
  explicit Ref(PyObject* x) : p(x) {
    if (p == nullptr) fail();
  }
  Ref(const Ref&) = delete;
  ~Ref() { Py_DECREF(p); }
};

int64_t to_int(PyObject* o) {
  if (THPVariable_Check(o)) fail(PyExc_ValueError, "arguments that are no operands must be plain numbers, not tensors");
  Ref index(PyNumber_Index(o));
  const long long x = PyLong_AsLongLong(index.p);
  if (x == -1 && PyErr_Occurred()) fail();
  return x;
}

void parse(PyObject* o, bool operand, Arg& a) {
  if (THPVariable_Check(o)) {
    if (!operand) fail(PyExc_ValueError, "arguments that are no operands must be plain numbers, not tensors");
    a.kind = Arg::kTensor;
    a.tensor = &THPVariable_Unpack(o);
    a.subclass = !THPVariable_CheckExact(o);
  } else if (o == Py_None) {
    a.kind = Arg::kNone;
  } else if (PyFloat_Check(o)) {
    a.kind = Arg::kFloat;
    a.d = PyFloat_AS_DOUBLE(o);
  } else if (PyTuple_Check(o)) {
    a.kind = Arg::kInts;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(o); ++i) a.list.push_back(to_int(PyTuple_GET_ITEM(o, i)));
  } else if (PyIndex_Check(o)) {
    a.kind = Arg::kInt;
    a.i = to_int(o);
  } else {  // numbers of other libraries
    a.kind = Arg::kFloat;
    a.d = PyFloat_AsDouble(o);
    if (a.d == -1.0 && PyErr_Occurred()) fail();
  }
}

void add_to_key(std::vector<int64_t>& key, const Arg& a) {
  key.push_back(a.kind);
  switch (a.kind) {
    case Arg::kNone:
      break;
    case Arg::kTensor: {
      const at::Tensor& t = *a.tensor;
      const auto device = t.device();
      key.push_back(static_cast<int64_t>(t.scalar_type()) | static_cast<int64_t>(device.type()) << 8 |
                    static_cast<int64_t>(static_cast<uint8_t>(device.index())) << 16 | t.dim() << 24);
      key.push_back(reinterpret_cast<int64_t>(t.const_data_ptr()) & 15);
      for (int64_t x : t.sizes()) key.push_back(x);
      for (int64_t x : t.strides()) key.push_back(x);
      break;
    }
    case Arg::kInt:
      key.push_back(a.i);
      break;
    case Arg::kFloat: {
      int64_t bits;
      std::memcpy(&bits, &a.d, 8);
      key.push_back(bits);
      break;
    }
    case Arg::kInts:
      key.push_back(static_cast<int64_t>(a.list.size()));
      for (int64_t x : a.list) key.push_back(x);
  }
}

PyObject* to_python(const Arg& a) {
  switch (a.kind) {
    case Arg::kTensor:
      return THPVariable_Wrap(*a.tensor);
    case Arg::kInt:
      return PyLong_FromLongLong(a.i);
    case Arg::kFloat:
      return PyFloat_FromDouble(a.d);
    default:
      Py_RETURN_NONE;
  }
}

std::vector<int64_t> int_list(PyObject* o) {
  Ref fast(PySequence_Fast(o, "a sequence of integers"));
  std::vector<int64_t> out;
  for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(fast.p); ++i) out.push_back(to_int(PySequence_Fast_GET_ITEM(fast.p, i)));
  return out;
}

// plan: (launches, outputs, returned); launch: (function, grid and block and LDS bytes, constants, name, pointers);
// output: (sizes, strides, dtype, zero)
std::shared_ptr<const Plan> read_plan(PyObject* o) {
  auto plan = std::make_shared<Plan>();
  PyObject *launches, *outputs;
  if (!PyArg_ParseTuple(o, "O!O!i", &PyTuple_Type, &launches, &PyTuple_Type, &outputs, &plan->returned)) fail();
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(launches); ++i) {
    unsigned long long function;
    PyObject *dims, *pointers;
    const char *constants, *name;
    Py_ssize_t size;
    if (!PyArg_ParseTuple(PyTuple_GET_ITEM(launches, i), "KOy#sO", &function, &dims, &constants, &size, &name, &pointers)) fail();
    Launch l;
    l.function = reinterpret_cast<void*>(function);
    const auto d = int_list(dims);
    for (int j = 0; j < 7; ++j) {
      if (d.size() != 7 || d[j] < 0 || d[j] > 0x7fffffff) fail(PyExc_ValueError, "a launch has seven dimensions that fit 31 bits");
      l.dims[j] = static_cast<uint32_t>(d[j]);
    }
    l.constants.assign(constants, size);
    l.name = name;
    for (int64_t x : int_list(pointers)) l.pointers.push_back(static_cast<int>(x));
    plan->launches.push_back(std::move(l));
  }
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(outputs); ++i) {
    PyObject *sizes, *strides, *dtype;
    int zero;
    if (!PyArg_ParseTuple(PyTuple_GET_ITEM(outputs, i), "OOO!p", &sizes, &strides, reinterpret_cast<PyObject*>(&THPDtypeType), &dtype, &zero))
      fail();
    plan->outputs.push_back({int_list(sizes), int_list(strides), reinterpret_cast<THPDtype*>(dtype)->scalar_type, zero != 0});
  }
  return plan;
}

// Whether somebody has to see this call through the dispatcher.  Tensors whose numbers are not those in their memory
// (a negative view) are made plain there too.
bool watched(const Arg* args, int n) {
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet rides({DispatchKey::Python, DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper,
                                       DispatchKey::BatchedNestedTensor, DispatchKey::Functionalize, DispatchKey::Conjugate,
                                       DispatchKey::Negative, DispatchKey::ZeroTensor});
  constexpr c10::DispatchKeySet here({DispatchKey::FuncTorchDynamicLayerFrontMode, DispatchKey::Functionalize, DispatchKey::PreDispatch});
  if (c10::impl::TorchDispatchModeTLS::any_modes_set() || c10::impl::tls_local_dispatch_key_set().included_.has_any(here) ||
      torch::jit::tracer::isTracing())
    return true;
  for (int i = 0; i < n; ++i)
    if (args[i].kind == Arg::kTensor && (args[i].subclass || args[i].tensor->key_set().has_any(rides))) return true;
  return false;
}

// The arguments as a tuple
PyObject* given(const Arg* args, int n, PyObject* const* objects) {
  Ref tuple(PyTuple_New(n));
  for (int i = 0; i < n; ++i) {
    PyObject* o = objects ? Py_NewRef(objects[i]) : to_python(args[i]);
    if (o == nullptr) fail();
    PyTuple_SET_ITEM(tuple.p, i, o);
  }
  return Py_NewRef(tuple.p);
}

// The outputs of a call (workspaces behind the returned ones); throws python_error.
void run(int which, const Arg* args, int n, PyObject* const* objects, std::vector<at::Tensor>& outs, int& returned) {
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode())
    for (int i = 0; i < n; ++i)
      if (args[i].kind == Arg::kTensor && args[i].tensor->_fw_grad(0).defined())  // a result without its tangent would read as constant
        fail(PyExc_NotImplementedError, "no forward-mode derivative here (decoder.rotary_axes has one outside of transforms)");
  Operator& op = *operators()[which];
  std::vector<int64_t> key;
  key.reserve(128);
  for (int i = 0; i < n; ++i) add_to_key(key, args[i]);
  std::shared_ptr<const Plan> plan;
  if (auto at = op.plans.find(key); at != op.plans.end()) {
    plan = at->second;
  } else {
    Ref arguments(given(args, n, objects));
    Ref made(PyObject_Call(op.maker, arguments.p, nullptr));
    plan = read_plan(made.p);
    const at::Tensor* tensors = nullptr;
    int count = static_cast<int>(plan->outputs.size());
    for (int i = 0; i < n; ++i) {
      if (op.operands >> i & 1) ++count;
      if (args[i].kind == Arg::kTensor && tensors == nullptr) tensors = args[i].tensor;
    }
    for (const Launch& l : plan->launches)
      for (int p : l.pointers)
        if (p < -1 || p >= count) fail(PyExc_ValueError, "a plan points past its tensors");
    if (tensors == nullptr || count > kMaxTensors) fail(PyExc_ValueError, "a plan needs an operand, and at most 24 tensors");
    if (op.plans.size() >= kMaxPlans) op.plans.clear();
    op.plans.emplace(std::move(key), plan);
  }

  const at::Tensor* first = nullptr;
  void* pointers[kMaxTensors];
  int tensors = 0;
  for (int i = 0; i < n; ++i) {
    if (!(op.operands >> i & 1)) continue;
    const bool there = args[i].kind == Arg::kTensor;
    if (there && first == nullptr) first = args[i].tensor;
    pointers[tensors++] = there ? const_cast<void*>(args[i].tensor->const_data_ptr()) : nullptr;
  }
  void* stream = nullptr;
  if (!plan->launches.empty()) {
    if (!first->is_cuda() || first->device().index() != c10::hip::current_device())
      fail(PyExc_ValueError, "tensors must live on the current GPU");
    stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(first->device().index()).stream();
  }
  for (const Output& o : plan->outputs) {
    outs.push_back(at::empty_strided(o.sizes, o.strides, first->options().dtype(o.dtype)));
    if (o.zero) outs.back().zero_();
    pointers[tensors++] = outs.back().data_ptr();
  }
  returned = plan->returned;
  if (plan->launches.empty()) return;
  PyObject* log = PyDict_GetItem(g_launcher_dict, g_log_name);  // borrowed
  char segment[1024];
  for (const Launch& l : plan->launches) {
    const size_t lead = 8 * l.pointers.size(), size = lead + l.constants.size();
    if (size > sizeof(segment)) fail(PyExc_ValueError, "a kernel's arguments must fit 1024 bytes");
    for (size_t i = 0; i < l.pointers.size(); ++i) {
      void* p = l.pointers[i] < 0 ? nullptr : pointers[l.pointers[i]];
      std::memcpy(segment + 8 * i, &p, 8);
    }
    std::memcpy(segment + lead, l.constants.data(), l.constants.size());
    if (log != nullptr && PyList_Check(log)) {
      Ref name(PyUnicode_FromString(l.name.c_str()));
      if (PyList_Append(log, name.p) != 0) fail();
    }
    const uint32_t* d = l.dims;
    const int err = g_launch(l.function, d[0], d[1], d[2], d[3], d[4], d[5], d[6], stream, segment, size);
    if (err != 0) {
      Ref raised(PyObject_CallFunction(g_launch_failed, "s(III)(III)Ii", l.name.c_str(), d[0], d[1], d[2], d[3], d[4], d[5], d[6], err));
      fail(PyExc_RuntimeError, "a launch failed");
    }
  }
}

// run(), or the registered op where somebody watches
void call(int which, const Arg* args, int n, PyObject* const* objects, std::vector<at::Tensor>& outs, int& returned) {
  if (!watched(args, n)) return run(which, args, n, objects, outs, returned);
  Ref arguments(given(args, n, objects));
  Ref result(PyObject_Call(operators()[which]->registered, arguments.p, nullptr));
  if (THPVariable_Check(result.p)) {
    outs.push_back(THPVariable_Unpack(result.p));
  } else {
    Ref all(PySequence_Fast(result.p, "tensors"));
    for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(all.p); ++i) {
      PyObject* o = PySequence_Fast_GET_ITEM(all.p, i);
      if (!THPVariable_Check(o)) fail(PyExc_TypeError, "an operator returns tensors");
      outs.push_back(THPVariable_Unpack(o));
    }
  }
  returned = static_cast<int>(outs.size());
}

// An incoming gradient as the kernels take it, with contiguous columns in 16-byte aligned rows: it may arrive in any
// layout (a sum's is one number everywhere) and at any address.
at::Tensor placed(const at::Tensor& dout) {
  bool fits = dout.dim() == 4 && dout.stride(3) == 1 && (reinterpret_cast<uintptr_t>(dout.const_data_ptr()) & 15) == 0;
  for (int i = 0; fits && i < 3; ++i) fits = dout.size(i) == 1 || dout.stride(i) % 8 == 0;
  return fits ? dout : dout.clone(at::MemoryFormat::Contiguous);
}

enum { kWindowForward, kWindowBackward };
int g_window[2] = {-1, -1};
PyObject* g_window_registered = nullptr;  // the op with its gradient

class WindowAttention : public torch::autograd::Function<WindowAttention> {
 public:
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            const std::optional<at::Tensor>& given_lengths, double scale, int64_t window, int64_t sinks) {
    const at::Tensor lengths = given_lengths.value_or(at::Tensor());
    const Arg args[] = {Arg(q), Arg(k), Arg(v), Arg(scale), Arg(window), Arg(sinks), Arg(lengths), Arg(int64_t{1})};
    std::vector<at::Tensor> outs;
    int returned;
    run(g_window[kWindowForward], args, 8, nullptr, outs, returned);  // py_window_attention looked for watchers
    ctx->save_for_backward({q, k, v, outs[0], outs[1], outs[2], lengths});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    return outs[0];
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    at::Tensor dout = grads[0];
    torch::autograd::variable_list given(7);
    if (!dout.defined()) return given;
    const Arg seen(dout);
    if (!watched(&seen, 1)) dout = placed(dout);  // else the op's implementation does
    const Arg args[] = {Arg(saved[0]), Arg(saved[1]), Arg(saved[2]), Arg(saved[3]), Arg(dout), Arg(saved[4]),
                        Arg(ctx->saved_data["scale"].toDouble()), Arg(ctx->saved_data["window"].toInt()),
                        Arg(ctx->saved_data["sinks"].toInt()), Arg(saved[6]), Arg(saved[5])};
    std::vector<at::Tensor> outs;
    int returned;
    {
      pybind11::gil_scoped_acquire lock;
      call(g_window[kWindowBackward], args, 11, nullptr, outs, returned);
    }
    torch::autograd::variable_list result(outs.begin(), outs.begin() + 3);
    if (at::GradMode::is_enabled()) {  // the kernels leave no graph behind: a gradient of these must not come out as none
      for (auto& t : result) t.set_requires_grad(true);
      auto refuse = std::make_shared<torch::autograd::DelayedError>(
          "trying to differentiate twice a function that was marked with @once_differentiable", 3);
      result = (*refuse)(std::move(result));
    }
    for (int i = 0; i < 3; ++i) given[i] = result[i];
    return given;
  }
};

PyObject* py_bind(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  unsigned long long address;
  PyObject *failed, *dict;
  if (!PyArg_ParseTuple(args, "KOO!", &address, &failed, &PyDict_Type, &dict)) return nullptr;
  g_launch = reinterpret_cast<LaunchFn>(address);
  g_launch_failed = Py_NewRef(failed);
  g_launcher_dict = Py_NewRef(dict);
  g_log_name = PyUnicode_InternFromString("launch_log");
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* py_operator(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *maker, *operands, *registered;
  if (!PyArg_ParseTuple(args, "OOO", &maker, &operands, &registered)) return nullptr;
  auto op = std::make_unique<Operator>();
  op->maker = Py_NewRef(maker);
  op->registered = Py_NewRef(registered);
  op->operands = 0;
  for (int64_t i : int_list(operands)) op->operands |= 1 << i;
  operators().push_back(std::move(op));
  return PyLong_FromSize_t(operators().size() - 1);
  END_HANDLE_TH_ERRORS
}

PyObject* py_window(PyObject*, PyObject* args) {
  PyObject* registered;
  if (!PyArg_ParseTuple(args, "iiO", &g_window[kWindowForward], &g_window[kWindowBackward], &registered)) return nullptr;
  g_window_registered = Py_NewRef(registered);
  Py_RETURN_NONE;
}

PyObject* py_forget(PyObject*, PyObject*) {
  for (auto& op : operators()) op->plans.clear();
  Py_RETURN_NONE;
}

PyObject* call_or_run(PyObject* const* objects, Py_ssize_t nargs, bool kernels) {
  HANDLE_TH_ERRORS
  const int64_t which = nargs > 0 ? to_int(objects[0]) : -1;
  const int n = static_cast<int>(nargs) - 1;
  if (which < 0 || which >= static_cast<int64_t>(operators().size()) || n > kMaxArgs || g_launch == nullptr)
    fail(PyExc_TypeError, "call(operator, at most 12 arguments) after bind()");
  Arg args[kMaxArgs];
  for (int i = 0; i < n; ++i) parse(objects[1 + i], operators()[which]->operands >> i & 1, args[i]);
  std::vector<at::Tensor> outs;
  outs.reserve(8);
  int returned;
  (kernels ? run : call)(static_cast<int>(which), args, n, objects + 1, outs, returned);
  if (returned == 1) return THPVariable_Wrap(outs[0]);
  Ref result(PyTuple_New(returned));
  for (int i = 0; i < returned; ++i) {
    PyObject* o = THPVariable_Wrap(outs[i]);
    if (o == nullptr) return nullptr;
    PyTuple_SET_ITEM(result.p, i, o);
  }
  return Py_NewRef(result.p);
  END_HANDLE_TH_ERRORS
}

PyObject* py_call(PyObject*, PyObject* const* objects, Py_ssize_t nargs) { return call_or_run(objects, nargs, false); }
PyObject* py_run(PyObject*, PyObject* const* objects, Py_ssize_t nargs) { return call_or_run(objects, nargs, true); }

PyObject* py_placed(PyObject*, PyObject* o) {
  HANDLE_TH_ERRORS
  if (!THPVariable_Check(o)) fail(PyExc_TypeError, "placed() takes a tensor");
  return THPVariable_Wrap(placed(THPVariable_Unpack(o)));
  END_HANDLE_TH_ERRORS
}

// watched(operands or None ...): whether a call with them goes through the dispatcher
PyObject* py_watched(PyObject*, PyObject* const* objects, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Arg args[kMaxArgs];
  if (nargs > kMaxArgs) fail(PyExc_TypeError, "watched() takes at most 12 operands");
  for (Py_ssize_t i = 0; i < nargs; ++i) parse(objects[i], true, args[i]);
  return PyBool_FromLong(watched(args, static_cast<int>(nargs)));
  END_HANDLE_TH_ERRORS
}

// window_attention_with_gradients(q, k, v, scale, window, sinks, lengths or None) -> out
PyObject* py_window_attention(PyObject*, PyObject* const* objects, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 7 || g_window[0] < 0) fail(PyExc_TypeError, "window_attention_with_gradients() takes 7 arguments");
  Arg a[7];
  for (int i = 0; i < 7; ++i) parse(objects[i], i < 3 || i == 6, a[i]);
  for (int i = 0; i < 3; ++i)
    if (a[i].kind != Arg::kTensor) fail(PyExc_TypeError, "q, k and v must be tensors");
  if (a[6].kind != Arg::kTensor && a[6].kind != Arg::kNone) fail(PyExc_TypeError, "lengths must be a tensor or None");
  if (a[3].kind == Arg::kInt) a[3].d = static_cast<double>(a[3].i);
  if ((a[3].kind != Arg::kInt && a[3].kind != Arg::kFloat) || a[4].kind != Arg::kInt || a[5].kind != Arg::kInt)
    fail(PyExc_TypeError, "scale must be a number, window and sinks integers");
  if (watched(a, 7)) return PyObject_Vectorcall(g_window_registered, objects, nargs, nullptr);
  std::optional<at::Tensor> lengths;
  if (a[6].kind == Arg::kTensor) lengths = *a[6].tensor;
  return THPVariable_Wrap(WindowAttention::apply(*a[0].tensor, *a[1].tensor, *a[2].tensor, lengths, a[3].d, a[4].i, a[5].i));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", py_bind, METH_VARARGS, "bind(address of mi_launch_packed, raise function for a failed launch, the launcher's namespace)"},
    {"operator", py_operator, METH_VARARGS, "operator(plan maker, indices of the arguments that may be tensors, the registered op) -> its number"},
    {"window", py_window, METH_VARARGS, "window(numbers of window attention's forward and backward, the registered op with its gradient)"},
    {"forget", py_forget, METH_NOARGS, "drop every plan"},
    {"call", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_call)), METH_FASTCALL, "call(operator, *arguments) -> its results"},
    {"run", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_run)), METH_FASTCALL,
     "run(operator, *arguments) -> its results, by the kernels whoever watches"},
    {"watched", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_watched)), METH_FASTCALL,
     "watched(*operands) -> whether a call with them goes to the registered op"},
    {"placed", py_placed, METH_O, "placed(gradient of an output) -> it, or a copy where the kernels do not take its layout or address"},
    {"window_attention_with_gradients", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_window_attention)), METH_FASTCALL,
     "window_attention_with_gradients(q, k, v, scale, window, sinks, lengths) -> out"},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mi_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mi_ops(void) { return PyModule_Create(&module); }
