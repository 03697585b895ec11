// luma_torch.cpp — the Python module luma_b200._grads_ext: lists of torch
// tensors for the gradient operators of include/luma_b200.h.
//
// A call on thousands of small gradients is bound by the host: reading each
// tensor's address, size, type, device and layout from Python costs about
// 0.6 us a tensor (7.1 ms of a 7.1 ms call on 10,000 tensors), here some tens
// of nanoseconds.  The module checks a list, allocates the results and the
// workspace from torch's allocator on the current stream, and makes the one
// library call; luma_b200/grads.py has the functions that users call.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <vector>

#include "luma_b200.h"

namespace {

// An owned Python reference.
struct Ref {
  PyObject* o;
  explicit Ref(PyObject* p = nullptr) : o(p) {}
  Ref(Ref&& r) noexcept : o(r.o) { r.o = nullptr; }
  Ref(const Ref&) = delete;
  ~Ref() { Py_XDECREF(o); }
};

[[noreturn]] void raise(PyObject* kind, const std::string& msg) {
  PyErr_SetString(kind, msg.c_str());
  throw python_error();
}

struct List {
  std::vector<const at::Tensor*> t;
  std::vector<uint64_t> ptr;
  std::vector<int64_t> numel;
  std::vector<uint8_t> code;
  c10::Device device{c10::kCPU};
  std::vector<std::pair<int64_t, PyObject*>> wrapped;  // DTensors, by their place in the list
  std::vector<Ref> keep;  // the sequence, and what its items were unwrapped to

  bool sharded() const { return !wrapped.empty(); }
  int64_t n() const { return (int64_t)t.size(); }
};

// Whether the elements are numel consecutive ones in some order of the
// dimensions (a transposed or channels-last gradient).
bool dense(const at::Tensor& t) {
  if (t.is_contiguous() || t.numel() <= 1) return true;
  std::vector<std::pair<int64_t, int64_t>> d;
  for (int64_t k = 0; k < t.dim(); ++k)
    if (t.size(k) != 1) d.emplace_back(t.stride(k), t.size(k));
  std::sort(d.begin(), d.end());
  int64_t room = 1;
  for (const auto& [stride, size] : d) {
    if (stride != room) return false;
    room *= size;
  }
  return true;
}

// Whether two dense tensors of one shape have their elements in one order.  A
// dimension of size 1 has no place in it, whatever its stride.
bool same_order(const at::Tensor& x, const at::Tensor& y) {
  for (int64_t k = 0; k < x.dim(); ++k)
    if (x.size(k) != 1 && x.stride(k) != y.stride(k)) return false;
  return true;
}

std::string shape_text(c10::IntArrayRef v) {
  std::string s = "(";
  for (size_t k = 0; k < v.size(); ++k) s += (k ? ", " : "") + std::to_string(v[k]);
  return s + (v.size() == 1 ? ",)" : ")");
}

void add(List& l, const at::Tensor& t, const char* name, bool written) {
  if (t.layout() != c10::kStrided)
    raise(PyExc_RuntimeError, std::string("LUMA does not support sparse gradients (") + name + ")");
  uint8_t code;
  switch (t.scalar_type()) {
    case at::kFloat: code = LUMA_F32; break;
    case at::kBFloat16: code = LUMA_BF16; break;
    case at::kHalf: code = LUMA_F16; break;
    default: {
      std::string type = c10::toString(t.scalar_type());
      std::transform(type.begin(), type.end(), type.begin(), ::tolower);
      if (type == "double") type = "float64";
      if (type == "short") type = "int16";
      raise(PyExc_ValueError, std::string(name) + " must be float32/bfloat16/float16 tensors (got " +
                                  type + ")");
    }
  }
  if (!t.is_cuda())
    raise(PyExc_RuntimeError, std::string("LUMA backend 'cuda' requires CUDA tensors (") + name +
                                  " on " + t.device().str() + ")");
  if (!dense(t))
    raise(PyExc_ValueError, std::string(name) + " must be dense in memory (got strides " +
                                shape_text(t.strides()) + " for shape " + shape_text(t.sizes()) +
                                ")");
  if (l.t.empty()) l.device = t.device();
  else if (t.device() != l.device)
    raise(PyExc_ValueError, std::string(name) + " must be on one device (got " + l.device.str() +
                                " and " + t.device().str() + ")");
  const int64_t n = t.numel();
  l.t.push_back(&t);
  l.numel.push_back(n);
  l.code.push_back(code);
  l.ptr.push_back(n == 0 ? 0
                         : reinterpret_cast<uint64_t>(written ? t.mutable_data_ptr()
                                                              : t.const_data_ptr()));
}

// The tensors of a Python iterable (or one tensor), checked.
void collect(List& l, PyObject* o, const char* name, bool written) {
  if (THPVariable_Check(o)) {
    Py_INCREF(o);
    l.keep.emplace_back(o);
    Ref one(PyTuple_Pack(1, o));
    if (one.o == nullptr) throw python_error();
    l.keep.push_back(std::move(one));
  } else {
    Ref seq(PySequence_Fast(o, (std::string(name) + " must be tensors").c_str()));
    if (seq.o == nullptr) throw python_error();
    // a list may be changed by the attribute lookups below: keep its items
    if (PyList_Check(seq.o)) {
      Ref t(PyList_AsTuple(seq.o));
      if (t.o == nullptr) throw python_error();
      l.keep.push_back(std::move(t));
    } else {
      l.keep.push_back(std::move(seq));
    }
  }
  PyObject* items = l.keep.back().o;
  const Py_ssize_t n = PyTuple_GET_SIZE(items);
  l.t.reserve(n);
  l.ptr.reserve(n);
  l.numel.reserve(n);
  l.code.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* item = PyTuple_GET_ITEM(items, i);
    if (!THPVariable_CheckExact(item)) {
      if (!THPVariable_Check(item))
        raise(PyExc_TypeError, std::string(name) + "[" + std::to_string(i) + "] is " +
                                   Py_TYPE(item)->tp_name + ", not a tensor");
      if (PyObject_HasAttrString(item, "_local_tensor")) {  // DTensor: this rank's shard
        Ref local(PyObject_GetAttrString(item, "_local_tensor"));
        if (local.o == nullptr) throw python_error();
        if (!THPVariable_Check(local.o)) raise(PyExc_TypeError, "_local_tensor is not a tensor");
        l.wrapped.emplace_back((int64_t)i, item);
        item = local.o;
        l.keep.push_back(std::move(local));
      }
    }
    add(l, THPVariable_Unpack(item), name, written);
  }
}

at::Tensor scalar(const List& l) {
  return at::empty({}, at::TensorOptions().dtype(at::kFloat).device(l.device));
}

struct Call {
  LumaGradArgs a{};
  at::Tensor workspace;
};

void set_list(Call& c, const List& l) {
  c.a.grads = l.ptr.data();
  c.a.numel = l.numel.data();
  c.a.dtypes = l.code.data();
  c.a.n = l.n();
  c.a.device = l.device.index();
  c.a.host_scale = 1.0f;
}

// Partial results of one call: memory of the current stream (of the graph,
// during a capture), so calls that overlap on the GPU never share it.
void set_workspace(Call& c, const List& l) {
  c.workspace = at::empty({LUMA_GRAD_PARTIALS(l.n())},
                          at::TensorOptions().dtype(at::kDouble).device(l.device));
  c.a.partials = static_cast<double*>(c.workspace.mutable_data_ptr());
  c.a.n_partials = c.workspace.numel();
}

void launch(const char* name, int (*fn)(const LumaGradArgs*, void*), const Call& c) {
  const int status = fn(&c.a, c10::cuda::getCurrentCUDAStream(c.a.device).stream());
  if (status == LUMA_OK) return;
  PyObject* kind = status == LUMA_ERR_INVALID ? PyExc_ValueError : PyExc_RuntimeError;
  Ref lib(PyImport_ImportModule("luma_b200._lib"));
  if (lib.o == nullptr) throw python_error();
  Ref own(PyObject_GetAttrString(lib.o, "LumaError"));
  if (own.o == nullptr) throw python_error();
  raise(status == LUMA_ERR_CUDA ? own.o : kind, std::string(name) + " failed (status " +
            std::to_string(status) + "): " + luma_last_error());
}

// Tell autograd that the tensors changed, as its own in-place operations do.
// A DTensor has a version of its own beside its local tensor's.
void written(const List& l) {
  const auto bump = [](const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  };
  for (const at::Tensor* t : l.t) bump(*t);
  for (const auto& [i, wrapper] : l.wrapped) bump(THPVariable_Unpack(wrapper));
}

// A one-element tensor's address.  That of a wrapper without memory of its own
// is 0, which the library takes for "no factor" or "no flag".
template <class T>
T* address(T* p, const char* name) {
  if (p == nullptr)
    raise(PyExc_ValueError, std::string(name) + " is a tensor without memory of its own");
  return p;
}

const at::Tensor& device_scalar(PyObject* o, const List& l, const char* name) {
  const at::Tensor* t = THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
  if (t == nullptr || t->layout() != c10::kStrided || t->numel() != 1 ||
      t->scalar_type() != at::kFloat || !t->is_cuda())
    raise(PyExc_ValueError,
          std::string(name) + " must be a one-element float32 CUDA tensor");
  if (t->device() != l.device)
    raise(PyExc_ValueError, std::string(name) + " must be on the gradients' device");
  return *t;
}

// A factor that the kernels read; `hold` keeps it.  A negated view's memory
// holds minus its value.
const float* reciprocal(PyObject* o, const List& l, const char* name, at::Tensor& hold) {
  if (o == Py_None) return nullptr;
  hold = device_scalar(o, l, name);
  if (hold.is_neg()) hold = hold.detach().resolve_neg();
  return static_cast<const float*>(address(hold.const_data_ptr(), name));
}

// A flag that they write.
float* flag(PyObject* o, const List& l, const char* name) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = device_scalar(o, l, name);
  if (t.is_neg()) raise(PyExc_ValueError, std::string(name) + " must not be a negated view");
  return static_cast<float*>(address(t.mutable_data_ptr(), name));
}

// A factor given as a number or a one-element tensor; `hold` keeps the tensor
// that the kernels read, where it lies on a GPU.
void factor(PyObject* o, const List& l, const char* name, Call& c, at::Tensor& hold) {
  if (!THPVariable_Check(o)) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    c.a.host_scale = (float)v;
    return;
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.layout() != c10::kStrided || t.numel() != 1 ||
      (t.scalar_type() != at::kFloat && t.scalar_type() != at::kBFloat16 &&
       t.scalar_type() != at::kHalf))
    raise(PyExc_ValueError, std::string(name) + " must be a number or a one-element float32, "
                                                "bfloat16 or float16 tensor");
  if (t.is_cpu()) {
    // read now: a copy would be queued, and read what is written here meanwhile
    // (in a captured call, before a replay)
    c.a.host_scale = t.item<float>();
    return;
  }
  hold = t.detach();
  if (hold.is_neg() || hold.scalar_type() != at::kFloat || hold.device() != l.device)
    hold = hold.resolve_neg().to(at::TensorOptions().dtype(at::kFloat).device(l.device), true);
  c.a.scale = static_cast<const float*>(address(hold.const_data_ptr(), name));
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}

void arity(const char* name, Py_ssize_t got, Py_ssize_t want) {
  if (got != want)
    raise(PyExc_TypeError, std::string(name) + ": " + std::to_string(want) + " arguments");
}

// (norm, coef or None, norms or None); clip: the grads are scaled in place.
// None where the list is empty.  Sharded lists are refused: their norm takes
// a process group.
PyObject* py_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  // grads, kind, max_norm or None, per_tensor, inv_scale, found_inf, clip
  arity("norm", n, 7);
  const bool clip = truth(args[6]);
  List l;
  collect(l, args[0], "grads", clip);
  if (l.sharded())
    raise(PyExc_ValueError, "the gradients are sharded (DTensor): pass process_group, over whose "
                            "ranks the norm is taken (per_tensor norms are of whole tensors)");
  if (l.n() == 0) Py_RETURN_NONE;
  Call c;
  set_list(c, l);
  c.a.norm_kind = (int32_t)PyLong_AsLong(args[1]);
  at::Tensor hold;
  c.a.inv_scale = reciprocal(args[4], l, "inv_scale", hold);
  c.a.found_inf = flag(args[5], l, "found_inf");
  at::Tensor norm = scalar(l), coef, norms;
  c.a.norm = norm.mutable_data_ptr<float>();
  if (args[2] != Py_None) {
    c.a.max_norm = PyFloat_AsDouble(args[2]);
    coef = scalar(l);
    c.a.coef = coef.mutable_data_ptr<float>();
  }
  if (PyErr_Occurred()) throw python_error();
  if (truth(args[3])) {
    norms = at::empty({l.n()}, norm.options());
    c.a.norms = norms.mutable_data_ptr<float>();
  }
  set_workspace(c, l);
  if (clip) {
    launch("luma_grad_clip", luma_grad_clip, c);
    written(l);
  } else {
    launch("luma_grad_norm", luma_grad_norm, c);
  }
  Ref out(PyTuple_New(3));
  if (out.o == nullptr) throw python_error();
  const at::Tensor* parts[3] = {&norm, &coef, &norms};
  for (int k = 0; k < 3; ++k) {
    PyObject* v = parts[k]->defined() ? THPVariable_Wrap(*parts[k]) : Py_NewRef(Py_None);
    if (v == nullptr) throw python_error();
    PyTuple_SET_ITEM(out.o, k, v);
  }
  return std::exchange(out.o, nullptr);
  END_HANDLE_TH_ERRORS
}

// The sum of powers (or the maximum) of a rank's shards, one float64 on their
// device; 0 on the current device where the list is empty.  None where there
// are DTensors: which ranks count them is the caller's to say.
PyObject* py_power(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity("power", n, 2);  // grads, kind
  List l;
  collect(l, args[0], "grads", false);
  if (l.n() == 0)
    return THPVariable_Wrap(at::zeros({1}, at::TensorOptions().dtype(at::kDouble).device(
        c10::Device(c10::kCUDA, c10::cuda::current_device()))));
  if (l.sharded()) Py_RETURN_NONE;
  Call c;
  set_list(c, l);
  c.a.norm_kind = (int32_t)PyLong_AsLong(args[1]);
  if (PyErr_Occurred()) throw python_error();
  at::Tensor power = at::empty({1}, at::TensorOptions().dtype(at::kDouble).device(l.device));
  c.a.power = power.mutable_data_ptr<double>();
  set_workspace(c, l);
  launch("luma_grad_norm", luma_grad_norm, c);
  return THPVariable_Wrap(power);
  END_HANDLE_TH_ERRORS
}

// (norm, coef or None) of a power that was reduced over ranks.
PyObject* py_finish(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity("finish", n, 5);  // power, kind, max_norm or None, inv_scale, found_inf
  const at::Tensor& power = THPVariable_Unpack(args[0]);
  List l;
  l.device = power.device();
  Call c;
  c.a.device = l.device.index();
  c.a.partials = power.mutable_data_ptr<double>();
  c.a.n_partials = 1;
  c.a.norm_kind = (int32_t)PyLong_AsLong(args[1]);
  at::Tensor norm = scalar(l), coef;
  c.a.norm = norm.mutable_data_ptr<float>();
  if (args[2] != Py_None) {
    c.a.max_norm = PyFloat_AsDouble(args[2]);
    coef = scalar(l);
    c.a.coef = coef.mutable_data_ptr<float>();
  }
  if (PyErr_Occurred()) throw python_error();
  at::Tensor hold;
  c.a.inv_scale = reciprocal(args[3], l, "inv_scale", hold);
  c.a.found_inf = flag(args[4], l, "found_inf");
  launch("luma_grad_finish", luma_grad_finish, c);
  Ref first(THPVariable_Wrap(norm));
  Ref second(coef.defined() ? THPVariable_Wrap(coef) : Py_NewRef(Py_None));
  if (first.o == nullptr || second.o == nullptr) throw python_error();
  return PyTuple_Pack(2, first.o, second.o);
  END_HANDLE_TH_ERRORS
}

PyObject* py_scale(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity("scale", n, 2);  // grads, coef
  List l;
  collect(l, args[0], "grads", true);
  if (l.n() == 0) Py_RETURN_NONE;
  Call c;
  set_list(c, l);
  at::Tensor hold;
  factor(args[1], l, "coef", c, hold);
  launch("luma_grad_scale", luma_grad_scale, c);
  written(l);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// Two DTensors of an accumulation hold the same part of tensors of one shape.
void same_part(int64_t i, PyObject* acc, PyObject* grad) {
  const std::string at = "[" + std::to_string(i) + "]";
  const std::string both = "acc" + at + " and grads" + at + " differ in ";
  const at::Tensor &x = THPVariable_Unpack(acc), &y = THPVariable_Unpack(grad);
  if (x.sizes() != y.sizes())
    raise(PyExc_ValueError, both + "shape (got " + shape_text(x.sizes()) + " and " +
                                shape_text(y.sizes()) + ")");
  for (const char* name : {"device_mesh", "placements"}) {
    Ref a(PyObject_GetAttrString(acc, name)), b(PyObject_GetAttrString(grad, name));
    if (a.o == nullptr || b.o == nullptr) throw python_error();
    const int same = PyObject_RichCompareBool(a.o, b.o, Py_EQ);
    if (same < 0) throw python_error();
    if (same) continue;
    Ref s(PyUnicode_FromFormat("%s%s (got %S and %S)", both.c_str(), name, a.o, b.o));
    if (s.o == nullptr) throw python_error();
    PyErr_SetObject(PyExc_ValueError, s.o);
    throw python_error();
  }
}

// (norm or None, coef or None); None where the lists are empty.
PyObject* py_accumulate(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity("accumulate", n, 6);  // acc, grads, scale, overwrite, kind, max_norm or None
  List d, s;
  collect(d, args[0], "acc", true);
  collect(s, args[1], "grads", false);
  if (d.n() != s.n())
    raise(PyExc_ValueError, "acc and grads must be as long as one another (got " +
                                std::to_string(d.n()) + " and " + std::to_string(s.n()) +
                                " tensors)");
  Call c;
  set_list(c, s);
  c.a.accs = d.ptr.data();
  c.a.acc_dtypes = d.code.data();
  c.a.overwrite = truth(args[3]);
  c.a.norm_kind = (int32_t)PyLong_AsLong(args[4]);
  if (PyErr_Occurred()) throw python_error();
  const bool norms = c.a.norm_kind != LUMA_NORM_NONE;
  if (norms && (d.sharded() || s.sharded()))
    raise(PyExc_ValueError, "the norm of sharded accumulators (DTensor): accumulate without one, "
                            "then clip_coef(acc, ..., process_group=...)");
  if (d.n() == 0) Py_RETURN_NONE;
  if (s.device != d.device) raise(PyExc_ValueError, "acc and grads must be on one device");
  for (auto x = d.wrapped.begin(), y = s.wrapped.begin();
       x != d.wrapped.end() && y != s.wrapped.end();) {
    if (x->first < y->first) ++x;
    else if (y->first < x->first) ++y;
    else same_part(x->first, x->second, y->second), ++x, ++y;
  }
  for (int64_t i = 0; i < d.n(); ++i) {
    const at::Tensor &x = *d.t[i], &y = *s.t[i];
    if (d.code[i] == LUMA_F16)
      raise(PyExc_ValueError, "acc must be float32 or bfloat16 tensors (got float16)");
    const bool shapes = x.sizes() == y.sizes();
    const bool orders = (x.is_contiguous() && y.is_contiguous()) || (shapes && same_order(x, y));
    if (shapes && orders && x.is_neg() == y.is_neg()) continue;
    const std::string at_i = "[" + std::to_string(i) + "]";
    const std::string both = "acc" + at_i + " and grads" + at_i;
    if (!shapes)
      raise(PyExc_ValueError, both + " differ in shape (got " + shape_text(x.sizes()) + " and " +
                                  shape_text(y.sizes()) + ")");
    if (!orders)
      raise(PyExc_ValueError, both + " differ in the order of their dimensions in memory (strides " +
                                  shape_text(x.strides()) + " and " + shape_text(y.strides()) +
                                  ")");
    raise(PyExc_ValueError, "acc" + at_i + " or grads" + at_i + " is a negated view");
  }
  at::Tensor hold, norm, coef;
  factor(args[2], d, "scale", c, hold);
  if (norms) {
    norm = scalar(d);
    c.a.norm = norm.mutable_data_ptr<float>();
    if (args[5] != Py_None) {
      c.a.max_norm = PyFloat_AsDouble(args[5]);
      if (PyErr_Occurred()) throw python_error();
      coef = scalar(d);
      c.a.coef = coef.mutable_data_ptr<float>();
    }
    set_workspace(c, d);
  }
  launch("luma_grad_accumulate", luma_grad_accumulate, c);
  written(d);
  Ref first(norm.defined() ? THPVariable_Wrap(norm) : Py_NewRef(Py_None));
  Ref second(coef.defined() ? THPVariable_Wrap(coef) : Py_NewRef(Py_None));
  if (first.o == nullptr || second.o == nullptr) throw python_error();
  return PyTuple_Pack(2, first.o, second.o);
  END_HANDLE_TH_ERRORS
}

// Whether a tensor's memory is dense, for the tests.
PyObject* py_dense(PyObject*, PyObject* o) {
  HANDLE_TH_ERRORS
  if (!THPVariable_Check(o)) raise(PyExc_TypeError, "not a tensor");
  return PyBool_FromLong(dense(THPVariable_Unpack(o)));
  END_HANDLE_TH_ERRORS
}

#define LUMA_FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f))
PyMethodDef kMethods[] = {
    {"norm", LUMA_FAST(py_norm), METH_FASTCALL, nullptr},
    {"power", LUMA_FAST(py_power), METH_FASTCALL, nullptr},
    {"finish", LUMA_FAST(py_finish), METH_FASTCALL, nullptr},
    {"scale", LUMA_FAST(py_scale), METH_FASTCALL, nullptr},
    {"accumulate", LUMA_FAST(py_accumulate), METH_FASTCALL, nullptr},
    {"dense", py_dense, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_grads_ext",
                       "Lists of tensors for the gradient operators.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__grads_ext(void) {
  if (luma_abi_version() != LUMA_ABI_VERSION) {
    PyErr_SetString(PyExc_ImportError, "libluma_b200.so and the tensor lists' module are of "
                                       "different builds");
    return nullptr;
  }
  // the layout of tensors and of Python objects is compiled in
  if ((Py_Version >> 16) != (PY_VERSION_HEX >> 16)) {
    PyErr_Format(PyExc_ImportError, "the tensor lists' module is built for Python %d.%d",
                 PY_MAJOR_VERSION, PY_MINOR_VERSION);
    return nullptr;
  }
  Ref torch(PyImport_ImportModule("torch"));
  if (torch.o == nullptr) return nullptr;
  Ref version(PyObject_GetAttrString(torch.o, "__version__"));
  if (version.o == nullptr) return nullptr;
  const char* text = PyUnicode_AsUTF8(version.o);
  if (text == nullptr) return nullptr;
  if (std::string(text) != LUMA_TORCH_VERSION) {
    PyErr_Format(PyExc_ImportError, "the tensor lists' module is built for torch %s, this is "
                                    "torch %s", LUMA_TORCH_VERSION, text);
    return nullptr;
  }
  return PyModule_Create(&kModule);
}
