// Python module that hands lists of torch tensors to the multi-tensor entries of libmi_ns.so.
//
// A call over a hundred small tensors takes the GPU a few microseconds.  Reading addresses, sizes, types and layouts of
// four lists through Python attributes takes about 0.4 us a tensor (111 us for 65 parameters with gradient and two
// moments); here it takes about 0.02 us.  Checks of arguments live here and nowhere else; the errors are Python's own
// (TypeError, ValueError, RuntimeError), and the entries' return codes go back to the caller.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <string>
#include <vector>

#include "../../include/mi_ns.h"

namespace {

// A refusal: the Python exception is raised where the call returns to Python.
struct Refused {
  PyObject* type;
  std::string text;
};
[[noreturn]] void refuse(PyObject* type, std::string text) { throw Refused{type, std::move(text)}; }

std::string number(int64_t v) { return std::to_string(v); }

int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? MI_DTYPE_F32 : t == at::kBFloat16 ? MI_DTYPE_BF16 : t == at::kHalf ? MI_DTYPE_F16 : -1;
}
std::string dtype_name(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    case at::kDouble: return "torch.float64";
    case at::kByte: return "torch.uint8";
    default: return c10::toString(t);
  }
}
std::string text_of(at::IntArrayRef v) {
  std::string s = "(";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + number(v[i]);
  return s + (v.size() == 1 ? ",)" : ")");
}

// The elements fill one block of memory, in whatever order of the dimensions.
bool is_dense(const at::Tensor& t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

// Tensors of a Python sequence; the sequence keeps them alive during the call.  What the checks ask of a tensor is read
// once, into a small record.
struct Item {
  const at::Tensor* t;
  int64_t n;
  at::ScalarType type;
  int gpu;  // -1: not on a GPU
  bool contiguous;
};
struct List {
  const char* who;
  const char* what;
  PyObject* fast = nullptr;
  std::vector<Item> items;

  List(const char* who_, const char* what_, PyObject* sequence) : who(who_), what(what_) {
    fast = PySequence_Fast(sequence, "");
    if (!fast) {
      PyErr_Clear();
      refuse(PyExc_TypeError, std::string(who) + ": " + what + " must be a sequence of tensors");
    }
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast);
    PyObject** objects = PySequence_Fast_ITEMS(fast);
    try {
      items.reserve(n);
      for (Py_ssize_t i = 0; i < n; ++i) {
        if (!THPVariable_Check(objects[i])) refuse(PyExc_TypeError, at_(i) + " is not a tensor");
        const at::Tensor& x = THPVariable_Unpack(objects[i]);
        // (values that are not what the memory holds)
        if (x.layout() != at::kStrided || x.is_neg()) refuse(PyExc_TypeError, at_(i) + " must be a plain strided tensor");
        items.push_back({&x, x.numel(), x.scalar_type(), x.is_cuda() ? (int)x.get_device() : -1, x.is_contiguous()});
      }
    } catch (...) {
      Py_DECREF(fast);
      throw;
    }
  }
  List(const List&) = delete;
  List& operator=(const List&) = delete;
  ~List() { Py_XDECREF(fast); }

  int64_t size() const { return (int64_t)items.size(); }
  const at::Tensor& operator[](size_t i) const { return *items[i].t; }
  std::string at_(size_t i) const { return std::string(who) + ": " + what + "[" + number((int64_t)i) + "]"; }

  // The one data type of the list, out of those whose bit is set (bit c for type code c).
  int dtype(int allowed) const {
    const int code = items.empty() ? -1 : dtype_code(items[0].type);
    bool ok = code >= 0 && (allowed >> code & 1);
    for (const Item& x : items) ok = ok && x.type == items[0].type;
    if (ok) return code;
    std::vector<std::string> found;
    for (const Item& x : items) found.push_back(dtype_name(x.type));
    std::sort(found.begin(), found.end());
    found.erase(std::unique(found.begin(), found.end()), found.end());
    std::string names, options;
    for (const std::string& f : found) names += (names.empty() ? "" : ", ") + f;
    for (int c = 0; c < 3; ++c)
      if (allowed >> c & 1) options += std::string(options.empty() ? "" : ", ") + (c == 0 ? "torch.float32" : c == 1 ? "torch.bfloat16" : "torch.float16");
    refuse(PyExc_TypeError, std::string(who) + ": " + what + " must have one data type out of " + options + ", got " + (names.empty() ? "nothing" : names));
  }

  // Shapes and memory order of another list, whose tensors' elements fill their memory.
  void like(const List& o) const {
    if (size() != o.size()) refuse(PyExc_ValueError, std::string(who) + ": " + number(size()) + " " + what + " for " + number(o.size()) + " " + o.what);
    for (size_t i = 0; i < items.size(); ++i) {
      const at::Tensor &x = *items[i].t, &p = *o.items[i].t;
      if (!x.sizes().equals(p.sizes()))
        refuse(PyExc_ValueError, at_(i) + " has shape " + text_of(x.sizes()) + ", its param " + text_of(p.sizes()));
      if (items[i].contiguous && o.items[i].contiguous) continue;
      if (!x.strides().equals(p.strides()) || !is_dense(p))
        refuse(PyExc_ValueError, at_(i) + " must fill its memory in the order of its param, got strides " + text_of(x.strides()) + " and " + text_of(p.strides()));
    }
  }

  void dense() const {
    for (const Item& x : items)
      if (!x.contiguous && !is_dense(*x.t)) refuse(PyExc_ValueError, std::string(who) + ": " + what + " must fill their memory");
  }

  // 8-bit forms of the moments of another list.
  void packed(const List& o) const {
    if (size() != o.size()) refuse(PyExc_ValueError, std::string(who) + ": " + number(size()) + " " + what + " for " + number(o.size()) + " tensors");
    for (size_t i = 0; i < items.size(); ++i) {
      if (items[i].type != at::kByte) refuse(PyExc_TypeError, at_(i) + " must be uint8, got " + dtype_name(items[i].type));
      const int64_t want = (int64_t)mi_moment_8bit_bytes(o.items[i].n);
      if (items[i].n != want || !items[i].contiguous)
        refuse(PyExc_ValueError, at_(i) + " must be " + number(want) + " contiguous bytes, got " + text_of((*this)[i].sizes()));
    }
  }

  std::vector<void*> pointers() const {
    std::vector<void*> p(items.size());
    for (size_t i = 0; i < items.size(); ++i) p[i] = items[i].t->data_ptr();
    return p;
  }
  // The call writes these tensors: autograd's version counters move as after an in-place operation, so a backward pass
  // over a graph that saved one of them is refused.
  void written() const {
    for (const Item& x : items)
      if (x.t->unsafeGetTensorImpl()->version_counter().enabled()) x.t->unsafeGetTensorImpl()->bump_version();
  }
  std::vector<int64_t> numels() const {
    std::vector<int64_t> n(items.size());
    for (size_t i = 0; i < items.size(); ++i) n[i] = items[i].n;
    return n;
  }
  // Data types of the list, which may differ.
  std::vector<int> dtypes() const {
    std::vector<int> d(items.size());
    for (size_t i = 0; i < items.size(); ++i) {
      d[i] = dtype_code(items[i].type);
      if (d[i] < 0) refuse(PyExc_TypeError, std::string(who) + ": " + what + " must be float32, bfloat16 or float16, got " + dtype_name(items[i].type));
    }
    return d;
  }
};

// The one GPU all tensors of the lists are on.
c10::Device one_gpu(const char* who, std::initializer_list<const List*> lists) {
  int gpu = -1;
  for (const List* l : lists) {
    if (!l) continue;
    for (const Item& x : l->items) {
      if (x.gpu < 0) refuse(PyExc_RuntimeError, std::string(who) + " runs on the GPU only; got a tensor on " + x.t->device().str());
      if (gpu < 0) gpu = x.gpu;
      if (x.gpu != gpu) refuse(PyExc_ValueError, std::string(who) + ": all tensors of a call must be on one GPU, got numbers " + number(gpu) + " and " + number(x.gpu));
    }
  }
  return gpu < 0 ? c10::Device(c10::kCPU) : c10::Device(c10::kCUDA, (c10::DeviceIndex)gpu);
}

const at::Tensor& device_scalar(const char* who, const char* what, PyObject* o, c10::Device device, const char* like) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, std::string(who) + ": " + what + " must be a tensor");
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.scalar_type() != at::kFloat || t.numel() != 1 || t.device() != device)
    refuse(PyExc_ValueError, std::string(who) + ": " + what + " must be one float32 value on the GPU of the " + like + ", got " + dtype_name(t.scalar_type()) + " " +
                                 text_of(t.sizes()) + " on " + t.device().str());
  return t;
}

double number_of(const char* who, const char* what, PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(PyExc_TypeError, std::string(who) + ": " + what + " must be a number");
  }
  return v;
}

void* current_stream(c10::Device device) {
  return c10::hip::getCurrentHIPStream(device.index()).stream();
}

const float* value(const at::Tensor& t) { return static_cast<const float*>(t.data_ptr()); }

template <class Body>
PyObject* guarded(Body body) {
  try {
    return body();
  } catch (const Refused& r) {
    PyErr_SetString(r.type, r.text.c_str());
  } catch (const std::bad_alloc&) {
    PyErr_NoMemory();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

constexpr int ANY_TYPE = 7, F32_ONLY = 1, HALF_TYPES = 6;

// adamw_update(who, bits (mi_adamw_update's moment_bits), params, grads, exp_avgs, exp_avg_sqs, model_params | None, step | steps, lr, beta1, beta2,
//              eps, weight_decay, method, grad_scale | None) -> return code
PyObject* adamw_update(PyObject*, PyObject* args) {
  const char* who;
  int bits, method;
  PyObject *p_, *g_, *m_, *v_, *low_, *step_, *lr_, *scale_;
  double beta1, beta2, eps, wd;
  if (!PyArg_ParseTuple(args, "siOOOOOOOddddiO", &who, &bits, &p_, &g_, &m_, &v_, &low_, &step_, &lr_, &beta1, &beta2, &eps, &wd, &method, &scale_)) return nullptr;
  return guarded([&]() -> PyObject* {
    const bool has_low = low_ != Py_None;
    PyObject* const no_list = has_low ? low_ : p_;  // (never read without copies)
    const List params(who, "params", p_), grads(who, "grads", g_), ms(who, "exp_avgs", m_), vs(who, "exp_avg_sqs", v_), low(who, "model_params", no_list);
    if (params.size() == 0 && grads.size() == 0 && ms.size() == 0 && vs.size() == 0 && low.size() == 0) return PyLong_FromLong(MI_OK);
    const int p_type = params.dtype(ANY_TYPE), g_type = grads.dtype(ANY_TYPE);
    grads.like(params);
    for (const List* l : {&ms, &vs}) {
      if (bits != 32) {
        l->packed(params);
      } else {
        l->dtype(F32_ONLY);
        l->like(params);
      }
    }
    int low_type = MI_DTYPE_BF16;
    if (has_low) {
      if (p_type != MI_DTYPE_F32) refuse(PyExc_TypeError, std::string(who) + ": model_params go with float32 params, got " + dtype_name(params[0].scalar_type()));
      low_type = low.dtype(HALF_TYPES);
      low.like(params);
    }
    const c10::Device device = one_gpu(who, {&params, &grads, &ms, &vs, has_low ? &low : nullptr});
    std::vector<const float*> steps;
    double step = 1.0, lr = 0.0;
    if (PyNumber_Check(step_) && !PySequence_Check(step_)) {
      step = number_of(who, "step", step_);
    } else {
      const List s(who, "step", step_);
      if (s.size() != params.size()) refuse(PyExc_ValueError, std::string(who) + ": " + number(s.size()) + " steps for " + number(params.size()) + " params");
      for (int64_t i = 0; i < s.size(); ++i) steps.push_back(value(device_scalar(who, "step", PySequence_Fast_GET_ITEM(s.fast, i), device, "params")));
    }
    const float* lr_dev = nullptr;
    if (THPVariable_Check(lr_)) lr_dev = value(device_scalar(who, "lr", lr_, device, "params"));
    else lr = number_of(who, "lr", lr_);
    const float* scale = scale_ == Py_None ? nullptr : value(device_scalar(who, "grad_scale", scale_, device, "params"));
    const std::vector<void*> p = params.pointers(), g = grads.pointers(), m = ms.pointers(), v = vs.pointers();
    std::vector<void*> l;
    if (has_low) l = low.pointers();
    const std::vector<int64_t> n = params.numels();
    const c10::DeviceGuard guard(device);
    const int rc = mi_adamw_update((int64_t)p.size(), p.data(), g.data(), m.data(), v.data(), has_low ? l.data() : nullptr,
                                   steps.empty() ? nullptr : steps.data(), n.data(), p_type, g_type, low_type, bits, step, lr, lr_dev, beta1, beta2, eps, wd, method,
                                   scale, current_stream(device));
    if (rc == MI_OK) {
      params.written();
      ms.written();
      vs.written();
      if (has_low) low.written();
    }
    return PyLong_FromLong(rc);
  });
}

// move_moments(who, pack, values, packed, second) -> return code
PyObject* move_moments(PyObject*, PyObject* args) {
  const char* who;
  int pack, second;
  PyObject *values_, *packed_;
  if (!PyArg_ParseTuple(args, "spOOi", &who, &pack, &values_, &packed_, &second)) return nullptr;
  return guarded([&]() -> PyObject* {
    const List values(who, "moments", values_), packed(who, "packed", packed_);
    packed.packed(values);
    if (values.size() == 0) return PyLong_FromLong(MI_OK);
    const int type = values.dtype(ANY_TYPE);
    values.dense();
    const c10::Device device = one_gpu(who, {&values, &packed});
    const std::vector<void*> x = values.pointers(), q = packed.pointers();
    const std::vector<int64_t> n = values.numels();
    const c10::DeviceGuard guard(device);
    void* const stream = current_stream(device);
    const int rc = pack ? mi_moments_8bit_pack((int64_t)x.size(), x.data(), q.data(), n.data(), type, second, stream)
                        : mi_moments_8bit_unpack((int64_t)x.size(), q.data(), x.data(), n.data(), type, second, stream);
    if (rc == MI_OK) (pack ? packed : values).written();
    return PyLong_FromLong(rc);
  });
}

// global_norm(who, tensors, max_norm, scale) -> (return code, norm, factor); with `scale` the tensors are multiplied by
// the factor.
PyObject* global_norm(PyObject*, PyObject* args) {
  const char* who;
  PyObject* tensors_;
  double max_norm;
  int scale;
  if (!PyArg_ParseTuple(args, "sOdp", &who, &tensors_, &max_norm, &scale)) return nullptr;
  return guarded([&]() -> PyObject* {
    const List tensors(who, "tensors", tensors_);
    if (tensors.size() == 0) refuse(PyExc_ValueError, std::string(who) + " needs at least one tensor");
    const std::vector<int> types = tensors.dtypes();
    tensors.dense();
    const c10::Device device = one_gpu(who, {&tensors});
    const std::vector<void*> x = tensors.pointers();
    const std::vector<int64_t> n = tensors.numels();
    const int64_t count = tensors.size();
    const c10::DeviceGuard guard(device);
    void* const stream = current_stream(device);
    // The scratch is this call's alone: it comes from the caching allocator for the current stream (while a graph is
    // captured, from the graph's own pool), so no two calls and no two graphs share it.
    const size_t length = mi_global_norm_partials_len(count, n.data());
    const at::Tensor partials = at::empty({(int64_t)length}, at::TensorOptions(device).dtype(at::kDouble));
    const at::Tensor out = at::empty({2}, at::TensorOptions(device).dtype(at::kFloat));
    float* const result = static_cast<float*>(out.data_ptr());
    double* const scratch = length ? static_cast<double*>(partials.data_ptr()) : nullptr;
    const int rc = scale ? mi_clip_by_global_norm(count, x.data(), n.data(), types.data(), max_norm, scratch, length, result, stream)
                         : mi_global_norm(count, x.data(), n.data(), types.data(), max_norm, scratch, length, result, stream);
    if (rc == MI_OK && scale) tensors.written();
    return Py_BuildValue("(iNN)", rc, THPVariable_Wrap(out.select(0, 0)), THPVariable_Wrap(out.select(0, 1)));
  });
}

// scale_tensors(who, tensors, factor) -> return code
PyObject* scale_tensors(PyObject*, PyObject* args) {
  const char* who;
  PyObject *tensors_, *factor_;
  if (!PyArg_ParseTuple(args, "sOO", &who, &tensors_, &factor_)) return nullptr;
  return guarded([&]() -> PyObject* {
    const List tensors(who, "tensors", tensors_);
    if (tensors.size() == 0) return PyLong_FromLong(MI_OK);
    const std::vector<int> types = tensors.dtypes();
    tensors.dense();
    const c10::Device device = one_gpu(who, {&tensors});
    const float* factor = value(device_scalar(who, "factor", factor_, device, "tensors"));
    const std::vector<void*> x = tensors.pointers();
    const std::vector<int64_t> n = tensors.numels();
    const c10::DeviceGuard guard(device);
    const int rc = mi_scale_tensors(tensors.size(), x.data(), n.data(), types.data(), factor, current_stream(device));
    if (rc == MI_OK) tensors.written();
    return PyLong_FromLong(rc);
  });
}

PyMethodDef METHODS[] = {
    {"adamw_update", adamw_update, METH_VARARGS, "mi_adamw_update over lists of tensors"},
    {"move_moments", move_moments, METH_VARARGS, "mi_moments_8bit_pack / mi_moments_8bit_unpack over lists of tensors"},
    {"global_norm", global_norm, METH_VARARGS, "mi_global_norm (and mi_scale_tensors) over a list of tensors"},
    {"scale_tensors", scale_tensors, METH_VARARGS, "mi_scale_tensors over a list of tensors"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef MODULE = {PyModuleDef_HEAD_INIT, "_mi_lists", "lists of tensors for libmi_ns.so", -1, METHODS, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mi_lists(void) { return PyModule_Create(&MODULE); }
