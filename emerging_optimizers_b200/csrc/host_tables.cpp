// Tables of tensor addresses for the operators over lists of tensors, built and checked in one pass over the Python lists.
// A call over a model's few hundred small tensors is bound by the host: asking every tensor from Python for its address,
// size, type, device and layout takes about two microseconds a parameter, here it takes some 20 nanoseconds a tensor.
//
// A Python extension module (emerging_optimizers_b200._host); everything below the tables stays behind the C ABI.
#include <torch/csrc/autograd/python_variable.h>

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <vector>

namespace {

constexpr int64_t kBlock = 256;  // elements that share an exponent byte of an 8-bit state

// A Python error is set.
struct Raised {};

class Owned {  // a new reference; a null one means that a Python error is set
 public:
  explicit Owned(PyObject* object) : object_(object) {
    if (object_ == nullptr) throw Raised{};
  }
  ~Owned() { Py_DECREF(object_); }
  Owned(const Owned&) = delete;
  PyObject* get() const { return object_; }

 private:
  PyObject* object_;
};

[[noreturn]] void raise(PyObject* type, const std::string& text) {
  PyErr_SetString(type, text.c_str());
  throw Raised{};
}

[[noreturn]] void raise_no_cpu_path(const std::string& name, const at::Tensor& t) {
  Owned module(PyImport_ImportModule("emerging_optimizers_b200._native"));
  Owned type(PyObject_GetAttrString(module.get(), "NativeLibraryError"));
  raise(type.get(), name + " is on " + t.device().str() +
                        "; emerging_optimizers_b200 runs on CUDA sm_100 devices only (there is no CPU path).");
}

enum Types : unsigned { kF32 = 1, kBF16 = 2, kU8 = 4, kI16 = 8, kI64 = 16 };

unsigned type_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return kF32;
    case at::kBFloat16: return kBF16;
    case at::kByte: return kU8;
    case at::kShort: return kI16;
    case at::kLong: return kI64;
    default: return 0;
  }
}

std::string names_of(unsigned types) {
  std::string s;
  const std::pair<unsigned, const char*> all[] = {
      {kF32, "torch.float32"}, {kBF16, "torch.bfloat16"}, {kU8, "torch.uint8"}, {kI16, "torch.int16"}, {kI64, "torch.int64"}};
  for (const auto& [bit, name] : all)
    if (types & bit) s += (s.empty() ? "" : " or ") + std::string(name);
  return s;
}

// A list or tuple of tensors, which the caller keeps until its launch: tensors that only an iterator holds would be gone by then.
class Tensors {
 public:
  Tensors(PyObject* object, const char* name) : seq_(object), name_(name) {
    if (THPVariable_Check(object)) raise(PyExc_TypeError, name_ + " must be a list of tensors, not a tensor");
    if (!PyList_Check(object) && !PyTuple_Check(object))
      raise(PyExc_TypeError, name_ + " must be a list of tensors, not " + Py_TYPE(object)->tp_name);
  }
  Tensors(const Tensors&) = delete;
  int64_t size() const { return PySequence_Fast_GET_SIZE(seq_); }
  PyObject* item(int64_t i) const { return PySequence_Fast_GET_ITEM(seq_, i); }
  const at::Tensor& operator[](int64_t i) const {
    PyObject* item = PySequence_Fast_GET_ITEM(seq_, i);
    if (!THPVariable_Check(item)) raise(PyExc_TypeError, at(i) + " is not a tensor");
    return THPVariable_Unpack(item);
  }
  std::string at(int64_t i) const { return name_ + "[" + std::to_string(i) + "]"; }
  const std::string& name() const { return name_; }

 private:
  PyObject* seq_;
  std::string name_;
};

// The checks that every tensor passes, and its address.  any_order: dense in any order of its dimensions, for operators to which
// the places of the elements are nothing.
int64_t address(const Tensors& ts, int64_t i, int device, unsigned types, int64_t numel, bool any_order = false) {
  const at::Tensor& t = ts[i];
  if (!t.is_cuda()) raise_no_cpu_path(ts.at(i), t);
  if (t.get_device() != device)
    raise(PyExc_ValueError, ts.at(i) + " is on " + t.device().str() + ", the first parameter on cuda:" + std::to_string(device));
  if (!(type_of(t) & types))
    raise(PyExc_TypeError, ts.name() + " must be " + names_of(types) + ", " + ts.at(i) + " is " + c10::toString(t.scalar_type()));
  if (numel >= 0 && t.numel() != numel)
    raise(PyExc_ValueError,
          ts.at(i) + " has " + std::to_string(t.numel()) + " elements where " + std::to_string(numel) + " are needed");
  if (!t.is_contiguous() && !(any_order && t.is_non_overlapping_and_dense()))
    raise(PyExc_ValueError, ts.at(i) + (any_order ? " is not dense" : " is not contiguous"));
  if (t.is_neg()) raise(PyExc_ValueError, ts.at(i) + " is a negated view");
  return reinterpret_cast<int64_t>(t.data_ptr());
}

void require_count(const Tensors& ts, int64_t n) {
  if (ts.size() != n)
    raise(PyExc_ValueError, ts.name() + ": " + std::to_string(ts.size()) + " tensors where " + std::to_string(n) + " are needed");
}

int first_device(const Tensors& ts) {
  const at::Tensor& t = ts[0];
  if (!t.is_cuda()) raise_no_cpu_path(ts.at(0), t);
  return static_cast<int>(t.get_device());
}

void require_distinct(std::vector<int64_t>& written, const char* what) {
  std::sort(written.begin(), written.end());
  if (std::adjacent_find(written.begin(), written.end()) != written.end())
    raise(PyExc_ValueError, std::string("a tensor appears twice among ") + what);
}

// Tells autograd that the tensor changes: a backward pass that saved it raises instead of using it.
void mark_written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

PyObject* bytes_of(const std::vector<int64_t>& table) {
  const auto bytes = static_cast<Py_ssize_t>(table.size() * sizeof(int64_t));
  return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(table.data()), bytes);
}

template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Raised&) {
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// adamw_table(params, grads, exp_avgs, exp_avg_sqs, exp_avg_exponents | None, exp_avg_sq_exponents | None,
//             remainders | None, steps | None) -> (device, table, kinds): the ten rows of eo_adamw_step and the set (bits) of
// kinds in it.  8-bit moments where exponents are given.
PyObject* adamw_table(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    if (nargs != 8) raise(PyExc_TypeError, "adamw_table takes 8 arguments");
    const bool bits8 = args[4] != Py_None, with_remainders = args[6] != Py_None, with_steps = args[7] != Py_None;
    Tensors p(args[0], "params"), g(args[1], "grads"), m(args[2], "exp_avgs"), v(args[3], "exp_avg_sqs");
    const int64_t n = p.size();
    if (n == 0) raise(PyExc_ValueError, "no parameters given");
    const int device = first_device(p);
    for (const Tensors* ts : {&g, &m, &v}) require_count(*ts, n);
    std::vector<int64_t> table(10 * n, 0), written;
    written.reserve(6 * n);
    const auto column = [&](int row) { return table.data() + row * n; };
    unsigned kinds = 0;
    for (int64_t i = 0; i < n; ++i) {
      column(0)[i] = address(p, i, device, kF32 | kBF16, -1);
      const int64_t numel = p[i].numel();
      column(1)[i] = address(g, i, device, kF32 | kBF16, numel);
      column(2)[i] = address(m, i, device, bits8 ? kU8 : kF32, numel);
      column(3)[i] = address(v, i, device, bits8 ? kU8 : kF32, numel);
      column(8)[i] = numel;
      column(9)[i] = (p[i].scalar_type() == at::kBFloat16 ? 1 : 0) | (g[i].scalar_type() == at::kBFloat16 ? 2 : 0) |
                     (with_remainders ? 4 : 0);
      kinds |= 1u << column(9)[i];
      if (numel > 0) written.insert(written.end(), {column(0)[i], column(2)[i], column(3)[i]});
    }
    if (bits8) {
      Tensors me(args[4], "exp_avg_exponents"), ve(args[5], "exp_avg_sq_exponents");
      require_count(me, n);
      require_count(ve, n);
      for (int64_t i = 0; i < n; ++i) {
        const int64_t blocks = (column(8)[i] + kBlock - 1) / kBlock;
        column(4)[i] = address(me, i, device, kU8, blocks);
        column(5)[i] = address(ve, i, device, kU8, blocks);
        if (blocks > 0) written.insert(written.end(), {column(4)[i], column(5)[i]});
      }
    }
    if (with_remainders) {
      Tensors r(args[6], "remainders");
      require_count(r, n);
      for (int64_t i = 0; i < n; ++i) {
        if (!(column(9)[i] & 1)) raise(PyExc_TypeError, "remainders go with bf16 parameters only");
        column(6)[i] = address(r, i, device, kI16, column(8)[i]);
        if (column(8)[i] > 0) written.push_back(column(6)[i]);
      }
    }
    if (with_steps) {
      if (THPVariable_Check(args[7])) {
        Owned one(PyTuple_Pack(1, args[7]));
        Tensors s(one.get(), "step");
        std::fill_n(column(7), n, address(s, 0, device, kI64, 1));
      } else {
        Tensors s(args[7], "step");
        require_count(s, n);
        for (int64_t i = 0; i < n; ++i) column(7)[i] = address(s, i, device, kI64, 1);
      }
    }
    require_distinct(written, "the parameters and their state");
    for (int64_t i = 0; i < n; ++i) mark_written(p[i]);
    Owned bytes(bytes_of(table));
    return Py_BuildValue("iOI", device, bytes.get(), kinds);
  });
}

// grads_table(grads, in_place) -> (device, table, types, elements): the three rows of eo_grad_norm, the set (bits) of types in it
// and the number of all elements.
PyObject* grads_table(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    if (nargs != 2) raise(PyExc_TypeError, "grads_table takes 2 arguments");
    Tensors g(args[0], "grads");
    const bool in_place = args[1] == Py_True;
    const int64_t n = g.size();
    if (n == 0) raise(PyExc_ValueError, "no gradients given");
    const int device = first_device(g);
    std::vector<int64_t> table(3 * n), written;
    unsigned types = 0;
    long long elements = 0;
    for (int64_t i = 0; i < n; ++i) {
      table[i] = address(g, i, device, kF32 | kBF16, -1, true);
      table[n + i] = g[i].numel();
      table[2 * n + i] = g[i].scalar_type() == at::kBFloat16 ? 1 : 0;
      types |= 1u << table[2 * n + i];
      elements += table[n + i];
      if (in_place && table[n + i] > 0) written.push_back(table[i]);
    }
    require_distinct(written, "the gradients");
    if (in_place)
      for (int64_t i = 0; i < n; ++i) mark_written(g[i]);
    Owned bytes(bytes_of(table));
    return Py_BuildValue("iOIL", device, bytes.get(), types, elements);
  });
}

// with_grads(params) -> (those with a gradient, their gradients, whether all of both are contiguous and the parameters of
// one device and type).
PyObject* with_grads(PyObject*, PyObject* arg) {
  return guarded([&]() -> PyObject* {
    Tensors p(arg, "params");
    Owned params(PyList_New(0)), grads(PyList_New(0));
    bool uniform = true;
    const at::Tensor* first = nullptr;
    for (int64_t i = 0; i < p.size(); ++i) {
      const at::Tensor& t = p[i];
      const at::Tensor& g = t.grad();
      if (!g.defined()) continue;
      if (g.layout() != at::kStrided) raise(PyExc_RuntimeError, "AdamW does not support sparse gradients");
      if (first == nullptr) first = &t;
      uniform = uniform && t.is_contiguous() && g.is_contiguous() && t.device() == first->device() &&
                t.scalar_type() == first->scalar_type();
      Owned wrapped(THPVariable_Wrap(g));
      if (PyList_Append(params.get(), p.item(i)) != 0 || PyList_Append(grads.get(), wrapped.get()) != 0) throw Raised{};
    }
    return Py_BuildValue("OOO", params.get(), grads.get(), uniform ? Py_True : Py_False);
  });
}

// stream(device) -> (address of the current stream, whether the device is the current one, whether it is being captured)
PyObject* stream(PyObject*, PyObject* arg) {
  return guarded([&]() -> PyObject* {
    const long device = PyLong_AsLong(arg);
    if (device == -1 && PyErr_Occurred()) throw Raised{};
    const auto s = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    const cudaError_t error = cudaStreamIsCapturing(s, &status);
    if (error != cudaSuccess) raise(PyExc_RuntimeError, cudaGetErrorString(error));
    return Py_BuildValue("KOO", static_cast<unsigned long long>(reinterpret_cast<uintptr_t>(s)),
                         c10::cuda::current_device() == device ? Py_True : Py_False,
                         status != cudaStreamCaptureStatusNone ? Py_True : Py_False);
  });
}

PyMethodDef methods[] = {
    {"adamw_table", reinterpret_cast<PyCFunction>(adamw_table), METH_FASTCALL, nullptr},
    {"grads_table", reinterpret_cast<PyCFunction>(grads_table), METH_FASTCALL, nullptr},
    {"with_grads", with_grads, METH_O, nullptr},
    {"stream", stream, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() {
  return PyModule_Create(&module);
}
