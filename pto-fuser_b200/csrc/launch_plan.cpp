// Launch plans: the host side of a call whose arguments have the same shapes, strides, types
// and device as an earlier call that was checked.
//
// The Python layer checks a call in full, once for each signature, and leaves a plan here: the
// C entry point, its parameter struct, where each pointer comes from, and what to allocate.
// Later calls with the signature skip the checks, which cost several times what the launch
// does: they allocate the outputs and scratch from torch's caching allocator, on the
// current stream of the tensors' device, and call the entry point. A signature holds no
// address, value or identity of a tensor. That is host time, which differs between machines: a
// pass through a single-token call took 5.5 us so on one (one output; 8 us with three) and 7 to 8
// (9.6) on others, 22 to 33 us through the checks. Calls that write into `out` have no plan.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>
#include <memory>
#include <unordered_map>
#include <vector>

namespace {

constexpr int kMaxTensors = 16, kMaxArgs = 16, kMaxOuts = 3, kMaxParams = 256;
constexpr int kMaxKey = 2 + kMaxTensors * 18;
constexpr size_t kMaxPlans = 4096;

// Where an argument of the entry point comes from.
enum Source : int { kNull = -1, kScratch = -2, kScratchBytes = -3, kOut0 = 100 };

struct Key {
  std::vector<int64_t> v;
  bool operator==(const Key& o) const { return v == o.v; }
};
struct KeyHash {
  size_t operator()(const Key& k) const {
    uint64_t h = 0x9e3779b97f4a7c15ull;
    for (int64_t x : k.v) {
      h ^= static_cast<uint64_t>(x);
      h *= 0xff51afd7ed558ccdull;
      h ^= h >> 32;
    }
    return static_cast<size_t>(h);
  }
};

struct Plan {
  void* fn = nullptr;
  alignas(16) unsigned char params[kMaxParams];
  int args[kMaxArgs];  // behind the params, before the stream
  int n_args = 0;
  std::vector<std::vector<int64_t>> out_sizes;
  std::vector<at::ScalarType> out_types;
  int64_t scratch = 0;
  int device = 0;
  int results[kMaxOuts];  // output indexes, kNull for None
  int n_results = 0;
  int writes = kNull;  // index of a tensor that the call updates
};

// A call holds its plan: making its results can run Python code that leaves other plans.
using Plans = std::unordered_map<Key, std::shared_ptr<const Plan>, KeyHash>;
Plans& plans() {
  static auto* m = new Plans();
  return *m;
}

// The signature of (op, flags, tensors...). False where a call has to take the checked way.
bool signature(PyObject* const* args, Py_ssize_t n, Key& key, const at::Tensor** t, int& count) {
  if (n < 2 || n - 2 > kMaxTensors) return false;
  key.v.clear();
  key.v.reserve(128);
  for (int i = 0; i < 2; ++i) {
    const int64_t x = PyLong_AsLongLong(args[i]);
    if (x == -1 && PyErr_Occurred()) return false;
    key.v.push_back(x);
  }
  const bool grad = c10::GradMode::is_enabled();
  const bool tangents = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  count = static_cast<int>(n - 2);
  for (int i = 0; i < count; ++i) {
    PyObject* o = args[i + 2];
    t[i] = nullptr;
    if (o == Py_None) {
      key.v.push_back(-1);
      continue;
    }
    if (!THPVariable_CheckExact(o)) return false;
    const at::Tensor& x = THPVariable_Unpack(o);
    if (x.layout() != at::kStrided || !x.is_cuda() || x.dim() > 8 || (grad && x.requires_grad()) ||
        x.is_neg() || x.is_conj() || !x.has_storage() || (tangents && x._fw_grad(0).defined()))
      return false;
    t[i] = &x;
    key.v.push_back((static_cast<int64_t>(x.dim()) << 32) |
                    (static_cast<int64_t>(x.scalar_type()) << 16) | x.get_device());
    const auto sizes = x.sizes(), strides = x.strides();
    key.v.insert(key.v.end(), sizes.begin(), sizes.end());
    key.v.insert(key.v.end(), strides.begin(), strides.end());
  }
  return true;
}

// First and last + 1 byte that a tensor can touch.
void span(const at::Tensor& t, uintptr_t& a, uintptr_t& b) {
  a = b = 0;
  if (t.numel() == 0) return;
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  a = reinterpret_cast<uintptr_t>(t.data_ptr());
  b = a + static_cast<uintptr_t>(last + 1) * t.element_size();
}
// Whether the memory of t[w], as a whole, reaches into another tensor's.
bool reaches(const at::Tensor* const* t, int count, int w) {
  uintptr_t a, b, c, d;
  span(*t[w], a, b);
  for (int i = 0; i < count; ++i) {
    if (i == w || !t[i]) continue;
    span(*t[i], c, d);
    if (c < b && a < d) return true;
  }
  return false;
}

using F = uintptr_t;
int invoke(void* fn, const F* a, int n) {  // the entry points take pointers and 64-bit integers only
  switch (n) {
    case 8: return reinterpret_cast<int (*)(F, F, F, F, F, F, F, F)>(fn)(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7]);
    case 9: return reinterpret_cast<int (*)(F, F, F, F, F, F, F, F, F)>(fn)(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8]);
    case 13: return reinterpret_cast<int (*)(F, F, F, F, F, F, F, F, F, F, F, F, F)>(fn)(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10], a[11], a[12]);
    case 16: return reinterpret_cast<int (*)(F, F, F, F, F, F, F, F, F, F, F, F, F, F, F, F)>(fn)(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10], a[11], a[12], a[13], a[14], a[15]);
  }
  return -1;
}

// run(op, flags, tensors...) -> None where no plan has the signature or the call has to be checked
// anew, the entry point's non-zero status as an int, or the tuple of results
PyObject* run(PyObject*, PyObject* const* args, Py_ssize_t n) {
  try {
    static thread_local Key key;
    const at::Tensor* t[kMaxTensors];
    int count = 0;
    if (!signature(args, n, key, t, count)) {
      if (PyErr_Occurred()) return nullptr;
      Py_RETURN_NONE;
    }
    const auto it = plans().find(key);
    if (it == plans().end()) Py_RETURN_NONE;
    const std::shared_ptr<const Plan> held = it->second;
    const Plan& p = *held;
    if (p.writes >= 0 && reaches(t, count, p.writes)) Py_RETURN_NONE;
    const c10::cuda::OptionalCUDAGuard guard(c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(p.device)));
    const auto on = at::TensorOptions().device(at::kCUDA, static_cast<c10::DeviceIndex>(p.device));
    at::Tensor outs[kMaxOuts], scratch;
    for (size_t i = 0; i < p.out_sizes.size(); ++i)
      outs[i] = at::empty(p.out_sizes[i], on.dtype(p.out_types[i]));
    if (p.scratch > 0) scratch = at::empty({p.scratch}, on.dtype(at::kByte));
    F a[kMaxArgs + 2];
    int k = 0;
    a[k++] = reinterpret_cast<F>(&p.params[0]);
    for (int i = 0; i < p.n_args; ++i) {
      const int s = p.args[i];
      if (s >= kOut0) a[k++] = reinterpret_cast<F>(outs[s - kOut0].data_ptr());
      else if (s == kScratch) a[k++] = p.scratch > 0 ? reinterpret_cast<F>(scratch.data_ptr()) : 0;
      else if (s == kScratchBytes) a[k++] = static_cast<F>(p.scratch);
      else a[k++] = s >= 0 && t[s] ? reinterpret_cast<F>(t[s]->data_ptr()) : 0;
    }
    a[k++] = reinterpret_cast<F>(c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(p.device)).stream());
    const int rc = invoke(p.fn, a, k);
    if (rc != 0) return PyLong_FromLong(rc);
    // a backward that saved the updated tensor must not use it
    if (p.writes >= 0 && !t[p.writes]->is_inference()) t[p.writes]->unsafeGetTensorImpl()->bump_version();
    PyObject* r = PyTuple_New(p.n_results);
    if (!r) return nullptr;
    for (int i = 0; i < p.n_results; ++i) {
      PyObject* o;
      if (p.results[i] < 0) {
        Py_INCREF(Py_None);
        o = Py_None;
      } else {
        o = THPVariable_Wrap(outs[p.results[i]]);
      }
      if (!o) {
        Py_DECREF(r);
        return nullptr;
      }
      PyTuple_SET_ITEM(r, i, o);
    }
    return r;
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    PyErr_SetString(type ? type : PyExc_RuntimeError, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// add((op, flags, tensors...), fn, params, args, outs, scratch, results, writes): leaves a plan.
// outs: ((sizes, type code), ...) with codes 0 f32, 1 f16, 2 bf16, 3 e4m3.
PyObject* add(PyObject*, PyObject* py) {
  try {
    PyObject *call, *args, *outs, *results;
    unsigned long long fn;
    const char* params;
    Py_ssize_t bytes;
    long long scratch;
    int writes;
    if (!PyArg_ParseTuple(py, "O!Ky#O!O!LO!i", &PyTuple_Type, &call, &fn, &params, &bytes,
                          &PyTuple_Type, &args, &PyTuple_Type, &outs, &scratch, &PyTuple_Type, &results,
                          &writes))
      return nullptr;
    Key key;
    const at::Tensor* t[kMaxTensors];
    int count = 0;
    std::vector<PyObject*> items(PyTuple_GET_SIZE(call));
    for (size_t i = 0; i < items.size(); ++i) items[i] = PyTuple_GET_ITEM(call, i);
    if (!signature(items.data(), static_cast<Py_ssize_t>(items.size()), key, t, count)) {
      if (PyErr_Occurred()) return nullptr;
      Py_RETURN_FALSE;
    }
    const auto made = std::make_shared<Plan>();
    Plan& p = *made;
    const Py_ssize_t na = PyTuple_GET_SIZE(args), no = PyTuple_GET_SIZE(outs),
                     nr = PyTuple_GET_SIZE(results);
    if (bytes > kMaxParams || na > kMaxArgs || no > kMaxOuts || nr > kMaxOuts) {
      PyErr_SetString(PyExc_ValueError, "plan too large");
      return nullptr;
    }
    p.fn = reinterpret_cast<void*>(static_cast<uintptr_t>(fn));
    std::memcpy(p.params, params, static_cast<size_t>(bytes));
    static const at::ScalarType kTypes[] = {at::kFloat, at::kHalf, at::kBFloat16, at::kFloat8_e4m3fn};
    for (Py_ssize_t i = 0; i < na; ++i) p.args[p.n_args++] = static_cast<int>(PyLong_AsLong(PyTuple_GET_ITEM(args, i)));
    for (Py_ssize_t i = 0; i < no; ++i) {
      PyObject *sizes;
      int code;
      if (!PyArg_ParseTuple(PyTuple_GET_ITEM(outs, i), "O!i", &PyTuple_Type, &sizes, &code)) return nullptr;
      std::vector<int64_t> s;
      for (Py_ssize_t j = 0; j < PyTuple_GET_SIZE(sizes); ++j) s.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(sizes, j)));
      p.out_sizes.push_back(std::move(s));
      p.out_types.push_back(kTypes[code & 3]);
    }
    for (Py_ssize_t i = 0; i < nr; ++i) p.results[p.n_results++] = static_cast<int>(PyLong_AsLong(PyTuple_GET_ITEM(results, i)));
    if (PyErr_Occurred()) return nullptr;
    p.scratch = scratch;
    p.writes = writes >= 0 && writes < count && t[writes] ? writes : kNull;
    for (int i = 0; i < count; ++i)
      if (t[i]) { p.device = t[i]->get_device(); break; }
    if (plans().size() >= kMaxPlans) plans().clear();
    plans().insert_or_assign(std::move(key), made);
    Py_RETURN_TRUE;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyMethodDef kMethods[] = {
    {"run", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(run)), METH_FASTCALL,
     "run(op, flags, *tensors): launch by plan; None without one, a status, or the results"},
    {"add", add, METH_VARARGS, "add(call, fn, params, args, outs, scratch, results, writes): leave a plan"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_launch", "launch plans of checked calls", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__launch() { return PyModule_Create(&kModule); }
