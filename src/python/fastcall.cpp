// The per-call half of the Python binding: the checks, pointers and stream of
// a collective on CUDA tensors, read from the tensors themselves instead of
// through a dozen Python attributes and ctypes conversions.
//
// Small messages are bound by the host: a 4 KiB world-size-1 allreduce spent
// 8 us per call, of which the launch itself is 2.3 us (an empty kernel, back
// to back) and the Python side most of the rest.  Everything that is not on
// the path of a collective (set-up, messaging, diagnostics) stays in ctypes.
//
// The functions raise the package's IbcommError and return None.  The GIL is
// released around the library call, as ctypes does.  Tensors without storage, a
// missing driver and the like are C++ exceptions in torch: the entry points turn
// them into the Python exceptions torch's own methods raise.
#include <Python.h>

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/Event.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/engine.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <memory>
#include <string>
#include <utility>
#include <vector>

#include "ibcomm/c_api.h"
#include "ibcomm/device_types.h"

namespace {

PyObject* g_error = nullptr;  // IbcommError(code, message)

constexpr int kInvalidArgument = 1, kNotSupported = 4;

PyObject* Raise(int code, const char* message) {
  PyObject* e = g_error != nullptr ? PyObject_CallFunction(g_error, "is", code, message) : nullptr;
  if (e != nullptr) {
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
  } else if (!PyErr_Occurred()) {
    PyErr_SetString(PyExc_RuntimeError, message);
  }
  return nullptr;
}

PyObject* RaiseLast(int code) {
  std::string m = ibcomm_last_error();
  while (!m.empty() && (m.back() == '\n' || m.back() == ' ')) m.pop_back();
  return Raise(code, m.c_str());
}

// Code of the library's element type, or -1.
int DTypeCode(c10::ScalarType t) {
  switch (t) {
    case c10::ScalarType::Float: return 0;
    case c10::ScalarType::Double: return 1;
    case c10::ScalarType::Int: return 2;
    case c10::ScalarType::Long: return 3;
    case c10::ScalarType::Half: return 4;
    case c10::ScalarType::BFloat16: return 5;
    default: return -1;
  }
}

// The tensor behind `o`; null with an exception set when it is none, has an
// unsupported type, is not contiguous or out of the GPU's reach.
const at::Tensor* Tensor(PyObject* o, int* dtype) {
  if (!THPVariable_Check(o)) {
    PyErr_SetString(PyExc_TypeError, "a torch.Tensor is expected");
    return nullptr;
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_contiguous()) {
    Raise(kInvalidArgument, "tensors must be contiguous");
    return nullptr;
  }
  const int d = DTypeCode(t.scalar_type());
  if (d < 0) {
    Raise(kNotSupported, (std::string("unsupported dtype ") + c10::toString(t.scalar_type())).c_str());
    return nullptr;
  }
  // A kernel reads and writes it: memory of a GPU, or pinned host memory.
  if (!t.is_cuda() && !t.is_pinned()) {
    Raise(kInvalidArgument, "tensors must live on the GPU");
    return nullptr;
  }
  *dtype = d;
  return &t;
}

// Whether a kernel that runs on the GPU of `a` can be given `b` too.
bool SameGpu(const at::Tensor& a, const at::Tensor& b) { return !a.is_cuda() || !b.is_cuda() || a.device() == b.device(); }

template <typename Handle>
bool ToHandle(PyObject* o, Handle** h) {
  *h = o == Py_None ? nullptr : static_cast<Handle*>(PyLong_AsVoidPtr(o));
  return !PyErr_Occurred();
}

// `stream` (a raw stream as an integer) or, for None, the current one of `device`.
bool ToStream(PyObject* stream, c10::DeviceIndex device, void** out) {
  if (stream == Py_None) {
    *out = c10::cuda::getCurrentCUDAStream(device).stream();
    return true;
  }
  *out = PyLong_AsVoidPtr(stream);
  return !PyErr_Occurred();
}

bool WantArgs(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%zd arguments are expected, got %zd", want, n);
  return false;
}

// The tensors of a sequence, one per rank.  It holds on to the sequence: one that
// makes its items as it is read (the rows of a tensor) has them live no longer
// than the list they were gathered in.
struct RankTensors {
  PyObject* list = nullptr;
  void* ptr[ibcomm::kMaxRanks] = {};
  const at::Tensor* first = nullptr;
  int dtype = 0;
  int64_t shortest = 0;  // fewest elements of one

  RankTensors() = default;
  RankTensors(const RankTensors&) = delete;
  RankTensors& operator=(const RankTensors&) = delete;
  ~RankTensors() { Py_XDECREF(list); }

  // `elements` fit into every tensor, and `o` is of the same type on the same GPU.
  bool Hold(int64_t elements, const RankTensors& o) const { return shortest >= elements && dtype == o.dtype && SameGpu(*first, *o.first); }

  // A short sequence leaves nulls, which the library refuses.
  bool Read(PyObject* seq, int ranks) {
    list = PySequence_Fast(seq, "a sequence of tensors is expected");
    if (list == nullptr) return false;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(list);
    if (n > ranks || n == 0) {
      PyErr_SetString(PyExc_IndexError, "one tensor per rank is expected");
      return false;
    }
    for (Py_ssize_t i = 0; i < n; ++i) {
      int d;
      const at::Tensor* t = Tensor(PySequence_Fast_GET_ITEM(list, i), &d);
      if (t == nullptr) return false;
      if (i == 0) first = t, dtype = d, shortest = t->numel();
      if (d != dtype || !SameGpu(*first, *t)) {
        Raise(kInvalidArgument, "the ranks' tensors must match in dtype and live on one GPU");
        return false;
      }
      if (t->numel() < shortest) shortest = t->numel();
      ptr[i] = t->data_ptr();
    }
    return true;
  }
};

PyObject* Done(int code) {
  if (code != 0) return RaiseLast(code);
  Py_RETURN_NONE;
}

// set_error(IbcommError)
PyObject* SetError(PyObject*, PyObject* cls) {
  Py_XDECREF(g_error);
  g_error = Py_NewRef(cls);
  Py_RETURN_NONE;
}

// allreduce(handle, send, recv, algo, scale, wire, stream, flags); wire < 0: the tensors' type
PyObject* Allreduce(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!WantArgs(n, 8)) return nullptr;
  ibcomm_comm* c;
  if (!ToHandle(a[0], &c)) return nullptr;
  int d, rd;
  const at::Tensor* s = Tensor(a[1], &d);
  if (s == nullptr) return nullptr;
  const at::Tensor* r = Tensor(a[2], &rd);
  if (r == nullptr) return nullptr;
  if (d != rd || s->numel() != r->numel()) return Raise(kInvalidArgument, "sendbuf and recvbuf must match in dtype and size");
  if (!SameGpu(*s, *r)) return Raise(kInvalidArgument, "sendbuf and recvbuf must live on the same GPU");
  const int algo = static_cast<int>(PyLong_AsLong(a[3]));
  const double scale = PyFloat_AsDouble(a[4]);
  const int wire = static_cast<int>(PyLong_AsLong(a[5]));
  const int flags = static_cast<int>(PyLong_AsLong(a[7]));
  void* stream;
  if (PyErr_Occurred() || !ToStream(a[6], s->device().index(), &stream)) return nullptr;
  const void* in = s->data_ptr();
  void* out = r->data_ptr();
  const size_t len = static_cast<size_t>(s->numel());
  if (len != 0 && (in == nullptr || out == nullptr)) return Raise(kInvalidArgument, "tensors must have memory");
  int code;
  Py_BEGIN_ALLOW_THREADS;
  code = ibcomm_allreduce_cuda(c, algo, d, in, out, len, scale, wire < 0 ? d : wire, stream, flags);
  Py_END_ALLOW_THREADS;
  return Done(code);
  END_HANDLE_TH_ERRORS
}

// copy_scale(src, dst, scale)
PyObject* CopyScale(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!WantArgs(n, 3)) return nullptr;
  int di, dout;
  const at::Tensor* s = Tensor(a[0], &di);
  if (s == nullptr) return nullptr;
  const at::Tensor* d = Tensor(a[1], &dout);
  if (d == nullptr) return nullptr;
  if (!s->is_cuda()) return Raise(kInvalidArgument, "src must be a CUDA tensor");
  if (d->numel() < s->numel() || !SameGpu(*s, *d)) return Raise(kInvalidArgument, "dst must hold every element of src, on the same GPU");
  const double scale = PyFloat_AsDouble(a[2]);
  if (PyErr_Occurred()) return nullptr;
  const void* in = s->data_ptr();
  void* out = d->data_ptr();
  const size_t len = static_cast<size_t>(s->numel());
  if (len != 0 && (in == nullptr || out == nullptr)) return Raise(kInvalidArgument, "tensors must have memory");
  void* stream = c10::cuda::getCurrentCUDAStream(s->device().index()).stream();
  int code;
  Py_BEGIN_ALLOW_THREADS;
  code = ibcomm_copy_scale(in, out, len, di, dout, scale, stream);
  Py_END_ALLOW_THREADS;
  return Done(code);
  END_HANDLE_TH_ERRORS
}

// emu_allreduce(handle, ranks, sends, recvs, algo, scale, wire, channels, stream, async)
PyObject* EmuAllreduce(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!WantArgs(n, 10)) return nullptr;
  ibcomm_emu* w;
  if (!ToHandle(a[0], &w)) return nullptr;
  const int ranks = static_cast<int>(PyLong_AsLong(a[1]));
  RankTensors in, out;
  if (PyErr_Occurred()) return nullptr;
  if (ranks < 1 || ranks > ibcomm::kMaxRanks) return Raise(kNotSupported, "the number of ranks is out of range");
  if (!in.Read(a[2], ranks) || !out.Read(a[3], ranks)) return nullptr;
  const int64_t len = in.first->numel();
  if (!in.Hold(len, out) || !out.Hold(len, in))
    return Raise(kInvalidArgument, "every rank's tensors must match in dtype and hold as many elements as the first");
  const int algo = static_cast<int>(PyLong_AsLong(a[4]));
  const double scale = PyFloat_AsDouble(a[5]);
  const int wire = static_cast<int>(PyLong_AsLong(a[6]));
  const int channels = static_cast<int>(PyLong_AsLong(a[7]));
  const int async = static_cast<int>(PyLong_AsLong(a[9]));
  void* stream;
  if (PyErr_Occurred() || !ToStream(a[8], -1, &stream)) return nullptr;
  int code;
  Py_BEGIN_ALLOW_THREADS;
  code = ibcomm_emu_allreduce(w, algo, in.dtype, in.ptr, out.ptr, static_cast<size_t>(len), scale, wire < 0 ? in.dtype : wire, channels, stream, async);
  Py_END_ALLOW_THREADS;
  return Done(code);
  END_HANDLE_TH_ERRORS
}

// emu_rsag(handle, ranks, all_gather, sends, recvs, scale, channels)
PyObject* EmuRsAg(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!WantArgs(n, 7)) return nullptr;
  ibcomm_emu* w;
  if (!ToHandle(a[0], &w)) return nullptr;
  const int ranks = static_cast<int>(PyLong_AsLong(a[1]));
  const int all_gather = static_cast<int>(PyLong_AsLong(a[2]));
  RankTensors in, out;
  if (PyErr_Occurred()) return nullptr;
  if (ranks < 1 || ranks > ibcomm::kMaxRanks) return Raise(kNotSupported, "the number of ranks is out of range");
  if (!in.Read(a[3], ranks) || !out.Read(a[4], ranks)) return nullptr;
  const int64_t block = (all_gather ? in : out).first->numel();
  if (!in.Hold(all_gather ? block : block * ranks, out) || !out.Hold(all_gather ? block * ranks : block, in))
    return Raise(kInvalidArgument, "every rank's tensors must match in dtype and hold a block, or a block per rank");
  const double scale = PyFloat_AsDouble(a[5]);
  const int channels = static_cast<int>(PyLong_AsLong(a[6]));
  void* stream;
  if (PyErr_Occurred() || !ToStream(Py_None, -1, &stream)) return nullptr;
  int code;
  Py_BEGIN_ALLOW_THREADS;
  code = ibcomm_emu_rsag(w, all_gather, in.dtype, in.ptr, out.ptr, static_cast<size_t>(block), scale, channels, stream, 0);
  Py_END_ALLOW_THREADS;
  return Done(code);
  END_HANDLE_TH_ERRORS
}

// The tensors of a list as the norm and clipping take them: dense, on one GPU.  It
// holds on to the sequences, like RankTensors.
struct GradList {
  PyObject* in = nullptr;
  PyObject* out = nullptr;
  std::vector<ibcomm_grad_tensor> tensors;
  c10::Device device{c10::DeviceType::CUDA, 0};
  bool any_double = false;

  GradList() = default;
  GradList(const GradList&) = delete;
  GradList& operator=(const GradList&) = delete;
  ~GradList() {
    Py_XDECREF(in);
    Py_XDECREF(out);
  }

  static const at::Tensor* Dense(PyObject* o, int* dtype) {
    if (!THPVariable_Check(o)) {
      PyErr_SetString(PyExc_TypeError, "a torch.Tensor is expected");
      return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    *dtype = DTypeCode(t.scalar_type());
    if (*dtype < 0) {
      Raise(kNotSupported, (std::string("unsupported dtype ") + c10::toString(t.scalar_type())).c_str());
      return nullptr;
    }
    if (!t.is_cuda()) {
      Raise(kInvalidArgument, "tensors must live on the GPU");
      return nullptr;
    }
    // The order of the elements does not matter, only that nothing lies between them.
    if (t.layout() != c10::kStrided || !(t.is_contiguous() || t.is_non_overlapping_and_dense())) {
      Raise(kInvalidArgument, "tensors must be dense");
      return nullptr;
    }
    return &t;
  }

  // `outs`: None for the norm alone, the same sequence for clipping in place.
  bool Read(PyObject* ins, PyObject* outs) {
    in = PySequence_Fast(ins, "a sequence of tensors is expected");
    if (in == nullptr) return false;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(in);
    const bool clip = outs != Py_None, in_place = outs == ins;
    if (n == 0) {
      Raise(kInvalidArgument, "a tensor is expected at least");
      return false;
    }
    if (clip && !in_place) {
      out = PySequence_Fast(outs, "a sequence of tensors is expected");
      if (out == nullptr) return false;
      if (PySequence_Fast_GET_SIZE(out) != n) {
        Raise(kInvalidArgument, "one output per tensor is expected");
        return false;
      }
    }
    tensors.resize(static_cast<size_t>(n));
    for (Py_ssize_t i = 0; i < n; ++i) {
      ibcomm_grad_tensor& g = tensors[static_cast<size_t>(i)];
      const at::Tensor* t = Dense(PySequence_Fast_GET_ITEM(in, i), &g.dtype_in);
      if (t == nullptr) return false;
      if (i == 0) device = t->device();
      g.len_elements = static_cast<size_t>(t->numel());
      any_double = any_double || g.dtype_in == 1;
      g.in = t->const_data_ptr();
      g.out = nullptr;
      g.dtype_out = g.dtype_in;
      const at::Tensor* o = t;
      if (clip && !in_place) {
        o = Dense(PySequence_Fast_GET_ITEM(out, i), &g.dtype_out);
        if (o == nullptr) return false;
        if (o->sizes() != t->sizes() || !(o->strides() == t->strides() || (o->is_contiguous() && t->is_contiguous()))) {
          Raise(kInvalidArgument, "an output must match its tensor in shape and strides");
          return false;
        }
      }
      if (t->device() != device || o->device() != device) {
        Raise(kInvalidArgument, "the tensors must live on one GPU");
        return false;
      }
      if (clip) g.out = o->data_ptr();
    }
    return true;
  }
};

// Device memory of this call; freed into the current stream's pool.
at::Tensor Empty(at::IntArrayRef sizes, c10::ScalarType type, c10::Device device) {
  return at::empty(sizes, at::TensorOptions().dtype(type).device(device));
}

// The ranks' sums (float64, on the list's GPU), or None.
bool ToSums(PyObject* o, const GradList& list, const double** sums, int* count) {
  *sums = nullptr;
  *count = 0;
  if (o == Py_None) return true;
  int d;
  const at::Tensor* t = Tensor(o, &d);
  if (t == nullptr) return false;
  if (d != 1 || t->device() != list.device || t->numel() < 1 || t->numel() > (1 << 20)) {
    Raise(kInvalidArgument, "the ranks' sums must be float64 on the tensors' GPU");
    return false;
  }
  *sums = static_cast<const double*>(t->const_data_ptr());
  *count = static_cast<int>(t->numel());
  return true;
}

// grad_norm(tensors, power, sums, want_sum) -> the norm, or with want_sum the sum that ranks have to join (float64, one element)
PyObject* GradNorm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!WantArgs(n, 4)) return nullptr;
  GradList list;
  if (!list.Read(a[0], Py_None)) return nullptr;
  const int power = static_cast<int>(PyLong_AsLong(a[1]));
  const int want_sum = static_cast<int>(PyLong_AsLong(a[3]));
  const double* sums;
  int num_sums;
  if (PyErr_Occurred() || !ToSums(a[2], list, &sums, &num_sums)) return nullptr;
  const c10::cuda::CUDAGuard guard(list.device);
  at::Tensor work = Empty({IBCOMM_NORM_WORK}, c10::kDouble, list.device);
  at::Tensor result = want_sum ? Empty({1}, c10::kDouble, list.device) : Empty({}, list.any_double ? c10::kDouble : c10::kFloat, list.device);
  void* stream = c10::cuda::getCurrentCUDAStream(list.device.index()).stream();
  void* norm = want_sum ? nullptr : result.data_ptr();
  double* sum = want_sum ? static_cast<double*>(result.data_ptr()) : nullptr;
  double* w = static_cast<double*>(work.data_ptr());
  int code;
  Py_BEGIN_ALLOW_THREADS;
  code = ibcomm_grad_norm(list.tensors.data(), static_cast<int>(list.tensors.size()), power, sums, num_sums, w, norm, list.any_double ? 1 : 0, sum, stream);
  Py_END_ALLOW_THREADS;
  if (code != 0) return RaiseLast(code);
  return THPVariable_Wrap(std::move(result));
  END_HANDLE_TH_ERRORS
}

// clip_grads(tensors, outs, power, max_norm, sums) -> the norm; outs None: in place
PyObject* ClipGrads(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!WantArgs(n, 5)) return nullptr;
  GradList list;
  if (!list.Read(a[0], a[1] == Py_None ? a[0] : a[1])) return nullptr;
  const int power = static_cast<int>(PyLong_AsLong(a[2]));
  const double max_norm = PyFloat_AsDouble(a[3]);
  const double* sums;
  int num_sums;
  if (PyErr_Occurred() || !ToSums(a[4], list, &sums, &num_sums)) return nullptr;
  const c10::cuda::CUDAGuard guard(list.device);
  at::Tensor work = Empty({IBCOMM_NORM_WORK}, c10::kDouble, list.device);
  at::Tensor result = Empty({}, list.any_double ? c10::kDouble : c10::kFloat, list.device);
  void* stream = c10::cuda::getCurrentCUDAStream(list.device.index()).stream();
  void* norm = result.data_ptr();
  double* w = static_cast<double*>(work.data_ptr());
  int code;
  Py_BEGIN_ALLOW_THREADS;
  code = ibcomm_clip_grads(list.tensors.data(), static_cast<int>(list.tensors.size()), power, max_norm, sums, num_sums, w, norm, list.any_double ? 1 : 0, stream);
  Py_END_ALLOW_THREADS;
  if (code != 0) return RaiseLast(code);
  return THPVariable_Wrap(std::move(result));
  END_HANDLE_TH_ERRORS
}

// An error of the library on its way to Python, or to autograd.
struct LibraryError {
  int code;
  std::string message;
};
void Want(bool ok, int code, const char* message) {
  if (!ok) throw LibraryError{code, message};
}
void CheckCode(int code) {
  if (code == 0) return;
  std::string m = ibcomm_last_error();
  while (!m.empty() && (m.back() == '\n' || m.back() == ' ')) m.pop_back();
  throw LibraryError{code, m};
}

int FloatCode(const at::Tensor& t) {
  const int d = DTypeCode(t.scalar_type());
  if (d != 0 && d != 4 && d != 5) throw LibraryError{kNotSupported, std::string("no embedding of ") + c10::toString(t.scalar_type())};
  return d;
}

// Without the GIL; `tokens` and `weight` contiguous.
at::Tensor Lookup(const at::Tensor& tokens, const at::Tensor& weight, int out_dtype, double scale) {
  const c10::Device device = weight.device();
  const c10::cuda::CUDAGuard guard(device);
  c10::SmallVector<int64_t, 8> sizes(tokens.sizes().begin(), tokens.sizes().end());
  sizes.push_back(weight.size(1));
  at::Tensor out = Empty(sizes, out_dtype == 0 ? c10::kFloat : out_dtype == 4 ? c10::kHalf : c10::kBFloat16, device);
  CheckCode(ibcomm_embedding(tokens.const_data_ptr(), DTypeCode(tokens.scalar_type()), static_cast<size_t>(tokens.numel()), weight.const_data_ptr(),
                             FloatCode(weight), static_cast<size_t>(weight.size(0)), static_cast<size_t>(weight.size(1)), out.data_ptr(), out_dtype, scale,
                             c10::cuda::getCurrentCUDAStream(device.index()).stream()));
  return out;
}

// Without the GIL; all contiguous, on one GPU.
void AddGradient(const at::Tensor& tokens, const at::Tensor& grad, const at::Tensor& out, int64_t padding, double scale, bool accumulate) {
  Want(out.dim() == 2, kInvalidArgument, "a table has rows and columns");
  const size_t count = static_cast<size_t>(tokens.numel()), rows = static_cast<size_t>(out.size(0)), width = static_cast<size_t>(out.size(1));
  Want(grad.dim() >= 1 && grad.size(-1) == out.size(1) && static_cast<size_t>(grad.numel()) == count * width, kInvalidArgument,
       "grad must hold a row of the table's width for every token");
  Want(tokens.is_cuda() && tokens.device() == out.device() && grad.device() == out.device(), kInvalidArgument,
       "tokens, grad and table must live on the same GPU");
  const c10::Device device = out.device();
  const c10::cuda::CUDAGuard guard(device);
  size_t bytes = 0;
  CheckCode(ibcomm_embedding_grad_work(count, rows, width, &bytes));
  at::Tensor work;
  if (bytes > 0) work = Empty({static_cast<int64_t>(bytes)}, c10::kByte, device);
  CheckCode(ibcomm_embedding_grad(tokens.const_data_ptr(), DTypeCode(tokens.scalar_type()), count, grad.const_data_ptr(), FloatCode(grad), out.data_ptr(),
                                  FloatCode(out), rows, width, padding, scale, accumulate ? 1 : 0, bytes > 0 ? work.data_ptr() : nullptr, bytes,
                                  c10::cuda::getCurrentCUDAStream(device.index()).stream()));
}

// The embedding's place in autograd's graph: the table's gradient, or with `into` its addition to that tensor.
struct EmbeddingBackward : public torch::autograd::Node {
  torch::autograd::SavedVariable tokens;
  at::Tensor weight, into;
  double scale = 1.0;
  int64_t padding = -1;

  std::string name() const override { return "EmbeddingBackward"; }
  void release_variables() override {
    tokens.reset_data();
    released = true;
  }
  bool released = false;

  // A hook's dictionary stays with the tensor when the hook is taken out of it.
  bool Hooked() const {
    const std::shared_ptr<torch::autograd::Node> from = weight.grad_fn();
    const auto& hooks = from != nullptr ? from->tensor_pre_hooks() : torch::autograd::impl::hooks(weight);
    if (hooks.size() != 1) return !hooks.empty();
    const pybind11::gil_scoped_acquire locked;
    const auto table = pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(weight));
    const pybind11::object dictionary = pybind11::getattr(table, "_backward_hooks", pybind11::none());
    return dictionary.is_none() || pybind11::len(dictionary) != 0;
  }
  bool GradIsInto() const {
    if (!weight.is_leaf() || !weight.grad().defined() || weight.grad().layout() != c10::kStrided) return false;
    const at::Tensor& grad = weight.grad();
    return grad.data_ptr() == into.data_ptr() && grad.scalar_type() == into.scalar_type() && grad.is_contiguous();
  }

  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    TORCH_CHECK(!released, "the embedding's gradient was taken already; specify retain_graph=True to take it again");
    const at::Tensor& grad = grads[0];
    if (!grad.defined()) return {at::Tensor()};
    TORCH_CHECK(!(at::GradMode::is_enabled() && grad.requires_grad()), "the embedding's gradient can be taken once, not differentiated again");
    TORCH_CHECK(!grad._fw_grad(0).defined(), "the embedding's gradient has no forward-mode derivative");
    const at::NoGradGuard no_grad;
    const at::Tensor ids = tokens.unpack(), rows = grad.contiguous();
    // A hook of the table is to see, and may change, what is added.
    const bool hooked = into.defined() && Hooked();
    TORCH_CHECK(!hooked || GradIsInto(), "the table has a hook, which would not see a gradient that is added to another tensor than weight.grad");
    try {
      if (!into.defined() || hooked) {
        at::Tensor out = at::empty(weight.sizes(), weight.options());
        AddGradient(ids, rows, out, padding, scale, false);
        return {out};
      }
      AddGradient(ids, rows, into, padding, scale, true);
    } catch (const LibraryError& e) {
      TORCH_CHECK(false, "[ibcomm error ", e.code, "] ", e.message);
    }
    // A gradient without entries costs nothing to add, and takes the way of every other one: autograd makes the stream
    // of weight.grad wait for this one, adds other uses of the table and runs the bucket's hook, in that order.
    if (weight.is_leaf() && weight.grad().defined()) return {at::empty(weight.sizes(), weight.options().layout(c10::kSparse))};
    // Where nothing is handed on, the stream of the backward call waits at its end.
    const c10::Device device = into.device();
    auto done = std::make_shared<c10::Event>(c10::DeviceType::CUDA);
    done->record(c10::cuda::getCurrentCUDAStream(device.index()).unwrap());
    torch::autograd::Engine::get_default_engine().queue_callback([done, device] { done->block(c10::cuda::getCurrentCUDAStream(device.index()).unwrap()); });
    return {at::Tensor()};
  }
};

// embedding(tokens, weight, out_dtype, scale, padding_row, grad_into) -> rows; out_dtype < 0: the table's type
PyObject* Embedding(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!WantArgs(n, 6)) return nullptr;
  int dt, dw;
  // What is computed from the memory alone would lack the tangent, or be a constant of the trace.
  if (THPVariable_Check(a[1]) && THPVariable_Unpack(a[1])._fw_grad(0).defined())
    return Raise(kNotSupported, "the embedding has no forward-mode derivative");
  if (c10::impl::tls_local_dispatch_key_set().included_.has(c10::DispatchKey::Tracer)) return Raise(kNotSupported, "the embedding cannot be traced");
  const at::Tensor* tokens = Tensor(a[0], &dt);
  if (tokens == nullptr) return nullptr;
  const at::Tensor* weight = Tensor(a[1], &dw);
  if (weight == nullptr) return nullptr;
  const int wanted = static_cast<int>(PyLong_AsLong(a[2]));
  const double scale = PyFloat_AsDouble(a[3]);
  const int64_t padding = PyLong_AsLongLong(a[4]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor* into = nullptr;
  if (a[5] != Py_None) {
    int d;
    if ((into = Tensor(a[5], &d)) == nullptr) return nullptr;
  }
  if (weight->dim() != 2) return Raise(kInvalidArgument, "a table has rows and columns");
  if (!tokens->is_cuda() || !weight->is_cuda() || tokens->device() != weight->device())
    return Raise(kInvalidArgument, "tokens and table must live on the same GPU");
  const int out_dtype = wanted < 0 ? dw : wanted;
  if (out_dtype != 0 && out_dtype != 4 && out_dtype != 5) return Raise(kNotSupported, "rows are float32, float16 or bfloat16");
  try {
    at::Tensor out;
    {
      const pybind11::gil_scoped_release unlocked;
      out = Lookup(*tokens, *weight, out_dtype, scale);
      if (at::GradMode::is_enabled() && weight->requires_grad()) {
        const std::shared_ptr<EmbeddingBackward> node(new EmbeddingBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(*weight));
        node->tokens = torch::autograd::SavedVariable(*tokens, false);
        node->weight = *weight;
        if (into != nullptr) node->into = *into;
        node->scale = scale;
        node->padding = padding;
        torch::autograd::set_history(out, node);
      }
    }
    return THPVariable_Wrap(std::move(out));
  } catch (const LibraryError& e) {
    return Raise(e.code, e.message.c_str());
  }
  END_HANDLE_TH_ERRORS
}

// embedding_grad(tokens, grad, out, padding_row, scale, accumulate)
PyObject* EmbeddingGrad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!WantArgs(n, 6)) return nullptr;
  int dt, dg, dout;
  const at::Tensor* tokens = Tensor(a[0], &dt);
  if (tokens == nullptr) return nullptr;
  const at::Tensor* grad = Tensor(a[1], &dg);
  if (grad == nullptr) return nullptr;
  const at::Tensor* out = Tensor(a[2], &dout);
  if (out == nullptr) return nullptr;
  const int64_t padding = PyLong_AsLongLong(a[3]);
  const double scale = PyFloat_AsDouble(a[4]);
  const int accumulate = PyObject_IsTrue(a[5]);
  if (PyErr_Occurred()) return nullptr;
  try {
    const pybind11::gil_scoped_release unlocked;
    AddGradient(*tokens, *grad, *out, padding, scale, accumulate != 0);
  } catch (const LibraryError& e) {
    return Raise(e.code, e.message.c_str());
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"set_error", SetError, METH_O, "set_error(exception_class)"},
    {"allreduce", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(Allreduce)), METH_FASTCALL, nullptr},
    {"copy_scale", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(CopyScale)), METH_FASTCALL, nullptr},
    {"emu_allreduce", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(EmuAllreduce)), METH_FASTCALL, nullptr},
    {"emu_rsag", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(EmuRsAg)), METH_FASTCALL, nullptr},
    {"grad_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(GradNorm)), METH_FASTCALL, nullptr},
    {"clip_grads", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(ClipGrads)), METH_FASTCALL, nullptr},
    {"embedding", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(Embedding)), METH_FASTCALL, nullptr},
    {"embedding_grad", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(EmbeddingGrad)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fastcall", "Collectives on CUDA tensors without ctypes.", -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fastcall(void) { return PyModule_Create(&kModule); }
