// Python extension `muon_b200._tables`: multi-tensor calls from lists of tensors. It checks the lists, lays
// out their pointer tables and calls the C entry points of libmuon_b200 (include/muon_b200.h) on the current
// stream of the tensors' device. With hundreds of tensors and five lists the same checks written in
// Python take longer than the kernel of the call. No arithmetic happens here.
#include <Python.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/muon_b200.h"

#include <algorithm>
#include <array>
#include <cstdint>
#include <utility>
#include <vector>

namespace {

// Bits of the element types, in the order of the MUON_B200_F32, _BF16, _F16 codes; then uint8.
constexpr int kF32 = 1, kBF16 = 2, kF16 = 4, kU8 = 8, kFloats = 7;
int type_bit(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return kF32;
    case at::kBFloat16: return kBF16;
    case at::kHalf: return kF16;
    case at::kByte: return kU8;
    default: return 0;
  }
}
int type_code(int bit) { return bit == kF32 ? MUON_B200_F32 : bit == kBF16 ? MUON_B200_BF16 : MUON_B200_F16; }
const char* type_names(int mask) {
  return mask == kF32 ? "float32" : mask == kU8 ? "uint8" : "float32, bfloat16 or float16";
}

// Whether two tensors have one shape and their elements in one order (dimensions of size 1 have none).
bool same_order(const at::Tensor& a, const at::Tensor& b) {
  if (a.sizes() != b.sizes()) return false;
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) != 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}

struct Ref {  // owned reference
  PyObject* p;
  explicit Ref(PyObject* o = nullptr) : p(o) {}
  Ref(const Ref&) = delete;
  Ref& operator=(const Ref&) = delete;
  ~Ref() { Py_XDECREF(p); }
  PyObject* release() { return std::exchange(p, nullptr); }
};

using Range = std::pair<uintptr_t, uintptr_t>;
using Table = std::vector<void*>;
enum Layout { kLikeFirst, kScales };  // sizes of a list: those of the first list, or one per block of its elements
// What a call does with a list. kUpdates: writes tensors that a backward pass may have saved, and counts a version of
// them as torch's in-place functions do. Moments, masters, codes and scales are state that nothing but a step reads: kWrites
// (counting a version takes 13 ns a tensor, a third of what the tensor takes in all).
enum Use { kReads, kWrites, kUpdates };

// The lists of one call. All tensors are on one device; what is written overlaps nothing else of the call (tensors
// that are only read may share memory).
struct Lists {
  // Part of the memory of a list: ranges[first .. last), all of it in [low, high). Lists mostly come in a few runs
  // that ascend, from as many segments of the allocator.
  struct Run {
    size_t first, last;
    uintptr_t low, high;
    bool written;
    bool ordered;  // ascending or descending, and apart from one another
  };
  static constexpr size_t kMostRuns = 24, kMostLists = 8;  // (seven, and the factor)
  const char* what;
  Py_ssize_t n = 0;
  int64_t device = -1;
  std::vector<int64_t> numel;
  std::vector<int> codes;  // element types of the first list
  std::vector<Range> ranges;
  std::array<Run, kMostRuns + kMostLists> runs;
  size_t n_runs = 0;
  std::vector<at::TensorImpl*> changed;
  std::array<Ref, kMostLists> held;  // the lists themselves (one made of an iterator's tensors may be all that holds them)
  int n_held = 0;
  const int most;  // lists, at most; 0: one, and nothing is written

  Lists(const char* w, int most_lists) : what(w), most(most_lists) {}

  // Adds a list; false with a Python error set. `found`: mask of the types in it.
  bool add(const char* name, PyObject* tensors, int types, Layout layout, Use use, Table& table, int& found) {
    Ref fast(PySequence_Fast(tensors, "lists of tensors are lists or tuples"));
    if (!fast.p) return false;
    const Py_ssize_t count = PySequence_Fast_GET_SIZE(fast.p);
    const bool is_first = n_held == 0;
    if (is_first) {
      n = count;
      numel.resize(n);
      codes.resize(n);
      if (most > 0) ranges.reserve(most * n + 1);
    } else if (count != n) {
      PyErr_Format(PyExc_ValueError, "%s: %zd %s tensors for %zd tensors", what, count, name, n);
      return false;
    }
    table.resize(n);
    found = 0;
    const bool writes = use != kReads;
    const size_t begin = ranges.size();
    if (use == kUpdates) changed.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* o = PySequence_Fast_GET_ITEM(fast.p, i);
      if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s: %s %zd is no tensor but %.80s", what, name, i, Py_TYPE(o)->tp_name);
        return false;
      }
      const at::Tensor& t = THPVariable_Unpack(o);
      const at::Device where = t.device();
      if (!where.is_cuda()) {
        PyErr_Format(PyExc_RuntimeError,
                     "muon_b200: every %s tensor of %s must live on a CUDA (sm_100) device, got device=%s; "
                     "there is no CPU implementation", name, what, where.str().c_str());
        return false;
      }
      if (device < 0) device = where.index();
      if (where.index() != device) {
        PyErr_Format(PyExc_ValueError, "%s: %s tensors must all be on cuda:%lld, got %s", what, name,
                     (long long)device, where.str().c_str());
        return false;
      }
      const int bit = type_bit(t.scalar_type());
      if (!(bit & types)) {
        Ref dtype(PyObject_GetAttrString(o, "dtype"));
        if (dtype.p)
          PyErr_Format(PyExc_ValueError, "%s: %s tensors must be %s, got %S", what, name, type_names(types), dtype.p);
        return false;
      }
      found |= bit;
      if (!t.has_storage() || t.is_neg()) {  // (sparse ones, say; the negative of another tensor's memory)
        PyErr_Format(PyExc_ValueError, "%s: %s %zd has no memory of its own", what, name, i);
        return false;
      }
      const int64_t size = t.numel();
      bool dense;
      if (is_first) {
        numel[i] = size;
        codes[i] = type_code(bit);
        dense = t.is_contiguous() || t.is_non_overlapping_and_dense();
      } else {
        const at::Tensor& ref = THPVariable_Unpack(PySequence_Fast_GET_ITEM(held[0].p, i));
        const int64_t want =
            layout == kLikeFirst ? numel[i] : (numel[i] + MUON_B200_STATE_BLOCK - 1) / MUON_B200_STATE_BLOCK;
        if (size != want) {
          PyErr_Format(PyExc_ValueError, "%s: %s tensor %zd has another number of elements than it must have "
                       "(%lld, not %lld)", what, name, i, (long long)size, (long long)want);
          return false;
        }
        dense = t.is_contiguous() && (layout == kScales || ref.is_contiguous());
        if (!dense && layout == kLikeFirst)  // the first list's tensor is dense
          dense = same_order(t, ref);
      }
      if (!dense && size > 1) {
        PyErr_Format(PyExc_ValueError, "%s: %s tensors must be contiguous, or dense with the strides of the tensor they "
                     "belong to (tensor %zd)", what, name, i);
        return false;
      }
      table[i] = size == 0 ? nullptr : writes ? t.mutable_data_ptr() : const_cast<void*>(t.const_data_ptr());
      if (use == kUpdates && !t.is_inference()) changed.push_back(t.unsafeGetTensorImpl());
      if (size > 0 && most > 0) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(table[i]);
        ranges.emplace_back(at, at + size * t.element_size());
      }
    }
    held[n_held++].p = fast.release();
    add_runs(begin, writes);
    return true;
  }

  // The ranges from `begin` on: the memory of one list, as runs that ascend or descend.
  void add_runs(size_t begin, bool written) {
    for (size_t i = begin; i < ranges.size();) {
      Run r = {i, i + 1, ranges[i].first, ranges[i].second, written, true};
      const bool rest = n_runs + 1 >= kMostRuns;  // too many to compare with one another
      bool up = true, down = true;
      for (; r.last < ranges.size(); ++r.last) {
        const Range &before = ranges[r.last - 1], &now = ranges[r.last];
        up = up && now.first >= before.second;
        down = down && now.second <= before.first;
        if (!up && !down && !rest) break;
        r.low = std::min(r.low, now.first);
        r.high = std::max(r.high, now.second);
      }
      r.ordered = up || down || !rest;
      runs[n_runs++] = r;
      i = r.last;
    }
  }

  // After the last list: false with a Python error set when memory that is written appears twice in the call. Runs
  // that share no span of addresses with another one are apart already; the others are sorted and compared.
  bool apart() const {
    std::vector<Range> written, read;
    for (size_t k = 0; k < n_runs; ++k) {
      const Run& r = runs[k];
      bool compare = r.written && !r.ordered;
      for (size_t j = 0; j < n_runs; ++j) {
        const Run& o = runs[j];
        compare = compare || (j != k && (o.written || r.written) && o.low < r.high && r.low < o.high);
      }
      if (!compare) continue;
      std::vector<Range>& to = r.written ? written : read;
      const size_t middle = to.size();
      to.insert(to.end(), ranges.begin() + r.first, ranges.begin() + r.last);
      if (!std::is_sorted(to.begin() + middle, to.end())) std::sort(to.begin() + middle, to.end());
      std::inplace_merge(to.begin(), to.begin() + middle, to.end());
    }
    for (size_t i = 1; i < written.size(); ++i)
      if (written[i - 1].second > written[i].first) {
        PyErr_Format(PyExc_ValueError, "%s: memory that is written appears twice in the call", what);
        return false;
      }
    size_t w = 0;  // first written range that ends behind the start of this read one
    for (const Range& r : read) {
      while (w < written.size() && written[w].second <= r.first) ++w;
      if (w < written.size() && written[w].first < r.second) {
        PyErr_Format(PyExc_ValueError, "%s: memory that is written overlaps memory that is read", what);
        return false;
      }
    }
    return true;
  }

  // After the library's call: autograd learns that the tensors have new values, as it does from torch's functions.
  int done(int rc) const {
    if (rc == 0)
      for (at::TensorImpl* t : changed) t->bump_version();
    return rc;
  }

  // The code of a list that must have one type; -1 with a Python error set.
  int one_type(int mask, const char* name) const {
    if (!(mask & (mask - 1))) return type_code(mask);
    PyErr_Format(PyExc_ValueError, "%s needs %s tensors of one dtype", what, name);
    return -1;
  }
};

// steps: one integer for all, or a sequence of n.
bool read_steps(const Lists& lists, PyObject* o, std::vector<int64_t>& steps) {
  steps.resize(lists.n);
  if (PyLong_Check(o)) {
    const int64_t s = PyLong_AsLongLong(o);
    if (s == -1 && PyErr_Occurred()) return false;
    std::fill(steps.begin(), steps.end(), s);
    return true;
  }
  Ref fast(PySequence_Fast(o, "steps are an integer or a list of integers"));
  if (!fast.p) return false;
  if (PySequence_Fast_GET_SIZE(fast.p) != lists.n) {
    PyErr_Format(PyExc_ValueError, "%s: %zd steps for %zd tensors", lists.what, PySequence_Fast_GET_SIZE(fast.p), lists.n);
    return false;
  }
  for (Py_ssize_t i = 0; i < lists.n; ++i) {
    steps[i] = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(fast.p, i));
    if (steps[i] == -1 && PyErr_Occurred()) return false;
  }
  return true;
}

// adamw(params, grads, masters or None, (moment lists), steps, lr, weight_decay, beta1, beta2, eps,
//       grad_scale or None, seed) -> status. Two moment lists: float32; four: 8-bit codes and scales of both.
PyObject* adamw(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *params, *grads, *masters, *moments, *steps_o, *scale;
  double lr, wd, b1, b2, eps;
  unsigned int seed;
  if (!PyArg_ParseTuple(args, "OOOO!OdddddOI", &params, &grads, &masters, &PyTuple_Type, &moments, &steps_o, &lr, &wd,
                        &b1, &b2, &eps, &scale, &seed))
    return nullptr;
  const bool eight = PyTuple_GET_SIZE(moments) == 4;
  if (!eight && PyTuple_GET_SIZE(moments) != 2) return PyErr_Format(PyExc_ValueError, "two or four lists of moments");
  Lists lists(eight ? "adamw8_step" : "adamw_step", eight ? 7 : 5);
  Table p, g, w, m[4];
  int p_types = 0, g_types = 0, found = 0;
  const bool has_masters = masters != Py_None;
  if (!lists.add("parameter", params, kFloats, kLikeFirst, kUpdates, p, p_types) ||
      !lists.add("gradient", grads, kFloats, kLikeFirst, kReads, g, g_types) ||
      (has_masters && !lists.add("master", masters, kF32, kLikeFirst, kWrites, w, found)))
    return nullptr;
  static const char* const names32[] = {"exp_avg", "exp_avg_sq"};
  static const char* const names8[] = {"exp_avg code", "exp_avg scale", "exp_avg_sq code", "exp_avg_sq scale"};
  for (int k = 0; k < (eight ? 4 : 2); ++k) {
    const bool scales = eight && k % 2 == 1;
    if (!lists.add(eight ? names8[k] : names32[k], PyTuple_GET_ITEM(moments, k), eight && !scales ? kU8 : kF32,
                   scales ? kScales : kLikeFirst, kWrites, m[k], found))
      return nullptr;
  }
  if (lists.n == 0) return PyLong_FromLong(0);
  const int code = lists.one_type(p_types, "parameter"), grad_code = code < 0 ? -1 : lists.one_type(g_types, "gradient");
  if (grad_code < 0) return nullptr;
  if (grad_code != code && grad_code != MUON_B200_F32)
    return PyErr_Format(PyExc_ValueError, "%s: gradient tensors must be of the parameters' type or float32", lists.what);
  if (has_masters && code == MUON_B200_F32)
    return PyErr_Format(PyExc_ValueError, "%s: float32 parameters have no master weights", lists.what);
  std::vector<int64_t> steps;
  if (!read_steps(lists, steps_o, steps)) return nullptr;
  const float* factor = nullptr;
  if (scale != Py_None) {
    const at::Tensor* t = THPVariable_Check(scale) ? &THPVariable_Unpack(scale) : nullptr;
    if (!t || !t->is_cuda() || t->get_device() != lists.device || t->scalar_type() != at::kFloat || t->numel() != 1)
      return PyErr_Format(PyExc_ValueError, "%s: grad_scale must be one float32 value on cuda:%lld", lists.what,
                          (long long)lists.device);
    factor = static_cast<const float*>(t->const_data_ptr());
    lists.ranges.emplace_back(reinterpret_cast<uintptr_t>(factor), reinterpret_cast<uintptr_t>(factor + 1));
    lists.add_runs(lists.ranges.size() - 1, false);
  }
  if (!lists.apart()) return nullptr;
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(lists.device));
  void* stream = c10::cuda::getCurrentCUDAStream().stream();
  void* const* wp = has_masters ? w.data() : nullptr;
  const int n = static_cast<int>(lists.n);
  const int rc = eight ? muon_b200_adamw8(p.data(), wp, g.data(), m[0].data(), m[1].data(), m[2].data(), m[3].data(),
                                          lists.numel.data(), steps.data(), n, code, grad_code, lr, wd, b1, b2, eps, seed,
                                          factor, stream)
                       : muon_b200_adamw(p.data(), wp, g.data(), m[0].data(), m[1].data(), lists.numel.data(),
                                         steps.data(), n, code, grad_code, lr, wd, b1, b2, eps, factor, stream);
  return PyLong_FromLong(lists.done(rc));
  END_HANDLE_TH_ERRORS
}

// convert(what, values, codes, scales, kind, to_codes) -> status
PyObject* convert(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  const char* what;
  PyObject *values, *codes, *scales;
  int kind, to_codes;
  if (!PyArg_ParseTuple(args, "sOOOip", &what, &values, &codes, &scales, &kind, &to_codes)) return nullptr;
  Lists lists(what, 3);
  Table x, c, s;
  int found = 0, types = 0;
  if (!lists.add("code", codes, kU8, kLikeFirst, to_codes ? kWrites : kReads, c, found) ||
      !lists.add("scale", scales, kF32, kScales, to_codes ? kWrites : kReads, s, found) ||
      !lists.add("value", values, kFloats, kLikeFirst, to_codes ? kReads : kUpdates, x, types))
    return nullptr;
  if (lists.n == 0) return PyLong_FromLong(0);
  const int code = lists.one_type(types, "value");
  if (code < 0 || !lists.apart()) return nullptr;
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(lists.device));
  void* stream = c10::cuda::getCurrentCUDAStream().stream();
  const int n = static_cast<int>(lists.n);
  const int rc = to_codes
      ? muon_b200_quantize_state(x.data(), c.data(), s.data(), lists.numel.data(), n, code, kind, stream)
      : muon_b200_dequantize_state(c.data(), s.data(), x.data(), lists.numel.data(), n, code, kind, stream);
  return PyLong_FromLong(lists.done(rc));
  END_HANDLE_TH_ERRORS
}

// grad_norm(tensors, max_norm, clip, scratch) -> (status, norm, factor; None with clip). scratch(device) returns the address of
// muon_b200_grad_norm_scratch_bytes() bytes that this call may use, as an integer.
PyObject* grad_norm(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *tensors, *scratch;
  double max_norm;
  int clip;
  if (!PyArg_ParseTuple(args, "OdpO", &tensors, &max_norm, &clip, &scratch)) return nullptr;
  Lists lists(clip ? "clip_grad_norm_" : "grad_norm", clip ? 1 : 0);
  Table x;
  int found = 0;
  if (!lists.add("gradient", tensors, kFloats, kLikeFirst, clip ? kUpdates : kReads, x, found)) return nullptr;
  if (lists.n == 0) return PyErr_Format(PyExc_ValueError, "%s: no tensors", lists.what);
  if (!lists.apart()) return nullptr;
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(lists.device));
  void* stream = c10::cuda::getCurrentCUDAStream().stream();
  Ref held(PyObject_CallFunction(scratch, "LN", (long long)lists.device, PyLong_FromVoidPtr(stream)));
  if (!held.p) return nullptr;
  if (!THPVariable_Check(held.p)) return PyErr_Format(PyExc_TypeError, "scratch is no tensor");
  const at::Tensor& room = THPVariable_Unpack(held.p);
  const uintptr_t at = (reinterpret_cast<uintptr_t>(room.data_ptr()) + 255) & ~uintptr_t(255);
  const int64_t bytes = room.numel() - static_cast<int64_t>(at - reinterpret_cast<uintptr_t>(room.data_ptr()));
  const at::Tensor out = at::empty({2}, at::TensorOptions().dtype(at::kFloat).device(at::kCUDA, lists.device));
  const int n = static_cast<int>(lists.n);
  float* result = out.mutable_data_ptr<float>();
  const int rc = clip ? muon_b200_clip_grads(x.data(), lists.numel.data(), lists.codes.data(), n, max_norm, result,
                                             reinterpret_cast<void*>(at), bytes, stream)
                      : muon_b200_grad_norm(x.data(), lists.numel.data(), lists.codes.data(), n, max_norm, result,
                                            reinterpret_cast<void*>(at), bytes, stream);
  return Py_BuildValue("iNN", lists.done(rc), THPVariable_Wrap(out.select(0, 0)),
                       clip ? Py_NewRef(Py_None) : THPVariable_Wrap(out.select(0, 1)));
  END_HANDLE_TH_ERRORS
}

// gradients(tensors) -> list: parameters give their .grad, other tensors themselves; None is left out.
PyObject* gradients(PyObject*, PyObject* tensors) {
  HANDLE_TH_ERRORS
  Ref fast(PySequence_Fast(tensors, "parameters or gradients are wanted")), out(PyList_New(0));
  if (!fast.p || !out.p) return nullptr;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast.p);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PySequence_Fast_GET_ITEM(fast.p, i);
    int parameter = 0;  // (a subclass of torch.Tensor may be one without being its subtype)
    if (Py_TYPE(o) == reinterpret_cast<PyTypeObject*>(ParameterClass)) parameter = 1;
    else if (Py_TYPE(o) != reinterpret_cast<PyTypeObject*>(THPVariableClass)) parameter = PyObject_IsInstance(o, ParameterClass);
    if (parameter < 0) return nullptr;
    if (!parameter && THPVariable_Check(o)) {  // or a plain leaf: an optimizer takes those too
      const at::Tensor& t = THPVariable_Unpack(o);
      parameter = t.requires_grad() && t.is_leaf();
    }
    Ref g(parameter ? PyObject_GetAttrString(o, "grad") : Py_NewRef(o));
    if (!g.p || (g.p != Py_None && PyList_Append(out.p, g.p) < 0)) return nullptr;
  }
  return out.release();
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"adamw", adamw, METH_VARARGS, "One AdamW step on lists of tensors."},
    {"convert", convert, METH_VARARGS, "Moments in 32 bits <-> codes and scales."},
    {"grad_norm", grad_norm, METH_VARARGS, "Norm of a list of tensors and the factor that clips it."},
    {"gradients", gradients, METH_O, "The gradients of parameters, or the tensors themselves."},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tables", "Multi-tensor calls from lists of tensors.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tables(void) { return PyModule_Create(&module); }
