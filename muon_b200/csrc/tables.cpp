// Python extension `muon_b200._tables`: checks the tensor lists of a multi-tensor call and lays out
// their pointer tables. With hundreds of tensors and five lists, the same checks written in Python take
// longer than the kernel of the call. No arithmetic and no CUDA call happens here; the tables go to the
// C entry points of libmuon_b200.
#include <Python.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <utility>
#include <vector>

namespace {

constexpr int kStateBlock = 256;  // elements per scale of 8-bit state (MUON_B200_STATE_BLOCK)

// Bits of the element types, in the order of the MUON_B200_F32, _BF16, _F16 codes; then uint8.
int type_bit(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return 1;
    case at::kBFloat16: return 2;
    case at::kHalf: return 4;
    case at::kByte: return 8;
    default: return 0;
  }
}
const char* type_names(int mask) {
  switch (mask) {
    case 1: return "float32";
    case 8: return "uint8";
    case 7: return "float32, bfloat16 or float16";
    case 3: return "float32 or bfloat16";
    case 5: return "float32 or float16";
    case 2: return "bfloat16";
    case 4: return "float16";
    default: return "of a supported type";
  }
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

// Sorted `more` into sorted `all`; false when two ranges overlap. Lists mostly come in ascending order of
// address, so this is linear.
bool merge_ranges(std::vector<Range>& all, std::vector<Range>& more) {
  if (!std::is_sorted(more.begin(), more.end())) std::sort(more.begin(), more.end());
  const size_t middle = all.size();
  all.insert(all.end(), more.begin(), more.end());
  std::inplace_merge(all.begin(), all.begin() + middle, all.end());
  for (size_t i = 1; i < all.size(); ++i)
    if (all[i - 1].second > all[i].first) return false;
  return true;
}

// collect(what, ((name, tensors, types, layout, written), ...)) ->
//   (device index, numel table, (address table per list, ...), (types found per list, ...), type codes of list 0)
// types: mask of type_bit; layout 0: the sizes and strides of the first list, 1: one float per
// kStateBlock elements of it; written: must not overlap another written tensor.
PyObject* collect(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  const char* what;
  PyObject* lists;
  if (!PyArg_ParseTuple(args, "sO!", &what, &PyTuple_Type, &lists)) return nullptr;
  const Py_ssize_t n_lists = PyTuple_GET_SIZE(lists);
  Ref tables(PyTuple_New(n_lists)), found(PyTuple_New(n_lists)), numel_table, code_table, first_fast;
  if (!tables.p || !found.p) return nullptr;
  Py_ssize_t n = 0;
  int64_t device = -1;
  int64_t* numel = nullptr;
  int32_t* codes = nullptr;
  std::vector<Range> written_ranges, ranges;
  for (Py_ssize_t l = 0; l < n_lists; ++l) {
    const char* name;
    PyObject* tensors;
    int types, layout, written;
    if (!PyArg_ParseTuple(PyTuple_GET_ITEM(lists, l), "sOiip", &name, &tensors, &types, &layout, &written)) return nullptr;
    Ref fast(PySequence_Fast(tensors, "lists of tensors are lists or tuples"));
    if (!fast.p) return nullptr;
    const Py_ssize_t count = PySequence_Fast_GET_SIZE(fast.p);
    if (l == 0) {
      n = count;
      numel_table.p = PyBytes_FromStringAndSize(nullptr, n * 8);
      code_table.p = PyBytes_FromStringAndSize(nullptr, n * 4);
      if (!numel_table.p || !code_table.p) return nullptr;
      numel = reinterpret_cast<int64_t*>(PyBytes_AS_STRING(numel_table.p));
      codes = reinterpret_cast<int32_t*>(PyBytes_AS_STRING(code_table.p));
    } else if (count != n) {
      return PyErr_Format(PyExc_ValueError, "%s: %zd %s tensors for %zd tensors", what, count, name, n);
    }
    Ref table(PyBytes_FromStringAndSize(nullptr, n * 8));
    if (!table.p) return nullptr;
    uint64_t* address = reinterpret_cast<uint64_t*>(PyBytes_AS_STRING(table.p));
    int mask = 0;
    ranges.clear();
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* o = PySequence_Fast_GET_ITEM(fast.p, i);
      if (!THPVariable_Check(o))
        return PyErr_Format(PyExc_TypeError, "%s: %s %zd is no tensor but %.80s", what, name, i, Py_TYPE(o)->tp_name);
      const at::Tensor& t = THPVariable_Unpack(o);
      if (!t.is_cuda())
        return PyErr_Format(PyExc_RuntimeError,
                            "muon_b200: every %s tensor of %s must live on a CUDA (sm_100) device, got device=%s; "
                            "there is no CPU implementation",
                            name, what, t.device().str().c_str());
      if (device < 0) device = t.get_device();
      else if (t.get_device() != device)
        return PyErr_Format(PyExc_ValueError, "%s: %s tensors must all be on cuda:%lld, got %s", what, name,
                            (long long)device, t.device().str().c_str());
      const int bit = type_bit(t.scalar_type());
      if (!(bit & types)) {
        Ref dtype(PyObject_GetAttrString(o, "dtype"));
        if (!dtype.p) return nullptr;
        return PyErr_Format(PyExc_ValueError, "%s: %s tensors must be %s, got %S", what, name, type_names(types), dtype.p);
      }
      mask |= bit;
      if (!t.has_storage())
        return PyErr_Format(PyExc_ValueError, "%s: %s %zd has no memory of its own (a sharded tensor? pass its local part)",
                            what, name, i);
      const int64_t size = t.numel();
      bool dense;
      if (l == 0) {
        numel[i] = size;
        codes[i] = bit == 1 ? 0 : bit == 2 ? 1 : 2;
        dense = t.is_contiguous() || t.is_non_overlapping_and_dense();
      } else {
        const at::Tensor& ref = THPVariable_Unpack(PySequence_Fast_GET_ITEM(first_fast.p, i));
        const int64_t want = layout == 0 ? numel[i] : (numel[i] + kStateBlock - 1) / kStateBlock;
        if (size != want)
          return PyErr_Format(PyExc_ValueError, "%s: %s tensor %zd has another number of elements than it must have "
                              "(%lld, not %lld)", what, name, i, (long long)size, (long long)want);
        dense = t.is_contiguous() && (layout == 1 || ref.is_contiguous());
        if (!dense && layout == 0)
          dense = t.sizes() == ref.sizes() && t.strides() == ref.strides();  // ref is dense
      }
      if (!dense && size > 1)
        return PyErr_Format(PyExc_ValueError, "%s: %s tensors must be contiguous, or dense with the strides of the "
                            "tensor they belong to (tensor %zd)", what, name, i);
      void* p = size == 0 ? nullptr : written ? t.mutable_data_ptr() : const_cast<void*>(t.const_data_ptr());
      address[i] = reinterpret_cast<uint64_t>(p);
      if (written && size > 0)
        ranges.emplace_back(reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + size * t.element_size());
    }
    if (written && !merge_ranges(written_ranges, ranges))
      return PyErr_Format(PyExc_ValueError, "%s: memory that is written (%s) appears twice in the call", what, name);
    PyObject* m = PyLong_FromLong(mask);
    if (!m) return nullptr;
    PyTuple_SET_ITEM(found.p, l, m);
    PyTuple_SET_ITEM(tables.p, l, table.release());
    if (l == 0) first_fast.p = fast.release();
  }
  return Py_BuildValue("LNNNN", (long long)device, numel_table.release(), tables.release(), found.release(),
                       code_table.release());
  END_HANDLE_TH_ERRORS
}

// gradients(tensors) -> list: parameters give their .grad, other tensors themselves; None is left out.
PyObject* gradients(PyObject*, PyObject* tensors) {
  HANDLE_TH_ERRORS
  Ref fast(PySequence_Fast(tensors, "a list of parameters or gradients is wanted")), out(PyList_New(0));
  if (!fast.p || !out.p) return nullptr;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast.p);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PySequence_Fast_GET_ITEM(fast.p, i);
    int parameter = 0;  // (a plain torch.Tensor is none; a subclass may be one without being its subtype)
    if (Py_TYPE(o) == reinterpret_cast<PyTypeObject*>(ParameterClass)) parameter = 1;
    else if (Py_TYPE(o) != reinterpret_cast<PyTypeObject*>(THPVariableClass)) parameter = PyObject_IsInstance(o, ParameterClass);
    if (parameter < 0) return nullptr;
    Ref g(parameter ? PyObject_GetAttrString(o, "grad") : Py_NewRef(o));
    if (!g.p || (g.p != Py_None && PyList_Append(out.p, g.p) < 0)) return nullptr;
  }
  return out.release();
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"gradients", gradients, METH_O, "The gradients of parameters, or the tensors themselves."},
                         {"collect", collect, METH_VARARGS, "Checks tensor lists and returns their pointer tables."},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tables", "Pointer tables of multi-tensor calls.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tables(void) { return PyModule_Create(&module); }
