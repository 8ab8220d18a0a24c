// A call's tensors looked over in native code: where Python asks each of eleven tensors for its shape, type, device, layout and address, a call for
// one short sequence is bound by the host (one tree of 8 nodes: 15 us, of them 5 these questions; here under 1).
#include <ATen/core/Tensor.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

// specs: a tuple of (name, tensor, shape or None, dtype).  0 and the tensors' addresses when each is a contiguous tensor of its dtype and shape on
// GPU `device`; otherwise 1, and the caller finds out which is not.  Never throws, and leaves no Python error behind.
extern "C" __attribute__((visibility("default"))) int llg_tensor_addresses(PyObject* specs, int device, unsigned long long* addresses) {
  if (!PyTuple_Check(specs)) return 1;
  const Py_ssize_t n = PyTuple_GET_SIZE(specs);
  try {
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* spec = PyTuple_GET_ITEM(specs, i);
      if (!PyTuple_Check(spec) || PyTuple_GET_SIZE(spec) != 4) return 1;
      PyObject *given = PyTuple_GET_ITEM(spec, 1), *shape = PyTuple_GET_ITEM(spec, 2), *dtype = PyTuple_GET_ITEM(spec, 3);
      if (!THPVariable_Check(given) || !THPDtype_Check(dtype)) return 1;
      const at::Tensor& t = THPVariable_Unpack(given);
      if (t.scalar_type() != reinterpret_cast<THPDtype*>(dtype)->scalar_type || !t.is_cuda() || t.get_device() != device || !t.is_contiguous()) return 1;
      if (shape != Py_None) {
        if (!PyTuple_Check(shape) || PyTuple_GET_SIZE(shape) != t.dim()) return 1;
        for (Py_ssize_t d = 0; d < t.dim(); ++d) {
          const long long want = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, d));
          if (want == -1 && PyErr_Occurred()) {
            PyErr_Clear();
            return 1;
          }
          if (want != t.size(d)) return 1;
        }
      }
      addresses[i] = reinterpret_cast<unsigned long long>(t.data_ptr());
    }
  } catch (...) {
    return 1;
  }
  return 0;
}
