// clip_list.cpp -- clip_gradients on Python's own lists of tensors.
//
// The dispatcher turns each tensor of a list argument into a value of its own
// and back: 0.17 us a tensor, which is most of a call with hundreds of small
// ones (157 gradients with outputs: 53 us).  This entry reads the lists
// where they are.  It uses no function of the Python library, only the layout
// of lists and tensors, so that the operator library still loads without one.
// What is not a plain tensor, or a call that something else listens to (a
// dispatch mode), goes through the operator.
#ifndef NDEBUG
#define NDEBUG  // the assertions of Python's macros refer to its types
#endif
#include <Python.h>

#include <c10/core/impl/TorchDispatchModeTLS.h>

#include <cstddef>
#include <cstring>
#include <string>
#include <vector>

#include "train_ops_common.h"

namespace {

using at::Tensor;

// How torch.Tensor begins (torch/csrc/autograd/python_variable.h, whose other
// contents would need the Python library).  Other versions of torch may hold the
// tensor another way: muon_ascend950_clip_reads tells.
struct PythonTensor {
  PyObject_HEAD Tensor tensor;
};
const Tensor& TensorOf(PyObject* object) { return reinterpret_cast<PythonTensor*>(object)->tensor; }

// Keys of tensors that stand for others, or need the dispatcher.
const c10::DispatchKeySet kSpecial = c10::functorch_transforms_ks | c10::python_ks |
                                     c10::DispatchKeySet({c10::DispatchKey::Functionalize, c10::DispatchKey::Conjugate,
                                                          c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor,
                                                          c10::DispatchKey::Sparse, c10::DispatchKey::SparseCsr,
                                                          c10::DispatchKey::Quantized});

bool Plain(const Tensor& t) { return t.defined() && t.has_storage() && !t.key_set().has_any(kSpecial); }

// Tensors of a list; false if one is not plain.
bool Unpack(PyObject* list, std::vector<const Tensor*>* to) {
  const Py_ssize_t n = PyList_GET_SIZE(list);
  to->reserve(static_cast<size_t>(n));
  for (Py_ssize_t i = 0; i < n; ++i) {
    to->push_back(&TensorOf(PyList_GET_ITEM(list, i)));
    if (!Plain(*to->back())) return false;
  }
  return true;
}

thread_local std::string message;

enum Status { kDone = 0, kValue = 1, kType = 2, kNotImplemented = 3, kRuntime = 4, kThroughTheOperator = 5 };

}  // namespace

// The word where this file takes the tensor of `object`, of the type torch.Tensor
// itself, to be; nothing is read through it.  It is the tensor's `_cdata` where the
// layout is as above, and only then may lists be passed to the entry below.
static_assert(sizeof(Tensor) == sizeof(uintptr_t), "a tensor is one pointer");
extern "C" __attribute__((visibility("default"))) uintptr_t muon_ascend950_clip_reads(PyObject* object) {
  if (static_cast<size_t>(Py_TYPE(object)->tp_basicsize) < sizeof(PythonTensor)) return 0;
  uintptr_t word;
  std::memcpy(&word, reinterpret_cast<const char*>(object) + offsetof(PythonTensor, tensor), sizeof(word));
  return word;
}

// `gradients` and `out` (or NULL): lists of objects of the type torch.Tensor
// itself, not empty; `norm`: such a tensor.  Called with the interpreter's lock.
// Errors come as a status; the message is this thread's until its next call.
extern "C" __attribute__((visibility("default"))) const char* muon_ascend950_clip_message() {
  return message.c_str();
}
extern "C" __attribute__((visibility("default"))) int muon_ascend950_clip_list(
    PyObject* gradients, PyObject* out, PyObject* norm, double max_norm, int largest) {
  const auto say = [](Status status, const char* what) {
    message = what;
    return static_cast<int>(status);
  };
  try {
    if (c10::impl::TorchDispatchModeTLS::any_modes_set()) return kThroughTheOperator;
    std::vector<const Tensor*> g, o;
    if (!Unpack(gradients, &g) || (out != nullptr && !Unpack(out, &o))) return kThroughTheOperator;
    const Tensor& n = TensorOf(norm);
    if (!Plain(n)) return kThroughTheOperator;
    if (out != nullptr && o.empty()) return say(kValue, "clip_gradients: out must have a tensor for each gradient");
    muon_train_ops::clip_gradients(g, o, max_norm, largest != 0, n);
    return kDone;
  } catch (const c10::ValueError& e) {
    return say(kValue, e.what_without_backtrace());
  } catch (const c10::TypeError& e) {
    return say(kType, e.what_without_backtrace());
  } catch (const c10::NotImplementedError& e) {
    return say(kNotImplemented, e.what_without_backtrace());
  } catch (const c10::Error& e) {
    return say(kRuntime, e.what_without_backtrace());
  } catch (const std::exception& e) {
    return say(kRuntime, e.what());
  }
}
