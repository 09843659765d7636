// CPython helper of the Python layer, for what costs more on the host than on the device:
//   - reading the pointers, sizes and types of a list of tensors (clip_grad_norm_ is handed
//     hundreds per step; asking each from Python takes about 0.3 us per property);
//   - the usual call of an entry point with tensors that need no explanation: checks,
//     outputs, workspace, stream and the library call in one step (joiner_logits of eight
//     rows: 21 us through ctypes, the kernels take 8).  Whatever is not the usual case is
//     answered with None, and the Python function then takes its own way and says what is
//     wrong;
//   - the autograd node of joiner_logits.
// libot_b200.so itself knows nothing of torch; its functions come in by address (bind).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdexcept>
#include <vector>

#include "../../include/ot_b200.h"

namespace {

// Element type as the library's flags say it; -1 for a type it does not take.
int type_flag(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return 0;
    case at::kDouble: return OT_B200_FP64;
    case at::kBFloat16: return OT_B200_BF16;
    case at::kHalf: return OT_B200_FP16;
    default: return -1;
  }
}

template <typename T> PyObject *as_bytes(const std::vector<T> &v) {
  return PyBytes_FromStringAndSize(reinterpret_cast<const char *>(v.data()), (Py_ssize_t)(v.size() * sizeof(T)));
}

// Runs f; what it throws becomes the Python exception that torch makes of it (a failed
// allocation torch.OutOfMemoryError).
template <typename F> PyObject *guarded(F f) {
  HANDLE_TH_ERRORS
  return f();
  END_HANDLE_TH_ERRORS
}

// Whether there may be forward-mode dual numbers at all: asking once spares hundreds of tensors the question (25 ns each).
bool forward_mode() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }

// Whether t is a forward-mode dual number (none is while forward mode is switched off).
bool has_tangent(const at::Tensor &t) { return t._fw_grad(/*level=*/0).defined(); }

// describe(list) -> (pointers, counts, type flags, device, index, why): three bytes objects
// with one 64-, 64- and 32-bit entry per tensor, and the CUDA device all are on; or, at the
// first tensor that will not do, None four times, its index and "tensor" / "layout" /
// "type" / "cpu" / "device" / "dual".  "Dense" means one stretch of memory, each element once.
PyObject *describe(PyObject *, PyObject *list) {
  PyObject *seq = PySequence_Fast(list, "expected a sequence of tensors");
  if (seq == nullptr) return nullptr;
  PyObject *result = guarded([&]() -> PyObject * {
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
    PyObject **items = PySequence_Fast_ITEMS(seq);
    std::vector<int64_t> pointers((size_t)n), counts((size_t)n);
    std::vector<int32_t> types((size_t)n);
    int device = -1;
    const bool duals = forward_mode();
    const char *why = nullptr;
    Py_ssize_t i = 0;
    for (; i < n; ++i) {
      if (!THPVariable_Check(items[i])) { why = "tensor"; break; }
      const at::Tensor &t = THPVariable_Unpack(items[i]);
      if (t.layout() != at::kStrided) { why = "layout"; break; }
      if (!t.is_cuda()) { why = "cpu"; break; }
      if (i == 0) device = (int)t.get_device();
      if ((int)t.get_device() != device) { why = "device"; break; }
      const int flag = type_flag(t.scalar_type());
      if (flag < 0) { why = "type"; break; }
      if (!t.is_contiguous() && !t.is_non_overlapping_and_dense()) { why = "layout"; break; }
      if (duals && has_tangent(t)) { why = "dual"; break; }
      pointers[(size_t)i] = (int64_t)reinterpret_cast<uintptr_t>(t.numel() > 0 ? t.data_ptr() : nullptr);
      counts[(size_t)i] = t.numel();
      types[(size_t)i] = flag;
    }
    if (why != nullptr) return Py_BuildValue("(OOOOns)", Py_None, Py_None, Py_None, Py_None, i, why);
    return Py_BuildValue("(NNNins)", as_bytes(pointers), as_bytes(counts), as_bytes(types), device, n, "");
  });
  Py_DECREF(seq);
  return result;
}

// alike(a, b): the index of the first pair of tensors whose shapes differ, or whose strides
// do where one of the two is not contiguous; -1 when there is none.
PyObject *alike(PyObject *, PyObject *args) {
  PyObject *a = nullptr, *b = nullptr;
  if (!PyArg_ParseTuple(args, "O!O!", &PyList_Type, &a, &PyList_Type, &b)) return nullptr;
  return guarded([&]() -> PyObject * {
    const Py_ssize_t n = PyList_GET_SIZE(a) < PyList_GET_SIZE(b) ? PyList_GET_SIZE(a) : PyList_GET_SIZE(b);
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject *x = PyList_GET_ITEM(a, i), *y = PyList_GET_ITEM(b, i);
      if (!THPVariable_Check(x) || !THPVariable_Check(y)) return PyLong_FromSsize_t(i);
      const at::Tensor &s = THPVariable_Unpack(x), &t = THPVariable_Unpack(y);
      if (s.layout() != at::kStrided || t.layout() != at::kStrided || s.sizes() != t.sizes() ||
          (s.strides() != t.strides() && !(s.is_contiguous() && t.is_contiguous())))
        return PyLong_FromSsize_t(i);
    }
    return PyLong_FromLong(-1);
  });
}

// writable(list): the index of the first tensor that autograd follows (a parameter, or a
// gradient that is part of a graph), -1 when there is none.
PyObject *writable(PyObject *, PyObject *list) {
  PyObject *seq = PySequence_Fast(list, "expected a sequence of tensors");
  if (seq == nullptr) return nullptr;
  Py_ssize_t found = -1;
  for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(seq) && found < 0; ++i)
    if (THPVariable_Check(PySequence_Fast_GET_ITEM(seq, i)) && THPVariable_Unpack(PySequence_Fast_GET_ITEM(seq, i)).requires_grad()) found = i;
  Py_DECREF(seq);
  return PyLong_FromSsize_t(found);
}

// tangent(list): the index of the first tensor with a forward-mode tangent, -1 when there is none.
PyObject *tangent(PyObject *, PyObject *list) {
  PyObject *seq = PySequence_Fast(list, "expected a sequence of tensors");
  if (seq == nullptr) return nullptr;
  Py_ssize_t found = -1;
  for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(seq) && found < 0; ++i)
    if (THPVariable_Check(PySequence_Fast_GET_ITEM(seq, i)) && has_tangent(THPVariable_Unpack(PySequence_Fast_GET_ITEM(seq, i)))) found = i;
  Py_DECREF(seq);
  return PyLong_FromSsize_t(found);
}

// written(list): the tensors' version counters move on, as after any write that autograd
// has to know of (inference tensors have none).
PyObject *written(PyObject *, PyObject *list) {
  PyObject *seq = PySequence_Fast(list, "expected a sequence of tensors");
  if (seq == nullptr) return nullptr;
  PyObject *result = guarded([&]() -> PyObject * {
    for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(seq); ++i) {
      const at::Tensor &t = THPVariable_Unpack(PySequence_Fast_GET_ITEM(seq, i));
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
    Py_RETURN_NONE;
  });
  Py_DECREF(seq);
  return result;
}

// ---------------------------------------------------------------------------
// the library's functions, by address
// ---------------------------------------------------------------------------
decltype(&ot_b200_last_error) f_last_error;
decltype(&ot_b200_sample) f_sample;
decltype(&ot_b200_joiner_logits) f_logits;
decltype(&ot_b200_joiner_logits_workspace_bytes) f_logits_bytes;
decltype(&ot_b200_joiner_train_bytes) f_train_bytes;
decltype(&ot_b200_joiner_train_forward_sized) f_train_forward;
decltype(&ot_b200_joiner_train_backward_sized) f_train_backward;
decltype(&ot_b200_clip_workspace_bytes) f_clip_bytes;
decltype(&ot_b200_clip_gradients) f_clip;

// bind(addresses): in the order above.
PyObject *bind(PyObject *, PyObject *args) {
  unsigned long long p[9];
  if (!PyArg_ParseTuple(args, "KKKKKKKKK", p, p + 1, p + 2, p + 3, p + 4, p + 5, p + 6, p + 7, p + 8)) return nullptr;
  f_last_error = reinterpret_cast<decltype(f_last_error)>(p[0]);
  f_sample = reinterpret_cast<decltype(f_sample)>(p[1]);
  f_logits = reinterpret_cast<decltype(f_logits)>(p[2]);
  f_logits_bytes = reinterpret_cast<decltype(f_logits_bytes)>(p[3]);
  f_train_bytes = reinterpret_cast<decltype(f_train_bytes)>(p[4]);
  f_train_forward = reinterpret_cast<decltype(f_train_forward)>(p[5]);
  f_train_backward = reinterpret_cast<decltype(f_train_backward)>(p[6]);
  f_clip_bytes = reinterpret_cast<decltype(f_clip_bytes)>(p[7]);
  f_clip = reinterpret_cast<decltype(f_clip)>(p[8]);
  Py_RETURN_NONE;
}

// A failed library call, as the Python layer raises it.
struct LibraryError : std::runtime_error {
  using std::runtime_error::runtime_error;
};
void check(int rc) {
  if (rc != OT_B200_OK) throw LibraryError(f_last_error());
}

void *stream_of(const at::Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// float32, bfloat16, float16: the flag; -1 for the rest.
int float_flag(at::ScalarType t) { return t == at::kDouble ? -1 : type_flag(t); }

bool plain_matrix(const at::Tensor &t) {
  return t.layout() == at::kStrided && t.is_cuda() && t.dim() == 2 && t.numel() > 0 && t.is_contiguous() && float_flag(t.scalar_type()) >= 0;
}

bool plain_vector(const at::Tensor &t, at::ScalarType type, int64_t n, int device) {
  return t.layout() == at::kStrided && t.is_cuda() && t.get_device() == device && t.scalar_type() == type && t.dim() == 1 && t.size(0) == n && t.is_contiguous();
}

// What Fp8Weight checks.  Its tensors may have been resized or exchanged since (Tensor.resize_,
// Tensor.data), so every call looks again.
bool plain_weight(const at::Tensor &w, const at::Tensor &scale) {
  if (w.layout() != at::kStrided || !w.is_cuda() || w.scalar_type() != at::kFloat8_e4m3fn || w.dim() != 2 || w.numel() == 0) return false;
  const int64_t v = w.size(0), d = w.size(1);
  return (d == 1 || w.stride(1) == 1) && (v == 1 || (w.stride(0) % 16 == 0 && w.stride(0) >= d)) &&
         reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0 && scale.layout() == at::kStrided && scale.is_cuda() &&
         scale.get_device() == w.get_device() && scale.scalar_type() == at::kFloat && scale.dim() == 2 &&
         scale.size(0) == (v + 127) / 128 && scale.size(1) == (d + 127) / 128 && scale.is_contiguous();
}

at::Tensor bytes_on(const at::Tensor &like, uint64_t n) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte).requires_grad(false)); }

// weight(data, scale): whether they are a quantised weight that the kernels can read.
PyObject *weight(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    return PyBool_FromLong(n == 2 && THPVariable_Check(args[0]) && THPVariable_Check(args[1]) &&
                           plain_weight(THPVariable_Unpack(args[0]), THPVariable_Unpack(args[1])));
  });
}

// sample(logits, uniforms, temperature, top_k, top_p, min_p): (tokens, logprobs) or None.
PyObject *sample(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (n != 6 || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1])) Py_RETURN_NONE;
    const at::Tensor &x = THPVariable_Unpack(args[0]), &u = THPVariable_Unpack(args[1]);
    if (!plain_matrix(x) || x.size(1) > OT_B200_SAMPLE_MAX_V) Py_RETURN_NONE;
    const int64_t rows = x.size(0);
    const int device = x.get_device();
    if (!plain_vector(u, at::kFloat, rows, device)) Py_RETURN_NONE;
    const void *ptr[4];
    float value[4] = {0, 0, 0, 0};
    int k = 0;
    for (int i = 0; i < 4; ++i) {
      PyObject *a = args[2 + i];
      ptr[i] = nullptr;
      if (i == 1 && PyLong_CheckExact(a)) {
        int overflow = 0;
        const long long v = PyLong_AsLongLongAndOverflow(a, &overflow);
        if (overflow || v < INT32_MIN || v > INT32_MAX) Py_RETURN_NONE;
        k = (int)v;
      } else if (i != 1 && PyFloat_CheckExact(a)) {
        const double v = PyFloat_AS_DOUBLE(a);
        if (v != v || (i == 0 && !(v >= 0.0 && v <= 1e6))) Py_RETURN_NONE;
        value[i] = (float)v;
      } else if (THPVariable_Check(a)) {
        const at::Tensor &t = THPVariable_Unpack(a);
        if (!plain_vector(t, i == 1 ? at::kInt : at::kFloat, rows, device)) Py_RETURN_NONE;
        ptr[i] = t.data_ptr();
      } else {
        Py_RETURN_NONE;
      }
    }
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
    const auto options = x.options().requires_grad(false);
    at::Tensor tokens = at::empty({rows}, options.dtype(at::kInt)), logprobs = at::empty({rows}, options.dtype(at::kFloat));
    check(f_sample(x.data_ptr(), rows, (int32_t)x.size(1), x.size(1), (uint32_t)float_flag(x.scalar_type()), u.data_ptr<float>(),
                   static_cast<const float *>(ptr[0]), value[0], static_cast<const int32_t *>(ptr[1]), k,
                   static_cast<const float *>(ptr[2]), value[2], static_cast<const float *>(ptr[3]), value[3],
                   tokens.data_ptr<int32_t>(), logprobs.data_ptr<float>(), stream_of(x)));
    PyObject *a = THPVariable_Wrap(std::move(tokens)), *b = THPVariable_Wrap(std::move(logprobs));
    PyObject *pair = PyTuple_Pack(2, a, b);
    Py_DECREF(a);
    Py_DECREF(b);
    return pair;
  });
}

// The autograd node of joiner_logits: everything the backward pass needs of the operands is
// in one buffer, W^T and X^T in e4m3.
struct JoinerLogits : torch::autograd::Function<JoinerLogits> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &x, const at::Tensor &w,
                            const std::optional<at::Tensor> &bias, int64_t out_type, int64_t report) {
    const int64_t rows = x.size(0), d = x.size(1), v = w.size(0);
    const bool need_x = x.requires_grad(), need_w = w.requires_grad(), need_b = bias && bias->requires_grad();
    const c10::cuda::CUDAGuard guard(x.device());
    uint64_t size[3];
    check(f_train_bytes(rows, (int32_t)d, (int32_t)v, need_x, need_w, need_b, size, size + 1, size + 2));
    at::Tensor saved = bytes_on(x, size[0]), ws = bytes_on(x, size[1]);
    const auto type = (at::ScalarType)out_type;
    at::Tensor out = at::empty({rows, v}, x.options().dtype(type).requires_grad(false));
    check(f_train_forward(x.data_ptr(), rows, (int32_t)d, rows > 1 ? x.stride(0) : d, (uint32_t)float_flag(x.scalar_type()), w.data_ptr(),
                          (int32_t)v, v > 1 ? w.stride(0) : d, (uint32_t)float_flag(w.scalar_type()), bias ? bias->data_ptr<float>() : nullptr,
                          (uint32_t)(float_flag(type) | report), need_x, need_w, saved.data_ptr(), size[0], ws.data_ptr(), size[1],
                          out.data_ptr(), stream_of(x)));
    ctx->save_for_backward({saved});
    ctx->saved_data["meta"] = std::vector<int64_t>{rows, d, v, (int64_t)x.scalar_type(), (int64_t)w.scalar_type(), need_x, need_w, need_b,
                                                   (int64_t)size[2], report};
    return out;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "joiner_logits cannot be differentiated twice");
    const std::vector<int64_t> m = ctx->saved_data["meta"].toIntVector();
    const int64_t rows = m[0], d = m[1], v = m[2];
    at::Tensor none, saved = ctx->get_saved_variables()[0], g = grads[0];
    if (!g.defined()) return {none, none, none, none, none};
    if ((v > 1 && g.stride(1) != 1) || (rows > 1 && g.stride(0) < v)) g = g.contiguous();
    const c10::cuda::CUDAGuard guard(g.device());
    const auto options = g.options().requires_grad(false);
    at::Tensor gx, gw, gb, ws = bytes_on(g, (uint64_t)m[8]);
    const auto x_type = (at::ScalarType)m[3], w_type = (at::ScalarType)m[4];
    if (m[5]) gx = at::empty({rows, d}, options.dtype(x_type));
    if (m[6]) gw = at::empty({v, d}, options.dtype(w_type));
    if (m[7]) gb = at::empty({v}, options.dtype(at::kFloat));
    check(f_train_backward(g.data_ptr(), rows, (int32_t)v, rows > 1 ? g.stride(0) : v, (uint32_t)float_flag(g.scalar_type()), (int32_t)d,
                           saved.data_ptr(), (uint64_t)saved.numel(), gx.defined() ? gx.data_ptr() : nullptr, (uint32_t)float_flag(x_type),
                           gw.defined() ? gw.data_ptr() : nullptr, (uint32_t)float_flag(w_type), gb.defined() ? gb.data_ptr<float>() : nullptr,
                           (uint32_t)m[9], ws.data_ptr(), (uint64_t)m[8], stream_of(g)));
    return {gx, gw, gb, none, none};
  }
};

// train(joiner_in, weight, bias or None, out dtype, report flag): the logits; arguments checked by the caller.
PyObject *train(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != 5 || !THPDtype_Check(args[3])) {
    PyErr_SetString(PyExc_TypeError, "train: wrong arguments");
    return nullptr;
  }
  return guarded([&]() -> PyObject * {
    std::optional<at::Tensor> bias;
    if (args[2] != Py_None) bias = THPVariable_Unpack(args[2]);
    return THPVariable_Wrap(JoinerLogits::apply(THPVariable_Unpack(args[0]), THPVariable_Unpack(args[1]), bias,
                                                (int64_t)reinterpret_cast<THPDtype *>(args[3])->scalar_type, (int64_t)PyLong_AsLong(args[4])));
  });
}

// logits(joiner_in, weight bytes, weight scales, bias or None, out dtype, report flag): the
// logits of a quantised weight, or None.
PyObject *logits(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (n != 6 || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) || !THPVariable_Check(args[2]) || !THPDtype_Check(args[4]))
      Py_RETURN_NONE;
    const at::Tensor &x = THPVariable_Unpack(args[0]), &w = THPVariable_Unpack(args[1]), &scale = THPVariable_Unpack(args[2]);
    const at::ScalarType type = reinterpret_cast<THPDtype *>(args[4])->scalar_type;
    if (!plain_matrix(x) || float_flag(type) < 0 || !plain_weight(w, scale) || has_tangent(x) || has_tangent(scale) || w.get_device() != x.get_device() || w.size(1) != x.size(1)) Py_RETURN_NONE;
    const int64_t rows = x.size(0), d = x.size(1), v = w.size(0);
    const float *bias = nullptr;
    bool grads = x.requires_grad();
    if (args[3] != Py_None) {
      if (!THPVariable_Check(args[3])) Py_RETURN_NONE;
      const at::Tensor &b = THPVariable_Unpack(args[3]);
      if (!plain_vector(b, at::kFloat, v, x.get_device()) || has_tangent(b)) Py_RETURN_NONE;
      bias = b.data_ptr<float>();
      grads = grads || b.requires_grad();
    }
    if (grads && at::GradMode::is_enabled()) Py_RETURN_NONE;
    const c10::cuda::CUDAGuard guard(x.device());
    uint64_t size = 0;
    check(f_logits_bytes(rows, (int32_t)d, (int32_t)v, &size));
    at::Tensor out = at::empty({rows, v}, x.options().dtype(type).requires_grad(false)), ws = bytes_on(x, size);
    check(f_logits(x.data_ptr(), rows, (int32_t)d, d, (uint32_t)float_flag(x.scalar_type()), w.data_ptr(), v > 1 ? w.stride(0) : (d + 15) / 16 * 16,
                   scale.data_ptr<float>(), (int32_t)v, bias, (uint32_t)(float_flag(type) | PyLong_AsLong(args[5])), ws.data_ptr(), size,
                   out.data_ptr(), stream_of(x)));
    return THPVariable_Wrap(std::move(out));
  });
}

// clip(pointers, counts, types, outs or None, out types or None, first tensor, norm kind,
// apply, max_norm): the norm; the lists come from describe().
PyObject *clip(PyObject *, PyObject *args) {
  const char *p, *c, *t, *o = nullptr, *ot = nullptr;
  Py_ssize_t np, nc, nt, no, not_;
  PyObject *like;
  int kind, apply;
  double max_norm;
  if (!PyArg_ParseTuple(args, "y#y#y#z#z#Oiid", &p, &np, &c, &nc, &t, &nt, &o, &no, &ot, &not_, &like, &kind, &apply, &max_norm)) return nullptr;
  return guarded([&]() -> PyObject * {
    const at::Tensor &x = THPVariable_Unpack(like);
    const c10::cuda::CUDAGuard guard(x.device());
    const int32_t n = (int32_t)(nc / (Py_ssize_t)sizeof(int64_t));
    uint64_t size = 0;
    check(f_clip_bytes(n, &size));
    at::Tensor ws = bytes_on(x, size), norm = at::empty({}, x.options().dtype(at::kFloat).requires_grad(false));
    check(f_clip(n, reinterpret_cast<const void *const *>(p), reinterpret_cast<const int64_t *>(c), reinterpret_cast<const int32_t *>(t),
                 reinterpret_cast<void *const *>(o), reinterpret_cast<const int32_t *>(ot), kind, apply, max_norm, ws.data_ptr(), size,
                 norm.data_ptr<float>(), stream_of(x)));
    return THPVariable_Wrap(std::move(norm));
  });
}

PyMethodDef methods[] = {{"describe", describe, METH_O, "pointers, counts and types of a list of tensors"},
                         {"alike", alike, METH_VARARGS, "whether two lists of tensors have the same shapes"},
                         {"writable", writable, METH_O, "the first tensor that requires a gradient"},
                         {"tangent", tangent, METH_O, "the first tensor with a forward-mode tangent"},
                         {"written", written, METH_O, "moves the tensors' version counters on"},
                         {"bind", bind, METH_VARARGS, "takes the addresses of the library's functions"},
                         {"weight", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(weight)), METH_FASTCALL, "whether two tensors are a quantised weight"},
                         {"sample", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(sample)), METH_FASTCALL, "the usual call of sample_tokens"},
                         {"logits", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(logits)), METH_FASTCALL, "the usual call of joiner_logits with a quantised weight"},
                         {"train", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(train)), METH_FASTCALL, "joiner_logits with gradients"},
                         {"clip", clip, METH_VARARGS, "grad_norm and clip_grad_norm_ of described tensors"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// built_for: the torch and the Python whose interfaces this file was compiled against.
PyMODINIT_FUNC PyInit__tensors(void) {
  PyObject *m = PyModule_Create(&module);
  if (m != nullptr && PyModule_AddStringConstant(m, "built_for", OT_BUILT_FOR) != 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
