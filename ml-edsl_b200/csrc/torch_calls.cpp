// Python module b200torch: the serving operators' calls on torch CUDA tensors
// (mlir_edsl/serving.py). Checks the arguments, makes the outputs and calls
// the C entry points of libb200edsl.so on the current stream of the tensors'
// device. A call for one token takes a few microseconds on the GPU; checks and
// allocations in C++ keep the host's share of it near that (measured per call
// with three outputs: 26 us through ctypes and torch.empty).
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>
#include <cmath>
#include <initializer_list>
#include <string>
#include "../../include/b200_edsl.h"

namespace {

using at::ScalarType;
using at::Tensor;

PyObject* g_b200_error = nullptr;    // mlir_edsl._native.B200Error
PyObject* g_memory_error = nullptr;  // torch.OutOfMemoryError

// A refused call: a Python exception to raise.
struct Refusal {
  PyObject* type;
  std::string text;
};
[[noreturn]] void type_error(std::string s) { throw Refusal{PyExc_TypeError, std::move(s)}; }
[[noreturn]] void value_error(std::string s) { throw Refusal{PyExc_ValueError, std::move(s)}; }
struct PythonError {};  // an exception that is set already

std::string text_of(PyObject* o) {
  PyObject* s = PyObject_Repr(o);
  const char* u = s ? PyUnicode_AsUTF8(s) : nullptr;
  std::string r = u ? u : "?";
  Py_XDECREF(s);
  if (!u) PyErr_Clear();
  return r;
}
std::string text_of(at::IntArrayRef v) {
  std::string s = "(";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + (v.size() == 1 ? ",)" : ")");
}
std::string text_of(ScalarType t) {
  switch (t) {
    case ScalarType::Float: return "torch.float32";
    case ScalarType::BFloat16: return "torch.bfloat16";
    case ScalarType::Half: return "torch.float16";
    case ScalarType::Float8_e4m3fn: return "torch.float8_e4m3fn";
    case ScalarType::Byte: return "torch.uint8";
    case ScalarType::Int: return "torch.int32";
    case ScalarType::Long: return "torch.int64";
    case ScalarType::Double: return "torch.float64";
    default: return std::string("torch.") + c10::toString(t);
  }
}

int code_of(ScalarType t) {
  return t == ScalarType::Float      ? B200_F32
         : t == ScalarType::BFloat16 ? B200_BF16
         : t == ScalarType::Half     ? B200_F16
                                     : B200_E4M3;
}
using Types = std::initializer_list<ScalarType>;
#define PLAIN_TYPES {ScalarType::Float, ScalarType::BFloat16, ScalarType::Half}

void check_type(ScalarType t, const char* name, Types types) {
  for (ScalarType k : types)
    if (k == t) return;
  std::string s = std::string(name) + ": dtype " + text_of(t) + " is not one of ";
  bool first = true;
  for (ScalarType k : types) {
    s += (first ? "" : ", ") + text_of(k);
    first = false;
  }
  type_error(s);
}

// `o` as an input: a CUDA tensor of one of `types`, on `device`.
const Tensor& tensor(PyObject* o, const char* name, Types types,
                     const c10::Device* device = nullptr) {
  if (!THPVariable_Check(o))
    type_error(std::string(name) + ": expected a torch tensor, got " + Py_TYPE(o)->tp_name);
  const Tensor& t = THPVariable_Unpack(o);
  check_type(t.scalar_type(), name, types);
  if (!t.is_cuda() || t.layout() != c10::kStrided)
    value_error(std::string(name) + ": expected a CUDA tensor, got one on " + t.device().str());
  if (t.is_neg())
    value_error(std::string(name) +
                ": stands for the negative of its memory (use torch.resolve_neg)");
  if (device && t.device() != *device)
    value_error(std::string(name) + ": on " + t.device().str() + ", but the call runs on " +
                device->str());
  if (t.requires_grad() && at::GradMode::is_enabled())
    value_error(std::string(name) +
                ": requires a gradient, and this operator has no backward pass (use "
                "torch.no_grad())");
  // the tangent is part of what a tensor without autograd data does not have
  if (t.unsafeGetTensorImpl()->autograd_meta() && t._fw_grad(0).defined() &&
      c10::AutogradState::get_tls_state().get_fw_grad_mode())
    value_error(std::string(name) +
                ": has a tangent, and this operator has no forward gradient (use "
                "torch.autograd.forward_ad.unpack_dual)");
  return t;
}

struct Rows {
  int64_t m, n, ld;
};

// A tensor as rows of its last dimension.
Rows rows(const Tensor& t, const char* name) {
  const auto shape = t.sizes(), stride = t.strides();
  const int64_t dims = t.dim();
  if (dims == 0) value_error(std::string(name) + ": expected at least one dimension");
  const int64_t n = shape[dims - 1], step = stride[dims - 1];
  int64_t m = 1, ld = n;
  bool first = true;
  int64_t last = 0;  // the pitch of the dimension inside
  for (int64_t d = dims - 2; d >= 0; --d) {
    if (shape[d] == 1) continue;
    if (first) ld = stride[d];
    else if (m && stride[d] != last)
      value_error(std::string(name) + ": the leading dimensions of shape " + text_of(shape) +
                  " with strides " + text_of(stride) + " cannot be viewed as one");
    first = false;
    m *= shape[d];
    last = stride[d] * shape[d];
  }
  if (m <= 1) ld = n;
  if (m && n && ((n > 1 && step != 1) || ld < n))
    value_error(std::string(name) + ": needs contiguous rows that do not overlap, got shape " +
                text_of(shape) + " with strides " + text_of(stride));
  return {m, n, std::max(ld, n)};
}

// The bytes of a tensor's rows: `rows` of them, `n` bytes each, `ld` apart.
struct Memory {
  const char* at;
  int64_t m, n, ld;
  const char* end() const { return at + (m - 1) * ld + n; }
};
Memory memory(const Tensor& t, const Rows& r) {
  const int64_t size = (int64_t)t.element_size();
  return {static_cast<const char*>(t.const_data_ptr()), r.n ? r.m : 0, r.n * size, r.ld * size};
}
Memory memory(const Tensor& t, const char* name) { return memory(t, rows(t, name)); }

bool same(const Memory& a, const Memory& b) {
  return a.at == b.at && a.m == b.m && a.n == b.n && (a.m == 1 || a.ld == b.ld);
}

// Whether two sets of rows share a byte. Rows of one pitch may lie side by side
// in one buffer; of other pitches, both are gone through in the order of their
// addresses.
bool overlap(const Memory& a, const Memory& b) {
  if (a.m == 0 || b.m == 0 || a.end() <= b.at || b.end() <= a.at) return false;
  if (a.ld == b.ld) {
    // a row of b starts d bytes behind one of a, and ld - d before the next (the
    // ends overlap, so at least one of the two is there)
    const int64_t d = ((b.at - a.at) % a.ld + a.ld) % a.ld;
    return d < a.n || a.ld - d < b.n;
  }
  for (int64_t i = 0, j = 0; i < a.m && j < b.m;) {
    const char *p = a.at + i * a.ld, *q = b.at + j * b.ld;
    if (p < q + b.n && q < p + a.n) return true;
    if (p < q) ++i;
    else ++j;
  }
  return false;
}

// Refuses an output that shares memory with `b`, unless it may take its place.
void check_apart(const Memory& out, const char* name, const Memory& b, const char* other,
                 bool in_place = false) {
  if (overlap(out, b) && !(in_place && same(out, b)))
    value_error(std::string(name) + ": overlaps " + other);
}

const void* vector(PyObject* o, int64_t n, const char* name, Types types,
                   const c10::Device& device, int* code) {
  const Tensor& t = tensor(o, name, types, &device);
  if (t.dim() != 1 || t.size(0) != n)
    value_error(std::string(name) + ": expected shape (" + std::to_string(n) + ",), got " +
                text_of(t.sizes()));
  if (n > 1 && t.stride(0) != 1) value_error(std::string(name) + ": needs contiguous elements");
  *code = code_of(t.scalar_type());
  return t.const_data_ptr();
}

Tensor empty(at::IntArrayRef shape, ScalarType type, const c10::Device& device) {
  return at::detail::empty_cuda(shape, type, device, std::nullopt);
}

// `o` as an output of this shape, or a new tensor where it is None.
Tensor output(PyObject* o, at::IntArrayRef shape, ScalarType type, const c10::Device& device,
              const char* name) {
  if (o == Py_None) return empty(shape, type, device);
  const Tensor& t = tensor(o, name, {type}, &device);
  if (t.sizes() != shape)
    value_error(std::string(name) + ": expected shape " + text_of(shape) + ", got " +
                text_of(t.sizes()));
  return t;
}

// A given output has new contents: backward passes that kept it have to notice.
void changed(PyObject* o, const Tensor& t) {
  if (o != Py_None && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

at::DimVector lead(const Tensor& t) {
  return at::DimVector(t.sizes().begin(), t.sizes().end() - 1);
}
at::DimVector lead_and(const Tensor& t, int64_t n) {
  at::DimVector s = lead(t);
  s.push_back(n);
  return s;
}

int64_t whole(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PythonError{};
  return v;
}
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PythonError{};
  return v;
}
int64_t one_of(PyObject* o, const char* name, const char* said, std::initializer_list<int64_t> of) {
  const int64_t v = whole(o);
  for (int64_t k : of)
    if (k == v) return v;
  value_error(std::string(name) + ": expected " + said + ", got " + std::to_string(v));
}

// Runs a C entry point on the current stream of `device`.
template <class Fn>
void call(const c10::Device& device, Fn fn) {
  c10::cuda::CUDAGuard guard(device);
  void* stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS;
  rc = fn(stream);
  Py_END_ALLOW_THREADS;
  if (rc) {
    PyObject* v = Py_BuildValue("(is)", rc, b200_last_error());
    if (v) PyErr_SetObject(g_b200_error ? g_b200_error : PyExc_RuntimeError, v);
    Py_XDECREF(v);
    throw PythonError{};
  }
}

PyObject* none() {
  Py_INCREF(Py_None);
  return Py_None;
}
PyObject* wrap(const Tensor& t) { return t.defined() ? THPVariable_Wrap(t) : none(); }
PyObject* wrap_all(std::initializer_list<Tensor> list) {
  PyObject* r = PyTuple_New((Py_ssize_t)list.size());
  if (!r) throw PythonError{};
  Py_ssize_t i = 0;
  for (const Tensor& t : list) {
    PyObject* o = wrap(t);
    if (!o) {
      Py_DECREF(r);
      throw PythonError{};
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

// ---------------------------------------------------------------- operators

// x, weight, residual, eps, quant, group, out, residual_out
PyObject* rms_norm(PyObject* const* a) {
  const Tensor& x = tensor(a[0], "x", PLAIN_TYPES);
  const c10::Device device = x.device();
  const ScalarType type = x.scalar_type();
  const int code = code_of(type);
  const Rows rx = rows(x, "x");
  const bool quant = a[4] != Py_None;
  if (quant && !(PyUnicode_Check(a[4]) && PyUnicode_CompareWithASCIIString(a[4], "e4m3") == 0))
    value_error("quant: expected None or 'e4m3', got " + text_of(a[4]));
  const int64_t group = one_of(a[5], "group", "0 (a row), 32, 64 or 128", {0, 32, 64, 128});
  if (group && !quant) value_error("group: only quantised outputs have groups");
  const float eps = (float)real(a[3]);
  if (!(eps > 0.0f) || std::isinf(eps))
    value_error("eps: must be positive and finite, got " + text_of(a[3]));
  const void* w = nullptr;
  int w_code = 0;
  if (a[1] != Py_None)
    w = vector(a[1], rx.n, "weight", {type, ScalarType::Float}, device, &w_code);
  const void* r = nullptr;
  Tensor h;
  int64_t ldr = 0, ldh = 0;
  auto apart = [&](const Memory& out, const char* name, bool in_place) {
    check_apart(out, name, memory(x, rx), "x", in_place);
    if (r) check_apart(out, name, memory(THPVariable_Unpack(a[2]), "residual"), "residual", in_place);
    if (w) check_apart(out, name, memory(THPVariable_Unpack(a[1]), "weight"), "weight");
  };
  if (a[2] != Py_None) {
    const Tensor& res = tensor(a[2], "residual", {type}, &device);
    if (res.sizes() != x.sizes())
      value_error("residual: expected shape " + text_of(x.sizes()) + ", got " +
                  text_of(res.sizes()));
    ldr = rows(res, "residual").ld;
    r = res.const_data_ptr();
    h = output(a[7], x.sizes(), type, device, "residual_out");
    ldh = rows(h, "residual_out").ld;
    if (a[7] != Py_None) apart(memory(h, "residual_out"), "residual_out", true);
  } else if (a[7] != Py_None) {
    value_error("residual_out: given without a residual");
  }
  Tensor y = output(a[6], x.sizes(), quant ? ScalarType::Float8_e4m3fn : type, device, "out");
  const int64_t ldy = rows(y, "out").ld;
  if (a[6] != Py_None) {
    const Memory my = memory(y, "out");
    apart(my, "out", !quant);
    if (h.defined()) check_apart(my, "out", memory(h, "residual_out"), "residual_out");
  }
  Tensor s;
  int64_t lds = 0;
  if (quant) {
    lds = group ? (rx.n + group - 1) / group : 1;
    s = empty(lead_and(x, lds), ScalarType::Float, device);
  }
  call(device, [&](void* stream) {
    return b200_rms_norm(x.const_data_ptr(), rx.ld, r, ldr, code, w, w_code, eps,
                         h.defined() ? h.data_ptr() : nullptr, ldh, y.data_ptr(), ldy,
                         quant ? B200_E4M3 : code,
                         quant ? static_cast<float*>(s.data_ptr()) : nullptr, lds, (int)group,
                         rx.m, rx.n, stream);
  });
  changed(a[6], y);
  changed(a[7], h);
  if (quant) return h.defined() ? wrap_all({y, s, h}) : wrap_all({y, s});
  return h.defined() ? wrap_all({y, h}) : wrap(y);
}

int64_t w4_group(PyObject* o) {
  const int64_t g = whole(o);
  if (g != 32 && (g <= 0 || g % 64 != 0 || g > INT32_MAX))
    value_error("group: expected 32 or a multiple of 64, got " + std::to_string(g));
  return g;
}

const Tensor& matrix(PyObject* o, const char* name, Types types, Rows* r) {
  const Tensor& t = tensor(o, name, types);
  if (t.dim() != 2)
    value_error(std::string(name) + ": expected two dimensions, got shape " + text_of(t.sizes()));
  *r = rows(t, name);
  return t;
}

// codes, scales, zeros, group -> the packed buffer
PyObject* pack_w4(PyObject* const* a) {
  const int64_t group = w4_group(a[3]);
  Rows c;
  const Tensor& codes = matrix(a[0], "codes", {ScalarType::Byte}, &c);
  const c10::Device device = codes.device();
  const int64_t K = codes.size(0), N = codes.size(1);
  const int64_t shape[2] = {(K + group - 1) / group, N};
  const Tensor& scales = tensor(a[1], "scales", PLAIN_TYPES, &device);
  const Tensor* zeros =
      a[2] == Py_None ? nullptr : &tensor(a[2], "zeros", {ScalarType::Byte}, &device);
  for (const Tensor* t : {&scales, zeros})
    if (t && t->sizes() != at::IntArrayRef(shape, 2))
      value_error(std::string(t == zeros ? "zeros" : "scales") + ": expected shape " +
                  text_of(at::IntArrayRef(shape, 2)) + ", got " + text_of(t->sizes()));
  const int64_t lds = rows(scales, "scales").ld, ldz = zeros ? rows(*zeros, "zeros").ld : 0;
  const int code = code_of(scales.scalar_type());
  const int64_t bytes = b200_w4_bytes(K, N, (int)group, code, zeros != nullptr);
  if (bytes < 0) value_error(std::string("codes: ") + b200_last_error());
  Tensor packed = empty({bytes}, ScalarType::Byte, device);
  call(device, [&](void* stream) {
    return b200_w4_pack(static_cast<const uint8_t*>(codes.const_data_ptr()), c.ld,
                        scales.const_data_ptr(), lds, code,
                        zeros ? static_cast<const uint8_t*>(zeros->const_data_ptr()) : nullptr, ldz,
                        K, N, (int)group, packed.data_ptr(), stream);
  });
  return wrap(packed);
}

ScalarType plain_type(PyObject* o, const char* name) {
  if (!THPDtype_Check(o))
    type_error(std::string(name) + ": expected a torch dtype, got " + Py_TYPE(o)->tp_name);
  const ScalarType t = reinterpret_cast<THPDtype*>(o)->scalar_type;
  check_type(t, name, PLAIN_TYPES);
  return t;
}

// W, group, scale_dtype -> codes, scales
PyObject* quantize_w4(PyObject* const* a) {
  const int64_t group = w4_group(a[1]);
  Rows r;
  const Tensor& W = matrix(a[0], "W", {ScalarType::Float}, &r);
  const ScalarType type = plain_type(a[2], "scale_dtype");
  const c10::Device device = W.device();
  const int64_t K = W.size(0), N = W.size(1);
  Tensor codes = empty({K, N}, ScalarType::Byte, device);
  Tensor scales = empty({(K + group - 1) / group, N}, type, device);
  call(device, [&](void* stream) {
    return b200_w4_quantize(static_cast<const float*>(W.const_data_ptr()), r.ld, K, N, (int)group,
                            static_cast<uint8_t*>(codes.data_ptr()), N, scales.data_ptr(), N,
                            code_of(type), stream);
  });
  return wrap_all({codes, scales});
}

// Packed weights: (buffer, K, N, group, type of scales, whether they have zeros).
struct Packed {
  const Tensor* buffer;
  int64_t K, N;
  int group, s_code, has_zeros;
};
Packed packed(PyObject* o) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 6) type_error("w: expected W4Weights");
  Packed p;
  p.buffer = &tensor(PyTuple_GET_ITEM(o, 0), "w", {ScalarType::Byte});
  p.K = whole(PyTuple_GET_ITEM(o, 1));
  p.N = whole(PyTuple_GET_ITEM(o, 2));
  p.group = (int)whole(PyTuple_GET_ITEM(o, 3));
  p.s_code = code_of(plain_type(PyTuple_GET_ITEM(o, 4), "w"));
  p.has_zeros = PyObject_IsTrue(PyTuple_GET_ITEM(o, 5));
  if (p.buffer->dim() != 1 || !p.buffer->is_contiguous() ||
      p.buffer->size(0) != b200_w4_bytes(p.K, p.N, p.group, p.s_code, p.has_zeros))
    value_error("w: the buffer is not that of its sizes");
  return p;
}

PyObject* dequantize_w4(PyObject* const* a) {
  const Packed w = packed(a[0]);
  const c10::Device device = w.buffer->device();
  Tensor out = empty({w.K, w.N}, ScalarType::Float, device);
  call(device, [&](void* stream) {
    return b200_w4_dequantize(w.buffer->const_data_ptr(), w.s_code, w.has_zeros, w.K, w.N, w.group,
                              static_cast<float*>(out.data_ptr()), w.N, stream);
  });
  return wrap(out);
}

// x, packed, bias, act, alpha, x_scales, x_group, out_dtype, out
PyObject* dense_w4(PyObject* const* a) {
  const Packed w = packed(a[1]);
  const Tensor& x = tensor(a[0], "x", {ScalarType::Float, ScalarType::BFloat16, ScalarType::Half,
                                       ScalarType::Float8_e4m3fn});
  const c10::Device device = x.device();
  if (w.buffer->device() != device)
    value_error("w: on " + w.buffer->device().str() + ", but the call runs on " + device.str());
  const Rows r = rows(x, "x");
  if (r.n != w.K)
    value_error("x: expected " + std::to_string(w.K) + " columns, got " + std::to_string(r.n));
  const int act = (int)one_of(a[3], "act", "0 (none), 1 (relu) or 2 (leaky relu)", {0, 1, 2});
  const float alpha = (float)real(a[4]);
  const bool e4m3 = x.scalar_type() == ScalarType::Float8_e4m3fn;
  ScalarType type = e4m3 ? ScalarType::BFloat16 : x.scalar_type();
  if (a[7] != Py_None) type = plain_type(a[7], "out_dtype");
  else if (a[8] != Py_None)
    type = tensor(a[8], "out", PLAIN_TYPES, &device).scalar_type();
  const int64_t x_group = one_of(a[6], "x_group", "0 (a row), 32, 64 or 128", {0, 32, 64, 128});
  const float* xs = nullptr;
  int64_t lds = 0;
  if (a[5] != Py_None) {
    if (!e4m3) type_error("x_scales: only an e4m3 x has scales");
    const Tensor& s = tensor(a[5], "x_scales", {ScalarType::Float}, &device);
    const at::DimVector shape = lead_and(x, x_group ? (w.K + x_group - 1) / x_group : 1);
    if (s.sizes() != at::IntArrayRef(shape))
      value_error("x_scales: expected shape " + text_of(shape) + ", got " + text_of(s.sizes()));
    lds = rows(s, "x_scales").ld;
    xs = static_cast<const float*>(s.const_data_ptr());
  } else if (x_group) {
    value_error("x_group: given without x_scales");
  }
  const void* b = nullptr;
  int b_code = 0;
  if (a[2] != Py_None) b = vector(a[2], w.N, "bias", PLAIN_TYPES, device, &b_code);
  Tensor y = output(a[8], lead_and(x, w.N), type, device, "out");
  const int64_t ldy = rows(y, "out").ld;
  if (a[8] != Py_None) {
    const Memory my = memory(y, "out");
    check_apart(my, "out", memory(x, r), "x");
    check_apart(my, "out", memory(*w.buffer, "w"), "w");
    if (b) check_apart(my, "out", memory(THPVariable_Unpack(a[2]), "bias"), "bias");
    if (xs) check_apart(my, "out", memory(THPVariable_Unpack(a[5]), "x_scales"), "x_scales");
  }
  call(device, [&](void* stream) {
    return b200_dense_w4(x.const_data_ptr(), r.ld, code_of(x.scalar_type()), xs, lds, (int)x_group,
                         w.buffer->const_data_ptr(), w.s_code, w.has_zeros, w.group, b, b_code,
                         y.data_ptr(), ldy, code_of(type), r.m, w.N, w.K, act, alpha, stream);
  });
  changed(a[8], y);
  return wrap(y);
}

// logits, tokens, top -> logprobs, entropy, top_logprobs, top_tokens
PyObject* token_logprobs(PyObject* const* a) {
  const Tensor& x = tensor(a[0], "logits", PLAIN_TYPES);
  const c10::Device device = x.device();
  const Rows r = rows(x, "logits");
  const int64_t top = whole(a[2]);
  if (top < 0 || top > 32) value_error("top: expected 0 to 32, got " + std::to_string(top));
  if (top > r.n || (r.n == 0 && r.m))
    value_error("top: " + std::to_string(top) + " of " + std::to_string(r.n) + " logits");
  const at::DimVector shape = lead(x);
  Tensor lp, top_lp, top_tok;
  const int32_t* tokens = nullptr;
  if (a[1] != Py_None) {
    const Tensor& t = tensor(a[1], "tokens", {ScalarType::Int}, &device);
    if (t.sizes() != at::IntArrayRef(shape))
      value_error("tokens: expected shape " + text_of(shape) + ", got " + text_of(t.sizes()));
    if (!t.is_contiguous()) value_error("tokens: needs contiguous elements");
    tokens = static_cast<const int32_t*>(t.const_data_ptr());
    lp = empty(shape, ScalarType::Float, device);
  }
  Tensor entropy = empty(shape, ScalarType::Float, device);
  if (top) {
    const at::DimVector with_top = lead_and(x, top);
    top_lp = empty(with_top, ScalarType::Float, device);
    top_tok = empty(with_top, ScalarType::Int, device);
  }
  auto f32 = [](const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; };
  call(device, [&](void* stream) {
    return b200_token_logprobs(x.const_data_ptr(), r.ld, code_of(x.scalar_type()), r.m, r.n, tokens,
                               f32(lp), f32(entropy), (int)top, f32(top_lp),
                               top ? static_cast<int32_t*>(top_tok.data_ptr()) : nullptr, stream);
  });
  return wrap_all({lp, entropy, top_lp, top_tok});
}

// tensor -> (rows, columns, pitch), of a tensor on any device
PyObject* rows_of(PyObject* const* a) {
  if (!THPVariable_Check(a[0])) type_error("expected a torch tensor");
  const Rows r = rows(THPVariable_Unpack(a[0]), "tensor");
  return Py_BuildValue("(LLL)", (long long)r.m, (long long)r.n, (long long)r.ld);
}

// two tensors on any device -> whether they share memory
PyObject* overlap_of(PyObject* const* a) {
  for (int i = 0; i < 2; ++i)
    if (!THPVariable_Check(a[i])) type_error("expected a torch tensor");
  return PyBool_FromLong(overlap(memory(THPVariable_Unpack(a[0]), "tensor"),
                                 memory(THPVariable_Unpack(a[1]), "tensor")));
}

// the exceptions of failed calls and of allocations
PyObject* set_errors(PyObject* const* a) {
  Py_INCREF(a[0]);
  Py_INCREF(a[1]);
  g_b200_error = a[0];
  g_memory_error = a[1];
  return none();
}

// No C++ exception leaves the module: each becomes a Python one.
template <PyObject* (*Fn)(PyObject* const*), Py_ssize_t Args>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != Args) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", Args, n);
    return nullptr;
  }
  try {
    return Fn(args);
  } catch (const PythonError&) {
  } catch (const Refusal& r) {
    PyErr_SetString(r.type, r.text.c_str());
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(g_memory_error ? g_memory_error : PyExc_RuntimeError,
                    e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

template <PyObject* (*Fn)(PyObject* const*), Py_ssize_t Args>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<Fn, Args>)),
          METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {
    method<rms_norm, 8>("rms_norm"),           method<pack_w4, 4>("pack_w4"),
    method<quantize_w4, 3>("quantize_w4"),     method<dequantize_w4, 1>("dequantize_w4"),
    method<dense_w4, 9>("dense_w4"),           method<token_logprobs, 3>("token_logprobs"),
    method<rows_of, 1>("rows_of"),             method<overlap_of, 2>("overlap_of"),
    method<set_errors, 2>("set_errors"),
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "b200torch", nullptr, -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_b200torch(void) { return PyModule_Create(&g_module); }
