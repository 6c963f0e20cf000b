// The host path of the feed-forward operators as a Python extension: for calls
// of a handful of microseconds on the GPU the interpreter's checks, allocations
// and foreign-function calls take longer than the kernels.
//
// Every function here serves the calls that pass all checks and answers None to
// anything else - another dtype, a wrong shape, an unusual argument - whereupon
// the Python front end (api.py, experts.py) runs its own checks, raises what
// there is to raise or makes the call itself.  So what is refused, and how, is
// written down once, in Python.  The launches go through the same C entry
// points; their addresses are handed over by bind().
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <cstring>
#include <optional>
#include <unordered_map>

#include "../../include/opengemm_b200.h"

namespace {

using at::ScalarType;
using at::Tensor;

struct Api {
  decltype(&og_b200_route) route = nullptr;
  decltype(&og_b200_route_gradient) route_gradient = nullptr;
  decltype(&og_b200_expert_plan) expert_plan = nullptr;
  decltype(&og_b200_expert_gather) expert_gather = nullptr;
  decltype(&og_b200_expert_product) expert_product = nullptr;
  decltype(&og_b200_expert_combine) expert_combine = nullptr;
  decltype(&og_b200_expert_combine_gradient) expert_combine_gradient = nullptr;
  decltype(&og_b200_activation_gradient) activation_gradient = nullptr;
  decltype(&og_b200_gemm_gradients) gemm_gradients = nullptr;
  decltype(&og_b200_gemm_gradients_workspace) gemm_gradients_workspace = nullptr;
  decltype(&og_b200_launch_fused) launch_fused = nullptr;
  decltype(&og_b200_routing_error) routing_error = nullptr;
  decltype(&og_b200_experts_error) experts_error = nullptr;
  decltype(&og_mm_error) error = nullptr;
} api;

// A launch that failed, as the Python front end would raise it.
PyObject* failed(const char* text) {
  PyErr_SetString(PyExc_RuntimeError, text);
  return nullptr;
}

// The tensor behind `o`, or null unless it is a plain CUDA tensor without gaps
// (no subclass, which may hold no memory at all).
const Tensor* cuda_tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.is_contiguous() && !t.is_neg() ? &t : nullptr;
}
bool is(const Tensor* t, ScalarType type, int device, std::initializer_list<int64_t> shape) {
  return t && t->scalar_type() == type && t->get_device() == device && t->sizes().equals(at::IntArrayRef(shape));
}
// An optional tensor argument: null for None; `ok` falls when it does not fit.
const Tensor* optional_tensor(PyObject* o, ScalarType type, int device, std::initializer_list<int64_t> shape, bool& ok) {
  if (o == Py_None) return nullptr;
  const Tensor* t = cuda_tensor(o);
  if (!is(t, type, device, shape)) ok = false;
  return t;
}
const void* data(const Tensor* t) { return t ? t->data_ptr() : nullptr; }
bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
bool overlap(const Tensor& s, const void* t, size_t bytes) {
  const char *a = static_cast<const char*>(s.data_ptr()), *b = static_cast<const char*>(t);
  return a < b + bytes && b < a + s.nbytes();
}
bool overlap(const Tensor& s, const Tensor& t) { return overlap(s, t.data_ptr(), t.nbytes()); }
Tensor empty(at::IntArrayRef shape, ScalarType type, int device) {
  return at::detail::empty_cuda(shape, type, c10::Device(c10::kCUDA, c10::DeviceIndex(device)), std::nullopt);
}
void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(device)).stream(); }

// A Python integer (or truth value) that fits `T`.
template <typename T>
bool integer(PyObject* o, T& v) {
  if (!PyLong_Check(o)) return false;
  int overflow = 0;
  const long long x = PyLong_AsLongLongAndOverflow(o, &overflow);
  if (overflow || x != (long long)(T)x) return false;
  v = T(x);
  return true;
}
bool number(PyObject* o, float& v) {
  if (PyFloat_CheckExact(o)) {
    v = float(PyFloat_AS_DOUBLE(o));
    return true;
  }
  if (!PyLong_CheckExact(o)) return false;
  const double x = PyLong_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) {  // past the floating range: the Python front end says so
    PyErr_Clear();
    return false;
  }
  v = float(x);
  return true;
}

int logits_type(ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1; }
const char* product_name(ScalarType t) {
  return t == at::kBFloat16 ? "bf16" : t == at::kHalf ? "f16" : t == at::kFloat8_e4m3fn ? "e4m3" : nullptr;
}

// Several tensors, None for those that are not there.
PyObject* tuple(std::initializer_list<Tensor> tensors) {
  PyObject* t = PyTuple_New(Py_ssize_t(tensors.size()));
  if (!t) return nullptr;
  Py_ssize_t i = 0;
  for (const Tensor& v : tensors) {
    PyObject* o = v.defined() ? THPVariable_Wrap(v) : Py_NewRef(Py_None);
    if (!o) {
      Py_DECREF(t);
      return nullptr;
    }
    PyTuple_SET_ITEM(t, i++, o);
  }
  return t;
}

#define NOT_SERVED Py_RETURN_NONE

// ------------------------------------------------------------------ routing

// route(logits, top_k, sigmoid, bias, groups, top_groups, group_top, renormalise, scale)
PyObject* route(PyObject*, PyObject* const* a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  OgRoute r{};
  const Tensor* logits = count == 9 ? cuda_tensor(a[0]) : nullptr;
  if (!logits || logits->dim() != 2 || (r.dtype = logits_type(logits->scalar_type())) < 0) NOT_SERVED;
  if (!integer(a[1], r.top_k) || !integer(a[2], r.sigmoid) || !integer(a[4], r.groups) || !integer(a[5], r.top_groups) || !integer(a[6], r.group_top) ||
      !integer(a[7], r.renormalise) || !number(a[8], r.scale) || r.top_k < 1 || r.top_k > 32)
    NOT_SERVED;
  const int device = logits->get_device();
  r.tokens = logits->size(0);
  if (logits->size(1) > 1024) NOT_SERVED;
  r.experts = int(logits->size(1));
  bool ok = true;
  const Tensor* bias = optional_tensor(a[3], at::kFloat, device, {r.experts}, ok);
  if (!ok) NOT_SERVED;
  Tensor weights = empty({r.tokens, r.top_k}, at::kFloat, device), indices = empty({r.tokens, r.top_k}, at::kInt, device);
  if (api.route(&r, logits->data_ptr(), static_cast<const float*>(data(bias)), weights.data_ptr<float>(), indices.data_ptr<int>(), device, stream_of(device)))
    return failed(api.routing_error());
  return tuple({weights, indices});
  END_HANDLE_TH_ERRORS
}

// route_backward(grad_weights, logits, indices, sigmoid, renormalise, scale)
PyObject* route_backward(PyObject*, PyObject* const* a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  OgRoute r{};
  const Tensor* logits = count == 6 ? cuda_tensor(a[1]) : nullptr;
  if (!logits || logits->dim() != 2 || (r.dtype = logits_type(logits->scalar_type())) < 0 || logits->size(1) > 1024) NOT_SERVED;
  const int device = logits->get_device();
  const Tensor *grad = cuda_tensor(a[0]), *indices = cuda_tensor(a[2]);
  if (!indices || indices->dim() != 2 || indices->size(1) > 32) NOT_SERVED;
  r.tokens = logits->size(0), r.experts = int(logits->size(1)), r.top_k = int(indices->size(1));
  r.groups = r.top_groups = r.group_top = 1;
  if (!is(indices, at::kInt, device, {r.tokens, r.top_k}) || !is(grad, at::kFloat, device, {r.tokens, r.top_k}) || !integer(a[3], r.sigmoid) ||
      !integer(a[4], r.renormalise) || !number(a[5], r.scale))
    NOT_SERVED;
  Tensor out = empty({r.tokens, r.experts}, logits->scalar_type(), device);
  if (api.route_gradient(&r, grad->data_ptr<float>(), logits->data_ptr(), indices->data_ptr<int>(), out.data_ptr(), device, stream_of(device)))
    return failed(api.routing_error());
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// expert_plan(indices, experts, chunk) -> (buffer of offsets, tokens and positions, its address, tokens, choices of each)
PyObject* expert_plan(PyObject*, PyObject* const* a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  const Tensor* indices = count == 3 ? cuda_tensor(a[0]) : nullptr;
  int experts = 0;
  int64_t chunk = 0;
  if (!indices || indices->dim() != 2 || indices->scalar_type() != at::kInt || indices->size(1) < 1 || !integer(a[1], experts) || experts < 1 || experts > 1024 ||
      !integer(a[2], chunk) || chunk < 1)
    NOT_SERVED;
  const int device = indices->get_device();
  const int64_t tokens = indices->size(0), top_k = indices->size(1), rows = tokens * top_k;
  if (rows > (int64_t(1) << 30)) NOT_SERVED;
  Tensor store = empty({experts + 1 + 2 * rows}, at::kInt, device), workspace;
  if (rows > chunk) workspace = empty({(rows + chunk - 1) / chunk * experts}, at::kInt, device);
  int* const base = store.data_ptr<int>();
  if (api.expert_plan(indices->data_ptr<int>(), tokens, int(top_k), experts, base, base + experts + 1, base + experts + 1 + rows,
                      workspace.defined() ? workspace.data_ptr<int>() : nullptr, device, stream_of(device)))
    return failed(api.routing_error());
  return Py_BuildValue("(NKLL)", THPVariable_Wrap(std::move(store)), (unsigned long long)reinterpret_cast<uintptr_t>(base), (long long)tokens, (long long)top_k);
  END_HANDLE_TH_ERRORS
}

// What a plan hands to the calls below: experts, tokens, choices of each, device index, address of its buffer.
struct Plan {
  int experts, top_k, device;
  int64_t tokens, rows;
  const int *offsets, *limit, *token_of_row, *positions;
};
bool plan_of(PyObject* o, Plan& p) {
  unsigned long long base = 0;
  if (!PyTuple_CheckExact(o) || PyTuple_GET_SIZE(o) != 5) return false;
  if (!integer(PyTuple_GET_ITEM(o, 0), p.experts) || !integer(PyTuple_GET_ITEM(o, 1), p.tokens) || !integer(PyTuple_GET_ITEM(o, 2), p.top_k) ||
      !integer(PyTuple_GET_ITEM(o, 3), p.device))
    return false;
  base = PyLong_AsUnsignedLongLong(PyTuple_GET_ITEM(o, 4));
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  p.rows = p.tokens * p.top_k;
  p.offsets = reinterpret_cast<const int*>(uintptr_t(base));
  p.limit = p.offsets + p.experts;
  p.token_of_row = p.limit + 1;
  p.positions = p.token_of_row + p.rows;
  return p.rows <= 0x7FFFFFFF;
}
size_t plan_bytes(const Plan& p) { return (size_t(p.experts) + 1 + 2 * size_t(p.rows)) * sizeof(int); }

// The tokens' rows in the plan's order, or an undefined tensor when the launch failed.
Tensor sorted_rows(const Tensor& x, const Plan& p, int64_t k) {
  Tensor rows = empty({p.rows, k}, x.scalar_type(), p.device);
  if (api.expert_gather(x.data_ptr(), p.token_of_row, p.limit, rows.data_ptr(), k * x.element_size(), int(p.rows), p.device, stream_of(p.device))) return Tensor();
  return rows;
}

// The checks that a product and its gradients share (experts.py, _check_product).
struct Product {
  const Tensor *x, *w;
  const char* name;
  int64_t n, k;
  int gather, activation;
  bool gated;
};
bool product_of(PyObject* x, PyObject* w, PyObject* gather, PyObject* activation, const Plan& p, Product& q) {
  q.x = cuda_tensor(x), q.w = cuda_tensor(w);
  if (!q.x || !q.w || q.w->dim() != 3 || !(q.name = product_name(q.x->scalar_type())) || !integer(gather, q.gather) || !integer(activation, q.activation)) return false;
  q.n = q.w->size(1), q.k = q.w->size(2);
  q.gated = q.activation >= 5;
  const int64_t multiple = 16 / q.x->element_size();
  return q.activation >= 0 && q.activation <= 6 && is(q.w, q.x->scalar_type(), p.device, {p.experts, q.n, q.k}) &&
         is(q.x, q.x->scalar_type(), p.device, {q.gather ? p.tokens : p.rows, q.k}) && q.n > 0 && q.k > 0 && q.n <= 0x7FFFFFFF && q.k <= 0x7FFFFFFF &&
         q.k % multiple == 0 && !(q.gated && q.n % 16) && aligned(*q.x) && aligned(*q.w);
}
OgExpertProduct launch_of(int mode, const Product& q, const Plan& p, const void* x, const void* w, void* out) {
  OgExpertProduct g{};
  g.x = x, g.w = w, g.offsets = p.offsets, g.out = out, g.mode = mode, g.groups = p.experts, g.rows = int(p.rows), g.x_rows = int(p.tokens);
  g.n = int(q.n), g.k = int(q.k), g.factor = 1.0f;
  std::strncpy(g.dtype, q.name, sizeof g.dtype - 1);
  return g;
}

// expert_gemm(x, w, plan, gather, activation, alpha, preactivation, rows gathered in the product)
PyObject* expert_gemm(PyObject*, PyObject* const* a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  Plan p;
  Product q;
  int64_t few = 0;
  if (count != 8 || !plan_of(a[2], p) || !product_of(a[0], a[1], a[3], a[4], p, q) || !integer(a[7], few)) NOT_SERVED;
  const ScalarType own = q.x->scalar_type() == at::kFloat8_e4m3fn ? at::kBFloat16 : q.x->scalar_type();
  bool ok = true;
  const Tensor* alpha = optional_tensor(a[5], at::kFloat, p.device, {p.experts}, ok);
  const Tensor* z = optional_tensor(a[6], own, p.device, {p.rows, q.n}, ok);
  if (!ok || (z && (overlap(*z, *q.x) || overlap(*z, *q.w) || (alpha && overlap(*z, *alpha)) || overlap(*z, p.offsets, plan_bytes(p))))) NOT_SERVED;
  Tensor out = empty({p.rows, q.gated ? q.n / 2 : q.n}, own, p.device), sorted;
  const void* x = q.x->data_ptr();
  bool gather = q.gather != 0;
  if (gather && p.rows > few * std::min<int64_t>(p.experts, p.rows)) {
    sorted = sorted_rows(*q.x, p, q.k);
    if (!sorted.defined()) return failed(api.routing_error());
    x = sorted.data_ptr(), gather = false;
  }
  OgExpertProduct g = launch_of(0, q, p, x, q.w->data_ptr(), out.data_ptr());
  g.tokens = gather ? p.token_of_row : nullptr;
  g.alpha = static_cast<const float*>(data(alpha)), g.preactivation = const_cast<void*>(data(z)), g.activation = q.activation;
  if (api.expert_product(&g, p.device, stream_of(p.device))) return failed(api.experts_error());
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// expert_gemm_backward(grad, x, w, plan, gather, activation, preactivation, want x, want w) for gradients of the operands' type
PyObject* expert_gemm_backward(PyObject*, PyObject* const* a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  Plan p;
  Product q;
  int want_x = 0, want_w = 0;
  if (count != 9 || !plan_of(a[3], p) || !product_of(a[1], a[2], a[4], a[5], p, q) || !integer(a[7], want_x) || !integer(a[8], want_w)) NOT_SERVED;
  const ScalarType type = q.x->scalar_type();
  const int code = logits_type(type);
  if (code < 1 || q.n % 8) NOT_SERVED;
  bool ok = true;
  const Tensor* grad = cuda_tensor(a[0]);
  const Tensor* z = optional_tensor(a[6], type, p.device, {p.rows, q.n}, ok);
  if (!ok || (q.activation != 0) != (z != nullptr) || !is(grad, type, p.device, {p.rows, q.gated ? q.n / 2 : q.n}) || !aligned(*grad) || (z && !aligned(*z)))
    NOT_SERVED;
  void* const stream = stream_of(p.device);
  // All outputs before the first launch: the weights' gradient, beside the rows', waits for
  // nothing before it writes (experts.py says what memory from between the two could be).
  Tensor dz = *grad, rows = *q.x, by_row, grad_x, grad_w;
  if (want_x) {  // a token's rows are added before anything is rounded
    by_row = empty({p.rows, q.k}, q.gather ? at::kFloat : type, p.device);
    grad_x = q.gather ? empty({p.tokens, q.k}, type, p.device) : by_row;
  }
  if (want_w) grad_w = empty({p.experts, q.n, q.k}, type, p.device);
  if (z) {
    dz = empty({p.rows, q.n}, type, p.device);
    if (api.activation_gradient(code, q.activation, grad->data_ptr(), z->data_ptr(), dz.data_ptr(), nullptr, nullptr, p.limit, p.rows, int(q.n), p.device, stream))
      return failed(api.routing_error());
  }
  if (want_w && q.gather) {
    rows = sorted_rows(*q.x, p, q.k);
    if (!rows.defined()) return failed(api.routing_error());
  }
  if (want_x) {
    OgExpertProduct g = launch_of(1, q, p, dz.data_ptr(), q.w->data_ptr(), by_row.data_ptr());
    g.out_f32 = q.gather;
    if (api.expert_product(&g, p.device, stream)) return failed(api.experts_error());
  }
  if (want_w) {
    OgExpertProduct g = launch_of(2, q, p, dz.data_ptr(), rows.data_ptr(), grad_w.data_ptr());
    g.beside_previous = want_x != 0;
    if (api.expert_product(&g, p.device, stream)) return failed(api.experts_error());
  }
  if (want_x && q.gather &&
      api.expert_combine(code, 1, by_row.data_ptr(), nullptr, p.positions, nullptr, grad_x.data_ptr(), p.tokens, p.top_k, int(q.k), p.device, stream))
    return failed(api.routing_error());
  return tuple({grad_x, grad_w});
  END_HANDLE_TH_ERRORS
}

// expert_combine(y, weights, plan, residual)
PyObject* expert_combine(PyObject*, PyObject* const* a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  Plan p;
  const Tensor* y = count == 4 ? cuda_tensor(a[0]) : nullptr;
  if (!y || !plan_of(a[2], p) || y->dim() != 2 || logits_type(y->scalar_type()) < 1) NOT_SERVED;
  const int64_t n = y->size(1);
  const ScalarType type = y->scalar_type();
  bool ok = n > 0 && n <= 0x7FFFFFFF;
  const Tensor* residual = optional_tensor(a[3], type, p.device, {p.tokens, n}, ok);
  const Tensor* weights = cuda_tensor(a[1]);
  if (!ok || !is(y, type, p.device, {p.rows, n}) || !is(weights, at::kFloat, p.device, {p.tokens, p.top_k})) NOT_SERVED;
  Tensor out = empty({p.tokens, n}, type, p.device);
  if (api.expert_combine(logits_type(type), 0, y->data_ptr(), weights->data_ptr<float>(), p.positions, data(residual), out.data_ptr(), p.tokens, p.top_k, int(n), p.device,
                         stream_of(p.device)))
    return failed(api.routing_error());
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// expert_combine_backward(grad, y, weights, plan)
PyObject* expert_combine_backward(PyObject*, PyObject* const* a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  Plan p;
  const Tensor* y = count == 4 ? cuda_tensor(a[1]) : nullptr;
  if (!y || !plan_of(a[3], p) || y->dim() != 2 || logits_type(y->scalar_type()) < 1) NOT_SERVED;
  const int64_t n = y->size(1);
  const ScalarType type = y->scalar_type();
  const Tensor *grad = cuda_tensor(a[0]), *weights = cuda_tensor(a[2]);
  if (n < 1 || n > 0x7FFFFFFF || !is(y, type, p.device, {p.rows, n}) || !is(grad, type, p.device, {p.tokens, n}) ||
      !is(weights, at::kFloat, p.device, {p.tokens, p.top_k}))
    NOT_SERVED;
  Tensor grad_y = empty({p.rows, n}, type, p.device), grad_weights = empty({p.tokens, p.top_k}, at::kFloat, p.device);
  if (api.expert_combine_gradient(logits_type(type), grad->data_ptr(), y->data_ptr(), weights->data_ptr<float>(), p.positions, grad_y.data_ptr(),
                                  grad_weights.data_ptr<float>(), p.tokens, p.top_k, int(n), p.device, stream_of(p.device)))
    return failed(api.routing_error());
  return tuple({grad_y, grad_weights});
  END_HANDLE_TH_ERRORS
}

// ----------------------------------------------------- the product's epilogue

// What a fused product of these types and extents launches, learnt from a call
// that the Python front end made.
struct Key {
  int64_t m, n, k;
  int a, b, scales, out, mode;
  bool operator==(const Key& o) const { return m == o.m && n == o.n && k == o.k && a == o.a && b == o.b && scales == o.scales && out == o.out && mode == o.mode; }
};
struct KeyHash {
  size_t operator()(const Key& k) const {
    size_t h = size_t(k.m) * 0x9E3779B97F4A7C15ull;
    for (int64_t v : {k.n, k.k, int64_t(k.a) << 40 | int64_t(k.b) << 32 | int64_t(k.scales + 1) << 16 | int64_t(k.out + 1) << 1 | k.mode}) h = (h ^ size_t(v)) * 0xD6E8FEB86659FD93ull, h ^= h >> 29;
    return h;
  }
};
struct Bound {
  OgGemm g;
  ScalarType out;
  int64_t scale_bytes_a, scale_bytes_b;
};
std::unordered_map<Key, Bound, KeyHash> bound;  // under the interpreter's lock

// The key of gemm's arguments, or false: a, b, sfa (or None), out_dtype (or None), launch mode.
bool key_of(const Tensor* a, const Tensor* b, PyObject* sfa, PyObject* out_dtype, PyObject* mode, Key& key) {
  if (!a || !b || a->dim() != 2 || b->dim() != 2 || !integer(mode, key.mode)) return false;
  key.m = a->size(0), key.n = b->size(0), key.k = a->size(1), key.a = int(a->scalar_type()), key.b = int(b->scalar_type());
  key.scales = key.out = -1;
  if (b->size(1) != key.k || a->get_device() != b->get_device()) return false;
  if (sfa != Py_None) {
    const Tensor* s = cuda_tensor(sfa);
    if (!s) return false;
    key.scales = int(s->scalar_type());
  }
  if (out_dtype != Py_None) {
    if (!THPDtype_Check(out_dtype)) return false;
    key.out = int(reinterpret_cast<THPDtype*>(out_dtype)->scalar_type);
  }
  return true;
}

// learn(a, b, sfa, out_dtype, launch mode, address of the OgGemm, C's dtype, bytes of the scales of a and b)
PyObject* learn(PyObject*, PyObject* const* a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  Key key;
  Bound value;
  if (count != 9 || !key_of(cuda_tensor(a[0]), cuda_tensor(a[1]), a[2], a[3], a[4], key) || !THPDtype_Check(a[6]) || !integer(a[7], value.scale_bytes_a) ||
      !integer(a[8], value.scale_bytes_b))
    NOT_SERVED;
  const unsigned long long address = PyLong_AsUnsignedLongLong(a[5]);
  if (PyErr_Occurred()) return nullptr;
  std::memcpy(&value.g, reinterpret_cast<const void*>(uintptr_t(address)), sizeof value.g);
  value.out = reinterpret_cast<THPDtype*>(a[6])->scalar_type;
  if (bound.size() >= 4096) bound.clear();  // a program that never stops meeting new shapes
  bound[key] = value;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* forget(PyObject*, PyObject* const*, Py_ssize_t) {
  bound.clear();
  Py_RETURN_NONE;
}

// gemm(a, b, sfa, sfb, out_dtype, alpha, bias, activation, residual, preactivation, launch mode)
PyObject* gemm(PyObject*, PyObject* const* v, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 11) NOT_SERVED;
  const Tensor *a = cuda_tensor(v[0]), *b = cuda_tensor(v[1]);
  Key key;
  if (!key_of(a, b, v[2], v[4], v[10], key)) NOT_SERVED;
  const auto found = bound.find(key);
  if (found == bound.end()) NOT_SERVED;
  const Bound& e = found->second;
  const int device = a->get_device();
  const Tensor *sfa = nullptr, *sfb = nullptr;
  if (key.scales >= 0) {
    sfa = cuda_tensor(v[2]), sfb = cuda_tensor(v[3]);
    if (!sfb || int(sfb->scalar_type()) != key.scales || sfa->get_device() != device || sfb->get_device() != device || sfa->numel() < e.scale_bytes_a ||
        sfb->numel() < e.scale_bytes_b)
      NOT_SERVED;
  } else if (v[3] != Py_None) {
    NOT_SERVED;
  }
  OgEpilogue epilogue{};
  epilogue.alpha = 1.0f;
  if ((v[5] != Py_None && !number(v[5], epilogue.alpha)) || !integer(v[7], epilogue.activation) || epilogue.activation < 0) NOT_SERVED;
  bool ok = true;
  const Tensor* bias = optional_tensor(v[6], at::kFloat, device, {key.n}, ok);
  const Tensor* residual = optional_tensor(v[8], e.out, device, {key.m, key.n}, ok);
  const Tensor* z = optional_tensor(v[9], e.out, device, {key.m, key.n}, ok);
  if (!ok || (z && !aligned(*z))) NOT_SERVED;
  for (const Tensor* read : {residual, a, b, sfa, sfb, bias})
    if (z && read && overlap(*z, *read)) NOT_SERVED;
  Tensor out = empty({key.m, key.n}, e.out, device);
  epilogue.bias = data(bias), epilogue.residual = data(residual), epilogue.preactivation = const_cast<void*>(data(z));
  if (api.launch_fused(&e.g, a->data_ptr(), b->data_ptr(), data(sfa), data(sfb), out.data_ptr(), device, stream_of(device), &epilogue)) return failed(api.error());
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// gemm_backward(grad, a, b, activation, preactivation, alpha, want a, want b, want bias) for gradients of the operands' type
PyObject* gemm_backward(PyObject*, PyObject* const* v, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  OgGemmGradients g{};
  const Tensor *grad = count == 9 ? cuda_tensor(v[0]) : nullptr, *a = grad ? cuda_tensor(v[1]) : nullptr, *b = a ? cuda_tensor(v[2]) : nullptr;
  if (!b || a->dim() != 2 || b->dim() != 2) NOT_SERVED;
  const ScalarType type = a->scalar_type();
  const int device = a->get_device();
  const int64_t m = a->size(0), n = b->size(0), k = a->size(1);
  int want_a = 0, want_b = 0, want_bias = 0;
  if ((type != at::kBFloat16 && type != at::kHalf) || n % 8 || k % 8 || !n || !k || m > 0x7FFFFFFF || n > 0x7FFFFFFF || k > 0x7FFFFFFF ||
      !is(b, type, device, {n, k}) || !is(grad, type, device, {m, n}) || !integer(v[3], g.activation) || g.activation < 0 || !integer(v[6], want_a) ||
      !integer(v[7], want_b) || !integer(v[8], want_bias))
    NOT_SERVED;
  bool ok = true;
  const Tensor* z = optional_tensor(v[4], type, device, {m, n}, ok);
  g.factor = 1.0f;
  if (!ok || (g.activation != 0) != (z != nullptr) || (v[5] != Py_None && !number(v[5], g.factor)) || !aligned(*a) || !aligned(*b) || !aligned(*grad) ||
      (z && !aligned(*z)))
    NOT_SERVED;
  Tensor grad_a, grad_b, grad_bias, workspace;
  if (want_a) g.grad_a = (grad_a = empty({m, k}, type, device)).data_ptr();
  if (want_b) g.grad_b = (grad_b = empty({n, k}, type, device)).data_ptr();
  if (want_bias) g.grad_bias = (grad_bias = empty({n}, at::kFloat, device)).data_ptr<float>();
  g.grad = grad->data_ptr(), g.a = a->data_ptr(), g.b = b->data_ptr(), g.z = data(z), g.m = int(m), g.n = int(n), g.k = int(k);
  std::strncpy(g.dtype, type == at::kBFloat16 ? "bf16" : "f16", sizeof g.dtype - 1);
  g.workspace_bytes = api.gemm_gradients_workspace(&g, device);
  if (g.workspace_bytes > 0) g.workspace = (workspace = empty({g.workspace_bytes}, at::kByte, device)).data_ptr();
  if (api.gemm_gradients(&g, device, stream_of(device))) return failed(api.experts_error());
  return tuple({grad_a, grad_b, grad_bias});
  END_HANDLE_TH_ERRORS
}

// bind({name: address}): where the library's entry points are.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t count) {
  if (count != 1 || !PyDict_Check(a[0])) return failed("bind takes a dict of addresses");
  const auto address = [&](const char* name) -> void* {
    PyObject* o = PyDict_GetItemString(a[0], name);
    return o ? PyLong_AsVoidPtr(o) : nullptr;
  };
#define BIND(field, name) api.field = reinterpret_cast<decltype(api.field)>(address(name))
  BIND(route, "og_b200_route");
  BIND(route_gradient, "og_b200_route_gradient");
  BIND(expert_plan, "og_b200_expert_plan");
  BIND(expert_gather, "og_b200_expert_gather");
  BIND(expert_product, "og_b200_expert_product");
  BIND(expert_combine, "og_b200_expert_combine");
  BIND(expert_combine_gradient, "og_b200_expert_combine_gradient");
  BIND(activation_gradient, "og_b200_activation_gradient");
  BIND(gemm_gradients, "og_b200_gemm_gradients");
  BIND(gemm_gradients_workspace, "og_b200_gemm_gradients_workspace");
  BIND(launch_fused, "og_b200_launch_fused");
  BIND(routing_error, "og_b200_routing_error");
  BIND(experts_error, "og_b200_experts_error");
  BIND(error, "og_mm_error");
#undef BIND
  if (PyErr_Occurred()) return nullptr;
  if (!api.route || !api.route_gradient || !api.expert_plan || !api.expert_gather || !api.expert_product || !api.expert_combine || !api.expert_combine_gradient ||
      !api.activation_gradient || !api.gemm_gradients || !api.gemm_gradients_workspace || !api.launch_fused || !api.routing_error || !api.experts_error || !api.error)
    return failed("an entry point is missing");
  Py_RETURN_NONE;
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind), METHOD(route), METHOD(route_backward), METHOD(expert_plan), METHOD(expert_gemm), METHOD(expert_gemm_backward), METHOD(expert_combine),
                         METHOD(expert_combine_backward), METHOD(gemm), METHOD(gemm_backward), METHOD(learn), METHOD(forget), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "front", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_front(void) { return PyModule_Create(&module); }
