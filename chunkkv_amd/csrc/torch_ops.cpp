// The torch-facing calls that a decoder layer makes many times per request, as one CPython call
// each: argument checks, output allocation and the C-ABI launch (include/chunkkv_amd.h) without the
// interpreter in between. chunkkv_amd/ops.py keeps their names, signatures and documentation and
// raises the same exceptions for the same misuse; everything else there calls the C ABI through
// ctypes.
//
// Bound: host time. A layer's launches take 3-15 us on the GPU at short requests, and a wrapper in
// Python (a dozen tensor attributes, an allocation, a 20-argument ctypes call) took 8-11 us of the
// host for each: attention_active 9.4 us, rope_qkv (k/v into a cache) 10.9, add_rmsnorm 8.0,
// silu_mul 12.2. The launch itself is 2-3 us of that.
#include <Python.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <torch/types.h>
#include <pybind11/pybind11.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <utility>
#include <vector>

#include "chunkkv_amd.h"

namespace {

using at::Tensor;

// A Python exception on its way out: ValueError, TypeError or RuntimeError with a message.
struct PyFailure {
  PyObject* type;
  std::string what;
};
[[noreturn]] void value_error(std::string s) { throw PyFailure{PyExc_ValueError, std::move(s)}; }
[[noreturn]] void type_error(std::string s) { throw PyFailure{PyExc_TypeError, std::move(s)}; }

#define CKV_PY_BEGIN HANDLE_TH_ERRORS try {
#define CKV_PY_END                          \
  }                                         \
  catch (const PyFailure& f) {              \
    PyErr_SetString(f.type, f.what.c_str()); \
    return nullptr;                         \
  }                                         \
  END_HANDLE_TH_ERRORS

void need_args(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) type_error("expected " + std::to_string(want) + " arguments, got " + std::to_string(got));
}
const Tensor& tensor(PyObject* o) {
  if (!THPVariable_Check(o)) type_error(std::string("expected a tensor, got ") + Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
Tensor optional_tensor(PyObject* o) { return o == Py_None ? Tensor() : tensor(o); }
int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
int32_t int32(int64_t v) { return (int32_t)v; }  // as a ctypes c_int32 argument takes it

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream_of(const Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream();
}
int dtype_code(const Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return CKV_DTYPE_BF16;
  if (t.scalar_type() == at::kFloat) return CKV_DTYPE_F32;
  type_error(std::string("unsupported K/V dtype ") + c10::toString(t.scalar_type()) +
             "; the HIP kernels take float32 or bfloat16");
}

// Every tensor on one HIP device.
template <typename... T>
void same_device(const Tensor& first, const T&... rest) {
  for (const Tensor* t : {&first, &rest...}) {
    if (!t->is_cuda()) value_error("chunkkv_amd ops run on a HIP device; got a tensor on " + t->device().str());
    if (t->device() != first.device())
      value_error("tensors on different devices: " + t->device().str() + " vs " + first.device().str());
  }
}
void need_dims(const Tensor& t, int64_t d, const char* what) {
  if (t.dim() != d) value_error(std::string(what) + " must have " + std::to_string(d) + " dimensions");
}
std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}
// Last dim contiguous, base and every other stride on a 16-byte boundary; else a contiguous copy.
Tensor rows_view(const Tensor& t) {
  bool ok = t.stride(-1) == 1 && (uintptr_t)t.data_ptr() % 16 == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && t.stride(i) * t.element_size() % 16 == 0;
  return ok ? t : t.contiguous();
}

// The status of a C-ABI call as the exception chunkkv_amd/_native.py:check raises.
void check(int32_t status, const char* what) {
  if (status == CKV_OK) return;
  const std::string msg =
      std::string(what) + ": " + ckv_status_string(status) + " (status " + std::to_string(status) + ")";
  if (status == CKV_ERR_INVALID_ARGUMENT || status == CKV_ERR_OUT_OF_RANGE || status == CKV_ERR_TOO_LARGE) value_error(msg);
  throw PyFailure{PyExc_RuntimeError, msg};
}
// The launch itself runs without the interpreter lock, as a ctypes call does. f looks up addresses
// and the stream too, which throw (a tensor without storage, a HIP error): the lock is taken back
// on that way out as well, before any handler touches the interpreter.
struct Unlocked {
  PyThreadState* const state = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  Unlocked& operator=(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state); }
};
template <typename F>
int32_t unlocked(F f) {
  const Unlocked section;
  return f();
}

// attention_active(q, K, V, positions, scale, err, out, split)
PyObject* attention_active(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  CKV_PY_BEGIN
  need_args(n_args, 8);
  Tensor q = tensor(a[0]);
  const Tensor &K = tensor(a[1]), &V = tensor(a[2]);
  Tensor pos = tensor(a[3]);
  const Tensor err = optional_tensor(a[5]);
  Tensor out = optional_tensor(a[6]);
  same_device(q, K, V, pos);
  need_dims(q, 4, "q");
  need_dims(K, 4, "K");
  const int64_t Hq = q.size(1), n = q.size(2), D = q.size(3), Hkv = K.size(1), N = K.size(2);
  if (q.scalar_type() != at::kBFloat16 || K.scalar_type() != at::kBFloat16 || V.scalar_type() != at::kBFloat16)
    type_error("attention_active runs on bf16 q/K/V");
  if (!K.is_contiguous() || !V.is_contiguous() || V.sizes() != K.sizes() || K.size(3) != D)
    value_error("K/V must be contiguous (1, Hkv, N, D) and match q's head_dim");
  if (q.stride(3) != 1) q = q.contiguous();
  if (pos.scalar_type() != at::kLong || pos.numel() != n) value_error("positions must be int64 (n,)");
  pos = pos.contiguous();
  if (!out.defined()) {
    out = at::empty({1, n, Hq, D}, q.options());
  } else if (out.sizes() != at::IntArrayRef({1, n, Hq, D}) || !out.is_contiguous() || out.scalar_type() != q.scalar_type()) {
    value_error("out must be contiguous (1, n, Hq, D) bf16");
  }
  const double scale = a[4] == Py_None ? 1.0 / std::sqrt((double)D) : real(a[4]);
  const int split = PyObject_IsTrue(a[7]);
  if (split < 0) throw python_error();
  const int64_t ws_bytes =
      split ? ckv_attention_workspace_bytes(int32(n), int32(N), int32(Hq), int32(D), nullptr, nullptr) : 0;
  Tensor ws;
  if (ws_bytes > 0) ws = at::empty({ws_bytes / 4}, q.options().dtype(at::kFloat));
  check(unlocked([&] {
          return ckv_attention_active(ptr(out), ptr(q), q.stride(1), q.stride(2), ptr(K), ptr(V), N * D,
                                      (const int64_t*)ptr(pos), int32(n), int32(N), int32(Hq), int32(Hkv), int32(D),
                                      CKV_DTYPE_BF16, scale, ptr(ws), ws_bytes, (int32_t*)ptr(err), stream_of(q));
        }),
        "ckv_attention_active");
  return THPVariable_Wrap(out);
  CKV_PY_END
}

// Pointer, head stride and token stride of a (1, n, n_heads * D) token-major tensor or a
// (1, H, n, D) tensor with contiguous rows.
struct Heads {
  void* p = nullptr;
  int64_t hs = 0, ts = 0;
};
Heads heads_view(const Tensor& t, int64_t n_heads, int64_t D) {
  if (t.dim() == 3) {
    if (t.stride(2) != 1 || t.size(2) != n_heads * D)
      value_error("projection output must have contiguous rows of n_heads * head_dim");
    return {ptr(t), D, t.stride(1)};
  }
  if (t.dim() == 4 && t.size(1) == n_heads && t.size(3) == D && t.stride(3) == 1) return {ptr(t), t.stride(1), t.stride(2)};
  value_error("unsupported layout " + shape_of(t));
}

// rope_qkv(q_in, k_in, v_in, positions, n_q_heads, n_kv_heads, head_dim, theta, q_out, k_out, v_out, rows, table, err)
PyObject* rope_qkv(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  CKV_PY_BEGIN
  need_args(n_args, 14);
  const Tensor &k_in = tensor(a[1]), v_in = optional_tensor(a[2]);
  Tensor pos = tensor(a[3]);
  const int64_t Hq = integer(a[4]), Hkv = integer(a[5]), D = integer(a[6]);
  const double theta = real(a[7]);
  const Tensor q_in = Hq == 0 ? k_in : tensor(a[0]);  // k/v only: q is not read
  Tensor q_out = optional_tensor(a[8]), k_out = optional_tensor(a[9]);
  const Tensor v_out = optional_tensor(a[10]), table = optional_tensor(a[12]), err = optional_tensor(a[13]);
  Tensor rows = optional_tensor(a[11]);
  if (table.defined()) {
    same_device(k_in, table);
    if (table.scalar_type() != at::kFloat || table.dim() != 3 || table.size(1) != D / 2 || table.size(2) != 2)
      value_error("table must be a rope_table() output (n, D/2, 2) float32");
  }
  same_device(k_in, pos);
  const int64_t n = pos.numel();
  if (pos.scalar_type() != at::kLong) value_error("positions must be int64");
  const bool rows_are_positions = rows.defined() && a[11] == a[3];
  pos = pos.contiguous();
  if (!q_out.defined() && Hq) q_out = at::empty({1, n, Hq, D}, q_in.options().device(k_in.device()));
  if (!k_out.defined()) {
    if (rows.defined()) value_error("rows needs k_out (the cache)");
    k_out = at::empty({1, Hkv, n, D}, q_in.options().device(k_in.device()));
  }
  const int64_t n_out = k_out.dim() == 4 ? k_out.size(2) : k_out.size(1);
  if (rows.defined()) {
    same_device(q_in, rows);
    if (rows.scalar_type() != at::kLong || rows.numel() != n) value_error("rows must be int64 (n,)");
    rows = rows_are_positions ? pos : rows.contiguous();
  }
  if (v_in.defined() != v_out.defined()) value_error("v_in and v_out go together");
  const auto dt = q_in.scalar_type();
  if (k_in.scalar_type() != dt || k_out.scalar_type() != dt || (Hq && q_out.scalar_type() != dt) ||
      (v_in.defined() && (v_in.scalar_type() != dt || v_out.scalar_type() != dt)))
    type_error("q/k/v and outputs must share a dtype");
  Heads qo, qi, vi, vo;
  if (Hq) {
    if (q_out.sizes() != at::IntArrayRef({1, n, Hq, D}) || !q_out.is_contiguous())
      value_error("q_out must be contiguous (1, n, Hq, D), token-major");
    qo = {ptr(q_out), D, Hq * D};
    qi = heads_view(q_in, Hq, D);
  }
  const Heads ki = heads_view(k_in, Hkv, D), ko = heads_view(k_out, Hkv, D);
  if (v_in.defined()) vi = heads_view(v_in, Hkv, D);
  if (v_out.defined()) vo = heads_view(v_out, Hkv, D);
  const int code = dtype_code(q_in);
  check(unlocked([&] {
          return ckv_rope_qkv(qo.p, qo.hs, qo.ts, ko.p, ko.hs, ko.ts, vo.p, vo.hs, vo.ts, (const int64_t*)ptr(rows),
                              int32(n_out), qi.p, qi.hs, qi.ts, ki.p, ki.hs, ki.ts, vi.p, vi.hs, vi.ts,
                              (const int64_t*)ptr(pos), ptr(table), table.defined() ? table.size(0) : 0, int32(n),
                              int32(Hq), int32(Hkv), int32(D), code, theta, (int32_t*)ptr(err), stream_of(k_in));
        }),
        "ckv_rope_qkv");
  PyObject* q_obj;
  if (q_out.defined()) {
    q_obj = THPVariable_Wrap(q_out);
  } else {
    Py_INCREF(Py_None);
    q_obj = Py_None;
  }
  return Py_BuildValue("(NN)", q_obj, THPVariable_Wrap(k_out));
  CKV_PY_END
}

// add_rmsnorm(h, delta, weight, eps, h_out, out)
PyObject* add_rmsnorm(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  CKV_PY_BEGIN
  need_args(n_args, 6);
  const Tensor &h = tensor(a[0]), delta = optional_tensor(a[1]), &weight = tensor(a[2]);
  const double eps = real(a[3]);
  Tensor h_out = optional_tensor(a[4]), out = optional_tensor(a[5]);
  if (delta.defined()) same_device(h, weight, delta);
  else same_device(h, weight);
  if (h.dim() == 0) throw PyFailure{PyExc_IndexError, "tuple index out of range"};
  const int64_t hidden = h.size(-1);
  if (!h.is_contiguous() || (delta.defined() && (!delta.is_contiguous() || delta.sizes() != h.sizes())))
    value_error("h and delta must be contiguous and of one shape");
  if (weight.dim() != 1 || weight.size(0) != hidden || weight.scalar_type() != h.scalar_type() ||
      (delta.defined() && delta.scalar_type() != h.scalar_type()))
    value_error("weight must be (hidden,) and every operand of h's dtype");
  auto fits = [&](const Tensor& t) { return t.sizes() == h.sizes() && t.is_contiguous() && t.scalar_type() == h.scalar_type(); };
  if (!out.defined()) out = at::empty(h.sizes(), h.options());
  else if (!fits(out)) value_error("out must be contiguous, of h's shape and dtype");
  if (delta.defined() && !h_out.defined()) h_out = at::empty(h.sizes(), h.options());
  else if (h_out.defined() && !fits(h_out)) value_error("h_out must be contiguous, of h's shape and dtype");
  const Tensor w = weight.contiguous();
  const int code = dtype_code(h);
  check(unlocked([&] {
          return ckv_add_rmsnorm(ptr(h_out), ptr(h), ptr(delta), ptr(out), ptr(w), hidden ? h.numel() / hidden : 0,
                                 int32(hidden), (float)eps, code, stream_of(h));
        }),
        "ckv_add_rmsnorm");
  return Py_BuildValue("(NN)", THPVariable_Wrap(delta.defined() ? h_out : h), THPVariable_Wrap(out));
  CKV_PY_END
}

// Row stride (elements) of a (..., width) tensor whose rows are contiguous and evenly spaced.
int64_t row_major(const Tensor& t, int64_t width, const char* what) {
  const std::string w(what);
  if (t.size(-1) != width || t.stride(-1) != 1 || (uintptr_t)t.data_ptr() % 16 != 0)
    value_error(w + " must have contiguous, 16-byte aligned rows of " + std::to_string(width) + " elements");
  if (t.dim() == 2) return t.size(0) > 1 ? t.stride(0) : width;
  int64_t step = -1, seen = 1;  // outer dimensions, innermost first: each must continue the ones inside it
  for (int64_t i = t.dim() - 2; i >= 0; --i) {
    if (t.size(i) == 0) return width;
    if (t.size(i) == 1) continue;
    if (step < 0) step = t.stride(i);
    else if (t.stride(i) != step * seen) value_error(w + " rows must be evenly spaced");
    seen *= t.size(i);
  }
  return step < 0 ? width : step;
}

// silu_mul(gate, up, out)
PyObject* silu_mul(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  CKV_PY_BEGIN
  need_args(n_args, 3);
  const Tensor &gate = tensor(a[0]), &up = tensor(a[1]);
  Tensor out = optional_tensor(a[2]);
  same_device(gate, up);
  if (gate.dim() == 0) throw PyFailure{PyExc_IndexError, "tuple index out of range"};
  const int64_t width = gate.size(-1);
  if (up.sizes() != gate.sizes() || up.scalar_type() != gate.scalar_type())
    value_error("gate and up must have one shape and dtype");
  const int64_t gs = row_major(gate, width, "gate"), us = row_major(up, width, "up");
  if (!out.defined()) {
    out = at::empty(gate.sizes(), gate.options());
  } else if (out.sizes() != gate.sizes() || !out.is_contiguous() || out.scalar_type() != gate.scalar_type()) {
    value_error("out must be contiguous, of gate's shape and dtype");
  }
  const int code = dtype_code(gate);
  check(unlocked([&] {
          return ckv_silu_mul(ptr(out), width, ptr(gate), gs, ptr(up), us, width ? gate.numel() / width : 0,
                              int32(width), code, stream_of(gate));
        }),
        "ckv_silu_mul");
  return THPVariable_Wrap(out);
  CKV_PY_END
}

// Whether a call with these operands would reach torch's device code with nothing in between: no
// tracing, transform (vmap), mode, autocast or tensor subclass takes part, which the kernels here
// know nothing of.
bool unintercepted(c10::DispatchKeySet operands) {
  static const c10::DispatchKeySet plain({c10::DispatchKey::CUDA, c10::DispatchKey::AutogradCUDA,
                                          c10::DispatchKey::ADInplaceOrView, c10::DispatchKey::BackendSelect});
  const auto tls = c10::impl::tls_local_dispatch_key_set();
  const c10::DispatchKeySet keys = (operands | tls.included_) - tls.excluded_;
  return (keys.raw_repr() & ~plain.raw_repr()) == 0;
}

// linear(x, weight, bias): ckv_linear where it is the better choice and takes the operands, else torch's
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  CKV_PY_BEGIN
  need_args(n_args, 3);
  const Tensor &x = tensor(a[0]), &w = tensor(a[1]), bias = optional_tensor(a[2]);
  auto plain = [&](const Tensor& t) {
    return t.is_cuda() && t.device() == x.device() && t.scalar_type() == at::kBFloat16 && t.is_contiguous() &&
           unintercepted(t.key_set()) && !t._fw_grad(/*level=*/0).defined() && (uintptr_t)t.data_ptr() % 16 == 0 &&
           !(at::GradMode::is_enabled() && t.requires_grad());
  };
  int64_t ws_bytes = -1;
  if (x.dim() >= 2 && w.dim() == 2 && x.size(-1) == w.size(1) && w.numel() > 0 && x.numel() > 0 && plain(x) && plain(w) &&
      (!bias.defined() || (bias.dim() == 1 && bias.size(0) == w.size(0) && plain(bias)))) {
    const int64_t rows = x.numel() / x.size(-1);
    if (rows <= INT32_MAX && w.size(0) <= INT32_MAX && w.size(1) <= INT32_MAX)
      ws_bytes = ckv_linear_workspace_bytes(int32(rows), int32(w.size(0)), int32(w.size(1)));
  }
  if (ws_bytes < 0) {
    Tensor out;
    {
      pybind11::gil_scoped_release off;
      out = at::linear(x, w, bias.defined() ? std::optional<Tensor>(bias) : std::nullopt);
    }
    return THPVariable_Wrap(out);
  }
  at::DimVector shape(x.sizes().begin(), x.sizes().end());
  shape.back() = w.size(0);
  Tensor out = at::empty(shape, x.options()), ws;
  if (ws_bytes > 0) ws = at::empty({ws_bytes / 4}, x.options().dtype(at::kFloat));
  check(unlocked([&] {
          return ckv_linear(ptr(out), ptr(x), x.size(-1), ptr(w), ptr(bias), int32(x.numel() / x.size(-1)),
                            int32(w.size(0)), int32(w.size(1)), CKV_DTYPE_BF16, ptr(ws), ws_bytes, stream_of(x));
        }),
        "ckv_linear");
  return THPVariable_Wrap(out);
  CKV_PY_END
}

// layer1_repair_gather(k_slab, v_slab, src_tab, layer, begin, end, segments, n_segs, max_seg_tokens, k, v, flags,
//                      local, spans, threshold, theta, workspace, err, out, diff_norm) with out None or the six
// tensors of a Selection and diff_norm None or two: (diff, norm, the six tensors)
PyObject* layer1_repair_gather(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  CKV_PY_BEGIN
  need_args(n_args, 20);
  const Tensor &ks = tensor(a[0]), &vs = tensor(a[1]), &tab = tensor(a[2]);
  const int64_t layer = integer(a[3]), begin = integer(a[4]), end = integer(a[5]);
  const Tensor& segs = tensor(a[6]);
  const int64_t n_segs = integer(a[7]), max_seg = integer(a[8]);
  Tensor k = tensor(a[9]), v = tensor(a[10]);
  const Tensor &flags = tensor(a[11]), &local = tensor(a[12]), &spans = tensor(a[13]);
  const bool has_thr = a[14] != Py_None;
  const double thr = has_thr ? real(a[14]) : 0.0, theta = real(a[15]);
  const Tensor &ws = tensor(a[16]), err = optional_tensor(a[17]);
  if (ks.dim() != 5 || vs.sizes() != ks.sizes() || !ks.is_contiguous() || !vs.is_contiguous())
    value_error("k_slab/v_slab must be contiguous (L, 1, H, N, D)");
  const int64_t L = ks.size(0), H = ks.size(2), N = ks.size(3), D = ks.size(4);
  if (!(0 <= begin && begin <= end && end <= L) || (begin <= layer && layer < end))
    value_error("gather layers (" + std::to_string(begin) + ", " + std::to_string(end) + ") must lie in [0, " +
                std::to_string(L) + ") and exclude layer " + std::to_string(layer));
  if (layer < -L || layer >= L) throw PyFailure{PyExc_IndexError, "layer out of range"};
  same_device(ks, vs, tab, segs, k, v, flags, local, spans, ws);
  k = rows_view(k);
  v = rows_view(v);
  if (ks.scalar_type() != k.scalar_type() || vs.scalar_type() != k.scalar_type() || v.scalar_type() != k.scalar_type())
    type_error("fresh and cached K/V must share a dtype");
  if (k.dim() != 4 || k.size(1) != H || k.size(3) != D || v.sizes() != k.sizes())
    value_error("fresh k/v shape " + shape_of(k) + " does not match cache " + shape_of(ks));
  if (flags.scalar_type() != at::kByte || local.scalar_type() != at::kInt || flags.numel() != N || local.numel() != N)
    value_error("flags must be uint8 (N,) and local int32 (N,)");
  if (!flags.is_contiguous() || !local.is_contiguous()) value_error("flags and local must be contiguous");
  if (tab.scalar_type() != at::kLong || tab.numel() % (2 * L)) value_error("src_tab must be int64 with 2 addresses per (chunk, layer)");
  if (segs.scalar_type() != at::kInt || segs.numel() < 6 * n_segs) value_error("segments must be int32 with 6 fields per segment");
  if (spans.scalar_type() != at::kInt || spans.numel() % 4) value_error("spans must be int32 (C, 4)");
  if ((int64_t)(ws.numel() * ws.element_size()) < CKV_LAYER1_REPAIR_WORKSPACE_BYTES || !ws.is_contiguous())
    value_error("workspace must come from layer1_repair_workspace()");
  const int64_t C = spans.numel() / 4;
  auto of = [&](at::ScalarType t, int64_t n) { return at::empty({n}, ks.options().dtype(t)); };
  Tensor dn[2], out[6];
  auto given = [](PyObject* o, Tensor* to, Py_ssize_t n) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != n) type_error("expected a tuple of " + std::to_string(n) + " tensors");
    for (Py_ssize_t i = 0; i < n; ++i) to[i] = tensor(PyTuple_GET_ITEM(o, i));
  };
  if (a[19] != Py_None) given(a[19], dn, 2);
  else for (Tensor& t : dn) t = of(at::kFloat, N);
  if (a[18] != Py_None) {
    given(a[18], out, 6);
  } else {
    out[0] = of(at::kLong, N);
    out[1] = of(at::kLong, N);
    out[2] = of(at::kInt, N);
    out[3] = of(at::kFloat, C);
    out[4] = of(at::kByte, C);
    out[5] = of(at::kInt, CKV_COUNT_N);
  }
  const int code = dtype_code(ks);
  check(unlocked([&] {
          return ckv_layer1_repair_gather(
              ptr(ks), ptr(vs), H * N * D, N * D, (const uint64_t*)ptr(tab), int32(tab.numel() / (2 * L)), int32(L),
              int32(layer), int32(begin), int32(end), (const ckv_segment*)ptr(segs), int32(n_segs), int32(max_seg),
              ptr(k), k.stride(1), k.stride(2), ptr(v), v.stride(1), v.stride(2), int32(k.size(2)),
              (const uint8_t*)ptr(flags), (const int32_t*)ptr(local), int32(N), int32(H), int32(D), code, theta,
              (const ckv_chunk_span*)ptr(spans), int32(C), has_thr, thr, (float*)ptr(dn[0]), (float*)ptr(dn[1]),
              (int64_t*)ptr(out[0]), (int64_t*)ptr(out[1]), (int32_t*)ptr(out[2]), (float*)ptr(out[3]),
              (uint8_t*)ptr(out[4]), (int32_t*)ptr(out[5]), ptr(ws), (int64_t)(ws.numel() * ws.element_size()),
              (int32_t*)ptr(err), stream_of(ks));
        }),
        "ckv_layer1_repair_gather");
  PyObject* r = PyTuple_New(8);
  if (r == nullptr) return nullptr;
  for (int i = 0; i < 8; ++i) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(i < 2 ? dn[i] : out[i - 2]));
  return r;
  CKV_PY_END
}

// extract_chunks(k_slab, v_slab, spans, err): a list of one (2, L, 1, H, end - start, D) tensor per span
PyObject* extract_chunks(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  CKV_PY_BEGIN
  need_args(n_args, 4);
  const Tensor &ks = tensor(a[0]), &vs = tensor(a[1]), err = optional_tensor(a[3]);
  same_device(ks, vs);
  if (!ks.is_contiguous() || !vs.is_contiguous() || ks.sizes() != vs.sizes())
    value_error("K/V slabs must be contiguous and of equal shape");
  need_dims(ks, 5, "K/V slabs");
  const int64_t L = ks.size(0), H = ks.size(2), N = ks.size(3), D = ks.size(4);
  // (start, end) pairs as any iterables of integers
  std::vector<std::pair<int64_t, int64_t>> spans;
  {
    THPObjectPtr seq(PySequence_Fast(a[2], "spans must be a sequence of (start, end) pairs"));
    if (!seq) throw python_error();
    auto whole = [](PyObject* o) {
      THPObjectPtr i(PyNumber_Long(o));
      if (!i) throw python_error();
      return integer(i.get());
    };
    for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(seq.get()); ++i) {
      THPObjectPtr pair(PySequence_Fast(PySequence_Fast_GET_ITEM(seq.get(), i), "a span is a (start, end) pair"));
      if (!pair) throw python_error();
      if (PySequence_Fast_GET_SIZE(pair.get()) != 2) value_error("a span is a (start, end) pair");
      const int64_t start = whole(PySequence_Fast_GET_ITEM(pair.get(), 0)), end = whole(PySequence_Fast_GET_ITEM(pair.get(), 1));
      if (!(0 <= start && start <= end && end <= N))
        value_error("span [" + std::to_string(start) + ", " + std::to_string(end) + ") outside the request of " +
                    std::to_string(N) + " tokens");
      spans.emplace_back(start, end);
    }
  }
  std::vector<Tensor> bufs;
  int64_t live = 0, most = 0;
  for (const auto& [start, end] : spans) {
    bufs.push_back(at::empty({2, L, 1, H, end - start, D}, ks.options()));
    live += end > start;
    most = std::max(most, end - start);
  }
  const int code = live > 0 ? dtype_code(ks) : 0;
  // Up to 64 segments go by value with the launch; a longer list goes through device memory.
  if (live > 0 && live <= 64) {
    uint64_t dst[64];
    int32_t rows[128];
    int32_t n = 0;
    for (size_t i = 0; i < spans.size(); ++i) {
      if (spans[i].second == spans[i].first) continue;
      dst[n] = (uint64_t)(uintptr_t)bufs[i].data_ptr();
      rows[2 * n] = (int32_t)spans[i].first;
      rows[2 * n++ + 1] = (int32_t)(spans[i].second - spans[i].first);
    }
    check(unlocked([&] {
            return ckv_extract_chunks_host(ptr(ks), ptr(vs), H * N * D, N * D, dst, rows, n, int32(L), int32(H), int32(N),
                                           int32(D), code, stream_of(ks));
          }),
          "ckv_extract_chunks_host");
  } else if (live > 0) {
    // descriptors: an address per span, then (start, length) pairs; pinned, one async copy (torch's
    // pinned allocator keeps the host block until the copy has run)
    Tensor host = at::empty({live * 2}, at::TensorOptions().dtype(at::kLong).pinned_memory(true));
    int64_t* at64 = host.data_ptr<int64_t>();
    int32_t* at32 = reinterpret_cast<int32_t*>(at64 + live);
    for (size_t i = 0; i < spans.size(); ++i) {
      if (spans[i].second == spans[i].first) continue;
      *at64++ = (int64_t)(uintptr_t)bufs[i].data_ptr();
      *at32++ = (int32_t)spans[i].first;
      *at32++ = (int32_t)(spans[i].second - spans[i].first);
    }
    const Tensor d = host.to(ks.device(), /*non_blocking=*/true);
    const uint64_t* dst = (const uint64_t*)ptr(d);
    check(unlocked([&] {
            return ckv_extract_chunks(ptr(ks), ptr(vs), H * N * D, N * D, dst, (const int32_t*)(dst + live),
                                      int32(live), int32(most), int32(L), int32(H), int32(N), int32(D), code,
                                      (int32_t*)ptr(err), stream_of(ks));
          }),
          "ckv_extract_chunks");
  }
  THPObjectPtr list(PyList_New((Py_ssize_t)bufs.size()));
  if (!list) return nullptr;
  for (size_t i = 0; i < bufs.size(); ++i) PyList_SET_ITEM(list.get(), (Py_ssize_t)i, THPVariable_Wrap(bufs[i]));
  return list.release();
  CKV_PY_END
}

// A new tensor beside `like`, without the dispatcher's round.
Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

// An 8-bit cache's four tensors of one shape: codes (1, H, N, D), scales (1, H, ceil(N / block)).
struct CodedCache {
  const Tensor &k, &v, &ks, &vs;
  int64_t block, H, N, D;
};
CodedCache coded_cache(PyObject* const* a) {
  const Tensor &k = tensor(a[0]), &v = tensor(a[1]), &ks = tensor(a[2]), &vs = tensor(a[3]);
  const int64_t block = integer(a[4]);
  if (block != 32 && block != 64 && block != 128) value_error("block_tokens must be 32, 64 or 128");
  need_dims(k, 4, "an 8-bit cache's codes");
  if (k.scalar_type() != at::kFloat8_e4m3fn || v.scalar_type() != at::kFloat8_e4m3fn ||
      ks.scalar_type() != at::kFloat8_e8m0fnu || vs.scalar_type() != at::kFloat8_e8m0fnu)
    type_error("an 8-bit cache has float8_e4m3fn codes and float8_e8m0fnu scales");
  const int64_t H = k.size(1), N = k.size(2), D = k.size(3), blocks = (N + block - 1) / block;
  if (k.size(0) != 1 || !k.is_contiguous() || !v.is_contiguous() || v.sizes() != k.sizes())
    value_error("an 8-bit cache's codes must be contiguous (1, Hkv, N, D)");
  if (ks.sizes() != at::IntArrayRef({1, H, blocks}) || vs.sizes() != ks.sizes() || !ks.is_contiguous() || !vs.is_contiguous())
    value_error("an 8-bit cache's scales must be contiguous (1, Hkv, ceil(N / block_tokens))");
  if (N > INT32_MAX) value_error("an 8-bit cache has at most 2^31 - 1 rows");
  return {k, v, ks, vs, block, H, N, D};
}

// Head stride (elements) of a (1, H, N, D) cache whose heads each have contiguous rows.
int64_t head_stride(const Tensor& t, const char* what) {
  const int64_t N = t.size(2), D = t.size(3);
  const bool rows = t.stride(3) == 1 && (N <= 1 || t.stride(2) == D);
  const int64_t hs = t.size(1) > 1 ? t.stride(1) : std::max(t.stride(1), N * D);
  if (!rows || hs < N * D) value_error(std::string(what) + " must have each head's rows contiguous");
  return t.size(1) > 1 ? hs : N * D;
}
// Stride of dimension d; where there is one element or none, any number serves: the packed one.
int64_t step(const Tensor& t, int64_t d, int64_t packed) { return t.size(d) > 1 ? t.stride(d) : packed; }
// An optional device status word.
int32_t* status_word(const Tensor& err, const Tensor& like) {
  if (!err.defined()) return nullptr;
  same_device(like, err);
  if (err.scalar_type() != at::kInt || err.numel() < 1) value_error("err must be an int32 tensor");
  return (int32_t*)ptr(err);
}

// quantize_rows(k codes, v codes, k scales, v scales, block, k, v, start, err)
PyObject* quantize_rows(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  CKV_PY_BEGIN
  need_args(n_args, 9);
  const CodedCache c = coded_cache(a);
  Tensor k = tensor(a[5]), v = tensor(a[6]);
  const Tensor err = optional_tensor(a[8]);
  same_device(c.k, c.v, c.ks, c.vs, k, v);
  need_dims(k, 4, "k");
  const int64_t n = k.size(2);
  if (k.size(0) != 1 || k.size(1) != c.H || k.size(3) != c.D || v.sizes() != k.sizes())
    value_error("rows " + shape_of(k) + " do not match the cache " + shape_of(c.k));
  if (v.scalar_type() != k.scalar_type()) type_error("k and v must share a dtype");
  const int code = dtype_code(k);
  int64_t start = 0;
  Tensor start_dev;
  if (THPVariable_Check(a[7])) {
    start_dev = tensor(a[7]);
    same_device(c.k, start_dev);
    if (start_dev.scalar_type() != at::kLong || start_dev.numel() != 1) value_error("start must be an int or one int64 on the device");
  } else {
    start = integer(a[7]);
    if (start < 0 || start > c.N - n)
      value_error("rows [" + std::to_string(start) + ", " + std::to_string(start + n) + ") outside the cache of " + std::to_string(c.N));
  }
  if (n > c.N) value_error("more rows than the cache has");
  if (n == 0) Py_RETURN_NONE;
  k = rows_view(k);
  v = rows_view(v);
  int32_t* const e = status_word(err, c.k);
  check(unlocked([&] {
          const c10::DeviceGuard on(c.k.device());
          return ckv_quantize_rows(ptr(c.k), ptr(c.v), ptr(c.ks), ptr(c.vs), ptr(k), step(k, 1, n * c.D),
                                   step(k, 2, c.D), ptr(v), step(v, 1, n * c.D), step(v, 2, c.D), start, (const int64_t*)ptr(start_dev), int32(n), int32(c.N),
                                   int32(c.H), int32(c.D), int32(c.block), code, e, stream_of(c.k));
        }),
        "ckv_quantize_rows");
  Py_RETURN_NONE;
  CKV_PY_END
}

// What attention calls take of their queries: (1, Hq, n, D) bf16, contiguous rows on 16-byte boundaries, int64 positions.
void query_args(Tensor& q, Tensor& pos, int64_t D, int64_t Hkv) {
  need_dims(q, 4, "q");
  if (q.scalar_type() != at::kBFloat16) type_error("q must be bf16");
  if (q.size(0) != 1 || q.size(3) != D) value_error("q " + shape_of(q) + " must be (1, Hq, n, D) and match the cache's head_dim");
  if (Hkv <= 0 || q.size(1) <= 0 || q.size(1) % Hkv) value_error("the query heads must be a multiple of the KV heads");
  q = rows_view(q);
  if (pos.scalar_type() != at::kLong || pos.numel() != q.size(2)) value_error("positions must be int64 (n,)");
  pos = pos.contiguous();
  if (q.size(2) > INT32_MAX || q.size(1) > INT32_MAX) value_error("too many query rows");
}
// attention_quantized(q, k codes, v codes, k scales, v scales, block, positions, scale, err, out, split)
PyObject* attention_quantized(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  CKV_PY_BEGIN
  need_args(n_args, 11);
  Tensor q = tensor(a[0]), pos = tensor(a[6]);
  const CodedCache c = coded_cache(a + 1);
  const Tensor err = optional_tensor(a[8]);
  Tensor out = optional_tensor(a[9]);
  same_device(q, c.k, c.v, c.ks, c.vs, pos);
  query_args(q, pos, c.D, c.H);
  const int64_t Hq = q.size(1), n = q.size(2);
  if (!out.defined()) {
    out = new_tensor({1, n, Hq, c.D}, q.scalar_type(), q);
  } else {
    same_device(q, out);
    if (out.sizes() != at::IntArrayRef({1, n, Hq, c.D}) || !out.is_contiguous() || out.scalar_type() != q.scalar_type())
      value_error("out must be contiguous (1, n, Hq, D) bf16");
  }
  const double scale = a[7] == Py_None ? 1.0 / std::sqrt((double)c.D) : real(a[7]);
  const int split = PyObject_IsTrue(a[10]);
  if (split < 0) throw python_error();
  const int64_t ws_bytes = split ? ckv_attention_quantized_workspace_bytes(int32(n), int32(c.N), int32(Hq), int32(c.H), int32(c.D)) : 0;
  Tensor ws;
  if (ws_bytes > 0) ws = new_tensor({(ws_bytes + 3) / 4}, at::kFloat, q);
  int32_t* const e = status_word(err, q);
  check(unlocked([&] {
          const c10::DeviceGuard on(q.device());
          return ckv_attention_quantized(ptr(out), ptr(q), step(q, 1, n * c.D), step(q, 2, c.D), ptr(c.k), ptr(c.v), ptr(c.ks),
                                         ptr(c.vs), (const int64_t*)ptr(pos), int32(n), int32(c.N), int32(Hq), int32(c.H),
                                         int32(c.D), int32(c.block), scale, ptr(ws), ws_bytes, e, stream_of(q));
        }),
        "ckv_attention_quantized");
  return THPVariable_Wrap(out);
  CKV_PY_END
}

// attention_weights(q, K, positions, scale, prior, out, err)
PyObject* attention_weights(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  CKV_PY_BEGIN
  need_args(n_args, 7);
  Tensor q = tensor(a[0]), pos = tensor(a[2]);
  const Tensor& K = tensor(a[1]);
  const Tensor prior = optional_tensor(a[4]), err = optional_tensor(a[6]);
  Tensor out = optional_tensor(a[5]);
  same_device(q, K, pos);
  need_dims(K, 4, "K");
  if (K.scalar_type() != at::kBFloat16) type_error("K must be bf16");
  if (K.size(0) != 1) value_error("K must be (1, Hkv, N, D)");
  const int64_t H = K.size(1), N = K.size(2), D = K.size(3);
  if (N > INT32_MAX) value_error("K has at most 2^31 - 1 rows");
  query_args(q, pos, D, H);
  const int64_t hs = head_stride(K, "K"), Hq = q.size(1), n = q.size(2);
  auto fits = [&](const Tensor& t, const char* what) {
    same_device(q, t);
    if (t.sizes() != at::IntArrayRef({1, H, N}) || !t.is_contiguous() || t.scalar_type() != at::kFloat)
      value_error(std::string(what) + " must be contiguous (1, Hkv, N) float32");
  };
  if (prior.defined()) fits(prior, "prior");
  if (!out.defined()) out = new_tensor({1, H, N}, at::kFloat, q);
  else fits(out, "out");
  const double scale = a[3] == Py_None ? 1.0 / std::sqrt((double)D) : real(a[3]);
  const int64_t ws_bytes = ckv_attention_weights_workspace_bytes(int32(n), int32(N), int32(Hq), int32(H), int32(D));
  Tensor ws;
  if (ws_bytes > 0) ws = new_tensor({(ws_bytes + 3) / 4}, at::kFloat, q);
  int32_t* const e = status_word(err, q);
  check(unlocked([&] {
          const c10::DeviceGuard on(q.device());
          return ckv_attention_weights((float*)ptr(out), (const float*)ptr(prior), ptr(q), step(q, 1, n * D), step(q, 2, D), ptr(K),
                                       hs, (const int64_t*)ptr(pos), int32(n), int32(N), int32(Hq), int32(H), int32(D),
                                       CKV_DTYPE_BF16, scale, ptr(ws), ws_bytes, e, stream_of(q));
        }),
        "ckv_attention_weights");
  return THPVariable_Wrap(out);
  CKV_PY_END
}

// The bytes of a tensor (1, H, ...): `count` heads of `size` each, `step` apart.
struct HeadBytes {
  uintptr_t at;
  int64_t size, step, count;
};
HeadBytes head_bytes(const Tensor& t, int64_t head_stride) {
  const int64_t e = t.element_size(), heads = t.size(1);
  return {(uintptr_t)t.data_ptr(), heads > 0 ? t.numel() / heads * e : 0, head_stride * e, heads};
}
// Whether two caches have a byte in common. Caches whose heads take turns in one buffer have none. Heads ascend, so of two that do
// not meet the lower one meets no later one either.
bool overlap(const HeadBytes& a, const HeadBytes& b) {
  for (int64_t i = 0, j = 0; i < a.count && j < b.count;) {
    const uintptr_t x = a.at + i * a.step, y = b.at + j * b.step;
    if (x < y + b.size && y < x + a.size) return true;
    x < y ? ++i : ++j;
  }
  return false;
}

// evict_rows(K, V, weights, n_keep, n_sink, n_recent, k_out, v_out): (K, V, rows, weights) of the kept rows
PyObject* evict_rows(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  CKV_PY_BEGIN
  need_args(n_args, 8);
  const Tensor &K = tensor(a[0]), &V = tensor(a[1]), &w = tensor(a[2]);
  const int64_t keep = integer(a[3]), sink = integer(a[4]), recent = integer(a[5]);
  Tensor ko = optional_tensor(a[6]), vo = optional_tensor(a[7]);
  same_device(K, V, w);
  need_dims(K, 4, "K");
  const int64_t H = K.size(1), N = K.size(2), D = K.size(3);
  if (K.size(0) != 1 || V.sizes() != K.sizes()) value_error("K/V must be (1, Hkv, N, D) of one shape");
  if (V.scalar_type() != K.scalar_type()) type_error("K and V must share a dtype");
  if (N > INT32_MAX || H <= 0) value_error("K/V have 1 to 2^31 - 1 rows and a head at least");
  const int64_t khs = head_stride(K, "K"), vhs = head_stride(V, "V");
  if (w.sizes() != at::IntArrayRef({1, H, N}) || w.scalar_type() != at::kFloat || (N > 1 && w.stride(2) != 1))
    value_error("weights must be (1, Hkv, N) float32 with contiguous rows");
  const int64_t whs = H > 1 ? w.stride(1) : N;
  if (sink < 0 || recent < 0 || keep < 0 || keep > N || sink > keep || recent > keep - sink)
    value_error("n_sink + n_recent <= n_keep <= N must hold: got " + std::to_string(sink) + " + " + std::to_string(recent) +
                ", " + std::to_string(keep) + ", " + std::to_string(N));
  const int code = dtype_code(K);
  auto to = [&](Tensor& t, const char* what) {
    if (!t.defined()) {
      t = new_tensor({1, H, keep, D}, K.scalar_type(), K);
      return;
    }
    same_device(K, t);
    if (t.sizes() != at::IntArrayRef({1, H, keep, D}) || t.scalar_type() != K.scalar_type())
      value_error(std::string(what) + " must be (1, Hkv, n_keep, D) of K's dtype");
  };
  const bool given = ko.defined() || vo.defined();
  to(ko, "k_out");
  to(vo, "v_out");
  const int64_t kohs = head_stride(ko, "k_out"), vohs = head_stride(vo, "v_out");
  const Tensor rows = new_tensor({1, H, keep}, at::kLong, K), wo = new_tensor({1, H, keep}, at::kFloat, K);
  if (keep > 0) {
    if (given) {
      const HeadBytes kb = head_bytes(K, khs), vb = head_bytes(V, vhs), kob = head_bytes(ko, kohs), vob = head_bytes(vo, vohs);
      const HeadBytes wb = head_bytes(w, whs);  // every workgroup reads all of a head's, others write by then
      if (overlap(kob, kb) || overlap(kob, vb) || overlap(vob, kb) || overlap(vob, vb) || overlap(kob, vob) || overlap(kob, wb) || overlap(vob, wb))
        value_error("k_out and v_out must overlap none of K, V, weights and each other");
    }
    check(unlocked([&] {
            const c10::DeviceGuard on(K.device());
            return ckv_evict_rows(ptr(ko), kohs, ptr(vo), vohs, (int64_t*)ptr(rows), (float*)ptr(wo), ptr(K), khs, ptr(V), vhs,
                                  (const float*)ptr(w), whs, int32(N), int32(keep), int32(sink), int32(recent), int32(H),
                                  int32(D), code, stream_of(K));
          }),
          "ckv_evict_rows");
  }
  return Py_BuildValue("(NNNN)", THPVariable_Wrap(ko), THPVariable_Wrap(vo), THPVariable_Wrap(rows), THPVariable_Wrap(wo));
  CKV_PY_END
}

// The book of a paged cache: table (S, M), lengths (S,) and refs (P,), int32 on one device.
struct PageBook {
  const Tensor &table, &lengths, &refs;
  int64_t S, M, P, T;
  int32_t* at(const Tensor& t) const { return (int32_t*)ptr(t); }
};
PageBook page_book(PyObject* const* a) {
  const Tensor &table = tensor(a[0]), &lengths = tensor(a[1]), &refs = tensor(a[2]);
  const int64_t T = integer(a[3]);
  same_device(table, lengths, refs);
  if (T != 32 && T != 64 && T != 128) value_error("page_tokens must be 32, 64 or 128");
  if (table.scalar_type() != at::kInt || lengths.scalar_type() != at::kInt || refs.scalar_type() != at::kInt)
    type_error("table, lengths and refs must be int32");
  if (table.dim() != 2 || lengths.dim() != 1 || refs.dim() != 1 || table.size(0) != lengths.size(0) || !table.is_contiguous() ||
      !lengths.is_contiguous() || !refs.is_contiguous())
    value_error("table must be (sequences, entries), lengths (sequences,) and refs (pages,), contiguous");
  if (table.numel() == 0 || refs.numel() == 0) value_error("a paged cache has a sequence, an entry and a page at least");
  if (table.size(0) > INT32_MAX || table.size(1) > INT32_MAX || refs.size(0) > INT32_MAX) value_error("too many pages");
  return {table, lengths, refs, table.size(0), table.size(1), refs.size(0), T};
}
// Pools (L, 1, H, P * T, D) of K and V.
struct PagePool {
  const Tensor &k, &v;
  int64_t L, H, D;
};
PagePool page_pool(const PageBook& b, PyObject* ko, PyObject* vo) {
  const Tensor &k = tensor(ko), &v = tensor(vo);
  same_device(b.table, k, v);
  need_dims(k, 5, "a paged cache's k");
  if (v.scalar_type() != k.scalar_type()) type_error("k and v must share a dtype");
  if (k.size(1) != 1 || k.size(3) != b.P * b.T || v.sizes() != k.sizes() || !k.is_contiguous() || !v.is_contiguous() || k.numel() == 0)
    value_error("a paged cache's k and v must be contiguous (layers, 1, Hkv, pages * page_tokens, D)");
  if (k.size(0) > INT32_MAX || k.size(2) > INT32_MAX || k.size(4) > INT32_MAX) value_error("a paged cache's k is too large");
  return {k, v, k.size(0), k.size(2), k.size(4)};
}
// An int32 vector on the book's device.
Tensor int_vector(PyObject* o, const PageBook& b, const char* what) {
  Tensor t = tensor(o);
  same_device(b.table, t);
  if (t.scalar_type() != at::kInt || t.dim() != 1) value_error(std::string(what) + " must be int32 of one dimension");
  if (t.numel() > INT32_MAX) value_error(std::string(what) + " is too long");
  return t.contiguous();
}

// extend_pages(table, lengths, refs, page_tokens, counts, n, err): (positions, rows, starts)
PyObject* extend_pages(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  CKV_PY_BEGIN
  need_args(n_args, 7);
  const PageBook b = page_book(a);
  const Tensor counts = int_vector(a[4], b, "counts"), err = optional_tensor(a[6]);
  int32_t* const e = status_word(err, b.table);
  const int64_t n = integer(a[5]);
  if (counts.numel() != b.S) value_error("counts must be (sequences,)");
  if (n < 0 || n > INT32_MAX) value_error("n must be 0 to 2^31 - 1");
  const Tensor positions = new_tensor({n}, at::kLong, b.table), rows = new_tensor({n}, at::kLong, b.table);
  const Tensor starts = new_tensor({b.S + 1}, at::kInt, b.table);
  check(unlocked([&] {
          const c10::DeviceGuard on(b.table.device());
          return ckv_extend_pages((int64_t*)ptr(positions), (int64_t*)ptr(rows), (int32_t*)ptr(starts), int32(n),
                                  (const int32_t*)ptr(counts), b.at(b.table), b.at(b.lengths), b.at(b.refs), int32(b.S), int32(b.M),
                                  int32(b.P), int32(b.T), e, stream_of(b.table));
        }),
        "ckv_extend_pages");
  return Py_BuildValue("(NNN)", THPVariable_Wrap(positions), THPVariable_Wrap(rows), THPVariable_Wrap(starts));
  CKV_PY_END
}

// fork_pages(table, lengths, refs, page_tokens, k, v, sources, targets, err)
PyObject* fork_pages(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  CKV_PY_BEGIN
  need_args(n_args, 9);
  const PageBook b = page_book(a);
  const PagePool p = page_pool(b, a[4], a[5]);
  const Tensor sources = int_vector(a[6], b, "sources"), targets = int_vector(a[7], b, "targets"), err = optional_tensor(a[8]);
  int32_t* const e = status_word(err, b.table);
  const int64_t n = sources.numel();
  if (targets.numel() != n) value_error("sources and targets must be of one length");
  const int code = dtype_code(p.k);
  const int64_t ws_bytes = ckv_fork_pages_workspace_bytes(int32(n));
  Tensor ws;
  if (ws_bytes > 0) ws = new_tensor({ws_bytes / 4}, at::kInt, b.table);
  check(unlocked([&] {
          const c10::DeviceGuard on(b.table.device());
          return ckv_fork_pages(ptr(p.k), ptr(p.v), p.k.stride(0), p.k.stride(2), int32(p.L), int32(p.H), int32(p.D), code,
                                (const int32_t*)ptr(sources), (const int32_t*)ptr(targets), int32(n), b.at(b.table), b.at(b.lengths),
                                b.at(b.refs), int32(b.S), int32(b.M), int32(b.P), int32(b.T), ptr(ws), ws_bytes, e, stream_of(b.table));
        }),
        "ckv_fork_pages");
  Py_RETURN_NONE;
  CKV_PY_END
}

// free_pages(table, lengths, refs, page_tokens, sequences, keep, err)
PyObject* free_pages(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  CKV_PY_BEGIN
  need_args(n_args, 7);
  const PageBook b = page_book(a);
  const Tensor sequences = int_vector(a[4], b, "sequences"), err = optional_tensor(a[6]);
  int32_t* const e = status_word(err, b.table);
  const int64_t n = sequences.numel();
  Tensor keep, ws;
  if (a[5] != Py_None) {
    keep = int_vector(a[5], b, "keep");
    if (keep.numel() != n) value_error("sequences and keep must be of one length");
    ws = new_tensor({n}, at::kInt, b.table);
  }
  check(unlocked([&] {
          const c10::DeviceGuard on(b.table.device());
          return ckv_free_pages((const int32_t*)ptr(sequences), (const int32_t*)ptr(keep), int32(n), b.at(b.table), b.at(b.lengths),
                                b.at(b.refs), int32(b.S), int32(b.M), int32(b.P), int32(b.T), ptr(ws), n * 4, e, stream_of(b.table));
        }),
        "ckv_free_pages");
  Py_RETURN_NONE;
  CKV_PY_END
}

// compact_pages(table, lengths, refs, page_tokens, k, v, err): used
PyObject* compact_pages(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  CKV_PY_BEGIN
  need_args(n_args, 7);
  const PageBook b = page_book(a);
  const PagePool p = page_pool(b, a[4], a[5]);
  const Tensor err = optional_tensor(a[6]);
  int32_t* const e = status_word(err, b.table);
  const int code = dtype_code(p.k);
  const int64_t ws_bytes = ckv_compact_pages_workspace_bytes(int32(b.P));
  const Tensor ws = new_tensor({ws_bytes / 4}, at::kInt, b.table), used = new_tensor({1}, at::kInt, b.table);
  check(unlocked([&] {
          const c10::DeviceGuard on(b.table.device());
          return ckv_compact_pages(ptr(p.k), ptr(p.v), p.k.stride(0), p.k.stride(2), int32(p.L), int32(p.H), int32(p.D), code,
                                   (int32_t*)ptr(used), b.at(b.table), b.at(b.lengths), b.at(b.refs), int32(b.S), int32(b.M), int32(b.P),
                                   int32(b.T), ptr(ws), ws_bytes, e, stream_of(b.table));
        }),
        "ckv_compact_pages");
  return THPVariable_Wrap(used);
  CKV_PY_END
}

// Whether `out`, contiguous, and t have a byte in common: of t, what dimensions d and behind it have from address `at` on.
bool meets(uintptr_t lo, uintptr_t hi, const Tensor& t, int64_t d, uintptr_t at) {
  const int64_t e = t.element_size();
  int64_t span = e, held = e;
  for (int64_t i = d; i < t.dim(); ++i) {
    if (t.stride(i) == 0) continue;  // the same bytes again
    span += (t.size(i) - 1) * t.stride(i) * e;
    held *= t.size(i);
  }
  if (at >= hi || at + (uintptr_t)span <= lo) return false;
  if (held >= span || at >= lo) return true;  // no gaps, or its first element
  const int64_t n = t.stride(d) == 0 ? 1 : t.size(d);
  for (int64_t i = 0; i < n; ++i)
    if (meets(lo, hi, t, d + 1, at + (uintptr_t)(i * t.stride(d) * e))) return true;
  return false;
}
bool meets(const Tensor& out, const Tensor& t) {
  if (!t.defined() || t.numel() == 0 || out.numel() == 0) return false;
  const uintptr_t lo = (uintptr_t)out.data_ptr();
  return meets(lo, lo + (uintptr_t)(out.numel() * out.element_size()), t, 0, (uintptr_t)t.data_ptr());
}

// attention_paged(q, table, lengths, refs, page_tokens, k, v, layer, starts, most, longest, total, scale, err, out, split)
PyObject* attention_paged(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  CKV_PY_BEGIN
  need_args(n_args, 16);
  Tensor q = tensor(a[0]);
  const PageBook b = page_book(a + 1);
  const PagePool p = page_pool(b, a[5], a[6]);
  const int64_t layer = integer(a[7]), most = a[9] == Py_None ? 0 : integer(a[9]), longest = a[10] == Py_None ? 0 : integer(a[10]),
                total = a[11] == Py_None ? 0 : integer(a[11]);
  const Tensor starts = int_vector(a[8], b, "starts"), err = optional_tensor(a[13]);
  int32_t* const e = status_word(err, q);
  Tensor out = optional_tensor(a[14]);
  same_device(q, p.k);
  need_dims(q, 4, "q");
  if (q.scalar_type() != at::kBFloat16 || p.k.scalar_type() != at::kBFloat16) type_error("attention_paged runs on bf16 q and cache");
  const int64_t Hq = q.size(1), n = q.size(2);
  if (q.size(0) != 1 || q.size(3) != p.D) value_error("q " + shape_of(q) + " must be (1, Hq, n, D) and match the cache's head_dim");
  if (Hq <= 0 || Hq % p.H) value_error("the query heads must be a multiple of the KV heads");
  if (n > INT32_MAX || Hq > INT32_MAX) value_error("too many query rows");
  if (layer < 0 || layer >= p.L) value_error("layer " + std::to_string(layer) + " of a cache of " + std::to_string(p.L));
  if (starts.numel() != b.S + 1) value_error("starts must be (sequences + 1,)");
  if (a[9] != Py_None && (most < 1 || most > INT32_MAX)) value_error("most must be 1 to 2^31 - 1");
  if (a[10] != Py_None && (longest < 1 || longest > INT32_MAX)) value_error("longest must be 1 to 2^31 - 1");
  if (a[11] != Py_None && total < 1) value_error("total must be 1 or more");
  q = rows_view(q);
  if (!out.defined()) {
    out = new_tensor({1, n, Hq, p.D}, at::kBFloat16, q);
  } else {
    same_device(q, out);
    if (out.sizes() != at::IntArrayRef({1, n, Hq, p.D}) || !out.is_contiguous() || out.scalar_type() != at::kBFloat16)
      value_error("out must be contiguous (1, n, Hq, D) bf16");
    // token-major queries may be written over: the workgroup that writes a row has read it, and no other reads it
    const bool in_place = out.data_ptr() == q.data_ptr() && step(q, 1, p.D) == p.D && step(q, 2, Hq * p.D) == Hq * p.D;
    if (!in_place && meets(out, q)) value_error("out overlaps q without being it");
    for (const Tensor* t : {&p.k, &p.v, &b.table, &b.lengths, &starts})
      if (meets(out, *t)) value_error("out overlaps the cache or starts");
  }
  const double scale = a[12] == Py_None ? 1.0 / std::sqrt((double)p.D) : real(a[12]);
  const int split = PyObject_IsTrue(a[15]);
  if (split < 0) throw python_error();
  const int64_t ws_bytes =
      split ? ckv_attention_paged_workspace_bytes(int32(n), int32(b.S), int32(most), int32(longest), total, int32(b.M), int32(b.T),
                                                  int32(Hq), int32(p.H), int32(p.D))
            : 0;
  Tensor ws;
  if (ws_bytes > 0) ws = new_tensor({(ws_bytes + 3) / 4}, at::kFloat, q);
  check(unlocked([&] {
          const c10::DeviceGuard on(q.device());
          const int64_t at = layer * p.k.stride(0) * 2;
          return ckv_attention_paged(ptr(out), ptr(q), step(q, 1, n * p.D), step(q, 2, p.D), (const char*)ptr(p.k) + at,
                                     (const char*)ptr(p.v) + at, p.k.stride(2), b.at(b.table), b.at(b.lengths), (const int32_t*)ptr(starts),
                                     int32(n), int32(most), int32(longest), total, int32(b.S), int32(b.M), int32(b.P), int32(b.T),
                                     int32(Hq), int32(p.H), int32(p.D), CKV_DTYPE_BF16, scale, ptr(ws), ws_bytes, e, stream_of(q));
        }),
        "ckv_attention_paged");
  return THPVariable_Wrap(out);
  CKV_PY_END
}

// What adjust_logits and next_tokens share: (logits, prompt, generated, repetition, frequency, presence, bias, allowed).
struct LogitArgs {
  const Tensor& logits;
  int64_t rows, vocab, row_stride;
  int code;
  Tensor prompt, generated, repetition, frequency, presence, bias, allowed;
  float repetition_all = 1.f, frequency_all = 0.f, presence_all = 0.f;
};
LogitArgs logit_args(PyObject* const* a) {
  const Tensor& x = tensor(a[0]);
  same_device(x);
  need_dims(x, 2, "logits");
  if (x.scalar_type() != at::kBFloat16 && x.scalar_type() != at::kFloat) type_error("logits must be bfloat16 or float32");
  LogitArgs r{x, x.size(0), x.size(1), 0, dtype_code(x), {}, {}, {}, {}, {}, {}, {}};
  if (r.vocab < 1 || r.vocab > INT32_MAX || r.rows > INT32_MAX) value_error("logits must be (rows, vocab)");
  if (r.vocab > 1 && x.stride(1) != 1) value_error("logits must have contiguous rows");
  r.row_stride = step(x, 0, r.vocab);
  if (r.row_stride < r.vocab) value_error("logits rows overlap");
  auto tokens = [&](PyObject* o, const char* what) {
    Tensor t = optional_tensor(o);
    if (!t.defined()) return t;
    same_device(x, t);
    if (t.scalar_type() != at::kLong || t.dim() != 2 || t.size(0) != r.rows || t.size(1) > INT32_MAX)
      value_error(std::string(what) + " must be int64 (rows, tokens)");
    if (t.size(1) > 1 && t.stride(1) != 1) t = t.contiguous();
    return t;
  };
  r.prompt = tokens(a[1], "prompt");
  r.generated = tokens(a[2], "generated");
  auto value = [&](PyObject* o, float& all, const char* what) {
    Tensor t;
    if (!THPVariable_Check(o)) {
      all = (float)real(o);
      return t;
    }
    t = tensor(o);
    same_device(x, t);
    if (t.scalar_type() != at::kFloat || t.dim() != 1 || t.size(0) != r.rows)
      value_error(std::string(what) + " must be a number or float32 (rows,)");
    return t.contiguous();
  };
  r.repetition = value(a[3], r.repetition_all, "repetition");
  r.frequency = value(a[4], r.frequency_all, "frequency");
  r.presence = value(a[5], r.presence_all, "presence");
  if (!(r.repetition_all > 0.f)) value_error("repetition must be above 0");
  auto per_row = [&](PyObject* o, at::ScalarType type, int64_t width, const char* what) {
    Tensor t = optional_tensor(o);
    if (!t.defined()) return t;
    same_device(x, t);
    if (t.dim() == 1) t = t.unsqueeze(0);
    if (t.scalar_type() != type || t.dim() != 2 || (t.size(0) != 1 && t.size(0) != r.rows) || t.size(1) != width)
      value_error(std::string(what) + " must be of " + std::to_string(width) + " for each row or for all, " + c10::toString(type));
    if (width > 1 && t.stride(1) != 1) t = t.contiguous();
    return t;
  };
  r.bias = per_row(a[6], at::kFloat, r.vocab, "bias");
  r.allowed = per_row(a[7], at::kInt, (r.vocab + 31) / 32, "allowed");
  return r;
}
int64_t rows_apart(const Tensor& t) { return t.defined() && t.size(0) > 1 ? t.stride(0) : 0; }
#define CKV_LOGIT_ARGS(r)                                                                                                          \
  ptr(r.logits), r.row_stride, int32(r.rows), int32(r.vocab), r.code, (const int64_t*)ptr(r.prompt), rows_apart(r.prompt),          \
      int32(r.prompt.defined() ? r.prompt.size(1) : 0), (const int64_t*)ptr(r.generated), rows_apart(r.generated),                  \
      int32(r.generated.defined() ? r.generated.size(1) : 0), (const float*)ptr(r.repetition), r.repetition_all,                    \
      (const float*)ptr(r.frequency), r.frequency_all, (const float*)ptr(r.presence), r.presence_all, (const float*)ptr(r.bias),    \
      rows_apart(r.bias), (const int32_t*)ptr(r.allowed), rows_apart(r.allowed)

// adjust_logits(logits, prompt, generated, repetition, frequency, presence, bias, allowed, out)
PyObject* adjust_logits(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  CKV_PY_BEGIN
  need_args(n_args, 9);
  const LogitArgs r = logit_args(a);
  Tensor out = optional_tensor(a[8]);
  if (!out.defined()) {
    out = new_tensor({r.rows, r.vocab}, at::kFloat, r.logits);
  } else {
    same_device(r.logits, out);
    if (out.sizes() != r.logits.sizes() || !out.is_contiguous() || out.scalar_type() != at::kFloat)
      value_error("out must be contiguous (rows, vocab) float32");
    // float32 logits, or a bias of each row, may be where the result goes: a thread reads what it writes
    auto there = [&](const Tensor& t) {
      return t.data_ptr() == out.data_ptr() && t.scalar_type() == at::kFloat && t.size(0) == r.rows && step(t, 0, r.vocab) == r.vocab;
    };
    if (!there(r.logits) && meets(out, r.logits)) value_error("out overlaps the logits without being them");
    if (r.bias.defined() && !there(r.bias) && meets(out, r.bias)) value_error("out overlaps the bias without being it");
    for (const Tensor* t : {&r.prompt, &r.generated, &r.repetition, &r.frequency, &r.presence, &r.allowed})
      if (meets(out, *t)) value_error("out overlaps what the logits are adjusted by");
  }
  check(unlocked([&] {
          const c10::DeviceGuard on(r.logits.device());
          return ckv_adjust_logits((float*)ptr(out), CKV_LOGIT_ARGS(r), stream_of(r.logits));
        }),
        "ckv_adjust_logits");
  return THPVariable_Wrap(out);
  CKV_PY_END
}

// next_tokens(logits, prompt, generated, repetition, frequency, presence, bias, allowed, err, out)
PyObject* next_tokens(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  CKV_PY_BEGIN
  need_args(n_args, 10);
  const LogitArgs r = logit_args(a);
  const Tensor err = optional_tensor(a[8]);
  int32_t* const e = status_word(err, r.logits);
  const int64_t ws_bytes = ckv_next_tokens_workspace_bytes(int32(r.rows), int32(r.vocab));
  Tensor out = optional_tensor(a[9]);
  if (!out.defined()) {
    out = new_tensor({r.rows}, at::kLong, r.logits);
  } else {
    same_device(r.logits, out);
    if (out.sizes() != at::IntArrayRef({r.rows}) || !out.is_contiguous() || out.scalar_type() != at::kLong)
      value_error("out must be contiguous (rows,) int64");
    // with a workspace a second launch writes the tokens; without it a row's workgroup does, when it has read all of its row
    if (ws_bytes == 0 && r.rows > 1)
      for (const Tensor* t : {&r.logits, &r.prompt, &r.generated, &r.repetition, &r.frequency, &r.presence, &r.bias, &r.allowed})
        if (meets(out, *t)) value_error("out overlaps what the tokens are chosen from");
  }
  Tensor ws;
  if (ws_bytes > 0) ws = new_tensor({ws_bytes / 8}, at::kLong, r.logits);
  check(unlocked([&] {
          const c10::DeviceGuard on(r.logits.device());
          return ckv_next_tokens((int64_t*)ptr(out), CKV_LOGIT_ARGS(r), ptr(ws), ws_bytes, e, stream_of(r.logits));
        }),
        "ckv_next_tokens");
  return THPVariable_Wrap(out);
  CKV_PY_END
}

PyMethodDef kMethods[] = {
    {"extend_pages", (PyCFunction)(void (*)(void))extend_pages, METH_FASTCALL, nullptr},
    {"fork_pages", (PyCFunction)(void (*)(void))fork_pages, METH_FASTCALL, nullptr},
    {"free_pages", (PyCFunction)(void (*)(void))free_pages, METH_FASTCALL, nullptr},
    {"compact_pages", (PyCFunction)(void (*)(void))compact_pages, METH_FASTCALL, nullptr},
    {"attention_paged", (PyCFunction)(void (*)(void))attention_paged, METH_FASTCALL, nullptr},
    {"adjust_logits", (PyCFunction)(void (*)(void))adjust_logits, METH_FASTCALL, nullptr},
    {"next_tokens", (PyCFunction)(void (*)(void))next_tokens, METH_FASTCALL, nullptr},
    {"quantize_rows", (PyCFunction)(void (*)(void))quantize_rows, METH_FASTCALL, nullptr},
    {"attention_quantized", (PyCFunction)(void (*)(void))attention_quantized, METH_FASTCALL, nullptr},
    {"attention_weights", (PyCFunction)(void (*)(void))attention_weights, METH_FASTCALL, nullptr},
    {"evict_rows", (PyCFunction)(void (*)(void))evict_rows, METH_FASTCALL, nullptr},
    {"attention_active", (PyCFunction)(void (*)(void))attention_active, METH_FASTCALL, nullptr},
    {"rope_qkv", (PyCFunction)(void (*)(void))rope_qkv, METH_FASTCALL, nullptr},
    {"add_rmsnorm", (PyCFunction)(void (*)(void))add_rmsnorm, METH_FASTCALL, nullptr},
    {"silu_mul", (PyCFunction)(void (*)(void))silu_mul, METH_FASTCALL, nullptr},
    {"linear", (PyCFunction)(void (*)(void))linear, METH_FASTCALL, nullptr},
    {"layer1_repair_gather", (PyCFunction)(void (*)(void))layer1_repair_gather, METH_FASTCALL, nullptr},
    {"extract_chunks", (PyCFunction)(void (*)(void))extract_chunks, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops() { return PyModule_Create(&kModule); }
