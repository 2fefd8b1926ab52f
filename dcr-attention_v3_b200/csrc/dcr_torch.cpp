// dcr_torch.cpp — the paged serving operators' binding to torch tensors (dcr_b200_torch.so).
//
// These operators run once per layer and decode step on calls of 5 to 20 us, where checking
// arguments and marshalling them through ctypes cost as much again: with the checks in Python a
// call took 17 to 30 us of host time, from here it took 11 to 13 (now 6 to 12, outputs allocated).
// So their argument checks, output
// allocations and the call of the C ABI live here; kernel/cuda/paged.py and logits.py give them
// their names, keywords and documentation.
//
// Every function takes its arguments by position, checks them (AssertionError for shapes, dtypes,
// layouts and values, RuntimeError for tensors that are not on a CUDA device), runs on the current
// stream of the tensors' device, and returns its result, or the dcr_status as an int where the C
// ABI refused. No exception leaves a function except as a Python error.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>

#include "dcr_b200.h"
#include "dcr_tables.h"

namespace {

struct Refused {};  // a Python error is set

[[noreturn]] void refuse(const std::string& msg) {
  PyErr_SetString(PyExc_AssertionError, msg.c_str());
  throw Refused{};
}

std::string dims(at::IntArrayRef s) {
  std::string r = "[";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + "]";
}

const char* type_name(at::ScalarType t) { return c10::toString(t); }

const at::Tensor& cuda_tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a tensor", name);
    throw Refused{};
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda()) {
    PyErr_SetString(PyExc_RuntimeError, "libdcr_b200 requires CUDA tensors (no CPU fallback).");
    throw Refused{};
  }
  return t;
}

int64_t integer(PyObject* o, const char* name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(std::string(name) + " must be an integer");
  }
  return v;
}

int dtype_code(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return DCR_DTYPE_BF16;
    case at::kHalf: return DCR_DTYPE_F16;
    case at::kFloat: return DCR_DTYPE_F32;
    default: refuse(std::string(name) + " must be bfloat16, float16 or float32, got " + type_name(t.scalar_type()));
  }
}

// A contiguous 1-D tensor of n elements.
void* vector_of(PyObject* o, const char* name, at::ScalarType type, int64_t n, int device) {
  const at::Tensor& t = cuda_tensor(o, name);
  if (!(t.dim() == 1 && t.size(0) == n && t.scalar_type() == type && t.get_device() == device &&
        t.is_contiguous()))
    refuse(std::string(name) + " must be a contiguous " + type_name(type) + " [" + std::to_string(n) +
           "] on cuda:" + std::to_string(device));
  return t.data_ptr();
}

void* optional_vector(PyObject* o, const char* name, at::ScalarType type, int64_t n, int device) {
  return o == Py_None ? nullptr : vector_of(o, name, type, n, device);
}

struct Pool {
  const at::Tensor* k;
  const at::Tensor* v;
  const at::Tensor* table;
  int dtype, device;
  int64_t pages, H_kv, page_size, D, max_pages, sequences, table_stride, slots;
};

Pool pool_of(PyObject* k_o, PyObject* v_o, PyObject* table_o) {
  Pool p;
  p.k = &cuda_tensor(k_o, "k_pages");
  p.v = &cuda_tensor(v_o, "v_pages");
  p.table = &cuda_tensor(table_o, "page_table");
  const at::Tensor &k = *p.k, &v = *p.v, &t = *p.table;
  p.dtype = dtype_code(k, "k_pages");
  p.device = k.get_device();
  if (!(k.dim() == 4 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() &&
        v.get_device() == p.device))
    refuse("k_pages and v_pages must be [pages, H_kv, page_size, D] of one shape, dtype and device");
  p.pages = k.size(0);
  p.H_kv = k.size(1);
  p.page_size = k.size(2);
  p.D = k.size(3);
  if (p.D != 64 && p.D != 128) refuse("head dim must be 64 or 128, got " + std::to_string(p.D));
  if (k.numel() == 0) refuse("k_pages must not be empty, got " + dims(k.sizes()));
  if (k.stride(3) != 1 || v.stride(3) != 1) refuse("page rows must be contiguous");
  if (!(t.scalar_type() == at::kInt && t.dim() == 2 && t.size(1) > 0 && t.get_device() == p.device &&
        t.stride(1) == 1))
    refuse("page_table must be [B, max_pages] int32 with contiguous rows, on the pool's device");
  p.sequences = t.size(0);
  p.max_pages = t.size(1);
  p.table_stride = p.sequences > 1 ? t.stride(0) : p.max_pages;
  p.slots = p.max_pages * p.page_size;
  if (p.pages > INT32_MAX || p.slots > INT32_MAX) refuse("pool or page_table too large");
  return p;
}

struct Table {
  void* data = nullptr;
  int64_t sb = 0, sh = 0;
};

// A per-slot table [B, H_kv, >= slots] with contiguous rows, or None; one that is written has no
// two rows that share elements (an expanded tensor, say).
Table slot_table(PyObject* o, const char* name, at::ScalarType type, const Pool& p, int64_t slots,
                 bool written = true) {
  Table r;
  if (o == Py_None) return r;
  const at::Tensor& t = cuda_tensor(o, name);
  if (!(t.scalar_type() == type && t.get_device() == p.device && t.dim() == 3 &&
        t.size(0) == p.sequences && t.size(1) == p.H_kv && t.size(2) >= slots && t.stride(2) == 1))
    refuse(std::string(name) + " must be " + type_name(type) + " [" + std::to_string(p.sequences) + ", " +
           std::to_string(p.H_kv) + ", >= " + std::to_string(slots) + "] with contiguous rows on cuda:" +
           std::to_string(p.device));
  r.data = t.data_ptr();
  r.sb = t.stride(0);
  r.sh = t.stride(1);
  if (written && !dcr::rows_apart(p.sequences, p.H_kv, slots, r.sb, r.sh))
    refuse(std::string(name) + " must not have rows that share elements");
  return r;
}

struct Rows {
  const void* data;
  int64_t st, sh;
};

// Rows [tokens, heads, D] of the pool's dtype with contiguous elements.
Rows rows_of(PyObject* o, const char* name, const Pool& p, int64_t tokens, int64_t heads) {
  const at::Tensor& t = cuda_tensor(o, name);
  if (!(t.dim() == 3 && t.size(0) == tokens && t.size(1) == heads && t.size(2) == p.D &&
        t.scalar_type() == p.k->scalar_type() && t.get_device() == p.device && t.stride(2) == 1))
    refuse(std::string(name) + " must be " + dims({tokens, heads, p.D}) + " " +
           type_name(p.k->scalar_type()) + " with contiguous rows on cuda:" + std::to_string(p.device));
  return {t.data_ptr(), tokens > 1 ? t.stride(0) : 0, heads > 1 ? t.stride(1) : 0};
}

// The [tokens, heads] of a query tensor.
std::pair<int64_t, int64_t> query_shape(PyObject* o, const Pool& p) {
  const at::Tensor& q = cuda_tensor(o, "q");
  if (q.dim() != 3) refuse("q must be [tokens, H, D]");
  if (q.size(1) <= 0 || q.size(1) % p.H_kv != 0)
    refuse("H=" + std::to_string(q.size(1)) + " must be a positive multiple of H_kv=" + std::to_string(p.H_kv));
  if (q.size(0) > INT32_MAX || q.size(1) > INT32_MAX) refuse("q too large");
  return {q.size(0), q.size(1)};
}

at::Tensor output(PyObject* o, at::IntArrayRef shape, const at::TensorOptions& opt) {
  if (o == Py_None) return at::empty(shape, opt);
  const at::Tensor& t = cuda_tensor(o, "out");
  if (!(t.sizes() == shape && t.scalar_type() == opt.dtype().toScalarType() &&
        t.device() == opt.device() && t.is_contiguous()))
    refuse(std::string("out must be a contiguous ") + type_name(opt.dtype().toScalarType()) + " " + dims(shape));
  return t;
}

// Refuses an output that reaches into the rows [tokens, heads, D] it is computed from.
void check_apart(PyObject* out, const at::Tensor& o, const Rows& q, const Pool& p, int64_t tokens, int64_t heads) {
  if (out != Py_None &&
      dcr::rows_meet(q.data, q.st, q.sh, o.data_ptr(), tokens, heads, p.D, o.element_size()))
    refuse("out must be q itself (contiguous) or share no memory with it");
}

// The caller's workspace (checked) or a fresh one from torch's allocator.
at::Tensor scratch(PyObject* o, size_t bytes, int device) {
  if (o == Py_None)
    return at::empty({static_cast<int64_t>(bytes)},
                     at::TensorOptions().dtype(at::kByte).device(at::kCUDA, device));
  const at::Tensor& t = cuda_tensor(o, "workspace");
  if (!(t.get_device() == device && t.scalar_type() == at::kByte && t.is_contiguous() &&
        t.numel() >= static_cast<int64_t>(bytes)))
    refuse("workspace must be a contiguous uint8 CUDA tensor of >= " + std::to_string(bytes) +
           " bytes on cuda:" + std::to_string(device));
  return t;
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

template <typename F>
PyObject* guarded(PyObject* const* a, Py_ssize_t n, Py_ssize_t want, F&& f) {
  if (n != want) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
    return nullptr;
  }
  try {
    return f();
  } catch (const Refused&) {
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    return nullptr;
  }
}

// (q, k_pages, v_pages, page_table, lengths, scale, window, weights, return_lse, out, workspace)
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(a, n, 11, [&]() -> PyObject* {
    const Pool p = pool_of(a[1], a[2], a[3]);
    const auto [B, H] = query_shape(a[0], p);
    const Rows q = rows_of(a[0], "q", p, B, H);
    if (p.sequences != B) refuse("page_table must have " + std::to_string(B) + " rows");
    const void* lengths = vector_of(a[4], "lengths", at::kInt, B, p.device);
    double scale = 1.0 / std::sqrt(static_cast<double>(p.D));
    if (a[5] != Py_None) {
      scale = PyFloat_AsDouble(a[5]);
      if (scale == -1.0 && PyErr_Occurred()) throw Refused{};
    }
    const int64_t window = integer(a[6], "window");
    if (window < 0 || window > INT32_MAX) refuse("window must be >= 0");
    const Table w = slot_table(a[7], "weights", at::kFloat, p, p.slots);
    const int truth = PyObject_IsTrue(a[8]);
    if (truth < 0) throw Refused{};
    const bool want_lse = truth != 0;
    const c10::cuda::OptionalCUDAGuard guard(p.k->device());
    const at::Tensor o = output(a[9], {B, H, p.D}, p.k->options());
    check_apart(a[9], o, q, p, B, H);
    at::Tensor lse;
    if (want_lse) lse = at::empty({B, H}, p.k->options().dtype(at::kFloat));
    if (B > 0) {
      const size_t bytes = dcr_paged_workspace_bytes(
          static_cast<int>(B), static_cast<int>(H), static_cast<int>(p.H_kv), static_cast<int>(p.D),
          static_cast<int>(p.slots), w.data != nullptr);
      const at::Tensor ws = scratch(a[10], bytes, p.device);
      const int st = dcr_paged_attend(
          q.data, q.st, q.sh, p.k->data_ptr(), p.v->data_ptr(), p.dtype, p.k->stride(0),
          p.k->stride(1), p.k->stride(2), p.v->stride(0), p.v->stride(1), p.v->stride(2),
          static_cast<int>(p.pages), static_cast<int>(p.page_size),
          static_cast<const int32_t*>(p.table->data_ptr()), p.table_stride,
          static_cast<int>(p.max_pages), static_cast<const int32_t*>(lengths), static_cast<int>(B),
          static_cast<int>(H), static_cast<int>(p.H_kv), static_cast<int>(p.D),
          static_cast<float>(scale), static_cast<int>(window), o.data_ptr(),
          want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr, static_cast<float*>(w.data),
          w.sb, w.sh, ws.data_ptr(), static_cast<size_t>(ws.numel()), stream_of(p.device));
      if (st != DCR_OK) return PyLong_FromLong(st);
    }
    if (!want_lse) return THPVariable_Wrap(o);
    PyObject* r = PyTuple_New(2);
    if (r == nullptr) return nullptr;
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(o));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(lse));
    return r;
  });
}

// (q, k, v, cos, sin, positions, k_pages, v_pages, page_table, slots, seq, q_weight, k_weight,
//  eps, weights, pos, out)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(a, n, 17, [&]() -> PyObject* {
    const Pool p = pool_of(a[6], a[7], a[8]);
    const auto [T, H] = query_shape(a[0], p);
    const Rows q = rows_of(a[0], "q", p, T, H);
    const Rows k = rows_of(a[1], "k", p, T, p.H_kv);
    const Rows v = rows_of(a[2], "v", p, T, p.H_kv);
    const at::Tensor &cos = cuda_tensor(a[3], "cos"), &sin = cuda_tensor(a[4], "sin");
    const at::ScalarType type = p.k->scalar_type(), table_type = cos.scalar_type();
    if (!(cos.dim() == 2 && sin.sizes() == cos.sizes() && cos.size(1) == p.D && cos.size(0) > 0 &&
          cos.size(0) <= INT32_MAX && sin.scalar_type() == table_type &&
          (table_type == type || table_type == at::kFloat) && cos.get_device() == p.device &&
          sin.get_device() == p.device && cos.is_contiguous() && sin.is_contiguous()))
      refuse("cos and sin must be contiguous [n, " + std::to_string(p.D) + "] tables of " +
             type_name(type) + " or float32 on cuda:" + std::to_string(p.device));
    const void* positions = vector_of(a[5], "positions", at::kInt, T, p.device);
    const void* slots = vector_of(a[9], "slots", at::kInt, T, p.device);
    const void* seq = optional_vector(a[10], "seq", at::kInt, T, p.device);
    if (seq == nullptr && T > p.sequences)
      refuse(std::to_string(T) + " tokens without seq need as many sequences, got " + std::to_string(p.sequences));
    const void* qw = optional_vector(a[11], "q_weight", type, p.D, p.device);
    const void* kw = optional_vector(a[12], "k_weight", type, p.D, p.device);
    const double eps = PyFloat_AsDouble(a[13]);
    if (eps == -1.0 && PyErr_Occurred()) throw Refused{};
    const Table w = slot_table(a[14], "weights", at::kFloat, p, p.slots);
    const Table pos = slot_table(a[15], "pos", at::kInt, p, p.slots);
    const c10::cuda::OptionalCUDAGuard guard(p.k->device());
    const at::Tensor o = output(a[16], {T, H, p.D}, p.k->options());
    check_apart(a[16], o, q, p, T, H);
    if (T > 0) {
      const int st = dcr_paged_append(
          q.data, q.st, q.sh, k.data, k.st, k.sh, v.data, v.st, v.sh, qw, kw,
          static_cast<float>(eps), cos.data_ptr(), sin.data_ptr(), dtype_code(cos, "cos"),
          static_cast<int>(cos.size(0)), static_cast<const int32_t*>(positions),
          static_cast<const int32_t*>(seq), static_cast<const int32_t*>(slots), p.dtype,
          static_cast<int>(T), static_cast<int>(H), static_cast<int>(p.H_kv),
          static_cast<int>(p.D), o.data_ptr(), p.k->data_ptr(), p.v->data_ptr(), p.k->stride(0),
          p.k->stride(1), p.k->stride(2), p.v->stride(0), p.v->stride(1), p.v->stride(2),
          static_cast<int>(p.pages), static_cast<int>(p.page_size),
          static_cast<const int32_t*>(p.table->data_ptr()), p.table_stride,
          static_cast<int>(p.sequences), static_cast<int>(p.max_pages),
          static_cast<float*>(w.data), w.sb, w.sh, static_cast<int32_t*>(pos.data), pos.sb, pos.sh,
          stream_of(p.device));
      if (st != DCR_OK) return PyLong_FromLong(st);
    }
    return THPVariable_Wrap(o);
  });
}

// (k_pages, v_pages, page_table, lengths, weights, pos, seen, budget, sinks, recent, weights_out,
//  pos_out, workspace)
PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(a, n, 13, [&]() -> PyObject* {
    const Pool p = pool_of(a[0], a[1], a[2]);
    const int64_t B = p.sequences;
    const void* lengths = vector_of(a[3], "lengths", at::kInt, B, p.device);
    cuda_tensor(a[4], "weights");
    cuda_tensor(a[5], "pos");
    const Table w = slot_table(a[4], "weights", at::kFloat, p, p.slots, false);
    const Table pos = slot_table(a[5], "pos", at::kInt, p, p.slots, false);
    const void* seen = vector_of(a[6], "seen", at::kInt, B, p.device);
    const int64_t budget = integer(a[7], "budget");
    const int64_t sinks = integer(a[8], "sinks"), recent = integer(a[9], "recent");
    if (budget <= 0 || budget > p.slots)
      refuse("budget must be in (0, " + std::to_string(p.slots) + "], got " + std::to_string(budget));
    if (sinks < 0 || sinks > INT32_MAX || recent < 0 || recent > INT32_MAX)
      refuse("sinks and recent must be >= 0");
    const c10::cuda::OptionalCUDAGuard guard(p.k->device());
    const at::TensorOptions i32 = p.table->options();
    at::Tensor wo, po;
    Table two, tpo;
    if (a[10] == Py_None) {
      wo = at::empty({B, p.H_kv, budget}, i32.dtype(at::kFloat));
      two = {wo.data_ptr(), p.H_kv * budget, budget};
    } else {
      wo = cuda_tensor(a[10], "weights_out");
      two = slot_table(a[10], "weights_out", at::kFloat, p, budget);
    }
    if (a[11] == Py_None) {
      po = at::empty({B, p.H_kv, budget}, i32);
      tpo = {po.data_ptr(), p.H_kv * budget, budget};
    } else {
      po = cuda_tensor(a[11], "pos_out");
      tpo = slot_table(a[11], "pos_out", at::kInt, p, budget);
    }
    const at::Tensor src = at::empty({B, p.H_kv, budget}, i32);
    const at::Tensor lengths_out = at::empty({B}, i32);
    if (B > 0) {
      auto span = [&](const Table& t, int64_t slots) {
        return dcr::TableSpan(t.data, B, p.H_kv, slots, t.sb, t.sh);
      };
      const dcr::TableSpan from[2] = {span(w, p.slots), span(pos, p.slots)};
      const dcr::TableSpan to[2] = {span(two, budget), span(tpo, budget)};
      if (dcr::tables_meet(from[0], to[0]) || dcr::tables_meet(from[1], to[0]) ||
          dcr::tables_meet(from[0], to[1]) || dcr::tables_meet(from[1], to[1]) ||
          dcr::tables_meet(to[0], to[1]))
        refuse("weights_out and pos_out must share no memory with weights, pos or one another");
      const size_t bytes = dcr_paged_evict_workspace_bytes(
          static_cast<int>(B), static_cast<int>(p.H_kv), static_cast<int>(budget));
      const at::Tensor ws = scratch(a[12], bytes, p.device);
      const int st = dcr_paged_evict(
          p.k->data_ptr(), p.v->data_ptr(), p.dtype, p.k->stride(0), p.k->stride(1), p.k->stride(2),
          p.v->stride(0), p.v->stride(1), p.v->stride(2), static_cast<int>(p.pages),
          static_cast<int>(p.page_size), static_cast<const int32_t*>(p.table->data_ptr()),
          p.table_stride, static_cast<int>(p.max_pages), static_cast<const int32_t*>(lengths),
          static_cast<const float*>(w.data), w.sb, w.sh, static_cast<const int32_t*>(pos.data),
          pos.sb, pos.sh, static_cast<const int32_t*>(seen), static_cast<int>(B),
          static_cast<int>(p.H_kv), static_cast<int>(p.D), static_cast<int>(budget),
          static_cast<int>(sinks), static_cast<int>(recent), static_cast<int32_t*>(src.data_ptr()),
          static_cast<float*>(two.data), two.sb, two.sh, static_cast<int32_t*>(tpo.data), tpo.sb,
          tpo.sh, static_cast<int32_t*>(lengths_out.data_ptr()), ws.data_ptr(),
          static_cast<size_t>(ws.numel()), stream_of(p.device));
      if (st != DCR_OK) return PyLong_FromLong(st);
    }
    PyObject* r = PyTuple_New(4);
    if (r == nullptr) return nullptr;
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(src));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(wo));
    PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(po));
    PyTuple_SET_ITEM(r, 3, THPVariable_Wrap(lengths_out));
    return r;
  });
}

// (logits, tokens, token_lengths, prompt_lengths, repetition, presence, frequency, bias, allowed,
//  out)
PyObject* process_logits(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(a, n, 10, [&]() -> PyObject* {
    const at::Tensor& x = cuda_tensor(a[0], "logits");
    const int dtype = dtype_code(x, "logits"), device = x.get_device();
    if (x.dim() != 2 || x.size(1) == 0 || x.stride(1) != 1) refuse("logits must be [B, V] with contiguous rows");
    const int64_t B = x.size(0), V = x.size(1);
    if (B > INT32_MAX || V > INT32_MAX) refuse("logits too large");
    const void* tokens = nullptr;
    int64_t L = 0, t_stride = 0;
    int tok64 = 0;
    if (a[1] != Py_None) {
      const at::Tensor& t = cuda_tensor(a[1], "tokens");
      if (!(t.dim() == 2 && t.size(0) == B && t.size(1) <= INT32_MAX && t.get_device() == device &&
            (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) &&
            (t.stride(1) == 1 || t.size(1) <= 1)))
        refuse("tokens must be int32 or int64 [" + std::to_string(B) + ", L] with contiguous rows on cuda:" +
               std::to_string(device));
      tokens = t.data_ptr();
      L = t.size(1);
      t_stride = t.stride(0);
      tok64 = t.scalar_type() == at::kLong;
    } else if (a[2] != Py_None || a[3] != Py_None) {
      refuse("token_lengths and prompt_lengths need tokens");
    }
    const void* n_tok = optional_vector(a[2], "token_lengths", at::kInt, B, device);
    const void* n_prompt = optional_vector(a[3], "prompt_lengths", at::kInt, B, device);
    const void* rep = optional_vector(a[4], "repetition", at::kFloat, B, device);
    const void* pres = optional_vector(a[5], "presence", at::kFloat, B, device);
    const void* freq = optional_vector(a[6], "frequency", at::kFloat, B, device);
    const void* bias = nullptr;
    int64_t b_stride = 0;
    if (a[7] != Py_None) {
      const at::Tensor& t = cuda_tensor(a[7], "bias");
      const int64_t d = t.dim();
      if (!(t.scalar_type() == at::kFloat && t.get_device() == device && (d == 1 || d == 2) &&
            t.size(d - 1) == V && (d == 1 || t.size(0) == B) && (V == 1 || t.stride(d - 1) == 1)))
        refuse("bias must be float32 [" + std::to_string(V) + "] or [" + std::to_string(B) + ", " +
               std::to_string(V) + "] with contiguous rows on cuda:" + std::to_string(device));
      bias = t.data_ptr();
      b_stride = d == 2 ? t.stride(0) : 0;
    }
    const void* allowed = nullptr;
    int64_t a_stride = 0;
    if (a[8] != Py_None) {
      const at::Tensor& t = cuda_tensor(a[8], "allowed");
      const int64_t words = (V + 31) / 32;
      if (!(t.scalar_type() == at::kInt && t.get_device() == device && t.dim() == 2 && t.size(0) == B &&
            t.size(1) == words && (words == 1 || t.stride(1) == 1)))
        refuse("allowed must be int32 " + dims({B, words}) + " with contiguous rows on cuda:" + std::to_string(device));
      allowed = t.data_ptr();
      a_stride = t.stride(0);
    }
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    at::Tensor out;
    if (a[9] == Py_None) {
      out = at::empty({B, V}, x.options());
    } else {
      out = cuda_tensor(a[9], "out");
      if (!(out.sizes() == x.sizes() && out.scalar_type() == x.scalar_type() &&
            out.get_device() == device && out.stride(1) == 1))
        refuse("out must match logits, with contiguous rows");
      if (out.data_ptr() == x.data_ptr() && out.strides() != x.strides())
        refuse("logits processed in place must keep their strides");
      if ((B <= 1 || out.stride(0) >= V) &&  // else refused below
          dcr::logits_meet(x.data_ptr(), x.stride(0), out.data_ptr(), out.stride(0), B, V,
                           x.element_size()))
        refuse("out must be the logits themselves or share no memory with them");
    }
    const at::Tensor token = at::empty({B}, x.options().dtype(at::kLong));
    if (B > 0) {
      const int st = dcr_process_logits(
          x.data_ptr(), x.stride(0), dtype, static_cast<int>(B), static_cast<int>(V), tokens, tok64,
          t_stride, static_cast<int>(L), static_cast<const int32_t*>(n_tok),
          static_cast<const int32_t*>(n_prompt), static_cast<const float*>(rep),
          static_cast<const float*>(pres), static_cast<const float*>(freq),
          static_cast<const float*>(bias), b_stride, static_cast<const uint32_t*>(allowed), a_stride,
          out.data_ptr(), out.stride(0), static_cast<int64_t*>(token.data_ptr()), stream_of(device));
      if (st != DCR_OK) return PyLong_FromLong(st);
    }
    PyObject* r = PyTuple_New(2);
    if (r == nullptr) return nullptr;
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(out));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(token));
    return r;
  });
}

PyMethodDef kMethods[] = {
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attend)), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL, nullptr},
    {"evict", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(evict)), METH_FASTCALL, nullptr},
    {"process_logits", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(process_logits)),
     METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "dcr_b200_torch",
                       "Paged serving operators of libdcr_b200 on torch tensors.", -1, kMethods};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_dcr_b200_torch() {
  return PyModule_Create(&kModule);
}
