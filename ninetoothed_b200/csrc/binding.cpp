// The serving operators' calls bound in C++: what serving.py does for a good
// call (checks, outputs, workspace, argument struct, launch on the current
// stream), without the interpreter's time for it, 11 to 20 us of a small call's.
//
// A call that anything is unusual about (a check fails, an output is empty, the
// tensors are not on the current device) is not made here: the function returns
// None, and serving.py's own path makes it or says what is wrong with it.  A
// nonzero launch code is returned as an int.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/nt_b200.h"

namespace {

decltype(&nt_b200_rotary) rotary_entry;
decltype(&nt_b200_paged_append) append_entry;
decltype(&nt_b200_paged_attention) paged_entry;
decltype(&nt_b200_prompt_attention) prompt_entry;
decltype(&nt_b200_chunk_attention) chunk_entry;
decltype(&nt_b200_rms_norm) norm_entry;
decltype(&nt_b200_int4_matmul) int4_entry;
decltype(&nt_b200_paged_attention_workspace_size) paged_workspace;
decltype(&nt_b200_prompt_attention_workspace_size) prompt_workspace;
decltype(&nt_b200_chunk_attention_workspace_size) chunk_workspace;

// The tensors of a call: all strided CUDA tensors of the current device.
struct Call {
  int device;
  bool good = true;
  Call() : device(c10::cuda::current_device()) {}
  const at::Tensor &tensor(PyObject *o, int64_t dim) {
    static const at::Tensor none;
    if (!THPVariable_Check(o)) {
      good = false;
      return none;
    }
    const at::Tensor &t = THPVariable_Unpack(o);
    good = good && t.defined() && t.layout() == at::kStrided && t.is_cuda() && t.get_device() == device && t.dim() == dim;
    return t;
  }
  void *stream() const { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }
};

int64_t code_of(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::kHalf: return NT_B200_FLOAT16;
    case at::kBFloat16: return NT_B200_BFLOAT16;
    case at::kFloat: return NT_B200_FLOAT32;
    case at::kInt: return NT_B200_INT32;
    case at::kLong: return NT_B200_INT64;
    case at::kChar: return NT_B200_INT8;
    case at::kFloat8_e4m3fn: return NT_B200_FLOAT8_E4M3FN;
    default: return -1;
  }
}
bool is_float(const at::Tensor &t) {
  return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat;
}
bool is_index(const at::Tensor &t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }

// Lets other Python threads run: allocations and launches can wait for the device
// (a full launch queue), and what they wait for may need the interpreter.
struct Released {
  PyThreadState *state = PyEval_SaveThread();
  void reset() {
    if (state) PyEval_RestoreThread(state);
    state = nullptr;
  }
  ~Released() { reset(); }
};

template <int N> void strides(const at::Tensor &t, int64_t (&to)[N]) {
  for (int i = 0; i < N; ++i) to[i] = t.stride(i);
}
at::Tensor like(const at::Tensor &t) { return at::empty(t.sizes(), t.options()); }

bool good_tables(const at::Tensor &cos, const at::Tensor &sin, int64_t dim) {
  return cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat && cos.sizes() == sin.sizes() &&
         2 * cos.size(1) <= dim && (cos.size(0) > 0 || cos.size(1) == 0) &&
         (cos.size(1) <= 1 || (cos.stride(1) == 1 && sin.stride(1) == 1));
}

bool cache_of(Call &call, PyObject *const *o, NtB200PagedCache &c) {
  const at::Tensor &k = call.tensor(o[0], 4), &v = call.tensor(o[1], 4);
  const at::Tensor &ks = call.tensor(o[2], 2), &vs = call.tensor(o[3], 2);
  if (!call.good || (k.scalar_type() != at::kChar && k.scalar_type() != at::kFloat8_e4m3fn) ||
      v.scalar_type() != k.scalar_type() || ks.scalar_type() != at::kFloat || vs.scalar_type() != at::kFloat ||
      v.sizes() != k.sizes() || ks.sizes() != k.sizes().slice(0, 2) || vs.sizes() != ks.sizes() || k.numel() == 0 ||
      k.size(2) % 16 || k.size(2) > 4096 || k.size(3) % 16 || k.stride(3) != 1 || v.stride(3) != 1)
    return false;
  c.key = k.data_ptr(); c.value = v.data_ptr();
  c.key_scale = static_cast<float *>(ks.data_ptr()); c.value_scale = static_cast<float *>(vs.data_ptr());
  c.pages = k.size(0); c.kv_heads = k.size(1); c.page = k.size(2); c.head_dim = k.size(3);
  c.code_dtype = code_of(k);
  strides(k, c.key_strides); strides(v, c.value_strides);
  strides(ks, c.key_scale_strides); strides(vs, c.value_scale_strides);
  return true;
}

PyObject *none() { Py_RETURN_NONE; }

// Whether an object has a truth value, and which.  One that has none is an odd
// call too: Python's own path raises for it.
bool flag(PyObject *o, bool &value) {
  const int truth = PyObject_IsTrue(o);
  if (truth < 0) PyErr_Clear();
  value = truth > 0;
  return truth >= 0;
}

// rotary(input, cos, sin, positions, interleaved, adjoint)
PyObject *rotary(PyObject *, PyObject *const *o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  bool interleaved, adjoint;
  if (n != 6 || !rotary_entry || !flag(o[4], interleaved) || !flag(o[5], adjoint)) return none();
  Call call;
  const at::Tensor &x = call.tensor(o[0], 3), &cos = call.tensor(o[1], 2), &sin = call.tensor(o[2], 2);
  const at::Tensor &at = call.tensor(o[3], 1);
  if (!call.good || !is_float(x) || !is_index(at) || at.size(0) != x.size(0) || x.numel() == 0 ||
      !good_tables(cos, sin, x.size(2)))
    return none();
  Released released;
  at::Tensor out = like(x);
  NtB200RotaryArgs a{};
  a.input = x.data_ptr(); a.output = out.data_ptr(); a.positions = at.data_ptr();
  a.cos = static_cast<const float *>(cos.data_ptr()); a.sin = static_cast<const float *>(sin.data_ptr());
  a.tokens = x.size(0); a.heads = x.size(1); a.head_dim = x.size(2); a.rotary_dim = 2 * cos.size(1); a.table_rows = cos.size(0);
  strides(x, a.input_strides); strides(out, a.output_strides);
  a.cos_stride = cos.stride(0); a.sin_stride = sin.stride(0); a.positions_stride = at.stride(0);
  a.interleaved = interleaved; a.adjoint = adjoint;
  a.dtype = code_of(x); a.index_dtype = code_of(at);
  const int code = rotary_entry(&a, call.stream());
  released.reset();
  return code ? PyLong_FromLong(code) : THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// paged_append(key, value, offsets, past, block_table, key_cache, value_cache,
// key_scale, value_scale, query, cos, sin, interleaved, return_key)
PyObject *paged_append(PyObject *, PyObject *const *o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  bool interleaved, return_key;
  if (n != 14 || !append_entry || !flag(o[12], interleaved) || !flag(o[13], return_key)) return none();
  Call call;
  const bool asks = o[9] != Py_None, turns = o[10] != Py_None;
  if (turns != (o[11] != Py_None) || (asks && !turns)) return none();
  const at::Tensor &k = call.tensor(o[0], 3), &v = call.tensor(o[1], 3);
  const at::Tensor &offsets = call.tensor(o[2], 1), &past = call.tensor(o[3], 1), &table = call.tensor(o[4], 2);
  NtB200PagedAppendArgs a{};
  if (!cache_of(call, o + 5, a.cache) || !is_float(k) || v.scalar_type() != k.scalar_type() || v.sizes() != k.sizes() ||
      k.numel() == 0 || k.size(1) != a.cache.kv_heads || k.size(2) != a.cache.head_dim || !is_index(offsets) ||
      past.scalar_type() != offsets.scalar_type() || table.scalar_type() != offsets.scalar_type() ||
      offsets.size(0) != past.size(0) + 1 || table.size(0) != past.size(0))
    return none();
  at::Tensor query_out, key_out;
  const at::Tensor *query = nullptr;
  if (turns) {
    const at::Tensor &cos = call.tensor(o[10], 2), &sin = call.tensor(o[11], 2);
    if (!call.good || !good_tables(cos, sin, k.size(2))) return none();
    a.cos = static_cast<const float *>(cos.data_ptr()); a.sin = static_cast<const float *>(sin.data_ptr());
    a.rotary_dim = 2 * cos.size(1); a.table_rows = cos.size(0);
    a.cos_stride = cos.stride(0); a.sin_stride = sin.stride(0);
  }
  if (asks) {
    const at::Tensor &q = call.tensor(o[9], 3);
    if (!call.good || q.scalar_type() != k.scalar_type() || q.size(0) != k.size(0) || q.size(2) != k.size(2)) return none();
    query = &q;
  }
  Released released;
  if (query) {
    query_out = like(*query);
    a.query = query->data_ptr(); a.query_out = query_out.data_ptr(); a.heads = query->size(1);
    strides(*query, a.query_strides); strides(query_out, a.query_out_strides);
  }
  if (return_key) {
    key_out = like(k);
    a.key_out = key_out.data_ptr();
    strides(key_out, a.key_out_strides);
  }
  a.key = k.data_ptr(); a.value = v.data_ptr();
  a.offsets = offsets.data_ptr(); a.past = past.data_ptr(); a.block_table = table.data_ptr();
  a.tokens = k.size(0); a.batch = past.size(0); a.table_columns = table.size(1);
  strides(k, a.key_strides); strides(v, a.value_strides); strides(table, a.block_table_strides);
  a.offsets_stride = offsets.stride(0); a.past_stride = past.stride(0);
  a.interleaved = interleaved; a.dtype = code_of(k); a.index_dtype = code_of(offsets);
  const int code = append_entry(&a, call.stream());
  released.reset();
  if (code) return PyLong_FromLong(code);
  PyObject *q = asks ? THPVariable_Wrap(query_out) : Py_NewRef(Py_None);
  PyObject *r = a.key_out ? THPVariable_Wrap(key_out) : Py_NewRef(Py_None);
  PyObject *both = q && r ? PyTuple_Pack(2, q, r) : nullptr;
  Py_XDECREF(q);
  Py_XDECREF(r);
  return both;
  END_HANDLE_TH_ERRORS
}

// scale: a number, or None for 1 / sqrt(dim); false if it is neither
bool scale_of(PyObject *o, int64_t dim, double &scale) {
  if (o == Py_None) {
    scale = 1.0 / std::sqrt((double)dim);
    return true;
  }
  if (!PyFloat_Check(o)) return false;
  scale = PyFloat_AS_DOUBLE(o);
  return true;
}

PyObject *with_lse(const at::Tensor &out, const at::Tensor &lse) {
  if (!lse.defined()) return THPVariable_Wrap(out);
  PyObject *a = THPVariable_Wrap(out), *b = THPVariable_Wrap(lse);
  PyObject *both = a && b ? PyTuple_Pack(2, a, b) : nullptr;
  Py_XDECREF(a);
  Py_XDECREF(b);
  return both;
}

// paged_attention(query, key_cache, value_cache, key_scale, value_scale,
// block_table, lengths, scale, return_lse)
PyObject *paged_attention(PyObject *, PyObject *const *o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  bool return_lse;
  if (n != 9 || !paged_entry || !flag(o[8], return_lse)) return none();
  Call call;
  const at::Tensor &q = call.tensor(o[0], 4), &table = call.tensor(o[5], 2), &lengths = call.tensor(o[6], 1);
  NtB200PagedAttentionArgs a{};
  if (!cache_of(call, o + 1, a.cache) || !is_float(q) || q.numel() == 0 || q.size(3) != a.cache.head_dim || q.size(3) > 256 ||
      q.size(2) % a.cache.kv_heads || !is_index(lengths) || table.scalar_type() != lengths.scalar_type() ||
      lengths.size(0) != q.size(0) || table.size(0) != q.size(0) || !scale_of(o[7], q.size(3), a.scale))
    return none();
  Released released;
  at::Tensor out = like(q), lse;
  if (return_lse) {
    lse = at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
    a.lse = static_cast<float *>(lse.data_ptr());
    strides(lse, a.lse_strides);
  }
  a.workspace_bytes = paged_workspace();
  at::Tensor workspace = at::empty({a.workspace_bytes}, q.options().dtype(at::kByte));
  a.query = q.data_ptr(); a.lengths = lengths.data_ptr(); a.block_table = table.data_ptr();
  a.output = out.data_ptr(); a.workspace = workspace.data_ptr();
  a.batch = q.size(0); a.queries = q.size(1); a.heads = q.size(2); a.table_columns = table.size(1);
  strides(q, a.query_strides); strides(out, a.output_strides); strides(table, a.block_table_strides);
  a.lengths_stride = lengths.stride(0); a.dtype = code_of(q); a.index_dtype = code_of(lengths);
  const int code = paged_entry(&a, call.stream());
  released.reset();
  return code ? PyLong_FromLong(code) : with_lse(out, lse);
  END_HANDLE_TH_ERRORS
}

// prompt_attention(query, key, value, offsets, key_offsets, is_causal, scale,
// return_lse)
PyObject *prompt_attention(PyObject *, PyObject *const *o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  bool is_causal, return_lse;
  if (n != 8 || !prompt_entry || !flag(o[5], is_causal) || !flag(o[7], return_lse)) return none();
  Call call;
  const at::Tensor &q = call.tensor(o[0], 3), &k = call.tensor(o[1], 3), &v = call.tensor(o[2], 3);
  const at::Tensor &qo = call.tensor(o[3], 1), &ko = call.tensor(o[4], 1);
  NtB200PromptAttentionArgs a{};
  if (!call.good || !is_float(q) || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() ||
      q.numel() == 0 || k.numel() == 0 || v.sizes() != k.sizes() || k.size(2) != q.size(2) || q.size(2) > 256 ||
      q.size(1) % k.size(1) || !is_index(qo) || ko.scalar_type() != qo.scalar_type() || qo.size(0) < 1 ||
      ko.sizes() != qo.sizes() || !scale_of(o[6], q.size(2), a.scale))
    return none();
  Released released;
  at::Tensor out = like(q), lse;
  if (return_lse) {
    lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
    a.lse = static_cast<float *>(lse.data_ptr());
    strides(lse, a.lse_strides);
  }
  a.query_tokens = q.size(0); a.key_tokens = k.size(0); a.batch = qo.size(0) - 1;
  a.heads = q.size(1); a.kv_heads = k.size(1); a.head_dim = q.size(2);
  a.workspace_bytes = prompt_workspace(a.query_tokens, a.batch, a.heads, a.kv_heads);
  at::Tensor workspace = at::empty({a.workspace_bytes}, q.options().dtype(at::kByte));
  a.query = q.data_ptr(); a.key = k.data_ptr(); a.value = v.data_ptr();
  a.query_offsets = qo.data_ptr(); a.key_offsets = ko.data_ptr();
  a.output = out.data_ptr(); a.workspace = workspace.data_ptr();
  strides(q, a.query_strides); strides(k, a.key_strides); strides(v, a.value_strides); strides(out, a.output_strides);
  a.query_offsets_stride = qo.stride(0); a.key_offsets_stride = ko.stride(0);
  a.is_causal = is_causal; a.dtype = code_of(q); a.index_dtype = code_of(qo);
  const int code = prompt_entry(&a, call.stream());
  released.reset();
  return code ? PyLong_FromLong(code) : with_lse(out, lse);
  END_HANDLE_TH_ERRORS
}

// chunk_attention(query, key_cache, value_cache, key_scale, value_scale,
// block_table, offsets, lengths, scale, return_lse)
PyObject *chunk_attention(PyObject *, PyObject *const *o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  bool return_lse;
  if (n != 10 || !chunk_entry || !flag(o[9], return_lse)) return none();
  Call call;
  const at::Tensor &q = call.tensor(o[0], 3), &table = call.tensor(o[5], 2), &offsets = call.tensor(o[6], 1);
  const at::Tensor &lengths = call.tensor(o[7], 1);
  NtB200ChunkAttentionArgs a{};
  if (!cache_of(call, o + 1, a.cache) || !is_float(q) || q.numel() == 0 || q.size(2) != a.cache.head_dim || q.size(2) > 256 ||
      q.size(1) % a.cache.kv_heads || !is_index(lengths) || table.scalar_type() != lengths.scalar_type() ||
      offsets.scalar_type() != lengths.scalar_type() || offsets.size(0) != lengths.size(0) + 1 ||
      table.size(0) != lengths.size(0) || !scale_of(o[8], q.size(2), a.scale))
    return none();
  Released released;
  at::Tensor out = like(q), lse;
  if (return_lse) {
    lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
    a.lse = static_cast<float *>(lse.data_ptr());
    strides(lse, a.lse_strides);
  }
  a.workspace_bytes = chunk_workspace();
  at::Tensor workspace = at::empty({a.workspace_bytes}, q.options().dtype(at::kByte));
  a.query = q.data_ptr(); a.offsets = offsets.data_ptr(); a.lengths = lengths.data_ptr(); a.block_table = table.data_ptr();
  a.output = out.data_ptr(); a.workspace = workspace.data_ptr();
  a.tokens = q.size(0); a.batch = lengths.size(0); a.heads = q.size(1); a.table_columns = table.size(1);
  strides(q, a.query_strides); strides(out, a.output_strides); strides(table, a.block_table_strides);
  a.offsets_stride = offsets.stride(0); a.lengths_stride = lengths.stride(0);
  a.dtype = code_of(q); a.index_dtype = code_of(lengths);
  const int code = chunk_entry(&a, call.stream());
  released.reset();
  return code ? PyLong_FromLong(code) : with_lse(out, lse);
  END_HANDLE_TH_ERRORS
}

// A whole number, or none; false if it is neither.
bool whole(PyObject *o, int64_t none, int64_t &value) {
  if (o == Py_None) {
    value = none;
    return true;
  }
  if (!PyLong_CheckExact(o)) return false;
  value = PyLong_AsLongLong(o);
  if (value == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

// rms_norm(input, weight, residual, eps, code_dtype, group)
PyObject *rms_norm(PyObject *, PyObject *const *o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !norm_entry || !PyFloat_Check(o[3])) return none();
  Call call;
  const bool adds = o[2] != Py_None, codes = o[4] != Py_None;
  const at::Tensor &x = call.tensor(o[0], 2), &w = call.tensor(o[1], 1);
  if (!call.good || !is_float(x) || x.numel() == 0 || w.size(0) != x.size(1) || x.size(1) > 131072 ||
      (w.scalar_type() != x.scalar_type() && w.scalar_type() != at::kFloat))
    return none();
  NtB200RmsNormArgs a{};
  a.eps = PyFloat_AS_DOUBLE(o[3]);
  at::ScalarType out_type = x.scalar_type();
  const int64_t width = x.size(1);
  if (!(a.eps >= 0) || !whole(o[5], 0, a.group) || a.group < 0 || (!codes && o[5] != Py_None)) return none();
  if (codes) {
    if (!THPDtype_Check(o[4])) return none();
    out_type = reinterpret_cast<THPDtype *>(o[4])->scalar_type;
    if (out_type != at::kChar && out_type != at::kFloat8_e4m3fn) return none();
    if (o[5] != Py_None && a.group < width && (a.group == 0 || a.group % 16)) return none();
  }
  if (o[5] == Py_None || a.group > width) a.group = width;
  const at::Tensor *residual = nullptr;
  if (adds) {
    const at::Tensor &r = call.tensor(o[2], 2);
    if (!call.good || r.scalar_type() != x.scalar_type() || r.sizes() != x.sizes()) return none();
    residual = &r;
  }
  Released released;
  at::Tensor out = at::empty(x.sizes(), x.options().dtype(out_type)), scale, total;
  if (codes) {
    scale = at::empty({x.size(0), (width + a.group - 1) / a.group}, x.options().dtype(at::kFloat));
    a.scale = static_cast<float *>(scale.data_ptr());
    strides(scale, a.scale_strides);
  }
  if (residual) {
    total = like(x);
    a.residual = residual->data_ptr(); a.total = total.data_ptr();
    strides(*residual, a.residual_strides); strides(total, a.total_strides);
  }
  a.input = x.data_ptr(); a.weight = w.data_ptr(); a.output = out.data_ptr();
  a.rows = x.size(0); a.width = width;
  strides(x, a.input_strides); strides(out, a.output_strides);
  a.weight_stride = w.stride(0);
  a.dtype = code_of(x); a.weight_dtype = code_of(w); a.output_dtype = code_of(out);
  const int code = norm_entry(&a, call.stream());
  released.reset();
  if (code) return PyLong_FromLong(code);
  if (!codes && !residual) return THPVariable_Wrap(out);
  PyObject *parts[3] = {THPVariable_Wrap(out), nullptr, nullptr};
  int count = 1;
  if (codes) parts[count++] = THPVariable_Wrap(scale);
  if (residual) parts[count++] = THPVariable_Wrap(total);
  PyObject *all = nullptr;
  if (parts[0] && parts[1] && (count < 3 || parts[2]))
    all = count == 2 ? PyTuple_Pack(2, parts[0], parts[1]) : PyTuple_Pack(3, parts[0], parts[1], parts[2]);
  for (PyObject *part : parts) Py_XDECREF(part);
  return all;
  END_HANDLE_TH_ERRORS
}

// int4_matmul(input, codes, scales, zeros, input_scale)
PyObject *int4_matmul(PyObject *, PyObject *const *o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5 || !int4_entry) return none();
  Call call;
  const at::Tensor &x = call.tensor(o[0], 2), &codes = call.tensor(o[1], 2), &scales = call.tensor(o[2], 2);
  if (!call.good || x.numel() == 0 || codes.numel() == 0 || scales.numel() == 0 || codes.scalar_type() != at::kByte ||
      !is_float(scales))
    return none();
  const bool eight = x.scalar_type() == at::kChar || x.scalar_type() == at::kFloat8_e4m3fn;
  const int64_t inner = x.size(1), groups = scales.size(1);
  if ((!eight && !is_float(x)) || codes.size(0) != scales.size(0) || codes.size(1) != inner / 2 || inner % groups ||
      inner / groups % 32)
    return none();
  NtB200Int4MatmulArgs a{};
  if (o[3] != Py_None) {
    const at::Tensor &zeros = call.tensor(o[3], 2);
    if (!call.good || zeros.scalar_type() != at::kByte || zeros.sizes() != scales.sizes()) return none();
    a.zeros = zeros.data_ptr();
    strides(zeros, a.zeros_strides);
  }
  if (o[4] != Py_None) {
    if (!THPVariable_Check(o[4])) return none();
    const int64_t dim = THPVariable_Unpack(o[4]).dim();
    const at::Tensor &by = call.tensor(o[4], dim);
    if (!call.good || by.scalar_type() != at::kFloat || dim < 1 || dim > 2 || by.size(0) != x.size(0) ||
        (dim == 2 && by.size(1) != 1))
      return none();
    a.input_scale = static_cast<const float *>(by.data_ptr());
    a.input_scale_stride = by.stride(0);
  }
  Released released;
  at::Tensor out = at::empty({x.size(0), scales.size(0)}, x.options().dtype(eight ? scales.scalar_type() : x.scalar_type()));
  a.input = x.data_ptr(); a.codes = codes.data_ptr(); a.scales = scales.data_ptr(); a.output = out.data_ptr();
  a.rows = x.size(0); a.inner = inner; a.outer = scales.size(0); a.group = inner / groups;
  strides(x, a.input_strides); strides(codes, a.codes_strides); strides(scales, a.scales_strides); strides(out, a.output_strides);
  a.dtype = code_of(x); a.scales_dtype = code_of(scales); a.output_dtype = code_of(out);
  const int code = int4_entry(&a, call.stream());
  released.reset();
  return code ? PyLong_FromLong(code) : THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// bind(addresses of the library's entry points, in the order above)
PyObject *bind(PyObject *, PyObject *const *o, Py_ssize_t n) {
  if (n != 10) {
    PyErr_SetString(PyExc_TypeError, "bind takes ten addresses");
    return nullptr;
  }
  void *at[10];
  for (int i = 0; i < 10; ++i) {
    at[i] = PyLong_AsVoidPtr(o[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  rotary_entry = reinterpret_cast<decltype(rotary_entry)>(at[0]);
  append_entry = reinterpret_cast<decltype(append_entry)>(at[1]);
  paged_entry = reinterpret_cast<decltype(paged_entry)>(at[2]);
  prompt_entry = reinterpret_cast<decltype(prompt_entry)>(at[3]);
  chunk_entry = reinterpret_cast<decltype(chunk_entry)>(at[4]);
  norm_entry = reinterpret_cast<decltype(norm_entry)>(at[5]);
  int4_entry = reinterpret_cast<decltype(int4_entry)>(at[6]);
  paged_workspace = reinterpret_cast<decltype(paged_workspace)>(at[7]);
  prompt_workspace = reinterpret_cast<decltype(prompt_workspace)>(at[8]);
  chunk_workspace = reinterpret_cast<decltype(chunk_workspace)>(at[9]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(bind), METH_FASTCALL, nullptr},
    {"rotary", reinterpret_cast<PyCFunction>(rotary), METH_FASTCALL, nullptr},
    {"paged_append", reinterpret_cast<PyCFunction>(paged_append), METH_FASTCALL, nullptr},
    {"paged_attention", reinterpret_cast<PyCFunction>(paged_attention), METH_FASTCALL, nullptr},
    {"prompt_attention", reinterpret_cast<PyCFunction>(prompt_attention), METH_FASTCALL, nullptr},
    {"chunk_attention", reinterpret_cast<PyCFunction>(chunk_attention), METH_FASTCALL, nullptr},
    {"rms_norm", reinterpret_cast<PyCFunction>(rms_norm), METH_FASTCALL, nullptr},
    {"int4_matmul", reinterpret_cast<PyCFunction>(int4_matmul), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&module_def); }
