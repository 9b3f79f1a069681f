// Direct Python entry points: the calls of a generation loop (attention over key lengths, decode against a dense or
// paged cache, a chunk behind a cached prefix) go from Python into the C ABI in one foreign call.
//
// The small calls of this package take 10-20 us on the GPU; through the ctypes binding the host needed 24 us
// (sdpa_forward) to 52 us (scaled_dot_product_attention with kv_lens) to enqueue one, so the GPU waited.  Here the
// whole call -- checks, output and scratch allocation, parameter block, launch -- is native.
//
// Every function returns None when the call is not one of the plain ones it serves (subclasses, active modes and
// transforms, tracing, forward-mode tangents, gradients, other dtypes, anything malformed); the Python layer then takes its own path, which serves the rest and
// raises the errors.  So nothing here raises for a bad argument.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/_scaled_dot_product_fused_attention_overrideable.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "ops_common.h"

namespace {

using namespace b200_ops;

struct NoGil {   // the interpreter lock is released for the lifetime of the object
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

// The record of the last forward's plan: the dict of the Python layer, filled under the interpreter lock.
PyObject* g_plan_record = nullptr;

bool record_plan(const B200SdpaPlan& plan) {
  if (g_plan_record == nullptr) return true;
  static PyObject* const names[] = {
      PyUnicode_InternFromString("path"),      PyUnicode_InternFromString("block_m"),    PyUnicode_InternFromString("block_n"),
      PyUnicode_InternFromString("grid"),      PyUnicode_InternFromString("threads"),    PyUnicode_InternFromString("smem_bytes"),
      PyUnicode_InternFromString("kv_splits"), PyUnicode_InternFromString("launches"),   PyUnicode_InternFromString("workspace_bytes")};
  static PyObject* const paths[] = {PyUnicode_InternFromString("auto"), PyUnicode_InternFromString("generic"),
                                    PyUnicode_InternFromString("prefill"), PyUnicode_InternFromString("decode")};
  PyObject* const values[] = {Py_NewRef(paths[plan.path & 3]),
                              PyLong_FromLong(plan.block_m),
                              PyLong_FromLong(plan.block_n),
                              Py_BuildValue("(iii)", plan.grid_x, plan.grid_y, plan.grid_z),
                              PyLong_FromLong(plan.threads),
                              PyLong_FromLong(plan.smem_bytes),
                              PyLong_FromLong(plan.kv_splits),
                              PyLong_FromLong(plan.launches),
                              PyLong_FromUnsignedLongLong(plan.workspace_bytes)};
  PyDict_Clear(g_plan_record);
  bool ok = true;
  for (int i = 0; i < 9; ++i) {
    ok = ok && values[i] != nullptr && PyDict_SetItem(g_plan_record, names[i], values[i]) == 0;
    Py_XDECREF(values[i]);
  }
  return ok;
}

// A plain strided CUDA tensor with nothing between it and the kernels; a dual tensor of forward-mode differentiation
// has the same keys but carries a tangent, which only the dispatcher's formulas see (and refuse).
bool plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  static const uint64_t expected = c10::DispatchKeySet({c10::DispatchKey::CUDA, c10::DispatchKey::AutogradCUDA,
                                                        c10::DispatchKey::ADInplaceOrView, c10::DispatchKey::AutocastCUDA})
                                       .raw_repr();
  return t.is_cuda() && (t.key_set().raw_repr() & ~expected) == 0 && !t._fw_grad(/*level=*/0).defined();
}
// Nothing on this thread stands between a call and the CUDA kernels.  The modes written in Python have stacks of their
// own; whatever else wants to see every call (the tracer, functorch's transforms, functionalization) includes a
// dispatch key.  Those included by default and autocast's, which these operations do not listen to, may be there.
bool no_modes() {
  static const c10::DispatchKeySet harmless = c10::default_included_set | c10::autocast_dispatch_keyset;
  return !at::impl::torch_function_mode_enabled() && !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
         (c10::impl::tls_local_dispatch_key_set().included_ - harmless).empty();
}
bool wants_grad(const at::Tensor& t) { return t.requires_grad(); }

// out := the tensor of `o`, or an undefined one for None; false when `o` is something else.
bool optional_plain(PyObject* o, at::Tensor* out) {
  if (o == Py_None) return true;
  if (!plain(o)) return false;
  *out = THPVariable_Unpack(o);
  return true;
}
bool as_int(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &overflow);
  return overflow == 0;
}
bool as_bool(PyObject* o, bool* v) {
  if (!PyBool_Check(o)) return false;
  *v = o == Py_True;
  return true;
}
bool as_scale(PyObject* o, int64_t head_dim, float* v) {
  if (o == Py_None) {
    *v = static_cast<float>(1.0 / std::sqrt(static_cast<double>(head_dim)));
    return true;
  }
  if (!PyFloat_CheckExact(o)) return false;
  *v = static_cast<float>(PyFloat_AS_DOUBLE(o));
  return true;
}

// The rules of the Python layer's validation for one forward call.
bool shapes_ok(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v) {
  return q.dim() == 4 && k.dim() == 4 && v.dim() == 4 && dtype_code(q.scalar_type()) >= 0 &&
         q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type() && q.device() == k.device() &&
         q.device() == v.device() && q.size(0) == k.size(0) && q.size(0) == v.size(0) && k.size(1) == v.size(1) &&
         k.size(2) == v.size(2) && q.size(3) == k.size(3) && k.size(1) != 0 && q.size(1) % k.size(1) == 0 &&
         q.numel() != 0 && k.size(3) != 0 && v.size(3) != 0;
}
bool lens_ok(const at::Tensor& lens, const at::Tensor& q) {
  return lens.scalar_type() == at::kInt && lens.device() == q.device() && lens.dim() == 1 && lens.size(0) == q.size(0) &&
         lens.is_contiguous();
}

void fill_common(B200SdpaParams& p, const at::Tensor& q, const at::Tensor& out, const at::Tensor& lse, int dev) {
  p.struct_size = sizeof(B200SdpaParams);
  p.dtype = dtype_code(q.scalar_type());
  p.device = dev;
  p.q = q.data_ptr();
  p.out = out.data_ptr();
  copy_strides(q, p.q_stride);
  copy_strides(out, p.out_stride);
  if (lse.defined()) {
    p.lse = lse.data_ptr<float>();
    copy_strides(lse, p.lse_stride);
  }
  p.B = static_cast<int32_t>(q.size(0));
  p.Hq = static_cast<int32_t>(q.size(1));
  p.L = static_cast<int32_t>(q.size(2));
  p.E = static_cast<int32_t>(q.size(3));
  p.status = device_state(dev).status.data_ptr<int32_t>();
}

// Plan, scratch, launch; the interpreter lock is not held.
void launch(B200SdpaParams& p, int dev, bool decode_only, B200SdpaPlan& plan) {
  at::Tensor ws;   // freed (stream-ordered) when the launch has been queued
  NoGil nogil;
  plan.struct_size = sizeof(B200SdpaPlan);
  int rc = b200_sdpa_query_plan(&p, &plan);
  TORCH_CHECK(rc == B200_SDPA_OK, "b200_sdpa_query_plan: ", b200_sdpa_strerror(rc));
  if (plan.workspace_bytes != 0) {
    ws = scratch(dev, plan.workspace_bytes);
    p.workspace = ws.data_ptr();
    p.workspace_bytes = static_cast<uint64_t>(ws.numel());
  }
  const auto stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  rc = decode_only ? b200_sdpa_decode(&p, stream) : b200_sdpa_fwd(&p, stream);
  TORCH_CHECK(rc == B200_SDPA_OK, decode_only ? "b200_sdpa_decode: " : "b200_sdpa_fwd: ", b200_sdpa_strerror(rc));
}

struct ForwardArgs {
  bool causal = false;
  float scale = 0.f;
  int64_t q_offset = 0, k_offset = 0, force_path = 0, kv_chunk = 0;
  at::Tensor lens;
};

// False: a Python error is set.
bool forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const ForwardArgs& a, const at::Tensor& out,
             const at::Tensor& lse) {
  const int dev = q.device().index();
  B200SdpaParams p{};
  fill_common(p, q, out, lse, dev);
  p.force_path = static_cast<int32_t>(a.force_path);
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  copy_strides(k, p.k_stride);
  copy_strides(v, p.v_stride);
  p.Hkv = static_cast<int32_t>(k.size(1));
  p.S = static_cast<int32_t>(k.size(2));
  p.Dv = static_cast<int32_t>(v.size(3));
  p.scale = a.scale;
  p.is_causal = a.causal ? 1 : 0;
  p.q_offset = a.q_offset;
  p.k_offset = a.k_offset;
  p.kv_chunk = static_cast<int32_t>(a.kv_chunk);
  if (a.lens.defined()) p.kv_lens = a.lens.data_ptr<int32_t>();
  B200SdpaPlan plan{};
  launch(p, dev, false, plan);
  return record_plan(plan);
}

#define NOT_SERVED() do { if (PyErr_Occurred()) PyErr_Clear(); Py_RETURN_NONE; } while (0)

// attention(query, key, value, is_causal, scale, enable_gqa, kv_lens) -> output or None
PyObject* py_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  ForwardArgs a;
  bool gqa = false;
  if (n != 7 || !plain(args[0]) || !plain(args[1]) || !plain(args[2]) || !as_bool(args[3], &a.causal) ||
      !as_bool(args[5], &gqa) || !optional_plain(args[6], &a.lens) || !no_modes())
    NOT_SERVED();
  const at::Tensor& q = THPVariable_Unpack(args[0]);
  const at::Tensor& k = THPVariable_Unpack(args[1]);
  const at::Tensor& v = THPVariable_Unpack(args[2]);
  if (!shapes_ok(q, k, v) || !as_scale(args[4], q.size(3), &a.scale)) NOT_SERVED();
  if (!gqa && q.size(1) != k.size(1)) NOT_SERVED();
  if (a.lens.defined() && !lens_ok(a.lens, q)) NOT_SERVED();
  at::Tensor out;
  if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(v))) {
    if (a.lens.defined()) NOT_SERVED();
    NoGil nogil;
    c10::optional<double> scale;
    if (args[4] != Py_None) scale = PyFloat_AS_DOUBLE(args[4]);
    out = std::get<0>(at::_scaled_dot_product_fused_attention_overrideable(q, k, v, c10::nullopt, 0.0, a.causal, false, scale));
  } else {
    const c10::cuda::CUDAGuard guard(q.device());
    out = alloc_like_query(q, {q.size(0), q.size(1), q.size(2), v.size(3)});
    if (!forward(q, k, v, a, out, at::Tensor())) return nullptr;
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// forward(query, key, value, is_causal, scale, kv_lens, q_offset, k_offset, need_lse, out, lse, force_path, kv_chunk)
//   -> (out, lse or None), or None
PyObject* py_forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  ForwardArgs a;
  bool need_lse = false;
  at::Tensor out, lse;
  if (n != 13 || !plain(args[0]) || !plain(args[1]) || !plain(args[2]) || !as_bool(args[3], &a.causal) ||
      !optional_plain(args[5], &a.lens) || !as_int(args[6], &a.q_offset) || !as_int(args[7], &a.k_offset) ||
      !as_bool(args[8], &need_lse) || !optional_plain(args[9], &out) || !optional_plain(args[10], &lse) ||
      !as_int(args[11], &a.force_path) || !as_int(args[12], &a.kv_chunk) || !no_modes())
    NOT_SERVED();
  const at::Tensor& q = THPVariable_Unpack(args[0]);
  const at::Tensor& k = THPVariable_Unpack(args[1]);
  const at::Tensor& v = THPVariable_Unpack(args[2]);
  if (!shapes_ok(q, k, v) || !as_scale(args[4], q.size(3), &a.scale)) NOT_SERVED();
  if (a.lens.defined() && !lens_ok(a.lens, q)) NOT_SERVED();
  const int64_t B = q.size(0), H = q.size(1), L = q.size(2), Dv = v.size(3);
  if (out.defined() && (out.dim() != 4 || out.size(0) != B || out.size(1) != H || out.size(2) != L || out.size(3) != Dv ||
                        out.scalar_type() != q.scalar_type() || out.device() != q.device()))
    NOT_SERVED();
  if (lse.defined() && (lse.dim() != 3 || lse.size(0) != B || lse.size(1) != H || lse.size(2) != L ||
                        lse.scalar_type() != at::kFloat || lse.device() != q.device()))
    NOT_SERVED();
  const c10::cuda::CUDAGuard guard(q.device());
  if (!out.defined()) out = alloc_like_query(q, {B, H, L, Dv});
  if (!lse.defined() && need_lse) lse = at::empty({B, H, L}, q.options().dtype(at::kFloat));
  if (!forward(q, k, v, a, out, lse)) return nullptr;
  PyObject* po = THPVariable_Wrap(out);
  PyObject* pl = lse.defined() ? THPVariable_Wrap(lse) : Py_NewRef(Py_None);
  return Py_BuildValue("(NN)", po, pl);
  END_HANDLE_TH_ERRORS
}

// decode(query, k_cache, v_cache, block_table, kv_lens, scale, layout, out, lse, need_lse, kv_chunk, k_new, v_new,
//        rope_cos, rope_sin, rope_interleaved) -> (out, lse or None, new_lens or None), or None
// layout: 0 a dense (B, Hkv, S, D) cache, 1 pages (pages, rows, Hkv, D), 2 pages (pages, Hkv, rows, D)
PyObject* py_decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  at::Tensor table, out, lse, k_new, v_new, cos, sin;
  int64_t layout = 0, kv_chunk = 0;
  bool need_lse = false, interleaved = false;
  if (n != 16 || !plain(args[0]) || !plain(args[1]) || !plain(args[2]) || !optional_plain(args[3], &table) ||
      !plain(args[4]) || !as_int(args[6], &layout) || !optional_plain(args[7], &out) || !optional_plain(args[8], &lse) ||
      !as_bool(args[9], &need_lse) || !as_int(args[10], &kv_chunk) || !optional_plain(args[11], &k_new) ||
      !optional_plain(args[12], &v_new) || !optional_plain(args[13], &cos) || !optional_plain(args[14], &sin) ||
      !as_bool(args[15], &interleaved) || !no_modes() || layout < 0 || layout > 2)
    NOT_SERVED();
  const at::Tensor& q = THPVariable_Unpack(args[0]);
  const at::Tensor& k = THPVariable_Unpack(args[1]);
  const at::Tensor& v = THPVariable_Unpack(args[2]);
  const at::Tensor& lens = THPVariable_Unpack(args[4]);
  const auto dt = q.scalar_type();
  if (q.dim() != 4 || q.size(2) != 1 || k.dim() != 4 || v.dim() != 4 || (dt != at::kHalf && dt != at::kBFloat16) ||
      k.scalar_type() != dt || v.scalar_type() != dt || k.device() != q.device() || v.device() != q.device() ||
      k.sizes() != v.sizes() || q.numel() == 0)
    NOT_SERVED();
  const bool paged = layout != 0;
  const int hd = layout == 1 ? 2 : 1, rd = layout == 1 ? 1 : 2;
  const int64_t B = q.size(0), Hq = q.size(1), E = q.size(3), Hkv = k.size(hd);
  if (Hkv == 0 || Hq % Hkv != 0 || k.size(3) != E || !lens_ok(lens, q)) NOT_SERVED();
  if (paged != table.defined() || (!paged && k.size(0) != B)) NOT_SERVED();
  if (paged && (table.scalar_type() != at::kInt || table.dim() != 2 || table.size(0) != B || table.device() != q.device() ||
                !table.is_contiguous()))
    NOT_SERVED();
  float scale = 0.f;
  if (!as_scale(args[5], E, &scale)) NOT_SERVED();
  const int64_t S = paged ? table.size(1) * k.size(rd) : k.size(2);
  if (k_new.defined() != v_new.defined() || cos.defined() != sin.defined() || (cos.defined() && !k_new.defined())) NOT_SERVED();
  for (const at::Tensor* t : {&k_new, &v_new}) {
    if (t->defined() && (t->dim() != 3 || t->size(0) != B || t->size(1) != Hkv || t->size(2) != E || t->scalar_type() != dt ||
                         t->device() != q.device() || t->stride(2) != 1))
      NOT_SERVED();
  }
  for (const at::Tensor* t : {&cos, &sin}) {
    if (t->defined() && (t->scalar_type() != at::kFloat || t->dim() != 2 || t->size(1) < E / 2 || t->stride(1) != 1 ||
                         t->device() != q.device() || t->size(0) < 1 || t->size(0) < S))
      NOT_SERVED();
  }
  if (cos.defined() && (cos.stride(0) != sin.stride(0) || cos.size(0) != sin.size(0))) NOT_SERVED();
  if (out.defined() && (out.sizes() != q.sizes() || out.scalar_type() != dt || out.device() != q.device())) NOT_SERVED();
  if (lse.defined() && (lse.dim() != 3 || lse.size(0) != B || lse.size(1) != Hq || lse.size(2) != 1 ||
                        lse.scalar_type() != at::kFloat || lse.device() != q.device()))
    NOT_SERVED();

  const c10::cuda::CUDAGuard guard(q.device());
  const int dev = q.device().index();
  if (!out.defined()) out = at::empty_like(q);
  if (!lse.defined() && need_lse) lse = at::empty({B, Hq, 1}, q.options().dtype(at::kFloat));
  at::Tensor new_lens;
  B200SdpaParams p{};
  fill_common(p, q, out, lse, dev);
  p.force_path = B200_SDPA_PATH_DECODE;
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  const int order[4] = {0, hd, rd, 3};
  for (int i = 0; i < 4; ++i) {
    p.k_stride[i] = k.stride(order[i]);
    p.v_stride[i] = v.stride(order[i]);
  }
  p.Hkv = static_cast<int32_t>(Hkv);
  p.S = static_cast<int32_t>(S);
  p.Dv = static_cast<int32_t>(E);
  p.scale = scale;
  p.kv_lens = lens.data_ptr<int32_t>();
  p.kv_chunk = static_cast<int32_t>(kv_chunk);
  if (paged) {
    p.block_table = table.data_ptr<int32_t>();
    p.block_table_stride = static_cast<int32_t>(table.size(1));
    p.page_size = static_cast<int32_t>(k.size(rd));
  }
  if (k_new.defined()) {
    p.k_new = k_new.data_ptr();
    p.v_new = v_new.data_ptr();
    for (int i = 0; i < 2; ++i) {
      p.k_new_stride[i] = k_new.stride(i);
      p.v_new_stride[i] = v_new.stride(i);
    }
    if (cos.defined()) {
      p.rope_cos = cos.data_ptr<float>();
      p.rope_sin = sin.data_ptr<float>();
      p.rope_positions = static_cast<int32_t>(cos.size(0));
      p.rope_stride = static_cast<int32_t>(cos.stride(0));
      p.rope_interleaved = interleaved ? 1 : 0;
    }
    new_lens = at::empty_like(lens);
    p.kv_lens_out = new_lens.data_ptr<int32_t>();
  }
  B200SdpaPlan plan{};
  launch(p, dev, true, plan);
  PyObject* po = THPVariable_Wrap(out);
  PyObject* pl = lse.defined() ? THPVariable_Wrap(lse) : Py_NewRef(Py_None);
  PyObject* pn = new_lens.defined() ? THPVariable_Wrap(new_lens) : Py_NewRef(Py_None);
  return Py_BuildValue("(NNN)", po, pl, pn);
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------------------------------
// Rotary embedding
// ---------------------------------------------------------------------------------------------------------------------

// The extents are counted in 32 bits (a broadcast dimension can have more without the memory for it).
bool in_32_bits(const at::Tensor& t) {
  for (int64_t n : t.sizes())
    if (n > 0x7fffffff) return false;
  return true;
}

struct RotaryRest {
  at::Tensor positions, inv_freq;   // (axes, B, L), (B, L) or (L,), extents of 1 broadcast
  std::vector<int64_t> sections;
  bool interleaved = false, inverse = false;
};

// (query', key') of plain CUDA tensors that hold something; key may be undefined.  Throws on a failed launch.
std::array<at::Tensor, 2> rotate(const at::Tensor& query, const at::Tensor& key, const RotaryRest& r) {
  const int dev = query.device().index();
  const c10::cuda::CUDAGuard guard(query.device());
  std::array<at::Tensor, 2> out;
  B200RotaryParams p{};
  p.struct_size = sizeof(p);
  p.dtype = dtype_code(query.scalar_type());
  p.device = dev;
  p.inverse = r.inverse ? 1 : 0;
  const at::Tensor* in[2] = {&query, &key};
  for (int w = 0; w < 2; ++w) {
    if (!in[w]->defined()) continue;
    const at::Tensor& x = *in[w];
    out[w] = alloc_like_query(x, {x.size(0), x.size(1), x.size(2), x.size(3)});
    p.x[w] = x.data_ptr();
    p.y[w] = out[w].data_ptr();
    copy_strides(x, p.x_stride[w]);
    copy_strides(out[w], p.y_stride[w]);
    p.heads[w] = static_cast<int32_t>(x.size(1));
  }
  p.B = static_cast<int32_t>(query.size(0));
  p.L = static_cast<int32_t>(query.size(2));
  p.D = static_cast<int32_t>(query.size(3));
  p.rot = static_cast<int32_t>(2 * r.inv_freq.size(0));
  p.axes = static_cast<int32_t>(r.sections.size());
  p.interleaved = r.interleaved ? 1 : 0;
  for (size_t i = 0; i < r.sections.size(); ++i) p.section[i] = static_cast<int32_t>(r.sections[i]);
  p.positions = r.positions.data_ptr();
  for (int64_t i = 0, pd = r.positions.dim(); i < pd; ++i)
    p.pos_stride[3 - pd + i] = r.positions.size(i) == 1 ? 0 : r.positions.stride(i);   // (dimensions in front: 0)
  p.inv_freq = r.inv_freq.data_ptr();
  p.positions_i64 = r.positions.scalar_type() == at::kLong;
  p.inv_freq_f64 = r.inv_freq.scalar_type() == at::kDouble;
  p.status = device_state(dev).status.data_ptr<int32_t>();
  const int rc = b200_sdpa_rotary(&p, c10::cuda::getCurrentCUDAStream(dev).stream());
  TORCH_CHECK(rc == B200_SDPA_OK, "b200_sdpa_rotary: ", b200_sdpa_strerror(rc));
  return out;
}

// Inside a stream capture a gradient cannot flow to a leaf whose accumulation node was made on the default stream, by an
// eager graph that is still alive: the engine would have the default stream wait for the capture, which ends the capture.
// This runs before that wait, so that the capture itself is still whole when the error reaches its caller.  (A leaf that the pass
// reaches with an undefined gradient is waited for too, one that it leaves out is not.)
void check_leaf_streams() {
  const auto node = torch::autograd::get_current_node();
  if (node == nullptr) return;
  for (uint32_t i = 0; i < node->num_outputs(); ++i) {
    const auto& edge = node->next_edge(i);
    if (!edge.is_valid() || !node->task_should_compute_output(i)) continue;
    if (dynamic_cast<torch::autograd::AccumulateGrad*>(edge.function.get()) == nullptr) continue;
    const auto made_on = edge.function->stream();
    if (!made_on.has_value() || made_on->device_type() != c10::kCUDA) continue;
    const auto now = c10::cuda::getCurrentCUDAStream(made_on->device_index());
    if (*made_on == now.unwrap() || *made_on != c10::cuda::getDefaultCUDAStream(made_on->device_index()).unwrap()) continue;
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    TORCH_CHECK(cudaStreamIsCapturing(now.stream(), &status) == cudaSuccess, "rotary_embedding: the stream's capture could not be queried");
    TORCH_CHECK(status == cudaStreamCaptureStatusNone,
                "rotary_embedding: a captured backward pass reaches a leaf that an eager graph from the default stream still holds; "
                "drop that graph, or build it on the stream that is captured");
  }
}

// A rotation's gradient is the rotation by the opposite angle, itself differentiable.
struct Rotary : torch::autograd::Function<Rotary> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& query, const std::optional<at::Tensor>& key,
                                                const at::Tensor& positions, const at::Tensor& inv_freq, std::vector<int64_t> sections,
                                                bool interleaved, bool inverse) {
    ctx->save_for_backward({positions, inv_freq});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["inverse"] = inverse;
    ctx->set_materialize_grads(false);
    const auto out = rotate(query, key.value_or(at::Tensor()), {positions, inv_freq, std::move(sections), interleaved, inverse});
    if (!key.has_value()) return {out[0]};
    return {out[0], out[1]};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    check_leaf_streams();
    const auto saved = ctx->get_saved_variables();
    const auto sections = ctx->saved_data["sections"].toIntVector();
    const bool interleaved = ctx->saved_data["interleaved"].toBool(), inverse = !ctx->saved_data["inverse"].toBool();
    torch::autograd::variable_list got(7);
    const bool q = grads[0].defined() && ctx->needs_input_grad(0);
    const bool k = grads.size() > 1 && grads[1].defined() && ctx->needs_input_grad(1);
    if (q) {
      auto r = Rotary::apply(grads[0], k ? std::optional<at::Tensor>(grads[1]) : std::nullopt, saved[0], saved[1], sections, interleaved, inverse);
      got[0] = r[0];
      if (k) got[1] = r[1];
    } else if (k) {
      got[1] = Rotary::apply(grads[1], std::optional<at::Tensor>(), saved[0], saved[1], sections, interleaved, inverse)[0];
    }
    return got;
  }
};

// check_leaf_streams(): the same for a backward pass in Python
PyObject* py_check_leaf_streams(PyObject*, PyObject*) {
  HANDLE_TH_ERRORS
  check_leaf_streams();
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// rotary(query, key, positions, inv_freq, sections, interleaved) -> (query', key' or None), or None
PyObject* py_rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  at::Tensor key;
  RotaryRest r;
  if (n != 6 || !plain(args[0]) || !optional_plain(args[1], &key) || !plain(args[2]) || !plain(args[3]) ||
      (args[4] != Py_None && !PyTuple_CheckExact(args[4]) && !PyList_CheckExact(args[4])) || !as_bool(args[5], &r.interleaved) || !no_modes())
    NOT_SERVED();
  const at::Tensor& q = THPVariable_Unpack(args[0]);
  const at::Tensor& positions = THPVariable_Unpack(args[2]);
  r.inv_freq = THPVariable_Unpack(args[3]);
  if (q.dim() != 4 || q.numel() == 0 || dtype_code(q.scalar_type()) < 0 || !in_32_bits(q)) NOT_SERVED();
  const int64_t B = q.size(0), L = q.size(2), D = q.size(3);
  if (key.defined() && (key.dim() != 4 || key.numel() == 0 || key.scalar_type() != q.scalar_type() || key.device() != q.device() ||
                        key.size(0) != B || key.size(2) != L || key.size(3) != D || !in_32_bits(key)))
    NOT_SERVED();
  if ((positions.scalar_type() != at::kInt && positions.scalar_type() != at::kLong) || positions.device() != q.device() ||
      positions.dim() < 1 || positions.dim() > 3)
    NOT_SERVED();
  const int64_t axes = positions.dim() == 3 ? positions.size(0) : 1, pd = positions.dim();
  if ((positions.size(pd - 1) != L && positions.size(pd - 1) != 1) || (pd > 1 && positions.size(pd - 2) != B && positions.size(pd - 2) != 1)) NOT_SERVED();
  if ((r.inv_freq.scalar_type() != at::kFloat && r.inv_freq.scalar_type() != at::kDouble) || r.inv_freq.dim() != 1 ||
      r.inv_freq.device() != q.device() || !r.inv_freq.is_contiguous() || (at::GradMode::is_enabled() && wants_grad(r.inv_freq)))
    NOT_SERVED();
  const int64_t pairs = r.inv_freq.size(0);
  if (pairs < 1 || 2 * pairs > D || axes < 1 || axes > 4) NOT_SERVED();
  if (args[4] == Py_None) {
    if (axes != 1) NOT_SERVED();
    r.sections = {pairs};
  } else {
    int64_t sum = 0;
    if (PySequence_Fast_GET_SIZE(args[4]) != axes) NOT_SERVED();
    for (int64_t i = 0; i < axes; ++i) {
      int64_t v = 0;
      if (!as_int(PySequence_Fast_GET_ITEM(args[4], i), &v) || v < 0 || v > pairs) NOT_SERVED();
      r.sections.push_back(v);
      sum += v;
    }
    if (sum != pairs) NOT_SERVED();
  }
  const bool grad = at::GradMode::is_enabled() && (q.requires_grad() || (key.defined() && key.requires_grad()));
  std::array<at::Tensor, 2> out;
  {
    NoGil nogil;
    r.positions = positions;
    if (grad) {
      auto got = Rotary::apply(q, key.defined() ? std::optional<at::Tensor>(key) : std::nullopt, r.positions, r.inv_freq, r.sections, r.interleaved, false);
      out[0] = got[0];
      if (key.defined()) out[1] = got[1];
    } else {
      out = rotate(q, key, r);
    }
  }
  PyObject* po = THPVariable_Wrap(out[0]);
  PyObject* pk = key.defined() ? THPVariable_Wrap(out[1]) : Py_NewRef(Py_None);
  return Py_BuildValue("(NN)", po, pk);
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------------------------------
// The 8-bit paged cache, and decode under a shared prefix
// ---------------------------------------------------------------------------------------------------------------------

bool scale_ok(const at::Tensor& t, const at::Tensor& pool) {
  return (t.scalar_type() == at::kFloat8_e8m0fnu || t.scalar_type() == at::kByte) && t.dim() == 3 && t.size(0) == pool.size(0) &&
         t.size(1) == pool.size(1) && t.size(2) == pool.size(2) && t.device() == pool.device();
}
bool table_ok(const at::Tensor& t, int64_t B, const at::Tensor& like) {
  return t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == B && t.device() == like.device() && t.is_contiguous();
}
bool vector_ok(const at::Tensor& t, int64_t B, const at::Tensor& like) {
  return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == B && t.device() == like.device() && t.is_contiguous();
}
bool pools_ok(const at::Tensor& k, const at::Tensor& v) {
  return k.dim() == 4 && v.dim() == 4 && k.sizes() == v.sizes() && k.size(0) > 0 && k.device() == v.device() && k.stride(3) == 1 &&
         v.stride(3) == 1 && k.scalar_type() == v.scalar_type();
}
void order(const at::Tensor& t, int hd, int rd, int64_t (&dst)[3]) {
  dst[0] = t.stride(0);
  dst[1] = t.stride(hd);
  dst[2] = t.stride(rd);
}

void fill_rows(B200CacheRowsParams& p, const at::Tensor& key, const at::Tensor& value, const at::Tensor& k, const at::Tensor& v,
               const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& table, int hd, int rd, int dev) {
  p.struct_size = sizeof(p);
  p.dtype = dtype_code(key.scalar_type());
  p.device = dev;
  p.page_size = static_cast<int32_t>(k.size(rd));
  p.k = key.data_ptr();
  p.v = value.data_ptr();
  for (int i = 0; i < 3; ++i) {
    p.k_stride[i] = key.stride(i);
    p.v_stride[i] = value.stride(i);
  }
  p.k_pages = k.data_ptr();
  p.v_pages = v.data_ptr();
  order(k, hd, rd, p.k_pages_stride);
  order(v, hd, rd, p.v_pages_stride);
  p.k_scales = ks.data_ptr();
  p.v_scales = vs.data_ptr();
  order(ks, hd, rd, p.k_scales_stride);
  order(vs, hd, rd, p.v_scales_stride);
  p.B = static_cast<int32_t>(key.size(0));
  p.Hkv = static_cast<int32_t>(key.size(1));
  p.L = static_cast<int32_t>(key.size(2));
  p.D = static_cast<int32_t>(key.size(3));
  p.block_table = table.data_ptr<int32_t>();
  p.block_table_stride = static_cast<int32_t>(table.size(1));
  p.n_pages = static_cast<int32_t>(k.size(0));
  p.status = device_state(dev).status.data_ptr<int32_t>();
}

// paged_write(key, value, k_pages, v_pages, k_scales, v_scales, block_table, start, lens, layout) -> True, or None
PyObject* py_paged_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  at::Tensor lens;
  int64_t layout = 0;
  if (n != 10 || !as_int(args[9], &layout) || layout < 1 || layout > 2 || !optional_plain(args[8], &lens) || !no_modes()) NOT_SERVED();
  for (int i = 0; i < 8; ++i)
    if (!plain(args[i])) NOT_SERVED();
  const at::Tensor& key = THPVariable_Unpack(args[0]);
  const at::Tensor& value = THPVariable_Unpack(args[1]);
  const at::Tensor& k = THPVariable_Unpack(args[2]);
  const at::Tensor& v = THPVariable_Unpack(args[3]);
  const at::Tensor& ks = THPVariable_Unpack(args[4]);
  const at::Tensor& vs = THPVariable_Unpack(args[5]);
  const at::Tensor& table = THPVariable_Unpack(args[6]);
  const at::Tensor& start = THPVariable_Unpack(args[7]);
  const int hd = layout == 1 ? 2 : 1, rd = layout == 1 ? 1 : 2;
  const auto dt = key.scalar_type();
  if (key.dim() != 4 || key.numel() == 0 || !in_32_bits(key) || value.sizes() != key.sizes() || (dt != at::kHalf && dt != at::kBFloat16) ||
      value.scalar_type() != dt || value.device() != key.device() || key.stride(3) != 1 || value.stride(3) != 1 || key.size(3) % 16 != 0 ||
      key.size(3) > 256)
    NOT_SERVED();
  if (!pools_ok(k, v) || k.device() != key.device() || k.scalar_type() != at::kFloat8_e4m3fn || k.size(hd) != key.size(1) ||
      k.size(3) != key.size(3) || !scale_ok(ks, k) || !scale_ok(vs, k))
    NOT_SERVED();
  const int64_t B = key.size(0);
  if (!table_ok(table, B, key) || !vector_ok(start, B, key) || (lens.defined() && !vector_ok(lens, B, key))) NOT_SERVED();
  const c10::cuda::CUDAGuard guard(key.device());
  const int dev = key.device().index();
  B200CacheRowsParams p{};
  fill_rows(p, key, value, k, v, ks, vs, table, hd, rd, dev);
  p.start = start.data_ptr<int32_t>();
  if (lens.defined()) p.lens = lens.data_ptr<int32_t>();
  int rc;
  {
    NoGil nogil;
    rc = b200_sdpa_cache_write(&p, c10::cuda::getCurrentCUDAStream(dev).stream());
  }
  TORCH_CHECK(rc == B200_SDPA_OK, "b200_sdpa_cache_write: ", b200_sdpa_strerror(rc));
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// paged_read(k_pages, v_pages, k_scales, v_scales, block_table, kv_lens, max_len, bf16, layout) -> (key, value), or None
PyObject* py_paged_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t layout = 0, max_len = -1;
  bool bf16 = false;
  if (n != 9 || !as_int(args[8], &layout) || layout < 1 || layout > 2 || !as_bool(args[7], &bf16) ||
      (args[6] != Py_None && !as_int(args[6], &max_len)) || !no_modes())
    NOT_SERVED();
  for (int i = 0; i < 6; ++i)
    if (!plain(args[i])) NOT_SERVED();
  const at::Tensor& k = THPVariable_Unpack(args[0]);
  const at::Tensor& v = THPVariable_Unpack(args[1]);
  const at::Tensor& ks = THPVariable_Unpack(args[2]);
  const at::Tensor& vs = THPVariable_Unpack(args[3]);
  const at::Tensor& table = THPVariable_Unpack(args[4]);
  const at::Tensor& lens = THPVariable_Unpack(args[5]);
  const int hd = layout == 1 ? 2 : 1, rd = layout == 1 ? 1 : 2;
  if (!pools_ok(k, v) || k.scalar_type() != at::kFloat8_e4m3fn || !scale_ok(ks, k) || !scale_ok(vs, k) || table.dim() != 2) NOT_SERVED();
  const int64_t B = table.size(0), H = k.size(hd), D = k.size(3), capacity = table.size(1) * k.size(rd);
  if (!table_ok(table, B, k) || !vector_ok(lens, B, k) || D % 16 != 0 || D < 16 || D > 256) NOT_SERVED();
  const int64_t L = args[6] == Py_None ? capacity : max_len;
  if (L < 1 || L > capacity || B < 1 || H < 1) NOT_SERVED();
  const c10::cuda::CUDAGuard guard(k.device());
  const int dev = k.device().index();
  const auto options = k.options().dtype(bf16 ? at::kBFloat16 : at::kHalf);
  at::Tensor key = at::empty({B, H, L, D}, options), value = at::empty({B, H, L, D}, options);
  B200CacheRowsParams p{};
  fill_rows(p, key, value, k, v, ks, vs, table, hd, rd, dev);
  p.lens = lens.data_ptr<int32_t>();
  int rc;
  {
    NoGil nogil;
    rc = b200_sdpa_cache_read(&p, c10::cuda::getCurrentCUDAStream(dev).stream());
  }
  TORCH_CHECK(rc == B200_SDPA_OK, "b200_sdpa_cache_read: ", b200_sdpa_strerror(rc));
  PyObject* pk = THPVariable_Wrap(key);
  PyObject* pv = THPVariable_Wrap(value);
  return Py_BuildValue("(NN)", pk, pv);
  END_HANDLE_TH_ERRORS
}

// cache_decode(query, k_pages, v_pages, k_scales, v_scales, prefix_table, prefix_len, block_table, kv_lens, scale, layout, out, lse,
//              need_lse, kv_chunk) -> (out, lse or None), or None
PyObject* py_cache_decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  at::Tensor ks, vs, prefix, out, lse;
  int64_t prefix_len = 0, layout = 0, kv_chunk = 0;
  bool need_lse = false;
  if (n != 15 || !plain(args[0]) || !plain(args[1]) || !plain(args[2]) || !optional_plain(args[3], &ks) || !optional_plain(args[4], &vs) ||
      !optional_plain(args[5], &prefix) || !as_int(args[6], &prefix_len) || !plain(args[7]) || !plain(args[8]) || !as_int(args[10], &layout) ||
      layout < 1 || layout > 2 || !optional_plain(args[11], &out) || !optional_plain(args[12], &lse) || !as_bool(args[13], &need_lse) ||
      !as_int(args[14], &kv_chunk) || !no_modes())
    NOT_SERVED();
  const at::Tensor& q = THPVariable_Unpack(args[0]);
  const at::Tensor& k = THPVariable_Unpack(args[1]);
  const at::Tensor& v = THPVariable_Unpack(args[2]);
  const at::Tensor& table = THPVariable_Unpack(args[7]);
  const at::Tensor& lens = THPVariable_Unpack(args[8]);
  const int hd = layout == 1 ? 2 : 1, rd = layout == 1 ? 1 : 2;
  const auto dt = q.scalar_type();
  if (q.dim() != 4 || q.size(2) != 1 || q.numel() == 0 || (dt != at::kHalf && dt != at::kBFloat16) || !pools_ok(k, v) || k.device() != q.device())
    NOT_SERVED();
  const bool quantised = ks.defined();
  if (ks.defined() != vs.defined() || (!quantised && prefix_len <= 0) || prefix_len < 0) NOT_SERVED();
  if (quantised ? (k.scalar_type() != at::kFloat8_e4m3fn || !scale_ok(ks, k) || !scale_ok(vs, k)) : k.scalar_type() != dt) NOT_SERVED();
  const int64_t B = q.size(0), Hq = q.size(1), D = q.size(3), Hkv = k.size(hd);
  if (k.size(3) != D || (D != 64 && D != 128) || Hkv == 0 || Hq % Hkv != 0) NOT_SERVED();
  if (!table_ok(table, B, q) || !vector_ok(lens, B, q)) NOT_SERVED();
  if (prefix_len > 0 && (!prefix.defined() || prefix.scalar_type() != at::kInt || prefix.dim() != 1 || prefix.device() != q.device() ||
                         !prefix.is_contiguous() || prefix.size(0) * k.size(rd) < prefix_len || prefix_len > 0x7fffffff))
    NOT_SERVED();
  if (prefix_len > 0 && (reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 != 0 || q.stride(3) != 1 || q.stride(0) <= 0 || q.stride(1) <= 0 ||
                         q.stride(0) % 8 != 0 || q.stride(1) % 8 != 0))
    NOT_SERVED();
  float scale = 0.f;
  if (!as_scale(args[9], D, &scale)) NOT_SERVED();
  if (out.defined() && (out.sizes() != q.sizes() || out.scalar_type() != dt || out.device() != q.device())) NOT_SERVED();
  if (lse.defined() && (lse.dim() != 3 || lse.size(0) != B || lse.size(1) != Hq || lse.size(2) != 1 || lse.scalar_type() != at::kFloat ||
                        lse.device() != q.device()))
    NOT_SERVED();
  const c10::cuda::CUDAGuard guard(q.device());
  const int dev = q.device().index();
  if (!out.defined()) out = at::empty_like(q);
  if (!lse.defined() && need_lse) lse = at::empty({B, Hq, 1}, q.options().dtype(at::kFloat));
  B200CacheDecodeParams p{};
  p.struct_size = sizeof(p);
  p.dtype = dtype_code(dt);
  p.device = dev;
  p.page_size = static_cast<int32_t>(k.size(rd));
  p.q = q.data_ptr();
  p.out = out.data_ptr();
  const int dims[3] = {0, 1, 3};
  for (int i = 0; i < 3; ++i) {
    p.q_stride[i] = q.stride(dims[i]);
    p.out_stride[i] = out.stride(dims[i]);
  }
  if (lse.defined()) {
    p.lse = lse.data_ptr<float>();
    p.lse_stride[0] = lse.stride(0);
    p.lse_stride[1] = lse.stride(1);
  }
  p.k_pages = k.data_ptr();
  p.v_pages = v.data_ptr();
  order(k, hd, rd, p.k_pages_stride);
  order(v, hd, rd, p.v_pages_stride);
  if (quantised) {
    p.k_scales = ks.data_ptr();
    p.v_scales = vs.data_ptr();
    order(ks, hd, rd, p.k_scales_stride);
    order(vs, hd, rd, p.v_scales_stride);
  }
  p.B = static_cast<int32_t>(B);
  p.Hq = static_cast<int32_t>(Hq);
  p.Hkv = static_cast<int32_t>(Hkv);
  p.D = static_cast<int32_t>(D);
  p.scale = scale;
  p.n_pages = static_cast<int32_t>(k.size(0));
  p.kv_lens = lens.data_ptr<int32_t>();
  p.block_table_stride = static_cast<int32_t>(table.size(1));
  if (table.size(1) > 0) p.block_table = table.data_ptr<int32_t>();
  p.prefix_len = static_cast<int32_t>(prefix_len);
  if (prefix_len > 0) p.prefix_table = prefix.data_ptr<int32_t>();
  p.kv_chunk = static_cast<int32_t>(kv_chunk);
  p.status = device_state(dev).status.data_ptr<int32_t>();
  at::Tensor ws;   // freed (stream-ordered) when the launches have been queued
  {
    NoGil nogil;
    B200SdpaPlan plan{};
    plan.struct_size = sizeof(plan);
    int rc = b200_sdpa_cache_decode_plan(&p, &plan);
    TORCH_CHECK(rc == B200_SDPA_OK, "b200_sdpa_cache_decode_plan: ", b200_sdpa_strerror(rc));
    if (plan.workspace_bytes != 0) {
      ws = scratch(dev, plan.workspace_bytes);
      p.workspace = ws.data_ptr();
      p.workspace_bytes = static_cast<uint64_t>(ws.numel());
    }
    rc = b200_sdpa_cache_decode(&p, c10::cuda::getCurrentCUDAStream(dev).stream());
    TORCH_CHECK(rc == B200_SDPA_OK, "b200_sdpa_cache_decode: ", b200_sdpa_strerror(rc));
  }
  PyObject* po = THPVariable_Wrap(out);
  PyObject* pl = lse.defined() ? THPVariable_Wrap(lse) : Py_NewRef(Py_None);
  return Py_BuildValue("(NN)", po, pl);
  END_HANDLE_TH_ERRORS
}

// set_plan_record(dict): where every forward made here leaves its plan
PyObject* py_set_plan_record(PyObject*, PyObject* record) {
  if (!PyDict_CheckExact(record)) {
    PyErr_SetString(PyExc_TypeError, "set_plan_record: a dict");
    return nullptr;
  }
  PyObject* old = g_plan_record;
  g_plan_record = Py_NewRef(record);
  Py_XDECREF(old);
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_attention)), METH_FASTCALL, nullptr},
    {"forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_forward)), METH_FASTCALL, nullptr},
    {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_decode)), METH_FASTCALL, nullptr},
    {"rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_rotary)), METH_FASTCALL, nullptr},
    {"check_leaf_streams", reinterpret_cast<PyCFunction>(py_check_leaf_streams), METH_NOARGS, nullptr},
    {"paged_write", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_paged_write)), METH_FASTCALL, nullptr},
    {"paged_read", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_paged_read)), METH_FASTCALL, nullptr},
    {"cache_decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_cache_decode)), METH_FASTCALL, nullptr},
    {"set_plan_record", py_set_plan_record, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&kModule); }
