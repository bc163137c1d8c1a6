// The Python wrappers' ordinary calls without their host work: argument checks, allocations and args structs of lq_zoo_simple_gla,
// lq_zoo_chunk_forward, lq_zoo_rotate_qkv, lq_split_rotate_quant_xBC, lq_ssd_combined and the serving entry points in native code.  Each function serves the
// ordinary form of its call (plain tensors on the current GPU, fp32 scales, shapes that need no padding) and returns None for any other,
// and for what is to be refused: the caller then takes the wrapper's general path, which converts, pads, copies or raises.  Nothing is
// kept from one call for the next.
//
// Host time of a call on one machine, general path -> here (the C entry with its launches in brackets): Mamba-2 cell B1 T2048 H8 26.5 ->
// 10.1 us (7.3 for two launches), KDA B1 T2048 H8 26.6 -> 10.3 (6.6), SSD layer B1 L512 H80, prologue and forward, 56 -> 25.3 (20.6 for
// five).  That was longer than the kernels of the first and the last (17 and 30 us): a ctypes struct of 30 to 60 fields, their conversions
// and attribute reads of tensors.  Whole calls 24.1 -> 16.7 and 52.3 -> 28.0.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/PythonTorchFunctionTLS.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <utility>
#include <vector>

#include "../../include/linquant_hip.h"

namespace {

// set once, while the module is loaded: entry points of liblinquant_hip.so and the function that raises for a failed call
decltype(&lq_zoo_simple_gla) simple_gla_entry;
decltype(&lq_zoo_simple_gla_workspace_bytes) simple_gla_bytes;
decltype(&lq_zoo_chunk_forward) chunk_forward_entry;
decltype(&lq_zoo_chunk_forward_workspace_bytes) chunk_forward_bytes;
decltype(&lq_zoo_rotate_qkv) rotate_entry;
decltype(&lq_split_rotate_quant_xBC) split_rotate_entry;
decltype(&lq_ssd_combined) ssd_entry;
decltype(&lq_ssd_combined_workspace_bytes) ssd_bytes;
decltype(&lq_quantize_rows) quantize_entry;
decltype(&lq_int8_matmul) matmul_entry;
decltype(&lq_residual_rmsnorm) norm_entry;
decltype(&lq_conv1d_prompt) conv_prompt_entry;
decltype(&lq_conv1d_step) conv_step_entry;
decltype(&lq_ssm_prompt) ssm_prompt_entry;
decltype(&lq_ssm_prompt_workspace_bytes) ssm_prompt_bytes;
decltype(&lq_ssm_step) ssm_step_entry;
decltype(&lq_linear_attention_prompt) attention_prompt_entry;
decltype(&lq_linear_attention_prompt_workspace_bytes) attention_prompt_bytes;
decltype(&lq_linear_attention_step) attention_step_entry;
decltype(&lq_groupnorm_gated) groupnorm_entry;
decltype(&lq_adapter_down) adapter_down_entry;
decltype(&lq_copy_slots) copy_slots_entry;
PyObject* raise_failed;

using at::ScalarType;
using at::Tensor;

// a plain tensor with memory of its own on the GPU of the call
bool plain(PyObject* o, const c10::Device& dev, Tensor& t) {
  if (!THPVariable_CheckExact(o)) return false;
  t = THPVariable_Unpack(o);
  return t.defined() && t.layout() == at::kStrided && t.unsafeGetTensorImpl()->has_storage() && t.device() == dev;
}
bool optional(PyObject* o, const c10::Device& dev, Tensor& t) { return o == Py_None || plain(o, dev, t); }

bool aligned(const Tensor& t, uintptr_t n = 16) { return (uintptr_t)t.const_data_ptr() % n == 0; }

// dense fp32 with `numel` entries
bool table(const Tensor& t, int64_t numel, uintptr_t align = 4) {
  return t.scalar_type() == ScalarType::Float && t.is_contiguous() && t.numel() == numel && aligned(t, align);
}
const float* f32(const Tensor& t) { return t.defined() ? (const float*)t.const_data_ptr() : nullptr; }

bool number(PyObject* o, double& x) {
  if (PyFloat_CheckExact(o)) return x = PyFloat_AS_DOUBLE(o), true;
  if (!PyLong_CheckExact(o)) return false;
  x = PyLong_AsDouble(o);
  return !(x == -1.0 && PyErr_Occurred() && (PyErr_Clear(), true));
}
bool integer(PyObject* o, int64_t& x) {
  if (!PyLong_CheckExact(o)) return false;
  x = PyLong_AsLongLong(o);
  return !(x == -1 && PyErr_Occurred() && (PyErr_Clear(), true)) && x >= 0 && x <= INT_MAX;
}
bool fits(at::IntArrayRef s) {
  for (const int64_t n : s)
    if (n <= 0 || n > INT_MAX) return false;
  return true;
}

// the GPU of the first tensor, if it is the current one and nothing watches the operators of this thread
bool device_of(PyObject* o, c10::Device& dev) {
  if (!THPVariable_CheckExact(o)) return false;
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.get_device() != c10::hip::current_device()) return false;
  if (c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::PythonTorchFunctionTLS::stack_len() > 0) return false;
  dev = t.device();
  return true;
}
hipStream_t stream_of(const c10::Device& dev) { return c10::hip::getCurrentHIPStream(dev.index()).stream(); }

Tensor empty(at::IntArrayRef size, ScalarType dt, const c10::Device& dev) { return at::empty(size, at::TensorOptions().dtype(dt).device(dev)); }

PyObject* failed(const char* entry, int rc) {
  PyObject* r = PyObject_CallFunction(raise_failed, "si", entry, rc);  // raises
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, entry);
  return nullptr;
}

// q, k, v of a zoo call: dense, one 16-bit type, whole 64-token chunks, widths that need no padding
bool operands(const Tensor& q, const Tensor& k, const Tensor& v) {
  const ScalarType act = v.scalar_type();
  if ((act != ScalarType::Half && act != ScalarType::BFloat16) || q.scalar_type() != act || k.scalar_type() != act) return false;
  if (q.dim() != 4 || v.dim() != 4 || k.sizes() != q.sizes() || !fits(q.sizes()) || !fits(v.sizes())) return false;
  for (int i = 0; i < 3; ++i)
    if (v.size(i) != q.size(i)) return false;
  if (q.size(1) % 64 != 0 || (q.size(3) != 64 && q.size(3) != 128) || v.size(3) % 64 != 0) return false;
  return q.is_contiguous() && k.is_contiguous() && v.is_contiguous();
}
// `n` scales of a call's dict by role; their entries
bool scales(PyObject* dict, const c10::Device& dev, const char* const* names, const int64_t* sizes, int n, int unaligned, Tensor* sc) {
  if (!PyDict_CheckExact(dict)) return false;
  for (int i = 0; i < n; ++i) {
    PyObject* o = PyDict_GetItemString(dict, names[i]);
    if (!o || !plain(o, dev, sc[i]) || !table(sc[i], sizes[i], i < unaligned ? 4 : 16)) return false;
  }
  return true;
}
bool output_type(PyObject* o, ScalarType act, ScalarType& ot) {
  ot = act;
  if (o == Py_None) return true;
  if (!THPDtype_Check(o)) return false;
  ot = ((THPDtype*)o)->scalar_type;
  return ot == act || ot == ScalarType::Float;
}

// ---- simple_gla(q, k, v, g, scales, eta, scale, final_state, bits, out_dtype, prologue): chunk_simple_gla_int8, chunks of 64 tokens
PyObject* simple_gla(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11) Py_RETURN_NONE;
  c10::Device dev(c10::DeviceType::CPU);
  Tensor q, k, v, g, sc[6], sg_qk, sg_v;
  if (!device_of(arg[0], dev) || !plain(arg[0], dev, q) || !plain(arg[1], dev, k) || !plain(arg[2], dev, v) || !optional(arg[3], dev, g)) Py_RETURN_NONE;
  if (!operands(q, k, v)) Py_RETURN_NONE;
  const ScalarType act = v.scalar_type();
  const int64_t B = q.size(0), T = q.size(1), H = q.size(2), K = q.size(3), V = v.size(3);
  if (g.defined() && (g.dim() != 3 || g.size(0) != B || g.size(1) != T || g.size(2) != H || !table(g, B * T * H))) Py_RETURN_NONE;
  static const char* const names[6] = {"q", "k", "kw", "vw", "vl", "state"};
  const int64_t sizes[6] = {H, H, H * K, H * V, H * V, H * V};
  if (!scales(arg[4], dev, names, sizes, 6, 2, sc)) Py_RETURN_NONE;
  double eta, scale = 0.0;
  int64_t bits;
  if (!number(arg[5], eta) || !(arg[6] == Py_None || number(arg[6], scale)) || !integer(arg[8], bits) || bits < 2 || bits > 8) Py_RETURN_NONE;
  if (arg[6] == Py_None) scale = std::pow((double)K, -0.5);
  const int final_state = PyObject_IsTrue(arg[7]);
  if (final_state < 0) return nullptr;
  ScalarType ot;
  if (!output_type(arg[9], act, ot)) Py_RETURN_NONE;
  if (arg[10] != Py_None) {  // the rotations; with D_QK (whose reciprocals are a tensor operation) the general path
    if (!PyDict_CheckExact(arg[10]) || (V != 64 && V != 128)) Py_RETURN_NONE;
    PyObject *key, *value;
    for (Py_ssize_t at = 0; PyDict_Next(arg[10], &at, &key, &value);) {
      if (!PyUnicode_CheckExact(key)) Py_RETURN_NONE;
      const bool qk = PyUnicode_CompareWithASCIIString(key, "signs_qk") == 0;
      if (!qk && PyUnicode_CompareWithASCIIString(key, "signs_v") != 0) Py_RETURN_NONE;
      Tensor& t = qk ? sg_qk : sg_v;
      if (!optional(value, dev, t) || (t.defined() && !table(t, qk ? K : V, 16))) Py_RETURN_NONE;
    }
  }
  lq_zoo_simple_gla_args a = {};
  a.q = q.const_data_ptr(), a.k = k.const_data_ptr(), a.v = v.const_data_ptr(), a.g = f32(g);
  a.sq = f32(sc[0]), a.sk = f32(sc[1]), a.skw = f32(sc[2]), a.svw = f32(sc[3]), a.svl = f32(sc[4]), a.ss = f32(sc[5]);
  a.eta = (float)eta, a.scale = (float)scale, a.qmax = (1 << (bits - 1)) - 1;
  a.batch = (int)B, a.seqlen = (int)T, a.nheads = (int)H, a.kdim = (int)K, a.vdim = (int)V, a.chunk_size = 64;
  a.act_dtype = act == ScalarType::BFloat16 ? LQ_DT_BF16 : LQ_DT_F16;
  a.signs_qk = f32(sg_qk), a.signs_v = f32(sg_v);
  int64_t bytes = 0;
  if (simple_gla_bytes(&a, &bytes) != 0) Py_RETURN_NONE;
  Tensor o, ht;
  int rc;
  {
    pybind11::gil_scoped_release no_gil;
    Tensor ws = empty({bytes}, ScalarType::Byte, dev);
    o = empty(v.sizes(), ot, dev);
    if (final_state) ht = empty({B, H, K, V}, ScalarType::Float, dev);
    a.o = o.data_ptr(), a.o_is_f32 = ot == ScalarType::Float, a.ht = final_state ? (float*)ht.data_ptr() : nullptr;
    a.workspace = ws.data_ptr(), a.workspace_bytes = bytes;
    rc = simple_gla_entry(&a, stream_of(dev));
  }
  if (rc != 0) return failed("lq_zoo_simple_gla", rc);
  PyObject* po = THPVariable_Wrap(o);
  PyObject* ph = final_state ? THPVariable_Wrap(ht) : (Py_INCREF(Py_None), Py_None);
  return Py_BuildValue("(NN)", po, ph);
  END_HANDLE_TH_ERRORS
}

// ---- chunk_forward(q, k, v, g, beta, scales, sigma, tau, eta, scale, final_state, bits, out_dtype, rot, dqk): chunk_gla_int8 (beta None),
// chunk_delta_int8 and chunk_kda_int8, chunks of 64 tokens
PyObject* chunk_forward(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 15) Py_RETURN_NONE;
  c10::Device dev(c10::DeviceType::CPU);
  Tensor q, k, v, g, beta, sc[7], rot, dqk;
  if (!device_of(arg[0], dev) || !plain(arg[0], dev, q) || !plain(arg[1], dev, k) || !plain(arg[2], dev, v) || !optional(arg[3], dev, g) ||
      !optional(arg[4], dev, beta) || !optional(arg[13], dev, rot) || !optional(arg[14], dev, dqk))
    Py_RETURN_NONE;
  if (!operands(q, k, v)) Py_RETURN_NONE;
  const ScalarType act = v.scalar_type();
  const int64_t B = q.size(0), T = q.size(1), H = q.size(2), K = q.size(3), V = v.size(3);
  const bool delta = beta.defined(), diag = g.defined() && g.dim() == 4;
  if (delta && (beta.dim() != 3 || beta.size(0) != B || beta.size(1) != T || !table(beta, B * T * H))) Py_RETURN_NONE;
  if (diag ? g.sizes() != q.sizes() || !table(g, B * T * H * K, 16)
           : !delta || (g.defined() && (g.dim() != 3 || g.size(0) != B || g.size(1) != T || !table(g, B * T * H))))
    Py_RETURN_NONE;
  if (rot.defined() && (!diag || rot.dim() != 2 || rot.size(0) != K || rot.size(1) != K || !rot.is_contiguous() || !aligned(rot) ||
                        (rot.scalar_type() != ScalarType::Float && rot.scalar_type() != ScalarType::Half)))
    Py_RETURN_NONE;
  if (dqk.defined() && (!delta || !diag || dqk.dim() != 2 || dqk.size(0) != H || !table(dqk, H * K, 16))) Py_RETURN_NONE;
  static const char* const linear_names[] = {"q", "k", "vw", "kw", "vl", "state"};
  static const char* const delta_names[] = {"q", "k", "ew", "kw", "el", "state", "w"};
  const int64_t sizes[7] = {H, H, H * V, H * K, H * V, H * V, H};
  if (!scales(arg[5], dev, delta ? delta_names : linear_names, sizes, 6, 3, sc)) Py_RETURN_NONE;
  if (delta && !scales(arg[5], dev, delta_names + 6, sizes + 6, 1, 1, sc + 6)) Py_RETURN_NONE;
  double sigma, tau, eta, scale = 0.0;
  int64_t bits;
  if (!number(arg[6], sigma) || !number(arg[7], tau) || !number(arg[8], eta) || !(arg[9] == Py_None || number(arg[9], scale)) || !integer(arg[11], bits) ||
      bits < 2 || bits > 8)
    Py_RETURN_NONE;
  if (arg[9] == Py_None) scale = std::pow((double)K, -0.5);
  const int final_state = PyObject_IsTrue(arg[10]);
  if (final_state < 0) return nullptr;
  ScalarType ot;
  if (!output_type(arg[12], act, ot)) Py_RETURN_NONE;
  lq_zoo_chunk_forward_args a = {};
  a.q = q.const_data_ptr(), a.k = k.const_data_ptr(), a.v = v.const_data_ptr(), a.g = f32(g), a.beta = f32(beta);
  a.sq = f32(sc[0]), a.sk = f32(sc[1]), a.svw = f32(sc[2]), a.skw = f32(sc[3]), a.svl = f32(sc[4]), a.ss = f32(sc[5]), a.sw = f32(sc[6]);
  if (rot.defined() && rot.scalar_type() == ScalarType::Float) a.rot_f32 = f32(rot);
  else if (rot.defined()) a.rot = rot.const_data_ptr();
  a.dqk = f32(dqk);
  a.sigma = (float)sigma, a.tau = (float)tau, a.eta = (float)eta, a.scale = (float)scale, a.qmax = (1 << (bits - 1)) - 1;
  a.family = delta ? LQ_FAMILY_DELTA : LQ_FAMILY_LINEAR, a.decay = diag ? LQ_DECAY_DIAGONAL : (g.defined() ? LQ_DECAY_SCALAR : LQ_DECAY_NONE);
  a.batch = (int)B, a.seqlen = (int)T, a.nheads = (int)H, a.kdim = (int)K, a.vdim = (int)V, a.chunk_size = 64;
  a.act_dtype = act == ScalarType::BFloat16 ? LQ_DT_BF16 : LQ_DT_F16;
  int64_t bytes = 0;
  if (chunk_forward_bytes(&a, &bytes) != 0) Py_RETURN_NONE;
  Tensor o, ht;
  int rc;
  {
    pybind11::gil_scoped_release no_gil;
    Tensor ws = empty({bytes + (rot.defined() ? 2 * K * K : 0)}, ScalarType::Byte, dev);
    o = empty(v.sizes(), ot, dev);
    if (final_state) ht = empty({B, H, K, V}, ScalarType::Float, dev);
    a.o = o.data_ptr(), a.o_is_f32 = ot == ScalarType::Float, a.ht = final_state ? (float*)ht.data_ptr() : nullptr;
    a.workspace = ws.data_ptr(), a.workspace_bytes = bytes;
    if (rot.defined()) a.rot_ws = (char*)ws.data_ptr() + bytes;
    rc = chunk_forward_entry(&a, stream_of(dev));
  }
  if (rc != 0) return failed("lq_zoo_chunk_forward", rc);
  PyObject* po = THPVariable_Wrap(o);
  PyObject* ph = final_state ? THPVariable_Wrap(ht) : (Py_INCREF(Py_None), Py_None);
  return Py_BuildValue("(NN)", po, ph);
  END_HANDLE_TH_ERRORS
}

// ---- rotate_qkv(q, k, v, signs_qk, signs_v): rotate_qkv into new tensors, without D_QK
PyObject* rotate_qkv(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) Py_RETURN_NONE;
  c10::Device dev(c10::DeviceType::CPU);
  Tensor in[3], sg_qk, sg_v, out[3];
  PyObject* first = arg[0] != Py_None ? arg[0] : (arg[1] != Py_None ? arg[1] : arg[2]);
  if (!device_of(first, dev) || !optional(arg[3], dev, sg_qk) || !optional(arg[4], dev, sg_v)) Py_RETURN_NONE;
  const Tensor& ref = THPVariable_Unpack(first);
  if (ref.dim() != 4 || (ref.scalar_type() != ScalarType::Half && ref.scalar_type() != ScalarType::BFloat16)) Py_RETURN_NONE;
  for (int i = 0; i < 3; ++i) {
    if (!optional(arg[i], dev, in[i])) Py_RETURN_NONE;
    const Tensor& t = in[i];
    if (!t.defined()) continue;
    if (t.dim() != 4 || t.scalar_type() != ref.scalar_type() || !t.is_contiguous() || !fits(t.sizes()) || (t.size(3) != 64 && t.size(3) != 128)) Py_RETURN_NONE;
    for (int d = 0; d < 3; ++d)
      if (t.size(d) != ref.size(d)) Py_RETURN_NONE;
  }
  if (in[0].defined() && in[1].defined() && in[0].size(3) != in[1].size(3)) Py_RETURN_NONE;
  const int64_t K = in[0].defined() ? in[0].size(3) : (in[1].defined() ? in[1].size(3) : 0), V = in[2].defined() ? in[2].size(3) : 0;
  if ((sg_qk.defined() && !table(sg_qk, K, 16)) || (sg_v.defined() && !table(sg_v, V, 16))) Py_RETURN_NONE;
  lq_zoo_rotate_qkv_args a = {};
  int rc;
  {
    pybind11::gil_scoped_release no_gil;
    for (int i = 0; i < 3; ++i)
      if (in[i].defined()) out[i] = empty(in[i].sizes(), in[i].scalar_type(), dev);
    auto at = [](const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; };
    a.q = at(in[0]), a.k = at(in[1]), a.v = at(in[2]);
    a.q_out = const_cast<void*>(at(out[0])), a.k_out = const_cast<void*>(at(out[1])), a.v_out = const_cast<void*>(at(out[2]));
    a.signs_qk = f32(sg_qk), a.signs_v = f32(sg_v);
    a.batch = (int)ref.size(0), a.seqlen = (int)ref.size(1), a.nheads = (int)ref.size(2), a.kdim = (int)K, a.vdim = (int)V;
    a.act_dtype = ref.scalar_type() == ScalarType::BFloat16 ? LQ_DT_BF16 : LQ_DT_F16;
    rc = rotate_entry(&a, stream_of(dev));
  }
  if (rc != 0) return failed("lq_zoo_rotate_qkv", rc);
  PyObject* o[3];
  for (int i = 0; i < 3; ++i) o[i] = in[i].defined() ? THPVariable_Wrap(out[i]) : (Py_INCREF(Py_None), Py_None);
  return Py_BuildValue("(NNN)", o[0], o[1], o[2]);
  END_HANDLE_TH_ERRORS
}

// ---- split_rotate(xBC, r_signs, nheads, ngroups, d_state, headdim, B_inv_scale, C_inv_scale, return_b_fp, return_b_rowmax):
// fused_split_rotate_quant_xBC without D_QK
PyObject* split_rotate(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10) Py_RETURN_NONE;
  c10::Device dev(c10::DeviceType::CPU);
  Tensor xBC, signs, binv, cinv;
  int64_t H, G, N, P;
  if (!device_of(arg[0], dev) || !plain(arg[0], dev, xBC) || !optional(arg[1], dev, signs) || !plain(arg[6], dev, binv) || !plain(arg[7], dev, cinv)) Py_RETURN_NONE;
  if (!integer(arg[2], H) || !integer(arg[3], G) || !integer(arg[4], N) || !integer(arg[5], P)) Py_RETURN_NONE;
  const int want_fp = PyObject_IsTrue(arg[8]), want_max = PyObject_IsTrue(arg[9]);
  if (want_fp < 0 || want_max < 0) return nullptr;
  if (xBC.dim() != 3 || xBC.scalar_type() != ScalarType::Half || !fits(xBC.sizes()) || xBC.stride(2) != 1) Py_RETURN_NONE;
  const int64_t B = xBC.size(0), T = xBC.size(1), d_ssm = H * P;
  if ((N != 64 && N != 128) || G <= 0 || d_ssm <= 0 || xBC.size(2) != d_ssm + 2 * G * N || (want_max && !want_fp)) Py_RETURN_NONE;
  if (!table(binv, G) || !table(cinv, G)) Py_RETURN_NONE;
  int signs_dtype = 0;
  if (signs.defined()) {
    const ScalarType st = signs.scalar_type();
    if ((st != ScalarType::Half && st != ScalarType::Float && st != ScalarType::Char) || !signs.is_contiguous() || signs.numel() != G * N) Py_RETURN_NONE;
    signs_dtype = st == ScalarType::Half ? LQ_DT_F16 : (st == ScalarType::Float ? LQ_DT_F32 : LQ_DT_I8);
  }
  Tensor x, qB, qC, b_fp, b_max;
  lq_split_rotate_quant_xBC_args a = {};
  int rc;
  {
    pybind11::gil_scoped_release no_gil;
    x = xBC.slice(2, 0, d_ssm).view({B, T, H, P});
    qB = empty({B, T, G, N}, ScalarType::Char, dev), qC = empty({B, T, G, N}, ScalarType::Char, dev);
    if (want_fp) b_fp = empty({B, T, G, N}, ScalarType::Half, dev);
    if (want_max) b_max = empty({B, T, G}, ScalarType::Float, dev);
    a.xBC = xBC.const_data_ptr(), a.xBC_stride_b = xBC.stride(0), a.xBC_stride_t = xBC.stride(1);
    a.qB = (int8_t*)qB.data_ptr(), a.qC = (int8_t*)qC.data_ptr(), a.b_fp = want_fp ? b_fp.data_ptr() : nullptr;
    a.signs = signs.defined() ? signs.const_data_ptr() : nullptr, a.signs_dtype = signs_dtype;
    a.B_inv_scale = f32(binv), a.C_inv_scale = f32(cinv);
    a.batch = (int)B, a.seqlen = (int)T, a.d_ssm = (int)d_ssm, a.ngroups = (int)G, a.dstate = (int)N;
    a.b_rowmax = want_max ? (float*)b_max.data_ptr() : nullptr;
    rc = split_rotate_entry(&a, stream_of(dev));
  }
  if (rc != 0) return failed("lq_split_rotate_quant_xBC", rc);
  PyObject *px = THPVariable_Wrap(x), *pb = THPVariable_Wrap(qB), *pc = THPVariable_Wrap(qC);
  if (want_max) return Py_BuildValue("(NNNNN)", px, pb, pc, THPVariable_Wrap(b_fp), THPVariable_Wrap(b_max));
  if (want_fp) return Py_BuildValue("(NNNN)", px, pb, pc, THPVariable_Wrap(b_fp));
  return Py_BuildValue("(NNN)", px, pb, pc);
  END_HANDLE_TH_ERRORS
}

bool scalar(const Tensor& t) { return t.scalar_type() == ScalarType::Float && t.numel() == 1; }
bool rows(const Tensor& t, int64_t B, int64_t L, ScalarType st) {  // (B, L, *, *) with dense rows
  return t.dim() == 4 && t.size(0) == B && t.size(1) == L && t.scalar_type() == st && t.stride(3) == 1 && fits(t.sizes());
}

// ---- ssd(x, dt, dt_scale, A_log, A_log_scale, q_B, B_scale, q_C, C_scale, chunk_size, D, D_scale, dt_bias, dt_softplus, dt_limit,
// state_scale, cb_scale, alpha_hp, bscale_g, keyside, x_scale_hp, b_fp, b_gate_scale, b_rowmax, gate_shift): the SSD forward
PyObject* ssd(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 25) Py_RETURN_NONE;
  c10::Device dev(c10::DeviceType::CPU);
  Tensor x, dt, dts, A, als, qB, Bs, qC, Cs, D, dsc, bias, ss, cbs, alpha, bsg, xs, bfp, bgs, bmax;
  if (!device_of(arg[0], dev)) Py_RETURN_NONE;
  const int keyside = PyObject_IsTrue(arg[19]), softplus = PyObject_IsTrue(arg[13]);
  if (keyside < 0 || softplus < 0) return nullptr;
  if (!plain(arg[0], dev, x) || !plain(arg[1], dev, dt) || !plain(arg[2], dev, dts) || !plain(arg[3], dev, A) || !plain(arg[4], dev, als) ||
      !plain(arg[5], dev, qB) || !plain(arg[6], dev, Bs) || !plain(arg[7], dev, qC) || !plain(arg[8], dev, Cs) || !optional(arg[10], dev, D) ||
      !optional(arg[12], dev, bias) || !plain(arg[15], dev, ss) || !plain(arg[16], dev, cbs))
    Py_RETURN_NONE;
  if (D.defined() && !plain(arg[11], dev, dsc)) Py_RETURN_NONE;
  if (x.dim() != 4 || qC.dim() != 4) Py_RETURN_NONE;
  const int64_t B = x.size(0), L = x.size(1), H = x.size(2), P = x.size(3), G = qC.size(2), N = qC.size(3);
  if (!rows(x, B, L, ScalarType::Half) || !rows(qC, B, L, ScalarType::Char) || qB.sizes() != qC.sizes()) Py_RETURN_NONE;
  if (dt.dim() != 3 || dt.size(0) != B || dt.size(1) != L || dt.size(2) != H) Py_RETURN_NONE;
  const ScalarType dtt = dt.scalar_type();
  if (dtt != ScalarType::Half && dtt != ScalarType::Float && dtt != ScalarType::Char) Py_RETURN_NONE;
  if (A.dim() != 1 || A.size(0) != H || A.scalar_type() != ScalarType::Char || !scalar(dts) || !scalar(als)) Py_RETURN_NONE;
  if (!table(Bs, G) || !table(Cs, G) || !table(cbs, G) || cbs.dim() != 1) Py_RETURN_NONE;
  if (ss.dim() != 2 || ss.size(0) != H || ss.size(1) != P || ss.scalar_type() != ScalarType::Float) Py_RETURN_NONE;
  if (bias.defined() && (bias.dim() != 1 || bias.size(0) != H || bias.scalar_type() != ScalarType::Float)) Py_RETURN_NONE;
  if (D.defined() && (D.scalar_type() != ScalarType::Char || D.dim() < 1 || D.dim() > 2 || D.size(0) != H || (D.dim() == 2 && D.size(1) != P) ||
                      D.stride(-1) != 1 || !scalar(dsc)))
    Py_RETURN_NONE;
  int64_t Q, shift;
  double lo, hi;
  if (!integer(arg[9], Q) || !integer(arg[24], shift)) Py_RETURN_NONE;
  if (!PyTuple_CheckExact(arg[14]) || PyTuple_GET_SIZE(arg[14]) != 2 || !number(PyTuple_GET_ITEM(arg[14], 0), lo) || !number(PyTuple_GET_ITEM(arg[14], 1), hi)) Py_RETURN_NONE;
  lq_ssd_combined_args a = {};
  if (keyside) {
    if (!plain(arg[20], dev, xs) || !plain(arg[21], dev, bfp) || !plain(arg[22], dev, bgs) || !optional(arg[23], dev, bmax)) Py_RETURN_NONE;
    if (xs.dim() != 2 || xs.size(0) != H || xs.size(1) != P || xs.scalar_type() != ScalarType::Float) Py_RETURN_NONE;
    if (!rows(bfp, B, L, ScalarType::Half) || bfp.sizes() != qC.sizes()) Py_RETURN_NONE;
    if (bgs.dim() != 4 || bgs.scalar_type() != ScalarType::Float) Py_RETURN_NONE;
    const int64_t full[4] = {B, (L + Q - 1) / std::max<int64_t>(Q, 1), H, N};
    int64_t st[4];
    for (int i = 0; i < 4; ++i) {
      if (bgs.size(i) != 1 && bgs.size(i) != full[i]) Py_RETURN_NONE;
      st[i] = bgs.size(i) > 1 ? bgs.stride(i) : 0;
    }
    if (bmax.defined() && (!table(bmax, B * L * G) || bmax.dim() != 3 || bmax.size(0) != B || bmax.size(1) != L)) Py_RETURN_NONE;
    a.b_fp = bfp.const_data_ptr(), a.bfp_stride_b = bfp.stride(0), a.bfp_stride_l = bfp.stride(1), a.bfp_stride_g = bfp.stride(2);
    a.x_scale_hp = f32(xs), a.xs_stride_h = xs.stride(0), a.xs_stride_p = xs.stride(1);
    a.b_gate_scale = f32(bgs), a.bgs_stride_b = st[0], a.bgs_stride_c = st[1], a.bgs_stride_h = st[2], a.bgs_stride_n = st[3];
    a.b_rowmax = f32(bmax);
  } else {
    if (!plain(arg[17], dev, alpha) || !plain(arg[18], dev, bsg)) Py_RETURN_NONE;
    if (!rows(qB, B, L, ScalarType::Char)) Py_RETURN_NONE;
    if (alpha.dim() != 2 || alpha.size(0) != H || alpha.size(1) != P || alpha.scalar_type() != ScalarType::Float) Py_RETURN_NONE;
    if (bsg.dim() != 1 || bsg.size(0) != G || bsg.scalar_type() != ScalarType::Float) Py_RETURN_NONE;
    a.qB = (const int8_t*)qB.const_data_ptr(), a.qB_stride_b = qB.stride(0), a.qB_stride_l = qB.stride(1), a.qB_stride_g = qB.stride(2);
    a.alpha_hp = f32(alpha), a.alpha_stride_h = alpha.stride(0), a.alpha_stride_p = alpha.stride(1);
    a.bscale_g = f32(bsg), a.bscale_stride_g = bsg.stride(0);
  }
  a.x = x.const_data_ptr(), a.x_stride_b = x.stride(0), a.x_stride_l = x.stride(1), a.x_stride_h = x.stride(2);
  a.dt = dt.const_data_ptr(), a.dt_dtype = dtt == ScalarType::Half ? LQ_DT_F16 : (dtt == ScalarType::Float ? LQ_DT_F32 : LQ_DT_I8);
  a.dt_stride_b = dt.stride(0), a.dt_stride_l = dt.stride(1), a.dt_stride_h = dt.stride(2), a.dt_scale = f32(dts);
  a.A_log = (const int8_t*)A.const_data_ptr(), a.A_log_stride_h = A.stride(0), a.A_log_scale = f32(als);
  a.dt_bias = f32(bias), a.dt_bias_stride_h = bias.defined() ? bias.stride(0) : 0;
  a.dt_softplus = softplus, a.dt_min = (float)lo, a.dt_max = (float)hi;
  a.qC = (const int8_t*)qC.const_data_ptr(), a.qC_stride_b = qC.stride(0), a.qC_stride_l = qC.stride(1), a.qC_stride_g = qC.stride(2);
  a.B_scale = f32(Bs), a.C_scale = f32(Cs), a.cb_scale = f32(cbs);
  if (D.defined()) a.D = (const int8_t*)D.const_data_ptr(), a.D_stride_h = D.stride(0), a.D_has_hdim = D.dim() == 2, a.D_scale = f32(dsc);
  a.state_scale = f32(ss), a.ss_stride_h = ss.stride(0), a.ss_stride_p = ss.stride(1);
  a.keyside = keyside, a.gate_shift = (int)shift;
  a.batch = (int)B, a.seqlen = (int)L, a.nheads = (int)H, a.headdim = (int)P, a.ngroups = (int)G, a.dstate = (int)N, a.chunk_size = (int)Q;
  int64_t bytes = 0;
  if (ssd_bytes(&a, &bytes) != 0) Py_RETURN_NONE;
  Tensor o;
  int rc;
  {
    pybind11::gil_scoped_release no_gil;
    o = empty({B, L, H, P}, ScalarType::Half, dev);
    Tensor ws = empty({bytes}, ScalarType::Byte, dev);
    a.out = o.data_ptr(), a.workspace = ws.data_ptr(), a.workspace_bytes = bytes;
    rc = ssd_entry(&a, stream_of(dev));
  }
  if (rc != 0) return failed("lq_ssd_combined", rc);
  return THPVariable_Wrap(o);
  END_HANDLE_TH_ERRORS
}

// ---- serving: ordinary calls of linquant_amd.w8a8_linear, norm.residual_rmsnorm, kernels.mamba2.conv1d_state and .ssm
bool act16(const Tensor& t) { return t.scalar_type() == ScalarType::Half || t.scalar_type() == ScalarType::BFloat16; }
int code(ScalarType st) { return st == ScalarType::Half ? LQ_DT_F16 : (st == ScalarType::BFloat16 ? LQ_DT_BF16 : LQ_DT_F32); }
bool floats(const Tensor& t) { return act16(t) || t.scalar_type() == ScalarType::Float; }
// unit last stride and every row on a 16-byte boundary (2-byte entries)
bool rows16(const Tensor& t) {
  if (t.dim() < 1 || t.stride(-1) != 1 || !aligned(t) || !fits(t.sizes())) return false;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.stride(i) % 8 != 0) return false;
  return true;
}
bool list32(const Tensor& t, int64_t n) { return t.scalar_type() == ScalarType::Int && t.dim() == 1 && t.size(0) == n && t.is_contiguous(); }
const int32_t* i32(const Tensor& t) { return t.defined() ? (const int32_t*)t.const_data_ptr() : nullptr; }
const void* at(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

// quantize_rows(x, pad): (codes in rows of `pad` bytes or multiples, scale) for a dense matrix
PyObject* quantize(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2) Py_RETURN_NONE;
  c10::Device dev(c10::DeviceType::CPU);
  Tensor x, codes, scale;
  int64_t pad;
  if (!device_of(arg[0], dev) || !plain(arg[0], dev, x) || !integer(arg[1], pad) || pad < 1) Py_RETURN_NONE;
  if (x.dim() != 2 || !floats(x) || !fits(x.sizes()) || x.stride(1) != 1 || x.size(1) > 16384) Py_RETURN_NONE;
  const int64_t M = x.size(0), K = x.size(1);
  lq_quantize_rows_args a = {};
  int rc;
  {
    pybind11::gil_scoped_release no_gil;
    codes = empty({M, (K + pad - 1) / pad * pad}, ScalarType::Char, dev), scale = empty({M}, ScalarType::Float, dev);
    a.x = x.const_data_ptr(), a.x_stride = x.stride(0), a.dtype = code(x.scalar_type());
    a.codes = (int8_t*)codes.data_ptr(), a.codes_stride = codes.stride(0), a.scale = (float*)scale.data_ptr(), a.rows = (int)M, a.cols = (int)K;
    rc = quantize_entry(&a, stream_of(dev));
  }
  if (rc != 0) return failed("lq_quantize_rows", rc);
  return Py_BuildValue("(NN)", THPVariable_Wrap(codes), THPVariable_Wrap(scale));
  END_HANDLE_TH_ERRORS
}

// int8_matmul(a, b, a_scale, b_scale, bias, out_dtype): matrices of whole 16-byte rows, fp32 scales on the GPU, a new output
PyObject* int8_matmul(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) Py_RETURN_NONE;
  c10::Device dev(c10::DeviceType::CPU);
  Tensor x, w, xs, ws, bias, out;
  if (!device_of(arg[0], dev) || !plain(arg[0], dev, x) || !plain(arg[1], dev, w) || !plain(arg[2], dev, xs) || !plain(arg[3], dev, ws) || !optional(arg[4], dev, bias)) Py_RETURN_NONE;
  if (!THPDtype_Check(arg[5])) Py_RETURN_NONE;
  const ScalarType ot = ((THPDtype*)arg[5])->scalar_type;
  if (ot != ScalarType::Half && ot != ScalarType::BFloat16 && ot != ScalarType::Float) Py_RETURN_NONE;
  for (const Tensor* t : {&x, &w})
    if (t->dim() != 2 || t->scalar_type() != ScalarType::Char || !fits(t->sizes()) || t->stride(1) != 1 || t->stride(0) % 16 != 0 || t->stride(0) >= 1 << 23 || !aligned(*t)) Py_RETURN_NONE;
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  if (w.size(1) != K || K % 16 != 0 || K > 131056) Py_RETURN_NONE;
  if (xs.scalar_type() != ScalarType::Float || !xs.is_contiguous() || (xs.numel() != 1 && xs.numel() != M)) Py_RETURN_NONE;
  if (ws.scalar_type() != ScalarType::Float || !ws.is_contiguous() || (ws.numel() != 1 && ws.numel() != N)) Py_RETURN_NONE;
  if (bias.defined() && (!floats(bias) || bias.dim() != 1 || bias.size(0) != N || !bias.is_contiguous())) Py_RETURN_NONE;
  lq_int8_matmul_args a = {};
  int rc;
  {
    pybind11::gil_scoped_release no_gil;
    out = empty({M, N}, ot, dev);
    a.a = (const int8_t*)x.const_data_ptr(), a.a_stride = x.stride(0), a.b = (const int8_t*)w.const_data_ptr(), a.b_stride = w.stride(0);
    a.a_scale = f32(xs), a.b_scale = f32(ws), a.a_scale_rows = xs.numel() != 1, a.b_scale_cols = ws.numel() != 1;
    a.bias = at(bias), a.bias_dtype = bias.defined() ? code(bias.scalar_type()) : 0;
    a.out = out.data_ptr(), a.out_stride = N, a.out_dtype = code(ot), a.rows = (int)M, a.cols = (int)N, a.inner = (int)K;
    rc = matmul_entry(&a, stream_of(dev));
  }
  if (rc != 0) return failed("lq_int8_matmul", rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// residual_rmsnorm(x, weight, residual, eps, gate, scale, post_weight, rows): rows that are dense, a gate for each channel or of x's shape,
// weights of one type; y in 16 bits, or with `rows` codes on a scale of each row
PyObject* residual_rmsnorm(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) Py_RETURN_NONE;
  c10::Device dev(c10::DeviceType::CPU);
  Tensor x, w, res, gate, post, y, r, codes, rs;
  double eps, scale;
  if (!device_of(arg[0], dev) || !plain(arg[0], dev, x) || !plain(arg[1], dev, w) || !plain(arg[2], dev, res) || !number(arg[3], eps) || !optional(arg[4], dev, gate) ||
      !number(arg[5], scale) || !optional(arg[6], dev, post))
    Py_RETURN_NONE;
  const int quant = PyObject_IsTrue(arg[7]);
  if (quant < 0) return nullptr;
  if (!act16(x) || x.dim() < 1 || !fits(x.sizes()) || !x.is_contiguous() || x.size(-1) > 16384) Py_RETURN_NONE;
  const int64_t D = x.size(-1), rows = x.numel() / D;
  if (rows > INT_MAX || res.sizes() != x.sizes() || !res.is_contiguous() || (res.scalar_type() != x.scalar_type() && res.scalar_type() != ScalarType::Float)) Py_RETURN_NONE;
  if (!floats(w) || w.dim() != 1 || w.size(0) != D || !w.is_contiguous()) Py_RETURN_NONE;
  if (post.defined() && (post.scalar_type() != w.scalar_type() || post.dim() != 1 || post.size(0) != D || !post.is_contiguous())) Py_RETURN_NONE;
  const bool channel = gate.defined() && gate.dim() == 1 && gate.size(0) == D;
  if (gate.defined() && (gate.scalar_type() != x.scalar_type() || !gate.is_contiguous() || !(channel || gate.sizes() == x.sizes()))) Py_RETURN_NONE;
  lq_residual_rmsnorm_args a = {};
  int rc;
  {
    pybind11::gil_scoped_release no_gil;
    r = empty(x.sizes(), res.scalar_type(), dev);
    if (quant) codes = empty(x.sizes(), ScalarType::Char, dev), rs = empty(x.sizes().slice(0, x.dim() - 1), ScalarType::Float, dev);
    else y = empty(x.sizes(), x.scalar_type(), dev);
    a.x = x.const_data_ptr(), a.x_stride = D, a.dtype = code(x.scalar_type()), a.residual = res.const_data_ptr(), a.residual_stride = D;
    a.residual_dtype = code(res.scalar_type()), a.gate = at(gate), a.gate_stride = channel ? 0 : D, a.gate_rows = 1, a.post_weight = at(post);
    a.weight = w.const_data_ptr(), a.weight_dtype = code(w.scalar_type()), a.scale = (float)scale, a.eps = (float)eps;
    a.residual_out = r.data_ptr(), a.residual_out_stride = D, a.out = quant ? nullptr : y.data_ptr(), a.out_stride = D;
    a.codes = quant ? (int8_t*)codes.data_ptr() : nullptr, a.codes_stride = D, a.row_scale = quant ? (float*)rs.data_ptr() : nullptr;
    a.rows = (int)rows, a.dim = (int)D;
    rc = norm_entry(&a, stream_of(dev));
  }
  if (rc != 0) return failed("lq_residual_rmsnorm", rc);
  if (quant) return Py_BuildValue("(NNN)", THPVariable_Wrap(codes), THPVariable_Wrap(rs), THPVariable_Wrap(r));
  return Py_BuildValue("(NN)", THPVariable_Wrap(y), THPVariable_Wrap(r));
  END_HANDLE_TH_ERRORS
}

bool activation(PyObject* o, int& silu) {
  silu = o != Py_None;
  return !silu || (PyUnicode_Check(o) && (PyUnicode_CompareWithASCIIString(o, "silu") == 0 || PyUnicode_CompareWithASCIIString(o, "swish") == 0));
}
// taps, bias and state of x's type that need no copy
bool conv_operands(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& state) {
  if (!act16(x) || !rows16(x) || w.dim() != 2 || w.scalar_type() != x.scalar_type() || !w.is_contiguous() || !aligned(w)) return false;
  const int64_t D = w.size(0), W = w.size(1);
  if (x.size(-1) != D || D % 8 != 0 || W < 2 || W > 4) return false;
  if (bias.defined() && (bias.scalar_type() != x.scalar_type() || bias.dim() != 1 || bias.size(0) != D || !bias.is_contiguous() || !aligned(bias))) return false;
  return !state.defined() || (state.dim() == 3 && state.size(1) == W - 1 && state.size(2) == D && state.scalar_type() == x.scalar_type() && rows16(state));
}
// n sequences, their slots (or none) in a state
bool slots_of(const Tensor& slots, int64_t n, const Tensor& state) { return slots.defined() ? list32(slots, n) : n <= state.size(0); }

// conv1d_step(x, state, weight, bias, activation, slots)
PyObject* conv1d_step(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) Py_RETURN_NONE;
  c10::Device dev(c10::DeviceType::CPU);
  Tensor x, state, w, bias, slots, out;
  int silu;
  if (!device_of(arg[0], dev) || !plain(arg[0], dev, x) || !plain(arg[1], dev, state) || !plain(arg[2], dev, w) || !optional(arg[3], dev, bias) || !activation(arg[4], silu) ||
      !optional(arg[5], dev, slots))
    Py_RETURN_NONE;
  if (x.dim() != 2 || !conv_operands(x, w, bias, state) || !slots_of(slots, x.size(0), state)) Py_RETURN_NONE;
  lq_conv1d_step_args a = {};
  int rc;
  {
    pybind11::gil_scoped_release no_gil;
    out = empty(x.sizes(), x.scalar_type(), dev);
    a.x = x.const_data_ptr(), a.x_stride = x.stride(0), a.dtype = code(x.scalar_type()), a.weight = w.const_data_ptr(), a.bias = at(bias), a.out = out.data_ptr();
    a.state = state.data_ptr(), a.state_stride_s = state.stride(0), a.state_stride_w = state.stride(1), a.slots = i32(slots), a.num_slots = (int)state.size(0);
    a.batch = (int)x.size(0), a.dim = (int)w.size(0), a.width = (int)w.size(1), a.silu = silu;
    rc = conv_step_entry(&a, stream_of(dev));
  }
  if (rc != 0) return failed("lq_conv1d_step", rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// conv1d_prompt(x, weight, bias, activation, state, slots, seq_starts), with a state
PyObject* conv1d_prompt(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) Py_RETURN_NONE;
  c10::Device dev(c10::DeviceType::CPU);
  Tensor x, w, bias, state, slots, starts, out;
  int silu;
  if (!device_of(arg[0], dev) || !plain(arg[0], dev, x) || !plain(arg[1], dev, w) || !optional(arg[2], dev, bias) || !activation(arg[3], silu) || !plain(arg[4], dev, state) ||
      !optional(arg[5], dev, slots) || !optional(arg[6], dev, starts))
    Py_RETURN_NONE;
  const bool packed = starts.defined();
  if (x.dim() != (packed ? 2 : 3) || !conv_operands(x, w, bias, state)) Py_RETURN_NONE;
  if (packed && (starts.dim() != 1 || starts.size(0) < 2 || !list32(starts, starts.size(0)))) Py_RETURN_NONE;
  const int64_t seqs = packed ? starts.size(0) - 1 : x.size(0);
  if (seqs > INT_MAX || !slots_of(slots, seqs, state)) Py_RETURN_NONE;
  lq_conv1d_prompt_args a = {};
  int rc;
  {
    pybind11::gil_scoped_release no_gil;
    out = empty(x.sizes(), x.scalar_type(), dev);
    a.x = x.const_data_ptr(), a.x_stride_b = packed ? 0 : x.stride(0), a.x_stride_l = x.stride(-2), a.dtype = code(x.scalar_type());
    a.weight = w.const_data_ptr(), a.bias = at(bias), a.out = out.data_ptr();
    a.state = state.data_ptr(), a.state_stride_s = state.stride(0), a.state_stride_w = state.stride(1), a.slots = i32(slots), a.seq_starts = i32(starts);
    a.num_slots = (int)state.size(0), a.nseq = (int)seqs, a.seqlen = packed ? 0 : (int)x.size(1), a.tokens = packed ? (int)x.size(0) : 0;
    a.dim = (int)w.size(0), a.width = (int)w.size(1), a.silu = silu;
    rc = conv_prompt_entry(&a, stream_of(dev));
  }
  if (rc != 0) return failed("lq_conv1d_prompt", rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// what both forms of the scan take: arg = x, dt, A, B, C, D, dt_bias, dt_softplus, dt_limit, state, slots
struct Scan {
  Tensor x, dt, A, B, C, D, bias, state, slots;
  int softplus = 0;
  double lo = 0.0, hi = 0.0;
  int64_t H = 0, P = 0, G = 0, N = 0;
};
bool scan_operands(PyObject* const* arg, const c10::Device& dev, int lead, Scan& s) {
  if (!plain(arg[0], dev, s.x) || !plain(arg[1], dev, s.dt) || !plain(arg[2], dev, s.A) || !plain(arg[3], dev, s.B) || !plain(arg[4], dev, s.C) || !optional(arg[5], dev, s.D) ||
      !optional(arg[6], dev, s.bias) || !plain(arg[9], dev, s.state) || !optional(arg[10], dev, s.slots))
    return false;
  if (!PyBool_Check(arg[7]) || !PyTuple_CheckExact(arg[8]) || PyTuple_GET_SIZE(arg[8]) != 2 || !number(PyTuple_GET_ITEM(arg[8], 0), s.lo) || !number(PyTuple_GET_ITEM(arg[8], 1), s.hi))
    return false;
  s.softplus = arg[7] == Py_True;
  const Tensor &x = s.x, &B = s.B, &C = s.C, &dt = s.dt;
  if (x.dim() != lead + 2 || B.dim() != lead + 2 || dt.dim() != lead + 1 || !act16(x) || B.scalar_type() != x.scalar_type() || C.scalar_type() != x.scalar_type() || !floats(dt)) return false;
  if (!rows16(x) || !rows16(B) || !rows16(C) || B.sizes() != C.sizes() || !fits(dt.sizes())) return false;
  s.H = x.size(lead), s.P = x.size(lead + 1), s.G = B.size(lead), s.N = B.size(lead + 1);
  for (int i = 0; i < lead; ++i)
    if (B.size(i) != x.size(i) || dt.size(i) != x.size(i)) return false;
  if (dt.size(lead) != s.H || s.H % s.G != 0 || s.P % 8 != 0 || s.N % 8 != 0 || s.N > 256 || x.stride(lead - 1) >= 1 << 24) return false;
  if (s.A.dim() != 1 || !table(s.A, s.H) || (s.bias.defined() && (s.bias.dim() != 1 || !table(s.bias, s.H)))) return false;
  if (s.D.defined() && !(s.D.dim() == 1 ? table(s.D, s.H) : s.D.dim() == 2 && s.D.size(0) == s.H && table(s.D, s.H * s.P))) return false;
  const Tensor& st = s.state;
  return st.dim() == 4 && st.scalar_type() == ScalarType::Float && fits(st.sizes()) && st.size(1) == s.H && st.size(2) == s.P && st.size(3) == s.N && st.stride(3) == 1 &&
         st.stride(2) == s.N && st.stride(1) == s.P * s.N && aligned(st);
}
template <typename Args>
void scan_args(const Scan& s, Args& a) {
  a.x = s.x.const_data_ptr(), a.dtype = code(s.x.scalar_type()), a.dt = s.dt.const_data_ptr(), a.dt_dtype = code(s.dt.scalar_type()), a.A = f32(s.A);
  a.B = s.B.const_data_ptr(), a.C = s.C.const_data_ptr(), a.D = f32(s.D), a.D_has_hdim = s.D.defined() && s.D.dim() == 2, a.dt_bias = f32(s.bias);
  a.dt_softplus = s.softplus, a.dt_min = (float)s.lo, a.dt_max = (float)s.hi;
  a.state = (float*)s.state.data_ptr(), a.state_stride_s = s.state.stride(0), a.slots = i32(s.slots), a.num_slots = (int)s.state.size(0);
  a.nheads = (int)s.H, a.headdim = (int)s.P, a.ngroups = (int)s.G, a.dstate = (int)s.N;
}

// ssm_step(x, dt, A, B, C, D, dt_bias, dt_softplus, dt_limit, state, slots)
PyObject* ssm_step(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11) Py_RETURN_NONE;
  c10::Device dev(c10::DeviceType::CPU);
  Scan s;
  Tensor out;
  if (!device_of(arg[0], dev) || !scan_operands(arg, dev, 1, s)) Py_RETURN_NONE;
  const int64_t B = s.x.size(0);
  if (B > 65535 || !slots_of(s.slots, B, s.state)) Py_RETURN_NONE;
  lq_ssm_step_args a = {};
  int rc;
  {
    pybind11::gil_scoped_release no_gil;
    out = empty(s.x.sizes(), s.x.scalar_type(), dev);
    scan_args(s, a);
    a.x_stride_b = s.x.stride(0), a.x_stride_h = s.x.stride(1), a.dt_stride_b = s.dt.stride(0), a.dt_stride_h = s.dt.stride(1);
    a.B_stride_b = s.B.stride(0), a.B_stride_g = s.B.stride(1), a.C_stride_b = s.C.stride(0), a.C_stride_g = s.C.stride(1);
    a.out = out.data_ptr(), a.batch = (int)B;
    rc = ssm_step_entry(&a, stream_of(dev));
  }
  if (rc != 0) return failed("lq_ssm_step", rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// ssm_prompt(x, dt, A, B, C, D, dt_bias, dt_softplus, dt_limit, state, slots, seq_starts), with a state
PyObject* ssm_prompt(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12) Py_RETURN_NONE;
  c10::Device dev(c10::DeviceType::CPU);
  Scan s;
  Tensor starts, out;
  if (!device_of(arg[0], dev) || !optional(arg[11], dev, starts)) Py_RETURN_NONE;
  const bool packed = starts.defined();
  if (!scan_operands(arg, dev, packed ? 1 : 2, s)) Py_RETURN_NONE;
  if (packed && (starts.dim() != 1 || starts.size(0) < 2 || !list32(starts, starts.size(0)))) Py_RETURN_NONE;
  const int64_t seqs = packed ? starts.size(0) - 1 : s.x.size(0);
  if (seqs > INT_MAX || !slots_of(s.slots, seqs, s.state)) Py_RETURN_NONE;
  lq_ssm_prompt_args a = {};
  scan_args(s, a);
  const int l = packed ? 0 : 1;
  auto batch = [&](const Tensor& t) { return packed ? 0 : t.stride(0); };
  a.x_stride_b = batch(s.x), a.x_stride_l = s.x.stride(l), a.x_stride_h = s.x.stride(l + 1);
  a.dt_stride_b = batch(s.dt), a.dt_stride_l = s.dt.stride(l), a.dt_stride_h = s.dt.stride(l + 1);
  a.B_stride_b = batch(s.B), a.B_stride_l = s.B.stride(l), a.B_stride_g = s.B.stride(l + 1);
  a.C_stride_b = batch(s.C), a.C_stride_l = s.C.stride(l), a.C_stride_g = s.C.stride(l + 1);
  a.seq_starts = i32(starts), a.nseq = (int)seqs, a.seqlen = packed ? 0 : (int)s.x.size(1), a.tokens = packed ? (int)s.x.size(0) : 0;
  int64_t bytes = 0;
  if (ssm_prompt_bytes(&a, &bytes) != 0) Py_RETURN_NONE;
  int rc;
  {
    pybind11::gil_scoped_release no_gil;
    out = empty(s.x.sizes(), s.x.scalar_type(), dev);
    Tensor ws = empty({bytes}, ScalarType::Byte, dev);
    a.out = out.data_ptr(), a.workspace = ws.data_ptr(), a.workspace_bytes = bytes;
    rc = ssm_prompt_entry(&a, stream_of(dev));
  }
  if (rc != 0) return failed("lq_ssm_prompt", rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// what both forms of linear attention take: q, k, v with `lead` token dimensions, decays for each head or each token, a state
struct Attention {
  Tensor q, k, v, g, state, slots;
  double scale = 0.0;
  int64_t H = 0, K = 0, V = 0;
};
bool attention_operands(PyObject* const* arg, const c10::Device& dev, int lead, Attention& a) {  // arg = q, k, v, g, scale, state, slots
  if (!plain(arg[0], dev, a.q) || !plain(arg[1], dev, a.k) || !plain(arg[2], dev, a.v) || !optional(arg[3], dev, a.g) || !(arg[4] == Py_None || number(arg[4], a.scale)) ||
      !plain(arg[5], dev, a.state) || !optional(arg[6], dev, a.slots))
    return false;
  const Tensor &q = a.q, &k = a.k, &v = a.v, &g = a.g, &st = a.state;
  if (v.dim() != lead + 2 || q.dim() != lead + 2 || !act16(v) || q.scalar_type() != v.scalar_type() || k.scalar_type() != v.scalar_type() || !rows16(q) || !rows16(k) || !rows16(v)) return false;
  a.H = v.size(lead), a.K = q.size(lead + 1), a.V = v.size(lead + 1);
  if (k.sizes() != q.sizes() || a.K % 8 != 0 || a.K > 256 || a.V % 8 != 0) return false;
  for (int i = 0; i <= lead; ++i)
    if (q.size(i) != v.size(i)) return false;
  for (const Tensor* t : {&q, &k, &v})
    if (t->stride(lead - 1) < 0 || t->stride(lead - 1) >= 1 << 24) return false;
  if (g.defined()) {
    if (g.scalar_type() != ScalarType::Float || !(g.dim() == 1 || g.dim() == lead + 1) || !fits(g.sizes()) || g.size(-1) != a.H) return false;
    for (int i = 0; g.dim() > 1 && i < lead; ++i)
      if (g.size(i) != v.size(i)) return false;
    if (g.dim() > 1 && (g.stride(-2) < 0 || g.stride(-2) >= 1 << 24)) return false;
  }
  if (arg[4] == Py_None) a.scale = std::pow((double)a.K, -0.5);
  return st.dim() == 4 && st.scalar_type() == ScalarType::Float && fits(st.sizes()) && st.size(1) == a.H && st.size(2) == a.K && st.size(3) == a.V && st.stride(3) == 1 &&
         st.stride(2) == a.V && st.stride(1) == a.K * a.V && st.stride(0) % 4 == 0 && (st.size(0) == 1 || st.stride(0) >= a.H * a.K * a.V) && aligned(st);
}
template <typename Args>
void attention_args(const Attention& s, Args& a) {
  a.q = s.q.const_data_ptr(), a.k = s.k.const_data_ptr(), a.v = s.v.const_data_ptr(), a.dtype = code(s.v.scalar_type()), a.g = f32(s.g), a.scale = (float)s.scale;
  a.state = (float*)s.state.data_ptr(), a.state_stride_s = s.state.stride(0), a.slots = i32(s.slots), a.num_slots = (int)s.state.size(0);
  a.nheads = (int)s.H, a.kdim = (int)s.K, a.vdim = (int)s.V;
}

// linear_attention_step(q, k, v, g, scale, state, slots)
PyObject* linear_attention_step(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) Py_RETURN_NONE;
  c10::Device dev(c10::DeviceType::CPU);
  Attention s;
  Tensor out;
  if (!device_of(arg[0], dev) || !attention_operands(arg, dev, 1, s)) Py_RETURN_NONE;
  const int64_t B = s.v.size(0);
  if (B > 65535 || !slots_of(s.slots, B, s.state)) Py_RETURN_NONE;
  lq_linear_attention_step_args a = {};
  int rc;
  {
    pybind11::gil_scoped_release no_gil;
    out = empty(s.v.sizes(), s.v.scalar_type(), dev);
    attention_args(s, a);
    a.q_stride_b = s.q.stride(0), a.q_stride_h = s.q.stride(1), a.k_stride_b = s.k.stride(0), a.k_stride_h = s.k.stride(1);
    a.v_stride_b = s.v.stride(0), a.v_stride_h = s.v.stride(1);
    a.g_dtype = LQ_DT_F32, a.g_stride_b = s.g.defined() && s.g.dim() == 2 ? s.g.stride(0) : 0, a.g_stride_h = s.g.defined() ? s.g.stride(-1) : 0;
    a.out = out.data_ptr(), a.batch = (int)B;
    rc = attention_step_entry(&a, stream_of(dev));
  }
  if (rc != 0) return failed("lq_linear_attention_step", rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// linear_attention_prompt(q, k, v, g, scale, state, slots, seq_starts), with a state
PyObject* linear_attention_prompt(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) Py_RETURN_NONE;
  c10::Device dev(c10::DeviceType::CPU);
  Attention s;
  Tensor starts, out;
  if (!device_of(arg[0], dev) || !optional(arg[7], dev, starts)) Py_RETURN_NONE;
  const bool packed = starts.defined();
  if (!attention_operands(arg, dev, packed ? 1 : 2, s)) Py_RETURN_NONE;
  if (packed && (starts.dim() != 1 || starts.size(0) < 2 || !list32(starts, starts.size(0)))) Py_RETURN_NONE;
  const int64_t seqs = packed ? starts.size(0) - 1 : s.v.size(0);
  if (seqs > INT_MAX || !slots_of(s.slots, seqs, s.state)) Py_RETURN_NONE;
  lq_linear_attention_prompt_args a = {};
  attention_args(s, a);
  const int l = packed ? 0 : 1;
  auto batch = [&](const Tensor& t) { return packed ? 0 : t.stride(0); };
  a.q_stride_b = batch(s.q), a.q_stride_l = s.q.stride(l), a.q_stride_h = s.q.stride(l + 1);
  a.k_stride_b = batch(s.k), a.k_stride_l = s.k.stride(l), a.k_stride_h = s.k.stride(l + 1);
  a.v_stride_b = batch(s.v), a.v_stride_l = s.v.stride(l), a.v_stride_h = s.v.stride(l + 1);
  if (s.g.defined()) {
    if (s.g.dim() > 1) a.g_stride_b = batch(s.g), a.g_stride_l = s.g.stride(l);
    a.g_stride_h = s.g.stride(-1);
  }
  a.seq_starts = i32(starts), a.nseq = (int)seqs, a.seqlen = packed ? 0 : (int)s.v.size(1), a.tokens = packed ? (int)s.v.size(0) : 0;
  int64_t bytes = 0;
  if (attention_prompt_bytes(&a, &bytes) != 0) Py_RETURN_NONE;
  int rc;
  {
    pybind11::gil_scoped_release no_gil;
    out = empty(s.v.sizes(), s.v.scalar_type(), dev);
    Tensor ws;
    if (bytes) ws = empty({bytes}, ScalarType::Byte, dev);
    a.out = out.data_ptr(), a.workspace = bytes ? ws.data_ptr() : nullptr, a.workspace_bytes = bytes;
    rc = attention_prompt_entry(&a, stream_of(dev));
  }
  if (rc != 0) return failed("lq_linear_attention_prompt", rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// entries from row to row of a tensor (..., D) with unit stride along D, if its rows are equally far apart in their order
bool row_distance(const Tensor& t, int64_t& s) {
  if (t.size(-1) != 1 && t.stride(-1) != 1) return false;
  int64_t next = 0;
  bool first = true;
  s = t.size(-1);
  for (int64_t i = t.dim() - 2; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (first) s = next = t.stride(i), first = false;
    else if (t.stride(i) != next) return false;
    next *= t.size(i);
  }
  return s >= 0;
}

// groupnorm_gated(x, z, weight, bias, num_groups, eps, act): equally distant rows, weights of one type
PyObject* groupnorm_gated(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) Py_RETURN_NONE;
  c10::Device dev(c10::DeviceType::CPU);
  Tensor x, z, w, b, out;
  int64_t groups, act;
  double eps;
  if (!device_of(arg[0], dev) || !plain(arg[0], dev, x) || !optional(arg[1], dev, z) || !optional(arg[2], dev, w) || !optional(arg[3], dev, b) || !integer(arg[4], groups) ||
      !number(arg[5], eps) || !integer(arg[6], act))
    Py_RETURN_NONE;
  int64_t xs = 0, zs = 0;
  if (!act16(x) || x.dim() < 1 || !fits(x.sizes()) || !row_distance(x, xs)) Py_RETURN_NONE;
  const int64_t D = x.size(-1), rows = x.numel() / D;
  if (rows > INT_MAX || groups < 1 || D % groups != 0 || D / groups > 16384) Py_RETURN_NONE;
  if (z.defined() && (z.scalar_type() != x.scalar_type() || z.sizes() != x.sizes() || !row_distance(z, zs))) Py_RETURN_NONE;
  for (const Tensor* t : {&w, &b})
    if (t->defined() && (!floats(*t) || t->dim() != 1 || t->size(0) != D || !t->is_contiguous())) Py_RETURN_NONE;
  if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type()) Py_RETURN_NONE;
  lq_groupnorm_gated_args a = {};
  int rc;
  {
    pybind11::gil_scoped_release no_gil;
    out = empty(x.sizes(), x.scalar_type(), dev);
    a.x = x.const_data_ptr(), a.x_stride = xs, a.z = at(z), a.z_stride = zs, a.dtype = code(x.scalar_type()), a.weight = at(w), a.bias = at(b);
    a.weight_dtype = w.defined() ? code(w.scalar_type()) : (b.defined() ? code(b.scalar_type()) : 0), a.out = out.data_ptr(), a.eps = (float)eps;
    a.rows = (int)rows, a.dim = (int)D, a.num_groups = (int)groups, a.act = (int)act;
    rc = groupnorm_entry(&a, stream_of(dev));
  }
  if (rc != 0) return failed("lq_groupnorm_gated", rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// adapted(x, scale, weight, weight_scale, bias, out_dtype, down, up, scaling, ids): a W8A8Linear with low-rank adapters.  x (..., K) in the
// adapters' type and scale None: quantized row by row here; or INT8 codes and their scale, one or one for each row
PyObject* adapted(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10) Py_RETURN_NONE;
  c10::Device dev(c10::DeviceType::CPU);
  Tensor x, xs, w, ws, bias, down, up, scaling, ids, codes, h, order, out;
  if (!device_of(arg[0], dev) || !plain(arg[0], dev, x) || !optional(arg[1], dev, xs) || !plain(arg[2], dev, w) || !plain(arg[3], dev, ws) || !optional(arg[4], dev, bias) ||
      !plain(arg[6], dev, down) || !plain(arg[7], dev, up) || !plain(arg[8], dev, scaling) || !plain(arg[9], dev, ids))
    Py_RETURN_NONE;
  if (!THPDtype_Check(arg[5])) Py_RETURN_NONE;
  const ScalarType ot = ((THPDtype*)arg[5])->scalar_type;
  if (ot != ScalarType::Half && ot != ScalarType::BFloat16 && ot != ScalarType::Float) Py_RETURN_NONE;
  const bool coded = xs.defined();
  if (x.dim() < 1 || !fits(x.sizes()) || !x.is_contiguous() || !aligned(x) || w.dim() != 2 || w.scalar_type() != ScalarType::Char || !fits(w.sizes()) || !w.is_contiguous() || !aligned(w)) Py_RETURN_NONE;
  const int64_t K = x.size(-1), M = x.numel() / K, N = w.size(0);
  if (K % 16 != 0 || K > 16384 || w.size(1) != K || M > INT_MAX || K >= 1 << 23) Py_RETURN_NONE;
  if (!act16(down) || x.scalar_type() != (coded ? ScalarType::Char : down.scalar_type()) || up.scalar_type() != down.scalar_type() || down.dim() != 3 || up.dim() != 3 || !fits(down.sizes()) ||
      !fits(up.sizes()) || !down.is_contiguous() || !up.is_contiguous() || !aligned(down) || !aligned(up))
    Py_RETURN_NONE;
  const int64_t count = down.size(0), R = down.size(1);
  if (R % 16 != 0 || R > 128 || down.size(2) != K || up.size(0) != count || up.size(1) != N || up.size(2) != R || !table(scaling, count)) Py_RETURN_NONE;
  if (ids.scalar_type() != ScalarType::Int || !ids.is_contiguous() || ids.numel() != M || ids.sizes() != x.sizes().slice(0, x.dim() - 1)) Py_RETURN_NONE;
  if (coded && (xs.scalar_type() != ScalarType::Float || !xs.is_contiguous() || (xs.numel() != 1 && xs.numel() != M))) Py_RETURN_NONE;
  if (ws.scalar_type() != ScalarType::Float || !ws.is_contiguous() || ws.numel() != N) Py_RETURN_NONE;
  if (bias.defined() && (!floats(bias) || bias.dim() != 1 || bias.size(0) != N || !bias.is_contiguous())) Py_RETURN_NONE;
  auto sizes = x.sizes().vec();
  sizes.back() = N;
  lq_adapter_down_args d = {};
  lq_int8_matmul_args a = {};
  const char* what = "lq_adapter_down";
  int rc = 0;
  {
    pybind11::gil_scoped_release no_gil;
    const hipStream_t stream = stream_of(dev);
    out = empty(sizes, ot, dev), h = empty({M, R}, ScalarType::Float, dev);
    if (!coded) {
      codes = empty({M, K}, ScalarType::Char, dev), xs = empty({M}, ScalarType::Float, dev);
      d.codes_out = (int8_t*)codes.data_ptr(), d.scale_out = (float*)xs.data_ptr();
    }
    if (M > 32) order = empty({M}, ScalarType::Int, dev);
    {
      d.x = x.const_data_ptr(), d.x_stride = K, d.x_dtype = coded ? LQ_DT_I8 : code(x.scalar_type()), d.x_scale = coded ? f32(xs) : nullptr, d.x_scale_rows = xs.numel() != 1;
      d.down = down.const_data_ptr(), d.dtype = code(down.scalar_type()), d.scaling = f32(scaling), d.ids = i32(ids), d.h = (float*)h.data_ptr();
      d.rows = (int)M, d.inner = (int)K, d.inner_padded = (int)K, d.rank = (int)R, d.count = (int)count, d.order = order.defined() ? (int32_t*)order.data_ptr() : nullptr;
      rc = adapter_down_entry(&d, stream);
    }
    if (rc == 0) {
      what = "lq_int8_matmul";
      a.a = (const int8_t*)(coded ? x : codes).const_data_ptr(), a.a_stride = K, a.b = (const int8_t*)w.const_data_ptr(), a.b_stride = K;
      a.a_scale = f32(xs), a.b_scale = f32(ws), a.a_scale_rows = xs.numel() != 1 || !coded, a.b_scale_cols = 1;
      a.bias = at(bias), a.bias_dtype = bias.defined() ? code(bias.scalar_type()) : 0;
      a.out = out.data_ptr(), a.out_stride = N, a.out_dtype = code(ot), a.rows = (int)M, a.cols = (int)N, a.inner = (int)K;
      a.adapter_h = f32(h), a.adapter_ids = i32(ids), a.adapter_up = up.const_data_ptr(), a.adapter_dtype = code(up.scalar_type()), a.adapter_rank = (int)R, a.adapter_count = (int)count, a.adapter_order = i32(order);
      rc = matmul_entry(&a, stream);
    }
  }
  if (rc != 0) return failed(what, rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// the tensors of nested lists and tuples (of ones that contain themselves: none): three numbers each
bool slot_tensors(PyObject* o, const c10::Device& dev, int64_t& slots, std::vector<int64_t>& out, int depth = 0) {
  if (THPVariable_CheckExact(o)) {
    Tensor t;
    if (!plain(o, dev, t) || t.dim() < 1 || !fits(t.sizes())) return false;
    if (slots == 0) slots = t.size(0);
    int64_t dense = 1;
    for (int64_t i = t.dim() - 1; i >= 1; --i) {
      if (t.size(i) != 1 && t.stride(i) != dense) return false;
      dense *= t.size(i);
    }
    if (t.size(0) != slots || (slots > 1 && t.stride(0) < dense)) return false;
    const int64_t size = t.element_size();
    out.push_back((int64_t)t.data_ptr()), out.push_back((slots > 1 ? t.stride(0) : dense) * size), out.push_back(dense * size);
    return true;
  }
  const bool list = PyList_CheckExact(o);
  if ((!list && !PyTuple_Check(o)) || depth == 16) return false;
  const Py_ssize_t n = list ? PyList_GET_SIZE(o) : PyTuple_GET_SIZE(o);
  for (Py_ssize_t i = 0; i < n; ++i)
    if (!slot_tensors(list ? PyList_GET_ITEM(o, i) : PyTuple_GET_ITEM(o, i), dev, slots, out, depth + 1)) return false;
  return true;
}

// copy_slots(states, src, dst) -> True
PyObject* copy_slots(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3) Py_RETURN_NONE;
  c10::Device dev(c10::DeviceType::CPU);
  Tensor src, dst;
  if (!device_of(arg[1], dev) || !plain(arg[1], dev, src) || !plain(arg[2], dev, dst)) Py_RETURN_NONE;
  const int64_t entries = src.numel();
  if (entries < 1 || entries > 8192 || !list32(src, entries) || !list32(dst, entries)) Py_RETURN_NONE;
  int64_t slots = 0;
  std::vector<int64_t> t;
  if (!slot_tensors(arg[0], dev, slots, t) || t.empty()) Py_RETURN_NONE;
  const size_t count = t.size() / 3;
  std::vector<std::pair<int64_t, int64_t>> spans(count);
  for (size_t i = 0; i < count; ++i) spans[i] = {t[3 * i], t[3 * i] + (slots - 1) * t[3 * i + 1] + t[3 * i + 2]};
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < count; ++i)
    if (spans[i].first < spans[i - 1].second) Py_RETURN_NONE;
  lq_copy_slots_args a = {};
  a.tensors = t.data(), a.num_tensors = (int)count, a.num_slots = (int)slots, a.src = i32(src), a.dst = i32(dst), a.entries = (int)entries;
  int rc;
  {
    pybind11::gil_scoped_release no_gil;
    rc = copy_slots_entry(&a, stream_of(dev));
  }
  if (rc != 0) return failed("lq_copy_slots", rc);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// whether the library was built from the header that this file was: its ABI version and the structs that are filled here
bool same_abi(decltype(&lq_abi_version) version, decltype(&lq_args_size) size) {
  const int v = version();
  if (v != LQ_ABI_VERSION) return PyErr_Format(PyExc_RuntimeError, "ABI version %d, the library has %d", LQ_ABI_VERSION, v), false;
#define LQ_SAME_SIZE(T)                                                                                                          \
  if (const int n = size(#T); n != (int)sizeof(T))                                                                               \
    return PyErr_Format(PyExc_RuntimeError, #T ": sizeof %d, the library has %d", (int)sizeof(T), n), false
  LQ_SAME_SIZE(lq_zoo_simple_gla_args);
  LQ_SAME_SIZE(lq_zoo_chunk_forward_args);
  LQ_SAME_SIZE(lq_zoo_rotate_qkv_args);
  LQ_SAME_SIZE(lq_split_rotate_quant_xBC_args);
  LQ_SAME_SIZE(lq_ssd_combined_args);
  LQ_SAME_SIZE(lq_quantize_rows_args);
  LQ_SAME_SIZE(lq_int8_matmul_args);
  LQ_SAME_SIZE(lq_residual_rmsnorm_args);
  LQ_SAME_SIZE(lq_conv1d_prompt_args);
  LQ_SAME_SIZE(lq_conv1d_step_args);
  LQ_SAME_SIZE(lq_ssm_prompt_args);
  LQ_SAME_SIZE(lq_ssm_step_args);
  LQ_SAME_SIZE(lq_linear_attention_prompt_args);
  LQ_SAME_SIZE(lq_linear_attention_step_args);
  LQ_SAME_SIZE(lq_groupnorm_gated_args);
  LQ_SAME_SIZE(lq_adapter_down_args);
  LQ_SAME_SIZE(lq_copy_slots_args);
#undef LQ_SAME_SIZE
  return true;
}

// init(raise_failed, {entry point: address})
PyObject* init(PyObject*, PyObject* const* arg, Py_ssize_t n) {
  if (n != 2 || !PyCallable_Check(arg[0]) || !PyDict_Check(arg[1])) {
    PyErr_SetString(PyExc_TypeError, "init(raise_failed, addresses)");
    return nullptr;
  }
  auto entry = [&](const char* name) { PyObject* o = PyDict_GetItemString(arg[1], name); return o ? PyLong_AsVoidPtr(o) : nullptr; };
  const auto version = (decltype(&lq_abi_version))entry("lq_abi_version");
  const auto size = (decltype(&lq_args_size))entry("lq_args_size");
  if (!version || !size) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_KeyError, "lq_abi_version or lq_args_size is missing");
    return nullptr;
  }
  if (!same_abi(version, size)) return nullptr;
  simple_gla_entry = (decltype(simple_gla_entry))entry("lq_zoo_simple_gla");
  simple_gla_bytes = (decltype(simple_gla_bytes))entry("lq_zoo_simple_gla_workspace_bytes");
  split_rotate_entry = (decltype(split_rotate_entry))entry("lq_split_rotate_quant_xBC");
  ssd_entry = (decltype(ssd_entry))entry("lq_ssd_combined");
  ssd_bytes = (decltype(ssd_bytes))entry("lq_ssd_combined_workspace_bytes");
  chunk_forward_entry = (decltype(chunk_forward_entry))entry("lq_zoo_chunk_forward");
  chunk_forward_bytes = (decltype(chunk_forward_bytes))entry("lq_zoo_chunk_forward_workspace_bytes");
  rotate_entry = (decltype(rotate_entry))entry("lq_zoo_rotate_qkv");
  quantize_entry = (decltype(quantize_entry))entry("lq_quantize_rows");
  matmul_entry = (decltype(matmul_entry))entry("lq_int8_matmul");
  norm_entry = (decltype(norm_entry))entry("lq_residual_rmsnorm");
  conv_prompt_entry = (decltype(conv_prompt_entry))entry("lq_conv1d_prompt");
  conv_step_entry = (decltype(conv_step_entry))entry("lq_conv1d_step");
  ssm_prompt_entry = (decltype(ssm_prompt_entry))entry("lq_ssm_prompt");
  ssm_prompt_bytes = (decltype(ssm_prompt_bytes))entry("lq_ssm_prompt_workspace_bytes");
  ssm_step_entry = (decltype(ssm_step_entry))entry("lq_ssm_step");
  attention_prompt_entry = (decltype(attention_prompt_entry))entry("lq_linear_attention_prompt");
  attention_prompt_bytes = (decltype(attention_prompt_bytes))entry("lq_linear_attention_prompt_workspace_bytes");
  attention_step_entry = (decltype(attention_step_entry))entry("lq_linear_attention_step");
  groupnorm_entry = (decltype(groupnorm_entry))entry("lq_groupnorm_gated");
  adapter_down_entry = (decltype(adapter_down_entry))entry("lq_adapter_down");
  copy_slots_entry = (decltype(copy_slots_entry))entry("lq_copy_slots");
  if (!quantize_entry || !matmul_entry || !norm_entry || !conv_prompt_entry || !conv_step_entry || !ssm_prompt_entry || !ssm_prompt_bytes || !ssm_step_entry ||
      !simple_gla_entry || !simple_gla_bytes || !chunk_forward_entry || !chunk_forward_bytes || !rotate_entry || !split_rotate_entry || !ssd_entry || !ssd_bytes ||
      !attention_prompt_entry || !attention_prompt_bytes || !attention_step_entry || !groupnorm_entry || !adapter_down_entry || !copy_slots_entry) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_KeyError, "an entry point is missing");
    return nullptr;
  }
  Py_INCREF(arg[0]);
  Py_XSETREF(raise_failed, arg[0]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"init", (PyCFunction)(void*)init, METH_FASTCALL, nullptr},
                         {"simple_gla", (PyCFunction)(void*)simple_gla, METH_FASTCALL, nullptr},
                         {"chunk_forward", (PyCFunction)(void*)chunk_forward, METH_FASTCALL, nullptr},
                         {"rotate_qkv", (PyCFunction)(void*)rotate_qkv, METH_FASTCALL, nullptr},
                         {"split_rotate", (PyCFunction)(void*)split_rotate, METH_FASTCALL, nullptr},
                         {"ssd", (PyCFunction)(void*)ssd, METH_FASTCALL, nullptr},
                         {"quantize_rows", (PyCFunction)(void*)quantize, METH_FASTCALL, nullptr},
                         {"int8_matmul", (PyCFunction)(void*)int8_matmul, METH_FASTCALL, nullptr},
                         {"residual_rmsnorm", (PyCFunction)(void*)residual_rmsnorm, METH_FASTCALL, nullptr},
                         {"conv1d_step", (PyCFunction)(void*)conv1d_step, METH_FASTCALL, nullptr},
                         {"conv1d_prompt", (PyCFunction)(void*)conv1d_prompt, METH_FASTCALL, nullptr},
                         {"ssm_step", (PyCFunction)(void*)ssm_step, METH_FASTCALL, nullptr},
                         {"ssm_prompt", (PyCFunction)(void*)ssm_prompt, METH_FASTCALL, nullptr},
                         {"linear_attention_step", (PyCFunction)(void*)linear_attention_step, METH_FASTCALL, nullptr},
                         {"linear_attention_prompt", (PyCFunction)(void*)linear_attention_prompt, METH_FASTCALL, nullptr},
                         {"groupnorm_gated", (PyCFunction)(void*)groupnorm_gated, METH_FASTCALL, nullptr},
                         {"adapted", (PyCFunction)(void*)adapted, METH_FASTCALL, nullptr},
                         {"copy_slots", (PyCFunction)(void*)copy_slots, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__binding() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", LQ_BUILT_FOR) < 0) Py_CLEAR(m);
  return m;
}
