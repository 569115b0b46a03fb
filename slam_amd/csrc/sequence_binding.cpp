// Python binding of the sequence-layer entry points: checks torch tensors, allocates a call's workspace and launches on the current
// stream of the tensors' device.  A call for single frames is bound by the host (its kernel takes 5 us): with the same checks in Python
// and ctypes the scan's call took 11 us, 8 of them for the checks; here it takes 4.
//
// The entry points are those of the library that capi.py has loaded, handed over by address (bind), so both use the same one.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cstring>
#include <initializer_list>

#include "../../include/slamhip.h"

namespace {

#define SLAMHIP_BOUND(X)                                                                                                         \
  X(last_error) X(rms_norm_fwd) X(rms_norm_bwd) X(rms_norm_bwd_workspace_bytes) X(quantize_fp8) X(quantize_fp8_blocks)           \
  X(gemm_nt_fp8) X(gemm_nt_fp8_workspace_bytes) X(causal_conv_fwd) X(causal_conv_bwd) X(causal_conv_bwd_workspace_bytes)         \
  X(selective_scan_kept_floats) X(selective_scan_fwd) X(selective_scan_fwd_workspace_bytes) X(selective_scan_bwd)                \
  X(selective_scan_bwd_workspace_bytes)

struct {
#define X(name) decltype(&slamhip_##name) name;
  SLAMHIP_BOUND(X)
#undef X
} lib;

[[noreturn]] void bad(const char* name, const at::Tensor* t, const std::string& want) {
  std::ostringstream got;
  if (t)
    got << t->dtype() << " " << t->sizes() << " on " << t->device() << ", strides " << t->strides();
  else
    got << "None";
  TORCH_CHECK_VALUE(false, name, ": expected ", want, ", got ", got.str());
}

std::string described(at::ScalarType type, at::IntArrayRef shape, c10::Device device) {
  std::ostringstream s;
  s << "a " << type << " tensor " << shape << " on " << device;
  return s.str();
}

const at::Tensor* tensor(PyObject* o, const char* name) {
  if (o == Py_None) return nullptr;
  TORCH_CHECK_VALUE(THPVariable_Check(o), name, ": expected a tensor, got ", Py_TYPE(o)->tp_name);
  return &THPVariable_Unpack(o);
}

int as_int(int64_t n, const char* name) {
  TORCH_CHECK_VALUE(n <= INT_MAX, name, ": more than 2^31 - 1 along an axis");
  return (int)n;
}

int type_code(at::ScalarType type) { return type == at::kBFloat16 ? SLAMHIP_BF16 : SLAMHIP_F32; }

bool is_value_type(at::ScalarType type) { return type == at::kBFloat16 || type == at::kFloat; }

// An activation, which says what type the others have and on which device they are.
const at::Tensor& leading(PyObject* o, const char* name, int dims) {
  const at::Tensor* t = tensor(o, name);
  if (!t || t->dim() != dims || !is_value_type(t->scalar_type()) || !t->is_cuda() || t->size(dims - 1) == 0)
    bad(name, t, dims == 3 ? "a float32 or bfloat16 GPU tensor [B, T, C] with channels" : "a float32 or bfloat16 GPU matrix with columns");
  return *t;
}

struct Call {
  c10::Device device;
  c10::DeviceGuard guard;
  at::Tensor workspace;
  size_t bytes = 0;
  static constexpr int kMost = 12;
  const char* names[kMost];
  const at::Tensor* sequences[kMost];
  void* addresses[kMost];
  long long strides[2 * kMost];
  int count = 0;

  explicit Call(const at::Tensor& t) : device(t.device()), guard(t.device()) {}

  // A contiguous tensor; its address, null for None.
  void* flat(PyObject* o, const char* name, at::ScalarType type, std::initializer_list<int64_t> shape) const {
    const at::Tensor* t = tensor(o, name);
    if (!t) return nullptr;
    const at::IntArrayRef want(shape.begin(), shape.size());
    if (t->scalar_type() != type || t->sizes() != want || t->device() != device || !t->is_contiguous())
      bad(name, t, "contiguous, " + described(type, want, device));
    return t->data_ptr();
  }

  void* need(PyObject* o, const char* name, at::ScalarType type, std::initializer_list<int64_t> shape) const {
    if (o == Py_None) bad(name, nullptr, described(type, at::IntArrayRef(shape.begin(), shape.size()), device));
    return flat(o, name, type, shape);
  }

  // A sequence [B, T, C] with unit stride over C; its strides over B and T join `strides`.  None has no address.
  void* sequence(PyObject* o, const char* name, at::ScalarType type, int64_t B, int64_t T, int64_t C, bool optional = false) {
    const at::Tensor* t = tensor(o, name);
    void* address = nullptr;
    long long sb = 0, st = 0;
    if (t || !optional) {
      const int64_t shape[3] = {B, T, C};
      if (!t || t->scalar_type() != type || t->sizes() != at::IntArrayRef(shape, 3) || t->device() != device)
        bad(name, t, described(type, at::IntArrayRef(shape, 3), device));
      if (t->stride(2) != 1 && C > 1) bad(name, t, "unit stride over the last axis");
      sb = t->stride(0);
      st = t->stride(1);
      address = t->data_ptr();
    }
    names[count] = name;
    sequences[count] = t;
    addresses[count] = address;
    strides[2 * count] = sb;
    strides[2 * count + 1] = st;
    ++count;
    return address;
  }

  // Sequences from `first` on are outputs: their rows do not overlap, and none begins where another sequence does (steps are
  // worked on at once).
  void outputs_from(int first) const {
    for (int i = first; i < count; ++i) {
      if (!addresses[i]) continue;
      const at::Tensor& t = *sequences[i];
      const int64_t B = t.size(0), T = t.size(1), C = t.size(2), sb = t.stride(0), st = t.stride(1);
      if ((T > 1 && st < C) || (B > 1 && sb < C) || (B > 1 && T > 1 && sb < (T - 1) * st + C && st < (B - 1) * sb + C))
        bad(names[i], &t, "rows that do not overlap");
      apart(addresses[i], names[i], 0, i);
    }
  }

  void apart(void* address, const char* name, int first, int last) const {
    if (address)
      for (int i = first; i < last; ++i) TORCH_CHECK_VALUE(address != addresses[i], name, " and ", names[i], " are the same memory");
  }

  // Launches f(workspace, its bytes, stream) without the interpreter's lock.
  template <typename F>
  PyObject* launch(const char* name, size_t workspace_bytes, F f) {
    int rc;
    bytes = workspace_bytes;
    {
      pybind11::gil_scoped_release free_interpreter;
      if (bytes) workspace = at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(device));
      rc = f(bytes ? workspace.data_ptr() : nullptr, bytes, (void*)c10::hip::getCurrentHIPStream(device.index()).stream());
    }
    if (rc != SLAMHIP_OK) {
      PyErr_Format(PyExc_RuntimeError, "%s failed (%d): %s", name, rc, lib.last_error());
      return nullptr;
    }
    Py_RETURN_NONE;
  }
};

void same(void* a, void* b, const char* a_name, const char* b_name) {
  TORCH_CHECK_VALUE(!a || a != b, a_name, " and ", b_name, " are the same memory");
}

#define BINDING(name, arguments)                                                                             \
  PyObject* name(PyObject*, PyObject* const* arg, Py_ssize_t given) {                                        \
    HANDLE_TH_ERRORS                                                                                         \
    TORCH_CHECK_TYPE(given == arguments, #name ": takes ", arguments, " arguments, got ", given);            \
    TORCH_CHECK(lib.last_error, #name ": not bound to a library");

#define END_BINDING \
  END_HANDLE_TH_ERRORS \
  }

const at::Tensor& matrix(PyObject* o, const char* name) {
  const at::Tensor& t = leading(o, name, 2);
  if (!t.is_contiguous()) bad(name, &t, "a contiguous float32 or bfloat16 GPU matrix with columns");
  return t;
}

// x, weight, eps, y, residual, sum_out, y8, scales, rstd
BINDING(rms_norm_fwd, 9)
  const at::Tensor& x = matrix(arg[0], "x");
  Call c(x);
  const at::ScalarType type = x.scalar_type();
  const int64_t rows = x.size(0);
  const int C = as_int(x.size(1), "x");
  const double eps = PyFloat_AsDouble(arg[2]);
  if (eps == -1.0 && PyErr_Occurred()) return nullptr;
  void* weight = c.need(arg[1], "weight", at::kFloat, {C});
  void* y = c.flat(arg[3], "y", type, {rows, C});
  void* residual = c.flat(arg[4], "residual", type, {rows, C});
  void* sum = c.flat(arg[5], "sum_out", type, {rows, C});
  void* y8 = c.flat(arg[6], "y8", at::kFloat8_e4m3fn, {rows, C});
  void* scales = c.flat(arg[7], "scales", at::kFloat, {rows, (C + 127LL) / 128});
  void* rstd = c.flat(arg[8], "rstd", at::kFloat, {rows});
  same(y, sum, "y", "sum_out");
  return c.launch("slamhip_rms_norm_fwd", 0, [&](void*, size_t, void* stream) {
    return lib.rms_norm_fwd(x.data_ptr(), residual, (float*)weight, (float)eps, rows, C, type_code(type), sum, y, y8,
                            (float*)scales, (float*)rstd, stream);
  });
END_BINDING

// dy, sum, weight, rstd, dx, dweight, d_sum
BINDING(rms_norm_bwd, 7)
  const at::Tensor& sum = matrix(arg[1], "sum");
  Call c(sum);
  const at::ScalarType type = sum.scalar_type();
  const int64_t rows = sum.size(0);
  const int C = as_int(sum.size(1), "sum");
  void* dy = c.need(arg[0], "dy", type, {rows, C});
  void* weight = c.need(arg[2], "weight", at::kFloat, {C});
  void* rstd = c.need(arg[3], "rstd", at::kFloat, {rows});
  void* dx = c.need(arg[4], "dx", type, {rows, C});
  void* dweight = c.need(arg[5], "dweight", at::kFloat, {C});
  void* d_sum = c.flat(arg[6], "d_sum", type, {rows, C});
  same(dweight, weight, "dweight", "weight");
  return c.launch("slamhip_rms_norm_bwd", lib.rms_norm_bwd_workspace_bytes(rows, C), [&](void* ws, size_t bytes, void* stream) {
    return lib.rms_norm_bwd(dy, sum.data_ptr(), (float*)weight, (float*)rstd, d_sum, rows, C, type_code(type), dx, (float*)dweight, ws, bytes,
                            stream);
  });
END_BINDING

// x, q, scales
BINDING(quantize_fp8, 3)
  const at::Tensor& x = matrix(arg[0], "x");
  Call c(x);
  const int64_t rows = x.size(0);
  const int C = as_int(x.size(1), "x");
  void* q = c.need(arg[1], "q", at::kFloat8_e4m3fn, {rows, C});
  void* scales = c.need(arg[2], "scales", at::kFloat, {rows, (C + 127LL) / 128});
  return c.launch("slamhip_quantize_fp8", 0, [&](void*, size_t, void* stream) {
    return lib.quantize_fp8(x.data_ptr(), rows, C, type_code(x.scalar_type()), q, (float*)scales, stream);
  });
END_BINDING

BINDING(quantize_fp8_blocks, 3)
  const at::Tensor& x = matrix(arg[0], "x");
  Call c(x);
  const int R = as_int(x.size(0), "x"), C = as_int(x.size(1), "x");
  void* q = c.need(arg[1], "q", at::kFloat8_e4m3fn, {R, C});
  void* scales = c.need(arg[2], "scales", at::kFloat, {(R + 127LL) / 128, (C + 127LL) / 128});
  return c.launch("slamhip_quantize_fp8_blocks", 0, [&](void*, size_t, void* stream) {
    return lib.quantize_fp8_blocks(x.data_ptr(), R, C, type_code(x.scalar_type()), q, (float*)scales, stream);
  });
END_BINDING

// a8, a_scales, b8, b_scales, out
BINDING(gemm_nt_fp8, 5)
  const at::Tensor *out = tensor(arg[4], "out"), *a = tensor(arg[0], "a8");
  if (!out || out->dim() != 2 || !out->is_cuda()) bad("out", out, "a bfloat16 GPU matrix");
  if (!a || a->dim() != 2 || a->size(1) == 0) bad("a8", a, "a matrix with columns");
  Call c(*out);
  const int M = as_int(out->size(0), "out"), N = as_int(out->size(1), "out"), K = as_int(a->size(1), "a8");
  const int64_t kb = (K + 127LL) / 128;
  void* a8 = c.need(arg[0], "a8", at::kFloat8_e4m3fn, {M, K});
  void* a_scales = c.need(arg[1], "a_scales", at::kFloat, {M, kb});
  void* b8 = c.need(arg[2], "b8", at::kFloat8_e4m3fn, {N, K});
  void* b_scales = c.need(arg[3], "b_scales", at::kFloat, {(N + 127LL) / 128, kb});
  void* to = c.need(arg[4], "out", at::kBFloat16, {M, N});
  TORCH_CHECK_VALUE(K % 16 == 0 && (uintptr_t)a8 % 16 == 0 && (uintptr_t)b8 % 16 == 0,
                    "gemm_nt_fp8: K must be a multiple of 16 and the operands 16-byte aligned, got K = ", K);
  return c.launch("slamhip_gemm_nt_fp8", lib.gemm_nt_fp8_workspace_bytes(M, N, K), [&](void* ws, size_t bytes, void* stream) {
    return lib.gemm_nt_fp8(a8, (float*)a_scales, b8, (float*)b_scales, M, N, K, to, ws, bytes, stream);
  });
END_BINDING

int taps(PyObject* o, int64_t C) {
  const at::Tensor* w = tensor(o, "weight");
  if (!w || w->dim() != 2 || w->size(1) < 2 || w->size(1) > 4) bad("weight", w, "[" + std::to_string(C) + ", K] with 2 <= K <= 4");
  return (int)w->size(1);
}

// x, weight, bias, y, state_in, state_out, lengths, silu
BINDING(causal_conv_fwd, 8)
  const at::Tensor& x = leading(arg[0], "x", 3);
  Call c(x);
  const at::ScalarType type = x.scalar_type();
  const int B = as_int(x.size(0), "x"), T = as_int(x.size(1), "x"), C = as_int(x.size(2), "x"), K = taps(arg[1], C);
  void* xp = c.sequence(arg[0], "x", type, B, T, C);
  void* y = c.sequence(arg[3], "y", type, B, T, C);
  c.outputs_from(1);
  void* weight = c.need(arg[1], "weight", at::kFloat, {C, K});
  void* bias = c.flat(arg[2], "bias", at::kFloat, {C});
  void* state_in = c.flat(arg[4], "state_in", type, {B, K - 1, C});
  void* state_out = c.flat(arg[5], "state_out", type, {B, K - 1, C});
  void* lengths = c.flat(arg[6], "lengths", at::kInt, {B});
  c.apart(state_in, "state_in", 1, 2);
  c.apart(state_out, "state_out", 0, 2);
  const int silu = PyObject_IsTrue(arg[7]);
  if (silu < 0) return nullptr;
  return c.launch("slamhip_causal_conv_fwd", 0, [&](void*, size_t, void* stream) {
    return lib.causal_conv_fwd(xp, c.strides, (float*)weight, (float*)bias, state_in, (int32_t*)lengths, B, T, C, K, silu, type_code(type), y,
                               state_out, stream);
  });
END_BINDING

// dy, x, weight, bias, dx, dweight, dbias, state_in, d_state_in, d_state_out, lengths, silu
BINDING(causal_conv_bwd, 12)
  const at::Tensor& x = leading(arg[1], "x", 3);
  Call c(x);
  const at::ScalarType type = x.scalar_type();
  const int B = as_int(x.size(0), "x"), T = as_int(x.size(1), "x"), C = as_int(x.size(2), "x"), K = taps(arg[2], C);
  void* dy = c.sequence(arg[0], "dy", type, B, T, C);
  void* xp = c.sequence(arg[1], "x", type, B, T, C);
  void* dx = c.sequence(arg[4], "dx", type, B, T, C);
  c.outputs_from(2);
  void* weight = c.need(arg[2], "weight", at::kFloat, {C, K});
  void* bias = c.flat(arg[3], "bias", at::kFloat, {C});
  void* dweight = c.need(arg[5], "dweight", at::kFloat, {C, K});
  void* dbias = c.flat(arg[6], "dbias", at::kFloat, {C});
  void* state_in = c.flat(arg[7], "state_in", type, {B, K - 1, C});
  void* d_state_in = c.flat(arg[8], "d_state_in", type, {B, K - 1, C});
  void* d_state_out = c.flat(arg[9], "d_state_out", type, {B, K - 1, C});
  void* lengths = c.flat(arg[10], "lengths", at::kInt, {B});
  c.apart(state_in, "state_in", 2, 3);
  c.apart(d_state_out, "d_state_out", 2, 3);
  c.apart(d_state_in, "d_state_in", 0, 3);
  same(d_state_in, state_in, "d_state_in", "state_in");
  same(d_state_in, d_state_out, "d_state_in", "d_state_out");
  const int silu = PyObject_IsTrue(arg[11]);
  if (silu < 0) return nullptr;
  return c.launch("slamhip_causal_conv_bwd", lib.causal_conv_bwd_workspace_bytes(B, T, C, K), [&](void* ws, size_t bytes, void* stream) {
    return lib.causal_conv_bwd(dy, xp, c.strides, (float*)weight, (float*)bias, state_in, d_state_out, (int32_t*)lengths, B, T, C, K, silu,
                               type_code(type), dx, (float*)dweight, (float*)dbias, d_state_in, ws, bytes, stream);
  });
END_BINDING

int states(PyObject* o, int64_t C) {
  const at::Tensor* A = tensor(o, "A");
  if (!A || A->dim() != 2 || A->size(1) < 1 || A->size(1) > 32) bad("A", A, "[" + std::to_string(C) + ", N] with 1 <= N <= 32");
  return (int)A->size(1);
}

// u, delta, A, Bm, Cm, y, D, z, delta_bias, softplus, state_in, state_out, kept_states, lengths
BINDING(selective_scan_fwd, 14)
  const at::Tensor& lead = leading(arg[0], "u", 3);
  Call c(lead);
  const at::ScalarType type = lead.scalar_type();
  const int B = as_int(lead.size(0), "u"), T = as_int(lead.size(1), "u"), C = as_int(lead.size(2), "u"), N = states(arg[2], C);
  void* u = c.sequence(arg[0], "u", type, B, T, C);
  void* delta = c.sequence(arg[1], "delta", type, B, T, C);
  void* z = c.sequence(arg[7], "z", type, B, T, C, true);
  void* Bm = c.sequence(arg[3], "Bm", type, B, T, N);
  void* Cm = c.sequence(arg[4], "Cm", type, B, T, N);
  void* y = c.sequence(arg[5], "y", type, B, T, C);
  c.outputs_from(5);
  void* A = c.need(arg[2], "A", at::kFloat, {C, N});
  void* D = c.flat(arg[6], "D", at::kFloat, {C});
  void* bias = c.flat(arg[8], "delta_bias", at::kFloat, {C});
  void* state_in = c.flat(arg[10], "state_in", at::kFloat, {B, C, N});
  void* state_out = c.flat(arg[11], "state_out", at::kFloat, {B, C, N});
  void* kept = nullptr;
  if (arg[12] != Py_None) kept = c.flat(arg[12], "kept_states", at::kFloat, {(int64_t)lib.selective_scan_kept_floats(B, T, C, N)});
  void* lengths = c.flat(arg[13], "lengths", at::kInt, {B});
  c.apart(state_in, "state_in", 5, 6);
  c.apart(state_out, "state_out", 0, 6);
  const int softplus = PyObject_IsTrue(arg[9]);
  if (softplus < 0) return nullptr;
  return c.launch("slamhip_selective_scan_fwd", lib.selective_scan_fwd_workspace_bytes(B, T, C, N), [&](void* ws, size_t bytes, void* stream) {
    return lib.selective_scan_fwd(u, delta, z, Bm, Cm, c.strides, (float*)A, (float*)D, (float*)bias, (float*)state_in, (int32_t*)lengths, B, T,
                                  C, N, softplus, type_code(type), y, (float*)state_out, (float*)kept, ws, bytes, stream);
  });
END_BINDING

// dy, u, delta, A, Bm, Cm, kept_states, du, ddelta, dA, dB, dC, D, z, delta_bias, softplus, dD, dz, d_delta_bias, d_state_in, d_state_out, lengths
BINDING(selective_scan_bwd, 22)
  const at::Tensor& lead = leading(arg[1], "u", 3);
  TORCH_CHECK_VALUE((arg[13] == Py_None) == (arg[17] == Py_None), "selective_scan_bwd: dz is wanted exactly when there is z");
  Call c(lead);
  const at::ScalarType type = lead.scalar_type();
  const int B = as_int(lead.size(0), "u"), T = as_int(lead.size(1), "u"), C = as_int(lead.size(2), "u"), N = states(arg[3], C);
  void* dy = c.sequence(arg[0], "dy", type, B, T, C);
  void* u = c.sequence(arg[1], "u", type, B, T, C);
  void* delta = c.sequence(arg[2], "delta", type, B, T, C);
  void* z = c.sequence(arg[13], "z", type, B, T, C, true);
  void* Bm = c.sequence(arg[4], "Bm", type, B, T, N);
  void* Cm = c.sequence(arg[5], "Cm", type, B, T, N);
  void* du = c.sequence(arg[7], "du", type, B, T, C);
  void* ddelta = c.sequence(arg[8], "ddelta", type, B, T, C);
  void* dz = c.sequence(arg[17], "dz", type, B, T, C, true);
  void* dB = c.sequence(arg[10], "dB", type, B, T, N);
  void* dC = c.sequence(arg[11], "dC", type, B, T, N);
  c.outputs_from(6);
  void* A = c.need(arg[3], "A", at::kFloat, {C, N});
  void* kept = c.need(arg[6], "kept_states", at::kFloat, {(int64_t)lib.selective_scan_kept_floats(B, T, C, N)});
  void* dA = c.need(arg[9], "dA", at::kFloat, {C, N});
  void* D = c.flat(arg[12], "D", at::kFloat, {C});
  void* bias = c.flat(arg[14], "delta_bias", at::kFloat, {C});
  void* dD = c.flat(arg[16], "dD", at::kFloat, {C});
  void* d_bias = c.flat(arg[18], "d_delta_bias", at::kFloat, {C});
  void* d_state_in = c.flat(arg[19], "d_state_in", at::kFloat, {B, C, N});
  void* d_state_out = c.flat(arg[20], "d_state_out", at::kFloat, {B, C, N});
  void* lengths = c.flat(arg[21], "lengths", at::kInt, {B});
  c.apart(d_state_in, "d_state_in", 0, 11);
  c.apart(d_state_out, "d_state_out", 6, 11);
  same(d_state_in, d_state_out, "d_state_in", "d_state_out");
  const int softplus = PyObject_IsTrue(arg[15]);
  if (softplus < 0) return nullptr;
  return c.launch("slamhip_selective_scan_bwd", lib.selective_scan_bwd_workspace_bytes(B, T, C, N), [&](void* ws, size_t bytes, void* stream) {
    return lib.selective_scan_bwd(dy, u, delta, z, Bm, Cm, c.strides, (float*)A, (float*)D, (float*)bias, (float*)kept, (float*)d_state_out,
                                  (int32_t*)lengths, B, T, C, N, softplus, type_code(type), du, ddelta, dz, dB, dC, (float*)dA, (float*)dD,
                                  (float*)d_bias, (float*)d_state_in, ws, bytes, stream);
  });
END_BINDING

// {name: address} of the library's functions
PyObject* bind(PyObject*, PyObject* addresses) {
  HANDLE_TH_ERRORS
#define X(name)                                                                                     \
  {                                                                                                 \
    PyObject* o = PyMapping_GetItemString(addresses, "slamhip_" #name);                             \
    if (!o) return nullptr;                                                                         \
    void* p = PyLong_AsVoidPtr(o);                                                                  \
    Py_DECREF(o);                                                                                   \
    if (PyErr_Occurred()) return nullptr;                                                           \
    std::memcpy(&lib.name, &p, sizeof(p));                                                          \
  }
  SLAMHIP_BOUND(X)
#undef X
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(rms_norm_fwd),       METHOD(rms_norm_bwd),       METHOD(quantize_fp8),
                         METHOD(quantize_fp8_blocks), METHOD(gemm_nt_fp8),        METHOD(causal_conv_fwd),
                         METHOD(causal_conv_bwd),    METHOD(selective_scan_fwd), METHOD(selective_scan_bwd),
                         {"bind", bind, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_sequence", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__sequence() { return PyModule_Create(&module); }
