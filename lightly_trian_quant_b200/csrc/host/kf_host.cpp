// Host side of the operator layer (ops.py) as a CPython extension: argument checks, output allocation, the current stream
// and the call into the C-ABI (libkf_b200.so) in one native call per operator.
//
// What bounds it: a small model called eagerly is a hundred launches of 3 to 10 us each, and the same steps in Python
// (attribute and dict look-ups, a ctypes structure of 30 fields, a stream object, a closure) took 12 to 16 us per operator.
// Here an operator costs its launch (about 2 us), one allocation where it returns a new tensor and about 1 us for the rest.
//
// Containers are the Python ones: an operand is any object with the attributes M, K, fmt, q, sf, ts (ops.ActBuf), a weight any
// object with N, K, fmt, q, sf, ts and optionally settled (ops.QWeight).  Errors are KfError of the package.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdarg>
#include <vector>

#include "../../../include/kf_b200.h"

namespace {

PyObject* g_error = nullptr;                                   // KfError
PyObject *s_M, *s_N, *s_K, *s_fmt, *s_q, *s_sf, *s_ts, *s_settled;         // interned attribute names
PyObject* g_fmt_names[4];                                      // interned "mx8", "nv4", "mx4", "bf16": index = KF_FMT_*

struct Failed {};                                              // a Python exception is set

[[noreturn]] void fail(const char* format, ...) {
  va_list ap;
  va_start(ap, format);
  PyErr_FormatV(g_error, format, ap);
  va_end(ap);
  throw Failed{};
}

void need(bool cond, const char* what) {
  if (!cond) fail("%s", what);
}

const at::Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) fail("%s must be a tensor", what);
  return THPVariable_Unpack(o);
}

const char* const NO_CPU = "operands must live on a CUDA device (there is no CPU path)";

const at::Tensor& cuda_tensor(PyObject* o, const char* what) {
  const at::Tensor& t = tensor(o, what);
  if (!t.is_cuda()) fail("%s", NO_CPU);
  return t;
}

[[noreturn]] void divides_by_zero(const char* what) {          // what Python arithmetic on the shapes raises
  PyErr_SetString(PyExc_ZeroDivisionError, what);
  throw Failed{};
}

// rows of x seen as [rows, d]
int64_t rows_of(const at::Tensor& x, int64_t d, const char* what) {
  if (d == 0) divides_by_zero(what);
  return x.numel() / d;
}

at::Tensor opt_tensor(PyObject* o, const char* what) { return o == Py_None ? at::Tensor() : cuda_tensor(o, what); }
// pointer of an optional CUDA tensor (None = null)
void* opt_ptr(PyObject* o, const char* what) { return o == Py_None ? nullptr : cuda_tensor(o, what).data_ptr(); }

// An owned reference: an attribute may be a property, whose value nobody else holds.
class Ref {
 public:
  explicit Ref(PyObject* p) : p_(p) {}
  Ref(Ref&& o) noexcept : p_(o.p_) { o.p_ = nullptr; }
  Ref(const Ref&) = delete;
  Ref& operator=(const Ref&) = delete;
  ~Ref() { Py_XDECREF(p_); }
  operator PyObject*() const { return p_; }

 private:
  PyObject* p_;
};

Ref attr(PyObject* o, PyObject* name) {
  PyObject* v = PyObject_GetAttr(o, name);
  if (!v) throw Failed{};
  return Ref(v);
}

int64_t to_int(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Failed{};
  return v;
}

double to_float(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Failed{};
  return v;
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Failed{};
  return v != 0;
}

int fmt_code(PyObject* name) {
  for (int i = 0; i < 4; ++i)
    if (name == g_fmt_names[i]) return i;
  if (PyUnicode_Check(name))
    for (int i = 0; i < 4; ++i)
      if (PyUnicode_Compare(name, g_fmt_names[i]) == 0) return i;
  fail("unknown operand format %R", name);
}

struct Operand {                                               // ActBuf or QWeight; holds its tensors until the launch is made
  int fmt;
  int64_t rows, K;
  at::Tensor q, sf, ts;                                        // sf: undefined for bf16, ts: undefined unless nv4
  void *pq, *psf, *pts;
};

Operand operand(PyObject* o, PyObject* rows_attr, const char* what) {
  Operand r;
  r.rows = to_int(attr(o, rows_attr));
  r.K = to_int(attr(o, s_K));
  r.fmt = fmt_code(attr(o, s_fmt));
  r.q = cuda_tensor(attr(o, s_q), what);
  r.pq = r.q.data_ptr();
  r.sf = opt_tensor(attr(o, s_sf), what);
  r.psf = r.sf.defined() ? r.sf.data_ptr() : nullptr;
  r.ts = opt_tensor(attr(o, s_ts), what);
  r.pts = r.ts.defined() ? r.ts.data_ptr() : nullptr;
  return r;
}
Operand act(PyObject* o, const char* what) { return operand(o, s_M, what); }
Operand weight(PyObject* o) { return operand(o, s_N, "weight"); }

int dtype_code(at::ScalarType t) { return t == at::kFloat ? KF_F32 : t == at::kBFloat16 ? KF_BF16 : t == at::kHalf ? KF_F16 : -1; }
at::ScalarType dtype_of(int code) { return code == KF_F32 ? at::kFloat : code == KF_BF16 ? at::kBFloat16 : at::kHalf; }

// fp32, contiguous, n elements; None passes
const float* f32_vec(PyObject* o, int64_t n, const char* what) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, what);
  if (t.scalar_type() != at::kFloat || !t.is_contiguous() || t.numel() != n) fail("gemm: %s must be contiguous fp32 with %lld elements", what, (long long)n);
  if (!t.is_cuda()) fail("%s", NO_CPU);
  return t.data_ptr<float>();
}

void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

void check(int status, const char* what) {
  if (status != 0) fail("%s failed with status %d: %s", what, status, kf_last_error_string());
}

// Other threads run while this one is inside an allocation or the library: a launch blocks when the stream's queue is full.
class Unlocked {
 public:
  Unlocked() : state_(PyEval_SaveThread()) {}
  Unlocked(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state_); }

 private:
  PyThreadState* state_;
};

// fn(args...) of the C-ABI without the interpreter lock; the arguments have been worked out with it
template <typename... P, typename... A>
void launch(const char* what, int (*fn)(P...), A... args) {
  int status;
  {
    const Unlocked unlocked;
    status = fn(args...);
  }
  check(status, what);
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType dtype, at::Device device) {
  const Unlocked unlocked;
  return at::Tensor(at::detail::empty_cuda(sizes, dtype, device, std::nullopt));
}

// `n` elements of t from `first` on as a tensor of its own: an allocation costs about 0.7 us of host time, this 0.1
at::Tensor piece(const at::Tensor& t, int64_t first, int64_t n) {
  auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(t.storage()), t.key_set(), t.dtype());
  impl->set_storage_offset(first);
  impl->set_sizes_contiguous({n});
  return at::Tensor(std::move(impl));
}

PyObject* new_ref(PyObject* o) {
  Py_INCREF(o);
  return o;
}

PyObject* pair(at::Tensor a, at::Tensor b) {
  PyObject *x = THPVariable_Wrap(std::move(a)), *y = THPVariable_Wrap(std::move(b));
  PyObject* t = PyTuple_New(2);
  PyTuple_SET_ITEM(t, 0, x);
  PyTuple_SET_ITEM(t, 1, y);
  return t;
}

// ------------------------------------------------------------------------------------------------ GEMM
// KF_G_W_STATIC lets the kernel read weights before the wait that makes the predecessor's writes visible, so it is claimed only for
// weights whose writes the host has seen complete and that nothing has written since: `settled` is (q, sf, sum of their version counters)
// at that moment (ops.settled), None where the host did not wait.  torch counts its in-place writes, writable() those of the operators
// here; other tensors in the place of those two, or an object without the attribute, claim nothing.  bmm_nt takes activations and does
// not claim it either.
bool weight_settled(PyObject* o, const at::Tensor& q, const at::Tensor& sf) {
  PyObject* p = PyObject_GetAttr(o, s_settled);
  if (!p) {
    if (!PyErr_ExceptionMatches(PyExc_AttributeError)) throw Failed{};
    PyErr_Clear();
    return false;
  }
  const Ref seen(p);
  if (!PyTuple_Check(p) || PyTuple_GET_SIZE(p) != 3) return false;
  auto same = [&](Py_ssize_t i, const at::Tensor& t) {
    PyObject* held = PyTuple_GET_ITEM(p, i);
    return t.defined() ? THPVariable_Check(held) && THPVariable_Unpack(held).is_same(t) : held == Py_None;
  };
  if (!same(0, q) || !same(1, sf) || q.is_inference() || (sf.defined() && sf.is_inference())) return false;   // an inference tensor has no version counter
  return (int64_t)q._version() + (sf.defined() ? (int64_t)sf._version() : 0) == to_int(PyTuple_GET_ITEM(p, 2));
}
int w_static(PyObject* o, const Operand& W) { return weight_settled(o, W.q, W.sf) ? KF_G_W_STATIC : 0; }

// out is about to be written: counted as torch counts an in-place operation
void writable(const at::Tensor& out) {
  if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
}
void writable(const Operand& out) {
  writable(out.q);
  if (out.sf.defined()) writable(out.sf);
}
// A side, W side and the common fields; returns M
int64_t gemm_fill(kf_gemm_params& p, PyObject* a, const Operand& W, int epi) {
  int64_t M;
  if (THPVariable_Check(a)) {
    const at::Tensor& t = THPVariable_Unpack(a);
    if (W.fmt != KF_FMT_BF16 || t.scalar_type() != at::kBFloat16 || t.dim() != 2 || !t.is_contiguous() || t.size(1) != W.K)
      fail("gemm: a plain tensor operand must be contiguous bf16 [M, K] with a bf16 weight");
    if (!t.is_cuda()) fail("%s", NO_CPU);
    M = t.size(0);
    p.A = t.data_ptr();
  } else {
    const Operand A = act(a, "gemm operand");
    if (A.fmt != W.fmt || A.K != W.K) fail("gemm: operand mismatch A %U K=%lld vs W %U K=%lld", g_fmt_names[A.fmt], (long long)A.K, g_fmt_names[W.fmt], (long long)W.K);
    M = A.rows;
    p.A = A.pq;
    p.SFA = A.psf;
    p.ts_a = static_cast<const float*>(A.pts);
  }
  p.fmt = W.fmt;
  p.epi = epi;
  p.M = (int)M;
  p.N = (int)W.rows;
  p.K = (int)W.K;
  p.W = W.pq;
  p.SFW = W.psf;
  p.ts_w = static_cast<const float*>(W.pts);
  return M;
}

void gemm_run(const kf_gemm_params& p, const char* what) { launch(what, kf_gemm_bs, &p, stream()); }

// a, W, bias, out | None, out dtype code, flags
PyObject* gemm_plain(PyObject* const* v) {
  const Operand W = weight(v[1]);
  kf_gemm_params p = {};
  const float* bias = f32_vec(v[2], W.rows, "bias");
  const int64_t M = gemm_fill(p, v[0], W, KF_EPI_PLAIN);
  p.bias = bias;
  p.flags = (int)to_int(v[5]) | w_static(v[1], W);
  if (v[3] == Py_None) {
    p.out_dtype = (int)to_int(v[4]);
    at::Tensor out = empty({M, W.rows}, dtype_of(p.out_dtype), W.q.device());
    p.C = out.data_ptr();
    gemm_run(p, "gemm_plain");
    return THPVariable_Wrap(std::move(out));
  }
  const at::Tensor& out = cuda_tensor(v[3], "out");
  p.out_dtype = dtype_code(out.scalar_type());
  p.C = out.data_ptr();
  writable(out);
  gemm_run(p, "gemm_plain");
  return new_ref(v[3]);
}

// (group, stride, offset) as any iterable of three integers
struct RowMap {
  int group, stride, offset;
};
RowMap row_map(PyObject* o) {
  PyObject* seq = PySequence_Fast(o, "gemm_res: row_map must be (group, stride, offset)");
  if (!seq) throw Failed{};
  int value[3] = {0, 0, 0};
  bool ok = PySequence_Fast_GET_SIZE(seq) == 3;
  if (!ok) PyErr_Format(PyExc_ValueError, "gemm_res: row_map must be (group, stride, offset), got %zd values", PySequence_Fast_GET_SIZE(seq));
  for (int i = 0; ok && i < 3; ++i) {
    const long n = PyLong_AsLong(PySequence_Fast_GET_ITEM(seq, i));
    ok = !(n == -1 && PyErr_Occurred());
    if (ok && n != (int)n) {
      PyErr_Format(PyExc_OverflowError, "gemm_res: row_map value %ld does not fit a 32-bit integer", n);
      ok = false;
    }
    value[i] = (int)n;
  }
  Py_DECREF(seq);
  if (!ok) throw Failed{};
  if (value[0] == 0) divides_by_zero("gemm_res: row_map with a group of 0 rows");
  return {value[0], value[1], value[2]};
}

// a, W, bias, gamma, res, out | None, row_map | None
PyObject* gemm_res(PyObject* const* v) {
  const Operand W = weight(v[1]);
  kf_gemm_params p = {};
  const float* bias = f32_vec(v[2], W.rows, "bias");
  const float* gamma = f32_vec(v[3], W.rows, "gamma");
  const int64_t M = gemm_fill(p, v[0], W, KF_EPI_RES);
  p.bias = bias;
  p.gamma = gamma;
  p.flags = w_static(v[1], W);
  p.R = f32_vec(v[4], M * W.rows, "res");
  p.out_dtype = KF_F32;
  if (v[5] == Py_None) {
    if (v[6] != Py_None) fail("gemm_res: a row mapping needs the output tensor");
    const at::Tensor& res = tensor(v[4], "res");
    at::Tensor out = [&] {
      const Unlocked unlocked;
      return at::empty_like(res);
    }();
    p.C = out.data_ptr();
    gemm_run(p, "gemm_res");
    return THPVariable_Wrap(std::move(out));
  }
  const at::Tensor& out = cuda_tensor(v[5], "out");
  need(out.scalar_type() == at::kFloat && out.is_contiguous(), "gemm_res: out must be contiguous fp32");
  if (v[6] != Py_None) {
    const RowMap m = row_map(v[6]);
    if (M % m.group || out.numel() != (M / m.group) * m.stride * W.rows || (int64_t)m.offset + m.group > m.stride)
      fail("gemm_res: row mapping (%d, %d, %d) does not fit M=%lld rows into an output of %lld values", m.group, m.stride, m.offset, (long long)M, (long long)out.numel());
    p.out_row_group = m.group;
    p.out_row_stride = m.stride;
    p.out_row_offset = m.offset;
  }
  p.C = out.data_ptr();
  writable(out);
  gemm_run(p, "gemm_res");
  return new_ref(v[5]);
}

// a, W, bias, sin, cos, Ntok, prefix, H, out dtype code, flags
PyObject* qkv_rope(PyObject* const* v) {
  const Operand W = weight(v[1]);
  kf_gemm_params p = {};
  const float* bias = f32_vec(v[2], W.rows, "bias");
  const at::Tensor &sin = tensor(v[3], "sin"), &cos = tensor(v[4], "cos");
  const int64_t Ntok = to_int(v[5]), prefix = to_int(v[6]), H = to_int(v[7]);
  need(sin.scalar_type() == at::kFloat && cos.scalar_type() == at::kFloat && sin.is_contiguous() && cos.is_contiguous() && sin.dim() > 0 && sin.size(-1) == 64 &&
           sin.size(0) >= Ntok - prefix && cos.sizes() == sin.sizes(),
       "qkv_rope: sin / cos must be contiguous fp32 [>= Ntok - prefix, 64]");
  need(sin.is_cuda() && cos.is_cuda(), NO_CPU);
  const int64_t M = gemm_fill(p, v[0], W, KF_EPI_ROPE);
  need(Ntok > 0 && M % Ntok == 0, "qkv_rope: M must be a multiple of Ntok");
  p.bias = bias;
  p.sin = sin.data_ptr<float>();
  p.cos = cos.data_ptr<float>();
  p.Ntok = (int)Ntok;
  p.prefix = (int)prefix;
  p.H = (int)H;
  p.out_dtype = (int)to_int(v[8]);
  p.flags = (int)to_int(v[9]) | w_static(v[1], W);
  at::Tensor out = empty({3, M / Ntok, Ntok, H, 64}, dtype_of(p.out_dtype), W.q.device());
  p.C = out.data_ptr();
  gemm_run(p, "qkv_rope");
  return THPVariable_Wrap(std::move(out));
}

// a, W, bias, out (ActBuf), flags, y_dbg | None
PyObject* gemm_gelu_q(PyObject* const* v) {
  const Operand W = weight(v[1]);
  kf_gemm_params p = {};
  const float* bias = f32_vec(v[2], W.rows, "bias");
  const int64_t M = gemm_fill(p, v[0], W, KF_EPI_QUANT);
  const Operand out = act(v[3], "out");
  if (out.rows != M || out.K != W.rows)
    fail("gemm_gelu_q: out must be [%lld, %lld], got [%lld, %lld]", (long long)M, (long long)W.rows, (long long)out.rows, (long long)out.K);
  p.bias = bias;
  p.y_dbg = const_cast<float*>(f32_vec(v[5], M * W.rows, "y_dbg"));
  p.out_dtype = KF_BF16;
  p.out_fmt = out.fmt;
  p.Qo = out.pq;
  p.SFo = out.psf;
  p.tso = static_cast<const float*>(out.pts);
  p.flags = (int)to_int(v[4]) | w_static(v[1], W);
  writable(out);
  gemm_run(p, "gemm_gelu_q");
  return new_ref(v[3]);
}

// a [B, Q, K], w [B, P, K], out | None
PyObject* bmm_nt(PyObject* const* v) {
  const at::Tensor &a = cuda_tensor(v[0], "a"), &w = cuda_tensor(v[1], "w");
  need(a.dim() == 3 && w.dim() == 3 && a.scalar_type() == at::kBFloat16 && w.scalar_type() == at::kBFloat16 && a.is_contiguous() && w.is_contiguous() &&
           a.size(0) == w.size(0) && a.size(2) == w.size(2),
       "bmm_nt: a [B, Q, K] and w [B, P, K] must be contiguous bf16 with equal B and K");
  const int64_t B = a.size(0), Q = a.size(1), K = a.size(2), P = w.size(1);
  at::Tensor out;
  if (v[2] == Py_None) {
    out = empty({B, Q, P}, at::kBFloat16, a.device());
  } else {
    out = cuda_tensor(v[2], "out");
    if (out.dim() != 3 || out.size(0) != B || out.size(1) != Q || out.size(2) != P || out.scalar_type() != at::kBFloat16 || !out.is_contiguous())
      fail("bmm_nt: out must be contiguous bf16 [%lld, %lld, %lld]", (long long)B, (long long)Q, (long long)P);
    writable(out);
  }
  kf_gemm_params p = {};
  p.fmt = KF_FMT_BF16;
  p.epi = KF_EPI_PLAIN;
  p.M = (int)(B * Q);
  p.N = (int)P;
  p.K = (int)K;
  p.A = a.data_ptr();
  p.W = w.data_ptr();
  p.C = out.data_ptr();
  p.out_dtype = KF_BF16;
  p.batch = (int)B;
  p.a_rows_per_batch = (int)Q;
  p.w_rows_per_batch = (int)P;
  gemm_run(p, "bmm_nt");
  return v[2] == Py_None ? THPVariable_Wrap(std::move(out)) : new_ref(v[2]);
}

// a, W, bias, out, rows per image, tokens per image, row offset, flags
PyObject* gemm_tokens(PyObject* const* v) {
  const at::Tensor &a = cuda_tensor(v[0], "a"), &out = cuda_tensor(v[3], "out");
  const Operand W = weight(v[1]);
  need(out.scalar_type() == at::kFloat && out.is_contiguous(), "gemm_tokens: out must be contiguous fp32");
  kf_gemm_params p = {};
  p.fmt = KF_FMT_BF16;
  p.epi = KF_EPI_PLAIN;
  p.M = (int)a.size(0);
  p.N = (int)W.rows;
  p.K = (int)W.K;
  p.A = a.data_ptr();
  p.W = W.pq;
  p.bias = static_cast<const float*>(opt_ptr(v[2], "bias"));
  p.C = out.data_ptr();
  p.out_dtype = KF_F32;
  p.out_row_group = (int)to_int(v[4]);
  p.out_row_stride = (int)to_int(v[5]);
  p.out_row_offset = (int)to_int(v[6]);
  p.flags = (int)to_int(v[7]) | w_static(v[1], W);
  writable(out);
  gemm_run(p, "gemm_tokens");
  return new_ref(v[3]);
}

// ------------------------------------------------------------------------------------------------ quantisers and LayerNorm
// x, out, bias, flags
PyObject* quant_rows(PyObject* const* v) {
  const at::Tensor& x = cuda_tensor(v[0], "x");
  const Operand out = act(v[1], "out");
  if (x.dim() != 2 || x.stride(1) != 1 || x.size(0) != out.rows || x.size(1) != out.K) {
    if (x.dim() == 2)
      fail("quant_rows: x must be [M=%lld, K=%lld] with a contiguous last dim, got (%lld, %lld)", (long long)out.rows, (long long)out.K, (long long)x.size(0), (long long)x.size(1));
    fail("quant_rows: x must be [M=%lld, K=%lld] with a contiguous last dim, got %lld dimensions", (long long)out.rows, (long long)out.K, (long long)x.dim());
  }
  const int dt = dtype_code(x.scalar_type());
  if (dt < 0) fail("quant_rows: unsupported dtype %s", c10::toString(x.scalar_type()));
  writable(out);
  launch("quant_rows", kf_quant_rows, out.fmt, dt, x.data_ptr(), x.stride(0), (int)out.rows, (int)out.K, static_cast<const float*>(out.pts),
         static_cast<const float*>(opt_ptr(v[2], "bias")), (int)to_int(v[3]), out.pq, out.psf, stream());
  return new_ref(v[1]);
}

// x, w, b, eps, out, flags, y_dbg
PyObject* ln_quant(PyObject* const* v) {
  const at::Tensor& x = cuda_tensor(v[0], "x");
  const Operand out = act(v[4], "out");
  const int64_t d = x.dim() > 0 ? x.size(-1) : 0, M = d > 0 ? x.numel() / d : 0;
  const bool bf16 = x.scalar_type() == at::kBFloat16;
  if ((x.scalar_type() != at::kFloat && !bf16) || !x.is_contiguous() || M != out.rows || d != out.K)
    fail("ln_quant: x must be contiguous fp32 or bf16 [M=%lld, d=%lld], got [%lld, %lld] %s", (long long)out.rows, (long long)out.K, (long long)M, (long long)d,
         c10::toString(x.scalar_type()));
  writable(out);
  launch("ln_quant", kf_ln_quant, out.fmt, static_cast<const float*>(x.data_ptr()), static_cast<const float*>(opt_ptr(v[1], "w")), static_cast<const float*>(opt_ptr(v[2], "b")),
         (float)to_float(v[3]), (int)M, (int)d, static_cast<const float*>(out.pts), (int)to_int(v[5]) | (bf16 ? KF_Q_IN_BF16 : 0), out.pq, out.psf,
         static_cast<float*>(opt_ptr(v[6], "y_dbg")), stream());
  return new_ref(v[4]);
}

// ts [1] fp32 and ws (two 32-bit words, zero before the first use)
float* scale_target(PyObject* ts, PyObject* ws, void** words) {
  const at::Tensor &t = cuda_tensor(ts, "ts"), &w = cuda_tensor(ws, "ws");
  need(t.scalar_type() == at::kFloat && t.numel() == 1 && w.scalar_type() == at::kInt && w.numel() >= 2 && w.is_contiguous(),
       "amax_scale: ts must be fp32 [1] and ws contiguous int32 [2]");
  *words = w.data_ptr();
  return t.data_ptr<float>();
}

// x, flags, factor, ts, ws
PyObject* amax_scale(PyObject* const* v) {
  const at::Tensor& x = cuda_tensor(v[0], "x");
  const int dt = dtype_code(x.scalar_type());
  need(x.dim() == 2 && x.stride(1) == 1 && dt >= 0, "amax_scale: x must be f32 | bf16 | f16 [M, K] with a contiguous last dim");
  void* ws;
  float* ts = scale_target(v[3], v[4], &ws);
  launch("amax_scale", kf_amax_scale, dt, x.data_ptr(), x.stride(0), (int)x.size(0), (int)x.size(1), (int)to_int(v[1]), (float)to_float(v[2]), ts, ws, stream());
  return new_ref(v[3]);
}

// x, w, b, eps, factor, ts, ws
PyObject* ln_amax_scale(PyObject* const* v) {
  const at::Tensor& x = cuda_tensor(v[0], "x");
  need(x.is_contiguous() && x.dim() > 0 && (x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16), "ln_amax_scale: x must be contiguous fp32 or bf16");
  const int64_t d = x.size(-1), M = rows_of(x, d, "ln_amax_scale: x has a last dimension of 0");
  void* ws;
  float* ts = scale_target(v[5], v[6], &ws);
  launch("ln_amax_scale", kf_ln_amax_scale, dtype_code(x.scalar_type()), x.data_ptr(), static_cast<const float*>(opt_ptr(v[1], "w")), static_cast<const float*>(opt_ptr(v[2], "b")),
         (float)to_float(v[3]), (int)M, (int)d, (float)to_float(v[4]), ts, ws, stream());
  return new_ref(v[5]);
}

// x, w, b, eps, dtype code
PyObject* ln_rows(PyObject* const* v) {
  const at::Tensor& x = cuda_tensor(v[0], "x");
  need(x.scalar_type() == at::kFloat && x.is_contiguous() && x.dim() > 0, "ln_rows: x must be contiguous fp32");
  const int64_t d = x.size(-1), M = rows_of(x, d, "ln_rows: x has a last dimension of 0");
  const int dt = (int)to_int(v[4]);
  at::Tensor y = empty(x.sizes(), dtype_of(dt), x.device());
  launch("ln_rows", kf_ln_rows, x.data_ptr<float>(), static_cast<const float*>(opt_ptr(v[1], "w")), static_cast<const float*>(opt_ptr(v[2], "b")), (float)to_float(v[3]), (int)M, (int)d, dt,
         y.data_ptr(), stream());
  return THPVariable_Wrap(std::move(y));
}

// src, dst, row offset
PyObject* broadcast_rows(PyObject* const* v) {
  const at::Tensor &src = cuda_tensor(v[0], "src"), &dst = cuda_tensor(v[1], "dst");
  need(src.scalar_type() == at::kFloat && dst.scalar_type() == at::kFloat && src.is_contiguous() && dst.is_contiguous() && dst.dim() == 3 && src.dim() > 0 &&
           src.size(-1) == dst.size(2),
       "broadcast_rows: src [R, d] and dst [B, Ntok, d] must be contiguous fp32");
  const int64_t d = dst.size(2), R = rows_of(src, d, "broadcast_rows: src and dst have a last dimension of 0");
  launch("broadcast_rows", kf_broadcast_rows, src.data_ptr<float>(), dst.data_ptr<float>(), (int)R, (int)d, (int)dst.size(0), dst.size(1) * d, to_int(v[2]), stream());
  return new_ref(v[1]);
}

// x, w, b, eps, Q, npre, wcls | None, bcls | None
PyObject* ln_tail(PyObject* const* v) {
  const at::Tensor& x = cuda_tensor(v[0], "x");
  need(x.scalar_type() == at::kFloat && x.is_contiguous() && x.dim() == 3, "ln_tail: x must be contiguous fp32");
  const int64_t B = x.size(0), Ntok = x.size(1), d = x.size(2), Q = to_int(v[4]), npre = to_int(v[5]);
  at::Tensor qb = empty({B * Q, d}, at::kBFloat16, x.device()), xb = empty({B * (Ntok - Q - npre), d}, at::kBFloat16, x.device()), cl;
  int ncls1 = 0;
  const void* wcls = nullptr;
  const float* bcls = nullptr;
  if (v[6] != Py_None) {
    const at::Tensor& wc = cuda_tensor(v[6], "wcls");
    const char* msg = "ln_tail: wcls must be contiguous bf16 [ncls1, d] and bcls fp32 [ncls1]";
    need(wc.scalar_type() == at::kBFloat16 && wc.is_contiguous() && wc.dim() == 2 && wc.size(1) == d && v[7] != Py_None, msg);
    const at::Tensor& bc = cuda_tensor(v[7], "bcls");
    need(bc.scalar_type() == at::kFloat && bc.numel() == wc.size(0), msg);
    ncls1 = (int)wc.size(0);
    wcls = wc.data_ptr();
    bcls = bc.data_ptr<float>();
    cl = empty({B * Q, wc.size(0)}, at::kBFloat16, x.device());
  }
  launch("ln_tail", kf_ln_tail, x.data_ptr<float>(), static_cast<const float*>(opt_ptr(v[1], "w")), static_cast<const float*>(opt_ptr(v[2], "b")), (float)to_float(v[3]), (int)B, (int)Ntok,
         (int)Q, (int)npre, (int)d, qb.data_ptr(), xb.data_ptr(), wcls, bcls, ncls1, ncls1 ? cl.data_ptr() : nullptr, stream());
  if (!ncls1) return pair(std::move(qb), std::move(xb));
  PyObject* t = PyTuple_New(3);
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(qb)));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(xb)));
  PyTuple_SET_ITEM(t, 2, THPVariable_Wrap(std::move(cl)));
  return t;
}

// ------------------------------------------------------------------------------------------------ attention
const at::Tensor& qkv_tensor(PyObject* o, const char* msg) {
  const at::Tensor& t = cuda_tensor(o, "qkv");
  need(t.dim() == 5 && t.size(0) == 3 && t.size(4) == 64 && t.is_contiguous() && (t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf), msg);
  return t;
}

// qkv, pre, out | None
PyObject* attn_fwd(PyObject* const* v) {
  const at::Tensor& qkv = qkv_tensor(v[0], "attn_fwd: qkv must be contiguous [3, B, N, H, 64] bf16 or f16");
  const int64_t B = qkv.size(1), N = qkv.size(2), H = qkv.size(3);
  at::Tensor out = v[2] == Py_None ? empty({B, N, H * 64}, qkv.scalar_type(), qkv.device()) : cuda_tensor(v[2], "out");
  if (v[2] != Py_None) writable(out);
  launch("attn_fwd", kf_attn_fwd, dtype_code(qkv.scalar_type()), qkv.data_ptr(), out.data_ptr(), (int)B, (int)N, (int)H, (float)to_float(v[1]), stream());
  return v[2] == Py_None ? THPVariable_Wrap(std::move(out)) : new_ref(v[2]);
}

// qkv, out (ActBuf), pre, flags
PyObject* attn_fwd_quant(PyObject* const* v) {
  const at::Tensor& qkv = qkv_tensor(v[0], "attn_fwd_quant: qkv must be contiguous [3, B, N, H, 64] bf16 or f16");
  const Operand out = act(v[1], "out");
  const int64_t B = qkv.size(1), N = qkv.size(2), H = qkv.size(3);
  if (out.rows != B * N || out.K != H * 64)
    fail("attn_fwd_quant: out must be [%lld, %lld], got [%lld, %lld]", (long long)(B * N), (long long)(H * 64), (long long)out.rows, (long long)out.K);
  writable(out);
  launch("attn_fwd_quant", kf_attn_fwd_quant, dtype_code(qkv.scalar_type()), qkv.data_ptr(), (int)B, (int)N, (int)H, (float)to_float(v[2]), out.fmt, out.pq, out.psf,
         static_cast<const float*>(out.pts), (int)to_int(v[3]), stream());
  return new_ref(v[1]);
}

// ------------------------------------------------------------------------------------------------ patch embed / head / pre / post
// x [B, 3, S, S] bf16
PyObject* im2col_patch16(PyObject* const* v) {
  const at::Tensor& x = cuda_tensor(v[0], "x");
  need(x.scalar_type() == at::kBFloat16 && x.dim() == 4 && x.size(1) == 3 && x.size(2) == x.size(3) && x.is_contiguous(),
       "im2col_patch16: x must be contiguous bf16 [B, 3, S, S]");
  const int64_t B = x.size(0), S = x.size(2), g = S / 16;
  at::Tensor out = empty({B * g * g, 768}, at::kBFloat16, x.device());
  launch("im2col_patch16", kf_im2col_patch16, x.data_ptr(), out.data_ptr(), (int)B, (int)S, stream());
  return THPVariable_Wrap(std::move(out));
}

// g, bias | None, dww, lnw, lnb, B, Hs, Ws, eps, pre_act
PyObject* dw_ln(PyObject* const* v) {
  const at::Tensor &g = cuda_tensor(v[0], "g"), &dww = cuda_tensor(v[2], "dww");
  const int64_t C = g.dim() == 2 ? g.size(1) / 4 : 0, B = to_int(v[5]), Hs = to_int(v[6]), Ws = to_int(v[7]);
  const bool pre = truth(v[9]);
  need(g.scalar_type() == at::kBFloat16 && g.is_contiguous() && g.dim() == 2 && g.size(0) == B * Hs * Ws && dww.dim() == 2 && dww.size(0) == 9 && dww.size(1) == C &&
           (v[1] != Py_None || pre),
       "dw_ln: g must be contiguous bf16 [B*Hs*Ws, 4C] and dww fp32 [9, C]");
  at::Tensor out = empty({B, 2 * Hs, 2 * Ws, C}, at::kBFloat16, g.device());
  launch("dw_ln", kf_dw_ln, g.data_ptr(), static_cast<const float*>(opt_ptr(v[1], "bias")), dww.data_ptr<float>(), static_cast<const float*>(opt_ptr(v[3], "lnw")),
         static_cast<const float*>(opt_ptr(v[4], "lnb")), out.data_ptr(), (int)B, (int)Hs, (int)Ws, (int)C, (float)to_float(v[8]), pre ? 1 : 0, stream());
  return THPVariable_Wrap(std::move(out));
}

// mask_logits, class_logits, want_scores
PyObject* semantic(PyObject* const* v) {
  const at::Tensor &ml = cuda_tensor(v[0], "mask_logits"), &cl = cuda_tensor(v[1], "class_logits");
  need(ml.scalar_type() == at::kBFloat16 && cl.scalar_type() == at::kBFloat16 && ml.is_contiguous() && cl.is_contiguous() && ml.dim() == 4 && cl.dim() > 0,
       "semantic: logits must be contiguous bf16");
  const int64_t B = ml.size(0), Q = ml.size(1), h = ml.size(2), w = ml.size(3), ncls1 = cl.size(-1);
  const bool want = truth(v[2]);
  at::Tensor labels = empty({B, h, w}, at::kByte, ml.device()), scores;
  if (want) scores = empty({B, ncls1, h, w}, at::kFloat, ml.device());
  launch("semantic", kf_semantic, ml.data_ptr(), cl.data_ptr(), (int)B, (int)Q, (int)ncls1 - 1, (int)(h * w), want ? scores.data_ptr<float>() : nullptr, labels.data_ptr<uint8_t>(), stream());
  if (want) return pair(std::move(labels), std::move(scores));
  PyObject* t = PyTuple_New(2);
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(labels)));
  PyTuple_SET_ITEM(t, 1, new_ref(Py_None));
  return t;
}

// ------------------------------------------------------------------------------------------------ operators for training
// These run on the device their first tensor lives on, on torch's current stream of that device; the others have to live there too.
void same_device(const at::Tensor& a, const at::Tensor& b, const char* op, const char* what) {
  if (a.device() != b.device()) fail("%s: %s lives on another device than the first operand", op, what);
}

// x as rows of its last dimension: the stride between them.  A 2-D tensor may have any (0 repeats one row), others are contiguous.
int64_t row_stride(const at::Tensor& x, const char* op, const char* what) {
  const int64_t d = x.size(-1);
  if (x.dim() == 2) {
    if (d > 1 && x.stride(1) != 1) fail("%s: %s must have a contiguous last dimension", op, what);
    return x.stride(0);
  }
  if (!x.is_contiguous()) fail("%s: %s must be contiguous (or two-dimensional with a contiguous last dimension)", op, what);
  return d;
}

const at::Tensor& affine(PyObject* o, const at::Tensor& x, int64_t d, const char* op, const char* what) {
  const at::Tensor& t = cuda_tensor(o, what);
  if (t.scalar_type() != at::kFloat || !t.is_contiguous() || t.numel() != d) fail("%s: %s must be contiguous fp32 with %lld elements", op, what, (long long)d);
  same_device(x, t, op, what);
  return t;
}

// rows and width of x as the kernels take them
void norm_shape(const at::Tensor& x, const char* op, int64_t* rows, int64_t* d) {
  if (x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > 8192) fail("%s: x must be [..., d] with d from 1 to 8192", op);
  if (dtype_code(x.scalar_type()) < 0) fail("%s: unsupported dtype %s", op, c10::toString(x.scalar_type()));
  *d = x.size(-1);
  *rows = x.numel() / *d;
  if (*rows > INT32_MAX) fail("%s: %lld rows are more than a call takes", op, (long long)*rows);
}

PyObject* tuple3(at::Tensor a, at::Tensor b, PyObject* c) {
  PyObject* t = PyTuple_New(3);
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(a)));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(b)));
  PyTuple_SET_ITEM(t, 2, c);
  return t;
}

// x, w, b | None, eps, out dtype code (-1: that of x)
PyObject* layer_norm_fwd(PyObject* const* v) {
  const char* const op = "layer_norm_fwd";
  const at::Tensor& x = cuda_tensor(v[0], "x");
  int64_t rows, d;
  norm_shape(x, op, &rows, &d);
  const int64_t ldx = row_stride(x, op, "x");
  const float* w = affine(v[1], x, d, op, "w").data_ptr<float>();
  const float* b = v[2] == Py_None ? nullptr : affine(v[2], x, d, op, "b").data_ptr<float>();
  const float eps = (float)to_float(v[3]);
  const int in = dtype_code(x.scalar_type()), asked = (int)to_int(v[4]), out = asked < 0 ? in : asked;
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor y = empty(x.sizes(), dtype_of(out), x.device()), stats = empty({2 * rows}, at::kFloat, x.device());
  float* const mean = stats.data_ptr<float>();
  launch(op, kf_layer_norm_fwd, in, (const void*)x.data_ptr(), ldx, w, b, eps, (int)rows, (int)d, out, y.data_ptr(), mean, mean + rows, stream());
  return tuple3(std::move(y), piece(stats, 0, rows), THPVariable_Wrap(piece(stats, rows, rows)));
}

// dy, x, w, mean, rstd, dres | None, want db, want dw
PyObject* layer_norm_bwd(PyObject* const* v) {
  const char* const op = "layer_norm_bwd";
  const at::Tensor &dy = cuda_tensor(v[0], "dy"), &x = cuda_tensor(v[1], "x");
  int64_t rows, d;
  norm_shape(x, op, &rows, &d);
  need(dy.sizes() == x.sizes() && dtype_code(dy.scalar_type()) >= 0, "layer_norm_bwd: dy must be f32, bf16 or f16 of the shape of x");
  same_device(x, dy, op, "dy");
  const int64_t ldx = row_stride(x, op, "x"), lddy = row_stride(dy, op, "dy");
  const float* w = affine(v[2], x, d, op, "w").data_ptr<float>();
  const float *mean = affine(v[3], x, rows, op, "mean").data_ptr<float>(), *rstd = affine(v[4], x, rows, op, "rstd").data_ptr<float>();
  const void* dres = nullptr;
  int64_t ldres = 0;
  if (v[5] != Py_None) {
    const at::Tensor& r = cuda_tensor(v[5], "dres");
    need(r.sizes() == x.sizes() && r.scalar_type() == x.scalar_type(), "layer_norm_bwd: dres must have the shape and type of x");
    same_device(x, r, op, "dres");
    ldres = row_stride(r, op, "dres");
    dres = r.data_ptr();
  }
  const bool want_dw = truth(v[7]), want_db = want_dw && truth(v[6]);
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t bytes = want_dw ? kf_layer_norm_ws_bytes(rows, (int)d) : 0;
  if (bytes < 0) check((int)bytes, "kf_layer_norm_ws_bytes");
  at::Tensor dx = empty(x.sizes(), x.scalar_type(), x.device()), dw, db, ws;
  if (want_dw) {
    dw = empty({d}, at::kFloat, x.device());
    ws = empty({bytes / 4}, at::kFloat, x.device());
  }
  if (want_db) db = empty({d}, at::kFloat, x.device());
  launch(op, kf_layer_norm_bwd, dtype_code(x.scalar_type()), (const void*)x.data_ptr(), ldx, dtype_code(dy.scalar_type()), (const void*)dy.data_ptr(), lddy, w, mean, rstd, dres, ldres,
         (int)rows, (int)d, dx.data_ptr(), want_dw ? dw.data_ptr<float>() : nullptr, want_db ? db.data_ptr<float>() : nullptr, want_dw ? ws.data_ptr() : nullptr, bytes, stream());
  if (!want_dw) {
    PyObject* t = PyTuple_New(3);
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(dx)));
    for (int i = 1; i < 3; ++i) PyTuple_SET_ITEM(t, i, new_ref(Py_None));
    return t;
  }
  return tuple3(std::move(dx), std::move(dw), want_db ? THPVariable_Wrap(std::move(db)) : new_ref(Py_None));
}

// [T, H, D] or [G, T, H, D], channels contiguous
struct Heads {
  int64_t g, t, h, d, sg, st, sh;
};
Heads heads_of(const at::Tensor& x, const char* op, const char* what) {
  if ((x.dim() != 3 && x.dim() != 4) || (x.size(-1) > 1 && x.stride(-1) != 1)) fail("%s: %s must be [T, H, D] or [G, T, H, D] with contiguous channels", op, what);
  const int o = (int)x.dim() - 3;
  return {o ? x.size(0) : 1, x.size(o), x.size(o + 1), x.size(o + 2), o ? x.stride(0) : 0, x.stride(o), x.stride(o + 1)};
}

// The bytes of a tensor of up to four dimensions: blocks of `len` (its last dimension where that is contiguous) at steps of the others.
struct Blocks {
  int64_t at, len, end;
  int n = 0;
  int64_t count[4], step[4];
  explicit Blocks(const at::Tensor& t) {
    const int64_t size = (int64_t)t.element_size(), dim = t.dim(), row = dim && (t.stride(-1) == 1 || t.size(-1) == 1);
    at = (int64_t)reinterpret_cast<uintptr_t>(t.data_ptr());
    len = t.numel() ? (row ? t.size(-1) : 1) * size : 0;
    end = at + len;
    for (int64_t i = 0; t.numel() && i < dim - row; ++i)
      if (t.size(i) > 1) {
        count[n] = t.size(i);
        step[n++] = t.stride(i) * size;
        end += (t.size(i) - 1) * t.stride(i) * size;
      }
  }
  bool operator==(const Blocks& o) const {
    return at == o.at && len == o.len && n == o.n && std::equal(count, count + n, o.count) && std::equal(step, step + n, o.step);
  }
};

// Whether two tensors share a byte; of a tensor with itself: whether two of its places do.  Looks for steps that bring a block of one to a block of
// the other, the longest first, each bounded by what the shorter ones can still make up: few to look at where dimensions lie inside one another, as
// parts of a projection do.  Where there are more than it looks at, the tensors count as overlapping.
class Overlap {
 public:
  static bool of(const Blocks& a, const Blocks& b) { return a.len && b.len && a.at < b.end && b.at < a.end && Overlap(a, b, false).found_; }
  static bool inside(const Blocks& a) { return a.len && Overlap(a, a, true).found_; }

 private:
  struct Dim {
    int64_t step, lo, hi;
  };
  Overlap(const Blocks& a, const Blocks& b, bool self) : low_(-b.len), high_(a.len), self_(self) {
    for (int i = 0; i < a.n; ++i) add(a.step[i], -(a.count[i] - 1), 0);
    for (int i = 0; i < b.n; ++i) add(b.step[i], 0, b.count[i] - 1);
    for (int i = 1; self && i < a.n; ++i) found_ |= std::find(a.step, a.step + i, a.step[i]) != a.step + i;      // (1, 0) and (0, 1) are one place
    if (found_) return;
    std::sort(dims_, dims_ + n_, [](const Dim& x, const Dim& y) { return x.step > y.step; });
    found_ = reaches(0, b.at - a.at, false);
  }
  void add(int64_t step, int64_t lo, int64_t hi) {
    if (step == 0) {                                               // the same place again
      found_ |= self_;
      return;
    }
    for (int i = 0; i < n_; ++i)
      if (dims_[i].step == step) {
        dims_[i].lo += lo;
        dims_[i].hi += hi;
        return;
      }
    dims_[n_++] = {step, lo, hi};
  }
  bool reaches(int i, int64_t apart, bool moved) {
    if (i == n_) return low_ < apart && apart < high_ && (moved || !self_);
    int64_t least = 0, most = 0;
    for (int k = i + 1; k < n_; ++k) {
      least += dims_[k].lo * dims_[k].step;
      most += dims_[k].hi * dims_[k].step;
    }
    const Dim& d = dims_[i];
    const auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
    const int64_t first = std::max(d.lo, floor_div(low_ - most - apart, d.step) + 1), last = std::min(d.hi, -floor_div(apart + least - high_, d.step) - 1);
    for (int64_t x = first; x <= last; ++x) {
      if (--budget_ < 0 || reaches(i + 1, apart + x * d.step, moved || x != 0)) return true;
    }
    return false;
  }
  Dim dims_[8];
  int n_ = 0, budget_ = 4096;
  int64_t low_, high_;
  bool self_, found_ = false;
};

// `out` is about to be written by an operator that reads (or writes) `other` as well
void apart(const at::Tensor& out, const at::Tensor& other, const char* op, const char* what, const char* from) {
  if (Overlap::of(Blocks(out), Blocks(other))) fail("%s: %s overlaps %s", op, what, from);
}

// x, pos, freq (fp64 [P]), axis (int32 [P]), axes, head channels, interleaved, inverse, out | None
PyObject* rope_axes(PyObject* const* v) {
  const char* const op = "rope_axes";
  const at::Tensor &x = cuda_tensor(v[0], "x"), &pos = cuda_tensor(v[1], "pos"), &freq = cuda_tensor(v[2], "freq"), &axis = cuda_tensor(v[3], "axis");
  const Heads s = heads_of(x, op, "x");
  const int64_t axes = to_int(v[4]), D = to_int(v[5]);
  if (dtype_code(x.scalar_type()) < 0) fail("%s: unsupported dtype %s", op, c10::toString(x.scalar_type()));
  if (s.d != D) fail("%s: the table is for %lld channels per head, x has %lld", op, (long long)D, (long long)s.d);
  if (pos.dim() != 2 || pos.size(0) != s.t || pos.size(1) != axes)
    fail("%s: pos must be [T=%lld, axes=%lld]", op, (long long)s.t, (long long)axes);
  const at::ScalarType pt = pos.scalar_type();
  need(pt == at::kInt || pt == at::kLong || pt == at::kFloat, "rope_axes: pos must be int32, int64 or fp32");
  if (s.g > INT32_MAX || s.t > INT32_MAX || s.h > INT32_MAX) fail("%s: shape does not fit 32-bit sizes", op);
  for (int i = 0; i < 3; ++i)
    if (x.device() != (i == 0 ? pos : i == 1 ? freq : axis).device()) fail("%s: pos and the table must live on the device of x", op);
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor out;
  if (v[8] == Py_None) {
    out = empty(x.sizes(), x.scalar_type(), x.device());
  } else {
    out = cuda_tensor(v[8], "out");
    need(out.sizes() == x.sizes() && out.scalar_type() == x.scalar_type(), "rope_axes: out must have the shape and type of x");
    same_device(x, out, op, "out");
  }
  const Heads o = heads_of(out, op, "out");
  if (v[8] != Py_None) {
    need((o.sg != 0 || o.g < 2) && (o.st != 0 || o.t < 2) && (o.sh != 0 || o.h < 2), "rope_axes: out must not be an expanded tensor");
    const Blocks to(out);
    need(!Overlap::inside(to), "rope_axes: out overlaps itself");
    need(Blocks(x) == to || !Overlap::of(to, Blocks(x)), "rope_axes: out must be x or not overlap it");
    apart(out, pos, op, "out", "pos");
    writable(out);
  }
  kf_rope_params p = {};
  p.x = x.data_ptr();
  p.y = out.data_ptr();
  p.pos = pos.data_ptr();
  p.freq = freq.data_ptr<double>();
  p.axis = axis.data_ptr<int>();
  p.xs_g = s.sg; p.xs_t = s.st; p.xs_h = s.sh; p.ys_g = o.sg; p.ys_t = o.st; p.ys_h = o.sh; p.ps_t = pos.stride(0); p.ps_a = pos.stride(1);
  p.dtype = dtype_code(x.scalar_type());
  p.pos_kind = pt == at::kInt ? KF_POS_I32 : pt == at::kLong ? KF_POS_I64 : KF_POS_F32;
  p.G = (int)s.g; p.T = (int)s.t; p.H = (int)s.h; p.D = (int)s.d; p.P = (int)freq.numel();
  p.interleaved = truth(v[6]);
  p.inverse = truth(v[7]);
  launch(op, kf_rope_axes, (const kf_rope_params*)&p, stream());
  return v[8] == Py_None ? THPVariable_Wrap(std::move(out)) : new_ref(v[8]);
}

// An operand [rows, heads, 64] of the packed attention.
kf_heads pack_heads(const at::Tensor& t) { return {t.data_ptr(), t.stride(0), t.stride(1)}; }
const at::Tensor& pack_tensor(PyObject* o, const at::Tensor* first, const char* op, const char* what) {
  const at::Tensor& t = cuda_tensor(o, what);
  if (t.dim() != 3 || t.size(2) != 64 || t.stride(2) != 1) fail("%s: %s must be [rows, heads, 64] with contiguous channels", op, what);
  if (first) {
    if (t.scalar_type() != first->scalar_type()) fail("%s: %s must have the type of q", op, what);
    same_device(*first, t, op, what);
  } else if (t.scalar_type() != at::kBFloat16 && t.scalar_type() != at::kHalf) {
    fail("%s: %s must be bf16 or f16", op, what);
  }
  return t;
}
void same_shape(const at::Tensor& a, const at::Tensor& b, const char* op, const char* what) {
  if (a.sizes() != b.sizes()) fail("%s: %s has another shape than the operand it belongs to", op, what);
}
void same_place(const at::Tensor& t, const char* op, const char* what) {          // written row by row from many threads
  for (int i = 0; i < 2; ++i)
    if (t.size(i) > 1 && t.stride(i) == 0) fail("%s: %s must not be an expanded tensor", op, what);
  if (Overlap::inside(Blocks(t))) fail("%s: %s overlaps itself", op, what);
}

// What both directions share.  v: q, k, v, q_tiles, k_tiles, query rows, key rows, longest, scale, cap, slopes | None
struct Pack {
  const at::Tensor &q, &k, &v;
  kf_attn_pack_params p;
  int64_t q_rows, k_rows;
};
const at::Tensor& pack_table(PyObject* o, const at::Tensor& q, const char* op) {
  const at::Tensor& t = cuda_tensor(o, "plan");
  if (t.scalar_type() != at::kInt || t.dim() != 2 || t.size(1) != 8 || !t.is_contiguous() || t.size(0) > INT32_MAX) fail("%s: the plan's tables must be contiguous int32 [n, 8]", op);
  same_device(q, t, op, "the plan");
  return t;
}
Pack pack_operands(PyObject* const* v, const char* op) {
  const at::Tensor& q = pack_tensor(v[0], nullptr, op, "q");
  Pack c{q, pack_tensor(v[1], &q, op, "k"), pack_tensor(v[2], &q, op, "v"), {}, to_int(v[5]), to_int(v[6])};
  same_shape(c.k, c.v, op, "v");
  if (c.q_rows > q.size(0) || c.k_rows > c.k.size(0))
    fail("%s: the plan is for %lld query and %lld key rows, there are %lld and %lld", op, (long long)c.q_rows, (long long)c.k_rows, (long long)q.size(0), (long long)c.k.size(0));
  if (q.size(1) < 1 || c.k.size(1) < 1 || q.size(1) > 65536 || q.size(1) % c.k.size(1))
    fail("%s: %lld query heads do not share %lld key heads evenly", op, (long long)q.size(1), (long long)c.k.size(1));
  const at::Tensor &qt = pack_table(v[3], q, op), &kt = pack_table(v[4], q, op);
  kf_attn_pack_params& p = c.p;
  p.dtype = dtype_code(q.scalar_type());
  p.Hq = (int)q.size(1);
  p.Hk = (int)c.k.size(1);
  p.n_q_tiles = (int)qt.size(0);
  p.n_k_tiles = (int)kt.size(0);
  p.longest = (int)to_int(v[7]);
  p.scale = (float)to_float(v[8]);
  const double cap = to_float(v[9]);
  p.cap = (float)cap;
  if (cap > 0 && p.cap == 0.f) fail("%s: the cap is 0 in fp32", op);
  p.Tq = q.size(0);
  p.Tk = c.k.size(0);
  p.q_tiles = qt.data_ptr<int>();
  p.k_tiles = kt.data_ptr<int>();
  if (v[10] != Py_None) p.slopes = affine(v[10], q, q.size(1), op, "slopes").data_ptr<float>();
  p.q = pack_heads(q);
  p.k = pack_heads(c.k);
  p.v = pack_heads(c.v);
  return c;
}
// A new tensor of this shape: the first `used` rows are written by the call, the others are zero.
at::Tensor pack_new(const at::Tensor& like, int64_t used) {
  at::Tensor t = empty(like.sizes(), like.scalar_type(), like.device());
  if (used < t.size(0)) {
    const Unlocked unlocked;
    t.narrow(0, used, t.size(0) - used).zero_();
  }
  return t;
}

// The lengths of a plan: any sequence of integers.
std::vector<int64_t> lengths(PyObject* o, const char* what) {
  PyObject* seq = PySequence_Fast(o, what);
  if (!seq) throw Failed{};
  std::vector<int64_t> v((size_t)PySequence_Fast_GET_SIZE(seq));
  for (size_t i = 0; i < v.size(); ++i) {
    PyObject* n = PyNumber_Index(PySequence_Fast_GET_ITEM(seq, (Py_ssize_t)i));
    v[i] = n ? PyLong_AsLongLong(n) : -1;
    Py_XDECREF(n);
    if (!n || (v[i] == -1 && PyErr_Occurred())) {
      Py_DECREF(seq);
      throw Failed{};
    }
  }
  Py_DECREF(seq);
  return v;
}

// q lengths, k lengths | None, causal, prefixes | None -> (table int32 [query tiles + key tiles, 8] on the CPU, query tiles, query rows, key rows, the most keys a query tile sees, the queries that see
// a key tile: of all, the most of one):
// the records of kf_attn_pack_params, of queries and then of keys, each with the longest work first
PyObject* attn_plan(PyObject* const* v) {
  constexpr int64_t T = 128, MOST = INT32_MAX - 256;
  const std::vector<int64_t> lq = lengths(v[0], "AttnPlan: q_lens must be a sequence of integers"),
                             lk = v[1] == Py_None ? lq : lengths(v[1], "AttnPlan: k_lens must be a sequence of integers");
  const bool causal = truth(v[2]);
  if (lq.size() != lk.size()) fail("AttnPlan: %zd sequences of queries, %zd of keys", (Py_ssize_t)lq.size(), (Py_ssize_t)lk.size());
  if (v[3] != Py_None && !causal) fail("AttnPlan: a prefix goes with causal=True (without it every key is seen)");
  const std::vector<int64_t> pre = v[3] == Py_None ? std::vector<int64_t>(lk.size(), 0) : lengths(v[3], "AttnPlan: prefix must be a sequence of integers");
  if (pre.size() != lk.size()) fail("AttnPlan: %zd sequences, %zd prefixes", (Py_ssize_t)lk.size(), (Py_ssize_t)pre.size());
  int64_t rows_q = 0, rows_k = 0, nq = 0, nk = 0;
  for (size_t d = 0; d < lq.size(); ++d) {
    if (lq[d] < 0 || lk[d] < 0 || pre[d] < 0 || pre[d] > lk[d]) fail("AttnPlan: lengths must not be negative, a prefix not longer than its sequence of keys");
    if (lq[d] >= MOST || lk[d] >= MOST || (rows_q += lq[d]) >= MOST || (rows_k += lk[d]) >= MOST) fail("AttnPlan: more rows than a call takes");
    nq += (lq[d] + T - 1) / T;
    nk += (lk[d] + T - 1) / T;
  }
  struct Tile {
    int64_t work;
    int32_t w[8];
  };
  std::vector<Tile> q, k;
  q.reserve((size_t)nq);
  k.reserve((size_t)nk);
  int64_t q0 = 0, k0 = 0;
  for (size_t d = 0; d < lq.size(); ++d) {
    const int64_t p = causal ? pre[d] : lk[d], off = lk[d] - lq[d], slot0 = (int64_t)q.size();
    for (int64_t i = 0; i < lq[d]; i += T) {
      const int64_t rows = std::min(T, lq[d] - i), seen = std::clamp(std::max(i + off + rows, p), (int64_t)0, lk[d]);
      q.push_back({seen, {(int32_t)(q0 + i), (int32_t)rows, (int32_t)k0, (int32_t)lk[d], (int32_t)(i + off), (int32_t)p, (int32_t)q.size(), 0}});
    }
    for (int64_t i = 0; i < lk[d]; i += T) {
      const int64_t low = i < p ? 0 : std::max(i - off, (int64_t)0);
      k.push_back({lq[d] - low, {(int32_t)(k0 + i), (int32_t)std::min(T, lk[d] - i), (int32_t)q0, (int32_t)lq[d], (int32_t)i, (int32_t)off, (int32_t)p, (int32_t)slot0}});
    }
    q0 += lq[d];
    k0 += lk[d];
  }
  const auto longer = [](const Tile& a, const Tile& b) { return a.work > b.work; };
  std::stable_sort(q.begin(), q.end(), longer);
  std::stable_sort(k.begin(), k.end(), longer);
  at::Tensor table = at::empty({nq + nk, 8}, at::TensorOptions().dtype(at::kInt));
  int32_t* to = table.data_ptr<int32_t>();
  for (const std::vector<Tile>* tiles : {&q, &k})
    for (const Tile& t : *tiles) to = std::copy(t.w, t.w + 8, to);
  int64_t k_work = 0;
  for (const Tile& t : k) k_work += std::max(t.work, (int64_t)0);
  PyObject* r = PyTuple_New(7);
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(table)));
  PyTuple_SET_ITEM(r, 1, PyLong_FromLongLong(nq));
  PyTuple_SET_ITEM(r, 2, PyLong_FromLongLong(rows_q));
  PyTuple_SET_ITEM(r, 3, PyLong_FromLongLong(rows_k));
  PyTuple_SET_ITEM(r, 4, PyLong_FromLongLong(q.empty() ? 0 : q[0].work));
  PyTuple_SET_ITEM(r, 5, PyLong_FromLongLong(k_work));
  PyTuple_SET_ITEM(r, 6, PyLong_FromLongLong(k.empty() ? 0 : std::max(k[0].work, (int64_t)0)));
  return r;
}

// ..., out | None
PyObject* attn_packed(PyObject* const* v) {
  const char* const op = "attn_packed";
  Pack c = pack_operands(v, op);
  const c10::cuda::CUDAGuard guard(c.q.device());
  at::Tensor out;
  if (v[11] == Py_None) {
    out = pack_new(c.q, c.q_rows);
  } else {
    out = pack_tensor(v[11], &c.q, op, "out");
    same_shape(c.q, out, op, "out");
    same_place(out, op, "out");
    apart(out, c.q, op, "out", "q");
    apart(out, c.k, op, "out", "k");
    apart(out, c.v, op, "out", "v");
    writable(out);
  }
  at::Tensor lse = empty({c.q.size(1), c.q.size(0)}, at::kFloat, c.q.device());
  if (c.q_rows < c.q.size(0)) {
    const Unlocked unlocked;
    lse.narrow(1, c.q_rows, c.q.size(0) - c.q_rows).zero_();
  }
  c.p.o = pack_heads(out);
  c.p.lse = lse.data_ptr<float>();
  launch(op, kf_attn_pack_fwd, (const kf_attn_pack_params*)&c.p, stream());
  if (v[11] == Py_None) return pair(std::move(out), std::move(lse));
  PyObject* t = PyTuple_New(2);
  PyTuple_SET_ITEM(t, 0, new_ref(v[11]));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(lse)));
  return t;
}

// ..., dout, out, lse, dq | None, dk | None, dv | None, want dk and dv, the plan's queries that see a key tile: of all, the most of one
PyObject* attn_packed_bwd(PyObject* const* v) {
  const char* const op = "attn_packed_bwd";
  Pack c = pack_operands(v, op);
  const at::Tensor &dout = pack_tensor(v[11], &c.q, op, "dout"), &out = pack_tensor(v[12], &c.q, op, "out"), &lse = cuda_tensor(v[13], "lse");
  same_shape(c.q, dout, op, "dout");
  same_shape(c.q, out, op, "out");
  if (lse.scalar_type() != at::kFloat || !lse.is_contiguous() || lse.dim() != 2 || lse.size(0) != c.q.size(1) || lse.size(1) != c.q.size(0))
    fail("%s: lse must be contiguous fp32 [query heads, query rows]", op);
  same_device(c.q, lse, op, "lse");
  const c10::cuda::CUDAGuard guard(c.q.device());
  const bool keys = truth(v[17]);
  need(keys || (v[15] == Py_None && v[16] == Py_None), "attn_packed_bwd: keys=False makes no dk and dv");
  const at::Tensor* const of[3] = {&c.q, &c.k, &c.v};
  const char* const names[3] = {"dq", "dk", "dv"};
  at::Tensor g[3];
  for (int i = 0; i < 3; ++i) {
    if (v[14 + i] == Py_None) continue;
    g[i] = pack_tensor(v[14 + i], &c.q, op, names[i]);
    same_shape(*of[i], g[i], op, names[i]);
    same_place(g[i], op, names[i]);
    const at::Tensor* const others[] = {&c.q, &c.k, &c.v, &dout, &out, &lse};
    const char* const from[] = {"q", "k", "v", "dout", "out", "lse"};
    for (int j = 0; j < 6; ++j) apart(g[i], *others[j], op, names[i], from[j]);
    for (int j = 0; j < i; ++j)
      if (g[j].defined()) apart(g[i], g[j], op, names[i], names[j]);
  }
  for (int i = 0; i < 3; ++i) {
    if (g[i].defined()) writable(g[i]);
    else if (keys || i == 0) g[i] = pack_new(*of[i], i ? c.k_rows : c.q_rows);
  }
  c.p.dout = pack_heads(dout);
  c.p.o = pack_heads(out);
  c.p.lse = lse.data_ptr<float>();
  c.p.dq = pack_heads(g[0]);
  if (keys) {
    c.p.dk = pack_heads(g[1]);
    c.p.dv = pack_heads(g[2]);
  }
  c.p.k_work = to_int(v[18]);
  c.p.k_longest = (int)to_int(v[19]);
  c.p.ws_bytes = kf_attn_pack_bwd_ws_bytes(&c.p);
  if (c.p.ws_bytes < 0) check((int)c.p.ws_bytes, "kf_attn_pack_bwd_ws_bytes");
  at::Tensor ws = empty({c.p.ws_bytes / 4}, at::kFloat, c.q.device());
  c.p.ws = ws.data_ptr();
  launch(op, kf_attn_pack_bwd, (const kf_attn_pack_params*)&c.p, stream());
  PyObject* t = PyTuple_New(3);
  for (int i = 0; i < 3; ++i) PyTuple_SET_ITEM(t, i, v[14 + i] == Py_None && g[i].defined() ? THPVariable_Wrap(std::move(g[i])) : new_ref(v[14 + i]));
  return t;
}

// kernels that this thread has launched through the library
PyObject* launch_count(PyObject* const*) { return PyLong_FromLongLong(kf_launch_count()); }

// a weight: does the next GEMM with it read it ahead of its predecessor's end?
PyObject* reads_weight_early(PyObject* const* v) {
  const Ref q = attr(v[0], s_q), sf = attr(v[0], s_sf);
  return PyBool_FromLong(weight_settled(v[0], tensor(q, "weight"), sf == Py_None ? at::Tensor() : tensor(sf, "weight")));
}

// ------------------------------------------------------------------------------------------------ module
template <PyObject* (*F)(PyObject* const*), int ARGS>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != ARGS) {
    PyErr_Format(PyExc_TypeError, "native operator takes %d arguments, got %zd", ARGS, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Failed&) {
    return nullptr;
  } catch (const c10::OutOfMemoryError& e) {                    // as torch raises it from its own allocations
    PyObject* t = PyImport_ImportModule("torch");
    PyObject* cls = t ? PyObject_GetAttrString(t, "OutOfMemoryError") : nullptr;
    PyErr_SetString(cls ? cls : PyExc_RuntimeError, e.what_without_backtrace());
    Py_XDECREF(cls);
    Py_XDECREF(t);
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

#define KF_ENTRY(f, n) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<f, n>)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {KF_ENTRY(quant_rows, 4),     KF_ENTRY(ln_quant, 7),   KF_ENTRY(ln_rows, 5),  KF_ENTRY(gemm_plain, 6),     KF_ENTRY(gemm_res, 7),
                           KF_ENTRY(qkv_rope, 10),      KF_ENTRY(gemm_gelu_q, 6), KF_ENTRY(bmm_nt, 3),   KF_ENTRY(gemm_tokens, 8),    KF_ENTRY(broadcast_rows, 3),
                           KF_ENTRY(ln_tail, 8),        KF_ENTRY(attn_fwd, 3),   KF_ENTRY(attn_fwd_quant, 4), KF_ENTRY(im2col_patch16, 1), KF_ENTRY(dw_ln, 10),
                           KF_ENTRY(semantic, 3),       KF_ENTRY(amax_scale, 5), KF_ENTRY(ln_amax_scale, 7),
                           KF_ENTRY(layer_norm_fwd, 5), KF_ENTRY(layer_norm_bwd, 8), KF_ENTRY(rope_axes, 9),
                           KF_ENTRY(attn_plan, 4),      KF_ENTRY(attn_packed, 12),   KF_ENTRY(attn_packed_bwd, 20),
                           KF_ENTRY(reads_weight_early, 1), KF_ENTRY(launch_count, 0), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_kf_host", "native operator layer over libkf_b200.so", -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kf_host() {
  PyObject* lib = PyImport_ImportModule("lightly_trian_quant_b200._lib");
  if (!lib) return nullptr;
  g_error = PyObject_GetAttrString(lib, "KfError");
  Py_DECREF(lib);
  if (!g_error) return nullptr;
  s_M = PyUnicode_InternFromString("M");
  s_N = PyUnicode_InternFromString("N");
  s_K = PyUnicode_InternFromString("K");
  s_fmt = PyUnicode_InternFromString("fmt");
  s_q = PyUnicode_InternFromString("q");
  s_sf = PyUnicode_InternFromString("sf");
  s_ts = PyUnicode_InternFromString("ts");
  s_settled = PyUnicode_InternFromString("settled");
  const char* names[4] = {"mx8", "nv4", "mx4", "bf16"};
  for (int i = 0; i < 4; ++i) g_fmt_names[i] = PyUnicode_InternFromString(names[i]);
  return PyModule_Create(&g_module);
}
