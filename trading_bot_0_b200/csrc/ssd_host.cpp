// Native host path of the Python entry points: argument checks, output allocation, geometry structs and the library call of
// ssd.py / prepost.py in one C++ function each, called with positional arguments (METH_FASTCALL).
//
// A small call is bound by this code and not by its kernels: four streams of one decode step keep the GPU busy for 3 us,
// while the same checks, struct fields and ctypes conversions written in Python took 25 us per step, 75 us per prefill and
// 200 us per fp32 training step (forward + backward under autograd).  The autograd nodes live here as well, so a backward
// pass runs without taking the interpreter lock.
//
// The module links to nothing of libssd_b200: bind() hands it the addresses of the C ABI functions of the library that
// _lib.py loaded.  Argument errors are ValueError, library errors the SsdError class handed to bind(), with the texts a
// caller of the Python functions sees.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <sstream>
#include <string>
#include <vector>

#include "../../include/ssd_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ---- the library's C ABI, bound at import ------------------------------------------------------------------------------
struct Api {
  decltype(&::ssd_workspace_bytes) workspace_bytes;
  decltype(&::ssd_forward_staged) forward_staged;
  decltype(&::ssd_backward_staged) backward_staged;
  decltype(&::ssd_state_update) state_update;
  decltype(&::ssd_state_update_host) state_update_host;
  decltype(&::ssd_last_error) last_error;
  decltype(&::ssd_conv1d_workspace_bytes) conv1d_workspace_bytes;
  decltype(&::ssd_conv1d_forward) conv1d_forward;
  decltype(&::ssd_conv1d_backward) conv1d_backward;
  decltype(&::ssd_rmsnorm_workspace_bytes) rmsnorm_workspace_bytes;
  decltype(&::ssd_rmsnorm_forward) rmsnorm_forward;
  decltype(&::ssd_rmsnorm_backward) rmsnorm_backward;
  decltype(&::ssd_selscan_workspace_bytes) selscan_workspace_bytes;
  decltype(&::ssd_selscan_forward) selscan_forward;
  decltype(&::ssd_selscan_backward) selscan_backward;
  decltype(&::ssd_selscan_step) selscan_step;
  decltype(&::ssd_conv1d_carry_workspace_bytes) conv1d_carry_workspace_bytes;
  decltype(&::ssd_conv1d_carry_forward) conv1d_carry_forward;
  decltype(&::ssd_conv1d_carry_backward) conv1d_carry_backward;
  decltype(&::ssd_conv1d_step) conv1d_step;
  decltype(&::ssd_linear_workspace_bytes) linear_workspace_bytes;
  decltype(&::ssd_linear_forward) linear_forward;
  decltype(&::ssd_linear_backward) linear_backward;
} api;
PyObject *ssd_error = nullptr, *oom_error = nullptr;   // _lib.SsdError, torch.OutOfMemoryError
constexpr int32_t kAllStages = SSD_STAGE_LOCAL | SSD_STAGE_FINISH;

// ---- errors ------------------------------------------------------------------------------------------------------------
struct ArgError : std::runtime_error { using std::runtime_error::runtime_error; };
struct LibError : std::runtime_error {
  int32_t code;
  LibError(int32_t c, const char* m) : std::runtime_error("ssd_b200 error " + std::to_string(c) + ": " + m), code(c), msg(m) {}
  std::string msg;
};
void check_rc(int32_t rc) { if (rc != SSD_OK) throw LibError(rc, api.last_error()); }

std::string str(at::ScalarType t) {
  return t == at::kBFloat16 ? "torch.bfloat16" : t == at::kFloat ? "torch.float32" : std::string("torch.") + c10::toString(t);
}
std::string str(at::IntArrayRef s) {
  std::ostringstream o;
  o << "(";
  for (size_t i = 0; i < s.size(); ++i) o << (i ? ", " : "") << s[i];
  o << (s.size() == 1 ? ",)" : ")");
  return o.str();
}
std::string str(const at::Device& d) { return d.str(); }
std::string str(const char* s) { return s; }
std::string str(const std::string& s) { return s; }
std::string str(int64_t v) { return std::to_string(v); }
template <class... A> [[noreturn]] void fail(const A&... a) { throw ArgError((str(a) + ...)); }

// Runs `f`, turning C++ exceptions into Python ones.
template <class F> PyObject* guarded(F f) {
  try {
    return f();
  } catch (const LibError& e) {
    PyObject* ex = PyObject_CallFunction(ssd_error, "is", (int)e.code, e.msg.c_str());
    if (ex) { PyErr_SetObject(ssd_error, ex); Py_DECREF(ex); }
  } catch (const ArgError& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(oom_error, e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// ---- Python arguments --------------------------------------------------------------------------------------------------
struct Args {
  PyObject* const* a;
  Py_ssize_t n;
  Args(PyObject* const* args, Py_ssize_t got, Py_ssize_t want) : a(args), n(got) {
    if (got != want) fail("expected ", (int64_t)want, " arguments, got ", (int64_t)got);
  }
  const Tensor& tensor(int i, const char* name) const {
    if (!THPVariable_Check(a[i])) fail(name, ": expected a tensor, got ", Py_TYPE(a[i])->tp_name);
    return THPVariable_Unpack(a[i]);
  }
  const Tensor* opt(int i, const char* name) const { return a[i] == Py_None ? nullptr : &tensor(i, name); }
  int64_t integer(int i) const {
    const long long v = PyLong_AsLongLong(a[i]);
    if (v == -1 && PyErr_Occurred()) throw std::runtime_error("bad integer argument");
    return v;
  }
  double real(int i) const {
    const double v = PyFloat_AsDouble(a[i]);
    if (v == -1.0 && PyErr_Occurred()) throw std::runtime_error("bad float argument");
    return v;
  }
  bool flag(int i) const { return PyObject_IsTrue(a[i]) == 1; }
};
PyObject* wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}

// ---- checks and geometry -----------------------------------------------------------------------------------------------
int32_t storage_type(const Tensor& x) {
  if (x.scalar_type() == at::kBFloat16) return SSD_BF16;
  if (x.scalar_type() != at::kFloat) fail("unsupported dtype ", x.scalar_type());
  return SSD_F32;
}
struct Shape {   // small fixed-size shape, no allocation
  int64_t v[4];
  int n;
  template <class... I> explicit Shape(I... i) : v{(int64_t)i...}, n((int)sizeof...(i)) {}
  operator at::IntArrayRef() const { return at::IntArrayRef(v, n); }
};
bool same(const Tensor& t, at::IntArrayRef s) { return t.sizes() == s; }

// The geometry structs take a stride of 0 as "dense", so rows that lie over one another cannot be described by them.
bool overlaid(const Tensor& t, int dims) {
  for (int i = 0; i < dims; ++i)
    if (t.size(i) > 1 && t.stride(i) == 0) return true;
  return false;
}
void check_seq(const char* name, const Tensor& t, const Shape& shape, at::ScalarType dtype, const at::Device& dev) {
  if (!same(t, shape)) {
    if (t.dim() != shape.n) fail(name, ": expected rank ", (int64_t)shape.n, ", got ", t.dim());
    fail(name, ": expected shape ", at::IntArrayRef(shape), ", got ", t.sizes());
  }
  if (t.scalar_type() != dtype) fail(name, ": expected dtype ", dtype, ", got ", t.scalar_type());
  if (t.device() != dev) fail(name, ": expected device ", dev, ", got ", t.device());
  if (t.stride(-1) != 1) fail(name, ": innermost stride must be 1");
  if (t.dim() == 4 && t.stride(2) != t.size(3)) fail(name, ": the last two dims must be dense");
  if (overlaid(t, 2)) fail(name, ": expanded over a dim (stride 0); make it contiguous");
}
void check_dense_f32(const char* name, const Tensor* t, const Shape& shape, const at::Device& dev) {
  if (!t) return;
  if (!same(*t, shape)) fail(name, ": expected shape ", at::IntArrayRef(shape), ", got ", t->sizes());
  if (t->scalar_type() != at::kFloat) fail(name, ": expected float32, got ", t->scalar_type());
  if (t->device() != dev || !t->is_contiguous()) fail(name, ": must be a contiguous tensor on ", dev);
}
void check_values_f32(const char* name, const Tensor* t, int64_t n, const at::Device& dev) {   // any shape
  if (t && (t->numel() != n || t->scalar_type() != at::kFloat || t->device() != dev || !t->is_contiguous()))
    fail(name, ": expected ", n, " contiguous fp32 values on ", dev, ", got ", t->sizes(), " ", t->scalar_type(), " on ", t->device());
}
Tensor empty(at::IntArrayRef shape, at::ScalarType dtype, const at::Device& dev) {
  return at::detail::empty_cuda(shape, dtype, dev, std::nullopt);
}
// A tensor of the caller's was written: autograd counts it, as of torch's own in-place calls, so that a node that saved the tensor
// refuses to go on with other values.  (Tensors of the inference mode keep no count.)
void written(const Tensor& t) { if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version(); }
void* ptr(const Tensor* t) { return t && t->defined() ? t->data_ptr() : nullptr; }
float* fptr(const Tensor* t) { return (float*)ptr(t); }
void* stream_of(const at::Device& d) { return c10::cuda::getCurrentCUDAStream(d.index()).stream(); }

// The operands of one scan, as both passes take them.
struct Scan {
  const Tensor &x, &dt, &A, &Bm, &Cm;
  const Tensor *D, *z, *init, *bias;
  int64_t chunk, algo;
  bool softplus;
};

// Validates the sequence operands and fills the geometry struct.
SsdDims seq_dims(const Tensor& x, const Tensor& dt, const Tensor& Bm, const Tensor& Cm, const Tensor* z, const Tensor* y, int64_t chunk,
                 int64_t algo, bool softplus) {
  if (!x.is_cuda()) fail("x must be a CUDA tensor (there is no CPU path)");
  if (x.dim() != 4) fail("x must be [batch, seqlen, nheads, headdim]");
  const int32_t dtype = storage_type(x);
  if (Bm.dim() != 4) fail("B must be [batch, seqlen, ngroups, dstate]");
  const int64_t B = x.size(0), L = x.size(1), H = x.size(2), P = x.size(3), G = Bm.size(2), N = Bm.size(3);
  const at::Device dev = x.device();
  const at::ScalarType st = x.scalar_type();
  check_seq("x", x, Shape(B, L, H, P), st, dev);
  check_seq("dt", dt, Shape(B, L, H), st, dev);
  check_seq("B", Bm, Shape(B, L, G, N), st, dev);
  check_seq("C", Cm, Shape(B, L, G, N), st, dev);
  if (G <= 0 || H % G) fail("nheads (", H, ") must be a multiple of ngroups (", G, ")");
  if (chunk < 1 || chunk > 256) fail("chunk must be in [1, 256], got ", chunk);
  SsdDims d;
  std::memset(&d, 0, sizeof d);
  d.batch = (int32_t)B; d.seqlen = (int32_t)L; d.nheads = (int32_t)H; d.headdim = (int32_t)P;
  d.dstate = (int32_t)N; d.ngroups = (int32_t)G; d.chunk = (int32_t)chunk;
  d.dtype = dtype; d.algo = (int32_t)algo; d.device = dev.index(); d.has_z = z ? 1 : 0; d.dt_softplus = softplus ? 1 : 0;
  d.x_stride_b = x.stride(0); d.x_stride_l = x.stride(1);
  d.dt_stride_b = dt.stride(0); d.dt_stride_l = dt.stride(1);
  d.b_stride_b = Bm.stride(0); d.b_stride_l = Bm.stride(1);
  d.c_stride_b = Cm.stride(0); d.c_stride_l = Cm.stride(1);
  if (z) {
    check_seq("z", *z, Shape(B, L, H, P), st, dev);
    d.z_stride_b = z->stride(0); d.z_stride_l = z->stride(1);
  }
  if (y) {
    check_seq("y/dy", *y, Shape(B, L, H, P), st, dev);
    d.y_stride_b = y->stride(0); d.y_stride_l = y->stride(1);
  }
  return d;
}
SsdDims make_dims(const Scan& s, const Tensor* y) {
  const SsdDims d = seq_dims(s.x, s.dt, s.Bm, s.Cm, s.z, y, s.chunk, s.algo, s.softplus);
  const at::Device dev = s.x.device();
  const int64_t H = d.nheads;
  check_dense_f32("A", &s.A, Shape(H), dev);
  check_dense_f32("D", s.D, Shape(H), dev);
  check_dense_f32("dt_bias", s.bias, Shape(H), dev);
  check_dense_f32("init_state", s.init, Shape(d.batch, H, d.headdim, d.dstate), dev);
  return d;
}
Tensor workspace_for(const SsdDims& d, const at::Device& dev, bool backward) {
  const size_t n = api.workspace_bytes(&d, backward ? SSD_PASS_BWD : SSD_PASS_FWD);
  if (!n) throw LibError(-1, api.last_error());
  const int64_t size = (int64_t)n;
  return empty(at::IntArrayRef(&size, 1), at::kByte, dev);
}

void check_workspace(const Tensor& ws, const at::Device& dev) {
  if (ws.device() != dev || !ws.is_contiguous()) fail("workspace: must be a contiguous tensor on ", dev);
}

// y, final_state, workspace; undefined ones among the three are allocated here (final_state only when `want_final`).
void scan_forward(const Scan& s, Tensor& y, Tensor& fin, Tensor& ws, bool want_final, bool for_backward, int32_t stages) {
  const at::Device dev = s.x.device();
  if (!y.defined()) {
    if (!s.x.is_cuda()) fail("x must be a CUDA tensor (there is no CPU path)");
    y = empty(s.x.sizes(), s.x.scalar_type(), dev);
  }
  const SsdDims d = make_dims(s, &y);
  const Shape state(d.batch, d.nheads, d.headdim, d.dstate);
  if (fin.defined()) check_dense_f32("final_state", &fin, state, dev);
  else if (want_final) fin = empty(state, at::kFloat, dev);
  if (ws.defined()) check_workspace(ws, dev);
  else ws = workspace_for(d, dev, for_backward);
  SsdFwdPtrs p;
  std::memset(&p, 0, sizeof p);
  p.x = ptr(&s.x); p.dt = ptr(&s.dt); p.A = fptr(&s.A); p.Bm = ptr(&s.Bm); p.Cm = ptr(&s.Cm); p.D = fptr(s.D); p.z = ptr(s.z);
  p.init_state = fptr(s.init); p.y = ptr(&y); p.final_state = fptr(&fin); p.dt_bias = fptr(s.bias);
  const c10::cuda::CUDAGuard guard(dev);
  check_rc(api.forward_staged(&d, &p, ws.data_ptr(), (size_t)ws.numel(), stream_of(dev), stages));
}

struct Grads { Tensor dx, ddt, dA, dB, dC, dD, dz, dinit, dbias; };

// A caller-provided output must be dense, 16-byte aligned and of the right shape; a missing one is allocated.
void out_slot(const char* key, Tensor& t, const Shape& shape, at::ScalarType dtype, const at::Device& dev) {
  if (!t.defined()) { t = empty(shape, dtype, dev); return; }
  if (!same(t, shape) || t.scalar_type() != dtype || t.device() != dev)
    fail("out['", key, "']: expected ", at::IntArrayRef(shape), " ", dtype, " on ", dev, ", got ", t.sizes(), " ", t.scalar_type(),
         " on ", t.device());
  if (!t.is_contiguous() || (uintptr_t)t.data_ptr() % 16) fail("out['", key, "']: must be contiguous and 16-byte aligned");
}

void scan_backward(const Scan& s, const Tensor& dy, const Tensor* dfin, Tensor& ws, bool fwd_saved, bool want_dinit, int32_t stages,
                   Grads& o) {
  const SsdDims d = make_dims(s, &dy);
  const at::Device dev = s.x.device();
  const at::ScalarType st = s.x.scalar_type();
  const int64_t B = d.batch, L = d.seqlen, H = d.nheads, P = d.headdim, N = d.dstate, G = d.ngroups;
  check_dense_f32("dfinal_state", dfin, Shape(B, H, P, N), dev);
  out_slot("dx", o.dx, Shape(B, L, H, P), st, dev);
  out_slot("ddt", o.ddt, Shape(B, L, H), at::kFloat, dev);
  out_slot("dA", o.dA, Shape(H), at::kFloat, dev);
  out_slot("dB", o.dB, Shape(B, L, G, N), st, dev);
  out_slot("dC", o.dC, Shape(B, L, G, N), st, dev);
  if (s.D) out_slot("dD", o.dD, Shape(H), at::kFloat, dev);
  if (s.z) out_slot("dz", o.dz, Shape(B, L, H, P), st, dev);
  if (want_dinit || s.init) out_slot("dinit", o.dinit, Shape(B, H, P, N), at::kFloat, dev);
  if (s.bias) out_slot("ddt_bias", o.dbias, Shape(H), at::kFloat, dev);
  if (ws.defined()) {
    check_workspace(ws, dev);
  } else {
    if (fwd_saved) fail("fwd_saved=True needs the workspace the forward ran in");
    ws = workspace_for(d, dev, true);
  }
  SsdBwdPtrs p;
  std::memset(&p, 0, sizeof p);
  p.x = ptr(&s.x); p.dt = ptr(&s.dt); p.A = fptr(&s.A); p.Bm = ptr(&s.Bm); p.Cm = ptr(&s.Cm); p.D = fptr(s.D); p.z = ptr(s.z);
  p.init_state = fptr(s.init); p.dy = ptr(&dy); p.dfinal_state = fptr(dfin); p.dx = ptr(&o.dx); p.ddt = fptr(&o.ddt);
  p.dA = fptr(&o.dA); p.dB = ptr(&o.dB); p.dC = ptr(&o.dC); p.dD = fptr(&o.dD); p.dz = ptr(&o.dz); p.dinit_state = fptr(&o.dinit);
  p.fwd_saved = fwd_saved ? 1 : 0; p.dt_bias = fptr(s.bias); p.ddt_bias = fptr(&o.dbias);
  const c10::cuda::CUDAGuard guard(dev);
  check_rc(api.backward_staged(&d, &p, ws.data_ptr(), (size_t)ws.numel(), stream_of(dev), stages));
}

// ---- conv1d and RMS norm -----------------------------------------------------------------------------------------------
void check_conv_weights(const Tensor& in, const Tensor& weight, const Tensor* bias) {
  if (weight.scalar_type() != at::kFloat || !weight.is_contiguous() || weight.dim() != 2)
    fail("conv1d: weight must be contiguous fp32 [channels, width]");
  if (weight.device() != in.device()) fail("conv1d: weight: expected device ", in.device(), ", got ", weight.device());
  if (weight.size(0) != in.size(2)) fail("conv1d: weight rows must equal the channel count");
  check_values_f32("conv1d: bias", bias, weight.size(0), in.device());
}
SsdConvDims conv_dims(const Tensor& in, const Tensor& out, int64_t width, bool activation) {
  if (!in.is_cuda() || in.dim() != 3 || (in.scalar_type() != at::kBFloat16 && in.scalar_type() != at::kFloat))
    fail("conv1d: input must be a CUDA [batch, seqlen, channels] bf16/fp32 tensor");
  if (in.stride(2) != 1 || out.stride(2) != 1) fail("conv1d: the channel dim must be dense");
  SsdConvDims d;
  std::memset(&d, 0, sizeof d);
  d.batch = (int32_t)in.size(0); d.seqlen = (int32_t)in.size(1); d.channels = (int32_t)in.size(2);
  d.width = (int32_t)width; d.dtype = storage_type(in); d.device = in.device().index(); d.activation = activation ? 1 : 0;
  d.in_stride_b = in.stride(0); d.in_stride_l = in.stride(1); d.out_stride_b = out.stride(0); d.out_stride_l = out.stride(1);
  return d;
}
void conv_forward(const Tensor& in, const Tensor& weight, const Tensor* bias, bool activation, Tensor& out) {
  if (!in.is_cuda() || in.dim() != 3) fail("conv1d: input must be a CUDA [batch, seqlen, channels] bf16/fp32 tensor");
  check_conv_weights(in, weight, bias);
  if (!out.defined()) out = empty(in.sizes(), in.scalar_type(), in.device());
  if (!same(out, in.sizes()) || out.scalar_type() != in.scalar_type() || out.device() != in.device())
    fail("conv1d: out: expected ", in.sizes(), " ", in.scalar_type(), " on ", in.device(), ", got ", out.sizes(), " ", out.scalar_type(),
         " on ", out.device());
  const SsdConvDims d = conv_dims(in, out, weight.size(1), activation);
  const c10::cuda::CUDAGuard guard(in.device());
  check_rc(api.conv1d_forward(&d, ptr(&in), fptr(&weight), fptr(bias), ptr(&out), stream_of(in.device())));
}
struct ConvGrads { Tensor din, dweight, dbias; };
ConvGrads conv_backward(const Tensor& in, const Tensor& weight, const Tensor* bias, const Tensor* const* douts, int ndout, bool activation) {
  const at::Device dev = in.device();
  if (!in.is_cuda() || in.dim() != 3) fail("conv1d: input must be a CUDA [batch, seqlen, channels] bf16/fp32 tensor");
  check_conv_weights(in, weight, bias);
  ConvGrads g;
  g.din = empty(in.sizes(), in.scalar_type(), dev);
  const SsdConvDims d = conv_dims(in, g.din, weight.size(1), activation);
  SsdConvGrad segs[3];
  std::memset(segs, 0, sizeof segs);
  if (ndout > 3) fail("conv1d backward: 1 to 3 gradient segments, got ", (int64_t)ndout);
  for (int i = 0; i < ndout; ++i) {
    const Tensor& t = *douts[i];
    if (t.dim() != 3 || t.scalar_type() != in.scalar_type() || t.stride(2) != 1 || t.size(0) != in.size(0) || t.size(1) != in.size(1) || t.device() != dev)
      fail("conv1d backward: bad gradient segment");
    segs[i].ptr = ptr(&t); segs[i].channels = (int32_t)t.size(2); segs[i].stride_b = t.stride(0); segs[i].stride_l = t.stride(1);
  }
  g.dweight = empty(weight.sizes(), at::kFloat, dev);
  g.dbias = empty(Shape(weight.size(0)), at::kFloat, dev);
  const size_t nbytes = api.conv1d_workspace_bytes(&d);
  if (!nbytes) fail(api.last_error());
  Tensor ws = empty(Shape((int64_t)nbytes), at::kByte, dev);
  const c10::cuda::CUDAGuard guard(dev);
  check_rc(api.conv1d_backward(&d, ptr(&in), fptr(&weight), fptr(bias), segs, ndout, ptr(&g.din), g.din.stride(0), g.din.stride(1),
                               fptr(&g.dweight), fptr(&g.dbias), ws.data_ptr(), nbytes, stream_of(dev)));
  return g;
}

void check_norm(const Tensor& in, const Tensor* weight) {
  if (!in.is_cuda() || (in.scalar_type() != at::kBFloat16 && in.scalar_type() != at::kFloat) || !in.is_contiguous() || in.dim() < 1)
    fail("rmsnorm: input must be a contiguous CUDA bf16/fp32 tensor");
  check_values_f32("rmsnorm: weight", weight, in.size(-1), in.device());
}
SsdNormDims norm_dims(const Tensor& in, double eps) {   // `in` contiguous: every dim but the last is a row
  SsdNormDims d;
  std::memset(&d, 0, sizeof d);
  d.width = (int32_t)in.size(-1); d.rows = d.width ? in.numel() / d.width : 0;
  d.dtype = storage_type(in); d.device = in.device().index(); d.eps = (float)eps;
  d.in_stride_row = d.out_stride_row = d.width;
  return d;
}
void norm_forward(const Tensor& in, const Tensor* weight, double eps, Tensor& out, Tensor& rstd) {
  check_norm(in, weight);
  const SsdNormDims d = norm_dims(in, eps);
  out = empty(in.sizes(), in.scalar_type(), in.device());
  rstd = empty(Shape(d.rows), at::kFloat, in.device());
  const c10::cuda::CUDAGuard guard(in.device());
  check_rc(api.rmsnorm_forward(&d, ptr(&in), fptr(weight), ptr(&out), fptr(&rstd), stream_of(in.device())));
}
void norm_backward(const Tensor& in, const Tensor* weight, const Tensor& rstd, const Tensor& dout_, double eps, Tensor& din, Tensor& dweight) {
  check_norm(in, weight);
  if (dout_.numel() != in.numel() || dout_.scalar_type() != in.scalar_type() || dout_.device() != in.device())
    fail("rmsnorm: dout: expected ", in.sizes(), " ", in.scalar_type(), " on ", in.device(), ", got ", dout_.sizes(), " ", dout_.scalar_type(),
         " on ", dout_.device());
  const Tensor dout = dout_.contiguous();
  const SsdNormDims d = norm_dims(in, eps);
  check_values_f32("rmsnorm: rstd", &rstd, d.rows, in.device());
  const at::Device dev = in.device();
  din = empty(in.sizes(), in.scalar_type(), dev);
  Tensor ws;
  if (weight) {
    dweight = empty(weight->sizes(), at::kFloat, dev);
    const size_t n = api.rmsnorm_workspace_bytes(&d);
    ws = empty(Shape((int64_t)n), at::kByte, dev);
  }
  const c10::cuda::CUDAGuard guard(dev);
  check_rc(api.rmsnorm_backward(&d, ptr(&in), fptr(weight), fptr(&rstd), ptr(&dout), d.width, ptr(&din), d.width, fptr(&dweight), ptr(&ws),
                                ws.defined() ? (size_t)ws.numel() : 0, stream_of(dev)));
}

// ---- selective scan, convolution with history, projection ---------------------------------------------------------------
// Distance between rows along `dim`; 0 ("dense") where there is one row, whose stride says nothing.
int64_t apart(const Tensor& t, int dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }
// A [.., rows, inner] operand whose inner dims (all from `outer` on) are dense and whose rows lie apart.
void check_rows(const char* name, const Tensor& t, at::IntArrayRef shape, int outer, at::ScalarType dtype, const at::Device& dev) {
  if (!same(t, shape)) fail(name, ": expected shape ", shape, ", got ", t.sizes());
  if (t.scalar_type() != dtype) fail(name, ": expected dtype ", dtype, ", got ", t.scalar_type());
  if (t.device() != dev) fail(name, ": expected device ", dev, ", got ", t.device());
  int64_t dense = 1;
  for (int i = (int)t.dim() - 1; i >= outer; --i) {
    if (t.size(i) > 1 && t.stride(i) != dense) fail(name, ": the dims from ", (int64_t)outer, " on must be dense");
    dense *= t.size(i);
  }
  if (overlaid(t, outer)) fail(name, ": expanded over a dim (stride 0); make it contiguous");
}
void check_lengths(const Tensor* t, int64_t batch, const at::Device& dev) {
  if (t && (t->dim() != 1 || t->size(0) != batch || t->scalar_type() != at::kInt || t->device() != dev || !t->is_contiguous()))
    fail("lengths: expected ", batch, " contiguous int32 values on ", dev, ", got ", t->sizes(), " ", t->scalar_type(), " on ", t->device());
}
// An incoming gradient as the kernels read it: storage type, dense channels, rows apart.
Tensor usable_rows(const Tensor& g, const Tensor& like, int outer) {
  if (!g.defined()) return at::zeros(like.sizes(), like.options().requires_grad(false));
  Tensor d = g.scalar_type() == like.scalar_type() ? g : g.to(like.scalar_type());
  int64_t dense = 1;
  bool ok = !overlaid(d, outer);
  for (int i = (int)d.dim() - 1; i >= outer; --i) {
    ok = ok && (d.size(i) <= 1 || d.stride(i) == dense);
    dense *= d.size(i);
  }
  return ok ? d : d.contiguous();
}

struct Sel {
  const Tensor &x, &dt, &A, &Bm, &Cm;
  const Tensor *D, *z, *init, *bias, *lengths;
  bool softplus;
};
SsdSelDims sel_dims(const Sel& s, const Tensor* y) {
  if (!s.x.is_cuda()) fail("x must be a CUDA tensor (there is no CPU path)");
  if (s.x.dim() != 3) fail("x must be [batch, seqlen, channels]");
  const int32_t dtype = storage_type(s.x);
  const at::Device dev = s.x.device();
  const at::ScalarType st = s.x.scalar_type();
  const int64_t B = s.x.size(0), L = s.x.size(1), D = s.x.size(2);
  if (s.A.dim() != 2) fail("A must be [channels, dstate]");
  const int64_t N = s.A.size(1);
  if (s.Bm.dim() != 3 && s.Bm.dim() != 4) fail("B must be [batch, seqlen, ngroups, dstate] or [batch, seqlen, dstate]");
  const int64_t G = s.Bm.dim() == 4 ? s.Bm.size(2) : 1;
  if (G <= 0 || D % G) fail("channels (", D, ") must be a multiple of ngroups (", G, ")");
  check_rows("x", s.x, Shape(B, L, D), 2, st, dev);
  check_rows("dt", s.dt, Shape(B, L, D), 2, st, dev);
  for (const Tensor* t : {&s.Bm, &s.Cm}) {
    const char* name = t == &s.Bm ? "B" : "C";
    if (s.Bm.dim() == 4) check_rows(name, *t, Shape(B, L, G, N), 2, st, dev);
    else check_rows(name, *t, Shape(B, L, N), 2, st, dev);
  }
  check_dense_f32("A", &s.A, Shape(D, N), dev);
  check_dense_f32("D", s.D, Shape(D), dev);
  check_dense_f32("dt_bias", s.bias, Shape(D), dev);
  check_dense_f32("init_state", s.init, Shape(B, D, N), dev);
  check_lengths(s.lengths, B, dev);
  SsdSelDims d;
  std::memset(&d, 0, sizeof d);
  d.batch = (int32_t)B; d.seqlen = (int32_t)L; d.channels = (int32_t)D; d.dstate = (int32_t)N; d.ngroups = (int32_t)G;
  d.dtype = dtype; d.device = dev.index(); d.dt_softplus = s.softplus ? 1 : 0;
  d.x_stride_b = apart(s.x, 0); d.x_stride_l = apart(s.x, 1);
  d.dt_stride_b = apart(s.dt, 0); d.dt_stride_l = apart(s.dt, 1);
  d.b_stride_b = apart(s.Bm, 0); d.b_stride_l = apart(s.Bm, 1);
  d.c_stride_b = apart(s.Cm, 0); d.c_stride_l = apart(s.Cm, 1);
  if (s.z) {
    check_rows("z", *s.z, Shape(B, L, D), 2, st, dev);
    d.z_stride_b = apart(*s.z, 0); d.z_stride_l = apart(*s.z, 1);
  }
  if (y) {
    check_rows("y/dy", *y, Shape(B, L, D), 2, st, dev);
    d.y_stride_b = apart(*y, 0); d.y_stride_l = apart(*y, 1);
  }
  return d;
}
Tensor bytes_on(size_t n, const at::Device& dev) {
  if (!n) throw LibError(-1, api.last_error());
  return empty(Shape((int64_t)n), at::kByte, dev);
}
void sel_forward(const Sel& s, Tensor& y, Tensor& fin, Tensor& ws, bool for_backward) {
  SsdSelDims d = sel_dims(s, nullptr);
  const at::Device dev = s.x.device();
  const c10::cuda::CUDAGuard guard(dev);
  y = empty(s.x.sizes(), s.x.scalar_type(), dev);
  fin = empty(Shape(d.batch, d.channels, d.dstate), at::kFloat, dev);
  const size_t need = api.selscan_workspace_bytes(&d, for_backward ? SSD_PASS_BWD : SSD_PASS_FWD);
  if (ws.defined()) check_workspace(ws, dev); else ws = bytes_on(need, dev);
  SsdSelFwdPtrs p;
  std::memset(&p, 0, sizeof p);
  p.x = ptr(&s.x); p.dt = ptr(&s.dt); p.A = fptr(&s.A); p.Bm = ptr(&s.Bm); p.Cm = ptr(&s.Cm); p.D = fptr(s.D); p.z = ptr(s.z);
  p.init_state = fptr(s.init); p.y = ptr(&y); p.final_state = fptr(&fin); p.dt_bias = fptr(s.bias); p.lengths = (const int32_t*)ptr(s.lengths);
  check_rc(api.selscan_forward(&d, &p, ws.data_ptr(), (size_t)ws.nbytes(), stream_of(dev)));
}
struct SelGrads { Tensor dx, ddt, dA, dB, dC, dD, dz, dinit, dbias; };
void sel_backward(const Sel& s, const Tensor& dy, const Tensor* dfin, Tensor& ws, bool saved, SelGrads& o) {
  const SsdSelDims d = sel_dims(s, &dy);
  const at::Device dev = s.x.device();
  const at::ScalarType st = s.x.scalar_type();
  check_dense_f32("dfinal_state", dfin, Shape(d.batch, d.channels, d.dstate), dev);
  const c10::cuda::CUDAGuard guard(dev);
  o.dx = empty(s.x.sizes(), st, dev); o.ddt = empty(s.x.sizes(), st, dev);
  o.dA = empty(s.A.sizes(), at::kFloat, dev);
  o.dB = empty(s.Bm.sizes(), st, dev); o.dC = empty(s.Cm.sizes(), st, dev);
  if (s.D) o.dD = empty(s.D->sizes(), at::kFloat, dev);
  if (s.z) o.dz = empty(s.x.sizes(), st, dev);
  if (s.init) o.dinit = empty(s.init->sizes(), at::kFloat, dev);
  if (s.bias) o.dbias = empty(s.bias->sizes(), at::kFloat, dev);
  if (ws.defined()) {
    check_workspace(ws, dev);
  } else {
    saved = false;
    ws = bytes_on(api.selscan_workspace_bytes(&d, SSD_PASS_BWD), dev);
  }
  SsdSelBwdPtrs p;
  std::memset(&p, 0, sizeof p);
  p.x = ptr(&s.x); p.dt = ptr(&s.dt); p.A = fptr(&s.A); p.Bm = ptr(&s.Bm); p.Cm = ptr(&s.Cm); p.D = fptr(s.D); p.z = ptr(s.z);
  p.init_state = fptr(s.init); p.dy = ptr(&dy); p.dfinal_state = fptr(dfin); p.dx = ptr(&o.dx); p.ddt = ptr(&o.ddt); p.dA = fptr(&o.dA);
  p.dB = ptr(&o.dB); p.dC = ptr(&o.dC); p.dD = fptr(&o.dD); p.dz = ptr(&o.dz); p.dinit_state = fptr(&o.dinit); p.dt_bias = fptr(s.bias);
  p.ddt_bias = fptr(&o.dbias); p.lengths = (const int32_t*)ptr(s.lengths); p.fwd_saved = saved ? 1 : 0;
  check_rc(api.selscan_backward(&d, &p, ws.data_ptr(), (size_t)ws.nbytes(), stream_of(dev)));
}

void check_history(const char* name, const Tensor* h, const Tensor& in, int64_t width) {
  if (!h) return;
  const Shape shape(in.size(0), width - 1, in.size(-1));
  if (!same(*h, shape) || h->scalar_type() != in.scalar_type() || h->device() != in.device() || !h->is_contiguous())
    fail("conv1d: ", name, ": expected a contiguous ", at::IntArrayRef(shape), " ", in.scalar_type(), " tensor on ", in.device(), ", got ",
         h->sizes(), " ", h->scalar_type(), " on ", h->device());
}
SsdConvDims carry_dims(const Tensor& in, const Tensor& weight, const Tensor* bias, bool activation) {
  if (!in.is_cuda() || in.dim() != 3) fail("conv1d: input must be a CUDA [batch, seqlen, channels] bf16/fp32 tensor");
  check_conv_weights(in, weight, bias);
  storage_type(in);
  check_rows("conv1d: input", in, Shape(in.size(0), in.size(1), in.size(2)), 2, in.scalar_type(), in.device());
  SsdConvDims d = conv_dims(in, in, weight.size(1), activation);
  const int64_t C = in.size(2);
  d.out_stride_l = C; d.out_stride_b = C * in.size(1);
  if (in.size(1) <= 1) d.in_stride_l = C;
  if (in.size(0) <= 1) d.in_stride_b = d.in_stride_l * in.size(1);
  return d;
}
void carry_forward(const Tensor& in, const Tensor& weight, const Tensor* bias, const Tensor* hist, const Tensor* lengths, bool activation,
                   Tensor& out, Tensor& nh) {
  const SsdConvDims d = carry_dims(in, weight, bias, activation);
  const at::Device dev = in.device();
  check_history("history", hist, in, d.width);
  check_lengths(lengths, d.batch, dev);
  const c10::cuda::CUDAGuard guard(dev);
  out = empty(in.sizes(), in.scalar_type(), dev);
  nh = empty(Shape(d.batch, d.width - 1, d.channels), in.scalar_type(), dev);
  check_rc(api.conv1d_carry_forward(&d, ptr(&in), fptr(&weight), fptr(bias), ptr(hist), (const int32_t*)ptr(lengths), ptr(&out), ptr(&nh),
                                    stream_of(dev)));
}
struct CarryGrads { Tensor din, dweight, dbias, dhist; };
CarryGrads carry_backward(const Tensor& in, const Tensor& weight, const Tensor* bias, const Tensor* hist, const Tensor& dout,
                          const Tensor* dnew, const Tensor* lengths, bool activation) {
  const SsdConvDims d = carry_dims(in, weight, bias, activation);
  const at::Device dev = in.device();
  check_history("history", hist, in, d.width);
  check_history("gradient of the new history", dnew, in, d.width);
  check_lengths(lengths, d.batch, dev);
  check_rows("conv1d: dout", dout, in.sizes(), 2, in.scalar_type(), dev);
  const c10::cuda::CUDAGuard guard(dev);
  CarryGrads g;
  g.din = empty(in.sizes(), in.scalar_type(), dev);
  g.dweight = empty(weight.sizes(), at::kFloat, dev);
  if (bias) g.dbias = empty(bias->sizes(), at::kFloat, dev);
  if (hist) g.dhist = empty(hist->sizes(), in.scalar_type(), dev);
  Tensor ws = bytes_on(api.conv1d_carry_workspace_bytes(&d), dev);
  const int64_t sl = dout.size(1) > 1 ? dout.stride(1) : (int64_t)d.channels, sb = dout.size(0) > 1 ? dout.stride(0) : sl * dout.size(1);
  check_rc(api.conv1d_carry_backward(&d, ptr(&in), fptr(&weight), fptr(bias), ptr(hist), (const int32_t*)ptr(lengths), ptr(&dout), sb, sl,
                                     ptr(dnew), ptr(&g.din), ptr(&g.dhist), fptr(&g.dweight), fptr(&g.dbias), ws.data_ptr(),
                                     (size_t)ws.numel(), stream_of(dev)));
  return g;
}

// [.., features] as rows of `features` dense values; a copy only where the rows have no one distance.
Tensor as_rows(const char* name, const Tensor& t, int64_t features) {
  if (t.dim() < 1 || t.size(-1) != features) fail("linear: ", name, ": expected ", features, " values in the last dim, got ", t.sizes());
  int64_t rows = 1;                                 // (not numel / features, which may be none; the library refuses that)
  for (int64_t i = 0; i + 1 < t.dim(); ++i) rows *= t.size(i);
  Tensor r = t.dim() == 2 ? t : t.reshape({rows, features});
  if ((features > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < features)) r = r.contiguous();
  return r;
}
SsdLinearDims linear_dims(const Tensor& x, const Tensor& w, int64_t act) {
  if (!x.is_cuda()) fail("x must be a CUDA tensor (there is no CPU path)");
  const int32_t dtype = storage_type(x);
  if (w.dim() != 2 || w.scalar_type() != x.scalar_type() || w.device() != x.device() || !w.is_contiguous())
    fail("linear: weight must be a contiguous [out_features, in_features] ", x.scalar_type(), " tensor on ", x.device());
  SsdLinearDims d;
  std::memset(&d, 0, sizeof d);
  d.in_features = (int32_t)w.size(1); d.out_features = (int32_t)w.size(0);
  d.dtype = dtype; d.device = x.device().index(); d.activation = (int32_t)act;
  return d;
}
Tensor like_rows(const Tensor& x, int64_t features, at::ScalarType st) {   // x's leading dims with `features` in the last one
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = features;
  return empty(shape, st, x.device());
}
void check_vec(const char* name, const Tensor* t, int64_t n, const Tensor& x) {
  if (t && (t->numel() != n || t->scalar_type() != x.scalar_type() || t->device() != x.device() || !t->is_contiguous()))
    fail("linear: ", name, ": expected ", n, " contiguous ", x.scalar_type(), " values on ", x.device(), ", got ", t->sizes(), " ",
         t->scalar_type(), " on ", t->device());
}
void linear_fwd(const Tensor& x, const Tensor& w, const Tensor* bias, const Tensor* res, int64_t act, bool for_backward, Tensor& out, Tensor& pre) {
  SsdLinearDims d = linear_dims(x, w, act);
  const at::Device dev = x.device();
  const int64_t N = d.out_features;
  check_vec("bias", bias, N, x);
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor xr = as_rows("x", x, d.in_features);
  d.rows = xr.size(0); d.x_stride_row = apart(xr, 0);
  Tensor rr;
  if (res) {
    if (res->scalar_type() != x.scalar_type() || res->device() != dev || res->dim() != x.dim() || res->numel() != d.rows * N || res->size(-1) != N)
      fail("linear: residual: expected x's leading dims with ", N, " values in the last, ", x.scalar_type(), " on ", dev, ", got ", res->sizes(),
           " ", res->scalar_type(), " on ", res->device());
    for (int64_t i = 0; i + 1 < x.dim(); ++i) if (res->size(i) != x.size(i)) fail("linear: residual: leading dims ", res->sizes(), " do not match x's ", x.sizes());
    rr = as_rows("residual", *res, N);
    d.residual_stride_row = apart(rr, 0);
  }
  const bool given = out.defined();
  if (given) {
    auto shares = [&](const Tensor& t, int64_t rows, int64_t stride, int64_t features) {   // bytes with `out`
      const char *a = (const char*)t.data_ptr(), *b = (const char*)out.data_ptr();
      return a < b + out.nbytes() && b < a + ((rows - 1) * stride + features) * t.element_size();
    };
    if (shares(xr, xr.size(0), xr.stride(0), d.in_features) || shares(w, N, d.in_features, d.in_features)) fail("linear: out: overlaps x or weight");
    if (bias && shares(*bias, 1, 0, N)) fail("linear: out: overlaps bias");
    // a value of the residual is read by the thread that writes the same element of `out`: its memory, or none of it
    if (rr.defined() && !(rr.data_ptr() == out.data_ptr() && (d.rows == 1 || rr.stride(0) == N)) && shares(rr, d.rows, rr.stride(0), N))
      fail("linear: out: overlaps a part of residual; it has to be the residual itself or apart from it");
    if (out.scalar_type() != x.scalar_type() || out.device() != dev || !out.is_contiguous() || out.dim() != x.dim() || out.numel() != d.rows * N || out.size(-1) != N)
      fail("linear: out: expected a contiguous tensor of x's leading dims with ", N, " values in the last, ", x.scalar_type(), " on ", dev,
           ", got ", out.sizes(), " ", out.scalar_type(), " on ", out.device());
  } else {
    out = like_rows(x, N, x.scalar_type());
  }
  if (for_backward && act) pre = like_rows(x, N, at::kFloat);
  Tensor ws = bytes_on(api.linear_workspace_bytes(&d, SSD_PASS_FWD), dev);
  check_rc(api.linear_forward(&d, ptr(&xr), ptr(&w), ptr(bias), ptr(&rr), ptr(&out), ptr(&pre), ws.data_ptr(), (size_t)ws.numel(), stream_of(dev)));
  if (given) written(out);
}
struct LinGrads { Tensor dx, dw, db; };
LinGrads linear_bwd(const Tensor& dout, const Tensor& x, const Tensor& w, const Tensor* pre, int64_t act, bool want_dx, bool want_dw, bool want_db) {
  SsdLinearDims d = linear_dims(x, w, act);
  const at::Device dev = x.device();
  const int64_t N = d.out_features;
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor xr = as_rows("x", x, d.in_features);
  d.rows = xr.size(0); d.x_stride_row = apart(xr, 0);
  auto check = [&](const char* name, const Tensor& t, at::ScalarType st) {
    if (t.scalar_type() != st || t.device() != dev || t.dim() < 1 || t.size(-1) != N || t.numel() != d.rows * N)
      fail("linear: ", name, ": expected x's leading dims with ", N, " values in the last, ", st, " on ", dev, ", got ", t.sizes(), " ",
           t.scalar_type(), " on ", t.device());
  };
  check("dout", dout, x.scalar_type());
  if (act && !pre) fail("linear: an activation needs the pre that the forward returned with for_backward");
  if (pre) { check("pre", *pre, at::kFloat); if (!pre->is_contiguous()) fail("linear: pre must be contiguous"); }
  const Tensor gr = as_rows("dout", dout, N);
  LinGrads g;
  if (want_dx) g.dx = empty(x.sizes(), x.scalar_type(), dev);
  if (want_dw) g.dw = empty(w.sizes(), x.scalar_type(), dev);
  if (want_db) g.db = empty(Shape(N), x.scalar_type(), dev);
  Tensor ws = bytes_on(api.linear_workspace_bytes(&d, SSD_PASS_BWD), dev);
  check_rc(api.linear_backward(&d, ptr(&xr), ptr(&w), ptr(pre), ptr(&gr), apart(gr, 0), ptr(&g.dx), ptr(&g.dw), ptr(&g.db), ws.data_ptr(),
                               (size_t)ws.numel(), stream_of(dev)));
  return g;
}

// ---- autograd nodes ----------------------------------------------------------------------------------------------------
bool any_requires_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts) if (t && t->requires_grad()) return true;
  return false;
}
// The nodes of the layer operators have no forward-mode derivative; a tangent must not be dropped.
void no_tangents(const char* what, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts) if (t && t->_fw_grad(0).defined()) fail(what, ": there is no forward-mode derivative");
}
// What a node's backward returns.  Where a graph of it is wanted (create_graph) the values are made to depend on what they were computed
// from, the node's operands and incoming gradients, by way of a function that raises: differentiated in turn they do not pass for constants.
variable_list once(const char* what, variable_list grads, const variable_list& operands, const variable_list& incoming) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list in;
  for (const Tensor& g : grads) if (g.defined()) in.push_back(g);
  for (const variable_list* l : {&operands, &incoming})
    for (const Tensor& t : *l) if (t.defined() && t.requires_grad()) in.push_back(t);
  const auto node = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " is differentiable once", (int64_t)in.size());
  const variable_list out = (*node)(std::move(in));
  size_t i = 0;
  for (Tensor& g : grads) if (g.defined()) g = out[i++];
  return grads;
}
using Opt = std::optional<Tensor>;   // an absent operand of a node: Function::apply takes no undefined tensors
Opt optional(const Tensor* t) { return t ? Opt(*t) : Opt(); }
const Tensor* or_null(const Opt& t) { return t.has_value() ? &*t : nullptr; }
Tensor or_undefined(const Opt& t) { return t.has_value() ? *t : Tensor(); }
Tensor or_undefined(const Tensor* t) { return t ? *t : Tensor(); }
const Tensor* or_null(const Tensor& t) { return t.defined() ? &t : nullptr; }
// An incoming gradient in the layout the kernels read: x's dtype, inner dims dense, rows apart (that of a sum or mean over the
// batch comes expanded).
Tensor usable_dy(const Tensor& g, const Tensor& x) {
  if (!g.defined()) return at::zeros(x.sizes(), x.options().requires_grad(false));
  Tensor dy = g.scalar_type() == x.scalar_type() ? g : g.to(x.scalar_type());
  if (dy.stride(-1) != 1 || dy.stride(2) != dy.size(3) || overlaid(dy, 2)) dy = dy.contiguous();
  return dy;
}
Tensor as_type(const Tensor& t, at::ScalarType st) { return t.scalar_type() == st ? t : t.to(st); }
int64_t pack(int64_t chunk, int64_t algo, bool softplus) { return chunk | (algo << 16) | ((int64_t)softplus << 24); }

struct ScanNode : public torch::autograd::Function<ScanNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& Bm, const Tensor& Cm,
                               const Opt& D, const Opt& z, const Opt& init, const Opt& bias, int64_t chunk, int64_t algo, bool softplus) {
    const Scan s{x, dt, A, Bm, Cm, or_null(D), or_null(z), or_null(init), or_null(bias), chunk, algo, softplus};
    Tensor y, fin, ws;
    scan_forward(s, y, fin, ws, true, true, kAllStages);
    ctx->set_materialize_grads(false);   // an unused final state has no gradient: no zeros to allocate, fill and read
    ctx->save_for_backward({x, dt, A, Bm, Cm, or_undefined(D), or_undefined(z), or_undefined(init), or_undefined(bias), ws});
    ctx->saved_data["how"] = pack(chunk, algo, softplus);
    return {y, fin};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list v = ctx->get_saved_variables();
    const int64_t how = ctx->saved_data["how"].toInt();
    const Scan s{v[0], v[1], v[2], v[3], v[4], or_null(v[5]), or_null(v[6]), or_null(v[7]), or_null(v[8]), how & 0xffff, (how >> 16) & 0xff,
                 ((how >> 24) & 1) != 0};
    const Tensor dy = usable_dy(grads[0], s.x);
    const Tensor dfin = grads[1].defined() ? grads[1].contiguous() : Tensor();
    Tensor ws = v[9];
    Grads g;
    scan_backward(s, dy, or_null(dfin), ws, true, false, kAllStages, g);
    return {g.dx, as_type(g.ddt, s.dt.scalar_type()), g.dA, g.dB, g.dC, g.dD, g.dz, g.dinit, g.dbias, Tensor(), Tensor(), Tensor()};
  }
};

// The whole mixer core as one node: conv + silu -> SSD (softplus step size and gate inside) -> RMS norm.
struct MixerNode : public torch::autograd::Function<MixerNode> {
  struct Parts { Tensor x, Bm, Cm; };
  static Parts parts(const Tensor& conv, int64_t H, int64_t P, int64_t G, int64_t N) {
    const int64_t B = conv.size(0), L = conv.size(1), c = conv.stride(1), b = conv.stride(0);
    return {conv.as_strided({B, L, H, P}, {b, c, P, 1}, 0), conv.as_strided({B, L, G, N}, {b, c, N, 1}, H * P),
            conv.as_strided({B, L, G, N}, {b, c, N, 1}, H * P + G * N)};
  }
  static variable_list forward(AutogradContext* ctx, const Tensor& xBC, const Tensor& dt, const Opt& z, const Tensor& cw, const Opt& cb,
                               const Opt& bias, const Tensor& A, const Opt& D, const Opt& nw, const Opt& init, int64_t H, int64_t P,
                               int64_t N, int64_t G, int64_t chunk, double eps, int64_t algo, bool save) {
    if (xBC.dim() != 3 || xBC.size(2) != H * P + 2 * G * N) fail("xBC: expected [batch, seqlen, ", H * P + 2 * G * N, "], got ", xBC.sizes());
    Tensor conv, y, fin, ws, out, rstd;
    conv_forward(xBC, cw, or_null(cb), true, conv);
    const Parts q = parts(conv, H, P, G, N);
    const Scan s{q.x, dt, A, q.Bm, q.Cm, or_null(D), or_null(z), or_null(init), or_null(bias), chunk, algo, true};
    scan_forward(s, y, fin, ws, true, save, kAllStages);
    norm_forward(y.view({y.size(0), y.size(1), H * P}), or_null(nw), eps, out, rstd);
    if (save) {
      ctx->set_materialize_grads(false);
      ctx->save_for_backward({xBC, dt, or_undefined(z), cw, or_undefined(cb), or_undefined(bias), A, or_undefined(D), or_undefined(nw),
                              or_undefined(init), conv, y, rstd, ws});
      ctx->saved_data["how"] = pack(chunk, algo, true);
      ctx->saved_data["geo"] = (int64_t)N;
      ctx->saved_data["ngroups"] = (int64_t)G;
      ctx->saved_data["eps"] = eps;
    }
    return {out, fin};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list v = ctx->get_saved_variables();
    const Tensor &xBC = v[0], &dt = v[1], &cw = v[3], &A = v[6], &conv = v[10], &y = v[11], &rstd = v[12];
    const int64_t how = ctx->saved_data["how"].toInt(), N = ctx->saved_data["geo"].toInt(), G = ctx->saved_data["ngroups"].toInt();
    const double eps = ctx->saved_data["eps"].toDouble();
    const int64_t B = y.size(0), L = y.size(1), H = y.size(2), P = y.size(3);
    const Tensor yr = y.view({B, L, H * P});
    const Tensor dout = grads[0].defined() ? as_type(grads[0], y.scalar_type()) : at::zeros(yr.sizes(), yr.options());
    Tensor dy, dnw;
    norm_backward(yr, or_null(v[8]), rstd, dout, eps, dy, dnw);
    const Parts q = parts(conv, H, P, G, N);
    const Scan s{q.x, dt, A, q.Bm, q.Cm, or_null(v[7]), or_null(v[2]), or_null(v[9]), or_null(v[5]), how & 0xffff, (how >> 16) & 0xff, true};
    const Tensor dfin = grads[1].defined() ? grads[1].contiguous() : Tensor();
    Tensor ws = v[13];
    Grads g;
    scan_backward(s, dy.view({B, L, H, P}), or_null(dfin), ws, true, false, kAllStages, g);
    const Tensor segs[3] = {g.dx.view({B, L, H * P}), g.dB.view({B, L, G * N}), g.dC.view({B, L, G * N})};
    const Tensor* douts[3] = {&segs[0], &segs[1], &segs[2]};
    ConvGrads c = conv_backward(xBC, cw, or_null(v[4]), douts, 3, true);
    return {c.din, as_type(g.ddt, dt.scalar_type()), g.dz, c.dweight, v[4].defined() ? c.dbias : Tensor(), g.dbias, g.dA, g.dD, dnw, g.dinit,
            Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

struct SelNode : public torch::autograd::Function<SelNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& Bm, const Tensor& Cm,
                               const Opt& D, const Opt& z, const Opt& init, const Opt& bias, const Opt& lengths, bool softplus) {
    const Sel s{x, dt, A, Bm, Cm, or_null(D), or_null(z), or_null(init), or_null(bias), or_null(lengths), softplus};
    Tensor y, fin, ws;
    sel_forward(s, y, fin, ws, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, dt, A, Bm, Cm, or_undefined(D), or_undefined(z), or_undefined(init), or_undefined(bias), or_undefined(lengths), ws});
    ctx->saved_data["softplus"] = softplus;
    return {y, fin};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list v = ctx->get_saved_variables();
    const Sel s{v[0], v[1], v[2], v[3], v[4], or_null(v[5]), or_null(v[6]), or_null(v[7]), or_null(v[8]), or_null(v[9]),
                ctx->saved_data["softplus"].toBool()};
    const Tensor dy = usable_rows(grads[0], s.x, 2);
    const Tensor dfin = grads[1].defined() ? grads[1].contiguous() : Tensor();
    Tensor ws = v[10];
    SelGrads g;
    sel_backward(s, dy, or_null(dfin), ws, true, g);
    return once("selective_scan", {g.dx, g.ddt, g.dA, g.dB, g.dC, g.dD, g.dz, g.dinit, g.dbias, Tensor(), Tensor()}, v, grads);
  }
};

struct CarryNode : public torch::autograd::Function<CarryNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& in, const Tensor& w, const Opt& b, const Opt& hist, const Opt& lengths,
                               bool activation) {
    Tensor out, nh;
    carry_forward(in, w, or_null(b), or_null(hist), or_null(lengths), activation, out, nh);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({in, w, or_undefined(b), or_undefined(hist), or_undefined(lengths)});
    ctx->saved_data["activation"] = activation;
    return {out, nh};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list v = ctx->get_saved_variables();
    Tensor dout = usable_rows(grads[0], v[0], 2);
    const int64_t e = dout.element_size();
    if ((uintptr_t)dout.data_ptr() % 16 || apart(dout, 1) * e % 16 || apart(dout, 0) * e % 16) dout = dout.contiguous().clone();
    Tensor dnew = grads[1].defined() ? as_type(grads[1], v[0].scalar_type()).contiguous() : Tensor();
    if (dnew.defined() && (uintptr_t)dnew.data_ptr() % 16) dnew = dnew.clone();
    CarryGrads g = carry_backward(v[0], v[1], or_null(v[2]), or_null(v[3]), dout, or_null(dnew), or_null(v[4]), ctx->saved_data["activation"].toBool());
    return once("causal_conv1d_carry", {g.din, g.dweight, g.dbias, g.dhist, Tensor(), Tensor()}, v, grads);
  }
};

struct LinearNode : public torch::autograd::Function<LinearNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Opt& b, const Opt& res, int64_t act) {
    Tensor out, pre;
    linear_fwd(x, w, or_null(b), or_null(res), act, true, out, pre);
    ctx->save_for_backward({x, w, pre});
    ctx->saved_data["act"] = act;
    ctx->saved_data["bias"] = b.has_value() ? b->sizes().vec() : std::vector<int64_t>{};
    ctx->saved_data["given"] = (int64_t)(b.has_value() + 2 * res.has_value());
    return {out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list v = ctx->get_saved_variables();
    const Tensor dout = as_type(grads[0], v[0].scalar_type());
    const int64_t given = ctx->saved_data["given"].toInt();   // absent operands have no place in the node's list of inputs
    const bool want_db = (given & 1) && ctx->needs_input_grad(2), want_dr = (given & 2) && ctx->needs_input_grad(given & 1 ? 3 : 2);
    LinGrads g;
    if (ctx->needs_input_grad(0) || ctx->needs_input_grad(1) || want_db)
      g = linear_bwd(dout, v[0], v[1], or_null(v[2]), ctx->saved_data["act"].toInt(), ctx->needs_input_grad(0), ctx->needs_input_grad(1), want_db);
    if (want_db) g.db = g.db.view(ctx->saved_data["bias"].toIntVector());
    variable_list r = once("linear", {g.dx, g.dw, g.db, Tensor(), Tensor()}, v, grads);
    if (want_dr) r[3] = dout;                          // (as often differentiable as dout is)
    return r;
  }
};

// ---- Python functions --------------------------------------------------------------------------------------------------
PyObject* pair(const Tensor& a, const Tensor& b) {
  PyObject* r = PyTuple_New(2);
  PyTuple_SET_ITEM(r, 0, wrap(a));
  PyTuple_SET_ITEM(r, 1, wrap(b));
  return r;
}
PyObject* triple(const Tensor& a, const Tensor& b, const Tensor& c) {
  PyObject* r = PyTuple_New(3);
  PyTuple_SET_ITEM(r, 0, wrap(a));
  PyTuple_SET_ITEM(r, 1, wrap(b));
  PyTuple_SET_ITEM(r, 2, wrap(c));
  return r;
}

// One step's operands: `where` is the device of the per-stream vectors (the state's, or the CPU).
struct Step {
  SsdStepDims d;
  SsdStepPtrs p;
  int64_t S, H, P;
};
Step step_of(const Tensor& state, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& Bm, const Tensor& Cm, const Tensor* D,
             const Tensor* z, const Tensor* bias, bool softplus, const at::Device& where) {
  const at::Device dev = state.device();
  if (state.dim() != 4 || state.scalar_type() != at::kFloat || !state.is_contiguous())
    fail("state must be a contiguous float32 [streams, nheads, headdim, dstate] tensor");
  const int64_t S = state.size(0), H = state.size(1), P = state.size(2), N = state.size(3);
  Step s;
  std::memset(&s, 0, sizeof s);
  SsdStepDims& d = s.d;
  d.dtype = storage_type(x);
  if (Bm.dim() != 3 || Bm.size(0) != S || Bm.size(2) != N) fail("B must be [streams, ngroups, dstate]");
  const int64_t G = Bm.size(1);
  if (G <= 0 || H % G) fail("nheads (", H, ") must be a multiple of ngroups (", G, ")");
  auto vec = [&](const char* name, const Tensor& t, const Shape& shape) {
    if (!same(t, shape) || t.scalar_type() != x.scalar_type() || t.device() != where)
      fail(name, ": expected ", at::IntArrayRef(shape), " ", x.scalar_type(), " on ", where);
    if (t.stride(-1) != 1 || (t.dim() >= 3 && t.stride(1) != t.size(2))) fail(name, ": inner dims must be dense");
    if (overlaid(t, 1)) fail(name, ": expanded over the streams (stride 0); make it contiguous");
  };
  vec("x", x, Shape(S, H, P)); vec("dt", dt, Shape(S, H)); vec("B", Bm, Shape(S, G, N)); vec("C", Cm, Shape(S, G, N));
  check_dense_f32("A", &A, Shape(H), dev);
  check_dense_f32("D", D, Shape(H), dev);
  check_dense_f32("dt_bias", bias, Shape(H), dev);
  if (z) vec("z", *z, Shape(S, H, P));
  d.streams = (int32_t)S; d.nheads = (int32_t)H; d.headdim = (int32_t)P; d.dstate = (int32_t)N; d.ngroups = (int32_t)G;
  d.device = dev.index(); d.dt_softplus = softplus ? 1 : 0;
  d.x_stride_s = x.stride(0); d.dt_stride_s = dt.stride(0); d.b_stride_s = Bm.stride(0); d.c_stride_s = Cm.stride(0);
  d.z_stride_s = z ? z->stride(0) : 0;
  SsdStepPtrs& p = s.p;
  p.state = fptr(&state); p.x = ptr(&x); p.dt = ptr(&dt); p.A = fptr(&A); p.Bm = ptr(&Bm); p.Cm = ptr(&Cm); p.D = fptr(D); p.z = ptr(z);
  p.dt_bias = fptr(bias);
  s.S = S; s.H = H; s.P = P;
  return s;
}

// state, x, dt, A, B, C, D, z, y, dt_bias, dt_softplus -> y
PyObject* py_state_update(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 11);
    const Tensor &state = a.tensor(0, "state"), &x = a.tensor(1, "x");
    if (!state.is_cuda()) fail("state must be a CUDA tensor (there is no CPU path)");
    const at::Device dev = state.device();
    Step s = step_of(state, x, a.tensor(2, "dt"), a.tensor(3, "A"), a.tensor(4, "B"), a.tensor(5, "C"), a.opt(6, "D"), a.opt(7, "z"),
                     a.opt(9, "dt_bias"), a.flag(10), dev);
    const Tensor* y_in = a.opt(8, "y");
    Tensor y = y_in ? *y_in : empty(Shape(s.S, s.H, s.P), x.scalar_type(), dev);
    if (y_in) {   // rows may lie apart, but not over one another
      const Shape shape(s.S, s.H, s.P);
      if (!same(y, shape) || y.scalar_type() != x.scalar_type() || y.device() != dev)
        fail("y: expected ", at::IntArrayRef(shape), " ", x.scalar_type(), " on ", dev, ", got ", y.sizes(), " ", y.scalar_type(), " on ", y.device());
      if ((s.P > 1 && y.stride(2) != 1) || (s.H > 1 && y.stride(1) != s.P) || (s.S > 1 && y.stride(0) < s.H * s.P)) fail("y: inner dims must be dense and rows apart");
    }
    s.d.y_stride_s = y.stride(0);
    s.p.y = ptr(&y);
    const c10::cuda::CUDAGuard guard(dev);
    check_rc(api.state_update(&s.d, &s.p, stream_of(dev)));
    written(state);
    if (y_in) written(y);
    return wrap(y);
  });
}

// state, x, dt, A, B, C, D, y, y_host: the vectors and y_host in pinned host memory -> None
PyObject* py_state_update_host(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 9);
    const Tensor &state = a.tensor(0, "state"), &y = a.tensor(7, "y"), &yh = a.tensor(8, "y_host");
    if (!state.is_cuda()) fail("state must be a CUDA tensor (there is no CPU path)");
    const at::Device dev = state.device();
    Step s = step_of(state, a.tensor(1, "x"), a.tensor(2, "dt"), a.tensor(3, "A"), a.tensor(4, "B"), a.tensor(5, "C"), a.opt(6, "D"), nullptr,
                     nullptr, false, at::Device(at::kCPU));
    for (const Tensor* t : {&y, &yh})
      if (!same(*t, Shape(s.S, s.H, s.P)) || t->scalar_type() != a.tensor(1, "x").scalar_type() || !t->is_contiguous())
        fail("y: expected a contiguous ", at::IntArrayRef(Shape(s.S, s.H, s.P)), " tensor");
    if (y.device() != dev) fail("y: expected device ", dev, ", got ", y.device());
    s.d.y_stride_s = s.H * s.P;
    s.p.y = ptr(&y);
    const c10::cuda::CUDAGuard guard(dev);
    check_rc(api.state_update_host(&s.d, &s.p, ptr(&yh), stream_of(dev)));
    Py_RETURN_NONE;
  });
}

Scan scan_of(const Args& a, int at, int chunk, int algo, int bias, int softplus) {
  return {a.tensor(at, "x"), a.tensor(at + 1, "dt"), a.tensor(at + 2, "A"), a.tensor(at + 3, "B"), a.tensor(at + 4, "C"), a.opt(at + 5, "D"),
          a.opt(at + 6, "z"), a.opt(at + 7, "init_state"), a.opt(bias, "dt_bias"), a.integer(chunk), a.integer(algo), a.flag(softplus)};
}

// x, dt, B, C, chunk, z, y, algo, dt_softplus -> the bytes of an SsdDims
PyObject* py_dims(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 9);
    const SsdDims d = seq_dims(a.tensor(0, "x"), a.tensor(1, "dt"), a.tensor(2, "B"), a.tensor(3, "C"), a.opt(5, "z"), a.opt(6, "y/dy"),
                               a.integer(4), a.integer(7), a.flag(8));
    return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(&d), sizeof d);
  });
}

// x, dt, A, B, C, D, z, init_state, chunk, algo, workspace, y, final_state, want_final, for_backward, stages, dt_bias, dt_softplus
//   -> y, final_state, workspace
PyObject* py_forward(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 18);
    const Scan s = scan_of(a, 0, 8, 9, 16, 17);
    Tensor ws = or_undefined(a.opt(10, "workspace")), y = or_undefined(a.opt(11, "y")), fin = or_undefined(a.opt(12, "final_state"));
    scan_forward(s, y, fin, ws, a.flag(13), a.flag(14), a.a[15] == Py_None ? kAllStages : (int32_t)a.integer(15));
    return triple(y, fin, ws);
  });
}

// dy, x, dt, A, B, C, D, z, init_state, dfinal_state, chunk, algo, workspace, fwd_saved, want_dinit, stages, out (dict), dt_bias,
// dt_softplus -> out
PyObject* py_backward(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 19);
    const Scan s = scan_of(a, 1, 10, 11, 17, 18);
    PyObject* out = a.a[16];
    Tensor ws = or_undefined(a.opt(12, "workspace"));
    Grads g;
    struct Slot { const char* key; Tensor* t; };
    const Slot slots[] = {{"dx", &g.dx}, {"ddt", &g.ddt}, {"dA", &g.dA}, {"dB", &g.dB}, {"dC", &g.dC}, {"dD", &g.dD}, {"dz", &g.dz},
                          {"dinit", &g.dinit}, {"ddt_bias", &g.dbias}};
    bool given[9] = {};
    for (int i = 0; i < 9; ++i) {
      PyObject* t = PyDict_GetItemString(out, slots[i].key);   // borrowed
      if (!t || t == Py_None) continue;
      if (!THPVariable_Check(t)) fail("out['", slots[i].key, "']: expected a tensor");
      *slots[i].t = THPVariable_Unpack(t);
      given[i] = true;
    }
    scan_backward(s, a.tensor(0, "dy"), a.opt(9, "dfinal_state"), ws, a.flag(13), a.flag(14),
                  a.a[15] == Py_None ? kAllStages : (int32_t)a.integer(15), g);
    auto put = [&](const char* key, const Tensor& t) {
      PyObject* o = wrap(t);
      const int bad = !o || PyDict_SetItemString(out, key, o);
      Py_XDECREF(o);
      if (bad) throw std::runtime_error("out: cannot store a result");
    };
    for (int i = 0; i < 9; ++i)
      if (!given[i] && slots[i].t->defined()) put(slots[i].key, *slots[i].t);
    put("workspace", ws);
    Py_INCREF(out);
    return out;
  });
}

// x, dt, A, B, C, D, z, init_state, chunk, algo, dt_bias, dt_softplus -> y, final_state (differentiable)
PyObject* py_scan(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 12);
    const Scan s = scan_of(a, 0, 8, 9, 10, 11);
    if (!any_requires_grad({&s.x, &s.dt, &s.A, &s.Bm, &s.Cm, s.D, s.z, s.init, s.bias})) {
      Tensor y, fin, ws;
      scan_forward(s, y, fin, ws, true, false, kAllStages);
      return pair(y, fin);
    }
    const variable_list r = ScanNode::apply(s.x, s.dt, s.A, s.Bm, s.Cm, optional(s.D), optional(s.z), optional(s.init), optional(s.bias),
                                            s.chunk, s.algo, s.softplus);
    return pair(r[0], r[1]);
  });
}

// xBC, dt, z, conv_weight, conv_bias, dt_bias, A, D, norm_weight, init_state, nheads, headdim, dstate, ngroups, chunk, eps, algo
//   -> out, final_state (differentiable)
PyObject* py_mixer(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 17);
    const char* names[] = {"xBC", "dt", "z", "conv_weight", "conv_bias", "dt_bias", "A", "D", "norm_weight", "init_state"};
    const Tensor* t[10];
    bool save = false;
    for (int i = 0; i < 10; ++i) {
      t[i] = i == 0 || i == 1 || i == 3 || i == 6 ? &a.tensor(i, names[i]) : a.opt(i, names[i]);   // the rest may be None
      save |= t[i] && t[i]->requires_grad();
    }
    save = save && at::GradMode::is_enabled();
    const variable_list r = MixerNode::apply(*t[0], *t[1], optional(t[2]), *t[3], optional(t[4]), optional(t[5]), *t[6], optional(t[7]),
                                             optional(t[8]), optional(t[9]), a.integer(10), a.integer(11), a.integer(12), a.integer(13),
                                             a.integer(14), a.real(15), a.integer(16), save);
    return pair(r[0], r[1]);
  });
}

// in, weight, bias, activation, out -> out
PyObject* py_conv_forward(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 5);
    Tensor out = or_undefined(a.opt(4, "out"));
    conv_forward(a.tensor(0, "input"), a.tensor(1, "weight"), a.opt(2, "bias"), a.flag(3), out);
    return wrap(out);
  });
}
// in, weight, bias, activation, dout_0 [, dout_1 [, dout_2]] -> din, dweight, dbias
PyObject* py_conv_backward(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, argc);
    if (argc < 4 || argc > 7) fail("conv1d backward: 1 to 3 gradient segments, got ", (int64_t)argc - 4);
    const Tensor* douts[3];
    for (int i = 4; i < argc; ++i) douts[i - 4] = &a.tensor(i, "gradient segment");
    const ConvGrads g = conv_backward(a.tensor(0, "input"), a.tensor(1, "weight"), a.opt(2, "bias"), douts, (int)argc - 4, a.flag(3));
    return triple(g.din, g.dweight, g.dbias);
  });
}
// in, weight, eps -> out, rstd
PyObject* py_norm_forward(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 3);
    Tensor out, rstd;
    norm_forward(a.tensor(0, "input"), a.opt(1, "weight"), a.real(2), out, rstd);
    return pair(out, rstd);
  });
}
// in, weight, rstd, dout, eps -> din, dweight
PyObject* py_norm_backward(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 5);
    Tensor din, dweight;
    norm_backward(a.tensor(0, "input"), a.opt(1, "weight"), a.tensor(2, "rstd"), a.tensor(3, "dout"), a.real(4), din, dweight);
    return pair(din, dweight);
  });
}

Sel sel_of(const Args& a, int at, int bias, int softplus, int lengths) {
  return {a.tensor(at, "x"), a.tensor(at + 1, "dt"), a.tensor(at + 2, "A"), a.tensor(at + 3, "B"), a.tensor(at + 4, "C"), a.opt(at + 5, "D"),
          a.opt(at + 6, "z"), a.opt(at + 7, "init_state"), a.opt(bias, "dt_bias"), a.opt(lengths, "lengths"), a.flag(softplus)};
}
// x, dt, A, B, C, D, z, init_state, dt_bias, dt_softplus, lengths, for_backward, workspace -> y, final_state, workspace
PyObject* py_sel_forward(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 13);
    Tensor y, fin, ws = or_undefined(a.opt(12, "workspace"));
    sel_forward(sel_of(a, 0, 8, 9, 10), y, fin, ws, a.flag(11));
    return triple(y, fin, ws);
  });
}
// dy, x, dt, A, B, C, D, z, init_state, dfinal_state, dt_bias, dt_softplus, lengths, workspace -> dict
PyObject* py_sel_backward(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 14);
    const Sel s = sel_of(a, 1, 10, 11, 12);
    Tensor ws = or_undefined(a.opt(13, "workspace"));
    SelGrads g;
    sel_backward(s, a.tensor(0, "dy"), a.opt(9, "dfinal_state"), ws, true, g);
    PyObject* out = PyDict_New();
    if (!out) throw std::runtime_error("out of memory");
    struct { const char* key; const Tensor* t; } const slots[] = {{"dx", &g.dx}, {"ddt", &g.ddt}, {"dA", &g.dA}, {"dB", &g.dB}, {"dC", &g.dC},
        {"dD", &g.dD}, {"dz", &g.dz}, {"dinit", &g.dinit}, {"ddt_bias", &g.dbias}};
    for (const auto& e : slots) {
      if (!e.t->defined()) continue;
      PyObject* o = wrap(*e.t);
      const int bad = !o || PyDict_SetItemString(out, e.key, o);
      Py_XDECREF(o);
      if (bad) { Py_DECREF(out); throw std::runtime_error("cannot store a result"); }
    }
    return out;
  });
}
// x, dt, A, B, C, D, z, init_state, dt_bias, dt_softplus, lengths -> y, final_state (differentiable)
PyObject* py_sel_scan(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 11);
    const Sel s = sel_of(a, 0, 8, 9, 10);
    no_tangents("selective_scan", {&s.x, &s.dt, &s.A, &s.Bm, &s.Cm, s.D, s.z, s.init, s.bias});
    if (!any_requires_grad({&s.x, &s.dt, &s.A, &s.Bm, &s.Cm, s.D, s.z, s.init, s.bias})) {
      Tensor y, fin, ws;
      sel_forward(s, y, fin, ws, false);
      return pair(y, fin);
    }
    const variable_list r = SelNode::apply(s.x, s.dt, s.A, s.Bm, s.Cm, optional(s.D), optional(s.z), optional(s.init), optional(s.bias),
                                           optional(s.lengths), s.softplus);
    return pair(r[0], r[1]);
  });
}
// state, x, dt, A, B, C, D, z, y, dt_bias, dt_softplus -> y
PyObject* py_sel_step(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 11);
    const Tensor &state = a.tensor(0, "state"), &x = a.tensor(1, "x"), &dt = a.tensor(2, "dt"), &A = a.tensor(3, "A"), &Bm = a.tensor(4, "B"),
                 &Cm = a.tensor(5, "C");
    const Tensor *D = a.opt(6, "D"), *z = a.opt(7, "z"), *y_in = a.opt(8, "y"), *bias = a.opt(9, "dt_bias");
    if (!state.is_cuda()) fail("state must be a CUDA tensor (there is no CPU path)");
    const at::Device dev = state.device();
    if (state.dim() != 3 || state.scalar_type() != at::kFloat || !state.is_contiguous())
      fail("state must be a contiguous float32 [streams, channels, dstate] tensor");
    const int64_t S = state.size(0), C = state.size(1), N = state.size(2);
    const at::ScalarType st = x.scalar_type();
    SsdSelStepDims d;
    std::memset(&d, 0, sizeof d);
    d.dtype = storage_type(x);
    if (Bm.dim() != 2 && Bm.dim() != 3) fail("B must be [streams, ngroups, dstate] or [streams, dstate]");
    const int64_t G = Bm.dim() == 3 ? Bm.size(1) : 1;
    if (G <= 0 || C % G) fail("channels (", C, ") must be a multiple of ngroups (", G, ")");
    check_rows("x", x, Shape(S, C), 1, st, dev);
    check_rows("dt", dt, Shape(S, C), 1, st, dev);
    for (const Tensor* t : {&Bm, &Cm}) {
      const char* name = t == &Bm ? "B" : "C";
      if (Bm.dim() == 3) check_rows(name, *t, Shape(S, G, N), 1, st, dev);
      else check_rows(name, *t, Shape(S, N), 1, st, dev);
    }
    if (z) check_rows("z", *z, Shape(S, C), 1, st, dev);
    check_dense_f32("A", &A, Shape(C, N), dev);
    check_dense_f32("D", D, Shape(C), dev);
    check_dense_f32("dt_bias", bias, Shape(C), dev);
    const c10::cuda::CUDAGuard guard(dev);
    if (y_in) check_rows("y", *y_in, Shape(S, C), 1, st, dev);
    Tensor y = y_in ? *y_in : empty(Shape(S, C), st, dev);
    d.streams = (int32_t)S; d.channels = (int32_t)C; d.dstate = (int32_t)N; d.ngroups = (int32_t)G; d.device = dev.index();
    d.dt_softplus = a.flag(10) ? 1 : 0;
    d.x_stride_s = apart(x, 0); d.dt_stride_s = apart(dt, 0); d.b_stride_s = apart(Bm, 0); d.c_stride_s = apart(Cm, 0);
    d.z_stride_s = z ? apart(*z, 0) : 0; d.y_stride_s = apart(y, 0);
    SsdStepPtrs p;
    std::memset(&p, 0, sizeof p);
    p.state = fptr(&state); p.x = ptr(&x); p.dt = ptr(&dt); p.A = fptr(&A); p.Bm = ptr(&Bm); p.Cm = ptr(&Cm); p.D = fptr(D); p.z = ptr(z);
    p.y = ptr(&y); p.dt_bias = fptr(bias);
    check_rc(api.selscan_step(&d, &p, stream_of(dev)));
    written(state);
    if (y_in) written(y);
    return wrap(y);
  });
}
// in, weight, bias, history, lengths, activation -> out, new_history
PyObject* py_carry_forward(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 6);
    Tensor out, nh;
    carry_forward(a.tensor(0, "input"), a.tensor(1, "weight"), a.opt(2, "bias"), a.opt(3, "history"), a.opt(4, "lengths"), a.flag(5), out, nh);
    return pair(out, nh);
  });
}
// in, weight, bias, history, dout, dnew_history, lengths, activation -> din, dweight, dbias, dhistory
PyObject* py_carry_backward(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 8);
    const CarryGrads g = carry_backward(a.tensor(0, "input"), a.tensor(1, "weight"), a.opt(2, "bias"), a.opt(3, "history"), a.tensor(4, "dout"),
                                        a.opt(5, "dnew_history"), a.opt(6, "lengths"), a.flag(7));
    return Py_BuildValue("(NNNN)", wrap(g.din), wrap(g.dweight), wrap(g.dbias), wrap(g.dhist));
  });
}
// in, weight, bias, history, lengths, activation -> out, new_history (differentiable)
PyObject* py_carry(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 6);
    const Tensor &in = a.tensor(0, "input"), &w = a.tensor(1, "weight");
    const Tensor *b = a.opt(2, "bias"), *h = a.opt(3, "history"), *l = a.opt(4, "lengths");
    no_tangents("causal_conv1d_carry", {&in, &w, b, h});
    if (!any_requires_grad({&in, &w, b, h})) {
      Tensor out, nh;
      carry_forward(in, w, b, h, l, a.flag(5), out, nh);
      return pair(out, nh);
    }
    const variable_list r = CarryNode::apply(in, w, optional(b), optional(h), optional(l), a.flag(5));
    return pair(r[0], r[1]);
  });
}
// history, in, weight, bias, activation, out -> out
PyObject* py_conv_step(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 6);
    const Tensor &hist = a.tensor(0, "history"), &in = a.tensor(1, "input"), &w = a.tensor(2, "weight");
    const Tensor *b = a.opt(3, "bias"), *out_in = a.opt(5, "out");
    if (!in.is_cuda() || in.dim() != 2) fail("conv1d: input of a step must be a CUDA [streams, channels] bf16/fp32 tensor");
    const at::Device dev = in.device();
    check_rows("conv1d: input", in, Shape(in.size(0), in.size(1)), 1, in.scalar_type(), dev);
    const Tensor in3 = in.unsqueeze(1);
    SsdConvDims d = carry_dims(in3, w, b, a.flag(4));
    check_history("history", &hist, in, d.width);
    const c10::cuda::CUDAGuard guard(dev);
    if (out_in) check_rows("conv1d: out", *out_in, Shape(in.size(0), in.size(1)), 1, in.scalar_type(), dev);
    Tensor out = out_in ? *out_in : empty(Shape(in.size(0), in.size(1)), in.scalar_type(), dev);
    d.out_stride_b = out.size(0) > 1 ? out.stride(0) : out.size(1);
    if (out.size(0) > 1 && out.stride(0) < out.size(1)) fail("conv1d: out: rows must lie apart");
    check_rc(api.conv1d_step(&d, ptr(&in), fptr(&w), fptr(b), ptr(&hist), ptr(&out), stream_of(dev)));
    written(hist);
    if (out_in) written(out);
    return wrap(out);
  });
}
// x, weight, bias, residual, activation, for_backward, out -> out, pre
PyObject* py_linear_forward(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 7);
    Tensor out = or_undefined(a.opt(6, "out")), pre;
    linear_fwd(a.tensor(0, "x"), a.tensor(1, "weight"), a.opt(2, "bias"), a.opt(3, "residual"), a.integer(4), a.flag(5), out, pre);
    return pair(out, pre);
  });
}
// dout, x, weight, pre, activation, want_dx, want_dweight, want_dbias -> dx, dweight, dbias
PyObject* py_linear_backward(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 8);
    const LinGrads g = linear_bwd(a.tensor(0, "dout"), a.tensor(1, "x"), a.tensor(2, "weight"), a.opt(3, "pre"), a.integer(4), a.flag(5), a.flag(6), a.flag(7));
    return triple(g.dx, g.dw, g.db);
  });
}
// x, weight, bias, residual, activation -> out (differentiable)
PyObject* py_linear(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 5);
    const Tensor &x = a.tensor(0, "x"), &w = a.tensor(1, "weight");
    const Tensor *b = a.opt(2, "bias"), *r = a.opt(3, "residual");
    no_tangents("linear", {&x, &w, b, r});
    if (!any_requires_grad({&x, &w, b, r})) {
      Tensor out, pre;
      linear_fwd(x, w, b, r, a.integer(4), false, out, pre);
      return wrap(out);
    }
    return wrap(LinearNode::apply(x, w, optional(b), optional(r), a.integer(4))[0]);
  });
}

// addresses (a tuple in Api's order), SsdError, torch.OutOfMemoryError
PyObject* py_bind(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  return guarded([&]() -> PyObject* {
    const Args a(argv, argc, 3);
    constexpr Py_ssize_t n = sizeof(Api) / sizeof(void*);
    if (!PyTuple_Check(argv[0]) || PyTuple_GET_SIZE(argv[0]) != n) fail("bind: expected ", (int64_t)n, " addresses");
    void** slot = reinterpret_cast<void**>(&api);
    for (Py_ssize_t i = 0; i < n; ++i) slot[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(argv[0], i));
    Py_INCREF(argv[1]);
    Py_INCREF(argv[2]);
    ssd_error = argv[1];   // the module is bound once and lives as long as the process
    oom_error = argv[2];
    Py_RETURN_NONE;
  });
}

#define FAST(name, fn) {name, (PyCFunction)(void (*)(void))fn, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST("bind", py_bind), FAST("dims", py_dims), FAST("state_update", py_state_update), FAST("state_update_host", py_state_update_host), FAST("forward", py_forward),
                         FAST("backward", py_backward), FAST("scan", py_scan), FAST("mixer", py_mixer),
                         FAST("conv1d_forward", py_conv_forward), FAST("conv1d_backward", py_conv_backward),
                         FAST("rmsnorm_forward", py_norm_forward), FAST("rmsnorm_backward", py_norm_backward),
                         FAST("selscan_forward", py_sel_forward), FAST("selscan_backward", py_sel_backward), FAST("selscan", py_sel_scan),
                         FAST("selscan_step", py_sel_step), FAST("carry_forward", py_carry_forward), FAST("carry_backward", py_carry_backward),
                         FAST("carry", py_carry), FAST("conv1d_step", py_conv_step), FAST("linear_forward", py_linear_forward),
                         FAST("linear_backward", py_linear_backward), FAST("linear", py_linear), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ssd_host", "native host path of the SSD entry points", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__ssd_host(void) { return PyModule_Create(&module); }
