// The host side of the 4-bit operators and of the distillation loss in native code: a call's allocations and launches in
// one step from Python, as host_path.cpp does for the 8-bit path (a single-token product runs for a few microseconds, which
// is what the Python around it would cost by itself).  Every function allocates through torch, launches on the stream that
// it is given through the C-ABI of include/mxfp4_ops.h, does not wait, and runs without the interpreter's lock.  Shapes,
// types, strides and devices are checked here; an error raises _native.NativeError.
#include <c10/core/DeviceGuard.h>
#include <torch/extension.h>

#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>

#include "../../include/mxfp4_ops.h"
#include "../../include/mxfp8_mlp.h"

namespace py = pybind11;
using at::Tensor;
using OptT = std::optional<Tensor>;

namespace {

PyObject* g_error = nullptr;  // _native.NativeError
struct NativeError : std::runtime_error {
  using std::runtime_error::runtime_error;
};
[[noreturn]] void raise(const std::string& msg) { throw NativeError(msg); }
void ok(int rc, const char* name) {
  if (rc) raise(std::string(name) + " failed with code " + std::to_string(rc) + ": " + mxfp8_last_error());
}
void need(bool cond, const char* what, const char* msg) {
  if (!cond) raise(std::string(what) + ": " + msg);
}

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t pad(int64_t a, int64_t b) { return cdiv(a, b) * b; }
int64_t code_bytes(int64_t rows, int64_t cols, int64_t fmt) {
  return pad(rows, 32) * pad(cols, 128) / (fmt == MXFP4_E4M3 ? 1 : 2);
}
int64_t scale_bytes(int64_t rows, int64_t cols) { return cdiv(rows, 128) * cdiv(cols, 128) * 512; }
void* stm(int64_t s) { return reinterpret_cast<void*>(s); }
void* ptr(const Tensor& t) { return t.data_ptr(); }
void* ptr(const OptT& t) { return t ? t->data_ptr() : nullptr; }

int64_t type_of(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return MXFP4_BF16;
    case at::kHalf: return MXFP4_F16;
    case at::kFloat: return MXFP4_F32;
    default: raise(std::string(what) + ": bfloat16, float16 or float32 tensors");
  }
}
int64_t half_type(const Tensor& t, const char* what) {
  need(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, what, "bfloat16 or float16 activations");
  return type_of(t, what);
}
void gpu(const Tensor& t, const char* what) {
  if (!t.is_cuda()) raise(std::string(what) + ": tensors must be on the GPU (there is no CPU implementation)");
}
void same(const Tensor& a, const Tensor& b, const char* what) {
  need(a.device() == b.device(), what, "tensors on different devices");
}
Tensor empty(at::IntArrayRef shape, at::ScalarType dt, const Tensor& like) {
  return at::empty(shape, like.options().dtype(dt).requires_grad(false).layout(at::kStrided));
}
// [.., C] as a matrix with unit column stride: a view where the strides allow it
Tensor rows_of(const Tensor& x) {
  Tensor m = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  return m.size(1) > 1 && m.stride(1) != 1 ? m.contiguous() : m;
}
// Row stride for the library; a matrix of one row (or one column) may carry any stride of its size-1 dimension
int64_t ld_of(const Tensor& m) { return m.size(0) <= 1 ? std::max<int64_t>(m.size(1), 1) : m.stride(0); }
Tensor shaped(Tensor y, const Tensor& x, int64_t cols) {
  if (x.dim() == 2) return y;
  auto s = x.sizes().vec();
  s.back() = cols;
  return y.view(s);
}

struct Operand {
  Tensor q, s;
};
Operand operand(int64_t rows, int64_t cols, int64_t fmt, const Tensor& like) {
  return {empty({code_bytes(rows, cols, fmt)}, at::kByte, like), empty({scale_bytes(rows, cols)}, at::kFloat8_e8m0fnu, like)};
}

// A pass's own operand (one allocation)
struct Temp {
  Tensor buf;
  char *q, *s;
  Temp(int64_t rows, int64_t cols, int64_t fmt, const Tensor& like) {
    const int64_t nq = code_bytes(rows, cols, fmt);  // a multiple of 2 KB
    buf = empty({nq + scale_bytes(rows, cols)}, at::kByte, like);
    q = static_cast<char*>(buf.data_ptr());
    s = q + nq;
  }
};

std::tuple<Tensor, Tensor> quant(const Tensor& x, int64_t fmt, int64_t order, int64_t stream) {
  const char* what = "mx4_quant";
  gpu(x, what);
  c10::OptionalDeviceGuard guard(x.device());
  need(x.dim() == 2, what, "a matrix");
  const Tensor m = rows_of(x);
  Operand o = operand(m.size(0), m.size(1), fmt, m);
  ok(mxfp4_quant(ptr(m), type_of(m, what), m.size(0), m.size(1), ld_of(m), fmt, ptr(o.q), ptr(o.s), order, nullptr, nullptr,
                 0, 0, 0, stm(stream)),
     "mxfp4_quant");
  return {o.q, o.s};
}

// both axes from one read, each in its row order
std::tuple<Tensor, Tensor, Tensor, Tensor> quant_both(const Tensor& x, int64_t fmt, int64_t order, int64_t stream) {
  const char* what = "mx4_quant";
  gpu(x, what);
  c10::OptionalDeviceGuard guard(x.device());
  need(x.dim() == 2, what, "a matrix");
  const Tensor m = rows_of(x);
  const int64_t R = m.size(0), C = m.size(1);
  Operand o = operand(R, C, fmt, m), t = operand(C, R, fmt, m);
  ok(mxfp4_quant(ptr(m), type_of(m, what), R, C, ld_of(m), fmt, ptr(o.q), ptr(o.s), order, ptr(t.q), ptr(t.s), order, 0,
                 cdiv(R, 128), stm(stream)),
     "mxfp4_quant");
  return {o.q, o.s, t.q, t.s};
}

// gate and up [N, K] -> their common operand along K and [K, 2 pad(N, 128)] along N
std::tuple<Tensor, Tensor, Tensor, Tensor> quant_gate_up(const Tensor& wg, const Tensor& wu, int64_t stream) {
  const char* what = "GatedWeight";
  gpu(wg, what);
  same(wg, wu, what);
  need(wg.dim() == 2 && wg.sizes() == wu.sizes() && wg.scalar_type() == wu.scalar_type() && wg.numel() > 0, what,
       "two matrices of one shape and type");
  c10::OptionalDeviceGuard guard(wg.device());
  const int64_t N = wg.size(0), K = wg.size(1), nt = cdiv(N, 128);
  Operand o = operand(2 * pad(N, 32), K, MXFP4_E2M1, wg), t = operand(K, 2 * nt * 128, MXFP4_E2M1, wg);
  for (int i = 0; i < 2; ++i) {
    const Tensor m = rows_of(i ? wu : wg);
    ok(mxfp4_quant(ptr(m), type_of(m, what), N, K, ld_of(m), MXFP4_E2M1, ptr(o.q), ptr(o.s),
                   i ? MXFP4_ROWS_UP : MXFP4_ROWS_GATE, ptr(t.q), ptr(t.s), MXFP4_ROWS_PI, i * nt, 2 * nt, stm(stream)),
       "mxfp4_quant");
  }
  return {o.q, o.s, t.q, t.s};
}

Tensor dequant(const Tensor& q, const Tensor& s, int64_t rows, int64_t cols, int64_t fmt, at::ScalarType dt, int64_t stream) {
  const char* what = "mx4_dequant";
  gpu(q, what);
  c10::OptionalDeviceGuard guard(q.device());
  need(q.numel() >= code_bytes(rows, cols, fmt) && s.numel() >= scale_bytes(rows, cols), what, "operand too small");
  Tensor out = empty({rows, cols}, dt, q);
  ok(mxfp4_dequant(ptr(q), ptr(s), rows, cols, fmt, ptr(out), type_of(out, what), stm(stream)), "mxfp4_dequant");
  return out;
}

Tensor gemm(const Tensor& q, const Tensor& s, int64_t fmt, const Tensor& bq, const Tensor& bs, int64_t order, int64_t M,
            int64_t N, int64_t K, at::ScalarType dt, int64_t stream) {
  const char* what = "mx4_mm";
  gpu(q, what);
  same(q, bq, what);
  c10::OptionalDeviceGuard guard(q.device());
  need(q.numel() >= code_bytes(M, K, fmt) && s.numel() >= scale_bytes(M, K) && bq.numel() >= code_bytes(N, K, MXFP4_E2M1) &&
           bs.numel() >= scale_bytes(N, K),
       what, "operand too small");
  Tensor out = empty({M, N}, dt, q);
  if (M && N && !K) return out.zero_();
  if (M && N)
    ok(mxfp4_gemm(ptr(q), ptr(s), fmt, ptr(bq), ptr(bs), order, M, N, pad(K, 128), ptr(out), N, type_of(out, what),
                  stm(stream)),
       "mxfp4_gemm");
  return out;
}

// x [.., K] with a weight [N, K] in the PI order
Tensor linear(const Tensor& x, const Tensor& wq, const Tensor& ws, int64_t N, int64_t K, int64_t fmt, int64_t stream) {
  const char* what = "mx4_linear";
  gpu(x, what);
  same(x, wq, what);
  const int64_t type = half_type(x, what);
  need(x.dim() >= 1 && x.size(-1) == K, what, "the last dimension is not the weight's input size");
  c10::OptionalDeviceGuard guard(x.device());
  const Tensor m = rows_of(x);
  const int64_t M = m.size(0);
  Tensor y = empty({M, N}, x.scalar_type(), x);
  if (M > MXFP4_FEW_ROWS) {
    Temp a(M, K, fmt, x);
    ok(mxfp4_quant(ptr(m), type, M, K, ld_of(m), fmt, a.q, a.s, MXFP4_ROWS_PLAIN, nullptr, nullptr, 0, 0, 0, stm(stream)),
       "mxfp4_quant");
    ok(mxfp4_gemm(a.q, a.s, fmt, ptr(wq), ptr(ws), MXFP4_ROWS_PI, M, N, pad(K, 128), ptr(y), N, type, stm(stream)),
       "mxfp4_gemm");
  } else if (M) {
    ok(mxfp4_few(ptr(m), ld_of(m), fmt, ptr(wq), ptr(ws), M, N, K, ptr(y), N, type, stm(stream)), "mxfp4_few");
  }
  return shaped(y, x, N);
}

// h [.., N]; with save also what the backward pass needs
std::tuple<Tensor, OptT> gated(const Tensor& x, const Tensor& wq, const Tensor& ws, int64_t N, int64_t K, const OptT& add,
                               int64_t fn, int64_t fmt, bool save, int64_t stream) {
  const char* what = "mx4_gated";
  gpu(x, what);
  same(x, wq, what);
  const int64_t type = half_type(x, what);
  need(x.dim() >= 1 && x.size(-1) == K, what, "the last dimension is not the weight's input size");
  c10::OptionalDeviceGuard guard(x.device());
  const Tensor m = rows_of(x);
  const int64_t M = m.size(0);
  Tensor ad;
  if (add) {
    same(x, *add, what);
    need(add->scalar_type() == x.scalar_type() && add->dim() >= 1 && add->size(-1) == 2 * N, what,
         "the addend has x's type and 2 N columns");
    ad = add->dim() == 1 ? add->unsqueeze(0) : rows_of(*add);
    need(ad.size(0) == M || ad.size(0) == 1, what, "the addend has x's rows, or one");
    if (ad.stride(1) != 1) ad = ad.contiguous();
  }
  const int64_t ld_add = !add || ad.size(0) == 1 ? 0 : ad.stride(0);
  if (add && ld_add != 0 && ld_add < 2 * N) ad = ad.contiguous();
  void* pa = add ? ptr(ad) : nullptr;
  const int64_t la = add && ld_add != 0 ? ad.stride(0) : 0;
  Tensor h = empty({M, N}, x.scalar_type(), x);
  OptT gu;
  if (save) gu = empty({mxfp4_gated_saved_elems(M, N)}, x.scalar_type(), x);
  if (M > MXFP4_FEW_ROWS || (save && M)) {
    Temp a(M, K, fmt, x);
    ok(mxfp4_quant(ptr(m), type, M, K, ld_of(m), fmt, a.q, a.s, MXFP4_ROWS_PLAIN, nullptr, nullptr, 0, 0, 0, stm(stream)),
       "mxfp4_quant");
    ok(mxfp4_gated(a.q, a.s, fmt, ptr(wq), ptr(ws), M, N, pad(K, 128), pa, la, fn, ptr(h), N, ptr(gu), type, stm(stream)),
       "mxfp4_gated");
  } else if (M) {
    ok(mxfp4_few_gated(ptr(m), ld_of(m), fmt, ptr(wq), ptr(ws), M, N, K, pa, la, fn, ptr(h), N, type, stm(stream)),
       "mxfp4_few_gated");
  }
  return {shaped(h, x, N), gu};
}

// dx [M, K] and, if wanted, [dg | du] [M, 2 N], from the saved gu and dh [.., N]
std::tuple<Tensor, OptT> gated_bwd(const Tensor& gu, const Tensor& dh, const Tensor& wtq, const Tensor& wts, int64_t N,
                                   int64_t K, int64_t fn, int64_t fmt, bool want_dx, bool want_dgu, int64_t stream) {
  const char* what = "mx4_gated backward";
  gpu(dh, what);
  c10::OptionalDeviceGuard guard(dh.device());
  const int64_t type = half_type(dh, what);
  Tensor d = rows_of(dh);
  if (d.size(0) > 1 && d.stride(0) < N) d = d.contiguous();  // a broadcast gradient
  const int64_t M = d.size(0), C = 2 * pad(N, 128);
  need(d.size(1) == N && gu.numel() == mxfp4_gated_saved_elems(M, N) && gu.scalar_type() == dh.scalar_type(), what,
       "dh does not belong to the saved pass");
  Tensor dx = empty({want_dx ? M : 0, K}, dh.scalar_type(), dh);
  OptT dgu;
  if (want_dgu) dgu = empty({M, 2 * N}, dh.scalar_type(), dh);
  if (M) {
    Temp a(M, C, fmt, dh);
    ok(mxfp4_gated_bwd(ptr(gu), ptr(d), ld_of(d), M, N, fn, type, fmt, a.q, a.s, ptr(dgu), stm(stream)), "mxfp4_gated_bwd");
    if (want_dx)
      ok(mxfp4_gemm(a.q, a.s, fmt, ptr(wtq), ptr(wts), MXFP4_ROWS_PI, M, K, C, ptr(dx), K, type, stm(stream)), "mxfp4_gemm");
  }
  return {dx, dgu};
}

// loss [T], gradient (or none), workspace of the statistics (kept by the autograd form).  stages as in distill_topk_kl.
std::tuple<OptT, OptT, OptT> topk_kl(const Tensor& z, const Tensor& idx, const Tensor& t, const OptT& weight, double tau,
                                     const OptT& lse, bool want_loss, bool want_grad, const OptT& out, const OptT& ws_in,
                                     int64_t stages, int64_t stream) {
  const char* what = "topk_kl";
  gpu(z, what);
  need(z.dim() == 2 && idx.dim() == 2 && t.dim() == 2 && idx.sizes() == t.sizes() && idx.size(0) == z.size(0), what,
       "logits [T, V] with the teacher's indices and logits [T, k]");
  const int64_t T = z.size(0), V = z.size(1), k = idx.size(1);
  need(V > 0 && k > 0, what, "empty vocabulary or no teacher entries");
  need(z.stride(1) == 1 || V == 1, what, "the logits' columns must be contiguous");
  need(T <= 1 || z.stride(0) >= V || !out, what, "rows of the logits overlap");
  need(idx.scalar_type() == at::kInt || idx.scalar_type() == at::kLong, what, "32- or 64-bit indices");
  same(z, idx, what);
  same(z, t, what);
  c10::OptionalDeviceGuard guard(z.device());
  auto vec = [&](const OptT& v, const char* msg) -> Tensor {
    if (!v) return Tensor();
    same(z, *v, what);
    need(v->dim() == 1 && v->size(0) == T, what, msg);
    return v->to(at::kFloat).contiguous();
  };
  const Tensor w = vec(weight, "one weight a row"), l = vec(lse, "one teacher logsumexp a row");
  const Tensor id = idx.stride(1) == 1 || k == 1 ? idx : idx.contiguous();
  Tensor tt = t.to(at::kFloat);
  if (tt.stride(1) != 1 && k > 1) tt = tt.contiguous();
  OptT loss, grad, ws = ws_in;
  if (want_loss) loss = empty({T}, at::kFloat, z);
  if (want_grad) {
    if (out) {
      same(z, *out, what);
      need(out->dim() == 2 && out->sizes() == z.sizes() && out->scalar_type() == z.scalar_type() &&
               (out->stride(1) == 1 || V == 1) && (T <= 1 || out->stride(0) >= V),
           what, "the gradient's buffer has the logits' shape and type and contiguous columns");
      grad = *out;
    } else {
      grad = empty({T, V}, z.scalar_type(), z);
    }
  }
  // the loss alone reads the logits once and is split the same; statistics that are kept always go through ws
  const int64_t parts = distill_parts(T, V, lse.has_value());
  if (T && !ws && (parts > 1 || stages != 3))
    ws = empty({distill_workspace_size(T, k, parts)}, at::kByte, z);
  if (T)
    ok(distill_topk_kl(ptr(z), type_of(z, what), T <= 1 ? V : z.stride(0), T, V, ptr(id), id.element_size(),
                       T <= 1 ? k : id.stride(0), tt.data_ptr<float>(), T <= 1 ? k : tt.stride(0), k, (float)tau,
                       l.defined() ? l.data_ptr<float>() : nullptr, w.defined() ? w.data_ptr<float>() : nullptr,
                       loss ? loss->data_ptr<float>() : nullptr, ptr(grad), grad ? (T <= 1 ? V : grad->stride(0)) : 0, parts,
                       stages, ptr(ws), stm(stream)),
       "distill_topk_kl");
  return {loss, grad, ws};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  py::register_local_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const NativeError& e) {
      PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, e.what());
    }
  });
  using Free = py::call_guard<py::gil_scoped_release>;
  m.def("set_error", [](py::object e) {
    Py_XINCREF(e.ptr());
    Py_XDECREF(g_error);
    g_error = e.ptr();
  });
  m.def("abi_version", [] { return (int64_t)MXFP4_OPS_ABI_VERSION; });
  m.def("code_bytes", &code_bytes);
  m.def("scale_bytes", &scale_bytes);
  m.def("quant", &quant, Free());
  m.def("quant_both", &quant_both, Free());
  m.def("quant_gate_up", &quant_gate_up, Free());
  m.def("dequant", &dequant, Free());
  m.def("gemm", &gemm, Free());
  m.def("linear", &linear, Free());
  m.def("gated", &gated, Free());
  m.def("gated_bwd", &gated_bwd, Free());
  m.def("topk_kl", &topk_kl, Free());
}
