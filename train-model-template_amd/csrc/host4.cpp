// The host side of the 4-bit operators and of the distillation loss in native code: a call's allocations and launches in
// one step from Python, as host_path.cpp does for the 8-bit path (a single-token product runs for a few microseconds, which
// is what the Python around it would cost by itself; a training step of a thousand tokens runs for 40, half of what the
// Python form of its backward nodes took).  Every function allocates through torch, launches on the current stream of the
// tensors' device through the C-ABI of include/mxfp4_ops.h, does not wait, and runs without the interpreter's lock.
// Shapes, types, strides and devices are checked here; an error raises _native.NativeError.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

#include <memory>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>

#include "../../include/mxfp4_ops.h"
#include "../../include/mxfp8_mlp.h"
#include "mx4_plan.h"

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
// What a call runs under: the tensors' device is current and torch records nothing (the nodes below do it by hand)
struct Scope {
  c10::OptionalDeviceGuard device;
  at::AutoDispatchBelowADInplaceOrView below;
  void* stream;
  explicit Scope(const Tensor& t) : device(t.device()), stream(c10::hip::getCurrentHIPStream(t.get_device()).stream()) {}
};
void* ptr(const Tensor& t) { return t.data_ptr(); }

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

// ------------------------------------------------------------------ quantization and products of MX operands
std::tuple<Tensor, Tensor> quant(const Tensor& x, int64_t fmt, int64_t order) {
  const char* what = "mx4_quant";
  gpu(x, what);
  const Scope sc(x);
  need(x.dim() == 2, what, "a matrix");
  const Tensor m = rows_of(x);
  Operand o = operand(m.size(0), m.size(1), fmt, m);
  ok(mxfp4_quant(ptr(m), type_of(m, what), m.size(0), m.size(1), ld_of(m), fmt, ptr(o.q), ptr(o.s), order, nullptr, nullptr,
                 0, 0, 0, sc.stream),
     "mxfp4_quant");
  return {o.q, o.s};
}

// both axes from one read, each in its row order
std::tuple<Tensor, Tensor, Tensor, Tensor> quant_both(const Tensor& x, int64_t fmt, int64_t order) {
  const char* what = "mx4_quant";
  gpu(x, what);
  const Scope sc(x);
  need(x.dim() == 2, what, "a matrix");
  const Tensor m = rows_of(x);
  const int64_t R = m.size(0), C = m.size(1);
  Operand o = operand(R, C, fmt, m), t = operand(C, R, fmt, m);
  ok(mxfp4_quant(ptr(m), type_of(m, what), R, C, ld_of(m), fmt, ptr(o.q), ptr(o.s), order, ptr(t.q), ptr(t.s), order, 0,
                 cdiv(R, 128), sc.stream),
     "mxfp4_quant");
  return {o.q, o.s, t.q, t.s};
}

Tensor dequant(const Tensor& q, const Tensor& s, int64_t rows, int64_t cols, int64_t fmt, at::ScalarType dt) {
  const char* what = "mx4_dequant";
  gpu(q, what);
  same(q, s, what);
  const Scope sc(q);
  need(q.numel() >= code_bytes(rows, cols, fmt) && s.numel() >= scale_bytes(rows, cols), what, "operand too small");
  Tensor out = empty({rows, cols}, dt, q);
  ok(mxfp4_dequant(ptr(q), ptr(s), rows, cols, fmt, ptr(out), type_of(out, what), sc.stream), "mxfp4_dequant");
  return out;
}

Tensor gemm(const Tensor& q, const Tensor& s, int64_t fmt, const Tensor& bq, const Tensor& bs, int64_t order, int64_t M,
            int64_t N, int64_t K, at::ScalarType dt) {
  const char* what = "mx4_mm";
  gpu(q, what);
  for (const Tensor* t : {&s, &bq, &bs}) same(q, *t, what);
  const Scope sc(q);
  need(q.numel() >= code_bytes(M, K, fmt) && s.numel() >= scale_bytes(M, K) && bq.numel() >= code_bytes(N, K, MXFP4_E2M1) &&
           bs.numel() >= scale_bytes(N, K),
       what, "operand too small");
  Tensor out = empty({M, N}, dt, q);
  if (M && N && !K) return out.zero_();
  if (M && N)
    ok(mxfp4_gemm(ptr(q), ptr(s), fmt, ptr(bq), ptr(bs), order, M, N, pad(K, 128), ptr(out), N, type_of(out, what), sc.stream),
       "mxfp4_gemm");
  return out;
}

// ------------------------------------------------------------------ the frozen weight of a linear layer
struct Weight {
  int64_t N, K;
  Tensor q, s;    // along K, rows in the PI order
  Tensor qt, st;  // of the transpose, along N; undefined without it
};
using WeightP = std::shared_ptr<Weight>;

WeightP make_weight(const Tensor& w, bool transpose) {
  gpu(w, "Weight");
  if (w.dim() != 2 || w.numel() == 0) throw std::invalid_argument("Weight: a matrix with rows and columns");
  auto r = std::make_shared<Weight>();
  r->N = w.size(0);
  r->K = w.size(1);
  if (transpose) std::tie(r->q, r->s, r->qt, r->st) = quant_both(w, MXFP4_E2M1, MXFP4_ROWS_PI);
  else std::tie(r->q, r->s) = quant(w, MXFP4_E2M1, MXFP4_ROWS_PI);
  return r;
}

// MX(x) [.., K] . MX(W)^T from an operand [N, K] in the PI order
Tensor product(const Tensor& x, const Tensor& wq, const Tensor& ws, int64_t N, int64_t K, int64_t fmt) {
  const char* what = "mx4_linear";
  gpu(x, what);
  same(x, wq, what);
  const int64_t type = half_type(x, what);
  need(x.dim() >= 1 && x.size(-1) == K, what, "the last dimension is not the weight's input size");
  const Scope sc(x);
  const Tensor m = rows_of(x);
  const int64_t M = m.size(0);
  Tensor y = empty({M, N}, x.scalar_type(), x);
  if (M > MXFP4_FEW_ROWS) {
    Temp a(M, K, fmt, x);
    ok(mxfp4_quant(ptr(m), type, M, K, ld_of(m), fmt, a.q, a.s, MXFP4_ROWS_PLAIN, nullptr, nullptr, 0, 0, 0, sc.stream),
       "mxfp4_quant");
    ok(mxfp4_gemm(a.q, a.s, fmt, ptr(wq), ptr(ws), MXFP4_ROWS_PI, M, N, pad(K, 128), ptr(y), N, type, sc.stream),
       "mxfp4_gemm");
  } else if (M) {
    ok(mxfp4_few(ptr(m), ld_of(m), fmt, ptr(wq), ptr(ws), M, N, K, ptr(y), N, type, sc.stream), "mxfp4_few");
  }
  return shaped(y, x, N);
}

using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

bool records(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }
// The nodes below know the backward pass alone: the tangent of a dual tensor would be lost
void no_tangent(const Tensor& t, const char* what) {
  need(!t._fw_grad(0).defined(), what, "no forward-mode derivative");
}
void once(const char* what) {
  need(!at::GradMode::is_enabled(), what, "the backward pass has no derivative of its own (create_graph)");
}
template <class T, class... A>
std::shared_ptr<T> make_node(A&&... a) {
  return std::shared_ptr<T>(new T(std::forward<A>(a)...), torch::autograd::deleteNode);
}

// dx = MX(dy) . MX(W^T)^T.  forward false: a product with the transpose, whose own gradient is one with W.
struct LinearNode : Node {
  WeightP w;
  int64_t fmt;
  bool forward;
  LinearNode(WeightP w_, int64_t f, bool fw) : w(std::move(w_)), fmt(f), forward(fw) {}
  std::string name() const override { return "Mx4Linear"; }
  variable_list apply(variable_list&& g) override;
};

Tensor linear(const WeightP& w, const Tensor& x, int64_t fmt, bool forward) {
  no_tangent(x, "mx4_linear");
  if (!records(x))
    return forward ? product(x, w->q, w->s, w->N, w->K, fmt) : product(x, w->qt, w->st, w->K, w->N, fmt);
  if (!w->qt.defined())
    throw std::invalid_argument("mx4_linear: this weight was made without its transpose, it has no input gradient");
  Tensor y = forward ? product(x, w->q, w->s, w->N, w->K, fmt) : product(x, w->qt, w->st, w->K, w->N, fmt);
  auto node = make_node<LinearNode>(w, fmt, forward);
  node->set_next_edges(torch::autograd::collect_next_edges(x));
  torch::autograd::set_history(y, node);
  return y;
}

variable_list LinearNode::apply(variable_list&& g) {
  if (!g[0].defined() || !task_should_compute_output(0)) return {Tensor()};
  return {linear(w, g[0], fmt, !forward)};
}

// ------------------------------------------------------------------ the gated block
struct Gated {
  int64_t N, K;
  Tensor q, s, qt, st;  // GATE and UP rows along K; [K, 2 pad(N, 128)] along N, rows in the PI order
};
using GatedP = std::shared_ptr<Gated>;

GatedP make_gated(const Tensor& wg, const Tensor& wu) {
  const char* what = "GatedWeight";
  gpu(wg, what);
  same(wg, wu, what);
  need(wg.dim() == 2 && wg.sizes() == wu.sizes() && wg.scalar_type() == wu.scalar_type() && wg.numel() > 0, what,
       "two matrices of one shape and type");
  const Scope sc(wg);
  const int64_t N = wg.size(0), K = wg.size(1), nt = cdiv(N, 128);
  Operand o = operand(2 * pad(N, 32), K, MXFP4_E2M1, wg), t = operand(K, 2 * nt * 128, MXFP4_E2M1, wg);
  for (int i = 0; i < 2; ++i) {
    const Tensor m = rows_of(i ? wu : wg);
    ok(mxfp4_quant(ptr(m), type_of(m, what), N, K, ld_of(m), MXFP4_E2M1, ptr(o.q), ptr(o.s),
                   i ? MXFP4_ROWS_UP : MXFP4_ROWS_GATE, ptr(t.q), ptr(t.s), MXFP4_ROWS_PI, i * nt, 2 * nt, sc.stream),
       "mxfp4_quant");
  }
  return std::make_shared<Gated>(Gated{N, K, o.q, o.s, t.q, t.s});
}

// h [.., N] and, with save, what the backward pass needs
std::tuple<Tensor, Tensor> gated_forward(const Gated& w, const Tensor& x, const OptT& add, int64_t fn, int64_t fmt,
                                         bool save) {
  const char* what = "mx4_gated";
  const int64_t type = half_type(x, what), N = w.N, K = w.K;
  const Scope sc(x);
  const Tensor m = rows_of(x);
  const int64_t M = m.size(0);
  Tensor ad;
  int64_t ld_add = 0;
  if (add) {
    ad = rows_of(*add);
    ld_add = M > 1 ? ad.stride(0) : 0;
    if (ld_add && ld_add < 2 * N) {  // overlapping rows
      ad = ad.contiguous();
      ld_add = 2 * N;
    }
  }
  const void* pa = add ? ptr(ad) : nullptr;
  Tensor h = empty({M, N}, x.scalar_type(), x), gu;
  if (save) gu = empty({mxfp4_gated_saved_elems(M, N)}, x.scalar_type(), x);
  if (M > MXFP4_FEW_ROWS || (save && M)) {
    Temp a(M, K, fmt, x);
    ok(mxfp4_quant(ptr(m), type, M, K, ld_of(m), fmt, a.q, a.s, MXFP4_ROWS_PLAIN, nullptr, nullptr, 0, 0, 0, sc.stream),
       "mxfp4_quant");
    ok(mxfp4_gated(a.q, a.s, fmt, ptr(w.q), ptr(w.s), M, N, pad(K, 128), pa, ld_add, fn, ptr(h), N,
                   save ? ptr(gu) : nullptr, type, sc.stream),
       "mxfp4_gated");
  } else if (M) {
    ok(mxfp4_few_gated(ptr(m), ld_of(m), fmt, ptr(w.q), ptr(w.s), M, N, K, pa, ld_add, fn, ptr(h), N, type, sc.stream),
       "mxfp4_few_gated");
  }
  return {shaped(h, x, N), gu};
}

struct GatedNode : Node {
  GatedP w;
  int64_t fn, fmt;
  std::vector<int64_t> lead;  // x's leading dimensions
  SavedVariable gu;
  std::string name() const override { return "Mx4Gated"; }
  void release_variables() override { gu.reset_data(); }
  variable_list apply(variable_list&& g) override {
    const char* what = "mx4_gated";
    const bool want_dx = task_should_compute_output(0), want_add = num_outputs() > 1 && task_should_compute_output(1);
    variable_list out(num_outputs());
    if (!g[0].defined()) return out;
    once(what);
    const Tensor saved = gu.unpack(), &dh = g[0];
    const int64_t N = w->N, K = w->K, C = 2 * pad(N, 128), type = half_type(dh, what);
    const Scope sc(dh);
    Tensor d = rows_of(dh);
    if (d.size(0) > 1 && d.stride(0) < N) d = d.contiguous();  // a broadcast gradient
    const int64_t M = d.size(0);
    Tensor dx, dgu;
    if (want_dx) dx = empty({M, K}, dh.scalar_type(), dh);
    if (want_add) dgu = empty({M, 2 * N}, dh.scalar_type(), dh);
    if (M) {
      Temp a(M, C, fmt, dh);
      ok(mxfp4_gated_bwd(ptr(saved), ptr(d), ld_of(d), M, N, fn, type, fmt, a.q, a.s, want_add ? ptr(dgu) : nullptr,
                         sc.stream),
         "mxfp4_gated_bwd");
      if (want_dx)
        ok(mxfp4_gemm(a.q, a.s, fmt, ptr(w->qt), ptr(w->st), MXFP4_ROWS_PI, M, K, C, ptr(dx), K, type, sc.stream),
           "mxfp4_gemm");
    }
    auto shape = lead;
    shape.push_back(K);
    if (want_dx) out[0] = dx.view(shape);
    shape.back() = 2 * N;
    if (want_add) out[1] = dgu.view(shape);
    return out;
  }
};

Tensor gated(const GatedP& w, const Tensor& x, const OptT& add_, int64_t fn, int64_t fmt) {
  const char* what = "mx4_gated";
  no_tangent(x, what);
  if (add_) no_tangent(*add_, what);
  gpu(x, what);
  same(x, w->q, what);
  half_type(x, what);
  need(x.dim() >= 1 && x.size(-1) == w->K, what, "the last dimension is not the weight's input size");
  auto lead = x.sizes().vec();
  OptT add;
  if (add_) {
    same(x, *add_, what);
    need(add_->scalar_type() == x.scalar_type(), what, "the addend has x's type");
    lead.back() = 2 * w->N;
    // expand is recorded: the gradient of what is broadcast is summed
    add = add_->sizes() == at::IntArrayRef(lead) ? *add_ : add_->expand(lead);
  }
  lead.pop_back();
  if (!records(x) && !(add && records(*add))) return std::get<0>(gated_forward(*w, x, add, fn, fmt, false));
  auto [h, gu] = gated_forward(*w, x, add, fn, fmt, true);
  auto node = make_node<GatedNode>();
  node->w = w;
  node->fn = fn;
  node->fmt = fmt;
  node->lead = lead;
  node->gu = SavedVariable(gu, false);
  if (add) node->set_next_edges(torch::autograd::collect_next_edges(x, *add));
  else node->set_next_edges(torch::autograd::collect_next_edges(x));
  torch::autograd::set_history(h, node);
  return h;
}

// ------------------------------------------------------------------ distillation
struct Kl {  // a checked call
  const Tensor& z;
  Tensor idx, t, lse;
  int64_t T, V, k, parts;
  double tau;
};

Kl kl_call(const Tensor& z, const Tensor& idx, const Tensor& t, double tau, const OptT& lse) {
  const char* what = "topk_kl";
  need(z.dim() == 2 && idx.dim() == 2 && t.dim() == 2 && idx.sizes() == t.sizes() && idx.size(0) == z.size(0), what,
       "logits [T, V] with the teacher's indices and logits [T, k]");
  const int64_t T = z.size(0), V = z.size(1), k = idx.size(1);
  need(V > 0 && k > 0, what, "empty vocabulary or no teacher entries");
  need(z.stride(1) == 1 || V == 1, what, "the logits' columns must be contiguous");
  need(idx.scalar_type() == at::kInt || idx.scalar_type() == at::kLong, what, "32- or 64-bit indices");
  same(z, idx, what);
  same(z, t, what);
  Kl c{z, idx.stride(1) == 1 || k == 1 ? idx : idx.contiguous(), t.to(at::kFloat), Tensor(), T, V, k, 1, tau};
  if (c.t.stride(1) != 1 && k > 1) c.t = c.t.contiguous();
  if (lse) {
    same(z, *lse, what);
    need(lse->dim() == 1 && lse->size(0) == T, what, "one teacher logsumexp a row");
    c.lse = lse->to(at::kFloat).contiguous();
  }
  c.parts = distill_parts(T, V, type_of(z, what));
  return c;
}

void kl_run(const Kl& c, const Tensor& weight, const Tensor& loss, const Tensor& grad, const Tensor& ws, int64_t stages,
            void* stream) {
  if (!c.T) return;
  auto f = [](const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; };
  const bool one = c.T == 1;
  ok(distill_topk_kl(ptr(c.z), type_of(c.z, "topk_kl"), one ? c.V : c.z.stride(0), c.T, c.V, ptr(c.idx),
                     c.idx.element_size(), one ? c.k : c.idx.stride(0), f(c.t), one ? c.k : c.t.stride(0), c.k, (float)c.tau,
                     f(c.lse), f(weight), f(loss), grad.defined() ? ptr(grad) : nullptr,
                     !grad.defined() ? 0 : one ? c.V : grad.stride(0), c.parts, stages, ws.defined() ? ptr(ws) : nullptr,
                     stream),
     "distill_topk_kl");
}
Tensor kl_workspace(const Kl& c) { return empty({distill_workspace_size(c.T, c.k, c.parts)}, at::kByte, c.z); }
Tensor row_weight(const Kl& c, const Tensor& w) {
  same(c.z, w, "topk_kl");
  need(w.dim() == 1 && w.size(0) == c.T, "topk_kl", "one weight a row");
  return w.to(at::kFloat).contiguous();
}

// Two matrices [T, V] with rows of contiguous columns that are the same memory, row by row, or share none
bool apart(const Tensor& a, const Tensor& b, int64_t T, int64_t V) {
  const int64_t es = (int64_t)a.element_size(), row = V * es;  // bytes from here on
  const int64_t la = T == 1 ? row : a.stride(0) * es, lb = T == 1 ? row : b.stride(0) * es;
  const int64_t pa = (int64_t)(uintptr_t)a.data_ptr(), pb = (int64_t)(uintptr_t)b.data_ptr();
  if (!T || (pa == pb && la == lb)) return true;
  if (pa + (T - 1) * la + row <= pb || pb + (T - 1) * lb + row <= pa) return true;
  if (la != lb || la == 0) return false;
  const int64_t d = ((pb - pa) % la + la) % la;  // columns of one buffer's rows beside each other
  return d >= row && d + row <= la;
}

std::tuple<Tensor, Tensor> topk_kl_rows(const Tensor& z, const Tensor& idx, const Tensor& t, const OptT& weight, double tau,
                                        const OptT& lse, const OptT& out) {
  const char* what = "topk_kl_rows";
  no_tangent(z, what);
  gpu(z, what);
  const Scope sc(z);
  const Kl c = kl_call(z, idx, t, tau, lse);
  Tensor w, grad, ws;
  if (weight) w = row_weight(c, *weight);
  if (out) {
    same(z, *out, what);
    need(out->dim() == 2 && out->sizes() == z.sizes() && out->scalar_type() == z.scalar_type() &&
             (out->stride(1) == 1 || c.V == 1) && (c.T <= 1 || out->stride(0) >= c.V),
         what, "the gradient's buffer has the logits' shape and type, contiguous columns and rows that do not overlap");
    need(apart(z, *out, c.T, c.V), what, "the gradient's buffer is the logits' own or does not overlap them");
    out->unsafeGetTensorImpl()->bump_version();  // autograd holds no value of it to be the one it saved
    grad = *out;
  } else {
    grad = empty({c.T, c.V}, z.scalar_type(), z);
  }
  Tensor loss = empty({c.T}, at::kFloat, z);
  if (c.parts > 1) ws = kl_workspace(c);
  kl_run(c, w, loss, grad, ws, DISTILL_STATS | DISTILL_FINISH, sc.stream);
  return {loss, grad};
}

struct KlNode : Node {
  SavedVariable z, idx, t, lse, ws;
  bool has_lse;
  double tau;
  std::string name() const override { return "TopkKl"; }
  void release_variables() override {
    for (SavedVariable* v : {&z, &idx, &t, &lse, &ws}) v->reset_data();
  }
  variable_list apply(variable_list&& g) override {
    if (!g[0].defined() || !task_should_compute_output(0)) return {Tensor()};
    once("topk_kl");
    const Tensor zz = z.unpack(), ii = idx.unpack(), tt = t.unpack(), w0 = ws.unpack();
    const OptT ll = has_lse ? OptT(lse.unpack()) : OptT();
    const Scope sc(zz);
    const Kl c = kl_call(zz, ii, tt, tau, ll);
    Tensor grad = empty({c.T, c.V}, zz.scalar_type(), zz);
    kl_run(c, row_weight(c, g[0]), Tensor(), grad, w0, DISTILL_FINISH, sc.stream);
    return {grad};
  }
};

Tensor topk_kl(const Tensor& z, const Tensor& idx, const Tensor& t, double tau, const OptT& lse) {
  no_tangent(z, "topk_kl");
  gpu(z, "topk_kl");
  const bool rec = records(z);
  Tensor loss, ws;
  {
    const Scope sc(z);
    const Kl c = kl_call(z, idx, t, tau, lse);
    loss = empty({c.T}, at::kFloat, z);
    if (c.parts > 1 || rec) ws = kl_workspace(c);
    if (rec) {  // the statistics are kept
      kl_run(c, Tensor(), Tensor(), Tensor(), ws, DISTILL_STATS, sc.stream);
      kl_run(c, Tensor(), loss, Tensor(), ws, DISTILL_FINISH, sc.stream);
    } else {
      kl_run(c, Tensor(), loss, Tensor(), ws, DISTILL_STATS | DISTILL_FINISH, sc.stream);
    }
  }
  if (!rec) return loss;
  auto node = make_node<KlNode>();
  node->z = SavedVariable(z, false);
  node->idx = SavedVariable(idx, false);
  node->t = SavedVariable(t.detach(), false);
  if (lse) node->lse = SavedVariable(lse->detach(), false);
  node->ws = SavedVariable(ws, false);
  node->has_lse = lse.has_value();
  node->tau = tau;
  node->set_next_edges(torch::autograd::collect_next_edges(z));
  torch::autograd::set_history(loss, node);
  return loss;
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
  m.def("shape", [](int64_t M, int64_t rows, int64_t K, bool e4m3, bool gated, bool thin, int64_t cus) {
    need(M > 0 && rows > 0 && K > 0 && cus > 0 && std::max({M, rows, K, cus}) < (1 << 30), "mx4_shape", "bad size");
    static const char* const names[] = {"256x128", "128x128", "64x128", "64x64", "thin"};
    return std::string(names[mx4_shape(M, rows, (K + 127) / 128, e4m3, gated, thin, (int)cus)]);
  });
  py::class_<Weight, WeightP>(m, "Weight")
      .def(py::init(&make_weight), Free())
      .def_readonly("N", &Weight::N)
      .def_readonly("K", &Weight::K)
      .def_property_readonly("nbytes", [](const Weight& w) {
        return w.q.nbytes() + w.s.nbytes() + (w.qt.defined() ? w.qt.nbytes() + w.st.nbytes() : 0);
      });
  py::class_<Gated, GatedP>(m, "Gated")
      .def(py::init(&make_gated), Free())
      .def_readonly("N", &Gated::N)
      .def_readonly("K", &Gated::K)
      .def_property_readonly("nbytes", [](const Gated& w) {
        return w.q.nbytes() + w.s.nbytes() + w.qt.nbytes() + w.st.nbytes();
      });
  m.def("quant", &quant, Free());
  m.def("quant_both", &quant_both, Free());
  m.def("dequant", &dequant, Free());
  m.def("gemm", &gemm, Free());
  m.def("linear", [](const WeightP& w, const Tensor& x, int64_t fmt) { return linear(w, x, fmt, true); }, Free());
  m.def("gated", &gated, Free());
  m.def("topk_kl_rows", &topk_kl_rows, Free());
  m.def("topk_kl", &topk_kl, Free());
}
