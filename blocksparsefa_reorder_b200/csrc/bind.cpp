// The host side of the operators that are called once a token: argument checks,
// output and workspace allocation and the C ABI call (include/bsattn_b200.h) in
// one native step, and their autograd nodes.  From Python (ctypes) the same
// steps took 22 to 30 us a call and 165 to 190 us a training step, several times
// the kernels; from here 9 to 12 us, and 97 us with PyTorch's own engine (80 us).
//
// Wrong types raise TypeError, wrong values ValueError, a refusal by the C ABI
// BsaError, as in the package's other entry points.
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/engine.h>
#include <torch/extension.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <limits>
#include <unordered_set>
#include <vector>

#include "../../include/bsattn_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A non-zero bsa_status, raised as the package's BsaError.
struct AbiError : std::runtime_error {
  AbiError(int s, const char* w) : std::runtime_error(std::string(w) + ": " + bsa_status_string(s)), status(s), what_(w) {}
  int status;
  std::string what_;
};

void check(int status, const char* what) {
  if (status != BSA_OK) throw AbiError(status, what);
}

int dtype_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return BSA_DTYPE_F32;
    case at::kHalf: return BSA_DTYPE_F16;
    case at::kBFloat16: return BSA_DTYPE_BF16;
    default: return -1;
  }
}

void require_cuda(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor (this library has no CPU path)");
}

void same_device(const Tensor& t, const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " is on another device");
}

int index_dtype(const Tensor& t, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " must be int32 or int64, got ",
                   t.scalar_type());
  return t.scalar_type() == at::kLong ? BSA_INDEX_I64 : BSA_INDEX_I32;
}

// A [B, H, N, D] (or [H, N, D]: no batch) view with contiguous rows.
bsa_tensor4d t4(const Tensor& t, const char* name) {
  const auto s = t.strides();
  const int d = static_cast<int>(s.size());
  TORCH_CHECK_VALUE(s[d - 1] == 1 || t.size(d - 1) <= 1, "the last (head) dimension of ", name, " must be contiguous");
  return {t.data_ptr(), d == 4 ? s[0] : 0, s[d - 3], s[d - 2]};
}

// Heads or tokens expanded from one (stride 0) get memory of their own: the TMA
// descriptors need real strides there.  An expanded batch of keys is kept.
Tensor spread(const Tensor& t, bool batch_too = false) {
  const int d = static_cast<int>(t.dim());
  for (int i = batch_too ? 0 : d - 3; i < d - 1; ++i)
    if (t.stride(i) == 0 && t.size(i) > 1) return t.contiguous();
  return t;
}

// An output gradient as the kernels read it (autograd hands out expanded and
// transposed ones).
Tensor rows(const Tensor& g) {
  const int64_t e = g.element_size();
  bool ok = g.stride(3) == 1 && reinterpret_cast<uintptr_t>(g.data_ptr()) % 16 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && g.stride(i) * e % 16 == 0 && (g.stride(i) != 0 || g.size(i) <= 1);
  return ok ? g : g.contiguous();
}

Tensor contiguous_like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }

// Memory of a strided tensor: runs of `run` bytes from `base` on, repeated over
// n dimensions (strides in bytes, ascending).
struct Extent {
  explicit Extent(const Tensor& t)
      : base(reinterpret_cast<intptr_t>(t.data_ptr())), run(static_cast<int64_t>(t.element_size())) {
    for (int64_t i = 0; i < t.dim() && n < kDims; ++i)
      if (t.size(i) > 1) dims[n++] = {t.stride(i) * static_cast<int64_t>(t.element_size()), t.size(i)};
    std::sort(dims.begin(), dims.begin() + n);
    int inner = 0;
    while (inner < n && dims[inner].first == run) run *= dims[inner++].second;
    std::copy(dims.begin() + inner, dims.begin() + n, dims.begin());
    n -= inner;
  }
  static constexpr int kDims = 5;
  intptr_t base;
  int64_t run;
  int n = 0;
  std::array<std::pair<int64_t, int64_t>, kDims> dims;  // stride, size
};

// Whether a sum at + sum d_i s_i, each d_i within its range, lies between -below
// and above (exclusive): largest stride first, so that what the smaller ones can
// still reach leaves a candidate or two for each d_i where the strides nest.
struct StridedSum {
  struct Term {
    int64_t s, lo, hi;
  };
  std::array<Term, 2 * Extent::kDims> terms;
  int n = 0;
  int64_t below, above;
  bool moved_only = false;  // not with every d_i zero
  int visits = 1 << 16;     // (more of them: taken as met)
  std::array<int64_t, 2 * Extent::kDims + 1> least, most;  // of the terms from i on

  void add(int64_t s, int64_t lo, int64_t hi) {
    for (int i = 0; i < n; ++i)
      if (terms[i].s == s) {
        terms[i].lo += lo, terms[i].hi += hi;
        return;
      }
    terms[n++] = {s, lo, hi};
  }
  bool hits(int64_t at) {
    std::sort(terms.begin(), terms.begin() + n, [](const Term& a, const Term& b) { return a.s > b.s; });
    least[n] = most[n] = 0;
    for (int i = n - 1; i >= 0; --i)
      least[i] = least[i + 1] + terms[i].s * terms[i].lo, most[i] = most[i + 1] + terms[i].s * terms[i].hi;
    return from(0, at, false);
  }
  bool from(int i, int64_t at, bool moved) {
    if (at + least[i] >= above || at + most[i] <= -below) return false;
    if (--visits < 0) return true;
    if (i == n) return moved || !moved_only;
    const Term& t = terms[i];
    if (t.s == 0) return from(i + 1, at, moved || t.hi > t.lo);
    // (the first candidate may miss by the division's rounding, which the test above sees)
    const int64_t lo = std::max(t.lo, (-below - at - most[i + 1]) / t.s - 1);
    const int64_t hi = std::min(t.hi, (above - at - least[i + 1]) / t.s + 1);
    for (int64_t d = lo; d <= hi; ++d)
      if (from(i + 1, at + d * t.s, moved || d != 0)) return true;
    return false;
  }
};

// The end of a tensor's memory.
intptr_t end_of(const Tensor& t) {
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += t.stride(i) * (t.size(i) - 1);
  return reinterpret_cast<intptr_t>(t.data_ptr()) + (last + 1) * static_cast<int64_t>(t.element_size());
}

// Whether two elements of a tensor share memory.
bool rows_overlap(const Tensor& t) {
  if (!t.numel()) return false;
  const Extent x(t);
  int64_t reach = x.run;
  bool nested = true;
  for (int i = 0; i < x.n; ++i) {
    if (i && x.dims[i].first == x.dims[i - 1].first) return true;  // (1, 0) and (0, 1) are one place
    nested = nested && x.dims[i].first >= reach;
    reach += x.dims[i].first * (x.dims[i].second - 1);
  }
  if (nested) return false;
  StridedSum sum;
  sum.below = sum.above = x.run;
  sum.moved_only = true;
  for (int i = 0; i < x.n; ++i) sum.add(x.dims[i].first, 1 - x.dims[i].second, x.dims[i].second - 1);
  return sum.hits(0);
}

enum class Overlap { kNone, kSame, kSome };

// What memory two tensors share (kSame: element for element).  PyTorch's own test
// does not answer for views that are not dense, as those of a fused projection or
// of a key cache are.
Overlap overlap_of(const Tensor& a, const Tensor& b) {
  if (!a.numel() || !b.numel() || a.device() != b.device()) return Overlap::kNone;
  if (end_of(a) <= reinterpret_cast<intptr_t>(b.data_ptr()) || end_of(b) <= reinterpret_cast<intptr_t>(a.data_ptr()))
    return Overlap::kNone;
  const Extent x(a), y(b);
  bool same = x.base == y.base && a.scalar_type() == b.scalar_type() && a.sizes() == b.sizes();
  for (int64_t i = 0; same && i < a.dim(); ++i) same = a.size(i) == 1 || a.stride(i) == b.stride(i);
  if (same) return Overlap::kSame;
  StridedSum sum;
  sum.below = x.run, sum.above = y.run;
  for (int i = 0; i < x.n; ++i) sum.add(x.dims[i].first, 0, x.dims[i].second - 1);
  for (int i = 0; i < y.n; ++i) sum.add(y.dims[i].first, 1 - y.dims[i].second, 0);
  return sum.hits(x.base - y.base) ? Overlap::kSome : Overlap::kNone;
}

// A tensor of the caller's that the call writes: as in PyTorch's own out=
// arguments its rows lie apart, and autograd learns that it changed.
void written(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(!rows_overlap(t), name, " must not be expanded or overlap itself: every row is written");
  TORCH_CHECK_VALUE(!(t.requires_grad() && at::GradMode::is_enabled()), name,
                    " requires a gradient: writing it is not differentiable");
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

Tensor output(const OptTensor& out, const Tensor& x, const char* name) {
  if (!out) return contiguous_like(x);
  TORCH_CHECK_VALUE(out->sizes() == x.sizes() && out->scalar_type() == x.scalar_type() && out->device() == x.device(), name,
                    " has the wrong shape, dtype or device");
  written(*out, name);
  return *out;
}

// Refuses an output over other memory of the call, which blocks still read (or
// write) when others write it; `same`: it may be that very tensor.
void apart(const Tensor& out, const Tensor& x, const char* name, const char* other, bool same = false) {
  const Overlap o = overlap_of(out, x);
  TORCH_CHECK_VALUE(o == Overlap::kNone || (same && o == Overlap::kSame), name, " overlaps ", other);
}
void apart(const OptTensor& out, const OptTensor& x, const char* name, const char* other, bool same = false) {
  if (out && x) apart(*out, *x, name, other, same);
}

void* ptr(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }
int32_t* flag(const OptTensor& t) { return t ? t->data_ptr<int32_t>() : nullptr; }
int dim(int64_t n, const char* what) {
  TORCH_CHECK_VALUE(n <= std::numeric_limits<int32_t>::max(), what, " is too large: ", n);
  return static_cast<int>(n);
}
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// ---------------------------------------------------------------------------
// Norm and rotation
// ---------------------------------------------------------------------------
struct RopeIn {
  OptTensor q, k, q_weight, k_weight, positions, cos, sin;
  double eps;
  bool interleaved;
};

void rope_weight(const Tensor& w, const Tensor& x, const char* name) {
  require_cuda(w, name);
  TORCH_CHECK_VALUE(w.dim() == 1 && w.size(0) == x.size(3) && w.is_contiguous(), name, " must be a contiguous [", x.size(3),
                    "] tensor, got ", w.sizes());
  TORCH_CHECK_TYPE(w.scalar_type() == at::kFloat || w.scalar_type() == x.scalar_type(), name, " must be float32 or ",
                   x.scalar_type(), ", got ", w.scalar_type());
  same_device(w, x, name);
}

// Checks, and the C arguments but for the outputs.
bsa_rope_args rope_args(const RopeIn& in) {
  TORCH_CHECK_VALUE(in.q || in.k, "pass q or k");
  const Tensor& x = in.q ? *in.q : *in.k;
  const OptTensor* sides[] = {&in.q, &in.k};
  const char* names[] = {"q", "k"};
  for (int i = 0; i < 2; ++i) {
    if (!*sides[i]) continue;
    const Tensor& t = **sides[i];
    require_cuda(t, names[i]);
    TORCH_CHECK_VALUE(t.dim() == 4, names[i], " must be [B, H, N, D], got ", t.sizes());
    TORCH_CHECK_TYPE(dtype_of(t.scalar_type()) >= 0, names[i], " must be float32, float16 or bfloat16, got ",
                     t.scalar_type());
  }
  if (in.q && in.k) {
    const Tensor& k = *in.k;
    TORCH_CHECK_VALUE(k.size(0) == x.size(0) && k.size(2) == x.size(2) && k.size(3) == x.size(3),
                      "q and k must share B, N and D, got ", x.sizes(), " and ", k.sizes());
    TORCH_CHECK_TYPE(k.scalar_type() == x.scalar_type(), "q and k must share a dtype, got ", x.scalar_type(), " and ",
                     k.scalar_type());
    TORCH_CHECK_VALUE(k.device() == x.device(), "q and k must be on one device");
  }
  bsa_rope_args a{};
  a.B = dim(x.size(0), "B"), a.N = dim(x.size(2), "N"), a.D = dim(x.size(3), "D");
  a.H = in.q ? dim(in.q->size(1), "H") : 0;
  a.Hk = in.k ? dim(in.k->size(1), "Hk") : 0;
  a.dtype = a.weight_dtype = dtype_of(x.scalar_type());
  if (in.q) {
    a.q = t4(*in.q, "q");
    if (in.q_weight) rope_weight(*in.q_weight, *in.q, "q_weight"), a.q_weight = in.q_weight->data_ptr();
  }
  if (in.k) {
    a.k = t4(*in.k, "k");
    if (in.k_weight) rope_weight(*in.k_weight, *in.k, "k_weight"), a.k_weight = in.k_weight->data_ptr();
  }
  if (a.q_weight && a.k_weight)
    TORCH_CHECK_TYPE(in.q_weight->scalar_type() == in.k_weight->scalar_type(), "q_weight and k_weight must share a dtype");
  if (a.q_weight || a.k_weight) a.weight_dtype = dtype_of((a.q_weight ? in.q_weight : in.k_weight)->scalar_type());
  TORCH_CHECK_VALUE(in.eps >= 0 && std::isfinite(in.eps), "eps must be finite and not negative");
  a.eps = static_cast<float>(in.eps);
  a.interleaved = in.interleaved;
  TORCH_CHECK_VALUE(in.cos.has_value() == in.sin.has_value(), "pass both cos and sin, or neither (norm only)");
  if (!in.cos) {
    TORCH_CHECK_VALUE(!in.positions, "positions need the cos and sin tables");
    return a;
  }
  const Tensor &c = *in.cos, &s = *in.sin;
  for (int i = 0; i < 2; ++i) {
    const Tensor& t = i ? s : c;
    const char* name = i ? "sin" : "cos";
    require_cuda(t, name);
    TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat && t.dim() == 2, name, " must be a float32 [length, R / 2] table");
    same_device(t, x, name);
  }
  TORCH_CHECK_VALUE(c.sizes() == s.sizes() && c.strides() == s.strides() && (c.stride(1) == 1 || c.size(1) <= 1),
                    "cos and sin must share their shape and strides, with contiguous rows");
  TORCH_CHECK_VALUE(c.numel() > 0, "cos and sin must not be empty (pass None for the norm alone)");
  a.R = dim(2 * c.size(1), "R");
  a.cos = c.data_ptr<float>(), a.sin = s.data_ptr<float>();
  a.table_len = dim(c.size(0), "the tables' length");
  // (an expanded row would be read as rows of its own, past its memory)
  TORCH_CHECK_VALUE(c.size(0) == 1 || c.stride(0) >= c.size(1), "the tables' rows must not overlap");
  a.table_stride = c.size(0) == 1 ? c.size(1) : c.stride(0);
  if (in.positions) {
    const Tensor& p = *in.positions;
    require_cuda(p, "positions");
    a.pos_dtype = index_dtype(p, "positions");
    same_device(p, x, "positions");
    const bool one = p.dim() == 1 && p.size(0) == a.N;
    TORCH_CHECK_VALUE((one || (p.dim() == 2 && p.size(0) == a.B && p.size(1) == a.N)) && (a.N <= 1 || p.stride(-1) == 1),
                      "positions must be [", a.N, "] or [", a.B, ", ", a.N, "] with contiguous rows, got ", p.sizes());
    a.positions = p.data_ptr();
    a.pos_stride_b = one ? 0 : p.stride(0);
  }
  return a;
}

bool rope_empty(const bsa_rope_args& a) { return a.B == 0 || a.N == 0 || a.H + a.Hk == 0; }

std::tuple<OptTensor, OptTensor> rope_forward(const RopeIn& in, const OptTensor& q_out, const OptTensor& k_out,
                                              const OptTensor& err) {
  bsa_rope_args a = rope_args(in);
  OptTensor oq, ok;
  const OptTensor* outs[] = {&q_out, &k_out};
  const char* names[] = {"q_out", "k_out"};
  for (int i = 0; i < 2; ++i) {
    if (!*outs[i]) continue;
    apart(*outs[i], in.q, names[i], "q", i == 0);
    apart(*outs[i], in.k, names[i], "k", i == 1);
    apart(*outs[i], in.q_weight, names[i], "q_weight");
    apart(*outs[i], in.k_weight, names[i], "k_weight");
    apart(*outs[i], in.positions, names[i], "positions");
    apart(*outs[i], in.cos, names[i], "cos");
    apart(*outs[i], in.sin, names[i], "sin");
  }
  apart(q_out, k_out, "q_out", "k_out");
  if (in.q) oq = output(q_out, *in.q, "q_out"), a.q_out = t4(*oq, "q_out");
  if (in.k) ok = output(k_out, *in.k, "k_out"), a.k_out = t4(*ok, "k_out");
  if (rope_empty(a)) return {oq, ok};
  const Tensor& x = in.q ? *in.q : *in.k;
  a.err_flag = flag(err);
  const c10::cuda::CUDAGuard guard(x.device());
  check(bsa_qk_norm_rope(&a, stream_of(x)), "bsa_qk_norm_rope");
  return {oq, ok};
}

std::tuple<OptTensor, OptTensor, OptTensor, OptTensor> rope_backward(const RopeIn& in, const OptTensor& dq_out,
                                                                     const OptTensor& dk_out, const OptTensor& err) {
  bsa_rope_args a = rope_args(in);
  OptTensor dx[2], dw[2];
  for (int i = 0; i < 2; ++i) {
    const OptTensor &t = i ? in.k : in.q, &g = i ? dk_out : dq_out, &w = i ? in.k_weight : in.q_weight;
    if (!t) continue;
    const char* name = i ? "dk_out" : "dq_out";
    TORCH_CHECK_VALUE(g.has_value(), name, " is missing");
    require_cuda(*g, name);
    TORCH_CHECK_VALUE(g->sizes() == t->sizes() && g->scalar_type() == t->scalar_type() && g->device() == t->device(), name,
                      " must have its input's shape, dtype and device");
    dx[i] = contiguous_like(*t);
    (i ? a.k_out : a.q_out) = t4(*dx[i], "dx");
    (i ? a.dk_out : a.dq_out) = t4(*g, name);
    if (w) {
      dw[i] = at::empty(w->sizes(), w->options());
      (i ? a.dk_weight : a.dq_weight) = dw[i]->data_ptr();
    }
  }
  if (rope_empty(a)) {
    for (auto& w : dw)
      if (w) w->zero_();
    return {dx[0], dx[1], dw[0], dw[1]};
  }
  const Tensor& x = in.q ? *in.q : *in.k;
  a.err_flag = flag(err);
  const c10::cuda::CUDAGuard guard(x.device());
  size_t n = 0;
  check(bsa_qk_norm_rope_bwd_workspace_bytes(&a, &n), "bsa_qk_norm_rope_bwd_workspace_bytes");
  Tensor ws;
  if (n) ws = at::empty({static_cast<int64_t>(n)}, x.options().dtype(at::kByte));
  check(bsa_qk_norm_rope_bwd(&a, n ? ws.data_ptr() : nullptr, n, stream_of(x)), "bsa_qk_norm_rope_bwd");
  return {dx[0], dx[1], dw[0], dw[1]};
}

Tensor or_none(const OptTensor& t) { return t ? *t : Tensor(); }
OptTensor if_defined(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

void once(const char* name) {
  TORCH_CHECK(!at::GradMode::is_enabled(), name, " is differentiable once: its gradient has none (create_graph)");
}

// A captured backward pass that reaches a node made on the default stream: a
// leaf's, which an eager graph, still alive, holds, or one of an eager graph
// behind this operator's inputs.  That stream cannot join the capture, which the
// engine's attempt invalidates (the process may end with it).  Refused here,
// before it gets there, through whatever lies between (views of a fused
// projection, casts).
void capturable_graph() {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  const auto self = torch::autograd::get_current_node();
  const auto* info = torch::autograd::get_current_graph_task_exec_info();
  if (!self) return;
  std::unordered_set<torch::autograd::Node*> seen;
  std::vector<torch::autograd::Node*> open{self.get()};
  while (!open.empty()) {
    auto* node = open.back();
    open.pop_back();
    for (const auto& edge : node->next_edges()) {
      auto* next = edge.function.get();
      if (!next || !seen.insert(next).second) continue;
      if (info && !info->empty()) {
        const auto it = info->find(next);
        if (it == info->end() || !it->second.should_execute()) continue;
      }
      const auto s = next->stream();
      TORCH_CHECK(!s || *s != c10::cuda::getDefaultCUDAStream(s->device_index()).unwrap(),
                  "a captured backward pass cannot reach a leaf (or another node) that an eager graph on the default "
                  "stream still holds: free that graph first, or run it on the capture's stream");
      open.push_back(next);
    }
  }
}

// Outputs and incoming gradients: those of q and k that are there, in that order.
struct RopeFn : torch::autograd::Function<RopeFn> {
  static variable_list forward(AutogradContext* ctx, const OptTensor& q, const OptTensor& k, const OptTensor& q_weight,
                               const OptTensor& k_weight, const OptTensor& positions, const OptTensor& cos,
                               const OptTensor& sin, double eps, bool interleaved) {
    auto [oq, ok] = rope_forward({q, k, q_weight, k_weight, positions, cos, sin, eps, interleaved}, {}, {}, {});
    ctx->save_for_backward({or_none(q), or_none(k), or_none(q_weight), or_none(k_weight), or_none(positions), or_none(cos),
                            or_none(sin)});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->set_materialize_grads(false);
    variable_list out;
    if (oq) out.push_back(*oq);
    if (ok) out.push_back(*ok);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    once("qk_norm_rope");
    capturable_graph();
    const auto s = ctx->get_saved_variables();
    // a side that is absent, or whose output took no part, has no gradient
    const Tensor gq = s[0].defined() ? g[0] : Tensor(), gk = s[1].defined() ? g[s[0].defined() ? 1 : 0] : Tensor();
    const bool hq = gq.defined(), hk = gk.defined();
    variable_list out(9);
    if (!hq && !hk) return out;
    RopeIn in{hq ? if_defined(s[0]) : OptTensor(), hk ? if_defined(s[1]) : OptTensor(),
              hq ? if_defined(s[2]) : OptTensor(), hk ? if_defined(s[3]) : OptTensor(), if_defined(s[4]),
              if_defined(s[5]), if_defined(s[6]), ctx->saved_data["eps"].toDouble(),
              ctx->saved_data["interleaved"].toBool()};
    auto [dq, dk, dwq, dwk] =
        rope_backward(in, hq ? OptTensor(rows(gq)) : OptTensor(), hk ? OptTensor(rows(gk)) : OptTensor(), {});
    out[0] = or_none(dq), out[1] = or_none(dk), out[2] = or_none(dwq), out[3] = or_none(dwk);
    return out;
  }
};

std::tuple<OptTensor, OptTensor> rope_autograd(const RopeIn& in) {
  TORCH_CHECK_VALUE(in.q || in.k, "pass q or k");
  const auto o = RopeFn::apply(in.q, in.k, in.q_weight, in.k_weight, in.positions, in.cos, in.sin, in.eps, in.interleaved);
  return {in.q ? OptTensor(o[0]) : OptTensor(), in.k ? OptTensor(o[in.q ? 1 : 0]) : OptTensor()};
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------
void half_type(const Tensor& q) {
  require_cuda(q, "q");
  TORCH_CHECK_TYPE(q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16, "q must be float16 or bfloat16, got ",
                   q.scalar_type());
}

void like_q(const Tensor& t, const Tensor& q, const char* name) {
  require_cuda(t, name);
  TORCH_CHECK_TYPE(t.scalar_type() == q.scalar_type(), name, " must have q's dtype ", q.scalar_type(), ", got ",
                   t.scalar_type());
  same_device(t, q, name);
}

int lens_dtype(const OptTensor& lens, const Tensor& q, const char* name) {
  if (!lens) return BSA_INDEX_I32;
  require_cuda(*lens, name);
  const int d = index_dtype(*lens, name);
  TORCH_CHECK_VALUE(lens->dim() == 1 && lens->size(0) == q.size(0) && lens->is_contiguous(), name,
                    " must be a contiguous [", q.size(0), "] tensor, got ", lens->sizes());
  same_device(*lens, q, name);
  return d;
}

float scale_of(const std::optional<double>& scale, int64_t D) {
  const double s = scale ? *scale : 1.0 / std::sqrt(static_cast<double>(D));
  TORCH_CHECK_VALUE(s > 0 && static_cast<float>(s) > 0 && std::isfinite(static_cast<float>(s)),
                    "sm_scale must be positive and finite");
  return static_cast<float>(s);
}

OptTensor lse_output(bool want, const OptTensor& out, const Tensor& q) {
  if (out) {
    TORCH_CHECK_VALUE(out->sizes() == q.sizes().slice(0, 3) && out->scalar_type() == at::kFloat && out->is_contiguous() &&
                          out->device() == q.device(),
                      "lse_out must be a contiguous float32 [B, H, tokens] tensor on q's device");
    written(*out, "lse_out");
    return out;
  }
  return want ? OptTensor(at::empty(q.sizes().slice(0, 3), q.options().dtype(at::kFloat))) : OptTensor();
}

// The caller's outputs lie apart from each other and from what the call reads.
void attention_outputs(const OptTensor& out, const OptTensor& lse_out, const OptTensor& o_rest,
                       std::initializer_list<std::pair<const Tensor&, const char*>> inputs, const OptTensor& lens,
                       const char* lens_name) {
  const std::pair<const OptTensor&, const char*> outs[] = {{out, "out"}, {lse_out, "lse_out"}, {o_rest, "o_rest"}};
  for (int i = 0; i < 3; ++i) {
    if (!outs[i].first) continue;
    for (const auto& x : inputs) apart(*outs[i].first, x.first, outs[i].second, x.second);
    apart(outs[i].first, lens, outs[i].second, lens_name);
    for (int j = 0; j < i; ++j) apart(outs[i].first, outs[j].first, outs[i].second, outs[j].second);
  }
}

template <typename Args>
void launch(const Args& a, int (*query)(const Args*, size_t*), int (*call)(const Args*, void*, size_t, void*),
            const Tensor& q, const char* name) {
  const c10::cuda::CUDAGuard guard(q.device());
  size_t n = 0;
  check(query(&a, &n), name);
  Tensor ws;
  if (n) ws = at::empty({static_cast<int64_t>(n)}, q.options().dtype(at::kByte));
  check(call(&a, n ? ws.data_ptr() : nullptr, n, stream_of(q)), name);
}

// The checks that forward and backward of cross attention share.
void cross_shapes(const Tensor& q, const Tensor& k, const Tensor& v) {
  half_type(q);
  TORCH_CHECK_VALUE(q.dim() == 4, "q must be [B, H, M, D], got ", q.sizes());
  like_q(k, q, "k");
  like_q(v, q, "v");
  TORCH_CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes() && k.size(0) == q.size(0) && k.size(3) == q.size(3),
                    "k and v must be [", q.size(0), ", Hk, N, ", q.size(3), "], got ", k.sizes(), " and ", v.sizes());
  TORCH_CHECK_VALUE(k.size(1) > 0 && q.size(1) % k.size(1) == 0, "the query heads (", q.size(1),
                    ") must be a multiple of the key / value heads (", k.size(1), ")");
}

std::tuple<Tensor, OptTensor> cross_forward(const Tensor& q_, const Tensor& k_, const Tensor& v_, const OptTensor& k_lens,
                                            const std::optional<double>& sm_scale, bool return_lse, const OptTensor& out,
                                            const OptTensor& lse_out, const OptTensor& o_rest, const OptTensor& err) {
  cross_shapes(q_, k_, v_);
  bsa_cross_args a{};
  a.lens_dtype = lens_dtype(k_lens, q_, "k_lens");
  a.sm_scale = scale_of(sm_scale, q_.size(3));
  attention_outputs(out, lse_out, o_rest, {{q_, "q"}, {k_, "k"}, {v_, "v"}}, k_lens, "k_lens");
  const Tensor o = output(out, q_, "out");
  const OptTensor lse = lse_output(return_lse, lse_out, q_);
  if (o_rest) {
    output(o_rest, q_, "o_rest");
    TORCH_CHECK_VALUE(o_rest->strides() == o.strides(), "o_rest must be laid out as the output");
    a.o_rest = o_rest->data_ptr();
  }
  if (q_.numel() == 0) return {o, lse};
  const Tensor q = spread(q_, true), k = spread(k_), v = spread(v_);
  a.B = dim(q.size(0), "B"), a.H = dim(q.size(1), "H"), a.Hk = dim(k.size(1), "Hk"), a.M = dim(q.size(2), "M");
  a.N = dim(k.size(2), "N"), a.D = dim(q.size(3), "D"), a.dtype = dtype_of(q.scalar_type());
  a.q = t4(q, "q"), a.o = t4(o, "out"), a.k = t4(k, "k"), a.v = t4(v, "v");
  a.k_lens = ptr(k_lens);
  a.lse = static_cast<float*>(ptr(lse));
  a.err_flag = flag(err);
  launch(a, bsa_cross_fwd_workspace_bytes, bsa_cross_fwd, q, "bsa_cross_fwd");
  return {o, lse};
}

std::tuple<Tensor, Tensor, Tensor> cross_backward(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& o_,
                                                  const Tensor& lse, const Tensor& dout_, const OptTensor& k_lens,
                                                  const std::optional<double>& sm_scale, const OptTensor& o_rest,
                                                  const OptTensor& err) {
  cross_shapes(q_, k_, v_);
  like_q(o_, q_, "o");
  like_q(dout_, q_, "dout");
  TORCH_CHECK_VALUE(o_.sizes() == q_.sizes() && dout_.sizes() == q_.sizes(), "o and dout must have q's shape");
  require_cuda(lse, "lse");
  TORCH_CHECK_VALUE(lse.sizes() == q_.sizes().slice(0, 3) && lse.scalar_type() == at::kFloat && lse.is_contiguous() &&
                        lse.device() == q_.device(),
                    "lse must be the forward's contiguous float32 [B, H, M] LSE");
  bsa_cross_bwd_args a{};
  if (o_rest) {
    like_q(*o_rest, q_, "o_rest");
    TORCH_CHECK_VALUE(o_rest->sizes() == q_.sizes() && o_rest->strides() == o_.strides(), "o_rest must be laid out as o");
    a.o_rest = o_rest->data_ptr();
  }
  a.lens_dtype = lens_dtype(k_lens, q_, "k_lens");
  a.sm_scale = scale_of(sm_scale, q_.size(3));
  Tensor dq = contiguous_like(q_), dk = contiguous_like(k_), dv = contiguous_like(v_);
  if (q_.numel() == 0) return {dq, dk.zero_(), dv.zero_()};
  const Tensor q = spread(q_, true), k = spread(k_), v = spread(v_), dout = spread(dout_, true);
  const Tensor o = o_rest ? o_ : spread(o_, true);
  // Delta of every row, then the maxima of |dout|
  const int64_t rows = lse.numel();
  const Tensor work = at::empty({2 * rows}, lse.options());
  a.B = dim(q.size(0), "B"), a.H = dim(q.size(1), "H"), a.Hk = dim(k.size(1), "Hk"), a.M = dim(q.size(2), "M");
  a.N = dim(k.size(2), "N"), a.D = dim(q.size(3), "D"), a.dtype = dtype_of(q.scalar_type());
  a.q = t4(q, "q"), a.k = t4(k, "k"), a.v = t4(v, "v"), a.o = t4(o, "o"), a.dout = t4(dout, "dout");
  a.dq = t4(dq, "dq"), a.dk = t4(dk, "dk"), a.dv = t4(dv, "dv");
  a.k_lens = ptr(k_lens);
  a.lse = lse.data_ptr<float>();
  a.delta = work.data_ptr<float>();
  a.err_flag = flag(err);
  const c10::cuda::CUDAGuard guard(q.device());
  check(bsa_cross_bwd_scaled(&a, a.delta + rows, stream_of(q)), "bsa_cross_bwd");
  return {dq, dk, dv};
}

struct CrossFn : torch::autograd::Function<CrossFn> {
  static Tensor forward(AutogradContext* ctx, Tensor q, Tensor k, Tensor v, const OptTensor& k_lens,
                        std::optional<double> sm_scale) {
    const Tensor rest = q.is_cuda() ? contiguous_like(q) : Tensor();
    auto [o, lse] = cross_forward(q, k, v, k_lens, sm_scale, true, {}, {}, if_defined(rest), {});
    ctx->save_for_backward({q, k, v, o, *lse, rest, or_none(k_lens)});
    ctx->saved_data["scale"] = sm_scale;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    once("cross_attention");
    capturable_graph();
    const auto s = ctx->get_saved_variables();
    const auto scale = ctx->saved_data["scale"].toOptional<double>();
    auto [dq, dk, dv] = cross_backward(s[0], s[1], s[2], s[3], s[4], rows(g[0]), if_defined(s[6]), scale, if_defined(s[5]), {});
    return {dq, dk, dv, Tensor(), Tensor()};
  }
};

Tensor cross_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& k_lens,
                      const std::optional<double>& sm_scale) {
  return CrossFn::apply(q, k, v, k_lens, sm_scale);
}

std::tuple<Tensor, OptTensor> prefix_forward(const Tensor& q_, const Tensor& kp_, const Tensor& vp_, const Tensor& k_,
                                             const Tensor& v_, const OptTensor& lens, const std::optional<double>& sm_scale,
                                             bool return_lse, const OptTensor& out, const OptTensor& lse_out,
                                             const OptTensor& err) {
  half_type(q_);
  TORCH_CHECK_VALUE(q_.dim() == 4, "q must be [B, H, T, D], got ", q_.sizes());
  like_q(kp_, q_, "k_prefix");
  like_q(vp_, q_, "v_prefix");
  like_q(k_, q_, "k");
  like_q(v_, q_, "v");
  TORCH_CHECK_VALUE(kp_.dim() == 3 && vp_.sizes() == kp_.sizes() && kp_.size(2) == q_.size(3),
                    "k_prefix and v_prefix must be [Hk, P, ", q_.size(3), "], got ", kp_.sizes(), " and ", vp_.sizes());
  TORCH_CHECK_VALUE(k_.dim() == 4 && v_.sizes() == k_.sizes() && k_.size(0) == q_.size(0) && k_.size(1) == kp_.size(0) &&
                        k_.size(3) == q_.size(3),
                    "k and v must be [", q_.size(0), ", ", kp_.size(0), ", C, ", q_.size(3), "], got ", k_.sizes(), " and ",
                    v_.sizes());
  TORCH_CHECK_VALUE(kp_.size(0) > 0 && q_.size(1) % kp_.size(0) == 0, "the query heads (", q_.size(1),
                    ") must be a multiple of the key / value heads (", kp_.size(0), ")");
  bsa_prefix_args a{};
  a.lens_dtype = lens_dtype(lens, q_, "lens");
  a.sm_scale = scale_of(sm_scale, q_.size(3));
  attention_outputs(out, lse_out, {}, {{q_, "q"}, {kp_, "k_prefix"}, {vp_, "v_prefix"}, {k_, "k"}, {v_, "v"}}, lens, "lens");
  const Tensor o = output(out, q_, "out");
  const OptTensor lse = lse_output(return_lse, lse_out, q_);
  if (q_.numel() == 0) return {o, lse};
  const Tensor q = spread(q_, true), kp = spread(kp_), vp = spread(vp_), k = spread(k_), v = spread(v_);
  a.B = dim(q.size(0), "B"), a.H = dim(q.size(1), "H"), a.Hk = dim(k.size(1), "Hk"), a.T = dim(q.size(2), "T");
  a.P = dim(kp.size(1), "P"), a.C = dim(k.size(2), "C"), a.D = dim(q.size(3), "D"), a.dtype = dtype_of(q.scalar_type());
  a.q = t4(q, "q"), a.o = t4(o, "out"), a.k_prefix = t4(kp, "k_prefix"), a.v_prefix = t4(vp, "v_prefix");
  a.k = t4(k, "k"), a.v = t4(v, "v");
  a.lens = ptr(lens);
  a.lse = static_cast<float*>(ptr(lse));
  a.err_flag = flag(err);
  launch(a, bsa_prefix_fwd_workspace_bytes, bsa_prefix_fwd, q, "bsa_prefix_fwd");
  return {o, lse};
}

}  // namespace

PYBIND11_MODULE(_bsattn_torch, m) {
  namespace py = pybind11;
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const AbiError& e) {
      const py::object cls = py::module_::import("blocksparsefa_reorder_b200._lib").attr("BsaError");
      const py::object err = cls(e.status, e.what_);
      PyErr_SetObject(cls.ptr(), err.ptr());
    }
  });
  using Release = py::call_guard<py::gil_scoped_release>;
  m.def("qk_norm_rope",
        [](OptTensor q, OptTensor k, OptTensor wq, OptTensor wk, OptTensor pos, OptTensor cos, OptTensor sin, double eps,
           bool il, OptTensor q_out, OptTensor k_out, OptTensor err) {
          return rope_forward({q, k, wq, wk, pos, cos, sin, eps, il}, q_out, k_out, err);
        },
        Release());
  m.def("qk_norm_rope_backward",
        [](OptTensor dq, OptTensor dk, OptTensor q, OptTensor k, OptTensor wq, OptTensor wk, OptTensor pos, OptTensor cos,
           OptTensor sin, double eps, bool il, OptTensor err) {
          return rope_backward({q, k, wq, wk, pos, cos, sin, eps, il}, dq, dk, err);
        },
        Release());
  m.def("qk_norm_rope_autograd",
        [](OptTensor q, OptTensor k, OptTensor wq, OptTensor wk, OptTensor pos, OptTensor cos, OptTensor sin, double eps,
           bool il) { return rope_autograd({q, k, wq, wk, pos, cos, sin, eps, il}); },
        Release());
  m.def("cross_attention", &cross_forward, Release());
  m.def("cross_attention_backward", &cross_backward, Release());
  m.def("cross_attention_autograd", &cross_autograd, Release());
  m.def("shared_prefix_attention", &prefix_forward, Release());
  // the memory tests behind the refusals of outputs, which work on any strided tensor
  m.def("overlap", [](const Tensor& a, const Tensor& b) { return static_cast<int>(overlap_of(a, b)); });
  m.def("rows_overlap", &rows_overlap);
}
