// Entry points of the decoder operators around the matrix products: checks of arguments, output allocation and
// gradients.  The autograd nodes are C++ because the smallest calls (one decoding step) are bound by the time to
// get from Python to the launch.
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/util/ArrayRef.h>
#include <c10/util/SmallVector.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <numeric>
#include <tuple>
#include <utility>
#include <vector>

#include "kernels/decoder_ops.h"

namespace mtorus {

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool is_act(const at::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf || t.scalar_type() == at::kFloat;
}

void check_act(const at::Tensor& t, const char* op, const char* name) {
  TORCH_CHECK_TYPE(is_act(t), op, ": ", name, " must be bf16, fp16 or fp32, not ", t.scalar_type());
}

// Last of the checks, so that every other refusal can be had without a GPU.
void check_cuda(std::initializer_list<const at::Tensor*> ts, const char* op) {
  const at::Tensor* first = nullptr;
  for (const at::Tensor* t : ts) {
    if (t->defined())
      TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), op, ": no forward-mode gradient");
  }
  for (const at::Tensor* t : ts) {
    if (!t->defined()) continue;
    TORCH_CHECK(t->is_cuda(), op, ": the tensors must be on a CUDA device (one is on ", t->device(), ")");
    if (first == nullptr) first = t;
    TORCH_CHECK(t->device() == first->device(), op, ": the tensors are on different devices (", first->device(),
                " and ", t->device(), ")");
  }
}

// Uninitialised memory on t's device, without the way through the dispatcher.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& t) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, t.device(), c10::nullopt));
}
at::Tensor fresh_like(const at::Tensor& t) { return fresh(t.sizes(), t.scalar_type(), t); }

at::Tensor last_dense(const at::Tensor& t) {
  return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

// [..., d] as [rows, d] with a dense last dimension, without a copy where the leading dimensions allow it.
at::Tensor rows_of(const at::Tensor& t) {
  const at::Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return last_dense(r);
}

// The same for the norm kernels, whose rows are less than 2^31 values apart.
at::Tensor near_rows_of(const at::Tensor& t) {
  const at::Tensor r = rows_of(t);
  return r.size(0) > 1 && r.stride(0) >= (int64_t(1) << 31) ? r.contiguous() : r;
}

at::Tensor or_undefined(const OptTensor& t) { return t.has_value() ? *t : at::Tensor(); }
OptTensor opt(const at::Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; }

bool needs_grad(std::initializer_list<const at::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts) {
    if (t->defined() && t->requires_grad()) return true;
  }
  return false;
}

void no_double_backward(const char* op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), op, ": the gradient has no gradient (backward with create_graph=True)");
}

// ------------------------------------------------------------------------------------------------ rotary

struct RotarySetup {
  at::Tensor turns;
  int64_t rot_dim = 0;
  bool interleaved = false;
  double scale = 1.0;
};

// [.., H, D] -> [B, S, H, D]
at::Tensor tokens_of(const at::Tensor& x) { return x.dim() == 3 ? x.unsqueeze(0) : x; }

OptTensor positions_of(const OptTensor& positions, int64_t B, int64_t S, int64_t offset) {
  if (!positions.has_value()) return c10::nullopt;
  TORCH_CHECK_VALUE(offset == 0, "rotary: an offset (", offset, ") goes with the default positions only");
  const at::Tensor& p = *positions;
  TORCH_CHECK_TYPE(p.scalar_type() == at::kLong || p.scalar_type() == at::kInt,
                   "rotary: positions must be int64 or int32, not ", p.scalar_type());
  const bool fits = (p.dim() == 1 && p.size(0) == S) ||
                    (p.dim() == 2 && (p.size(0) == B || p.size(0) == 1) && p.size(1) == S) ||
                    (p.dim() == 1 && B > 1 && S == 1 && p.size(0) == B);
  TORCH_CHECK_VALUE(fits, "rotary: positions ", p.sizes(), " do not fit ", B, " sequences of ", S, " tokens");
  if (p.dim() == 1 && p.size(0) != S) return p.unsqueeze(1);
  return p.dim() == 1 ? p.unsqueeze(0).expand({B, S}) : p.expand({B, S});
}

void check_rotary(const at::Tensor& x, const char* name, const RotarySetup& r) {
  check_act(x, "rotary", name);
  TORCH_CHECK_VALUE(x.dim() == 3 || x.dim() == 4, "rotary: ", name,
                    " must be [tokens, heads, dim] or [batch, tokens, heads, dim], not ", x.sizes());
  TORCH_CHECK_VALUE(x.size(-1) >= r.rot_dim && x.size(-1) <= 512, "rotary: ", name, " has head dim ", x.size(-1),
                    "; it must be at least rot_dim (", r.rot_dim, ") and at most 512");
  TORCH_CHECK_VALUE(x.size(-2) < (1 << 20), "rotary: too many heads: ", x.size(-2));
}

void check_pair(const at::Tensor& q, const at::Tensor& k) {
  TORCH_CHECK_TYPE(q.scalar_type() == k.scalar_type(), "rotary: q is ", q.scalar_type(), " but k is ",
                   k.scalar_type());
  TORCH_CHECK_VALUE(q.dim() == k.dim() && q.size(-1) == k.size(-1) &&
                        q.sizes().slice(0, q.dim() - 2) == k.sizes().slice(0, k.dim() - 2),
                    "rotary: q ", q.sizes(), " and k ", k.sizes(), " may differ in their heads only");
}

RotarySetup setup_of(const at::Tensor& turns, int64_t rot_dim, bool interleaved, double scale) {
  TORCH_CHECK_VALUE(rot_dim > 0 && rot_dim % 2 == 0 && turns.scalar_type() == at::kLong &&
                        turns.is_contiguous() && turns.numel() == rot_dim / 2,
                    "rotary: turns must hold rot_dim / 2 fixed-point values");
  return RotarySetup{turns, rot_dim, interleaved, scale};
}

std::vector<at::Tensor> rotary_raw(const std::vector<at::Tensor>& xs, const RotarySetup& r,
                                   const OptTensor& positions, int64_t offset, bool inverse,
                                   const std::vector<int64_t>& heads_rot) {
  c10::cuda::CUDAGuard guard(xs[0].device());
  std::vector<RotarySegment> segs;
  std::vector<at::Tensor> outs;
  for (size_t i = 0; i < xs.size(); ++i) {
    const at::Tensor in = last_dense(xs[i]);
    outs.push_back(fresh_like(xs[i]));
    segs.push_back({tokens_of(in), tokens_of(outs[i]), heads_rot[i]});
  }
  rotary_launch(segs, RotaryArgs{r.turns, r.rot_dim, r.interleaved, r.scale, positions, offset, inverse, false});
  return outs;
}

struct RotaryFn : torch::autograd::Function<RotaryFn> {
  // q and, where defined, k: [B, S, H, D] or [T, H, D]; heads_rot: heads of q that are rotated
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const OptTensor& k,
                               const at::Tensor& turns, const OptTensor& positions, int64_t rot_dim, bool interleaved, double scale,
                               int64_t offset, int64_t heads_rot) {
    at::AutoDispatchBelowADInplaceOrView g;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({turns, or_undefined(positions)});
    auto& d = ctx->saved_data;
    d["rot_dim"] = rot_dim;
    d["interleaved"] = interleaved;
    d["scale"] = scale;
    d["offset"] = offset;
    d["heads_rot"] = heads_rot;
    const RotarySetup r{turns, rot_dim, interleaved, scale};
    if (!k.has_value()) return rotary_raw({q}, r, positions, offset, false, {heads_rot});
    return rotary_raw({q, *k}, r, positions, offset, false, {heads_rot, k->size(-2)});
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    no_double_backward("rotary");
    const auto saved = ctx->get_saved_variables();
    auto& d = ctx->saved_data;
    const RotarySetup r{saved[0], d["rot_dim"].toInt(), d["interleaved"].toBool(), d["scale"].toDouble()};
    variable_list out(9);
    std::vector<at::Tensor> xs;
    std::vector<int64_t> heads, slot;
    for (size_t i = 0; i < g.size(); ++i) {
      if (!g[i].defined() || !ctx->needs_input_grad(i)) continue;
      xs.push_back(g[i]);
      heads.push_back(i == 0 ? d["heads_rot"].toInt() : g[i].size(-2));
      slot.push_back((int64_t)i);
    }
    if (xs.empty()) return out;
    const auto got = rotary_raw(xs, r, opt(saved[1]), d["offset"].toInt(), true, heads);
    for (size_t i = 0; i < got.size(); ++i) out[slot[i]] = got[i];
    return out;
  }
};

// A multiple of `step` from `low` to `high`.
struct Term {
  int64_t step, low, high;
};

// Whether `at` plus a multiple of each term's step (falling) can come within `width` of 0. Exact, but for a layout so
// entangled that `budget` trials do not settle it: true.
bool can_meet(c10::ArrayRef<Term> terms, size_t next, int64_t at, int64_t width, int& budget) {
  if (next == terms.size()) return std::abs(at) < width;
  if (--budget < 0) return true;
  const Term& t = terms[next];
  int64_t least = 0, most = 0;  // what the terms behind this one can add
  int64_t grid = t.step;        // all that can be added is a multiple of this
  for (size_t i = next + 1; i < terms.size(); ++i) {
    least += terms[i].step * terms[i].low;
    most += terms[i].step * terms[i].high;
    grid = std::gcd(grid, terms[i].step);
  }
  const int64_t off = std::abs(at) % grid;
  if (std::min(off, grid - off) >= width) return false;
  auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
  const int64_t from = std::max(t.low, -floor_div(at + most + width - 1, t.step)),
                to = std::min(t.high, floor_div(width - 1 - at - least, t.step));
  for (int64_t m = from; m <= to; ++m) {
    if (can_meet(terms, next + 1, at + m * t.step, width, budget)) return true;
  }
  return false;
}

// Whether heads of q and of k lie over one another, the same token's or different ones', as views of one buffer may. (Views
// that are not dense as a whole are beyond at::assert_no_overlap.)
bool share_heads(const at::Tensor& q, const at::Tensor& k) {
  if (q.numel() == 0 || k.numel() == 0) return false;
  const int64_t size = q.element_size(), width = q.size(-1) * size;
  auto extent = [&](const at::Tensor& t) {
    int64_t e = width;
    for (int64_t i = 0; i < t.dim() - 1; ++i) e += (t.size(i) - 1) * t.stride(i) * size;
    return e;
  };
  const int64_t between = reinterpret_cast<intptr_t>(k.data_ptr()) - reinterpret_cast<intptr_t>(q.data_ptr());
  if (between >= extent(q) || -between >= extent(k)) return false;
  // a head of k lies `between` + its own steps - those of the head of q from that
  c10::SmallVector<Term, 6> terms;
  for (int sign : {-1, 1}) {
    const at::Tensor& t = sign < 0 ? q : k;
    for (int64_t i = 0; i < t.dim() - 1; ++i) {
      if (t.size(i) == 1) continue;
      const int64_t step = t.stride(i) * size, n = t.size(i) - 1;
      auto same = std::find_if(terms.begin(), terms.end(), [&](const Term& o) { return o.step == step; });
      if (same == terms.end()) same = terms.insert(same, Term{step, 0, 0});
      (sign < 0 ? same->low : same->high) += sign * n;
    }
  }
  std::sort(terms.begin(), terms.end(), [](const Term& a, const Term& b) { return a.step > b.step; });
  int budget = 10000;
  return can_meet(terms, 0, between, width, budget);
}

// Whether the heads of x are known to lie apart from one another: each axis steps over all that the smaller ones cover.
bool heads_apart(const at::Tensor& x) {
  c10::SmallVector<std::pair<int64_t, int64_t>, 4> axes;
  for (int64_t i = 0; i < x.dim(); ++i) {
    if (x.size(i) > 1) axes.emplace_back(x.stride(i), x.size(i));
  }
  std::sort(axes.begin(), axes.end());
  int64_t covered = 1;
  for (const auto& [step, n] : axes) {
    if (step < covered) return false;
    covered += (n - 1) * step;
  }
  return true;
}

}  // namespace

std::tuple<at::Tensor, OptTensor> rotary(const at::Tensor& q, const OptTensor& k, const at::Tensor& turns,
                                         int64_t rot_dim, bool interleaved, double scale, const OptTensor& positions,
                                         int64_t offset) {
  const RotarySetup r = setup_of(turns, rot_dim, interleaved, scale);
  check_rotary(q, "q", r);
  if (k.has_value()) {
    check_rotary(*k, "k", r);
    check_pair(q, *k);
  }
  const at::Tensor qt = tokens_of(q), kt = or_undefined(k);
  const OptTensor pos = positions_of(positions, qt.size(0), qt.size(1), offset);
  check_cuda({&q, &kt, &turns, pos.has_value() ? &*pos : &turns}, "rotary");
  variable_list out;
  if (needs_grad({&q, &kt}))
    out = RotaryFn::apply(q, k, turns, pos, rot_dim, interleaved, scale, offset, q.size(-2));
  else if (kt.defined())
    out = rotary_raw({q, kt}, r, pos, offset, false, {q.size(-2), kt.size(-2)});
  else
    out = rotary_raw({q}, r, pos, offset, false, {q.size(-2)});
  return {out[0], k.has_value() ? OptTensor(out[1]) : c10::nullopt};
}

at::Tensor rotary_qkv(const at::Tensor& qkv, int64_t B, int64_t S, int64_t heads, int64_t kv_heads,
                      int64_t head_dim, const at::Tensor& turns, int64_t rot_dim, bool interleaved, double scale,
                      const OptTensor& positions, int64_t offset) {
  const RotarySetup r = setup_of(turns, rot_dim, interleaved, scale);
  check_act(qkv, "rotary_qkv", "qkv");
  TORCH_CHECK_VALUE(B >= 0 && S >= 0 && heads > 0 && kv_heads > 0 && qkv.dim() == 2 && qkv.size(0) == B * S &&
                        qkv.size(1) == (heads + 2 * kv_heads) * head_dim,
                    "rotary_qkv: qkv must be [B*S, (heads + 2 kv_heads) * head_dim] = [", B * S, ", ",
                    (heads + 2 * kv_heads) * head_dim, "], not ", qkv.sizes());
  const at::Tensor x = last_dense(qkv).unflatten(1, {heads + 2 * kv_heads, head_dim}).unflatten(0, {B, S});
  check_rotary(x, "qkv", r);
  const OptTensor pos = positions_of(positions, B, S, offset);
  check_cuda({&qkv, &turns, pos.has_value() ? &*pos : &turns}, "rotary_qkv");
  const auto out = needs_grad({&x}) ? RotaryFn::apply(x, OptTensor(), turns, pos, rot_dim, interleaved, scale, offset,
                                                      heads + kv_heads)
                                    : rotary_raw({x}, r, pos, offset, false, {heads + kv_heads});
  return out[0].view(qkv.sizes());
}

void rotary_inplace(at::Tensor q, const OptTensor& k, const at::Tensor& turns, int64_t rot_dim, bool interleaved,
                    double scale, const OptTensor& positions, int64_t offset, bool inverse) {
  const RotarySetup r = setup_of(turns, rot_dim, interleaved, scale);
  at::Tensor kt = or_undefined(k);
  for (const at::Tensor* t : {&q, &kt}) {
    if (!t->defined()) continue;
    check_rotary(*t, t == &q ? "q" : "k", r);
    TORCH_CHECK(!needs_grad({t}),
                "rotary_: works in place and records no gradient; use rotary() on tensors that require one");
    TORCH_CHECK_VALUE(t->size(-1) <= 1 || t->stride(-1) == 1, "rotary_: the head dim must have stride 1");
    if (t->numel() > 0 && !heads_apart(*t)) {
      at::assert_no_internal_overlap(*t);
      TORCH_CHECK_VALUE(false, "rotary_: ", t == &q ? "q" : "k", " has heads that are the same memory in some of their ",
                        "values (sizes ", t->sizes(), ", strides ", t->strides(), ")");
    }
  }
  if (kt.defined()) {
    check_pair(q, kt);
    TORCH_CHECK_VALUE(q.data_ptr() != kt.data_ptr() || q.numel() == 0, "rotary_: q and k are the same memory");
    if (share_heads(q, kt)) {
      at::assert_no_overlap(q, kt);
      TORCH_CHECK_VALUE(false, "rotary_: q and k are the same memory in some of their heads, or in a layout too entangled ",
                        "to tell (strides ", q.strides(), " and ", kt.strides(), ")");
    }
  }
  const at::Tensor qt = tokens_of(q);
  const OptTensor pos = positions_of(positions, qt.size(0), qt.size(1), offset);
  check_cuda({&q, &kt, &turns, pos.has_value() ? &*pos : &turns}, "rotary_");
  c10::cuda::CUDAGuard guard(q.device());
  std::vector<RotarySegment> segs{{qt, qt, qt.size(2)}};
  if (kt.defined()) segs.push_back({tokens_of(kt), tokens_of(kt), kt.size(-2)});
  q.unsafeGetTensorImpl()->bump_version();  // refuses inference tensors outside inference mode
  if (kt.defined()) kt.unsafeGetTensorImpl()->bump_version();
  rotary_launch(segs, RotaryArgs{turns, rot_dim, interleaved, scale, pos, offset, inverse, true});
}

// ------------------------------------------------------------------------------------------ residual norm

namespace {

int gate_kind(const at::Tensor& gate, const at::Tensor& x) {
  if (!gate.defined()) return kGateNone;
  const int64_t d = x.size(-1);
  auto lead = x.sizes().slice(0, x.dim() - 1);
  if (gate.sizes() == x.sizes() && gate.scalar_type() == x.scalar_type() && !(x.dim() == 1)) {
    if (!(d == 1 && gate.scalar_type() == at::kFloat)) return kGateFull;
  }
  if (gate.dim() == x.dim() && gate.size(-1) == 1 && gate.sizes().slice(0, gate.dim() - 1) == lead) {
    TORCH_CHECK_TYPE(gate.scalar_type() == at::kFloat, "residual_norm: a gate per row must be fp32, not ",
                     gate.scalar_type());
    return kGateRow;
  }
  if (gate.dim() == 1 && gate.size(0) == d) {
    TORCH_CHECK_TYPE(gate.scalar_type() == at::kFloat, "residual_norm: a gate per channel must be fp32, not ",
                     gate.scalar_type());
    return kGateChannel;
  }
  TORCH_CHECK_TYPE(gate.sizes() != x.sizes(), "residual_norm: a gate per element must have x's type (",
                   x.scalar_type(), "), not ", gate.scalar_type());
  TORCH_CHECK_VALUE(false, "residual_norm: the gate must be [d], [..., 1] or like x (", x.sizes(), "), not ",
                    gate.sizes());
}

ResidualNormArgs norm_args(const at::Tensor& x, const at::Tensor& h, const at::Tensor& pre, const at::Tensor& post,
                           const at::Tensor& gate, int kind, double beta, double alpha, double eps) {
  ResidualNormArgs a;
  a.x = near_rows_of(x);
  if (h.defined()) a.h = near_rows_of(h);
  if (pre.defined()) a.pre = pre.contiguous();
  if (post.defined()) a.post = post.contiguous();
  if (gate.defined()) a.gate = kind == kGateFull ? near_rows_of(gate) : gate.contiguous();
  a.gate_kind = kind;
  a.beta = beta;
  a.alpha = alpha;
  a.eps = eps;
  return a;
}

struct NormOutputs {
  at::Tensor y, n, rstd_h, rstd_y;
  variable_list list() const {
    variable_list out;
    if (y.defined()) out.push_back(y);
    if (n.defined()) out.push_back(n);
    return out;
  }
};

NormOutputs norm_forward(const at::Tensor& x, const at::Tensor& h, const at::Tensor& pre, const at::Tensor& post,
                         const at::Tensor& gate, int kind, double beta, double alpha, double eps, bool statistics) {
  c10::cuda::CUDAGuard guard(x.device());
  const ResidualNormArgs a = norm_args(x, h, pre, post, gate, kind, beta, alpha, eps);
  NormOutputs o;
  if (h.defined()) o.y = fresh_like(x);
  if (pre.defined()) o.n = fresh_like(x);
  if (statistics) {
    const at::Tensor stats = fresh({2, a.x.size(0)}, at::kFloat, x);
    if (post.defined()) o.rstd_h = stats.select(0, 0);
    if (pre.defined()) o.rstd_y = stats.select(0, 1);
  }
  residual_norm_fwd_launch(a, o.y, o.n, o.rstd_h, o.rstd_y);
  return o;
}

struct ResidualNormFn : torch::autograd::Function<ResidualNormFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& branch,
                               const OptTensor& pre_weight, const OptTensor& post_weight, const OptTensor& gate_,
                               int64_t kind, double beta, double alpha, double eps) {
    at::AutoDispatchBelowADInplaceOrView g;
    const at::Tensor h = or_undefined(branch), pre = or_undefined(pre_weight), post = or_undefined(post_weight),
                     gate = or_undefined(gate_);
    ctx->set_materialize_grads(false);
    const NormOutputs o = norm_forward(x, h, pre, post, gate, (int)kind, beta, alpha, eps, true);
    ctx->save_for_backward({x, h, pre, post, gate, o.rstd_h, o.rstd_y});
    auto& d = ctx->saved_data;
    d["kind"] = kind;
    d["beta"] = beta;
    d["alpha"] = alpha;
    d["eps"] = eps;
    return o.list();
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    no_double_backward("residual_norm");
    const auto s = ctx->get_saved_variables();
    const at::Tensor &x = s[0], &h = s[1], &pre = s[2], &post = s[3], &gate = s[4];
    c10::cuda::CUDAGuard guard(x.device());
    auto& d = ctx->saved_data;
    const int kind = (int)d["kind"].toInt();
    const ResidualNormArgs a = norm_args(x, h, pre, post, gate, kind, d["beta"].toDouble(), d["alpha"].toDouble(),
                                         d["eps"].toDouble());
    size_t at = 0;
    at::Tensor dy = h.defined() ? g[at++] : at::Tensor(), dn = pre.defined() ? g[at] : at::Tensor();
    variable_list out(9);
    if (!dy.defined() && !dn.defined()) return out;
    auto rows = [](const at::Tensor& t) { return t.defined() ? near_rows_of(t) : t; };
    // the node has an edge for each tensor that was given: i-th argument, next edge
    size_t edge = 0;
    for (size_t i = 0; i < 5; ++i) {
      if (s[i].defined() && ctx->needs_input_grad(edge++) && !(i == 2 && !dn.defined()))
        out[i] = fresh_like(s[i]);
    }
    residual_norm_bwd_launch(a, s[5], s[6], rows(dy), rows(dn), out[0], out[1], out[4], out[2], out[3]);
    return out;
  }
};

void check_weight(const at::Tensor& w, int64_t d, const char* name) {
  if (!w.defined()) return;
  TORCH_CHECK_TYPE(w.scalar_type() == at::kFloat, "residual_norm: ", name, " must be fp32, not ", w.scalar_type());
  TORCH_CHECK_VALUE(w.dim() == 1 && w.size(0) == d, "residual_norm: ", name, " must be [", d, "], not ", w.sizes());
}

void check_norm_x(const at::Tensor& x) {
  check_act(x, "residual_norm", "x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 16384,
                    "residual_norm: x must be [..., d] with d from 1 to 16384, not ", x.sizes());
}

}  // namespace

std::tuple<at::Tensor, OptTensor> residual_norm(const at::Tensor& x, const at::Tensor& branch, const OptTensor& pre,
                                                const OptTensor& post, const OptTensor& gate, double residual_scale,
                                                double branch_scale, double eps) {
  check_norm_x(x);
  TORCH_CHECK_TYPE(branch.scalar_type() == x.scalar_type(), "residual_norm: x is ", x.scalar_type(),
                   " but the branch is ", branch.scalar_type());
  TORCH_CHECK_VALUE(branch.sizes() == x.sizes(), "residual_norm: x ", x.sizes(), " and the branch ", branch.sizes(),
                    " must have the same shape");
  const at::Tensor pw = or_undefined(pre), qw = or_undefined(post), gt = or_undefined(gate);
  check_weight(pw, x.size(-1), "pre_weight");
  check_weight(qw, x.size(-1), "post_weight");
  const int kind = gate_kind(gt, x);
  TORCH_CHECK_VALUE(std::isfinite(residual_scale) && std::isfinite(branch_scale) && eps >= 0 && std::isfinite(eps),
                    "residual_norm: the scales must be finite and eps at least 0");
  check_cuda({&x, &branch, &pw, &qw, &gt}, "residual_norm");
  const auto out =
      needs_grad({&x, &branch, &pw, &qw, &gt})
          ? ResidualNormFn::apply(x, OptTensor(branch), pre, post, gate, (int64_t)kind, residual_scale, branch_scale, eps)
          : norm_forward(x, branch, pw, qw, gt, kind, residual_scale, branch_scale, eps, false).list();
  return {out[0], pw.defined() ? OptTensor(out[1]) : c10::nullopt};
}

at::Tensor rms_norm(const at::Tensor& x, const at::Tensor& weight, double eps) {
  check_norm_x(x);
  check_weight(weight, x.size(-1), "weight");
  TORCH_CHECK_VALUE(eps >= 0 && std::isfinite(eps), "rms_norm: eps must be at least 0");
  check_cuda({&x, &weight}, "rms_norm");
  if (!needs_grad({&x, &weight}))
    return norm_forward(x, at::Tensor(), weight, at::Tensor(), at::Tensor(), kGateNone, 1.0, 1.0, eps, false).n;
  const OptTensor none;
  return ResidualNormFn::apply(x, none, OptTensor(weight), none, none, (int64_t)kGateNone, 1.0, 1.0, eps)[0];
}

// ------------------------------------------------------------------------------------------ log probabilities

namespace {

struct LogprobOutputs {
  at::Tensor tokens, logprob, stats, entropy, top_lp, top_ids;
  variable_list list() const {
    variable_list out{logprob};
    for (const at::Tensor* t : {&entropy, &top_lp, &top_ids}) {
      if (t->defined()) out.push_back(*t);
    }
    return out;
  }
};

LogprobOutputs logprobs_forward(const at::Tensor& logits, const at::Tensor& tokens, double inv_tau, int64_t top,
                                bool entropy) {
  c10::cuda::CUDAGuard guard(logits.device());
  const at::Tensor x = rows_of(logits);
  LogprobOutputs o;
  o.tokens = tokens.dim() == 1 ? tokens.contiguous() : tokens.reshape({-1}).contiguous();
  o.logprob = fresh(tokens.sizes(), at::kFloat, logits);
  o.stats = fresh({x.size(0), 2}, at::kFloat, logits);
  if (entropy) o.entropy = fresh(tokens.sizes(), at::kFloat, logits);
  if (top > 0) {
    std::vector<int64_t> shape(tokens.sizes().begin(), tokens.sizes().end());
    shape.push_back(top);
    o.top_lp = fresh(shape, at::kFloat, logits);
    o.top_ids = fresh(shape, at::kLong, logits);
  }
  token_logprobs_fwd_launch(x, o.tokens, inv_tau, top, o.logprob, o.stats, o.entropy, o.top_lp, o.top_ids);
  return o;
}

struct TokenLogprobsFn : torch::autograd::Function<TokenLogprobsFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& tokens,
                               double inv_tau, int64_t top, bool entropy) {
    at::AutoDispatchBelowADInplaceOrView g;
    ctx->set_materialize_grads(false);
    const LogprobOutputs o = logprobs_forward(logits, tokens, inv_tau, top, entropy);
    ctx->save_for_backward({logits, o.tokens, o.stats, o.entropy, o.top_ids});
    ctx->saved_data["inv_tau"] = inv_tau;
    ctx->saved_data["top"] = top;
    ctx->saved_data["entropy"] = entropy;
    if (top > 0) ctx->mark_non_differentiable({o.top_ids});
    return o.list();
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    no_double_backward("token_logprobs");
    const auto s = ctx->get_saved_variables();
    const bool entropy = ctx->saved_data["entropy"].toBool();
    const int64_t top = ctx->saved_data["top"].toInt();
    c10::cuda::CUDAGuard guard(s[0].device());
    size_t at = 0;
    auto next = [&](bool there) {
      const at::Tensor t = there ? g[at++] : at::Tensor();
      return t.defined() ? t.contiguous() : t;
    };
    const at::Tensor gl = next(true), gh = next(entropy), gk = next(top > 0);
    variable_list out(5);
    if (!gl.defined() && !gh.defined() && !gk.defined()) return out;
    out[0] = fresh_like(s[0]);
    token_logprobs_bwd_launch(rows_of(s[0]), s[1], ctx->saved_data["inv_tau"].toDouble(), top, s[2], s[3], s[4], gl,
                              gh, gk, out[0]);
    return out;
  }
};

}  // namespace

std::tuple<at::Tensor, OptTensor, OptTensor, OptTensor> token_logprobs(const at::Tensor& logits,
                                                                       const at::Tensor& tokens, double temperature,
                                                                       int64_t top, bool entropy) {
  check_act(logits, "token_logprobs", "logits");
  TORCH_CHECK_TYPE(tokens.scalar_type() == at::kLong, "token_logprobs: tokens must be int64, not ",
                   tokens.scalar_type());
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.sizes().slice(0, logits.dim() - 1) == tokens.sizes(),
                    "token_logprobs: logits must be [..., vocabulary] for tokens [...], not ", logits.sizes(), " for ",
                    tokens.sizes());
  const int64_t V = logits.size(-1);
  TORCH_CHECK_VALUE(V >= 1 && V < (int64_t(1) << 31), "token_logprobs: a vocabulary of ", V, " values");
  TORCH_CHECK_VALUE(top >= 0 && top <= 64 && top <= V,
                    "token_logprobs: top must be from 0 to 64 and at most the vocabulary (", V, "), not ", top);
  TORCH_CHECK_VALUE(temperature >= 1e-6 && temperature <= 1e6,
                    "token_logprobs: the temperature must be from 1e-6 to 1e6, not ", temperature);
  check_cuda({&logits, &tokens}, "token_logprobs");
  const auto out = needs_grad({&logits}) ? TokenLogprobsFn::apply(logits, tokens, 1.0 / temperature, top, entropy)
                                         : logprobs_forward(logits, tokens, 1.0 / temperature, top, entropy).list();
  size_t at = 1;
  OptTensor ent, top_lp, top_ids;
  if (entropy) ent = out[at++];
  if (top > 0) {
    top_lp = out[at++];
    top_ids = out[at];
  }
  return {out[0], ent, top_lp, top_ids};
}

void bind_decoder_ops(pybind11::module& m) {
  namespace py = pybind11;
  m.def("rotary", &rotary);
  m.def("rotary_qkv", &rotary_qkv);
  m.def("rotary_inplace", &rotary_inplace);
  m.def("residual_norm", &residual_norm);
  m.def("rms_norm", &rms_norm);
  m.def("token_logprobs", &token_logprobs);
}

}  // namespace mtorus
