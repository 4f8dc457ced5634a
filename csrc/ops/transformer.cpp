// Operators of a transformer's training step (namespace catch_b200), each with its gradient:
//   qk_norm_rotary           -- RMS norm of query / key heads and the rotation by position
//   relative_bias_softmax    -- softmax over scores with a learned relative position bias, scale and mask
//   top_logits_distillation  -- loss against a teacher's top K logits
//
// The reference has no counterpart (its eager layers run these as separate norm, multiply, gather, add and softmax
// calls).  Every operator has a host path in elementary operations for host simulation and for tensors of other
// devices; gradients are wired up here, so torch.ops.catch_b200.<name> is differentiable as it is.  The autograd kernels go on through
// the dispatcher, so that what lies below them (torch.func's transforms, dispatch modes, fake tensors) sees the operators and their
// _backward forms.
#include <ATen/TensorSubclassLikeUtils.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/core/grad_mode.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <map>
#include <mutex>

#include "../runtime/graph.h"
#include "common.h"
#include "kernels.h"

namespace catch_b200 {
namespace ops {
namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

constexpr double kInf = std::numeric_limits<double>::infinity();

bool f_ok(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }
bool given(const OptTensor& t) { return t.has_value() && t->defined(); }
// Uninitialised device tensors without a trip through the dispatcher.
Tensor fresh(at::IntArrayRef sizes, const Tensor& like) { return empty_b200(sizes, like.scalar_type(), like.device().index()); }
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) { return empty_b200(sizes, type, like.device().index()); }
Tensor fresh_strided(const Tensor& like) { return empty_strided_b200(like.sizes(), like.strides(), like.scalar_type(), like.device().index()); }
bool on_device(const Tensor& t) { return !use_cpu_path() && is_b200(t); }

// ------------------------------------------------------------------------------------------ norm and rotation of q, k
struct RotaryArgs {
  Tensor q, k;
  OptTensor qw, kw;
  Tensor cos, sin;
  OptTensor positions;
  double eps;
  bool interleaved;
};

void check_rotary(const RotaryArgs& a) {
  const char* op = "qk_norm_rotary";
  TORCH_CHECK(a.q.dim() == 4 && a.k.dim() == 4, op, ": queries and keys are [batch, length, heads, head_dim], got ", a.q.sizes(),
              " and ", a.k.sizes());
  const int64_t B = a.q.size(0), L = a.q.size(1), D = a.q.size(3);
  TORCH_CHECK(a.k.size(0) == B && a.k.size(1) == L && a.k.size(3) == D, op,
              ": queries and keys differ in batch, length or head_dim: ", a.q.sizes(), " and ", a.k.sizes());
  TORCH_CHECK(f_ok(a.q.scalar_type()) && a.q.scalar_type() == a.k.scalar_type(), op,
              ": queries and keys are both float32, bfloat16 or float16, got ", a.q.scalar_type(), " and ", a.k.scalar_type());
  TORCH_CHECK(D >= 2 && D % 2 == 0 && D <= B200_QK_MAX_HEAD_DIM, op, ": head_dim must be even and at most ", B200_QK_MAX_HEAD_DIM,
              ", got ", D);
  TORCH_CHECK(a.cos.dim() == 2 && a.sin.sizes() == a.cos.sizes(), op, ": cos and sin are [positions, rotated / 2], got ", a.cos.sizes(),
              " and ", a.sin.sizes());
  TORCH_CHECK(f_ok(a.cos.scalar_type()) && f_ok(a.sin.scalar_type()), op, ": cos and sin are floating tables, got ",
              a.cos.scalar_type(), " and ", a.sin.scalar_type());
  TORCH_CHECK(2 * a.cos.size(1) <= D, op, ": cos and sin rotate ", 2 * a.cos.size(1), " dimensions of ", D);
  for (const OptTensor* w : {&a.qw, &a.kw})
    if (given(*w))
      TORCH_CHECK((*w)->dim() == 1 && (*w)->size(0) == D && f_ok((*w)->scalar_type()), op, ": weights are floating [head_dim], got ",
                  (*w)->scalar_type(), " ", (*w)->sizes());
  if (given(a.positions)) {
    TORCH_CHECK(a.positions->scalar_type() == at::kLong || a.positions->scalar_type() == at::kInt, op,
                ": positions are int64 or int32, got ", a.positions->scalar_type());
    TORCH_CHECK((a.positions->dim() == 2 && (a.positions->size(0) == B || a.positions->size(0) == 1) && a.positions->size(1) == L) ||
                    (a.positions->dim() == 1 && a.positions->size(0) == L),
                op, ": positions are [batch, length] or [length], got ", a.positions->sizes());
  } else {
    TORCH_CHECK(L <= a.cos.size(0), op, ": ", L, " tokens, but cos and sin have ", a.cos.size(0), " positions");
  }
  TORCH_CHECK(a.eps >= 0, op, ": eps must not be negative, got ", a.eps);
  TORCH_CHECK(B * L * std::max(a.q.size(2), a.k.size(2)) < (int64_t(1) << 31), op, ": more than 2^31 heads in one call");
  check_same_device(op, a.q, a.k, a.qw, a.kw, a.cos, a.sin, a.positions);
}

Tensor positions_of(const RotaryArgs& a) {  // [1 or B, L]
  if (!given(a.positions)) return at::arange(a.q.size(1), a.q.options().dtype(at::kLong)).unsqueeze(0);
  return a.positions->dim() == 1 ? a.positions->unsqueeze(0) : *a.positions;
}

// Host path: the tokens' cos / sin [*, L, 1, R/2] and whether each position lies inside the tables [*, L, 1, 1].
std::tuple<Tensor, Tensor, Tensor> host_angles(const RotaryArgs& a) {
  Tensor pos = positions_of(a).to(at::kLong);
  Tensor inside = pos.ge(0).logical_and(pos.lt(a.cos.size(0)));
  if (flags().async_disable && pos.numel() > 0)
    TORCH_CHECK_INDEX(pos.lt(a.cos.size(0)).all().item<bool>(), "qk_norm_rotary: index out of range");
  std::vector<int64_t> shape{pos.size(0), pos.size(1), 1, a.cos.size(1)};
  Tensor cos = at::zeros(shape, a.q.options().dtype(at::kFloat)), sin = at::zeros(shape, a.q.options().dtype(at::kFloat));
  if (a.cos.size(0) > 0) {
    Tensor at = pos.clamp(0, a.cos.size(0) - 1).reshape({-1});
    cos = a.cos.to(at::kFloat).index_select(0, at).view(shape);
    sin = a.sin.to(at::kFloat).index_select(0, at).view(shape);
  }
  return {cos, sin, inside.unsqueeze(-1).unsqueeze(-1)};
}
Tensor host_turn(const Tensor& n, const Tensor& cos, const Tensor& sin, bool interleaved) {
  const int64_t R = 2 * cos.size(-1), D = n.size(-1);
  if (R == 0) return n;
  Tensor x = interleaved ? n.slice(-1, 0, R, 2) : n.slice(-1, 0, R / 2), y = interleaved ? n.slice(-1, 1, R, 2) : n.slice(-1, R / 2, R);
  Tensor u = x * cos - y * sin, v = y * cos + x * sin;
  Tensor turned = interleaved ? at::stack({u, v}, -1).flatten(-2) : at::cat({u, v}, -1);
  return at::cat({turned, n.slice(-1, R, D)}, -1);
}
Tensor host_rotary_fwd(const RotaryArgs& a, const Tensor& x, const OptTensor& w) {
  auto [cos, sin, inside] = host_angles(a);
  Tensor t = x.to(at::kFloat);
  Tensor n = t * at::rsqrt((t * t).mean(-1, true) + a.eps);
  if (given(w)) n = n * w->to(at::kFloat);
  Tensor y = host_turn(n, cos, sin, a.interleaved);
  return at::where(inside, y, at::zeros_like(y)).to(x.scalar_type()).contiguous();
}
std::tuple<Tensor, Tensor> host_rotary_bwd(const RotaryArgs& a, const Tensor& x, const OptTensor& w, const Tensor& dy) {
  auto [cos, sin, inside] = host_angles(a);
  Tensor t = x.to(at::kFloat), r = at::rsqrt((t * t).mean(-1, true) + a.eps), n = t * r;
  Tensor g = host_turn(dy.to(at::kFloat), cos, -sin, a.interleaved);
  Tensor dw, zero = at::zeros_like(g);
  if (given(w)) {
    dw = at::where(inside, g * n, zero).sum({0, 1, 2}).to(w->scalar_type());
    g = g * w->to(at::kFloat);
  }
  Tensor dx = r * (g - n * (g * n).mean(-1, true));
  return {at::where(inside, dx, zero).to(x.scalar_type()).contiguous(), dw};
}

std::tuple<Tensor, Tensor> qk_norm_rotary_meta(const Tensor& q, const Tensor& k, const OptTensor& qw, const OptTensor& kw, const Tensor& cos,
                                               const Tensor& sin, const OptTensor& positions, double eps, bool interleaved) {
  check_rotary({q, k, qw, kw, cos, sin, positions, eps, interleaved});
  return {at::empty(q.sizes(), q.options()), at::empty(k.sizes(), k.options())};
}
void check_rotary_grads(const RotaryArgs& a, const Tensor& dyq, const Tensor& dyk) {
  check_rotary(a);
  TORCH_CHECK(dyq.sizes() == a.q.sizes() && dyk.sizes() == a.k.sizes() && dyq.scalar_type() == a.q.scalar_type() &&
                  dyk.scalar_type() == a.k.scalar_type(),
              "qk_norm_rotary_backward: the gradients have the shapes and the dtype of queries and keys");
  check_same_device("qk_norm_rotary_backward", a.q, dyq, dyk);
}
std::tuple<Tensor, Tensor, Tensor, Tensor> qk_norm_rotary_backward_meta(const Tensor& dyq, const Tensor& dyk, const Tensor& q, const Tensor& k,
                                                                        const OptTensor& qw, const OptTensor& kw, const Tensor& cos,
                                                                        const Tensor& sin, const OptTensor& positions, double eps,
                                                                        bool interleaved, bool need_qw, bool need_kw) {
  check_rotary_grads({q, k, qw, kw, cos, sin, positions, eps, interleaved}, dyq, dyk);
  return {at::empty(q.sizes(), q.options()), at::empty(k.sizes(), k.options()),
          given(qw) && need_qw ? at::empty(qw->sizes(), qw->options()) : Tensor(), given(kw) && need_kw ? at::empty(kw->sizes(), kw->options()) : Tensor()};
}

// The kernels read a row's two statistics at once; a caller's may begin anywhere.
Tensor by_pairs(const Tensor& stats) { return reinterpret_cast<uintptr_t>(stats.data_ptr()) % 8 == 0 ? stats : stats.clone(); }
Tensor dense_last(const Tensor& t) { return t.stride(-1) == 1 || t.numel() == 0 ? t : t.contiguous(); }

// The kernel's arguments that both directions share; `keep` holds what has to outlive the call.
B200QkNormRotary rotary_params(const RotaryArgs& a, const Tensor& q, const Tensor& k, const OptTensor& qw, const OptTensor& kw,
                               std::vector<Tensor>& keep) {
  B200QkNormRotary p{};
  p.B = q.size(0); p.L = q.size(1); p.D = (int)q.size(3); p.R = (int)(2 * a.cos.size(1));
  p.dtype = to_b200_dtype(q.scalar_type());
  p.interleaved = a.interleaved;
  Tensor cos = a.cos.to(at::kFloat).contiguous(), sin = a.sin.to(at::kFloat).contiguous();
  p.cos = cos.data_ptr<float>(); p.sin = sin.data_ptr<float>(); p.table_rows = cos.size(0);
  keep.push_back(cos); keep.push_back(sin);
  if (given(a.positions)) {
    const Tensor& t = *a.positions;
    const bool one = t.dim() == 1;
    p.positions = t.data_ptr();
    p.positions_dtype = to_b200_dtype(t.scalar_type());
    p.pos_stride[0] = one || t.size(0) == 1 ? 0 : t.stride(0);
    p.pos_stride[1] = t.stride(one ? 0 : 1);
    p.bad_flag = checked_index_flag(q);
  }
  p.eps = (float)a.eps;
  const Tensor* xs[2] = {&q, &k};
  const OptTensor* ws[2] = {&qw, &kw};
  for (int s = 0; s < 2; ++s) {
    B200QkSide& d = p.side[s];
    d.x = xs[s]->data_ptr();
    d.heads = (int)xs[s]->size(2);
    for (int i = 0; i < 3; ++i) d.x_stride[i] = xs[s]->stride(i);
    if (given(*ws[s])) {
      d.weight = (*ws[s])->data_ptr();
      d.weight_dtype = to_b200_dtype((*ws[s])->scalar_type());
    }
  }
  return p;
}
OptTensor dense_weight(const OptTensor& w) { return given(w) ? OptTensor(w->contiguous()) : OptTensor(); }

std::tuple<Tensor, Tensor> qk_norm_rotary(const Tensor& q_in, const Tensor& k_in, const OptTensor& qw_in, const OptTensor& kw_in, const Tensor& cos,
                                          const Tensor& sin, const OptTensor& positions, double eps, bool interleaved) {
  const RotaryArgs a{q_in, k_in, qw_in, kw_in, cos, sin, positions, eps, interleaved};
  check_rotary(a);
  if (!on_device(a.q)) return {host_rotary_fwd(a, a.q, a.qw), host_rotary_fwd(a, a.k, a.kw)};
  OpScope scope("qk_norm_rotary", a.q);
  Tensor q = dense_last(a.q), k = dense_last(a.k), yq = fresh(q.sizes(), q), yk = fresh(k.sizes(), k);
  const OptTensor qw = dense_weight(a.qw), kw = dense_weight(a.kw);
  std::vector<Tensor> keep;
  B200QkNormRotary p = rotary_params(a, q, k, qw, kw, keep);
  p.side[0].out = yq.data_ptr();
  p.side[1].out = yk.data_ptr();
  B200_KERNEL_CHECK(b200_qk_norm_rotary_fwd(&p, scope.stream()));
  if (p.bad_flag) report_bad_index("qk_norm_rotary", q);
  return {yq, yk};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> qk_norm_rotary_backward(const Tensor& dyq, const Tensor& dyk, const Tensor& q_in, const Tensor& k_in,
                                                                   const OptTensor& qw_in, const OptTensor& kw_in, const Tensor& cos,
                                                                   const Tensor& sin, const OptTensor& positions, double eps,
                                                                   bool interleaved, bool need_qw, bool need_kw) {
  const RotaryArgs a{q_in, k_in, qw_in, kw_in, cos, sin, positions, eps, interleaved};
  check_rotary_grads(a, dyq, dyk);
  if (!on_device(a.q)) {
    auto [dq, dqw] = host_rotary_bwd(a, a.q, a.qw, dyq);
    auto [dk, dkw] = host_rotary_bwd(a, a.k, a.kw, dyk);
    return {dq, dk, need_qw ? dqw : Tensor(), need_kw ? dkw : Tensor()};
  }
  OpScope scope("qk_norm_rotary_backward", a.q);
  Tensor q = dense_last(a.q), k = dense_last(a.k), gq = dense_last(dyq), gk = dense_last(dyk);
  Tensor dq = fresh(q.sizes(), q), dk = fresh(k.sizes(), k), dqw, dkw;
  const OptTensor qw = dense_weight(a.qw), kw = dense_weight(a.kw);
  if (given(qw) && need_qw) dqw = fresh(qw->sizes(), *qw);
  if (given(kw) && need_kw) dkw = fresh(kw->sizes(), *kw);
  std::vector<Tensor> keep;
  B200QkNormRotary p = rotary_params(a, q, k, qw, kw, keep);
  const Tensor* g[2] = {&gq, &gk};
  const Tensor* d[2] = {&dq, &dk};
  const Tensor* dw[2] = {&dqw, &dkw};
  for (int s = 0; s < 2; ++s) {
    p.side[s].dy = g[s]->data_ptr();
    p.side[s].out = d[s]->data_ptr();
    p.side[s].dweight = dw[s]->defined() ? dw[s]->data_ptr() : nullptr;
    for (int i = 0; i < 3; ++i) p.side[s].dy_stride[i] = g[s]->stride(i);
  }
  Workspace ws((size_t)b200_qk_norm_rotary_workspace(&p), scope);
  B200_KERNEL_CHECK(b200_qk_norm_rotary_bwd(&p, ws.get(), scope.stream()));
  if (p.bad_flag) report_bad_index("qk_norm_rotary_backward", q);
  return {dq, dk, dqw, dkw};
}

OptTensor saved_optional(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// ---- autograd.  Nodes of their own instead of torch::autograd::Function: the call of a small operator is as long as its bookkeeping.
bool wants_grad(std::initializer_list<const Tensor*> leaves) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : leaves)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
const Tensor& or_none(const OptTensor& t) {
  static const Tensor none;
  return given(t) ? *t : none;
}
// Calls go on below autograd.
using Below = at::AutoDispatchBelowADInplaceOrView;
// An output without a tangent would count as one that does not depend on the inputs.
void refuse_tangents(const char* op, std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), op, ": forward-mode derivatives are not implemented");
}
// The node of a gradient.  It leads to what the gradient was computed from, so that whoever differentiates it arrives here instead of
// taking it for a constant.
struct NoSecondDerivative : public torch::autograd::Node {
  std::string op;
  std::string name() const override { return "NoSecondDerivative"; }
  variable_list apply(variable_list&&) override { TORCH_CHECK(false, op, ": the gradient of the gradient is not implemented"); }
};
template <typename N>
std::shared_ptr<N> make_node() {
  return std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
}
// The autograd kernel of a _backward form: calls it below autograd and marks its results.
template <typename F>
auto first_derivative_only(const char* op, std::initializer_list<const Tensor*> inputs, F&& below) {
  refuse_tangents(op, inputs);
  auto grads = [&] {
    Below guard;
    return below();
  }();
  if (wants_grad(inputs)) {
    auto node = make_node<NoSecondDerivative>();
    node->op = op;
    for (const Tensor* t : inputs)
      if (t->defined()) node->add_next_edge(torch::autograd::impl::gradient_edge(*t));
    auto mark = [&](const Tensor& g) {
      if (g.defined()) torch::autograd::set_history(g, node);
    };
    if constexpr (std::is_same_v<std::decay_t<decltype(grads)>, Tensor>) mark(grads);
    else std::apply([&](const auto&... g) { (mark(g), ...); }, grads);
  }
  return grads;
}
SavedVariable save(const Tensor& t) { return SavedVariable(t, /*is_output=*/false); }
template <typename F>
c10::TypedOperatorHandle<F> find_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
// Whether nothing but the kernels looks on (no wrapper of a transform, no subclass, no dispatch mode), so that a shortcut may use the memory.
bool plain(const Tensor& t) { return !at::isTensorSubclassLike(t); }

// Autograd runs a backward on a thread of its own, whose memory does not come from the pool of a graph that the caller is capturing:
// a replay would write to memory that belongs to others by then.  The operators' _backward forms, called by the capturing thread, are fine.
void refuse_captured_backward(const char* op, const Tensor& t) {
  if (!on_device(t) || graphCaptureActive()) return;
  void* queue = getCurrentQueue(t.device().index()).handle();
  int capturing = 0;
  if (queue) TORCH_CHECK(b200_stream_is_capturing(queue, &capturing) == 0, op, ": the queue cannot be asked whether it is captured");
  TORCH_CHECK(!capturing, op, ": a backward pass through autograd cannot be captured into a device graph; capture torch.ops.catch_b200.", op,
              "_backward instead");
}

std::tuple<Tensor, Tensor, Tensor, Tensor> qk_norm_rotary_backward_autograd(const Tensor& dyq, const Tensor& dyk, const Tensor& q, const Tensor& k,
                                                                            const OptTensor& qw, const OptTensor& kw, const Tensor& cos,
                                                                            const Tensor& sin, const OptTensor& positions, double eps,
                                                                            bool interleaved, bool need_qw, bool need_kw) {
  static const auto op = find_op<decltype(qk_norm_rotary_backward)>("catch_b200::qk_norm_rotary_backward");
  return first_derivative_only("qk_norm_rotary_backward", {&dyq, &dyk, &q, &k, &or_none(qw), &or_none(kw), &cos, &sin},
                               [&] { return op.call(dyq, dyk, q, k, qw, kw, cos, sin, positions, eps, interleaved, need_qw, need_kw); });
}

struct RotaryNode : public torch::autograd::Node {
  SavedVariable q, k, qw, kw, cos, sin, positions;
  double eps = 0;
  bool interleaved = false;
  std::string name() const override { return "QkNormRotaryBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* s : {&q, &k, &qw, &kw, &cos, &sin, &positions}) s->reset_data();
  }
  variable_list apply(variable_list&& g) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(4);
    if (!g[0].defined() && !g[1].defined()) return out;
    const Tensor uq = q.unpack(), uk = k.unpack();
    refuse_captured_backward("qk_norm_rotary", uq);
    static const auto op = find_op<decltype(qk_norm_rotary_backward)>("catch_b200::qk_norm_rotary_backward");
    const Tensor gq = g[0].defined() ? g[0] : at::zeros_like(uq, at::MemoryFormat::Contiguous);
    const Tensor gk = g[1].defined() ? g[1] : at::zeros_like(uk, at::MemoryFormat::Contiguous);
    std::tie(out[0], out[1], out[2], out[3]) =
        op.call(gq, gk, uq, uk, saved_optional(qw.unpack()), saved_optional(kw.unpack()), cos.unpack(), sin.unpack(),
                saved_optional(positions.unpack()), eps, interleaved, task_should_compute_output(2), task_should_compute_output(3));
    return out;
  }
};

std::tuple<Tensor, Tensor> qk_norm_rotary_autograd(const Tensor& q, const Tensor& k, const OptTensor& qw, const OptTensor& kw,
                                                   const Tensor& cos, const Tensor& sin, const OptTensor& positions, double eps,
                                                   bool interleaved) {
  std::shared_ptr<RotaryNode> node;
  const Tensor &tqw = or_none(qw), &tkw = or_none(kw);
  refuse_tangents("qk_norm_rotary", {&q, &k, &tqw, &tkw, &cos, &sin});
  TORCH_CHECK(!cos.requires_grad() && !sin.requires_grad(), "qk_norm_rotary: cos and sin are constants, they get no gradient");
  if (wants_grad({&q, &k, &tqw, &tkw})) {
    node = make_node<RotaryNode>();
    node->set_next_edges(torch::autograd::collect_next_edges(q, k, tqw, tkw));
    node->q = save(q); node->k = save(k); node->qw = save(tqw); node->kw = save(tkw);
    node->cos = save(cos); node->sin = save(sin); node->positions = save(or_none(positions));
    node->eps = eps;
    node->interleaved = interleaved;
  }
  static const auto op = find_op<decltype(qk_norm_rotary)>("catch_b200::qk_norm_rotary");
  Tensor yq, yk;
  {
    Below below;
    std::tie(yq, yk) = op.call(q, k, qw, kw, cos, sin, positions, eps, interleaved);
  }
  if (node) {
    torch::autograd::set_history(yq, node);
    torch::autograd::set_history(yk, node);
  }
  return {yq, yk};
}

// ------------------------------------------------------------------------------------------------------ biased softmax
// The smallest distance of every far bucket, in integers: distance d has passed border k of m when
// d^m >= max_distance^k exact^(m - k), which is floor(log(d / exact) / log(max_distance / exact) m) >= k without a rounding.
struct BigInt {
  std::vector<uint32_t> w{1};
  void times(uint32_t f) {
    uint64_t carry = 0;
    for (auto& x : w) {
      carry += (uint64_t)x * f;
      x = (uint32_t)carry;
      carry >>= 32;
    }
    if (carry) w.push_back((uint32_t)carry);
  }
  static BigInt power(uint32_t base, int n) {
    BigInt r;
    for (int i = 0; i < n; ++i) r.times(base);
    return r;
  }
  bool at_least(const BigInt& o) const {
    if (w.size() != o.w.size()) return w.size() > o.w.size();
    for (size_t i = w.size(); i-- > 0;)
      if (w[i] != o.w[i]) return w[i] > o.w[i];
    return true;
  }
};

const B200RelativeBuckets& relative_buckets(int64_t num_buckets, bool bidirectional, int64_t max_distance) {
  static std::mutex mu;
  static std::map<std::tuple<int64_t, bool, int64_t>, B200RelativeBuckets> known;
  std::lock_guard<std::mutex> lk(mu);
  auto it = known.find({num_buckets, bidirectional, max_distance});
  if (it != known.end()) return it->second;
  B200RelativeBuckets r{};
  r.bidirectional = bidirectional;
  r.per_side = (int)(bidirectional ? num_buckets / 2 : num_buckets);
  r.exact = r.per_side / 2;
  r.max_distance = (int)max_distance;
  const int m = r.per_side - r.exact;
  int d = r.exact;
  for (int k = 0; k < m; ++k) {
    BigInt border = BigInt::power((uint32_t)max_distance, k);
    for (int i = 0; i < m - k; ++i) border.times((uint32_t)r.exact);
    while (!BigInt::power((uint32_t)d, m).at_least(border)) ++d;
    r.first[k] = d;
  }
  return known.emplace(std::make_tuple(num_buckets, bidirectional, max_distance), r).first->second;
}
int64_t bucket_of(const B200RelativeBuckets& r, int64_t rel) {
  const int64_t up = r.bidirectional && rel > 0 ? r.per_side : 0, d = r.bidirectional ? std::abs(rel) : std::max<int64_t>(0, -rel);
  if (d < r.exact) return up + d;
  int64_t b = r.exact;
  for (int k = 1; k < r.per_side - r.exact; ++k) b += d >= r.first[k];
  return up + b;
}

struct BiasArgs {
  Tensor scores, table;
  OptTensor mask;
  double scale;
  bool bidirectional;
  int64_t max_distance, query_offset;
};

void check_bias(const BiasArgs& a) {
  const char* op = "relative_bias_softmax";
  TORCH_CHECK(a.scores.dim() == 4, op, ": scores are [batch, heads, queries, keys], got ", a.scores.sizes());
  TORCH_CHECK(f_ok(a.scores.scalar_type()), op, ": scores are float32, bfloat16 or float16, got ", a.scores.scalar_type());
  TORCH_CHECK(a.table.dim() == 2 && a.table.size(1) == a.scores.size(1) && f_ok(a.table.scalar_type()), op,
              ": the table is floating [buckets, heads], got ", a.table.scalar_type(), " ", a.table.sizes(), " for ", a.scores.size(1),
              " heads");
  const int64_t n = a.table.size(0), side = a.bidirectional ? n / 2 : n, far = side - side / 2;
  TORCH_CHECK(side >= 2 && far <= B200_MAX_FAR_BUCKETS && (!a.bidirectional || n % 2 == 0), op, ": between ", a.bidirectional ? 4 : 2,
              " and ", (a.bidirectional ? 4 : 2) * B200_MAX_FAR_BUCKETS, " buckets", a.bidirectional ? ", an even number" : "", ", got ", n);
  TORCH_CHECK(a.max_distance > side / 2 && a.max_distance <= B200_MAX_BIAS_DISTANCE, op, ": max_distance must be above ", side / 2,
              " (the distances with a bucket each) and at most ", B200_MAX_BIAS_DISTANCE, ", got ", a.max_distance);
  const int64_t far_off = int64_t(1) << 30, Lq = a.scores.size(2), Lk = a.scores.size(3);
  TORCH_CHECK(a.query_offset > -far_off && a.query_offset < far_off && Lq < far_off && Lk < far_off, op,
              ": lengths and query_offset must stay below 2^30");
  // slots of distances are 32-bit numbers: reach - query_offset - query + key
  TORCH_CHECK(std::abs(a.query_offset) + std::max(Lq, Lk) < (int64_t(1) << 31) - 2 * B200_MAX_BIAS_DISTANCE, op,
              ": queries and keys lie too far apart: lengths of ", Lq, " and ", Lk, " with query_offset ", a.query_offset);
  TORCH_CHECK(a.scores.size(0) < (int64_t(1) << 31) && a.scores.size(0) * Lq < (int64_t(1) << 31), op,
              ": batch times queries must stay below 2^31");
  TORCH_CHECK(a.scores.size(1) < (int64_t(1) << 31), op, ": the number of heads must stay below 2^31");
  TORCH_CHECK(std::isfinite((float)a.scale), op, ": scale must be finite in fp32, got ", a.scale);
  if (given(a.mask)) {
    TORCH_CHECK(a.mask->scalar_type() == at::kBool || f_ok(a.mask->scalar_type()), op,
                ": the mask is bool (true keeps a key) or floating (added), got ", a.mask->scalar_type());
    TORCH_CHECK(a.mask->dim() <= 4, op, ": the mask has at most four dimensions, got ", a.mask->sizes());
    for (int64_t i = 1; i <= a.mask->dim(); ++i)
      TORCH_CHECK(a.mask->size(-i) == 1 || a.mask->size(-i) == a.scores.size(-i), op, ": the mask ", a.mask->sizes(),
                  " does not broadcast to the scores ", a.scores.sizes());
  }
  check_same_device(op, a.scores, a.table, a.mask);
}

// Host path: logits in fp32 and the bucket of every (query, key).
std::tuple<Tensor, Tensor> host_logits(const BiasArgs& a) {
  const int64_t Lq = a.scores.size(2), Lk = a.scores.size(3);
  const B200RelativeBuckets& rb = relative_buckets(a.table.size(0), a.bidirectional, a.max_distance);
  std::vector<int64_t> of(std::max<int64_t>(0, Lq + Lk - 1));  // by j - i + Lq - 1
  for (size_t x = 0; x < of.size(); ++x) of[x] = bucket_of(rb, (int64_t)x - (Lq - 1) - a.query_offset);
  auto iopt = at::TensorOptions().dtype(at::kLong);
  Tensor line = at::tensor(of, iopt);
  Tensor at = at::arange(Lk, iopt).unsqueeze(0) - at::arange(Lq, iopt).unsqueeze(1) + (Lq - 1);
  Tensor bucket = line.index_select(0, at.reshape({-1})).to(a.scores.device());  // [Lq * Lk]
  Tensor bias = a.table.to(at::kFloat).index_select(0, bucket).view({Lq, Lk, a.table.size(1)}).permute({2, 0, 1});
  Tensor x = a.scores.to(at::kFloat) * a.scale + bias;
  if (given(a.mask)) {
    if (a.mask->scalar_type() == at::kBool) x = x.masked_fill(a.mask->logical_not(), -kInf);
    else x = (x + a.mask->to(at::kFloat)).masked_fill(a.mask->eq(-kInf), -kInf);
  }
  return {x, bucket};
}
Tensor host_probs(const Tensor& x, const Tensor& stats) {
  return at::exp(x - stats.select(-1, 0).unsqueeze(-1)) * stats.select(-1, 1).unsqueeze(-1);  // x = -inf: 0, in a NaN row NaN
}

bool sixteen(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
// The kernels address scores, probabilities and gradients alike: dense, the last dimension innermost, from a 16-byte boundary on.
Tensor score_layout(const Tensor& t) {
  if (t.is_non_overlapping_and_dense() && (t.stride(-1) == 1 || t.size(-1) == 1) && sixteen(t)) return t;
  return t.clone(at::MemoryFormat::Contiguous);
}
Tensor in_layout_of(const Tensor& t, const Tensor& like) {
  if (t.strides() == like.strides() && sixteen(t)) return t;
  return fresh_strided(like).copy_(t);
}

B200BiasSoftmax bias_params(const BiasArgs& a, const Tensor& scores, const Tensor& table) {
  B200BiasSoftmax p{};
  p.scores = scores.data_ptr();
  p.table = table.data_ptr();
  for (int i = 0; i < 3; ++i) p.stride[i] = scores.stride(i);
  p.dtype = to_b200_dtype(scores.scalar_type());
  p.table_dtype = to_b200_dtype(table.scalar_type());
  if (given(a.mask)) {
    const Tensor& m = *a.mask;
    p.mask = m.data_ptr();
    p.mask_dtype = to_b200_dtype(m.scalar_type());
    for (int i = 0; i < 4; ++i) {
      const int64_t d = m.dim() - 4 + i;
      p.mask_stride[i] = d < 0 || m.size(d) == 1 ? 0 : m.stride(d);
    }
  }
  p.B = (int)scores.size(0); p.H = (int)scores.size(1); p.Lq = (int)scores.size(2); p.Lk = (int)scores.size(3);
  p.query_offset = (int)a.query_offset;
  p.scale = (float)a.scale;
  p.buckets = relative_buckets(table.size(0), a.bidirectional, a.max_distance);
  return p;
}

std::vector<int64_t> stats_sizes(const Tensor& scores) { return {scores.size(0), scores.size(1), scores.size(2), 2}; }

// (probabilities, statistics [batch, heads, queries, 2]: the maximum and 1 / sum of each row)
std::tuple<Tensor, Tensor> relative_bias_softmax(const Tensor& scores, const Tensor& table_in, const OptTensor& mask, double scale,
                                                 bool bidirectional, int64_t max_distance, int64_t query_offset) {
  const BiasArgs a{scores, table_in, mask, scale, bidirectional, max_distance, query_offset};
  check_bias(a);
  const std::vector<int64_t> ss = stats_sizes(scores);
  if (!on_device(a.scores)) {
    if (a.scores.numel() == 0) return {at::empty_like(a.scores), at::empty(ss, a.scores.options().dtype(at::kFloat))};
    auto [x, bucket] = host_logits(a);
    Tensor m = std::get<0>(x.max(-1));
    m = m.masked_fill(m.eq(-kInf), 0.0);  // a row with nothing left
    Tensor e = at::exp(x - m.unsqueeze(-1));
    Tensor sum = e.sum(-1), inv = at::where(sum.eq(0), at::zeros_like(sum), sum.reciprocal());
    Tensor stats = at::stack({m, inv}, -1);
    return {host_probs(x, stats).to(a.scores.scalar_type()), stats};
  }
  OpScope scope("relative_bias_softmax", a.scores);
  Tensor s = score_layout(a.scores), table = a.table.contiguous();
  Tensor probs = fresh_strided(s), stats = fresh(ss, at::kFloat, s);
  B200BiasSoftmax p = bias_params(a, s, table);
  p.out = probs.data_ptr();
  p.stats = stats.data_ptr<float>();
  B200_KERNEL_CHECK(b200_bias_softmax_fwd(&p, scope.stream()));
  return {probs, stats};
}

std::tuple<Tensor, Tensor> relative_bias_softmax_meta(const Tensor& scores, const Tensor& table, const OptTensor& mask, double scale,
                                                      bool bidirectional, int64_t max_distance, int64_t query_offset) {
  check_bias({scores, table, mask, scale, bidirectional, max_distance, query_offset});
  return {at::empty_like(scores), at::empty(stats_sizes(scores), scores.options().dtype(at::kFloat))};
}
void check_bias_grads(const BiasArgs& a, const Tensor& grad, const Tensor& stats) {
  check_bias(a);
  const char* op = "relative_bias_softmax_backward";
  TORCH_CHECK(grad.sizes() == a.scores.sizes() && grad.scalar_type() == a.scores.scalar_type(), op,
              ": the gradient has the shape and the dtype of the scores");
  TORCH_CHECK(stats.sizes() == at::IntArrayRef(stats_sizes(a.scores)) && stats.scalar_type() == at::kFloat && stats.is_contiguous(), op,
              ": statistics are the forward's");
  check_same_device(op, a.scores, grad, stats);
}
std::tuple<Tensor, Tensor> relative_bias_softmax_backward_meta(const Tensor& grad, const Tensor& scores, const Tensor& stats, const Tensor& table,
                                                               const OptTensor& mask, double scale, bool bidirectional, int64_t max_distance,
                                                               int64_t query_offset, bool need_table) {
  check_bias_grads({scores, table, mask, scale, bidirectional, max_distance, query_offset}, grad, stats);
  return {at::empty_like(scores), need_table ? at::empty(table.sizes(), table.options()) : Tensor()};
}

std::tuple<Tensor, Tensor> relative_bias_softmax_backward(const Tensor& grad, const Tensor& scores, const Tensor& stats, const Tensor& table_in,
                                                          const OptTensor& mask, double scale, bool bidirectional, int64_t max_distance,
                                                          int64_t query_offset, bool need_table) {
  const BiasArgs a{scores, table_in, mask, scale, bidirectional, max_distance, query_offset};
  check_bias_grads(a, grad, stats);
  if (!on_device(a.scores)) {
    if (a.scores.numel() == 0) return {at::empty_like(a.scores), need_table ? at::zeros_like(a.table) : Tensor()};
    auto [x, bucket] = host_logits(a);
    Tensor p = host_probs(x, stats), g = grad.to(at::kFloat).masked_fill(p.eq(0), 0.0);
    Tensor d = p * (g - (p * g).sum(-1, true)), dt;
    if (need_table) {
      const int64_t H = a.table.size(1);
      dt = at::zeros({a.table.size(0), H}, a.table.options().dtype(at::kDouble).device(at::kCPU));
      dt.index_add_(0, bucket.cpu(), d.cpu().to(at::kDouble).sum(0).permute({1, 2, 0}).reshape({-1, H}));
      dt = dt.to(a.table.scalar_type()).to(a.table.device());
    }
    return {(d * a.scale).to(a.scores.scalar_type()), dt};
  }
  OpScope scope("relative_bias_softmax_backward", a.scores);
  Tensor s = score_layout(a.scores), g = in_layout_of(grad, s), table = a.table.contiguous();
  Tensor ds = fresh_strided(s), pairs = by_pairs(stats), dt;
  B200BiasSoftmax p = bias_params(a, s, table);
  p.grad = g.data_ptr();
  p.out = ds.data_ptr();
  p.stats = pairs.data_ptr<float>();
  if (need_table) {
    dt = fresh(table.sizes(), table);
    p.dtable = dt.data_ptr();
  }
  Workspace ws((size_t)b200_bias_softmax_workspace(&p), scope);
  B200_KERNEL_CHECK(b200_bias_softmax_bwd(&p, ws.get(), scope.stream()));
  return {ds, dt};
}

std::tuple<Tensor, Tensor> relative_bias_softmax_backward_autograd(const Tensor& grad, const Tensor& scores, const Tensor& stats, const Tensor& table,
                                                                   const OptTensor& mask, double scale, bool bidirectional, int64_t max_distance,
                                                                   int64_t query_offset, bool need_table) {
  static const auto op = find_op<decltype(relative_bias_softmax_backward)>("catch_b200::relative_bias_softmax_backward");
  return first_derivative_only("relative_bias_softmax_backward", {&grad, &scores, &stats, &table, &or_none(mask)}, [&] {
    return op.call(grad, scores, stats, table, mask, scale, bidirectional, max_distance, query_offset, need_table);
  });
}

struct BiasNode : public torch::autograd::Node {
  SavedVariable scores, table, mask, stats;
  double scale = 1;
  bool bidirectional = true;
  int64_t max_distance = 0, query_offset = 0;
  std::string name() const override { return "RelativeBiasSoftmaxBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* s : {&scores, &table, &mask, &stats}) s->reset_data();
  }
  variable_list apply(variable_list&& g) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(2);
    if (!g[0].defined()) return out;
    Tensor s = scores.unpack();
    const Tensor t = table.unpack(), m = mask.unpack(), st = stats.unpack();
    // A copy in the kernels' layout stands for the scores, also to whoever differentiates the gradient.
    if (at::GradMode::is_enabled() && !s.requires_grad() && next_edge(0).is_valid()) {
      s = s.detach();
      torch::autograd::impl::set_gradient_edge(s, next_edge(0));
    }
    refuse_captured_backward("relative_bias_softmax", s);
    static const auto op = find_op<decltype(relative_bias_softmax_backward)>("catch_b200::relative_bias_softmax_backward");
    std::tie(out[0], out[1]) =
        op.call(g[0], s, st, t, saved_optional(m), scale, bidirectional, max_distance, query_offset, task_should_compute_output(1));
    return out;
  }
};

std::tuple<Tensor, Tensor> relative_bias_softmax_autograd(const Tensor& scores, const Tensor& table, const OptTensor& mask, double scale,
                                                          bool bidirectional, int64_t max_distance, int64_t query_offset) {
  refuse_tangents("relative_bias_softmax", {&scores, &table, &or_none(mask)});
  TORCH_CHECK(!or_none(mask).defined() || !mask->requires_grad(),
              "relative_bias_softmax: the mask gets no gradient; pass a mask that does not require one");
  static const auto op = find_op<decltype(relative_bias_softmax)>("catch_b200::relative_bias_softmax");
  const bool grad = wants_grad({&scores, &table});
  Tensor probs, stats, laid_out = scores;
  {
    Below below;
    if (grad && scores.dim() == 4 && on_device(scores) && plain(scores)) laid_out = score_layout(scores);  // once for both directions
    std::tie(probs, stats) = op.call(laid_out, table, mask, scale, bidirectional, max_distance, query_offset);
  }
  if (grad) {
    auto node = make_node<BiasNode>();
    node->set_next_edges(torch::autograd::collect_next_edges(scores, table));
    node->scores = save(laid_out); node->table = save(table); node->mask = save(or_none(mask)); node->stats = save(stats);
    node->scale = scale; node->bidirectional = bidirectional; node->max_distance = max_distance; node->query_offset = query_offset;
    torch::autograd::set_history(probs, node);
  }
  return {probs, stats};
}

// -------------------------------------------------------------------------------------------------------- distillation
struct DistillArgs {
  Tensor logits, teacher, index;
  double temperature;
  int64_t reduction;  // at::Reduction: None, Mean, Sum
};

void check_distill(const DistillArgs& a) {
  const char* op = "top_logits_distillation";
  TORCH_CHECK(a.logits.dim() == 2 && f_ok(a.logits.scalar_type()), op, ": logits are float32, bfloat16 or float16 [rows, vocabulary], got ",
              a.logits.scalar_type(), " ", a.logits.sizes());
  TORCH_CHECK(a.teacher.dim() == 2 && a.teacher.size(0) == a.logits.size(0) && f_ok(a.teacher.scalar_type()), op,
              ": the teacher's logits are floating [rows, kept], got ", a.teacher.scalar_type(), " ", a.teacher.sizes());
  TORCH_CHECK(a.index.sizes() == a.teacher.sizes() && (a.index.scalar_type() == at::kLong || a.index.scalar_type() == at::kInt), op,
              ": the teacher's indices are int64 or int32 of the shape of its logits, got ", a.index.scalar_type(), " ", a.index.sizes());
  TORCH_CHECK(a.teacher.size(1) <= B200_DISTILL_MAX_K, op, ": at most ", B200_DISTILL_MAX_K, " logits kept for a row, got ", a.teacher.size(1));
  TORCH_CHECK(a.logits.size(1) >= 1 && a.logits.size(1) < (int64_t(1) << 31) - 8192, op, ": unsupported vocabulary of ", a.logits.size(1));
  TORCH_CHECK(std::isfinite(a.temperature) && a.temperature >= 1e-3 && a.temperature <= 1e3, op, ": temperature must lie between 1e-3 and 1e3, got ",
              a.temperature);
  TORCH_CHECK(a.reduction == at::Reduction::None || a.reduction == at::Reduction::Mean || a.reduction == at::Reduction::Sum, op,
              ": reduction is 0 (none), 1 (mean) or 2 (sum), got ", a.reduction);
  check_same_device(op, a.logits, a.teacher, a.index);
}

// Host path: shares p, sum p log p, which entries and rows are there, clamped indices.
struct HostTeacher {
  Tensor share, plogp, rows, at;
};
HostTeacher host_teacher(const DistillArgs& a) {
  Tensor index = a.index.to(at::kLong), t = a.teacher.to(at::kFloat);
  Tensor inside = index.lt(a.logits.size(1));
  if (flags().async_disable && index.numel() > 0)
    TORCH_CHECK_INDEX(inside.all().item<bool>(), "top_logits_distillation: index out of range");
  Tensor there = index.ge(0).logical_and(inside).logical_and(t.ne(-kInf));
  t = (t / a.temperature).masked_fill(there.logical_not(), -kInf);
  HostTeacher h;
  if (t.size(1) == 0) {
    h.rows = at::zeros({t.size(0)}, t.options().dtype(at::kBool));
    h.share = t; h.plogp = at::zeros({t.size(0)}, t.options()); h.at = index;
    return h;
  }
  h.rows = there.any(1);
  Tensor lp = at::log_softmax(t, 1).masked_fill(there.logical_not(), -kInf);
  h.share = at::exp(lp);
  h.plogp = (h.share * lp).masked_fill(h.share.eq(0), 0.0).sum(1);
  h.at = index.clamp(0, a.logits.size(1) - 1).masked_fill(there.logical_not(), 0);
  return h;
}
Tensor host_distill_grad(const DistillArgs& a, const HostTeacher& h, const Tensor& factor /* [rows] */) {
  Tensor f = (factor * a.temperature).masked_fill(h.rows.logical_not(), 0.0).unsqueeze(1);
  Tensor q = at::softmax(a.logits.to(at::kFloat) / a.temperature, 1) * f;
  q = q.masked_fill(h.rows.logical_not().unsqueeze(1), 0.0);
  if (h.at.size(1) > 0) q = q.scatter_add(1, h.at, -(h.share * f));
  return q.to(a.logits.scalar_type());
}

// Rows of equal distance with a dense last dimension, each element at most once in memory.
Tensor row_layout(const Tensor& t) {
  if ((t.stride(1) == 1 || t.size(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1))) return t;
  return t.contiguous();
}
// An uninitialised tensor whose rows begin at the same place within 16 bytes as those of `t`, which lie `ld` apart: as close
// together as that allows (a token's logits of every sequence may lie a whole sequence apart).
Tensor empty_in_phase(const Tensor& t, int64_t ld) {
  const int64_t es = (int64_t)t.element_size(), vec = 16 / es, phase = (int64_t)(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) / es;
  const int64_t rows = t.size(0), V = t.size(1), apart = V + (ld - V) % vec;
  if (phase == 0 && apart == V) return fresh(t.sizes(), t);
  return fresh({(rows > 0 ? (rows - 1) * apart + V : 0) + phase}, t).as_strided(t.sizes(), {apart, 1}, phase);
}
// The distance of the rows of [N, V] logits or of their gradient.
int64_t row_distance(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// Whether `out` has the type of `t` and every row at the same place within 16 bytes.
bool in_phase(const Tensor& out, const Tensor& t) {
  return out.sizes() == t.sizes() && out.scalar_type() == t.scalar_type() &&
         (row_distance(out) - row_distance(t)) * (int64_t)t.element_size() % 16 == 0 &&
         (reinterpret_cast<uintptr_t>(out.data_ptr()) - reinterpret_cast<uintptr_t>(t.data_ptr())) % 16 == 0;
}

B200Distill distill_params(const DistillArgs& a, const Tensor& z, const Tensor& teacher, const Tensor& index) {
  B200Distill p{};
  p.logits = z.data_ptr(); p.teacher = teacher.data_ptr(); p.index = index.data_ptr();
  p.N = z.size(0); p.V = z.size(1); p.K = (int)teacher.size(1);
  p.ld = row_distance(z);
  p.teacher_ld = teacher.size(1); p.index_ld = index.size(1);
  p.dtype = to_b200_dtype(z.scalar_type());
  p.teacher_dtype = to_b200_dtype(teacher.scalar_type());
  p.index_dtype = to_b200_dtype(index.scalar_type());
  p.temperature = (float)a.temperature;
  p.inv_temperature = (float)(1.0 / a.temperature);
  p.bad_flag = checked_index_flag(z);
  return p;
}

// (loss, statistics [rows, 2], number of rows that count with the kernels' scratch behind it, gradient of the logits for a factor of 1 or undefined)
std::tuple<Tensor, Tensor, Tensor, Tensor> distill_fwd(const DistillArgs& a, bool need_grad) {
  check_distill(a);
  const bool mean = a.reduction == at::Reduction::Mean, each = a.reduction == at::Reduction::None;
  const int64_t N = a.logits.size(0);
  auto fopt = a.logits.options().dtype(at::kFloat);
  if (!on_device(a.logits)) {
    HostTeacher h = host_teacher(a);
    Tensor z = a.logits.to(at::kFloat) / a.temperature, lse = at::logsumexp(z, 1);
    Tensor rows = h.plogp;
    if (h.at.size(1) > 0)
      rows = rows - (h.share * at::log_softmax(z, 1).gather(1, h.at)).masked_fill(h.share.eq(0), 0.0).sum(1);
    rows = (rows * (a.temperature * a.temperature)).masked_fill(h.rows.logical_not(), 0.0);
    Tensor count = mean ? h.rows.sum().to(at::kFloat).reshape({1}) : at::ones({1}, fopt);
    Tensor loss = each ? rows : rows.sum() / count.clamp_min(1.0).squeeze(0);
    Tensor grad = need_grad && !each ? host_distill_grad(a, h, count.clamp_min(1.0).reciprocal().expand({N})) : Tensor();
    return {loss, at::stack({lse, lse}, 1), count, grad};
  }
  OpScope scope("top_logits_distillation", a.logits);
  Tensor z = row_layout(a.logits), teacher = a.teacher.contiguous(), index = a.index.contiguous();
  Tensor rows = fresh({N}, at::kFloat, z), stats = fresh({N, 2}, at::kFloat, z), count = fresh({1 + B200_DISTILL_SCRATCH}, at::kFloat, z);  // (count, scratch)
  Tensor loss = each ? rows : fresh({}, at::kFloat, z), grad;
  B200Distill p = distill_params(a, z, teacher, index);
  p.row_loss = rows.data_ptr<float>();
  p.stats = stats.data_ptr<float>();
  p.loss = each ? nullptr : loss.data_ptr<float>();
  p.count = mean ? count.data_ptr<float>() : nullptr;
  p.scratch = reinterpret_cast<unsigned*>(count.data_ptr<float>() + 1);
  // The gradient for a factor of 1, while the row is in the caches.  Not in half precision: its training scales the loss, so that the
  // factor is another one, and a gradient rounded before the scaling would lose what the scaling is there to keep.
  if (need_grad && !each && z.scalar_type() != at::kHalf) {
    grad = empty_in_phase(z, p.ld);
    p.dlogits = grad.data_ptr();
    p.dlogits_ld = row_distance(grad);
  }
  B200_KERNEL_CHECK(b200_distill_fwd(&p, scope.stream()));
  if (p.bad_flag) report_bad_index("top_logits_distillation", z);
  return {loss, stats, count, grad};
}

void check_distill_grads(const DistillArgs& a, const Tensor& grad, const Tensor& stats, const Tensor& count) {
  check_distill(a);
  const char* op = "top_logits_distillation_backward";
  const bool each = a.reduction == at::Reduction::None;
  const int64_t N = a.logits.size(0);
  TORCH_CHECK(each ? (grad.dim() == 1 && grad.size(0) == N) : grad.numel() == 1, op, ": the gradient has the shape of the loss, got ",
              grad.sizes());
  TORCH_CHECK(stats.dim() == 2 && stats.size(0) == N && stats.size(1) == 2 && stats.scalar_type() == at::kFloat && stats.is_contiguous() &&
                  count.numel() >= 1 && count.scalar_type() == at::kFloat,
              op, ": statistics are the forward's");
  check_same_device(op, a.logits, grad, stats, count);
}

// The gradient of the logits; `ready`: the forward's, which is taken when the factor turns out to be 1.
Tensor distill_bwd(const DistillArgs& a, const Tensor& grad, const Tensor& stats, const Tensor& count, const Tensor& ready) {
  check_distill_grads(a, grad, stats, count);
  const bool mean = a.reduction == at::Reduction::Mean, each = a.reduction == at::Reduction::None;
  const int64_t N = a.logits.size(0);
  if (!on_device(a.logits))
    return host_distill_grad(a, host_teacher(a), grad.to(at::kFloat).reshape({-1}).expand({N}) / count.to(at::kFloat).clamp_min(1.0));
  OpScope scope("top_logits_distillation_backward", a.logits);
  Tensor z = row_layout(a.logits), teacher = a.teacher.contiguous(), index = a.index.contiguous(), g = grad.to(at::kFloat), pairs = by_pairs(stats);
  B200Distill p = distill_params(a, z, teacher, index);
  // What backward() is given may lie elsewhere than what the forward saw (hooks on saved tensors, a recomputed forward): the kernel
  // takes the rows' place within 16 bytes from the logits.
  const bool keep = ready.defined() && in_phase(ready, z);
  Tensor out = keep ? ready : empty_in_phase(z, p.ld);
  p.stats = pairs.data_ptr<float>();
  p.count = mean ? count.data_ptr<float>() : nullptr;
  p.dlogits = out.data_ptr();
  p.dlogits_ld = row_distance(out);
  p.grad = g.data_ptr<float>();
  p.grad_per_row = each;
  p.grad_ld = each && N > 1 ? g.stride(0) : 0;
  p.skip_factor_one = keep;
  B200_KERNEL_CHECK(b200_distill_bwd(&p, scope.stream()));
  if (p.bad_flag) report_bad_index("top_logits_distillation_backward", z);
  return out;
}

Tensor top_logits_distillation(const Tensor& logits, const Tensor& teacher, const Tensor& index, double temperature, int64_t reduction,
                               bool /*early_gradient*/) {
  return std::get<0>(distill_fwd({logits, teacher, index, temperature, reduction}, false));
}
std::tuple<Tensor, Tensor, Tensor> top_logits_distillation_stats(const Tensor& logits, const Tensor& teacher, const Tensor& index,
                                                                 double temperature, int64_t reduction) {
  auto [loss, stats, count, ready] = distill_fwd({logits, teacher, index, temperature, reduction}, false);
  count = count.narrow(0, 0, 1);  // (behind it: the kernels' scratch)
  if (reduction != at::Reduction::Mean || logits.size(0) == 0) count.fill_(reduction != at::Reduction::Mean);
  return {loss, stats, count};
}
Tensor top_logits_distillation_backward(const Tensor& grad, const Tensor& logits, const Tensor& stats, const Tensor& count, const Tensor& teacher,
                                        const Tensor& index, double temperature, int64_t reduction) {
  return distill_bwd({logits, teacher, index, temperature, reduction}, grad, stats, count, Tensor());
}
Tensor top_logits_distillation_meta(const Tensor& logits, const Tensor& teacher, const Tensor& index, double temperature, int64_t reduction,
                                    bool early_gradient) {
  check_distill({logits, teacher, index, temperature, reduction});
  auto opt = logits.options().dtype(at::kFloat);
  return reduction == at::Reduction::None ? at::empty({logits.size(0)}, opt) : at::empty({}, opt);
}
std::tuple<Tensor, Tensor, Tensor> top_logits_distillation_stats_meta(const Tensor& logits, const Tensor& teacher, const Tensor& index,
                                                                      double temperature, int64_t reduction) {
  Tensor loss = top_logits_distillation_meta(logits, teacher, index, temperature, reduction, false);
  return {loss, at::empty({logits.size(0), 2}, loss.options()), at::empty({1}, loss.options())};
}
Tensor top_logits_distillation_backward_meta(const Tensor& grad, const Tensor& logits, const Tensor& stats, const Tensor& count, const Tensor& teacher,
                                             const Tensor& index, double temperature, int64_t reduction) {
  check_distill_grads({logits, teacher, index, temperature, reduction}, grad, stats, count);
  return at::empty(logits.sizes(), logits.options());
}

Tensor top_logits_distillation_backward_autograd(const Tensor& grad, const Tensor& logits, const Tensor& stats, const Tensor& count,
                                                 const Tensor& teacher, const Tensor& index, double temperature, int64_t reduction) {
  static const auto op = find_op<decltype(top_logits_distillation_backward)>("catch_b200::top_logits_distillation_backward");
  return first_derivative_only("top_logits_distillation_backward", {&grad, &logits, &stats, &count, &teacher},
                               [&] { return op.call(grad, logits, stats, count, teacher, index, temperature, reduction); });
}

struct DistillNode : public torch::autograd::Node {
  SavedVariable logits, teacher, index, stats, count;
  Tensor ready;  // the gradient for a factor of 1, handed out once: a second pass over a retained graph writes one of its own
  double temperature = 1;
  int64_t reduction = 0;
  std::string name() const override { return "TopLogitsDistillationBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* s : {&logits, &teacher, &index, &stats, &count}) s->reset_data();
    ready = Tensor();
  }
  variable_list apply(variable_list&& g) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(1);
    if (!g[0].defined()) return out;
    const Tensor z = logits.unpack(), t = teacher.unpack(), i = index.unpack(), st = stats.unpack(), n = count.unpack();
    refuse_captured_backward("top_logits_distillation", z);
    static const auto op = find_op<decltype(top_logits_distillation_backward)>("catch_b200::top_logits_distillation_backward");
    // The early gradient, if nobody but the kernels looks on; it is a constant to whoever differentiates once more.
    if (ready.defined() && !at::GradMode::is_enabled() && plain(z) && plain(g[0])) {
      refuse_tangents("top_logits_distillation", {&g[0]});
      Below below;
      out[0] = distill_bwd({z, t, i, temperature, reduction}, g[0], st, n, std::exchange(ready, Tensor()));
    } else {
      out[0] = op.call(g[0], z, st, n, t, i, temperature, reduction);
    }
    return out;
  }
};

// Records the node of a loss.
void record_distill(const Tensor& loss, const Tensor& logits, const Tensor& teacher, const Tensor& index, const Tensor& stats, const Tensor& count,
                    Tensor ready, double temperature, int64_t reduction) {
  auto node = make_node<DistillNode>();
  node->set_next_edges(torch::autograd::collect_next_edges(logits));
  node->logits = save(logits); node->teacher = save(teacher); node->index = save(index); node->stats = save(stats); node->count = save(count);
  node->ready = std::move(ready);
  node->temperature = temperature;
  node->reduction = reduction;
  torch::autograd::set_history(loss, node);
}
void refuse_teacher_grads(const Tensor& logits, const Tensor& teacher) {
  refuse_tangents("top_logits_distillation", {&logits, &teacher});
  TORCH_CHECK(!teacher.requires_grad(), "top_logits_distillation: the teacher's logits get no gradient; detach them");
}
std::tuple<Tensor, Tensor, Tensor> top_logits_distillation_stats_autograd(const Tensor& logits, const Tensor& teacher, const Tensor& index,
                                                                          double temperature, int64_t reduction) {
  refuse_teacher_grads(logits, teacher);
  static const auto op = find_op<decltype(top_logits_distillation_stats)>("catch_b200::top_logits_distillation_stats");
  Tensor loss, stats, count;
  {
    Below below;
    std::tie(loss, stats, count) = op.call(logits, teacher, index, temperature, reduction);
  }
  if (wants_grad({&logits})) record_distill(loss, logits, teacher, index, stats, count, Tensor(), temperature, reduction);
  return {loss, stats, count};
}
Tensor top_logits_distillation_autograd(const Tensor& logits, const Tensor& teacher, const Tensor& index, double temperature,
                                        int64_t reduction, bool early_gradient) {
  if (!plain(logits) || !plain(teacher) || !plain(index)) {  // an early gradient would be a constant to whatever else looks on
    static const auto op = find_op<decltype(top_logits_distillation_stats)>("catch_b200::top_logits_distillation_stats");
    return std::get<0>(op.call(logits, teacher, index, temperature, reduction));
  }
  refuse_teacher_grads(logits, teacher);
  const bool grad = wants_grad({&logits});
  Tensor loss, stats, count, ready;
  {
    Below below;
    std::tie(loss, stats, count, ready) = distill_fwd({logits, teacher, index, temperature, reduction}, grad && early_gradient);
  }
  if (grad) record_distill(loss, logits, teacher, index, stats, count, ready, temperature, reduction);
  return loss;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(catch_b200, m) {
  m.def("qk_norm_rotary(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor cos, Tensor sin, Tensor? positions=None, "
        "float eps=1e-06, bool interleaved=False) -> (Tensor, Tensor)");
  m.def("qk_norm_rotary_backward(Tensor grad_q, Tensor grad_k, Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor cos, "
        "Tensor sin, Tensor? positions, float eps, bool interleaved, bool need_q_weight=True, bool need_k_weight=True) -> "
        "(Tensor, Tensor, Tensor, Tensor)");
  // (probabilities, statistics of the rows for the backward)
  m.def("relative_bias_softmax(Tensor scores, Tensor table, Tensor? mask=None, float scale=1.0, bool bidirectional=True, "
        "int max_distance=128, int query_offset=0) -> (Tensor, Tensor)");
  m.def("relative_bias_softmax_backward(Tensor grad, Tensor scores, Tensor stats, Tensor table, Tensor? mask, float scale, "
        "bool bidirectional, int max_distance, int query_offset, bool need_table) -> (Tensor, Tensor)");
  // reduction: 0 a loss for each row, 1 their mean over the rows with entries, 2 their sum; early_gradient: the forward writes the
  // gradient for a factor of 1, where one is wanted
  m.def("top_logits_distillation(Tensor logits, Tensor teacher_logits, Tensor teacher_index, float temperature=1.0, int reduction=1, "
        "bool early_gradient=True) -> Tensor");
  // the loss with what its backward needs (statistics of the rows, number of rows that count), and that backward
  m.def("top_logits_distillation_stats(Tensor logits, Tensor teacher_logits, Tensor teacher_index, float temperature, int reduction) "
        "-> (Tensor, Tensor, Tensor)");
  m.def("top_logits_distillation_backward(Tensor grad, Tensor logits, Tensor stats, Tensor count, Tensor teacher_logits, "
        "Tensor teacher_index, float temperature, int reduction) -> Tensor");
}

TORCH_LIBRARY_IMPL(catch_b200, CompositeExplicitAutograd, m) {
  m.impl("top_logits_distillation_stats", TORCH_FN(top_logits_distillation_stats));
  m.impl("top_logits_distillation_backward", TORCH_FN(top_logits_distillation_backward));
  m.impl("qk_norm_rotary", TORCH_FN(qk_norm_rotary));
  m.impl("qk_norm_rotary_backward", TORCH_FN(qk_norm_rotary_backward));
  m.impl("relative_bias_softmax", TORCH_FN(relative_bias_softmax));
  m.impl("relative_bias_softmax_backward", TORCH_FN(relative_bias_softmax_backward));
  m.impl("top_logits_distillation", TORCH_FN(top_logits_distillation));
}

TORCH_LIBRARY_IMPL(catch_b200, Meta, m) {
  m.impl("qk_norm_rotary", TORCH_FN(qk_norm_rotary_meta));
  m.impl("qk_norm_rotary_backward", TORCH_FN(qk_norm_rotary_backward_meta));
  m.impl("relative_bias_softmax", TORCH_FN(relative_bias_softmax_meta));
  m.impl("relative_bias_softmax_backward", TORCH_FN(relative_bias_softmax_backward_meta));
  m.impl("top_logits_distillation", TORCH_FN(top_logits_distillation_meta));
  m.impl("top_logits_distillation_stats", TORCH_FN(top_logits_distillation_stats_meta));
  m.impl("top_logits_distillation_backward", TORCH_FN(top_logits_distillation_backward_meta));
}

TORCH_LIBRARY_IMPL(catch_b200, Autograd, m) {
  m.impl("qk_norm_rotary_backward", TORCH_FN(qk_norm_rotary_backward_autograd));
  m.impl("relative_bias_softmax_backward", TORCH_FN(relative_bias_softmax_backward_autograd));
  m.impl("top_logits_distillation_backward", TORCH_FN(top_logits_distillation_backward_autograd));
  m.impl("top_logits_distillation_stats", TORCH_FN(top_logits_distillation_stats_autograd));
  m.impl("qk_norm_rotary", TORCH_FN(qk_norm_rotary_autograd));
  m.impl("relative_bias_softmax", TORCH_FN(relative_bias_softmax_autograd));
  m.impl("top_logits_distillation", TORCH_FN(top_logits_distillation_autograd));
}

}  // namespace ops
}  // namespace catch_b200
