// The transformer-step operators of include/twg.h on webgpu tensors: webgpu::norm_rope,
// webgpu::token_logprobs, webgpu::dropout, each with its gradient, and aten::dropout (F.dropout,
// nn.Dropout), which ATen would compose of bernoulli_ and a stored mask.
//
// They have no counterpart in the reference, whose backend registers no autograd formulas
// (csrc/ops/webgpu_ops.cpp:63-66); these bring their own, at the AutogradPrivateUse1 key.  The
// formulas reach memory only through the dispatcher (the operators whose names start with an underscore
// are theirs), so that fake tensors, tracers and dispatch modes see every step; what a step
// gives for fake tensors is in torch_webgpu/fakes.py.
#include <ATen/EmptyTensor.h>
#include <ATen/MemoryOverlap.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <atomic>
#include <mutex>

#include "twg_torch.h"

namespace torch_webgpu {

namespace {
// State of the backend's generator: the seed and the offset the next dropout call takes.
std::mutex g_rng_lock;
uint64_t g_rng_seed = 67280421310721ull;  // torch's own default seed
uint64_t g_rng_offset = 0;
}  // namespace

void set_rng_state(uint64_t seed, uint64_t offset) {
  std::lock_guard<std::mutex> hold(g_rng_lock);
  g_rng_seed = seed;
  g_rng_offset = offset;
}
void get_rng_state(uint64_t *seed, uint64_t *offset) {
  std::lock_guard<std::mutex> hold(g_rng_lock);
  *seed = g_rng_seed;
  *offset = g_rng_offset;
}

namespace ops {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;
typedef std::optional<at::Tensor> MaybeTensor;

const at::Tensor &or_none(const MaybeTensor &t) {
  static const at::Tensor none;
  return t.has_value() ? *t : none;
}

void require_webgpu(const at::Tensor &t, const char *op, const char *what) {
  TORCH_CHECK(!t.defined() || is_webgpu(t), "webgpu ", op, ": ", what, " must be a webgpu tensor, got ", t.device());
}

int float_dtype(const at::Tensor &t, const char *op, const char *what) {
  const auto s = t.scalar_type();
  TORCH_CHECK(s == at::kHalf || s == at::kBFloat16 || s == at::kFloat, "webgpu ", op, ": ", what,
              " must be float16, bfloat16 or float32, got ", s);
  return twg_dtype_of(s);
}

void *ptr(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

at::Tensor unit_last(const at::Tensor &t) {
  return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

template <typename Fn>
c10::TypedOperatorHandle<Fn> handle(const char *name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Fn>();
}

// A gradient that is itself to be differentiated (create_graph=True) would silently be a constant.
void once(const char *op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "webgpu ", op, " has no second derivative (create_graph=True)");
}

// ------------------------------------------------------------------- norm_rope

struct RopeInputs {
  at::Tensor q, k, positions, inv_freq, q_weight, k_weight;
  std::optional<double> eps;
  std::vector<int64_t> pair_axis;
  bool adjacent = false;
};

// The geometry that the forward and the backward call share, checked.
twg_norm_rope_t rope_args(const RopeInputs &in) {
  const char *op = "norm_rope";
  require_webgpu(in.q, op, "q");
  require_webgpu(in.k, op, "k");
  require_webgpu(in.positions, op, "positions");
  require_webgpu(in.inv_freq, op, "inv_freq");
  require_webgpu(in.q_weight, op, "q_weight");
  require_webgpu(in.k_weight, op, "k_weight");
  TORCH_CHECK(in.q.dim() == 4, "webgpu norm_rope: q must be [batch, tokens, heads, head_dim], got ", in.q.sizes());
  const int64_t B = in.q.size(0), T = in.q.size(1), D = in.q.size(3);
  twg_norm_rope_t d{};
  d.dtype = float_dtype(in.q, op, "q");
  if (in.k.defined())
    TORCH_CHECK(in.k.dim() == 4 && in.k.size(0) == B && in.k.size(1) == T && in.k.size(3) == D &&
                    in.k.scalar_type() == in.q.scalar_type(),
                "webgpu norm_rope: k must have q's dtype and shape up to the number of heads, got ", in.k.sizes(), " beside ",
                in.q.sizes());
  TORCH_CHECK(in.inv_freq.dim() == 1 && in.inv_freq.scalar_type() == at::kFloat && in.inv_freq.is_contiguous(),
              "webgpu norm_rope: inv_freq must be a contiguous float32 vector, one entry per rotated pair");
  const int64_t pairs = in.inv_freq.size(0);
  TORCH_CHECK(D <= TWG_ROPE_MAX_HEAD_DIM && D % 2 == 0 && 2 * pairs <= D, "webgpu norm_rope: head_dim must be even, at most ",
              TWG_ROPE_MAX_HEAD_DIM, " and hold 2 * len(inv_freq) elements, got ", D, " and ", pairs, " pairs");
  const auto pt = in.positions.scalar_type();
  TORCH_CHECK(pt == at::kInt || pt == at::kLong || pt == at::kFloat,
              "webgpu norm_rope: positions must be int32, int64 or float32, got ", pt);
  const int64_t nd = in.positions.dim();
  TORCH_CHECK(nd >= 1 && nd <= 3 && in.positions.size(nd - 1) == T && (nd < 2 || in.positions.size(nd - 2) == B),
              "webgpu norm_rope: positions must be [tokens], [batch, tokens] or [axes, batch, tokens], got ",
              in.positions.sizes());
  const int64_t axes = nd == 3 ? in.positions.size(0) : 1;
  TORCH_CHECK(axes >= 1 && axes <= TWG_ROPE_MAX_AXES, "webgpu norm_rope: 1 to ", TWG_ROPE_MAX_AXES, " position axes, got ", axes);
  TORCH_CHECK(in.pair_axis.empty() ? axes == 1 || pairs == 0 : (int64_t)in.pair_axis.size() == pairs,
              "webgpu norm_rope: pair_axis must name a position axis for each rotated pair");
  for (size_t i = 0; i < in.pair_axis.size(); ++i) {
    TORCH_CHECK(in.pair_axis[i] >= 0 && in.pair_axis[i] < axes, "webgpu norm_rope: pair_axis names axis ", in.pair_axis[i],
                " of ", axes);
    d.pair_axis[i] = (uint8_t)in.pair_axis[i];
  }
  d.weight_dtype = d.dtype;
  const at::Tensor *weights[2] = {&in.q_weight, &in.k_weight};
  for (const at::Tensor *w : weights) {
    if (!w->defined()) continue;
    TORCH_CHECK(in.eps.has_value(), "webgpu norm_rope: weights without a norm (eps is None)");
    TORCH_CHECK(w->dim() == 1 && w->size(0) == D && w->is_contiguous() &&
                    (w->scalar_type() == at::kFloat || w->scalar_type() == in.q.scalar_type()),
                "webgpu norm_rope: a norm weight must be a contiguous vector [head_dim] of q's dtype or float32");
    d.weight_dtype = twg_dtype_of(w->scalar_type());
  }
  if (in.q_weight.defined() && in.k_weight.defined())
    TORCH_CHECK(in.q_weight.scalar_type() == in.k_weight.scalar_type(), "webgpu norm_rope: norm weights of two dtypes");
  d.position_dtype = twg_dtype_of(pt);
  d.norm = in.eps.has_value();
  d.eps = (float)in.eps.value_or(0.0);
  TORCH_CHECK(!d.norm || (d.eps >= 0 && std::isfinite(d.eps)), "webgpu norm_rope: eps must be finite and not negative");
  d.adjacent = in.adjacent;
  d.n_axes = (int32_t)axes;
  d.head_dim = (int32_t)D;
  d.rot_dim = (int32_t)(2 * pairs);
  d.batch = B;
  d.tokens = T;
  d.positions = in.positions.data_ptr();
  d.inv_freq = static_cast<const float *>(in.inv_freq.data_ptr());
  d.pos_stride[0] = nd == 3 ? in.positions.stride(0) : 0;
  d.pos_stride[1] = nd >= 2 ? in.positions.stride(nd - 2) : 0;
  d.pos_stride[2] = in.positions.stride(nd - 1);
  return d;
}

void set_strides(int64_t *to, const at::Tensor &t) {
  for (int i = 0; i < 3; ++i) to[i] = t.stride(i);
}

// The result keeps the order in which x's heads are stored where that leaves head_dim dense.
at::Tensor heads_like(const at::Tensor &x) {
  at::Tensor out = at::empty_like(x, x.options(), c10::MemoryFormat::Preserve);
  return x.size(3) <= 1 || out.stride(3) == 1 ? out : at::empty(x.sizes(), x.options());
}

variable_list norm_rope_run(const RopeInputs &in) {
  twg_norm_rope_t d = rope_args(in);
  variable_list outs, keep;
  const at::Tensor *xs[2] = {&in.q, &in.k}, *ws[2] = {&in.q_weight, &in.k_weight};
  for (int i = 0; i < 2; ++i) {
    if (!xs[i]->defined()) continue;
    const at::Tensor x = unit_last(*xs[i]);
    at::Tensor out = heads_like(x);
    twg_rope_part_t &p = d.part[i];
    p.heads = x.size(2);
    p.x = x.data_ptr();
    p.out = out.data_ptr();
    p.weight = ptr(*ws[i]);
    set_strides(p.x_stride, x);
    set_strides(p.out_stride, out);
    keep.push_back(x);
    outs.push_back(out);
  }
  TWG_CHECK(twg_norm_rope(&d, nullptr));
  return outs;
}

// Gradients of q, k and their weights; undefined where nothing flows back or nothing is asked for.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> norm_rope_gradients(
    const MaybeTensor &dq, const MaybeTensor &dk, const at::Tensor &q, const MaybeTensor &k, const at::Tensor &positions,
    const at::Tensor &inv_freq, const MaybeTensor &q_weight, const MaybeTensor &k_weight, std::optional<double> eps,
    at::IntArrayRef pair_axis, bool adjacent, bool q_weight_grad, bool k_weight_grad) {
  const RopeInputs in{q, or_none(k), positions, inv_freq, or_none(q_weight), or_none(k_weight), eps, pair_axis.vec(), adjacent};
  const at::Tensor *dys[2] = {&or_none(dq), &or_none(dk)}, *xs[2] = {&in.q, &in.k}, *ws[2] = {&in.q_weight, &in.k_weight};
  const bool weight_grads[2] = {q_weight_grad, k_weight_grad};
  twg_norm_rope_t d = rope_args(in);
  at::Tensor out[4];
  variable_list keep;
  for (int i = 0; i < 2; ++i) {
    if (!xs[i]->defined() || !dys[i]->defined()) continue;  // nothing flows back
    const at::Tensor x = unit_last(*xs[i]), dy = unit_last(*dys[i]);
    TORCH_CHECK(is_webgpu(dy) && dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type(),
                "webgpu norm_rope: an incoming gradient must have the dtype and shape of its result");
    at::Tensor dx = heads_like(x);
    twg_rope_part_t &p = d.part[i];
    p.heads = x.size(2);
    p.x = x.data_ptr();
    p.dy = dy.data_ptr();
    p.out = dx.data_ptr();
    p.weight = ptr(*ws[i]);
    set_strides(p.x_stride, x);
    set_strides(p.dy_stride, dy);
    set_strides(p.out_stride, dx);
    if (weight_grads[i]) {
      out[2 + i] = at::empty(ws[i]->sizes(), ws[i]->options());
      p.dweight = out[2 + i].data_ptr();
    }
    keep.push_back(x);
    keep.push_back(dy);
    out[i] = dx;
  }
  const size_t need = twg_norm_rope_backward_scratch_bytes(&d);
  at::Tensor scratch;
  if (need) scratch = at::empty({(int64_t)(need / 4)}, in.q.options().dtype(at::kFloat));
  TWG_CHECK(twg_norm_rope_backward(&d, ptr(scratch), need, nullptr));
  return {out[0], out[1], out[2], out[3]};
}

std::vector<at::Tensor> norm_rope(const at::Tensor &q, const MaybeTensor &k, const at::Tensor &positions,
                                  const at::Tensor &inv_freq, const MaybeTensor &q_weight, const MaybeTensor &k_weight,
                                  std::optional<double> eps, at::OptionalIntArrayRef pair_axis, bool adjacent);

struct NormRope : torch::autograd::Function<NormRope> {
  static variable_list forward(AutogradContext *ctx, const at::Tensor &q, const MaybeTensor &k, const at::Tensor &positions,
                               const at::Tensor &inv_freq, const MaybeTensor &q_weight, const MaybeTensor &k_weight,
                               std::optional<double> eps, std::vector<int64_t> pair_axis, bool adjacent) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = handle<decltype(norm_rope)>("webgpu::norm_rope");
    variable_list outs = op.call(q, k, positions, inv_freq, q_weight, k_weight, eps, at::IntArrayRef(pair_axis), adjacent);
    const at::Tensor &wq = or_none(q_weight), &wk = or_none(k_weight);
    ctx->save_for_backward({q, or_none(k), positions, inv_freq, wq, wk});
    ctx->saved_data["norm"] = eps.has_value();
    ctx->saved_data["eps"] = eps.value_or(0.0);
    ctx->saved_data["pair_axis"] = pair_axis;
    ctx->saved_data["adjacent"] = adjacent;
    // (needs_input_grad counts the tensors that are there, not the arguments)
    ctx->saved_data["weight_grads"] =
        std::vector<int64_t>{wq.defined() && wq.requires_grad(), wk.defined() && wk.requires_grad()};
    ctx->set_materialize_grads(false);
    return outs;
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    once("norm_rope");
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = handle<decltype(norm_rope_gradients)>("webgpu::_norm_rope_backward");
    const variable_list saved = ctx->get_saved_variables();
    const auto maybe = [](const at::Tensor &t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); };
    const std::vector<int64_t> pair_axis = ctx->saved_data["pair_axis"].toIntVector();
    const std::vector<int64_t> weight_grads = ctx->saved_data["weight_grads"].toIntVector();
    std::optional<double> eps;
    if (ctx->saved_data["norm"].toBool()) eps = ctx->saved_data["eps"].toDouble();
    const auto g = op.call(maybe(grads[0]), grads.size() > 1 ? maybe(grads[1]) : MaybeTensor(), saved[0], maybe(saved[1]),
                           saved[2], saved[3], maybe(saved[4]), maybe(saved[5]), eps, pair_axis,
                           ctx->saved_data["adjacent"].toBool(), weight_grads[0] != 0, weight_grads[1] != 0);
    variable_list out(9);
    std::tie(out[0], out[1], out[4], out[5]) = g;
    return out;
  }
};

std::vector<int64_t> axis_list(at::OptionalIntArrayRef a) {
  return a.has_value() ? a->vec() : std::vector<int64_t>();
}

std::vector<at::Tensor> norm_rope(const at::Tensor &q, const MaybeTensor &k, const at::Tensor &positions,
                                  const at::Tensor &inv_freq, const MaybeTensor &q_weight, const MaybeTensor &k_weight,
                                  std::optional<double> eps, at::OptionalIntArrayRef pair_axis, bool adjacent) {
  return norm_rope_run(RopeInputs{q, or_none(k), positions, inv_freq, or_none(q_weight), or_none(k_weight), eps,
                                  axis_list(pair_axis), adjacent});
}
std::vector<at::Tensor> norm_rope_autograd(const at::Tensor &q, const MaybeTensor &k, const at::Tensor &positions,
                                           const at::Tensor &inv_freq, const MaybeTensor &q_weight,
                                           const MaybeTensor &k_weight, std::optional<double> eps,
                                           at::OptionalIntArrayRef pair_axis, bool adjacent) {
  return NormRope::apply(q, k, positions, inv_freq, q_weight, k_weight, eps, axis_list(pair_axis), adjacent);
}

// -------------------------------------------------------------- token_logprobs

struct Logprobs {
  at::Tensor logits, targets;  // [rows, vocab], [rows]
  at::Tensor logprob, entropy, row_max, row_sum, top, ids;
};

twg_token_logprobs_t logprob_args(const at::Tensor &logits, const at::Tensor &targets, double scale, int64_t ignore_index) {
  twg_token_logprobs_t d{};
  d.dtype = twg_dtype_of(logits.scalar_type());
  d.target_dtype = twg_dtype_of(targets.scalar_type());
  d.rows = logits.size(0);
  d.vocab = logits.size(1);
  d.row_stride = logits.stride(0);
  d.logits = logits.data_ptr();
  d.targets = targets.data_ptr();
  d.ignore_index = ignore_index;
  d.scale = (float)scale;
  return d;
}

Logprobs token_logprobs_run(const at::Tensor &logits, const at::Tensor &targets, int64_t top_k, double scale,
                            int64_t ignore_index) {
  const char *op = "token_logprobs";
  require_webgpu(logits, op, "logits");
  require_webgpu(targets, op, "targets");
  float_dtype(logits, op, "logits");
  TORCH_CHECK(targets.scalar_type() == at::kInt || targets.scalar_type() == at::kLong,
              "webgpu token_logprobs: targets must be int32 or int64, got ", targets.scalar_type());
  TORCH_CHECK(logits.dim() >= 1 && logits.sizes().slice(0, logits.dim() - 1) == targets.sizes(),
              "webgpu token_logprobs: targets must be one per row of logits, got ", targets.sizes(), " beside ", logits.sizes());
  const int64_t vocab = logits.size(-1);
  TORCH_CHECK(vocab >= 1 && vocab <= TWG_LOGPROBS_MAX_VOCAB, "webgpu token_logprobs: a vocabulary of ", vocab, " entries");
  TORCH_CHECK(top_k >= 0 && top_k <= std::min<int64_t>(vocab, TWG_LOGPROBS_MAX_TOP_K),
              "webgpu token_logprobs: top_k must be in 0..min(", TWG_LOGPROBS_MAX_TOP_K, ", vocab), got ", top_k);
  TORCH_CHECK(scale > 0 && std::isfinite(scale) && (float)scale > 0 && std::isfinite((float)scale),
              "webgpu token_logprobs: scale must be positive and finite, got ", scale);
  const int64_t rows = targets.numel();
  Logprobs r;
  r.logits = unit_last(logits.reshape({rows, vocab}));
  r.targets = targets.reshape({rows}).contiguous();
  const auto f32 = logits.options().dtype(at::kFloat);
  std::vector<int64_t> top_sizes = targets.sizes().vec();
  top_sizes.push_back(top_k);
  r.logprob = at::empty(targets.sizes(), f32);
  r.entropy = at::empty(targets.sizes(), f32);
  r.row_max = at::empty({rows}, f32);
  r.row_sum = at::empty({rows}, f32);
  r.top = at::empty(top_sizes, f32);
  r.ids = at::empty(top_sizes, f32.dtype(at::kLong));
  twg_token_logprobs_t d = logprob_args(r.logits, r.targets, scale, ignore_index);
  d.top_k = (int32_t)top_k;
  d.logprob = static_cast<float *>(r.logprob.data_ptr());
  d.entropy = static_cast<float *>(r.entropy.data_ptr());
  d.row_max = static_cast<float *>(r.row_max.data_ptr());
  d.row_sum = static_cast<float *>(r.row_sum.data_ptr());
  d.top_logprobs = static_cast<float *>(r.top.data_ptr());
  d.top_ids = static_cast<int64_t *>(r.ids.data_ptr());
  const size_t need = twg_token_logprobs_scratch_bytes(&d);
  at::Tensor scratch;
  if (need) scratch = at::empty({(int64_t)(need / 8)}, f32.dtype(at::kLong));
  TWG_CHECK(twg_token_logprobs(&d, ptr(scratch), need, nullptr));
  return r;
}

// With the row's maximum and sum, which the gradient takes.
typedef std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> SixTensors;
SixTensors token_logprobs_stats(const at::Tensor &logits, const at::Tensor &targets, int64_t top_k, double scale,
                                int64_t ignore_index) {
  const Logprobs r = token_logprobs_run(logits, targets, top_k, scale, ignore_index);
  return {r.logprob, r.entropy, r.top, r.ids, r.row_max, r.row_sum};
}

at::Tensor token_logprobs_gradient(const MaybeTensor &g_logprob, const MaybeTensor &g_entropy, const at::Tensor &logits,
                                   const at::Tensor &targets, const at::Tensor &row_max, const at::Tensor &row_sum,
                                   const at::Tensor &entropy, double scale, int64_t ignore_index) {
  const int64_t rows = targets.numel();
  const at::Tensor x = unit_last(logits.reshape({rows, logits.size(-1)})), t = targets.reshape({rows}).contiguous();
  const at::Tensor h = entropy.reshape({rows}).contiguous();
  at::Tensor grad = at::empty(logits.sizes(), logits.options());
  twg_token_logprobs_t d = logprob_args(x, t, scale, ignore_index);
  at::Tensor g[2] = {or_none(g_logprob), or_none(g_entropy)};
  for (at::Tensor &v : g)
    if (v.defined()) v = v.reshape({rows}).contiguous();
  d.g_logprob = static_cast<const float *>(ptr(g[0]));
  d.g_entropy = static_cast<const float *>(ptr(g[1]));
  d.row_max = static_cast<float *>(row_max.data_ptr());
  d.row_sum = static_cast<float *>(row_sum.data_ptr());
  d.entropy = static_cast<float *>(h.data_ptr());
  d.grad = grad.data_ptr();
  d.grad_stride = logits.size(-1);
  TWG_CHECK(twg_token_logprobs_backward(&d, nullptr));
  return grad;
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static variable_list forward(AutogradContext *ctx, const at::Tensor &logits, const at::Tensor &targets, int64_t top_k,
                               double scale, int64_t ignore_index) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = handle<decltype(token_logprobs_stats)>("webgpu::_token_logprobs");
    const auto [logprob, entropy, top, ids, row_max, row_sum] = op.call(logits, targets, top_k, scale, ignore_index);
    ctx->save_for_backward({logits, targets, row_max, row_sum, entropy});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({top, ids});
    return {logprob, entropy, top, ids};
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    once("token_logprobs");
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = handle<decltype(token_logprobs_gradient)>("webgpu::_token_logprobs_backward");
    const variable_list saved = ctx->get_saved_variables();
    const auto maybe = [](const at::Tensor &t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); };
    return {op.call(maybe(grads[0]), maybe(grads[1]), saved[0], saved[1], saved[2], saved[3], saved[4],
                    ctx->saved_data["scale"].toDouble(), ctx->saved_data["ignore_index"].toInt()),
            Variable(), Variable(), Variable(), Variable()};
  }
};

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> token_logprobs(const at::Tensor &logits, const at::Tensor &targets,
                                                                          int64_t top_k, double scale, int64_t ignore_index) {
  const Logprobs r = token_logprobs_run(logits, targets, top_k, scale, ignore_index);
  return {r.logprob, r.entropy, r.top, r.ids};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> token_logprobs_autograd(const at::Tensor &logits,
                                                                                   const at::Tensor &targets, int64_t top_k,
                                                                                   double scale, int64_t ignore_index) {
  const variable_list r = TokenLogprobs::apply(logits, targets, top_k, scale, ignore_index);
  return {r[0], r[1], r[2], r[3]};
}

// --------------------------------------------------------------------- dropout

// out <- residual + dropout(x); the mask goes by the logical order of the elements
void dropout_into(at::Tensor &out, const at::Tensor &x, const at::Tensor &residual, double p, uint64_t seed, uint64_t offset) {
  require_webgpu(x, "dropout", "x");
  require_webgpu(residual, "dropout", "residual");
  const int dt = float_dtype(x, "dropout", "x");
  TORCH_CHECK(p >= 0 && p <= 1, "dropout probability has to be between 0 and 1, but got ", p);
  TORCH_CHECK(!residual.defined() || (residual.sizes() == x.sizes() && residual.scalar_type() == x.scalar_type()),
              "webgpu dropout: the residual must have x's shape and dtype");
  if (x.numel() == 0) return;
  // dimensions fastest first, adjacent ones merged where every operand is linear across them
  const at::Tensor *ops[3] = {&out, &x, &residual};
  const int n = residual.defined() ? 3 : 2;
  twg_iter_t it{};
  it.numel = x.numel();
  for (int64_t ld = x.dim() - 1; ld >= 0; --ld) {
    if (x.size(ld) == 1) continue;
    bool linear = it.ndim > 0;
    for (int o = 0; o < n && linear; ++o)
      linear = ops[o]->stride(ld) == it.stride[o][it.ndim - 1] * it.shape[it.ndim - 1];
    if (linear) {
      it.shape[it.ndim - 1] *= x.size(ld);
      continue;
    }
    TORCH_CHECK(it.ndim < TWG_MAX_DIMS, "webgpu dropout: more than ", TWG_MAX_DIMS, " dimensions after coalescing");
    it.shape[it.ndim] = x.size(ld);
    for (int o = 0; o < n; ++o) it.stride[o][it.ndim] = ops[o]->stride(ld);
    ++it.ndim;
  }
  TWG_CHECK(twg_dropout(out.data_ptr(), x.data_ptr(), ptr(residual), dt, p, seed, offset, nullptr, &it, nullptr));
}

at::Tensor dropout_run(const at::Tensor &x, double p, int64_t seed, int64_t offset, const at::Tensor &residual) {
  at::Tensor out = at::empty_like(x, x.options(), c10::MemoryFormat::Preserve);
  dropout_into(out, x, residual, p, (uint64_t)seed, (uint64_t)offset);
  return out;
}

at::Tensor dropout(const at::Tensor &x, double p, int64_t seed, int64_t offset, const MaybeTensor &residual) {
  return dropout_run(x, p, seed, offset, or_none(residual));
}

struct Dropout : torch::autograd::Function<Dropout> {
  static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x, double p, int64_t seed, int64_t offset,
                            const MaybeTensor &residual) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = handle<decltype(dropout)>("webgpu::dropout");
    ctx->saved_data["p"] = p;
    ctx->set_materialize_grads(false);  // (the device makes no zeros)
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["offset"] = offset;
    ctx->saved_data["residual"] = residual.has_value() && residual->defined();
    return op.call(x, p, seed, offset, residual);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    at::Tensor gx;  // the mask is found again from the seed, the offset and the elements' places
    if (grads[0].defined() && ctx->needs_input_grad(0))
      gx = apply(grads[0], ctx->saved_data["p"].toDouble(), ctx->saved_data["seed"].toInt(),
                 ctx->saved_data["offset"].toInt(), MaybeTensor());
    const bool residual = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1);
    return {gx, Variable(), Variable(), Variable(), residual ? grads[0] : Variable()};
  }
};

at::Tensor dropout_autograd(const at::Tensor &x, double p, int64_t seed, int64_t offset, const MaybeTensor &residual) {
  return Dropout::apply(x, p, seed, offset, residual);
}

// ---- aten::dropout: the seed and the offset are the backend's generator's.  A call leaves what it drew
// as a tensor in host memory, {seed, offset}, for its backward pass: a traced graph draws anew in each run.

void check_p(double p) {
  TORCH_CHECK(p >= 0 && p <= 1, "dropout probability has to be between 0 and 1, but got ", p);
}

at::Tensor next_draw() {
  at::Tensor draw = at::detail::empty_cpu({2}, at::kLong);
  int64_t *to = draw.mutable_data_ptr<int64_t>();
  std::lock_guard<std::mutex> hold(g_rng_lock);
  to[0] = (int64_t)g_rng_seed;
  to[1] = (int64_t)g_rng_offset++;
  return draw;
}

void dropout_drawn_into(at::Tensor out, const at::Tensor &x, double p, const at::Tensor &draw) {
  TORCH_CHECK(draw.is_cpu() && draw.scalar_type() == at::kLong && draw.numel() == 2 && draw.is_contiguous(),
              "webgpu dropout: not what a call drew");
  const int64_t *from = draw.const_data_ptr<int64_t>();
  dropout_into(out, x, at::Tensor(), p, (uint64_t)from[0], (uint64_t)from[1]);
}

std::tuple<at::Tensor, at::Tensor> draw_dropout(const at::Tensor &x, double p) {
  float_dtype(x, "dropout", "x");  // (refused before anything is drawn)
  check_p(p);
  at::Tensor out = at::empty_like(x, x.options(), c10::MemoryFormat::Preserve), draw = next_draw();
  dropout_drawn_into(out, x, p, draw);
  return {out, draw};
}
at::Tensor draw_dropout_(at::Tensor &x, double p) {
  float_dtype(x, "dropout", "x");
  check_p(p);
  at::assert_no_internal_overlap(x);
  const at::Tensor draw = next_draw();
  dropout_drawn_into(x, x, p, draw);
  return draw;
}
at::Tensor redo_dropout(const at::Tensor &x, double p, const at::Tensor &draw) {
  at::Tensor out = at::empty_like(x, x.options(), c10::MemoryFormat::Preserve);
  dropout_drawn_into(out, x, p, draw);
  return out;
}

variable_list redone(AutogradContext *ctx, const variable_list &grads) {
  static const auto op = handle<decltype(redo_dropout)>("webgpu::_redo_dropout");
  if (!grads[0].defined()) return {Variable(), Variable(), Variable()};  // nothing flows back
  return {op.call(grads[0], ctx->saved_data["p"].toDouble(), ctx->get_saved_variables()[0]), Variable(), Variable()};
}

struct RedoDropout : torch::autograd::Function<RedoDropout> {
  static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x, double p, const at::Tensor &draw) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = handle<decltype(redo_dropout)>("webgpu::_redo_dropout");
    ctx->saved_data["p"] = p;
    ctx->set_materialize_grads(false);  // (the device makes no zeros)
    ctx->save_for_backward({draw});
    return op.call(x, p, draw);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) { return redone(ctx, grads); }
};
at::Tensor redo_dropout_autograd(const at::Tensor &x, double p, const at::Tensor &draw) {
  return RedoDropout::apply(x, p, draw);
}

struct DrawDropout : torch::autograd::Function<DrawDropout> {
  static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x, double p) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = handle<decltype(draw_dropout)>("webgpu::_draw_dropout");
    const auto [out, draw] = op.call(x, p);
    ctx->saved_data["p"] = p;
    ctx->set_materialize_grads(false);  // (the device makes no zeros)
    ctx->save_for_backward({draw});
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list g = redone(ctx, grads);
    return {g[0], Variable()};
  }
};

// In place on a tensor with a history, as torch's own in-place operators are: the backward pass needs
// nothing of x.
struct DrawDropoutInPlace : torch::autograd::Function<DrawDropoutInPlace> {
  static at::Tensor forward(AutogradContext *ctx, at::Tensor x, double p) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = handle<decltype(draw_dropout_)>("webgpu::_draw_dropout_");
    ctx->saved_data["p"] = p;
    ctx->set_materialize_grads(false);  // (the device makes no zeros)
    ctx->save_for_backward({op.call(x, p)});
    x.unsafeGetTensorImpl()->bump_version();
    ctx->mark_dirty({x});
    return x;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list g = redone(ctx, grads);
    return {g[0], Variable()};
  }
};

at::Tensor aten_dropout(const at::Tensor &x, double p, bool train) {
  check_p(p);
  if (!train || p == 0 || x.numel() == 0) return x;
  return std::get<0>(draw_dropout(x, p));
}
at::Tensor aten_dropout_autograd(const at::Tensor &x, double p, bool train) {
  check_p(p);
  if (!train || p == 0 || x.numel() == 0) return x;
  return DrawDropout::apply(x, p);
}
at::Tensor &aten_dropout_(at::Tensor &x, double p, bool train) {
  check_p(p);
  if (!train || p == 0 || x.numel() == 0) return x;
  x.unsafeGetTensorImpl()->bump_version();  // (refuses a tensor of inference mode outside of it)
  draw_dropout_(x, p);
  return x;
}
at::Tensor &aten_dropout_autograd_(at::Tensor &x, double p, bool train) {
  check_p(p);
  if (!train || p == 0 || x.numel() == 0) return x;
  const bool grad = torch::autograd::compute_requires_grad(x);
  torch::autograd::check_inplace(x, grad);  // refuses leaves and views of them, before anything is drawn
  if (grad) {
    DrawDropoutInPlace::apply(x, p);
  } else {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = handle<decltype(draw_dropout_)>("webgpu::_draw_dropout_");
    x.unsafeGetTensorImpl()->bump_version();
    op.call(x, p);
  }
  return x;
}

}  // namespace
}  // namespace ops

TORCH_LIBRARY_FRAGMENT(webgpu, m) {
  m.def(
      "norm_rope(Tensor q, Tensor? k, Tensor positions, Tensor inv_freq, Tensor? q_weight=None, Tensor? k_weight=None, "
      "float? eps=1e-06, int[]? pair_axis=None, bool adjacent=False) -> Tensor[]");
  m.def(
      "token_logprobs(Tensor logits, Tensor targets, int top_k=0, float scale=1.0, int ignore_index=-100) -> "
      "(Tensor logprob, Tensor entropy, Tensor top_logprobs, Tensor top_ids)");
  m.def("dropout(Tensor x, float p, int seed, int offset=0, Tensor? residual=None) -> Tensor");
  m.def(
      "_norm_rope_backward(Tensor? dq, Tensor? dk, Tensor q, Tensor? k, Tensor positions, Tensor inv_freq, Tensor? q_weight, "
      "Tensor? k_weight, float? eps, int[] pair_axis, bool adjacent, bool q_weight_grad, bool k_weight_grad) -> "
      "(Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "_token_logprobs(Tensor logits, Tensor targets, int top_k, float scale, int ignore_index) -> "
      "(Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "_token_logprobs_backward(Tensor? g_logprob, Tensor? g_entropy, Tensor logits, Tensor targets, Tensor row_max, "
      "Tensor row_sum, Tensor entropy, float scale, int ignore_index) -> Tensor");
  m.def("_draw_dropout(Tensor x, float p) -> (Tensor, Tensor)", {at::Tag::nondeterministic_seeded});
  m.def("_draw_dropout_(Tensor(a!) x, float p) -> Tensor", {at::Tag::nondeterministic_seeded});
  m.def("_redo_dropout(Tensor x, float p, Tensor draw) -> Tensor");
}
TORCH_LIBRARY_IMPL(webgpu, PrivateUse1, m) {
  m.impl("norm_rope", TORCH_FN(ops::norm_rope));
  m.impl("token_logprobs", TORCH_FN(ops::token_logprobs));
  m.impl("dropout", TORCH_FN(ops::dropout));
  m.impl("_norm_rope_backward", TORCH_FN(ops::norm_rope_gradients));
  m.impl("_token_logprobs", TORCH_FN(ops::token_logprobs_stats));
  m.impl("_token_logprobs_backward", TORCH_FN(ops::token_logprobs_gradient));
  m.impl("_draw_dropout", TORCH_FN(ops::draw_dropout));
  m.impl("_draw_dropout_", TORCH_FN(ops::draw_dropout_));
  m.impl("_redo_dropout", TORCH_FN(ops::redo_dropout));
}
TORCH_LIBRARY_IMPL(webgpu, AutogradPrivateUse1, m) {
  m.impl("norm_rope", TORCH_FN(ops::norm_rope_autograd));
  m.impl("token_logprobs", TORCH_FN(ops::token_logprobs_autograd));
  m.impl("dropout", TORCH_FN(ops::dropout_autograd));
  m.impl("_redo_dropout", TORCH_FN(ops::redo_dropout_autograd));
}
TORCH_LIBRARY_IMPL(aten, PrivateUse1, m) {
  m.impl("dropout", TORCH_FN(ops::aten_dropout));
  m.impl("dropout_", TORCH_FN(ops::aten_dropout_));
}
TORCH_LIBRARY_IMPL(aten, AutogradPrivateUse1, m) {
  m.impl("dropout", TORCH_FN(ops::aten_dropout_autograd));
  m.impl("dropout_", TORCH_FN(ops::aten_dropout_autograd_));
}

}  // namespace torch_webgpu
