// torch.ops._b200_C: operators over rows of logits (log-probabilities of
// given tokens, distillation from a teacher's top values).
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>
#include <torch/torch.h>

#include <atomic>
#include <cmath>
#include <tuple>

#include "logits/logits_api.h"

namespace b200 {
namespace {

using OptTensor = c10::optional<at::Tensor>;

// at::empty without the dispatcher: at few rows the outputs' allocations are
// most of a call's time on the host.
at::Tensor make(at::IntArrayRef size, const at::TensorOptions& o) {
  return at::detail::empty_cuda(size, o);
}

cudaStream_t stream_now() { return at::cuda::getCurrentCUDAStream().stream(); }

LogitRows check_logits(const at::Tensor& x, const char* what) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2, what, ": logits must be a 2-D CUDA tensor [rows, V]");
  const bool bf = x.scalar_type() == at::kBFloat16;
  TORCH_CHECK(bf || x.scalar_type() == at::kFloat, what, ": logits must be bf16 or fp32");
  TORCH_CHECK(x.size(1) >= 1 && x.size(1) <= kMaxVocab, what, ": vocabulary outside [1, 2^22]");
  TORCH_CHECK(x.size(1) == 1 || x.stride(1) == 1, what, ": logits need a unit inner stride");
  return LogitRows{x.data_ptr(), bf, x.size(0), x.stride(0), (int)x.size(1)};
}

void check_temperature(double t, const char* what) {
  TORCH_CHECK(std::isfinite(t) && t >= 1e-3 && t <= 1e3, what,
              ": temperature must be in [1e-3, 1e3], got ", t);
}

void check_like(const at::Tensor& t, const at::Tensor& x, at::ScalarType type, const char* what,
                const char* name) {
  TORCH_CHECK(t.device() == x.device(), what, ": ", name, " must be on the logits' device");
  TORCH_CHECK(t.scalar_type() == type, what, ": ", name, " must be ", type);
  TORCH_CHECK(t.is_contiguous(), what, ": ", name, " must be contiguous");
}

void check_ids(const at::Tensor& ids, const at::Tensor& x, const char* what) {
  TORCH_CHECK(ids.device() == x.device(), what, ": token_ids must be on the logits' device");
  TORCH_CHECK(ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong, what,
              ": token_ids must be int32 or int64");
  TORCH_CHECK(ids.dim() == 1 && ids.size(0) == x.size(0) && ids.is_contiguous(), what,
              ": token_ids must be contiguous [rows]");
}

using Six = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor,
                       at::Tensor>;

Six token_logprobs(const at::Tensor& logits, const at::Tensor& ids, int64_t top_n,
                   double temperature) {
  const char* what = "token_logprobs";
  TokenLogprobsArgs a{};
  a.in = check_logits(logits, what);
  check_ids(ids, logits, what);
  check_temperature(temperature, what);
  TORCH_CHECK(top_n >= 0 && top_n <= kMaxTopN && top_n <= a.in.V, what,
              ": top_n must be in [0, min(64, V)], got ", top_n);
  c10::cuda::CUDAGuard g(logits.device());
  const auto f = logits.options().dtype(at::kFloat), i = logits.options().dtype(at::kInt);
  const int64_t T = a.in.rows;
  auto lp = make({T}, f), ent = make({T}, f), lse = make({T}, f);
  auto rank = make({T}, i), stats = make({T, 4}, f);
  auto top_ids = make({T, top_n}, i), top_lp = make({T, top_n}, f);
  a.ids = ids.data_ptr();
  a.ids64 = ids.scalar_type() == at::kLong;
  a.top_n = (int)top_n;
  a.temperature = (float)temperature;
  a.logprob = lp.data_ptr<float>();
  a.rank = rank.data_ptr<int>();
  a.entropy = ent.data_ptr<float>();
  a.lse = lse.data_ptr<float>();
  a.top_ids = top_ids.data_ptr<int>();
  a.top_lp = top_lp.data_ptr<float>();
  a.stats = stats.data_ptr<float>();
  token_logprobs_launch(a, stream_now());
  return {lp, rank, ent, lse, top_ids, top_lp, stats};
}

at::Tensor token_logprobs_bwd(const at::Tensor& logits, const at::Tensor& ids,
                              const at::Tensor& stats, const OptTensor& g_logprob,
                              const OptTensor& g_entropy, double temperature) {
  const char* what = "token_logprobs_bwd";
  TokenLogprobsBwdArgs a{};
  a.in = check_logits(logits, what);
  check_ids(ids, logits, what);
  check_temperature(temperature, what);
  check_like(stats, logits, at::kFloat, what, "stats");
  TORCH_CHECK(stats.numel() == 4 * a.in.rows, what, ": stats must be [rows, 4]");
  for (const OptTensor* t : {&g_logprob, &g_entropy})
    if (t->has_value()) {
      check_like(**t, logits, at::kFloat, what, "upstream gradient");
      TORCH_CHECK((*t)->numel() == a.in.rows, what, ": upstream gradients must be [rows]");
    }
  c10::cuda::CUDAGuard g(logits.device());
  auto grad = make({a.in.rows, a.in.V}, logits.options());
  a.ids = ids.data_ptr();
  a.ids64 = ids.scalar_type() == at::kLong;
  a.temperature = (float)temperature;
  a.stats = stats.data_ptr<float>();
  a.g_logprob = g_logprob ? g_logprob->data_ptr<float>() : nullptr;
  a.g_entropy = g_entropy ? g_entropy->data_ptr<float>() : nullptr;
  a.grad = grad.data_ptr();
  token_logprobs_bwd_launch(a, stream_now());
  return grad;
}

void check_teacher(const at::Tensor& logits, const at::Tensor& t_ids, const at::Tensor& t_lp,
                   const OptTensor& weights, const char* what) {
  check_like(t_ids, logits, at::kInt, what, "teacher_ids");
  check_like(t_lp, logits, at::kFloat, what, "teacher_logprobs");
  TORCH_CHECK(t_ids.dim() == 2 && t_ids.size(0) == logits.size(0) && t_ids.sizes() == t_lp.sizes(),
              what, ": teacher_ids and teacher_logprobs must be [rows, K]");
  TORCH_CHECK(t_ids.size(1) >= 1 && t_ids.size(1) <= kMaxTeacherK, what,
              ": K must be in [1, 128], got ", t_ids.size(1));
  if (weights) {
    check_like(*weights, logits, at::kFloat, what, "weights");
    TORCH_CHECK(weights->dim() == 1 && weights->size(0) == logits.size(0), what,
                ": weights must be [rows]");
  }
}

// (row losses, numbers for distill_loss_bwd, gradient or empty, loss or empty)
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> distill_loss(
    const at::Tensor& logits, const at::Tensor& t_ids, const at::Tensor& t_lp,
    const OptTensor& weights, double temperature, bool tail, double scale, bool with_loss,
    bool with_grad) {
  const char* what = "distill_loss";
  DistillArgs a{};
  a.in = check_logits(logits, what);
  check_teacher(logits, t_ids, t_lp, weights, what);
  check_temperature(temperature, what);
  c10::cuda::CUDAGuard g(logits.device());
  const auto f = logits.options().dtype(at::kFloat);
  auto rows = make({a.in.rows}, f), stats = make({a.in.rows, 8}, f);
  auto grad = make({with_grad ? a.in.rows : 0, a.in.V}, logits.options());
  auto loss = make({}, f);
  a.t_ids = t_ids.data_ptr<int>();
  a.t_lp = t_lp.data_ptr<float>();
  a.K = (int)t_ids.size(1);
  a.weights = weights ? weights->data_ptr<float>() : nullptr;
  a.temperature = (float)temperature;
  a.tail = tail;
  a.grad_scale = (float)scale;
  a.row_loss = rows.data_ptr<float>();
  a.stats = stats.data_ptr<float>();
  a.grad = with_grad ? grad.data_ptr() : nullptr;
  a.loss = with_loss ? loss.data_ptr<float>() : nullptr;
  a.counter = reinterpret_cast<int*>(loss.data_ptr<float>());  // until the loss is written
  distill_launch(a, stream_now());
  return {rows, stats, grad, loss};
}

void distill_bwd_into(const at::Tensor& grad, const at::Tensor& logits, const at::Tensor& t_ids,
                      const at::Tensor& t_lp, const OptTensor& weights, double temperature,
                      bool tail, const at::Tensor& stats, const at::Tensor& g_rows, double scale,
                      bool unless_one, const char* what) {
  DistillBwdArgs a{};
  a.in = check_logits(logits, what);
  check_teacher(logits, t_ids, t_lp, weights, what);
  check_temperature(temperature, what);
  check_like(stats, logits, at::kFloat, what, "stats");
  check_like(g_rows, logits, at::kFloat, what, "upstream gradient");
  TORCH_CHECK(stats.numel() == 8 * a.in.rows, what, ": stats must be [rows, 8]");
  TORCH_CHECK(g_rows.dim() == 0 || g_rows.numel() == a.in.rows, what,
              ": the upstream gradient must be a scalar or [rows]");
  a.t_ids = t_ids.data_ptr<int>();
  a.t_lp = t_lp.data_ptr<float>();
  a.K = (int)t_ids.size(1);
  a.weights = weights ? weights->data_ptr<float>() : nullptr;
  a.temperature = (float)temperature;
  a.tail = tail;
  a.stats = stats.data_ptr<float>();
  a.g_rows = g_rows.data_ptr<float>();
  a.g_stride = g_rows.dim() == 0 ? 0 : 1;
  a.g_scale = (float)scale;
  a.unless_one = unless_one;
  a.grad = grad.data_ptr();
  distill_bwd_launch(a, stream_now());
}

at::Tensor distill_loss_bwd(const at::Tensor& logits, const at::Tensor& t_ids,
                            const at::Tensor& t_lp, const OptTensor& weights, double temperature,
                            bool tail, const at::Tensor& stats, const at::Tensor& g_rows,
                            double scale) {
  const char* what = "distill_loss_bwd";
  const LogitRows in = check_logits(logits, what);
  c10::cuda::CUDAGuard g(logits.device());
  auto grad = make({in.rows, in.V}, logits.options());
  distill_bwd_into(grad, logits, t_ids, t_lp, weights, temperature, tail, stats, g_rows, scale,
                   false, what);
  return grad;
}

// The gradient for the upstream scalar `g` over that for 1, which `grad` holds.
void distill_loss_redo(at::Tensor& grad, const at::Tensor& logits, const at::Tensor& t_ids,
                       const at::Tensor& t_lp, const OptTensor& weights, double temperature,
                       bool tail, const at::Tensor& stats, const at::Tensor& g, double scale) {
  const char* what = "distill_loss_redo";
  check_logits(logits, what);
  check_like(grad, logits, logits.scalar_type(), what, "grad");
  TORCH_CHECK(grad.sizes() == logits.sizes() && g.dim() == 0, what,
              ": grad must have the logits' shape, the upstream gradient be a scalar");
  c10::cuda::CUDAGuard guard(logits.device());
  distill_bwd_into(grad, logits, t_ids, t_lp, weights, temperature, tail, stats, g, scale, true,
                   what);
}

// ---------------------------------------------------------------- training
// The autograd functions stand here and not in Python: at few rows a step is
// the host's time, and a backward pass that holds no Python function needs no
// change of threads for the interpreter (a step of 33 x 32003: 99 -> 85 us).
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

std::atomic<int64_t> g_backward_launches{0};
int64_t backward_launches() { return g_backward_launches.load(); }

// Through the dispatcher, so that fakes trace.
template <typename F>
c10::TypedOperatorHandle<F> handle(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
Six call_token_logprobs(const at::Tensor& x, const at::Tensor& ids, int64_t top_n, double t) {
  static auto op = handle<decltype(token_logprobs)>("_b200_C::token_logprobs");
  return op.call(x, ids, top_n, t);
}
at::Tensor call_token_logprobs_bwd(const at::Tensor& x, const at::Tensor& ids,
                                   const at::Tensor& stats, const OptTensor& g_lp,
                                   const OptTensor& g_ent, double t) {
  static auto op = handle<decltype(token_logprobs_bwd)>("_b200_C::token_logprobs_bwd");
  g_backward_launches += 1;
  return op.call(x, ids, stats, g_lp, g_ent, t);
}
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> call_distill(
    const at::Tensor& x, const at::Tensor& ids, const at::Tensor& lp, const OptTensor& w, double t,
    bool tail, double scale, bool with_loss, bool with_grad) {
  static auto op = handle<decltype(distill_loss)>("_b200_C::distill_loss");
  return op.call(x, ids, lp, w, t, tail, scale, with_loss, with_grad);
}
at::Tensor call_distill_bwd(const at::Tensor& x, const at::Tensor& ids, const at::Tensor& lp,
                            const OptTensor& w, double t, bool tail, const at::Tensor& stats,
                            const at::Tensor& g, double scale) {
  static auto op = handle<decltype(distill_loss_bwd)>("_b200_C::distill_loss_bwd");
  g_backward_launches += 1;
  return op.call(x, ids, lp, w, t, tail, stats, g, scale);
}
void call_distill_redo(at::Tensor& grad, const at::Tensor& x, const at::Tensor& ids,
                       const at::Tensor& lp, const OptTensor& w, double t, bool tail,
                       const at::Tensor& stats, const at::Tensor& g, double scale) {
  static auto op = handle<decltype(distill_loss_redo)>("_b200_C::distill_loss_redo");
  g_backward_launches += 1;
  op.call(grad, x, ids, lp, w, t, tail, stats, g, scale);
}

// Neither operator has forward-mode derivatives: a tangent is refused, not
// dropped (below the autograd keys nothing would know of it).
void refuse_tangent(const at::Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(/*level=*/0).defined(), what,
                              ": forward-mode derivatives are not implemented");
}
Six token_logprobs_ad(const at::Tensor& x, const at::Tensor& ids, int64_t top_n, double t) {
  refuse_tangent(x, "token_logprobs");
  at::AutoDispatchBelowADInplaceOrView guard;
  return call_token_logprobs(x, ids, top_n, t);
}
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> distill_loss_ad(
    const at::Tensor& x, const at::Tensor& ids, const at::Tensor& lp, const OptTensor& w, double t,
    bool tail, double scale, bool with_loss, bool with_grad) {
  for (const at::Tensor* p : {&x, &lp}) refuse_tangent(*p, "distill_loss");
  if (w) refuse_tangent(*w, "distill_loss");
  at::AutoDispatchBelowADInplaceOrView guard;
  return call_distill(x, ids, lp, w, t, tail, scale, with_loss, with_grad);
}

OptTensor opt(const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// A gradient that a graph of gradients may hold, and that raises where it is
// differentiated itself.
at::Tensor once(at::Tensor grad) {
  if (!at::GradMode::is_enabled()) return grad;
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "this operator's gradient cannot be differentiated again", 1);
  grad = grad.detach();
  grad.set_requires_grad(true);
  return (*error)({grad})[0];
}

struct TokenLogprobsFn : public Function<TokenLogprobsFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& ids,
                               int64_t top_n, double t) {
    auto [lp, rank, ent, lse, top_ids, top_lp, stats] = call_token_logprobs(x, ids, top_n, t);
    ctx->save_for_backward({x, ids, stats});
    ctx->saved_data["t"] = t;
    ctx->mark_non_differentiable({rank, lse, top_ids, top_lp});
    ctx->set_materialize_grads(false);
    return {lp, rank, ent, lse, top_ids, top_lp};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined() && !g[2].defined()) return variable_list(4);
    const auto saved = ctx->get_saved_variables();
    at::AutoDispatchBelowADInplaceOrView guard;
    const at::Tensor lp = g[0].defined() ? g[0].contiguous() : at::Tensor();
    const at::Tensor ent = g[2].defined() ? g[2].contiguous() : at::Tensor();
    at::Tensor grad = call_token_logprobs_bwd(saved[0], saved[1], saved[2], opt(lp), opt(ent),
                                              ctx->saved_data["t"].toDouble());
    return {once(grad), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

struct DistillRowsFn : public Function<DistillRowsFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& ids,
                            const at::Tensor& lp, const OptTensor& w, double t, bool tail) {
    auto [rows, stats, grad, loss] = call_distill(x, ids, lp, w, t, tail, 1.0, false, false);
    ctx->save_for_backward({x, ids, lp, w ? *w : at::Tensor(), stats});
    ctx->saved_data["t"] = t;
    ctx->saved_data["tail"] = tail;
    return rows;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    at::AutoDispatchBelowADInplaceOrView guard;
    at::Tensor grad = call_distill_bwd(s[0], s[1], s[2], opt(s[3]), ctx->saved_data["t"].toDouble(),
                                       ctx->saved_data["tail"].toBool(), s[4], g[0].contiguous(),
                                       1.0);
    return {once(grad), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// Loss and gradient in one pass over the logits, for the upstream scalar 1;
// where backward gets another, the gradient is computed anew there.
struct DistillScalarFn : public Function<DistillScalarFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& ids,
                            const at::Tensor& lp, const OptTensor& w, double t, bool tail,
                            double scale) {
    auto [rows, stats, grad, loss] = call_distill(x, ids, lp, w, t, tail, scale, true, true);
    ctx->save_for_backward({x, ids, lp, w ? *w : at::Tensor(), stats});
    ctx->saved_data["t"] = t;
    ctx->saved_data["tail"] = tail;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["grad"] = grad;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    at::AutoDispatchBelowADInplaceOrView guard;
    const double t = ctx->saved_data["t"].toDouble(), scale = ctx->saved_data["scale"].toDouble();
    const bool tail = ctx->saved_data["tail"].toBool();
    auto held = ctx->saved_data.find("grad");
    at::Tensor grad;
    if (held != ctx->saved_data.end()) {
      grad = held->second.toTensor();
      ctx->saved_data.erase(held);
      call_distill_redo(grad, s[0], s[1], s[2], opt(s[3]), t, tail, s[4], g[0], scale);
    } else {  // the graph is run again: the first run gave its gradient away
      grad = call_distill_bwd(s[0], s[1], s[2], opt(s[3]), t, tail, s[4], g[0], scale);
    }
    return {once(grad),   at::Tensor(), at::Tensor(), at::Tensor(),
            at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>
token_logprobs_train(const at::Tensor& x, const at::Tensor& ids, int64_t top_n, double t) {
  auto r = TokenLogprobsFn::apply(x, ids, top_n, t);
  return {r[0], r[1], r[2], r[3], r[4], r[5]};
}
at::Tensor distill_rows_train(const at::Tensor& x, const at::Tensor& ids, const at::Tensor& lp,
                              const OptTensor& w, double t, bool tail) {
  return DistillRowsFn::apply(x, ids, lp, w, t, tail);
}
at::Tensor distill_scalar_train(const at::Tensor& x, const at::Tensor& ids, const at::Tensor& lp,
                                const OptTensor& w, double t, bool tail, double scale) {
  return DistillScalarFn::apply(x, ids, lp, w, t, tail, scale);
}

}  // namespace
}  // namespace b200

TORCH_LIBRARY_FRAGMENT(_b200_C, m) {
  m.def("token_logprobs_train(Tensor logits, Tensor token_ids, int top_n, float temperature) -> "
        "(Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("distill_rows_train(Tensor logits, Tensor teacher_ids, Tensor teacher_logprobs, "
        "Tensor? weights, float temperature, bool tail) -> Tensor");
  m.def("distill_scalar_train(Tensor logits, Tensor teacher_ids, Tensor teacher_logprobs, "
        "Tensor? weights, float temperature, bool tail, float scale) -> Tensor");
  m.def("backward_launches() -> int", &b200::backward_launches);
  m.def("token_logprobs(Tensor logits, Tensor token_ids, int top_n, float temperature) -> "
        "(Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("token_logprobs_bwd(Tensor logits, Tensor token_ids, Tensor stats, Tensor? g_logprob, "
        "Tensor? g_entropy, float temperature) -> Tensor");
  m.def("distill_loss(Tensor logits, Tensor teacher_ids, Tensor teacher_logprobs, "
        "Tensor? weights, float temperature, bool tail, float scale, bool with_loss, "
        "bool with_grad) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("distill_loss_bwd(Tensor logits, Tensor teacher_ids, Tensor teacher_logprobs, "
        "Tensor? weights, float temperature, bool tail, Tensor stats, Tensor g_rows, "
        "float scale) -> Tensor");
  m.def("distill_loss_redo(Tensor(a!) grad, Tensor logits, Tensor teacher_ids, "
        "Tensor teacher_logprobs, Tensor? weights, float temperature, bool tail, Tensor stats, "
        "Tensor g, float scale) -> ()");
}

TORCH_LIBRARY_IMPL(_b200_C, CUDA, m) {
  m.impl("token_logprobs", &b200::token_logprobs);
  m.impl("token_logprobs_bwd", &b200::token_logprobs_bwd);
  m.impl("distill_loss", &b200::distill_loss);
  m.impl("distill_loss_bwd", &b200::distill_loss_bwd);
  m.impl("distill_loss_redo", &b200::distill_loss_redo);
}

TORCH_LIBRARY_IMPL(_b200_C, Autograd, m) {
  m.impl("token_logprobs", &b200::token_logprobs_ad);
  m.impl("distill_loss", &b200::distill_loss_ad);
}

TORCH_LIBRARY_IMPL(_b200_C, CompositeImplicitAutograd, m) {
  m.impl("token_logprobs_train", &b200::token_logprobs_train);
  m.impl("distill_rows_train", &b200::distill_rows_train);
  m.impl("distill_scalar_train", &b200::distill_scalar_train);
}
