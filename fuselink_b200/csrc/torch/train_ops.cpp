// Bindings of the operators around the expert layers of a training step: embedding, routing, log-probabilities and policy loss, AdamW.
// Each one that has a gradient is an autograd node of native code: the calls take the GPU a few microseconds, and a node in Python as many more.
#include <torch/extension.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <ATen/cuda/EmptyTensor.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <string>
#include <vector>

#include "../kernels/adamw.cuh"
#include "../kernels/embedding.cuh"
#include "../kernels/losses.cuh"
#include "../kernels/routing.cuh"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;
using OptTensor = c10::optional<Tensor>;

cudaStream_t stream_of() { return c10::cuda::getCurrentCUDAStream().stream(); }

void check(int rc, const char* what) {
  if (rc == 0) return;
  std::string msg = std::string(what) + " failed with code " + std::to_string(rc);
  if (rc > 0) msg += std::string(" (") + cudaGetErrorString((cudaError_t)rc) + ")";
  throw std::runtime_error(msg);
}

int dtype_of(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case torch::kBFloat16: return FL_BF16;
    case torch::kHalf: return FL_FP16;
    case torch::kFloat32: return FL_FP32;
    default: break;
  }
  TORCH_CHECK(false, what, ": bf16, fp16 or fp32 expected, not ", t.scalar_type());
}

// a new tensor without the dispatcher's part
Tensor new_like(const Tensor& as, c10::IntArrayRef sizes, torch::ScalarType type) {
  return Tensor(at::detail::empty_cuda(sizes, type, as.device(), c10::nullopt));
}
Tensor new_bytes(const Tensor& as, long long bytes) { return new_like(as, {(int64_t)bytes}, torch::kUInt8); }

bool records(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }
void first_derivative_only(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": the kernels' gradient cannot itself be differentiated");
}
const float* floats(const OptTensor& t, const Tensor& as, int64_t numel, const char* what) {
  if (!t.has_value()) return nullptr;
  TORCH_CHECK(t->device() == as.device() && t->scalar_type() == torch::kFloat32 && t->is_contiguous() && t->numel() == numel, what);
  return t->const_data_ptr<float>();
}

// ------------------------------------------------------------------------------------------------ embedding
FlEmbedArgs embed_args(const Tensor& tokens, int64_t vocab, int64_t hidden, double scale, int64_t status) {
  FlEmbedArgs a;
  memset(&a, 0, sizeof a);
  a.tokens = tokens.const_data_ptr(); a.token_bytes = tokens.scalar_type() == torch::kInt64 ? 8 : 4;
  a.n = tokens.numel(); a.vocab = vocab; a.hidden = hidden; a.scale = (float)scale; a.status = reinterpret_cast<int*>(status);
  return a;
}
Tensor embed_forward(const Tensor& table, const Tensor& tokens, double scale, int64_t status) {
  c10::cuda::CUDAGuard guard(table.device());
  const int dt = dtype_of(table, "embedding");
  FlEmbedArgs a = embed_args(tokens, table.size(0), table.size(1), scale, status);
  auto sizes = tokens.sizes().vec();
  sizes.push_back(table.size(1));
  const Tensor out = new_like(table, sizes, table.scalar_type());
  a.table = table.const_data_ptr(); a.table_stride = table.size(0) > 1 ? table.stride(0) : table.size(1);
  a.out = out.data_ptr();
  check(fl_embed(dt, &a, stream_of()), "fl_embed");
  return out;
}
struct Embed : torch::autograd::Function<Embed> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& tokens, double scale, int64_t status) {
    ctx->save_for_backward({tokens});
    ctx->saved_data["vocab"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    return embed_forward(table, tokens, scale, status);
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    first_derivative_only("embedding");
    const Tensor tokens = ctx->get_saved_variables()[0], dout = grads[0].contiguous();
    c10::cuda::CUDAGuard guard(dout.device());
    const int64_t vocab = ctx->saved_data["vocab"].toInt(), hidden = dout.size(-1);
    FlEmbedArgs a = embed_args(tokens, vocab, hidden, ctx->saved_data["scale"].toDouble(), 0);
    const Tensor dtable = new_like(dout, {vocab, hidden}, dout.scalar_type());
    const long long bytes = fl_embed_scratch(a.n, vocab, hidden);
    TORCH_CHECK(bytes >= 0, "embedding: too large");
    const Tensor scratch = new_bytes(dout, bytes);
    a.dout = dout.const_data_ptr(); a.dtable = dtable.data_ptr(); a.scratch = scratch.data_ptr();
    check(fl_embed_grad(dtype_of(dout, "embedding"), &a, stream_of()), "fl_embed_grad");
    return {dtable, Tensor(), Tensor(), Tensor()};
  }
};
Tensor embed_lookup(const Tensor& table, Tensor tokens, double scale, int64_t status) {
  TORCH_CHECK(table.is_cuda() && table.dim() == 2 && table.size(0) > 0 && table.size(1) > 0, "embedding: table [vocab, hidden] on the GPU");
  TORCH_CHECK(tokens.device() == table.device(), "embedding: tokens on ", table.device(), " expected, not on ", tokens.device());
  TORCH_CHECK(tokens.scalar_type() == torch::kInt64 || tokens.scalar_type() == torch::kInt32, "embedding: tokens of int64 or int32 expected");
  TORCH_CHECK(table.size(1) == 1 || table.stride(1) == 1, "embedding: a table of contiguous rows");
  TORCH_CHECK(table.size(0) == 1 || table.stride(0) >= table.size(1), "embedding: a table of rows that do not overlap");
  dtype_of(table, "embedding");
  tokens = tokens.contiguous();
  return records(table) ? Embed::apply(table, tokens, scale, status) : embed_forward(table, tokens, scale, status);
}

// ------------------------------------------------------------------------------------------------ routing
struct RouteHow {
  int64_t topk, score, groups, topk_groups, group_best;
  bool renormalize;
  double scale;
};
FlRouteArgs route_args(const Tensor& logits, const RouteHow& h, const OptTensor& offset) {
  FlRouteArgs a;
  memset(&a, 0, sizeof a);
  a.logits = logits.const_data_ptr(); a.tokens = logits.size(0); a.stride = logits.size(0) > 1 ? logits.stride(0) : logits.size(1);
  a.experts = (int)logits.size(1); a.topk = (int)h.topk; a.score = (int)h.score; a.groups = (int)h.groups; a.topk_groups = (int)h.topk_groups;
  a.group_best = (int)h.group_best; a.renormalize = h.renormalize; a.scale = (float)h.scale;
  a.offset = offset.has_value() ? offset->const_data_ptr<float>() : nullptr;
  return a;
}
// weights, experts, load and, where asked for, the balance term
tensor_list route_forward(const Tensor& logits, const RouteHow& h, const OptTensor& bias, const OptTensor& offset, bool balance) {
  c10::cuda::CUDAGuard guard(logits.device());
  FlRouteArgs a = route_args(logits, h, offset);
  a.bias = bias.has_value() ? bias->const_data_ptr<float>() : nullptr;
  const int64_t T = logits.size(0), E = logits.size(1);
  Tensor w = new_like(logits, {T, h.topk}, torch::kFloat32), chosen = new_like(logits, {T, h.topk}, torch::kInt32), load = new_like(logits, {E}, torch::kInt32), term;
  if (balance) term = new_like(logits, {}, torch::kFloat32);
  const long long bytes = fl_route_scratch(T, a.experts);
  Tensor scratch;
  if (bytes > 0) scratch = new_bytes(logits, bytes);
  a.weights = w.data_ptr<float>(); a.chosen = chosen.data_ptr<int>(); a.load = load.data_ptr<int>(); a.balance = balance ? term.data_ptr<float>() : nullptr;
  a.scratch = bytes > 0 ? scratch.data_ptr() : nullptr;
  check(fl_route(dtype_of(logits, "route"), &a, stream_of()), "fl_route");
  return {w, chosen, load, term};
}
struct Route : torch::autograd::Function<Route> {
  static tensor_list forward(AutogradContext* ctx, const Tensor& logits, int64_t topk, int64_t score, int64_t groups, int64_t topk_groups, int64_t group_best, bool renormalize,
                             double scale, const OptTensor& bias, const OptTensor& offset, bool balance) {
    const RouteHow h{topk, score, groups, topk_groups, group_best, renormalize, scale};
    tensor_list out = route_forward(logits, h, bias, offset, balance);
    ctx->save_for_backward({logits, out[0], out[1], out[2], offset.has_value() ? *offset : Tensor()});
    ctx->saved_data["how"] = std::vector<int64_t>{topk, score, groups, topk_groups, group_best, renormalize};
    ctx->saved_data["scale"] = scale;
    ctx->mark_non_differentiable({out[1], out[2]});
    ctx->set_materialize_grads(false);
    if (!balance) out.pop_back();
    return out;
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    tensor_list said(11);
    const Tensor dterm = grads.size() > 3 ? grads[3] : Tensor();
    if (!grads[0].defined() && !dterm.defined()) return said;
    first_derivative_only("route");
    const auto saved = ctx->get_saved_variables();
    const Tensor& logits = saved[0];
    c10::cuda::CUDAGuard guard(logits.device());
    const auto k = ctx->saved_data["how"].toIntVector();
    const RouteHow h{k[0], k[1], k[2], k[3], k[4], k[5] != 0, ctx->saved_data["scale"].toDouble()};
    FlRouteArgs a = route_args(logits, h, saved[4].defined() ? OptTensor(saved[4]) : OptTensor());
    const Tensor dw = grads[0].defined() ? grads[0].contiguous() : Tensor(), dlogits = new_like(logits, logits.sizes(), logits.scalar_type());
    a.weights = saved[1].data_ptr<float>(); a.chosen = saved[2].data_ptr<int>(); a.load = saved[3].data_ptr<int>();
    a.dweights = dw.defined() ? dw.const_data_ptr<float>() : nullptr;
    a.dbalance = dterm.defined() ? dterm.const_data_ptr<float>() : nullptr;
    a.dlogits = dlogits.data_ptr();
    check(fl_route_grad(dtype_of(logits, "route"), &a, stream_of()), "fl_route_grad");
    said[0] = dlogits;
    return said;
  }
};
// What is wrong with an argument's value is a ValueError, as from the plain form in Python; these checks are here because the calls are short.
void value(bool ok, const char* what) {
  if (!ok) throw pybind11::value_error(what);
}
std::tuple<Tensor, Tensor, Tensor, OptTensor> route(Tensor logits, int64_t topk, const std::string& score, int64_t groups, c10::optional<int64_t> topk_groups, int64_t group_best,
                                                    bool renormalize, double scale, OptTensor bias, OptTensor offset, bool balance) {
  TORCH_CHECK(logits.is_cuda(), "route: logits on the GPU");
  value(logits.dim() == 2 && logits.size(1) >= 1, "route: logits [tokens, experts] expected");
  const int64_t E = logits.size(1), how = score == "softmax" ? FL_ROUTE_SOFTMAX : score == "sigmoid" ? FL_ROUTE_SIGMOID : -1;
  value(how >= 0, "route: a score of softmax or sigmoid expected");
  value(groups >= 1 && E % groups == 0, "route: the experts do not make so many equal groups");
  const int64_t kept = topk_groups.value_or(groups);
  value(kept >= 1 && kept <= groups, "route: topk_groups, one at least and no more than there are groups");
  value(topk >= 1 && topk <= E / groups * kept, "route: topk, one at least and no more than the groups chosen from have experts");
  if (groups == 1) group_best = 1;
  value((group_best == 1 || group_best == 2) && group_best <= E / groups, "route: a group goes by its 1 or 2 best");
  value(scale != 0.0 && std::isfinite(scale), "route: a factor that is finite and not 0");
  TORCH_CHECK(E <= FL_ROUTE_MAX_EXPERTS && topk <= FL_ROUTE_MAX_TOPK && groups <= FL_ROUTE_MAX_GROUPS, "route: at most 1024 experts, 32 choices and 32 groups on the GPU");
  static_assert(FL_ROUTE_MAX_EXPERTS == 1024 && FL_ROUTE_MAX_TOPK == 32 && FL_ROUTE_MAX_GROUPS == 32, "what the message says");
  dtype_of(logits, "route");
  for (auto* t : {&bias, &offset}) {
    if (!t->has_value()) continue;
    value((*t)->dim() == 1 && (*t)->size(0) == E && (*t)->scalar_type() == torch::kFloat32, "route: bias and offset [experts] fp32");
    TORCH_CHECK((*t)->device() == logits.device(), "route: bias and offset on the logits' device");
    TORCH_CHECK(!records(**t), "route: bias and offset get no gradient; detach them");
    if (!(*t)->is_contiguous()) *t = (*t)->contiguous();
  }
  if ((E > 1 && logits.stride(1) != 1) || (logits.size(0) > 1 && logits.stride(0) < E)) logits = logits.contiguous();
  tensor_list out;
  if (records(logits)) out = Route::apply(logits, topk, how, groups, kept, group_best, renormalize, scale, bias, offset, balance);
  else out = route_forward(logits, RouteHow{topk, how, groups, kept, group_best, renormalize, scale}, bias, offset, balance);
  return {out[0], out[1], out[2], balance ? OptTensor(out[3]) : OptTensor()};
}

// ------------------------------------------------------------------------------------------------ losses
// The logits as rows at (i, j), or a contiguous copy of them where they do not lie so.  Without a value there is no row, whatever the sizes and strides are.
Tensor as_rows(const Tensor& logits, FlLossArgs& a) {
  const int64_t V = logits.size(-1);
  if (logits.numel() == 0) {
    a.logits = nullptr; a.vocab = V;
    a.outer = a.inner = 0; a.outer_stride = a.inner_stride = V;
    return logits;
  }
  const int d = (int)logits.dim() - 1;
  int64_t size[2] = {1, 1}, stride[2] = {V, V};             // [0]: the inner rows
  int n = 0;
  bool fits = V == 1 || logits.stride(-1) == 1;
  for (int i = d - 1; i >= 0 && fits; --i) {
    if (logits.size(i) == 1) continue;
    if (n > 0 && logits.stride(i) == stride[n - 1] * size[n - 1]) size[n - 1] *= logits.size(i);
    else if (n < 2) { size[n] = logits.size(i); stride[n] = logits.stride(i); ++n; }
    else fits = false;
  }
  for (int i = 0; i < n; ++i) fits = fits && stride[i] >= (i == 0 ? V : stride[0] * (size[0] - 1) + V);
  if (!fits) return as_rows(logits.contiguous(), a);
  a.logits = logits.const_data_ptr(); a.vocab = V;
  a.outer = size[1]; a.inner = size[0]; a.outer_stride = stride[1]; a.inner_stride = stride[0];
  TORCH_CHECK(a.outer * a.inner == logits.numel() / V, "losses: the logits' rows are not as many as they should be");
  return logits;
}
// A gradient whose rows begin as far behind multiples of 16 bytes as those of the logits: contiguous where that does it, else with up to 15 bytes
// between rows.
Tensor gradient_like(const Tensor& logits, FlLossArgs& a, const Tensor& ready = Tensor()) {
  const int64_t z = logits.element_size(), P = 16 / z, V = a.vocab, behind = ((uintptr_t)a.logits & 15) / z;
  auto up_to = [P](int64_t least, int64_t like) { return least + ((like - least) % P + P) % P; };
  a.dlogits_inner = a.inner > 1 ? up_to(V, a.inner_stride) : V;
  a.dlogits_outer = a.outer > 1 ? up_to(a.inner * a.dlogits_inner, a.outer_stride) : a.inner * a.dlogits_inner;
  Tensor out = ready;                                        // one that this function has made for the same logits
  if (out.defined()) {
    a.dlogits = out.data_ptr();
  } else if (behind == 0 && a.dlogits_inner == V && a.dlogits_outer == a.inner * V) {
    out = new_like(logits, logits.sizes(), logits.scalar_type());
    a.dlogits = out.data_ptr();
  } else {
    const Tensor all = new_like(logits, {behind + a.outer * a.dlogits_outer + V}, logits.scalar_type());
    auto strides = logits.sizes().vec();
    int64_t rows = 1;                                        // of the dimensions behind this one, of the inner rows or the outer ones
    bool outer = false;
    strides.back() = 1;
    for (int64_t i = logits.dim() - 2; i >= 0; --i) {
      if (!outer && rows == a.inner && logits.size(i) != 1) { outer = true; rows = 1; }
      strides[i] = (outer ? a.dlogits_outer : a.dlogits_inner) * rows;
      rows *= logits.size(i);
    }
    out = all.as_strided(logits.sizes(), strides, behind);
    a.dlogits = out.data_ptr();
  }
  if (a.inner <= 1) a.dlogits_inner = a.inner_stride;       // one row: no distance to keep
  if (a.outer <= 1) a.dlogits_outer = a.outer_stride;
  return out;
}
FlLossArgs loss_args(double temperature, const Tensor& tokens) {
  FlLossArgs a;
  memset(&a, 0, sizeof a);
  a.temperature = temperature;
  a.tokens = reinterpret_cast<const long long*>(tokens.const_data_ptr<int64_t>());
  return a;
}
// the gradient of rows whose log-probabilities' derivatives are `each` times `factor`; `ready`: what it is for a factor of 1, or nothing
Tensor rows_gradient(const Tensor& logits, const Tensor& tokens, double temperature, const Tensor& top, const Tensor& inverse, const Tensor& each, const Tensor& factor, const Tensor& ready) {
  FlLossArgs a = loss_args(temperature, tokens);
  c10::cuda::CUDAGuard guard(logits.device());
  const Tensor rows = as_rows(logits, a);
  if (logits.numel() == 0) return at::zeros_like(logits);
  const Tensor out = gradient_like(rows, a, ready);
  a.top = top.data_ptr<float>(); a.inverse = inverse.data_ptr<float>(); a.dlogprobs = each.const_data_ptr<float>();
  a.upstream = factor.defined() ? factor.const_data_ptr<float>() : nullptr;
  a.unless_one = ready.defined();
  check(fl_logprobs_grad(dtype_of(logits, "losses"), &a, stream_of()), "fl_logprobs_grad");
  return out;
}

Tensor logits_and_tokens(const Tensor& logits, Tensor tokens, double temperature) {
  TORCH_CHECK(logits.is_cuda(), "losses: logits on the GPU");
  value(logits.dim() >= 1 && logits.size(-1) > 0, "losses: logits [..., vocab] expected");
  value(tokens.sizes() == logits.sizes().slice(0, logits.dim() - 1), "losses: tokens, one for each row of the logits");
  value(tokens.scalar_type() == torch::kInt64 || tokens.scalar_type() == torch::kInt32, "losses: tokens of int64 or int32 expected");
  TORCH_CHECK(tokens.device() == logits.device(), "losses: tokens on ", logits.device(), " expected, not on ", tokens.device());
  value(temperature >= 1e-30 && std::isfinite(temperature), "losses: a temperature of 1e-30 at least");
  dtype_of(logits, "losses");
  return tokens.scalar_type() == torch::kInt64 && tokens.is_contiguous() ? tokens : tokens.to(torch::kInt64).contiguous();
}
// log-probabilities and, where the gradient will be asked for, the rows' largest logits and inverse sums
tensor_list logprobs_forward(const Tensor& logits, const Tensor& tokens, double temperature, bool gradient) {
  c10::cuda::CUDAGuard guard(logits.device());
  FlLossArgs a = loss_args(temperature, tokens);
  const Tensor rows = as_rows(logits, a);
  Tensor lp = new_like(logits, tokens.sizes(), torch::kFloat32), top, inverse;
  a.logprobs = lp.data_ptr<float>();
  if (gradient) {
    top = new_like(logits, {tokens.numel()}, torch::kFloat32); inverse = new_like(logits, {tokens.numel()}, torch::kFloat32);
    a.top = top.data_ptr<float>(); a.inverse = inverse.data_ptr<float>();
  }
  if (tokens.numel() > 0) check(fl_token_logprobs(dtype_of(logits, "token_logprobs"), &a, stream_of()), "fl_token_logprobs");
  return {lp, top, inverse};
}
struct LogProbs : torch::autograd::Function<LogProbs> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, double temperature) {
    const auto out = logprobs_forward(logits, tokens, temperature, true);
    ctx->save_for_backward({logits, tokens});
    ctx->saved_data["top"] = out[1];
    ctx->saved_data["inverse"] = out[2];
    ctx->saved_data["temperature"] = temperature;
    ctx->set_materialize_grads(false);
    return out[0];
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
    first_derivative_only("token_logprobs");
    const auto saved = ctx->get_saved_variables();
    return {rows_gradient(saved[0], saved[1], ctx->saved_data["temperature"].toDouble(), ctx->saved_data["top"].toTensor(), ctx->saved_data["inverse"].toTensor(),
                          grads[0].contiguous(), Tensor(), Tensor()),
            Tensor(), Tensor()};
  }
};
Tensor token_logprobs(const Tensor& logits, Tensor tokens, double temperature) {
  tokens = logits_and_tokens(logits, tokens, temperature);
  return records(logits) ? LogProbs::apply(logits, tokens, temperature) : logprobs_forward(logits, tokens, temperature, false)[0];
}

struct PolicyHow {
  double kl, low, high, temperature;
};
// loss, log-probabilities, divergence, clipped share; and for the gradient the rows' largest logits, inverse sums, derivatives, and the logits' gradient
tensor_list policy_forward(const Tensor& logits, const Tensor& tokens, const Tensor& old, const Tensor& advantages, const OptTensor& reference, const OptTensor& weights,
                           const OptTensor& total, const PolicyHow& h, bool gradient) {
  c10::cuda::CUDAGuard guard(logits.device());
  FlLossArgs a = loss_args(h.temperature, tokens);
  const Tensor rows = as_rows(logits, a);
  const int64_t n = tokens.numel();
  Tensor lp = new_like(logits, tokens.sizes(), torch::kFloat32), loss = new_like(logits, {}, torch::kFloat32), divergence = new_like(logits, {}, torch::kFloat32),
         clipped = new_like(logits, {}, torch::kFloat32), top, inverse, each, dlogits;
  const Tensor scratch = new_bytes(logits, fl_policy_scratch());
  a.logprobs = lp.data_ptr<float>();
  a.old = floats(old, logits, n, "policy_loss: old, fp32, like tokens"); a.advantages = floats(advantages, logits, n, "policy_loss: advantages, fp32, like tokens");
  a.reference = floats(reference, logits, n, "policy_loss: reference, fp32, like tokens"); a.weights = floats(weights, logits, n, "policy_loss: weights, fp32, like tokens");
  a.total = floats(total, logits, 1, "policy_loss: total, one fp32 value on the logits' device");
  a.kl = h.kl; a.clip_low = h.low; a.clip_high = h.high;
  a.loss = loss.data_ptr<float>(); a.divergence = divergence.data_ptr<float>(); a.clipped = clipped.data_ptr<float>();
  a.scratch = scratch.data_ptr();
  if (gradient && n > 0) {
    top = new_like(logits, {n}, torch::kFloat32); inverse = new_like(logits, {n}, torch::kFloat32); each = new_like(logits, {n}, torch::kFloat32);
    a.top = top.data_ptr<float>(); a.inverse = inverse.data_ptr<float>(); a.coefficient = each.data_ptr<float>();
    dlogits = gradient_like(rows, a);
  }
  check(fl_policy_loss(dtype_of(logits, "policy_loss"), &a, stream_of()), "fl_policy_loss");
  return {loss, lp, divergence, clipped, top, inverse, each, dlogits};
}
struct Policy : torch::autograd::Function<Policy> {
  static tensor_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, const Tensor& old, const Tensor& advantages, const OptTensor& reference,
                             const OptTensor& weights, const OptTensor& total, double kl, double low, double high, double temperature) {
    auto out = policy_forward(logits, tokens, old, advantages, reference, weights, total, PolicyHow{kl, low, high, temperature}, true);
    ctx->save_for_backward({logits, tokens});
    for (const auto& [name, at] : {std::pair<const char*, int>{"top", 4}, {"inverse", 5}, {"each", 6}, {"ready", 7}}) ctx->saved_data[name] = out[at];
    ctx->saved_data["temperature"] = temperature;
    ctx->mark_non_differentiable({out[1], out[2], out[3]});
    ctx->set_materialize_grads(false);
    out.resize(4);
    return out;
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    tensor_list said(11);
    if (!grads[0].defined()) return said;
    first_derivative_only("policy_loss");
    const auto saved = ctx->get_saved_variables();
    if (saved[0].numel() == 0) {
      said[0] = at::zeros_like(saved[0]);
      return said;
    }
    Tensor ready = ctx->saved_data["ready"].toTensor();      // given away once: its next owner may write into it
    ctx->saved_data["ready"] = Tensor();
    said[0] = rows_gradient(saved[0], saved[1], ctx->saved_data["temperature"].toDouble(), ctx->saved_data["top"].toTensor(), ctx->saved_data["inverse"].toTensor(),
                            ctx->saved_data["each"].toTensor(), grads[0].contiguous(), ready);
    return said;
  }
};
// `total`: None, a number, or one value on the device
std::tuple<Tensor, Tensor, Tensor, Tensor> policy_loss(const Tensor& logits, Tensor tokens, Tensor old, Tensor advantages, OptTensor reference, OptTensor weights,
                                                       pybind11::object total_of, double kl, double low, double high, double temperature) {
  tokens = logits_and_tokens(logits, tokens, temperature);
  value(low >= 0.0 && std::isfinite(low) && high >= 0.0 && std::isfinite(high) && kl >= 0.0 && std::isfinite(kl), "policy_loss: borders and a factor of the KL term that are not negative");
  auto like_tokens = [&](Tensor& t, const char* what) {
    TORCH_CHECK(t.device() == tokens.device(), "policy_loss: ", what, " on ", tokens.device(), " expected, not on ", t.device());
    TORCH_CHECK(!records(t), "policy_loss: only the logits get a gradient; detach ", what);
    if (t.scalar_type() != torch::kFloat32) t = t.to(torch::kFloat32);
    if (t.sizes() != tokens.sizes()) t = t.broadcast_to(tokens.sizes());
    if (!t.is_contiguous()) t = t.contiguous();
  };
  like_tokens(old, "old");
  like_tokens(advantages, "advantages");
  if (reference.has_value()) like_tokens(*reference, "reference");
  if (weights.has_value()) like_tokens(*weights, "weights");
  OptTensor total;
  if (!total_of.is_none()) {
    if (THPVariable_Check(total_of.ptr())) {
      total = THPVariable_Unpack(total_of.ptr());
      value(total->numel() == 1 && total->device() == logits.device(), "policy_loss: total, a number or one value on the logits' device");
      TORCH_CHECK(!records(*total), "policy_loss: only the logits get a gradient; detach total");
      if (total->scalar_type() != torch::kFloat32) total = total->to(torch::kFloat32);
    } else {
      total = torch::full({}, total_of.cast<double>(), logits.options().dtype(torch::kFloat32).requires_grad(false));
    }
  }
  tensor_list out;
  if (records(logits)) out = Policy::apply(logits, tokens, old, advantages, reference, weights, total, kl, low, high, temperature);
  else out = policy_forward(logits, tokens, old, advantages, reference, weights, total, PolicyHow{kl, low, high, temperature}, false);
  return {out[0], out[1], out[2], out[3]};
}

// ------------------------------------------------------------------------------------------------ AdamW
// The tensors of a list or tuple, borrowed from it: of some hundred a conversion to a vector is half of what the call costs the host.
struct Tensors {
  pybind11::object held;
  Tensors(const pybind11::object& from) : held(pybind11::reinterpret_steal<pybind11::object>(PySequence_Fast(from.ptr(), "adamw: lists of tensors expected"))) {
    if (!held) throw pybind11::error_already_set();
    for (size_t i = 0; i < size(); ++i) TORCH_CHECK(THPVariable_Check(PySequence_Fast_GET_ITEM(held.ptr(), (Py_ssize_t)i)), "adamw: lists of tensors expected");
  }
  size_t size() const { return (size_t)PySequence_Fast_GET_SIZE(held.ptr()); }
  bool empty() const { return size() == 0; }
  const Tensor& operator[](size_t i) const { return THPVariable_Unpack(PySequence_Fast_GET_ITEM(held.ptr(), (Py_ssize_t)i)); }
};
void adamw_step(const pybind11::object& params_, const pybind11::object& grads_, const pybind11::object& m_, const pybind11::object& v_, const pybind11::object& steps_,
                const pybind11::object& m_scales_, const pybind11::object& v_scales_, const pybind11::object& masters_, double lr, OptTensor lr_on_device, double beta1, double beta2, double eps,
                double weight_decay, bool codes, c10::optional<int64_t> seed) {
  const Tensors params(params_), grads(grads_), m(m_), v(v_), steps(steps_), m_scales(m_scales_), v_scales(v_scales_), masters(masters_);
  const size_t n = params.size();
  TORCH_CHECK(grads.size() == n && m.size() == n && v.size() == n && steps.size() == n && (!codes || (m_scales.size() == n && v_scales.size() == n)) &&
                  (masters.empty() || masters.size() == n), "adamw: one of each for every parameter");
  if (n == 0) return;
  const auto device = params[0].device();
  TORCH_CHECK(device.is_cuda(), "adamw: parameters on the GPU");
  c10::cuda::CUDAGuard guard(device);
  FlAdamwArgs a;
  memset(&a, 0, sizeof a);
  a.lr = lr; a.beta1 = beta1; a.beta2 = beta2; a.eps = eps; a.weight_decay = weight_decay; a.codes = codes; a.master = !masters.empty();
  a.random = seed.has_value(); a.seed = (uint32_t)seed.value_or(0);
  if (lr_on_device.has_value()) {
    TORCH_CHECK(lr_on_device->device() == device && lr_on_device->scalar_type() == torch::kFloat32 && lr_on_device->numel() == 1, "adamw: lr, one fp32 value on the parameters' device");
    a.lr_on_device = lr_on_device->const_data_ptr<float>();
  }
  std::vector<FlAdamwTensor> of[3];
  std::vector<Tensor> kept;                                  // gradients laid out anew, until the launches are on their way
  std::vector<const void*> seen;
  seen.reserve(n);
  const auto kind = codes ? torch::kFloat8_e4m3fn : torch::kFloat32;
  for (size_t i = 0; i < n; ++i) {
    const Tensor& p = params[i];
    const int dt = dtype_of(p, "adamw");
    TORCH_CHECK(p.device() == device && p.layout() == torch::kStrided && p.is_non_overlapping_and_dense(), "adamw: parameters without gaps, all on one device");
    TORCH_CHECK(grads[i].layout() == torch::kStrided && grads[i].device() == device && grads[i].scalar_type() == p.scalar_type() && grads[i].sizes() == p.sizes(),
                "adamw: a dense gradient of its parameter's type, shape and device");
    auto like = [&](const Tensor& t, torch::ScalarType type) { return t.device() == device && t.scalar_type() == type && t.sizes() == p.sizes() && t.strides() == p.strides(); };
    TORCH_CHECK(like(m[i], kind) && like(v[i], kind), "adamw: moments laid out as their parameter, fp32, or e4m3 codes where scales are given");
    TORCH_CHECK(steps[i].device() == device && steps[i].scalar_type() == torch::kInt64 && steps[i].numel() == 1, "adamw: steps, one int64 value per parameter on its device");
    FlAdamwTensor t;
    t.n = p.numel();
    t.m_scale = t.v_scale = t.master = nullptr;
    if (codes)
      for (const auto* s : {&m_scales[i], &v_scales[i]})
        TORCH_CHECK(s->device() == device && s->scalar_type() == torch::kFloat32 && s->is_contiguous() && s->numel() == (t.n + FL_ADAMW_BLOCK - 1) / FL_ADAMW_BLOCK,
                    "adamw: scales, one fp32 value per 256 values of the parameter");
    if (!masters.empty()) {
      TORCH_CHECK(dt != FL_FP32 && like(masters[i], torch::kFloat32), "adamw: fp32 copies are for bf16 and fp16 parameters, and laid out as they are");
      t.master = masters[i].data_ptr<float>();
    }
    Tensor g = grads[i];
    if (g.strides() != p.strides() && t.n > 1) {
      const at::NoGradGuard none;
      g = at::empty_like(p).copy_(g);
      kept.push_back(g);
    }
    t.param = p.data_ptr(); t.grad = const_cast<void*>(g.const_data_ptr()); t.m = m[i].data_ptr(); t.v = v[i].data_ptr();
    if (codes) { t.m_scale = m_scales[i].data_ptr<float>(); t.v_scale = v_scales[i].data_ptr<float>(); }
    t.step = reinterpret_cast<long long*>(steps[i].data_ptr<int64_t>());
    seen.push_back(t.step);
    if (t.n > 0) seen.push_back(t.param);
    of[dt].push_back(t);
  }
  std::sort(seen.begin(), seen.end());
  TORCH_CHECK(std::adjacent_find(seen.begin(), seen.end()) == seen.end(), "adamw: a parameter or its count of steps is given twice");
  for (int dt = 0; dt < 3; ++dt)
    if (!of[dt].empty()) check(fl_adamw(dt, of[dt].data(), (long long)of[dt].size(), &a, stream_of()), "fl_adamw");
  for (const auto* list : {&params, &m, &v, &steps, &m_scales, &v_scales, &masters})
    for (size_t i = 0; i < list->size(); ++i) (*list)[i].unsafeGetTensorImpl()->bump_version();
}

}  // namespace

void fl_train_bind(pybind11::module& m) {
  m.def("embed_lookup", &embed_lookup);
  m.def("route", &route);
  m.def("token_logprobs", &token_logprobs);
  m.def("policy_loss", &policy_loss);
  m.def("adamw_step", &adamw_step);
  m.attr("ROUTE_MAX_EXPERTS") = FL_ROUTE_MAX_EXPERTS;
  m.attr("ADAMW_BLOCK") = FL_ADAMW_BLOCK;
}
