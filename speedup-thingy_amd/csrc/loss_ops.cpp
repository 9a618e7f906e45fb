// Autograd nodes of the token losses and the pool balance (librte_ops.so, torch.ops.rte.*), over the C entry points
// of librte_hip.
//
// Small calls are bound by the host: forward and backward of a 64 x 2048 divergence take 85 us with a node in Python
// for 12 us of kernels (autograd's thread waits for the interpreter), and 58 with these.
//
// The Python wrappers (rte_amd/kernels/hip_ops.py) check arguments with the framework's errors; here only what a kernel
// could not survive is checked again.  `stream` is the current stream on the operands' device: a node's backward runs
// on the stream of its forward, so it is kept for that.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include "../../include/rte_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

void ok(int rc, const char* entry) { TORCH_CHECK(rc == 0, entry, " failed (code ", rc, "): ", rte_last_error()); }

Tensor dense(const Tensor& t, at::ScalarType dtype) {
  return t.scalar_type() == dtype && t.is_contiguous() ? t : t.contiguous().to(dtype);
}

// Rows x [..., V] on a device, in a type of the kernels.
void check_rows(const char* op, const Tensor& x) {
  TORCH_CHECK(x.is_cuda(), op, ": expects ROCm device tensors");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && (x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16), op,
              ": float32 or bfloat16 rows expected");
}
// An operand of n values for every row of x.
void check_beside(const char* op, const Tensor& x, const Tensor& t, int64_t n) {
  TORCH_CHECK(t.device() == x.device() && n >= 1 && t.numel() == x.numel() / x.size(-1) * n, op,
              ": an operand does not match the rows");
}

// Ids in 32 bits; wider ones that do not fit stay out of every range.
Tensor ids32(const Tensor& t) {
  return dense(t.scalar_type() == at::kLong ? t.clamp(-1, 0x7fffffff) : t, at::kInt);
}

// x [..., V] as rows with contiguous columns, a view where its strides allow, and their stride.
std::pair<Tensor, int64_t> rows_of(const Tensor& x) {
  const int64_t V = x.size(-1);
  if (x.is_contiguous()) return {x, V};
  Tensor r = x.reshape({-1, V});
  if (r.stride(1) != 1 && V > 1) r = r.contiguous();
  return {r, r.stride(0)};
}

Tensor scratch(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

template <class T>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

Tensor row_grad(const Tensor& g) { return g.defined() ? dense(g, at::kFloat) : g; }

// A gradient that a graph of gradients (create_graph) may pass on, but not differentiate.
Tensor once(Tensor dx, const char* op) {
  if (!at::GradMode::is_enabled() || !dx.defined()) return dx;
  const auto stop =
      std::make_shared<torch::autograd::DelayedError>(std::string(op) + ": its gradient cannot be differentiated", 1);
  return stop->apply(variable_list{dx.requires_grad_()})[0];
}

void* stream_of(AutogradContext* ctx) { return reinterpret_cast<void*>(ctx->saved_data["stream"].toInt()); }

bool wants_grad(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

// A call that passes its autograd node by would lose a tangent without a word, as a derivative of 0.
void no_tangent(const char* op, const Tensor& t) {
  TORCH_CHECK(!t._fw_grad(/*level=*/0).defined(), op, ": forward-mode derivatives are not implemented");
}

// ---------------------------------------------------------------- log probabilities from logits

struct Logprobs {
  Tensor lp, ent, top_lp, top_ids, stats, rows, tokens;
  int64_t ld;
};

Logprobs logprobs(const Tensor& logits, const Tensor& tokens, int64_t n_top, double temperature, bool need, int64_t stream) {
  check_rows("token_logprobs", logits);
  check_beside("token_logprobs", logits, tokens, 1);
  TORCH_CHECK(n_top >= 0 && n_top <= logits.size(-1), "token_logprobs: n_top must be in [0, V]");
  c10::DeviceGuard guard(logits.device());
  Logprobs r;
  std::tie(r.rows, r.ld) = rows_of(logits);
  r.tokens = dense(tokens, at::kLong);
  const int64_t T = r.tokens.numel(), V = logits.size(-1);
  const auto f32 = logits.options().dtype(at::kFloat).requires_grad(false);
  r.lp = at::empty(tokens.sizes(), f32);
  r.ent = at::empty(tokens.sizes(), f32);
  std::vector<int64_t> top = tokens.sizes().vec();
  top.push_back(n_top);
  r.top_lp = at::empty(top, f32);
  r.top_ids = at::empty(top, f32.dtype(at::kInt));
  if (need) r.stats = at::empty({T, 2}, f32);
  const size_t n = rte_token_logprobs_workspace_bytes((int)T, (int)V, (int)n_top);
  const Tensor ws = scratch(n, r.lp);
  ok(rte_token_logprobs_fwd(r.rows.data_ptr(), r.ld, logits.scalar_type() == at::kFloat, (int)T, (int)V,
                            ptr<int64_t>(r.tokens), (float)temperature, (int)n_top, ptr<float>(r.lp), ptr<float>(r.ent),
                            ptr<float>(r.top_lp), ptr<int32_t>(r.top_ids), ptr<float>(r.stats), ptr<void>(ws), n,
                            reinterpret_cast<void*>(stream)),
     "rte_token_logprobs_fwd");
  return r;
}

struct TokenLogprobs : Function<TokenLogprobs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, int64_t n_top,
                               double temperature, int64_t stream) {
    Logprobs r = logprobs(logits, tokens, n_top, temperature, true, stream);
    ctx->save_for_backward({r.rows, r.tokens, r.stats, r.ent});
    ctx->saved_data["ld"] = r.ld;
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["stream"] = stream;
    ctx->saved_data["shape"] = logits.sizes();
    ctx->mark_non_differentiable({r.top_lp, r.top_ids});
    ctx->set_materialize_grads(false);
    return {r.lp, r.ent, r.top_lp, r.top_ids};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined() && !g[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor &rows = saved[0], &tokens = saved[1];
    const Tensor gl = row_grad(g[0]), ge = row_grad(g[1]);
    const Tensor dx = at::empty(ctx->saved_data["shape"].toIntVector(), rows.options());
    ok(rte_token_logprobs_bwd(rows.data_ptr(), ctx->saved_data["ld"].toInt(), rows.scalar_type() == at::kFloat,
                              (int)tokens.numel(), (int)rows.size(-1), ptr<int64_t>(tokens),
                              (float)ctx->saved_data["temperature"].toDouble(), ptr<float>(saved[2]), ptr<float>(saved[3]),
                              ptr<float>(gl), ptr<float>(ge), dx.data_ptr(), stream_of(ctx)),
       "rte_token_logprobs_bwd");
    return {once(dx, "token_logprobs"), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};


std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs(const Tensor& logits, const Tensor& tokens, int64_t n_top,
                                                          double temperature, int64_t stream) {
  no_tangent("token_logprobs", logits);
  if (wants_grad(logits)) {
    const auto r = TokenLogprobs::apply(logits, tokens, n_top, temperature, stream);
    return {r[0], r[1], r[2], r[3]};
  }
  const Logprobs r = logprobs(logits.detach(), tokens, n_top, temperature, false, stream);
  return {r.lp, r.ent, r.top_lp, r.top_ids};
}

// ---------------------------------------------------------------- divergence from a teacher's list

struct Distill {
  Tensor loss, stats, cols, coef, rows;
  int64_t ld;
};

Distill distill(const Tensor& logits, const Tensor& ids, const Tensor& teacher, double temperature, bool tail, bool need,
                int64_t stream) {
  check_rows("topk_distill", logits);
  TORCH_CHECK(ids.dim() >= 1, "topk_distill: lists expected");
  check_beside("topk_distill", logits, ids, ids.size(-1));
  check_beside("topk_distill", logits, teacher, ids.size(-1));
  c10::DeviceGuard guard(logits.device());
  Distill r;
  std::tie(r.rows, r.ld) = rows_of(logits);
  const Tensor ic = ids32(ids), tc = dense(teacher, at::kFloat);
  const int64_t K = ids.size(-1), T = ids.numel() / K, V = logits.size(-1);
  const auto f32 = logits.options().dtype(at::kFloat).requires_grad(false);
  r.loss = at::empty(logits.sizes().slice(0, logits.dim() - 1), f32);
  if (need) {
    r.stats = at::empty({T, 2}, f32);
    r.cols = at::empty({T, K}, f32.dtype(at::kInt));
    r.coef = at::empty({T, K}, f32);
  }
  const auto kept = teacher.scalar_type();
  const int rest = !tail ? 0 : kept == at::kBFloat16 ? 2 : kept == at::kHalf ? 3 : 1;
  const size_t n = rte_topk_distill_workspace_bytes((int)T, (int)V, (int)K);
  const Tensor ws = scratch(n, r.loss);
  ok(rte_topk_distill_fwd(r.rows.data_ptr(), r.ld, logits.scalar_type() == at::kFloat, (int)T, (int)V, ptr<int32_t>(ic),
                          ptr<float>(tc), (int)K, (float)temperature, rest, ptr<float>(r.loss), ptr<float>(r.stats),
                          ptr<int32_t>(r.cols), ptr<float>(r.coef), ptr<void>(ws), n, reinterpret_cast<void*>(stream)),
     "rte_topk_distill_fwd");
  return r;
}

struct TopkDistill : Function<TopkDistill> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& ids, const Tensor& teacher,
                        double temperature, bool tail, int64_t stream) {
    Distill r = distill(logits, ids, teacher, temperature, tail, true, stream);
    ctx->save_for_backward({r.rows, r.stats, r.cols, r.coef});
    ctx->saved_data["ld"] = r.ld;
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["stream"] = stream;
    ctx->saved_data["shape"] = logits.sizes();
    ctx->set_materialize_grads(false);
    return r.loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor &rows = saved[0], &cols = saved[2];
    const Tensor gl = row_grad(g[0]);
    const Tensor dx = at::empty(ctx->saved_data["shape"].toIntVector(), rows.options());
    ok(rte_topk_distill_bwd(rows.data_ptr(), ctx->saved_data["ld"].toInt(), rows.scalar_type() == at::kFloat,
                            (int)cols.size(0), (int)rows.size(-1), (int)cols.size(1),
                            (float)ctx->saved_data["temperature"].toDouble(), ptr<float>(saved[1]), ptr<int32_t>(cols),
                            ptr<float>(saved[3]), ptr<float>(gl), dx.data_ptr(), stream_of(ctx)),
       "rte_topk_distill_bwd");
    return {once(dx, "topk_distill"), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor topk_distill(const Tensor& logits, const Tensor& ids, const Tensor& teacher, double temperature, bool tail,
                    int64_t stream) {
  no_tangent("topk_distill", logits);
  no_tangent("topk_distill", teacher);
  const Tensor t = teacher.detach();
  if (wants_grad(logits)) return TopkDistill::apply(logits, ids, t, temperature, tail, stream);
  return distill(logits.detach(), ids, t, temperature, tail, false, stream).loss;
}

// ---------------------------------------------------------------- load balance of routed pools

struct PoolBalance : Function<PoolBalance> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& ids, const OptTensor& mask,
                               int64_t stream) {
    check_rows("pool_balance", logits);
    TORCH_CHECK(ids.dim() >= 1, "pool_balance: lists expected");
    check_beside("pool_balance", logits, ids, ids.size(-1));
    if (mask) {
      check_beside("pool_balance", logits, *mask, 1);
      TORCH_CHECK(mask->scalar_type() == at::kBool, "pool_balance: mask must be bool");
    }
    c10::DeviceGuard guard(logits.device());
    const auto [rows, ld] = rows_of(logits);
    const int64_t C = logits.size(-1), k = ids.size(-1), T = ids.numel() / k;
    const Tensor ic = ids32(ids), mc = mask ? mask->contiguous() : Tensor();
    const auto f32 = logits.options().dtype(at::kFloat).requires_grad(false);
    const Tensor out = at::empty({2}, f32), counts = at::empty({C}, f32.dtype(at::kInt)), frac = at::empty({C + 1}, f32);
    const size_t n = rte_pool_balance_workspace_bytes((int)T, (int)C);
    const Tensor ws = scratch(n, out);
    ok(rte_pool_balance_fwd(rows.data_ptr(), ld, logits.scalar_type() == at::kFloat, (int)T, (int)C, ptr<int32_t>(ic), (int)k,
                            ptr<uint8_t>(mc), ptr<float>(out), ptr<int32_t>(counts), ptr<float>(frac), ptr<void>(ws), n,
                            reinterpret_cast<void*>(stream)),
       "rte_pool_balance_fwd");
    ctx->save_for_backward({rows, mc, frac});
    ctx->saved_data["ld"] = ld;
    ctx->saved_data["rows"] = T;
    ctx->saved_data["stream"] = stream;
    ctx->saved_data["shape"] = logits.sizes();
    ctx->mark_non_differentiable({counts});
    ctx->set_materialize_grads(false);
    // no views of each other for autograd: a caller may change one in place
    return {out.select(0, 0).variable_data(), out.select(0, 1).variable_data(), counts};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined() && !g[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor& rows = saved[0];
    const Tensor gb = row_grad(g[0]), gz = row_grad(g[1]);
    const Tensor dx = at::empty(ctx->saved_data["shape"].toIntVector(), rows.options());
    ok(rte_pool_balance_bwd(rows.data_ptr(), ctx->saved_data["ld"].toInt(), rows.scalar_type() == at::kFloat,
                            (int)ctx->saved_data["rows"].toInt(), (int)rows.size(-1), ptr<uint8_t>(saved[1]),
                            ptr<float>(saved[2]), ptr<float>(gb), ptr<float>(gz), dx.data_ptr(), stream_of(ctx)),
       "rte_pool_balance_bwd");
    return {once(dx, "pool_balance"), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor, Tensor> pool_balance(const Tensor& logits, const Tensor& ids, const OptTensor& mask,
                                                int64_t stream) {
  const auto r = PoolBalance::apply(logits, ids, mask, stream);
  return {r[0], r[1], r[2]};
}

// ---------------------------------------------------------------- log probabilities from hidden states

// hidden and w carry the graph; hb [T, d] and wb [V, d] are their bf16 values, of sizes that the tile product takes
// (rte_lm_head_logprobs_ok).  grad_bytes bounds the logits' gradient that is held at a time.
struct HeadLogprobs : Function<HeadLogprobs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& w, const Tensor& hb,
                               const Tensor& wb, const Tensor& tokens, double temperature, int64_t grad_bytes,
                               int64_t stream) {
    for (const Tensor* t : {&hb, &wb}) {
      check_rows("lm_head_logprobs", *t);
      TORCH_CHECK(t->dim() == 2 && t->scalar_type() == at::kBFloat16 && t->is_contiguous() && t->size(1) == hb.size(1) &&
                      t->device() == hb.device(),
                  "lm_head_logprobs: dense bfloat16 matrices of one width expected");
    }
    check_beside("lm_head_logprobs", hb, tokens, 1);
    TORCH_CHECK(hidden.numel() == hb.numel() && w.sizes() == wb.sizes(), "lm_head_logprobs: the copies do not match");
    c10::DeviceGuard guard(hb.device());
    const Tensor tk = dense(tokens, at::kLong);
    const int64_t T = hb.size(0), d = hb.size(1), V = wb.size(0);
    const auto f32 = hb.options().dtype(at::kFloat).requires_grad(false);
    const Tensor lp = at::empty(tokens.sizes(), f32), ent = at::empty(tokens.sizes(), f32), stats = at::empty({T, 2}, f32);
    const size_t n = rte_lm_head_logprobs_workspace_bytes((int)T, (int)V);
    const Tensor ws = scratch(n, lp);
    ok(rte_lm_head_logprobs_fwd(hb.data_ptr(), wb.data_ptr(), (int)T, (int)d, (int)V, ptr<int64_t>(tk), (float)temperature,
                                ptr<float>(lp), ptr<float>(ent), ptr<float>(stats), ptr<void>(ws), n,
                                reinterpret_cast<void*>(stream)),
       "rte_lm_head_logprobs_fwd");
    ctx->save_for_backward({hb, wb, tk, stats, ent});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["grad_bytes"] = grad_bytes;
    ctx->saved_data["stream"] = stream;
    ctx->saved_data["shape"] = hidden.sizes();
    ctx->saved_data["h_dtype"] = hidden.scalar_type();
    ctx->saved_data["w_dtype"] = w.scalar_type();
    ctx->set_materialize_grads(false);
    return {lp, ent};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(8);
    if (!g[0].defined() && !g[1].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor &hb = saved[0], &wb = saved[1];
    const Tensor gl = row_grad(g[0]), ge = row_grad(g[1]);
    const int64_t T = hb.size(0), d = hb.size(1), V = wb.size(0);
    const bool need_h = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const auto h_dtype = ctx->saved_data["h_dtype"].toScalarType(), w_dtype = ctx->saved_data["w_dtype"].toScalarType();
    const bool h_bf16 = h_dtype == at::kBFloat16, w_bf16 = w_dtype == at::kBFloat16;
    int64_t width = ctx->saved_data["grad_bytes"].toInt() / (2 * T);
    width = std::max<int64_t>(64, std::min(width, V) / 64 * 64);
    Tensor dh, dw;
    if (need_h) dh = at::empty({T, d}, hb.options().dtype(h_bf16 ? at::kBFloat16 : at::kFloat));
    if (need_w) dw = at::empty({V, d}, hb.options().dtype(w_bf16 ? at::kBFloat16 : at::kFloat));
    const int dh_type = need_h ? (h_bf16 ? 1 : 2) : 0;
    const size_t n = rte_lm_head_logprobs_bwd_workspace_bytes((int)T, (int)d, (int)V, (int)width, dh_type, need_w);
    const Tensor ws = scratch(n, hb);
    ok(rte_lm_head_logprobs_bwd(hb.data_ptr(), wb.data_ptr(), (int)T, (int)d, (int)V, ptr<int64_t>(saved[2]),
                                (float)ctx->saved_data["temperature"].toDouble(), ptr<float>(saved[3]), ptr<float>(saved[4]),
                                ptr<float>(gl), ptr<float>(ge), (int)width, ptr<void>(dh), ptr<void>(dw),
                                (w_bf16 ? 0 : 1) + (h_bf16 ? 0 : 2), ptr<void>(ws), n, stream_of(ctx)),
       "rte_lm_head_logprobs_bwd");
    if (need_h) out[0] = once(dh.view(ctx->saved_data["shape"].toIntVector()).to(h_dtype), "lm_head_logprobs");
    if (need_w) out[1] = once(dw.to(w_dtype), "lm_head_logprobs");
    return out;
  }
};

std::tuple<Tensor, Tensor> lm_head_logprobs(const Tensor& hidden, const Tensor& w, const Tensor& hb, const Tensor& wb,
                                            const Tensor& tokens, double temperature, int64_t grad_bytes, int64_t stream) {
  const auto r = HeadLogprobs::apply(hidden, w, hb, wb, tokens, temperature, grad_bytes, stream);
  return {r[0], r[1]};
}

}  // namespace

TORCH_LIBRARY(rte, m) {
  m.def("token_logprobs(Tensor logits, Tensor tokens, int n_top, float temperature, int stream) -> "
        "(Tensor, Tensor, Tensor, Tensor)", &token_logprobs);
  m.def("topk_distill(Tensor logits, Tensor ids, Tensor teacher, float temperature, bool tail, int stream) -> Tensor",
        &topk_distill);
  m.def("pool_balance(Tensor logits, Tensor ids, Tensor? mask, int stream) -> (Tensor, Tensor, Tensor)", &pool_balance);
  m.def("lm_head_logprobs(Tensor hidden, Tensor w, Tensor hb, Tensor wb, Tensor tokens, float temperature, "
        "int grad_bytes, int stream) -> (Tensor, Tensor)", &lm_head_logprobs);
}
