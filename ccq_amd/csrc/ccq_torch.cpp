// The operators around the token mixers as PyTorch sees them: argument checks, output and workspace tensors, autograd,
// one call of the C ABI (include/ccq_hip.h) each way.  In C++ because their calls are short: a training step of small
// rows costs the host half of what the same through Python costs, and the backward runs in autograd's own thread
// without waiting for the interpreter.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <algorithm>
#include <optional>
#include <string>
#include <tuple>

#include "../../include/ccq_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kMaxNorm = 8192, kMaxTop = 64, kMaxVocabulary = int64_t(1) << 30, kMaxStride = int64_t(1) << 22;

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }
const void* address(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out_address(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
Tensor value(const OptTensor& t) { return has(t) ? *t : Tensor(); }

bool known(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf || t == at::kFloat; }
int code(at::ScalarType t) { return t == at::kBFloat16 ? CCQ_DTYPE_BF16 : t == at::kHalf ? CCQ_DTYPE_F16 : CCQ_DTYPE_F32; }

void* stream_on(const Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

void check(int status, const char* what) {
  TORCH_CHECK(status == CCQ_OK, what, " failed (status ", status, "): ", ccq_last_error());
}

void require_gpu(const std::string& who, const Tensor& x) {
  TORCH_CHECK(x.is_cuda(), who, " runs on the GPU only (its input is on the ", x.device().str(), ")");
}
void require_on(const std::string& who, const char* name, const OptTensor& t, const Tensor& x) {
  TORCH_CHECK_VALUE(!has(t) || t->device() == x.device(), who, ": ", name, " must be on ", x.device().str(), " (got ",
                    t.has_value() ? t->device().str() : "", ")");
}

// x [..., D] as [rows, D] with consecutive elements and rows that do not overlap: a view where the strides allow one, a
// copy otherwise.
Tensor rows_of(const Tensor& x) {
  Tensor t = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  if (t.is_contiguous()) return t;
  const bool gaps = t.stride(1) != 1 && t.size(1) > 1, overlap = t.stride(0) < t.size(1) && t.size(0) > 1;
  return gaps || overlap ? t.contiguous() : t;
}
// elements between rows of such a view, at least the row (the stride of a single row is any number)
int64_t stride_of(const Tensor& rows) { return rows.defined() ? std::max(rows.stride(0), rows.size(1)) : 0; }

Tensor like(const Tensor& x) { return at::empty_like(x, at::MemoryFormat::Contiguous); }
Tensor fresh(const Tensor& x, at::IntArrayRef shape, at::ScalarType t) { return at::empty(shape, x.options().dtype(t)); }
Tensor bytes(const Tensor& x, size_t n) { return fresh(x, {(int64_t)n}, at::kByte); }

bool needs_grad(std::initializer_list<const Tensor*> xs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* x : xs)
    if (x->defined() && x->requires_grad()) return true;
  return false;
}

// The kernels have no forward-mode derivatives: an input or an arriving gradient with a tangent is refused, since results
// without one would stand for a derivative of zero.
void refuse_tangents(const std::string& who, std::initializer_list<const Tensor*> xs) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* x : xs)
    TORCH_CHECK_NOT_IMPLEMENTED(!x->defined() || !x->_fw_grad(0).defined(), who, " has no forward-mode derivatives");
}

// A leaf that an earlier graph still holds takes its gradients on the stream where that graph was made.  Under capture
// autograd would wait there for work that is not captured, which ends the process; raised here before it comes to that.
void check_capture(const Tensor& x) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  const c10::Stream here = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).unwrap();
  for (const auto& edge : node->next_edges()) {
    if (!dynamic_cast<torch::autograd::AccumulateGrad*>(edge.function.get())) continue;
    const auto stream = edge.function->stream();
    TORCH_CHECK(!stream || *stream == here, "a backward pass is captured into a graph while a graph of the same leaves from "
                "another stream is alive: drop that one's outputs first");
  }
}

// The kernels have no second derivatives: gradients asked for with a graph of their own carry one that raises.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice an operator that has first derivatives only", (int64_t)grads.size());
  return (*error)(std::move(grads));
}

// ---------------------------------------------------------------------------
// block norms
// ---------------------------------------------------------------------------
struct Normed {
  Tensor y, s, rows, stats;  // s with a residual; stats (mean, then 1 / deviation, of every row) where kept
};
Normed norm_forward(const Tensor& x, const Tensor& residual, const Tensor& weight, const Tensor& bias, bool layer,
                    double eps, bool keep) {
  c10::DeviceGuard guard(x.device());
  Normed o;
  o.rows = rows_of(x);
  const Tensor r = residual.defined() ? rows_of(residual) : Tensor();
  const int64_t rows = o.rows.size(0), D = o.rows.size(1);
  o.y = like(x);
  if (r.defined()) o.s = like(x);
  if (keep) o.stats = fresh(x, {2 * rows}, at::kFloat);
  float* stats = keep ? (float*)out_address(o.stats) : nullptr;
  const auto wtype = weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : x.scalar_type();
  check(ccq_norm_fwd(address(o.rows), stride_of(o.rows), address(r), stride_of(r), address(weight), address(bias),
                     out_address(o.y), out_address(o.s), layer ? stats : nullptr, keep ? stats + rows : nullptr, rows,
                     (int)D, code(x.scalar_type()), code(wtype), layer, (float)eps, stream_on(x)),
        "ccq_norm_fwd");
  return o;
}

struct BlockNorm : torch::autograd::Function<BlockNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& residual, const OptTensor& weight,
                               const OptTensor& bias, bool layer, double eps) {
    Normed o = norm_forward(x, value(residual), value(weight), value(bias), layer, eps, true);
    // the normalised rows: the stream where there is a residual (an output, saved as such), x otherwise
    ctx->save_for_backward({o.s.defined() ? o.s : o.rows, value(weight), o.stats});
    ctx->saved_data["layer"] = layer;
    ctx->saved_data["has"] = (int64_t)(has(residual) | has(weight) << 1 | has(bias) << 2);
    ctx->saved_data["bias"] = (int64_t)(has(bias) ? bias->scalar_type() : x.scalar_type());
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->set_materialize_grads(false);
    return o.s.defined() ? variable_list{o.y, o.s} : variable_list{o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor dx, dr, dw, db;
    {
      at::NoGradGuard no_grad;
      const auto saved = ctx->get_saved_variables();
      const bool layer = ctx->saved_data["layer"].toBool();
      const int64_t present = ctx->saved_data["has"].toInt();
      int edge = 0;
      const bool need_x = ctx->needs_input_grad(edge);
      const bool need_r = present & 1 && ctx->needs_input_grad(++edge);
      const bool need_w = present & 2 && ctx->needs_input_grad(++edge);
      const bool need_b = present & 4 && ctx->needs_input_grad(++edge);
      const Tensor ds = grads.size() > 1 ? grads[1] : Tensor();
      refuse_tangents(layer ? "layer_norm" : "rms_norm", {&grads[0], &ds});
      if (grads[0].defined() || ds.defined()) {
        c10::DeviceGuard guard(saved[0].device());
        check_capture(saved[0]);
        const auto shape = ctx->saved_data["shape"].toIntVector();
        const Tensor x = rows_of(saved[0]);
        const auto type = x.scalar_type();
        // (only the stream was used: no gradient of y)
        const Tensor dy = rows_of(grads[0].defined() ? grads[0] : at::zeros(shape, x.options()));
        const Tensor d = ds.defined() ? rows_of(ds) : Tensor();
        const Tensor& weight = saved[1];
        const auto wtype = weight.defined() ? weight.scalar_type()
                           : present & 4    ? (at::ScalarType)ctx->saved_data["bias"].toInt()
                                            : type;
        const int64_t rows = x.size(0), D = x.size(1);
        if (need_x || need_r) dx = fresh(x, shape, type);
        if (need_w) dw = fresh(x, {D}, wtype);
        if (need_b) db = fresh(x, {D}, wtype);
        Tensor ws;
        if (need_w || need_b) ws = bytes(x, ccq_norm_bwd_workspace_bytes(rows, (int)D, code(type)));
        const float* stats = (const float*)address(saved[2]);
        check(ccq_norm_bwd(address(x), stride_of(x), address(weight), layer ? stats : nullptr, stats + rows, address(dy),
                           stride_of(dy), address(d), stride_of(d), out_address(dx), out_address(dw), out_address(db),
                           out_address(ws), rows, (int)D, code(type), code(wtype), layer, stream_on(x)),
              "ccq_norm_bwd");
        if (need_r) dr = dx;
        if (!need_x) dx = Tensor();
      }
    }
    return once({dx, dr, dw, db, Tensor(), Tensor()});
  }
};

variable_list norm(const std::string& who, const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps,
                   const OptTensor& residual, bool layer) {
  TORCH_CHECK_TYPE(known(x.scalar_type()), who, " takes bf16, fp16 or fp32 rows (got ", x.scalar_type(), ")");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= kMaxNorm, who, ": x ", x.sizes(),
                    ": needs a last dimension in [1, ", kMaxNorm, "]");
  TORCH_CHECK_VALUE(eps >= 0, who, ": eps=", eps, " must not be negative");
  const OptTensor* vectors[] = {&weight, &bias};
  const char* names[] = {"weight", "bias"};
  for (int i = 0; i < 2; ++i) {
    const OptTensor& t = *vectors[i];
    require_on(who, names[i], t, x);
    if (!has(t)) continue;
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == x.size(-1), who, ": ", names[i], " ", t->sizes(), ": expected [",
                      x.size(-1), "]");
    TORCH_CHECK_TYPE(t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat, who, ": ", names[i], " ",
                     t->scalar_type(), ": expected x's type (", x.scalar_type(), ") or fp32");
  }
  TORCH_CHECK_TYPE(!has(weight) || !has(bias) || weight->scalar_type() == bias->scalar_type(), who,
                   ": weight and bias: expected one type");
  require_on(who, "residual", residual, x);
  TORCH_CHECK_VALUE(!has(residual) || (residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type()), who,
                    ": residual: expected x's shape ", x.sizes(), " and type ", x.scalar_type());
  const Tensor r = value(residual), w = has(weight) ? weight->contiguous() : Tensor(),
               b = has(bias) ? bias->contiguous() : Tensor();
  refuse_tangents(who, {&x, &r, &w, &b});
  require_gpu(who, x);
  if (needs_grad({&x, &r, &w, &b})) {
    auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    return BlockNorm::apply(x, opt(r), opt(w), opt(b), layer, eps);
  }
  Normed o = norm_forward(x, r, w, b, layer, eps, false);
  return o.s.defined() ? variable_list{o.y, o.s} : variable_list{o.y};
}

// ---------------------------------------------------------------------------
// log probabilities of given tokens
// ---------------------------------------------------------------------------
struct Scored {
  Tensor logp, entropy, top, top_ids, rows, ids, stats;
};
Scored score_forward(const Tensor& logits, const Tensor& ids, int64_t k, int64_t ignore, bool keep) {
  c10::DeviceGuard guard(logits.device());
  Scored o;
  o.rows = rows_of(logits);
  o.ids = ids.contiguous();
  const int64_t rows = o.rows.size(0), V = o.rows.size(1);
  o.logp = fresh(logits, ids.sizes(), at::kFloat);
  o.entropy = fresh(logits, ids.sizes(), at::kFloat);
  if (keep) o.stats = fresh(logits, {2 * rows}, at::kFloat);
  if (k) {
    auto shape = ids.sizes().vec();
    shape.push_back(k);
    o.top = fresh(logits, shape, at::kFloat);
    o.top_ids = fresh(logits, shape, at::kLong);
  }
  check(ccq_token_logprobs_fwd(address(o.rows), stride_of(o.rows), (const int64_t*)address(o.ids),
                               (float*)out_address(o.logp), (float*)out_address(o.entropy), (float*)out_address(o.stats),
                               (float*)out_address(o.top), (int64_t*)out_address(o.top_ids), rows, (int)V, (int)k, ignore,
                               code(logits.scalar_type()), stream_on(logits)),
        "ccq_token_logprobs_fwd");
  return o;
}

struct TokenScore : torch::autograd::Function<TokenScore> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& ids, int64_t k, int64_t ignore) {
    Scored o = score_forward(logits, ids, k, ignore, true);
    ctx->save_for_backward({o.rows, o.ids, o.entropy, o.stats});
    ctx->saved_data["shape"] = logits.sizes().vec();
    ctx->saved_data["ignore"] = ignore;
    ctx->set_materialize_grads(false);
    if (!k) return {o.logp, o.entropy};
    ctx->mark_non_differentiable({o.top, o.top_ids});
    return {o.logp, o.entropy, o.top, o.top_ids};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor dx;
    refuse_tangents("token_logprobs", {&grads[0], &grads[1]});
    if (grads[0].defined() || grads[1].defined()) {
      at::NoGradGuard no_grad;
      const auto saved = ctx->get_saved_variables();
      const Tensor& x = saved[0];
      c10::DeviceGuard guard(x.device());
      check_capture(x);
      const Tensor dlogp = grads[0].defined() ? grads[0].contiguous() : Tensor(),
                   dent = grads[1].defined() ? grads[1].contiguous() : Tensor();
      dx = fresh(x, ctx->saved_data["shape"].toIntVector(), x.scalar_type());
      check(ccq_token_logprobs_bwd(address(x), stride_of(x), (const int64_t*)address(saved[1]),
                                   (const float*)address(saved[2]), (const float*)address(saved[3]),
                                   (const float*)address(dlogp), (const float*)address(dent), out_address(dx), x.size(0),
                                   (int)x.size(1), ctx->saved_data["ignore"].toInt(), code(x.scalar_type()), stream_on(x)),
            "ccq_token_logprobs_bwd");
    }
    return once({dx, Tensor(), Tensor(), Tensor()});
  }
};

variable_list token_logprobs(const Tensor& logits, const Tensor& ids, int64_t top_k, int64_t ignore) {
  const char* who = "token_logprobs";
  TORCH_CHECK_TYPE(known(logits.scalar_type()), who, " takes bf16, fp16 or fp32 logits (got ", logits.scalar_type(), ")");
  TORCH_CHECK_TYPE(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, who,
                   " takes int64 or int32 ids (got ", ids.scalar_type(), ")");
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1 && ids.sizes() == logits.sizes().slice(0, logits.dim() - 1),
                    who, ": ids ", ids.sizes(), ": expected the positions of logits ", logits.sizes());
  TORCH_CHECK_VALUE(logits.size(-1) <= kMaxVocabulary, who, ": logits ", logits.sizes(), ": needs a last dimension of at most ",
                    kMaxVocabulary);
  require_on(who, "ids", ids, logits);
  const int64_t most = std::min(kMaxTop, logits.size(-1));
  TORCH_CHECK_VALUE(top_k >= 0 && top_k <= most, who, ": top_k=", top_k, " must lie in [0, ", most, "]");
  refuse_tangents(who, {&logits});
  require_gpu(who, logits);
  const Tensor i = ids.to(at::kLong);
  if (needs_grad({&logits})) return TokenScore::apply(logits, i, top_k, ignore);
  Scored o = score_forward(logits, i, top_k, ignore, false);
  return top_k ? variable_list{o.logp, o.entropy, o.top, o.top_ids} : variable_list{o.logp, o.entropy};
}

// ---------------------------------------------------------------------------
// linear map with an epilogue
// ---------------------------------------------------------------------------
// Rows as the products read them: 16-byte pieces, zeros up to a multiple of 8 columns.  A copy where the width, stride or
// address does not allow that.
Tensor operand(const Tensor& rows) {
  const int64_t n = rows.size(0), K = rows.size(1), ld = stride_of(rows);
  if (K % 8 == 0 && ld % 8 == 0 && ld <= kMaxStride && (size_t)address(rows) % 16 == 0) return rows;
  const int64_t ldd = (K + 7) / 8 * 8;
  Tensor out = fresh(rows, {n, ldd}, rows.scalar_type());
  check(ccq_pad_rows(address(rows), ld, out_address(out), ldd, n, K, stream_on(rows)), "ccq_pad_rows");
  return out;
}

struct Mapped {
  Tensor y, z, x, w;
};
Mapped linear_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, int act,
                      bool keep_z) {
  c10::DeviceGuard guard(x.device());
  Mapped o;
  o.x = rows_of(x);
  o.w = rows_of(weight);
  const int64_t M = o.x.size(0), K = o.x.size(1), outs = o.w.size(0), N = act == CCQ_ACT_SWIGLU ? outs / 2 : outs;
  const Tensor r = residual.defined() ? rows_of(residual) : Tensor();
  auto shape = x.sizes().vec();
  shape.back() = N;
  o.y = fresh(x, shape, x.scalar_type());
  if (keep_z && act != CCQ_ACT_NONE) o.z = bytes(x, 3 * M * ((outs + 7) / 8 * 8));  // 24 bits a value
  const Tensor a = operand(o.x), b = operand(o.w);
  const size_t n = ccq_linear_workspace_bytes(M, N, K, act);
  const Tensor ws = n ? bytes(x, n) : Tensor();
  check(ccq_linear_fwd(address(a), stride_of(a), address(b), stride_of(b), address(bias),
                       code(bias.defined() ? bias.scalar_type() : x.scalar_type()), address(r), stride_of(r),
                       out_address(o.y), out_address(o.z), out_address(ws), M, N, K, act, code(x.scalar_type()),
                       stream_on(x)),
        "ccq_linear_fwd");
  return o;
}

struct FusedLinear : torch::autograd::Function<FusedLinear> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& bias,
                               const OptTensor& residual, int64_t act) {
    const bool keep_z = x.requires_grad() || weight.requires_grad() || (has(bias) && bias->requires_grad());
    Mapped o = linear_forward(x, weight, value(bias), value(residual), (int)act, keep_z);
    ctx->save_for_backward({o.x, o.w, o.z});
    ctx->saved_data["act"] = act;
    ctx->saved_data["has"] = (int64_t)(has(bias) | has(residual) << 1);
    ctx->saved_data["bias"] = (int64_t)(has(bias) ? bias->scalar_type() : x.scalar_type());
    ctx->saved_data["shape"] = x.sizes().vec();
    return {o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor dx, dw, db, dr;
    {
      at::NoGradGuard no_grad;
      const auto saved = ctx->get_saved_variables();
      const Tensor &x = saved[0], &w = saved[1], &dy = grads[0];
      const int act = (int)ctx->saved_data["act"].toInt();
      const int64_t present = ctx->saved_data["has"].toInt();
      const auto btype = (at::ScalarType)ctx->saved_data["bias"].toInt();
      int edge = 1;
      refuse_tangents("fused_linear", {&dy});
      const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
      const bool need_b = present & 1 && ctx->needs_input_grad(++edge);
      const bool need_r = present & 2 && ctx->needs_input_grad(++edge);
      c10::DeviceGuard guard(x.device());
      check_capture(x);
      if (need_x || need_w || need_b) {
        const int64_t M = x.size(0), K = x.size(1), outs = w.size(0), N = act == CCQ_ACT_SWIGLU ? outs / 2 : outs;
        const int64_t ld = (K + 7) / 8 * 8;
        const auto type = x.scalar_type();
        const Tensor d = rows_of(dy);
        if (need_x) dx = fresh(x, ctx->saved_data["shape"].toIntVector(), type);
        if (need_w) dw = fresh(x, {outs, K}, type);
        if (need_b) db = fresh(x, {outs}, btype);
        const Tensor a = need_w ? operand(x) : Tensor(), b = need_x ? operand(w) : Tensor();
        const size_t n = ccq_linear_bwd_call_workspace_bytes(M, N, K, act, address(d), stride_of(d), need_x, need_w, need_b);
        const Tensor ws = n ? bytes(x, n) : Tensor();
        check(ccq_linear_bwd(address(a), need_w ? stride_of(a) : ld, address(b), need_x ? stride_of(b) : ld,
                             address(saved[2]), address(d), stride_of(d), out_address(dx), out_address(dw),
                             out_address(db), code(btype), out_address(ws), M, N, K, act, code(type), stream_on(x)),
              "ccq_linear_bwd");
      }
      if (need_r) dr = dy;
    }
    return once({dx, dw, db, dr, Tensor()});
  }
};

Tensor fused_linear(const Tensor& x, const Tensor& weight, const OptTensor& bias, int64_t act, const OptTensor& residual) {
  const char* who = "fused_linear";
  TORCH_CHECK_TYPE((x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf) && weight.scalar_type() == x.scalar_type(),
                   who, " takes bf16 or fp16 x and weight of one type (got ", x.scalar_type(), ", ", weight.scalar_type(), ")");
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 2 && weight.size(1) == x.size(-1) && x.size(-1) >= 1 &&
                        x.size(-1) <= kMaxStride && weight.size(0) >= 1 && weight.size(0) <= kMaxStride,
                    who, ": x ", x.sizes(), " and weight ", weight.sizes(),
                    ": expected [..., K] and [outputs, K], both at least 1 wide and at most ", kMaxStride);
  const int64_t outs = weight.size(0), N = act == CCQ_ACT_SWIGLU ? outs / 2 : outs;
  TORCH_CHECK_VALUE(act != CCQ_ACT_SWIGLU || outs % 2 == 0, who, ": swiglu needs as many gate as up rows (weight has ", outs, ")");
  require_on(who, "weight", weight, x);
  require_on(who, "bias", bias, x);
  require_on(who, "residual", residual, x);
  TORCH_CHECK_VALUE(!has(bias) || (bias->dim() == 1 && bias->size(0) == outs), who, ": bias: expected [", outs, "]");
  TORCH_CHECK_TYPE(!has(bias) || bias->scalar_type() == x.scalar_type() || bias->scalar_type() == at::kFloat, who,
                   ": bias: expected x's type (", x.scalar_type(), ") or fp32");
  auto shape = x.sizes().vec();
  shape.back() = N;
  TORCH_CHECK_VALUE(!has(residual) || (residual->sizes() == at::IntArrayRef(shape) && residual->scalar_type() == x.scalar_type()),
                    who, ": residual: expected ", at::IntArrayRef(shape), " ", x.scalar_type());
  const Tensor b = has(bias) ? bias->contiguous() : Tensor(), r = value(residual);
  refuse_tangents(who, {&x, &weight, &b, &r});
  require_gpu(who, x);
  if (needs_grad({&x, &weight, &b, &r})) {
    auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    return FusedLinear::apply(x, weight, opt(b), opt(r), act)[0];
  }
  return linear_forward(x, weight, b, r, (int)act, false).y;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("norm", [](const std::string& who, const Tensor& x, const OptTensor& w, const OptTensor& b, double eps, bool layer) {
    return norm(who, x, w, b, eps, OptTensor(), layer)[0];
  });
  m.def("norm_residual", [](const std::string& who, const Tensor& x, const OptTensor& w, const OptTensor& b, double eps,
                            const Tensor& residual, bool layer) {
    variable_list o = norm(who, x, w, b, eps, residual, layer);
    return std::make_tuple(o[0], o[1]);
  });
  m.def("token_logprobs", &token_logprobs);
  m.def("fused_linear", &fused_linear);
}
