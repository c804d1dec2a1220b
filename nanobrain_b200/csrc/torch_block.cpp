// PyTorch side of include/nb_block.h: the CUDA and autograd kernels of the nanobrain_b200::qk_norm_rope_* and
// gated_mlp_* ops (schemas and fake kernels: block_ops.py) and the two entry points that Python calls. Everything
// numeric stays behind the C ABI; arguments outside the supported subset raise.
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <array>
#include <cmath>
#include <optional>
#include <tuple>
#include <vector>

#include "../../include/nb_block.h"
#include "torch_common.h"

namespace {

using at::Tensor;
using nbt::check_rc;
using nbt::kHeadDim;
using nbt::new_tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

bool has(const MaybeTensor& t) { return t.has_value() && t->defined(); }
Tensor or_none(const MaybeTensor& t) { return has(t) ? *t : Tensor(); }
MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }
bool differentiable(const MaybeTensor& t) { return has(t) && t->requires_grad(); }

void* stream_of_current_device() { return at::cuda::getCurrentCUDAStream().stream(); }

template <typename Sig>
c10::TypedOperatorHandle<Sig> find_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
}

// ------------------------------------------------------------------------------------------
// Norms and rotation of queries and keys
// ------------------------------------------------------------------------------------------
#define QK_REQUIRE(cond, ...) TORCH_CHECK(cond, "nanobrain_b200.qk_norm_rope: ", __VA_ARGS__)

using Two = std::tuple<Tensor, Tensor>;
using Four = std::tuple<Tensor, Tensor, Tensor, Tensor>;
using QkFwdSig = Two(const Tensor&, const Tensor&, const MaybeTensor&, const MaybeTensor&, const MaybeTensor&,
                     const MaybeTensor&, const MaybeTensor&, double, bool);
using QkBwdSig = Four(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const MaybeTensor&, const MaybeTensor&,
                      const MaybeTensor&, const MaybeTensor&, const MaybeTensor&, double, bool);

void check_heads(const Tensor& t, const char* name) {
  QK_REQUIRE(t.is_cuda(), name, " must be a CUDA tensor (there is no CPU path)");
  QK_REQUIRE(t.scalar_type() == at::kBFloat16, name, " must be bfloat16, got ", t.scalar_type());
  QK_REQUIRE(t.dim() == 3 || t.dim() == 4, name, " must be [T, H, 64] or [B, H, L, 64], got ", t.dim(), " dimensions");
  QK_REQUIRE(t.size(-1) == kHeadDim, "head_dim must be ", kHeadDim, ", got ", t.size(-1));
}

struct QkCall {
  nb_qk_norm_rope_args args{};
  std::vector<Tensor> keep;  // copies that the arguments point into
};

nb_attn_tensor desc_of(const Tensor& t) { return t.dim() == 4 ? nbt::dense_desc(t) : nbt::packed_desc(t); }
Tensor layout_of(const Tensor& t) { return t.dim() == 4 ? nbt::dense_layout(t) : nbt::packed_layout(t); }
Tensor new_like(const Tensor& t) {
  return t.dim() == 4 ? nbt::new_dense(t) : new_tensor(t.sizes(), at::kBFloat16, t);
}

void check_qk(const Tensor& q, const Tensor& k) {
  check_heads(q, "q");
  check_heads(k, "k");
  QK_REQUIRE(q.device() == k.device(), "q and k must be on the same device");
  QK_REQUIRE(q.dim() == k.dim(), "q and k must both be packed or both dense");
  QK_REQUIRE(q.dim() == 3 || q.size(0) == k.size(0), "q and k must agree on the batch");
  for (const Tensor& t : {q, k}) {
    QK_REQUIRE(t.size(1) > 0 && t.size(1) <= 65535, "there must be 1 to 65535 heads, got ", t.size(1));
    QK_REQUIRE(t.numel() / (t.size(1) * kHeadDim) <= INT32_MAX, "there must be fewer than 2^31 tokens");
  }
}

void set_side(QkCall& c, nb_qk_side& s, const Tensor& x, const MaybeTensor& weight, const char* weight_name,
              const MaybeTensor& positions, const char* positions_name) {
  const bool dense = x.dim() == 4;
  s.x = desc_of(x);
  s.heads = int32_t(x.size(1));
  s.tokens = int32_t(dense ? x.size(2) : x.size(0));
  if (has(weight)) {
    QK_REQUIRE(weight->device() == x.device() && weight->dim() == 1 && weight->size(0) == kHeadDim,
               weight_name, " must be [64] on the device of q");
    QK_REQUIRE(weight->scalar_type() == at::kFloat || weight->scalar_type() == at::kBFloat16, weight_name,
               " must be float32 or bfloat16, got ", weight->scalar_type());
    const bool as_is = weight->scalar_type() == at::kFloat && weight->stride(0) == 1;
    if (!as_is) c.keep.push_back(weight->to(at::kFloat).contiguous());
    s.weight = (as_is ? *weight : c.keep.back()).data_ptr<float>();
  }
  if (c.args.axes == 0) return;
  QK_REQUIRE(has(positions), positions_name, " are missing");
  const Tensor& p = *positions;
  QK_REQUIRE(p.device() == x.device(), positions_name, " must be on the device of q");
  QK_REQUIRE(p.dim() >= 2 && p.size(-1) == c.args.axes && p.size(-2) == s.tokens &&
                 (p.dim() == 2 || (dense && p.dim() == 3 && p.size(0) == x.size(0))),
             positions_name, " must be [tokens, axes]", dense ? " or [batch, tokens, axes]" : "", ", got ", p.sizes());
  int32_t type = -1;
  if (p.scalar_type() == at::kInt) type = NB_POSITION_I32;
  if (p.scalar_type() == at::kLong) type = NB_POSITION_I64;
  if (p.scalar_type() == at::kFloat) type = NB_POSITION_F32;
  QK_REQUIRE(type >= 0, positions_name, " must be int32, int64 or float32, got ", p.scalar_type());
  QK_REQUIRE(c.args.position_type < 0 || c.args.position_type == type, "positions and k_positions must have one type");
  c.args.position_type = type;
  const bool as_is = p.size(-1) == 1 || p.stride(-1) == 1;
  if (!as_is) c.keep.push_back(p.contiguous());
  const Tensor& at = as_is ? p : c.keep.back();
  s.positions = at.data_ptr();
  s.position_stride_batch = at.dim() == 3 ? at.stride(0) : 0;
  s.position_stride_token = at.stride(-2);
}

QkCall make_call(const Tensor& q, const Tensor& k, const MaybeTensor& q_weight, const MaybeTensor& k_weight,
                 const MaybeTensor& positions, const MaybeTensor& k_positions, const MaybeTensor& freqs, double eps,
                 bool interleaved) {
  QkCall c;
  c.args.batch = int32_t(q.dim() == 4 ? q.size(0) : 1);
  c.args.interleaved = interleaved;
  c.args.eps = float(eps);
  c.args.position_type = -1;
  QK_REQUIRE(eps >= 0.0 && std::isfinite(eps), "eps must be finite and not negative, got ", eps);
  QK_REQUIRE(has(positions) == has(freqs), "positions and freqs come together");
  QK_REQUIRE(!has(k_positions) || has(positions), "k_positions need positions");
  if (has(freqs)) {
    QK_REQUIRE(freqs->device() == q.device() && freqs->scalar_type() == at::kFloat && freqs->dim() == 2 &&
                   freqs->size(1) == kHeadDim / 2 && freqs->size(0) >= 1 && freqs->size(0) <= NB_ROPE_MAX_AXES,
               "freqs must be float32 [axes, 32] with 1 to ", NB_ROPE_MAX_AXES, " axes on the device of q");
    c.args.axes = int32_t(freqs->size(0));
    const bool as_is = freqs->is_contiguous();
    if (!as_is) c.keep.push_back(freqs->contiguous());
    c.args.freqs = (as_is ? *freqs : c.keep.back()).data_ptr<float>();
  }
  set_side(c, c.args.q, q, q_weight, "q_weight", positions, "positions");
  const bool own = has(k_positions);
  set_side(c, c.args.k, k, k_weight, "k_weight", own ? k_positions : positions, own ? "k_positions" : "positions (as k's)");
  if (c.args.position_type < 0) c.args.position_type = 0;
  return c;
}

Two qk_fwd_cuda(const Tensor& q_, const Tensor& k_, const MaybeTensor& q_weight, const MaybeTensor& k_weight,
                const MaybeTensor& positions, const MaybeTensor& k_positions, const MaybeTensor& freqs, double eps,
                bool interleaved) {
  check_qk(q_, k_);
  const c10::cuda::CUDAGuard guard(q_.device());
  const Tensor q = layout_of(q_), k = layout_of(k_);
  QkCall c = make_call(q, k, q_weight, k_weight, positions, k_positions, freqs, eps, interleaved);
  Tensor yq = new_like(q), yk = new_like(k);
  c.args.q.y = desc_of(yq), c.args.k.y = desc_of(yk);
  check_rc(nb_qk_norm_rope_fwd(&c.args, stream_of_current_device()), "nb_qk_norm_rope_fwd");
  return {std::move(yq), std::move(yk)};
}

Four qk_bwd_cuda(const Tensor& dyq_, const Tensor& dyk_, const Tensor& q_, const Tensor& k_, const MaybeTensor& q_weight,
                 const MaybeTensor& k_weight, const MaybeTensor& positions, const MaybeTensor& k_positions,
                 const MaybeTensor& freqs, double eps, bool interleaved) {
  check_qk(q_, k_);
  QK_REQUIRE(dyq_.sizes() == q_.sizes() && dyk_.sizes() == k_.sizes() && dyq_.scalar_type() == at::kBFloat16 &&
                 dyk_.scalar_type() == at::kBFloat16 && dyq_.device() == q_.device() && dyk_.device() == q_.device(),
             "the gradients must be as q and k");
  const c10::cuda::CUDAGuard guard(q_.device());
  const Tensor q = layout_of(q_), k = layout_of(k_), dyq = layout_of(dyq_), dyk = layout_of(dyk_);
  QkCall c = make_call(q, k, q_weight, k_weight, positions, k_positions, freqs, eps, interleaved);
  Tensor dq = new_like(q), dk = new_like(k);
  Tensor dqw = new_tensor({kHeadDim}, at::kFloat, q), dkw = new_tensor({kHeadDim}, at::kFloat, q);
  c.args.q.y = desc_of(dq), c.args.k.y = desc_of(dk);
  c.args.q.dy = desc_of(dyq), c.args.k.dy = desc_of(dyk);
  c.args.q.d_weight = dqw.data_ptr<float>(), c.args.k.d_weight = dkw.data_ptr<float>();
  c.args.workspace_bytes = nb_qk_norm_rope_bwd_workspace_bytes();
  Tensor workspace = new_tensor({int64_t(c.args.workspace_bytes)}, at::kByte, q);
  c.args.workspace = workspace.data_ptr();
  check_rc(nb_qk_norm_rope_bwd(&c.args, stream_of_current_device()), "nb_qk_norm_rope_bwd");
  return {std::move(dq), std::move(dk), std::move(dqw), std::move(dkw)};
}

const auto& qk_fwd_op() {
  static const auto op = find_op<QkFwdSig>("nanobrain_b200::qk_norm_rope_fwd");
  return op;
}
const auto& qk_bwd_op() {
  static const auto op = find_op<QkBwdSig>("nanobrain_b200::qk_norm_rope_bwd");
  return op;
}

struct QkFunction : public torch::autograd::Function<QkFunction> {
  static constexpr bool is_traceable = true;  // compiled autograd may trace through backward
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const MaybeTensor& q_weight,
                               const MaybeTensor& k_weight, const MaybeTensor& positions, const MaybeTensor& k_positions,
                               const MaybeTensor& freqs, double eps, bool interleaved) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [yq, yk] = qk_fwd_op().call(q, k, q_weight, k_weight, positions, k_positions, freqs, eps, interleaved);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, k, or_none(q_weight), or_none(k_weight), or_none(positions), or_none(k_positions),
                            or_none(freqs)});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    return {yq, yk};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    auto [dq, dk, dqw, dkw] = qk_bwd_op().call(
        grads[0].defined() ? grads[0] : at::zeros_like(s[0]), grads[1].defined() ? grads[1] : at::zeros_like(s[1]), s[0],
        s[1], maybe(s[2]), maybe(s[3]), maybe(s[4]), maybe(s[5]), maybe(s[6]), ctx->saved_data["eps"].toDouble(),
        ctx->saved_data["interleaved"].toBool());
    const auto weight_grad = [](const Tensor& g, const Tensor& w) {
      if (!w.defined()) return Tensor();
      return w.scalar_type() == at::kFloat ? g : g.to(w.scalar_type());
    };
    return {dq, dk, weight_grad(dqw, s[2]), weight_grad(dkw, s[3]), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Two qk_fwd_autograd(const Tensor& q, const Tensor& k, const MaybeTensor& q_weight, const MaybeTensor& k_weight,
                    const MaybeTensor& positions, const MaybeTensor& k_positions, const MaybeTensor& freqs, double eps,
                    bool interleaved) {
  nbt::refuse_tangents("qk_norm_rope", q, k, q_weight, k_weight, positions, k_positions, freqs);
  if (at::GradMode::is_enabled()) {
    QK_REQUIRE(!differentiable(positions) && !differentiable(k_positions) && !differentiable(freqs),
               "there is no gradient for positions and freqs");
    if (q.requires_grad() || k.requires_grad() || differentiable(q_weight) || differentiable(k_weight)) {
      auto r = QkFunction::apply(q, k, q_weight, k_weight, positions, k_positions, freqs, eps, interleaved);
      return {r[0], r[1]};
    }
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return qk_fwd_op().call(q, k, q_weight, k_weight, positions, k_positions, freqs, eps, interleaved);
}

// ------------------------------------------------------------------------------------------
// The gated feed-forward block
// ------------------------------------------------------------------------------------------
#define MLP_REQUIRE(cond, ...) TORCH_CHECK(cond, "nanobrain_b200.gated_mlp: ", __VA_ARGS__)

using Three = std::tuple<Tensor, Tensor, Tensor>;
using Seven = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;
using MlpFwdSig = Three(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const MaybeTensor&, const MaybeTensor&,
                        const MaybeTensor&, int64_t, int64_t);
using MlpBwdSig = Seven(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                        const Tensor&, int64_t, int64_t, std::array<bool, 7>);

void check_matrix(const Tensor& t, const char* name, const Tensor& like) {
  MLP_REQUIRE(t.is_cuda(), name, " must be a CUDA tensor (there is no CPU path)");
  MLP_REQUIRE(t.scalar_type() == at::kBFloat16, name, " must be bfloat16, got ", t.scalar_type());
  MLP_REQUIRE(t.device() == like.device(), name, " must be on the device of x");
}

void check_mlp(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Tensor& w_down, int64_t activation) {
  check_matrix(x, "x", x);
  check_matrix(w_gate, "w_gate", x);
  check_matrix(w_up, "w_up", x);
  check_matrix(w_down, "w_down", x);
  MLP_REQUIRE(x.dim() >= 1 && w_gate.dim() == 2, "x must be [..., dim] and w_gate [hidden, dim]");
  const int64_t dim = x.size(-1), hidden = w_gate.size(0);
  MLP_REQUIRE(w_gate.size(1) == dim && w_up.sizes() == w_gate.sizes(), "w_gate and w_up must be [hidden, dim]; dim of x is ",
              dim, ", got ", w_gate.sizes(), " and ", w_up.sizes());
  MLP_REQUIRE(w_down.dim() == 2 && w_down.size(0) == dim && w_down.size(1) == hidden, "w_down must be [dim, hidden] = [", dim,
              ", ", hidden, "], got ", w_down.sizes());
  MLP_REQUIRE(dim > 0 && hidden > 0 && dim % 8 == 0 && hidden % 8 == 0, "dim and hidden must be multiples of 8, got ", dim,
              " and ", hidden);
  MLP_REQUIRE(dim <= 1 << 20 && hidden <= 1 << 20, "dim and hidden must be 2^20 at most, got ", dim, " and ", hidden);
  MLP_REQUIRE(activation == NB_ACT_SILU || activation == NB_ACT_GELU, "no such activation");
}

// Rows of `cols` values at a stride that the kernels can address; otherwise a copy.
Tensor rows_of(const Tensor& t, int64_t cols) {
  const Tensor m = t.dim() == 2 ? t : t.reshape({t.numel() / cols, cols});
  const bool fine = m.stride(1) == 1 && (m.size(0) <= 1 || (m.stride(0) >= cols && m.stride(0) % 8 == 0)) &&
                    (reinterpret_cast<uintptr_t>(m.data_ptr()) & 15u) == 0;
  return fine ? m : m.clone(at::MemoryFormat::Contiguous);
}
nb_matrix matrix(const Tensor& m) {
  if (!m.defined()) return {nullptr, 0};
  return {m.data_ptr(), m.size(0) > 1 ? m.stride(0) : m.size(1)};
}
Tensor bias_of(const MaybeTensor& b, const char* name, int64_t size, const Tensor& x) {
  if (!has(b)) return Tensor();
  check_matrix(*b, name, x);
  MLP_REQUIRE(b->dim() == 1 && b->size(0) == size, name, " must be [", size, "], got ", b->sizes());
  return b->is_contiguous() && (reinterpret_cast<uintptr_t>(b->data_ptr()) & 15u) == 0
             ? *b
             : b->clone(at::MemoryFormat::Contiguous);
}
void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Three mlp_fwd_cuda(const Tensor& x_, const Tensor& w_gate_, const Tensor& w_up_, const Tensor& w_down_,
                   const MaybeTensor& b_gate_, const MaybeTensor& b_up_, const MaybeTensor& b_down_, int64_t activation,
                   int64_t checkpoint) {
  check_mlp(x_, w_gate_, w_up_, w_down_, activation);
  MLP_REQUIRE(checkpoint >= 0 && checkpoint <= 2, "no such checkpoint");
  const int64_t dim = x_.size(-1), hidden = w_gate_.size(0), tokens = x_.numel() / dim;
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor b_gate = bias_of(b_gate_, "b_gate", hidden, x_), b_up = bias_of(b_up_, "b_up", hidden, x_),
               b_down = bias_of(b_down_, "b_down", dim, x_);
  const Tensor x = rows_of(x_, dim), w_gate = rows_of(w_gate_, dim), w_up = rows_of(w_up_, dim),
               w_down = rows_of(w_down_, hidden);
  nb_gated_mlp_fwd_args a{};
  a.shape = {tokens, int32_t(dim), int32_t(hidden), int32_t(activation), int32_t(checkpoint)};
  // Rows of h begin on lines of 128 bytes: with 1368 features side by side the product with w_down takes 160 instead of 132
  // us (131072 tokens, dim 512).
  const int64_t stride = (hidden + 63) / 64 * 64;
  Tensor y = new_tensor(x_.sizes(), at::kBFloat16, x), h = new_tensor({tokens, stride}, at::kBFloat16, x);
  Tensor codes = new_tensor({int64_t(nb_gated_mlp_checkpoint_bytes(&a.shape))}, at::kByte, x);
  const auto result = [&]() -> Three {  // the backward wants h from 16 bits; in 8 bits it makes h again
    if (checkpoint != NB_CHECKPOINT_16BIT) h = new_tensor({0}, at::kBFloat16, x);
    else if (stride != hidden) h = h.narrow(1, 0, hidden);
    return {y, h, codes};
  };
  if (tokens == 0) return result();
  a.x = matrix(x), a.w_gate = matrix(w_gate), a.w_up = matrix(w_up), a.w_down = matrix(w_down);
  a.y = {y.data_ptr(), dim}, a.h = {h.data_ptr(), stride};
  a.b_gate = address(b_gate), a.b_up = address(b_up), a.b_down = address(b_down);
  if (checkpoint != NB_CHECKPOINT_NONE) a.checkpoint = codes.data_ptr();
  volatile int32_t* word = nbt::status_ptr(x.get_device());
  nbt::raise_for_status(word);
  a.status = const_cast<int32_t*>(word);
  check_rc(nb_gated_mlp_fwd(&a, stream_of_current_device()), "nb_gated_mlp_fwd");
  nbt::after_launch(word);
  return result();
}

Seven mlp_bwd_cuda(const Tensor& dy_, const Tensor& x_, const Tensor& w_gate_, const Tensor& w_up_, const Tensor& w_down_,
                   const Tensor& h_, const Tensor& codes, int64_t activation, int64_t checkpoint, std::array<bool, 7> wanted) {
  check_mlp(x_, w_gate_, w_up_, w_down_, activation);
  MLP_REQUIRE(checkpoint == NB_CHECKPOINT_16BIT || checkpoint == NB_CHECKPOINT_8BIT, "there is no checkpoint to go back from");
  check_matrix(dy_, "the gradient", x_);
  MLP_REQUIRE(dy_.sizes() == x_.sizes(), "the gradient must have the shape of x");
  const int64_t dim = x_.size(-1), hidden = w_gate_.size(0), tokens = x_.numel() / dim;
  const c10::cuda::CUDAGuard guard(x_.device());
  const auto out = [&](int i, at::IntArrayRef sizes) {
    if (!wanted[i]) return Tensor();
    return tokens > 0 ? new_tensor(sizes, at::kBFloat16, x_) : at::zeros(sizes, x_.options());
  };
  const auto given = [&](const Tensor& t) { return t.defined() ? t : new_tensor({0}, at::kBFloat16, x_); };
  Tensor dx = out(0, x_.sizes()), dwg = out(1, {hidden, dim}), dwu = out(2, {hidden, dim}), dwd = out(3, {dim, hidden}),
         dbg = out(4, {hidden}), dbu = out(5, {hidden}), dbd = out(6, {dim});
  const auto result = [&]() -> Seven {
    return {given(dx), given(dwg), given(dwu), given(dwd), given(dbg), given(dbu), given(dbd)};
  };
  if (tokens == 0) return result();
  const Tensor x = rows_of(x_, dim), w_gate = rows_of(w_gate_, dim), w_up = rows_of(w_up_, dim),
               w_down = rows_of(w_down_, hidden), dy = rows_of(dy_, dim);
  nb_gated_mlp_bwd_args a{};
  a.shape = {tokens, int32_t(dim), int32_t(hidden), int32_t(activation), int32_t(checkpoint)};
  MLP_REQUIRE(codes.is_cuda() && codes.scalar_type() == at::kByte && codes.is_contiguous() &&
                  size_t(codes.numel()) == nb_gated_mlp_checkpoint_bytes(&a.shape),
              "this is not the checkpoint of such a call");
  Tensor h;
  if (checkpoint == NB_CHECKPOINT_16BIT) {
    MLP_REQUIRE(h_.dim() == 2 && h_.size(0) == tokens && h_.size(1) == hidden, "h must be [tokens, hidden]");
    check_matrix(h_, "h", x_);
    h = rows_of(h_, hidden);
  }
  a.x = matrix(x), a.w_gate = matrix(w_gate), a.w_up = matrix(w_up), a.w_down = matrix(w_down), a.dy = matrix(dy);
  a.h = matrix(h);
  a.checkpoint = codes.data_ptr();
  a.dx = {address(dx), dim}, a.d_w_gate = {address(dwg), dim}, a.d_w_up = {address(dwu), dim},
  a.d_w_down = {address(dwd), hidden};
  a.d_b_gate = address(dbg), a.d_b_up = address(dbu), a.d_b_down = address(dbd);
  a.workspace_bytes = nb_gated_mlp_bwd_workspace_bytes(&a);
  Tensor workspace = new_tensor({int64_t(a.workspace_bytes)}, at::kByte, x);
  a.workspace = workspace.data_ptr();
  volatile int32_t* word = nbt::status_ptr(x.get_device());
  nbt::raise_for_status(word);
  a.status = const_cast<int32_t*>(word);
  check_rc(nb_gated_mlp_bwd(&a, stream_of_current_device()), "nb_gated_mlp_bwd");
  nbt::after_launch(word);
  return result();
}

const auto& mlp_fwd_op() {
  static const auto op = find_op<MlpFwdSig>("nanobrain_b200::gated_mlp_fwd");
  return op;
}
const auto& mlp_bwd_op() {
  static const auto op = find_op<MlpBwdSig>("nanobrain_b200::gated_mlp_bwd");
  return op;
}

struct MlpFunction : public torch::autograd::Function<MlpFunction> {
  static constexpr bool is_traceable = true;  // compiled autograd may trace through backward
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w_gate, const Tensor& w_up,
                               const Tensor& w_down, const MaybeTensor& b_gate, const MaybeTensor& b_up,
                               const MaybeTensor& b_down, int64_t activation, int64_t checkpoint) {
    std::array<bool, 7> wanted = {x.requires_grad(),       w_gate.requires_grad(),  w_up.requires_grad(),
                                  w_down.requires_grad(),  differentiable(b_gate), differentiable(b_up),
                                  differentiable(b_down)};
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [y, h, codes] = mlp_fwd_op().call(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation, checkpoint);
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({h, codes});
    ctx->save_for_backward({x, w_gate, w_up, w_down, h, codes});
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["checkpoint"] = checkpoint;
    int64_t mask = 0;
    for (size_t i = 0; i < 7; ++i) mask |= int64_t(wanted[i]) << i;
    ctx->saved_data["wanted"] = mask;
    return {y, h, codes};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return variable_list(9);
    const variable_list s = ctx->get_saved_variables();
    const int64_t mask = ctx->saved_data["wanted"].toInt();
    std::array<bool, 7> wanted;
    for (size_t i = 0; i < 7; ++i) wanted[i] = (mask >> i) & 1;
    auto [dx, dwg, dwu, dwd, dbg, dbu, dbd] =
        mlp_bwd_op().call(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], ctx->saved_data["activation"].toInt(),
                          ctx->saved_data["checkpoint"].toInt(), wanted);
    variable_list all = {dx, dwg, dwu, dwd, dbg, dbu, dbd, Tensor(), Tensor()};
    for (size_t i = 0; i < 7; ++i)
      if (!wanted[i]) all[i] = Tensor();
    return all;
  }
};

bool wants_grad(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Tensor& w_down, const MaybeTensor& b_gate,
                const MaybeTensor& b_up, const MaybeTensor& b_down) {
  return at::GradMode::is_enabled() &&
         (x.requires_grad() || w_gate.requires_grad() || w_up.requires_grad() || w_down.requires_grad() ||
          differentiable(b_gate) || differentiable(b_up) || differentiable(b_down));
}

Three mlp_fwd_autograd(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Tensor& w_down,
                       const MaybeTensor& b_gate, const MaybeTensor& b_up, const MaybeTensor& b_down, int64_t activation,
                       int64_t checkpoint) {
  nbt::refuse_tangents("gated_mlp", x, w_gate, w_up, w_down, b_gate, b_up, b_down);
  if (!wants_grad(x, w_gate, w_up, w_down, b_gate, b_up, b_down)) {
    at::AutoDispatchBelowADInplaceOrView guard;
    return mlp_fwd_op().call(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation, checkpoint);
  }
  MLP_REQUIRE(checkpoint != NB_CHECKPOINT_NONE, "a call whose gradients are wanted needs a checkpoint");
  auto r = MlpFunction::apply(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation, checkpoint);
  return {r[0], r[1], r[2]};
}

// What Python calls outside of tracing: straight to the dispatcher.
Two qk_norm_rope(const Tensor& q, const Tensor& k, const MaybeTensor& q_weight, const MaybeTensor& k_weight,
                 const MaybeTensor& positions, const MaybeTensor& k_positions, const MaybeTensor& freqs, double eps,
                 bool interleaved) {
  return qk_fwd_op().call(q, k, q_weight, k_weight, positions, k_positions, freqs, eps, interleaved);
}
Tensor gated_mlp(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Tensor& w_down, const MaybeTensor& b_gate,
                 const MaybeTensor& b_up, const MaybeTensor& b_down, int64_t activation, int64_t checkpoint) {
  if (!wants_grad(x, w_gate, w_up, w_down, b_gate, b_up, b_down)) checkpoint = NB_CHECKPOINT_NONE;
  return std::get<0>(mlp_fwd_op().call(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation, checkpoint));
}

}  // namespace

TORCH_LIBRARY_IMPL(nanobrain_b200, CUDA, m) {
  m.impl("qk_norm_rope_fwd", qk_fwd_cuda);
  m.impl("qk_norm_rope_bwd", qk_bwd_cuda);
  m.impl("gated_mlp_fwd", mlp_fwd_cuda);
  m.impl("gated_mlp_bwd", mlp_bwd_cuda);
}

TORCH_LIBRARY_IMPL(nanobrain_b200, Autograd, m) {
  m.impl("qk_norm_rope_fwd", qk_fwd_autograd);
  m.impl("gated_mlp_fwd", mlp_fwd_autograd);
  // There is no second derivative.
  m.impl("qk_norm_rope_bwd", torch::autograd::autogradNotImplementedFallback());
  m.impl("gated_mlp_bwd", torch::autograd::autogradNotImplementedFallback());
}

void nbt::bind_block(pybind11::module_& m) {
  m.def("qk_norm_rope", &qk_norm_rope, py::call_guard<py::gil_scoped_release>());
  m.def("gated_mlp", &gated_mlp, py::call_guard<py::gil_scoped_release>());
}
