// C++ host layer of the operators in include/talos_b200_lm.h, in the manner of talos.hpp: modules and tape nodes over the C ABI.
// None of them is in the reference crate; LayerNorm stands beside its RMSNorm (src/nn.rs:145-304), policy_loss beside the loss of
// PPO::update (src/ppo.rs:702-755), long_attention beside the attention of src/transformer.rs:539-550.
#pragma once
#include "../../include/talos_b200_lm.h"
#include "talos.hpp"

namespace talos {

struct LayerNorm : Module {
  Tensor weight, bias; double eps; size_t dim;
  LayerNorm(size_t d, double e) : weight(Tensor::new_(std::vector<double>(d, 1.0), {d})), bias(Tensor::zeros({d})), eps(e), dim(d) {}
  Tensor forward(const Tensor& x) const override {
    TALOS_ASSERT(!x.shape.empty() && x.shape.back() == dim, "LayerNorm dim mismatch");
    const size_t rows = x.len() / dim, dm = dim;
    Buf mean = make_buf(rows, false), inv = make_buf(rows, false);
    Tensor out = Tensor::result(x.shape, {x, weight, bias}, [rows, dm, mean, inv](const Tensor& o, const std::vector<Tensor>& p) {
      check(talos_layernorm_bwd(ctx(), o.g(), p[0].d(), p[1].d(), mean->dev, inv->dev, (int64_t)rows, (int64_t)dm, p[0].g(), p[1].g(), p[2].g(), 7));
    });
    check(talos_layernorm_fwd(ctx(), x.d(), weight.d(), bias.d(), (float)eps, (int64_t)rows, (int64_t)dim, out.d(), mean->dev, inv->dev));
    return out;
  }
  std::vector<Tensor> parameters() const override { return {weight, bias}; }
};

// Dropout with the mask of (seed, offset); the tape keeps the two numbers, not the mask.
inline Tensor dropout(const Tensor& x, double p, uint64_t seed, uint64_t offset) {
  Tensor out = Tensor::result(x.shape, {x}, [p, seed, offset](const Tensor& o, const std::vector<Tensor>& q) {
    check(talos_dropout_bwd(ctx(), o.g(), q[0].g(), (int64_t)o.len(), (float)p, seed, offset, nullptr, 1));
  });
  check(talos_dropout_fwd(ctx(), x.d(), nullptr, out.d(), (int64_t)x.len(), (float)p, seed, offset, nullptr));
  return out;
}

// h = residual + dropout(x), y = norm(h), returned as {h, y}, each to be used by any number of nodes.  Backward is one pass, made when both
// gradients are complete: y's node hands nothing on by itself, h's node, which every path to y leads through, reads both.
inline std::pair<Tensor, Tensor> dropout_add_layernorm(const Tensor& x, const Tensor& residual, const LayerNorm& norm, double p, uint64_t seed, uint64_t offset) {
  TALOS_ASSERT(x.shape == residual.shape && !x.shape.empty() && x.shape.back() == norm.dim, "dropout_add_layernorm shape mismatch");
  const size_t rows = x.len() / norm.dim, dm = norm.dim;
  Buf mean = make_buf(rows, false), inv = make_buf(rows, false), dy = make_buf(x.len());
  Tensor h = Tensor::result(x.shape, {x, residual, norm.weight, norm.bias}, [=](const Tensor& o, const std::vector<Tensor>& q) {
    const bool same = q[0].grad == q[1].grad;                // x + dropout(x): two results into one buffer, one after the other
    Buf dx = same ? make_buf(o.len()) : nullptr;
    check(talos_dropout_add_layernorm_bwd(ctx(), dy->dev, o.g(), o.d(), q[2].d(), mean->dev, inv->dev, (float)p, seed, offset, nullptr, (int64_t)rows, (int64_t)dm,
                                          same ? dx->dev : q[0].g(), q[1].g(), q[2].g(), q[3].g(), 15));
    if (same) check(talos_eltwise_binary(ctx(), TALOS_EW_ADD, q[0].g(), dx->dev, q[0].g(), (int64_t)o.len()));
    check(talos_memset_zero(ctx(), dy->dev, sizeof(float) * dy->n));   // a later backward may reach h alone
  });
  Tensor y = Tensor::result(x.shape, {h}, [dy](const Tensor& o, const std::vector<Tensor>&) {
    check(talos_eltwise_binary(ctx(), TALOS_EW_ADD, dy->dev, o.g(), dy->dev, (int64_t)o.len()));
  });
  check(talos_dropout_add_layernorm_fwd(ctx(), x.d(), residual.d(), norm.weight.d(), norm.bias.d(), (float)norm.eps, (float)p, seed, offset, nullptr, (int64_t)rows,
                                        (int64_t)dm, h.d(), y.d(), mean->dev, inv->dev));
  return {h, y};
}

// Attention over q [B, Sq, H, d], k [B, Sk, Hk, d], v [B, Sk, Hk, dv] (what Linear layers leave); causal: 0, TALOS_ATTN_CAUSAL or TALOS_ATTN_CAUSAL_NEWEST;
// key_len: keys of each sequence (nullptr: all).
inline Tensor long_attention(const Tensor& q, const Tensor& k, const Tensor& v, int32_t causal, const std::vector<int32_t>* key_len = nullptr) {
  TALOS_ASSERT(q.shape.size() == 4 && k.shape.size() == 4 && v.shape.size() == 4 && q.shape[0] == k.shape[0] && q.shape[3] == k.shape[3] && k.shape[0] == v.shape[0] &&
                   k.shape[1] == v.shape[1] && k.shape[2] == v.shape[2], "long_attention shape mismatch");
  const int64_t B = q.shape[0], H = q.shape[2], Hk = k.shape[2], Sq = q.shape[1], Sk = k.shape[1], d = q.shape[3], dv = v.shape[3];
  const float scale = 1.f / std::sqrt((float)d);
  const int md = mode();
  Buf lens;
  if (key_len) {
    TALOS_ASSERT(key_len->size() == (size_t)B, "one key count a sequence");
    lens = make_buf(B, false);
    check(talos_copy_from_host(ctx(), lens->dev, key_len->data(), sizeof(int32_t) * B));
  }
  Buf lse = make_buf(B * H * Sq, false);
  Tensor out = Tensor::result({q.shape[0], q.shape[1], q.shape[2], v.shape[3]}, {q, k, v}, [=](const Tensor& o, const std::vector<Tensor>& p) {
    Buf g[3];
    for (int i = 0; i < 3; ++i) g[i] = make_buf(p[i].len(), false);
    check(talos_attention_lse_bwd(ctx(), p[0].d(), p[1].d(), p[2].d(), lens ? (const int32_t*)lens->dev : nullptr, o.d(), lse->dev, o.g(), g[0]->dev, g[1]->dev, g[2]->dev, B, H,
                                  Hk, Sq, Sk, d, dv, scale, causal, TALOS_ATTN_BSHD, md));
    for (int i = 0; i < 3; ++i) check(talos_eltwise_binary(ctx(), TALOS_EW_ADD, p[i].g(), g[i]->dev, p[i].g(), (int64_t)p[i].len()));
  });
  check(talos_attention_lse_fwd(ctx(), q.d(), k.d(), v.d(), lens ? (const int32_t*)lens->dev : nullptr, out.d(), lse->dev, B, H, Hk, Sq, Sk, d, dv, scale, causal, TALOS_ATTN_BSHD, md));
  return out;
}

struct PolicyLossConfig { double clip_low = 0.2, clip_high = 0.2, c_kl = 0.0, c_entropy = 0.0; };

// log pi(token) of each row of logits [rows, vocab] (negative tokens: padding, 0), graph-free: what a rollout stores and a reference policy answers.
inline Tensor token_log_probs(const Tensor& logits, const std::vector<int32_t>& tokens) {
  const size_t vocab = logits.shape.back(), rows = logits.len() / vocab;
  TALOS_ASSERT(tokens.size() == rows, "one token a row");
  Tensor out = Tensor::zeros({rows});
  Buf tok = make_buf(rows, false);
  check(talos_copy_from_host(ctx(), tok->dev, tokens.data(), sizeof(int32_t) * rows));
  check(talos_policy_loss_fwd_bwd(ctx(), logits.d(), (int64_t)vocab, (const int32_t*)tok->dev, nullptr, nullptr, nullptr, nullptr, (int64_t)rows, (int64_t)vocab, 0.2f, 0.2f, 0.f,
                                  0.f, 1.f, out.d(), nullptr, (int64_t)vocab, nullptr, 0));
  return out;
}

// The clipped policy loss with a KL term as a tape node on the logits: sum of the rows' losses / denom.  ref_logp and weights may be nullptr.
inline Tensor policy_loss(const Tensor& logits, const std::vector<int32_t>& tokens, const Tensor& old_logp, const Tensor* ref_logp, const Tensor& adv, const Tensor* weights,
                          const PolicyLossConfig& c, double denom) {
  const size_t vocab = logits.shape.back(), rows = logits.len() / vocab;
  TALOS_ASSERT(tokens.size() == rows && old_logp.len() == rows && adv.len() == rows && (!ref_logp || ref_logp->len() == rows) && (!weights || weights->len() == rows),
               "policy loss batch size mismatch");
  Buf tok = make_buf(rows, false), dz = make_buf(logits.len(), false), stats = make_buf(5, false);
  check(talos_copy_from_host(ctx(), tok->dev, tokens.data(), sizeof(int32_t) * rows));
  Tensor loss = Tensor::result({1}, {logits}, [dz](const Tensor& o, const std::vector<Tensor>& p) {
    const int64_t n = (int64_t)p[0].len();                   // dz holds the gradient for an upstream gradient of 1
    Buf scaled = make_buf((size_t)n, false);
    check(talos_fill_from_scalar(ctx(), o.g(), 1.f, scaled->dev, n, 0));
    check(talos_vector_fma(ctx(), p[0].g(), scaled->dev, dz->dev, n));
  });
  check(talos_policy_loss_fwd_bwd(ctx(), logits.d(), (int64_t)vocab, (const int32_t*)tok->dev, old_logp.d(), ref_logp ? ref_logp->d() : nullptr, adv.d(),
                                  weights ? weights->d() : nullptr, (int64_t)rows, (int64_t)vocab, (float)c.clip_low, (float)c.clip_high, (float)c.c_kl, (float)c.c_entropy,
                                  (float)denom, nullptr, dz->dev, (int64_t)vocab, stats->dev, 0));
  check(talos_fill_from_scalar(ctx(), stats->dev, (float)(1.0 / denom), loss.d(), 1, 0));
  return loss;
}

// Pre-norm block of a language-model-shaped policy: layer norm -> QKV -> attention over the whole sequence -> W_o -> dropout + residual + layer
// norm in one pass -> W_ff1 -> SiLU -> W_ff2 -> dropout + residual.  kv_heads may be fewer than heads.  `step` numbers the training step: every
// step and each of the block's two dropouts draw masks of their own.
struct LmBlock {
  size_t dim, heads, kv_heads; LayerNorm norm_1, norm_2; Linear w_q, w_k, w_v, w_o, w_ff1, w_ff2; double p; uint64_t seed;
  LmBlock(size_t d, size_t h, size_t hk, size_t ff, double eps, double dropout_p, uint64_t s)
      : dim(d), heads(h), kv_heads(hk), norm_1(d, eps), norm_2(d, eps), w_q(d, d, false, s), w_k(d, d / h * hk, false, s + 1), w_v(d, d / h * hk, false, s + 2), w_o(d, d, true, s + 3),
        w_ff1(d, ff, true, s + 4), w_ff2(ff, d, true, s + 5), p(dropout_p), seed(s) {}
  Tensor forward(const Tensor& x, uint64_t step, const std::vector<int32_t>* key_len = nullptr) const {
    TALOS_ASSERT(x.shape.size() == 3 && x.shape[2] == dim, "LmBlock expects [Batch, Seq, Dim]");
    const size_t B = x.shape[0], S = x.shape[1], dh = dim / heads;
    Tensor a = norm_1.forward(x);
    Tensor q = w_q.forward(a).reshape({B, S, heads, dh}), k = w_k.forward(a).reshape({B, S, kv_heads, dh}), v = w_v.forward(a).reshape({B, S, kv_heads, dh});
    Tensor att = long_attention(q, k, v, TALOS_ATTN_CAUSAL, key_len).reshape({B, S, dim});
    auto [h, y] = dropout_add_layernorm(w_o.forward(att), x, norm_2, p, seed, 2 * step);
    return h + dropout(w_ff2.forward(w_ff1.forward_act(y, TALOS_ACT_SILU)), p, seed, 2 * step + 1);
  }
  std::vector<Tensor> parameters() const {
    std::vector<Tensor> r = norm_1.parameters();
    for (const Linear* l : {&w_q, &w_k, &w_v, &w_o}) for (auto& t : l->parameters()) r.push_back(t);
    for (auto& t : norm_2.parameters()) r.push_back(t);
    for (const Linear* l : {&w_ff1, &w_ff2}) for (auto& t : l->parameters()) r.push_back(t);
    return r;
  }
};

}  // namespace talos
