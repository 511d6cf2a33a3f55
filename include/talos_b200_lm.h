/*
 * talos_b200 -- C ABI of the operators for training and serving language-model-shaped policies: layer norm, dropout from a
 * counter-based generator, their junction in a transformer block, the clipped policy loss over a vocabulary, and attention
 * over long sequences.  None of them is in the reference crate; they stand beside its RMSNorm (src/nn.rs:145-304), its
 * attention (src/transformer.rs:539-550) and its PPO loss (src/ppo.rs:702-752).
 *
 * The conventions are those of talos_b200.h: fp32 row-major device memory unless a parameter says otherwise, a talos_status
 * from every call, work enqueued on the ctx stream, results not over inputs unless a declaration allows it.
 *
 * CUDA graphs: calls may be captured.  Scratch comes from the ctx: reserve it (talos_ctx_reserve_workspace, or one call of the
 * same sizes) before the capture, and do not let the ctx grow it afterwards while the graph is in use.  Graphs captured from
 * one ctx share its scratch, so their replays must not overlap, like other calls on one ctx.
 */
#ifndef TALOS_B200_LM_H
#define TALOS_B200_LM_H

#include "talos_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- layer norm ------------------------------------------------------------------------------ */
/* y = (x - mean) * inv_std * gamma + beta over rows of `dim` <= 16384 values, inv_std = 1 / sqrt(var + eps), var the population
 * variance.  gamma, beta [dim] may each be NULL (1 and 0).  mean, inv_std [rows] are what the backward pass needs; each may be
 * NULL.  y may be x. */
talos_status talos_layernorm_fwd(talos_ctx* ctx, const float* x, const float* gamma, const float* beta, float eps, int64_t rows,
                                 int64_t dim, float* y, float* mean, float* inv_std);
/* With g = dy * gamma and xh = (x - mean) * inv_std: dx (+)= inv_std * (g - mean(g) - xh * mean(g * xh)), dgamma (+)= sum over
 * rows of dy * xh, dbeta (+)= sum over rows of dy; each of the three may be NULL.  accumulate bit0: dx +=, bit1: dgamma +=,
 * bit2: dbeta +=.  dx may be dy or x.  Sums are added in a fixed order: the same call gives the same bits. */
talos_status talos_layernorm_bwd(talos_ctx* ctx, const float* dy, const float* x, const float* gamma, const float* mean,
                                 const float* inv_std, int64_t rows, int64_t dim, float* dx, float* dgamma, float* dbeta,
                                 int32_t accumulate);

/* ---- dropout ---------------------------------------------------------------------------------- */
/* Element i draws word i % 4 of philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3",
 * SC 2011) with key = seed and counter = (i / 4, offset), both 64 bits, low word first.  It is kept where that word is at least
 * round(p * 2^32), and scaled by 1 / (1 - p); 0 <= p < 1.  Nothing is stored: the backward call with the same p, seed and
 * offset draws the same mask.  Another offset (a step number, a layer number) gives another, independent mask of any length.
 * offset_dev (nullable, device): a 64-bit count added to `offset` when the kernel runs, so that a captured graph whose
 * program advances it draws a new mask at each replay.
 *
 * y = residual + dropped(x), residual nullable.  y may be x or residual. */
talos_status talos_dropout_fwd(talos_ctx* ctx, const float* x, const float* residual, float* y, int64_t n, float p, uint64_t seed,
                               uint64_t offset, const uint64_t* offset_dev);
/* dx (+)= dropped(dy).  The residual's gradient is dy itself.  dx may be dy when it does not accumulate. */
talos_status talos_dropout_bwd(talos_ctx* ctx, const float* dy, float* dx, int64_t n, float p, uint64_t seed, uint64_t offset,
                               const uint64_t* offset_dev, int32_t accumulate);

/* ---- dropout, residual add and layer norm in one pass ------------------------------------------- */
/* h = residual + dropped(x), y = layer norm of h: the junction between the halves of a block.  Elements are counted as in
 * talos_dropout_fwd (i = row * dim + column).  residual, gamma, beta, mean, inv_std nullable; h may be x or residual; h is what
 * the next residual add and the backward pass read. */
talos_status talos_dropout_add_layernorm_fwd(talos_ctx* ctx, const float* x, const float* residual, const float* gamma, const float* beta,
                                             float eps, float p, uint64_t seed, uint64_t offset, const uint64_t* offset_dev, int64_t rows,
                                             int64_t dim, float* h, float* y, float* mean, float* inv_std);
/* dy: gradient of y; dh (nullable): gradient that reaches h past the norm.  dresidual (+)= dh + layer norm's dx, dx (+)=
 * dropped(that); dx, dresidual, dgamma, dbeta nullable.  accumulate bit0: dx +=, bit1: dgamma +=, bit2: dbeta +=, bit3:
 * dresidual +=.  dx and dresidual are different buffers; a result that does not accumulate may be dy or dh. */
talos_status talos_dropout_add_layernorm_bwd(talos_ctx* ctx, const float* dy, const float* dh, const float* h, const float* gamma,
                                             const float* mean, const float* inv_std, float p, uint64_t seed, uint64_t offset,
                                             const uint64_t* offset_dev, int64_t rows, int64_t dim, float* dx, float* dresidual, float* dgamma,
                                             float* dbeta, int32_t accumulate);

/* ---- clipped policy loss with a KL term, over a vocabulary ------------------------------------------ */
/* The per-row loss of a policy that chooses one of `vocab` tokens, and its gradient, from the head's logits [rows, vocab] (row
 * stride ld_logits >= vocab).  With lp = log softmax(logits)[token], r = exp(lp - old_logp), s1 = r * adv,
 * s2 = clip(r, 1 - clip_low, 1 + clip_high) * adv, d = ref_logp - lp, H the entropy of the row:
 *   loss = w * (-min(s1, s2) + c_kl * (exp(d) - d - 1) - c_entropy * H)
 * dlogits (row stride ld_out; nullable: evaluation only) is overwritten with the gradient of sum(loss) / denom; s2 passes its
 * gradient on the closed interval, as talos_ppo_loss_fwd_bwd does.  ref_logp NULL: no KL term (c_kl must be 0).  weights NULL: all 1.
 * logp (nullable) receives lp: with dlogits NULL, what a rollout stores as old_logp or a reference policy answers (old_logp and
 * adv may then be NULL, too: the loss terms that need them are 0).
 * stats[5] = {sum loss, sum w * kl, sum w * H, sum w where the clip held the ratio, sum w}, added to stats when `accumulate` is
 * set.  Sums are added in a fixed order.
 *
 * Padding: a row with a negative token or with weight 0 is not read; its logp and its gradient are 0, its terms left out.
 * Masked vocabulary: logits of -inf have probability 0, add nothing to H and have gradient 0.  A row whose logits are all -inf has
 * logp -inf and is left out otherwise, like padding.  (A token that is itself masked, in a row that is not, has logp -inf, and its loss
 * is what the formula gives.)  A token >= vocab: the row counts as padding, and the next call that waits for the stream returns
 * TALOS_ERR_ARG.
 * dlogits may be logits when the strides are equal. */
talos_status talos_policy_loss_fwd_bwd(talos_ctx* ctx, const float* logits, int64_t ld_logits, const int32_t* tokens, const float* old_logp,
                                       const float* ref_logp, const float* adv, const float* weights, int64_t rows, int64_t vocab,
                                       float clip_low, float clip_high, float c_kl, float c_entropy, float denom, float* logp, float* dlogits,
                                       int64_t ld_out, float* stats, int32_t accumulate);

/* ---- attention over long sequences ------------------------------------------------------------------- */
/* Layout of q, k, v, out and their gradients: [batch, heads, rows, width] or [batch, rows, heads, width] (what a Linear layer leaves). */
enum { TALOS_ATTN_BHSD = 0, TALOS_ATTN_BSHD = 1 };
/* Causal masks (0: none).  They differ where a sequence has fewer than sk keys. */
enum { TALOS_ATTN_CAUSAL = 1, TALOS_ATTN_CAUSAL_NEWEST = 3 };
/* out_i = sum_j p_ij v_j, p_i the softmax of scale * q_i . k_j over the keys that query i sees; the scores stay on chip, and one number
 * a row is saved, lse = log sum_j exp(scale * q_i . k_j).  q [batch, heads, sq, d], k [batch, kv_heads, sk, d], v [batch, kv_heads, sk, dv],
 * out [batch, heads, sq, dv]; lse [batch, heads, sq] (nullable) in every layout.  d, dv <= 128; kv_heads divides heads, query head h reads
 * key head h / (heads / kv_heads).
 * key_len (nullable, device, [batch]): sequence b has min(max(key_len[b], 0), sk) keys, the rows behind them are not read (padding, or a
 * cache that is not full).  A query that sees no key has out 0 and lse -inf.
 * causal: with TALOS_ATTN_CAUSAL query i sees the keys j <= i + sk - sq: the queries are the last sq of sk positions, whatever key_len says (training on
 * padded batches, sq = sk; a cache of one length for all sequences).  With TALOS_ATTN_CAUSAL_NEWEST it sees j <= i + n - sq, n the sequence's own keys:
 * the queries are the newest sq of them (several new tokens of each sequence over caches filled to different lengths; of a sequence with fewer
 * than sq keys the first queries see none).  A single query sees all its sequence's keys in either.
 * Rows of k and v before key_len are read in tiles and must be finite, in the backward pass q and dout, too.
 * A few queries over many keys (a decode step) are split over the keys and joined.  Larger products run on the tensor cores at fp32's
 * accuracy in modes FP32 and TF32X3 alike (three bf16 terms a value, six products, sums of a block added in fp32: closer to the exact result
 * than the CUDA-core kernel that serves up to 64 queries and keys); mode TF32 takes two terms and three products (2^-16 relative).
 * Scratch: the split tiles of as many sequences as fit 1 GiB, one at least (128 rows of a head and tensor: 48 KB, 96 KB above width 64). */
talos_status talos_attention_lse_fwd(talos_ctx* ctx, const float* q, const float* k, const float* v, const int32_t* key_len, float* out,
                                     float* lse, int64_t batch, int64_t heads, int64_t kv_heads, int64_t sq, int64_t sk, int64_t d, int64_t dv,
                                     float scale, int32_t causal, int32_t layout, int32_t mode);
/* Gradients from out, lse and the inputs: the probabilities are computed again.  dq, dk, dv_out are overwritten; dk and dv_out hold the
 * sums over the query heads that share a key head, 0 in the rows behind key_len.  The same call gives the same bits. */
talos_status talos_attention_lse_bwd(talos_ctx* ctx, const float* q, const float* k, const float* v, const int32_t* key_len, const float* out,
                                     const float* lse, const float* dout, float* dq, float* dk, float* dv_out, int64_t batch, int64_t heads,
                                     int64_t kv_heads, int64_t sq, int64_t sk, int64_t d, int64_t dv, float scale, int32_t causal,
                                     int32_t layout, int32_t mode);

#ifdef __cplusplus
}
#endif
#endif /* TALOS_B200_LM_H */
