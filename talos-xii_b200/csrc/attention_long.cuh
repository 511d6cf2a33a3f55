// What the kernels of attention over long sequences share: the problem's shape and where its rows lie.
#pragma once
#include "common.cuh"

#include "../../include/talos_b200_lm.h"

struct AttnShape {
  const int* key_len;
  int batch, heads, kv_heads, group, sq, sk, d, dv, causal;
  float scale;
  // elements between rows of one head, heads, sequences: of q / dq, of k / dk, of v / dv, of out / dout
  long long q_row, q_head, q_batch, k_row, k_head, k_batch, v_row, v_head, v_batch, o_row, o_head, o_batch;
};

#ifdef __CUDACC__
__device__ __forceinline__ int attn_keys(const AttnShape& s, int b) { return s.key_len ? min(max(s.key_len[b], 0), s.sk) : s.sk; }
// Causal: query i sees the keys up to i + attn_shift.
__device__ __forceinline__ int attn_shift(const AttnShape& s, int keys) { return (s.causal == TALOS_ATTN_CAUSAL_NEWEST ? keys : s.sk) - s.sq; }
// Keys that query i sees: the first attn_limit of its sequence's.
__device__ __forceinline__ int attn_limit(const AttnShape& s, int keys, int i) { return s.causal ? min(keys, max(0, i + attn_shift(s, keys) + 1)) : keys; }
#endif

// The tensor-core kernels (attention_long_tc.cu); false: not a shape of theirs, nothing launched.
bool talos_attn_tc_fwd(talos_ctx* ctx, const AttnShape& s, const float* q, const float* k, const float* v, float* out, float* lse, int mode);
bool talos_attn_tc_bwd(talos_ctx* ctx, const AttnShape& s, const float* q, const float* k, const float* v, const float* out, const float* lse, const float* dout, float* dq,
                       float* dk, float* dv, int mode);
