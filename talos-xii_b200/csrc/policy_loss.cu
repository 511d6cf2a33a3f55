// Clipped policy loss with a KL term over a vocabulary, and its gradient, from a head's logits.
//
// Mathematics, per row z with token a: lse = log sum exp z, lp = z_a - lse, H = -sum p log p.  One pass leaves, per warp, its
// maximum m, s = sum exp(z - m) and t = sum exp(z - m) (z - m); triples combine by rescaling to the larger maximum, and at the end
// lse = m + log s, H = log s - t / s.  The loss is a function of lp and H, so its gradient is
//   dz_j = g (1[j = a] - p_j) + e p_j (log p_j + H),    g = dL/dlp, e = c_entropy w / denom.
// Bound: HBM, 8 bytes a logit (read once, its gradient written once).  A row therefore stays in the registers of the threads that own
// it from the read to the write: 4 to 32 lanes for the few actions of a small policy, a CTA of 256 for up to 8 192 tokens, a
// cluster of two to eight CTAs beyond, whose warps push their triples into every CTA's shared memory, so that one cluster barrier
// a row is all they wait for.
#include <cooperative_groups.h>
#include <math.h>

#include "common.cuh"

#include "../../include/talos_b200_lm.h"

namespace {

namespace cg = cooperative_groups;

struct LossArgs {
  const float* logits; long long ld; const int* tokens; const float *old_logp, *ref_logp, *adv, *weights;
  long long rows; int vocab;
  float lo, hi, c_kl, c_entropy, inv_denom;
  float* logp; float* dlogits; long long ld_out; float* partial; int32_t* status;
};

struct Triple { float m, s, t; };
// (m = -inf: nothing but -inf so far.  A NaN survives in s.)
__device__ __forceinline__ float rescale(float m, float to) { return m == -INFINITY ? 0.f : expf(m - to); }
template <int G> __device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int G> __device__ __forceinline__ float group_add(float v) {
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What a row's loss says about it: dL/dlp (already divided by denom), the weight of its entropy gradient, its terms of the five sums.
struct RowLoss { float g, e, loss, kl, entropy, clipped; };
__device__ __forceinline__ RowLoss row_loss(const LossArgs& p, long long r, float w, float lp, float entropy) {
  RowLoss o{0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (p.adv) {
    const float adv = p.adv[r], ratio = expf(lp - p.old_logp[r]);
    const float s1 = ratio * adv, s2 = fminf(fmaxf(ratio, p.lo), p.hi) * adv;
    const bool first = s1 < s2, inside = ratio >= p.lo && ratio <= p.hi;
    o.loss = -(first ? s1 : s2);
    o.g = first || inside ? -s1 : 0.f;
    o.clipped = !first && !inside && s2 < s1 ? w : 0.f;
    if (s1 != s1) { o.loss = s1; o.g = s1; }                              // NaN stays NaN
  }
  if (p.ref_logp) {
    const float d = p.ref_logp[r] - lp, em1 = expm1f(d);
    o.kl = em1 - d;
    if (p.c_kl != 0.f) { o.loss += p.c_kl * o.kl; o.g -= p.c_kl * em1; }
  }
  if (p.c_entropy != 0.f) o.loss -= p.c_entropy * entropy;
  const float scale = w * p.inv_denom;
  o.g *= scale; o.e = p.c_entropy * scale;
  o.loss *= w; o.kl *= w; o.entropy = w * entropy;
  return o;
}

// One row's gradient values from its logits (ENT: z itself, otherwise exp(z - m) with c = exp(m - lse)).
template <bool ENT> __device__ __forceinline__ float dlogit(float v, float c, float lse, float H, const RowLoss& k, bool token) {
  float out;
  if constexpr (ENT) {
    const float lp = v - lse, q = expf(lp);
    out = q == 0.f ? 0.f : q * (k.e * (lp + H) - k.g);
  } else out = -k.g * (v * c);
  return token ? out + k.g : out;
}

template <int W> __device__ __forceinline__ void load_units(const float* p, float* a) {
  if constexpr (W == 4) { const float4 q = __ldcs((const float4*)p); a[0] = q.x; a[1] = q.y; a[2] = q.z; a[3] = q.w; }
  else a[0] = __ldcs(p);
}
template <int W> __device__ __forceinline__ void store_units(float* p, const float* a) {
  if constexpr (W == 4) __stcs((float4*)p, make_float4(a[0], a[1], a[2], a[3]));
  else __stcs(p, a[0]);
}

// Whether a row counts; reports a token outside the vocabulary.
__device__ __forceinline__ bool counts(const LossArgs& p, long long r, int& token, float& w, bool reports) {
  token = p.tokens[r]; w = p.weights ? p.weights[r] : 1.f;
  if (token >= p.vocab) { if (reports) atomicExch(p.status, TALOS_DEV_BAD_INDEX); return false; }
  return token >= 0 && w != 0.f;
}

template <int G> constexpr int block_of = G <= 32 ? 256 : G;

// G threads (of CL CTAs) own a row, NV groups of W values each.
template <int W, int G, int NV, int CL, bool ENT, int PER_SM>
__global__ void __launch_bounds__(block_of<G>, PER_SM) policy_loss_kernel(LossArgs p) {
  talos_pdl(p.logits, p.tokens, p.old_logp, p.ref_logp, p.adv, p.weights, p.logp, p.dlogits, p.partial, p.status);
  constexpr int RPB = G <= 32 ? 256 / G : 1, WARPS = G / 32 > 0 ? G / 32 : 1;
  __shared__ Triple parts[2][CL * WARPS];
  __shared__ float sums[8][5];
  const int l = G <= 32 ? threadIdx.x % G : threadIdx.x, sub = G <= 32 ? threadIdx.x / G : 0, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = CL > 1 ? (int)(blockIdx.x % CL) : 0;
  const long long first = (long long)(blockIdx.x / CL) * RPB, step = (long long)(gridDim.x / CL) * RPB;
  const int units = p.vocab / W, u0 = part * (G * NV) + l;
  int phase = 0;
  float acc[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
  if constexpr (CL > 1) cg::this_cluster().sync();                       // every CTA of the cluster runs before one writes into it
  for (long long r0 = first; r0 < p.rows; r0 += step) {
    const long long r = r0 + sub;
    const bool in = r < p.rows;
    int token = -1; float w = 0.f;
    const bool live = in && counts(p, r, token, w, l == 0 && part == 0);
    if (G > 32 && !live) {                                               // padding: nothing is read (the same for the row's threads)
      if (p.dlogits) {
        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int v = 0; v < NV; ++v) if (u0 + v * G < units) store_units<W>(p.dlogits + r * p.ld_out + (long long)(u0 + v * G) * W, zero);
      }
      if (p.logp && l == 0 && part == 0) p.logp[r] = 0.f;
      continue;
    }
    float z[NV][W];
    const float* row = p.logits + r * p.ld;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (live && u0 + v * G < units) load_units<W>(row + (long long)(u0 + v * G) * W, z[v]);
      else {
#pragma unroll
        for (int i = 0; i < W; ++i) z[v][i] = -INFINITY;
      }
    }
    const float zt = live ? row[token] : 0.f;                            // before any thread of the row writes over it
    float m = -INFINITY;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < W; ++i) m = fmaxf(m, z[v][i]);
    m = group_max<G>(m);
    const float mm = m == -INFINITY ? 0.f : m;
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float x = z[v][i] - mm, e = expf(x);
        s += e; t += e * fmaxf(x, -1e30f);                               // (0 for -inf)
        if constexpr (!ENT) z[v][i] = e;
      }
    s = group_add<G>(s); t = group_add<G>(t);
    float M = m, S = s, T = t;
    if constexpr (G > 32) {
      if (lane < CL) {
        Triple* to = &parts[phase][part * WARPS + warp];
        if constexpr (CL > 1) to = cg::this_cluster().map_shared_rank(to, lane);
        *to = Triple{m, s, t};
      }
      if constexpr (CL > 1) cg::this_cluster().sync(); else __syncthreads();
      // every warp combines the CL x WARPS triples, at most two a lane
      constexpr int N = CL * WARPS, PER = (N + 31) / 32;
      Triple q[PER];
      M = -INFINITY;
#pragma unroll
      for (int i = 0; i < PER; ++i) { const int j = lane + 32 * i; q[i] = j < N ? parts[phase][j] : Triple{-INFINITY, 0.f, 0.f}; M = fmaxf(M, q[i].m); }
      M = group_max<32>(M);
      S = T = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        // (a warp with nothing but -inf has s = 0; one with a NaN and -inf has m = -inf and s = NaN, which must stay)
        const float f = rescale(q[i].m, M), d = q[i].m == -INFINITY ? 0.f : q[i].m - M;
        S += q[i].m == -INFINITY ? q[i].s : q[i].s * f;
        T += q[i].m == -INFINITY ? q[i].t : (q[i].t + q[i].s * d) * f;
      }
      S = group_add<32>(S); T = group_add<32>(T);
      phase ^= 1;
    }
    const bool empty = S == 0.f;                                         // every logit -inf
    const float MM = M == -INFINITY ? 0.f : M, ls = logf(S), lse = empty ? -INFINITY : MM + ls, H = empty ? 0.f : ls - T / S;
    const float lp = empty ? -INFINITY : zt - lse;
    RowLoss k{0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (live && !empty) k = row_loss(p, r, w, lp, H);
    if (live && l == 0 && part == 0) {
      if (p.logp) p.logp[r] = lp;
      if (!empty) { acc[0] += k.loss; acc[1] += k.kl; acc[2] += k.entropy; acc[3] += k.clipped; acc[4] += w; }
    } else if (in && !live && l == 0 && p.logp) p.logp[r] = 0.f;
    if (p.dlogits && in) {
      const float c = live && !empty ? expf(mm - lse) : 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int u = u0 + v * G;
        if (u >= units) continue;
        float o[W];
#pragma unroll
        for (int i = 0; i < W; ++i) o[i] = live && !empty ? dlogit<ENT>(z[v][i], c, lse, H, k, u * W + i == token) : 0.f;
        store_units<W>(p.dlogits + r * p.ld_out + (long long)u * W, o);
      }
    }
  }
  if constexpr (CL > 1) cg::this_cluster().sync();                       // no CTA leaves while another may still write into it
  if (!p.partial || part != 0) return;
  // this CTA's rows: the leaders' sums, warp by warp
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    const float a = G <= 32 ? group_add<32>(acc[i]) : acc[i];
    if (G <= 32) { if (lane == 0) sums[warp][i] = a; }
    else if (threadIdx.x == 0) p.partial[(blockIdx.x / CL) * 5 + i] = a;
  }
  if constexpr (G <= 32) {
    __syncthreads();
    if (threadIdx.x < 5) {
      float a = 0.f;
      for (int i = 0; i < 8; ++i) a += sums[i][threadIdx.x];
      p.partial[blockIdx.x * 5 + threadIdx.x] = a;
    }
  }
}

// Rows that no cluster's registers hold: a CTA a row, the row read twice (the second time from L2).
template <bool ENT>
__global__ void __launch_bounds__(1024) policy_loss_long_kernel(LossArgs p) {
  talos_pdl(p.logits, p.tokens, p.old_logp, p.ref_logp, p.adv, p.weights, p.logp, p.dlogits, p.partial, p.status);
  __shared__ Triple parts[2][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int phase = 0;
  float acc[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    int token; float w;
    float* out = p.dlogits + r * p.ld_out;
    if (!counts(p, r, token, w, threadIdx.x == 0)) {
      if (p.dlogits) for (int j = threadIdx.x; j < p.vocab; j += 1024) out[j] = 0.f;
      if (p.logp && threadIdx.x == 0) p.logp[r] = 0.f;
      continue;
    }
    const float* row = p.logits + r * p.ld;
    const float zt = row[token];
    float m = -INFINITY, s = 0.f, t = 0.f;
    for (int j0 = threadIdx.x; j0 < p.vocab; j0 += 8 * 1024) {
      float z[8];
      float top = m;
#pragma unroll
      for (int i = 0; i < 8; ++i) { z[i] = j0 + i * 1024 < p.vocab ? row[j0 + i * 1024] : -INFINITY; top = fmaxf(top, z[i]); }
      const float mm = top == -INFINITY ? 0.f : top;
      if (m != -INFINITY) { const float f = expf(m - mm); t = (t + s * (m - mm)) * f; s *= f; }
#pragma unroll
      for (int i = 0; i < 8; ++i) { const float x = z[i] - mm, e = expf(x); s += e; t += e * fmaxf(x, -1e30f); }
      m = top;
    }
    auto join = [&](float M) {                                           // s, t relative to M (>= m)
      if (m != -INFINITY) { const float f = expf(m - M); t = (t + s * (m - M)) * f; s *= f; }
      m = M;
    };
    join(group_max<32>(m));
    s = group_add<32>(s); t = group_add<32>(t);
    if (lane == 0) parts[phase][warp] = Triple{m, s, t};
    __syncthreads();
    const Triple q = parts[phase][lane];
    m = q.m; s = q.s; t = q.t;
    join(group_max<32>(m));
    s = group_add<32>(s); t = group_add<32>(t);
    phase ^= 1;
    const bool empty = s == 0.f;
    const float mm = m == -INFINITY ? 0.f : m, ls = logf(s), lse = empty ? -INFINITY : mm + ls, H = empty ? 0.f : ls - t / s, lp = empty ? -INFINITY : zt - lse;
    RowLoss k{0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (!empty) k = row_loss(p, r, w, lp, H);
    if (threadIdx.x == 0) {
      if (p.logp) p.logp[r] = lp;
      if (!empty) { acc[0] += k.loss; acc[1] += k.kl; acc[2] += k.entropy; acc[3] += k.clipped; acc[4] += w; }
    }
    if (!p.dlogits) continue;
    const float c = empty ? 0.f : expf(mm - lse);
    for (int j = threadIdx.x; j < p.vocab; j += 1024) {
      const float z = row[j];
      out[j] = empty ? 0.f : dlogit<ENT>(ENT ? z : expf(z - mm), c, lse, H, k, j == token);
    }
  }
  if (p.partial && threadIdx.x == 0)
#pragma unroll
    for (int i = 0; i < 5; ++i) p.partial[blockIdx.x * 5 + i] = acc[i];
}

// stats (+)= the CTAs' sums, in 64 bits, in a fixed order.
__global__ void __launch_bounds__(256) policy_stats_kernel(const float* partial, int n, float* stats, int accumulate) {
  talos_pdl(partial, stats);
  __shared__ double sh[8][5];
  double a[5] = {0., 0., 0., 0., 0.};
  for (int i = threadIdx.x; i < n; i += 256)
#pragma unroll
    for (int j = 0; j < 5; ++j) a[j] += (double)partial[i * 5 + j];
#pragma unroll
  for (int j = 0; j < 5; ++j) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a[j] += __shfl_xor_sync(0xffffffffu, a[j], o);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5][j] = a[j];
  }
  __syncthreads();
  if (threadIdx.x < 5) {
    double t = accumulate ? (double)stats[threadIdx.x] : 0.;
    for (int i = 0; i < 8; ++i) t += sh[i][threadIdx.x];
    stats[threadIdx.x] = (float)t;
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Returns the number of partial sums that the launch leaves at p.partial.
template <bool ENT> int loss_launch(talos_ctx* ctx, LossArgs& p, bool want_stats) {
  int parts = 0;
  auto go = [&](auto kern, int rpb, int block, int per_sm, int cl) {
    const int64_t cap = std::max<int64_t>(1, (int64_t)ctx->sm_count * per_sm / cl);
    parts = (int)std::min<int64_t>(ceil_div(p.rows, rpb), cap);
    if (want_stats) p.partial = (float*)talos_workspace(ctx, sizeof(float) * 5 * (size_t)parts);
    talos_kernel_cluster(ctx, kern, (unsigned)(parts * cl), block, 0, (unsigned)cl, p);
  };
#define TALOS_L(LIM, W_, G_, NV_, CL_, PER_SM) if (p.vocab <= LIM) { go(policy_loss_kernel<W_, G_, NV_, CL_, ENT, PER_SM>, G_ <= 32 ? 256 / G_ : 1, block_of<G_>, PER_SM, CL_); return parts; }
  if (p.vocab % 4 == 0 && p.ld % 4 == 0 && aligned16(p.logits) && (!p.dlogits || (p.ld_out % 4 == 0 && aligned16(p.dlogits)))) {
    TALOS_L(16, 4, 4, 1, 1, 5) TALOS_L(64, 4, 8, 2, 1, 5) TALOS_L(256, 4, 32, 2, 1, 5) TALOS_L(1024, 4, 32, 8, 1, 3) TALOS_L(4096, 4, 256, 4, 1, 5)
    TALOS_L(8192, 4, 256, 8, 1, 3) TALOS_L(16384, 4, 256, 8, 2, 3) TALOS_L(32768, 4, 256, 8, 4, 3) TALOS_L(65536, 4, 256, 8, 8, 3) TALOS_L(131072, 4, 512, 8, 8, 1)
    TALOS_L(163840, 4, 512, 10, 8, 1)
  } else {
    TALOS_L(16, 1, 4, 4, 1, 5) TALOS_L(64, 1, 8, 8, 1, 5) TALOS_L(256, 1, 32, 8, 1, 5) TALOS_L(1024, 1, 32, 32, 1, 3) TALOS_L(4096, 1, 256, 16, 1, 5)
    TALOS_L(8192, 1, 256, 32, 1, 3) TALOS_L(16384, 1, 256, 32, 2, 3) TALOS_L(32768, 1, 256, 32, 4, 3) TALOS_L(65536, 1, 256, 32, 8, 3) TALOS_L(131072, 1, 512, 32, 8, 1)
    TALOS_L(163840, 1, 512, 40, 8, 1)
  }
#undef TALOS_L
  go(policy_loss_long_kernel<ENT>, 1, 1024, 2, 1);
  return parts;
}

}  // namespace

TALOS_API talos_status talos_policy_loss_fwd_bwd(talos_ctx* ctx, const float* logits, int64_t ld_logits, const int32_t* tokens, const float* old_logp,
                                                 const float* ref_logp, const float* adv, const float* weights, int64_t rows, int64_t vocab, float clip_low,
                                                 float clip_high, float c_kl, float c_entropy, float denom, float* logp, float* dlogits, int64_t ld_out,
                                                 float* stats, int32_t accumulate) {
  TALOS_ENTRY_BEGIN
  TALOS_REQUIRE(rows >= 0 && vocab >= 1 && vocab < (1 << 30), TALOS_ERR_SHAPE, "bad policy loss shape");
  TALOS_REQUIRE(ld_logits >= vocab && (!dlogits || ld_out >= vocab), TALOS_ERR_SHAPE, "row stride shorter than the vocabulary");
  TALOS_REQUIRE(clip_low >= 0.f && clip_low <= 1.f && clip_high >= 0.f && denom > 0.f, TALOS_ERR_ARG, "bad clip interval or denominator");
  TALOS_REQUIRE(accumulate == 0 || accumulate == 1, TALOS_ERR_ARG, "accumulate is 0 or 1");
  TALOS_REQUIRE(c_kl == 0.f || ref_logp, TALOS_ERR_ARG, "a KL term needs ref_logp");
  TALOS_REQUIRE(dlogits != logits || !dlogits || ld_out == ld_logits, TALOS_ERR_ARG, "dlogits over logits needs the same row stride");
  TALOS_REQUIRE((old_logp == nullptr) == (adv == nullptr) && (adv || !dlogits), TALOS_ERR_ARG, "the policy term needs old_logp and adv");
  TALOS_REQUIRE(rows == 0 || (logits && tokens), TALOS_ERR_ARG, "null pointer");
  talos_check_ctx(ctx);
  if (rows == 0) {
    if (stats && !accumulate) TALOS_CHECK_CUDA(cudaMemsetAsync(stats, 0, 5 * sizeof(float), ctx->stream));
    return TALOS_OK;
  }
  if (!logp && !dlogits && !stats) return TALOS_OK;
  LossArgs p{logits, (long long)ld_logits, tokens, old_logp, ref_logp, adv, weights, (long long)rows, (int)vocab, 1.f - clip_low, 1.f + clip_high, c_kl, c_entropy,
                   1.f / denom, logp, dlogits, (long long)ld_out, nullptr, ctx->dev_status};
  const int parts = c_entropy != 0.f ? loss_launch<true>(ctx, p, stats != nullptr) : loss_launch<false>(ctx, p, stats != nullptr);
  talos_launched(ctx, "policy_loss");
  if (stats) {
    talos_kernel(ctx, policy_stats_kernel, 1, 256, 0, p.partial, parts, stats, accumulate);
    talos_launched(ctx, "policy_stats");
  }
  TALOS_ENTRY_END
}
