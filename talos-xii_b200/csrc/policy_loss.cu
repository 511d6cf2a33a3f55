// Clipped policy loss with a KL term over a vocabulary, and its gradient, from a head's logits.
//
// Mathematics, per row z with token a: lse = log sum exp z, lp = z_a - lse, H = -sum p log p.  One pass leaves, per warp, its
// maximum m, s = sum exp(z - m) and t = sum exp(z - m) (z - m); triples combine by rescaling to the larger maximum, and at the end
// lse = m + log s, H = log s - t / s.  The loss is a function of lp and H, so its gradient is
//   dz_j = g (1[j = a] - p_j) + e p_j (log p_j + H),    g = dL/dlp, e = c_entropy w / denom.
// Bound: HBM, 8 bytes a logit (read once, its gradient written once).  A row therefore stays on chip, in the threads that own it, from the read to the write:
// in registers in 4 to 32 lanes for the few actions of a small policy (up to 1 024), in a CTA of 256 threads for up to 16 384 tokens, in a
// cluster of two to eight CTAs up to 131 072, whose warps push their triples into every CTA's shared memory, so that one cluster barrier a row is all they
// wait for; in the shared memory of a cluster of eight up to 425 984; longer rows are read twice by one CTA.  While a row is worked on, each thread
// copies its values of its group's next row into its own shared memory.  Units of four logits are dealt round the cluster, so that rows that
// are not aligned lose only their ends.  Measured: 4 096 x 32 000 in 174 us (6.0 TB/s), 2 048 x 50 257 in 189 (4.4), 1 024 x 128 256 in 186 (5.6), 1 024 x
// 151 936 in 292 (4.3), 64 x 430 000 in 254 (0.87), 65 536 x 16 in 9; the entropy term adds 3 to 9 %.
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

// Sums over a set of logits, relative to their maximum m and in base 2: x = (z - m) log2 e, s = sum 2^x, t = sum 2^x x.
// (m = -inf: nothing but -inf so far.  A NaN survives in s.)
struct Triple { float m, s, t; };
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
__device__ __forceinline__ float exp2_fast(float x) { float e; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x)); return e; }      // within 2^-22
// t of a triple whose maximum lies d (<= 0, base 2) below the new one, f = 2^d.  Where f is 0 nothing is left of it: a part whose logits are all some mask's low
// value is so far below that d or s d is infinite, and 0 inf would be NaN.
__device__ __forceinline__ float moved_t(float t, float s, float d, float f) { return f == 0.f ? 0.f : (t + s * d) * f; }
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
// The row's own numbers (read with its logits: behind the reductions they would cost a trip to memory a row).
struct RowIn { float w, adv, old, ref; };
__device__ __forceinline__ RowIn row_in(const LossArgs& p, long long r, float w) {
  RowIn i{w, 0.f, 0.f, 0.f};
  if (p.adv) { i.adv = p.adv[r]; i.old = p.old_logp[r]; }
  if (p.ref_logp) i.ref = p.ref_logp[r];
  return i;
}
__device__ __forceinline__ RowLoss row_loss(const LossArgs& p, const RowIn& in, float lp, float entropy) {
  RowLoss o{0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const float w = in.w;
  if (p.adv) {
    const float adv = in.adv, ratio = expf(lp - in.old);
    const float s1 = ratio * adv, s2 = fminf(fmaxf(ratio, p.lo), p.hi) * adv;
    const bool first = s1 < s2, inside = ratio >= p.lo && ratio <= p.hi;
    o.loss = -(first ? s1 : s2);
    o.g = first || inside ? -s1 : 0.f;
    o.clipped = !first && !inside && s2 < s1 ? w : 0.f;
    if (s1 != s1) { o.loss = s1; o.g = s1; }                              // NaN stays NaN
  }
  if (p.ref_logp) {
    const float d = in.ref - lp, em1 = expm1f(d);
    o.kl = em1 - d;
    if (p.c_kl != 0.f) { o.loss += p.c_kl * o.kl; o.g -= p.c_kl * em1; }
  }
  if (p.c_entropy != 0.f) o.loss -= p.c_entropy * entropy;
  const float scale = w * p.inv_denom;
  o.g *= scale; o.e = p.c_entropy * scale;
  o.loss *= w; o.kl *= w; o.entropy = w * entropy;
  return o;
}

// One of a row's gradient values, the token's own term left out, from its logit (ENT: v = z, otherwise v = 2^x, x relative to the warp's maximum, and
// c = -g p / v, the same for the warp).
template <bool ENT> __device__ __forceinline__ float dlogit(float v, float c, float top, float ls, float H, const RowLoss& k) {
  if constexpr (!ENT) return v * c;
  const float lp = (v - top) - ls, q = exp2_fast(lp * LOG2E);
  return q == 0.f ? 0.f : q * (k.e * (lp + H) - k.g);
}
// c of a warp with maximum m (mm: what its x are relative to).  One with nothing but -inf has values of 0 relative to mm = 0, which says nothing of where the row's
// logits lie: 2^(mm - lse) may be infinite there.  Its gradients are 0, in a row that has a NaN (S is one, too) NaN.
__device__ __forceinline__ float factor(float m, float mm, float top, float ls, float S, float g) {
  return m == -INFINITY ? S - S : -g * exp2_fast(((mm - top) - ls) * LOG2E);
}
// The token's own value.
__device__ __forceinline__ float dtoken(float lp, float H, const RowLoss& k) {
  const float q = expf(lp);
  return k.g * (1.f - q) + (q == 0.f ? 0.f : q * k.e * (lp + H));
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

// talos_pdl() of a launch whose clusters fill the SMs: the next kernel is let in only as this one's CTAs leave.  Let in at once, the next such launch
// would put clusters into the slots that this one leaves over, find the others one by one, and end up with fewer of its own resident at a
// time (2 048 rows of 50 257: 310 us instead of 220).
template <typename... T> __device__ __forceinline__ void pdl_late(T&... ptrs) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  ((void)([&] { asm volatile("" : "+l"(ptrs) : : "memory"); }()), ...);
}

// Where the rows of logits and gradient lie alike within 16 bytes, but not on them (SHIFT), units are the aligned groups of four around the row: the
// first and the last may hold less.  `a`: values of the first unit that lie before the row.
__device__ __forceinline__ int row_shift(const float* row) { return (int)(((uintptr_t)row >> 2) & 3); }

// G threads (of CL CTAs) own a row, NV groups of W values each.
template <int W, int G, int NV, int CL, bool ENT, int PER_SM, bool SHIFT>
__global__ void __launch_bounds__(block_of<G>, PER_SM) policy_loss_kernel(LossArgs p) {
  if constexpr (CL > 1) pdl_late(p.logits, p.tokens, p.old_logp, p.ref_logp, p.adv, p.weights, p.logp, p.dlogits, p.partial, p.status);
  else talos_pdl(p.logits, p.tokens, p.old_logp, p.ref_logp, p.adv, p.weights, p.logp, p.dlogits, p.partial, p.status);
  constexpr int RPB = G <= 32 ? 256 / G : 1, WARPS = G / 32 > 0 ? G / 32 : 1;
  __shared__ Triple parts[2][CL * WARPS];
  __shared__ float sums[8][5];
  const int l = G <= 32 ? threadIdx.x % G : threadIdx.x, sub = G <= 32 ? threadIdx.x / G : 0, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = CL > 1 ? (int)(blockIdx.x % CL) : 0;
  const long long first = (long long)(blockIdx.x / CL) * RPB, step = (long long)(gridDim.x / CL) * RPB;
  constexpr int HOP = G * CL;                                            // a row's units go round the threads of all its CTAs
  static_assert(!SHIFT || (W == 4 && G > 32), "shifted rows come in units of four");
  const int u0 = part * G + l;
  extern __shared__ float ahead[];                                       // G > 32: the next row, each thread its own units, while this one is worked on
  int phase = 0;
  float acc[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
  if constexpr (CL > 1) cg::this_cluster().sync();                       // every CTA of the cluster runs before one writes into it
  const uint32_t slot = (uint32_t)__cvta_generic_to_shared(ahead + threadIdx.x * W);
  auto request = [&](long long r) {
    const float* row = p.logits + r * p.ld;
    const int a = SHIFT ? row_shift(row) : 0, units = (p.vocab + a + W - 1) / W;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (u0 + v * HOP < units) {
        const int u = u0 + v * HOP;
        const float* src = row - a + (long long)u * W;
        if (SHIFT && (u == 0 || u == units - 1)) {
#pragma unroll
          for (int i = 0; i < W; ++i)
            if (u * W + i >= a && u * W + i < p.vocab + a) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(slot + v * (G * 16) + i * 4), "l"(src + i) : "memory");
          continue;
        }
        if constexpr (W == 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot + v * (G * 16)), "l"(src) : "memory");
        else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(slot + v * (G * 4)), "l"(src) : "memory");
      }
  };
  auto store = [&](float* out, int a, int units, int u, const float* o) {
    if (SHIFT && (u == 0 || u == units - 1)) {
#pragma unroll
      for (int i = 0; i < W; ++i) { const int j = u * W + i - a; if (j >= 0 && j < p.vocab) out[j] = o[i]; }
    } else store_units<W>(out - a + (long long)u * W, o);
  };
  int token = -1; float w = 0.f;
  bool live = false;
  if (G > 32 && first < p.rows) { live = counts(p, first, token, w, l == 0 && part == 0); if (live) request(first); }
  for (long long r0 = first; r0 < p.rows; r0 += step) {
    const long long r = r0 + sub;
    const bool in = r < p.rows;
    if constexpr (G <= 32) { token = -1; w = 0.f; live = in && counts(p, r, token, w, l == 0); }
    const float* row = p.logits + r * p.ld;
    const int a = SHIFT ? row_shift(row) : 0, units = (p.vocab + a + W - 1) / W;
    float z[NV][W];
    if constexpr (G > 32) {
      asm volatile("cp.async.wait_all;" ::: "memory");
      if (live) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          if (u0 + v * HOP < units) {
#pragma unroll
            for (int i = 0; i < W; ++i) z[v][i] = ahead[(v * G + threadIdx.x) * W + i];
            if (SHIFT && (u0 + v * HOP == 0 || u0 + v * HOP == units - 1)) {
#pragma unroll
              for (int i = 0; i < W; ++i) { const int j = (u0 + v * HOP) * W + i - a; if (j < 0 || j >= p.vocab) z[v][i] = -INFINITY; }
            }
          } else {
#pragma unroll
            for (int i = 0; i < W; ++i) z[v][i] = -INFINITY;
          }
        }
      }
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if (live && u0 + v * HOP < units) load_units<W>(row + (long long)(u0 + v * HOP) * W, z[v]);
        else {
#pragma unroll
          for (int i = 0; i < W; ++i) z[v][i] = -INFINITY;
        }
      }
    }
    RowIn own{};
    if (live) own = row_in(p, r, w);
    const float zt = live ? row[token] : 0.f;                            // before any thread of the row writes over it
    const int at = token;
    if constexpr (G > 32) {
      const bool now = live;
      live = r + step < p.rows && counts(p, r + step, token, w, l == 0 && part == 0);
      if (live) request(r + step);
      if (!now) {                                                        // padding: nothing is read (the same for the row's threads)
        if (p.dlogits) {
          const float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int v = 0; v < NV; ++v) if (u0 + v * HOP < units) store(p.dlogits + r * p.ld_out, a, units, u0 + v * HOP, zero);
        }
        if (p.logp && l == 0 && part == 0) p.logp[r] = 0.f;
        continue;
      }
    }
    const bool on = G > 32 || live;                                      // this row counts (`live` may speak of the next one)
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
        const float x = (z[v][i] - mm) * LOG2E, e = exp2_fast(x);
        s += e; t = fmaf(e, fmaxf(x, -1e30f), t);                        // (0 for -inf)
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
        const bool none = q[i].m == -INFINITY;
        const float d = none ? 0.f : (q[i].m - M) * LOG2E, f = exp2_fast(d);
        S += q[i].s * f; T += moved_t(q[i].t, q[i].s, d, f);
      }
      S = group_add<32>(S); T = group_add<32>(T);
      phase ^= 1;
    }
    const bool empty = S == 0.f;                                         // every logit -inf
    const float MM = M == -INFINITY ? 0.f : M, ls = logf(S), H = empty ? 0.f : ls - T / S * LN2;
    const float lp = empty ? -INFINITY : (zt - MM) - ls;      // (differences first: nothing is lost to large logits)
    RowLoss k{0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (on && !empty) k = row_loss(p, own, lp, H);
    if (on && l == 0 && part == 0) {
      if (p.logp) p.logp[r] = lp;
      if (!empty) { acc[0] += k.loss; acc[1] += k.kl; acc[2] += k.entropy; acc[3] += k.clipped; acc[4] += own.w; }
    } else if (in && !on && l == 0 && p.logp) p.logp[r] = 0.f;
    if (!p.dlogits || !in) continue;
    float* out = p.dlogits + r * p.ld_out;
    if (on && !empty) {
      const float c = factor(m, mm, MM, ls, S, k.g);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int u = u0 + v * HOP;
        if (u >= units) continue;
        float o[W];
#pragma unroll
        for (int i = 0; i < W; ++i) o[i] = dlogit<ENT>(z[v][i], c, MM, ls, H, k);
        store(out, a, units, u, o);
      }
      if (((at + a) / W) % HOP == u0) out[at] = dtoken(lp, H, k);              // the thread that wrote the token's unit
    } else {
      const float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < NV; ++v) if (u0 + v * HOP < units) store(out, a, units, u0 + v * HOP, zero);
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

// Rows that the registers of a cluster of eight do not hold: the same in their shared memory, W values at a time, without the look ahead.
template <int W, bool ENT>
__global__ void __launch_bounds__(512) policy_loss_wide_kernel(LossArgs p, int per) {      // per: units of W values a CTA holds
  pdl_late(p.logits, p.tokens, p.old_logp, p.ref_logp, p.adv, p.weights, p.logp, p.dlogits, p.partial, p.status);
  constexpr int CL = 8, G = 512, WARPS = G / 32;
  extern __shared__ float mine[];
  __shared__ Triple parts[2][CL * WARPS];
  cg::cluster_group cluster = cg::this_cluster();
  const int part = (int)(blockIdx.x % CL), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int units = p.vocab / W, first = part * per, n = max(0, min(per, units - first));
  const uint32_t slot = (uint32_t)__cvta_generic_to_shared(mine + threadIdx.x * W);
  int phase = 0;
  float acc[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
  cluster.sync();
  for (long long r = blockIdx.x / CL; r < p.rows; r += gridDim.x / CL) {
    int token; float w;
    float* out = p.dlogits + r * p.ld_out + (long long)first * W;
    if (!counts(p, r, token, w, threadIdx.x == 0 && part == 0)) {
      const float zero[4] = {0.f, 0.f, 0.f, 0.f};
      if (p.dlogits) for (int u = threadIdx.x; u < n; u += G) store_units<W>(out + (long long)u * W, zero);
      if (p.logp && threadIdx.x == 0 && part == 0) p.logp[r] = 0.f;
      continue;
    }
    const float* row = p.logits + r * p.ld;
    for (int u = threadIdx.x, k = 0; u < n; u += G, ++k) {
      const float* src = row + (long long)(first + u) * W;
      if constexpr (W == 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot + k * (G * 16)), "l"(src) : "memory");
      else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(slot + k * (G * 4)), "l"(src) : "memory");
    }
    const float zt = row[token];
    const RowIn own = row_in(p, r, w);
    asm volatile("cp.async.wait_all;" ::: "memory");
    float m = -INFINITY, s = 0.f, t = 0.f;
    for (int u = threadIdx.x; u < n; u += G)
#pragma unroll
      for (int i = 0; i < W; ++i) m = fmaxf(m, mine[u * W + i]);
    m = group_max<32>(m);
    const float mm = m == -INFINITY ? 0.f : m;
    for (int u = threadIdx.x; u < n; u += G)
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float x = (mine[u * W + i] - mm) * LOG2E, e = exp2_fast(x);
        s += e; t = fmaf(e, fmaxf(x, -1e30f), t);
        if constexpr (!ENT) mine[u * W + i] = e;
      }
    s = group_add<32>(s); t = group_add<32>(t);
    if (lane < CL) *cluster.map_shared_rank(&parts[phase][part * WARPS + warp], lane) = Triple{m, s, t};
    cluster.sync();
    Triple q[CL * WARPS / 32];
    float M = -INFINITY, S = 0.f, T = 0.f;
#pragma unroll
    for (int i = 0; i < CL * WARPS / 32; ++i) { q[i] = parts[phase][lane + 32 * i]; M = fmaxf(M, q[i].m); }
    M = group_max<32>(M);
#pragma unroll
    for (int i = 0; i < CL * WARPS / 32; ++i) {
      const float d = q[i].m == -INFINITY ? 0.f : (q[i].m - M) * LOG2E, f = exp2_fast(d);
      S += q[i].s * f; T += moved_t(q[i].t, q[i].s, d, f);
    }
    S = group_add<32>(S); T = group_add<32>(T);
    phase ^= 1;
    const bool empty = S == 0.f;
    const float MM = M == -INFINITY ? 0.f : M, ls = logf(S), H = empty ? 0.f : ls - T / S * LN2, lp = empty ? -INFINITY : (zt - MM) - ls;
    RowLoss k{0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (!empty) k = row_loss(p, own, lp, H);
    if (threadIdx.x == 0 && part == 0) {
      if (p.logp) p.logp[r] = lp;
      if (!empty) { acc[0] += k.loss; acc[1] += k.kl; acc[2] += k.entropy; acc[3] += k.clipped; acc[4] += w; }
    }
    if (!p.dlogits) continue;
    const float c = factor(m, mm, MM, ls, S, k.g);
    for (int u = threadIdx.x; u < n; u += G) {
      float o[W];
#pragma unroll
      for (int i = 0; i < W; ++i) o[i] = empty ? 0.f : dlogit<ENT>(mine[u * W + i], c, MM, ls, H, k);
      store_units<W>(out + (long long)u * W, o);
    }
    const int own_unit = token / W - first;
    if (!empty && own_unit >= 0 && own_unit < n && own_unit % G == (int)threadIdx.x) out[token - first * W] = dtoken(lp, H, k);
  }
  cluster.sync();
  if (p.partial && threadIdx.x == 0 && part == 0)
#pragma unroll
    for (int i = 0; i < 5; ++i) p.partial[(blockIdx.x / CL) * 5 + i] = acc[i];
}

// Rows that no cluster holds: a CTA a row, the row read twice.
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
    const RowIn own = row_in(p, r, w);
    float m = -INFINITY, s = 0.f, t = 0.f;
    auto join = [&](float M) {                                           // s, t relative to M (>= m)
      if (m != -INFINITY) { const float d = (m - M) * LOG2E, f = exp2_fast(d); t = moved_t(t, s, d, f); s *= f; }
      m = M;
    };
    for (int j0 = threadIdx.x; j0 < p.vocab; j0 += 8 * 1024) {
      float z[8];
      float top = m;
#pragma unroll
      for (int i = 0; i < 8; ++i) { z[i] = j0 + i * 1024 < p.vocab ? row[j0 + i * 1024] : -INFINITY; top = fmaxf(top, z[i]); }
      join(top);
      const float at = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int i = 0; i < 8; ++i) { const float x = (z[i] - at) * LOG2E, e = exp2_fast(x); s += e; t = fmaf(e, fmaxf(x, -1e30f), t); }
    }
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
    const float mm = m == -INFINITY ? 0.f : m, ls = logf(s), H = empty ? 0.f : ls - t / s * LN2, lp = empty ? -INFINITY : (zt - mm) - ls;
    RowLoss k{0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (!empty) k = row_loss(p, own, lp, H);
    if (threadIdx.x == 0) {
      if (p.logp) p.logp[r] = lp;
      if (!empty) { acc[0] += k.loss; acc[1] += k.kl; acc[2] += k.entropy; acc[3] += k.clipped; acc[4] += w; }
    }
    if (!p.dlogits) continue;
    const float c = empty ? 0.f : -k.g * exp2_fast(-ls * LOG2E);
    for (int j = threadIdx.x; j < p.vocab; j += 1024) {
      const float z = row[j];
      out[j] = empty ? 0.f : dlogit<ENT>(ENT ? z : exp2_fast((z - mm) * LOG2E), c, mm, ls, H, k);
    }
    if (!empty && token % 1024 == (int)threadIdx.x) out[token] = dtoken(lp, H, k);
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
  // (a cluster that is not resident at once would start when the first ones have finished their rows: a launch of 74 clusters of four, of which
  // the SMs' grouping holds 71, took 273 us instead of 176)
  auto go = [&](auto kern, int rpb, int block, int per_sm, int cl, size_t shmem, std::atomic<uint64_t>& done, std::atomic<int>& resident, auto... more) {
    if (shmem > 32 * 1024) talos_allow_smem(done, (const void*)kern, shmem, ctx->device);
    int64_t cap = std::max<int64_t>(1, (int64_t)ctx->sm_count * per_sm / cl);
    if (cl > 1) {
      int clusters = resident.load(std::memory_order_relaxed);
      if (clusters == 0) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)cl * (unsigned)cap); cfg.blockDim = dim3((unsigned)block); cfg.dynamicSmemBytes = shmem;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension; attr.val.clusterDim.x = (unsigned)cl; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
        cfg.attrs = &attr; cfg.numAttrs = 1;
        TALOS_CHECK_CUDA(cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg));
        resident.store(clusters = std::max(clusters, 1), std::memory_order_relaxed);
      }
      cap = std::min<int64_t>(cap, clusters) ;
    }
    parts = (int)std::min<int64_t>(ceil_div(p.rows, rpb), cap);
    if (want_stats) p.partial = (float*)talos_workspace(ctx, sizeof(float) * 5 * (size_t)parts);
    talos_kernel_cluster(ctx, kern, (unsigned)(parts * cl), block, shmem, (unsigned)cl, p, more...);
  };
  const bool vec = p.vocab % 4 == 0 && p.ld % 4 == 0 && aligned16(p.logits) && (!p.dlogits || (p.ld_out % 4 == 0 && aligned16(p.dlogits)));
  // rows of logits and gradient that lie alike within 16 bytes
  const bool alike = !p.dlogits || ((((uintptr_t)p.logits ^ (uintptr_t)p.dlogits) & 15) == 0 && ((p.ld ^ p.ld_out) & 3) == 0);
#define TALOS_L(LIM, W_, G_, NV_, CL_, PER_SM, SHIFT_) if (p.vocab <= LIM) { static std::atomic<uint64_t> done{0}; static std::atomic<int> resident{0}; \
    go(policy_loss_kernel<W_, G_, NV_, CL_, ENT, PER_SM, SHIFT_>, G_ <= 32 ? 256 / G_ : 1, block_of<G_>, PER_SM, CL_, G_ > 32 ? sizeof(float) * W_ * G_ * NV_ : 0, done, resident); return parts; }
  // (six and twelve units a thread between the powers of two: a row costs its slots, filled or not; 16 384 x 4 100 136 -> 129 us, 8 192 x 12 000 137 -> 130,
  // 4 096 x 40 001 352 -> 299, 2 048 x 70 001 378 -> 318)
  if (vec) {
    TALOS_L(16, 4, 4, 1, 1, 5, false) TALOS_L(64, 4, 8, 2, 1, 4, false) TALOS_L(256, 4, 32, 2, 1, 4, false) TALOS_L(1024, 4, 32, 8, 1, 3, false)
    TALOS_L(4096, 4, 256, 4, 1, 4, false) TALOS_L(6144, 4, 256, 6, 1, 3, false) TALOS_L(8192, 4, 256, 8, 1, 3, false) TALOS_L(12288, 4, 256, 12, 1, 2, false)
    TALOS_L(16384, 4, 256, 16, 1, 2, false) TALOS_L(24576, 4, 256, 12, 2, 2, false) TALOS_L(32768, 4, 256, 16, 2, 2, false) TALOS_L(49152, 4, 256, 12, 4, 2, false)
    TALOS_L(65536, 4, 256, 16, 4, 2, false) TALOS_L(98304, 4, 256, 12, 8, 2, false) TALOS_L(131072, 4, 256, 16, 8, 2, false)
  } else {
    TALOS_L(16, 1, 4, 4, 1, 5, false) TALOS_L(64, 1, 8, 8, 1, 5, false) TALOS_L(256, 1, 32, 8, 1, 5, false) TALOS_L(1024, 1, 32, 32, 1, 3, false)
    if (alike) {                                          // (three values of a unit may lie before the row)
      TALOS_L(4093, 4, 256, 4, 1, 4, true) TALOS_L(6141, 4, 256, 6, 1, 3, true) TALOS_L(8189, 4, 256, 8, 1, 3, true) TALOS_L(12285, 4, 256, 12, 1, 2, true)
      TALOS_L(16381, 4, 256, 16, 1, 2, true) TALOS_L(24573, 4, 256, 12, 2, 2, true) TALOS_L(32765, 4, 256, 16, 2, 2, true) TALOS_L(49149, 4, 256, 12, 4, 2, true)
      TALOS_L(65533, 4, 256, 16, 4, 2, true) TALOS_L(98301, 4, 256, 12, 8, 2, true) TALOS_L(131069, 4, 256, 16, 8, 2, true)
    } else {
      TALOS_L(4096, 1, 256, 16, 1, 4, false) TALOS_L(16384, 1, 256, 64, 1, 2, false) TALOS_L(32768, 1, 256, 64, 2, 2, false) TALOS_L(65536, 1, 256, 64, 4, 2, false)
      TALOS_L(131072, 1, 256, 64, 8, 2, false)
    }
  }
#undef TALOS_L
  constexpr int HELD = 8 * 53248;                         // 208 KB a CTA
  if (p.vocab <= HELD) {
    const int units = vec ? p.vocab / 4 : p.vocab, per = (int)ceil_div(units, 8);
    const size_t shmem = (size_t)per * (vec ? 16 : 4);
    const int per_sm = shmem <= 104 * 1024 ? 2 : 1;
    // (the kernel's shared memory limit is raised once, to the most; how many clusters are resident depends on the row)
    if (vec) {
      static std::atomic<uint64_t> done{0}; static std::atomic<int> resident[2];
      talos_allow_smem(done, (const void*)policy_loss_wide_kernel<4, ENT>, HELD / 8 * 4, ctx->device);
      go(policy_loss_wide_kernel<4, ENT>, 1, 512, per_sm, 8, shmem, done, resident[per_sm - 1], per);
    } else {
      static std::atomic<uint64_t> done{0}; static std::atomic<int> resident[2];
      talos_allow_smem(done, (const void*)policy_loss_wide_kernel<1, ENT>, HELD / 8 * 4, ctx->device);
      go(policy_loss_wide_kernel<1, ENT>, 1, 512, per_sm, 8, shmem, done, resident[per_sm - 1], per);
    }
    return parts;
  }
  static std::atomic<uint64_t> done{0}; static std::atomic<int> resident{0};
  go(policy_loss_long_kernel<ENT>, 1, 1024, 2, 1, 0, done, resident);
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
