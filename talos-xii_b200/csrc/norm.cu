// Layer norm, dropout, and their junction in a transformer block (h = residual + dropout(x), y = layer norm of h), forward and
// backward: one pass over the rows each way, the row in registers between the statistics and the result.
//
// Mathematics.  mean and the centred sum of squares are taken from the registers one after the other (two reductions, no
// E[x^2] - E[x]^2).  Backward, with g = dy * gamma and xh = (x - mean) * inv: dx = inv * (g - mean(g) - xh * mean(g * xh)); both
// means travel in one reduction.  The gradients of gamma and beta are column sums: every thread keeps its columns' sums over all the
// rows of its CTA, a CTA leaves one partial row of each, and a second small kernel adds the partial rows in order.
// Bound: HBM.  Layer norm moves 8 bytes an element forward and 12 backward, the junction 16 and 20.  Measured: layer norm 8 191 x 4 096
// 48 us forward (5.6 TB/s) and 78 backward (5.2, with the 10 us of the column sums' second kernel); junction 65 536 x 256 50 us (5.3) and 56 (6.0); dropout of
// 16.8 M elements with residual 35 us (5.8), its backward 25 (5.4).  Junction backward of 65 536 rows at other widths, with and without dropout: 257 160 and 134,
// 260 87 and 64, 253 121 and 104: an unaligned row loses most at its ends, which are copied, read and stored value by value.  Tensors that all lie
// four bytes off, whose units have factors of two draws: 256 209 and 129.
// Split: a group of G threads owns a row, G = 8 to 32 lanes of a warp (dim <= 256) or a CTA of 128 to 1 024 threads, so that a thread
// holds at most eight values of a row (16 above 8 192): no spills beside the column sums.  Each thread copies its own values of the next row into
// its own shared memory while it works on this one, so that loads are in flight during the reductions.
// Rows whose width is no multiple of four start anywhere: where all tensors of a call lie alike within 16 bytes, a row's units are the aligned groups of
// four around it (SHIFT); a group's rows are a multiple of four apart, so its shift, and with it its columns, stay the same.
#include <initializer_list>
#include <type_traits>

#include "philox.cuh"

#include "../../include/talos_b200_lm.h"

namespace {

constexpr int MAX_DIM = 16384;

template <int W> struct alignas(4 * W) Vec { float a[W]; };
// (__ldcs / __stcs: data that this kernel reads or writes once)
template <int W> __device__ __forceinline__ Vec<W> ldv(const float* p) {
  Vec<W> v;
  if constexpr (W == 4) { const float4 q = __ldcs((const float4*)p); v.a[0] = q.x; v.a[1] = q.y; v.a[2] = q.z; v.a[3] = q.w; }
  else v.a[0] = __ldcs(p);
  return v;
}
template <int W> __device__ __forceinline__ void stv(float* p, const Vec<W>& v) {
  if constexpr (W == 4) __stcs((float4*)p, make_float4(v.a[0], v.a[1], v.a[2], v.a[3]));
  else __stcs(p, v.a[0]);
}
template <int W> __device__ __forceinline__ Vec<W> fill(float f) { Vec<W> v; 
#pragma unroll
  for (int i = 0; i < W; ++i) v.a[i] = f;
  return v;
}
// (called where sixteen draws in line would spill)
__device__ __noinline__ float drop_one(uint32_t k0, uint32_t k1, uint32_t threshold, float scale, unsigned long long offset, unsigned long long i) {
  DropArgs d{};
  d.k0 = k0; d.k1 = k1; d.threshold = threshold; d.scale = scale;
  return talos_drop1(d, offset, i);
}
// Dropout factors of the W elements from `i` (i % 4 == 0 where W is 4).
template <int W> __device__ __forceinline__ Vec<W> drop(const DropArgs& d, unsigned long long offset, long long i) {
  Vec<W> v;
  if constexpr (W == 4) { const float4 f = talos_drop4(d, offset, (unsigned long long)i >> 2); v.a[0] = f.x; v.a[1] = f.y; v.a[2] = f.z; v.a[3] = f.w; }
  else v.a[0] = drop_one(d.k0, d.k1, d.threshold, d.scale, offset, (unsigned long long)i);
  return v;
}
__device__ __forceinline__ float dropped(float x, float f) { return f != 0.f ? x * f : 0.f; }     // a dropped NaN is 0, too
__device__ __forceinline__ unsigned long long run_offset(const DropArgs& d) { return d.offset + (d.offset_dev ? *d.offset_dev : 0ull); }

// Sums of (a, b) over a row's group; every thread gets them.  `phase` alternates between calls, so that one block barrier a call is enough.
template <int G> __device__ __forceinline__ float2 group_sum(float a, float b, float2 (*sh)[32], int& phase) {
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1) { a += __shfl_xor_sync(0xffffffffu, a, o); b += __shfl_xor_sync(0xffffffffu, b, o); }
  if constexpr (G > 32) {
    if ((threadIdx.x & 31) == 0) sh[phase][threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < G / 32; ++i) { const float2 s = sh[phase][i]; a += s.x; b += s.y; }
    phase ^= 1;
  }
  return make_float2(a, b);
}
template <int G> constexpr int block_of = G <= 32 ? 256 : G;
template <int G> constexpr int rows_per_block = G <= 32 ? 256 / G : 1;

template <int W> __device__ __forceinline__ void copy_unit(uint32_t dst, const float* src) {
  if constexpr (W == 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// A thread's share of its group's rows.  a: values of the first unit that lie before the row (SHIFT).
template <int W, int G, int NV, bool SHIFT> struct Share {
  int l, a, units, dim;
  __device__ __forceinline__ Share(const float* x, long long row, int d) {
    l = G <= 32 ? threadIdx.x % G : threadIdx.x; dim = d;
    a = SHIFT ? (int)((((uintptr_t)x >> 2) + (unsigned long long)row * (unsigned)d) & 3) : 0;
    units = (d + a + W - 1) / W;
  }
  __device__ __forceinline__ int unit(int v) const { return l + v * G; }
  __device__ __forceinline__ bool has(int v) const { return unit(v) < units; }
  __device__ __forceinline__ bool edge(int v) const { return SHIFT && (unit(v) == 0 || unit(v) == units - 1); }
  __device__ __forceinline__ int column(int v, int i) const { return unit(v) * W + i - a; }
  __device__ __forceinline__ bool in(int v, int i) const { const int c = column(v, i); return has(v) && (!SHIFT || (c >= 0 && c < dim)); }
  // Copies this thread's units of a row to its slots (blockDim units apart), waits for them elsewhere.
  __device__ __forceinline__ void request(uint32_t slot, const float* row) const {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (!has(v)) continue;
      const float* src = row - a + (long long)unit(v) * W;
      const uint32_t dst = slot + v * blockDim.x * (W * 4);
      if (edge(v)) {
#pragma unroll
        for (int i = 0; i < W; ++i) if (in(v, i)) copy_unit<1>(dst + i * 4, src + i);
      } else copy_unit<W>(dst, src);
    }
  }
  __device__ __forceinline__ Vec<W> clean(int v, Vec<W> x) const {      // zeros outside the row
    if (!has(v)) return fill<W>(0.f);
    if (edge(v)) {
#pragma unroll
      for (int i = 0; i < W; ++i) if (!in(v, i)) x.a[i] = 0.f;
    }
    return x;
  }
  __device__ __forceinline__ Vec<W> take(const float* slot, int v) const { return clean(v, *(const Vec<W>*)(slot + v * blockDim.x * W)); }
  __device__ __forceinline__ Vec<W> load(const float* row, int v) const {
    if (!has(v)) return fill<W>(0.f);
    const float* src = row - a + (long long)unit(v) * W;
    if (!edge(v)) return ldv<W>(src);
    Vec<W> x = fill<W>(0.f);
#pragma unroll
    for (int i = 0; i < W; ++i) if (in(v, i)) x.a[i] = src[i];
    return x;
  }
  __device__ __forceinline__ void store(float* row, int v, const Vec<W>& x) const {
    if (!has(v)) return;
    float* dst = row - a + (long long)unit(v) * W;
    if (!edge(v)) { stv<W>(dst, x); return; }
#pragma unroll
    for (int i = 0; i < W; ++i) if (in(v, i)) dst[i] = x.a[i];
  }
  // Dropout factors of a unit; `first`: the row's first element.
  __device__ __forceinline__ Vec<W> factors(const DropArgs& d, unsigned long long offset, long long first, int v) const {
    const long long e = first + column(v, 0);
    if constexpr (SHIFT) {
      if (e & 3) {                                        // the tensors themselves are not aligned: a unit has values of two draws
        Vec<W> f;
#pragma unroll
        for (int i = 0; i < W; ++i) f.a[i] = in(v, i) ? talos_drop1(d, offset, (unsigned long long)(e + i)) : 0.f;
        return f;
      }
    }
    return drop<W>(d, offset, e);
  }
};

struct NormFwd {
  const float *x, *residual, *gamma, *beta; float *h, *y, *mean, *inv;
  float eps; long long rows; int dim; DropArgs drop;
};

// AHEAD: the next row is copied to shared memory while this one is worked on.
template <int W, int G, int NV, bool FUSED, bool SHIFT, bool AHEAD>
__global__ void __launch_bounds__(block_of<G>) norm_fwd_kernel(NormFwd p) {
  talos_pdl(p.x, p.residual, p.gamma, p.beta, p.h, p.y, p.mean, p.inv, p.drop.offset_dev);
  extern __shared__ float ahead[];
  __shared__ float2 sh[2][32];
  int phase = 0;
  const int sub = G <= 32 ? threadIdx.x / G : 0;
  const float inv_dim = 1.f / (float)p.dim;
  const unsigned long long offset = FUSED ? run_offset(p.drop) : 0;
  const long long step = (long long)gridDim.x * rows_per_block<G>;
  const Share<W, G, NV, SHIFT> me(p.x, (long long)blockIdx.x * rows_per_block<G> + sub, p.dim);
  constexpr bool HOIST = NV * W <= 12;                    // gamma and beta stay in registers over the rows
  Vec<W> gam[HOIST ? NV : 1], bet[HOIST ? NV : 1];
  if constexpr (HOIST) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < W; ++i) {
        gam[v].a[i] = p.gamma && me.in(v, i) ? p.gamma[me.column(v, i)] : 1.f;
        bet[v].a[i] = p.beta && me.in(v, i) ? p.beta[me.column(v, i)] : 0.f;
      }
  }
  const float* mine = ahead + threadIdx.x * W;
  const uint32_t slot = (uint32_t)__cvta_generic_to_shared(mine), second = NV * block_of<G> * W * 4;
  auto request = [&](long long r) {
    if (r < p.rows) {
      me.request(slot, p.x + r * p.dim);
      if (FUSED && p.residual) me.request(slot + second, p.residual + r * p.dim);
    }
  };
  if constexpr (AHEAD) request((long long)blockIdx.x * rows_per_block<G> + sub);
  for (long long r0 = (long long)blockIdx.x * rows_per_block<G>; r0 < p.rows; r0 += step) {
    const long long r = r0 + sub, base = r * p.dim;
    const bool ok = r < p.rows;
    Vec<W> xv[NV], rv[FUSED ? NV : 1];
    if constexpr (AHEAD) {
      asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        xv[v] = ok ? me.take(mine, v) : fill<W>(0.f);
        if constexpr (FUSED) rv[v] = ok && p.residual ? me.take(mine + second / 4, v) : fill<W>(0.f);
      }
      request(r + step);
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        xv[v] = ok ? me.load(p.x + base, v) : fill<W>(0.f);
        if constexpr (FUSED) rv[v] = ok && p.residual ? me.load(p.residual + base, v) : fill<W>(0.f);
      }
    }
    if constexpr (FUSED) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if (!ok || !me.has(v)) continue;
        if (p.drop.threshold) {
          const Vec<W> f = me.factors(p.drop, offset, base, v);
#pragma unroll
          for (int i = 0; i < W; ++i) xv[v].a[i] = dropped(xv[v].a[i], f.a[i]);
        }
#pragma unroll
        for (int i = 0; i < W; ++i) xv[v].a[i] += rv[v].a[i];
        me.store(p.h + base, v, xv[v]);
      }
    }
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < W; ++i) s += xv[v].a[i];
    const float mean = group_sum<G>(s, 0.f, sh, phase).x * inv_dim;
    float q = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < W; ++i) { const float t = xv[v].a[i] - mean; if (me.in(v, i)) q = fmaf(t, t, q); }
    const float inv = 1.f / sqrtf(group_sum<G>(q, 0.f, sh, phase).x * inv_dim + p.eps);
    if (ok && me.l == 0) { if (p.mean) p.mean[r] = mean; if (p.inv) p.inv[r] = inv; }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (!ok || !me.has(v)) continue;
      Vec<W> o;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const bool in = me.in(v, i);
        const float gm = HOIST ? gam[HOIST ? v : 0].a[i] : p.gamma && in ? p.gamma[me.column(v, i)] : 1.f, bt = HOIST ? bet[HOIST ? v : 0].a[i] : p.beta && in ? p.beta[me.column(v, i)] : 0.f;
        o.a[i] = (xv[v].a[i] - mean) * inv * gm + bt;
      }
      me.store(p.y + base, v, o);
    }
  }
}

struct NormBwd {
  const float *dy, *dh, *x, *gamma, *mean, *inv; float *dx, *dresidual, *partial, *dgamma, *dbeta;
  long long rows; int dim; int accumulate; DropArgs drop;
};

// partial[CTA][2][dim]: this CTA's sums of dy * xh and of dy; a launch of one CTA writes dgamma and dbeta itself.  Without AHEAD (the widest rows)
// the column sums are held in shared memory, each thread its own.
template <int W, int G, int NV, bool FUSED, bool SHIFT, bool AHEAD>
__global__ void __launch_bounds__(block_of<G>) norm_bwd_kernel(NormBwd p) {
  talos_pdl(p.dy, p.dh, p.x, p.gamma, p.mean, p.inv, p.dx, p.dresidual, p.partial, p.dgamma, p.dbeta, p.drop.offset_dev);
  extern __shared__ float pool[];                       // AHEAD: the slots, then (G <= 32) the groups' sums over them; otherwise sums [2][units of a thread][threads]
  __shared__ float2 sh[2][32];
  int phase = 0;
  const int sub = G <= 32 ? threadIdx.x / G : 0;
  const float inv_dim = 1.f / (float)p.dim;
  const unsigned long long offset = FUSED ? run_offset(p.drop) : 0;
  const long long step = (long long)gridDim.x * rows_per_block<G>, start = (long long)blockIdx.x * rows_per_block<G> + sub;
  const Share<W, G, NV, SHIFT> me(p.x, start, p.dim);
  constexpr bool HOIST = NV * W <= 12;
  constexpr int HELD = AHEAD ? NV : 1;
  Vec<W> gam[HOIST ? NV : 1], dg[HELD], db[HELD];
  auto sum_at = [&](int which, int v) { return (Vec<W>*)(pool + ((which * NV + v) * block_of<G> + threadIdx.x) * W); };
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if constexpr (HOIST) {
#pragma unroll
      for (int i = 0; i < W; ++i) gam[v].a[i] = p.gamma && me.in(v, i) ? p.gamma[me.column(v, i)] : 1.f;
    }
    if constexpr (AHEAD) dg[v] = db[v] = fill<W>(0.f);
    else *sum_at(0, v) = *sum_at(1, v) = fill<W>(0.f);
  }
  const float* mine = pool + threadIdx.x * W;
  const uint32_t slot = (uint32_t)__cvta_generic_to_shared(mine);
  constexpr int NEXT = NV * block_of<G> * W;             // floats between the slots of dy, x, dh
  const bool wants = p.dx || p.dresidual;
  float mean_next = 0.f, inv_next = 0.f;
  auto request = [&](long long r) {
    if (r < p.rows) {
      me.request(slot, p.dy + r * p.dim);
      me.request(slot + NEXT * 4, p.x + r * p.dim);
      if (FUSED && p.dh) me.request(slot + 2 * NEXT * 4, p.dh + r * p.dim);
      mean_next = p.mean[r]; inv_next = p.inv[r];
    }
  };
  if constexpr (AHEAD) request(start);
  for (long long r0 = (long long)blockIdx.x * rows_per_block<G>; r0 < p.rows; r0 += step) {
    const long long r = r0 + sub, base = r * p.dim;
    const bool ok = r < p.rows;
    Vec<W> gv[NV], xv[NV], ev[FUSED && AHEAD ? NV : 1];
    float mean, inv;
    if constexpr (AHEAD) {
      asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        gv[v] = ok ? me.take(mine, v) : fill<W>(0.f);
        xv[v] = ok ? me.take(mine + NEXT, v) : fill<W>(0.f);
        if constexpr (FUSED) ev[v] = ok && p.dh ? me.take(mine + 2 * NEXT, v) : fill<W>(0.f);
      }
      mean = ok ? mean_next : 0.f; inv = ok ? inv_next : 0.f;
      request(r + step);
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v) { gv[v] = ok ? me.load(p.dy + base, v) : fill<W>(0.f); xv[v] = ok ? me.load(p.x + base, v) : fill<W>(0.f); }
      mean = ok ? p.mean[r] : 0.f; inv = ok ? p.inv[r] : 0.f;
    }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      Vec<W> sg, sb;
      if constexpr (!AHEAD) { sg = *sum_at(0, v); sb = *sum_at(1, v); }
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float gm = HOIST ? gam[HOIST ? v : 0].a[i] : p.gamma && me.in(v, i) ? p.gamma[me.column(v, i)] : 1.f;
        const float d = gv[v].a[i], xh = (xv[v].a[i] - mean) * inv;      // (d = 0 outside the row)
        if constexpr (AHEAD) { dg[v].a[i] = fmaf(d, xh, dg[v].a[i]); db[v].a[i] += d; }
        else { sg.a[i] = fmaf(d, xh, sg.a[i]); sb.a[i] += d; }
        xv[v].a[i] = xh; gv[v].a[i] = d * gm;
        s1 += gv[v].a[i]; s2 = fmaf(gv[v].a[i], xh, s2);
      }
      if constexpr (!AHEAD) { *sum_at(0, v) = sg; *sum_at(1, v) = sb; }
    }
    if (!wants) continue;                                 // (the same for all threads)
    const float2 s = group_sum<G>(s1, s2, sh, phase);
    const float m1 = s.x * inv_dim, m2 = s.y * inv_dim;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (!ok || !me.has(v)) continue;
      Vec<W> o;
#pragma unroll
      for (int i = 0; i < W; ++i) o.a[i] = inv * (gv[v].a[i] - m1 - xv[v].a[i] * m2);
      if constexpr (FUSED) {
        if (p.dh) {
          const Vec<W> e = AHEAD ? ev[AHEAD ? v : 0] : me.load(p.dh + base, v);
#pragma unroll
          for (int i = 0; i < W; ++i) o.a[i] += e.a[i];
        }
        Vec<W> t = o;
        if (p.dx && p.drop.threshold) {
          const Vec<W> f = me.factors(p.drop, offset, base, v);
#pragma unroll
          for (int i = 0; i < W; ++i) t.a[i] = dropped(t.a[i], f.a[i]);
        }
        if (p.dresidual) {
          if (p.accumulate & 8) {
            const Vec<W> old = me.load(p.dresidual + base, v);
#pragma unroll
            for (int i = 0; i < W; ++i) o.a[i] += old.a[i];
          }
          me.store(p.dresidual + base, v, o);
        }
        o = t;
      }
      if (p.dx) {
        if (p.accumulate & 1) {
          const Vec<W> old = me.load(p.dx + base, v);
#pragma unroll
          for (int i = 0; i < W; ++i) o.a[i] += old.a[i];
        }
        me.store(p.dx + base, v, o);
      }
    }
  }
  if (!p.dgamma && !p.dbeta) return;
  const bool only = gridDim.x == 1;
  auto put = [&](int c, float a, float b) {
    if (only) {
      if (p.dgamma) p.dgamma[c] = (p.accumulate & 2) ? p.dgamma[c] + a : a;
      if (p.dbeta) p.dbeta[c] = (p.accumulate & 4) ? p.dbeta[c] + b : b;
    } else {
      float* out = p.partial + (size_t)blockIdx.x * 2 * p.dim;
      out[c] = a; out[p.dim + c] = b;
    }
  };
  if constexpr (G <= 32) {
    __syncthreads();                                      // (no copies are in flight: the slots are free)
    float* sums = pool + (size_t)sub * 2 * p.dim;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < W; ++i) if (me.in(v, i)) { sums[me.column(v, i)] = dg[v].a[i]; sums[p.dim + me.column(v, i)] = db[v].a[i]; }
    __syncthreads();
    for (int c = threadIdx.x; c < p.dim; c += blockDim.x) {
      float a = 0.f, b = 0.f;
      for (int i = 0; i < rows_per_block<G>; ++i) { a += pool[(size_t)i * 2 * p.dim + c]; b += pool[(size_t)i * 2 * p.dim + p.dim + c]; }
      put(c, a, b);
    }
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      Vec<W> sg, sb;
      if constexpr (AHEAD) { sg = dg[v]; sb = db[v]; } else { sg = *sum_at(0, v); sb = *sum_at(1, v); }
#pragma unroll
      for (int i = 0; i < W; ++i) if (me.in(v, i)) put(me.column(v, i), sg.a[i], sb.a[i]);
    }
  }
}

// dgamma and dbeta from the CTAs' partial rows: 32 columns of [dgamma | dbeta] a CTA, 32 lanes down the parts, added in a fixed order.
__global__ void __launch_bounds__(1024)
norm_param_grads_kernel(const float* partial, int nparts, int dim, float* dgamma, float* dbeta, int accumulate) {
  talos_pdl(partial, dgamma, dbeta);
  __shared__ float sh[32][33];
  const int cl = threadIdx.x & 31, pl = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;
  float s = 0.f;
  if (c < 2 * dim) {
#pragma unroll 8
    for (int i = pl; i < nparts; i += 32) s += partial[(size_t)i * 2 * dim + c];
  }
  sh[pl][cl] = s;
  __syncthreads();
  // warp w sums column w over the lanes
  float t = sh[cl][pl];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  const int col = blockIdx.x * 32 + pl;
  if (cl == 0 && col < 2 * dim) {
    float* out = col < dim ? dgamma : dbeta;
    const int at = col < dim ? col : col - dim, acc = col < dim ? accumulate & 2 : accumulate & 4;
    if (out) out[at] = acc ? out[at] + t : t;
  }
}

// y = residual + dropped(x), or dx (+)= dropped(dy): four elements to a draw.  W = 1: buffers that are not 16-byte aligned.
// U draws a thread and step: their loads are in flight before the first draw's 20 products and 40 logic operations.
template <int W, int U>
__global__ void __launch_bounds__(256) dropout_kernel(const float* x, const float* residual, float* y, long long n, DropArgs d) {
  talos_pdl(x, residual, y, d.offset_dev);
  const unsigned long long offset = run_offset(d);
  const long long blocks = (n + 3) / 4, step = (long long)gridDim.x * blockDim.x;
  for (long long b0 = (long long)blockIdx.x * blockDim.x + threadIdx.x; b0 < blocks; b0 += U * step) {
    Vec<4> xv[U], rv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long i = (b0 + u * step) * 4;
      xv[u] = rv[u] = fill<4>(0.f);
      if (W == 4 && i + 4 <= n) {
        xv[u] = ldv<4>(x + i);
        if (residual) rv[u] = ldv<4>(residual + i);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) if (i + j < n) { xv[u].a[j] = x[i + j]; if (residual) rv[u].a[j] = residual[i + j]; }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long b = b0 + u * step, i = b * 4;
      if (d.threshold) {
        const Vec<4> f = drop<4>(d, offset, i);
#pragma unroll
        for (int j = 0; j < 4; ++j) xv[u].a[j] = dropped(xv[u].a[j], f.a[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) xv[u].a[j] += rv[u].a[j];
      if (W == 4 && i + 4 <= n) stv<4>(y + i, xv[u]);
      else {
#pragma unroll
        for (int j = 0; j < 4; ++j) if (i + j < n) y[i + j] = xv[u].a[j];
      }
    }
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// f(W, G, NV, SHIFT, AHEAD) by row width.  units: the most that a row has (a shifted row one more than its width needs).
enum { ROWS_ALIGNED, ROWS_SHIFTED, ROWS_ANY };
template <typename F> void by_width(int rows, int dim, F&& f) {
  using std::integral_constant; using std::true_type; using std::false_type;
#define TALOS_N(W_, G_, NV_, SHIFT_, AHEAD_) return f(integral_constant<int, W_>(), integral_constant<int, G_>(), integral_constant<int, NV_>(), SHIFT_(), AHEAD_())
#define TALOS_NS(G_, NV_, AHEAD_) { if (rows == ROWS_ALIGNED) TALOS_N(4, G_, NV_, false_type, AHEAD_); else TALOS_N(4, G_, NV_, true_type, AHEAD_); }
  if (rows != ROWS_ANY) {
    const int u = rows == ROWS_ALIGNED ? dim / 4 : (dim + 6) / 4;
    if (u <= 8) TALOS_NS(8, 1, true_type)
    if (u <= 16) TALOS_NS(16, 1, true_type)
    if (u <= 32) TALOS_NS(32, 1, true_type)
    if (u <= 64) TALOS_NS(32, 2, true_type)
    if (u <= 96) TALOS_NS(32, 3, true_type)
    if (u <= 128) TALOS_NS(128, 1, true_type)
    if (u <= 256) TALOS_NS(128, 2, true_type)
    if (u <= 384) TALOS_NS(128, 3, true_type)
    if (u <= 512) TALOS_NS(256, 2, true_type)
    if (u <= 768) TALOS_NS(256, 3, true_type)
    if (u <= 1024) TALOS_NS(512, 2, true_type)
    if (u <= 1536) TALOS_NS(512, 3, true_type)
    if (u <= 2048) TALOS_NS(512, 4, true_type)
    if (u <= 4096) TALOS_NS(1024, 4, false_type)
    // (a shifted row of 16 384 values may have 4 097 units)
  }
  if (dim <= 256) TALOS_N(1, 32, 8, false_type, true_type);
  if (dim <= 1024) TALOS_N(1, 128, 8, false_type, true_type);
  if (dim <= 8192) TALOS_N(1, 1024, 8, false_type, false_type);
  TALOS_N(1, 1024, 16, false_type, false_type);
#undef TALOS_NS
#undef TALOS_N
}
// How the rows of a call's tensors lie: all aligned, all alike within 16 bytes, or neither.
int rows_of(int dim, std::initializer_list<const void*> tensors) {
  uintptr_t low = 16;
  for (const void* t : tensors) {
    if (!t) continue;
    if (low == 16) low = (uintptr_t)t & 15;
    else if (((uintptr_t)t & 15) != low) return ROWS_ANY;
  }
  return low == 0 && dim % 4 == 0 ? ROWS_ALIGNED : ROWS_SHIFTED;
}

// A CTA a group of rows up to what is resident at once, then a multiple of four CTAs, so that a group's rows keep their shift.
template <typename K> unsigned row_grid(talos_ctx* ctx, std::atomic<int>& resident, K kern, int block, size_t shmem, int64_t rows, int64_t per_block) {
  int per_sm = resident.load(std::memory_order_relaxed);
  if (per_sm == 0) {
    TALOS_CHECK_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, block, shmem));
    resident.store(per_sm = std::max(per_sm, 1), std::memory_order_relaxed);
  }
  return (unsigned)std::min<int64_t>(ceil_div(rows, per_block), std::max<int64_t>(4, ((int64_t)ctx->sm_count * per_sm) & ~3ll));
}

template <bool FUSED> void norm_fwd_launch(talos_ctx* ctx, const NormFwd& p, const char* what) {
  by_width(rows_of(p.dim, {p.x, p.y, p.residual, p.h}), p.dim, [&](auto w, auto g, auto nv, auto shift, auto ahead) {
    constexpr int W = decltype(w)::value, G = decltype(g)::value, NV = decltype(nv)::value; constexpr bool SHIFT = decltype(shift)::value, AHEAD = decltype(ahead)::value;
    constexpr size_t shmem = AHEAD ? sizeof(float) * W * NV * block_of<G> * (FUSED ? 2 : 1) : 0;
    static std::atomic<uint64_t> done{0}; static std::atomic<int> resident{0};
    auto kern = norm_fwd_kernel<W, G, NV, FUSED, SHIFT, AHEAD>;
    if (shmem > 32 * 1024) talos_allow_smem(done, (const void*)kern, shmem, ctx->device);
    talos_kernel(ctx, kern, row_grid(ctx, resident, kern, block_of<G>, shmem, p.rows, rows_per_block<G>), block_of<G>, shmem, p);
  });
  talos_launched(ctx, what);
}

template <bool FUSED> void norm_bwd_launch(talos_ctx* ctx, NormBwd p, const char* what) {
  const bool params = p.dgamma || p.dbeta;
  unsigned grid = 1;
  by_width(rows_of(p.dim, {p.x, p.dy, p.dx, p.dh, p.dresidual}), p.dim, [&](auto w, auto g, auto nv, auto shift, auto ahead) {
    constexpr int W = decltype(w)::value, G = decltype(g)::value, NV = decltype(nv)::value; constexpr bool SHIFT = decltype(shift)::value, AHEAD = decltype(ahead)::value;
    constexpr size_t slots = sizeof(float) * W * NV * block_of<G> * (AHEAD ? (FUSED ? 3 : 2) : 2);
    const size_t shmem = std::max(slots, G <= 32 ? sizeof(float) * 2 * (size_t)p.dim * rows_per_block<G> : 0);
    static std::atomic<uint64_t> done{0}; static std::atomic<int> resident{0};
    auto kern = norm_bwd_kernel<W, G, NV, FUSED, SHIFT, AHEAD>;
    if (slots > 32 * 1024) talos_allow_smem(done, (const void*)kern, slots, ctx->device);
    // (two rows a thread group before there are more CTAs than SMs: every CTA leaves a partial row; 1 200 x 768 with one 12.7 us, two 10.2, eight 11.4)
    grid = std::min(row_grid(ctx, resident, kern, block_of<G>, shmem, p.rows, rows_per_block<G>),
                    (unsigned)std::max<int64_t>(ctx->sm_count & ~3, ceil_div(p.rows, 2 * rows_per_block<G>) & ~3ll));
    if (params && grid > 1) p.partial = (float*)talos_workspace(ctx, sizeof(float) * 2 * (size_t)p.dim * grid);
    talos_kernel(ctx, kern, grid, block_of<G>, shmem, p);
  });
  talos_launched(ctx, what);
  if (params && grid > 1) {
    talos_kernel(ctx, norm_param_grads_kernel, (unsigned)ceil_div(2 * p.dim, 32), 1024, 0, p.partial, (int)grid, p.dim, p.dgamma, p.dbeta, p.accumulate);
    talos_launched(ctx, "norm_param_grads");
  }
}

void norm_shape(int64_t rows, int64_t dim) {
  TALOS_REQUIRE(rows >= 0 && dim > 0 && dim <= MAX_DIM, TALOS_ERR_SHAPE, "layer norm supports rows of 1 to 16384 values");
  TALOS_REQUIRE(rows <= INT64_MAX / MAX_DIM / 4, TALOS_ERR_SHAPE, "too many rows");
}

void dropout_launch(talos_ctx* ctx, const float* x, const float* residual, float* y, int64_t n, const DropArgs& d, const char* what) {
  const int64_t ctas = ceil_div(ceil_div(n, 4), 256), most = (int64_t)ctx->sm_count * 4;
  const unsigned grid = (unsigned)std::min<int64_t>(ctas, most);
  if (!aligned16(x) || !aligned16(residual) || !aligned16(y)) talos_kernel(ctx, dropout_kernel<1, 1>, grid, 256, 0, x, residual, y, (long long)n, d);
  else if (ctas <= most) talos_kernel(ctx, dropout_kernel<4, 1>, grid, 256, 0, x, residual, y, (long long)n, d);
  else talos_kernel(ctx, dropout_kernel<4, 4>, grid, 256, 0, x, residual, y, (long long)n, d);
  talos_launched(ctx, what);
}

// Gradients of no rows: sums over nothing.
void no_rows(talos_ctx* ctx, int64_t dim, float* dgamma, float* dbeta, int32_t accumulate) {
  if (dgamma && !(accumulate & 2)) TALOS_CHECK_CUDA(cudaMemsetAsync(dgamma, 0, sizeof(float) * (size_t)dim, ctx->stream));
  if (dbeta && !(accumulate & 4)) TALOS_CHECK_CUDA(cudaMemsetAsync(dbeta, 0, sizeof(float) * (size_t)dim, ctx->stream));
}

}  // namespace

TALOS_API talos_status talos_layernorm_fwd(talos_ctx* ctx, const float* x, const float* gamma, const float* beta, float eps, int64_t rows, int64_t dim,
                                           float* y, float* mean, float* inv_std) {
  TALOS_ENTRY_BEGIN
  norm_shape(rows, dim);
  TALOS_REQUIRE(eps >= 0.f, TALOS_ERR_ARG, "layer norm eps must not be negative");
  TALOS_REQUIRE(rows == 0 || (x && y), TALOS_ERR_ARG, "null pointer");
  talos_check_ctx(ctx);
  if (rows == 0) return TALOS_OK;
  norm_fwd_launch<false>(ctx, NormFwd{x, nullptr, gamma, beta, nullptr, y, mean, inv_std, eps, (long long)rows, (int)dim, DropArgs{}}, "layernorm_fwd");
  TALOS_ENTRY_END
}

TALOS_API talos_status talos_layernorm_bwd(talos_ctx* ctx, const float* dy, const float* x, const float* gamma, const float* mean, const float* inv_std,
                                           int64_t rows, int64_t dim, float* dx, float* dgamma, float* dbeta, int32_t accumulate) {
  TALOS_ENTRY_BEGIN
  norm_shape(rows, dim);
  TALOS_REQUIRE(accumulate >= 0 && accumulate < 8, TALOS_ERR_ARG, "accumulate has bits 0 to 2");
  TALOS_REQUIRE(rows == 0 || (dy && x && mean && inv_std), TALOS_ERR_ARG, "null pointer");
  talos_check_ctx(ctx);
  if (rows == 0) { no_rows(ctx, dim, dgamma, dbeta, accumulate); return TALOS_OK; }
  if (!dx && !dgamma && !dbeta) return TALOS_OK;
  norm_bwd_launch<false>(ctx, NormBwd{dy, nullptr, x, gamma, mean, inv_std, dx, nullptr, nullptr, dgamma, dbeta, (long long)rows, (int)dim, accumulate, DropArgs{}},
                         "layernorm_bwd");
  TALOS_ENTRY_END
}

TALOS_API talos_status talos_dropout_fwd(talos_ctx* ctx, const float* x, const float* residual, float* y, int64_t n, float p, uint64_t seed, uint64_t offset,
                                         const uint64_t* offset_dev) {
  TALOS_ENTRY_BEGIN
  TALOS_REQUIRE(n >= 0, TALOS_ERR_SHAPE, "negative length");
  const DropArgs d = talos_drop_args(p, seed, offset, offset_dev);
  TALOS_REQUIRE(n == 0 || (x && y), TALOS_ERR_ARG, "null pointer");
  talos_check_ctx(ctx);
  if (n == 0) return TALOS_OK;
  dropout_launch(ctx, x, residual, y, n, d, "dropout_fwd");
  TALOS_ENTRY_END
}

TALOS_API talos_status talos_dropout_bwd(talos_ctx* ctx, const float* dy, float* dx, int64_t n, float p, uint64_t seed, uint64_t offset,
                                         const uint64_t* offset_dev, int32_t accumulate) {
  TALOS_ENTRY_BEGIN
  TALOS_REQUIRE(n >= 0, TALOS_ERR_SHAPE, "negative length");
  TALOS_REQUIRE(accumulate == 0 || accumulate == 1, TALOS_ERR_ARG, "accumulate is 0 or 1");
  const DropArgs d = talos_drop_args(p, seed, offset, offset_dev);
  TALOS_REQUIRE(n == 0 || (dy && dx), TALOS_ERR_ARG, "null pointer");
  talos_check_ctx(ctx);
  if (n == 0) return TALOS_OK;
  dropout_launch(ctx, dy, accumulate ? dx : nullptr, dx, n, d, "dropout_bwd");
  TALOS_ENTRY_END
}

TALOS_API talos_status talos_dropout_add_layernorm_fwd(talos_ctx* ctx, const float* x, const float* residual, const float* gamma, const float* beta, float eps,
                                                       float p, uint64_t seed, uint64_t offset, const uint64_t* offset_dev, int64_t rows, int64_t dim, float* h,
                                                       float* y, float* mean, float* inv_std) {
  TALOS_ENTRY_BEGIN
  norm_shape(rows, dim);
  TALOS_REQUIRE(eps >= 0.f, TALOS_ERR_ARG, "layer norm eps must not be negative");
  const DropArgs d = talos_drop_args(p, seed, offset, offset_dev);
  TALOS_REQUIRE(rows == 0 || (x && h && y), TALOS_ERR_ARG, "null pointer");
  TALOS_REQUIRE(rows == 0 || h != y, TALOS_ERR_ARG, "h and y are two results");
  talos_check_ctx(ctx);
  if (rows == 0) return TALOS_OK;
  norm_fwd_launch<true>(ctx, NormFwd{x, residual, gamma, beta, h, y, mean, inv_std, eps, (long long)rows, (int)dim, d}, "dropout_add_layernorm_fwd");
  TALOS_ENTRY_END
}

TALOS_API talos_status talos_dropout_add_layernorm_bwd(talos_ctx* ctx, const float* dy, const float* dh, const float* h, const float* gamma, const float* mean,
                                                       const float* inv_std, float p, uint64_t seed, uint64_t offset, const uint64_t* offset_dev, int64_t rows,
                                                       int64_t dim, float* dx, float* dresidual, float* dgamma, float* dbeta, int32_t accumulate) {
  TALOS_ENTRY_BEGIN
  norm_shape(rows, dim);
  TALOS_REQUIRE(accumulate >= 0 && accumulate < 16, TALOS_ERR_ARG, "accumulate has bits 0 to 3");
  const DropArgs d = talos_drop_args(p, seed, offset, offset_dev);
  TALOS_REQUIRE(rows == 0 || (dy && h && mean && inv_std), TALOS_ERR_ARG, "null pointer");
  TALOS_REQUIRE(!dx || dx != dresidual, TALOS_ERR_ARG, "dx and dresidual are two results");
  talos_check_ctx(ctx);
  if (rows == 0) { no_rows(ctx, dim, dgamma, dbeta, accumulate); return TALOS_OK; }
  if (!dx && !dresidual && !dgamma && !dbeta) return TALOS_OK;
  norm_bwd_launch<true>(ctx, NormBwd{dy, dh, h, gamma, mean, inv_std, dx, dresidual, nullptr, dgamma, dbeta, (long long)rows, (int)dim, accumulate, d},
                        "dropout_add_layernorm_bwd");
  TALOS_ENTRY_END
}
