// Layer norm, dropout, and their junction in a transformer block (h = residual + dropout(x), y = layer norm of h), forward and
// backward: one pass over the rows each way, the row in registers between the statistics and the result.
//
// Mathematics.  mean and the centred sum of squares are taken from the registers one after the other (two reductions, no
// E[x^2] - E[x]^2).  Backward, with g = dy * gamma and xh = (x - mean) * inv: dx = inv * (g - mean(g) - xh * mean(g * xh)); both
// means travel in one reduction.  The gradients of gamma and beta are column sums: every thread keeps its columns' sums over all the
// rows of its CTA, a CTA leaves one partial row of each, and a second small kernel adds the partial rows in order.
// Bound: HBM.  Layer norm moves 8 bytes an element forward and 12 backward, the junction 16 and 20.
// Split: a group of G threads owns a row, G = 8 to 32 lanes of a warp (dim <= 512) or a CTA of 128 to 1 024 threads, so that a thread
// holds at most 16 values of a row: enough loads in flight, no spills beside the column sums.
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
// Dropout factors of the W elements from `i` (i % 4 == 0 where W is 4).
template <int W> __device__ __forceinline__ Vec<W> drop(const DropArgs& d, unsigned long long offset, long long i) {
  Vec<W> v;
  if constexpr (W == 4) { const float4 f = talos_drop4(d, offset, (unsigned long long)i >> 2); v.a[0] = f.x; v.a[1] = f.y; v.a[2] = f.z; v.a[3] = f.w; }
  else v.a[0] = talos_drop1(d, offset, (unsigned long long)i);
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

struct NormFwd {
  const float *x, *residual, *gamma, *beta; float *h, *y, *mean, *inv;
  float eps; long long rows; int dim; DropArgs drop;
};

template <int W, int G, int NV, bool FUSED>
__global__ void __launch_bounds__(block_of<G>) norm_fwd_kernel(NormFwd p) {
  talos_pdl(p.x, p.residual, p.gamma, p.beta, p.h, p.y, p.mean, p.inv, p.drop.offset_dev);
  __shared__ float2 sh[2][32];
  int phase = 0;
  const int l = G <= 32 ? threadIdx.x % G : threadIdx.x, sub = G <= 32 ? threadIdx.x / G : 0;
  const int units = p.dim / W;
  const float inv_dim = 1.f / (float)p.dim;
  const unsigned long long offset = FUSED ? run_offset(p.drop) : 0;
  constexpr bool HOIST = NV * W <= 16;                   // gamma and beta stay in registers over the rows
  Vec<W> gam[HOIST ? NV : 1], bet[HOIST ? NV : 1];
  if constexpr (HOIST) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = l + v * G;
      gam[v] = fill<W>(1.f); bet[v] = fill<W>(0.f);
#pragma unroll
      for (int i = 0; i < W; ++i) if (c < units) { if (p.gamma) gam[v].a[i] = p.gamma[c * W + i]; if (p.beta) bet[v].a[i] = p.beta[c * W + i]; }
    }
  }
  for (long long r0 = (long long)blockIdx.x * rows_per_block<G>; r0 < p.rows; r0 += (long long)gridDim.x * rows_per_block<G>) {
    const long long r = r0 + sub, base = r * p.dim;
    const bool ok = r < p.rows;
    Vec<W> xv[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) { const int c = l + v * G; xv[v] = ok && c < units ? ldv<W>(p.x + base + c * W) : fill<W>(0.f); }
    if constexpr (FUSED) {
      Vec<W> rv[NV];
      if (p.residual) {
#pragma unroll
        for (int v = 0; v < NV; ++v) { const int c = l + v * G; rv[v] = ok && c < units ? ldv<W>(p.residual + base + c * W) : fill<W>(0.f); }
      } else {
#pragma unroll
        for (int v = 0; v < NV; ++v) rv[v] = fill<W>(0.f);
      }
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = l + v * G;
        if (ok && c < units) {
          if (p.drop.threshold) {
            const Vec<W> f = drop<W>(p.drop, offset, base + c * W);
#pragma unroll
            for (int i = 0; i < W; ++i) xv[v].a[i] = dropped(xv[v].a[i], f.a[i]);
          }
#pragma unroll
          for (int i = 0; i < W; ++i) xv[v].a[i] += rv[v].a[i];
          stv<W>(p.h + base + c * W, xv[v]);
        }
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
      if (l + v * G < units) {
#pragma unroll
        for (int i = 0; i < W; ++i) { const float t = xv[v].a[i] - mean; q += t * t; }
      }
    const float inv = 1.f / sqrtf(group_sum<G>(q, 0.f, sh, phase).x * inv_dim + p.eps);
    if (ok && l == 0) { if (p.mean) p.mean[r] = mean; if (p.inv) p.inv[r] = inv; }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = l + v * G;
      if (ok && c < units) {
        Vec<W> o;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float gm = HOIST ? gam[HOIST ? v : 0].a[i] : p.gamma ? p.gamma[c * W + i] : 1.f, bt = HOIST ? bet[HOIST ? v : 0].a[i] : p.beta ? p.beta[c * W + i] : 0.f;
          o.a[i] = (xv[v].a[i] - mean) * inv * gm + bt;
        }
        stv<W>(p.y + base + c * W, o);
      }
    }
  }
}

struct NormBwd {
  const float *dy, *dh, *x, *gamma, *mean, *inv; float *dx, *dresidual, *partial, *dgamma, *dbeta;
  long long rows; int dim; int accumulate; DropArgs drop;
};

// partial[CTA][2][dim]: this CTA's sums of dy * xh and of dy; a launch of one CTA writes dgamma and dbeta itself.
template <int W, int G, int NV, bool FUSED, bool ACC_SMEM>
__global__ void __launch_bounds__(block_of<G>) norm_bwd_kernel(NormBwd p) {
  talos_pdl(p.dy, p.dh, p.x, p.gamma, p.mean, p.inv, p.dx, p.dresidual, p.partial, p.dgamma, p.dbeta, p.drop.offset_dev);
  extern __shared__ float cols[];                       // G <= 32: [groups][2][dim] at the end; ACC_SMEM: [2][dim], each thread its own columns
  __shared__ float2 sh[2][32];
  int phase = 0;
  const int l = G <= 32 ? threadIdx.x % G : threadIdx.x, sub = G <= 32 ? threadIdx.x / G : 0;
  const int units = p.dim / W;
  const float inv_dim = 1.f / (float)p.dim;
  const unsigned long long offset = FUSED ? run_offset(p.drop) : 0;
  constexpr bool HOIST = NV * W <= 16;
  Vec<W> gam[HOIST ? NV : 1], dg[ACC_SMEM ? 1 : NV], db[ACC_SMEM ? 1 : NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = l + v * G;
    if constexpr (HOIST) {
      gam[v] = fill<W>(1.f);
#pragma unroll
      for (int i = 0; i < W; ++i) if (c < units && p.gamma) gam[v].a[i] = p.gamma[c * W + i];
    }
    if constexpr (!ACC_SMEM) { dg[v] = fill<W>(0.f); db[v] = fill<W>(0.f); }
    else if (c < units) {
#pragma unroll
      for (int i = 0; i < W; ++i) { cols[c * W + i] = 0.f; cols[p.dim + c * W + i] = 0.f; }
    }
  }
  for (long long r0 = (long long)blockIdx.x * rows_per_block<G>; r0 < p.rows; r0 += (long long)gridDim.x * rows_per_block<G>) {
    const long long r = r0 + sub, base = r * p.dim;
    const bool ok = r < p.rows;
    Vec<W> gv[NV], xv[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = l + v * G; const bool in = ok && c < units;
      gv[v] = in ? ldv<W>(p.dy + base + c * W) : fill<W>(0.f);
      xv[v] = in ? ldv<W>(p.x + base + c * W) : fill<W>(0.f);
    }
    const float mean = ok ? p.mean[r] : 0.f, inv = ok ? p.inv[r] : 0.f;
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = l + v * G;
      if (c < units) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float gm = HOIST ? gam[HOIST ? v : 0].a[i] : p.gamma ? p.gamma[c * W + i] : 1.f;
          const float d = gv[v].a[i], xh = (xv[v].a[i] - mean) * inv;
          if constexpr (ACC_SMEM) { cols[c * W + i] += d * xh; cols[p.dim + c * W + i] += d; }
          else { dg[v].a[i] += d * xh; db[v].a[i] += d; }
          xv[v].a[i] = xh; gv[v].a[i] = d * gm;
          s1 += gv[v].a[i]; s2 += gv[v].a[i] * xh;
        }
      }
    }
    if (!p.dx && !p.dresidual) continue;                  // (the same for all threads)
    const float2 s = group_sum<G>(s1, s2, sh, phase);
    const float m1 = s.x * inv_dim, m2 = s.y * inv_dim;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = l + v * G;
      if (!(ok && c < units)) continue;
      Vec<W> o;
#pragma unroll
      for (int i = 0; i < W; ++i) o.a[i] = inv * (gv[v].a[i] - m1 - xv[v].a[i] * m2);
      if constexpr (FUSED) {
        if (p.dh) {
          const Vec<W> e = ldv<W>(p.dh + base + c * W);
#pragma unroll
          for (int i = 0; i < W; ++i) o.a[i] += e.a[i];
        }
        Vec<W> t = o;
        if (p.dx && p.drop.threshold) {
          const Vec<W> f = drop<W>(p.drop, offset, base + c * W);
#pragma unroll
          for (int i = 0; i < W; ++i) t.a[i] = dropped(t.a[i], f.a[i]);
        }
        if (p.dresidual) {
          if (p.accumulate & 8) {
            const Vec<W> old = ldv<W>(p.dresidual + base + c * W);
#pragma unroll
            for (int i = 0; i < W; ++i) o.a[i] += old.a[i];
          }
          stv<W>(p.dresidual + base + c * W, o);
        }
        o = t;
      }
      if (p.dx) {
        if (p.accumulate & 1) {
          const Vec<W> old = ldv<W>(p.dx + base + c * W);
#pragma unroll
          for (int i = 0; i < W; ++i) o.a[i] += old.a[i];
        }
        stv<W>(p.dx + base + c * W, o);
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
      float* mine = p.partial + (size_t)blockIdx.x * 2 * p.dim;
      mine[c] = a; mine[p.dim + c] = b;
    }
  };
  if constexpr (G <= 32) {
    float* mine = cols + (size_t)sub * 2 * p.dim;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = l + v * G;
#pragma unroll
      for (int i = 0; i < W; ++i) if (c < units) { mine[c * W + i] = dg[v].a[i]; mine[p.dim + c * W + i] = db[v].a[i]; }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.dim; c += blockDim.x) {
      float a = 0.f, b = 0.f;
      for (int i = 0; i < rows_per_block<G>; ++i) { a += cols[(size_t)i * 2 * p.dim + c]; b += cols[(size_t)i * 2 * p.dim + p.dim + c]; }
      put(c, a, b);
    }
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = l + v * G;
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (c < units) { if constexpr (ACC_SMEM) put(c * W + i, cols[c * W + i], cols[p.dim + c * W + i]); else put(c * W + i, dg[v].a[i], db[v].a[i]); }
    }
  }
}

// dgamma and dbeta from the CTAs' partial rows: 32 columns of [dgamma | dbeta] a CTA, eight lanes down the parts, added in a fixed order.
__global__ void __launch_bounds__(256)
norm_param_grads_kernel(const float* partial, int nparts, int dim, float* dgamma, float* dbeta, int accumulate) {
  talos_pdl(partial, dgamma, dbeta);
  __shared__ float sh[8][33];
  const int cl = threadIdx.x & 31, pl = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;
  float s = 0.f;
  if (c < 2 * dim) {
#pragma unroll 8
    for (int i = pl; i < nparts; i += 8) s += partial[(size_t)i * 2 * dim + c];
  }
  sh[pl][cl] = s;
  __syncthreads();
  if (pl == 0 && c < 2 * dim) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += sh[i][cl];
    float* out = c < dim ? dgamma : dbeta;
    const int at = c < dim ? c : c - dim, acc = c < dim ? accumulate & 2 : accumulate & 4;
    if (out) out[at] = acc ? out[at] + t : t;
  }
}

// y = residual + dropped(x), or dx (+)= dropped(dy): four elements to a draw.  W = 1: buffers that are not 16-byte aligned.
// (Two draws a thread and step keep enough loads in flight to hide the draws' 40 products and logic operations.)
template <int W>
__global__ void __launch_bounds__(256) dropout_kernel(const float* x, const float* residual, float* y, long long n, DropArgs d) {
  talos_pdl(x, residual, y, d.offset_dev);
  const unsigned long long offset = run_offset(d);
  const long long blocks = (n + 3) / 4, step = (long long)gridDim.x * blockDim.x;
  for (long long b = (long long)blockIdx.x * blockDim.x + threadIdx.x; b < blocks; b += step) {
    const long long i = b * 4;
    float xv[4], rv[4] = {0.f, 0.f, 0.f, 0.f};
    const bool whole = W == 4 && i + 4 <= n;
    if (whole) {
      const float4 q = __ldcs((const float4*)(x + i));
      xv[0] = q.x; xv[1] = q.y; xv[2] = q.z; xv[3] = q.w;
      if (residual) { const float4 e = __ldcs((const float4*)(residual + i)); rv[0] = e.x; rv[1] = e.y; rv[2] = e.z; rv[3] = e.w; }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) { xv[j] = i + j < n ? x[i + j] : 0.f; if (residual && i + j < n) rv[j] = residual[i + j]; }
    }
    if (d.threshold) {
      const float4 f = talos_drop4(d, offset, (unsigned long long)b);
      xv[0] = dropped(xv[0], f.x); xv[1] = dropped(xv[1], f.y); xv[2] = dropped(xv[2], f.z); xv[3] = dropped(xv[3], f.w);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) xv[j] += rv[j];
    if (whole) __stcs((float4*)(y + i), make_float4(xv[0], xv[1], xv[2], xv[3]));
    else {
#pragma unroll
      for (int j = 0; j < 4; ++j) if (i + j < n) y[i + j] = xv[j];
    }
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// One launch by row width: f is called with the constants (W, G, NV).
template <typename F> void by_width(bool vec, int dim, F&& f) {
#define TALOS_N(W_, G_, NV_) return f(std::integral_constant<int, W_>(), std::integral_constant<int, G_>(), std::integral_constant<int, NV_>())
  if (vec) {
    const int u = dim / 4;
    if (u <= 8) TALOS_N(4, 8, 1);
    if (u <= 16) TALOS_N(4, 16, 1);
    if (u <= 32) TALOS_N(4, 32, 1);
    if (u <= 64) TALOS_N(4, 32, 2);
    if (u <= 128) TALOS_N(4, 32, 4);
    if (u <= 256) TALOS_N(4, 128, 2);
    if (u <= 512) TALOS_N(4, 128, 4);
    if (u <= 1024) TALOS_N(4, 256, 4);
    if (u <= 2048) TALOS_N(4, 512, 4);
    TALOS_N(4, 1024, 4);
  }
  if (dim <= 32) TALOS_N(1, 32, 1);
  if (dim <= 128) TALOS_N(1, 32, 4);
  if (dim <= 512) TALOS_N(1, 32, 16);
  if (dim <= 1024) TALOS_N(1, 128, 8);
  if (dim <= 2048) TALOS_N(1, 128, 16);
  if (dim <= 4096) TALOS_N(1, 256, 16);
  if (dim <= 8192) TALOS_N(1, 512, 16);
  TALOS_N(1, 1024, 16);
#undef TALOS_N
}

template <bool FUSED> void norm_fwd_launch(talos_ctx* ctx, const NormFwd& p, const char* what) {
  const bool vec = p.dim % 4 == 0 && aligned16(p.x) && aligned16(p.y) && (!FUSED || (aligned16(p.residual) && aligned16(p.h)));
  by_width(vec, p.dim, [&](auto w, auto g, auto nv) {
    constexpr int W = decltype(w)::value, G = decltype(g)::value, NV = decltype(nv)::value;
    const int64_t cap = (int64_t)ctx->sm_count * (2048 / block_of<G>);
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(p.rows, rows_per_block<G>), cap);
    talos_kernel(ctx, norm_fwd_kernel<W, G, NV, FUSED>, grid, block_of<G>, 0, p);
  });
  talos_launched(ctx, what);
}

template <bool FUSED> void norm_bwd_launch(talos_ctx* ctx, NormBwd p, const char* what) {
  const bool vec = p.dim % 4 == 0 && aligned16(p.dy) && aligned16(p.x) && aligned16(p.dx) && (!FUSED || (aligned16(p.dh) && aligned16(p.dresidual)));
  const bool params = p.dgamma || p.dbeta;
  unsigned grid = 1;
  by_width(vec, p.dim, [&](auto w, auto g, auto nv) {
    constexpr int W = decltype(w)::value, G = decltype(g)::value, NV = decltype(nv)::value;
    constexpr bool ACC_SMEM = G >= 512;                  // a CTA of 512 threads has 128 registers a thread: the column sums move to shared memory
    const int64_t cap = (int64_t)ctx->sm_count * (G >= 512 ? 1 : G == 256 ? 2 : G == 128 ? 4 : 3);
    grid = (unsigned)std::min<int64_t>(ceil_div(p.rows, rows_per_block<G>), cap);
    if (params && grid > 1) p.partial = (float*)talos_workspace(ctx, sizeof(float) * 2 * (size_t)p.dim * grid);
    const size_t shmem = G <= 32 ? sizeof(float) * 2 * (size_t)p.dim * rows_per_block<G> : ACC_SMEM ? sizeof(float) * 2 * (size_t)p.dim : 0;
    static std::atomic<uint64_t> done{0};
    auto kern = norm_bwd_kernel<W, G, NV, FUSED, ACC_SMEM>;
    if (ACC_SMEM) talos_allow_smem(done, (const void*)kern, sizeof(float) * 2 * (size_t)MAX_DIM, ctx->device);
    talos_kernel(ctx, kern, grid, block_of<G>, shmem, p);
  });
  talos_launched(ctx, what);
  if (params && grid > 1) {
    talos_kernel(ctx, norm_param_grads_kernel, (unsigned)ceil_div(2 * p.dim, 32), 256, 0, p.partial, (int)grid, p.dim, p.dgamma, p.dbeta, p.accumulate);
    talos_launched(ctx, "norm_param_grads");
  }
}

void norm_shape(int64_t rows, int64_t dim) {
  TALOS_REQUIRE(rows >= 0 && dim > 0 && dim <= MAX_DIM, TALOS_ERR_SHAPE, "layer norm supports rows of 1 to 16384 values");
  TALOS_REQUIRE(rows <= INT64_MAX / MAX_DIM / 4, TALOS_ERR_SHAPE, "too many rows");
}

void dropout_launch(talos_ctx* ctx, const float* x, const float* residual, float* y, int64_t n, const DropArgs& d, const char* what) {
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(ceil_div(n, 4), 256), (int64_t)ctx->sm_count * 8);
  if (aligned16(x) && aligned16(residual) && aligned16(y)) talos_kernel(ctx, dropout_kernel<4>, grid, 256, 0, x, residual, y, (long long)n, d);
  else talos_kernel(ctx, dropout_kernel<1>, grid, 256, 0, x, residual, y, (long long)n, d);
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
