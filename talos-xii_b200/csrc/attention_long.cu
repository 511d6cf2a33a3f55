// Attention over long sequences: the entry points, the kernels of the CUDA cores (forward with a running maximum and sum, backward from the saved
// log-sum-exp; up to 64 queries and keys, and every size where the tensor cores are switched off), and the decode step (few queries, many keys)
// split over the keys.  Larger products: attention_long_tc.cu.
//
// Mathematics.  Scores are kept in base 2: t = scale * log2(e) * q.k, p = 2^(t - m) with the running maximum m of a row; when m grows, sum and
// output are multiplied by 2^(m_old - m_new).  Backward: p = 2^(t - lse log2 e), dp = dout.v, ds = p (dp - delta) scale with
// delta = sum dout out; dv += p' dout, dk += ds' q, dq += ds k.  dk and dv have one owner per key block, which walks over the queries of
// every head that shares it; dq has one owner per query block and computes p and dp once more: no atomics, the same bits every time.
// Bound: fp32 FFMA and the shared-memory reads that feed it (12 128-bit reads for 128 FFMA of a thread); a row of 64 keeps 66 TFLOP/s
// at most.  Tiles: 128 or 64 queries by 64 keys, 256 threads in 16 x 16, rows padded by four values so that 8 rows lie in 8 bank groups.
// Measured: 512 heads of 64 x 64, widths 32, forward 18 us, backward 57.
#include <cooperative_groups.h>
#include <math.h>

#include <type_traits>

#include "attention_long.cuh"

namespace {

namespace cg = cooperative_groups;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int BK = 64;                                     // keys of a tile

__device__ __forceinline__ float4 ld4(const float* p) { return *(const float4*)p; }

// Copies `rows` rows of `width` values (row stride `stride`) into sh [R][W + 4]; zeros behind the width and behind the rows.
template <int R, int W, bool VEC> __device__ __forceinline__ void fetch(float* sh, const float* src, long long stride, int rows, int width) {
  if constexpr (VEC) {
    for (int e = threadIdx.x; e < R * (W / 4); e += 256) {
      const int r = e / (W / 4), c = e % (W / 4) * 4;
      *(float4*)(sh + r * (W + 4) + c) = r < rows && c < width ? ld4(src + r * stride + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  } else {
    for (int e = threadIdx.x; e < R * W; e += 256) {
      const int r = e / W, c = e % W;
      sh[r * (W + 4) + c] = r < rows && c < width ? src[r * stride + c] : 0.f;
    }
  }
}

// acc[i][j] += sum_c a[(ra + 16 i)][c] b[(rb + 16 j)][c]: rows against rows.
template <int TM, int TN, int W> __device__ __forceinline__ void rows_rows(float (&acc)[TM][TN], const float* a, int ra, const float* b, int rb) {
#pragma unroll 4
  for (int c = 0; c < W; c += 4) {
    float4 x[TM], y[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) x[i] = ld4(a + (ra + 16 * i) * (W + 4) + c);
#pragma unroll
    for (int j = 0; j < TN; ++j) y[j] = ld4(b + (rb + 16 * j) * (W + 4) + c);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = fmaf(x[i].w, y[j].w, fmaf(x[i].z, y[j].z, fmaf(x[i].y, y[j].y, fmaf(x[i].x, y[j].x, acc[i][j]))));
  }
}
// acc[i][4 v + w] += sum_k p[(r + 16 i)][k] b[k][64 v + 4 l + w] (or, W = 32, columns 2 l + w): probabilities against rows.
template <int TM, int NC, int W> __device__ __forceinline__ void probs_rows(float (&acc)[TM][NC], const float* p, int r, const float* b, int l) {
#pragma unroll 2
  for (int k = 0; k < BK; k += 4) {
    float4 x[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) x[i] = ld4(p + (r + 16 * i) * (BK + 4) + k);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      float y[NC];
#pragma unroll
      for (int j = 0; j < NC; ++j) y[j] = 0.f;
      if constexpr (NC == 2) { const float2 q = *(const float2*)(b + (k + kk) * (W + 4) + l * 2); y[0] = q.x; y[1] = q.y; }
      else {
#pragma unroll
        for (int j = 0; j < NC; j += 4) { const float4 q = ld4(b + (k + kk) * (W + 4) + j * 16 + l * 4); y[j] = q.x; y[j + 1] = q.y; y[j + 2] = q.z; y[j + 3] = q.w; }
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const float f = kk == 0 ? x[i].x : kk == 1 ? x[i].y : kk == 2 ? x[i].z : x[i].w;
#pragma unroll
        for (int j = 0; j < NC; ++j) acc[i][j] = fmaf(f, y[j], acc[i][j]);
      }
    }
  }
}
// acc[i][..] += sum_q p[q][r + 16 i] b[q][columns of l], q < 64: the transposed probabilities against rows.
template <int TM, int NC, int W> __device__ __forceinline__ void columns_rows(float (&acc)[TM][NC], const float* p, int r, const float* b, int l) {
#pragma unroll 4
  for (int q = 0; q < 64; ++q) {
    float x[TM], y[NC];
#pragma unroll
    for (int i = 0; i < TM; ++i) x[i] = p[q * (BK + 4) + r + 16 * i];
    if constexpr (NC == 2) { const float2 v = *(const float2*)(b + q * (W + 4) + l * 2); y[0] = v.x; y[1] = v.y; }
    else {
#pragma unroll
      for (int j = 0; j < NC; j += 4) { const float4 v = ld4(b + q * (W + 4) + j * 16 + l * 4); y[j] = v.x; y[j + 1] = v.y; y[j + 2] = v.z; y[j + 3] = v.w; }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < NC; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
  }
}
// Column of a thread's value j among W columns.
template <int W> __device__ __forceinline__ int column(int l, int j) { return W == 32 ? l * 2 + j : j / 4 * 64 + l * 4 + j % 4; }

__device__ __forceinline__ float over16(float v, bool max) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) { const float u = __shfl_xor_sync(0xffffffffu, v, o); v = max ? fmaxf(v, u) : v + u; }
  return v;
}

struct FwdArgs { AttnShape s; const float *q, *k, *v; float *out, *lse; };

template <int DQ, int DV, int BQ, bool VEC>
__global__ void __launch_bounds__(256) attn_fwd_kernel(FwdArgs p) {
  talos_pdl(p.q, p.k, p.v, p.out, p.lse, p.s.key_len);
  extern __shared__ float sh[];
  float *shq = sh, *shk = shq + BQ * (DQ + 4), *shv = shk + BK * (DQ + 4), *shp = shv + BK * (DV + 4);
  constexpr int TM = BQ / 16, NC = DV / 16;
  const AttnShape& s = p.s;
  const int tiles = (s.sq + BQ - 1) / BQ;
  const int i0 = (tiles - 1 - (int)(blockIdx.x % tiles)) * BQ, h = blockIdx.x / tiles % s.heads, b = blockIdx.x / tiles / s.heads;      // causal: the longest rows first
  const int l = threadIdx.x % 16, r = threadIdx.x / 16;
  const int rows = min(BQ, s.sq - i0), keys = attn_keys(s, b), limit = attn_limit(s, keys, i0 + rows - 1);
  const float* kp = p.k + b * s.k_batch + (h / s.group) * s.k_head;
  const float* vp = p.v + b * s.v_batch + (h / s.group) * s.v_head;
  fetch<BQ, DQ, VEC>(shq, p.q + b * s.q_batch + h * s.q_head + i0 * s.q_row, s.q_row, rows, s.d);
  float m[TM], sum[TM], acc[TM][NC];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    m[i] = -INFINITY; sum[i] = 0.f;
#pragma unroll
    for (int j = 0; j < NC; ++j) acc[i][j] = 0.f;
  }
  const float c = s.scale * LOG2E;
  for (int k0 = 0; k0 < limit; k0 += BK) {
    __syncthreads();
    fetch<BK, DQ, VEC>(shk, kp + k0 * s.k_row, s.k_row, limit - k0, s.d);
    fetch<BK, DV, VEC>(shv, vp + k0 * s.v_row, s.v_row, limit - k0, s.dv);
    __syncthreads();
    float t[TM][4];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) t[i][j] = 0.f;
    rows_rows<TM, 4, DQ>(t, shq, r, shk, l);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int lim = attn_limit(s, keys, i0 + r + 16 * i);
      float top = m[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) { t[i][j] = k0 + l + 16 * j < lim ? t[i][j] * c : -INFINITY; top = fmaxf(top, t[i][j]); }
      top = over16(top, true);
      const float at = top == -INFINITY ? 0.f : top;
      float part = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) { t[i][j] = exp2f(t[i][j] - at); part += t[i][j]; shp[(r + 16 * i) * (BK + 4) + l + 16 * j] = t[i][j]; }
      const float f = exp2f(m[i] - at);
      sum[i] = sum[i] * f + part; m[i] = top;                             // (the lanes' sums are joined at the end)
#pragma unroll
      for (int j = 0; j < NC; ++j) acc[i][j] *= f;
    }
    __syncwarp();                                                         // a warp reads the rows of shp that it wrote
    probs_rows<TM, NC, DV>(acc, shp, r, shv, l);
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int row = r + 16 * i;
    const float total = over16(sum[i], false), inv = total > 0.f ? 1.f / total : total == 0.f ? 0.f : total;      // (a NaN stays)
    if (row >= rows) continue;
    if (p.lse && l == 0) p.lse[((long long)b * s.heads + h) * s.sq + i0 + row] = total == 0.f ? -INFINITY : (m[i] + log2f(total)) * LN2;
    float* o = p.out + b * s.o_batch + h * s.o_head + (i0 + row) * s.o_row;
#pragma unroll
    for (int j = 0; j < NC; ++j) { const int col = column<DV>(l, j); if (col < s.dv) o[col] = acc[i][j] * inv; }
  }
}

// ---- backward ----------------------------------------------------------------------------------------------------------------------------
// One warp a row.
__global__ void __launch_bounds__(256) attn_delta_kernel(AttnShape s, const float* out, const float* dout, float* delta) {
  talos_pdl(out, dout, delta);
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), rows = (long long)s.batch * s.heads * s.sq;
  if (row >= rows) return;
  const int i = (int)(row % s.sq), h = (int)(row / s.sq % s.heads), b = (int)(row / s.sq / s.heads);
  const long long at = b * s.o_batch + h * s.o_head + i * s.o_row;
  float a = 0.f;
  for (int c = threadIdx.x & 31; c < s.dv; c += 32) a = fmaf(out[at + c], dout[at + c], a);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if ((threadIdx.x & 31) == 0) delta[row] = a;
}

struct BwdArgs { AttnShape s; const float *q, *k, *v, *dout, *lse, *delta; float *dq, *dk, *dv; };

// p and ds of a 64 x 64 tile from the rows in shared memory; shp / shs [query][key].  lo: first query, k0: first key.
template <int DQ, int DV> __device__ __forceinline__ void probs_and_grads(const BwdArgs& a, const float* shq, const float* shk, const float* shv, const float* shd, float* shp, float* shs,
                                                                          const float* lse, const float* delta, int i0, int rows, int k0, int keys, int r, int l) {
  float t[4][4], g[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) t[i][j] = g[i][j] = 0.f;
  rows_rows<4, 4, DQ>(t, shq, r, shk, l);
  rows_rows<4, 4, DV>(g, shd, r, shv, l);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = r + 16 * i, lim = row < rows ? attn_limit(a.s, keys, i0 + row) : 0;
    const float ls = row < rows ? lse[row] * LOG2E : 0.f, dl = row < rows ? delta[row] : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool sees = k0 + l + 16 * j < lim;
      const float pr = sees ? exp2f(t[i][j] * (a.s.scale * LOG2E) - ls) : 0.f;
      if (shp) shp[row * (BK + 4) + l + 16 * j] = pr;
      shs[row * (BK + 4) + l + 16 * j] = sees ? pr * (g[i][j] - dl) * a.s.scale : 0.f;
    }
  }
}

template <int DQ, int DV, bool VEC>
__global__ void __launch_bounds__(256) attn_bwd_kv_kernel(BwdArgs p) {
  talos_pdl(p.q, p.k, p.v, p.dout, p.lse, p.delta, p.dk, p.dv, p.s.key_len);
  extern __shared__ float sh[];
  float *shk = sh, *shv = shk + BK * (DQ + 4), *shq = shv + BK * (DV + 4), *shd = shq + 64 * (DQ + 4), *shp = shd + 64 * (DV + 4), *shs = shp + 64 * (BK + 4);
  constexpr int NQ = DQ / 16, NV = DV / 16;
  const AttnShape& s = p.s;
  const int tiles = (s.sk + BK - 1) / BK;
  const int k0 = (int)(blockIdx.x % tiles) * BK, hk = blockIdx.x / tiles % s.kv_heads, b = blockIdx.x / tiles / s.kv_heads;      // causal: the first keys have the most queries
  const int l = threadIdx.x % 16, r = threadIdx.x / 16, keys = attn_keys(s, b), n = min(BK, s.sk - k0);
  float dk[4][NQ], dv[4][NV];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < NQ; ++j) dk[i][j] = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) dv[i][j] = 0.f;
  }
  if (k0 < keys) {
    fetch<BK, DQ, VEC>(shk, p.k + b * s.k_batch + hk * s.k_head + k0 * s.k_row, s.k_row, keys - k0, s.d);
    fetch<BK, DV, VEC>(shv, p.v + b * s.v_batch + hk * s.v_head + k0 * s.v_row, s.v_row, keys - k0, s.dv);
    const int first = s.causal ? max(0, k0 - attn_shift(s, keys)) / 64 * 64 : 0;      // the first query that sees key k0
    for (int g = 0; g < s.group; ++g) {
      const int h = hk * s.group + g;
      for (int i0 = first; i0 < s.sq; i0 += 64) {
        const int rows = min(64, s.sq - i0);
        __syncthreads();
        fetch<64, DQ, VEC>(shq, p.q + b * s.q_batch + h * s.q_head + i0 * s.q_row, s.q_row, rows, s.d);
        fetch<64, DV, VEC>(shd, p.dout + b * s.o_batch + h * s.o_head + i0 * s.o_row, s.o_row, rows, s.dv);
        __syncthreads();
        const long long at = ((long long)b * s.heads + h) * s.sq + i0;
        probs_and_grads<DQ, DV>(p, shq, shk, shv, shd, shp, shs, p.lse + at, p.delta + at, i0, rows, k0, keys, r, l);
        __syncthreads();
        columns_rows<4, NV, DV>(dv, shp, r, shd, l);
        columns_rows<4, NQ, DQ>(dk, shs, r, shq, l);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = r + 16 * i;
    if (row >= n) continue;
    float* ok = p.dk + b * s.k_batch + hk * s.k_head + (k0 + row) * s.k_row;
    float* ov = p.dv + b * s.v_batch + hk * s.v_head + (k0 + row) * s.v_row;
#pragma unroll
    for (int j = 0; j < NQ; ++j) { const int col = column<DQ>(l, j); if (col < s.d) ok[col] = dk[i][j]; }
#pragma unroll
    for (int j = 0; j < NV; ++j) { const int col = column<DV>(l, j); if (col < s.dv) ov[col] = dv[i][j]; }
  }
}

template <int DQ, int DV, bool VEC>
__global__ void __launch_bounds__(256) attn_bwd_q_kernel(BwdArgs p) {
  talos_pdl(p.q, p.k, p.v, p.dout, p.lse, p.delta, p.dq, p.s.key_len);
  extern __shared__ float sh[];
  float *shq = sh, *shd = shq + 64 * (DQ + 4), *shk = shd + 64 * (DV + 4), *shv = shk + BK * (DQ + 4), *shs = shv + BK * (DV + 4);
  constexpr int NQ = DQ / 16;
  const AttnShape& s = p.s;
  const int tiles = (s.sq + 63) / 64;
  const int i0 = (tiles - 1 - (int)(blockIdx.x % tiles)) * 64, h = blockIdx.x / tiles % s.heads, b = blockIdx.x / tiles / s.heads;
  const int l = threadIdx.x % 16, r = threadIdx.x / 16, rows = min(64, s.sq - i0), keys = attn_keys(s, b), limit = attn_limit(s, keys, i0 + rows - 1);
  fetch<64, DQ, VEC>(shq, p.q + b * s.q_batch + h * s.q_head + i0 * s.q_row, s.q_row, rows, s.d);
  fetch<64, DV, VEC>(shd, p.dout + b * s.o_batch + h * s.o_head + i0 * s.o_row, s.o_row, rows, s.dv);
  const long long at = ((long long)b * s.heads + h) * s.sq + i0;
  float dq[4][NQ];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NQ; ++j) dq[i][j] = 0.f;
  for (int k0 = 0; k0 < limit; k0 += BK) {
    __syncthreads();
    fetch<BK, DQ, VEC>(shk, p.k + b * s.k_batch + (h / s.group) * s.k_head + k0 * s.k_row, s.k_row, limit - k0, s.d);
    fetch<BK, DV, VEC>(shv, p.v + b * s.v_batch + (h / s.group) * s.v_head + k0 * s.v_row, s.v_row, limit - k0, s.dv);
    __syncthreads();
    probs_and_grads<DQ, DV>(p, shq, shk, shv, shd, nullptr, shs, p.lse + at, p.delta + at, i0, rows, k0, keys, r, l);
    __syncwarp();
    probs_rows<4, NQ, DQ>(dq, shs, r, shk, l);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = r + 16 * i;
    if (row >= rows) continue;
    float* o = p.dq + b * s.q_batch + h * s.q_head + (i0 + row) * s.q_row;
#pragma unroll
    for (int j = 0; j < NQ; ++j) { const int col = column<DQ>(l, j); if (col < s.d) o[col] = dq[i][j]; }
  }
}

// ---- the decode step -----------------------------------------------------------------------------------------------------------------------
// The queries of all heads that share a key head, R a CTA, against one of `splits` parts of the keys.  A warp takes 32 / R keys at a time: D / 8
// lanes hold a key's row, eight values each, and multiply it with their columns of the R queries; a scatter-reduction over those lanes (each round
// halves the values a lane keeps: D / 8 - 1 shuffles) leaves one score a lane, row lane % R.  The maximum of a row is joined over the lanes
// that hold it, only when it grows; the probabilities go through 128 bytes of shared memory to the lanes that hold the values' rows.  Nothing is shared
// between the warps before the end of the part: no barrier in the loop.  The rows arrive by asynchronous copies in a ring that each lane fills and
// reads for itself, 8 KB a warp.  Up to eight parts are one cluster and join through distributed shared memory, more leave (m, sum) and
// the unnormalised output a row to attn_decode_join_kernel.
// Bound: HBM, the keys and values read once (by as many CTAs as there are groups of R rows, the later ones from L2), and close below it the
// instructions, about ten a score with packed FMA.  Measured, 4 queries a key head: 134 MB in 29 us (4.7 TB/s, 8 us of it start and join), 537 MB
// in 86 us (6.2 TB/s); 1 query: 537 MB in 77 us.
struct DecodeArgs { AttnShape s; const float *q, *k, *v; float *out, *lse, *part, *part_ms; int splits, chunks; };

struct Eight { ulonglong2 a, b; };                         // eight fp32 values as packed pairs: columns c .. c + 3 and c + W / 2 .. c + W / 2 + 3
__device__ __forceinline__ unsigned long long pack2(float x, float y) { unsigned long long r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y)); return r; }
__device__ __forceinline__ float2 unpack2(unsigned long long v) { float2 f; asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v)); return f; }
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) { unsigned long long r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ float dot8(const Eight& x, const Eight& y) {
  const float2 f = unpack2(fma2(x.b.y, y.b.y, fma2(x.b.x, y.b.x, fma2(x.a.y, y.a.y, mul2(x.a.x, y.a.x)))));
  return f.x + f.y;
}
// This lane's eight values of a row; zeros behind its width (VEC: 16-byte aligned rows whose width is a multiple of four).
template <int W, bool VEC> __device__ __forceinline__ Eight row8(const float* p, int c, int width) {
  Eight e;
  auto four = [&](int at) {
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (VEC) { if (at < width) f = __ldcs((const float4*)(p + at)); }
    else { if (at < width) f.x = p[at]; if (at + 1 < width) f.y = p[at + 1]; if (at + 2 < width) f.z = p[at + 2]; if (at + 3 < width) f.w = p[at + 3]; }
    return ulonglong2{pack2(f.x, f.y), pack2(f.z, f.w)};
  };
  e.a = four(c); e.b = four(c + W / 2);
  return e;
}

constexpr int DECODE_WARPS = 4;

__device__ __forceinline__ void copy16(uint32_t dst, const float* src, bool there) {      // zeros where it is not
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// The ring of a warp: 16-byte pieces a lane and step, steps in flight, bytes.  Steps of many pieces are enough in flight by themselves, in registers
// (two queries a key head at width 64: 50 us that way, 58 through the ring, 268 MB).  At width 128 with four queries or more a step's 16 pieces go through the
// ring (537 MB: 85 us, 96 without).  With one or two a step has 64 or 32 pieces, more than the ring takes, and they stay in registers: two queries
// 45 us of 268 MB (6.0 TB/s); one query spills 2.7 KB a thread, 113 us of 537 MB (4.8 TB/s, where width 64 takes 78).
template <int D, int DV, int R, bool VEC> struct Ring {
  static constexpr int PIECES = (D + DV) / 4 / R, STAGES = PIECES <= 4 ? 16 / PIECES : 2;
  static constexpr bool USED = VEC && PIECES <= (D > 64 ? 16 : 8);
  static constexpr int BYTES = USED ? STAGES * PIECES * 512 : 0;
};

template <int D, int DV, int R, bool VEC>
__global__ void __launch_bounds__(DECODE_WARPS * 32, R >= 4 && D <= 64 ? 3 : 1) attn_decode_kernel(DecodeArgs p) {
  extern __shared__ uint8_t ring[];
  using Rg = Ring<D, DV, R, VEC>;
  talos_pdl(p.q, p.k, p.v, p.out, p.lse, p.part, p.part_ms, p.s.key_len);
  constexpr int LK = D / 8, GK = 32 / LK, NK = LK / R, LV = DV / 8, GV = 32 / LV, NV = LV / R, STEP = 32 / R, HOP = DECODE_WARPS * STEP;
  static_assert(NK >= 1 && NV >= 1, "a lane holds at least one key and one value row of a step");
  __shared__ float sh_m[DECODE_WARPS][R], sh_s[DECODE_WARPS][R];
  __shared__ alignas(16) float sh_p[DECODE_WARPS][2][32];
  __shared__ float part_o[R * DV], part_m[R], part_l[R];   // this part's rows, for its cluster
  __shared__ float sh_o[DECODE_WARPS][R][DV];
  const AttnShape& s = p.s;
  const int split = blockIdx.x % p.splits, chunk = blockIdx.x / p.splits % p.chunks, hk = blockIdx.x / p.chunks / p.splits % s.kv_heads, b = blockIdx.x / p.chunks / p.splits / s.kv_heads;
  const int total = s.group * s.sq, r0 = chunk * R, rows = min(R, total - r0);      // row = (head of the group) * sq + query
  const int keys = attn_keys(s, b), per = ((keys + p.splits - 1) / p.splits + STEP - 1) / STEP * STEP, from = min(keys, split * per), to = min(keys, from + per);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gk = lane / LK, ck = lane % LK * 4, gv = lane / LV, cv = lane % LV * 4, mine = lane % R;      // (mine: the row whose scores this lane holds)
  const int score_key = lane % LK / R * GK + gk;           // the key of the step whose score this lane ends up with
  int k0 = from + warp * STEP;
  const float* kl = p.k + b * s.k_batch + hk * s.k_head + (k0 + gk) * s.k_row;
  const float* vl = p.v + b * s.v_batch + hk * s.v_head + (k0 + gv) * s.v_row;
  const long long krow = GK * s.k_row, vrow = GV * s.v_row, kstep = HOP * s.k_row, vstep = HOP * s.v_row;
  const Eight zero{{0ull, 0ull}, {0ull, 0ull}};
  struct Rows { Eight k[NK], v[NV]; };
  auto fetch_step = [&](Rows& x, int at) {                 // whole steps go without a bound a row
    if (at + STEP <= to) {
#pragma unroll
      for (int i = 0; i < NK; ++i) x.k[i] = row8<D, VEC>(kl + i * krow, ck, s.d);
#pragma unroll
      for (int i = 0; i < NV; ++i) x.v[i] = row8<DV, VEC>(vl + i * vrow, cv, s.dv);
    } else {
#pragma unroll
      for (int i = 0; i < NK; ++i) x.k[i] = at + i * GK + gk < to ? row8<D, VEC>(kl + i * krow, ck, s.d) : zero;
#pragma unroll
      for (int i = 0; i < NV; ++i) x.v[i] = at + i * GV + gv < to ? row8<DV, VEC>(vl + i * vrow, cv, s.dv) : zero;
    }
    kl += kstep; vl += vstep;
  };
  // the ring: each lane fills and reads its own pieces
  const uint32_t mine_at = Rg::USED ? (uint32_t)__cvta_generic_to_shared(ring + warp * Rg::BYTES + lane * 16) : 0u;
  int next = k0, fill = 0;
  auto request = [&] {
    if (next < to) {
      const uint32_t dst = mine_at + fill * (Rg::PIECES * 512);
      auto piece = [&](int at, const float* row, int c, int width, bool there) {
        there = there && c < width;
        copy16(dst + at * 512, there ? row + c : p.k, there);
      };
#pragma unroll
      for (int i = 0; i < NK; ++i) { const bool there = next + i * GK + gk < to; piece(2 * i, kl + i * krow, ck, s.d, there); piece(2 * i + 1, kl + i * krow, ck + D / 2, s.d, there); }
#pragma unroll
      for (int i = 0; i < NV; ++i) { const bool there = next + i * GV + gv < to; piece(2 * (NK + i), vl + i * vrow, cv, s.dv, there); piece(2 * (NK + i) + 1, vl + i * vrow, cv + DV / 2, s.dv, there); }
      kl += kstep; vl += vstep;
      fill = fill + 1 == Rg::STAGES ? 0 : fill + 1; next += HOP;
    }
    copy_commit();
  };
  Rows one;
  if constexpr (Rg::USED) {
#pragma unroll
    for (int i = 0; i < Rg::STAGES - 1; ++i) request();
  } else if (k0 < to) fetch_step(one, k0);
  Eight q[R], acc[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = r0 + r;
    q[r] = acc[r] = zero;
    if (r < rows) {
      const float c = s.scale * LOG2E;
      const unsigned long long cc = pack2(c, c);
      q[r] = row8<D, false>(p.q + b * s.q_batch + (hk * s.group + row / s.sq) * s.q_head + row % s.sq * s.q_row, ck, s.d);
      q[r].a.x = mul2(q[r].a.x, cc); q[r].a.y = mul2(q[r].a.y, cc); q[r].b.x = mul2(q[r].b.x, cc); q[r].b.y = mul2(q[r].b.y, cc);
    }
  }
  const int limit = mine < rows ? min(to, attn_limit(s, keys, (r0 + mine) % s.sq)) : 0;
  float m = -INFINITY, sum = 0.f;                          // of row `mine`, the sum over this lane's keys
  int turn = 0;
  auto work = [&](const Rows& x, int at) {
    float t[LK];
#pragma unroll
    for (int i = 0; i < NK; ++i)
#pragma unroll
      for (int r = 0; r < R; ++r) t[i * R + r] = dot8(x.k[i], q[r]);
#pragma unroll
    for (int o = LK / 2; o > 0; o >>= 1) {
      const bool up = lane & o;
#pragma unroll
      for (int i = 0; i < o; ++i) {
        const float keep = up ? t[i + o] : t[i], send = up ? t[i] : t[i + o];
        t[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
      }
    }
    const float y = at + score_key < limit ? t[0] : -INFINITY;
    if (__any_sync(0xffffffffu, y > m)) {
      float top = fmaxf(y, m);
#pragma unroll
      for (int o = 16; o >= R; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float f = top > m ? exp2f(m - top) : 1.f;      // (m = -inf: 0)
      m = top; sum *= f;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float fr = __shfl_sync(0xffffffffu, f, r);
        const unsigned long long ff = pack2(fr, fr);
        acc[r].a.x = mul2(acc[r].a.x, ff); acc[r].a.y = mul2(acc[r].a.y, ff); acc[r].b.x = mul2(acc[r].b.x, ff); acc[r].b.y = mul2(acc[r].b.y, ff);
      }
    }
    const float pr = exp2f(y - (m == -INFINITY ? 0.f : m));      // (0 for a key that is not seen; a NaN score, which never is a maximum, stays NaN)
    sum += pr;
    float* sp = sh_p[warp][turn];                          // [key][row]
    turn ^= 1;
    sp[score_key * R + mine] = pr;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float* w = sp + (i * GV + gv) * R;
      float wr[R];
      if constexpr (R >= 4) {
#pragma unroll
        for (int r = 0; r < R; r += 4) { const float4 f = *(const float4*)(w + r); wr[r] = f.x; wr[r + 1] = f.y; wr[r + 2] = f.z; wr[r + 3] = f.w; }
      } else if constexpr (R == 2) { const float2 f = *(const float2*)w; wr[0] = f.x; wr[1] = f.y; }
      else wr[0] = w[0];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const unsigned long long ww = pack2(wr[r], wr[r]);
        acc[r].a.x = fma2(ww, x.v[i].a.x, acc[r].a.x); acc[r].a.y = fma2(ww, x.v[i].a.y, acc[r].a.y);
        acc[r].b.x = fma2(ww, x.v[i].b.x, acc[r].b.x); acc[r].b.y = fma2(ww, x.v[i].b.y, acc[r].b.y);
      }
    }
  };
  if constexpr (Rg::USED) {
    int use = 0;
    for (; k0 < to; k0 += HOP) {
      request();
      copy_wait<Rg::STAGES - 1>();
      const ulonglong2* at = (const ulonglong2*)(ring + warp * Rg::BYTES + use * (Rg::PIECES * 512) + lane * 16);
#pragma unroll
      for (int i = 0; i < NK; ++i) one.k[i] = Eight{at[64 * i], at[64 * i + 32]};
#pragma unroll
      for (int i = 0; i < NV; ++i) one.v[i] = Eight{at[64 * (NK + i)], at[64 * (NK + i) + 32]};
      use = use + 1 == Rg::STAGES ? 0 : use + 1;
      work(one, k0);
    }
  } else {
    while (k0 < to) {
      work(one, k0);
      k0 += HOP;
      if (k0 < to) fetch_step(one, k0);
    }
  }
  // the lanes' sums, then the warps'
#pragma unroll
  for (int o = 16; o >= R; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float2 f[4] = {unpack2(acc[r].a.x), unpack2(acc[r].a.y), unpack2(acc[r].b.x), unpack2(acc[r].b.y)};
    float x[8] = {f[0].x, f[0].y, f[1].x, f[1].y, f[2].x, f[2].y, f[3].x, f[3].y};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int o = 16; o >= LV; o >>= 1) x[i] += __shfl_xor_sync(0xffffffffu, x[i], o);
      if (lane < LV) sh_o[warp][r][i / 4 * (DV / 2) + cv + i % 4] = x[i];
    }
  }
  if (lane < R) { sh_m[warp][lane] = m; sh_s[warp][lane] = sum; }
  __syncthreads();
  const long long at = ((long long)b * s.kv_heads + hk) * total + r0;      // first row in the joined order [batch][kv head][row]
  auto put = [&](int r, int c, float a, float l, float top) {
    const int row = r0 + r, h = hk * s.group + row / s.sq;
    if (c < s.dv) p.out[b * s.o_batch + h * s.o_head + row % s.sq * s.o_row + c] = l == 0.f ? 0.f : a / l;
    if (c == 0 && p.lse) p.lse[((long long)b * s.heads + h) * s.sq + row % s.sq] = l == 0.f ? -INFINITY : (top + log2f(l)) * LN2;
  };
  for (int e = threadIdx.x; e < rows * DV; e += DECODE_WARPS * 32) {
    const int r = e / DV, c = e % DV;
    float top = sh_m[0][r];
#pragma unroll
    for (int i = 1; i < DECODE_WARPS; ++i) top = fmaxf(top, sh_m[i][r]);
    const float ref = top == -INFINITY ? 0.f : top;
    float a = 0.f, l = 0.f;
#pragma unroll
    for (int i = 0; i < DECODE_WARPS; ++i) { const float f = exp2f(sh_m[i][r] - ref); a = fmaf(sh_o[i][r][c], f, a); l = fmaf(sh_s[i][r], f, l); }
    if (p.part) {
      p.part[((at + r) * p.splits + split) * DV + c] = a;
      if (c == 0) { float* ms = p.part_ms + ((at + r) * p.splits + split) * 2; ms[0] = top; ms[1] = l; }
    } else if (p.splits > 1) {
      part_o[e] = a;
      if (c == 0) { part_m[r] = top; part_l[r] = l; }
    } else put(r, c, a, l, top);
  }
  if (p.part || p.splits == 1) return;
  // the cluster's parts: each CTA joins its share of the rows' columns, in the order of the parts
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int e = split * DECODE_WARPS * 32 + threadIdx.x; e < rows * DV; e += p.splits * DECODE_WARPS * 32) {
    const int r = e / DV;
    float top = -INFINITY, a = 0.f, l = 0.f;
    for (int i = 0; i < p.splits; ++i) top = fmaxf(top, *cluster.map_shared_rank(part_m + r, i));
    const float ref = top == -INFINITY ? 0.f : top;
    for (int i = 0; i < p.splits; ++i) {
      const float f = exp2f(*cluster.map_shared_rank(part_m + r, i) - ref);
      a = fmaf(*cluster.map_shared_rank(part_o + e, i), f, a); l = fmaf(*cluster.map_shared_rank(part_l + r, i), f, l);
    }
    put(r, e % DV, a, l, top);
  }
  cluster.sync();                                          // nobody leaves while its part may still be read
}

// One CTA a row: the parts' outputs, weighted by 2^(m - max m).  256 / width threads share a column, each with every so many parts; their sums
// are added in order.
__global__ void __launch_bounds__(256) attn_decode_join_kernel(AttnShape s, const float* part, const float* part_ms, int splits, int width, float* out, float* lse) {
  talos_pdl(part, part_ms, out, lse);
  __shared__ float sh[256], sh_l[8];
  const int total = s.group * s.sq, c = threadIdx.x % width, g = threadIdx.x / width, groups = 256 / width;
  const long long at = blockIdx.x;
  const int row = (int)(at % total), hk = (int)(at / total % s.kv_heads), b = (int)(at / total / s.kv_heads), h = hk * s.group + row / s.sq, i = row % s.sq;
  const float2* ms = (const float2*)part_ms + at * splits;
  float m = -INFINITY;
  for (int j = threadIdx.x & 31; j < splits; j += 32) m = fmaxf(m, ms[j].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float mm = m == -INFINITY ? 0.f : m;
  float a = 0.f, l = 0.f;
#pragma unroll 4
  for (int j = g; j < splits; j += groups) {
    const float2 q = ms[j];
    const float f = exp2f(q.x - mm);
    l = fmaf(q.y, f, l); a = fmaf(part[(at * splits + j) * width + c], f, a);
  }
  sh[threadIdx.x] = a;
  if (c == 0) sh_l[g] = l;
  __syncthreads();
  if (g == 0) {
    for (int k = 1; k < groups; ++k) { a += sh[k * width + c]; l += sh_l[k]; }      // (l: the same for every column)
    if (lse && c == 0) lse[((long long)b * s.heads + h) * s.sq + i] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
    if (c < s.dv) out[b * s.o_batch + h * s.o_head + i * s.o_row + c] = l == 0.f ? 0.f : a / l;
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------------------
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

AttnShape attn_shape(int64_t batch, int64_t heads, int64_t kv_heads, int64_t sq, int64_t sk, int64_t d, int64_t dv, float scale, int causal, int layout, int mode, const int* key_len) {
  TALOS_REQUIRE(batch >= 0 && sq >= 0 && sk >= 0 && heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0, TALOS_ERR_SHAPE, "kv_heads must divide heads, sizes must not be negative");
  TALOS_REQUIRE(d >= 1 && dv >= 1 && d <= 128 && dv <= 128, TALOS_ERR_SHAPE, "attention supports head widths of 1 to 128");
  TALOS_REQUIRE(sq <= (1 << 24) && sk <= (1 << 24) && batch <= (1 << 20) && heads <= (1 << 16) && batch * heads * (sq / 64 + 1) < (1ll << 31) &&
                    batch * kv_heads * (sk / 64 + 1) < (1ll << 31), TALOS_ERR_SHAPE, "attention problem too large for one launch");
  TALOS_REQUIRE(layout == TALOS_ATTN_BHSD || layout == TALOS_ATTN_BSHD, TALOS_ERR_ARG, "bad layout");
  TALOS_REQUIRE(mode >= TALOS_MODE_FP32 && mode <= TALOS_MODE_TF32, TALOS_ERR_ARG, "bad mode");
  TALOS_REQUIRE(scale == scale && (causal == 0 || causal == TALOS_ATTN_CAUSAL || causal == TALOS_ATTN_CAUSAL_NEWEST), TALOS_ERR_ARG, "bad scale or causal value");
  AttnShape s{};
  s.key_len = key_len; s.batch = (int)batch; s.heads = (int)heads; s.kv_heads = (int)kv_heads; s.group = (int)(heads / kv_heads);
  s.sq = (int)sq; s.sk = (int)sk; s.d = (int)d; s.dv = (int)dv; s.scale = scale; s.causal = causal;
  const bool bshd = layout == TALOS_ATTN_BSHD;
  auto place = [&](int64_t h, int64_t n, int64_t w, long long& row, long long& head, long long& bat) { row = bshd ? h * w : w; head = bshd ? w : n * w; bat = h * n * w; };
  place(heads, sq, d, s.q_row, s.q_head, s.q_batch); place(kv_heads, sk, d, s.k_row, s.k_head, s.k_batch);
  place(kv_heads, sk, dv, s.v_row, s.v_head, s.v_batch); place(heads, sq, dv, s.o_row, s.o_head, s.o_batch);
  return s;
}

// f(DQ, DV, VEC) for the tile widths that hold d and dv.
template <typename F> void by_widths(const AttnShape& s, bool vec, F&& f) {
#define TALOS_W(DQ, DV) return vec ? f(std::integral_constant<int, DQ>(), std::integral_constant<int, DV>(), std::true_type()) : f(std::integral_constant<int, DQ>(), std::integral_constant<int, DV>(), std::false_type())
  if (s.d <= 32 && s.dv <= 32) TALOS_W(32, 32);
  if (s.d <= 64 && s.dv <= 64) TALOS_W(64, 64);
  if (s.dv <= 64) TALOS_W(128, 64);
  TALOS_W(128, 128);
#undef TALOS_W
}

template <typename K, typename A> void launch(talos_ctx* ctx, K kern, std::atomic<uint64_t>& done, int64_t grid, size_t shmem, const A& args) {
  talos_allow_smem(done, (const void*)kern, shmem, ctx->device);
  talos_kernel(ctx, kern, (unsigned)grid, 256, shmem, args);
}

void decode(talos_ctx* ctx, const AttnShape& s, const float* q, const float* k, const float* v, float* out, float* lse, bool vec) {
  by_widths(s, vec, [&](auto dq, auto dv, auto ve) {
    constexpr int DQ = decltype(dq)::value, DV = decltype(dv)::value; constexpr bool VEC = decltype(ve)::value;
    auto go = [&](auto rc) {
      constexpr int R = decltype(rc)::value;
      DecodeArgs a{s, q, k, v, out, lse, nullptr, nullptr, 1, (int)ceil_div(s.group * s.sq, R)};
      const int64_t ctas = (int64_t)s.batch * s.kv_heads * a.chunks, rows = (int64_t)s.batch * s.heads * s.sq;
      // parts: as many CTAs as are resident at once, of at least two steps a warp each; one cluster where eight will nearly do
      constexpr size_t shmem = (size_t)DECODE_WARPS * Ring<DQ, DV, R, VEC>::BYTES;
      static std::atomic<uint64_t> done{0};
      if (shmem) talos_allow_smem(done, (const void*)attn_decode_kernel<DQ, DV, R, VEC>, shmem, ctx->device);
      static std::atomic<int> resident{0};
      int per_sm = resident.load(std::memory_order_relaxed);
      if (per_sm == 0) {
        TALOS_CHECK_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, attn_decode_kernel<DQ, DV, R, VEC>, DECODE_WARPS * 32, shmem));
        resident.store(per_sm = std::max(per_sm, 1), std::memory_order_relaxed);
      }
      int64_t parts = std::max<int64_t>(1, std::min<int64_t>(per_sm * ctx->sm_count / ctas, s.sk / (2 * DECODE_WARPS * (32 / R))));
      if (parts > 8 && parts < 12) parts = 8;
      a.splits = (int)parts;
      if (parts > 8) {
        a.part = (float*)talos_workspace(ctx, sizeof(float) * (size_t)(rows * parts) * (DV + 2));
        a.part_ms = a.part + rows * parts * DV;
      }
      talos_kernel_cluster(ctx, attn_decode_kernel<DQ, DV, R, VEC>, (unsigned)(ctas * parts), DECODE_WARPS * 32, shmem, parts <= 8 ? (unsigned)parts : 1u, a);
      talos_launched(ctx, "attention_decode");
      if (parts > 8) {
        talos_kernel(ctx, attn_decode_join_kernel, (unsigned)rows, 256, 0, s, a.part, a.part_ms, a.splits, DV, out, lse);
        talos_launched(ctx, "attention_decode_join");
      }
    };
    const int total = s.group * s.sq;
    if (total <= 1) go(std::integral_constant<int, 1>());
    else if (total <= 2) go(std::integral_constant<int, 2>());
    else if (total <= 4 || DQ == 32) go(std::integral_constant<int, 4>());
    else if constexpr (DQ > 32) go(std::integral_constant<int, 8>());
  });
}

}  // namespace

TALOS_API talos_status talos_attention_lse_fwd(talos_ctx* ctx, const float* q, const float* k, const float* v, const int32_t* key_len, float* out, float* lse, int64_t batch,
                                               int64_t heads, int64_t kv_heads, int64_t sq, int64_t sk, int64_t d, int64_t dv, float scale, int32_t causal, int32_t layout, int32_t mode) {
  TALOS_ENTRY_BEGIN
  const AttnShape s = attn_shape(batch, heads, kv_heads, sq, sk, d, dv, scale, causal, layout, mode, key_len);
  const bool none = batch == 0 || sq == 0;
  TALOS_REQUIRE(none || (q && out && (sk == 0 || (k && v))), TALOS_ERR_ARG, "null pointer");
  talos_check_ctx(ctx);
  if (none) return TALOS_OK;
  const bool vec = d % 4 == 0 && dv % 4 == 0 && aligned16(q) && aligned16(k) && aligned16(v);
  // Few queries: one CTA reads a key head's rows for all of them.
  if (sq <= 8 && sk > 0) { decode(ctx, s, q, k, v, out, lse, vec); return TALOS_OK; }
  if (talos_attn_tc_fwd(ctx, s, q, k, v, out, lse, mode)) return TALOS_OK;
  by_widths(s, vec, [&](auto wq, auto wv, auto ve) {
    constexpr int DQ = decltype(wq)::value, DV = decltype(wv)::value; constexpr bool VEC = decltype(ve)::value;
    auto go = [&](auto bq) {
      constexpr int BQ = decltype(bq)::value;
      static std::atomic<uint64_t> done{0};
      const size_t shmem = sizeof(float) * (size_t)(BQ * (DQ + 4) + BK * (DQ + 4) + BK * (DV + 4) + BQ * (BK + 4));
      launch(ctx, attn_fwd_kernel<DQ, DV, BQ, VEC>, done, ceil_div(sq, BQ) * heads * batch, shmem, FwdArgs{s, q, k, v, out, lse});
    };
    if (DQ <= 64 && sq > 64) go(std::integral_constant<int, 128>()); else go(std::integral_constant<int, 64>());
  });
  talos_launched(ctx, "attention_lse_fwd");
  TALOS_ENTRY_END
}

TALOS_API talos_status talos_attention_lse_bwd(talos_ctx* ctx, const float* q, const float* k, const float* v, const int32_t* key_len, const float* out, const float* lse,
                                               const float* dout, float* dq, float* dk, float* dv_out, int64_t batch, int64_t heads, int64_t kv_heads, int64_t sq, int64_t sk,
                                               int64_t d, int64_t dv, float scale, int32_t causal, int32_t layout, int32_t mode) {
  TALOS_ENTRY_BEGIN
  const AttnShape s = attn_shape(batch, heads, kv_heads, sq, sk, d, dv, scale, causal, layout, mode, key_len);
  const bool no_q = batch == 0 || sq == 0, no_k = batch == 0 || sk == 0;
  TALOS_REQUIRE(no_q || (q && out && lse && dout && dq), TALOS_ERR_ARG, "null pointer");
  TALOS_REQUIRE(no_k || (k && v && dk && dv_out), TALOS_ERR_ARG, "null pointer");
  talos_check_ctx(ctx);
  if (no_q || no_k) {                                       // nothing saw anything: zeros
    if (!no_q) TALOS_CHECK_CUDA(cudaMemsetAsync(dq, 0, sizeof(float) * (size_t)(batch * heads * sq * d), ctx->stream));
    if (!no_k) TALOS_CHECK_CUDA(cudaMemsetAsync(dk, 0, sizeof(float) * (size_t)(batch * kv_heads * sk * d), ctx->stream));
    if (!no_k) TALOS_CHECK_CUDA(cudaMemsetAsync(dv_out, 0, sizeof(float) * (size_t)(batch * kv_heads * sk * dv), ctx->stream));
    return TALOS_OK;
  }
  if (talos_attn_tc_bwd(ctx, s, q, k, v, out, lse, dout, dq, dk, dv_out, mode)) return TALOS_OK;
  float* delta = (float*)talos_workspace(ctx, sizeof(float) * (size_t)(batch * heads * sq));
  talos_kernel(ctx, attn_delta_kernel, (unsigned)ceil_div(batch * heads * sq, 8), 256, 0, s, out, dout, delta);
  talos_launched(ctx, "attention_delta");
  const bool vec = d % 4 == 0 && dv % 4 == 0 && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(dout);
  const BwdArgs a{s, q, k, v, dout, lse, delta, dq, dk, dv_out};
  by_widths(s, vec, [&](auto wq, auto wv, auto ve) {
    constexpr int DQ = decltype(wq)::value, DV = decltype(wv)::value; constexpr bool VEC = decltype(ve)::value;
    static std::atomic<uint64_t> done_kv{0}, done_q{0};
    const size_t rows = sizeof(float) * 64 * (size_t)(2 * (DQ + 4) + 2 * (DV + 4)), tile = sizeof(float) * 64 * (BK + 4);
    launch(ctx, attn_bwd_kv_kernel<DQ, DV, VEC>, done_kv, ceil_div(sk, BK) * kv_heads * batch, rows + 2 * tile, a);
    talos_launched(ctx, "attention_lse_bwd_kv");
    launch(ctx, attn_bwd_q_kernel<DQ, DV, VEC>, done_q, ceil_div(sq, 64) * heads * batch, rows + tile, a);
  });
  talos_launched(ctx, "attention_lse_bwd_q");
  TALOS_ENTRY_END
}
