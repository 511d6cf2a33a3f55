// Attention over long sequences on the tensor cores (tcgen05), fp32-faithful: forward and backward, head widths up to 64 and (at the end) to 128.
//
// Mathematics.  An fp32 value is the sum of three bf16 terms x = x0 + x1 + x2 (8 bits each, rounded to nearest).  A product keeps the six
// of the nine term products that reach 2^-24: (2,0) (0,2) (1,1) (1,0) (0,1) (0,0), added in this order into one fp32 accumulator in tensor
// memory: the tensor core truncates when it adds, so the small ones come first and only the last one meets the full magnitude.  The
// fast mode keeps the last three (two terms, 2^-16).  Softmax and gradients as in attention_long.cu: base 2, q scaled by scale * log2(e) before it is
// split.  No accumulator lives longer than one block: its sums are added in registers, in fp32, rounded to nearest.
//
// A first kernel (attn_split_kernel) splits q, k, v and dout once, into tiles of [term][128 rows][64 values] that already have the
// 128-byte swizzle of the matrix descriptors, zeros behind a sequence's rows, so that every operand arrives by plain bulk copies.
//
// Bound: the tensor pipe, at the clock that the power limit leaves.  An MMA of 128 x N x 16 takes N / 2 cycles with A in tensor memory and
// max(N / 2, 32 + N / 4) with A in shared memory (its port; measured 48 at N = 64, 64 at N = 128), provided that one elected thread issues them back to
// back from descriptors in registers (issued one by one from a thread picked by its index they take 97, whatever N).  Cycles a 128 x 128 tile
// at width 64: forward 48 x 64, dk / dv 2 x (20 x 32 + 28 x 48 + 48 x 32), dq 2 x 72 x 32.
// Measured, 32 causal heads of 2 048 x 2 048, width 64 (29.4 tiles an SM; 1.75 GHz at 1 000 W): forward 96 us of 52 possible at that clock, dk / dv 172 of
// 118, dq 123 of 77; the split 24 us of q, k, v (5.2 TB/s, reads and writes), 29 with dout (5.8).  What is between: 4 us a CTA before its first scores and
// behind its last block, and 15 to 25 % in the loops, waits of the issuing warps that the queue of the tensor pipe is too short to cover.
//
// Roles of a CTA: warp 0 copies, warp 1 owns tensor memory and issues (in backward one more warp issues the products with the weights), sixteen warps work
// on the scores: four threads a row, a quarter of the columns each.  Every wait is bounded (mbar_wait); on expiry the CTA raises the error word
// and leaves.
#include <limits.h>
#include <math.h>

#include "attention_long.cuh"
#include "tc_common.cuh"

bool talos_tc_ready_for(talos_ctx* ctx);

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int WORKERS = 16, THREADS = (2 + WORKERS) * 32, TILE = 128 * 128;      // bytes of one term of 128 rows
// The term products in order: (2,0) (0,2) (1,1) (1,0) (0,1) (0,0).
__host__ __device__ constexpr int term_a(int i) { return i == 0 ? 2 : i == 2 || i == 3 ? 1 : 0; }
__host__ __device__ constexpr int term_b(int i) { return i == 1 ? 2 : i == 2 || i == 4 ? 1 : 0; }

// ---- the split ------------------------------------------------------------------------------------------------------------------------
// x [batch][heads][rows][width] at the given strides -> tiles [batch * heads][ceil(rows / 128)][chunks of 64 values][3][128 rows][64], the 16 bytes c of
// row r at c ^ (r % 8).
struct SplitJob { const float* x; uint8_t* tiles; long long row, head, bat; int heads, rows, width, keys, chunks; float factor; int first; };      // first: its first CTA
struct SplitArgs { SplitJob job[4]; int jobs, ctas; const int* key_len; };

// A CTA: 32 rows of one head, 64 values wide; a thread: 8 values of a row.
template <int TERMS> __global__ void __launch_bounds__(256) attn_split_kernel(SplitArgs a) {
  talos_pdl(a.job[0].x, a.job[1].x, a.job[2].x, a.job[3].x, a.key_len);      // (x: read by streaming loads)
  int j = 0;
#pragma unroll
  for (int i = 1; i < 4; ++i) if (i < a.jobs && (int)blockIdx.x >= a.job[i].first) j = i;
  const SplitJob q = j == 0 ? a.job[0] : j == 1 ? a.job[1] : j == 2 ? a.job[2] : a.job[3];
  const int per = (q.rows + 127) / 128 * 4, v = (int)blockIdx.x - q.first, chunk = v % q.chunks, u = v / q.chunks, bh = u / per, b = bh / q.heads, h = bh % q.heads;
  const int r = (u % per) * 32 + (threadIdx.x >> 3), c = threadIdx.x & 7, col = chunk * 64 + c * 8;
  const int rows = q.keys && a.key_len ? min(max(a.key_len[b], 0), q.rows) : q.rows;
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = 0.f;
  if (r < rows) {
    const float* src = q.x + b * q.bat + h * q.head + r * q.row + col;
    if (col + 8 <= q.width && ((uintptr_t)src & 15) == 0) {
      const float4 lo = __ldcs((const float4*)src), hi = __ldcs((const float4*)(src + 4));
      x[0] = lo.x; x[1] = lo.y; x[2] = lo.z; x[3] = lo.w; x[4] = hi.x; x[5] = hi.y; x[6] = hi.z; x[7] = hi.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) if (col + i < q.width) x[i] = src[i];
    }
  }
  uint8_t* tile = q.tiles + (((long long)bh * (per / 4) + r / 128) * q.chunks + chunk) * (3 * TILE) + (r % 128) * 128 + ((c ^ (r & 7)) << 4);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= q.factor;
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
      x[2 * i] -= __uint_as_float(w[i] << 16); x[2 * i + 1] -= __uint_as_float(w[i] & 0xffff0000u);
    }
    *(uint4*)(tile + t * TILE) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// (lse * log2 e, delta) a query, padded to 128 rows a head; +inf where a row is not there or sees no key: its probabilities are 0.
__global__ void __launch_bounds__(256) attn_rows_kernel(AttnShape s, const float* out, const float* dout, const float* lse, float2* rows) {
  talos_pdl(out, dout, lse, rows);
  const unsigned per_head = (unsigned)(s.sq + 127) / 128 * 2, bh = blockIdx.x / per_head;      // CTAs of 64 rows: 16 lanes four rows
  const int i0 = (int)(blockIdx.x % per_head) * 64 + (threadIdx.x >> 4), l = threadIdx.x & 15;
  const long long at = (bh / s.heads) * s.o_batch + (bh % s.heads) * s.o_head;
  const bool vec = (((uintptr_t)out | (uintptr_t)dout) & 15) == 0 && s.dv % 4 == 0;
  float d[4], ls[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) { d[j] = 0.f; ls[j] = i0 + j * 16 < s.sq ? lse[(long long)bh * s.sq + i0 + j * 16] : -INFINITY; }
  if (vec) {
    for (int c = l * 4; c < s.dv; c += 64) {
      float4 x[4], y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long o = at + (i0 + j * 16) * s.o_row + c;
        const bool in = i0 + j * 16 < s.sq;
        x[j] = in ? *(const float4*)(out + o) : make_float4(0.f, 0.f, 0.f, 0.f);
        y[j] = in ? *(const float4*)(dout + o) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) { d[j] = fmaf(x[j].x, y[j].x, d[j]); d[j] = fmaf(x[j].y, y[j].y, d[j]); d[j] = fmaf(x[j].z, y[j].z, d[j]); d[j] = fmaf(x[j].w, y[j].w, d[j]); }
    }
  } else {
    for (int c = l; c < s.dv; c += 16)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long o = at + (i0 + j * 16) * s.o_row + c;
        if (i0 + j * 16 < s.sq) d[j] = fmaf(out[o], dout[o], d[j]);
      }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) d[j] += __shfl_xor_sync(0xffffffffu, d[j], o);
    if (l == 0) rows[(long long)blockIdx.x * 64 + (threadIdx.x >> 4) + j * 16] = make_float2(ls[j] == -INFINITY ? INFINITY : ls[j] * LOG2E, d[j]);
  }
}

// ---- device pieces ------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.b32 %0, 1, 0, P;\n\t}" : "=r"(p));
  return p;
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
// bf16 operands, fp32 accumulator, M = 128; b_mn: B's rows run along the reduction.
__host__ __device__ constexpr uint32_t idesc_of(uint32_t n, uint32_t b_mn) { return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn << 16) | ((n >> 3) << 17) | (8u << 24); }
// A tile of 64 values a row: along the row (32 bytes a step of 16 values), or along the rows (2 048 bytes a step of 16 rows).
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr) { return make_desc(addr, 16, 1024, 2); }

// D = A . B over the term products: A rows of 128 in shared memory at terms TILE bytes apart, B rows at b_term bytes; both along their rows.
template <int PRODUCTS, int KD> __device__ __forceinline__ void issue_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t b_term, uint32_t idesc) {
#pragma unroll
  for (int i = 6 - PRODUCTS; i < 6; ++i)
#pragma unroll
    for (int k = 0; k < KD; ++k)
      mma_ss(d, a + (uint64_t)(term_a(i) * (TILE >> 4) + k * 2), b + (uint64_t)(term_b(i) * (b_term >> 4) + k * 2), idesc, (i > 6 - PRODUCTS || k > 0) ? 1u : 0u);
}
// A in tensor memory, terms a_term columns apart, 8 columns a step; B along its rows (MN false) or across them (MN true).
template <int PRODUCTS, int STEPS, bool MN> __device__ __forceinline__ void issue_ts(uint32_t d, uint32_t a, uint32_t a_term, uint64_t b, uint32_t b_term, uint32_t idesc) {
#pragma unroll
  for (int i = 6 - PRODUCTS; i < 6; ++i)
#pragma unroll
    for (int k = 0; k < STEPS; ++k)
      mma_ts(d, a + term_a(i) * a_term + k * 8, b + (uint64_t)(term_b(i) * (b_term >> 4) + k * (MN ? 128 : 2)), idesc, (i > 6 - PRODUCTS || k > 0) ? 1u : 0u);
}

__device__ __forceinline__ float exp2_fast(float x) { float e; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x)); return e; }
// The next term of a pair of values: packed bf16, and what it leaves.
__device__ __forceinline__ uint32_t take_term(float& lo, float& hi) {
  uint32_t w;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
  lo -= __uint_as_float(w << 16); hi -= __uint_as_float(w & 0xffff0000u);
  return w;
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// Stores N values of this thread's row as terms: N / 2 columns each, `term` columns apart.
template <int TERMS, int N> __device__ __forceinline__ void store_terms(uint32_t taddr, uint32_t term, float (&x)[N]) {
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = take_term(x[2 * i], x[2 * i + 1]);
    if constexpr (N == 32) tmem_st16(taddr + t * term, w); else tmem_st8(taddr + t * term, w);
  }
}
template <int N> __device__ __forceinline__ void load_values(uint32_t taddr, float (&x)[N]) {
  uint32_t r[N];
  if constexpr (N == 32) tmem_ld32(taddr, r); else tmem_ld16(taddr, r);
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = __uint_as_float(r[i]);
}
// For whole warps.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)); }
// The four threads of each of 32 rows.  Every warp comes here as often, also after a wait that gave up.
__device__ __forceinline__ void row_barrier(int quad) { asm volatile("bar.sync %0, 128;" ::"r"(quad + 1) : "memory"); }
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) { tc_fence_before(); __syncwarp(); if (lane == 0) mbar_arrive(bar); }

__device__ __forceinline__ void store_columns(float* d, const float4& v, int left) {
  if (left >= 4 && ((uintptr_t)d & 15) == 0) { *(float4*)d = v; return; }
  if (left > 0) d[0] = v.x;
  if (left > 1) d[1] = v.y;
  if (left > 2) d[2] = v.z;
  if (left > 3) d[3] = v.w;
}
// Writes W / 4 values of each thread's row, through shared memory: a warp's stores are whole rows (a row a lane they take 32 cycles each).  stage: 128 rows
// of W + 4 values; rows_left, o: of this quad's 32 rows.
template <int W> __device__ __forceinline__ void write_rows(float* stage, const float* x, int quad, int part, int lane, int rows_left, float* o, long long stride, int width) {
  stage += quad * 32 * (W + 4);
#pragma unroll
  for (int i = 0; i < W / 4; i += 4) *(float4*)(stage + lane * (W + 4) + part * (W / 4) + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
  row_barrier(quad);
  constexpr int LANES = W / 4, ROWS = 32 / LANES;
  const int c = lane % LANES * 4;
#pragma unroll
  for (int i = 0; i < 8; i += ROWS) {
    const int r = part * 8 + i + lane / LANES;
    if (r >= rows_left) continue;
    const float4 v = *(const float4*)(stage + r * (W + 4) + c);
    float* d = o + r * stride + c;
    store_columns(d, v, width - c);
  }
}

// Results whose blocks are shared out to the CTAs of a cluster (SHARED): each leaves its 128 rows of W values in shared memory (W + 4 apart), then each adds
// its share of the rows over the cluster, in the order of the ranks; in forward weighted by 2^(its maximum - the largest).
__device__ __forceinline__ void cluster_barrier() { asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ uint32_t peer_address(uint32_t own, int rank) { uint32_t a; asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(own), "r"(rank)); return a; }
__device__ __forceinline__ float4 peer_float4(uint32_t own, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(peer_address(own, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float2 peer_float2(uint32_t own, int rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(peer_address(own, rank)) : "memory");
  return v;
}
template <int W> __device__ __forceinline__ void stage_row(float* stage, const float* x, int row, int part) {
#pragma unroll
  for (int i = 0; i < W / 4; i += 4) *(float4*)(stage + row * (W + 4) + part * (W / 4) + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
}
template <int W> __device__ __forceinline__ void write_sums(const float* stage, int parts, int rank, int worker, int lane, int rows, float* o, long long stride, int width) {
  constexpr int LANES = W / 4, ROWS = 32 / LANES;
  const uint32_t own = smem_u32(stage);
  for (int k = rank + parts * worker; k < 128 / ROWS; k += parts * WORKERS) {
    const int r = ROWS * k + lane / LANES, c = lane % LANES * 4;
    if (r >= rows) continue;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int from = 0; from < parts; ++from) {
      const float4 v = peer_float4(own + (uint32_t)(r * (W + 4) + c) * 4, from);
      a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
    }
    store_columns(o + r * stride + c, a, width - c);
  }
}
// ms: (maximum, sum) of each row; lse nullable.
template <int W>
__device__ __forceinline__ void write_weighted(const float* stage, const float2* ms, int parts, int rank, int worker, int lane, int rows, float* o, long long stride, int width, float* lse) {
  constexpr int LANES = W / 4, ROWS = 32 / LANES;
  const uint32_t own = smem_u32(stage), own_ms = smem_u32(ms);
  for (int k = rank + parts * worker; k < 128 / ROWS; k += parts * WORKERS) {
    const int r = ROWS * k + lane / LANES, c = lane % LANES * 4;
    if (r >= rows) continue;
    float top = -INFINITY;
    for (int from = 0; from < parts; ++from) top = fmaxf(top, peer_float2(own_ms + r * 8, from).x);
    const float at = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int from = 0; from < parts; ++from) {
      const float2 q = peer_float2(own_ms + r * 8, from);
      const float4 v = peer_float4(own + (uint32_t)(r * (W + 4) + c) * 4, from);
      const float f = exp2_fast(q.x - at);
      sum = fmaf(q.y, f, sum);
      a.x = fmaf(v.x, f, a.x); a.y = fmaf(v.y, f, a.y); a.z = fmaf(v.z, f, a.z); a.w = fmaf(v.w, f, a.w);
    }
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
    if (lse && c == 0) lse[r] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * LN2;
    store_columns(o + r * stride + c, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv), width - c);
  }
}

struct TcAttn {
  AttnShape s; int parts;                                  // (parts: CTAs that share a tile's blocks)
  const uint8_t *q, *k, *v, *o;                           // split tiles of q, k, v, dout
  const float2* rows;
  float *out, *lse, *dq, *dk, *dv;
  int32_t* status; unsigned wait_spins; int skip;           // (skip: test hook, a load that the first CTA leaves out; -1: none)
};
__device__ __forceinline__ bool left_out(const TcAttn& p, int load) { return load == p.skip && blockIdx.x == 0; }

// Common start and end of the three kernels.
#define TC_SETUP(BARRIERS_INIT)                                                                                  \
  extern __shared__ uint8_t smem_raw[];                                                                          \
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);                                   \
  __shared__ uint64_t bars[24];                                                                                  \
  __shared__ uint32_t columns;                                                                                   \
  __shared__ int abort_words[2];                                                                                 \
  volatile int* abort_flag = abort_words;                                                                        \
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;                                                    \
  if (threadIdx.x == 0) { BARRIERS_INIT; abort_flag[0] = 0; abort_flag[1] = (int)p.wait_spins; fence_barrier_init(); } \
  if (warp == 1) { tmem_alloc(&columns, 512); tmem_relinquish(); }                                               \
  tc_fence_before(); __syncthreads(); tc_fence_after();                                                          \
  talos_pdl();                                            /* this CTA holds its tensor memory */                 \
  const uint32_t tmem = __shfl_sync(0xffffffffu, columns, 0);                                                    \
  const AttnShape& s = p.s;
__device__ __forceinline__ void tc_leave(volatile int* abort_flag, int32_t* status, int warp, uint32_t tmem) {
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) atomicExch(status, TALOS_DEV_TIMEOUT_BASE + 900 + (int)(blockIdx.x % 100));
    for (int i = 0; i < 64; ++i) __nanosleep(1000);       // copies in flight land before shared memory is given back
    __syncthreads();
  }
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem, 512); }
}

// This thread's quarter of its row's first N terms of an A operand, from a split tile in shared memory to tensor memory.  (Read from global memory, a
// row a lane, it took 3 us of a CTA's 7 beside its blocks.)
template <int N> struct RowTerms {
  uint4 w[N][2];
  __device__ __forceinline__ RowTerms(const uint8_t* tile, int row, int part) {
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) w[t][i] = *(const uint4*)(tile + t * TILE + row * 128 + (((part * 2 + i) ^ (row & 7)) << 4));
  }
  __device__ __forceinline__ void store(uint32_t taddr, int part) const {
#pragma unroll
    for (int t = 0; t < N; ++t) {
      const uint32_t r[8] = {w[t][0].x, w[t][0].y, w[t][0].z, w[t][0].w, w[t][1].x, w[t][1].y, w[t][1].z, w[t][1].w};
      tmem_st8(taddr + t * 32 + part * 8, r);
    }
  }
};

// The three kernels of widths up to 64 share one order of work.  The scores' columns are free once the workers have them in registers, so that the scores of
// block n + 1 are computed beside the work on block n; the weights have columns of their own, which the workers write when the products of block n - 1
// are done, beside the scores of block n + 1.  (Weights written over the scores in two buffers in turn, the scores of block n + 2 behind the products of
// block n, and the rows' operand in shared memory, whose port it filled: dk / dv 207 us, dq 147.)  In backward two warps issue, so
// that one's waits lie beside the other's products (dk / dv 186 to 180 us, dq 137 to 129); in forward one warp keeps the order, since
// the probabilities wait for the products before them: scores in between delay those (108 us with two, 102 with one).

// ---- forward ------------------------------------------------------------------------------------------------------------------------------
// 128 queries, blocks of 128 keys.  Shared memory: a ring of four 48 KB slots that k and v tiles pass through in the order in which they are used: k0 k1 v0
// k2 v1 ...  Tensor memory: the scores (128 columns), the probabilities (3 x 64), the block's output (64), q (3 x 32).
template <int PRODUCTS, int KD, bool SHARED>
__global__ void __launch_bounds__(THREADS, 1) attn_tc_fwd_kernel(TcAttn p) {
  constexpr int TERMS = PRODUCTS == 6 ? 3 : 2, SLOTS = 4, S_COL = 0, P_COL = 128, O_COL = 320, Q_COL = 384;
  __shared__ float sh_max[2][4][128], sh_sum[4][128];
  __shared__ float2 sh_ms[128];                            // (maximum, sum) a row of this CTA's share
  // barriers: full[4], empty[4], o_full, s_full, q_tile, then (all workers) q_full, s_empty, p_full
  TC_SETUP(for (int i = 0; i < 14; ++i) mbar_init(bars + i, i < 11 ? 1 : WORKERS))
  uint64_t *full = bars, *empty = bars + 4, *o_full = bars + 8, *s_full = bars + 9, *q_tile = bars + 10, *q_full = bars + 11, *s_empty = bars + 12, *p_full = bars + 13;
  uint8_t* sq = smem + 3 * (3 * TILE);                     // the last slot, before its first use
  const int tiles = (s.sq + 127) / 128, all = s.heads * s.batch;
  const int parts = SHARED ? p.parts : 1, unit = (int)blockIdx.x / parts, rank = (int)blockIdx.x % parts;
  const int tile = s.causal ? tiles - 1 - unit / all : unit % tiles, bh = s.causal ? unit % all : unit / tiles;      // causal: the longest first
  const int b = bh / s.heads, h = bh % s.heads, i0 = tile * 128, rows = min(128, s.sq - i0);
  const int keys = attn_keys(s, b), limit = attn_limit(s, keys, i0 + rows - 1), of_all = (limit + 127) / 128;
  const int n0 = of_all * rank / parts, blocks = of_all * (rank + 1) / parts - n0;      // this CTA's share of the blocks

  if (warp == 0) {
    if (lane == 0 && blocks > 0) {
      const int kt = (s.sk + 127) / 128;
      const long long kv = (long long)(b * s.kv_heads + h / s.group) * kt;
      mbar_expect_tx(q_tile, TERMS * TILE);
      bulk_load(sq, p.q + ((long long)bh * tiles + tile) * (3 * TILE), TERMS * TILE, q_tile);
      for (int i = 0; i < 2 * blocks; ++i) {               // use i: k0, k1, v0, k2, v1, ..., v(n-1)
        if (i == SLOTS - 1 && !mbar_wait(q_full, 0, abort_flag)) break;
        const bool is_v = i > 0 && (i == 2 * blocks - 1 || i % 2 == 0);
        const int n = i == 0 ? 0 : i == 2 * blocks - 1 ? blocks - 1 : is_v ? i / 2 - 1 : (i + 1) / 2, slot = i % SLOTS;
        if (!mbar_wait(empty + slot, ((i / SLOTS) & 1) ^ 1, abort_flag)) break;
        mbar_expect_tx(full + slot, TERMS * TILE);
        if (left_out(p, i)) continue;
        bulk_load(smem + slot * (3 * TILE), (is_v ? p.v : p.k) + (kv + n0 + n) * (3 * TILE), TERMS * TILE, full + slot);
      }
    }
  } else if (warp == 1) {
    const uint32_t ring_a = smem_u32(smem);
    const uint32_t idesc_o = idesc_of((uint32_t)((s.dv + 15) / 16 * 16), 1);
    bool ok = blocks > 0 && mbar_wait(q_full, 0, abort_flag);
    int use = 0;
    auto scores = [&](int n) {
      const int slot = use % SLOTS;
      ok = (n == 0 || mbar_wait(s_empty, (n - 1) & 1, abort_flag)) && mbar_wait(full + slot, (use / SLOTS) & 1, abort_flag);
      if (!ok) return;
      tc_fence_after();
      const uint64_t kd = tile_desc(ring_a + slot * (3 * TILE));
      if (elect_one()) {
        issue_ts<PRODUCTS, KD, false>(tmem + S_COL, tmem + Q_COL, 32, kd, TILE, idesc_of(128, 0));
        tc_commit(empty + slot); tc_commit(s_full);
      }
      __syncwarp();
      ++use;
    };
    if (ok) scores(0);
    for (int n = 0; n < blocks && ok; ++n) {
      if (n + 1 < blocks) { scores(n + 1); if (!ok) break; }
      const int slot = use % SLOTS;
      ok = mbar_wait(p_full, n & 1, abort_flag) && mbar_wait(full + slot, (use / SLOTS) & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const uint64_t vd = tile_desc(ring_a + slot * (3 * TILE));
      if (elect_one()) {
        issue_ts<PRODUCTS, 8, true>(tmem + O_COL, tmem + P_COL, 64, vd, TILE, idesc_o);
        tc_commit(empty + slot); tc_commit(o_full);
      }
      __syncwarp();
      ++use;
    }
  } else {
    const int quad = warp & 3, part = (warp - 2) >> 2, row = quad * 32 + lane;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const int lim = row < rows ? attn_limit(s, keys, i0 + row) : 0;
    float m = -INFINITY, sum = 0.f, acc[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
    bool ok = true;
    if (blocks > 0) {
      ok = warp_wait(q_tile, 0, abort_flag);
      if (ok) {
        RowTerms<TERMS>(sq, row, part).store(tmem + lanes + Q_COL, part);
        tmem_st_wait();
        warp_arrive(q_full, lane);
      }
    }
    for (int n = 0; n < blocks; ++n) {
      ok = ok && warp_wait(s_full, n & 1, abort_flag);
      if (!ok) { row_barrier(quad); continue; }
      tc_fence_after();
      float x[32];
      load_values(tmem + lanes + S_COL + part * 32, x);
      tmem_ld_wait();
      warp_arrive(s_empty, lane);
      const int see = lim - (n0 + n) * 128 - part * 32;             // columns of this part that the row sees
      if (!__all_sync(0xffffffffu, see >= 32)) {
#pragma unroll
        for (int i = 0; i < 32; ++i) if (i >= see) x[i] = -INFINITY;
      }
      float top = m;
#pragma unroll
      for (int i = 0; i < 32; ++i) top = fmaxf(top, x[i]);
      sh_max[n & 1][part][row] = top;
      row_barrier(quad);
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, sh_max[n & 1][i][row]);
      const float at = top == -INFINITY ? 0.f : top, f = exp2_fast(m - at);
      m = top;
      float even = 0.f, odd = 0.f;
#pragma unroll
      for (int i = 0; i < 32; i += 2) { x[i] = exp2_fast(x[i] - at); x[i + 1] = exp2_fast(x[i + 1] - at); even += x[i]; odd += x[i + 1]; }
      sum = sum * f + (even + odd);
      if (n > 0) {                                            // the block before: its output, and its probabilities are read
        ok = warp_wait(o_full, (n - 1) & 1, abort_flag);
        if (!ok) continue;
        tc_fence_after();
        float o[16];
        load_values(tmem + lanes + O_COL + part * 16, o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] = (acc[i] + o[i]) * f;
      }
      store_terms<TERMS>(tmem + lanes + P_COL + part * 16, 64, x);
      tmem_st_wait();
      warp_arrive(p_full, lane);
    }
    if (ok && blocks > 0) {
      ok = warp_wait(o_full, (blocks - 1) & 1, abort_flag);
      if (ok) {
        tc_fence_after();
        float o[16];
        load_values(tmem + lanes + O_COL + part * 16, o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] += o[i];
      }
    }
    sh_sum[part][row] = sum;
    row_barrier(quad);
    const float total = (sh_sum[0][row] + sh_sum[1][row]) + (sh_sum[2][row] + sh_sum[3][row]);
    if constexpr (!SHARED) {
      const float inv = total > 0.f ? 1.f / total : total == 0.f ? 0.f : total;
      if (ok && p.lse && part == 0 && row < rows) p.lse[(long long)bh * s.sq + i0 + row] = total == 0.f ? -INFINITY : (m + log2f(total)) * LN2;
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[i] *= inv;
      write_rows<64>((float*)smem, acc, quad, part, lane, ok ? rows - quad * 32 : 0, p.out + b * s.o_batch + h * s.o_head + (i0 + quad * 32) * s.o_row, s.o_row, s.dv);
    } else {
      stage_row<64>((float*)smem, acc, row, part);
      if (part == 0) sh_ms[row] = make_float2(m, total);
    }
  }
  if constexpr (SHARED) {
    cluster_barrier();
    if (warp >= 2)
      write_weighted<64>((float*)smem, sh_ms, parts, rank, warp - 2, lane, rows, p.out + b * s.o_batch + h * s.o_head + i0 * s.o_row, s.o_row, s.dv,
                         p.lse ? p.lse + (long long)bh * s.sq + i0 : nullptr);
    cluster_barrier();                                         // nobody leaves while its rows may still be read
  }
  tc_leave(abort_flag, p.status, warp, tmem);
}

// ---- backward: keys and values ----------------------------------------------------------------------------------------------------------------
// 128 keys, one a lane; blocks of 64 queries of every head that shares them.  Shared memory: k's third term, v, a ring of six 24 KB slots for q0 dout0 q1
// dout1 ..., and beside each q its rows' (lse, delta).  Tensor memory: [scores 64 | dp 64], the probabilities and ds (3 x 32 each), the block's dv and dk
// (64 each), and in the 64 columns that are left k's other two terms.
template <int PRODUCTS, int KD, bool SHARED>
__global__ void __launch_bounds__(THREADS + 32, 1) attn_tc_bwd_kv_kernel(TcAttn p) {
  constexpr int TERMS = PRODUCTS == 6 ? 3 : 2, HALF = TILE / 2, SLOT = 3 * HALF, SLOTS = 6, P_COL = 128, DS_COL = 224, DV_COL = 320, DK_COL = 384, K_COL = 448;
  __shared__ float4 sh_rows[SLOTS / 2][32];
  // barriers: kv_full, full[6], empty[6], sd_full, done, k_tile, then (all workers) k_full, sd_empty, pd_full
  TC_SETUP(for (int i = 0; i < 19; ++i) mbar_init(bars + i, i < 16 ? 1 : WORKERS))
  uint64_t *kv_full = bars, *full = bars + 1, *empty = bars + 7, *sd_full = bars + 13, *done = bars + 14, *k_tile = bars + 15, *k_full = bars + 16, *sd_empty = bars + 17, *pd_full = bars + 18;
  const int tiles = (s.sk + 127) / 128, all = s.kv_heads * s.batch;
  const int parts = SHARED ? p.parts : 1, unit = (int)blockIdx.x / parts, rank = (int)blockIdx.x % parts;
  const int tile = s.causal ? unit / all : unit % tiles, bh = s.causal ? unit % all : unit / tiles;      // causal: the first keys have the most queries
  const int b = bh / s.kv_heads, hk = bh % s.kv_heads, k0 = tile * 128, keys = attn_keys(s, b), offset = attn_shift(s, keys), q_tiles = (s.sq + 127) / 128;
  const int first = s.causal ? max(0, k0 - offset) / 64 : 0, per_head = k0 < keys ? max(0, (s.sq + 63) / 64 - first) : 0;
  const int n0 = per_head * s.group * rank / parts, blocks = per_head * s.group * (rank + 1) / parts - n0;      // this CTA's share of the blocks
  uint8_t *sk = smem, *sv = smem + TILE, *ring = smem + 4 * TILE, *sk01 = ring + 4 * SLOT;      // (the last: in two slots before their first use)

  if (warp == 0) {
    if (lane == 0 && blocks > 0) {
      const uint8_t* gk = p.k + ((long long)bh * tiles + tile) * (3 * TILE);
      mbar_expect_tx(k_tile, 2 * TILE);
      bulk_load(sk01, gk, 2 * TILE, k_tile);
      mbar_expect_tx(kv_full, (TERMS == 3 ? TILE : 0) + TERMS * TILE);
      if (TERMS == 3) bulk_load(sk, gk + 2 * TILE, TILE, kv_full);
      bulk_load(sv, p.v + ((long long)bh * tiles + tile) * (3 * TILE), TERMS * TILE, kv_full);
      for (int i = 0; i < 2 * blocks; ++i) {
        if (i == 4 && !mbar_wait(k_full, 0, abort_flag)) break;
        const int n = n0 + (i >> 1), blk = first + n % per_head, slot = i % SLOTS;
        const long long head = b * s.heads + hk * s.group + n / per_head;
        const uint8_t* src = (i & 1 ? p.o : p.q) + (head * q_tiles + blk / 2) * (3 * TILE) + (blk & 1) * HALF;
        if (!mbar_wait(empty + slot, ((i / SLOTS) & 1) ^ 1, abort_flag)) break;
        mbar_expect_tx(full + slot, TERMS * HALF + (i & 1 ? 0 : 512));
        if (left_out(p, i)) continue;
        for (int t = 0; t < TERMS; ++t) bulk_load(ring + slot * SLOT + t * HALF, src + t * TILE, HALF, full + slot);
        if ((i & 1) == 0) bulk_load(sh_rows[slot >> 1], p.rows + head * (q_tiles * 128) + blk * 64, 512, full + slot);
      }
    }
  } else if (warp == 1 || warp == 2 + WORKERS) {
    const uint32_t ring_a = smem_u32(ring);
    const uint64_t kd = tile_desc(smem_u32(sk)), vd = tile_desc(smem_u32(sv));
    const uint32_t idesc_v = idesc_of((uint32_t)((s.dv + 15) / 16 * 16), 1), idesc_k = idesc_of((uint32_t)((s.d + 15) / 16 * 16), 1);
    bool ok = blocks > 0 && (warp != 1 || (mbar_wait(kv_full, 0, abort_flag) && mbar_wait(k_full, 0, abort_flag)));
    for (int n = 0; n < blocks && ok && warp == 1; ++n) {
      const int uq = 2 * n, uo = 2 * n + 1;
      ok = (n == 0 || mbar_wait(sd_empty, (n - 1) & 1, abort_flag)) && mbar_wait(full + uq % SLOTS, (uq / SLOTS) & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const uint64_t qd = tile_desc(ring_a + (uq % SLOTS) * SLOT), od = tile_desc(ring_a + (uo % SLOTS) * SLOT);
      if (elect_one()) {
#pragma unroll
        for (int i = 6 - PRODUCTS; i < 6; ++i)
#pragma unroll
          for (int k = 0; k < KD; ++k) {
            const uint64_t bd = qd + (uint64_t)(term_b(i) * (HALF >> 4) + k * 2);
            const uint32_t more = (i > 6 - PRODUCTS || k > 0) ? 1u : 0u;
            if (term_a(i) == 2) mma_ss(tmem, kd + (uint64_t)(k * 2), bd, idesc_of(64, 0), more);
            else mma_ts(tmem, tmem + K_COL + term_a(i) * 32 + k * 8, bd, idesc_of(64, 0), more);
          }
      }
      __syncwarp();
      ok = mbar_wait(full + uo % SLOTS, (uo / SLOTS) & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) { issue_ss<PRODUCTS, KD>(tmem + 64, vd, od, HALF, idesc_of(64, 0)); tc_commit(sd_full); }
      __syncwarp();
    }
    for (int n = 0; n < blocks && ok && warp != 1; ++n) {
      const int uq = 2 * n, uo = 2 * n + 1;
      ok = mbar_wait(full + uq % SLOTS, (uq / SLOTS) & 1, abort_flag) && mbar_wait(full + uo % SLOTS, (uo / SLOTS) & 1, abort_flag) && mbar_wait(pd_full, n & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const uint64_t qd = tile_desc(ring_a + (uq % SLOTS) * SLOT), od = tile_desc(ring_a + (uo % SLOTS) * SLOT);
      if (elect_one()) {
        issue_ts<PRODUCTS, 4, true>(tmem + DK_COL, tmem + DS_COL, 32, qd, HALF, idesc_k);
        tc_commit(empty + uq % SLOTS);
        issue_ts<PRODUCTS, 4, true>(tmem + DV_COL, tmem + P_COL, 32, od, HALF, idesc_v);
        tc_commit(empty + uo % SLOTS); tc_commit(done);
      }
      __syncwarp();
    }
  } else {
    const int quad = warp & 3, part = (warp - 2) >> 2, row = quad * 32 + lane, key = k0 + row;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const int from = key >= keys ? INT_MAX : s.causal ? key - offset : 0;      // the first query that sees this key
    float dk[16], dv[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) dk[i] = dv[i] = 0.f;
    bool ok = true;
    auto gather = [&]() {                                     // adds a block's dv and dk
      float x[16], y[16];
      load_values(tmem + lanes + DV_COL + part * 16, x);
      load_values(tmem + lanes + DK_COL + part * 16, y);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) { dv[i] += x[i]; dk[i] += y[i]; }
    };
    if (blocks > 0) {
      ok = warp_wait(k_tile, 0, abort_flag);
      if (ok) {
        RowTerms<2>(sk01, row, part).store(tmem + lanes + K_COL, part);
        tmem_st_wait();
        warp_arrive(k_full, lane);
      }
    }
    for (int n = 0; n < blocks && ok; ++n) {
      const int q0 = (first + (n0 + n) % per_head) * 64 + part * 16, slot = 2 * n % SLOTS;
      ok = warp_wait(full + slot, (2 * n / SLOTS) & 1, abort_flag) && warp_wait(sd_full, n & 1, abort_flag);      // (the first for sh_rows)
      if (!ok) break;
      tc_fence_after();
      float x[16], y[16];
      load_values(tmem + lanes + part * 16, x);
      load_values(tmem + lanes + 64 + part * 16, y);
      tmem_ld_wait();
      warp_arrive(sd_empty, lane);
      const bool whole = __all_sync(0xffffffffu, q0 >= from);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 l = sh_rows[slot >> 1][part * 8 + i];     // (lse, delta) of two queries
        x[2 * i] = exp2_fast(x[2 * i] - l.x); x[2 * i + 1] = exp2_fast(x[2 * i + 1] - l.z);
        if (!whole) { if (q0 + 2 * i < from) x[2 * i] = 0.f; if (q0 + 2 * i + 1 < from) x[2 * i + 1] = 0.f; }
        y[2 * i] = x[2 * i] * (y[2 * i] - l.y); y[2 * i + 1] = x[2 * i + 1] * (y[2 * i + 1] - l.w);
      }
      if (n > 0) {                                             // the block before: its products have read their weights
        ok = warp_wait(done, (n - 1) & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
      }
      store_terms<TERMS>(tmem + lanes + P_COL + part * 8, 32, x);
      store_terms<TERMS>(tmem + lanes + DS_COL + part * 8, 32, y);
      if (n > 0) gather();
      tmem_st_wait();
      warp_arrive(pd_full, lane);
    }
    if (ok && blocks > 0) {
      ok = warp_wait(done, (blocks - 1) & 1, abort_flag);
      if (ok) { tc_fence_after(); gather(); }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) dk[i] *= LN2;                 // (q carries scale * log2 e)
    float* stage = (float*)ring;
    if constexpr (!SHARED) {
      const int left = ok ? s.sk - k0 - quad * 32 : 0;
      write_rows<64>(stage, dk, quad, part, lane, left, p.dk + b * s.k_batch + hk * s.k_head + (k0 + quad * 32) * s.k_row, s.k_row, s.d);
      write_rows<64>(stage + 128 * 68, dv, quad, part, lane, left, p.dv + b * s.v_batch + hk * s.v_head + (k0 + quad * 32) * s.v_row, s.v_row, s.dv);
    } else {
      stage_row<64>(stage, dk, row, part);
      stage_row<64>(stage + 128 * 68, dv, row, part);
    }
  }
  if constexpr (SHARED) {
    cluster_barrier();
    if (warp >= 2 && warp < 2 + WORKERS) {
      write_sums<64>((float*)ring, parts, rank, warp - 2, lane, s.sk - k0, p.dk + b * s.k_batch + hk * s.k_head + k0 * s.k_row, s.k_row, s.d);
      write_sums<64>((float*)ring + 128 * 68, parts, rank, warp - 2, lane, s.sk - k0, p.dv + b * s.v_batch + hk * s.v_head + k0 * s.v_row, s.v_row, s.dv);
    }
    cluster_barrier();                                         // nobody leaves while its rows may still be read
  }
  tc_leave(abort_flag, p.status, warp, tmem);
}

// ---- backward: queries ----------------------------------------------------------------------------------------------------------------------
// 128 queries, one a lane; blocks of 64 keys through a ring of four 48 KB slots (k, v).  Tensor memory: [scores 64 | dp 64], ds (3 x 32), q and dout (3 x 32
// each), the block's dq (64).
template <int PRODUCTS, int KD, bool SHARED>
__global__ void __launch_bounds__(THREADS + 32, 1) attn_tc_bwd_q_kernel(TcAttn p) {
  constexpr int TERMS = PRODUCTS == 6 ? 3 : 2, HALF = TILE / 2, SLOT = 6 * HALF, SLOTS = 4, DS_COL = 128, Q_COL = 224, O_COL = 320, DQ_COL = 416;
  // barriers: full[4], empty[4], sd_full, done, a_tile, then (all workers) a_full, sd_empty, ds_full
  TC_SETUP(for (int i = 0; i < 14; ++i) mbar_init(bars + i, i < 11 ? 1 : WORKERS))
  uint64_t *full = bars, *empty = bars + 4, *sd_full = bars + 8, *done = bars + 9, *a_tile = bars + 10, *a_full = bars + 11, *sd_empty = bars + 12, *ds_full = bars + 13;
  uint8_t *sq = smem + 2 * SLOT, *so = smem + 3 * SLOT;    // two slots before their first use
  const int tiles = (s.sq + 127) / 128, all = s.heads * s.batch;
  const int parts = SHARED ? p.parts : 1, unit = (int)blockIdx.x / parts, rank = (int)blockIdx.x % parts;
  const int tile = s.causal ? tiles - 1 - unit / all : unit % tiles, bh = s.causal ? unit % all : unit / tiles;
  const int b = bh / s.heads, h = bh % s.heads, i0 = tile * 128, rows = min(128, s.sq - i0);
  const int keys = attn_keys(s, b), limit = attn_limit(s, keys, i0 + rows - 1), of_all = (limit + 63) / 64;
  const int n0 = of_all * rank / parts, blocks = of_all * (rank + 1) / parts - n0;

  if (warp == 0) {
    if (lane == 0 && blocks > 0) {
      const long long kv = (long long)(b * s.kv_heads + h / s.group) * ((s.sk + 127) / 128), own = ((long long)bh * tiles + tile) * (3 * TILE);
      mbar_expect_tx(a_tile, 2 * TERMS * TILE);
      bulk_load(sq, p.q + own, TERMS * TILE, a_tile);
      bulk_load(so, p.o + own, TERMS * TILE, a_tile);
      for (int n = 0; n < blocks; ++n) {
        if (n == 2 && !mbar_wait(a_full, 0, abort_flag)) break;
        const int slot = n % SLOTS;
        const long long at = (kv + (n0 + n) / 2) * (3 * TILE) + ((n0 + n) & 1) * HALF;
        if (!mbar_wait(empty + slot, ((n / SLOTS) & 1) ^ 1, abort_flag)) break;
        mbar_expect_tx(full + slot, 2 * TERMS * HALF);
        if (left_out(p, n)) continue;
        for (int t = 0; t < TERMS; ++t) {
          bulk_load(smem + slot * SLOT + t * HALF, p.k + at + t * TILE, HALF, full + slot);
          bulk_load(smem + slot * SLOT + 3 * HALF + t * HALF, p.v + at + t * TILE, HALF, full + slot);
        }
      }
    }
  } else if (warp == 1 || warp == 2 + WORKERS) {
    const uint32_t ring_a = smem_u32(smem);
    const uint32_t idesc_q = idesc_of((uint32_t)((s.d + 15) / 16 * 16), 1);
    bool ok = blocks > 0 && (warp != 1 || mbar_wait(a_full, 0, abort_flag));
    for (int n = 0; n < blocks && ok && warp == 1; ++n) {
      const int slot = n % SLOTS;
      ok = (n == 0 || mbar_wait(sd_empty, (n - 1) & 1, abort_flag)) && mbar_wait(full + slot, (n / SLOTS) & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const uint64_t kd = tile_desc(ring_a + slot * SLOT), vd = tile_desc(ring_a + slot * SLOT + 3 * HALF);
      if (elect_one()) {
        issue_ts<PRODUCTS, KD, false>(tmem, tmem + Q_COL, 32, kd, HALF, idesc_of(64, 0));
        issue_ts<PRODUCTS, KD, false>(tmem + 64, tmem + O_COL, 32, vd, HALF, idesc_of(64, 0));
        tc_commit(sd_full);
      }
      __syncwarp();
    }
    for (int n = 0; n < blocks && ok && warp != 1; ++n) {
      const int slot = n % SLOTS;
      ok = mbar_wait(full + slot, (n / SLOTS) & 1, abort_flag) && mbar_wait(ds_full, n & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const uint64_t kd = tile_desc(ring_a + slot * SLOT);
      if (elect_one()) {
        issue_ts<PRODUCTS, 4, true>(tmem + DQ_COL, tmem + DS_COL, 32, kd, HALF, idesc_q);
        tc_commit(empty + slot); tc_commit(done);
      }
      __syncwarp();
    }
  } else {
    const int quad = warp & 3, part = (warp - 2) >> 2, row = quad * 32 + lane;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const int lim = row < rows ? attn_limit(s, keys, i0 + row) : 0;
    float acc[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
    bool ok = true;
    if (blocks > 0) {
      ok = warp_wait(a_tile, 0, abort_flag);
      if (ok) {
        RowTerms<TERMS>(sq, row, part).store(tmem + lanes + Q_COL, part);
        RowTerms<TERMS>(so, row, part).store(tmem + lanes + O_COL, part);
        tmem_st_wait();
        warp_arrive(a_full, lane);
      }
    }
    const float2 rl = p.rows[(long long)bh * (tiles * 128) + i0 + row];
    auto gather = [&]() {
      float x[16];
      load_values(tmem + lanes + DQ_COL + part * 16, x);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[i] += x[i];
    };
    for (int n = 0; n < blocks && ok; ++n) {
      ok = warp_wait(sd_full, n & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      float x[16], y[16];
      load_values(tmem + lanes + part * 16, x);
      load_values(tmem + lanes + 64 + part * 16, y);
      tmem_ld_wait();
      warp_arrive(sd_empty, lane);
      const int see = lim - (n0 + n) * 64 - part * 16;
      const bool whole = __all_sync(0xffffffffu, see >= 16);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float pr = exp2_fast(x[i] - rl.x);
        x[i] = whole || i < see ? pr * (y[i] - rl.y) : 0.f;
      }
      if (n > 0) {
        ok = warp_wait(done, (n - 1) & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
      }
      store_terms<TERMS>(tmem + lanes + DS_COL + part * 8, 32, x);
      if (n > 0) gather();
      tmem_st_wait();
      warp_arrive(ds_full, lane);
    }
    if (ok && blocks > 0) {
      ok = warp_wait(done, (blocks - 1) & 1, abort_flag);
      if (ok) { tc_fence_after(); gather(); }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] *= s.scale;
    if constexpr (!SHARED) write_rows<64>((float*)smem, acc, quad, part, lane, ok ? rows - quad * 32 : 0, p.dq + b * s.q_batch + h * s.q_head + (i0 + quad * 32) * s.q_row, s.q_row, s.d);
    else stage_row<64>((float*)smem, acc, row, part);
  }
  if constexpr (SHARED) {
    cluster_barrier();
    if (warp >= 2 && warp < 2 + WORKERS) write_sums<64>((float*)smem, parts, rank, warp - 2, lane, rows, p.dq + b * s.q_batch + h * s.q_head + i0 * s.q_row, s.q_row, s.d);
    cluster_barrier();
  }
  tc_leave(abort_flag, p.status, warp, tmem);
}

// ---- widths above 64 --------------------------------------------------------------------------------------------------------------------------
// Four passes of one shape: a tile of 128 rows r against blocks of 64 columns c of the other side,
//   scores S = X1 . Y1',  (dq, dk: D = X2 . Y2'),  weights W from them, result += W . Y
//   FORWARD  rows queries   X1 = q, Y1 = k, Y2 = v            W = 2^(S - running maximum)      out = sum W Y2
//   DV       rows keys      X1 = k, Y1 = q, Y2 = dout         W = p                            dv  = sum W Y2
//   DQ       rows queries   X1 = q, X2 = dout, Y1 = k, Y2 = v W = p (D - delta)                dq  = sum W Y1
//   DK       rows keys      X1 = k, X2 = v, Y1 = q, Y2 = dout W = p (D - delta)                dk  = sum W Y1
// X1 lies in shared memory (up to 96 KB), X2 in tensor memory, one block of Y1 and Y2 each in shared memory (up to 48 KB).  FORWARD and DV have two buffers of
// scores and compute those of block n + 1 beside the work on block n; DQ and DK hold X2 there instead and go step by step.  C1, C2: chunks of 64 columns
// of q / k and of v / dout.  Measured, 32 causal heads of 1 024 x 1 024, width 128: forward 74 us, dv 81, dk 113, dq 100.
enum { FORWARD, DV_PASS, DQ_PASS, DK_PASS };

template <int PRODUCTS, int C1, int C2, int PASS>
__global__ void __launch_bounds__(THREADS, 1) attn_tc_wide_kernel(TcAttn p) {
  constexpr bool GRAD = PASS == DQ_PASS || PASS == DK_PASS, KEY_ROWS = PASS == DV_PASS || PASS == DK_PASS;
  constexpr int TERMS = PRODUCTS == 6 ? 3 : 2, HALF = TILE / 2, CR = GRAD ? C1 : C2;      // (chunks of the result)
  constexpr int BUFS = GRAD ? 1 : 2, BUF = GRAD ? 128 : 96, R_COL = GRAD ? 128 : 192, X2_COL = 256;
  __shared__ float sh_max[2][4][128], sh_sum[4][128];
  __shared__ float2 sh_ms[128];
  // barriers: x1_full, y_full[2], y_empty[2], s_full[2], done, then (all workers) x2_full, w_full[2], r_empty
  TC_SETUP(for (int i = 0; i < 12; ++i) mbar_init(bars + i, i < 8 ? 1 : WORKERS))
  uint64_t *x1_full = bars, *y_full = bars + 1, *y_empty = bars + 3, *s_full = bars + 5, *done = bars + 7, *x2_full = bars + 8, *w_full = bars + 9, *r_empty = bars + 11;
  const int heads = KEY_ROWS ? s.kv_heads : s.heads, n_rows = KEY_ROWS ? s.sk : s.sq, n_cols = KEY_ROWS ? s.sq : s.sk;
  const int tiles = (n_rows + 127) / 128, col_tiles = (n_cols + 127) / 128, all = heads * s.batch;
  const int parts = p.parts, unit = (int)blockIdx.x / parts, rank = (int)blockIdx.x % parts, at_tile = unit / all;
  const int tile = s.causal && !KEY_ROWS ? tiles - 1 - at_tile : at_tile, bh = unit % all, b = bh / heads, h = bh % heads;
  const int r0 = tile * 128, rows = min(128, n_rows - r0), keys = attn_keys(s, b), offset = attn_shift(s, keys);
  // blocks of 64 columns: of one key head, or of the queries of every head that shares it
  const int first = KEY_ROWS && s.causal ? max(0, r0 - offset) / 64 : 0;
  const int per_head = KEY_ROWS ? (r0 < keys ? max(0, (s.sq + 63) / 64 - first) : 0) : (attn_limit(s, keys, r0 + rows - 1) + 63) / 64;
  const int of_all = per_head * (KEY_ROWS ? s.group : 1), n0 = of_all * rank / parts, blocks = of_all * (rank + 1) / parts - n0;      // this CTA's share
  const uint8_t *gx1 = KEY_ROWS ? p.k : p.q, *gx2 = KEY_ROWS ? p.v : p.o, *gy1 = KEY_ROWS ? p.q : p.k, *gy2 = KEY_ROWS ? p.o : p.v;
  uint8_t *x1 = smem, *y1 = smem + C1 * 3 * TILE, *y2 = y1 + C1 * 3 * HALF;
  float* o = PASS == FORWARD ? p.out + b * s.o_batch + h * s.o_head + r0 * s.o_row : PASS == DV_PASS ? p.dv + b * s.v_batch + h * s.v_head + r0 * s.v_row
           : PASS == DQ_PASS ? p.dq + b * s.q_batch + h * s.q_head + r0 * s.q_row : p.dk + b * s.k_batch + h * s.k_head + r0 * s.k_row;
  const long long stride = PASS == FORWARD ? s.o_row : PASS == DV_PASS ? s.v_row : PASS == DQ_PASS ? s.q_row : s.k_row;

  if (warp == 0) {
    if (lane == 0 && blocks > 0) {
      mbar_expect_tx(x1_full, C1 * TERMS * TILE);
      for (int c = 0; c < C1; ++c) bulk_load(x1 + c * 3 * TILE, gx1 + (((long long)bh * tiles + tile) * C1 + c) * (3 * TILE), TERMS * TILE, x1_full);
      for (int n = 0; n < blocks; ++n) {
        const int head = KEY_ROWS ? b * s.heads + h * s.group + (n0 + n) / per_head : b * s.kv_heads + h / s.group, blk = first + (n0 + n) % per_head;
        const long long at = (long long)head * col_tiles + blk / 2;
        // (which of the two comes first is which is free first: Y1 is read last where the result is summed over it)
        for (int k = 0; k < 2; ++k) {
          const int which = GRAD ? 1 - k : k, chunks = which ? C2 : C1;
          if (!mbar_wait(y_empty + which, (n & 1) ^ 1, abort_flag)) { n = blocks; break; }
          mbar_expect_tx(y_full + which, chunks * TERMS * HALF);
          if (left_out(p, 2 * n + k)) continue;
          for (int c = 0; c < chunks; ++c)
            for (int t = 0; t < TERMS; ++t)
              bulk_load((which ? y2 : y1) + (c * 3 + t) * HALF, (which ? gy2 : gy1) + (at * chunks + c) * (3 * TILE) + t * TILE + (blk & 1) * HALF, HALF, y_full + which);
        }
      }
    }
  } else if (warp == 1) {
    const uint64_t d1 = tile_desc(smem_u32(x1)), e1 = tile_desc(smem_u32(y1)), e2 = tile_desc(smem_u32(y2));
    const int width = GRAD ? s.d : s.dv;
    const int last1 = s.d - (C1 - 1) * 64 <= 32 ? 2 : 4;      // steps of 16 values in the last chunk of q and k
    bool ok = blocks > 0 && mbar_wait(x1_full, 0, abort_flag) && (!GRAD || mbar_wait(x2_full, 0, abort_flag));
    auto scores = [&](int n) {
      const int buf = GRAD ? 0 : n & 1;
      ok = (n < BUFS || mbar_wait(done, (n - BUFS) & 1, abort_flag)) && mbar_wait(y_full, n & 1, abort_flag) && (!GRAD || mbar_wait(y_full + 1, n & 1, abort_flag));
      if (!ok) return;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int i = 6 - PRODUCTS; i < 6; ++i)
#pragma unroll
          for (int c = 0; c < C1; ++c)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (c + 1 < C1 || k < last1)
                mma_ss(tmem + buf * BUF, d1 + (uint64_t)(((c * 3 + term_a(i)) * TILE >> 4) + k * 2), e1 + (uint64_t)(((c * 3 + term_b(i)) * HALF >> 4) + k * 2), idesc_of(64, 0),
                       (i > 6 - PRODUCTS || c > 0 || k > 0) ? 1u : 0u);
        if (GRAD) {
#pragma unroll
          for (int i = 6 - PRODUCTS; i < 6; ++i)
#pragma unroll
            for (int c = 0; c < C2; ++c)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                mma_ts(tmem + buf * BUF + 64, tmem + X2_COL + (c * 3 + term_a(i)) * 32 + k * 8, e2 + (uint64_t)(((c * 3 + term_b(i)) * HALF >> 4) + k * 2), idesc_of(64, 0),
                       (i > 6 - PRODUCTS || c > 0 || k > 0) ? 1u : 0u);
          tc_commit(y_empty + 1);
        } else tc_commit(y_empty);
        tc_commit(s_full + buf);
      }
      __syncwarp();
    };
    if (ok) scores(0);
    for (int n = 0; n < blocks && ok; ++n) {
      const int buf = GRAD ? 0 : n & 1;
      if (!GRAD && n + 1 < blocks) { scores(n + 1); if (!ok) break; }
      ok = mbar_wait(w_full + buf, (GRAD ? n : n >> 1) & 1, abort_flag) && (n == 0 || mbar_wait(r_empty, (n - 1) & 1, abort_flag)) && (GRAD || mbar_wait(y_full + 1, n & 1, abort_flag));
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int c = 0; c < CR; ++c) {
          const uint32_t idesc = idesc_of((uint32_t)(max(1, min(64, width - c * 64)) + 15) / 16 * 16, 1);      // (an empty chunk: zeros)
          issue_ts<PRODUCTS, 4, true>(tmem + R_COL + c * 64, tmem + buf * BUF, 32, (GRAD ? e1 : e2) + (uint64_t)(c * 3 * HALF >> 4), HALF, idesc);
        }
        tc_commit(y_empty + (GRAD ? 0 : 1)); tc_commit(done);
      }
      __syncwarp();
      if (GRAD && n + 1 < blocks) scores(n + 1);
    }
  } else {
    const int quad = warp & 3, part = (warp - 2) >> 2, row = quad * 32 + lane, at_row = r0 + row;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    // columns that the row sees: [from, lim) of the other side
    const int lim = KEY_ROWS ? (at_row < keys ? INT_MAX : 0) : row < rows ? attn_limit(s, keys, at_row) : 0, from = KEY_ROWS && s.causal ? at_row - offset : 0;
    float acc[CR * 16], m = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < CR * 16; ++i) acc[i] = 0.f;
    bool ok = true;
    if (GRAD && blocks > 0) {                                  // this thread's share of the row's X2 terms
#pragma unroll
      for (int c = 0; c < C2; ++c)
#pragma unroll
        for (int t = 0; t < TERMS; ++t) {
          const uint8_t* src = gx2 + ((((long long)bh * tiles + tile) * C2 + c) * 3 + t) * TILE + row * 128;
          uint32_t w[8];
#pragma unroll
          for (int i = 0; i < 2; ++i) { const uint4 v = *(const uint4*)(src + (((part * 2 + i) ^ (row & 7)) << 4)); w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w; }
          tmem_st8(tmem + lanes + X2_COL + (c * 3 + t) * 32 + part * 8, w);
        }
      tmem_st_wait();
      warp_arrive(x2_full, lane);
    }
    const int q_pad = (s.sq + 127) / 128 * 128;
    float2 rl = make_float2(0.f, 0.f);
    if (PASS == DQ_PASS) rl = p.rows[(long long)bh * q_pad + at_row];
    auto gather = [&](int n, float f) {                        // acc = (acc + block n's result) * f
      if (!warp_wait(done, n & 1, abort_flag)) { ok = false; return; }
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < CR; ++c) {
        float x[16];
        load_values(tmem + lanes + R_COL + part * (CR * 16) + c * 16, x);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[c * 16 + i] = (acc[c * 16 + i] + x[i]) * f;
      }
      warp_arrive(r_empty, lane);
    };
    for (int n = 0; n < blocks; ++n) {
      const int buf = GRAD ? 0 : n & 1, c0 = (first + (n0 + n) % per_head) * 64 + part * 16;
      const float4* cl = KEY_ROWS ? (const float4*)(p.rows + (long long)(b * s.heads + h * s.group + (n0 + n) / per_head) * q_pad + c0) : nullptr;
      ok = ok && warp_wait(s_full + buf, (GRAD ? n : n >> 1) & 1, abort_flag);
      if (!ok) { row_barrier(quad); continue; }
      tc_fence_after();
      float x[16], y[GRAD ? 16 : 1], f = 1.f;
      load_values(tmem + lanes + buf * BUF + part * 16, x);
      if constexpr (GRAD) load_values(tmem + lanes + buf * BUF + 64 + part * 16, y);
      tmem_ld_wait();
      const bool whole = __all_sync(0xffffffffu, c0 >= from && c0 + 16 <= lim);
      if constexpr (PASS == FORWARD) {
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 16; ++i) if (c0 + i >= lim) x[i] = -INFINITY;
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, x[i]);
        sh_max[n & 1][part][row] = top;
        tc_fence_before();
        row_barrier(quad);                                    // (also: the threads of the row hold their scores)
        tc_fence_after();
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, sh_max[n & 1][i][row]);
        const float ref = top == -INFINITY ? 0.f : top;
        f = exp2_fast(m - ref);
        m = top;
        float block = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) { x[i] = exp2_fast(x[i] - ref); block += x[i]; }
        sum = sum * f + block;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 l = KEY_ROWS ? cl[i] : make_float4(rl.x, rl.y, rl.x, rl.y);      // (lse, delta) of two columns, or of the row
          x[2 * i] = exp2_fast(x[2 * i] - l.x); x[2 * i + 1] = exp2_fast(x[2 * i + 1] - l.z);
          if (!whole) {
            if (c0 + 2 * i < from || c0 + 2 * i >= lim) x[2 * i] = 0.f;
            if (c0 + 2 * i + 1 < from || c0 + 2 * i + 1 >= lim) x[2 * i + 1] = 0.f;
          }
          if constexpr (GRAD) { x[2 * i] = x[2 * i] == 0.f ? 0.f : x[2 * i] * (y[2 * i] - l.y); x[2 * i + 1] = x[2 * i + 1] == 0.f ? 0.f : x[2 * i + 1] * (y[2 * i + 1] - l.w); }
        }
        tc_fence_before();
        row_barrier(quad);
        tc_fence_after();
      }
      store_terms<TERMS>(tmem + lanes + buf * BUF + part * 8, 32, x);
      tmem_st_wait();
      warp_arrive(w_full + buf, lane);
      if (n > 0) gather(n - 1, f);
    }
    if (ok && blocks > 0) gather(blocks - 1, 1.f);
    if constexpr (PASS == FORWARD) { sh_sum[part][row] = sum; row_barrier(quad); }
    float scale = PASS == DQ_PASS ? s.scale : PASS == DK_PASS ? LN2 : 1.f;      // (q carries scale * log2 e)
    if constexpr (PASS == FORWARD) {
      const float total = (sh_sum[0][row] + sh_sum[1][row]) + (sh_sum[2][row] + sh_sum[3][row]);
      if (parts == 1) {
        scale = total > 0.f ? 1.f / total : total == 0.f ? 0.f : total;
        if (ok && row < rows && p.lse && part == 0) p.lse[(long long)bh * s.sq + at_row] = total == 0.f ? -INFINITY : (m + log2f(total)) * LN2;
      } else if (part == 0) sh_ms[row] = make_float2(m, total);
    }
#pragma unroll
    for (int i = 0; i < CR * 16; ++i) acc[i] *= scale;
    // (the operands' space is free: all products are done)
    if (parts == 1) write_rows<CR * 64>((float*)smem, acc, quad, part, lane, ok ? rows - quad * 32 : 0, o + quad * 32 * stride, stride, GRAD ? s.d : s.dv);
    else stage_row<CR * 64>((float*)smem, acc, row, part);
  }
  if (parts > 1) {
    cluster_barrier();
    if (warp >= 2) {
      if constexpr (PASS == FORWARD)
        write_weighted<CR * 64>((float*)smem, sh_ms, parts, rank, warp - 2, lane, rows, o, stride, s.dv, p.lse ? p.lse + (long long)bh * s.sq + r0 : nullptr);
      else write_sums<CR * 64>((float*)smem, parts, rank, warp - 2, lane, rows, o, stride, GRAD ? s.d : s.dv);
    }
    cluster_barrier();
  }
  tc_leave(abort_flag, p.status, warp, tmem);
}

// Up to 64 queries and keys a tile is mostly padding, and the CUDA cores are ahead (512 heads of 64 x 64, widths 32: forward 18 us there, 40 here, backward
// 57 and 86; at 80 x 80 45 and 41, 135 and 109).
bool prepare(talos_ctx* ctx, const AttnShape& s) {
  if (s.sq <= 64 && s.sk <= 64) return false;
  return talos_tc_ready_for(ctx);
}

// The split tiles are larger than what they hold (1.5 times in full tiles, 48 KB for a head's rows however few and narrow): they are made for as many
// sequences at a time as fit this, the work of thousands of CTAs.
constexpr size_t SCRATCH = 1ull << 30;
// part(shape of some sequences, the first of them)
template <typename F> void in_slices(const AttnShape& s, size_t bytes, F&& part) {
  const int step = (int)std::max<int64_t>(1, (int64_t)(SCRATCH / std::max<size_t>(1, bytes / s.batch)));
  for (int b = 0; b < s.batch; b += std::min(step, s.batch - b)) {
    AttnShape t = s;
    t.batch = std::min(step, s.batch - b);
    if (s.key_len) t.key_len += b;
    part(t, (long long)b);
  }
}

// Space for the split tiles of one tensor.
size_t tile_bytes(int64_t heads, int64_t rows, int chunks) { return (size_t)(heads * ((rows + 127) / 128)) * 3 * TILE * chunks; }

// Of the whole problem, about (queries: 1 tensor of their rows forward, 2 backward).
size_t scratch(const AttnShape& s, int queries) {
  return (tile_bytes((int64_t)s.batch * s.heads, s.sq, 1) * queries + tile_bytes((int64_t)s.batch * s.kv_heads, s.sk, 1) * 2) * (s.d > 64 || s.dv > 64 ? 2 : 1);
}

struct Splitter {
  SplitArgs a{};
  void add(const float* x, uint8_t* tiles, long long row, long long head, long long bat, int heads, int batch, int rows, int width, bool keys, float factor, int chunks) {
    a.job[a.jobs++] = SplitJob{x, tiles, row, head, bat, heads, rows, width, keys ? 1 : 0, chunks, factor, a.ctas};
    a.ctas += batch * heads * ((rows + 127) / 128 * 4) * chunks;
  }
  void launch(talos_ctx* ctx, int mode) {
    if (mode == TALOS_MODE_TF32) talos_kernel(ctx, attn_split_kernel<2>, (unsigned)a.ctas, 256, 0, a);
    else talos_kernel(ctx, attn_split_kernel<3>, (unsigned)a.ctas, 256, 0, a);
    talos_launched(ctx, "attention_split");
  }
};

// CTAs of a cluster that share the blocks of each of `grid` tiles, `blocks` of the longest, where the tiles do not fill the SMs.  A CTA costs about two and a
// half blocks beside its own; causal: the mean tile has half of the longest one's.  Forward / backward in all, us, without and with: 12 heads on 4 key
// heads, 3 x 777 x 777, 51 / 159 and 51 / 141; 4 causal heads on one key head, 1 024 x 1 024, 26 / 183 and 17.5 / 48; 2 causal heads of 4 096 x 4 096 80 / 259
// and 43 / 107; 8 of 512 x 512 18 / 49 and 17 / 31; width 128, 4 causal heads on one key head, 1 024 x 1 024, 65 / 667 and 28 / 125.
int shares(talos_ctx* ctx, int64_t grid, int blocks, bool causal) {
  int best = 1;
  float least = INFINITY;
  for (int n : {1, 2, 3, 4, 6, 8}) {                          // (five or seven would leave SMs of a group of 16 to 18 without a cluster)
    if (n > 1 && 2 * n > blocks) break;
    const float rounds = (float)ceil_div(grid * n, ctx->sm_count), longest = (float)blocks / n + 2.5f, mean = (causal ? 0.5f : 1.f) * blocks / n + 2.5f;
    const float cost = std::max(longest, rounds * mean);
    if (cost < 0.95f * least) { least = cost; best = n; }
  }
  return best;
}

template <typename K> void run_tc(talos_ctx* ctx, K kern, std::atomic<uint64_t>& done, int64_t grid, size_t smem, const TcAttn& p, const char* what, int threads = THREADS) {
  talos_allow_smem(done, (const void*)kern, smem, ctx->device);
  talos_kernel_cluster(ctx, kern, (unsigned)(grid * p.parts), threads, smem, (unsigned)p.parts, p);
  talos_launched(ctx, what);
}

}  // namespace

template <int PRODUCTS, int C1, int C2, int PASS> void run_wide(talos_ctx* ctx, int64_t grid, const TcAttn& p, const char* what) {
  static std::atomic<uint64_t> done{0};
  run_tc(ctx, attn_tc_wide_kernel<PRODUCTS, C1, C2, PASS>, done, grid, (size_t)C1 * 3 * TILE + (C1 + C2) * (3 * TILE / 2) + 1024, p, what);
}

static void attn_tc_fwd_slice(talos_ctx* ctx, const AttnShape& s, const float* q, const float* k, const float* v, float* out, float* lse, int mode) {
  const int64_t hq = (int64_t)s.batch * s.heads, hk = (int64_t)s.batch * s.kv_heads;
  const int c1 = s.d > 64 || s.dv > 64 ? 2 : 1, c2 = s.dv > 64 ? 2 : 1;
  const size_t nq = tile_bytes(hq, s.sq, c1), nk = tile_bytes(hk, s.sk, c1), nv = tile_bytes(hk, s.sk, c2);
  uint8_t* ws = (uint8_t*)talos_workspace2(ctx, nq + nk + nv);
  TcAttn p{};
  p.s = s; p.parts = 1; p.q = ws; p.k = ws + nq; p.v = ws + nq + nk; p.out = out; p.lse = lse;
  p.status = ctx->dev_status; p.wait_spins = ctx->dbg_wait_spins ? ctx->dbg_wait_spins : WAIT_SPINS; p.skip = ctx->dbg_skip_kb;
  Splitter sp;
  sp.a.key_len = s.key_len;
  sp.add(q, ws, s.q_row, s.q_head, s.q_batch, s.heads, s.batch, s.sq, s.d, false, s.scale * LOG2E, c1);
  sp.add(k, ws + nq, s.k_row, s.k_head, s.k_batch, s.kv_heads, s.batch, s.sk, s.d, true, 1.f, c1);
  sp.add(v, ws + nq + nk, s.v_row, s.v_head, s.v_batch, s.kv_heads, s.batch, s.sk, s.dv, true, 1.f, c2);
  sp.launch(ctx, mode);
  const int64_t grid = hq * ((s.sq + 127) / 128);
  if (c1 == 2) {
    p.parts = shares(ctx, grid, (s.sk + 63) / 64, s.causal);
    if (mode == TALOS_MODE_TF32) { if (c2 == 2) run_wide<3, 2, 2, FORWARD>(ctx, grid, p, "attention_tc_fwd"); else run_wide<3, 2, 1, FORWARD>(ctx, grid, p, "attention_tc_fwd"); }
    else if (c2 == 2) run_wide<6, 2, 2, FORWARD>(ctx, grid, p, "attention_tc_fwd");
    else run_wide<6, 2, 1, FORWARD>(ctx, grid, p, "attention_tc_fwd");
    return;
  }
  const size_t smem = 4 * 3 * TILE + 1024;
  static std::atomic<uint64_t> done[8];
  p.parts = shares(ctx, grid, (s.sk + 127) / 128, s.causal);
  auto go = [&](auto kern, auto kern_shared, std::atomic<uint64_t>* d) {
    if (p.parts > 1) run_tc(ctx, kern_shared, d[1], grid, smem, p, "attention_tc_fwd"); else run_tc(ctx, kern, d[0], grid, smem, p, "attention_tc_fwd");
  };
  if (mode == TALOS_MODE_TF32) {
    if (s.d <= 32) go(attn_tc_fwd_kernel<3, 2, false>, attn_tc_fwd_kernel<3, 2, true>, done); else go(attn_tc_fwd_kernel<3, 4, false>, attn_tc_fwd_kernel<3, 4, true>, done + 2);
  } else {
    if (s.d <= 32) go(attn_tc_fwd_kernel<6, 2, false>, attn_tc_fwd_kernel<6, 2, true>, done + 4); else go(attn_tc_fwd_kernel<6, 4, false>, attn_tc_fwd_kernel<6, 4, true>, done + 6);
  }
}

bool talos_attn_tc_fwd(talos_ctx* ctx, const AttnShape& s, const float* q, const float* k, const float* v, float* out, float* lse, int mode) {
  if (!prepare(ctx, s)) return false;
  in_slices(s, scratch(s, 1), [&](const AttnShape& t, long long b) {
    attn_tc_fwd_slice(ctx, t, q + b * s.q_batch, k + b * s.k_batch, v + b * s.v_batch, out + b * s.o_batch, lse ? lse + b * s.heads * s.sq : nullptr, mode);
  });
  return true;
}

template <int PRODUCTS, int C2> void run_wide_bwd(talos_ctx* ctx, int64_t grid_kv, int64_t grid_q, TcAttn p) {
  p.parts = shares(ctx, grid_kv, p.s.group * ((p.s.sq + 63) / 64), p.s.causal);
  run_wide<PRODUCTS, 2, C2, DV_PASS>(ctx, grid_kv, p, "attention_tc_bwd_v");
  run_wide<PRODUCTS, 2, C2, DK_PASS>(ctx, grid_kv, p, "attention_tc_bwd_k");
  p.parts = shares(ctx, grid_q, (p.s.sk + 63) / 64, p.s.causal);
  run_wide<PRODUCTS, 2, C2, DQ_PASS>(ctx, grid_q, p, "attention_tc_bwd_q");
}

static void attn_tc_bwd_slice(talos_ctx* ctx, const AttnShape& s, const float* q, const float* k, const float* v, const float* out, const float* lse, const float* dout, float* dq,
                       float* dk, float* dv, int mode) {
  const int64_t hq = (int64_t)s.batch * s.heads, hk = (int64_t)s.batch * s.kv_heads, rows = hq * ((s.sq + 127) / 128 * 128);
  const int c1 = s.d > 64 || s.dv > 64 ? 2 : 1, c2 = s.dv > 64 ? 2 : 1;
  const size_t nq = tile_bytes(hq, s.sq, c1), no = tile_bytes(hq, s.sq, c2), nk = tile_bytes(hk, s.sk, c1), nv = tile_bytes(hk, s.sk, c2);
  uint8_t* ws = (uint8_t*)talos_workspace2(ctx, nq + no + nk + nv + sizeof(float2) * (size_t)rows);
  TcAttn p{};
  p.s = s; p.parts = 1; p.q = ws; p.o = ws + nq; p.k = ws + nq + no; p.v = ws + nq + no + nk; p.rows = (const float2*)(ws + nq + no + nk + nv);
  p.dq = dq; p.dk = dk; p.dv = dv;
  p.status = ctx->dev_status; p.wait_spins = ctx->dbg_wait_spins ? ctx->dbg_wait_spins : WAIT_SPINS; p.skip = ctx->dbg_skip_kb;
  Splitter sp;
  sp.a.key_len = s.key_len;
  sp.add(q, (uint8_t*)p.q, s.q_row, s.q_head, s.q_batch, s.heads, s.batch, s.sq, s.d, false, s.scale * LOG2E, c1);
  sp.add(dout, (uint8_t*)p.o, s.o_row, s.o_head, s.o_batch, s.heads, s.batch, s.sq, s.dv, false, 1.f, c2);
  sp.add(k, (uint8_t*)p.k, s.k_row, s.k_head, s.k_batch, s.kv_heads, s.batch, s.sk, s.d, true, 1.f, c1);
  sp.add(v, (uint8_t*)p.v, s.v_row, s.v_head, s.v_batch, s.kv_heads, s.batch, s.sk, s.dv, true, 1.f, c2);
  sp.launch(ctx, mode);
  talos_kernel(ctx, attn_rows_kernel, (unsigned)(rows / 64), 256, 0, s, out, dout, lse, (float2*)p.rows);
  talos_launched(ctx, "attention_rows");
  const int64_t grid_kv = hk * ((s.sk + 127) / 128), grid_q = hq * ((s.sq + 127) / 128);
  if (c1 == 2) {
    if (mode == TALOS_MODE_TF32) { if (c2 == 2) run_wide_bwd<3, 2>(ctx, grid_kv, grid_q, p); else run_wide_bwd<3, 1>(ctx, grid_kv, grid_q, p); }
    else if (c2 == 2) run_wide_bwd<6, 2>(ctx, grid_kv, grid_q, p);
    else run_wide_bwd<6, 1>(ctx, grid_kv, grid_q, p);
    return;
  }
  const size_t smem_kv = 4 * TILE + 6 * (3 * TILE / 2) + 1024, smem_q = 4 * 3 * TILE + 1024;
  static std::atomic<uint64_t> done[16];
  const int parts_kv = shares(ctx, grid_kv, s.group * ((s.sq + 63) / 64), s.causal), parts_q = shares(ctx, grid_q, (s.sk + 63) / 64, s.causal);
  auto go = [&](auto kern, auto kern_shared, int parts, int64_t grid, size_t smem, std::atomic<uint64_t>* d, const char* what) {
    p.parts = parts;
    if (parts > 1) run_tc(ctx, kern_shared, d[1], grid, smem, p, what, THREADS + 32); else run_tc(ctx, kern, d[0], grid, smem, p, what, THREADS + 32);
  };
#define TALOS_TC_BWD(PR, KD, I) { go(attn_tc_bwd_kv_kernel<PR, KD, false>, attn_tc_bwd_kv_kernel<PR, KD, true>, parts_kv, grid_kv, smem_kv, done + 4 * I, "attention_tc_bwd_kv"); \
                                  go(attn_tc_bwd_q_kernel<PR, KD, false>, attn_tc_bwd_q_kernel<PR, KD, true>, parts_q, grid_q, smem_q, done + 4 * I + 2, "attention_tc_bwd_q"); }
  const bool narrow = s.d <= 32 && s.dv <= 32;
  if (mode == TALOS_MODE_TF32) { if (narrow) TALOS_TC_BWD(3, 2, 0) else TALOS_TC_BWD(3, 4, 1) }
  else { if (narrow) TALOS_TC_BWD(6, 2, 2) else TALOS_TC_BWD(6, 4, 3) }
#undef TALOS_TC_BWD
}

bool talos_attn_tc_bwd(talos_ctx* ctx, const AttnShape& s, const float* q, const float* k, const float* v, const float* out, const float* lse, const float* dout, float* dq,
                       float* dk, float* dv, int mode) {
  if (!prepare(ctx, s)) return false;
  in_slices(s, scratch(s, 2), [&](const AttnShape& t, long long b) {
    attn_tc_bwd_slice(ctx, t, q + b * s.q_batch, k + b * s.k_batch, v + b * s.v_batch, out + b * s.o_batch, lse + b * s.heads * s.sq, dout + b * s.o_batch, dq + b * s.q_batch,
                      dk + b * s.k_batch, dv + b * s.v_batch, mode);
  });
  return true;
}
