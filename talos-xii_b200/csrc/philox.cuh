// The counter-based generator of the dropout kernels: philox4x32-10 of Salmon, Moraes, Dror and Shaw, "Parallel random
// numbers: as easy as 1, 2, 3" (SC 2011).  Four 32-bit words per call from a 128-bit counter and a 64-bit key: ten rounds of
// two 32 x 32 -> 64 bit products.
#pragma once
#include <math.h>

#include "common.cuh"

// What a dropout kernel is told: the generator's key and offset, the smallest word that is kept, the scale of what is kept.
struct DropArgs {
  uint32_t k0, k1; unsigned long long offset; const unsigned long long* offset_dev; uint32_t threshold; float scale;
};
inline DropArgs talos_drop_args(float p, uint64_t seed, uint64_t offset, const uint64_t* offset_dev) {
  TALOS_REQUIRE(p >= 0.f && p < 1.f, TALOS_ERR_ARG, "dropout probability must be in [0, 1)");
  DropArgs a;
  a.k0 = (uint32_t)seed; a.k1 = (uint32_t)(seed >> 32);
  a.offset = offset; a.offset_dev = (const unsigned long long*)offset_dev;
  a.threshold = (uint32_t)floor((double)p * 4294967296.0 + 0.5);      // p < 1 is at most 1 - 2^-24: below 2^32
  a.scale = (float)(1.0 / (1.0 - (double)p));
  return a;
}

#ifdef __CUDACC__
__device__ __forceinline__ uint4 talos_philox(unsigned long long block, unsigned long long offset, uint32_t k0, uint32_t k1) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long a = (unsigned long long)0xD2511F53u * c0, b = (unsigned long long)0xCD9E8D57u * c2;
    const uint32_t n0 = (uint32_t)(b >> 32) ^ c1 ^ k0, n2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)b; c3 = (uint32_t)a; c0 = n0; c2 = n2;
    k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}
// The factors (0 or scale) of elements 4 * block .. 4 * block + 3.
__device__ __forceinline__ float4 talos_drop4(const DropArgs& d, unsigned long long offset, unsigned long long block) {
  const uint4 w = talos_philox(block, offset, d.k0, d.k1);
  return make_float4(w.x >= d.threshold ? d.scale : 0.f, w.y >= d.threshold ? d.scale : 0.f, w.z >= d.threshold ? d.scale : 0.f,
                     w.w >= d.threshold ? d.scale : 0.f);
}
// The factor of one element.
__device__ __forceinline__ float talos_drop1(const DropArgs& d, unsigned long long offset, unsigned long long i) {
  const uint4 w = talos_philox(i >> 2, offset, d.k0, d.k1);
  const uint32_t lo = (i & 1) ? w.y : w.x, hi = (i & 1) ? w.w : w.z;
  return ((i & 2) ? hi : lo) >= d.threshold ? d.scale : 0.f;
}
#endif
