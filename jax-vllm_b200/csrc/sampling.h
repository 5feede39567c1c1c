// What the kernels that draw tokens share: the uniform numbers of a row, and the choice of the best token of a block.
#pragma once

#include "common.cuh"
#include <math.h>

__host__ __device__ __forceinline__ unsigned long long jv_mix64(unsigned long long z) {
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ULL;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBULL;
  return z ^ (z >> 31);
}

// What the numbers of one (seed, counter) have in common, and the 64 random bits of its vocabulary index v.
__host__ __device__ __forceinline__ unsigned long long jv_draw_base(unsigned long long seed, unsigned long long counter) {
  return jv_mix64(seed + 0x9E3779B97F4A7C15ULL * (counter + 1));
}
__host__ __device__ __forceinline__ unsigned long long jv_draw_bits(unsigned long long base, unsigned long long v) {
  return jv_mix64(base ^ (v * 0xD1342543DE82EF95ULL + 0x2545F4914F6CDD1DULL));
}

// The first 23 of them.  (The last shift of jv_mix64 reaches none but the lowest of the high word's bits.)
__host__ __device__ __forceinline__ unsigned jv_draw_first23(unsigned long long base, unsigned long long v) {
  unsigned long long z = base ^ (v * 0xD1342543DE82EF95ULL + 0x2545F4914F6CDD1DULL);
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ULL;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBULL;
  return (unsigned)(z >> 41);
}

// Uniform in (0, 1) with 24 of them: (n + 1/2) / 2^24, rounded to 32 bits.  The topmost would round to 1, whose score
// -log(-log(u)) is infinite: it is the largest number below.
__host__ __device__ __forceinline__ float jv_uniform_of(unsigned long long bits) {
  return fminf(((float)(unsigned)(bits >> 40) + 0.5f) * (1.0f / 16777216.0f), 1.0f - 1.0f / 16777216.0f);
}
__host__ __device__ __forceinline__ float jv_uniform(unsigned long long seed, unsigned long long counter,
                                                     unsigned long long v) {
  return jv_uniform_of(jv_draw_bits(jv_draw_base(seed, counter), v));
}

// (value, index) ordering: larger value wins, the lower index among equal values.
__device__ __forceinline__ void take_better(float& bv, int& bi, float ov, int oi) {
  if (ov > bv || (ov == bv && oi < bi)) { bv = ov; bi = oi; }
}

__device__ __forceinline__ void block_best(float& bv, int& bi, float* sv, int* si) {
  for (int o = 16; o > 0; o >>= 1)
    take_better(bv, bi, __shfl_xor_sync(0xffffffffu, bv, o), __shfl_xor_sync(0xffffffffu, bi, o));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) { sv[warp] = bv; si[warp] = bi; }
  __syncthreads();
  if (warp == 0) {
    const int nwarps = blockDim.x >> 5;
    bv = lane < nwarps ? sv[lane] : -INFINITY;
    bi = lane < nwarps ? si[lane] : 0x7fffffff;
    for (int o = 16; o > 0; o >>= 1)
      take_better(bv, bi, __shfl_xor_sync(0xffffffffu, bv, o), __shfl_xor_sync(0xffffffffu, bi, o));
  }
}
