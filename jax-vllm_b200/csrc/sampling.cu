// Token choice from 32-bit logits, one block per row.
//   temperature == 0: the index of the largest logit (the lowest index among equals).
//   temperature  > 0: a draw from softmax(logits / temperature) by the Gumbel-max rule,
//       argmax_v(logits[v] / temperature - log(-log(u_v))), with u_v in (0, 1) from a
//       counter-based generator keyed by (seed of the request, index of the output token,
//       v).  The draw therefore depends on the request and the place in its output only,
//       not on the batch it was sampled in.
#include "sampling.h"

// Stage 1: block (chunk, row) finds the best entry of its part of the vocabulary.
__global__ void sample_partial_kernel(const float* __restrict__ logits, int vocab, int chunk,
                                      const float* __restrict__ temperature, const long long* __restrict__ seeds,
                                      const long long* __restrict__ counters, float* __restrict__ part_v,
                                      int* __restrict__ part_i) {
  __shared__ float sv[32];
  __shared__ int si[32];
  pdl_trigger();
  pdl_wait();
  const int row = blockIdx.y;
  const float* lr = logits + (size_t)row * vocab;
  const float temp = temperature[row];
  const unsigned long long seed = (unsigned long long)seeds[row];
  const unsigned long long counter = (unsigned long long)counters[row];
  const int begin = blockIdx.x * chunk, end = min(vocab, begin + chunk);
  float bv = -INFINITY;
  int bi = 0x7fffffff;
  for (int v = begin + threadIdx.x; v < end; v += blockDim.x) {
    float x = lr[v];
    if (temp > 0.f) x = x / temp - logf(-logf(jv_uniform(seed, counter, (unsigned long long)v)));
    take_better(bv, bi, x, v);
  }
  block_best(bv, bi, sv, si);
  if (threadIdx.x == 0) {
    part_v[(size_t)row * gridDim.x + blockIdx.x] = bv;
    part_i[(size_t)row * gridDim.x + blockIdx.x] = bi;
  }
}

// Stage 2: one warp per row over the chunk winners.
__global__ void sample_final_kernel(const float* __restrict__ part_v, const int* __restrict__ part_i, int n_chunks,
                                    int* __restrict__ out) {
  pdl_trigger();
  pdl_wait();
  const int row = blockIdx.x;
  float bv = -INFINITY;
  int bi = 0x7fffffff;
  for (int c = threadIdx.x; c < n_chunks; c += 32)
    take_better(bv, bi, part_v[(size_t)row * n_chunks + c], part_i[(size_t)row * n_chunks + c]);
  for (int o = 16; o > 0; o >>= 1)
    take_better(bv, bi, __shfl_xor_sync(0xffffffffu, bv, o), __shfl_xor_sync(0xffffffffu, bi, o));
  if (threadIdx.x == 0) out[row] = (bi == 0x7fffffff) ? 0 : bi;
}

// Chunks that the vocabulary is cut into (scratch: rows * chunks floats and ints).
JV_EXPORT int jv_sample_chunks(int vocab) {
  int c = (vocab + 2047) / 2048;
  return c < 1 ? 1 : (c > 128 ? 128 : c);
}

// logits: [rows, vocab] float; temperature: [rows] float; seeds, counters: [rows] int64;
// part_v/part_i: scratch of rows * jv_sample_chunks(vocab) elements; out: [rows] int32.
JV_EXPORT int jv_sample(const float* logits, int rows, int vocab, const float* temperature,
                        const long long* seeds, const long long* counters, float* part_v, int* part_i,
                        int* out, cudaStream_t stream) {
  if (rows == 0) return JV_OK;
  const int chunks = jv_sample_chunks(vocab);
  const int chunk = (vocab + chunks - 1) / chunks;
  if (jv_launch(sample_partial_kernel, dim3(chunks, rows), dim3(256), 0, stream, logits, vocab, chunk, temperature,
                seeds, counters, part_v, part_i) != JV_OK)
    return JV_ERR_LAUNCH;
  return jv_launch(sample_final_kernel, dim3(rows), dim3(32), 0, stream, (const float*)part_v, (const int*)part_i, chunks,
                   out);
}
