// Log-probabilities of given tokens, and the likeliest tokens of every row with theirs:
//   logprob(v) = x_v - largest - log(sum_w exp(x_w - largest))
// in one pass over the row, with the running largest logit and the sum relative to it in every thread (32 bits), joined in a
// fixed order.  The `top` likeliest tokens (equal ones in the order of their indices) are found as in vocab_row.h.
// A NaN counts as minus infinity; a row that holds nothing else has no likely tokens (every logprob is minus infinity);
// where the largest logit is infinite, the infinite ones share the probability.
#include <math.h>
#include "vocab_row.h"

namespace {

using namespace vocab;

struct ScoreParams {
  const void* logits;
  long long stride;
  int rows, vocab, blocks, top;
  const int* tokens;
  float* logprob;
  int* top_tokens;
  float* top_logprobs;
  int* status;
};

// log-probability of a logit, from the row's largest and the logarithm of its sum
__device__ __forceinline__ float logprob_of(float x, float largest, float log_sum) {
  if (largest == -INFINITY || x == -INFINITY) return -INFINITY;
  return x == largest ? -log_sum : (x - largest) - log_sum;
}

constexpr float LOG2E = 1.4426950408889634f;

template <typename T>
__global__ void __launch_bounds__(NT, 2) token_logprobs_kernel(const ScoreParams p) {
  extern __shared__ __align__(16) unsigned char memory[];
  Shared& sh = *reinterpret_cast<Shared*>(memory);
  pdl_trigger();
  pdl_wait();
  const int r = blockIdx.x / p.blocks;
  Reader<T> rd;
  const T* row = reinterpret_cast<const T*>(p.logits) + (size_t)r * p.stride;
  rd.start(row, p.vocab, p.blocks, &sh);
  // largest and sum of this thread's elements; what is no number (a NaN, infinity less infinity) adds nothing
  float m = -INFINITY, s = 0.f;
  rd.template each<8>([&](const auto& x, int) {
    constexpr int V = sizeof(x) / sizeof(float);
    float big = x[0];
#pragma unroll
    for (int i = 1; i < V; ++i) big = fmaxf(big, x[i]);
    if (big > m) {
      s *= exp2_fast((m - big) * LOG2E);
      m = big;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) s += exp2_fast(fmaxf(x[i] - m, -1000.f) * LOG2E);
  });
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float mb = warp_max(m);
  double sum = m == mb ? (double)s : (double)(s * exp2_fast((m - mb) * LOG2E));
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) { sh.warp_v[warp] = mb; sh.warp_d[0][warp] = sum; }
  rd.started();
  rd.exchange_largest(m, p.top == 0 ? 1 : min((p.top - 1) / p.blocks + 1, MOST_OF_GROUPS), [&] {
    if (threadIdx.x == 0) {
      float block = -INFINITY;
      for (int w = 0; w < WARPS; ++w) block = fmaxf(block, sh.warp_v[w]);
      double all = 0.;
      for (int w = 0; w < WARPS; ++w) all += sh.warp_v[w] == block ? sh.warp_d[0][w] : sh.warp_d[0][w] * (double)exp2_fast((sh.warp_v[w] - block) * LOG2E);
      for (int b = 0; b < p.blocks; ++b) rd.of(&sh.part[rd.rank][0], b)[0] = all;
    }
  });
  sum = 0.;
  for (int b = 0; b < p.blocks; ++b)
    sum += sh.largest[b] == rd.largest ? sh.part[b][0] : sh.part[b][0] * (double)exp2_fast((sh.largest[b] - rd.largest) * LOG2E);
  if (rd.largest == INFINITY) {                        // the infinite ones share the probability: how many they are
    float count = 0.f;
    rd.template each<4>([&](const auto& x, int) {
      constexpr int V = sizeof(x) / sizeof(float);
#pragma unroll
      for (int i = 0; i < V; ++i) count += x[i] == INFINITY ? 1.f : 0.f;
    });
    double a = count, none = 0.;
    rd.block_sums(a, none);
    rd.sync();                                         // the others have read the last sums
    if (threadIdx.x == 0)
      for (int b = 0; b < p.blocks; ++b) rd.of(&sh.part[rd.rank][0], b)[0] = a;
    rd.sync();
    sum = 0.;
    for (int b = 0; b < p.blocks; ++b) sum += sh.part[b][0];
  }
  const float log_sum = logf((float)sum);
  if (rd.rank == 0 && threadIdx.x == 0) {
    const int token = p.tokens[r];
    if (token < 0 || token >= p.vocab) {
      atomicOr(p.status, JV_STATUS_BAD_TOKEN);
      p.logprob[r] = NAN;
    } else {
      p.logprob[r] = logprob_of(clean(to_f32(row[token])), rd.largest, log_sum);
    }
  }
  if (p.top == 0) return;

  const int j = (p.top - 1) / p.blocks + 1;
  bool found = false;
  unsigned total = 0;
  if (j <= MOST_OF_GROUPS) {
    const float least = rd.bound;
    rd.template each<4>([&](const auto& x, int at) {
      constexpr int V = sizeof(x) / sizeof(float);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (clean(x[i]) >= least) rd.put(compose(clean(x[i]), at + i));
    });
    total = rd.send_list([] {});
    found = total <= (unsigned)LIST;
    if (!found && threadIdx.x == 0) sh.listed = 0;
  }
  if (!found) {
    Range range;
    const float wide = 6.f * (rd.largest - rd.bound);
    rd.scale = 0.f;
    rd.template narrow<false>((u64)KEY_LOWEST << INDEX_BITS, wide > 0.f ? (float)BINS / wide : 1.f, (unsigned)(LIST - p.top), range,
                              [](unsigned, double) { return true; }, [&](unsigned n, double) { return n < (unsigned)p.top; });
    total = rd.gather(range.lo, ~0ull);                // what lies above the range too: fewer than `top`
  }
  if (rd.rank != 0) return;
  rd.sort_list((int)total);
  for (int i = threadIdx.x; i < p.top; i += NT) {
    const u64 c = sh.list[i];
    p.top_tokens[(size_t)r * p.top + i] = index_of(c);
    p.top_logprobs[(size_t)r * p.top + i] = logprob_of(logit_of(c), rd.largest, log_sum);
  }
}

template <typename T>
int launch(const ScoreParams& p, cudaStream_t stream) {
  static bool done[JV_MAX_DEVICES] = {};
  if (!jv_once_per_device(done, [&] {
        return cudaFuncSetAttribute(token_logprobs_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared)) == cudaSuccess;
      }))
    return JV_ERR_UNSUPPORTED;
  return launch_clusters(token_logprobs_kernel<T>, dim3((unsigned)(p.rows * p.blocks)), dim3(NT), sizeof(Shared), p.blocks, stream, p);
}

}  // namespace

// logits: [rows, vocab] with `stride` elements between rows; tokens: [rows] int32; logprob: [rows]; top_tokens and
// top_logprobs: [rows, top], at most 128 and at most vocab.  `blocks`: as in jv_sample_filtered.
JV_EXPORT int jv_token_logprobs(const void* logits, int dtype, long long stride, int rows, int vocab, const int* tokens, int top,
                                float* logprob, int* top_tokens, float* top_logprobs, int* status, int blocks, cudaStream_t stream) {
  if (rows == 0) return JV_OK;
  if (vocab < 1 || vocab > MAX_VOCAB || rows > (1 << 28) || top < 0 || top > 128 || top > vocab) return JV_ERR_UNSUPPORTED;
  if (blocks < 0 || blocks > MOST_BLOCKS || (blocks & (blocks - 1))) return JV_ERR_UNSUPPORTED;
  ScoreParams p{logits, stride, rows, vocab, blocks ? blocks : row_blocks(rows, vocab), top, tokens, logprob, top_tokens, top_logprobs, status};
  JV_DISPATCH_DTYPE(dtype, T, return launch<T>(p, stream));
}
