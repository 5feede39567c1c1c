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

template <typename T, int NT>
__global__ void __launch_bounds__(NT) token_logprobs_kernel(const ScoreParams p) {
  __shared__ Shared<NT> sh;
  pdl_trigger();
  pdl_wait();
  const int r = blockIdx.x / p.blocks;
  Reader<T, NT> rd;
  const T* row = reinterpret_cast<const T*>(p.logits) + (size_t)r * p.stride;
  rd.start(row, p.vocab, p.blocks, &sh);
  if (threadIdx.x == 0) sh.listed = 0;
  // largest and sum of this thread's elements
  float m = -INFINITY, s = 0.f;
  rd.template each<8>([&](float x, int) {
    if (x > m) { s = (m == -INFINITY ? 0.f : s * __expf(m - x)); m = x; }
    s += x == m ? 1.f : __expf(x - m);
  });
  const auto join = [](float& m, float& s, float om, float os) {
    const float big = fmaxf(m, om);
    s = (m == big ? s : s * expf(m - big)) + (om == big ? os : os * expf(om - big));
    m = big;
  };
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, s, o);
    join(m, s, om, os);
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) { sh.warp_v[warp] = m; sh.warp_i[warp] = __float_as_int(s); }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < NT / 32; ++w) join(m, s, sh.warp_v[w], __int_as_float(sh.warp_i[w]));
    sh.block_largest = m;
    sh.part_v[0] = s;
  }
  rd.sync();
  m = -INFINITY;
  s = 0.f;
  for (int b = 0; b < p.blocks; ++b) join(m, s, *rd.of(&sh.block_largest, b), *rd.of(&sh.part_v[0], b));
  rd.largest = m;
  rd.scale = 1.f;
  const float log_sum = logf(s);
  if (rd.rank == 0 && threadIdx.x == 0) {
    const int token = p.tokens[r];
    if (token < 0 || token >= p.vocab) {
      atomicOr(p.status, JV_STATUS_BAD_TOKEN);
      p.logprob[r] = NAN;
    } else {
      p.logprob[r] = logprob_of(clean(to_f32(row[token])), m, log_sum);
    }
  }
  if (p.top == 0) {
    rd.sync();                                         // the others' sums are read: they may leave
    return;
  }
  Range range{0, ~0ull, 0, 0, 0};
  rd.template narrow<false>(0, 1.f, (unsigned)(LIST - p.top), range, [&](unsigned n, u64) { return n > (unsigned)LIST; },
                            [&](unsigned n, u64) { return n < (unsigned)p.top; });
  rd.gather(range.lo, ~0ull);                          // what lies above the range too: fewer than `top`
  if (rd.rank != 0) return;
  rd.sort_list();
  for (int i = threadIdx.x; i < p.top; i += NT) {
    const u64 c = sh.list[i];
    p.top_tokens[(size_t)r * p.top + i] = index_of(c);
    p.top_logprobs[(size_t)r * p.top + i] = logprob_of(logit_of(c), m, log_sum);
  }
}

template <typename T>
int launch(const ScoreParams& p, cudaStream_t stream) {
  constexpr int NT = 256;
  return launch_clusters(token_logprobs_kernel<T, NT>, dim3((unsigned)(p.rows * p.blocks)), dim3(NT), p.blocks, stream, p);
}

}  // namespace

// logits: [rows, vocab] with `stride` elements between rows; tokens: [rows] int32; logprob: [rows]; top_tokens and
// top_logprobs: [rows, top], at most 128 and at most vocab.
JV_EXPORT int jv_token_logprobs(const void* logits, int dtype, long long stride, int rows, int vocab, const int* tokens, int top,
                                float* logprob, int* top_tokens, float* top_logprobs, int* status, cudaStream_t stream) {
  if (rows == 0) return JV_OK;
  if (vocab < 1 || vocab > MAX_VOCAB || top < 0 || top > 128 || top > vocab) return JV_ERR_UNSUPPORTED;
  ScoreParams p{logits, stride, rows, vocab, 8, top, tokens, logprob, top_tokens, top_logprobs, status};
  JV_DISPATCH_DTYPE(dtype, T, return launch<T>(p, stream));
}
