// Log-probabilities of given tokens, and the likeliest tokens of every row with theirs:
//   logprob(v) = x_v - largest - log(sum_w exp(x_w - largest))
// in one pass over the row, with the running largest logit and the sum relative to it in every thread (32 bits), joined in a
// fixed order.  The `top` likeliest tokens (equal ones in the order of their indices) are found as in vocab_row.h.
// Bound by memory where rows are many: 1,024 of 151,936 logits in 95.6 us, 6.51 TB/s.  Eight rows 5.4 us: one pass of a cluster of
// eight blocks and a barrier.  With likely tokens a second pass and a sort (64 rows of 50,021 16-bit logits, 20 tokens: 10.7 us).
// A NaN counts as minus infinity; a row that holds nothing else has no likely tokens (every logprob is minus infinity);
// where the largest logit is infinite, the infinite ones share the probability.
#include <math.h>
#include <stddef.h>
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

// Largest and sum of this thread's elements; what is no number (a NaN, infinity less infinity) adds nothing.
template <typename T, int AHEAD> __device__ __noinline__ float2 largest_and_sum() {
  constexpr int VEC = 16 / (int)sizeof(T);
  float m = -INFINITY, s = 0.f;
  each<T, AHEAD>([&](const auto& x, int) {
    float big = x[0];
#pragma unroll
    for (int i = 1; i < VEC; ++i) big = fmaxf(big, x[i]);
    if (big > m) {
      s *= exp2_fast((m - big) * LOG2E);
      m = big;
    }
    float q[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) q[i] = exp2_fast(fmaxf(x[i] - m, -1000.f) * LOG2E);
    s += sum_of(q);
  });
  return make_float2(m, s);
}

template <typename T> __device__ __noinline__ float count_infinite() {
  float count = 0.f;
  each<T, 4>([&](const auto& x, int) {
#pragma unroll
    for (int i = 0; i < 16 / (int)sizeof(T); ++i) count += x[i] == INFINITY ? 1.f : 0.f;
  });
  return count;
}

// Puts the tokens at or above `least`; a NaN is minus infinity, which may be among them.
template <typename T> __device__ __noinline__ void list_first(float least) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const int n = shared().n;
  each<T, 4>([&](const auto& x, int at) {
    float big = x[0];
#pragma unroll
    for (int i = 1; i < VEC; ++i) big = fmaxf(big, x[i]);
    if (big >= least || least == -INFINITY) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float y = asked<false>(x[i], at + i, n);
        if (y >= least) put(compose(y, at + i));
      }
    }
  });
}

// Without likely tokens a block needs little memory and few registers: four of them to a multiprocessor, with two loads ahead in
// each (1,024 rows of 151,936 logits: 95.6 us; three blocks with four loads 111, two with six 101, two with eight 107).
template <typename T, bool TOP>
__global__ void __launch_bounds__(NT, TOP ? 2 : 4) token_logprobs_kernel(const ScoreParams p) {
  Shared& sh = shared();
  constexpr int VEC = 16 / (int)sizeof(T);
  pdl_trigger();
  pdl_wait();
  const int r = blockIdx.x / p.blocks;
  const T* row = reinterpret_cast<const T*>(p.logits) + (size_t)r * p.stride;
  begin(row, p.vocab, p.blocks);
  const float2 mine = largest_and_sum<T, TOP ? 6 : 2>();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float of_warp = warp_max(mine.x);
  double sum = mine.x == of_warp ? (double)mine.y : (double)(mine.y * exp2_fast((mine.x - of_warp) * LOG2E));
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) { sh.warp_v[warp] = of_warp; sh.warp_d[0][warp] = sum; }
  started();
  __syncthreads();
  if (warp == 0) {
    const float v = lane < WARPS ? sh.warp_v[lane] : -INFINITY, block = warp_max(v);
    sum = lane < WARPS ? v == block ? sh.warp_d[0][lane] : sh.warp_d[0][lane] * (double)exp2_fast((v - block) * LOG2E) : 0.;
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane < p.blocks) {
      of(&sh.part[sh.rank][0], lane)[0] = sum;
      if (!TOP) *of(&sh.largest_of[sh.rank], lane) = block;
    }
  }
  float largest = -INFINITY;
  if (TOP) {
    exchange_largest(mine.x, (p.top - 1) / p.blocks + 1);
    largest = sh.largest;
  } else {
    sync_row();
    for (int b = 0; b < p.blocks; ++b) largest = fmaxf(largest, sh.largest_of[b]);
    if (sh.rank != 0 && largest != INFINITY) return;
  }
  sum = 0.;
  for (int b = 0; b < p.blocks; ++b) {
    const float v = sh.largest_of[b];
    sum += v == largest ? sh.part[b][0] : sh.part[b][0] * (double)exp2_fast((v - largest) * LOG2E);
  }
  if (largest == INFINITY) {                           // the infinite ones share the probability: how many they are
    const double2 a = block_sums((double)count_infinite<T>(), 0.);
    sync_row();                                        // the others have read the last sums
    if (threadIdx.x == 0)
      for (int b = 0; b < p.blocks; ++b) of(&sh.part[sh.rank][0], b)[0] = a.x;
    sync_row();
    sum = 0.;
    for (int b = 0; b < p.blocks; ++b) sum += sh.part[b][0];
  }
  const float log_sum = logf((float)sum);
  if (sh.rank == 0 && threadIdx.x == 0) {
    const int token = p.tokens[r];
    if (token < 0 || token >= p.vocab) {
      atomicOr(p.status, JV_STATUS_BAD_TOKEN);
      p.logprob[r] = NAN;
    } else {
      p.logprob[r] = logprob_of(clean(to_f32(row[token])), largest, log_sum);
    }
  }
  if (!TOP) return;

  bool found = false;
  unsigned total = 0;
  if (countable((p.top - 1) / p.blocks + 1, p.blocks)) {
    list_first<T>(sh.bound);
    total = send_list();
    found = total <= (unsigned)LIST;
    if (!found && threadIdx.x == 0) sh.listed = 0;
  }
  if (!found) {
    const float wide = 6.f * (largest - sh.bound);
    if (threadIdx.x == 0) sh.scale = 0.f;
    __syncthreads();
    narrow<T, false>(LOWEST, wide > 0.f ? (float)BINS / wide : 1.f, (unsigned)(LIST - p.top), (double)p.top, -1., -1.);
    // what lies above the range too: fewer than `top`
    const u64 high = sh.range.hi;
    put_range<T, false, false>([&](const auto& x, int at) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (x[i] == x[i] && compose(clean(x[i]), at + i) > high) put(compose(clean(x[i]), at + i));
    });
    total = send_list();
  }
  if (sh.rank != 0) return;
  sort_list((int)total);
  for (int i = threadIdx.x; i < p.top; i += NT) {
    const u64 c = sh.list[i];
    p.top_tokens[(size_t)r * p.top + i] = index_of(c);
    p.top_logprobs[(size_t)r * p.top + i] = logprob_of(logit_of(c), largest, log_sum);
  }
}

template <typename T, bool TOP>
int launch(const ScoreParams& p, cudaStream_t stream) {
  constexpr int bytes = TOP ? (int)sizeof(Shared) : (int)offsetof(Shared, list);
  static bool done[JV_MAX_DEVICES] = {};
  if (!jv_once_per_device(done, [&] {
        return cudaFuncSetAttribute(token_logprobs_kernel<T, TOP>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
      }))
    return JV_ERR_UNSUPPORTED;
  return launch_clusters(token_logprobs_kernel<T, TOP>, dim3((unsigned)(p.rows * p.blocks)), dim3(NT), bytes, p.blocks, stream, p);
}

}  // namespace

// logits: [rows, vocab] with `stride` elements between rows; tokens: [rows] int32; logprob: [rows]; top_tokens and
// top_logprobs: [rows, top], at most 128 and at most vocab.  `blocks`: as in jv_sample_filtered.
JV_EXPORT int jv_token_logprobs(const void* logits, int dtype, long long stride, int rows, int vocab, const int* tokens, int top,
                                float* logprob, int* top_tokens, float* top_logprobs, int* status, int blocks, cudaStream_t stream) {
  if (rows == 0) return JV_OK;
  if (vocab < 1 || vocab > MAX_VOCAB || rows > (1 << 28) || top < 0 || top > 128 || top > vocab) return JV_ERR_UNSUPPORTED;
  if (blocks < 0 || blocks > MOST_BLOCKS || (blocks & (blocks - 1))) return JV_ERR_UNSUPPORTED;
  ScoreParams p{logits, stride, rows, vocab, blocks ? blocks : row_blocks(rows, (long long)vocab * (dtype == 0 ? 4 : 2)), top, tokens, logprob, top_tokens, top_logprobs, status};
  JV_DISPATCH_DTYPE(dtype, T, return top > 0 ? launch<T, true>(p, stream) : launch<T, false>(p, stream));
}
