// One token per row of logits, drawn from softmax(logits / T) under filters.  With the tokens of a row in order of their
// logits (the lowest index first among equal ones), p = exp((x - largest) / T):
//   top_k > 0    only the first top_k tokens
//   min_p > 0    of these, the tokens with p >= min_p
//   top_p < 1    of these, the tokens before which less than top_p of their mass lies (the first always)
//   the token    argmax of x / T - log(-log(u)) over what is left, u = uniform(seed, counter, token id): a draw from the
//                softmax over it that depends on the row's own numbers only, as in sampling.cu and with its arithmetic
//   T == 0       the largest logit
// Every filter leaves the first tokens up to a boundary, so the kept ones are a range of the composed numbers of
// vocab_row.h, and only they need a random number.
#include <math.h>
#include "sampling.h"
#include "vocab_row.h"

namespace {

using namespace vocab;

struct SampleParams {
  const void* logits;
  long long stride;                                    // elements from one row to the next
  int rows, vocab, blocks;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const long long* seeds;
  const long long* counters;
  int* out;
};

// Exclusive prefix sum over the block of v (one value a thread); `warps`: NT / 32 numbers of shared memory.
template <int NT> __device__ __forceinline__ u64 block_before(u64 v, u64* warps) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 s = v;
  for (int o = 1; o < 32; o *= 2) {
    const u64 t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  __syncthreads();
  if (lane == 31) warps[warp] = s;
  __syncthreads();
  u64 base = 0;
  for (int w = 0; w < warp; ++w) base += warps[w];
  return base + s - v;
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT) sample_filtered_kernel(const SampleParams p) {
  __shared__ Shared<NT> sh;
  pdl_trigger();
  pdl_wait();
  const int r = blockIdx.x / p.blocks;
  Reader<T, NT> rd;
  rd.start(reinterpret_cast<const T*>(p.logits) + (size_t)r * p.stride, p.vocab, p.blocks, &sh);
  const float temp = p.temperature[r];
  const bool hot = temp > 0.f;
  const int top_k = p.top_k[r];
  const float top_p = p.top_p[r], min_p = p.min_p[r];
  const u64 seed = (u64)p.seeds[r], counter = (u64)p.counters[r];
  const bool by_count = hot && top_k > 0 && top_k < p.vocab, by_mass = hot && top_p < 1.f, by_share = hot && min_p > 0.f;

  const auto score = [&](float x, int i) {
    return hot ? x / temp - logf(-logf(jv_uniform(seed, counter, (u64)i))) : x;
  };
  float bv = -INFINITY;
  int bi = 0x7fffffff;
  bool in_list = false;                                // every kept token stands in the first block's list

  if (!by_count && !by_mass && !by_share) {
    rd.template each<4>([&](float x, int i) { take_better(bv, bi, score(x, i), i); });
    rd.sync();                                         // every block of the cluster runs: their memory may be written
  } else {
    rd.find_largest();
    rd.scale = 1.4426950408889634f / temp;
    u64 cut = 0;
    if (by_share) {
      double least = (double)rd.largest + (double)temp * log((double)fminf(min_p, 1.f));
      if (!(least <= (double)rd.largest)) least = (double)rd.largest;      // infinite numbers that make none
      cut = (u64)key_of(__double2float_ru(least) + 0.f) << INDEX_BITS;
    }
    u64 mass_kept = 0;                                 // of the tokens that the count and the share leave
    bool known = false;
    int listed = 0;                                    // first block: tokens kept in its sorted list
    Range range;
    if (by_count) {
      const auto whole = [&](unsigned n, u64 q) { mass_kept = q; return n > (unsigned)top_k; };
      if (rd.template narrow<true>(cut, 1.f / temp, LIST, range, whole, [&](unsigned n, u64) { return n < (unsigned)top_k; })) {
        rd.gather(range.lo, range.hi);
        in_list = range.count_above == 0;
        if (rd.rank == 0) {
          rd.sort_list();
          listed = top_k - (int)range.count_above;
          u64 q = 0;
          for (int i = threadIdx.x; i < listed; i += NT) q += mass_of(logit_of(sh.list[i]), rd.largest, rd.scale);
          const u64 before = block_before<NT>(q, sh.scan);
          if (threadIdx.x == NT - 1) { sh.told[0] = sh.list[listed - 1]; sh.told[1] = range.mass_above + before + q; }
          __syncthreads();
        }
        if (in_list && rd.rank != 0) return;
        if (!in_list) rd.sync();
        const u64* told = rd.of(&sh.told[0], 0);
        cut = told[0];
        mass_kept = told[1];
      }
      known = true;
    }
    if (by_mass) {
      double target = (double)top_p * (double)mass_kept;
      const auto before = [&](unsigned, u64 q) { return q == 0 || (double)q < target; };
      bool found = in_list;
      if (in_list) {
        range.mass_above = 0;
      } else {
        const auto whole = [&](unsigned, u64 q) {
          if (!known) { mass_kept = q; target = (double)top_p * (double)q; }
          return true;
        };
        if (rd.rank == 0 && threadIdx.x == 0) sh.listed = 0;   // the list may have served the count; the levels' barriers follow
        rd.template narrow<true>(cut, 1.f / temp, LIST, range, whole, before);
        rd.gather(range.lo, range.hi);
        in_list = range.count_above == 0;
        if (rd.rank == 0) listed = rd.sort_list();
      }
      if (rd.rank == 0) {
        // the kept tokens of the list: thread t has the places PER t .. PER t + PER - 1
        constexpr int PER = LIST / NT;
        u64 q[PER], sum = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const int i = threadIdx.x * PER + j;
          q[j] = i < listed ? mass_of(logit_of(sh.list[i]), rd.largest, rd.scale) : 0;
          sum += q[j];
        }
        u64 at = range.mass_above + block_before<NT>(sum, sh.scan);
        int mine = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          if (threadIdx.x * PER + j < listed && before(0, at)) mine = threadIdx.x * PER + j + 1;
          at += q[j];
        }
        for (int o = 16; o > 0; o >>= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
        if ((threadIdx.x & 31) == 0) sh.warp_i[threadIdx.x >> 5] = mine;
        __syncthreads();
        listed = 0;
        for (int w = 0; w < NT / 32; ++w) listed = max(listed, sh.warp_i[w]);
        if (threadIdx.x == 0) sh.told[2] = sh.list[max(listed, 1) - 1];
        __syncthreads();
      }
      if (in_list && rd.rank != 0) return;
      if (!found && !in_list) {
        rd.sync();
        cut = *rd.of(&sh.told[2], 0);
      }
    }
    if (in_list) {
      for (int i = threadIdx.x; i < listed; i += NT) {
        const u64 c = sh.list[i];
        take_better(bv, bi, score(logit_of(c), index_of(c)), index_of(c));
      }
    } else {
      rd.template each<4>([&](float x, int i) { if (compose(x, i) >= cut) take_better(bv, bi, score(x, i), i); });
    }
  }

  block_best(bv, bi, sh.warp_v, sh.warp_i);
  if (in_list) {
    if (threadIdx.x == 0) p.out[r] = bi == 0x7fffffff ? 0 : bi;
    return;
  }
  if (threadIdx.x == 0) { *rd.of(&sh.part_v[rd.rank], 0) = bv; *rd.of(&sh.part_i[rd.rank], 0) = bi; }
  rd.sync();
  if (rd.rank == 0 && threadIdx.x == 0) {
    for (int b = 0; b < p.blocks; ++b) take_better(bv, bi, sh.part_v[b], sh.part_i[b]);
    p.out[r] = bi == 0x7fffffff ? 0 : bi;
  }
}

template <typename T>
int launch(const SampleParams& p, cudaStream_t stream) {
  constexpr int NT = 256;
  return launch_clusters(sample_filtered_kernel<T, NT>, dim3((unsigned)(p.rows * p.blocks)), dim3(NT), p.blocks, stream, p);
}

}  // namespace

// logits: [rows, vocab] with `stride` elements between rows; the others one value a row (top_k int32, seeds and counters
// int64, the rest float).  out: [rows] int32.
JV_EXPORT int jv_sample_filtered(const void* logits, int dtype, long long stride, int rows, int vocab, const float* temperature,
                                 const int* top_k, const float* top_p, const float* min_p, const long long* seeds,
                                 const long long* counters, int* out, cudaStream_t stream) {
  if (rows == 0) return JV_OK;
  if (vocab < 1 || vocab > MAX_VOCAB) return JV_ERR_UNSUPPORTED;
  SampleParams p{logits, stride, rows, vocab, 8, temperature, top_k, top_p, min_p, seeds, counters, out};
  JV_DISPATCH_DTYPE(dtype, T, return launch<T>(p, stream));
}
