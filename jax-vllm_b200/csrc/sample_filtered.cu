// One token per row of logits, drawn from softmax(logits / T) under filters.  With the tokens of a row in order of their
// logits (the lowest index first among equal ones), p = exp((x - largest) / T):
//   top_k > 0    only the first top_k tokens
//   min_p > 0    of these, the tokens with p >= min_p
//   top_p < 1    of these, the tokens before which less than top_p of their mass lies (the first always)
//   the token    argmax of x / T - log(-log(u)) over what is left, u = uniform(seed, counter, token id): a draw from the
//                softmax over it that depends on the row's own numbers only, as in sampling.cu and with its arithmetic
//   T == 0       the largest logit
// Every filter leaves the first tokens up to a boundary, so the kept ones are a range of the composed numbers of
// vocab_row.h, and only they need a random number.  Tokens with (largest - x) / T > 30 are left out from the start where
// there is a filter: their mass is below 1e-13 of the largest's, and -log(-log(u)) lies between -2.9 and 16.7 (but for the
// one u in 2^24 that rounds to 1), so that they cannot be drawn before the largest.
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

constexpr float DEEPEST = 30.f;
constexpr int FIRST_LOOK = 128;                        // tokens that the list is meant to hold where no count says how many

// The best score so far and its token.
struct Best { float v; int i; };

// Scores of one row: x / T - log(-log(u)) in the arithmetic of sampling.cu.
struct Scores {
  float temp, inv;
  u64 seed, counter;

  __device__ __forceinline__ float of(float x, int i) const {
    return x / temp - logf(-logf(jv_uniform(seed, counter, (u64)i)));
  }
  // A number that no score of x with the uniform number of token i is above, but for roundings: -log(-log(u)) <= -log(1 - u).
  __device__ __forceinline__ float most(float x, int i) const {
    const float w = 1.f - jv_uniform(seed, counter, (u64)i);
    return fmaf(x, inv, -0.69314718f * __log2f(w));
  }
};

// The best score among the elements of this thread with c >= cut.  What a token can reach at most is compared with the best
// score that the warp knows, less what the roundings of both may be (scores are off by a few 2^-24 of themselves, `most` by
// a few more and by what the approximate logarithm lacks): few tokens need their logarithms.
template <typename T>
__device__ __forceinline__ void draw(const Reader<T>& rd, const Scores& sc, u64 cut, Best& best) {
  const float low = logit_of(cut);
  float enough = -INFINITY;
  const int n = rd.n;
  for_row<2, true>(rd.row, n, rd.me, rd.all, [&](const auto& x, int at) {
    constexpr int V = sizeof(x) / sizeof(float);
    bool better = false;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float y = clean(x[i]);
      if (y >= low && at + i < n && !(sc.most(y, at + i) < enough) && compose(y, at + i) >= cut) {
        const float v = best.v;
        take_better(best.v, best.i, sc.of(y, at + i), at + i);
        better |= best.v > v;
      }
    }
    if constexpr (V > 1) {
      if (__any_sync(0xffffffffu, better)) {
        const float known = value_of(__reduce_max_sync(0xffffffffu, key_of(best.v)));
        enough = known - (1e-5f * fabsf(known) + 1e-3f);
      }
    }
  });
}

// Prefix sums over the first block of the masses of the list's first `listed` tokens, two a thread: before[j] lies before
// the token 2 * threadIdx.x + j.  Returns the sum of all.
__device__ __forceinline__ double masses_before(Shared& sh, int listed, float largest, float scale, double (&before)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double q[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = 2 * threadIdx.x + j;
    q[j] = i < listed ? (double)mass_of(logit_of(sh.list[i]), largest, scale) : 0.;
  }
  double s = q[0] + q[1];
  for (int o = 1; o < 32; o *= 2) {
    const double t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  double own = __shfl_up_sync(0xffffffffu, s, 1);
  if (lane == 0) own = 0.;
  __syncthreads();
  if (lane == 31) sh.warp_d[0][warp] = s;
  __syncthreads();
  double base = 0., total = 0.;
  for (int w = 0; w < WARPS; ++w) {
    if (w == warp) base = total;
    total += sh.warp_d[0][w];
  }
  before[0] = base + own;
  before[1] = before[0] + q[0];
  return total;
}

static_assert(LIST == 2 * NT, "two tokens of the list a thread");

template <typename T>
__global__ void __launch_bounds__(NT, 2) sample_filtered_kernel(const SampleParams p) {
  extern __shared__ __align__(16) unsigned char memory[];
  Shared& sh = *reinterpret_cast<Shared*>(memory);
  pdl_trigger();
  pdl_wait();
  const int r = blockIdx.x / p.blocks;
  Reader<T> rd;
  rd.start(reinterpret_cast<const T*>(p.logits) + (size_t)r * p.stride, p.vocab, p.blocks, &sh);
  const float temp = p.temperature[r];
  const bool hot = temp > 0.f;
  const int top_k = p.top_k[r];
  const float top_p = p.top_p[r], min_p = p.min_p[r];
  const bool by_count = hot && top_k > 0 && top_k < p.vocab, by_mass = hot && top_p < 1.f, by_share = hot && min_p > 0.f;
  const Scores sc{temp, 1.f / temp, (u64)p.seeds[r], (u64)p.counters[r]};

  Best best{-INFINITY, 0x7fffffff};
  bool in_list = false;                                // every kept token stands in the first block's list
  int listed = 0;                                      // first block: kept tokens of its sorted list

  if (!hot) {
    rd.template each<8>([&](const auto& x, int at) {
      constexpr int V = sizeof(x) / sizeof(float);
#pragma unroll
      for (int i = 0; i < V; ++i) take_better(best.v, best.i, clean(x[i]), at + i);
    });
    rd.started();
  } else if (!by_count && !by_mass && !by_share) {
    draw(rd, sc, (u64)KEY_LOWEST << INDEX_BITS, best);
    rd.started();
  } else {
    // a list of the first tokens serves counts up to what the blocks' groups can bound
    const int j = by_count ? (top_k - 1) / p.blocks + 1 : (FIRST_LOOK - 1) / p.blocks + 1;
    const bool countable = j <= MOST_OF_GROUPS;
    float m = -INFINITY;
    rd.template each<8>([&](const auto& x, int) {
      constexpr int V = sizeof(x) / sizeof(float);
#pragma unroll
      for (int i = 0; i < V; ++i) m = fmaxf(m, x[i]);
    });
    rd.started();
    rd.exchange_largest(m, countable ? j : GROUPS / 2, [] {});
    if (rd.largest == -INFINITY) {                     // nothing is left in the row
      if (rd.rank == 0 && threadIdx.x == 0) p.out[r] = 0;
      return;
    }
    rd.scale = 1.4426950408889634f * sc.inv;
    // the lowest logit that any filter may keep
    float low = rd.largest - DEEPEST * temp;
    if (!(low <= rd.largest)) low = rd.largest;        // (infinite numbers that make none)
    if (by_share) {
      const double least = (double)rd.largest + (double)temp * log((double)fminf(min_p, 1.f));
      if (!(least <= (double)rd.largest)) low = rd.largest;
      else low = fmaxf(low, __double2float_ru(least));
    }
    u64 cut = (u64)max(key_of(low + 0.f), KEY_LOWEST + 1) << INDEX_BITS;
    low = logit_of(cut);

    if (by_count || by_mass) {
      const auto bounded = [&](double q, double target) { return q == 0. || q < target; };
      const bool summed = by_mass && !by_count;        // the mass that counts is that of the whole row
      double mass_kept = 0.;
      bool found = false;
      if (countable) {
        const float least = fmaxf(rd.bound, low);
        float all_mass = 0.f, list_mass = 0.f;
        rd.template each<4>([&](const auto& x, int at) {
          constexpr int V = sizeof(x) / sizeof(float);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float y = x[i];                      // a NaN is no smaller than anything
            float q = 0.f;
            if (summed) {
              q = y >= low ? mass_of(y, rd.largest, rd.scale) : 0.f;
              all_mass += q;
            }
            if (y >= least) {
              list_mass += q;
              rd.put(compose(clean(y), at + i));
            }
          }
        });
        double a = all_mass, l = list_mass;
        if (summed) rd.block_sums(a, l);
        const unsigned total = rd.send_list([&] {
          if (threadIdx.x == 0 && summed)
            for (int b = 0; b < p.blocks; ++b) {
              rd.of(&sh.part[rd.rank][0], b)[0] = a;
              rd.of(&sh.part[rd.rank][0], b)[1] = l;
            }
        });
        found = total <= (unsigned)LIST;
        if (summed) {
          l = 0.;
          for (int b = 0; b < p.blocks; ++b) { mass_kept += sh.part[b][0]; l += sh.part[b][1]; }
          found = found && (least == low || l >= (double)top_p * mass_kept);
        }
        if (found) {
          if (rd.rank != 0) return;
          in_list = true;
          rd.sort_list((int)total);
          listed = by_count ? min(top_k, (int)total) : (int)total;
        } else if (threadIdx.x == 0) {
          sh.listed = 0;
        }
      }
      Range range{0, 0, 0., 0u, 0u};
      if (!found) {
        const float step = DEEPEST * temp, wide = 6.f * (rd.largest - rd.bound);
        const float per = (float)BINS / (wide > 0.f ? fminf(step, wide) : step);
        bool counted = false;
        if (by_count) {
          const auto whole = [&](unsigned n, double q) { mass_kept = q; return n > (unsigned)top_k; };
          if (rd.template narrow<true>(cut, per, LIST, range, whole, [&](unsigned n, double) { return n < (unsigned)top_k; })) {
            const unsigned total = rd.gather(range.lo, range.hi);
            in_list = range.count_above == 0;
            if (in_list && rd.rank != 0) return;
            if (rd.rank == 0) {
              rd.sort_list((int)total);
              listed = top_k - (int)range.count_above;
              double before[2];
              const double q = masses_before(sh, listed, rd.largest, rd.scale, before);
              if (threadIdx.x == 0) { sh.told = sh.list[listed - 1]; sh.told_mass = range.mass_above + q; }
            }
            if (!in_list) {
              rd.sync();
              cut = *rd.of(&sh.told, 0);
              mass_kept = *rd.of(&sh.told_mass, 0);
              rd.sync();                               // they are read: the first block may go on to other ones
            }
          }
          counted = true;
        }
        if (by_mass && !in_list) {
          double target = (double)top_p * mass_kept;
          rd.template narrow<true>(cut, per, LIST, range, [&](unsigned, double q) {
            if (!counted) { mass_kept = q; target = (double)top_p * q; }
            return true;
          }, [&](unsigned, double q) { return bounded(q, target); });
          const unsigned total = rd.gather(range.lo, range.hi);
          in_list = range.count_above == 0;
          if (in_list && rd.rank != 0) return;
          if (rd.rank == 0) {
            rd.sort_list((int)total);
            listed = (int)total;
          }
        }
      }
      if (by_mass && (rd.rank == 0 || !in_list)) {
        if (rd.rank == 0) {
          double before[2];
          const double q = masses_before(sh, listed, rd.largest, rd.scale, before);
          if (in_list && by_count) mass_kept = q;
          const double target = (double)top_p * mass_kept, above = in_list ? 0. : range.mass_above;
          int mine = 0;
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (2 * threadIdx.x + k < listed && bounded(above + before[k], target)) mine = 2 * threadIdx.x + k + 1;
          mine = __reduce_max_sync(0xffffffffu, mine);
          if ((threadIdx.x & 31) == 0) sh.warp_i[threadIdx.x >> 5] = mine;
          __syncthreads();
          listed = 0;
          for (int w = 0; w < WARPS; ++w) listed = max(listed, sh.warp_i[w]);
          if (threadIdx.x == 0) sh.told = sh.list[max(listed, 1) - 1];
          __syncthreads();
        }
        if (!in_list) {
          rd.sync();
          cut = *rd.of(&sh.told, 0);
        }
      }
    }
    if (in_list) {
      for (int i = threadIdx.x; i < listed; i += NT) {
        const u64 c = sh.list[i];
        take_better(best.v, best.i, sc.of(logit_of(c), index_of(c)), index_of(c));
      }
    } else {
      draw(rd, sc, cut, best);
    }
  }

  block_best(best.v, best.i, sh.warp_v, sh.warp_i);
  if (in_list) {
    if (threadIdx.x == 0) p.out[r] = best.i == 0x7fffffff ? 0 : best.i;
    return;
  }
  if (threadIdx.x == 0) { *rd.of(&sh.part_v[rd.rank], 0) = best.v; *rd.of(&sh.part_i[rd.rank], 0) = best.i; }
  rd.sync();
  if (rd.rank == 0 && threadIdx.x == 0) {
    for (int b = 0; b < p.blocks; ++b) take_better(best.v, best.i, sh.part_v[b], sh.part_i[b]);
    p.out[r] = best.i == 0x7fffffff ? 0 : best.i;
  }
}

template <typename T>
int launch(const SampleParams& p, cudaStream_t stream) {
  static bool done[JV_MAX_DEVICES] = {};
  if (!jv_once_per_device(done, [&] {
        return cudaFuncSetAttribute(sample_filtered_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared)) == cudaSuccess;
      }))
    return JV_ERR_UNSUPPORTED;
  return launch_clusters(sample_filtered_kernel<T>, dim3((unsigned)(p.rows * p.blocks)), dim3(NT), sizeof(Shared), p.blocks, stream, p);
}

}  // namespace

// logits: [rows, vocab] with `stride` elements between rows; the others one value a row (top_k int32, seeds and counters
// int64, the rest float).  out: [rows] int32.  `blocks`: blocks a row, a power of two up to 8 (0: by the sizes).
JV_EXPORT int jv_sample_filtered(const void* logits, int dtype, long long stride, int rows, int vocab, const float* temperature,
                                 const int* top_k, const float* top_p, const float* min_p, const long long* seeds,
                                 const long long* counters, int* out, int blocks, cudaStream_t stream) {
  if (rows == 0) return JV_OK;
  if (vocab < 1 || vocab > MAX_VOCAB || rows > (1 << 28) || blocks < 0 || blocks > MOST_BLOCKS || (blocks & (blocks - 1))) return JV_ERR_UNSUPPORTED;
  SampleParams p{logits, stride, rows, vocab, blocks ? blocks : row_blocks(rows, vocab), temperature, top_k, top_p, min_p, seeds, counters, out};
  JV_DISPATCH_DTYPE(dtype, T, return launch<T>(p, stream));
}
