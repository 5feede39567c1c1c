// One token per row of logits, drawn from softmax(logits / T) under filters.  With the tokens of a row in order of their
// logits (the lowest index first among equal ones), p = exp((x - largest) / T):
//   top_k > 0    only the first top_k tokens
//   min_p > 0    of these, the tokens with p >= min_p
//   top_p < 1    of these, the tokens before which less than top_p of their mass lies (the first always)
//   the token    argmax of x / T - log(-log(u)) over what is left, u = uniform(seed, counter, token id): a draw from the
//                softmax over it that depends on the row's own numbers only, as in sampling.cu and with its arithmetic
//   T == 0       the largest logit
// Every filter leaves the first tokens up to a boundary, so the kept ones are a range of the composed numbers of
// vocab_row.h, and only they need a random number.  Counts and shares have exact boundaries, the same in every batch.  The
// boundary of a mass is a comparison of sums, 32-bit within a thread (columns of 64 bits would fill the shared memory of a
// multiprocessor with one block); which logits a thread adds follows the number of blocks that read the row, hence the number of rows,
// and the row's place beside 16-byte boundaries.  So a token whose border lies within the rounding of the sums (6e-5 of the mass at
// most, about 2e-8 as restated on the host) may be kept in one batch and left out in another: none of 10,240 even rows of
// 32,003 logits drew another token with eight blocks than with one.  Tokens with (largest - x) / T > 30 are left out from the start where
// there is a filter: their mass is below 1e-13 of the largest's, and -log(-log(u)) lies between -2.9 and 16.7, so that they
// cannot be drawn before the largest.
//
// What bounds it, and what it takes (alone on the device, calls behind one another): one row of 151,936 logits 10.4 us, a chain of
// two passes over 76 KB a block (2.4 and 1.8 us) and two barriers of the cluster with what they carry (2.3 and 1.5 us); 256 rows of which
// the first 40 tokens are kept 36.6 us, the memory's 23.8 and the ends of the rows' chains, which nothing covers; 64 nearly even
// rows under top-p 77 us, instructions: 5 a logit for the largest, 17 for each of two levels, 46 for the random number of a kept one.
// Tried and dropped: one pass with a bound from the row's start for clusters too (as a block by itself does it: 18 -> 31
// instructions a logit), the next round's loads ahead of a round (copies between registers: 46 -> 58 a drawn logit), and for
// top-p a draw from all tokens, repeated among those before it while it is not kept (138 -> 109 a logit, but a step waits for the
// row with the most rounds: 77 -> 100 us).
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
// Tokens that the list is meant to hold where no count says how many.  (64 rows of 151,936 with 200 peaks under top-p: 21.5 us; a list
// meant for 64 takes 19.1 where it does and 34 to 41 where it does not, one for 256 takes 22.9.)
constexpr int FIRST_LOOK = 128;
constexpr float LOG2E = 1.4426950408889634f;

// The best score so far and its token.
struct Best { float v; int i; };

// Scores of one row: x / T - log(-log(u)) in the arithmetic of sampling.cu.
struct Scores {
  float temp, per;                                     // T and log2(e) / T
  u64 base;

  __device__ __forceinline__ float of(float x, int i) const {
    return x / temp - logf(-logf(jv_uniform_of(jv_draw_bits(base, (unsigned)i))));
  }
  // Whether the score of token i may reach `enough` (given as enough * log2(e)), but for roundings: -log(-log(u)) <= -log(1 - u),
  // and 1 - u is no less than what the first 23 random bits leave of it.
  __device__ __forceinline__ bool may_reach(float x, int i, float enough2) const {
    return bits_may_reach(x, jv_draw_first23(base, (unsigned)i), enough2);
  }
  __device__ __forceinline__ bool bits_may_reach(float x, unsigned first23, float enough2) const {
    const float w = (2.f - 1.1920929e-7f) - __uint_as_float(0x3f800000u | first23);
    return !(w > exp2_fast(fmaf(x, per, -enough2)));
  }
};

// The best score of the tokens that it is called for, by whole warps.  What a token can reach at most is compared with the best
// score that the block knows (which a warp may see late: it only saves work), less what the roundings of both may be (scores
// are off by a few 2^-24 of themselves, the bound by a few more and by what the approximate exponential lacks): few tokens
// need their logarithms.
struct Draw {
  const Scores sc;
  Best best{-INFINITY, 0x7fffffff};
  float enough2 = -INFINITY;
  int queued = 0;

  __device__ __forceinline__ Draw(const Scores& sc_) : sc(sc_) {}

  // One token a lane, NaN: none.
  __device__ __forceinline__ void one(float y, int i) {
    const bool may = y == y && sc.may_reach(y, i, enough2);
    if (!__any_sync(0xffffffffu, may)) return;
    if (may) take_better(best.v, best.i, sc.of(y, i), i);
    const unsigned known = __reduce_max_sync(0xffffffffu, key_of(best.v));
    unsigned of_block = known;
    if ((threadIdx.x & 31) == 0) of_block = max(known, atomicMax(&shared().best_key, known));
    const float enough = value_of(__shfl_sync(0xffffffffu, of_block, 0));
    enough2 = (enough - (1e-5f * fabsf(enough) + 1e-3f)) * LOG2E;
  }
  // A vector a lane, of every token that is a number.  The largest logit and the largest random number bound them all.
  template <int VEC> __device__ __forceinline__ void all(const float (&x)[VEC], int at) {
    float big = x[0];
    unsigned luck = 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      big = fmaxf(big, x[i]);
      luck = max(luck, jv_draw_first23(sc.base, (unsigned)(at + i)));
    }
    if (!__any_sync(0xffffffffu, big == big && sc.bits_may_reach(big, luck, enough2))) return;
#pragma unroll 1
    for (int i = 0; i < VEC; ++i) {
      float y = x[0];
#pragma unroll
      for (int k = 1; k < VEC; ++k) y = i == k ? x[k] : y;
      one(y, at + i);
    }
  }
  // A vector a lane, of the tokens that are `kept`: where they are few, they wait until the warp has 32 of them.
  template <int VEC, typename K> __device__ __forceinline__ void some(const float (&x)[VEC], int at, K&& kept) {
    unsigned who[VEC];
    int number = 0;
    bool is[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      is[i] = kept(x[i], at + i);
      who[i] = __ballot_sync(0xffffffffu, is[i]);
      number += __popc(who[i]);
    }
    if (number >= 20 * VEC) {
      float y[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) y[i] = is[i] ? x[i] : nan_f();
      all(y, at);
      return;
    }
    if (number == 0) return;
    uint2* queue = shared().queue[threadIdx.x >> 5];
    const unsigned before = (1u << (threadIdx.x & 31)) - 1;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if (is[i]) queue[queued + __popc(who[i] & before)] = make_uint2(__float_as_uint(x[i]), (unsigned)(at + i));
      queued += __popc(who[i]);
    }
    while (queued >= 32) take(32);
  }
  // The last n of the warp's queue.
  __device__ __forceinline__ void take(int n) {
    __syncwarp();
    queued -= n;
    const int lane = threadIdx.x & 31;
    const uint2 token = lane < n ? shared().queue[threadIdx.x >> 5][queued + lane] : make_uint2(0x7fffffffu, 0u);
    __syncwarp();
    one(__uint_as_float(token.x), (int)token.y);
  }
  __device__ __forceinline__ void finish() {
    if (queued > 0) take(queued);
  }
};

// The best score of all tokens of the row.
template <typename T> __device__ __noinline__ Best draw_from_all(const Scores sc) {
  Draw draw(sc);
  each<T, 2, true>([&](const auto& x, int at) { draw.all(x, at); });
  return draw.best;
}
// The best score of the tokens with c >= cut, which no token of an equal logit is below.
template <typename T> __device__ __noinline__ Best draw_from(const Scores sc, u64 cut) {
  Draw draw(sc);
  const float lowest = logit_of(cut);
  each<T, 2, true>([&](const auto& x, int at) {
    draw.some(x, at, [&](float y, int) { return y >= lowest; });
  });
  draw.finish();
  return draw.best;
}
// Puts the tokens of the range and, with `score`, gives the best score of those above it.
template <typename T> __device__ __noinline__ Best draw_above(const Scores sc, bool score) {
  Draw draw(sc);
  const u64 high = shared().range.hi;
  const float next = value_of((unsigned)(high >> INDEX_BITS) + 1);     // the smallest logit above the range's
  const bool equal = (high & (MAX_VOCAB - 1)) != MAX_VOCAB - 1;        // tokens of the range's largest logit lie above it too
  put_range<T, true, true>([&](const auto& x, int at) {
    if (score) draw.some(x, at, [&](float y, int i) { return y >= next || (equal && compose(clean(y), i) > high); });
  });
  draw.finish();
  return draw.best;
}
template <typename T> __device__ __noinline__ Best largest_of_row() {
  Best best{-INFINITY, 0x7fffffff};
  each<T, 8>([&](const auto& x, int at) {
#pragma unroll
    for (int i = 0; i < 16 / (int)sizeof(T); ++i) take_better(best.v, best.i, x[i], at + i);
  });
  return best;
}

// The second pass of a row whose first tokens a list may hold: puts those at or above `least` in it.  SUMMED: returns the masses
// of the tokens from `low` up, and of those that are put.
template <typename T, bool SUMMED> __device__ __noinline__ float2 list_first(float low, float least) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const float largest = shared().largest, scale = shared().scale;
  float all = 0.f, listed = 0.f;
  each<T, 4>([&](const auto& x, int at) {
    float big = x[0];                                  // (a NaN is passed over)
#pragma unroll
    for (int i = 1; i < VEC; ++i) big = fmaxf(big, x[i]);
    if (SUMMED) {
      float q[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) q[i] = x[i] >= low ? exp2_fast(-(below(x[i], largest) * scale)) : 0.f;
      all += sum_of(q);
    }
    if (big >= least) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (x[i] >= least) {
          if (SUMMED) listed += exp2_fast(-(below(x[i], largest) * scale));
          put(compose(clean(x[i]), at + i));
        }
    }
  });
  return make_float2(all, listed);
}

// First block only: how many of the list's first m tokens have less than `part` of the mass that counts before them, with `above`
// before the first: `mass`, or the list's where that is negative.  `sum`: the list's.  A list of no more than 128 tokens is
// one warp's work.
static __device__ __noinline__ int kept_by_mass(int m, double above, double part, double mass, double& sum) {
  constexpr int PER = LIST / NT;
  Shared& sh = shared();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float largest = sh.largest, scale = sh.scale;
  const int warps = m <= 32 * PER ? 1 : WARPS;
  double to = 0., q[PER], s = 0.;
  if (warp < warps) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = PER * threadIdx.x + j;
      q[j] = i < m ? (double)exp2_fast(-(below(logit_of(sh.list[i]), largest) * scale)) : 0.;
      s += q[j];
    }
    to = s;
    for (int o = 1; o < 32; o *= 2) {
      const double t = __shfl_up_sync(0xffffffffu, to, o);
      if (lane >= o) to += t;
    }
    if (lane == 31) sh.warp_d[0][warp] = to;
  }
  __syncthreads();
  double before = above, total = 0.;
  for (int w = 0; w < warps; ++w) {
    if (w < warp) before += sh.warp_d[0][w];
    total += sh.warp_d[0][w];
  }
  sum = total;
  if (warp < warps) {
    const double first = __shfl_up_sync(0xffffffffu, to, 1), end = part * (mass < 0. ? total : mass);
    if (lane > 0) before += first;
    int mine = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = PER * threadIdx.x + j;
      if (i < m && (before == 0. || before < end)) mine = i + 1;
      before += q[j];
    }
    mine = __reduce_max_sync(0xffffffffu, mine);
    if (lane == 0) sh.warp_i[warp] = mine;
  }
  __syncthreads();
  int kept = 0;
  for (int w = 0; w < warps; ++w) kept = max(kept, sh.warp_i[w]);
  __syncthreads();
  return kept;
}

// A row with filters.  Returns the first token number that is kept where all tokens from there on are still to be drawn from;
// 0 where the first block has the others' best scores (with `drawn`) and `listed` kept tokens in its list; ~0 where nothing
// is left to do for this block.
template <typename T>
__device__ __forceinline__ u64 filtered(const SampleParams& p, const Scores& sc, int top_k, float top_p, float min_p, Best& best, int& listed,
                                        bool& drawn) {
  Shared& sh = shared();
  const float temp = sc.temp;
  const bool by_count = top_k > 0 && top_k < p.vocab, by_mass = top_p < 1.f, by_share = min_p > 0.f;
  // a list of the first tokens serves counts up to what the blocks' threads can bound
  const int j = ((by_count ? top_k : min(FIRST_LOOK, FEW * p.blocks)) - 1) / p.blocks + 1;
  const bool can_list = countable(j, p.blocks);
  const bool summed = by_mass && !by_count;            // the mass that counts is that of the whole row
  // one block a row: one pass, unless the mass that counts depends on the largest logit
  const bool once = p.blocks == 1 && (by_count || by_mass) && can_list && fits_once<T>(j, p.vocab) && !(summed && by_share);
  if (threadIdx.x == 0) sh.scale = fminf(fmaxf(sc.per, 1e-37f), 3e38f);
  float2 mine{-INFINITY, 0.f};
  if (once) {
    __syncthreads();
    mine = summed ? put_once<T, true>(j, DEEPEST * temp) : put_once<T, false>(j, DEEPEST * temp);
  } else {
    mine.x = my_largest<T>();
  }
  started();
  exchange_largest(mine.x, can_list ? j : FEW);
  const float largest = sh.largest;
  if (largest == -INFINITY) return ~0ull;              // nothing is left in the row (the output says 0 already)
  // the lowest logit that any filter may keep
  float low = largest - DEEPEST * temp;
  if (!(low <= largest)) low = largest;                // (infinite numbers that make none)
  if (by_share) {
    const double least = (double)largest + (double)temp * log((double)fminf(min_p, 1.f));
    if (!(least <= (double)largest)) low = largest;
    else low = fmaxf(low, __double2float_ru(least));
  }
  u64 cut = (u64)max(key_of(low + 0.f), KEY_LOWEST + 1) << INDEX_BITS;
  if (!by_count && !by_mass) return cut;
  low = logit_of(cut);

  const float least = fmaxf(sh.bound, low);
  unsigned total = LIST + 1;
  bool found = false;
  double mass = -1., list_mass = 0.;                   // mass: of what the count and the share leave, where it is known
  if (once) {
    total = keep_list(least);
    found = total <= (unsigned)LIST;
    if (found && summed) {
      const double2 a = block_sums((double)(mine.x == largest ? mine.y : mine.y * exp2_fast(-(below(mine.x, largest) * sh.scale))), 0.);
      if (threadIdx.x == 0) sh.part[0][0] = a.x;
      __syncthreads();
      mass = sh.part[0][0];
    }
  } else if (can_list && !(summed && largest - sh.bound < 3.f * temp)) {
    // Of nearly even logits, those from the bound up would hold too little of the mass.  (64 rows under top-p: even ones 73.6 us, 81.4
    // if the list is tried all the same; leaving it out up to 6 T, rows with 200 peaks take 35.5 instead of 21.7, rows of a spread
    // of 2.2 without peaks 62 instead of 70.)
    if (summed) {
      const float2 q = list_first<T, true>(low, least);
      const double2 a = block_sums((double)q.x, (double)q.y);
      if (threadIdx.x == 0)
        for (int b = 0; b < p.blocks; ++b) {
          of(&sh.part[sh.rank][0], b)[0] = a.x;
          of(&sh.part[sh.rank][0], b)[1] = a.y;
        }
    } else {
      list_first<T, false>(low, least);
    }
    total = send_list();
    found = total <= (unsigned)LIST;
    if (summed) {
      mass = 0.;
      for (int b = 0; b < p.blocks; ++b) { mass += sh.part[b][0]; list_mass += sh.part[b][1]; }
      found = found && (least == low || list_mass >= (double)top_p * mass);
    }
  }
  if (found) {
    if (sh.rank != 0) return ~0ull;
    sort_list((int)total);
    listed = by_count ? min(top_k, (int)total) : (int)total;
    if (by_mass) listed = kept_by_mass(listed, 0., (double)top_p, mass, list_mass);
    if (!(once && summed) || least == low || list_mass >= (double)top_p * mass) return 0;
  }
  if (threadIdx.x == 0) sh.listed = 0;

  // The first level's bins: from the largest logit to six times as deep as the bound of few tokens.  (64 even rows: top-p 0.9 73.6 us, with
  // three times as deep 92.3, with twelve 76.8; the first 1,500 tokens 52.9, 46.5 and 59.2.)
  const float step = DEEPEST * temp, wide = 6.f * (largest - sh.bound);
  const float per = (float)BINS / (wide > 0.f ? fminf(step, wide) : step);
  if (by_count) {                                      // the boundary by count
    if (!narrow<T, false>(cut, per, LIST, (double)top_k, -1., (double)top_k)) {
      if (!by_mass) return cut;                        // no more tokens than the count leaves
    } else {
      const double above = sh.range.above;
      best = draw_above<T>(sc, !by_mass);
      total = send_list();
      const bool last = !by_mass || above == 0.;
      if (!by_mass) {
        block_best(best.v, best.i, sh.warp_v, sh.warp_i);
        if (threadIdx.x == 0) { *of(&sh.part_v[sh.rank], 0) = best.v; *of(&sh.part_i[sh.rank], 0) = best.i; }
        sync_row();
        drawn = true;
      }
      if (last && sh.rank != 0) return ~0ull;
      if (sh.rank == 0) {
        sort_list((int)total);
        listed = top_k - (int)above;
      }
      if (last) {
        if (by_mass) listed = kept_by_mass(listed, 0., (double)top_p, -1., list_mass);
        return 0;
      }
      if (sh.rank == 0 && threadIdx.x == 0) sh.told = sh.list[listed - 1];
      sync_row();
      cut = *of(&sh.told, 0);
      sync_row();                                      // it is read: the first block may go on to another one
    }
  }
  narrow<T, true>(cut, per, LIST, 0., (double)top_p, -1.);
  best = draw_above<T>(sc, true);
  block_best(best.v, best.i, sh.warp_v, sh.warp_i);
  if (threadIdx.x == 0) { *of(&sh.part_v[sh.rank], 0) = best.v; *of(&sh.part_i[sh.rank], 0) = best.i; }
  total = send_list();
  drawn = true;
  if (sh.rank != 0) return ~0ull;
  sort_list((int)total);
  listed = kept_by_mass((int)total, sh.range.above, (double)top_p, sh.range.all, list_mass);
  return 0;
}

template <typename T>
__global__ void __launch_bounds__(NT, 2) sample_filtered_kernel(const SampleParams p) {
  Shared& sh = shared();
  pdl_trigger();
  pdl_wait();
  const int r = blockIdx.x / p.blocks;
  const float temp = p.temperature[r];
  const int top_k = p.top_k[r];
  const float top_p = p.top_p[r], min_p = p.min_p[r];
  const Scores sc{temp, LOG2E / temp, jv_draw_base((u64)p.seeds[r], (u64)p.counters[r])};
  begin(reinterpret_cast<const T*>(p.logits) + (size_t)r * p.stride, p.vocab, p.blocks);
  if (sh.rank == 0 && threadIdx.x == 0) p.out[r] = 0;
  Best best{-INFINITY, 0x7fffffff};
  int listed = 0;                                      // first block: kept tokens of its sorted list
  bool drawn = false;                                  // first block: it has the best scores of the tokens that are not listed
  u64 cut = LOWEST;
  const bool hot = temp > 0.f;
  if (hot && ((top_k > 0 && top_k < p.vocab) || top_p < 1.f || min_p > 0.f)) {
    cut = filtered<T>(p, sc, top_k, top_p, min_p, best, listed, drawn);
    if (cut == ~0ull) return;
  } else {
    started();
  }
  if (cut != 0) {
    best = !hot ? largest_of_row<T>() : cut == LOWEST ? draw_from_all<T>(sc) : draw_from<T>(sc, cut);
    block_best(best.v, best.i, sh.warp_v, sh.warp_i);
    if (threadIdx.x == 0) { *of(&sh.part_v[sh.rank], 0) = best.v; *of(&sh.part_i[sh.rank], 0) = best.i; }
    sync_row();
    drawn = true;
    if (sh.rank != 0) return;
  }
  if (listed > 0) {
    best = Best{-INFINITY, 0x7fffffff};
    const int threads = listed <= 64 ? 32 : NT;        // few tokens are one warp's work
    if ((int)threadIdx.x >= threads) return;
    for (int i = threadIdx.x; i < listed; i += threads) {
      const u64 c = sh.list[i];
      take_better(best.v, best.i, sc.of(logit_of(c), index_of(c)), index_of(c));
    }
    if (threads == 32) {
      for (int o = 16; o > 0; o >>= 1)
        take_better(best.v, best.i, __shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.i, o));
    } else {
      block_best(best.v, best.i, sh.warp_v, sh.warp_i);
    }
  }
  if (threadIdx.x == 0) {
    if (drawn)
      for (int b = 0; b < p.blocks; ++b) take_better(best.v, best.i, sh.part_v[b], sh.part_i[b]);
    if (best.v > -INFINITY) p.out[r] = best.i;
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
  SampleParams p{logits, stride, rows, vocab, blocks ? blocks : row_blocks(rows, (long long)vocab * (dtype == 0 ? 4 : 2)), temperature, top_k, top_p, min_p, seeds, counters, out};
  JV_DISPATCH_DTYPE(dtype, T, return launch<T>(p, stream));
}
