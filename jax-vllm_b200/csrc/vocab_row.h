// A row of logits as a cluster of blocks reads it, and the choice of its first tokens.
//
// The tokens of a row are in order of their logits, the lowest index first among equal ones.  Both are one number,
//   c = key(x) << 20 | (2^20 - 1 - index),     key: the bits of x, made to ascend with x
// so that "the first tokens up to some boundary" are the tokens with c >= cut.  A NaN counts as minus infinity and -0 as 0.
// A token weighs q = exp((x - largest) / T) * 2^43, cut to a whole number: sums of these are exact whatever their order.
//
// The boundary (the k-th token, or the first before which a given mass lies) is found by levels: every level cuts the
// range that holds it into 16 bins, sums up tokens and masses of each, and goes on in the bin that holds the boundary,
// until that bin has few enough tokens to be sorted.  The bins of a level are columns of shared memory that belong to one
// thread each (no atomics, no conflicts between banks, sums the same in every run).
#pragma once

#include <cooperative_groups.h>
#include "common.cuh"

namespace vocab {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int INDEX_BITS = 20, MAX_VOCAB = 1 << INDEX_BITS;
constexpr unsigned KEY_LOWEST = 0x007fffffu;           // of minus infinity
constexpr int MASS_BITS = 43, BINS = 16, LIST = 1024;
constexpr int COUNT_SHIFT = 54;                        // a cell: tokens (at most 1023 of a thread) above their mass
constexpr int CELL_MOST = 1000;

__device__ __forceinline__ float clean(float x) { return x == x ? x + 0.f : -INFINITY; }
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned u = __float_as_uint(x);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned key) {
  return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ u64 compose(float x, int index) {
  return (u64)key_of(x) << INDEX_BITS | (unsigned)(MAX_VOCAB - 1 - index);
}
__device__ __forceinline__ int index_of(u64 c) { return MAX_VOCAB - 1 - (int)(c & (MAX_VOCAB - 1)); }
__device__ __forceinline__ float logit_of(u64 c) { return value_of((unsigned)(c >> INDEX_BITS)); }

// exp((x - largest) / T) * 2^43 with scale = log2(e) / T.  The largest itself weighs 2^43 (also where it is infinite).
__device__ __forceinline__ u64 mass_of(float x, float largest, float scale) {
  const float e = x == largest ? 1.f : exp2f((x - largest) * scale);
  return __float2ull_rz(e * (float)(1ull << MASS_BITS));
}

// The elements of a row that thread `me` of `all` reads: f(value, index) for each, 16 bytes at a time from the first
// boundary on, AHEAD loads before the first is used; the elements before it and after the last one by themselves.
template <int AHEAD, typename T, typename F>
__device__ __forceinline__ void for_row(const T* __restrict__ row, int n, int me, int all, F&& f) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const int head = min(n, (VEC - off) % VEC);
  const int vectors = (n - head) / VEC;
  const uint4* body = reinterpret_cast<const uint4*>(row + head);
  for (int j = me; j < vectors; j += AHEAD * all) {
    uint4 raw[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (j + u * all < vectors) raw[u] = body[j + u * all];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (j + u * all < vectors) {
        const int at = head + (j + u * all) * VEC;
        if constexpr (sizeof(T) == 4) {
          f(clean(__uint_as_float(raw[u].x)), at);
          f(clean(__uint_as_float(raw[u].y)), at + 1);
          f(clean(__uint_as_float(raw[u].z)), at + 2);
          f(clean(__uint_as_float(raw[u].w)), at + 3);
        } else {
          const unsigned w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f(clean(__uint_as_float(w[i] << 16)), at + 2 * i);
            f(clean(__uint_as_float(w[i] & 0xffff0000u)), at + 2 * i + 1);
          }
        }
      }
  }
  const int rest = n - vectors * VEC;                  // the head, and what follows the last vector
  for (int e = me; e < rest; e += all) {
    const int at = e < head ? e : e + vectors * VEC;
    f(clean(to_f32(row[at])), at);
  }
}

template <int NT> struct Shared {
  u64 cells[BINS][NT];
  u64 list[LIST];
  u64 bin_mass[2][BINS], scan[NT / 32];
  unsigned bin_count[2][BINS];
  unsigned listed;
  u64 told[4];                                         // what the first block tells the others
  float block_largest;
  float part_v[16];                                    // one a block of the cluster
  int part_i[16];
  float warp_v[NT / 32];
  int warp_i[NT / 32];
  u64 pick[8];
};

// The tokens lo <= c <= hi that hold the boundary, and what lies above them.
struct Range {
  u64 lo, hi, mass_above;
  unsigned count_above, count;
};

// jv_launch with clusters of `blocks` blocks along x (at most eight, and a divisor of the grid's x).
template <typename... KArgs, typename... Args>
static inline int launch_clusters(void (*kernel)(KArgs...), dim3 grid, dim3 block, int blocks, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (blocks > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)blocks;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (jv_pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...) == cudaSuccess ? JV_OK : JV_ERR_LAUNCH;
}

// The cluster that reads one row.  `blocks` of NT threads; every member function is called by all threads of all blocks.
template <typename T, int NT> struct Reader {
  const T* row;
  int n, rank, blocks, me, all, parity;
  Shared<NT>* sh;
  float largest, scale;

  __device__ __forceinline__ void sync() {
    if (blocks > 1) cg::this_cluster().sync();
    else __syncthreads();
  }
  template <typename V> __device__ __forceinline__ V* of(V* mine, int r) {
    return blocks > 1 ? cg::this_cluster().map_shared_rank(mine, r) : mine;
  }
  template <int AHEAD, typename F> __device__ __forceinline__ void each(F&& f) { for_row<AHEAD>(row, n, me, all, f); }

  __device__ void start(const T* row_, int n_, int blocks_, Shared<NT>* sh_) {
    row = row_; n = n_; blocks = blocks_; sh = sh_; parity = 0;
    rank = blocks > 1 ? (int)cg::this_cluster().block_rank() : 0;
    me = rank * NT + threadIdx.x;
    all = blocks * NT;
  }

  __device__ void find_largest() {
    float m = -INFINITY;
    each<8>([&](float x, int) { m = fmaxf(m, x); });
    m = warp_max(m);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) sh->warp_v[warp] = m;
    if (threadIdx.x == 0) sh->listed = 0;
    __syncthreads();
    if (warp == 0) {
      m = warp_max(lane < NT / 32 ? sh->warp_v[lane] : -INFINITY);
      if (lane == 0) sh->block_largest = m;
    }
    sync();
    m = -INFINITY;
    for (int r = 0; r < blocks; ++r) m = fmaxf(m, *of(&sh->block_largest, r));
    largest = m;
  }

  // Tokens and masses of the bins over the whole row.  bin(x, c) in 0 .. 15 (15 the highest), or < 0: not counted.
  // The sums of the row are left in bin_count and bin_mass of this block ([parity ^ 1]: what the other blocks had is gone
  // after the next call but one).
  template <bool MASS, typename B> __device__ void level(u64 (&mass)[BINS], unsigned (&count)[BINS], B&& bin) {
    u64* mine = &sh->cells[0][threadIdx.x];
#pragma unroll
    for (int b = 0; b < BINS; ++b) mine[b * NT] = 0;
    each<4>([&](float x, int i) {
      const int b = bin(x, i);
      if (b >= 0) mine[b * NT] += (1ull << COUNT_SHIFT) + (MASS ? mass_of(x, largest, scale) : 0ull);
    });
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int b = warp; b < BINS; b += NT / 32) {
      u64 q = 0;
      unsigned c = 0;
      for (int t = lane; t < NT; t += 32) {
        const u64 v = sh->cells[b][t];
        c += (unsigned)(v >> COUNT_SHIFT);
        q += v & ((1ull << COUNT_SHIFT) - 1);
      }
      for (int o = 16; o > 0; o >>= 1) {
        c += __shfl_xor_sync(0xffffffffu, c, o);
        q += __shfl_xor_sync(0xffffffffu, q, o);
      }
      if (lane == 0) { sh->bin_count[parity][b] = c; sh->bin_mass[parity][b] = q; }
    }
    sync();
#pragma unroll
    for (int b = 0; b < BINS; ++b) { mass[b] = 0; count[b] = 0; }
    for (int r = 0; r < blocks; ++r) {
      const unsigned* c = of(&sh->bin_count[parity][0], r);
      const u64* q = of(&sh->bin_mass[parity][0], r);
#pragma unroll
      for (int b = 0; b < BINS; ++b) { count[b] += c[b]; mass[b] += q[b]; }
    }
    parity ^= 1;
  }

  // The smallest key whose value lies at least as near to the largest as `b` bins of width 1 / per.
  static __device__ __forceinline__ int linear_bin(float x, float largest, float per) {
    const float d = x == largest ? 0.f : (largest - x) * per;
    return BINS - 1 - min(BINS - 1, __float2int_rz(d));
  }
  __device__ unsigned first_key(int b, float per) const {
    const int lane = threadIdx.x & 31;
    unsigned a = KEY_LOWEST, z = key_of(largest);
    while (a < z) {
      const unsigned step = (z - a + 31) / 32, p = min(z - 1, a + lane * step);
      const unsigned yes = __ballot_sync(0xffffffffu, linear_bin(value_of(p), largest, per) >= b);
      if (yes == 0) { a = min(z - 1, a + 31 * step) + 1; continue; }
      const int f = __ffs(yes) - 1;
      const unsigned up = min(z - 1, a + f * step);
      a = f == 0 ? a : min(z - 1, a + (f - 1) * step) + 1;
      z = up;
    }
    return z;
  }

  // Finds a range of at most `most` tokens, among those with c >= lo, that holds the last token for which
  // before(count, mass) of the tokens before it is true (it is true for the first token, and stays false once it is false).
  // whole(count, mass) is told what all tokens with c >= lo make; where it says no, nothing is looked for.  The bins of
  // the first level are 1 / per wide, counted from the largest logit down.
  template <bool MASS, typename W, typename B>
  __device__ bool narrow(u64 lo, float per, unsigned most, Range& r, W&& whole, B&& before) {
    u64 mass[BINS];
    unsigned count[BINS];
    level<MASS>(mass, count, [&](float x, int i) { return compose(x, i) >= lo ? linear_bin(x, largest, per) : -1; });
    unsigned total = 0;
    u64 total_mass = 0;
#pragma unroll
    for (int b = 0; b < BINS; ++b) { total += count[b]; total_mass += mass[b]; }
    if (!whole(total, total_mass)) return false;
    r.count_above = 0;
    r.mass_above = 0;
    int b = choose(mass, count, r, before);
    const u64 low = (u64)first_key(b, per) << INDEX_BITS;
    r.lo = low > lo ? low : lo;
    r.hi = b == BINS - 1 ? ~0ull : ((u64)first_key(b + 1, per) << INDEX_BITS) - 1;
    if (r.hi == ~0ull) r.hi = compose(largest, 0);
    while (r.count > most) {
      const u64 span = r.hi - r.lo;
      const int shift = max(0, 60 - __clzll((long long)span));
      level<MASS>(mass, count, [&](float x, int i) {
        const u64 c = compose(x, i);
        return c >= r.lo && c <= r.hi ? (int)((c - r.lo) >> shift) : -1;
      });
      b = choose(mass, count, r, before);
      const u64 bottom = r.lo + ((u64)b << shift), top = bottom + ((1ull << shift) - 1);
      r.lo = bottom;
      r.hi = top < r.hi ? top : r.hi;
    }
    return true;
  }

  // The bin of the boundary; adds what lies above it.
  template <typename B> __device__ __forceinline__ int choose(const u64 (&mass)[BINS], const unsigned (&count)[BINS], Range& r, B&& before) {
    unsigned above = r.count_above, best_above = 0, best_count = 0;
    u64 mass_above = r.mass_above, best_mass = 0;
    int best = 0;
#pragma unroll
    for (int b = BINS - 1; b >= 0; --b) {
      if (count[b] > 0 && before(above, mass_above)) { best = b; best_above = above; best_mass = mass_above; best_count = count[b]; }
      above += count[b];
      mass_above += mass[b];
    }
    r.count_above = best_above;
    r.mass_above = best_mass;
    r.count = best_count;
    return best;
  }

  // The tokens of a range, in the first block's list.  A cluster barrier follows; `listed` is their number.
  __device__ void gather(u64 lo, u64 hi) {
    unsigned* listed = of(&sh->listed, 0);
    u64* list = of(&sh->list[0], 0);
    each<4>([&](float x, int i) {
      const u64 c = compose(x, i);
      if (c >= lo && c <= hi) {
        const unsigned at = atomicAdd(listed, 1u);
        if (at < (unsigned)LIST) list[at] = c;
      }
    });
    sync();
  }

  // First block only: sorts its list, the largest first.  Returns the number of tokens in it.
  __device__ int sort_list() {
    const int m = min((int)sh->listed, LIST);
    int padded = 32;
    while (padded < m) padded *= 2;
    for (int i = m + threadIdx.x; i < padded; i += NT) sh->list[i] = 0;
    __syncthreads();
    for (int size = 2; size <= padded; size *= 2)
      for (int stride = size / 2; stride > 0; stride /= 2) {
        for (int i = threadIdx.x; i < padded / 2; i += NT) {
          const int a = 2 * i - (i & (stride - 1)), b = a + stride;
          const bool down = (a & size) == 0;
          const u64 u = sh->list[a], v = sh->list[b];
          if ((u < v) == down) { sh->list[a] = v; sh->list[b] = u; }
        }
        __syncthreads();
      }
    return m;
  }
};

}  // namespace vocab
