// A row of logits as a cluster of blocks reads it, and the choice of its first tokens.
//
// The tokens of a row are in order of their logits, the lowest index first among equal ones.  Both are one number,
//   c = key(x) << 20 | (2^20 - 1 - index),     key: the bits of x, made to ascend with x
// so that "the first tokens up to some boundary" are the tokens with c >= cut.  A NaN counts as minus infinity and -0 as 0.
// A token weighs exp((x - largest) / T) in 32 bits; sums are 32-bit within a thread, 64-bit across threads, in a fixed order.
//
// Few first tokens are found in two passes.  In the first every block keeps the largest logit of each of its 128 groups of
// threads.  The j-th largest of these has at least j tokens at or above it in that block, and about as many in a row whose
// large logits lie anywhere; the lowest of the blocks' bounds therefore has at least j * blocks in the row.  The second
// pass puts the tokens at or above the bound in a list, which the first block sorts.
//
// Where that list does not do (the boundary lies deep in the row, or too many logits are equal), the boundary is found by
// levels: every level cuts the range that holds it into 16 bins, sums up tokens and masses of each, and goes on in the bin
// that holds the boundary, until that bin has few enough tokens to be sorted.  The bins are columns of shared memory that
// belong to one thread each: no atomics, no conflicts between banks, the same sums in every run.
#pragma once

#include <cooperative_groups.h>
#include "common.cuh"

namespace vocab {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int NT = 512, WARPS = NT / 32;               // threads of a block
constexpr int MOST_BLOCKS = 8;                         // of a cluster
constexpr int INDEX_BITS = 20, MAX_VOCAB = 1 << INDEX_BITS;
constexpr unsigned KEY_LOWEST = 0x007fffffu;           // of minus infinity
constexpr int BINS = 16, LIST = 1024;
constexpr int GROUP = 4, GROUPS = NT / GROUP;          // lanes that share a largest logit; such groups of a block
constexpr int MOST_OF_GROUPS = GROUPS * 7 / 8;         // the lowest of the groups' logits that is taken for a bound

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

__device__ __forceinline__ float exp2_fast(float y) {  // two steps off at most; results below 2^-126 are 0
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(e) : "f"(y));
  return e;
}
// exp((x - largest) / T) with scale = log2(e) / T; 1 for the largest itself (also where it is infinite).
__device__ __forceinline__ float mass_of(float x, float largest, float scale) {
  return x == largest ? 1.f : exp2_fast((x - largest) * scale);
}

// The elements of a row that thread `me` of `all` reads, 16 bytes at a time from the first boundary on, AHEAD loads before
// the first is used: f(values, index of the first), once for every load; elements before that boundary and behind the last
// vector come one by one, last.  With WHOLE the lanes of a warp come together for every load: those with nothing left get
// minus infinities behind the row's end.
template <int AHEAD, bool WHOLE = false, typename T, typename F>
__device__ __forceinline__ void for_row(const T* __restrict__ row, int n, int me, int all, F&& f) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const int head = min(n, (VEC - off) % VEC);
  const int vectors = (n - head) / VEC;
  const uint4* body = reinterpret_cast<const uint4*>(row + head);
  const int lane = WHOLE ? threadIdx.x & 31 : 0;
  for (int j = me; j - lane < vectors; j += AHEAD * all) {
    uint4 raw[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (j + u * all < vectors) raw[u] = body[j + u * all];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (j - lane + u * all < vectors) {
        float x[VEC];
        if constexpr (sizeof(T) == 4) {
          x[0] = __uint_as_float(raw[u].x); x[1] = __uint_as_float(raw[u].y);
          x[2] = __uint_as_float(raw[u].z); x[3] = __uint_as_float(raw[u].w);
        } else {
          const unsigned w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
          }
        }
        const bool in = !WHOLE || j + u * all < vectors;
        if (!in) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) x[i] = -INFINITY;
        }
        f(x, in ? head + (j + u * all) * VEC : MAX_VOCAB);
      }
  }
  const int rest = n - vectors * VEC;                  // the head, and what follows the last vector
  for (int e = me; e < rest; e += all) {
    const int at = e < head ? e : e + vectors * VEC;
    const float x[1] = {to_f32(row[at])};
    f(x, at);
  }
}

struct Cell { float mass; unsigned count; };
struct Sums { double mass; unsigned count, pad; };

struct Shared {
  union {
    Cell cells[BINS][NT];
    u64 own[LIST];                                     // this block's tokens on their way to the first block's list
  };
  u64 list[LIST];
  Sums bins[2][MOST_BLOCKS][BINS];                     // what the blocks counted
  double part[MOST_BLOCKS][2];                         // sums that the blocks exchange
  float largest[MOST_BLOCKS], bound[MOST_BLOCKS];
  unsigned tokens[MOST_BLOCKS];
  float part_v[MOST_BLOCKS];
  int part_i[MOST_BLOCKS];
  u64 told;                                            // the boundary, from the first block
  double told_mass;
  unsigned listed, mine, base;
  float group[GROUPS];
  double warp_d[2][WARPS];
  float warp_v[32];
  int warp_i[32];
};

// The tokens lo <= c <= hi that hold the boundary, and what lies above them.
struct Range {
  u64 lo, hi;
  double mass_above;
  unsigned count_above, count;
};

// jv_launch with clusters of `blocks` blocks along x (at most eight, and a divisor of the grid's x).
template <typename... KArgs, typename... Args>
static inline int launch_clusters(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, int blocks, cudaStream_t stream,
                                  Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
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

// Blocks a row.
static inline int row_blocks(int rows, int vocab) {
  const int room = 2 * jv_multiprocessors();
  int blocks = 1;
  while (blocks < MOST_BLOCKS && 2 * blocks * rows <= room && vocab > 4096 * blocks) blocks *= 2;
  return blocks;
}

// The cluster that reads one row: `blocks` of NT threads.  Every member function is called by all threads of all blocks,
// unless it says otherwise.
template <typename T> struct Reader {
  const T* row;
  int n, rank, blocks, me, all, parity;
  Shared* sh;
  float largest, scale, bound;                         // bound: at least `j * blocks` tokens are no smaller

  __device__ __forceinline__ void sync() {
    if (blocks > 1) cg::this_cluster().sync();
    else __syncthreads();
  }
  template <typename V> __device__ __forceinline__ V* of(V* mine, int r) {
    return blocks > 1 ? cg::this_cluster().map_shared_rank(mine, r) : mine;
  }
  // f(values, index of the first) for the elements of this thread
  template <int AHEAD, typename F> __device__ __forceinline__ void each(F&& f) {
    for_row<AHEAD>(row, n, me, all, f);
  }

  __device__ void start(const T* row_, int n_, int blocks_, Shared* sh_) {
    row = row_; n = n_; blocks = blocks_; sh = sh_; parity = 0;
    rank = blocks > 1 ? (int)cg::this_cluster().block_rank() : 0;
    me = rank * NT + threadIdx.x;
    all = blocks * NT;
    if (threadIdx.x == 0) sh->listed = sh->mine = 0;
    if (blocks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
  }
  // Every block of the cluster runs, and has its counters at zero: their memory may be written.
  __device__ __forceinline__ void started() {
    if (blocks > 1) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    else __syncthreads();
  }

  // From the largest logit of every thread: the row's, and the bound that at least j tokens of every block reach (the lowest
  // logit of all where a block has too few groups with any).  Holds one barrier of the cluster; before it, publish() may
  // write to other blocks.
  template <typename P> __device__ void exchange_largest(float m, int j, P&& publish) {
    float g = m;
#pragma unroll
    for (int o = 1; o < GROUP; o *= 2) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (threadIdx.x % GROUP == 0) sh->group[threadIdx.x / GROUP] = g;
    __syncthreads();
    // the place of group threadIdx.x / GROUP among all: each of its lanes compares with a share of the others
    const int mine = threadIdx.x / GROUP;
    int before = 0;
#pragma unroll 8
    for (int i = threadIdx.x % GROUP; i < GROUPS; i += GROUP) {
      const float o = sh->group[i];
      before += o > g || (o == g && i < mine);
    }
#pragma unroll
    for (int o = 1; o < GROUP; o *= 2) before += __shfl_xor_sync(0xffffffffu, before, o);
    if (threadIdx.x % GROUP == 0 && (before == 0 || before == j - 1)) {
      for (int b = 0; b < blocks; ++b) {
        if (before == 0) *of(&sh->largest[rank], b) = g;
        if (before == j - 1) *of(&sh->bound[rank], b) = g;
      }
    }
    publish();
    sync();
    largest = sh->largest[0];
    bound = sh->bound[0];
    for (int b = 1; b < blocks; ++b) {
      largest = fmaxf(largest, sh->largest[b]);
      bound = fminf(bound, sh->bound[b]);
    }
    largest += 0.f;                                    // never -0, as the keys
  }

  // Sums of a and b over the block, in a fixed order; valid in the first warp.
  __device__ void block_sums(double& a, double& b) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    __syncthreads();
    if (lane == 0) { sh->warp_d[0][warp] = a; sh->warp_d[1][warp] = b; }
    __syncthreads();
    if (warp == 0) {
      a = lane < WARPS ? sh->warp_d[0][lane] : 0.;
      b = lane < WARPS ? sh->warp_d[1][lane] : 0.;
      for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
      }
    }
  }

  // A token on its way to the list (any thread).
  __device__ __forceinline__ void put(u64 c) {
    const unsigned at = atomicAdd(&sh->mine, 1u);
    if (at < (unsigned)LIST) sh->own[at] = c;
  }
  // What every block has put goes to the first block's list, their number to `tokens` of every block.  Holds one barrier of
  // the cluster.  Returns the number of tokens put in the row: more than LIST, and the list is of no use.
  template <typename P> __device__ unsigned send_list(P&& publish) {
    __syncthreads();
    const unsigned count = sh->mine;
    const int mine = min((int)count, LIST);
    if (threadIdx.x == 0) sh->base = count == 0 ? 0 : atomicAdd(of(&sh->listed, 0), count);
    if (threadIdx.x < blocks) *of(&sh->tokens[rank], threadIdx.x) = count;
    publish();
    __syncthreads();
    const unsigned base = sh->base;
    u64* list = of(&sh->list[0], 0);
    for (int i = threadIdx.x; i < mine; i += NT)
      if (base + i < (unsigned)LIST) list[base + i] = sh->own[i];
    if (threadIdx.x == 0) sh->mine = 0;
    sync();
    unsigned total = 0;
    for (int b = 0; b < blocks; ++b) total += sh->tokens[b];
    return total;
  }
  // First block only: sorts its list, the largest first, and empties it for what is put next.
  __device__ void sort_list(int m) {
    int padded = 32;
    while (padded < m) padded *= 2;
    for (int i = m + threadIdx.x; i < padded; i += NT) sh->list[i] = 0;
    if (threadIdx.x == 0) sh->listed = 0;
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
  }

  // One level: tokens and masses of the 16 bins over the row, and the bin of the boundary: the lowest one that has tokens
  // and for which before(tokens above, mass above) is true.  bin(x, index) in 0 .. 15 (15 the highest), or < 0: not counted.
  // Takes the range over to that bin's sums and returns the bin; whole(tokens, mass) is told the sums of all bins first.
  template <bool MASS, typename N, typename W, typename B>
  __device__ int level(Range& r, N&& bin, W&& whole, B&& before) {
    Cell* mine = &sh->cells[0][threadIdx.x];
#pragma unroll
    for (int b = 0; b < BINS; ++b) mine[b * NT] = Cell{0.f, 0u};
    each<4>([&](const auto& x, int at) {
      constexpr int V = sizeof(x) / sizeof(float);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float y = clean(x[i]);
        const int b = bin(y, at + i);
        if (b >= 0) {
          Cell c = mine[b * NT];
          ++c.count;
          if (MASS) c.mass += mass_of(y, largest, scale);
          mine[b * NT] = c;
        }
      }
    });
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int b = warp; b < BINS; b += WARPS) {
      double q = 0;
      unsigned c = 0;
      for (int t = lane; t < NT; t += 32) {
        const Cell v = sh->cells[b][t];
        c += v.count;
        q += (double)v.mass;
      }
      for (int o = 16; o > 0; o >>= 1) {
        c += __shfl_xor_sync(0xffffffffu, c, o);
        q += __shfl_xor_sync(0xffffffffu, q, o);
      }
      if (lane < blocks) *of(&sh->bins[parity][rank][b], lane) = Sums{q, c, 0u};
    }
    sync();
    // lane l has bin 15 - l: what lies above it is what the lanes before it have
    double q = 0;
    unsigned c = 0;
    if (lane < BINS)
      for (int k = 0; k < blocks; ++k) {
        const Sums s = sh->bins[parity][k][BINS - 1 - lane];
        q += s.mass;
        c += s.count;
      }
    parity ^= 1;
    double q_to = q;
    unsigned c_to = c;
    for (int o = 1; o < BINS; o *= 2) {
      const double qo = __shfl_up_sync(0xffffffffu, q_to, o);
      const unsigned co = __shfl_up_sync(0xffffffffu, c_to, o);
      if (lane >= o) { q_to += qo; c_to += co; }
    }
    whole(__shfl_sync(0xffffffffu, c_to, BINS - 1), __shfl_sync(0xffffffffu, q_to, BINS - 1));
    double q_above = __shfl_up_sync(0xffffffffu, q_to, 1);
    unsigned c_above = __shfl_up_sync(0xffffffffu, c_to, 1);
    q_above = r.mass_above + (lane == 0 ? 0. : q_above);
    c_above = r.count_above + (lane == 0 ? 0u : c_above);
    const unsigned holds = __ballot_sync(0xffffffffu, lane < BINS && c > 0 && before(c_above, q_above));
    const int l = holds ? 31 - __clz(holds) : 0;
    r.count_above = __shfl_sync(0xffffffffu, c_above, l);
    r.mass_above = __shfl_sync(0xffffffffu, q_above, l);
    r.count = __shfl_sync(0xffffffffu, c, l);
    return BINS - 1 - l;
  }

  static __device__ __forceinline__ int linear_bin(float x, float top, float per) {
    const float d = x >= top ? 0.f : (top - x) * per;
    return BINS - 1 - min(BINS - 1, __float2int_rz(d));
  }
  // The smallest key from `a` to `z` whose value lies in linear bin b or above (that of z does).
  static __device__ unsigned first_key(unsigned a, unsigned z, int b, float top, float per) {
    const int lane = threadIdx.x & 31;
    while (a < z) {
      const unsigned step = (z - a + 31) / 32, p = min(z - 1, a + lane * step);
      const unsigned yes = __ballot_sync(0xffffffffu, linear_bin(value_of(p), top, per) >= b);
      if (yes == 0) { a = min(z - 1, a + 31 * step) + 1; continue; }
      const int f = __ffs(yes) - 1;
      const unsigned up = min(z - 1, a + f * step);
      a = f == 0 ? a : min(z - 1, a + (f - 1) * step) + 1;
      z = up;
    }
    return z;
  }

  // A level whose bins are 1 / per wide, from the range's highest logit down; the range becomes the boundary's bin.
  template <bool MASS, typename W, typename B>
  __device__ void linear_level(Range& r, float per, W&& whole, B&& before) {
    const unsigned low = (unsigned)(r.lo >> INDEX_BITS), high = (unsigned)(r.hi >> INDEX_BITS);
    const float top = value_of(high);
    const u64 lo = r.lo, hi = r.hi;
    const int b = level<MASS>(r, [&](float x, int i) {
      const u64 c = compose(x, i);
      return c >= lo && c <= hi ? linear_bin(x, top, per) : -1;
    }, whole, before);
    // (the last bin takes what lies deeper: it need not end at the range's lowest logit)
    const u64 from = b == 0 ? 0 : (u64)first_key(low, high, b, top, per) << INDEX_BITS;
    if (b < BINS - 1) r.hi = ((u64)first_key(low, high, b + 1, top, per) << INDEX_BITS) - 1;
    r.lo = from > lo ? from : lo;
  }

  // Finds a range of at most `most` tokens, among those with c >= lo, that holds the last token for which
  // before(count, mass) of the tokens before it is true (it is true for the first token, and stays false once it is false).
  // whole(count, mass) is told what all tokens with c >= lo make; where it says no, nothing is looked for.  The bins of
  // the first level are 1 / per wide.
  template <bool MASS, typename W, typename B>
  __device__ bool narrow(u64 lo, float per, unsigned most, Range& r, W&& whole, B&& before) {
    r = Range{lo, compose(largest, 0), 0., 0u, 0u};
    bool wanted = true;
    linear_level<MASS>(r, per, [&](unsigned c, double q) { wanted = whole(c, q); }, before);
    if (!wanted) return false;
    const auto nothing = [](unsigned, double) {};
    for (int depth = 1; r.count > most; ++depth) {
      const float high = logit_of(r.hi), wide = high - logit_of(r.lo);
      const float finer = (float)BINS / wide;
      if (depth < 3 && wide > 0.f && finer > 0.f && finer < INFINITY) {
        linear_level<MASS>(r, finer, nothing, before);
        continue;
      }
      // logits that crowd, or are equal: parts of the range of composed numbers, which ends with a single one
      const u64 span = r.hi - r.lo, from = r.lo, to = r.hi;
      const int shift = max(0, 60 - __clzll((long long)span));
      const int b = level<MASS>(r, [&](float x, int i) {
        const u64 c = compose(x, i);
        return c >= from && c <= to ? (int)((c - from) >> shift) : -1;
      }, nothing, before);
      r.lo = from + ((u64)b << shift);
      const u64 end = r.lo + ((1ull << shift) - 1);
      r.hi = end < to ? end : to;
    }
    return true;
  }

  // The tokens lo <= c <= hi go to the first block's list.
  __device__ unsigned gather(u64 lo, u64 hi) {
    const float low = logit_of(lo);
    __syncthreads();                                   // the cells are read: their place is the list's too
    each<4>([&](const auto& x, int at) {
      constexpr int V = sizeof(x) / sizeof(float);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float y = clean(x[i]);
        if (y >= low) {
          const u64 c = compose(y, at + i);
          if (c >= lo && c <= hi) put(c);
        }
      }
    });
    return send_list([] {});
  }
};

}  // namespace vocab
