// A row of logits as a cluster of blocks reads it, and the choice of its first tokens.
//
// The tokens of a row are in order of their logits, the lowest index first among equal ones.  Both are one number,
//   c = key(x) << 20 | (2^20 - 1 - index),     key: the bits of x, made to ascend with x
// so that "the first tokens up to some boundary" are the tokens with c >= cut.  A NaN counts as minus infinity and -0 as 0.
// A token weighs exp((x - largest) / T) in 32 bits; sums are 32-bit within a thread, 64-bit across threads, in an order that follows
// the row's length, its place beside 16-byte boundaries and the number of blocks that read it.
//
// Few first tokens are found in two passes.  In the first every thread keeps its largest logit.  The j-th largest of a block's
// (of its warps, of 128 groups of four threads, or of the threads where j is large) has at least j tokens at or above it in that block, and
// not many more in a row whose large logits lie anywhere; the lowest of the blocks' bounds therefore has at least j * blocks
// in the row.  The second pass puts the tokens at or above the bound in a list, which the first block sorts.
//
// Where that list does not do (the boundary lies deep in the row, or too many logits are equal), the boundary is found by
// levels: every level cuts the range that holds it into 31 bins, sums up the tokens or the masses of each, and goes on in the
// bin that holds the boundary, until that bin has few enough tokens to be sorted.  The bins are columns of shared memory that
// belong to one thread each: no atomics, no conflicts between banks, the same sums in every run.
//
// What all threads of a block know of its row stands in shared memory, and every pass over the row is a function of its own:
// with all of it in one, the passes ran out of registers.
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
constexpr u64 LOWEST = (u64)KEY_LOWEST << INDEX_BITS;  // no token's number is smaller
constexpr int BINS = 31, LIST = 2048, BUCKETS = NT;
constexpr unsigned CROWD = 64;                         // tokens up to which those of a bucket are compared with one another
constexpr int GROUP = 4, GROUPS = NT / GROUP;          // lanes that share a largest logit; such groups of a block
constexpr int FEW = GROUPS / 2;                        // tokens a block up to which the groups give the bound
constexpr float HUGE_F = 3.402823466e38f;

__device__ __forceinline__ float nan_f() { return __int_as_float(0x7fffffff); }
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
// How far x lies below the largest logit; not at all where both are infinite (the difference is no number then).
__device__ __forceinline__ float below(float x, float largest) { return fmaxf(largest - x, 0.f); }

// Sixteen bytes as 32-bit numbers.
template <typename T> __device__ __forceinline__ void unpack(const uint4& raw, float (&x)[16 / sizeof(T)]) {
  const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      x[i] = __uint_as_float(w[i]);
    } else {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

// By pairs: a thread adds a vector's sum to its own, which is rounded once for every vector.
template <int VEC> __device__ __forceinline__ float sum_of(const float (&x)[VEC]) {
  float s[VEC / 2];
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) s[i] = x[2 * i] + x[2 * i + 1];
#pragma unroll
  for (int n = VEC / 4; n > 0; n /= 2)
#pragma unroll
    for (int i = 0; i < n; ++i) s[i] += s[i + n];
  return s[0];
}

// A range of tokens that holds the boundary: lo <= c <= hi.  While it is cut into bins of equal width, it is the tokens with
// from <= largest - x < to (as 32 bits round it; no end where `to` is infinite) of those asked for.
struct Range {
  u64 lo, hi;
  float from, to, per;                                 // bins 1 / per wide
  int shift;                                           // bins of 2^shift composed numbers
  bool composed, found, enough;                        // enough: as few tokens as were looked for, or fewer, are all there are
  double above, all;                                   // tokens, or mass, above it and of all that were asked for
};

struct Shared {
  double bins[2][MOST_BLOCKS][BINS];                   // what the blocks counted
  double part[MOST_BLOCKS][2];                         // sums that the blocks exchange
  float part_v[MOST_BLOCKS];
  int part_i[MOST_BLOCKS];
  unsigned tokens[MOST_BLOCKS];
  float largest_of[MOST_BLOCKS], bound_of[MOST_BLOCKS];
  alignas(16) float group[GROUPS];
  double warp_d[2][WARPS];
  float warp_v[32];
  int warp_i[32];
  // the row: `vectors` of sixteen bytes from the first sixteen-byte boundary on, `head` elements before them, some behind
  const void* row;
  int n, head, vectors, blocks, rank, parity;
  float largest, scale, bound;                         // bound: at least `j * blocks` tokens are no smaller; scale: log2(e) / T
  Range range;
  u64 told;                                            // the boundary, from the first block
  unsigned listed, mine, base, best_key;
  // (a kernel that lists and counts nothing has no memory from here on)
  alignas(16) u64 list[LIST];
  union {
    float cells[BINS + 1][NT];                         // of a level: whole numbers or masses; the last row is not counted
    struct {
      u64 own[LIST];                                   // this block's tokens on their way to the first block's list
      uint2 queue[WARPS][32 * 9];                      // of a warp: logits and indices of tokens to draw from
    };
    struct {
      u64 sorted[LIST];
      unsigned bucket[BUCKETS + 1];
    };
  };
};
// The block's shared memory (named here, so that every function knows it for that).
extern __shared__ __align__(16) unsigned char shared_bytes[];
__device__ __forceinline__ Shared& shared() { return *reinterpret_cast<Shared*>(shared_bytes); }

// ---------------------------------------------------------------------------------------------------------- the cluster
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

// Blocks a row: as many as leave two blocks a multiprocessor room at once, while a block has 16 KB of its row or more.  Filtered
// sampling, us for one, two, four and eight blocks a row: one row of 608 KB 18.0, 13.9, 11.4, 10.5; 24 rows of 64 KB 11.5, 10.8, 10.9, 11.2;
// 40 rows of 608 KB 19.4, 16.8, 14.1, 20.7; 75 rows 24.7, 19.0, 24.6, 31.6; 128 rows 30.1, 27.4, 33.3, 52.7; 160 rows 31.5, 45.3,
// 44.4, 63.9; 256 rows 36.6, 52.3, 60.7, 95.6.  Where the device is filled to the last place the next smaller number is the
// faster one (74 rows: four blocks 24.2, two 16.9; 148 rows: two 31.2, one 28.4).
static inline int row_blocks(int rows, long long row_bytes) {
  const int room = 2 * jv_multiprocessors();
  int blocks = 1;
  while (blocks < MOST_BLOCKS && 2 * blocks * rows <= room && row_bytes >= 2 * blocks * 16384ll - 4096) blocks *= 2;
  return blocks;
}

// Every function below is called by all threads of all blocks of a row's cluster, unless it says otherwise.

// Notes down the row, and tells the other blocks that this one runs.
template <typename T> __device__ __forceinline__ void begin(const T* row, int n, int blocks) {
  Shared& sh = shared();
  if (threadIdx.x == 0) {
    constexpr int VEC = 16 / (int)sizeof(T);
    const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    sh.row = row;
    sh.n = n;
    sh.head = min(n, (VEC - off) % VEC);
    sh.vectors = (n - sh.head) / VEC;
    sh.blocks = blocks;
    sh.rank = blocks > 1 ? (int)cg::this_cluster().block_rank() : 0;
    sh.parity = 0;
    sh.listed = sh.mine = 0;
    sh.best_key = KEY_LOWEST;
  }
  __syncthreads();
  if (blocks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
}
// Every block of the cluster runs, and has its counters at zero: their memory may be written.  Called once.
__device__ __forceinline__ void started() {
  if (shared().blocks > 1) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void sync_row() {
  if (shared().blocks > 1) cg::this_cluster().sync();
  else __syncthreads();
}
// The place of `mine` in the memory of block b.
template <typename V> __device__ __forceinline__ V* of(V* mine, int b) {
  return shared().blocks > 1 ? cg::this_cluster().map_shared_rank(mine, b) : mine;
}

// ---------------------------------------------------------------------------------------------------------- passes
// The elements before the first vector and behind the last one, as two vectors that read as NaN elsewhere: `which` 0 or 1.
template <typename T> __device__ __forceinline__ int first_of_end(int which) {
  constexpr int VEC = 16 / (int)sizeof(T);
  return which == 0 ? shared().head - VEC : shared().head + shared().vectors * VEC;
}
template <typename T> __device__ __noinline__ uint4 load_end(int which) {
  const Shared& sh = shared();
  const T* row = reinterpret_cast<const T*>(sh.row);
  const int at = first_of_end<T>(which), from = which == 0 ? 0 : at, to = which == 0 ? sh.head : sh.n;
  unsigned w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      w[i] = at + i >= from && at + i < to ? reinterpret_cast<const unsigned*>(row)[at + i] : 0x7fffffffu;
    } else {
      const int l = at + 2 * i, h = l + 1;
      w[i] = (l >= from && l < to ? reinterpret_cast<const unsigned short*>(row)[l] : 0x7fffu) |
             (h >= from && h < to ? (unsigned)reinterpret_cast<const unsigned short*>(row)[h] : 0x7fffu) << 16;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 no_vector() { return make_uint4(0x7fffffffu, 0x7fffffffu, 0x7fffffffu, 0x7fffffffu); }   // NaNs of either type

// f(values, index of the first) for the vectors that this thread reads, AHEAD loads before the first is used, and then for the
// ends of the row; what lies outside the row is NaN.  With WHOLE the lanes of a warp come together for every vector: those
// with none left get NaNs.
template <typename T, int AHEAD, bool WHOLE = false, typename F> __device__ __forceinline__ void each(F&& f) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const Shared& sh = shared();
  const int step = sh.blocks * NT, start = sh.rank * NT + threadIdx.x, vectors = sh.vectors;
  const int lane = WHOLE ? threadIdx.x & 31 : 0;
  {
    const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(sh.row) + sh.head) + start;
    int at = sh.head + start * VEC;
    for (int left = vectors - start; left + lane > 0; left -= AHEAD * step) {
      uint4 raw[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
        if (left > u * step) raw[u] = p[u * step];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
        if (left + lane > u * step) {
          float x[VEC];
          if (WHOLE && left <= u * step) raw[u] = no_vector();
          unpack<T>(raw[u], x);
          f(x, at + u * step * VEC);
        }
      p += AHEAD * step;
      at += AHEAD * step * VEC;
    }
  }
  if (start - lane < 2) {                              // the row's first two threads (with WHOLE: their warp)
    float x[VEC];
    unpack<T>(start < 2 ? load_end<T>(start) : no_vector(), x);
    f(x, first_of_end<T>(start));
  }
}

// A logit that may be counted.  Where masses are, minus infinity and NaN are never asked for; elsewhere a NaN of the row is
// minus infinity, and one outside it stays what it is.
template <bool MASS> __device__ __forceinline__ float asked(float x, int index, int n) {
  return MASS || (unsigned)index >= (unsigned)n ? x : clean(x);
}

// This thread's largest logit.
template <typename T> __device__ __noinline__ float my_largest() {
  float m = -INFINITY;
  each<T, 8>([&](const auto& x, int) {
#pragma unroll
    for (int i = 0; i < 16 / (int)sizeof(T); ++i) m = fmaxf(m, x[i]);
  });
  return m;
}

// Whether a list of the tokens from the bound for j tokens a block up is likely to have room: of NT threads with their tokens
// anywhere, NT * log(NT / (NT - j)) tokens are expected where j threads have one.  A quarter of the list is left for rows that are
// not as expected.  (The first 1,000 tokens of 64 rows 26.0 us, 49.2 if half is left; the first 200 of 256 rows 58.1 us, which a
// list that is expected to be full would do in 50.5, and then a row that is not as expected pays for both.)
__device__ __forceinline__ bool countable(int j, int blocks) {
  return j < NT && (float)(blocks * NT) * -__logf(1.f - (float)j * (1.f / NT)) < 0.75f * LIST;
}

// From the largest logit of every thread: the row's, and the bound that at least j tokens of every block reach (minus infinity
// where a block has too few threads with any).  Holds one barrier of the cluster.
static __device__ __noinline__ void exchange_largest(float m, int j) {
  Shared& sh = shared();
  const int blocks = sh.blocks;
  if (j <= WARPS / 2) {
    // the warps' own largest do, and the first warp finds the place of each
    const unsigned k = __reduce_max_sync(0xffffffffu, key_of(m + 0.f));
    if (threadIdx.x % 32 == 0) sh.warp_i[threadIdx.x / 32] = (int)k;
    __syncthreads();
    if (threadIdx.x < 32) {
      const unsigned mine = threadIdx.x < WARPS ? (unsigned)sh.warp_i[threadIdx.x] : 0u;
      int above = 0, reach = 0;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const unsigned o = __shfl_sync(0xffffffffu, mine, w);
        above += o > mine;
        reach += o >= mine;
      }
      if (threadIdx.x < WARPS)
        for (int b = 0; b < blocks; ++b) {             // (equal ones write the same)
          if (above == 0) *of(&sh.largest_of[sh.rank], b) = value_of(mine);
          if (above < j && reach >= j) *of(&sh.bound_of[sh.rank], b) = value_of(mine);
        }
    }
  } else {
    float g = m;
#pragma unroll
    for (int o = 1; o < GROUP; o *= 2) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
    const int part = threadIdx.x % GROUP;
    if (part == 0) sh.group[threadIdx.x / GROUP] = g;
    __syncthreads();
    // the groups above this one's largest, and those at it: each of its lanes compares with a share of the others
    int both = 0;
    const float4* others = reinterpret_cast<const float4*>(sh.group);
#pragma unroll 4
    for (int i = 0; i < GROUPS / 4 / GROUP; ++i) {
      const float4 o = others[i * GROUP + part];
      both += ((o.x > g) + (o.y > g) + (o.z > g) + (o.w > g)) << 16;
      both += (o.x >= g) + (o.y >= g) + (o.z >= g) + (o.w >= g);
    }
#pragma unroll
    for (int o = 1; o < GROUP; o *= 2) both += __shfl_xor_sync(0xffffffffu, both, o);
    const int above = both >> 16, reach = both & 0xffff;
    if (above == 0)                                    // (equal ones write the same)
      for (int b = part; b < blocks; b += GROUP) *of(&sh.largest_of[sh.rank], b) = g;
    if (j <= FEW) {
      if (above < j && reach >= j)
        for (int b = part; b < blocks; b += GROUP) *of(&sh.bound_of[sh.rank], b) = g;
    } else {
      // the threads' own largest: a key that j of them reach, by halves
      unsigned lo = KEY_LOWEST, hi = 0xff800000u;      // at least j reach lo; fewer reach beyond hi
      const unsigned mine = key_of(m + 0.f);
      while (lo < hi) {
        const unsigned mid = lo + (hi - lo) / 2 + 1;
        const int c = __syncthreads_count(mine >= mid);
        if (c >= j) lo = mid; else hi = mid - 1;
        if (c >= j && c <= j + j / 16) break;
      }
      if (threadIdx.x < blocks) *of(&sh.bound_of[sh.rank], threadIdx.x) = value_of(lo);
    }
  }
  sync_row();
  // (every warp for itself; they write the same)
  const int lane = threadIdx.x & 31;
  float l = lane < blocks ? sh.largest_of[lane] : -INFINITY, low = lane < blocks ? sh.bound_of[lane] : INFINITY;
#pragma unroll
  for (int o = 1; o < MOST_BLOCKS; o *= 2) {
    l = fmaxf(l, __shfl_xor_sync(0xffffffffu, l, o));
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
  }
  if (lane == 0) {
    sh.largest = l + 0.f;                              // never -0, as the keys
    sh.bound = low;
  }
  __syncwarp();
}

// Sums of a and b over the block, in a fixed order; valid in the first warp.
static __device__ __noinline__ double2 block_sums(double a, double b) {
  Shared& sh = shared();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  __syncthreads();
  if (lane == 0) { sh.warp_d[0][warp] = a; sh.warp_d[1][warp] = b; }
  __syncthreads();
  if (warp == 0) {
    a = lane < WARPS ? sh.warp_d[0][lane] : 0.;
    b = lane < WARPS ? sh.warp_d[1][lane] : 0.;
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
  }
  return make_double2(a, b);
}

// ---------------------------------------------------------------------------------------------------------- the list
// A token on its way to the list (any thread).
__device__ __forceinline__ void put(u64 c) {
  const unsigned at = atomicAdd(&shared().mine, 1u);
  if (at < (unsigned)LIST) shared().own[at] = c;
}

// What every block has put goes to the first block's list, their number to `tokens` of every block.  Holds one barrier of the
// cluster.  Returns the number of tokens put in the row: more than LIST, and the list is of no use.
static __device__ __noinline__ unsigned send_list() {
  Shared& sh = shared();
  __syncthreads();
  const unsigned count = sh.mine;
  const int mine = min((int)count, LIST), blocks = sh.blocks;
  if (threadIdx.x == 0) sh.base = count == 0 ? 0 : atomicAdd(of(&sh.listed, 0), count);
  if (threadIdx.x < blocks) *of(&sh.tokens[sh.rank], threadIdx.x) = count;
  __syncthreads();
  const unsigned base = sh.base;
  u64* list = of(&sh.list[0], 0);
  for (int i = threadIdx.x; i < mine; i += NT)
    if (base + i < (unsigned)LIST) list[base + i] = sh.own[i];
  if (threadIdx.x == 0) sh.mine = 0;
  sync_row();
  unsigned total = 0;
  for (int b = 0; b < blocks; ++b) total += sh.tokens[b];
  return total;
}

// Whether what put_once puts is likely to have room: what the first vectors hold above their bound, and as much again whenever as
// many have been read as the bound was taken of.
template <typename T> __device__ __forceinline__ bool fits_once(int j, int n) {
  const float first = 6.f * NT * (16 / sizeof(T)), all = (float)n;
  const float own = (float)NT * -__logf(1.f - (float)j * (1.f / NT));
  return own * (1.f + fmaxf(0.f, fminf(all, 3.f * first) - first) / first + fmaxf(0.f, all - 3.f * first) / (3.f * first)) < 0.75f * LIST;
}
// One pass instead of two, where one block reads a row: the bound for j tokens of what has been read so far, taken after the
// first vectors and once more later, decides what is put, so that the list gets more tokens than it has to hold.  Minus
// infinity is not put, nor what lies more than `deepest` below the largest.  Returns this thread's largest logit and, SUMMED,
// the sum of its masses, relative to that one's.
template <typename T, bool SUMMED> __device__ __noinline__ float2 put_once(int j, float deepest) {
  constexpr int VEC = 16 / (int)sizeof(T), AHEAD = 6;
  const float scale = shared().scale;
  const int vectors = shared().vectors;
  float m = -INFINITY, s = 0.f, least = INFINITY;
  const auto take = [&](const uint4& raw, int at) {
    float x[VEC];
    unpack<T>(raw, x);
    float big = x[0];                                  // (a NaN is passed over)
#pragma unroll
    for (int i = 1; i < VEC; ++i) big = fmaxf(big, x[i]);
    if (SUMMED) {
      if (big > m) s *= exp2_fast(-(fminf(big - m, HUGE_F) * scale));
      const float to = fmaxf(big, m);
      float q[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) q[i] = x[i] > -INFINITY ? exp2_fast(-(below(x[i], to) * scale)) : 0.f;
      s += sum_of(q);
    }
    m = fmaxf(m, big);
    if (big >= least) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (x[i] >= least) put(compose(clean(x[i]), at + i));
    }
  };
  const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(shared().row) + shared().head) + threadIdx.x;
  int at = shared().head + threadIdx.x * VEC;
  for (int k = 0; k == 0 || k * AHEAD * NT < vectors; ++k) {
    uint4 raw[AHEAD];
    const int left = vectors - k * AHEAD * NT - (int)threadIdx.x;
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) raw[u] = left > u * NT ? p[u * NT] : no_vector();
    p += AHEAD * NT;
    // The bound of the first vectors, and once more when three times as many have been read.  (256
    // rows with peaks under top-p 46.2 us, 50.3 with the first bound alone, 64.3 with one in every round; rows in ascending order 168,
    // 166 and 185.)
    if (k == 0 || k == 3) {
      float g = m;
      if (k == 0) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          float x[VEC];
          unpack<T>(raw[u], x);
#pragma unroll
          for (int i = 0; i < VEC; ++i) g = fmaxf(g, x[i]);
        }
      }
      exchange_largest(g, j);
      least = fmaxf(fmaxf(shared().bound, -HUGE_F), shared().largest - deepest);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) take(raw[u], at + u * NT * VEC);
    at += AHEAD * NT * VEC;
  }
  if (threadIdx.x < 2) {
    take(load_end<T>(threadIdx.x), first_of_end<T>(threadIdx.x));
  }
  return make_float2(m, s);
}
// What has been put and is no smaller than `least` becomes the list (one block a row).  Returns the number of its tokens, or
// LIST + 1 where more had been put than there was room for; both counters are at zero then.
static __device__ __noinline__ unsigned keep_list(float least) {
  Shared& sh = shared();
  __syncthreads();
  const unsigned count = sh.mine;
  if (count <= (unsigned)LIST)
    for (int i = threadIdx.x; i < (int)count; i += NT) {
      const u64 c = sh.own[i];
      if (logit_of(c) >= least) sh.list[atomicAdd(&sh.listed, 1u)] = c;
    }
  __syncthreads();
  const unsigned kept = sh.listed;
  __syncthreads();                                     // both counters are read: they may be set again
  if (threadIdx.x == 0) sh.listed = sh.mine = 0;
  return count <= (unsigned)LIST ? kept : LIST + 1;
}

// First block only: sorts its list of m tokens by a bitonic network: the same steps whatever they are (2,048 tokens: 13 us).
static __device__ __noinline__ void sort_network(int m) {
  Shared& sh = shared();
  int n = 2 * NT / 4;
  while (n < m) n *= 2;
  for (int i = m + threadIdx.x; i < n; i += NT) sh.list[i] = 0;        // no token's number: behind all of them
  for (int k = 2; k <= n; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      __syncthreads();
      for (int t = threadIdx.x; t < n / 2; t += NT) {
        const int a = 2 * t - (t & (j - 1)), b = a + j;
        const u64 x = sh.list[a], y = sh.list[b];
        if ((x < y) == ((a & k) == 0)) { sh.list[a] = y; sh.list[b] = x; }
      }
    }
  __syncthreads();
}

// First block only: sorts its list of m tokens, the largest first, and empties it for what is put next.
static __device__ __noinline__ void sort_list(int m) {
  Shared& sh = shared();
  if (threadIdx.x == 0) sh.listed = 0;
  if (m <= NT / 4) {
    // every token's place is the number of tokens before it: four lanes count them, a quarter each
    const int i = threadIdx.x / 4;
    const u64 c = i < m ? sh.list[i] : 0;
    int place = 0;
    for (int k = threadIdx.x % 4; k < m; k += 4) place += sh.list[k] > c;
    place += __shfl_xor_sync(0xffffffffu, place, 1);
    place += __shfl_xor_sync(0xffffffffu, place, 2);
    __syncthreads();
    if (i < m && threadIdx.x % 4 == 0) sh.list[place] = c;
    __syncthreads();
    return;
  }
  // in buckets of equal width between the largest logit and the smallest (of indices, where all are equal), and within a
  // bucket by the number of its tokens that lie before one
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int PER = LIST / NT;
  unsigned small = ~0u, large = 0;
  for (int i = threadIdx.x; i < m; i += NT) {
    const unsigned k = (unsigned)(sh.list[i] >> INDEX_BITS);
    small = min(small, k);
    large = max(large, k);
  }
  small = __reduce_min_sync(0xffffffffu, small);
  large = __reduce_max_sync(0xffffffffu, large);
  sh.bucket[threadIdx.x] = 0;
  if (lane == 0) { sh.warp_i[warp] = (int)small; sh.warp_v[warp] = __uint_as_float(large); }
  __syncthreads();
  for (int w = 0; w < WARPS; ++w) {
    small = min(small, (unsigned)sh.warp_i[w]);
    large = max(large, __float_as_uint(sh.warp_v[w]));
  }
  const float top = value_of(large), per = fminf((float)BUCKETS / (top - value_of(small)), 1e37f);
  const auto bucket_of = [&](u64 c) {
    if (small == large) return (int)((long long)index_of(c) * BUCKETS / sh.n);
    return (int)fminf(fmaxf(top - logit_of(c), 0.f) * per, (float)(BUCKETS - 1));
  };
  unsigned at[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int i = e * NT + threadIdx.x;
    if (i < m) at[e] = atomicAdd(&sh.bucket[bucket_of(sh.list[i])], 1u);
  }
  __syncthreads();
  // where each bucket begins
  const unsigned own = sh.bucket[threadIdx.x];
  unsigned to = own;
  for (int o = 1; o < 32; o *= 2) {
    const unsigned t = __shfl_up_sync(0xffffffffu, to, o);
    if (lane >= o) to += t;
  }
  if (lane == 31) sh.warp_i[warp] = (int)to;
  // Many equal logits beside others, or a mask of a low finite value below a few: one bucket has nearly all, and its tokens
  // compared with one another would take longer than the network (1,900 equal ones beside one: 201 us a call, 41 by the
  // network).  Buckets of 32 and more occur in ordinary lists (700 of 32,003 16-bit logits: 18.6 us, 31.8 by the network).
  if (__syncthreads_or(own > CROWD)) {
    sort_network(m);
    return;
  }
  unsigned before = 0;
  for (int w = 0; w < warp; ++w) before += sh.warp_i[w];
  sh.bucket[threadIdx.x] = before + to - own;
  if (threadIdx.x == 0) sh.bucket[BUCKETS] = m;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int i = e * NT + threadIdx.x;
    if (i < m) {
      const u64 c = sh.list[i];
      sh.sorted[sh.bucket[bucket_of(c)] + at[e]] = c;
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int i = threadIdx.x; i < m; i += NT) {
    const u64 c = sh.sorted[i];
    const int b = bucket_of(c), end = sh.bucket[b + 1];
    int place = sh.bucket[b];
    for (int k = place; k < end; ++k) place += sh.sorted[k] > c;
    sh.list[place] = c;
  }
  __syncthreads();
}

// ---------------------------------------------------------------------------------------------------------- levels
// The bin, 1 / per wide, of a distance d from `from` on; the last one takes what lies deeper.
__device__ __forceinline__ int bin_of(float d, float from, float per) {
  const float t = fminf((d - from) * per, (float)(BINS - 1));
  return (int)(__float_as_uint(__fadd_rz(t, 8388608.f)) & 31u);
}

// Counts the tokens with c >= lo of the range [from, past) of distances in bins that are 1 / per wide; MASS: sums their masses.
template <typename T, bool MASS> __device__ __noinline__ void count_linear(u64 lo, float from, float past, float per) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const float lowest = logit_of(lo), largest = shared().largest, scale = shared().scale;
  const int n = shared().n;
  const bool ragged = (lo & (MAX_VOCAB - 1)) != 0;     // the tokens asked for begin among equal logits
  float* cells = &shared().cells[0][threadIdx.x];
#pragma unroll
  for (int b = 0; b < BINS; ++b) cells[b * NT] = 0.f;
  each<T, 4>([&](const auto& x, int at) {
    int bin[VEC];
    float share[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float y = asked<MASS>(x[i], at + i, n), d = below(y, largest);
      const bool in = y >= lowest && d >= from && !(d >= past);
      const float t = in ? fminf((d - from) * per, (float)(BINS - 1)) : (float)BINS;
      bin[i] = (int)(__float_as_uint(__fadd_rz(t, 8388608.f)) & 31u);
      share[i] = exp2_fast(-(d * scale));
    }
    if (ragged) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (x[i] == lowest && compose(clean(x[i]), at + i) < lo) bin[i] = BINS;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float& cell = cells[bin[i] * NT];
      cell = MASS ? cell + share[i] : __uint_as_float(__float_as_uint(cell) + 1u);
    }
  });
}
// The same of the tokens lo <= c <= hi, in bins of 2^shift composed numbers.
template <typename T, bool MASS> __device__ __noinline__ void count_composed(u64 lo, u64 hi, int shift) {
  const float largest = shared().largest, scale = shared().scale, lowest = logit_of(lo);
  const int n = shared().n;
  float* cells = &shared().cells[0][threadIdx.x];
#pragma unroll
  for (int b = 0; b < BINS; ++b) cells[b * NT] = 0.f;
  each<T, 2>([&](const auto& x, int at) {
#pragma unroll
    for (int i = 0; i < 16 / (int)sizeof(T); ++i) {
      const float y = asked<MASS>(x[i], at + i, n);
      if (!(y >= lowest)) continue;
      const u64 c = compose(clean(y), at + i);
      if (c < lo || c > hi) continue;
      float& cell = cells[(15 - (int)((c - lo) >> shift)) * NT];
      cell = MASS ? cell + exp2_fast(-(below(y, largest) * scale)) : __uint_as_float(__float_as_uint(cell) + 1u);
    }
  });
}

// After every block has counted: the sums of the bins over the blocks' threads go to every block.  Holds one barrier of the
// cluster.
template <bool MASS> __device__ __noinline__ void add_bins() {
  Shared& sh = shared();
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, blocks = sh.blocks, parity = sh.parity;
  for (int b = warp; b < BINS; b += WARPS) {
    float some[4] = {0.f, 0.f, 0.f, 0.f};
    unsigned c = 0;
#pragma unroll
    for (int t = 0; t < NT / 32; ++t) {
      const float v = sh.cells[b][t * 32 + lane];
      if (MASS) some[t % 4] += v;
      else c += __float_as_uint(v);
    }
    double q;
    if (MASS) {
      q = (double)((some[0] + some[1]) + (some[2] + some[3]));
      for (int o = 16; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
    } else {
      q = (double)__reduce_add_sync(0xffffffffu, c);
    }
    if (lane < blocks) *of(&sh.bins[parity][sh.rank][b], lane) = q;
  }
  sync_row();
}

// The smallest distance in bin b or deeper, of those from `from` to `to` (which is given where there is none).
static __device__ __noinline__ float first_distance(int b, float from, float to, float per) {
  const int lane = threadIdx.x & 31;
  unsigned a = __float_as_uint(from), z = __float_as_uint(to);
  // it lies within a few steps of where it would without rounding
  const float guess = from + (float)b / per;
  if (guess > from && guess < to) {
    const unsigned base = max(__float_as_uint(guess), 16u) - 16u, p = base + lane;
    const unsigned yes = __ballot_sync(0xffffffffu, bin_of(__uint_as_float(min(max(p, a), z - 1)), from, per) >= b);
    if (!(yes & 1u) && (yes >> 31)) { a = max(a, base); z = min(z, base + 31); }
  }
  while (a < z) {
    const unsigned step = (z - a + 31) / 32, p = min(z - 1, a + lane * step);
    const unsigned yes = __ballot_sync(0xffffffffu, bin_of(__uint_as_float(p), from, per) >= b);
    if (yes == 0) { a = min(z - 1, a + 31 * step) + 1; continue; }
    const int f = __ffs(yes) - 1;
    if (f == 0) return __uint_as_float(a);
    z = min(z - 1, a + f * step);
    a = min(z, a + (f - 1) * step) + 1;
  }
  return __uint_as_float(z);
}
// The smallest key from `a` to `z` whose value lies nearer to the largest logit than `to` (that of z does, or none).
static __device__ __noinline__ unsigned first_key(unsigned a, unsigned z, float to) {
  const int lane = threadIdx.x & 31;
  const float largest = shared().largest;
  // it lies within a step of where it would without rounding
  const float guess = largest - to, some = fmaxf(to, fabsf(largest)) * 2.4e-7f;
  const unsigned early = key_of(guess - some), late = key_of(guess + some);
  if (early >= a && late <= z && early < late && !(below(value_of(early), largest) < to) && below(value_of(late), largest) < to) {
    a = early + 1;
    z = late;
  }
  while (a < z) {
    const unsigned step = (z - a + 31) / 32, p = min(z - 1, a + lane * step);
    const unsigned yes = __ballot_sync(0xffffffffu, below(value_of(p), largest) < to);
    if (yes == 0) { a = min(z - 1, a + 31 * step) + 1; continue; }
    const int f = __ffs(yes) - 1;
    if (f == 0) return a;
    z = min(z - 1, a + f * step);
    a = min(z, a + (f - 1) * step) + 1;
  }
  return z;
}

// The first warp, after a level: takes the range over to the bin of the boundary, the last one that has tokens and before which
// the goal is not reached.
template <bool MASS> __device__ __noinline__ void take_bin(u64 lo, unsigned most, double goal, double part, double plenty, int depth) {
  Shared& sh = shared();
  Range& r = sh.range;
  const int lane = threadIdx.x & 31;
  const float largest = sh.largest, deepest = below(logit_of(lo), largest);
  // what lies above a lane's bin is what the lanes before it have
  double q = 0;
  if (lane < BINS)
    for (int k = 0; k < sh.blocks; ++k) q += sh.bins[sh.parity][k][lane];
  double sum = q;
  for (int o = 1; o < 32; o *= 2) {
    const double other = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += other;
  }
  const double all = depth == 0 ? __shfl_sync(0xffffffffu, sum, 31) : r.all;
  double above = __shfl_up_sync(0xffffffffu, sum, 1);
  above = r.above + (lane == 0 ? 0. : above);
  const double end = part >= 0. ? part * all : goal;
  const unsigned holds = __ballot_sync(0xffffffffu, lane < BINS && q > 0. && (above == 0. || above < end));
  const int b = holds ? 31 - __clz(holds) : 0;
  above = __shfl_sync(0xffffffffu, above, b);
  const double inside = __shfl_sync(0xffffffffu, q, b);
  const bool enough = depth == 0 && all <= plenty;

  float from = r.from, to = r.to, per = r.per, least;  // least: the deepest distance that the range may hold
  u64 low = r.lo, high = r.hi;
  bool composed = r.composed;
  if (!composed) {
    const float limit = fminf(to, HUGE_F);
    float first = from, last = to;
    if (b > 0) {
      first = first_distance(b, from, limit, per);
      if (first >= limit && bin_of(limit, from, per) < b) first = INFINITY;            // infinite distances alone
    }
    if (b < BINS - 1) {
      last = first_distance(b + 1, from, limit, per);
      if (last >= limit && bin_of(limit, from, per) <= b) last = to;
    }
    from = first;
    to = last;
    least = fminf(to, deepest);
  } else {
    low += (u64)(15 - b) << r.shift;
    const u64 last = low + ((1ull << r.shift) - 1);
    if (last < high) high = last;
    least = below(logit_of(low), largest);
  }
  // its tokens (where masses are summed, no fewer than that: no token of the range weighs less than one at its deepest)
  const unsigned count = MASS ? (unsigned)fmin(inside * (double)exp2f(least * sh.scale) * 1.0001 + 1., 4e9) : (unsigned)inside;
  const bool found = count <= most;
  if (!composed && !enough) {
    const float wide = fminf(to, deepest) - from;
    per = (float)BINS / wide;
    // (four levels of equal width at most: of logits that are cut off at one value 157 us for 64 rows, two levels 150, seven 189;
    // of many close to one another and a few far off 96, 98 and 96)
    if (found || depth > 3 || !(wide > 0.f && per > 0.f && per < 1e37f && wide > 1e-6f * fminf(to, deepest))) {
      // the logits crowd, or it is found: a range of composed numbers, of which the parts end with a single one
      const unsigned a = (unsigned)(lo >> INDEX_BITS), z = key_of(largest);
      const u64 bottom = to == INFINITY ? lo : (u64)first_key(a, z, to) << INDEX_BITS;
      if (from > 0.f) high = ((u64)first_key(a, z, from) << INDEX_BITS) - 1;
      low = bottom > lo ? bottom : lo;
      composed = true;
    }
  }
  __syncwarp();
  if (lane == 0)
    r = Range{low, high, from, to, fminf(per, 1e37f), max(0, 60 - __clzll((long long)(high - low))), composed, found, enough, above, all};
  if (lane == 0) sh.parity ^= 1;
}

// Finds the range of at most `most` tokens, among those with c >= lo, that holds the last token before which the goal is not
// reached: `goal` tokens, or (MASS) `part` of the mass of all tokens asked for.  range.all is what all of them make; where
// that is no more than `plenty`, nothing is looked for.  The first level's bins are 1 / per wide.
template <typename T, bool MASS> __device__ __noinline__ bool narrow(u64 lo, float per, unsigned most, double goal, double part, double plenty) {
  Shared& sh = shared();
  __syncthreads();
  if (threadIdx.x == 0) sh.range = Range{lo, compose(sh.largest, 0), 0.f, INFINITY, fminf(per, 1e37f), 0, false, false, false, 0., 0.};
  __syncthreads();
  for (int depth = 0;; ++depth) {
    if (sh.range.composed) count_composed<T, MASS>(sh.range.lo, sh.range.hi, sh.range.shift);
    else count_linear<T, MASS>(lo, sh.range.from, sh.range.to == INFINITY ? nan_f() : sh.range.to, sh.range.per);
    add_bins<MASS>();
    if (threadIdx.x < 32) take_bin<MASS>(lo, most, goal, part, plenty, depth);
    __syncthreads();
    if (sh.range.enough) return false;
    if (sh.range.found) return true;
  }
}

// The tokens of the range are put; above(values, index of the first) is called for every vector, by whole warps where WHOLE.
template <typename T, bool MASS, bool WHOLE, typename A> __device__ __forceinline__ void put_range(A&& above) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const u64 low = shared().range.lo, high = shared().range.hi;
  const float lowest = logit_of(low), highest = logit_of(high);
  const int n = shared().n;
  __syncthreads();                                     // the cells are read: their place is the list's too
  each<T, WHOLE ? 2 : 4, WHOLE>([&](const auto& x, int at) {
    bool any = false;
#pragma unroll
    for (int i = 0; i < VEC; ++i) any |= x[i] >= lowest && x[i] <= highest;
    if (any || lowest == -INFINITY) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float y = asked<MASS>(x[i], at + i, n);
        if (y >= lowest && y <= highest) {
          const u64 c = compose(clean(y), at + i);
          if (c >= low && c <= high) put(c);
        }
      }
    }
    above(x, at);
  });
}

}  // namespace vocab
