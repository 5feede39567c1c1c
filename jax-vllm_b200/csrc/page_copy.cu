// Copies of pages of a cache, and of rows of per-request state: what a fork of a request takes over, and what a pool of
// another size takes from the old one.
//   to[l][dst[i]][0 .. bytes_i) = from[l][src[i]][0 .. bytes_i)      for every plane, layer l of it and pair i
// A plane is a tensor [layers, pages, bytes of a page]; bytes_i is the whole page, or the first tokens of it.  The
// caller sees to it that no page is written twice and none both read and written.
//
// Bound by memory: every byte is read once and written once (a source with several destinations comes from L2 after
// its first read).  A warp takes one piece of PIECE bytes at a time, 16 bytes a lane and eight loads in flight before the
// first store, so that the few pieces of a single page still spread over many multiprocessors.  The pairs travel as
// parameters of the launch: no copy to the device, no workspace, and a captured launch keeps its own.
// 1,500 pages of 28 layers (5.5 GB moved) in 860 us, 6.40 TB/s; 64 pages of 36 layers 50 us, 6.0 TB/s; one page of 36 layers to
// three others 3.3 us, of which 0.9 are bytes; eight rows of 24 state tensors to three others each 69 us, 5.8 TB/s.
#include "common.cuh"

namespace {

constexpr int THREADS = 256, UNROLL = 8;

struct Plane {
  const char* from;
  char* to;
  long long from_layer, from_page, to_layer, to_page;  // bytes from one to the next
  long long page_bytes, token_bytes;
  int layers;
};

struct Pair { int src, dst, tokens; };                 // tokens < 0: the whole page
struct Pairs { const int *src, *dst, *tokens; int n; };   // on the host; tokens may be null: whole pages

template <int PLANES, int PAIRS> struct Job {
  Plane plane[PLANES];
  long long first[PLANES + 1];                         // pieces of the planes before
  Pair pair[PAIRS];
  int planes, pairs;
};

template <typename V, int PLANES, int PAIRS>
__global__ void __launch_bounds__(THREADS) page_copy_kernel(const __grid_constant__ Job<PLANES, PAIRS> job) {
  constexpr int PIECE = 32 * UNROLL * (int)sizeof(V);
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long warps = (long long)gridDim.x * (THREADS / 32);
  const long long total = job.first[job.planes];
  int p = 0;
  for (long long item = (long long)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5); item < total; item += warps) {
    while (item >= job.first[p + 1]) ++p;
    const Plane& pl = job.plane[p];
    const long long pieces = (pl.page_bytes + PIECE - 1) / PIECE;
    long long rest = item - job.first[p];
    const long long piece = rest % pieces;
    rest /= pieces;
    const Pair pr = job.pair[rest % job.pairs];
    const long long layer = rest / job.pairs;
    const long long end = pr.tokens < 0 ? pl.page_bytes : pr.tokens * pl.token_bytes;
    const long long at = piece * PIECE;
    if (at >= end) continue;
    const V* from = reinterpret_cast<const V*>(pl.from + layer * pl.from_layer + pr.src * pl.from_page + at);
    V* to = reinterpret_cast<V*>(pl.to + layer * pl.to_layer + pr.dst * pl.to_page + at);
    const int n = (int)(min((long long)PIECE, end - at) / (long long)sizeof(V));
    V v[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (u * 32 + lane < n) v[u] = from[u * 32 + lane];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (u * 32 + lane < n) to[u * 32 + lane] = v[u];
  }
}

template <typename V, int PLANES, int PAIRS>
int copy_some(const Plane* planes, int n_planes, const Pairs& pairs, int first, int n_pairs, cudaStream_t stream) {
  constexpr long long PIECE = 32 * UNROLL * (long long)sizeof(V);
  Job<PLANES, PAIRS> job;
  job.planes = n_planes;
  job.pairs = n_pairs;
  long long total = 0;
  for (int p = 0; p < n_planes; ++p) {
    job.plane[p] = planes[p];
    job.first[p] = total;
    total += (planes[p].page_bytes + PIECE - 1) / PIECE * planes[p].layers * n_pairs;
  }
  job.first[n_planes] = total;
  for (int i = 0; i < n_pairs; ++i)
    job.pair[i] = Pair{pairs.src[first + i], pairs.dst[first + i], pairs.tokens != nullptr ? pairs.tokens[first + i] : -1};
  if (total == 0) return JV_OK;
  const long long wanted = (total + THREADS / 32 - 1) / (THREADS / 32), most = (long long)jv_multiprocessors() * 8;
  return jv_launch(page_copy_kernel<V, PLANES, PAIRS>, dim3((unsigned)(wanted < most ? wanted : most)), dim3(THREADS), 0, stream, job);
}

// Parameters of a launch are copied with it: as few as serve (0.8 KB to 18 KB).
constexpr int FEW_PLANES = 4, FEW_PAIRS = 32, MANY_PLANES = 64, MANY_PAIRS = 1024;

template <typename V>
int copy_all(const Plane* planes, int n_planes, const Pairs& pairs, cudaStream_t stream) {
  for (int p = 0; p < n_planes; p += MANY_PLANES)
    for (int i = 0; i < pairs.n; i += MANY_PAIRS) {
      const int np = n_planes - p < MANY_PLANES ? n_planes - p : MANY_PLANES, ni = pairs.n - i < MANY_PAIRS ? pairs.n - i : MANY_PAIRS;
      const bool few_planes = np <= FEW_PLANES, few_pairs = ni <= FEW_PAIRS;
      const int rc = few_planes && few_pairs ? copy_some<V, FEW_PLANES, FEW_PAIRS>(planes + p, np, pairs, i, ni, stream)
                     : few_planes            ? copy_some<V, FEW_PLANES, MANY_PAIRS>(planes + p, np, pairs, i, ni, stream)
                     : few_pairs             ? copy_some<V, MANY_PLANES, FEW_PAIRS>(planes + p, np, pairs, i, ni, stream)
                                             : copy_some<V, MANY_PLANES, MANY_PAIRS>(planes + p, np, pairs, i, ni, stream);
      if (rc != JV_OK) return rc;
    }
  return JV_OK;
}

}  // namespace

// planes: n_planes records of nine int64: from, to, from_layer, from_page, to_layer, to_page, page_bytes, token_bytes, layers.
// src, dst, tokens: n_pairs int32 each (tokens null: whole pages).  All on the host.
JV_EXPORT int jv_page_copy(const long long* planes, int n_planes, const int* src, const int* dst, const int* tokens, int n_pairs,
                           cudaStream_t stream) {
  if (n_planes <= 0 || n_pairs <= 0) return JV_OK;
  const Pairs pairs{src, dst, tokens, n_pairs};
  constexpr int SOME = 64;
  Plane buf[SOME];
  for (int base = 0; base < n_planes; base += SOME) {
    const int n = n_planes - base < SOME ? n_planes - base : SOME;
    unsigned long long all = 0;                        // whatever a byte offset may be made of
    for (int p = 0; p < n; ++p) {
      const long long* r = planes + 9 * (base + p);
      buf[p] = Plane{reinterpret_cast<const char*>(r[0]), reinterpret_cast<char*>(r[1]), r[2], r[3], r[4], r[5], r[6], r[7], (int)r[8]};
      for (int k = 0; k < 8; ++k) all |= (unsigned long long)r[k];
    }
    const int rc = all % 16 == 0  ? copy_all<uint4>(buf, n, pairs, stream)
                   : all % 4 == 0 ? copy_all<uint32_t>(buf, n, pairs, stream)
                   : all % 2 == 0 ? copy_all<uint16_t>(buf, n, pairs, stream)
                                  : copy_all<uint8_t>(buf, n, pairs, stream);
    if (rc != JV_OK) return rc;
  }
  return JV_OK;
}
