// Stable counting sort of ids in one launch.
//
// A block owns a contiguous range of buckets and reads ALL the ids, twice: first it counts its own buckets and the ids below its
// range (which is where its output begins), then it places its own.  Blocks therefore depend on nothing but the input, and the
// n * 4 or 8 bytes that each of them reads come from L2 after the first.  Order within a bucket: a wave owns a contiguous part
// of the ids and each (wave, bucket) has its own counter, so an entry's place is the waves before, the earlier entries of its own
// wave and its rank among the lanes -- no atomic whose order could show.
#include "sort_ids.h"
#include <algorithm>

namespace sx {

constexpr int kSortWaves = 16;          // 1024 threads
constexpr int kSortBuckets = 1024;      // buckets per block: one per thread in the scan, 64 KB of counters
constexpr int kSortUnroll = 8;          // loads in flight per lane

template <typename I>
__global__ __launch_bounds__(1024) void sort_ids_kernel(const I* __restrict__ ids, int64_t n, int64_t rows, int per_block,
                                                        int* __restrict__ perm, int* __restrict__ key, int* __restrict__ start) {
  __shared__ int cnt[kSortWaves][kSortBuckets];
  __shared__ int red[2][kSortWaves];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int64_t lo = (int64_t)blockIdx.x * per_block;
  const int nb = (int)(rows + 1 - lo < per_block ? rows + 1 - lo : per_block);
  for (int w = 0; w < kSortWaves; ++w)
    if (tid < nb) cnt[w][tid] = 0;
  __syncthreads();
  const int64_t seg = (n + 1023) / 1024 * 64;              // this wave's part, a multiple of the lanes
  const int64_t s0 = std::min<int64_t>(n, wid * seg), s1 = std::min<int64_t>(n, s0 + seg);
  int below = 0;
  for (int64_t t0 = s0; t0 < s1; t0 += 64 * kSortUnroll) {
    int64_t b[kSortUnroll];
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      const int64_t t = t0 + u * 64 + lane;
      const int64_t id = t < s1 ? (int64_t)ids[t] : -1;
      b[u] = t >= s1 ? rows + 1 : (id < 0 || id >= rows ? rows : id);
    }
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      below += b[u] < lo ? 1 : 0;
      if (b[u] >= lo && b[u] < lo + nb) atomicAdd(&cnt[wid][(int)(b[u] - lo)], 1);
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) below += __shfl_xor(below, o, 64);
  if (lane == 0) red[0][wid] = below;
  __syncthreads();
  // exclusive scan over this block's buckets, one per thread
  int tot = 0;
  if (tid < nb)
    for (int w = 0; w < kSortWaves; ++w) tot += cnt[w][tid];
  int inc = tot;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(inc, o, 64);
    if (lane >= o) inc += v;
  }
  if (lane == 63) red[1][wid] = inc;
  __syncthreads();
  int base = 0;
  for (int w = 0; w < kSortWaves; ++w) {
    base += red[0][w];
    if (w < wid) base += red[1][w];
  }
  base += inc - tot;
  if (tid < nb) {
    start[lo + tid] = base;
    if (lo + tid == rows) start[rows + 1] = (int)n;
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = cnt[w][tid];
      cnt[w][tid] = base;
      base += c;
    }
  }
  __syncthreads();
  for (int64_t t0 = s0; t0 < s1; t0 += 64 * kSortUnroll) {
    int64_t b[kSortUnroll];
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      const int64_t t = t0 + u * 64 + lane;
      const int64_t id = t < s1 ? (int64_t)ids[t] : -1;
      b[u] = t >= s1 ? rows + 1 : (id < 0 || id >= rows ? rows : id);
    }
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      const int r = (b[u] >= lo && b[u] < lo + nb) ? (int)(b[u] - lo) : -1;
      unsigned long long todo = __ballot(r >= 0);
      while (todo) {                                       // one round per distinct bucket among the 64 lanes
        const int lead = __ffsll(todo) - 1;
        const int rl = __shfl(r, lead, 64);
        const unsigned long long same = __ballot(r == rl);
        int at = 0;
        if (lane == lead) at = atomicAdd(&cnt[wid][rl], __popcll(same));
        at = __shfl(at, lead, 64);
        if (r == rl) {
          const int p = at + __popcll(same & ((1ull << lane) - 1));
          perm[p] = (int)(t0 + u * 64 + lane);
          if (key) key[p] = (int)(lo + rl);
        }
        todo &= ~same;
      }
    }
  }
}

int launch_sort_ids(const void* ids, int ids64, int64_t n, int64_t rows, int* perm, int* key, int* start, hipStream_t st) {
  // enough blocks that a block's buckets hold few of the ids, no more than two per CU unless the counters need them
  const int64_t want = std::max<int64_t>(cdiv64(rows + 1, kSortBuckets), std::min<int64_t>(rows + 1, 512));
  const int per_block = (int)cdiv64(rows + 1, want);
  const int64_t blocks = cdiv64(rows + 1, per_block);
  if (ids64) hipLaunchKernelGGL(sort_ids_kernel<int64_t>, dim3((unsigned)blocks), dim3(1024), 0, st, (const int64_t*)ids, n, rows, per_block, perm, key, start);
  else hipLaunchKernelGGL(sort_ids_kernel<int32_t>, dim3((unsigned)blocks), dim3(1024), 0, st, (const int32_t*)ids, n, rows, per_block, perm, key, start);
  SX_LAUNCH_CHECK("sort_ids");
  return SX_OK;
}

}  // namespace sx
