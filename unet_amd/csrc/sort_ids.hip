// Stable counting sort of ids in one launch.
//
// A block owns some of the buckets and reads ALL the ids: first it counts its own buckets and the ids of the blocks before it (which is
// where its output begins), then it places its own.  Blocks therefore depend on nothing but the input, and the n * 4 or 8 bytes that each
// of them reads come from L2 after the first.  A block's time goes with the entries it places: with `spread` it owns every
// 2^shift-th bucket rather than a range, so that neighbouring frequent ids (the usual order of a vocabulary) lie in different blocks --
// 16384 ids of which half lie in one range of 256: 25 us by ranges.  Order within a bucket: a wave owns a contiguous part
// of the ids and each (wave, bucket) has its own counter, so an entry's place is the waves before, the earlier entries of its own
// wave and its rank among the lanes -- no atomic whose order could show.
#include "sort_ids.h"
#include <algorithm>
#include <type_traits>

namespace sx {

constexpr int kSortWaves = 16;          // 1024 threads
constexpr int kSortBuckets = 1024;      // buckets per block: one per thread in the scan, 64 KB of counters
constexpr int kSortUnroll = 8;          // loads in flight per lane
constexpr int kSortKeep = 16;           // ids per lane that stay in registers from the first pass to the second

// f(0), f(1) ... f(N - 1) with constant arguments: an array indexed by them stays in registers (#pragma unroll leaves loops around
// cross-lane operations rolled, and the array in memory)
template <int N, int I = 0, typename F>
__device__ __forceinline__ void unrolled(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>());
    unrolled<N, I + 1>(static_cast<F&&>(f));
  }
}

// Which block owns a bucket b and under which number: (b >> own_shift) & own_mask and (b >> num_shift) & num_mask
struct SortMap { int own_shift, own_mask, num_shift, num_mask, bits; };

// KEEP: a wave's part is at most 64 * kSortKeep ids and is read once
template <typename I, bool KEEP>
__global__ __launch_bounds__(1024) void sort_ids_kernel(const I* __restrict__ ids, int64_t n, int rows, SortMap q,
                                                        int* __restrict__ perm, int* __restrict__ key, int* __restrict__ start,
                                                        int* __restrict__ end) {
  __shared__ int cnt[kSortWaves][kSortBuckets];
  __shared__ int red[2][kSortWaves];
  constexpr int U = KEEP ? kSortKeep : kSortUnroll;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int me = blockIdx.x;
  auto bucket = [&](int num) { return me << q.own_shift | num << q.num_shift; };
  const bool mine = tid < (1 << q.bits) && bucket(tid) <= rows;      // thread = one of the block's buckets
  const int64_t seg = (n + 1023) / 1024 * 64;              // this wave's part, a multiple of the lanes
  const int64_t s0 = std::min<int64_t>(n, wid * seg), s1 = std::min<int64_t>(n, s0 + seg);
  int r[U], below = 0;                                     // this block's bucket of an id, -1 for another block's
  auto load = [&](int64_t t0, bool count) {
    I id[U];
    unrolled<U>([&](auto u) {
      const int64_t t = t0 + u * 64 + lane;
      id[u] = ids[t < s1 ? t : 0];
    });
    unrolled<U>([&](auto u) {
      const bool in = t0 + u * 64 + lane < s1;
      const int b = id[u] >= 0 && id[u] < (I)rows ? (int)id[u] : rows;
      const int own = (b >> q.own_shift) & q.own_mask;
      r[u] = in && own == me ? (b >> q.num_shift) & q.num_mask : -1;
      if (count) below += in && own < me ? 1 : 0;
    });
  };
  auto each = [&](auto&& f) {
    for (int64_t t0 = s0; t0 < s1; t0 += 64 * U) f(t0);
  };
  if constexpr (KEEP)
    if (n > 0) load(s0, true);
  for (int w = 0; w < kSortWaves; ++w) cnt[w][tid] = 0;
  __syncthreads();
  each([&](int64_t t0) {
    if constexpr (!KEEP) load(t0, true);
    if (q.bits == 0) {                                     // one bucket per block: counted without atomics
      int c = 0;
      unrolled<U>([&](auto u) { c += __popcll(__ballot(r[u] >= 0)); });
      if (lane == 0) cnt[wid][0] += c;
      return;
    }
    unrolled<U>([&](auto u) {
      if (r[u] >= 0) atomicAdd(&cnt[wid][r[u]], 1);
    });
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) below += __shfl_xor(below, o, 64);
  if (lane == 0) red[0][wid] = below;
  __syncthreads();
  // exclusive scan over this block's buckets, one per thread
  int tot = 0;
  if (mine)
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
  if (mine) {
    start[bucket(tid)] = base;
    end[bucket(tid)] = base + tot;
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = cnt[w][tid];
      cnt[w][tid] = base;
      base += c;
    }
  }
  __syncthreads();
  int next = cnt[wid][0];                                  // one bucket per block: where this wave's next entry goes
  each([&](int64_t t0) {
    if constexpr (!KEEP) load(t0, false);
    if (q.bits == 0) {
      unrolled<U>([&](auto u) {
        const unsigned long long same = __ballot(r[u] >= 0);
        if (r[u] >= 0) {
          const int p = next + __popcll(same & ((1ull << lane) - 1));
          perm[p] = (int)(t0 + u * 64 + lane);
          key[p] = me;
        }
        next += __popcll(same);
      });
      return;
    }
    unrolled<U>([&](auto u) {
      const int ru = r[u];
      unsigned long long same = __ballot(ru >= 0);
      if (!same) return;
      for (int k = same & (same - 1) ? 0 : q.bits; k < q.bits; ++k) {      // the lanes with this lane's bucket: one ballot per bit of its number
        const unsigned long long on = __ballot(ru >> k & 1);
        same &= (ru >> k & 1) ? on : ~on;
      }
      const int lead = __ffsll(same) - 1;
      int at = 0;
      if (ru >= 0 && lane == lead) at = atomicAdd(&cnt[wid][ru], __popcll(same));
      at = __shfl(at, lead & 63, 64);
      if (ru >= 0) {
        const int p = at + __popcll(same & ((1ull << lane) - 1));
        perm[p] = (int)(t0 + u * 64 + lane);
        key[p] = bucket(ru);
      }
    });
  });
}

template <typename I>
static void sort_launch(const void* ids, int64_t n, int rows, const SortMap& q, int blocks, int* perm, int* key, int* start, int* end, hipStream_t st) {
  if (n <= 1024 * kSortKeep) hipLaunchKernelGGL((sort_ids_kernel<I, true>), dim3(blocks), dim3(1024), 0, st, (const I*)ids, n, rows, q, perm, key, start, end);
  else hipLaunchKernelGGL((sort_ids_kernel<I, false>), dim3(blocks), dim3(1024), 0, st, (const I*)ids, n, rows, q, perm, key, start, end);
}

int launch_sort_ids(const void* ids, int ids64, int64_t n, int64_t rows, bool spread, int* perm, int* key, int* start, int* end, hipStream_t st) {
  // about 256 blocks, a power of two of buckets each
  SortMap q = {};
  while (q.bits < 10 && ((rows + 1) >> q.bits) > 256) ++q.bits;
  int blocks = (int)cdiv64(rows + 1, 1ll << q.bits);
  if (spread) {
    int s = 0;
    while ((1 << s) < blocks) ++s;
    q.own_mask = (1 << s) - 1;
    q.num_shift = s;
    q.num_mask = -1;
    blocks = (int)std::min<int64_t>(rows + 1, 1ll << s);
  } else {
    q.own_shift = q.bits;
    q.own_mask = -1;
    q.num_mask = (1 << q.bits) - 1;
  }
  if (ids64) sort_launch<int64_t>(ids, n, (int)rows, q, blocks, perm, key, start, end, st);
  else sort_launch<int32_t>(ids, n, (int)rows, q, blocks, perm, key, start, end, st);
  SX_LAUNCH_CHECK("sort_ids");
  return SX_OK;
}

}  // namespace sx
