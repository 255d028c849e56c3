// Stable counting sort of ids in one launch.
//
// A block owns a range of the buckets and reads ALL the ids, so that it depends on nothing but the input: it counts the ids of the blocks
// before it (which is where its output begins) and keeps its own in LDS, and only those, dense, are counted by bucket and placed.  A
// wave owns a contiguous part of the ids, and each (wave, bucket) has its own counter, so an entry's place is the waves before, the
// earlier entries of its own wave and its rank among the lanes -- no atomic whose order could show.
//
// Bound by latencies (a launch of this size alone is 4 us): 1024 ids 9 us, 16384 int64 ids over 32768 buckets 13 us evenly spread, 15 us with
// most of them in few buckets, 15 to 20 us all in one, 65536 45 us.  With every id of the block handled in place, 64 to a step whatever
// their number, the same were 14, 17, 22, 32 and 69 us.  Only a wave whose list cannot hold what the block owns of its part (16 million ids
// and more, or nearly all of them in one block's buckets) reads its part again.
//
// Up to 2^18 rows there are about 256 blocks, one a CU.  Beyond, a block has its 1024 buckets and there are rows / 1024 of them, all of which
// read all the ids: the work is n * rows / 1024 reads, from the caches.  The embedding's gradient, dominated by this, takes 0.36 ms for 65536
// ids of 2^22 rows, 1.3 ms of 2^24, 10 ms for 2^20 ids of 2^24 rows (16385 blocks of 8 MB each; the same ids of 2^18 rows: 0.39 ms).
#include "sort_ids.h"
#include <algorithm>
#include <atomic>

namespace sx {

constexpr int kSortWaves = 16;          // 1024 threads
constexpr int kSortBuckets = 1024;      // buckets per block: one per thread in the scan, 64 KB of counters
constexpr int kSortLds = 160 * 1024;    // counters, 2 * kSortWaves sums, and the rest for the lists

template <typename I>
__global__ __launch_bounds__(1024) void sort_ids_kernel(const I* __restrict__ ids, int64_t n, int rows, int bits, int* __restrict__ perm,
                                                        int* __restrict__ key, int* __restrict__ start, int* __restrict__ end) {
  extern __shared__ int lds[];
  constexpr int U = 8;                                     // loads in flight per lane
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int buckets = 1 << bits, cap = ((kSortLds / 4 - 2 * kSortWaves) / kSortWaves - buckets) & ~63;      // cap: entries of a wave's list
  int(*const red)[kSortWaves] = reinterpret_cast<int(*)[kSortWaves]>(lds);      // [2]
  int* const cnt = lds + 2 * kSortWaves;                   // [wave][bucket]
  int* const mycnt = cnt + wid * buckets;
  int* const list = cnt + kSortWaves * buckets + wid * cap;      // this wave's: entry << 10 | bucket, within what was gathered / the block
  const int me = blockIdx.x, first = me << bits;
  const bool mine = tid < buckets && first + tid <= rows;      // thread = one of the block's buckets
  const int64_t seg = (n + 1023) / 1024 * 64;              // this wave's part, a multiple of the lanes
  const int64_t s0 = std::min<int64_t>(n, wid * seg), s1 = std::min<int64_t>(n, s0 + seg);
  for (int i = tid; i < kSortWaves * buckets; i += 1024) cnt[i] = 0;
  int below = 0, len = 0;
  // the block's own ids among the `part` from t0 on -> list, in their order; len: how many there are, more than cap if they did not fit
  auto gather = [&](int64_t t0, int part, bool count) {
    len = 0;
    for (int p = 0; p < part; p += 64 * U) {
      I id[U];
#pragma unroll
      for (int u = 0; u < U; ++u) id[u] = ids[t0 + std::min(p + u * 64 + lane, part - 1)];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool in = p + u * 64 + lane < part;
        const int b = id[u] >= 0 && id[u] < (I)rows ? (int)id[u] : rows;
        const bool own = in && b >> bits == me;
        if (count) below += in && b < first ? 1 : 0;
        const unsigned long long all = __ballot(own);
        const int at = len + __popcll(all & ((1ull << lane) - 1));
        if (own && at < cap) list[at] = (p + u * 64 + lane) << 10 | (b - first);
        len += __popcll(all);
      }
    }
  };
  auto tally = [&]() {
    for (int i = lane; i - lane < len; i += 64) {
      const bool in = i < len;
      const int r = in ? list[i] & (kSortBuckets - 1) : -1, r0 = __builtin_amdgcn_readfirstlane(r);
      const unsigned long long all = __ballot(in);
      if (all == __ballot(r == r0)) {                      // one bucket: 64 additions to one address take 64 turns
        if (lane == 0) atomicAdd(&mycnt[r0], __popcll(all));
      } else if (in) {
        atomicAdd(&mycnt[r], 1);
      }
    }
  };
  // each(f): f for this wave's ids, whole if its list holds the block's own of them, else cap at a time
  bool whole = false;
  auto each = [&](bool again, auto&& f) {
    if (whole) { f(s0); return; }
    for (int64_t t0 = s0; t0 < s1; t0 += cap) {
      gather(t0, (int)std::min<int64_t>(cap, s1 - t0), !again && s1 - s0 > (1 << 20));
      f(t0);
    }
  };
  __syncthreads();
  if (s1 - s0 <= 1 << 20) {                                // (an entry has 22 bits)
    gather(s0, (int)(s1 - s0), true);
    whole = len <= cap;
  }
  each(false, [&](int64_t) { tally(); });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) below += __shfl_xor(below, o, 64);
  if (lane == 0) red[0][wid] = below;
  __syncthreads();
  // exclusive scan over this block's buckets, one per thread
  int tot = 0;
  if (mine)
    for (int w = 0; w < kSortWaves; ++w) tot += cnt[w * buckets + tid];
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
    start[first + tid] = base;
    end[first + tid] = base + tot;
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = cnt[w * buckets + tid];
      cnt[w * buckets + tid] = base;
      base += c;
    }
  }
  __syncthreads();
  each(true, [&](int64_t t0) {
    for (int i = lane; i - lane < len; i += 64) {
      const bool in = i < len;
      const int e = in ? list[i] : -1, r = e & (kSortBuckets - 1);
      unsigned long long same = __ballot(in);
      const int r0 = __builtin_amdgcn_readfirstlane(r);    // (the first lane always holds an entry)
      for (int k = same == __ballot(in && r == r0) ? bits : 0; k < bits; ++k) {      // the lanes with this lane's bucket: one ballot per bit of its number
        const unsigned long long on = __ballot(r >> k & 1);
        same &= (r >> k & 1) ? on : ~on;
      }
      const int lead = __ffsll(same) - 1;
      int at = 0;
      if (in && lane == lead) at = atomicAdd(&mycnt[r], __popcll(same));
      at = __shfl(at, lead & 63, 64);
      if (in) {
        const int p = at + __popcll(same & ((1ull << lane) - 1));
        perm[p] = (int)t0 + (e >> 10);
        key[p] = first + r;
      }
    }
  });
}

template <typename I>
static int sort_launch(const void* ids, int64_t n, int rows, int bits, int* perm, int* key, int* start, int* end, hipStream_t st) {
  static std::atomic<unsigned long long> done{0};
  SX_TRY(ensure_max_lds((const void*)sort_ids_kernel<I>, done, "sort_ids"));
  hipLaunchKernelGGL(sort_ids_kernel<I>, dim3((unsigned)cdiv64(rows + 1, 1ll << bits)), dim3(1024), kSortLds, st, (const I*)ids, n, rows, bits, perm, key, start, end);
  SX_LAUNCH_CHECK("sort_ids");
  return SX_OK;
}

int launch_sort_ids(const void* ids, int ids64, int64_t n, int64_t rows, int* perm, int* key, int* start, int* end, hipStream_t st) {
  // about 256 blocks, a power of two of buckets each, as long as those are no more than a block holds
  int bits = 0;
  while (bits < 10 && ((rows + 1) >> bits) > 256) ++bits;
  return ids64 ? sort_launch<int64_t>(ids, n, (int)rows, bits, perm, key, start, end, st)
               : sort_launch<int32_t>(ids, n, (int)rows, bits, perm, key, start, end, st);
}

}  // namespace sx
