// Scaled embedding lookup, out[t] = scale * table[ids[t]], and its gradient, dtable[v] = scale * sum_{t: ids[t] = v} dout[t].
//
// Ids outside [0, rows) are padding: a row of zeros, no gradient.  Both directions are bound by memory: the lookup reads and
// writes each row once; the gradient reads dout once and writes every row of the table once.  The sums run in fp32 over the
// entries sorted by id (sort_ids.hip), each row summed by one group of threads in the order of its tokens, so the result does
// not depend on the run.  A row with more than `run` tokens would keep its group busy long after the others: its entries are cut
// into runs, summed by groups of their own into partial rows, and joined in order by a second launch.
//
// Measured: 16384 tokens of 32768 x 1024 bf16, lookup 10.4 us (67 MB, 6.4 TB/s: hot rows come from the caches), gradient 18.6 us (101 MB, 5.4
// TB/s) behind a sort of 15 and before a join of 5.4.  5003 tokens of 9973 x 331 fp32 (4-byte loads): 6, 16, 7.4 and 4 us.
#include "sort_ids.h"
#include <algorithm>

namespace sx {

// Entries a group of threads sums in a row: about 1024 runs, more for small groups, kMinRun entries at least.  A group's time
// is a chain of memory latencies, eight rows at a time (16384 tokens of 1024 bf16: 18 us in runs of 16, 48 us in runs of 64), that of a
// row's join grows with its runs.
constexpr int kMinRun = 16;
static inline int embed_run(int64_t n, int group) {
  int run = kMinRun;
  while ((int64_t)run * (group >= 64 ? 1024 : 4096) < n) run *= 2;
  return run;
}
// pieces of 16 bytes at most in a row that a group of 16 threads may take (embed_bwd_pick): longer ones have groups of 64 and more
constexpr int kSmallPieces = 16;
// runs, whatever the width of the loads: small groups, which a row of few pieces may have, have the most
static inline int64_t embed_max_runs(int64_t n, int dim) {
  const int run = embed_run(n, dim <= kSmallPieces * 8 ? 16 : 64);
  return n > run ? cdiv64(n, run) : 0;
}
constexpr int64_t kMaxRows = 1 << 24;      // the gradient's grid gives every row of the table up to 128 threads of a 2^32 limit

// E elements as one load or store
template <typename T, int E> struct Piece { typedef __attribute__((ext_vector_type(E))) T type; };
template <typename T> struct Piece<T, 1> { typedef T type; };
template <typename T, int E> __device__ __forceinline__ float piece_get(const typename Piece<T, E>::type& p, int e) {
  if constexpr (E == 1) return to_f32(p);
  else return to_f32(p[e]);
}
template <typename T, int E> __device__ __forceinline__ void piece_set(typename Piece<T, E>::type& p, int e, float v) {
  if constexpr (E == 1) p = from_f32<T>(v);
  else p[e] = from_f32<T>(v);
}

template <typename T, typename I, int E>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const T* __restrict__ table, int64_t ld, const I* __restrict__ ids, int64_t n,
                                                        int64_t rows, int dim, float scale, T* __restrict__ out) {
  typedef typename Piece<T, E>::type P;
  const int pieces = dim / E;
  const int64_t total = n * pieces;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t t = i / pieces;
    const int c = (int)(i - t * pieces) * E;
    const int64_t id = (int64_t)ids[t];
    const bool ok = id >= 0 && id < rows;
    const T* src = table + (ok ? id : 0) * ld + c;
    T* dst = out + t * dim + c;
    P v = {};
    if (ok) v = *reinterpret_cast<const P*>(src);
    const float by = ok ? scale : 0.f;                     // (padding stays 0 whatever the scale is)
#pragma unroll
    for (int e = 0; e < E; ++e) piece_set<T, E>(v, e, piece_get<T, E>(v, e) * by);
    *reinterpret_cast<P*>(dst) = v;
  }
}

struct EmbedBwdArgs {
  const void* dout; int64_t ld;
  const int* perm; const int* key; const int* start; const int* end;
  int64_t rows; int dim; int64_t n;
  float scale;
  void* dtable;
  float* part;              // [runs][2][dim]: the first and the last long row that a run of entries holds part of
  int run;                  // entries per run
  int64_t run_blocks;       // blocks behind those of the rows
};

// Columns of a thread: NC pieces of E elements, GROUP * E apart, from column c on.  Group = GROUP threads that share a row.
template <typename T, int E, int GROUP, int NC>
struct RowSum {
  typedef typename Piece<T, E>::type P;
  float acc[NC][E];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[k][e] = 0.f;
  }
  static __device__ __forceinline__ void load(P (&x)[NC], const T* __restrict__ row, int c, int dim) {
#pragma unroll
    for (int k = 0; k < NC; ++k)
      if (c + k * GROUP * E < dim) x[k] = *reinterpret_cast<const P*>(row + c + k * GROUP * E);
  }
  __device__ __forceinline__ void add(const P (&x)[NC], int c, int dim) {
#pragma unroll
    for (int k = 0; k < NC; ++k)
      if (c + k * GROUP * E < dim) {
#pragma unroll
        for (int e = 0; e < E; ++e) acc[k][e] += piece_get<T, E>(x[k], e);
      }
  }
  // += dout rows perm[a .. b), in that order, U of them in flight
  __device__ __forceinline__ void rows(const EmbedBwdArgs& q, int a, int b, int c) {
    constexpr int U = NC == 1 ? 8 : 4;
    const T* dout = (const T*)q.dout;
    for (int i = a; i < b; i += U) {
      P x[U][NC];
      int t[U];
#pragma unroll
      for (int u = 0; u < U; ++u) t[u] = q.perm[std::min(i + u, b - 1)];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u < b) load(x[u], dout + (int64_t)t[u] * q.ld, c, q.dim);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u < b) add(x[u], c, q.dim);
    }
  }
  __device__ __forceinline__ void put(const EmbedBwdArgs& q, int64_t v, int c, float scale) const {
    T* dst = (T*)q.dtable + v * q.dim + c;
#pragma unroll
    for (int k = 0; k < NC; ++k)
      if (c + k * GROUP * E < q.dim) {
        P o;
#pragma unroll
        for (int e = 0; e < E; ++e) piece_set<T, E>(o, e, acc[k][e] * scale);
        *reinterpret_cast<P*>(dst + k * GROUP * E) = o;
      }
  }
};

// Blocks [0, gridDim.x - run_blocks) take the rows of the table, ROWS per group; the others take the runs of long rows.  Where most rows have
// no token or one the loads of four rows are what keeps memory busy; where they have several, four after another take longer.  Row length 1024
// in bf16, 16384 tokens evenly and unevenly spread, by four and by one: 32768 rows 19 and 22 us, 16384 rows 16.0 and 15.7, 4000 rows 12.8 and
// 9.1, uneven 17 and 12; 65000 tokens of 1000 rows of 500, 47 and 20
template <typename T, int E, int GROUP, int NC, int ROWS>
__global__ __launch_bounds__(256) void embed_bwd_kernel(EmbedBwdArgs q) {
  typedef RowSum<T, E, GROUP, NC> Sum;
  constexpr int STEP = GROUP * E * NC;
  const int sub = threadIdx.x / GROUP, li = threadIdx.x % GROUP;
  const int64_t row_blocks = gridDim.x - q.run_blocks;
  if ((int64_t)blockIdx.x < row_blocks) {
    const int64_t v0 = (blockIdx.x * (int64_t)(256 / GROUP) + sub) * ROWS;
    if (v0 >= q.rows) return;
    int st[ROWS], en[ROWS], first[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      st[i] = q.start[std::min<int64_t>(v0 + i, q.rows)];
      en[i] = q.end[std::min<int64_t>(v0 + i, q.rows)];
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) first[i] = en[i] > st[i] ? q.perm[st[i]] : -1;
    for (int c = li * E; c < q.dim; c += STEP) {
      typename Sum::P x[ROWS][NC];
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
        if (first[i] >= 0) Sum::load(x[i], (const T*)q.dout + (int64_t)first[i] * q.ld, c, q.dim);
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        if (v0 + i >= q.rows || en[i] - st[i] > q.run) continue;
        Sum s;
        s.clear();
        if (first[i] >= 0) {
          s.add(x[i], c, q.dim);
          s.rows(q, st[i] + 1, en[i], c);
        }
        s.put(q, v0 + i, c, first[i] >= 0 ? q.scale : 0.f);
      }
    }
  } else {
    const int64_t run = (blockIdx.x - row_blocks) * (int64_t)(256 / GROUP) + sub;
    const int64_t e0 = run * q.run, e1 = std::min<int64_t>(q.n, e0 + q.run);
    if (e0 >= q.n) return;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int v = q.key[side ? e1 - 1 : e0];
      if (v >= q.rows) continue;
      const int a = q.start[v], b = q.end[v];
      if (b - a <= q.run) continue;
      if (side && a < e0) continue;                      // one long row fills the run: it is its first
      const int f = (int)std::max<int64_t>(a, e0), t = (int)std::min<int64_t>(b, e1);
      if (!side && a >= e0 && t == e1) continue;         // it begins in this run and goes on: it is its last
      for (int c = li * E; c < q.dim; c += STEP) {
        Sum s;
        s.clear();
        s.rows(q, f, t, c);
        float* dst = q.part + (run * 2 + side) * q.dim + c;
#pragma unroll
        for (int k = 0; k < NC; ++k)
          if (c + k * GROUP * E < q.dim)
#pragma unroll
            for (int e = 0; e < E; ++e) dst[k * GROUP * E + e] = s.acc[k][e];
      }
    }
  }
}

// The long row that begins in a run (its last one) = that run's last part + the first parts of the runs it goes on into.  One run per
// block: its 512 / GROUP groups take every so many parts and add up through LDS, in the order of the groups.
template <typename T, int E, int GROUP, int NC>
__global__ __launch_bounds__(512) void embed_join_kernel(EmbedBwdArgs q) {
  typedef RowSum<T, E, GROUP, NC> Sum;
  constexpr int STEP = GROUP * E * NC, SUBS = 512 / GROUP;
  __shared__ float part[SUBS][GROUP][NC * E];
  const int sub = threadIdx.x / GROUP, li = threadIdx.x % GROUP;
  const int64_t run = blockIdx.x, e0 = run * q.run, e1 = std::min<int64_t>(q.n, e0 + q.run);
  const int v = q.key[e1 - 1];
  if (v >= q.rows) return;
  const int a = q.start[v], b = q.end[v];
  if (b - a <= q.run || a < e0) return;
  const int64_t last = (b - 1) / q.run;
  for (int c = li * E; c - li * E < q.dim; c += STEP) {
    Sum s;
    s.clear();
    constexpr int U = NC * E <= 8 ? 8 : 4;              // parts in flight; no branch around a load, columns behind the last read the first
    for (int64_t r0 = run + sub; r0 <= last; r0 += SUBS * U) {
      float x[U][NC][E];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t r = std::min(r0 + u * SUBS, last);
        const float* p = q.part + (r * 2 + (r == run ? 1 : 0)) * q.dim;
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
          for (int e = 0; e < E; ++e) x[u][k][e] = p[(c + k * GROUP * E < q.dim ? c + k * GROUP * E : 0) + e];
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
          for (int e = 0; e < E; ++e) s.acc[k][e] += r0 + u * SUBS <= last ? x[u][k][e] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) part[sub][li][k * E + e] = s.acc[k][e];
    __syncthreads();
    if (sub == 0) {
      for (int o = 1; o < SUBS; ++o)
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
          for (int e = 0; e < E; ++e) s.acc[k][e] += part[o][li][k * E + e];
      s.put(q, v, c, q.scale);
    }
    __syncthreads();
  }
}

struct EmbedWs { size_t perm, key, start, end, part, total; };
static EmbedWs embed_ws(int64_t n, int64_t rows, int dim) {
  EmbedWs w;
  size_t o = 0;
  w.perm = o; o = align_up(o + (size_t)n * 4, 256);
  w.key = o; o = align_up(o + (size_t)n * 4, 256);
  w.start = o; o = align_up(o + (size_t)(rows + 1) * 4, 256);
  w.end = o; o = align_up(o + (size_t)(rows + 1) * 4, 256);
  w.part = o; o = align_up(o + (size_t)embed_max_runs(n, dim) * 2 * (size_t)dim * 4, 256);
  w.total = o;
  return w;
}

template <typename T, int E, int GROUP, int NC>
static int embed_bwd_launch(EmbedBwdArgs q, hipStream_t st) {
  const int per = 256 / GROUP;
  q.run = embed_run(q.n, GROUP);
  const int64_t runs = q.n > q.run ? cdiv64(q.n, q.run) : 0;
  q.run_blocks = cdiv64(runs, per);
  const int by = q.n >= q.rows ? 1 : 4;
  const dim3 grid((unsigned)(cdiv64(q.rows, per * by) + q.run_blocks));
  if (by == 1) hipLaunchKernelGGL((embed_bwd_kernel<T, E, GROUP, NC, 1>), grid, dim3(256), 0, st, q);
  else hipLaunchKernelGGL((embed_bwd_kernel<T, E, GROUP, NC, 4>), grid, dim3(256), 0, st, q);
  SX_LAUNCH_CHECK("embed_bwd");
  if (runs) {
    hipLaunchKernelGGL((embed_join_kernel<T, E, GROUP, NC>), dim3((unsigned)runs), dim3(512), 0, st, q);
    SX_LAUNCH_CHECK("embed_join");
  }
  return SX_OK;
}

template <typename T, int E>
static int embed_bwd_pick(const EmbedBwdArgs& q, hipStream_t st) {
  const int pieces = q.dim / E;
  if (pieces <= kSmallPieces) return embed_bwd_launch<T, E, 16, 1>(q, st);
  if (pieces <= 64) return embed_bwd_launch<T, E, 64, 1>(q, st);
  if (pieces <= 128) return embed_bwd_launch<T, E, 128, 1>(q, st);
  return embed_bwd_launch<T, E, 128, 4>(q, st);
}

// elements of the widest load, up to 16 bytes, that rows of this length and stride from these addresses allow
static int embed_width(int size, int dim, int64_t ld, const void* a, const void* b) {
  int e = 16 / size;
  while (e > 1 && (dim % e || ld % e || ((uintptr_t)a | (uintptr_t)b) % (e * size))) e /= 2;
  return e;
}

template <typename T>
static int embed_bwd(const EmbedBwdArgs& q, hipStream_t st) {
  switch (embed_width(sizeof(T), q.dim, q.ld, q.dout, q.dtable)) {
    case 1: return embed_bwd_pick<T, 1>(q, st);
    case 2: return embed_bwd_pick<T, 2>(q, st);
    case 4: return embed_bwd_pick<T, 4>(q, st);
    default: return embed_bwd_pick<T, 16 / (int)sizeof(T)>(q, st);
  }
}

template <typename T, typename I, int E>
static int embed_fwd_launch(const void* table, int64_t ld, const void* ids, int64_t n, int64_t rows, int dim, float scale, void* out, hipStream_t st) {
  const unsigned blocks = (unsigned)std::max<int64_t>(1, std::min<int64_t>(cdiv64(n * (dim / E), 256), 256 * 32));
  hipLaunchKernelGGL((embed_fwd_kernel<T, I, E>), dim3(blocks), dim3(256), 0, st, (const T*)table, ld, (const I*)ids, n, rows, dim, scale, (T*)out);
  SX_LAUNCH_CHECK("embed_fwd");
  return SX_OK;
}

template <typename T, typename I>
static int embed_fwd(const void* table, int64_t ld, const void* ids, int64_t n, int64_t rows, int dim, float scale, void* out, hipStream_t st) {
  switch (embed_width(sizeof(T), dim, ld, table, out)) {
    case 1: return embed_fwd_launch<T, I, 1>(table, ld, ids, n, rows, dim, scale, out, st);
    case 2: return embed_fwd_launch<T, I, 2>(table, ld, ids, n, rows, dim, scale, out, st);
    case 4: return embed_fwd_launch<T, I, 4>(table, ld, ids, n, rows, dim, scale, out, st);
    default: return embed_fwd_launch<T, I, 16 / (int)sizeof(T)>(table, ld, ids, n, rows, dim, scale, out, st);
  }
}

static int embed_check(const char* who, int dtype, int64_t n, int64_t rows, int dim, int64_t ld) {
  SX_REQUIRE(dtype == SX_F32 || dtype == SX_BF16, "%s: dtype %d is neither fp32 nor bf16", who, dtype);
  SX_REQUIRE(n >= 0 && n < (1ll << 31) - 1024 && rows > 0 && rows <= kMaxRows && dim > 0 && ld >= dim, "%s: bad sizes n=%lld rows=%lld dim=%d ld=%lld", who,
             (long long)n, (long long)rows, dim, (long long)ld);
  return SX_OK;
}

}  // namespace sx

using namespace sx;

extern "C" int64_t sx_embedding_workspace_bytes(int64_t n, int64_t rows, int dim) {
  SX_TRY(embed_check("sx_embedding_workspace_bytes", SX_F32, n, rows, dim, dim));
  return (int64_t)embed_ws(n, rows, dim).total;
}

extern "C" int sx_embedding_forward(int dtype, int64_t n, int64_t rows, int dim, const void* table, int64_t ld, const void* ids, int ids64,
                                    float scale, void* out, void* stream) {
  SX_TRY(embed_check("sx_embedding_forward", dtype, n, rows, dim, ld));
  if (n == 0) return SX_OK;
  SX_REQUIRE(table && ids && out, "sx_embedding_forward: null pointer");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == SX_BF16)
    return ids64 ? embed_fwd<bf16, int64_t>(table, ld, ids, n, rows, dim, scale, out, st) : embed_fwd<bf16, int32_t>(table, ld, ids, n, rows, dim, scale, out, st);
  return ids64 ? embed_fwd<float, int64_t>(table, ld, ids, n, rows, dim, scale, out, st) : embed_fwd<float, int32_t>(table, ld, ids, n, rows, dim, scale, out, st);
}

extern "C" int sx_embedding_backward(int dtype, int64_t n, int64_t rows, int dim, const void* dout, int64_t ld, const void* ids, int ids64,
                                     float scale, void* dtable, void* workspace, int64_t workspace_bytes, void* stream) {
  SX_TRY(embed_check("sx_embedding_backward", dtype, n, rows, dim, ld));
  SX_REQUIRE(dtable && workspace && (n == 0 || (dout && ids)), "sx_embedding_backward: null pointer");
  const EmbedWs w = embed_ws(n, rows, dim);
  SX_REQUIRE(workspace_bytes >= (int64_t)w.total && (uintptr_t)workspace % 16 == 0, "sx_embedding_backward: workspace of %lld bytes, %lld needed, 16-byte aligned",
             (long long)workspace_bytes, (long long)w.total);
  char* ws = (char*)workspace;
  EmbedBwdArgs q = {};
  q.dout = dout; q.ld = ld; q.rows = rows; q.dim = dim; q.n = n; q.scale = scale; q.dtable = dtable;
  q.perm = (int*)(ws + w.perm); q.key = (int*)(ws + w.key); q.start = (int*)(ws + w.start); q.end = (int*)(ws + w.end); q.part = (float*)(ws + w.part);
  hipStream_t st = (hipStream_t)stream;
  SX_TRY(launch_sort_ids(ids, ids64, n, rows, (int*)q.perm, (int*)q.key, (int*)q.start, (int*)q.end, st));
  return dtype == SX_BF16 ? embed_bwd<bf16>(q, st) : embed_bwd<float>(q, st);
}
