// Low-rank adapters of many requests beside one shared projection.  Row t of a batch belongs to adapter a = ids[t] (or to none):
//
//   h[t]  = s_a A_a x[t]                   (r numbers)          y[t]  = W x[t] + b + B_a h[t]
//   dh[t] = s_a B_a^T dy[t]                                     dx[t] = W^T dy[t] + A_a^T dh[t]
//   dA_a  = sum_t dh[t] x[t]^T             dB_a = sum_t dy[t] h[t]^T          (W and b are frozen)
//
// The rows are taken in the order of their adapter (sort_ids.hip), so that a tile of rows meets few adapters and an adapter's
// gradient is a sum over consecutive rows.  Four kernels serve both directions:
//   pack    operands whose rows cannot be read 16 bytes at a time, and the transposed factors that the gradients multiply by, as
//           rows of whole 16-byte pieces
//   shrink  h and dh: skinny products over the long dimension, summed in fp32, in sorted order
//   project y and dx: the shared product by tiles, and behind its last K step one more short step per adapter that the tile
//           meets, with h (dh) as an operand: the adapter's share goes through the same accumulators and is rounded once, with
//           the product.  bf16 MFMA takes h as two bf16 parts (adapters.h).
//   outer   dA and dB: sums over an adapter's rows
//
// Measured at 4096 x 2048 -> 4096 bf16, four adapters of rank 32: sort 7, shrink 14 (forward, 17 MB of x, 1.2 TB/s) and 24 us (backward, 34 MB
// of dy, 1.4 TB/s; bound by the latencies of 256 blocks, one a CU), project 74 and 72, pack 9 (34 MB, 3.7 TB/s), outer 21 (50 MB, 2.4
// TB/s; each gathered row's 128-byte pieces once per block of columns).  At 8192 x 4096 -> 4096, rank 16: sort 8.6, shrink 25 (67 MB, 2.7 TB/s),
// project 244.
#include "adapters.h"
#include "sort_ids.h"
#include <algorithm>

namespace sx {

constexpr int kMaxRank = 128;

// ------------------------------------------------------------------ pack
// dst[b][i][j] (row length ld, rows * ld elements per b) = src[b * s_b + i * s_i + j * s_j] for j < cols, 0 up to ld; one of s_i, s_j is 1
struct PackJob {
  const void* src; int64_t s_b, s_i, s_j;
  void* dst; int ld, rows, cols, batch;
  int ti, tj; int64_t first;                  // 64 x 64 tiles along i and j; the job's first tile
};
constexpr int kMaxJobs = 5;
struct PackArgs { PackJob job[kMaxJobs]; int n; int64_t tiles; };

template <typename T>
__global__ __launch_bounds__(256) void adapter_pack_kernel(PackArgs a) {
  typedef __attribute__((ext_vector_type(4))) T T4;
  __shared__ __align__(16) T tile[64][64 + 2];
  const int lx = threadIdx.x & 15, ly = threadIdx.x >> 4;
  for (int64_t at = blockIdx.x; at < a.tiles; at += gridDim.x) {
    PackJob j = a.job[0];
    for (int k = 1; k < a.n; ++k)
      if (at >= a.job[k].first) j = a.job[k];
    int64_t t = at - j.first;
    const int j0 = (int)(t % j.tj) * 64;
    t /= j.tj;
    const int i0 = (int)(t % j.ti) * 64;
    const int64_t b = t / j.ti;
    const T* src = (const T*)j.src + b * j.s_b;
    T* dst = (T*)j.dst + b * j.rows * j.ld;
    if (j.s_j != 1 || j.s_i == 1) {           // transposed: i runs along memory
      const bool vec = j.s_j % 4 == 0 && j.s_b % 4 == 0 && (uintptr_t)j.src % (4 * sizeof(T)) == 0;
      __syncthreads();                        // the tile before has been read
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int jj = j0 + ly + 16 * k, i = i0 + lx * 4;
        T4 v = {};
        if (jj < j.cols) {
          if (vec && i + 3 < j.rows) v = *reinterpret_cast<const T4*>(src + jj * j.s_j + i);
          else
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (i + e < j.rows) v[e] = src[jj * j.s_j + i + e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) tile[ly + 16 * k][lx * 4 + e] = v[e];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i0 + ly + 16 * k, jj = j0 + lx * 4;
        T4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = tile[lx * 4 + e][ly + 16 * k];
        if (i < j.rows && jj < j.ld) *reinterpret_cast<T4*>(dst + (int64_t)i * j.ld + jj) = v;      // ld is a multiple of 4
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i0 + ly + 16 * k, jj = j0 + lx * 4;
        if (i >= j.rows || jj >= j.ld) continue;
        T4 v = {};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (jj + e < j.cols) v[e] = src[i * j.s_i + jj + e];
        *reinterpret_cast<T4*>(dst + (int64_t)i * j.ld + jj) = v;
      }
    }
  }
}

struct Packer {
  PackArgs a = {};
  void add(const void* src, int64_t s_b, int64_t s_i, int64_t s_j, void* dst, int ld, int rows, int cols, int batch) {
    PackJob& j = a.job[a.n++];
    j.src = src; j.s_b = s_b; j.s_i = s_i; j.s_j = s_j; j.dst = dst; j.ld = ld; j.rows = rows; j.cols = cols; j.batch = batch;
    j.ti = cdiv(rows, 64); j.tj = cdiv(ld, 64); j.first = a.tiles;
    a.tiles += (int64_t)j.ti * j.tj * batch;
  }
  template <typename T> int launch(hipStream_t st) {
    if (!a.n) return SX_OK;
    hipLaunchKernelGGL(adapter_pack_kernel<T>, dim3((unsigned)std::min<int64_t>(a.tiles, 1 << 16)), dim3(256), 0, st, a);
    SX_LAUNCH_CHECK("adapter_pack");
    return SX_OK;
  }
};

// ------------------------------------------------------------------ shrink
struct ShrinkArgs {
  const void* x; int64_t ldx;                 // rows of C elements
  const void* p; int64_t p_g; int p_ld;       // P(g, j, c) = p[g * p_g + j * p_ld + c]
  const float* scales;
  const int* perm; const int* key;
  int64_t T; int C, r, G, rp;
  void* h;                                    // see ProjectArgs
  bf16* ht; int64_t ldt;                      // bf16: [2][rp][ldt], hi and lo parts with the rows along memory; or null
};

// MT * 16 sorted rows and RT * 16 ranks per block; its NW waves split the columns
template <typename T, int MT, int RT, int NW>
__global__ __launch_bounds__(64 * NW) void adapter_shrink_kernel(ShrinkArgs a) {
  constexpr int EPL = Elem<T>::EPL, CK = Elem<T>::CK, RJ = RT * 16, U = MT == 1 && RT <= 2 ? 8 : 4, R = RT == 1 ? 4 : 3;      // U: chunks in flight per wave
  typedef typename Elem<T>::Vec Vec;
  __shared__ float red[NW][MT * 16][RJ + 1];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, gq = lane >> 4;
  const int64_t m0 = blockIdx.x * (int64_t)(MT * 16);
  const int j0 = blockIdx.y * RJ;
  const int rows = (int)std::min<int64_t>(MT * 16, a.T - m0);
  const T* xr[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xr[i] = (const T*)a.x + (int64_t)a.perm[m0 + std::min(i * 16 + n, rows - 1)] * a.ldx + gq * EPL;
  f32x4 tot[MT][RT] = {};
  const int own = a.key[m0 + std::min(lane, rows - 1)];      // the adapters of the block's rows, over the lanes
  for (int at = 0; at < rows;) {
    const int g = __builtin_amdgcn_readlane(own, at);
    const int end = at + __popcll(__ballot(lane < rows && own == g));
    if (g < a.G) {
      const T* pr[RT];                        // ranks past the last one read it again: their products are not stored
#pragma unroll
      for (int t = 0; t < RT; ++t) pr[t] = (const T*)a.p + g * a.p_g + (int64_t)std::min(j0 + t * 16 + n, a.r - 1) * a.p_ld + gq * EPL;
      f32x4 acc[MT][RT] = {};
      int c0 = wid * CK;
      for (; c0 + (U - 1) * NW * CK + CK <= a.C; c0 += U * NW * CK) {
        Vec xv[U][MT], pv[U][RT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int i = 0; i < MT; ++i) xv[u][i] = *reinterpret_cast<const Vec*>(xr[i] + c0 + u * NW * CK);
#pragma unroll
          for (int t = 0; t < RT; ++t) pv[u][t] = *reinterpret_cast<const Vec*>(pr[t] + c0 + u * NW * CK);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int t = 0; t < RT; ++t) acc[i][t] = Mma<T>::run(xv[u][i], pv[u][t], acc[i][t]);
      }
      for (; c0 < a.C; c0 += R * NW * CK) {   // the rest, R chunks in flight
        Vec xv[R][MT], pv[R][RT];
#pragma unroll
        for (int u = 0; u < R; ++u) {
          const int c = c0 + u * NW * CK;
          if (c >= a.C) continue;
#pragma unroll
          for (int i = 0; i < MT; ++i) xv[u][i] = load_piece<T>(xr[i] - gq * EPL, c + gq * EPL, a.C);
#pragma unroll
          for (int t = 0; t < RT; ++t) pv[u][t] = load_piece<T>(pr[t] - gq * EPL, c + gq * EPL, a.C);
        }
#pragma unroll
        for (int u = 0; u < R; ++u) {
          if (c0 + u * NW * CK >= a.C) continue;
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int t = 0; t < RT; ++t) acc[i][t] = Mma<T>::run(xv[u][i], pv[u][t], acc[i][t]);
        }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (i * 16 + 4 * gq + q >= at && i * 16 + 4 * gq + q < end)
#pragma unroll
            for (int t = 0; t < RT; ++t) tot[i][t][q] = acc[i][t][q];
    }
    at = end;
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q) red[wid][i * 16 + 4 * gq + q][t * 16 + n] = tot[i][t][q];
  __syncthreads();
  auto value = [&](int m, int j) {
    const int g = a.key[m0 + m];
    if (g >= a.G || j0 + j >= a.r) return 0.f;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += red[w][m][j];
    return a.scales ? a.scales[g] * v : v;
  };
  for (int i = tid; i < MT * 16 * RJ; i += 64 * NW) {
    const int m = i / RJ, j = i % RJ;
    if (m >= rows || j0 + j >= a.rp) continue;
    const float v = value(m, j);
    if constexpr (sizeof(T) == 2) {
      bf16* h = (bf16*)a.h + (m0 + m) * (2 * a.rp) + (j0 + j) / 16 * 32 + (j & 15);
      h[0] = (bf16)v;
      h[16] = h_lo(v);
    } else {
      ((float*)a.h)[(m0 + m) * a.rp + j0 + j] = v;
    }
  }
  if constexpr (sizeof(T) == 2) {
    if (!a.ht) return;
    for (int i = tid; i < MT * 16 * RJ; i += 64 * NW) {
      const int m = i % (MT * 16), j = i / (MT * 16);
      if (m >= rows || j0 + j >= a.rp) continue;
      const float v = value(m, j);
      bf16* h = a.ht + (int64_t)(j0 + j) * a.ldt + m0 + m;
      h[0] = (bf16)v;
      h[a.rp * a.ldt] = h_lo(v);
    }
  }
}

// Where rows seldom share an adapter: a block per sorted row, a wave per four ranks at a time, its lanes over the columns
template <typename T>
__global__ __launch_bounds__(256) void adapter_shrink_row_kernel(ShrinkArgs a) {
  constexpr int EPL = Elem<T>::EPL, J = 4;
  typedef typename Elem<T>::Vec Vec;
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t m = blockIdx.x;
  const int g = a.key[m];
  const T* x = (const T*)a.x + (int64_t)a.perm[m] * a.ldx;
  const float scale = g < a.G && a.scales ? a.scales[g] : 1.f;
  for (int j0 = wid * J; j0 < a.rp; j0 += 4 * J) {
    float acc[J] = {};
    if (g < a.G && j0 < a.r)
#pragma unroll 2
      for (int c = lane * EPL; c < a.C; c += 64 * EPL) {
        const Vec xv = *reinterpret_cast<const Vec*>(x + c);
        Vec pv[J];
#pragma unroll
        for (int j = 0; j < J; ++j) pv[j] = *reinterpret_cast<const Vec*>((const T*)a.p + g * a.p_g + (int64_t)std::min(j0 + j, a.r - 1) * a.p_ld + c);
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int e = 0; e < EPL; ++e) acc[j] = fmaf(to_f32(xv[e]), to_f32(pv[j][e]), acc[j]);
      }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const float sum = wave_sum(acc[j]), v = g < a.G && j0 + j < a.r ? scale * sum : 0.f;
      if (lane) continue;
      if constexpr (sizeof(T) == 2) {
        bf16* h = (bf16*)a.h + m * (2 * a.rp) + (j0 + j) / 16 * 32 + ((j0 + j) & 15);
        h[0] = (bf16)v;
        h[16] = h_lo(v);
        if (a.ht) {
          bf16* t = a.ht + (int64_t)(j0 + j) * a.ldt + m;
          t[0] = (bf16)v;
          t[a.rp * a.ldt] = h_lo(v);
        }
      } else {
        ((float*)a.h)[m * a.rp + j0 + j] = v;
      }
    }
  }
}

// ------------------------------------------------------------------ project (operands of 2 GiB and more; adapter_tiles.hip has the others)
// A block's tile is BM sorted rows x BN columns: four waves of (BM / 2) x (BN / 2), K steps of 128 bytes through LDS
template <typename T, int BM, int BN>
__global__ __launch_bounds__(256) void adapter_project_kernel(ProjectArgs a) {
  constexpr int EPL = Elem<T>::EPL, CK = Elem<T>::CK, BK = 2 * CK, LD = BK + EPL;
  typedef typename Elem<T>::Vec Vec;
  constexpr int MI = BM / 32, NI = BN / 32;
  __shared__ __align__(16) T As[BM][LD];
  __shared__ __align__(16) T Bs[BN][LD];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, n = lane & 15, gq = lane >> 4;
  const int64_t m0 = blockIdx.x * (int64_t)BM;
  const int n0 = blockIdx.y * BN;
  const int wm = (wid >> 1) * (BM / 2), wn = (wid & 1) * (BN / 2);
  const T* x = (const T*)a.x;
  const T* w = (const T*)a.w;
  f32x4 acc[MI][NI] = {};
  constexpr int PA = BM * 8 / 256, PB = BN * 8 / 256;
  const T *xrow[PA], *wrow[PB];
#pragma unroll
  for (int i = 0; i < PA; ++i) xrow[i] = x + (int64_t)a.perm[std::min<int64_t>(m0 + (i * 256 + tid) / 8, a.T - 1)] * a.ldx;
#pragma unroll
  for (int i = 0; i < PB; ++i) wrow[i] = w + (int64_t)std::min(n0 + (i * 256 + tid) / 8, a.N - 1) * a.ldw;
  for (int k0 = 0; k0 < a.K; k0 += BK) {
    Vec ra[PA], rb[PB];
#pragma unroll
    for (int i = 0; i < PA; ++i) ra[i] = load_piece<T>(xrow[i], k0 + (tid & 7) * EPL, a.K);
#pragma unroll
    for (int i = 0; i < PB; ++i) rb[i] = load_piece<T>(wrow[i], k0 + (tid & 7) * EPL, a.K);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PA; ++i) *reinterpret_cast<Vec*>(&As[(i * 256 + tid) / 8][(tid & 7) * EPL]) = ra[i];
#pragma unroll
    for (int i = 0; i < PB; ++i) *reinterpret_cast<Vec*>(&Bs[(i * 256 + tid) / 8][(tid & 7) * EPL]) = rb[i];
    __syncthreads();
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      Vec av[MI], bv[NI];
#pragma unroll
      for (int i = 0; i < MI; ++i) av[i] = *reinterpret_cast<const Vec*>(&As[wm + i * 16 + n][half * CK + gq * EPL]);
#pragma unroll
      for (int i = 0; i < NI; ++i) bv[i] = *reinterpret_cast<const Vec*>(&Bs[wn + i * 16 + n][half * CK + gq * EPL]);
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = Mma<T>::run(av[i], bv[j], acc[i][j]);
    }
  }
  // the adapters that this tile's rows meet, 16 ranks at a time
  const int rows = (int)std::min<int64_t>(BM, a.T - m0);
  for (int at = 0; at < rows;) {
    const int g = a.key[m0 + at];
    if (g >= a.G) break;                                  // the rows without an adapter come last
    const int end = (int)std::min<int64_t>(rows, a.end[g] - m0);
    const T* qg = (const T*)a.q + g * a.q_g;
    for (int j0 = 0; j0 < a.r; j0 += 16) {
      Vec bv[NI];
#pragma unroll
      for (int j = 0; j < NI; ++j) bv[j] = load_piece<T>(qg + (int64_t)std::min(n0 + wn + j * 16 + n, a.N - 1) * a.q_ld, j0 + h_rank<T>(gq), a.q_ld);
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int f = wm + i * 16;
        if (f >= end || f + 16 <= at) continue;
        const Vec av = load_h<T>(a, m0 + std::min(f + n, rows - 1), j0, gq);
#pragma unroll
        for (int j = 0; j < NI; ++j) {
          const f32x4 z = {0.f, 0.f, 0.f, 0.f};
          const f32x4 d = Mma<T>::run(av, bv[j], z);
#pragma unroll
          for (int q = 0; q < 4; ++q)                     // only this adapter's rows: 0 * NaN must not reach the others
            if (f + 4 * gq + q >= at && f + 4 * gq + q < end) acc[i][j][q] += d[q];
        }
      }
    }
    at = end;
  }
#pragma unroll
  for (int j = 0; j < NI; ++j) {
    const int cn = n0 + wn + j * 16 + n;
    if (cn >= a.N) continue;
    const float b = a.bias ? to_f32(((const T*)a.bias)[cn]) : 0.f;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t m = m0 + wm + i * 16 + 4 * gq + q;
        if (m < a.T) ((T*)a.y)[(int64_t)a.perm[m] * a.ldy + cn] = from_f32<T>(acc[i][j][q] + b);
      }
  }
}

// ------------------------------------------------------------------ outer
// out(g, j, c) = sum over the rows of adapter g of h[t][j] x[t][c]
struct OuterJob {
  const void* x; int64_t ldx; int C;          // rows of C elements, by perm
  const void* h;                              // fp32: [T][rp]; bf16: the transposed parts [2][rp][ldt]; sorted rows
  void* out; int64_t o_g, o_j, o_c;           // one of o_j and o_c is 1
  int vec;                                    // 4 columns can be read at once
  int cols, first;                            // 64-column blocks; the job's first block
};
struct OuterArgs {
  OuterJob job[2]; int n;
  const int* perm; const int* start; const int* end;
  int r, rp, G; int64_t ldt;
};

__device__ __forceinline__ void outer_block(const OuterArgs& a, OuterJob& j, int& c0, int& g) {
  j = a.n > 1 && (int)blockIdx.x >= a.job[1].first ? a.job[1] : a.job[0];
  const int t = blockIdx.x - j.first;
  c0 = t % j.cols * 64;
  g = t / j.cols;
}

// fp32: 64 columns and 16 ranks per block, its waves split the rows, four at a time; the places of the next four are on their way meanwhile
template <int NW>
__global__ __launch_bounds__(64 * NW) void adapter_outer_f32_kernel(OuterArgs a) {
  __shared__ float red[NW][16][64];
  constexpr int U = 4;
  OuterJob j;
  int c0, g;
  outer_block(a, j, c0, g);
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = c0 + lane, j0 = blockIdx.y * 16;
  const int t0 = a.start[g], t1 = a.end[g];
  float acc[16] = {};
  int p[U];
  auto load_perm = [&](int t) {
    if (t >= t1) return;
#pragma unroll
    for (int u = 0; u < U; ++u) p[u] = a.perm[std::min(t + u, t1 - 1)];
  };
  load_perm(t0 + wid * U);
  for (int t = t0 + wid * U; t < t1; t += NW * U) {
    float xv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) xv[u] = c < j.C ? ((const float*)j.x)[(int64_t)p[u] * j.ldx + c] : 0.f;
    load_perm(t + NW * U);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t + u >= t1) continue;
      const float* h = (const float*)j.h + (int64_t)(t + u) * a.rp + j0;
#pragma unroll
      for (int k = 0; k < 16; ++k) acc[k] = fmaf(h[k], xv[u], acc[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < 16; ++k) red[wid][k][lane] = acc[k];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * 64; i += 64 * NW) {
    const int k = j.o_j == 1 ? i & 15 : i >> 6, cc = j.o_j == 1 ? i >> 4 : i & 63;
    if (j0 + k < a.r && c0 + cc < j.C) {
      float v = red[0][k][cc];
#pragma unroll
      for (int w = 1; w < NW; ++w) v += red[w][k][cc];
      ((float*)j.out)[g * j.o_g + (j0 + k) * j.o_j + (int64_t)(c0 + cc) * j.o_c] = v;
    }
  }
}

// bf16: 64 columns and RT * 16 ranks per block; a wave takes every NW-th block of 32 rows, the next block's x on its way under the MFMAs
// of one.  h comes with the rows along memory (16 bytes = 8 rows of one rank); x comes as it lies, 4 columns of 8 rows per lane, and is
// turned in registers: fragment f holds columns 4 n + f.  32-row blocks are aligned, so that h's and perm's 16-byte reads are: rows of
// other adapters in the first and last one are cleared on both sides.
template <int RT, int NW>
__global__ __launch_bounds__(64 * NW) void adapter_outer_kernel(OuterArgs a) {
  typedef __attribute__((ext_vector_type(4))) int i32x4;
  __shared__ float red[NW / 2][RT * 16][64 + 1];
  OuterJob j;
  int c0, g;
  outer_block(a, j, c0, g);
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, n = lane & 15, gq = lane >> 4;
  const int j0 = blockIdx.y * (RT * 16), c = c0 + 4 * n;
  const int t0 = a.start[g], t1 = a.end[g];
  const bf16* x = (const bf16*)j.x;
  const bf16* ht = (const bf16*)j.h;
  f32x4 acc[RT][4] = {};
  auto load_perm = [&](int tb, int (&p)[8]) {               // (perm's storage reaches to a multiple of 64 rows)
    if (tb >= t1) return;
    const i32x4 lo = *reinterpret_cast<const i32x4*>(a.perm + tb + gq * 8), hi = *reinterpret_cast<const i32x4*>(a.perm + tb + gq * 8 + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) { p[e] = lo[e]; p[4 + e] = hi[e]; }
  };
  auto load_x = [&](int tb, const int (&p)[8], uint32_t (&v)[8][2]) {      // columns (0, 1) and (2, 3) of 8 rows
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e][0] = v[e][1] = 0;
      const int t = tb + gq * 8 + e;
      if (t >= t0 && t < t1) {
        const bf16* q = x + (int64_t)p[e] * j.ldx + c;
        if (j.vec) {
          if (c < j.C) {
            const uint64_t w = *reinterpret_cast<const uint64_t*>(q);
            v[e][0] = (uint32_t)w;
            v[e][1] = (uint32_t)(w >> 32);
          }
        } else {
          const uint16_t* q16 = reinterpret_cast<const uint16_t*>(q);
          if (c < j.C) v[e][0] = q16[0];
          if (c + 1 < j.C) v[e][0] |= (uint32_t)q16[1] << 16;
          if (c + 2 < j.C) v[e][1] = q16[2];
          if (c + 3 < j.C) v[e][1] |= (uint32_t)q16[3] << 16;
        }
      }
    }
  };
  auto multiply = [&](int tb, const uint32_t (&v)[8][2], const bf16x8 (&hv)[RT][2]) {
    bf16x8 xf[4];
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      union { uint32_t u[4]; bf16x8 b; } w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t p = v[2 * e][f >> 1], q = v[2 * e + 1][f >> 1];
        w.u[e] = f & 1 ? (p >> 16) | (q & 0xffff0000u) : (p & 0xffffu) | (q << 16);
      }
      xf[f] = w.b;
    }
    const bool whole = tb >= t0 && tb + 32 <= t1;
#pragma unroll
    for (int k = 0; k < RT; ++k)
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        bf16x8 h = hv[k][part];
        if (!whole)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (tb + gq * 8 + e < t0 || tb + gq * 8 + e >= t1) h[e] = (bf16)0.f;
#pragma unroll
        for (int f = 0; f < 4; ++f) acc[k][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(h, xf[f], acc[k][f], 0, 0, 0);
      }
  };
  auto load_h = [&](int tb, bf16x8 (&hv)[RT][2]) {
#pragma unroll
    for (int k = 0; k < RT; ++k) {
      const bf16* h = ht + (int64_t)std::min(j0 + k * 16 + n, a.rp - 1) * a.ldt + tb + gq * 8;
#pragma unroll
      for (int part = 0; part < 2; ++part) hv[k][part] = *reinterpret_cast<const bf16x8*>(h + part * (int64_t)a.rp * a.ldt);
    }
  };
  constexpr int STEP = NW * 32;
  int tb = (t0 & ~31) + wid * 32;
  if (t0 < t1) {
    int p[8];
    uint32_t va[8][2], vb[8][2];
    bf16x8 hv[RT][2];
    load_perm(tb, p);
    load_x(tb, p, va);
    load_perm(tb + STEP, p);
    for (; tb < t1; tb += 2 * STEP) {
      load_h(tb, hv);
      load_x(tb + STEP, p, vb);
      load_perm(tb + 2 * STEP, p);
      multiply(tb, va, hv);
      if (tb + STEP < t1) load_h(tb + STEP, hv);
      load_x(tb + 2 * STEP, p, va);
      load_perm(tb + 3 * STEP, p);
      if (tb + STEP < t1) multiply(tb + STEP, vb, hv);
    }
  }
  auto slot = [&](int k, int q, int f) -> float& { return red[wid & (NW / 2 - 1)][k * 16 + 4 * gq + q][4 * n + f]; };
  if (wid >= NW / 2)
#pragma unroll
    for (int k = 0; k < RT; ++k)
#pragma unroll
      for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int q = 0; q < 4; ++q) slot(k, q, f) = acc[k][f][q];
  __syncthreads();
  if (wid < NW / 2)
#pragma unroll
    for (int k = 0; k < RT; ++k)
#pragma unroll
      for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int q = 0; q < 4; ++q) slot(k, q, f) += acc[k][f][q];
  __syncthreads();
  for (int i = tid; i < RT * 16 * 64; i += 64 * NW) {
    const int k = j.o_j == 1 ? i % (RT * 16) : i >> 6, cc = j.o_j == 1 ? i / (RT * 16) : i & 63;
    if (j0 + k < a.r && c0 + cc < j.C) {
      float v = red[0][k][cc];
#pragma unroll
      for (int w = 1; w < NW / 2; ++w) v += red[w][k][cc];
      ((bf16*)j.out)[g * j.o_g + (j0 + k) * j.o_j + (int64_t)(c0 + cc) * j.o_c] = (bf16)v;
    }
  }
}

// ------------------------------------------------------------------ host
// kept: what a backward call needs of the forward one
struct AdapterKept { size_t perm, key, start, end, h, ht, total; int rp; int64_t ldt; };
static AdapterKept adapter_kept(int dtype, int64_t T, int r, int G) {
  AdapterKept w;
  size_t o = 0;
  w.rp = round_up(r, 16);
  w.ldt = (int64_t)align_up((size_t)T, 64);
  w.perm = o; o = align_up(o + (size_t)w.ldt * 4, 256);      // read 16 bytes at a time by adapter_outer_kernel
  w.key = o; o = align_up(o + (size_t)T * 4, 256);
  w.start = o; o = align_up(o + (size_t)(G + 1) * 4, 256);
  w.end = o; o = align_up(o + (size_t)(G + 1) * 4, 256);
  w.h = o; o = align_up(o + (size_t)T * w.rp * 4, 256);
  w.ht = o; o = align_up(o + (dtype == SX_BF16 ? (size_t)w.rp * w.ldt * 4 : 0), 256);
  w.total = o;
  return w;
}
// sizes that rows of K elements lie in whole 16-byte pieces for; other ones are packed into rows that do
static int padded(int dtype, int n) { return round_up(n, dtype == SX_BF16 ? 8 : 4); }

struct AdapterWs { size_t x, w, A, B, dy, wt, at, bt, dh, dht, part, total; };
static AdapterWs adapter_ws(int dtype, int64_t T, int K, int N, int r, int G, bool backward) {
  const size_t e = dtype_size(dtype);
  const int Kp = padded(dtype, K), Np = padded(dtype, N), r8 = padded(dtype, r);
  AdapterWs w = {};
  size_t o = 0;
  auto take = [&](size_t& at, size_t elems, size_t size) { at = o; o = align_up(o + elems * size, 256); };
  if (!backward) {
    if (Kp != K) { take(w.x, (size_t)T * Kp, e); take(w.w, (size_t)N * Kp, e); take(w.A, (size_t)G * r * Kp, e); }
    if (r8 != r) take(w.B, (size_t)G * N * r8, e);
  } else {
    const AdapterKept k = adapter_kept(dtype, T, r, G);
    if (Np != N) take(w.dy, (size_t)T * Np, e);
    take(w.wt, (size_t)K * Np, e);
    take(w.at, (size_t)G * K * r8, e);
    take(w.bt, (size_t)G * r * Np, e);
    take(w.dh, (size_t)T * k.rp, 4);
    if (dtype == SX_BF16) take(w.dht, (size_t)k.rp * k.ldt, 4);
  }
  int stages;
  const int out = backward ? K : N, parts = project_parts(dtype, T, backward ? Np : Kp, out, G, stages);
  take(w.part, (size_t)parts * T * round_up(out, 16), 4);
  w.total = std::max<size_t>(o, 256);
  return w;
}

template <typename T>
static int shrink_launch(const ShrinkArgs& a, hipStream_t st) {
  // 32 rows share an adapter's factor once there are rows enough for two such blocks a CU; below, 16 rows and, up to one block a CU, sixteen
  // waves and at most 32 ranks a block.  (32 rows from 8192 rows on: 32 us against 27 at 8192 x 4096, rank 16.  2481 x 3180, rank 40, fp32: 31 us
  // with sixteen waves, 41 with eight and 64 ranks.)  Rows that seldom share an adapter come one by one: 107 rows of 68 adapters 4 us against
  // 12, 256 of 16 adapters 3.5 against 4.6, 399 of 36 adapters, 2112 columns, rank 24: 10 against 22.
  const bool wide = a.T <= 16 * 256 && a.C >= 16 * Elem<T>::CK;
  const int rt = a.rp <= 16 ? 1 : a.rp <= 32 || wide ? 2 : 4;
  if (a.T <= 16 * (int64_t)a.G) {
    hipLaunchKernelGGL(adapter_shrink_row_kernel<T>, dim3((unsigned)a.T), dim3(256), 0, st, a);
  } else if (a.T >= 32 * 512) {
    const dim3 grid((unsigned)cdiv64(a.T, 32), cdiv(a.rp, rt * 16));
    if (rt == 1) hipLaunchKernelGGL((adapter_shrink_kernel<T, 2, 1, 4>), grid, dim3(256), 0, st, a);
    else if (rt == 2) hipLaunchKernelGGL((adapter_shrink_kernel<T, 2, 2, 4>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((adapter_shrink_kernel<T, 2, 4, 4>), grid, dim3(256), 0, st, a);
  } else {
    const dim3 grid((unsigned)cdiv64(a.T, 16), cdiv(a.rp, rt * 16));
    if (rt == 1 && wide) hipLaunchKernelGGL((adapter_shrink_kernel<T, 1, 1, 16>), grid, dim3(1024), 0, st, a);
    else if (rt == 1) hipLaunchKernelGGL((adapter_shrink_kernel<T, 1, 1, 8>), grid, dim3(512), 0, st, a);
    else if (rt == 2 && wide) hipLaunchKernelGGL((adapter_shrink_kernel<T, 1, 2, 16>), grid, dim3(1024), 0, st, a);
    else if (rt == 2) hipLaunchKernelGGL((adapter_shrink_kernel<T, 1, 2, 8>), grid, dim3(512), 0, st, a);
    else hipLaunchKernelGGL((adapter_shrink_kernel<T, 1, 4, 8>), grid, dim3(512), 0, st, a);
  }
  SX_LAUNCH_CHECK("adapter_shrink");
  return SX_OK;
}

template <typename T>
static int project_launch(ProjectArgs a, char* part, hipStream_t st) {
  a.parts = project_parts(Elem<T>::kDtype, a.T, a.K, a.N, a.G, a.part_stages);
  a.part = (float*)part;
  a.part_ld = round_up(a.N, 16);
  if (project_tiles_ok(a, Elem<T>::kDtype)) return project_tiles_launch(a, Elem<T>::kDtype, st);
  hipLaunchKernelGGL((adapter_project_kernel<T, 128, 128>), dim3((unsigned)cdiv64(a.T, 128), cdiv(a.N, 128)), dim3(256), 0, st, a);
  SX_LAUNCH_CHECK("adapter_project");
  return SX_OK;
}

template <typename T>
static int outer_launch(OuterArgs a, int64_t T_rows, hipStream_t st) {
  int blocks = 0;
  for (int i = 0; i < a.n; ++i) {
    a.job[i].cols = cdiv(a.job[i].C, 64);
    a.job[i].first = blocks;
    a.job[i].vec = a.job[i].C % 4 == 0 && a.job[i].ldx % 4 == 0 && (uintptr_t)a.job[i].x % 8 == 0;
    blocks += a.job[i].cols * a.G;
  }
  if (!blocks) return SX_OK;
  // Many rows per adapter: many waves for them, in fp32 only where there are very many or few blocks (the sum of sixteen waves through LDS costs
  // more than it gives).  fp32 with sixteen waves and with four: 6198 rows of 95 adapters 34 us and 23, 5684 of 25 35 and 30, 84 of one 6
  // and 8, 2481 of two 42 and 155 (then a row at a time).  bf16 with eight and with two: 1027 rows of 7 adapters 9 us and 18, 399 of 36 23 and 13.
  const bool tall = T_rows >= 64 * (int64_t)a.G && (sizeof(T) == 2 || T_rows >= 400 * (int64_t)a.G || (int64_t)blocks * cdiv(a.r, 16) <= 512);
  if (sizeof(T) == 4) {
    if (tall) hipLaunchKernelGGL(adapter_outer_f32_kernel<16>, dim3(blocks, cdiv(a.r, 16)), dim3(1024), 0, st, a);
    else hipLaunchKernelGGL(adapter_outer_f32_kernel<4>, dim3(blocks, cdiv(a.r, 16)), dim3(256), 0, st, a);
  } else if (a.rp <= 16) {
    if (tall) hipLaunchKernelGGL((adapter_outer_kernel<1, 8>), dim3(blocks, 1), dim3(512), 0, st, a);
    else hipLaunchKernelGGL((adapter_outer_kernel<1, 2>), dim3(blocks, 1), dim3(128), 0, st, a);
  } else {
    if (tall) hipLaunchKernelGGL((adapter_outer_kernel<2, 8>), dim3(blocks, cdiv(a.rp, 32)), dim3(512), 0, st, a);
    else hipLaunchKernelGGL((adapter_outer_kernel<2, 2>), dim3(blocks, cdiv(a.rp, 32)), dim3(128), 0, st, a);
  }
  SX_LAUNCH_CHECK("adapter_outer");
  return SX_OK;
}

struct AdapterCall {
  int dtype; int64_t T; int K, N, r, G;
  const void* x; int64_t ldx;
  const void* w; int64_t ldw;
  const void *bias, *A, *B;
  const float* scales;
};

template <typename T>
static int adapter_forward(const AdapterCall& c, const void* ids, int ids64, void* y, int64_t ldy, char* kept, char* ws, hipStream_t st) {
  const AdapterKept k = adapter_kept(c.dtype, c.T, c.r, c.G);
  const AdapterWs o = adapter_ws(c.dtype, c.T, c.K, c.N, c.r, c.G, false);
  const int Kp = padded(c.dtype, c.K), r8 = padded(c.dtype, c.r);
  int *perm = (int*)(kept + k.perm), *key = (int*)(kept + k.key), *start = (int*)(kept + k.start), *end = (int*)(kept + k.end);
  const void *x = c.x, *w = c.w, *A = c.A, *B = c.B;
  int64_t ldx = c.ldx, ldw = c.ldw;
  Packer pk;
  if (Kp != c.K) {
    pk.add(c.x, 0, c.ldx, 1, ws + o.x, Kp, (int)c.T, c.K, 1);
    pk.add(c.w, 0, c.ldw, 1, ws + o.w, Kp, c.N, c.K, 1);
    pk.add(c.A, 0, c.K, 1, ws + o.A, Kp, c.G * c.r, c.K, 1);
    x = ws + o.x; w = ws + o.w; A = ws + o.A; ldx = ldw = Kp;
  }
  if (r8 != c.r) {
    pk.add(c.B, (int64_t)c.N * c.r, c.r, 1, ws + o.B, r8, c.N, c.r, c.G);
    B = ws + o.B;
  }
  SX_TRY(pk.launch<T>(st));
  SX_TRY(launch_sort_ids(ids, ids64, c.T, c.G, perm, key, start, end, st));
  ShrinkArgs s = {};
  s.x = x; s.ldx = ldx; s.p = A; s.p_g = (int64_t)c.r * Kp; s.p_ld = Kp; s.scales = c.scales; s.perm = perm; s.key = key;
  s.T = c.T; s.C = Kp; s.r = c.r; s.G = c.G; s.rp = k.rp; s.h = kept + k.h; s.ht = sizeof(T) == 2 ? (bf16*)(kept + k.ht) : nullptr; s.ldt = k.ldt;
  SX_TRY(shrink_launch<T>(s, st));
  ProjectArgs p = {};
  p.x = x; p.ldx = ldx; p.w = w; p.ldw = ldw; p.bias = c.bias; p.q = B; p.q_g = (int64_t)c.N * r8; p.q_ld = r8; p.h = kept + k.h; p.rp = k.rp;
  p.perm = perm; p.key = key; p.end = end; p.T = c.T; p.K = Kp; p.N = c.N; p.r = c.r; p.G = c.G; p.y = y; p.ldy = ldy;
  return project_launch<T>(p, ws + o.part, st);
}

template <typename T>
static int adapter_backward(const AdapterCall& c, const void* dy, int64_t lddy, const char* kept, void* dx, void* dA, void* dB, char* ws, hipStream_t st) {
  const AdapterKept k = adapter_kept(c.dtype, c.T, c.r, c.G);
  const AdapterWs o = adapter_ws(c.dtype, c.T, c.K, c.N, c.r, c.G, true);
  const int Np = padded(c.dtype, c.N), r8 = padded(c.dtype, c.r);
  const int *perm = (const int*)(kept + k.perm), *key = (const int*)(kept + k.key), *start = (const int*)(kept + k.start), *end = (const int*)(kept + k.end);
  Packer pk;
  const void* d = dy;
  int64_t ldd = lddy;
  if (Np != c.N) {
    pk.add(dy, 0, lddy, 1, ws + o.dy, Np, (int)c.T, c.N, 1);
    d = ws + o.dy;
    ldd = Np;
  }
  if (dx || dA) pk.add(c.B, (int64_t)c.N * c.r, 1, c.r, ws + o.bt, Np, c.r, c.N, c.G);
  if (dx) {
    pk.add(c.w, 0, 1, c.ldw, ws + o.wt, Np, c.K, c.N, 1);
    pk.add(c.A, (int64_t)c.r * c.K, 1, c.K, ws + o.at, r8, c.K, c.r, c.G);
  }
  SX_TRY(pk.launch<T>(st));
  bf16* dht = sizeof(T) == 2 ? (bf16*)(ws + o.dht) : nullptr;
  if (dx || dA) {
    ShrinkArgs s = {};
    s.x = d; s.ldx = ldd; s.p = ws + o.bt; s.p_g = (int64_t)c.r * Np; s.p_ld = Np; s.scales = c.scales; s.perm = perm; s.key = key;
    s.T = c.T; s.C = Np; s.r = c.r; s.G = c.G; s.rp = k.rp; s.h = ws + o.dh; s.ht = dht; s.ldt = k.ldt;
    SX_TRY(shrink_launch<T>(s, st));
  }
  if (dx) {
    ProjectArgs p = {};
    p.x = d; p.ldx = ldd; p.w = ws + o.wt; p.ldw = Np; p.q = ws + o.at; p.q_g = (int64_t)c.K * r8; p.q_ld = r8; p.h = ws + o.dh; p.rp = k.rp;
    p.perm = perm; p.key = key; p.end = end; p.T = c.T; p.K = Np; p.N = c.K; p.r = c.r; p.G = c.G; p.y = dx; p.ldy = c.K;
    SX_TRY(project_launch<T>(p, ws + o.part, st));
  }
  OuterArgs q = {};
  q.perm = perm; q.start = start; q.end = end; q.r = c.r; q.rp = k.rp; q.G = c.G; q.ldt = k.ldt;
  if (dA) {
    OuterJob& j = q.job[q.n++];
    j.x = c.x; j.ldx = c.ldx; j.C = c.K; j.h = sizeof(T) == 2 ? (const void*)dht : ws + o.dh; j.out = dA; j.o_g = (int64_t)c.r * c.K; j.o_j = c.K; j.o_c = 1;
  }
  if (dB) {
    OuterJob& j = q.job[q.n++];
    j.x = d; j.ldx = ldd; j.C = c.N; j.h = kept + (sizeof(T) == 2 ? k.ht : k.h); j.out = dB; j.o_g = (int64_t)c.N * c.r; j.o_j = 1; j.o_c = c.r;
  }
  return outer_launch<T>(q, c.T, st);
}

static int adapter_check(const char* who, int dtype, int64_t T, int K, int N, int r, int G) {
  SX_REQUIRE(dtype == SX_F32 || dtype == SX_BF16, "%s: dtype %d is neither fp32 nor bf16", who, dtype);
  SX_REQUIRE(T >= 0 && T <= (1 << 24) && K > 0 && N > 0 && K <= (1 << 20) && N <= (1 << 20), "%s: bad sizes T=%lld K=%d N=%d", who, (long long)T, K, N);
  SX_REQUIRE((int64_t)G * std::max(K, N) <= (1 << 29), "%s: %d adapters of K=%d, N=%d: more than 2^29 rows", who, G, K, N);
  SX_REQUIRE(r >= 1 && r <= kMaxRank && G >= 1 && G <= 65535, "%s: rank %d must be 1..%d and the adapters %d 1..65535", who, r, kMaxRank, G);
  return SX_OK;
}

// rows of C elements that are read 16 bytes at a time; where C is no multiple of that, they are packed first and may lie anywhere
static bool rows_ok(int dtype, const void* p, int64_t ld, int C) {
  const int e = dtype == SX_BF16 ? 8 : 4;
  return ld >= C && (C % e != 0 || (ld % e == 0 && (uintptr_t)p % 16 == 0));
}

}  // namespace sx

using namespace sx;

extern "C" int64_t sx_adapter_kept_bytes(int dtype, int64_t T, int r, int G) {
  SX_TRY(adapter_check("sx_adapter_kept_bytes", dtype, T, 1, 1, r, G));
  return (int64_t)adapter_kept(dtype, T, r, G).total;
}

// what a forward call without `kept` needs besides: nothing more for a few rows, else the kept part itself, behind the rest
static size_t adapter_alone(int dtype, int64_t T, int K, int N, int r, int G) {
  return T <= kTokens ? tokens_workspace(dtype, (int)T, K, N, r) : adapter_ws(dtype, T, K, N, r, G, false).total + adapter_kept(dtype, T, r, G).total;
}

extern "C" int64_t sx_adapter_workspace_bytes(int dtype, int64_t T, int K, int N, int r, int G, int mode) {
  SX_TRY(adapter_check("sx_adapter_workspace_bytes", dtype, T, K, N, r, G));
  SX_REQUIRE(mode >= 0 && mode <= 2, "sx_adapter_workspace_bytes: mode %d", mode);
  return (int64_t)std::max<size_t>(256, mode == SX_ADAPTER_ALONE ? adapter_alone(dtype, T, K, N, r, G) : adapter_ws(dtype, T, K, N, r, G, mode == SX_ADAPTER_BACKWARD).total);
}

extern "C" int sx_adapter_forward(int dtype, int64_t T, int K, int N, int r, int G, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                                  const void* A, const void* B, const float* scales, const void* ids, int ids64, void* y, int64_t ldy, void* kept,
                                  int64_t kept_bytes, void* workspace, int64_t workspace_bytes, void* stream) {
  SX_TRY(adapter_check("sx_adapter_forward", dtype, T, K, N, r, G));
  if (T == 0) return SX_OK;
  SX_REQUIRE(x && w && A && B && ids && y && workspace, "sx_adapter_forward: null pointer");
  SX_REQUIRE(rows_ok(dtype, x, ldx, K) && rows_ok(dtype, w, ldw, K) && rows_ok(dtype, A, K, K) && rows_ok(dtype, B, r, r) && ldy >= N,
             "sx_adapter_forward: rows of x, w, A (K=%d) or B (r=%d) shorter than that or not 16-byte aligned (ldx=%lld ldw=%lld ldy=%lld)", K, r,
             (long long)ldx, (long long)ldw, (long long)ldy);
  const size_t need = adapter_ws(dtype, T, K, N, r, G, false).total;
  SX_REQUIRE(!kept || (kept_bytes >= (int64_t)adapter_kept(dtype, T, r, G).total && (uintptr_t)kept % 16 == 0), "sx_adapter_forward: kept too small or not 16-byte aligned");
  SX_REQUIRE(workspace_bytes >= (int64_t)(kept ? need : adapter_alone(dtype, T, K, N, r, G)) && (uintptr_t)workspace % 16 == 0,
             "sx_adapter_forward: workspace too small or not 16-byte aligned");
  if (!kept) {
    if (T <= kTokens)
      return tokens_forward(dtype, (int)T, K, N, r, G, x, ldx, w, ldw, bias, A, B, scales, ids, ids64, y, ldy, (char*)workspace, (hipStream_t)stream);
    kept = (char*)workspace + need;
  }
  const AdapterCall c = {dtype, T, K, N, r, G, x, ldx, w, ldw, bias, A, B, scales};
  return dtype == SX_BF16 ? adapter_forward<bf16>(c, ids, ids64, y, ldy, (char*)kept, (char*)workspace, (hipStream_t)stream)
                          : adapter_forward<float>(c, ids, ids64, y, ldy, (char*)kept, (char*)workspace, (hipStream_t)stream);
}

extern "C" int sx_adapter_backward(int dtype, int64_t T, int K, int N, int r, int G, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* A,
                                   const void* B, const float* scales, const void* dy, int64_t lddy, const void* kept, int64_t kept_bytes, void* dx, void* dA,
                                   void* dB, void* workspace, int64_t workspace_bytes, void* stream) {
  SX_TRY(adapter_check("sx_adapter_backward", dtype, T, K, N, r, G));
  SX_REQUIRE(T > 0, "sx_adapter_backward: T must be positive");
  SX_REQUIRE(x && w && A && B && dy && kept && workspace, "sx_adapter_backward: null pointer");
  SX_REQUIRE(ldx >= K && ldw >= K && rows_ok(dtype, dy, lddy, N), "sx_adapter_backward: rows of x, w (K=%d) or dy (N=%d) shorter than that or dy not 16-byte aligned (ldx=%lld ldw=%lld lddy=%lld)",
             K, N, (long long)ldx, (long long)ldw, (long long)lddy);
  SX_REQUIRE(kept_bytes >= (int64_t)adapter_kept(dtype, T, r, G).total && (uintptr_t)kept % 16 == 0 &&
                 workspace_bytes >= (int64_t)adapter_ws(dtype, T, K, N, r, G, true).total && (uintptr_t)workspace % 16 == 0,
             "sx_adapter_backward: kept or workspace too small or not 16-byte aligned");
  const AdapterCall c = {dtype, T, K, N, r, G, x, ldx, w, ldw, nullptr, A, B, scales};
  return dtype == SX_BF16 ? adapter_backward<bf16>(c, dy, lddy, (const char*)kept, dx, dA, dB, (char*)workspace, (hipStream_t)stream)
                          : adapter_backward<float>(c, dy, lddy, (const char*)kept, dx, dA, dB, (char*)workspace, (hipStream_t)stream);
}
