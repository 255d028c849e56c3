// Low-rank adapters of many requests beside one shared projection.  Row t of a batch belongs to adapter a = ids[t] (or to none):
//
//   h[t]  = s_a A_a x[t]                   (r numbers)          y[t]  = W x[t] + b + B_a h[t]
//   dh[t] = s_a B_a^T dy[t]                                     dx[t] = W^T dy[t] + A_a^T dh[t]
//   dA_a  = sum_t dh[t] x[t]^T             dB_a = sum_t dy[t] h[t]^T          (W and b are frozen)
//
// The rows are taken in the order of their adapter (sort_ids.hip), so that a tile of rows meets few adapters and an adapter's
// gradient is a sum over consecutive rows.  Three kernels serve both directions:
//   shrink  h and dh: skinny products over the long dimension, kept in fp32, in sorted order
//   project y and dx: the shared product by tiles, and behind its last K step one more short step per adapter that the tile
//           meets, with h (dh) as the left operand: the adapter's share goes through the same accumulators and is rounded
//           once, with the product.  bf16 MFMA takes h as two bf16 parts, hi + lo, side by side in one K block of 32: an error of
//           2^-17 of h where rounding h to bf16 alone would cost 2^-9.
//   outer   dA and dB: sums over an adapter's rows
#include "sort_ids.h"
#include <algorithm>

namespace sx {

constexpr int kMaxRank = 128;

template <typename T> struct Mma;
template <> struct Mma<bf16> {
  static __device__ __forceinline__ f32x4 run(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<float> {      // lane (n, g) feeds k = 4 g + i in MFMA i, on both sides
  static __device__ __forceinline__ f32x4 run(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};

// 16 bytes of a row from column c on, zeros from column C on; `vec`: 16-byte loads are possible and C is a multiple of them
template <typename T, bool VEC>
__device__ __forceinline__ typename Elem<T>::Vec load_piece(const T* __restrict__ row, int c, int C) {
  typename Elem<T>::Vec v = {};
  if constexpr (VEC) {
    if (c < C) v = *reinterpret_cast<const typename Elem<T>::Vec*>(row + c);
  } else {
#pragma unroll
    for (int i = 0; i < Elem<T>::EPL; ++i)
      if (c + i < C) v[i] = row[c + i];
  }
  return v;
}
// the same from elements `stride` apart
template <typename T>
__device__ __forceinline__ typename Elem<T>::Vec gather_piece(const T* __restrict__ p, int64_t stride, int c, int C) {
  typename Elem<T>::Vec v = {};
#pragma unroll
  for (int i = 0; i < Elem<T>::EPL; ++i)
    if (c + i < C) v[i] = p[(c + i) * stride];
  return v;
}

// ------------------------------------------------------------------ shrink
struct ShrinkArgs {
  const void* x; int64_t ldx;                 // rows of C elements
  const void* p; int64_t p_g, p_j, p_c;       // P(g, j, c) = p[g * p_g + j * p_j + c * p_c]
  const float* scales;
  const int* perm; const int* key; const int* start;
  int64_t T; int C, r, G, rp;
  float* h;                                   // [T][rp]
};

// 16 sorted rows and 64 ranks per block; the four waves split the columns
template <typename T, bool VEC, bool PC>
__global__ __launch_bounds__(256) void adapter_shrink_kernel(ShrinkArgs a) {
  constexpr int EPL = Elem<T>::EPL, CK = Elem<T>::CK;
  typedef typename Elem<T>::Vec Vec;
  __shared__ float red[4][16][64 + 1];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, n = lane & 15, gq = lane >> 4;
  const int64_t m0 = blockIdx.x * 16ll;
  const int j0 = blockIdx.y * 64;
  const int rows = (int)std::min<int64_t>(16, a.T - m0);
  const T* xr = (const T*)a.x + (int64_t)a.perm[m0 + std::min(n, rows - 1)] * a.ldx;
  f32x4 tot[4] = {};
  for (int at = 0; at < rows;) {
    const int g = a.key[m0 + at];
    const int end = (int)std::min<int64_t>(rows, a.start[g + 1] - m0);
    if (g < a.G) {
      const T* pg = (const T*)a.p + g * a.p_g;
      f32x4 acc[4] = {};
      for (int c0 = wid * CK; c0 < a.C; c0 += 4 * CK) {
        const int c = c0 + gq * EPL;
        const Vec xv = load_piece<T, VEC>(xr, c, a.C);
#pragma unroll
        for (int rt = 0; rt < 4; ++rt) {
          const int j = j0 + rt * 16 + n;
          if (j0 + rt * 16 >= a.r) continue;
          Vec pv = {};
          if (j < a.r) {
            if constexpr (PC) pv = load_piece<T, VEC>(pg + j * a.p_j, c, a.C);
            else pv = gather_piece<T>(pg + j * a.p_j, a.p_c, c, a.C);
          }
          acc[rt] = Mma<T>::run(xv, pv, acc[rt]);
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (4 * gq + q >= at && 4 * gq + q < end)
#pragma unroll
          for (int rt = 0; rt < 4; ++rt) tot[rt][q] = acc[rt][q];
    }
    at = end;
  }
#pragma unroll
  for (int rt = 0; rt < 4; ++rt)
#pragma unroll
    for (int q = 0; q < 4; ++q) red[wid][4 * gq + q][rt * 16 + n] = tot[rt][q];
  __syncthreads();
  for (int i = tid; i < rows * 64; i += 256) {
    const int m = i >> 6, j = i & 63;
    if (j0 + j >= a.rp) continue;
    const int g = a.key[m0 + m];
    const float s = g < a.G ? (a.scales ? a.scales[g] : 1.f) : 0.f;
    a.h[(m0 + m) * a.rp + j0 + j] = g < a.G ? s * (red[0][m][j] + red[1][m][j] + red[2][m][j] + red[3][m][j]) : 0.f;
  }
}

// ------------------------------------------------------------------ project
struct ProjectArgs {
  const void* x; int64_t ldx;                 // T rows of K elements, by perm
  const void* w; int64_t ldw;                 // WT = false: N rows of K elements; true: K rows of N elements
  const void* bias;                           // [N] or null
  const void* q; int64_t q_g, q_n, q_j;       // Q(g, n, j), the adapter's second factor
  const float* h; int rp;                     // [T][rp], sorted order
  const int* perm; const int* key; const int* start;
  int64_t T; int K, N, r, G;
  void* y; int64_t ldy;
};

// A block's tile is BM sorted rows x BN columns: four waves of (BM / 2) x (BN / 2), K steps of 128 bytes through LDS
template <typename T, bool VEC, bool WT, int BM, int BN>
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
  const T* xrow[PA];
#pragma unroll
  for (int i = 0; i < PA; ++i) {
    const int64_t m = std::min<int64_t>(m0 + (i * 256 + tid) / 8, a.T - 1);
    xrow[i] = x + (int64_t)a.perm[m] * a.ldx;
  }
  auto product = [&](int half) {
    Vec av[MI], bv[NI];
#pragma unroll
    for (int i = 0; i < MI; ++i) av[i] = *reinterpret_cast<const Vec*>(&As[wm + i * 16 + n][half * CK + gq * EPL]);
#pragma unroll
    for (int i = 0; i < NI; ++i) bv[i] = *reinterpret_cast<const Vec*>(&Bs[wn + i * 16 + n][half * CK + gq * EPL]);
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = Mma<T>::run(av[i], bv[j], acc[i][j]);
  };
  for (int k0 = 0; k0 < a.K; k0 += BK) {
    Vec ra[PA], rb[PB];
#pragma unroll
    for (int i = 0; i < PA; ++i) ra[i] = load_piece<T, VEC>(xrow[i], k0 + (tid & 7) * EPL, a.K);
#pragma unroll
    for (int i = 0; i < PB; ++i) {
      const int p = i * 256 + tid;
      if constexpr (WT) {
        const int nn = std::min(n0 + p % BN, a.N - 1);
        rb[i] = gather_piece<T>(w + nn, a.ldw, k0 + p / BN * EPL, a.K);
      } else {
        rb[i] = load_piece<T, VEC>(w + (int64_t)std::min(n0 + p / 8, a.N - 1) * a.ldw, k0 + (p & 7) * EPL, a.K);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PA; ++i) *reinterpret_cast<Vec*>(&As[(i * 256 + tid) / 8][(tid & 7) * EPL]) = ra[i];
#pragma unroll
    for (int i = 0; i < PB; ++i) {
      const int p = i * 256 + tid;
      if constexpr (WT) *reinterpret_cast<Vec*>(&Bs[p % BN][p / BN * EPL]) = rb[i];
      else *reinterpret_cast<Vec*>(&Bs[p / 8][(p & 7) * EPL]) = rb[i];
    }
    __syncthreads();
    product(0);
    product(1);
  }
  // the adapters that this tile's rows meet, 16 ranks at a time: fp32 one K block of 16; bf16 one of 32, 16 hi then 16 lo
  const int rows = (int)std::min<int64_t>(BM, a.T - m0);
  for (int at = 0; at < rows;) {
    const int g = a.key[m0 + at];
    if (g >= a.G) break;                                  // the rows without an adapter come last
    const int end = (int)std::min<int64_t>(rows, a.start[g + 1] - m0);
    for (int j0 = 0; j0 < a.r; j0 += 16) {
      __syncthreads();
      for (int i = tid; i < BM * 16; i += 256) {
        const int m = i >> 4, j = i & 15;
        const float h = (m >= at && m < end) ? a.h[(m0 + m) * a.rp + j0 + j] : 0.f;
        const T hi = from_f32<T>(h);
        As[m][j] = hi;
        if constexpr (CK == 32) As[m][16 + j] = from_f32<T>(fabsf(to_f32(hi)) == INFINITY ? 0.f : h - to_f32(hi));
      }
      for (int i = tid; i < BN * 16; i += 256) {
        const int nn = a.q_n == 1 ? i % BN : i >> 4, j = a.q_n == 1 ? i / BN : i & 15;
        const T v = (n0 + nn < a.N && j0 + j < a.r) ? ((const T*)a.q)[g * a.q_g + (n0 + nn) * a.q_n + (j0 + j) * a.q_j] : from_f32<T>(0.f);
        Bs[nn][j] = v;
        if constexpr (CK == 32) Bs[nn][16 + j] = v;
      }
      __syncthreads();
      // only this adapter's rows take the product: a NaN or an infinity in its factors must not reach the others as 0 * NaN
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int f = wm + i * 16;
        if (f >= end || f + 16 <= at) continue;
        const Vec av = *reinterpret_cast<const Vec*>(&As[f + n][gq * EPL]);
#pragma unroll
        for (int jj = 0; jj < NI; ++jj) {
          const Vec bv = *reinterpret_cast<const Vec*>(&Bs[wn + jj * 16 + n][gq * EPL]);
          const f32x4 z = {0.f, 0.f, 0.f, 0.f};
          const f32x4 d = Mma<T>::run(av, bv, z);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (f + 4 * gq + q >= at && f + 4 * gq + q < end) acc[i][jj][q] += d[q];
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
struct OuterArgs {
  const void* x; int64_t ldx;                 // rows of C elements, by perm
  const float* h; int rp;                     // [T][rp], sorted order
  const int* perm; const int* start;
  int C, r;
  void* out; int64_t o_g, o_j, o_c;           // out(g, j, c)
};

// out(g, j, c) = sum over the rows of adapter g of h[t][j] x[t][c]; 64 columns and 16 ranks per block, its waves split the rows
template <typename T>
__global__ __launch_bounds__(256) void adapter_outer_kernel(OuterArgs a) {
  __shared__ float red[4][16][64];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane, j0 = blockIdx.y * 16, g = blockIdx.z;
  const int t0 = a.start[g], t1 = a.start[g + 1];
  float acc[16] = {};
  for (int t = t0 + wid; t < t1; t += 4) {
    const float xv = c < a.C ? to_f32(((const T*)a.x)[(int64_t)a.perm[t] * a.ldx + c]) : 0.f;
    const float* h = a.h + (int64_t)t * a.rp + j0;
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[j] = fmaf(h[j], xv, acc[j]);
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) red[wid][j][lane] = acc[j];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * 64; i += 256) {
    const int j = a.o_j == 1 ? i & 15 : i >> 6, cc = a.o_j == 1 ? i >> 4 : i & 63;
    if (j0 + j < a.r && (int)blockIdx.x * 64 + cc < a.C)
      ((T*)a.out)[g * a.o_g + (j0 + j) * a.o_j + ((int64_t)blockIdx.x * 64 + cc) * a.o_c] =
          from_f32<T>(red[0][j][cc] + red[1][j][cc] + red[2][j][cc] + red[3][j][cc]);
  }
}

// ------------------------------------------------------------------ host
struct AdapterWs { size_t perm, key, start, h, total; };
static AdapterWs adapter_ws(int64_t T, int r, int G) {
  AdapterWs w;
  size_t o = 0;
  w.perm = o; o = align_up(o + (size_t)T * 4, 256);
  w.key = o; o = align_up(o + (size_t)T * 4, 256);
  w.start = o; o = align_up(o + (size_t)(G + 2) * 4, 256);
  w.h = o; o = align_up(o + (size_t)T * round_up(r, 16) * 4, 256);
  w.total = o;
  return w;
}
static size_t adapter_dh_bytes(int64_t T, int r) { return align_up((size_t)T * round_up(r, 16) * 4, 256); }

template <typename T>
static bool rows_vec(const void* p, int64_t ld, int C) {
  constexpr int E = Elem<T>::EPL;
  return C % E == 0 && ld % E == 0 && (uintptr_t)p % 16 == 0;
}

template <typename T>
static int shrink_launch(const ShrinkArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)cdiv64(a.T, 16), cdiv(a.rp, 64));
  const bool pc = a.p_c == 1;
  const bool vec = rows_vec<T>(a.x, a.ldx, a.C) && (!pc || (rows_vec<T>(a.p, a.p_j, a.C) && a.p_g % Elem<T>::EPL == 0));
  if (vec && pc) hipLaunchKernelGGL((adapter_shrink_kernel<T, true, true>), grid, dim3(256), 0, st, a);
  else if (vec) hipLaunchKernelGGL((adapter_shrink_kernel<T, true, false>), grid, dim3(256), 0, st, a);
  else if (pc) hipLaunchKernelGGL((adapter_shrink_kernel<T, false, true>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((adapter_shrink_kernel<T, false, false>), grid, dim3(256), 0, st, a);
  SX_LAUNCH_CHECK("adapter_shrink");
  return SX_OK;
}

template <typename T, bool WT>
static int project_launch(const ProjectArgs& a, hipStream_t st) {
  const bool vec = rows_vec<T>(a.x, a.ldx, a.K) && (WT || rows_vec<T>(a.w, a.ldw, a.K));
  const bool big = a.T >= 512 && a.N >= 512;
  const int b = big ? 128 : 64;
  const dim3 grid((unsigned)cdiv64(a.T, b), cdiv(a.N, b));
  if (big && vec) hipLaunchKernelGGL((adapter_project_kernel<T, true, WT, 128, 128>), grid, dim3(256), 0, st, a);
  else if (big) hipLaunchKernelGGL((adapter_project_kernel<T, false, WT, 128, 128>), grid, dim3(256), 0, st, a);
  else if (vec) hipLaunchKernelGGL((adapter_project_kernel<T, true, WT, 64, 64>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((adapter_project_kernel<T, false, WT, 64, 64>), grid, dim3(256), 0, st, a);
  SX_LAUNCH_CHECK("adapter_project");
  return SX_OK;
}

template <typename T>
static int outer_launch(const OuterArgs& a, int G, hipStream_t st) {
  hipLaunchKernelGGL(adapter_outer_kernel<T>, dim3(cdiv(a.C, 64), cdiv(a.r, 16), G), dim3(256), 0, st, a);
  SX_LAUNCH_CHECK("adapter_outer");
  return SX_OK;
}

template <typename T>
static int adapter_forward(int64_t Tn, int K, int N, int r, int G, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                           const void* A, const void* B, const float* scales, const void* ids, int ids64, void* y, int64_t ldy, char* ws, hipStream_t st) {
  const AdapterWs o = adapter_ws(Tn, r, G);
  int *perm = (int*)(ws + o.perm), *key = (int*)(ws + o.key), *start = (int*)(ws + o.start);
  float* h = (float*)(ws + o.h);
  SX_TRY(launch_sort_ids(ids, ids64, Tn, G, perm, key, start, st));
  ShrinkArgs s = {};
  s.x = x; s.ldx = ldx; s.p = A; s.p_g = (int64_t)r * K; s.p_j = K; s.p_c = 1; s.scales = scales; s.perm = perm; s.key = key; s.start = start;
  s.T = Tn; s.C = K; s.r = r; s.G = G; s.rp = round_up(r, 16); s.h = h;
  SX_TRY(shrink_launch<T>(s, st));
  ProjectArgs p = {};
  p.x = x; p.ldx = ldx; p.w = w; p.ldw = ldw; p.bias = bias; p.q = B; p.q_g = (int64_t)N * r; p.q_n = r; p.q_j = 1; p.h = h; p.rp = s.rp;
  p.perm = perm; p.key = key; p.start = start; p.T = Tn; p.K = K; p.N = N; p.r = r; p.G = G; p.y = y; p.ldy = ldy;
  return project_launch<T, false>(p, st);
}

template <typename T>
static int adapter_backward(int64_t Tn, int K, int N, int r, int G, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* A, const void* B,
                            const float* scales, const void* dy, int64_t lddy, const char* kept, void* dx, void* dA, void* dB, char* ws, hipStream_t st) {
  const AdapterWs o = adapter_ws(Tn, r, G);
  const int *perm = (const int*)(kept + o.perm), *key = (const int*)(kept + o.key), *start = (const int*)(kept + o.start);
  const float* h = (const float*)(kept + o.h);
  float* dh = (float*)ws;
  const int rp = round_up(r, 16);
  if (dx || dA) {
    ShrinkArgs s = {};
    s.x = dy; s.ldx = lddy; s.p = B; s.p_g = (int64_t)N * r; s.p_j = 1; s.p_c = r; s.scales = scales; s.perm = perm; s.key = key; s.start = start;
    s.T = Tn; s.C = N; s.r = r; s.G = G; s.rp = rp; s.h = dh;
    SX_TRY(shrink_launch<T>(s, st));
  }
  if (dx) {
    ProjectArgs p = {};
    p.x = dy; p.ldx = lddy; p.w = w; p.ldw = ldw; p.q = A; p.q_g = (int64_t)r * K; p.q_n = 1; p.q_j = K; p.h = dh; p.rp = rp;
    p.perm = perm; p.key = key; p.start = start; p.T = Tn; p.K = N; p.N = K; p.r = r; p.G = G; p.y = dx; p.ldy = K;
    SX_TRY((project_launch<T, true>(p, st)));
  }
  OuterArgs q = {};
  q.perm = perm; q.start = start; q.r = r; q.rp = rp;
  if (dA) {
    q.x = x; q.ldx = ldx; q.h = dh; q.C = K; q.out = dA; q.o_g = (int64_t)r * K; q.o_j = K; q.o_c = 1;
    SX_TRY(outer_launch<T>(q, G, st));
  }
  if (dB) {
    q.x = dy; q.ldx = lddy; q.h = h; q.C = N; q.out = dB; q.o_g = (int64_t)N * r; q.o_j = 1; q.o_c = r;
    SX_TRY(outer_launch<T>(q, G, st));
  }
  return SX_OK;
}

static int adapter_check(const char* who, int dtype, int64_t T, int K, int N, int r, int G) {
  SX_REQUIRE(dtype == SX_F32 || dtype == SX_BF16, "%s: dtype %d is neither fp32 nor bf16", who, dtype);
  SX_REQUIRE(T >= 0 && T <= (1 << 24) && K > 0 && N > 0 && K <= (1 << 20) && N <= (1 << 20), "%s: bad sizes T=%lld K=%d N=%d", who, (long long)T, K, N);
  SX_REQUIRE(r >= 1 && r <= kMaxRank && G >= 1 && G <= 65535, "%s: rank %d must be 1..%d and the adapters %d 1..65535", who, r, kMaxRank, G);
  return SX_OK;
}

}  // namespace sx

using namespace sx;

extern "C" int64_t sx_adapter_kept_bytes(int64_t T, int r, int G) {
  SX_TRY(adapter_check("sx_adapter_kept_bytes", SX_F32, T, 1, 1, r, G));
  return (int64_t)adapter_ws(T, r, G).total;
}

extern "C" int64_t sx_adapter_workspace_bytes(int dtype, int64_t T, int K, int N, int r, int G) {
  SX_TRY(adapter_check("sx_adapter_workspace_bytes", dtype, T, K, N, r, G));
  return (int64_t)std::max<size_t>(adapter_dh_bytes(T, r), 256);
}

extern "C" int sx_adapter_forward(int dtype, int64_t T, int K, int N, int r, int G, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                                  const void* A, const void* B, const float* scales, const void* ids, int ids64, void* y, int64_t ldy, void* kept,
                                  int64_t kept_bytes, void* workspace, int64_t workspace_bytes, void* stream) {
  SX_TRY(adapter_check("sx_adapter_forward", dtype, T, K, N, r, G));
  SX_REQUIRE(ldx >= K && ldw >= K && ldy >= N, "sx_adapter_forward: row strides %lld, %lld, %lld for K=%d, N=%d", (long long)ldx, (long long)ldw, (long long)ldy, K, N);
  if (T == 0) return SX_OK;
  SX_REQUIRE(x && w && A && B && ids && y && kept && workspace, "sx_adapter_forward: null pointer");
  SX_REQUIRE(kept_bytes >= (int64_t)adapter_ws(T, r, G).total && (uintptr_t)kept % 16 == 0 && workspace_bytes >= sx_adapter_workspace_bytes(dtype, T, K, N, r, G) &&
                 (uintptr_t)workspace % 16 == 0, "sx_adapter_forward: kept or workspace too small or not 16-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == SX_BF16) return adapter_forward<bf16>(T, K, N, r, G, x, ldx, w, ldw, bias, A, B, scales, ids, ids64, y, ldy, (char*)kept, st);
  return adapter_forward<float>(T, K, N, r, G, x, ldx, w, ldw, bias, A, B, scales, ids, ids64, y, ldy, (char*)kept, st);
}

extern "C" int sx_adapter_backward(int dtype, int64_t T, int K, int N, int r, int G, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* A,
                                   const void* B, const float* scales, const void* dy, int64_t lddy, const void* kept, int64_t kept_bytes, void* dx, void* dA,
                                   void* dB, void* workspace, int64_t workspace_bytes, void* stream) {
  SX_TRY(adapter_check("sx_adapter_backward", dtype, T, K, N, r, G));
  SX_REQUIRE(ldx >= K && ldw >= K && lddy >= N, "sx_adapter_backward: row strides %lld, %lld, %lld for K=%d, N=%d", (long long)ldx, (long long)ldw, (long long)lddy, K, N);
  SX_REQUIRE(T > 0, "sx_adapter_backward: T must be positive");
  SX_REQUIRE(x && w && A && B && dy && kept && workspace, "sx_adapter_backward: null pointer");
  SX_REQUIRE(kept_bytes >= (int64_t)adapter_ws(T, r, G).total && (uintptr_t)kept % 16 == 0 && workspace_bytes >= sx_adapter_workspace_bytes(dtype, T, K, N, r, G) &&
                 (uintptr_t)workspace % 16 == 0, "sx_adapter_backward: kept or workspace too small or not 16-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == SX_BF16) return adapter_backward<bf16>(T, K, N, r, G, x, ldx, w, ldw, A, B, scales, dy, lddy, (const char*)kept, dx, dA, dB, (char*)workspace, st);
  return adapter_backward<float>(T, K, N, r, G, x, ldx, w, ldw, A, B, scales, dy, lddy, (const char*)kept, dx, dA, dB, (char*)workspace, st);
}
