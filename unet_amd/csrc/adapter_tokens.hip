// The adapter projection of a few rows (single tokens of up to 64 requests) in two launches.
//
// Here the product is bound by reading W, and by the latencies of whatever runs one after the other.  Neither A x nor W x depends on the
// other, so one launch computes both (adapter_tokens_kernel): a block takes 64 columns of W (or 64 ranks of the adapter of the first row
// that names it, with all rows that do) and a part of the reduction.  Every element of W is read once, by one wave, straight into the
// MFMA's registers, a round of 1 KB per row at a time with all its loads in flight; the rows of x that the four waves share go through
// LDS (read by every wave for itself, x was the larger traffic: 28 us against 16 at 64 x 4096 x 4096).  The second launch
// (adapter_tokens_join_kernel) adds the parts, the bias and B (A x), in fp32 throughout, and rounds once.  Rows need no order by
// adapter: 64 ids fit a ballot.
//
// Measured in bf16: one token at 2048 x 2048, rank 8: 4.7 + 5.1 us, mostly the launches' own time (8.5 MB); 64 tokens of 64 adapters of rank 16
// at 4096 x 4096: 16.6 us (42 MB of W and A, 2.5 TB/s: one wave's round of 16 KB at a time, four waves a SIMD) + 4.8 (8.4 MB of B and the parts).
#include "adapters.h"
#include <algorithm>

namespace sx {

// 16 bytes of a row; VEC: as one load (rows aligned, C a multiple of the piece)
template <typename T, bool VEC>
__device__ __forceinline__ typename Elem<T>::Vec load_any(const T* __restrict__ row, int c, int C) {
  if constexpr (VEC) {
    return load_piece<T>(row, c, C);
  } else {
    typename Elem<T>::Vec v = {};
#pragma unroll
    for (int e = 0; e < Elem<T>::EPL; ++e)
      if (c + e < C) v[e] = row[c + e];
    return v;
  }
}

struct TokensArgs {
  const void* x; int64_t ldx;
  const void* w; int64_t ldw;
  const void* bias;
  const void *A, *B;
  const float* scales;
  const void* ids; int ids64;
  int T, K, N, r, G, rp, np;
  int splits, chunks;         // parts of the reduction; chunks (64 bytes of a row) per part
  float* part;                // [splits][T][np]
  float* h;                   // [splits][T][rp], unscaled; rows without an adapter are not written
  void* y; int64_t ldy;
};

__device__ __forceinline__ int64_t token_id(const TokensArgs& a, int t) {
  return a.ids64 ? ((const int64_t*)a.ids)[t] : (int64_t)((const int32_t*)a.ids)[t];
}

template <typename T, bool VEC, int F>
__global__ __launch_bounds__(256) void adapter_tokens_kernel(TokensArgs a) {
  constexpr int EPL = Elem<T>::EPL, CK = Elem<T>::CK, L = 16;
  typedef typename Elem<T>::Vec Vec;
  __shared__ Vec xs[F * 16][L * 4];                       // a round of x: piece p of row m at p ^ (m & 7), see adapter_tiles.hip
  __shared__ int member[64];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, n = lane & 15, gq = lane >> 4;
  const int nj = (a.rp + 63) / 64, shrink = a.T * nj * a.splits, all = (a.K + CK - 1) / CK;
  const bool is_h = (int)blockIdx.x < shrink;
  const int u0 = is_h ? blockIdx.x : blockIdx.x - shrink, s = u0 % a.splits, u1 = u0 / a.splits;
  int cnt = a.T, c0;                                      // rows of x; this wave's 16 rows of the left factor begin at c0
  const T* left;
  if (is_h) {
    const int i = u1 / nj;
    const int64_t g = token_id(a, i);
    const int64_t mine = lane < a.T ? token_id(a, lane) : -1;
    const unsigned long long same = __ballot(lane < a.T && mine == g);
    if (g < 0 || g >= a.G || __ffsll(same) - 1 != i) return;      // no adapter, or an earlier row's block computes it
    if (wid == 0 && (same >> lane & 1)) member[__popcll(same & ((1ull << lane) - 1))] = lane;
    cnt = __popcll(same);
    c0 = u1 % nj * 64 + wid * 16;
    left = (const T*)a.A + (g * a.r + std::min(c0 + n, a.r - 1)) * a.K;
  } else {
    if (tid < 64) member[tid] = std::min(tid, a.T - 1);
    c0 = u1 * 64 + wid * 16;
    left = (const T*)a.w + std::min(c0 + n, a.N - 1) * a.ldw;
  }
  const bool works = c0 < (is_h ? a.r : a.N);
  __syncthreads();
  const int k0 = s * a.chunks, k1 = std::min(all, k0 + a.chunks);
  f32x4 acc[F] = {};
  for (int c = k0; c < k1; c += L) {
    Vec lv[L], xv[F * 4];
#pragma unroll
    for (int u = 0; u < L; ++u) lv[u] = load_any<T, VEC>(left, works && c + u < k1 ? (c + u) * CK + gq * EPL : a.K, a.K);      // past the end: zeros
#pragma unroll
    for (int i = 0; i < F * 4; ++i) {
      const int m = i * 4 + wid, k = (c + (lane >> 2)) * CK + (lane & 3) * EPL;
      xv[i] = load_any<T, VEC>((const T*)a.x + member[std::min(m, cnt - 1)] * a.ldx, m < cnt && c + (lane >> 2) < k1 ? k : a.K, a.K);
    }
    if (c > k0) __syncthreads();
#pragma unroll
    for (int i = 0; i < F * 4; ++i) xs[i * 4 + wid][lane ^ ((i * 4 + wid) & 7)] = xv[i];
    __syncthreads();
    if (works)
#pragma unroll
      for (int u = 0; u < L; ++u)                           // behind k1 both sides are zeros
#pragma unroll
        for (int f = 0; f < F; ++f) acc[f] = Mma<T>::run(lv[u], xs[f * 16 + n][(u * 4 + gq) ^ (n & 7)], acc[f]);
  }
  if (!works) return;
  // lane: columns (ranks) c0 + 4 gq .. + 3 of row n of each fragment
  float* out = is_h ? a.h + (int64_t)s * a.T * a.rp : a.part + (int64_t)s * a.T * a.np;
  const int ld = is_h ? a.rp : a.np;
#pragma unroll
  for (int f = 0; f < F; ++f)
    if (f * 16 + n < cnt) *reinterpret_cast<f32x4*>(out + (int64_t)member[f * 16 + n] * ld + c0 + 4 * gq) = acc[f];
}

// one row and 256 columns per block
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void adapter_tokens_join_kernel(TokensArgs a) {
  constexpr int EPL = Elem<T>::EPL, PRE = 4;
  typedef typename Elem<T>::Vec Vec;
  __shared__ float h[128];
  const int tid = threadIdx.x, t = blockIdx.y, c = blockIdx.x * 256 + tid, cc = std::min(c, a.N - 1);
  const int64_t g = token_id(a, t);
  const bool has = g >= 0 && g < a.G;
  const T* b = has ? (const T*)a.B + (g * a.N + cc) * a.r : nullptr;
  Vec pre[PRE];                                             // the first ranks' factors are on their way before h is there
  if (has)
#pragma unroll
    for (int p = 0; p < PRE; ++p)
      if (p * EPL < a.r) pre[p] = load_any<T, VEC>(b, p * EPL, a.r);
  float v = a.bias ? to_f32(((const T*)a.bias)[cc]) : 0.f;
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) v += a.part[((int64_t)s * a.T + t) * a.np + cc];
  if (has && tid < a.r) {
    float d = 0.f;
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) d += a.h[((int64_t)s * a.T + t) * a.rp + tid];
    h[tid] = a.scales ? a.scales[g] * d : d;
  }
  __syncthreads();
  if (has) {
    float d = 0.f;
#pragma unroll
    for (int p = 0; p < PRE; ++p)
#pragma unroll
      for (int e = 0; e < EPL; ++e)
        if (p * EPL + e < a.r) d = fmaf(h[p * EPL + e], to_f32(pre[p][e]), d);
    for (int j = PRE * EPL; j < a.r; j += EPL) {
      const Vec q = load_any<T, VEC>(b, j, a.r);
#pragma unroll
      for (int e = 0; e < EPL; ++e)
        if (j + e < a.r) d = fmaf(h[j + e], to_f32(q[e]), d);
    }
    v += d;
  }
  if (c < a.N) ((T*)a.y)[(int64_t)t * a.ldy + c] = from_f32<T>(v);
}

// Parts of the reduction: about 512 blocks (two a CU; more write more parts), of at least four chunks
static void tokens_plan(int dtype, int K, int N, int& splits, int& chunks) {
  const int all = cdiv(K, dtype == SX_BF16 ? 32 : 16);
  splits = cdiv(512, cdiv(N, 64));
  chunks = std::max(4, cdiv(all, splits));
  splits = cdiv(all, chunks);
}

size_t tokens_workspace(int dtype, int T, int K, int N, int r) {
  int splits, chunks;
  tokens_plan(dtype, K, N, splits, chunks);
  return align_up((size_t)splits * T * round_up(N, 16) * 4, 256) + align_up((size_t)splits * T * round_up(r, 16) * 4, 256);
}

template <typename T, bool VEC>
static int tokens_launch(const TokensArgs& a, bool bvec, hipStream_t st) {
  const dim3 grid((a.T * cdiv(a.rp, 64) + cdiv(a.N, 64)) * a.splits);
  if (a.T <= 16) hipLaunchKernelGGL((adapter_tokens_kernel<T, VEC, 1>), grid, dim3(256), 0, st, a);
  else if (a.T <= 32) hipLaunchKernelGGL((adapter_tokens_kernel<T, VEC, 2>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((adapter_tokens_kernel<T, VEC, 4>), grid, dim3(256), 0, st, a);
  SX_LAUNCH_CHECK("adapter_tokens");
  if (bvec) hipLaunchKernelGGL((adapter_tokens_join_kernel<T, true>), dim3(cdiv(a.N, 256), a.T), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((adapter_tokens_join_kernel<T, false>), dim3(cdiv(a.N, 256), a.T), dim3(256), 0, st, a);
  SX_LAUNCH_CHECK("adapter_tokens_join");
  return SX_OK;
}

template <typename T>
static int tokens_typed(const TokensArgs& a, hipStream_t st) {
  constexpr int E = Elem<T>::EPL;
  const bool bvec = a.r % E == 0;                           // rows of such sizes are 16-byte aligned (checked at the entry)
  return a.K % E == 0 ? tokens_launch<T, true>(a, bvec, st) : tokens_launch<T, false>(a, bvec, st);
}

int tokens_forward(int dtype, int T, int K, int N, int r, int G, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* A,
                   const void* B, const float* scales, const void* ids, int ids64, void* y, int64_t ldy, char* ws, hipStream_t st) {
  TokensArgs a = {};
  a.x = x; a.ldx = ldx; a.w = w; a.ldw = ldw; a.bias = bias; a.A = A; a.B = B; a.scales = scales; a.ids = ids; a.ids64 = ids64;
  a.T = T; a.K = K; a.N = N; a.r = r; a.G = G; a.rp = round_up(r, 16); a.np = round_up(N, 16); a.y = y; a.ldy = ldy;
  tokens_plan(dtype, K, N, a.splits, a.chunks);
  a.part = (float*)ws;
  a.h = (float*)(ws + align_up((size_t)a.splits * T * a.np * 4, 256));
  return dtype == SX_BF16 ? tokens_typed<bf16>(a, st) : tokens_typed<float>(a, st);
}

}  // namespace sx
