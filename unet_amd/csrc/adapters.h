// Shared by the kernels of the adapter projection (adapters.hip, adapter_tiles.hip, adapter_tokens.hip).
#pragma once
#include "sx_common.h"
#include <type_traits>

namespace sx {

// f(0), f(1) ... f(N - 1) with constant arguments: an array indexed by them stays in registers (#pragma unroll leaves loops around
// cross-lane operations rolled, and the array in memory)
template <int N, int I = 0, typename F>
__device__ __forceinline__ void unrolled(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>());
    unrolled<N, I + 1>(static_cast<F&&>(f));
  }
}

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

// 16 bytes of a row from column c on, zeros from column C on (C a multiple of the piece, rows 16-byte aligned)
template <typename T>
__device__ __forceinline__ typename Elem<T>::Vec load_piece(const T* __restrict__ row, int c, int C) {
  typename Elem<T>::Vec v = {};
  if (c < C) v = *reinterpret_cast<const typename Elem<T>::Vec*>(row + c);
  return v;
}

// h in fp32 as the MFMA's operand.  fp32: as it is.  bf16: 16 ranks are 16 hi parts, then 16 lo parts (h - hi): one K block of 32, whose
// other side holds the 16 factors twice.  h loses 2^-17 of itself where one bf16 would cost 2^-9: a third part would take another MFMA per 16
// ranks.  An infinity among the factors meets both parts, lo may be 0 or of the other sign: what should be infinite may come out as NaN.
__device__ __forceinline__ bf16 h_lo(float v) {
  const float hi = (float)(bf16)v;
  return fabsf(hi) == INFINITY ? (bf16)0.f : (bf16)(v - hi);
}

struct ProjectArgs {
  const void* x; int64_t ldx;                 // T rows of K elements, by perm
  const void* w; int64_t ldw;                 // N rows of K elements
  const void* bias;                           // [N] or null
  const void* q; int64_t q_g; int q_ld;       // Q(g, n, j) = q[g * q_g + n * q_ld + j], the adapter's second factor; zeros for j in [r, q_ld)
  const void* h; int rp;                      // sorted rows: fp32 [T][rp], or bf16 [T][rp / 16][16 hi, 16 lo]
  const int* perm; const int* key; const int* end;
  int64_t T; int K, N, r, G;
  void* y; int64_t ldy;
  int parts, part_stages;                     // K in parts of that many stages, summed by a second launch; 0: in one
  float* part; int part_ld;                   // [parts][T][part_ld], sorted rows
};

// a lane's 16 bytes of h (row m, ranks from j0 on), and the first of the ranks whose factors they meet
template <typename T>
__device__ __forceinline__ int h_rank(int gq) { return sizeof(T) == 2 ? (gq & 1) * 8 : gq * 4; }
template <typename T>
__device__ __forceinline__ typename Elem<T>::Vec load_h(const ProjectArgs& a, int64_t m, int j0, int gq) {
  const T* h = (const T*)a.h + (sizeof(T) == 2 ? m * (2 * a.rp) + j0 * 2 + gq * 8 : m * a.rp + j0 + gq * 4);
  return *reinterpret_cast<const typename Elem<T>::Vec*>(h);
}

// the shared product by tiles (adapter_tiles.hip); false: not for this kernel
bool project_tiles_ok(const ProjectArgs& a, int dtype);
int project_parts(int dtype, int64_t T, int K, int N, int G, int& stages);
int project_tiles_launch(const ProjectArgs& a, int dtype, hipStream_t st);

// a few rows, forward alone (adapter_tokens.hip)
constexpr int kTokens = 64;
size_t tokens_workspace(int dtype, int T, int K, int N, int r);
int tokens_forward(int dtype, int T, int K, int N, int r, int G, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* A,
                   const void* B, const float* scales, const void* ids, int ids64, void* y, int64_t ldy, char* ws, hipStream_t st);

}  // namespace sx
