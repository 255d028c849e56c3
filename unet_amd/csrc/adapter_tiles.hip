// The shared product of the adapter projection (adapters.hip) by tiles.
//
// A block of WM x WN waves computes BM sorted rows x BN columns, each wave MI x NJ MFMA fragments of 16 x 16.  A stage is 128 bytes of K (64
// bf16, 32 fp32) of each row of x (gathered through perm by the addresses) and of w, brought by LDS-DMA as whole cache lines (3 % faster than
// stages of half a line).  x and w have rings of NA and NB stages (three or four of each: +- 3 %).  Fragments are read half a stage ahead of
// their MFMAs, so that the buffers of stage s are free in the middle of its MFMAs: there stands the one barrier of a stage, with a wait for
// stage s + 1 and the DMA of the stages NA and NB on.
// The eight 16-byte pieces of a row lie at (piece ^ row & 7): eight lanes that read one piece of consecutive rows then meet eight different
// parts of the banks (no conflicts counted).  The W fragment is the MFMA's left operand: a lane ends up with four consecutive columns of
// one row.
//
// Bound by the matrix cores and the clock that their power leaves: 8192 x 4096 -> 4096 bf16 with eight adapters of rank 16 244 us, 1.13 PFLOP/s,
// where the library's product alone takes 217 to 222; MFMAs busy 52 % of the time at 1.9 GHz, and 15 % faster on zeros.  4096 x 2048 ->
// 4096 with rank 32 75 us, of which the launch is 3, the adapters 10 and the stores 6.  fp32, 2048 x
// 2048 -> 2048: 185 us in all, the library's product alone 143.  Four waves on 128 x 128 of each instead of eight on 256 x 256: 347 us
// against 293 at that time.
#include "adapters.h"
#include <algorithm>
#include <atomic>

namespace sx {

template <int N> __device__ __forceinline__ void tiles_wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

template <typename T, int WM, int WN, int MI, int NJ, int OCC, int NA, int NB, bool SPLIT>
__global__ __launch_bounds__(64 * WM * WN, OCC) void adapter_tiles_kernel(ProjectArgs a, int gm, int gn, unsigned x_bytes, unsigned w_bytes) {
  constexpr int NT = 64 * WM * WN, BM = WM * MI * 16, BN = WN * NJ * 16, RPR = NT / 8;      // RPR: rows per DMA round
  constexpr int SA = BM * 128, SB = BN * 128, QA = SA / (NT * 16), QB = SB / (NT * 16);
  static_assert(SA % (NT * 16) == 0 && SB % (NT * 16) == 0 && RPR % 8 == 0, "whole DMA rounds");
  constexpr int E = sizeof(T), EPL = Elem<T>::EPL, KS = 128 / E;      // KS: K per stage
  typedef typename Elem<T>::Vec Vec;
  static_assert(NB >= 2 && NA >= NB, "the order of the DMA (w first) and the counts of the waits");
  extern __shared__ __align__(16) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, n = lane & 15, gq = lane >> 4;
  // consecutive blocks go to different XCDs: give each XCD a contiguous range of tiles, walked in patches of 8 row tiles
  int id = blockIdx.x;
  {
    const int total = gm * gn, per = total >> 3, rem = total & 7, xcd = id & 7, ix = id >> 3;
    id = xcd * per + std::min(xcd, rem) + ix;
  }
  constexpr int GM = 8;
  const int patch = GM * gn, first = id / patch * GM, width = std::min(gm - first, GM), in = id % patch;
  const int mt = first + in % width, nt = in / width;
  const int64_t m0 = (int64_t)mt * BM;
  const int n0 = nt * BN;
  const int wm = wid / WN, wn = wid % WN;

  unsigned xo[QA], wo[QB];
  const int piece = (tid & 7) ^ ((tid >> 3) & 7);          // rows advance by RPR, a multiple of 8, from round to round: the same piece in all
#pragma unroll
  for (int q = 0; q < QA; ++q) {
    const int64_t m = m0 + q * RPR + (tid >> 3);
    xo[q] = m < a.T ? (unsigned)((int64_t)a.perm[m] * a.ldx * E) + piece * 16 : 0x80000000u;
  }
#pragma unroll
  for (int q = 0; q < QB; ++q) {
    const int c = n0 + q * RPR + (tid >> 3);
    wo[q] = c < a.N ? (unsigned)(c * a.ldw * E) + piece * 16 : 0x80000000u;
  }
  const int64_t w0 = m0 + wm * MI * 16;
  const int rows = (int)std::min<int64_t>(MI * 16, a.T - w0);      // of this wave; <= 0: none, but it takes part in the DMA and the barriers
  const int g_first = __builtin_amdgcn_readfirstlane(a.key[std::min(w0, a.T - 1)]);
  // the stages of this block: all of K, or its part of them
  const int all = (a.K + KS - 1) / KS, sb = SPLIT ? blockIdx.y * a.part_stages : 0, nst = SPLIT ? std::min(all - sb, a.part_stages) : all;
  char* const sx = smem;
  char* const sw = smem + NA * SA;
  // past the end: zeros, which keep the count of loads uniform
  auto issue_x = [&](int s, int slot) {
    const unsigned far = piece * EPL + (sb + s) * KS < a.K ? 0u : 0x80000000u;
    __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)a.x, 0, s < nst ? x_bytes : 0, 0x00020000);
#pragma unroll
    for (int q = 0; q < QA; ++q) {
      const unsigned off = (xo[q] + (sb + s) * 128u) | far;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(sx + slot * SA + wid * 1024 + q * (NT * 16)), 16, off, 0, 0, 0);
    }
  };
  auto issue_w = [&](int s, int slot) {
    const unsigned far = piece * EPL + (sb + s) * KS < a.K ? 0u : 0x80000000u;
    __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)a.w, 0, s < nst ? w_bytes : 0, 0x00020000);
#pragma unroll
    for (int q = 0; q < QB; ++q) {
      const unsigned off = (wo[q] + (sb + s) * 128u) | far;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(sw + slot * SB + wid * 1024 + q * (NT * 16)), 16, off, 0, 0, 0);
    }
  };

  f32x4 acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // fragment row n of the first half of a stage; the other half's pieces differ in bit 2 of the position
  const int row_off = n * 128 + ((gq ^ (n & 7)) << 4);
  const int x_off = wm * MI * 2048 + row_off, w_off = wn * NJ * 2048 + row_off;
  Vec xa[MI], wa[NJ], xb[MI], wb[NJ];
  // multiply the fragments (xc, wc) while (xn, wn_) are read from (px, pw)
  auto half = [&](const char* px, const char* pw, Vec (&xc)[MI], Vec (&wc)[NJ], Vec (&xn)[MI], Vec (&wn_)[NJ]) {
    constexpr int READS = MI + NJ, GROUP = MI * NJ / READS;   // MFMAs between two reads
#pragma unroll
    for (int t = 0; t < READS; ++t) {
      if (t < NJ) wn_[t] = *reinterpret_cast<const Vec*>(pw + t * 2048);
      else xn[t - NJ] = *reinterpret_cast<const Vec*>(px + (t - NJ) * 2048);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int e = 0; e < (t == READS - 1 ? MI * NJ - GROUP * (READS - 1) : GROUP); ++e) {
        const int f = t * GROUP + e, i = f / NJ, j = f % NJ;
        acc[i][j] = Mma<T>::run(wc[j], xc[i], acc[i][j]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
#pragma unroll
  for (int s = -NA; s < 0; ++s) {
    if (s + NB >= 0) issue_w(s + NB, s + NB);
    issue_x(s + NA, s + NA);
  }
  tiles_wait_vm<(NA - 1) * QA + (NB - 1) * QB>();
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int j = 0; j < NJ; ++j) wa[j] = *reinterpret_cast<const Vec*>(sw + w_off + j * 2048);
#pragma unroll
  for (int i = 0; i < MI; ++i) xa[i] = *reinterpret_cast<const Vec*>(sx + x_off + i * 2048);
  int ax = 0, aw = 0;                                         // the slots of stage s
  for (int s = 0; s < nst; ++s) {
    half(sx + ax * SA + (x_off ^ 64), sw + aw * SB + (w_off ^ 64), xa, wa, xb, wb);
    tiles_wait_vm<(NA - 2) * QA + (NB - 2) * QB>();           // this wave's pieces of stage s + 1 have landed
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");        // and its reads of stage s
    __builtin_amdgcn_s_barrier();                             // ... for every wave: the buffers of stage s are free
    issue_w(s + NB, aw);
    issue_x(s + NA, ax);
    ax = ax + 1 == NA ? 0 : ax + 1;
    aw = aw + 1 == NB ? 0 : aw + 1;
    half(sx + ax * SA + x_off, sw + aw * SB + w_off, xb, wb, xa, wa);
  }
  tiles_wait_vm<0>();                                         // no DMA may land in LDS that this block has given back

  // The adapters that this wave's rows meet, 16 ranks at a time, as one more short K step each.  A fragment of 16 rows that one adapter
  // owns takes it in its accumulators; one that several share gets each adapter's product apart and picks its rows, in the epilogue:
  // masking h alone would let a NaN or an infinity of one adapter reach the others' rows as 0 * NaN.
  if (rows <= 0) return;
  if constexpr (SPLIT) {                                      // sums of a part of K, for adapter_join_kernel
    float* part = a.part + ((int64_t)blockIdx.y * a.T + w0) * a.part_ld;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int c = n0 + (wn * NJ + j) * 16 + 4 * gq;
        if (i * 16 + n < rows && c < a.part_ld) *reinterpret_cast<f32x4*>(part + (int64_t)(i * 16 + n) * a.part_ld + c) = acc[i][j];
      }
    return;
  }
  int at_y[MI], own[MI];                                      // all rows' places and adapters at once: one latency
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t m = w0 + std::min(i * 16 + n, rows - 1);
    at_y[i] = a.perm[m];
    own[i] = a.key[m];
  }
  auto q_piece = [&](int g, int j, int j0) {
    const int c = std::min(n0 + (wn * NJ + j) * 16 + n, a.N - 1);
    return load_piece<T>((const T*)a.q + g * a.q_g + (int64_t)c * a.q_ld, j0 + h_rank<T>(gq), a.q_ld);
  };
  auto h_piece = [&](int i, int j0) { return load_h<T>(a, w0 + std::min(i * 16 + n, rows - 1), j0, gq); };
  auto front = [&](int i) { return __builtin_amdgcn_readlane(own[i], 0); };
  auto back = [&](int i) { return __builtin_amdgcn_readlane(own[i], 15); };
  for (int j0 = 0; j0 < a.r && g_first < a.G; j0 += 16) {     // (the rows without an adapter come last)
    Vec hf[MI], qf[NJ];
    int g = g_first;                                          // known since the start: nothing to wait for in the usual case
#pragma unroll
    for (int j = 0; j < NJ; ++j) qf[j] = q_piece(g, j, j0);
#pragma unroll
    for (int i = 0; i < MI; ++i) hf[i] = h_piece(i, j0);
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int gi = front(i);
      if (gi != back(i) || gi >= a.G) continue;
      if (gi != g) {
        g = gi;
#pragma unroll
        for (int j = 0; j < NJ; ++j) qf[j] = q_piece(g, j, j0);
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j] = Mma<T>::run(qf[j], hf[i], acc[i][j]);
    }
  }
  f32x4 bias[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[j][e] = a.bias ? to_f32(((const T*)a.bias)[std::min(n0 + (wn * NJ + j) * 16 + 4 * gq + e, a.N - 1)]) : 0.f;
  const bool wide = a.N % 4 == 0 && a.ldy % 4 == 0 && (uintptr_t)a.y % (4 * E) == 0;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    if (i * 16 >= rows) continue;
    T* y = (T*)a.y + (int64_t)at_y[i] * a.ldy;
    f32x4 v[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) v[j] = acc[i][j];
    if (front(i) != back(i)) {
      constexpr int B = NJ == 1 ? 8 : 2;                      // adapters whose factors are in flight together
      for (int j0 = 0; j0 < a.r; j0 += 16) {
        const Vec hf = h_piece(i, j0);
        int at = 0;                                           // row of the fragment; its adapters in their order
        while (at < 16) {
          int g[B];
          Vec qb[B][NJ];
          unrolled<B>([&](auto b) {
            g[b] = at < 16 ? __builtin_amdgcn_readlane(own[i], at) : a.G;
            at = g[b] < a.G ? at + __popcll(__ballot(own[i] == g[b]) & 0xffffull) : 16;      // (the rows without an adapter come last)
          });
          unrolled<B>([&](auto b) {
            if (g[b] < a.G)
#pragma unroll
              for (int j = 0; j < NJ; ++j) qb[b][j] = q_piece(g[b], j, j0);
          });
          unrolled<B>([&](auto b) {
            if (g[b] < a.G)
#pragma unroll
              for (int j = 0; j < NJ; ++j) {
                const f32x4 d = Mma<T>::run(qb[b][j], hf, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int e = 0; e < 4; ++e) v[j][e] += own[i] == g[b] ? d[e] : 0.f;
              }
          });
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int c = n0 + (wn * NJ + j) * 16 + 4 * gq;
      v[j] += bias[j];
      if (i * 16 + n < rows) {
        if (wide) {
          if (c < a.N) store4(y + c, v[j]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + e < a.N) y[c + e] = from_f32<T>(v[j][e]);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

static void tiles_bytes(const ProjectArgs& a, int64_t size, int64_t& xb, int64_t& wb) {
  xb = ((a.T - 1) * a.ldx + a.K) * size;
  wb = ((int64_t)(a.N - 1) * a.ldw + a.K) * size;
}

// The DMA's offsets are 32-bit with bit 31 for "out of range"; operands of 2 GiB and more take the other kernel.
bool project_tiles_ok(const ProjectArgs& a, int dtype) {
  int64_t xb, wb;
  tiles_bytes(a, (int64_t)dtype_size(dtype), xb, wb);
  return xb < (1ll << 31) - 4096 && wb < (1ll << 31) - 4096;
}

template <typename T, int WM, int WN, int MI, int NJ, int OCC, int NA, int NB>
static int tiles_launch(const ProjectArgs& a, hipStream_t st) {
  constexpr int BM = WM * MI * 16, BN = WN * NJ * 16, LDS = (NA * BM + NB * BN) * 128;
  static std::atomic<unsigned long long> done{0};
  SX_TRY(ensure_max_lds((const void*)adapter_tiles_kernel<T, WM, WN, MI, NJ, OCC, NA, NB, false>, done, "adapter_tiles"));
  int64_t xb, wb;
  tiles_bytes(a, sizeof(T), xb, wb);
  const int gm = (int)cdiv64(a.T, BM), gn = cdiv(a.N, BN);
  hipLaunchKernelGGL((adapter_tiles_kernel<T, WM, WN, MI, NJ, OCC, NA, NB, false>), dim3((unsigned)(gm * gn)), dim3(64 * WM * WN), LDS, st, a, gm, gn, (unsigned)xb, (unsigned)wb);
  SX_LAUNCH_CHECK("adapter_tiles");
  return SX_OK;
}

// y of what the parts of K hold: one column of a row per thread, the parts in their order, then the row's adapter, one rounding
template <typename T>
__global__ __launch_bounds__(256) void adapter_join_kernel(ProjectArgs a) {
  typedef typename Elem<T>::Vec Vec;
  constexpr int EPL = Elem<T>::EPL;
  const int64_t at = blockIdx.x * 256ll + threadIdx.x;
  const int64_t m = at / a.N;
  const int c = (int)(at - m * a.N);
  if (m >= a.T) return;
  const int g = a.key[m];
  float v = a.bias ? to_f32(((const T*)a.bias)[c]) : 0.f;
#pragma unroll 4
  for (int s = 0; s < a.parts; ++s) v += a.part[((int64_t)s * a.T + m) * a.part_ld + c];
  if (g < a.G) {
    const T* q = (const T*)a.q + g * a.q_g + (int64_t)c * a.q_ld;
    float d = 0.f;
#pragma unroll 2
    for (int j = 0; j < a.r; j += EPL) {
      const Vec f = *reinterpret_cast<const Vec*>(q + j);
      Vec h, lo = {};
      if constexpr (sizeof(T) == 2) {
        const T* p = (const T*)a.h + m * (2 * a.rp) + j / 16 * 32 + (j & 15);
        h = *reinterpret_cast<const Vec*>(p);
        lo = *reinterpret_cast<const Vec*>(p + 16);
      } else {
        h = *reinterpret_cast<const Vec*>((const T*)a.h + m * a.rp + j);
      }
#pragma unroll
      for (int e = 0; e < EPL; ++e)
        if (j + e < a.r) d = fmaf(to_f32(h[e]) + to_f32(lo[e]), to_f32(f[e]), d);
    }
    v += d;
  }
  ((T*)a.y)[(int64_t)a.perm[m] * a.ldy + c] = from_f32<T>(v);
}

// Parts of K for a product of few tiles of 64 x 64; 0: none, the tiles kernel finishes by itself.  A stage of such a tile takes 0.5 to 0.7 us
// however deep its rings are (MFMA in fp32, the barriers in bf16), so few tiles with many stages leave most CUs idle: 84 x 2880 -> 128 in fp32
// 11 us in parts against 61, 2481 x 3180 -> 456 101 against 121.  The join costs a launch and its reads, six such stages and one more per
// 1.8 MB: 6198 x 896 -> 256 in fp32 54 us in parts, 44 without.  And where most fragments hold rows of several adapters, the join
// multiplies by them faster: 256 rows of 16 adapters, 256 -> 256, 9 us against 14; 82 rows of 118 adapters 7 against 26.
int project_parts(int dtype, int64_t T, int K, int N, int G, int& stages) {
  const int64_t tiles = cdiv64(T, 64) * cdiv(N, 64);
  const int all = cdiv(K, dtype == SX_BF16 ? 64 : 32);
  stages = all;
  if (tiles == 0 || tiles > 512) return 0;
  const bool mixed = tiles <= 128 && T <= 16 * (int64_t)G;
  const int parts = (int)std::max<int64_t>(1, std::min<int64_t>(cdiv64(1024, tiles), all / 3));
  stages = cdiv(all, parts);
  const int used = cdiv(all, stages);
  const int64_t one = cdiv64(tiles, 256) * all, split = cdiv64(tiles * used, 256) * stages + 6 + used * T * N * 8 / 1800000;
  return mixed || split < one ? used : 0;
}

template <typename T>
static int split_launch(const ProjectArgs& a, hipStream_t st) {
  constexpr int LDS = 3 * 128 * 128;
  static std::atomic<unsigned long long> done{0};
  SX_TRY(ensure_max_lds((const void*)adapter_tiles_kernel<T, 1, 4, 4, 1, 4, 3, 3, true>, done, "adapter_tiles"));
  int64_t xb, wb;
  tiles_bytes(a, sizeof(T), xb, wb);
  const int gm = (int)cdiv64(a.T, 64), gn = cdiv(a.N, 64);
  hipLaunchKernelGGL((adapter_tiles_kernel<T, 1, 4, 4, 1, 4, 3, 3, true>), dim3(gm * gn, a.parts), dim3(256), LDS, st, a, gm, gn, (unsigned)xb, (unsigned)wb);
  SX_LAUNCH_CHECK("adapter_tiles");
  hipLaunchKernelGGL(adapter_join_kernel<T>, dim3((unsigned)cdiv64(a.T * a.N, 256)), dim3(256), 0, st, a);
  SX_LAUNCH_CHECK("adapter_join");
  return SX_OK;
}

// Rounds of tiles over the 256 CUs times a tile's cost: its area, and more per area the smaller it is (LDS bytes per MFMA)
static double tiles_cost(const ProjectArgs& a, int bm, int bn, int per_cu, double per_area) {
  const int64_t tiles = cdiv64(a.T, bm) * cdiv(a.N, bn);
  return (double)cdiv64(tiles, 256 * per_cu) * per_cu * bm * bn * per_area;
}

template <typename T>
static int tiles_pick(const ProjectArgs& a, hipStream_t st) {
  if (a.parts) return split_launch<T>(a, st);
  const double c0 = tiles_cost(a, 256, 256, 1, 1.0), c1 = tiles_cost(a, 128, 256, 1, 1.2), c2 = tiles_cost(a, 128, 128, 2, 1.4), c3 = tiles_cost(a, 64, 64, 4, 2.0);
  if (c0 <= c1 && c0 <= c2 && c0 <= c3) return tiles_launch<T, 2, 4, 8, 4, 2, 3, 2>(a, st);
  if (c1 <= c2 && c1 <= c3) return tiles_launch<T, 2, 4, 4, 4, 2, 3, 3>(a, st);
  if (c2 <= c3) return tiles_launch<T, 2, 2, 4, 4, 2, 3, 2>(a, st);
  return tiles_launch<T, 1, 4, 4, 1, 4, 3, 3>(a, st);
}

int project_tiles_launch(const ProjectArgs& a, int dtype, hipStream_t st) { return dtype == SX_BF16 ? tiles_pick<bf16>(a, st) : tiles_pick<float>(a, st); }

}  // namespace sx
