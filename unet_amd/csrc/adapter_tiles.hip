// The shared product of the adapter projection (adapters.hip) on bf16 tiles.
//
// A block of WM x WN waves computes BM sorted rows x BN columns, each wave MI x NJ 16x16x32 MFMA fragments.  K steps of 32 go through
// a ring of four LDS buffers filled by LDS-DMA; x is gathered through perm by the DMA's addresses.  The fragments of step s + 1 are
// read while the MFMAs of step s run, so at the top of step s buffer s is free again: the DMA of step s + 4 goes there, with steps s + 2
// and s + 3 in flight behind it.  One barrier and one counted wait per step.  A 64-byte row of a step holds its four 16-byte pieces at
// (piece ^ (row >> 1) & 3): eight lanes that read one piece of consecutive rows then meet eight different parts of the banks.
// The W fragment is the MFMA's left operand: a lane ends up with four consecutive columns of one row.
#include "adapters.h"
#include <algorithm>
#include <atomic>

namespace sx {

template <int N> __device__ __forceinline__ void tiles_wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

template <int WM, int WN, int MI, int NJ, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC) void adapter_tiles_kernel(ProjectArgs a, int gm, int gn, unsigned x_bytes, unsigned w_bytes) {
  constexpr int NT = 64 * WM * WN, BM = WM * MI * 16, BN = WN * NJ * 16, NBUF = 4, RPR = NT / 4;      // RPR: rows per DMA round
  constexpr int SA = BM * 64, SB = BN * 64, STAGE = SA + SB;
  constexpr int QA = SA / (NT * 16), QB = SB / (NT * 16);
  static_assert(SA % (NT * 16) == 0 && SB % (NT * 16) == 0, "whole DMA rounds");
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
  const int piece = (tid & 3) ^ ((tid >> 3) & 3);          // rows advance by RPR, a multiple of 8, from round to round: the same piece in all
#pragma unroll
  for (int q = 0; q < QA; ++q) {
    const int64_t m = m0 + q * RPR + (tid >> 2);
    xo[q] = m < a.T ? (unsigned)((int64_t)a.perm[m] * a.ldx * 2) + piece * 16 : 0x80000000u;
  }
#pragma unroll
  for (int q = 0; q < QB; ++q) {
    const int c = n0 + q * RPR + (tid >> 2);
    wo[q] = c < a.N ? (unsigned)(c * a.ldw * 2) + piece * 16 : 0x80000000u;
  }
  const int nst = (a.K + 31) / 32;
  auto issue = [&](int s) {
    char* buf = smem + (s % NBUF) * STAGE + wid * 1024;
    const bool live = s < nst;                             // past the end: zeros, which keep the count of loads uniform
    const unsigned far = piece * 8 + s * 32 < a.K ? 0u : 0x80000000u;
    __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc((void*)a.x, 0, live ? x_bytes : 0, 0x00020000);
    __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc((void*)a.w, 0, live ? w_bytes : 0, 0x00020000);
#pragma unroll
    for (int q = 0; q < QA; ++q) {
      const unsigned off = (xo[q] + s * 64u) | far;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (__attribute__((address_space(3))) void*)(buf + q * (NT * 16)), 16, off, 0, 0, 0);
    }
#pragma unroll
    for (int q = 0; q < QB; ++q) {
      const unsigned off = (wo[q] + s * 64u) | far;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (__attribute__((address_space(3))) void*)(buf + SA + q * (NT * 16)), 16, off, 0, 0, 0);
    }
  };

  f32x4 acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int row_off = n * 64 + ((gq ^ ((n >> 1) & 3)) << 4);
  const int x_off = wm * MI * 1024 + row_off, w_off = SA + wn * NJ * 1024 + row_off;
  bf16x8 xa[MI], wa[NJ], xb[MI], wb[NJ];
  // step s: multiply the fragments in (xc, wc) while those of step s + 1 arrive in (xn, wn_)
  auto step = [&](int s, bf16x8 (&xc)[MI], bf16x8 (&wc)[NJ], bf16x8 (&xn)[MI], bf16x8 (&wn_)[NJ]) {
    tiles_wait_vm<2 * (QA + QB)>();                           // this wave's pieces of step s + 1 have landed
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");        // and its fragments of step s
    __builtin_amdgcn_s_barrier();                             // ... for every wave: buffer s is free
    issue(s + 4);
    const char* buf = smem + ((s + 1) % NBUF) * STAGE;
    constexpr int READS = MI + NJ, GROUP = MI * NJ / READS;   // MFMAs between two reads
    int done = 0;
#pragma unroll
    for (int t = 0; t < READS; ++t) {
      if (t < NJ) wn_[t] = *reinterpret_cast<const bf16x8*>(buf + w_off + t * 1024);
      else xn[t - NJ] = *reinterpret_cast<const bf16x8*>(buf + x_off + (t - NJ) * 1024);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int e = 0; e < (t == READS - 1 ? MI * NJ - GROUP * (READS - 1) : GROUP); ++e) {
        const int f = t * GROUP + e, i = f / NJ, j = f % NJ;
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wc[j], xc[i], acc[i][j], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
#pragma unroll
  for (int s = 0; s < 4; ++s) issue(s);
  tiles_wait_vm<3 * (QA + QB)>();
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int j = 0; j < NJ; ++j) wa[j] = *reinterpret_cast<const bf16x8*>(smem + w_off + j * 1024);
#pragma unroll
  for (int i = 0; i < MI; ++i) xa[i] = *reinterpret_cast<const bf16x8*>(smem + x_off + i * 1024);
  int s = 0;
  for (; s + 1 < nst; s += 2) {
    step(s, xa, wa, xb, wb);
    step(s + 1, xb, wb, xa, wa);
  }
  if (s < nst) step(s, xa, wa, xb, wb);
  tiles_wait_vm<0>();                                         // no DMA may land in LDS that this block has given back

  // the adapters that this wave's rows meet, 16 ranks at a time
  const int64_t w0 = m0 + wm * MI * 16;
  const int rows = (int)std::min<int64_t>(MI * 16, a.T - w0);
  for (int at = 0; at < rows;) {
    const int g = __builtin_amdgcn_readfirstlane(a.key[w0 + at]);
    if (g >= a.G) break;                                      // the rows without an adapter come last
    const int end = (int)std::min<int64_t>(rows, __builtin_amdgcn_readfirstlane(a.end[g]) - w0);
    const bf16* qg = (const bf16*)a.q + g * a.q_g;
    for (int j0 = 0; j0 < a.r; j0 += 16) {
      const int jr = j0 + (gq & 1) * 8;
      bf16x8 qf[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int c = std::min(n0 + (wn * NJ + j) * 16 + n, a.N - 1);
        qf[j] = load_piece<bf16>(qg + (int64_t)c * a.q_ld, jr, a.q_ld);
      }
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        if (i * 16 >= end || i * 16 + 16 <= at) continue;
        const int64_t m = w0 + std::min(i * 16 + n, rows - 1);
        const bf16x8 hf = *reinterpret_cast<const bf16x8*>((const bf16*)a.h + m * (2 * a.rp) + j0 * 2 + gq * 8);
        const bool mine = i * 16 + n >= at && i * 16 + n < end;     // only its rows: 0 * NaN must not reach the others
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const f32x4 z = {0.f, 0.f, 0.f, 0.f};
          const f32x4 d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qf[j], hf, z, 0, 0, 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] += mine ? d[e] : 0.f;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    at = end;
  }
  const bool wide = a.N % 4 == 0 && a.ldy % 4 == 0 && (uintptr_t)a.y % 8 == 0;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t m = w0 + i * 16 + n;
    if (m < a.T) {
      bf16* y = (bf16*)a.y + (int64_t)a.perm[m] * a.ldy;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int c = n0 + (wn * NJ + j) * 16 + 4 * gq;
        f32x4 v = acc[i][j];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (a.bias && c + e < a.N) v[e] += (float)((const bf16*)a.bias)[c + e];
        if (wide) {
          if (c < a.N) store4(y + c, v);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + e < a.N) y[c + e] = (bf16)v[e];
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

static void tiles_bytes(const ProjectArgs& a, int64_t& xb, int64_t& wb) {
  xb = ((a.T - 1) * a.ldx + a.K) * 2;
  wb = ((int64_t)(a.N - 1) * a.ldw + a.K) * 2;
}

// The DMA's offsets are 32-bit with bit 31 for "out of range"; operands of 2 GiB and more take the other kernel.
bool project_tiles_ok(const ProjectArgs& a) {
  int64_t xb, wb;
  tiles_bytes(a, xb, wb);
  return xb < (1ll << 31) - 4096 && wb < (1ll << 31) - 4096;
}

template <int WM, int WN, int MI, int NJ, int OCC>
static int tiles_launch(const ProjectArgs& a, hipStream_t st) {
  constexpr int BM = WM * MI * 16, BN = WN * NJ * 16, LDS = 4 * (BM + BN) * 64;
  static std::atomic<unsigned long long> done{0};
  SX_TRY(ensure_max_lds((const void*)adapter_tiles_kernel<WM, WN, MI, NJ, OCC>, done, "adapter_tiles"));
  int64_t xb, wb;
  tiles_bytes(a, xb, wb);
  const int gm = (int)cdiv64(a.T, BM), gn = cdiv(a.N, BN);
  hipLaunchKernelGGL((adapter_tiles_kernel<WM, WN, MI, NJ, OCC>), dim3((unsigned)(gm * gn)), dim3(64 * WM * WN), LDS, st, a, gm, gn, (unsigned)xb, (unsigned)wb);
  SX_LAUNCH_CHECK("adapter_tiles");
  return SX_OK;
}

// Rounds of tiles over the 256 CUs times a tile's cost: its area, and more per area the smaller it is (LDS bytes per MFMA)
static double tiles_cost(const ProjectArgs& a, int bm, int bn, int per_cu, double per_area) {
  const int64_t tiles = cdiv64(a.T, bm) * cdiv(a.N, bn);
  return (double)cdiv64(tiles, 256 * per_cu) * per_cu * bm * bn * per_area;
}

int project_tiles_launch(const ProjectArgs& a, hipStream_t st) {
  const double c0 = tiles_cost(a, 256, 256, 1, 1.0), c1 = tiles_cost(a, 128, 256, 1, 1.2), c2 = tiles_cost(a, 128, 128, 2, 1.4), c3 = tiles_cost(a, 64, 64, 4, 2.0);
  if (c0 <= c1 && c0 <= c2 && c0 <= c3) return tiles_launch<2, 4, 8, 4, 2>(a, st);
  if (c1 <= c2 && c1 <= c3) return tiles_launch<2, 4, 4, 4, 2>(a, st);
  if (c2 <= c3) return tiles_launch<2, 2, 4, 4, 2>(a, st);
  return tiles_launch<2, 2, 2, 2, 4>(a, st);
}

}  // namespace sx
