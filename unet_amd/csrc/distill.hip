// Distillation from a teacher's top logits: the loss of a row of student logits z against K (index, logit) pairs and its gradient.
//
//   p      = softmax over the row's valid pairs of top / tau          (valid: 0 <= index < V, top not -inf)
//   log q  = z / tau - lse(z / tau)
//   loss   = tau^2 * sum_k p_k (log p_k - log q_{idx_k})              (tau^2 keeps the gradient's size as tau changes)
//   dz_v   = c * (q_v - sum_{k: idx_k = v} p_k),   c = tau * weight / den
//
// A row of weight 0 or without a valid pair has loss 0 and gradient 0, whatever its logits hold.
//
// Both directions are bound by memory: what a pass cannot do without is one read of the logits and one write of the gradient.  A block
// therefore keeps its row in registers between the two (rows_kernel): up to 16 vectors of 16 bytes a thread, 1024 threads, 128 Ki bf16 or
// 64 Ki fp32 logits.  Maximum and sum run in one pass (a thread rescales its sum when its maximum grows).  Blocks are persistent, and as
// soon as a register's logits have done their work -- stored as gradients, or summed where no gradient is wanted -- the register takes
// the next row's: the loads of a row run under the work on the one before.  Longer rows, and gradients for another upstream factor
// than 1, read the logits twice (wide_kernel).
//
// Measured, bf16, 256 MB of logits: with the gradient (512 MB) rows of 32000 111 us, 4.8 TB/s, rows of 50000 118 us, of 131072 (512 MB of logits)
// 220 us, 4.9 TB/s; loss alone 50 us, 5.4 TB/s, for rows of 8000 to 50000.  A copy of that size moves 4.9 TB/s.  Shorter rows are bound
// by what a row costs besides (five sums over the lanes, the pairs): rows of 4000 128 us, of 1000 190 us.
#include "sx_common.h"
#include <algorithm>

namespace sx {

struct DistillArgs {
  const void* z; int64_t ldz;
  const void* top; int top_bf16;
  const void* idx; int idx64;
  int64_t N; int V, K;
  float tau;
  const float* weights;       // [N] or null
  const float* den;           // device scalar or null (then den_host)
  float den_host;
  float* row_loss;            // [N]: weight * loss (not divided by den)
  float* row_stats;           // [4][N]: maximum and sum of the logits and of the teacher's (what a later gradient pass needs); null: not kept
  void* dz; int64_t lddz;
  float* den_out;             // sum of the weights, taken and stored by the kernel itself; or null (then den / den_host)
  int ready;                  // gradient pass: dz is as the forward pass left it
  const float* g; int64_t g_stride;      // gradient pass: upstream gradient per row (stride 0: one for all)
};

constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}

// the same value in every thread
template <int NT>
__device__ __forceinline__ float all_max(float v, float* red) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) v = fmaxf(v, red[w]);
  return v;
}
template <int NT>
__device__ __forceinline__ float all_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) v += red[w];
  return v;
}

// the mean's divisor: the sum of the weights, at least 1e-8 (the masked losses' floor); NaN stays NaN
__device__ __forceinline__ float divisor(float sum) { return sum < 1e-8f ? 1e-8f : sum; }

__device__ __forceinline__ int64_t pair_idx(const DistillArgs& a, int64_t at) {
  return a.idx64 ? ((const int64_t*)a.idx)[at] : (int64_t)((const int32_t*)a.idx)[at];
}
__device__ __forceinline__ float pair_top(const DistillArgs& a, int64_t at) {
  return a.top_bf16 ? to_f32(((const bf16*)a.top)[at]) : ((const float*)a.top)[at];
}

// a * b rounded, never fused into a neighbouring addition (in a sum over lanes that would round each lane's own term, and not the others',
// away: the sum would differ from lane to lane)
__device__ __forceinline__ float mul_rn(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// exponent of 2 of a logit relative to the row's maximum.  z * c - m * c in one fma: m * c is rounded, but alike for all of the row (and
// sums move from one maximum to another by the difference of the rounded products).  What the maximum itself gets is that rounding's residual,
// up to half a last place of m * c, in the place of 0: it has to stay far below the 128 where exp2 leaves 32 bits on either side, or the sum is
// infinite or 0 (a masked logit of -1e10 at c = log2 e: 440).  So the form holds for |m * c| < 2^28, a residual of 8 at most, and beyond, rows
// of far values or temperatures near zero, the difference is taken first.
constexpr float kReach = 268435456.f;
// the largest logits that the fma form takes; a thread's maximum starts at minus that, so that a set without a logit above it joins the others
// as the little that it is beside any row maximum in reach
__device__ __forceinline__ float logit_reach(float c) { return fminf(1e30f, kReach / c); }
struct Expo {
  float c, m, mc;
  bool far;
  __device__ __forceinline__ Expo(float m_, float c_, float reach) : c(c_), m(m_), mc(mul_rn(m_, c_)), far(!(fabsf(m_) < reach)) {}
  __device__ __forceinline__ float at(float z) const { return far ? (z - m) * c : fmaf(z, c, -mc); }
};

__device__ __forceinline__ void keep_stats(const DistillArgs& a, int64_t row, float m, float s, float tm, float ts) {
  a.row_stats[row] = m;
  a.row_stats[a.N + row] = s;
  a.row_stats[2 * a.N + row] = tm;
  a.row_stats[3 * a.N + row] = ts;
}

constexpr int kKeptPairs = 256;        // pairs per row that rows_kernel takes at most: one per thread

// E logits of a row as they lie in memory, 16 bytes from 16-byte boundaries: element e of vector v is the row's element v * E + e - off,
// off being the row's start behind a boundary.  Elements before and behind the row read as -inf and are not stored.
template <typename T>
__device__ __forceinline__ typename Elem<T>::Vec load_row_vec(const T* __restrict__ z, int off, int V, int v) {
  constexpr int E = Elem<T>::EPL;
  const int i = v * E - off;
  typename Elem<T>::Vec r;
  if (i >= 0 && i + E <= V) return *reinterpret_cast<const typename Elem<T>::Vec*>(z + i);
#pragma unroll
  for (int e = 0; e < E; ++e) r[e] = (i + e >= 0 && i + e < V) ? z[i + e] : from_f32<T>(-INFINITY);
  return r;
}
template <typename T>
__device__ __forceinline__ void store_row_vec(T* __restrict__ d, int off, int V, int v, bool whole, typename Elem<T>::Vec r) {
  constexpr int E = Elem<T>::EPL;
  const int i = v * E - off;
  if (whole && i >= 0 && i + E <= V) { *reinterpret_cast<typename Elem<T>::Vec*>(d + i) = r; return; }
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (i + e >= 0 && i + e < V) d[i + e] = r[e];
}
template <typename T>
__device__ __forceinline__ int row_off(const T* z) { return (int)(((uintptr_t)z & 15) / sizeof(T)); }

// Row = nh elements up to the first 16-byte boundary, nb whole vectors, the rest.  Vector v belongs to thread v % NT, register v / NT; the
// elements before and behind the vectors to threads 0, 1, ... one each.  Pair k belongs to thread k; the gradient at its index is
// stored once more, over the plain q of the row's other elements, behind the next barrier that the block meets anyway.
template <typename T, int NT, int NV, bool GRAD>
__global__ __launch_bounds__(NT) void distill_rows_kernel(DistillArgs a) {
  constexpr int E = Elem<T>::EPL, NW = NT / 64, PAIRS = NT < kKeptPairs ? NT : kKeptPairs;
  typedef typename Elem<T>::Vec Vec;
  __shared__ float red[5][NW];                          // per wave: maximum and sum of the logits and of the teacher's, any pair
  __shared__ float red_kl[NW];
  __shared__ float pair_p[PAIRS];
  __shared__ int pair_i[PAIRS];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const float it = 1.f / a.tau, c = it * kLog2e, reach = logit_reach(c);
  float den = a.den_host;
  if (a.den_out) {
    float s = 0.f;
    for (int64_t i = tid; i < a.N; i += NT) s += a.weights[i];
    s = all_sum<NT>(s, red_kl);
    den = divisor(s);
    if (blockIdx.x == 0 && tid == 0) *a.den_out = den;
  } else if (a.den) {
    den = *a.den;
  }
  const unsigned my = tid * 16u;                        // bytes: with the block's own base in scalar registers, one offset for all vectors
  // vector k of a row, from its descriptor: behind the last one the load is not made, with no branch around it (a branch would leave the
  // number of loads in flight open, and a wait for one would be a wait for all)
  auto row_desc = [](const T* z, int nh, int nb) { return __builtin_amdgcn_make_buffer_rsrc((void*)(z + nh), 0, nb * 16, 0x00020000); };
  auto load_vec = [&](__amdgpu_buffer_rsrc_t d, int k) { return __builtin_bit_cast(Vec, __builtin_amdgcn_raw_buffer_load_b128(d, my, k * NT * 16, 0)); };
  auto shape = [&](const T* z, int& nh, int& nb) {
    nh = std::min(a.V, (int)((16 - ((uintptr_t)z & 15)) & 15) / (int)sizeof(T));
    nb = (a.V - nh) / E;
  };
  auto weight = [&](int64_t t) { return t < a.N ? (a.weights ? a.weights[t] : 1.f) : 0.f; };
  // a weight is the same in all lanes: its test in scalar registers, so that what it selects (the descriptors) stays there
  auto is_zero = [](float v) { return (__builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)) & 0x7fffffff) == 0; };
  Vec r[NV];
  T loose = {};                                         // as loaded: the conversions wait until the values are needed
  int64_t pair_raw = -1;
  unsigned top_raw = 0;
  auto load_head = [&](int64_t t, int nh, int nb) {     // row t's loose element and pair of this thread
    const T* z = (const T*)a.z + t * a.ldz;
    if (tid < a.V - nb * E) loose = z[tid < nh ? tid : tid + nb * E];
    if (tid < a.K) {
      const int64_t at = t * a.K + tid;
      if (a.idx64) pair_raw = ((const int64_t*)a.idx)[at];
      else pair_raw = ((const int32_t*)a.idx)[at];
      if (a.top_bf16) top_raw = ((const uint16_t*)a.top)[at];
      else top_raw = ((const uint32_t*)a.top)[at];
    }
  };
  int64_t row = blockIdx.x;
  float w = weight(row), wn = weight(row + gridDim.x);    // of this row and the next: loaded a row ahead, for nothing to wait on them
  {
    const T* z = (const T*)a.z + row * a.ldz;
    int nh, nb;
    shape(z, nh, nb);
    if (is_zero(w)) nb = 0;
    else load_head(row, nh, nb);
    const auto d = row_desc(z, nh, nb);
#pragma unroll
    for (int k = 0; k < NV; ++k) r[k] = load_vec(d, k);
  }
  T* fix_at = nullptr;                                  // the row before: where this thread's pair stands and the gradient there
  float fix = 0.f;
  for (; row < a.N; row += gridDim.x) {
    const T* z = (const T*)a.z + row * a.ldz;
    T* dz = GRAD ? (T*)a.dz + row * a.lddz : nullptr;
    const int64_t next = row + gridDim.x;
    const float wnn = weight(next + gridDim.x);
    int nh, nb;
    shape(z, nh, nb);
    const bool has_loose = tid < a.V - nb * E, on = !is_zero(w), onn = !is_zero(wn);
    const float pt = __builtin_bit_cast(float, a.top_bf16 ? top_raw << 16 : top_raw);
    const bool paired = on && tid < a.K && pair_raw >= 0 && pair_raw < a.V && pt != -INFINITY;
    const int pi = paired ? (int)pair_raw : -1;
    const float zp = paired ? to_f32(z[pi]) : 0.f;
    const float zl = to_f32(loose);
    const T* zn = (const T*)a.z + next * a.ldz;
    int nhn, nbn;
    shape(zn, nhn, nbn);
    if (!onn) nbn = 0;
    const auto dn = row_desc(zn, nhn, nbn);
    float m = -reach, s = 0.f;
    if (on && has_loose) {
      m = fmaxf(m, zl);
      s = __builtin_amdgcn_exp2f(fmaf(zl, c, -mul_rn(m, c)));
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (on && tid < nb - k * NT) {
        float f[E], mk = m;
#pragma unroll
        for (int e = 0; e < E; ++e) { f[e] = to_f32(r[k][e]); mk = fmaxf(mk, f[e]); }
        const float mc = mul_rn(mk, c);
        s *= __builtin_amdgcn_exp2f(mul_rn(m, c) - mc);
#pragma unroll
        for (int e = 0; e < E; ++e) s += __builtin_amdgcn_exp2f(fmaf(f[e], c, -mc));
        m = mk;
      }
      if (!GRAD) r[k] = load_vec(dn, k);                // without a gradient the row has done its work
      __builtin_amdgcn_sched_barrier(0);
    }
    float M = wave_max(m), S = wave_sum(mul_rn(s, __builtin_amdgcn_exp2f(mul_rn(m, c) - mul_rn(M, c))));
    float TM = wave_max(paired ? pt : -INFINITY), TS = wave_sum(paired ? expf((pt - TM) * it) : 0.f);
    float any = __ballot(paired) ? 1.f : 0.f;
    if (NW > 1 && lane == 0) { red[0][wid] = M; red[1][wid] = S; red[2][wid] = TM; red[3][wid] = TS; red[4][wid] = any; }
    __syncthreads();                                    // and every thread has stored its part of the row before
    if (fix_at) *fix_at = from_f32<T>(fix);
    fix_at = nullptr;
    if constexpr (NW > 1) {                             // every wave's results, over the lanes
      const int ww = lane & (NW - 1);
      const float m1 = red[0][ww], tm1 = red[2][ww], any1 = red[4][ww];
      M = wave_max(m1);
      TM = wave_max(tm1);
      any = wave_max(any1);
      S = wave_sum(lane < NW ? mul_rn(red[1][ww], __builtin_amdgcn_exp2f(mul_rn(m1, c) - mul_rn(M, c))) : 0.f);
      TS = wave_sum(lane < NW && any1 != 0.f ? mul_rn(red[3][ww], expf((tm1 - TM) * it)) : 0.f);
    }
    const bool live = on && any != 0.f;
    const bool far = live && !(fabsf(M) < reach);       // the row again, by differences
    if (far) {
      float mk = -INFINITY;
      for (int v = tid; v < a.V; v += NT) mk = fmaxf(mk, to_f32(z[v]));
      M = all_max<NT>(mk, red_kl);
      float sk = 0.f;
      for (int v = tid; v < a.V; v += NT) sk += __builtin_amdgcn_exp2f((to_f32(z[v]) - M) * c);
      S = all_sum<NT>(sk, red_kl);
      __syncthreads();
    }
    const float gc = w * a.tau / den, gs = gc / S, mc = mul_rn(M, c);
    if (tid < PAIRS) {
      float p = 0.f, kl = 0.f;
      if (live && paired) {
        const float lt = (pt - TM) * it;
        p = expf(lt) / TS;
        const Expo x(M, c, reach);
        if (!(p == 0.f)) kl = p * ((lt - logf(TS)) - (x.at(zp) * kLn2 - logf(S)));
      }
      pair_i[tid] = pi;
      pair_p[tid] = p;
      kl = wave_sum(kl);
      if (lane == 0) red_kl[wid] = kl;
    }
    __syncthreads();
    if (tid == 0) {
      float kl = 0.f;
#pragma unroll
      for (int i = 0; i < PAIRS / 64; ++i) kl += red_kl[i];
      a.row_loss[row] = live ? kl * a.tau * a.tau * w : 0.f;
      if (a.row_stats) keep_stats(a, row, M, S, TM, TS);
    }
    if (GRAD && live && wid * 64 < a.K) {                 // the gradient at the pairs' indices, in the order of the pairs
      const Expo x(M, c, reach);
      fix = gs * __builtin_amdgcn_exp2f(x.at(zp));
      for (int j = 0; j < a.K; ++j) fix = pair_i[j] == pi ? fmaf(-gc, pair_p[j], fix) : fix;
      if (paired) fix_at = dz + pi;
    }
    if (onn) load_head(next, nhn, nbn);
    if (GRAD && has_loose && !far) dz[tid < nh ? tid : tid + nb * E] = from_f32<T>(live ? gs * __builtin_amdgcn_exp2f(fmaf(zl, c, -mc)) : 0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (GRAD && !far && tid < nb - k * NT) {
        Vec o = {};
        if (live)
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] = from_f32<T>(gs * __builtin_amdgcn_exp2f(fmaf(to_f32(r[k][e]), c, -mc)));
        *reinterpret_cast<Vec*>(reinterpret_cast<char*>(dz + nh + k * NT * E) + my) = o;
      }
      if (GRAD) r[k] = load_vec(dn, k);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (GRAD && far)
      for (int v = tid; v < a.V; v += NT) dz[v] = from_f32<T>(gs * __builtin_amdgcn_exp2f((to_f32(z[v]) - M) * c));
    w = wn;
    wn = wnn;
  }
  __syncthreads();
  if (fix_at) *fix_at = from_f32<T>(fix);
}

// any row length and any number of pairs (each compared with every other: the time grows with K * K beyond the few hundred that a block of
// threads holds), the logits read once for the maximum and the sum and once for the gradient; with GRAD_ONLY, the gradient alone, from
// the maxima and sums of an earlier pass.  fmaxf drops a NaN; the sum brings it back
template <typename T, int NT, bool GRAD_ONLY>
__global__ __launch_bounds__(NT) void distill_wide_kernel(DistillArgs a) {
  constexpr int E = Elem<T>::EPL;
  typedef typename Elem<T>::Vec Vec;
  __shared__ float red[NT / 64];
  __shared__ int64_t pair_i[NT];
  __shared__ float pair_p[NT];
  const int tid = threadIdx.x;
  const float it = 1.f / a.tau, c = it * kLog2e, reach = logit_reach(c);
  if (GRAD_ONLY && a.ready && a.g_stride == 0 && *a.g == 1.f) return;      // dz still holds the forward pass's gradient, which is this one
  for (int64_t row = blockIdx.x; row < a.N; row += gridDim.x) {
    const T* z = (const T*)a.z + row * a.ldz;
    T* dz = a.dz ? (T*)a.dz + row * a.lddz : nullptr;
    const int off = row_off(z), nv = (a.V + off + E - 1) / E;
    const bool whole = dz && row_off(dz) == off;
    const float w = a.weights ? a.weights[row] : 1.f;
    const float gup = GRAD_ONLY ? a.g[row * a.g_stride] : 1.f;
    if (GRAD_ONLY && a.ready && gup == 1.f) continue;
    const int64_t k0 = row * a.K;
    float m, s, tm, ts;                                   // ts = 0: no valid pair, otherwise >= 1 or NaN
    if constexpr (GRAD_ONLY) {
      m = a.row_stats[row];
      s = a.row_stats[a.N + row];
      tm = a.row_stats[2 * a.N + row];
      ts = a.row_stats[3 * a.N + row];
    } else {
      tm = -INFINITY;
      float any = 0.f;
      for (int k = tid; k < a.K; k += NT) {
        const int64_t id = pair_idx(a, k0 + k);
        const float t = pair_top(a, k0 + k);
        if (id >= 0 && id < a.V && t != -INFINITY) { tm = fmaxf(tm, t); any = 1.f; }
      }
      tm = all_max<NT>(tm, red);
      any = all_max<NT>(any, red);
      ts = 0.f;
      for (int k = tid; k < a.K; k += NT) {
        const int64_t id = pair_idx(a, k0 + k);
        const float t = pair_top(a, k0 + k);
        if (id >= 0 && id < a.V && t != -INFINITY) ts += expf((t - tm) * it);
      }
      ts = all_sum<NT>(ts, red);
      if (any == 0.f) ts = 0.f;
      m = s = 0.f;
    }
    const bool live = w != 0.f && !(ts == 0.f);
    if (!GRAD_ONLY && live) {
      float mk = -reach;                                  // as in rows_kernel: a thread rescales its sum when its maximum grows
#pragma unroll 4
      for (int v = tid; v < nv; v += NT) {
        const Vec r = load_row_vec<T>(z, off, a.V, v);
        float f[E], mn = mk;
#pragma unroll
        for (int e = 0; e < E; ++e) { f[e] = to_f32(r[e]); mn = fmaxf(mn, f[e]); }
        const float mc = mul_rn(mn, c);
        s *= __builtin_amdgcn_exp2f(mul_rn(mk, c) - mc);
#pragma unroll
        for (int e = 0; e < E; ++e) s += __builtin_amdgcn_exp2f(fmaf(f[e], c, -mc));
        mk = mn;
      }
      m = all_max<NT>(mk, red);
      s = mul_rn(s, __builtin_amdgcn_exp2f(mul_rn(mk, c) - mul_rn(m, c)));
      if (!(fabsf(m) < reach)) {                          // the row again, by differences
        mk = -INFINITY;
        for (int v = tid; v < a.V; v += NT) mk = fmaxf(mk, to_f32(z[v]));
        m = all_max<NT>(mk, red);
        const Expo x(m, c, reach);
        s = 0.f;
        for (int v = tid; v < a.V; v += NT) s += __builtin_amdgcn_exp2f(x.at(to_f32(z[v])));
      }
      s = all_sum<NT>(s, red);
    }
    const Expo x(m, c, reach);
    if constexpr (!GRAD_ONLY) {
      const float ls = logf(s), lts = logf(ts);
      float kl = 0.f;
      if (live)
        for (int k = tid; k < a.K; k += NT) {
          const int64_t id = pair_idx(a, k0 + k);
          if (id < 0 || id >= a.V) continue;
          const float lp = (pair_top(a, k0 + k) - tm) * it;
          const float p = expf(lp) / ts;
          if (!(p == 0.f)) kl += p * ((lp - lts) - (x.at(to_f32(z[id])) * kLn2 - ls));
        }
      kl = all_sum<NT>(kl, red);
      if (tid == 0) {
        a.row_loss[row] = live ? kl * a.tau * a.tau * w : 0.f;
        if (a.row_stats) keep_stats(a, row, m, s, tm, ts);
      }
    }
    if (!dz) continue;
    const float gc = gup * w * a.tau / (a.den ? *a.den : a.den_host), gs = gc / s;
    for (int v = tid; v < nv; v += NT) {
      Vec o = {};
      if (live) {
        const Vec r = load_row_vec<T>(z, off, a.V, v);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = from_f32<T>(gs * __builtin_amdgcn_exp2f(x.at(to_f32(r[e]))));
      }
      store_row_vec<T>(dz, off, a.V, v, whole, o);
    }
    if (!live) continue;
    // the teacher's entries over what was just stored (behind the barriers below), NT pairs at a time against NT; entries that name the same
    // index all store the same value
    for (int kb = 0; kb < a.K; kb += NT) {
      int64_t id = -1;
      if (kb + tid < a.K) id = pair_idx(a, k0 + kb + tid);
      if (id >= a.V) id = -1;
      float g = id >= 0 ? gs * __builtin_amdgcn_exp2f(x.at(to_f32(z[id]))) : 0.f;
      for (int jb = 0; jb < a.K; jb += NT) {
        __syncthreads();
        if (jb + tid < a.K) {
          pair_i[tid] = pair_idx(a, k0 + jb + tid);
          pair_p[tid] = expf((pair_top(a, k0 + jb + tid) - tm) * it) / ts;
        }
        __syncthreads();
        for (int j = 0; j < std::min(NT, a.K - jb); ++j) g = pair_i[j] == id ? fmaf(-gc, pair_p[j], g) : g;
      }
      if (id >= 0) dz[id] = from_f32<T>(g);
    }
    __syncthreads();                                      // the pairs have been read
  }
}

// sum of n floats by one block of 1024 threads, four neighbours a thread at a time, in an order that depends on n alone (4 us for 16384)
__device__ __forceinline__ float sum_all(const float* __restrict__ p, int64_t n, float* red) {
  float s[4] = {};
  const bool whole = (uintptr_t)p % 16 == 0;
  const int64_t whole_end = whole ? n & ~3ll : 0;
  int64_t i = threadIdx.x * 4, base = 0;
  constexpr int U = 8;                                  // loads in flight, none behind a test of its own
  for (; base + U * 4096 <= whole_end; base += U * 4096, i += U * 4096) {
    f32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = *reinterpret_cast<const f32x4*>(p + i + u * 4096);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += v[u][e];
  }
  for (; i < whole_end; i += 4096) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(p + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += v[e];
  }
  for (; i < n; i += 4096)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i + e < n) s[e] += p[i + e];
  return all_sum<1024>((s[0] + s[1]) + (s[2] + s[3]), red);
}

__global__ __launch_bounds__(1024) void distill_den_kernel(const float* __restrict__ w, int64_t n, float* __restrict__ den) {
  __shared__ float red[16];
  const float s = sum_all(w, n, red);
  if (threadIdx.x == 0) *den = divisor(s);
}

__global__ __launch_bounds__(1024) void distill_total_kernel(const float* __restrict__ rows, int64_t n, const float* __restrict__ den, float den_host,
                                                             float* __restrict__ out) {
  __shared__ float red[16];
  const float s = sum_all(rows, n, red);
  if (threadIdx.x == 0) *out = s / (den ? *den : den_host);
}

template <typename T, int NT, int NV>
static int rows_launch(const DistillArgs& a, int per_cu, hipStream_t st) {
  const dim3 grid((unsigned)std::min<int64_t>(a.N, 256 * per_cu));
  if (a.dz) hipLaunchKernelGGL((distill_rows_kernel<T, NT, NV, true>), grid, dim3(NT), 0, st, a);
  else hipLaunchKernelGGL((distill_rows_kernel<T, NT, NV, false>), grid, dim3(NT), 0, st, a);
  SX_LAUNCH_CHECK("distill_rows");
  return SX_OK;
}

template <typename T, int NT>
static int wide_start(const DistillArgs& a, int grad_only, hipStream_t st) {
  const dim3 grid((unsigned)std::min<int64_t>(a.N, 256 * (2048 / NT)));
  if (grad_only) hipLaunchKernelGGL((distill_wide_kernel<T, NT, true>), grid, dim3(NT), 0, st, a);
  else hipLaunchKernelGGL((distill_wide_kernel<T, NT, false>), grid, dim3(NT), 0, st, a);
  SX_LAUNCH_CHECK("distill_wide");
  return SX_OK;
}

template <typename T>
static int wide_launch(const DistillArgs& a, int grad_only, hipStream_t st) {
  // a wave for a short row, more for a long one, most of them where there are few rows.  Gradient of 256 MB of bf16 logits with K = 16: rows of
  // 4000 by one wave 160 us, by four 222; of 50000 by four 122, by sixteen 137; of 131072 113 and 114
  // Many pairs: K * K comparisons of a row (distill_wide_kernel) over as many threads as there are, unless rows enough for a wave each to fill
  // the card have few of them.  fp32, loss and gradient, by one wave and by sixteen: 16 rows with K = 513 0.40 ms and 0.12, 1000 1.28 and 0.11,
  // 8000 76 and 4.2; 8192 rows with K = 513 1.05 and 1.4, 1000 3.0 and 2.4
  if (a.K > 768 || (a.K > 512 && a.N < 4096)) return wide_start<T, 1024>(a, grad_only, st);
  if (a.V <= 8192) return wide_start<T, 64>(a, grad_only, st);
  if (a.N >= 512) return wide_start<T, 256>(a, grad_only, st);
  return wide_start<T, 1024>(a, grad_only, st);
}

// rows_kernel: the row fits the registers, its pairs the threads, exponents the fma form, and the gradient's rows lie to the 16-byte
// boundaries as the logits' do
static bool rows_fit(const DistillArgs& a, int dtype) {
  const int64_t b = (int64_t)dtype_size(dtype), e = 16 / b;
  return a.V <= 16 * 1024 * e && a.K <= kKeptPairs && a.tau >= 1e-6f &&
         (!a.dz || (((uintptr_t)a.dz - (uintptr_t)a.z) % 16 == 0 && (a.N == 1 || (a.lddz - a.ldz) * b % 16 == 0)));
}

template <typename T>
static int distill_launch(const DistillArgs& a, hipStream_t st) {
  constexpr int E = Elem<T>::EPL;
  if (!rows_fit(a, Elem<T>::kDtype)) return wide_launch<T>(a, 0, st);
  const int nv = a.V / E;                               // whole vectors, at most
  // Few vectors a thread cost little to sum over the threads, many keep more of a row's loads in flight with fewer waves to wait for one
  // another: the latter wins nearly everywhere.  256 MB of bf16 logits with / without a gradient: rows of 1000 by one wave 190 / 91 us, by four
  // 643 / 450; of 2000 by one 151 / 64, by two 212 / 122; of 16000 by 256 threads 117 / 50, by 512 119 / 63; of 32000 by 256 115 / 51, by 512
  // 111 / 52; of 24000 without a gradient 50 and 58; of 50000 by 512 118 / 50, by 1024 131 / 62.
  if (a.K <= 64) {                                      // (one pair per thread)
    if (nv <= 64) return rows_launch<T, 64, 1>(a, 32, st);
    if (nv <= 128) return rows_launch<T, 64, 2>(a, 32, st);
    if (nv <= 256) return rows_launch<T, 64, 4>(a, 28, st);
    if (nv <= 512) return rows_launch<T, 64, 8>(a, 20, st);
    if (nv <= 1024) return rows_launch<T, 64, 16>(a, 16, st);
  }
  if (a.K <= 128) {
    if (nv <= 256) return rows_launch<T, 128, 2>(a, 16, st);
    if (nv <= 512) return rows_launch<T, 128, 4>(a, 14, st);
    if (nv <= 1024) return rows_launch<T, 128, 8>(a, 10, st);
  }
  if (nv <= 256) return rows_launch<T, 256, 1>(a, 8, st);
  if (nv <= 512) return rows_launch<T, 256, 2>(a, 8, st);
  if (nv <= 1024) return rows_launch<T, 256, 4>(a, 6, st);
  if (nv <= 2048) return rows_launch<T, 256, 8>(a, 5, st);
  if (nv <= 4096) return a.dz ? rows_launch<T, 512, 8>(a, 2, st) : rows_launch<T, 256, 16>(a, 4, st);
  if (nv <= 8192) return rows_launch<T, 512, 16>(a, 2, st);
  return rows_launch<T, 1024, 16>(a, 1, st);
}

static int distill_check(const char* who, int dtype, int64_t N, int V, int K, int64_t ld, int top_dtype, float tau) {
  SX_REQUIRE((dtype == SX_F32 || dtype == SX_BF16) && (top_dtype == SX_F32 || top_dtype == SX_BF16), "%s: dtypes %d / %d are neither fp32 nor bf16", who, dtype, top_dtype);
  SX_REQUIRE(N >= 0 && N < (1 << 22) && V > 0 && V <= (1 << 30) && K > 0 && K <= (1 << 30) && ld >= V, "%s: bad sizes N=%lld V=%d K=%d ld=%lld", who, (long long)N, V, K, (long long)ld);
  SX_REQUIRE(tau >= 1.17549435e-38f && tau < INFINITY, "%s: the temperature must be positive, normal and finite, got %g", who, (double)tau);      // 1 / tau is finite
  return SX_OK;
}

}  // namespace sx

using namespace sx;

extern "C" int sx_distill_forward(int dtype, int64_t N, int V, int K, const void* logits, int64_t ld, int top_dtype, const void* top, const void* idx,
                                  int idx64, float tau, const float* weights, int mean, float* row_loss, float* row_stats, float* den, float* loss,
                                  void* dlogits, int64_t ldd, void* stream) {
  SX_TRY(distill_check("sx_distill_forward", dtype, N, V, K, ld, top_dtype, tau));
  SX_REQUIRE((N == 0 || (logits && top && idx && row_loss)) && (!dlogits || ldd >= V) && (!mean || !weights || den), "sx_distill_forward: null pointer or bad stride");
  hipStream_t st = (hipStream_t)stream;
  DistillArgs a = {};
  a.z = logits; a.ldz = ld; a.top = top; a.top_bf16 = top_dtype == SX_BF16; a.idx = idx; a.idx64 = idx64; a.N = N; a.V = V; a.K = K; a.tau = tau;
  a.weights = weights; a.den_host = mean ? fmaxf((float)N, 1e-8f) : 1.f; a.row_loss = row_loss;
  a.row_stats = row_stats; a.dz = dlogits; a.lddz = ldd;
  if (mean && weights) {
    // few enough weights for every block to add up itself, sixteen a thread: 8192 rows of 1000 with a wave each 40 us, with a launch for
    // the sum 17
    const int64_t few = V <= 1024 * (16 / (int)dtype_size(dtype)) ? 1024 : V <= 8192 * (16 / (int)dtype_size(dtype)) ? 4096 : 16384;
    if (N > 0 && N <= few && rows_fit(a, dtype)) {
      a.den_out = den;
    } else {
      hipLaunchKernelGGL(distill_den_kernel, dim3(1), dim3(1024), 0, st, weights, N, den);
      SX_LAUNCH_CHECK("distill_den");
      a.den = den;
    }
  }
  if (N > 0) SX_TRY(dtype == SX_BF16 ? distill_launch<bf16>(a, st) : distill_launch<float>(a, st));
  if (loss) {
    hipLaunchKernelGGL(distill_total_kernel, dim3(1), dim3(1024), 0, st, row_loss, N, mean && weights ? den : nullptr, a.den_host, loss);
    SX_LAUNCH_CHECK("distill_total");
  }
  return SX_OK;
}

extern "C" int sx_distill_backward(int dtype, int64_t N, int V, int K, const void* logits, int64_t ld, int top_dtype, const void* top, const void* idx,
                                   int idx64, float tau, const float* weights, int mean, const float* row_stats, const float* den, const float* g,
                                   int64_t g_stride, int ready, void* dlogits, int64_t ldd, void* stream) {
  SX_TRY(distill_check("sx_distill_backward", dtype, N, V, K, ld, top_dtype, tau));
  if (N == 0) return SX_OK;
  SX_REQUIRE(logits && top && idx && row_stats && g && dlogits && ldd >= V && (!mean || !weights || den), "sx_distill_backward: null pointer or bad stride");
  DistillArgs a = {};
  a.z = logits; a.ldz = ld; a.top = top; a.top_bf16 = top_dtype == SX_BF16; a.idx = idx; a.idx64 = idx64; a.N = N; a.V = V; a.K = K; a.tau = tau;
  a.weights = weights; a.den_host = mean ? fmaxf((float)N, 1e-8f) : 1.f; a.den = mean && weights ? den : nullptr;
  a.row_stats = (float*)row_stats; a.dz = dlogits; a.lddz = ldd; a.g = g; a.g_stride = g_stride; a.ready = ready;
  return dtype == SX_BF16 ? wide_launch<bf16>(a, 1, (hipStream_t)stream) : wide_launch<float>(a, 1, (hipStream_t)stream);
}
