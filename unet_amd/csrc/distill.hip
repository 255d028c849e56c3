// Distillation from a teacher's top logits: the loss of a row of student logits z against K (index, logit) pairs and its gradient.
//
//   p      = softmax over the row's valid pairs of top / tau          (valid: 0 <= index < V)
//   log q  = z / tau - lse(z / tau)
//   loss   = tau^2 * sum_k p_k (log p_k - log q_{idx_k})              (tau^2 keeps the gradient's size as tau changes)
//   dz_v   = c * (q_v - sum_{k: idx_k = v} p_k),   c = tau * weight / den
//
// A row of weight 0 or without a valid pair has loss 0 and gradient 0, whatever its logits hold.
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
  float* row_max;             // [N] max of z, [N] log2 of the sum (what a later gradient pass needs); null: not kept
  float* row_sum;
  void* dz; int64_t lddz;
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

__device__ __forceinline__ int64_t pair_idx(const DistillArgs& a, int64_t at) {
  return a.idx64 ? ((const int64_t*)a.idx)[at] : (int64_t)((const int32_t*)a.idx)[at];
}
__device__ __forceinline__ float pair_top(const DistillArgs& a, int64_t at) {
  return a.top_bf16 ? to_f32(((const bf16*)a.top)[at]) : ((const float*)a.top)[at];
}

// fmaxf drops a NaN; the sum that follows brings it back, as exp(NaN - max) is NaN
template <typename T, int NT>
__global__ __launch_bounds__(NT) void distill_kernel(DistillArgs a, int grad_only) {
  __shared__ float red[NT / 64];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const T* z = (const T*)a.z + row * a.ldz;
  T* dz = a.dz ? (T*)a.dz + row * a.lddz : nullptr;
  const float w = a.weights ? a.weights[row] : 1.f;
  float gup = 1.f;
  if (grad_only) {
    gup = a.g[row * a.g_stride];
    if (a.ready && gup == 1.f) return;         // dz still holds the forward pass's gradient, which is this one
  }
  // teacher
  const int64_t k0 = row * a.K;
  float tm = -INFINITY, any = 0.f;
  for (int k = tid; k < a.K; k += NT) {
    const int64_t id = pair_idx(a, k0 + k);
    if (id >= 0 && id < a.V) { tm = fmaxf(tm, pair_top(a, k0 + k)); any = 1.f; }
  }
  tm = all_max<NT>(tm, red);
  any = all_max<NT>(any, red);
  if (w == 0.f || any == 0.f) {
    if (tid == 0) {
      if (!grad_only) a.row_loss[row] = 0.f;
      if (a.row_max) { a.row_max[row] = 0.f; a.row_sum[row] = 0.f; }
    }
    if (dz) for (int v = tid; v < a.V; v += NT) dz[v] = from_f32<T>(0.f);
    return;
  }
  const float it = 1.f / a.tau, it2 = it * kLog2e;
  float ts = 0.f;
  for (int k = tid; k < a.K; k += NT) {
    const int64_t id = pair_idx(a, k0 + k);
    if (id >= 0 && id < a.V) ts += expf((pair_top(a, k0 + k) - tm) * it);
  }
  ts = all_sum<NT>(ts, red);
  const float lts = logf(ts), its = 1.f / ts;
  // student
  float m, s;
  if (grad_only && a.row_max) {
    m = a.row_max[row];
    s = a.row_sum[row];
  } else {
    m = -INFINITY;
    for (int v = tid; v < a.V; v += NT) m = fmaxf(m, to_f32(z[v]));
    m = all_max<NT>(m, red);
    s = 0.f;
    for (int v = tid; v < a.V; v += NT) s += __builtin_amdgcn_exp2f((to_f32(z[v]) - m) * it2);
    s = all_sum<NT>(s, red);
    if (tid == 0 && a.row_max) { a.row_max[row] = m; a.row_sum[row] = s; }
  }
  if (!grad_only) {
    const float ls = logf(s);
    float kl = 0.f;
    for (int k = tid; k < a.K; k += NT) {
      const int64_t id = pair_idx(a, k0 + k);
      if (id < 0 || id >= a.V) continue;
      const float lp = (pair_top(a, k0 + k) - tm) * it;
      const float p = expf(lp) * its;
      if (!(p == 0.f)) kl += p * ((lp - lts) - ((to_f32(z[id]) - m) * it - ls));
    }
    kl = all_sum<NT>(kl, red);
    if (tid == 0) a.row_loss[row] = kl * a.tau * a.tau * w;
  }
  if (!dz) return;
  const float c = gup * w * a.tau / (a.den ? *a.den : a.den_host);
  const float cs = c / s;
  for (int v = tid; v < a.V; v += NT) dz[v] = from_f32<T>(cs * __builtin_amdgcn_exp2f((to_f32(z[v]) - m) * it2));
  __syncthreads();
  // the teacher's entries over what was just stored; entries that name the same index all store the same value
  for (int k = tid; k < a.K; k += NT) {
    const int64_t id = pair_idx(a, k0 + k);
    if (id < 0 || id >= a.V) continue;
    float p = 0.f;
    for (int j = 0; j < a.K; ++j)
      if (pair_idx(a, k0 + j) == id) p += expf((pair_top(a, k0 + j) - tm) * it) * its;
    const float q = __builtin_amdgcn_exp2f((to_f32(z[id]) - m) * it2) / s;
    dz[id] = from_f32<T>(c * (q - p));
  }
}

// den = max(sum of weights, 1e-8) (the masked losses' floor); one block, fixed order
__global__ __launch_bounds__(1024) void distill_den_kernel(const float* __restrict__ w, int64_t n, float* __restrict__ den) {
  __shared__ float red[16];
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += w[i];
  s = all_sum<1024>(s, red);
  if (threadIdx.x == 0) *den = fmaxf(s, 1e-8f);
}

__global__ __launch_bounds__(1024) void distill_total_kernel(const float* __restrict__ rows, int64_t n, const float* __restrict__ den, float den_host,
                                                             float* __restrict__ out) {
  __shared__ float red[16];
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += rows[i];
  s = all_sum<1024>(s, red);
  if (threadIdx.x == 0) *out = s / (den ? *den : den_host);
}

template <typename T>
static int distill_launch(const DistillArgs& a, int grad_only, hipStream_t st) {
  hipLaunchKernelGGL((distill_kernel<T, 256>), dim3((unsigned)a.N), dim3(256), 0, st, a, grad_only);
  SX_LAUNCH_CHECK("distill");
  return SX_OK;
}

static int distill_check(const char* who, int dtype, int64_t N, int V, int K, int64_t ld, int top_dtype, float tau) {
  SX_REQUIRE((dtype == SX_F32 || dtype == SX_BF16) && (top_dtype == SX_F32 || top_dtype == SX_BF16), "%s: dtypes %d / %d are neither fp32 nor bf16", who, dtype, top_dtype);
  SX_REQUIRE(N >= 0 && N < (1 << 22) && V > 0 && K > 0 && ld >= V, "%s: bad sizes N=%lld V=%d K=%d ld=%lld", who, (long long)N, V, K, (long long)ld);
  SX_REQUIRE(tau > 0.f && tau < INFINITY, "%s: the temperature must be positive and finite, got %g", who, (double)tau);
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
  a.row_max = row_stats; a.row_sum = row_stats ? row_stats + N : nullptr; a.dz = dlogits; a.lddz = ldd;
  if (mean && weights) {
    hipLaunchKernelGGL(distill_den_kernel, dim3(1), dim3(1024), 0, st, weights, N, den);
    SX_LAUNCH_CHECK("distill_den");
    a.den = den;
  }
  if (N > 0) SX_TRY(dtype == SX_BF16 ? distill_launch<bf16>(a, 0, st) : distill_launch<float>(a, 0, st));
  if (loss) {
    hipLaunchKernelGGL(distill_total_kernel, dim3(1), dim3(1024), 0, st, row_loss, N, a.den, a.den_host, loss);
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
  a.row_max = (float*)row_stats; a.row_sum = (float*)row_stats + N; a.dz = dlogits; a.lddz = ldd; a.g = g; a.g_stride = g_stride; a.ready = ready;
  return dtype == SX_BF16 ? distill_launch<bf16>(a, 1, (hipStream_t)stream) : distill_launch<float>(a, 1, (hipStream_t)stream);
}
