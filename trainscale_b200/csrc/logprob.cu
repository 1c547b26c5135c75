// Log-probabilities of chosen tokens, and entropies, out of logits [rows][V], forward and backward.
//
//   y_j = f z_j  or  f c tanh(z_j / c)          (f: logit scale / temperature, c: soft-cap)
//   logp = y_label - lse,  lse = log sum_j e^{y_j},  H = lse - sum_j p_j y_j,  p_j = e^{y_j - lse}
//   dz_j = slope_j f ([j = label] g - p_j (g + h (y_j - lse + H))),  slope_j = 1 - tanh(z_j / c)^2 or 1
//
// With v = z or tanh(z / c) and its maximum m, exponents are u_j = k (v_j - m) in units of log2: differences first, so that large
// logits cost no bits and rows of a type's lowest value do not overflow.  S = sum 2^u and U = sum u 2^u give
// logp = k ln2 (v_label - m) - ln S and H = ln S - ln2 U / S, both terms of which are positive: nothing cancels.
#include "common.cuh"
#include "host_common.h"

namespace ts {

constexpr int LP_THREADS = 512;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float LP_LOWEST = -1e30f;      // 2^u = 0, and u 2^u = 0 as well

// A maximum that keeps NaN (fmaxf drops it): a NaN anywhere in a row makes its results NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half(v); }

struct LogitRows {
  long long rows, inner;             // row r is (r / inner, r % inner)
  long long stride_outer, stride_inner;
  int V;
  float k, k2;                       // f or f c: y = k v; the same times log2(e)
  float inv_cap;                     // 1 / c, or 0
  long long ignore;
  __device__ __forceinline__ long long offset(long long r) const {
    return (r / inner) * stride_outer + (r % inner) * stride_inner;
  }
  __device__ __forceinline__ float capped(float z) const { return inv_cap > 0.f ? tanhf(z * inv_cap) : z; }
};

struct Softmax {
  float m = -INFINITY, s = 0.f, u = 0.f;      // maximum of v; S and U
  __device__ __forceinline__ void raise(float to, float k2) {
    if (!(to == m) && !(m == -INFINITY)) {
      const float d = max_nan(k2 * (m - to), LP_LOWEST), w = fast_ex2(d);
      u = w * (u + d * s);
      s = w * s;
    }
    m = to;
  }
  __device__ __forceinline__ void add(float v, float k2) {
    raise(max_nan(m, v), k2);
    const float t = max_nan(k2 * (v - (m == -INFINITY ? 0.f : m)), LP_LOWEST), e = fast_ex2(t);
    s += e;
    u += t * e;
  }
};

__device__ __forceinline__ float block_max_nan(float v, float* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarp = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  v = lane < nwarp ? scratch[lane] : -INFINITY;
#pragma unroll
  for (int o = 16; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) logprob_fwd_kernel(const T* __restrict__ logits, const long long* __restrict__ labels,
                                                                 float* __restrict__ logp, float* __restrict__ entropy,
                                                                 float4* __restrict__ kept, LogitRows a) {
  __shared__ float scratch[32];
  const long long row = blockIdx.x;
  const long long label = labels[row];
  if (label == a.ignore) {
    if (threadIdx.x == 0) {
      logp[row] = 0.f;
      if (entropy) entropy[row] = 0.f;
      if (kept) kept[row] = make_float4(0.f, 1.f, 0.f, 0.f);
    }
    return;
  }
  const T* z = logits + a.offset(row);
  Softmax acc;
  for (int i = threadIdx.x; i < a.V; i += LP_THREADS) acc.add(a.capped(to_f32(z[i])), a.k2);
  acc.raise(block_max_nan(acc.m, scratch), a.k2);
  const float s = block_sum(acc.s, scratch), u = block_sum(acc.u, scratch);
  if (threadIdx.x == 0) {
    const bool outside = label < 0 || label >= a.V;
    // a row whose largest logit is +inf, -inf or NaN has no distribution
    const bool proper = acc.m - acc.m == 0.f;
    const float v = outside ? NAN : a.capped(to_f32(z[label]));
    logp[row] = proper ? a.k * (v - acc.m) - logf(s) : v - acc.m;
    const float H = proper ? logf(s) - LN2 * (u / s) : NAN;
    if (entropy) entropy[row] = H;
    if (kept) kept[row] = make_float4(acc.m, s, H, 0.f);
  }
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) logprob_bwd_kernel(const T* __restrict__ logits, const long long* __restrict__ labels,
                                                                 const float4* __restrict__ kept, const float* __restrict__ grad_logp,
                                                                 const float* __restrict__ grad_entropy, T* __restrict__ grad,
                                                                 LogitRows a) {
  const long long row = blockIdx.x;
  const long long label = labels[row];
  const T* z = logits + a.offset(row);
  T* d = grad + row * a.V;
  const float g = grad_logp ? grad_logp[row] : 0.f, h = grad_entropy ? grad_entropy[row] : 0.f;
  if (label == a.ignore || (g == 0.f && h == 0.f)) {      // nothing flows back: the row is not read
    for (int i = threadIdx.x; i < a.V; i += LP_THREADS) d[i] = from_f32<T>(0.f);
    return;
  }
  const float4 k = kept[row];
  const float m = k.x, f = a.k * (a.inv_cap > 0.f ? a.inv_cap : 1.f);
  // p (g + h (ln p + H)) = 2^u (flat + tilt u)
  const float tilt = h * LN2 / k.y, flat = (g + (grad_entropy ? h * (k.z - logf(k.y)) : 0.f)) / k.y;
  for (int i = threadIdx.x; i < a.V; i += LP_THREADS) {
    const float v = a.capped(to_f32(z[i]));
    const float u = max_nan(a.k2 * (v - m), LP_LOWEST);
    const float r = (i == label ? g : 0.f) - fast_ex2(u) * (flat + tilt * u);
    d[i] = from_f32<T>(f * r * (a.inv_cap > 0.f ? 1.f - v * v : 1.f));
  }
}

template <typename F>
static int by_type(int dtype, F&& launch) {
  switch (dtype) {
    case 0: launch(static_cast<__nv_bfloat16*>(nullptr)); break;
    case 1: launch(static_cast<__half*>(nullptr)); break;
    case 2: launch(static_cast<float*>(nullptr)); break;
    default: return -1;
  }
  return static_cast<int>(cudaGetLastError());
}

static LogitRows logit_rows(long long rows, long long inner, long long stride_outer, long long stride_inner, int V, float factor,
                            float cap, long long ignore) {
  const float k = factor * (cap > 0.f ? cap : 1.f);
  return {rows, inner, stride_outer, stride_inner, V, k, k * LOG2E, cap > 0.f ? 1.f / cap : 0.f, ignore};
}

}  // namespace ts

using namespace ts;

TS_DEFINE_ERROR_API(ts_logprob)

// dtype: 0 bf16, 1 fp16, 2 fp32.  kept: (m, S, H, unused) of every row, for the backward pass.  entropy and kept may
// be null.
extern "C" int ts_logprob_fwd(const void* logits, int dtype, const long long* labels, float* logp, float* entropy, float4* kept,
                              long long rows, long long inner, long long stride_outer, long long stride_inner, int V, float factor,
                              float cap, long long ignore, void* stream) {
  if (rows <= 0 || inner <= 0 || V <= 0 || rows > 0x7fffffffll) return -1;
  const LogitRows a = logit_rows(rows, inner, stride_outer, stride_inner, V, factor, cap, ignore);
  return by_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    logprob_fwd_kernel<T><<<static_cast<unsigned>(rows), LP_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const T*>(logits), labels, logp, entropy, kept, a);
  });
}

// grad is dense [rows][V]; grad_logp / grad_entropy may be null (zero).
extern "C" int ts_logprob_bwd(const void* logits, int dtype, const long long* labels, const float4* kept, const float* grad_logp,
                              const float* grad_entropy, void* grad, long long rows, long long inner,
                              long long stride_outer, long long stride_inner, int V, float factor, float cap, long long ignore,
                              void* stream) {
  if (rows <= 0 || inner <= 0 || V <= 0 || rows > 0x7fffffffll || !kept) return -1;
  const LogitRows a = logit_rows(rows, inner, stride_outer, stride_inner, V, factor, cap, ignore);
  return by_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    logprob_bwd_kernel<T><<<static_cast<unsigned>(rows), LP_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const T*>(logits), labels, kept, grad_logp, grad_entropy, static_cast<T*>(grad), a);
  });
}
