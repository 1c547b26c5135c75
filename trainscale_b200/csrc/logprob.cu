// Log-probabilities of chosen tokens, and entropies, out of logits [rows][V], forward and backward.
//
//   y_j = f z_j  or  f c tanh(z_j / c)          (f: logit scale / temperature, c: soft-cap)
//   logp = y_label - lse,  lse = log sum_j e^{y_j},  H = lse - sum_j p_j y_j,  p_j = e^{y_j - lse}
//   dz_j = slope_j f ([j = label] g - p_j (g + h (y_j - lse + H))),  slope_j = 1 - tanh(z_j / c)^2 or 1
//
// With v = z or tanh(z / c) and its maximum m, exponents are u_j = k (v_j - m) in units of log2: differences first, so that large
// logits cost no bits and rows of a type's lowest value do not overflow.  S = sum 2^u and U = sum u 2^u give
// logp = k ln2 (v_label - m) - ln S and H = ln S - ln2 U / S, both terms of which are positive: nothing cancels.
//
// Forward reads the logits once: every thread keeps a running (m, S, U) over 16-byte vectors and raises m once for the vectors that
// it has in flight; the triples meet in the block and, where a row is split, in the cluster's shared memory.
#include <cooperative_groups.h>

#include "common.cuh"
#include "host_common.h"

namespace ts {

constexpr int LP_THREADS = 512;
constexpr int LP_FLIGHT = 4;             // vectors of a thread in flight
constexpr int LP_SPLIT = 8;              // most blocks of a row
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float LP_LOWEST = -1e30f;      // 2^u = 0, and u 2^u = 0 as well

// A maximum that keeps NaN (fmaxf drops it): a NaN anywhere in a row makes its results NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 bytes of logits: N values, their largest, and the pattern of a value that counts for nothing.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static constexpr uint32_t NOTHING = 0xff800000u;
  static __device__ __forceinline__ float value(float v) { return v; }
  static __device__ __forceinline__ float round(float v) { return v; }
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    f[0] = __uint_as_float(r.x), f[1] = __uint_as_float(r.y), f[2] = __uint_as_float(r.z), f[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ float largest(const uint4* r, int n) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      float f[N];
      unpack(r[i], f);
      m = max_nan(m, max_nan(max_nan(f[0], f[1]), max_nan(f[2], f[3])));
    }
    return m;
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr uint32_t NOTHING = 0xff80ff80u;
  static __device__ __forceinline__ float value(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 round(float v) { return __float2bfloat16(v); }
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
  static __device__ __forceinline__ __nv_bfloat162 as2(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
  static __device__ __forceinline__ float largest(const uint4* r, int n) {
    __nv_bfloat162 m = as2(NOTHING);
#pragma unroll
    for (int i = 0; i < n; ++i)
      m = __hmax2_nan(m, __hmax2_nan(__hmax2_nan(as2(r[i].x), as2(r[i].y)), __hmax2_nan(as2(r[i].z), as2(r[i].w))));
    return max_nan(__low2float(m), __high2float(m));
  }
};
template <>
struct Vec<__half> {
  static constexpr int N = 8;
  static constexpr uint32_t NOTHING = 0xfc00fc00u;
  static __device__ __forceinline__ float value(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half round(float v) { return __float2half(v); }
  static __device__ __forceinline__ __half2 as2(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __half22float2(as2(w[i]));
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 t = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float largest(const uint4* r, int n) {
    __half2 m = as2(NOTHING);
#pragma unroll
    for (int i = 0; i < n; ++i)
      m = __hmax2_nan(m, __hmax2_nan(__hmax2_nan(as2(r[i].x), as2(r[i].y)), __hmax2_nan(as2(r[i].z), as2(r[i].w))));
    return max_nan(__low2float(m), __high2float(m));
  }
};

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
};

// tanh(z / c) out of E = e^(-2 |z| / c) <= 1, so that the slope 1 - tanh^2 = 4 E / (1 + E)^2 keeps its bits where tanh is close to one
// (two special-function calls; off by 2^-23 of one).
template <bool CAP>
__device__ __forceinline__ float capped(float z, float inv_cap, float* slope = nullptr) {
  if (!CAP) return z;
  const float e = fast_ex2(fabsf(z) * (-2.f * LOG2E * inv_cap)), r = fast_rcp(1.f + e);
  if (slope) *slope = 4.f * e * r * r;
  return copysignf((1.f - e) * r, z);
}

struct Softmax {
  float m = -INFINITY, s = 0.f, u = 0.f;      // maximum of v; S and U
  template <bool ENT>
  __device__ __forceinline__ void raise(float to, float k2) {
    if (!(to == m) && !(m == -INFINITY)) {
      const float d = max_nan(k2 * (m - to), LP_LOWEST), w = fast_ex2(d);
      if (ENT) u = w * (u + d * s);
      s = w * s;
    }
    m = to;
  }
  template <bool ENT>
  __device__ __forceinline__ void join(const Softmax& o, float k2) {
    Softmax b = o;
    const float to = max_nan(m, b.m);
    raise<ENT>(to, k2);
    b.raise<ENT>(to, k2);
    s += b.s;
    u += b.u;
  }
};

// One block per row, or a cluster of them.
template <typename T, bool CAP, bool ENT>
__global__ void __launch_bounds__(LP_THREADS) logprob_fwd_kernel(const T* __restrict__ logits, const long long* __restrict__ labels,
                                                                 float* __restrict__ logp, float* __restrict__ entropy,
                                                                 float4* __restrict__ kept, LogitRows a) {
  using W = Vec<T>;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), parts = static_cast<int>(cluster.num_blocks());
  __shared__ Softmax by_warp[LP_THREADS / 32];
  __shared__ Softmax by_block[LP_SPLIT];
  const long long row = blockIdx.x / parts;
  const long long label = labels[row];
  if (label == a.ignore) {
    if (threadIdx.x == 0 && rank == 0) {
      logp[row] = 0.f;
      if (entropy) entropy[row] = 0.f;
      if (kept) kept[row] = make_float4(0.f, 1.f, 0.f, 0.f);
    }
    return;                                   // (the whole cluster: it has one row)
  }
  const T* z = logits + a.offset(row);
  // values before the first 16-byte boundary, vectors, values after the last one
  const int head = min(a.V, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / static_cast<int>(sizeof(T)));
  const int vectors = (a.V - head) / W::N, tail = head + vectors * W::N;
  const uint4* body = reinterpret_cast<const uint4*>(z + head);
  const int begin = static_cast<int>(static_cast<long long>(vectors) * rank / parts);
  const int end = static_cast<int>(static_cast<long long>(vectors) * (rank + 1) / parts);
  const uint4 nothing = make_uint4(W::NOTHING, W::NOTHING, W::NOTHING, W::NOTHING);

  Softmax acc;
  auto add = [&](float v, float m) {
    const float t = a.k2 * (v - m), e = fast_ex2(t);
    acc.s += e;
    if (ENT) acc.u += max_nan(t, LP_LOWEST) * e;
  };
  for (int i = begin + static_cast<int>(threadIdx.x); i < end; i += LP_THREADS * LP_FLIGHT) {
    uint4 r[LP_FLIGHT];
#pragma unroll
    for (int j = 0; j < LP_FLIGHT; ++j) r[j] = i + j * LP_THREADS < end ? __ldg(body + i + j * LP_THREADS) : nothing;
    const float top = max_nan(acc.m, capped<CAP>(W::largest(r, LP_FLIGHT), a.inv_cap));
    acc.raise<ENT>(top, a.k2);
    const float m = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int j = 0; j < LP_FLIGHT; ++j) {
      float f[W::N];
      W::unpack(r[j], f);
#pragma unroll
      for (int e = 0; e < W::N; ++e) add(capped<CAP>(f[e], a.inv_cap), m);
    }
  }
  if (rank == 0) {
    const int extra = a.V - vectors * W::N;   // fewer than two vectors
    if (static_cast<int>(threadIdx.x) < extra) {
      const int i = static_cast<int>(threadIdx.x) < head ? threadIdx.x : tail + (threadIdx.x - head);
      const float v = capped<CAP>(W::value(z[i]), a.inv_cap);
      acc.raise<ENT>(max_nan(acc.m, v), a.k2);
      add(v, acc.m == -INFINITY ? 0.f : acc.m);
    }
  }
  auto join_warp = [&](Softmax& x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      Softmax b;
      b.m = __shfl_xor_sync(0xffffffffu, x.m, o);
      b.s = __shfl_xor_sync(0xffffffffu, x.s, o);
      if (ENT) b.u = __shfl_xor_sync(0xffffffffu, x.u, o);
      x.join<ENT>(b, a.k2);
    }
  };
  join_warp(acc);
  if ((threadIdx.x & 31) == 0) by_warp[threadIdx.x >> 5] = acc;
  __syncthreads();
  if (threadIdx.x < 32) {
    acc = threadIdx.x < LP_THREADS / 32 ? by_warp[threadIdx.x] : Softmax();
    join_warp(acc);
  }
  if (parts > 1) {
    if (threadIdx.x == 0) *cluster.map_shared_rank(by_block + rank, 0) = acc;
    cluster.sync();
    if (rank != 0) return;
    if (threadIdx.x == 0) {
      acc = by_block[0];
      for (int i = 1; i < parts; ++i) acc.join<ENT>(by_block[i], a.k2);
    }
  }
  if (threadIdx.x == 0) {
    const bool outside = label < 0 || label >= a.V;
    // a row whose largest logit is +inf, -inf or NaN has no distribution
    const bool proper = acc.m - acc.m == 0.f;
    const float v = outside ? NAN : capped<CAP>(W::value(z[label]), a.inv_cap);
    logp[row] = proper ? a.k * (v - acc.m) - logf(acc.s) : v - acc.m;
    const float H = proper ? logf(acc.s) - LN2 * (acc.u / acc.s) : NAN;
    if (entropy) entropy[row] = H;
    if (kept) kept[row] = make_float4(acc.m, acc.s, H, 0.f);
  }
}

// A block takes LP_THREADS * LP_FLIGHT vectors of one row.
template <typename T, bool CAP, bool ENT>
__global__ void __launch_bounds__(LP_THREADS) logprob_bwd_kernel(const T* __restrict__ logits, const long long* __restrict__ labels,
                                                                 const float4* __restrict__ kept, const float* __restrict__ grad_logp,
                                                                 const float* __restrict__ grad_entropy, T* __restrict__ grad,
                                                                 LogitRows a, int parts) {
  using W = Vec<T>;
  const long long row = blockIdx.x / parts;
  const int part = static_cast<int>(blockIdx.x - row * parts);
  const long long label = labels[row];
  const T* z = logits + a.offset(row);
  T* d = grad + row * a.V;
  const float g = grad_logp ? grad_logp[row] : 0.f, h = ENT ? grad_entropy[row] : 0.f;
  const bool still = label == a.ignore || (g == 0.f && h == 0.f);       // nothing flows back: the row is not read
  // vectors start on the boundaries of the gradient; logits that lie otherwise are read one by one
  const int head = min(a.V, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(d) & 15)) & 15) / static_cast<int>(sizeof(T)));
  const int vectors = (a.V - head) / W::N, tail = head + vectors * W::N;
  uint4* out = reinterpret_cast<uint4*>(d + head);
  const int first = part * (LP_THREADS * LP_FLIGHT) + static_cast<int>(threadIdx.x);
  const int extra = part == 0 ? a.V - vectors * W::N : 0;
  const int lone = static_cast<int>(threadIdx.x) < head ? threadIdx.x : tail + (threadIdx.x - head);
  if (still) {
#pragma unroll
    for (int j = 0; j < LP_FLIGHT; ++j)
      if (first + j * LP_THREADS < vectors) out[first + j * LP_THREADS] = make_uint4(0, 0, 0, 0);
    if (static_cast<int>(threadIdx.x) < extra) d[lone] = W::round(0.f);
    return;
  }
  const bool aligned = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0;
  const uint4* body = reinterpret_cast<const uint4*>(z + head);
  uint4 r[LP_FLIGHT];
  if (aligned) {
#pragma unroll
    for (int j = 0; j < LP_FLIGHT; ++j) r[j] = first + j * LP_THREADS < vectors ? __ldg(body + first + j * LP_THREADS) : make_uint4(0, 0, 0, 0);
  }
  const float4 k = kept[row];
  const float m = k.x, f = a.k * (CAP ? a.inv_cap : 1.f);
  // f p (g + h (ln p + H)) = 2^u (flat + tilt u)
  const float tilt = ENT ? f * h * LN2 / k.y : 0.f, flat = f * (g + (ENT ? h * (k.z - logf(k.y)) : 0.f)) / k.y, fg = f * g;
  auto slope_of = [&](float value, bool chosen) {
    float slope = 1.f;
    const float u = a.k2 * (capped<CAP>(value, a.inv_cap, &slope) - m);
    const float r = (chosen ? fg : 0.f) - fast_ex2(u) * (ENT ? flat + tilt * max_nan(u, LP_LOWEST) : flat);
    return CAP ? slope * r : r;
  };
#pragma unroll
  for (int j = 0; j < LP_FLIGHT; ++j) {
    const int i = first + j * LP_THREADS;
    if (i >= vectors) break;
    float v[W::N], o[W::N];
    if (aligned) {
      W::unpack(r[j], v);
    } else {
#pragma unroll
      for (int e = 0; e < W::N; ++e) v[e] = W::value(z[head + i * W::N + e]);
    }
#pragma unroll
    for (int e = 0; e < W::N; ++e) o[e] = slope_of(v[e], false);
    const long long at = label - head - static_cast<long long>(i) * W::N;
    if (at >= 0 && at < W::N) {
#pragma unroll
      for (int e = 0; e < W::N; ++e)
        if (e == at) o[e] = slope_of(v[e], true);
    }
    out[i] = W::pack(o);
  }
  if (static_cast<int>(threadIdx.x) < extra) d[lone] = W::round(slope_of(W::value(z[lone]), lone == label));
}

// launch(type, cap, entropy) for the kernel's template arguments
template <typename F>
static int by_type(int dtype, bool cap, bool entropy, F&& launch) {
  auto flags = [&](auto* t) {
    using std::false_type;
    using std::true_type;
    return cap ? (entropy ? launch(t, true_type(), true_type()) : launch(t, true_type(), false_type()))
               : (entropy ? launch(t, false_type(), true_type()) : launch(t, false_type(), false_type()));
  };
  switch (dtype) {
    case 0: return flags(static_cast<__nv_bfloat16*>(nullptr));
    case 1: return flags(static_cast<__half*>(nullptr));
    case 2: return flags(static_cast<float*>(nullptr));
    default: return -1;
  }
}

static LogitRows logit_rows(long long rows, long long inner, long long stride_outer, long long stride_inner, int V, float factor,
                            float cap, long long ignore) {
  const float k = factor * (cap > 0.f ? cap : 1.f);
  return {rows, inner, stride_outer, stride_inner, V, k, k * LOG2E, cap > 0.f ? 1.f / cap : 0.f, ignore};
}

}  // namespace ts

using namespace ts;

TS_DEFINE_ERROR_API(ts_logprob)

// dtype: 0 bf16, 1 fp16, 2 fp32.  kept: (m, S, H, unused) of every row, for the backward pass; H counts only with `with_entropy`.
// entropy and kept may be null.
extern "C" int ts_logprob_fwd(const void* logits, int dtype, const long long* labels, float* logp, float* entropy, float4* kept,
                              long long rows, long long inner, long long stride_outer, long long stride_inner, int V, float factor,
                              float cap, long long ignore, void* stream) {
  if (rows <= 0 || inner <= 0 || V <= 0 || rows > 0x7fffffffll / LP_SPLIT) return -1;
  const LogitRows a = logit_rows(rows, inner, stride_outer, stride_inner, V, factor, cap, ignore);
  // a row is split while blocks are fewer than two to an SM and a part has a vector for every thread
  int parts = 1;
  const long long vectors = static_cast<long long>(V) * (dtype == 2 ? 4 : 2) / 16;
  while (parts < LP_SPLIT && rows * parts < 2 * sm_count() && vectors / parts >= 2 * LP_THREADS) parts *= 2;
  return by_type(dtype, cap > 0.f, entropy != nullptr, [&](auto* t, auto c, auto e) {
    using T = std::remove_pointer_t<decltype(t)>;
    return launch_chained(logprob_fwd_kernel<T, decltype(c)::value, decltype(e)::value>, dim3(static_cast<unsigned>(rows * parts)),
                          dim3(LP_THREADS), 0, static_cast<cudaStream_t>(stream), parts, false, static_cast<const T*>(logits), labels,
                          logp, entropy, kept, a);
  });
}

// grad is dense [rows][V]; grad_logp / grad_entropy may be null (zero).
extern "C" int ts_logprob_bwd(const void* logits, int dtype, const long long* labels, const float4* kept, const float* grad_logp,
                              const float* grad_entropy, void* grad, long long rows, long long inner, long long stride_outer,
                              long long stride_inner, int V, float factor, float cap, long long ignore, void* stream) {
  const long long vectors = static_cast<long long>(V) * (dtype == 2 ? 4 : 2) / 16;
  const long long parts = vectors / (LP_THREADS * LP_FLIGHT) + 1;
  if (rows <= 0 || inner <= 0 || V <= 0 || rows > 0x7fffffffll / parts || !kept) return -1;
  const LogitRows a = logit_rows(rows, inner, stride_outer, stride_inner, V, factor, cap, ignore);
  return by_type(dtype, cap > 0.f, grad_entropy != nullptr, [&](auto* t, auto c, auto e) {
    using T = std::remove_pointer_t<decltype(t)>;
    logprob_bwd_kernel<T, decltype(c)::value, decltype(e)::value>
        <<<static_cast<unsigned>(rows * parts), LP_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const T*>(logits), labels, kept, grad_logp, grad_entropy, static_cast<T*>(grad), a, static_cast<int>(parts));
    return static_cast<int>(cudaGetLastError());
  });
}
