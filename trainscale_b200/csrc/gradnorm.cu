// The global norm of a list of gradients, and their scaling by min(1, limit / (norm + 1e-6)).
//
// The list goes to the kernels by value (a launch takes up to 32 KB of parameters), so that nothing is copied to the device or
// kept between calls.  Norms: 2 (sqrt of the sum of squares), 1, inf.  A thread sums the 64 values that it has in flight in fp32
// and adds the sum to an fp64 one; where that sum leaves the range in which fp32 squares keep their bits it is made again in
// fp64.  The order of all sums depends on the sizes alone.
//
// Bounds: the memory.  1.05 GB of bf16 gradients: norm 163 to 170 us (6.2 to 6.4 TB/s), scaling 317 (6.6 TB/s); a norm below the
// limit ends the second kernel at its first instruction.  Blocks of 512 threads with eight vectors each in flight; plain loads of
// single values took 326 and 930. 128 tensors of 10 KB to 0.5 MB: 17 us on the GPU, 75 to 90 for the list's way through Python.
#include <algorithm>
#include <vector>

#include "common.cuh"
#include "host_common.h"

namespace ts {

constexpr int GN_THREADS = 512;
constexpr int GN_FLIGHT = 8;                       // 16-byte vectors of a thread in flight
constexpr int GN_CHUNK_BYTES = GN_THREADS * GN_FLIGHT * 16;      // of a block's turn
constexpr int GN_FEW = 256, GN_TENSORS = 1024;     // tensors of a launch: the parameters of a short list are quicker to pass

template <int TENSORS>
struct GradTable {
  void* data[TENSORS];
  long long size[TENSORS];
  int first[TENSORS + 1];                // first chunk of every tensor; [count] = number of chunks
  unsigned char type[TENSORS];           // 0 bf16, 1 fp16, 2 fp32
  int count;
};
static_assert(sizeof(GradTable<GN_TENSORS>) < 32000, "a launch takes 32764 bytes of parameters");

__host__ __device__ constexpr int width_of(int type) { return type == 2 ? 4 : 2; }
__host__ __device__ constexpr int chunk_of(int type) { return GN_CHUNK_BYTES / width_of(type); }

__device__ __forceinline__ double join(double a, double b, int kind) {
  return kind == 2 ? (a != a || a > b ? a : b) : a + b;        // a maximum that keeps NaN
}
__device__ __forceinline__ double join_block(double v, double* scratch, int kind) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarp = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o), kind);
  __syncthreads();
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  v = lane < nwarp ? scratch[lane] : 0.0;
#pragma unroll
  for (int o = 16; o; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o), kind);
  return v;
}

template <typename Table>
__device__ __forceinline__ int tensor_of(const Table& t, int chunk) {
  int lo = 0, hi = t.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

template <typename T>
struct Grad;
template <>
struct Grad<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    f[0] = __uint_as_float(r.x), f[1] = __uint_as_float(r.y), f[2] = __uint_as_float(r.z), f[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <>
struct Grad<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16(v); }
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
};
template <>
struct Grad<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half(v); }
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
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
};

// A chunk of a tensor: the values before its first 16-byte boundary, vectors, the values after the last.
template <typename T>
struct Span {
  T* p;
  int head, vectors, extra;
  __device__ __forceinline__ Span(void* data, long long size, long long at) : p(static_cast<T*>(data) + at) {
    const int n = static_cast<int>(min(static_cast<long long>(chunk_of(sizeof(T) == 4 ? 2 : 0)), size - at));
    head = min(n, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / static_cast<int>(sizeof(T)));
    vectors = (n - head) / Grad<T>::N;
    extra = n - vectors * Grad<T>::N;
  }
  __device__ __forceinline__ uint4* body() const { return reinterpret_cast<uint4*>(p + head); }
  __device__ __forceinline__ T& lone(int i) const { return p[i < head ? i : i + vectors * Grad<T>::N]; }
};

template <typename T, int KIND>
__device__ __forceinline__ double span_norm(const Span<T>& c) {
  const uint4* body = c.body();
  uint4 r[GN_FLIGHT];
#pragma unroll
  for (int j = 0; j < GN_FLIGHT; ++j) {
    const int i = static_cast<int>(threadIdx.x) + j * GN_THREADS;
    r[j] = i < c.vectors ? __ldg(body + i) : make_uint4(0, 0, 0, 0);
  }
  float alone = 0.f;
  if (static_cast<int>(threadIdx.x) < c.extra) alone = fabsf(Grad<T>::get(c.lone(threadIdx.x)));
  if (KIND == 2) {
    float m = alone;
#pragma unroll
    for (int j = 0; j < GN_FLIGHT; ++j) {
      float f[Grad<T>::N];
      Grad<T>::unpack(r[j], f);
#pragma unroll
      for (int e = 0; e < Grad<T>::N; ++e) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(f[e])));
    }
    return m;
  }
  uint64_t acc = pack_f32x2(KIND == 0 ? alone * alone : alone, 0.f);
#pragma unroll
  for (int j = 0; j < GN_FLIGHT; ++j) {
    float f[Grad<T>::N];
    Grad<T>::unpack(r[j], f);
#pragma unroll
    for (int e = 0; e < Grad<T>::N; e += 2) {
      if (KIND == 0) {
        const uint64_t v = pack_f32x2(f[e], f[e + 1]);
        acc = fma_f32x2(v, v, acc);
      } else {
        acc = add_f32x2(acc, pack_f32x2(fabsf(f[e]), fabsf(f[e + 1])));
      }
    }
  }
  const float2 two = unpack_f32x2(acc);
  const float s = two.x + two.y;
  if (s <= 1e37f && s >= 1e-30f) return s;
  uint32_t any = __float_as_uint(alone);
#pragma unroll
  for (int j = 0; j < GN_FLIGHT; ++j) any |= r[j].x | r[j].y | r[j].z | r[j].w;
  if ((any & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu)) == 0) return 0.0;      // (-0 and 0)
  double wide = KIND == 0 ? static_cast<double>(alone) * alone : alone;
#pragma unroll
  for (int j = 0; j < GN_FLIGHT; ++j) {
    float f[Grad<T>::N];
    Grad<T>::unpack(r[j], f);
#pragma unroll 1
    for (int e = 0; e < Grad<T>::N; ++e) wide += KIND == 0 ? static_cast<double>(f[e]) * f[e] : fabs(static_cast<double>(f[e]));
  }
  return wide;
}

// KIND: 0 squares, 1 absolute values, 2 their maximum.  Every block leaves one value.
template <typename Table, int KIND>
__global__ void __launch_bounds__(GN_THREADS) grad_norm_kernel(const __grid_constant__ Table t, double* __restrict__ partial) {
  __shared__ double scratch[32];
  double s = 0.0;
  for (int c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
    const int k = tensor_of(t, c), type = t.type[k];
    const long long at = static_cast<long long>(c - t.first[k]) * chunk_of(type);
    const double v = type == 0   ? span_norm<__nv_bfloat16, KIND>(Span<__nv_bfloat16>(t.data[k], t.size[k], at))
                     : type == 1 ? span_norm<__half, KIND>(Span<__half>(t.data[k], t.size[k], at))
                                 : span_norm<float, KIND>(Span<float>(t.data[k], t.size[k], at));
    s = join(v, s, KIND);
  }
  s = join_block(s, scratch, KIND);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__global__ void __launch_bounds__(1024) grad_norm_finish_kernel(const double* __restrict__ partial, int n, int kind,
                                                                float* __restrict__ norm) {
  __shared__ double scratch[32];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) s = join(partial[i], s, kind);
  s = join_block(s, scratch, kind);
  if (threadIdx.x == 0) *norm = static_cast<float>(kind == 0 ? sqrt(s) : s);
}

template <typename T>
__device__ __forceinline__ void span_scale(const Span<T>& c, float factor) {
  uint4* body = c.body();
  uint4 r[GN_FLIGHT];
#pragma unroll
  for (int j = 0; j < GN_FLIGHT; ++j) {
    const int i = static_cast<int>(threadIdx.x) + j * GN_THREADS;
    if (i < c.vectors) r[j] = body[i];
  }
#pragma unroll
  for (int j = 0; j < GN_FLIGHT; ++j) {
    const int i = static_cast<int>(threadIdx.x) + j * GN_THREADS;
    if (i >= c.vectors) break;
    float f[Grad<T>::N];
    Grad<T>::unpack(r[j], f);
#pragma unroll
    for (int e = 0; e < Grad<T>::N; ++e) f[e] *= factor;
    body[i] = Grad<T>::pack(f);
  }
  if (static_cast<int>(threadIdx.x) < c.extra) c.lone(threadIdx.x) = Grad<T>::put(Grad<T>::get(c.lone(threadIdx.x)) * factor);
}

// The coefficient stays fp32 and the product is rounded once.  Last chunks first: the norm has left them in the L2.
template <typename Table>
__global__ void __launch_bounds__(GN_THREADS) grad_scale_kernel(const __grid_constant__ Table t, const float* __restrict__ norm,
                                                                float limit) {
  const float f = limit / (*norm + 1e-6f);
  if (f >= 1.f) return;                    // (NaN goes on: it makes every gradient NaN)
  for (int c = t.first[t.count] - 1 - static_cast<int>(blockIdx.x); c >= 0; c -= gridDim.x) {
    const int k = tensor_of(t, c), type = t.type[k];
    const long long at = static_cast<long long>(c - t.first[k]) * chunk_of(type);
    if (type == 0) span_scale(Span<__nv_bfloat16>(t.data[k], t.size[k], at), f);
    else if (type == 1) span_scale(Span<__half>(t.data[k], t.size[k], at), f);
    else span_scale(Span<float>(t.data[k], t.size[k], at), f);
  }
}

// Calls launch(table) for every run of tensors that fits a launch.  -1: a bad argument, -4: more chunks than a launch can count.
template <typename Table, typename F>
static int for_tables(void* const* data, const long long* size, const unsigned char* type, int count, F&& launch) {
  constexpr int most = sizeof(Table::type);
  Table t;
  for (int at = 0; at < count;) {
    t.count = 0;
    long long chunks = 0;
    for (; at < count && t.count < most; ++at) {
      if (size[at] < 0 || type[at] > 2) return -1;
      if (size[at] == 0) continue;
      const long long more = (size[at] + chunk_of(type[at]) - 1) / chunk_of(type[at]);
      if (chunks + more > 0x40000000ll) {
        if (t.count == 0) return -4;
        break;
      }
      t.data[t.count] = data[at];
      t.size[t.count] = size[at];
      t.type[t.count] = type[at];
      t.first[t.count++] = static_cast<int>(chunks);
      chunks += more;
    }
    t.first[t.count] = static_cast<int>(chunks);
    if (t.count) launch(t);
  }
  return static_cast<int>(cudaGetLastError());
}
template <typename F>
static int for_lists(void* const* data, const long long* size, const unsigned char* type, int count, F&& launch) {
  return count <= GN_FEW ? for_tables<GradTable<GN_FEW>>(data, size, type, count, launch)
                         : for_tables<GradTable<GN_TENSORS>>(data, size, type, count, launch);
}

static int grad_blocks() { return sm_count() * 4; }

}  // namespace ts

using namespace ts;

TS_DEFINE_ERROR_API(ts_gradnorm)

// Number of doubles that ts_grad_norm needs as workspace: `elements` is the sum of the sizes.
extern "C" long long ts_grad_norm_workspace(int count, long long elements) {
  return (count / GN_TENSORS + 2 + elements / (0x20000000ll * chunk_of(2))) * static_cast<long long>(grad_blocks());
}

// norm: one float.  Tensors that share memory are refused (-2): blocks that scale them would race.
extern "C" int ts_grad_norm(void* const* data, const long long* size, const unsigned char* type, int count, int kind, double* workspace,
                            float* norm, void* stream) {
  if (count <= 0 || kind < 0 || kind > 2) return -1;
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;
  try {
    spans.reserve(count);
  } catch (...) {
    return -3;
  }
  for (int i = 0; i < count; ++i) {
    if (type[i] > 2) return -1;
    const uintptr_t p = reinterpret_cast<uintptr_t>(data[i]);
    if (size[i] > 0) spans.emplace_back(p, p + size[i] * width_of(type[i]));
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].first < spans[i - 1].second) return -2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int used = 0;
  const int rc = for_lists(data, size, type, count, [&](const auto& t) {
    using Table = std::remove_cv_t<std::remove_reference_t<decltype(t)>>;
    const int blocks = std::min(grad_blocks(), t.first[t.count]);
    if (kind == 0) grad_norm_kernel<Table, 0><<<blocks, GN_THREADS, 0, st>>>(t, workspace + used);
    else if (kind == 1) grad_norm_kernel<Table, 1><<<blocks, GN_THREADS, 0, st>>>(t, workspace + used);
    else grad_norm_kernel<Table, 2><<<blocks, GN_THREADS, 0, st>>>(t, workspace + used);
    used += blocks;
  });
  if (rc) return rc;
  grad_norm_finish_kernel<<<1, 1024, 0, st>>>(workspace, used, kind, norm);
  return static_cast<int>(cudaGetLastError());
}

extern "C" int ts_grad_scale(void* const* data, const long long* size, const unsigned char* type, int count, const float* norm, float limit,
                             void* stream) {
  if (count <= 0) return -1;
  return for_lists(data, size, type, count, [&](const auto& t) {
    grad_scale_kernel<<<std::min(grad_blocks(), t.first[t.count]), GN_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(t, norm, limit);
  });
}
