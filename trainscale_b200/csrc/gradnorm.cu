// The global norm of a list of gradients, and their scaling by min(1, limit / (norm + 1e-6)).
//
// The list goes to the kernels by value (a launch takes up to 32 KB of parameters), so that nothing is copied to the device or
// kept between calls.  Norms: 2 (sqrt of the sum of squares), 1, inf.  Sums are fp64 and made in an order that depends on the
// sizes alone.
#include <algorithm>
#include <vector>

#include "common.cuh"
#include "host_common.h"

namespace ts {

constexpr int GN_THREADS = 512;
constexpr int GN_TENSORS = 1024;          // of one launch
constexpr long long GN_CHUNK = 32768;     // elements of a block's turn

struct GradTable {
  void* data[GN_TENSORS];
  long long size[GN_TENSORS];
  int first[GN_TENSORS + 1];              // first chunk of every tensor; [count] = number of chunks
  unsigned char type[GN_TENSORS];         // 0 bf16, 1 fp16, 2 fp32
  int count;
};
static_assert(sizeof(GradTable) < 32000, "a launch takes 32764 bytes of parameters");

__device__ __forceinline__ double sum_all(double v, double* scratch, bool largest) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarp = blockDim.x >> 5;
  auto join = [&](double a, double b) { return largest ? (a != a || a > b ? a : b) : a + b; };     // a maximum that keeps NaN
#pragma unroll
  for (int o = 16; o; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  v = lane < nwarp ? scratch[lane] : 0.0;
#pragma unroll
  for (int o = 16; o; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__device__ __forceinline__ float gn_f32(float v) { return v; }
__device__ __forceinline__ float gn_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float gn_f32(__half v) { return __half2float(v); }

__device__ __forceinline__ int tensor_of(const GradTable& t, int chunk) {
  int lo = 0, hi = t.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

template <typename T>
__device__ __forceinline__ double chunk_norm(const T* p, long long n, int kind) {
  double s = 0.0;
  for (long long i = threadIdx.x; i < n; i += GN_THREADS) {
    const double v = fabs(static_cast<double>(gn_f32(p[i])));
    s = kind == 0 ? s + v * v : kind == 1 ? s + v : (v != v || v > s ? v : s);
  }
  return s;
}

// kind: 0 squares, 1 absolute values, 2 their maximum.  Every block leaves one value.
__global__ void __launch_bounds__(GN_THREADS) grad_norm_kernel(const __grid_constant__ GradTable t, int kind, double* __restrict__ partial) {
  __shared__ double scratch[32];
  double s = 0.0;
  for (int c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
    const int k = tensor_of(t, c);
    const long long at = (c - t.first[k]) * GN_CHUNK, n = min(GN_CHUNK, t.size[k] - at);
    const double v = t.type[k] == 0   ? chunk_norm(static_cast<const __nv_bfloat16*>(t.data[k]) + at, n, kind)
                     : t.type[k] == 1 ? chunk_norm(static_cast<const __half*>(t.data[k]) + at, n, kind)
                                      : chunk_norm(static_cast<const float*>(t.data[k]) + at, n, kind);
    s = kind == 2 ? (v != v || v > s ? v : s) : s + v;
  }
  s = sum_all(s, scratch, kind == 2);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__global__ void __launch_bounds__(1024) grad_norm_finish_kernel(const double* __restrict__ partial, int n, int kind, float* __restrict__ norm) {
  __shared__ double scratch[32];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) s = kind == 2 ? (partial[i] != partial[i] || partial[i] > s ? partial[i] : s) : s + partial[i];
  s = sum_all(s, scratch, kind == 2);
  if (threadIdx.x == 0) *norm = static_cast<float>(kind == 0 ? sqrt(s) : s);
}

__device__ __forceinline__ void scale_chunk(float* p, long long n, float c) {
  for (long long i = threadIdx.x; i < n; i += GN_THREADS) p[i] *= c;
}
__device__ __forceinline__ void scale_chunk(__nv_bfloat16* p, long long n, float c) {
  for (long long i = threadIdx.x; i < n; i += GN_THREADS) p[i] = __float2bfloat16(__bfloat162float(p[i]) * c);
}
__device__ __forceinline__ void scale_chunk(__half* p, long long n, float c) {
  for (long long i = threadIdx.x; i < n; i += GN_THREADS) p[i] = __float2half(__half2float(p[i]) * c);
}

// The coefficient stays fp32 and the product is rounded once.
__global__ void __launch_bounds__(GN_THREADS) grad_scale_kernel(const __grid_constant__ GradTable t, const float* __restrict__ norm, float limit) {
  const float c = limit / (*norm + 1e-6f);
  if (c >= 1.f) return;                    // (NaN goes on: it makes every gradient NaN)
  for (int i = blockIdx.x; i < t.first[t.count]; i += gridDim.x) {
    const int k = tensor_of(t, i);
    const long long at = (i - t.first[k]) * GN_CHUNK, n = min(GN_CHUNK, t.size[k] - at);
    if (t.type[k] == 0) scale_chunk(static_cast<__nv_bfloat16*>(t.data[k]) + at, n, c);
    else if (t.type[k] == 1) scale_chunk(static_cast<__half*>(t.data[k]) + at, n, c);
    else scale_chunk(static_cast<float*>(t.data[k]) + at, n, c);
  }
}

// Calls launch(table) for every run of tensors that fits a launch.  -1: a bad argument, -4: more chunks than a launch can count.
template <typename F>
static int for_tables(void* const* data, const long long* size, const unsigned char* type, int count, F&& launch) {
  GradTable t;
  for (int at = 0; at < count;) {
    t.count = 0;
    long long chunks = 0;
    for (; at < count && t.count < GN_TENSORS; ++at) {
      if (size[at] < 0 || type[at] > 2) return -1;
      if (size[at] == 0) continue;
      const long long more = (size[at] + GN_CHUNK - 1) / GN_CHUNK;
      if (chunks + more > 0x7fffffffll) {
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

static int grad_blocks() { return sm_count() * 4; }

}  // namespace ts

using namespace ts;

TS_DEFINE_ERROR_API(ts_gradnorm)

// Number of doubles that ts_grad_norm needs as workspace for `count` tensors of `elements` elements in all.
extern "C" long long ts_grad_norm_workspace(int count, long long elements) {
  return (count / GN_TENSORS + 2 + elements / (GN_CHUNK * 0x7fffffffll)) * static_cast<long long>(grad_blocks());
}

// norm: one float.  Tensors that share memory are refused (-2): blocks that scale them would race.
extern "C" int ts_grad_norm(void* const* data, const long long* size, const unsigned char* type, int count, int kind, double* workspace,
                            float* norm, void* stream) {
  if (count <= 0 || kind < 0 || kind > 2) return -1;
  static const int width[3] = {2, 2, 4};
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;
  try {
    spans.reserve(count);
  } catch (...) {
    return -3;
  }
  for (int i = 0; i < count; ++i) {
    if (type[i] > 2) return -1;
    const uintptr_t p = reinterpret_cast<uintptr_t>(data[i]);
    if (size[i] > 0) spans.emplace_back(p, p + size[i] * width[type[i]]);
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].first < spans[i - 1].second) return -2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int used = 0;
  const int rc = for_tables(data, size, type, count, [&](const GradTable& t) {
    const int blocks = std::min(grad_blocks(), t.first[t.count]);
    grad_norm_kernel<<<blocks, GN_THREADS, 0, st>>>(t, kind, workspace + used);
    used += blocks;
  });
  if (rc) return rc;
  grad_norm_finish_kernel<<<1, 1024, 0, st>>>(workspace, used, kind, norm);
  return static_cast<int>(cudaGetLastError());
}

extern "C" int ts_grad_scale(void* const* data, const long long* size, const unsigned char* type, int count, const float* norm, float limit,
                             void* stream) {
  if (count <= 0) return -1;
  return for_tables(data, size, type, count, [&](const GradTable& t) {
    grad_scale_kernel<<<std::min(grad_blocks(), t.first[t.count]), GN_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(t, norm, limit);
  });
}
