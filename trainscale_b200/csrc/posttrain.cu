// Losses over token log-probabilities [rows][T], with their gradients: the clipped policy loss with a KL term, and the losses of
// (chosen, rejected) pairs.
//
// Policy, for a token of weight m (its mask) in a row of advantage a:
//   r = e^(logp - old),  clipped = a > 0 ? r > 1 + high : a < 0 and r < 1 - low,  d = ref - logp
//   token = -a (clipped ? bound : r) + beta (e^d - 1 - d),  d token / d logp = (clipped ? 0 : -a r) - beta (e^d - 1)
//   loss  = sum m w token,  w = 1 / (rows sum_row m), 1 / sum m or 1 / (rows length); the sums of m are at least 1
// A token's gradient jumps at a bound, so the side that it is on is decided by logp - old without rounding (two fp32 numbers
// whose sum is the difference).  e^d - 1 - d is a power series near zero, where the difference would cancel.  Sums of four or
// eight tokens are fp32, sums of those fp64, in an order that depends on the sizes alone.
//
// Pairs, rows p (chosen) and P + p (rejected), of scores s = sum m (logp - ref), divided by max(sum m, 1) where asked:
//   x = s_p - s_(P + p),  q = beta x - gamma
//   sigmoid -(1 - eps) log sigma(q) - eps log sigma(-q);  robust: the same with + eps, / (1 - 2 eps);  hinge max(0, 1 - q);
//   ipo (x - 1 / (2 beta))^2;  and nll * the mean of -logp over the chosen row's tokens
// The scores are long sums whose difference decides: they, and all that is done per pair, are fp64.
//
// Gradients leave with the loss, for an upstream gradient of one.  Where it turns out to be another, fp32 gradients are
// multiplied by it; 16-bit ones, which that would round twice, are computed again (`Upstream`).
//
// Bounds: latencies (DRAM 26 % busy, issue slots 58 %, special functions 12 %): a thread has one vector in flight and asks for its inputs
// when its mask has come.  512 x 16384 tokens with a KL
// term, half of them masked: 10 us to count and 36 for the rest (168 MB without the masked tokens' would be 26 at the memory's
// rate); reading a masked token's inputs cost 42.  160 pairs of 16384 tokens 18 us (84 MB: 13), 600 of them 65 (255 MB: 39); a
// block's worth of fp64 exponentials instead of one thread's cost 3 us there.  Small calls are one or two launches of 5 to 9 us,
// behind 110 us of Python, half of which is what any autograd node takes there and back.
#include <cooperative_groups.h>

#include "common.cuh"
#include "host_common.h"

namespace ts {

namespace cg = cooperative_groups;

constexpr int PT_THREADS = 256;

template <typename T, int N>
struct alignas(sizeof(T) * N) Few {
  T v[N];
};
__device__ __forceinline__ float pt_f32(float v) { return v; }
__device__ __forceinline__ float pt_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float pt_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float pt_f32(unsigned char v) { return static_cast<float>(v); }
__device__ __forceinline__ float pt_f32(int v) { return static_cast<float>(v); }
__device__ __forceinline__ float pt_f32(long long v) { return static_cast<float>(v); }
template <typename T>
__device__ __forceinline__ T pt_from(float v);
template <>
__device__ __forceinline__ float pt_from<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 pt_from<__nv_bfloat16>(float v) { return __float2bfloat16(v); }
template <>
__device__ __forceinline__ __half pt_from<__half>(float v) { return __float2half(v); }

// N consecutive values, aligned to N of them where N > 1.
template <int N, typename T>
__device__ __forceinline__ void fetch(const T* p, float* f) {
  using V = Few<T, N>;
  if constexpr (sizeof(V) <= 16) {
    const V v = *reinterpret_cast<const V*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = pt_f32(v.v[i]);
  } else {
    fetch<N / 2>(p, f);
    fetch<N / 2>(p + N / 2, f + N / 2);
  }
}
template <int N, typename T>
__device__ __forceinline__ void put(T* p, const float* f) {
  Few<T, N> v;
#pragma unroll
  for (int i = 0; i < N; ++i) v.v[i] = pt_from<T>(f[i]);
  *reinterpret_cast<Few<T, N>*>(p) = v;
}

// N values of a mask.  They are loaded as they are and become fp32 when they are needed: a branch on their type that waited for
// them would keep the other loads waiting too.
template <int N>
struct MaskBits {
  uint32_t w[2 * N];
};
template <typename T, int N>
__device__ __forceinline__ float mask_value(const MaskBits<N>& b, int i) {
  if constexpr (sizeof(T) == 8)
    return static_cast<float>(static_cast<long long>(b.w[2 * i] | static_cast<unsigned long long>(b.w[2 * i + 1]) << 32));
  constexpr int in_word = 4 / sizeof(T) > 0 ? 4 / sizeof(T) : 1;
  const uint32_t word = b.w[i / in_word] >> (i % in_word * (32 / in_word));
  if constexpr (sizeof(T) == 1) return static_cast<float>(word & 0xff);
  if constexpr (sizeof(T) == 2) {
    const unsigned short half = static_cast<unsigned short>(word);
    return pt_f32(*reinterpret_cast<const T*>(&half));
  }
  return pt_f32(*reinterpret_cast<const T*>(&word));
}

struct Mask {
  const void* p;
  long long stride;                      // elements between rows
  int kind;                              // 0 bool / uint8, 1 int32, 2 int64, 3 fp32, 4 bf16, 5 fp16
  int shift;                             // log2 of their bytes
  template <int N>
  __device__ __forceinline__ void load(long long i, MaskBits<N>& b) const {
    const char* at = static_cast<const char*>(p) + (i << shift);
    if (shift == 0) {
      if (N == 4) b.w[0] = *reinterpret_cast<const uint32_t*>(at);
      else b.w[0] = *reinterpret_cast<const unsigned char*>(at);
    } else if (shift == 1) {
      if (N == 4) {
        const uint2 v = *reinterpret_cast<const uint2*>(at);
        b.w[0] = v.x, b.w[1] = v.y;
      } else {
        b.w[0] = *reinterpret_cast<const unsigned short*>(at);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (j == 1 && shift == 2) break;
        if (N == 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(at + 16 * j);
          b.w[4 * j] = v.x, b.w[4 * j + 1] = v.y, b.w[4 * j + 2] = v.z, b.w[4 * j + 3] = v.w;
        } else {
          b.w[j] = *reinterpret_cast<const uint32_t*>(at + 4 * j);
        }
      }
    }
  }
  template <typename T, int N>
  static __device__ __forceinline__ void values_of(const MaskBits<N>& b, float* f) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = mask_value<T, N>(b, i);
  }
  template <int N>
  __device__ __forceinline__ void values(const MaskBits<N>& b, float* f) const {
    switch (kind) {
      case 0: return values_of<unsigned char, N>(b, f);
      case 1: return values_of<int, N>(b, f);
      case 2: return values_of<long long, N>(b, f);
      case 3: return values_of<float, N>(b, f);
      case 4: return values_of<__nv_bfloat16, N>(b, f);
      default: return values_of<__half, N>(b, f);
    }
  }
  template <int N>
  __device__ __forceinline__ void get(long long i, float* f) const {
    MaskBits<N> b;
    load<N>(i, b);
    values<N>(b, f);
  }
};

// What flows into the loss: nothing known yet (null), or a factor of the gradient; `redo`: also where it is one.
struct Upstream {
  const float* factor;
  int redo;
  __device__ __forceinline__ bool done() const { return factor && !redo && *factor == 1.f; }
  __device__ __forceinline__ float get() const { return factor ? *factor : 1.f; }
};

// Sums over the block in a fixed order; every thread gets them.
template <int N>
__device__ __forceinline__ void block_sums(double* v, double (*scratch)[N]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarp = blockDim.x >> 5;
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int o = 16; o; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  __syncthreads();
  if (lane == 0)
#pragma unroll
    for (int k = 0; k < N; ++k) scratch[warp][k] = v[k];
  __syncthreads();
  if (threadIdx.x < N) {
    double t = scratch[0][threadIdx.x];
    for (int w = 1; w < nwarp; ++w) t += scratch[w][threadIdx.x];
    scratch[0][threadIdx.x] = t;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = scratch[0][k];
}

// ---------------------------------------------------------------------------------------------------
// Clipped policy loss.  Tokens are numbered row after row; a block takes a run of them, a thread VEC at a time.
// ---------------------------------------------------------------------------------------------------
constexpr int POLICY_PER_SM = 4;         // blocks of an SM
constexpr int POLICY_SUMS = 5;           // loss, kl m, clipped m, ratio m, m
constexpr int POLICY_SPLIT = 8;          // most blocks that count a row
// Tokens of a row that a warp counts (by warps and by blocks: 4096 x 128 12.6 and 18.3 us a call, 512 x 1024 12.1 and 12.9).
constexpr int POLICY_SHORT = 1024;
// Tokens that one block takes by itself, in one launch (8 x 64: 5.4 us, in two launches 7.8; 8 x 1024: 8.9 and 9.0; 16 x 1024:
// 13.1 and 8.1).
constexpr int POLICY_ALONE = 8192;
constexpr int POLICY_ALONE_THREADS = 1024, POLICY_ALONE_ROWS = 4096;

struct Policy {
  const void *logp, *old, *ref;
  long long s_logp, s_old, s_ref;        // elements between rows
  const float* advantages;               // [rows] or [rows][T]
  Mask mask;
  long long rows, T, tokens, run;        // tokens = rows T; run: tokens of a block
  double constant;                       // 1 / (rows length) of reduction 2
  float bound_low[2], bound_high[2];     // ln(1 - low) and ln(1 + high), each as a sum of two
  float low, high, beta;                 // 1 - low, 1 + high
  int per_token, reduction;              // 0 rows' means, 1 all tokens, 2 a constant
  int flat;                              // rows follow one another without gaps in every tensor
};

// e^d - 1 - d and e^d - 1
__device__ __forceinline__ float exp_rest(float d, float* less) {
  const float series = 0.5f + d * (1.f / 6.f + d * (1.f / 24.f + d * (1.f / 120.f + d * (1.f / 720.f + d * (1.f / 5040.f +
                       d * (1.f / 40320.f + d * (1.f / 362880.f)))))));
  const bool near = fabsf(d) < 0.5f;
  const float rest = d * d * series, e = expf(d) - 1.f;
  *less = near ? d + rest : e;
  return near ? rest : e - d;
}

// Where a thread's next tokens are: stepping by a block's width costs no division.
struct Place {
  int row, t, T, rows, rest;
  __device__ __forceinline__ Place(long long token, int width, long long length)
      : row(static_cast<int>(token / length)), t(static_cast<int>(token - row * length)), T(static_cast<int>(length)),
        rows(width / static_cast<int>(length)), rest(width - rows * static_cast<int>(length)) {}
  __device__ __forceinline__ void step() {
    row += rows;
    t += rest;
    if (t >= T) t -= T, ++row;
  }
  __device__ __forceinline__ long long in(long long stride) const { return row * stride + t; }
};

// A thread's part of the sum of the mask's values [begin, end), one of `threads`; four vectors in flight.
template <typename M, int VEC>
__device__ __forceinline__ double sum_values(const M* p, long long begin, long long end, int thread, int threads) {
  const long long width = static_cast<long long>(threads) * VEC;
  double n = 0.0;
  for (long long i = begin + static_cast<long long>(thread) * VEC; i < end; i += 4 * width) {
    float m[4][VEC], s = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) m[j][e] = 0.f;
      if (i + j * width < end) fetch<VEC>(p + i + j * width, m[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += m[j][e];
    n += s;
  }
  return n;
}

// Sum of the mask over tokens [begin, end), which lie in one row or are `flat`.
template <int VEC>
__device__ __forceinline__ double mask_run(const Policy& a, long long begin, long long end, int thread, int threads) {
  const long long at = a.flat ? 0 : begin / a.T * (a.mask.stride - a.T);
  switch (a.mask.kind) {
    case 0: return sum_values<unsigned char, VEC>(static_cast<const unsigned char*>(a.mask.p) + at, begin, end, thread, threads);
    case 1: return sum_values<int, VEC>(static_cast<const int*>(a.mask.p) + at, begin, end, thread, threads);
    case 2: return sum_values<long long, VEC>(static_cast<const long long*>(a.mask.p) + at, begin, end, thread, threads);
    case 3: return sum_values<float, VEC>(static_cast<const float*>(a.mask.p) + at, begin, end, thread, threads);
    case 4: return sum_values<__nv_bfloat16, VEC>(static_cast<const __nv_bfloat16*>(a.mask.p) + at, begin, end, thread, threads);
    default: return sum_values<__half, VEC>(static_cast<const __half*>(a.mask.p) + at, begin, end, thread, threads);
  }
}

// The same of any tokens.
template <int VEC>
__device__ __forceinline__ double mask_sum(const Policy& a, long long begin, long long end) {
  if (a.flat) return mask_run<VEC>(a, begin, end, threadIdx.x, blockDim.x);
  const int width = static_cast<int>(blockDim.x) * VEC;
  long long i = begin + static_cast<long long>(threadIdx.x) * VEC;
  double n = 0.0;
  for (Place at(i, width, a.T); i < end; i += width, at.step()) {
    float m[VEC], s = 0.f;
    a.mask.get<VEC>(at.in(a.mask.stride), m);
#pragma unroll
    for (int e = 0; e < VEC; ++e) s += m[e];
    n += s;
  }
  return n;
}

// Gradient and sums of tokens [begin, end).  Weights: of the row (`weights`), or the same for all.
template <typename T, int VEC, bool FLAT>
__device__ __forceinline__ void policy_tokens(const Policy& a, long long begin, long long end, const float* weights, float uniform,
                                              float factor, T* __restrict__ grad, double* sums) {
  const int width = static_cast<int>(blockDim.x) * VEC;
  const bool whole = a.T % VEC == 0;     // a thread's tokens are in one row
  long long next = begin + static_cast<long long>(threadIdx.x) * VEC;
  Place ahead(next, width, a.T);
  MaskBits<VEC> coming;                  // the mask is read a step ahead: tokens that it leaves out are not read at all
  if (next < end) a.mask.load<VEC>(FLAT ? next : ahead.in(a.mask.stride), coming);
  while (next < end) {
    const long long i = next;
    const Place at = ahead;
    float logp[VEC], old[VEC], ref[VEC], m[VEC], adv[VEC], w[VEC], slope[VEC], part[POLICY_SUMS] = {};
    bool any = false;
    a.mask.values<VEC>(coming, m);
#pragma unroll
    for (int e = 0; e < VEC; ++e) any |= m[e] != 0.f, slope[e] = 0.f;
    next += width;
    ahead.step();
    if (next < end) a.mask.load<VEC>(FLAT ? next : ahead.in(a.mask.stride), coming);
    if (!any) {
      if (grad) put<VEC>(grad + i, slope);
      continue;
    }
    fetch<VEC>(static_cast<const T*>(a.logp) + (FLAT ? i : at.in(a.s_logp)), logp);
    fetch<VEC>(static_cast<const T*>(a.old) + (FLAT ? i : at.in(a.s_old)), old);
    if (a.ref) fetch<VEC>(static_cast<const T*>(a.ref) + (FLAT ? i : at.in(a.s_ref)), ref);
    if (whole) {
      const float row_w = weights ? weights[at.row] : uniform, row_adv = a.per_token ? 0.f : a.advantages[at.row];
#pragma unroll
      for (int e = 0; e < VEC; ++e) w[e] = row_w, adv[e] = row_adv;
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int row = at.row + (at.t + e) / at.T;
        w[e] = weights ? weights[row] : uniform;
        adv[e] = a.per_token ? 0.f : a.advantages[row];
      }
    }
    if (a.per_token) fetch<VEC>(a.advantages + i, adv);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      // whatever a masked token holds reaches nothing
      const bool used = m[e] != 0.f;
      const float g = used ? adv[e] : 0.f, x = used ? logp[e] : 0.f, y = used ? old[e] : 0.f;
      const float moved = x - y;
      bool above = moved > a.bound_high[0], below = moved < a.bound_low[0];
      if (moved == a.bound_high[0] || moved == a.bound_low[0]) {
        // x - y = moved + lost exactly
        const float back = moved - x, lost = (x - (moved - back)) - (y + back);
        above = moved == a.bound_high[0] && lost > a.bound_high[1];
        below = moved == a.bound_low[0] && lost < a.bound_low[1];
      }
      const bool clipped = g > 0.f ? above : g < 0.f && below;
      const float ratio = expf(moved);
      // (0 * inf: a ratio that overflows has no say where the advantage is zero)
      const float gain = g == 0.f && ratio == INFINITY ? 0.f : g * (clipped ? (g > 0.f ? a.high : a.low) : ratio);
      float token = -gain;
      slope[e] = clipped ? 0.f : -gain;
      if (a.ref) {
        float less;
        const float kl = exp_rest(used ? ref[e] - x : 0.f, &less);
        if (a.beta != 0.f) {             // (0 * inf: a reference that is only looked at has no say)
          token += a.beta * kl;
          slope[e] -= a.beta * less;
        }
        part[1] += m[e] * kl;
      }
      const float mw = m[e] * w[e];
      part[0] += mw * token;
      part[2] += clipped ? m[e] : 0.f;
      part[3] += m[e] * ratio;
      part[4] += m[e];
      slope[e] *= mw * factor;
    }
#pragma unroll
    for (int k = 0; k < POLICY_SUMS; ++k) sums[k] += part[k];
    if (grad) put<VEC>(grad + i, slope);
  }
}

__device__ __forceinline__ void policy_results(const double* sums, float* loss, float* stats) {
  *loss = static_cast<float>(sums[0]);
  if (stats)
    for (int k = 1; k < 4; ++k) stats[k - 1] = static_cast<float>(sums[k] / fmax(sums[4], 1.0));
}

// What the tokens weigh: weights [rows] (reduction 0, a warp, a block or a cluster per row), sums of the mask by block (reduction 1); and
// the counter that tells the next kernel's last block.
template <int VEC>
__global__ void __launch_bounds__(PT_THREADS) policy_count_kernel(Policy a, float* __restrict__ weights, double* __restrict__ counts,
                                                                  unsigned* __restrict__ ticket, Upstream up) {
  __shared__ double scratch[32][1];
  __shared__ double by_block[POLICY_SPLIT];
  cg::cluster_group cluster = cg::this_cluster();
  if (up.done()) return;
  if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
  if (a.reduction == 2) return;
  const int parts = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  if (a.reduction == 1) {
    double n[1] = {mask_sum<VEC>(a, blockIdx.x * a.run, min(a.tokens, (blockIdx.x + 1ll) * a.run))};
    block_sums<1>(n, scratch);
    if (threadIdx.x == 0) counts[blockIdx.x] = n[0];
    return;
  }
  // (a row that starts between vectors is counted token by token)
  const bool vectors = a.T % VEC == 0;
  auto weight = [&](double n) { return static_cast<float>(1.0 / (fmax(n, 1.0) * static_cast<double>(a.rows))); };
  if (a.T <= POLICY_SHORT) {
    const long long row = blockIdx.x * static_cast<long long>(PT_THREADS / 32) + (threadIdx.x >> 5);
    if (row >= a.rows) return;
    const int lane = threadIdx.x & 31;
    double n = vectors ? mask_run<VEC>(a, row * a.T, (row + 1) * a.T, lane, 32) : mask_run<1>(a, row * a.T, (row + 1) * a.T, lane, 32);
#pragma unroll
    for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    if (lane == 0) weights[row] = weight(n);
    return;
  }
  if (parts > 1) cluster.barrier_arrive();      // (no block writes to another's shared memory before that one has begun)
  const long long row = blockIdx.x / parts, part = (a.T / VEC + parts - 1) / parts * VEC;
  const long long begin = row * a.T + rank * part, end = rank == parts - 1 ? (row + 1) * a.T : min((row + 1) * a.T, begin + part);
  double n[1] = {vectors ? mask_run<VEC>(a, begin, end, threadIdx.x, PT_THREADS) : mask_run<1>(a, begin, end, threadIdx.x, PT_THREADS)};
  block_sums<1>(n, scratch);
  if (parts > 1) {
    cluster.barrier_wait();
    if (threadIdx.x == 0) *cluster.map_shared_rank(by_block + rank, 0) = n[0];
    cluster.sync();
    if (rank != 0) return;
    n[0] = 0.0;
    for (int i = 0; i < parts; ++i) n[0] += by_block[i];
  }
  if (threadIdx.x == 0) weights[row] = weight(n[0]);
}

template <typename T, int VEC, bool FLAT>
__global__ void __launch_bounds__(PT_THREADS, POLICY_PER_SM)
    policy_kernel(Policy a, const float* __restrict__ weights, const double* __restrict__ counts, double* __restrict__ partial,
                  unsigned* __restrict__ ticket, T* __restrict__ grad, float* __restrict__ loss, float* __restrict__ stats, Upstream up) {
  __shared__ double scratch[32][POLICY_SUMS];
  __shared__ bool last;
  if (up.done()) return;
  float uniform = static_cast<float>(a.constant);
  if (a.reduction == 1) {
    double n[POLICY_SUMS] = {};
    for (unsigned i = threadIdx.x; i < gridDim.x; i += PT_THREADS) n[0] += counts[i];
    block_sums<POLICY_SUMS>(n, scratch);
    uniform = static_cast<float>(1.0 / fmax(n[0], 1.0));
  }
  double sums[POLICY_SUMS] = {};
  const long long begin = blockIdx.x * a.run;
  policy_tokens<T, VEC, FLAT>(a, begin, min(a.tokens, begin + a.run), a.reduction == 0 ? weights : nullptr, uniform, up.get(), grad, sums);
  if (!loss) return;
  block_sums<POLICY_SUMS>(sums, scratch);
  if (threadIdx.x == 0) {
#pragma unroll
    for (int k = 0; k < POLICY_SUMS; ++k) __stcg(partial + k * static_cast<long long>(gridDim.x) + blockIdx.x, sums[k]);
    __threadfence();
    last = atomicAdd(ticket, 1) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
#pragma unroll
  for (int k = 0; k < POLICY_SUMS; ++k) {
    sums[k] = 0.0;
    for (unsigned i = threadIdx.x; i < gridDim.x; i += PT_THREADS) sums[k] += __ldcg(partial + k * static_cast<long long>(gridDim.x) + i);
  }
  block_sums<POLICY_SUMS>(sums, scratch);
  if (threadIdx.x == 0) policy_results(sums, loss, stats);
}

// All of it in one block.
template <typename T, int VEC, bool FLAT>
__global__ void __launch_bounds__(POLICY_ALONE_THREADS) policy_alone_kernel(Policy a, T* __restrict__ grad, float* __restrict__ loss,
                                                                            float* __restrict__ stats, Upstream up) {
  __shared__ double scratch[32][POLICY_SUMS];
  __shared__ float weights[POLICY_ALONE_ROWS];
  if (up.done()) return;
  float uniform = static_cast<float>(a.constant);
  if (a.reduction == 0) {
    const int lanes = a.T >= 32 ? 32 : 1, lane = threadIdx.x % lanes;      // a warp counts a row, or a thread a short one
    for (int r = threadIdx.x / lanes; r < a.rows; r += POLICY_ALONE_THREADS / lanes) {
      double n = 0.0;
      for (long long t = lane; t < a.T; t += lanes) {
        float m;
        a.mask.get<1>(r * a.mask.stride + t, &m);
        n += m;
      }
      if (lanes == 32)
#pragma unroll
        for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
      if (lane == 0) weights[r] = static_cast<float>(1.0 / (fmax(n, 1.0) * static_cast<double>(a.rows)));
    }
    __syncthreads();
  } else if (a.reduction == 1) {
    double n[POLICY_SUMS] = {mask_sum<VEC>(a, 0, a.tokens)};
    block_sums<POLICY_SUMS>(n, scratch);
    uniform = static_cast<float>(1.0 / fmax(n[0], 1.0));
  }
  double sums[POLICY_SUMS] = {};
  policy_tokens<T, VEC, FLAT>(a, 0, a.tokens, a.reduction == 0 ? weights : nullptr, uniform, up.get(), grad, sums);
  if (!loss) return;
  block_sums<POLICY_SUMS>(sums, scratch);
  if (threadIdx.x == 0) policy_results(sums, loss, stats);
}

// grad *= *factor; a factor of one leaves it as it is
__global__ void __launch_bounds__(PT_THREADS) scale_kernel(float* __restrict__ grad, const float* __restrict__ factor, long long n) {
  const float f = *factor;
  if (f == 1.f) return;
  const long long step = gridDim.x * static_cast<long long>(PT_THREADS);
  const long long first = blockIdx.x * static_cast<long long>(PT_THREADS) + threadIdx.x;
  float4* fours = reinterpret_cast<float4*>(grad);
  for (long long i = first; i < n / 4; i += step) {
    const float4 v = fours[i];
    fours[i] = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
  }
  if (first < n % 4) grad[n - 1 - first] *= f;
}

// ---------------------------------------------------------------------------------------------------
// Pairs
// ---------------------------------------------------------------------------------------------------
constexpr int PAIR_SPLIT = 8;            // most blocks of a pair
constexpr int PAIR_TOKENS = 2048;        // tokens of a row that are worth a block

struct Pairs {
  const void *logp, *ref;
  long long s_logp, s_ref;
  Mask mask;
  long long pairs, T;
  double beta, gamma, smoothing, nll;
  int kind;                              // 0 sigmoid, 1 robust, 2 hinge, 3 ipo
  int normalized;
};

__device__ __forceinline__ double softplus(double v) { return fmax(v, 0.0) + log1p(exp(-fabs(v))); }   // -log sigma(-v)
__device__ __forceinline__ double sigmoid(double v) { return 1.0 / (1.0 + exp(-v)); }

// The loss of x and its derivative.
__device__ __forceinline__ double pair_loss(const Pairs& a, double x, double* slope) {
  const double q = a.beta * x - a.gamma, e = a.smoothing;
  if (a.kind <= 1) {
    const double sign = a.kind == 0 ? 1.0 : -1.0, f = a.kind == 0 ? 1.0 : 1.0 / (1.0 - 2.0 * e);
    *slope = a.beta * f * (sign * e * sigmoid(q) - (1.0 - e) * sigmoid(-q));
    return f * ((1.0 - e) * softplus(-q) + (e != 0.0 ? sign * e * softplus(q) : 0.0));      // (0 * inf: a token of no probability)
  }
  if (a.kind == 2) {
    *slope = q < 1.0 ? -a.beta : (q == q ? 0.0 : q);
    return q >= 1.0 ? 0.0 : 1.0 - q;
  }
  const double d = x - 0.5 / a.beta;
  *slope = 2.0 * d;
  return d * d;
}

// Calls f(t, N) over [begin, end) of a row whose token 0 is `phase` tokens behind a vector's boundary: single tokens up to the
// first boundary and behind the last, VEC at a time between them.
template <int VEC, typename F>
__device__ __forceinline__ void over_row(long long begin, long long end, int phase, F&& f) {
  const long long first = min(end, begin + (VEC - (begin + phase) % VEC) % VEC), past = first + (end - first) / VEC * VEC;
  for (long long t = first + static_cast<long long>(threadIdx.x) * VEC; t < past; t += PT_THREADS * VEC)
    f(t, std::integral_constant<int, VEC>());
  const int before = static_cast<int>(first - begin), singles = before + static_cast<int>(end - past), i = threadIdx.x;
  if (i < singles) f(i < before ? begin + i : past + (i - before), std::integral_constant<int, 1>());
}

// A block, or a cluster of them, per pair: scores, loss, rewards, and the gradient of both rows.
template <typename T, int VEC>
__global__ void __launch_bounds__(PT_THREADS, 5) pair_kernel(Pairs a, T* __restrict__ grad, double* __restrict__ loss,
                                                          float* __restrict__ rewards, Upstream up) {
  __shared__ double scratch[32][5];
  __shared__ double by_block[PAIR_SPLIT][5];
  __shared__ float weights[2];           // of the gradient's rows
  cg::cluster_group cluster = cg::this_cluster();
  if (up.done()) return;
  const int parts = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  if (parts > 1) cluster.barrier_arrive();      // (no block writes to another's shared memory before that one has begun)
  const long long p = blockIdx.x / parts;
  const long long begin = a.T * rank / parts, end = a.T * (rank + 1) / parts;
  double sums[5] = {};                   // score and tokens of the chosen, of the rejected row; the chosen's own log-probability
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const long long row = p + side * a.pairs;
    over_row<VEC>(begin, end, static_cast<int>(row * a.T % VEC), [&](long long t, auto n) {
      constexpr int N = decltype(n)::value;
      float m[N], v[N], r[N];
      MaskBits<N> bits;
      a.mask.load<N>(row * a.mask.stride + t, bits);
      fetch<N>(static_cast<const T*>(a.logp) + row * a.s_logp + t, v);
      if (a.ref) fetch<N>(static_cast<const T*>(a.ref) + row * a.s_ref + t, r);
      a.mask.values<N>(bits, m);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        // whatever a masked token holds reaches nothing (no branch: the next loads would wait behind it)
        const bool used = m[e] != 0.f;
        const double w = m[e], x = used ? v[e] : 0.f;
        sums[2 * side] += w * (a.ref ? x - (used ? r[e] : 0.f) : x);
        sums[2 * side + 1] += w;
        if (side == 0) sums[4] += w * x;
      }
    });
  }
  block_sums<5>(sums, scratch);
  if (parts > 1) {
    cluster.barrier_wait();
    if (static_cast<int>(threadIdx.x) < parts) {
      double* to = cluster.map_shared_rank(&by_block[rank][0], threadIdx.x);
#pragma unroll
      for (int k = 0; k < 5; ++k) to[k] = sums[k];
    }
    cluster.sync();
  }
  // (one thread: the pipe for fp64 would keep a block's worth of exponentials for a microsecond)
  if (threadIdx.x == 0) {
    for (int i = 0; parts > 1 && i < parts; ++i)
#pragma unroll
      for (int k = 0; k < 5; ++k) sums[k] = (i ? sums[k] : 0.0) + by_block[i][k];
    const double count[2] = {fmax(sums[1], 1.0), fmax(sums[3], 1.0)};
    const double score[2] = {a.normalized ? sums[0] / count[0] : sums[0], a.normalized ? sums[2] / count[1] : sums[2]};
    double slope;
    const double value = pair_loss(a, score[0] - score[1], &slope) - (a.nll != 0.0 ? a.nll * sums[4] / count[0] : 0.0);
    if (rank == 0 && rewards) {
      loss[p] = value;
      rewards[p] = static_cast<float>(a.beta * score[0]);
      rewards[p + a.pairs] = static_cast<float>(a.beta * score[1]);
    }
    const double scale = up.get() / static_cast<double>(a.pairs);
    weights[0] = static_cast<float>(((a.normalized ? slope / count[0] : slope) - a.nll / count[0]) * scale);
    weights[1] = static_cast<float>((a.normalized ? -slope / count[1] : -slope) * scale);
  }
  if (!grad) return;
  __syncthreads();
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const long long row = p + side * a.pairs;
    const float weight = weights[side];
    over_row<VEC>(begin, end, static_cast<int>(row * a.T % VEC), [&](long long t, auto n) {
      constexpr int N = decltype(n)::value;
      float m[N];
      a.mask.get<N>(row * a.mask.stride + t, m);
#pragma unroll
      for (int e = 0; e < N; ++e) m[e] = m[e] == 0.f ? 0.f : weight * m[e];
      put<N>(grad + row * a.T + t, m);
    });
  }
}

__global__ void __launch_bounds__(1024) pair_finish_kernel(const double* __restrict__ loss, long long pairs, float* __restrict__ out) {
  __shared__ double scratch[32][1];
  double v[1] = {0.0};
  for (long long i = threadIdx.x; i < pairs; i += blockDim.x) v[0] += loss[i];
  block_sums<1>(v, scratch);
  if (threadIdx.x == 0) *out = static_cast<float>(v[0] / static_cast<double>(pairs));
}

// ---------------------------------------------------------------------------------------------------
template <typename F>
static int pt_by_type(int dtype, F&& launch) {
  switch (dtype) {
    case 0: return launch(static_cast<__nv_bfloat16*>(nullptr));
    case 1: return launch(static_cast<__half*>(nullptr));
    case 2: return launch(static_cast<float*>(nullptr));
    default: return -1;
  }
}

static bool on_boundary(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
static Mask mask_of(const void* p, long long stride, long long kind) {
  static const int shift[6] = {0, 2, 3, 2, 1, 1};
  return {p, stride, static_cast<int>(kind), shift[kind]};
}
static int type_bytes(int dtype) { return dtype == 2 ? 4 : 2; }
static double high_part(double v) { return static_cast<double>(static_cast<float>(v)); }

}  // namespace ts

using namespace ts;

TS_DEFINE_ERROR_API(ts_posttrain)

// The arguments of a call, eight bytes each (ops/policy.py packs them).  dtype (of logp, old, ref and grad): 0 bf16, 1 fp16, 2
// fp32. ref, grad and stats may be null; loss too where only the gradient is wanted, times *factor (and where that is one, with
// `redo` alone).  stats: mean kl, share of clipped tokens, mean ratio.
struct PolicyCall {
  long long dtype;
  const void* logp;
  long long s_logp;
  const void* old;
  long long s_old;
  const void* ref;
  long long s_ref;
  const float* advantages;
  long long per_token;
  const void* mask;
  long long s_mask, mask_kind, rows, T;
  double log_low, log_high, low, high, beta;
  long long reduction;
  double constant;
  void* grad;
  float *loss, *stats;
  const float* factor;
  long long redo;
  double* workspace;
};

static bool policy_alone(long long rows, long long T) { return rows <= POLICY_ALONE_ROWS && rows * T <= POLICY_ALONE; }

// Number of doubles that ts_policy_loss needs as workspace: weights, counts, sums, a counter.  None where one block does it.
extern "C" long long ts_policy_workspace(long long rows, long long T) {
  return policy_alone(rows, T) ? 0 : rows + (POLICY_SUMS + 1) * static_cast<long long>(sm_count()) * POLICY_PER_SM + 1;
}

extern "C" int ts_policy_loss(const PolicyCall* c, void* stream) {
  const long long n = c->rows * c->T;
  if (c->rows <= 0 || c->T <= 0 || c->rows > 0x7fffffffll / POLICY_SPLIT || c->T > 0x3fffffffll || c->reduction < 0 || c->reduction > 2 ||
      c->mask_kind < 0 || c->mask_kind > 5 || c->dtype < 0 || c->dtype > 2)
    return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Policy a;
  a.logp = c->logp, a.old = c->old, a.ref = c->ref;
  a.s_logp = c->s_logp, a.s_old = c->s_old, a.s_ref = c->s_ref;
  a.advantages = c->advantages, a.per_token = static_cast<int>(c->per_token);
  a.mask = mask_of(c->mask, c->s_mask, c->mask_kind);
  a.rows = c->rows, a.T = c->T, a.tokens = n;
  a.constant = c->constant, a.reduction = static_cast<int>(c->reduction);
  a.bound_low[0] = static_cast<float>(c->log_low);
  a.bound_low[1] = c->log_low < -1e30 ? 0.f : static_cast<float>(c->log_low - high_part(c->log_low));
  a.bound_high[0] = static_cast<float>(c->log_high), a.bound_high[1] = static_cast<float>(c->log_high - high_part(c->log_high));
  a.low = static_cast<float>(c->low), a.high = static_cast<float>(c->high), a.beta = static_cast<float>(c->beta);
  // four tokens at a time where they lie together and on a boundary in every tensor: rows without gaps, or rows of whole fours
  const int e = type_bytes(static_cast<int>(c->dtype)), m = 1 << a.mask.shift;
  a.flat = a.s_logp == a.T && a.s_old == a.T && (!a.ref || a.s_ref == a.T) && a.mask.stride == a.T;
  const bool fours = (a.flat || ((a.T | a.s_logp | a.s_old | (a.ref ? a.s_ref : 0) | a.mask.stride) & 3) == 0) &&
                     on_boundary(a.logp, 4 * e) &&
                     on_boundary(a.old, 4 * e) && on_boundary(a.ref, 4 * e) && on_boundary(a.mask.p, m == 8 ? 16 : 4 * m) &&
                     on_boundary(c->grad, 4 * e) && (!a.per_token || on_boundary(a.advantages, 16)) && n % 4 == 0;
  const int vec = fours ? 4 : 1;
  const Upstream up{c->factor, static_cast<int>(c->redo)};
  const long long tile = static_cast<long long>(PT_THREADS) * vec, most = static_cast<long long>(sm_count()) * POLICY_PER_SM;
  const long long tiles = (n + tile - 1) / tile, blocks = tiles < most ? tiles : most;
  a.run = (tiles + blocks - 1) / blocks * tile;
  const unsigned used = static_cast<unsigned>((n + a.run - 1) / a.run);
  float* weights = reinterpret_cast<float*>(c->workspace);
  double *counts = c->workspace + a.rows, *partial = counts + most;
  unsigned* ticket = reinterpret_cast<unsigned*>(partial + POLICY_SUMS * most);
  return pt_by_type(static_cast<int>(c->dtype), [&](auto* t) {
    using E = std::remove_pointer_t<decltype(t)>;
    auto run = [&](auto v, auto f) {
      constexpr int VEC = decltype(v)::value;
      constexpr bool FLAT = decltype(f)::value;
      if (policy_alone(a.rows, a.T)) {
        policy_alone_kernel<E, VEC, FLAT><<<1, POLICY_ALONE_THREADS, 0, st>>>(a, static_cast<E*>(c->grad), c->loss, c->stats, up);
        return static_cast<int>(cudaGetLastError());
      }
      // a row is split while blocks are fewer than two to an SM and a part is worth one
      int parts = 1;
      if (a.reduction == 0)
        while (parts < POLICY_SPLIT && a.rows * parts < 2 * sm_count() && a.T / parts >= 8 * PT_THREADS * VEC) parts *= 2;
      constexpr int warps = PT_THREADS / 32;
      const unsigned by_row = static_cast<unsigned>(a.T <= POLICY_SHORT ? (a.rows + warps - 1) / warps : a.rows * parts);
      const unsigned counters = a.reduction == 0 ? by_row : a.reduction == 1 ? used : 1;
      const int rc = launch_chained(policy_count_kernel<VEC>, dim3(counters), dim3(PT_THREADS), 0, st, parts, false, a, weights, counts,
                                    ticket, up);
      if (rc) return rc;
      policy_kernel<E, VEC, FLAT><<<used, PT_THREADS, 0, st>>>(a, weights, counts, partial, ticket, static_cast<E*>(c->grad), c->loss,
                                                               c->stats, up);
      return static_cast<int>(cudaGetLastError());
    };
    using four = std::integral_constant<int, 4>;
    using one = std::integral_constant<int, 1>;
    return fours ? (a.flat ? run(four(), std::true_type()) : run(four(), std::false_type()))
                 : (a.flat ? run(one(), std::true_type()) : run(one(), std::false_type()));
  });
}

// grad [n] *= *factor; grad starts on a 16-byte boundary.
extern "C" int ts_scale_by(float* grad, const float* factor, long long n, void* stream) {
  if (n <= 0 || !on_boundary(grad, 16)) return -1;
  const long long blocks = (n + PT_THREADS * 8 - 1) / (PT_THREADS * 8), most = sm_count() * 8ll;
  scale_kernel<<<static_cast<unsigned>(blocks < most ? blocks : most), PT_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(grad, factor, n);
  return static_cast<int>(cudaGetLastError());
}

// Rows 0 .. pairs - 1 are the chosen, the next the rejected sequences.  loss: one float; rewards: 2 * pairs floats; workspace:
// `pairs` doubles.  ref and grad may be null; loss, rewards, factor and redo as above.
struct PairsCall {
  long long dtype;
  const void* logp;
  long long s_logp;
  const void* ref;
  long long s_ref;
  const void* mask;
  long long s_mask, mask_kind, pairs, T;
  double beta, gamma, smoothing, nll;
  long long kind, normalized;
  void* grad;
  float *loss, *rewards;
  const float* factor;
  long long redo;
  double* workspace;
};

extern "C" int ts_preference_loss(const PairsCall* c, void* stream) {
  if (c->pairs <= 0 || c->T <= 0 || c->pairs > 0x7fffffffll / PAIR_SPLIT || c->kind < 0 || c->kind > 3 || c->mask_kind < 0 ||
      c->mask_kind > 5 || c->dtype < 0 || c->dtype > 2)
    return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Pairs a{c->logp, c->ref, c->s_logp, c->s_ref, mask_of(c->mask, c->s_mask, c->mask_kind), c->pairs, c->T,
                c->beta, c->gamma, c->smoothing, c->nll, static_cast<int>(c->kind), static_cast<int>(c->normalized)};
  // four tokens at a time where all tensors start on a boundary and their rows are as far behind one (the gradient's rows are T
  // long)
  const int e = type_bytes(static_cast<int>(c->dtype)), m = 1 << a.mask.shift;
  const bool fours = ((a.s_logp ^ a.T) & 3) == 0 && (!a.ref || ((a.s_ref ^ a.T) & 3) == 0) && ((a.mask.stride ^ a.T) & 3) == 0 &&
                     on_boundary(a.logp, 4 * e) && on_boundary(a.ref, 4 * e) && on_boundary(a.mask.p, m == 8 ? 16 : 4 * m) &&
                     on_boundary(c->grad, 4 * e);
  // a pair is split while blocks are fewer than four to an SM and its parts are worth one (in one block and split: one pair of
  // 16384 24.3 and 10.6 us, 160 of them 31.9 and 18.9; one of 1024 7.2 and 8.9, 160 of 4096 in eight blocks each 12.5 and 23.4)
  int parts = 1;
  while (parts < PAIR_SPLIT && a.pairs * parts < 4 * sm_count() && a.T / parts >= 2 * PAIR_TOKENS) parts *= 2;
  return pt_by_type(static_cast<int>(c->dtype), [&](auto* t) {
    using E = std::remove_pointer_t<decltype(t)>;
    auto kernel = fours ? pair_kernel<E, 4> : pair_kernel<E, 1>;
    const int rc = launch_chained(kernel, dim3(static_cast<unsigned>(a.pairs * parts)), dim3(PT_THREADS), 0, st, parts, false, a,
                                  static_cast<E*>(c->grad), c->workspace, c->rewards, Upstream{c->factor, static_cast<int>(c->redo)});
    if (rc) return rc;
    if (c->loss) pair_finish_kernel<<<1, 1024, 0, st>>>(c->workspace, a.pairs, c->loss);
    return static_cast<int>(cudaGetLastError());
  });
}
