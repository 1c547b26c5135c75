// Losses over token log-probabilities [rows][T], with their gradients: the clipped policy loss with a KL term, and the losses of
// (chosen, rejected) pairs.
//
// Policy, for a token of weight m (its mask) in a row of advantage a:
//   r = e^(logp - old),  clipped = a > 0 ? r > 1 + high : a < 0 and r < 1 - low,  d = ref - logp
//   token = -a (clipped ? bound : r) + beta (e^d - 1 - d),  d token / d logp = (clipped ? 0 : -a r) - beta (e^d - 1)
//   loss  = sum m w token,  w = 1 / (rows sum_row m), 1 / sum m or 1 / (rows length); the sums of m are at least 1
// Which side of a bound a token is on is decided in 64 bits (the difference of two fp32 numbers is exact there): its gradient
// jumps at the bound.  e^d - 1 - d is a power series near zero, where the difference would cancel.  Sums are fp64.
//
// Pairs, rows p (chosen) and P + p (rejected), of scores s = sum m (logp - ref), divided by max(sum m, 1) where asked:
//   x = s_p - s_(P + p),  q = beta x - gamma
//   sigmoid -(1 - eps) log sigma(q) - eps log sigma(-q);  robust: the same with + eps, / (1 - 2 eps);  hinge max(0, 1 - q);
//   ipo (x - 1 / (2 beta))^2;  and nll * the mean of -logp over the chosen row's tokens
// The scores are long sums whose difference decides: they, and all that is done per pair, are fp64.
//
// Gradients leave with the loss, for an upstream gradient of one.  Where it turns out to be another, fp32 gradients are multiplied
// by it; 16-bit ones, which that would round twice, are computed again (`Upstream`).
#include "common.cuh"
#include "host_common.h"

namespace ts {

constexpr int PT_THREADS = 256;
constexpr int PT_TILE = 2048;            // tokens of a block

__device__ __forceinline__ float pt_f32(float v) { return v; }
__device__ __forceinline__ float pt_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float pt_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T pt_from(float v);
template <>
__device__ __forceinline__ float pt_from<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 pt_from<__nv_bfloat16>(float v) { return __float2bfloat16(v); }
template <>
__device__ __forceinline__ __half pt_from<__half>(float v) { return __float2half(v); }

// What flows into the loss: nothing known yet (null), or a factor of the gradient; `redo`: also where it is one.
struct Upstream {
  const float* factor;
  int redo;
  __device__ __forceinline__ bool done() const { return factor && !redo && *factor == 1.f; }
  __device__ __forceinline__ float get() const { return factor ? *factor : 1.f; }
};

struct Mask {
  const void* p;
  long long stride;                      // elements between rows
  int kind;                              // 0 bool / uint8, 1 int32, 2 int64, 3 fp32, 4 bf16, 5 fp16
  __device__ __forceinline__ float at(long long row, long long t) const {
    const long long i = row * stride + t;
    switch (kind) {
      case 0: return static_cast<float>(static_cast<const unsigned char*>(p)[i]);
      case 1: return static_cast<float>(static_cast<const int*>(p)[i]);
      case 2: return static_cast<float>(static_cast<const long long*>(p)[i]);
      case 3: return static_cast<const float*>(p)[i];
      case 4: return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
      default: return __half2float(static_cast<const __half*>(p)[i]);
    }
  }
};

// Sum over the block in a fixed order; every thread gets it.
__device__ __forceinline__ double block_sum64(double v, double* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarp = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  v = lane < nwarp ? scratch[lane] : 0.0;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ---------------------------------------------------------------------------------------------------
// Clipped policy loss
// ---------------------------------------------------------------------------------------------------
constexpr int POLICY_SUMS = 5;           // loss, kl m, clipped m, ratio m, m

struct Policy {
  const void *logp, *old, *ref;
  long long s_logp, s_old, s_ref;        // elements between rows
  const float* advantages;               // [rows] or [rows][T]
  int per_token;
  Mask mask;
  long long rows, T;
  double log_low, log_high;              // ln(1 - low), ln(1 + high)
  float low, high, beta;                 // 1 - low, 1 + high
  int reduction;                         // 0 rows' means, 1 all tokens, 2 a constant
  double constant;                       // 1 / (rows * length) of reduction 2
};

__global__ void __launch_bounds__(PT_THREADS) policy_count_kernel(Mask mask, long long T, double* __restrict__ counts, Upstream up) {
  __shared__ double scratch[32];
  if (up.done()) return;
  double n = 0.0;
  for (long long t = threadIdx.x; t < T; t += PT_THREADS) n += mask.at(blockIdx.x, t);
  n = block_sum64(n, scratch);
  if (threadIdx.x == 0) counts[blockIdx.x] = n;
}

// e^d - 1 - d, where e = e^d - 1
__device__ __forceinline__ float exp_rest(float d, float e) {
  const float series = 0.5f + d * (1.f / 6.f + d * (1.f / 24.f + d * (1.f / 120.f + d * (1.f / 720.f + d * (1.f / 5040.f +
                       d * (1.f / 40320.f + d * (1.f / 362880.f)))))));
  return fabsf(d) < 0.5f ? d * d * series : e - d;
}

template <typename T>
__global__ void __launch_bounds__(PT_THREADS) policy_kernel(Policy a, const double* __restrict__ counts, T* __restrict__ grad,
                                                            double* __restrict__ partial, Upstream up) {
  __shared__ double scratch[32];
  if (up.done()) return;
  const float factor = up.get();
  const long long n = a.rows * a.T;
  double all = 0.0;
  if (a.reduction == 1) {
    for (long long r = threadIdx.x; r < a.rows; r += PT_THREADS) all += counts[r];
    all = block_sum64(all, scratch);
  }
  double sums[POLICY_SUMS] = {};
  const long long end = min(n, (blockIdx.x + 1ll) * PT_TILE);
  for (long long i = blockIdx.x * static_cast<long long>(PT_TILE) + threadIdx.x; i < end; i += PT_THREADS) {
    const long long row = i / a.T, t = i - row * a.T;
    const float m = a.mask.at(row, t);
    float slope = 0.f;
    if (m != 0.f) {
      const double w = a.reduction == 0 ? 1.0 / (fmax(counts[row], 1.0) * static_cast<double>(a.rows))
                       : a.reduction == 1 ? 1.0 / fmax(all, 1.0) : a.constant;
      const float logp = pt_f32(static_cast<const T*>(a.logp)[row * a.s_logp + t]);
      const float old = pt_f32(static_cast<const T*>(a.old)[row * a.s_old + t]);
      const float adv = a.advantages[a.per_token ? i : row];
      const double moved = static_cast<double>(logp) - static_cast<double>(old);
      const float ratio = expf(static_cast<float>(moved));
      const bool clipped = (adv > 0.f && moved > a.log_high) || (adv < 0.f && moved < a.log_low);
      // (0 * inf: a ratio that overflows has no say where the advantage is zero)
      const float gain = adv == 0.f && ratio == INFINITY ? 0.f : adv * (clipped ? (adv > 0.f ? a.high : a.low) : ratio);
      float token = -gain, kl = 0.f;
      slope = clipped ? 0.f : -gain;
      if (a.ref) {
        const float d = static_cast<float>(static_cast<double>(pt_f32(static_cast<const T*>(a.ref)[row * a.s_ref + t])) - logp);
        const float e = expm1f(d);
        kl = exp_rest(d, e);
        token += a.beta * kl;
        slope -= a.beta * e;
      }
      sums[0] += m * w * token;
      sums[1] += static_cast<double>(m) * kl;
      sums[2] += clipped ? m : 0.f;
      sums[3] += static_cast<double>(m) * ratio;
      sums[4] += m;
      slope = static_cast<float>(slope * m * w * factor);
    }
    if (grad) grad[i] = pt_from<T>(slope);
  }
#pragma unroll
  for (int k = 0; k < POLICY_SUMS; ++k) {
    const double v = block_sum64(sums[k], scratch);
    if (threadIdx.x == 0) partial[blockIdx.x * static_cast<long long>(POLICY_SUMS) + k] = v;
  }
}

// stats: mean kl, share of clipped tokens, mean ratio
__global__ void __launch_bounds__(1024) policy_finish_kernel(const double* __restrict__ partial, int blocks, float* __restrict__ loss,
                                                             float* __restrict__ stats) {
  __shared__ double scratch[32];
  double v[POLICY_SUMS];
  for (int k = 0; k < POLICY_SUMS; ++k) {
    v[k] = 0.0;
    for (int i = threadIdx.x; i < blocks; i += blockDim.x) v[k] += partial[i * static_cast<long long>(POLICY_SUMS) + k];
    v[k] = block_sum64(v[k], scratch);
  }
  if (threadIdx.x == 0) {
    *loss = static_cast<float>(v[0]);
    for (int k = 1; k < 4; ++k) stats[k - 1] = static_cast<float>(v[k] / fmax(v[4], 1.0));
  }
}

// grad *= *factor; a factor of one leaves it as it is
__global__ void __launch_bounds__(PT_THREADS) scale_kernel(float* __restrict__ grad, const float* __restrict__ factor, long long n) {
  const float f = *factor;
  if (f == 1.f) return;
  for (long long i = blockIdx.x * static_cast<long long>(PT_THREADS) + threadIdx.x; i < n; i += gridDim.x * static_cast<long long>(PT_THREADS))
    grad[i] *= f;
}

// ---------------------------------------------------------------------------------------------------
// Pairs
// ---------------------------------------------------------------------------------------------------
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
    return f * ((1.0 - e) * softplus(-q) + sign * e * softplus(q));
  }
  if (a.kind == 2) {
    *slope = q < 1.0 ? -a.beta : (q == q ? 0.0 : q);
    return q >= 1.0 ? 0.0 : 1.0 - q;
  }
  const double d = x - 0.5 / a.beta;
  *slope = 2.0 * d;
  return d * d;
}

// One block per pair: scores, loss, rewards, and the gradient of both rows.
template <typename T>
__global__ void __launch_bounds__(PT_THREADS) pair_kernel(Pairs a, T* __restrict__ grad, double* __restrict__ loss,
                                                          float* __restrict__ rewards, Upstream up) {
  __shared__ double scratch[32];
  if (up.done()) return;
  const long long p = blockIdx.x;
  double score[2], count[2], own = 0.0;
  for (int side = 0; side < 2; ++side) {
    const long long row = p + side * a.pairs;
    double s = 0.0, c = 0.0, l = 0.0;
    for (long long t = threadIdx.x; t < a.T; t += PT_THREADS) {
      const float m = a.mask.at(row, t);
      if (m == 0.f) continue;
      const double v = pt_f32(static_cast<const T*>(a.logp)[row * a.s_logp + t]);
      const double r = a.ref ? pt_f32(static_cast<const T*>(a.ref)[row * a.s_ref + t]) : 0.f;
      s += m * (v - r);
      l += m * v;
      c += m;
    }
    score[side] = block_sum64(s, scratch);
    count[side] = fmax(block_sum64(c, scratch), 1.0);
    if (side == 0) own = block_sum64(l, scratch) / count[0];
    if (a.normalized) score[side] /= count[side];
  }
  double slope;
  const double value = pair_loss(a, score[0] - score[1], &slope) - (a.nll != 0.0 ? a.nll * own : 0.0);
  if (threadIdx.x == 0 && rewards) {
    loss[p] = value;
    rewards[p] = static_cast<float>(a.beta * score[0]);
    rewards[p + a.pairs] = static_cast<float>(a.beta * score[1]);
  }
  if (!grad) return;
  for (int side = 0; side < 2; ++side) {
    const long long row = p + side * a.pairs;
    double w = (side ? -slope : slope) / (a.normalized ? count[side] : 1.0);
    if (side == 0) w -= a.nll / count[0];
    w *= up.get() / static_cast<double>(a.pairs);
    for (long long t = threadIdx.x; t < a.T; t += PT_THREADS) {
      const float m = a.mask.at(row, t);
      grad[row * a.T + t] = pt_from<T>(m == 0.f ? 0.f : static_cast<float>(w * m));
    }
  }
}

__global__ void __launch_bounds__(1024) pair_finish_kernel(const double* __restrict__ loss, long long pairs, float* __restrict__ out) {
  __shared__ double scratch[32];
  double v = 0.0;
  for (long long i = threadIdx.x; i < pairs; i += blockDim.x) v += loss[i];
  v = block_sum64(v, scratch);
  if (threadIdx.x == 0) *out = static_cast<float>(v / static_cast<double>(pairs));
}

template <typename F>
static int pt_by_type(int dtype, F&& launch) {
  switch (dtype) {
    case 0: launch(static_cast<__nv_bfloat16*>(nullptr)); break;
    case 1: launch(static_cast<__half*>(nullptr)); break;
    case 2: launch(static_cast<float*>(nullptr)); break;
    default: return -1;
  }
  return static_cast<int>(cudaGetLastError());
}

}  // namespace ts

using namespace ts;

TS_DEFINE_ERROR_API(ts_posttrain)

// Number of doubles that ts_policy_loss needs as workspace.
extern "C" long long ts_policy_workspace(long long rows, long long T) {
  return rows + POLICY_SUMS * ((rows * T + PT_TILE - 1) / PT_TILE);
}

// dtype (of logp, old, ref and grad): 0 bf16, 1 fp16, 2 fp32.  ref and grad may be null.  loss: one float;
// stats: three; both null where only the gradient is wanted, times *factor (and where that is one, with `redo` alone).
extern "C" int ts_policy_loss(int dtype, const void* logp, long long s_logp, const void* old, long long s_old, const void* ref,
                              long long s_ref, const float* advantages, int per_token, const void* mask, long long s_mask,
                              int mask_kind, long long rows, long long T, double log_low, double log_high, double low, double high,
                              double beta, int reduction, double constant, void* grad, float* loss, float* stats, const float* factor,
                              int redo, double* workspace, void* stream) {
  const long long blocks = (rows * T + PT_TILE - 1) / PT_TILE;
  if (rows <= 0 || T <= 0 || rows > 0x7fffffffll || blocks > 0x7fffffffll || reduction < 0 || reduction > 2) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Mask m{mask, s_mask, mask_kind};
  const Policy a{logp, old, ref, s_logp, s_old, s_ref, advantages, per_token, m, rows, T, log_low, log_high,
                 static_cast<float>(low), static_cast<float>(high), static_cast<float>(beta), reduction, constant};
  const Upstream up{factor, redo};
  double *counts = workspace, *partial = workspace + rows;
  if (reduction != 2) policy_count_kernel<<<static_cast<unsigned>(rows), PT_THREADS, 0, st>>>(m, T, counts, up);
  return pt_by_type(dtype, [&](auto* t) {
    using E = std::remove_pointer_t<decltype(t)>;
    policy_kernel<E><<<static_cast<unsigned>(blocks), PT_THREADS, 0, st>>>(a, counts, static_cast<E*>(grad), partial, up);
    if (loss) policy_finish_kernel<<<1, 1024, 0, st>>>(partial, static_cast<int>(blocks), loss, stats);
  });
}

// grad [n] *= *factor.
extern "C" int ts_scale_by(float* grad, const float* factor, long long n, void* stream) {
  if (n <= 0) return -1;
  const long long blocks = (n + PT_THREADS * 4 - 1) / (PT_THREADS * 4);
  scale_kernel<<<static_cast<unsigned>(blocks < 2368 ? blocks : 2368), PT_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(grad, factor, n);
  return static_cast<int>(cudaGetLastError());
}

// Rows 0 .. pairs - 1 are the chosen, the next the rejected sequences.  loss: one float; rewards: 2 * pairs floats; workspace:
// `pairs` doubles.  ref and grad may be null; loss, rewards, factor and redo as above.
extern "C" int ts_preference_loss(int dtype, const void* logp, long long s_logp, const void* ref, long long s_ref, const void* mask,
                                  long long s_mask, int mask_kind, long long pairs, long long T, double beta, double gamma,
                                  double smoothing, double nll, int kind, int normalized, void* grad, float* loss, float* rewards,
                                  const float* factor, int redo, double* workspace, void* stream) {
  if (pairs <= 0 || T <= 0 || pairs > 0x3fffffffll || kind < 0 || kind > 3) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Pairs a{logp, ref, s_logp, s_ref, {mask, s_mask, mask_kind}, pairs, T, beta, gamma, smoothing, nll, kind, normalized};
  return pt_by_type(dtype, [&](auto* t) {
    using E = std::remove_pointer_t<decltype(t)>;
    pair_kernel<E><<<static_cast<unsigned>(pairs), PT_THREADS, 0, st>>>(a, static_cast<E*>(grad), workspace, rewards, {factor, redo});
    if (loss) pair_finish_kernel<<<1, 1024, 0, st>>>(workspace, pairs, loss);
  });
}
