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
// Forward reads the logits once: a thread keeps a running (m, S, U) over 16-byte vectors and raises m once for the vectors that
// it has in flight.  Few rows: a block or a cluster per row, one launch.  Many: a warp per part of a row, all of them alike, so
// that blocks end evenly and nothing waits inside a block; a second launch joins a row's parts.
//
// Bounds: 2 bytes of a logit and an exponential for each of them; at the memory's rate the special-function unit is busy 70 % of
// the time and the schedulers 60 %.  1644 rows of 128256 bf16 logits (421 MB) take 72 us, 79 with the entropy (5.8 and 5.3 TB/s,
// joining included; a plain copy moves 6.5).  A block of 512 threads a row took 89: 1.4 to 1.7 rounds of blocks, and waits at
// each row's end; clusters of two or four blocks 93 and 120; eight vectors in flight 105, parts of 512 vectors 89.  A quarter of
// the exponentials as polynomials freed the special-function unit and cost as much in instructions.  A cap's tanh asks for
// most of the instructions: 2103 rows of 32001 fp32 logits (269 MB) take 66 us, 41 of them the memory's; issue slots are 67 % busy.
#include <cooperative_groups.h>

#include "common.cuh"
#include "host_common.h"

namespace ts {

constexpr int LP_THREADS = 512;
constexpr int LP_FLIGHT = 4;             // vectors of a thread in flight
constexpr int LP_SPLIT = 8;              // most blocks of a row
constexpr int LP_BACK_THREADS = 64, LP_BACK_FLIGHT = 8;
constexpr int LP_PART_THREADS = 128, LP_PART_FLIGHT = 4, LP_PART = 1024;     // vectors of a warp's part
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

// Pairs of fp32 in one instruction.
struct Pair {
  uint64_t v;
  __device__ __forceinline__ Pair(uint64_t x) : v(x) {}
  __device__ __forceinline__ Pair(float a, float b) : v(pack_f32x2(a, b)) {}
  __device__ __forceinline__ Pair operator+(Pair o) const { return add_f32x2(v, o.v); }
  __device__ __forceinline__ Pair operator*(Pair o) const { return mul_f32x2(v, o.v); }
  __device__ __forceinline__ float2 get() const { return unpack_f32x2(v); }
};
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) { return fma_f32x2(a.v, b.v, c.v); }

// 16 bytes of logits: N values, their largest, and the pattern of a value that counts for nothing.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ uint4 nothing() { return make_uint4(NOTHING, NOTHING, NOTHING, NOTHING); }
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
  static __device__ __forceinline__ uint4 nothing() { return make_uint4(NOTHING, NOTHING, NOTHING, NOTHING); }
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
  static __device__ __forceinline__ uint4 nothing() { return make_uint4(NOTHING, NOTHING, NOTHING, NOTHING); }
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

// Logits are read once in each direction and are gone by then: they pass the L1 by.  (Not by the read-only path: a gradient may
// take their place.)
__device__ __forceinline__ uint4 load_once(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

struct LogitRows {
  long long rows, inner;             // row r is (r / inner, r % inner)
  long long stride_outer, stride_inner;
  int V;
  float k, k2;                       // f or f c: y = k v; the same times log2(e)
  float inv_cap;                     // 1 / c, or 0
  long long ignore;
  int lenient;                       // labels outside the vocabulary count as ignored
  __device__ __forceinline__ bool ignored(long long label) const { return label == ignore || (lenient && (label < 0 || label >= V)); }
  __device__ __forceinline__ long long offset(long long r) const {
    return (r / inner) * stride_outer + (r % inner) * stride_inner;
  }
};

// tanh(x), x = z / c, of two values: below a seam the odd polynomial x + x q P(q), q = x^2, above it 1 - E 2 / (1 + E), E = e^(-2 |x|).
// P is a minimax fit (Remez' exchange) to (tanh(x) / x - 1) / q, off by 2^-25.9 of tanh.  Rounding included, tanh is off by 2^-22.8 of its
// value at most and 2^-25 in the mean, as far as the library's is: at the seam an error of E counts a third of itself, and where E is
// closer to one and counts in full the polynomial has taken over.  (A seam at 0.15 took as long and was off by up to 2^-20.9.)
// Without a slope the quotient is a fit as well (2^-26, for E <= e^-1.8), which leaves one call of the special-function unit for an
// element; the forward pass asks for most of them.  With one it is a reciprocal, which also gives a quarter of the slope 1 - tanh^2,
// E / (1 + E)^2.  FINE: below the seam, where that is off by 2^-21.7, the slope is the difference, which cancels only above; results of 16
// bits do not show it (2103 x 32001 bf16 gradients take 74 us without and 85 with it, fp32 ones 92 and 92).
constexpr float TANH_SEAM = 0.9f;
enum Slope { NONE, COARSE, FINE };
template <bool CAP, Slope SLOPE>
__device__ __forceinline__ Pair capped2(float z, float w, float inv_cap, Pair* quarter = nullptr) {
  if (!CAP) return Pair(z, w);
  auto both = [](float v) { return Pair(v, v); };
  const Pair v = Pair(z, w) * both(inv_cap), q = v * v;
  const float2 x = v.get();
  const float2 e2 = make_float2(fast_ex2(fabsf(x.x) * (-2.f * LOG2E)), fast_ex2(fabsf(x.y) * (-2.f * LOG2E)));
  const Pair e(e2.x, e2.y);
  Pair p = fma2(q, both(1.30395975e-3f), both(-6.86005596e-3f));
  p = fma2(q, p, both(2.09041275e-2f));
  p = fma2(q, p, both(-5.37214912e-2f));
  p = fma2(q, p, both(1.33303598e-1f));
  p = fma2(q, p, both(-3.33332121e-1f));
  const Pair odd = fma2(v, q * p, v);
  const float2 low = odd.get();
  const bool poly_x = fabsf(x.x) < TANH_SEAM, poly_y = fabsf(x.y) < TANH_SEAM;
  float2 high;
  if (SLOPE != NONE) {
    const Pair r(fast_rcp(1.f + e2.x), fast_rcp(1.f + e2.y)), er = e * r;
    high = fma2(er, both(-2.f), both(1.f)).get();
    *quarter = er * r;
    if (SLOPE == FINE) {
      const float2 above = quarter->get(), below = fma2(odd * both(-0.25f), odd, both(0.25f)).get();
      *quarter = Pair(poly_x ? below.x : above.x, poly_y ? below.y : above.y);
    }
  } else {
    Pair r = fma2(e, both(-1.25909388f), both(1.87718737f));
    r = fma2(e, r, both(-1.99024522f));
    r = fma2(e, r, both(1.99965322f));
    r = fma2(e, r, both(-1.99999595f));
    high = fma2(e, r, both(1.f)).get();
  }
  return Pair(poly_x ? low.x : copysignf(high.x, x.x), poly_y ? low.y : copysignf(high.y, x.y));
}
// One value, with the bits of two.
template <bool CAP>
__device__ __forceinline__ float capped(float z, float inv_cap) {
  return CAP ? capped2<CAP, NONE>(z, z, inv_cap).get().x : z;
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

// u of one value, where m is a finite maximum or there is none yet; never below LP_LOWEST, so that u 2^u is zero where 2^u is.
__device__ __forceinline__ float exponent(float v, float m, float k2) { return max_nan(k2 * (v - (m == -INFINITY ? 0.f : m)), LP_LOWEST); }

template <bool CAP, bool ENT>
__device__ __forceinline__ void add_value(Softmax& acc, float z, float k2, float inv_cap) {
  const float v = capped<CAP>(z, inv_cap);
  acc.raise<ENT>(max_nan(acc.m, v), k2);
  const float t = exponent(v, acc.m, k2), e = fast_ex2(t);
  acc.s += e;
  if (ENT) acc.u += t * e;
}

// Adds the first `n` of N 16-byte vectors to a thread's (m, S, U); the others hold values of -inf, which count for nothing unless
// a cap makes them finite.  An entropy's 0 * -inf (logits of -inf) shows as NaN; it is then summed again with exponents that are
// bounded below.
template <typename T, bool CAP, bool ENT, int N>
__device__ __forceinline__ void add_vectors(Softmax& acc, const uint4* r, int n, float k2, float inv_cap) {
  using W = Vec<T>;
  const float top = max_nan(acc.m, capped<CAP>(W::largest(r, N), inv_cap));
  acc.raise<ENT>(top, k2);
  const float m = top == -INFINITY ? 0.f : top;
  const Pair minus(-m, -m), k(k2, k2);
  Pair s(0.f, 0.f), u(0.f, 0.f);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (CAP && j >= n) break;
    float f[W::N];
    W::unpack(r[j], f);
#pragma unroll
    for (int e = 0; e < W::N; e += 2) {
      const Pair t = (capped2<CAP, NONE>(f[e], f[e + 1], inv_cap) + minus) * k;
      const float2 x = t.get();
      const Pair p(fast_ex2(x.x), fast_ex2(x.y));
      s = s + p;
      if (ENT) u = fma2(t, p, u);
    }
  }
  const float2 x = s.get();
  acc.s += x.x + x.y;
  if (!ENT) return;
  const float2 y = u.get();
  float extra = y.x + y.y;
  if (extra != extra) {
    extra = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (CAP && j >= n) break;
      float f[W::N];
      W::unpack(r[j], f);
#pragma unroll 1
      for (int e = 0; e < W::N; ++e) {
        const float t = exponent(capped<CAP>(f[e], inv_cap), top, k2);
        extra += t * fast_ex2(t);
      }
    }
  }
  acc.u += extra;
}

template <bool ENT>
__device__ __forceinline__ void join_warp(Softmax& x, float k2) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    Softmax b;
    b.m = __shfl_xor_sync(0xffffffffu, x.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, x.s, o);
    if (ENT) b.u = __shfl_xor_sync(0xffffffffu, x.u, o);
    x.join<ENT>(b, k2);
  }
}

// A row: values before its first 16-byte boundary, vectors, values behind the last.
template <typename T>
struct Row {
  const T* z;
  int head, vectors, V;
  __device__ __forceinline__ Row(const T* at, int n) : z(at), V(n) {
    head = min(n, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(at) & 15)) & 15) / static_cast<int>(sizeof(T)));
    vectors = (n - head) / Vec<T>::N;
  }
  __device__ __forceinline__ const uint4* body() const { return reinterpret_cast<const uint4*>(z + head); }
  __device__ __forceinline__ int extra() const { return V - vectors * Vec<T>::N; }            // fewer than two vectors
  __device__ __forceinline__ int lone(int i) const { return i < head ? i : i + vectors * Vec<T>::N; }
};

// What a row's (m, S, U) come to.
template <typename T, bool CAP>
__device__ __forceinline__ void row_results(const Softmax& x, const Row<T>& row, long long r, long long label, const LogitRows& a,
                                            float* logp, float* entropy, float4* kept) {
  const bool outside = label < 0 || label >= a.V;
  // a row whose largest logit is +inf, -inf or NaN has no distribution
  const bool proper = x.m - x.m == 0.f;
  const float v = outside ? NAN : capped<CAP>(Vec<T>::value(row.z[label]), a.inv_cap);
  logp[r] = proper ? a.k * (v - x.m) - logf(x.s) : v - x.m;
  const float H = proper ? logf(x.s) - LN2 * (x.u / x.s) : NAN;
  if (entropy) entropy[r] = H;
  if (kept) kept[r] = make_float4(x.m, x.s, H, 0.f);
}
__device__ __forceinline__ void ignored_row(long long r, float* logp, float* entropy, float4* kept) {
  logp[r] = 0.f;
  if (entropy) entropy[r] = 0.f;
  if (kept) kept[r] = make_float4(0.f, 1.f, 0.f, 0.f);
}

// One block per row, or a cluster of them.
template <typename T, bool CAP, bool ENT>
__global__ void __launch_bounds__(LP_THREADS) logprob_row_kernel(const T* __restrict__ logits, const long long* __restrict__ labels,
                                                                 float* __restrict__ logp, float* __restrict__ entropy,
                                                                 float4* __restrict__ kept, LogitRows a) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), parts = static_cast<int>(cluster.num_blocks());
  __shared__ Softmax by_warp[LP_THREADS / 32];
  __shared__ Softmax by_block[LP_SPLIT];
  const long long r = blockIdx.x / parts, label = labels[r];
  if (a.ignored(label)) {
    if (threadIdx.x == 0 && rank == 0) ignored_row(r, logp, entropy, kept);
    return;                                   // (the whole cluster: it has one row)
  }
  if (parts > 1) cluster.barrier_arrive();    // (no block writes to another's shared memory before that one has begun)
  const Row<T> row(logits + a.offset(r), a.V);
  const uint4* body = row.body();
  const int begin = static_cast<int>(static_cast<long long>(row.vectors) * rank / parts);
  const int end = static_cast<int>(static_cast<long long>(row.vectors) * (rank + 1) / parts);
  Softmax acc;
  for (int i = begin + static_cast<int>(threadIdx.x); i < end; i += LP_THREADS * LP_FLIGHT) {
    uint4 v[LP_FLIGHT];
#pragma unroll
    for (int j = 0; j < LP_FLIGHT; ++j) v[j] = i + j * LP_THREADS < end ? load_once(body + i + j * LP_THREADS) : Vec<T>::nothing();
    add_vectors<T, CAP, ENT, LP_FLIGHT>(acc, v, (end - i + LP_THREADS - 1) / LP_THREADS, a.k2, a.inv_cap);
  }
  if (rank == 0 && static_cast<int>(threadIdx.x) < row.extra())
    add_value<CAP, ENT>(acc, Vec<T>::value(row.z[row.lone(threadIdx.x)]), a.k2, a.inv_cap);
  join_warp<ENT>(acc, a.k2);
  if ((threadIdx.x & 31) == 0) by_warp[threadIdx.x >> 5] = acc;
  __syncthreads();
  if (threadIdx.x < 32) {
    acc = threadIdx.x < LP_THREADS / 32 ? by_warp[threadIdx.x] : Softmax();
    join_warp<ENT>(acc, a.k2);
  }
  if (parts > 1) {
    cluster.barrier_wait();
    if (threadIdx.x == 0) *cluster.map_shared_rank(by_block + rank, 0) = acc;
    cluster.sync();
    if (rank != 0) return;
    if (threadIdx.x == 0) {
      acc = by_block[0];
      for (int i = 1; i < parts; ++i) acc.join<ENT>(by_block[i], a.k2);
    }
  }
  if (threadIdx.x == 0) row_results<T, CAP>(acc, row, r, label, a, logp, entropy, kept);
}

// A warp per part of a row: LP_PART vectors of it, or all where that is one part.
template <typename T, bool CAP, bool ENT>
__global__ void __launch_bounds__(LP_PART_THREADS) logprob_part_kernel(const T* __restrict__ logits, const long long* __restrict__ labels,
                                                                       Softmax* __restrict__ partial, float* __restrict__ logp,
                                                                       float* __restrict__ entropy, float4* __restrict__ kept,
                                                                       LogitRows a, int parts) {
  constexpr int step = 32 * LP_PART_FLIGHT;
  const long long unit = blockIdx.x * static_cast<long long>(LP_PART_THREADS / 32) + (threadIdx.x >> 5), r = unit / parts;
  const int lane = threadIdx.x & 31;
  if (r >= a.rows) return;
  const long long label = labels[r];
  if (a.ignored(label)) {
    if (parts == 1 && lane == 0) ignored_row(r, logp, entropy, kept);
    return;
  }
  const Row<T> row(logits + a.offset(r), a.V);
  const int begin = static_cast<int>(unit - r * parts) * LP_PART, end = parts == 1 ? row.vectors : min(row.vectors, begin + LP_PART);
  const uint4* body = row.body() + lane;
  Softmax acc;
  uint4 v[LP_PART_FLIGHT], next[LP_PART_FLIGHT];
  int i = begin;
  if (i + step <= end) {
#pragma unroll
    for (int j = 0; j < LP_PART_FLIGHT; ++j) next[j] = load_once(body + i + j * 32);
    for (; i + step <= end; i += step) {
#pragma unroll
      for (int j = 0; j < LP_PART_FLIGHT; ++j) v[j] = next[j];
      if (i + 2 * step <= end)
#pragma unroll
        for (int j = 0; j < LP_PART_FLIGHT; ++j) next[j] = load_once(body + i + step + j * 32);
      add_vectors<T, CAP, ENT, LP_PART_FLIGHT>(acc, v, LP_PART_FLIGHT, a.k2, a.inv_cap);
    }
  }
  if (i < end) {
#pragma unroll
    for (int j = 0; j < LP_PART_FLIGHT; ++j) v[j] = i + lane + j * 32 < end ? load_once(body + i + j * 32) : Vec<T>::nothing();
    add_vectors<T, CAP, ENT, LP_PART_FLIGHT>(acc, v, (end - i - lane + 31) / 32, a.k2, a.inv_cap);
  }
  if (parts == 1 && lane < row.extra()) add_value<CAP, ENT>(acc, Vec<T>::value(row.z[row.lone(lane)]), a.k2, a.inv_cap);
  join_warp<ENT>(acc, a.k2);
  if (lane != 0) return;
  if (parts == 1) row_results<T, CAP>(acc, row, r, label, a, logp, entropy, kept);
  else partial[unit] = acc;
}

// A warp per row joins its parts, and the values that are not in a vector.
template <typename T, bool CAP, bool ENT>
__global__ void __launch_bounds__(LP_PART_THREADS) logprob_join_kernel(const T* __restrict__ logits, const long long* __restrict__ labels,
                                                                       const Softmax* __restrict__ partial, float* __restrict__ logp,
                                                                       float* __restrict__ entropy, float4* __restrict__ kept,
                                                                       LogitRows a, int parts) {
  const long long r = blockIdx.x * static_cast<long long>(LP_PART_THREADS / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (r >= a.rows) return;
  grid_wait();
  const long long label = labels[r];
  if (a.ignored(label)) {
    if (lane == 0) ignored_row(r, logp, entropy, kept);
    return;
  }
  const Row<T> row(logits + a.offset(r), a.V);
  Softmax acc;
  if (lane < row.extra()) add_value<CAP, ENT>(acc, Vec<T>::value(row.z[row.lone(lane)]), a.k2, a.inv_cap);
  for (int i = lane; i < parts; i += 32) acc.join<ENT>(partial[r * parts + i], a.k2);
  join_warp<ENT>(acc, a.k2);
  if (lane == 0) row_results<T, CAP>(acc, row, r, label, a, logp, entropy, kept);
}

// A block takes LP_BACK_THREADS * LP_BACK_FLIGHT vectors of one row: small blocks that start with all their loads.  The gradient
// of the rows above (946 MB) takes 141 us, 6.7 TB/s; 512 threads with four vectors took 174, 128 with two 193, 64 with sixteen
// 151.  Streaming stores take 62 to 60 us off the gradient of 2934 rows of 32000.  A thread has read what it writes over before
// it writes, and no other thread reads that: the gradient may replace the logits.
template <typename T, bool CAP, bool ENT>
__global__ void __launch_bounds__(LP_BACK_THREADS) logprob_bwd_kernel(const T* logits, const long long* __restrict__ labels,
                                                                 const float4* __restrict__ kept, const float* __restrict__ grad_logp,
                                                                 const float* __restrict__ grad_entropy, T* grad,
                                                                 LogitRows a, long long grad_stride, int parts) {
  using W = Vec<T>;
  // (last rows first: the forward pass has left them in the L2)
  const unsigned unit = gridDim.x - 1 - blockIdx.x;
  const long long row = unit / parts;
  const int part = static_cast<int>(unit - row * parts);
  const long long label = labels[row];
  const T* z = logits + a.offset(row);
  T* d = grad + row * grad_stride;
  const float g = grad_logp ? grad_logp[row] : 0.f, h = ENT ? grad_entropy[row] : 0.f;
  const bool still = a.ignored(label) || (g == 0.f && h == 0.f);       // nothing flows back: the row is not read
  // vectors start on the boundaries of the gradient; logits that lie otherwise are read one by one
  const int head = min(a.V, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(d) & 15)) & 15) / static_cast<int>(sizeof(T)));
  const int vectors = (a.V - head) / W::N, tail = head + vectors * W::N;
  uint4* out = reinterpret_cast<uint4*>(d + head);
  const int first = part * (LP_BACK_THREADS * LP_BACK_FLIGHT) + static_cast<int>(threadIdx.x);
  const int extra = part == 0 ? a.V - vectors * W::N : 0;
  const int lone = static_cast<int>(threadIdx.x) < head ? threadIdx.x : tail + (threadIdx.x - head);
  if (still) {
#pragma unroll
    for (int j = 0; j < LP_BACK_FLIGHT; ++j)
      if (first + j * LP_BACK_THREADS < vectors) out[first + j * LP_BACK_THREADS] = make_uint4(0, 0, 0, 0);
    if (static_cast<int>(threadIdx.x) < extra) d[lone] = W::round(0.f);
    return;
  }
  const bool aligned = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0;
  const uint4* body = reinterpret_cast<const uint4*>(z + head);
  uint4 r[LP_BACK_FLIGHT];
  if (aligned) {
#pragma unroll
    for (int j = 0; j < LP_BACK_FLIGHT; ++j) {
      const int i = first + j * LP_BACK_THREADS;
      r[j] = i < vectors ? load_once(body + i) : make_uint4(0, 0, 0, 0);
    }
  }
  const float4 k = kept[row];
  const float m = k.x, f = a.k * (CAP ? 4.f * a.inv_cap : 1.f);     // (four quarters of a cap's slope)
  // f p (g + h (ln p + H)) = 2^u (flat + tilt u)
  const float tilt = ENT ? f * h * LN2 / k.y : 0.f, flat = f * (g + (ENT ? h * (k.z - logf(k.y)) : 0.f)) / k.y, fg = f * g;
  constexpr Slope SLOPE = sizeof(T) == 4 ? FINE : COARSE;
  auto slope_of = [&](float value, bool chosen) {
    Pair quarter(1.f, 1.f);
    const float u = exponent(capped2<CAP, SLOPE>(value, value, a.inv_cap, &quarter).get().x, m, a.k2);
    const float r = (chosen ? fg : 0.f) - fast_ex2(u) * (ENT ? flat + tilt * u : flat);
    return CAP ? quarter.get().x * r : r;
  };
  const int chosen = label >= head && label < a.V ? (static_cast<int>(label) - head) / W::N : -1;      // the label's vector
  const Pair minus(-m, -m), k2(a.k2, a.k2), flat2(-flat, -flat), tilt2(-tilt, -tilt);
  auto slope_of_two = [&](float x, float y) {
    Pair quarter(1.f, 1.f), t = (capped2<CAP, SLOPE>(x, y, a.inv_cap, &quarter) + minus) * k2;
    float2 u = t.get();
    if (ENT) {
      u.x = max_nan(u.x, LP_LOWEST), u.y = max_nan(u.y, LP_LOWEST);
      t = Pair(u.x, u.y);
    }
    const Pair r = Pair(fast_ex2(u.x), fast_ex2(u.y)) * (ENT ? fma2(tilt2, t, flat2) : flat2);
    return (CAP ? r * quarter : r).get();
  };
#pragma unroll
  for (int j = 0; j < LP_BACK_FLIGHT; ++j) {
    const int i = first + j * LP_BACK_THREADS;
    if (i >= vectors) break;
    float v[W::N], o[W::N];
    if (aligned) {
      W::unpack(r[j], v);
    } else {
#pragma unroll
      for (int e = 0; e < W::N; ++e) v[e] = W::value(z[head + i * W::N + e]);
    }
#pragma unroll
    for (int e = 0; e < W::N; e += 2) {
      const float2 t = slope_of_two(v[e], v[e + 1]);
      o[e] = t.x;
      o[e + 1] = t.y;
    }
    if (i == chosen) {
      const long long at = label - head - static_cast<long long>(i) * W::N;
#pragma unroll
      for (int e = 0; e < W::N; ++e)
        if (e == at) o[e] = slope_of(v[e], true);
    }
    __stcs(out + i, W::pack(o));
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

}  // namespace ts

using namespace ts;

TS_DEFINE_ERROR_API(ts_logprob)

// Parts of a row that warps of their own take; 0: a block or a cluster takes the row.  A row of one part always has a warp (4
// rows of 2000: 2.9 us, in blocks 3.2; 1200: 3.8 and 11).  Longer rows have blocks of their own while those are fewer than four
// to an SM, and need no second launch (rows of 128256 in blocks and in warps: 9.3 and 9.6 us for 100, 21.6 and 23.9 for 400, 33.3
// and 31.7 for 600; of 32000: 7.5 and 8.1, 8.4 and 9.7, 11.8 and 12.1).
static int row_parts(long long rows, long long V, int dtype) {
  const long long vectors = V * (dtype == 2 ? 4 : 2) / 16, parts = (vectors + LP_PART - 1) / LP_PART;
  return parts <= 1 ? 1 : rows < 4 * sm_count() ? 0 : static_cast<int>(parts);
}

// Fewer rows than these need no workspace.
extern "C" int ts_logprob_few_rows() { return 4 * sm_count(); }

// Bytes of workspace that ts_logprob_fwd needs.
extern "C" long long ts_logprob_workspace(long long rows, long long V, int dtype) {
  const int parts = row_parts(rows, V, dtype);
  return parts > 1 ? rows * parts * static_cast<long long>(sizeof(Softmax)) : 0;
}

// The arguments of a call, eight bytes each (ops/logprob.py packs them).  dtype: 0 bf16, 1 fp16, 2 fp32.  lenient: labels outside
// the vocabulary count as ignored; otherwise they give NaN.  kept: (m, S, H, unused) of every row, for the backward pass; H
// counts only with an entropy.  Forward: logp and, where they are not null, entropy and kept are results.  Backward: logp and
// entropy are what flows into them (null: zero), grad the result, its rows grad_stride elements apart; it may be the logits
// themselves, where their rows are.
struct LogprobCall {
  const void* logits;
  long long dtype;
  const long long* labels;
  float *logp, *entropy;
  float4* kept;
  void *workspace, *grad;
  long long grad_stride, rows, inner, stride_outer, stride_inner, V;
  double factor, cap;
  long long ignore, lenient;
};

static bool valid(const LogprobCall* c, long long units) {
  return c->rows > 0 && c->inner > 0 && c->V > 0 && c->V <= 0x7fffffffll && c->rows <= 0x7fffffffll / units && c->dtype >= 0 &&
         c->dtype <= 2;
}
static LogitRows logit_rows(const LogprobCall* c) {
  const double k = c->factor * (c->cap > 0.0 ? c->cap : 1.0);
  return {c->rows, c->inner, c->stride_outer, c->stride_inner, static_cast<int>(c->V), static_cast<float>(k),
          static_cast<float>(k * 1.4426950408889634), c->cap > 0.0 ? static_cast<float>(1.0 / c->cap) : 0.f, c->ignore,
          static_cast<int>(c->lenient)};
}

extern "C" int ts_logprob_fwd(const LogprobCall* c, void* stream) {
  constexpr int warps = LP_PART_THREADS / 32;
  const int dtype = static_cast<int>(c->dtype), units = row_parts(c->rows, c->V, dtype);
  if (!valid(c, units > LP_SPLIT ? units : LP_SPLIT)) return -1;
  const LogitRows a = logit_rows(c);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_type(dtype, c->cap > 0.0, c->entropy != nullptr, [&](auto* t, auto cap, auto e) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr bool CAP = decltype(cap)::value, ENT = decltype(e)::value;
    const T* z = static_cast<const T*>(c->logits);
    if (units) {
      Softmax* partial = static_cast<Softmax*>(c->workspace);
      if (units > 1 && !partial) return -1;
      logprob_part_kernel<T, CAP, ENT><<<static_cast<unsigned>((a.rows * units + warps - 1) / warps), LP_PART_THREADS, 0, st>>>(
          z, c->labels, partial, c->logp, c->entropy, c->kept, a, units);
      if (units == 1) return static_cast<int>(cudaGetLastError());
      const int rc = static_cast<int>(cudaGetLastError());
      if (rc) return rc;
      const dim3 joining(static_cast<unsigned>((a.rows + warps - 1) / warps));
      return launch_chained(logprob_join_kernel<T, CAP, ENT>, joining, dim3(LP_PART_THREADS), 0, st, 1, true, z, c->labels,
                            partial, c->logp, c->entropy, c->kept, a, units);
    }
    int parts = 1;                       // of a cluster, each with a vector or two for every thread
    const long long vectors = c->V * static_cast<int>(sizeof(T)) / 16;
    while (parts < LP_SPLIT && a.rows * parts < 2 * sm_count() && vectors / parts >= 2 * LP_THREADS) parts *= 2;
    const dim3 blocks(static_cast<unsigned>(a.rows * parts));
    return launch_chained(logprob_row_kernel<T, CAP, ENT>, blocks, dim3(LP_THREADS), 0, st, parts, false, z, c->labels,
                          c->logp, c->entropy, c->kept, a);
  });
}

extern "C" int ts_logprob_bwd(const LogprobCall* c, void* stream) {
  const int dtype = static_cast<int>(c->dtype);
  const long long vectors = c->V * (dtype == 2 ? 4 : 2) / 16, parts = vectors / (LP_BACK_THREADS * LP_BACK_FLIGHT) + 1;
  if (!valid(c, parts) || !c->kept || c->grad_stride < c->V) return -1;
  const LogitRows a = logit_rows(c);
  return by_type(dtype, c->cap > 0.0, c->entropy != nullptr, [&](auto* t, auto cap, auto e) {
    using T = std::remove_pointer_t<decltype(t)>;
    logprob_bwd_kernel<T, decltype(cap)::value, decltype(e)::value>
        <<<static_cast<unsigned>(a.rows * parts), LP_BACK_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const T*>(c->logits), c->labels, c->kept, c->logp, c->entropy, static_cast<T*>(c->grad), a, c->grad_stride,
            static_cast<int>(parts));
    return static_cast<int>(cudaGetLastError());
  });
}
