// Routing of tokens to experts.
//
// Choice: a warp per token, N consecutive experts in each lane's registers.  The top_k largest are taken one after another: a
// warp maximum of the lanes' best (redux), a vote for the lowest lane that holds it, and a new best in that lane.  Bound by
// instruction issue (a row of 256 logits is 1 KB; the choice of 8 of them some 600 instructions), so scores are computed with
// the hardware's approximate exponential and reciprocal.  Which of two near values is larger is a matter of rounding, so the
// choice is defined in 64 bits: where any two values that it hangs on are nearer than twice the error of a 32-bit score, the
// token's choice is made again in 64 bits (less than one token in a hundred of a usual batch).
//
// Order: one cluster counts the pairs of each expert (a histogram per warp, which also ranks them), adds the counts up over warps
// and CTAs (distributed shared memory), and each thread turns its pairs' ranks into rows, so that rows follow from the ids
// alone: no scratch, no atomics on global memory, one launch.
#include "route.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "dependent_launch.h"

namespace pmlb {
namespace {

constexpr int kRouteWarps = 4;
constexpr unsigned kAll = 0xffffffffu;
constexpr float kNoScore = -709.f;   // sigmoids of logits below are 0: in 64 bits, too, e^-z is infinite soon after
constexpr float kLog2e = 1.4426950408889634f;

struct RouteParams {
  const void* logits;
  const float* bias;
  float* weights;
  int32_t* ids;
  const int32_t* chosen;
  const float* dweights;
  void* dlogits;
  int tokens, experts, top_k, sigmoid, groups, top_groups, group_size, renormalise;
  int lanes_per_group;   // groups of whole lanes, a power of two of them; else 0
  int vec, vec_out, vec_bias;   // a lane's logits are loaded / gradients stored / biases loaded at once
  float scale;
  long long ld;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (sizeof(T) == 4) {
    return v;
  } else if constexpr (std::is_same<T, __half>::value) {
    return __float2half_rn(v);
  } else {
    return __float2bfloat16_rn(v);
  }
}

// A logit as it counts: NaN as minus infinity, plus infinity as the largest number.
__device__ __forceinline__ float logit(float z) { return fminf(fmaxf(z, -INFINITY), FLT_MAX); }   // (of a number and NaN, the number)

__device__ __forceinline__ float exp2_fast(float x) {   // relative error below 2^-22
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float reciprocal_fast(float x) {   // one unit in the last place
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <class F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kAll, v, d);
  return v;
}
// The larger of two, NaN only if both are.
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return a >= b || b != b ? a : b; }
__device__ __forceinline__ float smaller(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ double smaller(double a, double b) { return a <= b || b != b ? a : b; }

__device__ __forceinline__ float warp_max(float v) {   // (NaN does not count)
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(v));
  return y;
}
// By integers of the same order, the upper half first: two reductions in hardware where shuffles would be ten.
__device__ __forceinline__ double warp_max(double v) {
  const unsigned long long bits = static_cast<unsigned long long>(__double_as_longlong(v));
  const unsigned long long key = v != v ? 0ull : ((bits >> 63) != 0 ? ~bits : bits | (1ull << 63));
  const unsigned hi = static_cast<unsigned>(key >> 32), lo = static_cast<unsigned>(key);
  const unsigned top = __reduce_max_sync(kAll, hi), low = __reduce_max_sync(kAll, hi == top ? lo : 0u);
  const unsigned long long most = static_cast<unsigned long long>(top) << 32 | low;
  return __longlong_as_double(static_cast<long long>((most >> 63) != 0 ? most & ~(1ull << 63) : ~most));
}

// Scores of the row; -infinity scores 0 whatever the others are.
template <int N>
__device__ __forceinline__ void scores(const RouteParams& p, const float (&z)[N], float (&s)[N]) {
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = reciprocal_fast(1.f + exp2_fast(-kLog2e * z[i]));
    return;
  }
  float m = z[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, z[i]);
  m = fmaxf(warp_max(m), -FLT_MAX);   // (nothing but -infinity: every exponential is 0)
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s[i] = exp2_fast((z[i] - m) * kLog2e);
    sum += s[i];
  }
  sum = warp_sum(sum);
  const float r = sum > 0.f ? reciprocal_fast(sum) : 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] *= r;
}
template <int N>
__device__ __forceinline__ void scores(const RouteParams& p, const float (&z)[N], double (&s)[N]) {
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = 1.0 / (1.0 + exp(-static_cast<double>(z[i])));
    return;
  }
  float m = z[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, z[i]);
  m = fmaxf(warp_max(m), -FLT_MAX);
  double sum = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s[i] = exp(static_cast<double>(z[i]) - static_cast<double>(m));
    sum += s[i];
  }
  sum = warp_sum(sum);
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = sum > 0 ? s[i] / sum : 0.0;
}

// The token's experts: lane j gets the j-th choice.  Returns whether the choice hangs on values nearer than `F`'s errors.  `row`:
// room for a row in shared memory, used by groups that are not made of whole lanes.
template <class F, int N>
__device__ __forceinline__ bool choose(const RouteParams& p, const float (&z)[N], F* row, int lane, int* mine) {
  constexpr bool kExact = sizeof(F) == 8;
  const F kNone = -INFINITY, kTaken = NAN;
  const bool plain = p.bias == nullptr && p.groups == 1;   // the logits themselves: nothing is rounded
  const int held = min(max(p.experts - lane * N, 0), N);   // experts of this lane
  bool close = false;
  F r[N];
  // How near two values may be to be in either order, in units of u = 2^-24: `base`, and twice the larger one for the bias' rounding.
  // sigmoid 1 / (1 + e): e is off by 4 u (the exponential) and |z| u (its argument), which moves the score by s (1 - s) times
  // that, at most 1.4 u; the sum and the reciprocal by 3 u more.  softmax: 4 u, 2 d e^-d < 0.8 u for the argument, 37 u for a
  // sum of up to 1024 terms in chains of 32 and a tree of 5 (and 4 u of its terms), 3 u.  Twice that for two values.
  const F u = 0x1p-24f, base = (p.sigmoid ? 2 * 6 : 2 * 50) * u;
  if (plain) {
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = static_cast<F>(z[i]);
  } else {
    scores(p, z, r);
    if (p.bias != nullptr) {
      float b[N];
      if (p.vec_bias && held == N) {
        constexpr int kPiece = N < 4 ? N : 4;
#pragma unroll
        for (int i = 0; i < N; i += kPiece) {
          if constexpr (kPiece == 4) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(p.bias + lane * N + i));
            b[i] = v.x, b[i + 1] = v.y, b[i + 2] = v.z, b[i + 3] = v.w;
          } else {
            const float2 v = __ldg(reinterpret_cast<const float2*>(p.bias + lane * N + i));
            b[i] = v.x, b[i + 1] = v.y;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) b[i] = i < held ? __ldg(p.bias + lane * N + i) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = larger(r[i] + static_cast<F>(b[i]), kNone);   // (a bias that is NaN: never chosen)
    }
  }
  if (held < N) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i >= held) r[i] = kTaken;
    }
  }
  if (p.groups > 1) {
    F first = kNone, second = kNone;
    int group = lane, step = 1;   // the group whose value this lane holds, and the lanes between two groups' values
    if (p.lanes_per_group > 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        second = larger(smaller(r[i], first), second);
        first = larger(first, r[i]);
      }
      for (int d = 1; d < p.lanes_per_group; d <<= 1) {
        const F f = __shfl_xor_sync(kAll, first, d), s = __shfl_xor_sync(kAll, second, d);
        second = larger(smaller(f, first), larger(s, second));
        first = larger(f, first);
      }
      step = p.lanes_per_group;
      group = lane / step;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i < held) row[lane * N + i] = r[i];
      }
      __syncwarp();
      if (lane < p.groups) {
        for (int j = 0; j < p.group_size; ++j) {
          const F v = row[lane * p.group_size + j];
          second = larger(smaller(v, first), second);
          first = larger(first, v);
        }
      }
      __syncwarp();
    }
    const F value = larger(p.group_size > 1 ? first + second : first, kNone);
    int better = 0;
    for (int g = 0; g < p.groups; ++g) {
      const F v = __shfl_sync(kAll, value, g * step);
      better += v > value || (v == value && g < group);
    }
    const bool stays = group < p.groups && better < p.top_groups;
    if (!kExact && p.top_groups < p.groups) {
      // (a group's value: two scores, and a rounding of each bias and of the sum)
      F size = (first < 0 ? -first : first) + (p.group_size > 1 ? (second < 0 ? -second : second) : F(0));
      if (!(size < static_cast<F>(INFINITY))) size = 0;
      const F worst = -warp_max(stays ? -value : kNone), rest = warp_max(group < p.groups && !stays ? value : kNone);
      // (two infinities: sums of two large biases that 64 bits hold)
      close = !(worst - rest > 2 * base + 4 * u * warp_max(size));
    }
    // (the others' experts are taken, not minus infinity: that is what a bias may leave of an expert that stays)
    if (p.lanes_per_group > 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = stays ? r[i] : kTaken;
    } else {
      const unsigned kept = __ballot_sync(kAll, stays);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i < held && !((kept >> ((lane * N + i) / p.group_size)) & 1u)) r[i] = kTaken;
      }
    }
  }
  auto best = [&]() {
    F v = r[0];
#pragma unroll
    for (int i = 1; i < N; ++i) v = larger(v, r[i]);
    return v;
  };
  F v = best(), value_of_mine = 0;   // this lane's largest that is left, NaN for none; the value of the lane-th choice
  *mine = -1;
  // (the first one left out tells how near it was)
  const int picks = p.top_k + (kExact || plain || p.top_k == p.experts ? 0 : 1);
  F most = 0;
  for (int j = 0; j < picks; ++j) {
    most = warp_max(v);
    const int from = __ffs(__ballot_sync(kAll, v == most)) - 1;
    int at = 0;
    if (lane == from) {
      // the first of its registers that holds it is taken
      bool found = false;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool hit = !found && r[i] == most;
        if (hit) r[i] = kTaken, at = lane * N + i;
        found = found || hit;
      }
      v = best();
    }
    const int e = __shfl_sync(kAll, at, from);
    if (lane == j) *mine = e, value_of_mine = most;
  }
  if (!kExact && !plain) {
    // each choice with the one after it
    F next = __shfl_down_sync(kAll, value_of_mine, 1);
    if (lane == p.top_k - 1) next = most;   // (lane 31 has none after it)
    const F size = larger(value_of_mine < 0 ? -value_of_mine : value_of_mine, next < 0 ? -next : next);
    if (__any_sync(kAll, lane + 1 < picks && value_of_mine - next <= base + 2 * u * size)) close = true;
  }
  return close;
}

template <class T, int N>
__device__ __forceinline__ void load_row(const RouteParams& p, long long t, int lane, float (&z)[N]) {
  const T* row = static_cast<const T*>(p.logits) + t * p.ld + lane * N;
  constexpr int kBytes = N * sizeof(T);
  if (p.vec && lane * N + N <= p.experts) {
    T v[N];
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(v)[i] = __ldg(reinterpret_cast<const uint4*>(row) + i);
    } else if constexpr (kBytes == 8) {
      *reinterpret_cast<uint2*>(v) = __ldg(reinterpret_cast<const uint2*>(row));
    } else {
      *reinterpret_cast<uint32_t*>(v) = __ldg(reinterpret_cast<const uint32_t*>(row));
    }
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = logit(to_f32(v[i]));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = lane * N + i < p.experts ? logit(to_f32(row[i])) : -INFINITY;
  }
}

// The choice in 64 bits, for the tokens that need it.
template <class T, int N>
__device__ __noinline__ int choose_again(const RouteParams& p, long long t, int lane, double* row) {
  float z[N];
  load_row<T, N>(p, t, lane, z);
  int id;
  choose<double, N>(p, z, row, lane, &id);
  return id;
}

// e^(z - m), m >= z.  The difference's rounding is as much as |z - m| / 2 units of the last place of the exponential, so what it leaves
// out (Knuth's sum of two numbers: exact) goes into the result.
__device__ __forceinline__ float exp_between(float z, float m) {
  const float d = z - m, e = expf(d);
  const float back = d - z, rest = (z - (d - back)) - (m + back);
  return d > -128.f ? fmaf(e, rest, e) : e;   // (0 below; and the rest of an infinity is none)
}

// The chosen experts' weights before `scale`, lane j the j-th one's: scores over the row, or (renormalise) shares of the choice.
// `rest`: 1 - score for sigmoid.
template <class T, int N>
__device__ __forceinline__ float weight_of(const RouteParams& p, long long t, int lane, int id, const float (&z)[N], float* rest) {
  const bool mine = lane < p.top_k && static_cast<unsigned>(id) < static_cast<unsigned>(p.experts);
  const float zc = mine ? logit(to_f32(static_cast<const T*>(p.logits)[t * p.ld + id])) : -INFINITY;
  float w = 0.f;
  *rest = 0.f;
  if (p.sigmoid) {
    *rest = mine ? 1.f / (1.f + expf(zc)) : 0.f;
    if (!p.renormalise) return mine ? 1.f / (1.f + expf(-zc)) : 0.f;
    // Shares of scores that may all underflow in 32 bits: relative to e^m, m the largest logit or 0.
    const float m = fminf(warp_max(zc), 0.f);
    if (zc >= kNoScore) w = zc < 0.f ? exp_between(zc, m) / (1.f + expf(zc)) : 1.f / (1.f + expf(-zc));
  } else {
    float m = zc;
    if (!p.renormalise) {
#pragma unroll
      for (int i = 0; i < N; ++i) m = fmaxf(m, z[i]);
    }
    m = fmaxf(warp_max(m), -FLT_MAX);
    w = exp_between(zc, m);
    if (!p.renormalise) {
      // (the plain difference will do here: its rounding is worth u |z - m| of a term that is e^(z - m) of the sum or less)
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) sum += expf(z[i] - m);
      sum = warp_sum(sum);
      return sum > 0.f ? w / sum : 0.f;
    }
  }
  const float sum = warp_sum(w);
  return sum > 0.f ? w / sum : 0.f;
}

template <class T, int N>
__device__ __forceinline__ void route_token(const RouteParams& p, long long t, int lane, double* row) {
  float z[N];
  load_row<T, N>(p, t, lane, z);
  int id;
  if (choose<float, N>(p, z, reinterpret_cast<float*>(row), lane, &id)) id = choose_again<T, N>(p, t, lane, row);
  float rest;
  const float w = weight_of<T, N>(p, t, lane, id, z, &rest);
  if (lane < p.top_k) {
    p.weights[t * p.top_k + lane] = w * p.scale;
    p.ids[t * p.top_k + lane] = id;
  }
}

template <class T, int N>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const __grid_constant__ RouteParams p) {
  extern __shared__ double rows[];   // (groups that are not made of whole lanes) a row per warp
  dependent_entry();
  const int warp = threadIdx.x >> 5;
  const long long t = static_cast<long long>(blockIdx.x) * kRouteWarps + warp;
  if (t < p.tokens) route_token<T, N>(p, t, threadIdx.x & 31, rows + warp * p.experts);
}

// dz of w = scale * s_j, or scale * s_j / sum of the chosen s:
//   softmax              s_i (ds_i - sum_j ds_j s_j)          renormalised, the chosen alone:  q_j (g_j - sum g q)
//   sigmoid, chosen      s_j (1 - s_j) ds_j                   renormalised:                    q_j (1 - s_j) (g_j - sum g q)
// with g = scale * dw, q = w / scale.  The row is put together in shared memory: what all logits get, then the chosen ones'.
template <class T, int N>
__global__ void __launch_bounds__(kRouteWarps * 32) route_grad_kernel(const __grid_constant__ RouteParams p) {
  __shared__ __align__(16) T rows[kRouteWarps][32 * N];
  dependent_entry();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long t = static_cast<long long>(blockIdx.x) * kRouteWarps + warp;
  if (t >= p.tokens) return;
  T* row = rows[warp];
  float z[N];
  load_row<T, N>(p, t, lane, z);
  int id = -1;
  float g = 0.f;
  if (lane < p.top_k) {
    id = __ldg(p.chosen + t * p.top_k + lane);
    if (static_cast<unsigned>(id) < static_cast<unsigned>(p.experts)) g = p.scale * __ldg(p.dweights + t * p.top_k + lane);
    else id = -1;
  }
  float mine, dot = 0.f, out[N];
  if (!p.sigmoid && !p.renormalise) {   // every logit has a gradient
    const float zc = id >= 0 ? logit(to_f32(static_cast<const T*>(p.logits)[t * p.ld + id])) : -INFINITY;
    float m = z[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, z[i]);
    m = fmaxf(warp_max(m), -FLT_MAX);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      out[i] = expf(z[i] - m);
      sum += out[i];
    }
    sum = warp_sum(sum);
    const float r = sum > 0.f ? 1.f / sum : 0.f;
    const float w = expf(zc - m) * r;
    dot = warp_sum(g * w);
    mine = w * (g - dot);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] *= -r * dot;
  } else {
    float rest;
    const float w = weight_of<T, N>(p, t, lane, id, z, &rest);
    if (p.renormalise) dot = warp_sum(g * w);
    mine = w * (g - dot);
    if (p.sigmoid) mine *= rest;
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) row[lane * N + i] = from_f32<T>(out[i]);
  __syncwarp();
  if (id >= 0) row[id] = from_f32<T>(mine);
  __syncwarp();
  T* dst = static_cast<T*>(p.dlogits) + t * p.ld;
  constexpr int kWide = 16 / sizeof(T);
  if (p.vec_out) {
    for (int e = lane * kWide; e < p.experts; e += 32 * kWide) *reinterpret_cast<uint4*>(dst + e) = *reinterpret_cast<const uint4*>(row + e);
  } else {
    for (int e = lane; e < p.experts; e += 32) dst[e] = row[e];
  }
}

// ---------------------------------------------------------------- order

constexpr int kOrderThreads = 1024, kOrderWarps = kOrderThreads / 32, kMaxExperts = 1024;
// Steps of 32 pairs whose ranks a warp keeps in registers; longer runs keep theirs in `position` and place their rows one by one.  (256
// experts, 16 CTAs: 65536 pairs 8.4 us, 131072, which is eight steps, 11.0, 131080 12.7, 262144 20.8, 524288 37.5.)
constexpr int kKeep = 8;

struct OrderParams {
  const int32_t* ids;
  int32_t *offsets, *source, *position;
  int pairs, experts, rows, align, ctas;
};

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

constexpr int kStaged = kKeep * kOrderThreads;   // pairs that a CTA puts in order in shared memory

// Of a CTA with kOrderThreads threads: dynamic shared memory of order_smem() bytes.
__device__ __forceinline__ void order_pairs(const OrderParams& p, uint32_t* counts) {
  // counts: [warp][expert], the warp's pairs, then those of the warps before
  __shared__ uint32_t totals[kMaxExperts];      // this CTA's pairs of each expert
  __shared__ uint32_t bases[kMaxExperts];       // row of this CTA's first pair
  __shared__ uint32_t firsts[kMaxExperts];      // its place among the CTA's pairs in order
  __shared__ uint32_t begins[kMaxExperts + 1], filled[kMaxExperts];   // segments: first row, pairs
  __shared__ uint32_t sums[2][kOrderWarps + 1];
  uint32_t* staged = counts + kOrderWarps * p.experts;                            // the CTA's pairs in order,
  uint16_t* staged_id = reinterpret_cast<uint16_t*>(staged + kStaged);            // and their experts
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = p.ctas > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  // runs of whole 32 pairs, one after another: CTA, then warp
  const int runs = p.ctas * kOrderWarps;
  const int steps = (p.pairs + 31) / 32;
  const int run = rank * kOrderWarps + warp;
  const int begin = static_cast<int>(static_cast<long long>(steps) * run / runs) * 32;
  const int end = min(static_cast<int>(static_cast<long long>(steps) * (run + 1) / runs) * 32, p.pairs);
  const bool in_registers = (steps + runs - 1) / runs <= kKeep;   // of every warp
  int kept[kKeep];   // ids, then rank << 10 | id, -1 for pairs without an expert
#pragma unroll
  for (int k = 0; k < kKeep; ++k) kept[k] = begin + k * 32 + lane < end ? p.ids[begin + k * 32 + lane] : -1;
  for (int e = threadIdx.x; e < kOrderWarps * p.experts; e += kOrderThreads) {
    counts[e] = 0;
    if (kOrderWarps * p.experts * 4 <= kStaged * 6) staged[e] = 0;
  }
  __syncthreads();
  uint32_t* my = counts + warp * p.experts;
  // Lanes of the same expert: each sets its bit in the expert's word of the warp (in the place of the staged pairs, which come
  // later), or, for more experts than there is room for, a vote per bit of the id.  (131072 pairs of 256 experts: 18.8 us with
  // match.any, 14.5 with votes, 11.6 with the words.)  Ranks stay below the 2^24 pairs divided by the 256 runs that more
  // than 1024 pairs are cut into: 16 bits.
  const bool by_words = kOrderWarps * p.experts * 4 <= kStaged * 6;
  uint32_t* words = staged + warp * p.experts;
  const int id_bits = 32 - __clz(p.experts);
  auto ranked = [&](int id) {
    const bool there = static_cast<unsigned>(id) < static_cast<unsigned>(p.experts);
    unsigned same = kAll;
    if (by_words) {
      if (there) atomicOr(words + id, 1u << lane);
      __syncwarp();
      if (there) same = words[id];
    } else {
      const int key = there ? id : p.experts;
      for (int b = 0; b < id_bits; ++b) {
        const bool bit = (key >> b) & 1;
        const unsigned m = __ballot_sync(kAll, bit);
        same &= bit ? m : ~m;
      }
    }
    uint32_t r = 0;
    if (there) r = my[id] + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (there && (same >> lane) == 1u) {   // the last lane of its expert
      my[id] = r + 1;
      if (by_words) words[id] = 0;
    }
    __syncwarp();
    return there ? static_cast<int>(r << 10 | static_cast<uint32_t>(id)) : -1;
  };
#pragma unroll
  for (int k = 0; k < kKeep; ++k) {
    if (begin + k * 32 < end) kept[k] = ranked(kept[k]);
  }
  for (int i0 = begin + kKeep * 32; i0 < end; i0 += 4 * 32) {
    int id[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) id[k] = i0 + k * 32 + lane < end ? p.ids[i0 + k * 32 + lane] : -1;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (i0 + k * 32 >= end) break;
      id[k] = ranked(id[k]);
      if (i0 + k * 32 + lane < end) p.position[i0 + k * 32 + lane] = id[k];
    }
  }
  __syncthreads();
  const int e = threadIdx.x;
  uint32_t here = 0;
  if (e < p.experts) {
#pragma unroll 8
    for (int w = 0; w < kOrderWarps; ++w) {
      const uint32_t c = counts[w * p.experts + e];
      counts[w * p.experts + e] = here;
      here += c;
    }
    totals[e] = here;
  }
  __syncwarp();
  if (p.ctas > 1) cluster_sync_all(); else __syncthreads();
  uint32_t ahead = 0, all = here;
  if (e < p.experts && p.ctas > 1) {
    all = 0;
#pragma unroll 4
    for (int c = 0; c < p.ctas; ++c) {
      const uint32_t v = ld_cluster_u32(mapa_rank(smem_u32(totals + e), static_cast<uint32_t>(c)));
      if (c < rank) ahead += v;
      all += v;
    }
  }
  // segments, one after another; and the CTA's own pairs
  const uint32_t align = static_cast<uint32_t>(p.align);
  const uint32_t length = (all + align - 1) / align * align;
  uint32_t x = length, y = here;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t a = __shfl_up_sync(kAll, x, d), b = __shfl_up_sync(kAll, y, d);
    if (lane >= d) x += a, y += b;
  }
  if (lane == 31) sums[0][warp] = x, sums[1][warp] = y;
  __syncthreads();
  if (warp < 2) {
    uint32_t s = sums[warp][lane];
    const uint32_t own = s;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t a = __shfl_up_sync(kAll, s, d);
      if (lane >= d) s += a;
    }
    sums[warp][lane] = s - own;
    if (lane == 31) sums[warp][kOrderWarps] = s;
  }
  __syncthreads();
  const uint32_t used = sums[0][kOrderWarps];
  if (e < p.experts) {
    const uint32_t b = sums[0][warp] + x - length;
    begins[e] = b, filled[e] = all, bases[e] = b + ahead;
    firsts[e] = sums[1][warp] + y - here;
    if (rank == 0) p.offsets[e] = static_cast<int32_t>(b);
  }
  if (threadIdx.x == 0) {
    begins[p.experts] = used;
    if (rank == 0) p.offsets[p.experts] = static_cast<int32_t>(used);
  }
  __syncthreads();
  if (in_registers) {
    // The CTA's pairs in order in shared memory first: rows of an expert then leave side by side (scattered straight from
    // the threads they are 8192 stores of their own per SM, 4 of 16 us for 131072 pairs).
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
      const int i = begin + k * 32 + lane;
      if (i >= end) break;
      int row = -1;
      if (kept[k] >= 0) {
        const int id = kept[k] & 1023;
        const uint32_t nth = my[id] + static_cast<uint32_t>(kept[k] >> 10);   // of the CTA's pairs of this expert
        row = static_cast<int>(bases[id] + nth);
        staged[firsts[id] + nth] = static_cast<uint32_t>(i);
        staged_id[firsts[id] + nth] = static_cast<uint16_t>(id);
      }
      p.position[i] = row;
    }
    __syncthreads();
    const uint32_t placed = sums[1][kOrderWarps];
    for (uint32_t s = threadIdx.x; s < placed; s += kOrderThreads) {
      const int id = staged_id[s];
      const uint32_t row = bases[id] + s - firsts[id];
      if (row < static_cast<uint32_t>(p.rows)) p.source[row] = static_cast<int32_t>(staged[s]);
    }
  } else {
    auto place = [&](int i, int packed) {
      int row = -1;
      if (packed >= 0) {
        const int id = packed & 1023;
        row = static_cast<int>(bases[id] + my[id] + static_cast<uint32_t>(packed >> 10));
        if (row < p.rows) p.source[row] = i;
      }
      p.position[i] = row;
    };
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
      if (begin + k * 32 + lane < end) place(begin + k * 32 + lane, kept[k]);
    }
#pragma unroll 4
    for (int i = begin + kKeep * 32 + lane; i < end; i += 32) place(i, p.position[i]);
  }
  // rows without a pair
  if (p.align > 1) {
    for (int s = run; s < p.experts; s += runs) {
      const uint32_t to = begins[s + 1];
      for (uint32_t r = begins[s] + filled[s] + lane; r < to; r += 32) {
        if (r < static_cast<uint32_t>(p.rows)) p.source[r] = -1;
      }
    }
  }
  for (long long r = static_cast<long long>(used) + rank * kOrderThreads + threadIdx.x; r < p.rows; r += p.ctas * kOrderThreads) p.source[r] = -1;
  __syncwarp();
  if (p.ctas > 1) cluster_sync_all();   // no CTA leaves while another may read its totals
}

__global__ void __launch_bounds__(kOrderThreads, 1) route_order_kernel(const OrderParams p) {
  extern __shared__ __align__(16) uint32_t order_smem_raw[];
  dependent_entry();
  order_pairs(p, order_smem_raw);
}

// Few tokens: one CTA chooses for them and puts the pairs in order, one launch instead of two.
template <class T, int N>
__global__ void __launch_bounds__(kOrderThreads, 1) route_few_kernel(const __grid_constant__ RouteParams p, const OrderParams q) {
  extern __shared__ __align__(16) uint32_t order_smem_raw[];   // (aligned for rows of doubles: the arrays before it end 4 mod 8)
  dependent_entry();
  // (the counts come after the choice: its rows may take their place)
  const int warp = threadIdx.x >> 5;
  for (long long t = warp; t < p.tokens; t += kOrderWarps) {
    route_token<T, N>(p, t, threadIdx.x & 31, reinterpret_cast<double*>(order_smem_raw) + warp * p.experts);
  }
  __syncthreads();
  order_pairs(q, order_smem_raw);
}

int order_smem(int experts) { return kOrderWarps * experts * 4 + kStaged * 6; }
int few_smem(int experts) { return std::max(order_smem(experts), kOrderWarps * experts * 8); }

// A kernel's shared-memory limit (and whether clusters of 16 may be launched), set once per device.
template <class Kernel>
cudaError_t prepare(Kernel kernel, int smem, std::atomic<uint64_t>* done, int dev) {
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done->load(std::memory_order_acquire) & bit) != 0) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) done->fetch_or(bit, std::memory_order_release);
  return e;
}

OrderParams order_of(const pmlb_route_desc& d, const int32_t* ids, int32_t* offsets, int32_t* source, int32_t* position) {
  OrderParams p{};
  p.ids = ids, p.offsets = offsets, p.source = source, p.position = position;
  p.pairs = d.tokens * d.top_k, p.experts = d.experts, p.rows = d.rows;
  p.align = std::max(d.align, 1);   // (not looked at where there are no rows)
  p.ctas = 1;
  return p;
}

enum Job { kChoose, kChooseAndOrder, kGradient };

template <class T, int N>
cudaError_t launch_sized(RouteParams p, const OrderParams& q, Job job, cudaStream_t stream) {
  const int lanes = p.group_size % N == 0 ? p.group_size / N : 0;
  p.lanes_per_group = (lanes & (lanes - 1)) == 0 ? lanes : 0;
  constexpr int kLaneBytes = N * static_cast<int>(sizeof(T)), kVec = kLaneBytes < 16 ? kLaneBytes : 16;
  p.vec = reinterpret_cast<uintptr_t>(p.logits) % kVec == 0 && p.ld * static_cast<int>(sizeof(T)) % kVec == 0;
  constexpr int kWide = 16 / sizeof(T);
  p.vec_bias = reinterpret_cast<uintptr_t>(p.bias) % (N < 4 ? 4 * N : 16) == 0;
  p.vec_out = reinterpret_cast<uintptr_t>(p.dlogits) % 16 == 0 && p.ld % kWide == 0 && p.experts % kWide == 0;
  cudaLaunchAttribute attr = dependent_launch_attribute();
  cudaLaunchConfig_t cfg = {};
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (job == kChooseAndOrder) {
    if constexpr (N <= 8) {
      int dev = 0;
      cudaGetDevice(&dev);
      static std::atomic<uint64_t> done{0};
      const cudaError_t e = prepare(route_few_kernel<T, N>, few_smem(32 * N), &done, dev);
      if (e != cudaSuccess) return e;
      cfg.gridDim = dim3(1);
      cfg.blockDim = dim3(kOrderThreads);
      cfg.dynamicSmemBytes = few_smem(p.experts);
      return cudaLaunchKernelEx(&cfg, route_few_kernel<T, N>, p, q);
    }
    return cudaErrorInvalidValue;
  }
  cfg.gridDim = dim3(static_cast<unsigned>((p.tokens + kRouteWarps - 1) / kRouteWarps));
  cfg.blockDim = dim3(kRouteWarps * 32);
  if (job == kGradient) return cudaLaunchKernelEx(&cfg, route_grad_kernel<T, N>, p);
  cfg.dynamicSmemBytes = p.groups > 1 && p.lanes_per_group == 0 ? kRouteWarps * p.experts * sizeof(double) : 0;
  return cudaLaunchKernelEx(&cfg, route_kernel<T, N>, p);
}

template <class T>
cudaError_t launch_typed(const RouteParams& p, const OrderParams& q, Job job, cudaStream_t stream) {
  if (p.experts <= 64) return launch_sized<T, 2>(p, q, job, stream);
  if (p.experts <= 128) return launch_sized<T, 4>(p, q, job, stream);
  if (p.experts <= 256) return launch_sized<T, 8>(p, q, job, stream);
  if (p.experts <= 512) return launch_sized<T, 16>(p, q, job, stream);
  return launch_sized<T, 32>(p, q, job, stream);
}

cudaError_t launch_of(int dtype, const RouteParams& p, const OrderParams& q, Job job, cudaStream_t stream) {
  if (dtype == PMLB_F32) return launch_typed<float>(p, q, job, stream);
  return dtype == PMLB_BF16 ? launch_typed<__nv_bfloat16>(p, q, job, stream) : launch_typed<__half>(p, q, job, stream);
}

// 16 CTAs if the device can hold such a cluster of the order kernel, else 8.
int largest_cluster(int dev) {
  static std::atomic<uint64_t> known{0}, sixteen{0};
  const uint64_t bit = 1ull << (dev & 63);
  if (dev >= 64) return 8;
  if ((known.load(std::memory_order_acquire) & bit) == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(16);
    cfg.blockDim = dim3(kOrderThreads);
    cfg.dynamicSmemBytes = order_smem(kMaxExperts);
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 16;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, route_order_kernel, &cfg) == cudaSuccess && n > 0) {
      sixteen.fetch_or(bit);
    } else {
      cudaGetLastError();
    }
    known.fetch_or(bit, std::memory_order_release);
  }
  return (sixteen.load() & bit) != 0 ? 16 : 8;
}

RouteParams params_of(const pmlb_route_desc& d, const void* logits) {
  RouteParams p{};
  p.logits = logits;
  p.tokens = d.tokens, p.experts = d.experts, p.top_k = d.top_k, p.sigmoid = d.score == PMLB_ROUTE_SIGMOID;
  p.groups = d.groups, p.top_groups = d.top_groups, p.group_size = d.experts / d.groups, p.renormalise = d.renormalise;
  p.scale = static_cast<float>(d.scale);
  p.ld = d.ld;
  return p;
}

}  // namespace

cudaError_t launch_route(const pmlb_route_desc& d, const void* logits, const float* bias, float* weights, int32_t* ids,
                         int32_t* offsets, int32_t* source, int32_t* position, cudaStream_t stream) {
  RouteParams p = params_of(d, logits);
  p.bias = bias, p.weights = weights, p.ids = ids;
  // (few: two tokens per warp at most, and rows of logits that leave a thread of such a large CTA its registers)
  if (d.rows > 0 && d.tokens <= 2 * kOrderWarps && d.experts <= 256) {
    return launch_of(d.dtype, p, order_of(d, ids, offsets, source, position), kChooseAndOrder, stream);
  }
  const cudaError_t e = launch_of(d.dtype, p, OrderParams{}, kChoose, stream);
  return e != cudaSuccess || d.rows == 0 ? e : launch_route_order(d, ids, offsets, source, position, stream);
}

cudaError_t launch_route_grad(const pmlb_route_desc& d, const void* logits, const int32_t* ids, const float* dweights, void* dlogits,
                              cudaStream_t stream) {
  RouteParams p = params_of(d, logits);
  p.chosen = ids, p.dweights = dweights, p.dlogits = dlogits;
  return launch_of(d.dtype, p, OrderParams{}, kGradient, stream);
}

cudaError_t launch_route_order(const pmlb_route_desc& d, const int32_t* ids, int32_t* offsets, int32_t* source, int32_t* position,
                               cudaStream_t stream) {
  int dev = 0;
  cudaGetDevice(&dev);
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = prepare(route_order_kernel, order_smem(kMaxExperts), &done, dev);
  if (e != cudaSuccess) return e;
  OrderParams p = order_of(d, ids, offsets, source, position);
  // One CTA for few pairs (one step per warp); else as many as a cluster may have here, 16 where the device allows it: 131072 pairs
  // then are kKeep steps per warp.
  p.ctas = p.pairs <= kOrderThreads ? 1 : largest_cluster(dev);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.ctas);
  cfg.blockDim = dim3(kOrderThreads);
  cfg.dynamicSmemBytes = order_smem(d.experts);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0] = dependent_launch_attribute();
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.ctas > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, route_order_kernel, p);
}

}  // namespace pmlb
