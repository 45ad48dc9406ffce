// Routing of tokens to experts.
//
// Choice: a warp per token, the row of logits in registers (expert 32 i + lane in register i of a lane).  The top_k largest
// are taken one after another by warp maxima.  Which of two near values is larger is a matter of rounding, so the choice is
// defined in 64 bits; it is made in 32 bits first, together with whether any two values that the choice hangs on are nearer
// than twice the error of a 32-bit score, and made again in 64 bits for the few tokens where they are.
//
// Order: one cluster counts the pairs of each expert (a histogram per warp), adds the counts up over warps and CTAs (distributed
// shared memory), and walks the pairs again in the same order, so that rows follow from the ids alone: no scratch, no
// atomics on global memory, one launch.
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

struct RouteParams {
  const void* logits;
  const float* bias;
  float* weights;
  int32_t* ids;
  const int32_t* chosen;
  const float* dweights;
  void* dlogits;
  int tokens, experts, top_k, sigmoid, groups, top_groups, group_size, renormalise;
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
__device__ __forceinline__ float logit(float z) { return z != z ? -INFINITY : fminf(z, FLT_MAX); }

__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }

template <class F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kAll, v, d);
  return v;
}
template <class F>
__device__ __forceinline__ F warp_max(F v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const F u = __shfl_xor_sync(kAll, v, d);
    v = u > v ? u : v;
  }
  return v;
}

// The largest (value, lowest index) of the warp's; lanes without one hold minus infinity and an index of INT_MAX.
template <class F>
__device__ __forceinline__ void warp_best(F& v, int& at) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const F u = __shfl_xor_sync(kAll, v, d);
    const int k = __shfl_xor_sync(kAll, at, d);
    if (u > v || (u == v && k < at)) v = u, at = k;
  }
}

// Scores of the row; -infinity scores 0 whatever the others are.
template <class F, int N>
__device__ __forceinline__ void scores(const RouteParams& p, const float (&z)[N], F (&s)[N]) {
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = F(1) / (F(1) + exp_of(-static_cast<F>(z[i])));
    return;
  }
  float m = z[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, z[i]);
  m = warp_max(m);
  F sum = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s[i] = z[i] == -INFINITY ? F(0) : exp_of(static_cast<F>(z[i]) - static_cast<F>(m));
    sum += s[i];
  }
  sum = warp_sum(sum);
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = sum > F(0) ? s[i] / sum : F(0);
}

// The token's experts: lane j gets the j-th choice.  Returns whether the choice hangs on values nearer than `F`'s errors.
template <class F, int N>
__device__ __forceinline__ bool choose(const RouteParams& p, const float (&z)[N], F* row, int lane, int* mine) {
  const bool exact = sizeof(F) == 8;
  const bool plain = p.bias == nullptr && p.groups == 1;   // the logits themselves: nothing is rounded
  bool close = false;
  F r[N];
  F near = 0;   // values this near may be in either order
  if (plain) {
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = static_cast<F>(z[i]);
  } else {
    scores(p, z, r);
    F top = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = 32 * i + lane;
      if (e >= p.experts) continue;
      if (p.bias != nullptr) r[i] += static_cast<F>(__ldg(p.bias + e));
      if (r[i] != r[i]) r[i] = -INFINITY;
      const F size = r[i] < 0 ? -r[i] : r[i];
      if (size > top && size < static_cast<F>(INFINITY)) top = size;
    }
    // (sigmoid: four roundings of 2^-24 relative to at most 1.  softmax: the exponent's rounding, at most 2^-24 d e^-d < 0.37 * 2^-24,
    // expf's two units, and a sum of up to 1024 terms in chains of 32 and a tree of 5: less than 45 roundings of 2^-24.  The bias:
    // one rounding of the sum.  Twice that for two values.)
    if (!exact) near = static_cast<F>((p.sigmoid ? 2 * 5 : 2 * 48) * 0x1p-24f) + 2 * warp_max(top) * static_cast<F>(0x1p-24f);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (32 * i + lane >= p.experts) r[i] = -INFINITY;
  }
  if (p.groups > 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (32 * i + lane < p.experts) row[32 * i + lane] = r[i];
    }
    __syncwarp();
    F first = -INFINITY, second = -INFINITY;
    if (lane < p.groups) {
      for (int j = 0; j < p.group_size; ++j) {
        const F v = row[lane * p.group_size + (j + lane) % p.group_size];   // (another bank for each lane)
        if (v > first) {
          second = first;
          first = v;
        } else if (v > second) {
          second = v;
        }
      }
    }
    __syncwarp();
    F value = p.group_size > 1 ? first + second : first;
    if (value != value) value = -INFINITY;
    int better = 0;
    for (int g = 0; g < p.groups; ++g) {
      const F v = __shfl_sync(kAll, value, g);
      better += v > value || (v == value && g < lane);
    }
    const bool stays = lane < p.groups && better < p.top_groups;
    const unsigned kept = __ballot_sync(kAll, stays);
    if (!exact && p.top_groups < p.groups) {
      const F worst = -warp_max(stays ? -value : static_cast<F>(-INFINITY)), rest = warp_max(lane < p.groups && !stays ? value : static_cast<F>(-INFINITY));
      close = worst - rest <= 2 * near;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = 32 * i + lane;
      if (e < p.experts && !((kept >> (e / p.group_size)) & 1u)) r[i] = -INFINITY;
    }
  }
  F last = 0;
  unsigned taken = 0;   // bit i: register i has been chosen
  *mine = -1;
  for (int j = 0; j < p.top_k + (exact || plain ? 0 : 1); ++j) {
    F v = -INFINITY;
    int at = 0x7fffffff;
#pragma unroll
    for (int i = N - 1; i >= 0; --i) {
      if (32 * i + lane < p.experts && !((taken >> i) & 1u) && r[i] >= v) v = r[i], at = 32 * i + lane;
    }
    warp_best(v, at);
    if (!exact && !plain && j > 0 && last - v <= near) close = true;
    last = v;
    if (j < p.top_k && lane == j) *mine = at;
    if (at != 0x7fffffff && (at & 31) == lane) taken |= 1u << (at >> 5);
  }
  return close;
}

template <class T, int N>
__device__ __forceinline__ void load_row(const RouteParams& p, long long t, int lane, float (&z)[N]) {
  const T* row = static_cast<const T*>(p.logits) + t * p.ld;
#pragma unroll
  for (int i = 0; i < N; ++i) z[i] = 32 * i + lane < p.experts ? logit(to_f32(row[32 * i + lane])) : -INFINITY;
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
    if (zc >= kNoScore) w = zc < 0.f ? expf(zc - m) / (1.f + expf(zc)) : 1.f / (1.f + expf(-zc));
  } else {
    float m = zc;
    if (!p.renormalise) {
#pragma unroll
      for (int i = 0; i < N; ++i) m = fmaxf(m, z[i]);
    }
    m = warp_max(m);
    w = zc == -INFINITY ? 0.f : expf(zc - m);
    if (!p.renormalise) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) sum += z[i] == -INFINITY ? 0.f : expf(z[i] - m);
      sum = warp_sum(sum);
      return sum > 0.f ? w / sum : 0.f;
    }
  }
  const float sum = warp_sum(w);
  return sum > 0.f ? w / sum : 0.f;
}

template <class T, int N>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const RouteParams p) {
  extern __shared__ double rows[];   // (groups) a row per warp
  dependent_entry();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long t = static_cast<long long>(blockIdx.x) * kRouteWarps + warp;
  if (t >= p.tokens) return;
  double* row = rows + warp * p.experts;
  float z[N];
  load_row<T, N>(p, t, lane, z);
  int id;
  if (choose<float, N>(p, z, reinterpret_cast<float*>(row), lane, &id)) choose<double, N>(p, z, row, lane, &id);
  float rest;
  const float w = weight_of<T, N>(p, t, lane, id, z, &rest);
  if (lane < p.top_k) {
    p.weights[t * p.top_k + lane] = w * p.scale;
    p.ids[t * p.top_k + lane] = id;
  }
}

// dz of w = scale * s_j, or scale * s_j / sum of the chosen s:
//   softmax              s_i (ds_i - sum_j ds_j s_j)          renormalised, the chosen alone:  q_j (g_j - sum g q)
//   sigmoid, chosen      s_j (1 - s_j) ds_j                   renormalised:                    q_j (1 - s_j) (g_j - sum g q)
// with g = scale * dw, q = w / scale.
template <class T, int N>
__global__ void __launch_bounds__(kRouteWarps * 32) route_grad_kernel(const RouteParams p) {
  dependent_entry();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long t = static_cast<long long>(blockIdx.x) * kRouteWarps + warp;
  if (t >= p.tokens) return;
  float z[N], s[N];
  load_row<T, N>(p, t, lane, z);
  int id = -1;
  float g = 0.f;
  if (lane < p.top_k) {
    id = __ldg(p.chosen + t * p.top_k + lane);
    if (static_cast<unsigned>(id) < static_cast<unsigned>(p.experts)) g = p.scale * __ldg(p.dweights + t * p.top_k + lane);
    else id = -1;
  }
  float rest;
  const float w = weight_of<T, N>(p, t, lane, id, z, &rest);
  const bool dense = !p.sigmoid && !p.renormalise;   // every logit has a gradient
  const float dot = p.renormalise || dense ? warp_sum(id >= 0 ? g * w : 0.f) : 0.f;
  float mine = id >= 0 ? w * (g - dot) : 0.f;
  if (p.sigmoid && id >= 0) mine *= rest;
  float out[N];
  if (dense) {
    scores(p, z, s);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = -s[i] * dot;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = 0.f;
  }
  for (int j = 0; j < p.top_k; ++j) {
    const int e = __shfl_sync(kAll, id, j);
    const float v = __shfl_sync(kAll, mine, j);
    if (e >= 0 && (e & 31) == lane) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i == e >> 5) out[i] = v;
      }
    }
  }
  T* dst = static_cast<T*>(p.dlogits) + t * p.ld;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (32 * i + lane < p.experts) dst[32 * i + lane] = from_f32<T>(out[i]);
  }
}

// ---------------------------------------------------------------- order

constexpr int kOrderThreads = 1024, kOrderWarps = kOrderThreads / 32, kMaxExperts = 1024;

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

__global__ void __launch_bounds__(kOrderThreads, 1) route_order_kernel(const OrderParams p) {
  extern __shared__ uint32_t counts[];          // [warp][expert]: pairs, then the row of the warp's next pair
  __shared__ uint32_t totals[kMaxExperts];      // this CTA's pairs of each expert
  __shared__ uint32_t begins[kMaxExperts], filled[kMaxExperts];   // segments: first row, pairs
  __shared__ uint32_t sums[kOrderWarps + 1];
  dependent_entry();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = p.ctas > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  // runs of whole 32 pairs, one after another: CTA, then warp
  const int runs = p.ctas * kOrderWarps;
  const int steps = (p.pairs + 31) / 32;
  const int run = rank * kOrderWarps + warp;
  const int begin = static_cast<int>(static_cast<long long>(steps) * run / runs) * 32;
  const int end = min(static_cast<int>(static_cast<long long>(steps) * (run + 1) / runs) * 32, p.pairs);
  for (int e = threadIdx.x; e < kOrderWarps * p.experts; e += kOrderThreads) counts[e] = 0;
  __syncthreads();
  uint32_t* my = counts + warp * p.experts;
  for (int i = begin + lane; i < end; i += 32) {
    const int e = __ldg(p.ids + i);
    if (static_cast<unsigned>(e) < static_cast<unsigned>(p.experts)) atomicAdd(my + e, 1u);
  }
  __syncthreads();
  const int e = threadIdx.x;
  if (e < p.experts) {
    uint32_t sum = 0;
    for (int w = 0; w < kOrderWarps; ++w) {
      const uint32_t c = counts[w * p.experts + e];
      counts[w * p.experts + e] = sum;
      sum += c;
    }
    totals[e] = sum;
  }
  __syncwarp();
  if (p.ctas > 1) cluster_sync_all(); else __syncthreads();
  uint32_t ahead = 0, all = 0;
  if (e < p.experts) {
    if (p.ctas > 1) {
      for (int c = 0; c < p.ctas; ++c) {
        const uint32_t v = ld_cluster_u32(mapa_rank(smem_u32(totals + e), static_cast<uint32_t>(c)));
        if (c < rank) ahead += v;
        all += v;
      }
    } else {
      all = totals[e];
    }
  }
  // segments, one after another
  const uint32_t align = static_cast<uint32_t>(p.align);
  const uint32_t length = (all + align - 1) / align * align;
  uint32_t x = length;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t y = __shfl_up_sync(kAll, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    uint32_t s = sums[lane];
    const uint32_t own = s;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t y = __shfl_up_sync(kAll, s, d);
      if (lane >= d) s += y;
    }
    sums[lane] = s - own;
    if (lane == 31) sums[kOrderWarps] = s;
  }
  __syncthreads();
  const uint32_t used = sums[kOrderWarps];
  if (e < p.experts) {
    const uint32_t b = sums[warp] + x - length;
    begins[e] = b, filled[e] = all;
    if (rank == 0) p.offsets[e] = static_cast<int32_t>(b);
    for (int w = 0; w < kOrderWarps; ++w) counts[w * p.experts + e] += b + ahead;
  }
  if (rank == 0 && threadIdx.x == 0) p.offsets[p.experts] = static_cast<int32_t>(used);
  __syncthreads();
  for (int i0 = begin; i0 < end; i0 += 32) {
    const int i = i0 + lane;
    int id = -1;
    if (i < end) id = __ldg(p.ids + i);
    const bool there = static_cast<unsigned>(id) < static_cast<unsigned>(p.experts);
    const unsigned same = __match_any_sync(kAll, there ? id : -1);
    uint32_t row = 0;
    if (there) row = my[id] + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (there && (same >> lane) == 1u) my[id] = row + 1;   // the last lane of its expert
    __syncwarp();
    if (i < end) {
      p.position[i] = there ? static_cast<int32_t>(row) : -1;
      if (there && row < static_cast<uint32_t>(p.rows)) p.source[row] = i;
    }
  }
  // rows without a pair
  for (int s = rank * kOrderWarps + warp; s < p.experts; s += runs) {
    const uint32_t from = begins[s] + filled[s], to = s + 1 < p.experts ? begins[s + 1] : used;
    for (uint32_t r = from + lane; r < to; r += 32) {
      if (r < static_cast<uint32_t>(p.rows)) p.source[r] = -1;
    }
  }
  for (long long r = static_cast<long long>(used) + rank * kOrderThreads + threadIdx.x; r < p.rows; r += p.ctas * kOrderThreads) p.source[r] = -1;
  __syncwarp();
  if (p.ctas > 1) cluster_sync_all();   // no CTA leaves while another may read its totals
}

template <class T, int N>
cudaError_t launch_sized(const RouteParams& p, bool grad, cudaStream_t stream) {
  cudaLaunchAttribute attr = dependent_launch_attribute();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((p.tokens + kRouteWarps - 1) / kRouteWarps));
  cfg.blockDim = dim3(kRouteWarps * 32);
  cfg.dynamicSmemBytes = !grad && p.groups > 1 ? kRouteWarps * p.experts * sizeof(double) : 0;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return grad ? cudaLaunchKernelEx(&cfg, route_grad_kernel<T, N>, p) : cudaLaunchKernelEx(&cfg, route_kernel<T, N>, p);
}

template <class T>
cudaError_t launch_typed(const RouteParams& p, bool grad, cudaStream_t stream) {
  if (p.experts <= 64) return launch_sized<T, 2>(p, grad, stream);
  if (p.experts <= 128) return launch_sized<T, 4>(p, grad, stream);
  if (p.experts <= 256) return launch_sized<T, 8>(p, grad, stream);
  if (p.experts <= 512) return launch_sized<T, 16>(p, grad, stream);
  return launch_sized<T, 32>(p, grad, stream);
}

cudaError_t launch_of(int dtype, const RouteParams& p, bool grad, cudaStream_t stream) {
  if (dtype == PMLB_F32) return launch_typed<float>(p, grad, stream);
  return dtype == PMLB_BF16 ? launch_typed<__nv_bfloat16>(p, grad, stream) : launch_typed<__half>(p, grad, stream);
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
                         cudaStream_t stream) {
  RouteParams p = params_of(d, logits);
  p.bias = bias, p.weights = weights, p.ids = ids;
  return launch_of(d.dtype, p, false, stream);
}

cudaError_t launch_route_grad(const pmlb_route_desc& d, const void* logits, const int32_t* ids, const float* dweights, void* dlogits,
                              cudaStream_t stream) {
  RouteParams p = params_of(d, logits);
  p.chosen = ids, p.dweights = dweights, p.dlogits = dlogits;
  return launch_of(d.dtype, p, true, stream);
}

cudaError_t launch_route_order(const pmlb_route_desc& d, const int32_t* ids, int32_t* offsets, int32_t* source, int32_t* position,
                               cudaStream_t stream) {
  OrderParams p{};
  p.ids = ids, p.offsets = offsets, p.source = source, p.position = position;
  p.pairs = d.tokens * d.top_k, p.experts = d.experts, p.rows = d.rows, p.align = d.align;
  p.ctas = p.pairs <= 4096 ? 1 : 8;
  const int smem = kOrderWarps * d.experts * 4;
  int dev = 0;
  cudaGetDevice(&dev);
  static std::atomic<uint64_t> done{0};
  const uint64_t bit = 1ull << (dev & 63);
  if (dev >= 64 || (done.load(std::memory_order_acquire) & bit) == 0) {
    const cudaError_t e = cudaFuncSetAttribute(route_order_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kOrderWarps * kMaxExperts * 4);
    if (e != cudaSuccess) return e;
    done.fetch_or(bit, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.ctas);
  cfg.blockDim = dim3(kOrderThreads);
  cfg.dynamicSmemBytes = smem;
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
