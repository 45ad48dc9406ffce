// Weighted sums of the experts' rows of each token, and their gradients:
//
//   out[t] = sum_j w[t, j] * y[position[t, j]]
//   dy[position[t, j]] = w[t, j] * dout[t],   dw[t, j] = <dout[t], y[position[t, j]]>
//
// Memory-bound: each row of y is read once, each row of out (dout) written (read) once.  A block takes one token; the rows of
// its choices are loaded together, 16 bytes per lane.
#include "combine.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "dependent_launch.h"

namespace pmlb {
namespace {

constexpr int kThreads = 128;
constexpr int kAtOnce = 4;   // rows in flight per thread

struct CombineParams {
  const void *y, *dout;
  const float* weights;
  const int32_t *position, *source;
  void *out, *dy;
  float* dweights;
  int tokens, top_k, width, rows;
  long long ldy, ldo;
};

template <class T>
struct Elem;
template <>
struct Elem<float> {
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<__half> {
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};

// N elements: 16 bytes, or one where rows are not aligned.
template <class T, int N>
struct __align__(sizeof(T) * N) Pack {
  T e[N];
};

template <class T, int N>
__global__ void __launch_bounds__(kThreads) combine_kernel(const CombineParams p) {
  using P = Pack<T, N>;
  dependent_entry();
  const long long t = blockIdx.x;
  const int32_t* position = p.position + t * p.top_k;
  const T* y = static_cast<const T*>(p.y);
  T* out = static_cast<T*>(p.out) + t * p.ldo;
  for (int c = threadIdx.x * N; c < p.width; c += kThreads * N) {
    float sum[N];
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] = 0.f;
    for (int j0 = 0; j0 < p.top_k; j0 += kAtOnce) {
      P row[kAtOnce];
      float w[kAtOnce];
      bool there[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int r = j0 + u < p.top_k ? __ldg(position + j0 + u) : -1;
        there[u] = static_cast<unsigned>(r) < static_cast<unsigned>(p.rows);
        if (there[u]) {
          row[u] = *reinterpret_cast<const P*>(y + r * p.ldy + c);
          w[u] = p.weights != nullptr ? __ldg(p.weights + t * p.top_k + j0 + u) : 1.f;
        }
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if (!there[u]) continue;
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = fmaf(w[u], Elem<T>::get(row[u].e[e]), sum[e]);
      }
    }
    P o;
#pragma unroll
    for (int e = 0; e < N; ++e) o.e[e] = Elem<T>::put(sum[e]);
    *reinterpret_cast<P*>(out + c) = o;
  }
}

// Blocks [0, tokens): a token's rows.  The blocks behind them write zeros to rows that no pair has.
template <class T, int N>
__global__ void __launch_bounds__(kThreads) combine_grad_kernel(const CombineParams p) {
  using P = Pack<T, N>;
  __shared__ float part[kThreads / 32];
  dependent_entry();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x >= static_cast<unsigned>(p.tokens)) {
    const long long pairs = static_cast<long long>(p.tokens) * p.top_k;
    const int r0 = (blockIdx.x - p.tokens) * kThreads + warp * 32;
    int pair = 0;
    if (r0 + lane < p.rows) pair = __ldg(p.source + r0 + lane);
    unsigned empty = __ballot_sync(0xffffffffu, r0 + lane < p.rows && (pair < 0 || pair >= pairs));
    P zero;
#pragma unroll
    for (int e = 0; e < N; ++e) zero.e[e] = Elem<T>::put(0.f);
    while (empty != 0) {
      const int r = r0 + __ffs(empty) - 1;
      empty &= empty - 1;
      for (int c = lane * N; c < p.width; c += 32 * N) *reinterpret_cast<P*>(static_cast<T*>(p.dy) + r * p.ldy + c) = zero;
    }
    return;
  }
  const long long t = blockIdx.x;
  const T* dout = static_cast<const T*>(p.dout) + t * p.ldo;
  for (int j = 0; j < p.top_k; ++j) {
    const int r = __ldg(p.position + t * p.top_k + j);
    const bool there = static_cast<unsigned>(r) < static_cast<unsigned>(p.rows);
    const float w = p.weights != nullptr ? __ldg(p.weights + t * p.top_k + j) : 1.f;
    float dot = 0.f;
    if (there) {
      for (int c = threadIdx.x * N; c < p.width; c += kThreads * N) {
        const P g = *reinterpret_cast<const P*>(dout + c);
        if (p.dweights != nullptr) {
          const P v = *reinterpret_cast<const P*>(static_cast<const T*>(p.y) + r * p.ldy + c);
#pragma unroll
          for (int e = 0; e < N; ++e) dot = fmaf(Elem<T>::get(g.e[e]), Elem<T>::get(v.e[e]), dot);
        }
        if (p.dy != nullptr) {
          P o;
#pragma unroll
          for (int e = 0; e < N; ++e) o.e[e] = Elem<T>::put(w * Elem<T>::get(g.e[e]));
          *reinterpret_cast<P*>(static_cast<T*>(p.dy) + r * p.ldy + c) = o;
        }
      }
    }
    if (p.dweights != nullptr) {
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
      __syncthreads();
      if (lane == 0) part[warp] = dot;
      __syncthreads();
      if (threadIdx.x == 0) {
        float all = 0.f;
        for (int i = 0; i < kThreads / 32; ++i) all += part[i];
        p.dweights[t * p.top_k + j] = all;
      }
    }
  }
}

template <class T>
cudaError_t launch_typed(const CombineParams& p, bool grad, cudaStream_t stream) {
  constexpr int kWide = 16 / sizeof(T);
  auto aligned = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
  const bool wide = p.width % kWide == 0 && p.ldy % kWide == 0 && p.ldo % kWide == 0 && aligned(p.y) && aligned(p.dout) && aligned(p.out) &&
                    aligned(p.dy);
  unsigned grid = static_cast<unsigned>(p.tokens);
  if (!grad) return launch_dependent(wide ? combine_kernel<T, kWide> : combine_kernel<T, 1>, dim3(grid), kThreads, stream, p);
  if (p.dy != nullptr) grid += (p.rows + kThreads - 1) / kThreads;
  return launch_dependent(wide ? combine_grad_kernel<T, kWide> : combine_grad_kernel<T, 1>, dim3(grid), kThreads, stream, p);
}

cudaError_t launch_of(int dtype, const CombineParams& p, bool grad, cudaStream_t stream) {
  if (dtype == PMLB_F32) return launch_typed<float>(p, grad, stream);
  return dtype == PMLB_BF16 ? launch_typed<__nv_bfloat16>(p, grad, stream) : launch_typed<__half>(p, grad, stream);
}

CombineParams params_of(const pmlb_combine_desc& d) {
  CombineParams p{};
  p.tokens = d.tokens, p.top_k = d.top_k, p.width = d.width, p.rows = d.rows;
  p.ldy = d.ldy, p.ldo = d.ldo;
  return p;
}

}  // namespace

cudaError_t launch_combine(const pmlb_combine_desc& d, const void* y, const float* weights, const int32_t* position, void* out,
                           cudaStream_t stream) {
  CombineParams p = params_of(d);
  p.y = y, p.weights = weights, p.position = position, p.out = out;
  return launch_of(d.dtype, p, false, stream);
}

cudaError_t launch_combine_grad(const pmlb_combine_desc& d, const void* dout, const void* y, const float* weights,
                                const int32_t* position, const int32_t* source, void* dy, float* dweights, cudaStream_t stream) {
  CombineParams p = params_of(d);
  p.dout = dout, p.y = y, p.weights = weights, p.position = position, p.source = source, p.dy = dy, p.dweights = dweights;
  return launch_of(d.dtype, p, true, stream);
}

}  // namespace pmlb
