// Weighted sums of the experts' rows of each token, and their gradients:
//
//   out[t] = sum_j w[t, j] * y[position[t, j]]
//   dy[position[t, j]] = w[t, j] * dout[t],   dw[t, j] = <dout[t], y[position[t, j]]>
//
// Bound by memory: each row of y is read once, each row of out (dout) written (read) once.  A block takes one token, a thread 16
// bytes of a row at a time; what keeps the memory busy is that a thread's loads of up to eight rows are on their way
// together, so they are not made conditional: a pair without a row reads row 0 and leaves it out.
#include "combine.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "dependent_launch.h"

namespace pmlb {
namespace {

constexpr int kThreads = 256, kGradThreads = 128;
constexpr int kRowsPerWarp = 4;

struct CombineParams {
  const void *y, *dout;
  const float* weights;
  const int32_t *position, *source;
  void *out, *dy;
  float* dweights;
  int tokens, top_k, width, rows, row_blocks;
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

// N elements: 16 bytes, or as many as the rows' alignment allows (then a thread has more places of a row at a time, strips of
// a block's width apart, so that as much is on its way).
template <class T, int N>
struct __align__(sizeof(T) * N) Pack {
  T e[N];
};

template <class P>
__device__ __forceinline__ P load_once(const void* at) {   // (whole pieces are read once: no place in L1)
  if constexpr (sizeof(P) == 16) {
    uint4 u;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(at));
    return *reinterpret_cast<const P*>(&u);
  } else {
    return *static_cast<const P*>(at);
  }
}

template <class T, int N>
struct Strips {
  static constexpr int kBytes = N * static_cast<int>(sizeof(T)), value = kBytes >= 16 ? 1 : (kBytes == 8 ? 2 : 4);
};

// Adds U of the token's rows, from choice j on, to the sums of this thread's columns: N from c on, and N more every `step`.
template <class T, int N, int S, int U>
__device__ __forceinline__ void add_rows(const CombineParams& p, const int32_t* position, const float* weights, int j, int c, int step,
                                         float (&sum)[S][N]) {
  using P = Pack<T, N>;
  P row[U][S];
  float w[U];
  bool there[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int r = __ldg(position + j + u);
    there[u] = static_cast<unsigned>(r) < static_cast<unsigned>(p.rows);
    const T* y = static_cast<const T*>(p.y) + (there[u] ? r * p.ldy : 0);
#pragma unroll
    for (int s = 0; s < S; ++s) row[u][s] = load_once<P>(y + (s == 0 || c + s * step < p.width ? c + s * step : c));
    w[u] = weights != nullptr ? __ldg(weights + j + u) : 1.f;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float v = fmaf(w[u], Elem<T>::get(row[u][s].e[e]), sum[s][e]);
        sum[s][e] = there[u] ? v : sum[s][e];
      }
    }
  }
}

template <class T, int N>
__global__ void __launch_bounds__(kThreads) combine_kernel(const CombineParams p) {
  constexpr int S = Strips<T, N>::value, kStep = kThreads * N;
  dependent_entry();
  const long long t = blockIdx.x;
  const int32_t* position = p.position + t * p.top_k;
  const float* weights = p.weights != nullptr ? p.weights + t * p.top_k : nullptr;
  T* out = static_cast<T*>(p.out) + t * p.ldo;
  for (int c = threadIdx.x * N; c < p.width; c += S * kStep) {
    float sum[S][N];
#pragma unroll
    for (int s = 0; s < S; ++s) {
#pragma unroll
      for (int e = 0; e < N; ++e) sum[s][e] = 0.f;
    }
    int j = p.rows > 0 ? 0 : p.top_k;   // (without rows there is nothing to read, not even row 0)
    for (; j + 8 <= p.top_k; j += 8) add_rows<T, N, S, 8>(p, position, weights, j, c, kStep, sum);
    if (j + 4 <= p.top_k) add_rows<T, N, S, 4>(p, position, weights, j, c, kStep, sum), j += 4;
    if (j + 2 <= p.top_k) add_rows<T, N, S, 2>(p, position, weights, j, c, kStep, sum), j += 2;
    if (j < p.top_k) add_rows<T, N, S, 1>(p, position, weights, j, c, kStep, sum);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s > 0 && c + s * kStep >= p.width) break;
      Pack<T, N> o;
#pragma unroll
      for (int e = 0; e < N; ++e) o.e[e] = Elem<T>::put(sum[s][e]);
      *reinterpret_cast<Pack<T, N>*>(out + c + s * kStep) = o;
    }
  }
}

// The gradients of U of token t's choices, from choice j on.  `part`: [warps][8] in shared memory.
template <class T, int N, int U>
__device__ __forceinline__ void grad_rows(const CombineParams& p, long long t, int j, float (*part)[8]) {
  using P = Pack<T, N>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* dout = static_cast<const T*>(p.dout) + t * p.ldo;
  const bool dots = p.dweights != nullptr && p.rows > 0;
  int at[U];
  float w[U], dot[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    at[u] = __ldg(p.position + t * p.top_k + j + u);
    w[u] = p.weights != nullptr ? __ldg(p.weights + t * p.top_k + j + u) : 1.f;
    dot[u] = 0.f;
  }
  auto there = [&](int u) { return static_cast<unsigned>(at[u]) < static_cast<unsigned>(p.rows); };
  constexpr int S = Strips<T, N>::value, kStep = kGradThreads * N;
  for (int c0 = threadIdx.x * N; c0 < p.width; c0 += S * kStep) {
    P row[U][S], g[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int c = s == 0 || c0 + s * kStep < p.width ? c0 + s * kStep : c0;
      g[s] = load_once<P>(dout + c);
      if (dots) {
#pragma unroll
        for (int u = 0; u < U; ++u) row[u][s] = load_once<P>(static_cast<const T*>(p.y) + (there(u) ? at[u] * p.ldy : 0) + c);
      }
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int c = c0 + s * kStep;
      if (s > 0 && c >= p.width) break;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (dots) {
#pragma unroll
          for (int e = 0; e < N; ++e) dot[u] = fmaf(Elem<T>::get(g[s].e[e]), Elem<T>::get(row[u][s].e[e]), dot[u]);
        }
        if (p.dy != nullptr && there(u)) {
          P o;
#pragma unroll
          for (int e = 0; e < N; ++e) o.e[e] = Elem<T>::put(w[u] * Elem<T>::get(g[s].e[e]));
          *reinterpret_cast<P*>(static_cast<T*>(p.dy) + at[u] * p.ldy + c) = o;
        }
      }
    }
  }
  if (p.dweights == nullptr) return;
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], d);
  }
  __syncthreads();   // (the sums of the choices before have been read)
  if (lane == 0) {
#pragma unroll
    for (int u = 0; u < U; ++u) part[warp][u] = there(u) ? dot[u] : 0.f;
  }
  __syncthreads();
  if (threadIdx.x < U) {
    float all = 0.f;
#pragma unroll
    for (int i = 0; i < kGradThreads / 32; ++i) all += part[i][threadIdx.x];
    p.dweights[t * p.top_k + j + threadIdx.x] = all;
  }
}

// Blocks [0, row_blocks): zeros for rows that no pair has (first, and few rows per warp: the rows behind the last segment lie
// together, and a warp with many of them would end long after the others).  The others: a token each.
template <class T, int N>
__global__ void __launch_bounds__(kGradThreads) combine_grad_kernel(const CombineParams p) {
  using P = Pack<T, N>;
  __shared__ float part[kGradThreads / 32][8];
  dependent_entry();
  if (blockIdx.x < static_cast<unsigned>(p.row_blocks)) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r0 = (blockIdx.x * (kGradThreads / 32) + warp) * kRowsPerWarp;
    const bool mine = lane < kRowsPerWarp && r0 + lane < p.rows;
    const int pair = mine ? __ldg(p.source + r0 + lane) : 0;
    unsigned empty = __ballot_sync(0xffffffffu, mine && static_cast<unsigned>(pair) >= static_cast<unsigned>(p.tokens) * p.top_k);
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
  const long long t = blockIdx.x - p.row_blocks;
  int j = 0;
  for (; j + 8 <= p.top_k; j += 8) grad_rows<T, N, 8>(p, t, j, part);
  if (j + 4 <= p.top_k) grad_rows<T, N, 4>(p, t, j, part), j += 4;
  if (j + 2 <= p.top_k) grad_rows<T, N, 2>(p, t, j, part), j += 2;
  if (j < p.top_k) grad_rows<T, N, 1>(p, t, j, part);
}

template <class T, int N>
cudaError_t launch_sized(CombineParams p, bool grad, cudaStream_t stream) {
  if (!grad) return launch_dependent(combine_kernel<T, N>, dim3(static_cast<unsigned>(p.tokens)), kThreads, stream, p);
  constexpr int kRows = kGradThreads / 32 * kRowsPerWarp;
  p.row_blocks = p.dy != nullptr ? (p.rows + kRows - 1) / kRows : 0;
  return launch_dependent(combine_grad_kernel<T, N>, dim3(static_cast<unsigned>(p.row_blocks + p.tokens)), kGradThreads, stream, p);
}

template <class T>
cudaError_t launch_typed(const CombineParams& p, bool grad, cudaStream_t stream) {
  // bytes that every row starts on and is made of
  const uintptr_t bits = reinterpret_cast<uintptr_t>(p.y) | reinterpret_cast<uintptr_t>(p.dout) | reinterpret_cast<uintptr_t>(p.out) |
                         reinterpret_cast<uintptr_t>(p.dy) | static_cast<uintptr_t>((p.width | p.ldy | p.ldo) * sizeof(T));
  if (bits % 16 == 0) return launch_sized<T, 16 / sizeof(T)>(p, grad, stream);
  if (bits % 8 == 0) return launch_sized<T, 8 / sizeof(T)>(p, grad, stream);
  if constexpr (sizeof(T) == 2) {
    if (bits % 4 == 0) return launch_sized<T, 2>(p, grad, stream);
  }
  return launch_sized<T, 1>(p, grad, stream);
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
