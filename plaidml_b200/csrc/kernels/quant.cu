// Quantisation to 8-bit floats by blocks of 128:
//
//   scale = max(amax, 2^-100) / largest,   q = to_8_bits(x * (1 / scale))
//
// One read of x and one write of q: the values stay in registers between the block's maximum and the conversion.  All
// operations are IEEE ones in f32 (the two divisions are once per block), so that results are defined to the bit.
#include "quant.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "dependent_launch.h"

namespace pmlb {
namespace {

struct QuantParams {
  const void* x;
  const int32_t* source;   // rows to take, or null
  int source_rows, source_div;
  uint8_t* q;
  float* scale;
  int rows, cols;
  long long ldx, ldq, stride_x, stride_q, scale_row, scale_block, stride_scale;
  int vec_in, vec_out;     // four elements of x / sixteen bytes of q at a time
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

// Elements [0, n) of four from `src` on; the others 0.
template <class In>
__device__ __forceinline__ void load4(const In* src, int n, bool vec, float (&v)[4]) {
  if (n >= 4 && vec) {
    if constexpr (sizeof(In) == 4) {
      const float4 u = __ldg(reinterpret_cast<const float4*>(src));
      v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
    } else {
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(src));
      const In* e = reinterpret_cast<const In*>(&u);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = to_f32(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? to_f32(src[i]) : 0.f;
  }
}

template <bool E5M2>
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  constexpr __nv_fp8_interpretation_t kind = E5M2 ? __NV_E5M2 : __NV_E4M3;
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, kind);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, kind);
  return lo | hi << 16;
}

template <bool E5M2>
__device__ __forceinline__ float scale_of(float amax) {
  return __fdiv_rn(fmaxf(amax, 0x1p-100f), E5M2 ? 57344.f : 448.f);
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}

constexpr int kRowsThreads = 256, kRowsUnroll = 4;

// Blocks along a row: a warp takes four blocks at once, four elements per lane and block.
template <class In, bool E5M2>
__global__ void __launch_bounds__(kRowsThreads) quant_rows_kernel(const QuantParams p) {
  dependent_entry();
  const int lane = threadIdx.x & 31;
  const int blocks = (p.cols + 127) / 128, runs = (blocks + kRowsUnroll - 1) / kRowsUnroll;
  const long long job = static_cast<long long>(blockIdx.x) * (kRowsThreads / 32) + (threadIdx.x >> 5);
  const long long row = job / runs;
  if (row >= p.rows) return;
  const int first = static_cast<int>(job - row * runs) * kRowsUnroll, batch = blockIdx.y;
  long long from = row;
  if (p.source != nullptr) {
    const int pair = __ldg(p.source + row);
    from = pair < 0 ? -1 : pair / p.source_div;
    if (from >= p.source_rows) from = -1;
  }
  const In* x = static_cast<const In*>(p.x) + batch * p.stride_x + from * p.ldx;
  float v[kRowsUnroll][4];
#pragma unroll
  for (int u = 0; u < kRowsUnroll; ++u) {
    const int c = (first + u) * 128 + lane * 4;
    load4(x + c, from < 0 ? 0 : p.cols - c, p.vec_in, v[u]);
  }
#pragma unroll
  for (int u = 0; u < kRowsUnroll; ++u) {
    if (first + u >= blocks) break;
    const float amax = warp_max(fmaxf(fmaxf(fabsf(v[u][0]), fabsf(v[u][1])), fmaxf(fabsf(v[u][2]), fabsf(v[u][3]))));
    const float scale = scale_of<E5M2>(amax), inverse = __fdiv_rn(1.f, scale);
    const uint32_t bits = pack4<E5M2>(v[u][0] * inverse, v[u][1] * inverse, v[u][2] * inverse, v[u][3] * inverse);
    const int c = (first + u) * 128 + lane * 4;
    uint8_t* q = p.q + batch * p.stride_q + row * p.ldq + c;
    if (p.vec_out && c + 4 <= p.cols) {
      *reinterpret_cast<uint32_t*>(q) = bits;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (c + e < p.cols) q[e] = static_cast<uint8_t>(bits >> (8 * e));
      }
    }
    if (lane == 0) p.scale[batch * p.stride_scale + row * p.scale_row + (first + u) * p.scale_block] = scale;
  }
}

constexpr int kTileThreads = 256;

// The other forms: a tile of 128 x 128 in the registers of eight warps, 16 consecutive rows each, four columns per lane.  A lane
// thus holds 16 consecutive bytes of four of the transposed result's rows, which go through shared memory to be written in
// whole 128-byte rows.
template <class In, bool E5M2, bool COLUMNS, bool TRANSPOSED>
__global__ void __launch_bounds__(kTileThreads) quant_tile_kernel(const QuantParams p) {
  __shared__ float most[8][128];
  __shared__ uint4 turned[TRANSPOSED ? 128 * 8 : 1];   // [column][16-byte piece of its 128 rows], pieces permuted by the column
  dependent_entry();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, batch = blockIdx.z;
  const int row0 = blockIdx.y * 128 + warp * 16, col0 = blockIdx.x * 128 + lane * 4;
  const In* x = static_cast<const In*>(p.x) + batch * p.stride_x + row0 * p.ldx + col0;
  float v[16][4];
#pragma unroll
  for (int i = 0; i < 16; ++i) load4(x + i * p.ldx, row0 + i < p.rows ? p.cols - col0 : 0, p.vec_in, v[i]);
  float inverse[4];
  float m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e) m[e] = fmaxf(m[e], fabsf(v[i][e]));
  }
  float* scale = p.scale + batch * p.stride_scale;
  if constexpr (COLUMNS) {
    *reinterpret_cast<float4*>(&most[warp][lane * 4]) = make_float4(m[0], m[1], m[2], m[3]);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const float4 u = *reinterpret_cast<const float4*>(&most[w][lane * 4]);
      m[0] = fmaxf(m[0], u.x), m[1] = fmaxf(m[1], u.y), m[2] = fmaxf(m[2], u.z), m[3] = fmaxf(m[3], u.w);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float s = scale_of<E5M2>(m[e]);
      inverse[e] = __fdiv_rn(1.f, s);
      if (warp == 0 && col0 + e < p.cols) scale[(col0 + e) * p.scale_row + blockIdx.y * p.scale_block] = s;
    }
  } else {
    const float mine = warp_max(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
    if (lane == 0) most[0][warp] = mine;
    __syncthreads();
    float all = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) all = fmaxf(all, most[0][w]);
    const float s = scale_of<E5M2>(all);
#pragma unroll
    for (int e = 0; e < 4; ++e) inverse[e] = __fdiv_rn(1.f, s);
    if (threadIdx.x == 0) scale[(TRANSPOSED ? blockIdx.x : blockIdx.y) * p.scale_row + (TRANSPOSED ? blockIdx.y : blockIdx.x) * p.scale_block] = s;
  }
  uint8_t* q = p.q + batch * p.stride_q;
  if constexpr (TRANSPOSED) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = pack4<E5M2>(v[4 * i][e] * inverse[e], v[4 * i + 1][e] * inverse[e], v[4 * i + 2][e] * inverse[e], v[4 * i + 3][e] * inverse[e]);
      }
      turned[(lane * 4 + e) * 8 + (warp ^ (lane & 7))] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __syncthreads();
    const int piece = threadIdx.x & 7, r0 = blockIdx.y * 128 + piece * 16;
    for (int c = threadIdx.x >> 3; c < 128; c += kTileThreads / 8) {
      const int col = blockIdx.x * 128 + c;
      if (col >= p.cols || r0 >= p.rows) continue;
      const uint4 u = turned[c * 8 + (piece ^ ((c >> 2) & 7))];
      uint8_t* dst = q + col * p.ldq + r0;
      if (p.vec_out && r0 + 16 <= p.rows) {
        *reinterpret_cast<uint4*>(dst) = u;
      } else {
        const uint32_t words[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (r0 + i < p.rows) dst[i] = static_cast<uint8_t>(words[i / 4] >> (8 * (i % 4)));
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (row0 + i >= p.rows) break;
      const uint32_t bits = pack4<E5M2>(v[i][0] * inverse[0], v[i][1] * inverse[1], v[i][2] * inverse[2], v[i][3] * inverse[3]);
      uint8_t* dst = q + (row0 + i) * p.ldq + col0;
      if (p.vec_out && col0 + 4 <= p.cols) {
        *reinterpret_cast<uint32_t*>(dst) = bits;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (col0 + e < p.cols) dst[e] = static_cast<uint8_t>(bits >> (8 * e));
        }
      }
    }
  }
}

template <class In, bool E5M2>
cudaError_t launch_typed(const pmlb_quant_desc& d, const QuantParams& p, cudaStream_t stream) {
  if (d.form == PMLB_QUANT_ROWS) {
    const long long runs = ((p.cols + 127) / 128 + kRowsUnroll - 1) / kRowsUnroll;
    const long long grid = (runs * p.rows + kRowsThreads / 32 - 1) / (kRowsThreads / 32);
    return launch_dependent(quant_rows_kernel<In, E5M2>, dim3(static_cast<unsigned>(grid), d.batch), kRowsThreads, stream, p);
  }
  const dim3 grid((p.cols + 127) / 128, (p.rows + 127) / 128, d.batch);
  switch (d.form) {
    case PMLB_QUANT_COLUMNS: return launch_dependent(quant_tile_kernel<In, E5M2, true, true>, grid, kTileThreads, stream, p);
    case PMLB_QUANT_TILES: return launch_dependent(quant_tile_kernel<In, E5M2, false, false>, grid, kTileThreads, stream, p);
    default: return launch_dependent(quant_tile_kernel<In, E5M2, false, true>, grid, kTileThreads, stream, p);
  }
}

template <class In>
cudaError_t launch_from(const pmlb_quant_desc& d, const QuantParams& p, cudaStream_t stream) {
  return d.out_dtype == PMLB_F8E5M2 ? launch_typed<In, true>(d, p, stream) : launch_typed<In, false>(d, p, stream);
}

}  // namespace

cudaError_t launch_quant(const pmlb_quant_desc& d, const void* x, const int32_t* rows, void* q, float* scale, cudaStream_t stream) {
  QuantParams p{};
  p.x = x;
  p.source = d.source_rows > 0 ? rows : nullptr;
  p.source_rows = d.source_rows, p.source_div = d.source_div;
  p.q = static_cast<uint8_t*>(q), p.scale = scale;
  p.rows = d.rows, p.cols = d.cols;
  p.ldx = d.ldx, p.ldq = d.ldq, p.stride_x = d.stride_x, p.stride_q = d.stride_q;
  p.scale_row = d.scale_row, p.scale_block = d.scale_block, p.stride_scale = d.stride_scale;
  const int eb = d.in_dtype == PMLB_F32 ? 4 : 2;
  const long long batched = d.batch > 1 ? 1 : 0;
  p.vec_in = reinterpret_cast<uintptr_t>(x) % (4 * eb) == 0 && d.ldx % 4 == 0 && (batched * d.stride_x) % 4 == 0;
  const int wide = d.form == PMLB_QUANT_COLUMNS || d.form == PMLB_QUANT_TILES_TRANSPOSED ? 16 : 4;
  p.vec_out = reinterpret_cast<uintptr_t>(q) % wide == 0 && d.ldq % wide == 0 && (batched * d.stride_q) % wide == 0;
  if (d.in_dtype == PMLB_F32) return launch_from<float>(d, p, stream);
  return d.in_dtype == PMLB_BF16 ? launch_from<__nv_bfloat16>(d, p, stream) : launch_from<__half>(d, p, stream);
}

}  // namespace pmlb
