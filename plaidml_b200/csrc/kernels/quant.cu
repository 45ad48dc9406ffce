// Quantisation to 8-bit floats by blocks of 128:
//
//   scale = max(amax, 2^-100) / largest,   q = to_8_bits(x * (1 / scale))
//
// Bound by memory: one read of x and one write of q, the values staying in registers between the block's maximum and the
// conversion, eight elements (16 bytes of 16-bit ones) per lane and load.  All operations are those of IEEE f32 arithmetic, so
// that results are defined to the bit.
#include "quant.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cstring>
#include <type_traits>

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
  int vec_in, vec_out;     // eight elements of x / the bytes of q that a lane holds at a time
};

// Eight elements as they are stored.
template <class In>
struct Eight {
  uint4 raw[sizeof(In) / 2];

  // Elements [0, n) from `src` on; the others 0.
  __device__ __forceinline__ void load(const In* src, int n, bool vec) {
    if (n >= 8 && vec) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(In) / 2); ++i) raw[i] = __ldg(reinterpret_cast<const uint4*>(src) + i);
    } else if (sizeof(In) == 2 && n >= 8) {
      // rows that start anywhere: words, between two halves where the first one is not aligned
      const uint16_t* h = reinterpret_cast<const uint16_t*>(src);
      uint32_t w[4];
      if (reinterpret_cast<uintptr_t>(src) % 4 == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __ldg(reinterpret_cast<const uint32_t*>(h) + i);
      } else {
        const uint32_t *mid = reinterpret_cast<const uint32_t*>(h + 1), a = __ldg(mid), b = __ldg(mid + 1), c = __ldg(mid + 2);
        w[0] = __ldg(h) | a << 16;
        w[1] = a >> 16 | b << 16;
        w[2] = b >> 16 | c << 16;
        w[3] = c >> 16 | static_cast<uint32_t>(__ldg(h + 7)) << 16;
      }
      raw[0] = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      In v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < n ? src[i] : In(0.f);
      memcpy(raw, v, sizeof(raw));
    }
  }
  __device__ __forceinline__ uint32_t word(int i) const {
    const uint4& u = raw[i / 4];
    return i % 4 == 0 ? u.x : (i % 4 == 1 ? u.y : (i % 4 == 2 ? u.z : u.w));
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (sizeof(In) == 4) {
      return __uint_as_float(word(e));
    } else if constexpr (std::is_same<In, __nv_bfloat16>::value) {
      return __uint_as_float(e % 2 == 0 ? word(e / 2) << 16 : word(e / 2) & 0xffff0000u);
    } else {
      const uint32_t w = word(e / 2);
      const __half2 h = *reinterpret_cast<const __half2*>(&w);
      return e % 2 == 0 ? __low2float(h) : __high2float(h);
    }
  }
};

// The larger absolute values of pairs of words (two 16-bit elements, or one of 32 bits); NaN counts only beside NaN.
template <class In>
__device__ __forceinline__ uint32_t max_abs(uint32_t a, uint32_t b) {
  if constexpr (sizeof(In) == 4) {
    return __float_as_uint(fmaxf(fabsf(__uint_as_float(a)), fabsf(__uint_as_float(b))));
  } else {
    a &= 0x7fff7fffu, b &= 0x7fff7fffu;
    if constexpr (std::is_same<In, __nv_bfloat16>::value) {
      const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
      return *reinterpret_cast<const uint32_t*>(&m);
    } else {
      const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
      return *reinterpret_cast<const uint32_t*>(&m);
    }
  }
}

// The largest absolute value of a word's elements.
template <class In>
__device__ __forceinline__ float most_of(uint32_t w) {
  if constexpr (sizeof(In) == 4) {
    return fabsf(__uint_as_float(w));
  } else if constexpr (std::is_same<In, __nv_bfloat16>::value) {
    return fmaxf(__uint_as_float((w & 0x7fffu) << 16), __uint_as_float(w & 0x7fff0000u));
  } else {
    w &= 0x7fff7fffu;
    const __half2 h = *reinterpret_cast<const __half2*>(&w);
    return fmaxf(__low2float(h), __high2float(h));
  }
}

template <bool E5M2>
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  constexpr __nv_fp8_interpretation_t kind = E5M2 ? __NV_E5M2 : __NV_E4M3;
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, kind);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, kind);
  return lo | hi << 16;
}

// amax / largest, rounded to nearest: the quotient from the rounded reciprocal, corrected once by its remainder (Markstein 1990: with
// a correctly rounded reciprocal the correction gives the correctly rounded quotient): three operations.
template <bool E5M2>
__device__ __forceinline__ float scale_of(float amax) {
  constexpr float kLargest = E5M2 ? 57344.f : 448.f, kReciprocal = 1.f / kLargest;
  const float a = fmaxf(amax, 0x1p-100f);
  const float q = a * kReciprocal;
  const float exact = fmaf(fmaf(-q, kLargest, a), kReciprocal, q);
  return a == INFINITY ? a : exact;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}

__device__ __forceinline__ void store_bytes(uint8_t* q, uint32_t lo, uint32_t hi, int n) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (e < n) q[e] = static_cast<uint8_t>((e < 4 ? lo : hi) >> (8 * (e % 4)));
  }
}

constexpr int kRowWarps = 8;

// Blocks along a row: sixteen lanes per block, two blocks per load, UNROLL loads at once.  16-bit elements: 32 registers, so that
// the SM is full of warps (8192 x 4096 bf16 19.5 us, 20.5 with 46 registers; f32 elements need theirs: 27.6 us, 37 with 32).
template <class In, bool E5M2, int UNROLL>
__global__ void __launch_bounds__(kRowWarps * 32, sizeof(In) == 2 ? 8 : 1) quant_rows_kernel(const QuantParams p) {
  dependent_entry();
  const int lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5);
  if (row >= p.rows) return;
  const int batch = blockIdx.z, col0 = blockIdx.y * (UNROLL * 256) + lane * 8;
  long long from = row;
  if (p.source != nullptr) {
    const int pair = __ldg(p.source + row);
    from = pair < 0 ? -1 : pair / p.source_div;
    if (from >= p.source_rows) from = -1;
  }
  const In* x = static_cast<const In*>(p.x) + batch * p.stride_x + from * p.ldx;
  Eight<In> v[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) v[u].load(x + col0 + u * 256, from < 0 ? 0 : p.cols - col0 - u * 256, p.vec_in);
  float most[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    uint32_t m = max_abs<In>(v[u].word(0), v[u].word(1));
#pragma unroll
    for (int i = 2; i < static_cast<int>(2 * sizeof(In)); ++i) m = max_abs<In>(m, v[u].word(i));
    most[u] = most_of<In>(m);
  }
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) most[u] = fmaxf(most[u], __shfl_xor_sync(0xffffffffu, most[u], d));
  }
  uint8_t* q = p.q + batch * p.stride_q + row * p.ldq;
  float* scale = p.scale + batch * p.stride_scale + row * p.scale_row;
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const int c = col0 + u * 256;
    if (c >= p.cols) break;
    const float s = scale_of<E5M2>(most[u]), inverse = __frcp_rn(s);
    const uint32_t lo = pack4<E5M2>(v[u].get(0) * inverse, v[u].get(1) * inverse, v[u].get(2) * inverse, v[u].get(3) * inverse);
    const uint32_t hi = pack4<E5M2>(v[u].get(4) * inverse, v[u].get(5) * inverse, v[u].get(6) * inverse, v[u].get(7) * inverse);
    if (p.vec_out && c + 8 <= p.cols) {
      *reinterpret_cast<uint2*>(q + c) = make_uint2(lo, hi);
    } else {
      store_bytes(q + c, lo, hi, p.cols - c);
    }
    if ((lane & 15) == 0) scale[(c >> 7) * p.scale_block] = s;
  }
}

// The other forms: tiles of 128 rows and 64 columns per eight warps, four consecutive rows and eight columns per lane.  A lane
// then holds four consecutive bytes of eight of the transposed result's rows, which go through shared memory to be written
// in whole 128-byte rows; words are permuted by the column, so that a warp's stores and its 16-byte reads spread over the banks.
// The tile forms take 128 columns, a block, by sixteen warps.
template <class In, bool E5M2, bool COLUMNS, bool TRANSPOSED>
__global__ void __launch_bounds__(COLUMNS ? 256 : 512) quant_tile_kernel(const QuantParams p) {
  constexpr int kCols = COLUMNS ? 64 : 128, kWarps = COLUMNS ? 8 : 16;
  __shared__ float most[COLUMNS ? 8 : 1][COLUMNS ? 64 : 16];
  __shared__ float inverses[COLUMNS ? 64 : 1];
  __shared__ uint4 turned[TRANSPOSED ? kCols * 8 : 1];   // [column][16-byte piece of its 128 rows]
  dependent_entry();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, batch = blockIdx.z;
  const int rows4 = (warp & 7) * 4 + (lane >> 3), cols8 = (warp >> 3) * 8 + (lane & 7);   // which four rows, which eight columns
  const long long row0 = static_cast<long long>(blockIdx.y) * 128 + rows4 * 4;
  const int col0 = blockIdx.x * kCols + cols8 * 8;
  const In* x = static_cast<const In*>(p.x) + batch * p.stride_x + row0 * p.ldx + col0;
  Eight<In> v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i].load(x + i * p.ldx, row0 + i < p.rows ? p.cols - col0 : 0, p.vec_in);
  constexpr int kWords = 2 * sizeof(In);
  uint32_t m[kWords];
#pragma unroll
  for (int i = 0; i < kWords; ++i) m[i] = max_abs<In>(max_abs<In>(v[0].word(i), v[1].word(i)), max_abs<In>(v[2].word(i), v[3].word(i)));
  float* scale = p.scale + batch * p.stride_scale;
  float inverse[8];
  if constexpr (COLUMNS) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      m[i] = max_abs<In>(m[i], __shfl_xor_sync(0xffffffffu, m[i], 8));
      m[i] = max_abs<In>(m[i], __shfl_xor_sync(0xffffffffu, m[i], 16));
    }
    if (lane < 8) {
      Eight<In> all;
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) all.raw[i] = make_uint4(m[4 * i], m[4 * i + 1], m[4 * i + 2], m[4 * i + 3]);
      float4* to = reinterpret_cast<float4*>(&most[warp][lane * 8]);
      to[0] = make_float4(all.get(0), all.get(1), all.get(2), all.get(3));
      to[1] = make_float4(all.get(4), all.get(5), all.get(6), all.get(7));
    }
    __syncthreads();
    if (threadIdx.x < 64) {
      float a = most[0][threadIdx.x];
#pragma unroll
      for (int w = 1; w < 8; ++w) a = fmaxf(a, most[w][threadIdx.x]);
      const float s = scale_of<E5M2>(a);
      inverses[threadIdx.x] = __frcp_rn(s);
      const int c = blockIdx.x * kCols + threadIdx.x;
      if (c < p.cols) scale[c * p.scale_row + blockIdx.y * p.scale_block] = s;
    }
    __syncthreads();
    const float4* from = reinterpret_cast<const float4*>(&inverses[(lane & 7) * 8]);
    const float4 a = from[0], b = from[1];
    inverse[0] = a.x, inverse[1] = a.y, inverse[2] = a.z, inverse[3] = a.w, inverse[4] = b.x, inverse[5] = b.y, inverse[6] = b.z, inverse[7] = b.w;
  } else {
    float a = most_of<In>(m[0]);
#pragma unroll
    for (int i = 1; i < kWords; ++i) a = fmaxf(a, most_of<In>(m[i]));
    a = warp_max(a);
    if (lane == 0) most[0][warp] = a;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) a = fmaxf(a, most[0][w]);
    const float s = scale_of<E5M2>(a), one = __frcp_rn(s);
#pragma unroll
    for (int e = 0; e < 8; ++e) inverse[e] = one;
    if (threadIdx.x == 0) scale[(TRANSPOSED ? blockIdx.x : blockIdx.y) * p.scale_row + (TRANSPOSED ? blockIdx.y : blockIdx.x) * p.scale_block] = s;
  }
  uint8_t* q = p.q + batch * p.stride_q;
  if constexpr (TRANSPOSED) {
    uint32_t* words = reinterpret_cast<uint32_t*>(turned);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t w = pack4<E5M2>(v[0].get(e) * inverse[e], v[1].get(e) * inverse[e], v[2].get(e) * inverse[e], v[3].get(e) * inverse[e]);
      words[(cols8 * 8 + e) * 32 + (rows4 ^ ((cols8 & 7) * 4))] = w;
    }
    __syncthreads();
    const int piece = threadIdx.x & 7;
    const long long r0 = static_cast<long long>(blockIdx.y) * 128 + piece * 16;
#pragma unroll
    for (int c = threadIdx.x >> 3; c < kCols; c += kWarps * 4) {
      const int col = blockIdx.x * kCols + c;
      if (col >= p.cols || r0 >= p.rows) continue;
      const uint4 u = turned[c * 8 + (piece ^ ((c >> 3) & 7))];
      uint8_t* dst = q + col * p.ldq + r0;
      if (p.vec_out && r0 + 16 <= p.rows) {
        *reinterpret_cast<uint4*>(dst) = u;
      } else {
        const int n = static_cast<int>(min(p.rows - r0, 16LL));
        store_bytes(dst, u.x, u.y, n);
        store_bytes(dst + 8, u.z, u.w, n - 8);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (row0 + i >= p.rows || col0 >= p.cols) break;
      const uint32_t lo = pack4<E5M2>(v[i].get(0) * inverse[0], v[i].get(1) * inverse[1], v[i].get(2) * inverse[2], v[i].get(3) * inverse[3]);
      const uint32_t hi = pack4<E5M2>(v[i].get(4) * inverse[4], v[i].get(5) * inverse[5], v[i].get(6) * inverse[6], v[i].get(7) * inverse[7]);
      uint8_t* dst = q + (row0 + i) * p.ldq + col0;
      if (p.vec_out && col0 + 8 <= p.cols) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
      } else {
        store_bytes(dst, lo, hi, p.cols - col0);
      }
    }
  }
}

template <class In, bool E5M2>
cudaError_t launch_typed(const pmlb_quant_desc& d, const QuantParams& p, cudaStream_t stream) {
  if (d.form == PMLB_QUANT_ROWS) {
    // loads at once: four, or what a short row has (8192 x 4096 bf16, 46 registers and more: 20.5 us with four, 22.6 with eight)
    const unsigned x = static_cast<unsigned>((static_cast<long long>(p.rows) + kRowWarps - 1) / kRowWarps);
    if (p.cols > 512) return launch_dependent(quant_rows_kernel<In, E5M2, 4>, dim3(x, (p.cols + 1023) / 1024, d.batch), kRowWarps * 32, stream, p);
    if (p.cols > 256) return launch_dependent(quant_rows_kernel<In, E5M2, 2>, dim3(x, 1, d.batch), kRowWarps * 32, stream, p);
    return launch_dependent(quant_rows_kernel<In, E5M2, 1>, dim3(x, 1, d.batch), kRowWarps * 32, stream, p);
  }
  const int wide = d.form == PMLB_QUANT_COLUMNS ? 64 : 128;
  const dim3 grid((p.cols + wide - 1) / wide, (p.rows + 127) / 128, d.batch);
  switch (d.form) {
    case PMLB_QUANT_COLUMNS: return launch_dependent(quant_tile_kernel<In, E5M2, true, true>, grid, 256, stream, p);
    case PMLB_QUANT_TILES: return launch_dependent(quant_tile_kernel<In, E5M2, false, false>, grid, 512, stream, p);
    default: return launch_dependent(quant_tile_kernel<In, E5M2, false, true>, grid, 512, stream, p);
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
  p.vec_in = reinterpret_cast<uintptr_t>(x) % 16 == 0 && d.ldx * eb % 16 == 0 && batched * d.stride_x * eb % 16 == 0;
  const int wide = d.form == PMLB_QUANT_COLUMNS || d.form == PMLB_QUANT_TILES_TRANSPOSED ? 16 : 8;
  p.vec_out = reinterpret_cast<uintptr_t>(q) % wide == 0 && d.ldq % wide == 0 && (batched * d.stride_q) % wide == 0;
  if (d.in_dtype == PMLB_F32) return launch_from<float>(d, p, stream);
  return d.in_dtype == PMLB_BF16 ? launch_from<__nv_bfloat16>(d, p, stream) : launch_from<__half>(d, p, stream);
}

}  // namespace pmlb
