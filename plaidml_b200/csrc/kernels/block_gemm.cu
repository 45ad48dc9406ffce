// Products of 8-bit floats with a scale for each block of 128 terms:
//
//   C[i, j] = sum_b sa[i, b] * sb[j / 128 or j, b] * sum_{k in block b} A[i, k] * B[j, k]
//
// A block of 128 8-bit terms is one 128-byte row of a swizzled shared-memory tile: four tcgen05.mma.kind::f8f6f4 of 32 terms.
// The scales differ from block to block, so a block's products get a TMEM accumulator of their own, and eight warps that hold
// the tile's sums in registers add  sum += scale * accumulator  (packed f32 multiply-adds), while the tensor core works on the
// next block in another accumulator.  The tensor core thus never adds more than 128 terms, and the sums are f32.
#include "block_gemm.h"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cstring>
#include <mutex>

#include "dependent_launch.h"
#include "ptx.cuh"
#include "tc_launch.h"

namespace pmlb {
namespace {

constexpr int kBlock = 128;       // terms per scale, and rows of B per scale
constexpr int kMaxGroups = 1024;
constexpr int kSumWarps = 8;
constexpr int kThreads = 128 + kSumWarps * 32;   // warp 0 loads, warp 1 issues MMAs, warps 4..11 add
constexpr int kLoaderRegs = 56, kSumRegs = 224;  // (128 * 56 + 256 * 224 = 384 * 168, what the block is launched with)

// BN: columns of the accumulators.  SWAP: their rows are rows of B (weights) and their columns rows of A (tokens), for products
// of few tokens: the 128 rows of an MMA are then all of use, and BN need only be as large as there are tokens.
// VEC: each column has a scale of its own (else the tile's 128 columns of a warp share one).
template <int BN_, bool SWAP_, bool VEC_>
struct BlockCfg {
  static constexpr int BN = BN_;
  static constexpr bool kSwap = SWAP_, kVec = VEC_;
  static constexpr int kTileP = 128 * 128, kTileQ = BN * 128;
  static constexpr int kStageBytes = kTileP + kTileQ;
  static constexpr int kAccs = BN == 256 ? 2 : 4;
  static constexpr int kTmemCols = kAccs * BN;
  static constexpr int kPartBytes = kSwap ? BN * 128 * 4 : 0;                       // this CTA's sums, where K is split
  static constexpr int kTailBytes = 512 + 3 * (kMaxGroups + 4) * 4;
  static constexpr int kStages = std::min(10, (231000 - 1024 - kPartBytes - kTailBytes) / kStageBytes);
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kPartBytes + kTailBytes;
  static_assert(kStages >= 3 && kSmem <= 232448, "shared memory");
};

struct BlockGemmParams {
  int m, n, num_kb;
  int groups, terms;       // 0 = one product; groups along terms instead of rows
  int tiles_m, tiles_n;    // (rows of groups: tiles_m is not used)
  const int32_t* offsets;
  const float *a_scale, *b_scale;
  long long as_row, as_block, bs_row, bs_block, bs_group;
  int b_shift;             // rows of B per scale, as a power of two
  void* out;
  long long ldc, stride_c;
  int out_dtype, out_align;   // bytes that every row and the matrix start on: 32, 16, or less
  int split;               // CTAs of a cluster that share the tile's blocks
  uint32_t idesc;
  int* status;
};

struct Tile {
  int group, row0, row_end, n0, kb0, kb1;
};

__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}
__device__ __forceinline__ uint64_t pack2(float lo, float hi) { return pack2(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  uint32_t lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(v));
  return make_float2(__uint_as_float(lo), __uint_as_float(hi));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&v)[N]) {
  if constexpr (N == 32) {
    tmem_ld_32x32(taddr, v);
  } else if constexpr (N == 16) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
  } else {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr)
                 : "memory");
  }
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t cluster_addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
  return v;
}

// All threads of the cluster, from code where the warp's lanes may have parted.
__device__ __forceinline__ void cluster_sync_threads() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

__device__ __forceinline__ void store_one(const BlockGemmParams& p, long long at, float v) {
  if (p.out_dtype == PMLB_F32) {
    static_cast<float*>(p.out)[at] = v;
  } else if (p.out_dtype == PMLB_BF16) {
    static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
  } else {
    static_cast<__half*>(p.out)[at] = __float2half_rn(v);
  }
}

// Eight consecutive columns of a row from element `at` on, `n` of which exist.
__device__ __forceinline__ void store_eight(const BlockGemmParams& p, long long at, const float (&v)[8], int n) {
  if (n >= 8 && p.out_align >= 16) {
    if (p.out_dtype == PMLB_F32) {
      float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.out) + at);
      dst[0] = make_float4(v[0], v[1], v[2], v[3]);
      dst[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint4 u;
      if (p.out_dtype == PMLB_BF16) {
        u = make_uint4(cvt_pack16<true, false>(v[0], v[1]), cvt_pack16<true, false>(v[2], v[3]), cvt_pack16<true, false>(v[4], v[5]),
                       cvt_pack16<true, false>(v[6], v[7]));
      } else {
        u = make_uint4(cvt_pack16<false, false>(v[0], v[1]), cvt_pack16<false, false>(v[2], v[3]), cvt_pack16<false, false>(v[4], v[5]),
                       cvt_pack16<false, false>(v[6], v[7]));
      }
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at) = u;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e < n) store_one(p, at + e, v[e]);
    }
  }
}

template <class Cfg>
__global__ void __launch_bounds__(kThreads, 1)
    block_gemm_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ BlockGemmParams p) {
  constexpr int BN = Cfg::BN, kStages = Cfg::kStages, kAccs = Cfg::kAccs;
  constexpr bool SWAP = Cfg::kSwap, VEC = Cfg::kVec;
  constexpr int kTileRows = SWAP ? BN : 128, kTileCols = SWAP ? 128 : BN;   // of C
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t ring = (raw + 1023u) & ~1023u;
  uint8_t* after_ring = smem_raw + (ring - raw) + kStages * Cfg::kStageBytes;
  float* part = reinterpret_cast<float*>(after_ring);
  uint8_t* tail = after_ring + Cfg::kPartBytes;
  const uint32_t bar0 = smem_u32(tail);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (10 + s); };
  auto tfull_bar = [&](int a) { return bar0 + 8u * (20 + a); };
  auto tempty_bar = [&](int a) { return bar0 + 8u * (24 + a); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 256);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 264);   // flag, code, wait limit
  int* begins = reinterpret_cast<int*>(tail + 512);         // groups of rows: first row,
  int* ends = begins + kMaxGroups + 4;                      // row behind the last,
  int* before = ends + kMaxGroups + 4;                      // row tiles of the groups before
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 64) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < kAccs; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), kSumWarps);
    }
    abort_flag[0] = 0;
    abort_flag[1] = 0;
    abort_flag[2] = 0;
    fence_mbar_init();
  } else if (threadIdx.x == 96) {
    tma_prefetch_desc(&map_p);
    tma_prefetch_desc(&map_q);
  } else if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), Cfg::kTmemCols);
    tmem_relinquish();
    tc_fence_before_sync();
  }
  grid_dependency_wait();
  grid_launch_dependents();
  if (warp == 0 && p.groups > 0 && !p.terms) {
    // Row tiles of the groups, added up: a warp's prefix sums, 32 groups at a time.  An offset counts as the largest so far, so
    // that groups never share rows.
    int sum = 0, top = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 32) {
      const int g = g0 + lane;
      int hi = g < p.groups ? min(max(__ldg(p.offsets + g + 1), 0), p.m) : 0;
      if (g0 == 0) top = min(max(__ldg(p.offsets), 0), p.m);
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, hi, d);
        if (lane >= d) hi = max(hi, y);
      }
      hi = max(hi, top);
      int lo = __shfl_up_sync(0xffffffffu, hi, 1);
      if (lane == 0) lo = top;
      top = __shfl_sync(0xffffffffu, hi, 31);
      const int tiles = (hi - lo + kTileRows - 1) / kTileRows;
      int x = tiles;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      if (g < p.groups) begins[g] = lo, ends[g] = hi, before[g] = sum + x - tiles;
      sum += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) before[p.groups] = sum;
  }
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  const int units = static_cast<int>(gridDim.x) / p.split;
  const int rank = static_cast<int>(blockIdx.x) % p.split;
  const int first = static_cast<int>(blockIdx.x) / p.split;
  const int per_group = p.tiles_m * p.tiles_n;
  const int total = p.groups == 0 ? per_group : (p.terms ? p.groups * per_group : before[p.groups] * p.tiles_n);
  // Every role walks the same tiles.
  auto tile_at = [&](int t) {
    Tile x;
    x.group = 0, x.kb0 = 0, x.kb1 = p.num_kb;
    if (p.groups > 0 && !p.terms) {
      int lo = 0, hi = p.groups;   // the last group whose tiles begin at or before t
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (before[mid] * p.tiles_n <= t) lo = mid; else hi = mid;
      }
      // (groups without tiles begin where the next one does: the search ends on the last of them, the one with tiles)
      const int tiles = before[lo + 1] - before[lo];
      const int local = t - before[lo] * p.tiles_n;
      const int nt = local / tiles;
      x.group = lo;
      x.row0 = begins[lo] + (local - nt * tiles) * kTileRows;
      x.row_end = ends[lo];
      x.n0 = nt * kTileCols;
    } else {
      if (p.terms) {
        x.group = t / per_group;
        t -= x.group * per_group;
        const int lo = min(max(__ldg(p.offsets + x.group), 0), p.num_kb * kBlock);
        const int hi = min(max(__ldg(p.offsets + x.group + 1), lo), p.num_kb * kBlock);
        x.kb0 = lo / kBlock;
        x.kb1 = hi > lo ? (hi + kBlock - 1) / kBlock : x.kb0;
      }
      // bands of 16 row tiles, so that the tiles in flight share rows of A and of B in L2
      const int band = t / (16 * p.tiles_n);
      const int rows = min(16, p.tiles_m - band * 16);
      const int local = t - band * 16 * p.tiles_n;
      const int nt = local / rows;
      x.row0 = (band * 16 + local - nt * rows) * kTileRows;
      x.row_end = p.m;
      x.n0 = nt * kTileCols;
    }
    if (p.split > 1) {
      const int blocks = x.kb1 - x.kb0, base = x.kb0;
      x.kb0 = base + blocks * rank / p.split;
      x.kb1 = base + blocks * (rank + 1) / p.split;
    }
    return x;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLoaderRegs));
    if (warp == 0) {
      // ------------------------------------------------------------ loads
      const bool leader = elect_one();
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = first; t < total && ok; t += units) {
        const Tile x = tile_at(t);
        const int py = SWAP ? x.n0 : x.row0, qy = SWAP ? x.row0 : x.n0;
        const int z = p.terms ? 0 : x.group;
        for (int kb = x.kb0; kb < x.kb1; ++kb) {
          if (!mbar_wait_warp(empty_bar(stage), phase ^ 1u, abort_flag)) {
            if (leader && abort_flag[1] == 0) abort_flag[1] = 1;
            ok = false;
            break;
          }
          if (leader) {
            const uint32_t s = ring + static_cast<uint32_t>(stage) * Cfg::kStageBytes;
            mbar_arrive_expect_tx(full_bar(stage), Cfg::kStageBytes);
            tma_load_3d(s, &map_p, full_bar(stage), kb * kBlock, py, SWAP ? z : 0);
            tma_load_3d(s + Cfg::kTileP, &map_q, full_bar(stage), kb * kBlock, qy, SWAP ? 0 : z);
          }
          __syncwarp();
          if (++stage == kStages) stage = 0, phase ^= 1u;
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMAs
      const bool leader = elect_one();
      const uint64_t desc0 = make_smem_desc_sw128(0, 16, 1024);
      const uint32_t desc_hi = static_cast<uint32_t>(desc0 >> 32), desc_lo = static_cast<uint32_t>(desc0);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int t = first; t < total && ok; t += units) {
        const Tile x = tile_at(t);
        for (int kb = x.kb0; kb < x.kb1; ++kb) {
          if (!mbar_wait_warp(tempty_bar(acc), acc_phase ^ 1u, abort_flag)) {
            if (leader && abort_flag[1] == 0) abort_flag[1] = 2;
            ok = false;
            break;
          }
          if (!mbar_wait_warp(full_bar(stage), phase, abort_flag)) {
            if (leader && abort_flag[1] == 0) abort_flag[1] = 3;
            ok = false;
            break;
          }
          tc_fence_after_sync();
          if (leader) {
            const uint32_t s = ring + static_cast<uint32_t>(stage) * Cfg::kStageBytes;
            const uint32_t lo_p = desc_lo | ((s & 0x3FFFFu) >> 4), lo_q = desc_lo | (((s + Cfg::kTileP) & 0x3FFFFu) >> 4);
            tc_mma_x4<kMmaF8, 1>(tmem_base + static_cast<uint32_t>(acc * BN), lo_p, lo_q, desc_hi, desc_hi, p.idesc, 0u, 2u, 2u);
            tc_commit(empty_bar(stage));
            tc_commit(tfull_bar(acc));
          }
          __syncwarp();
          if (++stage == kStages) stage = 0, phase ^= 1u;
          if (++acc == kAccs) acc = 0, acc_phase ^= 1u;
        }
      }
    }
  } else {
    // ------------------------------------------------------------ sums
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSumRegs));
    const int w = warp - 4;
    const int quarter = warp & 3, half = w >> 2;     // TMEM lanes [32 quarter, ...), columns [half * BN / 2, ...)
    constexpr int kCols = BN / 2;
    constexpr int kChunk = kCols < 32 ? kCols : 32;
    constexpr int kMine = (kCols + 31) / 32;         // column scales that a lane fetches
    const uint32_t t_mine = tmem_base + static_cast<uint32_t>(half * kCols) + (static_cast<uint32_t>(quarter * 32) << 16);
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int t = first; t < total && ok; t += units) {
      const Tile x = tile_at(t);
      // scales of this thread's accumulator row, and of the columns
      const int i = quarter * 32 + lane;
      const int token = min(x.row0 + (SWAP ? 0 : i), p.m - 1), weight = min(x.n0 + (SWAP ? i : half * kCols), p.n - 1);
      const float* sa = p.a_scale + (SWAP ? 0 : token * p.as_row);
      const float* sb = p.b_scale + (p.terms ? 0 : x.group) * p.bs_group + (SWAP || !VEC ? (weight >> p.b_shift) * p.bs_row : 0);
      const float* row_scale = SWAP ? sb : sa;
      const float* col_scale = SWAP ? sa : sb;
      const long long row_step = SWAP ? p.bs_block : p.as_block, col_step = SWAP ? p.as_block : p.bs_block;
      long long col_at[kMine];
      if constexpr (VEC) {
#pragma unroll
        for (int e = 0; e < kMine; ++e) {
          const int j = half * kCols + e * 32 + min(lane, kCols - 1);
          col_at[e] = SWAP ? min(x.row0 + j, p.m - 1) * p.as_row : min(x.n0 + j, p.n - 1) * p.bs_row;
        }
      } else {
        col_at[0] = 0;
      }
      uint64_t sum[kCols / 2];
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j) sum[j] = 0;
      float next_row = 0.f, next_col[kMine];
      auto fetch = [&](int kb) {
        next_row = __ldg(row_scale + kb * row_step);
#pragma unroll
        for (int e = 0; e < (VEC ? kMine : 1); ++e) next_col[e] = __ldg(col_scale + col_at[e] + kb * col_step);
      };
      if (x.kb0 < x.kb1) fetch(x.kb0);
      for (int kb = x.kb0; kb < x.kb1; ++kb) {
        const float rs = next_row;
        float cs[kMine];
#pragma unroll
        for (int e = 0; e < (VEC ? kMine : 1); ++e) cs[e] = next_col[e];
        if (kb + 1 < x.kb1) fetch(kb + 1);
        if (!mbar_wait_warp(tfull_bar(acc), acc_phase, abort_flag)) {
          if (lane == 0 && abort_flag[1] == 0) abort_flag[1] = 4;
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t at = t_mine + static_cast<uint32_t>(acc * BN);
        const uint64_t one_scale = pack2(rs * cs[0], rs * cs[0]);
#pragma unroll
        for (int c = 0; c < kCols; c += kChunk) {
          uint32_t v[kChunk];
          tmem_ld<kChunk>(at + c, v);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < kChunk; e += 2) {
            uint64_t s = one_scale;
            if constexpr (VEC) {
              // (a column's scale is held by one lane)
              const float s0 = __shfl_sync(0xffffffffu, cs[c / 32], (c + e) & 31), s1 = __shfl_sync(0xffffffffu, cs[c / 32], (c + e + 1) & 31);
              s = pack2(rs * s0, rs * s1);
            }
            sum[(c + e) / 2] = fma2(pack2(v[e], v[e + 1]), s, sum[(c + e) / 2]);
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(tempty_bar(acc));
        if (++acc == kAccs) acc = 0, acc_phase ^= 1u;
      }
      if (!ok) break;
      if constexpr (SWAP) {
        if (p.split > 1) {
#pragma unroll
          for (int j = 0; j < kCols / 2; ++j) {
            const float2 v = unpack2(sum[j]);
            part[(half * kCols + 2 * j) * 128 + i] = v.x;
            part[(half * kCols + 2 * j + 1) * 128 + i] = v.y;
          }
        } else if (x.n0 + i < p.n) {
          const long long base = (p.terms ? x.group * p.stride_c : 0) + x.n0 + i;
#pragma unroll
          for (int j = 0; j < kCols; ++j) {
            const float2 v = unpack2(sum[j / 2]);
            const int row = x.row0 + half * kCols + j;
            if (row < x.row_end) store_one(p, base + row * p.ldc, j & 1 ? v.y : v.x);
          }
        }
      } else {
        const int row = x.row0 + i, col = x.n0 + half * kCols;
        if (row < x.row_end) {
          const long long base = (p.terms ? x.group * p.stride_c : 0) + row * p.ldc + col;
#pragma unroll
          for (int j = 0; j < kCols; j += 8) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              const float2 u = unpack2(sum[(j + e) / 2]);
              v[e] = u.x, v[e + 1] = u.y;
            }
            if (col + j < p.n) store_eight(p, base + j, v, p.n - col - j);
          }
        }
      }
    }
  }

  __syncwarp();
  tc_fence_before_sync();
  if (p.split > 1) {
    cluster_sync_threads();
  } else {
    __syncthreads();
  }
  const bool failed = abort_flag[0] != 0;
  if constexpr (SWAP) {
    if (p.split > 1) {
      // The cluster's one tile: each CTA adds a run of its columns over all parts, in the order of the blocks.
      if (first < total && !failed) {
        const Tile x = tile_at(first);
        const int begin = BN * 128 / p.split * rank, end = BN * 128 / p.split * (rank + 1);
        const long long base = (p.terms ? x.group * p.stride_c : 0) + x.n0;
        for (int e = begin + static_cast<int>(threadIdx.x); e < end; e += kThreads) {
          const int j = e >> 7, i = e & 127;
          const int row = x.row0 + j;
          if (row >= x.row_end || x.n0 + i >= p.n) continue;
          float v = 0.f;
          for (int r = 0; r < p.split; ++r) v += ld_cluster_f32(mapa_rank(smem_u32(part + e), static_cast<uint32_t>(r)));
          store_one(p, base + row * p.ldc + i, v);
        }
      }
      cluster_sync_threads();   // no CTA leaves while another may still read its part
    }
  }
  if (failed) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0, abort_flag[1] != 0 ? abort_flag[1] : 9);
    // copies and MMAs still in flight get a bounded time before TMEM and shared memory go away
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 2000000ull) __nanosleep(2000);
  }
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, Cfg::kTmemCols);
  }
}

using KernelPtr = void (*)(const CUtensorMap, const CUtensorMap, const BlockGemmParams);

// The shared-memory limit is an attribute per device.
template <class Cfg>
KernelPtr instance(int dev) {
  static std::atomic<uint64_t> done{0};
  const uint64_t bit = 1ull << (dev & 63);
  if (dev >= 64 || (done.load(std::memory_order_acquire) & bit) == 0) {
    if (cudaFuncSetAttribute(block_gemm_kernel<Cfg>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem) == cudaSuccess) {
      done.fetch_or(bit, std::memory_order_release);
    }
  }
  return block_gemm_kernel<Cfg>;
}

template <class Cfg>
cudaError_t launch(const CUtensorMap& mp, const CUtensorMap& mq, const BlockGemmParams& p, int grid, int dev, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Cfg::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0] = dependent_launch_attribute();
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.split > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, instance<Cfg>(dev), mp, mq, p);
}

uint32_t f8_format(int dtype) { return dtype == PMLB_F8E5M2 ? 1u : 0u; }

}  // namespace

int block_gemm_launch(const pmlb_block_gemm_desc& d, const void* a, const float* a_scale, const void* b, const float* b_scale,
                      const int32_t* offsets, void* c, int* status, cudaStream_t stream, std::string* err) {
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const bool by_rows = d.groups > 0 && d.group_dim == PMLB_GROUP_ROWS, by_terms = d.groups > 0 && !by_rows;
  BlockGemmParams p{};
  p.m = d.m, p.n = d.n, p.num_kb = (d.k + kBlock - 1) / kBlock;
  p.groups = d.groups, p.terms = by_terms;
  p.offsets = offsets;
  p.a_scale = a_scale, p.b_scale = b_scale;
  p.as_row = d.a_scale_row, p.as_block = d.a_scale_block;
  p.bs_row = d.b_scale_row, p.bs_block = d.b_scale_block, p.bs_group = d.b_scale_group;
  p.b_shift = d.b_scale_rows == 128 ? 7 : 0;
  p.out = c, p.ldc = d.ldc, p.stride_c = d.stride_c, p.out_dtype = d.out_dtype;
  const long long ob = d.out_dtype == PMLB_F32 ? 4 : 2;
  const long long bits = static_cast<long long>(reinterpret_cast<uintptr_t>(c)) | (d.ldc * ob) | (by_terms ? d.stride_c * ob : 0);
  p.out_align = bits % 32 == 0 ? 32 : (bits % 16 == 0 ? 16 : 1);
  p.status = status;

  // Rows that a tile of tokens has to hold: those of the product, or of a group on average.
  const long long rows = by_rows ? (d.m + d.groups - 1) / d.groups : d.m;
  const bool swap = rows <= 64;
  int bn = 128;
  if (swap) {
    bn = rows <= 16 ? 16 : (rows <= 32 ? 32 : 64);
  }
  const int tile_rows = swap ? bn : 128, tile_cols = swap ? 128 : bn;
  p.tiles_m = (d.m + tile_rows - 1) / tile_rows;
  p.tiles_n = (d.n + tile_cols - 1) / tile_cols;
  // (groups of rows: at most one tile more than whole ones for each group that has rows)
  const long long row_tiles = by_rows ? d.m / tile_rows + std::min(d.groups, d.m) : p.tiles_m;
  const long long tiles = row_tiles * p.tiles_n * (by_terms ? d.groups : 1);
  if (tiles > 0x07ffffff) {
    *err = "block_gemm: too many tiles";
    return PMLB_ERR_UNSUPPORTED;
  }
  p.split = 1;
  if (swap) {
    while (p.split < 8 && tiles * p.split * 2 <= sms && p.num_kb >= p.split * 4) p.split *= 2;
  }
  const int grid = p.split > 1 ? static_cast<int>(tiles) * p.split : static_cast<int>(std::min<long long>(tiles, sms));
  // bits: [4,6) f32 accumulators, [7,10) and [10,13) formats of the two operands, [17,23) N >> 3, [24,29) M >> 4
  p.idesc = 1u << 4 | f8_format(swap ? d.b_dtype : d.a_dtype) << 7 | f8_format(swap ? d.a_dtype : d.b_dtype) << 10 |
            static_cast<uint32_t>(bn >> 3) << 17 | 8u << 24;

  CUtensorMap ma, mb;
  if (!tc_encode_bytes(&ma, a, d.k, d.m, 1, d.lda, 16, tile_rows, err)) return PMLB_ERR_INVALID;
  if (!tc_encode_bytes(&mb, b, d.k, d.n, by_rows ? d.groups : 1, d.ldb, by_rows ? d.stride_b : 16, tile_cols, err)) return PMLB_ERR_INVALID;
  cudaError_t e = cudaSuccess;
  if (swap) {
    switch (bn) {
      case 16: e = launch<BlockCfg<16, true, true>>(mb, ma, p, grid, dev, stream); break;
      case 32: e = launch<BlockCfg<32, true, true>>(mb, ma, p, grid, dev, stream); break;
      default: e = launch<BlockCfg<64, true, true>>(mb, ma, p, grid, dev, stream); break;
    }
  } else if (d.b_scale_rows == 1) {
    e = launch<BlockCfg<128, false, true>>(ma, mb, p, grid, dev, stream);
  } else {
    e = launch<BlockCfg<128, false, false>>(ma, mb, p, grid, dev, stream);
  }
  if (e != cudaSuccess) {
    *err = std::string("block_gemm launch: ") + cudaGetErrorString(e);
    return PMLB_ERR_CUDA;
  }
  return 0;
}

}  // namespace pmlb
