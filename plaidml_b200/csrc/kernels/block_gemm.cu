// Products of 8-bit floats with a scale for each block of 128 terms:
//
//   C[i, j] = sum_b sa[i, b] * sb[j / 128 or j, b] * sum_{k in block b} A[i, k] * B[j, k]
//
// A block of 128 8-bit terms is one 128-byte row of a swizzled shared-memory tile: four tcgen05.mma.kind::f8f6f4 of 32 terms.
// The scales differ from block to block, so a block's products get a TMEM accumulator of their own, and eight warps that hold
// the tile's sums in registers add  sum += scale * accumulator  (packed f32 multiply-adds), while the tensor core works on the
// next block in another accumulator.  The tensor core thus never adds more than 128 terms, and the sums are f32.
//
// What bounds it.  Large products (CTA pairs on 256 x 256 tiles): a block's MMAs take 512 cycles, a block 700.  Two accumulators of
// 256 columns fill TMEM, and one's way round -- MMAs 512, their completion to both CTAs some 200, half of the sums' loads
// and additions before it can be handed back 330, that to the issuer and its first MMA 350 -- is 1400 for two blocks.  (Found
// with clock readings in a copy: the issuer waits for an accumulator in 62 of 64 blocks and for operands in 1; without the
// additions a block takes 620, with half of the MMAs 600.)  Around it, a tile's results cost 2000 cycles of which the two
// accumulators hide 1400.  Few rows: the weights' bytes from HBM (5.3 to 6.4 TB/s of them).
#include "block_gemm.h"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>
#include <mutex>
#include <type_traits>

#include "dependent_launch.h"
#include "ptx.cuh"
#include "tc_launch.h"

namespace pmlb {
namespace {

constexpr int kBlock = 128;       // terms per scale, and rows of B per scale
constexpr int kMaxGroups = 1024;

// Which scales differ within a warp's part of an accumulator (32 rows, half of the columns).
enum Scales { kOfRows, kOfBoth };

// BN: columns of the accumulators.  SWAP: their rows are rows of B (weights) and their columns rows of A (tokens), for products
// of few tokens: the 128 rows of an MMA are then all of use, and BN need only be as large as there are tokens.
// CTAS = 2: a cluster of two CTAs on one tile of 256 rows, each with 128 of them and half of the other operand.
template <int BN_, bool SWAP_, Scales SCALES_, int CTAS_ = 1>
struct BlockCfg {
  static constexpr int BN = BN_, CTAS = CTAS_;
  static constexpr bool kSwap = SWAP_;
  static constexpr Scales kScales = SCALES_;
  static constexpr int kSumWarps = 8;
  static constexpr int kThreads = 128 + kSumWarps * 32;   // warp 0 loads, warp 1 issues MMAs, warps 4 and up add
  static constexpr int kLoaderRegs = 56, kSumRegs = 224;  // (128 * 56 + 256 * 224 = 384 * 168, what the block is launched with)
  static constexpr int kCols = BN / (kSumWarps / 4);       // columns that a warp adds
  static constexpr int kTileP = 128 * 128, kTileQ = BN / CTAS * 128;
  static constexpr int kStageBytes = kTileP + kTileQ;
  static constexpr int kAccs = BN == 256 ? 2 : 4;
  static constexpr int kTmemCols = kAccs * BN;
  static constexpr bool kSplits = CTAS == 1;                                        // K may be shared by a cluster
  static constexpr int kPartBytes = kSwap ? BN * 128 * 4 : 0;                       // this CTA's sums, where it is (else in the place of the boxes)
  // Scales of a block: one for each row of the accumulator, then one for each column (or for each 128 of them); kAhead blocks are
  // on their way (see the warp that fetches them for what bounds it).
  static constexpr int kSlots = 16, kAhead = kSlots - 2 * kAccs - 1;
  static constexpr int kSlotFloats = 128 + (kScales == kOfBoth ? BN : 4);
  static constexpr int kScaleBytes = kSlots * kSlotFloats * 4;
  static constexpr int kStageOutBytes = kSwap ? 0 : kSumWarps * 8192;    // results on their way out: two boxes of 32 rows of 128 bytes per warp
  static constexpr int kTailBytes = 512 + 2 * (kMaxGroups + 4) * 4;
  static constexpr int kStages = std::min(10, (232448 - 1024 - kPartBytes - kScaleBytes - kStageOutBytes - kTailBytes) / kStageBytes);
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kPartBytes + kScaleBytes + kStageOutBytes + kTailBytes;
  static_assert(kStages >= kAccs && kStages >= 3 && kSmem <= 232448, "shared memory");   // (kAccs: see the warp that fetches scales)
  static_assert(kSwap || kCols == 64 || kCols == 128, "boxes");
  static_assert(kSwap || !kSplits || kStageOutBytes >= BN * 128 * 4, "room for a part");
};

struct BlockGemmParams {
  int m, n, num_kb;
  int groups, terms;       // 0 = one product; groups along terms instead of rows
  int tiles_m, tiles_n;    // (rows of groups: tiles_m is not used)
  const int32_t* offsets;
  const float *a_scale, *b_scale;
  long long as_row, as_block, bs_row, bs_block, bs_group;
  int b_shift;             // rows of B per scale, as a power of two
  int b_step;              // 1, or 0 where all groups share one B
  void* out;
  long long ldc, stride_c;
  int out_dtype, out_wide;   // every row and the matrix start on 16 bytes
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
// c += a * b.  (volatile: stays behind the wait for the TMEM loads whose registers it reads)
__device__ __forceinline__ void fma2(uint64_t& c, uint64_t a, uint64_t b) { asm volatile("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c) : "l"(a), "l"(b)); }

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm volatile("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

#define PMLB_OUT_8(i) \
  "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&v)[N]) {
  if constexpr (N == 64) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
        "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, "
        "%45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];"
        : PMLB_OUT_8(0), PMLB_OUT_8(8), PMLB_OUT_8(16), PMLB_OUT_8(24), PMLB_OUT_8(32), PMLB_OUT_8(40), PMLB_OUT_8(48), PMLB_OUT_8(56)
        : "r"(taddr)
        : "memory");
  } else if constexpr (N == 32) {
    tmem_ld_32x32(taddr, v);
  } else if constexpr (N == 16) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : PMLB_OUT_8(0), PMLB_OUT_8(8)
        : "r"(taddr)
        : "memory");
  } else {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : PMLB_OUT_8(0)
                 : "r"(taddr)
                 : "memory");
  }
}

#undef PMLB_OUT_8

__device__ __forceinline__ float ld_cluster_f32(uint32_t cluster_addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
  return v;
}

__device__ __forceinline__ float ld_shared_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// Four bytes from global to shared memory without a register; groups of them complete in order.
__device__ __forceinline__ void copy_async_4(uint32_t to, const float* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ float4 ld_cluster_v4(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
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

// Four consecutive columns of a row from element `at` on, `n` of which exist.
__device__ __forceinline__ void store_four(const BlockGemmParams& p, long long at, const float4& v, int n) {
  if (n >= 4 && p.out_wide) {
    if (p.out_dtype == PMLB_F32) {
      *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = v;
    } else {
      const bool bf16 = p.out_dtype == PMLB_BF16;
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) =
          make_uint2(bf16 ? cvt_pack16<true, false>(v.x, v.y) : cvt_pack16<false, false>(v.x, v.y),
                     bf16 ? cvt_pack16<true, false>(v.z, v.w) : cvt_pack16<false, false>(v.z, v.w));
    }
  } else {
    const float one[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e < n) store_one(p, at + e, one[e]);
    }
  }
}

// Part of a tile in shared memory: rows of BN floats, 16-byte pieces permuted by the row (a lane writes a row).
template <int BN>
__device__ __forceinline__ uint32_t part_piece(uint32_t row, uint32_t piece) { return row * (BN * 4u) + ((piece ^ (row & 7u)) << 4); }

// Results leave through shared memory in boxes of 32 rows of 128 bytes (64 columns of 16 bits, or 32 of 32 bits), in the layout
// of a TMA store with 128-byte swizzle: 16-byte pieces permuted by the row, which spreads a lane's row over the banks.
__device__ __forceinline__ uint32_t box_piece(uint32_t row, uint32_t piece) { return row * 128u + ((piece ^ (row & 7u)) << 4); }

// Eight sums as 16-bit values.
template <bool BF16>
__device__ __forceinline__ uint4 pack_eight(const uint64_t* sum) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = unpack2(sum[i]);
    u[i] = cvt_pack16<BF16, false>(v.x, v.y);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// A box by plain stores: rows [0, rows) of C from element `base` on, `n` columns of which exist.
__device__ __forceinline__ void store_box(const BlockGemmParams& p, uint32_t at, long long base, int rows, int n, int lane) {
  const int bytes = p.out_dtype == PMLB_F32 ? 4 : 2;
  char* dst = static_cast<char*>(p.out) + base * bytes;
  const long long step = p.ldc * bytes;
  if (n * bytes >= 128 && p.out_wide) {
    const int piece = lane & 7;
#pragma unroll 4
    for (int r = lane >> 3; r < 32; r += 4) {
      const uint4 u = ld_shared_v4(at + box_piece(r, piece));
      if (r < rows) *reinterpret_cast<uint4*>(dst + r * step + piece * 16) = u;
    }
  } else if (bytes == 4) {
#pragma unroll 1
    for (int r = 0; r < rows; ++r) {
      const float v = ld_shared_f32(at + box_piece(r, lane >> 2) + (lane & 3) * 4);
      if (lane < n) *reinterpret_cast<float*>(dst + r * step + lane * 4) = v;
    }
  } else {
#pragma unroll 1
    for (int r = 0; r < rows; ++r) {
#pragma unroll
      for (int c = lane; c < 64; c += 32) {
        uint16_t h;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(at + box_piece(r, c >> 3) + (c & 7) * 2) : "memory");
        if (c < n) *reinterpret_cast<uint16_t*>(dst + r * step + c * 2) = h;
      }
    }
  }
}

template <class Cfg>
__global__ void __launch_bounds__(Cfg::kThreads, 1)
    block_gemm_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_c,
                      const __grid_constant__ BlockGemmParams p) {
  constexpr int BN = Cfg::BN, kStages = Cfg::kStages, kAccs = Cfg::kAccs;
  constexpr int CTAS = Cfg::CTAS;
  constexpr bool SWAP = Cfg::kSwap, PAIR = CTAS == 2;
  constexpr Scales SCALES = Cfg::kScales;
  constexpr int kTileRows = SWAP ? BN : 128 * CTAS, kTileCols = SWAP ? 128 * CTAS : BN;   // of C
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t ring = (raw + 1023u) & ~1023u;
  uint8_t* after_ring = smem_raw + (ring - raw) + kStages * Cfg::kStageBytes;
  const uint32_t out_stage = smem_u32(after_ring);   // (1024-byte aligned, as the boxes' swizzle wants it)
  after_ring += Cfg::kStageOutBytes;
  float* part = reinterpret_cast<float*>(after_ring);
  const uint32_t scale_ring = smem_u32(after_ring + Cfg::kPartBytes);
  uint8_t* tail = after_ring + Cfg::kPartBytes + Cfg::kScaleBytes;
  const uint32_t bar0 = smem_u32(tail);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto done_bar = [&](int s) { return bar0 + 8u * (10 + s); };     // the stage's products (and their scales) are there, its operands free
  auto tempty_bar = [&](int a) { return bar0 + 8u * (20 + a); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 256);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 264);   // flag, code, wait limit
  int* begins = reinterpret_cast<int*>(tail + 512);         // groups of rows: first row (and, behind the last one, the end),
  int* before = begins + kMaxGroups + 4;                    // row tiles of the groups before
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int side = PAIR ? static_cast<int>(cluster_ctarank()) : 0;   // CTA of the pair

  if (threadIdx.x == 64) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(done_bar(s), 2);   // (the products, and their scales)
    }
    for (int a = 0; a < kAccs; ++a) {
      mbar_init(tempty_bar(a), Cfg::kSumWarps * CTAS);   // (pairs: both CTAs' warps, at the first CTA)
    }
    abort_flag[0] = 0;
    abort_flag[1] = 0;
    abort_flag[2] = 0;
    fence_mbar_init();
  } else if (threadIdx.x == 96) {
    tma_prefetch_desc(&map_p);
    tma_prefetch_desc(&map_q);
    if (!SWAP && p.out_wide) tma_prefetch_desc(&map_c);
  } else if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(smem_u32(tmem_slot), Cfg::kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), Cfg::kTmemCols);
      tmem_relinquish();
    }
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
      if (g < p.groups) begins[g] = lo, before[g] = sum + x - tiles;
      sum += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) begins[p.groups] = top, before[p.groups] = sum;
  }
  __syncwarp();
  if constexpr (PAIR) {
    cluster_sync_all();   // (the other CTA's barriers must exist before anything is sent to them)
  } else {
    __syncthreads();
  }
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  const int share = PAIR ? 2 : p.split;   // CTAs of a tile
  const int units = static_cast<int>(gridDim.x) / share;
  const int rank = PAIR ? 0 : static_cast<int>(blockIdx.x) % share;
  const int first = static_cast<int>(blockIdx.x) / share;
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
      x.row_end = begins[lo + 1];
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
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::kLoaderRegs));
    if (warp == 0) {
      // ------------------------------------------------------------ loads
      const bool leader = elect_one();
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = first; t < total && ok; t += units) {
        const Tile x = tile_at(t);
        const int py = (SWAP ? x.n0 : x.row0) + side * 128, qy = (SWAP ? x.row0 : x.n0) + side * (BN / CTAS);
        const int z = p.terms ? 0 : x.group * p.b_step;
        for (int kb = x.kb0; kb < x.kb1; ++kb) {
          if (!mbar_wait_warp(done_bar(stage), phase ^ 1u, abort_flag)) {
            if (leader && abort_flag[1] == 0) abort_flag[1] = 1;
            ok = false;
            break;
          }
          if (leader) {
            const uint32_t s = ring + static_cast<uint32_t>(stage) * Cfg::kStageBytes;
            if (side == 0) mbar_arrive_expect_tx(full_bar(stage), CTAS * Cfg::kStageBytes);
            if constexpr (PAIR) {   // both CTAs' bytes are counted at the first one
              const uint32_t fb = mapa_rank(full_bar(stage), 0);
              tma_load_3d_pair(s, &map_p, fb, kb * kBlock, py, SWAP ? z : 0);
              tma_load_3d_pair(s + Cfg::kTileP, &map_q, fb, kb * kBlock, qy, SWAP ? 0 : z);
            } else {
              tma_load_3d(s, &map_p, full_bar(stage), kb * kBlock, py, SWAP ? z : 0);
              tma_load_3d(s + Cfg::kTileP, &map_q, full_bar(stage), kb * kBlock, qy, SWAP ? 0 : z);
            }
          }
          __syncwarp();
          if (++stage == kStages) stage = 0, phase ^= 1u;
        }
      }
    } else if (warp == 1 && side == 0) {
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
          // (both barriers are asked before either answer is waited for, and one commit serves the loaders and the adding warps)
          const uint32_t s = ring + static_cast<uint32_t>(stage) * Cfg::kStageBytes;
          const uint32_t lo_p = desc_lo | ((s & 0x3FFFFu) >> 4), lo_q = desc_lo | (((s + Cfg::kTileP) & 0x3FFFFu) >> 4);
          const bool both = mbar_test_wait(full_bar(stage), phase) & mbar_test_wait(tempty_bar(acc), acc_phase ^ 1u);
          if (!__all_sync(0xffffffffu, both)) {
            if (!mbar_wait_warp(full_bar(stage), phase, abort_flag)) {
              if (leader && abort_flag[1] == 0) abort_flag[1] = 3;
              ok = false;
              break;
            }
            if (!mbar_wait_warp(tempty_bar(acc), acc_phase ^ 1u, abort_flag)) {
              if (leader && abort_flag[1] == 0) abort_flag[1] = 2;
              ok = false;
              break;
            }
          }
          tc_fence_after_sync();
          if (leader) {
            tc_mma_x4<kMmaF8, CTAS>(tmem_base + static_cast<uint32_t>(acc * BN), lo_p, lo_q, desc_hi, desc_hi, p.idesc, 0u, 2u, 2u);
            if constexpr (PAIR) {
              tc_commit_pair(done_bar(stage), 3);
            } else {
              tc_commit(done_bar(stage));
            }
          }
          __syncwarp();
          if (++stage == kStages) stage = 0, phase ^= 1u;
          if (++acc == kAccs) acc = 0, acc_phase ^= 1u;
        }
      }
    } else if (warp == 2) {
      // ------------------------------------------------------------ scales
      // Asynchronous copies, kAhead blocks ahead and across tiles: fetched by the warps that use them, scales cost those a trip to
      // L2 or HBM per block (4096^3, counted with clock reads: 510 of the 1710 cycles of a block).  A block's products are announced by
      // the tensor core and by this warp.  Step s waits for the products of block s - kAccs: they were begun after all of block
      // s - 2 kAccs - 1 had been added, so that its slot and those before it are free.
      constexpr int kRowCopies = 4, kColCopies = SCALES == kOfRows ? 1 : (BN + 31) / 32;
      int ahead_t = first, ahead_kb = 0, ahead_end = 0, to = 0;
      const float *row_from[kRowCopies], *col_from[kColCopies];
      const long long row_step = SWAP ? p.bs_block : p.as_block, col_step = SWAP ? p.as_block : p.bs_block;
      auto point_at = [&](int t) {   // the first block of tile t, or of the next one that has blocks
        for (; t < total; t += units) {
          const Tile x = tile_at(t);
          if (x.kb0 == x.kb1) continue;
          const float *sa = p.a_scale + x.kb0 * p.as_block, *sb = p.b_scale + (p.terms ? 0 : x.group) * p.bs_group + x.kb0 * p.bs_block;
          auto of_token = [&](int i) { return sa + min(x.row0 + i, p.m - 1) * p.as_row; };
          auto of_weight = [&](int i) { return sb + (min(x.n0 + i, p.n - 1) >> p.b_shift) * p.bs_row; };
#pragma unroll
          for (int e = 0; e < kRowCopies; ++e) {
            const int i = side * 128 + e * 32 + lane;
            row_from[e] = SWAP ? of_weight(i) : of_token(i);
          }
#pragma unroll
          for (int e = 0; e < kColCopies; ++e) {
            const int i = SCALES == kOfRows ? lane * 128 : e * 32 + lane;
            col_from[e] = SWAP ? of_token(i) : of_weight(i);
          }
          ahead_kb = x.kb0, ahead_end = x.kb1;
          break;
        }
        ahead_t = t;
      };
      auto request = [&]() {   // the next block's scales
        if (ahead_t < total) {
          const uint32_t at = scale_ring + static_cast<uint32_t>((to * Cfg::kSlotFloats + lane) * 4);
#pragma unroll
          for (int e = 0; e < kRowCopies; ++e) {
            copy_async_4(at + e * 128, row_from[e]);
            row_from[e] += row_step;
          }
#pragma unroll
          for (int e = 0; e < kColCopies; ++e) {
            if (SCALES == kOfRows ? lane < BN / 128 : e * 32 + lane < BN) copy_async_4(at + 512 + e * 128, col_from[e]);
            col_from[e] += col_step;
          }
          if (++ahead_kb == ahead_end) point_at(ahead_t + units);
        }
        copy_async_commit();
        if (++to == Cfg::kSlots) to = 0;
      };
      point_at(first);
      for (int e = 0; e < Cfg::kAhead; ++e) request();
      int stage = 0, old_stage = 0, step = 0;   // of this block, and of the block kAccs before it
      uint32_t old_phase = 0;
      bool ok = true;
      for (int t = first; t < total && ok; t += units) {
        const Tile x = tile_at(t);
        for (int kb = x.kb0; kb < x.kb1; ++kb) {
          if (step < kAccs) {
            ++step;
          } else {
            if (!mbar_wait_warp(done_bar(old_stage), old_phase, abort_flag)) {
              if (lane == 0 && abort_flag[1] == 0) abort_flag[1] = 5;
              ok = false;
              break;
            }
            if (++old_stage == kStages) old_stage = 0, old_phase ^= 1u;
          }
          request();
          copy_async_wait<Cfg::kAhead>();
          __syncwarp();
          if (lane == 0) mbar_arrive(done_bar(stage));
          if (++stage == kStages) stage = 0;
        }
      }
      copy_async_wait<0>();
    }
  } else {
    // ------------------------------------------------------------ sums
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::kSumRegs));
    const int w = warp - 4;
    constexpr int kCols = Cfg::kCols;
    const int quarter = warp & 3, first_col = (w >> 2) * kCols;   // TMEM lanes [32 quarter, ...), columns [first_col, ...)
    // Columns loaded from TMEM at a time.  Two warps take turns on a scheduler, so one set of registers is enough; what counts is
    // that the compiler finds them beside the sums without moving any (4096^3, bf16: 64 at a time 64.8 us, 16 67.1, 32 74.6; with
    // scales of rows and columns 16 at a time 89, 32 95, 64 95, and 100 where the two scales are multiplied first).
    constexpr int kChunk = kCols < 16 ? kCols : (SCALES == kOfRows && kCols >= 64 ? 64 : 16), kChunks = kCols / kChunk;
    const uint32_t t_mine = tmem_base + static_cast<uint32_t>(first_col) + (static_cast<uint32_t>(quarter * 32) << 16);
    int acc = 0, slot = 0, stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t tempty_at_first = PAIR ? mapa_rank(tempty_bar(0), 0) : 0u;
    // Waits for the accumulator's block and its scales; false: gave up.
    auto ready = [&]() {
      if (!mbar_wait_warp(done_bar(stage), phase, abort_flag)) {
        if (lane == 0 && abort_flag[1] == 0) abort_flag[1] = 4;
        return false;
      }
      if (++stage == kStages) stage = 0, phase ^= 1u;
      tc_fence_after_sync();
      return true;
    };
    // Hands the accumulator back (all of it is in registers) and goes on to the next.
    auto release = [&]() {
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) {
          mbar_arrive_cluster(tempty_at_first + 8u * acc);
        } else {
          mbar_arrive(tempty_bar(acc));
        }
      }
      if (++acc == kAccs) acc = 0;
    };
    for (int t = first; t < total && ok; t += units) {
      const Tile x = tile_at(t);
      const int i = side * 128 + quarter * 32 + lane;   // the accumulator row of this thread
      uint64_t sum[kCols / 2];
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j) sum[j] = 0;
      uint64_t row2 = 0;       // the row's scale (kOfRows: times that of the columns)
      uint32_t scales = 0;     // the columns' ones
      auto take_scales = [&]() {
        const uint32_t at = scale_ring + static_cast<uint32_t>(slot * Cfg::kSlotFloats * 4);
        float rs = ld_shared_f32(at + (quarter * 32 + lane) * 4);
        if constexpr (SCALES == kOfRows) rs *= ld_shared_f32(at + 512u + (first_col / 128) * 4);
        row2 = pack2(rs, rs);
        scales = at + 512u + first_col * 4;
        if (++slot == Cfg::kSlots) slot = 0;
      };
      auto add = [&](uint32_t (&v)[kChunk], int c) {
#pragma unroll
        for (int e = 0; e < kChunk; e += 4) {
          uint64_t v0 = pack2(v[e], v[e + 1]), v1 = pack2(v[e + 2], v[e + 3]);
          if constexpr (SCALES != kOfRows) {
            const uint4 u = ld_shared_v4(scales + (c + e) * 4);
            v0 = mul2(v0, pack2(u.x, u.y)), v1 = mul2(v1, pack2(u.z, u.w));
          }
          fma2(sum[(c + e) / 2], v0, row2);
          fma2(sum[(c + e) / 2 + 1], v1, row2);
        }
      };
      for (int kb = x.kb0; kb < x.kb1 && ok; ++kb) {
        ok = ready();
        if (!ok) break;
        const uint32_t at = t_mine + static_cast<uint32_t>(acc * BN);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          uint32_t v[kChunk];
          tmem_ld<kChunk>(at + c * kChunk, v);
          if (c == 0) take_scales();
          tmem_ld_wait();
          if (c == kChunks - 1) release();
          add(v, c * kChunk);
        }
      }
      if (!ok) break;
      if constexpr (SWAP) {
        if (Cfg::kSplits && p.split > 1) {
#pragma unroll
          for (int j = 0; j < kCols / 2; ++j) {
            const float2 v = unpack2(sum[j]);
            part[(first_col + 2 * j) * 128 + i] = v.x;
            part[(first_col + 2 * j + 1) * 128 + i] = v.y;
          }
        } else if (x.n0 + i < p.n) {
          // (the type and the first address outside the loop: with both inside, 64 columns took 27 of 51 us of a launch)
          const long long base = (p.terms ? x.group * p.stride_c : 0) + (x.row0 + first_col) * p.ldc + x.n0 + i;
          const int rows = x.row_end - x.row0 - first_col;
          auto leave = [&](auto* to, auto round) {
            to += base;
#pragma unroll
            for (int j = 0; j < kCols; ++j) {
              const float2 v = unpack2(sum[j / 2]);
              if (j < rows) *to = round(j & 1 ? v.y : v.x);
              to += p.ldc;
            }
          };
          if (p.out_dtype == PMLB_F32) {
            leave(static_cast<float*>(p.out), [](float v) { return v; });
          } else if (p.out_dtype == PMLB_BF16) {
            leave(static_cast<__nv_bfloat16*>(p.out), [](float v) { return __float2bfloat16_rn(v); });
          } else {
            leave(static_cast<__half*>(p.out), [](float v) { return __float2half_rn(v); });
          }
        }
      } else {
        if (Cfg::kSplits && p.split > 1) {
#pragma unroll
          for (int j = 0; j < kCols; j += 4) {
            const float2 a = unpack2(sum[j / 2]), b = unpack2(sum[j / 2 + 1]);
            st_shared_v4(out_stage + part_piece<BN>(i, (first_col + j) / 4),
                         make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y)));
          }
          continue;
        }
        // The results are rounded into shared memory and leave by TMA while the warp goes on with the next tile (written by the
        // warp itself, they held it up for 2 us per tile: no MMAs in that time, as both accumulators were full).
        const int row = x.row0 + side * 128 + quarter * 32, col = x.n0 + first_col;
        const int rows = min(x.row_end - row, 32);
        if (rows > 0) {
          const uint32_t places = out_stage + static_cast<uint32_t>(w) * 8192u;
          // (a box that holds rows of the next group is stored row by row)
          const bool by_tma = p.out_wide && (rows == 32 || x.row_end == p.m);
          // 16 bits: the warp's boxes of 64 columns together, one fence and one group of copies.  f32: boxes of 32 columns one
          // after the other, in the two places by turns, the next written while the last one leaves.  Every box is a group of
          // copies, an empty one where it leaves by plain stores or lies behind the last column: the wait for all groups but the
          // newest says only then that the box two before, which lay in this place, has been read.
          auto leave = [&](auto wide_tag, auto first_tag, auto pack) {
            constexpr int kWide = decltype(wide_tag)::value, kFirst = decltype(first_tag)::value;
            constexpr int kBoxes = kWide == 32 ? 1 : kCols / kWide;
            const uint32_t at = places + (kFirst & 1) * 4096u;
            if (lane == 0) bulk_wait_group_read<kWide == 32 ? 1 : 0>();
            __syncwarp();
            const uint32_t mine = at + box_piece(lane, 0);
#pragma unroll
            for (int b = 0; b < kBoxes; ++b) {
#pragma unroll
              for (int q = 0; q < 8; ++q) st_shared_v4((mine ^ (q << 4)) + b * 4096, pack((kFirst + b) * kWide + q * (kWide / 8)));
            }
            // (a TMA store writes whole 16-byte units: a row that ends inside one would lose what lies behind it)
            const int c0 = col + kFirst * kWide;
            const bool whole = c0 + kBoxes * kWide <= p.n || p.n % (kWide / 8) == 0;
            if (by_tma && whole) fence_proxy_async_smem();
            __syncwarp();
            if (by_tma && whole) {
              if (lane == 0) {
                if (c0 < p.n) tma_store_3d(&map_c, at, c0, row, p.terms ? x.group : 0);
                if (kBoxes == 2 && c0 + kWide < p.n) tma_store_3d(&map_c, at + 4096, c0 + kWide, row, p.terms ? x.group : 0);
              }
            } else {
#pragma unroll 1
              for (int b = 0; b < kBoxes; ++b) {
                const int c = c0 + b * kWide;
                if (c < p.n) store_box(p, at + b * 4096, (p.terms ? x.group * p.stride_c : 0) + row * p.ldc + c, rows, p.n - c, lane);
              }
            }
            if (lane == 0) bulk_commit_group();
          };
          using std::integral_constant;
          if (p.out_dtype == PMLB_F32) {
            auto pack = [&](int j) {
              const float2 u = unpack2(sum[j / 2]), v = unpack2(sum[j / 2 + 1]);
              return make_uint4(__float_as_uint(u.x), __float_as_uint(u.y), __float_as_uint(v.x), __float_as_uint(v.y));
            };
            leave(integral_constant<int, 32>(), integral_constant<int, 0>(), pack);
            leave(integral_constant<int, 32>(), integral_constant<int, 1>(), pack);
            if constexpr (kCols > 64) {
              leave(integral_constant<int, 32>(), integral_constant<int, 2>(), pack);
              leave(integral_constant<int, 32>(), integral_constant<int, 3>(), pack);
            }
          } else if (p.out_dtype == PMLB_BF16) {
            leave(integral_constant<int, 64>(), integral_constant<int, 0>(), [&](int j) { return pack_eight<true>(&sum[j / 2]); });
          } else {
            leave(integral_constant<int, 64>(), integral_constant<int, 0>(), [&](int j) { return pack_eight<false>(&sum[j / 2]); });
          }
        }
      }
    }
    if (lane == 0) bulk_wait_group_read<0>();   // (shared memory stays until the last box has left)
  }

  __syncwarp();
  tc_fence_before_sync();
  if (PAIR || p.split > 1) {
    cluster_sync_threads();
  } else {
    __syncthreads();
  }
  const bool failed = abort_flag[0] != 0;
  if constexpr (Cfg::kSplits) {
    if (p.split > 1 && first < total && !failed) {
      // The cluster's one tile: each CTA adds a run of its rows (SWAP: columns of the accumulator, which are rows of C) over all
      // parts, in the order of the blocks.
      const Tile x = tile_at(first);
      if constexpr (SWAP) {
        const int begin = BN * 128 / p.split * rank, end = BN * 128 / p.split * (rank + 1);
        const long long base = (p.terms ? x.group * p.stride_c : 0) + x.n0;
        for (int e = begin + static_cast<int>(threadIdx.x); e < end; e += Cfg::kThreads) {
          const int j = e >> 7, i = e & 127;
          const int row = x.row0 + j;
          if (row >= x.row_end || x.n0 + i >= p.n) continue;
          float v[8];
#pragma unroll
          for (int r = 0; r < 8; ++r) v[r] = r < p.split ? ld_cluster_f32(mapa_rank(smem_u32(part + e), static_cast<uint32_t>(r))) : 0.f;
#pragma unroll
          for (int r = 1; r < 8; ++r) v[0] += v[r];
          store_one(p, base + row * p.ldc + i, v[0]);
        }
      } else {
        constexpr int kPieces = BN / 4;
        const int begin = 128 / p.split * rank * kPieces, end = 128 / p.split * (rank + 1) * kPieces;
        const long long base = p.terms ? x.group * p.stride_c : 0;
        for (int e = begin + static_cast<int>(threadIdx.x); e < end; e += Cfg::kThreads) {
          const int row = x.row0 + e / kPieces, col = x.n0 + e % kPieces * 4;
          if (row >= x.row_end || col >= p.n) continue;
          const uint32_t at = out_stage + part_piece<BN>(e / kPieces, e % kPieces);
          float4 v[8];
#pragma unroll
          for (int r = 0; r < 8; ++r) v[r] = r < p.split ? ld_cluster_v4(mapa_rank(at, static_cast<uint32_t>(r))) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int r = 1; r < 8; ++r) v[0].x += v[r].x, v[0].y += v[r].y, v[0].z += v[r].z, v[0].w += v[r].w;
          store_four(p, base + row * p.ldc + col, v[0], p.n - col);
        }
      }
    }
  }
  if (failed) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0, abort_flag[1] != 0 ? abort_flag[1] : 9);
    // copies and MMAs still in flight get a bounded time before TMEM and shared memory go away
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 2000000ull) __nanosleep(2000);
  }
  __syncwarp();
  if (PAIR || p.split > 1) {
    cluster_sync_threads();   // no CTA leaves while another may still read its part, or before its MMAs have ended
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after_sync();
    if constexpr (PAIR) {
      tmem_dealloc_pair(tmem_base, Cfg::kTmemCols);
    } else {
      tmem_dealloc(tmem_base, Cfg::kTmemCols);
    }
  }
}

using KernelPtr = void (*)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const BlockGemmParams);

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
cudaError_t launch(const CUtensorMap& mp, const CUtensorMap& mq, const CUtensorMap& mc, const BlockGemmParams& p, int grid, int dev, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(Cfg::kThreads);
  cfg.dynamicSmemBytes = Cfg::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0] = dependent_launch_attribute();
  attr[1].id = cudaLaunchAttributeClusterDimension;
  const int share = Cfg::CTAS == 2 ? 2 : p.split;
  attr[1].val.clusterDim.x = share;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = share > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, instance<Cfg>(dev), mp, mq, mc, p);
}

// Clusters of `split` CTAs that the device holds at once (a GPC holds whole clusters only; every kernel here leaves room for one
// CTA per SM).
int resident_clusters(int dev, int split, int sms) {
  static std::mutex mutex;
  static int known[64][9];   // per device and split, 0 = not asked yet
  if (split == 1 || dev < 0 || dev >= 64) return sms / split;
  std::lock_guard<std::mutex> lock(mutex);
  if (known[dev][split] == 0) {
    using Cfg = BlockCfg<128, false, kOfRows>;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(split);
    cfg.blockDim = dim3(Cfg::kThreads);
    cfg.dynamicSmemBytes = Cfg::kSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, instance<Cfg>(dev), &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = 1;
    }
    known[dev][split] = n;
  }
  return known[dev][split];
}

struct Choice {
  bool swap = false, pair = false;
  int bn = 128, split = 1;
};

// Which tiles, and how many CTAs share the blocks of one.  Few rows: weights on the accumulator's rows and as few columns as hold
// the rows -- up to 64, or twice the average of groups, so that most groups are one tile (16 rows to each of 8 groups, 2048 x
// 1024: 5.7 us with 32 columns, 7.9 with 16; 48 rows to each of 16 groups, 1024 x 2048: single tiles 10.6 us, few rows 15.3).
// Else the smaller estimate, in cycles, of pairs of CTAs on 256 x 256 and of single ones on 128 x 128.  Measured per block: pairs
// 700 (1150 where rows and columns have scales of their own), single CTAs 540 (640), which is what an SM takes in of operands;
// around the blocks of a tile 3300 and 1500; 6500 for clusters that add parts up.  (4096 wide and deep, pairs / single / with K
// split: 100 rows 17.8 / 13.5 / 10.1 us, 256 18.0 / 13.9 / 13.0, 1024 20.5 / 26.0.)
Choice choose(const pmlb_block_gemm_desc& d, int dev, int sms) {
  const bool by_rows = d.groups > 0 && d.group_dim == PMLB_GROUP_ROWS, by_terms = d.groups > 0 && !by_rows;
  const int num_kb = (d.k + kBlock - 1) / kBlock, kb = by_terms ? (num_kb + d.groups - 1) / d.groups : num_kb;
  const int groups = by_rows ? std::min(d.groups, d.m) : 1;   // with rows of their own, at most
  const int rows = static_cast<int>((static_cast<long long>(d.m) + groups - 1) / groups);
  // (groups of rows end inside a tile: half a tile each on average)
  auto tiles = [&](int tile_rows, int tile_cols) {
    const double high = by_rows ? static_cast<double>(d.m) / tile_rows + 0.5 * groups : std::ceil(static_cast<double>(d.m) / tile_rows);
    return high * std::ceil(static_cast<double>(d.n) / tile_cols) * (by_terms ? d.groups : 1);
  };
  // (a launch with K split has one tile per cluster: the tiles there may be, not those there are on average)
  auto fits = [&](int tile_rows, int split) {
    const double high = by_rows ? d.m / tile_rows + groups : std::ceil(static_cast<double>(d.m) / tile_rows);
    return high * std::ceil(d.n / 128.0) * (by_terms ? d.groups : 1) <= resident_clusters(dev, split, sms);
  };
  Choice c;
  const int columns = groups > 1 ? 2 * rows : rows;
  if (d.tiles == PMLB_BLOCK_TILES_FEW || (d.tiles == 0 && columns <= 64)) {
    c.swap = true;
    c.bn = columns <= 16 ? 16 : (columns <= 32 ? 32 : 64);
    while (c.split < 8 && kb >= c.split * 4 && fits(c.bn, c.split * 2)) c.split *= 2;
    return c;
  }
  const bool both = d.b_scale_rows == 1;
  double best = std::ceil(tiles(256, 256) / (sms / 2)) * (kb * (both ? 1150.0 : 700.0) + 3300.0);
  c.pair = true, c.bn = 256;
  if (d.tiles == PMLB_BLOCK_TILES_PAIR) return c;
  if (d.tiles == PMLB_BLOCK_TILES_SINGLE) best = INFINITY;
  for (int split = 1; split <= 8 && split <= kb; split *= 2) {
    if (split > 1 && !fits(128, split)) break;
    const double waves = split > 1 ? 1.0 : std::ceil(tiles(128, 128) / sms);
    const double t = waves * ((kb + split - 1) / split * (both ? 640.0 : 540.0) + 1500.0) + (split > 1 ? 6500.0 : 0.0);
    if (t < best) best = t, c.pair = false, c.bn = 128, c.split = split;
  }
  return c;
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
  p.b_step = by_rows && d.stride_b == 0 ? 0 : 1;
  const bool many_c = by_terms && d.groups > 1;   // (a single group has no neighbour)
  p.out = c, p.ldc = d.ldc, p.stride_c = many_c ? d.stride_c : 0, p.out_dtype = d.out_dtype;
  const long long ob = d.out_dtype == PMLB_F32 ? 4 : 2;
  const long long bits = static_cast<long long>(reinterpret_cast<uintptr_t>(c)) | (d.ldc * ob) | (p.stride_c * ob);
  p.out_wide = bits % 16 == 0;
  p.status = status;

  const Choice choice = choose(d, dev, sms);
  const bool swap = choice.swap, pair = choice.pair;
  const int bn = choice.bn, ctas = pair ? 2 : 1;
  const int tile_rows = swap ? bn : 128 * ctas, tile_cols = swap ? 128 * ctas : bn;
  p.tiles_m = (d.m + tile_rows - 1) / tile_rows;
  p.tiles_n = (d.n + tile_cols - 1) / tile_cols;
  // (groups of rows: at most one tile more than whole ones for each group that has rows)
  const long long row_tiles = by_rows ? d.m / tile_rows + std::min(d.groups, d.m) : p.tiles_m;
  const long long tiles = row_tiles * p.tiles_n * (by_terms ? d.groups : 1);
  if (tiles > 0x07ffffff) {
    *err = "block_gemm: too many tiles";
    return PMLB_ERR_UNSUPPORTED;
  }
  p.split = choice.split;
  const int grid = p.split > 1 ? static_cast<int>(tiles) * p.split : static_cast<int>(std::min<long long>(tiles, sms / ctas)) * ctas;
  // bits: [4,6) f32 accumulators, [7,10) and [10,13) formats of the two operands, [17,23) N >> 3, [24,29) M >> 4
  p.idesc = 1u << 4 | f8_format(swap ? d.b_dtype : d.a_dtype) << 7 | f8_format(swap ? d.a_dtype : d.b_dtype) << 10 |
            static_cast<uint32_t>(bn >> 3) << 17 | static_cast<uint32_t>(8 * ctas) << 24;

  CUtensorMap ma, mb, mc;
  std::memset(&mc, 0, sizeof(mc));
  // (a CTA of a pair fetches 128 rows of one operand and its half of the other)
  const int box_a = tile_rows / ctas, box_b = tile_cols / ctas;
  if (!tc_encode_bytes(&ma, a, d.k, d.m, 1, d.lda, 16, box_a, err)) return PMLB_ERR_INVALID;
  const bool many_b = by_rows && d.stride_b != 0;
  if (!tc_encode_bytes(&mb, b, d.k, d.n, many_b ? d.groups : 1, d.ldb, many_b ? d.stride_b : 16, box_b, err)) return PMLB_ERR_INVALID;
  if (!swap && p.out_wide &&
      !tc_encode_boxes(&mc, d.out_dtype, c, d.n, d.m, many_c ? d.groups : 1, d.ldc, many_c ? d.stride_c : 8, err)) {
    return PMLB_ERR_INVALID;
  }
  cudaError_t e = cudaSuccess;
  // Rows and columns of an accumulator have scales of their own; where its rows are rows of B, the columns are tokens, which always do.
  const bool both = d.b_scale_rows == 1;
  if (swap) {
    if (bn == 16) {
      e = launch<BlockCfg<16, true, kOfBoth>>(mb, ma, mc, p, grid, dev, stream);
    } else if (bn == 32) {
      e = launch<BlockCfg<32, true, kOfBoth>>(mb, ma, mc, p, grid, dev, stream);
    } else {
      e = launch<BlockCfg<64, true, kOfBoth>>(mb, ma, mc, p, grid, dev, stream);
    }
  } else if (pair) {
    e = both ? launch<BlockCfg<256, false, kOfBoth, 2>>(ma, mb, mc, p, grid, dev, stream) : launch<BlockCfg<256, false, kOfRows, 2>>(ma, mb, mc, p, grid, dev, stream);
  } else {
    e = both ? launch<BlockCfg<128, false, kOfBoth>>(ma, mb, mc, p, grid, dev, stream) : launch<BlockCfg<128, false, kOfRows>>(ma, mb, mc, p, grid, dev, stream);
  }
  if (e != cudaSuccess) {
    *err = std::string("block_gemm launch: ") + cudaGetErrorString(e);
    return PMLB_ERR_CUDA;
  }
  return 0;
}

}  // namespace pmlb
