// Matrix products of the linear layers on tcgen05.
//
//   D[m][n] = act(sum_k A(m, k) B(n, k) + bias[n]) + residual[m][n]
//
// A persistent kernel: one warp loads 64-deep operand tiles by TMA into a ring of shared
// memory stages, one warp issues the MMAs into TMEM accumulators, warps of an epilogue read them
// back, apply the epilogue and hand finished 128-byte wide tiles to TMA stores. Two
// accumulator sets let the epilogue of one tile run under the main loop of the next. Either
// operand may be K-major or MN-major (dx reads W, dW reads dz and x as they lie in memory).
//
// Tiles. A 128 x 256 tile per CTA needs 96 operand bytes per clock and SM to keep the tensor
// core busy (two 16-bit operands, 384 rows of 64 per 512 cycles), more than an SM's share of
// L2. A pair of CTAs that multiply one 256 x 256 tile together (cta_group::2: each holds its
// own 128 rows of A and half of B) needs 64, so large products run on pairs; smaller ones
// on single CTAs with 128 or 64 columns, so that all SMs have a tile.
//
// float32 operands arrive as three bfloat16 terms each (x = x0 + x1 + x2, 24 significant
// bits); the six products down to 2^-24 are summed. The tensor core truncates each
// accumulation, an error that grows with the number of steps, so the leading product
// x0 y0 is collected in TMEM for 256 of k only and then added to float32 registers, while
// the five small products, 2^-8 of it and less, keep one accumulator for the whole tile.
//
// A long k with few tiles is cut into splits, whose float32 partial tiles a second launch
// adds in order before the epilogue: repeated calls give the same bits.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "activation.cuh"
#include "layers.cuh"
#include "pair.cuh"
#include "product.cuh"

namespace cnd {
namespace layers {
namespace {

constexpr int kBM = 128;
// Depth of an operand stage. Three-term operands take 32: six tiles of 64 leave room for two
// stages only.
constexpr int block_depth(int parts) { return parts == 3 ? 32 : 64; }
constexpr int kGroupThreads = 128;  // an epilogue group: four warps
constexpr int block_threads(int groups) { return 64 + groups * kGroupThreads; }
constexpr uint32_t kUnitBytes = kBM * 128;  // staging tile: 128 rows of 128 bytes
constexpr uint32_t kSharedLimit = 232448;
constexpr int kMostStages = 8;
constexpr int kChunkBlocks = 8;  // k blocks per float32 accumulation (three-term operands)
constexpr uint32_t kSiteLoad = 0x501, kSiteMma = 0x502, kSiteAccumulator = 0x503,
                   kSiteEpilogue = 0x504, kSiteDrain = 0x505, kSiteResidual = 0x506;

struct Maps {
  CUtensorMap a, b, out, pre, residual;
};

struct KernelArgs {
  int64_t m, n;
  int tiles_m, tiles_n, splits, k_blocks;
  int stages;         // operand stages
  int buffers, sets;  // staging tiles of an epilogue group; how many units they hold
  uint32_t idesc;
  uint32_t a_step, b_step;  // descriptor units (16 bytes) per 16 of k
  uint32_t a_lbo, b_lbo;
  uint32_t a_sbo, b_sbo, a_swizzle, b_swizzle;
  int a_k_major, b_k_major;
  int act, tma_out;
  int tma_residual;  // its rows are 16-byte aligned
  const void* bias;
  const void* residual;
  void* d;
  void* pre;
  unsigned int* error;
  uint64_t timeout_ns;
};

// Tiles in groups of 8 rows of tiles, walked down the rows first, so that the tiles in
// flight share both operands in L2.
__device__ __forceinline__ void tile_of(const KernelArgs& a, int index, int* tm, int* tn) {
  constexpr int kGroup = 8;
  const int per_group = kGroup * a.tiles_n;
  const int group = index / per_group;
  const int first = group * kGroup;
  const int rows = min(kGroup, a.tiles_m - first);
  const int inside = index - group * per_group;
  *tm = first + inside % rows;
  *tn = inside / rows;
}

template <int kPair>
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, dev::ErrorWord err,
                                     uint32_t site, uint64_t timeout_ns) {
  if constexpr (kPair == 1) {
    return dev::mbar_wait(bar, parity, err, site, timeout_ns);
  } else {
    if (dev::mbar_try_wait_cluster(bar, parity)) return true;
    const uint64_t start = dev::global_timer_ns();
    for (uint32_t spin = 0;; ++spin) {
      if (dev::mbar_try_wait_cluster(bar, parity)) return true;
      if ((spin & 63u) == 63u && dev::global_timer_ns() - start > timeout_ns) {
        atomicCAS(err.word, 0u, site);
        return false;
      }
    }
  }
}

template <int kPair>
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, dev::ErrorWord err,
                                          uint32_t site, uint64_t timeout_ns) {
  return __all_sync(0xffffffffu, wait<kPair>(bar, parity, err, site, timeout_ns)) != 0;
}

// Writes 32 values of a row (columns half * 32 ... of a unit) into a 128-byte-wide staging
// tile with the 128-byte TMA swizzle (16-byte chunk c of row r at chunk c ^ (r & 7)).
template <typename Out>
__device__ __forceinline__ void stage_row(uint8_t* tile, int row, int half, const Two (&v)[16]) {
  uint8_t* base = tile + row * 128;
  if constexpr (sizeof(Out) == 4) {
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      *reinterpret_cast<ulonglong2*>(base + ((c ^ (row & 7)) * 16)) =
          make_ulonglong2(v[2 * c].bits, v[2 * c + 1].bits);
    }
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      *reinterpret_cast<uint4*>(base + (((half * 4 + c) ^ (row & 7)) * 16)) =
          make_uint4(narrow2<Out>(v[4 * c]), narrow2<Out>(v[4 * c + 1]),
                     narrow2<Out>(v[4 * c + 2]), narrow2<Out>(v[4 * c + 3]));
    }
  }
}

// Copies between a staging tile and rows of a matrix that TMA cannot address, a warp per row
// and eight rows in flight: neighbouring lanes hold neighbouring columns.
template <bool kStore, typename Out>
__device__ __forceinline__ void copy_unit(uint8_t* tile, Out* d, int64_t row0, int64_t col0,
                                          int64_t m, int64_t n, int warp, int lane) {
  constexpr int kColumns = 128 / sizeof(Out), kEach = kColumns / 32;
  for (int r0 = warp; r0 < kBM && row0 + r0 < m; r0 += 32) {
    Out v[8][kEach];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int r = r0 + 4 * j, c = e * 32 + lane, byte = c * static_cast<int>(sizeof(Out));
        Out* at = reinterpret_cast<Out*>(tile + r * 128 + (((byte >> 4) ^ (r & 7)) << 4) + (byte & 15));
        const bool inside = row0 + r < m && col0 + c < n;
        if constexpr (kStore) {
          v[j][e] = *at;
        } else {
          v[j][e] = inside ? d[(row0 + r) * n + col0 + c] : narrow<Out>(0.0f);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int r = r0 + 4 * j, c = e * 32 + lane, byte = c * static_cast<int>(sizeof(Out));
        Out* at = reinterpret_cast<Out*>(tile + r * 128 + (((byte >> 4) ^ (r & 7)) << 4) + (byte & 15));
        const bool inside = row0 + r < m && col0 + c < n;
        if constexpr (kStore) {
          if (inside) d[(row0 + r) * n + col0 + c] = v[j][e];
        } else {
          *at = v[j][e];
        }
      }
    }
  }
}

// 32 residual values of a row, from a staging tile.
template <typename Out>
struct Residual {
  static constexpr int kPer = 16 / sizeof(Out);
  Pack<Out, kPer> q[32 / kPer];

  __device__ __forceinline__ void take(const uint8_t* tile, int row, int half) {
    constexpr int kChunks = 32 / kPer;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      q[c] = *reinterpret_cast<const Pack<Out, kPer>*>(
          tile + row * 128 + (((half * kChunks + c) ^ (row & 7)) * 16));
    }
  }

  __device__ __forceinline__ Two pair(int i) const {
    return two(widen(q[2 * i / kPer].v[2 * i % kPer]),
               widen(q[(2 * i + 1) / kPer].v[(2 * i + 1) % kPer]));
  }
};

template <int kPair, int kBN, int kParts, int kGroups, typename Out>
__global__ void __launch_bounds__(block_threads(kGroups), 1)
    product_tc_kernel(const __grid_constant__ Maps maps, const __grid_constant__ KernelArgs a) {
  constexpr bool kExact = sizeof(Out) == 4;
  constexpr int kColsB = kBN / kPair;  // rows of B that this CTA holds
  constexpr int kBK = block_depth(kParts);
  constexpr uint32_t kPartA = kBM * kBK * 2, kPartB = kColsB * kBK * 2;
  constexpr uint32_t kStageBytes = kParts * (kPartA + kPartB);
  constexpr int kUnit = 128 / sizeof(Out);      // columns of a staging tile
  constexpr int kGroupCols = kBN / kGroups;     // columns of an epilogue group
  constexpr int kEpilogueWarps = 4 * kGroups;
  constexpr int kHalves = kGroupCols / 32;
  constexpr uint32_t kColumns = kParts == 1 ? 2 * kBN : 512;

  extern __shared__ __align__(1024) uint8_t shared[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(shared) + 1023) & ~uintptr_t{1023});
  uint8_t* staging = smem + a.stages * kStageBytes;
  float* bias_s = reinterpret_cast<float*>(staging + kGroups * a.buffers * kUnitBytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(bias_s + kBN);
  uint64_t* empty = full + kMostStages;
  uint64_t* acc_full = empty + kMostStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* cross_empty = acc_empty + 2;  // three-term operands: the small products' sets
  uint64_t* residual_full = cross_empty + 2;  // a group's residual tile has arrived
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(residual_full + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = kPair == 2 ? dev::cluster_rank() : 0;
  const dev::ErrorWord err{a.error};

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      dev::mbar_init(&full[s], 1);
      dev::mbar_init(&empty[s], 1);
    }
    for (int g = 0; g < kGroups; ++g) dev::mbar_init(&residual_full[g], 1);
    for (int s = 0; s < 2; ++s) {
      dev::mbar_init(&acc_full[s], 1);
      dev::mbar_init(&acc_empty[s], kPair * kEpilogueWarps);
      dev::mbar_init(&cross_empty[s], kPair * kEpilogueWarps);
    }
    dev::fence_barrier_init();
  }
  if (warp == 0) {
    __syncwarp();
    dev::tmem_alloc_pair<kPair>(tmem_slot, kColumns);
  }
  dev::tc_fence_before();
  if constexpr (kPair == 2) {
    dev::cluster_sync();
  } else {
    __syncthreads();
  }
  dev::tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int workers = static_cast<int>(gridDim.x) / kPair;
  const int worker = static_cast<int>(blockIdx.x) / kPair;
  const int items = a.tiles_m * a.tiles_n * a.splits;

  if (warp == 0) {
    // ---- TMA loads: the converged warp, elect.sync issues ----
    if (lane == 0) {
      dev::prefetch_tensormap(&maps.a);
      dev::prefetch_tensormap(&maps.b);
    }
    __syncwarp();
    const uint32_t full_here = dev::smem_u32(full);
    const uint32_t full_signal = kPair == 2 ? dev::map_to_rank(full, 0) : full_here;
    const uint32_t stages_at = dev::smem_u32(smem);
    int stage = 0;
    uint32_t phase = 0, issued = 0;
    bool ok = true;
    for (int item = worker; item < items && ok; item += workers) {
      const int split = item % a.splits;
      int tm, tn;
      tile_of(a, item / a.splits, &tm, &tn);
      const int m0 = (tm * kPair + static_cast<int>(rank)) * kBM;
      const int n0 = tn * kBN + static_cast<int>(rank) * kColsB;
      const int first = static_cast<int>(static_cast<int64_t>(a.k_blocks) * split / a.splits);
      const int last = static_cast<int>(static_cast<int64_t>(a.k_blocks) * (split + 1) / a.splits);
      for (int kb = first; kb < last; ++kb) {
        if (!wait_warp<kPair>(&empty[stage], phase ^ 1u, err, kSiteLoad, a.timeout_ns)) {
          ok = false;
          break;
        }
        if (rank == 0) dev::mbar_expect_tx_warp(full_here + 8 * stage, kPair * kStageBytes);
        const uint32_t bar = full_signal + 8 * stage;
        const uint32_t dst = stages_at + stage * kStageBytes;
        const int k0 = kb * kBK;
        if (a.a_k_major) {
#pragma unroll
          for (int p = 0; p < kParts; ++p) {
            dev::tma_load_3d_to<kPair>(dst + p * kPartA, &maps.a, bar, k0, m0, p);
          }
        } else {
#pragma unroll
          for (int p = 0; p < kParts; ++p) {
#pragma unroll
            for (int i = 0; i < kBM / 64; ++i) {
              dev::tma_load_3d_to<kPair>(dst + p * kPartA + i * (kBK * 128), &maps.a, bar,
                                         m0 + 64 * i, k0, p);
            }
          }
        }
        if (a.b_k_major) {
#pragma unroll
          for (int p = 0; p < kParts; ++p) {
            dev::tma_load_3d_to<kPair>(dst + kParts * kPartA + p * kPartB, &maps.b, bar, k0, n0, p);
          }
        } else {
#pragma unroll
          for (int p = 0; p < kParts; ++p) {
#pragma unroll
            for (int i = 0; i < kColsB / 64; ++i) {
              dev::tma_load_3d_to<kPair>(dst + kParts * kPartA + p * kPartB + i * (kBK * 128),
                                         &maps.b, bar, n0 + 64 * i, k0, p);
            }
          }
        }
        ++issued;
        if (++stage == a.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    // The last loads of each stage land before the block may exit, or have had a bounded time to:
    // MMAs that gave up have not waited for them. (A pair's loads all signal the leader.)
    for (int left = rank == 0 ? min(issued, static_cast<uint32_t>(a.stages)) : 0; left > 0; --left) {
      if (stage == 0) {
        stage = a.stages;
        phase ^= 1u;
      }
      --stage;
      wait_warp<kPair>(&full[stage], phase, err, kSiteDrain, a.timeout_ns / 8 + 1);
    }
  } else if (warp == 1) {
    // ---- MMAs: the leader CTA's warp, converged; elect.sync issues ----
    if (rank == 0) {
      const uint32_t base = dev::warp_uniform(tmem);
      const uint64_t a_hi = dev::make_smem_desc(0, a.a_lbo, a.a_sbo, a.a_swizzle);
      const uint64_t b_hi = dev::make_smem_desc(0, a.b_lbo, a.b_sbo, a.b_swizzle);
      int stage = 0;
      uint32_t phase = 0;
      int set = 0, cross = 0;
      uint32_t set_phase = 0, cross_phase = 0;
      bool ok = true;
      for (int item = worker; item < items && ok; item += workers) {
        const int split = item % a.splits;
        const int first = static_cast<int>(static_cast<int64_t>(a.k_blocks) * split / a.splits);
        const int last = static_cast<int>(static_cast<int64_t>(a.k_blocks) * (split + 1) / a.splits);
        if constexpr (kParts == 3) {
          if (!wait_warp<kPair>(&cross_empty[cross], cross_phase ^ 1u, err, kSiteAccumulator,
                                a.timeout_ns)) {
            break;
          }
        }
        const uint32_t d_cross = base + 256 + cross * kBN;
        for (int kb = first; kb < last && ok;) {
          if (!wait_warp<kPair>(&acc_empty[set], set_phase ^ 1u, err, kSiteAccumulator,
                                a.timeout_ns)) {
            ok = false;
            break;
          }
          dev::tc_fence_after();
          const uint32_t d = base + set * kBN;
          const int stop = kParts == 3 ? min(kb + kChunkBlocks, last) : last;
          for (const int begin = kb; kb < stop; ++kb) {
            if (!wait_warp<kPair>(&full[stage], phase, err, kSiteMma, a.timeout_ns)) {
              ok = false;
              break;
            }
            dev::tc_fence_after();
            const uint32_t as = dev::warp_uniform(dev::smem_u32(smem + stage * kStageBytes) >> 4);
            const uint32_t bs = as + (kParts * kPartA >> 4);
#pragma unroll
            for (int ks = 0; ks < kBK / 16; ++ks) {
              const uint32_t ao = as + ks * a.a_step, bo = bs + ks * a.b_step;
              if constexpr (kParts == 1) {
                dev::mma_f16_pair<kPair>(d, a_hi | ao, b_hi | bo, a.idesc, kb > begin || ks > 0);
              } else {
                constexpr uint32_t pa = kPartA >> 4, pb = kPartB >> 4;
                const uint32_t more = kb > first || ks > 0;
                dev::mma_f16_pair<kPair>(d_cross, a_hi | (ao + 2 * pa), b_hi | bo, a.idesc, more);
                dev::mma_f16_pair<kPair>(d_cross, a_hi | ao, b_hi | (bo + 2 * pb), a.idesc, 1);
                dev::mma_f16_pair<kPair>(d_cross, a_hi | (ao + pa), b_hi | (bo + pb), a.idesc, 1);
                dev::mma_f16_pair<kPair>(d_cross, a_hi | (ao + pa), b_hi | bo, a.idesc, 1);
                dev::mma_f16_pair<kPair>(d_cross, a_hi | ao, b_hi | (bo + pb), a.idesc, 1);
                dev::mma_f16_pair<kPair>(d, a_hi | ao, b_hi | bo, a.idesc, kb > begin || ks > 0);
              }
            }
            dev::mma_commit_pair<kPair>(&empty[stage]);
            if (++stage == a.stages) {
              stage = 0;
              phase ^= 1u;
            }
          }
          dev::mma_commit_pair<kPair>(&acc_full[set]);
          if (++set == 2) {
            set = 0;
            set_phase ^= 1u;
          }
        }
        if constexpr (kParts == 3) {
          if (++cross == 2) {
            cross = 0;
            cross_phase ^= 1u;
          }
        }
      }
    }
  } else {
    // ---- epilogue: groups of four warps, each kGroupCols columns of the tile ----
    const int group = (warp - 2) >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int epi = threadIdx.x - 64;
    const bool leader = (epi & (kGroupThreads - 1)) == 0;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t release = kPair == 2 ? dev::map_to_rank(&acc_empty[0], 0) : 0;
    const uint32_t release_cross = kPair == 2 ? dev::map_to_rank(&cross_empty[0], 0) : 0;
    uint8_t* own = staging + group * a.buffers * kUnitBytes;
    const auto free_set = [&](uint64_t* bars, uint32_t remote, int s) {
      dev::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (kPair == 2) {
          dev::mbar_arrive_cluster(remote + 8 * s);
        } else {
          dev::mbar_arrive(&bars[s]);
        }
      }
    };
    int set = 0, cross = 0, buffer = 0;
    uint32_t set_phase = 0, residual_phase = 0;
    // Once false, on without waiting: the named barriers take all warps of a group, and one that
    // left them would hold the others for good.
    bool ok = true;
    // The residual's tile of a unit comes by TMA into the staging tile that its output will
    // take: each thread then reads its row's part and writes the output over it. It is asked
    // for while the unit before is worked on where there is a second tile, else once the
    // one tile is free. (Read by warps of the epilogue, a row each, it had waited for memory
    // there: 1M x 64 -> 256 in bf16 475 us, by TMA 253, without a residual 179;
    // 16384 x 1024 -> 4096 147 us, by TMA 116.)
    const auto ask_residual = [&](int64_t row0, int64_t col, uint8_t* into) {
      if (!ok) return;
      dev::mbar_arrive_expect_tx(&residual_full[group], kUnitBytes);
      dev::tma_load_2d(into, &maps.residual, &residual_full[group], static_cast<int>(col),
                       static_cast<int>(row0));
    };
    bool asked = false;  // the coming unit's residual is on its way
    int bias_tile = -1;
    for (int item = worker; item < items; item += workers) {
      const int split = item % a.splits;
      int tm, tn;
      tile_of(a, item / a.splits, &tm, &tn);
      const int64_t row0 = static_cast<int64_t>(tm * kPair + static_cast<int>(rank)) * kBM;
      const int64_t col0 = static_cast<int64_t>(tn) * kBN + group * kGroupCols;
      // bias of the tile's columns, where they change and after every thread has finished the
      // previous tile's (two barriers of all epilogue warps, 15 us of 1M x 64 -> 256's 313 when
      // done for every tile)
      if (tn != bias_tile) {
        bias_tile = tn;
        dev::named_barrier(1, 32 * kEpilogueWarps);
        for (int c = epi; c < kBN; c += 32 * kEpilogueWarps) {
          const int64_t column = static_cast<int64_t>(tn) * kBN + c;
          bias_s[c] = a.bias != nullptr && column < a.n
                          ? widen(static_cast<const Out*>(a.bias)[column])
                          : 0.0f;
        }
        dev::named_barrier(1, 32 * kEpilogueWarps);
      }
      float sums[kParts == 3 ? kHalves : 1][32];
      if constexpr (kParts == 3) {
        const int first = static_cast<int>(static_cast<int64_t>(a.k_blocks) * split / a.splits);
        const int last = static_cast<int>(static_cast<int64_t>(a.k_blocks) * (split + 1) / a.splits);
        for (int kb = first; kb < last; kb += kChunkBlocks) {
          ok = ok && wait_warp<kPair>(&acc_full[set], set_phase, err, kSiteEpilogue, a.timeout_ns);
          dev::tc_fence_after();
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            uint32_t v[32];
            dev::tmem_load32(tmem + lanes + set * kBN + group * kGroupCols + h * 32, v);
            dev::tmem_load_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              sums[h][i] = kb == first ? __uint_as_float(v[i]) : sums[h][i] + __uint_as_float(v[i]);
            }
          }
          free_set(acc_empty, release, set);
          if (++set == 2) {
            set = 0;
            set_phase ^= 1u;
          }
        }
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          uint32_t v[32];
          dev::tmem_load32(tmem + lanes + 256 + cross * kBN + group * kGroupCols + h * 32, v);
          dev::tmem_load_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) sums[h][i] += __uint_as_float(v[i]);
        }
        free_set(cross_empty, release_cross, cross);
        cross ^= 1;
      } else {
        if (ok && !wait_warp<kPair>(&acc_full[set], set_phase, err, kSiteEpilogue, a.timeout_ns)) {
          ok = false;
          if (asked) {  // the residual tile on its way has a bounded time to land
            dev::mbar_wait_warp(&residual_full[group], residual_phase, err, kSiteDrain,
                                a.timeout_ns / 8 + 1);
          }
        }
        dev::tc_fence_after();
      }

      const uint32_t acc = tmem + lanes + set * kBN + group * kGroupCols;
      uint8_t *tile = own, *pre_tile = own;
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        constexpr int kHalvesPerUnit = kUnit / 32;
        if (h % kHalvesPerUnit == 0) {
          // a free staging tile for this unit (and one for its pre-activation): the stores of
          // all but the other sets of tiles have read their shared memory
          if (leader) {
            if (a.sets == 2) {
              dev::bulk_wait_group_read<1>();
            } else {
              dev::bulk_wait_group_read<0>();
            }
          }
          dev::named_barrier(2 + group, kGroupThreads);
          tile = own + buffer * kUnitBytes;
          pre_tile = own + (buffer + a.sets) * kUnitBytes;
          if (a.buffers == 1) pre_tile = tile;
          if (a.sets == 2) buffer ^= 1;
          // (one tile for all: after the pre-activation has left it)
          if (a.tma_residual && !asked && leader && !(a.buffers == 1 && a.pre != nullptr)) {
            ask_residual(row0, col0 + h * 32, tile);
          }
          asked = false;
        }
        Two v[16];
        if constexpr (kParts == 3) {
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = two(sums[h][2 * i], sums[h][2 * i + 1]);
        } else {
          uint32_t raw[32];
          dev::tmem_load32(acc + h * 32, raw);
          dev::tmem_load_wait();
          if (h + 1 == kHalves) free_set(acc_empty, release, set);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            v[i] = two(__uint_as_float(raw[2 * i]), __uint_as_float(raw[2 * i + 1]));
          }
        }
        const float* bias = bias_s + group * kGroupCols + h * 32;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const ulonglong2 b2 = *reinterpret_cast<const ulonglong2*>(bias + 2 * i);
          v[i] = add2(v[i], Two{b2.x});
          v[i + 1] = add2(v[i + 1], Two{b2.y});
        }
        const int64_t unit_col = col0 + (h / kHalvesPerUnit) * kUnit;
        const bool unit_done = h % kHalvesPerUnit == kHalvesPerUnit - 1;
        if (a.pre != nullptr) {
          stage_row<Out>(pre_tile, row, h % kHalvesPerUnit, v);
          if (a.buffers == 1) {
            // one staging tile: the pre-activation leaves before the output is staged (units
            // of one half only: float32)
            dev::fence_proxy_async();
            dev::named_barrier(2 + group, kGroupThreads);
            if (a.tma_out) {
              if (leader && unit_col < a.n) {
                dev::tma_store_2d(&maps.pre, pre_tile, static_cast<int>(unit_col),
                                  static_cast<int>(row0));
                dev::bulk_commit_group();
                dev::bulk_wait_group_read<0>();
              }
            } else {
              copy_unit<true, Out>(pre_tile, static_cast<Out*>(a.pre), row0, unit_col, a.m, a.n, quarter,
                             lane);
            }
            dev::named_barrier(2 + group, kGroupThreads);
          }
        }
        const auto apply = [&](int act) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if constexpr (kExact) {
              float lo, hi;
              unpack(v[i], &lo, &hi);
              v[i] = two(activate(lo, act), activate(hi, act));
            } else {
              v[i] = activate2(v[i], act);
            }
          }
        };
        if (a.act == CND_ACT_GELU) {
          apply(CND_ACT_GELU);
        } else if (a.act == CND_ACT_SILU) {
          apply(CND_ACT_SILU);
        }
        if (a.residual != nullptr) {
          if (h % kHalvesPerUnit == 0) {
            if (a.tma_residual) {
              if (a.buffers == 1 && a.pre != nullptr && leader) ask_residual(row0, unit_col, tile);
              ok = ok && dev::mbar_wait_warp(&residual_full[group], residual_phase, err,
                                             kSiteResidual, a.timeout_ns);
              residual_phase ^= 1u;
            } else {
              // rows that are not 16-byte aligned
              copy_unit<false, Out>(tile, const_cast<Out*>(static_cast<const Out*>(a.residual)), row0,
                                    unit_col, a.m, a.n, quarter, lane);
              dev::named_barrier(2 + group, kGroupThreads);
            }
          }
          Residual<Out> residual;
          residual.take(tile, row, h % kHalvesPerUnit);
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = add2(v[i], residual.pair(i));
        }
        stage_row<Out>(tile, row, h % kHalvesPerUnit, v);
        if (unit_done) {
          dev::fence_proxy_async();
          dev::named_barrier(2 + group, kGroupThreads);
          if (a.tma_residual && a.sets == 2) {
            // The next unit's residual: the next of this tile, or the first of the next tile.
            // Asked for behind the barrier, when every warp has seen this unit's arrive: a
            // warp that came to its wait two phases late would wait for the next one.
            int64_t next_row = row0, next_col = unit_col + kUnit;
            bool more = h + 1 < kHalves;
            if (!more && item + workers < items) {
              int next_m, next_n;
              tile_of(a, (item + workers) / a.splits, &next_m, &next_n);
              next_row = static_cast<int64_t>(next_m * kPair + static_cast<int>(rank)) * kBM;
              next_col = static_cast<int64_t>(next_n) * kBN + group * kGroupCols;
              more = true;
            }
            if (more && leader) {
              dev::bulk_wait_group_read<0>();  // the other tile's store, a unit ago
              ask_residual(next_row, next_col, own + buffer * kUnitBytes);
            }
            asked = more;
          }
          if (a.tma_out) {
            if (leader && unit_col < a.n) {
              // partial tiles of a split lie below one another
              const int y = static_cast<int>(row0) + split * a.tiles_m * kPair * kBM;
              if (row0 < a.m) {
                dev::tma_store_2d(&maps.out, tile, static_cast<int>(unit_col), y);
                if (a.pre != nullptr && a.buffers > 1) {
                  dev::tma_store_2d(&maps.pre, pre_tile, static_cast<int>(unit_col),
                                    static_cast<int>(row0));
                }
              }
            }
            if (leader) dev::bulk_commit_group();
          } else {
            copy_unit<true, Out>(tile, static_cast<Out*>(a.d), row0, unit_col, a.m, a.n, quarter, lane);
            if (a.pre != nullptr && a.buffers > 1) {
              copy_unit<true, Out>(pre_tile, static_cast<Out*>(a.pre), row0, unit_col, a.m, a.n, quarter,
                             lane);
            }
          }
        }
      }
      if constexpr (kParts == 1) {
        if (++set == 2) {
          set = 0;
          set_phase ^= 1u;
        }
      }
    }
    if (leader) dev::bulk_wait_group<0>();
  }
  dev::tc_fence_before();
  if constexpr (kPair == 2) {
    dev::cluster_sync();
  } else {
    __syncthreads();
  }
  if (warp == 0) {
    dev::tc_fence_after();
    __syncwarp();
    dev::tmem_dealloc_pair<kPair>(tmem, kColumns);
  }
}

// Adds the partial tiles of a split product and applies the epilogue. A thread takes four
// columns and one of kRanges contiguous ranges of the splits, in split order; the ranges are
// added in order. (148 splits of 256 x 64: 14 us in one range.)
template <typename Out, int kRanges>
__global__ void __launch_bounds__(256)
    join_kernel(const float* partials, int splits, int64_t split_stride, int64_t pitch, int64_t m,
                int64_t n, const void* bias, const void* residual, void* d, void* pre, int act) {
  constexpr int kQuads = 256 / kRanges;
  __shared__ float4 part[kRanges][kQuads];
  const int64_t quads = pitch / 4, count = m * quads;
  const int range = threadIdx.x / kQuads, at = threadIdx.x % kQuads;
  const int first = splits * range / kRanges, last = splits * (range + 1) / kRanges;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kQuads; base < count;
       base += static_cast<int64_t>(gridDim.x) * kQuads) {
    const int64_t i = base + at;
    const int64_t row = i / quads, col = i % quads * 4;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (i < count) {
      const float* p = partials + row * pitch + col;
#pragma unroll 4
      for (int s = first; s < last; ++s) {
        const float4 v = *reinterpret_cast<const float4*>(p + s * split_stride);
        sum.x += v.x;
        sum.y += v.y;
        sum.z += v.z;
        sum.w += v.w;
      }
    }
    if constexpr (kRanges > 1) {
      part[range][at] = sum;
      __syncthreads();
      if (range == 0) {
#pragma unroll
        for (int r = 1; r < kRanges; ++r) {
          const float4 v = part[r][at];
          sum.x += v.x;
          sum.y += v.y;
          sum.z += v.z;
          sum.w += v.w;
        }
      }
      __syncthreads();
      if (range != 0) continue;
    }
    if (i >= count) continue;
    const float v4[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = col + j;
      if (c >= n) break;
      float v = v4[j];
      if (bias != nullptr) v += widen(static_cast<const Out*>(bias)[c]);
      if (pre != nullptr) static_cast<Out*>(pre)[row * n + c] = narrow<Out>(v);
      v = activate(v, act);
      if (residual != nullptr) v += widen(static_cast<const Out*>(residual)[row * n + c]);
      static_cast<Out*>(d)[row * n + c] = narrow<Out>(v);
    }
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult status;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &status) !=
            cudaSuccess ||
        status != cudaDriverEntryPointSuccess) {
      fn = nullptr;
    }
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  }();
  return encode;
}

bool encode_operand(CUtensorMap* map, const Operand& o, int64_t rows, int64_t k, int parts,
                    bool bf16, int box_rows) {
  const int depth = block_depth(parts);
  const cuuint64_t inner = static_cast<cuuint64_t>(o.k_major ? k : rows);
  const cuuint64_t outer = static_cast<cuuint64_t>(o.k_major ? rows : k);
  const cuuint64_t dims[3] = {inner, outer, static_cast<cuuint64_t>(parts)};
  const int64_t plane = parts > 1 ? o.plane : o.pitch * static_cast<int64_t>(outer);
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(o.pitch) * 2,
                                 static_cast<cuuint64_t>(plane) * 2};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(o.k_major ? depth : 64),
                             static_cast<cuuint32_t>(o.k_major ? box_rows : depth), 1};
  const cuuint32_t ones[3] = {1, 1, 1};
  return encoder()(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                   3, const_cast<void*>(o.data), dims, strides, box, ones,
                   CU_TENSOR_MAP_INTERLEAVE_NONE,
                   box[0] == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

using Kernel = void (*)(Maps, KernelArgs);

template <typename Out>
Kernel pick(const ProductPlan& plan, int parts) {
  if constexpr (sizeof(Out) == 4) {
    if (parts == 3) {
      return plan.pair == 2   ? product_tc_kernel<2, 128, 3, 2, Out>
             : plan.bn == 128 ? product_tc_kernel<1, 128, 3, 2, Out>
                              : product_tc_kernel<1, 64, 3, 1, Out>;
    }
  }
  if (plan.pair == 2) {
    return plan.groups == 4 ? product_tc_kernel<2, 256, 1, 4, Out>
                            : product_tc_kernel<2, 256, 1, 2, Out>;
  }
  return plan.bn == 128 ? product_tc_kernel<1, 128, 1, 2, Out>
                        : product_tc_kernel<1, 64, 1, 1, Out>;
}

int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

}  // namespace

bool encode_matrix(CUtensorMap* map, void* d, int dtype, int64_t rows, int64_t n, int64_t pitch,
                   int box_rows) {
  const int size = element_size(dtype);
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(n), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch) * size};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / size),
                             static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t ones[2] = {1, 1};
  const CUtensorMapDataType type = dtype == CND_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : dtype == CND_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                       : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (encoder() == nullptr) return false;
  return encoder()(map, type, 2, d, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

ProductPlan plan_product(int64_t m, int64_t n, int64_t k, int parts) {
  // Microseconds, fitted to runs over 16 to 4096 rows and 1024 or 4096 of n and k: a launch,
  // a block of k, and the epilogue of a tile (which runs under the next tile's main loop);
  // joining splits costs a launch and its traffic. The fit is within a few percent where two
  // cuts are close; the wrong one of a pair far apart costs half again (4096^3: 99 us on
  // pairs, 132 on single CTAs; 16 x 4096 -> 1024: 10.1 in 8 splits, 20 in one).
  struct Cut {
    int parts, pair, bn;
    double launch, block, tail;
  };
  static constexpr Cut kCuts[] = {
      {1, 2, 256, 8.5, 0.32, 5.5}, {1, 1, 128, 5.0, 0.27, 3.0}, {1, 1, 64, 4.3, 0.25, 1.9},
      {3, 2, 128, 8.0, 0.52, 4.0}, {3, 1, 128, 5.0, 0.62, 3.0}, {3, 1, 64, 4.3, 0.47, 2.0},
  };
  const int64_t sms = kSms, blocks = (k + block_depth(parts) - 1) / block_depth(parts);
  ProductPlan best{1, 64, 1, 1};
  double best_cost = 0;
  for (const Cut& c : kCuts) {
    if (c.parts != parts) continue;
    const int64_t rows = kBM * c.pair;
    const int64_t tiles = ((m + rows - 1) / rows) * ((n + c.bn - 1) / c.bn);
    const int64_t slots = sms / c.pair;
    for (int64_t splits = 1; splits <= 64; ++splits) {
      if (splits > 1 && (blocks / splits < 2 || tiles * splits > 2 * slots)) break;
      const int64_t waves = (tiles * splits + slots - 1) / slots;
      const double main = static_cast<double>((blocks + splits - 1) / splits) * c.block;
      double cost = c.launch + (waves - 1) * std::max(main, c.tail) + main;
      if (splits > 1) {
        cost += 2.2 + 0.3e-6 * static_cast<double>(splits) * ((m + rows - 1) / rows * rows) * n * 4;
      }
      if (best_cost == 0 || cost < best_cost) {
        best_cost = cost;
        // Four epilogue groups (four warps a scheduler) where the epilogue is the longer part:
        // with two, waits for TMEM, exponentials and staging left a scheduler issuing 27 % of
        // the time (1M x 64 -> 256 GELU: 369 us against 263). From a depth of 1024 on two
        // groups and more operand stages win (16384 x 1024 -> 4096 GELU: 123 us against 125,
        // without an activation 103 against 116).
        const int groups = c.bn == 64 ? 1 : c.bn == 256 && blocks / splits <= 8 ? 4 : 2;
        best = ProductPlan{c.pair, c.bn, static_cast<int>(splits), groups};
      }
    }
  }
  return best;
}

size_t product_workspace(const ProductPlan& plan, int64_t m, int64_t n) {
  if (plan.splits <= 1) return 0;
  return static_cast<size_t>(plan.splits) * round_up(m, kBM * plan.pair) * round_up(n, 4) *
         sizeof(float);
}

void join_partials(const Product& p, const float* partials, int splits, int64_t stride,
                   int64_t pitch, cudaStream_t stream) {
  const int64_t quads = p.m * (pitch / 4);
  const bool many = splits >= 16;
  const int per_block = many ? 32 : 256;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(
      (quads + per_block - 1) / per_block, static_cast<int64_t>(sm_count()) * 8));
  const auto join = [&](auto* kernel_join) {
    kernel_join<<<grid, 256, 0, stream>>>(partials, splits, stride, pitch, p.m, p.n, p.bias,
                                          p.residual, p.d, p.pre, p.act);
  };
  if (p.dtype == CND_F32) {
    many ? join(join_kernel<float, 8>) : join(join_kernel<float, 1>);
  } else if (p.dtype == CND_BF16) {
    many ? join(join_kernel<__nv_bfloat16, 8>) : join(join_kernel<__nv_bfloat16, 1>);
  } else {
    many ? join(join_kernel<__half, 8>) : join(join_kernel<__half, 1>);
  }
  count_launch();
}

int launch_product(const Product& p, const ProductPlan& plan, void* workspace,
                   cudaStream_t stream) {
  if (encoder() == nullptr) return fail(CND_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const int bm = kBM * plan.pair;
  const bool split = plan.splits > 1;
  const int depth = block_depth(p.parts);
  if (round_up(p.m, bm) * plan.splits > INT32_MAX || p.n > INT32_MAX - 256 ||
      p.k > INT32_MAX - 64) {
    return fail(CND_ERR_UNSUPPORTED, "linear: a matrix dimension exceeds 2^31");
  }
  KernelArgs a{};
  a.m = p.m;
  a.n = p.n;
  a.tiles_m = static_cast<int>((p.m + bm - 1) / bm);
  a.tiles_n = static_cast<int>((p.n + plan.bn - 1) / plan.bn);
  a.splits = plan.splits;
  a.k_blocks = static_cast<int>((p.k + depth - 1) / depth);
  if (static_cast<int64_t>(a.tiles_m) * a.tiles_n * a.splits > INT32_MAX) {
    return fail(CND_ERR_UNSUPPORTED, "linear: too many tiles");
  }
  const int out_dtype = split ? static_cast<int>(CND_F32) : p.dtype;
  // A second unit of staging hides the stores' latency behind the next unit; a unit with a
  // pre-activation takes two tiles. Two groups on a pair have main loops long enough to
  // hide it: there the room goes to a sixth operand stage.
  const bool wants_pre = !split && p.pre != nullptr;
  if (p.parts == 3) {
    a.buffers = 1;
  } else if (plan.pair == 2) {
    a.buffers = plan.groups == 4 || wants_pre || (!split && p.residual != nullptr) ? 2 : 1;
  } else {
    a.buffers = wants_pre ? 4 : 2;
  }
  a.sets = wants_pre ? std::max(1, a.buffers / 2) : a.buffers;
  const uint32_t stage = p.parts * (kBM + plan.bn / plan.pair) * depth * 2;
  const uint32_t fixed = 1024 + plan.groups * a.buffers * kUnitBytes + plan.bn * sizeof(float) + 256;
  a.stages = static_cast<int>(std::min<uint32_t>((kSharedLimit - fixed) / stage, kMostStages));
  const uint32_t shared = fixed + a.stages * stage;
  a.idesc = (1u << 4) | ((p.bf16 ? 1u : 0u) << 7) | ((p.bf16 ? 1u : 0u) << 10) |
            (p.a.k_major ? 0u : 1u << 15) | (p.b.k_major ? 0u : 1u << 16) |
            (static_cast<uint32_t>(plan.bn) >> 3 << 17) | (static_cast<uint32_t>(bm) >> 4 << 24);
  a.a_k_major = p.a.k_major;
  a.b_k_major = p.b.k_major;
  a.a_step = (p.a.k_major ? 32 : 16 * 128) >> 4;
  a.b_step = (p.b.k_major ? 32 : 16 * 128) >> 4;
  a.a_lbo = p.a.k_major ? 16 : depth * 128;
  a.b_lbo = p.b.k_major ? 16 : depth * 128;
  // eight rows of a swizzle atom: 128 bytes wide, or 64 (K-major blocks 32 deep)
  const uint32_t narrow_rows = depth == 32;
  a.a_sbo = p.a.k_major && narrow_rows ? 512 : 1024;
  a.b_sbo = p.b.k_major && narrow_rows ? 512 : 1024;
  a.a_swizzle = p.a.k_major && narrow_rows ? 4 : 2;
  a.b_swizzle = p.b.k_major && narrow_rows ? 4 : 2;
  a.error = device_error_word();
  a.timeout_ns = wait_timeout_ns();
  if (a.error == nullptr) return fail(CND_ERR_CUDA, "device error word unavailable");
  const Kernel kernel = out_dtype == CND_F32    ? pick<float>(plan, p.parts)
                        : out_dtype == CND_BF16 ? pick<__nv_bfloat16>(plan, p.parts)
                                                : pick<__half>(plan, p.parts);
  // (a runtime call before the tensor maps: encoding needs the thread to have a context)
  cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(kSharedLimit));
  if (e != cudaSuccess) return fail(CND_ERR_CUDA, "linear: %s", cudaGetErrorString(e));
  Maps maps{};
  if (!encode_operand(&maps.a, p.a, p.m, p.k, p.parts, p.bf16, kBM) ||
      !encode_operand(&maps.b, p.b, p.n, p.k, p.parts, p.bf16, plan.bn / plan.pair)) {
    return fail(CND_ERR_CUDA, "linear: encoding an operand's tensor map failed");
  }
  const int64_t pitch = round_up(p.n, 4);
  if (split) {
    // partial tiles below one another, each split's rows rounded up to whole tiles
    a.tma_out = 1;
    if (!encode_matrix(&maps.out, workspace, CND_F32, round_up(p.m, bm) * plan.splits, pitch,
                       pitch, kBM)) {
      return fail(CND_ERR_CUDA, "linear: encoding the partial sums' tensor map failed");
    }
  } else {
    const int size = element_size(p.dtype);
    a.bias = p.bias;
    a.residual = p.residual;
    a.d = p.d;
    a.pre = p.pre;
    a.act = p.act;
    a.tma_residual = p.residual != nullptr && aligned16(p.residual) && p.n * size % 16 == 0;
    a.tma_out = p.n * size % 16 == 0 && aligned16(p.d) && aligned16(p.pre);
    if (a.tma_out &&
        (!encode_matrix(&maps.out, p.d, p.dtype, p.m, p.n, p.n, kBM) ||
         (p.pre != nullptr && !encode_matrix(&maps.pre, p.pre, p.dtype, p.m, p.n, p.n, kBM)))) {
      return fail(CND_ERR_CUDA, "linear: encoding an output's tensor map failed");
    }
    if (a.tma_residual && !encode_matrix(&maps.residual, const_cast<void*>(p.residual), p.dtype, p.m,
                                         p.n, p.n, kBM)) {
      return fail(CND_ERR_CUDA, "linear: encoding an output's tensor map failed");
    }
  }
  const int items = a.tiles_m * a.tiles_n * a.splits;
  const int slots = sm_count() / plan.pair;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(std::min(items, slots) * plan.pair));
  config.blockDim = dim3(block_threads(plan.groups));
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  cudaLaunchAttribute attribute{};
  if (plan.pair == 2) {
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = 2;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
  }
  e = cudaLaunchKernelEx(&config, kernel, maps, a);
  if (e != cudaSuccess) return fail(CND_ERR_CUDA, "linear: %s", cudaGetErrorString(e));
  count_launch();
  if (split) {
    join_partials(p, static_cast<const float*>(workspace), plan.splits, round_up(p.m, bm) * pitch,
                  pitch, stream);
  }
  return launch_status("linear");
}

}  // namespace layers
}  // namespace cnd
