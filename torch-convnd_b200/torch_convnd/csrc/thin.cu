// Backward of a 16-bit linear layer with an activation and few features, in one pass:
//
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  dbias = column sums of dz.
//
// With up to 64 input and 256 output features, W and dW fit an SM, and the layer is bound by
// reading dy and z. Separate launches write dz and read it twice, 2.5 times the traffic of one
// pass that turns each tile of dy into dz where it lies in shared memory and feeds both products
// from there (1M x 64 -> 256 in bf16: 272 us, 4.9 TB/s of what has to be moved, and 8 us to join;
// 510 us in separate launches).
//
// A persistent block takes tiles of 128 rows. One lane loads 64-column chunks of dy and z by
// TMA into four slots and the tile's x into one of two; two teams of eight warps take
// alternate chunks, multiply dy by the slope in place and keep column sums; one warp issues
// the MMAs of a finished chunk:
//   dx [128 rows][64]  += dz chunk [128][64 n] * W chunk [64 n][64]   (K-major, MN-major)
//   dW^T [64][64 n]    += x^T [64][128 rows] * dz chunk [128 rows][64 n]  (both MN-major).
// dW^T stays in TMEM over all the block's tiles; an M = 128 product is issued, whose upper
// half reads the tile that follows x in shared memory and is dropped. Four warps
// write dx out. The blocks' dW and column sums are joined in block order: repeated calls give
// the same bits. dz is rounded to the operands' type for the products, as where it is stored;
// its column sums are not.
#include <cuda.h>

#include <algorithm>

#include "activation.cuh"
#include "layers.cuh"
#include "pair.cuh"
#include "product.cuh"

namespace cnd {
namespace layers {
namespace {

constexpr int kRows = 128, kChunk = 64;
constexpr int kMostChunks = kThinOut / kChunk;
constexpr int kSlots = 4, kTeams = 2, kTeamWarps = 8, kTeamThreads = kTeamWarps * 32;
constexpr int kFirstWorker = 6;  // after the TMA and MMA warps and the four that write dx
constexpr int kThreads = kFirstWorker * 32 + kTeams * kTeamThreads;
constexpr uint32_t kTileBytes = kRows * kChunk * 2;  // of dy, z, x and dx
constexpr uint32_t kWeightBytes = kChunk * kChunk * 2;
constexpr uint32_t kDxColumn = kThinOut;  // TMEM: dW^T, then two dx tiles
constexpr uint32_t kTmemColumns = 512;
constexpr uint32_t kSiteLoad = 0x511, kSiteMma = 0x512, kSiteSlope = 0x513, kSiteOut = 0x514,
                   kSiteDrain = 0x515;

struct ThinMaps {
  CUtensorMap dy, z, x, w, dx;
};

struct ThinArgs {
  int tiles, chunks, act;
  int n, k;
  uint32_t idesc_dx, idesc_dw;
  float* dw;  // [gridDim.x][n][k]
  float* db;  // [gridDim.x][n] or NULL
  unsigned int* error;
  uint64_t timeout_ns;
};

constexpr uint32_t kShared = 1024 + kSlots * 2 * kTileBytes + 2 * kTileBytes +
                             kMostChunks * kWeightBytes + kTileBytes +
                             kTeams * kTeamWarps * 2 * kChunk * 4 + 256;

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    thin_backward_kernel(const __grid_constant__ ThinMaps maps, const __grid_constant__ ThinArgs a) {
  extern __shared__ __align__(1024) uint8_t shared[];
  uint8_t* slots = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(shared) + 1023) & ~uintptr_t{1023});
  uint8_t* x_s = slots + kSlots * 2 * kTileBytes;
  uint8_t* w_s = x_s + 2 * kTileBytes;
  uint8_t* out_s = w_s + kMostChunks * kWeightBytes;
  float* sums_s = reinterpret_cast<float*>(out_s + kTileBytes);  // [team][warp][2][kChunk]
  uint64_t* full = reinterpret_cast<uint64_t*>(sums_s + kTeams * kTeamWarps * 2 * kChunk);
  uint64_t* ready = full + kSlots;  // the slot's dy is dz
  uint64_t* empty = ready + kSlots;
  uint64_t* x_full = empty + kSlots;
  uint64_t* x_empty = x_full + 2;
  uint64_t* dx_full = x_empty + 2;
  uint64_t* dx_empty = dx_full + 2;
  uint64_t* w_full = dx_empty + 2;
  uint64_t* done = w_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const dev::ErrorWord err{a.error};
  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) {
      dev::mbar_init(&full[s], 1);
      dev::mbar_init(&ready[s], kTeamWarps);
      dev::mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      dev::mbar_init(&x_full[b], 1);
      dev::mbar_init(&x_empty[b], 1);
      dev::mbar_init(&dx_full[b], 1);
      dev::mbar_init(&dx_empty[b], 4);
    }
    dev::mbar_init(w_full, 1);
    dev::mbar_init(done, 1);
    dev::fence_barrier_init();
  }
  if (warp == 0) {
    __syncwarp();
    dev::tmem_alloc(tmem_slot, kTmemColumns);
  }
  dev::tc_fence_before();
  __syncthreads();
  dev::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int first = static_cast<int>(blockIdx.x), step = static_cast<int>(gridDim.x);

  if (warp == 0) {
    if (lane == 0) {
      dev::mbar_arrive_expect_tx(w_full, a.chunks * kWeightBytes);
      for (int c = 0; c < a.chunks; ++c) {
        dev::tma_load_2d(w_s + c * kWeightBytes, &maps.w, w_full, 0, c * kChunk);
      }
      int slot = 0, buffer = 0;
      uint32_t phase = 0, x_phase = 0;
      uint32_t loaded = 0, x_loaded = 0;
      bool ok = true;
      for (int tile = first; tile < a.tiles && ok; tile += step) {
        const int row0 = tile * kRows;
        ok = dev::mbar_wait(&x_empty[buffer], x_phase ^ 1u, err, kSiteLoad, a.timeout_ns);
        if (!ok) break;
        dev::mbar_arrive_expect_tx(&x_full[buffer], kTileBytes);
        dev::tma_load_2d(x_s + buffer * kTileBytes, &maps.x, &x_full[buffer], 0, row0);
        ++x_loaded;
        if (++buffer == 2) {
          buffer = 0;
          x_phase ^= 1u;
        }
        for (int c = 0; c < a.chunks; ++c) {
          ok = dev::mbar_wait(&empty[slot], phase ^ 1u, err, kSiteLoad, a.timeout_ns);
          if (!ok) break;
          uint8_t* at = slots + slot * 2 * kTileBytes;
          dev::mbar_arrive_expect_tx(&full[slot], 2 * kTileBytes);
          dev::tma_load_2d(at, &maps.dy, &full[slot], c * kChunk, row0);
          dev::tma_load_2d(at + kTileBytes, &maps.z, &full[slot], c * kChunk, row0);
          ++loaded;
          if (++slot == kSlots) {
            slot = 0;
            phase ^= 1u;
          }
        }
      }
      // the last loads of each slot, of x and of W land before the block may exit, or have had a
      // bounded time to
      const uint64_t limit = a.timeout_ns / 8 + 1;
      dev::mbar_wait(w_full, 0, err, kSiteDrain, limit);
      for (int s = 0; s < kSlots; ++s) {
        if (loaded > static_cast<uint32_t>(s)) {
          dev::mbar_wait(&full[s], s < slot ? phase : phase ^ 1u, err, kSiteDrain, limit);
        }
      }
      for (int b = 0; b < 2; ++b) {
        if (x_loaded > static_cast<uint32_t>(b)) {
          dev::mbar_wait(&x_full[b], b < buffer ? x_phase : x_phase ^ 1u, err, kSiteDrain, limit);
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    const uint32_t base = dev::warp_uniform(tmem);
    // dz as A of dx (K-major, 32 bytes per 16 of k) and as B of dW (16 rows of 128 bytes)
    const uint64_t k_major = dev::make_smem_desc(0, 16, 1024, 2);
    const uint64_t mn_major = dev::make_smem_desc(0, kTileBytes, 1024, 2);
    const uint32_t slots_at = dev::warp_uniform(dev::smem_u32(slots) >> 4);
    const uint32_t x_at = dev::warp_uniform(dev::smem_u32(x_s) >> 4);
    const uint32_t w_at = dev::warp_uniform(dev::smem_u32(w_s) >> 4);
    int slot = 0, buffer = 0;
    uint32_t phase = 0, x_phase = 0;
    bool ok = dev::mbar_wait_warp(w_full, 0, err, kSiteMma, a.timeout_ns);
    for (int tile = first; tile < a.tiles && ok; tile += step) {
      ok = dev::mbar_wait_warp(&x_full[buffer], x_phase, err, kSiteMma, a.timeout_ns) &&
           dev::mbar_wait_warp(&dx_empty[buffer], x_phase ^ 1u, err, kSiteMma, a.timeout_ns);
      if (!ok) break;
      const uint32_t x_tile = x_at + buffer * (kTileBytes >> 4);
      const uint32_t d_dx = base + kDxColumn + buffer * kChunk;
      for (int c = 0; c < a.chunks; ++c) {
        ok = dev::mbar_wait_warp(&ready[slot], phase, err, kSiteMma, a.timeout_ns);
        if (!ok) break;
        dev::tc_fence_after();
        const uint32_t dz = slots_at + slot * (2 * kTileBytes >> 4);
        const uint32_t w = w_at + c * (kWeightBytes >> 4);
#pragma unroll
        for (int ks = 0; ks < kChunk / 16; ++ks) {
          dev::mma_f16_warp(d_dx, k_major | (dz + ks * 2), mn_major | (w + ks * 128), a.idesc_dx,
                            c > 0 || ks > 0);
        }
#pragma unroll
        for (int ks = 0; ks < kRows / 16; ++ks) {
          dev::mma_f16_warp(base + c * kChunk, mn_major | (x_tile + ks * 128),
                            mn_major | (dz + ks * 128), a.idesc_dw, tile != first || ks > 0);
        }
        dev::mma_commit_warp(&empty[slot]);
        if (++slot == kSlots) {
          slot = 0;
          phase ^= 1u;
        }
      }
      if (!ok) break;
      dev::mma_commit_warp(&x_empty[buffer]);
      dev::mma_commit_warp(&dx_full[buffer]);
      if (++buffer == 2) {
        buffer = 0;
        x_phase ^= 1u;
      }
    }
    dev::mma_commit_warp(done);
  } else if (warp < kFirstWorker) {
    // ---- dx out, then the block's dW ----
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const bool leader = threadIdx.x == 64;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    int buffer = 0;
    uint32_t phase = 0;
    bool ok = true;  // once false, on without waiting: the barriers below take all four warps
    for (int tile = first; tile < a.tiles; tile += step) {
      ok = ok && dev::mbar_wait_warp(&dx_full[buffer], phase, err, kSiteOut, a.timeout_ns);
      dev::tc_fence_after();
      uint32_t v[2][32];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        dev::tmem_load32(tmem + lanes + kDxColumn + buffer * kChunk + h * 32, v[h]);
      }
      dev::tmem_load_wait();
      dev::tc_fence_before();
      __syncwarp();
      if (lane == 0) dev::mbar_arrive(&dx_empty[buffer]);
      if (++buffer == 2) {
        buffer = 0;
        phase ^= 1u;
      }
      if (leader) dev::bulk_wait_group_read<0>();
      dev::named_barrier(1, 128);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        Two w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = two(__uint_as_float(v[c / 4][c % 4 * 8 + 2 * i]),
                     __uint_as_float(v[c / 4][c % 4 * 8 + 2 * i + 1]));
        }
        store_twos<T, 8>(out_s + row * 128 + ((c ^ (row & 7)) * 16), w);
      }
      dev::fence_proxy_async();
      dev::named_barrier(1, 128);
      if (leader) {
        dev::tma_store_2d(&maps.dx, out_s, 0, tile * kRows);
        dev::bulk_commit_group();
      }
    }
    ok = dev::mbar_wait_warp(done, 0, err, kSiteOut, ok ? a.timeout_ns : a.timeout_ns / 8 + 1) && ok;
    if (ok) {
      dev::tc_fence_after();
      float* dw = a.dw + static_cast<int64_t>(blockIdx.x) * a.n * a.k;
      for (int c0 = 0; c0 < a.n; c0 += 32) {
        uint32_t v[32];
        dev::tmem_load32(tmem + lanes + c0, v);
        dev::tmem_load_wait();
        if (row < a.k) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (c0 + i < a.n) dw[(c0 + i) * a.k + row] = __uint_as_float(v[i]);
          }
        }
      }
    }
    if (leader) dev::bulk_wait_group<0>();
  } else {
    // ---- dy to dz, in place; a thread keeps to eight columns of its team's chunks ----
    const int team = (warp - kFirstWorker) / kTeamWarps;
    const int tid = (threadIdx.x - kFirstWorker * 32) % kTeamThreads;
    const int piece = tid & 7, row0 = tid >> 3;
    uint8_t* mine = slots + row0 * 128 + ((piece ^ (row0 & 7)) * 16);
    Two sums[2][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[i / 4][i % 4] = same(0.0f);
    const auto slope_chunk = [&](uint8_t* at, Two (&sum)[4], int act) {
#pragma unroll
      for (int j = 0; j < kRows / 32; ++j) {
        Two w[4], z[4];
        load_twos<T, 8>(at + j * 32 * 128, w);
        load_twos<T, 8>(at + j * 32 * 128 + kTileBytes, z);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = mul2(w[i], slope2(z[i], act));
          sum[i] = add2(sum[i], w[i]);
        }
        store_twos<T, 8>(at + j * 32 * 128, w);
      }
    };
    bool ok = true;
    uint32_t chunk0 = 0;  // chunks before this tile
    for (int tile = first; tile < a.tiles && ok; tile += step, chunk0 += a.chunks) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = 2 * i + team;
        if (c < a.chunks && ok) {
          const uint32_t index = chunk0 + c, slot = index % kSlots;
          ok = dev::mbar_wait_warp(&full[slot], index / kSlots & 1u, err, kSiteSlope, a.timeout_ns);
          if (ok) {
            uint8_t* at = mine + slot * 2 * kTileBytes;
            if (a.act == CND_ACT_GELU) {
              slope_chunk(at, sums[i], CND_ACT_GELU);
            } else {
              slope_chunk(at, sums[i], CND_ACT_SILU);
            }
            dev::fence_proxy_async();
            __syncwarp();
            if (lane == 0) dev::mbar_arrive(&ready[slot]);
          }
        }
      }
    }
    // the four rows of a warp, then (below) the warps of a team
    float* out = sums_s + ((team * kTeamWarps + tid / 32) * 2) * kChunk;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float s[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) unpack(sums[i][j], &s[2 * j], &s[2 * j + 1]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[j] += __shfl_xor_sync(0xffffffffu, s[j], 8);
        s[j] += __shfl_xor_sync(0xffffffffu, s[j], 16);
        if (lane < 8) out[i * kChunk + piece * 8 + j] = s[j];
      }
    }
  }
  dev::tc_fence_before();
  __syncthreads();
  if (a.db != nullptr && static_cast<int>(threadIdx.x) < a.n) {
    const int c = threadIdx.x / kChunk;
    const float* in = sums_s + c % 2 * kTeamWarps * 2 * kChunk + c / 2 * kChunk + threadIdx.x % kChunk;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kTeamWarps; ++w) sum += in[w * 2 * kChunk];
    a.db[static_cast<int64_t>(blockIdx.x) * a.n + threadIdx.x] = sum;
  }
  if (warp == 0) {
    dev::tc_fence_after();
    __syncwarp();
    dev::tmem_dealloc(tmem, kTmemColumns);
  }
}

}  // namespace

int thin_blocks(int64_t rows) {
  return static_cast<int>(std::min<int64_t>((rows + kRows - 1) / kRows, kSms));
}

int launch_thin_backward(const ThinBackward& p, cudaStream_t stream) {
  ThinArgs a{};
  a.tiles = static_cast<int>((p.rows + kRows - 1) / kRows);
  a.n = static_cast<int>(p.n);
  a.k = static_cast<int>(p.k);
  a.chunks = (a.n + kChunk - 1) / kChunk;
  a.act = p.act;
  const uint32_t type = p.dtype == CND_BF16 ? 1u : 0u;
  const uint32_t idesc = (1u << 4) | (type << 7) | (type << 10) | (1u << 16) |
                         (static_cast<uint32_t>(kChunk) >> 3 << 17) |
                         (static_cast<uint32_t>(kRows) >> 4 << 24);
  a.idesc_dx = idesc;               // dz K-major, W MN-major
  a.idesc_dw = idesc | (1u << 15);  // both MN-major
  a.dw = p.dw;
  a.db = p.db;
  a.error = device_error_word();
  a.timeout_ns = wait_timeout_ns();
  if (a.error == nullptr) return fail(CND_ERR_CUDA, "device error word unavailable");
  // (a runtime call first: encoding needs the thread to have a context)
  const auto kernel = p.dtype == CND_BF16 ? thin_backward_kernel<__nv_bfloat16>
                                          : thin_backward_kernel<__half>;
  cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(kShared));
  if (e != cudaSuccess) return fail(CND_ERR_CUDA, "linear: %s", cudaGetErrorString(e));
  ThinMaps maps{};
  if (!encode_matrix(&maps.dy, const_cast<void*>(p.dy), p.dtype, p.rows, p.n, p.n, kRows) ||
      !encode_matrix(&maps.z, const_cast<void*>(p.z), p.dtype, p.rows, p.n, p.n, kRows) ||
      !encode_matrix(&maps.x, const_cast<void*>(p.x), p.dtype, p.rows, p.k, p.x_stride, kRows) ||
      !encode_matrix(&maps.w, const_cast<void*>(p.w), p.dtype, p.n, p.k, p.k, kChunk) ||
      !encode_matrix(&maps.dx, p.dx, p.dtype, p.rows, p.k, p.k, kRows)) {
    return fail(CND_ERR_CUDA, "linear: encoding a tensor map failed");
  }
  kernel<<<thin_blocks(p.rows), kThreads, kShared, stream>>>(maps, a);
  count_launch();
  return launch_status("linear");
}

}  // namespace layers
}  // namespace cnd
