// Layer norm over rows: forward, and the backward pass with the weight's and bias's
// gradients.
//
//   mean = sum(x) / C,  rstd = 1 / sqrt(sum((x - mean)^2) / C + eps),  u = (x - mean) rstd,
//   y = u w + b;
//   g = dy w,  dx = rstd (g - mean(g) - u mean(g u)),  dw = sum(dy u),  db = sum(dy).
//
// A row is held in registers between its two sums (the squares are of centred values, so a
// large mean costs no digits), so every element is read once: both passes are bound by
// memory traffic, 2 and 3 elements per position. A row belongs to G lanes of a warp or to a
// block of G threads; a block walks rows with a grid stride, each thread always holding the
// same columns, so the weight's gradient accumulates in registers, is combined once per
// block and leaves as one partial row per block, summed in order by a second launch. Rows
// wider than the register kernels take are walked in chunks and read again for each pass.
#include <algorithm>
#include <cstring>

#include "layers.cuh"

namespace cnd {
namespace layers {

int sm_count() {
  int device = 0, count = 0;
  if (cudaGetDevice(&device) != cudaSuccess ||
      cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device) != cudaSuccess ||
      count <= 0) {
    cudaGetLastError();
    return 148;
  }
  return count;
}

namespace {

struct NormArgs {
  const void* x;
  const void* dy;
  const void* weight;
  const void* bias;
  void* y;  // forward: y, backward: dx
  void* stats;
  void* partials;  // backward: [blocks][2][width]
  int64_t rows, width, x_stride, dy_stride;
  double eps;
  int param_f32;
  int want_dx, want_params;
};

// Sum over the G threads of a row's group; every thread gets it. G <= 32: lanes of one
// warp; else the whole block, with `scratch` holding one value per warp. The order is fixed.
template <int G, typename A>
__device__ __forceinline__ A group_sum(A v, A* scratch) {
#pragma unroll
  for (int d = (G < 32 ? G : 32) / 2; d > 0; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
  if constexpr (G > 32) {
    constexpr int kWarps = G / 32;
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[threadIdx.x & (kWarps - 1)];
#pragma unroll
    for (int d = kWarps / 2; d > 0; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
    __syncthreads();
  }
  return v;
}

// Block size of the register kernels: 256 threads, or the G of one row when it needs more.
template <int G>
constexpr int block_size() {
  return G > 256 ? G : (G > 32 ? G : 256);
}

template <typename T, int V, int NV, int G>
__global__ void __launch_bounds__(block_size<G>())
    norm_forward_kernel(const NormArgs a) {
  constexpr int kRows = block_size<G>() / G;
  __shared__ float scratch[32];
  const int lane = threadIdx.x % G;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  const float inverse = 1.0f / static_cast<float>(a.width);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows; base < a.rows; base += step) {
    const int64_t row = base + threadIdx.x / G;
    const bool live = row < a.rows;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    Pack<T, V> raw[NV];
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = static_cast<int64_t>(k * G + lane) * V;
      if (live && c < a.width) {
        raw[k] = *reinterpret_cast<const Pack<T, V>*>(x + c);
#pragma unroll
        for (int i = 0; i < V; ++i) sum += widen(raw[k].v[i]);
      }
    }
    const float mean = group_sum<G>(sum, scratch) * inverse;
    float squares = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = static_cast<int64_t>(k * G + lane) * V;
      if (live && c < a.width) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = widen(raw[k].v[i]) - mean;
          squares += d * d;
        }
      }
    }
    const float variance = group_sum<G>(squares, scratch) * inverse;
    const float rstd = rsqrtf(variance + static_cast<float>(a.eps));
    if (!live) continue;
    if (a.stats != nullptr && lane == 0) {
      static_cast<float*>(a.stats)[row] = mean;
      static_cast<float*>(a.stats)[a.rows + row] = rstd;
    }
    T* y = static_cast<T*>(a.y) + row * a.width;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = static_cast<int64_t>(k * G + lane) * V;
      if (c < a.width) {
        Pack<T, V> out;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float v = (widen(raw[k].v[i]) - mean) * rstd;
          if (a.weight != nullptr) v *= load_param<T>(a.weight, a.param_f32, c + i);
          if (a.bias != nullptr) v += load_param<T>(a.bias, a.param_f32, c + i);
          out.v[i] = narrow<T>(v);
        }
        *reinterpret_cast<Pack<T, V>*>(y + c) = out;
      }
    }
  }
}

template <typename T, int V, int NV, int G>
__global__ void __launch_bounds__(block_size<G>())
    norm_backward_kernel(const NormArgs a) {
  constexpr int kThreads = block_size<G>();
  constexpr int kRows = kThreads / G;
  extern __shared__ float columns[];  // [2][width], only when kRows > 1
  __shared__ float scratch[32];
  const int lane = threadIdx.x % G;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  const float inverse = 1.0f / static_cast<float>(a.width);
  const float* means = static_cast<const float*>(a.stats);
  float dw[NV][V], db[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
#pragma unroll
    for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = 0.0f;
  }
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows; base < a.rows; base += step) {
    const int64_t row = base + threadIdx.x / G;
    const bool live = row < a.rows;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
    const float mean = live ? means[row] : 0.0f;
    const float rstd = live ? means[a.rows + row] : 0.0f;
    Pack<T, V> rx[NV], rd[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = static_cast<int64_t>(k * G + lane) * V;
      if (live && c < a.width) {
        rx[k] = *reinterpret_cast<const Pack<T, V>*>(x + c);
        rd[k] = *reinterpret_cast<const Pack<T, V>*>(dy + c);
      }
    }
    float sum_g = 0.0f, sum_gu = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = static_cast<int64_t>(k * G + lane) * V;
      if (live && c < a.width) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = widen(rd[k].v[i]);
          const float u = (widen(rx[k].v[i]) - mean) * rstd;
          const float g =
              a.weight != nullptr ? d * load_param<T>(a.weight, a.param_f32, c + i) : d;
          sum_g += g;
          sum_gu += g * u;
          dw[k][i] += d * u;
          db[k][i] += d;
        }
      }
    }
    if (!a.want_dx) continue;
    const float mean_g = group_sum<G>(sum_g, scratch) * inverse;
    const float mean_gu = group_sum<G>(sum_gu, scratch) * inverse;
    if (!live) continue;
    T* dx = static_cast<T*>(a.y) + row * a.width;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = static_cast<int64_t>(k * G + lane) * V;
      if (c < a.width) {
        Pack<T, V> out;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = widen(rd[k].v[i]);
          const float u = (widen(rx[k].v[i]) - mean) * rstd;
          const float g =
              a.weight != nullptr ? d * load_param<T>(a.weight, a.param_f32, c + i) : d;
          out.v[i] = narrow<T>(rstd * (g - mean_g - u * mean_gu));
        }
        *reinterpret_cast<Pack<T, V>*>(dx + c) = out;
      }
    }
  }
  if (!a.want_params) return;
  float* partial = static_cast<float*>(a.partials) + static_cast<int64_t>(blockIdx.x) * 2 * a.width;
  if constexpr (kRows > 1) {
    // Rows of one warp first (lanes of the same columns), then the warps in order.
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int d = G; d < 32; d *= 2) {
          dw[k][i] += __shfl_xor_sync(0xffffffffu, dw[k][i], d);
          db[k][i] += __shfl_xor_sync(0xffffffffu, db[k][i], d);
        }
      }
    }
    for (int w = 0; w < kThreads / 32; ++w) {
      if (static_cast<int>(threadIdx.x) / 32 == w && (threadIdx.x & 31) < G) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int64_t c = static_cast<int64_t>(k * G + lane) * V;
          if (c < a.width) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
              columns[c + i] = w == 0 ? dw[k][i] : columns[c + i] + dw[k][i];
              columns[a.width + c + i] = w == 0 ? db[k][i] : columns[a.width + c + i] + db[k][i];
            }
          }
        }
      }
      __syncthreads();
    }
    for (int64_t c = threadIdx.x; c < 2 * a.width; c += kThreads) partial[c] = columns[c];
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = static_cast<int64_t>(k * G + lane) * V;
      if (c < a.width) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          partial[c + i] = dw[k][i];
          partial[a.width + c + i] = db[k][i];
        }
      }
    }
  }
}

// ---- rows of any width and type --------------------------------------------------------

constexpr int kLoopThreads = 512;

template <typename T>
__global__ void __launch_bounds__(kLoopThreads) norm_forward_loop_kernel(const NormArgs a) {
  using A = typename Wide<T>::type;
  __shared__ A scratch[32];
  const A inverse = A(1) / static_cast<A>(a.width);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    T* y = static_cast<T*>(a.y) + row * a.width;
    A sum = 0, squares = 0;
    for (int64_t c = threadIdx.x; c < a.width; c += kLoopThreads) sum += widen(x[c]);
    const A mean = group_sum<kLoopThreads>(sum, scratch) * inverse;
    for (int64_t c = threadIdx.x; c < a.width; c += kLoopThreads) {
      const A d = widen(x[c]) - mean;
      squares += d * d;
    }
    const A variance = group_sum<kLoopThreads>(squares, scratch) * inverse;
    const A rstd = A(1) / sqrt(variance + static_cast<A>(a.eps));
    if (a.stats != nullptr && threadIdx.x == 0) {
      static_cast<A*>(a.stats)[row] = mean;
      static_cast<A*>(a.stats)[a.rows + row] = rstd;
    }
    for (int64_t c = threadIdx.x; c < a.width; c += kLoopThreads) {
      A v = (widen(x[c]) - mean) * rstd;
      if (a.weight != nullptr) v *= load_param<T>(a.weight, a.param_f32, c);
      if (a.bias != nullptr) v += load_param<T>(a.bias, a.param_f32, c);
      y[c] = narrow<T>(v);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kLoopThreads) norm_dx_loop_kernel(const NormArgs a) {
  using A = typename Wide<T>::type;
  __shared__ A scratch[32];
  const A inverse = A(1) / static_cast<A>(a.width);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
    T* dx = static_cast<T*>(a.y) + row * a.width;
    const A mean = static_cast<const A*>(a.stats)[row];
    const A rstd = static_cast<const A*>(a.stats)[a.rows + row];
    A sum_g = 0, sum_gu = 0;
    for (int64_t c = threadIdx.x; c < a.width; c += kLoopThreads) {
      A g = widen(dy[c]);
      if (a.weight != nullptr) g *= load_param<T>(a.weight, a.param_f32, c);
      sum_g += g;
      sum_gu += g * ((widen(x[c]) - mean) * rstd);
    }
    const A mean_g = group_sum<kLoopThreads>(sum_g, scratch) * inverse;
    const A mean_gu = group_sum<kLoopThreads>(sum_gu, scratch) * inverse;
    for (int64_t c = threadIdx.x; c < a.width; c += kLoopThreads) {
      A g = widen(dy[c]);
      if (a.weight != nullptr) g *= load_param<T>(a.weight, a.param_f32, c);
      const A u = (widen(x[c]) - mean) * rstd;
      dx[c] = narrow<T>(rstd * (g - mean_g - u * mean_gu));
    }
  }
}

// Column sums of a row range (blockIdx.y of gridDim.y) into partial row blockIdx.y: a
// thread owns one column of 128.
template <typename T>
__global__ void __launch_bounds__(128) norm_columns_kernel(const NormArgs a) {
  using A = typename Wide<T>::type;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x;
  if (c >= a.width) return;
  const int64_t first = a.rows * blockIdx.y / gridDim.y;
  const int64_t last = a.rows * (blockIdx.y + 1) / gridDim.y;
  A dw = 0, db = 0;
  for (int64_t row = first; row < last; ++row) {
    const A mean = static_cast<const A*>(a.stats)[row];
    const A rstd = static_cast<const A*>(a.stats)[a.rows + row];
    const A d = widen((static_cast<const T*>(a.dy) + row * a.dy_stride)[c]);
    dw += d * ((widen((static_cast<const T*>(a.x) + row * a.x_stride)[c]) - mean) * rstd);
    db += d;
  }
  A* partial = static_cast<A*>(a.partials) + static_cast<int64_t>(blockIdx.y) * 2 * a.width;
  partial[c] = dw;
  partial[a.width + c] = db;
}

// Partial rows [blocks][2][width] summed in order: a block takes 32 columns, its 8 warps
// contiguous ranges of the rows, and the range sums are added in range order.
template <typename T>
__global__ void __launch_bounds__(256)
    norm_reduce_kernel(const void* partials, int blocks, int64_t width, void* dweight,
                       void* dbias, int param_f32) {
  using A = typename Wide<T>::type;
  __shared__ A part[8][32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  A sum = 0;
  if (j < 2 * width) {
    const A* p = static_cast<const A*>(partials) + j;
    const int last = blocks * (warp + 1) / 8;
#pragma unroll 8
    for (int b = blocks * warp / 8; b < last; ++b) sum += p[static_cast<int64_t>(b) * 2 * width];
  }
  part[warp][lane] = sum;
  __syncthreads();
  if (warp != 0 || j >= 2 * width) return;
  for (int w = 1; w < 8; ++w) sum += part[w][lane];
  if (j < width) {
    if (dweight != nullptr) store_param<T>(dweight, param_f32, j, sum);
  } else if (dbias != nullptr) {
    store_param<T>(dbias, param_f32, j - width, sum);
  }
}

// ---- choice of kernel ------------------------------------------------------------------

struct NormShape {
  int vector;   // elements per load: 16 bytes, or 1 where rows are not 16-byte aligned
  int chunks;   // vectors per row
  bool loops;   // wider than the register kernels (or float64)
};

constexpr int kMostChunks = 2048;

NormShape norm_shape(int dtype, int64_t width, bool aligned) {
  NormShape s{};
  const int wide = 16 / element_size(dtype);
  s.vector = aligned && width % wide == 0 ? wide : 1;
  s.loops = dtype == CND_F64 || width / s.vector > kMostChunks;
  s.chunks = s.loops ? 0 : static_cast<int>(width / s.vector);
  return s;
}

int norm_rows_per_block(const NormShape& s) {
  if (s.chunks <= 4) return 64;
  if (s.chunks <= 8) return 32;
  if (s.chunks <= 16) return 16;
  return s.chunks <= 128 ? 8 : 1;
}

// Blocks of the backward (one partial row each): enough to fill the SMs, no more than rows.
int norm_backward_blocks(const NormShape& s, int64_t rows, int64_t width) {
  if (s.loops) {
    // column kernel: row ranges of at least 64 rows
    const int64_t most = std::max<int64_t>(1, rows / 64);
    const int64_t across = (width + 127) / 128;
    return static_cast<int>(std::min<int64_t>(most, std::max<int64_t>(1, 8 * 148 / across)));
  }
  const int per_block = norm_rows_per_block(s);
  const int64_t need = (rows + per_block - 1) / per_block;
  return static_cast<int>(std::min<int64_t>(need, 4 * 148));
}

template <typename T, int V, typename F>
void with_shape(const NormShape& s, F&& f) {
  if (s.chunks <= 4) {
    f.template operator()<T, V, 1, 4>();
  } else if (s.chunks <= 8) {
    f.template operator()<T, V, 1, 8>();
  } else if (s.chunks <= 16) {
    f.template operator()<T, V, 1, 16>();
  } else if (s.chunks <= 32) {
    f.template operator()<T, V, 1, 32>();
  } else if (s.chunks <= 64) {
    f.template operator()<T, V, 2, 32>();
  } else if (s.chunks <= 128) {
    f.template operator()<T, V, 4, 32>();
  } else if (s.chunks <= 256) {
    f.template operator()<T, V, 2, 128>();
  } else if (s.chunks <= 512) {
    f.template operator()<T, V, 2, 256>();
  } else if (s.chunks <= 1024) {
    f.template operator()<T, V, 2, 512>();
  } else {
    f.template operator()<T, V, 2, 1024>();
  }
}

template <typename F>
void with_kernel(int dtype, const NormShape& s, F&& f) {
  if (dtype == CND_F32) {
    s.vector == 1 ? with_shape<float, 1>(s, f) : with_shape<float, 4>(s, f);
  } else if (dtype == CND_BF16) {
    s.vector == 1 ? with_shape<__nv_bfloat16, 1>(s, f) : with_shape<__nv_bfloat16, 8>(s, f);
  } else {
    s.vector == 1 ? with_shape<__half, 1>(s, f) : with_shape<__half, 8>(s, f);
  }
}

struct LaunchForward {
  const NormArgs& a;
  cudaStream_t stream;
  template <typename T, int V, int NV, int G>
  void operator()() const {
    constexpr int kRows = block_size<G>() / G;
    const int64_t need = (a.rows + kRows - 1) / kRows;
    const int64_t most = static_cast<int64_t>(sm_count()) * (2048 / block_size<G>()) * 4;
    norm_forward_kernel<T, V, NV, G>
        <<<static_cast<unsigned>(std::min(need, most)), block_size<G>(), 0, stream>>>(a);
  }
};

struct LaunchBackward {
  const NormArgs& a;
  int blocks;
  cudaStream_t stream;
  template <typename T, int V, int NV, int G>
  void operator()() const {
    constexpr int kRows = block_size<G>() / G;
    const size_t shared = kRows > 1 ? static_cast<size_t>(a.width) * 2 * sizeof(float) : 0;
    norm_backward_kernel<T, V, NV, G><<<blocks, block_size<G>(), shared, stream>>>(a);
  }
};

int check_norm(const char* who, int dtype, int param_dtype, int64_t rows, int64_t width,
               int64_t stride) {
  if (!known_dtype(dtype)) return fail(CND_ERR_UNSUPPORTED, "%s: unknown dtype %d", who, dtype);
  if (param_dtype != dtype && !(param_dtype == CND_F32 && dtype != CND_F64)) {
    return fail(CND_ERR_UNSUPPORTED, "%s: weight and bias must have the input's dtype or float32",
                who);
  }
  if (rows < 0 || width <= 0 || stride < width) {
    return fail(CND_ERR_INVALID, "%s: rows must be nonnegative, width positive and the row "
                "stride at least the width", who);
  }
  if (product(rows, std::max(stride, width)) < 0) {
    return fail(CND_ERR_INVALID, "%s: size overflows int64", who);
  }
  return CND_OK;
}

bool rows_aligned(int dtype, const void* p, int64_t stride) {
  return aligned16(p) && stride * element_size(dtype) % 16 == 0;
}

}  // namespace
}  // namespace layers
}  // namespace cnd

extern "C" {

int cnd_layer_norm_forward(int32_t dtype, int32_t param_dtype, int64_t rows, int64_t width,
                           int64_t x_stride, double eps, const void* x, const void* weight,
                           const void* bias, void* y, void* stats, void* stream_handle) {
  using namespace cnd;
  using namespace cnd::layers;
  clear_error();
  int rc = check_norm("cnd_layer_norm_forward", dtype, param_dtype, rows, width, x_stride);
  if (rc != CND_OK) return rc;
  if (rows == 0) return CND_OK;
  if (x == nullptr || y == nullptr) {
    return fail(CND_ERR_INVALID, "cnd_layer_norm_forward: x and y must not be NULL");
  }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  NormArgs a{};
  a.x = x;
  a.weight = weight;
  a.bias = bias;
  a.y = y;
  a.stats = stats;
  a.rows = rows;
  a.width = width;
  a.x_stride = x_stride;
  a.eps = eps;
  a.param_f32 = param_dtype == CND_F32;
  const NormShape s = norm_shape(dtype, width, rows_aligned(dtype, x, x_stride) && aligned16(y));
  if (s.loops) {
    const unsigned blocks =
        static_cast<unsigned>(std::min<int64_t>(rows, static_cast<int64_t>(sm_count()) * 16));
    if (dtype == CND_F64) {
      norm_forward_loop_kernel<double><<<blocks, kLoopThreads, 0, stream>>>(a);
    } else if (dtype == CND_F32) {
      norm_forward_loop_kernel<float><<<blocks, kLoopThreads, 0, stream>>>(a);
    } else if (dtype == CND_BF16) {
      norm_forward_loop_kernel<__nv_bfloat16><<<blocks, kLoopThreads, 0, stream>>>(a);
    } else {
      norm_forward_loop_kernel<__half><<<blocks, kLoopThreads, 0, stream>>>(a);
    }
  } else {
    with_kernel(dtype, s, LaunchForward{a, stream});
  }
  count_launch();
  return launch_status("cnd_layer_norm_forward");
}

size_t cnd_layer_norm_backward_workspace_size(int32_t dtype, int64_t rows, int64_t width,
                                              const int32_t output_mask[3]) {
  using namespace cnd::layers;
  if (!known_dtype(dtype) || rows <= 0 || width <= 0 || output_mask == nullptr) return 0;
  if (!output_mask[1] && !output_mask[2]) return 0;
  // the larger of what aligned and unaligned rows take
  int blocks = 0;
  for (const bool aligned : {false, true}) {
    blocks = std::max(blocks, norm_backward_blocks(norm_shape(dtype, width, aligned), rows, width));
  }
  return static_cast<size_t>(blocks) * 2 * static_cast<size_t>(width) *
         (dtype == CND_F64 ? sizeof(double) : sizeof(float));
}

int cnd_layer_norm_backward(int32_t dtype, int32_t param_dtype, int64_t rows, int64_t width,
                            int64_t dy_stride, int64_t x_stride, const void* dy, const void* x,
                            const void* weight, const void* stats, void* dx, void* dweight,
                            void* dbias, const int32_t output_mask[3], void* workspace,
                            size_t workspace_bytes, void* stream_handle) {
  using namespace cnd;
  using namespace cnd::layers;
  clear_error();
  int rc = check_norm("cnd_layer_norm_backward", dtype, param_dtype, rows, width,
                      std::min(dy_stride, x_stride));
  if (rc == CND_OK && product(rows, std::max(dy_stride, x_stride)) < 0) {
    rc = fail(CND_ERR_INVALID, "cnd_layer_norm_backward: size overflows int64");
  }
  if (rc != CND_OK) return rc;
  if (output_mask == nullptr) {
    return fail(CND_ERR_INVALID, "cnd_layer_norm_backward: output_mask must not be NULL");
  }
  const bool params = output_mask[1] || output_mask[2];
  if (!output_mask[0] && !params) return CND_OK;
  if ((output_mask[1] && dweight == nullptr) || (output_mask[2] && dbias == nullptr) ||
      (rows > 0 && (dy == nullptr || x == nullptr || stats == nullptr ||
                    (output_mask[0] && dx == nullptr)))) {
    return fail(CND_ERR_INVALID, "cnd_layer_norm_backward: a required buffer is NULL");
  }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  if (rows == 0) {
    const size_t bytes = static_cast<size_t>(width) * element_size(param_dtype);
    if (output_mask[1]) cudaMemsetAsync(dweight, 0, bytes, stream);
    if (output_mask[2]) cudaMemsetAsync(dbias, 0, bytes, stream);
    return launch_status("cnd_layer_norm_backward");
  }
  const size_t need = cnd_layer_norm_backward_workspace_size(dtype, rows, width, output_mask);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    return fail(CND_ERR_WORKSPACE, "cnd_layer_norm_backward: workspace of %zu bytes, %zu needed",
                workspace == nullptr ? size_t{0} : workspace_bytes, need);
  }
  NormArgs a{};
  a.x = x;
  a.dy = dy;
  a.weight = weight;
  a.y = dx;
  a.stats = const_cast<void*>(stats);
  a.partials = workspace;
  a.rows = rows;
  a.width = width;
  a.x_stride = x_stride;
  a.dy_stride = dy_stride;
  a.param_f32 = param_dtype == CND_F32;
  a.want_dx = output_mask[0] != 0;
  a.want_params = params;
  const bool aligned = rows_aligned(dtype, x, x_stride) && rows_aligned(dtype, dy, dy_stride) &&
                       (!a.want_dx || aligned16(dx));
  const NormShape s = norm_shape(dtype, width, aligned);
  const int blocks = norm_backward_blocks(s, rows, width);
  if (s.loops) {
    const unsigned grid =
        static_cast<unsigned>(std::min<int64_t>(rows, static_cast<int64_t>(sm_count()) * 16));
    const dim3 columns(static_cast<unsigned>((width + 127) / 128), static_cast<unsigned>(blocks));
    const auto run = [&](auto zero) {
      using T = decltype(zero);
      if (a.want_dx) {
        norm_dx_loop_kernel<T><<<grid, kLoopThreads, 0, stream>>>(a);
        count_launch();
      }
      if (params) {
        norm_columns_kernel<T><<<columns, 128, 0, stream>>>(a);
        count_launch();
      }
    };
    if (dtype == CND_F64) {
      run(double{});
    } else if (dtype == CND_F32) {
      run(float{});
    } else if (dtype == CND_BF16) {
      run(__nv_bfloat16{});
    } else {
      run(__half{});
    }
  } else {
    with_kernel(dtype, s, LaunchBackward{a, blocks, stream});
    count_launch();
  }
  if (params) {
    const unsigned grid = static_cast<unsigned>((2 * width + 31) / 32);
    void* w = output_mask[1] ? dweight : nullptr;
    void* b = output_mask[2] ? dbias : nullptr;
    if (dtype == CND_F64) {
      norm_reduce_kernel<double><<<grid, 256, 0, stream>>>(workspace, blocks, width, w, b, 0);
    } else if (dtype == CND_F32 || a.param_f32) {
      norm_reduce_kernel<float><<<grid, 256, 0, stream>>>(workspace, blocks, width, w, b, 1);
    } else if (dtype == CND_BF16) {
      norm_reduce_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(workspace, blocks, width, w, b, 0);
    } else {
      norm_reduce_kernel<__half><<<grid, 256, 0, stream>>>(workspace, blocks, width, w, b, 0);
    }
    count_launch();
  }
  return launch_status("cnd_layer_norm_backward");
}

}  // extern "C"
