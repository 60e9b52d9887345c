// Linear layers: y = act(x W^T + bias) + residual and their backward pass
//
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  dbias = column sums of dz.
//
// The products run on the CUDA cores: 64 x 64 tiles, each of 256 threads 4 x 4 of them,
// float32 sums (float64 for float64).
#include <algorithm>

#include "layers.cuh"

namespace cnd {
namespace layers {
namespace {

// GELU'(v) = Phi(v) + v phi(v); SiLU'(v) = s (1 + v (1 - s)), s = 1 / (1 + exp(-v)).
template <typename A>
__device__ __forceinline__ A activate(A v, int act) {
  if (act == CND_ACT_GELU) return A(0.5) * v * (A(1) + erf(v * A(0.70710678118654752440)));
  if (act == CND_ACT_SILU) return v / (A(1) + exp(-v));
  return v;
}

template <typename A>
__device__ __forceinline__ A activation_slope(A v, int act) {
  if (act == CND_ACT_GELU) {
    const A cdf = A(0.5) * (A(1) + erf(v * A(0.70710678118654752440)));
    return cdf + v * exp(A(-0.5) * v * v) * A(0.39894228040143267794);
  }
  if (act == CND_ACT_SILU) {
    const A s = A(1) / (A(1) + exp(-v));
    return s * (A(1) + v * (A(1) - s));
  }
  return A(1);
}

// d[m][n] = sum_k a(m, k) b(n, k), element (i, k) of an operand at i * row + k * col.
struct ProductArgs {
  const void *a, *b, *bias, *residual;
  void *d, *pre;
  int64_t m, n, k;
  int64_t a_row, a_col, b_row, b_col;
  int act;
};

constexpr int kTile = 64, kDepth = 16;

template <typename T>
__global__ void __launch_bounds__(256) product_kernel(const ProductArgs p) {
  using A = typename Wide<T>::type;
  __shared__ A sa[kDepth][kTile + 1], sb[kDepth][kTile + 1];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int64_t m0 = static_cast<int64_t>(blockIdx.x) * kTile;
  const int64_t n0 = static_cast<int64_t>(blockIdx.y) * kTile;
  const T* a = static_cast<const T*>(p.a);
  const T* b = static_cast<const T*>(p.b);
  A sum[4][4] = {};
  for (int64_t k0 = 0; k0 < p.k; k0 += kDepth) {
    for (int i = threadIdx.x; i < kTile * kDepth; i += 256) {
      const int r = p.a_col == 1 ? i / kDepth : i % kTile;
      const int k = p.a_col == 1 ? i % kDepth : i / kTile;
      const bool in = m0 + r < p.m && k0 + k < p.k;
      sa[k][r] = in ? widen(a[(m0 + r) * p.a_row + (k0 + k) * p.a_col]) : A(0);
    }
    for (int i = threadIdx.x; i < kTile * kDepth; i += 256) {
      const int r = p.b_col == 1 ? i / kDepth : i % kTile;
      const int k = p.b_col == 1 ? i % kDepth : i / kTile;
      const bool in = n0 + r < p.n && k0 + k < p.k;
      sb[k][r] = in ? widen(b[(n0 + r) * p.b_row + (k0 + k) * p.b_col]) : A(0);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
      A u[4], v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u[i] = sa[k][ty * 4 + i];
        v[i] = sb[k][tx + 16 * i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[i][j] += u[i] * v[j];
      }
    }
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty * 4 + i;
    if (m >= p.m) break;
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx + 16 * j;
      if (n >= p.n) break;
      A v = sum[i][j];
      if (p.bias != nullptr) v += widen(static_cast<const T*>(p.bias)[n]);
      if (p.pre != nullptr) static_cast<T*>(p.pre)[m * p.n + n] = narrow<T>(v);
      v = activate<A>(v, p.act);
      if (p.residual != nullptr) v += widen(static_cast<const T*>(p.residual)[m * p.n + n]);
      static_cast<T*>(p.d)[m * p.n + n] = narrow<T>(v);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
    slope_kernel(const T* dy, const T* pre, T* dz, int64_t count, int act) {
  using A = typename Wide<T>::type;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < count; i += step) {
    dz[i] = narrow<T>(widen(dy[i]) * activation_slope<A>(widen(pre[i]), act));
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
    column_sum_kernel(const T* dz, T* dbias, int64_t rows, int64_t width) {
  using A = typename Wide<T>::type;
  __shared__ A part[8][32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  A sum = 0;
  if (c < width) {
    for (int64_t r = rows * warp / 8; r < rows * (warp + 1) / 8; ++r) sum += widen(dz[r * width + c]);
  }
  part[warp][lane] = sum;
  __syncthreads();
  if (warp != 0 || c >= width) return;
  for (int w = 1; w < 8; ++w) sum += part[w][lane];
  dbias[c] = narrow<T>(sum);
}

template <typename F>
void with_dtype(int dtype, F&& f) {
  if (dtype == CND_F64) {
    f(double{});
  } else if (dtype == CND_F32) {
    f(float{});
  } else if (dtype == CND_BF16) {
    f(__nv_bfloat16{});
  } else {
    f(__half{});
  }
}

void launch_product(int dtype, const ProductArgs& p, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>((p.m + kTile - 1) / kTile),
                  static_cast<unsigned>((p.n + kTile - 1) / kTile));
  with_dtype(dtype, [&](auto zero) {
    product_kernel<decltype(zero)><<<grid, 256, 0, stream>>>(p);
  });
  count_launch();
}

int check_linear(const char* who, const cnd_linear* p) {
  if (p == nullptr) return fail(CND_ERR_INVALID, "%s: problem must not be NULL", who);
  if (!known_dtype(p->dtype)) {
    return fail(CND_ERR_UNSUPPORTED, "%s: unknown dtype %d", who, p->dtype);
  }
  if (p->activation != CND_ACT_NONE && p->activation != CND_ACT_GELU &&
      p->activation != CND_ACT_SILU) {
    return fail(CND_ERR_UNSUPPORTED, "%s: unknown activation %d", who, p->activation);
  }
  if (p->rows < 0 || p->in_features <= 0 || p->out_features <= 0 ||
      p->x_stride < p->in_features) {
    return fail(CND_ERR_INVALID, "%s: rows must be nonnegative, features positive and the row "
                "stride at least in_features", who);
  }
  if (product(p->rows, std::max(p->x_stride, p->out_features)) < 0 ||
      product(p->in_features, p->out_features) < 0) {
    return fail(CND_ERR_INVALID, "%s: size overflows int64", who);
  }
  return CND_OK;
}

int check_workspace(const char* who, const void* workspace, size_t bytes, size_t need) {
  if (need > 0 && (workspace == nullptr || bytes < need)) {
    return fail(CND_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who,
                workspace == nullptr ? size_t{0} : bytes, need);
  }
  return CND_OK;
}

}  // namespace
}  // namespace layers
}  // namespace cnd

extern "C" {

size_t cnd_linear_forward_workspace_size(const cnd_linear* problem) {
  (void)problem;
  return 0;
}

int cnd_linear_forward(const cnd_linear* problem, const void* x, const void* weight,
                       const void* bias, const void* residual, void* y, void* pre,
                       void* workspace, size_t workspace_bytes, void* stream_handle) {
  using namespace cnd;
  using namespace cnd::layers;
  clear_error();
  int rc = check_linear("cnd_linear_forward", problem);
  if (rc != CND_OK) return rc;
  if (problem->rows == 0) return CND_OK;
  if (x == nullptr || weight == nullptr || y == nullptr) {
    return fail(CND_ERR_INVALID, "cnd_linear_forward: x, weight and y must not be NULL");
  }
  rc = check_workspace("cnd_linear_forward", workspace, workspace_bytes,
                       cnd_linear_forward_workspace_size(problem));
  if (rc != CND_OK) return rc;
  ProductArgs p{};
  p.a = x;
  p.b = weight;
  p.bias = bias;
  p.residual = residual;
  p.d = y;
  p.pre = pre;
  p.m = problem->rows;
  p.n = problem->out_features;
  p.k = problem->in_features;
  p.a_row = problem->x_stride;
  p.a_col = 1;
  p.b_row = problem->in_features;
  p.b_col = 1;
  p.act = problem->activation;
  launch_product(problem->dtype, p, static_cast<cudaStream_t>(stream_handle));
  return launch_status("cnd_linear_forward");
}

size_t cnd_linear_backward_workspace_size(const cnd_linear* problem,
                                          const int32_t output_mask[3]) {
  (void)output_mask;
  if (problem == nullptr || problem->activation == CND_ACT_NONE) return 0;
  return static_cast<size_t>(problem->rows) * static_cast<size_t>(problem->out_features) *
         cnd::layers::element_size(problem->dtype);
}

int cnd_linear_backward(const cnd_linear* problem, const void* dy, const void* pre,
                        const void* x, const void* weight, void* dx, void* dweight, void* dbias,
                        const int32_t output_mask[3], void* workspace, size_t workspace_bytes,
                        void* stream_handle) {
  using namespace cnd;
  using namespace cnd::layers;
  clear_error();
  int rc = check_linear("cnd_linear_backward", problem);
  if (rc != CND_OK) return rc;
  if (output_mask == nullptr) {
    return fail(CND_ERR_INVALID, "cnd_linear_backward: output_mask must not be NULL");
  }
  if (!output_mask[0] && !output_mask[1] && !output_mask[2]) return CND_OK;
  const int64_t rows = problem->rows, in = problem->in_features, out = problem->out_features;
  const bool act = problem->activation != CND_ACT_NONE;
  if ((output_mask[1] && dweight == nullptr) || (output_mask[2] && dbias == nullptr) ||
      (rows > 0 && (dy == nullptr || (act && pre == nullptr) ||
                    (output_mask[0] && (dx == nullptr || weight == nullptr)) ||
                    (output_mask[1] && x == nullptr)))) {
    return fail(CND_ERR_INVALID, "cnd_linear_backward: a required buffer is NULL");
  }
  rc = check_workspace("cnd_linear_backward", workspace, workspace_bytes,
                       cnd_linear_backward_workspace_size(problem, output_mask));
  if (rc != CND_OK) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  const void* dz = dy;
  if (act && rows > 0) {
    const int64_t count = rows * out;
    const unsigned grid = static_cast<unsigned>(
        std::min<int64_t>((count + 255) / 256, static_cast<int64_t>(sm_count()) * 32));
    with_dtype(problem->dtype, [&](auto zero) {
      using T = decltype(zero);
      slope_kernel<T><<<grid, 256, 0, stream>>>(static_cast<const T*>(dy),
                                                static_cast<const T*>(pre),
                                                static_cast<T*>(workspace), count,
                                                problem->activation);
    });
    count_launch();
    dz = workspace;
  }
  if (output_mask[0] && rows > 0) {
    ProductArgs p{};
    p.a = dz;
    p.b = weight;
    p.d = dx;
    p.m = rows;
    p.n = in;
    p.k = out;
    p.a_row = out;
    p.a_col = 1;
    p.b_row = 1;
    p.b_col = in;
    launch_product(problem->dtype, p, stream);
  }
  if (output_mask[1]) {
    ProductArgs p{};
    p.a = dz;
    p.b = x;
    p.d = dweight;
    p.m = out;
    p.n = in;
    p.k = rows;
    p.a_row = 1;
    p.a_col = out;
    p.b_row = 1;
    p.b_col = problem->x_stride;
    launch_product(problem->dtype, p, stream);
  }
  if (output_mask[2]) {
    with_dtype(problem->dtype, [&](auto zero) {
      using T = decltype(zero);
      column_sum_kernel<T><<<static_cast<unsigned>((out + 31) / 32), 256, 0, stream>>>(
          static_cast<const T*>(dz), static_cast<T*>(dbias), rows, out);
    });
    count_launch();
  }
  return launch_status("cnd_linear_backward");
}

}  // extern "C"
