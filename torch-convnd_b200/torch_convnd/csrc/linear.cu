// Linear layers: y = act(x W^T + bias) + residual and their backward pass
//
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  dbias = column sums of dz.
//
// 16-bit and float32 products run on the tensor cores (product.cu). What they need beside
// the products is one kernel here, prepare_kernel: it reads a matrix once and writes it as a
// product's operand, multiplied by the activation's slope on the way (dz), split into three
// bfloat16 terms (float32), or with rows padded to 16 bytes (sizes that TMA cannot address),
// and sums its columns (dbias). Operands that TMA can read as they lie are not copied. The
// backward of thin 16-bit layers with an activation is one kernel (thin.cu). float64 runs on
// the CUDA cores.
//
// In 16-bit layers z and dz are rounded to the operands' type: dz has to be for the products
// (two terms of it would double them), z to be kept at half the traffic (float32 would move 1.07
// GB more for 1M x 64 -> 256, 164 us). Against float64 the gradients are 1.46 times as far off as
// with both in float32, 1.41 times with dz alone rounded; dbias sums dz before its rounding.
#include <algorithm>

#include "activation.cuh"
#include "layers.cuh"
#include "product.cuh"

namespace cnd {
namespace layers {
namespace {

// d[m][n] = sum_k a(m, k) b(n, k), element (i, k) of an operand at i * row + k * col.
struct DoubleProduct {
  const double *a, *b, *bias, *residual;
  double *d, *pre;
  int64_t m, n, k;
  int64_t a_row, a_col, b_row, b_col;
  int act;
};

constexpr int kTile = 64, kDepth = 16;

// 64 x 64 tiles, 4 x 4 values a thread.
__global__ void __launch_bounds__(256) double_product_kernel(const DoubleProduct p) {
  __shared__ double sa[kDepth][kTile + 1], sb[kDepth][kTile + 1];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int64_t m0 = static_cast<int64_t>(blockIdx.x) * kTile;
  // a grid has at most 65535 blocks in y
  for (int64_t n0 = static_cast<int64_t>(blockIdx.y) * kTile; n0 < p.n;
       n0 += static_cast<int64_t>(gridDim.y) * kTile) {
    double sum[4][4] = {};
    for (int64_t k0 = 0; k0 < p.k; k0 += kDepth) {
      for (int i = threadIdx.x; i < kTile * kDepth; i += 256) {
        const int r = p.a_col == 1 ? i / kDepth : i % kTile;
        const int k = p.a_col == 1 ? i % kDepth : i / kTile;
        const bool in = m0 + r < p.m && k0 + k < p.k;
        sa[k][r] = in ? p.a[(m0 + r) * p.a_row + (k0 + k) * p.a_col] : 0.0;
      }
      for (int i = threadIdx.x; i < kTile * kDepth; i += 256) {
        const int r = p.b_col == 1 ? i / kDepth : i % kTile;
        const int k = p.b_col == 1 ? i % kDepth : i / kTile;
        const bool in = n0 + r < p.n && k0 + k < p.k;
        sb[k][r] = in ? p.b[(n0 + r) * p.b_row + (k0 + k) * p.b_col] : 0.0;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kDepth; ++k) {
        double u[4], v[4];
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
        double v = sum[i][j];
        if (p.bias != nullptr) v += p.bias[n];
        if (p.pre != nullptr) p.pre[m * p.n + n] = v;
        v = activate(v, p.act);
        if (p.residual != nullptr) v += p.residual[m * p.n + n];
        p.d[m * p.n + n] = v;
      }
    }
  }
}

// ---- operands --------------------------------------------------------------------------

struct PrepareArgs {
  const void* src;  // [rows][width], rows src_stride apart
  const void* pre;  // [rows][width] dense, or NULL: no activation
  void* dst;        // NULL: column sums only
  void* sums;       // [gridDim.y][width] partial column sums, or NULL
  int64_t rows, width, src_stride, pitch, plane;
  int act;
  int lanes;  // lanes of a row (8 columns each): a power of two, all 32 from 256 columns on
};

constexpr int kPrepareColumns = 256;  // most columns of a block: 32 lanes of 8

// Writes 8 columns of a row as an operand: split into three bfloat16 terms (float32), or as they
// are (float64).
template <typename T, typename A>
__device__ __forceinline__ void store_operand(const PrepareArgs& a, int64_t row, int64_t col,
                                              const A (&w)[8]) {
  if constexpr (sizeof(T) == 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (col + i < a.width) static_cast<T*>(a.dst)[row * a.pitch + col + i] = w[i];
    }
  } else {
    // x = x0 + x1 + x2, each the nearest bfloat16 of what is left; an infinity or NaN is x0
    // alone
    Pack<__nv_bfloat16, 8> t[3];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      t[0].v[i] = __float2bfloat16_rn(w[i]);
      float rest = w[i] - __bfloat162float(t[0].v[i]);
      if (!isfinite(rest)) {
        // near the largest float32, x0 would round up to infinity: round it down
        t[0].v[i] = isfinite(w[i]) ? __float2bfloat16_rz(w[i]) : t[0].v[i];
        rest = isfinite(w[i]) ? w[i] - __bfloat162float(t[0].v[i]) : 0.0f;
      }
      t[1].v[i] = __float2bfloat16_rn(rest);
      t[2].v[i] = __float2bfloat16_rn(rest - __bfloat162float(t[1].v[i]));
    }
    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.dst) + row * a.pitch + col;
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      *reinterpret_cast<Pack<__nv_bfloat16, 8>*>(dst + p * a.plane) = t[p];
    }
  }
}

// T: source type. A block takes up to 256 columns and a range of rows, a lane 8 consecutive
// columns of a row: 16-byte loads and stores where rows allow them. A warp takes one row at a
// time, or several narrow ones.
template <typename T, bool kVectors>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 2) prepare_kernel(const PrepareArgs a) {
  using A = typename Wide<T>::type;
  constexpr int kBatch = 2;
  constexpr int kLoad = sizeof(T) == 2 ? 8 : 16 / sizeof(T);
  __shared__ A part[8][kPrepareColumns];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % a.lanes;
  const int rows = 256 / a.lanes, row_of = threadIdx.x / a.lanes;  // rows of the block at once
  const int64_t col = static_cast<int64_t>(blockIdx.x) * kPrepareColumns + lane * 8;
  const int64_t first = a.rows * blockIdx.y / gridDim.y;
  const int64_t last = a.rows * (blockIdx.y + 1) / gridDim.y;
  A sum[8] = {};
  Two sums[4] = {same(0.0f), same(0.0f), same(0.0f), same(0.0f)};
  if (col < a.width) {
    // Two rows are loaded before the first is worked on, and four blocks fit an SM: 4.8 TB/s on
    // 1M x 256 bf16; four rows in twice the registers reached 4.2.
    for (int64_t row0 = first + row_of; row0 < last; row0 += rows * kBatch) {
      alignas(16) T v[kBatch][8], z[kBatch][8];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int64_t row = row0 + rows * j;
        const bool live = row < last;
        const T* src = static_cast<const T*>(a.src) + row * a.src_stride + col;
        const T* pre = static_cast<const T*>(a.pre) + row * a.width + col;
        if constexpr (kVectors) {
#pragma unroll
          for (int i = 0; i < 8; i += kLoad) {
            if (live) {
              *reinterpret_cast<Pack<T, kLoad>*>(v[j] + i) =
                  *reinterpret_cast<const Pack<T, kLoad>*>(src + i);
            }
            if (live && a.pre != nullptr) {
              *reinterpret_cast<Pack<T, kLoad>*>(z[j] + i) =
                  *reinterpret_cast<const Pack<T, kLoad>*>(pre + i);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            v[j][i] = z[j][i] = narrow<T>(A(0));
            if (live && col + i < a.width) {
              v[j][i] = src[i];
              if (a.pre != nullptr) z[j][i] = pre[i];
            }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int64_t row = row0 + rows * j;
        if (row < last) {
          if constexpr (sizeof(T) == 2) {
            Two w[4];
            load_twos<T, 8>(v[j], w);
            if (a.pre != nullptr) {
              Two pre[4];
              load_twos<T, 8>(z[j], pre);
              if (a.act == CND_ACT_GELU) {
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = mul2(w[i], slope2(pre[i], CND_ACT_GELU));
              } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = mul2(w[i], slope2(pre[i], CND_ACT_SILU));
              }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[i] = add2(sums[i], w[i]);
            if (a.dst != nullptr) store_twos<T, 8>(static_cast<T*>(a.dst) + row * a.pitch + col, w);
          } else {
            A w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = widen(v[j][i]);
            if (a.pre != nullptr) {
#pragma unroll
              for (int i = 0; i < 8; ++i) w[i] *= activation_slope<A>(widen(z[j][i]), a.act);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += w[i];
            if (a.dst != nullptr) store_operand<T>(a, row, col, w);
          }
        }
      }
    }
  }
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) unpack(sums[i], &sum[2 * i], &sum[2 * i + 1]);
  }
  if (a.sums == nullptr) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) part[warp][threadIdx.x % 32 * 8 + i] = sum[i];
  __syncthreads();
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kPrepareColumns + threadIdx.x;
  if (c >= a.width || static_cast<int>(threadIdx.x) >= a.lanes * 8) return;
  A total = 0;
  for (int w = 0; w < 8; ++w) {
    for (int r = 0; r < 32 / a.lanes; ++r) total += part[w][r * a.lanes * 8 + threadIdx.x];
  }
  static_cast<A*>(a.sums)[blockIdx.y * a.width + c] = total;
}

// Partial column sums [count][width] added in order: a block takes 32 columns, its 32 warps
// contiguous ranges of the partial rows, and the range sums are added in range order.
constexpr int kJoinWarps = 32;
template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32)
    column_join_kernel(const void* sums, int count, int64_t width, T* out) {
  using A = typename Wide<T>::type;
  __shared__ A part[kJoinWarps][32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  A sum = 0;
  if (c < width) {
    const A* p = static_cast<const A*>(sums) + c;
#pragma unroll 8
    for (int r = count * warp / kJoinWarps; r < count * (warp + 1) / kJoinWarps; ++r) sum += p[r * width];
  }
  part[warp][lane] = sum;
  __syncthreads();
  if (warp != 0 || c >= width) return;
  for (int w = 1; w < kJoinWarps; ++w) sum += part[w][lane];
  out[c] = narrow<T>(sum);
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

void join_columns(int dtype, const void* sums, int count, int64_t width, void* out,
                  cudaStream_t stream) {
  with_dtype(dtype, [&](auto zero) {
    using T = decltype(zero);
    column_join_kernel<T><<<static_cast<unsigned>((width + 31) / 32), kJoinWarps * 32, 0, stream>>>(
        sums, count, width, static_cast<T*>(out));
  });
  count_launch();
}

// Elements between the rows of a prepared operand: whole 16-byte units, and whole 128-byte
// lines where that costs at most an eighth more (a 64-byte piece of a row that starts off a
// 32-byte sector is three sectors: float32 1999 x 771 -> 1280 took 46 us, 768 -> 1280 32).
int64_t row_pitch(int64_t width) {
  for (const int64_t unit : {64, 32, 16}) {
    const int64_t pitch = (width + unit - 1) / unit * unit;
    if (pitch <= width + width / 8) return pitch;
  }
  return (width + 7) / 8 * 8;
}
// Rows from which the one-pass backward of thin layers is taken: two of its tiles. At 512 rows
// it takes 23 us for 64 -> 256 in bf16 and separate launches 27, at 8192 rows 25 and 33, at
// 262144 rows 90 and 158; for 8 -> 8 14 and 23, 16 and 29, 41 and 84.
constexpr int64_t kThinRows = 256;

size_t up1024(size_t v) { return (v + 1023) / 1024 * 1024; }

// Row ranges of prepare_kernel's grid: about eight blocks an SM, 32 rows or more each.
int prepare_ranges(int64_t rows, int64_t width) {
  const int64_t across = (width + kPrepareColumns - 1) / kPrepareColumns;
  const int64_t ranges = std::min<int64_t>((rows + 31) / 32, (kSms * 8 + across - 1) / across);
  return static_cast<int>(std::max<int64_t>(1, ranges));
}

// Bytes of a prepared [rows][width] operand.
size_t operand_bytes(int dtype, int64_t rows, int64_t width) {
  return up1024(static_cast<size_t>(rows) * row_pitch(width) * (dtype == CND_F32 ? 6 : 2));
}

// Writes src (times the slope at pre) as an operand into dst (NULL: column sums only).
void prepare(int dtype, const void* src, const void* pre, int act, int64_t rows, int64_t width,
             int64_t stride, void* dst, int64_t pitch, void* sums, cudaStream_t stream) {
  PrepareArgs a{};
  a.src = src;
  a.pre = pre;
  a.dst = dst;
  a.sums = sums;
  a.rows = rows;
  a.width = width;
  a.src_stride = stride;
  a.pitch = pitch;
  a.plane = rows * pitch;
  a.act = act;
  const bool vectors = width % 8 == 0 && stride * element_size(dtype) % 16 == 0 &&
                       aligned16(src) && aligned16(pre);
  a.lanes = 1;
  while (a.lanes < 32 && a.lanes * 8 < width) a.lanes *= 2;
  const dim3 grid(static_cast<unsigned>((width + kPrepareColumns - 1) / kPrepareColumns),
                  static_cast<unsigned>(prepare_ranges(rows, width)));
  with_dtype(dtype, [&](auto zero) {
    using T = decltype(zero);
    vectors ? prepare_kernel<T, true><<<grid, 256, 0, stream>>>(a)
            : prepare_kernel<T, false><<<grid, 256, 0, stream>>>(a);
  });
  count_launch();
}

Operand operand_at(const void* data, int64_t rows, int64_t pitch, bool k_major) {
  return Operand{data, pitch, rows * pitch, k_major};
}

// What of a 16-bit or float32 problem has to be copied before TMA can read it.
bool copies_x(const cnd_linear& p) { return p.dtype == CND_F32 || p.x_stride % 8 != 0; }
bool copies_w(const cnd_linear& p) { return p.dtype == CND_F32 || p.in_features % 8 != 0; }
bool copies_dz(const cnd_linear& p) {
  return p.dtype == CND_F32 || p.activation != CND_ACT_NONE || p.out_features % 8 != 0;
}

// Whether the backward takes the one-pass kernel of thin layers.
bool one_pass(const cnd_linear& p, const int32_t mask[3]) {
  return (p.dtype == CND_BF16 || p.dtype == CND_F16) && p.activation != CND_ACT_NONE && mask[0] &&
         mask[1] && p.in_features <= kThinIn && p.out_features <= kThinOut &&
         p.in_features % 8 == 0 && p.out_features % 8 == 0 && p.x_stride % 8 == 0 &&
         p.rows >= kThinRows && p.rows < INT32_MAX - 128;
}

// Workspace of a call: byte offsets of its regions.
struct Layout {
  size_t dz = 0, x = 0, w = 0, sums = 0, splits = 0, total = 0;
};

size_t take(size_t* total, size_t bytes) {
  const size_t at = *total;
  *total += up1024(bytes);
  return at;
}

int parts_of(const cnd_linear& p) { return p.dtype == CND_F32 ? 3 : 1; }

Layout forward_layout(const cnd_linear& p) {
  Layout l;
  if (p.dtype == CND_F64) return l;
  if (copies_x(p)) l.x = take(&l.total, operand_bytes(p.dtype, p.rows, p.in_features));
  if (copies_w(p)) l.w = take(&l.total, operand_bytes(p.dtype, p.out_features, p.in_features));
  const ProductPlan plan = plan_product(p.rows, p.out_features, p.in_features, parts_of(p));
  l.splits = take(&l.total, product_workspace(plan, p.rows, p.out_features));
  return l;
}

Layout backward_layout(const cnd_linear& p, const int32_t mask[3]) {
  Layout l;
  if (one_pass(p, mask)) {
    const size_t blocks = thin_blocks(p.rows), out = p.out_features;
    if (mask[2]) l.sums = take(&l.total, blocks * out * sizeof(float));
    l.splits = take(&l.total, blocks * out * p.in_features * sizeof(float));
    return l;
  }
  const bool products = mask[0] || mask[1];
  if (p.dtype == CND_F64) {
    if (p.activation != CND_ACT_NONE) {
      l.dz = take(&l.total, static_cast<size_t>(p.rows) * p.out_features * sizeof(double));
    }
  } else {
    if (products && copies_dz(p)) {
      l.dz = take(&l.total, operand_bytes(p.dtype, p.rows, p.out_features));
    }
    if (mask[1] && copies_x(p)) l.x = take(&l.total, operand_bytes(p.dtype, p.rows, p.in_features));
    if (mask[0] && copies_w(p)) {
      l.w = take(&l.total, operand_bytes(p.dtype, p.out_features, p.in_features));
    }
  }
  if (mask[2]) {
    l.sums = take(&l.total, static_cast<size_t>(prepare_ranges(p.rows, p.out_features)) *
                                p.out_features * (p.dtype == CND_F64 ? 8 : 4));
  }
  if (p.dtype != CND_F64) {
    size_t splits = 0;
    if (mask[0]) {
      splits = product_workspace(plan_product(p.rows, p.in_features, p.out_features, parts_of(p)),
                                 p.rows, p.in_features);
    }
    if (mask[1]) {
      splits = std::max(splits, product_workspace(plan_product(p.out_features, p.in_features,
                                                               p.rows, parts_of(p)),
                                                  p.out_features, p.in_features));
    }
    l.splits = take(&l.total, splits);
  }
  return l;
}

void launch_double(const DoubleProduct& p, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>((p.m + kTile - 1) / kTile),
                  static_cast<unsigned>(std::min<int64_t>((p.n + kTile - 1) / kTile, 65535)));
  double_product_kernel<<<grid, 256, 0, stream>>>(p);
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
  if (need > 0 && !aligned16(workspace)) {
    return fail(CND_ERR_WORKSPACE, "%s: workspace must be 16-byte aligned", who);
  }
  return CND_OK;
}

}  // namespace
}  // namespace layers
}  // namespace cnd

extern "C" {

size_t cnd_linear_forward_workspace_size(const cnd_linear* problem) {
  using namespace cnd::layers;
  if (check_linear("cnd_linear_forward", problem) != CND_OK || problem->rows == 0) return 0;
  return forward_layout(*problem).total;
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
  if (!aligned_to(element_size(problem->dtype), {x, weight, bias, residual, y, pre})) {
    return misaligned("cnd_linear_forward");
  }
  const cnd_linear& q = *problem;
  const int64_t rows = q.rows, in = q.in_features, out = q.out_features;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  if (q.dtype == CND_F64) {
    DoubleProduct p{};
    p.a = static_cast<const double*>(x);
    p.b = static_cast<const double*>(weight);
    p.bias = static_cast<const double*>(bias);
    p.residual = static_cast<const double*>(residual);
    p.d = static_cast<double*>(y);
    p.pre = static_cast<double*>(pre);
    p.m = rows;
    p.n = out;
    p.k = in;
    p.a_row = q.x_stride;
    p.b_row = in;
    p.a_col = p.b_col = 1;
    p.act = q.activation;
    launch_double(p, stream);
    return launch_status("cnd_linear_forward");
  }
  if (!aligned16(x) || !aligned16(weight)) {
    return fail(CND_ERR_INVALID, "cnd_linear_forward: x and weight must be 16-byte aligned");
  }
  const Layout l = forward_layout(q);
  rc = check_workspace("cnd_linear_forward", workspace, workspace_bytes, l.total);
  if (rc != CND_OK) return rc;
  char* base = static_cast<char*>(workspace);
  Product p{};
  p.a = operand_at(x, rows, q.x_stride, true);
  p.b = operand_at(weight, out, in, true);
  if (copies_x(q)) {
    prepare(q.dtype, x, nullptr, CND_ACT_NONE, rows, in, q.x_stride, base + l.x, row_pitch(in), nullptr,
            stream);
    p.a = operand_at(base + l.x, rows, row_pitch(in), true);
  }
  if (copies_w(q)) {
    prepare(q.dtype, weight, nullptr, CND_ACT_NONE, out, in, in, base + l.w, row_pitch(in), nullptr,
            stream);
    p.b = operand_at(base + l.w, out, row_pitch(in), true);
  }
  p.m = rows;
  p.n = out;
  p.k = in;
  p.parts = parts_of(q);
  p.bf16 = q.dtype != CND_F16;
  p.dtype = q.dtype;
  p.d = y;
  p.pre = pre;
  p.bias = bias;
  p.residual = residual;
  p.act = q.activation;
  return launch_product(p, plan_product(rows, out, in, p.parts), base + l.splits, stream);
}

size_t cnd_linear_backward_workspace_size(const cnd_linear* problem,
                                          const int32_t output_mask[3]) {
  using namespace cnd::layers;
  if (check_linear("cnd_linear_backward", problem) != CND_OK || output_mask == nullptr ||
      problem->rows == 0) {
    return 0;
  }
  return backward_layout(*problem, output_mask).total;
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
  const bool want_x = output_mask[0], want_w = output_mask[1], want_b = output_mask[2];
  if (!want_x && !want_w && !want_b) return CND_OK;
  const cnd_linear& q = *problem;
  const int64_t rows = q.rows, in = q.in_features, out = q.out_features;
  const bool act = q.activation != CND_ACT_NONE;
  if ((want_w && dweight == nullptr) || (want_b && dbias == nullptr) ||
      (rows > 0 && (dy == nullptr || (act && pre == nullptr) ||
                    (want_x && (dx == nullptr || weight == nullptr)) ||
                    (want_w && x == nullptr)))) {
    return fail(CND_ERR_INVALID, "cnd_linear_backward: a required buffer is NULL");
  }
  if (!aligned_to(element_size(q.dtype), {dy, pre, x, weight, dx, dweight, dbias})) {
    return misaligned("cnd_linear_backward");
  }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  if (rows == 0) {
    const size_t size = element_size(q.dtype);
    if (want_w) cudaMemsetAsync(dweight, 0, static_cast<size_t>(out) * in * size, stream);
    if (want_b) cudaMemsetAsync(dbias, 0, static_cast<size_t>(out) * size, stream);
    return launch_status("cnd_linear_backward");
  }
  if (q.dtype != CND_F64 && (!aligned16(dy) || !aligned16(pre) || (want_w && !aligned16(x)) ||
                             (want_x && (!aligned16(weight) || !aligned16(dx))))) {
    return fail(CND_ERR_INVALID,
                "cnd_linear_backward: dy, pre, x, weight and dx must be 16-byte aligned");
  }
  const Layout l = backward_layout(q, output_mask);
  rc = check_workspace("cnd_linear_backward", workspace, workspace_bytes, l.total);
  if (rc != CND_OK) return rc;
  char* base = static_cast<char*>(workspace);
  if (one_pass(q, output_mask)) {
    ThinBackward t{};
    t.dtype = q.dtype;
    t.act = q.activation;
    t.rows = rows;
    t.n = out;
    t.k = in;
    t.x_stride = q.x_stride;
    t.dy = dy;
    t.z = pre;
    t.x = x;
    t.w = weight;
    t.dx = dx;
    t.dw = reinterpret_cast<float*>(base + l.splits);
    t.db = want_b ? reinterpret_cast<float*>(base + l.sums) : nullptr;
    rc = launch_thin_backward(t, stream);
    if (rc != CND_OK) return rc;
    Product p{};
    p.m = out;
    p.n = in;
    p.dtype = q.dtype;
    p.d = dweight;
    join_partials(p, t.dw, thin_blocks(rows), out * in, in, stream);
    if (want_b) join_columns(q.dtype, t.db, thin_blocks(rows), out, dbias, stream);
    return launch_status("cnd_linear_backward");
  }
  const bool copy = q.dtype == CND_F64 ? act : (want_x || want_w) && copies_dz(q);
  const int64_t pitch = q.dtype == CND_F64 ? out : row_pitch(out);
  if (copy || want_b) {
    prepare(q.dtype, dy, act ? pre : nullptr, q.activation, rows, out, out,
            copy ? base + l.dz : nullptr, pitch, want_b ? base + l.sums : nullptr, stream);
  }
  if (want_b) {
    join_columns(q.dtype, base + l.sums, prepare_ranges(rows, out), out, dbias, stream);
  }
  if (q.dtype == CND_F64) {
    DoubleProduct p{};
    p.a = copy ? reinterpret_cast<const double*>(base + l.dz) : static_cast<const double*>(dy);
    if (want_x) {
      p.b = static_cast<const double*>(weight);
      p.d = static_cast<double*>(dx);
      p.m = rows;
      p.n = in;
      p.k = out;
      p.a_row = out;
      p.a_col = 1;
      p.b_row = 1;
      p.b_col = in;
      launch_double(p, stream);
    }
    if (want_w) {
      p.b = static_cast<const double*>(x);
      p.d = static_cast<double*>(dweight);
      p.m = out;
      p.n = in;
      p.k = rows;
      p.a_row = 1;
      p.a_col = out;
      p.b_row = 1;
      p.b_col = q.x_stride;
      launch_double(p, stream);
    }
    return launch_status("cnd_linear_backward");
  }
  const Operand dz = copy ? operand_at(base + l.dz, rows, pitch, true)
                          : operand_at(dy, rows, out, true);
  Product p{};
  p.parts = parts_of(q);
  p.bf16 = q.dtype != CND_F16;
  p.dtype = q.dtype;
  if (want_x) {
    p.a = dz;
    p.b = operand_at(weight, out, in, false);
    if (copies_w(q)) {
      prepare(q.dtype, weight, nullptr, CND_ACT_NONE, out, in, in, base + l.w, row_pitch(in), nullptr,
              stream);
      p.b = operand_at(base + l.w, out, row_pitch(in), false);
    }
    p.m = rows;
    p.n = in;
    p.k = out;
    p.d = dx;
    rc = launch_product(p, plan_product(p.m, p.n, p.k, p.parts), base + l.splits, stream);
    if (rc != CND_OK) return rc;
  }
  if (want_w) {
    p.a = dz;
    p.a.k_major = false;
    p.b = operand_at(x, rows, q.x_stride, false);
    if (copies_x(q)) {
      prepare(q.dtype, x, nullptr, CND_ACT_NONE, rows, in, q.x_stride, base + l.x, row_pitch(in),
              nullptr, stream);
      p.b = operand_at(base + l.x, rows, row_pitch(in), false);
    }
    p.m = out;
    p.n = in;
    p.k = rows;
    p.d = dweight;
    rc = launch_product(p, plan_product(p.m, p.n, p.k, p.parts), base + l.splits, stream);
    if (rc != CND_OK) return rc;
  }
  return launch_status("cnd_linear_backward");
}

}  // extern "C"
