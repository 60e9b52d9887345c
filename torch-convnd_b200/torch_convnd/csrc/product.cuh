// Matrix products on the tensor cores for the linear layers: D[m][n] = sum_k A(m, k) B(n, k)
// with bias, activation, pre-activation output and residual in the epilogue.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace cnd {
namespace layers {

// One 16-bit operand in device memory. K-major: element (row, k) of part p at
// p * plane + row * pitch + k; else at p * plane + k * pitch + row. The base is 16-byte
// aligned, pitch and plane are multiples of 8 elements.
struct Operand {
  const void* data;
  int64_t pitch, plane;
  bool k_major;
};

struct Product {
  Operand a, b;
  int64_t m, n, k;
  int parts;    // 1, or 3: float32 operands as three bfloat16 terms each
  bool bf16;    // operand type: bfloat16, else float16
  int dtype;    // type of d, pre, bias and residual (CND_F16, CND_BF16, CND_F32)
  void* d;      // [m][n]
  void* pre;    // [m][n] pre-activation or NULL
  const void* bias;
  const void* residual;
  int act;
};

// How a product is cut: CTA pairs or single CTAs, tile width, splits of the k axis, epilogue
// groups.
struct ProductPlan {
  int pair, bn, splits, groups;
};

ProductPlan plan_product(int64_t m, int64_t n, int64_t k, int parts);

// float32 partial sums of a split product, [splits][m][round up n to 4]; 0 without splits.
size_t product_workspace(const ProductPlan& plan, int64_t m, int64_t n);

// Adds `splits` float32 partial results [m][pitch], `stride` elements apart, in order and applies
// the epilogue of `p`.
void join_partials(const Product& p, const float* partials, int splits, int64_t stride,
                   int64_t pitch, cudaStream_t stream);

// Tensor map of a [rows][n] matrix, rows `pitch` elements apart: boxes of 128 bytes by box_rows
// rows with the 128-byte swizzle.
bool encode_matrix(CUtensorMap* map, void* d, int dtype, int64_t rows, int64_t n, int64_t pitch,
                   int box_rows);

// The one-pass backward of a 16-bit layer with an activation, up to kThinIn input and kThinOut
// output features (thin.cu). All addresses and rows are whole 16-byte units.
constexpr int kThinIn = 64, kThinOut = 256;

struct ThinBackward {
  int dtype, act;
  int64_t rows, n, k, x_stride;  // n output features, k input features
  const void *dy, *z, *x, *w;
  void* dx;
  float* dw;  // partial sums [thin_blocks()][n][k]
  float* db;  // partial sums [thin_blocks()][n], or NULL
};

int thin_blocks(int64_t rows);
int launch_thin_backward(const ThinBackward& p, cudaStream_t stream);

int launch_product(const Product& p, const ProductPlan& plan, void* workspace, cudaStream_t stream);

}  // namespace layers
}  // namespace cnd
