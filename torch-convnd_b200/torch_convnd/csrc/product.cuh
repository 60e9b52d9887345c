// Matrix products on the tensor cores for the linear layers: D[m][n] = sum_k A(m, k) B(n, k)
// with bias, activation, pre-activation output and residual in the epilogue.
#pragma once

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

int launch_product(const Product& p, const ProductPlan& plan, void* workspace, cudaStream_t stream);

}  // namespace layers
}  // namespace cnd
