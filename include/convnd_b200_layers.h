/*
 * convnd_b200_layers.h — C ABI of the layers that stand around the convolutions: layer norm,
 * linear layers with a fused epilogue, and the gated linear recurrence.
 *
 * Conventions are those of convnd_b200.h: device pointers and sizes only, a caller-provided
 * workspace, a cudaStream_t as void* (NULL = legacy default stream), CND_OK or a negative
 * status with the message in cnd_last_error(). Every call only enqueues work on `stream`.
 * Every output is written in full. Buffers are aligned to their elements, a workspace to 16 bytes
 * (what is not is refused). None of these operators has a counterpart in the
 * reference.
 */
#ifndef CONVND_B200_LAYERS_H
#define CONVND_B200_LAYERS_H

#include "convnd_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- layer norm ------------------------------------------------------------------------
 * Over rows of `width` elements, in float32 (float64 for CND_F64):
 *   mean = sum(x) / width, rstd = 1 / sqrt(sum((x - mean)^2) / width + eps),
 *   y = (x - mean) * rstd * weight + bias.
 * x and dy rows start x_stride / dy_stride elements apart (>= width); y and dx are dense.
 * eps >= 0. weight and bias ([width], either may be NULL) have type param_dtype: `dtype`, or
 * CND_F32.
 * stats receives mean and rstd per row ([2][rows] float32, float64 for CND_F64; NULL in
 * cnd_layer_norm_forward when no backward follows).
 * The backward fills the gradients selected by output_mask = {dx, dweight, dbias}:
 *   g = dy * weight, u = (x - mean) * rstd,
 *   dx = rstd * (g - mean(g) - u * mean(g * u)), dweight = sum(dy * u), dbias = sum(dy).
 * Column sums have a fixed order: repeated calls give the same bits. */
CND_API int cnd_layer_norm_forward(int32_t dtype, int32_t param_dtype, int64_t rows,
                                   int64_t width, int64_t x_stride, double eps, const void* x,
                                   const void* weight, const void* bias, void* y, void* stats,
                                   void* stream);
CND_API size_t cnd_layer_norm_backward_workspace_size(int32_t dtype, int64_t rows, int64_t width,
                                                      const int32_t output_mask[3]);
CND_API int cnd_layer_norm_backward(int32_t dtype, int32_t param_dtype, int64_t rows,
                                    int64_t width, int64_t dy_stride, int64_t x_stride,
                                    const void* dy, const void* x, const void* weight,
                                    const void* stats, void* dx, void* dweight, void* dbias,
                                    const int32_t output_mask[3], void* workspace,
                                    size_t workspace_bytes, void* stream);

/* ---- linear layer with bias, activation and residual in its epilogue --------------------
 * z = x W^T + bias, y = act(z) + residual. x: [rows, in_features] with rows x_stride elements
 * apart; W: [out_features, in_features]; bias: [out_features] or NULL; residual and y:
 * [rows, out_features], residual may be NULL; everything of `dtype`, dense but for x.
 * 16-bit products accumulate in float32; float32 operands are split into three bfloat16
 * terms each and the six products above 2^-24 are summed (float32 accuracy; a non-finite
 * operand gives a non-finite result, but an infinity may come out as NaN); float64 runs on
 * the CUDA cores. cnd_linear_forward writes z to `pre` (same shape and type as y) when it is
 * not NULL; the backward of an activation needs it. Both z and the dz below are rounded to
 * `dtype` there. x, weight, dy, pre and dx are 16-byte
 * aligned (float64: their natural alignment):
 *   dz = dy * act'(z), dx = dz W, dW = dz^T x, dbias = column sums of dz
 * (the residual's gradient is dy itself). `pre` may be NULL for CND_ACT_NONE. The
 * gradients selected by output_mask = {dx, dW, dbias} are written; dy is dense. */
#define CND_ACT_SILU 2 /* v / (1 + exp(-v)); beside CND_ACT_NONE and CND_ACT_GELU */

typedef struct cnd_linear {
  int32_t dtype;      /* cnd_dtype */
  int32_t activation; /* CND_ACT_* */
  int64_t rows;
  int64_t in_features;
  int64_t out_features;
  int64_t x_stride; /* elements between rows of x, >= in_features */
} cnd_linear;

CND_API size_t cnd_linear_forward_workspace_size(const cnd_linear* problem);
CND_API int cnd_linear_forward(const cnd_linear* problem, const void* x, const void* weight,
                               const void* bias, const void* residual, void* y, void* pre,
                               void* workspace, size_t workspace_bytes, void* stream);
CND_API size_t cnd_linear_backward_workspace_size(const cnd_linear* problem,
                                                  const int32_t output_mask[3]);
CND_API int cnd_linear_backward(const cnd_linear* problem, const void* dy, const void* pre,
                                const void* x, const void* weight, void* dx, void* dweight,
                                void* dbias, const int32_t output_mask[3], void* workspace,
                                size_t workspace_bytes, void* stream);

/* ---- gated linear recurrence -----------------------------------------------------------
 * Along the middle axis of dense [outer][steps][inner] tensors x, gate, y of `dtype`:
 *   f_t = sigmoid(gate_t), h_t = f_t * h_{t-1} + (1 - f_t) * x_t, y_t = h_t,
 * with h_{-1} = initial ([outer][inner] float32, float64 for CND_F64; NULL = zeros) and
 * last = h_{steps-1} of the same type and shape. States are held in float32 (float64). A
 * gate of -inf restarts a column (h_t = x_t, h_{t-1} finite), +inf holds it (h_t = h_{t-1}, x_t
 * finite); what is not finite stays, as 0 * inf is NaN.
 * `states` (NULL when no backward follows) receives the states before each block of steps,
 * [cnd_gated_recurrence_blocks()][outer][inner]; the backward recomputes the others.
 * Backward, with dy ([outer][steps][inner], NULL = zeros) and dlast ([outer][inner], NULL =
 * zeros): G_t = dy_t + f_{t+1} G_{t+1} (the last step adds dlast),
 *   dx_t = (1 - f_t) G_t, dgate_t = f_t (1 - f_t) (h_{t-1} - x_t) G_t, dinitial = f_0 G_0.
 * Gradients selected by output_mask = {dx, dgate, dinitial} are written. */
CND_API int64_t cnd_gated_recurrence_blocks(int32_t dtype, int64_t outer, int64_t steps,
                                            int64_t inner);
CND_API size_t cnd_gated_recurrence_workspace_size(int32_t dtype, int64_t outer, int64_t steps,
                                                   int64_t inner);
CND_API int cnd_gated_recurrence_forward(int32_t dtype, int64_t outer, int64_t steps,
                                         int64_t inner, const void* x, const void* gate,
                                         const void* initial, void* y, void* last, void* states,
                                         void* workspace, size_t workspace_bytes, void* stream);
CND_API int cnd_gated_recurrence_backward(int32_t dtype, int64_t outer, int64_t steps,
                                          int64_t inner, const void* dy, const void* dlast,
                                          const void* x, const void* gate, const void* states,
                                          void* dx, void* dgate, void* dinitial,
                                          const int32_t output_mask[3], void* workspace,
                                          size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* CONVND_B200_LAYERS_H */
