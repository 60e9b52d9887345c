// Gated linear recurrence along the middle axis of [outer][steps][inner]:
//
//   f_t = sigmoid(g_t),  h_t = f_t h_{t-1} + (1 - f_t) x_t;
//   G_t = dy_t + f_{t+1} G_{t+1},  dx_t = (1 - f_t) G_t,
//   dg_t = f_t (1 - f_t) (h_{t-1} - x_t) G_t,  dh_{-1} = f_0 G_0.
//
// One thread per column walks the steps. The forward keeps the state before each block of
// kBlockSteps steps, from which the backward recomputes the others in float32, so it reads
// x, g and dy only and its h carry no rounding to the tensors' type.
#include <algorithm>

#include "layers.cuh"

namespace cnd {
namespace layers {
namespace {

constexpr int kBlockSteps = 16;
constexpr int kThreads = 128;

struct RecurrenceArgs {
  const void *x, *gate, *initial, *dy, *dlast, *states_in;
  void *y, *last, *states, *dx, *dgate, *dinitial;
  int64_t outer, steps, inner;
};

// f = sigmoid(g) and 1 - f, each to full relative accuracy (exact 0 and 1 at +-inf).
template <typename A>
__device__ __forceinline__ void gates(A g, A* f, A* keep) {
  const A e = exp(-fabs(g));
  const A r = A(1) / (A(1) + e);
  *f = g >= A(0) ? r : e * r;
  *keep = g >= A(0) ? e * r : r;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) recurrence_forward_kernel(const RecurrenceArgs a) {
  using A = typename Wide<T>::type;
  const int64_t columns = a.outer * a.inner;
  const int64_t column = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (column >= columns) return;
  const int64_t base = column / a.inner * a.steps * a.inner + column % a.inner;
  const T* x = static_cast<const T*>(a.x) + base;
  const T* gate = static_cast<const T*>(a.gate) + base;
  T* y = static_cast<T*>(a.y) + base;
  A h = a.initial != nullptr ? static_cast<const A*>(a.initial)[column] : A(0);
  for (int64_t t = 0; t < a.steps; ++t) {
    if (a.states != nullptr && t % kBlockSteps == 0) {
      static_cast<A*>(a.states)[t / kBlockSteps * columns + column] = h;
    }
    A f, keep;
    gates<A>(widen(gate[t * a.inner]), &f, &keep);
    h = f * h + keep * widen(x[t * a.inner]);
    y[t * a.inner] = narrow<T>(h);
  }
  static_cast<A*>(a.last)[column] = h;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) recurrence_backward_kernel(const RecurrenceArgs a) {
  using A = typename Wide<T>::type;
  const int64_t columns = a.outer * a.inner;
  const int64_t column = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (column >= columns) return;
  const int64_t base = column / a.inner * a.steps * a.inner + column % a.inner;
  const T* x = static_cast<const T*>(a.x) + base;
  const T* gate = static_cast<const T*>(a.gate) + base;
  const T* dy = a.dy != nullptr ? static_cast<const T*>(a.dy) + base : nullptr;
  A flow = a.dlast != nullptr ? static_cast<const A*>(a.dlast)[column] : A(0);
  for (int64_t block = (a.steps - 1) / kBlockSteps; block >= 0; --block) {
    const int64_t first = block * kBlockSteps;
    const int count = static_cast<int>(a.steps - first < kBlockSteps ? a.steps - first : kBlockSteps);
    A before[kBlockSteps];
    A h = static_cast<const A*>(a.states_in)[block * columns + column];
    for (int i = 0; i < count; ++i) {
      before[i] = h;
      A f, keep;
      gates<A>(widen(gate[(first + i) * a.inner]), &f, &keep);
      h = f * h + keep * widen(x[(first + i) * a.inner]);
    }
    for (int i = count - 1; i >= 0; --i) {
      const int64_t at = (first + i) * a.inner;
      A f, keep;
      gates<A>(widen(gate[at]), &f, &keep);
      const A total = flow + (dy != nullptr ? widen(dy[at]) : A(0));
      if (a.dx != nullptr) static_cast<T*>(a.dx)[base + at] = narrow<T>(keep * total);
      if (a.dgate != nullptr) {
        static_cast<T*>(a.dgate)[base + at] =
            narrow<T>(f * keep * (before[i] - widen(x[at])) * total);
      }
      flow = f * total;
    }
  }
  if (a.dinitial != nullptr) static_cast<A*>(a.dinitial)[column] = flow;
}

int check_recurrence(const char* who, int dtype, int64_t outer, int64_t steps, int64_t inner) {
  if (!known_dtype(dtype)) return fail(CND_ERR_UNSUPPORTED, "%s: unknown dtype %d", who, dtype);
  if (outer < 0 || steps < 0 || inner < 0) {
    return fail(CND_ERR_INVALID, "%s: sizes must be nonnegative", who);
  }
  const int64_t columns = product(outer, inner);
  if (columns < 0 || product(columns, std::max<int64_t>(steps, 1)) < 0) {
    return fail(CND_ERR_INVALID, "%s: size overflows int64", who);
  }
  return CND_OK;
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

}  // namespace
}  // namespace layers
}  // namespace cnd

extern "C" {

int64_t cnd_gated_recurrence_blocks(int32_t dtype, int64_t outer, int64_t steps, int64_t inner) {
  (void)dtype;
  (void)outer;
  (void)inner;
  return steps <= 0 ? 0 : (steps - 1) / cnd::layers::kBlockSteps + 1;
}

size_t cnd_gated_recurrence_workspace_size(int32_t dtype, int64_t outer, int64_t steps,
                                           int64_t inner) {
  (void)dtype;
  (void)outer;
  (void)steps;
  (void)inner;
  return 0;
}

int cnd_gated_recurrence_forward(int32_t dtype, int64_t outer, int64_t steps, int64_t inner,
                                 const void* x, const void* gate, const void* initial, void* y,
                                 void* last, void* states, void* workspace,
                                 size_t workspace_bytes, void* stream_handle) {
  using namespace cnd;
  using namespace cnd::layers;
  (void)workspace;
  (void)workspace_bytes;
  clear_error();
  const int rc = check_recurrence("cnd_gated_recurrence_forward", dtype, outer, steps, inner);
  if (rc != CND_OK) return rc;
  const int64_t columns = outer * inner;
  if (columns == 0) return CND_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  if (last == nullptr || (steps > 0 && (x == nullptr || gate == nullptr || y == nullptr))) {
    return fail(CND_ERR_INVALID, "cnd_gated_recurrence_forward: a required buffer is NULL");
  }
  RecurrenceArgs a{};
  a.x = x;
  a.gate = gate;
  a.initial = initial;
  a.y = y;
  a.last = last;
  a.states = states;
  a.outer = outer;
  a.steps = steps;
  a.inner = inner;
  with_dtype(dtype, [&](auto zero) {
    recurrence_forward_kernel<decltype(zero)>
        <<<static_cast<unsigned>((columns + kThreads - 1) / kThreads), kThreads, 0, stream>>>(a);
  });
  count_launch();
  return launch_status("cnd_gated_recurrence_forward");
}

int cnd_gated_recurrence_backward(int32_t dtype, int64_t outer, int64_t steps, int64_t inner,
                                  const void* dy, const void* dlast, const void* x,
                                  const void* gate, const void* states, void* dx, void* dgate,
                                  void* dinitial, const int32_t output_mask[3], void* workspace,
                                  size_t workspace_bytes, void* stream_handle) {
  using namespace cnd;
  using namespace cnd::layers;
  (void)workspace;
  (void)workspace_bytes;
  clear_error();
  const int rc = check_recurrence("cnd_gated_recurrence_backward", dtype, outer, steps, inner);
  if (rc != CND_OK) return rc;
  if (output_mask == nullptr) {
    return fail(CND_ERR_INVALID, "cnd_gated_recurrence_backward: output_mask must not be NULL");
  }
  const int64_t columns = outer * inner;
  if (columns == 0 || (!output_mask[0] && !output_mask[1] && !output_mask[2])) return CND_OK;
  if ((output_mask[2] && dinitial == nullptr) ||
      (steps > 0 && (x == nullptr || gate == nullptr || states == nullptr ||
                     (output_mask[0] && dx == nullptr) || (output_mask[1] && dgate == nullptr)))) {
    return fail(CND_ERR_INVALID, "cnd_gated_recurrence_backward: a required buffer is NULL");
  }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  RecurrenceArgs a{};
  a.x = x;
  a.gate = gate;
  a.dy = dy;
  a.dlast = dlast;
  a.states_in = states;
  a.dx = output_mask[0] ? dx : nullptr;
  a.dgate = output_mask[1] ? dgate : nullptr;
  a.dinitial = output_mask[2] ? dinitial : nullptr;
  a.outer = outer;
  a.steps = steps;
  a.inner = inner;
  with_dtype(dtype, [&](auto zero) {
    recurrence_backward_kernel<decltype(zero)>
        <<<static_cast<unsigned>((columns + kThreads - 1) / kThreads), kThreads, 0, stream>>>(a);
  });
  count_launch();
  return launch_status("cnd_gated_recurrence_backward");
}

}  // extern "C"
