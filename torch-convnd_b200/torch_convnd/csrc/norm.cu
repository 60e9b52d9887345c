// Layer norm over rows: forward, and the backward pass with the weight's and bias's
// gradients.
//
//   mean = sum(x) / C,  rstd = 1 / sqrt(sum((x - mean)^2) / C + eps),  u = (x - mean) rstd,
//   y = u w + b;
//   g = dy w,  dx = rstd (g - mean(g) - u mean(g u)),  dw = sum(dy u),  db = sum(dy).
//
// A row is held in registers or shared memory between its two sums (the squares are of centred
// values, so a large mean costs no digits), so every element is read once: both passes are
// bound by memory traffic, 2 and 3 elements per position. bf16 forward / backward: 1M x 64 in
// 58 / 92 us (4.6 / 4.4 TB/s), 16384 x 4096 in 52 / 85 us (5.2 / 4.7), of 6.55 TB/s copied.
// A row belongs to G lanes of a warp or to a block of G threads; a block walks rows with a
// grid stride, each thread always holding the same columns, so the weight's gradient
// accumulates in registers, is combined once per block and leaves as one partial row per
// block, summed in order by a second launch. Rows that are back to back come through a ring
// of bulk copies, whole rows of more than 64 vectors and tiles of shorter ones; rows that
// bulk copies cannot take stay in registers. Rows wider than 28 KB and float64 are walked
// in chunks, element by element, and read again for each pass: 8192 x 8192 float32 134 / 299 us,
// 4.0 and 2.7 TB/s of what one reading would move.
#include <algorithm>

#include "layers.cuh"
#include "pair.cuh"

namespace cnd {
namespace layers {

int sm_count() {
  int device = 0, count = 0;
  if (cudaGetDevice(&device) != cudaSuccess ||
      cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device) != cudaSuccess ||
      count <= 0) {
    cudaGetLastError();
    return kSms;
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
  int shift;  // rows shifted against 16-byte boundaries (ring and tile kernels)
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

// R sums at once: the same for every one, with one pair of block barriers.
template <int G, int R>
__device__ __forceinline__ void group_sums(float (&v)[R], float (*scratch)[32]) {
#pragma unroll
  for (int d = (G < 32 ? G : 32) / 2; d > 0; d /= 2) {
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] += __shfl_xor_sync(0xffffffffu, v[r], d);
  }
  if constexpr (G > 32) {
    constexpr int kWarps = G / 32;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int r = 0; r < R; ++r) scratch[r][threadIdx.x >> 5] = v[r];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      v[r] = scratch[r][threadIdx.x & (kWarps - 1)];
#pragma unroll
      for (int d = kWarps / 2; d > 0; d /= 2) v[r] += __shfl_xor_sync(0xffffffffu, v[r], d);
    }
    __syncthreads();
  }
}

// A thread's parameters, in float32 registers for all its rows: `absent` where there are none.
template <typename T, int V, int NV, int G>
__device__ __forceinline__ void load_params(const void* p, bool is_f32, int64_t width, int lane,
                                            float absent, float (&v)[NV][V]) {
#pragma unroll
  for (int k = 0; k < NV; ++k) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (k * G + lane) * V + i;
      v[k][i] = p != nullptr && c < width ? load_param<T>(p, is_f32, c) : absent;
    }
  }
}

// Block size of the register kernels: 256 threads, or one row's when it takes more than a warp.
template <int G>
constexpr int block_size() {
  return G > 32 ? G : 256;
}

__device__ __forceinline__ float both(Two v) {
  float lo, hi;
  unpack(v, &lo, &hi);
  return lo + hi;
}

// The arithmetic of a row's thread on vectors of V elements, two at a time: one instruction a
// pair where scalar code had the schedulers issuing more than half of the time.
template <typename T, int V, int NV, int G>
struct RowMath {
  static constexpr int kPairs = V / 2;

  static __device__ __forceinline__ float sum(const Two (&x)[kPairs]) {
    Two s = x[0];
#pragma unroll
    for (int i = 1; i < kPairs; ++i) s = add2(s, x[i]);
    return both(s);
  }
  static __device__ __forceinline__ float squares(const Two (&x)[kPairs], float mean) {
    Two s = same(0.0f);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const Two d = add2(x[i], same(-mean));
      s = fma2(d, d, s);
    }
    return both(s);
  }
  static __device__ __forceinline__ void normalise(Two (&x)[kPairs], float mean, float rstd,
                                                   const Two (&w)[kPairs], const Two (&b)[kPairs]) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      x[i] = fma2(mul2(add2(x[i], same(-mean)), same(rstd)), w[i], b[i]);
    }
  }
  // sums += (g, g u); dw += dy u, db += dy
  static __device__ __forceinline__ void collect(const Two (&x)[kPairs], const Two (&dy)[kPairs],
                                                 float mean, float rstd, const Two (&w)[kPairs],
                                                 Two (&sums)[2], Two (&dw)[kPairs],
                                                 Two (&db)[kPairs]) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const Two u = mul2(add2(x[i], same(-mean)), same(rstd));
      const Two g = mul2(dy[i], w[i]);
      sums[0] = add2(sums[0], g);
      sums[1] = fma2(g, u, sums[1]);
      dw[i] = fma2(dy[i], u, dw[i]);
      db[i] = add2(db[i], dy[i]);
    }
  }
  // dy becomes rstd (g - mean_g - u mean_gu)
  static __device__ __forceinline__ void gradient(const Two (&x)[kPairs], Two (&dy)[kPairs],
                                                  float mean, float rstd, const Two (&w)[kPairs],
                                                  float mean_g, float mean_gu) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const Two u = mul2(add2(x[i], same(-mean)), same(rstd));
      const Two t = fma2(dy[i], w[i], same(-mean_g));
      dy[i] = mul2(fma2(u, same(-mean_gu), t), same(rstd));
    }
  }
};

// Writes a block's column sums, held by groups of G <= 32 lanes, as one partial row: rows of
// one warp first (lanes of the same columns), then the warps in order. `columns`: [2][width].
template <typename T, int V, int NV, int G>
__device__ __forceinline__ void block_columns(const NormArgs& a, float (&dw)[NV][V],
                                              float (&db)[NV][V], float* columns) {
  const int lane = threadIdx.x % G;
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
  for (int w = 0; w < static_cast<int>(blockDim.x) / 32; ++w) {
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
  float* partial = static_cast<float*>(a.partials) + static_cast<int64_t>(blockIdx.x) * 2 * a.width;
  for (int64_t c = threadIdx.x; c < 2 * a.width; c += blockDim.x) partial[c] = columns[c];
}

// R rows of a group are in flight at once: their loads are issued before the first is summed,
// and their sums share the reductions' latency.
template <typename T, int V, int NV, int G, int R>
__global__ void __launch_bounds__(block_size<G>())
    norm_forward_kernel(const NormArgs a) {
  constexpr int kRows = block_size<G>() / G;
  __shared__ float scratch[R][32];
  const int lane = threadIdx.x % G;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows * R;
  const float inverse = 1.0f / static_cast<float>(a.width);
  float w[NV][V], b[NV][V];
  load_params<T, V, NV, G>(a.weight, a.param_f32, a.width, lane, 1.0f, w);
  load_params<T, V, NV, G>(a.bias, a.param_f32, a.width, lane, 0.0f, b);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows * R; base < a.rows; base += step) {
    const int64_t row0 = base + threadIdx.x / G;
    Pack<T, V> raw[R][NV];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = row0 + r * kRows;
      const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * G + lane) * V;
        if (row < a.rows && c < a.width) raw[r][k] = *reinterpret_cast<const Pack<T, V>*>(x + c);
      }
    }
    float mean[R], squares[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = squares[r] = 0.0f;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if ((k * G + lane) * V < a.width) {
#pragma unroll
          for (int i = 0; i < V; ++i) mean[r] += widen(raw[r][k].v[i]);
        }
      }
    }
    group_sums<G, R>(mean, scratch);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] *= inverse;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if ((k * G + lane) * V < a.width) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float d = widen(raw[r][k].v[i]) - mean[r];
            squares[r] += d * d;
          }
        }
      }
    }
    group_sums<G, R>(squares, scratch);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = row0 + r * kRows;
      if (row >= a.rows) continue;
      const float rstd = rsqrtf(squares[r] * inverse + static_cast<float>(a.eps));
      if (a.stats != nullptr && lane == 0) {
        static_cast<float*>(a.stats)[row] = mean[r];
        static_cast<float*>(a.stats)[a.rows + row] = rstd;
      }
      T* y = static_cast<T*>(a.y) + row * a.width;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * G + lane) * V;
        if (c < a.width) {
          Pack<T, V> out;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            out.v[i] = narrow<T>((widen(raw[r][k].v[i]) - mean[r]) * rstd * w[k][i] + b[k][i]);
          }
          *reinterpret_cast<Pack<T, V>*>(y + c) = out;
        }
      }
    }
  }
}

template <typename T, int V, int NV, int G, int R>
__global__ void __launch_bounds__(block_size<G>())
    norm_backward_kernel(const NormArgs a) {
  constexpr int kThreads = block_size<G>();
  constexpr int kRows = kThreads / G;
  extern __shared__ float columns[];  // [2][width], only when kRows > 1
  __shared__ float scratch[2 * R][32];
  const int lane = threadIdx.x % G;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows * R;
  const float inverse = 1.0f / static_cast<float>(a.width);
  const float* means = static_cast<const float*>(a.stats);
  float w[NV][V], dw[NV][V], db[NV][V];
  load_params<T, V, NV, G>(a.weight, a.param_f32, a.width, lane, 1.0f, w);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
#pragma unroll
    for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = 0.0f;
  }
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows * R; base < a.rows; base += step) {
    const int64_t row0 = base + threadIdx.x / G;
    Pack<T, V> rx[R][NV], rd[R][NV];
    float mean[R], rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = row0 + r * kRows;
      const bool live = row < a.rows;
      const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
      const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
      mean[r] = live ? means[row] : 0.0f;
      rstd[r] = live ? means[a.rows + row] : 0.0f;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * G + lane) * V;
        if (live && c < a.width) {
          rx[r][k] = *reinterpret_cast<const Pack<T, V>*>(x + c);
          rd[r][k] = *reinterpret_cast<const Pack<T, V>*>(dy + c);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) rx[r][k].v[i] = rd[r][k].v[i] = narrow<T>(0.0f);
        }
      }
    }
    float sums[2 * R];
#pragma unroll
    for (int r = 0; r < 2 * R; ++r) sums[r] = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = widen(rd[r][k].v[i]);
          const float u = (widen(rx[r][k].v[i]) - mean[r]) * rstd[r];
          const float g = d * w[k][i];
          sums[2 * r] += g;
          sums[2 * r + 1] += g * u;
          dw[k][i] += d * u;
          db[k][i] += d;
        }
      }
    }
    if (!a.want_dx) continue;
    group_sums<G, 2 * R>(sums, scratch);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = row0 + r * kRows;
      if (row >= a.rows) continue;
      const float mean_g = sums[2 * r] * inverse, mean_gu = sums[2 * r + 1] * inverse;
      T* dx = static_cast<T*>(a.y) + row * a.width;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * G + lane) * V;
        if (c < a.width) {
          Pack<T, V> out;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float d = widen(rd[r][k].v[i]);
            const float u = (widen(rx[r][k].v[i]) - mean[r]) * rstd[r];
            out.v[i] = narrow<T>(rstd[r] * (d * w[k][i] - mean_g - u * mean_gu));
          }
          *reinterpret_cast<Pack<T, V>*>(dx + c) = out;
        }
      }
    }
  }
  if (!a.want_params) return;
  if constexpr (kRows > 1) {
    block_columns<T, V, NV, G>(a, dw, db, columns);
  } else {
    float* partial = static_cast<float*>(a.partials) + static_cast<int64_t>(blockIdx.x) * 2 * a.width;
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

// ---- rows in vectors from shared memory ---------------------------------------------------
//
// Rows of any width and 16-byte vectors: row r of dense rows starts at element r * width,
// off a 16-byte boundary by (r * width) % V elements. A thread whose rows are all congruent
// modulo V (8 for 16 bits, 4 for float32) meets one such shift, so it can read aligned
// vectors with columns, parameters and column sums fixed in registers as if its rows began
// `shift` elements earlier; the first and the last vector of a row are masked. (Single
// elements took 171 + 217 us for 65536 x 1001 bf16.)

// A thread's vector: columns c ... c + V - 1 of which [lo, hi) exist. Without shifts (kShift)
// a vector exists or does not.
template <int V, bool kShift>
struct Span {
  int c, lo, hi;
  bool exists;
  __device__ __forceinline__ Span(int vector, int shift, int width) {
    c = vector * V - (kShift ? shift : 0);
    lo = kShift && c < 0 ? -c : 0;
    hi = kShift && width - c < V ? width - c : V;
    exists = kShift ? lo < hi : c < width;
  }
  __device__ __forceinline__ bool whole() const { return !kShift || (lo == 0 && hi == V); }
  __device__ __forceinline__ bool any() const { return exists; }
  // Whether column c + i exists (of a span that may not).
  __device__ __forceinline__ bool has(int i) const {
    return kShift ? i >= lo && i < hi : exists;
  }
};

template <typename T, int V, bool kShift>
__device__ __forceinline__ void store_span(T* row, const Span<V, kShift>& s, const Two (&v)[V / 2]) {
  if (s.whole()) {
    store_twos<T, V>(row + s.c, v);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      float lo, hi;
      unpack(v[i / 2], &lo, &hi);
      if (s.has(i)) row[s.c + i] = narrow<T>(lo);
      if (s.has(i + 1)) row[s.c + i + 1] = narrow<T>(hi);
    }
  }
}

// Values outside a span become `value`.
template <int V, bool kShift>
__device__ __forceinline__ void fill_outside(const Span<V, kShift>& s, float value, Two (&v)[V / 2]) {
#pragma unroll
  for (int i = 0; i < V; i += 2) {
    float lo, hi;
    unpack(v[i / 2], &lo, &hi);
    v[i / 2] = two(s.has(i) ? lo : value, s.has(i + 1) ? hi : value);
  }
}

template <typename T, int V, bool kShift>
__device__ __forceinline__ void load_span_params(const void* p, bool is_f32,
                                                 const Span<V, kShift>& s,
                                                 float absent, Two (&v)[V / 2]) {
  float f[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    f[i] = p != nullptr && s.has(i) ? load_param<T>(p, is_f32, s.c + i) : absent;
  }
#pragma unroll
  for (int i = 0; i < V / 2; ++i) v[i] = two(f[2 * i], f[2 * i + 1]);
}

// Elements between the 16-byte boundary before a row and the row.
template <int V>
__device__ __forceinline__ int row_shift(int64_t row, int64_t stride) {
  return static_cast<int>(row % V * (stride % V) % V);
}

// Adds a span's column sums to `to` ([2][width]), or starts them.
template <int V, bool kShift>
__device__ __forceinline__ void add_span(const Span<V, kShift>& s, const Two (&dw)[V / 2],
                                         const Two (&db)[V / 2], float* to, int width, bool first) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float w2[2], b2[2];
    unpack(dw[i / 2], &w2[0], &w2[1]);
    unpack(db[i / 2], &b2[0], &b2[1]);
    if (s.has(i)) {
      const int c = s.c + i;
      to[c] = first ? w2[i % 2] : to[c] + w2[i % 2];
      to[width + c] = first ? b2[i % 2] : to[width + c] + b2[i % 2];
    }
  }
}

// Blocks an SM of the ring kernels: 768 threads of 80 registers, 512 where the masks of shifted
// rows take more.
constexpr int ring_blocks_of(int threads, bool shift) {
  return threads >= 512 ? 1 : (shift ? 512 : 768) / threads;
}

// A block of G threads walks rows that bulk copies bring into a ring of stages ahead of it (x,
// and dy behind it in the backward), so the loads in flight depend neither on registers
// nor on the block's barriers: holding 16 KB rows in registers had left the memory system at
// 2.8 TB/s. A stage is refilled after the first barrier by which every thread has finished
// with its row. The backward takes two rows at a time, so that their four sums share one pair of
// barriers (84 us against 94 for 16384 x 4096 bf16), and reads them again from shared memory
// for its second pass; the forward, with two reductions a row but fewer registers, is faster
// row by row (53 us against 61). Short rows that lie back to back come by the tile, whose rows the
// block's warps share, with one barrier a tile.
struct Ring {
  int stages, tile;  // stages; rows of a stage
  uint32_t stage_bytes;  // the backward's second half holds dy
  unsigned int* error;
  uint64_t timeout_ns;
};

constexpr uint32_t kSiteRing = 0x701, kSiteRingDrain = 0x702;

template <bool kBackward, bool kShift>
struct RowRing {
  const NormArgs& a;
  const Ring& ring;
  uint8_t* data;
  uint64_t* full;
  int64_t next;  // the next row to ask for (thread 0)
  int fill = 0, stage = 0;
  uint32_t phase = 0;
  bool dead = false;

  // One operand's part of a stage: the 16-byte blocks that hold rows next ... next + count - 1
  // (they lie back to back where a stage holds several), but none past the tensor's end: what
  // the last rows have beyond the last whole block is stored element by element. Returns
  // the bytes that the copy will bring.
  __device__ __forceinline__ uint32_t bring(uint8_t* dst, const void* base, int64_t stride, int es,
                                            int count, bool copy) {
    const int64_t begin = next * stride * es, end = begin + ((count - 1) * stride + a.width) * es;
    const int64_t first = begin & ~int64_t{15};
    const int64_t limit = ((a.rows - 1) * stride + a.width) * es;
    int64_t last = (end + 15) & ~int64_t{15};
    if (last > limit) last = limit & ~int64_t{15};
    if (last < first) last = first;
    const char* src = static_cast<const char*>(base);
    if (!copy) {
      for (int64_t at = last; at < end; at += 2) {
        *reinterpret_cast<uint16_t*>(dst + (at - first)) = *reinterpret_cast<const uint16_t*>(src + at);
      }
    } else if (last > first) {
      dev::bulk_load(dst, src + first, static_cast<uint32_t>(last - first), &full[fill]);
    }
    return static_cast<uint32_t>(last - first);
  }

  __device__ __forceinline__ void ask(int es) {
    // thread 0: rows `next` ... into stage `fill`
    if (next >= a.rows || dead) return;
    const int64_t left = a.rows - next;
    const int count = left < ring.tile ? static_cast<int>(left) : ring.tile;
    uint8_t* dst = data + fill * ring.stage_bytes;
    uint8_t* second = dst + ring.stage_bytes / 2;
    if constexpr (!kShift) {
      const uint32_t whole = static_cast<uint32_t>(count) * static_cast<uint32_t>(a.width) * es;
      dev::mbar_arrive_expect_tx(&full[fill], kBackward ? 2 * whole : whole);
      dev::bulk_load(dst, static_cast<const char*>(a.x) + next * a.x_stride * es, whole, &full[fill]);
      if (kBackward) {
        dev::bulk_load(second, static_cast<const char*>(a.dy) + next * a.dy_stride * es, whole,
                       &full[fill]);
      }
      next += static_cast<int64_t>(gridDim.x) * ring.tile;
      if (++fill == ring.stages) fill = 0;
      return;
    }
    uint32_t bytes = bring(dst, a.x, a.x_stride, es, count, false);
    if (kBackward) bytes += bring(second, a.dy, a.dy_stride, es, count, false);
    dev::mbar_arrive_expect_tx(&full[fill], bytes);
    bring(dst, a.x, a.x_stride, es, count, true);
    if (kBackward) bring(second, a.dy, a.dy_stride, es, count, true);
    next += static_cast<int64_t>(gridDim.x) * ring.tile;
    if (++fill == ring.stages) fill = 0;
  }

  // Waits for the current stage. After a wait that expired no other one waits or asks, and the
  // copies on their way are drained: here (kHere), as the tile kernels do it, or behind the
  // last row. Which one only decides what registers the compiler finds for the loop: 65536 x
  // 512 bf16 by the tile 31 us here and 43 behind it, 16384 x 4096 row by row 58 and 54.
  template <bool kHere>
  __device__ __forceinline__ const uint8_t* wait() {
    if (!dead && !dev::mbar_wait(&full[stage], phase, dev::ErrorWord{ring.error}, kSiteRing,
                                 ring.timeout_ns)) {
      dead = true;
      if (kHere) drain();
    }
    return data + stage * ring.stage_bytes;
  }

  __device__ __forceinline__ void advance() {
    if (++stage == ring.stages) {
      stage = 0;
      phase ^= 1u;
    }
  }

  // After a wait that expired: thread 0 gives the copies that it asked for a bounded time to land
  // before the block may exit. Of a barrier's two phases the one in progress ends when its copy has
  // landed, the other has ended; both are waited for, as the walk does not keep which is which.
  __device__ __forceinline__ void drain() {
    if (!dead || threadIdx.x != 0) return;
#pragma unroll 1
    for (uint32_t i = 0; i < 2u * ring.stages; ++i) {
      dev::mbar_wait(&full[i / 2], i & 1u, dev::ErrorWord{ring.error}, kSiteRingDrain,
                     ring.timeout_ns / 16 + 1);
    }
  }
};

template <typename T, int V, int NV, int G, bool kShift>
__global__ void __launch_bounds__(G, ring_blocks_of(G, kShift))
    norm_forward_ring_kernel(const __grid_constant__ NormArgs a, const __grid_constant__ Ring ring_args) {
  extern __shared__ __align__(128) uint8_t shared[];
  __shared__ float scratch[1][32];
  __shared__ uint64_t full[16];
  const int lane = threadIdx.x;
  const float inverse = 1.0f / static_cast<float>(a.width);
  if (lane == 0) {
    for (int s = 0; s < ring_args.stages; ++s) dev::mbar_init(&full[s], 1);
    dev::fence_barrier_init();
  }
  __syncthreads();
  RowRing<false, kShift> ring{a, ring_args, shared, full, blockIdx.x};
  if (lane == 0) {
    for (int s = 0; s < ring_args.stages; ++s) ring.ask(sizeof(T));
  }
  using M = RowMath<T, V, NV, G>;
  Two w[NV][V / 2], b[NV][V / 2];
  const int width = static_cast<int>(a.width);
  const int shift = row_shift<V>(blockIdx.x, a.x_stride);  // the same for all the block's rows
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const Span<V, kShift> s(k * G + lane, shift, width);
    load_span_params<T>(a.weight, a.param_f32, s, 1.0f, w[k]);
    load_span_params<T>(a.bias, a.param_f32, s, 0.0f, b[k]);
  }
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* data = reinterpret_cast<const T*>(ring.template wait<false>());
    Two x[NV][V / 2];
    float sum[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const Span<V, kShift> s(k * G + lane, shift, width);
      if (s.any()) {
        load_twos<T, V>(data + (k * G + lane) * V, x[k]);
        if (!s.whole()) fill_outside(s, 0.0f, x[k]);
        sum[0] += M::sum(x[k]);
      }
    }
    group_sums<G, 1>(sum, scratch);
    // every thread has passed the previous row: its stage is free
    if (lane == 0 && row != blockIdx.x) ring.ask(sizeof(T));
    const float mean = sum[0] * inverse;
    float squares[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const Span<V, kShift> s(k * G + lane, shift, width);
      if (s.any()) {
        if (!s.whole()) fill_outside(s, mean, x[k]);
        squares[0] += M::squares(x[k], mean);
      }
    }
    group_sums<G, 1>(squares, scratch);
    const float rstd = rsqrtf(squares[0] * inverse + static_cast<float>(a.eps));
    if (a.stats != nullptr && lane == 0) {
      static_cast<float*>(a.stats)[row] = mean;
      static_cast<float*>(a.stats)[a.rows + row] = rstd;
    }
    T* y = static_cast<T*>(a.y) + row * width;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const Span<V, kShift> s(k * G + lane, shift, width);
      if (s.any()) {
        M::normalise(x[k], mean, rstd, w[k], b[k]);
        store_span<T>(y, s, x[k]);
      }
    }
    ring.advance();
  }
  ring.drain();
}

template <typename T, int V, int NV, int G, bool kShift>
__global__ void __launch_bounds__(G, ring_blocks_of(G, kShift))
    norm_backward_ring_kernel(const __grid_constant__ NormArgs a, const __grid_constant__ Ring ring_args) {
  extern __shared__ __align__(128) uint8_t shared[];
  __shared__ float scratch[4][32];
  __shared__ uint64_t full[16];
  const int lane = threadIdx.x;
  const float inverse = 1.0f / static_cast<float>(a.width);
  const float* means = static_cast<const float*>(a.stats);
  if (lane == 0) {
    for (int s = 0; s < ring_args.stages; ++s) dev::mbar_init(&full[s], 1);
    dev::fence_barrier_init();
  }
  __syncthreads();
  RowRing<true, kShift> ring{a, ring_args, shared, full, blockIdx.x};
  if (lane == 0) {
    for (int s = 0; s < ring_args.stages; ++s) ring.ask(sizeof(T));
  }
  using M = RowMath<T, V, NV, G>;
  const int width = static_cast<int>(a.width);
  const int shift = row_shift<V>(blockIdx.x, a.x_stride);  // the same for all the block's rows
  Two w[NV][V / 2], dw[NV][V / 2], db[NV][V / 2];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    load_span_params<T>(a.weight, a.param_f32, Span<V, kShift>(k * G + lane, shift, width), 1.0f, w[k]);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) dw[k][i] = db[k][i] = same(0.0f);
  }
  // Two rows at a time: their sums share the reductions' barriers. The statistics of the next
  // two are fetched ahead.
  const int64_t step = gridDim.x;
  float2 ahead[2];
  const auto fetch = [&](int64_t row0) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t row = row0 + r * step;
      if (row < a.rows) ahead[r] = make_float2(means[row], means[a.rows + row]);
    }
  };
  fetch(blockIdx.x);
  for (int64_t row0 = blockIdx.x; row0 < a.rows; row0 += 2 * step) {
    const float2 stats[2] = {ahead[0], ahead[1]};
    fetch(row0 + 2 * step);
    const uint8_t* at[2];
    float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (row0 + r * step < a.rows) {
        at[r] = ring.template wait<false>();
        ring.advance();
        Two pairs[2] = {same(0.0f), same(0.0f)};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const Span<V, kShift> s(k * G + lane, shift, width);
          if (s.any()) {
            Two x[V / 2], dy[V / 2];
            load_twos<T, V>(reinterpret_cast<const T*>(at[r]) + (k * G + lane) * V, x);
            load_twos<T, V>(reinterpret_cast<const T*>(at[r] + ring_args.stage_bytes / 2) + (k * G + lane) * V, dy);
            if (!s.whole()) {  // nothing is collected outside the row
              fill_outside(s, 0.0f, x);
              fill_outside(s, 0.0f, dy);
            }
            M::collect(x, dy, stats[r].x, stats[r].y, w[k], pairs, dw[k], db[k]);
          }
        }
        sums[2 * r] = both(pairs[0]);
        sums[2 * r + 1] = both(pairs[1]);
      }
    }
    group_sums<G, 4>(sums, scratch);
    // every thread has finished with the two rows before these: their stages are free
    if (lane == 0 && row0 != blockIdx.x) {
      ring.ask(sizeof(T));
      ring.ask(sizeof(T));
    }
    if (!a.want_dx) continue;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t row = row0 + r * step;
      if (row >= a.rows) break;
      T* dx = static_cast<T*>(a.y) + row * width;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const Span<V, kShift> s(k * G + lane, shift, width);
        if (s.any()) {
          Two x[V / 2], dy[V / 2];
          load_twos<T, V>(reinterpret_cast<const T*>(at[r]) + (k * G + lane) * V, x);
          load_twos<T, V>(reinterpret_cast<const T*>(at[r] + ring_args.stage_bytes / 2) + (k * G + lane) * V, dy);
          M::gradient(x, dy, stats[r].x, stats[r].y, w[k], sums[2 * r] * inverse,
                      sums[2 * r + 1] * inverse);
          store_span<T>(dx, s, dy);
        }
      }
    }
  }
  ring.drain();
  if (!a.want_params) return;
  float* partial = static_cast<float*>(a.partials) + static_cast<int64_t>(blockIdx.x) * 2 * width;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    add_span(Span<V, kShift>(k * G + lane, shift, width), dw[k], db[k], partial, width, true);
  }
}

// Short rows in tiles: G lanes of a warp to a row, as in the register kernels.
constexpr int tile_blocks_of(int vectors, bool shift, bool backward) {
  return backward ? (vectors == 1 && !shift ? 3 : 2) : (vectors == 1 && !shift ? 4 : 3);
}
constexpr int kTileThreads = 256, kMostTile = 256;

template <typename T, int V, int NV, int G, bool kShift>
__global__ void __launch_bounds__(kTileThreads, tile_blocks_of(NV, kShift, false))
    norm_forward_tile_kernel(const __grid_constant__ NormArgs a, const __grid_constant__ Ring ring_args) {
  constexpr int kGroups = kTileThreads / G;
  extern __shared__ __align__(128) uint8_t shared[];
  __shared__ uint64_t full[16];
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  const int width = static_cast<int>(a.width), tile = ring_args.tile;
  const float inverse = 1.0f / static_cast<float>(width);
  if (threadIdx.x == 0) {
    for (int s = 0; s < ring_args.stages; ++s) dev::mbar_init(&full[s], 1);
    dev::fence_barrier_init();
  }
  __syncthreads();
  RowRing<false, kShift> ring{a, ring_args, shared, full, static_cast<int64_t>(blockIdx.x) * tile};
  if (threadIdx.x == 0) {
    for (int s = 0; s < ring_args.stages; ++s) ring.ask(sizeof(T));
  }
  using M = RowMath<T, V, NV, G>;
  Two w[NV][V / 2], b[NV][V / 2];
  const int shift = row_shift<V>(group, width);  // tiles and steps are multiples of V rows
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const Span<V, kShift> s(k * G + lane, shift, width);
    load_span_params<T>(a.weight, a.param_f32, s, 1.0f, w[k]);
    load_span_params<T>(a.bias, a.param_f32, s, 0.0f, b[k]);
  }
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * tile; row0 < a.rows;
       row0 += static_cast<int64_t>(gridDim.x) * tile) {
    const T* data = reinterpret_cast<const T*>(ring.template wait<true>());
#pragma unroll 2
    for (int i0 = 0; i0 < tile; i0 += kGroups) {
      const int64_t row = row0 + i0 + group;
      const bool live = i0 + group < tile && row < a.rows;
      Two x[NV][V / 2];
      float mean = 0.0f, squares = 0.0f;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const Span<V, kShift> s(k * G + lane, shift, width);
        if (live && s.any()) {
          load_twos<T, V>(data + (i0 + group) * width + s.c, x[k]);
          if (!s.whole()) fill_outside(s, 0.0f, x[k]);
          mean += M::sum(x[k]);
        }
      }
      mean = group_sum<G, float>(mean, nullptr) * inverse;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const Span<V, kShift> s(k * G + lane, shift, width);
        if (live && s.any()) {
          if (!s.whole()) fill_outside(s, mean, x[k]);
          squares += M::squares(x[k], mean);
        }
      }
      squares = group_sum<G, float>(squares, nullptr);
      if (!live) continue;
      const float rstd = rsqrtf(squares * inverse + static_cast<float>(a.eps));
      if (a.stats != nullptr && lane == 0) {
        static_cast<float*>(a.stats)[row] = mean;
        static_cast<float*>(a.stats)[a.rows + row] = rstd;
      }
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const Span<V, kShift> s(k * G + lane, shift, width);
        if (s.any()) {
          M::normalise(x[k], mean, rstd, w[k], b[k]);
          store_span<T>(static_cast<T*>(a.y) + row * width, s, x[k]);
        }
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) ring.ask(sizeof(T));
    ring.advance();
  }
}

template <typename T, int V, int NV, int G, bool kShift>
__global__ void __launch_bounds__(kTileThreads, tile_blocks_of(NV, kShift, true))
    norm_backward_tile_kernel(const __grid_constant__ NormArgs a, const __grid_constant__ Ring ring_args) {
  constexpr int kGroups = kTileThreads / G;
  extern __shared__ __align__(128) uint8_t shared[];
  __shared__ uint64_t full[16];
  __shared__ float2 stats[2][kMostTile];  // of this tile and the next
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  const int width = static_cast<int>(a.width), tile = ring_args.tile;
  const float inverse = 1.0f / static_cast<float>(width);
  const float* means = static_cast<const float*>(a.stats);
  const auto fetch = [&](int64_t row0, int slot) {
    const int64_t row = row0 + threadIdx.x;
    if (static_cast<int>(threadIdx.x) < tile && row < a.rows) {
      stats[slot][threadIdx.x] = make_float2(means[row], means[a.rows + row]);
    }
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < ring_args.stages; ++s) dev::mbar_init(&full[s], 1);
    dev::fence_barrier_init();
  }
  fetch(static_cast<int64_t>(blockIdx.x) * tile, 0);
  __syncthreads();
  RowRing<true, kShift> ring{a, ring_args, shared, full, static_cast<int64_t>(blockIdx.x) * tile};
  if (threadIdx.x == 0) {
    for (int s = 0; s < ring_args.stages; ++s) ring.ask(sizeof(T));
  }
  using M = RowMath<T, V, NV, G>;
  Two w[NV][V / 2], dw[NV][V / 2], db[NV][V / 2];
  const int shift = row_shift<V>(group, width);  // tiles and steps are multiples of V rows
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    load_span_params<T>(a.weight, a.param_f32, Span<V, kShift>(k * G + lane, shift, width), 1.0f, w[k]);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) dw[k][i] = db[k][i] = same(0.0f);
  }
  int slot = 0;
  const int64_t step = static_cast<int64_t>(gridDim.x) * tile;
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * tile; row0 < a.rows; row0 += step) {
    fetch(row0 + step, slot ^ 1);
    const uint8_t* at = ring.template wait<true>();
    const T* xs = reinterpret_cast<const T*>(at);
    const T* ds = reinterpret_cast<const T*>(at + ring_args.stage_bytes / 2);
#pragma unroll 2
    for (int i0 = 0; i0 < tile; i0 += kGroups) {
      const int64_t row = row0 + i0 + group;
      const bool live = i0 + group < tile && row < a.rows;
      const float2 st = live ? stats[slot][i0 + group] : make_float2(0.0f, 0.0f);
      Two x[NV][V / 2], dy[NV][V / 2];
      Two pairs[2] = {same(0.0f), same(0.0f)};
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const Span<V, kShift> s(k * G + lane, shift, width);
        if (live && s.any()) {
          load_twos<T, V>(xs + (i0 + group) * width + s.c, x[k]);
          load_twos<T, V>(ds + (i0 + group) * width + s.c, dy[k]);
          if (!s.whole()) {  // nothing is collected outside the row
            fill_outside(s, 0.0f, x[k]);
            fill_outside(s, 0.0f, dy[k]);
          }
          M::collect(x[k], dy[k], st.x, st.y, w[k], pairs, dw[k], db[k]);
        }
      }
      if (!a.want_dx) continue;
      float sums[2] = {both(pairs[0]), both(pairs[1])};
      group_sums<G, 2>(sums, nullptr);
      if (!live) continue;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const Span<V, kShift> s(k * G + lane, shift, width);
        if (s.any()) {
          M::gradient(x[k], dy[k], st.x, st.y, w[k], sums[0] * inverse, sums[1] * inverse);
          store_span<T>(static_cast<T*>(a.y) + row * width, s, dy[k]);
        }
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) ring.ask(sizeof(T));
    ring.advance();
    slot ^= 1;
  }
  if (!a.want_params) return;
  __syncthreads();
  float* columns = reinterpret_cast<float*>(shared);
  if constexpr (kShift) {
    // the groups' columns are offset against one another, so they add theirs one by one
    for (int g = 0; g < kGroups; ++g) {
      if (group == g) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          add_span(Span<V, kShift>(k * G + lane, shift, width), dw[k], db[k], columns, width, g == 0);
        }
      }
      __syncthreads();
    }
    float* partial = static_cast<float*>(a.partials) + static_cast<int64_t>(blockIdx.x) * 2 * width;
    for (int c = threadIdx.x; c < 2 * width; c += kTileThreads) partial[c] = columns[c];
  } else {
    float wide_dw[NV][V], wide_db[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        unpack(dw[k][i], &wide_dw[k][2 * i], &wide_dw[k][2 * i + 1]);
        unpack(db[k][i], &wide_db[k][2 * i], &wide_db[k][2 * i + 1]);
      }
    }
    block_columns<T, V, NV, G>(a, wide_dw, wide_db, columns);
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

// Partial rows [blocks][2][width] summed in order: a block takes 32 columns, its 32 warps
// contiguous ranges of the rows, and the range sums are added in range order.
constexpr int kReduceWarps = 32;
template <typename T>
__global__ void __launch_bounds__(kReduceWarps * 32)
    norm_reduce_kernel(const void* partials, int blocks, int64_t width, void* dweight,
                       void* dbias, int param_f32) {
  using A = typename Wide<T>::type;
  __shared__ A part[kReduceWarps][32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  A sum = 0;
  if (j < 2 * width) {
    const A* p = static_cast<const A*>(partials) + j;
    const int last = blocks * (warp + 1) / kReduceWarps;
#pragma unroll 8
    for (int b = blocks * warp / kReduceWarps; b < last; ++b) sum += p[static_cast<int64_t>(b) * 2 * width];
  }
  part[warp][lane] = sum;
  __syncthreads();
  if (warp != 0 || j >= 2 * width) return;
  for (int w = 1; w < kReduceWarps; ++w) sum += part[w][lane];
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
  bool loops;   // wider than the block kernels (or float64)
  bool shift;   // dense rows of another width, read in vectors from shifted starts
  bool ring;    // more than 64 vectors a row
};

// Four stages of two such rows (28 KB each) fit the ring of the backward.
constexpr int kMostChunks = 1792;

// aligned: data on 16-byte boundaries; whole: rows a multiple of 16 bytes apart; dense: rows
// back to back.
NormShape norm_shape(int dtype, int64_t width, bool aligned, bool whole, bool dense) {
  NormShape s{};
  const int wide = 16 / element_size(dtype);
  s.shift = aligned && dense && width % wide != 0 && width > 2 * wide && dtype != CND_F64 &&
            (width + 2 * wide - 2) / wide <= kMostChunks;
  if (s.shift) {
    s.vector = wide;
    s.chunks = static_cast<int>((width + 2 * wide - 2) / wide);
    s.ring = s.chunks > 64;
    return s;
  }
  s.vector = aligned && whole && width % wide == 0 ? wide : 1;
  s.loops = dtype == CND_F64 || width / s.vector > kMostChunks;
  s.chunks = s.loops ? 0 : static_cast<int>(width / s.vector);
  s.ring = s.vector > 1 && s.chunks > 64;
  return s;
}

int ring_threads(int chunks) {
  return chunks <= 128 ? 64 : chunks <= 256 ? 128 : chunks <= 512 ? 256 : chunks <= 1024 ? 512 : 1024;
}
int ring_blocks(const NormShape& s) { return ring_blocks_of(ring_threads(s.chunks), s.shift); }

int norm_rows_per_block(const NormShape& s) {
  if (s.chunks <= 4) return 64;
  if (s.chunks <= 8) return 32;
  if (s.chunks <= 16) return 16;
  return s.chunks <= 64 ? 8 : 1;
}

// Short rows back to back, in vectors, come by the tile; others (rows apart from one another,
// single elements) are held in registers as they are loaded. bf16, forward / backward, registers
// against tiles: 1M x 64 76 / 109 us and 56 / 98, 65536 x 512 64 / 99 and 31 / 64,
// 65536 x 64 11.5 / 26 and 8 / 19; the same from 1 to 1024 rows.
bool norm_tiles(const NormShape& s, int64_t width, int64_t x_stride, int64_t dy_stride) {
  return !s.loops && !s.ring && s.vector > 1 && x_stride == width && dy_stride == width;
}

// Blocks of the backward (one partial row each): enough to fill the SMs, no more than rows.
int norm_backward_blocks(const NormShape& s, int64_t rows, int64_t width) {
  if (s.loops) {
    // column kernel: row ranges of at least 64 rows
    const int64_t most = std::max<int64_t>(1, rows / 64);
    const int64_t across = (width + 127) / 128;
    return static_cast<int>(std::min<int64_t>(most, std::max<int64_t>(1, 8 * kSms / across)));
  }
  if (s.ring) {
    // a multiple of 8 where blocks take several rows: one shift a block
    return static_cast<int>(std::min<int64_t>(rows, kSms * ring_blocks(s) / 8 * 8));
  }
  const int per_block = norm_rows_per_block(s);
  const int64_t need = (rows + per_block - 1) / per_block;
  return static_cast<int>(std::min<int64_t>(need, 4 * kSms));
}

// Vectors a thread, threads a row, rows in flight.
template <bool kBackward, typename T, int V, typename F>
void with_shape(const NormShape& s, F&& f) {
  constexpr int kThin = kBackward ? 2 : 4;
  if (s.chunks <= 4) {
    f.template operator()<T, V, 1, 4, kThin>();
  } else if (s.chunks <= 8) {
    f.template operator()<T, V, 1, 8, kThin>();
  } else if (s.chunks <= 16) {
    f.template operator()<T, V, 1, 16, kThin>();
  } else if (s.chunks <= 32) {
    f.template operator()<T, V, 1, 32, kThin>();
  } else if (V > 1 || s.chunks <= 64) {
    f.template operator()<T, V, 2, 32, 2>();
  } else if constexpr (V == 1) {  // longer rows of vectors run on the ring kernels
    if (s.chunks <= 128) {
      f.template operator()<T, V, 2, 64, 2>();
    } else if (s.chunks <= 256) {
      f.template operator()<T, V, 2, 128, 2>();
    } else if (s.chunks <= 512) {
      f.template operator()<T, V, 2, 256, 2>();
    } else if (s.chunks <= 1024) {
      f.template operator()<T, V, 2, 512, 2>();
    } else {
      f.template operator()<T, V, 2, 1024, 2>();
    }
  }
}

template <bool kBackward, typename F>
void with_kernel(int dtype, const NormShape& s, F&& f) {
  if (dtype == CND_F32) {
    s.vector == 1 ? with_shape<kBackward, float, 1>(s, f) : with_shape<kBackward, float, 4>(s, f);
  } else if (dtype == CND_BF16) {
    s.vector == 1 ? with_shape<kBackward, __nv_bfloat16, 1>(s, f) : with_shape<kBackward, __nv_bfloat16, 8>(s, f);
  } else {
    s.vector == 1 ? with_shape<kBackward, __half, 1>(s, f) : with_shape<kBackward, __half, 8>(s, f);
  }
}

// Blocks an SM of the tile kernels.
int tile_blocks(const NormShape& s, bool backward) {
  return tile_blocks_of(s.chunks <= 32 ? 1 : 2, s.shift, backward);
}

// The ring of a block: its share of 200 KB, at most 16 stages but four at least. Tiles of short
// rows are 8 KB.
constexpr int kRingTotal = 200 * 1024;
// The most that any call of a tile kernel (two blocks an SM and more) and of a ring kernel (four
// stages of two rows) takes. A kernel's limit is set to this in every call, not to what the call
// takes: another thread's call may come between setting the limit and the launch.
constexpr int kTileShared = kRingTotal / 2, kRingShared = 4 * 2 * kMostChunks * 16;
static_assert(kRingShared >= kRingTotal);
Ring make_ring(const NormShape& s, int dtype, int64_t width, bool backward) {
  Ring r{};
  if (s.ring) {
    r.tile = 1;
    r.stage_bytes = static_cast<uint32_t>(s.chunks) * 16;
  } else {
    // whole multiples of 8 rows; a vector before and behind for the masked ends
    const uint32_t row = static_cast<uint32_t>(width) * element_size(dtype);
    r.tile = static_cast<int>(std::max<uint32_t>(8, std::min<uint32_t>(kMostTile, 8192 / row / 8 * 8)));
    r.stage_bytes = (row * r.tile + 31) / 16 * 16;
  }
  if (backward) r.stage_bytes *= 2;
  const uint32_t share = kRingTotal / (s.ring ? ring_blocks(s) : tile_blocks(s, backward));
  r.stages = static_cast<int>(std::min<uint32_t>(16, std::max<uint32_t>(4, share / r.stage_bytes)));
  r.error = device_error_word();
  r.timeout_ns = wait_timeout_ns();
  return r;
}

template <typename T, int V, typename F>
void with_ring(const NormShape& s, F&& f) {
  switch (ring_threads(s.chunks)) {
    case 64:
      return f.template operator()<T, V, 2, 64>();
    case 128:
      return f.template operator()<T, V, 2, 128>();
    case 256:
      return f.template operator()<T, V, 2, 256>();
    case 512:
      return f.template operator()<T, V, 2, 512>();
    default:
      return f.template operator()<T, V, 2, 1024>();
  }
}

template <typename F>
void with_ring_dtype(int dtype, const NormShape& s, F&& f) {
  if (dtype == CND_F32) {
    with_ring<float, 4>(s, f);
  } else if (dtype == CND_BF16) {
    with_ring<__nv_bfloat16, 8>(s, f);
  } else {
    with_ring<__half, 8>(s, f);
  }
}

template <bool kBackward>
struct LaunchTile {
  const NormArgs& a;
  const Ring& ring;
  int blocks;
  cudaStream_t stream;
  // R (rows in flight) is the register kernels': a tile kernel's are in its ring
  template <typename T, int V, int NV, int G, int R>
  void operator()() const {
    if constexpr (V > 1 && G <= 32) {
      const auto kernel = a.shift ? (kBackward ? norm_backward_tile_kernel<T, V, NV, G, true>
                                               : norm_forward_tile_kernel<T, V, NV, G, true>)
                                  : (kBackward ? norm_backward_tile_kernel<T, V, NV, G, false>
                                               : norm_forward_tile_kernel<T, V, NV, G, false>);
      const uint32_t bytes = std::max<uint32_t>(ring.stage_bytes * ring.stages,
                                                static_cast<uint32_t>(a.width) * 2 * sizeof(float));
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTileShared);
      kernel<<<blocks, kTileThreads, bytes, stream>>>(a, ring);
    }
  }
};

template <bool kBackward>
struct LaunchRing {
  const NormArgs& a;
  const Ring& ring;
  int blocks;
  cudaStream_t stream;
  template <typename T, int V, int NV, int G>
  void operator()() const {
    const auto kernel = a.shift ? (kBackward ? norm_backward_ring_kernel<T, V, NV, G, true>
                                             : norm_forward_ring_kernel<T, V, NV, G, true>)
                                : (kBackward ? norm_backward_ring_kernel<T, V, NV, G, false>
                                             : norm_forward_ring_kernel<T, V, NV, G, false>);
    const uint32_t bytes = ring.stage_bytes * ring.stages;
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingShared);
    kernel<<<blocks, G, bytes, stream>>>(a, ring);
  }
};

struct LaunchForward {
  const NormArgs& a;
  cudaStream_t stream;
  template <typename T, int V, int NV, int G, int R>
  void operator()() const {
    constexpr int kRows = block_size<G>() / G * R;
    const int64_t need = (a.rows + kRows - 1) / kRows;
    const int64_t most = static_cast<int64_t>(sm_count()) * (2048 / block_size<G>()) * 4;
    norm_forward_kernel<T, V, NV, G, R>
        <<<static_cast<unsigned>(std::min(need, most)), block_size<G>(), 0, stream>>>(a);
  }
};

struct LaunchBackward {
  const NormArgs& a;
  int blocks;
  cudaStream_t stream;
  template <typename T, int V, int NV, int G, int R>
  void operator()() const {
    constexpr int kRows = block_size<G>() / G;
    const size_t shared = kRows > 1 ? static_cast<size_t>(a.width) * 2 * sizeof(float) : 0;
    norm_backward_kernel<T, V, NV, G, R><<<blocks, block_size<G>(), shared, stream>>>(a);
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

bool rows_whole(int dtype, int64_t stride) { return stride * element_size(dtype) % 16 == 0; }

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
  if (!(eps >= 0)) return fail(CND_ERR_INVALID, "cnd_layer_norm_forward: eps must be nonnegative");
  if (rows == 0) return CND_OK;
  if (x == nullptr || y == nullptr) {
    return fail(CND_ERR_INVALID, "cnd_layer_norm_forward: x and y must not be NULL");
  }
  if (!aligned_to(element_size(dtype), {x, y}) ||
      !aligned_to(element_size(param_dtype), {weight, bias}) || !aligned_to(wide_size(dtype), {stats})) {
    return misaligned("cnd_layer_norm_forward");
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
  const NormShape s = norm_shape(dtype, width, aligned16(x) && aligned16(y),
                                 rows_whole(dtype, x_stride), x_stride == width);
  a.shift = s.shift;
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
  } else if (s.ring) {
    const Ring ring = make_ring(s, dtype, width, false);
    if (ring.error == nullptr) return fail(CND_ERR_CUDA, "device error word unavailable");
    const int blocks =
        static_cast<int>(std::min<int64_t>(rows, sm_count() * ring_blocks(s) / 8 * 8));
    with_ring_dtype(dtype, s, LaunchRing<false>{a, ring, blocks, stream});
  } else if (norm_tiles(s, width, x_stride, width)) {
    const Ring ring = make_ring(s, dtype, width, false);
    if (ring.error == nullptr) return fail(CND_ERR_CUDA, "device error word unavailable");
    const int64_t tiles = (rows + ring.tile - 1) / ring.tile;
    const int blocks =
        static_cast<int>(std::min<int64_t>(tiles, sm_count() * tile_blocks(s, false)));
    with_kernel<false>(dtype, s, LaunchTile<false>{a, ring, blocks, stream});
  } else {
    with_kernel<false>(dtype, s, LaunchForward{a, stream});
  }
  count_launch();
  return launch_status("cnd_layer_norm_forward");
}

size_t cnd_layer_norm_backward_workspace_size(int32_t dtype, int64_t rows, int64_t width,
                                              const int32_t output_mask[3]) {
  using namespace cnd::layers;
  if (!known_dtype(dtype) || rows <= 0 || width <= 0 || output_mask == nullptr) return 0;
  if (!output_mask[1] && !output_mask[2]) return 0;
  // the largest of what the data's alignment can lead to
  int blocks = 0;
  for (int kind = 0; kind < 8; ++kind) {
    const NormShape s = norm_shape(dtype, width, (kind & 1) != 0, (kind & 2) != 0, (kind & 4) != 0);
    blocks = std::max(blocks, norm_backward_blocks(s, rows, width));
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
  if (!aligned_to(element_size(dtype), {dy, x, dx}) ||
      !aligned_to(element_size(param_dtype), {weight, dweight, dbias}) ||
      !aligned_to(wide_size(dtype), {stats})) {
    return misaligned("cnd_layer_norm_backward");
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
  if (need > 0 && !aligned16(workspace)) {
    return fail(CND_ERR_WORKSPACE, "cnd_layer_norm_backward: workspace must be 16-byte aligned");
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
  const NormShape s =
      norm_shape(dtype, width, aligned16(x) && aligned16(dy) && (!a.want_dx || aligned16(dx)),
                 rows_whole(dtype, x_stride) && rows_whole(dtype, dy_stride),
                 x_stride == width && dy_stride == width);
  a.shift = s.shift;
  int blocks = norm_backward_blocks(s, rows, width);
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
  } else if (s.ring) {
    const Ring ring = make_ring(s, dtype, width, true);
    if (ring.error == nullptr) return fail(CND_ERR_CUDA, "device error word unavailable");
    with_ring_dtype(dtype, s, LaunchRing<true>{a, ring, blocks, stream});
    count_launch();
  } else if (norm_tiles(s, width, x_stride, dy_stride)) {
    const Ring ring = make_ring(s, dtype, width, true);
    if (ring.error == nullptr) return fail(CND_ERR_CUDA, "device error word unavailable");
    blocks = std::min(blocks, sm_count() * tile_blocks(s, true));
    with_kernel<true>(dtype, s, LaunchTile<true>{a, ring, blocks, stream});
    count_launch();
  } else {
    with_kernel<true>(dtype, s, LaunchBackward{a, blocks, stream});
    count_launch();
  }
  if (params) {
    const unsigned grid = static_cast<unsigned>((2 * width + 31) / 32);
    void* w = output_mask[1] ? dweight : nullptr;
    void* b = output_mask[2] ? dbias : nullptr;
    if (dtype == CND_F64) {
      norm_reduce_kernel<double><<<grid, kReduceWarps * 32, 0, stream>>>(workspace, blocks, width, w, b, 0);
    } else if (dtype == CND_F32 || a.param_f32) {
      norm_reduce_kernel<float><<<grid, kReduceWarps * 32, 0, stream>>>(workspace, blocks, width, w, b, 1);
    } else if (dtype == CND_BF16) {
      norm_reduce_kernel<__nv_bfloat16><<<grid, kReduceWarps * 32, 0, stream>>>(workspace, blocks, width, w, b, 0);
    } else {
      norm_reduce_kernel<__half><<<grid, kReduceWarps * 32, 0, stream>>>(workspace, blocks, width, w, b, 0);
    }
    count_launch();
  }
  return launch_status("cnd_layer_norm_backward");
}

}  // extern "C"
