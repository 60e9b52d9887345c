// Gated linear recurrence along the middle axis of [outer][steps][inner]:
//
//   f_t = sigmoid(g_t),  h_t = f_t h_{t-1} + (1 - f_t) x_t;
//   q_t = f_t (dy_t + q_{t+1}),  dx_t = (1 - f_t) (dy_t + q_{t+1}),
//   dg_t = f_t (1 - f_t) (h_{t-1} - x_t) (dy_t + q_{t+1}),  dh_{-1} = q_0.
//
// A run of steps acts on a state as one affine map h -> a h + b, and maps compose:
// (a1, b1) then (a2, b2) is (a1 a2, a2 b1 + b2). So a thread reduces a few consecutive steps
// to a map, a block composes its threads' maps in shared memory to find the state each of
// them starts from, and the thread then walks its steps from that state: x, g and dy are
// read once and stay in registers between the two walks. The traffic is 3 elements a step
// forward, 5 backward. float32, 8 x 33 x 129600: 98 / 180 us, 4.2 / 3.8 TB/s. What is
// between that and the 6.55 TB/s of a copy is latency: a block loads, composes, waits and
// stores one after the other, and 128 registers leave room for two blocks on an SM. Most of
// it is seen where 16-bit columns share the time axis (65536 x 512 bf16, 87 / 176 us).
//
// Column layout (inner > 1): the lanes of a warp hold two columns each, in packed float32
// pairs, the warps of a block follow one another in time. Step layout (inner = 1, steps
// contiguous): the lanes of a warp hold neighbouring runs of steps of one column and compose
// their maps by shuffles.
//
// A block that has its columns to itself loops over the chunks of the time axis. Where
// the columns are too few to fill the SMs, every (chunk, column block) is a block of its own
// and chunks exchange their maps through global memory: blocks take tickets in time order,
// so whoever a block waits for is already running; each chunk composes the maps of the
// chunks before it in its group of kGroup, in order, with the state that the last chunk
// of the group before published. The association is fixed, so repeated calls give the
// same bits. The exchange area starts as all ones, a NaN that is never sent, and a
// map (a state) is stored at once, so a reader polls the value itself: no flag, no fence, one
// trip to L2. Waits are bounded and end at once when any wait of the launch has expired.
//
// The forward keeps the state before each block of 64 steps (256 in step layout), from which
// the backward recomputes the others in float32: it reads x, g and dy only, and its states
// carry no rounding to the tensors' type.
#include <algorithm>
#include <type_traits>

#include "layers.cuh"
#include "ptx.cuh"

namespace cnd {
namespace layers {
namespace {

constexpr int kWarps = 8;       // most warps of a block
// Chunks that are composed without an intermediate state. Forward / backward, 65536 steps of
// 512 and of 64 bf16 columns: 16 chunks 104 / 190 and 70 / 122 us, 32 chunks 103 / 194 and
// 57 / 93, 64 chunks 121 / 224 and 45 / 73.
constexpr int kGroup = 32;
constexpr uint32_t kSiteForward = 0x601, kSiteBackward = 0x602;

// Steps a thread holds: forward (by element size: what its registers take of two columns) and
// backward in column layout, both in step layout.
constexpr int forward_steps(size_t size) { return size == 2 ? 16 : 8; }
constexpr int kBackwardSteps = 8, kAlongSteps = 8;
constexpr int kStateBlock = kBackwardSteps * kWarps;  // 64
constexpr int kAlongBlock = 32 * kAlongSteps;         // 256

template <typename A>
struct Map {
  A a, b;
};

// `first`, then `second`.
template <typename A>
__device__ __forceinline__ Map<A> then(const Map<A>& first, const Map<A>& second) {
  return {first.a * second.a, second.a * first.b + second.b};
}

struct RecurrenceArgs {
  const void *x, *gate, *initial, *dy, *dlast, *states_in;
  void *y, *last, *states, *dx, *dgate, *dinitial;
  int64_t outer, steps, inner, columns;
  int64_t chunks;
  int column_blocks;
  int lanes, per_block;  // step layout: lanes of a column, columns of a block
  int balanced;  // steps a thread takes when one chunk holds them all, 0: the most it can
  // exchange between chunks (shared != 0): maps [chunks][padded], states [groups][padded],
  // a ticket counter and a word that an expired wait clears; all bits set at the start
  int shared;
  void *maps, *bases;
  unsigned int *ticket, *waiting, *error;
  uint64_t timeout_ns;
};

__device__ __forceinline__ int steps_here(int64_t left, int most) {
  return left < 0 ? 0 : left < most ? static_cast<int>(left) : most;
}

// f = sigmoid(g) and 1 - f, each to full relative accuracy (exact 0 and 1 at +-inf). For
// 16-bit tensors by the fast exponential and reciprocal, good to 2^-20; what falls below
// 2^-126 (|g| > 87) is zero.
template <typename T, typename A>
__device__ __forceinline__ void gates(A g, A* f, A* keep) {
  A e, r;
  if constexpr (sizeof(T) == 2) {
    e = exp2_fast(-fabsf(g * 1.44269504089f));
    r = reciprocal_fast(1.0f + e);
  } else {
    e = exp(-fabs(g));
    const A d = A(1) + e;
    if constexpr (sizeof(T) == 4) {
      // d is in [1, 2]: the approximate reciprocal and one Newton step
      r = reciprocal_fast(d);
      r = fmaf(r, fmaf(-d, r, 1.0f), r);
    } else {
      r = A(1) / d;
    }
  }
  const A s = e * r;
  *f = g >= A(0) ? r : s;
  *keep = g >= A(0) ? s : r;
}

// Values of the exchange area, read and written at once: 32 bits (a float32 state), 64
// bits (a float32 map, a float64).
template <typename Bits>
__device__ __forceinline__ Bits load_exchange(const Bits* p) {
  Bits v;
  if constexpr (sizeof(Bits) == 4) {
    asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  } else {
    asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  }
  return v;
}

// (All ones would read as not written yet. float32 arithmetic never gives that NaN, float64
// arithmetic may hand on a NaN operand's bits: it leaves as another NaN.)
template <typename Bits>
__device__ __forceinline__ void store_exchange(Bits* p, Bits v) {
  if (v == ~Bits{0}) v >>= 1;
  if constexpr (sizeof(Bits) == 4) {
    asm volatile("st.relaxed.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
  } else {
    asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
  }
}

// Reads *p again until it has been written. Gives up (error word set) after the timeout, or
// as soon as another wait of this launch has. (Not by the error word, which may hold what some
// other kernel's wait left there.)
template <typename Bits>
__device__ __forceinline__ Bits settle(const Bits* p, Bits v, const RecurrenceArgs& a,
                                       unsigned int site) {
  if (v != ~Bits{0}) return v;
  const uint64_t start = dev::global_timer_ns();
  for (uint32_t spin = 1;; ++spin) {
    v = load_exchange(p);
    if (v != ~Bits{0}) return v;
    if (spin % 64 == 0) {
      const bool late = dev::global_timer_ns() - start > a.timeout_ns;
      if (late) {
        *static_cast<volatile unsigned int*>(a.waiting) = 0;
        atomicCAS(a.error, 0u, site);
      }
      if (late || *static_cast<volatile unsigned int*>(a.waiting) == 0) return v;
    }
  }
}

// Words of a map: one of 64 bits for float32, two for float64.
template <typename A>
constexpr int kMapWords = sizeof(A) / 4;

template <typename A>
__device__ __forceinline__ void store_map(void* maps, int64_t i, const Map<A>& m) {
  auto* p = static_cast<unsigned long long*>(maps) + i * kMapWords<A>;
  if constexpr (sizeof(A) == 4) {
    store_exchange(p, static_cast<unsigned long long>(__float_as_uint(m.a)) |
                          static_cast<unsigned long long>(__float_as_uint(m.b)) << 32);
  } else {
    store_exchange(p, static_cast<unsigned long long>(__double_as_longlong(m.a)));
    store_exchange(p + 1, static_cast<unsigned long long>(__double_as_longlong(m.b)));
  }
}

template <typename A>
__device__ __forceinline__ Map<A> map_of(const unsigned long long (&w)[kMapWords<A>]) {
  if constexpr (sizeof(A) == 4) {
    return {__uint_as_float(static_cast<unsigned int>(w[0])),
            __uint_as_float(static_cast<unsigned int>(w[0] >> 32))};
  } else {
    return {__longlong_as_double(static_cast<long long>(w[0])),
            __longlong_as_double(static_cast<long long>(w[1]))};
  }
}

template <typename A>
__device__ __forceinline__ void store_base(void* bases, int64_t i, A v) {
  if constexpr (sizeof(A) == 4) {
    store_exchange(static_cast<unsigned int*>(bases) + i, __float_as_uint(v));
  } else {
    store_exchange(static_cast<unsigned long long*>(bases) + i,
                   static_cast<unsigned long long>(__double_as_longlong(v)));
  }
}

template <typename A>
__device__ __forceinline__ A load_base(const RecurrenceArgs& a, int64_t i, unsigned int site) {
  if constexpr (sizeof(A) == 4) {
    const auto* p = static_cast<const unsigned int*>(a.bases) + i;
    return __uint_as_float(settle(p, load_exchange(p), a, site));
  } else {
    const auto* p = static_cast<const unsigned long long*>(a.bases) + i;
    return __longlong_as_double(static_cast<long long>(settle(p, load_exchange(p), a, site)));
  }
}

// A step past the end is given the gate +inf and x = dy = 0: it holds the state and passes the
// flow on, so the walks need no branches (a branch per step had kept the exponentials of
// different steps from overlapping).

template <typename A>
__device__ __forceinline__ Map<A> shuffle_up(const Map<A>& m, int d) {
  return {__shfl_up_sync(0xffffffffu, m.a, d), __shfl_up_sync(0xffffffffu, m.b, d)};
}
template <typename A>
__device__ __forceinline__ Map<A> shuffle_down(const Map<A>& m, int d) {
  return {__shfl_down_sync(0xffffffffu, m.a, d), __shfl_down_sync(0xffffffffu, m.b, d)};
}

// The one column of a block in step layout, as Steps are the columns of the other.
struct OneColumn {
  static constexpr int kColumns = 1;
  static __device__ __forceinline__ int slot(int, int) { return 0; }
};
template <typename S>
constexpr int slots_of() {
  if constexpr (std::is_same_v<S, OneColumn>) {
    return 1;
  } else {
    return 32 * S::kColumns;
  }
}

// The state before this chunk, for the columns a lane holds (S::slot of them), from the chunks
// before it (order = 0, 1, ... in the direction of the walk) and `state`, the state before
// the first. `scratch`: [kWarps][slots] maps. The whole block calls it: warp w composes maps
// w * 4 ... of the group.
template <typename A, typename S>
__device__ __forceinline__ void carry_in(const RecurrenceArgs& a, int64_t order, int64_t block,
                                         Map<A>* scratch, unsigned int site,
                                         A (&state)[S::kColumns]) {
  constexpr int kEach = kGroup / kWarps, kWords = kMapWords<A>, kPer = S::kColumns;
  constexpr int kSlots = slots_of<S>();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t group = order / kGroup;
  const int64_t padded = static_cast<int64_t>(a.column_blocks) * kSlots;
  const auto* maps = static_cast<const unsigned long long*>(a.maps);
  unsigned long long raw[kEach][kPer][kWords];
  const auto place = [&](int i, int v) {
    return ((group * kGroup + warp * kEach + i) * padded + block * kSlots + S::slot(lane, v)) * kWords;
  };
  const int known = static_cast<int>(order - group * kGroup) - warp * kEach;  // maps of this warp
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (i < known) {
#pragma unroll
      for (int v = 0; v < kPer; ++v) {
#pragma unroll
        for (int k = 0; k < kWords; ++k) raw[i][v][k] = load_exchange(maps + place(i, v) + k);
      }
    }
  }
  if (group > 0) {
#pragma unroll
    for (int v = 0; v < kPer; ++v) {
      state[v] = load_base<A>(a, group * padded + block * kSlots + S::slot(lane, v), site);
    }
  }
#pragma unroll
  for (int v = 0; v < kPer; ++v) {
    Map<A> m{A(1), A(0)};
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (i < known) {
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
          raw[i][v][k] = settle(maps + place(i, v) + k, raw[i][v][k], a, site);
        }
        m = then(m, map_of<A>(raw[i][v]));
      }
    }
    if (kSlots > 1 || lane == 0) scratch[warp * kSlots + S::slot(lane, v)] = m;
  }
  __syncthreads();
#pragma unroll
  for (int v = 0; v < kPer; ++v) {
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const Map<A> m = scratch[w * kSlots + S::slot(lane, v)];
      state[v] = m.a * state[v] + m.b;
    }
  }
}

// Column `column`'s first element in [outer][steps][inner].
__device__ __forceinline__ int64_t column_base(const RecurrenceArgs& a, int64_t column) {
  int64_t outer;
  if (a.columns <= INT32_MAX) {
    outer = static_cast<uint32_t>(column) / static_cast<uint32_t>(a.inner);
  } else {
    outer = column / a.inner;
  }
  return outer * a.steps * a.inner + (column - outer * a.inner);
}

// What a lane holds of a step: two columns (of float32 arithmetic, in packed pairs) or, for
// float64, one.
template <typename T>
struct Held {
  using P = Two;
  static constexpr int kColumns = 2;
  static __device__ __forceinline__ P value(float v) { return same(v); }
  static __device__ __forceinline__ P join(const float (&v)[2]) { return two(v[0], v[1]); }
  static __device__ __forceinline__ void part(P p, float (&v)[2]) { unpack(p, &v[0], &v[1]); }
  static __device__ __forceinline__ P mad(P a, P b, P c) { return fma2(a, b, c); }
  static __device__ __forceinline__ P mul(P a, P b) { return mul2(a, b); }
  static __device__ __forceinline__ P add(P a, P b) { return add2(a, b); }
};
template <>
struct Held<double> {
  using P = double;
  static constexpr int kColumns = 1;
  static __device__ __forceinline__ P value(double v) { return v; }
  static __device__ __forceinline__ P join(const double (&v)[1]) { return v[0]; }
  static __device__ __forceinline__ void part(P p, double (&v)[1]) { v[0] = p; }
  static __device__ __forceinline__ P mad(P a, P b, P c) { return fma(a, b, c); }
  static __device__ __forceinline__ P mul(P a, P b) { return a * b; }
  static __device__ __forceinline__ P add(P a, P b) { return a + b; }
};

// A map of the held columns.
template <typename T>
struct HeldMap {
  typename Held<T>::P a, b;
};
template <typename T>
__device__ __forceinline__ HeldMap<T> then(const HeldMap<T>& first, const HeldMap<T>& second) {
  using H = Held<T>;
  return {H::mul(first.a, second.a), H::mad(second.a, first.b, second.b)};
}

// The addresses of a thread's steps. Adjacent: its columns are neighbours read at once (two
// 16-bit columns are 4 bytes); else they lie 32 apart, each warp reading 32 neighbours, which
// needs no alignment (32768 bf16 columns of 1024 steps: forward 76 us adjacent, 87 apart).
// Step i of every tensor lies i strides behind the same offset.
// Offset: uint32_t bytes where the tensors are below 4 GB (one 32-bit addition serves all
// tensors, whose bases stay in uniform registers), else int64_t.
template <typename T, bool kAdjacent, typename Offset>
struct Steps {
  static constexpr int kColumns = Held<T>::kColumns, kParts = kAdjacent ? 1 : kColumns;
  Offset first[kParts], stride;
  bool live[kParts];

  __device__ __forceinline__ Steps(const RecurrenceArgs& a, int64_t block, int lane)
      : stride(static_cast<Offset>(a.inner * static_cast<int64_t>(sizeof(T)))) {
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      const int64_t c = column(block, lane, p);
      live[p] = c < a.columns;
      first[p] = live[p] ? static_cast<Offset>(column_base(a, c) * static_cast<int64_t>(sizeof(T)))
                         : Offset(0);
    }
  }
  // Column of held column `i`.
  static __device__ __forceinline__ int64_t column(int64_t block, int lane, int i) {
    return block * 32 * kColumns + (kAdjacent ? lane * kColumns + i : i * 32 + lane);
  }
  // Slot of held column `i` among the block's.
  static __device__ __forceinline__ int slot(int lane, int i) {
    return kAdjacent ? lane * kColumns + i : i * 32 + lane;
  }
  __device__ __forceinline__ bool lives(int i) const { return live[kAdjacent ? 0 : i]; }

  __device__ __forceinline__ Pack<T, kColumns> read(const void* base, Offset ahead) const {
    Pack<T, kColumns> v;
    if constexpr (kAdjacent) {
      v = *reinterpret_cast<const Pack<T, kColumns>*>(static_cast<const char*>(base) + (first[0] + ahead));
    } else {
#pragma unroll
      for (int p = 0; p < kColumns; ++p) {
        v.v[p] = *reinterpret_cast<const T*>(static_cast<const char*>(base) + (first[p] + ahead));
      }
    }
    return v;
  }
  // The held columns that exist, `other` for the rest.
  __device__ __forceinline__ Pack<T, kColumns> read_live(const void* base, Offset ahead,
                                                         float other) const {
    Pack<T, kColumns> v;
#pragma unroll
    for (int i = 0; i < kColumns; ++i) {
      v.v[i] = narrow<T>(static_cast<typename Wide<T>::type>(other));
    }
    if constexpr (kAdjacent) {
      if (live[0]) v = read(base, ahead);
    } else {
#pragma unroll
      for (int p = 0; p < kColumns; ++p) {
        if (live[p]) {
          v.v[p] = *reinterpret_cast<const T*>(static_cast<const char*>(base) + (first[p] + ahead));
        }
      }
    }
    return v;
  }
  __device__ __forceinline__ void write(void* base, Offset ahead, typename Held<T>::P value) const {
    typename Wide<T>::type w[kColumns];
    Held<T>::part(value, w);
    if constexpr (kAdjacent) {
      if (!live[0]) return;
      char* to = static_cast<char*>(base) + (first[0] + ahead);
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint32_t*>(to) = narrow2<T>(value);
      } else {
        Pack<T, kColumns> v;
#pragma unroll
        for (int i = 0; i < kColumns; ++i) v.v[i] = narrow<T>(w[i]);
        *reinterpret_cast<Pack<T, kColumns>*>(to) = v;
      }
    } else {
#pragma unroll
      for (int p = 0; p < kColumns; ++p) {
        if (live[p]) {
          *reinterpret_cast<T*>(static_cast<char*>(base) + (first[p] + ahead)) = narrow<T>(w[p]);
        }
      }
    }
  }
  // A step's pack past the end of the steps.
  static __device__ __forceinline__ Pack<T, kColumns> all(float value) {
    Pack<T, kColumns> v;
#pragma unroll
    for (int i = 0; i < kColumns; ++i) {
      v.v[i] = narrow<T>(static_cast<typename Wide<T>::type>(value));
    }
    return v;
  }
};

template <typename T, int N>
__device__ __forceinline__ typename Held<T>::P held(const Pack<T, N>& p) {
  typename Wide<T>::type w[N];
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = widen(p.v[i]);
  return Held<T>::join(w);
}

// f and 1 - f of the held columns.
template <typename T, int N>
__device__ __forceinline__ void held_gates(const Pack<T, N>& g, typename Held<T>::P* f,
                                           typename Held<T>::P* keep) {
  if constexpr (sizeof(T) == 2) {  // gates() in pairs
    const Two pair = held<T>(g);
    float lo, hi, m0, m1, r0, r1, s0, s1;
    unpack(pair, &lo, &hi);
    unpack(mul2(pair, same(1.44269504089f)), &m0, &m1);
    const Two e = two(exp2_fast(-fabsf(m0)), exp2_fast(-fabsf(m1)));
    float d0, d1;
    unpack(add2(e, same(1.0f)), &d0, &d1);
    r0 = reciprocal_fast(d0);
    r1 = reciprocal_fast(d1);
    unpack(mul2(e, two(r0, r1)), &s0, &s1);
    *f = two(lo >= 0.0f ? r0 : s0, hi >= 0.0f ? r1 : s1);
    *keep = two(lo >= 0.0f ? s0 : r0, hi >= 0.0f ? s1 : r1);
  } else {
    typename Wide<T>::type w[N], v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) gates<T>(widen(g.v[i]), &w[i], &v[i]);
    *f = Held<T>::join(w);
    *keep = Held<T>::join(v);
  }
}

// Values kept per column ([..][columns] of type Wide<T>), zero where there are none.
template <typename T, typename S>
__device__ __forceinline__ typename Held<T>::P load_columns(const void* p, const S& at,
                                                            const RecurrenceArgs& a, int64_t row,
                                                            int64_t block, int lane) {
  using A = typename Wide<T>::type;
  A w[S::kColumns];
#pragma unroll
  for (int i = 0; i < S::kColumns; ++i) {
    w[i] = p != nullptr && at.lives(i)
               ? static_cast<const A*>(p)[row * a.columns + S::column(block, lane, i)]
               : A(0);
  }
  return Held<T>::join(w);
}

template <typename T, typename S>
__device__ __forceinline__ void store_columns(void* p, const S& at, const RecurrenceArgs& a,
                                              int64_t row, int64_t block, int lane,
                                              typename Held<T>::P value) {
  using A = typename Wide<T>::type;
  A w[S::kColumns];
  Held<T>::part(value, w);
#pragma unroll
  for (int i = 0; i < S::kColumns; ++i) {
    if (at.lives(i)) static_cast<A*>(p)[row * a.columns + S::column(block, lane, i)] = w[i];
  }
}

// Sends this chunk's map (and, from the last chunk of a group, the state behind it) and returns
// the state before the chunk.
template <typename T, typename S>
__device__ __forceinline__ typename Held<T>::P exchange(const RecurrenceArgs& a, int64_t order,
                                                        int64_t block, int lane, bool sends,
                                                        const HeldMap<T>& whole,
                                                        typename Held<T>::P begin,
                                                        Map<typename Wide<T>::type>* scratch,
                                                        unsigned int site) {
  using A = typename Wide<T>::type;
  constexpr int kSlots = 32 * S::kColumns;
  const int64_t padded = static_cast<int64_t>(a.column_blocks) * kSlots;
  A map_a[S::kColumns], map_b[S::kColumns], state[S::kColumns];
  Held<T>::part(whole.a, map_a);
  Held<T>::part(whole.b, map_b);
  Held<T>::part(begin, state);
  if (sends) {
#pragma unroll
    for (int i = 0; i < S::kColumns; ++i) {
      store_map<A>(a.maps, order * padded + block * kSlots + S::slot(lane, i),
                   Map<A>{map_a[i], map_b[i]});
    }
  }
  carry_in<A, S>(a, order, block, scratch, site, state);
  if (sends && (order + 1) % kGroup == 0) {
#pragma unroll
    for (int i = 0; i < S::kColumns; ++i) {
      store_base<A>(a.bases, (order + 1) / kGroup * padded + block * kSlots + S::slot(lane, i),
                    map_a[i] * state[i] + map_b[i]);
    }
  }
  return Held<T>::join(state);
}

// Blocks an SM: what two columns of forward_steps() cost in registers.
template <typename T, bool kAdjacent, typename Offset>
__global__ void __launch_bounds__(kWarps * 32, sizeof(T) == 4 ? 4 : 2)
    columns_forward_kernel(const __grid_constant__ RecurrenceArgs a) {
  using H = Held<T>;
  using S = Steps<T, kAdjacent, Offset>;
  using A = typename Wide<T>::type;
  using P = typename H::P;
  constexpr int kSteps = forward_steps(sizeof(T)), kColumns = H::kColumns;
  __shared__ HeldMap<T> maps[kWarps][32];
  __shared__ Map<A> before[kWarps * 32 * kColumns];
  __shared__ unsigned int taken;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int warps = blockDim.x >> 5;
  int64_t block = blockIdx.x, chunk = 0, stop = a.chunks;
  if (a.shared) {
    if (threadIdx.x == 0) taken = atomicAdd(a.ticket, 1u) + 1u;
    __syncthreads();
    chunk = taken / a.column_blocks;
    block = taken - static_cast<uint32_t>(chunk) * a.column_blocks;
    stop = chunk + 1;
  }
  const S at(a, block, lane);
  P begin = load_columns<T>(a.initial, at, a, 0, block, lane);
  for (; chunk < stop; ++chunk) {
    const int most = a.balanced ? a.balanced : kSteps;
    const int64_t first = (chunk * warps + warp) * most;
    const Offset offset = static_cast<Offset>(first) * at.stride;
    const int count = steps_here(a.steps - first, most);
    Pack<T, kColumns> px[kSteps], pg[kSteps];
    if (count > 0 && at.lives(0) && at.lives(kColumns - 1)) {
      // steps past the end read the last one again: no branches between the loads
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const Offset ahead = offset + min(i, count - 1) * at.stride;
        px[i] = at.read(a.x, ahead);
        pg[i] = at.read(a.gate, ahead);
      }
      if (count < kSteps) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          px[i] = i < count ? px[i] : S::all(0.0f);
          pg[i] = i < count ? pg[i] : S::all(INFINITY);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        px[i] = S::all(0.0f);
        pg[i] = S::all(INFINITY);
        if (i < count) {
          px[i] = at.read_live(a.x, offset + i * at.stride, 0.0f);
          pg[i] = at.read_live(a.gate, offset + i * at.stride, INFINITY);
        }
      }
    }
    P f[kSteps], b[kSteps];
    HeldMap<T> own{H::value(1), H::value(0)};
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      P keep;
      held_gates<T>(pg[i], &f[i], &keep);
      b[i] = H::mul(keep, held<T>(px[i]));
      own = then<T>(own, HeldMap<T>{f[i], b[i]});
    }
    maps[warp][lane] = own;
    __syncthreads();
    HeldMap<T> earlier{H::value(1), H::value(0)};  // the block's warps before this one
#pragma unroll
    for (int w = 0; w < kWarps - 1; ++w) {
      if (w < warp) earlier = then<T>(earlier, maps[w][lane]);
    }
    P state;
    if (a.shared) {
      state = exchange<T, S>(a, chunk, block, lane, warp == warps - 1 && chunk + 1 < a.chunks,
                             then<T>(earlier, own), begin, before, kSiteForward);
    } else {
      state = begin;
      if (chunk + 1 < stop) {
        HeldMap<T> all = earlier;
        for (int w = warp; w < warps; ++w) all = then<T>(all, maps[w][lane]);
        begin = H::mad(all.a, begin, all.b);
        __syncthreads();
      }
    }
    state = H::mad(earlier.a, state, earlier.b);
    if (a.states != nullptr && first < a.steps && first % kStateBlock == 0) {
      store_columns<T>(a.states, at, a, first / kStateBlock, block, lane, state);
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      state = H::mad(f[i], state, b[i]);
      if (i < count) at.write(a.y, offset + i * at.stride, state);
    }
    const int64_t end = a.steps > 0 ? a.steps - 1 : 0;
    if (first <= end && end < first + most) store_columns<T>(a.last, at, a, 0, block, lane, state);
  }
}

template <typename T, bool kAdjacent, typename Offset>
__global__ void __launch_bounds__(kWarps * 32, 2)
    columns_backward_kernel(const __grid_constant__ RecurrenceArgs a) {
  using H = Held<T>;
  using S = Steps<T, kAdjacent, Offset>;
  using A = typename Wide<T>::type;
  using P = typename H::P;
  constexpr int kSteps = kBackwardSteps, kColumns = H::kColumns;
  __shared__ HeldMap<T> forward[kWarps][32];
  __shared__ P backward[kWarps][32];  // the flow's map: same factor, own offset
  __shared__ Map<A> after[kWarps * 32 * kColumns];
  __shared__ unsigned int taken;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int warps = blockDim.x >> 5;
  int64_t block = blockIdx.x, order = 0, stop = a.chunks;  // chunks from the last to the first
  if (a.shared) {
    if (threadIdx.x == 0) taken = atomicAdd(a.ticket, 1u) + 1u;
    __syncthreads();
    order = taken / a.column_blocks;
    block = taken - static_cast<uint32_t>(order) * a.column_blocks;
    stop = order + 1;
  }
  const S at(a, block, lane);
  P begin = load_columns<T>(a.dlast, at, a, 0, block, lane);
  for (; order < stop; ++order) {
    const int64_t chunk = a.chunks - 1 - order;
    const int most = a.balanced ? a.balanced : kSteps;
    const int64_t first = (chunk * warps + warp) * most;
    const Offset offset = static_cast<Offset>(first) * at.stride;
    const int count = steps_here(a.steps - first, most);
    Pack<T, kColumns> px[kSteps], pg[kSteps], pd[kSteps];
    if (count > 0 && a.dy != nullptr && at.lives(0) && at.lives(kColumns - 1)) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const Offset ahead = offset + min(i, count - 1) * at.stride;
        px[i] = at.read(a.x, ahead);
        pg[i] = at.read(a.gate, ahead);
        pd[i] = at.read(a.dy, ahead);
      }
      if (count < kSteps) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          px[i] = i < count ? px[i] : S::all(0.0f);
          pg[i] = i < count ? pg[i] : S::all(INFINITY);
          pd[i] = i < count ? pd[i] : S::all(0.0f);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        px[i] = pd[i] = S::all(0.0f);
        pg[i] = S::all(INFINITY);
        if (i < count) {
          px[i] = at.read_live(a.x, offset + i * at.stride, 0.0f);
          pg[i] = at.read_live(a.gate, offset + i * at.stride, INFINITY);
          if (a.dy != nullptr) pd[i] = at.read_live(a.dy, offset + i * at.stride, 0.0f);
        }
      }
    }
    // the state before the chunk
    P state = a.steps > 0 ? load_columns<T>(a.states_in, at, a, chunk, block, lane) : H::value(0);
    P f[kSteps], keep[kSteps];
    HeldMap<T> own{H::value(1), H::value(0)};
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      held_gates<T>(pg[i], &f[i], &keep[i]);
      own = then<T>(own, HeldMap<T>{f[i], H::mul(keep[i], held<T>(px[i]))});
    }
    P flow = H::value(0);
#pragma unroll
    for (int i = kSteps - 1; i >= 0; --i) flow = H::mul(f[i], H::add(held<T>(pd[i]), flow));
    forward[warp][lane] = own;
    backward[warp][lane] = flow;
    __syncthreads();
    HeldMap<T> later{H::value(1), H::value(0)};  // the block's warps after this one, backwards
#pragma unroll
    for (int w = 0; w < kWarps - 1; ++w) {
      if (w < warp) state = H::mad(forward[w][lane].a, state, forward[w][lane].b);
    }
#pragma unroll
    for (int w = kWarps - 1; w > 0; --w) {
      if (w > warp && w < warps) {
        later = then<T>(later, HeldMap<T>{forward[w][lane].a, backward[w][lane]});
      }
    }
    P q;
    if (a.shared) {
      q = exchange<T, S>(a, order, block, lane, warp == 0 && order + 1 < a.chunks,
                         then<T>(later, HeldMap<T>{own.a, flow}), begin, after, kSiteBackward);
    } else {
      q = begin;
      if (order + 1 < stop) {
        HeldMap<T> all = later;
        for (int w = warp; w >= 0; --w) {
          all = then<T>(all, HeldMap<T>{forward[w][lane].a, backward[w][lane]});
        }
        begin = H::mad(all.a, begin, all.b);
        __syncthreads();
      }
    }
    q = H::mad(later.a, q, later.b);
    P slope[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      // f (1 - f) (h_{t-1} - x), what the gate's gradient takes of the flow
      const P x = held<T>(px[i]);
      const P difference = H::mad(x, H::value(-1), state);
      slope[i] = H::mul(H::mul(f[i], keep[i]), difference);
      state = H::mad(f[i], state, H::mul(keep[i], x));
    }
#pragma unroll
    for (int i = kSteps - 1; i >= 0; --i) {
      const P total = H::add(held<T>(pd[i]), q);
      q = H::mul(f[i], total);
      if (i < count) {
        if (a.dx != nullptr) at.write(a.dx, offset + i * at.stride, H::mul(keep[i], total));
        if (a.dgate != nullptr) at.write(a.dgate, offset + i * at.stride, H::mul(slope[i], total));
      }
    }
    if (a.dinitial != nullptr && first == 0) {
      store_columns<T>(a.dinitial, at, a, 0, block, lane, q);
    }
  }
}

// ---- step layout -----------------------------------------------------------------------

// Column c starts at element c * steps, off a 16-byte boundary of its tensor by `shift` elements
// where steps is no multiple of one. Its runs start `shift` elements earlier, so that in an aligned
// tensor every run is read and written in aligned vectors; the column's first run then begins, like
// its last one ends, with steps that do not exist and hold the state. The runs lie the same
// whatever the alignment of the data, which only decides between vectors and single elements: the
// backward, whose tensors may be aligned otherwise, looks for the kept states where the
// forward put them. A column takes `lanes` lanes of a warp (a short column less than a warp, a
// block then several columns) or a block's warps one behind the other.
template <typename T>
struct Run {
  static constexpr int kPer = 16 / sizeof(T);
  int64_t first;  // step of the run's first element, negative in a shifted column's first run
  int lo, hi;     // steps of the run that exist
  bool vectors;   // whole, of tensors that start on 16-byte boundaries

  __device__ __forceinline__ Run(int64_t index, int shift, int64_t steps, bool aligned)
      : first(index * kAlongSteps - shift) {
    lo = first < 0 ? static_cast<int>(-first) : 0;
    hi = steps_here(steps - first, kAlongSteps);
    vectors = aligned && lo == 0 && hi == kAlongSteps;
  }
  __device__ __forceinline__ bool has(int i) const { return i >= lo && i < hi; }

  // `column`: the column's first element.
  __device__ __forceinline__ void load(const T* column, float other, T (&v)[kAlongSteps]) const {
    const T* p = column + first;
    if (vectors) {
#pragma unroll
      for (int i = 0; i < kAlongSteps; i += kPer) {
        *reinterpret_cast<Pack<T, kPer>*>(v + i) = *reinterpret_cast<const Pack<T, kPer>*>(p + i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kAlongSteps; ++i) {
        v[i] = narrow<T>(static_cast<typename Wide<T>::type>(other));
        if (has(i)) v[i] = p[i];
      }
    }
  }
  __device__ __forceinline__ void store(T* column, const T (&v)[kAlongSteps]) const {
    T* p = column + first;
    if (vectors) {
#pragma unroll
      for (int i = 0; i < kAlongSteps; i += kPer) {
        *reinterpret_cast<Pack<T, kPer>*>(p + i) = *reinterpret_cast<const Pack<T, kPer>*>(v + i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kAlongSteps; ++i) {
        if (has(i)) p[i] = v[i];
      }
    }
  }
};

// Places of a thread in step layout: its column, its lane among the column's and its warp.
struct Along {
  int64_t column, chunk;  // chunk: the walk's first
  int warp, warps, lane, lanes;

  __device__ __forceinline__ Along(const RecurrenceArgs& a, unsigned int* taken) {
    lanes = a.lanes;
    chunk = 0;
    if (a.shared) {
      if (threadIdx.x == 0) *taken = atomicAdd(a.ticket, 1u) + 1u;
      __syncthreads();
      chunk = *taken / a.column_blocks;
      column = *taken - static_cast<uint32_t>(chunk) * a.column_blocks;
    } else {
      column = blockIdx.x;
    }
    warp = threadIdx.x >> 5;
    warps = blockDim.x >> 5;
    lane = threadIdx.x & 31;
    if (a.per_block > 1) {  // several columns a block, each within a warp
      column = static_cast<int64_t>(blockIdx.x) * a.per_block + threadIdx.x / lanes;
      warp = 0;
      warps = 1;
      lane = threadIdx.x % lanes;
    }
  }
};

// Three blocks an SM: at the 94 registers of two, 8 x 1022 columns of 4097 float32 steps took 187 us,
// at 78 133.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32, sizeof(T) == 8 ? 2 : 3)
    steps_forward_kernel(const __grid_constant__ RecurrenceArgs a, bool aligned) {
  using A = typename Wide<T>::type;
  __shared__ Map<A> maps[kWarps];
  __shared__ Map<A> before[kWarps];
  __shared__ unsigned int taken;
  const Along at(a, &taken);
  const bool live = at.column < a.columns;
  const int64_t column = live ? at.column : 0;
  const int shift = static_cast<int>(column * a.steps % Run<T>::kPer);
  const int64_t stop = a.shared ? at.chunk + 1 : a.chunks;
  const T* x_column = static_cast<const T*>(a.x) + column * a.steps;
  const T* g_column = static_cast<const T*>(a.gate) + column * a.steps;
  T* y_column = static_cast<T*>(a.y) + column * a.steps;
  A begin = a.initial != nullptr ? static_cast<const A*>(a.initial)[column] : A(0);
  for (int64_t chunk = at.chunk; chunk < stop; ++chunk) {
    const Run<T> run((chunk * at.warps + at.warp) * at.lanes + at.lane, shift, a.steps, aligned);
    alignas(16) T x[kAlongSteps], g[kAlongSteps];
    run.load(x_column, 0.0f, x);
    run.load(g_column, INFINITY, g);
    A f[kAlongSteps], b[kAlongSteps];
    Map<A> own{A(1), A(0)};
#pragma unroll
    for (int i = 0; i < kAlongSteps; ++i) {
      A keep;
      gates<T>(widen(g[i]), &f[i], &keep);
      b[i] = keep * widen(x[i]);
      own = then(own, Map<A>{f[i], b[i]});
    }
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      if (d >= at.lanes) break;
      const Map<A> m = shuffle_up(own, d);
      if (at.lane >= d) own = then(m, own);
    }
    Map<A> earlier = shuffle_up(own, 1);
    if (at.lane == 0) earlier = {A(1), A(0)};
    Map<A> lead{A(1), A(0)};  // the block's warps before this one
    if (at.warps > 1) {
      if (at.lane == 31) maps[at.warp] = own;
      __syncthreads();
      for (int w = 0; w < at.warp; ++w) lead = then(lead, maps[w]);
    }
    A state = begin;
    if (a.shared) {
      const bool sends = at.warp == at.warps - 1 && at.lane == 31 && chunk + 1 < a.chunks;
      if (sends) store_map<A>(a.maps, chunk * a.column_blocks + column, then(lead, own));
      A carried[1] = {begin};
      carry_in<A, OneColumn>(a, chunk, column, before, kSiteForward, carried);
      state = carried[0];
      if (sends && (chunk + 1) % kGroup == 0) {
        const Map<A> all = then(lead, own);
        store_base<A>(a.bases, (chunk + 1) / kGroup * a.column_blocks + column, all.a * state + all.b);
      }
    } else if (chunk + 1 < stop) {
      Map<A> all = lead;
      for (int w = at.warp; w < at.warps; ++w) all = then(all, maps[w]);
      begin = all.a * begin + all.b;
      __syncthreads();
    }
    state = lead.a * state + lead.b;
    if (a.states != nullptr && at.lane == 0 && live && run.first < a.steps) {
      static_cast<A*>(a.states)[(run.first + shift) / kAlongBlock * a.columns + column] = state;
    }
    state = earlier.a * state + earlier.b;
    alignas(16) T y[kAlongSteps];
#pragma unroll
    for (int i = 0; i < kAlongSteps; ++i) {
      state = f[i] * state + b[i];
      y[i] = narrow<T>(state);
    }
    if (!live) continue;
    run.store(y_column, y);
    const int64_t end = a.steps - 1;
    if (run.first <= end && end < run.first + kAlongSteps) static_cast<A*>(a.last)[column] = state;
  }
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
    steps_backward_kernel(const __grid_constant__ RecurrenceArgs a, bool aligned) {
  using A = typename Wide<T>::type;
  __shared__ Map<A> maps[kWarps];
  __shared__ Map<A> after[kWarps];
  __shared__ unsigned int taken;
  const Along at(a, &taken);
  const bool live = at.column < a.columns;
  const int64_t column = live ? at.column : 0;
  const int shift = static_cast<int>(column * a.steps % Run<T>::kPer);
  const int64_t stop = a.shared ? at.chunk + 1 : a.chunks;
  const int64_t base = column * a.steps;
  A begin = a.dlast != nullptr ? static_cast<const A*>(a.dlast)[column] : A(0);
  for (int64_t order = at.chunk; order < stop; ++order) {
    const int64_t chunk = a.chunks - 1 - order;
    const int64_t warp_run = (chunk * at.warps + at.warp) * at.lanes;
    const Run<T> run(warp_run + at.lane, shift, a.steps, aligned);
    alignas(16) T x[kAlongSteps], g[kAlongSteps], d[kAlongSteps];
    run.load(static_cast<const T*>(a.x) + base, 0.0f, x);
    run.load(static_cast<const T*>(a.gate) + base, INFINITY, g);
    if (a.dy != nullptr) {
      run.load(static_cast<const T*>(a.dy) + base, 0.0f, d);
    } else {
#pragma unroll
      for (int i = 0; i < kAlongSteps; ++i) d[i] = narrow<T>(A(0));
    }
    A state = warp_run * kAlongSteps - shift < a.steps
                  ? static_cast<const A*>(a.states_in)[warp_run * kAlongSteps / kAlongBlock * a.columns + column]
                  : A(0);
    A f[kAlongSteps], keep[kAlongSteps];
    Map<A> own{A(1), A(0)};
#pragma unroll
    for (int i = 0; i < kAlongSteps; ++i) {
      gates<T>(widen(g[i]), &f[i], &keep[i]);
      own = then(own, Map<A>{f[i], keep[i] * widen(x[i])});
    }
    Map<A> back{own.a, A(0)};
#pragma unroll
    for (int i = kAlongSteps - 1; i >= 0; --i) back.b = f[i] * (widen(d[i]) + back.b);
#pragma unroll
    for (int k = 1; k < 32; k *= 2) {
      if (k >= at.lanes) break;
      const Map<A> m = shuffle_up(own, k);
      if (at.lane >= k) own = then(m, own);
      const Map<A> n = shuffle_down(back, k);
      if (at.lane < at.lanes - k) back = then(n, back);
    }
    Map<A> earlier = shuffle_up(own, 1), later = shuffle_down(back, 1);
    if (at.lane > 0) state = earlier.a * state + earlier.b;
    if (at.lane == at.lanes - 1) later = {A(1), A(0)};
    Map<A> lead{A(1), A(0)};  // the block's warps after this one
    if (at.warps > 1) {
      if (at.lane == 0) maps[at.warp] = back;
      __syncthreads();
      for (int w = at.warps - 1; w > at.warp; --w) lead = then(lead, maps[w]);
    }
    A q = begin;
    if (a.shared) {
      const bool sends = at.warp == 0 && at.lane == 0 && order + 1 < a.chunks;
      if (sends) store_map<A>(a.maps, order * a.column_blocks + column, then(lead, back));
      A carried[1] = {begin};
      carry_in<A, OneColumn>(a, order, column, after, kSiteBackward, carried);
      q = carried[0];
      if (sends && (order + 1) % kGroup == 0) {
        const Map<A> all = then(lead, back);
        store_base<A>(a.bases, (order + 1) / kGroup * a.column_blocks + column, all.a * q + all.b);
      }
    } else if (order + 1 < stop) {
      Map<A> all = lead;
      for (int w = at.warp; w >= 0; --w) all = then(all, maps[w]);
      begin = all.a * begin + all.b;
      __syncthreads();
    }
    q = lead.a * q + lead.b;
    q = later.a * q + later.b;
    A slope[kAlongSteps];
#pragma unroll
    for (int i = 0; i < kAlongSteps; ++i) {
      const A value = widen(x[i]);
      slope[i] = f[i] * keep[i] * (state - value);
      state = f[i] * state + keep[i] * value;
    }
    alignas(16) T dx[kAlongSteps], dg[kAlongSteps];
#pragma unroll
    for (int i = kAlongSteps - 1; i >= 0; --i) {
      const A total = widen(d[i]) + q;
      dx[i] = narrow<T>(keep[i] * total);
      dg[i] = narrow<T>(slope[i] * total);
      q = f[i] * total;
    }
    if (!live) continue;
    if (a.dx != nullptr) run.store(static_cast<T*>(a.dx) + base, dx);
    if (a.dgate != nullptr) run.store(static_cast<T*>(a.dgate) + base, dg);
    if (a.dinitial != nullptr && run.first <= 0 && run.first + kAlongSteps > 0) {
      static_cast<A*>(a.dinitial)[column] = q;
    }
  }
}

// ---- choice of kernel and layout of the workspace --------------------------------------

struct RecurrencePlan {
  bool along;  // step layout
  int warps;   // warps a block
  int64_t chunks;
  int64_t column_blocks;
  int lanes, per_block;  // step layout
  int balanced;
  bool shared;
  size_t maps = 0, bases = 0, ticket = 0, waiting = 0, total = 0;
};

RecurrencePlan plan_recurrence(int dtype, int64_t outer, int64_t steps, int64_t inner,
                               bool backward) {
  RecurrencePlan p{};
  const int64_t columns = outer * inner;
  const int held = dtype == CND_F64 ? 1 : 2;  // columns a lane
  p.along = inner == 1 && steps > 1;
  p.lanes = 32;
  p.per_block = 1;
  if (p.along) {
    // runs of a column: one more where its start is shifted
    const int per = 16 / element_size(dtype);
    const int64_t ahead = steps % per != 0 ? per - 1 : 0;
    const int64_t runs = (steps + ahead + kAlongSteps - 1) / kAlongSteps;
    p.warps = static_cast<int>(std::min<int64_t>(kWarps, (runs + 31) / 32));
    p.chunks = (runs + p.warps * 32 - 1) / (p.warps * 32);
    if (runs <= 32) {
      p.lanes = 1;
      while (p.lanes < runs) p.lanes *= 2;
      p.warps = kWarps;
      p.per_block = kWarps * 32 / p.lanes;
    }
  } else {
    const int64_t per_warp = backward ? kBackwardSteps : forward_steps(element_size(dtype));
    p.warps = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kWarps, (steps + per_warp - 1) / per_warp)));
    p.chunks = std::max<int64_t>(1, (steps + p.warps * per_warp - 1) / (p.warps * per_warp));
  }
  // Up to 64 steps (one kept state), the warps share them evenly: 33 steps as 11 + 11 + 11.
  if (!p.along && steps <= kStateBlock) p.balanced = static_cast<int>((steps + p.warps - 1) / p.warps);
  p.column_blocks = p.along ? (columns + p.per_block - 1) / p.per_block
                            : (columns + 32 * held - 1) / (32 * held);
  // Too few column blocks to give each SM more than one share the time axis. bf16, 4096
  // steps, forward / backward: 128 blocks 114 / 232 us alone and 90 / 180 shared, 160 blocks
  // 131 / 264 and 106 / 220, 200 blocks 133 / 269 and 129 / 270; 2048 steps, 256 blocks 77 / 146
  // and 89 / 175.
  p.shared = p.chunks > 1 && p.column_blocks < 200;
  if (p.shared) {
    const int64_t padded = p.along ? columns : p.column_blocks * 32 * held;
    const int64_t groups = (p.chunks + kGroup - 1) / kGroup;
    const size_t wide = dtype == CND_F64 ? 8 : 4;
    const auto take = [&](size_t bytes) {
      const size_t at = p.total;
      p.total += (bytes + 255) / 256 * 256;
      return at;
    };
    p.ticket = take(sizeof(unsigned int));
    p.waiting = take(sizeof(unsigned int));
    p.maps = take(static_cast<size_t>(p.chunks * padded) * 2 * wide);
    p.bases = take(static_cast<size_t>(groups * padded) * wide);
  }
  return p;
}

// Binds the exchange area and sets its bits.
int bind_exchange(const char* who, const RecurrencePlan& p, void* workspace, size_t bytes,
                  RecurrenceArgs* a, cudaStream_t stream) {
  a->chunks = p.chunks;
  a->column_blocks = static_cast<int>(p.column_blocks);
  a->shared = p.shared;
  a->balanced = p.balanced;
  a->lanes = p.lanes;
  a->per_block = p.per_block;
  if (p.column_blocks > INT32_MAX) {
    return fail(CND_ERR_UNSUPPORTED, "%s: too many columns", who);
  }
  if (!p.shared) return CND_OK;
  if (workspace == nullptr || bytes < p.total) {
    return fail(CND_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who,
                workspace == nullptr ? size_t{0} : bytes, p.total);
  }
  if (!aligned16(workspace)) {
    return fail(CND_ERR_WORKSPACE, "%s: workspace must be 16-byte aligned", who);
  }
  char* base = static_cast<char*>(workspace);
  a->maps = base + p.maps;
  a->bases = base + p.bases;
  a->ticket = reinterpret_cast<unsigned int*>(base + p.ticket);
  a->waiting = reinterpret_cast<unsigned int*>(base + p.waiting);
  a->error = device_error_word();
  a->timeout_ns = wait_timeout_ns();
  if (a->error == nullptr) return fail(CND_ERR_CUDA, "device error word unavailable");
  if (cudaMemsetAsync(workspace, 0xff, p.total, stream) != cudaSuccess) return launch_status(who);
  return CND_OK;
}

unsigned recurrence_grid(const RecurrencePlan& p) {
  return static_cast<unsigned>(p.shared ? p.column_blocks * p.chunks : p.column_blocks);
}

// Whether two neighbouring columns can be read and written at once.
bool pairs_aligned(int dtype, int64_t inner, std::initializer_list<const void*> pointers) {
  if (inner % 2 != 0) return false;
  for (const void* p : pointers) {
    if (reinterpret_cast<uintptr_t>(p) % (2 * element_size(dtype)) != 0) return false;
  }
  return true;
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
  using namespace cnd::layers;
  if (steps <= 0) return 0;
  // in step layout a column's runs may start up to 7 steps before it
  if (inner == 1 && steps > 1) return (steps + 6) / kAlongBlock + 1;
  return (steps - 1) / kStateBlock + 1;
}

size_t cnd_gated_recurrence_workspace_size(int32_t dtype, int64_t outer, int64_t steps,
                                           int64_t inner) {
  using namespace cnd::layers;
  if (check_recurrence("cnd_gated_recurrence", dtype, outer, steps, inner) != CND_OK ||
      outer == 0 || inner == 0) {
    return 0;
  }
  size_t bytes = 0;
  for (const bool backward : {false, true}) {
    bytes = std::max(bytes, plan_recurrence(dtype, outer, steps, inner, backward).total);
  }
  return bytes;
}

int cnd_gated_recurrence_forward(int32_t dtype, int64_t outer, int64_t steps, int64_t inner,
                                 const void* x, const void* gate, const void* initial, void* y,
                                 void* last, void* states, void* workspace,
                                 size_t workspace_bytes, void* stream_handle) {
  using namespace cnd;
  using namespace cnd::layers;
  clear_error();
  int rc = check_recurrence("cnd_gated_recurrence_forward", dtype, outer, steps, inner);
  if (rc != CND_OK) return rc;
  const int64_t columns = outer * inner;
  if (columns == 0) return CND_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  if (last == nullptr || (steps > 0 && (x == nullptr || gate == nullptr || y == nullptr))) {
    return fail(CND_ERR_INVALID, "cnd_gated_recurrence_forward: a required buffer is NULL");
  }
  if (!aligned_to(element_size(dtype), {x, gate, y}) ||
      !aligned_to(wide_size(dtype), {initial, last, states})) {
    return misaligned("cnd_gated_recurrence_forward");
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
  a.columns = columns;
  const RecurrencePlan p = plan_recurrence(dtype, outer, steps, inner, false);
  rc = bind_exchange("cnd_gated_recurrence_forward", p, workspace, workspace_bytes, &a, stream);
  if (rc != CND_OK) return rc;
  const unsigned grid = recurrence_grid(p);
  const bool vectors = aligned_to(16, {x, gate, y});
  const bool small = columns * std::max<int64_t>(steps, 1) * element_size(dtype) <= UINT32_MAX;
  with_dtype(dtype, [&](auto zero) {
    using T = decltype(zero);
    if (p.along) {
      steps_forward_kernel<T><<<grid, p.warps * 32, 0, stream>>>(a, vectors);
      return;
    }
    const auto run = [&](auto kernel) { kernel<<<grid, p.warps * 32, 0, stream>>>(a); };
    if (sizeof(T) < 8 && pairs_aligned(dtype, inner, {x, gate, y})) {
      return small ? run(columns_forward_kernel<T, true, uint32_t>)
                   : run(columns_forward_kernel<T, true, int64_t>);
    }
    small ? run(columns_forward_kernel<T, false, uint32_t>)
          : run(columns_forward_kernel<T, false, int64_t>);
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
  clear_error();
  int rc = check_recurrence("cnd_gated_recurrence_backward", dtype, outer, steps, inner);
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
  if (!aligned_to(element_size(dtype), {dy, x, gate, dx, dgate}) ||
      !aligned_to(wide_size(dtype), {dlast, states, dinitial})) {
    return misaligned("cnd_gated_recurrence_backward");
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
  a.columns = columns;
  const RecurrencePlan p = plan_recurrence(dtype, outer, steps, inner, true);
  rc = bind_exchange("cnd_gated_recurrence_backward", p, workspace, workspace_bytes, &a, stream);
  if (rc != CND_OK) return rc;
  const unsigned grid = recurrence_grid(p);
  const bool vectors = aligned_to(16, {x, gate, dy, dx, dgate});
  const bool small = columns * std::max<int64_t>(steps, 1) * element_size(dtype) <= UINT32_MAX;
  with_dtype(dtype, [&](auto zero) {
    using T = decltype(zero);
    if (p.along) {
      steps_backward_kernel<T><<<grid, p.warps * 32, 0, stream>>>(a, vectors);
      return;
    }
    const auto run = [&](auto kernel) { kernel<<<grid, p.warps * 32, 0, stream>>>(a); };
    if (sizeof(T) < 8 && pairs_aligned(dtype, inner, {x, gate, dy, dx, dgate})) {
      return small ? run(columns_backward_kernel<T, true, uint32_t>)
                   : run(columns_backward_kernel<T, true, int64_t>);
    }
    small ? run(columns_backward_kernel<T, false, uint32_t>)
          : run(columns_backward_kernel<T, false, int64_t>);
  });
  count_launch();
  return launch_status("cnd_gated_recurrence_backward");
}

}  // extern "C"
