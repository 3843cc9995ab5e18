// The gate of a mixture: the k largest of a row's logits and their softmax weights, and the gradient.
#include "row_common.h"

namespace spnc_hip {
namespace {

// Unsigned keys in the order of the values: NaN above everything, both zeros the same, 0 for "taken out". Keys of 16-bit types
// carry the expert below the value, descending, so that one maximum finds both. They have 29 bits and bit 30, which makes them
// normal positive floats in the same order: v_med3_f32 sorts them into lists.
template <typename T> struct GateKey;
template <> struct GateKey<float> {
  using key = uint32_t;
  static constexpr bool packed = false;
  __device__ static key of(float x, int) {  // not of NaN
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
  }
  __device__ static key ofNan(int) { return 0xFFFFFFFFu; }
  __device__ static float value(key k) {
    return k == 0xFFFFFFFFu ? __uint_as_float(0x7FC00000u) : __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
  }
  __device__ static bool open(key k) { return k > 0x007FFFFFu; }  // above minus infinity
};
template <> struct GateKey<double> {
  using key = uint64_t;
  static constexpr bool packed = false;
  __device__ static key of(double x, int) {
    const uint64_t u = uint64_t(__double_as_longlong(x + 0.0));
    return (u >> 63) ? ~u : u | (1ull << 63);
  }
  __device__ static key ofNan(int) { return ~0ull; }
  __device__ static double value(key k) {
    if (k == ~0ull) return __longlong_as_double(0x7FF8000000000000ll);
    return __longlong_as_double((long long)((k >> 63) ? k ^ (1ull << 63) : ~k));
  }
  __device__ static bool open(key k) { return k > 0x000FFFFFFFFFFFFFull; }
};
struct GateKey16 {
  using key = uint32_t;
  static constexpr bool packed = true;
  // As float these have at most 19 leading bits that are not zero.
  __device__ static key of(float x, int e) {
    const uint32_t u = GateKey<float>::of(x, e);
    return ((u >> 3) & 0x1FFFFC00u) | (0x40000000u | ((1023u - unsigned(e)) & 1023u));
  }
  __device__ static key ofNan(int e) { return 0x5FFFFC00u | ((1023u - unsigned(e)) & 1023u); }
  __device__ static float value(key k) {
    const uint32_t u = (k << 3) & 0xFFFFE000u;
    return u == 0xFFFFE000u ? __uint_as_float(0x7FC00000u) : __uint_as_float((u & 0x80000000u) ? u ^ 0x80000000u : ~(u | 0x1FFFu));
  }
  __device__ static bool open(key k) { return k > 0x400FFFFFu; }  // above minus infinity, whose value is 0x3FF
};
template <> struct GateKey<__bf16> : GateKey16 {};
template <> struct GateKey<_Float16> : GateKey16 {};

// How a row's logits lie in its lanes: one after the other, four at a time where widths and addresses allow it, or, for 16-bit
// types in rows of any width, the two of an aligned word at a time. A row that begins in the middle of a word is `odd`.
enum GateLayout { GATE_SINGLES, GATE_FOURS, GATE_PAIRS };
constexpr int gateStep(int layout) { return layout == GATE_FOURS ? 4 : layout == GATE_PAIRS ? 2 : 1; }

template <typename T>
__device__ inline int gateOdd(const T* row) {
  return int(reinterpret_cast<uintptr_t>(row) / 2) & 1;
}

// The expert of a lane's i-th logit: -1 before an odd row, and past the last expert in the lanes that have none left.
template <int G, int LAYOUT>
__device__ inline int gateExpert(int i, int lane, int odd) {
  constexpr int STEP = gateStep(LAYOUT);
  return i / STEP * (STEP * G) + STEP * lane + i % STEP - (LAYOUT == GATE_PAIRS ? odd : 0);
}

// The rows of a block as a buffer: loads beyond its end return zero without touching memory, so places without an expert need
// no care, and one address with a constant per load serves a lane. Its size is rounded down to `unit` bytes.
typedef __amdgpu_buffer_rsrc_t GateRows;

template <typename T>
__device__ inline GateRows gateRows(const T* first, size_t elements, unsigned unit) {
  const size_t bytes = elements * sizeof(T) / unit * unit;
  // word 3: 32-bit data, no stride
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(first), 0, int(bytes < 0x7FFFFFF0u ? bytes : 0x7FFFFFF0u), 0x00027000);
}

// Steps whose places are experts in every lane: the same for the whole kernel. Opaque, or the comparisons with it would be
// kept from one tile to the next in registers that are not there.
template <int G, int LAYOUT>
__device__ inline int gateWholeSteps(int experts) {
  int steps = experts / (gateStep(LAYOUT) * G);
  asm volatile("" : "+s"(steps));
  return steps;
}
template <int LAYOUT>
__device__ inline bool gateWhole(int i, int steps) {
  return (LAYOUT != GATE_PAIRS || i > 0) && i / gateStep(LAYOUT) < steps;
}

// A row's logits, minus infinity in places without an expert. `at` is where it begins, in elements from the buffer's start.
template <typename T, int G, int V, int LAYOUT>
__device__ inline void gateLoad(GateRows rows, const T* row, unsigned at, int experts, int lane, int odd, bool last, wide_t<T> (&z)[V]) {
  constexpr int STEP = gateStep(LAYOUT);
  constexpr unsigned BYTES = STEP * sizeof(T);
  const int from = int((at + STEP * lane - (LAYOUT == GATE_PAIRS ? odd : 0)) * sizeof(T));
  Pack<T, STEP> raw[V / STEP];
#pragma unroll
  for (int i = 0; i < V / STEP; ++i) {
    const int offset = from + i * int(BYTES * G);
    if constexpr (BYTES == 2) raw[i] = __builtin_bit_cast(Pack<T, STEP>, __builtin_amdgcn_raw_buffer_load_b16(rows, offset, 0, 0));
    if constexpr (BYTES == 4) raw[i] = __builtin_bit_cast(Pack<T, STEP>, __builtin_amdgcn_raw_buffer_load_b32(rows, offset, 0, 0));
    if constexpr (BYTES == 8) raw[i] = __builtin_bit_cast(Pack<T, STEP>, __builtin_amdgcn_raw_buffer_load_b64(rows, offset, 0, 0));
    if constexpr (BYTES == 16) raw[i] = __builtin_bit_cast(Pack<T, STEP>, __builtin_amdgcn_raw_buffer_load_b128(rows, offset, 0, 0));
    if constexpr (BYTES == 32) {
      const Words4 words[2] = {__builtin_amdgcn_raw_buffer_load_b128(rows, offset, 0, 0), __builtin_amdgcn_raw_buffer_load_b128(rows, offset + 16, 0, 0)};
      raw[i] = __builtin_bit_cast(Pack<T, STEP>, words);
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) z[i] = wide_t<T>(raw[i / STEP].v[i % STEP]);
  const int steps = gateWholeSteps<G, LAYOUT>(experts);
#pragma unroll
  for (int i = 0; i < V; i += STEP)
    if (!gateWhole<LAYOUT>(i, steps)) {
#pragma unroll
      for (int q = 0; q < STEP; ++q) {
        const int e = gateExpert<G, LAYOUT>(i + q, lane, odd);
        if (unsigned(e) >= unsigned(experts)) z[i + q] = -INFINITY;
        else if (LAYOUT == GATE_PAIRS && last && e == experts - 1) z[i + q] = wide_t<T>(row[e]);  // half a word at the buffer's end
      }
    }
}

// The largest keys of a lane in descending order, 0 where there are none.
template <int DEPTH>
__device__ inline void gateInsert(uint32_t (&list)[4], uint32_t key) {
#pragma unroll
  for (int d = DEPTH - 1; d > 0; --d)  // the middle of two neighbours and the new key, which is one or the other or the new one
    list[d] = __float_as_uint(__builtin_amdgcn_fmed3f(__uint_as_float(list[d - 1]), __uint_as_float(list[d]), __uint_as_float(key)));
  list[0] = key > list[0] ? key : list[0];
}

// G lanes hold a row, V logits each, so the logits are read once. k rounds: the largest key of the group, the lowest expert that has it, and
// out it goes; lane j keeps the choice of round j, and the softmax is computed by the lanes that have one. Bound by instructions: 262144
// rows of 64 float32, four choices, take 17 us (76 MB, 4.4 TB/s), 65537 of 509 bfloat16, eight choices over all, 26 us (71 MB; 800
// vector instructions a wave of four rows are 21 us of issue). Every round of float32 and float64 looks at all logits again, so the time grows with
// experts times choices: 262144 rows of 128 float32, eight choices, take 47 us, of 256 93, twice what their bytes take.
template <typename T, int G, int V, int LAYOUT>
__global__ __launch_bounds__(BLOCK) void gateKernel(const T* __restrict__ logits, size_t n, unsigned experts, size_t stride, unsigned k,
                                                    unsigned flags, int32_t* __restrict__ index, wide_t<T>* __restrict__ weight) {
  using R = wide_t<T>;
  using O = GateKey<T>;
  using K = typename O::key;
  const int lane = threadIdx.x % G;
  forTiles((n + BLOCK / G - 1) / (BLOCK / G), gridDim.x, false, [&](size_t tile) {
    const size_t row = tile * (BLOCK / G) + threadIdx.x / G;
    if (row >= n) return;  // whole groups leave; lanes are paired inside a group
    const T* const from = logits + row * stride;
    const int odd = LAYOUT == GATE_PAIRS ? gateOdd(from) : 0;
    const size_t first = tile * (BLOCK / G);
    const GateRows rows = gateRows(logits + first * stride, (n - 1 - first) * stride + experts, gateStep(LAYOUT) * sizeof(T));
    R z[V];
    gateLoad<T, G, V, LAYOUT>(rows, from, unsigned(threadIdx.x / G) * unsigned(stride), experts, lane, odd, row == n - 1, z);
    K key[V];
    bool nan = false;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      key[i] = O::of(z[i], gateExpert<G, LAYOUT>(i, lane, odd));
      nan |= z[i] != z[i];
    }
    if (nan) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (z[i] != z[i]) key[i] = O::ofNan(gateExpert<G, LAYOUT>(i, lane, odd));
    }
    K myKey = 0, topKey = 0;
    int myIndex = 0;
    R total = 0;
    [[maybe_unused]] uint32_t list[4] = {};
    if constexpr (O::packed) {
      // Every lane's four largest (two, if no more are asked for): four instructions a logit, after which a round only looks at the
      // lists' heads. A lane that has more of the k largest than its list holds makes a new one of what is below.
      if (k > 2) {
#pragma unroll
        for (int i = 0; i < V; ++i) gateInsert<4>(list, key[i]);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) gateInsert<2>(list, key[i]);
      }
    }
    for (int j = 0; j < int(k); ++j) {
      K best = 0;
      int at = 0;
      if constexpr (O::packed) {
        best = groupMax<G>(list[0]);
        at = 1023 - int(best & 1023u);
        if (list[0] == best) {  // keys are distinct: one lane
          list[0] = list[1], list[1] = list[2], list[2] = list[3], list[3] = 0;
          if (V > 4 && list[0] == 0 && j + 1 < int(k)) {
#pragma unroll
            for (int i = 0; i < V; ++i) gateInsert<4>(list, key[i] < best ? key[i] : 0u);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) best = key[i] > best ? key[i] : best;
        best = groupMax<G>(best);
        at = INT32_MAX;
#pragma unroll
        for (int i = V - 1; i >= 0; --i) at = key[i] == best ? gateExpert<G, LAYOUT>(i, lane, odd) : at;
        at = groupMin<G>(at);
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (gateExpert<G, LAYOUT>(i, lane, odd) == at) key[i] = 0;
      }
      if (j == 0) {
        topKey = best;
        if ((flags & SPNC_HIP_GATE_ALL) && O::open(best)) {
          const R top = O::value(best);
#pragma unroll
          for (int i = 0; i < V; ++i) total += expTerm(z[i] - top);
          total = groupSum<G>(total);
        }
      }
      if (lane == j) myKey = best, myIndex = at;
    }
    const bool open = lane < int(k) && O::open(myKey);
    const R shifted = open ? O::value(myKey) - O::value(topKey) : R(0);
    const R e = open ? expOf(shifted) : R(0);
    if (!(flags & SPNC_HIP_GATE_ALL)) total = groupSum<G>(e);
    if (lane < int(k)) {
      index[row * k + lane] = open ? myIndex : -1;
      weight[row * k + lane] = (flags & SPNC_HIP_GATE_LOG) ? (open ? shifted - logOf(total) : R(-INFINITY)) : open ? e / total : R(0);
    }
  });
}

// dz_e of the experts that were not chosen is 0, or -p_e times the sum over the slots under "all"; the k chosen ones get their
// slot's term on top. A block's rows are one stretch of the output. It is put together in LDS, the chosen entries over the others,
// and goes out 16 bytes a lane whatever the width of a row: 65537 rows of 509 bfloat16 take 29 us, 40 if every group
// writes its own row.
template <typename T, int G, int V, int LAYOUT>
__global__ __launch_bounds__(BLOCK) void gateBackwardKernel(const T* __restrict__ logits, size_t n, unsigned experts, size_t stride, unsigned k,
                                                            unsigned flags, const int32_t* __restrict__ index, const wide_t<T>* __restrict__ weight,
                                                            const wide_t<T>* __restrict__ gradWeight, T* __restrict__ gradLogits) {
  using R = wide_t<T>;
  constexpr int ROWS = BLOCK / G, E16 = 16 / sizeof(T);
  __shared__ alignas(16) T stretch[ROWS * V * G + E16];
  const int lane = threadIdx.x % G, local = threadIdx.x / G;
  const bool all = flags & SPNC_HIP_GATE_ALL, logs = flags & SPNC_HIP_GATE_LOG;
  forTiles((n + ROWS - 1) / ROWS, gridDim.x, false, [&](size_t tile) {
    const size_t row = tile * ROWS + local;
    const int rows = n - tile * ROWS < size_t(ROWS) ? int(n - tile * ROWS) : ROWS;
    T* const to = gradLogits + tile * ROWS * experts;
    const int skew = int(reinterpret_cast<uintptr_t>(to) % 16 / sizeof(T));  // LDS is aligned as the output is
    T* const mine = stretch + skew + local * int(experts);
    if (row < n) {
      int32_t at = -1;
      R d = 0, w = 0;
      if (lane < int(k)) {
        at = index[row * k + lane];
        if (at >= int32_t(experts)) at = -1;
        if (at >= 0) {
          d = gradWeight[row * k + lane];
          w = weight[row * k + lane];
          if (logs) w = expOf(w);
          else d *= w;
        }
      }
      const R common = groupSum<G>(d);
      if (all) {
        R z[V];
        const T* const from = logits + row * stride;
        const int32_t first = index[row * k];  // the largest logit's, or NaN's; none: closed altogether
        const bool any = first >= 0 && first < int32_t(experts);
        const int odd = LAYOUT == GATE_PAIRS ? gateOdd(from) : 0;
        const GateRows buffer = gateRows(logits + tile * ROWS * stride, (n - 1 - tile * ROWS) * stride + experts, gateStep(LAYOUT) * sizeof(T));
        gateLoad<T, G, V, LAYOUT>(buffer, from, unsigned(local) * unsigned(stride), experts, lane, odd, row == n - 1, z);
        const R top = any ? R(from[first]) : R(0);
        R total = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          z[i] = sizeof(T) == 2 ? expTerm(z[i] - top) : expOf(z[i] - top);
          total += z[i];
        }
        total = groupSum<G>(total);
        const R factor = total == 0 ? R(0) : -common / total;
        const int steps = gateWholeSteps<G, LAYOUT>(experts);
#pragma unroll
        for (int i = 0; i < V; i += gateStep(LAYOUT)) {
          const int e = gateExpert<G, LAYOUT>(i, lane, odd);
          if constexpr (LAYOUT == GATE_FOURS) {
            const Pack<T, 4> p{{T(z[i] * factor), T(z[i + 1] * factor), T(z[i + 2] * factor), T(z[i + 3] * factor)}};
            if (e < int(experts)) *reinterpret_cast<Pack<T, 4>*>(mine + e) = p;
          } else if (gateWhole<LAYOUT>(i, steps)) {
#pragma unroll
            for (int q = 0; q < gateStep(LAYOUT); ++q) mine[e + q] = T(z[i + q] * factor);
          } else {
#pragma unroll
            for (int q = 0; q < gateStep(LAYOUT); ++q)
              if (unsigned(e + q) < experts) mine[e + q] = T(z[i + q] * factor);
          }
        }
      } else {
        constexpr int STEP = LAYOUT == GATE_FOURS ? 4 : 1;
#pragma unroll
        for (int i = 0; i < V; i += STEP) {
          const int e = i * G + STEP * lane;
          if (e < int(experts)) *reinterpret_cast<Pack<T, STEP>*>(mine + e) = Pack<T, STEP>{};
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the group is part of one wave, whose LDS accesses stay in order
      if (at >= 0) mine[at] = T(d - w * common);
    }
    __syncthreads();
    const int begin = skew, end = skew + rows * int(experts);
    for (int i = int(threadIdx.x) * E16; i < end; i += BLOCK * E16) {
      if (i >= begin && i + E16 <= end) {
        *reinterpret_cast<Pack<T, E16>*>(to + (i - skew)) = *reinterpret_cast<const Pack<T, E16>*>(stretch + i);
      } else {
#pragma unroll
        for (int q = 0; q < E16; ++q)
          if (i + q >= begin && i + q < end) to[i + q - skew] = stretch[i + q];
      }
    }
    __syncthreads();
  });
}

constexpr size_t GATE_MANY_ROWS = 8192;
constexpr size_t GATE_MAX_STRIDE = 1u << 20;  // a block's rows, 256 at the most, lie within 2^31 bytes

// calls fn(G, V, LAYOUT): a row's logits in G lanes of V, at least as many lanes as choices. A round costs a wave about 5 V + 14
// instructions (3 V / 2 + 14 with packed keys) for 64 / G rows, so with many rows few lanes of many logits are cheapest, as far as the
// registers go; with few rows a row is spread over as many lanes as have four logits, which is done sooner.
template <typename T, typename Fn>
void withGateShape(size_t n, unsigned experts, unsigned k, size_t stride, uintptr_t addresses, Fn&& fn) {
  constexpr bool packed = sizeof(T) == 2;
  const bool fours = (experts | stride) % 4 == 0 && addresses % alignof(Pack<T, 4>) == 0;
  const bool pairs = packed && !fours && experts >= 16 && experts < SPNC_HIP_MAX_EXPERTS && addresses % 4 == 0;
  const unsigned places = experts + (pairs ? 1 : 0);  // an odd row's first word begins a place earlier
  unsigned group = 0, logits = 0, best = ~0u;
  for (unsigned v : {4u, 8u, 16u, 32u}) {
    if ((v > 16 && !packed) || (v > 4 && (sizeof(T) == 8 || n < GATE_MANY_ROWS) && places <= 256)) continue;
    unsigned g = 1;
    while (g < WAVE && (v * g < places || g < k)) g *= 2;
    if (v * g < places || (v == 8 && (g < 2 || sizeof(T) == 8) && g < WAVE) || (v == 16 && g < (sizeof(T) == 8 ? WAVE : 2)) || (v == 32 && (g < 4 || g > 32))) continue;
    const unsigned cost = n < GATE_MANY_ROWS ? v : packed ? g * (3 * v + 28) : g * (10 * v + 28);
    if (cost < best) group = g, logits = v, best = cost;
  }
  auto shape = [&](auto g, auto v) {
    if (fours) return fn(g, v, std::integral_constant<int, GATE_FOURS>());
    if constexpr (packed)
      if (pairs) return fn(g, v, std::integral_constant<int, GATE_PAIRS>());
    fn(g, v, std::integral_constant<int, GATE_SINGLES>());
  };
#define SPN_GATE_SHAPE(G, V) \
  if (group == G && logits == V) return shape(std::integral_constant<int, G>(), std::integral_constant<int, V>())
  SPN_GATE_SHAPE(1, 4);
  SPN_GATE_SHAPE(2, 4);
  SPN_GATE_SHAPE(4, 4);
  SPN_GATE_SHAPE(8, 4);
  SPN_GATE_SHAPE(16, 4);
  SPN_GATE_SHAPE(32, 4);
  SPN_GATE_SHAPE(64, 4);
  SPN_GATE_SHAPE(64, 8);
  SPN_GATE_SHAPE(64, 16);
  if constexpr (sizeof(T) < 8) {
    SPN_GATE_SHAPE(2, 8);
    SPN_GATE_SHAPE(4, 8);
    SPN_GATE_SHAPE(8, 8);
    SPN_GATE_SHAPE(16, 8);
    SPN_GATE_SHAPE(32, 8);
    SPN_GATE_SHAPE(2, 16);
    SPN_GATE_SHAPE(4, 16);
    SPN_GATE_SHAPE(8, 16);
    SPN_GATE_SHAPE(16, 16);
    SPN_GATE_SHAPE(32, 16);
  }
  if constexpr (packed) {
    SPN_GATE_SHAPE(4, 32);
    SPN_GATE_SHAPE(8, 32);
    SPN_GATE_SHAPE(16, 32);
    SPN_GATE_SHAPE(32, 32);
  }
#undef SPN_GATE_SHAPE
  refuse("no gate kernel for this shape");
}

void checkGate(int dtype, size_t n, unsigned experts, size_t stride, unsigned k, unsigned flags) {
  elementBytes(dtype);
  checkExperts(experts);
  if (k == 0 || k > experts || k > SPNC_HIP_MAX_CHOICES)
    refuse("k must be between 1 and the number of experts, at most " + std::to_string(SPNC_HIP_MAX_CHOICES));
  if (n > 1 && stride < experts) refuse("rows of logits overlap");
  if (stride >= GATE_MAX_STRIDE) refuse("rows of logits must be less than 2^20 elements apart");
  if (flags & ~unsigned(SPNC_HIP_GATE_ALL | SPNC_HIP_GATE_LOG)) refuse("unknown gate flags");
}

}  // namespace
}  // namespace spnc_hip

using namespace spnc_hip;

extern "C" {

int spnc_hip_gate(const void* logits, int dtype, size_t n, unsigned experts, size_t stride, unsigned k, unsigned flags, int32_t* index,
                  void* weight, void* stream) {
  return guarded([&] {
    checkGate(dtype, n, experts, stride, k, flags);
    if (n == 0) return;
    if (!logits || !index || !weight) refuse("null argument");
    if (address(logits) % elementBytes(dtype)) refuse("gate: pointers are not aligned to the element type");
    const size_t bytes = elementBytes(dtype), slots = n * k;
    const Span read{logits, n, experts * bytes, stride * bytes}, chosen = block(index, slots * sizeof(int32_t));
    const Span weights = block(weight, slots * (bytes < sizeof(float) ? sizeof(float) : bytes));
    checkApart("gate", chosen, {read, weights});
    checkApart("gate", weights, {read});
    withType(dtype, [&](auto t) {
      using T = decltype(t);
      withGateShape<T>(n, experts, k, stride, address(logits), [&](auto g, auto v, auto layout) {
        constexpr int G = decltype(g)::value, V = decltype(v)::value;
        launch("gate", gateKernel<T, G, V, decltype(layout)::value>, tileGrid((n + BLOCK / G - 1) / (BLOCK / G)), BLOCK, 0, stream,
               static_cast<const T*>(logits), n, experts, stride, k, flags, index, static_cast<wide_t<T>*>(weight));
      });
    });
  });
}

int spnc_hip_gate_backward(const void* logits, int dtype, size_t n, unsigned experts, size_t stride, unsigned k, unsigned flags,
                           const int32_t* index, const void* weight, const void* grad_weight, void* grad_logits, void* stream) {
  return guarded([&] {
    checkGate(dtype, n, experts, stride, k, flags);
    if (n == 0) return;
    if ((!logits && (flags & SPNC_HIP_GATE_ALL)) || !index || !weight || !grad_weight || !grad_logits) refuse("null argument");
    if ((address(logits) | address(grad_logits)) % elementBytes(dtype)) refuse("gate gradient: pointers are not aligned to the element type");
    const size_t bytes = elementBytes(dtype), slots = n * k, weightBytes = slots * (bytes < sizeof(float) ? sizeof(float) : bytes);
    checkApart("gate gradient", block(grad_logits, n * experts * bytes),
               {{logits, (flags & SPNC_HIP_GATE_ALL) ? n : 0, experts * bytes, stride * bytes}, block(index, slots * sizeof(int32_t)),
                block(weight, weightBytes), block(grad_weight, weightBytes)});
    withType(dtype, [&](auto t) {
      using T = decltype(t);
      using R = wide_t<T>;
      withGateShape<T>(n, experts, k, (flags & SPNC_HIP_GATE_ALL) ? stride : experts,
                       address(grad_logits) | ((flags & SPNC_HIP_GATE_ALL) ? address(logits) : 0), [&](auto g, auto v, auto layout) {
        constexpr int G = decltype(g)::value, V = decltype(v)::value;
        launch("gate gradient", gateBackwardKernel<T, G, V, decltype(layout)::value>, tileGrid((n + BLOCK / G - 1) / (BLOCK / G)), BLOCK, 0, stream,
               static_cast<const T*>(logits), n, experts, stride, k, flags, index, static_cast<const R*>(weight), static_cast<const R*>(grad_weight),
               static_cast<T*>(grad_logits));
      });
    });
  });
}

}  // extern "C"
