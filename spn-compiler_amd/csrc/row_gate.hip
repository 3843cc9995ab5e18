// The gate of a mixture: the k largest of a row's logits and their softmax weights, and the gradient.
#include "row_common.h"

namespace spnc_hip {
namespace {

// Unsigned keys in the order of the values: NaN above everything, both zeros the same, 0 for "taken out". Keys of 16-bit types
// carry the expert below the value, descending, so that one maximum finds both; 29 bits in all.
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
    return ((u >> 3) & 0x1FFFFC00u) | ((1023u - unsigned(e)) & 1023u);
  }
  __device__ static key ofNan(int e) { return 0x1FFFFC00u | ((1023u - unsigned(e)) & 1023u); }
  __device__ static float value(key k) {
    const uint32_t u = k >> 10 << 13;
    return (k >> 10) == 0x7FFFFu ? __uint_as_float(0x7FC00000u) : __uint_as_float((u & 0x80000000u) ? u ^ 0x80000000u : ~(u | 0x1FFFu));
  }
  __device__ static bool open(key k) { return k >> 10 > 0x007FFFFFu >> 13; }
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

// A row's logits, minus infinity in places without an expert. All loads are unconditional (a place past the end reads the last
// one), so that they are under way together. A word at the border of a row reaches into the row beside it, which the first and
// the last row do not have: `edge` reads those one by one.
template <typename T, int G, int V, int LAYOUT>
__device__ inline void gateLoad(const T* row, int experts, int lane, int odd, bool edge, wide_t<T> (&z)[V]) {
  T raw[V];
  auto single = [&](int i) {
    const int e = gateExpert<G, LAYOUT>(i, lane, odd);
    raw[i] = row[e < 0 ? 0 : e < experts ? e : experts - 1];
  };
  if constexpr (LAYOUT == GATE_FOURS) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const int e = gateExpert<G, LAYOUT>(i, lane, odd);
      const Pack<T, 4> p = *reinterpret_cast<const Pack<T, 4>*>(row + (e < experts ? e : experts - 4));
#pragma unroll
      for (int q = 0; q < 4; ++q) raw[i + q] = p.v[q];
    }
  } else if constexpr (LAYOUT == GATE_PAIRS) {
    if (edge) {
#pragma unroll
      for (int i = 0; i < V; ++i) single(i);
    } else {
      const int last = ((experts - 1 + odd) & ~1) - odd;
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        const int e = gateExpert<G, LAYOUT>(i, lane, odd);
        const Pack<T, 2> p = *reinterpret_cast<const Pack<T, 2>*>(row + (e < last ? e : last));
        raw[i] = p.v[0], raw[i + 1] = p.v[1];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) single(i);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) z[i] = unsigned(gateExpert<G, LAYOUT>(i, lane, odd)) < unsigned(experts) ? wide_t<T>(raw[i]) : wide_t<T>(-INFINITY);
}

// G lanes hold a row, V logits each. k rounds: the largest key of the group, the lowest expert that has it, and out it goes; lane
// j keeps the choice of round j. The whole row is in registers, so the logits are read once.
template <typename T, int G, int V, int LAYOUT>
__global__ __launch_bounds__(BLOCK) void gateKernel(const T* __restrict__ logits, size_t n, unsigned experts, size_t stride, unsigned k,
                                                    unsigned flags, int32_t* __restrict__ index, wide_t<T>* __restrict__ weight) {
  using R = wide_t<T>;
  using O = GateKey<T>;
  using K = typename O::key;
  const int lane = threadIdx.x % G;
  forTiles((n + BLOCK / G - 1) / (BLOCK / G), gridDim.x, [&](size_t tile) {
    const size_t row = tile * (BLOCK / G) + threadIdx.x / G;
    if (row >= n) return;  // whole groups leave; lanes are paired inside a group
    const T* const from = logits + row * stride;
    const int odd = LAYOUT == GATE_PAIRS ? gateOdd(from) : 0;
    R z[V];
    gateLoad<T, G, V, LAYOUT>(from, experts, lane, odd, row == 0 || row == n - 1, z);
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
    K myKey = 0, topKey = 0, last = 0;
    int myIndex = 0;
    R total = 0;
    for (int j = 0; j < int(k); ++j) {
      K best = 0;
      int at = 0;
      if constexpr (O::packed) {
        // Keys are distinct and have 29 bits: modulo 2^32, key - last is above 2^31 for keys below the last choice and below 2^29
        // for the others, so its maximum belongs to the largest key below, and nothing has to be taken out.
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const K below = j == 0 ? key[i] : key[i] - last;
          best = below > best ? below : best;
        }
        best = groupMax<G>(best);
        best = j == 0 ? best : best >> 31 ? best + last : K(0);
        last = best ? best : last;
        at = 1023 - int(best & 1023u);
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
// slot's term on top, through LDS: every lane has V of the row's entries in registers, and a slot's expert may be any of them.
template <typename T, int G, int V, int LAYOUT>
__global__ __launch_bounds__(BLOCK) void gateBackwardKernel(const T* __restrict__ logits, size_t n, unsigned experts, size_t stride, unsigned k,
                                                            unsigned flags, const int32_t* __restrict__ index, const wide_t<T>* __restrict__ weight,
                                                            const wide_t<T>* __restrict__ gradWeight, T* __restrict__ gradLogits) {
  using R = wide_t<T>;
  __shared__ R entries[BLOCK / G][V * G];
  const int lane = threadIdx.x % G;
  R* const mine = entries[threadIdx.x / G];
  const bool all = flags & SPNC_HIP_GATE_ALL, logs = flags & SPNC_HIP_GATE_LOG;
  forTiles((n + BLOCK / G - 1) / (BLOCK / G), gridDim.x, [&](size_t tile) {
    const size_t row = tile * (BLOCK / G) + threadIdx.x / G;
    if (row >= n) return;
    int32_t at = -1;
    R d = 0, w = 0;
    if (lane < int(k)) {
      at = index[row * k + lane];
      if (at >= int32_t(experts)) at = -1;
      if (at >= 0) {
        d = gradWeight[row * k + lane];
        w = weight[row * k + lane];
        if (logs) w = w == -INFINITY ? R(0) : expOf(w);
        else d *= w;
      }
    }
    R dz[V] = {};
    R total = 0;
    int odd = 0;  // any layout of the entries will do without logits
    const int32_t first = all ? index[row * k] : -1;  // the largest logit's, or NaN's; none: closed altogether
    if (first >= 0 && first < int32_t(experts)) {
      const T* const from = logits + row * stride;
      const R top = R(from[first]);
      if (LAYOUT == GATE_PAIRS) odd = gateOdd(from);
      gateLoad<T, G, V, LAYOUT>(from, experts, lane, odd, row == 0 || row == n - 1, dz);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        dz[i] = sizeof(T) == 2 ? expTerm(dz[i] - top) : expOf(dz[i] - top);
        total += dz[i];
      }
      total = groupSum<G>(total);
    }
    const R common = groupSum<G>(d);
    if (!all) d -= w * common;
    const R factor = total == 0 ? R(0) : -common / total;
#pragma unroll
    for (int i = 0; i < V; i += gateStep(LAYOUT)) {
      const int e = gateExpert<G, LAYOUT>(i, lane, odd);
      if constexpr (LAYOUT == GATE_FOURS) {
        Pack<R, 4> p;
#pragma unroll
        for (int q = 0; q < 4; ++q) p.v[q] = dz[i + q] * factor;
        *reinterpret_cast<Pack<R, 4>*>(mine + e) = p;
      } else {
#pragma unroll
        for (int q = 0; q < gateStep(LAYOUT); ++q)
          if (unsigned(e + q) < experts) mine[e + q] = dz[i + q] * factor;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the group is part of one wave, whose LDS accesses stay in order
    if (at >= 0) mine[at] += d;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    T* const to = gradLogits + row * experts;
    if (LAYOUT == GATE_PAIRS) odd = gateOdd(to);
#pragma unroll
    for (int i = 0; i < V; i += gateStep(LAYOUT)) {
      const int e = gateExpert<G, LAYOUT>(i, lane, odd);
      if constexpr (LAYOUT == GATE_FOURS) {
        const Pack<R, 4> p = *reinterpret_cast<const Pack<R, 4>*>(mine + e);
        Pack<T, 4> o;
#pragma unroll
        for (int q = 0; q < 4; ++q) o.v[q] = T(p.v[q]);
        if (e < int(experts)) *reinterpret_cast<Pack<T, 4>*>(to + e) = o;
      } else if constexpr (LAYOUT == GATE_PAIRS) {
        if (e >= 0 && e + 1 < int(experts)) *reinterpret_cast<Pack<T, 2>*>(to + e) = Pack<T, 2>{{T(mine[e]), T(mine[e + 1])}};
        else if (unsigned(e) < experts) to[e] = T(mine[e]);
        else if (unsigned(e + 1) < experts) to[e + 1] = T(mine[e + 1]);
      } else if (e < int(experts)) {
        to[e] = T(mine[e]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  });
}

constexpr size_t GATE_MANY_ROWS = 8192;

// calls fn(G, V, LAYOUT): a row's logits in G lanes of V, at least as many lanes as choices. A round costs a wave about 5 V + 14
// instructions (3 V / 2 + 14 with packed keys) for 64 / G rows, so with many rows few lanes of many logits are cheapest, as far as the
// registers go; with few rows a row is spread over as many lanes as have four logits, which is done sooner.
template <typename T, typename Fn>
void withGateShape(size_t n, unsigned experts, unsigned k, size_t stride, uintptr_t addresses, Fn&& fn) {
  constexpr bool packed = sizeof(T) == 2;
  const bool fours = (experts | stride) % 4 == 0 && addresses % alignof(Pack<T, 4>) == 0;
  const bool pairs = packed && !fours && experts >= 16 && experts < SPNC_HIP_MAX_EXPERTS;
  const unsigned places = experts + (pairs ? 1 : 0);  // an odd row's first word begins a place earlier
  unsigned group = 0, logits = 0, best = ~0u;
  for (unsigned v : {4u, 8u, 16u, 32u}) {
    if ((v == 8 && places <= 256) || (v > 16 && !packed) || (v > 4 && (sizeof(T) == 8 || n < GATE_MANY_ROWS) && places <= 256)) continue;
    unsigned g = 1;
    while (g < WAVE && (v * g < places || g < k)) g *= 2;
    if (v * g < places || (v == 8 && g < WAVE) || (v == 16 && g < (sizeof(T) == 8 ? WAVE : 2)) || (v == 32 && (g < 4 || g > 32))) continue;
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
    withType(dtype, [&](auto t) {
      using T = decltype(t);
      withGateShape<T>(n, experts, k, stride, address(logits), [&](auto g, auto v, auto layout) {
        constexpr int G = decltype(g)::value, V = decltype(v)::value;
        gateKernel<T, G, V, decltype(layout)::value><<<tileGrid((n + BLOCK / G - 1) / (BLOCK / G)), BLOCK, 0, static_cast<hipStream_t>(stream)>>>(
            static_cast<const T*>(logits), n, experts, stride, k, flags, index, static_cast<wide_t<T>*>(weight));
      });
    });
    launched("gate");
  });
}

int spnc_hip_gate_backward(const void* logits, int dtype, size_t n, unsigned experts, size_t stride, unsigned k, unsigned flags,
                           const int32_t* index, const void* weight, const void* grad_weight, void* grad_logits, void* stream) {
  return guarded([&] {
    checkGate(dtype, n, experts, stride, k, flags);
    if (n == 0) return;
    if ((!logits && (flags & SPNC_HIP_GATE_ALL)) || !index || !weight || !grad_weight || !grad_logits) refuse("null argument");
    withType(dtype, [&](auto t) {
      using T = decltype(t);
      using R = wide_t<T>;
      withGateShape<T>(n, experts, k, (flags & SPNC_HIP_GATE_ALL) ? stride : experts,
                       address(grad_logits) | ((flags & SPNC_HIP_GATE_ALL) ? address(logits) : 0), [&](auto g, auto v, auto layout) {
        constexpr int G = decltype(g)::value, V = decltype(v)::value;
        gateBackwardKernel<T, G, V, decltype(layout)::value><<<tileGrid((n + BLOCK / G - 1) / (BLOCK / G)), BLOCK, 0, static_cast<hipStream_t>(stream)>>>(
            static_cast<const T*>(logits), n, experts, stride, k, flags, index, static_cast<const R*>(weight), static_cast<const R*>(grad_weight),
            static_cast<T*>(grad_logits));
      });
    });
    launched("gate gradient");
  });
}

}  // extern "C"
