// Operators on device-resident rows around compiled kernels (include/spnc_hip_rows.h): gate, routing, combination,
// dropout. Device code, launch shapes and the extern "C" entry points.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "../../include/spnc_hip_rows.h"
#include "guard.h"
#include "philox.h"

namespace spnc_hip {
namespace {

constexpr unsigned WAVE = 64;
constexpr unsigned BLOCK = 256;
constexpr unsigned XCDS = 8;             // blocks go to the chip's dies in turn
constexpr size_t MAX_GRID = 1u << 22;    // a launch must stay below 2^32 threads

template <typename T> struct Wide { using type = float; };
template <> struct Wide<double> { using type = double; };
template <typename T> using wide_t = typename Wide<T>::type;

template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
  T v[N];
};

// Accesses that are not kept in the caches. A piece of another size than 16 bytes goes the ordinary way.
typedef uint32_t Words4 __attribute__((ext_vector_type(4)));

template <typename P>
__device__ inline P streamLoad(const P* p) {
  if constexpr (sizeof(P) == 16) return __builtin_bit_cast(P, __builtin_nontemporal_load(reinterpret_cast<const Words4*>(p)));
  else return *p;
}

template <typename P>
__device__ inline void streamStore(P* p, const P& v) {
  if constexpr (sizeof(P) == 16) __builtin_nontemporal_store(__builtin_bit_cast(Words4, v), reinterpret_cast<Words4*>(p));
  else *p = v;
}

// Neighbouring tiles of rows go to one die: rows that are neighbours in the sorted buffer come from neighbouring rows,
// and a cache line of narrow rows is then filled or read within one L2.
template <typename Body>
__device__ inline void forTiles(size_t tiles, unsigned grid, Body&& body) {
  const size_t perDie = (tiles + XCDS - 1) / XCDS, first = size_t(blockIdx.x % XCDS) * perDie;
  for (size_t t = blockIdx.x / XCDS; t < perDie; t += grid / XCDS)
    if (first + t < tiles) body(first + t);
}

unsigned tileGrid(size_t tiles) {
  const size_t g = (tiles + XCDS - 1) / XCDS * XCDS;
  return unsigned(g < MAX_GRID ? g : MAX_GRID);
}

// ---- lanes ----------------------------------------------------------------------------------------------------------

// For a lane, its word and that of the lane it is paired with at distance D, in an order that is the same for both lanes or
// does not matter to a symmetric operation. D = 4 and 8 mirror instead of exchanging: all lanes at smaller distances must hold the
// same already. Vector instructions throughout (DPP, and row swaps of gfx950 for 16 and 32), no LDS.
template <int D>
__device__ inline void lanePair(uint32_t x, uint32_t& a, uint32_t& b) {
  if constexpr (D <= 8) {
    constexpr int control = D == 1 ? 0xB1 : D == 2 ? 0x4E : D == 4 ? 0x141 : 0x140;  // quad_perm, half row and row mirror
    a = x;
    b = uint32_t(__builtin_amdgcn_update_dpp(0, int(x), control, 0xF, 0xF, true));
  } else if constexpr (D == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    a = r[0], b = r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    a = r[0], b = r[1];
  }
}

template <int D, int G, typename R, typename Op>
__device__ inline R groupFrom(R x, Op op) {
  if constexpr (D >= G) {
    return x;
  } else {
    R a, b;
    if constexpr (sizeof(R) == 4) {
      uint32_t wa, wb;
      lanePair<D>(__builtin_bit_cast(uint32_t, x), wa, wb);
      a = __builtin_bit_cast(R, wa), b = __builtin_bit_cast(R, wb);
    } else {
      const uint64_t w = __builtin_bit_cast(uint64_t, x);
      uint32_t la, lb, ha, hb;
      lanePair<D>(uint32_t(w), la, lb);
      lanePair<D>(uint32_t(w >> 32), ha, hb);
      a = __builtin_bit_cast(R, uint64_t(ha) << 32 | la), b = __builtin_bit_cast(R, uint64_t(hb) << 32 | lb);
    }
    return groupFrom<D * 2, G>(op(a, b), op);
  }
}

// The sum, maximum or minimum over a group of G lanes, in all of them.
template <int G, typename R> __device__ inline R groupSum(R x) {
  return groupFrom<1, G>(x, [](R a, R b) { return a + b; });
}
template <int G, typename R> __device__ inline R groupMax(R x) {
  return groupFrom<1, G>(x, [](R a, R b) { return a > b ? a : b; });
}
template <int G, typename R> __device__ inline R groupMin(R x) {
  return groupFrom<1, G>(x, [](R a, R b) { return a < b ? a : b; });
}

// exp(x): x log2(e) in two parts, the hardware's exp2 of the first, the second as a factor 1 + r ln 2. Within two units in the
// last place; below exp(-87) the result is 0.
__device__ inline float expOf(float x) {
  x = x < -200.0f ? -200.0f : x;  // minus infinity has no second part
  const float t = x * 1.44269502f, r = __builtin_fmaf(x, 1.92596299e-8f, __builtin_fmaf(x, 1.44269502f, -t));
  const float y = __builtin_amdgcn_exp2f(t);
  return __builtin_fmaf(y, r * 0.693147182f, y);
}
__device__ inline double expOf(double x) { return exp(x); }
__device__ inline float logOf(float x) { return logf(x); }
__device__ inline double logOf(double x) { return log(x); }

// ---- gate -----------------------------------------------------------------------------------------------------------

// Unsigned keys in the order of the values: NaN above everything, both zeros the same, 0 for "no value". Keys of 16-bit types
// carry the expert below the value, descending, so that one maximum finds both; 26 bits in all.
template <typename T> struct GateKey;
template <> struct GateKey<float> {
  using key = uint32_t;
  static constexpr bool packed = false;
  __device__ static key of(float x, unsigned) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return x != x ? 0xFFFFFFFFu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  }
  __device__ static float value(key k) {
    return k == 0xFFFFFFFFu ? __uint_as_float(0x7FC00000u) : __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
  }
  __device__ static bool open(key k) { return k > 0x007FFFFFu; }  // above minus infinity
};
template <> struct GateKey<double> {
  using key = uint64_t;
  static constexpr bool packed = false;
  __device__ static key of(double x, unsigned) {
    const uint64_t u = uint64_t(__double_as_longlong(x + 0.0));
    return x != x ? ~0ull : (u >> 63) ? ~u : u | (1ull << 63);
  }
  __device__ static double value(key k) {
    if (k == ~0ull) return __longlong_as_double(0x7FF8000000000000ll);
    return __longlong_as_double((long long)((k >> 63) ? k ^ (1ull << 63) : ~k));
  }
  __device__ static bool open(key k) { return k > 0x000FFFFFFFFFFFFFull; }
};
template <typename T, uint32_t INF> struct GateKey16 {
  using key = uint32_t;
  static constexpr bool packed = true;
  __device__ static key of(T x, unsigned e) {
    uint32_t u = __builtin_bit_cast(uint16_t, x);
    const bool nan = (u & 0x7FFFu) > INF;
    u = u == 0x8000u ? 0u : u;
    u = nan ? 0xFFFFu : (u & 0x8000u) ? u ^ 0xFFFFu : u | 0x8000u;
    return u << 10 | (1023u - e);
  }
  __device__ static float value(key k) {
    const uint32_t u = k >> 10;
    const float x = float(__builtin_bit_cast(T, uint16_t((u & 0x8000u) ? u ^ 0x8000u : u ^ 0xFFFFu)));
    return u == 0xFFFFu ? __uint_as_float(0x7FC00000u) : x;
  }
  __device__ static bool open(key k) { return k >> 10 > (INF ^ 0x7FFFu); }
};
template <> struct GateKey<__bf16> : GateKey16<__bf16, 0x7F80u> {};
template <> struct GateKey<_Float16> : GateKey16<_Float16, 0x7C00u> {};

// The expert of a lane's i-th logit. VEC: read four at a time.
template <int G, bool VEC>
__device__ inline unsigned gateExpert(int i, unsigned lane) {
  return VEC ? (i / 4) * (4 * G) + 4 * lane + i % 4 : i * G + lane;
}

template <typename T, int G, int V, bool VEC>
__device__ inline void gateLoad(const T* row, unsigned experts, unsigned lane, T (&z)[V]) {
#pragma unroll
  for (int i = 0; i < V; i += VEC ? 4 : 1) {
    const unsigned e = gateExpert<G, VEC>(i, lane);
    if constexpr (VEC) {
      if (e < experts) {
        const Pack<T, 4> p = *reinterpret_cast<const Pack<T, 4>*>(row + e);
#pragma unroll
        for (int q = 0; q < 4; ++q) z[i + q] = p.v[q];
      }
    } else if (e < experts) {
      z[i] = row[e];
    }
  }
}

// G lanes hold a row, V logits each. k rounds: the largest key of the group, the lowest expert that has it, and out it goes; lane
// j keeps the choice of round j. The whole row is in registers, so the logits are read once.
template <typename T, int G, int V, bool VEC>
__global__ __launch_bounds__(BLOCK) void gateKernel(const T* __restrict__ logits, size_t n, unsigned experts, size_t stride, unsigned k,
                                                    unsigned flags, int32_t* __restrict__ index, wide_t<T>* __restrict__ weight) {
  using R = wide_t<T>;
  using O = GateKey<T>;
  using K = typename O::key;
  const unsigned lane = threadIdx.x % G;
  forTiles((n + BLOCK / G - 1) / (BLOCK / G), gridDim.x, [&](size_t tile) {
    const size_t row = tile * (BLOCK / G) + threadIdx.x / G;
    if (row >= n) return;  // whole groups leave; lanes are paired inside a group
    T z[V];
    K key[V];
    gateLoad<T, G, V, VEC>(logits + row * stride, experts, lane, z);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const unsigned e = gateExpert<G, VEC>(i, lane);
      key[i] = e < experts ? O::of(z[i], e) : K(0);
    }
    K myKey = 0, topKey = 0, last = 0;
    unsigned myIndex = 0;
    R total = 0;
    for (unsigned j = 0; j < k; ++j) {
      K best = 0;
      unsigned at = 0;
      if constexpr (O::packed) {
        // Keys are distinct and have 26 bits: modulo 2^32, key - last is above 2^31 for keys below the last choice and below 2^26
        // for the others, so its maximum belongs to the largest key below, and nothing has to be taken out.
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const K below = j == 0 ? key[i] : key[i] - last;
          best = below > best ? below : best;
        }
        best = groupMax<G>(best);
        best = j == 0 ? best : best >> 31 ? best + last : K(0);
        last = best ? best : last;
        at = 1023u - (best & 1023u);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) best = key[i] > best ? key[i] : best;
        best = groupMax<G>(best);
        at = ~0u;
#pragma unroll
        for (int i = V - 1; i >= 0; --i) at = key[i] == best ? gateExpert<G, VEC>(i, lane) : at;
        at = groupMin<G>(at);
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (gateExpert<G, VEC>(i, lane) == at) key[i] = 0;
      }
      if (j == 0) {
        topKey = best;
        if ((flags & SPNC_HIP_GATE_ALL) && O::open(best)) {
          const R top = O::value(best);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const unsigned e = gateExpert<G, VEC>(i, lane);
            if (e < experts && R(z[i]) != -INFINITY) total += expOf(R(z[i]) - top);
          }
          total = groupSum<G>(total);
        }
      }
      if (lane == j) myKey = best, myIndex = at;
    }
    const bool open = lane < k && O::open(myKey);
    const R shifted = open ? O::value(myKey) - O::value(topKey) : R(0);
    const R e = open ? expOf(shifted) : R(0);
    if (!(flags & SPNC_HIP_GATE_ALL)) total = groupSum<G>(e);
    if (lane < k) {
      index[row * k + lane] = open ? int32_t(myIndex) : -1;
      weight[row * k + lane] = (flags & SPNC_HIP_GATE_LOG) ? (open ? shifted - logOf(total) : R(-INFINITY)) : open ? e / total : R(0);
    }
  });
}

// dz_e of the experts that were not chosen is 0, or -p_e times the sum over the slots under "all"; the k chosen ones get their
// slot's term on top, through LDS: every lane has V of the row's entries in registers, and a slot's expert may be any of them.
template <typename T, int G, int V, bool VEC>
__global__ __launch_bounds__(BLOCK) void gateBackwardKernel(const T* __restrict__ logits, size_t n, unsigned experts, size_t stride, unsigned k,
                                                            unsigned flags, const int32_t* __restrict__ index, const wide_t<T>* __restrict__ weight,
                                                            const wide_t<T>* __restrict__ gradWeight, T* __restrict__ gradLogits) {
  using R = wide_t<T>;
  __shared__ R entries[BLOCK / G][V * G];
  const unsigned lane = threadIdx.x % G;
  R* const mine = entries[threadIdx.x / G];
  const bool all = flags & SPNC_HIP_GATE_ALL, logs = flags & SPNC_HIP_GATE_LOG;
  forTiles((n + BLOCK / G - 1) / (BLOCK / G), gridDim.x, [&](size_t tile) {
    const size_t row = tile * (BLOCK / G) + threadIdx.x / G;
    if (row >= n) return;
    int32_t at = -1;
    R d = 0, w = 0;
    if (lane < k) {
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
    R top = -INFINITY, total = 0;
    if (all) {
      T z[V];
      gateLoad<T, G, V, VEC>(logits + row * stride, experts, lane, z);
      int bad = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        dz[i] = gateExpert<G, VEC>(i, lane) < experts ? R(z[i]) : R(-INFINITY);
        bad |= dz[i] != dz[i];
        top = dz[i] > top ? dz[i] : top;
      }
      top = groupMax<G>(top);
      if (groupMax<G>(bad)) top = NAN;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        dz[i] = dz[i] == -INFINITY ? R(0) : expOf(dz[i] - top);
        total += dz[i];
      }
      total = groupSum<G>(total);
    }
    const R common = groupSum<G>(d);
    if (!all) d -= w * common;
    const R factor = total == 0 ? R(0) : -common / total;
#pragma unroll
    for (int i = 0; i < V; i += VEC ? 4 : 1) {
      const unsigned e = gateExpert<G, VEC>(i, lane);
      if constexpr (VEC) {
        Pack<R, 4> p;
#pragma unroll
        for (int q = 0; q < 4; ++q) p.v[q] = dz[i + q] * factor;
        *reinterpret_cast<Pack<R, 4>*>(mine + e) = p;
      } else {
        mine[e] = dz[i] * factor;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the group is part of one wave, whose LDS accesses stay in order
    if (at >= 0) mine[at] += d;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int i = 0; i < V; i += VEC ? 4 : 1) {
      const unsigned e = gateExpert<G, VEC>(i, lane);
      if constexpr (VEC) {
        const Pack<R, 4> p = *reinterpret_cast<const Pack<R, 4>*>(mine + e);
        Pack<T, 4> o;
#pragma unroll
        for (int q = 0; q < 4; ++q) o.v[q] = T(p.v[q]);
        if (e < experts) *reinterpret_cast<Pack<T, 4>*>(gradLogits + row * experts + e) = o;
      } else if (e < experts) {
        gradLogits[row * experts + e] = T(mine[e]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  });
}

// ---- routing --------------------------------------------------------------------------------------------------------

constexpr unsigned ROUTE_BLOCK = 1024, ROUTE_WAVES = ROUTE_BLOCK / WAVE, ROUTE_MAX_BLOCKS = 256;
constexpr size_t ROUTE_SINGLE = 8192;      // slots one block sorts by itself
constexpr unsigned ROUTE_MAX_COUNTS = 65536;  // counters (blocks * experts) that every block adds up

struct RouteShape {
  size_t chunk;     // slots a block sorts, a multiple of ROUTE_BLOCK
  unsigned blocks;
};

RouteShape routeShape(size_t slots, unsigned experts) {
  if (slots <= ROUTE_SINGLE) return {(slots + ROUTE_BLOCK - 1) / ROUTE_BLOCK * ROUTE_BLOCK, 1};
  size_t blocks = (slots + 4 * ROUTE_BLOCK - 1) / (4 * ROUTE_BLOCK);
  const size_t most = ROUTE_MAX_COUNTS / experts < ROUTE_MAX_BLOCKS ? ROUTE_MAX_COUNTS / experts : ROUTE_MAX_BLOCKS;
  if (blocks > most) blocks = most;
  const size_t chunk = ((slots + blocks - 1) / blocks + ROUTE_BLOCK - 1) / ROUTE_BLOCK * ROUTE_BLOCK;
  return {chunk, unsigned((slots + chunk - 1) / chunk)};
}

// Lanes of the wave that hold the same expert, found by one vote per bit of the expert number.
__device__ inline uint64_t sameExpert(bool routed, uint32_t expert, unsigned bits) {
  uint64_t same = __ballot(routed);
  for (unsigned b = 0; b < bits; ++b) {
    const bool one = (expert >> b) & 1;
    const uint64_t votes = __ballot(one);
    same &= one ? votes : ~votes;
  }
  return same;
}

// counter[wave][expert] of this block's slots; every wave sorts a contiguous part of the chunk.
__device__ inline void countSlots(const int32_t* index, size_t begin, size_t end, unsigned experts, unsigned bits, uint32_t* counter) {
  const unsigned lane = threadIdx.x % WAVE;
  for (size_t s = begin; s < end; s += WAVE) {
    const size_t slot = s + lane;
    const uint32_t e = slot < end ? uint32_t(index[slot]) : ~0u;
    const bool routed = e < experts;
    const uint64_t same = sameExpert(routed, e, bits);
    if (routed && __ffsll((unsigned long long)same) - 1 == int(lane)) atomicAdd(&counter[e], uint32_t(__popcll(same)));
  }
}

__global__ __launch_bounds__(ROUTE_BLOCK) void routeCountKernel(const int32_t* __restrict__ index, size_t slots, unsigned experts, unsigned bits,
                                                                size_t chunk, uint32_t* __restrict__ counts) {
  extern __shared__ uint32_t routeLds[];  // [experts]
  for (unsigned e = threadIdx.x; e < experts; e += ROUTE_BLOCK) routeLds[e] = 0;
  __syncthreads();
  const size_t begin = blockIdx.x * chunk + threadIdx.x / WAVE * (chunk / ROUTE_WAVES);
  size_t end = begin + chunk / ROUTE_WAVES;
  if (end > slots) end = slots;
  countSlots(index, begin, end, experts, bits, routeLds);
  __syncthreads();
  for (unsigned e = threadIdx.x; e < experts; e += ROUTE_BLOCK) counts[size_t(blockIdx.x) * experts + e] = routeLds[e];
}

// blockCounts [gridDim.x][experts] of routeCountKernel; unused by a single block.
__global__ __launch_bounds__(ROUTE_BLOCK) void routeKernel(const int32_t* __restrict__ index, size_t slots, unsigned experts, unsigned bits,
                                                           unsigned align, size_t chunk, const uint32_t* __restrict__ blockCounts,
                                                           int32_t* __restrict__ position, int32_t* __restrict__ starts, int32_t* __restrict__ counts) {
  extern __shared__ uint32_t routeLds[];  // counter[ROUTE_WAVES][experts]
  __shared__ uint32_t waveSum[ROUTE_WAVES], total[ROUTE_BLOCK], earlier[ROUTE_BLOCK];
  const unsigned t = threadIdx.x, lane = t % WAVE, wave = t / WAVE;
  for (unsigned i = t; i < ROUTE_WAVES * experts; i += ROUTE_BLOCK) routeLds[i] = 0;
  total[t] = earlier[t] = 0;
  __syncthreads();
  // what all blocks, and the blocks before this one, hold of every expert: integer sums, the same in any order
  if (gridDim.x > 1) {
    const unsigned slices = ROUTE_BLOCK / experts, slice = t / experts, e = t % experts;
    uint32_t all = 0, before = 0;
    if (slice < slices)
      for (unsigned b = slice; b < gridDim.x; b += slices) {
        const uint32_t c = blockCounts[size_t(b) * experts + e];
        all += c;
        before += b < blockIdx.x ? c : 0;
      }
    if (all) atomicAdd(&total[e], all);
    if (before) atomicAdd(&earlier[e], before);
  }
  const size_t begin = blockIdx.x * chunk + wave * (chunk / ROUTE_WAVES);
  size_t end = begin + chunk / ROUTE_WAVES;
  if (end > slots) end = slots;
  countSlots(index, begin, end, experts, bits, routeLds + wave * experts);
  __syncthreads();
  uint32_t all = total[t];
  if (gridDim.x == 1 && t < experts)
    for (unsigned w = 0; w < ROUTE_WAVES; ++w) all += routeLds[w * experts + t];
  // where each segment starts: an exclusive scan of the totals, rounded up
  const uint32_t rounded = (all + (align - 1)) / align * align;
  uint32_t scan = rounded;
  for (unsigned d = 1; d < WAVE; d *= 2) {
    const uint32_t below = __shfl_up(scan, d);
    if (lane >= d) scan += below;
  }
  if (lane == WAVE - 1) waveSum[wave] = scan;
  __syncthreads();
  uint32_t start = scan - rounded;
  for (unsigned w = 0; w < wave; ++w) start += waveSum[w];
  if (t < experts) {
    if (blockIdx.x == 0) {
      starts[t] = int32_t(start);
      counts[t] = int32_t(all);
      if (t == experts - 1) starts[experts] = int32_t(start + rounded);
    }
    uint32_t next = start + earlier[t];
    for (unsigned w = 0; w < ROUTE_WAVES; ++w) {
      const uint32_t c = routeLds[w * experts + t];
      routeLds[w * experts + t] = next;
      next += c;
    }
  }
  __syncthreads();
  uint32_t* counter = routeLds + wave * experts;
  for (size_t s = begin; s < end; s += WAVE) {
    const size_t slot = s + lane;
    const uint32_t e = slot < end ? uint32_t(index[slot]) : ~0u;
    const bool routed = e < experts;
    const uint64_t same = sameExpert(routed, e, bits);
    const int leader = __ffsll((unsigned long long)same) - 1;
    uint32_t base = 0;
    if (routed && leader == int(lane)) base = atomicAdd(&counter[e], uint32_t(__popcll(same)));
    base = __shfl(base, routed ? leader : int(lane));
    if (slot < end) position[slot] = routed ? int32_t(base + __popcll(same & ((1ull << lane) - 1))) : -1;
  }
}

// ---- rows there and back --------------------------------------------------------------------------------------------

// A group of 2^shift lanes handles a row, a piece of up to 16 bytes a lane at a time.
//
// Rows that are written to scattered places bypass the caches where they consist of whole 64-byte halves of cache lines: 1 M rows
// of 64 bytes to two places each take 36 us instead of 50, of 2 KB to four places 52 instead of 67 (a consumer that reads
// them next loses up to half of that where they would have fit the last-level cache). Rows that share their halves must not: 48
// bytes take 87 us instead of 61, since each piece goes to memory by itself.
struct RowShape {
  unsigned pieces;  // of a row
  unsigned shift;
  size_t tiles;
  bool stream;      // scattered rows are written past the caches
};

RowShape rowShape(size_t n, size_t rowBytes, unsigned pieceBytes, const void* scattered = nullptr) {
  RowShape s;
  s.pieces = unsigned(rowBytes / pieceBytes);
  s.shift = 0;
  while (s.shift < 6 && (1u << s.shift) < s.pieces) ++s.shift;
  const size_t rows = BLOCK >> s.shift;
  s.tiles = (n + rows - 1) / rows;
  s.stream = pieceBytes == 16 && rowBytes % 64 == 0 && reinterpret_cast<uintptr_t>(scattered) % 64 == 0;
  return s;
}

// Rows of the sorted buffer that belong to no segment, cleared by blocks of their own behind the rowBlocks that write the
// others: a wave for what follows each segment, all of them for what follows the last one.
struct Unused {
  unsigned rowBlocks, blocks;
  const int32_t *starts, *counts;
  unsigned experts;
  size_t capacity, rowBytes;
  unsigned char* out;
};

__device__ inline void clearUnused(const Unused& u) {
  const unsigned lane = threadIdx.x % WAVE;
  const size_t wave = size_t(blockIdx.x - u.rowBlocks) * (BLOCK / WAVE) + threadIdx.x / WAVE, waves = size_t(u.blocks) * (BLOCK / WAVE);
  auto clear = [&](size_t from, size_t to, size_t first, size_t step) {  // bytes; pointers may have any alignment
    if (((reinterpret_cast<uintptr_t>(u.out) | from | to) & 15) == 0) {
      Pack<uint32_t, 4>* words = reinterpret_cast<Pack<uint32_t, 4>*>(u.out);
      for (size_t i = from / 16 + first; i < to / 16; i += step) words[i] = Pack<uint32_t, 4>{};
    } else if (((reinterpret_cast<uintptr_t>(u.out) | from | to) & 3) == 0) {
      uint32_t* words = reinterpret_cast<uint32_t*>(u.out);
      for (size_t i = from / 4 + first; i < to / 4; i += step) words[i] = 0;
    } else {
      for (size_t i = from + first; i < to; i += step) u.out[i] = 0;
    }
  };
  for (size_t e = wave; e < u.experts; e += waves) {
    size_t from = size_t(u.starts[e]) + size_t(u.counts[e]), to = size_t(u.starts[e + 1]);
    if (to > u.capacity) to = u.capacity;
    if (from < to) clear(from * u.rowBytes, to * u.rowBytes, lane, WAVE);
  }
  const size_t end = size_t(u.starts[u.experts]);
  if (end < u.capacity) clear(end * u.rowBytes, u.capacity * u.rowBytes, wave * WAVE + lane, waves * WAVE);
}

unsigned clearBlocks(size_t capacity, size_t rowBytes) {
  const size_t b = capacity * rowBytes / 65536 + 1;
  return unsigned(b < 256 ? b : 256);
}

// Positions of KB slots from `first` on, -1 where there is no slot or it is not routed.
template <int KB>
__device__ inline void loadPositions(const int32_t* position, size_t row, unsigned k, unsigned first, size_t capacity, int32_t (&at)[KB]) {
#pragma unroll
  for (int j = 0; j < KB; ++j) {
    at[j] = first + j < k ? position[row * k + first + j] : -1;
    if (at[j] >= 0 && size_t(at[j]) >= capacity) at[j] = -1;
  }
}

template <int KB, typename W, typename R>
__device__ inline void loadWeights(const W* weight, size_t row, unsigned k, unsigned first, R (&w)[KB]) {
#pragma unroll
  for (int j = 0; j < KB; ++j) w[j] = !weight ? R(1) : first + j < k ? R(weight[row * k + first + j]) : R(0);
}

template <typename P, int KB, bool STREAM>
__global__ __launch_bounds__(BLOCK) void dispatchKernel(const unsigned char* __restrict__ rows, size_t n, size_t strideBytes, RowShape shape,
                                                        const int32_t* __restrict__ position, unsigned k, size_t capacity, P* __restrict__ out,
                                                        Unused unused) {
  if (blockIdx.x >= unused.rowBlocks) return clearUnused(unused);
  const unsigned lane = threadIdx.x & ((1u << shape.shift) - 1);
  forTiles(shape.tiles, unused.rowBlocks, [&](size_t tile) {
    const size_t row = tile * (BLOCK >> shape.shift) + (threadIdx.x >> shape.shift);
    if (row >= n) return;
    const P* source = reinterpret_cast<const P*>(rows + row * strideBytes);
    for (unsigned first = 0; first < k; first += KB) {
      int32_t at[KB];
      loadPositions<KB>(position, row, k, first, capacity, at);
      for (unsigned c = lane; c < shape.pieces; c += 1u << shape.shift) {
        const P piece = source[c];
#pragma unroll
        for (int j = 0; j < KB; ++j)
          if (at[j] >= 0) {
            P* const to = &out[size_t(at[j]) * shape.pieces + c];
            if constexpr (STREAM) streamStore(to, piece);
            else *to = piece;
          }
      }
    }
  });
}

// Slots are read KB at a time, all loads before the first product; a slot that is not routed reads row 0 and drops it. Results
// bypass the caches, which leaves the values there for the backward pass (32769 x 4 rows of 2 KB, forward and backward: 164 us
// instead of 191), and so do values without weights: gradients of dispatch, whose last use this is (139 instead of 150 us for the
// whole of routing, dispatch and its gradient at that size).
template <typename T, int N, typename W, int KB, bool ONE, bool WEIGHTED>
__global__ __launch_bounds__(BLOCK) void combineKernel(const T* __restrict__ values, size_t capacity, size_t stride, RowShape shape,
                                                       const int32_t* __restrict__ position, size_t n, unsigned k, const W* __restrict__ weight,
                                                       Pack<T, N>* __restrict__ out) {
  using R = wide_t<T>;
  const unsigned lane = threadIdx.x & ((1u << shape.shift) - 1);
  forTiles(shape.tiles, gridDim.x, [&](size_t tile) {
    const size_t row = tile * (BLOCK >> shape.shift) + (threadIdx.x >> shape.shift);
    if (row >= n) return;
    int32_t at[KB];
    R w[KB];
    if (ONE) {
      loadPositions<KB>(position, row, k, 0, capacity, at);
      loadWeights<KB>(WEIGHTED ? weight : nullptr, row, k, 0, w);
    }
    for (unsigned c = lane; c < shape.pieces; c += 1u << shape.shift) {
      R sum[N] = {};
      for (unsigned first = 0; first < (ONE ? 1 : k); first += KB) {
        if (!ONE) {
          loadPositions<KB>(position, row, k, first, capacity, at);
          loadWeights<KB>(WEIGHTED ? weight : nullptr, row, k, first, w);
        }
        Pack<T, N> v[KB];
#pragma unroll
        for (int j = 0; j < KB; ++j)
          if (capacity) {
            const Pack<T, N>* from = reinterpret_cast<const Pack<T, N>*>(values + size_t(at[j] >= 0 ? at[j] : 0) * stride + size_t(c) * N);
            v[j] = WEIGHTED ? *from : streamLoad(from);
          }
#pragma unroll
        for (int j = 0; j < KB; ++j)
#pragma unroll
          for (int i = 0; i < N; ++i) sum[i] += at[j] >= 0 ? w[j] * R(v[j].v[i]) : R(0);
      }
      Pack<T, N> o;
#pragma unroll
      for (int i = 0; i < N; ++i) o.v[i] = T(sum[i]);
      streamStore(&out[row * shape.pieces + c], o);
    }
  });
}

template <typename T, int N, typename W, int KB, bool STREAM>
__global__ __launch_bounds__(BLOCK) void combineBackwardKernel(const T* __restrict__ values, size_t capacity, size_t stride, RowShape shape,
                                                               const int32_t* __restrict__ position, size_t n, unsigned k,
                                                               const W* __restrict__ weight, const T* __restrict__ gradOut, size_t gradStride,
                                                               Pack<T, N>* __restrict__ gradValues, W* __restrict__ gradWeight, Unused unused) {
  using R = wide_t<T>;
  if (blockIdx.x >= unused.rowBlocks) return clearUnused(unused);
  const unsigned group = 1u << shape.shift, lane = threadIdx.x & (group - 1);
  forTiles(shape.tiles, unused.rowBlocks, [&](size_t tile) {
    const size_t row = tile * (BLOCK >> shape.shift) + (threadIdx.x >> shape.shift);
    if (row >= n) return;
    for (unsigned first = 0; first < k; first += KB) {
      int32_t at[KB];
      R w[KB], dot[KB] = {};
      loadPositions<KB>(position, row, k, first, capacity, at);
      loadWeights<KB>(weight, row, k, first, w);
      for (unsigned c = lane; c < shape.pieces; c += group) {
        const Pack<T, N> g = streamLoad(reinterpret_cast<const Pack<T, N>*>(gradOut + row * gradStride + size_t(c) * N));
        if (gradWeight && capacity) {
          Pack<T, N> v[KB];
#pragma unroll
          for (int j = 0; j < KB; ++j) v[j] = *reinterpret_cast<const Pack<T, N>*>(values + size_t(at[j] >= 0 ? at[j] : 0) * stride + size_t(c) * N);
#pragma unroll
          for (int j = 0; j < KB; ++j)
#pragma unroll
            for (int i = 0; i < N; ++i) dot[j] += at[j] >= 0 ? R(g.v[i]) * R(v[j].v[i]) : R(0);
        }
        if (gradValues) {
#pragma unroll
          for (int j = 0; j < KB; ++j)
            if (at[j] >= 0) {
              Pack<T, N> o;
#pragma unroll
              for (int i = 0; i < N; ++i) o.v[i] = T(w[j] * R(g.v[i]));
              Pack<T, N>* const to = &gradValues[size_t(at[j]) * shape.pieces + c];
              if constexpr (STREAM) streamStore(to, o);
              else *to = o;
            }
        }
      }
      if (gradWeight) {
#pragma unroll
        for (int j = 0; j < KB; ++j) {
          for (unsigned d = 1; d < group; d *= 2) dot[j] += __shfl_xor(dot[j], int(d));
          if (lane == 0 && first + j < k) gradWeight[row * k + first + j] = W(dot[j]);
        }
      }
    }
  });
}

// The largest value of the row's slots is taken out before its log weight is added: values of some thousands differ by
// little, and the difference is exact where the sum would be rounded. Shares are computed from the same terms, not from the
// rounded result.

// A row's slots. K > 0: held in registers, read as one piece each of positions and weights; K = 0: read again for every use.
template <typename R, typename W, int K>
struct LogTerms {
  const R* values;
  size_t capacity;
  const int32_t* position;
  const W* logWeight;
  unsigned k;
  int32_t at[K > 0 ? K : 1];
  R value[K > 0 ? K : 1], weight[K > 0 ? K : 1];

  __device__ unsigned count() const { return K > 0 ? K : k; }
  // false: the slot is left out
  __device__ bool read(size_t s, R& v, R& lw, int32_t& p) const {
    p = position[s];
    if (p >= 0 && size_t(p) >= capacity) p = -1;
    lw = p >= 0 ? R(logWeight[s]) : R(-INFINITY);
    if (lw == -INFINITY) return false;
    v = values[p];
    return true;
  }
  __device__ void load(size_t row) {
    if constexpr (K > 0) {
      const Pack<int32_t, K> p = *reinterpret_cast<const Pack<int32_t, K>*>(position + row * K);
      const Pack<W, K> w = *reinterpret_cast<const Pack<W, K>*>(logWeight + row * K);
#pragma unroll
      for (int j = 0; j < K; ++j) {
        at[j] = p.v[j] >= 0 && size_t(p.v[j]) < capacity ? p.v[j] : -1;
        weight[j] = at[j] >= 0 ? R(w.v[j]) : R(-INFINITY);
        value[j] = capacity ? values[at[j] >= 0 ? at[j] : 0] : R(0);
      }
    }
  }
  __device__ bool slot(size_t row, unsigned j, R& v, R& lw) const {
    if constexpr (K > 0) {
      v = value[j];
      lw = weight[j];
      return lw != -INFINITY;
    } else {
      int32_t p;
      return read(row * k + j, v, lw, p);
    }
  }
};

// peak: the largest value; shift: the largest log weight + (value - peak); total: sum of exp(that - shift)
template <typename R, typename W, int K>
__device__ inline void logSum(const LogTerms<R, W, K>& terms, size_t row, R& peak, R& shift, R& total) {
  peak = -INFINITY;
  R v, lw;
#pragma unroll
  for (unsigned j = 0; j < terms.count(); ++j)
    if (terms.slot(row, j, v, lw)) peak = v > peak || v != v ? v : peak;
  shift = -INFINITY;
  total = 0;
  if (peak == -INFINITY) return;  // nothing possible
#pragma unroll
  for (unsigned j = 0; j < terms.count(); ++j)
    if (terms.slot(row, j, v, lw)) {
      const R t = lw + (v - peak);
      shift = t > shift || t != t ? t : shift;
    }
#pragma unroll
  for (unsigned j = 0; j < terms.count(); ++j)
    if (terms.slot(row, j, v, lw)) total += expOf(lw + (v - peak) - shift);
}

template <typename R, typename W, int K>
__global__ __launch_bounds__(BLOCK) void combineLogKernel(const R* __restrict__ values, size_t capacity, const int32_t* __restrict__ position,
                                                          const W* __restrict__ logWeight, size_t n, unsigned k, R* __restrict__ out) {
  forTiles((n + BLOCK - 1) / BLOCK, gridDim.x, [&](size_t tile) {
    const size_t row = tile * BLOCK + threadIdx.x;
    if (row >= n) return;
    LogTerms<R, W, K> terms{values, capacity, position, logWeight, k};
    terms.load(row);
    R peak, shift, total;
    logSum(terms, row, peak, shift, total);
    out[row] = peak == -INFINITY || peak == INFINITY ? peak : peak + (shift + logOf(total));
  });
}

template <typename R, typename W, int K>
__global__ __launch_bounds__(BLOCK) void combineLogBackwardKernel(const R* __restrict__ values, size_t capacity, const int32_t* __restrict__ position,
                                                                  const W* __restrict__ logWeight, size_t n, unsigned k, const R* __restrict__ gradOut,
                                                                  R* __restrict__ gradValues, W* __restrict__ gradLogWeight, Unused unused) {
  if (blockIdx.x >= unused.rowBlocks) return clearUnused(unused);
  forTiles((n + BLOCK - 1) / BLOCK, unused.rowBlocks, [&](size_t tile) {
    const size_t row = tile * BLOCK + threadIdx.x;
    if (row >= n) return;
    LogTerms<R, W, K> terms{values, capacity, position, logWeight, k};
    terms.load(row);
    R peak, shift, total;
    logSum(terms, row, peak, shift, total);
    const R g = gradOut[row];
    if constexpr (K > 0) {
      Pack<W, K> o;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        R v, lw, share = 0;
        if (peak != -INFINITY && terms.slot(row, j, v, lw)) share = g * (expOf(lw + (v - peak) - shift) / total);
        if (gradValues && terms.at[j] >= 0) gradValues[terms.at[j]] = share;
        o.v[j] = W(share);
      }
      if (gradLogWeight) *reinterpret_cast<Pack<W, K>*>(gradLogWeight + row * K) = o;
    } else {
      for (unsigned j = 0; j < k; ++j) {
        const size_t s = row * k + j;
        R v, lw, share = 0;
        int32_t p;
        if (terms.read(s, v, lw, p) && peak != -INFINITY) share = g * (expOf(lw + (v - peak) - shift) / total);
        if (gradValues && p >= 0) gradValues[p] = share;
        if (gradLogWeight) gradLogWeight[s] = W(share);
      }
    }
  });
}

// ---- dropout --------------------------------------------------------------------------------------------------------

template <typename R>
struct Dropout {
  uint64_t threshold;
  R scale, fill;
  uint64_t seed, offset;
  const uint64_t* offsetDevice;

  __device__ Philox4 words(size_t block, uint64_t at) const {
    return philox4x32(uint32_t(block), uint32_t(block >> 32), uint32_t(at), uint32_t(at >> 32), uint32_t(seed), uint32_t(seed >> 32));
  }
  template <typename T>
  __device__ T apply(uint32_t word, T x) const {
    return T(word >= threshold ? R(x) * scale : fill);
  }
};

template <typename T> constexpr int DROPOUT_UNIT = sizeof(T) == 2 ? 8 : 4;  // elements of 16 bytes, at least the four of one counter
constexpr unsigned DROPOUT_UNITS = 2;                                       // of a thread

// Contiguous elements; VEC: read and written 16 bytes at a time.
template <typename T, bool VEC>
__global__ __launch_bounds__(BLOCK) void dropoutFlatKernel(const T* x, size_t elements, T* out, Dropout<wide_t<T>> d) {
  constexpr int E = DROPOUT_UNIT<T>;
  using P = Pack<T, E>;
  const uint64_t at = d.offsetDevice ? *d.offsetDevice : d.offset;
  const size_t units = (elements + E - 1) / E, tiles = (units + DROPOUT_UNITS * BLOCK - 1) / (DROPOUT_UNITS * BLOCK);
  for (size_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const size_t first = tile * (DROPOUT_UNITS * BLOCK) + threadIdx.x;
    P v[DROPOUT_UNITS];
#pragma unroll
    for (unsigned i = 0; i < DROPOUT_UNITS; ++i) {
      const size_t e = (first + i * BLOCK) * E;
      if (VEC && e + E <= elements) v[i] = *reinterpret_cast<const P*>(x + e);
      else
#pragma unroll
        for (int q = 0; q < E; ++q)
          if (e + q < elements) v[i].v[q] = x[e + q];
    }
#pragma unroll
    for (unsigned i = 0; i < DROPOUT_UNITS; ++i) {
      const size_t e = (first + i * BLOCK) * E;
      if (e >= elements) continue;
#pragma unroll
      for (int b = 0; b < E / 4; ++b) {
        const Philox4 r = d.words(e / 4 + b, at);
#pragma unroll
        for (int q = 0; q < 4; ++q) v[i].v[4 * b + q] = d.apply(r.w[q], v[i].v[4 * b + q]);
      }
      if (VEC && e + E <= elements) *reinterpret_cast<P*>(out + e) = v[i];
      else
#pragma unroll
        for (int q = 0; q < E; ++q)
          if (e + q < elements) out[e + q] = v[i].v[q];
    }
  }
}

// Rows that are not adjacent; VEC: widths, strides and addresses in multiples of four elements, so that a counter's four
// elements are neighbours. Otherwise a counter whose elements lie in two rows is computed for both.
template <typename T, bool VEC>
__global__ __launch_bounds__(BLOCK) void dropoutRowsKernel(const T* x, size_t n, size_t width, size_t stride, T* out, size_t outStride, RowShape shape,
                                                           Dropout<wide_t<T>> d) {
  const uint64_t at = d.offsetDevice ? *d.offsetDevice : d.offset;
  const unsigned lane = threadIdx.x & ((1u << shape.shift) - 1);
  forTiles(shape.tiles, gridDim.x, [&](size_t tile) {
    const size_t row = tile * (BLOCK >> shape.shift) + (threadIdx.x >> shape.shift);
    if (row >= n) return;
    const size_t begin = row * width, end = begin + width;
    const T* from = x + row * stride;
    T* to = out + row * outStride;
    for (size_t b = begin / 4 + lane; 4 * b < end; b += size_t(1) << shape.shift) {
      const Philox4 r = d.words(b, at);
      if constexpr (VEC) {
        Pack<T, 4> v = *reinterpret_cast<const Pack<T, 4>*>(from + (4 * b - begin));
#pragma unroll
        for (int q = 0; q < 4; ++q) v.v[q] = d.apply(r.w[q], v.v[q]);
        *reinterpret_cast<Pack<T, 4>*>(to + (4 * b - begin)) = v;
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const size_t e = 4 * b + q;
          if (e >= begin && e < end) to[e - begin] = d.apply(r.w[q], from[e - begin]);
        }
      }
    }
  });
}

// ---- host side ------------------------------------------------------------------------------------------------------

[[noreturn]] void refuse(const std::string& what) { throw std::runtime_error(what); }

void launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) refuse(std::string(what) + " launch: " + hipGetErrorString(e));
}

size_t elementBytes(int dtype) {
  switch (dtype) {
    case SPNC_HIP_FLOAT32: return 4;
    case SPNC_HIP_FLOAT64: return 8;
    case SPNC_HIP_FLOAT16:
    case SPNC_HIP_BFLOAT16: return 2;
  }
  refuse("unknown element type " + std::to_string(dtype));
}

// calls fn(T()) for the element type
template <typename Fn>
void withType(int dtype, Fn&& fn) {
  switch (dtype) {
    case SPNC_HIP_FLOAT32: return fn(float());
    case SPNC_HIP_FLOAT64: return fn(double());
    case SPNC_HIP_FLOAT16: return fn(_Float16());
    case SPNC_HIP_BFLOAT16: return fn(__bf16());
  }
  refuse("unknown element type " + std::to_string(dtype));
}

// the widest piece, in bytes, that a row of rowBytes at these addresses and strides consists of; `least` at the least
unsigned pieceBytes(unsigned least, std::initializer_list<uintptr_t> addresses) {
  uintptr_t bits = 16;
  for (uintptr_t a : addresses) bits |= a;
  const unsigned widest = unsigned(bits & (~bits + 1));
  return widest < least ? 0 : widest;
}

uintptr_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }

void checkAligned(unsigned piece, const char* what) {
  if (piece == 0) refuse(std::string(what) + ": pointers are not aligned to the element type");
}

void checkSlots(size_t n, unsigned k, size_t capacity) {
  if (k == 0) refuse("k must be at least 1");
  if (n > (size_t(1) << 31) / k) refuse("too many slots: n * k must be below 2^31");
  if (capacity >= (size_t(1) << 31)) refuse("too many rows: the capacity must be below 2^31");
}

void checkExperts(unsigned experts) {
  if (experts == 0 || experts > SPNC_HIP_MAX_EXPERTS) refuse("experts must be between 1 and " + std::to_string(SPNC_HIP_MAX_EXPERTS));
}

void checkWeightType(int dtype, int weightDtype) {
  if (weightDtype != SPNC_HIP_FLOAT32 && !(weightDtype == SPNC_HIP_FLOAT64 && dtype == SPNC_HIP_FLOAT64))
    refuse("weights must be float32, or float64 with float64 values");
}

// calls fn(G, V, VEC): a row's logits in G lanes of V; at least as many lanes as choices, four logits a lane until 64 lanes are used
template <typename T, typename Fn>
void withGateShape(unsigned experts, unsigned k, size_t stride, uintptr_t addresses, Fn&& fn) {
  unsigned group = 1;
  while (group < WAVE && (4 * group < experts || group < k)) group *= 2;
  const bool vec = (experts | stride) % 4 == 0 && addresses % alignof(Pack<T, 4>) == 0;
  auto shape = [&](auto g, auto v) { vec ? fn(g, v, std::true_type()) : fn(g, v, std::false_type()); };
#define SPN_GATE_SHAPE(G, V) return shape(std::integral_constant<int, G>(), std::integral_constant<int, V>())
  switch (group) {
    case 1: SPN_GATE_SHAPE(1, 4);
    case 2: SPN_GATE_SHAPE(2, 4);
    case 4: SPN_GATE_SHAPE(4, 4);
    case 8: SPN_GATE_SHAPE(8, 4);
    case 16: SPN_GATE_SHAPE(16, 4);
    case 32: SPN_GATE_SHAPE(32, 4);
  }
  if (experts <= 256) SPN_GATE_SHAPE(64, 4);
  if (experts <= 512) SPN_GATE_SHAPE(64, 8);
  SPN_GATE_SHAPE(64, 16);
#undef SPN_GATE_SHAPE
}

void checkGate(int dtype, size_t n, unsigned experts, size_t stride, unsigned k, unsigned flags) {
  elementBytes(dtype);
  checkExperts(experts);
  if (k == 0 || k > experts || k > SPNC_HIP_MAX_CHOICES)
    refuse("k must be between 1 and the number of experts, at most " + std::to_string(SPNC_HIP_MAX_CHOICES));
  if (n > 1 && stride < experts) refuse("rows of logits overlap");
  if (flags & ~unsigned(SPNC_HIP_GATE_ALL | SPNC_HIP_GATE_LOG)) refuse("unknown gate flags");
}

template <typename Fn>
void withPieces(unsigned piece, Fn&& fn) {
  switch (piece) {
    case 16: return fn(Pack<uint32_t, 4>());
    case 8: return fn(Pack<uint32_t, 2>());
    case 4: return fn(uint32_t());
    case 2: return fn(uint16_t());
    default: return fn(uint8_t());
  }
}

// calls fn(N) with N elements of T to a piece
template <typename T, typename Fn>
void withPack(unsigned piece, Fn&& fn) {
  if (piece == 16) return fn(std::integral_constant<int, 16 / sizeof(T)>());
  if constexpr (sizeof(T) <= 8)
    if (piece == 8) return fn(std::integral_constant<int, 8 / sizeof(T)>());
  if constexpr (sizeof(T) <= 4)
    if (piece == 4) return fn(std::integral_constant<int, 4 / sizeof(T)>());
  if constexpr (sizeof(T) <= 2)
    if (piece == 2) return fn(std::integral_constant<int, 1>());
}

template <typename T, typename Fn>
void withWeight(int weightDtype, Fn&& fn) {
  if constexpr (std::is_same<T, double>::value)
    if (weightDtype == SPNC_HIP_FLOAT64) return fn(double());
  fn(float());
}

// Clearing rides along with the kernel that writes the used rows: its blocks follow that kernel's.
Unused unusedRows(unsigned rowBlocks, const int32_t* starts, const int32_t* counts, unsigned experts, size_t capacity, size_t rowBytes, void* out) {
  Unused u{rowBlocks, 0, starts, counts, experts, capacity, rowBytes, static_cast<unsigned char*>(out)};
  if (out && capacity && rowBytes) u.blocks = clearBlocks(capacity, rowBytes);
  return u;
}

// calls fn(STREAM); only 16-byte pieces are ever written past the caches
template <size_t PIECE, typename Fn>
void withStream(const RowShape& shape, Fn&& fn) {
  if constexpr (PIECE == 16)
    if (shape.stream) return fn(std::true_type());
  fn(std::false_type());
}

// calls fn(KB, ONE): slots are taken KB at a time; ONE says that this is all of them
template <typename Fn>
void withChoices(unsigned k, Fn&& fn) {
  if (k == 1) return fn(std::integral_constant<int, 1>(), std::true_type());
  if (k == 2) return fn(std::integral_constant<int, 2>(), std::true_type());
  if (k <= 4) return fn(std::integral_constant<int, 4>(), std::true_type());
  if (k <= 8) return fn(std::integral_constant<int, 8>(), std::true_type());
  fn(std::integral_constant<int, 8>(), std::false_type());
}

void checkSegments(const int32_t* starts, const int32_t* counts, unsigned experts) {
  checkExperts(experts);
  if (!starts || !counts) refuse("null argument");
}

// calls fn(K): K slots a row read as one piece each of positions and weights, or 0 for any number and alignment
template <typename W, typename Fn>
void withLogChoices(unsigned k, const void* position, const void* weight, const void* gradWeight, Fn&& fn) {
  const uintptr_t bits = address(position) | address(weight) | address(gradWeight);
  if (k == 1) return fn(std::integral_constant<int, 1>());
  if (k == 2 && bits % (2 * sizeof(W)) == 0) return fn(std::integral_constant<int, 2>());
  if (k == 4 && bits % 16 == 0) return fn(std::integral_constant<int, 4>());
  if (k == 8 && bits % 16 == 0) return fn(std::integral_constant<int, 8>());
  fn(std::integral_constant<int, 0>());
}

void checkLogTypes(int dtype, int weightDtype) {
  if (dtype != SPNC_HIP_FLOAT32 && dtype != SPNC_HIP_FLOAT64) refuse("log-likelihoods must be float32 or float64");
  if (weightDtype != SPNC_HIP_FLOAT32 && weightDtype != SPNC_HIP_FLOAT64) refuse("log weights must be float32 or float64");
}

template <typename Fn>
void withLogTypes(int dtype, int weightDtype, Fn&& fn) {
  if (dtype == SPNC_HIP_FLOAT32) return weightDtype == SPNC_HIP_FLOAT32 ? fn(float(), float()) : fn(float(), double());
  return weightDtype == SPNC_HIP_FLOAT32 ? fn(double(), float()) : fn(double(), double());
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
      withGateShape<T>(experts, k, stride, address(logits), [&](auto g, auto v, auto vec) {
        constexpr int G = decltype(g)::value, V = decltype(v)::value;
        gateKernel<T, G, V, decltype(vec)::value><<<tileGrid((n + BLOCK / G - 1) / (BLOCK / G)), BLOCK, 0, static_cast<hipStream_t>(stream)>>>(
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
      withGateShape<T>(experts, k, (flags & SPNC_HIP_GATE_ALL) ? stride : experts,
                       address(grad_logits) | ((flags & SPNC_HIP_GATE_ALL) ? address(logits) : 0), [&](auto g, auto v, auto vec) {
        constexpr int G = decltype(g)::value, V = decltype(v)::value;
        gateBackwardKernel<T, G, V, decltype(vec)::value><<<tileGrid((n + BLOCK / G - 1) / (BLOCK / G)), BLOCK, 0, static_cast<hipStream_t>(stream)>>>(
            static_cast<const T*>(logits), n, experts, stride, k, flags, index, static_cast<const R*>(weight), static_cast<const R*>(grad_weight),
            static_cast<T*>(grad_logits));
      });
    });
    launched("gate gradient");
  });
}

size_t spnc_hip_route_workspace(size_t slots, unsigned experts) {
  const RouteShape shape = routeShape(slots, experts);
  return shape.blocks <= 1 ? 0 : size_t(shape.blocks) * experts * sizeof(uint32_t);
}

int spnc_hip_route(const int32_t* index, size_t slots, unsigned experts, unsigned align, int32_t* position, int32_t* starts, int32_t* counts,
                   void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&] {
    checkExperts(experts);
    if (align == 0) refuse("align must be at least 1");
    if (slots >= (size_t(1) << 31) || slots + size_t(experts) * (align - 1) >= (size_t(1) << 31))
      refuse("too many slots: slots + experts * (align - 1) must be below 2^31");
    if ((slots && (!index || !position)) || !starts || !counts) refuse("null argument");
    const RouteShape shape = routeShape(slots, experts);
    const size_t need = spnc_hip_route_workspace(slots, experts);
    if (workspace_bytes < need || (need && !workspace)) refuse("the workspace must hold " + std::to_string(need) + " bytes");
    unsigned bits = 0;
    while ((1u << bits) < experts) ++bits;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (shape.blocks > 1) {
      routeCountKernel<<<shape.blocks, ROUTE_BLOCK, experts * sizeof(uint32_t), s>>>(index, slots, experts, bits, shape.chunk,
                                                                                     static_cast<uint32_t*>(workspace));
      launched("route");
    }
    const size_t lds = ROUTE_WAVES * experts * sizeof(uint32_t);
    if (lds > 48 * 1024) {
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(routeKernel), hipFuncAttributeMaxDynamicSharedMemorySize, int(lds));
      if (e != hipSuccess) refuse(std::string("route: ") + hipGetErrorString(e));
    }
    routeKernel<<<shape.blocks, ROUTE_BLOCK, lds, s>>>(
        index, slots, experts, bits, align, shape.chunk, static_cast<const uint32_t*>(workspace), position, starts, counts);
    launched("route");
  });
}

int spnc_hip_dispatch(const void* rows, size_t n, size_t row_bytes, size_t stride_bytes, const int32_t* position, unsigned k, size_t capacity,
                      const int32_t* starts, const int32_t* counts, unsigned experts, int zero_unused, void* out, void* stream) {
  return guarded([&] {
    checkSlots(n, k, capacity);
    if (row_bytes >> 32) refuse("a row must be shorter than 4 GiB");
    if (zero_unused) checkSegments(starts, counts, experts);
    if (capacity == 0 || row_bytes == 0) return;
    if (!out || (n && (!rows || !position))) refuse("null argument");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const unsigned piece = pieceBytes(1, {address(rows), address(out), row_bytes, stride_bytes});
    const RowShape shape = rowShape(n, row_bytes, piece, out);
    const Unused unused = unusedRows(tileGrid(shape.tiles), starts, counts, experts, capacity, row_bytes, zero_unused ? out : nullptr);
    if (unused.rowBlocks + unused.blocks == 0) return;
    withPieces(piece, [&](auto p) {
      using P = decltype(p);
      withChoices(k, [&](auto kb, auto) {
        constexpr int KB = decltype(kb)::value;
        withStream<sizeof(P)>(shape, [&](auto stream) {
          dispatchKernel<P, KB, decltype(stream)::value><<<unused.rowBlocks + unused.blocks, BLOCK, 0, s>>>(
              static_cast<const unsigned char*>(rows), n, stride_bytes, shape, position, k, capacity, static_cast<P*>(out), unused);
        });
      });
    });
    launched("dispatch");
  });
}

int spnc_hip_combine(const void* values, int dtype, size_t capacity, size_t width, size_t stride, const int32_t* position, size_t n, unsigned k,
                     const void* weight, int weight_dtype, void* out, void* stream) {
  return guarded([&] {
    const size_t bytes = elementBytes(dtype);
    checkSlots(n, k, capacity);
    if (weight) checkWeightType(dtype, weight_dtype);
    if (width * bytes >> 32) refuse("a row must be shorter than 4 GiB");
    if (n == 0 || width == 0) return;
    if ((capacity && !values) || !position || !out) refuse("null argument");
    const unsigned piece = pieceBytes(unsigned(bytes), {address(values), address(out), width * bytes, stride * bytes});
    checkAligned(piece, "combine");
    const RowShape shape = rowShape(n, width * bytes, piece);
    withType(dtype, [&](auto t) {
      using T = decltype(t);
      withPack<T>(piece, [&](auto count) {
        constexpr int N = decltype(count)::value;
        withWeight<T>(weight_dtype, [&](auto w) {
          using W = decltype(w);
          withChoices(k, [&](auto kb, auto one) {
            auto launch = [&](auto weighted) {
              combineKernel<T, N, W, decltype(kb)::value, decltype(one)::value, decltype(weighted)::value>
                  <<<tileGrid(shape.tiles), BLOCK, 0, static_cast<hipStream_t>(stream)>>>(
                      static_cast<const T*>(values), capacity, stride, shape, position, n, k, static_cast<const W*>(weight), static_cast<Pack<T, N>*>(out));
            };
            weight ? launch(std::true_type()) : launch(std::false_type());
          });
        });
      });
    });
    launched("combine");
  });
}

int spnc_hip_combine_backward(const void* values, int dtype, size_t capacity, size_t width, size_t stride, const int32_t* position, size_t n,
                              unsigned k, const void* weight, int weight_dtype, const void* grad_out, size_t grad_stride, const int32_t* starts,
                              const int32_t* counts, unsigned experts, void* grad_values, void* grad_weight, void* stream) {
  return guarded([&] {
    const size_t bytes = elementBytes(dtype);
    checkSlots(n, k, capacity);
    checkWeightType(dtype, weight_dtype);
    if (width * bytes >> 32) refuse("a row must be shorter than 4 GiB");
    if (grad_values) checkSegments(starts, counts, experts);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (!grad_values && !grad_weight) return;
    if (n && ((capacity && width && !values) || !position || !weight || (width && !grad_out))) refuse("null argument");
    const unsigned piece = pieceBytes(unsigned(bytes), {address(values), address(grad_out), address(grad_values), width * bytes, stride * bytes,
                                                        grad_stride * bytes});
    checkAligned(piece, "combine gradient");
    const RowShape shape = rowShape(n, width * bytes, piece, grad_values);
    const Unused unused = unusedRows(tileGrid(shape.tiles), starts, counts, experts, capacity, width * bytes, grad_values);
    if (unused.rowBlocks + unused.blocks == 0) return;
    withType(dtype, [&](auto t) {
      using T = decltype(t);
      withPack<T>(piece, [&](auto count) {
        constexpr int N = decltype(count)::value;
        withWeight<T>(weight_dtype, [&](auto w) {
          using W = decltype(w);
          withChoices(k, [&](auto kb, auto) {
            withStream<sizeof(T) * N>(shape, [&](auto past) {
              combineBackwardKernel<T, N, W, decltype(kb)::value, decltype(past)::value><<<unused.rowBlocks + unused.blocks, BLOCK, 0, s>>>(
                  static_cast<const T*>(values), capacity, stride, shape, position, n, k, static_cast<const W*>(weight),
                  static_cast<const T*>(grad_out), grad_stride, static_cast<Pack<T, N>*>(grad_values), static_cast<W*>(grad_weight), unused);
            });
          });
        });
      });
    });
    launched("combine gradient");
  });
}

int spnc_hip_combine_log(const void* values, int dtype, size_t capacity, const int32_t* position, size_t n, unsigned k, const void* log_weight,
                         int weight_dtype, void* out, void* stream) {
  return guarded([&] {
    checkLogTypes(dtype, weight_dtype);
    checkSlots(n, k, capacity);
    if (n == 0) return;
    if ((capacity && !values) || !position || !log_weight || !out) refuse("null argument");
    withLogTypes(dtype, weight_dtype, [&](auto r, auto w) {
      using R = decltype(r);
      using W = decltype(w);
      withLogChoices<W>(k, position, log_weight, nullptr, [&](auto kb) {
        combineLogKernel<R, W, decltype(kb)::value><<<tileGrid((n + BLOCK - 1) / BLOCK), BLOCK, 0, static_cast<hipStream_t>(stream)>>>(
            static_cast<const R*>(values), capacity, position, static_cast<const W*>(log_weight), n, k, static_cast<R*>(out));
      });
    });
    launched("combine_log");
  });
}

int spnc_hip_combine_log_backward(const void* values, int dtype, size_t capacity, const int32_t* position, size_t n, unsigned k,
                                  const void* log_weight, int weight_dtype, const void* grad_out, const int32_t* starts, const int32_t* counts,
                                  unsigned experts, void* grad_values, void* grad_log_weight, void* stream) {
  return guarded([&] {
    checkLogTypes(dtype, weight_dtype);
    checkSlots(n, k, capacity);
    if (grad_values) checkSegments(starts, counts, experts);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (!grad_values && !grad_log_weight) return;
    if (n && ((capacity && !values) || !position || !log_weight || !grad_out)) refuse("null argument");
    const Unused unused =
        unusedRows(tileGrid((n + BLOCK - 1) / BLOCK), starts, counts, experts, capacity, elementBytes(dtype), grad_values);
    if (unused.rowBlocks + unused.blocks == 0) return;
    withLogTypes(dtype, weight_dtype, [&](auto r, auto w) {
      using R = decltype(r);
      using W = decltype(w);
      withLogChoices<W>(k, position, log_weight, grad_log_weight, [&](auto kb) {
        combineLogBackwardKernel<R, W, decltype(kb)::value><<<unused.rowBlocks + unused.blocks, BLOCK, 0, s>>>(
            static_cast<const R*>(values), capacity, position, static_cast<const W*>(log_weight), n, k, static_cast<const R*>(grad_out),
            static_cast<R*>(grad_values), static_cast<W*>(grad_log_weight), unused);
      });
    });
    launched("combine_log gradient");
  });
}

int spnc_hip_dropout(const void* x, int dtype, size_t n, size_t width, size_t stride, void* out, size_t out_stride, double p, int mode,
                     uint64_t seed, uint64_t offset, const uint64_t* offset_device, void* stream) {
  return guarded([&] {
    elementBytes(dtype);
    if (!(p >= 0.0 && p <= 1.0)) refuse("the probability of dropping an element must be between 0 and 1");
    if (mode < SPNC_HIP_DROPOUT_ZERO || mode > SPNC_HIP_DROPOUT_MASK) refuse("unknown dropout mode " + std::to_string(mode));
    if (n > 1 && (stride < width || out_stride < width)) refuse("rows overlap");
    if (n == 0 || width == 0) return;
    if (!x || !out) refuse("null argument");
    const uint64_t threshold = uint64_t(std::llrint(p * 4294967296.0));
    const double scale = mode != SPNC_HIP_DROPOUT_ZERO ? 1.0 : threshold >> 32 ? 0.0 : 1.0 / (1.0 - p);
    const double fill = mode == SPNC_HIP_DROPOUT_MARGINAL ? NAN : 0.0;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    withType(dtype, [&](auto t) {
      using T = decltype(t);
      using R = wide_t<T>;
      const Dropout<R> d{threshold, R(scale), R(fill), seed, offset, offset_device};
      const uintptr_t bits = address(x) | address(out);
      if (n == 1 || (stride == width && out_stride == width)) {
        constexpr int E = DROPOUT_UNIT<T>;
        const size_t elements = n * width, units = (elements + E - 1) / E, blocks = (units + DROPOUT_UNITS * BLOCK - 1) / (DROPOUT_UNITS * BLOCK);
        const unsigned grid = unsigned(blocks < MAX_GRID ? blocks : MAX_GRID);
        if (bits % (sizeof(Pack<T, E>) < 16 ? sizeof(Pack<T, E>) : 16) == 0)
          dropoutFlatKernel<T, true><<<grid, BLOCK, 0, s>>>(static_cast<const T*>(x), elements, static_cast<T*>(out), d);
        else
          dropoutFlatKernel<T, false><<<grid, BLOCK, 0, s>>>(static_cast<const T*>(x), elements, static_cast<T*>(out), d);
      } else {
        const RowShape shape = rowShape(n, (width + 3) / 4, 1);
        if (((width | stride | out_stride) % 4 | bits % (4 * sizeof(T) < 16 ? 4 * sizeof(T) : 16)) == 0)
          dropoutRowsKernel<T, true><<<tileGrid(shape.tiles), BLOCK, 0, s>>>(static_cast<const T*>(x), n, width, stride, static_cast<T*>(out), out_stride, shape, d);
        else
          dropoutRowsKernel<T, false><<<tileGrid(shape.tiles), BLOCK, 0, s>>>(static_cast<const T*>(x), n, width, stride, static_cast<T*>(out), out_stride, shape, d);
      }
    });
    launched("dropout");
  });
}

}  // extern "C"
