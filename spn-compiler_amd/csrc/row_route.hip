// Rows sorted by expert and back: the sort, the copy into its order, the weighted sum and the log-sum-exp back in row order,
// and their gradients.
#include "row_common.h"

namespace spnc_hip {
namespace {

// ---- routing --------------------------------------------------------------------------------------------------------

// A stable counting sort in two launches, or one for up to 8192 slots. Blocks count the experts of a chunk of slots each; then every
// block adds up what all and what the earlier ones counted, and places its own chunk. Within a wave slots of one expert find each other
// by votes, a bit of the expert's number at a time, and are numbered by the lanes below; waves and tiles follow each other by
// counters in LDS. 2 M slots of 10 experts take 5 + 9 us: 16 MB of traffic is less than a third of that, the rest is the chain of votes
// and LDS round trips and the launch of the second kernel.
constexpr unsigned ROUTE_BLOCK = 1024, ROUTE_WAVES = ROUTE_BLOCK / WAVE, ROUTE_MAX_BLOCKS = 256;
constexpr unsigned ROUTE_MAX_ITEMS = 8;                               // slots a lane sorts at a time
constexpr size_t ROUTE_SINGLE = ROUTE_BLOCK * ROUTE_MAX_ITEMS;        // slots one block sorts by itself
constexpr unsigned ROUTE_MAX_COUNTS = 65536;                          // counters (blocks * experts) that every block adds up

struct RouteShape {
  size_t chunk;  // slots a block sorts, a multiple of its tile of `items` slots a lane
  unsigned blocks, items;
};

RouteShape routeShape(size_t slots, unsigned experts) {
  size_t blocks = 1;
  if (slots > ROUTE_SINGLE) {
    const size_t most = ROUTE_MAX_COUNTS / experts < ROUTE_MAX_BLOCKS ? ROUTE_MAX_COUNTS / experts : ROUTE_MAX_BLOCKS;
    blocks = (slots + 2 * ROUTE_BLOCK - 1) / (2 * ROUTE_BLOCK);
    if (blocks > most) blocks = most;
  }
  const size_t each = (slots + blocks - 1) / blocks;
  const unsigned items = each <= 2 * ROUTE_BLOCK ? 2 : each <= 4 * ROUTE_BLOCK ? 4 : 8;
  const size_t tile = size_t(items) * ROUTE_BLOCK, tiles = each ? (each + tile - 1) / tile : 1;
  return {tiles * tile, unsigned(slots > ROUTE_SINGLE ? (slots + tiles * tile - 1) / (tiles * tile) : 1), items};
}

// An expert's number for each of a lane's slots, ~0 where there is none or it is not routed.
template <int ITEMS>
__device__ inline void routeLoad(const int32_t* index, size_t slot, size_t slots, unsigned experts, uint32_t (&e)[ITEMS]) {
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) e[i] = slot + i * WAVE < slots ? uint32_t(index[slot + i * WAVE]) : ~0u;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
    if (e[i] >= experts) e[i] = ~0u;
}

template <int ITEMS>
__global__ __launch_bounds__(ROUTE_BLOCK) void routeCountKernel(const int32_t* __restrict__ index, size_t slots, unsigned experts, size_t chunk,
                                                                uint32_t* __restrict__ counts) {
  extern __shared__ uint32_t routeLds[];  // [ROUTE_WAVES][experts]: waves do not get in each other's way
  const unsigned t = threadIdx.x;
  for (unsigned i = t; i < ROUTE_WAVES * experts; i += ROUTE_BLOCK) routeLds[i] = 0;
  __syncthreads();
  uint32_t* const mine = routeLds + t / WAVE * experts;
  for (size_t tile = 0; tile < chunk; tile += ROUTE_BLOCK * ITEMS) {
    uint32_t e[ITEMS];
    routeLoad<ITEMS>(index, blockIdx.x * chunk + tile + t / WAVE * (WAVE * ITEMS) + t % WAVE, slots, experts, e);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (e[i] != ~0u) atomicAdd(&mine[e[i]], 1u);
  }
  __syncthreads();
  if (t < experts) {
    uint32_t sum = 0;
    for (unsigned w = 0; w < ROUTE_WAVES; ++w) sum += routeLds[w * experts + t];
    counts[size_t(blockIdx.x) * experts + t] = sum;
  }
}

// A lane's slots numbered among those of the same expert in the wave, counted on from counter[expert] and added to it.
template <int ITEMS>
__device__ inline void routeRank(const uint32_t (&e)[ITEMS], unsigned bits, uint32_t* counter, uint32_t (&rank)[ITEMS]) {
  const unsigned lane = threadIdx.x % WAVE;
  uint64_t same[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) same[i] = __ballot(e[i] != ~0u);
  for (unsigned b = 0; b < bits; ++b)
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const bool one = (e[i] >> b) & 1;
      const uint64_t votes = __ballot(one);
      same[i] &= one ? votes : ~votes;
    }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const unsigned below = unsigned(__popcll(same[i] & ((1ull << lane) - 1)));
    rank[i] = 0;
    if (e[i] != ~0u && below == 0) rank[i] = atomicAdd(&counter[e[i]], uint32_t(__popcll(same[i])));  // the first lane, for all
    const int first = e[i] != ~0u ? __ffsll((unsigned long long)same[i]) - 1 : int(lane);
    rank[i] = __shfl(rank[i], first) + below;
  }
}

// blockCounts [gridDim.x][experts] of routeCountKernel; unused by a single block.
template <int ITEMS>
__global__ __launch_bounds__(ROUTE_BLOCK) void routeKernel(const int32_t* __restrict__ index, size_t slots, unsigned experts, unsigned bits,
                                                           unsigned align, size_t chunk, const uint32_t* __restrict__ blockCounts,
                                                           int32_t* __restrict__ position, int32_t* __restrict__ starts, int32_t* __restrict__ counts) {
  extern __shared__ uint32_t routeLds[];  // counter[ROUTE_WAVES][experts]
  __shared__ uint32_t waveSum[ROUTE_WAVES], total[ROUTE_BLOCK], next[ROUTE_BLOCK];
  const unsigned t = threadIdx.x, lane = t % WAVE, wave = t / WAVE;
  const size_t begin = blockIdx.x * chunk + wave * (WAVE * ITEMS) + lane;
  uint32_t e[ITEMS], rank[ITEMS];
  routeLoad<ITEMS>(index, begin, slots, experts, e);
  for (unsigned i = t; i < ROUTE_WAVES * experts; i += ROUTE_BLOCK) routeLds[i] = 0;
  total[t] = next[t] = 0;
  __syncthreads();
  // what all blocks, and the blocks before this one, hold of every expert: integer sums, the same in any order
  if (gridDim.x > 1) {
    const unsigned slices = ROUTE_BLOCK / experts, slice = t / experts, expert = t % experts;
    uint32_t all = 0, before = 0;
    if (slice < slices) {
#pragma unroll 4
      for (unsigned b = slice; b < gridDim.x; b += slices) {
        const uint32_t c = blockCounts[size_t(b) * experts + expert];
        all += c;
        before += b < blockIdx.x ? c : 0;
      }
    }
    if (all) atomicAdd(&total[expert], all);
    if (before) atomicAdd(&next[expert], before);
  }
  uint32_t* const counter = routeLds + wave * experts;
  routeRank<ITEMS>(e, bits, counter, rank);
  __syncthreads();
  uint32_t all = total[t];
  if (gridDim.x == 1 && t < experts)
    for (unsigned w = 0; w < ROUTE_WAVES; ++w) all += routeLds[w * experts + t];
  // where each segment starts: an exclusive scan of the totals, rounded up
  const uint32_t rounded = align == 1 ? all : (all + (align - 1)) / align * align;
  uint32_t scan = rounded;
#pragma unroll
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
    next[t] += start;
  }
  for (size_t tile = 0;;) {
    if (t < experts) {  // the waves' counters become the first positions of their slots
      uint32_t at = next[t];
      for (unsigned w = 0; w < ROUTE_WAVES; ++w) {
        const uint32_t c = routeLds[w * experts + t];
        routeLds[w * experts + t] = at;
        at += c;
      }
      next[t] = at;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const size_t slot = begin + tile + i * WAVE;
      if (slot < slots) position[slot] = e[i] != ~0u ? int32_t(counter[e[i]] + rank[i]) : -1;
    }
    tile += ROUTE_BLOCK * ITEMS;
    if (tile >= chunk) break;
    routeLoad<ITEMS>(index, begin + tile, slots, experts, e);
    __syncthreads();
    for (unsigned i = t; i < ROUTE_WAVES * experts; i += ROUTE_BLOCK) routeLds[i] = 0;
    __syncthreads();
    routeRank<ITEMS>(e, bits, counter, rank);
    __syncthreads();
  }
}

// ---- rows there and back --------------------------------------------------------------------------------------------

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
    unsigned char *const begin = u.out + from, *const end = u.out + to;
    const uintptr_t low = (reinterpret_cast<uintptr_t>(begin) + 15) & ~uintptr_t(15), high = reinterpret_cast<uintptr_t>(end) & ~uintptr_t(15);
    if (low >= high) {
      for (size_t i = first; i < to - from; i += step) begin[i] = 0;
      return;
    }
    Pack<uint32_t, 4>* const pieces = reinterpret_cast<Pack<uint32_t, 4>*>(low);
    for (size_t i = first; i < (high - low) / 16; i += step) pieces[i] = Pack<uint32_t, 4>{};
    unsigned char* const tail = reinterpret_cast<unsigned char*>(high);
    if (first < low - reinterpret_cast<uintptr_t>(begin)) begin[first] = 0;  // fewer than 16 bytes, of which there are as many lanes
    if (first < reinterpret_cast<uintptr_t>(end) - high) tail[first] = 0;
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

// out[position_ij] = x_i: a row is read once and written to all its places. Bound by the writes: 1 M rows of 64 bytes to two places
// take 36 us, 5.6 TB/s; 32769 rows of 2 KB to four, 53 us, 6.3 TB/s. Rows that share cache lines with rows of other blocks cost more: of 24
// bytes, 2 M to two of ten experts' places 55 us, 3.1 TB/s, to four of 64 experts' places 102 us, 2.8 TB/s.
template <typename P, int KB, bool STREAM>
__global__ __launch_bounds__(BLOCK) void dispatchKernel(const unsigned char* __restrict__ rows, size_t n, size_t strideBytes, RowShape shape,
                                                        const int32_t* __restrict__ position, unsigned k, size_t capacity, P* __restrict__ out,
                                                        Unused unused) {
  if (blockIdx.x >= unused.rowBlocks) return clearUnused(unused);
  const unsigned lane = threadIdx.x & ((1u << shape.shift) - 1);
  forTiles(shape.tiles, unused.rowBlocks, shape.byDie, [&](size_t tile) {
    const size_t row = tile * (BLOCK >> shape.shift) + (threadIdx.x >> shape.shift);
    if (row >= n) return;
    const P* source = reinterpret_cast<const P*>(rows + row * strideBytes);
    for (unsigned first = 0; first < k; first += KB) {
      int32_t at[KB];
      loadPositions<KB>(position, row, k, first, capacity, at);
      // H pieces a lane at a time, H - 1 of which may lie behind the row's end
      auto copy = [&](auto h) {
        constexpr unsigned H = decltype(h)::value;
        for (unsigned c = lane; c < shape.pieces; c += H << shape.shift) {
          P piece[H];
#pragma unroll
          for (unsigned i = 0; i < H; ++i)
            if (i == 0 || c + (i << shape.shift) < shape.pieces) piece[i] = source[c + (i << shape.shift)];
#pragma unroll
          for (unsigned i = 0; i < H; ++i)
            if (i == 0 || c + (i << shape.shift) < shape.pieces)
#pragma unroll
              for (int j = 0; j < KB; ++j)
                if (at[j] >= 0) {
                  P* const to = &out[size_t(at[j]) * shape.pieces + c + (i << shape.shift)];
                  if constexpr (STREAM) streamStore(to, piece[i]);
                  else *to = piece[i];
                }
        }
      };
      if (shape.pieces > 1u << shape.shift) copy(std::integral_constant<unsigned, 2>());
      else copy(std::integral_constant<unsigned, 1>());
    }
  });
}

// out[i] = sum_j w_ij v[position_ij] in the order of j. Bound by memory: 32769 rows of four slots of 2 KB take 59 us, 5.5 TB/s. Slots
// are read KB at a time, all loads before the first product (a slot that is not routed reads row 0 and drops it), and two pieces a
// lane at a time where a row has them for all lanes, which is 10 us of these. Results go past the caches, which leaves the
// values there for the backward pass (both together are 27 us shorter at that size), and so do values without weights: gradients of
// dispatch, whose last use this is (54 us; 11 us of routing, dispatch and gradient together).
template <typename T, int N, typename W, int KB, bool ONE, bool WEIGHTED>
__global__ __launch_bounds__(BLOCK) void combineKernel(const T* __restrict__ values, size_t capacity, size_t stride, RowShape shape,
                                                       const int32_t* __restrict__ position, size_t n, unsigned k, const W* __restrict__ weight,
                                                       Pack<T, N>* __restrict__ out) {
  using R = wide_t<T>;
  const unsigned lane = threadIdx.x & ((1u << shape.shift) - 1);
  forTiles(shape.tiles, gridDim.x, shape.byDie, [&](size_t tile) {
    const size_t row = tile * (BLOCK >> shape.shift) + (threadIdx.x >> shape.shift);
    if (row >= n) return;
    int32_t at[KB];
    R w[KB];
    if (ONE) {
      loadPositions<KB>(position, row, k, 0, capacity, at);
      loadWeights<KB>(WEIGHTED ? weight : nullptr, row, k, 0, w);
    }
    auto join = [&](auto h) {
      constexpr unsigned H = decltype(h)::value;
      for (unsigned c = lane; c < shape.pieces; c += H << shape.shift) {
        const unsigned place[2] = {c, c + (1u << shape.shift)};
        R sum[H][N] = {};
        for (unsigned first = 0; first < (ONE ? 1 : k); first += KB) {
          if (!ONE) {
            loadPositions<KB>(position, row, k, first, capacity, at);
            loadWeights<KB>(WEIGHTED ? weight : nullptr, row, k, first, w);
          }
          Pack<T, N> v[H][KB];
#pragma unroll
          for (unsigned q = 0; q < H; ++q)
#pragma unroll
            for (int j = 0; j < KB; ++j) {
              const Pack<T, N>* from = reinterpret_cast<const Pack<T, N>*>(values + size_t(at[j] >= 0 ? at[j] : 0) * stride + size_t(place[q]) * N);
              v[q][j] = WEIGHTED ? *from : streamLoad(from);
            }
#pragma unroll
          for (unsigned q = 0; q < H; ++q)
#pragma unroll
            for (int j = 0; j < KB; ++j)
#pragma unroll
              for (int i = 0; i < N; ++i) sum[q][i] += at[j] >= 0 ? w[j] * R(v[q][j].v[i]) : R(0);
        }
#pragma unroll
        for (unsigned q = 0; q < H; ++q) {
          Pack<T, N> o;
#pragma unroll
          for (int i = 0; i < N; ++i) o.v[i] = T(sum[q][i]);
          streamStore(&out[row * shape.pieces + place[q]], o);
        }
      }
    };
    if (shape.pieces % (2u << shape.shift) == 0) join(std::integral_constant<unsigned, 2>());
    else join(std::integral_constant<unsigned, 1>());
  });
}

// dv[position_ij] = w_ij g_i and dw_ij = <g_i, v[position_ij]> in one pass over the values. Bound by memory: 32769 rows of four slots
// of 2 KB take 94 us, 6.3 TB/s; the gradient of the output is read past the caches, where it has no further use (8 us).
template <typename T, int N, typename W, int KB, bool STREAM>
__global__ __launch_bounds__(BLOCK) void combineBackwardKernel(const T* __restrict__ values, size_t capacity, size_t stride, RowShape shape,
                                                               const int32_t* __restrict__ position, size_t n, unsigned k,
                                                               const W* __restrict__ weight, const T* __restrict__ gradOut, size_t gradStride,
                                                               Pack<T, N>* __restrict__ gradValues, W* __restrict__ gradWeight, Unused unused) {
  using R = wide_t<T>;
  if (blockIdx.x >= unused.rowBlocks) return clearUnused(unused);
  const unsigned group = 1u << shape.shift, lane = threadIdx.x & (group - 1);
  forTiles(shape.tiles, unused.rowBlocks, shape.byDie, [&](size_t tile) {
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
// rounded result. A slot that is not routed or has log weight minus infinity is left out, whatever value stands there.
//
// K slots a row in registers, EXACT: k of them, positions and weights one piece each; otherwise the last ones may be missing. Bound by
// the gather of single values: lanes next to each other hold rows of different experts, so nearly every lane is an access of its own.
// Two rows a thread keep more of them under way. 4 M rows of two slots take 26 us, 4.5 TB/s, and 30 with the shares for a backward pass: the address
// units, which take a lane a cycle here, are busy for three quarters of that.
template <typename R, typename W, int K, bool EXACT>
struct LogRow {
  int32_t at[K];
  R weight[K], term[K];  // term: the value, then exp(log weight + (value - peak) - shift)
  R peak, shift, total;  // the largest value, the largest log weight + (value - peak), the sum of the terms

  __device__ void slots(const int32_t* position, const W* logWeight, size_t row, unsigned k, size_t capacity) {
    Pack<int32_t, K> p;
    Pack<W, K> w;
    if constexpr (EXACT) {
      p = *reinterpret_cast<const Pack<int32_t, K>*>(position + row * K);
      w = *reinterpret_cast<const Pack<W, K>*>(logWeight + row * K);
    } else {
#pragma unroll
      for (int j = 0; j < K; ++j) {
        p.v[j] = j < int(k) ? position[row * k + j] : -1;
        w.v[j] = j < int(k) ? logWeight[row * k + j] : W(0);
      }
    }
#pragma unroll
    for (int j = 0; j < K; ++j) {
      at[j] = p.v[j] >= 0 && size_t(p.v[j]) < capacity ? p.v[j] : -1;
      weight[j] = at[j] >= 0 ? R(w.v[j]) : R(-INFINITY);
    }
  }
  __device__ void values(const R* from) {
#pragma unroll
    for (int j = 0; j < K; ++j) term[j] = from[at[j] >= 0 ? at[j] : 0];
  }
  __device__ void solve() {
    peak = shift = -INFINITY;
    total = 0;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (weight[j] == -INFINITY) term[j] = -INFINITY;
      peak = term[j] > peak || term[j] != term[j] ? term[j] : peak;
    }
#pragma unroll
    for (int j = 0; j < K; ++j) {
      term[j] = weight[j] + (term[j] - peak);
      shift = term[j] > shift || term[j] != term[j] ? term[j] : shift;
    }
#pragma unroll
    for (int j = 0; j < K; ++j) {
      term[j] = expOf(term[j] - shift);
      total += term[j];
    }
  }
  __device__ R result() const { return peak == -INFINITY || peak == INFINITY ? peak : peak + (shift + logOf(total)); }
  __device__ R share(int j) const { return weight[j] == -INFINITY || peak == -INFINITY ? R(0) : term[j] / total; }
};

template <typename T, int K, bool EXACT>
__device__ inline void storeSlots(T* to, size_t row, unsigned k, const Pack<T, K>& v) {
  if constexpr (EXACT) {
    *reinterpret_cast<Pack<T, K>*>(to + row * K) = v;
  } else {
#pragma unroll
    for (int j = 0; j < K; ++j)
      if (j < int(k)) to[row * k + j] = v.v[j];
  }
}

template <int K> constexpr int LOG_ROWS = K <= 2 ? 2 : 1;  // of a thread

template <typename R, typename W, int K, bool EXACT>
__global__ __launch_bounds__(BLOCK) void combineLogKernel(const R* __restrict__ values, size_t capacity, const int32_t* __restrict__ position,
                                                          const W* __restrict__ logWeight, size_t n, unsigned k, R* __restrict__ out,
                                                          R* __restrict__ shares) {
  constexpr int ROWS = LOG_ROWS<K>;
  forTiles((n + ROWS * BLOCK - 1) / (ROWS * BLOCK), gridDim.x, true, [&](size_t tile) {
    const size_t first = tile * (ROWS * BLOCK) + threadIdx.x;
    LogRow<R, W, K, EXACT> r[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) r[i].slots(position, logWeight, first + i * BLOCK < n ? first + i * BLOCK : n - 1, k, capacity);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) r[i].values(values);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const size_t row = first + i * BLOCK;
      if (row >= n) continue;
      r[i].solve();
      out[row] = r[i].result();
      if (shares) {
        Pack<R, K> o;
#pragma unroll
        for (int j = 0; j < K; ++j) o.v[j] = r[i].share(j);
        storeSlots<R, K, EXACT>(shares, row, k, o);
      }
    }
  });
}

// dv[position_ij] = dl_ij = g_i times the share that the forward pass wrote: nothing is gathered again. A share of 0 passes no gradient
// whatever g is: its slot may have been left out. 4 M rows of two slots take 34 us, bound by
// the scatter, and 16 us, 5.2 TB/s, without the values' gradient (compiled kernels want none); 41 where values and weights are read again.
template <typename R, typename W, int K, bool EXACT>
__global__ __launch_bounds__(BLOCK) void combineLogBackwardKernel(const R* __restrict__ shares, const int32_t* __restrict__ position, size_t n, unsigned k,
                                                                  size_t capacity, const R* __restrict__ gradOut, R* __restrict__ gradValues,
                                                                  W* __restrict__ gradLogWeight, Unused unused) {
  if (blockIdx.x >= unused.rowBlocks) return clearUnused(unused);
  constexpr int ROWS = LOG_ROWS<K>;
  forTiles((n + ROWS * BLOCK - 1) / (ROWS * BLOCK), unused.rowBlocks, true, [&](size_t tile) {
    const size_t first = tile * (ROWS * BLOCK) + threadIdx.x;
    Pack<R, K> share[ROWS];
    int32_t at[ROWS][K];
    R g[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const size_t row = first + i * BLOCK < n ? first + i * BLOCK : n - 1;
      g[i] = gradOut[row];
      Pack<int32_t, K> p;
      if constexpr (EXACT) {
        share[i] = *reinterpret_cast<const Pack<R, K>*>(shares + row * K);
        if (gradValues) p = *reinterpret_cast<const Pack<int32_t, K>*>(position + row * K);
      } else {
#pragma unroll
        for (int j = 0; j < K; ++j) {
          share[i].v[j] = j < int(k) ? shares[row * k + j] : R(0);
          if (gradValues) p.v[j] = j < int(k) ? position[row * k + j] : -1;
        }
      }
#pragma unroll
      for (int j = 0; j < K; ++j) at[i][j] = gradValues && p.v[j] >= 0 && size_t(p.v[j]) < capacity ? p.v[j] : -1;
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const size_t row = first + i * BLOCK;
      if (row >= n) continue;
      Pack<W, K> o;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const R d = share[i].v[j] == 0 ? R(0) : g[i] * share[i].v[j];
        if (at[i][j] >= 0) gradValues[at[i][j]] = d;
        o.v[j] = W(d);
      }
      if (gradLogWeight) storeSlots<W, K, EXACT>(gradLogWeight, row, k, o);
    }
  });
}

// Any number of slots, read again for every use: one thread a row, three passes over its slots and a fourth for the shares, neighbouring lanes
// k slots apart. Simple and far from its bytes: 262144 rows of 16 slots take 477 us and 147 for the gradients (11 us each at 6.2 TB/s), of 64 slots
// 3526 and 884 (44 us each).
template <typename R, typename W>
struct LogSlots {
  const R* values;
  size_t capacity;
  const int32_t* position;
  const W* logWeight;
  unsigned k;
  R peak, shift, total;

  __device__ bool read(size_t s, R& v, R& lw, int32_t& at) const {
    at = position[s];
    if (at >= 0 && size_t(at) >= capacity) at = -1;
    lw = at >= 0 ? R(logWeight[s]) : R(-INFINITY);
    if (lw == -INFINITY) return false;
    v = values[at];
    return true;
  }
  __device__ void solve(size_t row) {
    peak = shift = -INFINITY;
    total = 0;
    R v, lw;
    int32_t at;
    for (unsigned j = 0; j < k; ++j)
      if (read(row * k + j, v, lw, at)) peak = v > peak || v != v ? v : peak;
    if (peak == -INFINITY) return;  // nothing possible
    for (unsigned j = 0; j < k; ++j)
      if (read(row * k + j, v, lw, at)) {
        const R t = lw + (v - peak);
        shift = t > shift || t != t ? t : shift;
      }
    for (unsigned j = 0; j < k; ++j)
      if (read(row * k + j, v, lw, at)) total += expOf(lw + (v - peak) - shift);
  }
};

template <typename R, typename W>
__global__ __launch_bounds__(BLOCK) void combineLogManyKernel(LogSlots<R, W> given, size_t n, R* __restrict__ out, R* __restrict__ shares) {
  forTiles((n + BLOCK - 1) / BLOCK, gridDim.x, true, [&](size_t tile) {
    const size_t row = tile * BLOCK + threadIdx.x;
    if (row >= n) return;
    LogSlots<R, W> r = given;
    r.solve(row);
    out[row] = r.peak == -INFINITY || r.peak == INFINITY ? r.peak : r.peak + (r.shift + logOf(r.total));
    if (!shares) return;
    for (unsigned j = 0; j < r.k; ++j) {
      R v, lw, share = 0;
      int32_t at;
      if (r.read(row * r.k + j, v, lw, at) && r.peak != -INFINITY) share = expOf(lw + (v - r.peak) - r.shift) / r.total;
      shares[row * r.k + j] = share;
    }
  });
}

template <typename R, typename W>
__global__ __launch_bounds__(BLOCK) void combineLogManyBackwardKernel(const R* __restrict__ shares, const int32_t* __restrict__ position, size_t n,
                                                                      unsigned k, size_t capacity, const R* __restrict__ gradOut,
                                                                      R* __restrict__ gradValues, W* __restrict__ gradLogWeight, Unused unused) {
  if (blockIdx.x >= unused.rowBlocks) return clearUnused(unused);
  forTiles((n + BLOCK - 1) / BLOCK, unused.rowBlocks, true, [&](size_t tile) {
    const size_t row = tile * BLOCK + threadIdx.x;
    if (row >= n) return;
    const R g = gradOut[row];
    for (size_t s = row * k; s < row * k + k; ++s) {
      const R d = shares[s] == 0 ? R(0) : g * shares[s];
      if (gradValues) {
        const int32_t at = position[s];
        if (at >= 0 && size_t(at) < capacity) gradValues[at] = d;
      }
      if (gradLogWeight) gradLogWeight[s] = W(d);
    }
  });
}

// ---- host side ------------------------------------------------------------------------------------------------------

template <typename Fn>
void withItems(unsigned items, Fn&& fn) {
  if (items == 2) return fn(std::integral_constant<int, 2>());
  if (items == 4) return fn(std::integral_constant<int, 4>());
  fn(std::integral_constant<int, 8>());
}

void checkSlots(size_t n, unsigned k, size_t capacity) {
  if (k == 0) refuse("k must be at least 1");
  if (n > ((size_t(1) << 31) - 1) / k) refuse("too many slots: n * k must be below 2^31");
  if (capacity >= (size_t(1) << 31)) refuse("too many rows: the capacity must be below 2^31");
}

void checkWeightType(int dtype, int weightDtype) {
  if (weightDtype != SPNC_HIP_FLOAT32 && !(weightDtype == SPNC_HIP_FLOAT64 && dtype == SPNC_HIP_FLOAT64))
    refuse("weights must be float32, or float64 with float64 values");
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

// Fewer rows than the chip has places for waves: a row is spread over a block. Eight rows of 4096 bfloat16 go to four places each in
// 3.9 us instead of 6.7 and are combined in 3.6 instead of 6.0, of 16384 in 7.1 instead of 20.5 and 5.8 instead of 15.6. The gradient of
// combine keeps a wave a row, whose dot products stay in the wave: 11 us and 35 us there.
constexpr size_t FEW_ROWS = 2048;

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

Span startsBlock(const int32_t* starts, unsigned experts) { return block(starts, experts ? (size_t(experts) + 1) * sizeof(int32_t) : 0); }
Span countsBlock(const int32_t* counts, unsigned experts) { return block(counts, experts * sizeof(int32_t)); }

// calls fn(K, EXACT), see LogRow; K = 0 for more than eight. W: the widest type that is read or written k at a time.
template <typename W, typename Fn>
void withLogChoices(unsigned k, uintptr_t addresses, Fn&& fn) {
  const bool exact = (k & (k - 1)) == 0 && addresses % (k * sizeof(W) < 16 ? k * sizeof(W) : 16) == 0;
  auto choose = [&](auto kb) { exact ? fn(kb, std::true_type()) : fn(kb, std::false_type()); };
  if (k == 1) return fn(std::integral_constant<int, 1>(), std::true_type());
  if (k == 2) return choose(std::integral_constant<int, 2>());
  if (k <= 4) return choose(std::integral_constant<int, 4>());
  if (k <= 8) return choose(std::integral_constant<int, 8>());
  fn(std::integral_constant<int, 0>(), std::false_type());
}

// the blocks of the kernel that withLogChoices picks
inline unsigned logGrid(size_t n, unsigned k) {
  const size_t rows = BLOCK * (k <= 2 ? LOG_ROWS<2> : 1);
  return tileGrid((n + rows - 1) / rows);
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

size_t spnc_hip_route_workspace(size_t slots, unsigned experts) {
  if (experts == 0 || experts > SPNC_HIP_MAX_EXPERTS) return 0;  // refused by spnc_hip_route
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
    if (address(workspace) % sizeof(uint32_t)) refuse("the workspace must be aligned to 4 bytes");
    if (workspace_bytes < need || (need && !workspace)) refuse("the workspace must hold " + std::to_string(need) + " bytes");
    const Span placed = block(position, slots * sizeof(int32_t)), begins = startsBlock(starts, experts), sizes = countsBlock(counts, experts);
    const Span read = block(index, slots * sizeof(int32_t)), scratch = block(workspace, need);
    checkApart("route", placed, {read, begins, sizes, scratch});
    checkApart("route", begins, {read, sizes, scratch});
    checkApart("route", sizes, {read, scratch});
    checkApart("route", scratch, {read});
    unsigned bits = 0;
    while ((1u << bits) < experts) ++bits;
    const size_t lds = ROUTE_WAVES * experts * sizeof(uint32_t);
    withItems(shape.items, [&](auto items) {
      constexpr int ITEMS = decltype(items)::value;
      if (lds > 48 * 1024)
        for (const void* kernel : {reinterpret_cast<const void*>(routeCountKernel<ITEMS>), reinterpret_cast<const void*>(routeKernel<ITEMS>)})
          checkCall("route", hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, int(lds)));
      if (shape.blocks > 1)
        launch("route", routeCountKernel<ITEMS>, shape.blocks, ROUTE_BLOCK, lds, stream, index, slots, experts, shape.chunk, static_cast<uint32_t*>(workspace));
      launch("route", routeKernel<ITEMS>, shape.blocks, ROUTE_BLOCK, lds, stream, index, slots, experts, bits, align, shape.chunk,
             static_cast<const uint32_t*>(workspace), position, starts, counts);
    });
  });
}

int spnc_hip_dispatch(const void* rows, size_t n, size_t row_bytes, size_t stride_bytes, const int32_t* position, unsigned k, size_t capacity,
                      const int32_t* starts, const int32_t* counts, unsigned experts, int zero_unused, void* out, void* stream) {
  return guarded([&] {
    checkSlots(n, k, capacity);
    if (row_bytes >> 31) refuse("a row must be shorter than 2 GiB");
    if (zero_unused) checkSegments(starts, counts, experts);
    if (capacity == 0 || row_bytes == 0) return;
    if (!out || (n && (!rows || !position))) refuse("null argument");
    if (!zero_unused) experts = 0;  // the segments are not read
    checkApart("dispatch", block(out, capacity * row_bytes),
               {{rows, n, row_bytes, stride_bytes}, block(position, n * k * sizeof(int32_t)), startsBlock(starts, experts), countsBlock(counts, experts)});
    const unsigned piece = pieceBytes(1, {address(rows), address(out), row_bytes, stride_bytes});
    const RowShape shape = rowShape(n, row_bytes, piece, out, n < FEW_ROWS ? 8 : 6);
    const Unused unused = unusedRows(tileGrid(shape.tiles), starts, counts, experts, capacity, row_bytes, zero_unused ? out : nullptr);
    if (unused.rowBlocks + unused.blocks == 0) return;
    withPieces(piece, [&](auto p) {
      using P = decltype(p);
      withChoices(k, [&](auto kb, auto) {
        constexpr int KB = decltype(kb)::value;
        withStream<sizeof(P)>(shape, [&](auto past) {
          launch("dispatch", dispatchKernel<P, KB, decltype(past)::value>, unused.rowBlocks + unused.blocks, BLOCK, 0, stream,
                 static_cast<const unsigned char*>(rows), n, stride_bytes, shape, position, k, capacity, static_cast<P*>(out), unused);
        });
      });
    });
  });
}

int spnc_hip_combine(const void* values, int dtype, size_t capacity, size_t width, size_t stride, const int32_t* position, size_t n, unsigned k,
                     const void* weight, int weight_dtype, void* out, void* stream) {
  return guarded([&] {
    const size_t bytes = elementBytes(dtype);
    checkSlots(n, k, capacity);
    if (weight) checkWeightType(dtype, weight_dtype);
    if (width >> 31 || width * bytes >> 31) refuse("a row must be shorter than 2 GiB");
    if (n == 0 || width == 0) return;
    if ((capacity && !values) || !position || !out) refuse("null argument");
    const Span read{values, capacity, width * bytes, stride * bytes};
    if (capacity == 0) values = out, stride = width;  // no slot is routed; there has to be a row to read and drop
    const unsigned piece = pieceBytes(unsigned(bytes), {address(values), address(out), width * bytes, stride * bytes});
    checkAligned(piece, "combine");
    checkApart("combine", block(out, n * width * bytes),
               {read, block(position, n * k * sizeof(int32_t)), block(weight, weight ? n * k * elementBytes(weight_dtype) : 0)});
    const RowShape shape = rowShape(n, width * bytes, piece, nullptr, n < FEW_ROWS ? 8 : 6);
    withType(dtype, [&](auto t) {
      using T = decltype(t);
      withPack<T>(piece, [&](auto count) {
        constexpr int N = decltype(count)::value;
        withWeight<T>(weight_dtype, [&](auto w) {
          using W = decltype(w);
          withChoices(k, [&](auto kb, auto one) {
            launch("combine",
                   weight ? combineKernel<T, N, W, decltype(kb)::value, decltype(one)::value, true>
                          : combineKernel<T, N, W, decltype(kb)::value, decltype(one)::value, false>,
                   tileGrid(shape.tiles), BLOCK, 0, stream, static_cast<const T*>(values), capacity, stride, shape, position, n, k,
                   static_cast<const W*>(weight), static_cast<Pack<T, N>*>(out));
          });
        });
      });
    });
  });
}

int spnc_hip_combine_backward(const void* values, int dtype, size_t capacity, size_t width, size_t stride, const int32_t* position, size_t n,
                              unsigned k, const void* weight, int weight_dtype, const void* grad_out, size_t grad_stride, const int32_t* starts,
                              const int32_t* counts, unsigned experts, void* grad_values, void* grad_weight, void* stream) {
  return guarded([&] {
    const size_t bytes = elementBytes(dtype);
    checkSlots(n, k, capacity);
    checkWeightType(dtype, weight_dtype);
    if (width >> 31 || width * bytes >> 31) refuse("a row must be shorter than 2 GiB");
    if (grad_values) checkSegments(starts, counts, experts);
    if (!grad_values && !grad_weight) return;
    if (n && ((capacity && width && !values) || !position || !weight || (width && !grad_out))) refuse("null argument");
    const unsigned piece = pieceBytes(unsigned(bytes), {address(values), address(grad_out), address(grad_values), width * bytes, stride * bytes,
                                                        grad_stride * bytes});
    checkAligned(piece, "combine gradient");
    const size_t weightBytes = n * k * elementBytes(weight_dtype);
    const Span toValues = block(grad_values, capacity * width * bytes), toWeight = block(grad_weight, weightBytes);
    const Span read{values, grad_weight ? capacity : 0, width * bytes, stride * bytes}, gradient{grad_out, n, width * bytes, grad_stride * bytes};
    const Span slots = block(position, n * k * sizeof(int32_t)), weights = block(weight, weightBytes);
    const Span begins = startsBlock(starts, grad_values ? experts : 0), sizes = countsBlock(counts, grad_values ? experts : 0);
    checkApart("combine gradient", toValues, {read, gradient, slots, weights, begins, sizes, toWeight});
    checkApart("combine gradient", toWeight, {read, gradient, slots, weights, begins, sizes});
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
              launch("combine gradient", combineBackwardKernel<T, N, W, decltype(kb)::value, decltype(past)::value>, unused.rowBlocks + unused.blocks,
                     BLOCK, 0, stream, static_cast<const T*>(values), capacity, stride, shape, position, n, k, static_cast<const W*>(weight),
                     static_cast<const T*>(grad_out), grad_stride, static_cast<Pack<T, N>*>(grad_values), static_cast<W*>(grad_weight), unused);
            });
          });
        });
      });
    });
  });
}

int spnc_hip_combine_log(const void* values, int dtype, size_t capacity, const int32_t* position, size_t n, unsigned k, const void* log_weight,
                         int weight_dtype, void* out, void* share, void* stream) {
  return guarded([&] {
    checkLogTypes(dtype, weight_dtype);
    checkSlots(n, k, capacity);
    if (n == 0) return;
    if ((capacity && !values) || !position || !log_weight || !out) refuse("null argument");
    const size_t bytes = elementBytes(dtype);
    const Span read = block(values, capacity * bytes), slots = block(position, n * k * sizeof(int32_t));
    const Span weights = block(log_weight, n * k * elementBytes(weight_dtype)), shares = block(share, n * k * bytes);
    checkApart("combine_log", block(out, n * bytes), {read, slots, weights, shares});
    checkApart("combine_log", shares, {read, slots, weights});
    if (capacity == 0) values = out;  // no slot is routed; there has to be a value to read and drop
    withLogTypes(dtype, weight_dtype, [&](auto r, auto w) {
      using R = decltype(r);
      using W = decltype(w);
      using Widest = typename std::conditional<(sizeof(R) > sizeof(W)), R, W>::type;
      withLogChoices<Widest>(k, address(position) | address(log_weight) | address(share), [&](auto kb, auto exact) {
        constexpr int K = decltype(kb)::value;
        if constexpr (K > 0)
          launch("combine_log", combineLogKernel<R, W, K, decltype(exact)::value>, logGrid(n, k), BLOCK, 0, stream, static_cast<const R*>(values), capacity,
                 position, static_cast<const W*>(log_weight), n, k, static_cast<R*>(out), static_cast<R*>(share));
        else
          launch("combine_log", combineLogManyKernel<R, W>, logGrid(n, k), BLOCK, 0, stream,
                 LogSlots<R, W>{static_cast<const R*>(values), capacity, position, static_cast<const W*>(log_weight), k}, n, static_cast<R*>(out),
                 static_cast<R*>(share));
      });
    });
  });
}

int spnc_hip_combine_log_backward(const void* share, int dtype, size_t capacity, const int32_t* position, size_t n, unsigned k, int weight_dtype,
                                  const void* grad_out, const int32_t* starts, const int32_t* counts, unsigned experts, void* grad_values,
                                  void* grad_log_weight, void* stream) {
  return guarded([&] {
    checkLogTypes(dtype, weight_dtype);
    checkSlots(n, k, capacity);
    if (grad_values) checkSegments(starts, counts, experts);
    if (!grad_values && !grad_log_weight) return;
    if (n && (!share || (grad_values && !position) || !grad_out)) refuse("null argument");
    const size_t bytes = elementBytes(dtype);
    const Span toValues = block(grad_values, capacity * bytes), toWeight = block(grad_log_weight, n * k * elementBytes(weight_dtype));
    const Span read = block(share, n * k * bytes), gradient = block(grad_out, n * bytes), slots = block(position, grad_values ? n * k * sizeof(int32_t) : 0);
    const Span begins = startsBlock(starts, grad_values ? experts : 0), sizes = countsBlock(counts, grad_values ? experts : 0);
    checkApart("combine_log gradient", toValues, {read, gradient, slots, begins, sizes, toWeight});
    checkApart("combine_log gradient", toWeight, {read, gradient, slots, begins, sizes});
    const Unused unused = unusedRows(logGrid(n, k), starts, counts, experts, capacity, bytes, grad_values);
    if (unused.rowBlocks + unused.blocks == 0) return;
    withLogTypes(dtype, weight_dtype, [&](auto r, auto w) {
      using R = decltype(r);
      using W = decltype(w);
      using Widest = typename std::conditional<(sizeof(R) > sizeof(W)), R, W>::type;
      withLogChoices<Widest>(k, address(share) | address(grad_log_weight) | (grad_values ? address(position) : 0), [&](auto kb, auto exact) {
        constexpr int K = decltype(kb)::value;
        if constexpr (K > 0)
          launch("combine_log gradient", combineLogBackwardKernel<R, W, K, decltype(exact)::value>, unused.rowBlocks + unused.blocks, BLOCK, 0, stream,
                 static_cast<const R*>(share), position, n, k, capacity, static_cast<const R*>(grad_out), static_cast<R*>(grad_values),
                 static_cast<W*>(grad_log_weight), unused);
        else
          launch("combine_log gradient", combineLogManyBackwardKernel<R, W>, unused.rowBlocks + unused.blocks, BLOCK, 0, stream, static_cast<const R*>(share),
                 position, n, k, capacity, static_cast<const R*>(grad_out), static_cast<R*>(grad_values), static_cast<W*>(grad_log_weight), unused);
      });
    });
  });
}

}  // extern "C"
