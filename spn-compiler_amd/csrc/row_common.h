// What the kernels on device-resident rows share (row_gate.hip, row_route.hip, row_dropout.hip): launch shapes, packed accesses,
// operations over groups of lanes, and argument checks of their entry points (include/spnc_hip_rows.h).
#pragma once
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <stdexcept>
#include <string>
#include <tuple>
#include <type_traits>

#include "../../include/spnc_hip_rows.h"
#include "guard.h"

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

// Tiles of rows, one a block at a time. byDie: neighbouring tiles go to one die (blocks are dealt to the dies in turn): rows that are
// neighbours in the sorted buffer come from neighbouring rows, and a cache line of narrow rows is then filled or read within one L2.
template <typename Body>
__device__ inline void forTiles(size_t tiles, unsigned grid, bool byDie, Body&& body) {
  const size_t perDie = (tiles + XCDS - 1) / XCDS;
  const size_t first = byDie ? size_t(blockIdx.x % XCDS) * perDie : 0, begin = byDie ? blockIdx.x / XCDS : blockIdx.x;
  const size_t end = byDie ? (first + perDie < tiles ? perDie : tiles > first ? tiles - first : 0) : tiles, step = byDie ? grid / XCDS : grid;
  for (size_t t = begin; t < end; t += step) body(first + t);
}

inline unsigned tileGrid(size_t tiles) {
  const size_t g = (tiles + XCDS - 1) / XCDS * XCDS;
  return unsigned(g < MAX_GRID ? g : MAX_GRID);
}

// A group of 2^shift lanes, a wave or with few rows up to a block, handles a row, a piece of up to 16 bytes a lane at a time.
//
// Rows that are written to scattered places bypass the caches where they consist of whole 64-byte halves of cache lines: 1 M rows
// of 64 bytes to two places each take 36 us instead of 53, 32769 of 2 KB to four places 53 instead of 65 (a consumer that reads
// them next loses up to half of that where they would have fit the last-level cache). Rows that share their halves must not: 1 M of 48
// bytes to two places take 70 us instead of 53, since each piece goes to memory by itself.
struct RowShape {
  unsigned pieces;  // of a row
  unsigned shift;
  size_t tiles;
  bool stream;      // scattered rows are written past the caches
  bool byDie;
};

inline RowShape rowShape(size_t n, size_t rowBytes, unsigned pieceBytes, const void* scattered = nullptr, unsigned most = 6) {
  RowShape s;
  s.pieces = unsigned(rowBytes / pieceBytes);
  s.shift = 0;
  while (s.shift < most && (1u << s.shift) < s.pieces) ++s.shift;
  const size_t rows = BLOCK >> s.shift;
  s.tiles = (n + rows - 1) / rows;
  // In the order of the blocks from 1 KB on: 4 x 32769 rows of 2 KB are combined in 60 us instead of 63. 4 x 2 M rows of 8 bytes take 38
  // instead of 37 that way, of 24 bytes 93 instead of 82, and to be dispatched 114 instead of 102.
  s.byDie = rowBytes < 1024;
  s.stream = pieceBytes == 16 && rowBytes % 64 == 0 && reinterpret_cast<uintptr_t>(scattered) % 64 == 0;
  return s;
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

// The same over a whole wave for operations on words with 0 as neutral element, in fewer instructions: lane 15 of a row to the
// next row, lane 31 to the upper half, and lane 63, which then has everything, to all lanes as a scalar.
template <typename R, typename Op>
__device__ inline R waveFrom(R x, Op op) {
  x = groupFrom<1, 16>(x, op);
  x = op(x, __builtin_bit_cast(R, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x142, 0xF, 0xF, true)));  // row_bcast:15
  x = op(x, __builtin_bit_cast(R, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x143, 0xF, 0xF, true)));  // row_bcast:31
  return __builtin_bit_cast(R, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

// The sum, maximum or minimum over a group of G lanes, in all of them.
template <int G, typename R> __device__ inline R groupSum(R x) {
  auto op = [](R a, R b) { return a + b; };
  if constexpr (G == WAVE && sizeof(R) == 4) return waveFrom(x, op);
  else return groupFrom<1, G>(x, op);
}
template <int G, typename R> __device__ inline R groupMax(R x) {
  auto op = [](R a, R b) { return a > b ? a : b; };
  if constexpr (G == WAVE && std::is_same<R, uint32_t>::value) return waveFrom(x, op);
  else return groupFrom<1, G>(x, op);
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
// Without the second part: x log2(e) is rounded, an error of |x| 2^-24 relative to the result, which is that of a difference x
// already. For terms of a sum, where it is weighted with exp(x), and for results of 16 bits. The difference is taken first: a logit of
// the type's lowest value, times log2(e), would be infinite.
__device__ inline float expTerm(float x) { return __builtin_amdgcn_exp2f(x * 1.44269502f); }
__device__ inline double expTerm(double x) { return exp(x); }
__device__ inline float logOf(float x) { return logf(x); }
__device__ inline double logOf(double x) { return log(x); }

// ---- host side ------------------------------------------------------------------------------------------------------

[[noreturn]] inline void refuse(const std::string& what) { throw std::runtime_error(what); }

// Calls of the runtime return their own status, and what others left to be read by hipGetLastError is neither read nor cleared. An error
// of one's own replaces that, so it is taken back: it is reported here.
inline void checkCall(const char* what, hipError_t e) {
  if (e == hipSuccess) return;
  (void)hipGetLastError();
  refuse(std::string(what) + " launch: " + hipGetErrorString(e));
}

template <typename... P, typename... A>
void launch(const char* what, void (*kernel)(P...), unsigned grid, unsigned blockSize, size_t lds, void* stream, const A&... given) {
  std::tuple<P...> parameters(given...);
  std::apply(
      [&](P&... p) {
        void* pointers[] = {const_cast<void*>(static_cast<const void*>(&p))...};
        checkCall(what, hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(grid), dim3(blockSize), pointers, lds, static_cast<hipStream_t>(stream)));
      },
      parameters);
}

inline size_t elementBytes(int dtype) {
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
inline unsigned pieceBytes(unsigned least, std::initializer_list<uintptr_t> addresses) {
  uintptr_t bits = 16;
  for (uintptr_t a : addresses) bits |= a;
  const unsigned widest = unsigned(bits & (~bits + 1));
  return widest < least ? 0 : widest;
}

inline uintptr_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }

inline void checkAligned(unsigned piece, const char* what) {
  if (piece == 0) refuse(std::string(what) + ": pointers are not aligned to the element type");
}

// Rows of `bytes` bytes in memory, `stride` bytes apart.
struct Span {
  const void* at;
  size_t rows, bytes, stride;
};

// whether contiguous memory and rows share a byte; rows may lie around it
inline bool overlap(const void* out, size_t outBytes, const Span& in) {
  if (outBytes == 0 || in.rows == 0 || in.bytes == 0) return false;
  const uintptr_t o = address(out), r = address(in.at), step = in.stride ? in.stride : 1;
  const size_t behind = r + in.bytes > o ? 0 : (o - r - in.bytes) / step + 1;  // rows that end before it begins
  return behind < (in.stride ? in.rows : 1) && r + behind * in.stride < o + outBytes;
}

// contiguous memory
inline Span block(const void* at, size_t bytes) { return {at, at ? 1u : 0u, bytes, 0}; }

// whether rows of both share a byte; they may lie between each other
inline bool overlap(const Span& a, const Span& b) {
  if (a.rows == 0 || b.rows == 0 || a.bytes == 0 || b.bytes == 0) return false;
  if (a.rows == 1 || b.rows == 1) return a.rows == 1 ? overlap(a.at, a.bytes, b) : overlap(b.at, b.bytes, a);
  if (a.stride == b.stride && a.stride >= a.bytes && a.stride >= b.bytes) {
    const Span &low = address(a.at) <= address(b.at) ? a : b, &high = &low == &a ? b : a;
    const uintptr_t apart = address(high.at) - address(low.at), skip = apart / a.stride, rest = apart % a.stride;
    return (skip < low.rows && rest < low.bytes) || (skip + 1 < low.rows && a.stride - rest < high.bytes);
  }
  if (!overlap(a.at, (a.rows - 1) * a.stride + a.bytes, b)) return false;
  for (size_t i = 0; i < a.rows; ++i)
    if (overlap(static_cast<const char*>(a.at) + i * a.stride, a.bytes, b)) return true;
  return false;
}

// Kernels read through __restrict__ pointers, and while others write: no output lies in an input or in another output.
inline void checkApart(const char* what, const Span& out, std::initializer_list<Span> others) {
  for (const Span& other : others)
    if (overlap(out, other)) refuse(std::string(what) + ": an output overlaps an input or another output");
}

inline void checkExperts(unsigned experts) {
  if (experts == 0 || experts > SPNC_HIP_MAX_EXPERTS) refuse("experts must be between 1 and " + std::to_string(SPNC_HIP_MAX_EXPERTS));
}

}  // namespace
}  // namespace spnc_hip
