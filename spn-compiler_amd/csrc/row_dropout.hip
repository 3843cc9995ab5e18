// Dropout whose mask is a function of the element's number: it is computed where it is needed and never stored.
#include "philox.h"
#include "row_common.h"

namespace spnc_hip {
namespace {

template <typename R>
struct Dropout {
  uint32_t last;  // the largest word that drops an element
  bool none;      // no word does
  R scale, fill;
  uint64_t seed, offset;
  const uint64_t* offsetDevice;

  __device__ Philox4 words(uint32_t low, uint32_t high, uint64_t at) const {
    return philox4x32(low, high, uint32_t(at), uint32_t(at >> 32), uint32_t(seed), uint32_t(seed >> 32));
  }
  template <typename T>
  __device__ T apply(uint32_t word, T x) const {
    return T(word > last || none ? R(x) * scale : fill);
  }
};

template <typename T> constexpr int DROPOUT_UNIT = sizeof(T) == 2 ? 8 : 4;  // elements of a thread: 16 bytes, at least the four of one counter

// Contiguous elements; VEC: read and written 16 bytes at a time. One unit a thread: 4 M x 16 float32 take 88 us or 6.1 TB/s (95 with two,
// 98 with four), which is what a copy of that size reaches. For 16-bit types the generator counts, eighteen 32-bit products at a quarter of
// the rate for four elements: 33 M bfloat16 take 27 us, 23 without it (31 with two exclusive ors an instruction each and a counter
// whose upper half is a lane's own). Results stay on the ordinary way through the caches: past them the kernel alone is a
// few us faster, but what reads them next loses more than that.
template <typename T, bool VEC>
__global__ __launch_bounds__(BLOCK) void dropoutFlatKernel(const T* x, size_t elements, T* out, Dropout<wide_t<T>> d) {
  constexpr uint32_t E = DROPOUT_UNIT<T>, TILE = BLOCK * E;  // elements; TILE / 4 divides 2^32, so a tile's counters have one upper half
  using P = Pack<T, E>;
  const uint64_t at = d.offsetDevice ? *d.offsetDevice : d.offset;
  const size_t tiles = (elements + TILE - 1) / TILE;
  for (size_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const T* const from = x + tile * TILE;
    T* const to = out + tile * TILE;
    const size_t left = elements - tile * TILE;
    const uint32_t here = left < TILE ? uint32_t(left) : TILE, e = threadIdx.x * E;
    if (e >= here) continue;
    P v;
    if (VEC && e + E <= here) v = *reinterpret_cast<const P*>(from + e);
    else
#pragma unroll
      for (uint32_t q = 0; q < E; ++q)
        if (e + q < here) v.v[q] = from[e + q];
    const uint64_t counter = uint64_t(tile) * (TILE / 4);
#pragma unroll
    for (uint32_t b = 0; b < E / 4; ++b) {
      const Philox4 r = d.words(uint32_t(counter) + e / 4 + b, uint32_t(counter >> 32), at);
#pragma unroll
      for (int q = 0; q < 4; ++q) v.v[4 * b + q] = d.apply(r.w[q], v.v[4 * b + q]);
    }
    if (VEC && e + E <= here) *reinterpret_cast<P*>(to + e) = v;
    else
#pragma unroll
      for (uint32_t q = 0; q < E; ++q)
        if (e + q < here) to[e + q] = v.v[q];
  }
}

// Rows that are not adjacent; VEC: widths, strides and addresses in multiples of four elements, so that a counter's four
// elements are neighbours. Otherwise a counter whose elements lie in two rows is computed for both.
template <typename T, bool VEC>
__global__ __launch_bounds__(BLOCK) void dropoutRowsKernel(const T* x, size_t n, size_t width, size_t stride, T* out, size_t outStride, RowShape shape,
                                                           Dropout<wide_t<T>> d) {
  const uint64_t at = d.offsetDevice ? *d.offsetDevice : d.offset;
  const unsigned lane = threadIdx.x & ((1u << shape.shift) - 1);
  forTiles(shape.tiles, gridDim.x, false, [&](size_t tile) {
    const size_t row = tile * (BLOCK >> shape.shift) + (threadIdx.x >> shape.shift);
    if (row >= n) return;
    const size_t begin = row * width, end = begin + width;
    const T* from = x + row * stride;
    T* to = out + row * outStride;
    for (size_t b = begin / 4 + lane; 4 * b < end; b += size_t(1) << shape.shift) {
      const Philox4 r = d.words(uint32_t(b), uint32_t(b >> 32), at);
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

}  // namespace
}  // namespace spnc_hip

using namespace spnc_hip;

extern "C" {

int spnc_hip_dropout(const void* x, int dtype, size_t n, size_t width, size_t stride, void* out, size_t out_stride, double p, int mode,
                     uint64_t seed, uint64_t offset, const uint64_t* offset_device, void* stream) {
  return guarded([&] {
    elementBytes(dtype);
    if (!(p >= 0.0 && p <= 1.0)) refuse("the probability of dropping an element must be between 0 and 1");
    if (mode < SPNC_HIP_DROPOUT_ZERO || mode > SPNC_HIP_DROPOUT_MASK) refuse("unknown dropout mode " + std::to_string(mode));
    if (n > 1 && (stride < width || out_stride < width)) refuse("rows overlap");
    if (n == 0 || width == 0) return;
    if (!x || !out) refuse("null argument");
    if ((address(x) | address(out)) % elementBytes(dtype)) refuse("dropout: pointers are not aligned to the element type");
    const size_t bytes = elementBytes(dtype);
    const Span read{x, n, width * bytes, stride * bytes}, written{out, n, width * bytes, out_stride * bytes};
    if (x != out || (n > 1 && stride != out_stride)) checkApart("dropout", written, {read});  // in place every element is read by who writes it
    checkApart("dropout", written, {block(offset_device, sizeof(uint64_t))});
    const uint64_t threshold = uint64_t(std::llrint(p * 4294967296.0));
    const double scale = mode != SPNC_HIP_DROPOUT_ZERO ? 1.0 : threshold >> 32 ? 0.0 : 1.0 / (1.0 - p);
    const double fill = mode == SPNC_HIP_DROPOUT_MARGINAL ? NAN : 0.0;
    withType(dtype, [&](auto t) {
      using T = decltype(t);
      using R = wide_t<T>;
      const Dropout<R> d{uint32_t(threshold - 1), threshold == 0, R(scale), R(fill), seed, offset, offset_device};
      const uintptr_t bits = address(x) | address(out);
      const T* const from = static_cast<const T*>(x);
      T* const to = static_cast<T*>(out);
      if (n == 1 || (stride == width && out_stride == width)) {
        constexpr int E = DROPOUT_UNIT<T>;
        const size_t elements = n * width, blocks = (elements + BLOCK * E - 1) / (BLOCK * E);
        const bool vec = bits % (sizeof(Pack<T, E>) < 16 ? sizeof(Pack<T, E>) : 16) == 0;
        launch("dropout", vec ? dropoutFlatKernel<T, true> : dropoutFlatKernel<T, false>, unsigned(blocks < MAX_GRID ? blocks : MAX_GRID), BLOCK, 0, stream, from,
               elements, to, d);
      } else {
        const RowShape shape = rowShape(n, (width + 3) / 4, 1);
        const bool vec = ((width | stride | out_stride) % 4 | bits % (4 * sizeof(T) < 16 ? 4 * sizeof(T) : 16)) == 0;
        launch("dropout", vec ? dropoutRowsKernel<T, true> : dropoutRowsKernel<T, false>, tileGrid(shape.tiles), BLOCK, 0, stream, from, n, width, stride, to,
               out_stride, shape, d);
      }
    });
  });
}

}  // extern "C"
