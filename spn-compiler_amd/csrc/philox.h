// The counter-based generator Philox4x32 with ten rounds, from its published definition: J. K. Salmon, M. A. Moraes,
// R. O. Dror and D. E. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011. Host and device.
#pragma once
#include <stdint.h>

#ifndef SPN_HD
#if defined(__HIPCC__)
#define SPN_HD __host__ __device__ inline
#else
#define SPN_HD inline
#endif
#endif

namespace spnc_hip {

struct Philox4 {
  uint32_t w[4];
};

SPN_HD uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);  // one instruction instead of two
#else
  return a ^ b ^ c;
#endif
}

// c1 to c3 and the key are best the same for a whole wave: two of the first four products are then scalar.
SPN_HD Philox4 philox4x32(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    const uint64_t p0 = uint64_t(0xD2511F53u) * c0, p1 = uint64_t(0xCD9E8D57u) * c2;
    c0 = xor3(uint32_t(p1 >> 32), c1, k0);
    c1 = uint32_t(p1);
    c2 = xor3(uint32_t(p0 >> 32), c3, k1);
    c3 = uint32_t(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Philox4{{c0, c1, c2, c3}};
}

}  // namespace spnc_hip
