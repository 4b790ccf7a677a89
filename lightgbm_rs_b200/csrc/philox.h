// The counter-based generator of dropout; for host and device.
#pragma once

#include <cstdint>

#include "host_device.h"

namespace lgbm_b200 {
namespace experts {

// Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", 2011): ten rounds of two 32 x 32 -> 64 bit products and xors on a counter of
// 128 bits, keyed by 64 bits.
LGBM_HOST_DEVICE void philox(uint64_t block, uint64_t offset, uint32_t k0, uint32_t k1,
                             uint32_t (&words)[4]) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32);
  uint32_t c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  LGBM_UNROLL
  for (int r = 0; r < 10; ++r) {
    const uint64_t p = (uint64_t)0xD2511F53u * c0, q = (uint64_t)0xCD9E8D57u * c2;
    const uint32_t n0 = (uint32_t)(q >> 32) ^ c1 ^ k0, n2 = (uint32_t)(p >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)q;
    c3 = (uint32_t)p;
    c0 = n0;
    c2 = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  words[0] = c0;
  words[1] = c1;
  words[2] = c2;
  words[3] = c3;
}

}  // namespace experts
}  // namespace lgbm_b200
