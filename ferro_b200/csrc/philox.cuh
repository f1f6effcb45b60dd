// Philox4x32-10, the counter-based generator of Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3" (SC 2011): ten rounds of two
// 32 x 32 -> 64 bit products over a four-word counter, the two-word key moved on
// by a Weyl sequence between rounds.
#pragma once
#include <stdint.h>

namespace fb {

__host__ __device__ __forceinline__ void philox_round(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
  const uint64_t p = (uint64_t)0xD2511F53u * c[0], q = (uint64_t)0xCD9E8D57u * c[2];
  const uint32_t a = (uint32_t)(q >> 32) ^ c[1] ^ k0, b = (uint32_t)(p >> 32) ^ c[3] ^ k1;
  c[0] = a;
  c[1] = (uint32_t)q;
  c[2] = b;
  c[3] = (uint32_t)p;
}
// The four words at counter n (upper two counter words 0) under `key`.
__host__ __device__ __forceinline__ void philox4(uint64_t n, uint64_t key, uint32_t (&c)[4]) {
  c[0] = (uint32_t)n;
  c[1] = (uint32_t)(n >> 32);
  c[2] = 0;
  c[3] = 0;
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    philox_round(c, k0, k1);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

}  // namespace fb
