#pragma once
#include <stdint.h>

namespace fb {

// n / d for any 32-bit n and d >= 1 with one multiply-high.  With 2^shift >= d and M = 2^32 + magic =
// (2^(32 + shift) + e) / d, 0 < e <= d, the product n M / 2^(32 + shift) exceeds n / d by
// n e / (d 2^(32 + shift)) < 1 / d: too little to reach the next whole number.
struct FastDiv {
  uint32_t d, magic, shift;
};
inline FastDiv make_fastdiv(uint32_t d) {
  FastDiv f;
  f.d = d;
  uint32_t shift = 0;
  while (shift < 32 && (1ull << shift) < d) ++shift;
  f.shift = shift;
  f.magic = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  return f;
}
__device__ __forceinline__ uint32_t fdiv(uint32_t n, const FastDiv& f) {
  return (uint32_t)(((uint64_t)__umulhi(n, f.magic) + n) >> f.shift);
}

}  // namespace fb
