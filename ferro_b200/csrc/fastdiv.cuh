#pragma once
#include <stdint.h>

namespace fb {

// n / d for n < 2^31 with one multiply-high (d >= 1).
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
