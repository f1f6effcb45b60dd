// Scratch that could not be had: the C++ mirror forgets the one it gave back and goes on.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdio>
#include <memory>
#include <stdexcept>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#define private public
#include "../../ferro_b200/host/ferro_b200.hpp"
#undef private

#define EXPECT(cond)                                                        \
  do {                                                                      \
    if (!(cond)) { std::printf("FAIL %s:%d %s\n", __FILE__, __LINE__, #cond); return 1; } \
  } while (0)

int main() {
  fb::CudaBackend be(0);
  EXPECT(be.scratch(1 << 16) != nullptr && be.scratch_bytes_ == 1 << 16);
  bool threw = false;
  try { be.scratch(1ull << 56); } catch (const fb::Unsupported&) { threw = true; }
  EXPECT(threw && be.scratch_ == nullptr && be.scratch_bytes_ == 0);
  // a call that needs scratch, on new memory: 2 ids for 9000 assignments
  std::vector<int64_t> ids(9000);
  for (size_t i = 0; i < ids.size(); ++i) ids[i] = (int64_t)(i & 1);
  auto plan = be.moe_sort_dev(*be.alloc_i64_from_host(ids), 9000, 1, 2);
  EXPECT(be.scratch_ != nullptr);
  auto off = be.copy_i64_to_host(*plan.offsets);
  EXPECT(off[0] == 0 && off[1] == 4500 && off[2] == 9000);
  std::printf("scratch_test ok\n");
  return 0;
}
