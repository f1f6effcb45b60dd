// Plans made by hand: the C++ mirror refuses a rotary plan whose table does not fit it, before any launch.
#include <cstdio>

#include "../../ferro_b200/host/ferro_b200.hpp"

#define EXPECT(cond)                                                        \
  do {                                                                      \
    if (!(cond)) { std::printf("FAIL %s:%d %s\n", __FILE__, __LINE__, #cond); return 1; } \
  } while (0)

template <typename E, typename F>
static bool throws(F f) {
  try { f(); } catch (const E&) { return true; }
  return false;
}

int main() {
  fb::CudaBackend be(0);
  auto x = be.alloc_from_host({1.f, 2.f, 3.f, 4.f, 5.f, 6.f, 7.f, 8.f});
  const std::vector<uint64_t> shape = {1, 1, 1, 8};
  const auto launches = fb_launch_count();
  fb::RopePlan shorter{be.alloc_i64_from_host({1, 2, 3}), 8, FB_ROPE_HALF, 1.f};
  EXPECT(throws<fb::InvalidShape>([&] { be.rope_dev(*x, shape, shorter, nullptr); }));
  EXPECT(throws<fb::InvalidShape>([&] { be.rope_backward_dev(*x, shape, shorter, nullptr); }));
  fb::RopePlan floats{be.alloc_from_host({1.f, 2.f, 3.f, 4.f}), 8, FB_ROPE_HALF, 1.f};
  EXPECT(throws<fb::Unsupported>([&] { be.rope_dev(*x, shape, floats, nullptr); }));
  fb::RopePlan none{nullptr, 8, FB_ROPE_HALF, 1.f};
  EXPECT(throws<fb::InvalidShape>([&] { be.rope_dev(*x, shape, none, nullptr); }));
  EXPECT(fb_launch_count() == launches);
  auto plan = be.rope_plan(8, 10000.0, FB_ROPE_HALF);
  auto y = be.copy_to_host(*be.rope_dev(*x, shape, plan, nullptr));  // position 0 turns nothing
  for (int i = 0; i < 8; ++i) EXPECT(y[i] == 1.f + i);
  std::printf("layer_plans_test ok\n");
  return 0;
}
