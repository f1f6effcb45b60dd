// The layer operators through ferro_b200/host/ferro_b200.hpp: known answers of rotary positions, dropout,
// the router's gate, the expert sort and the rows' way to the experts and back.
#include <cmath>
#include <cstdio>

#include "../../ferro_b200/host/ferro_b200.hpp"

#define EXPECT(cond)                                                        \
  do {                                                                      \
    if (!(cond)) { std::printf("FAIL %s:%d %s\n", __FILE__, __LINE__, #cond); return 1; } \
  } while (0)

int main() {
  fb::CudaBackend be(0);
  {
    // one pair at position 2 with base 1: an angle of 2 radians, and back
    auto plan = be.rope_plan(2, 1.0, FB_ROPE_HALF);
    auto x = be.alloc_from_host({3.f, 4.f, 5.f});
    auto y = be.rope_dev(*x, {1, 1, 1, 3}, plan, nullptr, 2);
    auto v = be.copy_to_host(*y);
    EXPECT(std::fabs(v[0] - (3 * std::cos(2.0) - 4 * std::sin(2.0))) < 1e-5);
    EXPECT(std::fabs(v[1] - (4 * std::cos(2.0) + 3 * std::sin(2.0))) < 1e-5);
    EXPECT(v[2] == 5.f);
    auto b = be.copy_to_host(*be.rope_backward_dev(*y, {1, 1, 1, 3}, plan, nullptr, 2));
    EXPECT(std::fabs(b[0] - 3.f) < 1e-5 && std::fabs(b[1] - 4.f) < 1e-5 && b[2] == 5.f);
    bool threw = false;
    try { be.rope_dev(*x, {1, 1, 1, 4}, plan, nullptr, 0); } catch (const fb::InvalidShape&) { threw = true; }
    EXPECT(threw);
  }
  {
    // Philox4x32-10 at counter 0 under key 0: 6627e8d5 e169c58d bc57ac4c 9b00dbd8; p = 0.5 keeps words from 2^31
    auto x = be.alloc_from_host({1.f, 2.f, 3.f, 4.f}), r = be.alloc_from_host({10.f, 20.f, 30.f, 40.f}), b = be.alloc_from_host({1.f, 1.f});
    auto v = be.copy_to_host(*be.dropout_dev(*x, b.get(), r.get(), 2, 2, 0.5f, 0, 0));
    EXPECT(v[0] == 10.f && v[1] == 26.f && v[2] == 38.f && v[3] == 50.f);
    auto [dx, db] = be.dropout_backward_dev(*x, 2, 2, 0.5f, 0, 0);
    auto d = be.copy_to_host(*dx), s = be.copy_to_host(*db);
    EXPECT(d[0] == 0.f && d[1] == 4.f && d[2] == 6.f && d[3] == 8.f && s[0] == 6.f && s[1] == 12.f);
  }
  {
    const float inf = INFINITY;
    auto l = be.alloc_from_host({0.f, 1.f, 1.f, -inf, -inf, -inf, std::log(3.f), 0.f, -inf});
    auto [w, ids] = be.moe_gate_dev(*l, 3, 3, 2, true);
    auto id = be.copy_i64_to_host(*ids);
    auto wt = be.copy_to_host(*w);
    EXPECT(id[0] == 1 && id[1] == 2 && id[2] == -1 && id[3] == -1 && id[4] == 0 && id[5] == 1);
    EXPECT(wt[0] == 0.5f && wt[1] == 0.5f && wt[2] == 0.f && wt[3] == 0.f && std::fabs(wt[4] - 0.75f) < 1e-6f);
    auto dw = be.alloc_from_host({1.f, 0.f, 1.f, 1.f, 1.f, 0.f});
    auto dl = be.copy_to_host(*be.moe_gate_backward_dev(*dw, *l, *w, *ids, 3, 3, 2, true));
    EXPECT(dl[0] == 0.f && dl[1] == 0.25f && dl[2] == -0.25f && dl[3] == 0.f && std::fabs(dl[6] - 0.1875f) < 1e-6f);
    auto plan = be.moe_sort_dev(*ids, 3, 2, 3);
    auto place = be.copy_i64_to_host(*plan.place), off = be.copy_i64_to_host(*plan.offsets);
    EXPECT(place[0] == 1 && place[1] == 3 && place[2] == -1 && place[3] == -1 && place[4] == 0 && place[5] == 2);
    EXPECT(off[0] == 0 && off[1] == 1 && off[2] == 3 && off[3] == 4);
    auto x = be.alloc_from_host({1.f, 2.f, 3.f});
    auto xs = be.moe_dispatch_dev(*x, plan, 1);
    auto xv = be.copy_to_host(*xs);
    EXPECT(xv[0] == 3.f && xv[1] == 1.f && xv[2] == 3.f && xv[3] == 1.f);
    auto y = be.copy_to_host(*be.moe_combine_dev(*xs, *w, plan, 1));
    EXPECT(y[0] == 1.f && y[1] == 0.f && std::fabs(y[2] - 3.f) < 1e-6f);
    auto dx = be.copy_to_host(*be.moe_dispatch_backward_dev(*xs, plan, 1));
    EXPECT(dx[0] == 2.f && dx[1] == 0.f && dx[2] == 6.f);
    auto [dys, dww] = be.moe_combine_backward_dev(*x, *xs, *w, plan, 1);
    auto dv = be.copy_to_host(*dww);
    EXPECT(dv[0] == 1.f && dv[1] == 1.f && dv[2] == 0.f && dv[3] == 0.f && dv[4] == 9.f && dv[5] == 9.f);
    be.check_experts();
    auto wrong = be.alloc_i64_from_host({2, 3, 0, -2, 1, 0});
    auto partial = be.moe_sort_dev(*wrong, 3, 2, 3);
    auto at = be.copy_i64_to_host(*partial.place);
    EXPECT(at[0] == 3 && at[1] == -1 && at[2] == 0 && at[3] == -1 && at[4] == 2 && at[5] == 1);
    std::string said;
    try { be.check_experts(); } catch (const fb::InvalidShape& e) { said = e.what(); }
    EXPECT(said.find("assignment 3 ") != std::string::npos);
    be.check_experts();  // said once
    partial.tokens = 4;  // places of three tokens
    bool refused = false;
    auto four = be.alloc_from_host({1.f, 2.f, 3.f, 4.f});
    try { be.moe_dispatch_dev(*four, partial, 1); } catch (const fb::InvalidShape&) { refused = true; }
    EXPECT(refused);
  }
  std::printf("layer_ops_test ok, %llu kernel launches\n", (unsigned long long)fb_launch_count());
  return 0;
}
