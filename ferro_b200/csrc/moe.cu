// The memory-bound half of a layer of routed experts: the router's choice, the
// stable sort of its assignments by expert, and the movement of token rows to
// their experts' rows and back, forward and backward.
//
// Every row that is written has one writer, every sum a fixed order (choices of a
// token ascending), integers are counted with commutative adds only: results do
// not depend on scheduling.
#include "common.cuh"
#include "fastdiv.cuh"
#include "math.cuh"
#include "reduce.cuh"

namespace fb {

// ---------------------------------------------------------------- gate
// A logit is turned into an unsigned key whose order is the order of choice: -inf
// (masked) lowest, then the finite values ascending, +inf, NaN highest.  Adding +0
// first makes -0 and +0 the same key and every NaN the one positive NaN the adder
// returns.
constexpr uint32_t kGateMasked = 0x007fffffu;  // the key of -inf
__device__ __forceinline__ uint32_t gate_key(float v) {
  const int32_t u = __float_as_int(v + 0.0f);
  return (uint32_t)u ^ ((uint32_t)(u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float gate_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

constexpr int kGateThreads = 128;
constexpr int kGateWarps = kGateThreads / 32;

// Choice j of a row for lane j (-1 where there is none): k rounds of a warp-wide maximum over whole
// keys, then of the lowest index among the lanes that hold it.
template <int NPL>
__device__ __forceinline__ int32_t gate_choose_exact(const float* __restrict__ row, uint32_t experts, uint32_t k, int lane) {
  uint32_t key[NPL];
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    const uint32_t e = i * 32 + lane;
    key[i] = e < experts ? gate_key(__ldca(row + e)) : 0u;
  }
  int32_t mine = -1;
  for (uint32_t j = 0; j < k; ++j) {
    uint32_t lb = 0, li = 0;
#pragma unroll
    for (int i = 0; i < NPL; ++i)
      if (key[i] > lb) {
        lb = key[i];
        li = i * 32 + lane;
      }
    const uint32_t win = __reduce_max_sync(0xffffffffu, lb);
    if (win <= kGateMasked) break;
    const uint32_t id = __reduce_min_sync(0xffffffffu, lb == win ? li : 0xffffffffu);
    if ((uint32_t)lane == j) mine = (int32_t)id;
#pragma unroll
    for (int i = 0; i < NPL; ++i)
      if (i * 32 + lane == id) key[i] = 0;
  }
  return mine;
}

// e^x for x <= 0: 2^(x log2 e) with the rounding of that product put back, so what is left is the
// instruction's 2^-22 whatever x is.  Results below 2^-126 are 0.  NaN stays NaN.
__device__ __forceinline__ float gate_exp(float x) {
  x = fmax_nan(x, -200.0f);  // -inf would turn the correction into a NaN
  const float t = x * 1.4426950408889634f;
  float r = fmaf(x, 1.4426950408889634f, -t);
  r = fmaf(x, 1.925963033500e-8f, r);  // log2 e - its f32 value
  const float e = ex2_approx_ftz(t);
  return fmaf(e, r * 0.6931471805599453f, e);
}

// ---- lists in registers, largest first
__device__ __forceinline__ void gate_order(uint32_t& a, uint32_t& b) {
  const uint32_t hi = max(a, b), lo = min(a, b);
  a = hi;
  b = lo;
}
// Batcher's odd-even merge sort of v[LO .. LO + N) (19 exchanges for 8), as compile-time recursion.
template <int N, int LO, int R, int M>
__device__ __forceinline__ void gate_sort_merge(uint32_t (&v)[M]) {
  if constexpr (2 * R < N) {
    gate_sort_merge<N, LO, 2 * R>(v);
    gate_sort_merge<N, LO + R, 2 * R>(v);
#pragma unroll
    for (int i = LO + R; i + R < LO + N; i += 2 * R) gate_order(v[i], v[i + R]);
  } else {
    gate_order(v[LO], v[LO + R]);
  }
}
template <int N, int LO, int M>
__device__ __forceinline__ void gate_sort(uint32_t (&v)[M]) {
  if constexpr (N > 1) {
    gate_sort<N / 2, LO>(v);
    gate_sort<N / 2, LO + N / 2>(v);
    gate_sort_merge<N, LO, 1>(v);
  }
}
// a = the N largest of two sorted lists, sorted: the larger of a_i and b_(N-1-i) are those N and form a
// bitonic sequence.
template <int N>
__device__ __forceinline__ void gate_merge(uint32_t (&a)[N], const uint32_t (&b)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = max(a[i], b[N - 1 - i]);
#pragma unroll
  for (int s = N / 2; s >= 1; s /= 2)
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((i & s) == 0) gate_order(a[i], a[i + s]);
}
// The N largest of v, sorted; the lists of N are sorted and merged one after the other.
template <int N, int LO, int M>
__device__ __forceinline__ void gate_top(uint32_t (&v)[M], uint32_t (&top)[N]) {
  if constexpr (LO < M) {
    gate_sort<N, LO>(v);
    uint32_t b[N];
#pragma unroll
    for (int i = 0; i < N; ++i) b[i] = v[LO + i];
    if constexpr (LO == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) top[i] = b[i];
    } else {
      gate_merge<N>(top, b);
    }
    gate_top<N, LO + N>(v, top);
  }
}

// L lanes of a warp hold a token's row, V values each.  Where the row is read in vectors of 4, register
// r of lane l is expert (r / 4) * 4 L + 4 l + r % 4, else r L + l.
template <int L, int V>
__device__ __forceinline__ uint32_t gate_expert(int r, int l, bool vec) {
  return V % 4 == 0 && vec ? (r / 4) * (4 * L) + 4 * l + r % 4 : r * L + l;
}
template <int L, int V>
__device__ __forceinline__ void gate_load(const float* __restrict__ row, uint32_t experts, int l, bool vec, bool live, float (&v)[V]) {
  if (V % 4 == 0 && vec) {
#pragma unroll
    for (int r = 0; r < V; r += 4) {
      const uint32_t e = gate_expert<L, V>(r, l, true);
      const float4 t = live && e < experts ? __ldca(reinterpret_cast<const float4*>(row + e)) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      v[r] = t.x;
      if constexpr (V % 4 == 0) { v[r + 1] = t.y; v[r + 2] = t.z; v[r + 3] = t.w; }
    }
  } else {
#pragma unroll
    for (int r = 0; r < V; ++r) {
      const uint32_t e = r * L + l;
      v[r] = live && e < experts ? __ldca(row + e) : -INFINITY;
    }
  }
}
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Choice through packed words: the expert's number, complemented, takes the place of the key's lowest
// bits, so that integer maxima order value, then index (ties: lowest first), and carry the index along.
// A lane sorts its values' KL largest, lists are merged across the token's L lanes by shuffles; two
// instructions an exchange instead of the five that separate keys and indices would take.
//
// The order found is exact unless entries that differ only in the bits cut off were met: two neighbours
// among the chosen that agree in the kept bits but not in value, or one left out that agrees in the
// kept bits with the last chosen.  Such a token is chosen again on whole keys by the whole warp.  The
// second condition also meets a left-out entry equal to the last chosen, whose order is right already: with
// logits rounded to bf16 32768 tokens of 128 experts, 8 choices, take 10.2 us for 7.9 (back to back in a
// graph, rows in L2), with all logits equal 22.8.
//
// Bound by the integer pipe, which issues half the rate of the others: per token of 128 experts and 8
// choices 190 instructions, 11.6 us for 32768 tokens; one warp-wide maximum per choice took 407 (16 us).
template <int KL, int L, int V>
__global__ void __launch_bounds__(kGateThreads, V <= 16 ? 8 : 4)
moe_gate_fwd_kernel(const float* __restrict__ logits, uint64_t tokens, uint32_t experts, uint32_t k, bool renorm, bool vec,
                    float* __restrict__ weights, int64_t* __restrict__ ids) {
  static_assert(KL <= L, "lane l of a token reports choice l");
  constexpr uint32_t kIds = L * V, kKept = ~(kIds - 1);  // a power of two
  constexpr int kTokens = 32 / L;                        // per warp
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % L, g = lane / L;
  const uint64_t step = (uint64_t)gridDim.x * kGateWarps * kTokens;
  for (uint64_t t0 = ((uint64_t)blockIdx.x * kGateWarps + warp) * kTokens; t0 < tokens; t0 += step) {
    const uint64_t t = t0 + g;
    const bool live = t < tokens;
    const float* row = logits + t * experts;
    float v[V];
    gate_load<L, V>(row, experts, l, vec, live, v);
    uint32_t w[V], top[KL];
#pragma unroll
    for (int r = 0; r < V; ++r) w[r] = (gate_key(v[r]) & kKept) | (kIds - 1 - gate_expert<L, V>(r, l, vec));
    {
      uint32_t c[V < KL ? KL : V];
#pragma unroll
      for (int r = 0; r < (V < KL ? KL : V); ++r) c[r] = r < V ? w[r] : 0u;
      gate_top<KL, 0>(c, top);
    }
#pragma unroll
    for (int o = 1; o < L; o <<= 1) {
      uint32_t b[KL];
#pragma unroll
      for (int i = 0; i < KL; ++i) b[i] = __shfl_xor_sync(0xffffffffu, top[i], o);
      gate_merge<KL>(top, b);
    }
    // lane l: choice l, the one behind it and the last
    uint32_t mine = 0, after = 0, last = 0;
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      if (i == l) mine = top[i];
      if (i == l + 1) after = top[i];
      if (i + 1 == (int)k) last = top[i];
    }
    const bool mine_in = l < (int)k && mine > kGateMasked;
    int32_t id = mine_in ? (int32_t)(kIds - 1 - (mine & (kIds - 1))) : -1;
    float value = mine_in ? __ldca(row + id) : 0.0f;
    const float after_value = __shfl_down_sync(0xffffffffu, value, 1);
    bool clash = false;
    if (mine_in && l + 1 < (int)k && after > kGateMasked)
      clash = ((mine ^ after) & kKept) == 0 && __float_as_uint(value + 0.0f) != __float_as_uint(after_value + 0.0f);
    // How many get as far as the last chosen in the kept bits: k, or too many.  Counted for every token,
    // with or without a last: all lanes of the warp have to meet in the shuffles.
    uint32_t reach = 0;
#pragma unroll
    for (int r = 0; r < V; ++r) reach += w[r] >= (last & kKept);
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) reach += __shfl_xor_sync(0xffffffffu, reach, o);
    clash |= last > kGateMasked && reach > k;
    const uint32_t groups = L == 32 ? 0xffffffffu : ((1u << (L & 31)) - 1u);
    uint32_t again = __ballot_sync(0xffffffffu, clash);
    while (again) {  // rare; every lane works on the token of the lowest lane that asks
      const int who = (__ffs(again) - 1) / L;
      again &= ~(groups << (who * L));
      const int32_t found = gate_choose_exact<L * V / 32>(logits + (t0 + who) * experts, experts, k, lane);
      const int32_t theirs = __shfl_sync(0xffffffffu, found, l);
      if (g == who) {
        id = l < (int)k ? theirs : -1;
        value = id >= 0 ? __ldca(row + id) : 0.0f;
      }
    }
    const float m = __shfl_sync(0xffffffffu, value, g * L);  // the largest, where there is one
    const float mass = id >= 0 ? gate_exp(value - m) : 0.0f;
    float total;
    if (renorm) {
      total = lanes_sum<L>(mass);
    } else {
      total = 0.0f;
#pragma unroll
      for (int r = 0; r < V; ++r) total += gate_exp(v[r] - m);
      total = lanes_sum<L>(total);
    }
    if (live && l < (int)k) {
      weights[t * k + l] = id >= 0 ? mass / total : 0.0f;
      ids[t * k + l] = id;
    }
  }
}

// More than 8 choices: a warp per token, k warp-wide maxima over the lanes' largest packed words, one
// more for the first left out.  A lane keeps its words sorted and moves them up when its head is taken
// (up to 8 a lane), or strikes the taken one out.  Lists of 16 merged as above would take 24.7 to 30.5 us
// for 32768 tokens, 10 choices of 32 to 128 experts.
template <int NPL>
__global__ void __launch_bounds__(kGateThreads)
moe_gate_fwd_many_kernel(const float* __restrict__ logits, uint64_t tokens, uint32_t experts, uint32_t k, bool renorm,
                         float* __restrict__ weights, int64_t* __restrict__ ids) {
  pdl_wait();
  pdl_trigger();
  constexpr uint32_t kIds = 32 * NPL, kKept = ~(kIds - 1);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (uint64_t t = (uint64_t)blockIdx.x * kGateWarps + warp; t < tokens; t += (uint64_t)gridDim.x * kGateWarps) {
    const float* row = logits + t * experts;
    float v[NPL];
    gate_load<32, NPL>(row, experts, lane, false, true, v);
    uint32_t w[NPL];
#pragma unroll
    for (int r = 0; r < NPL; ++r) w[r] = (gate_key(v[r]) & kKept) | (kIds - 1 - (r * 32 + lane));
    if constexpr (NPL <= 8) gate_sort<NPL, 0>(w);
    uint32_t mine = 0, next = 0;  // next: the first left out
    for (uint32_t j = 0;; ++j) {
      uint32_t head = w[0];
      if constexpr (NPL > 8) {
#pragma unroll
        for (int r = 1; r < NPL; ++r) head = max(head, w[r]);
      }
      const uint32_t win = __reduce_max_sync(0xffffffffu, head);
      if (j == k) {
        next = win;
        break;
      }
      mine = (uint32_t)lane == j ? win : mine;
      if constexpr (NPL <= 8) {
        const bool hit = head == win;
#pragma unroll
        for (int r = 0; r < NPL; ++r) w[r] = hit ? (r + 1 < NPL ? w[r + 1] : 0u) : w[r];
      } else {
#pragma unroll
        for (int r = 0; r < NPL; ++r) w[r] = w[r] == win ? 0u : w[r];
      }
    }
    const bool in = mine > kGateMasked;  // lanes from k on hold 0
    int32_t id = in ? (int32_t)(kIds - 1 - (mine & (kIds - 1))) : -1;
    float value = in ? __ldca(row + id) : 0.0f;
    uint32_t after = __shfl_down_sync(0xffffffffu, mine, 1);
    const float after_value = __shfl_down_sync(0xffffffffu, value, 1);
    bool clash = in && (uint32_t)lane + 1 < k && after > kGateMasked && ((mine ^ after) & kKept) == 0 &&
                 __float_as_uint(value + 0.0f) != __float_as_uint(after_value + 0.0f);
    clash |= in && (uint32_t)lane + 1 == k && next > kGateMasked && ((mine ^ next) & kKept) == 0;
    if (__any_sync(0xffffffffu, clash)) {
      id = gate_choose_exact<NPL>(row, experts, k, lane);
      value = id >= 0 ? __ldca(row + id) : 0.0f;
    }
    const float m = __shfl_sync(0xffffffffu, value, 0);
    const float mass = id >= 0 ? gate_exp(value - m) : 0.0f;
    float total = mass;
    if (!renorm) {
      total = 0.0f;
#pragma unroll
      for (int r = 0; r < NPL; ++r) total += gate_exp(v[r] - m);
    }
    total = warp_sum(total);
    if ((uint32_t)lane < k) {
      weights[t * k + lane] = id >= 0 ? mass / total : 0.0f;
      ids[t * k + lane] = id;
    }
  }
}

// L lanes per token; lane l takes choices l, l + L, ...  The row is laid out in shared memory and the
// chosen entries written over it.  A chosen entry is w_j (dw_j - sum w dw) in both forms: the saved
// weight is its probability.
template <int L, int V, int MINE>
__global__ void __launch_bounds__(kGateThreads)
moe_gate_bwd_kernel(const float* __restrict__ dweights, const float* __restrict__ logits, const float* __restrict__ weights,
                    const int64_t* __restrict__ ids, uint64_t tokens, uint32_t experts, uint32_t k, bool renorm, bool vec,
                    float* __restrict__ dlogits) {
  pdl_wait();
  pdl_trigger();
  constexpr int kTokens = 32 / L;  // MINE choices a lane
  __shared__ __align__(16) float rows[kGateThreads / L][L * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % L, g = lane / L;
  float* out = rows[warp * kTokens + g];
  const uint64_t step = (uint64_t)gridDim.x * kGateWarps * kTokens;
  for (uint64_t t0 = ((uint64_t)blockIdx.x * kGateWarps + warp) * kTokens; t0 < tokens; t0 += step) {
    const uint64_t t = t0 + g;
    const bool live = t < tokens;
    float v[V];
    if (!renorm) gate_load<L, V>(logits + t * experts, experts, l, vec, live, v);
    float w[MINE], dw[MINE], dot = 0.0f;
    int32_t id[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const uint32_t j = i * L + l;
      id[i] = -1;
      w[i] = dw[i] = 0.0f;
      if (live && j < k) {
        const int64_t e = __ldca(ids + t * k + j);
        if (e >= 0 && e < (int64_t)experts) {
          id[i] = (int32_t)e;
          w[i] = __ldca(weights + t * k + j);
          dw[i] = __ldca(dweights + t * k + j);
          dot = fmaf(w[i], dw[i], dot);
        }
      }
    }
    dot = lanes_sum<L>(dot);
    if (renorm) {
#pragma unroll
      for (int r = 0; r < V; ++r) v[r] = 0.0f;
    } else {
      float m = v[0];
#pragma unroll
      for (int r = 1; r < V; ++r) m = fmax_nan(m, v[r]);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) m = fmax_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
      // a row of nothing but masked entries: every exponent NaN, every entry 0 below
      float total = 0.0f;
      uint32_t masked = 0;
#pragma unroll
      for (int r = 0; r < V; ++r) {
        if (v[r] == -INFINITY) masked |= 1u << r;
        v[r] = v[r] == -INFINITY ? 0.0f : gate_exp(v[r] - m);
        total += v[r];
      }
      total = lanes_sum<L>(total);
      const float f = -dot / total;
#pragma unroll
      for (int r = 0; r < V; ++r) v[r] = (masked >> r) & 1 ? 0.0f : v[r] * f;
    }
    if (V % 4 == 0 && vec) {
#pragma unroll
      for (int r = 0; r < V; r += 4)
        if constexpr (V % 4 == 0) *reinterpret_cast<float4*>(out + gate_expert<L, V>(r, l, true)) = make_float4(v[r], v[r + 1], v[r + 2], v[r + 3]);
    } else {
#pragma unroll
      for (int r = 0; r < V; ++r) out[r * L + l] = v[r];
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < MINE; ++i)
      if (id[i] >= 0) out[id[i]] = w[i] * (dw[i] - dot);
    __syncwarp();
    if (live) {
      float* to = dlogits + t * experts;
      if (V % 4 == 0 && vec) {
#pragma unroll
        for (int r = 0; r < V; r += 4) {
          const uint32_t e = gate_expert<L, V>(r, l, true);
          if (e < experts) *reinterpret_cast<float4*>(to + e) = *reinterpret_cast<const float4*>(out + e);
        }
      } else {
#pragma unroll
        for (int r = 0; r < V; ++r)
          if (r * L + l < experts) to[r * L + l] = out[r * L + l];
      }
    }
    __syncwarp();
  }
}

// ---------------------------------------------------------------- sort
// Counting sort.  A CTA owns a chunk of neighbouring assignments, a warp 32 * R of them.  Within a
// warp the rank of an assignment among those of its expert comes from the lanes that hold the same id
// (ballots) plus the warp's running count; between warps and chunks counts are summed in order.
constexpr int kSortThreads = 1024;
constexpr int kSortRounds = 4;  // R where one assignment per thread would take too many chunks

__device__ __forceinline__ uint32_t sort_id(int64_t e, uint32_t experts) {
  return e >= 0 && e < (int64_t)experts ? (uint32_t)e : experts;  // `experts`: goes nowhere
}

// Lanes that hold the same id, by one ballot per bit: 10.3 us for 4096 assignments to 128 experts in one
// CTA, where the match instruction, which grows with the number of different ids, takes 12.3 us.
__device__ __forceinline__ uint32_t lanes_alike(uint32_t id, int bits) {
  uint32_t same = 0xffffffffu;
  for (int b = 0; b < bits; ++b) {
    const bool set = (id >> b) & 1;
    const uint32_t v = __ballot_sync(0xffffffffu, set);
    same &= set ? v : ~v;
  }
  return same;
}

// counts[b][e] = how many assignments of chunk b go to expert e.
template <int R>
__global__ void __launch_bounds__(kSortThreads)
moe_count_kernel(const int64_t* __restrict__ ids, uint32_t n, uint32_t experts, uint32_t* __restrict__ counts) {
  pdl_wait();  // before the trigger: moe_place_kernel relies on what this kernel waited for
  pdl_trigger();
  extern __shared__ uint32_t hist[];
  const uint32_t base = blockIdx.x * (kSortThreads * R);
  uint32_t id[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t i = base + r * kSortThreads + threadIdx.x;
    id[r] = i < n ? sort_id(__ldca(ids + i), experts) : experts;
  }
  for (uint32_t e = threadIdx.x; e < experts; e += kSortThreads) hist[e] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (id[r] < experts) atomicAdd(&hist[id[r]], 1u);
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < experts; e += kSortThreads) counts[(uint64_t)blockIdx.x * experts + e] = hist[e];
}

// In place: counts[b][e] becomes the number of e's assignments in the chunks before b, totals[e] their
// number in all.  A CTA owns 32 experts (lanes) and splits the chunks into 32 runs (warps).
__global__ void __launch_bounds__(1024)
moe_scan_kernel(uint32_t* __restrict__ counts, uint32_t chunks, uint32_t experts, uint32_t* __restrict__ totals) {
  pdl_wait();
  pdl_trigger();
  __shared__ uint32_t part[32][33];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
  const uint32_t run = (chunks + 31) / 32, lo = min(chunks, warp * run), hi = min(chunks, lo + run);
  uint32_t sum = 0;
  if (e < experts)
    for (uint32_t b = lo; b < hi; ++b) sum += counts[(uint64_t)b * experts + e];
  part[warp][lane] = sum;
  __syncthreads();
  uint32_t acc = 0;
  for (uint32_t w = 0; w < warp; ++w) acc += part[w][lane];
  if (e < experts) {
    for (uint32_t b = lo; b < hi; ++b) {
      const uint32_t c = counts[(uint64_t)b * experts + e];
      counts[(uint64_t)b * experts + e] = acc;
      acc += c;
    }
    if (warp == 31) totals[e] = acc;
  }
}

// How a CTA learns what the other chunks hold: there are none; it adds up the counts of all chunks
// (kSortDirect chunks and kSortCounts counts at most); moe_scan_kernel has left prefixes and totals.
enum { SORT_ALONE = 0, SORT_DIRECT = 1, SORT_SCANNED = 2 };
constexpr uint32_t kSortDirect = 128, kSortCounts = 32768;

// blockDim.x is a multiple of 32 and at least `experts`.
template <int R>
__global__ void __launch_bounds__(kSortThreads, 1)
moe_place_kernel(const int64_t* __restrict__ ids, uint32_t n, uint32_t experts, uint32_t chunks, int mode,
                 const uint32_t* __restrict__ counts, const uint32_t* __restrict__ totals, int64_t* __restrict__ place,
                 int64_t* __restrict__ order, int64_t* __restrict__ offsets, int64_t* __restrict__ bad) {
  extern __shared__ uint32_t sm[];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const uint32_t stride = experts | 1;  // odd: a column of hist touches every bank
  uint32_t* total = sm;                 // [experts] over all chunks, then first rows
  uint32_t* before = total + experts;   // [experts] in the chunks before this one
  uint32_t* hist = before + experts;    // [warps][stride]
  __shared__ uint32_t wsum[32];
  // Behind moe_count_kernel (or moe_scan_kernel) the ids may be read before pdl_wait: those kernels only
  // let this one start after they had waited for whatever wrote them.
  if (mode == SORT_ALONE) pdl_wait();
  pdl_trigger();
  const uint32_t base = blockIdx.x * (blockDim.x * R) + warp * 32 * R + lane;
  uint32_t id[R], rank[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t i = base + r * 32;
    id[r] = experts;
    if (i < n) {
      const int64_t e = __ldca(ids + i);
      id[r] = sort_id(e, experts);
      if (id[r] == experts && e != -1 && bad) atomicMax(reinterpret_cast<long long*>(bad), (long long)i + 1);
    }
  }
  for (uint32_t i = threadIdx.x; i < warps * stride; i += blockDim.x) hist[i] = 0;
  for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) total[e] = before[e] = 0;
  __syncthreads();
  // ranks within the warp
  uint32_t* mine = hist + warp * stride;
  const int bits = 32 - __clz(experts);  // of the largest id, `experts`
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t same = lanes_alike(id[r], bits);
    const uint32_t old = id[r] < experts ? mine[id[r]] : 0u;
    rank[r] = old + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (id[r] < experts && lane == (uint32_t)__ffs(same) - 1) mine[id[r]] = old + __popc(same);
    __syncwarp();
  }
  if (mode != SORT_ALONE) pdl_wait();
  if (mode == SORT_DIRECT) {
    // groups of `experts` threads take the chunks in turn
    const uint32_t groups = blockDim.x / experts, g = threadIdx.x / experts, e = threadIdx.x - g * experts;
    if (g < groups) {
      uint32_t all = 0, pre = 0;
      for (uint32_t b0 = g; b0 < chunks; b0 += 8 * groups) {
        uint32_t c[8];  // eight loads in flight
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = b0 + i * groups < chunks ? __ldcg(counts + (uint64_t)(b0 + i * groups) * experts + e) : 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          all += c[i];
          if (b0 + i * groups < blockIdx.x) pre += c[i];
        }
      }
      atomicAdd(&total[e], all);
      atomicAdd(&before[e], pre);
    }
  } else if (mode == SORT_SCANNED && threadIdx.x < experts) {
    total[threadIdx.x] = __ldcg(totals + threadIdx.x);
    before[threadIdx.x] = __ldcg(counts + (uint64_t)blockIdx.x * experts + threadIdx.x);
  }
  __syncthreads();
  // exclusive prefix over the warps of this CTA: a warp per expert, lanes along the warps
  for (uint32_t e = warp; e < experts; e += warps) {
    const uint32_t c = lane < warps ? hist[lane * stride + e] : 0u;
    uint32_t inc = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= (uint32_t)o) inc += up;
    }
    if (lane < warps) hist[lane * stride + e] = inc - c;
    if (lane == 31 && mode == SORT_ALONE) total[e] = inc;
  }
  __syncthreads();
  // exclusive scan over the experts (at most one per thread)
  const uint32_t v = threadIdx.x < experts ? total[threadIdx.x] : 0u;
  uint32_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= (uint32_t)o) inc += up;
  }
  if (lane == 31) wsum[warp] = inc;
  __syncthreads();
  uint32_t lower = 0;  // what the warps below hold
  {
    uint32_t s = lane < warp ? wsum[lane] : 0u;
    lower = __reduce_add_sync(0xffffffffu, s);
  }
  const uint32_t excl = inc - v + lower;
  if (threadIdx.x < experts) {
    total[threadIdx.x] = excl + before[threadIdx.x];
    if (blockIdx.x == 0) {
      offsets[threadIdx.x] = excl;
      if (threadIdx.x + 1 == experts) offsets[experts] = excl + v;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t i = base + r * 32;
    if (i >= n) continue;
    int64_t at = -1;
    if (id[r] < experts) {
      at = (int64_t)total[id[r]] + mine[id[r]] + rank[r];
      if (order) order[at] = i;
    }
    place[i] = at;
  }
}

// ---------------------------------------------------------------- rows
constexpr int kRowThreads = 256;

// What a thread moves of one row at a time: N accesses of VEC floats, `step` floats apart.  N is more
// than 1 where rows fit no 16-byte access or a token has few choices, so that the bytes in flight stay.
template <int VEC, int N>
struct RowPart {
  static_assert(VEC == 1 || VEC == 2 || VEC == 4, "floats of one access");
  float v[N][VEC];
  // The first access stands at p, the i-th exists where i < have.
  __device__ __forceinline__ void load(const float* p, uint64_t step, uint32_t have) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < (int)have) {
        const float* q = p + i * step;
        if constexpr (VEC == 4) {
          const float4 t = ld_stream4(q);
          v[i][0] = t.x; v[i][1] = t.y; v[i][2] = t.z; v[i][3] = t.w;
        } else if constexpr (VEC == 2) {
          const float2 t = __ldcs(reinterpret_cast<const float2*>(q));
          v[i][0] = t.x; v[i][1] = t.y;
        } else {
          v[i][0] = ld_stream(q);
        }
      }
  }
  __device__ __forceinline__ void store(float* p, uint64_t step, uint32_t have) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < (int)have) {
        float* q = p + i * step;
        if constexpr (VEC == 4) st_stream4(q, make_float4(v[i][0], v[i][1], v[i][2], v[i][3]));
        else if constexpr (VEC == 2) __stcs(reinterpret_cast<float2*>(q), make_float2(v[i][0], v[i][1]));
        else st_stream(q, v[i][0]);
      }
  }
};

// Where a thread stands.  A row is cut into vectors of VEC floats; `width` threads share a token, thread l
// of them takes vectors l, l + width, ... of its piece, N at a time.  Narrow rows: a CTA takes `tpb` tokens.
// Wider ones: a CTA takes a token, or, where that gives too few CTAs, one of `bpt` pieces of a token.  With
// 8192 tokens, 8 choices and 2048 columns the gather runs at 102 % of the copy rate with a CTA per token and
// at 80 % with two CTAs per token, whose halves of a row reach DRAM at different times.
struct RowMap {
  uint64_t tokens, cols, slots, blocks;
  uint32_t k, vpt;    // vectors per row
  uint32_t width;     // threads per token
  uint32_t tpb, bpt;
  uint32_t piece;     // vectors per piece (bpt > 1)
  FastDiv d_width;
};
// Token and first vector of this thread and one behind the last of its piece; false: nothing to do.
__device__ __forceinline__ bool row_place(const RowMap& M, uint64_t blk, uint64_t& t, uint32_t& vec, uint32_t& end) {
  end = M.vpt;
  if (M.tpb > 1) {
    const uint32_t tl = fdiv(threadIdx.x, M.d_width);
    vec = threadIdx.x - tl * M.width;
    t = blk * M.tpb + tl;
    return tl < M.tpb && t < M.tokens;
  }
  vec = threadIdx.x;
  t = blk;
  if (M.bpt > 1) {
    t = blk / M.bpt;
    const uint32_t lo = (uint32_t)(blk - t * M.bpt) * M.piece;
    vec += lo;
    end = min(lo + M.piece, M.vpt);
  }
  return true;
}
// How many of a thread's next N vectors lie before `end`.
template <int N>
__device__ __forceinline__ uint32_t row_have(uint32_t vec, uint32_t end, uint32_t width) {
  if (N == 1) return 1;
  uint32_t have = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) have += vec + i * width < end;
  return have;
}

__device__ __forceinline__ int64_t slot_of(const int64_t* place, uint64_t a, uint64_t slots) {
  const int64_t s = __ldca(place + a);
  return s >= 0 && (uint64_t)s < slots ? s : -1;
}

// xs[place[t, j]] = x[t], KU choices at a time: their places are loaded before the first store.
template <int VEC, int N, int KU>
__global__ void __launch_bounds__(kRowThreads, KU == 8 ? 4 : KU == 4 ? 5 : 6)
moe_scatter_kernel(const float* __restrict__ x, const int64_t* __restrict__ place, const __grid_constant__ RowMap M,
                   float* __restrict__ xs) {
  pdl_wait();
  pdl_trigger();
  const uint64_t step = (uint64_t)M.width * VEC;
  for (uint64_t blk = blockIdx.x; blk < M.blocks; blk += gridDim.x) {
    uint64_t t;
    uint32_t vec, end;
    if (!row_place(M, blk, t, vec, end)) continue;
    for (; vec < end; vec += M.width * N) {
      const uint64_t c = (uint64_t)vec * VEC;
      const uint32_t have = row_have<N>(vec, end, M.width);
      RowPart<VEC, N> v;
      v.load(x + t * M.cols + c, step, have);
      for (uint32_t j0 = 0; j0 < M.k; j0 += KU) {
        int64_t s[KU];
#pragma unroll
        for (int j = 0; j < KU; ++j) s[j] = j0 + j < M.k ? slot_of(place, t * M.k + j0 + j, M.slots) : -1;
#pragma unroll
        for (int j = 0; j < KU; ++j)
          if (s[j] >= 0) v.store(xs + (uint64_t)s[j] * M.cols + c, step, have);
      }
    }
  }
}

// y[t] = sum over j of (weights[t, j] *) ys[place[t, j]], KU rows in flight, added in the order of j.
// Bound by HBM; what counts is enough CTAs per SM (five with KU 4) to cover the load of the places.
template <int VEC, int N, int KU, bool WEIGHTED>
__global__ void __launch_bounds__(kRowThreads, KU == 8 ? 3 : N == 1 ? 5 : 4)
moe_gather_kernel(const float* __restrict__ ys, const float* __restrict__ weights, const int64_t* __restrict__ place,
                  const __grid_constant__ RowMap M, float* __restrict__ y) {
  pdl_wait();
  pdl_trigger();
  const uint64_t step = (uint64_t)M.width * VEC;
  for (uint64_t blk = blockIdx.x; blk < M.blocks; blk += gridDim.x) {
    uint64_t t;
    uint32_t vec, end;
    if (!row_place(M, blk, t, vec, end)) continue;
    for (; vec < end; vec += M.width * N) {
      const uint64_t c = (uint64_t)vec * VEC;
      const uint32_t have = row_have<N>(vec, end, M.width);
      RowPart<VEC, N> acc;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc.v[n][i] = 0.0f;
      for (uint32_t j0 = 0; j0 < M.k; j0 += KU) {
        int64_t s[KU];
        float w[KU];
#pragma unroll
        for (int j = 0; j < KU; ++j) {
          s[j] = j0 + j < M.k ? slot_of(place, t * M.k + j0 + j, M.slots) : -1;
          if (WEIGHTED) w[j] = j0 + j < M.k ? __ldca(weights + t * M.k + j0 + j) : 0.0f;
        }
        RowPart<VEC, N> r[KU];
#pragma unroll
        for (int j = 0; j < KU; ++j)
          if (s[j] >= 0) r[j].load(ys + (uint64_t)s[j] * M.cols + c, step, have);
#pragma unroll
        for (int j = 0; j < KU; ++j)
          if (s[j] >= 0) {
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
              for (int i = 0; i < VEC; ++i)
                acc.v[n][i] = WEIGHTED ? fmaf(r[j].v[n][i], w[j], acc.v[n][i]) : acc.v[n][i] + r[j].v[n][i];
          }
      }
      acc.store(y + t * M.cols + c, step, have);
    }
  }
}

// dys[place[t, j]] = weights[t, j] * dy[t]; dweights[t, j] = dy[t] . ys[place[t, j]].  A token is owned by
// `lanes` lanes of a warp (a power of two; 0: by the CTA), which walk the columns with KU rows of ys in
// flight; dy is read once per KU choices.  dys may be ys: an element is read by the thread that writes it,
// before it does.
template <int VEC, int N, int KU>
__global__ void __launch_bounds__(kRowThreads, KU == 8 ? 2 : 3)
moe_combine_bwd_kernel(const float* __restrict__ dy, const float* ys, const float* __restrict__ weights,
                       const int64_t* __restrict__ place, uint64_t tokens, uint32_t k, uint64_t cols, uint64_t slots,
                       uint32_t lanes, float* dys, float* __restrict__ dweights) {
  pdl_wait();
  pdl_trigger();
  __shared__ float part[kRowThreads / 32][KU];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const uint32_t width = lanes ? lanes : blockDim.x, l = lanes ? lane & (lanes - 1) : threadIdx.x;
  const uint32_t per_cta = lanes ? blockDim.x / lanes : 1, mine = lanes ? threadIdx.x / lanes : 0;
  const uint32_t vpt = (uint32_t)(cols / VEC);
  const uint64_t step = (uint64_t)width * VEC;
  for (uint64_t t0 = (uint64_t)blockIdx.x * per_cta; t0 < tokens; t0 += (uint64_t)gridDim.x * per_cta) {
    const uint64_t t = t0 + mine;
    const bool live = t < tokens;  // all lanes meet in the sums below
    for (uint32_t j0 = 0; j0 < k; j0 += KU) {
      int64_t s[KU];
      float w[KU], dot[KU];
#pragma unroll
      for (int j = 0; j < KU; ++j) {
        s[j] = live && j0 + j < k ? slot_of(place, t * k + j0 + j, slots) : -1;
        w[j] = live && j0 + j < k ? __ldca(weights + t * k + j0 + j) : 0.0f;
        dot[j] = 0.0f;
      }
      if (live) {
        for (uint32_t vec = l; vec < vpt; vec += width * N) {
          const uint64_t c = (uint64_t)vec * VEC;
          const uint32_t have = row_have<N>(vec, vpt, width);
          RowPart<VEC, N> g, r[KU];
          g.load(dy + t * cols + c, step, have);
          if (dweights) {
#pragma unroll
            for (int j = 0; j < KU; ++j)
              if (s[j] >= 0) r[j].load(ys + (uint64_t)s[j] * cols + c, step, have);
#pragma unroll
            for (int j = 0; j < KU; ++j)
              if (s[j] >= 0) {
#pragma unroll
                for (int n = 0; n < N; ++n)
                  if (n < (int)have) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) dot[j] = fmaf(g.v[n][i], r[j].v[n][i], dot[j]);
                  }
              }
          }
          if (dys) {
#pragma unroll
            for (int j = 0; j < KU; ++j)
              if (s[j] >= 0) {
                RowPart<VEC, N> o;
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                  for (int i = 0; i < VEC; ++i) o.v[n][i] = g.v[n][i] * w[j];
                o.store(dys + (uint64_t)s[j] * cols + c, step, have);
              }
          }
        }
      }
      if (!dweights) continue;
      if (lanes && lanes < 32) {
#pragma unroll
        for (int j = 0; j < KU; ++j)
          for (uint32_t o = lanes / 2; o > 0; o >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
#pragma unroll
        for (int j = 0; j < KU; ++j)
          if (live && l == (uint32_t)j % lanes && j0 + j < k) dweights[t * k + j0 + j] = dot[j];
        continue;
      }
      const float sum = lanes_transpose_sum<32, KU>(dot, lane);  // choice lane / (32 / KU)
      const uint32_t which = lane / (32 / KU);
      if (lanes) {
        if (live && lane % (32 / KU) == 0 && j0 + which < k) dweights[t * k + j0 + which] = sum;
      } else {
        if (lane % (32 / KU) == 0) part[warp][which] = sum;
        __syncthreads();
        if (threadIdx.x < KU && j0 + threadIdx.x < k) {
          float all = 0.0f;
          for (uint32_t i = 0; i < warps; ++i) all += part[i][threadIdx.x];
          dweights[t * k + j0 + threadIdx.x] = all;
        }
        __syncthreads();
      }
    }
  }
}

static int gate_check(const char* name, uint64_t tokens, uint64_t experts, uint64_t k) {
  uint64_t n;
  if (experts == 0 || experts > FB_MOE_MAX_EXPERTS)
    return fail(FB_ERR_INVALID_SHAPE, "%s: %llu experts, not 1 to %d", name, (unsigned long long)experts, FB_MOE_MAX_EXPERTS);
  if (k == 0 || k > experts || k > FB_MOE_MAX_K)
    return fail(FB_ERR_INVALID_SHAPE, "%s: k %llu is not 1 to min(experts, %d)", name, (unsigned long long)k, FB_MOE_MAX_K);
  if (mul_overflows(tokens, experts, &n) || n > (UINT64_MAX >> 4)) return fail(FB_ERR_INVALID_SHAPE, "%s: tokens * experts overflows", name);
  return FB_OK;
}

static int rows_check(const char* name, uint64_t tokens, uint64_t k, uint64_t cols, uint64_t slots) {
  uint64_t n;
  if (k == 0 || k > FB_MOE_MAX_K) return fail(FB_ERR_INVALID_SHAPE, "%s: k %llu is not 1 to %d", name, (unsigned long long)k, FB_MOE_MAX_K);
  if (mul_overflows(tokens, k, &n) || n > (UINT64_MAX >> 4) || mul_overflows(tokens, cols, &n) || n > (UINT64_MAX >> 3) ||
      mul_overflows(slots, cols, &n) || n > (UINT64_MAX >> 3))
    return fail(FB_ERR_INVALID_SHAPE, "%s: size overflow", name);
  if (cols >= (1ull << 31)) return fail(FB_ERR_UNSUPPORTED, "%s: rows of 2^31 or more elements are not supported", name);
  return FB_OK;
}

// Fewer CTAs than the SMs hold when each takes a token: rows are cut into pieces and all choices of a
// token taken at once, for the shortest chain of loads instead of the best stream.
static bool few_tokens(uint64_t tokens) { return tokens < (uint64_t)device_info().sm_count * 4; }

static RowMap row_map(uint64_t tokens, uint64_t k, uint64_t cols, uint64_t slots, int vec, int n, uint32_t* threads) {
  RowMap m = {};
  m.tokens = tokens;
  m.cols = cols;
  m.slots = slots;
  m.k = (uint32_t)k;
  m.vpt = (uint32_t)(cols / vec);
  m.bpt = 1;
  const uint32_t most = kRowThreads * n, rounds = (m.vpt + most - 1) / most;
  const uint32_t need = (m.vpt + rounds * n - 1) / (rounds * n);  // threads that divide a row into equal shares
  if (need <= kRowThreads / 2) {
    m.tpb = kRowThreads / need;
    m.width = need;
    *threads = kRowThreads;
    m.blocks = (tokens + m.tpb - 1) / m.tpb;
  } else {
    m.tpb = 1;
    m.width = *threads = (need + 31) / 32 * 32;
    if (rounds > 1 && few_tokens(tokens)) {
      m.piece = m.width * n;
      m.bpt = (m.vpt + m.piece - 1) / m.piece;
    }
    m.blocks = tokens * m.bpt;
  }
  m.d_width = make_fastdiv(m.width);
  return m;
}

// Floats of one access: as many of 4, 2, 1 as the row length and both addresses allow.
static int row_vec(uint64_t cols, const void* a, const void* b, const void* c = nullptr) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c);
  return cols % 4 == 0 && at % 16 == 0 ? 4 : cols % 2 == 0 && at % 8 == 0 ? 2 : 1;
}

// Accesses per thread and row: 8 floats of each of two rows, 4 of more.
static constexpr int row_n(int vec, int ku) { return (ku == 2 ? 8 : 4) / vec; }
// CALL(VEC, KU) for the access width and the number of choices taken at a time.
#define FB_ROW_KU(VEC, ku, CALL)         \
  if ((ku) == 2) { CALL(VEC, 2); }       \
  else if ((ku) == 4) { CALL(VEC, 4); }  \
  else { CALL(VEC, 8); }
#define FB_ROW_DISPATCH(vec, ku, CALL)             \
  do {                                             \
    if ((vec) == 4) { FB_ROW_KU(4, ku, CALL) }     \
    else if ((vec) == 2) { FB_ROW_KU(2, ku, CALL) }\
    else { FB_ROW_KU(1, ku, CALL) }                \
  } while (0)

// CALL(L, V): lanes per token and values per lane that hold the experts of a row.
#define FB_GATE_ROWS(experts, CALL)                                              \
  do {                                                                           \
    if ((experts) <= 32) { CALL(8, 4); }                           \
    else if ((experts) <= 64) { CALL(8, 8); }                      \
    else if ((experts) <= 128) { CALL(8, 16); }                    \
    else if ((experts) <= 256) { CALL(16, 16); }                                 \
    else if ((experts) <= 512) { CALL(32, 16); }                                 \
    else { CALL(32, 32); }                                                       \
  } while (0)
// CALL(NPL): experts per lane of a whole warp.
#define FB_GATE_WARP(experts, CALL)                \
  do {                                             \
    if ((experts) <= 32) { CALL(1); }              \
    else if ((experts) <= 64) { CALL(2); }         \
    else if ((experts) <= 128) { CALL(4); }        \
    else if ((experts) <= 256) { CALL(8); }        \
    else if ((experts) <= 512) { CALL(16); }       \
    else { CALL(32); }                             \
  } while (0)

// One CTA up to 4096 assignments (one launch; two take less time on the GPU but more on the host).  Beyond,
// chunks of 1024 (a thread each) up to kSortDirect of them, else of 4096; every CTA adds the counts up itself
// while there are few.  131072 assignments to 64 / 128 / 256 experts take 6.8 / 7.1 / 9.5 us in 128 chunks,
// 9.4 / 10.2 / 11.4 in 32; to 1024 experts 23.8 against 18.6.  With 128 chunks of 4096 and 1024 experts the
// scan of its own takes 20.1 us, adding up in every CTA 27.7.
struct SortPlan {
  uint32_t rounds, threads, chunks;
  int mode;
};
static SortPlan sort_plan(uint64_t n, uint64_t experts) {
  SortPlan p;
  const uint64_t most = n > experts ? n : experts;
  p.rounds = n <= kSortThreads || (n > kSortThreads * kSortRounds && n <= (uint64_t)kSortThreads * kSortDirect && experts <= 512) ? 1 : kSortRounds;
  p.threads = most < kSortThreads ? (uint32_t)(most + 31) / 32 * 32 : kSortThreads;
  const uint64_t chunk = (uint64_t)p.threads * p.rounds;
  p.chunks = n ? (uint32_t)((n + chunk - 1) / chunk) : 1;
  p.mode = p.chunks == 1 ? SORT_ALONE : p.chunks <= kSortDirect && p.chunks * experts <= kSortCounts ? SORT_DIRECT : SORT_SCANNED;
  return p;
}

}  // namespace fb

using namespace fb;

extern "C" {

int fb_moe_gate_fwd(fb_stream_t stream, const float* logits, uint64_t tokens, uint64_t experts, uint64_t k, int renorm,
                    float* weights, int64_t* ids) {
  const char* name = "fb_moe_gate_fwd";
  if (int rc = gate_check(name, tokens, experts, k)) return rc;
  if (tokens == 0) return FB_OK;
  if (!logits || !weights || !ids) return fail(FB_ERR_INVALID_ARG, "%s: null buffer", name);
  const uint64_t n = tokens * experts, m = tokens * k;
  if (overlaps(weights, m, logits, n) || overlaps(ids, 2 * m, logits, n) || overlaps(ids, 2 * m, weights, m))
    return fail(FB_ERR_INVALID_ARG, "%s: an output overlaps another buffer", name);
  const bool vec = experts % 4 == 0 && aligned16(logits);
  const uint32_t E = (uint32_t)experts, K = (uint32_t)k;
#define FB_CALL(KL, L, V)                                                                                        \
  FB_CUDA(launch_pdl(moe_gate_fwd_kernel<KL, L, V>, dim3(grid_full((tokens + kGateThreads / L - 1) / (kGateThreads / L))), dim3(kGateThreads), 0, stream, \
      logits, tokens, E, K, renorm != 0, vec, weights, ids))
#define FB_CALL2(L, V) FB_CALL(2, L, V)
#define FB_CALL8(L, V) FB_CALL(8, L, V)
#define FB_MANY(NPL)                                                                                             \
  FB_CUDA(launch_pdl(moe_gate_fwd_many_kernel<NPL>, dim3(grid_full((tokens + kGateWarps - 1) / kGateWarps)), dim3(kGateThreads), 0, stream, \
      logits, tokens, E, K, renorm != 0, weights, ids))
  if (k <= 2) FB_GATE_ROWS(experts, FB_CALL2);
  else if (k <= 8) FB_GATE_ROWS(experts, FB_CALL8);
  else FB_GATE_WARP(experts, FB_MANY);
#undef FB_CALL
#undef FB_CALL2
#undef FB_CALL8
#undef FB_MANY
  FB_LAUNCHED(name);
  return FB_OK;
}

int fb_moe_gate_bwd(fb_stream_t stream, const float* dweights, const float* logits, const float* weights,
                    const int64_t* ids, uint64_t tokens, uint64_t experts, uint64_t k, int renorm, float* dlogits) {
  const char* name = "fb_moe_gate_bwd";
  if (int rc = gate_check(name, tokens, experts, k)) return rc;
  if (tokens == 0) return FB_OK;
  if (!dweights || !weights || !ids || !dlogits || (!renorm && !logits)) return fail(FB_ERR_INVALID_ARG, "%s: null buffer", name);
  const uint64_t n = tokens * experts, m = tokens * k;
  if ((!renorm && overlaps(dlogits, n, logits, n)) || overlaps(dlogits, n, weights, m) || overlaps(dlogits, n, dweights, m) ||
      overlaps(dlogits, n, ids, 2 * m))
    return fail(FB_ERR_INVALID_ARG, "%s: dlogits overlaps an input", name);
  const bool vec = experts % 4 == 0 && aligned16(dlogits) && (renorm || aligned16(logits));
#define FB_CALL(L, V, MINE)                                                                                      \
  FB_CUDA(launch_pdl(moe_gate_bwd_kernel<L, V, MINE>, dim3(grid_full((tokens + kGateThreads / L - 1) / (kGateThreads / L))), dim3(kGateThreads), 0, stream, \
      dweights, logits, weights, ids, tokens, (uint32_t)experts, (uint32_t)k, renorm != 0, vec, dlogits))
#define FB_CALL1(L, V) FB_CALL(L, V, 1)
#define FB_CALL_ALL(L, V) FB_CALL(L, V, (FB_MOE_MAX_K / L))
  if (k <= 8) FB_GATE_ROWS(experts, FB_CALL1);
  else FB_GATE_ROWS(experts, FB_CALL_ALL);
#undef FB_CALL
#undef FB_CALL1
#undef FB_CALL_ALL
  FB_LAUNCHED(name);
  return FB_OK;
}

uint64_t fb_moe_sort_workspace_bytes(uint64_t n, uint64_t experts) {
  if (n > 0x7fffffffull || experts == 0 || experts > FB_MOE_MAX_EXPERTS) return 0;
  const SortPlan p = sort_plan(n, experts);
  return p.chunks > 1 ? ((uint64_t)p.chunks + 1) * experts * sizeof(uint32_t) : 0;
}

int fb_moe_sort(fb_stream_t stream, const int64_t* ids, uint64_t n, uint64_t experts, int64_t* place, int64_t* order,
                int64_t* offsets, int64_t* bad_index, void* workspace, uint64_t workspace_bytes) {
  const char* name = "fb_moe_sort";
  if (experts == 0 || experts > FB_MOE_MAX_EXPERTS)
    return fail(FB_ERR_INVALID_SHAPE, "%s: %llu experts, not 1 to %d", name, (unsigned long long)experts, FB_MOE_MAX_EXPERTS);
  if (n > 0x7fffffffull) return fail(FB_ERR_UNSUPPORTED, "%s: 2^31 or more assignments are not supported", name);
  if (!offsets || (n && (!ids || !place))) return fail(FB_ERR_INVALID_ARG, "%s: null buffer", name);
  if (overlaps(place, n, ids, n, 8) || overlaps(order, n, ids, n, 8) || overlaps(offsets, experts + 1, ids, n, 8) ||
      overlaps(place, n, order, n, 8) || overlaps(place, n, offsets, experts + 1, 8) || overlaps(order, n, offsets, experts + 1, 8))
    return fail(FB_ERR_INVALID_ARG, "%s: an output overlaps another buffer", name);
  const uint64_t need = fb_moe_sort_workspace_bytes(n, experts);
  if (need && (!workspace || workspace_bytes < need))
    return fail(FB_ERR_WORKSPACE, "%s: needs %llu bytes of scratch", name, (unsigned long long)need);
  const uint32_t E = (uint32_t)experts, n32 = (uint32_t)n;
  const SortPlan p = sort_plan(n, experts);
  const size_t smem = (2 * (size_t)E + (size_t)(p.threads / 32) * (E | 1)) * sizeof(uint32_t);
  const bool one = p.rounds == 1;
  if (smem > 48 * 1024) FB_CUDA(allow_dyn_smem(one ? (const void*)moe_place_kernel<1> : (const void*)moe_place_kernel<kSortRounds>, smem));
  uint32_t* counts = static_cast<uint32_t*>(workspace);
  uint32_t* totals = counts + (uint64_t)p.chunks * E;
  if (p.mode == SORT_ALONE) {
    if (one) FB_CUDA(launch_pdl(moe_place_kernel<1>, dim3(1), dim3(p.threads), smem, stream, ids, n32, E, 1, p.mode, nullptr, nullptr, place, order, offsets, bad_index));
    else FB_CUDA(launch_pdl(moe_place_kernel<kSortRounds>, dim3(1), dim3(p.threads), smem, stream, ids, n32, E, 1, p.mode, nullptr, nullptr, place, order, offsets, bad_index));
    FB_LAUNCHED(name);
    return FB_OK;
  }
  if (one) FB_CUDA(launch_pdl(moe_count_kernel<1>, dim3(p.chunks), dim3(kSortThreads), E * sizeof(uint32_t), stream, ids, n32, E, counts));
  else FB_CUDA(launch_pdl(moe_count_kernel<kSortRounds>, dim3(p.chunks), dim3(kSortThreads), E * sizeof(uint32_t), stream, ids, n32, E, counts));
  FB_LAUNCHED(name);
  if (p.mode == SORT_SCANNED) {
    FB_CUDA(launch_pdl(moe_scan_kernel, dim3((E + 31) / 32), dim3(1024), 0, stream, counts, p.chunks, E, totals));
    FB_LAUNCHED(name);
  }
  FB_CUDA(launch_pdl(one ? moe_place_kernel<1> : moe_place_kernel<kSortRounds>, dim3(p.chunks), dim3(p.threads), smem, stream, ids,
                     n32, E, p.chunks, p.mode, (const uint32_t*)counts, (const uint32_t*)totals, place, order, offsets, bad_index));
  FB_LAUNCHED(name);
  return FB_OK;
}

int fb_moe_dispatch_fwd(fb_stream_t stream, const float* x, const int64_t* place, uint64_t tokens, uint64_t k,
                        uint64_t cols, float* xs, uint64_t slots) {
  const char* name = "fb_moe_dispatch_fwd";
  if (int rc = rows_check(name, tokens, k, cols, slots)) return rc;
  if (tokens == 0 || cols == 0 || slots == 0) return FB_OK;
  if (!x || !place || !xs) return fail(FB_ERR_INVALID_ARG, "%s: null buffer", name);
  if (overlaps(xs, slots * cols, x, tokens * cols) || overlaps(xs, slots * cols, place, 2 * tokens * k))
    return fail(FB_ERR_INVALID_ARG, "%s: xs must not overlap an input", name);
  const int vec = row_vec(cols, x, xs), ku = k <= 2 ? 2 : k <= 4 ? 4 : 8;
  uint32_t threads;
  const RowMap m = row_map(tokens, k, cols, slots, vec, row_n(vec, ku), &threads);
  const unsigned grid = grid_full(m.blocks);
#define FB_CALL(VEC, KU) FB_CUDA(launch_pdl(moe_scatter_kernel<VEC, row_n(VEC, KU), KU>, dim3(grid), dim3(threads), 0, stream, x, place, m, xs))
  FB_ROW_DISPATCH(vec, ku, FB_CALL);
#undef FB_CALL
  FB_LAUNCHED(name);
  return FB_OK;
}

static int gather_rows(cudaStream_t stream, const char* name, const float* ys, const float* weights, const int64_t* place,
                       uint64_t tokens, uint64_t k, uint64_t cols, uint64_t slots, float* y) {
  if (int rc = rows_check(name, tokens, k, cols, slots)) return rc;
  if (tokens == 0 || cols == 0) return FB_OK;
  if ((slots && !ys) || !place || !y) return fail(FB_ERR_INVALID_ARG, "%s: null buffer", name);
  if (overlaps(y, tokens * cols, ys, slots * cols) || overlaps(y, tokens * cols, weights, tokens * k) ||
      overlaps(y, tokens * cols, place, 2 * tokens * k))
    return fail(FB_ERR_INVALID_ARG, "%s: the output must not overlap an input", name);
  const int vec = row_vec(cols, ys, y), ku = k <= 2 ? 2 : k <= 4 || !few_tokens(tokens) ? 4 : 8;
  uint32_t threads;
  const RowMap m = row_map(tokens, k, cols, slots, vec, row_n(vec, ku), &threads);
  const unsigned grid = grid_full(m.blocks);
#define FB_CALL(VEC, KU)                                                                                                   \
  if (weights) FB_CUDA(launch_pdl(moe_gather_kernel<VEC, row_n(VEC, KU), KU, true>, dim3(grid), dim3(threads), 0, stream, ys, weights, place, m, y)); \
  else FB_CUDA(launch_pdl(moe_gather_kernel<VEC, row_n(VEC, KU), KU, false>, dim3(grid), dim3(threads), 0, stream, ys, weights, place, m, y))
  FB_ROW_DISPATCH(vec, ku, FB_CALL);
#undef FB_CALL
  FB_LAUNCHED(name);
  return FB_OK;
}

int fb_moe_dispatch_bwd(fb_stream_t stream, const float* dxs, const int64_t* place, uint64_t tokens, uint64_t k,
                        uint64_t cols, uint64_t slots, float* dx) {
  return gather_rows(stream, "fb_moe_dispatch_bwd", dxs, nullptr, place, tokens, k, cols, slots, dx);
}

int fb_moe_combine_fwd(fb_stream_t stream, const float* ys, const float* weights, const int64_t* place,
                       uint64_t tokens, uint64_t k, uint64_t cols, uint64_t slots, float* y) {
  if (tokens && cols && !weights) return fail(FB_ERR_INVALID_ARG, "fb_moe_combine_fwd: null buffer");
  return gather_rows(stream, "fb_moe_combine_fwd", ys, weights, place, tokens, k, cols, slots, y);
}

int fb_moe_combine_bwd(fb_stream_t stream, const float* dy, const float* ys, const float* weights, const int64_t* place,
                       uint64_t tokens, uint64_t k, uint64_t cols, uint64_t slots, float* dys, float* dweights) {
  const char* name = "fb_moe_combine_bwd";
  if (int rc = rows_check(name, tokens, k, cols, slots)) return rc;
  if (tokens == 0 || (!dys && !dweights)) return FB_OK;
  if (cols == 0) return dweights ? fb_fill(stream, dweights, 0.0f, tokens * k) : FB_OK;
  if (!dy || !weights || !place || (dweights && slots && !ys)) return fail(FB_ERR_INVALID_ARG, "%s: null buffer", name);
  const uint64_t n = slots * cols, m = tokens * k;
  if ((dys != ys && overlaps(dys, n, ys, n)) || overlaps(dys, n, dy, tokens * cols) || overlaps(dys, n, weights, m) ||
      overlaps(dys, n, place, 2 * m) || overlaps(dweights, m, weights, m) || overlaps(dweights, m, dy, tokens * cols) ||
      overlaps(dweights, m, ys, n) || overlaps(dweights, m, dys, n) || overlaps(dweights, m, place, 2 * m))
    return fail(FB_ERR_INVALID_ARG, "%s: an output must not overlap another buffer, but dys may be ys", name);
  const int vec = row_vec(cols, dy, dweights ? ys : dy, dys);
  const int ku = k <= 2 ? 2 : k <= 4 ? 4 : 8;
  // Up to 64 threads' worth of a row: by a warp or as many of its lanes as have something to do.  Wider: by
  // a CTA that divides the row into equal shares.
  const uint32_t each = (uint32_t)row_n(vec, ku), vpt = (uint32_t)(cols / vec), most = kRowThreads * each;
  const uint32_t need = (vpt + each - 1) / each, rounds = (vpt + most - 1) / most;
  uint32_t lanes = 0, threads = kRowThreads;
  if (need <= 64) {
    for (lanes = 1; lanes < 32 && lanes < need; lanes <<= 1) {
    }
  } else {
    threads = ((vpt + rounds * each - 1) / (rounds * each) + 31) / 32 * 32;
  }
  const uint32_t per_cta = lanes ? threads / lanes : 1;
  const unsigned grid = grid_full((tokens + per_cta - 1) / per_cta);
  const uint32_t k32 = (uint32_t)k;
#define FB_CALL(VEC, KU) \
  FB_CUDA(launch_pdl(moe_combine_bwd_kernel<VEC, row_n(VEC, KU), KU>, dim3(grid), dim3(threads), 0, stream, dy, ys, weights, place, \
                     tokens, k32, cols, slots, lanes, dys, dweights))
  FB_ROW_DISPATCH(vec, ku, FB_CALL);
#undef FB_CALL
  FB_LAUNCHED(name);
  return FB_OK;
}

}  // extern "C"
