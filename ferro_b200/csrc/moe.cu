// The memory-bound half of a layer of routed experts: the router's choice, the
// stable sort of its assignments by expert, and the movement of token rows to
// their experts' rows and back, forward and backward.
//
// Every row that is written has one writer, every sum a fixed order (choices of a
// token ascending), integers are counted with commutative adds only: results do
// not depend on scheduling.
#include "common.cuh"

namespace fb {

// ---------------------------------------------------------------- gate
// One warp per token; lane l holds experts l, l + 32, ...  A logit is turned into
// an unsigned key whose order is the order of choice: -inf (masked) 0, then the
// finite values ascending (-0 and +0 equal), +inf, NaN highest.
__device__ __forceinline__ uint32_t gate_key(float v) {
  if (v != v) return 0xffffffffu;
  if (v == -INFINITY) return 0u;
  const uint32_t u = __float_as_uint(v + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float gate_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

constexpr int kGateThreads = 256;

template <int NPL>
__global__ void __launch_bounds__(kGateThreads)
moe_gate_fwd_kernel(const float* __restrict__ logits, uint64_t tokens, uint32_t experts, uint32_t k, int renorm,
                    float* __restrict__ weights, int64_t* __restrict__ ids) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (uint64_t t = (uint64_t)blockIdx.x * (kGateThreads / 32) + warp; t < tokens; t += (uint64_t)gridDim.x * (kGateThreads / 32)) {
    uint32_t key[NPL];
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      const uint32_t e = i * 32 + lane;
      key[i] = e < experts ? gate_key(__ldg(logits + t * experts + e)) : 0u;
    }
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < NPL; ++i) best = max(best, key[i]);
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    const float m = gate_value(top);
    float total = 0.0f;
    if (!renorm && top) {
#pragma unroll
      for (int i = 0; i < NPL; ++i)
        if (key[i]) total += expf(gate_value(key[i]) - m);
      total = warp_sum(total);
    }
    uint32_t my_key = 0, my_id = 0;  // lane j keeps choice j
    for (uint32_t j = 0; j < k; ++j) {
      uint32_t lb = 0, li = 0;
#pragma unroll
      for (int i = 0; i < NPL; ++i)
        if (key[i] > lb) {
          lb = key[i];
          li = i * 32 + lane;
        }
      const uint32_t win = __reduce_max_sync(0xffffffffu, lb);
      if (win == 0) break;
      const uint32_t id = __reduce_min_sync(0xffffffffu, lb == win ? li : 0xffffffffu);
      if ((uint32_t)lane == j) {
        my_key = win;
        my_id = id;
      }
#pragma unroll
      for (int i = 0; i < NPL; ++i)
        if (i * 32 + lane == id) key[i] = 0;
    }
    const float mass = my_key ? expf(gate_value(my_key) - m) : 0.0f;
    const float sum = renorm ? warp_sum(mass) : total;
    if ((uint32_t)lane < k) {
      weights[t * k + lane] = my_key ? mass / sum : 0.0f;
      ids[t * k + lane] = my_key ? (int64_t)my_id : -1;
    }
  }
}

template <int NPL>
__global__ void __launch_bounds__(kGateThreads)
moe_gate_bwd_kernel(const float* __restrict__ dweights, const float* __restrict__ logits, const float* __restrict__ weights,
                    const int64_t* __restrict__ ids, uint64_t tokens, uint32_t experts, uint32_t k, int renorm,
                    float* __restrict__ dlogits) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (uint64_t t = (uint64_t)blockIdx.x * (kGateThreads / 32) + warp; t < tokens; t += (uint64_t)gridDim.x * (kGateThreads / 32)) {
    float w = 0.0f, dw = 0.0f;
    uint32_t id = 0xffffffffu;
    if ((uint32_t)lane < k) {
      const int64_t e = __ldg(ids + t * k + lane);
      if (e >= 0 && e < (int64_t)experts) {
        id = (uint32_t)e;
        w = __ldg(weights + t * k + lane);
        dw = __ldg(dweights + t * k + lane);
      }
    }
    const float dot = warp_sum(w * dw);
    float p[NPL], acc[NPL];
    if (!renorm) {
      uint32_t best = 0;
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        const uint32_t e = i * 32 + lane;
        const float v = e < experts ? __ldg(logits + t * experts + e) : -INFINITY;
        p[i] = v;
        best = max(best, gate_key(v));
      }
      const uint32_t top = __reduce_max_sync(0xffffffffu, best);
      const float m = gate_value(top);
      float total = 0.0f;
      uint32_t live = 0;
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        const bool on = p[i] != -INFINITY;
        live |= (uint32_t)on << i;
        p[i] = on ? expf(p[i] - m) : 0.0f;
        total += p[i];
      }
      total = warp_sum(total);
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        p[i] = (live >> i) & 1 ? p[i] / total : 0.0f;
        acc[i] = -p[i] * dot;
      }
    } else {
#pragma unroll
      for (int i = 0; i < NPL; ++i) acc[i] = 0.0f;
    }
    for (uint32_t j = 0; j < k; ++j) {
      const uint32_t e = __shfl_sync(0xffffffffu, id, j);
      const float wj = __shfl_sync(0xffffffffu, w, j), dwj = __shfl_sync(0xffffffffu, dw, j);
      if (e == 0xffffffffu) continue;
#pragma unroll
      for (int i = 0; i < NPL; ++i)
        if (i * 32 + lane == e) acc[i] = renorm ? wj * (dwj - dot) : p[i] * (dwj - dot);
    }
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      const uint32_t e = i * 32 + lane;
      if (e < experts) dlogits[t * experts + e] = acc[i];
    }
  }
}

// ---------------------------------------------------------------- sort
// Counting sort.  A CTA owns kSortChunk neighbouring assignments, a warp 32 *
// kSortRounds of them.  Within a warp the rank of an assignment among those of
// its expert comes from the lanes that hold the same id (match) plus the warp's
// running count; between warps and CTAs counts are summed in order.
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortRounds = 4;
constexpr uint32_t kSortChunk = kSortThreads * kSortRounds;

__device__ __forceinline__ uint32_t sort_id(int64_t e, uint32_t experts) {
  return e >= 0 && e < (int64_t)experts ? (uint32_t)e : experts;  // `experts`: goes nowhere
}

// counts[b][e] = how many assignments of chunk b go to expert e.
__global__ void __launch_bounds__(kSortThreads)
moe_count_kernel(const int64_t* __restrict__ ids, uint32_t n, uint32_t experts, uint32_t* __restrict__ counts) {
  extern __shared__ uint32_t hist[];
  for (uint32_t e = threadIdx.x; e < experts; e += kSortThreads) hist[e] = 0;
  __syncthreads();
  const uint32_t base = blockIdx.x * kSortChunk;
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const uint32_t i = base + r * kSortThreads + threadIdx.x;
    if (i < n) {
      const uint32_t e = sort_id(__ldg(ids + i), experts);
      if (e < experts) atomicAdd(&hist[e], 1u);
    }
  }
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < experts; e += kSortThreads) counts[(uint64_t)blockIdx.x * experts + e] = hist[e];
}

// In place: counts[b][e] becomes the number of e's assignments in the chunks before b, totals[e] their
// number in all.  A CTA owns 32 experts (lanes) and splits the chunks into 32 runs (warps).
__global__ void __launch_bounds__(1024)
moe_scan_kernel(uint32_t* __restrict__ counts, uint32_t chunks, uint32_t experts, uint32_t* __restrict__ totals) {
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
// (kSortDirect at most); moe_scan_kernel has left prefixes and totals.
enum { SORT_ALONE = 0, SORT_DIRECT = 1, SORT_SCANNED = 2 };
constexpr uint32_t kSortDirect = 64;

__global__ void __launch_bounds__(kSortThreads)
moe_place_kernel(const int64_t* __restrict__ ids, uint32_t n, uint32_t experts, uint32_t chunks, int mode,
                 const uint32_t* __restrict__ counts, const uint32_t* __restrict__ totals, int64_t* __restrict__ place, int64_t* __restrict__ order,
                 int64_t* __restrict__ offsets, int64_t* __restrict__ bad) {
  extern __shared__ uint32_t sm[];
  uint32_t* total = sm;                // [experts + 1] over all chunks, then first rows
  uint32_t* before = total + experts + 1;  // [experts] in the chunks before this one
  uint32_t* hist = before + experts;   // [warps][experts]
  __shared__ uint32_t wsum[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (uint32_t i = threadIdx.x; i < kSortWarps * experts; i += kSortThreads) hist[i] = 0;
  for (uint32_t e = threadIdx.x; e < experts; e += kSortThreads) total[e] = before[e] = 0;
  __syncthreads();
  // ranks within the warp
  const uint32_t base = blockIdx.x * kSortChunk + warp * 32 * kSortRounds + lane;
  uint32_t id[kSortRounds], rank[kSortRounds];
  uint32_t* mine = hist + warp * experts;
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const uint32_t i = base + r * 32;
    id[r] = experts;
    if (i < n) {
      const int64_t e = __ldg(ids + i);
      id[r] = sort_id(e, experts);
      if (id[r] == experts && e != -1 && bad) atomicMax(reinterpret_cast<long long*>(bad), (long long)i + 1);
    }
  }
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const uint32_t same = __match_any_sync(0xffffffffu, id[r]);
    const uint32_t old = id[r] < experts ? mine[id[r]] : 0u;
    rank[r] = old + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (id[r] < experts && lane == __ffs(same) - 1) mine[id[r]] = old + __popc(same);
    __syncwarp();
  }
  __syncthreads();
  // exclusive prefix over the warps of this CTA; its total
  for (uint32_t e = threadIdx.x; e < experts; e += kSortThreads) {
    uint32_t acc = 0;
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t c = hist[w * experts + e];
      hist[w * experts + e] = acc;
      acc += c;
    }
    if (mode == SORT_ALONE) total[e] = acc;
    if (mode == SORT_SCANNED) {
      total[e] = totals[e];
      before[e] = counts[(uint64_t)blockIdx.x * experts + e];
    }
  }
  if (mode == SORT_DIRECT) {
    for (uint64_t i = threadIdx.x; i < (uint64_t)chunks * experts; i += kSortThreads) {
      const uint32_t b = (uint32_t)(i / experts), e = (uint32_t)(i - (uint64_t)b * experts);
      const uint32_t c = __ldg(counts + i);
      if (c) {
        atomicAdd(&total[e], c);
        if (b < blockIdx.x) atomicAdd(&before[e], c);
      }
    }
  }
  __syncthreads();
  // exclusive scan over the experts (at most one per thread)
  uint32_t v = threadIdx.x < experts ? total[threadIdx.x] : 0u, inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) wsum[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    uint32_t s = wsum[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += up;
    }
    wsum[lane] = s;
  }
  __syncthreads();
  const uint32_t excl = inc - v + (warp ? wsum[warp - 1] : 0u);
  if (threadIdx.x < experts) {
    total[threadIdx.x] = excl + before[threadIdx.x];
    if (blockIdx.x == 0) offsets[threadIdx.x] = excl;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) offsets[experts] = wsum[kSortWarps - 1];
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
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
// A token is owned by TPT threads (a power of two from 32 to 256); a thread walks the columns in
// vectors of VEC floats.
constexpr int kRowThreads = 256;

template <int VEC>
struct RowVec;
template <>
struct RowVec<4> {
  using T = float4;
  static __device__ __forceinline__ T load(const float* p) { return ld_stream4(p); }
  static __device__ __forceinline__ void store(float* p, T v) { st_stream4(p, v); }
  static __device__ __forceinline__ T zero() { return make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
  static __device__ __forceinline__ T mul(T a, float s) { return make_float4(a.x * s, a.y * s, a.z * s, a.w * s); }
  static __device__ __forceinline__ T add(T a, T b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
  static __device__ __forceinline__ T fma(T a, float s, T c) {
    return make_float4(fmaf(a.x, s, c.x), fmaf(a.y, s, c.y), fmaf(a.z, s, c.z), fmaf(a.w, s, c.w));
  }
  static __device__ __forceinline__ float dot(T a, T b, float c) {
    return fmaf(a.w, b.w, fmaf(a.z, b.z, fmaf(a.y, b.y, fmaf(a.x, b.x, c))));
  }
};
template <>
struct RowVec<1> {
  using T = float;
  static __device__ __forceinline__ T load(const float* p) { return ld_stream(p); }
  static __device__ __forceinline__ void store(float* p, T v) { st_stream(p, v); }
  static __device__ __forceinline__ T zero() { return 0.0f; }
  static __device__ __forceinline__ T mul(T a, float s) { return a * s; }
  static __device__ __forceinline__ T add(T a, T b) { return a + b; }
  static __device__ __forceinline__ T fma(T a, float s, T c) { return fmaf(a, s, c); }
  static __device__ __forceinline__ float dot(T a, T b, float c) { return fmaf(a, b, c); }
};

__device__ __forceinline__ int64_t slot_of(const int64_t* place, uint64_t a, uint64_t slots) {
  const int64_t s = __ldg(place + a);
  return s >= 0 && (uint64_t)s < slots ? s : -1;
}

// xs[place[t, j]] = x[t]
template <int VEC>
__global__ void __launch_bounds__(kRowThreads)
moe_scatter_kernel(const float* __restrict__ x, const int64_t* __restrict__ place, uint64_t tokens, uint32_t k,
                   uint64_t cols, uint64_t slots, uint32_t tpt, float* __restrict__ xs) {
  using R = RowVec<VEC>;
  const uint32_t per_cta = kRowThreads / tpt, mine = threadIdx.x / tpt, l = threadIdx.x % tpt;
  for (uint64_t t = (uint64_t)blockIdx.x * per_cta + mine; t < tokens; t += (uint64_t)gridDim.x * per_cta)
    for (uint64_t c = (uint64_t)l * VEC; c < cols; c += (uint64_t)tpt * VEC) {
      const typename R::T v = R::load(x + t * cols + c);
      for (uint32_t j = 0; j < k; ++j) {
        const int64_t s = slot_of(place, t * k + j, slots);
        if (s >= 0) R::store(xs + (uint64_t)s * cols + c, v);
      }
    }
}

// y[t] = sum over j of (weights[t, j] *) ys[place[t, j]]
template <int VEC, bool WEIGHTED>
__global__ void __launch_bounds__(kRowThreads)
moe_gather_kernel(const float* __restrict__ ys, const float* __restrict__ weights, const int64_t* __restrict__ place,
                  uint64_t tokens, uint32_t k, uint64_t cols, uint64_t slots, uint32_t tpt, float* __restrict__ y) {
  using R = RowVec<VEC>;
  const uint32_t per_cta = kRowThreads / tpt, mine = threadIdx.x / tpt, l = threadIdx.x % tpt;
  for (uint64_t t = (uint64_t)blockIdx.x * per_cta + mine; t < tokens; t += (uint64_t)gridDim.x * per_cta)
    for (uint64_t c = (uint64_t)l * VEC; c < cols; c += (uint64_t)tpt * VEC) {
      typename R::T acc = R::zero();
      for (uint32_t j = 0; j < k; ++j) {
        const int64_t s = slot_of(place, t * k + j, slots);
        if (s < 0) continue;
        const typename R::T v = R::load(ys + (uint64_t)s * cols + c);
        acc = WEIGHTED ? R::fma(v, __ldg(weights + t * k + j), acc) : R::add(acc, v);
      }
      R::store(y + t * cols + c, acc);
    }
}

// dys[place[t, j]] = weights[t, j] * dy[t]; dweights[t, j] = dy[t] . ys[place[t, j]].  One CTA per token.
template <int VEC>
__global__ void __launch_bounds__(kRowThreads)
moe_combine_bwd_kernel(const float* __restrict__ dy, const float* ys, const float* __restrict__ weights,
                       const int64_t* __restrict__ place, uint64_t tokens, uint32_t k, uint64_t cols, uint64_t slots,
                       float* dys, float* __restrict__ dweights) {
  using R = RowVec<VEC>;
  __shared__ float red[32];
  for (uint64_t t = blockIdx.x; t < tokens; t += gridDim.x)
    for (uint32_t j = 0; j < k; ++j) {
      const int64_t s = slot_of(place, t * k + j, slots);
      float dot = 0.0f;
      if (s >= 0) {
        const float w = __ldg(weights + t * k + j);
        for (uint64_t c = (uint64_t)threadIdx.x * VEC; c < cols; c += (uint64_t)kRowThreads * VEC) {
          const typename R::T g = R::load(dy + t * cols + c);
          if (dweights) dot = R::dot(g, R::load(ys + (uint64_t)s * cols + c), dot);
          if (dys) R::store(dys + (uint64_t)s * cols + c, R::mul(g, w));
        }
      }
      if (dweights) {
        dot = block_sum(dot, red);
        if (threadIdx.x == 0) dweights[t * k + j] = dot;
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
  return FB_OK;
}

static uint32_t threads_per_token(uint64_t vecs) {
  uint32_t t = 32;
  while (t < kRowThreads && t < vecs) t <<= 1;
  return t;
}

// f(std::integral_constant<int, NPL>) for the number of experts a lane holds.
#define FB_GATE_DISPATCH(experts, CALL)            \
  do {                                             \
    if ((experts) <= 32) { CALL(1); }              \
    else if ((experts) <= 64) { CALL(2); }         \
    else if ((experts) <= 128) { CALL(4); }        \
    else if ((experts) <= 256) { CALL(8); }        \
    else if ((experts) <= 512) { CALL(16); }       \
    else { CALL(32); }                             \
  } while (0)

static uint32_t sort_chunks(uint64_t n) { return (uint32_t)((n + kSortChunk - 1) / kSortChunk); }

}  // namespace fb

using namespace fb;

extern "C" {

int fb_moe_gate_fwd(fb_stream_t stream, const float* logits, uint64_t tokens, uint64_t experts, uint64_t k, int renorm,
                    float* weights, int64_t* ids) {
  const char* name = "fb_moe_gate_fwd";
  if (int rc = gate_check(name, tokens, experts, k)) return rc;
  if (tokens == 0) return FB_OK;
  if (!logits || !weights || !ids) return fail(FB_ERR_INVALID_ARG, "%s: null buffer", name);
  const unsigned grid = grid_full((tokens + kGateThreads / 32 - 1) / (kGateThreads / 32));
#define FB_CALL(NPL) \
  moe_gate_fwd_kernel<NPL><<<grid, kGateThreads, 0, stream>>>(logits, tokens, (uint32_t)experts, (uint32_t)k, renorm != 0, weights, ids)
  FB_GATE_DISPATCH(experts, FB_CALL);
#undef FB_CALL
  FB_LAUNCHED(name);
  return FB_OK;
}

int fb_moe_gate_bwd(fb_stream_t stream, const float* dweights, const float* logits, const float* weights,
                    const int64_t* ids, uint64_t tokens, uint64_t experts, uint64_t k, int renorm, float* dlogits) {
  const char* name = "fb_moe_gate_bwd";
  if (int rc = gate_check(name, tokens, experts, k)) return rc;
  if (tokens == 0) return FB_OK;
  if (!dweights || !weights || !ids || !dlogits || (!renorm && !logits)) return fail(FB_ERR_INVALID_ARG, "%s: null buffer", name);
  const unsigned grid = grid_full((tokens + kGateThreads / 32 - 1) / (kGateThreads / 32));
#define FB_CALL(NPL)                                                                                               \
  moe_gate_bwd_kernel<NPL><<<grid, kGateThreads, 0, stream>>>(dweights, logits, weights, ids, tokens, (uint32_t)experts, \
                                                              (uint32_t)k, renorm != 0, dlogits)
  FB_GATE_DISPATCH(experts, FB_CALL);
#undef FB_CALL
  FB_LAUNCHED(name);
  return FB_OK;
}

uint64_t fb_moe_sort_workspace_bytes(uint64_t n, uint64_t experts) {
  if (n > 0x7fffffffull || experts == 0 || experts > FB_MOE_MAX_EXPERTS) return 0;
  const uint64_t chunks = sort_chunks(n);
  return chunks > 1 ? (chunks + 1) * experts * sizeof(uint32_t) : 0;
}

int fb_moe_sort(fb_stream_t stream, const int64_t* ids, uint64_t n, uint64_t experts, int64_t* place, int64_t* order,
                int64_t* offsets, int64_t* bad_index, void* workspace, uint64_t workspace_bytes) {
  const char* name = "fb_moe_sort";
  if (experts == 0 || experts > FB_MOE_MAX_EXPERTS)
    return fail(FB_ERR_INVALID_SHAPE, "%s: %llu experts, not 1 to %d", name, (unsigned long long)experts, FB_MOE_MAX_EXPERTS);
  if (n > 0x7fffffffull) return fail(FB_ERR_UNSUPPORTED, "%s: 2^31 or more assignments are not supported", name);
  if (!offsets || (n && (!ids || !place))) return fail(FB_ERR_INVALID_ARG, "%s: null buffer", name);
  const uint64_t need = fb_moe_sort_workspace_bytes(n, experts);
  if (need && (!workspace || workspace_bytes < need))
    return fail(FB_ERR_WORKSPACE, "%s: needs %llu bytes of scratch", name, (unsigned long long)need);
  const uint32_t chunks = n ? sort_chunks(n) : 1, E = (uint32_t)experts;
  const size_t smem = (2 * (size_t)E + 1 + (size_t)kSortWarps * E) * sizeof(uint32_t);
  if (smem > 48 * 1024) FB_CUDA(allow_dyn_smem((const void*)moe_place_kernel, smem));
  uint32_t* counts = static_cast<uint32_t*>(workspace);
  uint32_t* totals = counts + (uint64_t)chunks * E;
  const int mode = chunks == 1 ? SORT_ALONE : chunks <= kSortDirect ? SORT_DIRECT : SORT_SCANNED;
  if (chunks > 1) {
    moe_count_kernel<<<chunks, kSortThreads, E * sizeof(uint32_t), stream>>>(ids, (uint32_t)n, E, counts);
    FB_LAUNCHED(name);
  }
  if (mode == SORT_SCANNED) {
    moe_scan_kernel<<<(E + 31) / 32, 1024, 0, stream>>>(counts, chunks, E, totals);
    FB_LAUNCHED(name);
  }
  moe_place_kernel<<<chunks, kSortThreads, smem, stream>>>(ids, (uint32_t)n, E, chunks, mode, counts, totals, place, order, offsets, bad_index);
  FB_LAUNCHED(name);
  return FB_OK;
}

int fb_moe_dispatch_fwd(fb_stream_t stream, const float* x, const int64_t* place, uint64_t tokens, uint64_t k,
                        uint64_t cols, float* xs, uint64_t slots) {
  const char* name = "fb_moe_dispatch_fwd";
  if (int rc = rows_check(name, tokens, k, cols, slots)) return rc;
  if (tokens == 0 || cols == 0 || slots == 0) return FB_OK;
  if (!x || !place || !xs) return fail(FB_ERR_INVALID_ARG, "%s: null buffer", name);
  if (xs == x) return fail(FB_ERR_INVALID_ARG, "%s: xs must not be x", name);
  const bool vec = cols % 4 == 0 && aligned16(x) && aligned16(xs);
  const uint32_t tpt = threads_per_token(vec ? cols / 4 : cols);
  const unsigned grid = grid_full((tokens + kRowThreads / tpt - 1) / (kRowThreads / tpt));
  if (vec) moe_scatter_kernel<4><<<grid, kRowThreads, 0, stream>>>(x, place, tokens, (uint32_t)k, cols, slots, tpt, xs);
  else moe_scatter_kernel<1><<<grid, kRowThreads, 0, stream>>>(x, place, tokens, (uint32_t)k, cols, slots, tpt, xs);
  FB_LAUNCHED(name);
  return FB_OK;
}

static int gather_rows(cudaStream_t stream, const char* name, const float* ys, const float* weights, const int64_t* place,
                       uint64_t tokens, uint64_t k, uint64_t cols, uint64_t slots, float* y) {
  if (int rc = rows_check(name, tokens, k, cols, slots)) return rc;
  if (tokens == 0 || cols == 0) return FB_OK;
  if ((slots && !ys) || !place || !y) return fail(FB_ERR_INVALID_ARG, "%s: null buffer", name);
  if (ys == y) return fail(FB_ERR_INVALID_ARG, "%s: the output must not be the input", name);
  const bool vec = cols % 4 == 0 && aligned16(ys) && aligned16(y);
  const uint32_t tpt = threads_per_token(vec ? cols / 4 : cols), k32 = (uint32_t)k;
  const unsigned grid = grid_full((tokens + kRowThreads / tpt - 1) / (kRowThreads / tpt));
  if (weights) {
    if (vec) moe_gather_kernel<4, true><<<grid, kRowThreads, 0, stream>>>(ys, weights, place, tokens, k32, cols, slots, tpt, y);
    else moe_gather_kernel<1, true><<<grid, kRowThreads, 0, stream>>>(ys, weights, place, tokens, k32, cols, slots, tpt, y);
  } else {
    if (vec) moe_gather_kernel<4, false><<<grid, kRowThreads, 0, stream>>>(ys, weights, place, tokens, k32, cols, slots, tpt, y);
    else moe_gather_kernel<1, false><<<grid, kRowThreads, 0, stream>>>(ys, weights, place, tokens, k32, cols, slots, tpt, y);
  }
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
  if (dys == dy || dweights == weights) return fail(FB_ERR_INVALID_ARG, "%s: an output is one of the inputs it must not be", name);
  const bool vec = cols % 4 == 0 && aligned16(dy) && (!dweights || aligned16(ys)) && (!dys || aligned16(dys));
  const unsigned grid = grid_full(tokens);
  if (vec) moe_combine_bwd_kernel<4><<<grid, kRowThreads, 0, stream>>>(dy, ys, weights, place, tokens, (uint32_t)k, cols, slots, dys, dweights);
  else moe_combine_bwd_kernel<1><<<grid, kRowThreads, 0, stream>>>(dy, ys, weights, place, tokens, (uint32_t)k, cols, slots, dys, dweights);
  FB_LAUNCHED(name);
  return FB_OK;
}

}  // extern "C"
