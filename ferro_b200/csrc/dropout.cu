// Dropout with bias and residual, forward and backward, whose mask is a pure
// function of (seed, counter, element number): the backward draws it again
// instead of reading a stored one.
//
// Element e is kept when word e % 4 of Philox4x32-10 at counter
// offset + counter[0] + e / 4 is at least round(p * 2^32).  One generator call
// serves four neighbouring elements, which is one float4.
//
// Roofline: HBM.  Algorithmic bytes: 8 per element forward (12 with a
// residual), 8 backward; the generator adds about 10 instructions per element
// (20 wide products and 20 three-way xors per four elements).
#include <cmath>

#include "common.cuh"
#include "fastdiv.cuh"
#include "philox.cuh"

namespace fb {

constexpr int kDropThreads = 256;
constexpr int kDropUnroll = 4;  // groups of four elements per thread

struct DropMask {
  uint64_t seed, offset;
  const int64_t* counter;
  uint32_t least;  // smallest word that keeps its element
  float factor;    // 1 / (1 - p)
  __device__ __forceinline__ uint64_t first() const { return offset + (counter ? (uint64_t)__ldca(counter) : 0ull); }
  __device__ __forceinline__ bool keep(uint32_t word) const { return word >= least; }
};

enum { DROP_NO_BIAS = 0, DROP_BIAS_VEC = 1, DROP_BIAS_SCALAR = 2 };

// VEC: x, residual and out are 16-byte aligned.  DROP_BIAS_VEC: cols % 4 == 0 and the bias is aligned too.
template <bool VEC, int BIAS, bool RES>
__global__ void __launch_bounds__(kDropThreads)
dropout_kernel(const float* x, const float* __restrict__ bias, const float* residual, uint64_t n, uint32_t cols,
               FastDiv d_cols, DropMask M, float* out) {
  pdl_wait();
  pdl_trigger();
  const uint64_t groups = (n + 3) / 4;
  const uint64_t first = M.first();
  for (uint64_t base = (uint64_t)blockIdx.x * kDropThreads * kDropUnroll; base < groups;
       base += (uint64_t)gridDim.x * kDropThreads * kDropUnroll) {
    float v[kDropUnroll][4], r[kDropUnroll][4];
#pragma unroll
    for (int k = 0; k < kDropUnroll; ++k) {
      const uint64_t q = base + (uint64_t)k * kDropThreads + threadIdx.x;
      const uint64_t e = q * 4;
      if (VEC && e + 4 <= n) {
        const float4 t = ld_stream4(x + e);
        v[k][0] = t.x; v[k][1] = t.y; v[k][2] = t.z; v[k][3] = t.w;
        if (RES) {
          const float4 w = ld_stream4(residual + e);
          r[k][0] = w.x; r[k][1] = w.y; r[k][2] = w.z; r[k][3] = w.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[k][j] = e + j < n ? x[e + j] : 0.0f;
          if (RES) r[k][j] = e + j < n ? residual[e + j] : 0.0f;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kDropUnroll; ++k) {
      const uint64_t q = base + (uint64_t)k * kDropThreads + threadIdx.x;
      const uint64_t e = q * 4;
      if (e >= n) continue;
      if (BIAS != DROP_NO_BIAS) {
        uint32_t c = (e >> 32) ? (uint32_t)(e % cols) : (uint32_t)e - fdiv((uint32_t)e, d_cols) * cols;
        if (BIAS == DROP_BIAS_VEC) {
          const float4 b = __ldca(reinterpret_cast<const float4*>(bias + c));
          v[k][0] += b.x; v[k][1] += b.y; v[k][2] += b.z; v[k][3] += b.w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v[k][j] += __ldca(bias + c);
            if (++c == cols) c = 0;
          }
        }
      }
      uint32_t w[4];
      philox4(first + q, M.seed, w);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool keep = M.keep(w[j]);
        if (RES) v[k][j] = keep ? fmaf(v[k][j], M.factor, r[k][j]) : r[k][j];
        else v[k][j] = keep ? v[k][j] * M.factor : 0.0f;
      }
      if (VEC && e + 4 <= n) {
        st_stream4(out + e, make_float4(v[k][0], v[k][1], v[k][2], v[k][3]));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (e + j < n) out[e + j] = v[k][j];
      }
    }
  }
}

// ---- backward with the bias gradient
// The tensor is walked flat, in periods of P elements, P a multiple of cols and of 4: a thread that takes
// the same group of four in every period meets the same columns each time and keeps their sums in
// registers, whatever the width, with one generator call and one 16-byte access per four elements.  A CTA
// takes 1024 neighbouring places of the period (a tile) in a slab of periods; P is the multiple of
// lcm(cols, 4) that fills its last tile best.
//
// What a CTA leaves behind is, for cols >= 1024, its tile of a row of P sums, which is P / cols rows of
// cols; for fewer columns it first adds up the places of a column and leaves one row.  dropout_bias_kernel
// adds the rows in order.
//
// Bound by HBM as far as a grid of resident CTAs allows that reads and writes in equal measure: 16384 x
// 4096 in 95 us, 87 % of the copy rate.  Seven groups are in flight per thread while seven go through the
// generator, on two CTAs per SM; four on three, four or five CTAs took 103 to 125 us, without the early
// loads 109 us at best, a column sum that draws the mask at each load 107 us, staging through shared
// memory by bulk copies (2 to 8 stages of 8 KB, 3 to 8 CTAs per SM) 94 to 113 us.
constexpr int kDropBwdUnroll = 7;      // groups in flight per thread: 8 spill
constexpr int kDropBwdPerSm = 2;       // CTAs, by registers
constexpr uint32_t kDropTile = kDropThreads * 4;

struct DropBwdPlan {
  uint64_t period, periods;   // elements; how many begin in the tensor
  uint64_t per_slab;          // periods
  uint32_t tiles, slabs;
  uint64_t sum_rows;          // rows of cols partial sums
};

static DropBwdPlan drop_bwd_plan(uint64_t rows, uint64_t cols) {
  DropBwdPlan p;
  const uint64_t n = rows * cols, unit = cols % 4 == 0 ? cols : cols % 2 == 0 ? 2 * cols : 4 * cols;
  const uint64_t target = (uint64_t)device_info().sm_count * kDropBwdPerSm;  // one wave
  p.period = unit;
  double best = 0.0;
  for (uint64_t m = 1; best < 0.98 && (m <= 16 || unit * m <= kDropTile); ++m) {
    const uint64_t P = unit * m, tiles = (P + kDropTile - 1) / kDropTile;
    if (m > 1 && (tiles > target || P > n / kDropBwdUnroll)) break;
    const double full = (double)P / ((double)tiles * kDropTile);
    if (full > best + 0.02) {
      best = full;
      p.period = P;
    }
  }
  p.periods = (n + p.period - 1) / p.period;
  p.tiles = (uint32_t)((p.period + kDropTile - 1) / kDropTile);
  uint64_t slabs = target / p.tiles ? target / p.tiles : 1;
  const uint64_t most = (p.periods + 3) / 4;  // a few groups per thread at least
  if (slabs > most) slabs = most;
  p.per_slab = (p.periods + slabs - 1) / slabs;
  p.slabs = (uint32_t)((p.periods + p.per_slab - 1) / p.per_slab);
  p.sum_rows = cols < kDropTile ? (uint64_t)p.tiles * p.slabs : p.period / cols * p.slabs;
  return p;
}

// One group of four: masked, scaled, added to the column sums.
__device__ __forceinline__ float4 drop_group(const DropMask& M, uint64_t counter, float4 v, float (&acc)[4]) {
  uint32_t w[4];
  philox4(counter, M.seed, w);
  v.x = M.keep(w[0]) ? v.x * M.factor : 0.0f;
  v.y = M.keep(w[1]) ? v.y * M.factor : 0.0f;
  v.z = M.keep(w[2]) ? v.z * M.factor : 0.0f;
  v.w = M.keep(w[3]) ? v.w * M.factor : 0.0f;
  acc[0] += v.x;
  acc[1] += v.y;
  acc[2] += v.z;
  acc[3] += v.w;
  return v;
}
// Four elements at p, `have` of which exist (4 outside the tensor's last group).
template <bool VEC>
__device__ __forceinline__ float4 drop_load(const float* p, uint32_t have = 4) {
  if (VEC && have == 4) return ld_stream4(p);
  return make_float4(ld_stream(p), have > 1 ? ld_stream(p + 1) : 0.0f, have > 2 ? ld_stream(p + 2) : 0.0f, have > 3 ? ld_stream(p + 3) : 0.0f);
}
template <bool VEC>
__device__ __forceinline__ void drop_store(float* p, float4 v, uint32_t have = 4) {
  if (VEC && have == 4) {
    st_stream4(p, v);
  } else {
    st_stream(p, v.x);
    if (have > 1) st_stream(p + 1, v.y);
    if (have > 2) st_stream(p + 2, v.z);
    if (have > 3) st_stream(p + 3, v.w);
  }
}

template <bool VEC, bool DX>
__global__ void __launch_bounds__(kDropThreads, kDropBwdPerSm)
dropout_bwd_kernel(const float* g, uint64_t n, uint32_t cols, const __grid_constant__ DropBwdPlan P, DropMask M,
                   float* dx, float* __restrict__ sums) {
  pdl_wait();
  pdl_trigger();
  __shared__ __align__(16) float sm[kDropTile];
  __shared__ float part[kDropThreads];
  constexpr int U = kDropBwdUnroll;
  const uint32_t tile = blockIdx.x % P.tiles, slab = blockIdx.x / P.tiles;
  const uint64_t place = (uint64_t)tile * kDropTile + 4 * threadIdx.x;  // in the period
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const uint64_t i0 = (uint64_t)slab * P.per_slab, i1 = i0 + P.per_slab < P.periods ? i0 + P.per_slab : P.periods;
  const uint64_t at = i0 * P.period + place;
  if (place < P.period && at < n) {
    uint64_t left = i1 - i0;  // groups of this thread; in the last period there may be none, or a short one
    const uint64_t last = at + (left - 1) * P.period;
    uint32_t have = 0;
    if (last + 4 > n) {
      --left;
      have = last < n ? (uint32_t)(n - last) : 0;
    }
    const float* gp = g + at;
    float* dp = DX ? dx + at : nullptr;
    uint64_t ctr = M.first() + (at >> 2);
    const uint64_t down = P.period, ctr_down = P.period >> 2;
    // Columns are summed in blocks of U: the error grows with U + groups / U roundings instead of their number.
    float sub[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    auto put = [&](float4 v) {
      v = drop_group(M, ctr, v, sub);
      ctr += ctr_down;
      if (DX) {
        drop_store<VEC>(dp, v);
        dp += down;
      }
    };
    auto fold = [&] {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc[j] += sub[j];
        sub[j] = 0.0f;
      }
    };
    // The next groups' loads are issued before the present ones go through the generator.
    float4 v[U];
    if (left >= U) {
#pragma unroll
      for (int u = 0; u < U; ++u, gp += down) v[u] = drop_load<VEC>(gp);
      for (left -= U; left >= U; left -= U) {
        float4 next[U];
#pragma unroll
        for (int u = 0; u < U; ++u, gp += down) next[u] = drop_load<VEC>(gp);
#pragma unroll
        for (int u = 0; u < U; ++u) put(v[u]);
        fold();
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = next[u];
      }
      float4 rest[U - 1];
#pragma unroll
      for (int u = 0; u < U - 1; ++u)
        if (u < (int)left) rest[u] = drop_load<VEC>(gp + u * down);
#pragma unroll
      for (int u = 0; u < U; ++u) put(v[u]);
      fold();
#pragma unroll
      for (int u = 0; u < U - 1; ++u)
        if (u < (int)left) put(rest[u]);
    } else {
#pragma unroll
      for (int u = 0; u < U - 1; ++u)
        if (u < (int)left) v[u] = drop_load<VEC>(gp + u * down);
#pragma unroll
      for (int u = 0; u < U - 1; ++u)
        if (u < (int)left) put(v[u]);
    }
    fold();
    if (have) {  // the tensor's last group, whole or short
      const float4 w = drop_group(M, M.first() + (last >> 2), drop_load<VEC>(g + last, have), acc);
      if (DX) drop_store<VEC>(dx + last, w, have);
    }
  }
  if (cols >= kDropTile) {  // places of a tile are different columns
    if (place < P.period) {
      float* to = sums + (uint64_t)slab * P.period + place;
#pragma unroll
      for (int j = 0; j < 4; ++j) to[j] = acc[j];
    }
    return;
  }
  *reinterpret_cast<float4*>(sm + 4 * threadIdx.x) = make_float4(acc[0], acc[1], acc[2], acc[3]);
  __syncthreads();
  // Column c's places in the tile are first, first + cols, ...; `share` threads take them in turn.
  const uint32_t begin = (uint32_t)(((uint64_t)tile * kDropTile) % cols);
  const uint32_t share = cols < kDropThreads ? kDropThreads / cols : 1;
  float* row = sums + (uint64_t)blockIdx.x * cols;
  for (uint32_t k = threadIdx.x; k < cols * share; k += kDropThreads) {
    const uint32_t c = k % cols, q = k / cols, first = c >= begin ? c - begin : c + cols - begin;
    float t = 0.0f;
    for (uint32_t i = first + q * cols; i < kDropTile; i += share * cols) t += sm[i];  // places behind the period hold 0
    if (share == 1) row[c] = t;
    else part[k] = t;
  }
  if (share > 1) {
    __syncthreads();
    if (threadIdx.x < cols) {
      float t = 0.0f;
      for (uint32_t q = 0; q < share; ++q) t += part[q * cols + threadIdx.x];
      row[threadIdx.x] = t;
    }
  }
}

// dbias[c] = sum over rows of part[row][c]: 32 threads per column take every 32nd row, then a fixed order.
// A chain of loads whatever it does; eight threads per column took 8.3 us for 293 rows of 64, this 4 to 5.
__global__ void __launch_bounds__(1024)
dropout_bias_kernel(const float* __restrict__ part, uint32_t rows, uint64_t cols, float* __restrict__ dbias) {
  pdl_wait();
  pdl_trigger();
  __shared__ float sm[32][33];
  const uint32_t lane = threadIdx.x & 31, y = threadIdx.x >> 5;
  const uint64_t c = (uint64_t)blockIdx.x * 32 + lane;
  float t = 0.0f;
  if (c < cols) {
    uint32_t s = y;
    for (; s + 96 < rows; s += 128) {
      const float a = __ldcg(part + (uint64_t)s * cols + c), b = __ldcg(part + (uint64_t)(s + 32) * cols + c);
      const float d = __ldcg(part + (uint64_t)(s + 64) * cols + c), f = __ldcg(part + (uint64_t)(s + 96) * cols + c);
      t = (((t + a) + b) + d) + f;
    }
    for (; s < rows; s += 32) t += __ldcg(part + (uint64_t)s * cols + c);
  }
  sm[y][lane] = t;
  __syncthreads();
  // warp y adds up column y of the CTA's 32
  const float sum = warp_sum(sm[lane][y]);
  const uint64_t mine = (uint64_t)blockIdx.x * 32 + y;
  if (lane == 0 && mine < cols) dbias[mine] = sum;
}

__global__ void dropout_advance_kernel(int64_t* counter, uint64_t n) {
  pdl_wait();
  pdl_trigger();
  if (threadIdx.x == 0) counter[0] = (int64_t)((uint64_t)counter[0] + n);
}

// *none: p is 1 (or rounds to it), nothing is kept; no kernel is needed for that.
static int make_mask(const char* name, float p, uint64_t seed, uint64_t offset, const int64_t* counter, DropMask* m, bool* none) {
  if (!(p >= 0.0f && p <= 1.0f)) return fail(FB_ERR_INVALID_ARG, "%s: p must lie in [0, 1]", name);
  const double t = std::nearbyint((double)p * 4294967296.0);
  *none = t >= 4294967296.0;
  m->least = *none ? 0u : (uint32_t)t;
  m->factor = *none ? 0.0f : (float)(1.0 / (1.0 - (double)p));
  m->seed = seed;
  m->offset = offset;
  m->counter = counter;
  return FB_OK;
}

template <bool VEC, int BIAS>
static int drop_launch(cudaStream_t s, unsigned grid, const float* x, const float* bias, const float* residual,
                        uint64_t n, uint64_t cols, const DropMask& m, float* out) {
  const uint32_t c32 = (uint32_t)cols;
  const FastDiv d = make_fastdiv(BIAS == DROP_NO_BIAS ? 1 : c32);
  if (residual) FB_CUDA(launch_pdl(dropout_kernel<VEC, BIAS, true>, dim3(grid), dim3(kDropThreads), 0, s, x, bias, residual, n, c32, d, m, out));
  else FB_CUDA(launch_pdl(dropout_kernel<VEC, BIAS, false>, dim3(grid), dim3(kDropThreads), 0, s, x, bias, residual, n, c32, d, m, out));
  FB_LAUNCHED("fb_dropout");
  return FB_OK;
}

static int run_dropout(cudaStream_t s, const float* x, const float* bias, const float* residual,
                       uint64_t n, uint64_t cols, const DropMask& m, float* out) {
  const bool vec = aligned16(x) && aligned16(out) && (!residual || aligned16(residual));
  const uint64_t per_cta = (uint64_t)kDropThreads * kDropUnroll;
  const unsigned grid = grid_full(((n + 3) / 4 + per_cta - 1) / per_cta);
  if (!bias)
    return vec ? drop_launch<true, DROP_NO_BIAS>(s, grid, x, bias, residual, n, cols, m, out)
               : drop_launch<false, DROP_NO_BIAS>(s, grid, x, bias, residual, n, cols, m, out);
  if (vec && cols % 4 == 0 && aligned16(bias)) return drop_launch<true, DROP_BIAS_VEC>(s, grid, x, bias, residual, n, cols, m, out);
  return vec ? drop_launch<true, DROP_BIAS_SCALAR>(s, grid, x, bias, residual, n, cols, m, out)
             : drop_launch<false, DROP_BIAS_SCALAR>(s, grid, x, bias, residual, n, cols, m, out);
}

}  // namespace fb

using namespace fb;

extern "C" {

int fb_dropout_fwd(fb_stream_t stream, const float* x, const float* bias, const float* residual, uint64_t rows,
                   uint64_t cols, float p, uint64_t seed, uint64_t offset, const int64_t* counter, float* out) {
  const char* name = "fb_dropout_fwd";
  DropMask m;
  bool none;
  if (int rc = make_mask(name, p, seed, offset, counter, &m, &none)) return rc;
  uint64_t n;
  if (mul_overflows(rows, cols, &n) || n > (UINT64_MAX >> 3)) return fail(FB_ERR_INVALID_SHAPE, "%s: rows * cols overflows", name);
  if (n == 0) return FB_OK;
  if (!x || !out) return fail(FB_ERR_INVALID_ARG, "%s: null buffer", name);
  if ((out != x && overlaps(out, n, x, n)) || (out != residual && overlaps(out, n, residual, n)) || overlaps(out, n, bias, cols))
    return fail(FB_ERR_INVALID_ARG, "%s: out overlaps an input without being x or residual", name);
  if (bias && cols >= (1ull << 31)) return fail(FB_ERR_UNSUPPORTED, "%s: a bias of 2^31 or more elements is not supported", name);
  if (none) return !residual ? fb_fill(stream, out, 0.0f, n) : out == residual ? FB_OK : fb_copy(stream, out, residual, n);
  return run_dropout(stream, x, bias, residual, n, cols, m, out);
}

uint64_t fb_dropout_bwd_workspace_bytes(uint64_t rows, uint64_t cols) {
  uint64_t n;
  if (mul_overflows(rows, cols, &n) || n == 0 || cols >= (1ull << 31)) return 0;
  const DropBwdPlan p = drop_bwd_plan(rows, cols);
  return p.sum_rows > 1 ? p.sum_rows * cols * sizeof(float) : 0;
}

int fb_dropout_bwd(fb_stream_t stream, const float* g, uint64_t rows, uint64_t cols, float p, uint64_t seed,
                   uint64_t offset, const int64_t* counter, float* dx, float* dbias, void* workspace,
                   uint64_t workspace_bytes) {
  const char* name = "fb_dropout_bwd";
  DropMask m;
  bool none;
  if (int rc = make_mask(name, p, seed, offset, counter, &m, &none)) return rc;
  uint64_t n;
  if (mul_overflows(rows, cols, &n) || n > (UINT64_MAX >> 3)) return fail(FB_ERR_INVALID_SHAPE, "%s: rows * cols overflows", name);
  if (cols == 0) return FB_OK;
  if (rows == 0) return dbias ? fb_fill(stream, dbias, 0.0f, cols) : FB_OK;
  if (!g) return fail(FB_ERR_INVALID_ARG, "%s: null buffer", name);
  if (!dx && !dbias) return FB_OK;
  if ((dx != g && overlaps(dx, n, g, n)) || overlaps(dbias, cols, g, n) || overlaps(dbias, cols, dx, n))
    return fail(FB_ERR_INVALID_ARG, "%s: dx overlaps g without being it, or dbias overlaps either", name);
  if (none) {
    if (dx)
      if (int rc = fb_fill(stream, dx, 0.0f, n)) return rc;
    return dbias ? fb_fill(stream, dbias, 0.0f, cols) : FB_OK;
  }
  if (!dbias) return run_dropout(stream, g, nullptr, nullptr, n, cols, m, dx);
  if (cols >= (1ull << 31)) return fail(FB_ERR_UNSUPPORTED, "%s: a bias of 2^31 or more elements is not supported", name);
  const DropBwdPlan plan = drop_bwd_plan(rows, cols);
  const uint64_t need = fb_dropout_bwd_workspace_bytes(rows, cols);
  if (need && (!workspace || workspace_bytes < need))
    return fail(FB_ERR_WORKSPACE, "%s: needs %llu bytes of scratch", name, (unsigned long long)need);
  float* sums = need ? static_cast<float*>(workspace) : dbias;
  const unsigned grid = plan.tiles * plan.slabs;
  const bool vec = aligned16(g) && (!dx || aligned16(dx));
  if (vec && dx) FB_CUDA(launch_pdl(dropout_bwd_kernel<true, true>, dim3(grid), dim3(kDropThreads), 0, stream, g, n, (uint32_t)cols, plan, m, dx, sums));
  else if (vec) FB_CUDA(launch_pdl(dropout_bwd_kernel<true, false>, dim3(grid), dim3(kDropThreads), 0, stream, g, n, (uint32_t)cols, plan, m, dx, sums));
  else if (dx) FB_CUDA(launch_pdl(dropout_bwd_kernel<false, true>, dim3(grid), dim3(kDropThreads), 0, stream, g, n, (uint32_t)cols, plan, m, dx, sums));
  else FB_CUDA(launch_pdl(dropout_bwd_kernel<false, false>, dim3(grid), dim3(kDropThreads), 0, stream, g, n, (uint32_t)cols, plan, m, dx, sums));
  FB_LAUNCHED(name);
  if (need) {
    FB_CUDA(launch_pdl(dropout_bias_kernel, dim3((unsigned)((cols + 31) / 32)), dim3(1024), 0, stream, (const float*)sums,
                       (uint32_t)plan.sum_rows, cols, dbias));
    FB_LAUNCHED(name);
  }
  return FB_OK;
}

int fb_dropout_advance(fb_stream_t stream, int64_t* counter, uint64_t n) {
  if (!counter) return fail(FB_ERR_INVALID_ARG, "fb_dropout_advance: null counter");
  FB_CUDA(launch_pdl(dropout_advance_kernel, dim3(1), dim3(32), 0, stream, counter, n));
  FB_LAUNCHED("fb_dropout_advance");
  return FB_OK;
}

}  // extern "C"
