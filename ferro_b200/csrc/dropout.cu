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
  int none;        // p == 1: nothing is kept
  float factor;    // 1 / (1 - p)
  __device__ __forceinline__ uint64_t first() const { return offset + (counter ? (uint64_t)__ldg(counter) : 0ull); }
  __device__ __forceinline__ bool keep(uint32_t word) const { return word >= least && !none; }
};

enum { DROP_NO_BIAS = 0, DROP_BIAS_VEC = 1, DROP_BIAS_SCALAR = 2 };

// VEC: x, residual and out are 16-byte aligned.  DROP_BIAS_VEC: cols % 4 == 0 and the bias is aligned too.
template <bool VEC, int BIAS, bool RES>
__global__ void __launch_bounds__(kDropThreads)
dropout_kernel(const float* x, const float* __restrict__ bias, const float* residual, uint64_t n, uint32_t cols,
               FastDiv d_cols, DropMask M, float* out) {
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
          const float4 b = __ldg(reinterpret_cast<const float4*>(bias + c));
          v[k][0] += b.x; v[k][1] += b.y; v[k][2] += b.z; v[k][3] += b.w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v[k][j] += __ldg(bias + c);
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
// A thread walks down rows with the column sums of one group of four neighbours in registers.  The group
// is one of the generator's (elements 4 q .. 4 q + 3), so a row costs one generator call and one 16-byte
// access whatever the width: where cols is no multiple of 4 the groups of row r begin s = r cols mod 4
// columns to the left of the row's own fours, and a thread takes only rows r + 4 m, for which s, and with
// it the thread's columns, stay the same.  A warp holds `lx` groups of 32 / lx rows; a CTA `wx` warps side
// by side (one or two where s is not 0, so that its row step is a multiple of 4) and 8 / wx below each other.
// A tile of columns is one group narrower than its lanes where s may be 1, 2 or 3.
//
// CTAs of a slab of rows write their sums to part[slab]; dropout_bias_kernel adds the slabs up in order.
constexpr int kDropBwdUnroll = 4;  // rows in flight per thread

struct DropBwdPlan {
  uint32_t lx, wx;       // lanes per row of a warp; warps side by side
  uint32_t tile, tiles;  // columns of a CTA; CTAs across
  uint32_t slabs;
  uint64_t rows_per_slab;
};

static DropBwdPlan drop_bwd_plan(uint64_t rows, uint64_t cols) {
  DropBwdPlan p;
  const bool even = cols % 4 == 0;
  const uint64_t groups = even ? cols / 4 : (cols + 2) / 4 + 1;  // of one row, at most
  p.lx = 1;
  while (p.lx < 32 && p.lx < groups) p.lx <<= 1;
  const uint64_t warp_cols = 4ull * (even || groups <= 32 ? p.lx : p.lx - 1);
  p.wx = 1;
  while (p.wx < (even ? 8u : 2u) && p.wx * warp_cols < cols) p.wx <<= 1;
  p.tile = (uint32_t)(p.wx * warp_cols);
  p.tiles = (uint32_t)((cols + p.tile - 1) / p.tile);
  const uint64_t step = 8 / p.wx * (32 / p.lx), target = (uint64_t)device_info().sm_count * 6;
  uint64_t slabs = (target + p.tiles - 1) / p.tiles;
  const uint64_t most = rows / (step * kDropBwdUnroll) + 1;  // a slab fills a thread's loads once
  if (slabs > most) slabs = most;
  p.rows_per_slab = (rows + slabs - 1) / slabs;
  p.slabs = (uint32_t)((rows + p.rows_per_slab - 1) / p.rows_per_slab);
  return p;
}

template <bool VEC, bool DX>
__global__ void __launch_bounds__(kDropThreads, 4)
dropout_bwd_kernel(const float* g, uint64_t rows, uint64_t cols, const __grid_constant__ DropBwdPlan P, DropMask M,
                   float* dx, float* __restrict__ sums) {
  pdl_trigger();
  __shared__ float sm[kDropThreads / 32][128 + 4];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t li = lane & (P.lx - 1), sub = lane / P.lx, rpw = 32 / P.lx;
  const uint32_t wx = warp & (P.wx - 1), wy = warp / P.wx, step = 8 / P.wx * rpw;
  const uint32_t tile = blockIdx.x % P.tiles, slab = blockIdx.x / P.tiles;
  const uint32_t warp_cols = P.tile / P.wx;
  const uint64_t c0 = (uint64_t)tile * P.tile + wx * warp_cols;  // columns [c0, c1) are this warp's
  const uint64_t c1 = c0 + warp_cols < cols ? c0 + warp_cols : cols;
  const uint64_t n = rows * cols, first = M.first();
  const uint64_t r0 = (uint64_t)slab * P.rows_per_slab + wy * rpw + sub;
  const uint64_t r1 = (uint64_t)(slab + 1) * P.rows_per_slab < rows ? (uint64_t)(slab + 1) * P.rows_per_slab : rows;
  const uint32_t s = (uint32_t)(r0 * cols) & 3;
  const int64_t c = (int64_t)(c0 + 4 * li) - s;  // column of the group's first element; c0 is a multiple of 4
  uint32_t mine = 0;                             // which of the four are this warp's
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (c + j >= (int64_t)c0 && c + j < (int64_t)c1) mine |= 1u << j;
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (mine) {
    // element of the group's first member in row r0; n - 1 is the last there is
    uint64_t e = r0 * cols + (uint64_t)c;
    const uint64_t down = (uint64_t)step * cols;
    for (uint64_t r = r0; r < r1; r += (uint64_t)step * kDropBwdUnroll) {
      float v[kDropBwdUnroll][4];
#pragma unroll
      for (int u = 0; u < kDropBwdUnroll; ++u) {
        const uint64_t at = e + u * down;
        if (r + (uint64_t)u * step < r1) {
          if (VEC && at + 4 <= n) {
            const float4 t = ld_stream4(g + at);
            v[u][0] = t.x; v[u][1] = t.y; v[u][2] = t.z; v[u][3] = t.w;
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[u][j] = (mine >> j) & 1 ? ld_stream(g + at + j) : 0.0f;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kDropBwdUnroll; ++u) {
        const uint64_t at = e + u * down;
        if (r + (uint64_t)u * step < r1) {
          uint32_t w[4];
          philox4(first + (at >> 2), M.seed, w);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v[u][j] = M.keep(w[j]) ? v[u][j] * M.factor : 0.0f;
            acc[j] += v[u][j];
          }
          if (DX) {
            if (VEC && mine == 15u) {
              st_stream4(dx + at, make_float4(v[u][0], v[u][1], v[u][2], v[u][3]));
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if ((mine >> j) & 1) st_stream(dx + at + j, v[u][j]);
            }
          }
        }
      }
      e += kDropBwdUnroll * down;
    }
  }
  // Rows of a warp have columns of their own where s is not 0: sums meet in shared memory by column.
  // One pass per row of the warp, so that a place has one writer at a time and a fixed order.
  const uint32_t places = 4 * P.lx;  // at most this many columns
  for (uint32_t i = lane; i < places; i += 32) sm[warp][i] = 0.0f;
  for (uint32_t q = 0; q < rpw; ++q) {
    __syncwarp();
    if (sub == q) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((mine >> j) & 1) sm[warp][(uint32_t)(c + j - (int64_t)c0)] += acc[j];
    }
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < P.tile; i += kDropThreads) {
    const uint32_t w = i / warp_cols, k = i - w * warp_cols;
    const uint64_t col = (uint64_t)tile * P.tile + i;
    if (col < cols) {
      float t = 0.0f;
      for (uint32_t y = w; y < 8; y += P.wx) t += sm[y][k];
      sums[(uint64_t)slab * cols + col] = t;
    }
  }
}

// dbias[c] = sum over slabs of part[slab][c]: eight threads per column take every eighth slab, then a
// fixed order.
__global__ void __launch_bounds__(256)
dropout_bias_kernel(const float* __restrict__ part, uint32_t slabs, uint64_t cols, float* __restrict__ dbias) {
  pdl_wait();
  pdl_trigger();
  __shared__ float sm[8][32];
  const uint32_t lane = threadIdx.x & 31, y = threadIdx.x >> 5;
  const uint64_t c = (uint64_t)blockIdx.x * 32 + lane;
  float t = 0.0f;
  if (c < cols) {
    uint32_t s = y;
    for (; s + 24 < slabs; s += 32) {
      const float a = __ldcg(part + (uint64_t)s * cols + c), b = __ldcg(part + (uint64_t)(s + 8) * cols + c);
      const float d = __ldcg(part + (uint64_t)(s + 16) * cols + c), f = __ldcg(part + (uint64_t)(s + 24) * cols + c);
      t = (((t + a) + b) + d) + f;
    }
    for (; s < slabs; s += 8) t += __ldcg(part + (uint64_t)s * cols + c);
  }
  sm[y][lane] = t;
  __syncthreads();
  if (y == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < 8; ++i) t += sm[i][lane];
    dbias[c] = t;
  }
}

__global__ void dropout_advance_kernel(int64_t* counter, uint64_t n) {
  if (threadIdx.x == 0) counter[0] = (int64_t)((uint64_t)counter[0] + n);
}

static int make_mask(const char* name, float p, uint64_t seed, uint64_t offset, const int64_t* counter, DropMask* m) {
  if (!(p >= 0.0f && p <= 1.0f)) return fail(FB_ERR_INVALID_ARG, "%s: p must lie in [0, 1]", name);
  const double t = std::nearbyint((double)p * 4294967296.0);
  m->none = t >= 4294967296.0;
  m->least = m->none ? 0xffffffffu : (uint32_t)t;
  m->factor = m->none ? 0.0f : (float)(1.0 / (1.0 - (double)p));
  m->seed = seed;
  m->offset = offset;
  m->counter = counter;
  return FB_OK;
}

template <bool VEC, int BIAS>
static void drop_launch(cudaStream_t s, unsigned grid, const float* x, const float* bias, const float* residual,
                        uint64_t n, uint64_t cols, const DropMask& m, float* out) {
  const uint32_t c32 = (uint32_t)cols;
  const FastDiv d = make_fastdiv(BIAS == DROP_NO_BIAS ? 1 : c32);
  if (residual) dropout_kernel<VEC, BIAS, true><<<grid, kDropThreads, 0, s>>>(x, bias, residual, n, c32, d, m, out);
  else dropout_kernel<VEC, BIAS, false><<<grid, kDropThreads, 0, s>>>(x, bias, residual, n, c32, d, m, out);
}

static int run_dropout(cudaStream_t s, const char* name, const float* x, const float* bias, const float* residual,
                       uint64_t n, uint64_t cols, const DropMask& m, float* out) {
  const bool vec = aligned16(x) && aligned16(out) && (!residual || aligned16(residual));
  const uint64_t per_cta = (uint64_t)kDropThreads * kDropUnroll;
  const unsigned grid = grid_full(((n + 3) / 4 + per_cta - 1) / per_cta);
  if (!bias) {
    if (vec) drop_launch<true, DROP_NO_BIAS>(s, grid, x, bias, residual, n, cols, m, out);
    else drop_launch<false, DROP_NO_BIAS>(s, grid, x, bias, residual, n, cols, m, out);
  } else if (vec && cols % 4 == 0 && aligned16(bias)) {
    drop_launch<true, DROP_BIAS_VEC>(s, grid, x, bias, residual, n, cols, m, out);
  } else if (vec) {
    drop_launch<true, DROP_BIAS_SCALAR>(s, grid, x, bias, residual, n, cols, m, out);
  } else {
    drop_launch<false, DROP_BIAS_SCALAR>(s, grid, x, bias, residual, n, cols, m, out);
  }
  FB_LAUNCHED(name);
  return FB_OK;
}

}  // namespace fb

using namespace fb;

extern "C" {

int fb_dropout_fwd(fb_stream_t stream, const float* x, const float* bias, const float* residual, uint64_t rows,
                   uint64_t cols, float p, uint64_t seed, uint64_t offset, const int64_t* counter, float* out) {
  const char* name = "fb_dropout_fwd";
  DropMask m;
  if (int rc = make_mask(name, p, seed, offset, counter, &m)) return rc;
  uint64_t n;
  if (mul_overflows(rows, cols, &n) || n > (UINT64_MAX >> 3)) return fail(FB_ERR_INVALID_SHAPE, "%s: rows * cols overflows", name);
  if (n == 0) return FB_OK;
  if (!x || !out) return fail(FB_ERR_INVALID_ARG, "%s: null buffer", name);
  if (bias && cols >= (1ull << 31)) return fail(FB_ERR_UNSUPPORTED, "%s: a bias of 2^31 or more elements is not supported", name);
  return run_dropout(stream, name, x, bias, residual, n, cols, m, out);
}

uint64_t fb_dropout_bwd_workspace_bytes(uint64_t rows, uint64_t cols) {
  uint64_t n;
  if (mul_overflows(rows, cols, &n) || n == 0 || cols >= (1ull << 31)) return 0;
  const DropBwdPlan p = drop_bwd_plan(rows, cols);
  return p.slabs > 1 ? (uint64_t)p.slabs * cols * sizeof(float) : 0;
}

int fb_dropout_bwd(fb_stream_t stream, const float* g, uint64_t rows, uint64_t cols, float p, uint64_t seed,
                   uint64_t offset, const int64_t* counter, float* dx, float* dbias, void* workspace,
                   uint64_t workspace_bytes) {
  const char* name = "fb_dropout_bwd";
  DropMask m;
  if (int rc = make_mask(name, p, seed, offset, counter, &m)) return rc;
  uint64_t n;
  if (mul_overflows(rows, cols, &n) || n > (UINT64_MAX >> 3)) return fail(FB_ERR_INVALID_SHAPE, "%s: rows * cols overflows", name);
  if (cols == 0) return FB_OK;
  if (rows == 0) return dbias ? fb_fill(stream, dbias, 0.0f, cols) : FB_OK;
  if (!g) return fail(FB_ERR_INVALID_ARG, "%s: null buffer", name);
  if (!dx && !dbias) return FB_OK;
  if (!dbias) return run_dropout(stream, name, g, nullptr, nullptr, n, cols, m, dx);
  if (cols >= (1ull << 31)) return fail(FB_ERR_UNSUPPORTED, "%s: a bias of 2^31 or more elements is not supported", name);
  const DropBwdPlan plan = drop_bwd_plan(rows, cols);
  const uint64_t need = fb_dropout_bwd_workspace_bytes(rows, cols);
  if (need && (!workspace || workspace_bytes < need))
    return fail(FB_ERR_WORKSPACE, "%s: needs %llu bytes of scratch", name, (unsigned long long)need);
  float* sums = plan.slabs > 1 ? static_cast<float*>(workspace) : dbias;
  const unsigned grid = plan.tiles * plan.slabs;
  const bool vec = aligned16(g) && (!dx || aligned16(dx));
  if (vec && dx) dropout_bwd_kernel<true, true><<<grid, kDropThreads, 0, stream>>>(g, rows, cols, plan, m, dx, sums);
  else if (vec) dropout_bwd_kernel<true, false><<<grid, kDropThreads, 0, stream>>>(g, rows, cols, plan, m, dx, sums);
  else if (dx) dropout_bwd_kernel<false, true><<<grid, kDropThreads, 0, stream>>>(g, rows, cols, plan, m, dx, sums);
  else dropout_bwd_kernel<false, false><<<grid, kDropThreads, 0, stream>>>(g, rows, cols, plan, m, dx, sums);
  FB_LAUNCHED(name);
  if (plan.slabs > 1) {
    FB_CUDA(launch_pdl(dropout_bias_kernel, dim3((unsigned)((cols + 31) / 32)), dim3(256), 0, stream, (const float*)sums,
                       plan.slabs, cols, dbias));
    FB_LAUNCHED(name);
  }
  return FB_OK;
}

int fb_dropout_advance(fb_stream_t stream, int64_t* counter, uint64_t n) {
  if (!counter) return fail(FB_ERR_INVALID_ARG, "fb_dropout_advance: null counter");
  dropout_advance_kernel<<<1, 32, 0, stream>>>(counter, n);
  FB_LAUNCHED("fb_dropout_advance");
  return FB_OK;
}

}  // extern "C"
