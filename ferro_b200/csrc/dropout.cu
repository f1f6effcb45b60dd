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
#include "reduce.cuh"

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

// Column-sum source of the bias gradient: the masked gradient, stored to dx on the way.
struct DropBwdSrc {
  const float* g;
  float* dx;
  uint64_t cols;
  DropMask M;
  template <int VEC>
  __device__ __forceinline__ void load(uint64_t, uint64_t r, uint64_t c, float (&v)[1][VEC]) const {
    const uint64_t e = r * cols + c;
    uint32_t w[4];
    philox4(M.first() + (e >> 2), M.seed, w);
    if constexpr (VEC == 4) {  // cols % 4 == 0, so e % 4 == 0
      const float4 t = ld_stream4(g + e);
      v[0][0] = M.keep(w[0]) ? t.x * M.factor : 0.0f;
      v[0][1] = M.keep(w[1]) ? t.y * M.factor : 0.0f;
      v[0][2] = M.keep(w[2]) ? t.z * M.factor : 0.0f;
      v[0][3] = M.keep(w[3]) ? t.w * M.factor : 0.0f;
      if (dx) st_stream4(dx + e, make_float4(v[0][0], v[0][1], v[0][2], v[0][3]));
    } else {
      const uint32_t j = (uint32_t)e & 3;
      const uint32_t word = j == 0 ? w[0] : j == 1 ? w[1] : j == 2 ? w[2] : w[3];
      v[0][0] = M.keep(word) ? g[e] * M.factor : 0.0f;
      if (dx) dx[e] = v[0][0];
    }
  }
};

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
  if (mul_overflows(rows, cols, &n) || n == 0) return 0;
  const uint64_t a = col_scratch_bytes(col_plan(1, rows, cols, true), 1, cols, 1);
  const uint64_t b = col_scratch_bytes(col_plan(1, rows, cols, false), 1, cols, 1);
  return a > b ? a : b;
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
  const DropBwdSrc src{g, dx, cols, m};
  const bool al = aligned16(g) && (!dx || aligned16(dx));
  return run_col_sum<1>(stream, src, 1, rows, cols, al, dbias, nullptr, 1.0f, workspace, workspace_bytes, name);
}

int fb_dropout_advance(fb_stream_t stream, int64_t* counter, uint64_t n) {
  if (!counter) return fail(FB_ERR_INVALID_ARG, "fb_dropout_advance: null counter");
  dropout_advance_kernel<<<1, 32, 0, stream>>>(counter, n);
  FB_LAUNCHED("fb_dropout_advance");
  return FB_OK;
}

}  // extern "C"
