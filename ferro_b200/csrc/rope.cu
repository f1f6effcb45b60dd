// Rotary positions: pairs of channels of a [batch, seq, heads, head_dim] view
// turned by position * theta_i, forward and (with the angle negated) backward.
//
// Angle.  theta_i is given in turns as a 64-bit fixed-point fraction, so the
// fraction of a turn at position p is the low 64 bits of p * turns_i: integer
// arithmetic without range reduction.  The fraction's last place costs |p| * 2^-64
// turns, the cut to 32 bits 2^-32, which is the larger up to position 2^32.
//
// Roofline: HBM, 8 bytes per element.  A thread owns one group of pairs of one
// token and walks HPT heads with it, so cosine and sine are paid once per HPT
// heads; all of a thread's loads are issued before the first product.  Measured
// against the copy rate: 4 x 4096 tokens of 32 heads of 128 100 % in both layouts
// (82 us), 64 of 256 channels turned 104 %, 40 of 80 89 to 95 %, 126 channels (no
// 16-byte access fits) 88 to 96 %, one head of 128 62 % at 65536 tokens (16.5 us),
// 94 % at 524288 (88 us): a thread has one pair of accesses in flight and its
// angles to form before it can store, and neither limit is reached (schedulers
// issue in 75 % of the cycles, DRAM is busy for 68 %).
#include <cmath>

#include "common.cuh"
#include "fastdiv.cuh"

namespace fb {

constexpr int kRopeThreads = 128;  // 256: 2 to 20 % slower throughout

struct RopeArgs {
  const float* x;
  float* out;
  const int64_t* pos;    // NULL: start + s
  const int64_t* turns;
  int64_t start;
  int64_t xs[4], os[4];  // element strides of batch, seq, head, channel
  uint32_t tokens, seq, heads, half;  // half = rot_dim / 2 pairs
  uint32_t pair_units, units;  // groups of pairs per head; with the groups of copied channels
  uint32_t upt;                // threads per token: head chunks * units
  uint32_t tpb, bpt;           // tokens per CTA; CTAs per token
  uint32_t pos_batch;          // 1: positions have a row per batch entry
  uint32_t rot, dim;
  FastDiv d_upt, d_units, d_seq;
  uint64_t blocks;
  float scale;
  uint32_t flip;               // sign bit where the angle is negated
};

template <int V>
struct Vec;
template <> struct Vec<1> { using T = float; };
template <> struct Vec<2> { using T = float2; };
template <> struct Vec<4> { using T = float4; };

template <int VEC>
__device__ __forceinline__ void rope_load(const float* p, float (&v)[VEC]) {
  using T = typename Vec<VEC>::T;
  const T t = __ldcs(reinterpret_cast<const T*>(p));
  *reinterpret_cast<T*>(v) = t;
}
template <int VEC>
__device__ __forceinline__ void rope_store(float* p, const float (&v)[VEC]) {
  using T = typename Vec<VEC>::T;
  __stcs(reinterpret_cast<T*>(p), *reinterpret_cast<const T*>(v));
}

// Cosine and sine of a fraction of a turn (top 32 bits of the fixed-point word), from their Taylor series
// after the nearest quarter turn is taken off exactly: x, half turns in [-1/4, 1/4], is the integer
// remainder times a power of two.  The terms left out are below 2e-9 (sine, from x^11) and 2e-10 (cosine,
// from x^12); pi is kept in two floats, so that what counts is the rounding of x and of the result.
// About 25 instructions.  Where one head has to pay for them alone (8 x 8192 tokens of 128 channels, half
// layout) the kernel takes 16.5 us, with sincospif, which reduces a float argument first, 18.6.
__device__ __forceinline__ void turn_sincos(uint64_t turns, float scale, uint32_t flip, float& s, float& c) {
  const uint32_t t = (uint32_t)(turns >> 32), q = (t + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(t - (q << 30)) * 4.656612873077393e-10f;  // 2^-31
  const float y = x * x;
  float a = 0.08214588661112822f;  // pi^9 / 9!
  a = fmaf(a, y, -0.5992645293207921f);
  a = fmaf(a, y, 2.550164039877345f);
  a = fmaf(a, y, -5.16771278004997f);
  a = fmaf(x, 3.1415927410125732f, x * fmaf(a, y, -8.742278e-8f));
  float b = -0.02580689139001406f;  // -pi^10 / 10!
  b = fmaf(b, y, 0.23533063035889312f);
  b = fmaf(b, y, -1.3352627688545893f);
  b = fmaf(b, y, 4.058712126416768f);
  b = fmaf(b, y, -4.934802200544679f);
  b = fmaf(b, y, 1.0f);
  const bool odd = q & 1;
  // quarter turns: (c, s) -> (-s, c) each
  s = (odd ? b : a) * __uint_as_float(__float_as_uint(scale) ^ ((q & 2) << 30) ^ flip);
  c = (odd ? a : b) * __uint_as_float(__float_as_uint(scale) ^ (((q + 1) & 2) << 30));
}

// A group of pairs is, in the half layout, VEC neighbours of the first half and the VEC across from
// them; in the interleaved layout VEC / 2 pairs in one vector (VEC 1: the two channels of one pair,
// any channel stride).
template <int VEC, int LAYOUT, int HPT>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const __grid_constant__ RopeArgs A) {
  constexpr bool kTwo = LAYOUT == FB_ROPE_HALF || VEC == 1;  // two vectors per group
  constexpr int kPairs = LAYOUT == FB_ROPE_HALF ? VEC : (VEC + 1) / 2;
  pdl_wait();
  pdl_trigger();
  for (uint64_t blk = blockIdx.x; blk < A.blocks; blk += gridDim.x) {
    uint32_t token, rem;
    if (A.bpt == 1) {
      const uint32_t tl = fdiv(threadIdx.x, A.d_upt);
      rem = threadIdx.x - tl * A.upt;
      token = (uint32_t)blk * A.tpb + tl;
      if (tl >= A.tpb || token >= A.tokens) continue;
    } else {
      const uint64_t t = blk / A.bpt;
      token = (uint32_t)t;
      rem = (uint32_t)(blk - t * A.bpt) * kRopeThreads + threadIdx.x;
      if (rem >= A.upt) continue;
    }
    const uint32_t chunk = fdiv(rem, A.d_units), u = rem - chunk * A.units;
    const uint32_t b = fdiv(token, A.d_seq), s = token - b * A.seq;
    const uint32_t h0 = chunk * HPT, hn = min((uint32_t)HPT, A.heads - h0);
    const float* xp = A.x + (int64_t)b * A.xs[0] + (int64_t)s * A.xs[1] + (int64_t)h0 * A.xs[2];
    float* op = A.out + (int64_t)b * A.os[0] + (int64_t)s * A.os[1] + (int64_t)h0 * A.os[2];
    // Groups of copied channels go through the same loads and stores, so that a warp that holds both
    // kinds waits for memory once.
    const bool turn = u < A.pair_units;
    const uint32_t pair = u * kPairs;
    uint32_t ca, cb;  // channels of the first and, where there is one, the second vector
    bool second = kTwo;
    if (turn) {
      ca = LAYOUT == FB_ROPE_HALF ? pair : 2 * pair;
      cb = LAYOUT == FB_ROPE_HALF ? pair + A.half : 2 * pair + 1;
    } else {
      ca = A.rot + (u - A.pair_units) * (kTwo ? 2 * VEC : VEC);
      cb = ca + VEC;
      second = kTwo && cb < A.dim;
    }
    const float* xa = xp + (int64_t)ca * A.xs[3];
    const float* xb = xp + (int64_t)cb * A.xs[3];
    float va[HPT][VEC], vb[HPT][VEC];
#pragma unroll
    for (int h = 0; h < HPT; ++h)
      if (h < (int)hn) {
        rope_load<VEC>(xa + (int64_t)h * A.xs[2], va[h]);
        if (kTwo && second) rope_load<VEC>(xb + (int64_t)h * A.xs[2], vb[h]);
      }
    if (turn) {
      const uint64_t p = A.pos ? (uint64_t)__ldca(A.pos + (A.pos_batch ? token : s)) : (uint64_t)A.start + s;
      float sn[kPairs], cs[kPairs];
#pragma unroll
      for (int i = 0; i < kPairs; ++i) turn_sincos(p * (uint64_t)__ldca(A.turns + pair + i), A.scale, A.flip, sn[i], cs[i]);
#pragma unroll
      for (int h = 0; h < HPT; ++h)
        if (h < (int)hn) {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            float& a = kTwo ? va[h][i] : va[h][2 * i];
            float& c = kTwo ? vb[h][i] : va[h][2 * i + 1];
            const float t = a * cs[i] - c * sn[i];
            c = c * cs[i] + a * sn[i];
            a = t;
          }
        }
    }
    float* oa = op + (int64_t)ca * A.os[3];
    float* ob = op + (int64_t)cb * A.os[3];
#pragma unroll
    for (int h = 0; h < HPT; ++h)
      if (h < (int)hn) {
        rope_store<VEC>(oa + (int64_t)h * A.os[2], va[h]);
        if (kTwo && second) rope_store<VEC>(ob + (int64_t)h * A.os[2], vb[h]);
      }
  }
}

template <int VEC, int LAYOUT>
static int rope_launch(cudaStream_t stream, RopeArgs& A, bool in_place, uint32_t head_dim) {
  A.pair_units = LAYOUT == FB_ROPE_HALF ? A.half / VEC : (VEC == 1 ? A.half : A.half / (VEC / 2));
  constexpr uint32_t kUnit = LAYOUT == FB_ROPE_HALF || VEC == 1 ? 2 * VEC : VEC;  // channels of a group
  A.units = A.pair_units + (in_place ? 0 : (head_dim - A.rot + kUnit - 1) / kUnit);
  A.dim = head_dim;
  const uint64_t work = (uint64_t)A.tokens * A.units;
  // Heads per thread: four share the cost of cosine and sine and keep their loads in flight, as far as
  // there are heads, and threads enough to fill the SMs.
  const bool few = work * ((A.heads + 3) / 4) < (uint64_t)device_info().sm_count * 2048;
  const uint32_t most = VEC == 4 ? 4 : 8;  // eight where an access is narrower
  uint32_t hpt = 1;
  while (!few && hpt < most && hpt < A.heads) hpt <<= 1;
  A.upt = (A.heads + hpt - 1) / hpt * A.units;
  A.tpb = A.upt < kRopeThreads ? kRopeThreads / A.upt : 1;
  A.bpt = A.upt < kRopeThreads ? 1 : (A.upt + kRopeThreads - 1) / kRopeThreads;
  A.d_upt = make_fastdiv(A.upt);
  A.d_units = make_fastdiv(A.units);
  A.d_seq = make_fastdiv(A.seq);
  A.blocks = (uint64_t)((A.tokens + A.tpb - 1) / A.tpb) * A.bpt;
  const unsigned grid = grid_full(A.blocks);
  if (hpt == 1) FB_CUDA(launch_pdl(rope_kernel<VEC, LAYOUT, 1>, dim3(grid), dim3(kRopeThreads), 0, stream, A));
  else if (hpt == 2) FB_CUDA(launch_pdl(rope_kernel<VEC, LAYOUT, 2>, dim3(grid), dim3(kRopeThreads), 0, stream, A));
  else if (hpt == 4) FB_CUDA(launch_pdl(rope_kernel<VEC, LAYOUT, 4>, dim3(grid), dim3(kRopeThreads), 0, stream, A));
  else if constexpr (VEC < 4) FB_CUDA(launch_pdl(rope_kernel<VEC, LAYOUT, 8>, dim3(grid), dim3(kRopeThreads), 0, stream, A));
  FB_LAUNCHED("fb_rope");
  return FB_OK;
}

template <int LAYOUT>
static int rope_vec(cudaStream_t stream, RopeArgs& A, bool in_place, uint32_t head_dim, int vec) {
  if (vec == 4) return rope_launch<4, LAYOUT>(stream, A, in_place, head_dim);
  if (vec == 2) return rope_launch<2, LAYOUT>(stream, A, in_place, head_dim);
  return rope_launch<1, LAYOUT>(stream, A, in_place, head_dim);
}

// Whether two elements of the view may share an address: dims sorted by stride, each must step over
// everything the smaller ones span.
static bool may_self_overlap(const uint64_t* shape, const int64_t* strides, int rank) {
  int idx[FB_MAX_RANK], n = 0;
  for (int d = 0; d < rank; ++d)
    if (shape[d] > 1) idx[n++] = d;
  auto mag = [&](int d) { return strides[d] < 0 ? -(__int128)strides[d] : (__int128)strides[d]; };
  for (int i = 1; i < n; ++i)
    for (int j = i; j > 0 && mag(idx[j]) < mag(idx[j - 1]); --j) {
      const int t = idx[j];
      idx[j] = idx[j - 1];
      idx[j - 1] = t;
    }
  __int128 span = 0;  // largest offset reached by the dims so far
  for (int i = 0; i < n; ++i) {
    if (mag(idx[i]) <= span) return true;
    span += mag(idx[i]) * (__int128)(shape[idx[i]] - 1);
  }
  return false;
}

// Addresses [lo, hi) that a view touches (bounds already checked, not empty).
static void touched(const fb_view& v, uintptr_t* lo, uintptr_t* hi) {
  int64_t a = v.offset, b = v.offset;
  for (int d = 0; d < v.rank; ++d) {
    const int64_t span = (int64_t)(v.shape[d] - 1) * v.strides[d];
    if (span >= 0) b += span;
    else a += span;
  }
  *lo = reinterpret_cast<uintptr_t>(v.ptr + a);
  *hi = reinterpret_cast<uintptr_t>(v.ptr + b + 1);
}

}  // namespace fb

using namespace fb;

extern "C" {

int fb_rope_turns(uint64_t rot_dim, double base, int scaling, double factor, double original_len, double low,
                  double high, int64_t* turns_host) {
  const char* name = "fb_rope_turns";
  if (rot_dim < 2 || (rot_dim & 1) || rot_dim > (1u << 30))
    return fail(FB_ERR_INVALID_SHAPE, "%s: rot_dim %llu is not an even number from 2 on", name, (unsigned long long)rot_dim);
  if (scaling < FB_ROPE_PLAIN || scaling > FB_ROPE_BY_PARTS) return fail(FB_ERR_INVALID_ARG, "%s: unknown scaling %d", name, scaling);
  if (!(base > 0.0) || std::isinf(base)) return fail(FB_ERR_INVALID_ARG, "%s: base must be positive and finite", name);
  if (scaling != FB_ROPE_PLAIN && (!(factor > 0.0) || std::isinf(factor)))
    return fail(FB_ERR_INVALID_ARG, "%s: factor must be positive and finite", name);
  if (scaling == FB_ROPE_BASE && rot_dim == 2) return fail(FB_ERR_INVALID_ARG, "%s: one pair has no base to change", name);
  if (scaling == FB_ROPE_BY_PARTS && (!(original_len > 0.0) || std::isinf(original_len) || !(high > low) || std::isinf(high) || std::isinf(low)))
    return fail(FB_ERR_INVALID_ARG, "%s: original_len must be positive and low < high", name);
  if (!turns_host) return fail(FB_ERR_INVALID_ARG, "%s: null table", name);
  const long double two_pi = 6.283185307179586476925286766559005768L;
  long double b = base;
  if (scaling == FB_ROPE_BASE) b *= powl((long double)factor, (long double)rot_dim / (long double)(rot_dim - 2));
  for (uint64_t i = 0; i < rot_dim / 2; ++i) {
    long double theta = powl(b, -2.0L * (long double)i / (long double)rot_dim);
    if (scaling == FB_ROPE_LINEAR) theta /= (long double)factor;
    if (scaling == FB_ROPE_BY_PARTS) {
      long double keep = ((long double)original_len * theta / two_pi - low) / ((long double)high - low);
      keep = keep < 0.0L ? 0.0L : keep > 1.0L ? 1.0L : keep;
      theta = theta * keep + theta / (long double)factor * (1.0L - keep);
    }
    long double t = theta / two_pi;
    t -= floorl(t);  // whole turns change nothing
    const long double f = ldexpl(t, 64);  // below 2^64: t < 1
    uint64_t r = (uint64_t)f;
    if (f - (long double)r >= 0.5L) ++r;
    turns_host[i] = (int64_t)r;
  }
  return FB_OK;
}

int fb_rope(fb_stream_t stream, const fb_view* x, const int64_t* positions, uint64_t position_rows, int64_t start,
            const int64_t* turns, uint64_t rot_dim, int layout, float scale, int inverse, float* out,
            uint64_t out_len, const int64_t* out_strides, int64_t out_offset) {
  const char* name = "fb_rope";
  if (layout != FB_ROPE_INTERLEAVED && layout != FB_ROPE_HALF) return fail(FB_ERR_INVALID_ARG, "%s: unknown layout %d", name, layout);
  if (int rc = check_view(name, x)) return rc;
  if (x->rank != 4) return fail(FB_ERR_INVALID_SHAPE, "%s: the view has rank %d, not [batch, seq, heads, head_dim]", name, x->rank);
  const uint64_t B = x->shape[0], S = x->shape[1], H = x->shape[2], D = x->shape[3];
  if (rot_dim < 2 || (rot_dim & 1) || rot_dim > D)
    return fail(FB_ERR_INVALID_SHAPE, "%s: rot_dim %llu is not an even number from 2 to head_dim %llu", name,
                (unsigned long long)rot_dim, (unsigned long long)D);
  if (positions && position_rows != 1 && position_rows != B)
    return fail(FB_ERR_INVALID_SHAPE, "%s: %llu rows of positions for a batch of %llu", name,
                (unsigned long long)position_rows, (unsigned long long)B);
  if (B == 0 || S == 0 || H == 0) return FB_OK;
  fb_view o = *x;
  o.ptr = out;
  o.len = out_len;
  o.offset = out_offset;
  int64_t expect = 1;
  for (int d = 3; d >= 0; --d) {
    o.strides[d] = out_strides ? out_strides[d] : expect;
    expect *= (int64_t)x->shape[d];
  }
  if (int rc = check_view(name, &o)) return rc;
  if (!turns) return fail(FB_ERR_INVALID_ARG, "%s: null table of frequencies", name);
  if (B * S >= (1ull << 31) || H * D >= (1ull << 31))
    return fail(FB_ERR_UNSUPPORTED, "%s: batch * seq or heads * head_dim of 2^31 or more is not supported", name);
  if (may_self_overlap(o.shape, o.strides, 4)) return fail(FB_ERR_INVALID_ARG, "%s: elements of out share addresses", name);
  bool in_place = o.ptr + o.offset == x->ptr + x->offset;
  for (int d = 0; d < 4; ++d) in_place = in_place && (o.shape[d] == 1 || o.strides[d] == x->strides[d]);
  if (!in_place) {
    uintptr_t xl, xh, ol, oh;
    touched(*x, &xl, &xh);
    touched(o, &ol, &oh);
    if (xl < oh && ol < xh) return fail(FB_ERR_INVALID_ARG, "%s: out overlaps x without being the same view", name);
  }
  RopeArgs A = {};
  A.x = x->ptr + x->offset;
  A.out = out + out_offset;
  A.pos = positions;
  A.pos_batch = positions && position_rows == B;
  A.turns = turns;
  A.start = start;
  // A vector of `vec` channels needs unit channel strides, addresses that are multiples of its size
  // and group ends that fall on vector ends.
  int vec = 4;
  auto fits = [&](const float* p, const int64_t* st) {
    for (int d = 0; d < 3; ++d)
      if (o.shape[d] > 1 && st[d] % vec) return false;
    return st[3] == 1 && reinterpret_cast<uintptr_t>(p) % (4u * vec) == 0;
  };
  while (vec > 1 && !((layout == FB_ROPE_HALF ? rot_dim / 2 : rot_dim) % vec == 0 && D % vec == 0 && fits(A.x, x->strides) && fits(A.out, o.strides)))
    vec >>= 1;
  for (int d = 0; d < 4; ++d) {
    A.xs[d] = o.shape[d] == 1 ? 0 : x->strides[d];
    A.os[d] = o.shape[d] == 1 ? 0 : o.strides[d];
  }
  A.tokens = (uint32_t)(B * S);
  A.seq = (uint32_t)S;
  A.heads = (uint32_t)H;
  A.half = (uint32_t)(rot_dim / 2);
  A.rot = (uint32_t)rot_dim;
  A.scale = scale;
  A.flip = inverse ? 0x80000000u : 0u;
  return layout == FB_ROPE_HALF ? rope_vec<FB_ROPE_HALF>(stream, A, in_place, (uint32_t)D, vec)
                                : rope_vec<FB_ROPE_INTERLEAVED>(stream, A, in_place, (uint32_t)D, vec);
}

}  // extern "C"
