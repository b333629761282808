// AdamW (Adam with decoupled weight decay) over many tensors in one launch,
// with the two moments in float32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2       t = step + 1
//   p = p - lr wd p - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// A 16-bit parameter has a float32 master that is stepped and rounded into it.
//
// 8-bit states: every 256 values of a tensor share one float scale per moment,
// their largest magnitude / 448; m and r = sqrt(v) -- whose range is half that
// of v in powers of two -- are e4m3 codes, four to a word.
//  * Rounding is stochastic.  A step moves v by a thousandth of itself while
//    neighbouring codes are 6 to 12 % apart: rounded to the nearest, v would
//    never move.  floor(x + u) with uniform u keeps the expectation.  u are 16
//    bits of Philox4x32-10 with the counter (element / 4, step) and the seed as
//    key: a function of seed, step and place, the same on every run.
//  * What is divided by never rounds to zero: r > 0 keeps at least the smallest
//    code, which can only shorten a step.
//  * A moment that is not finite is left out of its block's scale and stored as
//    NaN: it spoils its own element, as a float32 state would, not 255 others.
//  * The step itself uses the moments before they are rounded.
//
// float32 states are bound by memory: p, g, m, v are read and p, m, v written, 28
// bytes an element; bfloat16 with masters and 8-bit states moves 16.  A workgroup
// of 256 has 4096 elements in registers, all their loads issued before the first
// is used; a whole chunk of them is accessed without bounds.  141 M parameters:
// float32 680 us (5.8 TB/s), bfloat16 with masters 726 us (5.5 TB/s), 8-bit
// states 397 us with float32 and 400 us with bfloat16 parameters (5.7 TB/s),
// where a large copy reaches 5.1 TB/s.  The 8-bit kernel issues some 390
// instructions for each four elements of a lane, which keeps the vector units
// busy throughout: they bound it, not the memory.  Compiled without contraction,
// so that a state is the same value a plain evaluation of the formula in float32
// gives.
//
// The reference has Adam only (python/singa/opt.py:608-683), one element-wise
// launch for each operation.
#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace sa {

namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 256;   // values under one scale: four for each lane
constexpr int64_t kLaunchChunks = (1 << 24) - 1;

struct Consts {
  float lr, decay, eps, b1, k1, b2, k2, c1, c2, root_c2, scale;
};

// 1 - b^t for b = 1 - k without the cancellation of a b near 1, good to some
// 2^-20: the logarithm from its series where k is small, 1 - exp from its series
// where the exponent is.  The library's log1p and expm1 cost four times as much
// (141 M bf16 parameters with 8-bit states, otherwise as then: 501
// us instead of 533).
__device__ __forceinline__ float one_minus_power(float k, float t) {
  float y;   // log b
  if (k < 0.125f) {
    float s = 1.f / 8.f;
#pragma unroll
    for (int i = 7; i >= 1; --i) s = fmaf(s, k, 1.f / (float)i);
    y = -s * k;
  } else {
    y = 0.6931471806f * __builtin_amdgcn_logf(1.f - k);   // log2
  }
  y *= t;
  if (y < -0.35f) return 1.f - __builtin_amdgcn_exp2f(1.442695041f * y);
  float s = 1.f;
#pragma unroll
  for (int i = 7; i >= 2; --i) s = fmaf(s * y, 1.f / (float)i, 1.f);
  return -s * y;
}

__device__ __forceinline__ Consts constants(const AdamwHyper &h) {
  Consts c;
  c.lr = h.lr[0];
  c.decay = c.lr * h.wd[0];
  c.eps = h.eps[0];
  c.b1 = h.b1[0];
  c.b2 = h.b2[0];
  c.k1 = 1.f - c.b1;
  c.k2 = 1.f - c.b2;
  const float t = h.step[0] + 1.f;
  c.c1 = 1.f / one_minus_power(c.k1, t);
  c.c2 = 1.f / one_minus_power(c.k2, t);
  c.root_c2 = sqrtf(c.c2);
  c.scale = h.scale;
  return c;
}

__device__ __forceinline__ void advance(const Consts &c, float g, float &p,
                                        float &m, float &v) {
  g = g * c.scale;
  m = c.b1 * m + c.k1 * g;
  v = c.b2 * v + c.k2 * (g * g);
  p = p - c.decay * p;
  p = p - c.lr * ((m * c.c1) / (sqrtf(v * c.c2) + c.eps));
}

// The square root rounded to nearest: the hardware's, good to one unit in the
// last place, or the neighbour whose product with it says so.  (A v below
// 2^-126 may count as 0: its root, 2^-63 at most, is nothing beside eps.)
__device__ __forceinline__ float root(float v) {
  const float s = __builtin_amdgcn_sqrtf(v);
  const float down = __uint_as_float(__float_as_uint(s) - 1u);
  const float up = __uint_as_float(__float_as_uint(s) + 1u);
  const float too_large = fmaf(-down, s, v), too_small = fmaf(-up, s, v);
  float r = too_large <= 0.f ? down : s;
  return too_small > 0.f ? up : r;
}

// The same with r = sqrt(v) in the place of v.  The step takes the root that
// the state needs anyway, and a reciprocal good to one unit in the last place.
__device__ __forceinline__ void advance8(const Consts &c, float g, float &p,
                                         float &m, float &r) {
  g = g * c.scale;
  m = c.b1 * m + c.k1 * g;
  r = root(c.b2 * (r * r) + c.k2 * (g * g));
  const float u =
      (m * c.c1) * __builtin_amdgcn_rcpf(fmaf(r, c.root_c2, c.eps));
  p = fmaf(-c.decay, p, p);
  p = fmaf(-c.lr, u, p);
}

// the tensor that workgroup `chunk` works on
__device__ __forceinline__ int tensor_of(const AdamwBatch &b, int chunk) {
  const int lane = threadIdx.x & 63;
  const bool behind =
      lane > 0 && lane < b.count && chunk >= b.chunk_start[lane < b.count ? lane : 0];
  return __popcll(__ballot(behind));
}

// How a chunk is accessed: a whole and aligned one in vectors, kStream past the
// caches; the others with their bounds.
enum Access { kBounded, kWhole, kStream };

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Four {
  using Raw = typename std::conditional<sizeof(T) == 4, u32x4, u32x2>::type;
  T v[4];
};

// four values of which the first `n` exist
template <Access A, typename T>
__device__ __forceinline__ void load4(float *f, const T *p, int n, bool wide) {
  if (A == kBounded && !(wide && n >= 4)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = j < n ? to_f<T>(p[j]) : 0.f;
    return;
  }
  using Raw = typename Four<T>::Raw;
  const Raw *at = reinterpret_cast<const Raw *>(p);
  const Four<T> k = __builtin_bit_cast(
      Four<T>, A == kStream ? __builtin_nontemporal_load(at) : *at);
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = to_f<T>(k.v[j]);
}

template <Access A, typename T>
__device__ __forceinline__ void store4(T *p, const float *f, int n, bool wide) {
  if (A == kBounded && !(wide && n >= 4)) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) p[j] = from_f<T>(f[j]);
    return;
  }
  Four<T> k;
#pragma unroll
  for (int j = 0; j < 4; ++j) k.v[j] = from_f<T>(f[j]);
  using Raw = typename Four<T>::Raw;
  Raw *at = reinterpret_cast<Raw *>(p);
  const Raw raw = __builtin_bit_cast(Raw, k);
  if (A == kStream)
    __builtin_nontemporal_store(raw, at);
  else
    *at = raw;
}

template <Access A>
__device__ __forceinline__ uint32_t load_word(const uint32_t *p) {
  return A == kStream ? __builtin_nontemporal_load(p) : *p;
}

template <Access A>
__device__ __forceinline__ void store_word(uint32_t *p, uint32_t v) {
  if (A == kStream)
    __builtin_nontemporal_store(v, p);
  else
    *p = v;
}

__device__ __forceinline__ bool aligned16(const void *a, const void *b,
                                          const void *c, const void *d,
                                          const void *e) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) |
           reinterpret_cast<uintptr_t>(c) | reinterpret_cast<uintptr_t>(d) |
           reinterpret_cast<uintptr_t>(e)) & 15) == 0;
}

template <Access A, typename T, bool MASTER, typename P>
__device__ __forceinline__ void chunk32(const Consts &c, T *p16, P *p,
                                        const T *g, float *m, float *v, int len,
                                        bool wide) {
  constexpr int kSteps = kAdamwChunk / (4 * kThreads);
  float pf[kSteps][4], gf[kSteps][4], mf[kSteps][4], vf[kSteps][4];
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int i = 4 * (k * kThreads + (int)threadIdx.x), n = len - i;
    load4<A, P>(pf[k], p + i, n, wide);
    load4<A, T>(gf[k], g + i, n, wide);
    load4<A, float>(mf[k], m + i, n, wide);
    load4<A, float>(vf[k], v + i, n, wide);
  }
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int i = 4 * (k * kThreads + (int)threadIdx.x), n = len - i;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      advance(c, gf[k][j], pf[k][j], mf[k][j], vf[k][j]);
    store4<A, P>(p + i, pf[k], n, wide);
    if (MASTER) store4<A, T>(p16 + i, pf[k], n, wide);
    store4<A, float>(m + i, mf[k], n, wide);
    store4<A, float>(v + i, vf[k], n, wide);
  }
}

// T: type of parameter and gradient; MASTER: the step is taken on a float copy
template <typename T, bool MASTER, bool STREAM>
__global__ void __launch_bounds__(kThreads)
    adamw_kernel(AdamwBatch b, AdamwHyper h) {
  using P = typename std::conditional<MASTER, float, T>::type;
  const int t = tensor_of(b, blockIdx.x);
  const int64_t base = (int64_t)((int)blockIdx.x - b.chunk_start[t]) * kAdamwChunk;
  const int64_t left = b.n[t] - base;
  const int len = left < kAdamwChunk ? (int)left : kAdamwChunk;
  T *p16 = static_cast<T *>(b.p[t]) + base;
  P *p = MASTER ? reinterpret_cast<P *>(b.master[t]) + base
                : reinterpret_cast<P *>(p16);
  const T *g = static_cast<const T *>(b.g[t]) + base;
  float *m = static_cast<float *>(b.m[t]) + base;
  float *v = static_cast<float *>(b.v[t]) + base;
  const bool wide = aligned16(p16, p, g, m, v);
  const Consts c = constants(h);
  // a whole chunk has no bounds to look at
  constexpr Access kFull = STREAM ? kStream : kWhole;
  if (wide && len == kAdamwChunk)
    chunk32<kFull, T, MASTER>(c, p16, p, g, m, v, len, wide);
  else
    chunk32<kBounded, T, MASTER>(c, p16, p, g, m, v, len, wide);
}

struct Words { uint32_t w[4]; };

__device__ __forceinline__ Words philox(uint32_t c0, uint32_t c1, uint32_t c2,
                                        uint32_t c3, uint64_t key) {
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0;
    const uint64_t b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// Magnitudes are compared as integers: the bits of non-negative floats are in
// their order, infinity and NaN above all numbers, and no instruction is spent
// on quieting NaN.
constexpr uint32_t kInfinity = 0x7f800000u;

__device__ __forceinline__ uint32_t magnitude(float x) {
  return __float_as_uint(x) & 0x7fffffffu;
}

// the larger of x and of what the lane pattern brings (0 where nothing)
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t max_dpp(uint32_t x) {
  const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(
      0, (int)x, CTRL, ROWS, 0xf, ROWS == 0xf);
  return x > other ? x : other;
}

// The largest of a wave's values, in a scalar register: within rows of 16 lanes
// (neighbours, pairs, half rows, rows), then into the following rows.
__device__ __forceinline__ uint32_t wave_top(uint32_t x) {
  x = max_dpp<0xb1, 0xf>(x);    // quad_perm 1 0 3 2
  x = max_dpp<0x4e, 0xf>(x);    // quad_perm 2 3 0 1
  x = max_dpp<0x141, 0xf>(x);   // row_half_mirror
  x = max_dpp<0x140, 0xf>(x);   // row_mirror
  x = max_dpp<0x142, 0xa>(x);   // row_bcast15 into rows 1 and 3
  x = max_dpp<0x143, 0xc>(x);   // row_bcast31 into rows 2 and 3
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) {
  return a > b ? a : b;
}

// The largest finite magnitude of the wave's 256 values; `finite`: whether all
// are (what is not is looked for only where there is some).
__device__ __forceinline__ float block_top(const float *x, bool &finite) {
  uint32_t top = wave_top(umax(umax(magnitude(x[0]), magnitude(x[1])),
                               umax(magnitude(x[2]), magnitude(x[3]))));
  finite = top < kInfinity;
  if (!finite) {
    top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t a = magnitude(x[j]);
      top = umax(top, a < kInfinity ? a : 0u);
    }
    top = wave_top(top);
  }
  // below this the reciprocal of the scale would overflow: zeros
  return __uint_as_float(top > 0x08800000u ? top : 0u);   // 2^-110
}

// x times inv, rounded to e4m3 by the 16 bits of noise: floor(s / unit + u) of
// the codes' spacing.  A normal code keeps three bits of the fraction: the
// noise is added behind them, a carry goes where it should, the rest is cut
// off.  Below 2^-6 the spacing is 2^-9 throughout.  ROOT: x is not negative,
// and what is positive does not become zero.  FINITE: so are all values.
template <bool ROOT, bool FINITE>
__device__ __forceinline__ float to_code(float x, float inv, uint32_t noise) {
  const float s = x * inv;
  const uint32_t size = magnitude(s);
  const uint32_t normal = (size + (noise << 4)) & 0xfff00000u;
  float small = floorf(fmaf((float)noise, 0x1p-16f,
                            __uint_as_float(size) * 512.f)) * 0x1p-9f;
  if (ROOT)
    small = size > 0 ? __uint_as_float(umax(__float_as_uint(small), 0x3b000000u))
                     : small;   // 2^-9
  uint32_t q = size < 0x3c800000u ? __float_as_uint(small) : normal;   // 2^-6
  q = q < 0x43e00000u ? q : 0x43e00000u;   // 448
  if (!FINITE) q = size < kInfinity ? q : 0x7fc00000u;
  const float f = __uint_as_float(q);
  return ROOT ? f : copysignf(f, s);
}

template <bool FINITE>
__device__ __forceinline__ void to_codes(float *m, float *r, float mi, float ri,
                                         const uint32_t *words) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m[j] = to_code<false, FINITE>(m[j], mi, words[j] & 0xffffu);
    r[j] = to_code<true, FINITE>(r[j], ri, words[j] >> 16);
  }
}

__device__ __forceinline__ uint32_t pack_codes(const float *q) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
}

__device__ __forceinline__ void unpack_codes(float *f, uint32_t w, float scale) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  f[0] = lo[0] * scale;
  f[1] = lo[1] * scale;
  f[2] = hi[0] * scale;
  f[3] = hi[1] * scale;
}

template <Access A, typename T, bool MASTER, typename P>
__device__ __forceinline__ void chunk8(const Consts &c, T *p16, P *p,
                                       const T *g, uint32_t *mw, uint32_t *rw,
                                       float *ms, float *rs, int64_t base,
                                       int len, bool wide, uint32_t step,
                                       uint64_t seed) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int kSteps = kAdamwChunk / (4 * kBlock);
  float pf[kSteps][4], gf[kSteps][4], msf[kSteps], rsf[kSteps];
  uint32_t mc[kSteps], rc[kSteps];
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int blk = 4 * k + wave, i = kBlock * blk + 4 * lane, n = len - i;
    mc[k] = rc[k] = 0;
    msf[k] = rsf[k] = 0.f;
    if (A != kBounded || kBlock * blk < len) {   // the last block's words are all there
      mc[k] = load_word<A>(mw + i / 4);
      rc[k] = load_word<A>(rw + i / 4);
      msf[k] = ms[blk];
      rsf[k] = rs[blk];
    }
    load4<A, P>(pf[k], p + i, n, wide);
    load4<A, T>(gf[k], g + i, n, wide);
  }
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int blk = 4 * k + wave, i = kBlock * blk + 4 * lane, n = len - i;
    if (A == kBounded && kBlock * blk >= len) break;   // the same for the whole wave
    float m[4], v[4];
    unpack_codes(m, mc[k], msf[k]);
    unpack_codes(v, rc[k], rsf[k]);
    // behind the end of the tensor gradients and states are zero and stay so
#pragma unroll
    for (int j = 0; j < 4; ++j)
      advance8(c, gf[k][j], pf[k][j], m[j], v[j]);
    store4<A, P>(p + i, pf[k], n, wide);
    if (MASTER) store4<A, T>(p16 + i, pf[k], n, wide);
    bool m_finite, r_finite;
    const float mt = block_top(m, m_finite), rt = block_top(v, r_finite);
    const float mi = mt > 0.f ? 448.f * (1.f / mt) : 0.f;
    const float ri = rt > 0.f ? 448.f * (1.f / rt) : 0.f;
    const int64_t group = (base + i) / 4;
    const Words u = philox((uint32_t)group, (uint32_t)((uint64_t)group >> 32),
                           step, 0u, seed);
    if (m_finite && r_finite)   // the same for the whole wave
      to_codes<true>(m, v, mi, ri, u.w);
    else
      to_codes<false>(m, v, mi, ri, u.w);
    store_word<A>(mw + i / 4, pack_codes(m));
    store_word<A>(rw + i / 4, pack_codes(v));
    if (lane == 0) {
      ms[blk] = mt * (1.f / 448.f);
      rs[blk] = rt * (1.f / 448.f);
    }
  }
}

// A wave takes a block of 256 values, four for each lane; the blocks of a
// chunk go to the workgroup's four waves in turn.
template <typename T, bool MASTER, bool STREAM>
__global__ void __launch_bounds__(kThreads)
    adamw8_kernel(AdamwBatch b, AdamwHyper h) {
  using P = typename std::conditional<MASTER, float, T>::type;
  const int t = tensor_of(b, blockIdx.x);
  const int64_t base = (int64_t)((int)blockIdx.x - b.chunk_start[t]) * kAdamwChunk;
  const int64_t left = b.n[t] - base;
  const int len = left < kAdamwChunk ? (int)left : kAdamwChunk;
  T *p16 = static_cast<T *>(b.p[t]) + base;
  P *p = MASTER ? reinterpret_cast<P *>(b.master[t]) + base
                : reinterpret_cast<P *>(p16);
  const T *g = static_cast<const T *>(b.g[t]) + base;
  uint32_t *mw = static_cast<uint32_t *>(b.m[t]) + base / 4;
  uint32_t *rw = static_cast<uint32_t *>(b.v[t]) + base / 4;
  float *ms = b.m_scale[t] + base / kBlock;
  float *rs = b.v_scale[t] + base / kBlock;
  const bool wide = aligned16(p16, p, g, mw, rw);
  const Consts c = constants(h);
  const uint32_t step = (uint32_t)h.step[0];
  constexpr Access kFull = STREAM ? kStream : kWhole;
  if (wide && len == kAdamwChunk)
    chunk8<kFull, T, MASTER>(c, p16, p, g, mw, rw, ms, rs, base, len, wide,
                             step, h.seed);
  else
    chunk8<kBounded, T, MASTER>(c, p16, p, g, mw, rw, ms, rs, base, len, wide,
                                step, h.seed);
}

template <typename T, bool MASTER, bool STREAM>
void launch(const AdamwBatch &b, const AdamwHyper &h, bool eight, int chunks,
            hipStream_t s) {
  if (eight)
    hipLaunchKernelGGL((adamw8_kernel<T, MASTER, STREAM>), dim3(chunks),
                       dim3(kThreads), 0, s, b, h);
  else
    hipLaunchKernelGGL((adamw_kernel<T, MASTER, STREAM>), dim3(chunks),
                       dim3(kThreads), 0, s, b, h);
}

// A step that moves more than half the 256 MB last-level cache reads and writes
// past it (141 M parameters: float32 683 us instead of 753, bfloat16 with
// masters 730 instead of 776, with 8-bit states 438 instead of 463); what a
// smaller one touches may still be there for the next forward pass.
constexpr int64_t kStreamBytes = 128 << 20;

}  // namespace

}  // namespace sa

using namespace sa;

int sa_adamw_update_multi(int dtype, int state_bits, int count, void *const *p,
                          const void *const *g, float *const *master,
                          void *const *m, void *const *v, float *const *m_scale,
                          float *const *v_scale, const int64_t *n,
                          const AdamwHyper *hyper, hipStream_t s) {
  if (state_bits != 8 && state_bits != 32) return -2;
  if (state_bits == 8 && (!m_scale || !v_scale)) return -2;
  int64_t all = 0;
  for (int i = 0; i < count; ++i) all += n[i];
  const bool stream = all * (state_bits == 8 ? 16 : 28) > kStreamBytes;
  for (int first = 0; first < count;) {
    AdamwBatch b;
    int64_t chunks = 0;
    int k = 0;
    for (; k < kAdamwMaxTensors && first + k < count; ++k) {
      const int i = first + k;
      const int64_t mine = (n[i] + kAdamwChunk - 1) / kAdamwChunk;
      // a launch counts its threads in 32 bits
      if (mine > kLaunchChunks) return -2;
      if (chunks + mine > kLaunchChunks) break;   // the rest in the next one
      b.p[k] = p[i];
      b.g[k] = g[i];
      b.master[k] = master ? master[i] : nullptr;
      b.m[k] = m[i];
      b.v[k] = v[i];
      b.m_scale[k] = m_scale ? m_scale[i] : nullptr;
      b.v_scale[k] = v_scale ? v_scale[i] : nullptr;
      b.n[k] = n[i];
      b.chunk_start[k] = (int)chunks;
      chunks += mine;
    }
    b.count = k;
    first += k;
    if (chunks == 0) continue;
    const bool eight = state_bits == 8;
    SA_DISPATCH_FLOAT(dtype, T, {
      if (master)
        stream ? launch<T, true, true>(b, *hyper, eight, (int)chunks, s)
               : launch<T, true, false>(b, *hyper, eight, (int)chunks, s);
      else
        stream ? launch<T, false, true>(b, *hyper, eight, (int)chunks, s)
               : launch<T, false, false>(b, *hyper, eight, (int)chunks, s);
    });
  }
  return 0;
}
