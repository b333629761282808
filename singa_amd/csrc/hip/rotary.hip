// Rotary positions of queries and keys, with the root-mean-square norm of
// every head in the same pass, forward and backward.
//
//   x' = x * rstd * w          rstd = 1 / sqrt(mean(x^2) + eps), per head
//   y  = R(position) x'        pair i of the first R channels turns by the
//                              angle position * f_i, the rest passes through
// backward, with g = R^T dy (the transposed rotation, amplitude included):
//   dw = sum over tokens and heads of g * x * rstd
//   dx = rstd * (g w - xh * mean(g w xh)),  xh = x * rstd
// rstd is computed again from x, which the backward pass reads anyway: nothing
// but x is kept.
//
// Angles: a position times f_i in float32 is off by 2^-24 of the angle, at a
// position of a million by 0.06 of a radian.  Here f_i / (2 pi) is a 64-bit
// fixed-point fraction of a turn and the product with the integer position is
// taken modulo 2^64, that is modulo whole turns, exactly; only the remaining
// fraction becomes a float.  Any 32-bit position, negative ones too, has an
// angle good to 2^-24 of a half turn.
//
// Bound by memory: read x, write y (backward: read dy and x, write dx), about
// 30 operations for 4 bytes moved.  A team of lanes owns one head of one token:
// each lane holds V pairs (two 16-byte loads), so the pair partners are in the
// same lane in both layouts and the norm is one reduction between lanes.  cos /
// sin of a token are computed once by the workgroup into LDS and shared by its
// heads.  The frequencies travel in the kernel arguments, so a handle owns no
// device memory.  2 x 4096 tokens of 32 + 8 heads of 128, bfloat16, normed:
// forward 34 us, backward 50 us (4.9 and 5.0 TB/s; a large copy reaches 5.1), and
// 4 us to add up the scale gradients; one token for each of 16 sequences 4.5 us.
//
// The reference has no such operator.
#include "common.cuh"
#include "kernels.h"

namespace sa {

namespace {

constexpr int kThreads = 256;
constexpr int kTableMax = 1024;   // cos / sin pairs a workgroup keeps
constexpr int kTileMax = 32;      // tokens of a tile

struct RotaryPart {
  const void *x, *dy, *w;
  void *y;            // forward: y; backward: dx; contiguous (tokens, H, D)
  float *partial;     // (blocks, D): this workgroup's share of dw
  int64_t x_sb, x_ss, x_sh, g_sb, g_ss, g_sh;
  int H;
  unsigned magic;     // ceil(2^32 / H): row / H by one multiplication, which is
                      // exact below 2^32 / H rows; 0: one head
  int tile;           // tokens of a tile
  int blocks;         // workgroups of this part
};

struct RotaryArgs {
  RotaryPart part[2];
  const int *pos;
  int64_t p_sb, p_ss;
  int S, tokens, D, R;
  int units;          // D / (2 V): what a team of lanes shares
  int lanes;          // of a team: the next power of two of units, at most 64
  int flat;           // all tensors: batch stride = S times token stride
  int half;           // 1: pairs (i, i + R / 2), 0: pairs (2 i, 2 i + 1)
  float eps, amplitude;
  uint64_t freq[kRotaryMaxPairs];
};

template <typename T, int V> struct alignas(sizeof(T) * V) Vec { T v[V]; };

// the two loads of a unit, as they are in memory
template <typename T, int V> struct Unit {
  Vec<T, V> a, b;

  __device__ __forceinline__ void load(const T *row, int lo, int hi, bool ok) {
    if (ok) {
      a = *reinterpret_cast<const Vec<T, V> *>(row + lo);
      b = *reinterpret_cast<const Vec<T, V> *>(row + hi);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) a.v[j] = b.v[j] = from_f<T>(0.f);
    }
  }
  __device__ __forceinline__ void widen(float *e) const {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      e[j] = to_f<T>(a.v[j]);
      e[V + j] = to_f<T>(b.v[j]);
    }
  }
};

template <int CTRL>
__device__ __forceinline__ float add_dpp(float x) {
  const int other = __builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf,
                                                0xf, false);
  return x + __int_as_float(other);
}

// sum over each aligned group of `lanes` lanes (a power of two), in all of them
__device__ __forceinline__ float group_sum(float x, int lanes) {
  if (lanes > 1) x = add_dpp<0xb1>(x);    // quad_perm 1 0 3 2
  if (lanes > 2) x = add_dpp<0x4e>(x);    // quad_perm 2 3 0 1
  if (lanes > 4) x = add_dpp<0x141>(x);   // row_half_mirror
  if (lanes > 8) x = add_dpp<0x140>(x);   // row_mirror
  if (lanes > 16) x += __shfl_xor(x, 16, 64);
  if (lanes > 32) x += __shfl_xor(x, 32, 64);
  return x;
}

template <typename T, int V>
__device__ __forceinline__ void store_unit(T *row, int lo, int hi,
                                           const float *e) {
  Vec<T, V> a, b;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    a.v[j] = from_f<T>(e[j]);
    b.v[j] = from_f<T>(e[V + j]);
  }
  *reinterpret_cast<Vec<T, V> *>(row + lo) = a;
  *reinterpret_cast<Vec<T, V> *>(row + hi) = b;
}

// V pairs by their angles; the sign of the sine turns back
template <int V>
__device__ __forceinline__ void turn(float *e, const float2 *cs, float sign,
                                     bool half) {
  if (half) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float c = cs[j].x, s = sign * cs[j].y, a = e[j], b = e[V + j];
      e[j] = a * c - b * s;
      e[V + j] = a * s + b * c;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float c = cs[j].x, s = sign * cs[j].y, a = e[2 * j],
                  b = e[2 * j + 1];
      e[2 * j] = a * c - b * s;
      e[2 * j + 1] = a * s + b * c;
    }
  }
}

// V: pairs of a unit.  NU: units a lane holds (more than one only where a head
// has over 64 of them).  The loads of a team's next row fly while the present
// one is computed, and those of a tile's first row while the workgroup computes
// its table.
template <typename T, int V, int NU, bool NORM, bool BWD>
__global__ void __launch_bounds__(kThreads, NU == 1 ? 4 : 2)
    rotary_kernel(RotaryArgs a) {
  __shared__ float2 cs[kTableMax];
  constexpr bool kSums = NORM && BWD, kReadX = !BWD || NORM;
  __shared__ float sums[kSums ? 4 * 128 * V * NU : 1];
  const int which = (int)blockIdx.x >= a.part[0].blocks;
  const RotaryPart &p = a.part[which];
  const int block = (int)blockIdx.x - (which ? a.part[0].blocks : 0);
  const int tid = threadIdx.x;
  const int lane = tid & (a.lanes - 1), team = tid / a.lanes;
  const int teams = kThreads / a.lanes;
  const int D = a.D, R = a.R, pairs = R >> 1, H = p.H;
  const bool half = a.half != 0;
  const float inv_D = 1.f / (float)D;

  int lo[NU], hi[NU], at[NU];   // element offsets, first pair in the table
  bool mine[NU], turns[NU];
  float w[NU][2 * V], acc[NU][2 * V];
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    const int unit = lane + u * a.lanes;
    mine[u] = unit < a.units;
    at[u] = unit * V;
    turns[u] = mine[u] && at[u] < pairs;
    if (half && turns[u]) {
      lo[u] = unit * V;
      hi[u] = lo[u] + pairs;
    } else {
      lo[u] = 2 * unit * V;
      hi[u] = lo[u] + V;
    }
#pragma unroll
    for (int j = 0; j < 2 * V; ++j) {
      w[u][j] = 1.f;
      acc[u][j] = 0.f;
    }
    if (NORM) {
      Unit<T, V> raw;
      raw.load((const T *)p.w, lo[u], hi[u], mine[u]);
      raw.widen(w[u]);
    }
  }

  for (int64_t tile = block; tile * p.tile < a.tokens; tile += p.blocks) {
    const int first = (int)(tile * p.tile);
    const int count = a.tokens - first < p.tile ? a.tokens - first : p.tile;
    const int rows = count * H;
    Unit<T, V> x_next[NU], g_next[NU];
    int t_next = 0, head_next = 0;
    auto fetch = [&](int row) {
      const bool ok = row < rows;
      const int t = !ok ? 0 : p.magic ? (int)__umulhi((unsigned)row, p.magic)
                                      : row;
      t_next = t;
      head_next = ok ? row - t * H : 0;
      // tokens are one after another in memory, or batches lie apart
      int64_t b = 0, s = first + t;
      if (!a.flat) {
        b = (first + t) / a.S;
        s -= b * a.S;
      }
      const T *xr = (const T *)p.x + b * p.x_sb + s * p.x_ss +
                    head_next * p.x_sh;
      const T *gr = (const T *)p.dy + b * p.g_sb + s * p.g_ss +
                    head_next * p.g_sh;
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        if (kReadX) x_next[u].load(xr, lo[u], hi[u], ok && mine[u]);
        if (BWD) g_next[u].load(gr, lo[u], hi[u], ok && mine[u]);
      }
    };
    fetch(team);
    __syncthreads();   // the previous tile's table has been used
    for (int e = tid; e < count * pairs; e += kThreads) {
      const int t = e / pairs, i = e - t * pairs;
      const int b = (first + t) / a.S, s = (first + t) - b * a.S;
      const int64_t position =
          a.pos ? (int64_t)a.pos[b * a.p_sb + s * a.p_ss] : (int64_t)s;
      const uint64_t turn64 = (uint64_t)position * a.freq[i];
      // signed fraction of a half turn in [-1, 1)
      const float f = (float)(int32_t)(turn64 >> 32) * 0x1p-31f;
      float sn, c;
      sincospif(f, &sn, &c);
      cs[e] = make_float2(c * a.amplitude, sn * a.amplitude);
    }
    __syncthreads();
    for (int base = 0; base < rows; base += teams) {
      const bool ok = base + team < rows;
      const int t = t_next;
      T *out = (T *)p.y + ((int64_t)(first + t) * H + head_next) * D;
      float e[NU][2 * V], g[NU][2 * V];
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        if (kReadX) x_next[u].widen(e[u]);
        if (BWD) g_next[u].widen(g[u]);
      }
      if (base + teams < rows) fetch(base + teams + team);
      float rstd = 1.f;
      if (NORM) {
        float sq = 0.f;
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) sq += e[u][j] * e[u][j];
        // a team without a row: nothing, also where eps is 0
        rstd = ok ? rsqrtf(group_sum(sq, a.lanes) * inv_D + a.eps) : 0.f;
      }
      if (!BWD) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          if (!(ok && mine[u])) continue;
          if (NORM) {
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) e[u][j] = e[u][j] * rstd * w[u][j];
          }
          if (turns[u]) turn<V>(e[u], cs + t * pairs + at[u], 1.f, half);
          store_unit<T, V>(out, lo[u], hi[u], e[u]);
        }
        continue;
      }
      float dot = 0.f;
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        if (turns[u]) turn<V>(g[u], cs + t * pairs + at[u], -1.f, half);
        if (NORM) {
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) {
            e[u][j] *= rstd;
            acc[u][j] += g[u][j] * e[u][j];
            g[u][j] *= w[u][j];
            dot += g[u][j] * e[u][j];
          }
        }
      }
      if (NORM) dot = group_sum(dot, a.lanes) * inv_D;
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        if (!(ok && mine[u])) continue;
        if (NORM) {
#pragma unroll
          for (int j = 0; j < 2 * V; ++j)
            g[u][j] = rstd * (g[u][j] - e[u][j] * dot);
        }
        store_unit<T, V>(out, lo[u], hi[u], g[u]);
      }
    }
  }

  if (kSums) {
    // teams of a wave, then the four waves, in a fixed order
    const int wave = tid >> 6;
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int j = 0; j < 2 * V; ++j)
        for (int off = 32; off >= a.lanes; off >>= 1)
          acc[u][j] += __shfl_xor(acc[u][j], off, 64);
    if ((tid & 63) < a.lanes) {
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        if (!mine[u]) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          sums[wave * D + lo[u] + j] = acc[u][j];
          sums[wave * D + hi[u] + j] = acc[u][V + j];
        }
      }
    }
    __syncthreads();
    for (int d = tid; d < D; d += kThreads)
      p.partial[(int64_t)block * D + d] =
          (sums[d] + sums[D + d]) + (sums[2 * D + d] + sums[3 * D + d]);
  }
}

// dw[d] = sum over workgroups of partial[., d], in a fixed order: 16 columns
// of one part per workgroup, 64 rows of threads over the partial sums
template <typename T>
__global__ void __launch_bounds__(1024)
    rotary_scale_kernel(const float *p0, const float *p1, int n0, int n1, T *w0,
                        T *w1, int D) {
  __shared__ float s[64][17];
  const float *p = blockIdx.y ? p1 : p0;
  const int n = blockIdx.y ? n1 : n0;
  T *w = blockIdx.y ? w1 : w0;
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
  const int d = blockIdx.x * 16 + c;
  float v = 0.f;
  if (d < D) {
#pragma unroll 8
    for (int i = r; i < n; i += 64) v += p[(int64_t)i * D + d];
  }
  s[r][c] = v;
  __syncthreads();
  for (int k = 32; k > 0; k >>= 1) {
    if (r < k) s[r][c] += s[r + k][c];
    __syncthreads();
  }
  if (r == 0 && d < D) w[d] = from_f<T>(s[0][c]);
}

template <typename T, int V, bool NORM, bool BWD>
void launch(const RotaryArgs &a, int grid, hipStream_t s) {
  constexpr int kMany = 8 / V > 1 ? 8 / V : 1;
  if (a.units <= 64)
    hipLaunchKernelGGL((rotary_kernel<T, V, 1, NORM, BWD>), dim3(grid),
                       dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((rotary_kernel<T, V, kMany, NORM, BWD>), dim3(grid),
                       dim3(kThreads), 0, s, a);
}

template <typename T, int V>
void launch(const RotaryArgs &a, bool norm, bool bwd, int grid, hipStream_t s) {
  if (norm)
    bwd ? launch<T, V, true, true>(a, grid, s)
        : launch<T, V, true, false>(a, grid, s);
  else
    bwd ? launch<T, V, false, true>(a, grid, s)
        : launch<T, V, false, false>(a, grid, s);
}

}  // namespace

static int rotary_run(int dtype, const RotaryDesc *d, bool bwd, hipStream_t s) {
  const int size = dtype == kF32 ? 4 : 2;
  if (dtype != kF32 && dtype != kF16 && dtype != kBF16) return -1;
  if (d->D < 2 || d->D > kRotaryMaxDim || (d->D & 1) || d->R < 2 ||
      d->R > d->D || (d->R & 1) || d->R > 2 * kRotaryMaxPairs || d->B < 0 ||
      d->S < 0 || (int64_t)d->B * d->S > 1ll << 30)
    return -2;
  RotaryArgs a;
  a.tokens = (int)(d->B * d->S);
  if (a.tokens == 0) return 0;
  a.pos = d->pos;
  a.p_sb = d->pos_stride[0];
  a.p_ss = d->pos_stride[1];
  a.S = (int)d->S;
  a.D = d->D;
  a.R = d->R;
  a.half = d->half;
  a.flat = 1;
  a.eps = d->eps;
  a.amplitude = d->amplitude;
  for (int i = 0; i < d->R / 2; ++i) a.freq[i] = d->freq[i];
  // pairs of a unit: the widest access that divides the rotated and the passed
  // channels and that every row's address allows
  int V = 16 / size;
  // the backward pass of the norm holds six values for each of its inputs: with
  // eight 16-bit pairs a lane it spills (2 x 4096 x 40 heads of 128, bf16: 66 us
  // instead of 61)
  if (bwd && d->norm && V > 4) V = 4;
  auto fits = [&](int v) {
    if (d->R % (2 * v) || d->D % (2 * v)) return false;
    // the two halves of the half layout start R / 2 apart: a multiple of v
    const uintptr_t bytes = (uintptr_t)v * size - 1;
    for (int i = 0; i < d->parts; ++i) {
      const RotaryTensor &t = d->part[i];
      const void *ptr[] = {t.x, t.dy, t.w, t.y};
      for (const void *q : ptr)
        if (reinterpret_cast<uintptr_t>(q) & bytes) return false;
      for (int k = 0; k < 3; ++k)
        if ((bwd && t.dy_stride[k] % v) || (t.x && t.x_stride[k] % v))
          return false;
    }
    return true;
  };
  while (V > 1 && !fits(V)) V >>= 1;
  a.units = d->D / (2 * V);
  if (a.units > 64 * (8 / V > 1 ? 8 / V : 1)) return -2;
  a.lanes = 1;
  while (a.lanes < a.units && a.lanes < 64) a.lanes <<= 1;
  const int teams = kThreads / a.lanes, pairs = d->R / 2;
  int grid = 0;
  const bool sums = bwd && d->norm;
  for (int i = 0; i < 2; ++i) {
    RotaryPart &p = a.part[i];
    p = RotaryPart{};
    p.tile = 1;
    if (i >= d->parts) continue;
    const RotaryTensor &t = d->part[i];
    if (t.H <= 0 || t.H > 65536) return -2;
    p.x = t.x; p.dy = t.dy; p.w = t.w; p.y = t.y; p.partial = t.partial;
    p.x_sb = t.x_stride[0]; p.x_ss = t.x_stride[1]; p.x_sh = t.x_stride[2];
    p.g_sb = t.dy_stride[0]; p.g_ss = t.dy_stride[1]; p.g_sh = t.dy_stride[2];
    p.H = t.H;
    if (d->B > 1 && ((t.x && p.x_sb != d->S * p.x_ss) ||
                     (bwd && p.g_sb != d->S * p.g_ss)))
      a.flat = 0;
    p.magic = t.H == 1 ? 0 : (unsigned)((0x100000000ull + t.H - 1) / t.H);
    // four rows for each team, fewer where that leaves CUs idle (3 x 1021 tokens
    // of 15 heads: 27 us for both directions, 34 when 1024 tiles are asked for)
    int tile = 4 * teams / t.H;
    tile = tile < 1 ? 1 : tile > kTileMax ? kTileMax : tile;
    while (tile > 1 && tile * pairs > kTableMax) tile >>= 1;
    while (tile > 1 && a.tokens / tile < 512) tile >>= 1;
    p.tile = tile;
    p.blocks = (a.tokens + tile - 1) / tile;
    // (a launch counts its threads in 32 bits; workgroups stride over the tiles)
    if (p.blocks > 1 << 22) p.blocks = 1 << 22;
    if (sums && p.blocks > kRotaryMaxBlocks) p.blocks = kRotaryMaxBlocks;
    grid += p.blocks;
  }
  const int v = V;
#define SA_ROTARY(T)                                                  \
  switch (v) {                                                        \
    case 8: launch<T, sizeof(T) == 4 ? 4 : 8>(a, d->norm, bwd, grid, s); break; \
    case 4: launch<T, 4>(a, d->norm, bwd, grid, s); break;            \
    case 2: launch<T, 2>(a, d->norm, bwd, grid, s); break;            \
    default: launch<T, 1>(a, d->norm, bwd, grid, s);                  \
  }
  SA_DISPATCH_FLOAT(dtype, T, {
    SA_ROTARY(T)
    if (sums)
      hipLaunchKernelGGL((rotary_scale_kernel<T>),
                         dim3((a.D + 15) / 16, d->parts), dim3(1024), 0, s,
                         a.part[0].partial, a.part[1].partial, a.part[0].blocks,
                         a.part[1].blocks, (T *)d->part[0].dw,
                         (T *)d->part[1].dw, a.D);
  });
#undef SA_ROTARY
  return 0;
}

}  // namespace sa

int sa_rotary_fwd(int dtype, const sa::RotaryDesc *d, hipStream_t s) {
  return sa::rotary_run(dtype, d, false, s);
}

int sa_rotary_bwd(int dtype, const sa::RotaryDesc *d, hipStream_t s) {
  return sa::rotary_run(dtype, d, true, s);
}
