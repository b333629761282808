// Losses over the log-probabilities of given tokens, forward and backward.
//
//   lp[r] = x[r, t[r]] - log sum_v exp(x[r, v])           logits x (rows, V)
//
//   log-probabilities  y[r] = lp[r]
//   preference         rows are 2 P sequences of S tokens, the P chosen ones
//                      first; a[i] = sum over sequence i of (lp - ref),
//                      z = beta (a[chosen] - a[rejected]),
//                      loss = -mean((1 - s) log sigma(z) + s log sigma(-z))
//   policy             r = exp(lp - old), d = ref - lp,
//                      loss = sum w (-min(r A, clip(r) A) + kl (exp d - d - 1))
//                             / sum w
// A row whose label lies outside [0, V) -- and for the policy loss one whose
// weight is 0 -- takes no part: its logits are not read and its gradient is 0.
// The gradient of every loss is c[r] (1[v = t[r]] - softmax(x[r])[v]).
//
// Bound by memory: the forward pass reads the logits once (running maximum and
// sum of the exponentials), the backward pass reads them again -- c[r] depends
// on every row -- and writes the gradient; the probabilities never reach
// memory.  Maxima, sums and log-probabilities are float32, sums over tokens
// float64.  8192 x 50257 bfloat16 logits, three tenths of the tokens ignored:
// forward 102 us (5.6 TB/s of what is read), backward 252 us (5.5 TB/s); a large
// copy reaches 5.1 TB/s.  Few rows are cut into pieces (8 x 131071 float32: 4 us
// and 3.5 us to join them).
//
// The reference has no such operators (its soft-max loss,
// python/singa/autograd.py:1204-1271, keeps the probabilities and averages over
// the rows).
#include "common.cuh"
#include "kernels.h"

namespace sa {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kUnroll = 4;   // 16-byte loads a thread has in flight

__device__ __forceinline__ float fexp(float v) {
  return __builtin_amdgcn_exp2f(v * kLog2e);
}

// A running (maximum, sum of exp(v - maximum)).  A maximum of minus infinity
// is replaced by 0 as the reference point: exp(-inf) adds nothing, while NaN
// and plus infinity turn the sum into NaN, as in the definition.
struct Running {
  float m = -INFINITY, s = 0.f;
};

__device__ __forceinline__ float reference_point(float m) {
  return m == -INFINITY ? 0.f : m;
}

template <int N>
__device__ __forceinline__ void add(Running &r, const float (&v)[N]) {
  float top = r.m;
#pragma unroll
  for (int i = 0; i < N; ++i) top = fmaxf(top, v[i]);
  const float ref = reference_point(top);
  float s = r.s * fexp(r.m - ref);
#pragma unroll
  for (int i = 0; i < N; ++i) s += fexp(v[i] - ref);
  r.m = top;
  r.s = s;
}

__device__ __forceinline__ Running join(const Running &a, const Running &b) {
  Running r;
  r.m = fmaxf(a.m, b.m);
  const float ref = reference_point(r.m);
  r.s = a.s * fexp(a.m - ref) + b.s * fexp(b.m - ref);
  return r;
}

template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <bool STREAM, typename P>
__device__ __forceinline__ void put(P *at, const P &v) {
  if constexpr (STREAM && sizeof(P) == 16)
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v),
                                reinterpret_cast<u32x4 *>(at));
  else
    *at = v;
}

// Elements before the first 16-byte boundary of p, at most n
template <typename T, int VEC>
__device__ __forceinline__ int64_t lead(const T *p, int64_t n) {
  if (VEC == 1) return 0;
  const int64_t h =
      (int64_t)((0 - reinterpret_cast<uintptr_t>(p)) & 15) / (int)sizeof(T);
  return h < n ? h : n;
}

// n logits at p, shared by `threads` threads
template <typename T, int VEC>
__device__ __forceinline__ Running scan(const T *p, int64_t n, int tid,
                                        int threads) {
  Running r;
  const int64_t h = lead<T, VEC>(p, n), packs = (n - h) / VEC;
  const Pack<T, VEC> *q = reinterpret_cast<const Pack<T, VEC> *>(p + h);
  int64_t i = tid;
  for (; i + (kUnroll - 1) * (int64_t)threads < packs;
       i += kUnroll * (int64_t)threads) {
    Pack<T, VEC> k[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) k[u] = q[i + u * threads];
    float v[kUnroll * VEC];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[u * VEC + j] = to_f<T>(k[u].v[j]);
    add(r, v);
  }
  for (; i < packs; i += threads) {
    const Pack<T, VEC> k = q[i];
    float v[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = to_f<T>(k.v[j]);
    add(r, v);
  }
  // the elements in front of and behind the aligned packs
  if (tid < h) {
    const float v[1] = {to_f<T>(p[tid])};
    add(r, v);
  }
  const int64_t rest = h + packs * VEC;
  if (tid < n - rest) {
    const float v[1] = {to_f<T>(p[rest + tid])};
    add(r, v);
  }
  return r;
}

__device__ __forceinline__ Running join_wave(Running r) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    Running o;
    o.m = __shfl_xor(r.m, off, 64);
    o.s = __shfl_xor(r.s, off, 64);
    r = join(r, o);
  }
  return r;
}

__device__ __forceinline__ bool takes_part(const TokenLossDesc &d, int64_t r) {
  const int t = d.label[r];
  return t >= 0 && t < d.V &&
         (d.mode != kPolicy || !d.weight || d.weight[r] != 0.f);
}

// what follows for one row from its maximum and sum: one thread
template <typename T>
__device__ void finish_row(const TokenLossDesc &d, int64_t r, bool used,
                           Running run) {
  if (!used) {
    d.top[r] = d.norm[r] = 0.f;
    d.value[r] = 0.f;
    if (d.mode == kPolicy) d.coef[r] = 0.f;
    return;
  }
  const float ls = logf(run.s);
  const float lp =
      (to_f<T>(((const T *)d.x)[r * d.V + d.label[r]]) - run.m) - ls;
  d.top[r] = run.m;
  d.norm[r] = ls;
  if (d.mode == kLogProb) {
    d.value[r] = lp;
  } else if (d.mode == kPreference) {
    d.value[r] = lp - d.ref[r];
  } else {
    const float w = d.weight ? d.weight[r] : 1.f, A = d.adv[r];
    const float ratio = expf(lp - d.old[r]);
    const float plain = ratio * A;
    const float cut =
        (ratio < d.clip_lo ? d.clip_lo : ratio > d.clip_hi ? d.clip_hi : ratio) *
        A;
    // NaN goes through both
    const bool clipped = cut < plain;
    float each = -(clipped ? cut : plain), c = clipped ? 0.f : -plain;
    if (d.ref) {
      const float diff = d.ref[r] - lp, e = expm1f(diff);
      each += d.kl * (e - diff);
      c -= d.kl * e;
    }
    d.value[r] = w * each;
    d.coef[r] = w * c;
  }
}

constexpr int threads_of(int waves) { return waves == 1 ? 256 : 64 * waves; }

// WPR waves share a row, a workgroup has one row (WPR 1: four); gridDim.y
// pieces of a row (not with WPR 1) leave their (maximum, sum) in d.part for
// the join kernel.
template <typename T, int VEC, int WPR>
__global__ void __launch_bounds__(threads_of(WPR))
    token_rows_kernel(TokenLossDesc d) {
  const int wave = threadIdx.x >> 6;
  const int64_t r =
      d.first + (WPR == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x);
  const bool used = r < d.rows && takes_part(d, r);
  Running run;
  if (used) {
    const int64_t c0 = (int64_t)blockIdx.y * d.piece;
    const int64_t n = d.V - c0 < d.piece ? d.V - c0 : d.piece;
    run = scan<T, VEC>((const T *)d.x + r * d.V + c0, n,
                       threadIdx.x & (64 * WPR - 1), 64 * WPR);
    run = join_wave(run);
  }
  if (WPR > 1) {   // one row for the whole workgroup: `used` is uniform
    __shared__ float2 all[WPR];
    if ((threadIdx.x & 63) == 0) all[wave] = make_float2(run.m, run.s);
    __syncthreads();
    run = Running{all[0].x, all[0].y};
#pragma unroll
    for (int i = 1; i < WPR; ++i) run = join(run, Running{all[i].x, all[i].y});
  }
  if ((threadIdx.x & (64 * WPR - 1)) != 0 || r >= d.rows) return;
  if (WPR > 1 && gridDim.y > 1)
    d.part[r * gridDim.y + blockIdx.y] = make_float2(run.m, run.s);
  else
    finish_row<T>(d, r, used, run);
}

// the pieces of a row joined by one wave
template <typename T>
__global__ void __launch_bounds__(64)
    token_join_kernel(TokenLossDesc d, int pieces) {
  const int64_t r = blockIdx.x;   // few rows: one launch
  const bool used = takes_part(d, r);
  Running run;
  if (used) {
    for (int i = threadIdx.x; i < pieces; i += 64) {
      const float2 p = d.part[r * pieces + i];
      run = join(run, Running{p.x, p.y});
    }
    run = join_wave(run);
  }
  if (threadIdx.x == 0) finish_row<T>(d, r, used, run);
}

// sums of two doubles over a workgroup of 1024 threads, in a fixed order
__device__ __forceinline__ void block_sums(double &a, double &b) {
  __shared__ double sa_[16], sb_[16];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    a += __shfl_xor(a, off, 64);
    b += __shfl_xor(b, off, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    sa_[threadIdx.x >> 6] = a;
    sb_[threadIdx.x >> 6] = b;
  }
  __syncthreads();
  a = b = 0.0;
  for (int i = 0; i < 16; ++i) {
    a += sa_[i];
    b += sb_[i];
  }
}

// -log sigma(z) = log(1 + exp(-z)), without overflow
__device__ __forceinline__ double soft_plus(double v) {
  return fmax(v, 0.0) + log1p(exp(-fabs(v)));
}

// What the rows left is added up by one workgroup up to kOneBlockRows rows (16
// loads for each thread and value, 4 to 5 us), above that by many first.
constexpr int64_t kOneBlockRows = 32768;
constexpr int kParts = 256;

// loss and weight of every `step`-th row
__device__ __forceinline__ void add_rows(const TokenLossDesc &d, int64_t first,
                                         int64_t step, double &loss,
                                         double &total) {
#pragma unroll 4
  for (int64_t r = first; r < d.rows; r += step) {
    const int t = d.label[r];
    const float w = d.weight ? d.weight[r] : 1.f;
    loss += (double)d.value[r];
    total += t >= 0 && t < d.V ? (double)w : 0.0;
  }
}

__global__ void __launch_bounds__(1024) policy_parts_kernel(TokenLossDesc d) {
  double loss = 0.0, total = 0.0;
  add_rows(d, (int64_t)blockIdx.x * 1024 + threadIdx.x, 1024 * kParts, loss,
           total);
  block_sums(loss, total);
  if (threadIdx.x == 0) {
    d.sums[2 * blockIdx.x] = loss;
    d.sums[2 * blockIdx.x + 1] = total;
  }
}

__global__ void __launch_bounds__(1024)
    policy_total_kernel(TokenLossDesc d, bool parts) {
  double loss = 0.0, total = 0.0;
  if (!parts) {
    add_rows(d, threadIdx.x, 1024, loss, total);
  } else if (threadIdx.x < kParts) {
    loss = d.sums[2 * threadIdx.x];
    total = d.sums[2 * threadIdx.x + 1];
  }
  block_sums(loss, total);
  if (threadIdx.x != 0) return;
  if (!(total > 0.0)) total = 1.0;   // no token takes part
  d.loss[0] = (float)(loss / total);
  d.total[0] = (float)(1.0 / total);
}

// sum of a sequence's values, a workgroup for each
__global__ void __launch_bounds__(1024)
    preference_parts_kernel(TokenLossDesc d) {
  const float *v = d.value + (int64_t)blockIdx.x * d.seq;
  double sum = 0.0, none = 0.0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < d.seq; i += 1024) sum += (double)v[i];
  block_sums(sum, none);
  if (threadIdx.x == 0) d.sums[blockIdx.x] = sum;
}

__global__ void __launch_bounds__(1024)
    preference_total_kernel(TokenLossDesc d, bool parts) {
  __shared__ double share[16];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t seqs = 2 * d.pairs;
  // several waves take a sequence where there are few of them
  int each = 1;
  while (each < 16 && 2 * each * seqs <= 16) each <<= 1;
  const int at_once = 16 / each, mine = wave / each, sub = wave % each;
  for (int64_t first = 0; !parts && first < seqs; first += at_once) {
    const int64_t q = first + mine;
    double sum = 0.0;
    if (q < seqs) {
      const float *v = d.value + q * d.seq;
#pragma unroll 4
      for (int64_t i = sub * 64 + lane; i < d.seq; i += 64 * each)
        sum += (double)v[i];
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if (lane == 0) share[wave] = sum;
    __syncthreads();
    if ((int)threadIdx.x < at_once && first + threadIdx.x < seqs) {
      double a = 0.0;
      for (int k = 0; k < each; ++k) a += share[threadIdx.x * each + k];
      d.sums[first + threadIdx.x] = a;
    }
    __syncthreads();
  }
  __threadfence_block();
  __syncthreads();
  double loss = 0.0, none = 0.0;
  const double smooth = d.smoothing, beta = d.beta;
  for (int64_t i = threadIdx.x; i < d.pairs; i += 1024) {
    const double z = beta * (d.sums[i] - d.sums[d.pairs + i]);
    loss += (1.0 - smooth) * soft_plus(-z) + smooth * soft_plus(z);
    const double up = 1.0 / (1.0 + exp(-z)), down = 1.0 / (1.0 + exp(z));
    d.total[i] = (float)((smooth * up - (1.0 - smooth) * down) * beta /
                         (double)d.pairs);
  }
  block_sums(loss, none);
  if (threadIdx.x == 0) d.loss[0] = (float)(loss / (double)d.pairs);
}

// dx[r, v] = c[r] (1[v = t[r]] - exp((x[r, v] - max[r]) - log sum[r])).  The two
// are kept apart: added up, a row of large logits would lose the logarithm.
// Rows are taken from the last to the first, so that the logits the forward
// pass read last are met while they are still in the last-level cache.
// STREAM: the gradient is stored past the caches.
template <typename T, int VEC, int WPR, bool STREAM>
__global__ void __launch_bounds__(threads_of(WPR))
    token_grad_kernel(TokenLossDesc d) {
  const int64_t q = d.first + (WPR == 1 ? (int64_t)blockIdx.x * 4 +
                                              (threadIdx.x >> 6)
                                        : blockIdx.x);
  if (q >= d.rows) return;
  const int64_t r = d.rows - 1 - q;
  const int tid = threadIdx.x & (64 * WPR - 1), threads = 64 * WPR;
  const int64_t c0 = (int64_t)blockIdx.y * d.piece;
  const int64_t n = d.V - c0 < d.piece ? d.V - c0 : d.piece;
  const T *x = (const T *)d.x + r * d.V + c0;
  T *dx = (T *)d.dx + r * d.V + c0;
  float c = 0.f;
  if (takes_part(d, r)) {
    if (d.mode == kLogProb) {
      c = d.dy[r];
    } else {
      c = d.dy_scale * (d.dy ? d.dy[0] : 1.f);
      if (d.mode == kPolicy) {
        c *= d.coef[r] * d.total[0];
      } else {
        const int64_t s = r / d.seq;
        c *= s < d.pairs ? d.total[s] : -d.total[s - d.pairs];
      }
    }
  }
  const int64_t h = lead<T, VEC>(x, n), packs = (n - h) / VEC;
  Pack<T, VEC> *o = reinterpret_cast<Pack<T, VEC> *>(dx + h);
  const int64_t rest = h + packs * VEC;
  if (c == 0.f) {
    Pack<T, VEC> z;
#pragma unroll
    for (int j = 0; j < VEC; ++j) z.v[j] = from_f<T>(0.f);
    for (int64_t i = tid; i < packs; i += threads) put<STREAM>(o + i, z);
    if (tid < h) dx[tid] = from_f<T>(0.f);
    if (tid < n - rest) dx[rest + tid] = from_f<T>(0.f);
    return;
  }
  const float top = d.top[r], norm = d.norm[r];
  const int64_t label = d.label[r] - c0;   // within this piece
  auto grad = [&](T v) { return -c * fexp((to_f<T>(v) - top) - norm); };
  const Pack<T, VEC> *p = reinterpret_cast<const Pack<T, VEC> *>(x + h);
  auto one = [&](int64_t i, const Pack<T, VEC> &k) {
    float g[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) g[j] = grad(k.v[j]);
    const int64_t at = label - (h + i * VEC);
    if (at >= 0 && at < VEC) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) g[j] += j == at ? c : 0.f;
    }
    Pack<T, VEC> out;
#pragma unroll
    for (int j = 0; j < VEC; ++j) out.v[j] = from_f<T>(g[j]);
    put<STREAM>(o + i, out);
  };
  int64_t i = tid;
  for (; i + (kUnroll - 1) * (int64_t)threads < packs;
       i += kUnroll * (int64_t)threads) {
    Pack<T, VEC> k[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) k[u] = p[i + u * threads];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) one(i + u * threads, k[u]);
  }
  for (; i < packs; i += threads) one(i, p[i]);
  if (tid < h)
    dx[tid] = from_f<T>(grad(x[tid]) + (label == tid ? c : 0.f));
  if (tid < n - rest)
    dx[rest + tid] =
        from_f<T>(grad(x[rest + tid]) + (label == rest + tid ? c : 0.f));
}

int check_desc(const TokenLossDesc &d) {
  if (d.rows < 0 || d.V < 1 || d.rows > 0x7fffffffll || d.V > 0x7fffffffll)
    return -2;
  if (d.mode == kPreference && d.rows != 2 * d.pairs * d.seq) return -2;
  return 0;
}

// A row for each wave up to this many logits: 64 lanes then have no more than
// four (16 bits: two) of the unrolled steps.
constexpr int64_t kWaveRow = 4096;
// A row (or piece) of at least 32 KB, one unrolled step of 512 threads, is
// taken by eight waves, a shorter one by four: bf16, both directions, 8192 x
// 50257 356 us with eight and 377 with four, 4096 x 30522 114 and 119, but
// 16384 x 10007 (20 KB) 166 and 141.
constexpr int64_t kLongRow = 32 << 10;
// A gradient of over half the 256 MB last-level cache is stored past it: it
// would not stay there for whoever reads it next, and throws out the logits
// (8192 x 50257 bf16: 356 us instead of 388, 4096 x 30522 114 instead of 134).
constexpr int64_t kStreamBytes = 128 << 20;

// rows of one launch: its threads are counted in 32 bits
constexpr int64_t kLaunchRows = 1 << 22;

template <typename T, int VEC>
void launch_rows(const TokenLossDesc &d, int64_t rows, int pieces,
                 hipStream_t s) {
  if (d.V <= kWaveRow)
    hipLaunchKernelGGL((token_rows_kernel<T, VEC, 1>),
                       dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, d);
  else if (d.piece * (int64_t)sizeof(T) < kLongRow)
    hipLaunchKernelGGL((token_rows_kernel<T, VEC, 4>),
                       dim3((unsigned)rows, pieces), dim3(256), 0, s, d);
  else
    hipLaunchKernelGGL((token_rows_kernel<T, VEC, 8>),
                       dim3((unsigned)rows, pieces), dim3(512), 0, s, d);
}

template <typename T, int VEC, bool STREAM>
void launch_grad(const TokenLossDesc &d, int64_t rows, int pieces,
                 hipStream_t s) {
  if (d.V <= kWaveRow)
    hipLaunchKernelGGL((token_grad_kernel<T, VEC, 1, STREAM>),
                       dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, d);
  else if (d.piece * (int64_t)sizeof(T) < kLongRow)
    hipLaunchKernelGGL((token_grad_kernel<T, VEC, 4, STREAM>),
                       dim3((unsigned)rows, pieces), dim3(256), 0, s, d);
  else
    hipLaunchKernelGGL((token_grad_kernel<T, VEC, 8, STREAM>),
                       dim3((unsigned)rows, pieces), dim3(512), 0, s, d);
}

// whether every row of a and b has its 16-byte boundaries at the same places
bool same_phase(const void *a, const void *b) {
  return ((reinterpret_cast<uintptr_t>(a) ^ reinterpret_cast<uintptr_t>(b)) &
          15) == 0;
}

}  // namespace

}  // namespace sa

using namespace sa;

// Workgroups for each row: one, unless the rows alone leave most of the 256
// CUs idle; then pieces of at least 4096 logits until about 1024 workgroups
// run.
int sa_token_loss_pieces(int64_t rows, int64_t V) {
  if (V <= kWaveRow || rows >= 512 || rows < 1) return 1;
  const int64_t want = 1024 / rows, most = V / 4096;
  const int64_t p = want < most ? want : most;
  return p < 1 ? 1 : (int)p;
}

// float64 words of `sums` that a loss needs
int64_t sa_token_loss_sums(int mode, int64_t rows, int64_t pairs) {
  if (mode == kPreference) return 2 * pairs;
  return mode == kPolicy && rows > kOneBlockRows ? 2 * kParts : 0;
}

static int64_t piece_of(int64_t V, int pieces) {
  return ((V + pieces - 1) / pieces + 63) / 64 * 64;
}

int sa_token_loss_fwd(int dtype, const TokenLossDesc *desc, hipStream_t s) {
  TokenLossDesc d = *desc;
  if (int rc = check_desc(d)) return rc;
  const int pieces = sa_token_loss_pieces(d.rows, d.V);
  d.piece = piece_of(d.V, pieces);
  const bool parts = d.rows > kOneBlockRows;
  if ((pieces > 1 && !d.part) ||
      (sa_token_loss_sums(d.mode, d.rows, d.pairs) > 0 && !d.sums))
    return -2;
  SA_DISPATCH_FLOAT(dtype, T, {
    for (d.first = 0; d.first < d.rows; d.first += kLaunchRows)
      launch_rows<T, 16 / (int)sizeof(T)>(d, i64min(kLaunchRows, d.rows - d.first),
                                          pieces, s);
    if (pieces > 1)
      hipLaunchKernelGGL((token_join_kernel<T>), dim3((unsigned)d.rows),
                         dim3(64), 0, s, d, pieces);
  });
  if (d.mode == kPolicy) {
    if (parts)
      hipLaunchKernelGGL(policy_parts_kernel, dim3(kParts), dim3(1024), 0, s, d);
    hipLaunchKernelGGL(policy_total_kernel, dim3(1), dim3(1024), 0, s, d, parts);
  } else if (d.mode == kPreference && d.pairs > 0) {
    // (a workgroup for each of up to 2^21 sequences: threads in 32 bits)
    const bool many = parts && d.pairs <= (1 << 20);
    if (many)
      hipLaunchKernelGGL(preference_parts_kernel, dim3((unsigned)(2 * d.pairs)),
                         dim3(1024), 0, s, d);
    hipLaunchKernelGGL(preference_total_kernel, dim3(1), dim3(1024), 0, s, d,
                       many);
  }
  return 0;
}

int sa_token_loss_bwd(int dtype, const TokenLossDesc *desc, hipStream_t s) {
  TokenLossDesc d = *desc;
  if (int rc = check_desc(d)) return rc;
  const int pieces = sa_token_loss_pieces(d.rows, d.V);
  d.piece = piece_of(d.V, pieces);
  const bool wide = same_phase(d.x, d.dx);
  SA_DISPATCH_FLOAT(dtype, T, {
    const bool stream = d.rows * d.V * (int64_t)sizeof(T) > kStreamBytes;
    constexpr int kVec = 16 / (int)sizeof(T);
    for (d.first = 0; d.first < d.rows; d.first += kLaunchRows) {
      const int64_t rows = i64min(kLaunchRows, d.rows - d.first);
      if (!wide)
        launch_grad<T, 1, false>(d, rows, pieces, s);
      else if (stream)
        launch_grad<T, kVec, true>(d, rows, pieces, s);
      else
        launch_grad<T, kVec, false>(d, rows, pieces, s);
    }
  });
  return 0;
}
