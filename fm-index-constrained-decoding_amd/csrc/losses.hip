// losses.hip -- log-probabilities of chosen tokens under the document
// constraint, the losses on them, and their gradients.
//
// Row n holds V scores s and a mask value v per token (row_mask.h).  A token
// is IN when v != -inf; then z = s + v, added in f32 and rounded to the scores
// dtype exactly as the epilogue does, so z is the score the sampler saw:
//     logp[n] = z_a / T - log sum_{IN} exp(z_t / T)          (a = the row's token)
//     dlogp / ds_t = (1[t = a] - exp(z_t / T - lse)) / T     (0 where t is not IN)
// The rounding's derivative is taken as 1.  A row whose token lies outside
// [0, V) counts nowhere (logp 0); a row whose z_a is -inf has logp -inf and
// also adds no loss and no gradient.
//
// Every sum is kept relative to the row's maximum m: sum_t exp2((z_t - m) k)
// with k = log2(e) / T.  The difference is taken before the scale, so scores
// near the dtype's lowest value neither overflow nor lose digits; m starts at
// -FLT_MAX, so a row of nothing but -inf gives a sum of 0 and no NaN.
// Log-probabilities are finished in f64 (one log per row), because sequences
// add up hundreds of them and clip borders compare them.
#include "fmidx_internal.h"
#include "row_mask.h"
#include "../../include/fmidx.h"

#include <algorithm>
#include <cfloat>
#include <cmath>

namespace fmidx {
namespace {

constexpr int kRowThreads = 256;
constexpr int kOneThreads = 1024;      // the single-workgroup loss kernels

struct Rows {
  const void* scores;
  uint64_t ld, ld_outer;      // row n: (n / inner) * ld_outer + (n % inner) * ld
  uint32_t inner, N, V;
  const int64_t* tokens;
  const uint32_t* bits;
  uint64_t ldb;
  const uint32_t* uni;
  const RowParams* rp;
  int64_t eos;
  float k;                    // log2(e) / T
  float inv_t;
  double inv_t64;
};

typedef unsigned los_v4u __attribute__((ext_vector_type(4)));
// rows start wherever their stride puts them: 16-B accesses of the element's alignment
typedef los_v4u los_v4u_a2 __attribute__((aligned(2)));
typedef los_v4u los_v4u_a4 __attribute__((aligned(4)));

template <typename T>
__device__ __forceinline__ float bits16_to_f(uint32_t h) {
  return to_f<T>(__builtin_bit_cast(T, (unsigned short)h));
}
template <typename T>
__device__ __forceinline__ uint32_t f_to_bits16(float x) {
  return (uint32_t)__builtin_bit_cast(unsigned short, from_f<T>(x));
}

// 8 consecutive scores as f32
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const los_v4u a = *reinterpret_cast<const los_v4u_a4*>(p);
    const los_v4u b = *reinterpret_cast<const los_v4u_a4*>(p + 4);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      x[q] = __uint_as_float(a[q]);
      x[q + 4] = __uint_as_float(b[q]);
    }
  } else {
    const los_v4u a = *reinterpret_cast<const los_v4u_a2*>(p);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      x[2 * q] = bits16_to_f<T>(a[q] & 0xFFFFu);
      x[2 * q + 1] = bits16_to_f<T>(a[q] >> 16);
    }
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    los_v4u a, b;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      a[q] = __float_as_uint(x[q]);
      b[q] = __float_as_uint(x[q + 4]);
    }
    *reinterpret_cast<los_v4u_a4*>(p) = a;
    *reinterpret_cast<los_v4u_a4*>(p + 4) = b;
  } else {
    los_v4u a;
#pragma unroll
    for (int q = 0; q < 4; ++q) a[q] = f_to_bits16<T>(x[2 * q]) | (f_to_bits16<T>(x[2 * q + 1]) << 16);
    *reinterpret_cast<los_v4u_a2*>(p) = a;
  }
}

// One row's scores and rules, uniform over the workgroup.
template <typename T>
struct Row {
  const T* s;
  const uint32_t* bits;
  const uint32_t* uni;
  RowSel sel;
  bool masked;
};

template <typename T>
__device__ __forceinline__ Row<T> open_row(const Rows& R, uint32_t n) {
  Row<T> r;
  const uint32_t o = n / R.inner, i = n - o * R.inner;
  r.s = reinterpret_cast<const T*>(R.scores) + (uint64_t)o * R.ld_outer + (uint64_t)i * R.ld;
  r.bits = R.bits ? R.bits + (uint64_t)n * R.ldb : nullptr;
  r.uni = R.uni;
  RowParams p;
  if (R.rp) {
    p = R.rp[n];
    if (!r.bits) p.flags &= ~kUseBits;
    if (!r.uni) p.flags &= ~kUnigram;
  } else {                              // the allowed bits alone: a hard mask
    p.base = r.bits ? -INFINITY : 0.f;
    p.v_dist = p.v_uni = p.v_eos = 0.f;
    p.flags = r.bits ? kUseBits : 0u;
    p.special = -1;
  }
  r.sel = row_sel(p, R.V, R.eos);
  r.masked = p.flags != 0 || p.base != 0.f;
  return r;
}

// s + v in f32, rounded to T; -inf when the mask value forbids the token
// (whatever its score, NaN and inf included)
template <typename T>
__device__ __forceinline__ float masked_score(float s, float v) {
  float z = s + v;
  if constexpr (sizeof(T) == 2) z = to_f<T>(from_f<T>(z));
  return v == -INFINITY ? -INFINITY : z;
}

// the scores of chunk j (tokens 8 j .. 8 j + cnt - 1) under the mask; -inf past cnt
template <typename T>
__device__ __forceinline__ void chunk_z(const Row<T>& r, uint32_t j, uint32_t cnt, float (&z)[8]) {
  if (cnt == 8) {
    load8<T>(r.s + 8 * j, z);
  } else {
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q) z[q] = q < cnt ? to_f<T>(r.s[8 * j + q]) : -INFINITY;
  }
  if (r.masked) {
    uint32_t H, L;
    chunk_codes(r.sel, j, r.sel.dm ? r.bits[j >> 2] : 0u, r.sel.um ? r.uni[j >> 2] : 0u, H, L);
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q) {
      const float v = mask_at(r.sel, H, L, q);
      z[q] = q < cnt ? masked_score<T>(z[q], v) : -INFINITY;
    }
  }
}

// z of one token
template <typename T>
__device__ __forceinline__ float token_z(const Row<T>& r, uint32_t t) {
  const float s = to_f<T>(r.s[t]);
  if (!r.masked) return s;
  uint32_t H, L;
  chunk_codes(r.sel, t >> 3, r.sel.dm ? r.bits[t >> 5] : 0u, r.sel.um ? r.uni[t >> 5] : 0u, H, L);
  return masked_score<T>(s, mask_at(r.sel, H, L, t & 7));
}

// running (maximum, sum of exp2((z - maximum) k))
struct MaxSum {
  float m, s;
};

__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b, float k) {
  MaxSum c;
  c.m = fmaxf(a.m, b.m);
  c.s = a.s * exp2f((a.m - c.m) * k) + b.s * exp2f((b.m - c.m) * k);
  return c;
}

__device__ __forceinline__ void add8(MaxSum& a, const float (&z)[8], float k) {
  float m = a.m;
#pragma unroll
  for (int q = 0; q < 8; ++q) m = fmaxf(m, z[q]);
  float s = a.s * exp2f((a.m - m) * k);
#pragma unroll
  for (int q = 0; q < 8; ++q) s += exp2f((z[q] - m) * k);
  a.m = m;
  a.s = s;
}

template <int kThreads>
__device__ MaxSum block_join(MaxSum a, float k, MaxSum* sh) {
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    MaxSum b;
    b.m = __shfl_xor(a.m, d);
    b.s = __shfl_xor(a.s, d);
    a = join(a, b, k);
  }
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) sh[w] = a;
  __syncthreads();
  MaxSum t = sh[0];
#pragma unroll
  for (int i = 1; i < kThreads / 64; ++i) t = join(t, sh[i], k);
  return t;
}

// Workgroup (slice, row): the slice's maximum and sum.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) k_part(Rows R, uint32_t S, MaxSum* __restrict__ parts) {
  __shared__ MaxSum sh[kRowThreads / 64];
  const uint32_t n = blockIdx.x / S, sl = blockIdx.x - n * S;
  const Row<T> r = open_row<T>(R, n);
  const uint32_t chunks = (R.V + 7) / 8;
  const uint32_t per = (chunks + S - 1) / S;
  const uint32_t c0 = sl * per, c1 = min(chunks, c0 + per);
  MaxSum a{-FLT_MAX, 0.f};
  for (uint32_t j = c0 + threadIdx.x; j < c1; j += kRowThreads) {
    float z[8];
    chunk_z<T>(r, j, min(8u, R.V - 8 * j), z);
    add8(a, z, R.k);
  }
  a = block_join<kRowThreads>(a, R.k, sh);
  if (threadIdx.x == 0) parts[(uint64_t)n * S + sl] = a;
}

// A row's log-probability from its maximum and sum, in f64, and what the
// gradient needs: {m, -log2(sum)}, or {0, +inf} for a row that has none.
struct RowStat {
  float m, nls;
};

__device__ __forceinline__ double row_logp(int64_t tok, uint32_t V, float za, MaxSum a, double inv_t, RowStat& st) {
  st = RowStat{0.f, INFINITY};
  if (tok < 0 || tok >= (int64_t)V) return 0.0;
  if (za == -INFINITY) return -INFINITY;
  const double ls = log((double)a.s);
  st.m = a.m;
  st.nls = (float)(-ls * 1.4426950408889634);
  return ((double)za - (double)a.m) * inv_t - ls;
}

// One thread per row: the S parts joined in slice order.
template <typename T>
__global__ void __launch_bounds__(64) k_finish(Rows R, uint32_t S, const MaxSum* __restrict__ parts,
                                               float* __restrict__ logp, double* __restrict__ logp64,
                                               RowStat* __restrict__ stats) {
  const uint32_t n = blockIdx.x * 64 + threadIdx.x;
  if (n >= R.N) return;
  MaxSum a = parts[(uint64_t)n * S];
  for (uint32_t i = 1; i < S; ++i) a = join(a, parts[(uint64_t)n * S + i], R.k);
  const int64_t tok = R.tokens[n];
  const bool in = tok >= 0 && tok < (int64_t)R.V;
  const float za = in ? token_z<T>(open_row<T>(R, n), (uint32_t)tok) : 0.f;
  RowStat st;
  const double lp = row_logp(tok, R.V, za, a, R.inv_t64, st);
  if (logp) logp[n] = (float)lp;
  if (logp64) logp64[n] = lp;
  if (stats) stats[n] = st;
}

// ds_t = c (1[t = a] - exp2((z_t - m) k - log2 sum)), c = coef[n] * scale / T.
// Workgroup (slice, row).
template <typename T>
__global__ void __launch_bounds__(kRowThreads) k_grad(Rows R, uint32_t S, const RowStat* __restrict__ stats,
                                                      const float* __restrict__ coef, const float* __restrict__ scale,
                                                      T* __restrict__ out, uint64_t ldo) {
  const uint32_t n = blockIdx.x / S, sl = blockIdx.x - n * S;
  const uint32_t chunks = (R.V + 7) / 8;
  const uint32_t per = (chunks + S - 1) / S;
  const uint32_t c0 = sl * per, c1 = min(chunks, c0 + per);
  const RowStat st = stats[n];
  const float c = st.nls == INFINITY ? 0.f : coef[n] * (scale ? *scale : 1.f) * R.inv_t;
  const Row<T> r = open_row<T>(R, n);
  T* o = out + (uint64_t)n * ldo;
  const int64_t tok = R.tokens[n];
  const uint32_t ja = c != 0.f ? (uint32_t)((uint64_t)tok >> 3) : ~0u, qa = (uint32_t)tok & 7u;
  for (uint32_t j = c0 + threadIdx.x; j < c1; j += kRowThreads) {
    const uint32_t cnt = min(8u, R.V - 8 * j);
    float z[8];
    if (c == 0.f) {
#pragma unroll
      for (int q = 0; q < 8; ++q) z[q] = 0.f;
    } else {
      chunk_z<T>(r, j, cnt, z);
#pragma unroll
      for (uint32_t q = 0; q < 8; ++q) {
        z[q] = -c * exp2f(fmaf(z[q] - st.m, R.k, st.nls));
        if (j == ja && q == qa) z[q] += c;
      }
    }
    if (cnt == 8) {
      store8<T>(o + 8 * j, z);
    } else {
      for (uint32_t q = 0; q < cnt; ++q) o[8 * j + q] = from_f<T>(z[q]);
    }
  }
}

// ---- the losses: one workgroup, sums in f64 in a fixed order -----------------

__device__ double block_sum64(double x, double* sh) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
  __syncthreads();
  double t = 0;
  for (uint32_t i = 0; i < blockDim.x / 64; ++i) t += sh[i];
  return t;
}

struct PolicyIn {
  const float *old_logp, *ref_logp, *adv, *weights;
  double lo, hi, kl;     // 1 - clip_low, 1 + clip_high, the KL coefficient
  double w;              // every position's weight when weights is null
};

// One position's loss and its derivative by logp:
//   r = exp(logp - old), pg = -min(r A, clip(r) A), kl = e^d - d - 1 with d = ref - logp
//   d pg = -r A where r A is the smaller (or equal) one, else 0; d kl = 1 - e^d
__device__ __forceinline__ double policy_term(const PolicyIn& P, uint32_t n, double lp, bool live, float& coef) {
  const double w = P.weights ? (double)P.weights[n] : P.w;
  coef = 0.f;
  if (!live || w == 0.0) return 0.0;
  const double A = P.adv[n];
  const double r = exp(lp - (double)P.old_logp[n]);
  const double a = r * A, b = fmin(fmax(r, P.lo), P.hi) * A;
  double l = A == 0.0 ? 0.0 : (a <= b ? -a : -b);
  double g = A != 0.0 && a <= b ? -a : 0.0;
  if (P.kl != 0.0) {
    const double d = (double)P.ref_logp[n] - lp, e = exp(d);
    l += P.kl * (expm1(d) - d);
    g += P.kl * (1.0 - e);
  }
  coef = (float)(w * g);
  return w * l;
}

__global__ void __launch_bounds__(kOneThreads) k_policy(uint32_t N, PolicyIn P, const double* __restrict__ logp,
                                                        const RowStat* __restrict__ stats,
                                                        float* __restrict__ coef, float* __restrict__ loss) {
  __shared__ double sh[kOneThreads / 64];
  double sum = 0;
  for (uint32_t n = threadIdx.x; n < N; n += kOneThreads) {
    float c;
    sum += policy_term(P, n, logp[n], stats[n].nls != INFINITY, c);
    coef[n] = c;
  }
  sum = block_sum64(sum, sh);
  if (threadIdx.x == 0) *loss = (float)sum;
}

struct PreferenceIn {
  const int64_t* cu;             // 2 P + 1 row bounds; sequence 2 i is pair i's preferred one
  const float *weights, *ref;    // either may be null (1, 0)
  uint32_t pairs;
  double beta, ls, margin;
};

__device__ __forceinline__ double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }

// Waves take sequences: their weighted sums; threads take pairs: loss and
// slope; waves write every row's coefficient.  ws: 2 P sums + P slopes, f64.
__global__ void __launch_bounds__(kOneThreads) k_preference(uint32_t N, PreferenceIn P,
                                                            const double* __restrict__ logp,
                                                            const RowStat* __restrict__ stats, double* ws,
                                                            float* __restrict__ seq_logp, float* __restrict__ coef,
                                                            float* __restrict__ loss) {
  __shared__ double sh[kOneThreads / 64];
  double* sums = ws;
  double* slope = ws + 2 * (uint64_t)P.pairs;
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63, waves = kOneThreads / 64;
  const uint32_t Q = 2 * P.pairs;
  for (uint32_t n = threadIdx.x; n < N; n += kOneThreads) coef[n] = 0.f;
  for (uint32_t q = wave; q < Q; q += waves) {
    const int64_t b = min(max(P.cu[q], (int64_t)0), (int64_t)N), e = min(max(P.cu[q + 1], b), (int64_t)N);
    double s = 0;
    for (int64_t n = b + lane; n < e; n += 64) {
      const double w = P.weights ? (double)P.weights[n] : 1.0;
      if (w != 0.0 && stats[n].nls != INFINITY) s += w * logp[n];
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    if (lane == 0) {
      sums[q] = s;
      seq_logp[q] = (float)s;
    }
  }
  __syncthreads();
  double total = 0;
  for (uint32_t i = threadIdx.x; i < P.pairs; i += kOneThreads) {
    const double a = sums[2 * i] - (P.ref ? (double)P.ref[2 * i] : 0.0);
    const double b = sums[2 * i + 1] - (P.ref ? (double)P.ref[2 * i + 1] : 0.0);
    const double D = P.beta * (a - b) - P.margin;
    total += (1.0 - P.ls) * softplus(-D) + P.ls * softplus(D);
    slope[i] = P.beta / P.pairs * (1.0 / (1.0 + exp(-D)) - 1.0 + P.ls);
  }
  total = block_sum64(total, sh);       // its barriers also publish slope
  if (threadIdx.x == 0) *loss = P.pairs ? (float)(total / P.pairs) : 0.f;
  for (uint32_t q = wave; q < Q; q += waves) {
    const int64_t b = min(max(P.cu[q], (int64_t)0), (int64_t)N), e = min(max(P.cu[q + 1], b), (int64_t)N);
    const double g = (q & 1) ? -slope[q >> 1] : slope[q >> 1];
    for (int64_t n = b + lane; n < e; n += 64) {
      const double w = P.weights ? (double)P.weights[n] : 1.0;
      if (w != 0.0 && stats[n].nls != INFINITY) coef[n] = (float)(w * g);
    }
  }
}

// ---- launch ----------------------------------------------------------------

// Slices per row: enough workgroups to fill the chip, none below 512 tokens.
uint32_t slices(uint64_t N, uint64_t V) {
  const uint64_t want = (2048 + N - 1) / N;
  const uint64_t most = (V + 511) / 512;
  return (uint32_t)std::max<uint64_t>(1, std::min({want, most, (uint64_t)256}));
}

uint64_t up16(uint64_t x) { return (x + 15) & ~(uint64_t)15; }

struct Layout {            // the workspace: slice parts, f64 log-probabilities, preference sums
  uint64_t parts, logp, pref, bytes;
};
Layout layout(uint64_t N, uint64_t V, uint64_t pairs) {
  Layout l;
  l.parts = 0;
  l.logp = up16(N * slices(std::max<uint64_t>(N, 1), V) * sizeof(MaxSum));
  l.pref = l.logp + up16(N * 8);
  l.bytes = l.pref + up16(pairs * 24);
  return l;
}

int as_rows(const fm_score_rows* a, Rows& R) {
  if (!a) {
    set_error("score rows: null");
    return -1;
  }
  if (a->dtype < 0 || a->dtype > 2) {
    set_error("unsupported scores dtype code %d", a->dtype);
    return -1;
  }
  if (a->N >= (1ull << 22) || a->V == 0 || a->V > (1ull << 30)) {
    set_error("score rows: N = %llu, V = %llu out of range (N < 2^22, 1 <= V <= 2^30)", (unsigned long long)a->N,
              (unsigned long long)a->V);
    return -1;
  }
  const double k = 1.4426950408889634 / a->temperature;
  if (!(a->temperature > 0) || !std::isfinite(a->temperature) || !(k <= 1e30) || !(k >= 1e-30)) {
    set_error("score rows: temperature %g must be positive, between 1e-30 and 1e30", a->temperature);
    return -1;
  }
  if (a->inner == 0 || a->inner > (1ull << 31)) {
    set_error("score rows: inner = %llu rows per outer stride", (unsigned long long)a->inner);
    return -1;
  }
  if (a->d_bits && a->ld_bits < (a->V + 31) / 32) {
    set_error("score rows: ld_bits = %llu words < ceil(V / 32)", (unsigned long long)a->ld_bits);
    return -1;
  }
  if (a->N && (!a->d_scores || !a->d_tokens)) {
    set_error("score rows: null scores or tokens");
    return -1;
  }
  static_assert(sizeof(RowParams) == sizeof(fm_row_params), "row record layout");
  R = Rows{a->d_scores, a->ld_scores, a->ld_outer, (uint32_t)a->inner, (uint32_t)a->N, (uint32_t)a->V, a->d_tokens,
           a->d_bits, a->ld_bits, a->d_unigram_bits, reinterpret_cast<const RowParams*>(a->d_rows), a->eos,
           (float)k, (float)(1.0 / a->temperature), 1.0 / a->temperature};
  return 0;
}

int check_ws(const void* ws, uint64_t have, uint64_t need) {
  if (have >= need && (ws || !need) && (reinterpret_cast<uintptr_t>(ws) & 15) == 0) return 0;
  set_error("score workspace: %llu bytes at a 16-B aligned address needed, %llu given", (unsigned long long)need,
            (unsigned long long)have);
  return -1;
}

// A launch's threads, N * S * 256, stay below 2^32: N < 2^22, and S > 1 only below 2048 rows.
template <typename F>
int by_dtype(int dtype, F f) {
  switch (dtype) {
    case 0: f((float*)nullptr); break;
    case 1: f((__hip_bfloat16*)nullptr); break;
    default: f((__half*)nullptr); break;
  }
  FM_HIP(hipGetLastError());
  return 0;
}

int run_logp(int dtype, const Rows& R, float* logp, double* logp64, RowStat* stats, MaxSum* parts, hipStream_t s) {
  const uint32_t S = slices(R.N, R.V);
  return by_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    k_part<T><<<R.N * S, kRowThreads, 0, s>>>(R, S, parts);
    k_finish<T><<<(R.N + 63) / 64, 64, 0, s>>>(R, S, parts, logp, logp64, stats);
  });
}

int run_grad(int dtype, const Rows& R, const RowStat* stats, const float* coef, const float* scale, void* out,
             uint64_t ldo, hipStream_t s) {
  const uint32_t S = slices(R.N, R.V);
  return by_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    k_grad<T><<<R.N * S, kRowThreads, 0, s>>>(R, S, stats, coef, scale, reinterpret_cast<T*>(out), ldo);
  });
}

}  // namespace

int score_workspace(uint64_t N, uint64_t V, uint64_t pairs, uint64_t* bytes) {
  if (!bytes) {
    set_error("score_workspace: null result");
    return -1;
  }
  *bytes = layout(N, V, pairs).bytes;
  return 0;
}

int token_logprobs(const fm_score_rows* a, float* logp, float* stats, void* ws, uint64_t ws_bytes, hipStream_t s) {
  Rows R;
  if (as_rows(a, R)) return -1;
  if (R.N == 0) return 0;
  const Layout l = layout(R.N, R.V, 0);
  if (check_ws(ws, ws_bytes, l.bytes)) return -1;
  return run_logp(a->dtype, R, logp, nullptr, reinterpret_cast<RowStat*>(stats), reinterpret_cast<MaxSum*>(ws), s);
}

int token_logprobs_grad(const fm_score_rows* a, const float* stats, const float* coef, const float* scale, void* grad,
                        uint64_t ld_grad, hipStream_t s) {
  Rows R;
  if (as_rows(a, R)) return -1;
  if (R.N == 0) return 0;
  if (!stats || !coef || !grad || ld_grad < R.V) {
    set_error("token_logprobs_grad: null buffer, or ld_grad < V");
    return -1;
  }
  return run_grad(a->dtype, R, reinterpret_cast<const RowStat*>(stats), coef, scale, grad, ld_grad, s);
}

int policy_loss(const fm_score_rows* a, const fm_policy_args* p, hipStream_t s) {
  Rows R;
  if (as_rows(a, R)) return -1;
  if (!p || !p->d_loss || (R.N && (!p->d_logp || !p->d_stats || !p->d_coef || !p->d_old_logp || !p->d_advantages))) {
    set_error("policy_loss: null argument");
    return -1;
  }
  if (!(p->clip_low >= 0 && p->clip_low <= 1 && p->clip_high >= 0 && std::isfinite(p->clip_high)) ||
      !std::isfinite(p->kl_coef)) {
    set_error("policy_loss: clip_low must be in [0, 1], clip_high >= 0 and finite, kl_coef finite");
    return -1;
  }
  if (p->kl_coef != 0 && R.N && !p->d_ref_logp) {
    set_error("policy_loss: a KL term needs reference log-probabilities");
    return -1;
  }
  const Layout l = layout(R.N, R.V, 0);
  if (check_ws(p->d_ws, p->ws_bytes, l.bytes)) return -1;
  char* ws = reinterpret_cast<char*>(p->d_ws);
  double* lp = reinterpret_cast<double*>(ws + l.logp);
  RowStat* st = reinterpret_cast<RowStat*>(p->d_stats);
  if (R.N && run_logp(a->dtype, R, p->d_logp, lp, st, reinterpret_cast<MaxSum*>(ws), s)) return -1;
  const PolicyIn in{p->d_old_logp, p->d_ref_logp, p->d_advantages, p->d_weights, 1.0 - p->clip_low, 1.0 + p->clip_high,
                    p->kl_coef, 1.0 / std::max<uint32_t>(R.N, 1)};
  k_policy<<<1, kOneThreads, 0, s>>>(R.N, in, lp, st, p->d_coef, p->d_loss);
  FM_HIP(hipGetLastError());
  return 0;
}

int preference_loss(const fm_score_rows* a, const fm_preference_args* p, hipStream_t s) {
  Rows R;
  if (as_rows(a, R)) return -1;
  if (!p || !p->d_loss || !p->d_cu || (p->pairs && !p->d_seq_logp) || (R.N && (!p->d_stats || !p->d_coef))) {
    set_error("preference_loss: null argument");
    return -1;
  }
  if (p->pairs >= (1ull << 30) || !std::isfinite(p->beta) || !std::isfinite(p->margin) ||
      !(p->label_smoothing >= 0 && p->label_smoothing <= 1)) {
    set_error("preference_loss: pairs < 2^30, beta and margin finite, label_smoothing in [0, 1]");
    return -1;
  }
  const Layout l = layout(R.N, R.V, p->pairs);
  if (check_ws(p->d_ws, p->ws_bytes, l.bytes)) return -1;
  char* ws = reinterpret_cast<char*>(p->d_ws);
  double* lp = reinterpret_cast<double*>(ws + l.logp);
  RowStat* st = reinterpret_cast<RowStat*>(p->d_stats);
  if (R.N && run_logp(a->dtype, R, nullptr, lp, st, reinterpret_cast<MaxSum*>(ws), s)) return -1;
  const PreferenceIn in{p->d_cu, p->d_weights, p->d_ref_logp, (uint32_t)p->pairs, p->beta, p->label_smoothing,
                        p->margin};
  k_preference<<<1, kOneThreads, 0, s>>>(R.N, in, lp, st, reinterpret_cast<double*>(ws + l.pref), p->d_seq_logp,
                                         p->d_coef, p->d_loss);
  FM_HIP(hipGetLastError());
  return 0;
}

}  // namespace fmidx
