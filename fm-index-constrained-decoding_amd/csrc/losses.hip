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

constexpr int kRowThreads = 256;       // few rows: a slice of one row
constexpr int kWholeThreads = 512;     // many rows: a row
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

// One row's scores and rules, uniform over the workgroup.  Its mode picks the
// cheapest form of z; every form gives the same z.
enum Mode : uint32_t {
  kFree,       // no mask: z = s
  kHard,       // every value 0 or -inf: z = s for the tokens of the set
  kSoft,       // every value finite
  kAny         // anything else (-inf beside boosts)
};

template <typename T>
struct Row {
  const T* s;
  const uint32_t* bits;     // null: the row uses none
  const uint32_t* uni;
  RowSel sel;
  Mode mode;
};

template <typename T>
__device__ __forceinline__ Row<T> open_row(const Rows& R, uint32_t n) {
  Row<T> r;
  const uint32_t o = n / R.inner, i = n - o * R.inner;
  r.s = reinterpret_cast<const T*>(R.scores) + (uint64_t)o * R.ld_outer + (uint64_t)i * R.ld;
  RowParams p;
  if (R.rp) {
    p = R.rp[n];
    if (!R.bits) p.flags &= ~kUseBits;
    if (!R.uni) p.flags &= ~kUnigram;
  } else {                              // the allowed bits alone: a hard mask
    p.base = R.bits ? -INFINITY : 0.f;
    p.v_dist = p.v_uni = p.v_eos = 0.f;
    p.flags = R.bits ? kUseBits : 0u;
    p.special = -1;
  }
  r.bits = (p.flags & kUseBits) ? R.bits + (uint64_t)n * R.ldb : nullptr;
  r.uni = (p.flags & kUnigram) ? R.uni : nullptr;
  // values of classes the row does not have count as its base
  const float vd = (p.flags & (kUseBits | kSpecial)) ? p.v_dist : p.base;
  const float vu = (p.flags & kUnigram) ? p.v_uni : p.base;
  const float ve = (p.flags & kEos) ? p.v_eos : p.base;
  const float lo = fminf(fminf(p.base, vd), fminf(vu, ve)), hi = fmaxf(fmaxf(p.base, vd), fmaxf(vu, ve));
  const bool zeros = (vd == 0.f || vd == p.base) && (vu == 0.f || vu == p.base) && (ve == 0.f || ve == p.base);
  // a class at -inf over a base of -inf would join the set below, so kHard wants its classes at 0
  const bool sets = (!(p.flags & (kUseBits | kSpecial)) || p.v_dist == 0.f) &&
                    (!(p.flags & kUnigram) || p.v_uni == 0.f) && (!(p.flags & kEos) || p.v_eos == 0.f);
  r.mode = lo == 0.f && hi == 0.f ? kFree : p.base == -INFINITY && zeros && sets ? kHard : lo > -INFINITY ? kSoft : kAny;
  r.sel = row_sel(p, R.V, R.eos);
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

// z of one token
template <typename T>
__device__ __forceinline__ float token_z(const Row<T>& r, uint32_t t) {
  const float s = to_f<T>(r.s[t]);
  if (r.mode == kFree) return s;
  uint32_t H, L;
  chunk_codes(r.sel, t >> 3, r.bits ? r.bits[t >> 5] : 0u, r.uni ? r.uni[t >> 5] : 0u, H, L);
  return masked_score<T>(s, mask_at(r.sel, H, L, t & 7));
}

// z of chunk j's 8 tokens (kFree, kSoft, kAny: x = their scores)
template <typename T, Mode M>
__device__ __forceinline__ void chunk_z(const Row<T>& r, uint32_t j, uint32_t dw, uint32_t uw, float (&x)[8]) {
  if constexpr (M == kFree) return;
  uint32_t H, L;
  if (M == kSoft && j != r.sel.je && j != r.sel.js) {      // three values: two selects
    H = (dw >> ((8 * j) & 31u)) & r.sel.dm;
    L = (uw >> ((8 * j) & 31u)) & r.sel.um;
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q) {
      const uint32_t v = bit_sel(bit_mask(H, q), r.sel.fd, bit_sel(bit_mask(L, q), r.sel.fu, r.sel.fb));
      x[q] += __uint_as_float(v);
    }
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (uint32_t q = 0; q < 8; ++q) x[q] = to_f<T>(from_f<T>(x[q]));
    }
  } else {
    chunk_codes(r.sel, j, dw, uw, H, L);
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q) x[q] = masked_score<T>(x[q], mask_at(r.sel, H, L, q));
  }
}

// the tokens of a kHard row's set among 32 w .. 32 w + 31
template <typename T>
__device__ __forceinline__ uint32_t hard_word(const Row<T>& r, uint32_t w) {
  uint32_t x = (r.bits ? r.bits[w] : 0u) | (r.uni ? r.uni[w] : 0u);
  if (w == r.sel.je >> 2) x |= r.sel.eb << (8 * (r.sel.je & 3));
  if (w == r.sel.js >> 2) x |= r.sel.sb << (8 * (r.sel.js & 3));
  return x;
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

// Adds kN values.  The exponents are taken against the whole number n nearest
// to m k, which a fused multiply-add subtracts without a rounding of its own
// (one instruction less per value than (z - m) k); the sum moves to m at the
// end.  Where m k has no such neighbour (rows of the lowest values, extreme
// temperatures) the difference is taken first.
template <int kN>
__device__ __forceinline__ void add_values(MaxSum& a, const float (&z)[kN], float k) {
  float m = a.m;
#pragma unroll
  for (int q = 0; q < kN; ++q) m = fmaxf(m, z[q]);
  const float mk = m * k;
  float t = 0.f;
  if (fabsf(mk) < 1e30f) {
    const float n = rintf(mk);
#pragma unroll
    for (int q = 0; q < kN; ++q) t += __builtin_amdgcn_exp2f(fmaf(z[q], k, -n));
    t *= __builtin_amdgcn_exp2f(fmaf(-m, k, n));
  } else {
#pragma unroll
    for (int q = 0; q < kN; ++q) t += __builtin_amdgcn_exp2f((z[q] - m) * k);
  }
  a.s = a.s * __builtin_amdgcn_exp2f((a.m - m) * k) + t;
  a.m = m;
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

// A wave takes a row in segments of 2048 tokens: 4 chunks of 8 tokens per lane,
// 64 chunks apart, so every access is 1 KB (16-bit) of one row per instruction;
// or one 32-token word of the set per lane.
constexpr uint32_t kSeg = 2048;
// Up to this many tokens in every lane's word, a kHard segment is walked token
// by token; with more, chunk by chunk.
constexpr int kSparse = 4;

template <typename T, Mode M>
__device__ __forceinline__ void scan_chunks(const Row<T>& r, uint32_t V, uint32_t seg, uint32_t lane, float k,
                                            MaxSum& a) {
  const uint32_t j0 = seg * (kSeg / 8) + lane;
  if ((seg + 1) * kSeg <= V) {
    float z[32];
    float x[4][8];
    uint32_t dw[4], uw[4];
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      const uint32_t j = j0 + 64 * u;
      if (M != kFree) {
        dw[u] = r.bits ? r.bits[j >> 2] : 0u;
        uw[u] = r.uni ? r.uni[j >> 2] : 0u;
      }
      load8<T>(r.s + 8 * j, x[u]);
    }
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      chunk_z<T, M>(r, j0 + 64 * u, dw[u], uw[u], x[u]);
#pragma unroll
      for (uint32_t q = 0; q < 8; ++q) z[8 * u + q] = x[u][q];
    }
    add_values(a, z, k);
  } else {                               // the row's end
    for (uint32_t j = j0; 8 * j < V && j < (seg + 1) * (kSeg / 8); j += 64) {
      float x[8];
      if (8 * j + 8 <= V) {
        load8<T>(r.s + 8 * j, x);
      } else {
#pragma unroll
        for (uint32_t q = 0; q < 8; ++q) x[q] = 8 * j + q < V ? to_f<T>(r.s[8 * j + q]) : -INFINITY;
      }
      chunk_z<T, M>(r, j, r.bits ? r.bits[j >> 2] : 0u, r.uni ? r.uni[j >> 2] : 0u, x);
      if (8 * j + 8 > V) {
#pragma unroll
        for (uint32_t q = 0; q < 8; ++q)
          if (8 * j + q >= V) x[q] = -INFINITY;
      }
      add_values(a, x, k);
    }
  }
}

template <typename T>
__device__ __forceinline__ void scan_hard(const Row<T>& r, uint32_t V, uint32_t seg, uint32_t lane, float k,
                                          MaxSum& a) {
  const uint32_t w = seg * 64 + lane;
  uint32_t x = 32 * w < V ? hard_word(r, w) : 0u;
  if (32 * w < V && V - 32 * w < 32) x &= (1u << (V - 32 * w)) - 1;       // the last word's spare bits
  if (__any(__popc(x) > kSparse)) {
    for (uint32_t u = 0; u < 4; ++u) {
      const uint32_t j = seg * (kSeg / 8) + 64 * u + lane;
      const uint32_t h = (uint32_t)__shfl((int)x, 16 * u + (lane >> 2)) >> (8 * (lane & 3)) & 0xFFu;
      if (!h) continue;
      float z[8];
      if (8 * j + 8 <= V) {
        load8<T>(r.s + 8 * j, z);
      } else {
#pragma unroll
        for (uint32_t q = 0; q < 8; ++q) z[q] = 8 * j + q < V ? to_f<T>(r.s[8 * j + q]) : 0.f;
      }
#pragma unroll
      for (uint32_t q = 0; q < 8; ++q)
        z[q] = __uint_as_float(bit_sel(bit_mask(h, q), __float_as_uint(z[q]), 0xFF800000u));
      add_values(a, z, k);
    }
  } else {
    while (x) {
      const float z[1] = {to_f<T>(r.s[32 * w + __ffs((int)x) - 1])};
      x &= x - 1;
      add_values(a, z, k);
    }
  }
}

// the row's segments s0 + wave, s0 + wave + waves, ... below s1
template <typename T>
__device__ __forceinline__ MaxSum scan_row(const Row<T>& r, uint32_t V, uint32_t s0, uint32_t s1, uint32_t waves,
                                           float k) {
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t first = s0 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  MaxSum a{-FLT_MAX, 0.f};
  switch (r.mode) {
    case kFree:
      for (uint32_t s = first; s < s1; s += waves) scan_chunks<T, kFree>(r, V, s, lane, k, a);
      break;
    case kHard:
      for (uint32_t s = first; s < s1; s += waves) scan_hard<T>(r, V, s, lane, k, a);
      break;
    case kSoft:
      for (uint32_t s = first; s < s1; s += waves) scan_chunks<T, kSoft>(r, V, s, lane, k, a);
      break;
    default:
      for (uint32_t s = first; s < s1; s += waves) scan_chunks<T, kAny>(r, V, s, lane, k, a);
  }
  return a;
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

template <typename T>
__device__ __forceinline__ double row_logp(const Rows& R, uint32_t n, const Row<T>& r, MaxSum a, RowStat& st) {
  const int64_t tok = R.tokens[n];
  const bool in = tok >= 0 && tok < (int64_t)R.V;
  return row_logp(tok, R.V, in ? token_z<T>(r, (uint32_t)tok) : 0.f, a, R.inv_t64, st);
}

// What the passes over rows leave: either may be null.
struct RowOut {
  float* logp;
  double* logp64;
  RowStat* stats;
};

__device__ __forceinline__ void put_row(const RowOut& o, uint32_t n, double lp, RowStat st) {
  if (o.logp) o.logp[n] = (float)lp;
  if (o.logp64) o.logp64[n] = lp;
  if (o.stats) o.stats[n] = st;
}

// Few rows: workgroup (slice, row) leaves its slice's maximum and sum.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) k_part(Rows R, uint32_t S, uint32_t per, MaxSum* __restrict__ parts) {
  __shared__ MaxSum sh[kRowThreads / 64];
  const uint32_t n = blockIdx.x / S, sl = blockIdx.x - n * S;
  const Row<T> r = open_row<T>(R, n);
  const uint32_t segs = (R.V + kSeg - 1) / kSeg;
  MaxSum a = scan_row<T>(r, R.V, sl * per, min(segs, (sl + 1) * per), kRowThreads / 64, R.k);
  a = block_join<kRowThreads>(a, R.k, sh);
  if (threadIdx.x == 0) parts[(uint64_t)n * S + sl] = a;
}

// its S parts joined in slice order
template <typename T>
__device__ __forceinline__ double finish_row(const Rows& R, uint32_t n, uint32_t S, const MaxSum* parts, RowStat& st) {
  MaxSum a = parts[(uint64_t)n * S];
  for (uint32_t i = 1; i < S; ++i) a = join(a, parts[(uint64_t)n * S + i], R.k);
  return row_logp<T>(R, n, open_row<T>(R, n), a, st);
}

template <typename T>
__global__ void __launch_bounds__(64) k_finish(Rows R, uint32_t S, const MaxSum* __restrict__ parts, RowOut o) {
  const uint32_t n = blockIdx.x * 64 + threadIdx.x;
  if (n >= R.N) return;
  RowStat st;
  const double lp = finish_row<T>(R, n, S, parts, st);
  put_row(o, n, lp, st);
}

// Many rows: a workgroup each.
template <typename T>
__global__ void __launch_bounds__(kWholeThreads) k_row(Rows R, RowOut o) {
  __shared__ MaxSum sh[kWholeThreads / 64];
  const uint32_t n = blockIdx.x;
  const Row<T> r = open_row<T>(R, n);
  MaxSum a = scan_row<T>(r, R.V, 0, (R.V + kSeg - 1) / kSeg, kWholeThreads / 64, R.k);
  a = block_join<kWholeThreads>(a, R.k, sh);
  if (threadIdx.x == 0) {
    RowStat st;
    const double lp = row_logp<T>(R, n, r, a, st);
    put_row(o, n, lp, st);
  }
}

// ---- the gradient: ds_t = c (1[t = a] - exp2((z_t - m) k - log2 sum)) --------

struct GradRow {
  float c, m, nls, k;
  uint32_t a;             // the token
};

__device__ __forceinline__ float grad_at(const GradRow& g, float z, uint32_t t) {
  const float v = -g.c * exp2f(fmaf(z - g.m, g.k, g.nls));
  return t == g.a ? v + g.c : v;
}

// 8 of them at chunk j
__device__ __forceinline__ void grad8(const GradRow& g, uint32_t j, float (&z)[8]) {
#pragma unroll
  for (uint32_t q = 0; q < 8; ++q) z[q] = -g.c * exp2f(fmaf(z[q] - g.m, g.k, g.nls));
  if (j == g.a >> 3) {
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q)
      if (q == (g.a & 7u)) z[q] += g.c;
  }
}

template <typename T>
__device__ __forceinline__ void store_chunk(T* o, uint32_t j, uint32_t V, const float (&x)[8]) {
  if (8 * j + 8 <= V) {
    store8<T>(o + 8 * j, x);
  } else {
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q)
      if (8 * j + q < V) o[8 * j + q] = from_f<T>(x[q]);
  }
}

template <typename T>
__device__ __forceinline__ void zero_segment(T* o, uint32_t V, uint32_t seg, uint32_t lane) {
  const float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (uint32_t u = 0; u < 4; ++u) {
    const uint32_t j = seg * (kSeg / 8) + 64 * u + lane;
    if (8 * j < V) store_chunk<T>(o, j, V, x);
  }
}

template <typename T, Mode M>
__device__ __forceinline__ void grad_chunks(const Row<T>& r, const GradRow& g, T* o, uint32_t V, uint32_t seg,
                                            uint32_t lane) {
  const uint32_t j0 = seg * (kSeg / 8) + lane;
  if ((seg + 1) * kSeg <= V) {
    float x[4][8];
    uint32_t dw[4], uw[4];
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      const uint32_t j = j0 + 64 * u;
      if (M != kFree) {
        dw[u] = r.bits ? r.bits[j >> 2] : 0u;
        uw[u] = r.uni ? r.uni[j >> 2] : 0u;
      }
      load8<T>(r.s + 8 * j, x[u]);
    }
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      const uint32_t j = j0 + 64 * u;
      chunk_z<T, M>(r, j, dw[u], uw[u], x[u]);
      grad8(g, j, x[u]);
      store8<T>(o + 8 * j, x[u]);
    }
  } else {
    for (uint32_t j = j0; 8 * j < V && j < (seg + 1) * (kSeg / 8); j += 64) {
      float x[8];
      if (8 * j + 8 <= V) {
        load8<T>(r.s + 8 * j, x);
      } else {
#pragma unroll
        for (uint32_t q = 0; q < 8; ++q) x[q] = 8 * j + q < V ? to_f<T>(r.s[8 * j + q]) : 0.f;
      }
      chunk_z<T, M>(r, j, r.bits ? r.bits[j >> 2] : 0u, r.uni ? r.uni[j >> 2] : 0u, x);
      grad8(g, j, x);
      store_chunk<T>(o, j, V, x);
    }
  }
}

// A sparse kHard segment is put together in the wave's own LDS (zeros, then the
// few values at their tokens) and leaves it in whole 16-B stores.
template <typename T>
__device__ __forceinline__ void grad_hard(const Row<T>& r, const GradRow& g, T* o, uint32_t V, uint32_t seg,
                                          uint32_t lane, T* stage) {
  const uint32_t w = seg * 64 + lane;
  uint32_t x = 32 * w < V ? hard_word(r, w) : 0u;
  if (32 * w < V && V - 32 * w < 32) x &= (1u << (V - 32 * w)) - 1;
  if (!__any(x != 0)) {
    zero_segment<T>(o, V, seg, lane);
  } else if (__any(__popc(x) > kSparse)) {
    for (uint32_t u = 0; u < 4; ++u) {
      const uint32_t j = seg * (kSeg / 8) + 64 * u + lane;
      const uint32_t h = (uint32_t)__shfl((int)x, 16 * u + (lane >> 2)) >> (8 * (lane & 3)) & 0xFFu;
      if (8 * j >= V) continue;
      float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (h) {
        if (8 * j + 8 <= V) {
          load8<T>(r.s + 8 * j, z);
        } else {
#pragma unroll
          for (uint32_t q = 0; q < 8; ++q) z[q] = 8 * j + q < V ? to_f<T>(r.s[8 * j + q]) : 0.f;
        }
        grad8(g, j, z);
#pragma unroll
        for (uint32_t q = 0; q < 8; ++q)
          z[q] = __uint_as_float(__float_as_uint(z[q]) & bit_mask(h, q));     // NaN of an out token included
      }
      store_chunk<T>(o, j, V, z);
    }
  } else {
    const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) store8<T>(stage + 8 * (64 * u + lane), zero);
    __syncwarp();
    while (x) {
      const uint32_t t = 32 * w + __ffs((int)x) - 1;
      x &= x - 1;
      stage[t - seg * kSeg] = from_f<T>(grad_at(g, to_f<T>(r.s[t]), t));
    }
    __syncwarp();
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      const uint32_t j = seg * (kSeg / 8) + 64 * u + lane;
      float z[8];
      load8<T>(stage + 8 * (64 * u + lane), z);
      if (8 * j < V) store_chunk<T>(o, j, V, z);
    }
    __syncwarp();
  }
}

// the row's segments s0 + wave, s0 + wave + waves, ... below s1
template <typename T>
__device__ __forceinline__ void grad_row(const Row<T>& r, const GradRow& g, T* o, uint32_t V, uint32_t s0, uint32_t s1,
                                         uint32_t waves, T* stage) {
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  stage += wave * kSeg;
  if (g.c == 0.f) {
    for (uint32_t s = s0 + wave; s < s1; s += waves) zero_segment<T>(o, V, s, lane);
    return;
  }
  switch (r.mode) {
    case kFree:
      for (uint32_t s = s0 + wave; s < s1; s += waves) grad_chunks<T, kFree>(r, g, o, V, s, lane);
      break;
    case kHard:
      for (uint32_t s = s0 + wave; s < s1; s += waves) grad_hard<T>(r, g, o, V, s, lane, stage);
      break;
    case kSoft:
      for (uint32_t s = s0 + wave; s < s1; s += waves) grad_chunks<T, kSoft>(r, g, o, V, s, lane);
      break;
    default:
      for (uint32_t s = s0 + wave; s < s1; s += waves) grad_chunks<T, kAny>(r, g, o, V, s, lane);
  }
}

// Workgroup (slice, row).
template <typename T>
__global__ void __launch_bounds__(kRowThreads) k_grad(Rows R, uint32_t S, uint32_t per,
                                                      const RowStat* __restrict__ stats,
                                                      const float* __restrict__ coef, const float* __restrict__ scale,
                                                      T* __restrict__ out, uint64_t ldo) {
  __shared__ __attribute__((aligned(16))) T stage[kRowThreads / 64 * kSeg];
  const uint32_t n = blockIdx.x / S, sl = blockIdx.x - n * S;
  const RowStat st = stats[n];
  GradRow g;
  g.c = st.nls == INFINITY ? 0.f : coef[n] * (scale ? *scale : 1.f) * R.inv_t;
  g.m = st.m;
  g.nls = st.nls;
  g.k = R.k;
  g.a = (uint32_t)R.tokens[n];
  const uint32_t segs = (R.V + kSeg - 1) / kSeg;
  grad_row<T>(open_row<T>(R, n), g, out + (uint64_t)n * ldo, R.V, sl * per, min(segs, (sl + 1) * per),
              kRowThreads / 64, stage);
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

// How a row is cut.  One workgroup takes a whole row from kManyRows rows on;
// below, slices of at least one segment per wave fill the chip.
constexpr uint64_t kManyRows = 1024;
struct Cut {
  uint32_t S, per;      // slices per row, segments per slice
};
Cut cut(uint64_t N, uint64_t V, uint64_t groups) {
  const uint64_t segs = (V + kSeg - 1) / kSeg, waves = kRowThreads / 64;
  const uint64_t most = (segs + waves - 1) / waves;
  const uint64_t S0 = std::max<uint64_t>(1, std::min(most, groups / std::max<uint64_t>(N, 1)));
  const uint64_t per = (segs + S0 - 1) / S0;
  return Cut{(uint32_t)((segs + per - 1) / per), (uint32_t)per};
}
Cut scan_cut(uint64_t N, uint64_t V) { return cut(N, V, N >= kManyRows ? 0 : 2048); }
Cut grad_cut(uint64_t N, uint64_t V) { return cut(N, V, 8192); }

uint64_t up16(uint64_t x) { return (x + 15) & ~(uint64_t)15; }

struct Layout {            // the workspace: slice parts, f64 log-probabilities, preference sums
  uint64_t parts, logp, pref, bytes;
};
Layout layout(uint64_t N, uint64_t V, uint64_t pairs) {
  Layout l;
  l.parts = 0;
  l.logp = up16(N * scan_cut(N, V).S * sizeof(MaxSum));
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

// A launch's threads stay below 2^32: N < 2^22 rows of 512, or at most 8192 slices of 256 when rows are cut.
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

int run_logp(int dtype, const Rows& R, const RowOut& o, MaxSum* parts, hipStream_t s) {
  const Cut c = scan_cut(R.N, R.V);
  return by_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (R.N >= kManyRows) {
      k_row<T><<<R.N, kWholeThreads, 0, s>>>(R, o);
    } else {
      k_part<T><<<R.N * c.S, kRowThreads, 0, s>>>(R, c.S, c.per, parts);
      k_finish<T><<<(R.N + 63) / 64, 64, 0, s>>>(R, c.S, parts, o);
    }
  });
}

int run_grad(int dtype, const Rows& R, const RowStat* stats, const float* coef, const float* scale, void* out,
             uint64_t ldo, hipStream_t s) {
  const Cut c = grad_cut(R.N, R.V);
  return by_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    k_grad<T><<<R.N * c.S, kRowThreads, 0, s>>>(R, c.S, c.per, stats, coef, scale, reinterpret_cast<T*>(out), ldo);
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
  return run_logp(a->dtype, R, RowOut{logp, nullptr, reinterpret_cast<RowStat*>(stats)}, reinterpret_cast<MaxSum*>(ws),
                  s);
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
  if (R.N && run_logp(a->dtype, R, RowOut{p->d_logp, lp, st}, reinterpret_cast<MaxSum*>(ws), s)) return -1;
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
  if (R.N && run_logp(a->dtype, R, RowOut{nullptr, lp, st}, reinterpret_cast<MaxSum*>(ws), s)) return -1;
  const PreferenceIn in{p->d_cu, p->d_weights, p->d_ref_logp, (uint32_t)p->pairs, p->beta, p->label_smoothing,
                        p->margin};
  k_preference<<<1, kOneThreads, 0, s>>>(R.N, in, lp, st, reinterpret_cast<double*>(ws + l.pref), p->d_seq_logp,
                                         p->d_coef, p->d_loss);
  FM_HIP(hipGetLastError());
  return 0;
}

}  // namespace fmidx
