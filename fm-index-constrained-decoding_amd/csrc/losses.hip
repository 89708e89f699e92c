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
// -FLT_MAX, so a row of nothing but -inf gives a sum of 0 and no NaN.  The sum
// is over the tokens other than a: where a has nearly all of the probability,
// logp = -log1p(rest) and 1 - p_a = -expm1(logp) then keep all their digits,
// which 1 + rest in f32 has lost.
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

// words read by plain global loads wherever the pointer came from
typedef const __attribute__((address_space(1))) uint32_t* Words;

// 8 consecutive scores as they lie in memory, and as f32
template <typename T>
struct Raw8 {
  los_v4u v[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw8<T> raw8(const T* p) {
  Raw8<T> r;
  if constexpr (sizeof(T) == 4) {
    r.v[0] = *reinterpret_cast<const los_v4u_a4*>(p);
    r.v[1] = *reinterpret_cast<const los_v4u_a4*>(p + 4);
  } else {
    r.v[0] = *reinterpret_cast<const los_v4u_a2*>(p);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void widen8(const Raw8<T>& r, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      x[q] = __uint_as_float(r.v[0][q]);
      x[q + 4] = __uint_as_float(r.v[1][q]);
    }
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      x[2 * q] = bits16_to_f<T>(r.v[0][q] & 0xFFFFu);
      x[2 * q + 1] = bits16_to_f<T>(r.v[0][q] >> 16);
    }
  }
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  widen8<T>(raw8<T>(p), x);
}

// Gradients leave by nontemporal stores: they are not read again here, and kept
// in the caches they push out the scores that are (213 us for 240 at 1500 rows
// of 151936 bf16, read twice and written once by k_policy_row).
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    los_v4u a, b;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      a[q] = __float_as_uint(x[q]);
      b[q] = __float_as_uint(x[q + 4]);
    }
    __builtin_nontemporal_store(a, reinterpret_cast<los_v4u_a4*>(p));
    __builtin_nontemporal_store(b, reinterpret_cast<los_v4u_a4*>(p + 4));
  } else {
    los_v4u a;
#pragma unroll
    for (int q = 0; q < 4; ++q) a[q] = pack16<T>(x[2 * q], x[2 * q + 1]);
    __builtin_nontemporal_store(a, reinterpret_cast<los_v4u_a2*>(p));
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
  Words bits_at, uni_at;    // the same, or for none some words of the row itself (never used, but loads
                            // without a branch can be kept in flight)
  RowSel sel;
  Mode mode;
};

template <typename T>
__device__ __forceinline__ Row<T> open_row(const Rows& R, uint32_t n, bool hard = true) {
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
  const uint32_t* any = reinterpret_cast<const uint32_t*>((reinterpret_cast<uintptr_t>(r.s) + 3) & ~(uintptr_t)3);
  r.bits_at = (Words)(r.bits ? r.bits : any);
  r.uni_at = (Words)(r.uni ? r.uni : any);
  // values of classes the row does not have count as its base
  const float vd = (p.flags & (kUseBits | kSpecial)) ? p.v_dist : p.base;
  const float vu = (p.flags & kUnigram) ? p.v_uni : p.base;
  const float ve = (p.flags & kEos) ? p.v_eos : p.base;
  const float lo = fminf(fminf(p.base, vd), fminf(vu, ve)), hi = fmaxf(fmaxf(p.base, vd), fmaxf(vu, ve));
  // kHard: every class the row has is at 0 (one at -inf would join the set below), its base at -inf
  const bool sets = (!(p.flags & (kUseBits | kSpecial)) || p.v_dist == 0.f) &&
                    (!(p.flags & kUnigram) || p.v_uni == 0.f) && (!(p.flags & kEos) || p.v_eos == 0.f);
  r.mode = lo == 0.f && hi == 0.f ? kFree : hard && p.base == -INFINITY && sets ? kHard : lo > -INFINITY ? kSoft : kAny;
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
    for (uint32_t q = 0; q < 8; ++q)
      x[q] += __uint_as_float(pick(sign_bit(H, q), r.sel.fd, pick(sign_bit(L, q), r.sel.fu, r.sel.fb)));
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (uint32_t q = 0; q < 8; q += 2) {
        const uint32_t h = pack16<T>(x[q], x[q + 1]);
        x[q] = bits16_to_f<T>(h & 0xFFFFu);
        x[q + 1] = bits16_to_f<T>(h >> 16);
      }
    }
  } else {
    chunk_codes(r.sel, j, dw, uw, H, L);
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q) x[q] = masked_score<T>(x[q], mask_at(r.sel, H, L, q));
  }
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
// end, by 2^(n - m k), where n is within 1 of m k.  That holds below 2^22, where
// the product's own rounding is under a quarter: from 2^24 on it reaches whole
// numbers, and from 2^32 on 2^(n - m k) overflows.  There (large boosts, rows of
// large negative values, extreme temperatures) the difference is taken first.
template <int kN>
__device__ __forceinline__ void add_values(MaxSum& a, const float (&z)[kN], float k) {
  float m = a.m;
#pragma unroll
  for (int q = 0; q < kN; ++q) m = fmaxf(m, z[q]);
  const float mk = m * k;
  float t = 0.f;
  if (fabsf(mk) < 0x1p22f) {
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
// 64 chunks apart, so every access is 1 KB (16-bit) of one row per instruction.
constexpr uint32_t kSeg = 2048;

// one lane's share of a whole segment, in registers
template <typename T, Mode M>
struct SegLoad {
  Raw8<T> s[4];
  uint32_t dw[4], uw[4];
  __device__ __forceinline__ void load(const Row<T>& r, uint32_t seg, uint32_t lane) {
    const uint32_t j0 = seg * (kSeg / 8) + lane;
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      const uint32_t j = j0 + 64 * u;
      if constexpr (M != kFree) {
        dw[u] = r.bits_at[j >> 2];          // a whole segment's words lie within its row's scores too
        uw[u] = r.uni_at[j >> 2];
      }
      s[u] = raw8<T>(r.s + 8 * j);
    }
  }
  __device__ __forceinline__ void values(const Row<T>& r, uint32_t seg, uint32_t lane, uint32_t u,
                                         float (&x)[8]) const {
    widen8<T>(s[u], x);
    chunk_z<T, M>(r, seg * (kSeg / 8) + 64 * u + lane, M == kFree ? 0u : dw[u], M == kFree ? 0u : uw[u], x);
  }
};

// chunk j of the row's last, partial segment: z, -inf past the row
template <typename T, Mode M>
__device__ __forceinline__ void edge_chunk(const Row<T>& r, uint32_t V, uint32_t j, float (&x)[8]) {
  if (8 * j + 8 <= V) {
    load8<T>(r.s + 8 * j, x);
  } else {
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q) x[q] = 8 * j + q < V ? to_f<T>(r.s[8 * j + q]) : 0.f;
  }
  chunk_z<T, M>(r, j, r.bits ? r.bits[j >> 2] : 0u, r.uni ? r.uni[j >> 2] : 0u, x);
  if (8 * j + 8 > V) {
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q)
      if (8 * j + q >= V) x[q] = -INFINITY;
  }
}

// the row's segments first, first + waves, ... below s1, without token `not_t`;
// the next one's loads are issued before the present one is added up
template <typename T, Mode M>
__device__ __forceinline__ void scan_chunks(const Row<T>& r, uint32_t V, uint32_t first, uint32_t s1, uint32_t waves,
                                            uint32_t lane, float k, uint32_t not_t, MaxSum& a) {
  const uint32_t whole = min(s1, V / kSeg);
  uint32_t s = first;
  if (s < whole) {
    SegLoad<T, M> cur, nxt;
    auto add = [&](const SegLoad<T, M>& l, uint32_t seg) {
      float z[32];
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u) {
        float x[8];
        l.values(r, seg, lane, u, x);
#pragma unroll
        for (uint32_t q = 0; q < 8; ++q) z[8 * u + q] = x[q];
      }
      if (seg == not_t / kSeg && lane == (not_t >> 3 & 63u)) {
#pragma unroll
        for (uint32_t i = 0; i < 32; ++i)
          if (i == ((not_t >> 9 & 3u) << 3 | (not_t & 7u))) z[i] = -INFINITY;
      }
      add_values(a, z, k);
    };
    cur.load(r, s, lane);
    for (; s + waves < whole; s += waves) {
      nxt.load(r, s + waves, lane);
      add(cur, s);
      cur = nxt;
    }
    add(cur, s);
    s += waves;
  }
  if (s < s1) {                          // the row's end
    for (uint32_t j = s * (kSeg / 8) + lane; 8 * j < V && j < (s + 1) * (kSeg / 8); j += 64) {
      float x[8];
      edge_chunk<T, M>(r, V, j, x);
      if (j == not_t >> 3) {
#pragma unroll
        for (uint32_t q = 0; q < 8; ++q)
          if (q == (not_t & 7u)) x[q] = -INFINITY;
      }
      add_values(a, x, k);
    }
  }
}

template <typename T>
__device__ __forceinline__ MaxSum scan_other(const Row<T>& r, uint32_t V, uint32_t first, uint32_t s1, uint32_t waves,
                                             uint32_t lane, float k, uint32_t not_t) {
  MaxSum a{-FLT_MAX, 0.f};
  switch (r.mode) {
    case kFree: scan_chunks<T, kFree>(r, V, first, s1, waves, lane, k, not_t, a); break;
    case kSoft: scan_chunks<T, kSoft>(r, V, first, s1, waves, lane, k, not_t, a); break;
    default: scan_chunks<T, kAny>(r, V, first, s1, waves, lane, k, not_t, a);
  }
  return a;
}

// ---- kHard rows --------------------------------------------------------------
// The set's words of the workgroup's range (32 w0 .. 32 (w0 + nw)) go to LDS in
// one round trip.  Up to kList tokens: their numbers are written to a list (a
// prefix sum of the words' counts), their scores are gathered all at once, one
// per thread, and stay in LDS, so that a gradient made by the same workgroup
// reads nothing again.  More: chunks of 8 that hold a token are read whole.
// Walking the words in registers instead (10 segments per wave, unrolled) took
// 413 us where this takes 298 with its gradient, at 4096 rows of 128256 with about 400 tokens.
constexpr uint32_t kList = 2048;
// The longest range: 6 bytes of LDS per word beside the list's 16 KB, in the 64 KB
// of a launch.  Whole rows past it (245760 tokens) take the general form, which
// reads every score: 8 x 256000 bf16 48 us for 19 at 245760, 2048 rows 318 for 74.
constexpr uint32_t kHardWords = 7680;

struct HardLds {
  uint32_t* word;       // [nw]
  uint32_t* tok;        // [kList] token - 32 w0
  float* val;           // [kList] its score, later its gradient
  uint16_t* before;     // [nw] tokens of the list before the word
  uint32_t* wave_sum;   // [16]
  uint32_t nw, w0, total;
};

__host__ __device__ constexpr uint32_t hard_bytes(uint32_t nw) { return nw * 6 + kList * 8 + 64; }

__device__ __forceinline__ HardLds hard_lds(uint32_t* base, uint32_t w0, uint32_t nw) {
  HardLds h;
  h.wave_sum = base;
  h.tok = base + 16;
  h.val = reinterpret_cast<float*>(h.tok + kList);
  h.word = reinterpret_cast<uint32_t*>(h.val + kList);
  h.before = reinterpret_cast<uint16_t*>(h.word + nw);
  h.nw = nw;
  h.w0 = w0;
  h.total = 0;
  return h;
}

// words and, if they fit, the list; every thread of the workgroup
template <typename T, int kThreads>
__device__ void hard_open(const Row<T>& r, uint32_t V, HardLds& h) {
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  for (uint32_t i = tid; i < h.nw; i += kThreads) {
    const uint32_t w = h.w0 + i;
    uint32_t x = 0;
    if (32 * w < V) {
      x = (r.bits ? r.bits[w] : 0u) | (r.uni ? r.uni[w] : 0u);
      if (w == r.sel.je >> 2) x |= r.sel.eb << (8 * (r.sel.je & 3));
      if (w == r.sel.js >> 2) x |= r.sel.sb << (8 * (r.sel.js & 3));
      if (V - 32 * w < 32) x &= (1u << (V - 32 * w)) - 1;       // the last word's spare bits
    }
    h.word[i] = x;
  }
  __syncthreads();
  const uint32_t per = (h.nw + kThreads - 1) / kThreads;
  const uint32_t i0 = min(h.nw, tid * per), i1 = min(h.nw, i0 + per);
  uint32_t mine = 0;
  for (uint32_t i = i0; i < i1; ++i) mine += __popc(h.word[i]);
  uint32_t upto = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = (uint32_t)__shfl_up((int)upto, d);
    if (lane >= (uint32_t)d) upto += o;
  }
  if (lane == 63) h.wave_sum[tid >> 6] = upto;
  __syncthreads();
  uint32_t at = upto - mine, total = 0;
  for (uint32_t i = 0; i < kThreads / 64; ++i) {
    if (i < tid >> 6) at += h.wave_sum[i];
    total += h.wave_sum[i];
  }
  h.total = total;
  if (total > kList) return;
  for (uint32_t i = i0; i < i1; ++i) {
    h.before[i] = (uint16_t)at;
    for (uint32_t x = h.word[i]; x; x &= x - 1) h.tok[at++] = 32 * i + __ffs((int)x) - 1;
  }
  __syncthreads();
}

// chunk j's (of the range) part of the set, and its scores as they lie in memory
// (0 where no token is in, and past the row)
template <typename T>
__device__ __forceinline__ uint32_t hard_chunk(const Row<T>& r, uint32_t V, const HardLds& h, uint32_t j, Raw8<T>& z) {
  const uint32_t b = h.word[j >> 2] >> (8 * (j & 3)) & 0xFFu, t = 32 * h.w0 + 8 * j;
#pragma unroll
  for (uint32_t q = 0; q < sizeof(T) / 2; ++q) z.v[q] = los_v4u{0, 0, 0, 0};
  if (b) {
    if (t + 8 <= V) {
      z = raw8<T>(r.s + t);
    } else if constexpr (sizeof(T) == 4) {
      for (uint32_t q = 0; t + q < V; ++q) {
        const uint32_t e = __float_as_uint(to_f<T>(r.s[t + q]));
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
          if (i == q) z.v[i >> 2][i & 3] = e;
      }
    } else {
      const unsigned short* p = reinterpret_cast<const unsigned short*>(r.s + t);
      for (uint32_t q = 0; t + q < V; ++q) {
        const uint32_t e = (uint32_t)p[q] << (16 * (q & 1));
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
          if (i == q >> 1) z.v[0][i] |= e;
      }
    }
  }
  return b;
}

template <typename T, int kThreads>
__device__ MaxSum scan_hard(const Row<T>& r, uint32_t V, float k, uint32_t not_t, HardLds& h) {
  MaxSum a{-FLT_MAX, 0.f};
  hard_open<T, kThreads>(r, V, h);
  if (h.total <= kList) {
    constexpr uint32_t kEach = kList / kThreads;
    float z[kEach];
#pragma unroll
    for (uint32_t e = 0; e < kEach; ++e) {
      const uint32_t i = e * kThreads + threadIdx.x;
      z[e] = i < h.total ? to_f<T>(r.s[32 * h.w0 + h.tok[i]]) : -INFINITY;
    }
#pragma unroll
    for (uint32_t e = 0; e < kEach; ++e) {
      const uint32_t i = e * kThreads + threadIdx.x;
      if (i < h.total) {
        h.val[i] = z[e];
        if (32 * h.w0 + h.tok[i] == not_t) z[e] = -INFINITY;
      }
    }
    add_values(a, z, k);
  } else {
    const uint32_t n = 4 * h.nw;
    for (uint32_t j0 = threadIdx.x; j0 < n; j0 += 4 * kThreads) {
      Raw8<T> raw[4];
      float y[32];
      uint32_t b[4];
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u) {
        const uint32_t j = j0 + u * kThreads;
        b[u] = 0;
        if (j < n) b[u] = hard_chunk<T>(r, V, h, j, raw[u]);
        if (4 * h.w0 + j == not_t >> 3) b[u] &= ~(1u << (not_t & 7u));
      }
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u) {
        float z[8];
        widen8<T>(raw[u], z);
#pragma unroll
        for (uint32_t q = 0; q < 8; ++q)
          y[8 * u + q] = __uint_as_float(pick(sign_bit(b[u], q), __float_as_uint(z[q]), 0xFF800000u));
      }
      add_values(a, y, k);
    }
  }
  return a;
}

// the workgroup's share of a row, its token left out: segments s0 .. s1 - 1 (kHard:
// words held in LDS, or null: the row's mode is not kHard)
template <typename T, int kThreads>
__device__ __forceinline__ MaxSum scan_row(const Row<T>& r, uint32_t V, uint32_t s0, uint32_t s1, float k,
                                           int64_t tok, HardLds& h) {
  // a token outside the vocabulary is never met: V <= 2^30
  const uint32_t not_t = __builtin_amdgcn_readfirstlane(tok >= 0 && tok < (int64_t)V ? (uint32_t)tok : ~0u);
  if (r.mode == kHard) return scan_hard<T, kThreads>(r, V, k, not_t, h);
  return scan_other<T>(r, V, s0 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), s1, kThreads / 64,
                       threadIdx.x & 63, k, not_t);
}

// A row's log-probability, in f64, from its token's z and the other tokens'
// maximum and sum, and what the gradient needs: {m, -log2(sum)} with the token
// in them, or {0, +inf} for a row that has none.
struct RowStat {
  float m, nls;
};

__device__ __forceinline__ double row_logp(int64_t tok, uint32_t V, float za, MaxSum a, double inv_t, RowStat& st) {
  st = RowStat{0.f, INFINITY};
  if (tok < 0 || tok >= (int64_t)V) return 0.0;
  if (za == -INFINITY) return -INFINITY;
  const double d = ((double)za - (double)a.m) * inv_t;
  double ls, lp;
  if (d >= 0) {
    ls = log1p((double)a.s * exp(-d) + ((double)za - (double)za));      // z_a = +inf: NaN, as exp(inf - inf)
    lp = -ls;
    st.m = za;
  } else {
    ls = log((double)a.s + exp(d));
    lp = d - ls;
    st.m = a.m;
  }
  st.nls = (float)(-ls * 1.4426950408889634);
  return lp;
}

// A row's token and its z (0 for a token outside the vocabulary): read before
// the row is scanned, so their latency is not the row's tail.
struct Chosen {
  int64_t tok;
  float z;
};
template <typename T>
__device__ __forceinline__ Chosen chosen(const Rows& R, uint32_t n, const Row<T>& r) {
  Chosen c;
  c.tok = R.tokens[n];
  c.z = c.tok >= 0 && c.tok < (int64_t)R.V ? token_z<T>(r, (uint32_t)c.tok) : 0.f;
  return c;
}

// What the passes over rows leave (each may be null), and which rows they leave
// out unread: those of weight 0 and those of no sequence, when the caller
// returns nothing per row.
struct RowOut {
  float* logp;
  double* logp64;
  RowStat* stats;
  const float* weights;
  const int64_t* cu;
  uint32_t seqs;

  __device__ __forceinline__ bool skips(uint32_t n) const {
    if (!cu) return false;
    return (weights && weights[n] == 0.f) || (int64_t)n < cu[0] || (int64_t)n >= cu[seqs];
  }
};

__device__ __forceinline__ void put_row(const RowOut& o, uint32_t n, double lp, RowStat st) {
  if (o.logp) o.logp[n] = (float)lp;
  if (o.logp64) o.logp64[n] = lp;
  if (o.stats) o.stats[n] = st;
}

// Few rows: workgroup (slice, row) leaves its slice's maximum and sum.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) k_part(Rows R, uint32_t S, uint32_t per, bool hard, RowOut o,
                                                      MaxSum* __restrict__ parts) {
  __shared__ MaxSum sh[kRowThreads / 64];
  extern __shared__ uint32_t lds[];
  const uint32_t n = blockIdx.x / S, sl = blockIdx.x - n * S;
  if (o.skips(n)) return;
  const Row<T> r = open_row<T>(R, n, hard);
  const uint32_t s0 = sl * per, s1 = min((R.V + kSeg - 1) / kSeg, s0 + per);
  HardLds h = hard_lds(lds, s0 * (kSeg / 32), (s1 - s0) * (kSeg / 32));
  MaxSum a = scan_row<T, kRowThreads>(r, R.V, s0, s1, R.k, R.tokens[n], h);
  a = block_join<kRowThreads>(a, R.k, sh);
  if (threadIdx.x == 0) parts[(uint64_t)n * S + sl] = a;
}

// A row's S parts, joined by a wave: lane i takes parts i, i + 64, ...
// All lanes return the row's log-probability.
template <typename T>
__device__ __forceinline__ double finish_row(const Rows& R, uint32_t n, uint32_t S, const MaxSum* parts, RowStat& st) {
  const uint32_t lane = threadIdx.x & 63;
  const Chosen c = chosen<T>(R, n, open_row<T>(R, n));
  MaxSum a{-FLT_MAX, 0.f};
  for (uint32_t i = lane; i < S; i += 64) a = join(a, parts[(uint64_t)n * S + i], R.k);
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    MaxSum b;
    b.m = __shfl_xor(a.m, d);
    b.s = __shfl_xor(a.s, d);
    a = join(a, b, R.k);
  }
  return row_logp(c.tok, R.V, c.z, a, R.inv_t64, st);
}

template <typename T>
__global__ void __launch_bounds__(64) k_finish(Rows R, uint32_t S, const MaxSum* __restrict__ parts, RowOut o) {
  const uint32_t n = blockIdx.x;
  RowStat st{0.f, INFINITY};
  const double lp = o.skips(n) ? 0.0 : finish_row<T>(R, n, S, parts, st);
  if (threadIdx.x == 0) put_row(o, n, lp, st);
}

// A workgroup per row.  2048 x 128256 bf16 under soft masks: 116 us = 4.8 TB/s
// in a settled loop (the first tens of calls after a pause up to 145), the vector units as busy as the memory (11 instructions per score: widen, two
// bit-field extracts and two selects, add, round, maximum, fused multiply-add,
// exponential at a quarter of the rate, add).
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads) k_row(Rows R, bool hard, RowOut o) {
  __shared__ MaxSum sh[kThreads / 64];
  extern __shared__ uint32_t lds[];
  const uint32_t n = blockIdx.x, segs = (R.V + kSeg - 1) / kSeg;
  if (o.skips(n)) {
    if (threadIdx.x == 0) put_row(o, n, 0.0, RowStat{0.f, INFINITY});
    return;
  }
  const Row<T> r = open_row<T>(R, n, hard);
  const Chosen c = chosen<T>(R, n, r);
  HardLds h = hard_lds(lds, 0, segs * (kSeg / 32));
  MaxSum a = scan_row<T, kThreads>(r, R.V, 0, segs, R.k, c.tok, h);
  a = block_join<kThreads>(a, R.k, sh);
  if (threadIdx.x == 0) {
    RowStat st;
    const double lp = row_logp(c.tok, R.V, c.z, a, R.inv_t64, st);
    put_row(o, n, lp, st);
  }
}

// ---- the gradient: ds_t = c (1[t = a] - exp2((z_t - m) k - log2 sum)) --------
// At t = a it is -c expm1(logp): the difference 1 - p has lost its digits where
// p is near 1.

struct GradRow {
  float c, m, nls, k;     // c: what v_t's exponential is multiplied with
  float hot_c, hot_nls;   // the same at the chosen token
  uint32_t a;             // the token
};

// The hardware's exp2 gives 0 below 2^-126.  f16 gradients vanish long before;
// bf16's go on into subnormals, so there 2^32 more is raised and taken back by c
// (the exponent then rounds at 2^-19, far below bf16's 2^-9) -- from |c| = 2^-8
// on: below, what the exponential gives up is under 2^-134, half of bf16's
// smallest, and a small c would lose its own digits to the 2^-32.  f32 takes the
// full exp2f.
template <typename T>
__device__ __forceinline__ GradRow grad_of(float c, RowStat st, float k, uint32_t tok) {
  GradRow g;
  const bool lift = std::is_same_v<T, __hip_bfloat16> && fabsf(c) >= 0x1p-8f;
  g.c = lift ? c * 0x1p-32f : c;
  g.hot_c = c;
  g.hot_nls = st.nls;
  g.m = st.m;
  g.nls = lift ? st.nls + 32.f : st.nls;
  g.k = k;
  g.a = tok;
  return g;
}

template <typename T>
__device__ __forceinline__ float grad_out(const GradRow& g, float z) {
  const float x = fmaf(z - g.m, g.k, g.nls);
  return -g.c * (std::is_same_v<T, float> ? exp2f(x) : __builtin_amdgcn_exp2f(x));
}

__device__ __forceinline__ float grad_hot(const GradRow& g, float z) {
  return -g.hot_c * expm1f(fmaf(z - g.m, g.k, g.hot_nls) * 0.6931471805599453f);
}

template <typename T>
__device__ __forceinline__ float grad_at(const GradRow& g, float z, uint32_t t) {
  return t == g.a ? grad_hot(g, z) : grad_out<T>(g, z);
}

// 8 of them at chunk j.  kAny rows hold tokens that are out (z = -inf): theirs is
// 0 whatever the coefficient and the row's statistics are, NaN included.
template <typename T, Mode M>
__device__ __forceinline__ void grad8(const GradRow& g, uint32_t j, float (&z)[8]) {
  float za = 0.f;
  if (j == g.a >> 3) {
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q)
      if (q == (g.a & 7u)) za = z[q];
  }
#pragma unroll
  for (uint32_t q = 0; q < 8; ++q) z[q] = M == kAny && z[q] == -INFINITY ? 0.f : grad_out<T>(g, z[q]);
  if (j == g.a >> 3) {
    const float v = grad_hot(g, za);
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q)
      if (q == (g.a & 7u)) z[q] = v;
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

// segments last, last - waves, ... down to s0: backwards, so a workgroup that
// has just read the row finds its latest part in cache
template <typename T, Mode M>
__device__ __forceinline__ void grad_chunks(const Row<T>& r, const GradRow& g, T* o, uint32_t V, uint32_t s0,
                                            uint32_t last, uint32_t waves, uint32_t lane) {
  for (int64_t s = last; s >= (int64_t)s0; s -= waves) {
    const uint32_t seg = (uint32_t)s;
    if ((seg + 1) * kSeg <= V) {
      SegLoad<T, M> cur;
      cur.load(r, seg, lane);
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u) {
        const uint32_t j = seg * (kSeg / 8) + 64 * u + lane;
        float x[8];
        cur.values(r, seg, lane, u, x);
        grad8<T, M>(g, j, x);
        store8<T>(o + 8 * j, x);
      }
    } else {
      for (uint32_t j = seg * (kSeg / 8) + lane; 8 * j < V && j < (seg + 1) * (kSeg / 8); j += 64) {
        float x[8];
        edge_chunk<T, M>(r, V, j, x);
        grad8<T, M>(g, j, x);
        store_chunk<T>(o, j, V, x);
      }
    }
  }
}

// A kHard range.  A listed token's gradient is worked out once, by the thread
// that has it; then every chunk is stored whole, zeros or zeros and its few
// values.  opened: h holds the range's words, list and scores.
template <typename T, int kThreads>
__device__ void grad_hard(const Row<T>& r, const GradRow& g, T* o, uint32_t V, HardLds& h, bool opened) {
  if (!opened) hard_open<T, kThreads>(r, V, h);
  const uint32_t n = 4 * h.nw, t0 = 32 * h.w0;
  if (h.total > kList) {
    for (uint32_t j0 = threadIdx.x; j0 < n && t0 + 8 * j0 < V; j0 += 4 * kThreads) {
      Raw8<T> raw[4];
      uint32_t b[4];
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u) {
        const uint32_t j = j0 + u * kThreads;
        b[u] = 0;
        if (j < n) b[u] = hard_chunk<T>(r, V, h, j, raw[u]);
      }
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u) {
        const uint32_t j = j0 + u * kThreads;
        if (j >= n || t0 + 8 * j >= V) break;
        float z[8];
        widen8<T>(raw[u], z);
        if (b[u]) grad8<T, kHard>(g, (t0 >> 3) + j, z);
#pragma unroll
        for (uint32_t q = 0; q < 8; ++q)
          z[q] = __uint_as_float(__float_as_uint(z[q]) & sign_bit(b[u], q));     // NaN of an out token included
        store_chunk<T>(o, (t0 >> 3) + j, V, z);
      }
    }
    return;
  }
  for (uint32_t i = threadIdx.x; i < h.total; i += kThreads) {
    const uint32_t t = t0 + h.tok[i];
    const float z = opened ? h.val[i] : to_f<T>(r.s[t]);
    h.val[i] = grad_at<T>(g, z, t);
  }
  __syncthreads();
  for (uint32_t j = threadIdx.x; j < n && t0 + 8 * j < V; j += kThreads) {
    const uint32_t x = h.word[j >> 2], sh = 8 * (j & 3);
    float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (x >> sh & 0xFFu) {
      const uint32_t at = h.before[j >> 2];
#pragma unroll
      for (uint32_t q = 0; q < 8; ++q)
        if (x >> (sh + q) & 1u) z[q] = h.val[at + __popc(x & ((1u << (sh + q)) - 1u))];
    }
    store_chunk<T>(o, (t0 >> 3) + j, V, z);
  }
}

// The workgroup's share, segments s0 .. s1 - 1, of a row's gradient.
template <typename T, int kThreads>
__device__ __forceinline__ void grad_row(const Row<T>& r, const GradRow& g, T* o, uint32_t V, uint32_t s0, uint32_t s1,
                                         HardLds& h, bool opened) {
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr uint32_t waves = kThreads / 64;
  const uint32_t first = s0 + wave;
  if (g.c == 0.f) {
    for (uint32_t s = first; s < s1; s += waves) zero_segment<T>(o, V, s, lane);
    return;
  }
  if (r.mode == kHard) {
    grad_hard<T, kThreads>(r, g, o, V, h, opened);
    return;
  }
  if (first >= s1) return;
  const uint32_t last = first + (s1 - 1 - first) / waves * waves;
  switch (r.mode) {
    case kFree: grad_chunks<T, kFree>(r, g, o, V, s0, last, waves, lane); break;
    case kSoft: grad_chunks<T, kSoft>(r, g, o, V, s0, last, waves, lane); break;
    default: grad_chunks<T, kAny>(r, g, o, V, s0, last, waves, lane);
  }
}

// 3001 x 128256 bf16, a quarter of the rows without weight: 221 us = 6.1 TB/s
// of reads and stores, part of the reads from the last-level cache.
// Workgroup (slice, row), the last row first: what a scan of all rows has just
// read is still in the last-level cache.  skip_unit: the gradient is there
// already unless the scale is another than 1.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) k_grad(Rows R, uint32_t S, uint32_t per, bool hard,
                                                      const RowStat* __restrict__ stats,
                                                      const float* __restrict__ coef, const float* __restrict__ scale,
                                                      bool skip_unit, T* __restrict__ out, uint64_t ldo) {
  extern __shared__ uint32_t lds[];
  const float f = scale ? *scale : 1.f;
  if (skip_unit && f == 1.f) return;
  const uint32_t i = blockIdx.x / S, sl = blockIdx.x - i * S, n = R.N - 1 - i;
  const RowStat st = stats[n];
  const GradRow g = grad_of<T>(st.nls == INFINITY ? 0.f : coef[n] * f * R.inv_t, st, R.k, (uint32_t)R.tokens[n]);
  const uint32_t s0 = sl * per, s1 = min((R.V + kSeg - 1) / kSeg, s0 + per);
  HardLds h = hard_lds(lds, s0 * (kSeg / 32), (s1 - s0) * (kSeg / 32));
  grad_row<T, kRowThreads>(open_row<T>(R, n, hard), g, out + (uint64_t)n * ldo, R.V, s0, s1, h, false);
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
// The ratio is clipped by comparisons, which keep a NaN (fmin and fmax would put
// a border in its place): NaN in the row's scores, old_logp or A makes the loss
// and the row's gradient NaN.  A = 0 counts as 0 beside an infinite ratio too.
__device__ __forceinline__ double policy_term(const PolicyIn& P, uint32_t n, double lp, bool live, float& coef) {
  const double w = P.weights ? (double)P.weights[n] : P.w;
  coef = 0.f;
  if (!live || w == 0.0) return 0.0;
  const double A = P.adv[n];
  const double r = exp(lp - (double)P.old_logp[n]);
  double l = 0.0, g = 0.0;
  if (A != 0.0 || isnan(r)) {
    const double a = r * A, b = (r < P.lo ? P.lo : r > P.hi ? P.hi : r) * A;
    l = a <= b ? -a : -b;
    g = a <= b ? -a : a > b ? 0.0 : a + b;
  }
  if (P.kl != 0.0) {
    const double d = (double)P.ref_logp[n] - lp, e = exp(d);
    l += P.kl * (expm1(d) - d);
    g += P.kl * (1.0 - e);
  }
  coef = (float)(w * g);
  return w * l;
}

// Few rows: a wave each joins its row's S parts and takes the row's term; one
// workgroup (up to 16 rows) also adds the terms up, more leave them to k_sum.
constexpr uint32_t kOneRows = kOneThreads / 64;
template <typename T>
__global__ void __launch_bounds__(kOneThreads) k_policy_few(Rows R, uint32_t S, const MaxSum* __restrict__ parts,
                                                            PolicyIn P, RowOut o, float* __restrict__ coef,
                                                            double* __restrict__ terms, float* __restrict__ loss) {
  __shared__ double sh[kOneThreads / 64];
  const uint32_t n = blockIdx.x * kOneRows + (threadIdx.x >> 6);
  double term = 0;
  if (n < R.N) {
    RowStat st;
    const double lp = finish_row<T>(R, n, S, parts, st);
    if ((threadIdx.x & 63) == 0) {
      float c;
      term = policy_term(P, n, lp, st.nls != INFINITY, c);
      put_row(o, n, lp, st);
      coef[n] = c;
      if (gridDim.x > 1) terms[n] = term;
    }
  }
  if (gridDim.x > 1) return;
  term = block_sum64(term, sh);
  if (threadIdx.x == 0) *loss = (float)term;
}

// Many rows: a workgroup reads its row, knows its coefficient, and writes the
// row's gradient (scale 1) from a second read of the same row, backwards and so
// largely from the caches: a row between its first and second read is at most
// 512 KB old per workgroup, 512 workgroups apart, where the gradient as a
// kernel of its own found 456 MB of other rows in between.
// 1500 x 151936 bf16: 199 us, 4.6 TB/s of the scores read once and the gradient;
// 4096 x 128256 with about 400 tokens a row: 282 us.
// terms[n]: the row's loss, for k_sum.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads) k_policy_row(Rows R, bool hard, PolicyIn P, RowOut o,
                                                              float* __restrict__ coef, double* __restrict__ terms,
                                                              T* __restrict__ grad, uint64_t ldg) {
  __shared__ MaxSum sh[kThreads / 64];
  __shared__ GradRow gs;
  extern __shared__ uint32_t lds[];
  const uint32_t n = blockIdx.x, segs = (R.V + kSeg - 1) / kSeg;
  const Row<T> r = open_row<T>(R, n, hard);
  const Chosen c = chosen<T>(R, n, r);
  HardLds h = hard_lds(lds, 0, segs * (kSeg / 32));
  MaxSum a = scan_row<T, kThreads>(r, R.V, 0, segs, R.k, c.tok, h);
  a = block_join<kThreads>(a, R.k, sh);
  if (threadIdx.x == 0) {
    RowStat st;
    const double lp = row_logp(c.tok, R.V, c.z, a, R.inv_t64, st);
    float cf;
    terms[n] = policy_term(P, n, lp, st.nls != INFINITY, cf);
    put_row(o, n, lp, st);
    coef[n] = cf;
    gs = grad_of<T>(cf * R.inv_t, st, R.k, (uint32_t)c.tok);
  }
  if (!grad) return;
  __syncthreads();
  grad_row<T, kThreads>(r, gs, grad + (uint64_t)n * ldg, R.V, 0, segs, h, true);
}

__global__ void __launch_bounds__(kOneThreads) k_sum(uint32_t N, const double* __restrict__ terms,
                                                     float* __restrict__ loss) {
  __shared__ double sh[kOneThreads / 64];
  double sum = 0;
  for (uint32_t n = threadIdx.x; n < N; n += kOneThreads) sum += terms[n];
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
// One workgroup's chains of reads are its time, so every lane has kAhead rows'
// under way, whether they count or not (3001 rows in 16 sequences: 10.9 us, one
// row at a time 14.6).
constexpr int kAhead = 4;
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
    for (int64_t n0 = b + lane; n0 < e; n0 += 64 * kAhead) {
      double w[kAhead], lp[kAhead];
      bool live[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int64_t n = min(n0 + 64 * u, e - 1);
        w[u] = P.weights ? (double)P.weights[n] : 1.0;
        live[u] = stats[n].nls != INFINITY && n0 + 64 * u < e;
        lp[u] = logp[n];
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (w[u] != 0.0 && live[u]) s += w[u] * lp[u];
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
    for (int64_t n0 = b + lane; n0 < e; n0 += 64 * kAhead) {
      double w[kAhead];
      bool live[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int64_t n = min(n0 + 64 * u, e - 1);
        w[u] = P.weights ? (double)P.weights[n] : 1.0;
        live[u] = stats[n].nls != INFINITY && n0 + 64 * u < e;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (w[u] != 0.0 && live[u]) coef[n0 + 64 * u] = (float)(w[u] * g);
    }
  }
}

// ---- launch ----------------------------------------------------------------

// Whether one workgroup takes a whole row: from kManyRows rows on, and for rows
// of up to kShortRow tokens whatever their number.  Slices of a row fill more of
// the chip, and pay for it with a launch or two more: at 4 rows of 2^20 tokens
// 20 us for 48 (bf16), at 128256 tokens 20 for 17, at 800 rows 40 us either way.
constexpr uint64_t kManyRows = 256, kShortRow = 1 << 18;
bool whole_rows(uint64_t N, uint64_t V) { return N >= kManyRows || V <= kShortRow; }

// How a row is cut otherwise: slices of at least one segment per wave.
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
Cut scan_cut(uint64_t N, uint64_t V) { return cut(N, V, whole_rows(N, V) ? 0 : 2048); }
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

// LDS of a launch whose workgroups take `segs` segments of a row each; 0: rows
// go without the kHard form (no constraint, or a range past kHardWords)
uint32_t hard_lds_bytes(const Rows& R, uint64_t segs) {
  const uint64_t nw = segs * (kSeg / 32);
  return (R.bits || R.uni || R.rp) && nw <= kHardWords ? hard_bytes((uint32_t)nw) : 0u;
}
uint64_t segments(uint64_t V) { return (V + kSeg - 1) / kSeg; }

// Threads of a whole row's workgroup.  Short rows want more, smaller workgroups
// (4096 x 50265 bf16, log-probabilities: 90 us with 256 threads, 106 with 512),
// long ones fewer rows at a time, so that the gradient's second read still finds
// them in the caches (1500 x 151936, policy: 209 us with 512 threads, 238 with
// 256; at 1024, one workgroup per CU, 2048 x 128256 log-probabilities took 158
// us for 126).
template <typename F>
void by_row_length(uint64_t segs, F f) {
  if (segs <= 1) f(std::integral_constant<int, 64>());
  else if (segs <= 32) f(std::integral_constant<int, 256>());
  else f(std::integral_constant<int, 512>());
}

int run_logp(int dtype, const Rows& R, const RowOut& o, MaxSum* parts, hipStream_t s) {
  const Cut c = scan_cut(R.N, R.V);
  return by_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (whole_rows(R.N, R.V)) {
      const uint32_t lds = hard_lds_bytes(R, segments(R.V));
      by_row_length(segments(R.V), [&](auto n) {
        k_row<T, decltype(n)::value><<<R.N, decltype(n)::value, lds, s>>>(R, lds != 0, o);
      });
    } else {
      const uint32_t lds = hard_lds_bytes(R, c.per);
      k_part<T><<<R.N * c.S, kRowThreads, lds, s>>>(R, c.S, c.per, lds != 0, o, parts);
      k_finish<T><<<R.N, 64, 0, s>>>(R, c.S, parts, o);
    }
  });
}

int run_grad(int dtype, const Rows& R, const RowStat* stats, const float* coef, const float* scale, bool skip_unit,
             void* out, uint64_t ldo, hipStream_t s) {
  const Cut c = grad_cut(R.N, R.V);
  return by_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const uint32_t lds = hard_lds_bytes(R, c.per);
    k_grad<T><<<R.N * c.S, kRowThreads, lds, s>>>(R, c.S, c.per, lds != 0, stats, coef, scale, skip_unit,
                                                  reinterpret_cast<T*>(out), ldo);
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
  return run_logp(a->dtype, R, RowOut{logp, nullptr, reinterpret_cast<RowStat*>(stats), nullptr, nullptr, 0}, reinterpret_cast<MaxSum*>(ws),
                  s);
}

int token_logprobs_grad(const fm_score_rows* a, const float* stats, const float* coef, const float* scale,
                        int skip_unit, void* grad, uint64_t ld_grad, hipStream_t s) {
  Rows R;
  if (as_rows(a, R)) return -1;
  if (R.N == 0) return 0;
  if (!stats || !coef || !grad || ld_grad < R.V) {
    set_error("token_logprobs_grad: null buffer, or ld_grad < V");
    return -1;
  }
  return run_grad(a->dtype, R, reinterpret_cast<const RowStat*>(stats), coef, scale, skip_unit != 0, grad, ld_grad, s);
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
  if (p->d_grad && p->ld_grad < R.V) {
    set_error("policy_loss: ld_grad < V");
    return -1;
  }
  const Layout l = layout(R.N, R.V, 0);
  if (check_ws(p->d_ws, p->ws_bytes, l.bytes)) return -1;
  char* ws = reinterpret_cast<char*>(p->d_ws);
  double* terms = reinterpret_cast<double*>(ws + l.logp);
  MaxSum* parts = reinterpret_cast<MaxSum*>(ws);
  const RowOut o{p->d_logp, nullptr, reinterpret_cast<RowStat*>(p->d_stats), nullptr, nullptr, 0};
  const PolicyIn in{p->d_old_logp, p->d_ref_logp, p->d_advantages, p->d_weights, 1.0 - p->clip_low, 1.0 + p->clip_high,
                    p->kl_coef, 1.0 / std::max<uint32_t>(R.N, 1)};
  if (R.N && whole_rows(R.N, R.V))
    return by_dtype(a->dtype, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      const uint32_t lds = hard_lds_bytes(R, segments(R.V));
      by_row_length(segments(R.V), [&](auto n) {
        k_policy_row<T, decltype(n)::value><<<R.N, decltype(n)::value, lds, s>>>(
            R, lds != 0, in, o, p->d_coef, terms, reinterpret_cast<T*>(p->d_grad), p->ld_grad);
      });
      k_sum<<<1, kOneThreads, 0, s>>>(R.N, terms, p->d_loss);
    });
  const Cut c = scan_cut(R.N, R.V);
  if (by_dtype(a->dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const uint32_t lds = hard_lds_bytes(R, c.per);
        if (R.N) k_part<T><<<R.N * c.S, kRowThreads, lds, s>>>(R, c.S, c.per, lds != 0, o, parts);
        const uint32_t groups = std::max(1u, (R.N + kOneRows - 1) / kOneRows);
        k_policy_few<T><<<groups, kOneThreads, 0, s>>>(R, c.S, parts, in, o, p->d_coef, terms, p->d_loss);
        if (groups > 1) k_sum<<<1, kOneThreads, 0, s>>>(R.N, terms, p->d_loss);
      }))
    return -1;
  return R.N && p->d_grad ? run_grad(a->dtype, R, o.stats, p->d_coef, nullptr, false, p->d_grad, p->ld_grad, s) : 0;
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
  if (R.N && run_logp(a->dtype, R, RowOut{nullptr, lp, st, p->d_weights, p->d_cu, (uint32_t)(2 * p->pairs)},
                      reinterpret_cast<MaxSum*>(ws), s)) return -1;
  const PreferenceIn in{p->d_cu, p->d_weights, p->d_ref_logp, (uint32_t)p->pairs, p->beta, p->label_smoothing,
                        p->margin};
  k_preference<<<1, kOneThreads, 0, s>>>(R.N, in, lp, st, reinterpret_cast<double*>(ws + l.pref), p->d_seq_logp,
                                         p->d_coef, p->d_loss);
  FM_HIP(hipGetLastError());
  return 0;
}

}  // namespace fmidx
