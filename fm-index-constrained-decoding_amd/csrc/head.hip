// head.hip -- the scores product with the document constraint in its epilogue.
//
//     x[b, t]   = sum_k hidden[b, k] weight[t, k] + bias[t]          (f32)
//     y[b, t]   = softcap ? softcap tanh(x / softcap) : x
//     out[b, t] = y + residual[b, t] + mask[b, t], rounded once;  -inf where mask is -inf
//
// mask is the row's value of row_mask.h (what fm_apply_boosts adds).  16-bit
// operands, f32 accumulation on the matrix cores (16x16x32: 8 consecutive k per
// lane of either operand, 4 consecutive tokens of one row per lane of the
// result).
#include "fmidx_internal.h"
#include "row_mask.h"
#include "../../include/fmidx.h"

#include <algorithm>
#include <cmath>

namespace fmidx {
namespace {

typedef unsigned hd_v4u __attribute__((ext_vector_type(4)));
typedef hd_v4u hd_v4u_a2 __attribute__((aligned(2)));     // rows start wherever their stride puts them
typedef hd_v4u hd_v4u_a4 __attribute__((aligned(4)));
typedef float hd_v4f __attribute__((ext_vector_type(4)));
typedef __bf16 hd_v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 hd_v8h __attribute__((ext_vector_type(8)));

struct Head {
  const void *hidden, *weight, *bias, *residual;
  void* out;
  uint64_t ldh, ldw, ldr, ldo;
  uint32_t B, V, d;
  const uint32_t* bits;
  uint64_t ldb;
  const uint32_t* uni;
  const RowParams* rp;
  int64_t eos;
  float cap, inv_cap;
};

template <typename T>
__device__ __forceinline__ hd_v4f mma(hd_v4u a, hd_v4u b, hd_v4f c) {
  if constexpr (std::is_same_v<T, __hip_bfloat16>)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(hd_v8bf, a), __builtin_bit_cast(hd_v8bf, b), c,
                                                   0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(hd_v8h, a), __builtin_bit_cast(hd_v8h, b), c, 0,
                                                  0, 0);
}

// 8 elements of a row from k on; zeros from d on
template <typename T>
__device__ __forceinline__ hd_v4u frag(const T* row, uint32_t k, uint32_t d) {
  hd_v4u x = {0, 0, 0, 0};
  if (k >= d) return x;
  if (k + 8 <= d) return *reinterpret_cast<const hd_v4u_a2*>(row + k);
  const unsigned short* p = reinterpret_cast<const unsigned short*>(row + k);
#pragma unroll
  for (uint32_t q = 0; q < 8; ++q)
    if (k + q < d) x[q >> 1] |= (uint32_t)p[q] << (16 * (q & 1));
  return x;
}

// the mask values of batch row b, and their rules
__device__ __forceinline__ RowParams head_row(const Head& H, uint32_t b, RowSel& r) {
  RowParams p;
  if (H.rp) {
    p = H.rp[b];
    if (!H.bits) p.flags &= ~kUseBits;
    if (!H.uni) p.flags &= ~kUnigram;
  } else {
    p.base = H.bits ? -INFINITY : 0.f;
    p.v_dist = p.v_uni = p.v_eos = 0.f;
    p.flags = H.bits ? kUseBits : 0u;
    p.special = -1;
  }
  r = row_sel(p, H.V, H.eos);
  return p;
}

// tanh, off by under 5 half-steps of itself: 1 - 2 / (e^2x + 1) from 0.7 on, and
// below, where that cancels (6 half-steps at 0.25), x + x^3 q(x^2), q fitted to
// tanh by least squares of the relative error on [0, 0.7] (1.5 half-steps).
__device__ __forceinline__ float soft(float x) {
  const float t = x * x;
  const float q = fmaf(t, fmaf(t, fmaf(t, fmaf(t, -0.005138651933521032f, 0.020091958343982697f), -0.05355885624885559f),
                               0.1332911103963852f), -0.3333319127559662f);
  const float near = fmaf(x * t, q, x);
  const float e = __builtin_amdgcn_exp2f(2.8853900817779268f * x);
  const float far = fmaf(-2.f, __builtin_amdgcn_rcpf(e + 1.f), 1.f);
  return fabsf(x) < 0.7f ? near : far;
}

// one element's epilogue; everything it reads is asked for before the first use
template <typename T, typename O>
__device__ __forceinline__ void finish(const Head& H, const RowSel& r, uint32_t b, uint32_t t, float x) {
  const uint32_t dw = H.bits ? H.bits[(uint64_t)b * H.ldb + (t >> 5)] : 0u;
  const uint32_t uw = H.uni ? H.uni[t >> 5] : 0u;
  const float bias = H.bias ? to_f<T>(reinterpret_cast<const T*>(H.bias)[t]) : 0.f;
  const float res = H.residual ? to_f<O>(reinterpret_cast<const O*>(H.residual)[(uint64_t)b * H.ldr + t]) : 0.f;
  uint32_t hi, lo;
  chunk_codes(r, t >> 3, dw, uw, hi, lo);
  const float v = mask_at(r, hi, lo, t & 7);
  x += bias;
  if (H.cap != 0.f) x = H.cap * soft(x * H.inv_cap);
  x = (x + res) + v;
  reinterpret_cast<O*>(H.out)[(uint64_t)b * H.ldo + t] = from_f<O>(v == -INFINITY ? -INFINITY : x);
}

// 8 tokens t0 .. t0 + 7 of row b (t0 a multiple of 8), all inside the row
template <typename T>
__device__ __forceinline__ void load8f(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const hd_v4u a = *reinterpret_cast<const hd_v4u_a4*>(p), b = *reinterpret_cast<const hd_v4u_a4*>(p + 4);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      x[q] = __uint_as_float(a[q]);
      x[q + 4] = __uint_as_float(b[q]);
    }
  } else {
    const hd_v4u a = *reinterpret_cast<const hd_v4u_a2*>(p);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      x[2 * q] = to_f<T>(__builtin_bit_cast(T, (unsigned short)(a[q] & 0xFFFFu)));
      x[2 * q + 1] = to_f<T>(__builtin_bit_cast(T, (unsigned short)(a[q] >> 16)));
    }
  }
}

template <typename O>
__device__ __forceinline__ void store8f(O* p, const float (&x)[8]) {
  if constexpr (sizeof(O) == 4) {
    hd_v4u a, b;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      a[q] = __float_as_uint(x[q]);
      b[q] = __float_as_uint(x[q + 4]);
    }
    *reinterpret_cast<hd_v4u_a4*>(p) = a;
    *reinterpret_cast<hd_v4u_a4*>(p + 4) = b;
  } else {
    hd_v4u a;
#pragma unroll
    for (int q = 0; q < 4; ++q) a[q] = pack16<O>(x[2 * q], x[2 * q + 1]);
    *reinterpret_cast<hd_v4u_a2*>(p) = a;
  }
}

template <typename T, typename O>
__device__ __forceinline__ void finish8(const Head& H, bool masked, const RowParams& p, uint32_t dw, uint32_t uw,
                                        uint32_t b, uint32_t t0, const float (&bias)[8], float (&x)[8]) {
#pragma unroll
  for (int q = 0; q < 8; ++q) x[q] += bias[q];
  if (H.cap != 0.f) {
#pragma unroll
    for (int q = 0; q < 8; ++q) x[q] = H.cap * soft(x[q] * H.inv_cap);
  }
  if (H.residual) {
    float y[8];
    load8f<O>(reinterpret_cast<const O*>(H.residual) + (uint64_t)b * H.ldr + t0, y);
#pragma unroll
    for (int q = 0; q < 8; ++q) x[q] += y[q];
  }
  if (masked) {
    const RowSel r = row_sel(p, H.V, H.eos);
    uint32_t hi, lo;
    chunk_codes(r, t0 >> 3, dw, uw, hi, lo);
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q) {
      const uint32_t ml = sign_bit(lo, q);
      const float v = __uint_as_float(pick(sign_bit(hi, q), pick(ml, r.fe, r.fd), pick(ml, r.fu, r.fb)));
      x[q] = v == -INFINITY ? -INFINITY : x[q] + v;
    }
  }
  store8f<O>(reinterpret_cast<O*>(H.out) + (uint64_t)b * H.ldo + t0, x);
}

// ---- which weight rows are needed ---------------------------------------------
// A token's weight row is needed if its mask value is above -inf in some row.
// k_need: per 512 tokens, the needed ones listed in order and counted.
// k_fill: -inf where the mask says so, the chunks' lists joined (the order
// stays), and for every listed token the rows that it is in for, as bits.
// Neither does more when above half of the vocabulary is needed: then the
// product runs over all of it and writes every score itself, which costs less
// than gathering.
constexpr uint32_t kChunk = 2048;           // tokens per workgroup of k_fill and k_fill_few
constexpr uint32_t kSub = 512;              // of k_need
constexpr uint32_t kMaxChunks = 512;        // lists up to 2^20 tokens; above, no list is made

struct Need {
  uint32_t* count;       // [lists], then how many are listed in all (V: no list, all are taken)
  uint32_t* part;        // [chunks * kChunk]
  uint32_t* list;        // [listed <= V / 2]; null: no lists
  uint32_t* rows;        // [ceil(B / 32)][cap]: bit b % 32 of word b / 32: the listed token is in for row b
  uint32_t chunks, lists, cap;    // lists: as many as k_need (k_fill_few) has workgroups
};

// The tokens of word w that a row's mask leaves in; dw, uw: the row's allowed
// bits and the corpus's tokens there, read by the caller whether the row uses
// them or not, so that many rows' reads are under way together.
__device__ __forceinline__ uint32_t need_word(const RowParams& p, const RowSel& r, uint32_t dw, uint32_t uw,
                                              uint32_t w) {
  const uint32_t d = (r.dm ? dw : 0u) | (w == r.js >> 2 ? r.sb << (8 * (r.js & 3)) : 0u);
  const uint32_t u = r.um ? uw : 0u;
  const uint32_t e = w == r.je >> 2 ? r.eb << (8 * (r.je & 3)) : 0u;
  uint32_t x = p.base != -INFINITY ? ~0u : 0u;
  x = (x & ~u) | (p.v_uni != -INFINITY ? u : 0u);
  x = (x & ~d) | (p.v_dist != -INFINITY ? d : 0u);
  return (x & ~e) | (p.v_eos != -INFINITY ? e : 0u);
}

// word w of rows first, first + step, ... (kRows of them; past the last row: the last one again)
template <int kRows>
__device__ __forceinline__ void need_words(const Head& H, uint32_t first, uint32_t step, uint32_t w,
                                           uint32_t (&x)[kRows]) {
  const uint32_t uw = H.uni ? H.uni[w] : 0u;
  uint32_t dw[kRows];
#pragma unroll
  for (uint32_t i = 0; i < kRows; ++i)
    dw[i] = H.bits ? H.bits[(uint64_t)min(first + i * step, H.B - 1) * H.ldb + w] : 0u;
#pragma unroll
  for (uint32_t i = 0; i < kRows; ++i) {
    RowSel r;
    const RowParams p = head_row(H, min(first + i * step, H.B - 1), r);
    x[i] = need_word(p, r, dw[i], uw, w);
  }
}

// a wave's inclusive prefix sum
__device__ __forceinline__ uint32_t wave_upto(uint32_t x, uint32_t lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = (uint32_t)__shfl_up((int)x, d);
    if (lane >= (uint32_t)d) x += o;
  }
  return x;
}

// Workgroup (512 tokens).  16 lanes take a row's 16 words, so the rows' rules
// are worked out by lanes, 64 rows at a time, and every CU has a workgroup; with
// a row per wave they were scalar work on a quarter of the CUs (11 us for 9 at
// 256 x 151936).
__global__ void __launch_bounds__(1024) k_need(Head H, Need N) {
  __shared__ uint32_t sh[64][17];
  const uint32_t word = threadIdx.x & 15, slot = threadIdx.x >> 4, lane = threadIdx.x & 63;
  const uint32_t w = blockIdx.x * (kSub / 32) + word;
  uint32_t x = 0;
  if (32 * w < H.V)
    for (uint32_t b = slot; b < H.B && x != ~0u; b += 256) {       // one soft row needs all
      uint32_t y[4];
      need_words<4>(H, b, 64, w, y);
#pragma unroll
      for (int i = 0; i < 4; ++i) x |= y[i];
    }
  sh[slot][word] = x;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  x = 0;
#pragma unroll
  for (uint32_t i = 0; i < 16; ++i) x |= sh[16 * (lane >> 4) + i][word];
  x |= (uint32_t)__shfl_xor((int)x, 16);
  x |= (uint32_t)__shfl_xor((int)x, 32);
  if (32 * w >= H.V) x = 0;
  else if (H.V - 32 * w < 32) x &= (1u << (H.V - 32 * w)) - 1;
  const uint32_t upto = wave_upto(lane < 16 ? __popc(x) : 0u, lane);
  if (lane == 63) N.count[blockIdx.x] = upto;
  // every lane a byte of its word
  uint32_t* list = N.part + (uint64_t)blockIdx.x * kSub + ((uint32_t)__shfl((int)upto, (int)word) - __popc(x));
  for (uint32_t y = x & (0xFFu << (8 * (lane >> 4))); y; y &= y - 1) {
    const uint32_t q = (uint32_t)__ffs((int)y) - 1;
    list[__popc(x & ((1u << q) - 1u))] = 32 * w + q;
  }
}

// the sums of all counts and of those before list c, by the whole workgroup; sh: 32 words
__device__ __forceinline__ uint2 count_sums(const Need& N, uint32_t c, uint32_t* sh) {
  uint32_t s = 0, before = 0;
  for (uint32_t i = threadIdx.x; i < N.lists; i += blockDim.x) {
    const uint32_t v = N.count[i];
    s += v;
    before += i < c ? v : 0u;
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    s += (uint32_t)__shfl_xor((int)s, d);
    before += (uint32_t)__shfl_xor((int)before, d);
  }
  if ((threadIdx.x & 63) == 0) {
    sh[threadIdx.x >> 6] = s;
    sh[16 + (threadIdx.x >> 6)] = before;
  }
  __syncthreads();
  s = before = 0;
  for (uint32_t i = 0; i < blockDim.x / 64; ++i) {
    s += sh[i];
    before += sh[16 + i];
  }
  __syncthreads();
  return make_uint2(s, before);
}

// how many tokens are listed; V: all of them, without a list
__device__ __forceinline__ uint32_t listed(const Head& H, const Need& N) { return N.list ? N.count[N.lists] : H.V; }

// Workgroup (chunk of tokens, 32 rows).
template <typename O>
__global__ void __launch_bounds__(256) k_fill(Head H, Need N) {
  __shared__ uint32_t sh[32];
  __shared__ uint32_t in[32][65];
  const uint32_t c = blockIdx.x, b0 = blockIdx.y * 32;
  constexpr uint32_t kSubs = kChunk / kSub;
  const uint2 sums = count_sums(N, c * kSubs, sh);
  const bool all = 2 * sums.x > H.V;
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) N.count[N.lists] = all ? H.V : sums.x;
  if (all) return;
  const uint32_t w0 = c * (kChunk / 32);
  // the rows' words: 64 lanes a row, 4 rows at a time
  {
    const uint32_t lane = threadIdx.x & 63, part = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (32 * (w0 + lane) < H.V) need_words<8>(H, b0 + part, 4, w0 + lane, x);
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) in[i * 4 + part][lane] = b0 + i * 4 + part < H.B ? x[i] : 0u;
  }
  __syncthreads();
  uint32_t at = sums.y;
  for (uint32_t k = c * kSubs; k < min(N.lists, (c + 1) * kSubs); ++k) {
    const uint32_t n = N.count[k];
    for (uint32_t i = threadIdx.x; i < n; i += 256) {
      const uint32_t t = N.part[(uint64_t)k * kSub + i], w = (t >> 5) - w0, q = t & 31;
      uint32_t m = 0;
#pragma unroll
      for (uint32_t rr = 0; rr < 32; ++rr) m |= (in[rr][w] >> q & 1u) << rr;
      N.rows[(uint64_t)blockIdx.y * N.cap + at + i] = m;
      if (blockIdx.y == 0) N.list[at + i] = t;
    }
    at += n;
  }
  // 256 chunks of 8 tokens a row, one per thread
  const uint32_t j = c * (kChunk / 8) + threadIdx.x;
  if (8 * j >= H.V) return;
  const float none[8] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY};
  const uint32_t rows = min(32u, H.B - b0);
  O* o = reinterpret_cast<O*>(H.out) + (uint64_t)b0 * H.ldo + 8 * j;
  for (uint32_t rr = 0; rr < rows; ++rr, o += H.ldo) {
    const uint32_t x = in[rr][threadIdx.x >> 2] >> (8 * (threadIdx.x & 3)) & 0xFFu;
    if (x == 0 && 8 * j + 8 <= H.V) {
      store8f<O>(o, none);
    } else {
      for (uint32_t q = 0; q < 8; ++q)
        if (8 * j + q < H.V && !(x >> q & 1)) o[q] = from_f<O>(-INFINITY);
    }
  }
}

// ---- up to 16 rows of the batch -----------------------------------------------------
// One kernel in the place of k_need and k_fill: every workgroup has all rows'
// words of its chunk, so it lists the chunk's tokens (part, rows: at 2048 chunk
// + place) and writes the -inf's at once.  When the product then takes the
// whole vocabulary, it writes them again.
constexpr uint32_t kFewRows = 16;

template <typename O>
__global__ void __launch_bounds__(256) k_fill_few(Head H, Need N) {
  __shared__ uint32_t in[kFewRows][65], any[64], base[64];
  const uint32_t c = blockIdx.x, w0 = c * (kChunk / 32), lane = threadIdx.x & 63, part = threadIdx.x >> 6;
  const uint32_t w = w0 + lane;
  {
    const uint32_t first = __builtin_amdgcn_readfirstlane(part);
    uint32_t x[kFewRows / 4] = {};
    if (32 * w < H.V) need_words<kFewRows / 4>(H, first, 4, w, x);
#pragma unroll
    for (uint32_t i = 0; i < kFewRows / 4; ++i) {
      const uint32_t spare = 32 * w < H.V && H.V - 32 * w < 32 ? (1u << (H.V - 32 * w)) - 1 : ~0u;
      in[i * 4 + first][lane] = i * 4 + first < H.B ? x[i] & spare : 0u;
    }
  }
  __syncthreads();
  if (part == 0) {
    uint32_t x = 0;
#pragma unroll
    for (uint32_t row = 0; row < kFewRows; ++row) x |= in[row][lane];
    const uint32_t upto = wave_upto(__popc(x), lane);
    any[lane] = x;
    base[lane] = upto - __popc(x);
    if (lane == 63) N.count[c] = upto;
  }
  __syncthreads();
  for (uint32_t x = any[lane] & (0xFFu << (8 * part)); x; x &= x - 1) {
    const uint32_t q = (uint32_t)__ffs((int)x) - 1;
    uint32_t m = 0;
#pragma unroll
    for (uint32_t row = 0; row < kFewRows; ++row) m |= (in[row][lane] >> q & 1u) << row;
    const uint64_t at = (uint64_t)c * kChunk + base[lane] + __popc(any[lane] & ((1u << q) - 1u));
    N.part[at] = 32 * w + q;
    N.rows[at] = m;
  }
  const uint32_t j = c * (kChunk / 8) + threadIdx.x;
  if (8 * j >= H.V) return;
  const float none[8] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY};
  O* o = reinterpret_cast<O*>(H.out) + 8 * j;
  for (uint32_t row = 0; row < H.B; ++row, o += H.ldo) {
    const uint32_t x = in[row][threadIdx.x >> 2] >> (8 * (threadIdx.x & 3)) & 0xFFu;
    if (x == 0 && 8 * j + 8 <= H.V) {
      store8f<O>(o, none);
    } else {
      for (uint32_t q = 0; q < 8; ++q)
        if (8 * j + q < H.V && !(x >> q & 1)) o[q] = from_f<O>(-INFINITY);
    }
  }
}

// 16 listed tokens per workgroup at a time, its waves each a share of k
// straight from memory into the matrix cores (a lane's 8 k's are 16 B of one
// row), joined in LDS: a few hundred tokens are a few dozen workgroups, one
// round trip each.  (Over the whole vocabulary the tiles below are faster even
// for one row: 179 us for 193 at 1 x 4096 x 128256, 184 for 248 at 8 rows.)
constexpr int kFewWaves = 8;
static_assert(kFewWaves * 64 >= kMaxChunks, "a thread per chunk");

template <typename T, typename O>
__global__ void __launch_bounds__(kFewWaves * 64) k_head_few(Head H, Need N) {
  __shared__ hd_v4f sh[kFewWaves][64];
  __shared__ uint32_t start[kFewWaves * 64 + 1], sums[kFewWaves];
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  // where each chunk's tokens start in the joined list
  const uint32_t mine = threadIdx.x < N.chunks ? N.count[threadIdx.x] : 0u, upto = wave_upto(mine, lane);
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  uint32_t before = 0, total = 0;
#pragma unroll
  for (uint32_t q = 0; q < (uint32_t)kFewWaves; ++q) {
    before += q < wave ? sums[q] : 0u;
    total += sums[q];
  }
  start[threadIdx.x + 1] = before + upto;
  if (threadIdx.x == 0) start[0] = 0;
  const bool all = 2 * total > H.V;
  if (blockIdx.x == 0 && threadIdx.x == 0) N.count[N.lists] = all ? H.V : total;
  if (all) return;                      // the tiles' turn
  __syncthreads();
  auto find = [&](uint32_t e) {         // entry e's place: the last chunk that starts at or before it
    uint32_t lo = 0, hi = N.chunks;     // start[lo] <= e < start[hi]
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (start[mid] <= e) lo = mid;
      else hi = mid;
    }
    return lo * kChunk + (e - start[lo]);
  };
  // lanes without a row or a token of their own repeat a valid one; their results are not stored
  const T* h = reinterpret_cast<const T*>(H.hidden) + (uint64_t)min(i, H.B - 1) * H.ldh + 8 * g;
  RowSel r;
  if (i < H.B) head_row(H, i, r);
  constexpr uint32_t kStep = kFewWaves * 32, kAhead = 8;       // requests in flight per operand and lane
  for (uint32_t e0 = blockIdx.x * 16; e0 < total; e0 += gridDim.x * 16) {
    const uint32_t at = find(min(e0 + i, total - 1));
    const uint32_t t = N.part[at], rows = N.rows[at];
    const T* w = reinterpret_cast<const T*>(H.weight) + (uint64_t)t * H.ldw + 8 * g;
    hd_v4f acc = {0, 0, 0, 0};
    uint32_t k = wave * 32;
    for (; k + (kAhead - 1) * kStep + 32 <= H.d; k += kAhead * kStep) {
      hd_v4u a[kAhead], b[kAhead];
#pragma unroll
      for (uint32_t u = 0; u < kAhead; ++u) {
        a[u] = *reinterpret_cast<const hd_v4u_a2*>(w + k + u * kStep);
        b[u] = *reinterpret_cast<const hd_v4u_a2*>(h + k + u * kStep);
      }
#pragma unroll
      for (uint32_t u = 0; u < kAhead; ++u) acc = mma<T>(a[u], b[u], acc);
    }
    for (; k < H.d; k += kStep) acc = mma<T>(frag<T>(w - 8 * g, k + 8 * g, H.d), frag<T>(h - 8 * g, k + 8 * g, H.d), acc);
    __syncthreads();
    sh[wave][lane] = acc;
    __syncthreads();
    if (wave) continue;
#pragma unroll
    for (int q = 1; q < kFewWaves; ++q) acc += sh[q][lane];
#pragma unroll
    for (uint32_t q = 0; q < 4; ++q) {
      const uint32_t eq = e0 + 4 * g + q, tq = (uint32_t)__shfl((int)t, (int)(4 * g + q));
      const uint32_t rq = (uint32_t)__shfl((int)rows, (int)(4 * g + q));
      // a listed token's other rows are -inf already
      if (eq < total && i < H.B && (rq >> i & 1)) finish<T, O>(H, r, i, tq, acc[q]);
    }
  }
}

// ---- larger batches: tiles through LDS ---------------------------------------------
// TM tokens x TN rows per workgroup, WM x WN waves, k in steps of 32: a stage is
// 64 B of every row of the tile.  The tokens' stages lie in a ring of kA, the
// rows' in one of kB: weights come from memory and are asked for many steps
// ahead, hidden rows from the caches, fewer steps ahead.  Both are requested
// straight into LDS (16 B per lane), by different waves, each waiting for its
// own: a wave's requests return in order, and the near ones would make the far
// ones wait.  While stage s is multiplied, stage s + 1's operands are read from
// LDS into the other half of the registers; one barrier per stage says that
// every wave's part of the next stage has arrived and that the oldest has been
// read.  The 16-B quarters of a row are exchanged by swz() so that the 16 rows
// of a read spread over the banks (no conflicts are counted).
// Measured in a settled loop: 2048 x 2048 x 128256 958 us = 1125 TFLOP/s (a large
// library product 1383), of it about 12 us per tile of 59 outside the loop, where
// the matrix cores wait; 256 x 4096 x 128256 291 us = 4.1 TB/s with an f32 result
// (307 with a soft mask and cap), 1 x 4096 x 128256 180 us = 5.9 TB/s.
__device__ __forceinline__ uint32_t swz(uint32_t row) { return (row >> 1) & 3u; }

template <int TM_, int TN_, int WM_, int WN_, int kA_, int kB_, int WA_>
struct Tile {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, kA = kA_, kB = kB_;
  static constexpr int kWaves = WM * WN, kThreads = kWaves * 64;
  static constexpr int WA = WA_, WB = kWaves - WA;              // waves that request weights, hidden rows
  static constexpr int LA = TM / 16 / WA, LB = TN / 16 / WB;    // their 1-KB requests per stage
  static constexpr int L = LA > LB ? LA : LB;
  static constexpr int MI = TM / WM / 16, NI = TN / WN / 16;
  static constexpr int kPitch = TM / WM + 4;                    // floats per row of a wave's share of the result
  static constexpr int kRing = (kA * TM + kB * TN) * 64;
  static constexpr int kWords = TM / 32;                        // mask words of a row of the tile
  static constexpr int kSide = TN * (32 + kWords * 4);          // the rows' records and words
  static constexpr int kLds = kRing + kSide;
  static_assert(LA * WA * 16 == TM && LB * WB * 16 == TN, "whole requests per wave");
  static_assert(kWaves * 16 * kPitch * 4 <= kRing, "a wave's 16 result rows fit its share");
  static_assert(kA >= kB && kB >= 3 && (kA - 2) * LA < 63 && kLds <= 160 * 1024, "rings");
};

typedef __attribute__((address_space(3))) void* LdsPtr;
typedef const __attribute__((address_space(1))) void* GlobalPtr;

template <int kLeft>
__device__ __forceinline__ void arrive() {     // all but the newest kLeft requests, then every wave
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLeft) : "memory");
}

template <typename T, typename O, typename C, bool kDirect, bool kList>
__global__ void __launch_bounds__(C::kThreads) k_head_tile(Head H, Need N, uint32_t ntiles) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  RowParams* srow = reinterpret_cast<RowParams*>(lds + C::kRing);
  uint32_t* sword = reinterpret_cast<uint32_t*>(lds + C::kRing + C::TN * 32);
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t wm = wave / C::WN, wn = wave % C::WN;
  uint32_t total = H.V;
  if (N.list) {
    total = listed(H, N);
    if (kList != (total != H.V)) return;       // the other form's turn
  }
  // 8 XCDs take every 8th tile of tokens; the row tiles of one are neighbours in time
  const uint32_t x = blockIdx.x & 7u, y = blockIdx.x >> 3;
  const uint32_t mt = (y / ntiles) * 8 + x, nt = y % ntiles;
  const uint32_t m0 = mt * C::TM, n0 = nt * C::TN;
  if (m0 >= total) return;
  auto token = [&](uint32_t e) {               // entry e of the tile (past the end: the last one, not stored)
    return kList ? N.list[min(m0 + e, total - 1)] : min(m0 + e, H.V - 1);
  };
  // what the epilogue reads of the mask, on its way before the product starts
  const bool masked = H.rp || H.bits;
  if (masked) {
    if constexpr (kList) {                     // [32 rows][token]: which rows each token is in for
      for (uint32_t i = tid; i < C::TN / 32 * C::TM; i += C::kThreads) {
        const uint32_t g = n0 / 32 + i / C::TM, e = m0 + i % C::TM;
        sword[i] = 32 * g < H.B && e < total ? N.rows[(uint64_t)g * N.cap + e] : 0u;
      }
    } else {
      for (uint32_t i = tid; i < C::TN; i += C::kThreads) {
        RowSel r;
        srow[i] = head_row(H, min(n0 + i, H.B - 1), r);
      }
      for (uint32_t i = tid; i < C::TN * C::kWords; i += C::kThreads) {
        const uint32_t row = n0 + i / C::kWords, w = m0 / 32 + i % C::kWords;
        sword[i] = H.bits && row < H.B && 32 * w < H.V ? H.bits[(uint64_t)row * H.ldb + w] : 0u;
      }
    }
  }
  const uint32_t steps = (H.d + 31) / 32, unbroken = H.d / 32;
  const uint32_t full = kDirect ? unbroken : 0;          // stages that are requested straight into LDS

  // this lane's part of request i: 16 B of a row
  const bool forA = wave < (uint32_t)C::WA;
  const uint32_t unit0 = forA ? wave * C::LA : (wave - C::WA) * C::LB;
  const T* src[C::L];
#pragma unroll
  for (int i = 0; i < C::L; ++i) {
    const uint32_t row = (unit0 + i) * 16 + (lane >> 2);
    const T* base = forA ? reinterpret_cast<const T*>(H.weight) + (uint64_t)token(row) * H.ldw
                         : reinterpret_cast<const T*>(H.hidden) + (uint64_t)min(n0 + row, H.B - 1) * H.ldh;
    src[i] = base + ((lane & 3u) ^ swz(row)) * 8;
  }
  auto place = [&](uint32_t s) {        // where this wave's part of stage s goes
    return lds + (forA ? (s % C::kA) * (C::TM * 64) : C::kA * C::TM * 64 + (s % C::kB) * (C::TN * 64)) + unit0 * 1024;
  };
  // tiles start at different k's: weight rows lie a power of two apart, and all
  // workgroups at one k would ask the same few memory channels (350 us for 375
  // at 256 x 4096 x 128256)
  const uint32_t turn0 = unbroken ? mt * 17 % unbroken : 0;
  auto turned = [&](uint32_t s) { return (s + turn0 < unbroken ? s + turn0 : s + turn0 - unbroken) * 32; };
  auto request = [&](uint32_t s) {
    char* at = place(s);
    const uint32_t k = turned(s);
#pragma unroll
    for (int i = 0; i < C::L; ++i)
      if ((C::LA == C::L && C::LB == C::L) || i < (forA ? C::LA : C::LB))
        __builtin_amdgcn_global_load_lds((GlobalPtr)(src[i] + k), (LdsPtr)(at + i * 1024), 16, 0, 0);
  };
  auto fetch = [&](uint32_t s, hd_v4u (&x)[C::L]) {        // a whole stage
    const uint32_t k = turned(s);
#pragma unroll
    for (int i = 0; i < C::L; ++i)
      if (i < (forA ? C::LA : C::LB)) x[i] = *reinterpret_cast<const hd_v4u_a2*>(src[i] + k);
  };
  auto put = [&](uint32_t s, const hd_v4u (&x)[C::L]) {
    char* at = place(s);
#pragma unroll
    for (int i = 0; i < C::L; ++i)
      if (i < (forA ? C::LA : C::LB)) *reinterpret_cast<hd_v4u*>(at + i * 1024 + lane * 16) = x[i];
  };

  hd_v4f acc[C::MI][C::NI];
#pragma unroll
  for (int a = 0; a < C::MI; ++a)
#pragma unroll
    for (int b = 0; b < C::NI; ++b) acc[a][b] = hd_v4f{0, 0, 0, 0};
  const uint32_t frow = lane & 15, fat = frow * 64 + (((lane >> 4) ^ swz(frow)) * 16);
  const uint32_t aoff = wm * (C::TM / C::WM) * 64 + fat;
  const uint32_t boff = C::kA * C::TM * 64 + wn * (C::TN / C::WN) * 64 + fat;
  struct Frags {
    hd_v4u a[C::MI], b[C::NI];
  };
  auto read = [&](Frags& f, uint32_t s) {
    const char* ata = lds + (s % C::kA) * (C::TM * 64) + aoff;
    const char* atb = lds + (s % C::kB) * (C::TN * 64) + boff;
#pragma unroll
    for (int i = 0; i < C::MI; ++i) f.a[i] = *reinterpret_cast<const hd_v4u*>(ata + i * 1024);
#pragma unroll
    for (int i = 0; i < C::NI; ++i) f.b[i] = *reinterpret_cast<const hd_v4u*>(atb + i * 1024);
  };
  auto multiply = [&](const Frags& f) {
#pragma unroll
    for (int a = 0; a < C::MI; ++a)
#pragma unroll
      for (int b = 0; b < C::NI; ++b) acc[a][b] = mma<T>(f.a[a], f.b[b], acc[a][b]);
  };

  Frags f0, f1;
  if (full) {
    const uint32_t mine = forA ? C::kA : C::kB;
    for (uint32_t s = 0; s + 1 < mine && s < full; ++s) request(s);
    if (forA) {
      if (full >= C::kA - 1) arrive<(C::kA - 2) * C::LA>();
      else arrive<0>();
    } else {
      if (full >= C::kB - 1) arrive<(C::kB - 2) * C::LB>();
      else arrive<0>();
    }
    read(f0, 0);
    // stage s + 1 has to be there; this wave's requests of later ones may be under way
    auto step = [&](uint32_t s, const Frags& now, Frags& next) {
      if (forA) {
        if (s + C::kA - 2 < full) arrive<(C::kA - 3) * C::LA>();
        else arrive<0>();
      } else {
        if (s + C::kB - 2 < full) arrive<(C::kB - 3) * C::LB>();
        else arrive<0>();
      }
      if (s + mine - 1 < full) request(s + mine - 1);
      if (s + 1 < full) read(next, s + 1);
      multiply(now);
    };
    auto steady = [&](uint32_t s, const Frags& now, Frags& next) {
      if (forA) arrive<(C::kA - 3) * C::LA>();
      else arrive<(C::kB - 3) * C::LB>();
      request(s + mine - 1);
      read(next, s + 1);
      multiply(now);
      // the next stage's reads in among the products: issued together, they
      // hold the products back until the last of 8 waves has been served
#pragma unroll
      for (int i = 0; i < C::MI + C::NI; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, C::MI * C::NI / (C::MI + C::NI), 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
    };
    uint32_t s = 0;
    for (; s + C::kA < full; s += 2) {        // stages s + kA - 1 and s + kA exist
      steady(s, f0, f1);
      steady(s + 1, f1, f0);
    }
    for (; s + 2 <= full; s += 2) {
      step(s, f0, f1);
      step(s + 1, f1, f0);
    }
    if (s < full) step(s, f0, f1);
  }
  // Rows off 16-B alignment: stages through registers, two at a time, the next
  // two fetched while these are multiplied (2048 x 2052 x 64128: 747 us, one at
  // a time 885; 1 x 1470 x 50265: 63 for 72).  They go to the ring's other two
  // places, which everyone has read by the barrier before.  No branch parts a
  // fetch from its use (the last two are fetched again), or the wait for it
  // moves there.
  uint32_t next = full;
  if constexpr (!kDirect) {
    constexpr uint32_t kHeld = 2;
    static_assert(C::kB >= 2 * kHeld, "two groups of places");
    hd_v4u held[kHeld][C::L];
    const uint32_t groups = unbroken / kHeld;
    if (groups) {
#pragma unroll
      for (uint32_t i = 0; i < kHeld; ++i) fetch(i, held[i]);
      for (uint32_t g = 0; g < groups; ++g) {
#pragma unroll
        for (uint32_t i = 0; i < kHeld; ++i) put(g * kHeld + i, held[i]);
        __syncthreads();
        const uint32_t then = min(g + 1, groups - 1) * kHeld;
#pragma unroll
        for (uint32_t i = 0; i < kHeld; ++i) fetch(then + i, held[i]);
        __builtin_amdgcn_sched_barrier(0);      // else the fetches sink behind the products
#pragma unroll
        for (uint32_t i = 0; i < kHeld; ++i) {
          read(f0, g * kHeld + i);
          multiply(f0);
        }
      }
    }
    next = groups * kHeld;
  }
  for (uint32_t s = next; s < steps; ++s) {      // what is left of the whole stages, and the partial one
    hd_v4u x[C::L];
#pragma unroll
    for (int i = 0; i < C::L; ++i) {
      const uint32_t row = (unit0 + i) * 16 + (lane >> 2), k = ((lane & 3u) ^ swz(row)) * 8;
      if (i < (forA ? C::LA : C::LB)) x[i] = frag<T>(src[i] - k, (s < unbroken ? turned(s) : s * 32) + k, H.d);
    }
    __syncthreads();                    // whoever still reads the ring's place
    put(s, x);
    __syncthreads();
    read(f0, s);
    multiply(f0);
  }

  __syncthreads();                      // the ring is read, the side tables are written
  if constexpr (kList) {
    // Only what the mask leaves in: the rest is -inf already.  A wave first puts
    // its (value, place) pairs together in its share of the LDS, then finishes
    // them 64 at a time: mostly few, and each needs a chain of small reads, which
    // taken one element after the other cost 60 us of 76 at 256 rows and 18000 tokens.
    constexpr uint32_t kBlock = C::MI * 256, kCap = C::kRing / C::kWaves / 48 * 8;      // a block's pairs; a share's
    static_assert(kCap >= kBlock && C::TM * C::TN <= 65536, "a block's pairs fit a share");
    float* val = reinterpret_cast<float*>(lds + wave * kCap * 6);
    uint16_t* at = reinterpret_cast<uint16_t*>(val + kCap);
    uint32_t n = 0;
#pragma unroll
    for (int b = 0; b < C::NI; ++b) {
      const uint32_t in = wn * (C::TN / C::WN) + b * 16 + (lane & 15);
#pragma unroll
      for (int a = 0; a < C::MI; ++a)
#pragma unroll
        for (uint32_t q = 0; q < 4; ++q) {
          const uint32_t e = wm * (C::TM / C::WM) + a * 16 + 4 * (lane >> 4) + q;
          const bool set = sword[(in >> 5) * C::TM + e] >> (in & 31) & 1;
          const uint64_t m = __ballot(set);
          if (set) {
            const uint32_t i = n + __popcll(m & ((1ull << lane) - 1));
            val[i] = acc[a][b][q];
            at[i] = (uint16_t)(in * C::TM + e);
          }
          n += (uint32_t)__popcll(m);
        }
      if (b + 1 < C::NI && n + kBlock <= kCap) continue;
      __syncwarp();
      for (uint32_t i = lane; i < n; i += 64) {
        const uint32_t row = n0 + at[i] / C::TM, t = token(at[i] % C::TM);
        RowSel r;
        head_row(H, row, r);
        finish<T, O>(H, r, row, t, val[i]);
      }
      __syncwarp();
      n = 0;
    }
  } else {
    // A wave's result, 16 rows at a time, turned in its share of the LDS: 4
    // tokens of one row per lane come in, 8 tokens of one row go out.  A lane's
    // 8 tokens are the same in all rows.
    float* turn = reinterpret_cast<float*>(lds) + wave * 16 * C::kPitch;
    constexpr uint32_t kTok = C::TM / C::WM, kPer = kTok / 8, kRows = 64 / kPer;    // lanes and rows per pass
    const uint32_t tt = lane % kPer * 8, t0 = m0 + wm * kTok + tt;
    const bool whole = t0 + 8 <= H.V;
    float bias[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (H.bias && whole) load8f<T>(reinterpret_cast<const T*>(H.bias) + t0, bias);
    const uint32_t uw = masked && H.uni && t0 < H.V ? H.uni[t0 >> 5] : 0u;
#pragma unroll
    for (int b = 0; b < C::NI; ++b) {
#pragma unroll
      for (int a = 0; a < C::MI; ++a)
        *reinterpret_cast<hd_v4f*>(turn + (lane & 15) * C::kPitch + a * 16 + 4 * (lane >> 4)) = acc[a][b];
      __syncwarp();
#pragma unroll
      for (uint32_t i = 0; i < 16 / kRows; ++i) {
        const uint32_t rr = i * kRows + lane / kPer, in = wn * (C::TN / C::WN) + b * 16 + rr, row = n0 + in;
        if (row >= H.B || t0 >= H.V) continue;
        const hd_v4f lo = *reinterpret_cast<const hd_v4f*>(turn + rr * C::kPitch + tt);
        const hd_v4f hi = *reinterpret_cast<const hd_v4f*>(turn + rr * C::kPitch + tt + 4);
        float v[8];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          v[q] = lo[q];
          v[q + 4] = hi[q];
        }
        if (!whole) {                    // the row's end
          RowSel r;
          head_row(H, row, r);
          for (uint32_t q = 0; q < 8; ++q)
            if (t0 + q < H.V) finish<T, O>(H, r, row, t0 + q, v[q]);
          continue;
        }
        finish8<T, O>(H, masked, srow[in], sword[in * C::kWords + ((wm * kTok + tt) >> 5)], uw, row, t0, bias, v);
      }
      __syncwarp();
    }
  }
}

template <typename T, typename O, typename C, bool kList>
int launch_tile(const Head& H, const Need& N, bool direct, uint32_t tokens, hipStream_t s) {
  const uint32_t mt = (tokens + C::TM - 1) / C::TM, nt = (H.B + C::TN - 1) / C::TN;
  const uint64_t grid64 = (uint64_t)((mt + 7) / 8 * 8) * nt;
  if (grid64 * C::kThreads >= (1ull << 32)) {
    set_error("head_scores: %u rows x %u tokens are too many for one call", H.B, H.V);
    return -1;
  }
  const uint32_t grid = (uint32_t)grid64;
  if (direct) {
    FM_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(k_head_tile<T, O, C, true, kList>),
                               hipFuncAttributeMaxDynamicSharedMemorySize, C::kLds));
    k_head_tile<T, O, C, true, kList><<<grid, C::kThreads, C::kLds, s>>>(H, N, nt);
  } else {
    FM_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(k_head_tile<T, O, C, false, kList>),
                               hipFuncAttributeMaxDynamicSharedMemorySize, C::kLds));
    k_head_tile<T, O, C, false, kList><<<grid, C::kThreads, C::kLds, s>>>(H, N, nt);
  }
  return 0;
}

// Rings measured at 256 x 4096 x 128256 and 2048 x 2048 x 128256: (4, 4) 324
// and 964 us, (6, 4) 350 and 1040 (the longer ring's LDS cost the epilogue its
// tables); 256 x 128 tiles of 4 waves, two workgroups per CU, 365 and 1348 (one
// stage ahead is all their LDS allows).  Listed tokens, 18000 of 151936 at
// 256 x 1024: 128 x 256 tiles 59 us (142 workgroups, all at once), 64 x 128 67,
// 64 x 256 70 (a second, nearly empty round).
typedef Tile<256, 256, 2, 4, 4, 4, 4> Tile256;      // more than 128 rows
typedef Tile<256, 128, 4, 2, 7, 4, 4> Tile128;      // 65 .. 128
typedef Tile<256, 64, 4, 1, 8, 4, 2> Tile64;        // up to 64
typedef Tile<128, 256, 2, 4, 6, 4, 4> TileList;     // listed tokens, more than 64 rows
typedef Tile<128, 64, 4, 1, 8, 4, 2> TileList64;    // up to 64
typedef Tile<128, 128, 2, 4, 6, 4, 4> TileHalf;     // small products, below
typedef Tile<64, 64, 2, 2, 4, 4, 2> TileSmall;    // four workgroups per CU

// Whether a product in tiles C is at most one tile per CU.
constexpr uint64_t kCus = 256;
template <typename C>
bool one_round(const Head& H) {
  return ((uint64_t)H.V + C::TM - 1) / C::TM * ((H.B + C::TN - 1) / C::TN) <= kCus;
}

// The whole vocabulary's tiles: the batch's largest, smaller ones as long as
// those too are done in one round (each then takes less, on more CUs).  Measured
// at 256 x 1024 x V, 256 x 256 / 128 x 256 / 128 x 128 / 64 x 64 tiles: V = 12000
// 28 / 20 / 16 / 19 us, 24000 30 / 23 / 28 / 33, 32768 37 / 29 / 37 / 52, 40960
// (320 tiles of 128 x 256) 38 / 47 / 51 / 63; at 472 x 64 x 1171 30 / 17 / 11 /
// 6.5; at 64 x 1024 x V, 256 x 64 / 128 x 64 / 64 x 64: V = 8000 (32 rows) 17 / 12 / 10,
// 32000 26 / 19 / 21, 40000 30 / 34 / 30.  Up to 64 rows of little depth are
// mostly the tiles' beginnings and ends, which overlap where a CU has several
// tiles, 256 x 64 / 64 x 64: 64 x 64 x 151936 17 / 11 us, 16 x 512 x 151936 46 /
// 38, 4 x 768 x 151936 61 / 53, 64 x 768 x 100000 49 / 50, 64 x 1024 x 128256 66
// / 74, 16 x 4096 x 128256 192 / 215.
template <typename T, typename O>
int launch_all(const Head& H, const Need& N, bool direct, hipStream_t s) {
  // (64 tokens a tile reach a launch's 2^32 threads at 2^30 tokens)
  if (one_round<TileSmall>(H) || (H.B <= 64 && H.d <= 768 && H.V <= 1u << 29))
    return launch_tile<T, O, TileSmall, false>(H, N, direct, H.V, s);
  if (H.B <= 64)
    return one_round<TileList64>(H) ? launch_tile<T, O, TileList64, false>(H, N, direct, H.V, s)
                                    : launch_tile<T, O, Tile64, false>(H, N, direct, H.V, s);
  if (one_round<TileHalf>(H)) return launch_tile<T, O, TileHalf, false>(H, N, direct, H.V, s);
  if (H.B <= 128) return launch_tile<T, O, Tile128, false>(H, N, direct, H.V, s);
  return one_round<TileList>(H) ? launch_tile<T, O, TileList, false>(H, N, direct, H.V, s)
                                : launch_tile<T, O, Tile256, false>(H, N, direct, H.V, s);
}

template <typename T, typename O>
int launch_head_t(const Head& H, const Need& N, bool direct, hipStream_t s) {
  if (N.list && H.B <= kFewRows) {
    k_fill_few<O><<<N.chunks, 256, 0, s>>>(H, N);
    k_head_few<T, O><<<std::min<uint32_t>((H.V / 2 + 16) / 16, 1024), kFewWaves * 64, 0, s>>>(H, N);
  } else if (N.list) {
    k_need<<<N.lists, 1024, 0, s>>>(H, N);
    k_fill<O><<<dim3(N.chunks, (H.B + 31) / 32), 256, 0, s>>>(H, N);
    const uint32_t most = std::max(1u, H.V / 2);
    if (H.B > 64 ? launch_tile<T, O, TileList, true>(H, N, direct, most, s)
                 : launch_tile<T, O, TileList64, true>(H, N, direct, most, s))
      return -1;
  }
  return launch_all<T, O>(H, N, direct, s);
}

}  // namespace

namespace {
uint64_t chunks_of(uint64_t V) { return (V + kChunk - 1) / kChunk; }
uint64_t list_cap(uint64_t V) { return (V / 2 + 4) / 4 * 4; }
uint64_t lists_of(uint64_t B, uint64_t V) { return B <= kFewRows ? chunks_of(V) : (V + kSub - 1) / kSub; }
// count[lists + 1], part[chunks * kChunk], then (few rows) rows[chunks * kChunk] or list[cap], rows[B / 32][cap]
uint64_t need_bytes(uint64_t B, uint64_t V) {
  const uint64_t c = chunks_of(V);
  if (B == 0 || c > kMaxChunks) return 0;
  const uint64_t lists = B <= kFewRows ? c * kChunk : (1 + (B + 31) / 32) * list_cap(V);
  return (lists_of(B, V) + 4) / 4 * 16 + c * kChunk * 4 + lists * 4;
}

// Whether the needed tokens are listed first.  Lists cost two or three launches
// (about 6 us up to 16 rows, 20 above) whatever they save, so the whole product
// has to move some bytes for them to pay.  Lists / whole, 0.03 to 1 % of the
// tokens allowed per row, us: 8 x 256 x 16384 (8 MB) 12 / 6, 1 x 512 x 32000 (33
// MB) 11 / 11, 4 x 1024 x 20000 (41 MB) 11 / 13, 1 x 2048 x 32000 (131 MB) 12 /
// 34; 64 x 512 x 20000 (23 MB) 28 / 11, 256 x 512 x 32000 (49 MB) 34 / 20, 32 x
// 1024 x 40000 (84 MB) 29 / 29, 32 x 1024 x 64000 (135 MB) 29 / 34, 64 x 4096 x
// 32000 (266 MB) 54 / 69.
bool lists_pay(uint64_t B, uint64_t V, uint64_t d, uint64_t out_bytes) {
  return V * d * 2 + B * V * out_bytes > (B <= kFewRows ? 36ull << 20 : 96ull << 20);
}

bool aligned16(const void* p, uint64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0; }
}  // namespace

int head_workspace(uint64_t B, uint64_t V, uint64_t* bytes) {
  if (!bytes) {
    set_error("head_workspace: null result");
    return -1;
  }
  *bytes = need_bytes(B, V);
  return 0;
}

int head_scores(const fm_head_args* a, hipStream_t s) {
  if (!a) {
    set_error("head_scores: null");
    return -1;
  }
  if ((a->dtype != 1 && a->dtype != 2) || (a->out_dtype != 0 && a->out_dtype != a->dtype)) {
    set_error("head_scores: dtype codes %d -> %d (bf16 or f16 operands; their dtype or f32 out)", a->dtype,
              a->out_dtype);
    return -1;
  }
  if (a->B > (1u << 20) || a->V > (1u << 30) || a->d > (1u << 30)) {
    set_error("head_scores: B = %llu, V = %llu, d = %llu out of range (B <= 2^20, V, d <= 2^30)",
              (unsigned long long)a->B, (unsigned long long)a->V, (unsigned long long)a->d);
    return -1;
  }
  if (a->B == 0 || a->V == 0) return 0;
  if (!a->d_out || (a->d && (!a->d_hidden || !a->d_weight))) {
    set_error("head_scores: null buffer");
    return -1;
  }
  if (a->ld_hidden < a->d || a->ld_weight < a->d || a->ld_out < a->V || (a->d_residual && a->ld_residual < a->V)) {
    set_error("head_scores: a row stride is shorter than its row");
    return -1;
  }
  if (a->d_bits && a->ld_bits < (a->V + 31) / 32) {
    set_error("head_scores: ld_bits = %llu words < ceil(V / 32)", (unsigned long long)a->ld_bits);
    return -1;
  }
  const float cap = (float)a->softcap;
  if (!(a->softcap >= 0) || !std::isfinite(cap) || (a->softcap > 0 && !std::isfinite(1.f / cap))) {
    set_error("head_scores: softcap %g must be 0 (none) or positive", a->softcap);
    return -1;
  }
  const Head H{a->d_hidden, a->d_weight, a->d_bias, a->d_residual, a->d_out, a->ld_hidden, a->ld_weight,
               a->ld_residual, a->ld_out, (uint32_t)a->B, (uint32_t)a->V, (uint32_t)a->d, a->d_bits, a->ld_bits,
               a->d_unigram_bits, reinterpret_cast<const RowParams*>(a->d_rows), a->eos, cap,
               cap != 0.f ? 1.f / cap : 0.f};
  Need N{};
  const uint64_t need = a->d_bits || a->d_rows ? need_bytes(a->B, a->V) : 0;
  if (need) {
    if (!a->d_ws || (reinterpret_cast<uintptr_t>(a->d_ws) & 15) || a->ws_bytes < need) {
      set_error("head_scores: workspace of %llu bytes at a 16-B aligned address needed, %llu given",
                (unsigned long long)need, (unsigned long long)a->ws_bytes);
      return -1;
    }
  }
  if (need && lists_pay(a->B, a->V, a->d, a->out_dtype == 0 ? 4 : 2)) {
    N.chunks = (uint32_t)chunks_of(a->V);
    N.count = reinterpret_cast<uint32_t*>(a->d_ws);
    N.lists = (uint32_t)lists_of(a->B, a->V);
    N.part = N.count + (N.lists + 4) / 4 * 4;
    N.list = N.part + (uint64_t)N.chunks * kChunk;
    N.cap = (uint32_t)list_cap(a->V);
    N.rows = a->B <= kFewRows ? N.list : N.list + N.cap;
  }
  // 16-B requests straight into LDS need rows on 16 bytes
  const bool direct = a->d >= 32 && a->d % 8 == 0 && aligned16(a->d_hidden, a->ld_hidden) &&
                      aligned16(a->d_weight, a->ld_weight);
  int rc;
  if (a->dtype == 1)
    rc = a->out_dtype == 0 ? launch_head_t<__hip_bfloat16, float>(H, N, direct, s)
                           : launch_head_t<__hip_bfloat16, __hip_bfloat16>(H, N, direct, s);
  else
    rc = a->out_dtype == 0 ? launch_head_t<__half, float>(H, N, direct, s) : launch_head_t<__half, __half>(H, N, direct, s);
  if (rc) return rc;
  FM_HIP(hipGetLastError());
  return 0;
}

}  // namespace fmidx
