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

__device__ __forceinline__ float head_mask(const Head& H, const RowSel& r, uint32_t b, uint32_t t) {
  uint32_t hi, lo;
  chunk_codes(r, t >> 3, r.dm ? H.bits[(uint64_t)b * H.ldb + (t >> 5)] : 0u, r.um ? H.uni[t >> 5] : 0u, hi, lo);
  return mask_at(r, hi, lo, t & 7);
}

// one element's epilogue
template <typename T, typename O>
__device__ __forceinline__ void finish(const Head& H, const RowSel& r, uint32_t b, uint32_t t, float x) {
  const float v = head_mask(H, r, b, t);
  O* o = reinterpret_cast<O*>(H.out) + (uint64_t)b * H.ldo + t;
  if (v == -INFINITY) {
    *o = from_f<O>(-INFINITY);
    return;
  }
  if (H.bias) x += to_f<T>(reinterpret_cast<const T*>(H.bias)[t]);
  if (H.cap != 0.f) x = H.cap * tanhf(x * H.inv_cap);
  if (H.residual) x += to_f<O>(reinterpret_cast<const O*>(H.residual)[(uint64_t)b * H.ldr + t]);
  *o = from_f<O>(x + v);
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
    for (int q = 0; q < 4; ++q)
      a[q] = (uint32_t)__builtin_bit_cast(unsigned short, from_f<O>(x[2 * q])) |
             ((uint32_t)__builtin_bit_cast(unsigned short, from_f<O>(x[2 * q + 1])) << 16);
    *reinterpret_cast<hd_v4u_a2*>(p) = a;
  }
}

template <typename T, typename O>
__device__ __forceinline__ void finish8(const Head& H, const RowSel& r, bool masked, uint32_t b, uint32_t t0,
                                        float (&x)[8]) {
  if (t0 + 8 > H.V) {
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q)
      if (t0 + q < H.V) finish<T, O>(H, r, b, t0 + q, x[q]);
    return;
  }
  float y[8];
  if (H.bias) {
    load8f<T>(reinterpret_cast<const T*>(H.bias) + t0, y);
#pragma unroll
    for (int q = 0; q < 8; ++q) x[q] += y[q];
  }
  if (H.cap != 0.f) {
#pragma unroll
    for (int q = 0; q < 8; ++q) x[q] = H.cap * tanhf(x[q] * H.inv_cap);
  }
  if (H.residual) {
    load8f<O>(reinterpret_cast<const O*>(H.residual) + (uint64_t)b * H.ldr + t0, y);
#pragma unroll
    for (int q = 0; q < 8; ++q) x[q] += y[q];
  }
  if (masked) {
    uint32_t hi, lo;
    chunk_codes(r, t0 >> 3, r.dm ? H.bits[(uint64_t)b * H.ldb + (t0 >> 5)] : 0u, r.um ? H.uni[t0 >> 5] : 0u, hi, lo);
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q) {
      const float v = mask_at(r, hi, lo, q);
      x[q] = v == -INFINITY ? -INFINITY : x[q] + v;
    }
  }
  store8f<O>(reinterpret_cast<O*>(H.out) + (uint64_t)b * H.ldo + t0, x);
}

// ---- which weight rows are needed ---------------------------------------------
// A token's weight row is needed if its mask value is above -inf in some row.
// k_need: per chunk of 2048 tokens, the needed ones listed in order (at
// list[2048 chunk ..]) and counted.  k_fill: -inf where the mask says so, and
// the chunks' lists joined (the order stays); neither does anything when more
// than half of the vocabulary is needed: then the product runs over all of it
// and writes every score itself, which costs less than gathering.
constexpr uint32_t kChunk = 2048;
constexpr uint32_t kMaxChunks = 512;        // lists up to 2^20 tokens; above, no list is made

struct Need {
  uint32_t* count;       // [chunks]
  uint32_t* part;        // [chunks * kChunk]
  uint32_t* list;        // [V]; null: no lists
  uint32_t chunks;
};

// the tokens of word w that row b's mask leaves in
__device__ __forceinline__ uint32_t need_word(const Head& H, const RowParams& p, const RowSel& r, uint32_t b,
                                              uint32_t w) {
  const uint32_t d = (r.dm ? H.bits[(uint64_t)b * H.ldb + w] : 0u) | (w == r.js >> 2 ? r.sb << (8 * (r.js & 3)) : 0u);
  const uint32_t u = r.um ? H.uni[w] : 0u;
  const uint32_t e = w == r.je >> 2 ? r.eb << (8 * (r.je & 3)) : 0u;
  uint32_t x = p.base != -INFINITY ? ~0u : 0u;
  x = (x & ~u) | (p.v_uni != -INFINITY ? u : 0u);
  x = (x & ~d) | (p.v_dist != -INFINITY ? d : 0u);
  return (x & ~e) | (p.v_eos != -INFINITY ? e : 0u);
}

__global__ void __launch_bounds__(1024) k_need(Head H, Need N) {
  __shared__ uint32_t sh[16][64];
  const uint32_t lane = threadIdx.x & 63, grp = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t w = blockIdx.x * (kChunk / 32) + lane;
  uint32_t x = 0;
  if (32 * w < H.V)
    for (uint32_t b = grp; b < H.B; b += 16) {
      RowSel r;
      const RowParams p = head_row(H, b, r);
      x |= need_word(H, p, r, b, w);
    }
  sh[grp][lane] = x;
  __syncthreads();
  if (grp) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) x |= sh[i][lane];
  if (32 * w < H.V && H.V - 32 * w < 32) x &= (1u << (H.V - 32 * w)) - 1;
  if (32 * w >= H.V) x = 0;
  uint32_t upto = __popc(x);
  const uint32_t mine = upto;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = (uint32_t)__shfl_up((int)upto, d);
    if (lane >= (uint32_t)d) upto += o;
  }
  if (lane == 63) N.count[blockIdx.x] = upto;
  uint32_t* at = N.part + (uint64_t)blockIdx.x * kChunk + (upto - mine);
  for (; x; x &= x - 1) *at++ = 32 * w + __ffs((int)x) - 1;
}

// the sum of count[0 .. n) by the whole workgroup (n <= kMaxChunks)
__device__ __forceinline__ uint32_t count_sum(const Need& N, uint32_t n, uint32_t* sh) {
  uint32_t s = 0;
  for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) s += N.count[i];
#pragma unroll
  for (int d = 32; d; d >>= 1) s += (uint32_t)__shfl_xor((int)s, d);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  s = 0;
  for (uint32_t i = 0; i < blockDim.x / 64; ++i) s += sh[i];
  __syncthreads();
  return s;
}

// how many tokens are listed; V: all of them, without a list
__device__ __forceinline__ uint32_t listed(const Head& H, const Need& N, uint32_t* sh) {
  if (!N.list) return H.V;
  const uint32_t s = count_sum(N, N.chunks, sh);
  return 2 * s > H.V ? H.V : s;
}

template <typename O>
__global__ void __launch_bounds__(256) k_fill(Head H, Need N) {
  __shared__ uint32_t sh[16];
  if (listed(H, N, sh) == H.V) return;
  const uint32_t flat = blockIdx.y * gridDim.x + blockIdx.x;
  for (uint32_t c = flat; c < N.chunks; c += gridDim.x * gridDim.y) {
    const uint32_t at = count_sum(N, c, sh), n = N.count[c];
    for (uint32_t i = threadIdx.x; i < n; i += 256) N.list[at + i] = N.part[(uint64_t)c * kChunk + i];
  }
  const uint32_t chunks = (H.V + 7) / 8;
  for (uint32_t b = blockIdx.y; b < H.B; b += gridDim.y) {
    RowSel r;
    const RowParams p = head_row(H, b, r);
    O* o = reinterpret_cast<O*>(H.out) + (uint64_t)b * H.ldo;
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      const uint32_t j = blockIdx.x * 1024 + u * 256 + threadIdx.x;
      if (j >= chunks) continue;
      const uint32_t in = need_word(H, p, r, b, j >> 2) >> (8 * (j & 3)) & 0xFFu;
      if (in == 0 && 8 * j + 8 <= H.V) {
        const float x[8] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY};
        store8f<O>(o + 8 * j, x);
      } else {
        for (uint32_t q = 0; q < 8; ++q)
          if (8 * j + q < H.V && !(in >> q & 1)) o[8 * j + q] = from_f<O>(-INFINITY);
      }
    }
  }
}

// ---- up to 16 rows of the batch --------------------------------------------------
// 16 tokens per workgroup at a time, its waves each a share of k straight from
// memory into the matrix cores (a lane's 8 k's are 16 B of one row), joined in LDS.
constexpr int kFewWaves = 4;

template <typename T, typename O>
__global__ void __launch_bounds__(kFewWaves * 64) k_head_few(Head H, Need N) {
  __shared__ hd_v4f sh[kFewWaves][64];
  __shared__ uint32_t shc[16];
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const uint32_t total = listed(H, N, shc);
  const bool gather = total != H.V;
  // lanes without a row or a token of their own repeat a valid one; their results are not stored
  const T* h = reinterpret_cast<const T*>(H.hidden) + (uint64_t)min(i, H.B - 1) * H.ldh + 8 * g;
  RowSel r;
  if (i < H.B) head_row(H, i, r);
  constexpr uint32_t kStep = kFewWaves * 32, kAhead = 8;       // requests in flight per operand and lane
  for (uint32_t e0 = blockIdx.x * 16; e0 < total; e0 += gridDim.x * 16) {
    const uint32_t e = min(e0 + i, total - 1);
    const uint32_t t = gather ? N.list[e] : e;
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
      const uint32_t tq = (uint32_t)__shfl((int)t, (int)(4 * g + q));
      if (e0 + 4 * g + q < total && i < H.B) finish<T, O>(H, r, i, tq, acc[q]);
    }
  }
}

// ---- larger batches: tiles through LDS ---------------------------------------------
// TM tokens x TN rows per workgroup, WM x WN waves, k in steps of 32: a stage
// is 64 B of every row of the tile, kStages of them in a ring.  Stage s + kStages
// - 1 is requested (straight into LDS, 16 B per lane) while stage s is
// multiplied, and stage s + 1's operands are read from LDS into the other half
// of the registers meanwhile; one barrier per stage says that every wave's part
// of the next stage has arrived and that the oldest stage has been read.
// The 16-B quarters of a row are exchanged by swz() so that the 16 rows of a
// read spread over the banks.
__device__ __forceinline__ uint32_t swz(uint32_t row) { return (row >> 1) & 3u; }

template <int TM_, int TN_, int WM_, int WN_, int kStages_>
struct Tile {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, kStages = kStages_;
  static constexpr int kThreads = WM * WN * 64;
  static constexpr int MI = TM / WM / 16, NI = TN / WN / 16;
  static constexpr int kStage = (TM + TN) * 64;                 // bytes
  static constexpr int kLoads = (TM + TN) / 16 / (WM * WN);     // 1-KB requests per wave and stage
  static constexpr int kPitch = TM / WM + 4;                    // floats per row of a wave's share of the result
  static constexpr int kLds = kStages * kStage;
  static_assert((TM + TN) / 16 % (WM * WN) == 0, "whole requests per wave");
  static_assert(WM * WN * 16 * kPitch * 4 <= kLds, "a wave's 16 result rows fit its share");
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
  __shared__ uint32_t shc[16];
  __shared__ uint32_t shl[kList ? C::TM : 1];
  constexpr int S = C::kStages;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t wm = wave / C::WN, wn = wave % C::WN;
  uint32_t total = H.V;
  if (N.list) {
    total = listed(H, N, shc);
    if (kList != (total != H.V)) return;       // the other form's turn
  }
  // 8 XCDs take every 8th tile of tokens; the row tiles of one are neighbours in time
  const uint32_t x = blockIdx.x & 7u, y = blockIdx.x >> 3;
  const uint32_t mt = (y / ntiles) * 8 + x, nt = y % ntiles;
  const uint32_t m0 = mt * C::TM, n0 = nt * C::TN;
  if (m0 >= total) return;
  if constexpr (kList) {
    for (uint32_t i = tid; i < C::TM; i += C::kThreads) shl[i] = N.list[min(m0 + i, total - 1)];
    __syncthreads();
  }
  const uint32_t steps = (H.d + 31) / 32;
  const uint32_t full = kDirect ? H.d / 32 : 0;       // stages that are requested straight into LDS

  // this lane's part of request i: 16 B of a row (a row past the end repeats the last one; it is not stored)
  const T* src[C::kLoads];
#pragma unroll
  for (int i = 0; i < C::kLoads; ++i) {
    const uint32_t u = wave * C::kLoads + i, row = u * 16 + (lane >> 2);
    const uint32_t k = ((lane & 3u) ^ swz(row)) * 8;
    const T* base;
    if (row < (uint32_t)C::TM) {
      const uint32_t t = kList ? shl[row] : min(m0 + row, H.V - 1);
      base = reinterpret_cast<const T*>(H.weight) + (uint64_t)t * H.ldw;
    } else {
      base = reinterpret_cast<const T*>(H.hidden) + (uint64_t)min(n0 + row - C::TM, H.B - 1) * H.ldh;
    }
    src[i] = base + k;
  }
  auto request = [&](uint32_t s) {      // stage s into its place in the ring
    char* at = lds + (s % S) * C::kStage + wave * C::kLoads * 1024;
#pragma unroll
    for (int i = 0; i < C::kLoads; ++i)
      __builtin_amdgcn_global_load_lds((GlobalPtr)(src[i] + s * 32), (LdsPtr)(at + i * 1024), 16, 0, 0);
  };
  hd_v4u held[C::kLoads];               // a stage on its way through registers
  auto fetch = [&](uint32_t s) {
#pragma unroll
    for (int i = 0; i < C::kLoads; ++i) {
      const uint32_t row = (wave * C::kLoads + i) * 16 + (lane >> 2), k = ((lane & 3u) ^ swz(row)) * 8;
      held[i] = frag<T>(src[i] - k, s * 32 + k, H.d);
    }
  };
  auto put = [&](uint32_t s) {
    char* at = lds + (s % S) * C::kStage + wave * C::kLoads * 1024;
#pragma unroll
    for (int i = 0; i < C::kLoads; ++i) *reinterpret_cast<hd_v4u*>(at + i * 1024 + lane * 16) = held[i];
  };

  hd_v4f acc[C::MI][C::NI];
#pragma unroll
  for (int a = 0; a < C::MI; ++a)
#pragma unroll
    for (int b = 0; b < C::NI; ++b) acc[a][b] = hd_v4f{0, 0, 0, 0};
  const uint32_t frow = lane & 15, fat = frow * 64 + (((lane >> 4) ^ swz(frow)) * 16);
  const uint32_t aoff = wm * (C::TM / C::WM) * 64 + fat, boff = (C::TM + wn * (C::TN / C::WN)) * 64 + fat;
  struct Frags {
    hd_v4u a[C::MI], b[C::NI];
  };
  auto read = [&](Frags& f, uint32_t s) {
    const char* at = lds + (s % S) * C::kStage;
#pragma unroll
    for (int i = 0; i < C::MI; ++i) f.a[i] = *reinterpret_cast<const hd_v4u*>(at + aoff + i * 1024);
#pragma unroll
    for (int i = 0; i < C::NI; ++i) f.b[i] = *reinterpret_cast<const hd_v4u*>(at + boff + i * 1024);
  };
  auto multiply = [&](const Frags& f) {
#pragma unroll
    for (int a = 0; a < C::MI; ++a)
#pragma unroll
      for (int b = 0; b < C::NI; ++b) acc[a][b] = mma<T>(f.a[a], f.b[b], acc[a][b]);
  };

  Frags f0, f1;
  if (full) {
#pragma unroll
    for (uint32_t s = 0; s < S - 1; ++s)
      if (s < full) request(s);
    if (full >= S - 1) arrive<(S - 2) * C::kLoads>();
    else arrive<0>();
    read(f0, 0);
    auto step = [&](uint32_t s, const Frags& now, Frags& next) {
      // the requests of stages s + 2 .. s + S - 2 may still be under way
      if (s + S - 2 < full) arrive<(S - 3) * C::kLoads>();
      else arrive<0>();
      if (s + S - 1 < full) request(s + S - 1);
      if (s + 1 < full) read(next, s + 1);
      multiply(now);
    };
    auto steady = [&](uint32_t s, const Frags& now, Frags& next) {
      arrive<(S - 3) * C::kLoads>();
      request(s + S - 1);
      read(next, s + 1);
      multiply(now);
    };
    uint32_t s = 0;
    for (; s + S < full; s += 2) {        // both stages s + S - 1 and s + S exist
      steady(s, f0, f1);
      steady(s + 1, f1, f0);
    }
    for (; s + 2 <= full; s += 2) {
      step(s, f0, f1);
      step(s + 1, f1, f0);
    }
    if (s < full) step(s, f0, f1);
  }
  // stages through registers: the last, partial one, or (rows off 16-B alignment) all of them
  if (full < steps) {
    fetch(full);
    for (uint32_t s = full; s < steps; ++s) {
      __syncthreads();                  // whoever still reads the ring's place
      put(s);
      __syncthreads();
      if (s + 1 < steps) fetch(s + 1);
      read(f0, s);
      multiply(f0);
    }
  }

  if constexpr (kList) {
    // only what the mask leaves in: the rest is -inf already
#pragma unroll
    for (int b = 0; b < C::NI; ++b) {
      const uint32_t row = n0 + wn * (C::TN / C::WN) + b * 16 + (lane & 15);
      if (row >= H.B) continue;
      RowSel r;
      const RowParams p = head_row(H, row, r);
#pragma unroll
      for (int a = 0; a < C::MI; ++a)
#pragma unroll
        for (uint32_t q = 0; q < 4; ++q) {
          const uint32_t e = wm * (C::TM / C::WM) + a * 16 + 4 * (lane >> 4) + q;
          if (m0 + e >= total) continue;
          const uint32_t t = shl[e];
          if (need_word(H, p, r, row, t >> 5) >> (t & 31) & 1) finish<T, O>(H, r, row, t, acc[a][b][q]);
        }
    }
  } else {
    // A wave's result, 16 rows at a time, turned in its share of the LDS: 4
    // tokens of one row per lane come in, 8 tokens of one row go out.
    __syncthreads();
    float* turn = reinterpret_cast<float*>(lds) + wave * 16 * C::kPitch;
    constexpr uint32_t kTok = C::TM / C::WM;
    const bool masked = H.rp || H.bits;
#pragma unroll
    for (int b = 0; b < C::NI; ++b) {
#pragma unroll
      for (int a = 0; a < C::MI; ++a)
        *reinterpret_cast<hd_v4f*>(turn + (lane & 15) * C::kPitch + a * 16 + 4 * (lane >> 4)) = acc[a][b];
      __syncwarp();
      for (uint32_t c = lane; c < 16 * (kTok / 8); c += 64) {
        const uint32_t rr = c / (kTok / 8), tt = c % (kTok / 8) * 8;
        const uint32_t row = n0 + wn * (C::TN / C::WN) + b * 16 + rr, t0 = m0 + wm * kTok + tt;
        if (row >= H.B || t0 >= H.V) continue;
        float v[8];
        const hd_v4f lo = *reinterpret_cast<const hd_v4f*>(turn + rr * C::kPitch + tt);
        const hd_v4f hi = *reinterpret_cast<const hd_v4f*>(turn + rr * C::kPitch + tt + 4);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          v[q] = lo[q];
          v[q + 4] = hi[q];
        }
        RowSel r;                        // without a mask: no flags, and no memory behind them
        head_row(H, row, r);
        finish8<T, O>(H, r, masked, row, t0, v);
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

typedef Tile<256, 256, 2, 4, 4> Tile256;     // more than 128 rows
typedef Tile<256, 128, 4, 2, 4> Tile128;     // 65 .. 128
typedef Tile<256, 64, 4, 1, 4> Tile64;       // 17 .. 64
typedef Tile<64, 256, 1, 4, 4> TileList;     // listed tokens

template <typename T, typename O>
int launch_head_t(const Head& H, const Need& N, bool direct, hipStream_t s) {
  if (N.list) {
    k_need<<<N.chunks, 1024, 0, s>>>(H, N);
    k_fill<O><<<dim3((H.V + 8191) / 8192, std::min<uint32_t>(H.B, 32768)), 256, 0, s>>>(H, N);
  }
  if (H.B <= 16) {
    k_head_few<T, O><<<std::min<uint32_t>((H.V + 15) / 16, 1u << 16), kFewWaves * 64, 0, s>>>(H, N);
    return 0;
  }
  if (N.list && launch_tile<T, O, TileList, true>(H, N, direct, std::max(1u, H.V / 2), s)) return -1;
  if (H.B > 128) return launch_tile<T, O, Tile256, false>(H, N, direct, H.V, s);
  if (H.B > 64) return launch_tile<T, O, Tile128, false>(H, N, direct, H.V, s);
  return launch_tile<T, O, Tile64, false>(H, N, direct, H.V, s);
}

}  // namespace

namespace {
uint64_t chunks_of(uint64_t V) { return (V + kChunk - 1) / kChunk; }
uint64_t need_bytes(uint64_t B, uint64_t V) {
  const uint64_t c = chunks_of(V);
  return B == 0 || c > kMaxChunks ? 0 : (c + 3) / 4 * 16 + 2 * c * kChunk * 4;
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
    N.chunks = (uint32_t)chunks_of(a->V);
    N.count = reinterpret_cast<uint32_t*>(a->d_ws);
    N.part = N.count + (N.chunks + 3) / 4 * 4;
    N.list = N.part + (uint64_t)N.chunks * kChunk;
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
