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

// 8 elements of a row from k on; zeros from d on (and for no row)
template <typename T>
__device__ __forceinline__ hd_v4u frag(const T* row, uint32_t k, uint32_t d) {
  hd_v4u x = {0, 0, 0, 0};
  if (!row || k >= d) return x;
  if (k + 8 <= d) return *reinterpret_cast<const hd_v4u_a2*>(row + k);
  const unsigned short* p = reinterpret_cast<const unsigned short*>(row + k);
#pragma unroll
  for (uint32_t q = 0; q < 8; ++q)
    if (k + q < d) x[q >> 1] |= (uint32_t)p[q] << (16 * (q & 1));
  return x;
}

// the mask values' rules of batch row b
__device__ __forceinline__ RowSel head_sel(const Head& H, uint32_t b) {
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
  return row_sel(p, H.V, H.eos);
}

__device__ __forceinline__ float head_mask(const Head& H, const RowSel& r, uint32_t b, uint32_t t) {
  uint32_t hi, lo;
  chunk_codes(r, t >> 3, r.dm ? H.bits[(uint64_t)b * H.ldb + (t >> 5)] : 0u, r.um ? H.uni[t >> 5] : 0u, hi, lo);
  return mask_at(r, hi, lo, t & 7);
}

// one element's epilogue
template <typename T, typename O>
__device__ __forceinline__ void finish(const Head& H, const RowSel& r, uint32_t b, uint32_t t, float x) {
  if (H.bias) x += to_f<T>(reinterpret_cast<const T*>(H.bias)[t]);
  if (H.cap != 0.f) x = H.cap * tanhf(x * H.inv_cap);
  const float v = head_mask(H, r, b, t);
  if (H.residual) x += to_f<O>(reinterpret_cast<const O*>(H.residual)[(uint64_t)b * H.ldr + t]);
  x = v == -INFINITY ? -INFINITY : x + v;
  reinterpret_cast<O*>(H.out)[(uint64_t)b * H.ldo + t] = from_f<O>(x);
}

constexpr int kFewWaves = 4;

// 16 tokens x 16 rows per workgroup, its waves each a share of k, joined in LDS.
template <typename T, typename O>
__global__ void __launch_bounds__(kFewWaves * 64) k_head_few(Head H) {
  __shared__ hd_v4f sh[kFewWaves][64];
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const uint32_t t0 = blockIdx.x * 16, b0 = blockIdx.y * 16;
  const T* w = t0 + i < H.V ? reinterpret_cast<const T*>(H.weight) + (uint64_t)(t0 + i) * H.ldw : nullptr;
  const T* h = b0 + i < H.B ? reinterpret_cast<const T*>(H.hidden) + (uint64_t)(b0 + i) * H.ldh : nullptr;
  hd_v4f acc = {0, 0, 0, 0};
  for (uint32_t k = wave * 32; k < H.d; k += kFewWaves * 32)
    acc = mma<T>(frag<T>(w, k + 8 * g, H.d), frag<T>(h, k + 8 * g, H.d), acc);
  sh[wave][lane] = acc;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int q = 1; q < kFewWaves; ++q) acc += sh[q][lane];
  const uint32_t b = b0 + i;
  if (b >= H.B) return;
  const RowSel r = head_sel(H, b);
#pragma unroll
  for (uint32_t q = 0; q < 4; ++q) {
    const uint32_t t = t0 + 4 * g + q;
    if (t < H.V) finish<T, O>(H, r, b, t, acc[q]);
  }
}

template <typename T, typename O>
void launch_head_t(const Head& H, hipStream_t s) {
  k_head_few<T, O><<<dim3((H.V + 15) / 16, (H.B + 15) / 16), kFewWaves * 64, 0, s>>>(H);
}

}  // namespace

int head_workspace(uint64_t, uint64_t, uint64_t* bytes) {
  if (!bytes) {
    set_error("head_workspace: null result");
    return -1;
  }
  *bytes = 0;
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
  if (a->dtype == 1) {
    if (a->out_dtype == 0) launch_head_t<__hip_bfloat16, float>(H, s);
    else launch_head_t<__hip_bfloat16, __hip_bfloat16>(H, s);
  } else {
    if (a->out_dtype == 0) launch_head_t<__half, float>(H, s);
    else launch_head_t<__half, __half>(H, s);
  }
  FM_HIP(hipGetLastError());
  return 0;
}

}  // namespace fmidx
