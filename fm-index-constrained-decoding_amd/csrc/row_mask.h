// row_mask.h -- a row's mask value per token, shared by the kernels that read
// or write scores under a document constraint (epilogue.hip, losses.hip,
// head.hip): the 32-byte row records of fm_row_params, the packed allowed and
// all_unigrams bits, and the scores dtypes' conversions.
#pragma once
#include "fmidx_internal.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace fmidx {
namespace {

// row flags
constexpr uint32_t kUseBits = 1u;      // allowed tokens from the bit row
constexpr uint32_t kUnigram = 2u;      // all_unigrams get v_uni
constexpr uint32_t kEos = 4u;          // eos gets v_eos (last, overrides)
constexpr uint32_t kSpecial = 8u;      // the single token `special` is the distinct set

struct RowParams {
  float base, v_dist, v_uni, v_eos;
  uint32_t flags;
  int32_t pad;
  int64_t special;
};

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f<__hip_bfloat16>(__hip_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __hip_bfloat16 from_f<__hip_bfloat16>(float x) { return __float2bfloat16(x); }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half(x); }

template <typename T>
__device__ __forceinline__ uint32_t add16(uint32_t h, float m) {   // one 16-bit element, as bits
  const T x = __builtin_bit_cast(T, (unsigned short)h);
  return (uint32_t)__builtin_bit_cast(unsigned short, from_f<T>(to_f<T>(x) + m));
}

// A row's mask values and rules as uniform constants.  The mask value of a
// token follows the reference's assignment order -- base, all_unigrams,
// distinct (the allowed bits, plus `special`), eos -- and is selected with
// bit operations on the four values' f32 bits (a select between struct
// fields was compiled as an LDS copy of the struct and an indexed read per
// token).  eos and `special` are found by chunk index, not by a 64-bit
// compare per token.
struct RowSel {
  uint32_t fb, fu, fd, fe;   // base, v_uni, v_dist, v_eos (f32 bits)
  uint32_t dm, um;           // 0xFF if the allowed / unigram bits apply, else 0
  uint32_t je, eb;           // chunk holding eos and its bit (je = ~0: none)
  uint32_t js, sb;           // the same for `special`
};

__device__ __forceinline__ RowSel row_sel(const RowParams& p, uint32_t V, int64_t eos) {
  RowSel r;
  r.fb = __float_as_uint(p.base);
  r.fu = __float_as_uint(p.v_uni);
  r.fd = __float_as_uint(p.v_dist);
  r.fe = __float_as_uint(p.v_eos);
  r.dm = (p.flags & kUseBits) ? 0xFFu : 0u;
  r.um = (p.flags & kUnigram) ? 0xFFu : 0u;
  const bool he = (p.flags & kEos) && eos >= 0 && eos < (int64_t)V;
  r.je = he ? (uint32_t)(eos >> 3) : ~0u;
  r.eb = he ? 1u << (uint32_t)(eos & 7) : 0u;
  const bool hs = (p.flags & kSpecial) && p.special >= 0 && p.special < (int64_t)V;
  r.js = hs ? (uint32_t)(p.special >> 3) : ~0u;
  r.sb = hs ? 1u << (uint32_t)(p.special & 7) : 0u;
  return r;
}

// Chunk j (tokens 8 j .. 8 j + 7): bit k of H = "token k gets v_dist or
// v_eos", bit k of L = "the upper value of its pair" (v_eos over v_dist,
// v_uni over base).  dw / uw: the bit words holding the chunk's byte.
__device__ __forceinline__ void chunk_codes(const RowSel& r, uint32_t j, uint32_t dw, uint32_t uw, uint32_t& H,
                                            uint32_t& L) {
  const uint32_t sh = (8 * j) & 31u;
  const uint32_t d = ((dw >> sh) & r.dm) | (j == r.js ? r.sb : 0u);
  const uint32_t u = (uw >> sh) & r.um;
  const uint32_t e = j == r.je ? r.eb : 0u;
  H = d | e;
  L = e | (u & ~H);
}

__device__ __forceinline__ uint32_t bit_mask(uint32_t X, uint32_t k) {   // all ones iff bit k of X
  return (uint32_t)((int32_t)(X << (31 - k)) >> 31);
}
__device__ __forceinline__ uint32_t bit_sel(uint32_t M, uint32_t a, uint32_t b) { return (a & M) | (b & ~M); }

__device__ __forceinline__ float mask_at(const RowSel& r, uint32_t H, uint32_t L, uint32_t k) {
  const uint32_t mh = bit_mask(H, k), ml = bit_mask(L, k);
  return __uint_as_float(bit_sel(mh, bit_sel(ml, r.fe, r.fd), bit_sel(ml, r.fu, r.fb)));
}

template <typename T>
__device__ __forceinline__ float bits16_to_f(uint32_t h) {
  return to_f<T>(__builtin_bit_cast(T, (unsigned short)h));
}
template <typename T>
__device__ __forceinline__ uint32_t f_to_bits16(float x) {
  return (uint32_t)__builtin_bit_cast(unsigned short, from_f<T>(x));
}

// two f32 rounded to nearest even and packed (one instruction for bf16)
template <typename T>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (std::is_same_v<T, __hip_bfloat16>) {
    typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
    typedef float v2f __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{a, b}), v2bf));
  } else {
    return f_to_bits16<T>(a) | (f_to_bits16<T>(b) << 16);
  }
}
// All ones where bit q (a constant) of x is set: one bit-field extract.  As an
// asm because the compiler takes such masks apart again, into a test, a compare
// and a conditional move per select.
__device__ __forceinline__ uint32_t sign_bit(uint32_t x, uint32_t q) {
  uint32_t r;
  asm("v_bfe_i32 %0, %1, %2, 1" : "=v"(r) : "v"(x), "n"(q));
  return r;
}
// a where the mask is set, else b
__device__ __forceinline__ uint32_t pick(uint32_t mask, uint32_t a, uint32_t b) {
  uint32_t r;
  asm("v_bfi_b32 %0, %1, %2, %3" : "=v"(r) : "v"(mask), "v"(a), "v"(b));
  return r;
}
}  // namespace
}  // namespace fmidx
