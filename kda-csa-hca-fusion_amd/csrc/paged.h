// Rows of the paged HCA cache in their storage formats (gfx950).
//
// bf16, or 8-bit codes with one power of two per row: value = code 2^e, with e
// the least integer for which the row's largest magnitude fits the codes (448 for
// e4m3, 127 for int8), held as the E8M0 code e + 127. A row's scale is a power of
// two because then nothing past the code's own rounding is lost: e4m3 steps are
// relative, and every value (at most 7 significant bits) is exact in bf16, so
// the attention's products see the stored values themselves and no scale enters
// its scores. A row that is written with a non-finite channel is NaN in every channel
// (its norm is no number): code 255 (NaN in E8M0), or bf16 NaNs.
#pragma once

#include "attn_common.h"
#include "kch_kernels.h"

namespace kch {

constexpr int kScaleNan = 255;
constexpr float kRowTiny = 7.8886090522101181e-31f;  // 2^-100: rows below it are held as zeros

template <int FMT> struct PagedFmt;
template <> struct PagedFmt<PF_BF16> {
  typedef bf16_t elem;
};
template <> struct PagedFmt<PF_E4M3> {
  typedef uint8_t elem;
  // 448 = 1.75 2^8: the exponent of amax less 8, one more past 1.75
  static constexpr int top_exp = 8;
  static constexpr uint32_t top_frac = 0x600000u;
};
template <> struct PagedFmt<PF_INT8> {
  typedef uint8_t elem;
  static constexpr int top_exp = 6;  // 127 = 1.984375 2^6
  static constexpr uint32_t top_frac = 0x7e0000u;
};

// Whether a row of this largest magnitude has a channel that is infinite or NaN.
__device__ __forceinline__ bool not_finite(float amax) { return __float_as_uint(amax) >= 0x7f800000u; }

// The E8M0 code of a row whose largest magnitude is amax (NaN or infinite: 255).
template <int FMT>
__device__ __forceinline__ int row_scale_code(float amax) {
  const uint32_t u = __float_as_uint(amax);
  if (not_finite(amax)) return kScaleNan;
  if (amax < kRowTiny) return 127;
  return (int)(u >> 23) - PagedFmt<FMT>::top_exp + ((u & 0x7fffffu) > PagedFmt<FMT>::top_frac ? 1 : 0);
}
// Largest magnitude with NaN kept (fmaxf drops it).
__device__ __forceinline__ float amax_nan(float a, float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu, v = __float_as_uint(a);
  return __uint_as_float(u > v ? u : v);
}

// Four values times 2^-(code - 127) as four codes. A row of code 255 gets zeros.
template <int FMT>
__device__ __forceinline__ uint32_t quant4(float a, float b, float c, float d, int code) {
  if (code == kScaleNan) return 0u;
  const float f = __uint_as_float((uint32_t)(254 - code) << 23);  // 2^(127 - code); 19 <= code <= 249
  if constexpr (FMT == PF_E4M3) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * f, b * f, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c * f, d * f, w, true);
  } else {
    const int i0 = (int)rintf(a * f), i1 = (int)rintf(b * f), i2 = (int)rintf(c * f), i3 = (int)rintf(d * f);
    return (uint32_t)(i0 & 255) | ((uint32_t)(i1 & 255) << 8) | ((uint32_t)(i2 & 255) << 16) |
           ((uint32_t)i3 << 24);
  }
}

// 2^(code - 127), NaN for 255.
__device__ __forceinline__ float row_scale(int code) {
  return __uint_as_float(code == kScaleNan ? 0x7fc00000u : (uint32_t)code << 23);
}

// Rows as the operands of the attention's products, bf16 or fp16 (E). In fp16 the
// 8-bit formats' values are held as a quarter: their largest may be rounded up past fp16's
// (65504 to 65536), and at a quarter every row of values of fp16 fits. `top`: codes
// of larger scales, and bf16 values of larger magnitude (past 65536, itself taken as
// 65504), are rows beyond that, which read as NaN.
template <int FMT, typename E> struct PagedKey {
  static constexpr float held = 1.f;
  static constexpr int top = FMT == PF_BF16 ? 0x7f7f : kScaleNan - 1;
};
template <int FMT> struct PagedKey<FMT, _Float16> {
  static constexpr float held = FMT == PF_BF16 ? 1.f : 0.25f;
  static constexpr int top = FMT == PF_BF16 ? 0x4780 : FMT == PF_E4M3 ? 127 + 9 : 127 + 11;
};

// Four codes as values (exact in bf16, and in fp16 down to its least steps).
template <int FMT, typename E>
__device__ __forceinline__ uint2 dequant4(uint32_t w, float scale) {
  typedef E ex2 __attribute__((ext_vector_type(2)));
  typedef E ex4 __attribute__((ext_vector_type(4)));
  if constexpr (FMT == PF_E4M3) {
    ex2 lo, hi;
    if constexpr (__is_same(E, _Float16)) {
      lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false);
      hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true);
    } else {
      lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false);
      hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true);
    }
    return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
  } else {
    ex4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (E)((float)(int8_t)(w >> (8 * i)) * scale);
    return __builtin_bit_cast(uint2, r);
  }
}
// Two bf16 values of a word as two of E (fp16: towards zero, which only values below
// its normal range meet, and 65536).
template <typename E> __device__ __forceinline__ uint32_t bf16_pair(uint32_t w) {
  if constexpr (__is_same(E, _Float16))
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(__uint_as_float(w << 16),
                                                                   __uint_as_float(w & 0xffff0000u)));
  else
    return w;
}
template <typename E> __device__ __forceinline__ uint4 bf16_pairs(uint4 v) {
  return make_uint4(bf16_pair<E>(v.x), bf16_pair<E>(v.y), bf16_pair<E>(v.z), bf16_pair<E>(v.w));
}

// A sequence of the step: its slot, the rows that the arrays give it, its length (0
// where they do not describe rows of this call: it is passed over), and the tokens
// cached before it. Positions are below 2^32: ctx and len are ints.
struct PagedSeq {
  int slot, row0, end, len;
  uint32_t ctx;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedPool& p, int i) {
  PagedSeq s;
  s.slot = p.slots[i];
  s.row0 = p.cu[i];
  s.end = p.cu[i + 1];
  const int ctx = p.ctx[i];
  s.ctx = (uint32_t)ctx;
  s.len = s.end - s.row0;
  if (s.row0 < 0 || s.end > p.N || s.end < s.row0 || s.slot < 0 || s.slot >= p.n_slots || ctx < 0) s.len = 0;
  return s;
}

// The pool row of a slot's row r, or -1 where the table has no such row or names
// no page of the pool.
__device__ __forceinline__ long long pool_row(const PagedPool& p, const int* table, int width, int slot,
                                              uint32_t r) {
  const uint32_t pg = r >> p.log2page;
  if (pg >= (uint32_t)width) return -1;
  const int page = table[(size_t)slot * width + pg];
  if ((unsigned)page >= (unsigned)p.P) return -1;
  return ((long long)page << p.log2page) + (r & ((1u << p.log2page) - 1));
}

}  // namespace kch
