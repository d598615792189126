// The 8-bit cache format, shared by the kernels that write it, read it back and attend over it (gfx950).
//
// One layer's K (and V) is codes [pages][16][heads][D], int8 or e4m3 (the OCP float8 with a largest value of
// 448), and one exponent byte for every 32 dims of a token's head, [pages][heads][ceil(D/32)][16]: a code c in
// a block with byte s stands for c * 2^(s - 127). Powers of two make both directions exact: scaling a row never
// rounds, so a code is one rounding of the value away from it, and the exponents' limits (QuantFmt::kLow,
// kHigh) keep every value c * 2^e a number of fp16 and of bf16, so that reading back never rounds and
// the matrix cores take the values as fp16 whatever the model's type. The byte 255 marks a block that held a NaN
// or an infinity (codes 0, or e4m3's NaN); it reads as NaN. The sixteen tokens of a block lie together,
// because a lane of the attention kernels holds four tokens of one block: one dword.
#pragma once

#include "ukv_common.h"

namespace ukv {

// One layer of the cache; strides in bytes (= elements): page, token, head of the codes; page, head,
// block of the exponents.
struct QuantLayer {
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* ks;
  const uint8_t* vs;
  int64_t k_sp, k_st, k_sh, v_sp, v_st, v_sh;
  int64_t ks_sp, ks_sh, ks_sb, vs_sp, vs_sh, vs_sb;
  int num_pages;
};

constexpr int kQuantBlock = 32;  // dims that share an exponent
constexpr int kCache16 = -1;     // in place of a format: pages of the model's type

template <int QF> struct QuantFmt;

// kLow: the step 2^e of the smallest exponent is fp16's smallest number (e4m3: 2^-9 of it). kHigh: the
// largest code times 2^e stays below fp16's end. kFraction: the fraction bits of the largest code.
template <> struct QuantFmt<UKV_CACHE_INT8> {
  static constexpr float kTop = 127.f;
  static constexpr int kTopPower = 6, kLow = -24, kHigh = 9;
  static constexpr uint32_t kFraction = 0x7E0000u, kNanCodes = 0u;
};
template <> struct QuantFmt<UKV_CACHE_FP8> {
  static constexpr float kTop = 448.f;
  static constexpr int kTopPower = 8, kLow = -15, kHigh = 7;
  static constexpr uint32_t kFraction = 0x600000u, kNanCodes = 0x7F7F7F7Fu;
};

// The exponent of a block whose largest magnitude is the finite `largest`: the smallest e with
// kTop * 2^e >= largest, within the limits. (The fp32 exponent, one more where the fraction is above kTop's.)
template <int QF> __device__ __forceinline__ int quant_exponent(float largest) {
  using F = QuantFmt<QF>;
  const int p = (int)((__float_as_uint(largest) + (0x7FFFFFu - F::kFraction)) >> 23) - 127 - F::kTopPower;
  return min(max(p, F::kLow), F::kHigh);
}

// Four values as four codes: RNE of x * 2^-e, `inv` = 2^-e (exact; a magnitude beyond kTop, which the
// highest exponent alone allows, becomes kTop).
template <int QF> __device__ __forceinline__ uint32_t quant_codes4(const float (&x)[4], float inv) {
  constexpr float top = QuantFmt<QF>::kTop;
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = __builtin_amdgcn_fmed3f(x[i] * inv, -top, top);
  if constexpr (QF == UKV_CACHE_INT8) {
    // 1.5 * 2^23 has a step of one: the sum's low byte is the rounded value in two's complement
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(y[i] + 12582912.f);
    const uint32_t lo = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(u[3], u[2], 0x0c0c0400u);
    return lo | (hi << 16);
  } else {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
  }
}

// 2^(s - 127) of an exponent byte in fp32; NaN for 255.
__device__ __forceinline__ float quant_scale(uint32_t s) {
  return __uint_as_float(s == 255u ? 0x7FC00000u : s << 23);
}

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Four codes as two packed pairs of fp16 values, code * scale (scale: quant_scale of their block).
//   int8: u = code ^ 0x80 is code + 128; the fp16 with bits 0x6400 | u is 1024 + u, less 1152 the code itself.
//   e4m3: one conversion for two codes takes the block's exponent along.
template <int QF> __device__ __forceinline__ u32x2 quant_f16x4(uint32_t w, float scale) {
  if constexpr (QF == UKV_CACHE_INT8) {
    const uint32_t u = w ^ 0x80808080u;
    const f16x2 s = {(_Float16)scale, (_Float16)scale}, off = {(_Float16)1152.f, (_Float16)1152.f};
    const f16x2 a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u));
    const f16x2 b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
    return u32x2{__builtin_bit_cast(uint32_t, (a - off) * s), __builtin_bit_cast(uint32_t, (b - off) * s)};
  } else {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false);
    const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true);
    return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
  }
}

// Four codes as two packed pairs of values of a 16-bit type (exact in either). int8 to bf16, whose eight significant
// bits leave no room for the offset above: through fp32, code + 128 from its byte, times scale, less 128 * scale.
template <int QF, int DT> __device__ __forceinline__ u32x2 quant_elems4(uint32_t w, float scale) {
  if constexpr (DT == UKV_DTYPE_F16) {
    return quant_f16x4<QF>(w, scale);
  } else if constexpr (QF == UKV_CACHE_INT8) {
    const uint32_t u = w ^ 0x80808080u;
    const float off = -128.f * scale;
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __builtin_fmaf((float)(uint8_t)(u >> (8 * i)), scale, off);
    return u32x2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
  } else {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true))};
  }
}

// One code as a float.
template <int QF> __device__ __forceinline__ float quant_one(uint8_t c, float scale) {
  if constexpr (QF == UKV_CACHE_INT8) return (float)(int8_t)c * scale;
  return __builtin_amdgcn_cvt_f32_fp8((int)c, 0) * scale;
}

// bf16 queries as fp16 operands: every row is moved by a power of two that its scores' scale takes back. A row whose
// largest magnitude has the exponent field `top` lands in [2^13, 2^14) with query_to_f16(.., top); 28 binades below
// that are exact, smaller elements are off by 2^-39 of the largest at most.
//
// The largest exponent field of a row, in each of its four lanes (lanes i16 + 16 kg hold eight dims of each step).
template <int STEPS> __device__ __forceinline__ int query_top(const u32x4 (&q)[STEPS]) {
  u16x2 m = {0, 0};
#pragma unroll
  for (int s = 0; s < STEPS; ++s)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t w = q[s][c];
      m = __builtin_elementwise_max(m, as_u16x2(w & 0x7fff7fffu));
    }
  int top = max((int)m[0], (int)m[1]) >> 7;
  top = max(top, __shfl_xor(top, 16));
  return max(top, __shfl_xor(top, 32));
}
template <int STEPS> __device__ __forceinline__ void query_to_f16(u32x4 (&q)[STEPS], int top) {
  const float down = __uint_as_float((uint32_t)min(267 - top, 254) << 23);
#pragma unroll
  for (int s = 0; s < STEPS; ++s)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t w = q[s][c];
      q[s][c] = pack_f16(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xffff0000u) * down);
    }
}
// What query_to_f16 divided by.
__device__ __forceinline__ float query_scale(int top) {
  return top > 13 ? __uint_as_float((uint32_t)(top - 13) << 23) : 0x1p-127f;
}

}  // namespace ukv
