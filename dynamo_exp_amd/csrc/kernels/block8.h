// The 8-bit KV cache with a scale for each block and key/value head: codes [num_blocks, Hkv, BS, 128] (int8, or e4m3fn),
// scales [num_blocks, Hkv] fp32, value = code * scale.  Shared by its writer (block_cache.hip) and its readers.
#pragma once
#include "common.h"

typedef unsigned int raw2 __attribute__((ext_vector_type(2)));
typedef unsigned int raw4 __attribute__((ext_vector_type(4)));

enum : int { kInt8 = 0, kE4m3 = 1 };

// four codes of a word as fp32 (exact)
template <int CODE> __device__ __forceinline__ void widen4(uint32_t w, float (&f)[4]) {
  if constexpr (CODE == kE4m3) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    f[0] = lo[0], f[1] = lo[1], f[2] = hi[0], f[3] = hi[1];
  } else {
    f[0] = (float)(int8_t)w, f[1] = (float)(int8_t)(w >> 8), f[2] = (float)(int8_t)(w >> 16), f[3] = (float)((int32_t)w >> 24);
  }
}

// ... times a scale, as bf16 pairs (exact where the scale is a power of two: a code has at most 7 bits)
template <int CODE, bool SCALED> __device__ __forceinline__ raw2 widen4_bf16(uint32_t w, float s) {
  float f[4];
  widen4<CODE>(w, f);
  if constexpr (SCALED) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] *= s;
  }
  return raw2{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])};
}

// ---- codes in fp16, which holds them and their products with small powers of two exactly
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {  // (one v_cvt_pk_f16_f32, half-even)
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{lo, hi}, f16x2));
}
// four codes of a word: e4m3 by the conversion instruction; an int8 code c as (1024 + (c + 128)) - 1152, its byte put in the mantissa of
// 1024 (1.25 instructions a code; by fp32 it would be 1.5)
template <int CODE> __device__ __forceinline__ raw2 widen4_f16(uint32_t w) {
  if constexpr (CODE == kE4m3) {
    return raw2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, false)),
                __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, true))};
  } else {
    const f16x2 bias = {(_Float16)-1152.f, (_Float16)-1152.f};
    const uint32_t u = w ^ 0x80808080u;
    return raw2{__builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + bias),
                __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + bias)};
  }
}
// 16 codes, times a factor where SCALED
template <int CODE, bool SCALED> __device__ __forceinline__ void widen16_f16(const raw4& w, float factor, raw4 (&o)[2]) {
  const f16x2 f = {(_Float16)factor, (_Float16)factor};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const raw2 x = widen4_f16<CODE>(w[i]);
    uint32_t lo = x[0], hi = x[1];  // (a bit cast of a vector's element itself takes the first one, whichever is named)
    if constexpr (SCALED) {
      lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, lo) * f);
      hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, hi) * f);
    }
    o[i >> 1][2 * (i & 1)] = lo, o[i >> 1][2 * (i & 1) + 1] = hi;
  }
}
// the power of two that brings |x| <= amax under 2 (exact inverse in fp32; 1 for 0)
__device__ __forceinline__ float unit_factor(float amax) {
  const int e = (int)(__float_as_uint(amax) >> 23) - 127;
  return amax > 0.f ? __uint_as_float((uint32_t)(127 - max(min(e, 126), -126)) << 23) : 1.f;
}
