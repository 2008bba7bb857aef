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
  if constexpr (CODE == kE4m3 && !SCALED) {
    return raw2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, false)),
                __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, true))};
  }
  float f[4];
  widen4<CODE>(w, f);
  if constexpr (SCALED) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] *= s;
  }
  return raw2{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])};
}
