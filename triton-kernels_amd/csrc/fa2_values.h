// fa2_values.h - 16 bytes of tensor values to fp32 and back, and words of 4-bit codes
// (E2M1 at a power of two) to 16 bits.
#pragma once

#include "fa2_device.h"

namespace fa2 {

// 16 bytes of values as fp32
template <int DT>
__device__ __forceinline__ void unpack16(u32x4 r, float* x) {
  if constexpr (DT == FA2_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = r[i];
      x[i] = __builtin_bit_cast(float, w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = r[i];
      if constexpr (DT == FA2_DTYPE_BF16) {
        x[2 * i] = __builtin_bit_cast(float, w << 16);
        x[2 * i + 1] = __builtin_bit_cast(float, w & 0xFFFF0000u);
      } else {
        const f32x2 f = __builtin_convertvector(__builtin_bit_cast(f16x2, w), f32x2);
        x[2 * i] = f[0];
        x[2 * i + 1] = f[1];
      }
    }
  }
}

// ... and back, rounded
template <int DT>
__device__ __forceinline__ u32x4 pack16(const float* x) {
  u32x4 r;
  if constexpr (DT == FA2_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(uint32_t, x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = pack2<DT == FA2_DTYPE_BF16>(x[2 * i], x[2 * i + 1]);
  }
  return r;
}

// The 8 values of a code word at the scale with E8M0 byte `sb` (255: NaN).
template <bool BF>
__device__ __forceinline__ u32x4 fp4_values(uint32_t w, uint32_t sb) {
  const float f = __builtin_bit_cast(float, sb << 23);
  if constexpr (BF)
    return (u32x4){
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 0)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 1)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 2)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 3))};
  else
    return (u32x4){
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 0)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 1)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 2)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 3))};
}

}  // namespace fa2
