// 8-bit KV cache pages: the row format and its conversions.
//
// A page of one KV head is a record of 256 rows x 128 e4m3 codes followed by the
// 256 rows' scale bytes; pages are [num_pages][Hkv] records.  All rows of a (page,
// head) are contiguous, so attention streams 32 KiB runs whatever the number of
// heads (with heads inside a row, as in the bf16 cache, a head's rows lie
// Hkv * 128 bytes apart and every 64 scale bytes come from 64 lines).
//
// Row x[0..127] with finite maximum a = m * 2^E (1 <= m < 2) has the scale 2^e,
//   e = max(E - 8 + (m > 1.75), -117),
// the smallest power of two with a <= 448 * 2^e (448: the largest e4m3 value),
// kept as the byte e + 127 in [10, 247], and the codes e4m3(x_i * 2^-e), rounded to
// nearest even.  A power of two costs at most one of e4m3's 18 octaves; in return
// the product is exact, so is the border between two codes, and code * 2^e is a
// bf16 value: e >= -117 keeps the smallest one, 2^-9 * 2^e, normal.  NaN and
// infinities are left out of the maximum and stored as NaN (e4m3 has no infinity).
#pragma once

#include "common.h"

namespace dllm {

constexpr int kPageRows = 256;
constexpr int kQuantD = 128;
constexpr int kScaleOff = kPageRows * kQuantD;      // scale bytes behind the codes
constexpr int kRecord = kScaleOff + kPageRows;      // 33024 bytes of a (page, KV head)

// Record byte offset of the row in `slot`'s page and head; the row is slot & 255.
__device__ __forceinline__ int64_t record_off(uint32_t slot, int Hkv, int h) {
  return ((int64_t)(slot >> 8) * Hkv + h) * kRecord;
}

// Scale byte of a row whose finite maximum has the bf16 bits `amax` (sign cleared).
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  const int b = (int)(amax >> 7) - 8 + ((amax & 0x7f) > 0x60 ? 1 : 0);
  return (uint32_t)max(b, 10);
}
// 2^e and 2^-e of a scale byte (both normal).
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ float inv_scale_of(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// Eight bf16 values (x_i in order) of a row piece -> eight codes.
__device__ __forceinline__ u32x2_t quant8(u32x4_t x, float inv) {
  u32x2_t r;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float f[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f[2 * i] = __uint_as_float(x[2 * w + i] << 16) * inv;
      f[2 * i + 1] = __uint_as_float(x[2 * w + i] & 0xffff0000u) * inv;
    }
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
    r[w] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], c, true);
  }
  return r;
}

// Eight codes -> eight bf16 values, exact (v_cvt_scalef32_pk_bf16_fp8 multiplies
// by the scale's power of two).
__device__ __forceinline__ u32x4_t dequant8(u32x2_t c, float scale) {
  u32x4_t r;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    r[2 * w] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[w], scale, false));
    r[2 * w + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[w], scale, true));
  }
  return r;
}

typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
// One row spread over 16 lanes, eight values each: its codes and scale byte.
// Every lane of the wavefront must be active.
__device__ __forceinline__ u32x2_t quant_row16(u32x4_t x, uint32_t& byte) {
  u16x2_t m = {0, 0};
#pragma unroll
  for (int w = 0; w < 4; ++w) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, x[w] & 0x7fff7fffu));
  uint32_t a = m[0] > m[1] ? m[0] : m[1];
#pragma unroll
  for (int j = 1; j < 16; j <<= 1) a = max(a, lane_xor(a, j));
  if (__builtin_amdgcn_ballot_w64(a >= 0x7f80u)) {  // a row with NaN or an infinity
    uint32_t f = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t h = (x[w] >> (16 * i)) & 0x7fffu;
        if (h < 0x7f80u)
          f = max(f, h);
        else
          x[w] |= 0x7fffu << (16 * i);  // a NaN
      }
#pragma unroll
    for (int j = 1; j < 16; j <<= 1) f = max(f, lane_xor(f, j));
    a = f;
  }
  byte = scale_byte(a);
  return quant8(x, inv_scale_of(byte));
}

}  // namespace dllm
