// MXFP4, the microscaled 4-bit format (OCP Microscaling Formats v1.0): a row
// of k elements is ceil(k / 32) blocks of 16 bytes, two elements a byte (the
// first in the low half), each sign, two exponent bits and one mantissa bit
// (0, 0.5, 1, 1.5, 2, 3, 4, 6); a scale byte b for each block stands for the
// factor 2^(b - 127), 255 for NaN.
//
// gfx950 converts two elements an instruction and takes the factor from the
// exponent bits of an f32 operand alone (sign and mantissa are ignored, all
// ones give NaN), so a scale byte need only be shifted to bits 30:23.
#pragma once

#include "dw_device.h"

namespace dw {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// A scale byte as the conversions' factor operand.
__device__ __forceinline__ float mx_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// The scale byte of a block whose largest magnitude has these f32 bits
// (without the sign): floor(log2) - 2, at least the format's smallest, and
// 255 where an infinity or NaN is among the elements.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits, uint32_t least) {
  const uint32_t e = amax_bits >> 23;
  return e == 255u ? 255u : max(e, least + 2u) - 2u;
}

// Eight values over one factor, to nearest even, saturated at 6: one word.
__device__ __forceinline__ uint32_t mx_encode8(const float* v, float scale) {
  uint32_t q = 0;
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], scale, 0);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], scale, 1);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], scale, 2);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], scale, 3);
  return q;
}

// The largest over each aligned group of four lanes.
__device__ __forceinline__ uint32_t max_of_quad(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));   // lanes 1 0 3 2
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));  // lanes 2 3 0 1
}

// Sums up to and with each lane, in the lanes' registers (six steps of data
// parallel primitives; each shuffle through LDS would cost several times one).
__device__ __forceinline__ int sums_upto(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);   // the lane one to the left in its row of 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);   // two
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);   // four
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);   // eight
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // the last of row 0 to row 1, of 2 to 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // the last of row 1 to rows 2 and 3
  return v;
}

// The 8 values of one word, exact in f32.
__device__ __forceinline__ void mx_decode8(uint32_t q, float scale, float* v) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 0);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 1);
  const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 2);
  const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 3);
  v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
  v[4] = c[0]; v[5] = c[1]; v[6] = d[0]; v[7] = d[1];
}

// n elements of 16 or 32 bits from any element's address: one wide access
// each way (global memory takes unaligned ones).
template <typename T, int N>
struct Loose {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Loose<T, N> load_loose(const T* p) {
  Loose<T, N> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <typename T, int N>
__device__ __forceinline__ void store_loose(T* p, const Loose<T, N>& r) {
  __builtin_memcpy(p, &r, sizeof(r));
}
__device__ __forceinline__ float widen(uint16_t h) { return h2f_ieee(h); }
__device__ __forceinline__ float widen(float f) { return f; }
template <typename T>
__device__ __forceinline__ T narrow(float f);
template <>
__device__ __forceinline__ uint16_t narrow<uint16_t>(float f) {
  return __builtin_bit_cast(uint16_t, (_Float16)f);
}
template <>
__device__ __forceinline__ float narrow<float>(float f) {
  return f;
}

}  // namespace dw
