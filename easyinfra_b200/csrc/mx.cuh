// Microscaled (MX) number formats: blocks of 32 elements that share one power-of-two
// scale, held as its biased exponent (e8m0: 2^(byte - 127), byte 255 = NaN).
//   MX8  e4m3 elements (largest value 448): activations.  One row of K elements is
//        [K element bytes][K/32 scale bytes][padding to 16 bytes], so a row moves as one
//        piece (permute, exchange) and its scales are 16-byte loads.
//   MX4  e2m1 elements (largest value 6), two per byte, the even one in the low half:
//        weights.
// The scale of a block is the smallest power of two, 2^-127 at least, with which the
// block's largest magnitude does not pass the element type's largest value: no element
// saturates, and the elements use the type's top binade.  (The OCP specification's
// conversion takes floor(log2 amax) - emax, with which magnitudes above the largest value
// saturate.  The formats are the same, so blocks that were quantised that way can be read;
// codes and scales of the same values differ where it would saturate.)  A block that holds a NaN or an
// infinity gets the scale byte 255, so that everything computed from it is NaN.
// Elements are rounded once, to the nearest with ties to even.
#pragma once

#include "common.cuh"

namespace b200moe {

constexpr int MX_BLOCK = 32;

// Bytes of an MX8 row of K elements (K a multiple of 32).
__host__ __device__ constexpr int64_t mx8_row_bytes(int64_t K) { return K + (K / MX_BLOCK + 15) / 16 * 16; }

// Scale byte from the largest |x| of a block as fp32 bits (sign cleared; comparing the
// bits as integers keeps NaN and infinity on top).  EMAX, LIMIT: the element type's
// largest value is (1 + LIMIT / 2^23) 2^EMAX.
template <int EMAX, uint32_t LIMIT>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255u;
  const int e = static_cast<int>(amax_bits >> 23) - EMAX + ((amax_bits & 0x7fffffu) > LIMIT ? 1 : 0);
  return static_cast<uint32_t>(max(e, 0));
}
__device__ __forceinline__ uint32_t mx8_scale_byte(uint32_t amax_bits) { return mx_scale_byte<8, 0x600000u>(amax_bits); }
__device__ __forceinline__ uint32_t mx4_scale_byte(uint32_t amax_bits) { return mx_scale_byte<2, 0x400000u>(amax_bits); }

// 2^(127 - byte), which turns a block's values into elements: exact in fp32 for every
// byte up to 253, the largest one of a finite block (e2m1, magnitudes from 1.5 * 2^127 on),
// NaN for 255.
__device__ __forceinline__ float mx_inverse_scale(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float((254u - byte) << 23);
}

// The value of a scale byte in fp32 (byte 0 is the subnormal 2^-127).
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
  if (byte == 0u) return __uint_as_float(0x00400000u);
  return byte == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(byte << 23);
}

// Two values to two e4m3 bytes (lo in the low byte); NaN becomes the type's NaN.
__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t cvt_e4m3x4(float a, float b, float c, float d) {
  return cvt_e4m3x2(a, b) | (cvt_e4m3x2(c, d) << 16);
}

// Two values to one byte of e2m1 (lo in the low half).  The type has no NaN.
__device__ __forceinline__ uint32_t cvt_e2m1x2(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 t;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\t"
      "cvt.u32.u8 %0, t;\n\t}"
      : "=r"(r)
      : "f"(hi), "f"(lo));
  return r;
}

// Packed elements back to values (half precision holds every e4m3 and e2m1 value).
__device__ __forceinline__ float2 half2_bits_to_float2(uint32_t bits) {
  float lo, hi;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
      : "=f"(lo), "=f"(hi)
      : "r"(bits));
  return make_float2(lo, hi);
}
__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t two_bytes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(two_bytes)));
  return half2_bits_to_float2(h);
}
__device__ __forceinline__ float2 e2m1x2_to_float2(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h) : "r"(byte));
  return half2_bits_to_float2(h);
}

// ---- quantisation (mx_quant.cu)
struct MxQuantParams {
  const void* x;        // [rows, K], row stride ldx elements
  int64_t ldx;
  int64_t rows;
  int64_t K;            // multiple of 32
  uint8_t* data;        // elements, row stride ld_data bytes
  int64_t ld_data;
  uint8_t* scales;      // scale bytes, row stride ld_scales
  int64_t ld_scales;
  int pad;              // MX8 rows: zero bytes written after the K/32 scale bytes
};

struct MxDequantParams {
  const uint8_t* data;
  int64_t ld_data;
  const uint8_t* scales;
  int64_t ld_scales;
  int64_t rows;
  int64_t K;
  void* out;            // [rows, K], row stride ldo elements
  int64_t ldo;
};

int launch_mx_quantize(const MxQuantParams& p, int dtype, bool four_bit, cudaStream_t stream);
int launch_mx_dequantize(const MxDequantParams& p, int dtype, bool four_bit, cudaStream_t stream);

}  // namespace b200moe
