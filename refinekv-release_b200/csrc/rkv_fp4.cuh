// Rows held in 4 bits: 16 channels share a scale s, an e4m3 number, and each
// channel a code c, an e2m1 number (a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4,
// 6).  The channel stands for c s, times the KV head's fp32 factor where there
// is one.  c s has six significant bits and lies between 2^-10 and 2688, so it
// is exact in fp16 (and in bf16).
//
// A page's KV head is one slab of block * dim * 9 / 16 contiguous bytes: the
// codes of its rows, row after row (dim / 2 bytes each, channel 2i in the low
// half of byte i), then the scales of its rows (dim / 16 bytes each).  One bulk
// copy fetches it: dim and block are multiples of 32 and 16, so slabs are
// multiples of 16 bytes whatever the shape.
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

namespace rkv {

__host__ __device__ constexpr int fp4_slab_bytes(int block, int dim) {
  return block * (dim / 2 + dim / 16);
}

constexpr float kFp4Most = 6.f;  // the largest code
constexpr uint32_t kFp4NanScale = 0x7f;

// Eight codes (a word) as four fp16 pairs, in channel order.
__device__ __forceinline__ void fp4_decode(uint32_t codes, uint32_t (&pairs)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(pairs[0]), "=r"(pairs[1]), "=r"(pairs[2]), "=r"(pairs[3])
      : "r"(codes));
}

// Two scales (the low 16 bits) as an fp16 pair.
__device__ __forceinline__ uint32_t fp4_scales(uint32_t two) {
  uint32_t pair;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(pair) : "h"(static_cast<uint16_t>(two)));
  return pair;
}

__device__ __forceinline__ float fp4_scale_value(uint32_t scale) {
  const uint32_t pair = fp4_scales(scale);
  return __low2float(*reinterpret_cast<const __half2*>(&pair));
}

// Eight quotients x / s to the nearest codes, ties to the even one, beyond 6 to 6.
__device__ __forceinline__ uint32_t fp4_encode(const float (&y)[8]) {
  uint32_t codes;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(codes)
      : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
  return codes;
}

// The scale of 16 channels whose greatest magnitude has the bits `most`: most /
// 6 rounded to e4m3, at most 448.  A channel that is infinite or NaN makes it
// NaN, and with it all 16.
__device__ __forceinline__ uint32_t fp4_scale_of(uint32_t most) {
  if (most >= 0x7f800000u) return kFp4NanScale;
  uint16_t two;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %1;"
      : "=h"(two)
      : "f"(__fdiv_rn(__uint_as_float(most), kFp4Most)));
  return two & 0xffu;
}

}  // namespace rkv
