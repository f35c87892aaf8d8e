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

constexpr uint32_t kFp4NanScale = 0x7f;

// Two codes, byte I of a word, as an fp16 pair.  (An assembler block for each: one with
// four conversions whose results were not all used gave wrong ones with nvcc 12.9.)
template <int I>
__device__ __forceinline__ uint32_t fp4_decode2(uint32_t codes) {
  uint32_t pair;
  if constexpr (I == 0)
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t}" : "=r"(pair) : "r"(codes));
  if constexpr (I == 1)
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(pair) : "r"(codes));
  if constexpr (I == 2)
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, c;\n\t}" : "=r"(pair) : "r"(codes));
  if constexpr (I == 3)
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, d;\n\t}" : "=r"(pair) : "r"(codes));
  return pair;
}

// Eight codes (a word) as four fp16 pairs, in channel order.
__device__ __forceinline__ void fp4_decode(uint32_t codes, uint32_t (&pairs)[4]) {
  pairs[0] = fp4_decode2<0>(codes);
  pairs[1] = fp4_decode2<1>(codes);
  pairs[2] = fp4_decode2<2>(codes);
  pairs[3] = fp4_decode2<3>(codes);
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

// Two quotients x / s to the nearest codes, ties to the even one, beyond 6 to 6.
__device__ __forceinline__ uint32_t fp4_encode2(float first, float second) {
  uint32_t codes;
  asm("{\n\t.reg .b8 a;\n\tcvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.u32.u8 %0, a;\n\t}" : "=r"(codes) : "f"(first), "f"(second));
  return codes;
}

// Eight of them, a word.
__device__ __forceinline__ uint32_t fp4_encode(const float (&y)[8]) {
  return __byte_perm(__byte_perm(fp4_encode2(y[0], y[1]), fp4_encode2(y[2], y[3]), 0x0040),
                     __byte_perm(fp4_encode2(y[4], y[5]), fp4_encode2(y[6], y[7]), 0x0040), 0x5410);
}

}  // namespace rkv
