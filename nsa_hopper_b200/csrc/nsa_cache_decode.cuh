// From the 4-bit cache's codes and scales to operands of the tensor core.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

namespace nsa {
namespace cache {

// Two codes of byte I of `w` as fp16 pair (low nibble in the low half).
template <int I>
__device__ __forceinline__ uint32_t decode_byte(uint32_t w) {
  uint32_t r;
  if constexpr (I == 0)
    asm("{.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b0;}" : "=r"(r) : "r"(w));
  else if constexpr (I == 1)
    asm("{.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b1;}" : "=r"(r) : "r"(w));
  else if constexpr (I == 2)
    asm("{.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b2;}" : "=r"(r) : "r"(w));
  else
    asm("{.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b3;}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// A scale byte in both halves of an fp16 pair.
__device__ __forceinline__ uint32_t scale2(uint32_t byte) { return byte * 0x00800080u; }

// m16n8k16, fp16 in, fp32 out.
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

}  // namespace cache
}  // namespace nsa
