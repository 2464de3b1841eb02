// Matrix instructions (mma.sync, 16 rows by 8 columns, fp32 sums) and the
// splitting of fp32 operands into parts that they take.
#pragma once

#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace sc {
namespace mma {

// Operand types; Wide: fp32 on one side, split into parts of the other side's type.
enum Mode { kTF32, kBF16, kBF16Wide, kBF16Wide4, kF16, kF16Wide };
__host__ __device__ constexpr bool is_f16(int mode) { return mode == kF16 || mode == kF16Wide; }

template <int MODE>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  if (MODE == kTF32)
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else if (is_f16(MODE))
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The TF32 head of x: x rounded to 11 significant bits; x - head is exact.  The
// instruction cuts the tail to 11 bits too, which loses a unit of x's last place
// at most.  With a head cut off in place of a rounded one the tail loses up to
// three units, always towards zero: that put results off by 5e-7 (attention) and
// 1.3e-6 (adapters) of their size, one way, where fp32 sums are off by 2e-7 and
// 4e-7 either way.  A NaN that the addition carries over stays one in the tail.
__device__ __forceinline__ uint32_t tf32_head(float x) { return (__float_as_uint(x) + 0x1000u) & 0xffffe000u; }
__device__ __forceinline__ uint32_t tf32_tail(float x) { return __float_as_uint(x - __uint_as_float(tf32_head(x))); }

// The power of two that brings a row of largest value `top` to below 2^15 for a
// split into two fp16 parts: no part overflows, and values down to 2^-40 of the
// largest are not lost below fp16's smallest.  Rows below 2^-112 are brought up
// by no more than 2^126, so that the inverse is a normal number too.
__device__ __forceinline__ float f16_scale(float top) {
  const int e = (int)(__float_as_uint(top) >> 23) - 127;  // floor(log2(top)) of a normal number; 128: not finite
  return e < 128 ? __uint_as_float((uint32_t)((e > -112 ? e : -112) - 14 + 127) << 23) : 1.f;
}

// Two floats as packed 16-bit values, and what the packing lost of them.
template <int MODE>
__device__ __forceinline__ uint32_t pack2(float &a, float &b) {
  if (is_f16(MODE)) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    a -= f.x;
    b -= f.y;
    return *reinterpret_cast<const uint32_t *>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    const float2 f = __bfloat1622float2(h);
    a -= f.x;
    b -= f.y;
    return *reinterpret_cast<const uint32_t *>(&h);
  }
}

}  // namespace mma
}  // namespace sc
