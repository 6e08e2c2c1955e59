// Formats of the low-precision operands (8-bit rows, microscaled 4-bit floating point).
//
// mxfp4: E2M1 codes, one E8M0 byte (a power of two, 255 = NaN) per 32 columns.
// nvfp4: E2M1 codes, one E4M3 byte per 16 columns and one fp32 scale per row.
// int8:  int8 codes, one fp32 scale per row.
// 4-bit codes are packed two to a byte, low nibble = even column.  The block
// scales lie in tiles of 128 rows x 4 blocks (512 bytes): row r, block b at
// tile (r/128, b/4), byte (r%32)*16 + (r%128/32)*4 + b%4, the order in which
// tcgen05.cp takes them to tensor memory; the bytes of rows and blocks beyond
// the matrix are zero.
#pragma once
#include "common.cuh"

namespace ic {

constexpr float LOWP_SCALE_FLOOR = 1e-30f;  // smallest per-row scale: an all-zero row keeps a finite reciprocal

inline int64_t fp4_block(int fmt) { return fmt == IC_MXFP4 ? 32 : 16; }
inline int64_t fp4_ktiles(int fmt, int64_t kp) { return cdiv(kp, fp4_block(fmt) * 4); }

__host__ __device__ __forceinline__ int64_t scale_word(int64_t row, int64_t ktile, int64_t ktiles) {
  return ((row >> 7) * ktiles + ktile) * 512 + (row & 31) * 16 + ((row & 127) >> 5) * 4;
}

// packed fp32 pairs: one .f32x2 instruction for both halves, each rounded as alone
typedef unsigned long long f2;
__device__ __forceinline__ f2 pk2(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float lo2(f2 r) { return __uint_as_float((uint32_t)(r & 0xffffffffull)); }
__device__ __forceinline__ float hi2(f2 r) { return __uint_as_float((uint32_t)(r >> 32)); }
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f2 sub2(f2 a, f2 b) {
  f2 d;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

}  // namespace ic
