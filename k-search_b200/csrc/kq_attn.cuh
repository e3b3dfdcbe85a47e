// Device helpers of the tensor-core attention kernels: packed fp32 arithmetic,
// score reads from TMEM, conversions.
#pragma once

#include <cuda_bf16.h>

#include "kq_device.cuh"
#include "kq_tc.cuh"

namespace kq {
namespace attn {

#ifdef __CUDACC__
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void store_f(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// (a, b) rounded to two values of T in one register, a in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Two fp32 lanes per instruction.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack(F2 a, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// Largest of N scores (N a multiple of 8), in a few parallel chains.
template <int N>
__device__ __forceinline__ float row_max(const uint32_t (&s)[N]) {
  float mx[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) mx[x] = fmaxf(__uint_as_float(s[x]), __uint_as_float(s[x + 4]));
#pragma unroll
  for (int x = 8; x < N; x += 8)
#pragma unroll
    for (int y = 0; y < 4; ++y) mx[y] = max3(mx[y], __uint_as_float(s[x + y]), __uint_as_float(s[x + y + 4]));
  return fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
}

// o *= f on `cols` accumulator columns of this thread's TMEM lane, in small
// pieces (the caller's scores are still in registers).
__device__ __forceinline__ void rescale_row(uint32_t taddr, int cols, float f) {
#pragma unroll 1
  for (int x = 0; x < cols; x += 16) {
    uint32_t o[16];
    tc::tmem_ld16(taddr + x, o);
    tc::tmem_ld_wait();
#pragma unroll
    for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
    tc::tmem_st16(taddr + x, o);
  }
}

// A warp's 32 rows of 64 bytes, staged in shared memory (2 KB): lane l holds
// row l as 4 pieces of 16 bytes; in the transposed view it holds piece l % 4 of
// rows l / 4 + 8 x, so that a global access covers whole 64-byte row pieces
// instead of 32 scattered ones of 16. Piece c of row r lies at c ^ (r / 2 % 4):
// eight rows hit distinct banks.
__device__ __forceinline__ uint4* stage_row(uint8_t* stage, int lane, int x) {
  return reinterpret_cast<uint4*>(stage + lane * 64 + ((x ^ ((lane >> 1) & 3)) << 4));
}
__device__ __forceinline__ uint4* stage_piece(uint8_t* stage, int lane, int x) {
  const int r = 8 * x + (lane >> 2);
  return reinterpret_cast<uint4*>(stage + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4));
}
// The same with rows of 128 bytes (4 KB): 8 pieces, a lane moves piece l % 8 of
// rows l / 8 + 4 x.
__device__ __forceinline__ uint4* stage128_row(uint8_t* stage, int lane, int x) {
  return reinterpret_cast<uint4*>(stage + lane * 128 + ((x ^ (lane & 7)) << 4));
}
__device__ __forceinline__ uint4* stage128_piece(uint8_t* stage, int lane, int x) {
  const int r = 4 * x + (lane >> 3);
  return reinterpret_cast<uint4*>(stage + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
}
#endif

}  // namespace attn
}  // namespace kq
