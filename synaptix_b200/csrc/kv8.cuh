// The format of keys and values held in eight bits, shared by the kernels that write and read it.
//
// A head's row of a token, x[0 .. hd), is one exponent byte e and hd e4m3 codes c_i and stands for c_i 2^(e - 127).  With a
// the row's largest magnitude, a = m 2^x and 1 <= m < 2, e - 127 is x - 8 where m <= 1.75 and x - 7 above (448 = 1.75 2^8 is
// the largest e4m3 number), kept in -117 .. 119; codes are rounded to nearest even and saturate.  e = 255: the row was not
// finite and reads as NaN; its codes are e4m3's NaN (0x7f) too, so a kernel may look at either.  A scale that is a power of two takes nothing from a floating format: all
// magnitudes within 2^13 of the row's largest keep their three bits of mantissa, as with any other scale, and in return x / scale and
// code * scale are exact in bfloat16, float16 (within its range) and float32.  So writing rounds once, whatever
// else a kernel does in which order, and reading back rounds never.
//
// Pages hold 64 tokens of all kv heads.  Keys: [hd / CB][64 keys][CB], CB the largest of 64, 32, 16 that divides hd; values:
// [hd][64 keys], exponents: [64].  Both are made for the tensor cores' fragments.  A thread of a fragment wants pairs of
// neighbours along the product's inner axis, which are dims of one key in q k^T and KEYS of one dim in p v: with values stored
// dim by dim both are plain 16-byte loads (16 codes), and rows of 64 bytes spread the eight rows a load touches over all banks.
#pragma once
#include "common.cuh"

#include <cuda_fp8.h>

#define KV8_NAN 255
#define KV8_MIN 10
#define KV8_MAX 246

__host__ __device__ __forceinline__ int kv8_block(int hd) { return hd % 64 == 0 ? 64 : hd % 32 == 0 ? 32 : 16; }
// byte of key `key`, element d within a head's K (or V) page
__device__ __forceinline__ int kv8_k_at(int key, int d, int cb) { return (d / cb) * (SX_PAGE * cb) + key * cb + d % cb; }
__device__ __forceinline__ int kv8_v_at(int key, int d) { return d * SX_PAGE + key; }

// the exponent byte of a row whose largest magnitude is `a`; `finite`: no element is an infinity or NaN
__device__ __forceinline__ int kv8_exponent(float a, bool finite) {
  if (!finite) return KV8_NAN;
  const int bits = __float_as_int(a);
  const int e = (bits >> 23) - ((bits & 0x7fffff) <= 0x600000 ? 8 : 7);
  return a == 0.f ? KV8_MIN : min(max(e, KV8_MIN), KV8_MAX);
}
// 2^(127 - e), what a row's elements are multiplied by ahead of their rounding (NaN for a row that is not finite)
__device__ __forceinline__ float kv8_inverse(int e) { return __int_as_float(e == KV8_NAN ? 0x7fffffff : (254 - e) << 23); }
// 2^(e - 127); NaN for 255
__device__ __forceinline__ float kv8_scale(int e) { return e == KV8_NAN ? __int_as_float(0x7fffffff) : __int_as_float(e << 23); }
// two codes at once: `lo` in the low byte
__device__ __forceinline__ uint32_t kv8_codes2(float lo, float hi) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
// four codes as half precision, exactly: the two of the low 16 bits, the two of the high ones
__device__ __forceinline__ void kv8_half4(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}\n" : "=r"(lo), "=r"(hi) : "r"(codes));
}
__device__ __forceinline__ uint32_t kv8_half2(uint32_t codes) {
  uint32_t lo, hi;
  kv8_half4(codes, lo, hi);
  return lo;
}
__device__ __forceinline__ float2 kv8_float2(uint32_t codes) {
  const uint32_t h = kv8_half2(codes);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ void kv8_float16(const uint4 c, float (&x)[16]) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = kv8_float2(w[i]), b = kv8_float2(w[i] >> 16);
    x[4 * i] = a.x; x[4 * i + 1] = a.y; x[4 * i + 2] = b.x; x[4 * i + 3] = b.y;
  }
}
// what the attention kernels are made of: c += a b of 16 x 8 x 16 halves and of 16 x 8 x 32 codes, 2^x, and two numbers as halves
__device__ __forceinline__ void kv8_mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void kv8_mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float kv8_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t kv8_pack2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
