// The paged cache held in 8 bits: shared pieces of its append, decode and prefill kernels.
//
// K and V are e4m3 numbers [num_blocks, block_size, num_kv_heads, head_dim]; a scale per block and kv head ([num_blocks,
// num_kv_heads] f32, K and V apart) says what one unit is worth: value = number * scale.  The append makes scales that are powers
// of two between 2^-117 and 2^119, so that
//   * dividing by one is exact: a value is rounded once, by the conversion to e4m3;
//   * a block whose scale grows is rescaled exactly, but for numbers that leave e4m3's normal range;
//   * number * scale is a bf16 and an f32 number exactly, down to the smallest subnormal e4m3 (2^-9 * 2^-117 = 2^-126).
#pragma once

#include <cuda_fp8.h>

#include <type_traits>

#include "nvj_common.cuh"

namespace nvj {

constexpr int kQLowExp = -117, kQHighExp = 119;

// Head layouts and block sizes that the kernels take: rows of 64, 128 or 256 elements, blocks of 16, 32, 48 or 64 tokens (a key tile of 16
// lies in one block; a block's rows fit a 64-bit mask).
inline bool quantized_cache_shape_ok(int block_size, int num_kv_heads, int head_dim) {
  return (head_dim == 64 || head_dim == 128 || head_dim == 256) && block_size >= 16 && block_size <= 64 && block_size % 16 == 0 &&
         num_kv_heads >= 1 && num_kv_heads <= 1024;
}
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// 2^e for -126 <= e <= 127.
__host__ __device__ __forceinline__ float q_pow2(int e) {
#ifdef __CUDA_ARCH__
  return __int_as_float((e + 127) << 23);
#else
  union { int i; float f; } u;
  u.i = (e + 127) << 23;
  return u.f;
#endif
}
// The scale for a block whose largest finite magnitude is `largest`: 2^e with the least e such that largest <= 448 * 2^e
// (448 = 1.75 * 2^8), within the range above.  Past its upper end values are held at 448 * 2^119.
__device__ __forceinline__ float q_scale_for(float largest) {
  const int bits = __float_as_int(largest);
  const int e = (bits >> 23) - 135 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return q_pow2(e < kQLowExp ? kQLowExp : (e > kQHighExp ? kQHighExp : e));
}
// Two e4m3 numbers (x in the low byte): rounded to nearest even, magnitudes over 448 and infinities held at 448, NaN kept.
__device__ __forceinline__ uint32_t q_pack2(float x, float y) {
  return __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3);
}
// The two numbers in the low half of w as an f16 pair: exact.
__device__ __forceinline__ uint32_t q_half2(uint32_t w) {
  uint32_t h;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(h) : "r"(w));
  return h;
}
// ... and in its high half.
__device__ __forceinline__ uint32_t q_half2_high(uint32_t w) {
  uint32_t h;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(h) : "r"(w));
  return h;
}
__device__ __forceinline__ float2 q_float2(uint32_t half2) {
  return __half22float2(*reinterpret_cast<const __half2*>(&half2));
}

__device__ __forceinline__ void q_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t q_transpose(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t q_pair(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// What the rounding of q_pair(x, y) left over.
__device__ __forceinline__ uint32_t q_pair_rest(float x, float y, uint32_t high) {
  const float2 f = q_float2(high);
  return q_pair(x - f.x, y - f.y);
}

// Eight elements of a row of activations, as loaded and as floats.
template <typename T>
struct QRaw {
  uint4 v;
};
template <>
struct QRaw<float> {
  uint4 v, w;
};
template <typename T>
__device__ __forceinline__ QRaw<T> q_load8(const T* p) {
  QRaw<T> r;
  r.v = ld_stream_u4(p);
  if constexpr (sizeof(T) == 4) r.w = ld_stream_u4(p + 4);
  return r;
}
template <typename T>
__device__ __forceinline__ void q_floats(const QRaw<T>& r, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const uint32_t u[8] = {r.v.x, r.v.y, r.v.z, r.v.w, r.w.x, r.w.y, r.w.z, r.w.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(u[i]);
  } else {
    const uint32_t u[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 f;
      if constexpr (sizeof(T) == 2 && !std::is_same<T, __half>::value) f = bf16x2_to_float2(u[i]);
      else f = q_float2(u[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}
// The largest of m and the finite magnitudes among x.
__device__ __forceinline__ float q_largest(float m, const float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = fabsf(x[i]);
    if (a < __int_as_float(0x7f800000)) m = fmaxf(m, a);
  }
  return m;
}

}  // namespace nvj
