// Shared definitions of the 8-bit kernels: e4m3 (OCP float8_e4m3fn: 4
// exponent bits, 3 of mantissa, largest value 448, no infinity) with one fp32
// scale per block of 128.
#pragma once

#include "tjk_common.h"

namespace tjk {

constexpr int kF8Block = 128;
constexpr float kF8Max = 448.0f;
// The smallest scale, the least normal fp32: a block of zeros takes it, and
// its reciprocal is finite.
constexpr float kF8MinScale = 1.1754943508222875e-38f;  // 2^-126

// Scale of a block whose largest magnitude is `top`: top / 448 (to within one
// unit in the last place), at least kF8MinScale.  A block that holds an
// infinity has scale inf (its finite values become 0, its infinities NaN);
// NaN elements stay NaN and do not count in `top` (fmaxf drops them).
__device__ __forceinline__ float f8_scale(float top) { return fmaxf(top * (1.0f / kF8Max), kF8MinScale); }

// Four values times `inv`, the reciprocal of their block's scale, rounded
// to nearest even in e4m3, value i in byte i.  A reciprocal good to one unit in
// the last place leaves |v inv| <= 448 (1 + 2^-22), which rounds to at most
// 448: nothing saturates.  A quotient that close to a tie may go either way.
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d, float inv) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, w, true);
  return (uint32_t)w;
}

// Largest of the 16 lanes of a DPP row, in each of them.
__device__ __forceinline__ float row16_max(float v) {
  auto step = [](float x, float y) { return fmaxf(x, y); };
  v = step(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true)));
  v = step(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, true)));
  v = step(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x141, 0xF, 0xF, true)));
  v = step(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x140, 0xF, 0xF, true)));
  return v;
}

// Eight consecutive elements in fp32; a raw piece is 16 bytes of a 2-byte
// type, 32 of fp32.
template <typename T> struct Oct;
template <> struct Oct<float> {
  struct raw { float4 lo, hi; };
  static __device__ __forceinline__ raw load(const float* p) {
    return raw{reinterpret_cast<const float4*>(p)[0], reinterpret_cast<const float4*>(p)[1]};
  }
  static __device__ __forceinline__ void to(const raw& r, float (&v)[8]) {
    v[0] = r.lo.x; v[1] = r.lo.y; v[2] = r.lo.z; v[3] = r.lo.w;
    v[4] = r.hi.x; v[5] = r.hi.y; v[6] = r.hi.z; v[7] = r.hi.w;
  }
  static __device__ __forceinline__ raw from(const float (&v)[8]) {
    return raw{make_float4(v[0], v[1], v[2], v[3]), make_float4(v[4], v[5], v[6], v[7])};
  }
};
template <typename T> struct Oct {
  typedef uint4 raw;
  static __device__ __forceinline__ raw load(const T* p) { return *reinterpret_cast<const uint4*>(p); }
  static __device__ __forceinline__ void to(const raw& r, float (&v)[8]) {
    const float4 a = Quad<T>::to(make_uint2(r.x, r.y)), b = Quad<T>::to(make_uint2(r.z, r.w));
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  static __device__ __forceinline__ raw from(const float (&v)[8]) {
    const uint2 a = Quad<T>::from(make_float4(v[0], v[1], v[2], v[3]));
    const uint2 b = Quad<T>::from(make_float4(v[4], v[5], v[6], v[7]));
    return make_uint4(a.x, a.y, b.x, b.y);
  }
};

}  // namespace tjk
