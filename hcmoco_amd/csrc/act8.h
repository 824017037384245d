// The 8-bit block format shared by act8.hip, norm.hip and fp8mm.hip (device side).
//
// 128 neighbouring values of a row (a 128 x 128 block of a weight) are held as e4m3 numbers q (OCP: 448 the largest, no
// infinity) times one power of two 2^E, stored as the biased byte E + 127:
//     E = the smallest exponent with max|x| <= 448 * 2^E,  at least -126;  0 for a block without a nonzero value
//     q = e4m3(x * 2^-E), to nearest, ties to even; a value that is not finite becomes NaN and does not count in the maximum
// Why a power of two and not max|x| / 448: x * 2^-E and q * 2^E are exact, so the stored value does not depend on the order or
// the rounding of whatever computes it; q * 2^E is exact in bf16 (3 fraction bits) for -124 <= E <= 119, that is, for blocks whose largest
// magnitude is in 2^-116 .. 2^127, so that a checkpoint enters a bf16 matrix instruction without a second rounding; and the scaled matrix
// instructions of this chip take exactly this byte.  (Below: bf16's steps are 2^-133.  Above, E = 120: what rounds up to 256, from 248 * 2^120
// = 3.3e38 on, is 2^128, infinite in bf16 as in fp32.)  Cost: up to one binade of e4m3's range of eighteen, none of its precision.
#pragma once
#include "hcm_common.h"

namespace hcm {

enum : int { kF32 = 0, kBF16 = 1, kF16 = 2 };      // dtype codes of the C ABI (HCM_DT_*)

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v8f __attribute__((ext_vector_type(8)));

template <typename T> struct Vec8;
template <> struct Vec8<float> { typedef v8f type; };
template <> struct Vec8<__bf16> { typedef v8bf type; };
template <> struct Vec8<_Float16> { typedef v8h type; };

// Eight consecutive elements as floats.  The address needs the element's alignment only (a global load of 4 dwords does not ask
// for more), so odd row lengths take the same path.  `left` (> 0) elements of the row remain: the others read as zero.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int left, float (&v)[8]) {
  if (left >= 8) {
    typename Vec8<T>::type r;
    __builtin_memcpy(&r, p, 8 * sizeof(T));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)r[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? (float)p[i] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int left, const float (&v)[8]) {
  if (left >= 8) {
    typename Vec8<T>::type r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (T)v[i];
    __builtin_memcpy(p, &r, 8 * sizeof(T));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = (T)v[i];
  }
}
// the same from a float / bf16 / fp16 vector whose type is known at run time only (parameters, read once per workgroup)
__device__ __forceinline__ void load8_dt(const void* p, int dt, int64_t at, int left, float (&v)[8]) {
  if (dt == kF32) load8((const float*)p + at, left, v);
  else if (dt == kBF16) load8((const __bf16*)p + at, left, v);
  else load8((const _Float16*)p + at, left, v);
}
__device__ __forceinline__ float load_dt(const void* p, int dt, int64_t at) {
  return dt == kF32 ? ((const float*)p)[at] : dt == kBF16 ? (float)((const __bf16*)p)[at] : (float)((const _Float16*)p)[at];
}
__device__ __forceinline__ void store_dt(void* p, int dt, int64_t at, float v) {
  if (dt == kF32) ((float*)p)[at] = v;
  else if (dt == kBF16) ((__bf16*)p)[at] = (__bf16)v;
  else ((_Float16*)p)[at] = (_Float16)v;
}

__device__ __forceinline__ bool finite_f(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }
__device__ __forceinline__ float finite_abs(float x) { return finite_f(x) ? fabsf(x) : 0.f; }

// the biased exponent byte of a block whose largest finite magnitude is amax (448 = 1.75 * 2^8)
__device__ __forceinline__ int act8_byte(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return u == 0 ? 127 : max(e, 1);
}
__device__ __forceinline__ float pow2_of_byte(int b) { return __uint_as_float((uint32_t)b << 23); }            // 2^(b - 127), b >= 1
__device__ __forceinline__ float inv_pow2_of_byte(int b) { return __uint_as_float((uint32_t)(254 - b) << 23); }  // b <= 253

// eight values -> eight e4m3 bytes
__device__ __forceinline__ v2i act8_bytes(const float (&x)[8], float inv) {
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = finite_f(x[i]) ? x[i] * inv : __uint_as_float(0x7fc00000u);
  v2i q;
  q[0] = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
  q[0] = __builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], q[0], true);
  q[1] = __builtin_amdgcn_cvt_pk_fp8_f32(s[4], s[5], 0, false);
  q[1] = __builtin_amdgcn_cvt_pk_fp8_f32(s[6], s[7], q[1], true);
  return q;
}
// eight e4m3 bytes -> the values they stand for
__device__ __forceinline__ void act8_values(v2i q, float scale, float (&x)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    x[4 * h + 0] = __builtin_amdgcn_cvt_f32_fp8(q[h], 0) * scale;
    x[4 * h + 1] = __builtin_amdgcn_cvt_f32_fp8(q[h], 1) * scale;
    x[4 * h + 2] = __builtin_amdgcn_cvt_f32_fp8(q[h], 2) * scale;
    x[4 * h + 3] = __builtin_amdgcn_cvt_f32_fp8(q[h], 3) * scale;
  }
}

}  // namespace hcm
