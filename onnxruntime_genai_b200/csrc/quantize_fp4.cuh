// Rules of the quantisation to 4-bit floating point, shared by the kernels that do it (compiled with IEEE denormals).
//
// nvfp4: the row's scale is s = the smallest power of two >= max|x| / 2688 (2688 = 6 * 448, the largest e2m1 times the largest e4m3), at least
// 2^-100; a block's scale is e4m3(max|block| / s / 6), to nearest; an element's code is e2m1(x / (scale * s)), to nearest with ties to the even
// code, 0 where the block's scale is.  A power of two leaves x / s exact, so that no step before the last rounding moves a value across a tie.
// mxfp4: a block's scale is 2^(floor(log2 max|block|) - 2), clamped to e8m0's range; an element's code is e2m1(x / scale), at most 6.  s = 1.
// A row that holds an infinity or a NaN gets s = NaN, and everything computed from it is NaN.
#pragma once
#include <cuda_fp16.h>

#include "fp4_matrix.cuh"

namespace ogb {

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ float pow2(int e) { return e >= -126 ? __uint_as_float(uint32_t(e + 127) << 23) : __uint_as_float(1u << (e + 149)); }   // -149 <= e <= 127
// exponent of the row's scale, from the bits of its largest magnitude
__device__ __forceinline__ int row_exponent(uint32_t top) {
  const int e = int(top >> 23) - 127;                       // max|x| = m 2^e, 1 <= m < 2; 2688 = 1.3125 * 2^11
  return max((top & 0x7fffffu) <= 0x280000u ? e - 11 : e - 10, -100);
}
__device__ __forceinline__ uint32_t e4m3_of(float v) {      // 0 <= v <= 448, to nearest even
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(v));
  return r & 0xffu;
}
__device__ __forceinline__ float e4m3_value(uint32_t code) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(code)));
  return __half2float(__ushort_as_half(uint16_t(h)));
}
// eight numbers to eight codes, the first in the lowest four bits: to nearest, ties to the even code, at most 6
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// Eight consecutive elements as they lie in memory.
template <typename T> struct Raw8;
template <> struct Raw8<__nv_bfloat16> {
  uint4 q;
  template <bool VEC> __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    if constexpr (VEC) q = *reinterpret_cast<const uint4*>(p);
    else {
      const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
      q = make_uint4(u[0] | uint32_t(u[1]) << 16, u[2] | uint32_t(u[3]) << 16, u[4] | uint32_t(u[5]) << 16, u[6] | uint32_t(u[7]) << 16);
    }
  }
  __device__ __forceinline__ void zero() { q = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ uint32_t largest() const {        // bits of the largest magnitude, as fp32 (a NaN: of a NaN)
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(part(q.x), part(q.y)), __hmax2_nan(part(q.z), part(q.w)));
    return uint32_t(__bfloat16_as_ushort(__hmax_nan(m.x, m.y))) << 16;
  }
  static __device__ __forceinline__ __nv_bfloat162 part(uint32_t w) { return __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w)); }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
};
template <> struct Raw8<float> {
  float4 a, b;
  template <bool VEC> __device__ __forceinline__ void load(const float* p) {
    if constexpr (VEC) { a = reinterpret_cast<const float4*>(p)[0]; b = reinterpret_cast<const float4*>(p)[1]; }
    else { a = make_float4(p[0], p[1], p[2], p[3]); b = make_float4(p[4], p[5], p[6], p[7]); }
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ uint32_t largest() const {
    float v[8];
    get(v);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[i]));
    return m;
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
};

// Eight elements a lane of a row's k-block (32 lanes in order): their codes, and the byte of their block's scale, which the block's lanes share.
// m: bits of the largest magnitude of the lane's eight; s, over: the row's scale and its reciprocal; bad: the row holds what is not a number.
template <typename T, int FORM>
__device__ __forceinline__ uint32_t fp4_codes8(const Raw8<T>& r, uint32_t m, float s, float over, bool bad, uint32_t& code) {
  float v[8];
  r.get(v);
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  if (FORM == FP4_NV) {
    // Quotients are products with a reciprocal.  One that is a tie has to come out as that tie, and one that is not on its side of it; the powers of two of
    // the row's scale change no rounding.
    constexpr float sixth = 1.f / 6.f;
    const float t = __uint_as_float(m) * over, h = t * sixth;
    if constexpr (sizeof(T) == 2) {
      // Of numbers of eight bits: a sixth of such a number is a tie of e4m3 only where the product with the rounded 1/6 comes out exact (tested for all of
      // them), and a quotient by a scale of four bits is a tie or at least 2^-10 away from it, so that rounding it to whole 2^-14, by an addition, puts it right.
      constexpr float grid = 768.f;                                       // 1.5 * 2^9; quotients are at most 9
      code = bad ? 0u : e4m3_of(h);
      const float inv = code ? reciprocal(e4m3_value(code)) * over : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __fsub_rn(fmaf(v[i], inv, grid), grid);
    } else {
      // Else: one correction by the exact remainder, with reciprocals that a Newton step makes the nearest ones.
      code = bad ? 0u : e4m3_of(fmaf(fmaf(-h, 6.f, t), sixth, h));
      const float sc = e4m3_value(code), by = sc * s, near = reciprocal(sc);
      const float inv = code ? fmaf(fmaf(-sc, near, 1.f), near, near) * over : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float q = v[i] * inv;
        v[i] = fmaf(fmaf(-q, by, v[i]), inv, q);
      }
    }
  } else {
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    int e = int(m >> 23) - 127;
    if (m < 0x00800000u) e = m ? -118 - __clz(m) : -127;                 // below the normal numbers: m 2^-149
    e = max(e - 2, -127);
    code = bad ? 0u : uint32_t(e + 127);
    const float inv = __uint_as_float(uint32_t(127 - e) << 23);          // (of a row that is not numbers: whatever)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= inv;
  }
  return bad ? 0u : e2m1x8(v);
}

}  // namespace ogb
