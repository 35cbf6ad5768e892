// Rows to 4-bit floating point in blocks, and back (layout: fp4_matrix.cuh).
//
// nvfp4: the row's scale is s = the smallest power of two >= max|x| / 2688 (2688 = 6 * 448, the largest e2m1 times the largest e4m3), at least
// 2^-100; a block's scale is e4m3(max|block| / s / 6), to nearest; an element's code is e2m1(x / (scale * s)), to nearest with ties to the even
// code, 0 where the block's scale is.  A power of two leaves x / s exact, so that no step before the last rounding moves a value across a tie.
// mxfp4: a block's scale is 2^(floor(log2 max|block|) - 2), clamped to e8m0's range; an element's code is e2m1(x / scale), at most 6.  s = 1.
// A row that holds an infinity or a NaN gets s = NaN, and everything computed from it is NaN.
#include <cuda_fp16.h>

#include "fp4_matrix.cuh"
#include "kernels.h"

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
__device__ __forceinline__ void values8(uint32_t codes, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
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

// A warp turns a row's k-blocks of 256, eight elements a lane: a block of 16 (32) belongs to two (four) lanes, the codes of a k-block go out as one
// line of 128 bytes.  `wpr` warps share a row (a power of two up to THREADS / 32) and meet once, at the row's largest value; up to
// HELD k-blocks a warp stay in registers between the two passes, later ones are read again.
// With many rows bound by the instructions of a number (some twelve) beside the bytes: 256 threads with eight pieces each, four CTAs an SM (4096 x 14336 bf16 in 36.5 us,
// 4.1 TB/s; three an SM: 38.8; five with four pieces each, whose rows are partly read twice: 45.8; a CTA that fetches its next row ahead: no gain).  fp32 rows to mxfp4 do
// not fit 64 registers: three an SM (777 x 2880 in 3.2 us, else 3.8).  Bound by latency with few rows, where twice the warps share a row.
constexpr int quantize_ctas(int bytes, int form, int threads) { return threads == 512 ? 2 : bytes == 4 && form == FP4_MX ? 3 : 4; }
template <typename T, int FORM, bool VEC, int HELD, int THREADS>
__global__ void __launch_bounds__(THREADS, quantize_ctas(sizeof(T), FORM, THREADS)) quantize_fp4_kernel(const T* __restrict__ x, long long ldx, int K, int wpr, Fp4View out) {
  __shared__ uint32_t s_top[16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, first = warp & (wpr - 1);
  const int row = blockIdx.x * (THREADS / 32 / wpr) + warp / wpr;
  const bool here = row < out.rows;
  const T* src = x + (long long)(here ? row : 0) * ldx;
  pdl_wait();
  pdl_launch_dependents();     // after the wait: whoever starts now may read what the kernels before this one wrote (linear_fp4.cu does)
  Raw8<T> held[HELD];
  uint32_t top = 0, most[HELD];
  auto fetch = [&](int kb) {
    Raw8<T> r;
    const int k = kb * FP4_KB + lane * 8;
    if (here && k < K) r.template load<VEC>(src + k); else r.zero();        // K is a multiple of 16: all eight or none
    return r;
  };
#pragma unroll
  for (int i = 0; i < HELD; ++i) held[i] = fetch(first + i * wpr);
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    most[i] = held[i].largest();
    top = max(top, most[i]);
  }
  for (int kb = first + HELD * wpr; kb < out.num_kb; kb += wpr) top = max(top, fetch(kb).largest());
  top = __reduce_max_sync(0xffffffffu, top);
  if (wpr > 1) {
    if (lane == 0) s_top[warp] = top;
    __syncthreads();
    for (int w = 0; w < wpr; ++w) top = max(top, s_top[(warp & ~(wpr - 1)) + w]);
  }
  if (!here) return;
  const bool bad = top >= 0x7f800000u;
  const int re = FORM == FP4_NV ? row_exponent(top) : 0;
  const float s = pow2(re), over = pow2(-re);
  if (first == 0 && lane == 0) out.row_scale[row] = bad ? __uint_as_float(0x7fc00000u) : s;

  constexpr int PER = FORM == FP4_NV ? 2 : 4;                              // lanes of a block
  uint8_t* codes_to = out.codes + fp4_code_at(out, first, row, lane >> 2) + (lane & 3) * 4;
  uint8_t* scales_to = out.scales + fp4_scale_at(out, FORM, first, row, lane / (4 * PER), lane / PER & 3);
  const long long codes_step = (long long)wpr * out.padded * 128, scales_step = (long long)wpr * (out.padded >> 7) * (fp4_steps(FORM) * FP4_SCALE_STEP);
  auto emit = [&](const Raw8<T>& r, uint32_t m) {
    float v[8];
    r.get(v);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    uint32_t code;
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
        const float inv = code ? __fdividef(1.f, fp4_scale_nv(code)) * over : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fsub_rn(fmaf(v[i], inv, grid), grid);
      } else {
        // Else: one correction by the exact remainder, with reciprocals that a Newton step makes the nearest ones.
        code = bad ? 0u : e4m3_of(fmaf(fmaf(-h, 6.f, t), sixth, h));
        const float sc = fp4_scale_nv(code), by = sc * s, near = __fdividef(1.f, sc);
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
    *reinterpret_cast<uint32_t*>(codes_to) = bad ? 0u : e2m1x8(v);
    if (lane % PER == 0) *scales_to = uint8_t(code);
    codes_to += codes_step;
    scales_to += scales_step;
  };
#pragma unroll
  for (int i = 0; i < HELD; ++i)
    if (first + i * wpr < out.num_kb) emit(held[i], most[i]);
  for (int kb = first + HELD * wpr; kb < out.num_kb; kb += wpr) {
    const Raw8<T> r = fetch(kb);
    emit(r, r.largest());
  }
}

// A warp reads four rows of a k-block (512 bytes of codes), eight elements a lane and row.
constexpr int DEQUANT_ROWS = 4;
template <typename T, int FORM>
__global__ void __launch_bounds__(256) dequantize_fp4_kernel(Fp4View m, int K, T* __restrict__ out, long long ldo, int vec) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, row0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * DEQUANT_ROWS, kb = blockIdx.y;
  const int k = kb * FP4_KB + lane * 8, b = lane / (FORM == FP4_NV ? 2 : 4);
  if (k >= K) return;
  uint32_t codes[DEQUANT_ROWS];
  float scale[DEQUANT_ROWS];
#pragma unroll
  for (int i = 0; i < DEQUANT_ROWS; ++i) {
    const int r = min(row0 + i, m.rows - 1);
    codes[i] = *reinterpret_cast<const uint32_t*>(m.codes + fp4_code_at(m, kb, r, lane >> 2) + (lane & 3) * 4);
    scale[i] = fp4_scale(FORM, m.scales[fp4_scale_at(m, FORM, kb, r, b >> 2, b & 3)]) * m.row_scale[r];
  }
#pragma unroll
  for (int i = 0; i < DEQUANT_ROWS; ++i) {
    if (row0 + i >= m.rows) break;
    float v[8];
    values8(codes[i], v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= scale[i];
    T* dst = out + (long long)(row0 + i) * ldo + k;
    if constexpr (sizeof(T) == 4) {
      if (vec) { reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]); reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]); }
      else for (int j = 0; j < 8; ++j) dst[j] = v[j];
    } else {
      if (vec) *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
      else for (int j = 0; j < 8; ++j) dst[j] = f2bf(v[j]);
    }
  }
}

template <typename T, int FORM, bool VEC>
static bool LaunchQuantize(const T* x, long long ldx, int K, const Fp4View& v, cudaStream_t s) {
  const bool few = v.rows <= 296;                   // two CTAs of 512 threads an SM
  constexpr int HELD = sizeof(T) == 2 ? 8 : 4;
  const int warps = few ? 16 : 8, each = few ? 1 : HELD;      // k-blocks that a warp is to have of a row, where it has so many
  int wpr = 1;
  while (wpr * each < v.num_kb && wpr < warps) wpr *= 2;
  const int rows_per_cta = warps / wpr;
  const dim3 grid(unsigned((v.rows + rows_per_cta - 1) / rows_per_cta)), block(unsigned(warps * 32));
  return few ? launch_pdl(quantize_fp4_kernel<T, FORM, VEC, 4, 512>, grid, block, 0, s, x, ldx, K, wpr, v)
             : launch_pdl(quantize_fp4_kernel<T, FORM, VEC, HELD, 256>, grid, block, 0, s, x, ldx, K, wpr, v);
}
template <typename T, int FORM>
static bool LaunchQuantize(const void* x, long long ldx, int K, const Fp4View& v, cudaStream_t s) {
  const T* p = static_cast<const T*>(x);
  const bool vec = ((reinterpret_cast<uintptr_t>(x) | uintptr_t(ldx * (long long)sizeof(T))) & 15) == 0;
  return vec ? LaunchQuantize<T, FORM, true>(p, ldx, K, v, s) : LaunchQuantize<T, FORM, false>(p, ldx, K, v, s);
}
template <typename T>
static bool LaunchDequantize(const Fp4View& v, int K, int form, void* out, long long ldo, cudaStream_t s) {
  const dim3 grid(unsigned((v.rows + 8 * DEQUANT_ROWS - 1) / (8 * DEQUANT_ROWS)), unsigned(v.num_kb));
  T* p = static_cast<T*>(out);
  const int vec = ((reinterpret_cast<uintptr_t>(out) | uintptr_t(ldo * (long long)sizeof(T))) & 15) == 0;
  return form == FP4_NV ? launch_pdl(dequantize_fp4_kernel<T, FP4_NV>, grid, dim3(256), 0, s, v, K, p, ldo, vec)
                        : launch_pdl(dequantize_fp4_kernel<T, FP4_MX>, grid, dim3(256), 0, s, v, K, p, ldo, vec);
}

}  // namespace ogb

using namespace ogb;

OGB_API long long ogb_fp4_matrix_bytes(int rows, int K, int form) {
  return rows < 0 || K <= 0 || (form != FP4_NV && form != FP4_MX) ? -1 : fp4_bytes(rows, K, form);
}

static bool BadFp4(const void* data, const void* other, int rows, int K, int form) {      // (empty tensors have no address)
  return rows < 0 || K <= 0 || (form != FP4_NV && form != FP4_MX) || K % fp4_block(form) || (rows > 0 && (!data || !other)) || (reinterpret_cast<uintptr_t>(data) & 15);
}

OGB_API int ogb_quantize_fp4(const void* x, long long ldx, int x_fp32, int rows, int K, int form, void* data, void* stream) {
  if (BadFp4(data, x, rows, K, form)) return -1;
  if (rows == 0) return 0;
  const Fp4View v = fp4_view(data, rows, K, form);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool ok = x_fp32 ? (form == FP4_NV ? LaunchQuantize<float, FP4_NV>(x, ldx, K, v, s) : LaunchQuantize<float, FP4_MX>(x, ldx, K, v, s))
                         : (form == FP4_NV ? LaunchQuantize<__nv_bfloat16, FP4_NV>(x, ldx, K, v, s) : LaunchQuantize<__nv_bfloat16, FP4_MX>(x, ldx, K, v, s));
  return ok ? 0 : -4;
}

OGB_API int ogb_dequantize_fp4(const void* data, int rows, int K, int form, void* out, long long ldo, int out_fp32, void* stream) {
  if (BadFp4(data, out, rows, K, form)) return -1;
  if (rows == 0) return 0;
  const Fp4View v = fp4_view(const_cast<void*>(data), rows, K, form);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (v.num_kb > 65535) return -5;
  return (out_fp32 ? LaunchDequantize<float>(v, K, form, out, ldo, s) : LaunchDequantize<__nv_bfloat16>(v, K, form, out, ldo, s)) ? 0 : -4;
}
