// Rows to 4-bit floating point in blocks, and back (layout: fp4_matrix.cuh).
//
// nvfp4: the row's scale is s = the smallest power of two >= max|x| / 2688 (2688 = 6 * 448, the largest e2m1 times the largest e4m3), at least
// 2^-100; a block's scale is e4m3(max|block| / s / 6), to nearest; an element's code is e2m1(x / (scale * s)), to nearest with ties to the even
// code, 0 where the block's scale is.  A power of two leaves x / s exact, so that no step before the last rounding moves a value across a tie.
// mxfp4: a block's scale is 2^(floor(log2 max|block|) - 2), clamped to e8m0's range; an element's code is e2m1(x / scale), at most 6.  s = 1.
// A row that holds an infinity or a NaN gets s = NaN, and everything computed from it is NaN.
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
__device__ __forceinline__ uint32_t e2m1_of(float q) {      // to nearest, ties to even, at most 6
  const float a = fabsf(q);
  const uint32_t c = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.f);
  return c | (q < 0.f && c ? 8u : 0u);
}
__device__ __forceinline__ uint32_t e4m3_of(float v) {      // 0 <= v <= 448, to nearest even
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(v));
  return r & 0xffu;
}

template <typename T>
__device__ __forceinline__ float load_one(const T* p) {
  if constexpr (sizeof(T) == 4) return *p; else return bf2f(*p);
}

// One CTA per row; a thread takes whole blocks.
template <typename T, int FORM>
__global__ void quantize_fp4_kernel(const T* x, long long ldx, int K, Fp4View out) {
  constexpr int B = FORM == FP4_NV ? 16 : 32;
  __shared__ uint32_t s_top[32];
  const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* src = x + (long long)row * ldx;
  pdl_wait();
  pdl_launch_dependents();     // after the wait: whoever starts now may read what the kernels before this one wrote (linear_fp4.cu does)
  uint32_t top = 0;
  for (int k = threadIdx.x; k < K; k += blockDim.x) top = max(top, abs_bits(load_one(src + k)));
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) s_top[warp] = top;
  __syncthreads();
  for (int w = 0; w < int(blockDim.x >> 5); ++w) top = max(top, s_top[w]);
  const bool bad = top >= 0x7f800000u;
  const int re = FORM == FP4_NV ? row_exponent(top) : 0;
  if (threadIdx.x == 0) out.row_scale[row] = bad ? __uint_as_float(0x7fc00000u) : pow2(re);
  const float over = bad ? 0.f : pow2(-re);
  for (int b = threadIdx.x; b < out.num_kb * (FP4_KB / B); b += blockDim.x) {
    float v[B];
    uint32_t m = 0;
    for (int i = 0; i < B; ++i) {
      const int k = b * B + i;
      v[i] = k < K && !bad ? load_one(src + k) * over : 0.f;
      m = max(m, abs_bits(v[i]));
    }
    uint32_t code;
    if (FORM == FP4_NV) {
      code = e4m3_of(__fdiv_rn(__uint_as_float(m), 6.f));
      const float sc = fp4_scale_nv(code);
      for (int i = 0; i < B; ++i) v[i] = code ? __fdiv_rn(v[i], sc) : 0.f;
    } else {
      const float top_v = __uint_as_float(m);
      int e = m >= 0x00800000u ? int(m >> 23) - 127 : (m ? ilogbf(top_v) : -127);
      e = max(e - 2, -127);
      code = uint32_t(e + 127);
      for (int i = 0; i < B; ++i) v[i] *= pow2(-e);
    }
    const int kb = b / (FP4_KB / B), in = b % (FP4_KB / B);
    out.scales[fp4_scale_at(out, FORM, kb, row, in >> 2, in & 3)] = uint8_t(code);
    for (int i = 0; i < B; i += 2) {
      const int k = in * B + i;
      out.codes[fp4_code_at(out, kb, row, k >> 5) + ((k & 31) >> 1)] = uint8_t(e2m1_of(v[i]) | (e2m1_of(v[i + 1]) << 4));
    }
  }
}

template <typename T, int FORM>
__global__ void dequantize_fp4_kernel(Fp4View m, int K, T* out, long long ldo) {
  constexpr int B = FORM == FP4_NV ? 16 : 32;
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.x;
  const float s = m.row_scale[row];
  for (int k = threadIdx.x; k < K; k += blockDim.x) {
    const int kb = k / FP4_KB, in = k % FP4_KB, b = in / B;
    const uint32_t byte = m.codes[fp4_code_at(m, kb, row, in >> 5) + ((in & 31) >> 1)];
    const float v = fp4_value((in & 1) ? byte >> 4 : byte & 15u) * fp4_scale(FORM, m.scales[fp4_scale_at(m, FORM, kb, row, b >> 2, b & 3)]) * s;
    if constexpr (sizeof(T) == 4) out[(long long)row * ldo + k] = v; else out[(long long)row * ldo + k] = f2bf(v);
  }
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
  bool ok;
  if (x_fp32) {
    ok = form == FP4_NV ? launch_pdl(quantize_fp4_kernel<float, FP4_NV>, dim3(rows), dim3(256), 0, s, static_cast<const float*>(x), ldx, K, v)
                        : launch_pdl(quantize_fp4_kernel<float, FP4_MX>, dim3(rows), dim3(256), 0, s, static_cast<const float*>(x), ldx, K, v);
  } else {
    ok = form == FP4_NV ? launch_pdl(quantize_fp4_kernel<__nv_bfloat16, FP4_NV>, dim3(rows), dim3(256), 0, s, static_cast<const __nv_bfloat16*>(x), ldx, K, v)
                        : launch_pdl(quantize_fp4_kernel<__nv_bfloat16, FP4_MX>, dim3(rows), dim3(256), 0, s, static_cast<const __nv_bfloat16*>(x), ldx, K, v);
  }
  return ok ? 0 : -4;
}

OGB_API int ogb_dequantize_fp4(const void* data, int rows, int K, int form, void* out, long long ldo, int out_fp32, void* stream) {
  if (BadFp4(data, out, rows, K, form)) return -1;
  if (rows == 0) return 0;
  const Fp4View v = fp4_view(const_cast<void*>(data), rows, K, form);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (out_fp32) {
    if (form == FP4_NV) dequantize_fp4_kernel<float, FP4_NV><<<rows, 256, 0, s>>>(v, K, static_cast<float*>(out), ldo);
    else dequantize_fp4_kernel<float, FP4_MX><<<rows, 256, 0, s>>>(v, K, static_cast<float*>(out), ldo);
  } else {
    if (form == FP4_NV) dequantize_fp4_kernel<__nv_bfloat16, FP4_NV><<<rows, 256, 0, s>>>(v, K, static_cast<__nv_bfloat16*>(out), ldo);
    else dequantize_fp4_kernel<__nv_bfloat16, FP4_MX><<<rows, 256, 0, s>>>(v, K, static_cast<__nv_bfloat16*>(out), ldo);
  }
  return cudaPeekAtLastError() == cudaSuccess ? 0 : -4;
}
