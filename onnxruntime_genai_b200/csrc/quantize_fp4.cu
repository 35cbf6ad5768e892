// Rows to 4-bit floating point in blocks, and back (layout: fp4_matrix.cuh; rules: quantize_fp4.cuh).
#include "kernels.h"
#include "quantize_fp4.cuh"

namespace ogb {

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

// A warp turns a row's k-blocks of 256, eight elements a lane: a block of 16 (32) belongs to two (four) lanes, the codes of a k-block go out as one
// line of 128 bytes.  `wpr` warps share a row (a power of two up to THREADS / 32) and meet once, at the row's largest value; up to
// HELD k-blocks a warp stay in registers between the two passes, later ones are read again.
// With many rows bound by the instructions of a number (some ten) beside the bytes: 256 threads with eight pieces each, four CTAs an SM (4096 x 14336 bf16 in 33.9 us,
// 4.4 TB/s; when that took 36.5: three an SM 38.8, five with four pieces each, whose rows are partly read twice, 45.8, a CTA that fetches its next row ahead no gain).  fp32
// rows to mxfp4 do not fit 64 registers: three an SM (777 x 2880 in 3.2 us, else 3.8).  Bound by latency with few rows, where twice the warps share a row.
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
    uint32_t code;
    *reinterpret_cast<uint32_t*>(codes_to) = fp4_codes8<T, FORM>(r, m, s, over, bad, code);
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
