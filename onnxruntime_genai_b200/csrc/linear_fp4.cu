// Linear layers on 4-bit floating-point rows and weights (layout: fp4_matrix.cuh):
//   C[t, n] = a_row[t] * w_row[n] * sum_blocks a_scale * w_scale * sum_k a_code * w_code   (+ bias, residual, or the gated activation)
#include "fp4_matrix.cuh"
#include "kernels.h"

namespace ogb {

struct Fp4LinearArgs {
  Fp4View a, w;
  int N;
  void* C;
  long long ldc;
  int out_fp32, pair;
  const __nv_bfloat16* bias;
  const void* residual;
  long long ldr;
  int res_fp32;
};

constexpr int TILE = 16;
template <int FORM>
__global__ void linear_fp4_simple_kernel(Fp4LinearArgs p) {
  constexpr int B = FORM == FP4_NV ? 16 : 32;
  __shared__ float sa[TILE][FP4_KB], sw[2][TILE][FP4_KB];
  const int tx = threadIdx.x % TILE, ty = threadIdx.x / TILE;
  const int n_out = p.pair ? p.N / 2 : p.N, t0 = blockIdx.y * TILE, col = blockIdx.x * TILE + tx;
  float acc[2] = {0.f, 0.f};
  auto value = [&](const Fp4View& m, int kb, int r, int k) {
    if (r >= m.rows) return 0.f;
    const uint32_t byte = m.codes[fp4_code_at(m, kb, r, k >> 5) + ((k & 31) >> 1)];
    return fp4_value((k & 1) ? byte >> 4 : byte & 15u) * fp4_scale(FORM, m.scales[fp4_scale_at(m, FORM, kb, r, (k / B) >> 2, (k / B) & 3)]);
  };
  auto weight_row = [&](int c) { return p.pair ? c / 64 * 128 + c % 64 : c; };   // gate row of an output column; its up row is 64 further
  for (int kb = 0; kb < p.a.num_kb; ++kb) {
    __syncthreads();
    for (int i = threadIdx.x; i < TILE * FP4_KB; i += blockDim.x) {
      const int r = i / FP4_KB, k = i % FP4_KB, wr = weight_row(blockIdx.x * TILE + r);
      sa[r][k] = value(p.a, kb, t0 + r, k);
      sw[0][r][k] = value(p.w, kb, wr, k);
      if (p.pair) sw[1][r][k] = value(p.w, kb, wr + 64, k);
    }
    __syncthreads();
    for (int k = 0; k < FP4_KB; ++k) {
      acc[0] += sa[ty][k] * sw[0][tx][k];
      if (p.pair) acc[1] += sa[ty][k] * sw[1][tx][k];
    }
  }
  const int t = t0 + ty, wr = weight_row(col);
  if (t >= p.a.rows || col >= n_out) return;
  const float s = p.a.row_scale[t];
  float v = acc[0] * s * p.w.row_scale[wr] + (p.bias ? bf2f(p.bias[wr]) : 0.f);
  if (p.pair) {
    const float u = acc[1] * s * p.w.row_scale[wr + 64] + (p.bias ? bf2f(p.bias[wr + 64]) : 0.f);
    v = v / (1.f + __expf(-v)) * u;
  }
  if (p.residual) v += p.res_fp32 ? static_cast<const float*>(p.residual)[t * p.ldr + col] : bf2f(static_cast<const __nv_bfloat16*>(p.residual)[t * p.ldr + col]);
  if (p.out_fp32) static_cast<float*>(p.C)[t * p.ldc + col] = v; else static_cast<__nv_bfloat16*>(p.C)[t * p.ldc + col] = f2bf(v);
}

}  // namespace ogb

using namespace ogb;

OGB_API int ogb_linear_fp4(const void* x, long long ldx, int x_fp32, void* a_data, int T, const void* w_data, int N, int K, int form, void* out, long long ldc,
                           int out_fp32, int pair, const void* bias, const void* residual, long long ldr, int res_fp32, int* status, void* stream) {
  if (!w_data || T < 0 || (T > 0 && (!a_data || !out)) || N <= 0 || K <= 0 || (form != FP4_NV && form != FP4_MX) || K % fp4_block(form)) return -1;
  if ((reinterpret_cast<uintptr_t>(a_data) | reinterpret_cast<uintptr_t>(w_data)) & 15) return -1;
  if (pair && (N % 128 || residual)) return -1;
  if (T == 0) return 0;
  if (x) {
    const int rc = ogb_quantize_fp4(x, ldx, x_fp32, T, K, form, a_data, stream);
    if (rc) return rc;
  }
  Fp4LinearArgs p{fp4_view(a_data, T, K, form), fp4_view(const_cast<void*>(w_data), N, K, form), N, out, ldc, out_fp32, pair,
                  static_cast<const __nv_bfloat16*>(bias), residual, ldr, res_fp32};
  const dim3 grid(unsigned(((pair ? N / 2 : N) + TILE - 1) / TILE), unsigned((T + TILE - 1) / TILE));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (form == FP4_NV) linear_fp4_simple_kernel<FP4_NV><<<grid, TILE * TILE, 0, s>>>(p); else linear_fp4_simple_kernel<FP4_MX><<<grid, TILE * TILE, 0, s>>>(p);
  return cudaPeekAtLastError() == cudaSuccess ? 0 : -4;
}
