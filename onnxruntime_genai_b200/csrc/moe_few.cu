// A whole mixture-of-experts layer for up to eight tokens: router, choice of experts, gate / up products with the activation, down products and the
// weighted sum.
#include <math.h>

#include "common.cuh"
#include "kernels.h"

namespace ogb {

enum FewWeights : int { FEW_BF16 = 0, FEW_FP4_F16 = 1, FEW_FP4_BF16 = 2 };   // packed: the records of gemm_fp4.cu in their two forms
constexpr int FEW_TOKENS = 8, FEW_TOP = 32;

struct FewArgs {
  const __nv_bfloat16* x;
  long long ldx;
  const __nv_bfloat16* router;
  const __nv_bfloat16* router_b;
  const void* gate_up;
  const __nv_bfloat16* gate_up_b;
  const void* down;
  const __nv_bfloat16* down_b;
  __nv_bfloat16* out;
  int T, H, I, E, top, rule, act;
  float alpha, limit;
  int* ids;          // [T, top]
  float* share;      // [T, top]
  float* h;          // [T, top, I]
};

template <int W>
__device__ __forceinline__ float few_weight(const void* w, int e, int N, int K, int row, int k) {
  if constexpr (W == FEW_BF16) {
    return bf2f(static_cast<const __nv_bfloat16*>(w)[((long long)e * N + row) * K + k]);
  } else {
    const int tiles = (N + 127) / 128, c = (k & 63) >> 3, i = k & 7;
    const uint8_t* rec = static_cast<const uint8_t*>(w) + (((long long)e * (K / 64) + k / 64) * tiles + row / 128) * 4352;
    const int word = W == FEW_FP4_F16 ? ((c & 3) << 1) | (c >> 2) : c;
    const int shift = W == FEW_FP4_F16 ? (i & 3) * 8 + (i >> 2) * 4 : (i >> 1) * 4 + (i & 1) * 16;
    const uint32_t code = reinterpret_cast<const uint32_t*>(rec + (row & 127) * 32)[word] >> shift & 15u, m = code & 7u;
    const float a = m < 2u ? 0.5f * float(m) : __uint_as_float(((126u + (m >> 1)) << 23) | ((m & 1u) << 22));
    const int s = int(rec[4096 + (row & 127) * 2 + ((k & 63) >> 5)]);
    return ldexpf((code & 8u) ? -a : a, W == FEW_FP4_F16 ? s - 6 - 127 : ((s - 126) & 255) - 127);
  }
}

__global__ void few_route_kernel(FewArgs p) {
  extern __shared__ float logits[];
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = warp; e < p.E; e += blockDim.x >> 5) {
    float s = 0.f;
    for (int k = lane; k < p.H; k += 32) s += bf2f(p.x[t * p.ldx + k]) * bf2f(p.router[(long long)e * p.H + k]);
    s = warp_sum(s);
    if (lane == 0) logits[e] = s + (p.router_b ? bf2f(p.router_b[e]) : 0.f);
  }
  __syncthreads();
  if (threadIdx.x) return;
  float most = -INFINITY, sum = 0.f, all = 0.f;
  for (int e = 0; e < p.E; ++e) most = fmaxf(most, logits[e]);
  for (int e = 0; e < p.E; ++e) all += expf(logits[e] - most);
  for (int j = 0; j < p.top; ++j) {
    int best = 0;
    for (int e = 1; e < p.E; ++e) if (logits[e] > logits[best]) best = e;
    const float w = expf(logits[best] - most);
    p.ids[t * p.top + j] = best;
    p.share[t * p.top + j] = w;
    sum += w;
    logits[best] = -INFINITY;
  }
  for (int j = 0; j < p.top; ++j) p.share[t * p.top + j] /= p.rule == 1 ? all : sum;
}

template <int W>
__global__ void few_gate_up_kernel(FewArgs p) {
  const int item = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (item >= p.T * p.top * p.I) return;
  const int pair = item / p.I, i = item % p.I, e = p.ids[pair], t = pair / p.top, row = i / 64 * 128 + i % 64;
  float g = 0.f, u = 0.f;
  for (int k = lane; k < p.H; k += 32) {
    const float v = bf2f(p.x[t * p.ldx + k]);
    g += v * few_weight<W>(p.gate_up, e, 2 * p.I, p.H, row, k);
    u += v * few_weight<W>(p.gate_up, e, 2 * p.I, p.H, row + 64, k);
  }
  g = warp_sum(g);
  u = warp_sum(u);
  if (lane) return;
  if (p.gate_up_b) { g += bf2f(p.gate_up_b[e * 2 * p.I + row]); u += bf2f(p.gate_up_b[e * 2 * p.I + row + 64]); }
  if (p.act == 2) {
    if (p.limit > 0.f) { g = fminf(g, p.limit); u = fminf(fmaxf(u, -p.limit), p.limit); }
    p.h[item] = g / (1.f + expf(-p.alpha * g)) * (u + 1.f);
  } else {
    p.h[item] = g / (1.f + expf(-g)) * u;
  }
}

template <int W>
__global__ void few_down_kernel(FewArgs p) {
  const int item = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (item >= p.T * p.H) return;
  const int t = item / p.H, n = item % p.H;
  float sum = 0.f;
  for (int j = 0; j < p.top; ++j) {
    const int e = p.ids[t * p.top + j];
    float y = 0.f;
    for (int k = lane; k < p.I; k += 32) y += p.h[(t * p.top + j) * p.I + k] * few_weight<W>(p.down, e, p.H, p.I, n, k);
    sum += p.share[t * p.top + j] * (warp_sum(y) + (p.down_b ? bf2f(p.down_b[e * p.H + n]) : 0.f));
  }
  if (lane == 0) p.out[item] = f2bf(sum);
}

}  // namespace ogb

using namespace ogb;

OGB_API long long ogb_moe_few_scratch_bytes(int T, int top, int I) {
  return T < 1 || T > FEW_TOKENS || top < 1 || top > FEW_TOP || I < 1 ? -1 : (long long)T * top * (8 + 4LL * I);
}

OGB_API int ogb_moe_few_tokens(const void* x, long long ldx, const void* router, const void* router_b, const void* gate_up, const void* gate_up_b,
                               const void* down, const void* down_b, void* out, int T, int H, int I, int E, int top, int rule, int weights, int act,
                               float alpha, float limit, void* scratch, void* stream) {
  if (ogb_moe_few_scratch_bytes(T, top, I) < 0 || !x || !router || !gate_up || !down || !out || !scratch || H < 1 || E < top || E > 1024 || I % 64 ||
      (weights != FEW_BF16 && H % 64) || rule < 0 || rule > 2 || weights < 0 || weights > 2 || (act != 1 && act != 2)) return -1;
  FewArgs p{static_cast<const __nv_bfloat16*>(x), ldx, static_cast<const __nv_bfloat16*>(router), static_cast<const __nv_bfloat16*>(router_b), gate_up,
            static_cast<const __nv_bfloat16*>(gate_up_b), down, static_cast<const __nv_bfloat16*>(down_b), static_cast<__nv_bfloat16*>(out), T, H, I, E, top,
            rule, act, alpha, limit, nullptr, nullptr, nullptr};
  p.ids = static_cast<int*>(scratch);
  p.share = reinterpret_cast<float*>(p.ids + T * top);
  p.h = p.share + T * top;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  few_route_kernel<<<T, 256, E * 4, s>>>(p);
  const unsigned a = unsigned((T * top * I + 7) / 8), b = unsigned((T * H + 7) / 8);
  if (weights == FEW_BF16) { few_gate_up_kernel<FEW_BF16><<<a, 256, 0, s>>>(p); few_down_kernel<FEW_BF16><<<b, 256, 0, s>>>(p); }
  else if (weights == FEW_FP4_F16) { few_gate_up_kernel<FEW_FP4_F16><<<a, 256, 0, s>>>(p); few_down_kernel<FEW_FP4_F16><<<b, 256, 0, s>>>(p); }
  else { few_gate_up_kernel<FEW_FP4_BF16><<<a, 256, 0, s>>>(p); few_down_kernel<FEW_FP4_BF16><<<b, 256, 0, s>>>(p); }
  return cudaPeekAtLastError() == cudaSuccess ? 0 : -4;
}
