// What the 4-bit products share (linear_fp4.cu: few tokens, linear_fp4_pair.cu: prompts): arguments, tensor-core wrappers, the store of results.
#pragma once
#include "gemm_common.cuh"
#include "fp4_matrix.cuh"

namespace ogb {

struct Fp4LinearArgs {
  Fp4View a, w;
  int N, n_out;
  void* C;
  long long ldc;
  int out_fp32, pair;
  const __nv_bfloat16* bias;
  const void* residual;
  long long ldr;
  int res_fp32;
  int whole;                    // every eight columns of an output and residual row are aligned for 16-byte accesses
  int splits, kb_per_split;     // parts of the k-blocks, none of them empty
  int stages;
  const void* x;                // rows that the kernel quantises itself (else they are in `a`), K of them and ldx apart; x_vec: every eight aligned for 16-byte loads
  long long ldx;
  int K, x_fp32, x_vec;
  int early;                    // weights may be fetched before the kernel in front has finished (it does not write them, nor do those before it)
  int* status;
  int pdl;
};

constexpr int FP4_TILE = 128;                                    // weight rows of a CTA
constexpr int FP4_W_BYTES = FP4_TILE * 128;                      // codes of a k-block
__host__ __device__ constexpr int fp4_sf_bytes(int form) { return fp4_steps(form) * FP4_SCALE_STEP; }

// ------------------------------------------------------------------------------- tensor-core wrappers
// Instruction descriptor of the block-scaled e2m1 products: both operands e2m1 and K-major; bit 23 tells e8m0 from e4m3 scales; the scale ids say which of
// a column's four bytes belong to this instruction (0, or 2 where it takes two).
__host__ __device__ constexpr uint32_t fp4_idesc(int form, int m, int n, int id) {
  return (1u << 7) | (1u << 10) | (uint32_t(id) << 4) | (uint32_t(n >> 3) << 17) | (form == FP4_MX ? 1u << 23 : 0u) | (uint32_t(m >> 7) << 27) | (uint32_t(id) << 29);
}
// Shared-memory descriptor of 32 x 16 bytes without swizzle (groups of eight rows 128 bytes apart): what a copy of scales reads.
__device__ __forceinline__ uint64_t fp4_scale_desc(uint32_t addr) {
  return uint64_t((addr & 0x3FFFF) >> 4) | (uint64_t(1) << 16) | (uint64_t(128 >> 4) << 32) | (uint64_t(1) << 46);
}
template <int CTAS>
__device__ __forceinline__ void fp4_copy_scales(uint32_t taddr, uint64_t desc) {     // 512 bytes -> four columns, in all four lane quarters
  if constexpr (CTAS == 1) asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
#define FP4_MMA(GROUP, VEC)                                                                                                              \
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                                                           \
               "tcgen05.mma.cta_group::" GROUP ".kind::mxf4nvf4.block_scale.scale_vec::" VEC " [%0], %1, %2, %3, [%4], [%5], p;\n\t}"           \
               ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory")
template <int CTAS, int FORM>
__device__ __forceinline__ void fp4_mma(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
  if constexpr (CTAS == 1) { if constexpr (FORM == FP4_NV) FP4_MMA("1", "4X"); else FP4_MMA("1", "2X"); }
  else { if constexpr (FORM == FP4_NV) FP4_MMA("2", "4X"); else FP4_MMA("2", "2X"); }
}

// ------------------------------------------------------------------------------- results
// v / (1 + exp(-v)) by the approximate power of two and reciprocal, a few 2^-23 off; below some -87, where the result is under 2^-119, zero.  Neither looks at subnormal
// numbers, which one added to an exponential that small would not show.  (8192 gated tokens of 4096 -> 2 x 14336: 420 us; with __expf, 424; with an IEEE division, some 510.)
__device__ __forceinline__ float fp4_silu(float v) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * -1.44269504f));
  return v * reciprocal(1.f + e);
}
// Eight columns of token row m: residual and store.
__device__ __forceinline__ void fp4_store8(const Fp4LinearArgs& p, int m, int col, float (&v)[8]) {
  const int n = min(8, p.n_out - col);
  const bool whole = p.whole && n == 8;
  if (p.residual) {
    if (p.res_fp32) {
      const float* r = static_cast<const float*>(p.residual) + m * p.ldr + col;
      if (whole) {
        const float4 x = reinterpret_cast<const float4*>(r)[0], y = reinterpret_cast<const float4*>(r)[1];
        v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w; v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (j < n) v[j] += r[j];
      }
    } else {
      const __nv_bfloat16* r = static_cast<const __nv_bfloat16*>(p.residual) + m * p.ldr + col;
      if (whole) {
        const uint4 q = *reinterpret_cast<const uint4*>(r);
        const float2 x0 = unpack_bf16x2(q.x), x1 = unpack_bf16x2(q.y), x2 = unpack_bf16x2(q.z), x3 = unpack_bf16x2(q.w);
        v[0] += x0.x; v[1] += x0.y; v[2] += x1.x; v[3] += x1.y; v[4] += x2.x; v[5] += x2.y; v[6] += x3.x; v[7] += x3.y;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (j < n) v[j] += bf2f(r[j]);
      }
    }
  }
  if (p.out_fp32) {
    float* c = static_cast<float*>(p.C) + m * p.ldc + col;
    if (whole) {
      reinterpret_cast<float4*>(c)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(c)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) if (j < n) c[j] = v[j];
    }
  } else {
    __nv_bfloat16* c = static_cast<__nv_bfloat16*>(p.C) + m * p.ldc + col;
    if (whole) {
      *reinterpret_cast<uint4*>(c) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) if (j < n) c[j] = f2bf(v[j]);
    }
  }
}

int LaunchPairLinearFp4(const Fp4LinearArgs& p, int form, int sm_count, cudaStream_t stream);   // linear_fp4_pair.cu

}  // namespace ogb
