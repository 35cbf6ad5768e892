// A whole mixture-of-experts layer for up to eight tokens in two kernels, bound by the bytes of the experts that the tokens meet.
//
// few_gate_up_kernel: every cluster of eight CTAs computes all router logits for itself (an eighth of the experts per CTA, exchanged through distributed
// shared memory), so that each CTA can choose the experts, list those that any token meets, and go on to their gate and up rows without a kernel or a
// grid barrier in between; the router is small beside the experts and comes from L2.  A warp computes eight features of one expert for all tokens: the
// rows of an `mma.sync` tile of 16 are eight gate rows and the eight up rows of the same features, its columns the tokens, so that a thread holds a
// gate and its up value and writes share * act(gate, up).
// few_down_kernel: a CTA computes 16 columns of the output; its warps take equal parts of the sequence (expert, k) and are summed in warp order.
//
// `mma.sync` is used on purpose: its eight columns are the eight tokens, and the operands go from memory to registers in the order in which they lie:
// the k index of a product is permuted alike for both operands, so a lane's share of a row is one contiguous load.  A lane keeps several chunks of 64 k
// values in flight, in a ring that runs on from one unit of work to the next.
//
// Roundings: the router's logits, all sums and the activation are fp32.  The activations times routing weights travel between the kernels in 16 bits (the
// operand type of the second product): bf16, or, with packed experts in their fp16 form, fp16, where values beyond 65504 become that.  The rows meet packed
// experts of that form as fp16 after a scaling by a power of two per token, which loses nothing within 2^-38 of a row's largest value.
#include <cuda_fp16.h>
#include <math.h>

#include "kernels.h"
#include "packed_weights.cuh"

namespace ogb {

enum FewWeights : int { FEW_BF16 = 0, FEW_FP4_F16 = 1, FEW_FP4_BF16 = 2 };   // packed: the records of gemm_fp4.cu in their two forms
constexpr int FEW_TOKENS = 8, FEW_TOP = 32, FEW_EXPERTS = 1024, FEW_MET = FEW_TOKENS * FEW_TOP;
constexpr int FEW_CLUSTER = 8;
constexpr int FEW_A_THREADS = 256, FEW_B_THREADS = 512;
constexpr size_t FEW_SMEM_TWO = 112 * 1024;

// What the first kernel leaves for the second.
struct FewPlan {
  int met, unused[3];                       // experts that any token meets, in ascending order
  int expert[FEW_MET];
  uint8_t slot[FEW_MET][FEW_TOKENS];        // which choice of the token the expert is; 255: none
  int ids[FEW_TOKENS * FEW_TOP];            // [token][choice]
  float share[FEW_TOKENS * FEW_TOP];
};
static_assert(sizeof(FewPlan) % 16 == 0, "h follows the plan");

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
  FewPlan* plan;
  uint16_t* h;          // [T * top, I], in groups of eight as the second product reads them
};

// ------------------------------------------------------------------------------- operands
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  const uint32_t a[4] = {a0, a1, a2, a3};
  mma_bf16_16816(d, a, b0, b1);
}
// two mma of 16 k values each: a lane brings eight values of each of its rows (in pairs) and of its token
__device__ __forceinline__ void mma_bf16_32(float (&d)[4], const uint4& r0, const uint4& r1, const uint4& b) {
  mma_bf16_16816(d, r0.x, r1.x, r0.y, r1.y, b.x, b.y);
  mma_bf16_16816(d, r0.z, r1.z, r0.w, r1.w, b.z, b.w);
}
__device__ __forceinline__ uint4 ld_stream(const void* p) {         // weights are read once: they need no place in L1
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld_stream2(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

// Two weight rows of a warp's tile (row lane / 4 of each half), k values 64 c .. 64 c + 63: a lane's 16 of each row.
template <int W> struct FewChunk;
template <> struct FewChunk<FEW_BF16> {
  uint4 a[2][2];
  // p0, p1: the lane's place in the rows; left: k values from there to the rows' end
  __device__ __forceinline__ void load(const uint8_t* p0, const uint8_t* p1, int left) {
    const uint4 zero = make_uint4(0, 0, 0, 0);
    a[0][0] = left > 0 ? ld_stream(p0) : zero;
    a[1][0] = left > 0 ? ld_stream(p1) : zero;
    a[0][1] = left > 32 ? ld_stream(p0 + 64) : zero;
    a[1][1] = left > 32 ? ld_stream(p1 + 64) : zero;
  }
  __device__ __forceinline__ void mma(float (&acc)[4], const uint4 (&b)[2]) const {
    mma_bf16_32(acc, a[0][0], a[1][0], b[0]);
    mma_bf16_32(acc, a[0][1], a[1][1], b[1]);
  }
};
__device__ __forceinline__ float fp4_half_scale(uint32_t s) { return __uint_as_float((s - 6u) << 23); }      // the records hold code + 6
template <> struct FewChunk<FEW_FP4_F16> {
  uint2 q[2];
  uint16_t s[2];
  // p: the lane's eight bytes of a row's record, ps: the row's two scales
  __device__ __forceinline__ void load(const uint8_t* p0, const uint8_t* p1, const uint8_t* ps0, const uint8_t* ps1) {
    q[0] = ld_stream2(p0);
    q[1] = ld_stream2(p1);
    s[0] = __ldg(reinterpret_cast<const uint16_t*>(ps0));
    s[1] = __ldg(reinterpret_cast<const uint16_t*>(ps1));
  }
  // a block of 32 has one scale per row: its sum is scaled as a whole
  __device__ __forceinline__ void mma(float (&acc)[4], const uint4 (&b)[2]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t u[4], v[4];
      cvt_e2m1x8_f16(i ? q[0].y : q[0].x, u);
      cvt_e2m1x8_f16(i ? q[1].y : q[1].x, v);
      float t[4] = {0.f, 0.f, 0.f, 0.f};
      mma_f16_16816(t, u[0], v[0], u[1], v[1], b[i].x, b[i].y);
      mma_f16_16816(t, u[2], v[2], u[3], v[3], b[i].z, b[i].w);
      const float s0 = fp4_half_scale(i ? s[0] >> 8 : s[0] & 255), s1 = fp4_half_scale(i ? s[1] >> 8 : s[1] & 255);
      acc[0] = fmaf(t[0], s0, acc[0]);
      acc[1] = fmaf(t[1], s0, acc[1]);
      acc[2] = fmaf(t[2], s1, acc[2]);
      acc[3] = fmaf(t[3], s1, acc[3]);
    }
  }
};
template <> struct FewChunk<FEW_FP4_BF16> {
  uint32_t q[2][2];
  uint16_t s[2];
  __device__ __forceinline__ void load(const uint8_t* p0, const uint8_t* p1, const uint8_t* ps0, const uint8_t* ps1) {
    q[0][0] = __ldg(reinterpret_cast<const uint32_t*>(p0));
    q[0][1] = __ldg(reinterpret_cast<const uint32_t*>(p0 + 16));
    q[1][0] = __ldg(reinterpret_cast<const uint32_t*>(p1));
    q[1][1] = __ldg(reinterpret_cast<const uint32_t*>(p1 + 16));
    s[0] = __ldg(reinterpret_cast<const uint16_t*>(ps0));
    s[1] = __ldg(reinterpret_cast<const uint16_t*>(ps1));
  }
  __device__ __forceinline__ void mma(float (&acc)[4], const uint4 (&b)[2]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      mma_bf16_32(acc, deq_fp4_word_bf16(q[0][i], i ? s[0] >> 8 : s[0] & 255), deq_fp4_word_bf16(q[1][i], i ? s[1] >> 8 : s[1] & 255), b[i]);
  }
};

// A place in the weights: the rows r0 and r1 (in one tile of 128) of expert e, going up in steps of 64 k values.
template <int W>
struct FewRows {
  const uint8_t *p0, *p1, *s0, *s1;
  long long step;
  int left;
  __device__ __forceinline__ void seek(const void* w, int e, int N, int K, int r0, int r1, int chunk, int q) {
    const uint8_t* base = static_cast<const uint8_t*>(w);
    if constexpr (W == FEW_BF16) {
      left = K - chunk * 64 - q * 8;
      p0 = base + (((long long)e * N + r0) * K + chunk * 64 + q * 8) * 2;
      p1 = base + (((long long)e * N + r1) * K + chunk * 64 + q * 8) * 2;
      step = 128;
    } else {
      const int tiles = (N + 127) >> 7;
      const uint8_t* rec = base + (((long long)e * (K >> 6) + chunk) * tiles + (r0 >> 7)) * FP4_RECORD_BYTES;
      const int at = W == FEW_FP4_F16 ? q * 8 : q * 4;
      p0 = rec + (r0 & 127) * 32 + at;
      p1 = rec + (r1 & 127) * 32 + at;
      s0 = rec + 128 * 32 + (r0 & 127) * 2;
      s1 = rec + 128 * 32 + (r1 & 127) * 2;
      step = (long long)tiles * FP4_RECORD_BYTES;
    }
  }
  __device__ __forceinline__ void load(FewChunk<W>& c) const {
    if constexpr (W == FEW_BF16) c.load(p0, p1, left); else c.load(p0, p1, s0, s1);
  }
  __device__ __forceinline__ void next() {
    p0 += step;
    p1 += step;
    if constexpr (W == FEW_BF16) left -= 64; else { s0 += step; s1 += step; }
  }
};

// Eight 16-bit values in the order in which a lane's eight weights of a row come out of their load: pairs (0, 1) (2, 3) .. or, from records in fp16 form,
// (0, 4) (1, 5) (2, 6) (3, 7).
template <int W> __device__ __forceinline__ int few_place(int i) { return W == FEW_FP4_F16 ? (i & 3) * 2 + (i >> 2) : i; }
__device__ __forceinline__ uint32_t f16x2_sat(float lo, float hi) {          // NaN stays NaN
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// ------------------------------------------------------------------------------- router, choice
// Shared memory of the first kernel.
struct FewShared {
  float red[8][16 * FEW_TOKENS];
  uint32_t top[FEW_TOKENS];          // bits of the rows' largest magnitudes
  uint32_t mask[FEW_EXPERTS];        // tokens that meet an expert
  FewPlan plan;
};

// Power of two that brings a row's largest magnitude (its bits) to 2^14 .. 2^15
__device__ __forceinline__ int few_shift(uint32_t top) { return top >= 0x7f800000u ? 0 : min(14 - (int(top >> 23) - 127), 126); }
// A float as an unsigned number of the same order; 0: not a number.
__device__ __forceinline__ uint32_t few_key(float v) {
  const uint32_t u = __float_as_uint(v);
  return v != v ? 0u : u & 0x80000000u ? ~u : u | 0x80000000u;
}
// Choice of `top` experts for a token by one warp: the largest logits, the lowest index among equal ones; a token whose logits are not numbers takes
// expert 0.  A lane holds every 32nd expert and looks for its best one anew only when that was taken.
__device__ __forceinline__ void few_choose(const float* row, int E, int top, int rule, int lane, int& id, float& share) {
  uint32_t taken = 0, best = 0;      // taken, bit i: expert lane + 32 i
  int at = 0x7fffffff;
  bool bad = false;
  auto scan = [&]() {
    best = 0;
    at = 0x7fffffff;
    for (int i = 0, e = lane; e < E; ++i, e += 32) {
      const uint32_t k = taken >> i & 1 ? 0u : few_key(row[e]);
      if (k > best) { best = k; at = e; }
    }
  };
  for (int e = lane; e < E; e += 32) bad |= row[e] != row[e];
  bad = __any_sync(0xffffffffu, bad);
  scan();
  float most = 0.f, mine = 0.f;
  id = 0;
  for (int j = 0; j < top; ++j) {
    const uint32_t k = __reduce_max_sync(0xffffffffu, best);
    const int e = int(__reduce_min_sync(0xffffffffu, best == k && k ? uint32_t(at) : 0x7fffffffu));
    const float v = __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
    if (j == 0) most = v;
    if (lane == j) { mine = v; id = k ? e : 0; }
    if (k && at == e) { taken |= 1u << (e >> 5); scan(); }
  }
  const float w = lane < top ? expf(mine - most) : 0.f;
  float sum = warp_sum(w);
  if (rule == 1) {
    sum = 0.f;
    for (int e = lane; e < E; e += 32) sum += expf(row[e] - most);
    sum = warp_sum(sum);
  }
  share = bad ? __uint_as_float(0x7fc00000u) : w / sum;
}

template <int W>
__global__ void __launch_bounds__(FEW_A_THREADS, 2) few_gate_up_kernel(const FewArgs p) {
  constexpr int DEPTH = W == FEW_BF16 ? 4 : 8;
  extern __shared__ __align__(16) uint8_t smem[];
  FewShared& sh = *reinterpret_cast<FewShared*>(smem);
  float* logits = reinterpret_cast<float*>(smem + sizeof(FewShared));                       // [T][E]
  const int Hp = (p.H + 63) / 64 * 64, xs_ld = Hp + 32;              // 16-bit values a row: neighbours start 64 bytes apart in the banks
  uint16_t* xs = reinterpret_cast<uint16_t*>(smem + sizeof(FewShared) + (size_t(p.T) * p.E * 4 + 15) / 16 * 16);
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int rank = int(cluster_ctarank());
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");      // the others' shared memory is written only once they run
  for (int e = threadIdx.x; e < p.E; e += FEW_A_THREADS) sh.mask[e] = 0;
  if (threadIdx.x < FEW_TOKENS) sh.top[threadIdx.x] = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();

  // the largest magnitude of every row, where the rows are to be scaled: a warp takes 256 values of a token at a time
  const int parts = (Hp + 255) >> 8, pieces = p.T * parts;
  if (W == FEW_FP4_F16) {
#pragma unroll 4
    for (int i = warp; i < pieces; i += 8) {
      const int t = i / parts, k = (i - t * parts) * 256 + lane * 8;
      const uint4 v = k < p.H ? *reinterpret_cast<const uint4*>(p.x + t * p.ldx + k) : make_uint4(0, 0, 0, 0);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) top = max(top, max(w[j] << 16 & 0x7fffffffu, w[j] & 0x7fff0000u));
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0) atomicMax(&sh.top[t], top);
    }
  }

  // router logits of this CTA's experts: 16 experts x 8 tokens at a time, the warps share k
  const int per = (p.E + FEW_CLUSTER - 1) / FEW_CLUSTER, e_end = min(p.E, (rank + 1) * per);
  bool met_cluster = false;
  for (int e0 = rank * per; e0 < (rank + 1) * per; e0 += 16) {               // (the same number of rounds in every CTA)
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    const bool r0 = e0 + g < e_end, r1 = e0 + g + 8 < e_end;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const __nv_bfloat16* w0 = p.router + (long long)(r0 ? e0 + g : 0) * p.H;
    const __nv_bfloat16* w1 = p.router + (long long)(r1 ? e0 + g + 8 : 0) * p.H;
#pragma unroll 4
    for (int k = warp * 32 + q * 8; k < (p.H + 31) / 32 * 32; k += 256) {
      const bool in = k < p.H;
      const uint4 a0 = r0 && in ? *reinterpret_cast<const uint4*>(w0 + k) : zero, a1 = r1 && in ? *reinterpret_cast<const uint4*>(w1 + k) : zero;
      const uint4 b = g < p.T && in ? *reinterpret_cast<const uint4*>(p.x + g * p.ldx + k) : zero;
      mma_bf16_32(acc, a0, a1, b);
    }
    *reinterpret_cast<float2*>(&sh.red[warp][g * 8 + q * 2]) = make_float2(acc[0], acc[1]);
    *reinterpret_cast<float2*>(&sh.red[warp][(g + 8) * 8 + q * 2]) = make_float2(acc[2], acc[3]);
    __syncthreads();
    if (!met_cluster) { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); met_cluster = true; }
    if (threadIdx.x < 128) {
      const int e = e0 + int(threadIdx.x >> 3), t = threadIdx.x & 7;
      if (e < e_end && t < p.T) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) v += sh.red[w][threadIdx.x];
        if (p.router_b) v += bf2f(p.router_b[e]);
        const uint32_t at = smem_u32(logits + t * p.E + e);
#pragma unroll
        for (uint32_t r = 0; r < FEW_CLUSTER; ++r) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dsmem_addr(at, r)), "f"(v) : "memory");
      }
    }
    __syncthreads();
  }
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  // the rows as the products read them
#pragma unroll 4
  for (int i = warp; i < pieces; i += 8) {
    const int t = i / parts, k = (i - t * parts) * 256 + lane * 8;
    uint4 v = k < p.H ? *reinterpret_cast<const uint4*>(p.x + t * p.ldx + k) : make_uint4(0, 0, 0, 0);
    if (W == FEW_FP4_F16) {
      const float scale = __uint_as_float(uint32_t(few_shift(sh.top[t]) + 127) << 23);
      const float2 a = unpack_bf16x2(v.x), b = unpack_bf16x2(v.y), c = unpack_bf16x2(v.z), d = unpack_bf16x2(v.w);
      v = make_uint4(pack_f16x2(a.x * scale, c.x * scale), pack_f16x2(a.y * scale, c.y * scale), pack_f16x2(b.x * scale, d.x * scale),
                     pack_f16x2(b.y * scale, d.y * scale));
    }
    if (k < Hp) *reinterpret_cast<uint4*>(xs + t * xs_ld + k) = v;
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

  // choices, and the experts that any token meets
  if (warp < p.T) {
    int id;
    float share;
    few_choose(logits + warp * p.E, p.E, p.top, p.rule, lane, id, share);
    if (lane < p.top) {
      sh.plan.ids[warp * p.top + lane] = id;
      sh.plan.share[warp * p.top + lane] = share;
      atomicOr(&sh.mask[id], 1u << warp);
    }
  }
  __syncthreads();
  if (warp == 0) {
    int n = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const bool here = e0 + lane < p.E && sh.mask[e0 + lane];
      const uint32_t b = __ballot_sync(0xffffffffu, here);
      const int at = n + __popc(b & ((1u << lane) - 1));
      if (here) {
        sh.plan.expert[at] = e0 + lane;
        *reinterpret_cast<uint2*>(sh.plan.slot[at]) = make_uint2(0xffffffffu, 0xffffffffu);
        sh.mask[e0 + lane] = uint32_t(at);         // from here on: the expert's place in the list
      }
      n += __popc(b);
    }
    if (lane == 0) sh.plan.met = n;
    __syncwarp();
    for (int i = lane; i < p.T * p.top; i += 32) sh.plan.slot[sh.mask[sh.plan.ids[i]]][i / p.top] = uint8_t(i % p.top);
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    const uint4* src = reinterpret_cast<const uint4*>(&sh.plan);
    for (int i = threadIdx.x; i < int(sizeof(FewPlan) / 16); i += FEW_A_THREADS) reinterpret_cast<uint4*>(p.plan)[i] = src[i];
  }

  // gate and up rows: a unit is eight features of a met expert; neighbours in memory are at work at the same time
  const int blocks = p.I >> 3, units = sh.plan.met * blocks, stride = int(gridDim.x) * 8, chunks = Hp >> 6;
  FewChunk<W> ring[DEPTH];
  FewRows<W> rows;
  int lu = int(blockIdx.x) + int(gridDim.x) * warp, lc = 0;                  // where the loads are
  auto seek = [&]() {
    if (lu < units) {
      const int d = lu / blocks, f = (lu - d * blocks) * 8 + g, r = (f >> 6) * 128 + (f & 63);
      rows.seek(p.gate_up, sh.plan.expert[d], 2 * p.I, p.H, r, r + 64, 0, q);
    }
  };
  auto fetch = [&](FewChunk<W>& c) {
    if (lu >= units) return;
    rows.load(c);
    if (++lc < chunks) { rows.next(); return; }
    lc = 0;
    lu += stride;
    seek();
  };
  seek();
#pragma unroll
  for (int i = 0; i < DEPTH; ++i) fetch(ring[i]);
  const uint16_t* xt = xs + (g < p.T ? g : 0) * xs_ld + q * 8;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  int u = int(blockIdx.x) + int(gridDim.x) * warp, c = 0;                    // where the products are
  while (u < units) {
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
      if (u >= units) break;
      // columns beyond the tokens: any numbers, they are not looked at
      const uint4 b[2] = {*reinterpret_cast<const uint4*>(xt + c * 64), *reinterpret_cast<const uint4*>(xt + c * 64 + 32)};
      ring[i].mma(acc, b);
      fetch(ring[i]);
      if (++c < chunks) continue;
      const int d = u / blocks, i0 = (u - d * blocks) * 8, e = sh.plan.expert[d], r = ((i0 + g) >> 6) * 128 + ((i0 + g) & 63);
      const float bg = p.gate_up_b ? bf2f(p.gate_up_b[(long long)e * 2 * p.I + r]) : 0.f, bu = p.gate_up_b ? bf2f(p.gate_up_b[(long long)e * 2 * p.I + r + 64]) : 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int t = q * 2 + j, slot = sh.plan.slot[d][t];
        if (slot != 255) {
          const float s = W == FEW_FP4_F16 ? __uint_as_float(uint32_t(127 - few_shift(sh.top[t])) << 23) : 1.f;
          float gate = fmaf(acc[j], s, bg), up = fmaf(acc[2 + j], s, bu), v;
          if (p.act == 2) {
            if (p.limit > 0.f) {             // (comparisons, not minima: what is not a number stays that)
              gate = gate > p.limit ? p.limit : gate;
              up = up > p.limit ? p.limit : up < -p.limit ? -p.limit : up;
            }
            v = gate / (1.f + expf(-p.alpha * gate)) * (up + 1.f);
          } else {
            v = gate / (1.f + expf(-gate)) * up;
          }
          const int pair = t * p.top + slot;
          v *= sh.plan.share[pair];
          const uint32_t bits = W == FEW_FP4_F16 ? f16x2_sat(v, 0.f) : pack_bf16x2(v, 0.f);
          p.h[(long long)pair * p.I + i0 + few_place<W>(g)] = uint16_t(bits);
        }
        acc[j] = acc[2 + j] = 0.f;
      }
      c = 0;
      u += stride;
    }
  }
}

template <int W>
__global__ void __launch_bounds__(FEW_B_THREADS, 1) few_down_kernel(const FewArgs p) {
  constexpr int DEPTH = W == FEW_BF16 ? 3 : 6, WARPS = FEW_B_THREADS / 32;
  __shared__ FewPlan plan;
  __shared__ float red[WARPS][16 * FEW_TOKENS];
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int n0 = blockIdx.x * 16;
  pdl_wait();
  pdl_launch_dependents();
  {
    const uint4* src = reinterpret_cast<const uint4*>(p.plan);
    for (int i = threadIdx.x; i < int(sizeof(FewPlan) / 16); i += FEW_B_THREADS) reinterpret_cast<uint4*>(&plan)[i] = src[i];
  }
  __syncthreads();
  const int chunks = p.I >> 6, total = plan.met * chunks;
  const int lo = int((long long)total * warp / WARPS), hi = int((long long)total * (warp + 1) / WARPS);
  const int r0 = min(n0 + g, p.H - 1), r1 = min(n0 + g + 8, p.H - 1);        // rows past the end: any, they are not stored

  struct Item { FewChunk<W> w; uint4 h[2]; };
  Item ring[DEPTH];
  FewRows<W> rows;
  const uint16_t* hp = nullptr;                                               // this lane's token's activations of the expert; null: it does not meet it
  int at = lo, ld = 0, lc = 0;
  auto seek = [&]() {
    if (at >= hi) return;
    ld = at / chunks;
    lc = at - ld * chunks;
    rows.seek(p.down, plan.expert[ld], p.H, p.I, r0, r1, lc, q);
    const int slot = plan.slot[ld][g];
    hp = slot == 255 ? nullptr : p.h + (long long)(g * p.top + slot) * p.I + lc * 64 + q * 8;
  };
  auto fetch = [&](Item& it) {
    if (at >= hi) return;
    rows.load(it.w);
    it.h[0] = hp ? *reinterpret_cast<const uint4*>(hp) : make_uint4(0, 0, 0, 0);
    it.h[1] = hp ? *reinterpret_cast<const uint4*>(hp + 32) : make_uint4(0, 0, 0, 0);
    ++at;
    if (++lc < chunks) { rows.next(); if (hp) hp += 64; } else seek();
  };
  seek();
#pragma unroll
  for (int i = 0; i < DEPTH; ++i) fetch(ring[i]);
  float sum[4] = {0.f, 0.f, 0.f, 0.f}, acc[4] = {0.f, 0.f, 0.f, 0.f};
  int c = lo < hi ? lo % chunks : 0, d = lo < hi ? lo / chunks : 0;
  for (int i0 = lo; i0 < hi; i0 += DEPTH) {
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
      if (i0 + i >= hi) break;
      ring[i].w.mma(acc, ring[i].h);
      fetch(ring[i]);
      if (++c < chunks && i0 + i + 1 < hi) continue;
      // an expert's part is done: it counts for the tokens that meet it (weights that are not numbers stay with them)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (plan.slot[d][q * 2 + j] != 255) { sum[j] += acc[j]; sum[2 + j] += acc[2 + j]; }
        acc[j] = acc[2 + j] = 0.f;
      }
      c = 0;
      ++d;
    }
  }
  *reinterpret_cast<float2*>(&red[warp][g * 8 + q * 2]) = make_float2(sum[0], sum[1]);
  *reinterpret_cast<float2*>(&red[warp][(g + 8) * 8 + q * 2]) = make_float2(sum[2], sum[3]);
  __syncthreads();
  if (threadIdx.x < 128) {
    const int n = n0 + int(threadIdx.x & 15), t = threadIdx.x >> 4;
    if (t < p.T && n < p.H) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) v += red[w][(threadIdx.x & 15) * 8 + t];
      if (p.down_b)
        for (int j = 0; j < p.top; ++j) v += plan.share[t * p.top + j] * bf2f(p.down_b[(long long)plan.ids[t * p.top + j] * p.H + n]);
      p.out[(long long)t * p.H + n] = f2bf(v);
    }
  }
}

template <int W>
static int LaunchFew(const FewArgs& p, cudaStream_t stream) {
  const int Hp = (p.H + 63) / 64 * 64, xs_ld = Hp + 32;
  const size_t smem = sizeof(FewShared) + (size_t(p.T) * p.E * 4 + 15) / 16 * 16 + size_t(p.T) * xs_ld * 2;
  if (smem > 227 * 1024) return -5;
  static bool configured[OGB_MAX_DEVICES] = {};
  if (!set_max_dyn_smem(few_gate_up_kernel<W>, 227 * 1024, configured)) return -3;
  static const int pdl = [] { const char* e = getenv("OGB_PDL"); return (e && e[0] == '0') ? 0 : 1; }();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {FEW_CLUSTER, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(FEW_A_THREADS);
  cfg.stream = stream;
  cfg.gridDim = dim3(FEW_CLUSTER);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // As many clusters as run at once, two CTAs an SM or, with long rows, one.
  static int clusters_at[OGB_MAX_DEVICES][2] = {};
  const int two = smem <= FEW_SMEM_TWO;
  int dev = 0, clusters = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -4;
  const bool tracked = dev >= 0 && dev < OGB_MAX_DEVICES;
  if (tracked) clusters = clusters_at[dev][two];
  if (!clusters) {
    cfg.dynamicSmemBytes = two ? FEW_SMEM_TWO : 227 * 1024;
    if (cudaOccupancyMaxActiveClusters(&clusters, few_gate_up_kernel<W>, &cfg) != cudaSuccess || clusters < 1) return -4;
    if (tracked) clusters_at[dev][two] = clusters;
  }
  cfg.dynamicSmemBytes = smem;
  cfg.gridDim = dim3(unsigned(clusters * FEW_CLUSTER));
  cfg.numAttrs = pdl ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, few_gate_up_kernel<W>, p) != cudaSuccess) return -4;
  return launch_pdl(few_down_kernel<W>, dim3(unsigned((p.H + 15) / 16)), dim3(FEW_B_THREADS), 0, stream, p) ? 0 : -4;
}

}  // namespace ogb

using namespace ogb;

OGB_API long long ogb_moe_few_scratch_bytes(int T, int top, int I) {
  return T < 1 || T > FEW_TOKENS || top < 1 || top > FEW_TOP || I < 1 ? -1 : (long long)sizeof(FewPlan) + (long long)T * top * I * 2;
}

OGB_API int ogb_moe_few_tokens(const void* x, long long ldx, const void* router, const void* router_b, const void* gate_up, const void* gate_up_b,
                               const void* down, const void* down_b, void* out, int T, int H, int I, int E, int top, int rule, int weights, int act,
                               float alpha, float limit, void* scratch, void* stream) {
  if (ogb_moe_few_scratch_bytes(T, top, I) < 0 || !x || !router || !gate_up || !down || !out || !scratch || H < 1 || H % 8 || E < top || E > FEW_EXPERTS ||
      I % 64 || (weights != FEW_BF16 && H % 64) || rule < 0 || rule > 2 || weights < 0 || weights > 2 || (act != 1 && act != 2)) return -1;
  if ((reinterpret_cast<uintptr_t>(x) | uintptr_t(ldx * 2) | reinterpret_cast<uintptr_t>(router) | reinterpret_cast<uintptr_t>(gate_up) | reinterpret_cast<uintptr_t>(down) | reinterpret_cast<uintptr_t>(scratch)) & 15)
    return -1;
  FewArgs p{static_cast<const __nv_bfloat16*>(x), ldx, static_cast<const __nv_bfloat16*>(router), static_cast<const __nv_bfloat16*>(router_b), gate_up,
            static_cast<const __nv_bfloat16*>(gate_up_b), down, static_cast<const __nv_bfloat16*>(down_b), static_cast<__nv_bfloat16*>(out), T, H, I, E, top,
            rule, act, alpha, limit, static_cast<FewPlan*>(scratch), reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(scratch) + sizeof(FewPlan))};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (weights == FEW_BF16) return LaunchFew<FEW_BF16>(p, s);
  return weights == FEW_FP4_F16 ? LaunchFew<FEW_FP4_F16>(p, s) : LaunchFew<FEW_FP4_BF16>(p, s);
}
