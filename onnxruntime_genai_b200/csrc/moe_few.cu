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
constexpr int FEW_THREADS = 288, FEW_STAGES = 16;
constexpr size_t FEW_SMEM_TWO = 112 * 1024, FEW_SMEM_ONE = 227 * 1024;          // shared memory of a CTA, with two or one on an SM
constexpr int FEW_DOWN_RING = 72 * 1024;

// What the first kernel leaves for the second.
struct alignas(16) FewPlan {
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
  int stages, splits;   // of the first kernel's ring; CTAs of a cluster of the second
  int* status;
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
// A stage of the ring holds CHUNKS steps of 64 k values of a tile of 128 weight rows, as they lie in memory: packed records, or (bf16) a box of 64 columns with
// the 128-byte swizzle.  A warp multiplies 16 of the rows, r0 = the row of lanes 4 g .. 4 g + 3 in the tile's first half of its 16, r1 in the second.
template <int W>
struct FewTile {
  static constexpr int CHUNKS = W == FEW_BF16 ? 1 : 2;
  static constexpr int BYTES = W == FEW_BF16 ? 128 * 128 : FP4_RECORD_BYTES;       // of a step
  static __device__ __forceinline__ void mma(float (&acc)[4], const uint8_t* tile, int r0, int r1, int g, int q, const uint4 (&b)[2]) {
    if constexpr (W == FEW_BF16) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = ((q + 4 * i) ^ g) << 4;
        mma_bf16_32(acc, *reinterpret_cast<const uint4*>(tile + r0 * 128 + c), *reinterpret_cast<const uint4*>(tile + r1 * 128 + c), b[i]);
      }
    } else if constexpr (W == FEW_FP4_F16) {
      const uint2 q0 = *reinterpret_cast<const uint2*>(tile + r0 * 32 + q * 8), q1 = *reinterpret_cast<const uint2*>(tile + r1 * 32 + q * 8);
      const uint32_t s0 = *reinterpret_cast<const uint16_t*>(tile + 128 * 32 + r0 * 2), s1 = *reinterpret_cast<const uint16_t*>(tile + 128 * 32 + r1 * 2);
#pragma unroll
      for (int i = 0; i < 2; ++i) {                       // a block of 32 has one scale per row (the records hold code + 6): its sum is scaled as a whole
        uint32_t u[4], v[4];
        cvt_e2m1x8_f16(i ? q0.y : q0.x, u);
        cvt_e2m1x8_f16(i ? q1.y : q1.x, v);
        float t[4] = {0.f, 0.f, 0.f, 0.f};
        mma_f16_16816(t, u[0], v[0], u[1], v[1], b[i].x, b[i].y);
        mma_f16_16816(t, u[2], v[2], u[3], v[3], b[i].z, b[i].w);
        const float f0 = __uint_as_float(((i ? s0 >> 8 : s0 & 255u) - 6u) << 23), f1 = __uint_as_float(((i ? s1 >> 8 : s1 & 255u) - 6u) << 23);
        acc[0] = fmaf(t[0], f0, acc[0]);
        acc[1] = fmaf(t[1], f0, acc[1]);
        acc[2] = fmaf(t[2], f1, acc[2]);
        acc[3] = fmaf(t[3], f1, acc[3]);
      }
    } else {
      const uint32_t s0 = *reinterpret_cast<const uint16_t*>(tile + 128 * 32 + r0 * 2), s1 = *reinterpret_cast<const uint16_t*>(tile + 128 * 32 + r1 * 2);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        mma_bf16_32(acc, deq_fp4_word_bf16(*reinterpret_cast<const uint32_t*>(tile + r0 * 32 + i * 16 + q * 4), i ? s0 >> 8 : s0 & 255u),
                    deq_fp4_word_bf16(*reinterpret_cast<const uint32_t*>(tile + r1 * 32 + i * 16 + q * 4), i ? s1 >> 8 : s1 & 255u), b[i]);
    }
  }
};
// Copies step `chunk` of 128 weight rows (tile `tile` of expert e's rows) to shared memory; by one thread.
template <int W>
__device__ __forceinline__ void few_copy(uint8_t* dst, uint64_t* bar, const CUtensorMap* map, const void* packed, int e, int tile, int chunk, int N, int K) {
  if constexpr (W == FEW_BF16) {
    tma_load_2d(dst, map, bar, chunk * 64, e * N + tile * 128);
  } else {
    const int tiles = (N + 127) >> 7;
    bulk_copy_g2s(dst, static_cast<const uint8_t*>(packed) + (((long long)e * (K >> 6) + chunk) * tiles + tile) * FP4_RECORD_BYTES, FP4_RECORD_BYTES, bar);
  }
}

// Eight 16-bit values in the order in which a lane's eight weights of a row come out of their load: pairs (0, 1) (2, 3) .. or, from records in fp16 form,
// (0, 4) (1, 5) (2, 6) (3, 7).
template <int W> __device__ __forceinline__ int few_place(int i) { return W == FEW_FP4_F16 ? (i & 3) * 2 + (i >> 2) : i; }
__device__ __forceinline__ uint32_t f16x2_sat(float lo, float hi) {          // NaN stays NaN
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// ------------------------------------------------------------------------------- ring of copies
// Warp 8 copies, warps 0 .. 7 multiply.  All waits are bounded; after a failed one every warp leaves its loop.
struct FewBars { uint64_t full[FEW_STAGES], empty[FEW_STAGES]; int abort; };
__device__ __forceinline__ void few_init(FewBars& b, int stages) {
  for (int s = 0; s < stages; ++s) { mbar_init(&b.full[s], 1); mbar_init(&b.empty[s], 8); }
  b.abort = 0;
  mbar_fence_init();
}
struct FewRing {
  int stages, s = 0, filled = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void next() {
    ++filled;
    if (++s == stages) { s = 0; ph ^= 1; }
  }
  __device__ __forceinline__ bool fail(FewBars& b, int* status) { atomicMax(status, OGB_ERR_WAIT_TMA); *reinterpret_cast<volatile int*>(&b.abort) = 1; return false; }
  __device__ __forceinline__ bool wait_empty(FewBars& b, int* status) {
    if (filled < stages) return true;
    return __all_sync(0xffffffffu, mbar_wait_bounded(&b.empty[s], ph ^ 1, &b.abort)) || fail(b, status);
  }
  // A consumer warp hands the stage before this one back only here.  Directly behind the products of its own stage the arrival could overtake reads of shared
  // memory that are still on their way (the compiler may put it in front of the products that wait for them; seen as single wrong rows); behind the wait for the
  // next stage all products, and so all reads, have been issued and answered.
  __device__ __forceinline__ bool wait_full(FewBars& b, int* status, int lane) {
    if (!__all_sync(0xffffffffu, mbar_wait_bounded(&b.full[s], ph, &b.abort))) return fail(b, status);
    if (filled > 0 && lane == 0) mbar_arrive(&b.empty[(s == 0 ? stages : s) - 1]);
    return true;
  }
  __device__ __forceinline__ void drain(FewBars& b) {          // copies in flight still write shared memory: give them time to land
    volatile int never = 0;
    for (int i = max(0, filled - stages); i < filled; ++i) mbar_wait_bounded(&b.full[i % stages], (i / stages) & 1, &never, 200000000ull);
  }
};

// ------------------------------------------------------------------------------- router, choice
// Shared memory of the first kernel.
struct FewShared {
  FewBars bars;
  float red[FEW_THREADS / 32][16 * FEW_TOKENS];
  uint32_t top[FEW_TOKENS];          // bits of the rows' largest magnitudes
  uint32_t mask[FEW_EXPERTS];        // tokens that meet an expert
  FewPlan plan;
};
static_assert(sizeof(FewShared) % 16 == 0, "16-byte accesses to what follows");

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
__global__ void __launch_bounds__(FEW_THREADS, 2) few_gate_up_kernel(const __grid_constant__ CUtensorMap map, const FewArgs p) {
  using Tile = FewTile<W>;
  constexpr int STAGE = Tile::CHUNKS * Tile::BYTES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  FewShared& sh = *reinterpret_cast<FewShared*>(ring + p.stages * STAGE);
  float* logits = reinterpret_cast<float*>(&sh + 1);                                         // [T][E]
  const int Hp = (p.H + 63) / 64 * 64, xs_ld = Hp + 32;              // 16-bit values a row: neighbours start 64 bytes apart in the banks
  uint16_t* xs = reinterpret_cast<uint16_t*>(reinterpret_cast<uint8_t*>(logits) + (size_t(p.T) * p.E * 4 + 15) / 16 * 16);
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int rank = int(cluster_ctarank());
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");      // the others' shared memory is written only once they run
  for (int e = threadIdx.x; e < p.E; e += FEW_THREADS) sh.mask[e] = 0;
  if (threadIdx.x < FEW_TOKENS) sh.top[threadIdx.x] = 0;
  if (threadIdx.x == 0) few_init(sh.bars, p.stages);
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();

  // the largest magnitude of every row, where the rows are to be scaled: a warp takes 256 values of a token at a time
  const int parts = (Hp + 255) >> 8, pieces = p.T * parts;
  if (W == FEW_FP4_F16) {
#pragma unroll 4
    for (int i = warp; i < pieces; i += FEW_THREADS / 32) {
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
    for (int k = warp * 32 + q * 8; k < (p.H + 31) / 32 * 32; k += FEW_THREADS) {
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
        for (int w = 0; w < FEW_THREADS / 32; ++w) v += sh.red[w][threadIdx.x];
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
  for (int i = warp; i < pieces; i += FEW_THREADS / 32) {
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
    for (int i = threadIdx.x; i < int(sizeof(FewPlan) / 16); i += FEW_THREADS) reinterpret_cast<uint4*>(p.plan)[i] = src[i];
  }

  // gate and up rows: an item is 64 features of a met expert, 128 rows that lie together; a warp takes eight features
  const int tiles = p.I >> 6, items = sh.plan.met * tiles, chunks = Hp >> 6;
  if (warp == 8) {
    FewRing r{p.stages};
    bool ok = true;
    for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
      const int e = sh.plan.expert[item / tiles], tile = item % tiles;
      for (int c = 0; c < chunks; c += Tile::CHUNKS) {
        ok = r.wait_empty(sh.bars, p.status);
        if (!ok) break;
        if (elect_one()) {
          const int n = min(Tile::CHUNKS, chunks - c);
          uint64_t* bar = &sh.bars.full[r.s];
          mbar_expect_tx(bar, n * Tile::BYTES);
          for (int i = 0; i < n; ++i) few_copy<W>(ring + r.s * STAGE + i * Tile::BYTES, bar, &map, p.gate_up, e, tile, c + i, 2 * p.I, p.H);
        }
        __syncwarp();
        r.next();
      }
    }
    if (!ok) r.drain(sh.bars);
    return;
  }
  FewRing r{p.stages};
  const uint16_t* xt = xs + (g < p.T ? g : 0) * xs_ld + q * 8;           // (columns beyond the tokens: any numbers, they are not looked at)
  const int r0 = warp * 8 + g;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int d = item / tiles, tile = item - d * tiles, e = sh.plan.expert[d], i0 = tile * 64 + warp * 8;
    const long long row = (long long)e * 2 * p.I + tile * 128 + r0;
    const float bg = p.gate_up_b ? bf2f(p.gate_up_b[row]) : 0.f, bu = p.gate_up_b ? bf2f(p.gate_up_b[row + 64]) : 0.f;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < chunks; c += Tile::CHUNKS) {
      if (!r.wait_full(sh.bars, p.status, lane)) return;
#pragma unroll
      for (int i = 0; i < Tile::CHUNKS; ++i) {
        if (i > 0 && c + i >= chunks) break;
        const uint4 b[2] = {*reinterpret_cast<const uint4*>(xt + (c + i) * 64), *reinterpret_cast<const uint4*>(xt + (c + i) * 64 + 32)};
        Tile::mma(acc, ring + r.s * STAGE + i * Tile::BYTES, r0, r0 + 64, g, q, b);
      }
      r.next();
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int t = q * 2 + j, slot = sh.plan.slot[d][t];
      if (slot == 255) continue;
      const float s = W == FEW_FP4_F16 ? __uint_as_float(uint32_t(127 - few_shift(sh.top[t])) << 23) : 1.f;
      float gate = fmaf(acc[j], s, bg), up = fmaf(acc[2 + j], s, bu), v = gate;
      if (p.act == 2) {
        if (p.limit > 0.f) {             // (comparisons, not minima: what is not a number stays that)
          gate = gate > p.limit ? p.limit : gate;
          up = up > p.limit ? p.limit : up < -p.limit ? -p.limit : up;
        }
        v = p.alpha * gate;
        up += 1.f;
      }
      const int pair = t * p.top + slot;
      v = gate / (1.f + expf(-v)) * up * sh.plan.share[pair];
      p.h[(long long)pair * p.I + i0 + few_place<W>(g)] = uint16_t(W == FEW_FP4_F16 ? f16x2_sat(v, 0.f) : pack_bf16x2(v, 0.f));
    }
  }
}

// A cluster computes 128 columns of the output, its CTAs take equal parts of the sequence (expert, k); partial sums are sent to the CTA that finishes their rows.
template <int W>
__global__ void __launch_bounds__(FEW_THREADS, 2) few_down_kernel(const __grid_constant__ CUtensorMap map, const FewArgs p) {
  using Tile = FewTile<W>;
  constexpr int H_LD = Tile::CHUNKS * 128 + 64, H_OFF = Tile::CHUNKS * Tile::BYTES, STAGE = (H_OFF + FEW_TOKENS * H_LD + 1023) / 1024 * 1024;
  constexpr int STAGES = FEW_DOWN_RING / STAGE < FEW_STAGES ? FEW_DOWN_RING / STAGE : FEW_STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ FewBars bars;
  __shared__ __align__(16) FewPlan plan;
  __shared__ __align__(16) float red[128 * FEW_TOKENS];                         // [sender][rows of this CTA: 128 / splits][token]
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int rank = int(cluster_ctarank()), splits = p.splits, tile = blockIdx.x / splits;
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  if (threadIdx.x == 0) few_init(bars, STAGES);
  pdl_wait();
  pdl_launch_dependents();
  {
    const uint4* src = reinterpret_cast<const uint4*>(p.plan);
    for (int i = threadIdx.x; i < int(sizeof(FewPlan) / 16); i += FEW_THREADS) reinterpret_cast<uint4*>(&plan)[i] = src[i];
  }
  __syncthreads();
  const int chunks = p.I >> 6, steps = (chunks + Tile::CHUNKS - 1) / Tile::CHUNKS, total = plan.met * steps;
  const int lo = int((long long)total * rank / splits), hi = int((long long)total * (rank + 1) / splits);
  bool ok = true;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  if (warp == 8) {
    FewRing r{STAGES};
    int d = lo / steps, c = (lo - d * steps) * Tile::CHUNKS;
    for (int i = lo; i < hi; ++i) {
      ok = r.wait_empty(bars, p.status);
      if (!ok) break;
      if (elect_one()) {
        const int n = min(Tile::CHUNKS, chunks - c), e = plan.expert[d];
        const uint2 sl = *reinterpret_cast<const uint2*>(plan.slot[d]);
        uint8_t* st = ring + r.s * STAGE;
        uint64_t* bar = &bars.full[r.s];
        int meet = 0;
        for (int t = 0; t < p.T; ++t) meet += ((t < 4 ? sl.x : sl.y) >> (t & 3) * 8 & 255u) != 255u;
        mbar_expect_tx(bar, n * (Tile::BYTES + meet * 128));
        for (int j = 0; j < n; ++j) few_copy<W>(st + j * Tile::BYTES, bar, &map, p.down, e, tile, c + j, p.H, p.I);
        for (int t = 0; t < p.T; ++t) {
          const uint32_t slot = (t < 4 ? sl.x : sl.y) >> (t & 3) * 8 & 255u;
          if (slot != 255u) bulk_copy_g2s(st + H_OFF + t * H_LD, p.h + (long long)(t * p.top + slot) * p.I + c * 64, n * 128, bar);
        }
      }
      __syncwarp();
      r.next();
      c += Tile::CHUNKS;
      if (c >= chunks) { c = 0; ++d; }
    }
    if (!ok) r.drain(bars);
  } else {
    FewRing r{STAGES};
    int d = lo / steps, c = (lo - d * steps) * Tile::CHUNKS;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    const int r0 = warp * 16 + g;
    for (int i = lo; i < hi; ++i) {
      ok = r.wait_full(bars, p.status, lane);
      if (!ok) break;
      const uint8_t* st = ring + r.s * STAGE;
      const bool mine = plan.slot[d][g] != 255;
#pragma unroll
      for (int j = 0; j < Tile::CHUNKS; ++j) {
        if (j > 0 && c + j >= chunks) break;
        const uint8_t* hs = st + H_OFF + g * H_LD + j * 128 + q * 16;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        const uint4 b[2] = {mine ? *reinterpret_cast<const uint4*>(hs) : zero, mine ? *reinterpret_cast<const uint4*>(hs + 64) : zero};
        Tile::mma(acc, st + j * Tile::BYTES, r0, r0 + 8, g, q, b);
      }
      r.next();
      c += Tile::CHUNKS;
      if (c < chunks && i + 1 < hi) continue;
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
  // rows of the tile are dealt out to the cluster's CTAs, a multiple of 16 each
  __syncwarp();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");        // of the arrival at the start
  const int rows = 128 / splits;
  if (warp < 8) {
    const int owner = warp * 16 / rows, l = warp * 16 - owner * rows;
    const uint32_t at = dsmem_addr(smem_u32(&red[(rank * rows + l + g) * FEW_TOKENS + q * 2]), uint32_t(owner));
#pragma unroll
    for (int j = 0; j < 2; ++j)
      asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(at + j * 8 * FEW_TOKENS * 4), "f"(sum[j * 2]), "f"(sum[j * 2 + 1]) : "memory");
  }
  cluster_sync_all();
  for (int i = threadIdx.x; i < rows * FEW_TOKENS; i += FEW_THREADS) {
    const int t = i / rows, l = i - t * rows, n = tile * 128 + rank * rows + l;
    if (t >= p.T || n >= p.H) continue;
    float v = 0.f;
    for (int s = 0; s < splits; ++s) v += red[(s * rows + l) * FEW_TOKENS + t];
    if (p.down_b)
      for (int j = 0; j < p.top; ++j) v += plan.share[t * p.top + j] * bf2f(p.down_b[(long long)plan.ids[t * p.top + j] * p.H + n]);
    p.out[(long long)t * p.H + n] = f2bf(v);
  }
}

// --------------------------------------------------------------------------------- host side
bool MakeMapBf16(CUtensorMap* out, const void* ptr, int rows, int cols, int ld, int box_rows);  // gemm_tcgen05.cu

template <int W>
static int LaunchFew(FewArgs p, int sm_count, cudaStream_t stream) {
  using Tile = FewTile<W>;
  constexpr int STAGE = Tile::CHUNKS * Tile::BYTES;
  const int Hp = (p.H + 63) / 64 * 64;
  const size_t fixed = 1024 + sizeof(FewShared) + (size_t(p.T) * p.E * 4 + 15) / 16 * 16 + size_t(p.T) * (Hp + 32) * 2;
  // Two CTAs an SM where that leaves each a ring of 48 KiB: more warps to expand and multiply; else one with what there is.
  const int two = fixed + 48 * 1024 <= FEW_SMEM_TWO;
  const size_t room = two ? FEW_SMEM_TWO : FEW_SMEM_ONE;
  if (fixed + 2 * STAGE > room) return -5;
  p.stages = int(min(size_t(FEW_STAGES), (room - fixed) / STAGE));
  CUtensorMap gate_up = {}, down = {};
  if (W == FEW_BF16 && (!MakeMapBf16(&gate_up, p.gate_up, p.E * 2 * p.I, p.H, p.H, 128) || !MakeMapBf16(&down, p.down, p.E * p.H, p.I, p.I, 128))) return -2;
  static bool configured[OGB_MAX_DEVICES] = {}, configured_down[OGB_MAX_DEVICES] = {};
  if (!set_max_dyn_smem(few_gate_up_kernel<W>, int(FEW_SMEM_ONE), configured) || !set_max_dyn_smem(few_down_kernel<W>, FEW_DOWN_RING + 1024, configured_down)) return -3;
  static const int pdl = [] { const char* e = getenv("OGB_PDL"); return (e && e[0] == '0') ? 0 : 1; }();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {FEW_CLUSTER, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(FEW_THREADS);
  cfg.stream = stream;
  cfg.gridDim = dim3(FEW_CLUSTER);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // as many clusters as run at once
  static int clusters_at[OGB_MAX_DEVICES][2] = {};
  int dev = 0, clusters = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -4;
  const bool tracked = dev >= 0 && dev < OGB_MAX_DEVICES;
  if (tracked) clusters = clusters_at[dev][two];
  if (!clusters) {
    cfg.dynamicSmemBytes = room;
    if (cudaOccupancyMaxActiveClusters(&clusters, few_gate_up_kernel<W>, &cfg) != cudaSuccess || clusters < 1) return -4;
    if (tracked) clusters_at[dev][two] = clusters;
  }
  cfg.dynamicSmemBytes = fixed + p.stages * STAGE;
  cfg.gridDim = dim3(unsigned(clusters * FEW_CLUSTER));
  cfg.numAttrs = pdl ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, few_gate_up_kernel<W>, gate_up, p) != cudaSuccess) return -4;
  const int tiles = (p.H + 127) / 128;
  p.splits = FEW_CLUSTER;
  while (p.splits > 1 && tiles * p.splits > 2 * sm_count) p.splits /= 2;
  attr[0].val.clusterDim = {unsigned(p.splits), 1, 1};
  cfg.dynamicSmemBytes = FEW_DOWN_RING + 1024;
  cfg.gridDim = dim3(unsigned(tiles * p.splits));
  return cudaLaunchKernelEx(&cfg, few_down_kernel<W>, down, p) == cudaSuccess ? 0 : -4;
}

}  // namespace ogb

using namespace ogb;

OGB_API long long ogb_moe_few_scratch_bytes(int T, int top, int I) {
  return T < 1 || T > FEW_TOKENS || top < 1 || top > FEW_TOP || I < 1 ? -1 : (long long)sizeof(FewPlan) + (long long)T * top * I * 2;
}

OGB_API int ogb_moe_few_tokens(const void* x, long long ldx, const void* router, const void* router_b, const void* gate_up, const void* gate_up_b,
                               const void* down, const void* down_b, void* out, int T, int H, int I, int E, int top, int rule, int weights, int act,
                               float alpha, float limit, void* scratch, int* status, int sm_count, void* stream) {
  if (ogb_moe_few_scratch_bytes(T, top, I) < 0 || !x || !router || !gate_up || !down || !out || !scratch || H < 1 || H % 8 || E < top || E > FEW_EXPERTS ||
      I % 64 || (weights != FEW_BF16 && H % 64) || rule < 0 || rule > 2 || weights < 0 || weights > 2 || (act != 1 && act != 2)) return -1;
  if ((reinterpret_cast<uintptr_t>(x) | uintptr_t(ldx * 2) | reinterpret_cast<uintptr_t>(router) | reinterpret_cast<uintptr_t>(gate_up) | reinterpret_cast<uintptr_t>(down) | reinterpret_cast<uintptr_t>(scratch)) & 15)
    return -1;
  FewArgs p{static_cast<const __nv_bfloat16*>(x), ldx, static_cast<const __nv_bfloat16*>(router), static_cast<const __nv_bfloat16*>(router_b), gate_up,
            static_cast<const __nv_bfloat16*>(gate_up_b), down, static_cast<const __nv_bfloat16*>(down_b), static_cast<__nv_bfloat16*>(out), T, H, I, E, top,
            rule, act, alpha, limit, static_cast<FewPlan*>(scratch), reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(scratch) + sizeof(FewPlan)), 0, 0, status};
  if ((long long)E * 2 * I > 0x7fffffff || (long long)E * H > 0x7fffffff) return -5;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (weights == FEW_BF16) return LaunchFew<FEW_BF16>(p, sm_count, s);
  return weights == FEW_FP4_F16 ? LaunchFew<FEW_FP4_F16>(p, sm_count, s) : LaunchFew<FEW_FP4_BF16>(p, sm_count, s);
}
