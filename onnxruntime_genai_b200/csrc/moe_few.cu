// A whole mixture-of-experts layer for up to eight tokens in two kernels, bound by the bytes of the experts that the tokens meet and, with few bytes, by latency.
//
// few_gate_up_kernel: every cluster of eight CTAs computes all router logits for itself (an eighth of the experts per CTA, exchanged through distributed
// shared memory), so that each CTA can choose the experts, list those that any token meets, and go on to their gate and up rows without a kernel or a
// grid barrier in between; the router is small beside the experts and comes from L2.  A warp computes sixteen features of one expert for all tokens: the
// rows of an `mma.sync` tile of 16 are eight gate rows and the eight up rows of the same features, its columns the tokens, so that a thread holds a
// gate and its up value and writes share * act(gate, up).  The work of a cluster (items of 64 features, in steps of k) is cut into eight equal ranges; of an
// item that a range border cuts, the later parts' sums go through memory to the CTA that began it.
// few_down_kernel: a cluster computes 64 columns of the output; its CTAs take equal parts of the sequence (expert, k); their sums are sent to the CTA that finishes
// an output and added there in a fixed order.
// In both the warps of a CTA form teams that take turns at the stages of a ring and add their sums in a fixed order: more stages are in work at once.
//
// `mma.sync` is used on purpose: its eight columns are the eight tokens, and weights go from shared memory to registers in the order in which they lie in
// memory, with the k index of a product permuted alike for both operands.  A ring of bulk copies per CTA keeps 50 to 70 KB in flight, twice an SM.  A bulk copy costs
// some 30 ns of an SM however small it is, so that what is in small pieces (scales of half a record, a step's activations) is copied by a warp's threads: the down products
// of 7 tokens in 30 us instead of 40.
//
// Measured (us a layer, weights from memory; both kernels take 18 of them with hardly any weights: launches, the router, the choice, the first bytes, the sums):
// 1 token, 4 of 32 mxfp4 experts of 2880: 28 (in their bf16 form 32); 7 tokens of the same 86 (3.0 TB/s; 115); 8 tokens, 8 of 128 of 1472: 109.5 (3.2); 1 token, 8 of 128
// bf16 experts of 768: 26 to 28; 8 tokens, 2 of 8 bf16 experts of 14336: 438 to 454 on different cards (5.6 to 5.8).  With the products left out 7 mxfp4 tokens save 15 us of 98, with the activations' bulk copies left out 10.
//
// Roundings: the router's logits, all sums and the activation are fp32.  The activations times routing weights travel between the kernels in 16 bits (the
// operand type of the second product): bf16, or, with packed experts in their fp16 form, fp16 after a scaling by a power of two per token, expert and 64 features
// (an item of the first product and a step of the second), which the second product's sums undo: eleven bits down to 2^-28 of the largest of the 64, whatever its size.
// The rows meet packed experts of that form as fp16 after a scaling by a power of two per token, which loses nothing within 2^-38 of a row's largest value.
#include <cuda_fp16.h>
#include <math.h>

#include "kernels.h"
#include "packed_weights.cuh"
#include "tensor_map.cuh"

namespace ogb {

template <int N> struct Int { static constexpr int value = N; };
enum FewWeights : int { FEW_BF16 = 0, FEW_FP4_F16 = 1, FEW_FP4_BF16 = 2 };   // packed: the records of gemm_fp4.cu in their two forms
constexpr int FEW_TOKENS = 8, FEW_TOP = 32, FEW_EXPERTS = 1024, FEW_MET = FEW_TOKENS * FEW_TOP;
constexpr int FEW_CLUSTER = 8, FEW_AGAIN = 0x8000;
constexpr int FEW_THREADS = 288, FEW_DOWN_THREADS = 320, FEW_STAGES = 16;
constexpr size_t FEW_SMEM_TWO = 113 * 1024, FEW_SMEM_ONE = 227 * 1024;          // shared memory of a CTA, with two or one on an SM
constexpr int FEW_DOWN_ROWS = 64, FEW_DOWN_RING = 96 * 1024, FEW_OUT = FEW_DOWN_ROWS * FEW_TOKENS;
constexpr int FEW_MAX_CTAS = 320;                                               // of the first kernel: partial sums of a cut item, 4 KB each
constexpr long long FEW_PREFETCH = 40 << 20;

// What the first kernel leaves for the second.
struct alignas(16) FewPlan {
  int met, unused[3];                       // experts that any token meets, in ascending order
  uint16_t expert[FEW_MET];
  uint8_t slot[FEW_MET][FEW_TOKENS];        // which choice of the token the expert is; 255: none
  uint16_t ids[FEW_TOKENS * FEW_TOP];       // [token][choice]; FEW_AGAIN: expert 0 again
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
  float4* parts;        // [CTA][warp][half][lane] sums of the first kernel's cut items
  uint16_t* h;          // [T * top, I], in groups of eight as the second product reads them
  float* h_scale;       // [met expert, I / 64, token], fp16 form: what the second product's sums over 64 features are multiplied by
  int stages, ring_bytes, splits;   // of the first kernel's ring, and its room; CTAs of a cluster of the second
  int* status;
};

// ------------------------------------------------------------------------------- operands
// (volatile: they are for whole warps, and must not be moved into a branch that some lanes take)
__device__ __forceinline__ void few_mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void few_mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 32 k values: a lane brings eight values of each of its rows (in pairs) and of its token; two sums, so that the two products do not wait for each other
__device__ __forceinline__ void mma_bf16_32(float (&d)[2][4], const uint4& r0, const uint4& r1, const uint4& b) {
  few_mma_bf16(d[0], r0.x, r1.x, r0.y, r1.y, b.x, b.y);
  few_mma_bf16(d[1], r0.z, r1.z, r0.w, r1.w, b.z, b.w);
}

// Reads of shared memory by 32-bit address (volatile: they stay between the waits around them)
template <int OFF> __device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4+%5];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at), "n"(OFF));
  return v;
}
template <int OFF> __device__ __forceinline__ uint2 lds64(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2+%3];" : "=r"(v.x), "=r"(v.y) : "r"(at), "n"(OFF));
  return v;
}
template <int OFF> __device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1+%2];" : "=r"(v) : "r"(at), "n"(OFF));
  return v;
}
template <int OFF> __device__ __forceinline__ uint32_t lds8(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1+%2];" : "=r"(v) : "r"(at), "n"(OFF));
  return v;
}

// A thread's arrival on a barrier when its copies so far have landed
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory"); }

// A stage of the ring holds CHUNKS steps of 64 k values of a tile of ROWS weight rows, as they lie in memory: packed records (codes, then scales), or (bf16) a
// box of 64 columns with the 128-byte swizzle.  A warp multiplies 32 of the rows in two tiles of 16: row r0 of the first (lanes 4 g .. 4 g + 3) and the row APART behind it, and
// those NEXT behind both.
template <int W, int ROWS>
struct FewTile {
  static constexpr int CHUNKS = W == FEW_BF16 && ROWS == 128 ? 1 : 2;
  static constexpr int BYTES = W == FEW_BF16 ? ROWS * 128 : ROWS * 34;             // of a step
  // Groups of warps that take turns at the stages.  A ring has a multiple of so many: a place of the ring belongs to one team, which then has seen every phase of its
  // barrier (a team that came to a place whose stage before was another team's, and still on its way, would take the barrier's old parity for its own stage's).
  static constexpr int TEAMS = 8 / (ROWS / 32);
  static constexpr int ring(int room, int stage) { return (room / stage < FEW_STAGES ? room / stage : FEW_STAGES) / TEAMS * TEAMS; }
  static constexpr int APART = ROWS == 128 ? 64 : 8, NEXT = ROWS == 128 ? 8 : 16;  // r1 - r0: gate and up rows, or eight rows on; the warp's second tile of 16
  static constexpr float SCALE = W == FEW_FP4_F16 ? 0.015625f : 1.f;               // of the sums: the records hold a scale's code + 6
  // a lane's place in a step: its part of row r0, and (packed) its scales
  static __device__ __forceinline__ uint32_t place(int r0, int g, int q) { return W == FEW_BF16 ? r0 * 128 + ((q ^ g) << 4) : r0 * 32 + q * (W == FEW_FP4_F16 ? 8 : 4); }
  static __device__ __forceinline__ uint32_t scales(int r0) { return ROWS * 32 + r0 * 2; }
  // A step: every load, then every product.  at, sc: addresses of the lane's place and scales in it; b: the tokens' values; by (fp16 form, where the tokens' values are
  // scaled step by step): what the sums of the lane's two tokens are multiplied by
  template <bool SCALED = false>
  static __device__ __forceinline__ void mma(float (&acc)[2][4], uint32_t at, uint32_t sc, const uint4 (&b)[2], float2 by = make_float2(1.f, 1.f)) {
    if constexpr (W == FEW_BF16) {
      uint4 a[2][2][2];                                                            // [tile of 16][half of the step][row]
      const uint32_t x = at ^ 64u;                                                 // places 4 and more of a row's eight: (q + 4) ^ g
      a[0][0][0] = lds128<0>(at);
      a[0][0][1] = lds128<APART * 128>(at);
      a[0][1][0] = lds128<0>(x);
      a[0][1][1] = lds128<APART * 128>(x);
      a[1][0][0] = lds128<NEXT * 128>(at);
      a[1][0][1] = lds128<(NEXT + APART) * 128>(at);
      a[1][1][0] = lds128<NEXT * 128>(x);
      a[1][1][1] = lds128<(NEXT + APART) * 128>(x);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          few_mma_bf16(acc[m], a[m][i][0].x, a[m][i][1].x, a[m][i][0].y, a[m][i][1].y, b[i].x, b[i].y);
          few_mma_bf16(acc[m], a[m][i][0].z, a[m][i][1].z, a[m][i][0].w, a[m][i][1].w, b[i].z, b[i].w);
        }
    } else if constexpr (W == FEW_FP4_F16) {
      const uint2 q00 = lds64<0>(at), q01 = lds64<APART * 32>(at), q10 = lds64<NEXT * 32>(at), q11 = lds64<(NEXT + APART) * 32>(at);
      const uint32_t f[2][2][2] = {{{lds8<0>(sc), lds8<1>(sc)}, {lds8<APART * 2>(sc), lds8<APART * 2 + 1>(sc)}},
                                   {{lds8<NEXT * 2>(sc), lds8<NEXT * 2 + 1>(sc)}, {lds8<(NEXT + APART) * 2>(sc), lds8<(NEXT + APART) * 2 + 1>(sc)}}};
      float t[2][2][4];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i) {                     // a block of 32 has one scale per row: its sum is scaled as a whole
          uint32_t u[4], v[4];
          cvt_e2m1x8_f16(i ? (m ? q10.y : q00.y) : (m ? q10.x : q00.x), u);
          cvt_e2m1x8_f16(i ? (m ? q11.y : q01.y) : (m ? q11.x : q01.x), v);
          few_mma_f16_first(t[m][i], u[0], v[0], u[1], v[1], b[i].x, b[i].y);
          mma_m16n8k16_f16(t[m][i], u[2], v[2], u[3], v[3], b[i].z, b[i].w);
        }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        float z[4] = {};
        float (&to)[4] = SCALED ? z : acc[m];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float x0 = __uint_as_float(f[m][0][i] << 23), x1 = __uint_as_float(f[m][1][i] << 23);
          to[0] = fmaf(t[m][i][0], x0, to[0]);
          to[1] = fmaf(t[m][i][1], x0, to[1]);
          to[2] = fmaf(t[m][i][2], x1, to[2]);
          to[3] = fmaf(t[m][i][3], x1, to[3]);
        }
        if constexpr (SCALED) {
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[m][j] = fmaf(z[j], j & 1 ? by.y : by.x, acc[m][j]);
        }
      }
    } else {
      auto half = [&](auto i, auto m) {
        constexpr int I_ = decltype(i)::value, R = decltype(m)::value * NEXT;
        const uint4 a0 = deq_fp4_word_bf16(lds32<R * 32 + I_ * 16>(at), lds8<R * 2 + I_>(sc));
        const uint4 a1 = deq_fp4_word_bf16(lds32<(R + APART) * 32 + I_ * 16>(at), lds8<(R + APART) * 2 + I_>(sc));
        few_mma_bf16(acc[R ? 1 : 0], a0.x, a1.x, a0.y, a1.y, b[I_].x, b[I_].y);
        few_mma_bf16(acc[R ? 1 : 0], a0.z, a1.z, a0.w, a1.w, b[I_].z, b[I_].w);
      };
      half(Int<0>{}, Int<0>{});
      half(Int<0>{}, Int<1>{});
      half(Int<1>{}, Int<0>{});
      half(Int<1>{}, Int<1>{});
    }
  }
  // Copies n steps from `chunk` on of rows row .. row + ROWS - 1 of expert e to a stage, counted in bytes on its barrier; by one thread.  Of half a
  // record's rows: their codes ..
  static constexpr int COPIED = W == FEW_BF16 || ROWS == 128 ? BYTES : ROWS * 32;
  static __device__ __forceinline__ void copy(uint8_t* dst, uint64_t* bar, const CUtensorMap* map, const void* packed, int e, int row, int chunk, int n, int N, int K) {
    if constexpr (W == FEW_BF16) {
      for (int j = 0; j < n; ++j) tma_load_2d(dst + j * BYTES, map, bar, (chunk + j) * 64, e * N + row);
    } else {
      const int tiles = (N + 127) >> 7;
      const uint8_t* rec = static_cast<const uint8_t*>(packed) + (((long long)e * (K >> 6) + chunk) * tiles + (row >> 7)) * FP4_RECORD_BYTES;
      for (int j = 0; j < n; ++j, rec += (long long)tiles * FP4_RECORD_BYTES) {
        if constexpr (ROWS == 128) {
          bulk_copy_g2s(dst + j * BYTES, rec, FP4_RECORD_BYTES, bar);
        } else {
          bulk_copy_g2s(dst + j * BYTES, rec + (row & 127) * 32, ROWS * 32, bar);
        }
      }
    }
  }
  // .. and the scales of half a record's rows in pieces of 16 bytes, EACH of them a step: where piece i of a record lies, and where it belongs in a step
  static constexpr int EACH = ROWS * 2 / 16;
  static __device__ __forceinline__ int scales_in_record(int row, int i) { return 128 * 32 + (row & 127) * 2 + i * 16; }
  static __device__ __forceinline__ int scales_in_step(int i) { return ROWS * 32 + i * 16; }
};

// Eight 16-bit values in the order in which a lane's eight weights of a row come out of their load: pairs (0, 1) (2, 3) .. or, from records in fp16 form,
// (0, 4) (1, 5) (2, 6) (3, 7).
template <int W> __device__ __forceinline__ int few_place(int i) { return W == FEW_FP4_F16 ? (i & 3) * 2 + (i >> 2) : i; }

// ------------------------------------------------------------------------------- ring of copies
// Warps 0 .. 7 multiply, the others copy.  All waits are bounded; after a failed one every warp leaves its loop.
struct FewBars { uint64_t full[FEW_STAGES], empty[FEW_STAGES]; int abort; };
__device__ __forceinline__ void few_init(FewBars& b, int stages, int writers, int warps) {      // warps that copy to a stage, and that read it
  for (int s = 0; s < stages; ++s) { mbar_init(&b.full[s], writers); mbar_init(&b.empty[s], warps); }
  b.abort = 0;
  mbar_fence_init();
}
struct FewRing {                       // the copying side
  int stages, s = 0, filled = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void next() {
    ++filled;
    if (++s == stages) { s = 0; ph ^= 1; }
  }
  __device__ __forceinline__ bool wait_empty(FewBars& b, int* status) {
    if (filled < stages || __all_sync(0xffffffffu, mbar_wait_bounded(&b.empty[s], ph ^ 1, &b.abort))) return true;
    atomicMax(status, OGB_ERR_WAIT_TMA);
    *reinterpret_cast<volatile int*>(&b.abort) = 1;
    return false;
  }
  __device__ __forceinline__ void drain(FewBars& b) {          // copies in flight still write shared memory: give them time to land
    volatile int never = 0;
    for (int i = max(0, filled - stages); i < filled; ++i) mbar_wait_bounded(&b.full[i % stages], (i / stages) & 1, &never, 200000000ull);
  }
};
static __device__ __noinline__ bool few_wait_slow(FewBars* b, uint32_t full, uint32_t ph, int* status) {
  const uint64_t t0 = global_timer_ns();
  uint32_t spins = 0, ok = 0;
  while (!ok) {
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(full), "r"(ph) : "memory");
    if (!ok && (++spins & 0x3ff) == 0 && (*reinterpret_cast<volatile int*>(&b->abort) || global_timer_ns() - t0 > 2000000000ull)) break;
  }
  if (__all_sync(0xffffffffu, ok != 0)) return true;
  atomicMax(status, OGB_ERR_WAIT_TMA);
  *reinterpret_cast<volatile int*>(&b->abort) = 1;
  return false;
}
template <int STAGE, int TEAMS>
struct FewReader {                     // the multiplying side: every TEAMS-th stage
  FewBars* b;
  uint32_t data, full, ph = 0, end, ring;                // addresses: this stage, its barrier; end of the ring, its bytes
  __device__ __forceinline__ FewReader(FewBars* bars, const void* first, int stages, int team)
      : b(bars), data(smem_u32(first) + team * STAGE), full(smem_u32(bars->full) + team * 8), end(smem_u32(first) + stages * STAGE), ring(stages * STAGE) {}
  __device__ __forceinline__ void next() {
    data += TEAMS * STAGE;
    full += TEAMS * 8;
    if (data >= end) { data -= ring; full -= ring / STAGE * 8; ph ^= 1; }
  }
  // false: the wait ran out; the warp goes through its loop without reading, so that it meets the barriers that the others wait at
  __device__ __forceinline__ bool wait(int* status) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(full), "r"(ph) : "memory");
    return __all_sync(0xffffffffu, ok) || few_wait_slow(b, full, ph, status);
  }
  // Hands back the stage, behind all loads from it: every sum's last product has to have its operands first (in fp16 form rows g and g + 8 have scales of their own).
  __device__ __forceinline__ void release(int lane, const float (&acc)[2][4]) {
    const uint32_t read = __float_as_uint(acc[0][0]) | __float_as_uint(acc[0][2]) | __float_as_uint(acc[1][0]) | __float_as_uint(acc[1][2]);
    mbar_arrive_behind_reads(full + uint32_t(sizeof(uint64_t)) * FEW_STAGES, read, blockIdx.z, lane);       // (the stage's `empty`; grids have one layer)
  }
};

// ------------------------------------------------------------------------------- router, choice
// Shared memory of the first kernel: what stands where the ring comes, until the experts are chosen (then logits [T][E]) ..
struct FewBefore {
  float red[FEW_THREADS / 32][16 * FEW_TOKENS];
  uint32_t mask[FEW_EXPERTS];        // tokens that meet an expert
};
// .. and behind the ring
struct alignas(16) FewShared {
  FewBars bars;
  float4 teams[2][4][64];             // [item][warp][half of its rows, lane] sums of the second team
  uint32_t top[FEW_TOKENS];          // bits of the rows' largest magnitudes
  alignas(16) uint32_t item_top[2][4][4];        // [turn][pair of tokens][warp]: exponents of the largest of an item's activations
  FewPlan plan;
};
static_assert(sizeof(FewShared) % 16 == 0, "16-byte accesses to what follows");

// Power of two that brings a largest magnitude (its bits) to 2^14 .. 2^15; none for one that is no number
__device__ __forceinline__ int few_shift(uint32_t top) { return top >= 0x7f800000u ? 0 : min(14 - (int(top >> 23) - 127), 126); }
// A float as an unsigned number of the same order; 0: not a number.
__device__ __forceinline__ uint32_t few_key(float v) {
  const uint32_t u = __float_as_uint(v);
  return v != v ? 0u : u & 0x80000000u ? ~u : u | 0x80000000u;
}
// Choice of `top` experts for a token by one warp: the largest logits, the lowest index among equal ones; where logits are not numbers, expert 0 stands for
// what is missing (several times then), and all shares are no numbers.  A lane holds every 32nd expert, up to 32 R, and looks for its best one anew only when that was taken.
template <int R>
__device__ __forceinline__ void few_choose(const float* row, int E, int top, int rule, int lane, int& id, float& share) {
  uint32_t key[R];                   // 0: nothing to choose
  bool bad = false;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const float v = i * 32 + lane < E ? row[i * 32 + lane] : -INFINITY;
    key[i] = i * 32 + lane < E ? few_key(v) : 0u;
    bad |= v != v;
  }
  bad = __any_sync(0xffffffffu, bad);
  uint32_t best = 0;
  int at = 0x7fffffff;
  auto scan = [&]() {
    best = 0;
    at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < R; ++i) if (key[i] > best) { best = key[i]; at = i * 32 + lane; }
  };
  scan();
  float most = 0.f, mine = 0.f;
  id = 0;
  for (int j = 0; j < top; ++j) {
    const uint32_t k = __reduce_max_sync(0xffffffffu, best);
    const int e = int(__reduce_min_sync(0xffffffffu, best == k && k ? uint32_t(at) : 0x7fffffffu));
    const float v = __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
    if (j == 0) most = v;
    if (lane == j) { mine = v; id = k ? e : 0; }
    if (k && at == e) {
#pragma unroll
      for (int i = 0; i < R; ++i) if (i == e >> 5) key[i] = 0;
      scan();
    }
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
  using Tile = FewTile<W, 128>;
  constexpr int STAGE = Tile::CHUNKS * Tile::BYTES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  FewBefore& pre = *reinterpret_cast<FewBefore*>(ring);
  float* logits = reinterpret_cast<float*>(&pre + 1);                                        // [T][E]
  FewShared& sh = *reinterpret_cast<FewShared*>(ring + p.ring_bytes);
  const int Hp = (p.H + 63) / 64 * 64, xs_ld = Hp + 32;              // 16-bit values a row: neighbours start 64 bytes apart in the banks
  uint16_t* xs = reinterpret_cast<uint16_t*>(&sh + 1);
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int rank = int(cluster_ctarank());
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");      // the others' shared memory is written only once they run
  // The rows: a warp takes 256 values of a token at a time and keeps the first pieces in registers until the rows' largest magnitudes are known (packed experts:
  // fp16 after a scaling).
  constexpr int HELD = 6, WARPS = FEW_THREADS / 32;
  const int parts = (Hp + 255) >> 8, pieces = p.T * parts;
  auto piece = [&](int i) {
    const int t = i / parts, k = (i - t * parts) * 256 + lane * 8;
    return i < pieces && k < p.H ? *reinterpret_cast<const uint4*>(p.x + t * p.ldx + k) : make_uint4(0, 0, 0, 0);
  };
  uint4 held[HELD];
#pragma unroll
  for (int h = 0; h < HELD; ++h) held[h] = piece(warp + h * WARPS);
  for (int e = threadIdx.x; e < p.E; e += FEW_THREADS) pre.mask[e] = 0;
  if (threadIdx.x < FEW_TOKENS) sh.top[threadIdx.x] = 0;
  if (threadIdx.x == 0) few_init(sh.bars, p.stages, 1, 8 / Tile::TEAMS);
  __syncwarp();
  __syncthreads();

  auto tops = [&]() {                     // behind the router's loads, so that these are on their way first
    auto largest = [&](int i, const uint4& v) {
      if (i >= pieces) return;
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) top = max(top, max(w[j] << 16 & 0x7fffffffu, w[j] & 0x7fff0000u));
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0) atomicMax(&sh.top[i / parts], top);
    };
#pragma unroll
    for (int h = 0; h < HELD; ++h) largest(warp + h * WARPS, held[h]);
    for (int i = warp + HELD * WARPS; i < pieces; i += WARPS) largest(i, piece(i));
  };

  // router logits of this CTA's experts: 16 experts x 8 tokens at a time, the warps share k
  const int per = (p.E + FEW_CLUSTER - 1) / FEW_CLUSTER, e_end = min(p.E, (rank + 1) * per);
  bool met_cluster = false;
  for (int e0 = rank * per; e0 < (rank + 1) * per; e0 += 16) {               // (the same number of rounds in every CTA)
    float acc[2][4] = {};
    const bool r0 = e0 + g < e_end, r1 = e0 + g + 8 < e_end;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const __nv_bfloat16* w0 = p.router + (long long)(r0 ? e0 + g : 0) * p.H;
    const __nv_bfloat16* w1 = p.router + (long long)(r1 ? e0 + g + 8 : 0) * p.H;
    auto fetch = [&](const __nv_bfloat16* at, bool there) { return there ? *reinterpret_cast<const uint4*>(at) : zero; };
    if (e0 + 8 < e_end) {
#pragma unroll 5
      for (int k = warp * 32 + q * 8; k < (p.H + 31) / 32 * 32; k += FEW_THREADS) {
        const bool in = k < p.H;
        const uint4 a0 = fetch(w0 + k, r0 && in), a1 = fetch(w1 + k, r1 && in), b = fetch(p.x + g * p.ldx + k, g < p.T && in);
        mma_bf16_32(acc, a0, a1, b);
      }
    } else {                                             // (up to eight: more of k on its way at once)
#pragma unroll 10
      for (int k = warp * 32 + q * 8; k < (p.H + 31) / 32 * 32; k += FEW_THREADS) {
        const bool in = k < p.H;
        const uint4 a0 = fetch(w0 + k, r0 && in), b = fetch(p.x + g * p.ldx + k, g < p.T && in);
        mma_bf16_32(acc, a0, zero, b);
      }
    }
    if (W == FEW_FP4_F16 && !met_cluster) tops();
    *reinterpret_cast<float2*>(&pre.red[warp][g * 8 + q * 2]) = make_float2(acc[0][0] + acc[1][0], acc[0][1] + acc[1][1]);
    *reinterpret_cast<float2*>(&pre.red[warp][(g + 8) * 8 + q * 2]) = make_float2(acc[0][2] + acc[1][2], acc[0][3] + acc[1][3]);
    __syncthreads();
    if (!met_cluster) { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); met_cluster = true; }
    if (threadIdx.x < 128) {
      const int e = e0 + int(threadIdx.x >> 3), t = threadIdx.x & 7;
      if (e < e_end && t < p.T) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < FEW_THREADS / 32; ++w) v += pre.red[w][threadIdx.x];
        if (p.router_b) v += bf2f(p.router_b[e]);
        const uint32_t at = smem_u32(logits + t * p.E + e);
#pragma unroll
        for (uint32_t r = 0; r < FEW_CLUSTER; ++r) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dsmem_addr(at, r)), "f"(v) : "memory");
      }
    }
    __syncthreads();
  }
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  // the rows as the products read them
  auto put = [&](int i, uint4 v) {
    const int t = i / parts, k = (i - t * parts) * 256 + lane * 8;
    if (i >= pieces || k >= Hp) return;
    if (W == FEW_FP4_F16) {
      const float scale = __uint_as_float(uint32_t(few_shift(sh.top[t]) + 127) << 23);
      const float2 a = unpack_bf16x2(v.x), b = unpack_bf16x2(v.y), c = unpack_bf16x2(v.z), d = unpack_bf16x2(v.w);
      v = make_uint4(pack_f16x2(a.x * scale, c.x * scale), pack_f16x2(a.y * scale, c.y * scale), pack_f16x2(b.x * scale, d.x * scale),
                     pack_f16x2(b.y * scale, d.y * scale));
    }
    *reinterpret_cast<uint4*>(xs + t * xs_ld + k) = v;
  };
#pragma unroll
  for (int h = 0; h < HELD; ++h) put(warp + h * WARPS, held[h]);
  for (int i = warp + HELD * WARPS; i < pieces; i += WARPS) put(i, piece(i));
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

  // choices, and the experts that any token meets
  if (warp < p.T) {
    int id;
    float share;
    const float* row = logits + warp * p.E;
    if (p.E <= 128) few_choose<4>(row, p.E, p.top, p.rule, lane, id, share);
    else if (p.E <= 256) few_choose<8>(row, p.E, p.top, p.rule, lane, id, share);
    else few_choose<32>(row, p.E, p.top, p.rule, lane, id, share);
    // expert 0 may stand there several times: the first counts, so that all clusters look for its activations in the same place
    const uint32_t zeros = __ballot_sync(0xffffffffu, id == 0);
    const bool again = id == 0 && (zeros & ((1u << lane) - 1)) != 0;
    if (lane < p.top) {
      sh.plan.ids[warp * p.top + lane] = uint16_t(again ? FEW_AGAIN : id);
      sh.plan.share[warp * p.top + lane] = share;
      atomicOr(&pre.mask[id], 1u << warp);
    }
  }
  __syncthreads();
  if (warp == 0) {
    int n = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const bool here = e0 + lane < p.E && pre.mask[e0 + lane];
      const uint32_t b = __ballot_sync(0xffffffffu, here);
      const int at = n + __popc(b & ((1u << lane) - 1));
      if (here) {
        sh.plan.expert[at] = uint16_t(e0 + lane);
        *reinterpret_cast<uint2*>(sh.plan.slot[at]) = make_uint2(0xffffffffu, 0xffffffffu);
        pre.mask[e0 + lane] = uint32_t(at);         // from here on: the expert's place in the list
      }
      n += __popc(b);
    }
    if (lane == 0) sh.plan.met = n;
    __syncwarp();
    for (int i = lane; i < p.T * p.top; i += 32)
      if (const int id = sh.plan.ids[i]; id < FEW_AGAIN) sh.plan.slot[pre.mask[id]][i / p.top] = uint8_t(i % p.top);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // copies take the place of what stood in the ring's
  __syncthreads();
  if (blockIdx.x == 0) {
    const uint4* src = reinterpret_cast<const uint4*>(&sh.plan);
    for (int i = threadIdx.x; i < int(sizeof(FewPlan) / 16); i += FEW_THREADS) reinterpret_cast<uint4*>(p.plan)[i] = src[i];
  }

  // Gate and up rows: an item is 64 features of a met expert, 128 rows that lie together; a warp takes eight features.  The clusters share the items, the CTAs
  // of a cluster the steps of its items.
  const int tiles = p.I >> 6, items = sh.plan.met * tiles, chunks = Hp >> 6, steps = (chunks + Tile::CHUNKS - 1) / Tile::CHUNKS;
  const unsigned clusters = gridDim.x / FEW_CLUSTER, cluster = blockIdx.x / FEW_CLUSTER;
  const int item0 = int(unsigned(items) * cluster / clusters), mine = int(unsigned(items) * (cluster + 1) / clusters) - item0;
  const unsigned all_steps = unsigned(mine * steps);
  const int lo = int(all_steps * rank / FEW_CLUSTER), hi = int(all_steps * (rank + 1) / FEW_CLUSTER);
  // Activations of 16 features x 2 tokens a lane: acc[m] the sums of features m * 8 + g of the warp's 16 (gate, gate, up, up).  For the first four warps together.
  int turn = 0;
  auto finish = [&](int item, const float (&acc)[2][4]) {
    const int d = item / tiles, f0 = (item - d * tiles) * 64 + (warp & 3) * 16;
    float h[2][2];                                       // [feature][token]
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const long long row = (long long)sh.plan.expert[d] * 2 * p.I + (f0 >> 6) * 128 + (f0 & 63) + m * 8 + g;
      const float bg = p.gate_up_b ? bf2f(p.gate_up_b[row]) : 0.f, bu = p.gate_up_b ? bf2f(p.gate_up_b[row + 64]) : 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int t = q * 2 + j, slot = sh.plan.slot[d][t];
        h[m][j] = 0.f;
        if (slot == 255) continue;
        const float s = W == FEW_FP4_F16 ? __uint_as_float(uint32_t(127 - few_shift(sh.top[t])) << 23) * Tile::SCALE : 1.f;
        float gate = fmaf(acc[m][j], s, bg), up = fmaf(acc[m][2 + j], s, bu), v = gate;
        if (p.act == 2) {
          if (p.limit > 0.f) {             // (comparisons, not minima: what is not a number stays that)
            gate = gate > p.limit ? p.limit : gate;
            up = up > p.limit ? p.limit : up < -p.limit ? -p.limit : up;
          }
          v = p.alpha * gate;
          up += 1.f;
        }
        h[m][j] = gate / (1.f + expf(-v)) * up * sh.plan.share[t * p.top + slot];
      }
    }
    float scale[2] = {1.f, 1.f};
    if (W == FEW_FP4_F16) {
      // the largest of the item's 64 features, per token (its exponent, two tokens in a word): over the lanes of the warp that share the token, then over the four
      // warps.  Two buffers: a warp is at most one item ahead of the others
      __syncwarp();
      auto exponent = [&](int j) { return max(__float_as_uint(h[0][j]) & 0x7fffffffu, __float_as_uint(h[1][j]) & 0x7fffffffu) >> 23; };
      uint32_t top = exponent(0) | exponent(1) << 16;
#pragma unroll
      for (int o = 4; o < 32; o *= 2) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
      uint32_t (&all)[4][4] = sh.item_top[turn & 1];
      ++turn;
      if (g == 0) all[q][warp & 3] = top;
      __syncwarp();
      asm volatile("bar.sync 2, 128;" ::: "memory");
      const uint4 w = *reinterpret_cast<const uint4*>(all[q]);
      top = __vmaxu2(__vmaxu2(w.x, w.y), __vmaxu2(w.z, w.w));
      float undo[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int shift = few_shift((top >> (16 * j) & 0xffffu) << 23);
        scale[j] = __uint_as_float(uint32_t(127 + shift) << 23);
        undo[j] = __uint_as_float(uint32_t(127 - shift) << 23) * Tile::SCALE;
      }
      if (warp == 0 && g == 0) *reinterpret_cast<float2*>(p.h_scale + ((long long)d * tiles + (f0 >> 6)) * FEW_TOKENS + q * 2) = make_float2(undo[0], undo[1]);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int t = q * 2 + j, slot = sh.plan.slot[d][t];
        if (slot == 255) continue;
        p.h[(long long)(t * p.top + slot) * p.I + f0 + m * 8 + few_place<W>(g)] = uint16_t(W == FEW_FP4_F16 ? pack_f16x2(h[m][j] * scale[j], 0.f) : pack_bf16x2(h[m][j], 0.f));
      }
  };
  const int last_item = hi > lo ? (hi - 1) / steps : 0;
  const bool open_end = hi > lo && hi % steps != 0 && last_item * steps >= lo;        // began here, ends elsewhere: finished below
  float left[2][4] = {};                               // its sums
  if (warp == 8) {
    FewRing r{p.stages};
    bool ok = true;
    const int item = lo / steps;
    int c = (lo - item * steps) * Tile::CHUNKS, d = (item0 + item) / tiles, tile = item0 + item - d * tiles;
    for (int i = lo; i < hi; ++i) {
      ok = r.wait_empty(sh.bars, p.status);
      if (!ok) break;
      const int n = min(Tile::CHUNKS, chunks - c);
      uint64_t* bar = &sh.bars.full[r.s];
      if (elect_one()) {
        mbar_expect_tx(bar, n * Tile::BYTES);
        Tile::copy(ring + r.s * STAGE, bar, &map, p.gate_up, sh.plan.expert[d], tile * 128, c, n, 2 * p.I, p.H);
      }
      __syncwarp();
      r.next();
      c += Tile::CHUNKS;
      if (c >= chunks) {
        c = 0;
        if (++tile == tiles) { tile = 0; ++d; }
      }
    }
    if (!ok) r.drain(sh.bars);
    // While the rest of this kernel runs, memory is idle: where the met experts' down rows are few enough to stay in L2, they are fetched there
    const long long per_expert = W == FEW_BF16 ? (long long)p.H * p.I * 2 : (long long)(p.I >> 6) * ((p.H + 127) >> 7) * FP4_RECORD_BYTES;
    if (per_expert * sh.plan.met <= FEW_PREFETCH) {
      constexpr int PIECE = 16384;
      const int per = int((per_expert + PIECE - 1) / PIECE), all = per * sh.plan.met;
      for (int i = int(blockIdx.x) * 32 + lane; i < all; i += int(gridDim.x) * 32) {
        const int d = i / per;
        const long long at = (long long)(i - d * per) * PIECE;
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;"
                     ::"l"(static_cast<const uint8_t*>(p.down) + per_expert * sh.plan.expert[d] + at), "r"(uint32_t(min((long long)PIECE, per_expert - at))) : "memory");
      }
    }
  } else {
    const uint32_t xt = smem_u32(xs + (g < p.T ? g : 0) * xs_ld + q * 8);    // (columns beyond the tokens: any numbers, they are not looked at)
    const int team = warp >> 2;
    const uint32_t place = Tile::place((warp & 3) * 16 + g, g, q), scales = Tile::scales((warp & 3) * 16 + g);
    float acc[2][4] = {};
    FewReader<STAGE, Tile::TEAMS> r(&sh.bars, ring, p.stages, team);
    bool ok = true;
    int item = lo / steps, i = lo + team;              // i: this team's next step
    for (int from = lo; from < hi; ++item) {
      const int first = item * steps, to = min(hi, first + steps);
      const bool whole = from == first;
      for (; i < to; i += Tile::TEAMS) {
        if (ok && (ok = r.wait(p.status))) {
          const int c = (i - first) * Tile::CHUNKS;
          const uint32_t x = xt + c * 128;
          uint4 b[2] = {lds128<0>(x), lds128<64>(x)};
          Tile::mma(acc, r.data + place, r.data + scales, b);
          if (Tile::CHUNKS == 2 && c + 1 < chunks) {
            b[0] = lds128<128>(x);
            b[1] = lds128<192>(x);
            Tile::mma(acc, r.data + Tile::BYTES + place, r.data + Tile::BYTES + scales, b);
          }
          r.release(lane, acc);
        }
        r.next();
      }
      // The item's part in this range is done: the second team's sums go to the first, which finishes the item, leaves a part of it to the CTA that began it, or
      // keeps what it has until the others' parts are there.  Two buffers: a team is at most one item ahead of the other.
      float4* mine_ = sh.teams[item & 1][warp & 3];
      if (team == 1) {
        mine_[lane] = make_float4(acc[0][0], acc[0][1], acc[0][2], acc[0][3]);
        mine_[32 + lane] = make_float4(acc[1][0], acc[1][1], acc[1][2], acc[1][3]);
      }
      __syncwarp();                                    // (lanes may still be apart behind the last item's activations: barriers want whole warps)
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (team == 0) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const float4 v = mine_[m * 32 + lane];
          acc[m][0] += v.x; acc[m][1] += v.y; acc[m][2] += v.z; acc[m][3] += v.w;
        }
        if (!whole) {
          for (int m = 0; m < 2; ++m) p.parts[((blockIdx.x * 4 + warp) * 2 + m) * 32 + lane] = make_float4(acc[m][0], acc[m][1], acc[m][2], acc[m][3]);
        } else if (to == first + steps) {
          finish(item0 + item, acc);
        } else {
          for (int m = 0; m < 2; ++m) for (int j = 0; j < 4; ++j) left[m][j] = acc[m][j];
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[0][j] = acc[1][j] = 0.f;
      from = to;
    }
  }
  __syncwarp();
  cluster_sync_all();                                    // the cluster's partial sums are in memory
  if (warp < 4 && open_end) {
    const int end = (last_item + 1) * steps;             // ranges behind this one, up to the item's end, in order
    for (int o = rank + 1; o < FEW_CLUSTER; ++o) {
      const int from = int(all_steps * o / FEW_CLUSTER);
      if (from >= end) break;
      const int to = int(all_steps * (o + 1) / FEW_CLUSTER);
      if (from == to) continue;
      for (int m = 0; m < 2; ++m) {
        const float4 v = __ldcg(&p.parts[(((cluster * FEW_CLUSTER + o) * 4 + warp) * 2 + m) * 32 + lane]);
        left[m][0] += v.x; left[m][1] += v.y; left[m][2] += v.z; left[m][3] += v.w;
      }
    }
    finish(item0 + last_item, left);
  }
}

template <int W>
__global__ void __launch_bounds__(FEW_DOWN_THREADS, 2) few_down_kernel(const __grid_constant__ CUtensorMap map, const FewArgs p) {
  using Tile = FewTile<W, FEW_DOWN_ROWS>;
  constexpr bool SCALED = W == FEW_FP4_F16;            // a stage: weights, the tokens' activations, and (fp16 form) these's scales [step][token]
  constexpr int H_LD = Tile::CHUNKS * 128 + 64, H_OFF = Tile::CHUNKS * Tile::BYTES, S_OFF = H_OFF + FEW_TOKENS * H_LD,
                STAGE = (S_OFF + (SCALED ? Tile::CHUNKS * FEW_TOKENS * 4 : 0) + 1023) / 1024 * 1024;
  constexpr int STAGES = Tile::ring(FEW_DOWN_RING, STAGE), TEAMS = Tile::TEAMS;
  static_assert(STAGES >= TEAMS, "a place for every team");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ FewBars bars;
  __shared__ FewPlan plan;
  __shared__ __align__(16) float red[TEAMS * (FEW_OUT + 2 * FEW_CLUSTER)];     // [sender: CTA, team][outputs of this CTA]
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int rank = int(cluster_ctarank()), splits = p.splits, n0 = int(blockIdx.x) / splits * FEW_DOWN_ROWS;
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  if (threadIdx.x == FEW_DOWN_THREADS - 1) few_init(bars, STAGES, 1 + 32, 8 / TEAMS);       // (a thread that has nothing of the plan to fetch)
  static_assert(sizeof(FewPlan) / 16 < FEW_DOWN_THREADS, "one piece a thread");
  pdl_launch_dependents();
  {
    const uint4* src = reinterpret_cast<const uint4*>(p.plan);
    for (int i = threadIdx.x; i < int(sizeof(FewPlan) / 16); i += FEW_DOWN_THREADS) reinterpret_cast<uint4*>(&plan)[i] = src[i];
  }
  __syncthreads();
  const int chunks = p.I >> 6, steps = (chunks + Tile::CHUNKS - 1) / Tile::CHUNKS, total = plan.met * steps;
  const int lo = int(unsigned(total) * rank / splits), hi = int(unsigned(total) * (rank + 1) / splits);
  // outputs [row of the tile][token], dealt out to the cluster's CTAs in runs of `per`
  const int per = ((FEW_OUT + splits - 1) / splits + 1) & ~1, first = rank * per, last = min(FEW_OUT, first + per);
  auto output = [&](int i, int& n, int& t) {
    n = n0 + (first + i) / FEW_TOKENS;
    t = (first + i) % FEW_TOKENS;
    return first + i < last && n < p.H && t < p.T;
  };
  float bias[2] = {0.f, 0.f};                          // of this thread's outputs, fetched while the first stages are on their way
  if (p.down_b) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      int n, t;
      if (output(int(threadIdx.x) + k * FEW_DOWN_THREADS, n, t))
        for (int j = 0; j < p.top; ++j) bias[k] += plan.share[t * p.top + j] * bf2f(p.down_b[(long long)(plan.ids[t * p.top + j] & (FEW_AGAIN - 1)) * p.H + n]);
    }
  }
  bool ok = true;
  float sum[2][4] = {};
  const int team = warp >> 1, r0 = (warp & 1) * 32 + g;
  int d = lo / steps, c = (lo - d * steps) * Tile::CHUNKS;
  if (warp == 8) {                       // weights
    FewRing r{STAGES};
    for (int i = lo; i < hi; ++i) {
      ok = r.wait_empty(bars, p.status);
      if (!ok) break;
      const int n = min(Tile::CHUNKS, chunks - c);
      if (elect_one()) {
        mbar_expect_tx(&bars.full[r.s], n * Tile::COPIED);
        Tile::copy(ring + r.s * STAGE, &bars.full[r.s], &map, p.down, plan.expert[d], n0, c, n, p.H, p.I);
      }
      __syncwarp();
      r.next();
      c += Tile::CHUNKS;
      if (c >= chunks) { c = 0; ++d; }
    }
    if (!ok) r.drain(bars);
  } else if (warp == 9) {                // scales of half records, and the activations of the tokens that meet the expert
    FewRing r{STAGES};
    constexpr int PAIRS = FEW_TOKENS / 2;
    const int piece = lane & 15;                         // a half of the warp takes a token at a time, 16 bytes a lane
    const uint16_t* from[PAIRS] = {};                    // every second one of the tokens that meet expert `now`: its activations, and its place in a stage
    int place[PAIRS] = {}, pairs = 0, now = -1;
    // What is small goes by pieces of 16 bytes, one a lane: scales of the weights' half records, then (fp16 form) the activations'.  A lane's piece is of step `of`.
    constexpr bool HALVES = Tile::COPIED < Tile::BYTES;
    constexpr int FIRST = HALVES ? Tile::CHUNKS * Tile::EACH : 0, LAST = FIRST + (SCALED ? Tile::CHUNKS * 2 : 0);
    static_assert(LAST <= 32, "a piece a lane");
    const bool weights = lane < FIRST;
    const int of = lane >= LAST ? Tile::CHUNKS : weights ? lane / Tile::EACH : (lane - FIRST) >> 1;
    const int small_to = weights ? of * Tile::BYTES + Tile::scales_in_step(lane % Tile::EACH) : S_OFF + (lane - FIRST) * 16;
    const long long record = (long long)((p.H + 127) >> 7) * FP4_RECORD_BYTES, small_step = Tile::CHUNKS * (weights ? record : FEW_TOKENS * 4);
    const uint8_t* small = nullptr;
    for (int i = lo; i < hi; ++i) {
      if (d != now) {
        now = d;
        uint32_t left = __ballot_sync(0xffffffffu, lane < p.T && plan.slot[d][lane & 7] != 255);
        pairs = (__popc(left) + 1) / 2;
        if (lane >= 16) left &= left - 1;
#pragma unroll
        for (int u = 0; u < PAIRS; ++u) {
          const int t = left ? __ffs(left) - 1 : -1;
          left &= left - 1;
          left &= left - 1;
          place[u] = t < 0 ? -1 : H_OFF + t * H_LD + piece * 16;
          if (t >= 0) from[u] = p.h + (long long)(t * p.top + plan.slot[d][t]) * p.I + piece * 8;
        }
        if (LAST > 0) {
          const uint8_t* tile = static_cast<const uint8_t*>(p.down) + (n0 >> 7) * FP4_RECORD_BYTES + Tile::scales_in_record(n0, lane % Tile::EACH);
          small = weights ? tile + ((long long)plan.expert[d] * chunks + c + of) * record
                          : reinterpret_cast<const uint8_t*>(p.h_scale + ((long long)d * chunks + c + of) * FEW_TOKENS) + (lane & 1) * 16;
        }
      }
      ok = r.wait_empty(bars, p.status);
      if (!ok) break;
      const int n = min(Tile::CHUNKS, chunks - c);
      uint8_t* st = ring + r.s * STAGE;
      if (LAST > 0) {
        if (of < n) cp_async16(st + small_to, small, true);
        small += small_step;
      }
#pragma unroll
      for (int u = 0; u < PAIRS; ++u) {
        if (u >= pairs) break;
        if (place[u] >= 0 && piece < n * 8) cp_async16(st + place[u], from[u] + c * 64, true);
      }
      __syncwarp();
      cp_async_arrive(&bars.full[r.s]);
      r.next();
      c += Tile::CHUNKS;
      if (c >= chunks) { c = 0; ++d; }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    float acc[2][4] = {};
    FewReader<STAGE, TEAMS> r(&bars, ring, STAGES, team);
    const uint32_t place = Tile::place(r0, g, q), scales = Tile::scales(r0), hs = H_OFF + g * H_LD + q * 16, ss = S_OFF + q * 8;
    auto scaling = [](const uint2& v) { return make_float2(__uint_as_float(v.x), __uint_as_float(v.y)); };
    auto masked = [](const uint4& v, uint32_t m) { return make_uint4(v.x & m, v.y & m, v.z & m, v.w & m); };
    int i = lo + team;                                   // this team's next step
    for (int from = lo; from < hi; ++d) {
      const int begin = d * steps, to = min(hi, begin + steps);
      const uint32_t meets = plan.slot[d][g] != 255 ? ~0u : 0u;        // else what lies in the token's place is left over
      for (; i < to; i += TEAMS) {
        if (ok && (ok = r.wait(p.status))) {
          const uint32_t x = r.data + hs;
          uint4 b[2] = {masked(lds128<0>(x), meets), masked(lds128<64>(x), meets)};
          Tile::template mma<SCALED>(acc, r.data + place, r.data + scales, b, scaling(SCALED ? lds64<0>(r.data + ss) : make_uint2(0u, 0u)));
          if ((i - begin) * Tile::CHUNKS + 1 < chunks) {
            b[0] = masked(lds128<128>(x), meets);
            b[1] = masked(lds128<192>(x), meets);
            Tile::template mma<SCALED>(acc, r.data + Tile::BYTES + place, r.data + Tile::BYTES + scales, b, scaling(SCALED ? lds64<FEW_TOKENS * 4>(r.data + ss) : make_uint2(0u, 0u)));
          }
          r.release(lane, acc);
        }
        r.next();
      }
      // an expert's part is done: it counts for the tokens that meet it (weights that are not numbers stay with them)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (plan.slot[d][q * 2 + (j & 1)] != 255) { sum[0][j] += acc[0][j]; sum[1][j] += acc[1][j]; }
        acc[0][j] = acc[1][j] = 0.f;
      }
      from = to;
    }
  }
  __syncwarp();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");        // of the arrival at the start
  if (warp < 8) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int o = (r0 + j * 8) * FEW_TOKENS + q * 2, owner = o / per;
      asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};"
                   ::"r"(dsmem_addr(smem_u32(&red[(rank * TEAMS + team) * per + o - owner * per]), uint32_t(owner))), "f"(sum[j >> 1][(j & 1) * 2]), "f"(sum[j >> 1][(j & 1) * 2 + 1])
                   : "memory");
    }
  }
  __syncwarp();
  cluster_sync_all();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    int n, t;
    const int i = int(threadIdx.x) + k * FEW_DOWN_THREADS;
    if (!output(i, n, t)) continue;
    float v = 0.f;
    for (int s = 0; s < splits * TEAMS; ++s) v += red[s * per + i];
    p.out[(long long)t * p.H + n] = f2bf(v + bias[k]);
  }
}

// --------------------------------------------------------------------------------- host side
// Shared memory of the first kernel: besides its ring's, and what its ring has to have room for at least (a place for each team, of the largest stage)
static size_t few_fixed(int T, int H) { return 1024 + sizeof(FewShared) + size_t(T) * ((H + 63) / 64 * 64 + 32) * 2; }
static size_t few_before(int T, int E) { return (sizeof(FewBefore) + size_t(T) * E * 4 + 15) / 16 * 16; }
static bool few_fits(int T, int H, int E) {
  using Tile = FewTile<FEW_BF16, 128>;
  constexpr size_t least = Tile::TEAMS * Tile::CHUNKS * Tile::BYTES;
  static_assert(Tile::CHUNKS * Tile::BYTES >= FewTile<FEW_FP4_F16, 128>::CHUNKS * FewTile<FEW_FP4_F16, 128>::BYTES, "the largest stage");
  return H <= 65536 && few_fixed(T, H) + max(least, few_before(T, E)) <= FEW_SMEM_ONE;
}

template <int W>
static int LaunchFew(FewArgs p, int sm_count, cudaStream_t stream) {
  using Tile = FewTile<W, 128>;
  constexpr int STAGE = Tile::CHUNKS * Tile::BYTES;
  const size_t fixed = few_fixed(p.T, p.H), before = few_before(p.T, p.E);
  // Two CTAs an SM where that leaves each a ring of 48 KiB: more warps to multiply, more stages in work (7 mxfp4 tokens of 2880 columns: 98 us, one CTA with 16 stages 123);
  // else one with what there is (8 bf16 tokens of 4096 columns: 453 us, two with two stages each 497).
  const int two = fixed + max(size_t(48 * 1024), before) <= FEW_SMEM_TWO;
  const size_t room = two ? FEW_SMEM_TWO : FEW_SMEM_ONE;
  p.stages = Tile::ring(int(room - fixed), STAGE);
  p.ring_bytes = int(max(size_t(p.stages * STAGE), before));
  CUtensorMap gate_up = {}, down = {};
  if (W == FEW_BF16 && (!encode_map_2d(&gate_up, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.gate_up, uint64_t(p.E) * 2 * p.I, p.H, uint64_t(p.H) * 2, 128, 64, CU_TENSOR_MAP_SWIZZLE_128B) ||
                        !encode_map_2d(&down, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.down, uint64_t(p.E) * p.H, p.I, uint64_t(p.I) * 2, FEW_DOWN_ROWS, 64, CU_TENSOR_MAP_SWIZZLE_128B)))
    return -2;
  static bool configured[OGB_MAX_DEVICES] = {}, configured_down[OGB_MAX_DEVICES] = {};
  if (!set_max_dyn_smem(few_gate_up_kernel<W>, int(FEW_SMEM_ONE), configured) || !set_max_dyn_smem(few_down_kernel<W>, FEW_DOWN_RING + 1024, configured_down)) return -3;
  // Both kernels are launched behind the complete kernels in front of them: CTAs that come in as others leave are placed so that some clusters find no room until the
  // rest is done (8 tokens of 2 of 8 bf16 experts of 14336 in a row: 913 us a layer with programmatic launches of an earlier form, 590 without; the second kernel's alone: 1 mxfp4 token
  // 37 to 38 us instead of 31).
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {FEW_CLUSTER, 1, 1};
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
    clusters = min(clusters, FEW_MAX_CTAS / FEW_CLUSTER);
    if (tracked) clusters_at[dev][two] = clusters;
  }
  cfg.dynamicSmemBytes = fixed + p.ring_bytes;
  cfg.gridDim = dim3(unsigned(clusters * FEW_CLUSTER));
  if (cudaLaunchKernelEx(&cfg, few_gate_up_kernel<W>, gate_up, p) != cudaSuccess) return -4;
  const int tiles = (p.H + FEW_DOWN_ROWS - 1) / FEW_DOWN_ROWS;
  p.splits = max(1, min(FEW_CLUSTER, 2 * sm_count / tiles));                          // two CTAs an SM
  attr[0].val.clusterDim = {unsigned(p.splits), 1, 1};
  cfg.blockDim = dim3(FEW_DOWN_THREADS);
  cfg.dynamicSmemBytes = FEW_DOWN_RING + 1024;
  cfg.gridDim = dim3(unsigned(tiles * p.splits));
  return cudaLaunchKernelEx(&cfg, few_down_kernel<W>, down, p) == cudaSuccess ? 0 : -4;
}

}  // namespace ogb

using namespace ogb;

OGB_API long long ogb_moe_few_scratch_bytes(int T, int top, int I) {
  return T < 1 || T > FEW_TOKENS || top < 1 || top > FEW_TOP || I < 1 ? -1 : (long long)sizeof(FewPlan) + FEW_MAX_CTAS * 4096LL + (long long)T * top * (I * 2LL + I / 64 * (FEW_TOKENS * 4LL));
}

OGB_API int ogb_moe_few_takes(int T, int H, int I, int E, int top) {
  return ogb_moe_few_scratch_bytes(T, top, I) >= 0 && H >= 1 && H % 8 == 0 && I % 64 == 0 && E >= top && E <= FEW_EXPERTS && few_fits(T, H, E);
}

OGB_API int ogb_moe_few_tokens(const void* x, long long ldx, const void* router, const void* router_b, const void* gate_up, const void* gate_up_b,
                               const void* down, const void* down_b, void* out, int T, int H, int I, int E, int top, int rule, int weights, int act,
                               float alpha, float limit, void* scratch, int* status, int sm_count, void* stream) {
  if (!ogb_moe_few_takes(T, H, I, E, top) || !x || !router || !gate_up || !down || !out || !scratch || (weights != FEW_BF16 && H % 64) || rule < 0 || rule > 2 ||
      weights < 0 || weights > 2 || (act != 1 && act != 2)) return -1;
  if ((reinterpret_cast<uintptr_t>(x) | uintptr_t(ldx * 2) | reinterpret_cast<uintptr_t>(router) | reinterpret_cast<uintptr_t>(gate_up) | reinterpret_cast<uintptr_t>(down) | reinterpret_cast<uintptr_t>(scratch)) & 15)
    return -1;
  FewArgs p{static_cast<const __nv_bfloat16*>(x), ldx, static_cast<const __nv_bfloat16*>(router), static_cast<const __nv_bfloat16*>(router_b), gate_up,
            static_cast<const __nv_bfloat16*>(gate_up_b), down, static_cast<const __nv_bfloat16*>(down_b), static_cast<__nv_bfloat16*>(out), T, H, I, E, top,
            rule, act, alpha, limit, static_cast<FewPlan*>(scratch), reinterpret_cast<float4*>(static_cast<uint8_t*>(scratch) + sizeof(FewPlan)),
            reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(scratch) + sizeof(FewPlan) + FEW_MAX_CTAS * 4096LL), nullptr, 0, 0, 0, status};
  p.h_scale = reinterpret_cast<float*>(p.h + (long long)T * top * I);
  if ((long long)E * 2 * I > 0x7fffffff || (long long)E * H > 0x7fffffff || (long long)min(E, T * top) * I * H > 1LL << 37) return -5;   // (32-bit counts of steps)
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (weights == FEW_BF16) return LaunchFew<FEW_BF16>(p, sm_count, s);
  return weights == FEW_FP4_F16 ? LaunchFew<FEW_FP4_F16>(p, sm_count, s) : LaunchFew<FEW_FP4_BF16>(p, sm_count, s);
}
