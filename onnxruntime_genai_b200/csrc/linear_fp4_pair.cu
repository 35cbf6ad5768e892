// 4-bit products of prompts on pairs of SMs (see linear_fp4.cu for the operation): a cluster of two CTAs walks a list of output tiles of 256 weight rows x up to
// 192 tokens (`tcgen05.mma.cta_group::2`, M = 256).  Each CTA holds 128 of the weight rows and half of the token rows, the scales of its weight rows and of all
// tokens, and the accumulator of its own 128 rows in its tensor memory.
//
// Bound by what an SM can take in from L2 beside the tensor cores: a k-block of 256 takes the pair 384 cycles of MMAs and brings 34 KB into each SM; one CTA per
// 128 x 128 tile needs 36 KB for 256 cycles.  192 tokens, because two accumulators (drained in turns) and two sets of scales then share the 512 columns of tensor
// memory: 2 x 192 + 2 x (16 + 32).  A tile starts at a multiple of 64 tokens, two columns of scales.
//
// Warps of a CTA: 0 and 2 copy weights and tokens, 1 issues scale copies and MMAs (of the cluster's first CTA), all as whole warps with one elected lane; 3..10 drain
// accumulators, two teams 16 tokens at a time through staging tiles that turn a weight row per thread into 16-byte row segments.  Copies of both CTAs are counted on the first CTA's
// barrier of a stage; a commit frees the stage in both.  All waits are bounded; after a failed one every role leaves its loop, both CTAs meet at the last cluster
// barrier and return with the status word set.
#include "kernels.h"
#include "linear_fp4.cuh"
#include "pair.cuh"
#include "tensor_map.cuh"

namespace ogb {

constexpr int FP4P_BT = 192, FP4P_LD = FP4_TILE + 4;
template <int FORM>
struct Fp4PairCfg {
  static constexpr int SF = fp4_sf_bytes(FORM);
  static constexpr int X_OFF = FP4_W_BYTES, SFW_OFF = X_OFF + FP4P_BT / 2 * 128, SFX_OFF = SFW_OFF + SF;
  static constexpr int BLOCK = SFX_OFF + 2 * SF;                       // a k-block: codes of 128 weight rows and half of the tokens, scales of 128 weight rows and 256 tokens
  static constexpr int KB = 2, STAGE = KB * BLOCK, STAGES = 3;         // a role's pass over a stage costs some 650 cycles whatever it holds: two k-blocks
  static constexpr int STAGING = STAGES * STAGE, BARS = STAGING + 32 * FP4P_LD * 4, SMEM = BARS + 256 + 1024;
  static constexpr int SF_COL = 2 * FP4P_BT, SF_SET = 64;              // tensor memory: accumulators, then two sets of scales (16 columns of weights, 32 of tokens)
  static_assert(BLOCK % 1024 == 0 && SMEM <= 227 * 1024 && SF_COL + 2 * SF_SET <= 512, "memory");
};

struct Fp4PairArgs {
  int bt, m_tiles, n_pairs;      // tokens of a tile, tiles along the tokens, pairs of weight tiles
};

template <int FORM>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(352, 1)
linear_fp4_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_sw,
                       const __grid_constant__ CUtensorMap map_sx, const Fp4LinearArgs p, const Fp4PairArgs a) {
  using Cfg = Fp4PairCfg<FORM>;
  constexpr int S = Cfg::STAGES, STEPS = fp4_steps(FORM);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* staging = reinterpret_cast<float*>(smem + Cfg::STAGING);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::BARS);      // [S] copies -> MMA (first CTA's)
  uint64_t* empty = full + S;                                          // [S] MMA -> copies (both)
  uint64_t* acc_full = empty + S;                                      // [2] MMA -> drain (both)
  uint64_t* acc_empty = acc_full + 2;                                  // [2] drain of both CTAs -> MMA (first CTA's)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* epi_abort = reinterpret_cast<volatile int*>(tmem_slot + 2);     // [team]

  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1, num_kb = p.w.num_kb, total = a.m_tiles * a.n_pairs;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 16); }
    *abort_flag = 0;
    epi_abort[0] = epi_abort[1] = 0;
    mbar_fence_init();
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_sw);
    tma_prefetch_desc(&map_sx);
  }
  __syncwarp();
  if (warp == 2) pair_tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  cluster_sync_all();                      // barriers of both CTAs are initialised, tensor memory is allocated
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (p.pdl) pdl_launch_dependents();
  // Tiles that run at the same time share the weight rows of the moment and all tokens in L2.
  struct Tile { int n_tile, row0, rows, cols; };
  auto tile_at = [&](int t) {
    const int n = t / a.m_tiles;
    Tile x;
    x.n_tile = n * 2 + int(rank);
    x.row0 = (t - n * a.m_tiles) * a.bt;
    x.rows = min(a.bt, p.a.rows - x.row0);
    x.cols = (x.rows + 31) & ~31;          // token columns of the MMA
    return x;
  };
  auto fail = [&](int code) { atomicMax(p.status, code); *abort_flag = 1; };

  if (warp == 0 || warp == 2) {
    // ------------------------------------------------------------------ copies of all tiles' k-blocks, back to back: weights (warp 0) and tokens (warp 2)
    const bool tokens = warp == 2;
    bool ok = true;
    int it = 0, s = 0;
    uint32_t ph = 1;
    const int tiles_w = p.w.padded >> 7, tiles_x = p.a.padded >> 7;
    const uint32_t bytes = uint32_t(FP4_W_BYTES + a.bt / 2 * 128 + Cfg::SF + (a.bt > 128 ? 2 : 1) * Cfg::SF);
    // the weights may be fetched before the kernel in front has finished, where it writes none; tokens may not
    if (p.pdl && (tokens || !p.early)) pdl_wait();
    for (int t = first; t < total && ok; t += step) {
      const Tile x = tile_at(t);
      int row = tokens ? x.row0 + int(rank) * (x.cols >> 1) : x.n_tile * FP4_TILE, sf = (tokens ? x.row0 >> 7 : x.n_tile) * STEPS;
      const int row_step = tokens ? p.a.padded : p.w.padded, sf_step = (tokens ? tiles_x : tiles_w) * STEPS;
      for (int kb = 0; kb < num_kb; kb += Cfg::KB) {
        if (it >= S) ok = __all_sync(0xffffffffu, mbar_wait_bounded(&empty[s], ph, abort_flag));
        if (!ok) { fail(OGB_ERR_WAIT_TMA); break; }
        if (elect_one()) {
          const int n = min(Cfg::KB, num_kb - kb);
          const uint32_t bar = dsmem_addr(smem_u32(&full[s]), 0);
          if (!tokens && rank == 0) mbar_expect_tx(&full[s], 2 * n * bytes);
#pragma unroll
          for (int h = 0; h < Cfg::KB; ++h) {
            if (h >= n) break;
            uint8_t* st = smem + s * Cfg::STAGE + h * Cfg::BLOCK;
            pair_tma_load_2d(st + (tokens ? Cfg::X_OFF : 0), tokens ? &map_x : &map_w, bar, 0, row + h * row_step);
            pair_tma_load_2d(st + (tokens ? Cfg::SFX_OFF : Cfg::SFW_OFF), tokens ? &map_sx : &map_sw, bar, 0, sf + h * sf_step);
          }
        }
        row += Cfg::KB * row_step;
        sf += Cfg::KB * sf_step;
        __syncwarp();
        ++it;
        if (++s == S) { s = 0; ph ^= 1; }
      }
    }
    if (!ok) {   // copies already issued still write the pair's shared memory: give them time to land
      volatile int never = 0;
      if (rank == 0) for (int i = max(0, it - S); i < it; ++i) mbar_wait_bounded(&full[i % S], (i / S) & 1, &never, 200000000ull);
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // ------------------------------------------------------------------ MMAs of the pair: the two accumulators in turns
      int s = 0, j = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = first; t < total && ok; t += step, ++j) {
        const int buf = j & 1;
        if (j >= 2) ok = __all_sync(0xffffffffu, cluster_wait_bounded(&acc_empty[buf], ((j >> 1) & 1) ^ 1, abort_flag));
        if (!ok) { fail(OGB_ERR_WAIT_MMA); break; }
        tc_fence_after();
        const Tile x = tile_at(t);
        const uint32_t acc = tmem + uint32_t(buf * FP4P_BT), off = uint32_t(x.row0 & 127) >> 5;      // the tile's first column in a step's scales
        const uint32_t idesc = fp4_idesc(FORM, 2 * FP4_TILE, x.cols, 0);
        const bool wide = a.bt > 128;
        for (int kb = 0; kb < num_kb; kb += Cfg::KB) {
          if (!__all_sync(0xffffffffu, mbar_wait_bounded(&full[s], ph, abort_flag))) { fail(OGB_ERR_WAIT_TMA); ok = false; break; }
          tc_fence_after();
          if (elect_one()) {
            const int n = min(Cfg::KB, num_kb - kb);
#pragma unroll
            for (int h = 0; h < Cfg::KB; ++h) {
              if (h >= n) break;
              const uint32_t base = smem_u32(smem + s * Cfg::STAGE + h * Cfg::BLOCK), sf = tmem + Cfg::SF_COL + h * Cfg::SF_SET;
              const uint64_t dw = umma_desc_sw128(base), dx = umma_desc_sw128(base + Cfg::X_OFF);
              const uint64_t dsw = fp4_scale_desc(base + Cfg::SFW_OFF), dsx = fp4_scale_desc(base + Cfg::SFX_OFF);
#pragma unroll
              for (int k = 0; k < STEPS; ++k) {
                fp4_copy_scales<2>(sf + k * 4, dsw + k * (FP4_SCALE_STEP >> 4));
                fp4_copy_scales<2>(sf + 16 + k * 8, dsx + k * (FP4_SCALE_STEP >> 4));
                if (wide) fp4_copy_scales<2>(sf + 16 + k * 8 + 4, dsx + (STEPS + k) * (FP4_SCALE_STEP >> 4));
              }
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int st = FORM == FP4_NV ? k : k >> 1;
                const uint32_t id = FORM == FP4_NV ? 0u : uint32_t(k & 1) * 2u;
                fp4_mma<2, FORM>(acc, dw + k * 2, dx + k * 2, idesc | id << 4 | id << 29, sf + st * 4, sf + 16 + st * 8 + off, kb > 0 || h > 0 || k > 0 ? 1u : 0u);
              }
            }
            pair_commit(&empty[s]);
            if (kb + Cfg::KB >= num_kb) pair_commit(&acc_full[buf]);
          }
          __syncwarp();
          if (++s == S) { s = 0; ph ^= 1; }
        }
      }
    }
  } else {
    // -------------------------------------------------------------------- drain: two teams of four warps take turns at 16 tokens
    const int et = (int(threadIdx.x) - 96) & 127, team = (warp - 3) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const bool pair = p.pair != 0;
    float* mine = staging + team * 16 * FP4P_LD;
    auto meet = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(1 + team) : "memory"); };
    // the eight columns of a token row that this thread finishes: plain, of its own warp's rows; paired, of the 64 gate rows
    const int seg = pair ? (et & 7) * 8 : quarter * 32 + (lane & 3) * 8, tok = pair ? et >> 3 : lane >> 2;
    if (p.pdl) pdl_wait();
    int j = 0;
    for (int t = first; t < total; t += step, ++j) {
      const int buf = j & 1;
      const Tile x = tile_at(t);
      const int n0 = x.n_tile * FP4_TILE, rows = n0 < p.N ? x.rows : 0, col = x.n_tile * (pair ? 64 : FP4_TILE) + seg;
      float ws[8], us[8], wb[8], ub[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool in = n0 + seg + k < p.N;             // (past the last tile: nothing is stored)
        ws[k] = in ? p.w.row_scale[n0 + seg + k] : 0.f;
        wb[k] = in && p.bias ? bf2f(p.bias[n0 + seg + k]) : 0.f;
        us[k] = in && pair ? p.w.row_scale[n0 + seg + 64 + k] : 0.f;
        ub[k] = in && pair && p.bias ? bf2f(p.bias[n0 + seg + 64 + k]) : 0.f;
      }
      // a failed wait is published in a word, before the barrier: the team takes the same branch
      if (!mbar_wait_bounded(&acc_full[buf], (j >> 1) & 1, abort_flag, 4000000000ull)) { fail(OGB_ERR_WAIT_MMA); epi_abort[team] = 1; }
      __syncwarp();
      meet();
      if (epi_abort[team]) break;
      tc_fence_after();
      const uint32_t taddr = tmem + (uint32_t(quarter * 32) << 16) + uint32_t(buf * FP4P_BT);
      for (int c0 = team * 16; c0 < rows; c0 += 32) {
        uint32_t r[16];
        __syncwarp();
        tmem_ld16(taddr + c0, r);
        tmem_ld_wait();
#pragma unroll
        for (int q = 0; q < 16; ++q) mine[q * FP4P_LD + row] = __uint_as_float(r[q]);
        // all values of the chunk are read before the first store: a store through a generic pointer would order the reads behind it
        if (pair) {
          meet();
          const float4* src = reinterpret_cast<const float4*>(mine + tok * FP4P_LD + seg);
          const float4 g0 = src[0], g1 = src[1], h0 = src[16], h1 = src[17];
          const float sc = p.a.row_scale[x.row0 + c0 + tok];                      // (padded to whole tiles)
          meet();
          float v[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w};
          const float u[8] = {h0.x, h0.y, h0.z, h0.w, h1.x, h1.y, h1.z, h1.w};
#pragma unroll
          for (int q = 0; q < 8; ++q) v[q] = fp4_silu(fmaf(v[q], sc * ws[q], wb[q])) * fmaf(u[q], sc * us[q], ub[q]);
          if (c0 + tok < rows && col < p.n_out) fp4_store8(p, x.row0 + c0 + tok, col, v);
        } else {
          __syncwarp();
          float4 g[2][2];
          float sc[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float4* src = reinterpret_cast<const float4*>(mine + (tok + k * 8) * FP4P_LD + seg);
            g[k][0] = src[0]; g[k][1] = src[1];
            sc[k] = p.a.row_scale[x.row0 + c0 + tok + k * 8];
          }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int m = c0 + tok + k * 8;
            float v[8] = {g[k][0].x, g[k][0].y, g[k][0].z, g[k][0].w, g[k][1].x, g[k][1].y, g[k][1].z, g[k][1].w};
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = fmaf(v[q], sc[k] * ws[q], wb[q]);
            if (m < rows && col < p.n_out) fp4_store8(p, x.row0 + m, col, v);
          }
        }
      }
      // accumulator drained: hand it back to the MMA warp of the pair
      tc_fence_before();
      __syncwarp();
      if (lane == 0) cluster_arrive(dsmem_addr(smem_u32(&acc_empty[buf]), 0));
    }
  }

  __syncwarp();
  tc_fence_before();
  cluster_sync_all();      // no CTA leaves while the pair's MMAs, copies or arrivals may still reach its memory
  if (warp == 2) pair_tmem_dealloc(tmem, 512);
}

// --------------------------------------------------------------------------------- host side
template <int FORM>
static int LaunchPair(const Fp4LinearArgs& p, int sm_count, cudaStream_t stream) {
  using Cfg = Fp4PairCfg<FORM>;
  static bool configured[OGB_MAX_DEVICES] = {};
  if (!set_max_dyn_smem(linear_fp4_pair_kernel<FORM>, Cfg::SMEM, configured)) return -3;
  const int pairs = sm_count / 2, T = p.a.rows;
  Fp4PairArgs a = {};
  a.n_pairs = (p.N + 2 * FP4_TILE - 1) / (2 * FP4_TILE);
  // Tiles of 64, 128 or 192 tokens: rounds of the pairs x the time of a k-block, which is the MMAs' down to what a role's pass over a stage takes
  double best = 0;
  for (int bt = 64; bt <= FP4P_BT; bt += 64) {
    const int m = (T + bt - 1) / bt;
    const double ns = double((m * a.n_pairs + pairs - 1) / pairs) * p.w.num_kb * (1.1 * bt > 150. ? 1.1 * bt : 150.) + bt * 10.;
    if (a.bt == 0 || ns < best) { best = ns; a.bt = bt; a.m_tiles = m; }
  }
  CUtensorMap mw, mx, msw, msx;
  const uint32_t steps = fp4_steps(FORM), wide = a.bt > 128 ? 2 : 1;
  const auto words = CU_TENSOR_MAP_DATA_TYPE_UINT32;
  const auto plain = CU_TENSOR_MAP_SWIZZLE_NONE;
  if (!encode_map_2d(&mw, words, p.w.codes, uint64_t(p.w.num_kb) * p.w.padded, 32, 128, FP4_TILE, 32, plain) ||
      !encode_map_2d(&mx, words, p.a.codes, uint64_t(p.a.num_kb) * p.a.padded, 32, 128, a.bt / 2, 32, plain) ||
      !encode_map_2d(&msw, words, p.w.scales, uint64_t(p.w.num_kb) * (p.w.padded >> 7) * steps, 128, 512, steps, 128, plain) ||
      !encode_map_2d(&msx, words, p.a.scales, uint64_t(p.a.num_kb) * (p.a.padded >> 7) * steps, 128, 512, steps * wide, 128, plain)) return -2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(2 * min(pairs, a.n_pairs * a.m_tiles)));
  cfg.blockDim = dim3(352);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = p.pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, linear_fp4_pair_kernel<FORM>, mw, mx, msw, msx, p, a) == cudaSuccess ? 0 : -4;
}

int LaunchPairLinearFp4(const Fp4LinearArgs& p, int form, int sm_count, cudaStream_t stream) {
  return form == FP4_NV ? LaunchPair<FP4_NV>(p, sm_count, stream) : LaunchPair<FP4_MX>(p, sm_count, stream);
}

}  // namespace ogb
