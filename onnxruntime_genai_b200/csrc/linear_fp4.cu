// Linear layers on 4-bit floating-point rows and weights (layout: fp4_matrix.cuh):
//   C[t, n] = a_row[t] * w_row[n] * sum_blocks a_scale * w_scale * sum_k a_code * w_code   (+ bias, residual, or the gated activation)
//
// Both operands go to the block-scaled tensor-core product (`tcgen05.mma.kind::mxf4nvf4.block_scale`) as they are: codes from shared memory, block
// scales from tensor memory, fp32 accumulators.  Weights are the M operand (128 rows a CTA), tokens the N operand.
//
// Up to 64 tokens (linear_fp4_kernel): bound by the weights' bytes.  A CTA holds one tile of 128 weight rows x BT tokens of a part of the k-blocks; the parts of a
// tile form a cluster that sums its accumulators through distributed shared memory, always in the same order.  One or two rows are quantised here too.  More tokens: linear_fp4_pair.cu.
#include "kernels.h"
#include "linear_fp4.cuh"
#include "packed_weights.cuh"
#include "quantize_fp4.cuh"

namespace ogb {

// ------------------------------------------------------------------------------- few tokens
// ROWS: the rows are there in 4 bits (FP4_GIVEN), or a CTA quantises what it needs of one or two of them, bf16 or fp32, while its weights are on the way.
enum Fp4Rows : int { FP4_GIVEN = 0, FP4_BF16 = 1, FP4_FP32 = 2 };
constexpr int FP4_OWN_ROWS = 2, FP4_OWN_WORK = 40, FP4_OWN_PART = 13;           // rows; k-blocks of them that a CTA reads, twice its own; most of its own then

template <int BT, int FORM, int ROWS = FP4_GIVEN>
struct Fp4Cfg {
  static constexpr int SF = fp4_sf_bytes(FORM);
  static constexpr int X_OFF = FP4_W_BYTES, SFW_OFF = X_OFF + (ROWS ? 0 : BT * 128), SFX_OFF = SFW_OFF + SF;
  static constexpr int STAGE = ROWS ? SFX_OFF : SFX_OFF + SF;                    // codes of weights and tokens, scales of weights and of 128 tokens
  // Rows that the CTA quantises lie behind the ring: of a k-block eight rows of codes, then (of all k-blocks) 128 bytes of scales a step.  The tensor core reads sixteen
  // rows and scales of 32; what it takes for the others is what lies behind, and goes into columns that nobody reads.
  static constexpr int OWN_SF = fp4_steps(FORM) * 128;
  static constexpr int own(int kbs) { return ROWS ? (kbs * (1024 + OWN_SF) + 1024 + 1023) / 1024 * 1024 : 0; }
  // Partial sums that other CTAs of the cluster send: up to 32 tokens have a place of their own, more take the stages once the whole cluster is done with them
  static constexpr bool APART = BT <= 32;
  static constexpr int SUMS = (BT + 8) * FP4_TILE * 4;
  static constexpr int ROOM = 110 * 1024 - (APART ? SUMS : 0);                     // two CTAs per SM
  static constexpr int STAGES = ROWS ? 5 : ROOM / STAGE;
  static constexpr int SF_COL = BT < 32 ? 32 : BT;                                // first tensor-memory column of the scales: two sets of 16 + 16
  static constexpr int COLS = 128;
  static_assert(STAGE % 1024 == 0 && STAGES >= 2 && SF_COL + 64 <= COLS, "stages, tensor memory");
  static constexpr int smem(int stages, int kbs) {
    const int ring = stages * STAGE + own(kbs);
    return (APART ? ring + SUMS : ring > SUMS ? ring : SUMS) + 1024 + 256;
  }
};

template <int BT, int FORM, int ROWS>
__global__ void __launch_bounds__(192, 3) linear_fp4_kernel(const Fp4LinearArgs p) {
  using Cfg = Fp4Cfg<BT, FORM, ROWS>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int stages = p.stages, kb_room = p.kb_per_split, ring = stages * Cfg::STAGE + Cfg::own(kb_room);
  uint8_t* own_codes = smem + stages * Cfg::STAGE;
  uint8_t* own_scales = own_codes + kb_room * 1024;
  __shared__ uint32_t s_top[FP4_OWN_ROWS];                  // bits of the rows' largest magnitudes
  float* sums = reinterpret_cast<float*>(smem + (Cfg::APART ? ring : 0));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::smem(stages, kb_room) - 1024 - 256);
  uint64_t* empty = full + Cfg::STAGES;
  uint64_t* accum = empty + Cfg::STAGES;
  uint64_t* quantised = accum + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(quantised + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int n_tile = blockIdx.x, rows = p.a.rows;           // at most BT
  const int kb0 = blockIdx.z * p.kb_per_split, num = min(p.kb_per_split, p.w.num_kb - kb0);       // at least one
  auto fail = [&](int code) { atomicMax(p.status, code); *abort_flag = 1; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    mbar_init(accum, 1);
    mbar_init(quantised, 128);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (ROWS && threadIdx.x >= 64 && threadIdx.x < 64 + FP4_OWN_ROWS) s_top[threadIdx.x - 64] = 0;
  if (warp == 1) { tmem_alloc(tmem_slot, Cfg::COLS); tmem_relinquish(); }
  __syncwarp();                                             // (lanes may be apart behind the branches above: the arrival wants whole warps)
  if (p.splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");         // sums are sent to CTAs that run
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (p.pdl) pdl_launch_dependents();

  if (warp == 0) {
    // ---------------------------------------------------------------- copies
    const uint8_t* w = p.w.codes + (long long)n_tile * FP4_W_BYTES;
    const uint8_t* sw = p.w.scales + (long long)n_tile * Cfg::SF;
    const uint8_t* x = p.a.codes;
    const uint8_t* sx = p.a.scales;
    const long long w_step = (long long)p.w.padded * 128, x_step = (long long)p.a.padded * 128;
    const long long sw_step = (long long)(p.w.padded >> 7) * Cfg::SF, sx_step = (long long)(p.a.padded >> 7) * Cfg::SF;
    auto weights = [&](int i, int s) {
      uint8_t* st = smem + s * Cfg::STAGE;
      mbar_expect_tx(&full[s], Cfg::STAGE);
      bulk_copy_g2s(st, w + (kb0 + i) * w_step, FP4_W_BYTES, &full[s]);
      bulk_copy_g2s(st + Cfg::SFW_OFF, sw + (kb0 + i) * sw_step, Cfg::SF, &full[s]);
    };
    auto tokens = [&](int i, int s) {
      if (ROWS) return;
      uint8_t* st = smem + s * Cfg::STAGE;
      bulk_copy_g2s(st + Cfg::X_OFF, x + (kb0 + i) * x_step, BT * 128, &full[s]);
      bulk_copy_g2s(st + Cfg::SFX_OFF, sx + (kb0 + i) * sx_step, Cfg::SF, &full[s]);
    };
    const int ahead = min(num, stages);
    if (p.pdl && !p.early) pdl_wait();
    if (elect_one()) for (int i = 0; i < ahead; ++i) weights(i, i);
    __syncwarp();
    if (p.pdl && p.early) pdl_wait();
    if (elect_one()) for (int i = 0; i < ahead; ++i) tokens(i, i);
    __syncwarp();
    bool ok = true;
    int s = 0, filled = ahead;
    uint32_t ph = 0;
    for (int i = ahead; i < num; ++i) {
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&empty[s], ph, abort_flag));
      if (!ok) { fail(OGB_ERR_WAIT_TMA); break; }
      if (elect_one()) { weights(i, s); tokens(i, s); }
      __syncwarp();
      ++filled;
      if (++s == stages) { s = 0; ph ^= 1; }
    }
    if (!ok || *abort_flag) {     // copies in flight still write this shared memory: give them time to land
      volatile int never = 0;
      for (int i = max(0, filled - stages); i < filled; ++i) mbar_wait_bounded(&full[i % stages], (i / stages) & 1, &never, 200000000ull);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- products
    int s = 0;
    uint32_t ph = 0;
    const bool there = !ROWS || __all_sync(0xffffffffu, mbar_wait_bounded(quantised, 0, abort_flag));
    if (!there) fail(OGB_ERR_WAIT_TMA);
    for (int i = 0; there && i < num; ++i) {
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&full[s], ph, abort_flag))) { fail(OGB_ERR_WAIT_TMA); break; }
      tc_fence_after();
      if (elect_one()) {
        const uint32_t base = smem_u32(smem + s * Cfg::STAGE), sf = tmem + Cfg::SF_COL + (i & 1) * 32;
        const uint64_t dw = umma_desc_sw128(base), dx = umma_desc_sw128(ROWS ? smem_u32(own_codes + i * 1024) : base + Cfg::X_OFF);
        const uint64_t dsw = fp4_scale_desc(base + Cfg::SFW_OFF), dsx = fp4_scale_desc(ROWS ? smem_u32(own_scales + i * Cfg::OWN_SF) : base + Cfg::SFX_OFF);
#pragma unroll
        for (int j = 0; j < fp4_steps(FORM); ++j) {
          fp4_copy_scales<1>(sf + j * 4, dsw + j * (FP4_SCALE_STEP >> 4));
          fp4_copy_scales<1>(sf + 16 + j * 4, dsx + j * ((ROWS ? 128 : FP4_SCALE_STEP) >> 4));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {                       // 64 k values: 32 bytes of a row
          const int col = FORM == FP4_NV ? j * 4 : (j >> 1) * 4;
          fp4_mma<1, FORM>(tmem, dw + j * 2, dx + j * 2, fp4_idesc(FORM, FP4_TILE, BT, FORM == FP4_NV ? 0 : (j & 1) * 2), sf + col, sf + 16 + col,
                           i > 0 || j > 0 ? 1u : 0u);
        }
        umma_commit(&empty[s]);
        if (i == num - 1) umma_commit(accum);
      }
      __syncwarp();
      if (++s == stages) { s = 0; ph ^= 1; }
    }
  }

  // ------------------------------------------------------------------ results (warps 2..5)
  // Token rows are dealt out to the CTAs of the cluster; every CTA sends its part of a row's sums to the row's CTA, at [sender][row][128 outputs].
  const int rank = p.splits > 1 ? int(cluster_ctarank()) : 0, per = (rows + p.splits - 1) / p.splits;
  const int et = int(threadIdx.x) - 64, segs = p.pair ? 8 : 16, seg = (et & (segs - 1)) * 8, g = n_tile * FP4_TILE + seg;
  const int first = min(rows, rank * per), last = min(rows, first + per);
  float ws[8], us[8], wb[8], ub[8];
  if (warp >= 2) {
    if (p.pdl) pdl_wait();
    if constexpr (ROWS != FP4_GIVEN) {
      // The rows' largest magnitudes, then this CTA's k-blocks; a warp takes a row's k-block at a time.
      using T = std::conditional_t<ROWS == FP4_BF16, __nv_bfloat16, float>;
      const T* x = static_cast<const T*>(p.x);
      auto fetch = [&](int t, int kb) {
        Raw8<T> r;
        const int k = kb * FP4_KB + lane * 8;
        const T* from = x + t * p.ldx + k;
        if (k >= p.K) r.zero(); else if (p.x_vec) r.template load<true>(from); else r.template load<false>(from);
        return r;
      };
      constexpr int AT_ONCE = ROWS == FP4_BF16 ? 8 : 4;
      for (int i = warp - 2; i < rows * p.w.num_kb; i += 4 * AT_ONCE) {
        Raw8<T> r[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
          const int n = i + 4 * j, t = n / p.w.num_kb;
          if (n < rows * p.w.num_kb) r[j] = fetch(t, n - t * p.w.num_kb); else r[j].zero();
        }
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
          const int n = i + 4 * j;
          if (n >= rows * p.w.num_kb) break;
          const uint32_t top = __reduce_max_sync(0xffffffffu, r[j].largest());
          if (lane == 0) atomicMax(&s_top[n / p.w.num_kb], top);
        }
      }
      __syncwarp();
      asm volatile("bar.sync 1, 128;" ::: "memory");
      constexpr int PER = FORM == FP4_NV ? 2 : 4;                              // lanes of a block
      for (int i = warp - 2; i < rows * num; i += 4) {
        const int t = i / num, kb = i - t * num;
        const uint32_t top = s_top[t];
        const int e = FORM == FP4_NV ? row_exponent(top) : 0;
        const Raw8<T> r = fetch(t, kb0 + kb);
        uint32_t code;
        const uint32_t codes = fp4_codes8<T, FORM>(r, r.largest(), pow2(e), pow2(-e), top >= 0x7f800000u, code);
        *reinterpret_cast<uint32_t*>(own_codes + kb * 1024 + t * 128 + (((lane >> 2) ^ t) << 4) + (lane & 3) * 4) = codes;
        if (lane % PER == 0) own_scales[kb * Cfg::OWN_SF + lane / (4 * PER) * 128 + t * 16 + (lane / PER & 3)] = uint8_t(code);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");             // written by threads, read by the tensor core
      mbar_arrive(quantised);
    }
    if (first < last) {                       // row scales and bias of this thread's columns, fetched under the main loop
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        ws[j] = p.w.row_scale[g + j];
        wb[j] = p.bias && g + j < p.N ? bf2f(p.bias[g + j]) : 0.f;
        us[j] = p.pair ? p.w.row_scale[g + 64 + j] : 0.f;
        ub[j] = p.pair && p.bias ? bf2f(p.bias[g + 64 + j]) : 0.f;
      }
    }
    if (!mbar_wait_bounded(accum, 0, abort_flag, 4000000000ull)) fail(OGB_ERR_WAIT_MMA);
    asm volatile("bar.sync 1, 128;" ::: "memory");
    tc_fence_after();
  }
  __syncwarp();
  if (p.splits > 1) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");                            // of the arrival at the start
    if (!Cfg::APART) cluster_sync_all();                                                // nobody's stages are in use any more
  }
  if (warp >= 2 && *abort_flag == 0) {
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t at = smem_u32(sums);
#pragma unroll 1
    for (int c0 = 0; c0 < rows; c0 += 16) {
      uint32_t r[16];
      tmem_ld16(tmem + (uint32_t(quarter * 32) << 16) + c0, r);
      tmem_ld_wait();
      if (p.splits > 1) {
        int m = c0, o = c0 / per, l = c0 - o * per;                                       // token, its CTA and its place there
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (m < rows) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dsmem_addr(at + uint32_t((rank * per + l) * FP4_TILE + row) * 4, uint32_t(o))), "r"(r[j]) : "memory");
          ++m;
          if (++l == per) { l = 0; ++o; }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) sums[(c0 + j) * FP4_TILE + row] = __uint_as_float(r[j]);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  if (p.splits > 1) cluster_sync_all(); else __syncthreads();
  if (warp >= 2 && *abort_flag == 0) {
    const int col = n_tile * (p.pair ? 64 : 128) + seg;
    if (col < p.n_out) {
      for (int m = first + (p.pair ? et >> 3 : et >> 4); m < last; m += 128 / segs) {
        float scale;
        if constexpr (ROWS == FP4_GIVEN) scale = p.a.row_scale[m];
        else scale = s_top[m] >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : FORM == FP4_NV ? pow2(row_exponent(s_top[m])) : 1.f;
        float v[8], u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = u[j] = 0.f;
        for (int q = 0; q < p.splits; ++q) {
          const float4* l = reinterpret_cast<const float4*>(sums + (q * per + m - first) * FP4_TILE + seg);
          const float4 x = l[0], y = l[1];
          v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w; v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
          if (p.pair) {
            const float4 a = l[16], b = l[17];
            u[0] += a.x; u[1] += a.y; u[2] += a.z; u[3] += a.w; u[4] += b.x; u[5] += b.y; u[6] += b.z; u[7] += b.w;
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = fmaf(v[j], scale * ws[j], wb[j]);
        if (p.pair) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = fp4_silu(v[j]) * fmaf(u[j], scale * us[j], ub[j]);
        }
        fp4_store8(p, m, col, v);
      }
    }
  }
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, Cfg::COLS);
}

template <int BT, int FORM, int ROWS = FP4_GIVEN>
static int LaunchFew(Fp4LinearArgs p, int splits, cudaStream_t stream) {
  using Cfg = Fp4Cfg<BT, FORM, ROWS>;
  static bool configured[OGB_MAX_DEVICES] = {};
  if (!set_max_dyn_smem(linear_fp4_kernel<BT, FORM, ROWS>, Cfg::smem(Cfg::STAGES, FP4_OWN_PART), configured)) return -3;
  p.kb_per_split = (p.w.num_kb + splits - 1) / splits;
  p.splits = splits = (p.w.num_kb + p.kb_per_split - 1) / p.kb_per_split;
  p.stages = min(ROWS ? min(Cfg::STAGES, (Cfg::ROOM - Cfg::own(p.kb_per_split)) / Cfg::STAGE) : Cfg::STAGES, p.kb_per_split);       // no more shared memory than the CTA has k-blocks: the next kernel's CTAs find room
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(p.w.padded / FP4_TILE), 1u, unsigned(splits));
  cfg.blockDim = dim3(192);
  cfg.dynamicSmemBytes = Cfg::smem(p.stages, p.kb_per_split);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (p.pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (splits > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim = {1, 1, unsigned(splits)};
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, linear_fp4_kernel<BT, FORM, ROWS>, p) == cudaSuccess ? 0 : -4;
}

static int fp4_splits(int N, int num_kb, int sm_count) { return max(1, min(min(8, num_kb), 2 * sm_count / (fp4_padded(N) / FP4_TILE))); }

template <int FORM>
static int LaunchLinear(const Fp4LinearArgs& p, int sm_count, cudaStream_t stream) {
  const int T = p.a.rows, bt = T <= 16 ? 16 : T <= 32 ? 32 : 64;
  // (65 / 128 tokens, us with 128 token columns here, a form that was not kept, against pairs of SMs: 6144 x 4096 14.5 / 20.4 against 7.1 / 7.5, 28672 x 4096 14.5 / 17.6
  // against 12.2 / 13.7; only few weight tiles with a long k were faster here, and by 65 tokens only: 4096 x 14336 11.8 / 16.1 against 14.5 / 14.7)
  if (T > 64) return LaunchPairLinearFp4(p, FORM, sm_count, stream);
  const int splits = fp4_splits(p.N, p.w.num_kb, sm_count);
  if (p.x) return p.x_fp32 ? LaunchFew<16, FORM, FP4_FP32>(p, splits, stream) : LaunchFew<16, FORM, FP4_BF16>(p, splits, stream);
  if (bt == 16) return LaunchFew<16, FORM>(p, splits, stream);
  if (bt == 32) return LaunchFew<32, FORM>(p, splits, stream);
  return LaunchFew<64, FORM>(p, splits, stream);
}

}  // namespace ogb

using namespace ogb;

// Whether the product quantises its rows itself: one or two of them, where all CTAs run at once and each has few k-blocks to look through for the rows' largest
// magnitudes and to turn (us, against a kernel for the rows in front, which costs a launch more: 1 x 4096 -> 6144 7.5 / 9.9, 2 rows 8.5 / 9.9, 4 rows 10.7 / 10.1, 8 x 1024
// 6.4 / 5.2; 1 x 4096 -> 4096 6.0 / 6.6; 1 x 14336 -> 4096 11.8 / 10.5; 1 x 4096 -> 128256, in waves, 53.5 / 48.8).
OGB_API int ogb_linear_fp4_own_rows(int T, int N, int K, int sm_count) {
  if (T < 1 || T > FP4_OWN_ROWS || N < 1 || K < 1) return 0;
  const int kbs = (K - 1) / FP4_KB + 1, splits = fp4_splits(N, kbs, sm_count), part = (kbs + splits - 1) / splits;
  return splits > 1 && part <= FP4_OWN_PART && T * (kbs + part) <= FP4_OWN_WORK;
}

OGB_API int ogb_linear_fp4(const void* x, long long ldx, int x_fp32, void* a_data, int T, const void* w_data, int N, int K, int form, void* out, long long ldc,
                           int out_fp32, int pair, const void* bias, const void* residual, long long ldr, int res_fp32, int* status, int sm_count, void* stream) {
  if (!w_data || T < 0 || (T > 0 && ((!a_data && !x) || !out)) || N <= 0 || K <= 0 || (form != FP4_NV && form != FP4_MX) || K % fp4_block(form)) return -1;
  if ((reinterpret_cast<uintptr_t>(a_data) | reinterpret_cast<uintptr_t>(w_data)) & 15) return -1;
  if (pair && (N % 128 || residual)) return -1;
  if (T == 0) return 0;
  const bool own = x && !a_data;
  if (own && !ogb_linear_fp4_own_rows(T, N, K, sm_count)) return -1;
  if (x && !own) {
    const int rc = ogb_quantize_fp4(x, ldx, x_fp32, T, K, form, a_data, stream);
    if (rc) return rc;
  }
  static const int pdl = [] { const char* e = getenv("OGB_PDL"); return (e && e[0] == '0') ? 0 : 1; }();
  Fp4LinearArgs p = {};
  p.a = fp4_view(a_data, T, K, form);
  if (own) {
    p.x = x;
    p.ldx = ldx;
    p.x_fp32 = x_fp32;
    p.x_vec = ((reinterpret_cast<uintptr_t>(x) | uintptr_t(ldx * (x_fp32 ? 4 : 2))) & 15) == 0;
  }
  p.K = K;
  p.w = fp4_view(const_cast<void*>(w_data), N, K, form);
  p.N = N;
  p.n_out = pair ? N / 2 : N;
  p.C = out;
  p.ldc = ldc;
  p.out_fp32 = out_fp32;
  p.pair = pair;
  p.bias = static_cast<const __nv_bfloat16*>(bias);
  p.residual = residual;
  p.ldr = ldr;
  p.res_fp32 = res_fp32;
  p.whole = ((reinterpret_cast<uintptr_t>(out) | uintptr_t(ldc * (out_fp32 ? 4 : 2))) & 15) == 0 &&
            (!residual || ((reinterpret_cast<uintptr_t>(residual) | uintptr_t(ldr * (res_fp32 ? 4 : 2))) & 15) == 0);
  p.status = status;
  p.pdl = pdl;
  p.early = x && !own;         // the quantisation in front has waited for everything before it, and writes only the rows
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return form == FP4_NV ? LaunchLinear<FP4_NV>(p, sm_count, s) : LaunchLinear<FP4_MX>(p, sm_count, s);
}
