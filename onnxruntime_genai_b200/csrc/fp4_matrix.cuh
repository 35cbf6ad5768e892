// Rows of 4-bit floating-point numbers (e2m1) in blocks with a scale each, laid out as the block-scaled tensor-core product reads them.
//
//   nvfp4: blocks of 16 along K, scale e4m3;  mxfp4: blocks of 32, scale a power of two (e8m0).  Both: one fp32 scale per row.
//   value[r, k] = row_scale[r] * scale[r, k / block] * e2m1(code[r, k])
//
// One buffer: codes, block scales, row scales.  Rows are padded to whole tiles of 128, K to whole k-blocks of 256 (codes and scales of 0).
//   codes       [k-block][row / 8][8 rows x 128 bytes]: a row's 256 codes of a k-block, two to a byte (the even k in the low half), in eight
//               chunks of 16 bytes, chunk c of row r at place c ^ (r % 8).  This is the shared-memory image of a K-major operand with the
//               128-byte swizzle, so any multiple of eight rows of a k-block is one contiguous copy without a tensor map.
//   scales      [k-block][row / 128][step][512 bytes]: a step is what four scales of a row cover (nvfp4: the K of one tensor-core instruction,
//               mxfp4: of two); scale b of row r at byte (r % 32) * 16 + (r % 128) / 32 * 4 + b, the order in which 32 rows of 16 bytes become
//               four columns of tensor memory.
//   row scales  [rows padded]
#pragma once
#include "common.cuh"

namespace ogb {

enum Fp4Form : int { FP4_NV = 0, FP4_MX = 1 };

constexpr int FP4_KB = 256;                                  // k values of a k-block: a row's 128 bytes
constexpr int FP4_SCALE_STEP = 512;                          // bytes of a scale step of 128 rows
__host__ __device__ constexpr int fp4_block(int form) { return form == FP4_NV ? 16 : 32; }
__host__ __device__ constexpr int fp4_steps(int form) { return form == FP4_NV ? 4 : 2; }   // scale steps of a k-block

struct Fp4View {
  uint8_t* codes;
  uint8_t* scales;
  float* row_scale;
  int rows, padded, num_kb;     // rows, rows in whole tiles, k-blocks
};
__host__ __device__ inline int fp4_padded(int rows) { return (rows + 127) / 128 * 128; }
__host__ __device__ inline long long fp4_bytes(int rows, int K, int form) {
  const long long padded = fp4_padded(rows), kb = (K + FP4_KB - 1) / FP4_KB;
  return padded * (kb * (FP4_KB / 2 + fp4_steps(form) * 4) + 4);
}
__host__ __device__ inline Fp4View fp4_view(void* data, int rows, int K, int form) {
  Fp4View v;
  v.rows = rows;
  v.padded = fp4_padded(rows);
  v.num_kb = (K + FP4_KB - 1) / FP4_KB;
  v.codes = static_cast<uint8_t*>(data);
  v.scales = v.codes + (long long)v.num_kb * v.padded * (FP4_KB / 2);
  v.row_scale = reinterpret_cast<float*>(v.scales + (long long)v.num_kb * v.padded * (fp4_steps(form) * 4));
  return v;
}
// byte of row r's 16-byte chunk c (32 codes) of k-block kb
__host__ __device__ inline long long fp4_code_at(const Fp4View& v, int kb, int r, int c) {
  return ((long long)kb * v.padded + r) * 128 + ((c ^ (r & 7)) << 4);
}
// byte of row r's scale b (0..3) of a step of k-block kb
__host__ __device__ inline long long fp4_scale_at(const Fp4View& v, int form, int kb, int r, int step, int b) {
  return (((long long)kb * (v.padded >> 7) + (r >> 7)) * fp4_steps(form) + step) * FP4_SCALE_STEP + (r & 31) * 16 + ((r & 127) >> 5) * 4 + b;
}

__device__ __forceinline__ float reciprocal(float v) {      // within a last place or two, of a normal number
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Codes to numbers, by their fields.
__device__ __forceinline__ float fp4_value(uint32_t code) {     // e2m1
  const uint32_t m = code & 7u;
  const float a = m < 2u ? 0.5f * float(m) : __uint_as_float(((126u + (m >> 1)) << 23) | ((m & 1u) << 22));
  return (code & 8u) ? -a : a;
}
__device__ __forceinline__ float fp4_scale_nv(uint32_t s) {     // e4m3, no sign
  const uint32_t e = (s >> 3) & 15u, m = s & 7u;
  return e == 0u ? float(m) * 0.001953125f : __uint_as_float(((e + 120u) << 23) | (m << 20));
}
__device__ __forceinline__ float fp4_scale_mx(uint32_t s) {     // e8m0
  return s == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(s << 23);
}
__device__ __forceinline__ float fp4_scale(int form, uint32_t s) { return form == FP4_NV ? fp4_scale_nv(s) : fp4_scale_mx(s); }

}  // namespace ogb
