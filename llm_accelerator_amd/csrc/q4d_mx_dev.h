// Microscaled 4-bit floats (gfx950): a row of K values is K / 32 blocks; a block is 32 codes of
// sign, 2 exponent bits and 1 mantissa bit (0, 0.5, 1, 1.5, 2, 3, 4, 6) and one scale byte s that
// stands for 2^(s - 127), 255 for NaN.  Codes lie two a byte, the even column in the low nibble;
// 16 bytes are one block.
//
// In memory a matrix is tiles of 32 rows x 128 columns, those of 32 rows side by side: codes
// [4 blocks][32 rows][16 bytes], scales [32 rows][4 blocks].  What a wave loads for a matrix
// instruction, 64 blocks of 16 or 32 rows, is then 1 KB in one or four pieces (row by row it was 32
// pieces of 32 bytes: 4096 x 8192 x 4096 in 4 bits took 214 us, all of it waiting).  Rows and columns past the
// matrix's are there: columns as zeros, rows as anything.
#pragma once

#include <math.h>

#include "q4d_device.h"
#include "q4d_mx.h"

namespace q4d {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kMxRows = 32, kMxCols = 128;              // of a tile
constexpr int kMxTile = kMxRows * kMxCols / 2;          // bytes of its codes
constexpr int kMxScales = kMxRows * kMxCols / 32;       // ... and of its scales

__host__ __device__ inline int mx_col_tiles(int cols) { return (cols + kMxCols - 1) / kMxCols; }
__host__ __device__ inline int mx_row_tiles(int rows) { return (rows + kMxRows - 1) / kMxRows; }

// A scale byte as the conversions take it: they read the exponent field alone, 0 as 2^-127 and 255 as NaN.
__device__ __forceinline__ float mx_scale(uint32_t s) { return __builtin_bit_cast(float, s << 23); }

// Two codes (byte SEL of w) as fp32, and as a pair of 16-bit floats: one instruction each, exact but where
// the type cannot hold the value (fp16: blocks of scales outside 2^-23 .. 2^13, rounded or Inf).
template <int SEL, bool BF>
__device__ __forceinline__ uint32_t mx_pair(uint32_t w, float scale) {
  if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, SEL));
}
// Eight codes (columns 8 j .. + 7 of a block are its word j) as 16-bit floats.
template <bool BF>
__device__ __forceinline__ u32x4 mx_dequant8(uint32_t w, float scale) {
  return u32x4{mx_pair<0, BF>(w, scale), mx_pair<1, BF>(w, scale), mx_pair<2, BF>(w, scale), mx_pair<3, BF>(w, scale)};
}

// Sum / maximum of a wave, in every lane: in the 16-lane rows by DPP, then over the rows by lane swaps (shuffles
// through LDS would be a few hundred clocks of a chain).
// No addition takes in the product that v may be: fused, it would be rounded for the other lane and not for the own,
// and the lanes would hold sums a rounding apart.
template <bool SUM>
__device__ __forceinline__ float wave_all(float v) {
  const auto op = [](float a, float b) {
#pragma clang fp contract(off)
    return SUM ? a + b : fmaxf(a, b);
  };
  v = op(v, dpp_f<kDppQuadSwap1>(v));
  v = op(v, dpp_f<kDppQuadSwap2>(v));
  v = op(v, dpp_f<kDppRowHalfMirror>(v));
  v = op(v, dpp_f<kDppRowMirror>(v));
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  const uint32_t x = __builtin_bit_cast(uint32_t, op(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1)));
  const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return op(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}

// A softmax's sums over some logits z: the maximum m, l = sum e^(z - m) and t = sum (z - m) e^(z - m), from
// which log(sum e^z) = m + log l and the entropy log l - t / l.  fp32; a NaN among the logits makes l NaN,
// and where all are -Inf l is 0 (and the joined l NaN at the end, as the softmax is).
struct SoftSum {
  float m, l, t;
};
// e^d, d <= 0, by the hardware's 2^x (what would be subnormal is 0).
constexpr float kLog2e = 1.44269504f;
__device__ __forceinline__ float exp_neg(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }
// The sums of N logits given their maximum.
template <int N, class F>
__device__ __forceinline__ SoftSum soft_sum(float m, F z) {
  const float ms = m == -INFINITY ? 0.f : m;
  SoftSum s = {m, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = z(i) - ms, e = exp_neg(d);
    s.l += e;
    s.t = fmaf(fmaxf(d, -1000.f), e, s.t);  // (e is 0 long before; -Inf x 0 would be NaN)
  }
  return s;
}
__device__ __forceinline__ SoftSum soft_join(SoftSum a, SoftSum b) {
  const float m = fmaxf(a.m, b.m), ms = m == -INFINITY ? 0.f : m;
  const float da = a.m - ms, db = b.m - ms, fa = exp_neg(da), fb = exp_neg(db);
  return {m, fmaf(a.l, fa, b.l * fb),
          (fa > 0.f ? fa * fmaf(da, a.l, a.t) : 0.f) + (fb > 0.f ? fb * fmaf(db, b.l, b.t) : 0.f)};
}

// Of the lanes of a wave, in every lane.
__device__ __forceinline__ SoftSum soft_wave(SoftSum s) {
  const float m = wave_all<false>(s.m), d = s.m - (m == -INFINITY ? 0.f : m), f = exp_neg(d);
  return {m, wave_all<true>(s.l * f), wave_all<true>(f > 0.f ? f * fmaf(d, s.l, s.t) : 0.f)};
}

// Four outputs rounded once to a 16-bit type.
__device__ __forceinline__ u32x2 pack_out4(int dtype, f32x4 v) {
  uint32_t u[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    u[e] = dtype == Q4D_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)v[e]) : __builtin_bit_cast(uint16_t, (_Float16)v[e]);
  return u32x2{u[0] | u[1] << 16, u[2] | u[3] << 16};
}
// Outputs n .. n + 3 of row m, those below N, rounded once to the output's type.
__device__ __forceinline__ void store_out4(const MxProduct& a, int m, int n, f32x4 v) {
  const size_t at = (size_t)m * a.N + n;
  const bool whole = n + 4 <= a.N && a.N % 4 == 0;
  if (a.y_dtype == Q4D_F32) {
    float* y = static_cast<float*>(a.y) + at;
    if (whole) {
      *reinterpret_cast<f32x4*>(y) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < a.N) y[e] = v[e];
    }
    return;
  }
  const u32x2 u = pack_out4(a.y_dtype, v);
  uint16_t* y = static_cast<uint16_t*>(a.y) + at;
  if (whole) {
    *reinterpret_cast<u32x2*>(y) = u;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < a.N) y[e] = (uint16_t)(u[e / 2] >> (16 * (e & 1)));
  }
}

}  // namespace q4d
