// Products of a few rows with microscaled 4-bit weights (gfx950, wave64): y = x W^T.
//
// A block takes 16 weight rows and up to 16 MT rows of x; its waves share K, 128 columns at a time: lane
// (r, g) loads the 16 bytes of weight row r's block g and the 32 values of x's row r there.  The
// order of K inside a product is free, so that both operands go to the matrix unit as they were loaded:
// four 16x16x32 products of 8 columns a lane after the codes are made 16-bit floats, or with x in 4 bits
// one 16x16x128 product that takes codes and scales as they are.  The waves' sums meet in LDS.
#include "q4d_mx.h"
#include "q4d_mx_dev.h"

namespace q4d {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kRowTile = 16;  // weight rows of a block

template <bool BF>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ i32x8 codes_operand(u32x4 v) {
  return i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
}

template <MxKind KIND, int MT, int NW>
__global__ __launch_bounds__(64 * NW) void mx_rows_kernel(const MxProduct a) {
  __shared__ f32x4 part[NW][MT][64];
  const int t = threadIdx.x, lane = t & 63, r = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int n0 = blockIdx.x * kRowTile, m0 = blockIdx.y * (16 * MT);
  const int blocks = a.K / 32, steps = mx_col_tiles(a.K);
  const size_t at = (size_t)(n0 / kMxRows) * steps;  // first tile
  const uint8_t* wp = a.w + at * kMxTile + g * (kMxRows * 16) + (n0 % kMxRows + r) * 16;
  const uint8_t* sp = a.ws + at * kMxScales + 4 * (n0 % kMxRows + r) + g;
  const u32x4 none = {0u, 0u, 0u, 0u};

  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int it = w; it < steps; it += NW) {
    const u32x4 wq = *reinterpret_cast<const u32x4*>(wp + (size_t)it * kMxTile);
    const uint32_t ws = sp[(size_t)it * kMxScales];
    if constexpr (KIND == MX_X4) {
      u32x4 x[MT];
      uint32_t xs[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        // (16-row halves of tiles that are there: rows past the last go to outputs that are not stored)
        const int m = min(m0 + 16 * i, (a.M - 1) & ~15);
        const size_t tile = (size_t)(m / kMxRows) * steps + it;
        x[i] = *reinterpret_cast<const u32x4*>(static_cast<const uint8_t*>(a.x) + tile * kMxTile + g * (kMxRows * 16) + (m % kMxRows + r) * 16);
        xs[i] = a.xs[tile * kMxScales + 4 * (m % kMxRows + r) + g];
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
        acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(codes_operand(wq), codes_operand(x[i]), acc[i], 4, 4, 0,
                                                                  (int)ws, 0, (int)xs[i]);
    } else {
      const int b = 4 * it + g;
      u32x4 x[MT][4];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int m = m0 + 16 * i + r;
        const bool have = b < blocks && m < a.M;
        const uint16_t* xp = static_cast<const uint16_t*>(a.x) + (have ? m * a.x_stride + 32 * b : 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[i][j] = have ? *reinterpret_cast<const u32x4*>(xp + 8 * j) : none;
      }
      const float f = mx_scale(ws);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u32x4 v = mx_dequant8<KIND == MX_BF16>(wq[j], f);
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i] = mfma16<KIND == MX_BF16>(v, x[i][j], acc[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) part[w][i][lane] = acc[i];
  __syncthreads();
  // lane (r, g) of row tile i: outputs 4 g .. + 3 of x's row 16 i + r
  for (int i = w; i < MT; i += NW) {
    f32x4 s = part[0][i][lane];
#pragma unroll
    for (int k = 1; k < NW; ++k) {
      const f32x4 v = part[k][i][lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += v[e];
    }
    const int m = m0 + 16 * i + r, at = n0 + 4 * g;
    if (m < a.M) store_out4(a, m, at, s);
  }
}

template <MxKind KIND, int MT>
int launch(const MxProduct& p, hipStream_t st) {
  const dim3 grid((unsigned)((p.N + kRowTile - 1) / kRowTile), (unsigned)((p.M + 16 * MT - 1) / (16 * MT)));
  if (grid.y > 65535u) return Q4D_ERR_SHAPE;
  hipLaunchKernelGGL((mx_rows_kernel<KIND, MT, 4>), grid, dim3(256), 0, st, p);
  return check_launch();
}
template <MxKind KIND>
int launch(const MxProduct& p, hipStream_t st) {
  if (p.M <= 16) return launch<KIND, 1>(p, st);
  if (p.M <= 32) return launch<KIND, 2>(p, st);
  return launch<KIND, 4>(p, st);
}

}  // namespace

int launch_mx_rows(const MxProduct& p, MxKind kind, hipStream_t st) {
  if (kind == MX_X4) return launch<MX_X4>(p, st);
  return kind == MX_BF16 ? launch<MX_BF16>(p, st) : launch<MX_F16>(p, st);
}

}  // namespace q4d
