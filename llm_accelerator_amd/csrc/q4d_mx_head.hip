// Products of up to 64 rows of 16-bit x with many microscaled 4-bit weights, as an output head's (gfx950,
// wave64): y = x W^T, and the score of given outputs (see q4d_mx_gemm.hip).
//
// x lies in LDS as the matrix instruction's operands, made once a block; a wave streams tiles of 32
// weight rows through registers, kAhead tile columns ahead (2 KB each), and needs no other wave until its
// end.  The operands and their order are those of q4d_mx_rows.hip.  A score's waves keep the softmax's
// sums of their outputs, so that a block leaves one set a row.
// Bound by the weight stream.
#include <math.h>

#include <algorithm>

#include "q4d_mx.h"
#include "q4d_mx_dev.h"

namespace q4d {
namespace {

constexpr int kAhead = 8;
constexpr int kHeadLds = 128 << 10;  // x's operands at most
constexpr int kHeadBlocks = 256;     // one or two a CU

template <bool BF>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <bool BF, int MT, int NW, bool SCORE>
__global__ __launch_bounds__(64 * NW) void mx_head_kernel(const MxProduct a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];  // [column tile][4 parts j][MT][64 lanes][16 bytes]
  const int t = threadIdx.x, lane = t & 63, r = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int steps = mx_col_tiles(a.K), tiles = mx_row_tiles(a.N), stride = gridDim.x * NW;

  struct Step {
    u32x4 w[2];
    uint32_t s[2];
  } ring[kAhead];
  // The wave's steps in order: (tile, column tile); `ahead` names the next to load.
  int tile = blockIdx.x * NW + w, ahead_tile = tile, ahead = 0;
  const auto load = [&](Step& s) {
    const size_t at = (size_t)min(ahead_tile, tiles - 1) * steps + ahead;  // (past the last: not used)
    const uint8_t* p = a.w + at * kMxTile + g * (kMxRows * 16) + r * 16;
    const uint8_t* q = a.ws + at * kMxScales + 4 * r + g;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      s.w[k] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + 256 * k));
      s.s[k] = q[64 * k];
    }
    if (++ahead == steps) {
      ahead = 0;
      ahead_tile += stride;
    }
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u) load(ring[u]);

  for (int c = t; c < steps * 16 * (16 * MT); c += 64 * NW) {  // 16-byte groups of x, along its rows
    const int m = c / (steps * 16), k = c - m * (steps * 16);
    u32x4 v = {0u, 0u, 0u, 0u};
    if (m < a.M && 8 * k < a.K) v = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.x) + m * a.x_stride + 8 * k);
    // column tile k / 16, block k / 4 % 4 (the lanes' g), part k % 4
    *reinterpret_cast<u32x4*>(lds + (((k >> 4) * 4 + (k & 3)) * MT + (m >> 4)) * 1024 + ((k >> 2 & 3) * 16 + (m & 15)) * 16) = v;
  }
  __syncthreads();

  f32x4 acc[2][MT];
  const auto clear = [&]() {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[k][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  };
  SoftSum sums[MT];
  int target[MT];
  if constexpr (SCORE) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      sums[i] = SoftSum{-INFINITY, 0.f, 0.f};
      target[i] = 16 * i + r < a.M ? a.targets[16 * i + r] : -1;
    }
  }
  // lane (r, g) holds outputs 32 tile + 16 k + 4 g .. + 3 of x's row 16 i + r
  const auto finish = [&]() {
    const int n0 = kMxRows * tile + 4 * g;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if constexpr (!SCORE) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (16 * i + r < a.M && n0 + 16 * k < a.N) store_out4(a, 16 * i + r, n0 + 16 * k, acc[k][i]);
      } else {
        float z[8], top = -INFINITY;
        const int hit = target[i] - n0;  // 16 k + e of the lane's
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const int n = 16 * (c >> 2) + (c & 3);
          if (hit == n && n0 + n < a.N) a.hit[16 * i + r] = acc[c >> 2][i][c & 3];
          z[c] = n0 + n < a.N ? acc[c >> 2][i][c & 3] : -INFINITY;
          top = fmaxf(top, z[c]);
        }
        sums[i] = soft_join(sums[i], soft_sum<8>(top, [&](int c) { return z[c]; }));
      }
    }
  };

  clear();
  int step = 0;
  while (tile < tiles) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (tile >= tiles) break;
      const char* x = lds + step * (4 * MT * 1024) + 16 * lane;
      const float f0 = mx_scale(ring[u].s[0]), f1 = mx_scale(ring[u].s[1]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u32x4 v0 = mx_dequant8<BF>(ring[u].w[0][j], f0), v1 = mx_dequant8<BF>(ring[u].w[1][j], f1);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const u32x4 xv = *reinterpret_cast<const u32x4*>(x + (j * MT + i) * 1024);
          acc[0][i] = mfma16<BF>(v0, xv, acc[0][i]);
          acc[1][i] = mfma16<BF>(v1, xv, acc[1][i]);
        }
      }
      load(ring[u]);
      if (++step == steps) {
        finish();
        clear();
        step = 0;
        tile += stride;
      }
    }
  }

  if constexpr (SCORE) {
    __syncthreads();  // everybody is done with x
    float* s_stat = reinterpret_cast<float*>(lds);  // [NW][16 MT][3]
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      SoftSum s = sums[i];
#pragma unroll
      for (int v = 16; v <= 32; v *= 2) s = soft_join(s, SoftSum{__shfl_xor(s.m, v), __shfl_xor(s.l, v), __shfl_xor(s.t, v)});
      if (g == 0) {
        float* at = s_stat + (w * 16 * MT + 16 * i + r) * 3;
        at[0] = s.m;
        at[1] = s.l;
        at[2] = s.t;
      }
    }
    __syncthreads();
    if (t < 16 * MT && t < a.M) {
      SoftSum s = {s_stat[t * 3], s_stat[t * 3 + 1], s_stat[t * 3 + 2]};
#pragma unroll
      for (int v = 1; v < NW; ++v) {
        const float* at = s_stat + (v * 16 * MT + t) * 3;
        s = soft_join(s, SoftSum{at[0], at[1], at[2]});
      }
      a.stats[(size_t)t * gridDim.x + blockIdx.x] = f32x4{s.m, s.l, s.t, 0.f};
    }
  }
}

int row_tiles16(int M) { return M <= 16 ? 1 : M <= 32 ? 2 : 4; }
size_t lds_bytes(int M, int K) { return (size_t)mx_col_tiles(K) * 4 * row_tiles16(M) * 1024; }
// Waves of a block, and blocks: as many as fit, but no wave without a tile.
constexpr int kWaves = 4, kWavesMost = 8;
int head_waves(int M) { return row_tiles16(M) == 4 ? kWavesMost : kWaves; }
int head_blocks(int M, int N, int K) {
  const int waves = head_waves(M), fit = lds_bytes(M, K) <= 72 << 10 ? 2 : 1;
  return std::max(1, std::min(kHeadBlocks * fit, (mx_row_tiles(N) + waves - 1) / waves));
}

template <bool BF, bool SCORE>
int launch(const MxProduct& p, hipStream_t st) {
  const dim3 grid((unsigned)head_blocks(p.M, p.N, p.K));
  const size_t bytes = lds_bytes(p.M, p.K);
  switch (row_tiles16(p.M)) {
    case 1: hipLaunchKernelGGL((mx_head_kernel<BF, 1, kWaves, SCORE>), grid, dim3(64 * kWaves), bytes, st, p); break;
    case 2: hipLaunchKernelGGL((mx_head_kernel<BF, 2, kWaves, SCORE>), grid, dim3(64 * kWaves), bytes, st, p); break;
    default: hipLaunchKernelGGL((mx_head_kernel<BF, 4, kWavesMost, SCORE>), grid, dim3(64 * kWavesMost), bytes, st, p);
  }
  return check_launch();
}

}  // namespace

bool mx_head_fits(int M, int K) { return M <= 64 && lds_bytes(M, K) <= (size_t)kHeadLds; }
int mx_head_parts(int M, int N, int K) { return head_blocks(M, N, K); }
int launch_mx_head(const MxProduct& p, MxKind kind, hipStream_t st) {
  return kind == MX_BF16 ? launch<true, false>(p, st) : launch<false, false>(p, st);
}
int launch_mx_head_score(const MxProduct& p, MxKind kind, hipStream_t st) {
  return kind == MX_BF16 ? launch<true, true>(p, st) : launch<false, true>(p, st);
}

}  // namespace q4d
