// Products of up to 32 rows of 16-bit x with many microscaled 4-bit weights, as an output head's (gfx950,
// wave64): y = x W^T, and the score of given outputs (see q4d_mx_gemm.hip).
//
// x lies in LDS as the matrix instruction's operands, made once a block; a wave streams units of 16 NT
// weight rows through registers, kAhead tile columns ahead (1 KB a unit), and needs no other wave until its
// end.  The operands and their order are those of q4d_mx_rows.hip.  A score's waves keep the softmax's
// sums of their outputs, so that a block leaves one set a row.
// Bound by the weight stream and by the vector units, which make 16-bit floats of it (41 % busy): 21 rows of 151936 x
// 1024, 83 MB, 20-21.6 us, 4 TB/s (36 us on the kernel of few rows, which loads x for every weight tile).
#include <math.h>

#include <algorithm>

#include "q4d_mx.h"
#include "q4d_mx_dev.h"

namespace q4d {
namespace {

constexpr int kAhead = 3;
constexpr int kHeadLds = 128 << 10;  // x's operands at most
constexpr int kHeadBlocks = 256;     // one a CU
constexpr int kWavesLeast = 8, kWavesMost = 16;

template <bool BF>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <bool BF, int MT, int NT, bool SCORE>
__global__ __launch_bounds__(64 * kWavesMost) void mx_head_kernel(const MxProduct a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];  // [column tile][4 parts j][MT][64 lanes][16 bytes]
  const int t = threadIdx.x, lane = t & 63, r = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6), waves = blockDim.x >> 6;
  const int steps = mx_col_tiles(a.K), units = (a.N + 16 * NT - 1) / (16 * NT), stride = gridDim.x * waves;

  struct Step {
    u32x4 w[NT];
    uint32_t s[NT];
  } ring[kAhead];
  // The wave's steps in order: (unit, column tile); `ahead` names the next to load.
  int unit = blockIdx.x * waves + w, ahead_unit = unit, ahead = 0;
  const auto load = [&](Step& s) {
    const int u = min(ahead_unit, units - 1), half = NT == 1 ? u & 1 : 0;  // (past the last: not used)
    const size_t at = (size_t)(NT == 1 ? u >> 1 : u) * steps + ahead;
    const uint8_t* p = a.w + at * kMxTile + g * (kMxRows * 16) + (16 * half + r) * 16;
    const uint8_t* q = a.ws + at * kMxScales + 4 * (16 * half + r) + g;
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      s.w[k] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + 256 * k));
      s.s[k] = q[64 * k];
    }
    if (++ahead == steps) {
      ahead = 0;
      ahead_unit += stride;
    }
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u) load(ring[u]);

  for (int c = t; c < steps * 16 * (16 * MT); c += blockDim.x) {  // 16-byte groups of x, along its rows
    const int m = c / (steps * 16), k = c - m * (steps * 16);
    u32x4 v = {0u, 0u, 0u, 0u};
    if (m < a.M && 8 * k < a.K) v = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.x) + m * a.x_stride + 8 * k);
    // column tile k / 16, block k / 4 % 4 (the lanes' g), part k % 4
    *reinterpret_cast<u32x4*>(lds + (((k >> 4) * 4 + (k & 3)) * MT + (m >> 4)) * 1024 + ((k >> 2 & 3) * 16 + (m & 15)) * 16) = v;
  }
  __syncthreads();

  f32x4 acc[NT][MT];
  const auto clear = [&]() {
#pragma unroll
    for (int k = 0; k < NT; ++k)
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
  // lane (r, g) holds outputs 16 (NT unit + k) + 4 g .. + 3 of x's row 16 i + r
  const auto finish = [&]() {
    const int n0 = 16 * NT * unit + 4 * g;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if constexpr (!SCORE) {
#pragma unroll
        for (int k = 0; k < NT; ++k)
          if (16 * i + r < a.M && n0 + 16 * k < a.N) store_out4(a, 16 * i + r, n0 + 16 * k, acc[k][i]);
      } else {
        float z[4 * NT], top = -INFINITY;
        const int hit = target[i] - n0;  // 16 k + e of the lane's
#pragma unroll
        for (int c = 0; c < 4 * NT; ++c) {
          const int n = 16 * (c >> 2) + (c & 3);
          if (hit == n && n0 + n < a.N) a.hit[16 * i + r] = acc[c >> 2][i][c & 3];
          z[c] = n0 + n < a.N ? acc[c >> 2][i][c & 3] : -INFINITY;
          top = fmaxf(top, z[c]);
        }
        sums[i] = soft_join(sums[i], soft_sum<4 * NT>(top, [&](int c) { return z[c]; }));
      }
    }
  };

  clear();
  int step = 0;
  while (unit < units) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (unit >= units) break;
      const char* x = lds + step * (4 * MT * 1024) + 16 * lane;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x4 v[NT];
#pragma unroll
        for (int k = 0; k < NT; ++k) v[k] = mx_dequant8<BF>(ring[u].w[k][j], mx_scale(ring[u].s[k]));
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const u32x4 xv = *reinterpret_cast<const u32x4*>(x + (j * MT + i) * 1024);
#pragma unroll
          for (int k = 0; k < NT; ++k) acc[k][i] = mfma16<BF>(v[k], xv, acc[k][i]);
        }
      }
      load(ring[u]);
      if (++step == steps) {
        finish();
        clear();
        step = 0;
        unit += stride;
      }
    }
  }

  if constexpr (SCORE) {
    __syncthreads();  // everybody is done with x
    float* s_stat = reinterpret_cast<float*>(lds);  // [waves][16 MT][3]
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
      for (int v = 1; v < waves; ++v) {
        const float* at = s_stat + (v * 16 * MT + t) * 3;
        s = soft_join(s, SoftSum{at[0], at[1], at[2]});
      }
      a.stats[(size_t)t * gridDim.x + blockIdx.x] = f32x4{s.m, s.l, s.t, 0.f};
    }
  }
}

constexpr int kUnit = 2;  // NT
size_t lds_bytes(int M, int K) { return (size_t)mx_col_tiles(K) * 4 * (M <= 16 ? 1 : 2) * 1024; }
struct Shape {
  int blocks, waves;
};
// One block a CU, of as many waves as leave the fewest places without a unit in the last round (an LM head of 151936
// rows: 10 waves have two rounds, 93 % full; 8 would have three, 77 %).
Shape head_shape(int N) {
  const int units = (int)((N + 16LL * kUnit - 1) / (16 * kUnit));
  const int blocks = std::min(kHeadBlocks, (units + kWavesLeast - 1) / kWavesLeast), each = (units + blocks - 1) / blocks;
  int best = kWavesLeast;
  for (int w = kWavesLeast; w <= kWavesMost; ++w)
    if ((each + w - 1) / w * w < (each + best - 1) / best * best) best = w;
  return {blocks, best};
}

template <bool BF, bool SCORE>
int launch(const MxProduct& p, hipStream_t st) {
  const Shape s = head_shape(p.N);
  const dim3 grid(s.blocks), block(64 * s.waves);
  const size_t bytes = lds_bytes(p.M, p.K);
  if (p.M <= 16) hipLaunchKernelGGL((mx_head_kernel<BF, 1, kUnit, SCORE>), grid, block, bytes, st, p);
  else hipLaunchKernelGGL((mx_head_kernel<BF, 2, kUnit, SCORE>), grid, block, bytes, st, p);
  return check_launch();
}

}  // namespace

bool mx_head_fits(int M, int K) { return M <= 32 && lds_bytes(M, K) <= (size_t)kHeadLds; }
MxForm mx_head_form(int M, int N) { return {MX_HEAD, M <= 16 ? 1 : 2, kUnit, head_shape(N).waves}; }
int mx_head_parts(int N) { return head_shape(N).blocks; }
int launch_mx_head(const MxProduct& p, MxKind kind, hipStream_t st) {
  return kind == MX_BF16 ? launch<true, false>(p, st) : launch<false, false>(p, st);
}
int launch_mx_head_score(const MxProduct& p, MxKind kind, hipStream_t st) {
  return kind == MX_BF16 ? launch<true, true>(p, st) : launch<false, true>(p, st);
}

}  // namespace q4d
