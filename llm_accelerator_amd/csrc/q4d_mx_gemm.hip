// Products of many rows with microscaled 4-bit weights (gfx950, wave64): y = x W^T, and the score of
// given outputs, which keeps of each row's products only the sums of a softmax.
//
// A block takes 128 NT weight rows and 32 MT rows of x, a wave 32 NT weight rows and all of x's.  Both go to
// LDS by DMA, RING - 1 stages ahead (64 columns with x in 16 bits, 128 in 4).  Lane (r, h) takes row r's block
// 2 i + h, and since the order of K inside a product is free, its 32 columns are the lane's share of 64:
// with 16-bit x four 32x32x16 products of 8 columns a lane after the codes are made 16-bit floats, with x
// in 4 bits one 32x32x64 product that takes codes and scales as they are.
// The weights are the first operand, so that a lane holds outputs of one row of x.
//
// Bound by the matrix units and the clock that they leave (1.5 GHz): 2000 x 6144 x 1024 28 us, 0.90 PFLOP/s (units busy
// 56 %; one round of blocks), 8192 x 8192 x 8192 844 us, 1.30 PFLOP/s, a score of 1999 rows of 151936 x
// 1024 560 us, 1.11 PFLOP/s (68 %).  In 4 bits, where a stage is 16 products a wave, by the stages' start: 4096 x 8192
// x 4096 76 us, 3.6 PFLOP/s (units busy 52 %), waves wait 28 % of their time for the stage, for each other and for the first
// operands, which are read after the barrier.
#include <math.h>

#include <type_traits>

#include "q4d_mx.h"
#include "q4d_mx_dev.h"

namespace q4d {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kXcds = 8, kCus = 256;

template <bool BF>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ i32x8 codes_operand(u32x4 v) {
  return i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
}
// Blocks 2 I + h of a tile: its rows' scales were shifted by 8 h, so that byte 2 I serves.
template <int I>
__device__ __forceinline__ f32x16 mfma_codes(u32x4 a, uint32_t as, u32x4 b, uint32_t bs, f32x16 c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(codes_operand(a), codes_operand(b), c, 4, 4, 2 * I, (int)as, 2 * I, (int)bs);
}

// Lane i writes the 16 (or 4) bytes at base + offset to LDS address lds + 16 i (4 i); lds, base wave-uniform.
// Ordered by the kernel's own wait and barrier.
__device__ __forceinline__ void dma16(const void* base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ void dma4(const void* base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(offset), "s"(base)
               : "memory", "m0");
}

template <bool SUM>
__device__ __forceinline__ float halves(float v) {  // of lanes l and l ^ 32, in both
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  const float x0 = __builtin_bit_cast(float, a0), x1 = __builtin_bit_cast(float, a1);
  return SUM ? x0 + x1 : fmaxf(x0, x1);
}

// s_waitcnt vmcnt(N) lgkmcnt(0)
template <int N>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);
}

template <MxKind KIND, bool SCORE, int NT, int MT, int RING, int PER_CU>
__global__ __launch_bounds__(256, PER_CU) void mx_gemm_kernel(const MxProduct a) {
  constexpr bool X4 = KIND == MX_X4;
  constexpr int kTileN = 128 * NT, kTileM = 32 * MT;
  constexpr int kCols = X4 ? 128 : 64;                     // columns of a stage
  // bytes of a stage: x (16 bits: 128 a row; 4 bits: tiles), weights, their scales and x's, 256 a wave
  constexpr int kWaveX = kTileM * (X4 ? 64 : 128) / 4, kWaveW = NT * kMxTile * kCols / kMxCols;  // of a wave
  constexpr int kX = 4 * kWaveX, kW = 4 * kWaveW, kS = 1024;
  constexpr int kStage = kX + kW + kS * (X4 ? 2 : 1);
  constexpr int kLoads = (kWaveX + kWaveW) / 1024 + (X4 ? 2 : 1);  // DMA instructions of a wave and stage
  static_assert((MT == 2 || MT == 4) && RING >= 3 && RING <= 6 && kLoads * (RING - 2) < 64 && RING * kStage * PER_CU <= 160 << 10, "");
  static_assert(!SCORE || (NT == 2 && 4 * kTileM * 12 <= RING * kStage), "");
  __shared__ __attribute__((aligned(16))) char lds[RING * kStage];
  const int t = threadIdx.x, lane = t & 63, r = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  // Of a CU's two blocks one goes first, so that one's outputs leave beside the other's products (4096 x 8192 x 4096 76
  // instead of 79 us, 4096 x 8192 x 1024 32.3 / 33.7; in 16 bits, three a CU, 2000 x 16384 x 1024 68 instead of 65).
  if constexpr (X4 && MT == 4) {
    if (blockIdx.x / kCus & 1) __builtin_amdgcn_s_setprio(1);
  }
  const int tm = (a.M + kTileM - 1) / kTileM, tiles = gridDim.x;
  // an XCD takes consecutive tiles, those of one weight range after each other
  const int xcd = blockIdx.x % kXcds, per = tiles / kXcds, more = tiles % kXcds;
  const int tile = xcd * per + min(xcd, more) + blockIdx.x / kXcds;
  const int n0 = tile / tm * kTileN, m0 = tile % tm * kTileM;
  const int col_tiles = mx_col_tiles(a.K), stages = (a.K + kCols - 1) / kCols;

  // ---- to LDS ------------------------------------------------------------------------------------
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  // x in 16 bits: slot s of row i holds the row's 16-byte group s ^ (i / 2 & 7), so that 16 rows' same group
  // falls on all banks.  Tiles lie as they are.
  const size_t x_row = 2 * (size_t)a.x_stride;
  const char* xb = static_cast<const char*>(a.x) + (X4 ? 0 : m0 * x_row);
  const auto group = [&](int j) { return (lane & 7) ^ ((4 * j + (lane >> 4)) & 7); };
  uint32_t from[MT];
  if constexpr (!X4) {
#pragma unroll
    for (int j = 0; j < MT; ++j) from[j] = (uint32_t)(min(8 * (MT * w + j) + (lane >> 3), a.M - 1 - m0) * x_row) + 16 * group(MT * w + j);
  }
  const size_t x_tile = (size_t)min(m0 / kMxRows + w * MT / 4, (a.M - 1) / kMxRows) * col_tiles;  // this wave's first
  // the wave's tiles of weight rows (past the last: the last, not stored)
  const int w_tiles = mx_row_tiles(a.N), wt0 = min(n0 / kMxRows + NT * w, w_tiles - 1), wt1 = min(wt0 + NT - 1, w_tiles - 1);
  const uint8_t* const wp0 = a.w + (size_t)wt0 * col_tiles * kMxTile;
  const uint8_t* const wp1 = a.w + (size_t)wt1 * col_tiles * kMxTile;
  const uint8_t* const sp = a.ws + (size_t)wt0 * col_tiles * kMxScales;
  const uint32_t sfrom = 4 * r + h * (wt1 - wt0) * col_tiles * kMxScales;
  const auto issue = [&](int st, int at) {
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + at);
    if constexpr (X4) {
      const uint8_t* p = static_cast<const uint8_t*>(a.x) + (x_tile + st) * kMxTile + (MT == 2 ? 1024 * (w & 1) : 0);
#pragma unroll
      for (int j = 0; j < kWaveX / 1024; ++j) dma16(p, 16 * lane + 1024 * j, to + kWaveX * w + 1024 * j);
#pragma unroll
      for (int j = 0; j < 2 * NT; ++j)
        dma16((j < 2 ? wp0 : wp1) + (size_t)st * kMxTile, 16 * lane + 1024 * (j & 1), to + kX + kWaveW * w + 1024 * j);
      dma4(sp + (size_t)st * kMxScales, sfrom, to + kX + kW + 256 * w);
      dma4(a.xs + (x_tile + st) * kMxScales, 4 * r, to + kX + kW + kS + 256 * w);
    } else {
      const char* base = xb + (size_t)st * 128;
      const int have = a.K / 8 - 8 * st;  // groups left in the row
      if (have >= 8) {
#pragma unroll
        for (int j = 0; j < MT; ++j) dma16(base, from[j], to + kWaveX * w + 1024 * j);
      } else {  // groups past the row's end are zeros
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          u32x4 v = {0u, 0u, 0u, 0u};
          if (group(MT * w + j) < have) v = *reinterpret_cast<const u32x4*>(base + from[j]);
          *reinterpret_cast<u32x4*>(lds + at + kWaveX * w + 1024 * j + 16 * lane) = v;
        }
        // This stage, the last, has MT DMA loads fewer than the loop counts on: with those of all stages before it
        // complete here, the loop's waits for them are met whatever they count.
        wait_loads<0>();
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
        dma16((j ? wp1 : wp0) + (size_t)st * (kMxTile / 2), 16 * lane, to + kX + kWaveW * w + 1024 * j);
      dma4(sp + (size_t)(st / 2) * kMxScales, sfrom, to + kX + kW + 256 * w);
    }
  };

  f32x16 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

#pragma unroll
  for (int c = 0; c < RING - 1; ++c)
    if (c < stages) issue(c, c * kStage);
  int at = 0, ahead = (RING - 1) * kStage;  // of this stage in the ring, and of the one to load next
  for (int st = 0; st < stages; ++st) {
    // this wave's part of the stage is there (the loads of later ones may be under way), then everybody's,
    // and the stage before is read
    const int later = min(stages - 1 - st, RING - 2);
    if (later >= 4) wait_loads<4 * kLoads>();
    else if (later == 3) wait_loads<3 * kLoads>();
    else if (later == 2) wait_loads<2 * kLoads>();
    else if (later == 1) wait_loads<kLoads>();
    else wait_loads<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (st + RING - 1 < stages) issue(st + RING - 1, ahead);
    const char* stage = lds + at;
    if constexpr (X4) {
      uint32_t xs[MT], ws[NT];
#pragma unroll
      for (int j = 0; j < MT; ++j) xs[j] = *reinterpret_cast<const uint32_t*>(stage + kX + kW + kS + 256 * (j * 4 / MT) + 4 * r) >> (8 * h);
#pragma unroll
      for (int k = 0; k < NT; ++k) ws[k] = *reinterpret_cast<const uint32_t*>(stage + kX + kW + 256 * w + 128 * k + 4 * r) >> (8 * h);
      const auto step = [&](auto i_) {
        constexpr int I = decltype(i_)::value;
        u32x4 q[NT];
#pragma unroll
        for (int k = 0; k < NT; ++k) q[k] = *reinterpret_cast<const u32x4*>(stage + kX + kWaveW * w + 2048 * k + 1024 * I + 16 * lane);
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(stage + 2048 * j + 1024 * I + 16 * lane);
#pragma unroll
          for (int k = 0; k < NT; ++k) acc[k][j] = mfma_codes<I>(q[k], ws[k], x, xs[j], acc[k][j]);
        }
      };
      step(std::integral_constant<int, 0>());
      step(std::integral_constant<int, 1>());
    } else {
      u32x4 q[NT];
      float f[NT];
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        q[k] = *reinterpret_cast<const u32x4*>(stage + kX + kWaveW * w + 1024 * k + 16 * lane);
        f[k] = mx_scale(*reinterpret_cast<const uint32_t*>(stage + kX + kW + 256 * w + 128 * k + 4 * r) >> (16 * (st & 1) + 8 * h) & 255u);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u32x4 wd[NT];
#pragma unroll
        for (int k = 0; k < NT; ++k) wd[k] = mx_dequant8<KIND == MX_BF16>(q[k][i], f[k]);
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(stage + 128 * r + 4096 * j + (((4 * h + i) ^ (r >> 1 & 7)) << 4));
#pragma unroll
          for (int k = 0; k < NT; ++k) acc[k][j] = mfma32<KIND == MX_BF16>(wd[k], x, acc[k][j]);
        }
      }
    }
    at = at == (RING - 1) * kStage ? 0 : at + kStage;
    ahead = ahead == (RING - 1) * kStage ? 0 : ahead + kStage;
  }

  // lane (r, h) holds outputs n0 + 32 NT w + 32 i + 8 (e / 4) + 4 h + e % 4 of x's row m0 + 32 j + r
  const int nb = n0 + 32 * NT * w + 4 * h;
  if constexpr (!SCORE) {
    // Through LDS, so that a row's outputs leave as 64 or 128 bytes together (straight from the registers, 8 bytes
    // of 32 rows an instruction, 2000 x 16384 x 1024 in 4 bits took 61 us).
    __syncthreads();  // everybody is done with the last stage
    constexpr int kPitch = 64 * NT + 16;  // bytes of a row of 32 NT 16-bit outputs, or of 16 NT floats
    char* own = lds + w * (32 * kPitch);
    const bool wide = a.y_dtype == Q4D_F32;
    const int size = wide ? 4 : 2;
    const bool whole = a.N % (16 / size) == 0;  // rows of 16-byte pieces
#pragma unroll
    for (int j = 0; j < MT; ++j) {
#pragma unroll
      for (int pass = 0; pass < 2; ++pass) {
        if (!whole) {
          const int m = m0 + 32 * j + r;
#pragma unroll
          for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 8 * pass; e < 8 * pass + 8; e += 4) {
              const int n = nb + 32 * i + 2 * e;
              if (m < a.M && n < a.N) store_out4(a, m, n, f32x4{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]});
            }
          continue;
        }
        if (pass && !wide) continue;
        // a pass: 16 columns of each tile of 32 as floats, all of them in 16 bits
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            if (wide) {
              if (e / 8 == pass)
                *reinterpret_cast<f32x4*>(own + r * kPitch + 64 * i + 4 * (2 * e - 16 * pass + 4 * h)) =
                    f32x4{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
            } else {
              *reinterpret_cast<u32x2*>(own + r * kPitch + 64 * i + 2 * (2 * e + 4 * h)) =
                  pack_out4(a.y_dtype, f32x4{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]});
            }
          }
#pragma unroll
        for (int c = 0; c < 2 * NT; ++c) {  // 16 bytes a lane, 4 NT lanes a row
          const int row = (64 * c + lane) / (4 * NT), col = (64 * c + lane) % (4 * NT);  // (in order: LDS answers a wave so)
          const int m = m0 + 32 * j + row;
          // of tile col / 4: floats 16 pass + 4 (col % 4) .., or 16-bit outputs 8 (col % 4) ..
          const int n = n0 + 32 * NT * w + 32 * (col / 4) + (wide ? 16 * pass + 4 * (col % 4) : 8 * (col % 4));
          const u32x4 v = *reinterpret_cast<const u32x4*>(own + row * kPitch + 16 * col);
          if (m < a.M && n < a.N) *reinterpret_cast<u32x4*>(static_cast<char*>(a.y) + ((size_t)m * a.N + n) * size) = v;
        }
      }
    }
  } else {
    __syncthreads();  // everybody is done with x's tiles
    float* s_stat = reinterpret_cast<float*>(lds);  // [4 waves][32 MT rows][3]
    const bool part = n0 + kTileN > a.N;            // outputs past the last are as -Inf
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const int m = m0 + 32 * j + r;
      const int hit = m < a.M ? a.targets[m] - nb : -1;  // 32 i + 8 (e / 4) + e % 4 of the lane's
      if (__ballot((unsigned)hit < 64u)) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (hit == 32 * i + 8 * (e >> 2) + (e & 3) && nb + hit < a.N) a.hit[m] = acc[i][j][e];
      }
      if (part) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (nb + 32 * i + 8 * (e >> 2) + (e & 3) >= a.N) acc[i][j][e] = -INFINITY;
      }
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, acc[i][j][e]);
      top = halves<false>(top);
      const float base = top == -INFINITY ? 0.f : top;
      float l = 0.f, u = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float d = acc[i][j][e] - base, p = exp_neg(d);
          l += p;
          u = fmaf(p, d, u);
        }
      if (__ballot(u != u && l == l)) {  // 0 x -Inf (seldom: an operation an output otherwise)
        u = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float d = acc[i][j][e] - base;
            u = fmaf(exp_neg(d), fmaxf(d, -1000.f), u);
          }
      }
      l = halves<true>(l);
      u = halves<true>(u);
      if (h == 0) {
        float* at = s_stat + (w * kTileM + 32 * j + r) * 3;
        at[0] = top;
        at[1] = l;
        at[2] = u;
      }
    }
    __syncthreads();
    if (t < kTileM && m0 + t < a.M) {
      SoftSum s = {s_stat[t * 3], s_stat[t * 3 + 1], s_stat[t * 3 + 2]};
#pragma unroll
      for (int i = 1; i < 4; ++i) {
        const float* at = s_stat + (i * kTileM + t) * 3;
        s = soft_join(s, SoftSum{at[0], at[1], at[2]});
      }
      a.stats[(size_t)(m0 + t) * mx_gemm_parts(a.N) + n0 / kTileN] = f32x4{s.m, s.l, s.t, 0.f};
    }
  }
}

long long tile_count(int M, int N, int nt, int mt) {
  return (N + 128LL * nt - 1) / (128 * nt) * ((M + 32LL * mt - 1) / (32 * mt));
}
template <MxKind KIND, bool SCORE, int NT, int MT, int RING, int PER_CU>
int launch(const MxProduct& p, hipStream_t st) {
  const long long tiles = tile_count(p.M, p.N, NT, MT);
  static_assert(KIND == MX_X4 || MT == 2, "");  // x's offsets in a tile, 64 rows of 2 kMxStride bytes, are 32 bits
  if (tiles > kMxTiles) return Q4D_ERR_SHAPE;
  hipLaunchKernelGGL((mx_gemm_kernel<KIND, SCORE, NT, MT, RING, PER_CU>), dim3((unsigned)tiles), dim3(256), 0, st, p);
  return check_launch();
}
template <MxKind KIND>
int launch(const MxProduct& p, hipStream_t st) {
  const MxForm f = mx_gemm_form(p.M, p.N, KIND);
  if constexpr (KIND == MX_X4) {
    if (f.mt == 4) return launch<KIND, false, 2, 4, 3, 2>(p, st);
  }
  if (f.nt == 2) return launch<KIND, false, 2, 2, 3, KIND == MX_X4 ? 2 : 3>(p, st);
  return launch<KIND, false, 1, 2, KIND == MX_X4 ? 5 : 6, 2>(p, st);
}
constexpr int kScoreNT = 2, kScoreMT = 2;

}  // namespace

// Tiles of 256 x 64, three blocks a CU (two with x in 4 bits); 128 x 64 where those are no more than one a CU:
// 1024 x 4096 x 4096 in 16 bits 42 / 39 us, 512 x 16384 x 1024 (two a CU) 20 / 24.  With x in 4 bits, whose
// products take a quarter of the time their operands are moved for, 256 x 128 where that gives two a CU:
// 4096 x 8192 x 4096 78 instead of 98 us, 2000 x 4096 x 4096 (one a CU) 31 instead of 28; in 16 bits the
// larger tile is no faster (8192 x 8192 x 8192 864 instead of 844, 2000 x 16384 x 1024 66 instead of 68).
MxForm mx_gemm_form(int M, int N, MxKind kind) {
  const int cus = device_cus();
  if (kind == MX_X4 && tile_count(M, N, 2, 4) >= 2 * cus) return {MX_TILES, 4, 2, 4};
  return {MX_TILES, 2, tile_count(M, N, 2, 2) > cus ? 2 : 1, 4};
}
MxForm mx_gemm_score_form() { return {MX_TILES, kScoreMT, kScoreNT, 4}; }
int launch_mx_gemm(const MxProduct& p, MxKind kind, hipStream_t st) {
  if (kind == MX_X4) return launch<MX_X4>(p, st);
  return kind == MX_BF16 ? launch<MX_BF16>(p, st) : launch<MX_F16>(p, st);
}
bool mx_gemm_scores(int M, int N) { return tile_count(M, N, kScoreNT, kScoreMT) <= kMxTiles; }
int launch_mx_gemm_score(const MxProduct& p, MxKind kind, hipStream_t st) {
  return kind == MX_BF16 ? launch<MX_BF16, true, kScoreNT, kScoreMT, 3, 3>(p, st) : launch<MX_F16, true, kScoreNT, kScoreMT, 3, 3>(p, st);
}

}  // namespace q4d
