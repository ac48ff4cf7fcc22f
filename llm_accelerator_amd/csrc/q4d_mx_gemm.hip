// Products of many rows with microscaled 4-bit weights (gfx950, wave64): y = x W^T, and the score of
// given outputs, which keeps of each row's products only the sums of a softmax.
//
// A block takes 256 weight rows and 128 rows of x, a wave 64 x 128 of that.  x goes to LDS by DMA, 128
// bytes a row and stage (64 columns of 16 bits, 256 of 4), one stage ahead; weights go from memory to the
// registers of the one wave that needs them: lane (r, h) loads row r's block 2 i + h, and since the
// order of K inside a product is free, its 32 columns are the lane's share of 64: with 16-bit x four
// 32x32x16 products of 8 columns a lane after the codes are made 16-bit floats, with x in 4 bits one
// 32x32x64 product that takes codes and scales as they are.
// The weights are the first operand, so that a lane holds outputs of one row of x.
#include <float.h>
#include <math.h>

#include <type_traits>

#include "q4d_mx.h"
#include "q4d_mx_dev.h"

namespace q4d {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kTileN = 256, kTileM = 128;
constexpr int kRowBytes = 128;                // of x a stage
constexpr int kStage = kTileM * kRowBytes;
constexpr int kXcds = 8;

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
// Blocks 2 SEL' + h of a stage: the scale bytes were shifted by 8 h, so that byte 0 and 2 of word I / 2 serve.
template <int I>
__device__ __forceinline__ f32x16 mfma_codes(u32x4 a, uint32_t as, u32x4 b, uint32_t bs, f32x16 c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(codes_operand(a), codes_operand(b), c, 4, 4, 2 * (I & 1), (int)as,
                                                         2 * (I & 1), (int)bs);
}

// Lane i writes the 16 bytes at base + offset to LDS address lds + 16 i (lds, base wave-uniform).
// Ordered by the kernel's own wait and barrier.
__device__ __forceinline__ void dma16(const void* base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base)
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

// Up to 8 scale bytes from p on, `count` of them there, as two words shifted by 8 h.
__device__ __forceinline__ void load_scales(const uint8_t* p, int count, int h, uint32_t (&s)[2]) {
  uint64_t v = 0;
  if (count >= 8) {
    __builtin_memcpy(&v, p, 8);
  } else {
    for (int i = 0; i < count; ++i) v |= (uint64_t)p[i] << (8 * i);
  }
  s[0] = (uint32_t)v >> (8 * h);
  s[1] = (uint32_t)(v >> 32) >> (8 * h);
}

template <MxKind KIND, bool SCORE>
__global__ __launch_bounds__(256, 2) void mx_gemm_kernel(const MxProduct a) {
  constexpr bool X4 = KIND == MX_X4;
  constexpr int kCols = X4 ? 256 : 64;        // columns of a stage
  constexpr int kLoads = X4 ? 4 : 1;          // 16-byte weight loads of a lane and tile of 32 rows
  __shared__ __attribute__((aligned(16))) char lds[2 * kStage];
  const int t = threadIdx.x, lane = t & 63, r = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int tm = (a.M + kTileM - 1) / kTileM, tiles = gridDim.x;
  // an XCD takes consecutive tiles, those of one weight range after each other
  const int xcd = blockIdx.x % kXcds, per = tiles / kXcds, more = tiles % kXcds;
  const int tile = xcd * per + min(xcd, more) + blockIdx.x / kXcds;
  const int n0 = tile / tm * kTileN, m0 = tile % tm * kTileM;
  const int blocks = a.K / 32, stages = (a.K + kCols - 1) / kCols;
  const size_t x_row = X4 ? a.K / 2 : 2 * (size_t)a.x_stride;  // bytes

  // ---- x to LDS: slot s of row i holds the row's 16-byte group s ^ (i & 7) -----------------------
  const char* xb = static_cast<const char*>(a.x) + m0 * x_row;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const int group = (lane & 7) ^ (lane >> 3);
  uint32_t from[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) from[j] = (uint32_t)(min(32 * w + 8 * j + (lane >> 3), a.M - 1 - m0) * x_row) + 16 * group;
  const int x_groups = X4 ? blocks : a.K / 8;  // of a row
  const auto issue_x = [&](int st, int sg) {
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + sg * kStage + 32 * w * kRowBytes);
    const char* base = xb + (size_t)st * kRowBytes;
    const int have = x_groups - 8 * st;
    if (have >= 8) {
#pragma unroll
      for (int j = 0; j < 4; ++j) dma16(base, from[j], to + 1024 * j);
    } else {  // groups past the row's end are zeros
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x4 v = {0u, 0u, 0u, 0u};
        if (group < have) v = *reinterpret_cast<const u32x4*>(base + from[j]);
        *reinterpret_cast<u32x4*>(lds + sg * kStage + 32 * w * kRowBytes + 1024 * j + 16 * lane) = v;
      }
    }
  };

  // ---- weights to registers --------------------------------------------------------------------
  const uint8_t* wp[2];
  const uint8_t* sp[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int n = min(n0 + 64 * w + 32 * i + r, a.N - 1);
    wp[i] = a.w + (size_t)n * (a.K / 2);
    sp[i] = a.ws + (size_t)n * blocks;
  }
  const uint8_t* xsp[4];
  if constexpr (X4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) xsp[i] = a.xs + (size_t)min(m0 + 32 * i + r, a.M - 1) * blocks;
  }
  struct Weights {
    u32x4 q[2][kLoads];
    uint32_t s[2][2];
    uint32_t xs[X4 ? 4 : 1][2];
  };
  const auto load_w = [&](int st, Weights& v) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int k = 0; k < kLoads; ++k) {
        const int b = 2 * (kLoads * st + k) + h;
        v.q[i][k] = u32x4{0u, 0u, 0u, 0u};
        if (b < blocks) v.q[i][k] = *reinterpret_cast<const u32x4*>(wp[i] + 16 * b);
      }
      if constexpr (X4) {
        load_scales(sp[i] + 8 * st, blocks - 8 * st, h, v.s[i]);
      } else {
        const int b = 2 * st + h;
        v.s[i][0] = b < blocks ? sp[i][b] : 0u;
      }
    }
    if constexpr (X4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) load_scales(xsp[i] + 8 * st, blocks - 8 * st, h, v.xs[i]);
    }
  };

  f32x16 acc[2][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  const auto compute = [&](int sg, const Weights& v) {
    const char* xt = lds + sg * kStage + r * kRowBytes;
    const auto operand = [&](int j, int slot) {
      return *reinterpret_cast<const u32x4*>(xt + j * (32 * kRowBytes) + ((slot ^ (r & 7)) << 4));
    };
    if constexpr (X4) {
      const auto step = [&](auto k) {
        constexpr int I = decltype(k)::value;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x4 x = operand(j, 2 * I + h);
#pragma unroll
          for (int i = 0; i < 2; ++i) acc[i][j] = mfma_codes<I>(v.q[i][I], v.s[i][I >> 1], x, v.xs[j][I >> 1], acc[i][j]);
        }
      };
      step(std::integral_constant<int, 0>());
      step(std::integral_constant<int, 1>());
      step(std::integral_constant<int, 2>());
      step(std::integral_constant<int, 3>());
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        u32x4 wd[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) wd[i] = mx_dequant8<KIND == MX_BF16>(v.q[i][0][s], mx_scale(v.s[i][0]));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x4 x = operand(j, 4 * h + s);
#pragma unroll
          for (int i = 0; i < 2; ++i) acc[i][j] = mfma32<KIND == MX_BF16>(wd[i], x, acc[i][j]);
        }
      }
    }
  };

  Weights now, next;
  issue_x(0, 0);
  load_w(0, now);
  for (int st = 0; st < stages; ++st) {
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0): this wave's rows of x are there
    __builtin_amdgcn_s_barrier();        // everybody's are, and the other stage is read
    asm volatile("" ::: "memory");
    if (st + 1 < stages) {
      issue_x(st + 1, (st + 1) & 1);
      load_w(st + 1, next);
    }
    compute(st & 1, now);
    now = next;
  }

  // lane (r, h) holds outputs n0 + 64 w + 32 i + 8 (e / 4) + 4 h + e % 4 of x's row m0 + 32 j + r
  const int nb = n0 + 64 * w + 4 * h;
  if constexpr (!SCORE) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + 32 * j + r;
      if (m >= a.M) continue;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const int n = nb + 32 * i + 2 * e;
          if (n < a.N) store_out4(a, m, n, f32x4{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]});
        }
    }
  } else {
    __syncthreads();  // everybody is done with x's tiles
    float* s_stat = reinterpret_cast<float*>(lds);  // [4 waves][128 rows][3]
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + 32 * j + r;
      const int target = m < a.M ? a.targets[m] : -1;
      const bool mine = target >= n0 + 64 * w && target < n0 + 64 * w + 64;
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int n = nb + 32 * i + 8 * (e >> 2) + (e & 3);
          if (mine && n == target && n < a.N) a.hit[m] = acc[i][j][e];
          if (n >= a.N) acc[i][j][e] = -INFINITY;
          top = fmaxf(top, acc[i][j][e]);
        }
      top = halves<false>(top);
      const SoftSum s = soft_sum<32>(top, [&](int k) { return acc[k >> 4][j][k & 15]; });
      const float l = halves<true>(s.l), u = halves<true>(s.t);
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
      float* to = a.stats + ((size_t)(n0 / kTileN) * a.M + m0 + t) * 3;
      to[0] = s.m;
      to[1] = s.l;
      to[2] = s.t;
    }
  }
}

template <bool SCORE>
int launch(const MxProduct& p, MxKind kind, hipStream_t st) {
  const long long tiles = ((long long)p.N + kTileN - 1) / kTileN * ((p.M + kTileM - 1) / kTileM);
  const long long row = kind == MX_X4 ? p.K / 2 : 2 * p.x_stride;
  if (tiles > (1 << 23) || row * kTileM > 0x7FFFFFFFLL) return Q4D_ERR_SHAPE;  // a tile's offsets are 32 bits
  const dim3 grid((unsigned)tiles);
  if (kind == MX_X4) {
    if constexpr (SCORE) return Q4D_ERR_DTYPE;
    else hipLaunchKernelGGL((mx_gemm_kernel<MX_X4, false>), grid, dim3(256), 0, st, p);
  } else if (kind == MX_BF16) {
    hipLaunchKernelGGL((mx_gemm_kernel<MX_BF16, SCORE>), grid, dim3(256), 0, st, p);
  } else {
    hipLaunchKernelGGL((mx_gemm_kernel<MX_F16, SCORE>), grid, dim3(256), 0, st, p);
  }
  return check_launch();
}

}  // namespace

int launch_mx_gemm(const MxProduct& p, MxKind kind, hipStream_t st) { return launch<false>(p, kind, st); }
int mx_gemm_parts(int N) { return (N + kTileN - 1) / kTileN; }
int launch_mx_gemm_score(const MxProduct& p, MxKind kind, hipStream_t st) { return launch<true>(p, kind, st); }

}  // namespace q4d
