// Products of a few rows with microscaled 4-bit weights (gfx950, wave64): y = x W^T, and the score of
// given outputs (see q4d_mx_gemm.hip).
//
// A block takes 16 NT weight rows and 16 MT rows of x; its waves share K, 128 columns at a time: lane
// (r, g) loads the 16 bytes of weight row r's block g and the 32 values of x's row r there.  The
// order of K inside a product is free, so that both operands go to the matrix unit as they were loaded:
// four 16x16x32 products of 8 columns a lane after the codes are made 16-bit floats, or with x in 4 bits
// one 16x16x128 product that takes codes and scales as they are.  The waves' sums meet in LDS.
//
// Bound by a launch and its one or two memory round trips, for which the waves wait 70 % of their time: one row of
// 4096 x 1024 3.1 us, 48 of 1024 x 2048 4.7, five in 4 bits of 6144 x 1024 3.2.  Hence small blocks, K over a block's
// waves and two steps' loads in flight.
#include "q4d_mx.h"
#include "q4d_mx_dev.h"

namespace q4d {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

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

template <MxKind KIND, int MT, int NT>
struct RowsStep {  // a wave's operands of 128 columns
  u32x4 w[NT];
  uint32_t ws[NT];
  u32x4 x[MT][KIND == MX_X4 ? 1 : 4];
  uint32_t xs[KIND == MX_X4 ? MT : 1];
};

template <MxKind KIND, int MT, int NT, int NW, bool SCORE>
__global__ __launch_bounds__(64 * NW) void mx_rows_kernel(const MxProduct a) {
  __shared__ f32x4 part[NW][NT][MT][64];
  const int t = threadIdx.x, lane = t & 63, r = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int n0 = blockIdx.x * (16 * NT), m0 = blockIdx.y * (16 * MT);
  const int blocks = a.K / 32, steps = mx_col_tiles(a.K), row_tiles = mx_row_tiles(a.N);
  const auto load = [&](int it, RowsStep<KIND, MT, NT>& s) {
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      // (16-row halves of tiles that are there: outputs past the last are not stored)
      const int half = min(n0 / 16 + k, 2 * row_tiles - 1), row = 16 * (half & 1) + r;
      const size_t tile = (size_t)(half >> 1) * steps + it;
      s.w[k] = *reinterpret_cast<const u32x4*>(a.w + tile * kMxTile + g * (kMxRows * 16) + row * 16);
      s.ws[k] = a.ws[tile * kMxScales + 4 * row + g];
    }
    if constexpr (KIND == MX_X4) {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int m = min(m0 + 16 * i, (a.M - 1) & ~15);
        const size_t tile = (size_t)(m / kMxRows) * steps + it;
        s.x[i][0] = *reinterpret_cast<const u32x4*>(static_cast<const uint8_t*>(a.x) + tile * kMxTile + g * (kMxRows * 16) + (m % kMxRows + r) * 16);
        s.xs[i] = a.xs[tile * kMxScales + 4 * (m % kMxRows + r) + g];
      }
    } else {
      const int b = 4 * it + g;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int m = m0 + 16 * i + r;
#pragma unroll
        for (int j = 0; j < 4; ++j) s.x[i][j] = u32x4{0u, 0u, 0u, 0u};
        if (b < blocks && m < a.M) {
          const uint16_t* p = static_cast<const uint16_t*>(a.x) + m * a.x_stride + 32 * b;
#pragma unroll
          for (int j = 0; j < 4; ++j) s.x[i][j] = *reinterpret_cast<const u32x4*>(p + 8 * j);
        }
      }
    }
  };
  f32x4 acc[NT][MT];
#pragma unroll
  for (int k = 0; k < NT; ++k)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[k][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const auto take = [&](const RowsStep<KIND, MT, NT>& s) {
    if constexpr (KIND == MX_X4) {
#pragma unroll
      for (int k = 0; k < NT; ++k)
#pragma unroll
        for (int i = 0; i < MT; ++i)
          acc[k][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(codes_operand(s.w[k]), codes_operand(s.x[i][0]), acc[k][i],
                                                                       4, 4, 0, (int)s.ws[k], 0, (int)s.xs[i]);
    } else {
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        const float f = mx_scale(s.ws[k]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x4 v = mx_dequant8<KIND == MX_BF16>(s.w[k][j], f);
#pragma unroll
          for (int i = 0; i < MT; ++i) acc[k][i] = mfma16<KIND == MX_BF16>(v, s.x[i][j], acc[k][i]);
        }
      }
    }
  };
  // two steps' loads in flight
  for (int it = w; it < steps; it += 2 * NW) {
    RowsStep<KIND, MT, NT> s0, s1;
    load(it, s0);
    if (it + NW < steps) load(it + NW, s1);
    take(s0);
    if (it + NW < steps) take(s1);
  }
#pragma unroll
  for (int k = 0; k < NT; ++k)
#pragma unroll
    for (int i = 0; i < MT; ++i) part[w][k][i][lane] = acc[k][i];
  __syncthreads();
  // lane (r, g) of row tiles (k, i): outputs 16 k + 4 g .. + 3 of x's row 16 i + r
  const auto sum = [&](int k, int i) {
    f32x4 s = part[0][k][i][lane];
#pragma unroll
    for (int v = 1; v < NW; ++v)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += part[v][k][i][lane][e];
    return s;
  };
  if constexpr (!SCORE) {
    for (int c = w; c < NT * MT; c += NW) {
      const int k = c / MT, i = c - k * MT, m = m0 + 16 * i + r, n = n0 + 16 * k + 4 * g;
      const f32x4 s = sum(k, i);
      if (m < a.M && n < a.N) store_out4(a, m, n, s);
    }
  } else {
    for (int i = w; i < MT; i += NW) {
      const int m = m0 + 16 * i + r, hit = m < a.M ? a.targets[m] - n0 - 4 * g : -1;  // 16 k + e of the lane's
      float z[4 * NT], top = -INFINITY;
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        const f32x4 s = sum(k, i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool have = n0 + 16 * k + 4 * g + e < a.N;
          if (have && hit == 16 * k + e) a.hit[m] = s[e];
          z[4 * k + e] = have ? s[e] : -INFINITY;
          top = fmaxf(top, z[4 * k + e]);
        }
      }
      SoftSum s = soft_sum<4 * NT>(top, [&](int c) { return z[c]; });
#pragma unroll
      for (int v = 16; v <= 32; v *= 2) s = soft_join(s, SoftSum{__shfl_xor(s.m, v), __shfl_xor(s.l, v), __shfl_xor(s.t, v)});
      if (g == 0 && m < a.M) a.stats[(size_t)m * gridDim.x + blockIdx.x] = f32x4{s.m, s.l, s.t, 0.f};
    }
  }
}

template <MxKind KIND, int MT, int NT, int NW>
int launch(const MxProduct& p, hipStream_t st) {
  const dim3 grid((unsigned)((p.N + 16LL * NT - 1) / (16 * NT)), (unsigned)((p.M + 16 * MT - 1) / (16 * MT)));
  if (grid.y > 65535u || (long long)grid.x * (64 * NW) > 0xFFFFFFFFLL) return Q4D_ERR_SHAPE;
  hipLaunchKernelGGL((mx_rows_kernel<KIND, MT, NT, NW, false>), grid, dim3(64 * NW), 0, st, p);
  return check_launch();
}
template <MxKind KIND>
int launch(const MxProduct& p, hipStream_t st) {
  const MxForm f = mx_rows_form(p.M, p.N, p.K);
  if (f.mt == 4) return f.waves == 8 ? launch<KIND, 4, 2, 8>(p, st) : launch<KIND, 4, 2, 4>(p, st);
  if (f.mt == 2) {
    if (f.nt == 4) return launch<KIND, 2, 4, 4>(p, st);
    return f.waves == 8 ? launch<KIND, 2, 2, 8>(p, st) : launch<KIND, 2, 2, 4>(p, st);
  }
  if (f.nt == 4) return launch<KIND, 1, 4, 4>(p, st);
  if (f.nt == 2) return f.waves == 8 ? launch<KIND, 1, 2, 8>(p, st) : launch<KIND, 1, 2, 4>(p, st);
  return f.waves == 8 ? launch<KIND, 1, 1, 8>(p, st) : launch<KIND, 1, 1, 4>(p, st);
}

template <MxKind KIND, int MT, int NT>
int launch_score(const MxProduct& p, hipStream_t st) {
  const dim3 grid((unsigned)((p.N + 16LL * NT - 1) / (16 * NT)));
  if ((long long)grid.x * 256 > 0xFFFFFFFFLL) return Q4D_ERR_SHAPE;
  hipLaunchKernelGGL((mx_rows_kernel<KIND, MT, NT, 4, true>), grid, dim3(256), 0, st, p);
  return check_launch();
}
template <MxKind KIND>
int launch_score(const MxProduct& p, hipStream_t st) {
  const MxForm f = mx_rows_score_form(p.M);
  if (f.mt == 1) return launch_score<KIND, 1, 4>(p, st);
  return f.mt == 2 ? launch_score<KIND, 2, 4>(p, st) : launch_score<KIND, 4, 2>(p, st);
}

}  // namespace

// x's rows a block (16 mt): the fewest that leave no more blocks of 16 weight rows than two a CU.
// Weight rows a block (16 nt): 16 where those are at most one a CU, else 32, which share what is loaded of x: one row of
// 4096 x 1024 3.2 / 3.4 us, 16 of 8192 x 1024 4.7 / 4.1, 64 of 4096 x 4096 17.8 / 11.3.  64 for very many (16 rows
// of 24000 x 1024 6.7 / 6.6).  Eight waves where K is long (one row of 8192 x 8192 10.2 instead of 12.5 us).
MxForm mx_rows_form(int M, int N, int K) {
  const long long tiles = (N + 15LL) / 16;
  const int cus = device_cus();
  const auto blocks = [&](int mt) { return tiles * ((M + 16LL * mt - 1) / (16 * mt)); };
  const int mt = M <= 16 || blocks(1) <= 2 * cus ? 1 : M <= 32 || blocks(2) <= 2 * cus ? 2 : 4;
  const bool deep = K > 1024;
  if (N >= 32768 && !deep) return {MX_ROWS, mt, mt == 4 ? 2 : 4, 4};
  return {MX_ROWS, mt, blocks(mt) > cus ? 2 : 1, deep ? 8 : 4};  // (mt > 1: more than one a CU)
}
MxForm mx_rows_score_form(int M) { return M <= 16 ? MxForm{MX_ROWS, 1, 4, 4} : M <= 32 ? MxForm{MX_ROWS, 2, 4, 4} : MxForm{MX_ROWS, 4, 2, 4}; }

int launch_mx_rows(const MxProduct& p, MxKind kind, hipStream_t st) {
  if (kind == MX_X4) return launch<MX_X4>(p, st);
  return kind == MX_BF16 ? launch<MX_BF16>(p, st) : launch<MX_F16>(p, st);
}
int launch_mx_rows_score(const MxProduct& p, MxKind kind, hipStream_t st) {
  return kind == MX_BF16 ? launch_score<MX_BF16>(p, st) : launch_score<MX_F16>(p, st);
}
int mx_rows_parts(int M, int N) {
  const int n = 16 * mx_rows_score_form(M).nt;
  return (int)((N + n - 1LL) / n);
}

}  // namespace q4d
