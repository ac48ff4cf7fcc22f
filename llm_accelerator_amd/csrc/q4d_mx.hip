// Quantisation to microscaled 4-bit floats and back (gfx950, wave64).
//
// A thread takes 8 consecutive values (16 or 32 bytes), four threads a block of 32.  The block's
// largest magnitude is a maximum over the values' fp32 bit patterns without their signs, which order
// like the values, Inf and NaN last; its exponent field E (biased, 0 for subnormals) gives the scale
// byte: floor(log2) - 2 is E - 2, clamped at 0.  Rounding to the eight magnitudes is one conversion
// instruction per two values (nearest, ties to even, past 6 to 6: exactly the format's rule).
// Bound by memory: 17/32 bytes a value written against 2 or 4 read.
#include <algorithm>

#include "q4d_internal.h"
#include "q4d_mx_dev.h"

namespace q4d {
namespace {

struct MxArgs {
  const void* x;     // values in (quantise) or codes in (dequantise)
  void* y;           // codes out or values out
  uint8_t* scale;
  long long ld;      // elements from row to row of x
  uint32_t groups;   // of 8 values
  uint32_t per_row;  // groups a row
};

constexpr int kUnroll = 4;  // groups a thread has in flight

__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kDppQuadSwap1, 0xF, 0xF, false));
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kDppQuadSwap2, 0xF, 0xF, false));
}

// Scale byte of a block whose largest magnitude has these fp32 bits.
template <bool CEIL>
__device__ __forceinline__ uint32_t block_scale(uint32_t bits) {
  if (bits >= 0x7F800000u) return 255;  // Inf or NaN: the block is NaN
  int s = (int)(bits >> 23) - 2;
  if (CEIL && (bits & 0x7FFFFFu) > 0x400000u) ++s;  // past 1.5 2^E: past 6 2^s
  return (uint32_t)max(s, 0);
}

template <int DT, bool CEIL, bool ROWS>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const MxArgs a) {
  constexpr int kWords = DT == Q4D_F32 ? 8 : 4;
  const uint32_t stride = gridDim.x * 256u;
  for (uint64_t g0 = blockIdx.x * 256u + threadIdx.x; g0 < a.groups; g0 += (uint64_t)stride * kUnroll) {
    uint32_t x[kUnroll][kWords];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint64_t g = g0 + (uint64_t)stride * u;
      if (g >= a.groups) break;
      size_t at = (size_t)g * 8;
      if constexpr (ROWS) {
        const uint32_t row = (uint32_t)g / a.per_row;
        at = (size_t)((long long)row * a.ld) + ((uint32_t)g - row * a.per_row) * 8u;
      }
      const u32x4* p = reinterpret_cast<const u32x4*>(static_cast<const char*>(a.x) + at * (DT == Q4D_F32 ? 4 : 2));
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const u32x4 v = __builtin_nontemporal_load(p + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[u][4 * i + e] = v[e];
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint64_t g = g0 + (uint64_t)stride * u;
      if (g >= a.groups) break;
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        const uint32_t v = x[u][i];
        if constexpr (DT == Q4D_F32) {
          top = max(top, v & 0x7FFFFFFFu);
        } else if constexpr (DT == Q4D_BF16) {
          top = max(top, max(v << 16 & 0x7FFF0000u, v & 0x7FFF0000u));
        } else {  // fp16 magnitudes order like their bits; widened below
          top = max(top, max(v & 0x7FFFu, v >> 16 & 0x7FFFu));
        }
      }
      top = quad_max(top);
      if constexpr (DT == Q4D_F16)
        top = __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(_Float16, (uint16_t)top)) & 0x7FFFFFFFu;
      const uint32_t s = block_scale<CEIL>(top);
      const float f = mx_scale(s);
      uint32_t w = 0;
      if constexpr (DT == Q4D_F32) {
        const auto at = [&](int i) { return __builtin_bit_cast(float, x[u][i]); };
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, at(0), at(1), f, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, at(2), at(3), f, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, at(4), at(5), f, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, at(6), at(7), f, 3);
      } else if constexpr (DT == Q4D_BF16) {
        const auto at = [&](int i) { return __builtin_bit_cast(bf16x2, x[u][i]); };
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, at(0), f, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, at(1), f, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, at(2), f, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, at(3), f, 3);
      } else {
        const auto at = [&](int i) { return __builtin_bit_cast(f16x2, x[u][i]); };
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, at(0), f, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, at(1), f, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, at(2), f, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, at(3), f, 3);
      }
      static_cast<uint32_t*>(a.y)[g] = s == 255 ? 0u : w;
      if ((threadIdx.x & 3) == 0) a.scale[g >> 2] = (uint8_t)s;
    }
  }
}

template <int DT>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const MxArgs a) {
  const uint32_t stride = gridDim.x * 256u;
  for (uint64_t g0 = blockIdx.x * 256u + threadIdx.x; g0 < a.groups; g0 += (uint64_t)stride * kUnroll) {
    uint32_t w[kUnroll], s[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint64_t g = g0 + (uint64_t)stride * u;
      if (g >= a.groups) break;
      w[u] = static_cast<const uint32_t*>(a.x)[g];
      s[u] = a.scale[g >> 2];
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint64_t g = g0 + (uint64_t)stride * u;
      if (g >= a.groups) break;
      const float f = mx_scale(s[u]);
      if constexpr (DT == Q4D_F32) {
        const auto v0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], f, 0), v1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], f, 1);
        const auto v2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], f, 2), v3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], f, 3);
        f32x4* y = static_cast<f32x4*>(a.y) + 2 * g;
        __builtin_nontemporal_store(f32x4{v0[0], v0[1], v1[0], v1[1]}, y);
        __builtin_nontemporal_store(f32x4{v2[0], v2[1], v3[0], v3[1]}, y + 1);
      } else {
        __builtin_nontemporal_store(mx_dequant8<DT == Q4D_BF16>(w[u], f), static_cast<u32x4*>(a.y) + g);
      }
    }
  }
}

bool mx_kind(int dtype) { return dtype == Q4D_F16 || dtype == Q4D_BF16 || dtype == Q4D_F32; }

// Groups of 8 in a matrix (0: not a shape that the kernels take).
uint32_t mx_groups(int32_t rows, int32_t cols) {
  if (rows <= 0 || cols <= 0 || cols % 32) return 0;
  const unsigned long long g = (unsigned long long)rows * (cols / 8);
  return g > 0xFFF00000ull ? 0 : (uint32_t)g;
}
// Blocks of 256 threads, each with kUnroll groups a round; past 8192 they go round.
unsigned mx_blocks(uint32_t groups) {
  return (unsigned)std::min<unsigned long long>(((unsigned long long)groups + 256 * kUnroll - 1) / (256 * kUnroll), 8192);
}

template <int DT, bool CEIL>
void quantize(const MxArgs& a, bool rows, unsigned blocks, hipStream_t st) {
  if (rows) hipLaunchKernelGGL((mx_quantize_kernel<DT, CEIL, true>), dim3(blocks), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((mx_quantize_kernel<DT, CEIL, false>), dim3(blocks), dim3(256), 0, st, a);
}
template <int DT>
void quantize(const MxArgs& a, bool ceil, bool rows, unsigned blocks, hipStream_t st) {
  if (ceil) quantize<DT, true>(a, rows, blocks, st);
  else quantize<DT, false>(a, rows, blocks, st);
}

}  // namespace

int check_mx(const q4d_mx_t* t) {
  if (!t || !t->w || !t->s) return Q4D_ERR_NULL;
  if (!mx_groups(t->rows, t->cols)) return Q4D_ERR_SHAPE;
  return aligned(t->w, 16) ? Q4D_OK : Q4D_ERR_BAD_ADDR;
}

}  // namespace q4d

using namespace q4d;

extern "C" int q4d_mx_quantize(const void* x, int32_t dtype, int64_t ld, int32_t rows, int32_t cols, int32_t rule,
                               uint8_t* packed, uint8_t* scale, void* stream) {
  if (!x || !packed || !scale) return Q4D_ERR_NULL;
  if (!mx_kind(dtype)) return Q4D_ERR_DTYPE;
  const uint32_t groups = mx_groups(rows, cols);
  if (!groups || ld < cols || (rule != Q4D_MX_FLOOR && rule != Q4D_MX_CEIL)) return Q4D_ERR_SHAPE;
  const int size = dtype == Q4D_F32 ? 4 : 2;
  if (!aligned(x, 16) || (ld * size) % 16 || !aligned(packed, 16)) return Q4D_ERR_BAD_ADDR;
  const MxArgs a = {x, packed, scale, ld, groups, (uint32_t)cols / 8};
  const bool strided = ld != cols && rows > 1, ceil = rule == Q4D_MX_CEIL;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == Q4D_F32) quantize<Q4D_F32>(a, ceil, strided, mx_blocks(groups), st);
  else if (dtype == Q4D_BF16) quantize<Q4D_BF16>(a, ceil, strided, mx_blocks(groups), st);
  else quantize<Q4D_F16>(a, ceil, strided, mx_blocks(groups), st);
  return check_launch();
}

extern "C" int q4d_mx_dequantize(const q4d_mx_t* t, void* y, int32_t y_dtype, void* stream) {
  if (const int rc = check_mx(t)) return rc;
  if (!y) return Q4D_ERR_NULL;
  if (!mx_kind(y_dtype)) return Q4D_ERR_DTYPE;
  if (!aligned(y, 16)) return Q4D_ERR_BAD_ADDR;
  const uint32_t groups = mx_groups(t->rows, t->cols);
  const MxArgs a = {t->w, y, const_cast<uint8_t*>(t->s), t->cols, groups, (uint32_t)t->cols / 8};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (y_dtype == Q4D_F32) hipLaunchKernelGGL(mx_dequantize_kernel<Q4D_F32>, dim3(mx_blocks(groups)), dim3(256), 0, st, a);
  else if (y_dtype == Q4D_BF16) hipLaunchKernelGGL(mx_dequantize_kernel<Q4D_BF16>, dim3(mx_blocks(groups)), dim3(256), 0, st, a);
  else hipLaunchKernelGGL(mx_dequantize_kernel<Q4D_F16>, dim3(mx_blocks(groups)), dim3(256), 0, st, a);
  return check_launch();
}
