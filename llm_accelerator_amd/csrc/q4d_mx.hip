// Quantisation to microscaled 4-bit floats and back, and rows of them from and to tiles (gfx950, wave64).
//
// A thread takes 8 consecutive values (16 or 32 bytes), four threads a block of 32, a wave 4 rows of a
// tile's 128 columns, so that it reads 256 or 512 bytes a row and writes 64-byte pieces of the tile.  The
// block's largest magnitude is a maximum over the values' bit patterns without their signs, which order
// like the values, Inf and NaN last; its exponent field E (biased, 0 for subnormals) gives the scale
// byte: floor(log2) - 2 is E - 2, clamped at 0.  Rounding to the eight magnitudes is one conversion
// instruction per two values (nearest, ties to even, past 6 to 6: exactly the format's rule).
// Bound by memory, 17/32 bytes a value written against 2 or 4 read, with the vector units busy 57 % of it: 151936 x
// 1024 in bf16 69-78 us, 5.0-5.7 TB/s, and back 58 us, 6.8 TB/s.  One row of 1024 is a launch, 2.4 us.
#include <algorithm>

#include "q4d_internal.h"
#include "q4d_mx_dev.h"

namespace q4d {
namespace {

struct MxArgs {
  const void* x;       // values (quantise) or rows of codes (pack)
  void* y;             // values (dequantise) or rows of codes (unpack)
  uint8_t* row_scale;  // [rows][cols / 32] (pack, unpack)
  uint32_t* codes;     // tiles
  uint8_t* scale;      // ... their scales
  long long ld;        // elements from row to row of x
  int rows, cols, col_tiles;
  uint32_t groups;     // of 4 rows of a tile
};

// Groups a wave has in flight.
constexpr int kUnroll = 4;

// A wave's lane (i, c) of group g: row 4 (g % 8) + i of tile g / 8, columns 8 c .. + 7.  Groups beside each
// other write the lines of one tile together.
struct MxPlace {
  int row, col;    // of the matrix
  size_t codes;    // 32-bit word of the tiles, scale byte
  size_t scale;
  bool in;         // the columns and the row are the matrix's
};
__device__ __forceinline__ MxPlace mx_place(const MxArgs& a, uint32_t g, int lane) {
  const uint32_t tile = g >> 3, rt = tile / (uint32_t)a.col_tiles, kt = tile - rt * a.col_tiles;
  const int i = lane >> 4, c = lane & 15, r = 4 * (g & 7) + i;
  MxPlace p;
  p.row = kMxRows * rt + r;
  p.col = kMxCols * kt + 8 * c;
  p.codes = ((size_t)tile * kMxTile + (c >> 2) * (kMxRows * 16) + r * 16) / 4 + (c & 3);
  p.scale = (size_t)tile * kMxScales + 4 * r + (c >> 2);
  p.in = p.row < a.rows && p.col < a.cols;
  return p;
}

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

template <int DT, bool CEIL>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const MxArgs a) {
  constexpr int kWords = DT == Q4D_F32 ? 8 : 4;
  const int lane = threadIdx.x & 63;
  const uint32_t stride = gridDim.x * 4;
  for (uint32_t g0 = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); g0 < a.groups; g0 += stride * kUnroll) {
    uint32_t x[kUnroll][kWords];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) x[u][i] = 0;  // columns past the last
      if (g0 + stride * u >= a.groups) continue;
      const MxPlace at = mx_place(a, g0 + stride * u, lane);
      if (!at.in) continue;
      const u32x4* p = reinterpret_cast<const u32x4*>(static_cast<const char*>(a.x) +
                                                      ((size_t)(at.row * a.ld) + at.col) * (DT == Q4D_F32 ? 4 : 2));
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const u32x4 v = __builtin_nontemporal_load(p + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[u][4 * i + e] = v[e];
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (g0 + stride * u >= a.groups) break;
      const MxPlace at = mx_place(a, g0 + stride * u, lane);
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
        const auto v = [&](int i) { return __builtin_bit_cast(float, x[u][i]); };
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v(0), v(1), f, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v(2), v(3), f, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v(4), v(5), f, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v(6), v(7), f, 3);
      } else if constexpr (DT == Q4D_BF16) {
        const auto v = [&](int i) { return __builtin_bit_cast(bf16x2, x[u][i]); };
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, v(0), f, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, v(1), f, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, v(2), f, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, v(3), f, 3);
      } else {
        const auto v = [&](int i) { return __builtin_bit_cast(f16x2, x[u][i]); };
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, v(0), f, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, v(1), f, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, v(2), f, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, v(3), f, 3);
      }
      if (at.row >= a.rows) continue;
      a.codes[at.codes] = s == 255 ? 0u : w;
      if ((lane & 3) == 0) a.scale[at.scale] = (uint8_t)s;
    }
  }
}

template <int DT>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const MxArgs a) {
  const int lane = threadIdx.x & 63;
  const uint32_t stride = gridDim.x * 4;
  for (uint32_t g0 = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); g0 < a.groups; g0 += stride * kUnroll) {
    uint32_t w[kUnroll], s[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (g0 + stride * u >= a.groups) continue;
      const MxPlace at = mx_place(a, g0 + stride * u, lane);
      if (!at.in) continue;
      w[u] = a.codes[at.codes];
      s[u] = a.scale[at.scale];
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (g0 + stride * u >= a.groups) break;
      const MxPlace at = mx_place(a, g0 + stride * u, lane);
      if (!at.in) continue;
      const float f = mx_scale(s[u]);
      const size_t to = (size_t)at.row * a.cols + at.col;
      if constexpr (DT == Q4D_F32) {
        const auto v0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], f, 0), v1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], f, 1);
        const auto v2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], f, 2), v3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], f, 3);
        f32x4* y = reinterpret_cast<f32x4*>(static_cast<float*>(a.y) + to);
        __builtin_nontemporal_store(f32x4{v0[0], v0[1], v1[0], v1[1]}, y);
        __builtin_nontemporal_store(f32x4{v2[0], v2[1], v3[0], v3[1]}, y + 1);
      } else {
        __builtin_nontemporal_store(mx_dequant8<DT == Q4D_BF16>(w[u], f),
                                    reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.y) + to));
      }
    }
  }
}

// Rows of codes and scales to tiles (PACK) or back.
template <bool PACK>
__global__ __launch_bounds__(256) void mx_rows_tiles_kernel(const MxArgs a) {
  const int lane = threadIdx.x & 63;
  for (uint32_t g = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); g < a.groups; g += gridDim.x * 4) {
    const MxPlace at = mx_place(a, g, lane);
    if (at.row >= a.rows) continue;
    const size_t word = ((size_t)at.row * a.cols + at.col) / 8, s = (size_t)at.row * (a.cols / 32) + at.col / 32;
    if constexpr (PACK) {
      a.codes[at.codes] = at.in ? static_cast<const uint32_t*>(a.x)[word] : 0u;
      if ((lane & 3) == 0) a.scale[at.scale] = at.in ? a.row_scale[s] : (uint8_t)0;
    } else if (at.in) {
      static_cast<uint32_t*>(a.y)[word] = a.codes[at.codes];
      if ((lane & 3) == 0) a.row_scale[s] = a.scale[at.scale];
    }
  }
}

bool mx_kind(int dtype) { return dtype == Q4D_F16 || dtype == Q4D_BF16 || dtype == Q4D_F32; }

MxArgs mx_args(const void* w, const void* s, int32_t rows, int32_t cols) {
  MxArgs a = {};
  a.codes = static_cast<uint32_t*>(const_cast<void*>(w));
  a.scale = static_cast<uint8_t*>(const_cast<void*>(s));
  a.rows = rows;
  a.cols = cols;
  a.col_tiles = mx_col_tiles(cols);
  a.groups = (uint32_t)mx_row_tiles(rows) * a.col_tiles * 8;
  return a;
}
// Blocks of four waves, each with `each` groups a round; past 8192 they go round.
dim3 mx_blocks(const MxArgs& a, int each) {
  return dim3(std::min<unsigned>((a.groups + 4 * each - 1) / (4 * each), 8192));
}

template <int DT>
void quantize(const MxArgs& a, bool ceil, hipStream_t st) {
  if (ceil) hipLaunchKernelGGL((mx_quantize_kernel<DT, true>), mx_blocks(a, kUnroll), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((mx_quantize_kernel<DT, false>), mx_blocks(a, kUnroll), dim3(256), 0, st, a);
}

}  // namespace

// Up to 2^27 tiles (2^38 codes): groups, and a round past the last, are counted in 32 bits.
bool mx_shape(int32_t rows, int32_t cols) {
  return rows > 0 && cols > 0 && cols % 32 == 0 && rows <= 0x7FFFFF00 && cols <= 0x7FFFFF00 &&
         (long long)mx_row_tiles(rows) * mx_col_tiles(cols) <= 1LL << 27;
}
int check_mx(const q4d_mx_t* t) {
  if (!t || !t->w || !t->s) return Q4D_ERR_NULL;
  if (!mx_shape(t->rows, t->cols)) return Q4D_ERR_SHAPE;
  return aligned(t->w, 16) && aligned(t->s, 4) ? Q4D_OK : Q4D_ERR_BAD_ADDR;
}

}  // namespace q4d

using namespace q4d;

extern "C" size_t q4d_mx_code_bytes(int32_t rows, int32_t cols) {
  return mx_shape(rows, cols) ? (size_t)mx_row_tiles(rows) * mx_col_tiles(cols) * kMxTile : 0;
}
extern "C" size_t q4d_mx_scale_bytes(int32_t rows, int32_t cols) {
  return mx_shape(rows, cols) ? (size_t)mx_row_tiles(rows) * mx_col_tiles(cols) * kMxScales : 0;
}

extern "C" int q4d_mx_quantize(const void* x, int32_t dtype, int64_t ld, int32_t rule, const q4d_mx_t* t, void* stream) {
  if (const int rc = check_mx(t)) return rc;
  if (!x) return Q4D_ERR_NULL;
  if (!mx_kind(dtype)) return Q4D_ERR_DTYPE;
  if ((t->rows > 1 && ld < t->cols) || (rule != Q4D_MX_FLOOR && rule != Q4D_MX_CEIL)) return Q4D_ERR_SHAPE;
  if (!aligned(x, 16) || (t->rows > 1 && ld % (dtype == Q4D_F32 ? 4 : 8))) return Q4D_ERR_BAD_ADDR;
  MxArgs a = mx_args(t->w, t->s, t->rows, t->cols);
  a.x = x;
  a.ld = ld;
  const bool ceil = rule == Q4D_MX_CEIL;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == Q4D_F32) quantize<Q4D_F32>(a, ceil, st);
  else if (dtype == Q4D_BF16) quantize<Q4D_BF16>(a, ceil, st);
  else quantize<Q4D_F16>(a, ceil, st);
  return check_launch();
}

extern "C" int q4d_mx_dequantize(const q4d_mx_t* t, void* y, int32_t y_dtype, void* stream) {
  if (const int rc = check_mx(t)) return rc;
  if (!y) return Q4D_ERR_NULL;
  if (!mx_kind(y_dtype)) return Q4D_ERR_DTYPE;
  if (!aligned(y, 16)) return Q4D_ERR_BAD_ADDR;
  MxArgs a = mx_args(t->w, t->s, t->rows, t->cols);
  a.y = y;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (y_dtype == Q4D_F32) hipLaunchKernelGGL(mx_dequantize_kernel<Q4D_F32>, mx_blocks(a, kUnroll), dim3(256), 0, st, a);
  else if (y_dtype == Q4D_BF16) hipLaunchKernelGGL(mx_dequantize_kernel<Q4D_BF16>, mx_blocks(a, kUnroll), dim3(256), 0, st, a);
  else hipLaunchKernelGGL(mx_dequantize_kernel<Q4D_F16>, mx_blocks(a, kUnroll), dim3(256), 0, st, a);
  return check_launch();
}

extern "C" int q4d_mx_pack(const uint8_t* packed, const uint8_t* scale, const q4d_mx_t* t, void* stream) {
  if (const int rc = check_mx(t)) return rc;
  if (!packed || !scale) return Q4D_ERR_NULL;
  if (!aligned(packed, 4)) return Q4D_ERR_BAD_ADDR;
  MxArgs a = mx_args(t->w, t->s, t->rows, t->cols);
  a.x = packed;
  a.row_scale = const_cast<uint8_t*>(scale);
  hipLaunchKernelGGL(mx_rows_tiles_kernel<true>, mx_blocks(a, 1), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), a);
  return check_launch();
}

extern "C" int q4d_mx_unpack(const q4d_mx_t* t, uint8_t* packed, uint8_t* scale, void* stream) {
  if (const int rc = check_mx(t)) return rc;
  if (!packed || !scale) return Q4D_ERR_NULL;
  if (!aligned(packed, 4)) return Q4D_ERR_BAD_ADDR;
  MxArgs a = mx_args(t->w, t->s, t->rows, t->cols);
  a.y = packed;
  a.row_scale = scale;
  hipLaunchKernelGGL(mx_rows_tiles_kernel<false>, mx_blocks(a, 1), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), a);
  return check_launch();
}
