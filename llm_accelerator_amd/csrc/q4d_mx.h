// Products with microscaled 4-bit weights: what the kernels' files share.
#pragma once

#include "q4d_internal.h"

namespace q4d {

struct MxProduct {
  const uint8_t* w;   // tiles of codes, of scales
  const uint8_t* ws;
  const void* x;      // 16-bit rows x_stride elements apart, or tiles of codes
  const uint8_t* xs;  // ... of their scales
  long long x_stride;
  int M, N, K;
  void* y;  // [M][N]
  int y_dtype;
  // of a score: row m's target (outside [0, N): none), the target's logit, and of each `parts` range of
  // the N outputs (max, sum of e^(z - max), sum of (z - max) e^(z - max), 0)
  const int32_t* targets;
  float* hit;  // [M]
  float __attribute__((ext_vector_type(4)))* stats;  // [M][parts]
};

enum MxKind { MX_X4 = 0, MX_F16 = 1, MX_BF16 = 2 };  // x: codes or 16-bit floats

// x's rows lie less than this many elements apart (64 of them within 32 bits), a score has up to so many rows (a
// launch's threads are counted in 32 bits, the join's are 256 a row).
constexpr long long kMxStride = 1 << 24;
constexpr int kMxScored = 1 << 23;
// ... and the tiles' kernel so many blocks.
constexpr long long kMxTiles = 1 << 23;

bool mx_shape(int32_t rows, int32_t cols);
int check_mx(const q4d_mx_t* t);

// A product's kernel, and its form: the blocks' rows of x and of weights in units of 16 (32 and 128 for tiles).
enum MxPath { MX_ROWS = 0, MX_HEAD = 1, MX_TILES = 2 };
struct MxForm {
  int path, mt, nt, waves;
};
MxForm mx_form(int M, int N, int K, MxKind kind);
MxForm mx_score_form(int M, int N, int K);

// Few rows (q4d_mx_rows.hip; a score: up to kMxFewRows) and tiles of many (q4d_mx_gemm.hip), and the ranges of N
// that a score's blocks leave.
constexpr int kMxFewRows = 64;
int launch_mx_rows(const MxProduct& p, MxKind kind, hipStream_t st);
int launch_mx_rows_score(const MxProduct& p, MxKind kind, hipStream_t st);
int mx_rows_parts(int M, int N);
MxForm mx_rows_form(int M, int N, int K);
MxForm mx_rows_score_form(int M);
// Few rows and many weights (q4d_mx_head.hip), where x fits in LDS.
bool mx_head_fits(int M, int K);
int mx_head_parts(int N);
MxForm mx_head_form(int M, int N);
int launch_mx_head(const MxProduct& p, MxKind kind, hipStream_t st);
int launch_mx_head_score(const MxProduct& p, MxKind kind, hipStream_t st);
MxForm mx_gemm_form(int M, int N, MxKind kind);
MxForm mx_gemm_score_form();
int launch_mx_gemm(const MxProduct& p, MxKind kind, hipStream_t st);
__host__ __device__ inline int mx_gemm_parts(int N) { return (int)((N + 255LL) / 256); }
bool mx_gemm_scores(int M, int N);  // no more tiles than that
int launch_mx_gemm_score(const MxProduct& p, MxKind kind, hipStream_t st);

}  // namespace q4d
