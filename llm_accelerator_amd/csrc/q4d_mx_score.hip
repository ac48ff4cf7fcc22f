// Entry points of the products with microscaled 4-bit weights, and the last step of a score: the sums
// that the product's blocks left of each row are joined.
#include <math.h>

#include "q4d_mx.h"
#include "q4d_mx_dev.h"

namespace q4d {
namespace {

struct JoinArgs {
  const f32x4* stats;  // [M][parts]
  const float* hit;    // [M]
  const int32_t* targets;
  int parts, M, N;
  float *logprob, *entropy, *best;
};

// A block a row: a thread's parts in order, then the threads'.  21 rows of 256 parts 3.9 us, a launch and two round
// trips; 1999 of 594, 19 MB, 6.5 us.
__global__ __launch_bounds__(256) void mx_score_join_kernel(const JoinArgs a) {
  __shared__ float s_stat[4][3];
  const int t = threadIdx.x, m = blockIdx.x;
  const f32x4* at = a.stats + (size_t)m * a.parts;
  SoftSum s = {-INFINITY, 0.f, 0.f};
#pragma unroll 4
  for (int p = t; p < a.parts; p += 256) {
    const f32x4 v = at[p];
    s = soft_join(s, SoftSum{v[0], v[1], v[2]});
  }
  s = soft_wave(s);
  if ((t & 63) == 0) {
    s_stat[t >> 6][0] = s.m;
    s_stat[t >> 6][1] = s.l;
    s_stat[t >> 6][2] = s.t;
  }
  __syncthreads();
  if (t) return;
#pragma unroll
  for (int i = 1; i < 4; ++i) s = soft_join(s, SoftSum{s_stat[i][0], s_stat[i][1], s_stat[i][2]});
  const float ll = s.m == -INFINITY ? NAN : logf(s.l);
  const int target = a.targets[m];
  a.logprob[m] = target >= 0 && target < a.N ? (a.hit[m] - s.m) - ll : NAN;
  a.entropy[m] = ll - s.t / s.l;
  a.best[m] = -ll;
}

int check_x(const q4d_mx_t* w, const void* x, int32_t x_dtype, int64_t x_stride, int32_t M) {
  if (const int rc = check_mx(w)) return rc;
  if (!x) return Q4D_ERR_NULL;
  if (x_dtype != Q4D_F16 && x_dtype != Q4D_BF16) return Q4D_ERR_DTYPE;
  if (M <= 0 || (M > 1 && (x_stride < w->cols || x_stride >= kMxStride))) return Q4D_ERR_SHAPE;
  return aligned(x, 16) && (M == 1 || x_stride % 8 == 0) ? Q4D_OK : Q4D_ERR_BAD_ADDR;
}
int check_y(const void* y, int32_t y_dtype) {
  if (!y) return Q4D_ERR_NULL;
  if (y_dtype != Q4D_F16 && y_dtype != Q4D_BF16 && y_dtype != Q4D_F32) return Q4D_ERR_DTYPE;
  return aligned(y, 16) ? Q4D_OK : Q4D_ERR_BAD_ADDR;
}
// Few outputs go to the kernel of few rows, which reads x once a weight tile but whose waves share K (us, rows' kernel
// / tiles): with 16-bit x up to 750000 (64 rows of 8192 x 1024 7.6 / 9.5, of 12288 11.4 / 9.5; 128 of 4096 x 4096
// 19.1 / 27.4, of 8192 x 4096 37.8 / 27.8), with x in 4 bits, a quarter of the bytes, up to a million or 16 rows
// (64 of 12288 x 1024 5.2 / 5.8, of 17408 7.3 / 5.9; 16 of 151936 18.2 / 19.8).  Beside the lines K and the last round
// of blocks decide, and outputs alone may miss: 64 of 11718 12.5 / 11.9 with K = 1024 and 38.7 / 30.1 with 4096, in
// 4 bits 64 of 16384 5.3 / 5.8 and 15.2 / 12.8.
// Up to 32 rows of many more weights: the kernel that holds x in LDS, from 49152 on (24 rows, rows / tiles / LDS: of
// 32768 x 1024 8.9 / 9.7 / 10.8, 49152 12.2 / 12.2 / 11.7, 65536 15.1 / 16.1 / 12.6, 151936 31 / 29 / 22; with
// K = 512 it is the faster one from 65536 on, with 2048 from 40960).
constexpr long long kFewOutputs = 750000, kFewOutputs4 = 1000000;
constexpr int kHeadRows = 49152;
MxPath product_path(int M, int N, int K, MxKind kind) {
  const long long outputs = (long long)M * N;
  if (kind == MX_X4) return outputs <= kFewOutputs4 || M <= 16 ? MX_ROWS : MX_TILES;
  if (outputs <= kFewOutputs) return MX_ROWS;
  return N >= kHeadRows && mx_head_fits(M, K) ? MX_HEAD : MX_TILES;
}
int product(const MxProduct& p, MxKind kind, hipStream_t st) {
  const MxPath path = product_path(p.M, p.N, p.K, kind);
  if (path == MX_ROWS) return launch_mx_rows(p, kind, st);
  return path == MX_HEAD ? launch_mx_head(p, kind, st) : launch_mx_gemm(p, kind, st);
}
// A score's kernels: the same three, few outputs being up to 1100000 and 64 rows (rows' kernel / tiles: 32 rows of
// 32768 x 1024 13.9 / 15.1 us, 40960 18.2 / 15.6; 48 of 16384 13.4 / 15.6, 24576 18.3 / 15.7; 64 of 12288 15.1 / 15.6,
// just below the line 64 of 17187 20.0 / 15.6), the one with x in LDS from 49152 tokens on (24 rows 17.4 / 15.6 / 14.7; 16
// rows 13.1 on the rows' kernel / 13.2, of 65536 15.0 / 14.3; one row 11.5 / 12.2, of 98304 17.0 / 15.9).
constexpr long long kFewScores = 1100000;
MxPath score_path(int M, int N, int K) {
  if (N >= kHeadRows && mx_head_fits(M, K)) return MX_HEAD;
  return M <= 16 || (M <= kMxFewRows && (long long)M * N <= kFewScores) ? MX_ROWS : MX_TILES;
}
MxKind kind_of(int32_t x_dtype) { return x_dtype == Q4D_BF16 ? MX_BF16 : MX_F16; }

size_t hit_bytes(int M) { return align_up((size_t)M * 4, 256); }
// Whether a score has these sizes: what a launch of its path holds.
bool score_shape(int M, int N, int K) {
  return mx_shape(N, K) && M > 0 && M <= kMxScored && (score_path(M, N, K) != MX_TILES || mx_gemm_scores(M, N));
}
int score_parts(int M, int N, int K) {
  const MxPath path = score_path(M, N, K);
  return path == MX_HEAD ? mx_head_parts(N) : path == MX_ROWS ? mx_rows_parts(M, N) : mx_gemm_parts(N);
}

}  // namespace

MxForm mx_form(int M, int N, int K, MxKind kind) {
  const MxPath path = product_path(M, N, K, kind);
  return path == MX_ROWS ? mx_rows_form(M, N, K) : path == MX_HEAD ? mx_head_form(M, N) : mx_gemm_form(M, N, kind);
}
MxForm mx_score_form(int M, int N, int K) {
  const MxPath path = score_path(M, N, K);
  return path == MX_ROWS ? mx_rows_score_form(M) : path == MX_HEAD ? mx_head_form(M, N) : mx_gemm_score_form();
}

}  // namespace q4d

using namespace q4d;

extern "C" int q4d_mx_linear(const q4d_mx_t* w, const void* x, int32_t x_dtype, int64_t x_stride, int32_t M, void* y,
                             int32_t y_dtype, void* stream) {
  int rc = check_x(w, x, x_dtype, x_stride, M);
  if (rc || (rc = check_y(y, y_dtype))) return rc;
  MxProduct p = {};
  p.w = w->w;
  p.ws = w->s;
  p.x = x;
  p.x_stride = M == 1 ? w->cols : x_stride;
  p.M = M;
  p.N = w->rows;
  p.K = w->cols;
  p.y = y;
  p.y_dtype = y_dtype;
  return product(p, kind_of(x_dtype), reinterpret_cast<hipStream_t>(stream));
}

extern "C" int q4d_mx_matmul(const q4d_mx_t* w, const q4d_mx_t* x, void* y, int32_t y_dtype, void* stream) {
  int rc = check_mx(w);
  if (rc || (rc = check_mx(x)) || (rc = check_y(y, y_dtype))) return rc;
  if (x->cols != w->cols) return Q4D_ERR_SHAPE;
  MxProduct p = {};
  p.w = w->w;
  p.ws = w->s;
  p.x = x->w;
  p.xs = x->s;
  p.M = x->rows;
  p.N = w->rows;
  p.K = w->cols;
  p.y = y;
  p.y_dtype = y_dtype;
  return product(p, MX_X4, reinterpret_cast<hipStream_t>(stream));
}

extern "C" size_t q4d_mx_score_workspace_bytes(int32_t rows, int32_t cols, int32_t M) {
  if (!score_shape(M, rows, cols)) return 0;
  return hit_bytes(M) + (size_t)score_parts(M, rows, cols) * M * sizeof(f32x4);
}

extern "C" int q4d_mx_score(const q4d_mx_t* w, const void* x, int32_t x_dtype, int64_t x_stride, int32_t M,
                            const int32_t* targets, float* logprob, float* entropy, float* best, void* ws, size_t ws_bytes,
                            void* stream) {
  int rc = check_x(w, x, x_dtype, x_stride, M);
  if (rc) return rc;
  if (!score_shape(M, w->rows, w->cols)) return Q4D_ERR_SHAPE;
  if (!targets || !logprob || !entropy || !best || !ws) return Q4D_ERR_NULL;
  if (!aligned(targets, 4) || !aligned(logprob, 4) || !aligned(entropy, 4) || !aligned(best, 4) || !aligned(ws, 256))
    return Q4D_ERR_BAD_ADDR;
  if (ws_bytes < q4d_mx_score_workspace_bytes(w->rows, w->cols, M)) return Q4D_ERR_CAPACITY;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  MxProduct p = {};
  p.w = w->w;
  p.ws = w->s;
  p.x = x;
  p.x_stride = M == 1 ? w->cols : x_stride;
  p.M = M;
  p.N = w->rows;
  p.K = w->cols;
  p.targets = targets;
  p.hit = ws_ptr<float>(ws, 0);
  p.stats = ws_ptr<f32x4>(ws, hit_bytes(M));
  const int parts = score_parts(M, p.N, p.K);
  const MxKind kind = kind_of(x_dtype);
  const MxPath path = score_path(M, p.N, p.K);
  if (path == MX_HEAD) rc = launch_mx_head_score(p, kind, st);
  else rc = path == MX_ROWS ? launch_mx_rows_score(p, kind, st) : launch_mx_gemm_score(p, kind, st);
  if (rc) return rc;
  const JoinArgs j = {p.stats, p.hit, targets, parts, M, p.N, logprob, entropy, best};
  hipLaunchKernelGGL(mx_score_join_kernel, dim3((unsigned)M), dim3(256), 0, st, j);
  return check_launch();
}
