// Log probabilities of given tokens, ranks, entropy and the most likely alternatives out of logits
// (gfx950, wave64), in one pass over them.
//
// A row is cut into parts of 256 x 64 logits; a block holds a part in registers, 64 logits a thread, and
// leaves the part's softmax sums, how many of its logits come before the target, and its K best.  The
// K best: of each thread's best the K-th best over the block is a bound that K logits reach, and the few
// that reach it are gathered in LDS and ordered by counting.  A second kernel joins a row's parts.
//
// Logits are ordered by value, then by index, the lower first; NaN comes last, after -Inf.
#include <math.h>

#include "q4d_internal.h"
#include "q4d_mx_dev.h"

namespace q4d {
namespace {

constexpr int kThreads = 256;
constexpr int kHeld = 64;                     // logits of a thread
constexpr int kPart = kThreads * kHeld;
constexpr int kTop = 32;                      // alternatives at most
constexpr int kMaxParts = 64;                 // of a row: vocabularies of up to 2^20

struct LogprobArgs {
  const void* logits;
  long long stride;
  int rows, vocab, parts, top;
  const int32_t* targets;
  float* stats;      // [rows][parts][3]
  int32_t* before;   // [rows][parts]
  uint64_t* best;    // [rows][parts][top] keys
  float* logprob;
  int32_t* rank;
  float* entropy;
  float* top_logprobs;
  int32_t* top_ids;
};

// A key that orders like (value, then lower index): the value's bits made monotonic, the index inverted.
// NaN and what is not there are below -Inf.
__device__ __forceinline__ uint32_t order_bits(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v == 0.f ? 0.f : v);  // -0 is 0
  return v != v ? 1u : u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_key(float v, int i) { return (uint64_t)order_bits(v) << 32 | (uint32_t)~i; }
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t u = (uint32_t)(k >> 32);
  if (u <= 1) return NAN;
  return __builtin_bit_cast(float, u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ int key_index(uint64_t k) { return (int)~(uint32_t)k; }

template <int DT>
__device__ __forceinline__ float logit(const void* p, size_t i) {
  if constexpr (DT == Q4D_F32) return static_cast<const float*>(p)[i];
  else if constexpr (DT == Q4D_BF16) return (float)static_cast<const __bf16*>(p)[i];
  else return (float)static_cast<const _Float16*>(p)[i];
}

template <int DT>
__global__ __launch_bounds__(kThreads) void logprob_part_kernel(const LogprobArgs a) {
  __shared__ float s_stat[4][3];
  __shared__ int s_before[4];
  __shared__ uint64_t s_key[kThreads];
  __shared__ uint64_t s_cand[kHeld * kTop];
  __shared__ uint64_t s_bound;
  __shared__ int s_count;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
  const int base = part * kPart;
  const size_t row0 = (size_t)((long long)row * a.stride);

  float x[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int at = base + i * kThreads + t;
    x[i] = at < a.vocab ? logit<DT>(a.logits, row0 + at) : -INFINITY;
  }
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) top = fmaxf(top, x[i]);
  SoftSum s = soft_sum<kHeld>(top, [&](int i) { return x[i]; });
#pragma unroll
  for (int m = 32; m; m >>= 1)
    s = soft_join(s, SoftSum{__shfl_xor(s.m, m), __shfl_xor(s.l, m), __shfl_xor(s.t, m)});

  int before = 0;
  if (a.targets) {
    const int target = a.targets[row];
    if (target >= 0 && target < a.vocab) {
      const uint64_t key = order_key(logit<DT>(a.logits, row0 + target), target);
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int at = base + i * kThreads + t;
        before += at < a.vocab && order_key(x[i], at) > key;
      }
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) before += __shfl_xor(before, m);
  }
  if (lane == 0) {
    s_stat[w][0] = s.m;
    s_stat[w][1] = s.l;
    s_stat[w][2] = s.t;
    s_before[w] = before;
  }
  const size_t slot = (size_t)row * a.parts + part;
  if (a.top) {
    uint64_t mine = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int at = base + i * kThreads + t;
      const uint64_t k = at < a.vocab ? order_key(x[i], at) : 0;
      mine = k > mine ? k : mine;
    }
    s_key[t] = mine;
    if (t == 0) {
      s_count = 0;
      s_bound = 1;  // (fewer than `top` threads have any: all are candidates)
    }
    __syncthreads();
    int ahead = 0;
    for (int i = 0; i < kThreads; ++i) ahead += s_key[i] > mine;
    if (mine && ahead == a.top - 1) s_bound = mine;
    __syncthreads();
    const uint64_t bound = s_bound;
    if (mine >= bound) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int at = base + i * kThreads + t;
        const uint64_t k = at < a.vocab ? order_key(x[i], at) : 0;
        if (k >= bound) s_cand[atomicAdd(&s_count, 1)] = k;
      }
    }
    __syncthreads();
    const int count = s_count;
    uint64_t* out = a.best + slot * a.top;
    for (int c = t; c < count; c += kThreads) {
      const uint64_t k = s_cand[c];
      int rank = 0;
      for (int i = 0; i < count; ++i) rank += s_cand[i] > k;
      if (rank < a.top) out[rank] = k;
    }
    for (int c = count + t; c < a.top; c += kThreads) out[c] = 0;
  }
  __syncthreads();
  if (t == 0) {
    s = SoftSum{s_stat[0][0], s_stat[0][1], s_stat[0][2]};
    for (int i = 1; i < 4; ++i) s = soft_join(s, SoftSum{s_stat[i][0], s_stat[i][1], s_stat[i][2]});
    a.stats[slot * 3] = s.m;
    a.stats[slot * 3 + 1] = s.l;
    a.stats[slot * 3 + 2] = s.t;
    a.before[slot] = s_before[0] + s_before[1] + s_before[2] + s_before[3];
  }
}

// A wave a row.
template <int DT>
__global__ __launch_bounds__(64) void logprob_join_kernel(const LogprobArgs a) {
  __shared__ uint64_t s_key[kMaxParts * kTop];
  const int row = blockIdx.x, lane = threadIdx.x;
  const size_t slot0 = (size_t)row * a.parts;
  SoftSum s = {-INFINITY, 0.f, 0.f};
  int before = 0;
  for (int p = lane; p < a.parts; p += 64) {
    const float* at = a.stats + (slot0 + p) * 3;
    s = soft_join(s, SoftSum{at[0], at[1], at[2]});
    before += a.before[slot0 + p];
  }
#pragma unroll
  for (int m = 32; m; m >>= 1) {
    s = soft_join(s, SoftSum{__shfl_xor(s.m, m), __shfl_xor(s.l, m), __shfl_xor(s.t, m)});
    before += __shfl_xor(before, m);
  }
  const float ll = s.m == -INFINITY ? NAN : logf(s.l);
  if (lane == 0) {
    a.entropy[row] = ll - s.t / s.l;
    if (a.targets) {
      const int target = a.targets[row];
      const bool have = target >= 0 && target < a.vocab;
      a.logprob[row] = have ? (logit<DT>(a.logits, (size_t)((long long)row * a.stride) + target) - s.m) - ll : NAN;
      a.rank[row] = have ? before : -1;
    }
  }
  const int count = a.parts * a.top;
  for (int c = lane; c < count; c += 64) s_key[c] = a.best[slot0 * a.top + c];
  __syncthreads();
  for (int c = lane; c < count; c += 64) {
    const uint64_t k = s_key[c];
    if (!k) continue;
    int rank = 0;
    for (int i = 0; i < count; ++i) rank += s_key[i] > k;
    if (rank < a.top) {
      a.top_logprobs[(size_t)row * a.top + rank] = (key_value(k) - s.m) - ll;
      a.top_ids[(size_t)row * a.top + rank] = key_index(k);
    }
  }
}

struct LogprobLayout {
  size_t before, best, total;
  int parts;
};
LogprobLayout layout(int rows, int vocab, int top) {
  LogprobLayout l;
  l.parts = (vocab + kPart - 1) / kPart;
  const size_t slots = (size_t)rows * l.parts;
  l.before = align_up(slots * 12, 256);
  l.best = align_up(l.before + slots * 4, 256);
  l.total = l.best + slots * top * 8;
  return l;
}

bool logprob_shape(int rows, int vocab, int top) {
  return rows > 0 && vocab > 0 && vocab <= kMaxParts * kPart && top >= 0 && top <= kTop && top <= vocab &&
         (long long)rows * ((vocab + kPart - 1) / kPart) <= (1 << 23);
}

template <int DT>
int launch(const LogprobArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(logprob_part_kernel<DT>, dim3((unsigned)(a.rows * a.parts)), dim3(kThreads), 0, st, a);
  hipLaunchKernelGGL(logprob_join_kernel<DT>, dim3((unsigned)a.rows), dim3(64), 0, st, a);
  return check_launch();
}

}  // namespace
}  // namespace q4d

using namespace q4d;

extern "C" size_t q4d_token_logprobs_workspace_bytes(int32_t rows, int32_t vocab, int32_t top) {
  return logprob_shape(rows, vocab, top) ? layout(rows, vocab, top).total : 0;
}

extern "C" int q4d_token_logprobs(const void* logits, int32_t dtype, int64_t stride, int32_t rows, int32_t vocab,
                                  const int32_t* targets, int32_t top, float* logprob, int32_t* rank, float* entropy,
                                  float* top_logprobs, int32_t* top_ids, void* ws, size_t ws_bytes, void* stream) {
  if (!logits || !entropy || !ws || (targets && (!logprob || !rank)) || (top > 0 && (!top_logprobs || !top_ids))) return Q4D_ERR_NULL;
  if (dtype != Q4D_F16 && dtype != Q4D_BF16 && dtype != Q4D_F32) return Q4D_ERR_DTYPE;
  if (!logprob_shape(rows, vocab, top) || (rows > 1 && stride < vocab)) return Q4D_ERR_SHAPE;
  if (!aligned(logits, dtype == Q4D_F32 ? 4 : 2) || !aligned(targets, 4) || !aligned(logprob, 4) || !aligned(rank, 4) ||
      !aligned(entropy, 4) || !aligned(top_logprobs, 4) || !aligned(top_ids, 4) || !aligned(ws, 256))
    return Q4D_ERR_BAD_ADDR;
  const LogprobLayout l = layout(rows, vocab, top);
  if (ws_bytes < l.total) return Q4D_ERR_CAPACITY;
  const LogprobArgs a = {logits, stride, rows, vocab, l.parts, top, targets, ws_ptr<float>(ws, 0), ws_ptr<int32_t>(ws, l.before),
                         ws_ptr<uint64_t>(ws, l.best), logprob, rank, entropy, top_logprobs, top_ids};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == Q4D_F32) return launch<Q4D_F32>(a, st);
  return dtype == Q4D_BF16 ? launch<Q4D_BF16>(a, st) : launch<Q4D_F16>(a, st);
}
