// Log probabilities of given tokens, ranks, entropy and the most likely alternatives out of logits
// (gfx950, wave64), in one pass over them.
//
// A row is cut into parts of 64 W x HELD logits; a block of W waves holds a part in registers, HELD logits a
// thread, and leaves the part's softmax sums, how many of its logits come before the target, and its K best.  A row
// of one part is finished there; else a second kernel joins a row's parts, a block a row.
//
// The K best: of the lanes' own maxima in a wave the K-th largest, found bit by bit with ballots, is reached by
// K logits, and so is the smallest of the waves' K/W-th largest; the larger of such bounds serves.  The few logits
// that reach it are gathered in LDS and ordered by counting.  Where masks leave fewer than K numbers, -Inf follows by
// index (64 rows of 151936 with 15 tokens left, K = 20, 21 us instead of 75; 1100 bf16 rows with 150 left, K = 5, 116
// instead of 287).  Where the logits are too many (equal ones) or NaN matters the bound is found again among keys of
// value and index, which no two logits share.  The parts' lists are joined by such a bound, too.
//
// Logits are ordered by value, then by index, the lower first; NaN comes last, after -Inf.
//
// Bound by the vector units, about twelve operations a logit and an exponential, and by loads that wait for the
// blocks before: 1100 bf16 rows of 151669 with one alternative 88-95 us, 3.5-3.8 TB/s (units busy 76 %; 102 registers,
// four waves a SIMD, which wait 55 % of their time), 64 fp32 rows of 151936 with 20 15 us, 2.6 TB/s (66 %; 2432 blocks on
// 2048 places, each its load, its sums and its search: the second round is a fifth full).  One row: 6.3 us, and 3-5 us
// for a join, both latency.
#include <float.h>
#include <math.h>

#include "q4d_internal.h"
#include "q4d_mx_dev.h"

namespace q4d {
namespace {

constexpr int kJoinThreads = 256;
constexpr int kHeldMost = 64;                 // logits of a thread, kHeldFew where there are few parts or short rows
constexpr int kHeldFew = 16;
constexpr int kTop = 32;                      // alternatives at most
constexpr int kMaxParts = 64;                 // of a row: vocabularies of up to 2^20
constexpr int kGather = 256;                  // logits that are ordered without a second bound

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
// V consecutive logits, 16 bytes at any alignment of the type.
template <int DT, int V>
__device__ __forceinline__ void load_logits(const void* p, size_t i, float* x) {
  u32x4 v;
  __builtin_memcpy(&v, static_cast<const char*>(p) + i * (16 / V), 16);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t u = v[e];
    if constexpr (DT == Q4D_F32) {
      x[e] = __builtin_bit_cast(float, u);
    } else if constexpr (DT == Q4D_BF16) {
      x[2 * e] = __builtin_bit_cast(float, u << 16);
      x[2 * e + 1] = __builtin_bit_cast(float, u & 0xFFFF0000u);
    } else {
      const f16x2 h = __builtin_bit_cast(f16x2, u);
      x[2 * e] = (float)h[0];
      x[2 * e + 1] = (float)h[1];
    }
  }
}
// A number that at least n of the lanes' u reach, and not many more: their n-th largest but for lower bits
// that do not tell them apart.
__device__ __forceinline__ uint32_t wave_reach(uint32_t u, int n) {
  uint32_t bound = 0;
  for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
    const int reach = __popcll(__ballot(u >= (bound | bit)));
    if (reach >= n) bound |= bit;
    if (reach == n) break;
  }
  return bound;
}

// Sum of a count of up to 2^16 a lane: exact in fp32.
__device__ __forceinline__ int wave_count(int c) { return (int)wave_all<true>((float)c); }

// What a row's outputs are once its sums are whole.
template <int DT>
__device__ __forceinline__ void finish_row(const LogprobArgs& a, int row, const SoftSum& s, float ll, int before) {
  a.entropy[row] = ll - s.t / s.l;
  if (!a.targets) return;
  const int target = a.targets[row];
  const bool have = target >= 0 && target < a.vocab;
  a.logprob[row] = have ? (logit<DT>(a.logits, (size_t)((long long)row * a.stride) + target) - s.m) - ll : NAN;
  a.rank[row] = have ? before : -1;
}
__device__ __forceinline__ void finish_top(const LogprobArgs& a, int row, const SoftSum& s, float ll, int rank, uint64_t key) {
  a.top_logprobs[(size_t)row * a.top + rank] = (key_value(key) - s.m) - ll;
  a.top_ids[(size_t)row * a.top + rank] = key_index(key);
}
__device__ __forceinline__ float log_sum(const SoftSum& s) { return s.m == -INFINITY ? NAN : logf(s.l); }

template <int DT, int HELD, int W>
__global__ __launch_bounds__(64 * W) void logprob_part_kernel(const LogprobArgs a) {
  constexpr int kThreads = 64 * W;
  constexpr int V = DT == Q4D_F32 ? 4 : 8, CH = HELD / V, kPart = kThreads * HELD;
  constexpr int kCand = HELD * kTop;
  static_assert(kCand >= kGather, "");
  __shared__ float s_stat[W][3];
  __shared__ int s_before[W];
  __shared__ uint32_t s_wave[2][W];
  __shared__ uint64_t s_key[kThreads];
  __shared__ uint64_t s_cand[kCand];
  __shared__ uint64_t s_bound;
  __shared__ int s_count, s_fill, s_more;
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
  const int base = part * kPart;
  const size_t row0 = (size_t)((long long)row * a.stride);
  const auto index = [&](int c) { return base + (c * kThreads + t) * V; };  // of a thread's chunk
  // Chunk c again from memory, for what is seldom needed: kept in registers, its masks and keys were spilled.
  const auto again = [&](int c, float (&v)[V]) {
    const int at = index(c);
    if (at + V <= a.vocab) {
      load_logits<DT, V>(a.logits, row0 + at, v);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = at + e < a.vocab ? logit<DT>(a.logits, row0 + at + e) : -INFINITY;
    }
  };
  const auto key_of = [&](const float (&v)[V], int c, int e) { return index(c) + e < a.vocab ? order_key(v[e], index(c) + e) : 0; };

  float x[HELD];
  if (base + kPart <= a.vocab) {
#pragma unroll
    for (int c = 0; c < CH; ++c) load_logits<DT, V>(a.logits, row0 + index(c), x + c * V);
  } else {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = index(c);
      if (at + V <= a.vocab) {
        load_logits<DT, V>(a.logits, row0 + at, x + c * V);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) x[c * V + e] = at + e < a.vocab ? logit<DT>(a.logits, row0 + at + e) : -INFINITY;
      }
    }
  }
  int target = -1;
  float goal = 0.f;
  if (a.targets) {
    target = a.targets[row];
    if (target < 0 || target >= a.vocab) target = -1;
    else goal = logit<DT>(a.logits, row0 + target);
  }
  if (t == 0) s_count = s_more = 0;

  // ---- softmax sums --------------------------------------------------------------------------
  float most[CH], mine = -INFINITY;  // of the chunks, of the thread
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    most[c] = x[c * V];
#pragma unroll
    for (int e = 1; e < V; ++e) most[c] = fmaxf(most[c], x[c * V + e]);
    mine = fmaxf(mine, most[c]);
  }
  const float top = wave_all<false>(mine);
  SoftSum s = soft_sum<HELD>(top, [&](int i) { return x[i]; });
  s.l = wave_all<true>(s.l);
  s.t = wave_all<true>(s.t);

  // ---- logits before the target ----------------------------------------------------------------
  // (of the wave: a comparison's lanes are counted by the scalar unit)
  int before = 0;
  if (target >= 0) {
    if (goal != goal) {  // NaN: all that are not, and the NaN of lower index
#pragma unroll 1
      for (int c = 0; c < CH; ++c) {
        float v[V];
        again(c, v);
#pragma unroll
        for (int e = 0; e < V; ++e) before += __popcll(__ballot(index(c) + e < a.vocab && (v[e] == v[e] || index(c) + e < target)));
      }
    } else {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int last = base + (c * kThreads + 64 * w + 64) * V;  // of the wave's 64 V
        if (last <= target) {
#pragma unroll
          for (int e = 0; e < V; ++e) before += __popcll(__ballot(x[c * V + e] >= goal));
        } else {  // (what lies past the row's end is -Inf, above which no goal lies)
#pragma unroll
          for (int e = 0; e < V; ++e) before += __popcll(__ballot(x[c * V + e] > goal));
        }
      }
      const int c = (target - base) / (kThreads * V);  // the target's own: equal ones of lower index
      if (target >= base && target - base < kPart && (target - base) / (64 * V) % W == w) {
        float v[V];
        again(c, v);
#pragma unroll
        for (int e = 0; e < V; ++e) before += __popcll(__ballot(v[e] == goal && index(c) + e < target));
      }
    }
  }
  if (lane == 0) {
    s_stat[w][0] = s.m;
    s_stat[w][1] = s.l;
    s_stat[w][2] = s.t;
    s_before[w] = before;
  }

  // ---- the K best ------------------------------------------------------------------------------
  int count = 0;
  if (a.top) {
    // (a thread without a number has the bits of -Inf or NaN, which the keys tell apart)
    const uint32_t u = order_bits(mine);
    uint32_t bound = a.top == 1 ? order_bits(top) : wave_reach(u, a.top);
    if constexpr (W > 1) {
      // (the second for more than a few, of which one wave's K best are not the part's)
      const uint32_t share = a.top > W ? wave_reach(u, (a.top + W - 1) / W) : 0;
      if (lane == 0) {
        s_wave[0][w] = bound;
        s_wave[1][w] = share;
      }
      __syncthreads();
      uint32_t least = s_wave[1][0];
#pragma unroll
      for (int i = 0; i < W; ++i) {
        bound = max(bound, s_wave[0][i]);
        least = min(least, s_wave[1][i]);
      }
      bound = max(bound, least);
    } else {
      __syncthreads();  // (s_count is set)
    }
    // A bound of -Inf, where masks leave few lanes a number: all numbers, if they are not too many.
    float least = key_value((uint64_t)bound << 32);
    if (!(least > -INFINITY)) least = -FLT_MAX;
    if (mine >= least) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (most[c] >= least) {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (x[c * V + e] >= least) {
              const int at = atomicAdd(&s_count, 1);
              if (at < kGather) s_cand[at] = order_key(x[c * V + e], index(c) + e);
            }
        }
      }
    }
    __syncthreads();
    count = s_count;
    if (count < a.top) {
      // Those of -Inf come next, the lowest index first: with fewer than K numbers in the part the first 64 indices hold
      // as many as are missing, or NaN.
      static_assert(2 * kTop <= 64, "");
      if (w == 0) {
        const float v = base + lane < a.vocab ? logit<DT>(a.logits, row0 + base + lane) : 0.f;
        const uint64_t low = __ballot(v == -INFINITY);
        if (v == -INFINITY) s_cand[count + __popcll(low & ((1ull << lane) - 1))] = order_key(v, base + lane);
        if (lane == 0) s_fill = __popcll(low);
      }
      __syncthreads();
      count += s_fill;
    }
    if (count < min(a.top, a.vocab - base) || count > kGather) {
      // by keys: of each thread's best the K-th best of the block is reached by K logits, and at most
      // HELD K reach it
      uint64_t best = 0;
#pragma unroll 1
      for (int c = 0; c < CH; ++c) {
        float v[V];
        again(c, v);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const uint64_t k = key_of(v, c, e);
          best = k > best ? k : best;
        }
      }
      s_key[t] = best;
      if (t == 0) s_bound = 1;  // (fewer than K threads have any: all are taken)
      __syncthreads();
      int ahead = 0;
      for (int i = 0; i < kThreads; ++i) ahead += s_key[i] > best;
      if (best && ahead == a.top - 1) s_bound = best;
      __syncthreads();
      const uint64_t floor = s_bound;
      if (best >= floor) {
#pragma unroll 1
        for (int c = 0; c < CH; ++c) {
          float v[V];
          again(c, v);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const uint64_t k = key_of(v, c, e);
            if (k >= floor) s_cand[atomicAdd(&s_more, 1)] = k;
          }
        }
      }
      __syncthreads();
      count = s_more;
    }
  }
  __syncthreads();
  if (w && 64 * w >= count) return;  // nothing of the wave's is among the candidates
  s = SoftSum{s_stat[0][0], s_stat[0][1], s_stat[0][2]};
#pragma unroll
  for (int i = 1; i < W; ++i) s = soft_join(s, SoftSum{s_stat[i][0], s_stat[i][1], s_stat[i][2]});
  before = s_before[0];
#pragma unroll
  for (int i = 1; i < W; ++i) before += s_before[i];
  const size_t slot = (size_t)row * a.parts + part;
  const bool whole = a.parts == 1;
  const float ll = whole ? log_sum(s) : 0.f;
  if (t == 0) {
    if (whole) {
      finish_row<DT>(a, row, s, ll, before);
    } else {
      a.stats[slot * 3] = s.m;
      a.stats[slot * 3 + 1] = s.l;
      a.stats[slot * 3 + 2] = s.t;
      a.before[slot] = before;
    }
  }
  const auto place = [&](uint64_t k, int rank) {
    if (rank >= a.top) return;
    if (whole) finish_top(a, row, s, ll, rank, k);
    else a.best[slot * a.top + rank] = k;
  };
  constexpr int kAt = W == 1 ? 2 : 1;  // of a lane, side by side: 64 lanes have up to 256 (50 rows of 1000, K = 32, 27 -> 19 us)
  for (int c = t; c < count; c += kAt * kThreads) {
    const bool second = W == 1 && c + kThreads < count;
    const uint64_t k = s_cand[c], k2 = second ? s_cand[c + kThreads] : ~0ull;
    int rank = 0, rank2 = 0;
#pragma unroll 4
    for (int i = 0; i < count; ++i) {
      rank += s_cand[i] > k;
      if (W == 1) rank2 += s_cand[i] > k2;
    }
    place(k, rank);
    if (second) place(k2, rank2);
  }
  if (!whole)
    for (int c = count + t; c < a.top; c += kThreads) a.best[slot * a.top + c] = 0;  // a last part of fewer logits
}

// A block a row, a part a lane of each wave.  Of the parts' J-th best keys as many as K / J reach their K/J-th
// largest, and so do K keys; J such that this is about the middle one.
template <int DT>
__global__ __launch_bounds__(kJoinThreads) void logprob_join_kernel(const LogprobArgs a) {
  constexpr int kEach = kMaxParts * kTop / kJoinThreads;  // keys of a thread
  __shared__ uint64_t s_key[kMaxParts * kTop];
  __shared__ int s_count;
  const int row = blockIdx.x, t = threadIdx.x, lane = t & 63;
  const size_t slot0 = (size_t)row * a.parts;
  const int all = a.parts * a.top;
  uint64_t key[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) key[i] = i * kJoinThreads + t < all ? a.best[slot0 * a.top + i * kJoinThreads + t] : 0;
  SoftSum s = {-INFINITY, 0.f, 0.f};
  int before = 0;
  uint32_t bound = 0, last = 0;
  const int nth = min(a.top, (2 * a.top + a.parts - 1) / a.parts);
  if (lane < a.parts) {
    const float* at = a.stats + (slot0 + lane) * 3;
    s = SoftSum{at[0], at[1], at[2]};
    before = a.before[slot0 + lane];
    if (a.top) {
      bound = (uint32_t)(a.best[(slot0 + lane) * a.top + nth - 1] >> 32);
      last = (uint32_t)(a.best[(slot0 + lane) * a.top + a.top - 1] >> 32);
    }
  }
  s = soft_wave(s);
  before = wave_count(before & 0xFFFF) + (wave_count(before >> 16) << 16);
  const float ll = log_sum(s);
  if (t == 0) finish_row<DT>(a, row, s, ll, before);
  if (!a.top) return;
  // (by value alone: keys of the bound's value all reach it, but earlier parts' come before them, and one such part
  // may have K: masked rows' -Inf, equal logits)
  const uint32_t least = wave_reach(bound, (a.top + nth - 1) / nth);
  const uint64_t reach = __ballot(bound >= least), full = __ballot(last >= least);
  if (t == 0) s_count = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (key[i] && (uint32_t)(key[i] >> 32) >= least) {
      if ((uint32_t)(key[i] >> 32) == least) {
        const uint64_t earlier = (1ull << ((i * kJoinThreads + t) / a.top)) - 1;
        if ((full & earlier) || __popcll(reach & earlier) * nth >= a.top) continue;
      }
      s_key[atomicAdd(&s_count, 1)] = key[i];
    }
  __syncthreads();
  const int count = s_count;
  for (int c = t; c < count; c += kJoinThreads) {
    const uint64_t k = s_key[c];
    int rank = 0;
#pragma unroll 4
    for (int i = 0; i < count; ++i) rank += s_key[i] > k;
    if (rank < a.top) finish_top(a, row, s, ll, rank, k);
  }
}

// How a row is cut: short rows are a wave's, others parts of four waves, of 16 logits a thread up to 4096 such blocks
// and of 64 past them (16 / 64 a thread, rows of 151936 in fp32 with 20 alternatives: 53 rows, 2014 blocks of 16 a
// thread, 17.9 / 19.7 us; 107 rows 25.2 / 26.2, 161 31.2 / 31.0, 315 49.9 / 45.7; with one alternative 107 rows 18.4 / 21.0,
// 315 40.9 / 39.8; in bf16 with 20 107 rows 26.3 / 27.2, 131 29.7 / 29.2).  Rows that 64 a thread hold in one part, up to
// 16384, want them earlier: 1000 rows of 10000 22.3 / 18.5 with 20, 13.6 / 12.8 with none.
struct Cut {
  int held, waves, parts;
};
Cut cut(int rows, int vocab) {
  if (vocab <= 64 * kHeldFew) return {kHeldFew, 1, 1};
  const auto parts = [&](int held) { return (vocab + 256 * held - 1) / (256 * held); };
  const bool few = parts(kHeldFew) <= kMaxParts && (parts(kHeldFew) == 1 || (long long)rows * parts(kHeldFew) <= 4096);
  return {few ? kHeldFew : kHeldMost, 4, parts(few ? kHeldFew : kHeldMost)};
}

struct LogprobLayout {
  size_t before, best, total;
};
LogprobLayout layout(int rows, int parts, int top) {
  LogprobLayout l;
  const size_t slots = (size_t)rows * parts;
  l.before = align_up(slots * 12, 256);
  l.best = align_up(l.before + slots * 4, 256);
  l.total = l.best + slots * top * 8;
  return l;
}

bool logprob_shape(int rows, int vocab, int top) {
  constexpr int kPart = 256 * kHeldMost;
  return rows > 0 && vocab > 0 && vocab <= kMaxParts * kPart && top >= 0 && top <= kTop && top <= vocab &&
         (long long)rows * ((vocab + kPart - 1) / kPart) <= (1 << 23);
}

template <int DT>
int launch(const LogprobArgs& a, const Cut& c, hipStream_t st) {
  const dim3 grid((unsigned)(a.rows * a.parts)), block(64 * c.waves);
  if (c.waves == 1) hipLaunchKernelGGL((logprob_part_kernel<DT, kHeldFew, 1>), grid, block, 0, st, a);
  else if (c.held == kHeldFew) hipLaunchKernelGGL((logprob_part_kernel<DT, kHeldFew, 4>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((logprob_part_kernel<DT, kHeldMost, 4>), grid, block, 0, st, a);
  if (a.parts > 1) hipLaunchKernelGGL(logprob_join_kernel<DT>, dim3((unsigned)a.rows), dim3(kJoinThreads), 0, st, a);
  return check_launch();
}

}  // namespace
}  // namespace q4d

using namespace q4d;

extern "C" size_t q4d_token_logprobs_workspace_bytes(int32_t rows, int32_t vocab, int32_t top) {
  if (!logprob_shape(rows, vocab, top)) return 0;
  return layout(rows, cut(rows, vocab).parts, top).total;
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
  const Cut c = cut(rows, vocab);
  const LogprobLayout l = layout(rows, c.parts, top);
  if (ws_bytes < l.total) return Q4D_ERR_CAPACITY;
  const LogprobArgs a = {logits, stride, rows, vocab, c.parts, top, targets, ws_ptr<float>(ws, 0), ws_ptr<int32_t>(ws, l.before),
                         ws_ptr<uint64_t>(ws, l.best), logprob, rank, entropy, top_logprobs, top_ids};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == Q4D_F32) return launch<Q4D_F32>(a, c, st);
  return dtype == Q4D_BF16 ? launch<Q4D_BF16>(a, c, st) : launch<Q4D_F16>(a, c, st);
}
