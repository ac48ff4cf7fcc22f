// Attention of a ragged batch's new tokens over a paged KV cache (gfx950, wave64).
//
// A kv head's query rows of a sequence are its new tokens times the G = q heads / kv heads that
// share the kv head: row r is token r / G, head r % G.  Sequences of up to 16 rows (decode steps,
// a few proposed tokens; 16 is what one MFMA takes) are bound by reading K and V once: rows_part.
// More rows share what is read: chunk_part.  A call is one launch.
// Both sides of the 16: decode steps on chunk_part would take 15 us instead of 8.0 (one sequence of
// 700 positions), 151 instead of 122 (64 of up to 4000), 31 instead of 22 (3 of up to 32700); 24 sequences of
// 5 tokens and 10 rows 34 instead of 26.  Batches of up to 32 rows a sequence take rows_part too, in two
// groups (4 tokens of 8 heads a kv head, two groups / chunk_part: one sequence of 700 positions 13.0 /
// 15.7 us, one of 6000 with two kv heads 17.4 / 21.0, 24 of up to 1500 21.8 / 22.4, 64 of up to 4000 144 / 154).
#include <float.h>
#include <math.h>

#include <type_traits>

#include "q4d_device.h"
#include "q4d_paged.h"

namespace q4d {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kRows = 16;             // query rows of a group of rows_part, which takes one or two
constexpr int kStep = 128;            // positions of a block's step there: 32 a wave
constexpr int kJoin = 8;              // parts joined at a time
constexpr int kLevels = 4;            // of joins: up to 8^4 parts
constexpr int kCounters = 1024;       // counters of a level, one per block
constexpr int kChunkCounters = 2048;  // the same of chunk_part, one per part

template <bool BF>
__device__ __forceinline__ float to_f32(uint16_t u) {
  if constexpr (BF) return __builtin_bit_cast(float, (uint32_t)u << 16);
  else return (float)__builtin_bit_cast(_Float16, u);
}
template <bool BF>
__device__ __forceinline__ uint16_t from_f32(float x) {
  if constexpr (BF) return __builtin_bit_cast(uint16_t, (__bf16)x);
  else return __builtin_bit_cast(uint16_t, (_Float16)x);
}
template <bool BF>
__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  if constexpr (BF) {
    bf16x8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (__bf16)x[e];
    return __builtin_bit_cast(u32x4, y);
  } else {
    f16x8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (_Float16)x[e];
    return __builtin_bit_cast(u32x4, y);
  }
}
// x as value and remainder: v = x in 16 bits, rest = x - v (exact in fp32) in 16 bits.
template <bool BF>
__device__ __forceinline__ void pack8_rest(float (&x)[8], u32x4& v, u32x4& rest) {
  v = pack8<BF>(x);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF) {
      x[2 * i] -= to_f32<BF>((uint16_t)v[i]);
      x[2 * i + 1] -= to_f32<BF>((uint16_t)(v[i] >> 16));
    } else {  // one mixed multiply-add each out of the pair (seen through, the compiler would round every x once more)
      uint32_t u = v[i];
      float minus = -1.f;
      asm("" : "+v"(u));
      asm("" : "+s"(minus));
      x[2 * i] = fmaf(to_f32<BF>((uint16_t)u), minus, x[2 * i]);
      x[2 * i + 1] = fmaf(to_f32<BF>((uint16_t)(u >> 16)), minus, x[2 * i + 1]);
    }
  }
  rest = pack8<BF>(x);
}
template <bool BF>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// Inf and NaN of V.  A row that does not see such a value gives it the weight 0, and so does the product's
// 16-bit type to a small weight or to what the rounding of one leaves: 0 x Inf is NaN.  So the products are
// taken as if there were none, which a part's sums show at its end: 0 x Inf and a weight x Inf stay Inf or
// NaN through every later sum and rescaling.  Only then the part is done again with those values set to
// zero, and they are added after the loop for the rows that see them (with the weight 1, which does as well:
// what is added is Inf or NaN; as NaN where the score is -Inf and the weight 0).  Which 64ths of the part's steps have some is kept as bits.  The sum l of such
// a row's weights is stored with a minus sign: see join_factor.

// Inf and NaN (the exponent is all ones) among eight 16-bit floats become 0; whether there were any.
template <bool BF>
__device__ __forceinline__ bool drop_odd(u32x4& v) {
  constexpr uint32_t e = BF ? 0x7F80u : 0x7C00u;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool lo = (v[i] & e) == e, hi = (v[i] & e << 16) == e << 16;
    v[i] &= (lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u);
    odd |= lo || hi;
  }
  return odd;
}
// Eight products of 16-bit floats, summed.
template <bool BF>
__device__ __forceinline__ float dot8(u32x4 a, u32x4 b) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s = fmaf(to_f32<BF>((uint16_t)a[i]), to_f32<BF>((uint16_t)b[i]), s);
    s = fmaf(to_f32<BF>((uint16_t)(a[i] >> 16)), to_f32<BF>((uint16_t)(b[i] >> 16)), s);
  }
  return s;
}
__device__ __forceinline__ bool not_finite(float x) { return !(fabsf(x) < INFINITY); }
__device__ __forceinline__ uint32_t sign_of(float x) { return __builtin_bit_cast(uint32_t, x) & 0x80000000u; }
__device__ __forceinline__ float with_sign(float x, uint32_t sign) {
  return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) | sign);
}

// What a part's sums (maximum m, sum of weights l) are multiplied with when they are joined to others with the
// maximum M; never 0 where l says that there is Inf or NaN among them, which have to stay what they are.
__device__ __forceinline__ float join_factor(float m, float l, float M) {
  const float f = m == -INFINITY ? 0.f : exp2f(m - M);
  return sign_of(l) ? fmaxf(f, 0x1p-149f) : f;
}

// 1 / the sum of a row's weights.  That is 0 where the row sees no position (its output is then zeros), and
// where every score that it sees is -Inf, for which the softmax is NaN: the pages up to position `last` tell.
__device__ __forceinline__ float inverse_sum(float l, const PagedView& p, const int32_t* tab, int last) {
  if (l != 0.f) return 1.0f / fabsf(l);
  for (int i = 0; i <= last >> p.page_shift; ++i)
    if (in_range(tab[i], p.num_pages)) return NAN;
  return 0.f;
}

// Max / sum over the four 16-lane rows of a wave, in every lane (as in q4d_attention.hip).
template <bool SUM>
__device__ __forceinline__ float rows4(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  const float x0 = __builtin_bit_cast(float, a0), x1 = __builtin_bit_cast(float, a1);
  const float s = SUM ? x0 + x1 : fmaxf(x0, x1);
  const uint32_t w = __builtin_bit_cast(uint32_t, s);
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  const float y0 = __builtin_bit_cast(float, b0), y1 = __builtin_bit_cast(float, b1);
  return SUM ? y0 + y1 : fmaxf(y0, y1);
}

__device__ __forceinline__ void store_dev(float* p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float load_dev(const float* p) {
  return __hip_atomic_load(const_cast<float*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// 4 keys of one dim out of row-major rows in LDS: lane i of each 16 addresses 4 dims (8 bytes) of
// key i / 4 and receives dim i of the four keys.
__device__ __forceinline__ u32x2 read_tr4(const char* p) {
  return __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p)));
}

// `bytes` from p on as a buffer: loads past them give zeros and read nothing.
// (p and bytes are the same in every lane, which the compiler does not always see.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* p, int bytes) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  const uint64_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)u);
  const uint64_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(u >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(lo | hi << 32), (short)0,
                                           __builtin_amdgcn_readfirstlane(bytes), 0x00027000);
}
// Non-temporal: every row is read once (64 sequences of up to 4000 positions 122 instead of 138 us; 3 of
// up to 32700 with 16-position pages 22.0 instead of 20.9).
__device__ __forceinline__ u32x4 rows_load(__amdgpu_buffer_rsrc_t r, int offset) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, 2));
}

// Four floats that another XCD's block writes or reads in this launch: the same accesses as
// store_dev / load_dev (device scope, past the caches that are not shared), 16 bytes at a time.
constexpr int kDeviceScope = 16;  // sc1
__device__ __forceinline__ void store_dev4(__amdgpu_buffer_rsrc_t r, int offset, f32x4 v) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, v), r, offset, 0, kDeviceScope);
}
__device__ __forceinline__ f32x4 load_dev4(__amdgpu_buffer_rsrc_t r, int offset) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, kDeviceScope));
}

// The running max moves only when a score exceeds it by more than this (log2 units): P = 2^(s - m)
// stays below 2^8, far inside fp16's range, and the rescaling of the output is rare (whole prompts
// 182 instead of 187 us, nothing where K and V are streamed).
constexpr float kRescale = 8.0f;
// bf16 values reach 3e38, and their sums pass fp32 where their mean does not.  A part whose sums came out
// Inf (see drop_odd) is done again with weights of 2^(8 - 32) at most, so that 2^24 positions have room, and
// every join of up to eight parts leaves room for four bits.  Powers of two change no result but those that
// fp32 would hold as subnormals.
constexpr float kHeadroom = 32.0f;
template <bool BF>
__device__ __forceinline__ float join_max(float M) {
  return BF ? M + 4.0f : M;
}

// ---- up to 16 query rows a sequence --------------------------------------------------------
// The work of a kv head is a line of steps of 128 positions, the sequences one after the other;
// `blocks` blocks take S = ceil(steps / blocks) consecutive steps each, so every block streams as
// many bytes whatever the lengths are.  A cut within `slack` steps of a sequence's end moves there,
// which saves its join (24 sequences of up to 1500 positions and 5 tokens 26.3 instead of 26.8 us).  A
// block's first and last sequences may be parts: their softmax states go to the workspace (slot 1:
// the sequence begins in this block; slot 0: it began in an earlier one), where they are joined.
// A step: S^T = K . Q^T (16x16x32 MFMA, K rows straight from memory in operand order, two tiles of 16
// positions a wave), online softmax per row, O^T += V^T . P^T, where the S^T accumulators already are
// the operand layout of P^T and V^T comes out of the wave's own LDS rows with the transposing read, so
// that the waves meet only at a sequence's end.  The product takes P as two numbers of the cache's
// type, the rounded value and what that leaves (22 or 16 bits together; the stream hides the second
// product: 1 % of a long batch's time, and outputs as close to 64 bits as their own rounding lets
// them be instead of 1.4 times as far).
// Bound by the K and V stream: 64 sequences of up to 4000 positions (790 MB) 120-123 us, 6.4 TB/s, which is
// what reads alone reach; short ones by a chain of ten dependent memory round trips (cut, page, rows,
// join): 7.9 us for one of 700 positions, 21-22 us (3.4 TB/s) for 3 of up to 32700, 26 us (4.2 TB/s) for 24
// of up to 1500 and 5 tokens.  One block a CU: two take 126 / 8.1 / 25.5 / 29.2 us.
struct Cut {
  int S, slack;
};
// A sequence's steps [lo, hi) of the line: the cuts inside are those of blocks first .. last.
__device__ __forceinline__ int cut_first(const Cut& c, int lo) { return (lo + c.slack + c.S) / c.S; }
__device__ __forceinline__ int cut_last(const Cut& c, int hi) { return (hi - c.slack - 1 + c.S) / c.S - 1; }

// The kernels' argument block as the hardware passes it (both have it as their only argument).  Read
// through this at the end of a sequence, its fields are not kept in scalar registers through the loops
// (kept, they pushed the loop's own scalars out: 60 v_readlane of 150 vector instructions a step).
typedef const __attribute__((address_space(4))) PagedAttnArgs* KernelArgs;
__device__ __forceinline__ KernelArgs late_args() {
  KernelArgs p = (KernelArgs)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

// Shared memory of a block: V rows or tiles, a little more, and per-sequence arrays past 64 sequences
// (up to 64 every wave holds one a lane).
template <int D>
struct Shared {
  static constexpr int kRowsV = 4 * 32 * 2 * D;      // rows: 32 rows of V a wave, also 16 rows of floats
  static constexpr int kChunkV = 2 * 2 * 64 * 2 * D;  // chunk: two stages of 64 rows of K and V
  static constexpr int kMore = 4 * kRows * 2 * 4 + 64;
};
constexpr int kLanes = 64;

// The steps (or items) of up to 64 sequences as one line, a sequence a lane: the lane whose part of
// the line, which ends at `end`, holds x.
__device__ __forceinline__ int lane_of(int end, int x) { return __builtin_ctzll(__ballot(end > x) | 1ULL << 63); }

template <int D, bool BF, int R>
__device__ __forceinline__ void rows_part(const PagedAttnArgs& a, char* lds, int* seqs, int block) {
  constexpr int KS = D / 32, DT = D / 16, NV = D / 16, LR = D / 8;  // LR lanes of 16 bytes a row
  constexpr int kRowBytes = 2 * D, kWaveBytes = 32 * kRowBytes;
  float* sml = reinterpret_cast<float*>(lds + Shared<D>::kRowsV);  // [4 waves][16 rows] of (m, l)
  int* s_sum = reinterpret_cast<int*>(sml + 4 * kRows * 2);        // [4]
  int* s_last = s_sum + 4;
  int* s_end = seqs;               // [n] steps of the sequences up to and with b
  int* s_len = s_end + a.r.n;      // positions
  int* s_first = s_len + a.r.n;    // first token row
  int* s_row = s_first + a.r.n;    // table row and new tokens << 16
  const int t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int kvh = a.p.kvh, G = a.qh / kvh;
  const int k = block / kvh, j = block - k * kvh;

  // ---- the cut -----------------------------------------------------------------------------
  const bool few = a.r.n <= kLanes;
  int W = 0, l_end = 0, l_row = 0;
  SeqSpan l_span = {0, 0, 0, 0};
  bool bad = false;
  const auto steps_of = [&](const SeqSpan& s) {
    return s.count > 0 && s.count * G <= R * kRows ? (s.len + kStep - 1) / kStep : 0;
  };
  if (few) {
    if (lane < a.r.n) l_span = seq_span(a.p, a.r, lane);
    bad = l_span.count < 0;
    l_row = l_span.row | l_span.count << 16;
    l_end = wave_incl(steps_of(l_span));
    W = __builtin_amdgcn_readlane(l_end, 63);
  } else {
    for (int g = 0; g < a.r.n; g += 256) {
      const int b = g + t;
      int steps = 0;
      if (b < a.r.n) {
        const SeqSpan s = seq_span(a.p, a.r, b);
        bad |= s.count < 0;
        steps = steps_of(s);
        s_len[b] = s.len;
        s_first[b] = s.first;
        s_row[b] = s.row | s.count << 16;
      }
      const int x = wave_incl(steps);
      if (g) block_sync_lds();  // the last round's sums have been read
      if (lane == 63) s_sum[w] = x;
      block_sync_lds();
      int before = 0, all = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        before += i < w ? s_sum[i] : 0;
        all += s_sum[i];
      }
      if (b < a.r.n) s_end[b] = W + before + x;
      W += all;
    }
    block_sync_lds();
    W = __builtin_amdgcn_readfirstlane(W);
  }
  if (bad && block == 0) atomicOr(a.p.status, Q4D_STATUS_BAD_SEQUENCE);
  Cut c;
  c.S = (W + a.blocks - 1) / a.blocks;
  c.slack = min(c.S / 4, 2);
  if (k * c.S >= W) return;
  const auto lds_at = [&](const int* p) { return __builtin_amdgcn_readfirstlane(*p); };  // the same in every lane
  const auto end_of = [&](int b) {  // steps up to and with sequence b (-1: none)
    if (b < 0) return 0;
    return few ? __builtin_amdgcn_readlane(l_end, b) : lds_at(s_end + b);
  };
  const auto find = [&](int x) {  // the sequence whose steps hold step x < W
    if (few) return lane_of(l_end, x);
    int lo = 0, hi = a.r.n - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (lds_at(s_end + mid) > x) hi = mid; else lo = mid + 1;
    }
    return lo;
  };
  const auto snap = [&](int x, int lo, int hi) {
    if (x - lo <= c.slack && x - lo <= hi - x) return lo;
    return hi - x <= c.slack ? hi : x;
  };
  int b = find(k * c.S);
  const int from = snap(k * c.S, end_of(b - 1), end_of(b));
  int to = W;
  if ((k + 1) * c.S < W) {
    const int e = find((k + 1) * c.S);
    to = snap((k + 1) * c.S, end_of(e - 1), end_of(e));
  }

  const int r = lane & 15, g = lane >> 4;
  char* vl = lds + w * kWaveBytes;
  for (; b < a.r.n; ++b) {
    const int lo = end_of(b - 1), hi = end_of(b);
    if (lo >= to) break;
    const int x0 = max(lo, from), x1 = min(hi, to);
    if (x0 >= x1) continue;
    const int row_count = few ? __builtin_amdgcn_readlane(l_row, b) : lds_at(s_row + b);
    const SeqSpan s = {row_count & 0xFFFF, few ? __builtin_amdgcn_readlane(l_span.first, b) : lds_at(s_first + b),
                       row_count >> 16, few ? __builtin_amdgcn_readlane(l_span.len, b) : lds_at(s_len + b)};
    const int rows = s.count * G;
    const int32_t* tab = a.p.table + (size_t)s.row * a.p.max_pages;
    const int shift = a.p.page_shift, inpage = (1 << shift) - 1;
    // of one or two groups of 16 query rows
    const auto serve = [&](auto groups) {
      constexpr int H = decltype(groups)::value;
      // this lane's query row of either 16, its last visible position, and the operand Q^T: dims 32 i + 8 g .. + 7
      int qpos[H];
      u32x4 q[H][KS];
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const int rr = min(kRows * h + r, rows - 1), tok = rr / G;
        qpos[h] = s.len - s.count + tok;
        const KernelArgs late = late_args();
        const uint16_t* qp = late->q + (s.first + tok) * late->q_stride + (j * G + rr - tok * G) * D + 8 * g;
#pragma unroll
        for (int i = 0; i < KS; ++i) q[h][i] = *reinterpret_cast<const u32x4*>(qp + 32 * i);
      }
      const int first_hidden = s.len - s.count + 1;  // positions from here on are hidden from some row

      const int s0 = x0 - lo, s1 = x1 - lo;
      struct Stage {
        u32x4 k[2][KS], v[NV];
        bool ok0, ok1;  // the first and second 16 positions' pages are there
      } d;
      // The page of lanes 0-31's and of lanes 32-63's 16 positions of step `it`.
      const auto page_of = [&](int it) {
        const int e = (it * kStep + 32 * w + ((lane & 32) >> 1)) >> shift;
        return tab[min(e, a.p.max_pages - 1)];
      };
      int page = page_of(s0);
      bool bad_page = false;
      uint64_t odd = 0;  // 64ths of the steps where Inf and NaN of V were set to zero
      const int per = (s1 - s0 + 63) / 64;
      // Loads of step `it`, without a branch, so that the next steps' loads stay in flight while this
      // one's are waited for: through descriptors that end with the sequence's last row (rows past it,
      // of a page that is not there or of a step past the part's end are zeros and cost nothing).  K in
      // operand order (score tile h row r is position 16 h + r), V row by row.
      const auto issue = [&](int it) {
        const int base = it * kStep + 32 * w;
        const int p0 = __builtin_amdgcn_readlane(page, 0), p1 = __builtin_amdgcn_readlane(page, 32);
        page = page_of(it + 1);
        const int end = it < s1 ? s.len : 0;
        const int n0 = min(max(end - base, 0), 16), n1 = min(max(end - base - 16, 0), 16);
        d.ok0 = in_range(p0, a.p.num_pages);
        d.ok1 = in_range(p1, a.p.num_pages);
        bad_page |= (n0 && !d.ok0) || (n1 && !d.ok1);
        const size_t o0 = page_elem(a.p, d.ok0 ? p0 : 0, j) + (size_t)(base & inpage) * D;
        const size_t o1 = page_elem(a.p, d.ok1 ? p1 : 0, j) + (size_t)((base + 16) & inpage) * D;
        const int b0 = d.ok0 ? n0 * kRowBytes : 0, b1 = d.ok1 ? n1 * kRowBytes : 0;
        const auto k0 = rows_rsrc(a.kplane + o0, b0), k1 = rows_rsrc(a.kplane + o1, b1);
        const auto v0 = rows_rsrc(a.vplane + o0, b0), v1 = rows_rsrc(a.vplane + o1, b1);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          d.k[0][i] = rows_load(k0, r * kRowBytes + 16 * g + 64 * i);
          d.k[1][i] = rows_load(k1, r * kRowBytes + 16 * g + 64 * i);
        }
#pragma unroll
        for (int i = 0; i < NV / 2; ++i) {
          d.v[i] = rows_load(v0, 16 * lane + 1024 * i);
          d.v[NV / 2 + i] = rows_load(v1, 16 * lane + 1024 * i);
        }
      };

      f32x4 o[H][DT];
      float m[H], l[H];  // of query rows r and 16 + r; l of this lane's positions only
      const auto consume = [&](int it, auto again) {
        const int base = it * kStep + 32 * w;
        const bool ok0 = d.ok0, ok1 = d.ok1;
        const bool hides = base + 32 > first_hidden;
        if constexpr (again) {
          bool any = false;
#pragma unroll
          for (int i = 0; i < NV; ++i) any |= drop_odd<BF>(d.v[i]);
          if (__ballot(any)) odd |= 1ULL << ((it - s0) / per);
        }
        // V into this wave's LDS rows: 32-byte chunk c of row x at c ^ f(x), f chosen so that the 16
        // rows of a transposing read fall on all banks
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int row = i * (64 / LR) + lane / LR, slot = lane % LR;
          const int f = D == 128 ? row & 7 : (row >> 1) & 3;
          *reinterpret_cast<u32x4*>(vl + row * kRowBytes + ((slot ^ (f << 1)) << 4)) = d.v[i];
        }
        f32x4 st[H][2];
#pragma unroll
        for (int h = 0; h < H; ++h) st[h][0] = st[h][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
          for (int h = 0; h < H; ++h) {
            st[h][0] = mfma16<BF>(d.k[0][i], q[h][i], st[h][0]);
            st[h][1] = mfma16<BF>(d.k[1][i], q[h][i], st[h][1]);
          }
        issue(it + 1);
        u32x4 pp[H], pr[H];
#pragma unroll
        for (int h = 0; h < H; ++h) {
          // this lane's positions: 4 g .. + 3 of either 16
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = st[h][e >> 2][e & 3] * a.scale;
          if (hides || !ok0 || !ok1) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (base + 16 * (e >> 2) + 4 * g + (e & 3) > qpos[h] || !(e < 4 ? ok0 : ok1)) y[e] = -INFINITY;
          }
          float mx = y[0];
#pragma unroll
          for (int e = 1; e < 8; ++e) mx = fmaxf(mx, y[e]);
          mx = rows4<false>(mx);
          if constexpr (BF && again) mx += kHeadroom;
          const bool move = mx > m[h] + kRescale || (m[h] == -INFINITY && mx > m[h]);
          if (__ballot(move)) {
            const float mn = move ? mx : m[h];
            const float f = m[h] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[h] - mn);
            m[h] = mn;
            l[h] *= f;
#pragma unroll
            for (int i = 0; i < DT; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[h][i][e] *= f;
          }
          const float ms = m[h] == -INFINITY ? 0.f : m[h];
          float p[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            p[e] = __builtin_amdgcn_exp2f(y[e] - ms);
            l[h] += p[e];
          }
          pack8_rest<BF>(p, pp[h], pr[h]);
        }
        // V^T operand: dim 16 i + r, the same eight positions
        const auto vt = [&](int i) {
          u32x4 v;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int row = 16 * h + 4 * g + (r >> 2);
            const int f = D == 128 ? row & 7 : (row >> 1) & 3;
            const u32x2 x = read_tr4(vl + row * kRowBytes + ((i ^ f) << 5) + 8 * (r & 3));
            v[2 * h] = x[0];
            v[2 * h + 1] = x[1];
          }
          return v;
        };
#pragma unroll
        for (int i = 0; i < DT; ++i) {
          const u32x4 v = vt(i);
#pragma unroll
          for (int h = 0; h < H; ++h) {
            o[h][i] = mfma16<BF>(v, pp[h], o[h][i]);
            o[h][i] = mfma16<BF>(v, pr[h], o[h][i]);
          }
        }
      };
      const auto pass = [&](auto again) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
          m[h] = -INFINITY;
          l[h] = 0.f;
#pragma unroll
          for (int i = 0; i < DT; ++i) o[h][i] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        issue(s0);
        for (int it = s0; it < s1; ++it) consume(it, again);
#pragma unroll
        for (int h = 0; h < H; ++h) l[h] = rows4<true>(l[h]);
      };
      pass(std::false_type());
      float zero = 0.f;  // NaN if a sum is Inf or NaN
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) zero = fmaf(o[h][i][e], 0.f, zero);
      if (__builtin_expect(__ballot(zero != 0.f) != 0, 0)) {
        page = page_of(s0);
        pass(std::true_type());
        const KernelArgs late = late_args();
        for (; odd; odd &= odd - 1)
          for (int i = 0, it = s0 + __builtin_ctzll(odd) * per; i < per && it < s1; ++i, ++it) {
            const int base = it * kStep + 32 * w;  // this wave's positions
            for (int pos = base; pos < min(s.len, base + 32); ++pos) {
              const int pg = tab[min(pos >> shift, a.p.max_pages - 1)];
              if (!in_range(pg, a.p.num_pages)) continue;
              const size_t at = page_elem(a.p, pg, j) + (size_t)(pos & inpage) * D;
              bool none[H];  // the weight is 0
#pragma unroll
              for (int h = 0; h < H; ++h) {
                float score = 0.f;
#pragma unroll
                for (int i = 0; i < KS; ++i)
                  score += dot8<BF>(q[h][i], *reinterpret_cast<const u32x4*>(late->kplane + at + 32 * i + 8 * g));
                none[h] = rows4<true>(score) * late->scale == -INFINITY;
                if (pos <= qpos[h]) {
                  m[h] = fmaxf(m[h], -FLT_MAX);  // (joined whatever the scores are)
                  l[h] = with_sign(l[h], 0x80000000u);
                }
              }
              const uint16_t* v = late->vplane + at + 4 * g;
#pragma unroll
              for (int i = 0; i < DT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float x = to_f32<BF>(v[16 * i + e]);
#pragma unroll
                  for (int h = 0; h < H; ++h)
                    if (pos <= qpos[h] && not_finite(x)) o[h][i][e] += none[h] ? NAN : x;
                }
            }
          }
      }
      if (bad_page && lane == 0) atomicOr(a.p.status, Q4D_STATUS_BAD_PAGE);

      // ---- the four waves' states ----------------------------------------------------------------
      // a thread takes row t / 16 of either 16 and D / 64 slots of 4 dims each: sl, sl + 16
      const int row = t >> 4, sl = t & 15;
      constexpr int NS = D / 64;
      float M[H], L[H];
      f32x4 acc[H][NS];
#pragma unroll
      for (int h = 0; h < H; ++h) {
        if (h) block_sync_lds();  // the first rows' states have been read
        if (g == 0) {
          sml[(w * kRows + r) * 2] = m[h];
          sml[(w * kRows + r) * 2 + 1] = l[h];
        }
        // lane holds O^T[dim 16 i + 4 g + e][row r]: 16-byte slot 4 i + g of row r at slot ^ r
#pragma unroll
        for (int i = 0; i < DT; ++i)
          *reinterpret_cast<f32x4*>(vl + r * (4 * D) + (((4 * i + g) ^ r) << 4)) = o[h][i];
        block_sync_lds();
        M[h] = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) M[h] = fmaxf(M[h], sml[(i * kRows + row) * 2]);
        M[h] = join_max<BF>(M[h]);
        L[h] = 0.f;
        uint32_t sign = 0;
#pragma unroll
        for (int n = 0; n < NS; ++n) acc[h][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float li = sml[(i * kRows + row) * 2 + 1], f = join_factor(sml[(i * kRows + row) * 2], li, M[h]);
          L[h] = fmaf(fabsf(li), f, L[h]);
          sign |= sign_of(li);
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(lds + i * kWaveBytes + row * (4 * D) + (((sl + 16 * n) ^ row) << 4));
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[h][n][e] = fmaf(x[e], f, acc[h][n][e]);
          }
        }
        L[h] = with_sign(L[h], sign);
      }
      // The parts' states are joined eight at a time: of each eight the block that counts in last adds
      // them in order and goes on with the sum as one of the next level's parts.
      const KernelArgs late = late_args();
      const auto pacc = rows_rsrc(late->pacc, 1 << 30);
      float* pml = late->pml;
      const int kf = cut_first(c, lo);
      int count = max(0, cut_last(c, hi) - kf + 1) + 1, part = x0 == lo ? 0 : k - kf + 1;
      // part 0 lies in block kf - 1's slot 1, part i in block kf - 1 + i's slot 0; a sum lies where its
      // first part did, and its counter is that block's
      for (int level = 0, step = 1; count > 1; ++level, step *= kJoin) {
        const auto place = [&](int i, int h) {
          return ((((kf - 1 + i * step) * 2 + (i == 0)) * kvh + j) * R + h) * kRows + row;
        };
        const int first = part / kJoin * kJoin, size = min(kJoin, count - first);
        if (size > 1) {
#pragma unroll
          for (int h = 0; h < H; ++h) {
            if (kRows * h + row >= rows) continue;
            const int at = place(part, h);
#pragma unroll
            for (int n = 0; n < NS; ++n) store_dev4(pacc, (at * D + 64 * n + 4 * sl) * 4, acc[h][n]);
            if (sl == 0) {
              store_dev(pml + at * 2, M[h]);
              store_dev(pml + at * 2 + 1, L[h]);
            }
          }
          __builtin_amdgcn_s_waitcnt(0);  // this thread's stores are performed
          __syncthreads();                // ... and every other thread's
          int* counter = late->counters + level * kCounters + (kf - 1 + first * step) * kvh + j;
          if (t == 0) *s_last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == size - 1;
          __syncthreads();
          if (!*s_last) break;
          if (t == 0) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // next call
#pragma unroll
          for (int h = 0; h < H; ++h) {
            if (kRows * h + row >= rows) continue;
            float mi[kJoin], li[kJoin];
            f32x4 ai[kJoin][NS];
#pragma unroll
            for (int i = 0; i < kJoin; ++i) {
              const int at = place(first + min(i, size - 1), h);
              mi[i] = load_dev(pml + at * 2);
              li[i] = load_dev(pml + at * 2 + 1);
#pragma unroll
              for (int n = 0; n < NS; ++n) ai[i][n] = load_dev4(pacc, (at * D + 64 * n + 4 * sl) * 4);
            }
            M[h] = -INFINITY;
#pragma unroll
            for (int i = 0; i < kJoin; ++i) M[h] = fmaxf(M[h], mi[i]);
            M[h] = join_max<BF>(M[h]);
            L[h] = 0.f;
            uint32_t sign = 0;
#pragma unroll
            for (int n = 0; n < NS; ++n) acc[h][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kJoin; ++i) {
              if (i >= size) continue;
              const float f = join_factor(mi[i], li[i], M[h]);
              L[h] = fmaf(fabsf(li[i]), f, L[h]);
              sign |= sign_of(li[i]);
#pragma unroll
              for (int n = 0; n < NS; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[h][n][e] = fmaf(ai[i][n][e], f, acc[h][n][e]);
            }
            L[h] = with_sign(L[h], sign);
          }
        }
        part = first / kJoin;
        count = (count + kJoin - 1) / kJoin;
      }
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const int at = kRows * h + row;
        if (count > 1 || at >= rows) continue;
        const int otok = at / G;
        uint16_t* op = late->out + (s.first + otok) * late->out_stride + (j * G + at - otok * G) * D + 4 * sl;
        const float inv = inverse_sum(L[h], a.p, tab, s.len - s.count + otok);
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          const uint32_t u0 = from_f32<BF>(acc[h][n][0] * inv), u1 = from_f32<BF>(acc[h][n][1] * inv);
          const uint32_t u2 = from_f32<BF>(acc[h][n][2] * inv), u3 = from_f32<BF>(acc[h][n][3] * inv);
          *reinterpret_cast<u32x2*>(op + 64 * n) = u32x2{u0 | u1 << 16, u2 | u3 << 16};
        }
      }
    };
    if (R > 1 && rows > kRows) serve(std::integral_constant<int, R>());
    else serve(std::integral_constant<int, 1>());
    block_sync_lds();  // the next sequence's V rows go where the states were
  }
}

// ---- more rows ------------------------------------------------------------------------------
// A block takes 128 query rows of a sequence for one kv head, a wave 32 of them, over a part of the
// positions that they see, 64 at a time:
//   S^T = K . Q^T (32x32x16 MFMA; K rows from LDS, Q^T in registers); online softmax per row; O^T +=
//   V^T . P^T, where the S^T accumulators already are the operand layout of P^T (a lane holds 4 + 4
//   keys of each 16 for one row) and V^T comes out of the row-major tile with the transposing read.
// The product takes P as two numbers of the cache's type, as in rows_part: rounded once it was as far again
// from 64 bits as the output's own rounding (2.9e-4 instead of 2.1e-4 in fp16, 2.1e-3 instead of 1.6e-3 in
// bf16), and a token's precision went by how many came with it.  The second product costs prompts 212 instead of
// 165 us, 512 tokens after 4097 44 instead of 39.
// K and V tiles go from the pages to LDS by DMA one tile ahead, 16 rows a wave (one page at most).
// Two blocks a CU, so that one's products run under the other's softmax.  4 prompts of up to 3500
// positions, 16 / 8 heads: 212-220 us, 660-690 TFLOP/s of what rows see and, with the remainder's product,
// 990-1030 of what the matrix units do, which are busy 54 % of the time (a product of 8192^3 reaches 1365);
// 512 tokens after 4097 44 us.  Measured with one product and no faster than this order's 178 us: the next
// step's first product interleaved with this one's exponentials in a wave (180), the same with 8 waves that
// share tiles two or three steps ahead (185), with 64 rows a wave and 512 registers (264: accumulators move
// between the register files).
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kTile = 128;  // query rows of a block
constexpr int kKeys = 64;   // positions of a step

template <bool BF>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Max / sum of lanes l and l ^ 32, in both.
template <bool SUM>
__device__ __forceinline__ float halves(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  const float x0 = __builtin_bit_cast(float, a0), x1 = __builtin_bit_cast(float, a1);
  return SUM ? x0 + x1 : fmaxf(x0, x1);
}

// Lane i writes the 16 bytes at base + offset to LDS address lds + 16 i (lds, base wave-uniform).
// Ordered by the kernel's own wait and barrier.
__device__ __forceinline__ void dma16(const uint16_t* base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base)
               : "memory", "m0");
}

// A tile of n steps is cut into round(n / S) parts, S the steps that fill the device's blocks once (two
// a CU; at least kMinSplit, so that a part pays for its join).  Parts then have 3/4 S .. 3/2 S steps.
// kMinSplit 2 / 4 / 6: one sequence of 1500 positions and 20 tokens 19.2 / 17.8 / 19.7 us, 2 of 200 fresh
// ones 14.8 / 12.7 / 12.6, 3 of 900 and 40 tokens 18.9 / 19.4 / 20.2.
constexpr int kMinSplit = 4;
// One block a CU instead of two where that leaves two under kOneSteps steps each (the joins of twice the
// parts cost more than the overlap gives), or where rows_part's blocks have more steps than these and
// keep the CU busy beside.  Two / one, us: 64 tokens after 20000 (4.9 steps) 48 / 40, 40 sequences of 500
// positions and 20 tokens (5) 43 / 29, 16 of 3000 with two kv heads (2.9) 36.2 / 34.7; two chunks of 700
// after 1500 beside 9 decode steps (7) 64 / 70, 60 tokens after 30000 (7.3) 56 / 50, 2048 fresh ones (8.3) 42 /
// 47, 512 after 4097 (8.7) 43.4 / 42.9, 24 of 1500 and 20 tokens (9) 57 / 45: past the line it goes by how full
// the tiles are, too, which the rule does not look at.  Those two chunks beside 17 / 31 / 60 decode steps of 3000
// positions (0.9 / 1.6 / 3.1 of their steps): 79 / 82, 101 / 104, 163 / 147; two of up to 700 of 3000 beside 38
// (3.2) 100 / 93.
constexpr int kOneSteps = 6;
// A sequence's tiles are at most its rows / kTile, rounded up.
__host__ __device__ inline long long tiles_most(int tokens, int G, int n) { return (long long)tokens * G / kTile + n; }
__device__ __forceinline__ int split_parts(int steps, int S) { return max(1, (2 * steps + S) / (2 * S)); }
constexpr int kMaxParts = 64;

template <int D, bool BF>
__device__ __forceinline__ void chunk_part(const PagedAttnArgs& a, char* lds, int* seqs, int block) {
  constexpr int KS = D / 16, DT = D / 32, LR = D / 8;  // LR slots of 16 bytes a row
  constexpr int kRowBytes = 2 * D, kPlane = kKeys * kRowBytes, kStage = 2 * kPlane;
  int* s_sum = reinterpret_cast<int*>(lds + 2 * kStage);  // [2][4]
  int* s_again = s_sum + 8;  // [4]
  unsigned long long* s_odd = reinterpret_cast<unsigned long long*>(s_again + 4);
  int* s_last = s_again + 6;
  int* s_end = seqs;               // [n] items of the sequences up to and with b
  int* s_split = s_end + a.r.n;    // [n] the same of sequences in parts
  const int t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int kvh = a.p.kvh, G = a.qh / kvh;
  const int idx = block / kvh, j = block - idx * kvh;

  // ---- which item ----------------------------------------------------------------------------
  const auto tiles_of = [&](const SeqSpan& s) { return s.count * G > kRows ? (s.count * G + kTile - 1) / kTile : 0; };
  const auto steps_of = [&](int len) { return (len + kKeys - 1) / kKeys; };
  // steps of a sequence's tile, and of all its tiles (they grow evenly from the first to the last)
  const auto tile_steps = [&](const SeqSpan& s, int tile) {
    return steps_of(s.len - s.count + (min(s.count * G, (tile + 1) * kTile) - 1) / G + 1);
  };
  const auto work_of = [&](const SeqSpan& s) {
    const int n = tiles_of(s);
    return n ? (int)min((long long)n * (tile_steps(s, 0) + steps_of(s.len)) / 2, 1LL << 18) : 0;
  };
  // steps of rows_part's sequences, which stream K and V beside these
  const auto beside_of = [&](const SeqSpan& s) {
    return s.count > 0 && s.count * G <= kRows ? (s.len + kStep - 1) / kStep : 0;
  };
  const auto share = [&](int W, int most, int beside) {
    const int slots = W < kOneSteps * a.slots || beside > W ? (a.slots + 1) / 2 : a.slots;
    return max(max(kMinSplit, (W + slots - 1) / slots), (most + kMaxParts - 2) / (kMaxParts - 1));
  };
  // Starts that go back and forth (a bad batch) can ask for more tiles than the launch has blocks: then no
  // block does anything, so that no part waits for one that never comes.
  const long long most_tiles = tiles_most(a.r.tokens, G, a.r.n);
  SeqSpan s = {0, 0, 0, 0};
  int parts, tile, part, slots;  // slots: lane i's is the workspace slot of the tile's part i
  if (a.r.n <= kLanes) {
    // A sequence a lane.
    SeqSpan l = {0, 0, 0, 0};
    if (lane < a.r.n) l = seq_span(a.p, a.r, lane);
    const int l_nt = tiles_of(l), l_rows = l_nt ? l.count * G : 0, l_old = l.len - l.count;
    const auto sum = [&](int x) { return __builtin_amdgcn_readlane(wave_incl(x), 63); };
    // tiles of v steps and more, of a sequence with `rows` rows after `old` positions: the last ones
    const auto at_least = [&](int v, int nt, int rows, int old) {
      const long long x = ((long long)kKeys * (v - 1) - old) * G;  // that many rows before the tile's last
      if (x <= 0) return nt;
      return x < rows ? nt - (int)(x / kTile) : 0;
    };
    const int tiles = sum(l_nt);
    if (tiles == 0 || tiles > most_tiles) return;
    int most = l_nt ? steps_of(l.len) : 0;
#pragma unroll
    for (int m = 32; m; m >>= 1) most = max(most, __shfl_xor(most, m));
    most = __builtin_amdgcn_readfirstlane(most);
    // Layer p = lane + 1: the tiles of p parts and more, which have steps >= p S - S / 2; layer 1 counts
    // those of two and more, like layer 2.  Sizes of the layers, and of lane b's sequences' share.
    int S = share(sum(work_of(l)), most, sum(beside_of(l))), size = 0, end = 0;
    const auto in_layer = [&](int b) {
      return at_least(S * max(lane + 1, 2) - S / 2, __builtin_amdgcn_readlane(l_nt, b),
                      __builtin_amdgcn_readlane(l_rows, b), __builtin_amdgcn_readlane(l_old, b));
    };
    const uint64_t mine = __ballot(l_nt > 0);
    for (;; S += (S + 3) / 4) {
      size = 0;
      if (2 * most + S >= 4 * S)  // (otherwise nothing is cut)
        for (uint64_t todo = mine; todo; todo &= todo - 1) size += in_layer(__builtin_ctzll(todo));
      end = wave_incl(size);
      if (__builtin_amdgcn_readlane(end, 63) <= a.max_splits) break;  // (always, but for roundings and steps past what W counts)
    }
    const int split = __builtin_amdgcn_readlane(end, 63), first = __builtin_amdgcn_readlane(end, 0);
    int b, rank;  // the tile's, from the sequence's last
    if (idx >= split - first + tiles) return;
    if (idx < split - first) {
      // second and later parts, which are about S steps each, come first
      const int layer = lane_of(end, first + idx);
      const int at = first + idx - (__builtin_amdgcn_readlane(end, layer) - __builtin_amdgcn_readlane(size, layer));
      const int n = at_least(S * (layer + 1) - S / 2, l_nt, l_rows, l_old), upto = wave_incl(n);
      b = lane_of(upto, at);
      rank = at - (__builtin_amdgcn_readlane(upto, b) - __builtin_amdgcn_readlane(n, b));
      part = layer;
    } else {
      // then the first (or only) parts, the tiles of the most steps first, whatever their sequence (one
      // that sees much and starts last keeps a few CUs busy alone): more than `at` tiles have v steps
      const int at = idx - (split - first);
      int v = 1, hi = most;
      while (v < hi) {
        const int mid = (v + hi + 1) >> 1;
        if (sum(at_least(mid, l_nt, l_rows, l_old)) > at) v = mid; else hi = mid - 1;
      }
      const int more = at_least(v + 1, l_nt, l_rows, l_old), here = at_least(v, l_nt, l_rows, l_old) - more;
      const int upto = wave_incl(here), left = at - sum(more);
      b = lane_of(upto, left);
      rank = __builtin_amdgcn_readlane(more, b) + left -
             (__builtin_amdgcn_readlane(upto, b) - __builtin_amdgcn_readlane(here, b));
      part = 0;
    }
    s = {__builtin_amdgcn_readlane(l.row, b), __builtin_amdgcn_readlane(l.first, b),
         __builtin_amdgcn_readlane(l.count, b), __builtin_amdgcn_readlane(l.len, b)};
    tile = tiles_of(s) - 1 - rank;
    parts = split_parts(tile_steps(s, tile), S);
    slots = end - size + rank;
    if (parts > 1)
      for (uint64_t todo = mine & ((1ULL << b) - 1); todo; todo &= todo - 1) slots += in_layer(__builtin_ctzll(todo));
  } else {
    const auto block_scan = [&](int x, int y, int* ex, int* ey, int* allx, int* ally) {
      const int u = wave_incl(x), v = wave_incl(y);
      block_sync_lds();  // the last round's sums have been read
      if (lane == 63) {
        s_sum[w] = u;
        s_sum[4 + w] = v;
      }
      block_sync_lds();
      *ex = u; *ey = v; *allx = *ally = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        *ex += i < w ? s_sum[i] : 0;
        *ey += i < w ? s_sum[4 + i] : 0;
        *allx += s_sum[i];
        *ally += s_sum[4 + i];
      }
    };
    // More: every tile of a sequence in as many parts as its last, by the batch's lengths alone (the table's
    // room for 2^20 positions in their place left a chunk of 512 tokens after 4097 beside 64 decode steps
    // whole: 108 us instead of 56; with 63 beside it, planned above, 50).
    int S = 0, W = 0, beside = 0, most = 0, items, splits;
    long long tiles = 0;
    for (int g = 0; g < a.r.n; g += 256) {
      const int b = g + t;
      SeqSpan l = {0, 0, 0, 0};
      if (b < a.r.n) l = seq_span(a.p, a.r, b);
      int ex, ey, aw, at;
      most = max(most, tiles_of(l) ? steps_of(l.len) : 0);
      block_scan(work_of(l), beside_of(l), &ex, &ey, &aw, &at);
      W += aw;
      beside += at;
      block_scan(tiles_of(l) & 0xFFF, tiles_of(l) >> 12, &ex, &ey, &aw, &at);
      tiles += aw + ((long long)at << 12);
    }
    if (tiles == 0 || tiles > most_tiles) return;
#pragma unroll
    for (int m = 32; m; m >>= 1) most = max(most, __shfl_xor(most, m));
    block_sync_lds();  // the last round's sums have been read
    if (lane == 0) s_sum[w] = most;
    block_sync_lds();
    most = max(max(s_sum[0], s_sum[1]), max(s_sum[2], s_sum[3]));
    for (S = share(W, most, beside);; S += (S + 3) / 4) {
      items = splits = 0;
      for (int g = 0; g < a.r.n; g += 256) {
        const int b = g + t;
        SeqSpan l = {0, 0, 0, 0};
        if (b < a.r.n) l = seq_span(a.p, a.r, b);
        const int np = split_parts(steps_of(l.len), S), n = tiles_of(l) * np;
        int ex, ey, ax, ay;
        block_scan(n, np > 1 ? n : 0, &ex, &ey, &ax, &ay);
        if (b < a.r.n) {
          s_end[b] = items + ex;
          s_split[b] = splits + ey;
        }
        items += ax;
        splits += ay;
      }
      if (splits <= a.max_splits) break;
    }
    block_sync_lds();
    if (idx >= items) return;
    const auto lds_at = [&](const int* p) { return __builtin_amdgcn_readfirstlane(*p); };
    int b = 0;
    for (int hi = a.r.n - 1; b < hi;) {
      const int mid = (b + hi) >> 1;
      if (lds_at(s_end + mid) > idx) hi = mid; else b = mid + 1;
    }
    s = seq_span(a.p, a.r, b);
    s.row = __builtin_amdgcn_readfirstlane(s.row);
    s.first = __builtin_amdgcn_readfirstlane(s.first);
    s.count = __builtin_amdgcn_readfirstlane(s.count);
    s.len = __builtin_amdgcn_readfirstlane(s.len);
    parts = split_parts(steps_of(s.len), S);
    const int nt = tiles_of(s), in = idx - (lds_at(s_end + b) - nt * parts);
    tile = nt - 1 - in / parts;  // a sequence's last tiles, which see the most, first
    part = in % parts;
    slots = lds_at(s_split + b) - (tile + 1) * parts + lane;
  }
  const int rows = s.count * G, row0 = tile * kTile + 32 * w;  // this wave's first row
  const int old = s.len - s.count;
  const int kend = old + (min(rows, (tile + 1) * kTile) - 1) / G + 1;
  const int steps = steps_of(kend), st0 = part * steps / parts, st1 = (part + 1) * steps / parts;
  const bool active = row0 < rows;  // the wave has rows

  // the first tiles' pages, the query rows and the first tile are on their way together
  const int32_t* tab = a.p.table + (size_t)s.row * a.p.max_pages;
  const int shift = a.p.page_shift, inpage = (1 << shift) - 1;
  const auto pages_at = [&](int st) {  // lanes 16 i ..: the page of the step's 16 i .. + 15
    const int pos = st * kKeys + 16 * (lane >> 4);
    return tab[min(pos >> shift, a.p.max_pages - 1)];
  };
  int pages = pages_at(st0), pages_next = pages_at(st0 + 1);

  // Q^T operand: lane (row l % 32, half l / 32) holds dims 16 i + 8 half .. + 7
  const int qc = lane & 31, hf = lane >> 5;
  const int row = min(row0 + qc, rows - 1), tok = row / G, head = j * G + row - tok * G;
  const int qpos = old + tok;
  const int first_hidden = old + min(row0, rows - 1) / G + 1;  // hidden from some row of the wave
  u32x4 q[KS];
  {
    const uint16_t* qp = a.q + (s.first + tok) * a.q_stride + head * D + 8 * hf;
#pragma unroll
    for (int i = 0; i < KS; ++i) q[i] = *reinterpret_cast<const u32x4*>(qp + 16 * i);
  }
  // Scores are scaled as they enter the exponential, hidden ones at -Inf by then: the scale is positive, its
  // sign and a scale of 0 go to the query.
  const float scale = a.scale == 0.f ? 1.f : fabsf(a.scale);

  // ---- K / V tiles ---------------------------------------------------------------------------
  constexpr int RI = 64 / LR;  // rows a DMA instruction
  const int drow = lane / LR, dslot = lane % LR;
  const auto kswz = [](int r) { return D == 128 ? r & 15 : (r >> 1) & 7; };
  const auto vswz = [](int r) { return D == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1); };
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  uint32_t kfrom[16 / RI], vfrom[16 / RI];  // slot s of row r is column group s ^ swz(r)
#pragma unroll
  for (int i = 0; i < 16 / RI; ++i) {
    const int r = i * RI + drow;
    kfrom[i] = r * kRowBytes + ((dslot ^ kswz(r)) << 4);
    vfrom[i] = r * kRowBytes + ((dslot ^ vswz(r)) << 4);
  }
  uint64_t gone = 0;  // 16-row groups of the tile last issued whose page is not there (bits 16 i)
  bool bad_page = false;
  const auto issue = [&](int st, int sg) {
    const int pos = st * kKeys + 16 * w;
    const int page = __builtin_amdgcn_readlane(pages, 16 * w);
    gone = __ballot(!in_range(pages, a.p.num_pages) && st * kKeys + 16 * (lane >> 4) < kend);
    char* to = lds + sg * kStage + 16 * w * kRowBytes;
    if (pos >= kend || !in_range(page, a.p.num_pages)) {  // nothing there: zeros
      bad_page |= pos < kend;
#pragma unroll
      for (int i = 0; i < 16 / RI; ++i) {
        *reinterpret_cast<u32x4*>(to + i * 1024 + 16 * lane) = u32x4{0u, 0u, 0u, 0u};
        *reinterpret_cast<u32x4*>(to + kPlane + i * 1024 + 16 * lane) = u32x4{0u, 0u, 0u, 0u};
      }
    } else {
      const size_t at = page_elem(a.p, page, j) + (size_t)(pos & inpage) * D;
      const uint16_t* kp = a.kplane + at;
      const uint16_t* vp = a.vplane + at;
      const uint32_t l0 = __builtin_amdgcn_readfirstlane(lds0 + sg * kStage + 16 * w * kRowBytes);
      const int last = kend - 1 - pos;
      if (last >= 15) {
#pragma unroll
        for (int i = 0; i < 16 / RI; ++i) {
          dma16(kp, kfrom[i], l0 + i * 1024);
          dma16(vp, vfrom[i], l0 + kPlane + i * 1024);
        }
      } else {  // rows past the last position repeat it (masked)
#pragma unroll
        for (int i = 0; i < 16 / RI; ++i) {
          const uint32_t up = max(i * RI + drow - last, 0) * kRowBytes;
          dma16(kp, kfrom[i] - up, l0 + i * 1024);
          dma16(vp, vfrom[i] - up, l0 + kPlane + i * 1024);
        }
      }
    }
  };
  uint32_t ko[KS], vo[DT];  // K: row l % 32, slot 2 i + half; V: 4 dims of key 4 half + l % 16 / 4
#pragma unroll
  for (int i = 0; i < KS; ++i) ko[i] = qc * kRowBytes + (((2 * i + hf) ^ kswz(qc)) << 4);
  {
    const int i = lane & 15, key = 4 * hf + (i >> 2), db = (lane >> 4) & 1;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      vo[dt] = kPlane + key * kRowBytes + (((4 * dt + 2 * db + ((i >> 1) & 1)) ^ vswz(key)) << 4) + 8 * (i & 1);
  }

  f32x16 o[DT];
  float m, l;  // l of this lane's keys only
  const int per = (st1 - st0 + 63) / 64;

  // Step `st`, in LDS stage SG (the loop takes two at a time, so that operand addresses are immediates).
  const auto take = [&](int st, auto stage_no, auto again) {
    constexpr int SG = decltype(stage_no)::value;
    const char* stage = lds + SG * kStage;
    const int key0 = st * kKeys;
    const uint64_t none = gone;
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) expcnt(7) lgkmcnt(0): this wave's rows are there
    if constexpr (again) {
      bool odd = false;
#pragma unroll
      for (int i = 0; i < 16 / RI; ++i) {
        u32x4* at = reinterpret_cast<u32x4*>(lds + SG * kStage + kPlane + 16 * w * kRowBytes + i * 1024 + 16 * lane);
        u32x4 v = *at;
        if (drop_odd<BF>(v)) {
          *at = v;
          odd = true;
        }
      }
      if (odd) atomicOr(s_odd, 1ULL << ((st - st0) / per));
      __builtin_amdgcn_s_waitcnt(0xc07f);
    }
    __builtin_amdgcn_s_barrier();  // everybody's rows are there, and the other stage is read
    asm volatile("" ::: "memory");
    if (st + 1 < st1) {
      issue(st + 1, SG ^ 1);
      pages = pages_at(st + 2);
    }
    if (!active || key0 > old + min(row0 + 31, rows - 1) / G) return;  // nothing the wave's rows see
    f32x16 x[2];
    {
      u32x4 kop[KS][2];  // all of the tile's operands on their way before the first product waits
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) kop[i][h] = *reinterpret_cast<const u32x4*>(stage + ko[i] + 32 * h * kRowBytes);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          x[h] = mfma32<BF>(kop[i][h], q[i], i ? x[h] : zero);
        }
    }
    // V^T operands of 16 keys: dims 32 dt + l % 32, the lane's eight keys of 16 i ..
    const auto load_v = [&](int i, u32x4 (&v)[DT]) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const u32x2 v0 = read_tr4(stage + vo[dt] + 16 * i * kRowBytes);
        const u32x2 v1 = read_tr4(stage + vo[dt] + (16 * i + 8) * kRowBytes);
        v[dt] = u32x4{v0[0], v0[1], v1[0], v1[1]};
      }
    };
    u32x4 v[2][DT];
    load_v(0, v[0]);
    // lane holds keys 32 h + 8 (r / 4) + 4 half + r % 4
    if (key0 + kKeys > first_hidden || none) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = 32 * h + 8 * (r >> 2) + 4 * hf + (r & 3);
          if (key0 + key > qpos || (none >> (16 * (2 * h + (r >> 3))) & 1)) x[h][r] = -INFINITY;
        }
    }
    float mx = x[0][0];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, x[h][r]);
    mx = halves<false>(mx) * scale;
    if constexpr (BF && again) mx += kHeadroom;
    const bool move = mx > m + kRescale || (m == -INFINITY && mx > m);
    if (__ballot(move)) {
      const float mn = move ? mx : m;
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= f;
    }
    const float ms = m == -INFINITY ? 0.f : m;
    // the lane's eight probabilities of each 16 keys, as value and remainder; l sums them unrounded
    const auto probs = [&](int i, u32x4& p, u32x4& rest) {
      float e[8], sum = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        e[k] = __builtin_amdgcn_exp2f(fmaf(x[i >> 1][8 * (i & 1) + k], scale, -ms));
        sum += e[k];
      }
      l += sum;
      pack8_rest<BF>(e, p, rest);
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < 3) load_v(i + 1, v[(i + 1) & 1]);
      u32x4 p, rest;
      probs(i, p, rest);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] = mfma32<BF>(v[i & 1][dt], p, o[dt]);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] = mfma32<BF>(v[i & 1][dt], rest, o[dt]);
    }
  };
  const auto pass = [&](auto again) {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
    for (int st = st0; st < st1; st += 2) {
      take(st, std::integral_constant<int, 0>(), again);
      if (st + 1 < st1) take(st + 1, std::integral_constant<int, 1>(), again);
    }
    l = halves<true>(l);
  };
  if (st0 < st1) issue(st0, 0);
  pages = pages_next;
  if (a.scale < 0.f) {
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) q[i][e] ^= 0x80008000u;
  } else if (a.scale == 0.f) {  // (Inf x 0 is NaN)
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = 0.f * to_f32<BF>((uint16_t)(e & 1 ? q[i][e >> 1] >> 16 : q[i][e >> 1]));
      q[i] = pack8<BF>(y);
    }
  }
  pass(std::false_type());
  float zero = 0.f;  // NaN if a sum is Inf or NaN
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) zero = fmaf(o[dt][r], 0.f, zero);
  s_again[w] = __ballot(zero != 0.f) != 0;
  if (t == 0) *s_odd = 0;
  __syncthreads();
  if (__builtin_expect(s_again[0] | s_again[1] | s_again[2] | s_again[3], 0)) {  // (then the part has steps)
    pages = pages_at(st0);
    issue(st0, 0);
    pages = pages_at(st0 + 1);
    pass(std::true_type());
    __syncthreads();
    if (active)
      for (uint64_t odd = *s_odd; odd; odd &= odd - 1) {
        const int key0 = (st0 + __builtin_ctzll(odd) * per) * kKeys;
        for (int key = key0; key < min(min(st1 * kKeys, key0 + per * kKeys), kend); ++key) {
          const int page = tab[min(key >> shift, a.p.max_pages - 1)];
          if (!in_range(page, a.p.num_pages)) continue;
          const size_t at = page_elem(a.p, page, j) + (size_t)(key & inpage) * D;
          float score = 0.f;
#pragma unroll
          for (int i = 0; i < KS; ++i)
            score += dot8<BF>(q[i], *reinterpret_cast<const u32x4*>(a.kplane + at + 16 * i + 8 * hf));
          const bool none = halves<true>(score) * scale == -INFINITY;  // the weight is 0
          if (key > qpos) continue;
          m = fmaxf(m, -FLT_MAX);  // (joined whatever the scores are)
          l = with_sign(l, 0x80000000u);
          const uint16_t* v = a.vplane + at + 4 * hf;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const float x = to_f32<BF>(v[32 * dt + 8 * (r >> 2) + (r & 3)]);
              if (not_finite(x)) o[dt][r] += none ? NAN : x;
            }
        }
      }
  }
  if (bad_page && lane == 0) atomicOr(a.p.status, Q4D_STATUS_BAD_PAGE);

  // ---- parts, joined as in rows_part; a lane's values lie together by fours ---------------------
  const KernelArgs late = late_args();
  int count = parts, at_part = part;
  for (int level = 0, step = 1; count > 1; ++level, step *= kJoin) {
    const int first = at_part / kJoin * kJoin, size = min(kJoin, count - first);
    const auto slot = [&](int i) { return (size_t)__builtin_amdgcn_readlane(slots, i * step) * kvh + j; };
    const auto place = [&](int i) { return slot(i) * 4 + w; };
    if (size > 1) {
      if (active) {
        const auto acc = rows_rsrc(late->cacc + place(at_part) * (32 * D), 32 * D * 4);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; r += 4)
            store_dev4(acc, (16 * dt + r) * 256 + 16 * lane, f32x4{o[dt][r], o[dt][r + 1], o[dt][r + 2], o[dt][r + 3]});
        store_dev(late->cml + place(at_part) * 64 + lane, hf ? l : m);
      }
      __builtin_amdgcn_s_waitcnt(0);  // this thread's stores are performed
      __syncthreads();                // ... and every other thread's
      int* counter = late->ccounters + level * kChunkCounters + slot(first);
      if (t == 0) *s_last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == size - 1;
      __syncthreads();
      if (!*s_last) return;
      if (t == 0) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // next call
      if (active) {
        const auto ml = [&](int i) { return late->cml + place(first + i) * 64 + qc; };
        float M = -INFINITY;
        uint32_t sign = 0;
#pragma unroll
        for (int i = 0; i < kJoin; ++i) M = fmaxf(M, load_dev(ml(min(i, size - 1))));
        M = join_max<BF>(M);
        l = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
        // two parts' values are in flight together
        for (int i0 = 0; i0 < size; i0 += 2) {
          f32x4 v[2][4 * DT];
          float mv[2], lv[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int i = min(i0 + k, size - 1);
            mv[k] = load_dev(ml(i));
            lv[k] = load_dev(ml(i) + 32);
            const auto acc = rows_rsrc(late->cacc + place(first + i) * (32 * D), 32 * D * 4);
#pragma unroll
            for (int n = 0; n < 4 * DT; ++n) v[k][n] = load_dev4(acc, n * 1024 + 16 * lane);
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (i0 + k >= size) break;
            const float f = join_factor(mv[k], lv[k], M);
            l = fmaf(fabsf(lv[k]), f, l);
            sign |= sign_of(lv[k]);
#pragma unroll
            for (int n = 0; n < 4 * DT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float y = o[n >> 2][4 * (n & 3) + e];
                o[n >> 2][4 * (n & 3) + e] = fmaf(v[k][n][e], f, y);
              }
          }
        }
        l = with_sign(l, sign);
        m = M;
      }
      __syncthreads();  // s_last has been read
    }
    at_part = first / kJoin;
    count = (count + kJoin - 1) / kJoin;
  }

  // ---- rows out, through LDS -------------------------------------------------------------------
  __syncthreads();  // everybody is done with the tiles
  if (!active) return;
  const float inv = inverse_sum(l, a.p, tab, qpos);
  char* T0 = lds + w * (32 * kRowBytes);  // 32 rows of D values, slot s of row r at s ^ (r & (LR - 1))
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u0 = from_f32<BF>(o[dt][4 * i] * inv), u1 = from_f32<BF>(o[dt][4 * i + 1] * inv);
      const uint32_t u2 = from_f32<BF>(o[dt][4 * i + 2] * inv), u3 = from_f32<BF>(o[dt][4 * i + 3] * inv);
      *reinterpret_cast<u32x2*>(T0 + qc * kRowBytes + (((4 * dt + i) ^ (qc & (LR - 1))) << 4) + 8 * hf) =
          u32x2{u0 | u1 << 16, u2 | u3 << 16};
    }
#pragma unroll
  for (int i = 0; i < 32 / RI; ++i) {
    const int r = i * RI + drow, rr = row0 + r;
    if (rr >= rows) continue;
    const int tk = rr / G;
    *reinterpret_cast<u32x4*>(late->out + (s.first + tk) * late->out_stride + (j * G + rr - tk * G) * D + 8 * dslot) =
        *reinterpret_cast<const u32x4*>(T0 + r * kRowBytes + ((dslot ^ (r & (LR - 1))) << 4));
  }
}

template <int D, bool BF, int R>
__global__ __launch_bounds__(256, 2) void rows_kernel(const PagedAttnArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[Shared<D>::kRowsV + Shared<D>::kMore];
  extern __shared__ int seqs[];
  rows_part<D, BF, R>(a, lds, seqs, blockIdx.x);
}

// Both: the first blocks * kvh blocks take the sequences of few rows, which stream K and V, and run
// beside the others, which compute: 38 decode steps of up to 3000 positions and two chunks of up to 700 tokens
// 86 us (as two launches, one after the other, they took 7 us more than together).
template <int D, bool BF>
__global__ __launch_bounds__(256, 2) void chunk_kernel(const PagedAttnArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[Shared<D>::kChunkV + Shared<D>::kMore];
  extern __shared__ int seqs[];
  const int rows = a.blocks * a.p.kvh;
  if ((int)blockIdx.x < rows) rows_part<D, BF, 1>(a, lds, seqs, blockIdx.x);
  else chunk_part<D, BF>(a, lds, seqs, blockIdx.x - rows);
}

// Blocks per kv head of rows_part.
int rows_blocks(int kvh) { return max(1, min(device_cus(), kCounters) / kvh); }
// Blocks per kv head that chunk_part's parts are to fill: two a CU.  Tiles in parts have 4/3 of that
// many parts at most: round(n / S) is at most n / S + 1/2, and two or more says n / S >= 3/2.
int chunk_slots(int kvh) { return max(1, 2 * min(device_cus(), kChunkCounters / 4) / kvh); }
int chunk_splits(int kvh) { return chunk_slots(kvh) * 4 / 3 + 1; }

// The counters lie at the same place for every shape, since calls of several may share a workspace.
struct Layout {
  size_t pml, pacc, cml, cacc, total;
};
Layout layout(int kvh, int d, bool chunks) {
  Layout l;
  const size_t slots = 2 * (size_t)rows_blocks(kvh) * kvh, items = chunks ? (size_t)chunk_splits(kvh) * kvh : 0;
  l.pml = paged_attention_ws_counters();
  l.pacc = l.pml + align_up(slots * 2 * kRows * 2 * 4, 256);
  l.cml = l.pacc + align_up(slots * 2 * kRows * d * 4, 256);
  l.cacc = l.cml + align_up(items * kTile * 2 * 4, 256);
  l.total = l.cacc + items * kTile * d * 4;
  return l;
}
// Groups of 16 query rows that the batch's sequences have at most: rows_part takes all of them if that is one
// or two, else (0) the sequences of one, and chunk_part the others.  Two groups beside chunks, or in the
// kernel for one, cost that one 3 to 12 % (mixed 94.6 / 97, 64 decode steps 128.3 / 133.3, one 8.7 / 9.8 us).
int row_groups(int qh, int kvh, int max_new) {
  const long long rows = (long long)max_new * (qh / kvh);
  return rows <= kRows ? 1 : rows <= 2 * kRows ? 2 : 0;
}
bool has_chunks(int qh, int kvh, int max_new) { return row_groups(qh, kvh, max_new) == 0; }

template <int D, bool BF>
int launch(const PagedAttnArgs& a, hipStream_t st) {
  const int kvh = a.p.kvh, G = a.qh / kvh;
  const size_t seqs = a.r.n > kLanes ? (size_t)a.r.n * 16 : 0;
  const long long rows = (long long)a.blocks * kvh;
  if (const int groups = row_groups(a.qh, kvh, a.r.max_new)) {
    if (groups == 1) hipLaunchKernelGGL((rows_kernel<D, BF, 1>), dim3((unsigned)rows), dim3(256), seqs, st, a);
    else hipLaunchKernelGGL((rows_kernel<D, BF, 2>), dim3((unsigned)rows), dim3(256), seqs, st, a);
    return check_launch();
  }
  // items: tiles, and more parts of them at most chunk_splits
  const long long items = tiles_most(a.r.tokens, G, a.r.n) + chunk_splits(kvh);
  if (rows + items * kvh > kMaxBlocks) return Q4D_ERR_SHAPE;
  hipLaunchKernelGGL((chunk_kernel<D, BF>), dim3((unsigned)(rows + items * kvh)), dim3(256), seqs, st, a);
  return check_launch();
}

}  // namespace

size_t paged_attention_ws_counters() { return (kLevels * kCounters + kLevels * kChunkCounters) * 4; }
size_t paged_attention_ws_bytes(int kvh, int d, int qh, int, int, int max_new) {
  return layout(kvh, d, has_chunks(qh, kvh, max_new)).total;
}

int launch_paged_attention(const PagedAttnArgs& args, hipStream_t st) {
  PagedAttnArgs a = args;
  const Layout l = layout(a.p.kvh, a.p.d, has_chunks(a.qh, a.p.kvh, a.r.max_new));
  a.counters = ws_ptr<int>(a.ws, 0);
  a.ccounters = a.counters + kLevels * kCounters;
  a.pml = ws_ptr<float>(a.ws, l.pml);
  a.pacc = ws_ptr<float>(a.ws, l.pacc);
  a.cml = ws_ptr<float>(a.ws, l.cml);
  a.cacc = ws_ptr<float>(a.ws, l.cacc);
  a.blocks = rows_blocks(a.p.kvh);
  a.slots = chunk_slots(a.p.kvh);
  a.max_splits = chunk_splits(a.p.kvh);
  if (a.p.d == 128) return a.bf16 ? launch<128, true>(a, st) : launch<128, false>(a, st);
  return a.bf16 ? launch<64, true>(a, st) : launch<64, false>(a, st);
}

}  // namespace q4d
