// The paged KV cache as its kernels see it: descriptors by value, and the checks of what only
// the device knows (sequences, counts, pages).  The checks are host functions too, so that they
// can be tested without a device.
#pragma once

#include "q4d_internal.h"

namespace q4d {

struct PagedView {
  uint16_t* data;  // [num_layers][2][num_pages][kvh][page_size][d]
  int32_t* table;
  int32_t* lengths;
  int32_t* refs;
  int32_t* status;
  int num_layers, num_pages, kvh, page_shift, d, num_seqs, max_pages;
  int max_ctx;  // positions that a row may grow to
};

struct RaggedView {
  const int32_t* seqs;
  const int32_t* starts;
  int n, tokens, max_new;
};

// New tokens [first, first + count) of the token rows, the last of table row `row`'s `len`
// positions.  count 0: nothing to do; count < 0: cannot be (Q4D_STATUS_BAD_SEQUENCE).
struct SeqSpan {
  int row, first, count, len;
};

__host__ __device__ inline int seq_count(int s0, int s1, int tokens, int max_new) {
  return s0 >= 0 && s0 <= s1 && s1 <= tokens && s1 - s0 <= max_new ? s1 - s0 : -1;
}
__host__ __device__ inline bool in_range(int i, int n) { return (unsigned)i < (unsigned)n; }

// Span of batch entry b (in [0, n)) whose new tokens are already counted in lengths.
__host__ __device__ inline SeqSpan seq_span(const PagedView& p, const RaggedView& r, int b) {
  const int s0 = r.starts[b], s1 = r.starts[b + 1];
  SeqSpan s = {0, s0, seq_count(s0, s1, r.tokens, r.max_new), 0};
  if (s.count <= 0) return s;
  s.row = r.seqs ? r.seqs[b] : b;
  if (!in_range(s.row, p.num_seqs)) {
    s.count = -1;
    return s;
  }
  s.len = p.lengths[s.row];
  if (s.len < s.count || s.len > p.max_pages << p.page_shift) s.count = -1;
  return s;
}

#ifdef __HIPCC__
// Inclusive sum over the lanes of a wave (DPP row shifts, then the row totals).
__device__ __forceinline__ int wave_incl(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast 15 into rows 1, 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast 31 into rows 2, 3
  return x;
}
#endif

// Elements of one (layer, K or V) plane, and the first element of a page's rows of kv head j.
__host__ __device__ inline size_t plane_elems(const PagedView& p) {
  return ((size_t)p.num_pages * p.kvh * p.d) << p.page_shift;
}
__host__ __device__ inline size_t page_elem(const PagedView& p, int page, int j) {
  return (((size_t)page * p.kvh + j) << p.page_shift) * p.d;
}

constexpr long long kMaxBlocks = (1 << 24) - 1;  // of 256 threads: a launch has fewer than 2^32

// Host: the descriptors' checks (Q4D_OK or an error code).
int check_pages(const q4d_pages_t* p);
int check_ragged(const q4d_ragged_t* r);
PagedView paged_view(const q4d_pages_t* p);
RaggedView ragged_view(const q4d_ragged_t* r);

// Attention over the pages (q4d_paged_attn.hip).
struct PagedAttnArgs {
  PagedView p;
  RaggedView r;
  const uint16_t* q;
  uint16_t* out;
  long long q_stride, out_stride;
  const uint16_t* kplane;
  const uint16_t* vplane;
  float scale;  // scaling * log2(e)
  int qh, bf16;
  void* ws;
  // set by launch_paged_attention
  // of rows_part
  int* counters;  // parts that have arrived, by join level and block
  float* pml;     // [block][2 slots][kvh][16 or 32 rows][m, l]
  float* pacc;    // [block][2 slots][kvh][16 or 32 rows][d]
  int blocks;     // per kv head
  // of chunk_part
  int* ccounters;  // by join level and part
  float* cml;     // [parts][kvh][4 waves][m, l of 32 rows]
  float* cacc;    // [parts][kvh][4 waves][32 x d]
  int slots, max_splits;  // per kv head: blocks that parts are to fill, parts at most
};
size_t paged_attention_ws_bytes(int kvh, int d, int qh, int n, int tokens, int max_new);
size_t paged_attention_ws_counters();  // bytes at the workspace's start that are zero between calls
int launch_paged_attention(const PagedAttnArgs& a, hipStream_t st);

}  // namespace q4d
