// Attention of a ragged batch's new tokens over a paged KV cache (gfx950, wave64).
//
// One wave per (token, q head): the lanes hold D / 64 dims each and walk the positions with an
// online softmax (running maximum and sum).
#include <math.h>

#include "q4d_device.h"
#include "q4d_paged.h"

namespace q4d {

namespace {

template <bool BF>
__device__ __forceinline__ float to_f32(uint16_t u) {
  if constexpr (BF) return __builtin_bit_cast(float, (uint32_t)u << 16);
  else return (float)__builtin_bit_cast(_Float16, u);
}

template <int D, bool BF>
__global__ __launch_bounds__(256) void paged_attn_simple(const PagedAttnArgs a) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int b = blockIdx.x;
  const SeqSpan s = seq_span(a.p, a.r, b);
  if (s.count <= 0) {
    if (s.count < 0 && blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0)
      atomicOr(a.p.status, Q4D_STATUS_BAD_SEQUENCE);
    return;
  }
  const int h = blockIdx.y, j = h / (a.qh / a.p.kvh);
  const int32_t* tab = a.p.table + (size_t)s.row * a.p.max_pages;
  for (int i = blockIdx.z * 4 + w; i < s.count; i += 4 * gridDim.z) {
    const size_t tok = s.first + i;
    float q[E], o[E], m = -INFINITY, l = 0.f;
    for (int e = 0; e < E; ++e) {
      q[e] = to_f32<BF>(a.q[tok * a.q_stride + h * D + lane * E + e]) * a.scale;
      o[e] = 0.f;
    }
    const int end = s.len - s.count + i + 1;
    for (int pos = 0; pos < end; ++pos) {
      const int page = tab[pos >> a.p.page_shift];
      if (!in_range(page, a.p.num_pages)) {
        if (lane == 0) atomicOr(a.p.status, Q4D_STATUS_BAD_PAGE);
        continue;
      }
      const size_t at = page_elem(a.p, page, j) + (size_t)(pos & ((1 << a.p.page_shift) - 1)) * D + lane * E;
      float x = 0.f;
      for (int e = 0; e < E; ++e) x = fmaf(q[e], to_f32<BF>(a.kplane[at + e]), x);
      x = wave_sum(x);
      const float mn = fmaxf(m, x), f = m == -INFINITY ? 0.f : exp2f(m - mn), pr = exp2f(x - mn);
      l = fmaf(l, f, pr);
      for (int e = 0; e < E; ++e) o[e] = fmaf(o[e], f, pr * to_f32<BF>(a.vplane[at + e]));
      m = mn;
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    for (int e = 0; e < E; ++e) {
      const float y = o[e] * inv;
      a.out[tok * a.out_stride + h * D + lane * E + e] =
          BF ? __builtin_bit_cast(uint16_t, (__bf16)y) : __builtin_bit_cast(uint16_t, (_Float16)y);
    }
  }
}

}  // namespace

size_t paged_attention_ws_bytes(int, int, int, int, int, int) { return 256; }

int launch_paged_attention(const PagedAttnArgs& a, hipStream_t st) {
  const dim3 grid(a.r.n, a.qh, (unsigned)min((a.r.max_new + 3) / 4, 1024));
  if (a.p.d == 128) {
    if (a.bf16) hipLaunchKernelGGL((paged_attn_simple<128, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_attn_simple<128, false>), grid, dim3(256), 0, st, a);
  } else {
    if (a.bf16) hipLaunchKernelGGL((paged_attn_simple<64, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_attn_simple<64, false>), grid, dim3(256), 0, st, a);
  }
  return check_launch();
}

}  // namespace q4d
