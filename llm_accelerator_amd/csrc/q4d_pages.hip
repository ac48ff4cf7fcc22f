// Pages of the paged KV cache: reserving, forking, truncating and compacting them, and the append
// of a ragged batch's k / v rows (with the head norm and rotation of q and k).
//
// The integers (table, lengths, refs) stay on the device, so that a captured step can take pages
// without the host.  A page is free when its refs are 0; the free pages of the lowest numbers go
// first, in the order of the batch, which makes every call's result a function of its inputs: no
// stack of free pages whose order depends on the past, no atomics whose order matters (refs are
// sums, the keeper of a shared page a maximum).
#include <string.h>

#include "q4d_device.h"
#include "q4d_paged.h"

namespace q4d {

int check_pages(const q4d_pages_t* p) {
  if (!p || !p->data || !p->table || !p->lengths || !p->refs || !p->status) return Q4D_ERR_NULL;
  if (p->dtype != Q4D_F16 && p->dtype != Q4D_BF16) return Q4D_ERR_DTYPE;
  const int ps = p->page_size;
  if (ps != 16 && ps != 32 && ps != 64 && ps != 128 && ps != 256) return Q4D_ERR_SHAPE;
  if (p->head_dim != 64 && p->head_dim != 128) return Q4D_ERR_SHAPE;
  if (p->num_layers <= 0 || p->num_pages <= 0 || p->num_pages > 1 << 22 || p->num_kv_heads <= 0 ||
      p->num_kv_heads > 256 || p->num_seqs <= 0 || p->num_seqs > 65536 || p->max_pages <= 0 ||
      (long long)p->max_pages * ps > 1 << 24 || p->max_ctx < 0 || p->max_ctx > p->max_pages * ps)
    return Q4D_ERR_SHAPE;
  if (!aligned(p->data, 16) || !aligned(p->table, 4) || !aligned(p->lengths, 4) || !aligned(p->refs, 4) ||
      !aligned(p->status, 4))
    return Q4D_ERR_BAD_ADDR;
  return Q4D_OK;
}

int check_ragged(const q4d_ragged_t* r) {
  if (!r || !r->starts) return Q4D_ERR_NULL;
  if (r->n <= 0 || r->n > 4096 || r->tokens <= 0 || r->tokens > 1 << 24 || r->max_new <= 0) return Q4D_ERR_SHAPE;
  if (!aligned(r->starts, 4) || !aligned(r->seqs, 4)) return Q4D_ERR_BAD_ADDR;
  return Q4D_OK;
}

PagedView paged_view(const q4d_pages_t* p) {
  PagedView v;
  v.data = static_cast<uint16_t*>(p->data);
  v.table = p->table;
  v.lengths = p->lengths;
  v.refs = p->refs;
  v.status = p->status;
  v.num_layers = p->num_layers;
  v.num_pages = p->num_pages;
  v.kvh = p->num_kv_heads;
  v.page_shift = __builtin_ctz((unsigned)p->page_size);
  v.d = p->head_dim;
  v.num_seqs = p->num_seqs;
  v.max_pages = p->max_pages;
  v.max_ctx = p->max_ctx ? p->max_ctx : p->max_pages * p->page_size;
  return v;
}

RaggedView ragged_view(const q4d_ragged_t* r) { return {r->seqs, r->starts, r->n, r->tokens, r->max_new}; }

namespace {

constexpr int kMaxBatch = 4096;

// Workspace of the page calls: the list of page rows to copy, and a few ints per page.
struct PageWs {
  int32_t* copies;  // [1] number of entries of src / dst / rows
  int32_t* ids;     // [num_pages] compact: holes in order
  int32_t* a;       // [num_pages] compact: movers in order
  int32_t* b;       // [num_pages] compact: where a page goes
  int32_t *src, *dst, *rows;  // [max(num_pages, kMaxBatch)]
};

__host__ size_t page_ws_ints(int num_pages) {
  return 64 + 3 * (size_t)num_pages + 3 * (size_t)max(num_pages, kMaxBatch);
}
PageWs page_ws(void* ws, int num_pages) {
  PageWs w;
  const size_t np = num_pages, nl = max(num_pages, kMaxBatch);
  w.copies = static_cast<int32_t*>(ws);
  w.ids = w.copies + 64;
  w.a = w.ids + np;
  w.b = w.a + np;
  w.src = w.b + np;
  w.dst = w.src + nl;
  w.rows = w.dst + nl;
  return w;
}

__device__ __forceinline__ int load_now(const int32_t* p) {
  return __hip_atomic_load(const_cast<int32_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Sum over the waves below of the block's 16 and over all, of what each wave gives; `sums` int[16] of
// LDS, aligned to 16 bytes.
__device__ __forceinline__ int waves_excl(int wave_total, int t, int* sums, int* total) {
  typedef int i32x4 __attribute__((ext_vector_type(4)));
  block_sync_lds();  // the last call's sums have been read
  if ((t & 63) == 0) sums[t >> 6] = wave_total;
  block_sync_lds();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const i32x4 s = reinterpret_cast<const i32x4*>(sums)[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      before += 4 * i + e < (t >> 6) ? s[e] : 0;
      all += s[e];
    }
  }
  *total = all;
  return before;
}
// Exclusive sum over the block's 1024 threads and the block's total.
__device__ __forceinline__ int block_excl(int v, int t, int* sums, int* total) {
  const int incl = wave_incl(v);
  return waves_excl(__builtin_amdgcn_readlane(incl, 63), t, sums, total) + incl - v;
}

__device__ __forceinline__ int pages_of(int len, int shift) { return (len + (1 << shift) - 1) >> shift; }

// One block, since every decision hangs on all of them: the batch is at most 4096 sequences (four a
// thread, read once) and the refs a few 10,000 ints, of which a round looks at 16384 (a wave at 1024
// in a row, four loads a lane), the first of them read ahead.  What it costs is the chain of dependent
// reads (starts and seqs, lengths, the last page, its refs) and a round's scan: 7 us for 200 sequences that
// grow by a token, 10 where they take 2300 of 19000 pages.
// Shared last pages are few: they are counted in a hash table in LDS (by atomics on global memory it
// took 5 us more), whose place the list of free pages takes over.
constexpr int kRound = 16384;
constexpr int kIds = 16384;        // free pages listed at a time
constexpr int kSlots = kIds / 3;   // of the hash table, for up to kMaxBatch pages
static_assert(kSlots > kMaxBatch, "an empty slot ends every search");

__global__ __launch_bounds__(1024) void reserve_kernel(const PagedView p, const RaggedView r, const PageWs w) {
  constexpr int B = kMaxBatch / 1024;
  __shared__ uint32_t seen[65536 / 32];
  __shared__ int end[kMaxBatch];  // pages taken by sequences up to and with b
  __shared__ int row_of[kMaxBatch], have_of[kMaxBatch];  // have: pages held, bit 31: the last is copied first
  __shared__ int ids[kIds];
  __shared__ __attribute__((aligned(16))) int sums[16];
  __shared__ int s_err, s_copies;
  const int t = threadIdx.x, lane = t & 63;
  const int ps = 1 << p.page_shift;

  // Pages 1024 w + 256 i + 4 lane .. + 3 of a round, -1 past the pool.
  typedef int i32x4 __attribute__((ext_vector_type(4)));
  struct Refs {
    i32x4 v[4];
  };
  const auto load_round = [&](int p0) {
    Refs f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = p0 + (t >> 6) * 1024 + 256 * i + 4 * lane;
      if (at + 4 <= p.num_pages && ((uintptr_t)p.refs & 15) == 0) {
        f.v[i] = *reinterpret_cast<const i32x4*>(p.refs + at);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) f.v[i][e] = at + e < p.num_pages ? p.refs[at + e] : -1;
      }
    }
    return f;
  };
  const Refs ahead = load_round(0);

  int s0[B], count[B], row[B], len[B], last[B], refs[B];
#pragma unroll
  for (int i = 0; i < B; ++i) {
    const int b = t + 1024 * i;
    s0[i] = b < r.n ? r.starts[b] : 0;
    count[i] = b < r.n ? r.starts[b + 1] : 0;
    row[i] = b < r.n ? (r.seqs ? r.seqs[b] : b) : 0;
  }
  const int held_back = t ? 0 : *p.status & Q4D_STATUS_NOT_RESERVED;
  for (int i = t; i < 65536 / 32; i += 1024) seen[i] = 0;
  if (t == 0) s_err = s_copies = 0;
  __syncthreads();
  int err = held_back;
#pragma unroll
  for (int i = 0; i < B; ++i) {
    const int b = t + 1024 * i;
    count[i] = b < r.n ? seq_count(s0[i], count[i], r.tokens, r.max_new) : 0;
    len[i] = 0;
    if (count[i] == 0) continue;
    if (count[i] < 0 || !in_range(row[i], p.num_seqs)) {
      err |= Q4D_STATUS_BAD_SEQUENCE;
      count[i] = 0;
      continue;
    }
    if (atomicOr(&seen[row[i] >> 5], 1u << (row[i] & 31)) >> (row[i] & 31) & 1) err |= Q4D_STATUS_BAD_SEQUENCE;
    len[i] = p.lengths[row[i]];
  }
  const long long most = (long long)p.max_pages << p.page_shift;
  bool shared = false;
#pragma unroll
  for (int i = 0; i < B; ++i) {
    last[i] = -1;  // the partly filled last page
    refs[i] = 0;
    if (!count[i]) continue;
    if (len[i] < 0 || len[i] > most) {
      err |= Q4D_STATUS_BAD_SEQUENCE;
    } else if (len[i] + (long long)count[i] > p.max_ctx) {
      err |= Q4D_STATUS_BAD_POSITION;
    } else if (len[i] & (ps - 1)) {
      last[i] = p.table[(size_t)row[i] * p.max_pages + (len[i] >> p.page_shift)];
      if (!in_range(last[i], p.num_pages)) {
        err |= Q4D_STATUS_BAD_PAGE;
        last[i] = -1;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < B; ++i) {
    if (last[i] >= 0) refs[i] = p.refs[last[i]];
    shared |= refs[i] > 1;
  }
  if (err) atomicOr(&s_err, err);
  shared = __syncthreads_or(shared);
  if (s_err) {
    if (t == 0) {
      atomicOr(p.status, s_err | Q4D_STATUS_NOT_RESERVED);
      *w.copies = 0;
    }
    return;
  }
  // a page that several rows hold: how many of the batch, and which of them is the last
  int slot[B];
  int *key = ids, *holders = ids + kSlots, *last_of = ids + 2 * kSlots;
  if (shared) {
    for (int i = t; i < kSlots; i += 1024) {
      key[i] = last_of[i] = -1;
      holders[i] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < B; ++i) {
      if (refs[i] <= 1) continue;
      slot[i] = (uint32_t)last[i] * 2654435761u % kSlots;
      for (;;) {
        const int old = atomicCAS(&key[slot[i]], -1, last[i]);
        if (old == -1 || old == last[i]) break;
        slot[i] = slot[i] + 1 == kSlots ? 0 : slot[i] + 1;
      }
      atomicAdd(&holders[slot[i]], 1);
      atomicMax(&last_of[slot[i]], t + 1024 * i);
    }
    __syncthreads();
  }
  int total = 0;
#pragma unroll
  for (int i = 0; i < B; ++i) {
    const int b = t + 1024 * i;
    if (1024 * i >= r.n) break;
    const bool cow = refs[i] > 1 && !(holders[slot[i]] == refs[i] && last_of[slot[i]] == b);
    const int have = pages_of(len[i], p.page_shift);
    const int take = count[i] ? pages_of(len[i] + count[i], p.page_shift) - have + cow : 0;
    int sum;
    const int before = block_excl(take, t, sums, &sum);
    end[b] = total + before + take;
    row_of[b] = row[i];
    have_of[b] = have | (cow ? 1 << 31 : 0);
    total += sum;
  }

  // The free pages of the lowest numbers: a round's have the numbers from `found` on, and those below
  // base + kIds are listed in LDS.  (block_excl's barriers lie between the table's last use and this.)
  const auto collect = [&](const Refs& f, int p0, int found, int base) {
    const uint64_t below = lane ? ~0ULL >> (64 - lane) : 0;
    int first[4], wave_total = 0;  // of this lane's load i, in the wave's order: by load, lane, element
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      first[i] = wave_total;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t z = __ballot(f.v[i][e] == 0);
        first[i] += __popcll(z & below);
        wave_total += __popcll(z);
      }
    }
    int n;
    const int before = found - base + waves_excl(wave_total, t, sums, &n);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      int k = before + first[i];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (f.v[i][e] == 0) {
          if (k < kIds) ids[k] = p0 + (t >> 6) * 1024 + 256 * i + 4 * lane + e;
          ++k;
        }
    }
    return n;
  };
  int found = 0;  // all rounds that it takes, so that it is known whether there are enough
  for (int p0 = 0; p0 < p.num_pages && found < total; p0 += kRound)
    found += collect(p0 ? load_round(p0) : ahead, p0, found, 0);
  if (found < total) {
    if (t == 0) {
      atomicOr(p.status, Q4D_STATUS_NO_PAGES | Q4D_STATUS_NOT_RESERVED);
      *w.copies = 0;
    }
    return;
  }
  for (int base = 0; base < total; base += kIds) {
    if (base) {  // what is given is free no more, so the next ones are the lowest
      __syncthreads();
      found = base;
      for (int p0 = 0; p0 < p.num_pages && found < min(total, base + kIds); p0 += kRound)
        found += collect(load_round(p0), p0, found, base);
    }
    __syncthreads();  // ids (and end, row_of, have_of)
    for (int k = base + t; k < min(total, base + kIds); k += 1024) {
      const int id = ids[k - base];
      int lo = 0, hi = r.n - 1;  // the first b with end[b] > k
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (end[mid] > k) hi = mid; else lo = mid + 1;
      }
      const int b = lo, j = k - (b ? end[b - 1] : 0), have = have_of[b] & 0x7FFFFFFF, cow = have_of[b] < 0;
      int32_t* tab = p.table + (size_t)row_of[b] * p.max_pages;
      p.refs[id] = 1;
      if (cow && j == 0) {
        const int old = tab[have - 1], n = atomicAdd(&s_copies, 1);
        w.src[n] = old;
        w.dst[n] = id;
        w.rows[n] = p.lengths[row_of[b]] & (ps - 1);
        tab[have - 1] = id;
        atomicSub(&p.refs[old], 1);
      } else {
        tab[have + j - cow] = id;
      }
    }
  }
  __syncthreads();  // the copies have read the lengths, and are counted
#pragma unroll
  for (int i = 0; i < B; ++i)
    if (count[i]) p.lengths[row[i]] = len[i] + count[i];
  if (t == 0) *w.copies = s_copies;
}

// The listed pages' first rows[i] rows, in every layer, K and V: a unit is one head of one page.  70 whole
// pages of 28 layers and 8 heads (1.03 GB) move at 5.0 TB/s, a large copy's rate.
__device__ __forceinline__ void copy_pages(const PagedView& p, const PageWs& w, int block, int blocks) {
  const int planes = 2 * p.num_layers;
  const long long units = (long long)*w.copies * planes * p.kvh;
  for (long long u = block; u < units; u += blocks) {
    const int j = (int)(u % p.kvh);
    const long long v = u / p.kvh;
    const int plane = (int)(v % planes), i = (int)(v / planes);
    uint16_t* base = p.data + plane * plane_elems(p);
    const u32x4* src = reinterpret_cast<const u32x4*>(base + page_elem(p, w.src[i], j));
    u32x4* dst = reinterpret_cast<u32x4*>(base + page_elem(p, w.dst[i], j));
    const int n = w.rows[i] * p.d / 8;
    for (int e0 = threadIdx.x; e0 < n; e0 += 1024) {  // four loads in flight
      u32x4 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (e0 + 256 * k < n) x[k] = __builtin_nontemporal_load(src + e0 + 256 * k);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (e0 + 256 * k < n) __builtin_nontemporal_store(x[k], dst + e0 + 256 * k);
    }
  }
}

__global__ __launch_bounds__(256) void copy_kernel(const PagedView p, const PageWs w) {
  copy_pages(p, w, blockIdx.x, gridDim.x);
}

// Block i copies pair i.  Whether a pair can be is decided from what no block changes: the
// lists, the source rows (a source that is somebody's destination refuses that pair), and the
// destination's length, which only this block changes.
__global__ __launch_bounds__(256) void fork_kernel(const PagedView p, const int32_t* src, const int32_t* dst, int n) {
  const int i = blockIdx.x, t = threadIdx.x;
  const int s = src[i], d = dst[i];
  bool bad = !in_range(s, p.num_seqs) || !in_range(d, p.num_seqs);
  if (!bad) {
    for (int j = t; j < n; j += 256) bad |= src[j] == d || (j < i && dst[j] == d);
  }
  bad = __syncthreads_or(bad);
  int len = 0;
  if (!bad) {
    len = p.lengths[s];
    bad = p.lengths[d] != 0 || len < 0 || len > p.max_pages << p.page_shift;
  }
  bad = __syncthreads_or(bad);
  if (bad) {
    if (t == 0) atomicOr(p.status, Q4D_STATUS_BAD_SEQUENCE);
    return;
  }
  const int held = pages_of(len, p.page_shift);
  const int32_t* from = p.table + (size_t)s * p.max_pages;
  int32_t* to = p.table + (size_t)d * p.max_pages;
  for (int k = t; k < held; k += 256) bad |= !in_range(from[k], p.num_pages);
  if (__syncthreads_or(bad)) {
    if (t == 0) atomicOr(p.status, Q4D_STATUS_BAD_PAGE);
    return;
  }
  for (int k = t; k < held; k += 256) {
    const int page = from[k];
    to[k] = page;
    atomicAdd(&p.refs[page], 1);
  }
  if (t == 0) p.lengths[d] = len;
}

__global__ __launch_bounds__(256) void truncate_kernel(const PagedView p, const int32_t* seqs, const int32_t* lens,
                                                       int n) {
  const int i = blockIdx.x, t = threadIdx.x;
  const int row = seqs[i];
  int bad = !in_range(row, p.num_seqs);
  for (int j = t; j < i; j += 256) bad |= seqs[j] == row;
  bad = __syncthreads_or(bad);  // (an entry that occurs earlier never looks at the row)
  int len = 0, keep = 0;
  if (!bad) {
    len = p.lengths[row];
    keep = lens ? lens[i] : 0;
    bad = keep < 0 || keep > len || len > p.max_pages << p.page_shift;
  }
  __syncthreads();  // everybody has read the length
  if (bad) {
    if (t == 0) atomicOr(p.status, Q4D_STATUS_BAD_SEQUENCE);
    return;
  }
  int32_t* tab = p.table + (size_t)row * p.max_pages;
  for (int k = pages_of(keep, p.page_shift) + t; k < pages_of(len, p.page_shift); k += 256) {
    const int page = tab[k];
    if (in_range(page, p.num_pages)) {
      atomicSub(&p.refs[page], 1);
    } else {
      atomicOr(p.status, Q4D_STATUS_BAD_PAGE);
    }
    tab[k] = -1;
  }
  if (t == 0) p.lengths[row] = keep;
}

// One block: how many pages are held, and which of them goes where.
__global__ __launch_bounds__(1024) void compact_plan_kernel(const PagedView p, const PageWs w, int32_t* used) {
  __shared__ __attribute__((aligned(16))) int sums[16];
  const int t = threadIdx.x;
  int mine = 0, count;
  for (int i = t; i < p.num_pages; i += 1024) mine += p.refs[i] != 0;
  block_excl(mine, t, sums, &count);
  int holes = 0, movers = 0;
  for (int p0 = 0; p0 < p.num_pages; p0 += 1024) {
    const int i = p0 + t;
    const bool in = i < p.num_pages, held = in && p.refs[i] != 0;
    const int hole = in && !held && i < count, mover = held && i >= count;
    int sum;
    const int k = block_excl(hole | mover << 16, t, sums, &sum);  // both counts of a round fit 16 bits
    if (hole) w.ids[holes + (k & 0xFFFF)] = i;
    if (mover) w.a[movers + (k >> 16)] = i;
    if (in && !mover) w.b[i] = i;
    holes += sum & 0xFFFF;
    movers += sum >> 16;
  }
  __threadfence();
  __syncthreads();
  for (int k = t; k < movers; k += 1024) {
    const int from = load_now(&w.a[k]), to = load_now(&w.ids[k]);
    w.src[k] = from;
    w.dst[k] = to;
    w.rows[k] = 1 << p.page_shift;
    w.b[from] = to;
    p.refs[to] = p.refs[from];
    p.refs[from] = 0;
  }
  if (t == 0) {
    *w.copies = movers;
    w.copies[1] = count;
    if (used) *used = count;
  }
}

// Blocks below copy_blocks copy the pages, the others rename them in the table.
__global__ __launch_bounds__(256) void compact_apply_kernel(const PagedView p, const PageWs w, int copy_blocks) {
  if ((int)blockIdx.x < copy_blocks) {
    copy_pages(p, w, blockIdx.x, copy_blocks);
    return;
  }
  const int count = w.copies[1];
  for (int row = blockIdx.x - copy_blocks; row < p.num_seqs; row += gridDim.x - copy_blocks) {
    const int len = p.lengths[row];
    if (len <= 0 || len > p.max_pages << p.page_shift) continue;
    int32_t* tab = p.table + (size_t)row * p.max_pages;
    for (int k = threadIdx.x; k < pages_of(len, p.page_shift); k += 256) {
      const int page = tab[k];
      if (!in_range(page, p.num_pages)) atomicOr(p.status, Q4D_STATUS_BAD_PAGE);
      else if (page >= count) tab[k] = w.b[page];
    }
  }
}

// ---- append -----------------------------------------------------------------------------
struct AppendArgs {
  PagedView p;
  RaggedView r;
  const void *q, *k, *v;
  long long qs, ks, vs;
  const float *q_gamma, *k_gamma;
  float eps;
  const float *cos, *sin;  // NULL: no rotation
  int rope_ctx, rot, inter;
  uint16_t* q_out;
  uint16_t *kplane, *vplane;
  int qh, per;  // head rows (q, k, v) of a token: qh + 2 kvh; waves per token
};

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 f8 __attribute__((ext_vector_type(8)));

template <int XT>
__device__ __forceinline__ void load8(const void* p, long long i, float (&x)[8]) {
  if constexpr (XT == Q4D_F32) {
    const f32x4* s = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
    const f32x4 a = s[0], b = s[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = a[e];
      x[e + 4] = b[e];
    }
  } else if constexpr (XT == Q4D_F16) {
    const f8 a = *reinterpret_cast<const f8*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)a[e];
  } else {
    const b8 a = *reinterpret_cast<const b8*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)a[e];
  }
}

template <bool BF>
__device__ __forceinline__ void store8(uint16_t* p, const float (&x)[8]) {
  if constexpr (BF) {
    b8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (__bf16)x[e];
    *reinterpret_cast<b8*>(p) = y;
  } else {
    f8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (_Float16)x[e];
    *reinterpret_cast<f8*>(p) = y;
  }
}

// Which batch entry token t is of: entries whose end is at or below t, counted 64 at a time.
__device__ __forceinline__ int entry_of(const RaggedView& r, int t, int lane) {
  int b = 0;
  for (int g = 0; g < r.n; g += 64) {
    const int i = g + lane;
    const int c = __popcll(__ballot(i < r.n && r.starts[min(i, r.n - 1) + 1] <= t));
    b += c;
    if (c < 64) break;
  }
  return b;
}

// A wave takes one token and some of its head rows; D / 8 lanes hold a head row, 8 dims each, so that
// the norm's sum and the rotation's partners are lane exchanges and a row is read and written once, 16
// or 32 bytes a lane.  Bound by those bytes (4900 tokens of 16 / 8 heads, 79 MB: 17 us, 4.6 TB/s with
// the launch) or by the chain of reads before them (starts, lengths, page, angles; 16 tokens 3.7 us).
template <int D, int XT, bool BF>
__global__ __launch_bounds__(256) void append_kernel(const AppendArgs a) {
  constexpr int L = D / 8, R = 64 / L;  // lanes a row, rows at a time
  const int lane = threadIdx.x & 63;
  const long long wave = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int tok = (int)(wave / a.per), part = (int)(wave % a.per);
  if (tok >= a.r.tokens) return;
  const int refused = *a.p.status & Q4D_STATUS_NOT_RESERVED;  // (nobody sets this bit meanwhile)
  const int b = entry_of(a.r, tok, lane);
  if (b >= a.r.n || refused) return;
  const SeqSpan s = seq_span(a.p, a.r, b);
  if (s.count < 0 || tok < s.first || tok >= s.first + s.count) {
    if (lane == 0 && s.count < 0) atomicOr(a.p.status, Q4D_STATUS_BAD_SEQUENCE);
    return;
  }
  const int pos = s.len - s.count + (tok - s.first);
  if (a.cos && pos >= a.rope_ctx) {
    if (lane == 0) atomicOr(a.p.status, Q4D_STATUS_BAD_POSITION);
    return;
  }
  const int page = a.p.table[(size_t)s.row * a.p.max_pages + (pos >> a.p.page_shift)];
  const bool page_ok = in_range(page, a.p.num_pages);
  if (!page_ok && lane == 0) atomicOr(a.p.status, Q4D_STATUS_BAD_PAGE);

  const int sub = lane & (L - 1), d0 = 8 * sub, half = a.rot / 2;
  // the angles of this lane's dims: one per dim in halves (dim mod half), one per pair interleaved
  float c[8], sn[8];
  const bool turned = a.cos && d0 < a.rot;
  if (turned) {
    const size_t at = (size_t)pos * half;
    if (a.inter) {
      const f32x4 cv = *reinterpret_cast<const f32x4*>(a.cos + at + d0 / 2);
      const f32x4 sv = *reinterpret_cast<const f32x4*>(a.sin + at + d0 / 2);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        c[e] = cv[e / 2];
        sn[e] = sv[e / 2];
      }
    } else {
      const int i = d0 < half ? d0 : d0 - half;
      load8<Q4D_F32>(a.cos, at + i, c);
      load8<Q4D_F32>(a.sin, at + i, sn);
    }
  }
  const int rows = a.qh + 2 * a.p.kvh, off = pos & ((1 << a.p.page_shift) - 1);
  for (int g = part * R; g < rows; g += a.per * R) {
    const int h = g + lane / L;
    const bool on = h < rows;
    const int kind = h < a.qh ? 0 : h < a.qh + a.p.kvh ? 1 : 2;
    const int j = kind == 0 ? h : kind == 1 ? h - a.qh : h - a.qh - a.p.kvh;
    const void* src = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
    const long long stride = kind == 0 ? a.qs : kind == 1 ? a.ks : a.vs;
    float x[8] = {};
    if (on) load8<XT>(src, tok * stride + j * D + d0, x);
    const float* gamma = kind == 0 ? a.q_gamma : kind == 1 ? a.k_gamma : nullptr;
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
    ss += dpp_f<kDppQuadSwap1>(ss);
    ss += dpp_f<kDppQuadSwap2>(ss);
    ss += dpp_f<kDppRowHalfMirror>(ss);
    if constexpr (L == 16) ss += dpp_f<kDppRowMirror>(ss);
    if (gamma) {
      const float inv = 1.0f / sqrtf(ss / (float)D + a.eps);
      float gm[8];
      load8<Q4D_F32>(gamma, d0, gm);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (x[e] * inv) * gm[e];
    }
    if (a.cos) {
      float y[8];
      if (a.inter) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = x[e ^ 1];
      } else {  // the partner dims are the same 8 of a lane half / 8 away
        const int from = d0 < half ? lane + half / 8 : lane - half / 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = __shfl(x[e], from);
      }
      if (turned && kind != 2) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool lo = a.inter ? !(e & 1) : d0 < half;
          x[e] = fmaf(x[e], c[e], lo ? -(y[e] * sn[e]) : y[e] * sn[e]);
        }
      }
    }
    if (!on) continue;
    if (kind == 0) {
      store8<BF>(a.q_out + ((size_t)tok * a.qh + j) * D + d0, x);
    } else if (page_ok) {
      store8<BF>((kind == 1 ? a.kplane : a.vplane) + page_elem(a.p, page, j) + (size_t)off * D + d0, x);
    }
  }
}

template <int D, bool BF>
void launch_append(const AppendArgs& a, int xt, unsigned blocks, hipStream_t st) {
  if (xt == Q4D_F32) hipLaunchKernelGGL((append_kernel<D, Q4D_F32, BF>), dim3(blocks), dim3(256), 0, st, a);
  else if (xt == Q4D_F16) hipLaunchKernelGGL((append_kernel<D, Q4D_F16, BF>), dim3(blocks), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((append_kernel<D, Q4D_BF16, BF>), dim3(blocks), dim3(256), 0, st, a);
}

// Groups of head rows (512 / D of them) that a wave takes one after the other: the chain of reads is
// then paid once for all.  One while the groups are few waves a CU, so that none waits for another;
// 1 / 2 / 4 measured, us, groups per CU: 0.5: 3.7 / 4.3 / 5.3, 8: 4.6 / 5.0 / 6.0, 16: 7.5 / 7.2 / 8.2,
// 64: 23.5 / 18.0 / 18.7, 150: 21 / 17.2 / 17.3 (of bf16), 400: 135 / 95 / 86.
int groups_per_wave(long long groups) {
  const long long cus = device_cus();
  return groups < 16 * cus ? 1 : groups < 128 * cus ? 2 : 4;
}

int check_page_ws(const q4d_pages_t* p, const void* ws, size_t bytes) {
  if (!ws) return Q4D_ERR_NULL;
  if (!aligned(ws, 16)) return Q4D_ERR_BAD_ADDR;
  return bytes < q4d_pages_workspace_bytes(p) ? Q4D_ERR_CAPACITY : Q4D_OK;
}

// Blocks of a copy: a unit is 4 to 64 KB, and blocks with one or two units each keep more reads in
// flight than few with many (48 partly filled pages of 28 layers, 1024 / 4096 / 8192 blocks: a step
// of beams 85 / 70 / 71 us when its other kernels took 21; 70 whole pages moved 211 / 213 / 205 us; nothing to copy: no difference).
constexpr int kCopyBlocks = 8192;

}  // namespace
}  // namespace q4d

using namespace q4d;

extern "C" {

size_t q4d_pages_workspace_bytes(const q4d_pages_t* pages) {
  return check_pages(pages) == Q4D_OK ? page_ws_ints(pages->num_pages) * 4 : 0;
}

int q4d_pages_reserve(const q4d_pages_t* pages, const q4d_ragged_t* batch, void* ws, size_t ws_bytes, void* stream) {
  int rc;
  if ((rc = check_pages(pages)) || (rc = check_ragged(batch)) || (rc = check_page_ws(pages, ws, ws_bytes))) return rc;
  const PagedView p = paged_view(pages);
  const PageWs w = page_ws(ws, p.num_pages);
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(reserve_kernel, dim3(1), dim3(1024), 0, st, p, ragged_view(batch), w);
  if ((rc = check_launch())) return rc;
  const long long units = 2LL * p.num_layers * p.kvh * batch->n;
  hipLaunchKernelGGL(copy_kernel, dim3((unsigned)min(units, (long long)kCopyBlocks)), dim3(256), 0, st, p, w);
  return check_launch();
}

int q4d_pages_fork(const q4d_pages_t* pages, const int32_t* src, const int32_t* dst, int32_t n, void* stream) {
  if (const int rc = check_pages(pages)) return rc;
  if (!src || !dst) return Q4D_ERR_NULL;
  if (n <= 0 || n > 65536) return Q4D_ERR_SHAPE;
  if (!aligned(src, 4) || !aligned(dst, 4)) return Q4D_ERR_BAD_ADDR;
  hipLaunchKernelGGL(fork_kernel, dim3(n), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), paged_view(pages), src,
                     dst, n);
  return check_launch();
}

int q4d_pages_truncate(const q4d_pages_t* pages, const int32_t* seqs, const int32_t* lengths, int32_t n, void* stream) {
  if (const int rc = check_pages(pages)) return rc;
  if (!seqs) return Q4D_ERR_NULL;
  if (n <= 0 || n > 65536) return Q4D_ERR_SHAPE;
  if (!aligned(seqs, 4) || !aligned(lengths, 4)) return Q4D_ERR_BAD_ADDR;
  hipLaunchKernelGGL(truncate_kernel, dim3(n), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), paged_view(pages),
                     seqs, lengths, n);
  return check_launch();
}

int q4d_pages_compact(const q4d_pages_t* pages, int32_t* used, void* ws, size_t ws_bytes, void* stream) {
  int rc;
  if ((rc = check_pages(pages)) || (rc = check_page_ws(pages, ws, ws_bytes))) return rc;
  if (!aligned(used, 4)) return Q4D_ERR_BAD_ADDR;
  const PagedView p = paged_view(pages);
  const PageWs w = page_ws(ws, p.num_pages);
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(1024), 0, st, p, w, used);
  if ((rc = check_launch())) return rc;
  hipLaunchKernelGGL(compact_apply_kernel, dim3(kCopyBlocks + min(p.num_seqs, 256)), dim3(256), 0, st, p, w,
                     (int)kCopyBlocks);
  return check_launch();
}

int q4d_paged_append(const q4d_pages_t* pages, int32_t layer, const q4d_ragged_t* batch, const void* q, int64_t q_stride,
                     int32_t q_heads, const void* k, int64_t k_stride, const void* v, int64_t v_stride, int32_t x_dtype,
                     const float* q_gamma, const float* k_gamma, float eps, const q4d_rope_t* rope, void* q_out,
                     void* stream) {
  int rc;
  if ((rc = check_pages(pages)) || (rc = check_ragged(batch))) return rc;
  if (!k || !v || !q != !q_out) return Q4D_ERR_NULL;
  if (layer < 0 || layer >= pages->num_layers) return Q4D_ERR_BAD_LAYER;
  if (x_dtype != Q4D_F32 && x_dtype != Q4D_F16 && x_dtype != Q4D_BF16) return Q4D_ERR_DTYPE;
  const int kvh = pages->num_kv_heads, d = pages->head_dim, ew = x_dtype == Q4D_F32 ? 4 : 2;
  if (q ? q_heads <= 0 || q_heads > 16 * 256 : q_heads != 0) return Q4D_ERR_SHAPE;
  if ((q && q_stride < (int64_t)q_heads * d) || k_stride < (int64_t)kvh * d || v_stride < (int64_t)kvh * d)
    return Q4D_ERR_SHAPE;
  if (q_stride > INT64_C(1) << 32 || k_stride > INT64_C(1) << 32 || v_stride > INT64_C(1) << 32) return Q4D_ERR_SHAPE;
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(q_out, 16) || !aligned(q_gamma, 16) ||
      !aligned(k_gamma, 16) || (q && q_stride * ew % 16) || k_stride * ew % 16 || v_stride * ew % 16)
    return Q4D_ERR_BAD_ADDR;
  if (rope) {
    if (!rope->cos || !rope->sin) return Q4D_ERR_NULL;
    if (rope->max_ctx <= 0 || rope->rotary_dim <= 0 || rope->rotary_dim > d || rope->rotary_dim % 16 ||
        (rope->interleaved != 0 && rope->interleaved != 1))
      return Q4D_ERR_SHAPE;
    if (!aligned(rope->cos, 16) || !aligned(rope->sin, 16)) return Q4D_ERR_BAD_ADDR;
  }
  AppendArgs a;
  memset(&a, 0, sizeof(a));
  a.p = paged_view(pages);
  a.r = ragged_view(batch);
  a.q = q; a.k = k; a.v = v;
  a.qs = q_stride; a.ks = k_stride; a.vs = v_stride;
  a.q_gamma = q_gamma; a.k_gamma = k_gamma;
  a.eps = eps;
  if (rope) {
    a.cos = rope->cos;
    a.sin = rope->sin;
    a.rope_ctx = rope->max_ctx;
    a.rot = rope->rotary_dim;
    a.inter = rope->interleaved;
  }
  a.q_out = static_cast<uint16_t*>(q_out);
  a.qh = q_heads;
  a.kplane = a.p.data + (size_t)layer * 2 * plane_elems(a.p);
  a.vplane = a.kplane + plane_elems(a.p);
  const int at_a_time = 512 / d, groups = (q_heads + 2 * kvh + at_a_time - 1) / at_a_time;
  const int each = groups_per_wave((long long)batch->tokens * groups);
  a.per = (groups + each - 1) / each;
  const long long waves = (long long)batch->tokens * a.per;
  if ((waves + 3) / 4 > kMaxBlocks) return Q4D_ERR_SHAPE;
  const unsigned blocks = (unsigned)((waves + 3) / 4);
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const bool bf = pages->dtype == Q4D_BF16;
  if (d == 128) bf ? launch_append<128, true>(a, x_dtype, blocks, st) : launch_append<128, false>(a, x_dtype, blocks, st);
  else bf ? launch_append<64, true>(a, x_dtype, blocks, st) : launch_append<64, false>(a, x_dtype, blocks, st);
  return check_launch();
}

size_t q4d_paged_attention_workspace_bytes(const q4d_pages_t* pages, int32_t q_heads, int32_t n, int32_t tokens,
                                           int32_t max_new) {
  if (check_pages(pages) || n <= 0 || n > 4096 || tokens <= 0 || tokens > 1 << 24 || max_new <= 0) return 0;
  const int kvh = pages->num_kv_heads;
  if (q_heads <= 0 || q_heads % kvh || q_heads / kvh > 16) return 0;
  return paged_attention_ws_bytes(kvh, pages->head_dim, q_heads, n, tokens, max_new);
}

int q4d_paged_attention_workspace_init(void* ws, size_t ws_bytes, void* stream) {
  if (!ws) return Q4D_ERR_NULL;
  if (!aligned(ws, 256)) return Q4D_ERR_BAD_ADDR;
  const size_t n = paged_attention_ws_counters();
  if (ws_bytes < n) return Q4D_ERR_CAPACITY;
  return launch_fill_i32(static_cast<int32_t*>(ws), 0, n / 4, reinterpret_cast<hipStream_t>(stream));
}

int q4d_paged_attention(const q4d_pages_t* pages, int32_t layer, const q4d_ragged_t* batch, const void* q,
                        int64_t q_stride, int32_t q_heads, float scaling, void* out, int64_t out_stride, void* ws,
                        size_t ws_bytes, void* stream) {
  int rc;
  if ((rc = check_pages(pages)) || (rc = check_ragged(batch))) return rc;
  if (!q || !out || !ws) return Q4D_ERR_NULL;
  if (layer < 0 || layer >= pages->num_layers) return Q4D_ERR_BAD_LAYER;
  const int kvh = pages->num_kv_heads, d = pages->head_dim;
  if (q_heads <= 0 || q_heads % kvh || q_heads / kvh > 16 || !__builtin_isfinite(scaling)) return Q4D_ERR_SHAPE;
  if (q_stride < (int64_t)q_heads * d || out_stride < (int64_t)q_heads * d || q_stride > INT64_C(1) << 32 ||
      out_stride > INT64_C(1) << 32)
    return Q4D_ERR_SHAPE;
  if (!aligned(q, 16) || !aligned(out, 16) || q_stride % 8 || out_stride % 8 || !aligned(ws, 256)) return Q4D_ERR_BAD_ADDR;
  if (ws_bytes < paged_attention_ws_bytes(kvh, d, q_heads, batch->n, batch->tokens, batch->max_new))
    return Q4D_ERR_CAPACITY;
  PagedAttnArgs a;
  memset(&a, 0, sizeof(a));
  a.p = paged_view(pages);
  a.r = ragged_view(batch);
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.kplane = a.p.data + (size_t)layer * 2 * plane_elems(a.p);
  a.vplane = a.kplane + plane_elems(a.p);
  a.scale = scaling * 1.4426950408889634f;
  a.qh = q_heads;
  a.bf16 = pages->dtype == Q4D_BF16;
  a.ws = ws;
  return launch_paged_attention(a, reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
