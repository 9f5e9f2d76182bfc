// Pages of the KV cache between steps: rows of the page table replaced by forks of them, and the pages that are held moved to the front.
// The reference keeps its pages' owners on the host (astrai/inference/core/cache.py:18-185: a bitmask, reference counts, a queue of
// prompts' pages) and gives every sequence pages of its own; here table, counts and caches stay on the device and no call waits for it,
// so that a step of a search can be captured with the decode steps around it.
//
// refs[page] counts who holds a page: rows of the table, and whoever else (a cache of prompts).  0: free.
#include "aq_common.h"

namespace aq {

constexpr int PG_THREADS = 256, PG_PAGES = 4096;  // pages of a workgroup that numbers them: 16 to a thread
constexpr int PG_UNIT = 16 * 1024;                // bytes of a copying workgroup's turn: 4 x 16 to a thread

struct ForkArgs {
  const int64_t* table;    // [B, P]
  const int32_t* refs;     // [n_pages]
  const int64_t* parents;  // [R]
  const int64_t* lens;     // [B] or null: all T
  int64_t* new_table;      // [R, P]
  int32_t* new_refs;       // [n_pages]
  int32_t* missing;        // [1]
  int32_t* gone;           // [n_pages] entries of the old rows that name the page
  int32_t* come;           // [n_pages] entries of the new rows that name it
  int32_t* source;         // [R] the page that the row needs a copy of, or -1
  int32_t* wanting;        // [R] rows that need one, ascending
  int32_t* fresh;          // [R] the pages they get, ascending
  int32_t* counts;         // [2] rows that need a page, rows that get one
  uint8_t *k, *v;          // [layers][n_pages][page][row_bytes]
  int64_t layer_bytes, row_bytes, page, T, n_pages;
  int B, R, P, layers;
};

// Sum over the workgroup, in every thread.
__device__ __forceinline__ int wg_sum(int v, int* s) {
  const int tid = threadIdx.x;
  __syncthreads();
#pragma unroll
  for (int off = 32; off; off >>= 1) v += __shfl_xor(v, off, 64);
  if ((tid & 63) == 0) s[tid >> 6] = v;
  __syncthreads();
  return s[0] + s[1] + s[2] + s[3];
}

// Sum over the threads before this one; *all: over all of them.
__device__ __forceinline__ int wg_before(int v, int* s, int* all) {
  const int tid = threadIdx.x, lane = tid & 63;
  __syncthreads();
  int x = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(x, off, 64);
    if (lane >= off) x += y;
  }
  if (lane == 63) s[tid >> 6] = x;
  __syncthreads();
  int base = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < PG_THREADS / 64; ++w) {
    if (w < tid >> 6) base += s[w];
    sum += s[w];
  }
  *all = sum;
  return base + x - v;
}

__global__ __launch_bounds__(PG_THREADS) void fork_clear_kernel(int32_t* p, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * PG_THREADS + threadIdx.x;
  if (i < n) p[i] = 0;
}

// A row of the old table (the workgroups from R on: whose pages they let go), or of the new one.  Counts are whole numbers: the order of
// the atomics changes nothing.
__global__ __launch_bounds__(PG_THREADS) void fork_rows_kernel(ForkArgs a) {
  const int tid = threadIdx.x;
  auto entry = [&](int row, int l) -> int {
    const int64_t e = a.table[(int64_t)row * a.P + l];
    return e >= 0 && e < a.n_pages ? (int)e : -1;
  };
  if ((int)blockIdx.x >= a.R) {
    const int row = (int)blockIdx.x - a.R;
    for (int l = tid; l < a.P; l += PG_THREADS) {
      const int e = entry(row, l);
      if (e >= 0) atomicAdd(a.gone + e, 1);
    }
    return;
  }
  const int i = (int)blockIdx.x;
  const int64_t parent = a.parents[i];
  const bool known = parent >= 0 && parent < a.B;
  int before = 0;  // an earlier child of the same parent
  for (int j = tid; j < i; j += PG_THREADS) before |= a.parents[j] == parent;
  const bool first = known && !__syncthreads_or(before);
  const int p = known ? (int)parent : 0;
  int64_t n = a.lens ? a.lens[p] : a.T;
  n = n < 0 ? 0 : n > a.T ? a.T : n;
  const int64_t whole = n / a.page, rest = n - whole * a.page;
  for (int l = tid; l < a.P; l += PG_THREADS) {
    const int e = known && (first || l < whole) ? entry(p, l) : -1;
    a.new_table[(int64_t)i * a.P + l] = e;
    if (e >= 0) atomicAdd(a.come + e, 1);
  }
  if (tid == 0) a.source[i] = known && !first && rest > 0 && whole < a.P ? entry(p, (int)whole) : -1;
}

// The new counts, and the free pages for the rows that need one: the k-th free page to the k-th row.  Every workgroup counts the free
// pages in front of its own by itself.  The last workgroup numbers the rows.
__global__ __launch_bounds__(PG_THREADS) void fork_refs_kernel(ForkArgs a, int groups) {
  __shared__ int s[PG_THREADS / 64];
  const int tid = threadIdx.x;
  if ((int)blockIdx.x == groups) {
    int done = 0;
    for (int i0 = 0; i0 < a.R; i0 += PG_THREADS) {
      const int i = i0 + tid;
      const int want = i < a.R && a.source[i] >= 0;
      int all;
      const int at = done + wg_before(want, s, &all);
      if (want) a.wanting[at] = i;
      done += all;
    }
    if (tid == 0) a.counts[0] = done;
    return;
  }
  int need = 0;
  for (int i = tid; i < a.R; i += PG_THREADS) need += a.source[i] >= 0;
  need = wg_sum(need, s);
  auto count = [&](int64_t x) -> int {
    const int left = a.refs[x] - a.gone[x];
    return (left > 0 ? left : 0) + a.come[x];
  };
  const int64_t x0 = (int64_t)blockIdx.x * PG_PAGES;
  int base = 0;
  for (int64_t x = tid; x < x0; x += PG_THREADS) base += count(x) == 0;
  base = wg_sum(base, s);
  for (int64_t x = x0 + tid; x - tid < x0 + PG_PAGES; x += PG_THREADS) {
    int c = x < a.n_pages ? count(x) : 1;
    const int is_free = c == 0;
    int all;
    const int at = base + wg_before(is_free, s, &all);
    if (is_free && at < need) {
      a.fresh[at] = (int)x;
      c = 1;
    }
    if (x < a.n_pages) a.new_refs[x] = c;
    base += all;
  }
  if ((int)blockIdx.x == groups - 1 && tid == 0) {
    a.counts[1] = need < base ? need : base;
    a.missing[0] = need > base ? need - base : 0;
  }
}

// 16 bytes a thread at a time, four in flight.
__device__ __forceinline__ void copy_unit(const uint8_t* from, uint8_t* to, int64_t bytes) {
  uint4 x[PG_UNIT / 16 / PG_THREADS];
#pragma unroll
  for (int u = 0; u < PG_UNIT / 16 / PG_THREADS; ++u) {
    const int64_t at = (int64_t)(u * PG_THREADS + threadIdx.x) * 16;
    if (at < bytes) x[u] = *reinterpret_cast<const uint4*>(from + at);
  }
#pragma unroll
  for (int u = 0; u < PG_UNIT / 16 / PG_THREADS; ++u) {
    const int64_t at = (int64_t)(u * PG_THREADS + threadIdx.x) * 16;
    if (at < bytes) *reinterpret_cast<uint4*>(to + at) = x[u];
  }
}

// The copies' first rest positions, in units of PG_UNIT bytes of one layer's keys or values, and their entries of the table.
__global__ __launch_bounds__(PG_THREADS) void fork_copy_kernel(ForkArgs a) {
  const int got = a.counts[1];
  const int64_t per_page = (a.page * a.row_bytes + PG_UNIT - 1) / PG_UNIT, per_copy = per_page * 2 * a.layers;
  for (int64_t u = blockIdx.x; u < got * per_copy; u += gridDim.x) {
    const int c = (int)(u / per_copy);
    const int64_t w = u - c * per_copy, lkv = w / per_page, chunk = w - lkv * per_page;
    const int i = a.wanting[c], p = (int)a.parents[i];
    int64_t n = a.lens ? a.lens[p] : a.T;
    n = n < 0 ? 0 : n > a.T ? a.T : n;
    const int64_t whole = n / a.page, bytes = (n - whole * a.page) * a.row_bytes - chunk * PG_UNIT;
    if (w == 0 && threadIdx.x == 0) a.new_table[(int64_t)i * a.P + whole] = a.fresh[c];
    if (bytes <= 0) continue;
    uint8_t* const base = (lkv & 1 ? a.v : a.k) + (lkv >> 1) * a.layer_bytes + chunk * PG_UNIT;
    const int64_t page_bytes = a.page * a.row_bytes;
    copy_unit(base + a.source[i] * page_bytes, base + a.fresh[c] * page_bytes, bytes < PG_UNIT ? bytes : PG_UNIT);
  }
}

struct CompactArgs {
  const int64_t* table;  // [B, P] entries in all
  const int32_t* refs;
  int64_t* new_table;
  int32_t* new_refs;
  int64_t* where;  // [n_pages] where a held page went, -1: free
  int32_t* live;   // [1]
  int32_t* source;  // [n_pages] of the k-th move: the k-th page held from the top,
  int32_t* hole;    // [n_pages] the k-th free one from the bottom
  int32_t* move;    // [n_pages] of a held page past the last place: which move is its own
  int32_t* moves;   // [1]
  uint8_t *k, *v;
  int64_t layer_bytes, page_bytes, n_pages, entries;
  int layers;
};

// Numbers the pages: live of them are held, places 0 .. live - 1 are to hold them.  Every workgroup counts what lies in front of its own
// pages, and all, by itself.
__global__ __launch_bounds__(PG_THREADS) void compact_rank_kernel(CompactArgs a) {
  __shared__ int s[PG_THREADS / 64];
  const int tid = threadIdx.x;
  const int64_t x0 = (int64_t)blockIdx.x * PG_PAGES;
  int before = 0, rest = 0;
  for (int64_t x = tid; x < x0; x += PG_THREADS) before += a.refs[x] > 0;
  for (int64_t x = x0 + tid; x < a.n_pages; x += PG_THREADS) rest += a.refs[x] > 0;
  before = wg_sum(before, s);
  const int live = before + wg_sum(rest, s);
  int base = before;
  for (int64_t x = x0 + tid; x - tid < x0 + PG_PAGES; x += PG_THREADS) {
    const int r = x < a.n_pages ? a.refs[x] : 0;
    const int held = r > 0;
    int all;
    const int at = base + wg_before(held, s, &all);  // held pages in front of x
    base += all;
    if (x >= a.n_pages) continue;
    a.where[x] = held && x < live ? x : -1;  // moved pages: their move says
    a.new_refs[x] = held && x < live ? r : 0;
    if (held && x >= live) {
      a.source[live - 1 - at] = (int)x;
      a.move[x] = live - 1 - at;
    }
    if (!held && x < live) a.hole[x - at] = (int)x;
    if (x == live - 1) a.moves[0] = live - (at + held);  // free pages among the first live
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.live[0] = live;
    if (live == 0) a.moves[0] = 0;
  }
}

// Moves the pages, in units of PG_UNIT bytes of one layer's keys or values, and renumbers the table.  Sources lie behind the last place,
// holes in front of it: no page is both.
__global__ __launch_bounds__(PG_THREADS) void compact_move_kernel(CompactArgs a) {
  const int moves = a.moves[0], live = a.live[0];
  const int64_t stride = (int64_t)gridDim.x * PG_THREADS, me = (int64_t)blockIdx.x * PG_THREADS + threadIdx.x;
  for (int64_t i = me; i < a.entries; i += stride) {
    const int64_t e = a.table[i];
    int64_t to = -1;
    if (e >= 0 && e < a.n_pages && a.refs[e] > 0) to = e < live ? e : a.hole[a.move[e]];
    a.new_table[i] = to;
  }
  for (int64_t i = me; i < moves; i += stride) {
    const int from = a.source[i], to = a.hole[i];
    a.where[from] = to;
    a.new_refs[to] = a.refs[from];
  }
  const int64_t per_page = (a.page_bytes + PG_UNIT - 1) / PG_UNIT, per_move = per_page * 2 * a.layers;
  for (int64_t u = blockIdx.x; u < moves * per_move; u += gridDim.x) {
    const int c = (int)(u / per_move);
    const int64_t w = u - c * per_move, lkv = w / per_page, chunk = w - lkv * per_page, left = a.page_bytes - chunk * PG_UNIT;
    uint8_t* const base = (lkv & 1 ? a.v : a.k) + (lkv >> 1) * a.layer_bytes + chunk * PG_UNIT;
    copy_unit(base + a.source[c] * a.page_bytes, base + a.hole[c] * a.page_bytes, left < PG_UNIT ? left : PG_UNIT);
  }
}

static int check_caches(const void* k, const void* v, int64_t layers, int64_t layer_bytes, int64_t n_pages, int64_t page_size, int64_t row_bytes) {
  if (layers <= 0 || n_pages <= 0 || page_size <= 0 || row_bytes <= 0) return AQ_E_SHAPE;
  if (layers > 65535 || n_pages > 0x7fffffff - PG_PAGES || page_size > (1 << 30) || row_bytes > (1 << 30)) return AQ_E_RANGE;
  if ((row_bytes & 15) || (layer_bytes & 15)) return AQ_E_ALIGN;
  if (layers > 1 && layer_bytes / row_bytes / page_size < n_pages) return AQ_E_SHAPE;  // layers that overlap
  if (!k || !v) return AQ_E_NULL;
  return check_ptr16(k) || check_ptr16(v) ? AQ_E_ALIGN : AQ_OK;
}

static unsigned copy_groups(int64_t units) {
  const int64_t most = (int64_t)device_cus() * 8;  // 8 workgroups of 256 threads fill a compute unit
  return (unsigned)(units < 1 ? 1 : units < most ? units : most);
}

}  // namespace aq

extern "C" int64_t aq_fork_pages_workspace_bytes(int64_t n_pages, int64_t R) {
  return n_pages <= 0 || R < 0 ? 0 : (2 * n_pages + 3 * R + 2) * (int64_t)sizeof(int32_t);
}

extern "C" int aq_fork_pages(const int64_t* page_table, int64_t B, int64_t P, const int32_t* refs, const int64_t* parents, int64_t R,
                             int64_t total_len, const int64_t* seq_lens, void* k_layers, void* v_layers, int64_t layers,
                             int64_t layer_bytes, int64_t n_pages, int64_t page_size, int64_t row_bytes, int64_t* new_table,
                             int32_t* new_refs, int32_t* missing, void* workspace, int64_t workspace_bytes, void* stream) {
  if (B < 0 || R < 0 || P <= 0 || total_len < 0) return AQ_E_SHAPE;
  if (const int rc = aq::check_caches(k_layers, v_layers, layers, layer_bytes, n_pages, page_size, row_bytes)) return rc;
  if (B > (1 << 24) || R > (1 << 24) || P > 0x7fffffff) return AQ_E_RANGE;
  if ((B > 0 && !page_table) || (R > 0 && (!parents || !new_table)) || !refs || !new_refs || !missing || !workspace) return AQ_E_NULL;
  if (aq::check_ptr(page_table, 8) || aq::check_ptr(parents, 8) || aq::check_ptr(seq_lens, 8) || aq::check_ptr(new_table, 8) ||
      aq::check_ptr(refs, 4) || aq::check_ptr(new_refs, 4) || aq::check_ptr(missing, 4) || aq::check_ptr(workspace, 4))
    return AQ_E_ALIGN;
  if (workspace_bytes < aq_fork_pages_workspace_bytes(n_pages, R)) return AQ_E_WORKSPACE;
  aq::ForkArgs a{};
  a.table = page_table;
  a.refs = refs;
  a.parents = parents;
  a.lens = seq_lens;
  a.new_table = new_table;
  a.new_refs = new_refs;
  a.missing = missing;
  a.gone = static_cast<int32_t*>(workspace);
  a.come = a.gone + n_pages;
  a.source = a.come + n_pages;
  a.wanting = a.source + R;
  a.fresh = a.wanting + R;
  a.counts = a.fresh + R;
  a.k = static_cast<uint8_t*>(k_layers);
  a.v = static_cast<uint8_t*>(v_layers);
  a.layer_bytes = layer_bytes;
  a.row_bytes = row_bytes;
  a.page = page_size;
  a.T = total_len;
  a.n_pages = n_pages;
  a.B = (int)B;
  a.R = (int)R;
  a.P = (int)P;
  a.layers = (int)layers;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 block(aq::PG_THREADS);
  const int groups = (int)((n_pages + aq::PG_PAGES - 1) / aq::PG_PAGES);
  aq::queue_kernel(aq::fork_clear_kernel, dim3((unsigned)((2 * n_pages + aq::PG_THREADS - 1) / aq::PG_THREADS)), block, 0, st, a.gone, 2 * n_pages);
  if (R + B > 0) aq::queue_kernel(aq::fork_rows_kernel, dim3((unsigned)(R + B)), block, 0, st, a);
  aq::queue_kernel(aq::fork_refs_kernel, dim3((unsigned)(groups + 1)), block, 0, st, a, groups);
  if (R > 1) {  // (a single row is its parent's first child)
    const int64_t units = (R - 1) * 2 * layers * ((page_size * row_bytes + aq::PG_UNIT - 1) / aq::PG_UNIT);
    aq::queue_kernel(aq::fork_copy_kernel, dim3(aq::copy_groups(units)), block, 0, st, a);
  }
  return (int)hipGetLastError();
}

extern "C" int64_t aq_compact_pages_workspace_bytes(int64_t n_pages) { return n_pages <= 0 ? 0 : (3 * n_pages + 1) * (int64_t)sizeof(int32_t); }

extern "C" int aq_compact_pages(const int64_t* page_table, int64_t entries, const int32_t* refs, void* k_layers, void* v_layers,
                                int64_t layers, int64_t layer_bytes, int64_t n_pages, int64_t page_size, int64_t row_bytes,
                                int64_t* new_table, int32_t* new_refs, int64_t* where, int32_t* live, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  if (entries < 0) return AQ_E_SHAPE;
  if (const int rc = aq::check_caches(k_layers, v_layers, layers, layer_bytes, n_pages, page_size, row_bytes)) return rc;
  if ((entries > 0 && (!page_table || !new_table)) || !refs || !new_refs || !where || !live || !workspace) return AQ_E_NULL;
  if (aq::check_ptr(page_table, 8) || aq::check_ptr(new_table, 8) || aq::check_ptr(where, 8) || aq::check_ptr(refs, 4) ||
      aq::check_ptr(new_refs, 4) || aq::check_ptr(live, 4) || aq::check_ptr(workspace, 4))
    return AQ_E_ALIGN;
  if (workspace_bytes < aq_compact_pages_workspace_bytes(n_pages)) return AQ_E_WORKSPACE;
  aq::CompactArgs a{};
  a.table = page_table;
  a.refs = refs;
  a.new_table = new_table;
  a.new_refs = new_refs;
  a.where = where;
  a.live = live;
  a.source = static_cast<int32_t*>(workspace);
  a.hole = a.source + n_pages;
  a.move = a.hole + n_pages;
  a.moves = a.move + n_pages;
  a.k = static_cast<uint8_t*>(k_layers);
  a.v = static_cast<uint8_t*>(v_layers);
  a.layer_bytes = layer_bytes;
  a.page_bytes = page_size * row_bytes;
  a.n_pages = n_pages;
  a.entries = entries;
  a.layers = (int)layers;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 block(aq::PG_THREADS);
  aq::queue_kernel(aq::compact_rank_kernel, dim3((unsigned)((n_pages + aq::PG_PAGES - 1) / aq::PG_PAGES)), block, 0, st, a);
  const int64_t units = n_pages / 2 * 2 * layers * ((a.page_bytes + aq::PG_UNIT - 1) / aq::PG_UNIT), rows = (entries + aq::PG_THREADS - 1) / aq::PG_THREADS;
  aq::queue_kernel(aq::compact_move_kernel, dim3(aq::copy_groups(units > rows ? units : rows)), block, 0, st, a);
  return (int)hipGetLastError();
}
