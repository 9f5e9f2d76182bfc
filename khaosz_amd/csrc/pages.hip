// Pages of the KV cache between steps: rows of the page table replaced by forks of them, and the pages that are held moved to the front.
// The reference keeps its pages' owners on the host (astrai/inference/core/cache.py:18-185: a bitmask, reference counts, a queue of
// prompts' pages) and gives every sequence pages of its own; here table, counts and caches stay on the device and no call waits for it,
// so that a step of a search can be captured with the decode steps around it.
//
// What bounds them: pages that move, HBM (500 of 1024 pages, 24 layers, 1.6 GB: 300 to 340 us by the card, 5.2 TB/s; 64 beams of which 24 go on, 220 MB:
// 46.3); else launches and the chain of reads in each: table, counts, free pages, copies (from a graph 1 row into 8, 24 layers, 22 MB: 6.7; 40 of 128
// pages: 4.7; 256 rows into 300 over 40000 pages, five launches: 16.8; queued one by one 6.8, 6.8 and 19.6, what the host takes for them).
//
// refs[page] counts who holds a page: rows of the table, and whoever else (a cache of prompts).  0: free.
#include "aq_common.h"

namespace aq {

constexpr int PG_THREADS = 1024, PG_PAGES = 4 * PG_THREADS;  // of a workgroup that numbers pages: 4 to a thread
constexpr int PG_COPY = 256, PG_UNIT = 8 * 1024;              // a copying workgroup, and the bytes of its turn: 2 x 16 to a thread
constexpr int PG_TURN = 4 * PG_COPY, PG_SEGMENTS = 1024;      // where pages are counted in segments: pages of a turn, at most so many segments

// Turns of a segment; as many segments as the pages take.
static int64_t segment_turns(int64_t n_pages) { return (n_pages + PG_TURN * PG_SEGMENTS - 1) / (PG_TURN * PG_SEGMENTS); }
static int64_t segments(int64_t n_pages) {
  const int64_t size = segment_turns(n_pages) * PG_TURN;
  return (n_pages + size - 1) / size;
}

// A copy that a row needs: the page, its written positions, the row, and the entry of the row that gets the new page.
struct ForkCopy {
  int32_t source, rows, row, column;
};

struct ForkArgs {
  const int64_t* table;    // [B, P]
  const int32_t* refs;     // [n_pages]
  const int64_t* parents;  // [R]
  const int64_t* lens;     // [B] or null: all T
  int64_t* new_table;      // [R, P]
  int32_t* new_refs;       // [n_pages]
  int32_t* missing;        // [1]
  ForkCopy* wants;         // [R] of a row, source -1: none
  ForkCopy* copies;        // [R] the same, the rows that need one only
  int32_t* fresh;          // [R] the pages they get, ascending
  int32_t* got;            // [1] rows that get one
  int32_t* need;           // [1] rows that need one
  int32_t* free_pages;     // [segments] free pages of each segment, these rows not yet served
  int32_t* gone;           // [n_pages] entries of the old rows that name the page
  int32_t* come;           // [n_pages] entries of the new rows that name it
  uint8_t *k, *v;          // [layers][n_pages][page][row_bytes]
  int64_t layer_bytes, row_bytes, page_bytes, T, n_pages;
  int B, R, P, layers, page, turns;
  UDiv by_p;  // (one-workgroup form)
};

// Sum over the threads before this one; *all: over all of them.
template <int THREADS>
__device__ __forceinline__ int wg_before(int v, int* s, int* all) {
  const int tid = threadIdx.x, lane = tid & 63;
  int x = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(x, off, 64);
    if (lane >= off) x += y;
  }
  __syncthreads();  // s may still be read by an earlier call
  if (lane == 63) s[tid >> 6] = x;
  __syncthreads();
  int base = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < tid >> 6) base += s[w];
    sum += s[w];
  }
  *all = sum;
  return base + x - v;
}

// f(i) summed over the workgroup, i in [i0, i1); several loads in flight.
template <int THREADS, class F>
__device__ __forceinline__ int wg_count(int64_t i0, int64_t i1, int* s, F&& f) {
  int n = 0;
#pragma unroll 8
  for (int64_t i = i0 + threadIdx.x; i < i1; i += THREADS) n += f(i);
  int all;
  wg_before<THREADS>(n, s, &all);
  return all;
}

__device__ __forceinline__ int fork_entry(const ForkArgs& a, int row, int l) {
  const int64_t e = a.table[(int64_t)row * a.P + l];
  return e >= 0 && e < a.n_pages ? (int)e : -1;
}

__device__ __forceinline__ int64_t fork_length(const ForkArgs& a, int row) {
  const int64_t n = a.lens ? a.lens[row] : a.T;
  return n < 0 ? 0 : n > a.T ? a.T : n;
}

// refs, with the old rows' entries taken away (none is left at least) and the new rows' added
__device__ __forceinline__ int fork_count(int refs, int gone, int come) {
  return (refs > gone ? refs - gone : 0) + come;
}

// Four pages' new counts: the free ones among them get numbers from `at` on, the first `need` of which are handed out.
__device__ __forceinline__ void fork_hand_out(const ForkArgs& a, int64_t x, int (&c)[4], int at, int need) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if (x + u >= a.n_pages) break;
    if (c[u] == 0) {
      if (at < need) {
        a.fresh[at] = (int)(x + u);
        c[u] = 1;
      }
      ++at;
    }
    a.new_refs[x + u] = c[u];
  }
}

__global__ __launch_bounds__(PG_THREADS) void fork_clear_kernel(v4i* p, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * PG_THREADS + threadIdx.x;
  if (i < n) p[i] = v4i{0, 0, 0, 0};
}

// ROWS rows of the new table, or (the workgroups behind those) of the old one, whose pages are let go; a thread has a column, so that
// neighbouring rows with the same page (what sequences share) are one atomic.  (256 old and 300 new rows of 129 columns, 63 of them
// alike: 9.5 us with one row to a workgroup, most of it 556 atomics on each shared page in turn; 6.9 with two, 5.7 with four, 7.0 with eight,
// 12.8 with 16, which are 35 workgroups.)  Counts are whole numbers: the order
// of the atomics changes nothing.
constexpr int FORK_ROWS = 4;
__global__ __launch_bounds__(PG_COPY) void fork_rows_kernel(ForkArgs a, int new_wgs, int chunks) {
  __shared__ int parent_s[FORK_ROWS], whole_s[FORK_ROWS], rest_s[FORK_ROWS], later_s[FORK_ROWS];
  const int tid = threadIdx.x;
  const bool old = (int)blockIdx.x >= new_wgs;
  const int wg = old ? (int)blockIdx.x - new_wgs : (int)blockIdx.x, rows = old ? a.B : a.R;
  const int i0 = wg / chunks * FORK_ROWS, l = (wg - wg / chunks * chunks) * PG_COPY + tid;
  const int n_rows = rows - i0 < FORK_ROWS ? rows - i0 : FORK_ROWS;
  if (!old) {
    if (tid < n_rows) {
      const int64_t p = a.parents[i0 + tid];
      const bool known = p >= 0 && p < a.B;
      parent_s[tid] = known ? (int)p : -1;
      const int64_t n = known ? fork_length(a, (int)p) : 0;
      whole_s[tid] = (int)(n / a.page);
      rest_s[tid] = (int)(n - n / a.page * a.page);
      later_s[tid] = 0;
    }
    __syncthreads();
    for (int j = tid; j < i0 + n_rows; j += PG_COPY) {  // which rows have an earlier sibling
      const int64_t p = a.parents[j];
#pragma unroll
      for (int r = 0; r < FORK_ROWS; ++r)
        if (r < n_rows && j < i0 + r && p == parent_s[r]) later_s[r] = 1;
    }
    __syncthreads();
  }
  if (l >= a.P) return;
  int e[FORK_ROWS];  // all requested before any is used
#pragma unroll
  for (int r = 0; r < FORK_ROWS; ++r) {
    const int p = old ? i0 + r : r < n_rows ? parent_s[r] : -1;
    e[r] = r < n_rows && p >= 0 ? fork_entry(a, p, l) : -1;
  }
  int at = -1, run = 0;
  int32_t* const counts = old ? a.gone : a.come;
#pragma unroll
  for (int r = 0; r < FORK_ROWS; ++r) {
    if (r >= n_rows) break;
    if (!old) {
      const int i = i0 + r;
      if (l == whole_s[r]) a.wants[i] = {later_s[r] && rest_s[r] > 0 ? e[r] : -1, rest_s[r], i, l};
      if (l == 0 && whole_s[r] >= a.P) a.wants[i] = {-1, 0, i, 0};
      if (later_s[r] && l >= whole_s[r]) e[r] = -1;
      a.new_table[(int64_t)i * a.P + l] = e[r];
    }
    if (e[r] != at) {
      if (at >= 0) atomicAdd(counts + at, run);
      at = e[r];
      run = 0;
    }
    ++run;
  }
  if (at >= 0) atomicAdd(counts + at, run);
}

// The rows that need a page, numbered: returns how many.
template <int THREADS>
__device__ __forceinline__ int fork_number(const ForkArgs& a, int* s) {
  int done = 0;
  for (int i0 = 0; i0 < a.R; i0 += THREADS) {
    const int i = i0 + (int)threadIdx.x;
    ForkCopy w = {-1, 0, 0, 0};
    if (i < a.R) w = a.wants[i];
    int all;
    const int at = done + wg_before<THREADS>(w.source >= 0, s, &all);
    if (w.source >= 0) a.copies[at] = w;
    done += all;
  }
  return done;
}

// New counts of the pages x .. x + 3, of those that are there (others: 1).
__device__ __forceinline__ void fork_counts(const ForkArgs& a, int64_t x, int (&c)[4]) {
  if (x + 4 <= a.n_pages) {
    const int64_t i = x / 4;
    const v4i r = reinterpret_cast<const v4i*>(a.refs)[i], g = reinterpret_cast<const v4i*>(a.gone)[i], n = reinterpret_cast<const v4i*>(a.come)[i];
#pragma unroll
    for (int u = 0; u < 4; ++u) c[u] = fork_count(r[u], g[u], n[u]);
    return;
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) c[u] = x + u < a.n_pages ? fork_count(a.refs[x + u], a.gone[x + u], a.come[x + u]) : 1;
}

// The free pages of each segment; the last workgroup numbers the rows.  (Every workgroup counting what lies in front of its own pages
// instead, in one launch: 40000 pages 12 us, this and the next kernel 4.0 and 3.3.)
__global__ __launch_bounds__(PG_COPY) void fork_free_kernel(ForkArgs a) {
  __shared__ int s[PG_COPY / 64];
  if (blockIdx.x == gridDim.x - 1) {
    const int need = fork_number<PG_COPY>(a, s);
    if (threadIdx.x == 0) a.need[0] = need;
    return;
  }
  const int64_t x0 = (int64_t)blockIdx.x * a.turns * PG_TURN;
  const int n = wg_count<PG_COPY>(0, (int64_t)a.turns * PG_COPY, s, [&](int64_t i) {
    const int64_t x = x0 + 4 * i;
    int c[4] = {1, 1, 1, 1};
    if (x < a.n_pages) fork_counts(a, x, c);
    return (c[0] == 0) + (c[1] == 0) + (c[2] == 0) + (c[3] == 0);
  });
  if (threadIdx.x == 0) a.free_pages[blockIdx.x] = n;
}

// The new counts, and the free pages for the rows that need one: the k-th free page to the k-th row.
__global__ __launch_bounds__(PG_COPY) void fork_refs_kernel(ForkArgs a) {
  __shared__ int s[PG_COPY / 64];
  const int need = a.need[0];
  int base = wg_count<PG_COPY>(0, blockIdx.x, s, [&](int64_t i) { return a.free_pages[i]; });
  for (int turn = 0; turn < a.turns; ++turn) {
    const int64_t x = (((int64_t)blockIdx.x * a.turns + turn) * PG_COPY + threadIdx.x) * 4;
    int c[4] = {1, 1, 1, 1}, all;
    if (x < a.n_pages) fork_counts(a, x, c);
    const int at = base + wg_before<PG_COPY>((c[0] == 0) + (c[1] == 0) + (c[2] == 0) + (c[3] == 0), s, &all);
    fork_hand_out(a, x, c, at, need);
    base += all;
  }
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) {
    a.got[0] = need < base ? need : base;
    a.missing[0] = need > base ? need - base : 0;
  }
}

// All of the above by one workgroup, its counts and rows in LDS, for small tables and caches: one launch instead of four.  What it waits for is
// a chain of reads, so that the counts are requested first and each row's parent and length looked up once (1 row into 8, 64 pages, and
// 64 into 64, 2048 pages: 4.7 and 6.4 us with every entry looking them up and the list of copies read back from memory, 4.5 and 5.8).
constexpr int FORK_ONE_PAGES = 8192, FORK_ONE_ROWS = 4096, FORK_ONE_ENTRIES = 32768;
struct ForkRow {
  int parent, whole, rest, source;  // row of the table or -1, pages that are full, rows of the next one, and its page if it is copied, or -1
};
static size_t fork_one_lds(int64_t n_pages, int64_t B, int64_t R) { return (n_pages + 3) / 4 * 8 * sizeof(int) + (B + 3) / 4 * 4 * sizeof(int) + R * sizeof(ForkRow); }

__global__ __launch_bounds__(PG_THREADS) void fork_one_kernel(ForkArgs a) {
  __shared__ int s[PG_THREADS / 64];
  extern __shared__ __align__(16) int pg_lds[];
  const int tid = threadIdx.x, pages = ((int)a.n_pages + 3) & ~3;
  int *const gone = pg_lds, *const come = gone + pages, *const first_of = come + pages;
  ForkRow* const rows = reinterpret_cast<ForkRow*>(first_of + ((a.B + 3) & ~3));
  int refs[FORK_ONE_PAGES / PG_PAGES][4];
#pragma unroll
  for (int t = 0; t < FORK_ONE_PAGES / PG_PAGES; ++t)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int x = t * PG_PAGES + 4 * tid + u;
      refs[t][u] = x < (int)a.n_pages ? a.refs[x] : 1;
    }
  for (int x = tid; x < 2 * pages; x += PG_THREADS) gone[x] = 0;
  for (int p = tid; p < a.B; p += PG_THREADS) first_of[p] = a.R;
  __syncthreads();
  for (int i = tid; i < a.R; i += PG_THREADS) {
    const int64_t p = a.parents[i];
    ForkRow r = {-1, 0, 0, -1};
    if (p >= 0 && p < a.B) {
      const int64_t n = fork_length(a, (int)p);
      r.parent = (int)p;
      r.whole = (int)(n / a.page);
      r.rest = (int)(n - (int64_t)r.whole * a.page);
      atomicMin(first_of + p, i);
    }
    rows[i] = r;
  }
#pragma unroll 2
  for (int x = tid; x < a.B * a.P; x += PG_THREADS) {
    const int64_t e = a.table[x];
    if (e >= 0 && e < a.n_pages) atomicAdd(gone + e, 1);
  }
  __syncthreads();
#pragma unroll 2
  for (int x = tid; x < a.R * a.P; x += PG_THREADS) {
    const int i = a.by_p((uint32_t)x), l = x - i * a.P;
    const ForkRow r = rows[i];
    const int mine = r.parent >= 0 ? fork_entry(a, r.parent, l) : -1;
    const bool first = r.parent >= 0 && first_of[r.parent] == i;
    const int e = first || l < r.whole ? mine : -1;
    a.new_table[x] = e;
    if (e >= 0) atomicAdd(come + e, 1);
    if (l == r.whole && !first && r.rest > 0) rows[i].source = mine;
  }
  __syncthreads();
  int need = 0, base = 0;
  for (int i0 = 0; i0 < a.R; i0 += PG_THREADS) {
    const int i = i0 + tid;
    ForkRow r = {-1, 0, 0, -1};
    if (i < a.R) r = rows[i];
    int all;
    const int at = need + wg_before<PG_THREADS>(r.source >= 0, s, &all);
    if (r.source >= 0) a.copies[at] = {r.source, r.rest, i, r.whole};
    need += all;
  }
#pragma unroll
  for (int t = 0; t < FORK_ONE_PAGES / PG_PAGES; ++t) {
    if (t * PG_PAGES >= pages) break;
    const int x = t * PG_PAGES + 4 * tid;
    int c[4] = {1, 1, 1, 1}, all;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (x + u < (int)a.n_pages) c[u] = fork_count(refs[t][u], gone[x + u], come[x + u]);
    const int at = base + wg_before<PG_THREADS>((c[0] == 0) + (c[1] == 0) + (c[2] == 0) + (c[3] == 0), s, &all);
    fork_hand_out(a, x, c, at, need);
    base += all;
  }
  if (tid == 0) {
    a.got[0] = need < base ? need : base;
    a.missing[0] = need > base ? need - base : 0;
  }
}

// 16 bytes a thread at a time, two in flight, past the L2: what is copied is not read again soon (1920 copies of 56 KB, two at a time
// and four: 42.0 and 45 us, through the L2 46 and 50).  Of HIP's uint4 the compiler makes an array in LDS, three times slower.
__device__ __forceinline__ void copy_unit(const uint8_t* from, uint8_t* to, int bytes) {
  v4i x[PG_UNIT / 16 / PG_COPY];
#pragma unroll
  for (int u = 0; u < PG_UNIT / 16 / PG_COPY; ++u) {
    const int at = (u * PG_COPY + (int)threadIdx.x) * 16;
    if (at < bytes) x[u] = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(from + at));
  }
#pragma unroll
  for (int u = 0; u < PG_UNIT / 16 / PG_COPY; ++u) {
    const int at = (u * PG_COPY + (int)threadIdx.x) * 16;
    if (at < bytes) __builtin_nontemporal_store(x[u], reinterpret_cast<v4i*>(to + at));
  }
}

// How the units (chunks of PG_UNIT bytes, of keys and of values, of each layer) of a page fall on workgroups: unit w of page c follows unit
// w - 1, the workgroups take turns, and turn (pages, rest) is what one turn of all of them is, so that none divides.
struct CopyPlan {
  int units, chunks, turn_pages, turn_rest;
  UDiv by_units, by_chunks;
};

// f(c, layer, values?, offset into the page) for every unit of pages 0 .. n - 1 that is this workgroup's; the first one's page: copy_first.
__device__ __forceinline__ int copy_first(const CopyPlan& p) { return (int)p.by_units(blockIdx.x); }
template <class F>
__device__ __forceinline__ void each_unit(const CopyPlan& p, int c0, int n, F&& f) {
  int c = c0, w = (int)blockIdx.x - c0 * p.units;
  while (c < n) {
    const int lkv = p.by_chunks(w);
    f(c, lkv >> 1, lkv & 1, (int64_t)(w - lkv * p.chunks) * PG_UNIT);
    c += p.turn_pages;
    w += p.turn_rest;
    if (w >= p.units) {
      w -= p.units;
      ++c;
    }
  }
}

// The copies' written positions, and their entries of the table.
__global__ __launch_bounds__(PG_COPY) void fork_copy_kernel(ForkArgs a, CopyPlan plan) {
  const int c0 = copy_first(plan), got = a.got[0];
  const ForkCopy w0 = a.copies[c0];  // requested with the count, one round trip less: not looked at if it is not one
  const int fresh0 = a.fresh[c0];
  each_unit(plan, c0, got, [&](int c, int64_t layer, int values, int64_t at) {
    const ForkCopy w = c == c0 ? w0 : a.copies[c];
    const int fresh = c == c0 ? fresh0 : a.fresh[c];
    if (layer == 0 && !values && at == 0 && threadIdx.x == 0) a.new_table[(int64_t)w.row * a.P + w.column] = fresh;
    const int64_t bytes = w.rows * a.row_bytes - at;
    if (bytes <= 0) return;
    uint8_t* const base = (values ? a.v : a.k) + layer * a.layer_bytes + at;
    copy_unit(base + w.source * a.page_bytes, base + fresh * a.page_bytes, (int)(bytes < PG_UNIT ? bytes : PG_UNIT));
  });
}

// Numbering and copies in one launch for small tables and caches: every workgroup numbers the rows by itself, a thread to a row and to four
// pages, and the last one writes table and counts.  (us in two launches | one: 1 row into 8 over 64 pages, a layer 7.5 | 4.8, 24 layers 9.4 | 7.2; 16 rows
// into 16 of 13 columns 7.9 | 5.7; 64 into 64 of 8 8.0 | 6.1; but 200 into 250 of 4 8.2 | 9.2.)
constexpr int FORK_SMALL_PAGES = 4 * PG_COPY, FORK_SMALL_ROWS = PG_COPY, FORK_SMALL_ENTRIES = 1024;
constexpr int64_t FORK_SMALL_BYTES = (int64_t)1 << 27;  // copied at most
__global__ __launch_bounds__(PG_COPY) void fork_small_kernel(ForkArgs a, CopyPlan plan, int copy_wgs) {
  __shared__ int s[PG_COPY / 64], gone[FORK_SMALL_PAGES], come[FORK_SMALL_PAGES], first_of[FORK_SMALL_ROWS], slot[FORK_SMALL_ROWS], order[FORK_SMALL_ROWS],
      fresh[FORK_SMALL_ROWS];
  __shared__ ForkRow rows[FORK_SMALL_ROWS];
  const int tid = threadIdx.x, x0 = 4 * tid;
  const int64_t parent = tid < a.R ? a.parents[tid] : -1;
  int c[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    c[u] = x0 + u < (int)a.n_pages ? a.refs[x0 + u] : 1;
    gone[x0 + u] = come[x0 + u] = 0;
  }
  first_of[tid] = a.R;
  __syncthreads();
  ForkRow mine = {-1, 0, 0, -1};
  if (parent >= 0 && parent < a.B) {
    const int64_t n = fork_length(a, (int)parent);
    mine.parent = (int)parent;
    mine.whole = (int)(n / a.page);
    mine.rest = (int)(n - (int64_t)mine.whole * a.page);
    atomicMin(first_of + parent, tid);
  }
  rows[tid] = mine;
#pragma unroll 4
  for (int x = tid; x < a.B * a.P; x += PG_COPY) {
    const int64_t e = a.table[x];
    if (e >= 0 && e < a.n_pages) atomicAdd(gone + e, 1);
  }
  __syncthreads();
  // entry x of the new table, but that of a copy
  auto entry = [&](int x, int* row, int* copied) __attribute__((always_inline)) {
    const int i = a.by_p((uint32_t)x), l = x - i * a.P;
    const ForkRow r = rows[i];
    const int e = r.parent >= 0 ? fork_entry(a, r.parent, l) : -1;
    const bool first = r.parent >= 0 && first_of[r.parent] == i;
    *row = i;
    *copied = l == r.whole && !first && r.rest > 0 ? e : -1;
    return first || l < r.whole ? e : -1;
  };
#pragma unroll 4
  for (int x = tid; x < a.R * a.P; x += PG_COPY) {
    int i, copied;
    const int e = entry(x, &i, &copied);
    if (e >= 0) atomicAdd(come + e, 1);
    if (copied >= 0) rows[i].source = copied;
  }
  __syncthreads();
  int need, base;
  const bool wants = tid < a.R && rows[tid].source >= 0;
  const int mine_at = wg_before<PG_COPY>(wants, s, &need);
  slot[tid] = mine_at;
  if (wants) order[mine_at] = tid;
#pragma unroll
  for (int u = 0; u < 4; ++u) c[u] = x0 + u < (int)a.n_pages ? fork_count(c[u], gone[x0 + u], come[x0 + u]) : 1;
  int at = wg_before<PG_COPY>((c[0] == 0) + (c[1] == 0) + (c[2] == 0) + (c[3] == 0), s, &base);
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (c[u] == 0) {
      if (at < need) {
        fresh[at] = x0 + u;
        c[u] = 1;
      }
      ++at;
    }
  __syncthreads();
  const int got = need < base ? need : base;
  if ((int)blockIdx.x < copy_wgs) {
    each_unit(plan, copy_first(plan), got, [&](int k, int64_t layer, int values, int64_t from) {
      const int i = order[k];
      const int rest = __builtin_amdgcn_readfirstlane(rows[i].rest), source = __builtin_amdgcn_readfirstlane(rows[i].source);
      const int to = __builtin_amdgcn_readfirstlane(fresh[k]);
      const int64_t bytes = rest * a.row_bytes - from;
      if (bytes <= 0) return;
      uint8_t* const base = (values ? a.v : a.k) + layer * a.layer_bytes + from;
      copy_unit(base + source * a.page_bytes, base + to * a.page_bytes, (int)(bytes < PG_UNIT ? bytes : PG_UNIT));
    });
    return;
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (x0 + u < (int)a.n_pages) a.new_refs[x0 + u] = c[u];
  for (int x = tid; x < a.R * a.P; x += PG_COPY) {
    int i, copied;
    const int e = entry(x, &i, &copied);
    a.new_table[x] = copied < 0 ? e : slot[i] < got ? fresh[slot[i]] : -1;
  }
  if (tid == 0) a.missing[0] = need - got;
}

struct CompactArgs {
  const int64_t* table;  // entries in all
  const int32_t* refs;
  int64_t* new_table;
  int32_t* new_refs;
  int64_t* where;   // [n_pages] where a held page went, -1: free
  int32_t* live;    // [1]
  int32_t* source;  // [n_pages] of the k-th move: the k-th page held from the top,
  int32_t* hole;    // [n_pages] the k-th free one from the bottom
  int32_t* move;    // [n_pages] of a held page past the last place: which move is its own
  int32_t* moves;   // [1]
  int32_t* held;    // [segments] held pages of each segment
  uint8_t *k, *v;
  int64_t layer_bytes, page_bytes, n_pages, entries;
  int layers, copy_wgs, turns;
};

__device__ __forceinline__ void compact_refs(const CompactArgs& a, int64_t x, int (&r)[4]) {  // of the pages x .. x + 3 that are there (others: 0)
  if (x + 4 <= a.n_pages) {
    const v4i y = reinterpret_cast<const v4i*>(a.refs)[x / 4];
#pragma unroll
    for (int u = 0; u < 4; ++u) r[u] = y[u];
    return;
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) r[u] = x + u < a.n_pages ? a.refs[x + u] : 0;
}

__device__ __forceinline__ int compact_held(const CompactArgs& a, int64_t x) {
  int r[4] = {0, 0, 0, 0};
  if (x < a.n_pages) compact_refs(a, x, r);
  return (r[0] > 0) + (r[1] > 0) + (r[2] > 0) + (r[3] > 0);
}

__global__ __launch_bounds__(PG_COPY) void compact_count_kernel(CompactArgs a) {
  __shared__ int s[PG_COPY / 64];
  const int64_t i0 = (int64_t)blockIdx.x * a.turns * PG_COPY;
  const int n = wg_count<PG_COPY>(i0, i0 + (int64_t)a.turns * PG_COPY, s, [&](int64_t i) { return compact_held(a, 4 * i); });
  if (threadIdx.x == 0) a.held[blockIdx.x] = n;
}

// Numbers the pages: live of them are held, places 0 .. live - 1 are to hold them.  THREADS x 4 pages a turn.  Up to 16384 pages every
// workgroup counts what lies in front of its own turn, and all, by itself (COUNT): a launch less.  (60000 pages: 12.3 us; counted in
// segments first, 4.6 and 4.8.)
constexpr int COMPACT_COUNT = 16384;
template <int THREADS, bool COUNT>
__global__ __launch_bounds__(THREADS) void compact_rank_kernel(CompactArgs a) {
  __shared__ int s[THREADS / 64];
  const int64_t turns = COUNT ? 1 : a.turns, i0 = (int64_t)blockIdx.x * turns * THREADS;
  int before, live;
  if constexpr (COUNT) {
    auto held = [&](int64_t i) { return compact_held(a, 4 * i); };
    before = wg_count<THREADS>(0, i0, s, held);
    live = before + wg_count<THREADS>(i0, (a.n_pages + 3) / 4, s, held);
  } else {
    auto held = [&](int64_t i) { return a.held[i]; };
    before = wg_count<THREADS>(0, blockIdx.x, s, held);
    live = before + wg_count<THREADS>(blockIdx.x, gridDim.x, s, held);
  }
  for (int64_t turn = 0; turn < turns; ++turn) {
    const int64_t x = 4 * (i0 + turn * THREADS + threadIdx.x);
    int r[4] = {0, 0, 0, 0}, mine;
    if (x < a.n_pages) compact_refs(a, x, r);
    int at = before + wg_before<THREADS>((r[0] > 0) + (r[1] > 0) + (r[2] > 0) + (r[3] > 0), s, &mine);  // held pages in front of x
    before += mine;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t y = x + u;
      if (y >= a.n_pages) break;
      const bool held = r[u] > 0;
      a.where[y] = held && y < live ? y : -1;  // moved pages: their move says
      a.new_refs[y] = held && y < live ? r[u] : 0;
      if (held && y >= live) {
        a.source[live - 1 - at] = (int)y;
        a.move[y] = live - 1 - at;
      }
      if (!held && y < live) a.hole[y - at] = (int)y;
      at += held;
      if (y == live - 1) a.moves[0] = live - at;  // free pages among the first live
    }
    if (x == 0) {
      a.live[0] = live;
      if (live == 0) a.moves[0] = 0;
    }
  }
}

// Moves the pages; the workgroups behind those renumber the table and fill in the counts.  Sources lie behind the last place, holes in
// front of it: no page is both.
__global__ __launch_bounds__(PG_COPY) void compact_move_kernel(CompactArgs a, CopyPlan plan) {
  const int moves = a.moves[0];
  if ((int)blockIdx.x >= a.copy_wgs) {
    const int live = a.live[0];
    const int64_t stride = (int64_t)(gridDim.x - a.copy_wgs) * PG_COPY, me = (int64_t)((int)blockIdx.x - a.copy_wgs) * PG_COPY + threadIdx.x;
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
    return;
  }
  const int c0 = copy_first(plan), source0 = a.source[c0], hole0 = a.hole[c0];  // requested with the count
  each_unit(plan, c0, moves, [&](int c, int64_t layer, int values, int64_t at) {
    const int64_t left = a.page_bytes - at;
    uint8_t* const base = (values ? a.v : a.k) + layer * a.layer_bytes + at;
    copy_unit(base + (c == c0 ? source0 : a.source[c]) * a.page_bytes, base + (c == c0 ? hole0 : a.hole[c]) * a.page_bytes, (int)(left < PG_UNIT ? left : PG_UNIT));
  });
}

// Both of the above in one launch for small caches: every workgroup numbers all pages by itself, 4 to a thread, and keeps the moves in LDS.
// us in two launches | one, half the pages held: 128 pages of 64 KB 7.9 | 6.1, 128 of 256 KB 12.1 | 9.4, 512 of them (128 MB of keys) 29.7 | 28.4,
// but 1000 of them 49.5 | 51.1 and in two layers 105 | 114.  (16 pages to a thread, 4096 pages: 9.1 | 14.4.)
constexpr int COMPACT_SMALL = 4 * PG_COPY;
constexpr int64_t COMPACT_SMALL_BYTES = (int64_t)1 << 27;  // of all keys
__global__ __launch_bounds__(PG_COPY) void compact_small_kernel(CompactArgs a, CopyPlan plan) {
  __shared__ int s[PG_COPY / 64], moves_s, source[COMPACT_SMALL / 2], hole[COMPACT_SMALL / 2];
  const int x = (int)threadIdx.x * 4, n_pages = (int)a.n_pages;
  int r[4] = {0, 0, 0, 0}, live;
  if (x < n_pages) compact_refs(a, x, r);
  if (threadIdx.x == 0) moves_s = 0;
  const int at0 = wg_before<PG_COPY>((r[0] > 0) + (r[1] > 0) + (r[2] > 0) + (r[3] > 0), s, &live);
  int at = at0;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int y = x + u;
    const bool held = r[u] > 0;
    if (held && y >= live) source[live - 1 - at] = y;
    if (!held && y < live) hole[y - at] = y;
    at += held;
    if (y == live - 1) moves_s = live - at;  // free pages among the first live
  }
  __syncthreads();
  const int moves = moves_s;
  if ((int)blockIdx.x < a.copy_wgs) {
    each_unit(plan, copy_first(plan), moves, [&](int c, int64_t layer, int values, int64_t at) {
      const int64_t left = a.page_bytes - at;
      uint8_t* const base = (values ? a.v : a.k) + layer * a.layer_bytes + at;
      const int from = __builtin_amdgcn_readfirstlane(source[c]), to = __builtin_amdgcn_readfirstlane(hole[c]);
      copy_unit(base + from * a.page_bytes, base + to * a.page_bytes, (int)(left < PG_UNIT ? left : PG_UNIT));
    });
    return;
  }
  const int64_t stride = (int64_t)(gridDim.x - a.copy_wgs) * PG_COPY, me = (int64_t)((int)blockIdx.x - a.copy_wgs) * PG_COPY + threadIdx.x;
  for (int64_t i = me; i < a.entries; i += stride) {
    const int64_t e = a.table[i];
    int64_t to = -1;
    if (e >= 0 && e < n_pages && a.refs[e] > 0) {
      to = e;
      if (e >= live) {  // source[] falls
        int lo = 0;
        for (int step = COMPACT_SMALL / 4; step; step >>= 1)
          if (lo + step < moves && source[lo + step] >= (int)e) lo += step;
        to = hole[lo];
      }
    }
    a.new_table[i] = to;
  }
  if ((int)blockIdx.x != a.copy_wgs) return;
  at = at0;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int y = x + u;
    const bool held = r[u] > 0;
    if (y < n_pages) {
      a.where[y] = !held ? -1 : y < live ? y : hole[live - 1 - at];
      a.new_refs[y] = y >= live ? 0 : held ? r[u] : a.refs[source[y - at]];
    }
    at += held;
  }
  if (threadIdx.x == 0) a.live[0] = live;
}

// At most `most` pages are copied, at most `bytes` of each; 8 workgroups fill a compute unit.  Returns the workgroups.
static unsigned copy_plan(CopyPlan& p, int64_t most, int64_t layers, int64_t bytes) {
  const int64_t chunks = (bytes + PG_UNIT - 1) / PG_UNIT, units = 2 * layers * chunks, room = (int64_t)device_cus() * 8;
  const int64_t wgs = most < 1 ? 1 : most < room / units + 1 && most * units < room ? most * units : room;
  p.units = (int)units;
  p.chunks = (int)chunks;
  p.turn_pages = (int)(wgs / units);
  p.turn_rest = (int)(wgs - wgs / units * units);
  p.by_units = UDiv::of((uint32_t)units);
  p.by_chunks = UDiv::of((uint32_t)chunks);
  return (unsigned)wgs;
}

static int check_caches(const void* k, const void* v, int64_t layers, int64_t layer_bytes, int64_t n_pages, int64_t page_size, int64_t row_bytes) {
  if (layers <= 0 || n_pages <= 0 || page_size <= 0 || row_bytes <= 0) return AQ_E_SHAPE;
  if (layers > 4096 || n_pages > 0x7fffffff - PG_PAGES || page_size > (1 << 30) || row_bytes > (1 << 30) || page_size * row_bytes > (int64_t)1 << 31)
    return AQ_E_RANGE;  // (units of a copied page: 31 bits)
  if ((row_bytes & 15) || (layer_bytes & 15)) return AQ_E_ALIGN;
  if (layers > 1 && layer_bytes / row_bytes / page_size < n_pages) return AQ_E_SHAPE;  // layers that overlap
  if (!k || !v) return AQ_E_NULL;
  return check_ptr16(k) || check_ptr16(v) ? AQ_E_ALIGN : AQ_OK;
}

// Workspace of a fork: the list of copies, then the counts.
static int64_t fork_words(int64_t n_pages, int64_t R) { return 8 * R + (R + 4 + segments(n_pages) + 1) / 4 * 4 + 2 * ((n_pages + 3) / 4 * 4); }

}  // namespace aq

extern "C" int64_t aq_fork_pages_workspace_bytes(int64_t n_pages, int64_t R) {
  return n_pages <= 0 || R < 0 ? 0 : aq::fork_words(n_pages, R) * (int64_t)sizeof(int32_t);
}

extern "C" int aq_fork_pages(const int64_t* page_table, int64_t B, int64_t P, const int32_t* refs, const int64_t* parents, int64_t R,
                             int64_t total_len, const int64_t* seq_lens, void* k_layers, void* v_layers, int64_t layers,
                             int64_t layer_bytes, int64_t n_pages, int64_t page_size, int64_t row_bytes, int64_t* new_table,
                             int32_t* new_refs, int32_t* missing, void* workspace, int64_t workspace_bytes, void* stream) {
  if (B < 0 || R < 0 || P <= 0 || total_len < 0) return AQ_E_SHAPE;
  if (const int rc = aq::check_caches(k_layers, v_layers, layers, layer_bytes, n_pages, page_size, row_bytes)) return rc;
  if (B > (1 << 24) || R > (1 << 16) || P > 0x7fffffff) return AQ_E_RANGE;  // (every row looks for earlier siblings)
  if (total_len > P * page_size) return AQ_E_SHAPE;  // positions the page table does not cover
  if ((B > 0 && !page_table) || (R > 0 && (!parents || !new_table)) || !refs || !new_refs || !missing || !workspace) return AQ_E_NULL;
  if (aq::check_ptr(page_table, 8) || aq::check_ptr(parents, 8) || aq::check_ptr(seq_lens, 8) || aq::check_ptr(new_table, 8) ||
      aq::check_ptr16(refs) || aq::check_ptr(new_refs, 4) || aq::check_ptr(missing, 4) || aq::check_ptr16(workspace))
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
  a.wants = static_cast<aq::ForkCopy*>(workspace);
  a.copies = a.wants + R;
  a.fresh = reinterpret_cast<int32_t*>(a.copies + R);
  a.got = a.fresh + R;
  a.need = a.got + 1;
  a.free_pages = a.need + 1;
  a.gone = a.fresh + (R + 4 + aq::segments(n_pages) + 1) / 4 * 4;
  a.come = a.gone + (n_pages + 3) / 4 * 4;
  a.k = static_cast<uint8_t*>(k_layers);
  a.v = static_cast<uint8_t*>(v_layers);
  a.layer_bytes = layer_bytes;
  a.row_bytes = row_bytes;
  a.page_bytes = page_size * row_bytes;
  a.page = (int)page_size;
  a.T = total_len;
  a.n_pages = n_pages;
  a.B = (int)B;
  a.R = (int)R;
  a.P = (int)P;
  a.layers = (int)layers;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 one(aq::PG_THREADS), threads(aq::PG_COPY);
  // Written rows of a page that is partly filled: one number for all, or anything where sequences have lengths of their own.
  const int64_t written = !seq_lens ? total_len % page_size : total_len < page_size ? total_len : page_size - 1;
  aq::CopyPlan plan{};
  unsigned copy_wgs = 0;  // (a single row is its parent's first child)
  if (R > 1 && written > 0) copy_wgs = aq::copy_plan(plan, R - 1, layers, written * row_bytes);
  if (P <= aq::FORK_ONE_ENTRIES) a.by_p = aq::UDiv::of((uint32_t)P);
  if (n_pages <= aq::FORK_SMALL_PAGES && B <= aq::FORK_SMALL_ROWS && R <= aq::FORK_SMALL_ROWS && (B + R) * P <= aq::FORK_SMALL_ENTRIES &&
      2 * layers * R * written * row_bytes <= aq::FORK_SMALL_BYTES) {
    aq::queue_kernel(aq::fork_small_kernel, dim3(copy_wgs + 1), threads, 0, st, a, plan, (int)copy_wgs);
    return (int)hipGetLastError();
  }
  if (n_pages <= aq::FORK_ONE_PAGES && B <= aq::FORK_ONE_ROWS && R <= aq::FORK_ONE_ROWS && (B + R) * P <= aq::FORK_ONE_ENTRIES) {
    aq::queue_kernel(aq::fork_one_kernel, dim3(1), one, aq::fork_one_lds(n_pages, B, R), st, a);
  } else {
    const int64_t quads = (n_pages + 3) / 4 * 2, groups = aq::segments(n_pages);
    a.turns = (int)aq::segment_turns(n_pages);
    const int64_t chunks = (P + aq::PG_COPY - 1) / aq::PG_COPY, new_wgs = (R + aq::FORK_ROWS - 1) / aq::FORK_ROWS * chunks;
    const int64_t wgs = new_wgs + (B + aq::FORK_ROWS - 1) / aq::FORK_ROWS * chunks;
    if (wgs > 0x7fffffff) return AQ_E_RANGE;
    aq::queue_kernel(aq::fork_clear_kernel, dim3((unsigned)((quads + aq::PG_THREADS - 1) / aq::PG_THREADS)), one, 0, st,
                     reinterpret_cast<v4i*>(a.gone), quads);
    if (wgs > 0) aq::queue_kernel(aq::fork_rows_kernel, dim3((unsigned)wgs), threads, 0, st, a, (int)new_wgs, (int)chunks);
    aq::queue_kernel(aq::fork_free_kernel, dim3((unsigned)groups + 1), threads, 0, st, a);
    aq::queue_kernel(aq::fork_refs_kernel, dim3((unsigned)groups), threads, 0, st, a);
  }
  if (copy_wgs) aq::queue_kernel(aq::fork_copy_kernel, dim3(copy_wgs), threads, 0, st, a, plan);
  return (int)hipGetLastError();
}

extern "C" int64_t aq_compact_pages_workspace_bytes(int64_t n_pages) {
  return n_pages <= 0 ? 0 : (3 * n_pages + 1 + aq::segments(n_pages)) * (int64_t)sizeof(int32_t);
}

extern "C" int aq_compact_pages(const int64_t* page_table, int64_t entries, const int32_t* refs, void* k_layers, void* v_layers,
                                int64_t layers, int64_t layer_bytes, int64_t n_pages, int64_t page_size, int64_t row_bytes,
                                int64_t* new_table, int32_t* new_refs, int64_t* where, int32_t* live, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  if (entries < 0) return AQ_E_SHAPE;
  if (const int rc = aq::check_caches(k_layers, v_layers, layers, layer_bytes, n_pages, page_size, row_bytes)) return rc;
  if ((entries > 0 && (!page_table || !new_table)) || !refs || !new_refs || !where || !live || !workspace) return AQ_E_NULL;
  if (aq::check_ptr(page_table, 8) || aq::check_ptr(new_table, 8) || aq::check_ptr(where, 8) || aq::check_ptr16(refs) ||
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
  a.held = a.moves + 1;
  a.turns = (int)aq::segment_turns(n_pages);
  a.k = static_cast<uint8_t*>(k_layers);
  a.v = static_cast<uint8_t*>(v_layers);
  a.layer_bytes = layer_bytes;
  a.page_bytes = page_size * row_bytes;
  a.n_pages = n_pages;
  a.entries = entries;
  a.layers = (int)layers;
  hipStream_t st = static_cast<hipStream_t>(stream);
  aq::CopyPlan plan;
  a.copy_wgs = (int)aq::copy_plan(plan, n_pages / 2, layers, a.page_bytes);
  const int64_t work = entries > n_pages / 2 ? entries : n_pages / 2, rest = (work + aq::PG_COPY - 1) / aq::PG_COPY;
  const dim3 wgs((unsigned)(a.copy_wgs + (rest < 1 ? 1 : rest < 256 ? rest : 256))), threads(aq::PG_COPY);
  if (n_pages <= aq::COMPACT_SMALL && layers * n_pages * a.page_bytes <= aq::COMPACT_SMALL_BYTES) {
    aq::queue_kernel(aq::compact_small_kernel, wgs, threads, 0, st, a, plan);
    return (int)hipGetLastError();
  }
  if (n_pages <= aq::COMPACT_COUNT) {
    aq::queue_kernel(aq::compact_rank_kernel<aq::PG_THREADS, true>, dim3((unsigned)((n_pages + aq::PG_PAGES - 1) / aq::PG_PAGES)), dim3(aq::PG_THREADS), 0, st, a);
  } else {
    const dim3 groups((unsigned)aq::segments(n_pages));
    aq::queue_kernel(aq::compact_count_kernel, groups, threads, 0, st, a);
    aq::queue_kernel(aq::compact_rank_kernel<aq::PG_COPY, false>, groups, threads, 0, st, a);
  }
  aq::queue_kernel(aq::compact_move_kernel, wgs, threads, 0, st, a, plan);
  return (int)hipGetLastError();
}
