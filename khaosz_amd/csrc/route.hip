// The two ends of a layer of routed experts: from the router's logits to each token's experts and the order in which the experts work
// through the tokens, and from the experts' outputs back to the tokens.
//
// route: a token's k largest logits x_1 >= .. >= x_k (equal ones: the lowest expert first), their weights exp(x_j - x_1) / sum, and a
// counting sort of the T k choices by expert, in the tokens' order inside an expert.  16 lanes hold a token's logits as keys that order like
// (logit, lowest index), so that a choice is a maximum over a few registers and four DPP steps.  A token names an expert at most once:
// a workgroup's 64 tokens leave a bit each in a 64-bit word per expert (an OR: any order gives the same word), and the number of
// bits below a token's own is its place among them.  No atomic whose order shows.
// What bounds it: launches and chains of latencies; the bytes (10.5 MB for 16384 tokens of 256 experts) would take 2 us.  Measured: 1 token's 6 of 64 experts
// 3.6 us (one launch), 333 tokens' 4 of 60 8.2 (two launches, the host's time), 16384 tokens' 8 of 256 15.0 (three: choices 8.7, sums 4.1, rows 4.1 under
// the profiler).  A workgroup of 256 threads for up to 16 tokens is level (64 experts) to 0.4 us faster (256): not built.
#include <type_traits>

#include "aq_grouped.h"

namespace aq {

constexpr int RT_THREADS = 1024, RT_TOKENS = RT_THREADS / 16;  // a workgroup's tokens: 16 lanes each
constexpr int RT_ONE_PASSES = 2;  // of the kernel that does it all in one workgroup (64 experts, 6 choices: 128 tokens 6.1 us, by two launches 6.7; 256 10.0 and 6.7)
constexpr int RT_FEW_THREADS = 256, RT_FEW_TOKENS = RT_FEW_THREADS / 16, RT_FEW_T = 2048;  // up to RT_FEW_T tokens: more, smaller workgroups
constexpr int RT_MAX_E = 512, RT_MAX_K = 16;
constexpr int RT_MOST_CHUNKS = 512;  // larger batches: more passes to a chunk
constexpr int RT_GROUP = RT_TOKENS / RT_FEW_TOKENS;  // chunks of a workgroup that hands out rows, at most

struct RouteArgs {
  const void* logits;
  int64_t ld;  // logits between tokens
  float* weights;
  int32_t *experts, *rows, *tokens, *offsets;
  uint16_t* counts;            // [chunks][pitch]
  uint32_t *before, *totals;   // [chunks][pitch], [pitch]: many chunks
  int T, E, k, renormalize, passes, chunks;
  int chunk;  // tokens of a chunk
  int group;  // chunks of a workgroup that hands out rows
  int pitch;  // of counts
  int whole;  // lanes' runs of logits are whole, aligned vectors
};

typedef unsigned long long u64;
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}
template <int CTRL>
__device__ __forceinline__ u64 dpp(u64 v) {
  return (u64)dpp<CTRL>((uint32_t)(v >> 32)) << 32 | dpp<CTRL>((uint32_t)v);
}
template <class K>
__device__ __forceinline__ K larger(K a, K b) {
  return a > b ? a : b;
}
// over each row of 16 lanes, in all of them
template <class K>
__device__ __forceinline__ K row_max(K v) {
  v = larger(v, dpp<0xB1>(v));
  v = larger(v, dpp<0x4E>(v));
  v = larger(v, dpp<0x141>(v));
  return larger(v, dpp<0x140>(v));
}
__device__ __forceinline__ float row_sum(float v) {
  v += __uint_as_float(dpp<0xB1>(__float_as_uint(v)));
  v += __uint_as_float(dpp<0x4E>(__float_as_uint(v)));
  v += __uint_as_float(dpp<0x141>(__float_as_uint(v)));
  return v + __uint_as_float(dpp<0x140>(__float_as_uint(v)));
}

// A key per logit: its bits, made to order like the number, then the expert's number counted down.  bf16 logits have room for both in
// 32 bits.  0: not to be chosen (-inf, NaN).
template <bool BF16>
struct Key;
template <>
struct Key<true> {
  using type = uint32_t;
  // logits l V .. l V + V - 1 of token t, as the bits of fp32; -inf behind the last
  template <int V>
  static __device__ __forceinline__ void load(const RouteArgs& a, int t, int l, uint32_t (&bits)[V]) {
    const uint16_t* const p = static_cast<const uint16_t*>(a.logits) + (int64_t)t * a.ld + l * V;
    if (a.whole && t < a.T) {
#pragma unroll
      for (int v = 0; v < V; v += 4) {
        const uint2 q = *reinterpret_cast<const uint2*>(p + v);
        bits[v] = q.x << 16, bits[v + 1] = q.x & 0xffff0000u, bits[v + 2] = q.y << 16, bits[v + 3] = q.y & 0xffff0000u;
      }
      return;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) bits[v] = t < a.T && l * V + v < a.E ? (uint32_t)p[v] << 16 : 0xff800000u;
  }
  static __device__ __forceinline__ type make(uint32_t ordered, int e) { return (ordered & 0xffff0000u) | (0xffffu - (uint32_t)e); }
  static __device__ __forceinline__ int expert(type k) { return (int)(0xffffu - (k & 0xffffu)); }
  static __device__ __forceinline__ float value(type k) { return __uint_as_float((k >> 31 ? k ^ 0x80000000u : ~k) & 0xffff0000u); }
};
template <>
struct Key<false> {
  using type = u64;
  template <int V>
  static __device__ __forceinline__ void load(const RouteArgs& a, int t, int l, uint32_t (&bits)[V]) {
    const uint32_t* const p = static_cast<const uint32_t*>(a.logits) + (int64_t)t * a.ld + l * V;
    if (a.whole && t < a.T) {
#pragma unroll
      for (int v = 0; v < V; v += 4) {
        const uint4 q = *reinterpret_cast<const uint4*>(p + v);
        bits[v] = q.x, bits[v + 1] = q.y, bits[v + 2] = q.z, bits[v + 3] = q.w;
      }
      return;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) bits[v] = t < a.T && l * V + v < a.E ? p[v] : 0xff800000u;
  }
  static __device__ __forceinline__ type make(uint32_t ordered, int e) { return (u64)ordered << 32 | (0xffffu - (uint32_t)e); }
  static __device__ __forceinline__ int expert(type k) { return (int)(0xffffu - ((uint32_t)k & 0xffffu)); }
  static __device__ __forceinline__ float value(type k) {
    const uint32_t h = (uint32_t)(k >> 32);
    return __uint_as_float(h >> 31 ? h ^ 0x80000000u : ~h);
  }
};

// exp(x - most), most the largest of them: 1 for it, infinite or not.
__device__ __forceinline__ float exp_below(float x, float most) {
  const float e = exp_hw(fmaxf(x - most, -150.0f));  // (2^-216 is 0)
  return x == most ? 1.0f : e;
}

// The choices of token t by the 16 lanes that hold it: lane j has choice j < k (expert -1: there is none) and its weight.
template <bool BF16, int V>
__device__ __forceinline__ int choose(const RouteArgs& a, int t, int l, float* weight) {
  using K = Key<BF16>;
  using key_t = typename K::type;
  key_t key[V];
  uint32_t bits[V];
  K::template load<V>(a, t, l, bits);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float x = __uint_as_float(bits[v]) + 0.0f;  // (-0 counts as 0)
    const uint32_t u = __float_as_uint(x);
    key[v] = x > -__builtin_inff() ? K::make(u >> 31 ? ~u : u | 0x80000000u, l * V + v) : 0;
  }
  key_t b = key[0], mine = 0;
#pragma unroll
  for (int v = 1; v < V; ++v) b = larger(b, key[v]);
  b = row_max(b);
  const float most = K::value(b);
  float total = 0.0f;
  if (!a.renormalize && b) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (key[v]) total += exp_below(K::value(key[v]), most);
    total = row_sum(total);
  }
  for (int j = 0;;) {
    if (l == j) mine = b;
    if (++j == a.k) break;
    // the largest key below b: those that are not wrap around in the difference and come last
    key_t d = key[0] - b;
#pragma unroll
    for (int v = 1; v < V; ++v) d = larger(d, key[v] - b);
    b = b ? row_max(d) + b : 0;
  }
  const float e = mine ? exp_below(K::value(mine), most) : 0.0f;
  const float chosen = row_sum(e);
  *weight = mine ? e / (a.renormalize ? chosen : total) : 0.0f;
  return mine ? K::expert(mine) : -1;
}

// first[e] = total of the experts before e, for e <= E, by one wavefront
__device__ __forceinline__ void experts_scan(const uint32_t* counts, uint32_t* first, int E, int lane) {
  constexpr int PER = RT_MAX_E / 64;
  int c[PER], sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane * PER + i;
    c[i] = e < E ? (int)counts[e] : 0;
    sum += c[i];
  }
  int at = wave_scan(sum) - sum;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane * PER + i;
    if (e <= E) first[e] = (uint32_t)at;
    at += c[i];
  }
  if (lane == 63 && E == RT_MAX_E) first[E] = (uint32_t)at;
}

// ONE: all tokens in one workgroup's passes, rows handed out at the end.  Otherwise a chunk of `passes` passes: the choices, each with its
// place among the chunk's choices of its expert (in `rows` until the next launch), and the chunk's counts.
template <bool BF16, int V, int THREADS, bool ONE>
__global__ __launch_bounds__(THREADS) void route_choose_kernel(RouteArgs a) {
  constexpr int TOKENS = THREADS / 16;
  __shared__ u64 asked[RT_MAX_E];
  __shared__ uint32_t count[RT_MAX_E], first[RT_MAX_E + 1];
  const int tid = threadIdx.x, lane = tid & 63, l = lane & 15, place = tid >> 4;
  for (int e = tid; e < a.E; e += THREADS) count[e] = 0;
  int chose[ONE ? RT_ONE_PASSES : 1], rank[ONE ? RT_ONE_PASSES : 1];
  auto pass = [&](int t, int& ce, int& cr) {
    for (int e = tid; e < a.E; e += THREADS) asked[e] = 0;
    float w;
    ce = choose<BF16, V>(a, t, l, &w);
    __syncthreads();
    if (ce >= 0) atomicOr(&asked[ce], 1ull << place);
    __syncthreads();
    cr = ce >= 0 ? (int)count[ce] + __popcll(asked[ce] & ((1ull << place) - 1)) : -1;
    if (t < a.T && l < a.k) {
      const int64_t at = (int64_t)t * a.k + l;
      a.weights[at] = w;
      a.experts[at] = ce;
      if constexpr (!ONE) a.rows[at] = cr;
    }
    __syncthreads();
    for (int e = tid; e < a.E; e += THREADS) count[e] += (uint32_t)__popcll(asked[e]);
  };
  if constexpr (ONE) {
#pragma unroll
    for (int i = 0; i < RT_ONE_PASSES; ++i) {
      chose[i] = rank[i] = -1;
      if (i * TOKENS < a.T) pass(i * TOKENS + place, chose[i], rank[i]);
    }
    __syncthreads();
    if (tid < 64) experts_scan(count, first, a.E, lane);
    __syncthreads();
    for (int e = tid; e <= a.E; e += THREADS) a.offsets[e] = (int32_t)first[e];
#pragma unroll
    for (int i = 0; i < RT_ONE_PASSES; ++i) {
      const int t = i * TOKENS + place;
      if (t < a.T && l < a.k) {
        const int r = chose[i] >= 0 ? (int)first[chose[i]] + rank[i] : -1;
        a.rows[t * a.k + l] = r;
        if (r >= 0) a.tokens[r] = t;
      }
    }
    for (int r = (int)first[a.E] + tid; r < a.T * a.k; r += THREADS) a.tokens[r] = -1;
  } else {
    for (int i = 0; i < a.passes; ++i) pass(((int)blockIdx.x * a.passes + i) * TOKENS + place, chose[0], rank[0]);
    __syncthreads();
    for (int e = tid; e < a.E; e += THREADS) a.counts[(int64_t)blockIdx.x * a.pitch + e] = (uint16_t)count[e];
  }
}

// Many chunks: each expert's choices in the chunks before, summed once for everybody.  A workgroup has 32 experts, two to a thread, and its 16 rows of
// threads a run of chunks each.
constexpr int RT_SUM_THREADS = 256, RT_SUM_E = 32, RT_SUM_RUNS = RT_SUM_THREADS * 2 / RT_SUM_E;
__global__ __launch_bounds__(RT_SUM_THREADS) void route_sums_kernel(RouteArgs a) {
  __shared__ uint32_t run_sum[RT_SUM_RUNS][RT_SUM_E];
  const int e = (int)blockIdx.x * RT_SUM_E + 2 * (threadIdx.x & (RT_SUM_E / 2 - 1)), run = threadIdx.x / (RT_SUM_E / 2), i = e & (RT_SUM_E - 1);
  const int per = (a.chunks + RT_SUM_RUNS - 1) / RT_SUM_RUNS, c0 = run * per, c1 = c0 + per < a.chunks ? c0 + per : a.chunks;
  auto counts = [&](int c) { return *reinterpret_cast<const uint32_t*>(a.counts + (int64_t)c * a.pitch + e); };
  uint32_t lo = 0, hi = 0;
  if (e < a.E) {
#pragma unroll 16
    for (int c = c0; c < c1; ++c) {
      const uint32_t two = counts(c);
      lo += two & 0xffffu, hi += two >> 16;
    }
  }
  run_sum[run][i] = lo, run_sum[run][i + 1] = hi;
  __syncthreads();
  if (e >= a.E) return;
  uint32_t at_lo = 0, at_hi = 0, all_lo = 0, all_hi = 0;
#pragma unroll
  for (int r = 0; r < RT_SUM_RUNS; ++r) {
    const uint32_t x = run_sum[r][i], y = run_sum[r][i + 1];
    if (r < run) at_lo += x, at_hi += y;
    all_lo += x, all_hi += y;
  }
  if (run == 0) *reinterpret_cast<uint2*>(a.totals + e) = make_uint2(all_lo, all_hi);
#pragma unroll 16
  for (int c = c0; c < c1; ++c) {
    const uint32_t two = counts(c);
    *reinterpret_cast<uint2*>(a.before + (int64_t)c * a.pitch + e) = make_uint2(at_lo, at_hi);
    at_lo += two & 0xffffu, at_hi += two >> 16;
  }
}

// Rows for the choices of a group of chunks: the experts' first rows, the choices of the chunks before, the place among the chunk's.  Few
// chunks: every workgroup adds up all their counts by itself (256 workgroups, chunks and experts: 15 us, SUMMED 4 and 4).  Its first choices (of 64 tokens:
// all there are) are on their way meanwhile.
template <bool SUMMED>
__global__ __launch_bounds__(RT_THREADS) void route_rows_kernel(RouteArgs a) {
  __shared__ uint32_t total[RT_MAX_E], before[RT_MAX_E], first[RT_MAX_E + 1], base[RT_GROUP][RT_MAX_E];
  const int tid = threadIdx.x, E = a.E;
  const int c0 = (int)blockIdx.x * a.group;
  const int64_t all = (int64_t)a.T * a.k, from = (int64_t)c0 * a.chunk * a.k;
  const int64_t room = (int64_t)a.group * a.chunk * a.k, to = from + room < all ? from + room : all;
  int64_t s = from + tid;
  int expert = -1, place = 0;
  if (s < to) expert = a.experts[s], place = a.rows[s];
  if constexpr (SUMMED) {
    for (int i = tid; i < E; i += RT_THREADS) {
      total[i] = a.totals[i];
      before[i] = a.before[(int64_t)blockIdx.x * a.pitch + i];
      base[0][i] = 0;
    }
    __syncthreads();
  } else {
    for (int i = tid; i < E; i += RT_THREADS) total[i] = before[i] = 0;
    __syncthreads();
    int width = 32;  // threads to a chunk's counts, two experts each
    while (2 * width < E) width *= 2;
    const int e = 2 * (tid & (width - 1)), turns = RT_THREADS / width;
    if (e < E) {
      uint32_t sum[2] = {0, 0}, early[2] = {0, 0};
#pragma unroll 16
      for (int c = tid / width; c < a.chunks; c += turns) {
        const uint32_t two = *reinterpret_cast<const uint32_t*>(a.counts + (int64_t)c * a.pitch + e);
        const uint32_t n[2] = {two & 0xffffu, two >> 16};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          sum[i] += n[i];
          early[i] += c < c0 ? n[i] : 0;
          if (c >= c0 && c < c0 + a.group && e + i < E) base[c - c0][e + i] = n[i];
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (e + i < E) {
          atomicAdd(&total[e + i], sum[i]);  // whole numbers: any order
          atomicAdd(&before[e + i], early[i]);
        }
    }
    __syncthreads();
  }
  if (tid < 64) experts_scan(total, first, E, tid);
  __syncthreads();
  for (int i = tid; i < E; i += RT_THREADS) {
    uint32_t at = first[i] + before[i];
    for (int c = 0; c < a.group; ++c) {
      const uint32_t n = base[c][i];
      base[c][i] = at;
      at += n;
    }
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int i = tid; i <= E; i += RT_THREADS) a.offsets[i] = (int32_t)first[i];
  while (s < to) {
    if (expert >= 0) {
      const int t = (int)((uint32_t)s / (uint32_t)a.k), r = (int)base[a.group == 1 ? 0 : (t - c0 * a.chunk) / a.chunk][expert] + place;
      a.rows[s] = r;
      a.tokens[r] = t;
    }
    s += RT_THREADS;
    if (s < to) expert = a.experts[s], place = a.rows[s];
  }
  for (int64_t r = (int64_t)first[E] + (int64_t)blockIdx.x * RT_THREADS + tid; r < all; r += (int64_t)gridDim.x * RT_THREADS) a.tokens[r] = -1;
}

static int route_passes(int64_t T) {
  const int64_t n = (T + RT_TOKENS - 1) / RT_TOKENS;
  return (int)((n + RT_MOST_CHUNKS - 1) / RT_MOST_CHUNKS);
}
static int64_t route_chunk(int64_t T) { return T <= RT_FEW_T ? RT_FEW_TOKENS : (int64_t)route_passes(T) * RT_TOKENS; }
static int64_t route_chunks(int64_t T) { return (T + route_chunk(T) - 1) / route_chunk(T); }

// Whether the counts are summed by a launch of their own (64 experts, 4096 tokens: 10.4 us, without it 7.6; 256 and 16384: 15.3 and 21.8).
// (Its chunks are a workgroup's each: not those of RT_FEW_TOKENS.)
static bool route_sums(int64_t T, int64_t E) { return T > RT_FEW_T && route_chunks(T) * E > 16384; }

template <bool BF16, int V>
static void launch_route(const RouteArgs& a, hipStream_t st) {
  if (a.T <= RT_ONE_PASSES * RT_TOKENS) {
    queue_kernel((route_choose_kernel<BF16, V, RT_THREADS, true>), dim3(1), dim3(RT_THREADS), 0, st, a);
    return;
  }
  if (a.T <= RT_FEW_T)
    queue_kernel((route_choose_kernel<BF16, V, RT_FEW_THREADS, false>), dim3((unsigned)a.chunks), dim3(RT_FEW_THREADS), 0, st, a);
  else
    queue_kernel((route_choose_kernel<BF16, V, RT_THREADS, false>), dim3((unsigned)a.chunks), dim3(RT_THREADS), 0, st, a);
  const dim3 groups((unsigned)((a.chunks + a.group - 1) / a.group)), threads(RT_THREADS);
  if (!route_sums(a.T, a.E)) {
    queue_kernel(route_rows_kernel<false>, groups, threads, 0, st, a);
  } else {
    queue_kernel(route_sums_kernel, dim3((unsigned)((a.E + RT_SUM_E - 1) / RT_SUM_E)), dim3(RT_SUM_THREADS), 0, st, a);
    queue_kernel(route_rows_kernel<true>, groups, threads, 0, st, a);
  }
}
template <bool BF16>
static void launch_route(const RouteArgs& a, hipStream_t st) {
  if (a.E <= 64) launch_route<BF16, 4>(a, st);
  else if (a.E <= 128) launch_route<BF16, 8>(a, st);
  else if (a.E <= 256) launch_route<BF16, 16>(a, st);
  else launch_route<BF16, 32>(a, st);
}

// ---- the experts' outputs back to the tokens ------------------------------------------------------------------------
// out[t] = sum_j weights[t, j] y[rows[t, j]] (+ residual[t]), in fp32 in the order of j, the residual last, rounded once.  A wavefront has 64
// units of 16 bytes of a token's row (VEC; single values where rows are not whole units): its rows and weights are scalar loads, and it asks for up
// to 8 rows before it adds the first.  What bounds it: HBM (16384 tokens' 8 of 2048 bf16 with the residual: 565 MB in 111 us, 5.1 TB/s); a few tokens: the
// launch (11 tokens 4.0 us).
struct CombineArgs {
  const void *y, *res;
  void* out;
  const int32_t* rows;
  const float* weights;
  int64_t waves, R;
  int k, per;  // units of a token
  UDiv chunks; // wavefronts of a token
  int n_chunks;
};

template <bool BF16, bool VEC>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a) {
  constexpr int N = VEC ? (BF16 ? 8 : 4) : 1, AHEAD = 8;
  using unit = std::conditional_t<VEC, uint4, std::conditional_t<BF16, uint16_t, uint32_t>>;
  const int64_t w = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (w >= a.waves) return;
  const int t = (int)a.chunks((uint32_t)w), u = ((int)w - t * a.n_chunks) * 64 + (int)(threadIdx.x & 63);
  const bool in = u < a.per;
  auto at = [&](const void* p, int64_t row) { return static_cast<const unit*>(p) + row * a.per + u; };
  auto value = [](const unit& q, int c) {
    if constexpr (!VEC) return BF16 ? bf16_bits_to_f32(q) : __uint_as_float(q);
    else {
      const uint32_t* const d = &q.x;
      if constexpr (!BF16) return __uint_as_float(d[c]);
      else return __uint_as_float(c & 1 ? d[c / 2] & 0xffff0000u : d[c / 2] << 16);
    }
  };
  const int32_t* const rows = a.rows + (int64_t)t * a.k;
  const float* const weights = a.weights + (int64_t)t * a.k;
  float sum[N];
#pragma unroll
  for (int c = 0; c < N; ++c) sum[c] = 0.0f;
  unit r{};
  if (a.res && in) r = *at(a.res, t);
  for (int j0 = 0; j0 < a.k; j0 += AHEAD) {
    int row[AHEAD];
    unit q[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      row[j] = j0 + j < a.k ? rows[j0 + j] : -1;
      if (row[j] >= a.R) row[j] = -1;
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (row[j] >= 0 && in) q[j] = *at(a.y, row[j]);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (row[j] >= 0) {
        const float x = weights[j0 + j];
#pragma unroll
        for (int c = 0; c < N; ++c) sum[c] += x * value(q[j], c);
      }
  }
  if (a.res) {
#pragma unroll
    for (int c = 0; c < N; ++c) sum[c] += value(r, c);
  }
  if (!in) return;
  unit* const out = static_cast<unit*>(a.out) + (int64_t)t * a.per + u;
  if constexpr (VEC && BF16) *out = make_uint4(pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3]), pack_bf16x2(sum[4], sum[5]), pack_bf16x2(sum[6], sum[7]));
  else if constexpr (VEC) *out = make_uint4(__float_as_uint(sum[0]), __float_as_uint(sum[1]), __float_as_uint(sum[2]), __float_as_uint(sum[3]));
  else if constexpr (BF16) *out = (uint16_t)f32_to_bf16_bits(sum[0]);
  else *out = __float_as_uint(sum[0]);
}

}  // namespace aq

extern "C" int64_t aq_route_topk_workspace_bytes(int64_t T, int64_t E) {
  if (T <= aq::RT_ONE_PASSES * aq::RT_TOKENS || T > (int64_t)1 << 24 || E <= 0) return 0;
  const int64_t chunks = aq::route_chunks(T), pitch = (E + 1) / 2 * 2;
  return (aq::route_sums(T, E) ? (chunks + 1) * pitch * 4 : 0) + chunks * pitch * 2;
}

extern "C" int aq_route_topk(const void* logits, int dtype, int64_t T, int64_t E, int64_t ld, int64_t k, int renormalize, float* weights,
                             int32_t* experts, int32_t* rows, int32_t* tokens, int32_t* offsets, void* workspace, int64_t workspace_bytes,
                             void* stream) {
  if (dtype != AQ_F32 && dtype != AQ_BF16) return AQ_E_DTYPE;
  if (T < 0 || E <= 0 || k <= 0 || k > E || ld < E) return AQ_E_SHAPE;
  if (E > aq::RT_MAX_E || k > aq::RT_MAX_K || T > (int64_t)1 << 24) return AQ_E_RANGE;
  if (!offsets || (T > 0 && (!logits || !weights || !experts || !rows || !tokens))) return AQ_E_NULL;
  if (aq::check_ptr(logits, dtype == AQ_BF16 ? 2 : 4) || aq::check_ptr(weights, 4) || aq::check_ptr(experts, 4) || aq::check_ptr(rows, 4) ||
      aq::check_ptr(tokens, 4) || aq::check_ptr(offsets, 4))
    return AQ_E_ALIGN;
  const int64_t need = aq_route_topk_workspace_bytes(T, E);
  if (need > 0 && !workspace) return AQ_E_NULL;
  if (workspace_bytes < need) return AQ_E_WORKSPACE;
  if (need > 0 && aq::check_ptr(workspace, 8)) return AQ_E_ALIGN;
  aq::RouteArgs a{};
  a.logits = logits;
  a.ld = ld;
  a.weights = weights;
  a.experts = experts;
  a.rows = rows;
  a.tokens = tokens;
  a.offsets = offsets;
  a.T = (int)T;
  a.E = (int)E;
  a.k = (int)k;
  a.renormalize = renormalize != 0;
  a.passes = T <= aq::RT_FEW_T ? 1 : aq::route_passes(T);
  a.chunk = T > 0 ? (int)aq::route_chunk(T) : 0;
  a.group = T <= aq::RT_FEW_T ? aq::RT_GROUP : 1;
  a.chunks = T > 0 ? (int)aq::route_chunks(T) : 0;
  a.pitch = (int)((E + 1) / 2 * 2);
  a.totals = static_cast<uint32_t*>(workspace);  // (many chunks; then their sums, then the counts)
  a.before = a.totals + a.pitch;
  a.counts = reinterpret_cast<uint16_t*>(aq::route_sums(T, E) ? a.before + (int64_t)a.chunks * a.pitch : a.totals);
  const int run = E <= 64 ? 4 : E <= 128 ? 8 : E <= 256 ? 16 : 32, unit = dtype == AQ_BF16 ? 8 : 16;  // a lane's logits; bytes of four
  a.whole = E == 16 * run && !aq::check_ptr(logits, unit) && (T <= 1 || ld * (unit / 4) % unit == 0);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == AQ_BF16) aq::launch_route<true>(a, st);
  else aq::launch_route<false>(a, st);
  return (int)hipGetLastError();
}

extern "C" int aq_combine_rows(const void* y, int dtype, int64_t R, int64_t N, const int32_t* rows, const float* weights, int64_t T, int64_t k,
                               const void* residual, void* out, void* stream) {
  if (dtype != AQ_F32 && dtype != AQ_BF16) return AQ_E_DTYPE;
  if (R < 0 || N <= 0 || T < 0 || k <= 0) return AQ_E_SHAPE;
  if (R > 0x7fffffff || N > (1 << 24) || T > (int64_t)1 << 24 || k > 64) return AQ_E_RANGE;
  if (T == 0) return AQ_OK;
  if ((R > 0 && !y) || !rows || !weights || !out) return AQ_E_NULL;
  const int size = dtype == AQ_BF16 ? 2 : 4;
  if (aq::check_ptr(y, size) || aq::check_ptr(residual, size) || aq::check_ptr(out, size) || aq::check_ptr(rows, 4) || aq::check_ptr(weights, 4))
    return AQ_E_ALIGN;
  const bool vec = (N * size) % 16 == 0 && !aq::check_ptr16(y) && !aq::check_ptr16(out) && !aq::check_ptr16(residual);
  aq::CombineArgs a{};
  a.y = y;
  a.res = residual;
  a.out = out;
  a.rows = rows;
  a.weights = weights;
  a.R = R;
  a.k = (int)k;
  a.per = (int)(vec ? N * size / 16 : N);
  a.n_chunks = (a.per + 63) / 64;
  a.chunks = aq::UDiv::of((uint32_t)a.n_chunks);
  a.waves = T * a.n_chunks;
  if (a.waves > 0x7fffffff) return AQ_E_RANGE;
  const int64_t wgs = (a.waves + 3) / 4;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 g((unsigned)wgs), b(256);
  if (dtype == AQ_BF16) {
    if (vec) aq::queue_kernel((aq::combine_kernel<true, true>), g, b, 0, st, a);
    else aq::queue_kernel((aq::combine_kernel<true, false>), g, b, 0, st, a);
  } else {
    if (vec) aq::queue_kernel((aq::combine_kernel<false, true>), g, b, 0, st, a);
    else aq::queue_kernel((aq::combine_kernel<false, false>), g, b, 0, st, a);
  }
  return (int)hipGetLastError();
}
