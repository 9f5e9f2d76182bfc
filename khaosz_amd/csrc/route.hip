// The two ends of a layer of routed experts: from the router's logits to each token's experts and the order in which the experts work
// through the tokens, and from the experts' outputs back to the tokens.
//
// route: a token's k largest logits x_1 >= .. >= x_k (equal ones: the lowest expert first), their weights exp(x_j - x_1) / sum, and a
// counting sort of the T k choices by expert, in the tokens' order inside an expert.  16 lanes hold a token's logits as keys that order like
// (logit, lowest index), so that a choice is a maximum over a few registers and four DPP steps.  A token names an expert at most once:
// a workgroup's 64 tokens leave a bit each in a 64-bit word per expert (an OR: any order gives the same word), and the number of
// bits below a token's own is its place among them.  No atomic whose order shows.
// What bounds it: launches and chains of latencies; the bytes (10.5 MB for 16384 tokens of 256 experts) would take 2 us.
#include "aq_grouped.h"

namespace aq {

constexpr int RT_THREADS = 1024;
constexpr int RT_TOKENS = RT_THREADS / 16;  // tokens of a pass: 16 lanes each, 64 of them
constexpr int RT_ONE_PASSES = 4;            // passes of the kernel that does it all in one workgroup
constexpr int RT_MAX_E = 512, RT_MAX_K = 16;
constexpr int RT_MOST_CHUNKS = 512;  // larger batches: more passes to a chunk
constexpr int RT_GROUP = 4;          // chunks of a workgroup that hands out rows

struct RouteArgs {
  const void* logits;
  int64_t ld;  // logits between tokens
  float* weights;
  int32_t *experts, *rows, *tokens, *offsets;
  uint16_t* counts;  // [chunks][E]
  int T, E, k, renormalize, passes, chunks;
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
  static __device__ __forceinline__ uint32_t load(const void* p, int64_t i) { return (uint32_t)static_cast<const uint16_t*>(p)[i] << 16; }
  static __device__ __forceinline__ type make(uint32_t ordered, int e) { return (ordered & 0xffff0000u) | (0xffffu - (uint32_t)e); }
  static __device__ __forceinline__ int expert(type k) { return (int)(0xffffu - (k & 0xffffu)); }
  static __device__ __forceinline__ float value(type k) { return __uint_as_float((k >> 31 ? k ^ 0x80000000u : ~k) & 0xffff0000u); }
};
template <>
struct Key<false> {
  using type = u64;
  static __device__ __forceinline__ uint32_t load(const void* p, int64_t i) { return static_cast<const uint32_t*>(p)[i]; }
  static __device__ __forceinline__ type make(uint32_t ordered, int e) { return (u64)ordered << 32 | (0xffffu - (uint32_t)e); }
  static __device__ __forceinline__ int expert(type k) { return (int)(0xffffu - ((uint32_t)k & 0xffffu)); }
  static __device__ __forceinline__ float value(type k) {
    const uint32_t h = (uint32_t)(k >> 32);
    return __uint_as_float(h >> 31 ? h ^ 0x80000000u : ~h);
  }
};

// exp(x - most), most the largest of them: 1 for it, infinite or not
__device__ __forceinline__ float exp_below(float x, float most) { return x == most ? 1.0f : expf(x - most); }

// The choices of token t by the 16 lanes that hold it: lane j has choice j < k (expert -1: there is none) and its weight.
template <bool BF16, int V>
__device__ __forceinline__ int choose(const RouteArgs& a, int t, int l, float* weight) {
  using K = Key<BF16>;
  typename K::type key[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * 16 + l;
    uint32_t bits = 0xff800000u;  // -inf
    if (t < a.T && e < a.E) bits = K::load(a.logits, (int64_t)t * a.ld + e);
    const float x = __uint_as_float(bits) + 0.0f;  // (-0 counts as 0)
    const uint32_t u = __float_as_uint(x);
    key[v] = x > -__builtin_inff() ? K::make(u >> 31 ? ~u : u | 0x80000000u, e) : 0;
  }
  auto best = [&]() {
    auto b = key[0];
#pragma unroll
    for (int v = 1; v < V; ++v) b = larger(b, key[v]);
    return row_max(b);
  };
  typename K::type mine = 0, b = best();
  const float most = K::value(b);
  float total = 0.0f;
  if (!a.renormalize && b) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (key[v]) total += exp_below(K::value(key[v]), most);
    total = row_sum(total);
  }
  for (int j = 0; j < a.k; ++j) {
    if (j) b = best();
    if (l == j) mine = b;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (key[v] == b) key[v] = 0;
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
template <bool BF16, int V, bool ONE>
__global__ __launch_bounds__(RT_THREADS) void route_choose_kernel(RouteArgs a) {
  __shared__ u64 asked[RT_MAX_E];
  __shared__ uint32_t count[RT_MAX_E], first[RT_MAX_E + 1];
  const int tid = threadIdx.x, lane = tid & 63, l = lane & 15, place = tid >> 4;
  for (int e = tid; e < a.E; e += RT_THREADS) count[e] = 0;
  int chose[ONE ? RT_ONE_PASSES : 1], rank[ONE ? RT_ONE_PASSES : 1];
  auto pass = [&](int i, int t, int& ce, int& cr) {
    for (int e = tid; e < a.E; e += RT_THREADS) asked[e] = 0;
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
    for (int e = tid; e < a.E; e += RT_THREADS) count[e] += (uint32_t)__popcll(asked[e]);
  };
  if constexpr (ONE) {
#pragma unroll
    for (int i = 0; i < RT_ONE_PASSES; ++i) {
      chose[i] = rank[i] = -1;
      if (i * RT_TOKENS < a.T) pass(i, i * RT_TOKENS + place, chose[i], rank[i]);
    }
    __syncthreads();
    if (tid < 64) experts_scan(count, first, a.E, lane);
    __syncthreads();
    for (int e = tid; e <= a.E; e += RT_THREADS) a.offsets[e] = (int32_t)first[e];
#pragma unroll
    for (int i = 0; i < RT_ONE_PASSES; ++i) {
      const int t = i * RT_TOKENS + place;
      if (t < a.T && l < a.k) {
        const int r = chose[i] >= 0 ? (int)first[chose[i]] + rank[i] : -1;
        a.rows[t * a.k + l] = r;
        if (r >= 0) a.tokens[r] = t;
      }
    }
    for (int r = (int)first[a.E] + tid; r < a.T * a.k; r += RT_THREADS) a.tokens[r] = -1;
  } else {
    for (int i = 0; i < a.passes; ++i) pass(i, ((int)blockIdx.x * a.passes + i) * RT_TOKENS + place, chose[0], rank[0]);
    __syncthreads();
    for (int e = tid; e < a.E; e += RT_THREADS) a.counts[(int64_t)blockIdx.x * a.E + e] = (uint16_t)count[e];
  }
}

// Rows for the choices of RT_GROUP chunks: the experts' first rows, the choices of the chunks before, the place among the chunk's.  Every
// workgroup adds up all chunks' counts by itself.
__global__ __launch_bounds__(RT_THREADS) void route_rows_kernel(RouteArgs a) {
  __shared__ uint32_t total[RT_MAX_E], before[RT_MAX_E], first[RT_MAX_E + 1], base[RT_GROUP][RT_MAX_E];
  const int tid = threadIdx.x, E = a.E;
  const int c0 = (int)blockIdx.x * RT_GROUP;
  for (int e = tid; e < E; e += RT_THREADS) total[e] = before[e] = 0;
  __syncthreads();
  int width = 64;  // threads to a run of experts
  while (width < E) width *= 2;
  const int e = tid & (width - 1), turns = RT_THREADS / width;
  if (e < E) {
    uint32_t all = 0, early = 0;
#pragma unroll 8
    for (int c = tid / width; c < a.chunks; c += turns) {
      const uint32_t n = a.counts[(int64_t)c * E + e];
      all += n;
      early += c < c0 ? n : 0;
      if (c >= c0 && c < c0 + RT_GROUP) base[c - c0][e] = n;
    }
    atomicAdd(&total[e], all);  // whole numbers: any order
    atomicAdd(&before[e], early);
  }
  __syncthreads();
  if (tid < 64) experts_scan(total, first, E, tid);
  __syncthreads();
  for (int i = tid; i < E; i += RT_THREADS) {
    uint32_t at = first[i] + before[i];
#pragma unroll
    for (int c = 0; c < RT_GROUP; ++c) {
      const uint32_t n = base[c][i];
      base[c][i] = at;
      at += n;
    }
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int i = tid; i <= E; i += RT_THREADS) a.offsets[i] = (int32_t)first[i];
  const int chunk = a.passes * RT_TOKENS, k = a.k;
  const int64_t all = (int64_t)a.T * k;
  for (int c = 0; c < RT_GROUP; ++c) {
    const int64_t from = (int64_t)(c0 + c) * chunk * k, to = from + (int64_t)chunk * k < all ? from + (int64_t)chunk * k : all;
    for (int64_t s = from + tid; s < to; s += RT_THREADS) {
      const int ex = a.experts[s];
      if (ex < 0) continue;
      const int r = (int)base[c][ex] + a.rows[s];
      a.rows[s] = r;
      a.tokens[r] = (int)((uint32_t)s / (uint32_t)k);
    }
  }
  for (int64_t r = (int64_t)first[E] + (int64_t)blockIdx.x * RT_THREADS + tid; r < all; r += (int64_t)gridDim.x * RT_THREADS) a.tokens[r] = -1;
}

static int route_passes(int64_t T) {
  const int64_t n = (T + RT_TOKENS - 1) / RT_TOKENS;
  return (int)((n + RT_MOST_CHUNKS - 1) / RT_MOST_CHUNKS);
}
static int64_t route_chunks(int64_t T) {
  const int64_t chunk = (int64_t)route_passes(T) * RT_TOKENS;
  return (T + chunk - 1) / chunk;
}

template <bool BF16, int V>
static void launch_route(const RouteArgs& a, hipStream_t st) {
  if (a.T <= RT_ONE_PASSES * RT_TOKENS) {
    queue_kernel((route_choose_kernel<BF16, V, true>), dim3(1), dim3(RT_THREADS), 0, st, a);
  } else {
    queue_kernel((route_choose_kernel<BF16, V, false>), dim3((unsigned)a.chunks), dim3(RT_THREADS), 0, st, a);
    queue_kernel(route_rows_kernel, dim3((unsigned)((a.chunks + RT_GROUP - 1) / RT_GROUP)), dim3(RT_THREADS), 0, st, a);
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
// out[t] = sum_j weights[t, j] y[rows[t, j]] (+ residual[t]), in fp32 in the order of j, the residual last, rounded once.  A thread has 16 bytes of a
// token's row (VEC; single values where rows are not whole vectors) and asks for up to 8 choices' before it adds.
// What bounds it: HBM.
struct CombineArgs {
  const void *y, *res;
  void* out;
  const int32_t* rows;
  const float* weights;
  int64_t units;  // of 16 bytes (values), in all
  int64_t R;
  int k, per;     // units of a token
};

template <bool BF16, bool VEC>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a) {
  constexpr int N = VEC ? (BF16 ? 8 : 4) : 1, AHEAD = 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.units) return;
  const int64_t t = a.per == 256 ? (int64_t)blockIdx.x : i / a.per;
  const int u = (int)(i - t * a.per);
  auto load = [&](const void* p, int64_t row, float* v) {
    if constexpr (VEC) {
      const uint4 q = static_cast<const uint4*>(p)[row * a.per + u];
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if constexpr (BF16) {
          v[2 * c] = __uint_as_float(w[c] << 16);
          v[2 * c + 1] = __uint_as_float(w[c] & 0xffff0000u);
        } else {
          v[c] = __uint_as_float(w[c]);
        }
      }
    } else {
      v[0] = BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(p)[row * a.per + u]) : static_cast<const float*>(p)[row * a.per + u];
    }
  };
  float sum[N];
#pragma unroll
  for (int c = 0; c < N; ++c) sum[c] = 0.0f;
  for (int j0 = 0; j0 < a.k; j0 += AHEAD) {
    int row[AHEAD];
    float w[AHEAD], v[AHEAD][N];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      row[j] = -1;
      if (j0 + j < a.k) {
        row[j] = a.rows[t * a.k + j0 + j];
        w[j] = a.weights[t * a.k + j0 + j];
        if (row[j] >= a.R) row[j] = -1;
      }
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (row[j] >= 0) load(a.y, row[j], v[j]);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (row[j] >= 0) {
#pragma unroll
        for (int c = 0; c < N; ++c) sum[c] += w[j] * v[j][c];
      }
  }
  if (a.res) {
    float v[N];
    load(a.res, t, v);
#pragma unroll
    for (int c = 0; c < N; ++c) sum[c] += v[c];
  }
  if constexpr (VEC && BF16) {
    static_cast<uint4*>(a.out)[i] = make_uint4(pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3]), pack_bf16x2(sum[4], sum[5]), pack_bf16x2(sum[6], sum[7]));
  } else if constexpr (VEC) {
    static_cast<float4*>(a.out)[i] = make_float4(sum[0], sum[1], sum[2], sum[3]);
  } else if constexpr (BF16) {
    static_cast<uint16_t*>(a.out)[i] = (uint16_t)f32_to_bf16_bits(sum[0]);
  } else {
    static_cast<float*>(a.out)[i] = sum[0];
  }
}

}  // namespace aq

extern "C" int64_t aq_route_topk_workspace_bytes(int64_t T, int64_t E) {
  if (T <= aq::RT_ONE_PASSES * aq::RT_TOKENS || T > (int64_t)1 << 24 || E <= 0) return 0;
  return aq::route_chunks(T) * E * (int64_t)sizeof(uint16_t);
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
  if (need > 0 && aq::check_ptr(workspace, 4)) return AQ_E_ALIGN;
  aq::RouteArgs a{};
  a.logits = logits;
  a.ld = ld;
  a.weights = weights;
  a.experts = experts;
  a.rows = rows;
  a.tokens = tokens;
  a.offsets = offsets;
  a.counts = static_cast<uint16_t*>(workspace);
  a.T = (int)T;
  a.E = (int)E;
  a.k = (int)k;
  a.renormalize = renormalize != 0;
  a.passes = aq::route_passes(T);
  a.chunks = T > 0 ? (int)aq::route_chunks(T) : 0;
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
  a.units = T * a.per;
  const int64_t wgs = (a.units + 255) / 256;
  if (wgs > 0x7fffffff) return AQ_E_RANGE;
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
