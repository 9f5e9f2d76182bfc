// Decode attention of a batch whose sequences begin with the same pages (samples of one prompt, beams, requests behind one
// system prompt; the reference's prefix cache maps such pages into every sequence's table, astrai/inference/core/cache.py:68-185, and its
// attention then gathers and reads them once per sequence, cache.py:254-274).  Here the shared positions are read and multiplied
// once for the whole batch:
//
//   prefix   the G query heads of a KV head of all B sequences are B G rows of one product against the shared keys: scores,
//            softmax statistics and values per tile of rows and slice of positions, left as partial results;
//   tail     the same for the G rows of one sequence against its own positions;
//   merge    the partial results of a row are weighed by exp2(maximum - overall maximum) and added up.
//
// softmax over two ranges is the softmax over both: with m, l, n the maximum, denominator and numerator of each range,
// out = (n1 2^(m1 - m) + n2 2^(m2 - m)) / (l1 2^(m1 - m) + l2 2^(m2 - m)), m = max(m1, m2).  All of them are fp32; probabilities
// are rounded to bf16 (off by 2^-8 of themselves at most) where the matrix core takes them, in the prefix and in the tails alike, the denominator
// sums them unrounded.
//
// Prefix and tail are workgroups of one launch, the prefix's first: those multiply while the tails read.  Both compute S^T = K Q^T and
// O^T = V^T P^T as the prefill kernel does (attn_prefill.hip has the layout): a lane has the scores of one row, nothing changes lanes,
// K and V rows go straight into LDS ahead of the products.
//
// us a call; what its bytes take at the 5.2 TB/s of a large copy; the decode kernel, which reads the prefix for every sequence; what bounds the call:
//   8 x 2591 positions of which 2048 shared, 16/4 heads of 128     9.3   2.5   13.8  the latency of two launches
//   33 x 1401 of 1008, own lengths, 24/4 of 64, pages of 16        10.8  1.5   12.6  the same
//   64 x 8448 of 8192, 32/8 of 128                                 34.8  19.6   208  a wavefront's chain in the prefix beside the tails' loads
//   16 x 65600 of 65536, 16/4 of 128                               36.0  26.3   350  HBM: 6.5 TB/s inside the loop, 20.6 of the launch's 32.3; the merge 4.8
//   256 x 4500 of 4096, own lengths, 16/4 of 128                   39.4  22.5   222  tails of 200 positions, mostly beginning and end; the merge 5.3
#include "aq_attn.h"
#include "aq_common.h"
#include "aq_rows.h"

#include <type_traits>

namespace aq {

struct SharedArgs {
  const uint16_t* q;     // [B, Hq, D]
  const uint16_t* kc;    // [n_pages, page, Hkv, D]
  const uint16_t* vc;
  const int64_t* table;  // [B, P]; row 0 has the shared pages
  const int64_t* lens;   // [B] or null
  float* ws;             // partial results: [slices][Hkv][tiles of 32 rows] of the prefix, then [B][Hkv][tails]
  int64_t page, n_pages, P;
  float scale_log2e;
  int T, s0, rows, Hq, Hkv, G;      // positions, of which the prefix takes s0 (a multiple of 64); B G
  int slice, slices, tiles, tiles32;  // positions of a prefix slice; slices; tiles of rows of a workgroup, of 32
  int tail, tails;                  // positions of a tail's slice, slices of a sequence
  int prefix_wgs;                   // the workgroups behind them are tails
  int page_shift;                   // log2 of the page size, or -1
  int page_rows;                    // pages hold whole loads of 1 KiB of one head's rows: 512 / D of them
  int table_lds;                    // entries of the page table that a workgroup may need, kept in LDS (0: read from memory)
  UDiv by_g, by_page, by_tiles, by_hkv, by_tails;
};

constexpr float SHARED_MASKED = -1.0e30f;  // score of every position of a sequence without any length: it weighs them alike, as in the decode kernel

// A partial result of n rows: numerators as 16-byte groups of 4 dimensions, the n rows of a group side by side (what the lanes of a
// product hold, so that it is stored and read by whole lines), then the n maxima and the n denominators.
__host__ __device__ constexpr int part_floats(int D, int n) { return (D + 4) * n; }

// s_waitcnt for n vector-memory operations still in flight (gfx9 encoding), and a barrier that leaves them in flight.
#define SH_WAIT_VMCNT(n) __builtin_amdgcn_s_waitcnt(0x0f70 | ((n) & 15) | (((n) >> 4) << 14))
#define SH_WAIT_LGKM() __builtin_amdgcn_s_waitcnt(0xc07f)
__device__ __forceinline__ void sh_barrier() {
  asm volatile("" ::: "memory");
  SH_WAIT_LGKM();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// What a wavefront keeps of its 32 rows: lane = (row col, half g of the positions of a 32 x 32 product).
template <int D>
struct SharedRows {
  uint4 qf[D / 16];    // Q^T operand: dimensions 16 step + 8 g .. + 8
  pa_f32x16 o[D / 32];  // O^T: register r of tile dt is dimension 32 dt + 8 (r / 4) + 4 g + r % 4
  float m, l;          // bound of the row's scores; this lane's half of its denominator
  int vis;             // positions the row may attend to, 0 .. T

  __device__ __forceinline__ void start(const uint16_t* q, int g, int visible) {
#pragma unroll
    for (int st = 0; st < D / 16; ++st) qf[st] = *reinterpret_cast<const uint4*>(q + g * 8 + st * 16);
    vis = visible;
    clear();
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] = 0.0f;
    m = -INFINITY;
    l = 0.0f;
  }

  // Whether some numerator is infinite or NaN; wavefront-uniform.
  __device__ __forceinline__ bool odd() const {
    float x = 0.0f;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) x = __builtin_fmaf(o[dt][r], 0.0f, x);
    return __builtin_amdgcn_ballot_w64(x != 0.0f) != 0;  // (0 times either is NaN)
  }

  // 32 NT positions from kb0 on, K rows at ks and V rows at vs.  masked (wavefront-uniform): some row may not attend to some of them, or
  // (not ALL) there are only T.
  // keys_read() is called when the last K row has been read, values_needed() before the first V row is.  APART: infinite
  // values are among V, which 0 does not mask: a row's product leaves out what the row must not see.
  template <int NT, bool ALL, bool APART, class FK, class FV>
  __device__ __forceinline__ void attend(const uint8_t* ks, const uint8_t* vs, int kb0, bool masked, int T, float scale_log2e,
                                         FK&& keys_read, FV&& values_needed) {
    constexpr int DSTEPS = D / 16, DT = D / 32, ROWB = 2 * D;
    const int lane = threadIdx.x & 63, col = lane & 31, g = lane >> 5;
    // fragment addresses inside a block: K row `col`, piece 2 step + g; V rows 4 g + i / 4 (and 8 further), i = lane % 16,
    // dimensions 16 (lane / 16 % 2) + 4 (i % 4) of a 32-dimension tile
    const int kfr = col * ROWB + ((g ^ row_key<D>(col)) << 4);  // ^ (2 step) << 4
    const int vrow = 4 * g + (lane & 15) / 4, vpiece = ((lane >> 4) & 1) * 2 + (lane & 3) / 2;
    const int vfr0 = vrow * ROWB + ((vpiece ^ row_key<D>(vrow)) << 4) + (lane & 1) * 8;  // ^ dt << 6
    const int vfr1 = (vrow + 8) * ROWB + ((vpiece ^ row_key<D>(vrow + 8)) << 4) + (lane & 1) * 8;
    // ---- scores; the fragments of K are read two groups of steps ahead of the products that take them
    pa_f32x16 s[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[t][r] = 0.0f;
    {
      constexpr int GRP = 4 / NT, NG = DSTEPS / GRP;
      uint4 fa[2][GRP][NT];
      auto ldk = [&](int buf, int st0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < GRP; ++i)
#pragma unroll
          for (int t = 0; t < NT; ++t)
            fa[buf][i][t] = *reinterpret_cast<const uint4*>(ks + t * 32 * ROWB + (kfr ^ ((2 * (st0 + i)) << 4)));
      };
      ldk(0, 0);
      if (NG > 1) ldk(1, GRP);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int gi = 0; gi < NG; ++gi) {
#pragma unroll
        for (int i = 0; i < GRP; ++i) {
          const pa_bf16x8 qv = __builtin_bit_cast(pa_bf16x8, qf[gi * GRP + i]);
#pragma unroll
          for (int t = 0; t < NT; ++t)
            s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(pa_bf16x8, fa[gi & 1][i][t]), qv, s[t], 0, 0, 0);
        }
        if (gi + 2 < NG) ldk(gi & 1, (gi + 2) * GRP);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    keys_read();
    // ---- softmax of this lane's row; register r of tile kt is position kb0 + 32 kt + 8 (r / 4) + 4 g + r % 4
    float sc = scale_log2e;
    if (masked) {  // the scores are scaled here: those of a sequence without any length have the same value in every slice
      const float hidden = vis ? -INFINITY : SHARED_MASKED;
      const int end = vis - kb0 - 4 * g, all = T - kb0 - 4 * g;
#pragma unroll
      for (int kt = 0; kt < NT; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = kt * 32 + 8 * (r / 4) + r % 4;
          s[kt][r] = key < end ? s[kt][r] * sc : ALL || key < all ? hidden : -INFINITY;
        }
      sc = 1.0f;
    }
    softmax_values<NT, APART>(s, vs, vfr0, vfr1, kb0, masked, T, sc, values_needed);
  }

  template <int NT, bool APART, class FV>
  __device__ __forceinline__ void softmax_values(pa_f32x16 (&s)[NT], const uint8_t* vs, int vfr0, int vfr1, int kb0, bool masked, int T, float sc,
                                                 FV&& values_needed) {
    constexpr int DT = D / 32, ROWB = 2 * D;
    float bm = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < NT; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r) bm = fmaxf(bm, s[kt][r]);
    const LanePair b2 = lanes32_pair(bm);
    bm = fmaxf(b2.x, b2.y) * sc;
    // m only has to bound the exponents: it is raised, and the sums rescaled, when a row of the wavefront would see one above 2^8
    if (__builtin_amdgcn_ballot_w64(bm > m + 8.0f) != 0) {  // wavefront-uniform
      const float mn = fmaxf(m, bm), alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
    }
    const float mb = m == -INFINITY ? 0.0f : m;  // (so far every score is -infinity, and weighs nothing, or NaN, and stays that)
    uint4 pf[NT][2];  // P^T operands: tile kt, positions 16 s2 .. + 16
#pragma unroll
    for (int kt = 0; kt < NT; ++kt) {
      float pv[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        pv[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][r], sc, -mb));
        l += pv[r];
      }
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2)
        pf[kt][s2] = make_uint4(pack_bf16x2(pv[8 * s2 + 0], pv[8 * s2 + 1]), pack_bf16x2(pv[8 * s2 + 2], pv[8 * s2 + 3]),
                                pack_bf16x2(pv[8 * s2 + 4], pv[8 * s2 + 5]), pack_bf16x2(pv[8 * s2 + 6], pv[8 * s2 + 7]));
    }
    values_needed();
    constexpr int KK = 2 * NT;
    auto fragment = [&](int dt, int kk) __attribute__((always_inline)) {  // V^T operand: tile dt, positions 16 kk .. + 16
      const uint8_t* at = vs + kk * 16 * ROWB;
      const pa_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_lds_s16x4*)(at + (vfr0 ^ (dt << 6))));
      const pa_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_lds_s16x4*)(at + (vfr1 ^ (dt << 6))));
      return __builtin_bit_cast(pa_bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    if constexpr (APART) {  // a product for each length, of the values that rows of this length see
      const int g = (threadIdx.x & 63) >> 5, mine = vis ? vis : T;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        uint64_t left = ~0ull;
        do {
          const int n = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
          left &= ~__builtin_amdgcn_ballot_w64(mine == n);
          int end = n - kb0 - 4 * g;
          asm volatile("" : "+v"(end)::"memory");  // (compared, and the values read, here: nothing of it kept in registers)
          pa_f32x16 x = o[dt];
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) {
            pa_bf16x8 v = fragment(dt, kk);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (16 * kk + 8 * (j / 4) + j % 4 >= end) v[j] = static_cast<__bf16>(0.0f);
            x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, __builtin_bit_cast(pa_bf16x8, pf[kk >> 1][kk & 1]), x, 0, 0, 0);
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) o[dt][r] = mine == n ? x[r] : o[dt][r];
        } while (left);
      }
      return;
    }
    // ---- O^T += V^T P^T; all fragments of V are read before the products, whose chains alternate
    pa_bf16x8 fv[DT][KK];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) fv[dt][kk] = fragment(dt, kk);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d0 = 0; d0 < DT; d0 += 2)
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int dt = d0; dt < d0 + 2; ++dt)
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fv[dt][kk], __builtin_bit_cast(pa_bf16x8, pf[kk >> 1][kk & 1]), o[dt], 0, 0, 0);
  }

  // Whether some row may not attend to some of the positions kb0 .. kb0 + n - 1; *none: no row to any.
  __device__ __forceinline__ bool masked(int kb0, int n, bool* none) const {
    *none = false;
    if (__builtin_amdgcn_ballot_w64(kb0 + n > vis) == 0) return false;
    *none = __builtin_amdgcn_ballot_w64(vis == 0 || kb0 < vis) == 0;
    return true;
  }

  // A partial result of n rows; a row that saw nothing, or scores of -infinity only, leaves its maximum only.  One whose scores are NaN has a NaN
  // for a maximum, which fmaxf leaves out and the sums take in.
  __device__ __forceinline__ void store(float* part, int n) const {
    const int lane = threadIdx.x & 63, col = lane & 31, g = lane >> 5;
    const LanePair l2 = lanes32_pair(l);
    const float sum = l2.x + l2.y, most = sum != sum ? sum : m;
    if (col >= n) return;
    if (most != -INFINITY) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        *reinterpret_cast<v4f*>(part + ((2 * i + g) * n + col) * 4) = v4f{o[i / 4][4 * (i % 4)], o[i / 4][4 * (i % 4) + 1], o[i / 4][4 * (i % 4) + 2],
                                                                         o[i / 4][4 * (i % 4) + 3]};
    }
    part[(g == 0 ? D : D + 1) * n + col] = g == 0 ? most : sum;
  }

  // The same of the KW wavefronts that share these rows (as the tile-th of `tiles`), whose sums meet in LDS: each adds up and stores its
  // share of the dimensions.  lds: 32 D numbers a wavefront that no load is still to arrive in; ml: 128.  (One wavefront that adds up and
  // stores everything takes 2.0 us of a tail's 8.7, this 1.)
  template <int KW>
  __device__ __forceinline__ void join_and_store(v4f* lds, float* ml, int kw, int tile, int tiles, float* part, int n) const {
    constexpr int GROUPS = D / 8, SHARE = GROUPS / KW;  // groups of 4 sums
    const int lane = threadIdx.x & 63, col = lane & 31, g = lane >> 5, at = kw * tiles + tile;
    const LanePair l2 = lanes32_pair(l);
#pragma unroll
    for (int i = 0; i < GROUPS; ++i)
      lds[(at * GROUPS + i) * 64 + lane] = v4f{o[i / 4][4 * (i % 4)], o[i / 4][4 * (i % 4) + 1], o[i / 4][4 * (i % 4) + 2], o[i / 4][4 * (i % 4) + 3]};
    ml[at * 128 + lane] = m;
    ml[at * 128 + 64 + lane] = l2.x + l2.y;
    sh_barrier();
    float w[KW], most = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      w[k] = ml[(k * tiles + tile) * 128 + lane];
      most = fmaxf(most, w[k]);
    }
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      w[k] = w[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(w[k] - most);
      sum = __builtin_fmaf(ml[(k * tiles + tile) * 128 + 64 + lane], w[k], sum);
    }
    if (sum != sum) most = sum;
    if (col >= n) return;
    if (most != -INFINITY) {
#pragma unroll
      for (int i = 0; i < SHARE; ++i) {
        const int c = kw * SHARE + i;
        v4f x = lds[(tile * GROUPS + c) * 64 + lane];
#pragma unroll
        for (int d = 0; d < 4; ++d) x[d] *= w[0];
#pragma unroll
        for (int k = 1; k < KW; ++k) {
          const v4f y = lds[((k * tiles + tile) * GROUPS + c) * 64 + lane];
#pragma unroll
          for (int d = 0; d < 4; ++d) x[d] = __builtin_fmaf(y[d], w[k], x[d]);
        }
        *reinterpret_cast<v4f*>(part + ((2 * c + g) * n + col) * 4) = x;
      }
    }
    if (kw == 0) part[(g == 0 ? D : D + 1) * n + col] = g == 0 ? most : sum;
  }
};

__device__ __forceinline__ const uint16_t* uniform(const uint16_t* p) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  return reinterpret_cast<const uint16_t*>((uint64_t)__builtin_amdgcn_readfirstlane((int)(a >> 32)) << 32 |
                                           (uint32_t)__builtin_amdgcn_readfirstlane((int)a));
}

// The page table of one sequence.
struct SharedPages {
  const int64_t* table;
  int* lds;  // ids of the pages from lp0 on, or null
  int lp0;

  __device__ __forceinline__ int phys(const SharedArgs& p, int lp) const {
    const int64_t t = lp < p.P ? table[lp] : -1;
    return t >= 0 && t < p.n_pages ? (int)t : -1;
  }
  // (a barrier has to follow before load() is called)
  __device__ __forceinline__ void fetch(const SharedArgs& p, int first, int* place, int threads) {
    lds = nullptr;
    lp0 = 0;
    if (!p.table_lds) return;
    lds = place;
    lp0 = (int)p.by_page((uint32_t)first);
    for (int i = threadIdx.x; i < p.table_lds; i += threads) lds[i] = phys(p, lp0 + i);
  }

  // The page of the block at kb0 (before `end`), where a block lies in one page; requested a block ahead, so that no load waits for it.
  // SCALAR: a vector load would count among the rows on their way.
  template <int KB, bool SCALAR = true>
  __device__ __forceinline__ int64_t page_of(const SharedArgs& p, int kb0, int end) const {
    if (p.page_shift < (KB == 64 ? 6 : 5)) return -1;
    const int lp = __builtin_amdgcn_readfirstlane(kb0 >> p.page_shift);
    typedef const __attribute__((address_space(4))) int64_t* constant;
    if (kb0 >= end || lp >= p.P) return -1;
    if constexpr (SCALAR) return ((constant)(uintptr_t)table)[lp];
    else return table[lp];
  }

  // N loads of 1 KiB: rows r0, r0 + rows of a load, .. of the block of KB positions at kb0, into LDS from `dst` on, those of keys and (BOTH) of
  // values `apart` bytes further.  Rows from `seen` on, which no one looks at, are zeros whatever is stored there; so are unmapped pages.
  template <int D, int KB, int N, bool KEYS, bool VALUES>
  __device__ __forceinline__ void load(const SharedArgs& p, int kvh, int kb0, int64_t id, int seen, int r0, uint32_t dst, uint32_t apart) const {
    constexpr int ROWB = 2 * D, RPI = 1024 / ROWB, LPR = 64 / RPI;
    const int lane = threadIdx.x & 63;
    const int rows = seen - kb0;
    const uint16_t* const zero = reinterpret_cast<const uint16_t*>(pa_zero_row);
    int pc[N];  // this lane's piece of the rows: elements into the row
#pragma unroll
    for (int c = 0; c < N; ++c) pc[c] = ((lane % LPR) ^ row_key<D>(r0 + c * RPI + lane / LPR)) * 8;
    constexpr int SHIFT = KB == 64 ? 6 : 5;
    if (p.page_shift >= SHIFT) {  // the whole block lies in one page
      const int lp = __builtin_amdgcn_readfirstlane(kb0 >> p.page_shift);
      const bool mapped = id >= 0 && id < p.n_pages;
      const int64_t first = mapped ? (((id << p.page_shift) + (kb0 - (lp << p.page_shift))) * p.Hkv + kvh) * D : 0;
      const int step = p.Hkv * D;
      if (mapped && rows >= KB) {  // (wavefront-uniform) the whole block is there: only the base changes from block to block
        const uint16_t *const kc = uniform(p.kc + first), *const vc = uniform(p.vc + first);
#pragma unroll
        for (int c = 0; c < N; ++c) {
          const uint32_t at = 2 * (uint32_t)((r0 + c * RPI + lane / LPR) * step + pc[c]);
          if (KEYS) load_row_lds(kc, at, dst + c * 1024);
          if (VALUES) load_row_lds(vc, at, dst + (KEYS ? apart : 0) + c * 1024);
        }
        return;
      }
#pragma unroll
      for (int c = 0; c < N; ++c) {
        const int r = r0 + c * RPI + lane / LPR;
        const bool there = mapped && r < rows;
        const uint32_t at = (uint32_t)(r * step + pc[c]);
        if (KEYS) load_row_lds(there ? p.kc + first + at : zero + pc[c], dst + c * 1024);
        if (VALUES) load_row_lds(there ? p.vc + first + at : zero + pc[c], dst + (KEYS ? apart : 0) + c * 1024);
      }
      return;
    }
    if (p.page_rows && lds && rows >= KB) {  // the rows of a load lie in one page: a lookup and a base per load
      int id[N];
      bool mapped = true;
#pragma unroll
      for (int c = 0; c < N; ++c) id[c] = lds[p.by_page((uint32_t)(kb0 + r0 + c * RPI)) - lp0];
#pragma unroll
      for (int c = 0; c < N; ++c) {
        id[c] = __builtin_amdgcn_readfirstlane(id[c]);
        mapped = mapped && id[c] >= 0;
      }
      if (mapped) {
        const int step = p.Hkv * D, row = (lane / LPR) * step;
#pragma unroll
        for (int c = 0; c < N; ++c) {
          const int key = __builtin_amdgcn_readfirstlane(kb0 + r0 + c * RPI), in_page = key - (int)p.by_page((uint32_t)key) * (int)p.page;
          const int64_t first = (((int64_t)id[c] * p.page + in_page) * p.Hkv + kvh) * D;
          const uint32_t at = 2 * (uint32_t)(row + pc[c]);
          if (KEYS) load_row_lds(uniform(p.kc + first), at, dst + c * 1024);
          if (VALUES) load_row_lds(uniform(p.vc + first), at, dst + (KEYS ? apart : 0) + c * 1024);
        }
        return;
      }
    }
    // every address first, then the loads: a load is a fence to the compiler, and a lookup behind each one would wait for LDS once per row
    int64_t at[N];
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int r = r0 + c * RPI + lane / LPR, key = kb0 + r;
      const int lp = p.by_page((uint32_t)key), in_page = key - lp * (int)p.page;
      const int id = r >= rows ? -1 : lds ? lds[lp - lp0] : phys(p, lp);
      at[c] = id < 0 ? -1 : (((int64_t)id * p.page + in_page) * p.Hkv + kvh) * D;
    }
#pragma unroll
    for (int c = 0; c < N; ++c) {
      if (KEYS) load_row_lds((at[c] < 0 ? zero : p.kc + at[c]) + pc[c], dst + c * 1024);
      if (VALUES) load_row_lds((at[c] < 0 ? zero : p.vc + at[c]) + pc[c], dst + (KEYS ? apart : 0) + c * 1024);
    }
  }
};

__device__ __forceinline__ int visible(const SharedArgs& p, int b) {
  if (!p.lens) return p.T;
  const int64_t n = p.lens[b];
  return n <= 0 ? 0 : n < p.T ? (int)n : p.T;
}

// A tile of 32 QW rows of all sequences against a slice of the shared positions.  QW x KW wavefronts: QW tiles of 32 rows side by side on
// the same block of KB positions, KW blocks at a time, the next KW ahead of the products.  (More buffers gain nothing: 64 x 8192 positions
// of 32/8 heads of 128 20.0 us with two, 22.2 with four that leave room for one workgroup per compute unit.)
// Few rows: bound by HBM (16 x 65536 positions, 16/4 heads of 128: 20.6 us for 134 MB in the loop).  Many: 64 x 8192 positions take 12.0 us in the
// loop, 6.9 without the products, 10 without the loads; the matrix core is busy for 3.9, and the store of the partial results adds 1.4.
template <int D, int QW, int KW, int KB, bool LENS>
__device__ __forceinline__ void shared_prefix(const SharedArgs& p, uint8_t* lds, float* ml, int* table_lds) {
  constexpr int ROWB = 2 * D, RPI = 1024 / ROWB;    // bytes of a K or V row; rows of a 1 KiB load
  constexpr int TILE = KB * ROWB;                   // bytes of a block's K (or V)
  constexpr int LOADS = TILE / 1024 / QW;           // 1 KiB loads of K (and of V) per wavefront and block
  constexpr int BUF = KW * 2 * TILE;
  static_assert(LOADS >= 1 && TILE % (1024 * QW) == 0, "whole loads per wavefront");
  static_assert(KW == 1 || KW * QW * 128 * D <= 2 * BUF, "the wavefronts' sums fit the buffers");
  __shared__ int seen_s[QW];
  const int lane = threadIdx.x & 63, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), qw = wave % QW, kw = wave / QW;
  // Workgroups i and i + 8 run on one XCD: the tiles of a (KV head, slice) follow one another there, so that its L2 has the keys and
  // values the first one read.
  const int turn = (int)blockIdx.x >> 3, ty = p.by_tiles(turn), tile = turn - ty * p.tiles, combo = ty * 8 + ((int)blockIdx.x & 7);
  if (combo >= p.slices * p.Hkv) return;
  const int slice = p.by_hkv(combo), kvh = combo - slice * p.Hkv;
  const int k0 = slice * p.slice, k1 = k0 + p.slice < p.s0 ? k0 + p.slice : p.s0;

  const int t32 = tile * QW + qw, r0 = t32 * 32, row = r0 + col < p.rows ? r0 + col : p.rows - 1;  // rows past the end: the last one again
  const int b = p.by_g(row), head = kvh * p.G + (row - b * p.G);
  SharedPages pages{p.table, nullptr, 0};
  pages.fetch(p, k0, table_lds, QW * KW * 64);
  const int vis = visible(p, b);
  int seen = k1;  // positions that any row of the workgroup looks at
  if constexpr (LENS) {
    int most = vis ? vis : p.T;  // a row without any length weighs every position alike
#pragma unroll
    for (int off = 32; off; off >>= 1) {
      const int o = __shfl_xor(most, off, 64);
      most = o > most ? o : most;
    }
    if (kw == 0 && lane == 0) seen_s[qw] = most;
    __syncthreads();
    most = seen_s[0];
#pragma unroll
    for (int i = 1; i < QW; ++i) most = seen_s[i] > most ? seen_s[i] : most;
    seen = most < k1 ? most : k1;
  } else if (p.table_lds) {
    __syncthreads();
  }
  const int nit = __builtin_amdgcn_readfirstlane(seen > k0 ? (seen - k0 + KW * KB - 1) / (KW * KB) : 0);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(pa_lds_void*)lds;
  int64_t page = pages.template page_of<KB>(p, k0 + kw * KB, seen);
  auto issue = [&](int it, int buf) __attribute__((always_inline)) {
    const uint32_t dst = __builtin_amdgcn_readfirstlane(lds0 + buf * BUF + kw * 2 * TILE + qw * LOADS * 1024);
    const int kb0 = k0 + (it * KW + kw) * KB;
    pages.template load<D, KB, LOADS, true, true>(p, kvh, kb0, page, seen, qw * LOADS * RPI, dst, TILE);
    page = pages.template page_of<KB>(p, kb0 + KW * KB, seen);
  };
  if (nit) issue(0, 0);
  SharedRows<D> rows;
  rows.start(p.q + ((int64_t)b * p.Hq + head) * D, lane >> 5, vis);
  const bool idle = r0 >= p.rows;  // wavefront-uniform: no row here, only loads

  bool hidden = false;  // some row must not see some of the positions
  auto blocks = [&](auto apart) __attribute__((always_inline)) {
    constexpr bool APART = decltype(apart)::value;
    for (int it = 0; it < nit; ++it) {
      SH_WAIT_VMCNT(0);  // this wavefront's part of the blocks has landed
      sh_barrier();      // ... everyone's, and everyone is done with the ones before
      if (it + 1 < nit) issue(it + 1, (it + 1) & 1);
      const int kb0 = k0 + (it * KW + kw) * KB;
      const uint8_t* ks = lds + (it & 1) * BUF + kw * 2 * TILE;
      if (idle || kb0 >= k1) continue;  // wavefront-uniform, as all below
      bool masked = false, none = false;
      if constexpr (LENS) {
        masked = rows.masked(kb0, KB, &none);
        hidden |= masked;
      }
      if (none) continue;
      if constexpr (APART) {
#pragma unroll 1
        for (int at = 0; at < KB; at += 32)
          rows.template attend<1, true, true>(ks + at * ROWB, ks + TILE + at * ROWB, kb0 + at, masked, p.T, p.scale_log2e, [] {}, [] {});
      } else {
        rows.template attend<KB / 32, true, false>(ks, ks + TILE, kb0, masked, p.T, p.scale_log2e, [] {}, [] {});
      }
    }
  };
  blocks(std::false_type{});
  if constexpr (LENS) {
    // 0 masks no infinity and no NaN: where some came out, which other sequences' positions may have brought in, the slice is done again
    // with every row's own values.  (Looking for them in each block first: 64 x 8448 positions, lengths from 4096 on, 37.2 us instead of 28.2.)
    __shared__ int odd_s[QW * KW];
    const bool odd = hidden && rows.odd();
    if (lane == 0) odd_s[wave] = odd;
    sh_barrier();
    int any = 0;
#pragma unroll
    for (int i = 0; i < QW * KW; ++i) any |= odd_s[i];
    if (__builtin_amdgcn_readfirstlane(any)) {  // workgroup-uniform
      page = pages.template page_of<KB>(p, k0 + kw * KB, seen);
      issue(0, 0);
      rows.clear();
      blocks(std::true_type{});
    }
  }
  const int n = p.rows - r0 < 32 ? p.rows - r0 : 32;  // idle: none
  float* const part = p.ws + (((int64_t)slice * p.Hkv + kvh) * p.tiles32 + t32) * part_floats(D, 32);
  if constexpr (KW > 1) {
    sh_barrier();  // everyone is done with the blocks
    rows.template join_and_store<KW>(reinterpret_cast<v4f*>(lds), ml, kw, qw, QW, part, n);
  } else if (!idle) {
    rows.store(part, n);
  }
}

// The G rows of one sequence against a slice of its own positions.  Bound by HBM and by what a workgroup waits for before its first and after
// its last block (64 sequences of 256 positions, 32/8 heads of 128: 67 MB in 15.5 us; 256 of 404, 16/4: 212 MB in 46).  KW wavefronts, each
// by itself: blocks of 32 positions in turn, the next block's keys requested when the last key has been read, its values when the last
// value has.
template <int D, int KW, bool LENS>
__device__ __forceinline__ void shared_tail(const SharedArgs& p, uint8_t* lds, float* ml, int* table_lds) {
  constexpr int KB = 32, TILE = KB * 2 * D, LOADS = TILE / 1024;
  static_assert(128 * D <= 2 * TILE, "the wavefronts' sums fit the buffers");
  const int lane = threadIdx.x & 63, col = lane & 31, kw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wg = (int)blockIdx.x - p.prefix_wgs, bh = p.by_tails(wg), slice = wg - bh * p.tails, b = p.by_hkv(bh), kvh = bh - b * p.Hkv;
  const int k0 = p.s0 + slice * p.tail, k1 = k0 + p.tail < p.T ? k0 + p.tail : p.T;
  const int vis = visible(p, b), seen = vis && vis < k1 ? vis : k1;  // rows behind the sequence's length: zeros
  SharedPages pages{p.table + (int64_t)b * p.P, nullptr, 0};
  pages.fetch(p, k0, table_lds, KW * 64);
  if (p.table_lds) __syncthreads();
  const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(pa_lds_void*)lds + kw * 2 * TILE);
  uint8_t* const ks = lds + kw * 2 * TILE;
  int kb0 = k0 + kw * KB;
  SharedRows<D> rows;
  rows.start(p.q + ((int64_t)b * p.Hq + kvh * p.G + (col < p.G ? col : 0)) * D, lane >> 5, vis);
  if (kb0 < seen) {  // wavefront-uniform, as all below
    // (us with a vector and a scalar load here: 8 x 2591 positions of which 2048 shared 9.7 | 10.0, 256 x 4500 of 4096 with lengths 40.6 | 38.8)
    int64_t page = pages.template page_of<KB, LENS>(p, kb0, seen);
    pages.template load<D, KB, LOADS, true, false>(p, kvh, kb0, page, seen, 0, at, 0);
    pages.template load<D, KB, LOADS, false, true>(p, kvh, kb0, page, seen, 0, at + TILE, 0);
    page = pages.template page_of<KB>(p, kb0 + KW * KB, seen);
    // The queries have arrived, as far as the compiler knows too: otherwise it waits for them in every turn, by a count that takes in
    // the blocks on their way.
    SH_WAIT_VMCNT(0);
    for (;;) {
      const int next = kb0 + KW * KB;
      const bool more = next < seen;
      asm volatile("" ::: "memory");
      rows.template attend<1, false, false>(
          ks, ks + TILE, kb0, kb0 + KB > vis, p.T, p.scale_log2e,
          [&] {
            SH_WAIT_LGKM();
            if (more) pages.template load<D, KB, LOADS, true, false>(p, kvh, next, page, seen, 0, at, 0);
          },
          [&] {
            if (more) SH_WAIT_VMCNT(LOADS);  // this block's values have landed
            else SH_WAIT_VMCNT(0);
            asm volatile("" ::: "memory");
          });
      if (!more) break;
      SH_WAIT_LGKM();
      pages.template load<D, KB, LOADS, false, true>(p, kvh, next, page, seen, 0, at + TILE, 0);
      page = pages.template page_of<KB>(p, next + KW * KB, seen);
      SH_WAIT_VMCNT(LOADS);  // the next block's keys have
      kb0 = next;
    }
  }
  // (the sums go where this wavefront's own blocks were)
  const int64_t prefix = (int64_t)p.slices * p.Hkv * p.tiles32 * part_floats(D, 32);
  rows.template join_and_store<KW>(reinterpret_cast<v4f*>(lds), ml, kw, 0, 1, p.ws + prefix + (int64_t)wg * part_floats(D, p.G), p.G);
}

constexpr int SHARED_LDS = 512;  // bytes of the blocks of either kind of workgroup, per dimension

template <int D, int QW, int KW, int KB, bool LENS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void shared_attn_kernel(SharedArgs p) {
  static_assert(QW * KW == 4 && 2 * KW * KB * 4 * D == SHARED_LDS * D, "four wavefronts, 128 D bytes each");
  __shared__ float ml[4 * 128];
  extern __shared__ __align__(1024) uint8_t sh_lds[];  // blocks; page table
  int* const table = reinterpret_cast<int*>(sh_lds + SHARED_LDS * D);
  if ((int)blockIdx.x < p.prefix_wgs) shared_prefix<D, QW, KW, KB, LENS>(p, sh_lds, ml, table);
  else shared_tail<D, 4, LENS>(p, sh_lds, ml, table);
}

// The slices of a row added up: a half wavefront has 4 dimensions of the 32 rows of a tile, so that the prefix's slices are read by whole
// lines, and every PARTS-th slice, four of them requested before any is used; the parts meet in LDS.  (64 x 8448 positions: 17 MB in 5.4 us; 16 parts
// 36.6 us for the call instead of 33.8, eight slices requested at once 35.4; 8 x 2591 with four parts 10.0 instead of 9.6.)
template <int D, int PARTS>
__global__ __launch_bounds__(PARTS * 32) void shared_merge_kernel(const float* ws, uint16_t* out, int slices, int tails, int tiles32, int rows, int Hkv, int G) {
  constexpr int GRP = 4;
  __shared__ float sums[PARTS][6][32];
  const int col = threadIdx.x & 31, part = threadIdx.x >> 5, c = blockIdx.y;  // group of 4 dimensions
  const int kvh = (int)blockIdx.x / tiles32, t32 = (int)blockIdx.x - kvh * tiles32;
  const int n32 = rows - t32 * 32 < 32 ? rows - t32 * 32 : 32, row = t32 * 32 + (col < n32 ? col : n32 - 1);
  const int b = row / G, g = row - b * G;
  const int64_t step = (int64_t)Hkv * tiles32 * part_floats(D, 32);
  const float* const prefix = ws + (int64_t)blockIdx.x * part_floats(D, 32);
  const float* const tail = ws + slices * step + ((int64_t)b * Hkv + kvh) * tails * part_floats(D, G);
  float mm = -INFINITY, den = 0.0f, n[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = part; s0 < slices + tails; s0 += PARTS * GRP) {
    float m[GRP], l[GRP];
    v4f v[GRP];
    float mx = mm;
#pragma unroll
    for (int i = 0; i < GRP; ++i) {
      const int s = s0 + i * PARTS;
      const bool is_tail = s >= slices;
      const float* from = is_tail ? tail + (s - slices) * part_floats(D, G) : prefix + s * step;
      const int k = is_tail ? G : n32, at = is_tail ? g : row - t32 * 32;
      m[i] = -INFINITY;
      l[i] = 0.0f;
      v[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
      if (s < slices + tails) {
        m[i] = from[D * k + at];
        l[i] = from[(D + 1) * k + at];
        v[i] = *reinterpret_cast<const v4f*>(from + (c * k + at) * 4);
      }
    }
#pragma unroll
    for (int i = 0; i < GRP; ++i) mx = fmaxf(mx, m[i]);
    const float old = mm == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mm - mx);
    mm = mx;
    den *= old;
#pragma unroll
    for (int d = 0; d < 4; ++d) n[d] *= old;
#pragma unroll
    for (int i = 0; i < GRP; ++i) {
      const bool some = m[i] != -INFINITY;  // otherwise only the maximum was written
      const float w = some ? __builtin_amdgcn_exp2f(m[i] - mm) : 0.0f;
      den = __builtin_fmaf(some ? l[i] : 0.0f, w, den);
#pragma unroll
      for (int d = 0; d < 4; ++d) n[d] = __builtin_fmaf(some ? v[i][d] : 0.0f, w, n[d]);
    }
  }
  sums[part][0][col] = mm;
  sums[part][1][col] = den;
#pragma unroll
  for (int d = 0; d < 4; ++d) sums[part][2 + d][col] = n[d];
  __syncthreads();
  if (part > 0 || col >= n32) return;
  float mx = mm;
#pragma unroll
  for (int i = 1; i < PARTS; ++i) mx = fmaxf(mx, sums[i][0][col]);
  den = 0.0f;
#pragma unroll
  for (int d = 0; d < 4; ++d) n[d] = 0.0f;
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    const float mi = sums[i][0][col], w = mi == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mi - mx);
    den = __builtin_fmaf(sums[i][1][col], w, den);
#pragma unroll
    for (int d = 0; d < 4; ++d) n[d] = __builtin_fmaf(sums[i][2 + d][col], w, n[d]);
  }
  const float r = attn_inv_denominator(den);
  *reinterpret_cast<uint2*>(out + (((int64_t)b * Hkv + kvh) * G + g) * D + c * 4) =
      make_uint2(pack_bf16x2(__fmul_rn(n[0], r), __fmul_rn(n[1], r)), pack_bf16x2(__fmul_rn(n[2], r), __fmul_rn(n[3], r)));
}

// How a call is cut.
struct SharedPlan {
  int64_t s0;  // positions that the prefix takes; 0: none, the decode kernel takes all of them
  int qw, slice, slices, tail, tails;
  int64_t bytes;
};

constexpr int SHARED_TABLE_MAX = 2048;  // page-table entries kept in LDS

// Whether reading the first s0 positions once is the faster form: what each form has beside the other.  The decode kernel reads the keys and
// values of B x T positions (0.1 a megabyte), and past 2048 of them it has two launches with a merge of more slices (4).  Here there is the
// merge (2, and 2 more where the decode kernel is a single launch), the tails' megabytes, and 0.6 a million products of a row with a
// position and 128 dimensions.  The weights are fitted to both forms' times from a graph at 11168 random sizes (2 to 128 sequences, 2 to 8 KV heads
// of 1 to 8 rows, both head dimensions, pages of 16 to 256, 64 to 10000 positions): at 15385 others the rule's choice costs 1.008 times the
// better form's time in the mean, always sharing 1.098, never 1.63.  us, decode kernel | shared: 2 x 1088 positions of which 1024 shared, 16/4 heads of
// 128 7.8 | 8.6; 2 x 2112 of 2048 9.5 | 8.7; 8 x 2112 of 2048 12.2 | 8.9; 32 x 576 of 512 10.4 | 9.5; 32 x 1024 of 512 12.0 | 14.4;
// 32 x 2560 of 2048 23.3 | 16.3; 122 x 152 of 128 8.9 | 15.8.
static bool sharing_pays(int64_t B, int64_t Hkv, int64_t G, int64_t D, int64_t T, int64_t s0) {
  const double position = 4e-6 * (double)(Hkv * D);  // megabytes
  const double apart = 0.1 * position * (double)(B * T) + (T > 2048 ? 4.0 : 0.0);
  const double shared = 2.0 + (T > 256 ? 0.0 : 2.0) + 0.1 * position * (double)(B * (T - s0)) + 0.6e-6 / 128 * (double)(D * Hkv * G) * (double)B * (double)s0;
  return shared < apart;
}

// The same for a model's step.  Its other form rotates, writes the pages and attends in one launch (and a merge); sharing has a launch in front
// for the first two.  Weights fitted to blocks' times in a graph at 1550 random sizes that the rule above shares (7 head layouts), of
// which a third lost by it; the merge that sharing saves past 2048 positions counts by how much of them is shared, and by more than the fit
// gives it (1.6), so that few sequences, level within 1 us there, share.  At 840 sizes it was not fitted to, a third of them with lengths: 28 lose
// more than 1 us by this rule (8 of 129 at most), 123 by the operator's (8 of 129 at most), 94 us and 333 in all; 91 us of the 1441 that sharing can gain are
// left; 0.5 % above the better form's time in the mean, 1.0 % by the operator's rule.  us a block, apart | shared:
// not shared  57 x 217 positions of which 208 shared, 32/8 heads of 128 105.9 | 115.9; 49 x 1162 of 400, 8/8 of 64 47.0 | 51.3; 3 x 2097 of 592,
//             32/8 of 128 81.5 | 85.0;
// shared      16 x 2101 of 2096, 24/4 heads of 64 41.5 | 39.5; 40 x 4096 of 4000 63.8 | 47.0; 16 x 8200 of 8000, 16/4 of 128 73.2 | 49.5;
//             8 x 2101 of 2096 37.6 | 35.7; 2 x 2101 of 2096 31.6 | 32.7.
static bool step_sharing_pays(int64_t B, int64_t Hkv, int64_t G, int64_t D, int64_t T, int64_t s0) {
  const double position = 4e-6 * (double)(Hkv * D);  // megabytes
  const double apart = (0.05 + 0.006 * (double)G) * position * (double)(B * T) + (T > 2048 ? 2.1 * (double)s0 / (double)T : 0.0);
  const double shared = 2.2 + (T > 256 ? 0.0 : 3.0) + 0.09 * position * (double)(B * (T - s0));
  return shared < apart;
}

static SharedPlan shared_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t T, int64_t shared) {
  SharedPlan p{};
  const int64_t G = Hq / Hkv, rows = B * G, s0 = (shared < T ? shared : T) / 64 * 64, cus = device_cus();
  if (B < 2 || s0 < 64 || !sharing_pays(B, Hkv, G, D, T, s0)) return p;
  p.s0 = s0;
  // A workgroup has 64 rows, or 128 where there are many: fewer keys and values go into the compute units then (64 x 8448 positions of which
  // 8192 shared, 32/8 heads of 128 39.2 | 36.3 us), but too few workgroups otherwise (32 x 4300 of 4096, 16/4 heads of 128 14.6 | 16.0).
  p.qw = rows > 128 && (rows + 63) / 64 * Hkv * (s0 / 256) > 2 * cus ? 4 : 2;
  // As many slices as fill the compute units once, half (three quarters) as many where the tails are most of the work anyway (with lengths, 256 x 4500
  // positions of which 4096 shared, 16/4 heads of 128, half, three quarters, all: 38.1, 39.9, 41.6; 256 x 2400 of 2048, 24/4 of 64: 27.9, 21.8, 22.9; over
  // the best of the three in the mean of random sizes of 8 head layouts 1.009, 1.011, 1.020 at 218 such of 128, 1.019, 1.012, 1.019 at 328 of 64, and
  // 1.038, 1.012, 1.011 at 654 with shorter tails); but short ones cost the merge more than they save (16 x 8300 of 8192, 16/4 heads of 128,
  // slices of 64, 128, 256, 512: 24.5, 18.4, 15.4, 17.7; 8 x 2591 of 2048, 64, 128, 256: 13.7, 11.4, 12.3).
  const int64_t tiles = (rows + 32 * p.qw - 1) / (32 * p.qw), shortest = s0 < 4096 ? 128 : 256;
  int64_t want = (B * (T - s0) < 8 * s0 ? cus : D == 64 ? cus * 3 / 4 : cus / 2) / (tiles * Hkv);
  if (want < 1) want = 1;
  int64_t slice = ((s0 + want - 1) / want + 63) / 64 * 64;
  if (slice < shortest) slice = shortest;
  p.slice = (int)slice;
  p.slices = (int)((s0 + slice - 1) / slice);
  if (T > s0) {
    // one workgroup of tails per compute unit, two of half the size at head dimension 64; 128 positions are one block for each wavefront.  (One, two
    // or four, over the best of them in the mean of random sizes: 1.019, 1.015, 1.029 at 750 of head dimension 64, 1.014, 1.022, 1.043 at 450 of 128; us
    // 100 x 900 of 768, 24/4 of 64, with lengths 12.2, 12.2, 14.5; 33 x 1401 of 1008 12.3, 10.7, 10.6; 64 x 1000 of 512, 16/4 of 128 19.5, 21.1, 23.6.)
    int64_t n = (D == 64 ? 2 : 1) * cus / (B * Hkv), most = (T - s0 + 127) / 128;
    if (n > most) n = most;
    if (n < 1) n = 1;
    p.tail = (int)(((T - s0 + n - 1) / n + 127) / 128 * 128);
    p.tails = (int)((T - s0 + p.tail - 1) / p.tail);
  }
  p.bytes = ((int64_t)p.slices * Hkv * ((rows + 31) / 32) * part_floats((int)D, 32) + B * Hkv * p.tails * part_floats((int)D, (int)G)) * (int64_t)sizeof(float);
  return p;
}

template <int D, int QW>
static int launch_shared(SharedArgs& a, int64_t tail_wgs, uint16_t* out, hipStream_t st) {
  constexpr int KW = 4 / QW, KB = 64 / KW;
  size_t lds = SHARED_LDS * D;
  a.tiles = (a.rows + 32 * QW - 1) / (32 * QW);
  a.by_tiles = UDiv::of((uint32_t)a.tiles);
  if (a.page_shift < (KB == 64 ? 6 : 5) || (tail_wgs && a.page_shift < 5)) {
    const int64_t most = a.slice > a.tail ? a.slice : a.tail, entries = (most + a.page - 1) / a.page + 1;
    a.table_lds = entries <= SHARED_TABLE_MAX ? (int)entries : 0;
    lds += (size_t)a.table_lds * sizeof(int);
  }
  const int64_t combos = (int64_t)a.slices * a.Hkv, prefix_wgs = (combos + 7) / 8 * 8 * a.tiles;
  if (prefix_wgs + tail_wgs > 0x7fffffff) return AQ_E_RANGE;
  a.prefix_wgs = (int)prefix_wgs;
  // (a form of its own where sequences may end anywhere: its masks cost the others 3 to 7 % of their time)
  queue_kernel(a.lens ? shared_attn_kernel<D, QW, KW, KB, true> : shared_attn_kernel<D, QW, KW, KB, false>,
               dim3((unsigned)(prefix_wgs + tail_wgs)), dim3(256), lds, st, a);
  if (const int rc = (int)hipGetLastError()) return rc;
  const int64_t tiles = (int64_t)a.Hkv * a.tiles32;
  const bool few = tiles * (D / 4) < 16 * device_cus();
  queue_kernel(few ? shared_merge_kernel<D, 8> : shared_merge_kernel<D, 4>, dim3((unsigned)tiles, D / 4), dim3(few ? 256 : 128), 0, st, a.ws, out,
               a.slices, a.tails, a.tiles32, a.rows, a.Hkv, a.G);
  return (int)hipGetLastError();
}

}  // namespace aq

extern "C" int64_t aq_paged_attn_decode_shared_positions(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t total_len, int64_t shared_len) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || total_len <= 0 || shared_len < 0 || total_len > (1 << 30) || (D != 64 && D != 128) ||
      !aq::attn_group_ok(Hq / Hkv))
    return 0;
  return aq::shared_plan(B, Hq, Hkv, D, total_len, shared_len).s0;
}

extern "C" int64_t aq_paged_attn_decode_shared_step_positions(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t total_len, int64_t shared_len) {
  const int64_t s0 = aq_paged_attn_decode_shared_positions(B, Hq, Hkv, D, total_len, shared_len);
  return s0 && aq::step_sharing_pays(B, Hkv, Hq / Hkv, D, total_len, s0) ? s0 : 0;
}

extern "C" int64_t aq_paged_attn_decode_shared_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t total_len,
                                                               int64_t shared_len) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || total_len <= 0 || shared_len < 0 || total_len > (1 << 30) || (D != 64 && D != 128)) return 0;
  const aq::SharedPlan p = aq::shared_plan(B, Hq, Hkv, D, total_len, shared_len);
  return p.s0 ? p.bytes : aq_paged_attn_decode_workspace_bytes(B, Hq, Hkv, total_len);
}

extern "C" int aq_paged_attn_decode_shared(const void* q, const void* k_cache, const void* v_cache, const int64_t* page_table,
                                           int64_t P, int64_t total_len, int64_t shared_len, const int64_t* seq_lens,
                                           int64_t page_size, int64_t n_pages, float scale, void* out, int64_t B, int64_t Hq,
                                           int64_t Hkv, int64_t D, void* workspace, int64_t workspace_bytes, void* stream) {
  if (D != 64 && D != 128) return AQ_E_SHAPE;
  if (B < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || P <= 0 || total_len <= 0 || shared_len < 0 || page_size <= 0 || n_pages <= 0 ||
      !(scale > 0.0f) || !aq::attn_group_ok(Hq / Hkv))
    return AQ_E_SHAPE;
  if (B == 0) return AQ_OK;
  if (!q || !k_cache || !v_cache || !page_table || !out) return AQ_E_NULL;
  if (aq::check_ptr16(q) || aq::check_ptr16(k_cache) || aq::check_ptr16(v_cache) || aq::check_ptr16(out)) return AQ_E_ALIGN;
  // 32-bit positions and page ids, 32-bit offsets inside a block of 64 positions, one workgroup index
  if (total_len > (1 << 30) || n_pages > 0x7fffffff || B > (1 << 24) / Hq || Hkv * D > (1 << 24)) return AQ_E_RANGE;
  const aq::SharedPlan plan = aq::shared_plan(B, Hq, Hkv, D, total_len, shared_len);
  if (!plan.s0)
    return aq_paged_attn_decode(q, k_cache, v_cache, page_table, P, total_len, seq_lens, page_size, n_pages, scale, out, B, Hq, Hkv, D,
                                workspace, workspace_bytes, stream);
  if (!workspace) return AQ_E_NULL;
  if (aq::check_ptr16(workspace)) return AQ_E_ALIGN;
  if (workspace_bytes < plan.bytes) return AQ_E_WORKSPACE;
  hipStream_t st = static_cast<hipStream_t>(stream);
  aq::SharedArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.kc = static_cast<const uint16_t*>(k_cache);
  a.vc = static_cast<const uint16_t*>(v_cache);
  a.table = page_table;
  a.lens = seq_lens;
  a.ws = static_cast<float*>(workspace);
  a.page = page_size;
  a.n_pages = n_pages;
  a.P = P;
  a.scale_log2e = scale * 1.44269504088896341f;
  a.T = (int)total_len;
  a.s0 = (int)plan.s0;
  a.rows = (int)(B * (Hq / Hkv));
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.G = (int)(Hq / Hkv);
  a.slice = plan.slice;
  a.slices = plan.slices;
  a.tiles32 = (a.rows + 31) / 32;
  a.tail = plan.tail;
  a.tails = plan.tails;
  a.page_shift = -1;
  for (int sh = 5; sh < 31; ++sh)
    if (page_size == ((int64_t)1 << sh)) a.page_shift = sh;
  a.by_g = aq::UDiv::of((uint32_t)a.G);
  a.by_hkv = aq::UDiv::of((uint32_t)a.Hkv);
  a.by_tails = aq::UDiv::of((uint32_t)(a.tails ? a.tails : 1));
  a.page_rows = page_size % (512 / D) == 0;
  // (pages above 2^30 hold every position: the quotient is 0 for any divisor as large)
  a.by_page = aq::UDiv::of((uint32_t)(page_size < (1 << 30) ? page_size : 1 << 30));
  const int64_t tail_wgs = B * Hkv * plan.tails;
  uint16_t* const o = static_cast<uint16_t*>(out);
  if (D == 128) return plan.qw == 2 ? aq::launch_shared<128, 2>(a, tail_wgs, o, st) : aq::launch_shared<128, 4>(a, tail_wgs, o, st);
  return plan.qw == 2 ? aq::launch_shared<64, 2>(a, tail_wgs, o, st) : aq::launch_shared<64, 4>(a, tail_wgs, o, st);
}
