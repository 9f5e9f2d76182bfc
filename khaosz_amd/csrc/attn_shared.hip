// Decode attention of a batch whose sequences begin with the same pages (samples of one prompt, beams, requests behind one
// system prompt; the reference's prefix cache maps such pages into every sequence's table, astrai/inference/core/cache.py:68-185, and its
// attention then gathers and reads them once per sequence, cache.py:254-274).  Here the shared positions are read and multiplied
// once for the whole batch:
//
//   prefix   the G query heads of a KV head of all B sequences are B G rows of one product against the shared keys: scores,
//            softmax statistics and values per tile of rows and range of positions, left as partial results;
//   tail     each sequence's own positions, by the decode kernel (attn_tail);
//   merge    the partial results of a (sequence, query head) are weighed by exp2(maximum - overall maximum) and added up.
//
// softmax over two ranges is the softmax over both: with m, l, n the maximum, denominator and numerator of each range,
// out = (n1 2^(m1 - m) + n2 2^(m2 - m)) / (l1 2^(m1 - m) + l2 2^(m2 - m)), m = max(m1, m2).  All of them are fp32; probabilities
// are rounded to bf16 (off by 2^-9 of themselves at most) where the matrix core takes them, the denominator sums them unrounded.
//
// The prefix kernel computes S^T = K Q^T and O^T = V^T P^T as the prefill kernel does (attn_prefill.hip has the layout): a lane
// has the scores of one row, nothing changes lanes, K and V rows go straight into LDS one block ahead of the products.
#include "aq_attn.h"
#include "aq_common.h"
#include "aq_rows.h"

namespace aq {

struct SharedArgs {
  const uint16_t* q;     // [B, Hq, D]
  const uint16_t* kc;    // [n_pages, page, Hkv, D]
  const uint16_t* vc;
  const int64_t* table;  // the first sequence's row of the page table: the shared pages
  const int64_t* lens;   // [B] or null
  float* ws;             // [B, Hq, NS, D + 4]; slots 0 .. slices - 1 are written
  int64_t page, n_pages, P;
  float scale_log2e;
  int T, rows, Hq, Hkv, G, NS;
  int blocks, per_slice, slices, tiles;  // blocks of 64 shared positions, of one slice; slices; tiles of rows
  int page_shift;                        // log2 of the page size, or -1
  int table_lds;                         // entries of the page table that a slice may need, kept in LDS (0: read from memory)
  UDiv by_g, by_page, by_tiles, by_hkv;
};

constexpr float SHARED_MASKED = -1.0e30f;  // score (exp2 domain) of a position the sequence may not attend to, as in the decode kernel

// QW x KW wavefronts: QW tiles of 32 rows side by side on the same block of 64 positions, KW blocks at a time.
template <int D, int QW, int KW>
__global__ __launch_bounds__(QW* KW * 64) __attribute__((amdgpu_waves_per_eu(D == 128 && KW == 2 ? 1 : 2))) void shared_attn_kernel(SharedArgs p) {
  constexpr int KB = 64, NT = KB / 32, DSTEPS = D / 16, DT = D / 32;
  constexpr int ROWB = 2 * D;                       // bytes of a K or V row
  constexpr int RPI = 1024 / ROWB, LPR = 64 / RPI;  // rows of a 1 KiB load, lanes of a row
  constexpr int TILE = KB * ROWB;                   // bytes of a block's K (or V)
  constexpr int LOADS = TILE / 1024 / QW;           // 1 KiB loads of K (and of V) per wavefront and block
  constexpr int BUF = KW * 2 * TILE;
  static_assert(LOADS >= 1 && TILE % (1024 * QW) == 0, "whole loads per wavefront");
  static_assert((KW - 1) * QW * (DT * 16 + 2) * 256 <= 2 * BUF, "the wavefronts' sums fit the buffers");
  __shared__ int seen_s[QW];
  extern __shared__ __align__(1024) uint8_t sh_lds[];  // 2 buffers of KW [K block | V block]; page table
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qw = wave % QW, kw = wave / QW;
  const int col = lane & 31, g = lane >> 5;
  // Workgroups i and i + 8 run on one XCD: the tiles of a (KV head, slice) follow one another there, so that its L2 has the keys and
  // values the first one read.
  const int turn = (int)blockIdx.x >> 3, ty = p.by_tiles(turn), tile = turn - ty * p.tiles, combo = ty * 8 + ((int)blockIdx.x & 7);
  if (combo >= p.slices * p.Hkv) return;
  const int slice = p.by_hkv(combo), kvh = combo - slice * p.Hkv;
  const int j0 = slice * p.per_slice, j1 = j0 + p.per_slice < p.blocks ? j0 + p.per_slice : p.blocks;
  const int nit = (j1 - j0 + KW - 1) / KW;

  const int r0 = (tile * QW + qw) * 32, row = r0 + col < p.rows ? r0 + col : p.rows - 1;  // rows past the end: the last one again
  const int b = p.by_g(row), head = kvh * p.G + (row - b * p.G);
  int vis = p.T, seen = p.T;  // positions this lane's row may attend to; that any row of the workgroup looks at
  int* const table = reinterpret_cast<int*>(sh_lds + 2 * BUF);
  auto phys_of = [&](int lp) -> int {
    const int64_t t = lp < p.P ? p.table[lp] : -1;
    return t >= 0 && t < p.n_pages ? (int)t : -1;
  };
  const int lp0 = p.table_lds ? (int)p.by_page((uint32_t)(j0 * KB)) : 0;
  if (p.table_lds) {
    for (int i = tid; i < p.table_lds; i += QW * KW * 64) table[i] = phys_of(lp0 + i);
    if (!p.lens) __syncthreads();
  }
  if (p.lens) {
    const int64_t n = p.lens[b];
    vis = n <= 0 ? 0 : n < p.T ? (int)n : p.T;
    int most = vis ? vis : p.T;  // a row without any length weighs every position alike
#pragma unroll
    for (int off = 32; off; off >>= 1) {
      const int o = __shfl_xor(most, off, 64);
      most = o > most ? o : most;
    }
    if (kw == 0 && lane == 0) seen_s[qw] = most;
    __syncthreads();
    seen = seen_s[0];
#pragma unroll
    for (int i = 1; i < QW; ++i) seen = seen_s[i] > seen ? seen_s[i] : seen;
  }

  const int chunk0 = qw * LOADS;
  int pc[LOADS];  // this lane's piece of the rows that the wavefront's loads bring: elements into the row
#pragma unroll
  for (int c = 0; c < LOADS; ++c) pc[c] = ((lane % LPR) ^ row_key<D>((chunk0 + c) * RPI + lane / LPR)) * 8;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(pa_lds_void*)sh_lds;
  auto issue = [&](int it, int buf) __attribute__((always_inline)) {
    const int j = j0 + it * KW + kw;
    if (j >= j1) return;  // wavefront-uniform
    const uint32_t dst = __builtin_amdgcn_readfirstlane(lds0 + buf * BUF + kw * 2 * TILE + chunk0 * 1024);
    const int rows = seen - j * KB;  // rows that no one looks at are zeros, whatever is stored there
    const uint16_t* const zero = reinterpret_cast<const uint16_t*>(pa_zero_row);
    if (p.page_shift >= 6) {  // the whole block lies in one page
      const int lp = __builtin_amdgcn_readfirstlane((j * KB) >> p.page_shift);
      const int64_t phys = lp < p.P ? p.table[lp] : -1;
      const bool mapped = phys >= 0 && phys < p.n_pages;
      const int64_t first = mapped ? (((phys << p.page_shift) + (j * KB - (lp << p.page_shift))) * p.Hkv + kvh) * D : 0;
      const int step = p.Hkv * D;
#pragma unroll
      for (int c = 0; c < LOADS; ++c) {
        const int r = (chunk0 + c) * RPI + lane / LPR;
        const bool there = mapped && r < rows;
        const uint32_t at = (uint32_t)(r * step + pc[c]);
        load_row_lds(there ? p.kc + first + at : zero + pc[c], dst + c * 1024);
        load_row_lds(there ? p.vc + first + at : zero + pc[c], dst + TILE + c * 1024);
      }
      return;
    }
    // every address first, then the loads: a load is a fence to the compiler, and a lookup behind each one would wait for LDS once per row
    int64_t at[LOADS];
#pragma unroll
    for (int c = 0; c < LOADS; ++c) {
      const int r = (chunk0 + c) * RPI + lane / LPR, key = j * KB + r;
      const int lp = p.by_page((uint32_t)key), in_page = key - lp * (int)p.page;
      const int phys = r >= rows ? -1 : p.table_lds ? table[lp - lp0] : phys_of(lp);
      at[c] = phys < 0 ? -1 : (((int64_t)phys * p.page + in_page) * p.Hkv + kvh) * D;
    }
#pragma unroll
    for (int c = 0; c < LOADS; ++c) {
      load_row_lds((at[c] < 0 ? zero : p.kc + at[c]) + pc[c], dst + c * 1024);
      load_row_lds((at[c] < 0 ? zero : p.vc + at[c]) + pc[c], dst + TILE + c * 1024);
    }
  };
  issue(0, 0);

  uint4 qf[DSTEPS];  // Q^T operand: lane = (row col, dimensions 16 step + 8 g .. + 8)
  {
    const uint16_t* src = p.q + ((int64_t)b * p.Hq + head) * D + g * 8;
#pragma unroll
    for (int st = 0; st < DSTEPS; ++st) qf[st] = *reinterpret_cast<const uint4*>(src + st * 16);
  }
  // fragment addresses inside a block: K row `col`, piece 2 step + g; V rows 4 g + i / 4 (and 8 further), i = lane % 16,
  // dimensions 16 (lane / 16 % 2) + 4 (i % 4) of a 32-dimension tile
  const int kfr = col * ROWB + ((g ^ row_key<D>(col)) << 4);  // ^ (2 step) << 4
  const int vrow = 4 * g + (lane & 15) / 4, vpiece = ((lane >> 4) & 1) * 2 + (lane & 3) / 2;
  const int vfr0 = vrow * ROWB + ((vpiece ^ row_key<D>(vrow)) << 4) + (lane & 1) * 8;  // ^ dt << 6
  const int vfr1 = (vrow + 8) * ROWB + ((vpiece ^ row_key<D>(vrow + 8)) << 4) + (lane & 1) * 8;

  pa_f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.0f;
  float m = -INFINITY, l = 0.0f;  // bound of this lane's row's scores; this lane's half of its denominator
  const bool idle = r0 >= p.rows;  // wavefront-uniform: no row here, only loads

  for (int it = 0; it < nit; ++it) {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): block `it` has landed
    __syncthreads();                     // ... everyone's part of it, and everyone is done with the one before
    if (it + 1 < nit) issue(it + 1, (it + 1) & 1);
    const int j = j0 + it * KW + kw, kb0 = j * KB;
    if (idle || j >= j1) continue;  // wavefront-uniform
    const bool some = p.lens && __builtin_amdgcn_ballot_w64(kb0 + KB > vis) != 0;  // some row may not attend to some position
    if (some && __builtin_amdgcn_ballot_w64(vis == 0 || kb0 < vis) == 0) continue;  // none to any
    const uint8_t* ks = sh_lds + (it & 1) * BUF + kw * 2 * TILE;
    const uint8_t* vs = ks + TILE;
    // ---- scores; the fragments of K are read two steps ahead of the products that take them
    pa_f32x16 s[NT];
    {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[t][r] = 0.0f;
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
    // ---- softmax of this lane's row; register r of tile kt is position kb0 + 32 kt + 8 (r / 4) + 4 g + r % 4
    float sc = p.scale_log2e;
    if (some) {  // the scores are scaled here, so that a masked one has the same value in every slice
#pragma unroll
      for (int kt = 0; kt < NT; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = kb0 + kt * 32 + 8 * (r / 4) + 4 * g + (r % 4);
          s[kt][r] = key < vis ? s[kt][r] * sc : SHARED_MASKED;
        }
      sc = 1.0f;
    }
    float bm = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < NT; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r) bm = fmaxf(bm, s[kt][r]);
    const LanePair b2 = lanes32_pair(bm);
    bm = fmaxf(b2.x, b2.y) * sc;
    // m only has to bound the exponents: it is raised, and the sums rescaled, when a row of the wavefront would see one above 2^8
    if (__builtin_amdgcn_ballot_w64(bm > m + 8.0f) != 0) {  // wavefront-uniform
      const float mn = fmaxf(m, bm), alpha = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
    }
    uint4 pf[NT][2];  // P^T operands: tile kt, positions 16 s2 .. + 16
#pragma unroll
    for (int kt = 0; kt < NT; ++kt) {
      float pv[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        pv[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][r], sc, -m));
        l += pv[r];
      }
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2)
        pf[kt][s2] = make_uint4(pack_bf16x2(pv[8 * s2 + 0], pv[8 * s2 + 1]), pack_bf16x2(pv[8 * s2 + 2], pv[8 * s2 + 3]),
                                pack_bf16x2(pv[8 * s2 + 4], pv[8 * s2 + 5]), pack_bf16x2(pv[8 * s2 + 6], pv[8 * s2 + 7]));
    }
    // ---- O^T += V^T P^T; all fragments of V are read before the products, whose chains alternate
    constexpr int KK = 2 * NT;
    pa_bf16x8 fv[DT][KK];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const uint8_t* at = vs + kk * 16 * ROWB;
        const pa_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_lds_s16x4*)(at + (vfr0 ^ (dt << 6))));
        const pa_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_lds_s16x4*)(at + (vfr1 ^ (dt << 6))));
        fv[dt][kk] = __builtin_bit_cast(pa_bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d0 = 0; d0 < DT; d0 += 2)
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int dt = d0; dt < d0 + 2; ++dt)
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fv[dt][kk], __builtin_bit_cast(pa_bf16x8, pf[kk >> 1][kk & 1]), o[dt], 0, 0, 0);
  }
  const LanePair l2 = lanes32_pair(l);
  l = l2.x + l2.y;
  // ---- the KW wavefronts of a tile of rows add up their sums
  if constexpr (KW > 1) {
    constexpr int SUMS = DT * 16 * 64;  // floats
    float* const to = reinterpret_cast<float*>(sh_lds) + ((kw - 1) * QW + qw) * (SUMS + 128) + lane;
    __syncthreads();  // everyone is done with the blocks
    if (kw > 0) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) to[(dt * 16 + r) * 64] = o[dt][r];
      to[SUMS] = m;
      to[SUMS + 64] = l;
    }
    __syncthreads();
    if (kw > 0) return;
#pragma unroll
    for (int k = 1; k < KW; ++k) {
      const float* from = reinterpret_cast<const float*>(sh_lds) + ((k - 1) * QW + qw) * (SUMS + 128) + lane;
      const float mk = from[SUMS], lk = from[SUMS + 64], mn = fmaxf(m, mk);
      const float a0 = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn), a1 = mk == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mk - mn);
      m = mn;
      l = l * a0 + lk * a1;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] = __builtin_fmaf(from[(dt * 16 + r) * 64], a1, o[dt][r] * a0);
    }
  }
  // ---- register r of tile dt is dimension 32 dt + 8 (r / 4) + 4 g + r % 4 of row col
  if (r0 + col < p.rows) {
    float* part = p.ws + (((int64_t)b * p.Hq + head) * p.NS + slice) * (D + 4);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int a = 0; a < 4; ++a)
        *reinterpret_cast<float4*>(part + dt * 32 + 8 * a + 4 * g) = make_float4(o[dt][4 * a], o[dt][4 * a + 1], o[dt][4 * a + 2], o[dt][4 * a + 3]);
    if (g == 0) *reinterpret_cast<float2*>(part + D) = make_float2(m, l);
  }
}

// How a call is cut: `blocks` blocks of 64 shared positions (a part of one is left to the tails), per_slice of them to a workgroup.
struct SharedPlan {
  int64_t s0;  // positions that the prefix kernel takes; 0: none, the decode kernel takes all of them
  int qw, kw, blocks, per_slice, slices, tail;
};

constexpr int SHARED_TABLE_MAX = 2048;  // page-table entries kept in LDS

static SharedPlan shared_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t T, int64_t shared) {
  SharedPlan p{};
  const int64_t rows = B * (Hq / Hkv), s0 = (shared < T ? shared : T) / 64 * 64;
  if (B < 2 || s0 < 64) {
    p.tail = (int)attn_tail_slices(T);
    return p;
  }
  p.s0 = s0;
  p.blocks = (int)(s0 / 64);
  if (rows <= 64) p.qw = 2, p.kw = 2;
  else p.qw = 4, p.kw = 1;
  const int64_t tiles = (rows + 32 * p.qw - 1) / (32 * p.qw), per_cu = p.kw == 1 ? 2 : D == 64 ? 2 : 1;
  int64_t want = device_cus() * per_cu / (tiles * Hkv);
  if (want < 1) want = 1;
  int64_t per = (p.blocks + want - 1) / want;
  per = (per + p.kw - 1) / p.kw * p.kw;
  p.per_slice = (int)per;
  p.slices = (int)((p.blocks + per - 1) / per);
  p.tail = T > s0 ? (int)attn_tail_slices(T - s0) : 0;
  return p;
}

template <int D, int QW, int KW>
static int launch_shared(SharedArgs& a, hipStream_t st) {
  constexpr int BUFS = 2 * KW * 2 * 64 * 2 * D;
  size_t lds = BUFS;
  a.tiles = (a.rows + 32 * QW - 1) / (32 * QW);
  a.by_tiles = UDiv::of((uint32_t)a.tiles);
  if (a.page_shift < 6) {
    const int64_t entries = ((int64_t)a.per_slice * 64 + a.page - 1) / a.page + 1;
    a.table_lds = entries <= SHARED_TABLE_MAX ? (int)entries : 0;
    lds += (size_t)a.table_lds * sizeof(int);
  }
  const int64_t combos = (int64_t)a.slices * a.Hkv;
  queue_kernel(shared_attn_kernel<D, QW, KW>, dim3((unsigned)((combos + 7) / 8 * 8 * a.tiles)), dim3(QW * KW * 64), lds, st, a);
  return (int)hipGetLastError();
}

}  // namespace aq

extern "C" int64_t aq_paged_attn_decode_shared_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t total_len,
                                                               int64_t shared_len) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || total_len <= 0 || shared_len < 0 || total_len > (1 << 30) || (D != 64 && D != 128)) return 0;
  const aq::SharedPlan p = aq::shared_plan(B, Hq, Hkv, D, total_len, shared_len);
  if (!p.s0) return aq_paged_attn_decode_workspace_bytes(B, Hq, Hkv, total_len);
  return aq::attn_workspace_bytes(B, Hq, p.slices + p.tail);
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
  const int ns = plan.slices + plan.tail;
  const int64_t tiles = (B * (Hq / Hkv) + 32 * plan.qw - 1) / (32 * plan.qw);
  if (((int64_t)plan.slices * Hkv + 8) * tiles > 0x7fffffff || B * Hkv * plan.tail > 0x7fffffff) return AQ_E_RANGE;
  if (!workspace) return AQ_E_NULL;
  if (aq::check_ptr16(workspace)) return AQ_E_ALIGN;
  if (workspace_bytes < aq::attn_workspace_bytes(B, Hq, ns)) return AQ_E_WORKSPACE;
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
  a.rows = (int)(B * (Hq / Hkv));
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.G = (int)(Hq / Hkv);
  a.NS = ns;
  a.blocks = plan.blocks;
  a.per_slice = plan.per_slice;
  a.slices = plan.slices;
  a.page_shift = -1;
  for (int sh = 6; sh < 31; ++sh)
    if (page_size == ((int64_t)1 << sh)) a.page_shift = sh;
  a.by_g = aq::UDiv::of((uint32_t)a.G);
  a.by_hkv = aq::UDiv::of((uint32_t)a.Hkv);
  // (pages above 2^30 hold every position: the quotient is 0 for any divisor as large)
  a.by_page = aq::UDiv::of((uint32_t)(page_size < (1 << 30) ? page_size : 1 << 30));
  int rc;
  if (D == 128)
    rc = plan.kw == 2 ? aq::launch_shared<128, 2, 2>(a, st) : aq::launch_shared<128, 4, 1>(a, st);
  else
    rc = plan.kw == 2 ? aq::launch_shared<64, 2, 2>(a, st) : aq::launch_shared<64, 4, 1>(a, st);
  if (rc) return rc;
  if (plan.tail) {
    rc = aq::attn_tail({q, k_cache, v_cache, page_table, seq_lens, a.ws, P, plan.s0, total_len, page_size, n_pages, B, Hq, Hkv, D, scale, ns,
                        plan.slices}, st);
    if (rc) return rc;
  }
  return aq::attn_merge(a.ws, out, B, Hq, ns, D, st);
}
