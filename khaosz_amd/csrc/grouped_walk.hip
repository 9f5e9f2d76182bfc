// Grouped products of many rows an expert: tiles of 128 rows x 256 weight rows, walked by one workgroup per compute unit whose K loop does not stop
// between them (as gemm_walk.hip walks the tiles of a single Linear).
//
// Inside an expert tiles go in groups of 8 by rows, then by columns: the 32 tiles that an XCD works on at a time share 2 MB of rows and 2 MB of
// weights.  The rows' tokens of the next tile are fetched into LDS under this tile's first step, for its first stages are requested in the
// last steps.
#include "aq_grouped.h"

namespace aq {

typedef int v2i_t __attribute__((ext_vector_type(2)));

constexpr int GW_BM = 128, GW_BK = 128, GW_THREADS = 512, GW_GROUP = 8;

// WM x WN wavefronts, each 32 TM rows by 32 TN weight rows of a tile of 128 x BN, K steps through NST stages.
template <int WM_, int TN_, int NST_>
struct GroupedShape {
  static constexpr int WM = WM_, WN = 8 / WM_, TM = 4 / WM_, TN = TN_, BN = 32 * TN * WN, NST = NST_;
  static constexpr int STAGE = (GW_BM + BN) * GW_BK;
  static constexpr int SX = NST * STAGE, TOK = SX + 8 * 64 * 4, OFF = TOK + GW_BM * 4, LDS = OFF + (GP_MAX_E + 1) * 4;
  static_assert(LDS <= 160 * 1024, "LDS of one compute unit");
  static_assert(NST >= 3, "a stage in use, one that lands, one on its way");
};

__device__ __forceinline__ void fetch_dword_to_lds(__amdgpu_buffer_rsrc_t r, void* to, uint32_t at) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)to, 4, at, 0, 0, 0);
}
__device__ __forceinline__ uint32_t load_dword(__amdgpu_buffer_rsrc_t r, uint32_t at) { return (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, (int)at, 0, 0); }
__device__ __forceinline__ uint32_t load_word(__amdgpu_buffer_rsrc_t r, uint32_t at) { return (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(r, (int)at, 0, 0); }
template <int POLICY = STORE_WT>
__device__ __forceinline__ void store_dword(uint32_t v, __amdgpu_buffer_rsrc_t r, uint32_t at) { __builtin_amdgcn_raw_buffer_store_b32(v, r, at, 0, POLICY); }
__device__ __forceinline__ void store_word(uint32_t v, __amdgpu_buffer_rsrc_t r, uint32_t at) { __builtin_amdgcn_raw_buffer_store_b16((uint16_t)v, r, at, 0, 0); }
__device__ __forceinline__ void store_pair(float a, float b, __amdgpu_buffer_rsrc_t r, uint32_t at) {
  const v2i_t two = {__float_as_int(a), __float_as_int(b)};
  __builtin_amdgcn_raw_buffer_store_b64(two, r, at, 0, STORE_WT);
}
// Values of rows a (low half) and b of this lane's column and its neighbour's -> the even lane both columns of row a, the odd one of row b
__device__ __forceinline__ uint32_t pair_columns(uint32_t mine, bool odd) {
  const uint32_t other = (uint32_t)__builtin_amdgcn_mov_dpp((int)mine, 0xB1 /* quad_perm [1,0,3,2] */, 0xf, 0xf, true);
  return __builtin_amdgcn_perm(other, mine, odd ? 0x03020706u : 0x05040100u);
}

struct WalkTile {
  int e, first, end, n0;  // rows first .. end - 1 (end of the expert's rows) by columns from n0 (SwiGLU: of h)
};

template <class S, int OUT, bool SWI>
__global__ __launch_bounds__(GW_THREADS) void grouped_walk_kernel(GroupedArgs p, int tiles_n, UDiv by_tiles_n) {
#ifdef __HIP_DEVICE_COMPILE__  // (the host pass drops a kernel in whose generic lambdas it finds the device's operations)
  __shared__ __attribute__((aligned(1024))) uint8_t smem[S::LDS];
  constexpr int BK = GW_BK, BN = S::BN, TM = S::TM, TN = S::TN, A_LOADS = GW_BM / 64, B_LOADS = BN / 64, NLOADS = A_LOADS + B_LOADS, NKS = 4;
  constexpr int NST = S::NST, AHEAD = NST - 1;     // a step requests the stage that many steps on
  constexpr int BEHIND = (NST - 2) * NLOADS;       // loads behind the next stage's when a step ends
  static_assert(!SWI || TN == 2, "up and gate in one lane");
  constexpr int V = SWI || TN == 1 ? 1 : 2;  // neighbouring outputs of a lane
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wave_m = wave / S::WN, wave_n = wave % S::WN;
  const int K = p.K, N = p.N, FH = SWI ? N / 2 : N;
  const int steps = (K + BK - 1) / BK, nk = steps < 2 * AHEAD ? 2 * AHEAD : steps;  // (steps past K are of zeros)
  const int col = lane & 31, rq = (lane >> 5) * 4;
  float* const sx_lds = reinterpret_cast<float*>(smem + S::SX) + wave * 64;
  int32_t* const tok_lds = reinterpret_cast<int32_t*>(smem + S::TOK);
  int32_t* const off = reinterpret_cast<int32_t*>(smem + S::OFF);

  GroupTiles<GW_BM> tiles;
  tiles.init(p, off, tid, GW_THREADS);
  const int count = tiles.count(tiles_n);
  int id = blockIdx.x;
  if (id >= count) return;

  auto locate = [&](int pid) {
    // a contiguous run of tiles per XCD, to which workgroup ids are dealt round-robin
    const int share = count / NUM_XCD, rest = count % NUM_XCD, xcd = pid % NUM_XCD;
    const int t = xcd * share + (xcd < rest ? xcd : rest) + pid / NUM_XCD;
    const int q = (int)by_tiles_n((uint32_t)t);  // tiles of rows before it, of experts before its own for sure
    const auto expert = tiles.find(q, lane);
    const int rem = t - expert.before * tiles_n;
    const int group_sz = GW_GROUP * tiles_n, group = rem / group_sz, first_m = group * GW_GROUP;
    const int gm = expert.tiles - first_m < GW_GROUP ? expert.tiles - first_m : GW_GROUP, in_group = rem - group * group_sz;
    const int n_at = in_group / gm;
    WalkTile w;
    w.e = __builtin_amdgcn_readfirstlane(expert.e);
    w.first = __builtin_amdgcn_readfirstlane(off[w.e] + (first_m + in_group - n_at * gm) * GW_BM);
    w.end = __builtin_amdgcn_readfirstlane(off[w.e + 1]);
    w.n0 = __builtin_amdgcn_readfirstlane(n_at * (SWI ? BN / 2 : BN));
    return w;
  };

  const __amdgpu_buffer_rsrc_t Ar = make_rsrc(p.x, (uint32_t)p.x_rows * (uint32_t)K), Sr = make_rsrc(p.sx, (uint32_t)p.x_rows * 4u);
  const bool gather = p.tokens != nullptr;
  __amdgpu_buffer_rsrc_t Br = make_rsrc(p.w, 0);

  // A load instruction of a wavefront fills 1 KiB = 8 rows of a stage; the 16-byte pieces of a row are permuted as in gemm_kernel: piece c of
  // row r at slot c ^ (r / 2 % 8).
  const int ld_row = wave * 8 + lane / 8;  // + 64 i
  const int ld_piece = ((lane % 8) ^ (ld_row / 2 % 8)) * 16;
  uint32_t vo[NLOADS];
  // The token of row r of a tile, -1: none (its codes and its scale are zeros).
  auto token = [&](const WalkTile& t, int r) {
    const int row = t.first + r;
    const int tok = gather ? tok_lds[r] : row;
    return row < t.end && tok >= 0 && tok < p.x_rows ? tok : -1;
  };
  // Rows of weights in a stage: a wavefront's 64 columns are 32 of up and the same 32 of gate (SwiGLU), or pairs of neighbours, column 2 c + j behind
  // accumulator j of lane c, so that a row's 32 lanes store whole lines.
  auto aim = [&](const WalkTile& t) {
    Br = make_rsrc(p.w + t.e * p.w_bytes, (uint32_t)p.w_bytes);
#pragma unroll
    for (int i = 0; i < A_LOADS; ++i) {
      const int tok = token(t, ld_row + 64 * i);
      vo[i] = tok >= 0 ? (uint32_t)tok * (uint32_t)K + (uint32_t)ld_piece : OOB_OFFSET;
    }
    const int j = TN == 2 ? ld_row / 32 : 0, c = TN == 2 ? ld_row % 32 : ld_row;
#pragma unroll
    for (int i = 0; i < B_LOADS; ++i) {
      const int h = t.n0 + (SWI ? i * 32 + c : i * 64 + V * c + (V == 2 ? j : 0));
      vo[A_LOADS + i] = h < FH ? (uint32_t)(SWI ? j * FH + h : h) * (uint32_t)K + (uint32_t)ld_piece : OOB_OFFSET;
    }
  };
  auto issue_load = [&](int k0, int buf, int idx) {  // pieces past K: outside the descriptor, zeros in LDS
    uint8_t* st = smem + buf * S::STAGE + wave * 1024;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(idx < A_LOADS ? Ar : Br,
                                             (lds_void*)(st + (idx < A_LOADS ? idx * 8192 : GW_BM * BK + (idx - A_LOADS) * 8192)), 16,
                                             k0 + ld_piece < K ? vo[idx] : OOB_OFFSET, k0, 0, 0);
  };

  v16i acc[TM][TN];
  v4i af[2][TM], bf[2][TN];
  // Tiles of up to 64 rows, where wavefronts have 64: the first 32 of them are the tile's, half the products.
  auto is_short = [&](const WalkTile& t) { return TM == 2 && t.end - t.first <= 64; };
  auto first_row = [&](const WalkTile& t) { return wave_m * (is_short(t) ? 32 : 32 * TM); };  // of this wavefront's
  auto fragments_of = [&](const WalkTile& t) { return (first_row(t) + col) * BK; };
  int fr_a = 0;
  const int fr_b = GW_BM * BK + (wave_n * 32 * TN + col) * BK;
  const int swz = ((lane >> 5) ^ (col / 2 % 8)) << 4;
  auto load_frag = [&](const uint8_t* st, int ks, int f, v4i (&a)[TM], v4i (&b)[TN]) {
    const bool is_a = f == 0 || f > TN;  // in the order the products need them: A0, B0, B1, A1
    const int idx = f == 0 ? 0 : f <= TN ? f - 1 : f - TN;
    const v4i v = *reinterpret_cast<const v4i*>(st + (is_a ? fr_a : fr_b) + idx * 32 * BK + (((ks * 2) << 4) ^ swz));
    if (is_a) a[idx] = v;
    else b[idx] = v;
  };
  // One sub-step: its products, the next sub-step's fragment reads and the loads [LD0, LD1) of the requested stage between them
  auto slot = [&](auto tm_c, auto cur_c, const uint8_t* st_next, int ks_next, int k_ld, int b_ld, auto lo_c, auto hi_c) {
    constexpr int CUR = decltype(cur_c)::value, LD0 = decltype(lo_c)::value, NLD = decltype(hi_c)::value - LD0;
    constexpr int NMMA = decltype(tm_c)::value * TN, NFR = TM + TN;
#pragma unroll
    for (int m = 0; m < NMMA; ++m) {
      acc[m / TN][m % TN] = mma<false>(af[CUR][m / TN], bf[CUR][m % TN], acc[m / TN][m % TN]);
#pragma unroll
      for (int f = (m * NFR) / NMMA; f < ((m + 1) * NFR) / NMMA; ++f) load_frag(st_next, ks_next, f, af[CUR ^ 1], bf[CUR ^ 1]);
#pragma unroll
      for (int q = (m * NLD) / NMMA; q < ((m + 1) * NLD) / NMMA; ++q) issue_load(k_ld, b_ld, LD0 + q);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  using c0 = std::integral_constant<int, 0>;
  using c1 = std::integral_constant<int, 1>;
  using c2 = std::integral_constant<int, 2>;
  using l1 = std::integral_constant<int, NLOADS / 3>;
  using l2 = std::integral_constant<int, NLOADS * 2 / 3>;
  using all = std::integral_constant<int, NLOADS>;
  int b_cur = 0;  // buffer of the current stage
  // A K step of a tile with TMV accumulator rows: its first fragments are in af[0].  Requests the stage AHEAD steps on into the buffer that the
  // step before left, and waits for the next one: `behind` says how.
  auto step = [&](auto tm_c, int k_ld, auto&& behind) {
    const int b_next = b_cur == NST - 1 ? 0 : b_cur + 1, b_prev = b_cur == 0 ? NST - 1 : b_cur - 1;
    const uint8_t *st = smem + b_cur * S::STAGE, *st_next = smem + b_next * S::STAGE;
    slot(tm_c, c0{}, st, 1, k_ld, b_prev, c0{}, l1{});
    slot(tm_c, c1{}, st, 2, k_ld, b_prev, l1{}, l2{});
    slot(tm_c, c0{}, st, 3, k_ld, b_prev, l2{}, all{});
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the last fragments of the stage are in registers
    behind();                            // the next stage has landed
    AQ_BARRIER();
    slot(tm_c, c1{}, st_next, 0, k_ld, b_cur, all{}, all{});
    b_cur = b_next;
  };
  static_assert(NKS == 4, "four sub-steps");
  auto landed = [&]() { AQ_WAIT_VMCNT(BEHIND); };  // nothing behind the next stage's loads but the later stages'

  WalkTile now = locate(id);
  if (gather) {
    if (tid < GW_BM) tok_lds[tid] = now.first + tid < now.end ? p.tokens[now.first + tid] : -1;
    __syncthreads();
  }
  aim(now);
  fr_a = fragments_of(now);
  int my_tok = token(now, first_row(now) + (lane & (32 * TM - 1)));  // of the row whose scale this lane fetches
#pragma unroll
  for (int s = 0; s < AHEAD; ++s)
#pragma unroll
    for (int q = 0; q < NLOADS; ++q) issue_load(s * BK, s, q);
  __builtin_amdgcn_s_waitcnt(0xc07f);  // the tokens are read: the next tile's may come
  AQ_WAIT_VMCNT(BEHIND);               // stage 0 has landed
  AQ_BARRIER();
#pragma unroll
  for (int f = 0; f < TM + TN; ++f) load_frag(smem, 0, f, af[0], bf[0]);

  constexpr int ESZ = OUT == OUT_BF16 ? 2 : 4;
  constexpr int ROW_STORES = V == 1 && OUT == OUT_BF16 ? 8 : 16;  // of an accumulator row, per lane, at least
  const __amdgpu_buffer_rsrc_t Tr = make_rsrc(p.tokens, gather ? (uint32_t)p.R * 4u : 0u);
  int stores = 0;  // accumulator rows that the tile before stored
  auto tile = [&](auto tm_c) {  // false: it was the last
    constexpr int TMV = decltype(tm_c)::value;
#pragma unroll
    for (int i = 0; i < TMV; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    id += gridDim.x;
    const bool last = id >= count;
    WalkTile next = now;
    if (!last) next = locate(id);
    // its tokens, 16 rows to a wavefront (one operation of each, counted below); they are there before step AHEAD
    if (lane < 16)
      fetch_dword_to_lds(Tr, tok_lds + wave * 16, (uint32_t)(next.first + wave * 16 + lane) * 4u);
    int k0 = AHEAD * BK;
#pragma unroll
    for (int s = 0; s < NST - 2; ++s, k0 += BK)
      step(tm_c, k0, [&]() {  // behind the next stage's loads: the stores of the tile before and the tokens, too
        if (stores == 2) AQ_WAIT_VMCNT(BEHIND + 1 + 2 * ROW_STORES);
        else if (stores == 1) AQ_WAIT_VMCNT(BEHIND + 1 + ROW_STORES);
        else AQ_WAIT_VMCNT(BEHIND + 1);
      });
    for (int s = NST - 2; s < nk - AHEAD; ++s, k0 += BK) step(tm_c, k0, landed);
    // the epilogue's operands, then the next tile's first stages
    const int mw = now.first + first_row(now), nt = now.n0, end = now.end;
    const int64_t scales = (int64_t)now.e * N;
    auto my_column = [&](int j) { return nt + (V == 2 ? wave_n * 64 + 2 * col + j : wave_n * 32 + col); };  // of h or y
    float swn[TN], bn[TN];
    const __amdgpu_buffer_rsrc_t Wr = make_rsrc(p.sw + scales, (uint32_t)N * 4u);
    if (lane < 32 * TM)
      fetch_dword_to_lds(Sr, sx_lds, my_tok >= 0 ? (uint32_t)my_tok * 4u : OOB_OFFSET);
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int c = my_column(j);
      swn[j] = __uint_as_float(load_dword(Wr, c < FH ? (uint32_t)(SWI ? j * FH + c : c) * 4u : OOB_OFFSET));
    }
    [[maybe_unused]] uint32_t braw[TN];
    const bool has_bias = !SWI && p.bias != nullptr, bias_bf16 = p.bias_dtype == AQ_BF16;
    if constexpr (!SWI) {
      const uint32_t bsz = bias_bf16 ? 2u : 4u;
      const __amdgpu_buffer_rsrc_t Bsr = make_rsrc(has_bias ? static_cast<const uint8_t*>(p.bias) + scales * bsz : (const uint8_t*)p.sw, has_bias ? (uint32_t)N * bsz : 0u);
#pragma unroll
      for (int j = 0; j < TN; ++j)
        braw[j] = bias_bf16 ? load_word(Bsr, (uint32_t)my_column(j) * 2u) : load_dword(Bsr, (uint32_t)my_column(j) * 4u);
    }
    asm volatile("" ::: "memory");
    int next_fr_a = fr_a;
    if (!last) {
      now = next;
      aim(now);
      next_fr_a = fragments_of(now);
      my_tok = token(now, first_row(now) + (lane & (32 * TM - 1)));
    } else {  // nothing: loads outside the descriptors touch no memory
#pragma unroll
      for (int i = 0; i < NLOADS; ++i) vo[i] = OOB_OFFSET;
    }
#pragma unroll
    for (int s = 0; s < AHEAD - 1; ++s) step(tm_c, s * BK, landed);
    step(tm_c, (AHEAD - 1) * BK, [&]() {
      landed();
      fr_a = next_fr_a;  // (the fragments read behind this step's barrier are the next tile's)
    });
    asm volatile("" ::: "memory");

    // ---- epilogue: three rounded operations, then bf16 rows of neighbouring columns a dword a lane
    const uint32_t rowb = (uint32_t)FH * ESZ;
    const int rows = end - mw < 32 * TMV ? end - mw : 32 * TMV;
    const uint32_t window = rows > 0 ? (uint32_t)rows * rowb - (uint32_t)nt * ESZ : 0u;
    const __amdgpu_buffer_rsrc_t Cr =
        make_rsrc(static_cast<uint8_t*>(p.y) + (rows > 0 ? ((int64_t)mw * FH + nt) * ESZ : 0), window);
#pragma unroll
    for (int j = 0; j < TN; ++j) bn[j] = !has_bias ? 0.0f : bias_bf16 ? bf16_bits_to_f32(braw[j]) : __uint_as_float(braw[j]);
    const bool odd = lane & 1, even_n = SWI || (N & 1) == 0;
    const uint32_t c = (uint32_t)(my_column(0) - nt);
    uint32_t at = OOB_OFFSET, at1 = OOB_OFFSET;  // at1: an odd N's second column, by itself
    if (my_column(0) < FH) at = (uint32_t)rq * rowb + (V == 1 && OUT == OUT_BF16 && even_n ? (c & ~1u) * 2 + (odd ? rowb : 0u) : c * ESZ);
    if (V == 2 && my_column(1) < FH) at1 = (uint32_t)rq * rowb + (c + 1) * ESZ;
#pragma unroll
    for (int i = 0; i < TMV; ++i) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int r0 = i * 32 + g * 8;
        const v4f sxq = *reinterpret_cast<const v4f*>(sx_lds + r0 + rq);
        float y[TN][4], o[V][4];
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            y[j][q] = __fmul_rn(__fmul_rn((float)acc[i][j][g * 4 + q], sxq[q]), swn[j]);
            if constexpr (!SWI) y[j][q] = has_bias ? __fadd_rn(y[j][q], bn[j]) : y[j][q];
          }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if constexpr (SWI) o[0][q] = grouped_swiglu<OUT>(y[0][q], y[1][q]);
          else
#pragma unroll
            for (int v = 0; v < V; ++v) o[v][q] = y[v][q];
        }
        if constexpr (V == 1 && OUT == OUT_F32) {
#pragma unroll
          for (int q = 0; q < 4; ++q) store_dword(__float_as_uint(o[0][q]), Cr, at + (r0 + q) * rowb);
        } else if constexpr (V == 1) {
          if (even_n) {
#pragma unroll
            for (int h = 0; h < 2; ++h) store_dword(pair_columns(pack_bf16x2(o[0][2 * h], o[0][2 * h + 1]), odd), Cr, at + (r0 + 2 * h) * rowb);
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) store_word(f32_to_bf16_bits(o[0][q]), Cr, at + (r0 + q) * rowb);
          }
        } else if (even_n) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if constexpr (OUT == OUT_F32) store_pair(o[0][q], o[V - 1][q], Cr, at + (r0 + q) * rowb);
            else store_dword(pack_bf16x2(o[0][q], o[V - 1][q]), Cr, at + (r0 + q) * rowb);
          }
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if constexpr (OUT == OUT_F32) {
              store_dword<0>(__float_as_uint(o[0][q]), Cr, at + (r0 + q) * rowb);
              store_dword<0>(__float_as_uint(o[V - 1][q]), Cr, at1 + (r0 + q) * rowb);
            } else {
              store_word(f32_to_bf16_bits(o[0][q]), Cr, at + (r0 + q) * rowb);
              store_word(f32_to_bf16_bits(o[V - 1][q]), Cr, at1 + (r0 + q) * rowb);
            }
          }
        }
      }
    }
    stores = TMV;
    return !last;
  };
  if constexpr (TM == 2) {
    while (is_short(now) ? tile(c1{}) : tile(c2{})) {}
  } else {
    while (tile(c1{})) {}
  }
  AQ_WAIT_VMCNT(0);  // nothing lands in LDS behind the walk
  AQ_BARRIER();
#endif
}

template <class S, int OUT, bool SWI>
static int walk_launch(const GroupedArgs& a, hipStream_t st) {
  const int tiles_n = (a.N + S::BN - 1) / S::BN;
  const int64_t most = grouped_most_tiles(a.R, a.E, GW_BM) * tiles_n;
  if (most > 0x7fffffff) return AQ_E_RANGE;
  const int cus = device_cus();
  queue_kernel(grouped_walk_kernel<S, OUT, SWI>, dim3((unsigned)(most < cus ? most : cus)), dim3(GW_THREADS), 0, st, a, tiles_n,
               UDiv::of((uint32_t)tiles_n));
  return (int)hipGetLastError();
}
template <int OUT, bool SWI>
int grouped_walk_launch(const GroupedArgs& a, int width, hipStream_t st) {
  if (width == 256) return walk_launch<GroupedShape<2, 2, 3>, OUT, SWI>(a, st);
  if constexpr (!SWI)
    if (width == 64) return walk_launch<GroupedShape<4, 1, 6>, OUT, SWI>(a, st);
  return walk_launch<GroupedShape<4, 2, 4>, OUT, SWI>(a, st);
}
template int grouped_walk_launch<OUT_BF16, false>(const GroupedArgs&, int, hipStream_t);
template int grouped_walk_launch<OUT_F32, false>(const GroupedArgs&, int, hipStream_t);
template int grouped_walk_launch<OUT_BF16, true>(const GroupedArgs&, int, hipStream_t);
template int grouped_walk_launch<OUT_F32, true>(const GroupedArgs&, int, hipStream_t);

}  // namespace aq
