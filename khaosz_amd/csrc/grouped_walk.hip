// Grouped products of many rows an expert: tiles of 128 rows x 256 weight rows, walked by one workgroup per compute unit whose K loop does not stop
// between them (as gemm_walk.hip walks the tiles of a single Linear).
//
// Inside an expert tiles go in groups of 8 by rows, then by columns: the 32 tiles that an XCD works on at a time share 2 MB of rows and 2 MB of
// weights.  The rows' tokens of the next tile are fetched into LDS under this tile's first step, for its first stages are requested in the
// last steps.
//
// What bounds it, and what was measured.  Many rows an expert: the clock that power leaves and, of its cycles, the loads (48000 rows of 64 experts, 1408 ->
// 2048: 171 us, 1.6 POP/s of the 2.36 that torch's product of 8192 x 8192 x 8192 reaches on this card; 1.64 GHz of 2.4, the matrix core at work in 51 % of the
// cycles; on codes of zeros, the same instructions and bytes, 145; without its stores 148, with loads that all hit the L2 147).  A few dozen rows: the weights (96 of 60
// experts, SwiGLU of 2048 -> 1408: 280 MB in 50 us, 5.6 TB/s, the launch included).  A few hundred: both (12000 of 64 experts, SwiGLU of 1536 -> 1408: 342 MB in 94 us,
// 1.1 POP/s, the matrix core 38 % of the cycles; on zeros 88).  A ragged last round is left as it is: its tiles' columns dealt out
// to two or four workgroups each take as many K steps (500 tokens' 2 of 8, SwiGLU: 73 us, 79 that way).
#include "aq_grouped.h"

namespace aq {

typedef int v2i_t __attribute__((ext_vector_type(2)));

constexpr int GW_BM = 128, GW_BK = 128, GW_THREADS = 512, GW_GROUP = 8;

// WM x WN wavefronts, each 32 TM rows by 32 TN weight rows of a tile of 128 x BN, K steps through NST stages.
template <int WM_, int TN_, int NST_>
struct GroupedShape {
  static constexpr int WM = WM_, WN = 8 / WM_, TM = 4 / WM_, TN = TN_, BN = 32 * TN * WN, NST = NST_;
  static constexpr int STAGE = (GW_BM + BN) * GW_BK;
  static constexpr int SX = NST * STAGE, TOK = SX + 2 * 8 * 64 * 4, OFF = TOK + GW_BM * 4, LDS = OFF + (GP_MAX_E + 1) * 4;
  static_assert(LDS <= 160 * 1024, "LDS of one compute unit");
  static_assert(NST >= 3, "a stage in use, one that lands, one on its way");
};

__device__ __forceinline__ void fetch_dword_to_lds(__amdgpu_buffer_rsrc_t r, void* to, uint32_t at) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)to, 4, at, 0, 0, 0);
}
__device__ __forceinline__ uint32_t load_dword(__amdgpu_buffer_rsrc_t r, uint32_t at) { return (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, (int)at, 0, 0); }
__device__ __forceinline__ uint32_t load_word(__amdgpu_buffer_rsrc_t r, uint32_t at) { return (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(r, (int)at, 0, 0); }
template <int POLICY>
__device__ __forceinline__ void store_dword(uint32_t v, __amdgpu_buffer_rsrc_t r, uint32_t at) { __builtin_amdgcn_raw_buffer_store_b32(v, r, at, 0, POLICY); }
__device__ __forceinline__ void store_word(uint32_t v, __amdgpu_buffer_rsrc_t r, uint32_t at) { __builtin_amdgcn_raw_buffer_store_b16((uint16_t)v, r, at, 0, 0); }
template <int POLICY>
__device__ __forceinline__ void store_pair(float a, float b, __amdgpu_buffer_rsrc_t r, uint32_t at) {
  const v2i_t two = {__float_as_int(a), __float_as_int(b)};
  __builtin_amdgcn_raw_buffer_store_b64(two, r, at, 0, POLICY);
}
// Values of rows a (low half) and b of this lane's column and its neighbour's -> the even lane both columns of row a, the odd one of row b
__device__ __forceinline__ uint32_t pair_columns(uint32_t mine, bool odd) {
  const uint32_t other = (uint32_t)__builtin_amdgcn_mov_dpp((int)mine, 0xB1 /* quad_perm [1,0,3,2] */, 0xf, 0xf, true);
  return __builtin_amdgcn_perm(other, mine, odd ? 0x03020706u : 0x05040100u);
}

struct WalkTile {
  int e, first, end, n0;  // rows first .. end - 1 (end of the expert's rows) by columns from n0 (SwiGLU: of h)
  int rot;                // the K step it begins with
};

// Rows of the output: whole 128-byte lines, whole dwords (with bf16: an even number), or neither.  Parts of lines stay in the L2 until the rest is there;
// written through, they go to memory by themselves (43000 rows of 608 -> 3060: 191 us, 244 written through; whole lines 1 % faster written through
// where the next launch reads them, 4096 tokens' 6 of 64 320.6 and 322.2).
enum { ROWS_LINES, ROWS_DWORDS, ROWS_ODD };

template <class S, int OUT, bool SWI, int ROWS>
__global__ __launch_bounds__(GW_THREADS) void grouped_walk_kernel(GroupedArgs p, int tiles_n, UDiv by_tiles_n) {
#ifdef __HIP_DEVICE_COMPILE__  // (the host pass drops a kernel in whose generic lambdas it finds the device's operations)
  __shared__ __attribute__((aligned(1024))) uint8_t smem[S::LDS];
  constexpr int BK = GW_BK, BN = S::BN, TM = S::TM, TN = S::TN, A_LOADS = GW_BM / 64, B_LOADS = BN / 64, NLOADS = A_LOADS + B_LOADS, NKS = 4;
  constexpr int NST = S::NST, AHEAD = NST - 1;     // a step requests the stage that many steps on
  constexpr int BEHIND = (NST - 2) * NLOADS;       // loads behind the next stage's when a step ends
  static_assert(!SWI || TN == 2, "up and gate in one lane");
  constexpr int V = SWI || TN == 1 ? 1 : 2;  // neighbouring outputs of a lane
  constexpr int ESZ = OUT == OUT_BF16 ? 2 : 4;
  constexpr int EPI = 4;                     // steps that finish the tile before
  constexpr bool ODD = ROWS == ROWS_ODD;
  constexpr int POLICY = ROWS == ROWS_LINES ? STORE_WT : 0;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wave_m = wave / S::WN, wave_n = wave % S::WN;
  const int K = p.K, N = p.N, FH = SWI ? N / 2 : N;
  const int steps = (K + BK - 1) / BK, least = EPI + AHEAD > 2 * AHEAD ? EPI + AHEAD : 2 * AHEAD;
  const int nk = steps < least ? least : steps;  // (steps past K are of zeros)
  const int col = lane & 31, rq = (lane >> 5) * 4;
  float* sx_lds = reinterpret_cast<float*>(smem + S::SX) + wave * 128;  // row scales of this wavefront, of this tile ..
  float* sx_done = sx_lds + 64;                                         // .. and of the one before
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
    w.rot = __builtin_amdgcn_readfirstlane((in_group % gm + n_at) % 8 * steps / 8);
    return w;
  };
  // K step s of a tile.  Tiles beside each other begin at different steps: what they share is then brought by one of them at a time and found in the L2 by the
  // others, where all of them in step would wait for each line's way from memory.
  auto k_of = [&](int s, const WalkTile& t) {
    const int k = s + t.rot;
    return (s >= steps ? steps : k >= steps ? k - steps : k) * BK;
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
  // The tile before, as its sums and what finishes them: every step of the first EPI has two or four of its rows' outputs between its products
  // (finished in one go, with the matrix core idle, they took a quarter of the time at K = 1408: 48000 rows of 1408 -> 2048 182 us).  Rows that it did
  // not have fall outside the window.
  struct Done {
    v16i acc[TM][TN];
    float sw[TN], bias[TN];
    __amdgpu_buffer_rsrc_t out;
    uint32_t at, at1;  // at1: an odd N's second column, by itself
  };
  Done done;
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = done.acc[i][j][r] = 0;
#pragma unroll
  for (int j = 0; j < TN; ++j) done.sw[j] = done.bias[j] = 0.0f;
  done.out = make_rsrc(p.y, 0);
  done.at = done.at1 = OOB_OFFSET;
  const uint32_t rowb = (uint32_t)FH * ESZ;
  const bool odd_lane = lane & 1;
  constexpr int ROW_STORES = V == 1 && OUT == OUT_BF16 && !ODD ? 2 : V == 2 && ODD ? 8 : 4;  // of four rows, per lane
  v4f sxq;
  float held = 0.0f;
  // row q of the four rows 8 g + rq .. of accumulator row i: three rounded operations; bf16 neighbours go as a dword
  auto finish = [&](int i, int g, int q) {
    const int r0 = i * 32 + g * 8;
    if (q == 0) sxq = *reinterpret_cast<const v4f*>(sx_done + r0 + rq);
    float y[TN], o[V];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      y[j] = __fmul_rn(__fmul_rn((float)done.acc[i][j][g * 4 + q], sxq[q]), done.sw[j]);
      if constexpr (!SWI) y[j] = __fadd_rn(y[j], done.bias[j]);
    }
    if constexpr (SWI) {
      o[0] = grouped_swiglu<OUT>(y[0], y[1]);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) o[v] = y[v];
    }
    const uint32_t at = done.at + (r0 + q) * rowb;
    if constexpr (V == 2 && ODD) {
      const uint32_t at1 = done.at1 + (r0 + q) * rowb;
      if constexpr (OUT == OUT_F32) {
        store_dword<POLICY>(__float_as_uint(o[0]), done.out, at);
        store_dword<POLICY>(__float_as_uint(o[V - 1]), done.out, at1);
      } else {
        store_word(f32_to_bf16_bits(o[0]), done.out, at);
        store_word(f32_to_bf16_bits(o[V - 1]), done.out, at1);
      }
    } else if constexpr (V == 2) {
      if constexpr (OUT == OUT_F32) store_pair<POLICY>(o[0], o[V - 1], done.out, at);
      else store_dword<POLICY>(pack_bf16x2(o[0], o[V - 1]), done.out, at);
    } else if constexpr (OUT == OUT_F32) {
      store_dword<POLICY>(__float_as_uint(o[0]), done.out, at);
    } else if constexpr (ODD) {
      store_word(f32_to_bf16_bits(o[0]), done.out, at);
    } else {  // two rows of two neighbouring lanes
      if (q & 1) store_dword<POLICY>(pair_columns(pack_bf16x2(held, o[0]), odd_lane), done.out, at - rowb);
      held = o[0];
    }
  };
  // One sub-step: its products (FIRST: of a tile), the next sub-step's fragment reads and the loads [LD0, LD1) of the requested stage between them,
  // and, with ROW >= 0, four rows (part `g`) of accumulator row ROW of the tile before.
  auto slot = [&](auto tm_c, auto first_c, auto row_c, int g, auto cur_c, const uint8_t* st_next, int ks_next, int k_ld, int b_ld, auto lo_c, auto hi_c) {
    constexpr int CUR = decltype(cur_c)::value, LD0 = decltype(lo_c)::value, NLD = decltype(hi_c)::value - LD0, ROW = decltype(row_c)::value;
    constexpr int NMMA = decltype(tm_c)::value * TN, NFR = TM + TN;
#pragma unroll
    for (int m = 0; m < NMMA; ++m) {
      v16i c = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
      if constexpr (!decltype(first_c)::value) c = acc[m / TN][m % TN];
      acc[m / TN][m % TN] = mma<false>(af[CUR][m / TN], bf[CUR][m % TN], c);
#pragma unroll
      for (int f = (m * NFR) / NMMA; f < ((m + 1) * NFR) / NMMA; ++f) load_frag(st_next, ks_next, f, af[CUR ^ 1], bf[CUR ^ 1]);
#pragma unroll
      for (int q = (m * NLD) / NMMA; q < ((m + 1) * NLD) / NMMA; ++q) issue_load(k_ld, b_ld, LD0 + q);
      if constexpr (ROW >= 0) {
#pragma unroll
        for (int q = (m * 4) / NMMA; q < ((m + 1) * 4) / NMMA; ++q) finish(ROW, g, q);
      }
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
  using no = std::false_type;
  using none = std::integral_constant<int, -1>;
  // A K step of a tile with TMV accumulator rows: its first fragments are in af[0].  Requests the stage AHEAD steps on into the buffer that the
  // step before left, and waits for the next one: `behind` says how.  FIRST: of the tile.  DONE: part `g` of the tile before is finished in it.
  auto step = [&](auto tm_c, auto first_c, auto done_c, int g, int k_ld, auto&& behind) {
    constexpr bool DONE = decltype(done_c)::value;
    using row0 = std::integral_constant<int, DONE ? 0 : -1>;
    using row1 = std::integral_constant<int, DONE && TM == 2 ? 1 : -1>;
    const int b_next = b_cur == NST - 1 ? 0 : b_cur + 1, b_prev = b_cur == 0 ? NST - 1 : b_cur - 1;
    const uint8_t *st = smem + b_cur * S::STAGE, *st_next = smem + b_next * S::STAGE;
    slot(tm_c, first_c, row0{}, g, c0{}, st, 1, k_ld, b_prev, c0{}, l1{});
    slot(tm_c, no{}, none{}, g, c1{}, st, 2, k_ld, b_prev, l1{}, l2{});
    slot(tm_c, no{}, row1{}, g, c0{}, st, 3, k_ld, b_prev, l2{}, all{});
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the last fragments of the stage are in registers
    behind();                            // the next stage has landed
    AQ_BARRIER();
    slot(tm_c, no{}, none{}, g, c1{}, st_next, 0, k_ld, b_cur, all{}, all{});
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
    for (int q = 0; q < NLOADS; ++q) issue_load(k_of(s, now), s, q);
  __builtin_amdgcn_s_waitcnt(0xc07f);  // the tokens are read: the next tile's may come
  AQ_WAIT_VMCNT(BEHIND);               // stage 0 has landed
  AQ_BARRIER();
#pragma unroll
  for (int f = 0; f < TM + TN; ++f) load_frag(smem, 0, f, af[0], bf[0]);

  const __amdgpu_buffer_rsrc_t Tr = make_rsrc(p.tokens, gather ? (uint32_t)p.R * 4u : 0u);
  auto tile = [&](auto tm_c) {  // false: it was the last
    constexpr int TMV = decltype(tm_c)::value;
    id += gridDim.x;
    const bool last = id >= count;
    WalkTile next = now;
    if (!last) next = locate(id);
    // its tokens, 16 rows to a wavefront (one operation of each, counted below); they are there before step AHEAD
    if (lane < 16)
      fetch_dword_to_lds(Tr, tok_lds + wave * 16, (uint32_t)(next.first + wave * 16 + lane) * 4u);
    // behind the next stage's loads: the step's stores, and in the first step the tokens
    step(tm_c, std::true_type{}, std::true_type{}, 0, k_of(AHEAD, now), [&]() { AQ_WAIT_VMCNT(BEHIND + 1 + TM * ROW_STORES); });
#pragma unroll
    for (int g = 1; g < EPI; ++g) step(tm_c, no{}, std::true_type{}, g, k_of(AHEAD + g, now), [&]() { AQ_WAIT_VMCNT(BEHIND + TM * ROW_STORES); });
    for (int s = EPI; s < nk - AHEAD; ++s) step(tm_c, no{}, no{}, 0, k_of(AHEAD + s, now), landed);
    // the epilogue's operands, then the next tile's first stages
    const int mw = now.first + first_row(now), nt = now.n0, end = now.end;
    const int64_t scales = (int64_t)now.e * N;
    auto my_column = [&](int j) { return nt + (V == 2 ? wave_n * 64 + 2 * col + j : wave_n * 32 + col); };  // of h or y
    float swn[TN];
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
    for (int s = 0; s < AHEAD - 1; ++s) step(tm_c, no{}, no{}, 0, k_of(s, now), landed);
    step(tm_c, no{}, no{}, 0, k_of(AHEAD - 1, now), [&]() {
      landed();
      fr_a = next_fr_a;  // (the fragments read behind this step's barrier are the next tile's)
    });
    asm volatile("" ::: "memory");

    // what finishes it, under the next tile's first steps
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) done.acc[i][j] = acc[i][j];
    const int rows = end - mw < 32 * TMV ? end - mw : 32 * TMV;
    const uint32_t window = rows > 0 ? (uint32_t)rows * rowb - (uint32_t)nt * ESZ : 0u;
    done.out = make_rsrc(static_cast<uint8_t*>(p.y) + (rows > 0 ? ((int64_t)mw * FH + nt) * ESZ : 0), window);
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      done.sw[j] = swn[j];
      if constexpr (!SWI) done.bias[j] = !has_bias ? 0.0f : bias_bf16 ? bf16_bits_to_f32(braw[j]) : __uint_as_float(braw[j]);
    }
    const uint32_t c = (uint32_t)(my_column(0) - nt);
    done.at = done.at1 = OOB_OFFSET;
    if (my_column(0) < FH)  // (two lanes' columns of two rows: the even lane has the first row of the two)
      done.at = (uint32_t)rq * rowb + (V == 1 && OUT == OUT_BF16 && !ODD ? (c & ~1u) * 2 + (odd_lane ? rowb : 0u) : c * ESZ);
    if (V == 2 && my_column(1) < FH) done.at1 = (uint32_t)rq * rowb + (c + 1) * ESZ;
    float* const other = sx_lds;
    sx_lds = sx_done;
    sx_done = other;
    return !last;
  };
  if constexpr (TM == 2) {
    while (is_short(now) ? tile(c1{}) : tile(c2{})) {}
  } else {
    while (tile(c1{})) {}
  }
#pragma unroll
  for (int g = 0; g < EPI; ++g)
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) finish(i, g, q);
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
  const dim3 grid((unsigned)(most < cus ? most : cus)), block(GW_THREADS);
  const UDiv by_tiles_n = UDiv::of((uint32_t)tiles_n);
  const bool lines = (SWI ? a.N / 2 : a.N) * (OUT == OUT_BF16 ? 2 : 4) % 128 == 0;
  if (lines) {
    queue_kernel((grouped_walk_kernel<S, OUT, SWI, ROWS_LINES>), grid, block, 0, st, a, tiles_n, by_tiles_n);
  } else if (SWI || a.N % 2 == 0) {
    queue_kernel((grouped_walk_kernel<S, OUT, SWI, ROWS_DWORDS>), grid, block, 0, st, a, tiles_n, by_tiles_n);
  } else if constexpr (!SWI) {
    queue_kernel((grouped_walk_kernel<S, OUT, SWI, ROWS_ODD>), grid, block, 0, st, a, tiles_n, by_tiles_n);
  }
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
