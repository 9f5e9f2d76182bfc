// Grouped products of many rows an expert: tiles of 128 rows x 256 weight rows, walked by one workgroup per compute unit whose K loop does not stop
// between them (as gemm_walk.hip walks the tiles of a single Linear).
//
// Every workgroup takes the offsets into LDS, and a wavefront's lanes hold the running count of tiles, so that a tile's expert is two ballots
// away.  Inside an expert tiles go in groups of 8 by rows, then by columns: the 32 tiles that an XCD works on at a time share 2 MB of rows and 2 MB of
// weights.  The rows' tokens of the next tile are fetched into LDS under this tile's first step, for its first two stages are requested in the
// last two.
#include "aq_grouped.h"

namespace aq {

typedef int v2i_t __attribute__((ext_vector_type(2)));

constexpr int GW_BM = 128, GW_BN = 256, GW_BK = 128, GW_STAGES = 3, GW_THREADS = 512, GW_GROUP = 8;
constexpr int GW_STAGE = (GW_BM + GW_BN) * GW_BK;
constexpr int GW_SX = GW_STAGES * GW_STAGE, GW_TOK = GW_SX + 8 * 64 * 4, GW_OFF = GW_TOK + GW_BM * 4, GW_LDS = GW_OFF + (GP_MAX_E + 1) * 4;
static_assert(GW_LDS <= 160 * 1024, "LDS of one compute unit");

struct WalkTile {
  int e, first, end, n0;  // rows first .. end - 1 (end of the expert's rows) by columns from n0 (SwiGLU: of h)
};

template <int OUT, bool SWI>
__global__ __launch_bounds__(GW_THREADS) void grouped_walk_kernel(GroupedArgs p, int tiles_n, UDiv by_tiles_n) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[GW_LDS];
  constexpr int BK = GW_BK, TM = 2, TN = 2, A_LOADS = 2, B_LOADS = 4, NLOADS = A_LOADS + B_LOADS, NKS = 4;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wave_m = wave >> 2, wave_n = wave & 3;
  const int K = p.K, N = p.N, FH = SWI ? N / 2 : N;
  const int steps = (K + BK - 1) / BK, nk = steps < 4 ? 4 : steps;  // (steps past K are of zeros)
  const int col = lane & 31, rq = (lane >> 5) * 4;
  float* const sx_lds = reinterpret_cast<float*>(smem + GW_SX) + wave * 64;
  int32_t* const tok_lds = reinterpret_cast<int32_t*>(smem + GW_TOK);
  int32_t* const off = reinterpret_cast<int32_t*>(smem + GW_OFF);

  for (int e = tid; e <= p.E; e += GW_THREADS) {
    const int o = p.offsets[e];
    off[e] = o < 0 ? 0 : o > p.R ? p.R : o;
  }
  __syncthreads();
  const int per = (p.E + 63) >> 6;  // experts of a lane
  auto tiles_of = [&](int e) {
    const int rows = e < p.E ? off[e + 1] - off[e] : 0;
    return rows > 0 ? (rows + GW_BM - 1) / GW_BM : 0;
  };
  int mine = 0;
  for (int i = 0; i < per; ++i) mine += tiles_of(lane * per + i);
  const int upto = wave_scan(mine);
  const int64_t all_tiles = (int64_t)__builtin_amdgcn_readlane(upto, 63) * tiles_n;  // (offsets that fall can make it more than was launched for)
  const int count = all_tiles < 0x7fffffff ? (int)all_tiles : 0x7fffffff;
  int id = blockIdx.x;
  if (id >= count) return;

  auto locate = [&](int pid) {
    // a contiguous run of tiles per XCD, to which workgroup ids are dealt round-robin
    const int share = count / NUM_XCD, rest = count % NUM_XCD, xcd = pid % NUM_XCD;
    const int t = xcd * share + (xcd < rest ? xcd : rest) + pid / NUM_XCD;
    const int q = (int)by_tiles_n((uint32_t)t);  // tiles of rows before it, of experts before its own for sure
    const int at = __builtin_ctzll(__ballot(upto > q));
    const int e0 = at * per, before = __builtin_amdgcn_readlane(upto - mine, at);
    const int n = lane < per ? tiles_of(e0 + lane) : 0;  // (per <= 8: a row of 16 lanes)
    int in = n;
    in += __builtin_amdgcn_update_dpp(0, in, 0x111, 0xf, 0xf, false);
    in += __builtin_amdgcn_update_dpp(0, in, 0x112, 0xf, 0xf, false);
    in += __builtin_amdgcn_update_dpp(0, in, 0x114, 0xf, 0xf, false);
    const int sub = __builtin_ctzll(__ballot(lane < per && before + in > q));
    const int tiles_m = __builtin_amdgcn_readlane(n, sub);
    const int rem = t - (before + __builtin_amdgcn_readlane(in, sub) - tiles_m) * tiles_n;
    const int group_sz = GW_GROUP * tiles_n, group = rem / group_sz, first_m = group * GW_GROUP;
    const int gm = tiles_m - first_m < GW_GROUP ? tiles_m - first_m : GW_GROUP, in_group = rem - group * group_sz;
    const int n_at = in_group / gm;
    WalkTile w;
    w.e = __builtin_amdgcn_readfirstlane(e0 + sub);
    w.first = __builtin_amdgcn_readfirstlane(off[w.e] + (first_m + in_group - n_at * gm) * GW_BM);
    w.end = __builtin_amdgcn_readfirstlane(off[w.e + 1]);
    w.n0 = __builtin_amdgcn_readfirstlane(n_at * (SWI ? GW_BN / 2 : GW_BN));
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
    const int j = ld_row / 32, c = ld_row % 32;
#pragma unroll
    for (int i = 0; i < B_LOADS; ++i) {
      const int h = t.n0 + (SWI ? i * 32 + c : i * 64 + 2 * c + j);
      vo[A_LOADS + i] = h < FH ? (uint32_t)(SWI ? j * FH + h : h) * (uint32_t)K + (uint32_t)ld_piece : OOB_OFFSET;
    }
  };
  auto issue_load = [&](int k0, int buf, int idx) {  // pieces past K: outside the descriptor, zeros in LDS
    uint8_t* st = smem + buf * GW_STAGE + wave * 1024;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(idx < A_LOADS ? Ar : Br,
                                             (lds_void*)(st + (idx < A_LOADS ? idx * 8192 : GW_BM * BK + (idx - A_LOADS) * 8192)), 16,
                                             k0 + ld_piece < K ? vo[idx] : OOB_OFFSET, k0, 0, 0);
  };

  v16i acc[TM][TN];
  v4i af[2][TM], bf[2][TN];
  const int fr_a = (wave_m * 32 * TM + col) * BK, fr_b = GW_BM * BK + (wave_n * 32 * TN + col) * BK;
  const int swz = ((lane >> 5) ^ (col / 2 % 8)) << 4;
  auto load_frag = [&](const uint8_t* st, int ks, int f, v4i (&a)[TM], v4i (&b)[TN]) {
    const bool is_a = f == 0 || f > TN;  // in the order the products need them: A0, B0, B1, A1
    const int idx = f == 0 ? 0 : f <= TN ? f - 1 : f - TN;
    const v4i v = *reinterpret_cast<const v4i*>(st + (is_a ? fr_a : fr_b) + idx * 32 * BK + (((ks * 2) << 4) ^ swz));
    if (is_a) a[idx] = v;
    else b[idx] = v;
  };
  // One sub-step: its products, the next sub-step's fragment reads and the loads [LD0, LD1) of the requested stage between them
  auto slot = [&](auto cur_c, const uint8_t* st_next, int ks_next, int k_ld, int b_ld, auto lo_c, auto hi_c) {
    constexpr int CUR = decltype(cur_c)::value, LD0 = decltype(lo_c)::value, NLD = decltype(hi_c)::value - LD0;
    constexpr int NMMA = TM * TN, NFR = TM + TN;
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
  using l1 = std::integral_constant<int, NLOADS / 3>;
  using l2 = std::integral_constant<int, NLOADS * 2 / 3>;
  using all = std::integral_constant<int, NLOADS>;
  int b_cur = 0;  // buffer of the current stage
  // A K step: its first fragments are in af[0].  Requests the stage two steps on into the buffer that the step before left.
  // BEHIND: vector memory operations that may be in flight behind the next stage's loads, besides this step's own loads.
  auto step = [&](int k_ld, auto behind_c) {
    constexpr int BEHIND = NLOADS + decltype(behind_c)::value;
    const int b_next = b_cur == GW_STAGES - 1 ? 0 : b_cur + 1, b_prev = b_cur == 0 ? GW_STAGES - 1 : b_cur - 1;
    const uint8_t *st = smem + b_cur * GW_STAGE, *st_next = smem + b_next * GW_STAGE;
    slot(c0{}, st, 1, k_ld, b_prev, c0{}, l1{});
    slot(c1{}, st, 2, k_ld, b_prev, l1{}, l2{});
    slot(c0{}, st, 3, k_ld, b_prev, l2{}, all{});
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the last fragments of the stage are in registers
    AQ_WAIT_VMCNT(BEHIND < 63 ? BEHIND : 63);  // the next stage has landed
    AQ_BARRIER();
    slot(c1{}, st_next, 0, k_ld, b_cur, all{}, all{});
    b_cur = b_next;
  };
  static_assert(NKS == 4, "four sub-steps");

  WalkTile now = locate(id);
  if (gather) {
    if (tid < GW_BM) tok_lds[tid] = now.first + tid < now.end ? p.tokens[now.first + tid] : -1;
    __syncthreads();
  }
  aim(now);
  int my_tok = token(now, wave_m * 64 + lane);  // of the row whose scale this lane fetches
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int q = 0; q < NLOADS; ++q) issue_load(s * BK, s, q);
  __builtin_amdgcn_s_waitcnt(0xc07f);  // the tokens are read: the next tile's may come
  AQ_WAIT_VMCNT(NLOADS);               // stage 0 has landed
  AQ_BARRIER();
#pragma unroll
  for (int f = 0; f < TM + TN; ++f) load_frag(smem, 0, f, af[0], bf[0]);

  constexpr int ESZ = OUT == OUT_BF16 ? 2 : 4;
  constexpr int STORES = SWI ? (OUT == OUT_BF16 ? 16 : 32) : 32;  // per lane and tile, at least
  const __amdgpu_buffer_rsrc_t Tr = make_rsrc(p.tokens, gather ? (uint32_t)p.R * 4u : 0u);
  for (bool first = true;; first = false) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    id += gridDim.x;
    const bool last = id >= count;
    WalkTile next = now;
    if (!last) next = locate(id);
    // its tokens, 16 rows to a wavefront (one operation of each, counted below); they are there two steps on
    if (lane < 16)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(Tr, (lds_void*)(tok_lds + wave * 16), 4, (uint32_t)(next.first + wave * 16 + lane) * 4u, 0, 0, 0);
    int k0 = 2 * BK;
    if (first)
      step(k0, c1{});
    else
      step(k0, std::integral_constant<int, STORES + 1>{});  // the stores of the tile before
    for (int s = 1; s < nk - 2; ++s) step(k0 += BK, c0{});
    // the epilogue's operands, then the next tile's first two stages
    const int mw = now.first + wave_m * 32 * TM, nt = now.n0, end = now.end;
    const int64_t scales = (int64_t)now.e * N;
    auto my_column = [&](int j) { return nt + (SWI ? wave_n * 32 + col : wave_n * 64 + 2 * col + j); };  // of h or y
    float swn[TN], bn[TN];
    const __amdgpu_buffer_rsrc_t Wr = make_rsrc(p.sw + scales, (uint32_t)N * 4u);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(Sr, (lds_void*)sx_lds, 4, my_tok >= 0 ? (uint32_t)my_tok * 4u : OOB_OFFSET, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int c = my_column(j);
      swn[j] = __uint_as_float((uint32_t)__builtin_amdgcn_raw_buffer_load_b32(Wr, c < FH ? (SWI ? j * FH + c : c) * 4 : (int)OOB_OFFSET, 0, 0));
    }
    [[maybe_unused]] uint32_t braw[TN];
    const bool has_bias = !SWI && p.bias != nullptr, bias_bf16 = p.bias_dtype == AQ_BF16;
    if constexpr (!SWI) {
      const uint32_t bsz = bias_bf16 ? 2u : 4u;
      const __amdgpu_buffer_rsrc_t Bsr = make_rsrc(has_bias ? static_cast<const uint8_t*>(p.bias) + scales * bsz : (const uint8_t*)p.sw, has_bias ? (uint32_t)N * bsz : 0u);
#pragma unroll
      for (int j = 0; j < TN; ++j)
        braw[j] = bias_bf16 ? (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(Bsr, my_column(j) * 2, 0, 0)
                            : (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(Bsr, my_column(j) * 4, 0, 0);
    }
    asm volatile("" ::: "memory");
    if (!last) {
      now = next;
      aim(now);
      my_tok = token(now, wave_m * 64 + lane);
    } else {  // nothing: loads outside the descriptors touch no memory
#pragma unroll
      for (int i = 0; i < NLOADS; ++i) vo[i] = OOB_OFFSET;
    }
    step(0, c0{});
    step(BK, c0{});
    asm volatile("" ::: "memory");

    // ---- epilogue: three rounded operations, then bf16 rows of neighbouring columns a dword a lane
    const uint32_t rowb = (uint32_t)FH * ESZ;
    const int rows = end - mw < 32 * TM ? end - mw : 32 * TM;
    const uint32_t window = rows > 0 ? (uint32_t)rows * rowb - (uint32_t)nt * ESZ : 0u;
    const __amdgpu_buffer_rsrc_t Cr =
        make_rsrc(static_cast<uint8_t*>(p.y) + (rows > 0 ? ((int64_t)mw * FH + nt) * ESZ : 0), window);
#pragma unroll
    for (int j = 0; j < TN; ++j) bn[j] = !has_bias ? 0.0f : bias_bf16 ? bf16_bits_to_f32(braw[j]) : __uint_as_float(braw[j]);
    const bool odd = lane & 1, pairs = (N & 1) == 0;
    const uint32_t c = (uint32_t)(my_column(0) - nt);
    uint32_t at = OOB_OFFSET;
    if (my_column(0) < FH) at = (uint32_t)rq * rowb + (SWI && OUT == OUT_BF16 ? (c & ~1u) * 2 + (odd ? rowb : 0u) : c * ESZ);
    const uint32_t at1 = !SWI && my_column(1) < FH ? (uint32_t)rq * rowb + (c + 1) * ESZ : OOB_OFFSET;  // odd N: the second column by itself
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int r0 = i * 32 + g * 8;
        const v4f sxq = *reinterpret_cast<const v4f*>(sx_lds + r0 + rq);
        float y[TN][4];
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            y[j][q] = __fmul_rn(__fmul_rn((float)acc[i][j][g * 4 + q], sxq[q]), swn[j]);
            if constexpr (!SWI) y[j][q] = has_bias ? __fadd_rn(y[j][q], bn[j]) : y[j][q];
          }
        if constexpr (SWI) {
          float h[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) h[q] = grouped_swiglu<OUT>(y[0][q], y[1][q]);
          if constexpr (OUT == OUT_F32) {
#pragma unroll
            for (int q = 0; q < 4; ++q) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(h[q]), Cr, at + (r0 + q) * rowb, 0, STORE_WT);
          } else {
#pragma unroll
            for (int s = 0; s < 2; ++s) {  // rows 2s, 2s + 1 of two lanes -> two columns of one row: the even lane the first row
              const uint32_t mine2 = pack_bf16x2(h[2 * s], h[2 * s + 1]);
              const uint32_t other = (uint32_t)__builtin_amdgcn_mov_dpp((int)mine2, 0xB1 /* quad_perm [1,0,3,2] */, 0xf, 0xf, true);
              __builtin_amdgcn_raw_buffer_store_b32(__builtin_amdgcn_perm(other, mine2, odd ? 0x03020706u : 0x05040100u), Cr,
                                                    at + (r0 + 2 * s) * rowb, 0, STORE_WT);
            }
          }
        } else if (pairs) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if constexpr (OUT == OUT_F32) {
              const v2i_t o = {__float_as_int(y[0][q]), __float_as_int(y[1][q])};
              __builtin_amdgcn_raw_buffer_store_b64(o, Cr, at + (r0 + q) * rowb, 0, STORE_WT);
            } else {
              __builtin_amdgcn_raw_buffer_store_b32(pack_bf16x2(y[0][q], y[1][q]), Cr, at + (r0 + q) * rowb, 0, STORE_WT);
            }
          }
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if constexpr (OUT == OUT_F32) {
              __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(y[0][q]), Cr, at + (r0 + q) * rowb, 0, 0);
              __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(y[1][q]), Cr, at1 + (r0 + q) * rowb, 0, 0);
            } else {
              const uint32_t pk = pack_bf16x2(y[0][q], y[1][q]);
              __builtin_amdgcn_raw_buffer_store_b16((uint16_t)pk, Cr, at + (r0 + q) * rowb, 0, 0);
              __builtin_amdgcn_raw_buffer_store_b16((uint16_t)(pk >> 16), Cr, at1 + (r0 + q) * rowb, 0, 0);
            }
          }
        }
      }
    }
    if (last) break;
  }
  AQ_WAIT_VMCNT(0);  // nothing lands in LDS behind the walk
  AQ_BARRIER();
}

template <int OUT, bool SWI>
int grouped_walk_launch(const GroupedArgs& a, hipStream_t st) {
  const int tiles_n = (a.N + GW_BN - 1) / GW_BN;
  const int64_t most = grouped_most_tiles(a.R, a.E, GW_BM) * tiles_n;
  if (most > 0x7fffffff) return AQ_E_RANGE;
  const int cus = device_cus();
  queue_kernel(grouped_walk_kernel<OUT, SWI>, dim3((unsigned)(most < cus ? most : cus)), dim3(GW_THREADS), 0, st, a, tiles_n,
               UDiv::of((uint32_t)tiles_n));
  return (int)hipGetLastError();
}
template int grouped_walk_launch<OUT_BF16, false>(const GroupedArgs&, hipStream_t);
template int grouped_walk_launch<OUT_F32, false>(const GroupedArgs&, hipStream_t);
template int grouped_walk_launch<OUT_BF16, true>(const GroupedArgs&, hipStream_t);
template int grouped_walk_launch<OUT_F32, true>(const GroupedArgs&, hipStream_t);

}  // namespace aq
