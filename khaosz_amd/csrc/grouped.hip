// One Linear per expert on the rows of that expert, any number of rows each: y[r] = (float(sum_k xq[t, k] wq[e, n, k]) sx[t]) sw[e, n] (+ bias[e, n])
// for the rows offsets[e] <= r < offsets[e + 1] of expert e, t = tokens[r] or r itself: the arithmetic of the single Linear, three rounded
// operations and one cast.  SwiGLU: the weights are up and gate stacked, both rounded to the output's type, h = up silu(gate).
//
// The groups' sizes are known on the device alone.  A launch has workgroups for the most tiles of rows that any split of R rows over
// E experts can need; each finds its own by a scan over the offsets, and those past the last one end.
#include <cmath>

#include "aq_grouped.h"
#include "aq_rows.h"

namespace aq {

struct RowTile {
  int e, first, end;  // rows first .. end - 1; end of the expert's rows
};

// Tile `idx` of the list that has ceil(rows / BM) tiles of every expert: every lane looks at a run of experts.  false: there is none.
// Offsets outside 0 .. R, or that fall, count as the nearest that do not: nothing is read or written outside the R rows.
// (GroupTiles answers the same of offsets in LDS, for workgroups that ask again and again.  Of one question this is the shorter chain, without a store, a
// barrier and reads of LDS: 16 tokens' 6 of 64 experts, the layer 90.0 us, by GroupTiles 93.8; one token's 21.2 and 21.6; 10 rows of 8 experts 4.9 and 5.2.  Of 512
// experts, eight to a lane, it is the longer one: 64 rows of 512 -> 512 10.6 and 9.3.)
template <int BM, int PER>
__device__ __forceinline__ bool find_tile(const GroupedArgs& p, int idx, int lane, RowTile& t) {
  int o[PER + 1], n = 0, mine[PER];
#pragma unroll
  for (int i = 0; i <= PER; ++i) {
    const int e = lane * PER + i;
    o[i] = p.offsets[e < p.E ? e : p.E];
  }
#pragma unroll
  for (int i = 0; i <= PER; ++i) o[i] = o[i] < 0 ? 0 : o[i] > p.R ? p.R : o[i];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int rows = o[i + 1] - o[i];
    mine[i] = rows > 0 ? (rows + BM - 1) / BM : 0;
    n += mine[i];
  }
  const int upto = wave_scan(n);
  const unsigned long long past = __ballot(upto > idx);
  if (!past) return false;
  const int at = __builtin_ctzll(past);
  int before = upto - n, e = lane * PER, first = o[0], end = o[1];
#pragma unroll
  for (int i = 1; i < PER; ++i)
    if (before + mine[i - 1] <= idx) before += mine[i - 1], e = lane * PER + i, first = o[i], end = o[i + 1];
    else break;
  t.e = __builtin_amdgcn_readlane(e, at);
  t.first = __builtin_amdgcn_readlane(first, at) + (idx - __builtin_amdgcn_readlane(before, at)) * BM;
  t.end = __builtin_amdgcn_readlane(end, at);
  return true;
}
template <int BM>
__device__ __forceinline__ bool find_tile(const GroupedArgs& p, int idx, int lane, RowTile& t) {
  return p.E <= 64    ? find_tile<BM, 1>(p, idx, lane, t)
         : p.E <= 128 ? find_tile<BM, 2>(p, idx, lane, t)
         : p.E <= 256 ? find_tile<BM, 4>(p, idx, lane, t)
                      : find_tile<BM, GP_MAX_E / 64>(p, idx, lane, t);
}

__device__ __forceinline__ float load_bias(const GroupedArgs& p, int64_t i) {
  return p.bias_dtype == AQ_BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(p.bias)[i]) : static_cast<const float*>(p.bias)[i];
}
template <int OUT>
__device__ __forceinline__ void store_out(void* y, int64_t i, float v) {
  if constexpr (OUT == OUT_BF16) static_cast<uint16_t*>(y)[i] = (uint16_t)f32_to_bf16_bits(v);
  else static_cast<float*>(y)[i] = v;
}
// Tiles of 16 rows x 32 weight rows: four wavefronts take every fourth 128-byte line of K, weights straight from memory into registers, the sums
// meet in LDS.  Rows come as codes, from memory like the weights (IN = CODES), or as they are, and every workgroup quantises its own while its
// weights are on their way (the row quantiser's arithmetic): a launch less for a few rows.
// What bounds it: HBM (16 tokens' 6 of 64 experts, SwiGLU of 2048 -> 1408 from codes: 293 MB in 49 us, 6.0 TB/s, the launch included); of one token the
// chain of launch, offsets, row and weights (35 MB in 11 us).  A workgroup that walks units, the next one's weights on their way, is slower (one token
// 14.6 us, 16 tokens 54): two of its size fit a compute unit where four of these do.
constexpr int GP_MAX_TOKEN_K = 64;  // choices of a token
enum { IN_CODES = 0, IN_BF16 = 1, IN_F32 = 2 };
constexpr int GF_ROWS = 16, GF_COLS = 32, GF_WAVES = 4;
// bytes between rows of codes in LDS: 16 of them then begin 4 banks apart
__host__ __device__ inline int few_pitch(int K) { return (K + 127) / 128 * 128 + 16; }

// A row of x (rows: they are, in its type) on its way into a wavefront's registers; -1: zeros.
template <bool BF16, int VPL>
__device__ __forceinline__ void ask_for_row(RowsToLds<BF16, 1, VPL>& r, const uint8_t* x, int K, int row, int lane) {
  const uint32_t bytes = (uint32_t)K * (BF16 ? 2 : 4);
  const __amdgpu_buffer_rsrc_t R = make_rsrc(x + (row < 0 ? 0 : row) * (int64_t)bytes, row < 0 ? 0u : bytes);
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const v4i v = __builtin_amdgcn_raw_buffer_load_b128(R, (i * 64 + lane) * 16, 0, 0);
    r.c[0][i] = make_uint4((uint32_t)v[0], (uint32_t)v[1], (uint32_t)v[2], (uint32_t)v[3]);
  }
}

// DEEP: lines of a wavefront on their way at a time, cut to the rows' length class (a load of nothing takes its turn in the address path all the
// same, and branches around loads make them wait for each other: 24.7 -> 66 us for four tokens' up and gate).
template <int OUT, bool SWI, int IN, int VPL, int DEEP>
__global__ __launch_bounds__(GF_WAVES * 64, VPL == 8 ? 3 : VPL == 16 ? 2 : 1) void grouped_few_kernel(GroupedArgs p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t xs[];  // IN: the rows' codes
  __shared__ int part[GF_WAVES][2][GF_ROWS][17];
  __shared__ float scale[GF_ROWS];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // tokens of up to 64 rows come beside the offsets: x is then asked for without another wait
  const bool near = p.R <= 64;
  int my_token = -1;
  if (p.tokens && near) my_token = p.tokens[lane < p.R ? lane : 0];
  RowTile t;
  if (!find_tile<GF_ROWS>(p, blockIdx.y, lane, t)) return;
  const int K = p.K, FH = SWI ? p.N / 2 : p.N;
  const int n0 = (int)blockIdx.x * (SWI ? 16 : GF_COLS);
  const __amdgpu_buffer_rsrc_t Wr = make_rsrc(p.w + t.e * p.w_bytes, (uint32_t)p.w_bytes);
  const int r16 = lane & 15, q16 = (lane >> 4) * 16;
  const int na = n0 + r16, nb = SWI ? FH + na : na + 16;
  const bool ina = na < FH, inb = SWI ? ina : nb < FH;
  const uint32_t ao = (uint32_t)na * (uint32_t)K + q16, bo = (uint32_t)nb * (uint32_t)K + q16;
  const int lines = (K + 127) / 128;
  auto token = [&](int row) {  // -1: none
    int tok = row;
    if (p.tokens && near) tok = __shfl(my_token, row & 63);
    else if (p.tokens) tok = row < t.end ? p.tokens[row] : -1;
    return row < t.end && tok >= 0 && tok < p.x_rows ? tok : -1;
  };
  v4i av[2 * DEEP], bv[2 * DEEP];
  auto k_of = [&](int l0, int i) { return (l0 + i / 2 * GF_WAVES) * 128 + i % 2 * 64; };
  auto load_weights = [&](int l0) {
#pragma unroll
    for (int i = 0; i < 2 * DEEP; ++i) {
      const int k = k_of(l0, i);
      const bool in = k + q16 < K;
      av[i] = __builtin_amdgcn_raw_buffer_load_b128(Wr, in && ina ? ao + k : OOB_OFFSET, 0, 2);
      bv[i] = __builtin_amdgcn_raw_buffer_load_b128(Wr, in && inb ? bo + k : OOB_OFFSET, 0, 2);
    }
  };
  // The first row of each wavefront before the weights, as it is rounded while they come (behind them if its token takes a wait of its own).
  constexpr bool BF16 = IN == IN_BF16;
  const int rows = t.end - t.first < GF_ROWS ? t.end - t.first : GF_ROWS;
  const bool known = !p.tokens || near;
  int tok = -1;
  [[maybe_unused]] RowsToLds<BF16, 1, VPL> ahead;
  if constexpr (IN != IN_CODES) {
    if (known) tok = __builtin_amdgcn_readfirstlane(token(t.first + wave));
    ask_for_row<BF16>(ahead, p.x, K, tok, lane);
  }
  load_weights(wave);
  // the epilogue's operands, one tile row and two columns (SwiGLU: one) to a thread
  const int m = tid >> 4, c = tid & 15, out_row = t.first + m;
  float sw[2], bias[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int n = SWI ? g * FH + n0 + c : n0 + g * 16 + c;
    const int64_t at = (int64_t)t.e * p.N + (n < p.N ? n : 0);
    sw[g] = p.sw[at];
    bias[g] = !SWI && p.bias ? load_bias(p, at) : 0.0f;
  }
  float sx = 0.0f;
  if constexpr (IN == IN_CODES) {
    const int tok = token(out_row);
    if (tok >= 0) sx = p.sx[tok];
  }
  const int pitch = few_pitch(K);
  [[maybe_unused]] const uint8_t* const held = xs + (r16 < p.held ? r16 : 0) * pitch;  // (rows past the tile's: any)
  __amdgpu_buffer_rsrc_t Xr = make_rsrc(p.x, IN == IN_CODES ? (uint32_t)p.x_rows * (uint32_t)K : 0u);
  uint32_t xo = OOB_OFFSET;
  if constexpr (IN == IN_CODES) {
    const int tok = token(t.first + r16);
    if (tok >= 0) xo = (uint32_t)tok * (uint32_t)K + q16;
  } else {
    auto round_row = [&](RowsToLds<BF16, 1, VPL>& r, int m, int tok) {
      r.finish(1, 1, K, xs + m * pitch, pitch, scale + m, 0, 1, lane);
      if (tok < 0 && lane == 0) scale[m] = 0.0f;  // a row of zeros
    };
    if (known && wave < rows) round_row(ahead, wave, tok);
    for (int m = known ? wave + GF_WAVES : wave; m < rows; m += GF_WAVES) {
      const int tok = __builtin_amdgcn_readfirstlane(token(t.first + m));
      RowsToLds<BF16, 1, VPL> r;
      ask_for_row<BF16>(r, p.x, K, tok, lane);
      round_row(r, m, tok);
    }
    __syncthreads();
  }
  v4i acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  for (int l0 = wave; l0 < lines;) {
    v4i xv[2 * DEEP];
#pragma unroll
    for (int i = 0; i < 2 * DEEP; ++i) {
      const int k = k_of(l0, i);
      if constexpr (IN == IN_CODES) {
        xv[i] = __builtin_amdgcn_raw_buffer_load_b128(Xr, k + q16 < K && xo != OOB_OFFSET ? xo + k : OOB_OFFSET, 0, 0);
      } else {
        xv[i] = v4i{0, 0, 0, 0};  // (past K the weights are zeros)
        if (k < K) xv[i] = *reinterpret_cast<const v4i*>(held + k + q16);
      }
    }
#pragma unroll
    for (int i = 0; i < 2 * DEEP; ++i) {
      acc[0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xv[i], av[i], acc[0], 0, 0, 0);
      acc[1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xv[i], bv[i], acc[1], 0, 0, 0);
    }
    l0 += GF_WAVES * DEEP;
    if (l0 < lines) load_weights(l0);
  }
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[wave][g][(lane >> 4) * 4 + i][r16] = acc[g][i];
  __syncthreads();
  if (out_row >= t.end) return;
  if constexpr (IN != IN_CODES) sx = scale[m];
  float y[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    int s = 0;
#pragma unroll
    for (int v = 0; v < GF_WAVES; ++v) s += part[v][g][m][c];
    y[g] = __fmul_rn(__fmul_rn((float)s, sx), sw[g]);
    if constexpr (!SWI) {
      if (p.bias) y[g] = __fadd_rn(y[g], bias[g]);
      const int n = n0 + g * 16 + c;
      if (n < FH) store_out<OUT>(p.y, (int64_t)out_row * FH + n, y[g]);
    }
  }
  if constexpr (SWI) store_out<OUT>(p.y, (int64_t)out_row * FH + n0 + c, grouped_swiglu<OUT>(y[0], y[1]));  // (F is a multiple of 16)
}

// The second product and the weighted sum in one launch, for a few tokens: a workgroup has 8 columns of one token's output, a wavefront one of its
// choices at a time: it quantises that row of h, multiplies it with its expert's 8 weight rows and leaves the rounded output times its weight in LDS,
// where the choices are added in their order: the bits of the grouped Linear and combine_rows.  Experts that several tokens chose are read for each.
// The matrix core's 16 columns are the 8 weight rows' two halves of K, and rows 0 and 1 of its other operand the same halves of the row: half the
// loads and products of 16 columns in a row, on twice the compute units (one token, 6 of 64 experts of 2048 / 1408: 9.8 us).
constexpr int GT_WAVES = 8, GT_COLS = 8;
struct TokenArgs {
  GroupedArgs g;  // x: h [R, K]
  const int32_t* rows;
  const float* weights;
  const void* res;
  int k;
};
// GT_LINES: of 128 bytes of each half on their way at a time.  With 8 or 12 a compute unit has room for one workgroup, with 4 for two (8 tokens' 8 of 256
// experts of 1024 / 512, the layer: 38.2, 43.9 and 33.5 us; one token's 6 of 64 of 2048 / 1408: 22.0, 22.8 and 22.3).
constexpr int GT_LINES = 4;
template <int OUT, int VPL>
__global__ __launch_bounds__(GT_WAVES * 64, VPL == 4 ? 4 : 2) void grouped_token_kernel(TokenArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t xs[];  // a row of codes per wavefront
  __shared__ float term[GP_MAX_TOKEN_K][GT_COLS];
  __shared__ float scale[GT_WAVES];
  constexpr bool BF16 = OUT == OUT_BF16;
  const GroupedArgs& p = a.g;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int K = p.K, N = p.N, t = blockIdx.y, n0 = (int)blockIdx.x * GT_COLS, pitch = few_pitch(K);
  const int r16 = lane & 15, q16 = (lane >> 4) * 16, n = n0 + (r16 & 7);
  const int half = (K + 31) / 32 * 16, k_of_lane = (r16 >> 3) * half, k_end = r16 >> 3 ? K - half : half;
  uint8_t* const mine = xs + wave * pitch;
  const uint8_t* const operand = mine + (r16 & 1) * half + q16;
  for (int j = wave; j < a.k; j += GT_WAVES) {
    const int row = __builtin_amdgcn_readfirstlane(a.rows[(int64_t)t * a.k + j]);
    float y = 0.0f, w = 0.0f;
    if (row >= 0 && row < p.R) {
      int e = 0;  // experts whose rows end at or before it
      for (int i = lane; i < p.E; i += 64) e += __popcll(__ballot(p.offsets[i + 1] <= row));
      e = __builtin_amdgcn_readfirstlane(e);
      if (e < p.E) {
        const __amdgpu_buffer_rsrc_t Wr = make_rsrc(p.w + e * p.w_bytes, (uint32_t)p.w_bytes);
        const uint32_t wo = (uint32_t)n * (uint32_t)K + k_of_lane + q16;
        w = a.weights[(int64_t)t * a.k + j];
        const float sw = p.sw[(int64_t)e * N + n];
        RowsToLds<BF16, 1, VPL> r;
        r.issue(p.x + (int64_t)row * K * (BF16 ? 2 : 4), 1, K, K, 0, 1, lane);
        v4i acc = {0, 0, 0, 0};
        for (int k0 = 0; k0 < half; k0 += GT_LINES * 128) {
          v4i wv[2 * GT_LINES];
#pragma unroll
          for (int i = 0; i < 2 * GT_LINES; ++i) {
            const int k = k0 + i * 64;
            wv[i] = __builtin_amdgcn_raw_buffer_load_b128(Wr, k + q16 < k_end ? wo + k : OOB_OFFSET, 0, 2);
          }
          if (k0 == 0) {
            r.finish(1, 1, K, mine, pitch, scale + wave, 0, 1, lane);
            __builtin_amdgcn_wave_barrier();  // (a wavefront's LDS operations keep their order)
          }
#pragma unroll
          for (int i = 0; i < 2 * GT_LINES; ++i) {
            const int k = k0 + i * 64;
            if (k < half) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const v4i*>(operand + k), wv[i], acc, 0, 0, 0);
          }
        }
        const int sum = acc[0] + __builtin_amdgcn_update_dpp(0, acc[1], 0x128 /* row_ror:8 */, 0xf, 0xf, false);  // lanes 0 .. 7: both halves
        y = __fmul_rn(__fmul_rn((float)sum, scale[wave]), sw);
        if constexpr (BF16) y = bf16_bits_to_f32(f32_to_bf16_bits(y));
      }
    }
    if (lane < GT_COLS) term[j][lane] = __fmul_rn(w, y);
  }
  __syncthreads();
  if (tid >= GT_COLS) return;
  float sum = 0.0f;
  for (int j = 0; j < a.k; ++j) {
    const int row = a.rows[(int64_t)t * a.k + j];
    if (row >= 0 && row < p.R) sum = __fadd_rn(sum, term[j][tid]);
  }
  const int64_t at = (int64_t)t * N + n0 + tid;
  if (a.res) sum = __fadd_rn(sum, BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(a.res)[at]) : static_cast<const float*>(a.res)[at]);
  store_out<OUT>(p.y, at, sum);
}

#ifdef AQ_LAB
static int g_forced_grouped = 0;  // lab build only: 0 = by size
#endif

// Experts with rows, of E, when R rows are dealt out evenly.
static double experts_used(int64_t R, int64_t E) { return E * (1.0 - std::exp(-(double)R / E)); }

// Which kernel: the one whose estimated time, in us, is least.  Tiles of 16 rows: units of 32 weight rows, four to a compute unit at a time.  Walked
// tiles: rounds of tiles (mostly whole ones: the last takes as long), each of its steps and a beginning and an end, beside the weights' way from memory.
// Fitted to 900 random sizes of experts that are asked for alike (1 to 256 experts, 1 to 8192 tokens, K 128 to 6912), 400 of uneven ones (2 to 128 experts, 20 to
// 600 rows each) and 350 with 0.2 to 300 rows each: 1.5, 0.9 and 1.4 % slower than the best kernel in the mean, one in twenty 12, 6 and 11 % or more.  At 199
// other sizes, asked for as routers ask, 3.9 % in the mean, one in twenty 20 % or more (always 128 x 256 59 %, always 128 x 128 36 %).
// Chosen by the launch itself, from the tiles that there are, the width was 0.3 % off on the second, but three widths in one kernel cost 1 to 2 % and the
// choice 0.5 to 1 us.
enum { GROUPED_FEW = 1, GROUPED_WALK_256 = 2, GROUPED_WALK_128 = 3, GROUPED_WALK_64 = 4 };
static double walk_us(const GroupedArgs& a, double used, int width, int least_steps, double launch, double ends, double step, double tb_s, double tail, double even) {
  const double avg = a.R / used / 128 + tail, steps = (a.K + 127) / 128;
  const double part = used * (avg > 1 ? avg : 1) * ((a.N + width - 1) / width) / device_cus();
  const double rounds = even * part + (1 - even) * std::ceil(part);
  const double c = (rounds > 1 ? rounds : 1) * (ends + step * (steps > least_steps ? steps : least_steps)), m = used * a.N * a.K * 1e-6 / tb_s;
  return launch + std::sqrt(std::sqrt(c * c * c * c + m * m * m * m));
}
static bool few_fits(int64_t R, int64_t E) { return grouped_most_tiles(R, E, GF_ROWS) <= 65535; }  // (the grid's second axis)
static int choose_grouped(const GroupedArgs& a, bool swiglu) {
  if (a.N > (1 << 20)) return GROUPED_FEW;  // (a tile's rows by 32-bit offsets)
#ifdef AQ_LAB
  if (g_forced_grouped) return g_forced_grouped;
#endif
  const double used = experts_used(a.R, a.E), rows = a.R / used / 16 + 0.58;
  const double units = used * (rows > 1 ? rows : 1) * ((a.N + GF_COLS - 1) / GF_COLS);
  const double us[] = {units / (4 * device_cus()) * (2.24 + 12.82 * a.K / 1024) + 1.80 * ((a.K + 2047) / 2048),
                       walk_us(a, used, 256, 6, 1.49, 3.80, 1.085, 4.53, 0.544, 0.127), walk_us(a, used, 128, 7, 3.55, 2.36, 0.626, 4.84, 0.527, 0.205),
                       walk_us(a, used, 64, 10, 3.36, 0.335, 0.507, 6.36, 0.532, 0.217)};
  int best = few_fits(a.R, a.E) ? 0 : 1;
  for (int i = best + 1; i < (swiglu ? 3 : 4); ++i)
    if (us[i] < us[best]) best = i;
  return GROUPED_FEW + best;
}

template <int OUT, bool SWI, int IN, int VPL, int DEEP>
static int launch_few_of(const GroupedArgs& a, hipStream_t st) {
  const int64_t tiles = grouped_most_tiles(a.R, a.E, GF_ROWS), cols = (a.N + GF_COLS - 1) / GF_COLS;
  if (tiles > 65535 || cols > 0x7fffffff) return AQ_E_RANGE;  // (more rows of N > 2^20 columns than memory holds)
  queue_kernel((grouped_few_kernel<OUT, SWI, IN, VPL, DEEP>), dim3((unsigned)cols, (unsigned)tiles), dim3(GF_WAVES * 64),
               IN == IN_CODES ? 0 : a.held * few_pitch(a.K), st, a);
  return (int)hipGetLastError();
}

// VPL: 16-byte vectors of a row in a lane (rows as they are), 4, 8 or 16: rows of the length class below are not its own.
template <int OUT, bool SWI, int IN, int VPL>
static int launch_few(const GroupedArgs& a, hipStream_t st) {
  constexpr int DEEP_3 = GF_WAVES * 3 * 128, MOST = IN == IN_CODES ? 1 << 30 : VPL * 64 * (IN == IN_BF16 ? 8 : 4), LEAST = VPL <= 4 ? 0 : MOST / 2;
  if constexpr (LEAST < DEEP_3)
    if (a.K <= DEEP_3) return launch_few_of<OUT, SWI, IN, VPL, 3>(a, st);
  if constexpr (MOST > DEEP_3) return launch_few_of<OUT, SWI, IN, VPL, 4>(a, st);
  return AQ_E_RANGE;
}

// Rows as they are (a.x of `dtype`, which is the output's type too), quantised in the launch.  A workgroup has their codes in LDS: up to 16 rows of 4096,
// or fewer of up to 8192, so that a compute unit has room for two.
static int64_t most_in_launch(int dtype) { return dtype == AQ_BF16 ? 8192 : 4096; }  // of 16 vectors a lane
static int rows_held(int64_t R) { return R < GF_ROWS ? (int)R : GF_ROWS; }
static bool rows_fit(int64_t K, int64_t R) { return rows_held(R) * few_pitch((int)K) <= GF_ROWS * few_pitch(4096); }
template <int OUT, int IN, bool SWI>
static int launch_rows_of(const GroupedArgs& a, hipStream_t st) {
  constexpr int CLASS = 256 * (IN == IN_BF16 ? 8 : 4);
  return a.K <= CLASS       ? launch_few<OUT, SWI, IN, 4>(a, st)
         : a.K <= 2 * CLASS ? launch_few<OUT, SWI, IN, 8>(a, st)
                            : launch_few<OUT, SWI, IN, 16>(a, st);
}
template <bool SWI>
static int launch_rows(GroupedArgs a, int dtype, hipStream_t st) {
  a.held = rows_held(a.R);
  return dtype == AQ_BF16 ? launch_rows_of<OUT_BF16, IN_BF16, SWI>(a, st) : launch_rows_of<OUT_F32, IN_F32, SWI>(a, st);
}
// Whether a product of a layer quantises its rows itself: a launch less, but every workgroup reads and rounds its tile's rows, one after the other in a
// wavefront, holds up to 16 of them in LDS and longer ones in more registers.  So the weights times 1 + rows an expert have a limit by the rows' length
// (us of the layer, with | without.  Up to 2048: 16 tokens' 6 of 64 of 2048 / 1408, x 93.1 | 95.8, then h 89.8 | 93.1; 16 tokens' 4 of 16 of 2048 / 5632, x 123.2 | 121.5.  Up
// to 4096: 4 tokens' 2 of 8 of 3584 / 4096, x 63.2 | 69.8, 8 tokens' 80.5 | 77.7.  Up to 8192: one token's 2 of 8 of 1536 / 6912, h 25.6 | 35.0, of 4096 / 8192 67.8 | 65.7,
// 4 tokens' 143 | 123), and rows an expert by themselves (32 tokens' 8 of 16 of 5120 / 144, h 50.0 | 43.4).  At 200 sizes, with the rule
// of the sum below, 2.0 % slower than the best of the three ways in the mean, one in twenty 11 %; always apart 33 %, always in the launch 13 %.
static bool rows_in_launch(int64_t R, int64_t E, int64_t N, int64_t K, int dtype) {
  if (K > most_in_launch(dtype) || !few_fits(R, E)) return false;
#ifdef AQ_LAB
  if (g_forced_grouped) return g_forced_grouped == GROUPED_FEW;
#endif
  const double limit = 4 * K <= most_in_launch(dtype) ? 8e8 : 2 * K <= most_in_launch(dtype) ? 3e8 : 1.2e8;
  return R <= 8 * E && experts_used(R, E) * (double)(N * K) * (1.0 + (double)R / E) <= limit;
}

// The second product with the weighted sum (dim is a multiple of 16, and so of GT_COLS).
template <int OUT, int VPL>
static int launch_token(const TokenArgs& a, int64_t T, hipStream_t st) {
  const dim3 grid((unsigned)(a.g.N / GT_COLS), (unsigned)T), block(GT_WAVES * 64);
  const size_t lds = (size_t)(a.k < GT_WAVES ? a.k : GT_WAVES) * few_pitch(a.g.K);
  queue_kernel((grouped_token_kernel<OUT, VPL>), grid, block, lds, st, a);
  return (int)hipGetLastError();
}
template <int OUT>
static int launch_tokens_of(const TokenArgs& a, int64_t T, hipStream_t st) {
  constexpr int CLASS = 256 * (OUT == OUT_BF16 ? 8 : 4);
  return a.g.K <= CLASS ? launch_token<OUT, 4>(a, T, st) : a.g.K <= 2 * CLASS ? launch_token<OUT, 8>(a, T, st) : launch_token<OUT, 16>(a, T, st);
}
static int launch_tokens(const TokenArgs& a, int64_t T, int dtype, hipStream_t st) {
  return dtype == AQ_BF16 ? launch_tokens_of<OUT_BF16>(a, T, st) : launch_tokens_of<OUT_F32>(a, T, st);
}
// Whether it is: what the experts of several tokens cost more, read for each, is then less than the launch saved (us of the layer, with | without: 64
// choices of 256 experts of 1024 / 512, 4 MB more, 33.4 | 36.0; 18 of 64 of 2048 / 1408, 7 MB, 42.7 | 40.2; 24 of them, 11 MB, 48.8 | 46.3).  And its workgroups, of a
// token's 8 columns each, are at most four to a compute unit, which has room for one or two at a time: of wide layers with narrow experts there are many with little
// to do (54 tokens' 1 of 128 of 3568 / 80 112.7 | 31.1; 8 tokens' 1 of 60 of 5200 / 80 35.5 | 22.1; 7 tokens' 8 of 64 of 592 / 256 14.9 | 16.0).  At 835 sizes 0.8 % slower than
// the better of the two in the mean, one in twenty 4 % or more (without the second condition 5.2 and 32 %).
static bool tokens_in_launch(int64_t T, int64_t k, int64_t E, int64_t dim, int64_t F) {
  return T * (dim / GT_COLS) <= 4 * device_cus() && ((double)(T * k) - experts_used(T * k, E)) * (double)(dim * F) <= 5e6;
}

template <int OUT, bool SWI>
static int launch_grouped(const GroupedArgs& a, hipStream_t st) {
  const int kind = choose_grouped(a, SWI);
  if (kind != GROUPED_FEW) return grouped_walk_launch<OUT, SWI>(a, kind == GROUPED_WALK_256 ? 256 : kind == GROUPED_WALK_128 ? 128 : 64, st);
  return launch_few<OUT, SWI, IN_CODES, 1>(a, st);
}

static int grouped(const int8_t* xq, const float* sx, int64_t x_rows, const int8_t* wq, const float* sw, const void* bias, int bias_dtype,
                   const int32_t* offsets, int64_t E, const int32_t* tokens, int64_t R, void* y, int y_dtype, int64_t N, int64_t K, bool swiglu,
                   void* stream) {
  if (y_dtype != AQ_F32 && y_dtype != AQ_BF16) return AQ_E_DTYPE;
  if (bias && bias_dtype != AQ_F32 && bias_dtype != AQ_BF16) return AQ_E_DTYPE;
  if (x_rows < 0 || E <= 0 || R < 0 || N <= 0 || K <= 0 || K % 16 || (!tokens && x_rows != R)) return AQ_E_SHAPE;
  if (E > GP_MAX_E || R > GP_MAX_R || N > 0x7fffffff || N * K > (int64_t)OOB_OFFSET || x_rows * K > (int64_t)OOB_OFFSET) return AQ_E_RANGE;
  if (R == 0) return AQ_OK;
  if (!offsets || !wq || !sw || !y || (x_rows > 0 && (!xq || !sx))) return AQ_E_NULL;
  if (check_ptr16(xq) || check_ptr16(wq) || check_ptr16(y) || check_ptr(sx, 4) || check_ptr(sw, 4) || check_ptr(offsets, 4) || check_ptr(tokens, 4) ||
      check_ptr(bias, bias_dtype == AQ_BF16 ? 2 : 4))
    return AQ_E_ALIGN;
  GroupedArgs a{};
  a.x = reinterpret_cast<const uint8_t*>(xq);
  a.sx = sx;
  a.w = reinterpret_cast<const uint8_t*>(wq);
  a.sw = sw;
  a.bias = bias;
  a.bias_dtype = bias_dtype;
  a.offsets = offsets;
  a.tokens = tokens;
  a.y = y;
  a.w_bytes = N * K;
  a.x_rows = (int)x_rows;
  a.R = (int)R;
  a.E = (int)E;
  a.N = (int)N;
  a.K = (int)K;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (swiglu) return y_dtype == AQ_BF16 ? launch_grouped<OUT_BF16, true>(a, st) : launch_grouped<OUT_F32, true>(a, st);
  return y_dtype == AQ_BF16 ? launch_grouped<OUT_BF16, false>(a, st) : launch_grouped<OUT_F32, false>(a, st);
}

// Scratch of a whole layer: codes and scales of x, h, its codes and scales, the experts' outputs.
struct ExpertsScratch {
  int64_t xq, sx, h, hq, sh, y, bytes;
  ExpertsScratch(int64_t T, int64_t R, int64_t dim, int64_t F, int size) {
    auto take = [&](int64_t n) {
      const int64_t at = bytes;
      bytes += (n + 255) / 256 * 256;
      return at;
    };
    bytes = 0;
    xq = take(T * dim);
    sx = take(T * 4);
    h = take(R * F * size);
    hq = take(R * F);
    sh = take(R * 4);
    y = take(R * dim * size);
  }
};

}  // namespace aq

extern "C" int aq_linear_w8a8_grouped(const int8_t* xq, const float* sx, int64_t x_rows, const int8_t* wq, const float* sw, const void* bias,
                                      int bias_dtype, const int32_t* offsets, int64_t E, const int32_t* tokens, int64_t R, void* y, int y_dtype,
                                      int64_t N, int64_t K, void* stream) {
  return aq::grouped(xq, sx, x_rows, wq, sw, bias, bias_dtype, offsets, E, tokens, R, y, y_dtype, N, K, false, stream);
}

extern "C" int aq_swiglu_w8a8_grouped(const int8_t* xq, const float* sx, int64_t x_rows, const int8_t* wq, const float* sw, const int32_t* offsets,
                                      int64_t E, const int32_t* tokens, int64_t R, void* h, int h_dtype, int64_t F, int64_t K, void* stream) {
  if (F <= 0 || F % 16) return AQ_E_SHAPE;
  return aq::grouped(xq, sx, x_rows, wq, sw, nullptr, AQ_F32, offsets, E, tokens, R, h, h_dtype, 2 * F, K, true, stream);
}

extern "C" int64_t aq_experts_w8a8_workspace_bytes(int x_dtype, int64_t T, int64_t k, int64_t dim, int64_t F) {
  if (T <= 0 || k <= 0 || dim <= 0 || F <= 0 || T > (int64_t)1 << 24 || k > 64 || dim > (1 << 24) || F > (1 << 24)) return 0;
  return aq::ExpertsScratch(T, T * k, dim, F, x_dtype == AQ_BF16 ? 2 : 4).bytes;
}

extern "C" int aq_experts_w8a8(const void* x, int x_dtype, int64_t T, int64_t dim, const int32_t* offsets, int64_t E, const int32_t* tokens,
                               const int32_t* rows, const float* weights, int64_t k, const int8_t* up_gate, const float* up_gate_scale,
                               const int8_t* down, const float* down_scale, int64_t F, const void* residual, void* out, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  if (x_dtype != AQ_F32 && x_dtype != AQ_BF16) return AQ_E_DTYPE;
  if (T < 0 || dim <= 0 || dim % 16 || E <= 0 || k <= 0 || F <= 0 || F % 16) return AQ_E_SHAPE;
  if (E > aq::GP_MAX_E || k > 64 || T > (int64_t)1 << 24 || dim > (1 << 24) || F > (1 << 24) || T * k > aq::GP_MAX_R || T * k * F > (int64_t)aq::OOB_OFFSET ||
      T * dim > (int64_t)aq::OOB_OFFSET || 2 * F * dim > (int64_t)aq::OOB_OFFSET)
    return AQ_E_RANGE;
  if (T == 0) return AQ_OK;
  if (!x || !offsets || !tokens || !rows || !weights || !up_gate || !up_gate_scale || !down || !down_scale || !out || !workspace) return AQ_E_NULL;
  if (aq::check_ptr16(x) || aq::check_ptr16(up_gate) || aq::check_ptr16(down) || aq::check_ptr16(out) || aq::check_ptr16(workspace) ||
      aq::check_ptr(up_gate_scale, 4) || aq::check_ptr(down_scale, 4) || aq::check_ptr(offsets, 4) ||
      aq::check_ptr(tokens, 4) || aq::check_ptr(rows, 4) || aq::check_ptr(weights, 4) || aq::check_ptr(residual, x_dtype == AQ_BF16 ? 2 : 4))
    return AQ_E_ALIGN;
  if (workspace_bytes < aq_experts_w8a8_workspace_bytes(x_dtype, T, k, dim, F)) return AQ_E_WORKSPACE;
  const int64_t R = T * k;
  const aq::ExpertsScratch s(T, R, dim, F, x_dtype == AQ_BF16 ? 2 : 4);
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  int8_t *const xq = reinterpret_cast<int8_t*>(ws + s.xq), *const hq = reinterpret_cast<int8_t*>(ws + s.hq);
  float *const sx = reinterpret_cast<float*>(ws + s.sx), *const sh = reinterpret_cast<float*>(ws + s.sh);
  void *const h = ws + s.h, *const y = ws + s.y;
  hipStream_t st = static_cast<hipStream_t>(stream);
  aq::GroupedArgs a{};
  a.offsets = offsets;
  a.R = (int)R;
  a.E = (int)E;
  int rc;
  if (aq::rows_in_launch(R, E, 2 * F, dim, x_dtype) && aq::rows_fit(dim, R)) {
    a.x = static_cast<const uint8_t*>(x);
    a.x_rows = (int)T;
    a.w = reinterpret_cast<const uint8_t*>(up_gate);
    a.sw = up_gate_scale;
    a.tokens = tokens;
    a.y = h;
    a.w_bytes = 2 * F * dim;
    a.N = (int)(2 * F);
    a.K = (int)dim;
    rc = aq::launch_rows<true>(a, x_dtype, st);
  } else {
    rc = aq_quant_rowwise_i8(x, x_dtype, T, dim, dim, xq, sx, stream);
    if (rc == AQ_OK) rc = aq_swiglu_w8a8_grouped(xq, sx, T, up_gate, up_gate_scale, offsets, E, tokens, R, h, x_dtype, F, dim, stream);
  }
  if (rc != AQ_OK) return rc;
  const bool few = aq::rows_in_launch(R, E, dim, F, x_dtype), token = few && aq::tokens_in_launch(T, k, E, dim, F);
  if (token || (few && aq::rows_fit(F, R))) {
    a.x = static_cast<const uint8_t*>(h);
    a.x_rows = (int)R;
    a.w = reinterpret_cast<const uint8_t*>(down);
    a.sw = down_scale;
    a.tokens = nullptr;
    a.y = token ? out : y;
    a.w_bytes = dim * F;
    a.N = (int)dim;
    a.K = (int)F;
    if (token) return aq::launch_tokens(aq::TokenArgs{a, rows, weights, residual, (int)k}, T, x_dtype, st);
    rc = aq::launch_rows<false>(a, x_dtype, st);
  } else {
    rc = aq_quant_rowwise_i8(h, x_dtype, R, F, F, hq, sh, stream);
    if (rc == AQ_OK) rc = aq_linear_w8a8_grouped(hq, sh, R, down, down_scale, nullptr, AQ_F32, offsets, E, nullptr, R, y, x_dtype, dim, F, stream);
  }
  if (rc == AQ_OK) rc = aq_combine_rows(y, x_dtype, R, dim, rows, weights, T, k, residual, out, stream);
  return rc;
}

#ifdef AQ_LAB
extern "C" int aq_lab_set_grouped_kernel(int kind) {
  if (kind < 0 || kind > aq::GROUPED_WALK_64) return AQ_E_SHAPE;
  aq::g_forced_grouped = kind;
  return AQ_OK;
}
#endif
