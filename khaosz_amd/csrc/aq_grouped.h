// What the grouped products (one Linear per expert, ragged rows) share.
#ifndef AQ_GROUPED_H
#define AQ_GROUPED_H

#include "aq_gemm.h"

namespace aq {

constexpr int GP_MAX_E = 512;
constexpr int64_t GP_MAX_R = 1 << 25;  // counts of tiles fit 31 bits, whatever the offsets say

struct GroupedArgs {
  const uint8_t* x;
  const float* sx;
  const uint8_t* w;
  const float* sw;
  const void* bias;
  int bias_dtype;
  const int32_t* offsets;
  const int32_t* tokens;
  void* y;
  int64_t w_bytes;  // of one expert
  int x_rows, R, E;
  int N;            // weight rows of an expert (SwiGLU: up and gate)
  int K;
  int held;         // rows that a workgroup has room for in LDS, where it quantises them
};

// Inclusive sum over the 64 lanes
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1 and so on
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
  return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
}

// The most tiles of BM rows that R rows over E experts can need.
inline int64_t grouped_most_tiles(int64_t R, int64_t E, int64_t BM) {
  const int64_t used = R < E ? R : E;
  return used + (R - used) / BM;
}

// The tiles of BM rows that every expert's rows need, numbered expert by expert.  A workgroup takes the offsets into LDS (off: GP_MAX_E + 1); a
// wavefront's lanes hold the running count over runs of experts, so that a tile's expert is two ballots away.  Offsets outside 0 .. R, or that fall, count
// as the nearest that do not: nothing is read or written outside the R rows.
template <int BM>
struct GroupTiles {
  const int32_t* off;
  int E, per, upto, mine;  // per: experts of a lane; upto: tiles of the lanes up to this one
  struct At {
    int e, before, tiles;  // the expert, the tiles of the experts before it, its own
  };
  __device__ __forceinline__ int tiles_of(int e) const {
    const int rows = e < E ? off[e + 1] - off[e] : 0;
    return rows > 0 ? (rows + BM - 1) / BM : 0;
  }
  __device__ __forceinline__ void init(const GroupedArgs& p, int32_t* lds, int tid, int threads) {
    for (int e = tid; e <= p.E; e += threads) {
      const int o = p.offsets[e];
      lds[e] = o < 0 ? 0 : o > p.R ? p.R : o;
    }
    __syncthreads();
    off = lds;
    E = p.E;
    per = (E + 63) >> 6;
    const int lane = tid & 63;
    mine = 0;
    for (int i = 0; i < per; ++i) mine += tiles_of(lane * per + i);
    upto = wave_scan(mine);
  }
  // all tiles times `times` (offsets that fall can make it more than was launched for)
  __device__ __forceinline__ int count(int times) const {
    const int64_t all = (int64_t)__builtin_amdgcn_readlane(upto, 63) * times;
    return all < 0x7fffffff ? (int)all : 0x7fffffff;
  }
  __device__ __forceinline__ At find(int q, int lane) const {  // q below count(1)
    const int at = __builtin_ctzll(__ballot(upto > q));
    const int e0 = at * per, before = __builtin_amdgcn_readlane(upto - mine, at);
    const int n = lane < per ? tiles_of(e0 + lane) : 0;  // (per <= 8: inside a row of 16 lanes)
    int in = n;
    in += __builtin_amdgcn_update_dpp(0, in, 0x111, 0xf, 0xf, false);
    in += __builtin_amdgcn_update_dpp(0, in, 0x112, 0xf, 0xf, false);
    in += __builtin_amdgcn_update_dpp(0, in, 0x114, 0xf, 0xf, false);
    const int sub = __builtin_ctzll(__ballot(lane < per && before + in > q));
    At a;
    a.e = e0 + sub;
    a.tiles = __builtin_amdgcn_readlane(n, sub);
    a.before = before + __builtin_amdgcn_readlane(in, sub) - a.tiles;
    return a;
  }
};
static_assert(GP_MAX_E <= 64 * 8, "a lane's run of experts");

// e^t, -150 <= t <= 87, as 2^(t log2 e) by the hardware's exponential (one step of fp32), the product's rounding taken back to first order: without
// that it is |t| log2 e half steps off.
__device__ __forceinline__ float exp_hw(float t) {
  const float y = t * 1.44269502e0f;
  const float rest = __builtin_fmaf(t, 1.92596303e-8f, __builtin_fmaf(t, 1.44269502e0f, -y));
  const float e = __builtin_amdgcn_exp2f(y);
  return __builtin_fmaf(e * 0.693147182f, rest, e);
}

// up silu(gate) of fp32 projections, which are rounded to the output's type first.  fp32: the layer's frozen arithmetic.  bf16: the same steps, as
// exact: the exponential above (within the frozen one's two steps), one sum, a quotient by the hardware's reciprocal and one correction, which for d = 1 + e^-g
// rounds it correctly but next to a tie (v_div_fixup: infinities and zeros as a division has them), and one product: 7 half steps of fp32 before
// the rounding to 2^-8.  (SwiGLU of 2000 tokens' 6 of 64, 1536 -> 1408: 94.1 us; by the frozen exponential 97.0, all of the frozen form 100.2.  A product with the reciprocal in the
// quotient's place, nothing taken back in the exponential: 91.3, and ten times as many values of h on the other side of a rounding.)
template <int OUT>
__device__ __forceinline__ float grouped_swiglu(float up, float gate) {
  if constexpr (OUT == OUT_F32) {
    return swiglu_repro(up, gate);
  } else {
    const uint32_t pair = pack_bf16x2(up, gate);
    const float u = __uint_as_float(pair << 16), g = __uint_as_float(pair & 0xffff0000u);
    const float d = 1.0f + exp_hw(__builtin_amdgcn_fmed3f(-g, -87.0f, 87.0f)), r = __builtin_amdgcn_rcpf(d), q = g * r;
    return u * __builtin_amdgcn_div_fixupf(__builtin_fmaf(__builtin_fmaf(-d, q, g), r, q), d, g);
  }
}

// grouped_walk.hip: tiles of 128 rows and 256, 128 or 64 (not SwiGLU: 128) weight rows
template <int OUT, bool SWI>
int grouped_walk_launch(const GroupedArgs& a, int width, hipStream_t st);

}  // namespace aq

#endif  // AQ_GROUPED_H
