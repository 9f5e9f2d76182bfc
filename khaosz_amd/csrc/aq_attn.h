// What the attention kernels share that bring rows of keys and values into LDS and multiply them on the matrix core.
#pragma once
#include "aq_common.h"

namespace aq {

typedef __bf16 pa_bf16x8 __attribute__((ext_vector_type(8)));
typedef short pa_s16x4 __attribute__((ext_vector_type(4)));
typedef float pa_f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void pa_lds_void;
typedef __attribute__((address_space(3))) pa_s16x4 pa_lds_s16x4;

__device__ const uint4 pa_zero_row[16] = {};  // what a row of an unmapped page reads as

// 16 bytes per lane from memory to LDS, 1 KiB in lane order from byte `at` (wavefront-uniform).  Written out because the compiler,
// given the builtin, waits for every such load in flight before the next LDS read of any kind -- here the other buffer's,
// requested a moment earlier.  The kernel waits itself, before the barrier that hands a buffer over.
__device__ __forceinline__ void load_row_lds(const uint16_t* src, uint32_t at) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(at) : "memory");  // m0 needs a wait state
}

// The same, the address a wavefront-uniform base and an offset in bytes.  A memory instruction that reads a scalar register which a vector
// instruction (v_readfirstlane, or v_readlane of a spilled register) has written needs 5 wait states; the compiler cannot see that this is one.
__device__ __forceinline__ void load_row_lds(const uint16_t* base, uint32_t offset, uint32_t at) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "{m0}"(at) : "memory");
}

// The 16-byte piece of row r that sits in slot s of the row is s ^ row_key(r): the low bits of r, reversed.  16 rows
// reading the same piece (K) fall on all slots of the bank lines; the 8 neighbouring rows x 64 bytes of a transposing
// read (V) are told apart by their lowest bits, which reversed move a row's pieces by 64 bytes and more.
template <int D>
__device__ __forceinline__ int row_key(int row) {
  if constexpr (D == 64)  // 128-byte rows: two to a bank line
    return (int)(__builtin_bitreverse32((uint32_t)(row >> 1) & 7u) >> 29);
  else
    return (int)(__builtin_bitreverse32((uint32_t)row & 15u) >> 28);
}

// Query heads per KV head that the decode kernels are made for.
inline bool attn_group_ok(int64_t G) { return G == 1 || G == 2 || G == 3 || G == 4 || G == 6 || G == 8; }

}  // namespace aq
