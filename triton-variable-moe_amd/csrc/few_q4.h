// 4-bit matrices in the order the matrix instructions take them.
//
// A value is an e2m1 float: a sign and a place among 0, 0.5, 1, 1.5, 2, 3, 4, 6
// (bits 0-2, the sign in bit 3). The hardware turns eight of them into an
// operand in four instructions, and each is exact in bf16, so a product rounds
// nothing; the scale of a group (32, 64 or 128 values of a column along the
// summed axis) multiplies the group's fp32 sum.
//
// Block (nb, kb) of a matrix: 16 columns x 128 rows, 1 KB. Lane l holds 16 bytes
// = four dwords; dword j is the operand of rows 128 kb + 32 j + 8 (l / 16) + 0..7
// of column 16 nb + l % 16, the first row in the lowest bits. The blocks of a
// column follow one another: a wave walks them as one stream. Scales: bf16
// [block][16 columns][128 / group]. Rows and columns past the matrix hold 0 (and
// a scale of 0). A stack's matrices follow one another, each from a whole block.
#pragma once

#include <type_traits>

#include "vmoe_common.h"

namespace vmoe {

constexpr int kQ4Rows = 128, kQ4Cols = 16, kQ4BlockBytes = 1024;

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// The weights of a stack of matrices: row-major bf16 or fp32 with a row stride,
// or 4-bit blocks with their scales.
struct Stack {
  const void* w;
  const uint16_t* scales;
  int64_t ld;
};

// A matrix of a stack: where it starts along the axis the matrices share
// (column of W1, row of W2), its length along it, its first block (4-bit), its
// first tile of 64 along that axis.
struct alignas(16) MatEntry {
  int32_t off, len, base, first_tile;
};

// (One 16-byte load; a struct copied under a condition would go through memory.)
__device__ __forceinline__ MatEntry load_entry(const MatEntry* p) {
  typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
  const i32x4 v = *reinterpret_cast<const i32x4*>(p);
  return {v[0], v[1], v[2], v[3]};
}
__device__ __forceinline__ void store_entry(MatEntry* p, const MatEntry& m) {
  typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<i32x4*>(p) = i32x4{m.off, m.len, m.base, m.first_tile};
}

// Eight values of a dword as bf16, the lowest bits first (exact).
__device__ __forceinline__ bf16x8_t q4_values(uint32_t codes) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  u32x4 v;
  v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.0f, 0));
  v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.0f, 1));
  v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.0f, 2));
  v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.0f, 3));
  return __builtin_bit_cast(bf16x8_t, v);
}

// Orders LDS accesses of the workgroup; global loads stay in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

}  // namespace vmoe
