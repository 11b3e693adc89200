// What the attention kernels share: the 32 x 32 x 16 bf16 product, 64-row tiles in
// LDS and their fragments, and values combined over lanes l and l ^ 32.
#pragma once

#include "common.h"

namespace abacus {

typedef __bf16 attn_bf16x8 __attribute__((ext_vector_type(8)));
typedef float attn_f32x16 __attribute__((ext_vector_type(16)));
__device__ inline void mfma32(attn_f32x16& acc, const Vec16& a, const Vec16& b) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(attn_bf16x8, a), __builtin_bit_cast(attn_bf16x8, b),
                                                acc, 0, 0, 0);
}

// A K or V tile in LDS: 64 rows (keys) of HD / 8 16-byte chunks (dims), the chunk
// index XOR-swizzled by row.  Head dim 64: with m = row / 2, swz = (m % 2) * 4 +
// (m / 2) % 4.  Rows 2 apart land 128 bytes apart in the bank space, so a K
// fragment read (16 consecutive rows, one chunk) needs the 8 even rows of a block
// of 16 on 8 different chunks (swz is a permutation of 0..7 over them), and a V^T
// read (rows r..r+3, r a multiple of 4, chunks c..c+3 of 8) needs rows r and r+2
// on complementary halves of the chunks (swz(r+2) = swz(r) ^ 4).  Head dim 128: a
// row is a whole turn of the banks, so 16 consecutive rows need 16 different
// chunks and rows r..r+3 four different groups of 4: swz = (row % 4) * 4 +
// (row / 4) % 4.  Either way both reads are free of bank conflicts.
template <int HD> __device__ inline int tile_swz(int row) {
  return HD == 64 ? (((row >> 1) & 1) << 2) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3);
}
template <int HD> __device__ inline int tile_off(int row, int chunk) {
  return (row * (HD / 8) + (chunk ^ tile_swz<HD>(row))) * 16;
}

// K fragment (A of S^T): key `row0 + l % 32`, dims 16 c + 8 (l / 32) .. +7.
template <int HD>
__device__ inline Vec16 frag_k(const char* tile, int row0, int c, int lane) {
  return *reinterpret_cast<const Vec16*>(tile + tile_off<HD>(row0 + (lane & 31), 2 * c + (lane >> 5)));
}

// v_permlane32_swap: lanes 32..63 of a take lanes 0..31 of b, and lanes 0..31
// of b take lanes 32..63 of a (one VALU instruction, no LDS round trip).
__device__ inline void swap_halves(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}

// max and sum of a value over lanes l and l ^ 32 (the same on both lanes)
__device__ inline float pair_max(float x) {
  uint32_t a = __builtin_bit_cast(uint32_t, x), b = a;
  swap_halves(a, b);
  return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ inline float pair_sum(float x) {
  uint32_t a = __builtin_bit_cast(uint32_t, x), b = a;
  swap_halves(a, b);  // lanes < 32: (own, partner); lanes >= 32: (partner, own)
  return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}

}  // namespace abacus
