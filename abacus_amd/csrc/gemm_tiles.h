// Tiles of a pipelined GEMM on gfx950 MFMA, as the grouped GEMMs and the products of the linear cross-entropy use them:
// MFMA operand policies, the geometry of a block tile, direct global->LDS DMA of an operand's k-tiles, fragment reads and
// the order in which a launch walks its tiles.
#pragma once

#include "common.h"

namespace abacus {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

typedef float f32x16_t __attribute__((ext_vector_type(16)));

// MFMA policies.  A fragment is 16 bytes per lane: lane l supplies row
// (l % kRows) and the VEC consecutive k at (l / kRows) * VEC of a k-block of
// kKB.  For fp32 the 4 values of a fragment feed 4 successive MFMAs (lane
// group g supplies k = 4g + j in step j; A and B agree, so the sum over k is
// complete).  Output: lane l holds column (l % kRows) and, in register q,
// row out_row(l, q).
template <typename T, int SHAPE> struct MfmaOp;
template <> struct MfmaOp<uint16_t, 32> {
  static constexpr int kRows = 32, kKB = 16, kAcc = 16;
  using Acc = f32x16_t;
  __device__ static inline void run(Acc& acc, const Vec16& a, const Vec16& b) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                  __builtin_bit_cast(bf16x8_t, b), acc, 0, 0, 0);
  }
  __device__ static inline int out_row(int lane, int q) { return 8 * (q >> 2) + 4 * (lane >> 5) + (q & 3); }
};
template <> struct MfmaOp<float, 32> {
  static constexpr int kRows = 32, kKB = 8, kAcc = 16;
  using Acc = f32x16_t;
  __device__ static inline void run(Acc& acc, const Vec16& a, const Vec16& b) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(bits_f32(a.w[j]), bits_f32(b.w[j]), acc, 0, 0, 0);
  }
  __device__ static inline int out_row(int lane, int q) { return 8 * (q >> 2) + 4 * (lane >> 5) + (q & 3); }
};

namespace pipe {

#ifndef ABACUS_PIPE_BK
#define ABACUS_PIPE_BK 64
#endif
#ifndef ABACUS_PIPE_STAGES
#define ABACUS_PIPE_STAGES 2
#endif
constexpr int BM = 256, BN = 256, BK = ABACUS_PIPE_BK, STAGES = ABACUS_PIPE_STAGES;
constexpr int CPR = BK / 8;        // 16-byte chunks per k-contiguous LDS row
static_assert(STAGES >= 2 && STAGES <= 5, "2..5 LDS stages");
constexpr int NSTEP = BK / 16;     // MFMA k-steps per k-tile
#ifndef ABACUS_PIPE_WAVES_N
#define ABACUS_PIPE_WAVES_N 2
#endif
constexpr int WAVES_M = 2, WAVES_N = ABACUS_PIPE_WAVES_N;  // wave grid over the block tile
constexpr int NWAVES = WAVES_M * WAVES_N, NT = NWAVES * 64;
constexpr int WTM = BM / WAVES_M, WTN = BN / WAVES_N;     // wave tile
constexpr int FM = WTM / 32, FN = WTN / 32;                // 32 x 32 fragments per wave
constexpr int TILE_BYTES = 256 * BK * 2;          // one operand tile: 16 KB
constexpr int STAGE_BYTES = 2 * TILE_BYTES;       // A + B
constexpr int LDC = BN + 8;                        // epilogue C tile row stride (bf16)
constexpr int LDS_BYTES = STAGES * STAGE_BYTES > BM * LDC * 2 ? STAGES * STAGE_BYTES : BM * LDC * 2;
static_assert(LDS_BYTES <= 160 * 1024, "LDS is 160 KB per work-group");
constexpr int TILE_CHUNKS = TILE_BYTES / 16;
constexpr int DMA_PER_OPERAND = TILE_CHUNKS / NT;   // 16-byte chunks per thread per operand tile
constexpr int LOADS_PER_TILE = 2 * DMA_PER_OPERAND; // DMA instructions per thread per k-tile

// Row-grouped kinds cut each expert's rows into BM-row tiles; a remainder of
// at most THIN rows goes to a thin tile of THIN rows (same MFMAs and k order,
// so the same results) instead of a mostly empty full one.  bf16 thin tiles
// keep 256 columns and a 3-stage ring of 48 KB stages: with few rows per
// expert they mostly stream weights, and a third stage doubles the DMA a CU
// keeps in flight (gate/up forward at 6 rows per expert 205 -> 184 us;
// Mixtral's remainder tiles 1889 -> 1847 us); 128-column thin tiles measured
// slower there (more, shorter weight-row segments per tile: T = 512 gate/up
// 177 -> 190 us).  fp32 thin tiles have 128 columns and 4 stages of 32 KB (the
// fp32 gate/up data gradient 3885 -> 3566 us at the mid-size layer).  Full
// tiles keep 2 stages (2 x 64 KB).
constexpr int THIN = 128;
template <typename T> constexpr int kThinN = sizeof(T) == 4 ? 128 : 256;
template <typename T> constexpr int kThinStages = sizeof(T) == 4 ? 4 : 3;
template <int BMT, typename T = uint16_t>
struct Geo {
  static_assert(BMT == BM || BMT == THIN, "full or thin tiles");
  static constexpr int WTM = BMT / WAVES_M, FM = WTM / 32;
  static constexpr int BN = BMT == BM ? pipe::BN : kThinN<T>;  // tile columns
  static constexpr int WTN = BN / WAVES_N, FN = WTN / 32;
  static constexpr int LDC = BN + 8;                           // epilogue C tile row stride (bf16)
  static constexpr int A_BYTES = BMT * BK * 2;                 // A operand tile
  static constexpr int B_BYTES = BN * BK * 2;                  // B operand tile
  static constexpr int STAGE = A_BYTES + B_BYTES;              // A + B
  static constexpr int ST = BMT == BM ? STAGES : kThinStages<T>;  // ring depth
  static constexpr int DMA_A = A_BYTES / 16 / NT, DMA_B = B_BYTES / 16 / NT;
  static constexpr int LOADS = DMA_A + DMA_B;                  // DMA instructions per thread per k-tile
  static constexpr int LDS = ST * STAGE > BMT * LDC * 2 ? ST * STAGE : BMT * LDC * 2;
};
static_assert(Geo<BM>::LDS == LDS_BYTES, "full tiles");
constexpr int kThinLds = Geo<THIN, uint16_t>::LDS > Geo<THIN, float>::LDS ? Geo<THIN, uint16_t>::LDS
                                                                          : Geo<THIN, float>::LDS;
constexpr int LDS_ALLOC = kThinLds > LDS_BYTES ? kThinLds : LDS_BYTES;
static_assert(LDS_ALLOC <= 160 * 1024, "LDS is 160 KB per work-group");

typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;

// 16 zero bytes: the DMA source for k beyond a ragged segment's end.
static __device__ __attribute__((aligned(16))) uint32_t g_zero16[4];

// kc rows are CPR chunks; 256 bytes of LDS banks hold 16 / CPR rows, so rows
// of one bank period get distinct chunk permutations.
__device__ inline int kc_off(int row, int chunk) { return (row * CPR + (chunk ^ ((row / (16 / CPR)) % CPR))) * 16; }
// The mn-contiguous tile: [k][MCC chunks] (MCC = 16-byte chunks per k row,
// 32 for a 256-wide bf16 tile), chunks XOR-swizzled per k row.  bf16: by
// (k % 4) * 4.  fp32: by groups of 8 chunks per 4 k rows, so that the two
// half-waves of a fragment read (rows k and k + 4) hit different banks.
template <typename T, int MCC> __device__ inline int mc_swz(int k);
template <> __device__ inline int mc_swz<uint16_t, 16>(int k) { return (k & 3) << 2; }
template <> __device__ inline int mc_swz<uint16_t, 32>(int k) { return (k & 3) << 2; }
template <> __device__ inline int mc_swz<float, 32>(int k) { return ((k >> 2) & 3) << 3; }
template <> __device__ inline int mc_swz<float, 64>(int k) { return ((k >> 2) & 7) << 3; }
template <typename T, int MCC>
__device__ inline int mc_off(int k, int chunk) { return (k * MCC + (chunk ^ mc_swz<T, MCC>(k))) * 16; }
// k-tile depth in elements: 128 bytes of k per row for either dtype
template <typename T> constexpr int kBKT = 128 / (int)sizeof(T);
static_assert(kBKT<uint16_t> == BK, "the bf16 k-tile");

// One operand's DMA stream.  Chunk p of an operand tile (p = 0 .. TILE_CHUNKS-1)
// is written by instruction i = p / NT of wave (p / 64) % NWAVES, lane p % 64:
//   kc: p -> (row = p / CPR, chunk = swizzle^-1(p % CPR)): element (r0 + row, k0 + 8 c)
//   mc: p -> (k = p / 32, chunk = swizzle^-1(p % 32)):    element (k0 + k, r0 + 8 c)
// Everything but k0 is fixed for a tile, so setup() computes each lane's
// source pointers once and issue() adds the k0 step (kc: k0 elements, mc:
// k0 rows) -- one 64-bit add per DMA.  Chunks whose k lies beyond k_lim
// (a ragged segment's tail) read the zero page instead.
template <typename T, bool MC, int N = DMA_PER_OPERAND, int BNT = BN>
struct DmaStream {
  static constexpr int EPC = 16 / (int)sizeof(T);        // elements per 16-byte chunk
  static constexpr int MCC = BNT * (int)sizeof(T) / 16;  // chunks per mn-contiguous k row
  const T* base[N];
  int koff[N];   // k of the chunk relative to k0
  int64_t ld;

  __device__ inline void setup(const T* b0, const T* b1, int64_t ld_, int r0, int r_lim, int wave, int lane) {
    ld = ld_;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int p = (i * NWAVES + wave) * 64 + lane;
      if (!MC) {
        const int row = p / CPR;
        const int c = (p % CPR) ^ ((row / (16 / CPR)) % CPR);
        int gr = r0 + row;
        gr = gr < r_lim ? gr : r_lim - 1;
        base[i] = b0 + (int64_t)gr * ld + c * EPC;
        koff[i] = c * EPC;
      } else {
        const int k = p / MCC;
        const int c = (p % MCC) ^ mc_swz<T, MCC>(k);
        int mn = c * EPC;
        const T* b = b0;
        if (b1 != nullptr && mn >= BNT / 2) {
          b = b1;
          mn -= BNT / 2;
        }
        int gm = r0 + mn;
        gm = gm < r_lim ? gm : r_lim - EPC;
        base[i] = b + (int64_t)k * ld + gm;
        koff[i] = k;
      }
    }
  }

  // Instruction i of this operand's k-tile at k0.  LDS destinations are
  // wave-uniform: tile + (i * NWAVES + wave) * 1024.
  template <bool MAYBE_RAGGED>
  __device__ inline void issue_one(int i, uint32_t tile, int wave_u, int k0, int k_lim) const {
    const void* src = MC ? (const void*)(base[i] + (int64_t)k0 * ld) : (const void*)(base[i] + k0);
    if (MAYBE_RAGGED && k0 + koff[i] >= k_lim) src = (const void*)g_zero16;
    dma16_to(src, tile + (uint32_t)((i * NWAVES + wave_u) * 1024));
  }
};

// 32 x 16 MFMA operand fragment (rows or columns f0 .. f0+31, k-step t of 2).
__device__ inline Vec16 frag_kc(const char* tile, int f0, int t, int lane) {
  const int r = f0 + (lane & 31);
  return *reinterpret_cast<const Vec16*>(tile + kc_off(r, 2 * t + (lane >> 5)));
}
// 32 x 16 MFMA operand fragment of an mn-contiguous tile (MCC chunks per k
// row).  fp32: lane l gets the 4 k at 8 t + 4 (l / 32) of column f0 + l % 32
// (one 32-bit read each; the MFMA's k order, as frag_kc's 16-byte chunk).
// bf16: two transposed reads (ds_read_b64_tr_b16) of 4 k each.
template <typename T, int MCC>
__device__ inline Vec16 frag_mc(const char* tile, int f0, int t, int lane) {
  Vec16 v;
  if constexpr (sizeof(T) == 4) {
    const int cc = f0 + (lane & 31), k0 = 8 * t + 4 * (lane >> 5);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v.w[j] = *reinterpret_cast<const uint32_t*>(tile + mc_off<T, MCC>(k0 + j, cc >> 2) + (cc & 3) * 4);
  } else {
    const int grp = lane >> 4, s = lane & 15;
    const int mn = f0 + 16 * (grp & 1) + 4 * (s & 3);
    const int k = 16 * t + 8 * (grp >> 1) + (s >> 2);
    const int b = (mn & 7) * 2;
    const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) v4i16*)(tile + mc_off<T, MCC>(k, mn >> 3) + b));
    const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) v4i16*)(tile + mc_off<T, MCC>(k + 4, mn >> 3) + b));
    v.w[0] = (uint16_t)lo[0] | ((uint32_t)(uint16_t)lo[1] << 16);
    v.w[1] = (uint16_t)lo[2] | ((uint32_t)(uint16_t)lo[3] << 16);
    v.w[2] = (uint16_t)hi[0] | ((uint32_t)(uint16_t)hi[1] << 16);
    v.w[3] = (uint16_t)hi[2] | ((uint32_t)(uint16_t)hi[3] << 16);
  }
  return v;
}

constexpr int GM = 8, GN = 4;


// Real tile r of mt_real row tiles x NT column tiles -> its row and column tile:
// groups of GM rows x GN columns, column group by column group, the last rows'
// and the last columns' groups short.  Every number is a real tile: a block
// without one, between others, costs more than its launch, because the dispatcher
// gives the shader engines their blocks in a fixed turn, whatever they still run.
// With NT padded to whole column groups, N = 320 (two tiles of four real) left
// half of each XCD idle (us, padded -> now): bf16 E 64 D 320 M 11456, 2135 tokens
// top-2, sliced down forward 240 -> 151; E 128 D 2048 M 768, 8192 tokens top-8,
// gate/up forward (6 of 8) 669 -> 551, down backward (3 of 4) 663 -> 608.
__device__ inline void row_tile(int r, int mt_real, int NT, int& mt, int& nt) {
  const int full = (mt_real / GM) * GM * NT;  // tiles in whole groups of GM rows
  int rows = GM, m0 = 0;
  if (r < full) {
    m0 = r / (GM * NT) * GM;
    r %= GM * NT;
  } else {
    rows = mt_real % GM;  // the short last group (nonzero when r >= full)
    m0 = mt_real / GM * GM;
    r -= full;
  }
  const int c0 = r / (rows * GN) * GN;  // this column group's first tile
  const int cols = min(GN, NT - c0);
  r -= c0 * rows;
  mt = m0 + r / cols;
  nt = c0 + r % cols;
}

// The first n (all 8 when n >= 8) bf16 of v to p, at any alignment.
__device__ inline void st8_any(uint16_t* p, const Vec16& v, int n) {
  if (n >= 8) {
    typedef uint32_t u32x4_ua __attribute__((ext_vector_type(4), aligned(2)));
    *reinterpret_cast<u32x4_ua*>(p) = u32x4_ua{v.w[0], v.w[1], v.w[2], v.w[3]};
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) p[i] = (uint16_t)(v.w[i >> 1] >> (16 * (i & 1)));
  }
}

}  // namespace pipe
}  // namespace abacus
