// Cross-entropy of a linear head, x W against targets, with the gradients of both operands: the logits never whole in
// memory.  No counterpart in the reference, whose head and loss are two steps (transformer_moe.py:75,
// trainer.py:77-85).
//
//   l = x W  (fp32),   lse_t = log sum_v exp l_tv,   loss_t = lse_t - l[t, target_t]
//   P_tv = s_t (exp(l_tv - lse_t) - [v = target_t]),   dx = P W^T,   dw = x^T P
//
// s_t is 1 / kept rows (mean), 1 (sum) or a weight of each row.  Rows whose target is ignore_index are left out before
// any product: the kept rows are packed (their count stays on the device) and every launch ends at that count, so a
// batch of prompts costs what its answers cost.
//
// One pass over a chunk of kept rows (all of them while their P takes at most kChunkBytes):
//   1. logits: a tile of x W stays in registers; of each row and strip of columns its maximum m and the sum of
//      exp(l - m) go out, and with gradients exp(l - m) itself, in 16 bits of which 10 are mantissa for bf16
//      operands (it is in [0, 1], so 6 bits of exponent and no sign do; rounded four times finer than P).
//   2. rows: the strips' (m, sum) joined to lse and the loss; P in place of the exponentials, rounded once to the
//      operands' type, which the matrix instructions take.
//   3. dx and dw: two products on P.  Where their tiles are fewer than the CUs, slices of the reduction in fp32,
//      added in slice order.  Over several chunks dw adds up in fp32.
// So 6 n D V operations of matrix products in all: the logits are not computed again for the gradient.
#include <algorithm>
#include <type_traits>

#include "gemm_tiles.h"

namespace abacus {
namespace {

using namespace pipe;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kCUs = 256;
constexpr int64_t kChunkBytes = 1ll << 30;       // of P, or of the strips' statistics where there is no P
constexpr int kUnits = 512;                       // tiles x slices of a sliced product at most
constexpr int kSlices = 16;
constexpr int kReduceRows = 16;                   // rows of a tile that a block of the adding pass takes

enum Kind : int { kLogits = 0, kDx = 1, kDw = 2 };

struct LceArgs {
  const void* x;
  int64_t x_stride;
  const void* w;          // (D, ldv)
  const int64_t* targets;
  int64_t ignore_index;
  int T, D, V, Dp, Vp;    // Dp, Vp: whole vectors; also the pitches of xc, P and the padded w
  int64_t ldv;
  int chunk, chunk_rows;  // this chunk's number, rows a chunk
  int chunks;
  int reduction;          // ABACUS_LOSS_*
  int grad;               // P is wanted
  const float* row_grad;  // weights of the rows, or NULL
  float* loss;
  void* dx;               // NULL: not wanted
  void* dw;
  // workspace
  int* kept;              // one int: the number of kept rows
  int* idx;               // kept row -> row
  int* tgt;               // kept row -> target (-1: outside the vocabulary)
  float* target_logit;    // of each kept row; NaN until its strip writes it
  float* row_loss;        // of each kept row
  void* xc;               // kept rows of x
  float2* stats;          // (strip, chunk row): maximum, sum
  void* p;                // (chunk rows, Vp)
  float* acc;             // dw over several chunks
  float* parts;           // tiles of a sliced product
};

template <typename T> constexpr int kVec = VecTraits<T>::kN;
// columns of one wave: a row's statistics go by these strips
template <typename T, int BMT> constexpr int kStrip = Geo<BMT, T>::WTN;

__device__ inline int chunk_kept(const LceArgs& a) {
  return max(0, min(a.chunk_rows, *a.kept - a.chunk * a.chunk_rows));
}

// About what a tile's k-tile takes (us, with every CU at work), and its prologue and epilogue.
template <typename T, int BMT> constexpr float kTileUs = sizeof(T) == 2 ? (BMT == BM ? 1.9f : 1.15f) : (BMT == BM ? 7.0f : 1.9f);
template <int KIND, int BMT> constexpr float kEndsUs = (BMT == BM ? 8.f : 4.f) * (KIND == kLogits ? 1.5f : 1.f);

// The time of a product cut into `slices` of its reduction: rounds of the CUs, and for partial tiles another launch
// and their way out and back at 4 TB/s.
template <typename T, int KIND, int BMT>
__host__ __device__ inline float product_us(int64_t tiles, int ktiles, int slices) {
  const float rounds = (float)((tiles * slices + kCUs - 1) / kCUs);
  const float us = rounds * ((float)((ktiles + slices - 1) / slices) * kTileUs<T, BMT> + kEndsUs<KIND, BMT>);
  return slices == 1 ? us : us + 6.f + (float)(tiles * slices) * (BMT * Geo<BMT, T>::BN * 4) * 2.f / 4.0e6f;
}
template <typename T, int KIND, int BMT>
__host__ __device__ inline int slices_of(int64_t tiles, int ktiles) {
  int best = 1;
  if constexpr (KIND != kLogits) {
    float least = product_us<T, KIND, BMT>(tiles, ktiles, 1);
    for (int s = 2; s <= kSlices && tiles * s <= kUnits && ktiles >= 4 * s; ++s) {
      const float us = product_us<T, KIND, BMT>(tiles, ktiles, s);
      if (us < least) {
        least = us;
        best = s;
      }
    }
  }
  return best;
}

// ---------------------------------------------------------------- packing the kept rows

// A block takes rows_per rows: it counts the kept rows before them, so that no block waits for another, and copies
// its kept rows to their places; the rows left out get a gradient of 0.
template <typename T>
__global__ __launch_bounds__(256) void pack_rows_kernel(LceArgs a, int rows_per) {
  constexpr int VEC = kVec<T>;
  extern __shared__ int place_s[];  // rows_per
  __shared__ int wave_s[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row0 = blockIdx.x * rows_per, rows = min(rows_per, a.T - row0);
  int before = 0;
  for (int i = tid; i < row0; i += 256) before += a.targets[i] != a.ignore_index;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) before += __shfl_xor(before, off, 64);
  if (lane == 0) wave_s[wave] = before;
  __syncthreads();
  before = wave_s[0] + wave_s[1] + wave_s[2] + wave_s[3];
  if (wave == 0) {
    for (int r0 = 0; r0 < rows; r0 += 64) {
      const int r = r0 + lane;
      const int64_t t = r < rows ? a.targets[row0 + r] : a.ignore_index;
      const bool kept = r < rows && t != a.ignore_index;
      const uint64_t mask = __ballot(kept);
      const int at = before + __popcll(mask & ((1ull << lane) - 1));
      if (r < rows) place_s[r] = kept ? at : -1;
      if (kept) {
        a.idx[at] = row0 + r;
        a.tgt[at] = t >= 0 && t < a.V ? (int)t : -1;
        a.target_logit[at] = __builtin_nanf("");
      }
      before += __popcll(mask);
    }
    if (lane == 0 && row0 + rows == a.T) *a.kept = before;
  }
  __syncthreads();
  const bool whole = a.D == a.Dp && a.x_stride % VEC == 0 && (uintptr_t)a.x % 16 == 0;
  for (int r = wave; r < rows; r += 4) {
    const int at = place_s[r];
    const T* src = (const T*)a.x + (int64_t)(row0 + r) * a.x_stride;
    if (at < 0) {
      if (a.reduction == ABACUS_LOSS_ROWS && a.loss && lane == 0) a.loss[row0 + r] = 0.f;
      if (!a.dx) continue;
      T* dx = (T*)a.dx + (int64_t)(row0 + r) * a.D;
      if (a.D == a.Dp) {
        for (int c = lane * VEC; c < a.D; c += 64 * VEC) st16(dx + c, zero16());
      } else {
        for (int c = lane; c < a.D; c += 64) dx[c] = from_f32<T>(0.f);
      }
      continue;
    }
    T* dst = (T*)a.xc + (int64_t)at * a.Dp;
    if (whole) {
      for (int c = lane * VEC; c < a.D; c += 64 * VEC) st16(dst + c, ld16(src + c));
    } else {
      for (int c = lane; c < a.Dp; c += 64) dst[c] = c < a.D ? src[c] : from_f32<T>(0.f);
    }
  }
}

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

// The vector at column c of a row of V values (V at least a vector), zeros past its end.  One load, always in bounds: near the
// row's end that of its last vector, shifted.
template <typename T>
__device__ inline Vec16 load_end(const T* row, int c, int V) {
  constexpr int VEC = kVec<T>, BITS = 8 * (int)sizeof(T);
  const int at = min(c, V - VEC);
  const u32x4_any v = *reinterpret_cast<const u32x4_any*>(row + at);
  uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
  if (at < c) {
    int sh = min(c - at, VEC) * BITS;
    if (sh >= 64) {
      lo = sh < 128 ? hi : 0;
      hi = 0;
      sh -= 64;
    }
    if (sh > 0 && sh < 64) {
      lo = lo >> sh | hi << (64 - sh);
      hi >>= sh;
    }
  }
  Vec16 o;
  o.w[0] = (uint32_t)lo;
  o.w[1] = (uint32_t)(lo >> 32);
  o.w[2] = (uint32_t)hi;
  o.w[3] = (uint32_t)(hi >> 32);
  return o;
}

// w's rows of V values at a pitch of whole vectors, zeros behind them.  A thread takes a column of kPadRows vectors, so
// that as many loads are in flight (2048 x 50257 bf16: 110 us a vector at a time).
constexpr int kPadRows = 8;
template <typename T>
__global__ __launch_bounds__(256) void pad_w_kernel(const T* __restrict__ w, int D, int V, int Vp, T* __restrict__ out) {
  constexpr int VEC = kVec<T>;
  const int c = ((int)blockIdx.x * 256 + threadIdx.x) * VEC, row0 = blockIdx.y * kPadRows;
  if (c >= Vp) return;
  Vec16 v[kPadRows];
#pragma unroll
  for (int r = 0; r < kPadRows; ++r) {
    const T* row = w + (int64_t)min(row0 + r, D - 1) * V;
    if (V >= VEC) {
      v[r] = load_end<T>(row, c, V);
    } else {
      T e[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) e[k] = k < V ? row[k] : from_f32<T>(0.f);
      __builtin_memcpy(&v[r], e, 16);
    }
  }
#pragma unroll
  for (int r = 0; r < kPadRows; ++r)
    if (row0 + r < D) st16(out + (int64_t)(row0 + r) * Vp + c, v[r]);
}

// ---------------------------------------------------------------- the products

// exp(l - m) in [0, 1] as 16 bits: 6 of exponent (2^-63 and less is 0) and 10 of mantissa, two values a word.
__device__ inline uint32_t encode2(float a, float b) {
  constexpr uint32_t kBias = (64u << 23) - 0x1000u;  // with half a step, so that the shift rounds
  const uint32_t x = __builtin_elementwise_sub_sat(f32_bits(a), kBias);
  const uint32_t y = __builtin_elementwise_sub_sat(f32_bits(b), kBias);
  return (x >> 13) | (y >> 13 << 16);
}
__device__ inline float decode(uint32_t h) { return h ? bits_f32((h << 13) + (64u << 23)) : 0.f; }

// acc[i][j] += A B over the k-tiles kbase .. kbase + ktiles - 1: the operands' tiles come by DMA into a ring of LDS
// stages, the matrix instructions of one k-step cover the fragment reads of the next, and the last step's the DMA.
template <typename T, bool A_MC, bool B_NC, int BMT, bool RK>
struct TileProduct {
  using Op = MfmaOp<T, 32>;
  using GE = Geo<BMT, T>;
  static constexpr int FM = GE::FM, FN = GE::FN, WTM = GE::WTM, WTN = GE::WTN, ST = GE::ST;
  static constexpr int MCC_A = BMT * (int)sizeof(T) / 16, MCC_B = GE::BN * (int)sizeof(T) / 16;
  static constexpr int BKT = kBKT<T>;
  using Acc = typename Op::Acc;

  static __device__ __attribute__((always_inline)) inline void run(Acc (&acc)[FM][FN], const T* A, int64_t lda, int row0, int a_lim, const T* B,
                                    int64_t ldb, int n0, int b_lim, int kbase, int ktiles, int k_lim, int wave_rows,
                                    char* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave / WAVES_N, wn = wave % WAVES_N;
    const int wave_u = __builtin_amdgcn_readfirstlane(wave);
    DmaStream<T, A_MC, GE::DMA_A, BMT> sa;
    DmaStream<T, B_NC, GE::DMA_B, GE::BN> sb;
    sa.setup(A, nullptr, lda, row0, a_lim, wave, lane);
    sb.setup(B, nullptr, ldb, n0, b_lim, wave, lane);
    const uint32_t lds32 = lds_addr32(lds);
    uint32_t stage = lds32;
    int k0 = 0;
    auto prep = [&](int kt) __attribute__((always_inline)) {
      stage = lds32 + (uint32_t)((kt % ST) * GE::STAGE);
      k0 = (kt + kbase) * BKT;
    };
    auto dma = [&](int n) __attribute__((always_inline)) {
      if (n < GE::DMA_A) sa.template issue_one<RK>(n, stage, wave_u, k0, k_lim);
      else sb.template issue_one<RK>(n - GE::DMA_A, stage + GE::A_BYTES, wave_u, k0, k_lim);
    };
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int q = 0; q < Op::kAcc; ++q) acc[i][j][q] = 0.f;
    if (ktiles <= 0) return;

    constexpr int NFRAG = FM + FN, MF = FM * FN;
    static_assert(MF >= NFRAG, "one fragment read per MFMA at most");
    Vec16 af[2][FM], bf[2][FN];
    auto read_frag = [&](const char* st, int t, int slot, int f) __attribute__((always_inline)) {
      if (f == 0 || f > FN) {
        const int i = f == 0 ? 0 : f - FN;
        af[slot][i] = A_MC ? frag_mc<T, MCC_A>(st, wm * WTM + i * 32, t, lane) : frag_kc(st, wm * WTM + i * 32, t, lane);
      } else {
        const int j = f - 1;
        bf[slot][j] = B_NC ? frag_mc<T, MCC_B>(st + GE::A_BYTES, wn * WTN + j * 32, t, lane)
                           : frag_kc(st + GE::A_BYTES, wn * WTN + j * 32, t, lane);
      }
    };
    // LF: how many of the wave's row fragments hold rows of the product
    auto kstep = [&](auto lfc, int slot, bool with_read, const char* rd, int rd_t, int rd_slot, bool with_dma)
                     __attribute__((always_inline)) {
      constexpr int LF = decltype(lfc)::value;
#pragma unroll
      for (int m = 0; m < MF; ++m) {
        // operands swapped: a fragment is C^T, so a lane holds runs of 4 columns of one row
        if (m / FN < LF) Op::run(acc[m / FN][m % FN], bf[slot][m % FN], af[slot][m / FN]);
        if (with_read && m < NFRAG) read_frag(rd, rd_t, rd_slot, m);
        if (with_dma) {
#pragma unroll
          for (int n = m * GE::LOADS / MF; n < (m + 1) * GE::LOADS / MF; ++n) dma(n);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // at most `later` k-tiles' DMA may still be in flight
    auto wait_for = [&](int later) __attribute__((always_inline)) {
      if (ST >= 4 && later >= 3) wait_vmcnt<(ST >= 4 ? 3 : 0) * GE::LOADS>();
      else if (ST >= 3 && later >= 2) wait_vmcnt<(ST >= 3 ? 2 : 0) * GE::LOADS>();
      else if (later >= 1) wait_vmcnt<GE::LOADS>();
      else wait_vmcnt<0>();
    };
    auto ktile = [&](auto lfc, int kt, bool next, bool dma_next) __attribute__((always_inline)) {
      const char* st = lds + (kt % ST) * GE::STAGE;
      const char* st_next = lds + ((kt + 1) % ST) * GE::STAGE;
#pragma unroll
      for (int t = 0; t < NSTEP - 1; ++t) kstep(lfc, t & 1, true, st, t + 1, (t + 1) & 1, false);
      wait_for(min(ST - 2, ktiles - 2 - kt));
      __builtin_amdgcn_s_waitcnt(0xc07f);  // this wave's reads of the stage are back: it may be refilled
      __syncthreads();
      if (dma_next) prep(kt + ST);
      __builtin_amdgcn_sched_barrier(0);
      kstep(lfc, (NSTEP - 1) & 1, next, st_next, 0, 0, dma_next);
    };
#pragma unroll
    for (int p = 0; p < ST; ++p)
      if (p < ktiles) {
        prep(p);
#pragma unroll
        for (int n = 0; n < GE::LOADS; ++n) dma(n);
      }
    wait_for(min(ST, ktiles) - 1);
    __syncthreads();
#pragma unroll
    for (int f = 0; f < NFRAG; ++f) read_frag(lds, 0, 0, f);
    auto run_tiles = [&](auto lfc) __attribute__((always_inline)) {
      int kt = 0;
      for (; kt + ST < ktiles; ++kt) ktile(lfc, kt, true, true);
      for (; kt + 1 < ktiles; ++kt) ktile(lfc, kt, true, false);
      ktile(lfc, kt, false, false);
    };
    // few rows fill one fragment of a thin tile, or none of a wave's
    if (FM > 2 || wave_rows > 32) run_tiles(std::integral_constant<int, FM>());
    else if (wave_rows > 0) run_tiles(std::integral_constant<int, 1>());
    else run_tiles(std::integral_constant<int, 0>());
  }
};

// n (at most VEC) values to p at any alignment of T.
template <typename T>
__device__ inline void store_any(T* p, const float* f, int n) {
  if constexpr (sizeof(T) == 2) {
    Vec16 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v.w[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
    st8_any(p, v, n);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = f[i];
  }
}

// VEC finished values of a gradient at (row, col) of dx or dw; whole: rows of it are whole vectors.
template <typename T, int KIND>
__device__ inline void store_grad(const LceArgs& a, int row, int col, const float* f, bool whole) {
  const int N = KIND == kDx ? a.D : a.V;
  T* out = KIND == kDx ? (T*)a.dx + (int64_t)a.idx[a.chunk * a.chunk_rows + row] * N + col : (T*)a.dw + (int64_t)row * N + col;
  if (whole) {
    Vec16 v;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v.w[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v.w[i] = f32_bits(f[i]);
    }
    st16(out, v);
  } else {
    store_any<T>(out, f, N - col);
  }
}

// What a product's launch covers: tiles of rows x tiles of columns x slices.
template <typename T, int KIND, int BMT>
struct Cover {
  int M, N, K, ktiles, mt, nt, slices;
  __device__ inline Cover(const LceArgs& a, int n) {
    M = KIND == kDw ? a.D : n;
    N = KIND == kDx ? a.D : a.V;
    K = KIND == kLogits ? a.D : KIND == kDx ? a.Vp : n;
    ktiles = (K + kBKT<T> - 1) / kBKT<T>;
    mt = (M + BMT - 1) / BMT;
    nt = (N + Geo<BMT, T>::BN - 1) / Geo<BMT, T>::BN;
    // (over several chunks dw's tiles are cut alike in each, as their sums go from one to the next)
    const int most = KIND == kDw && a.chunks > 1 ? (a.chunk_rows + kBKT<T> - 1) / kBKT<T> : ktiles;
    slices = slices_of<T, KIND, BMT>((int64_t)mt * nt, most);
  }
};

template <typename T, int KIND, int BMT, bool RK>
__global__ __launch_bounds__(NT, 1) void lce_product_kernel(LceArgs a) {
  using GE = Geo<BMT, T>;
  using TP = TileProduct<T, KIND == kDw, KIND != kDx, BMT, RK>;
  constexpr int FM = GE::FM, FN = GE::FN, WTM = GE::WTM, WTN = GE::WTN, BN = GE::BN, VEC = kVec<T>;
  __shared__ __attribute__((aligned(1024))) char lds[LDS_ALLOC];
  const int kept = *a.kept, n = chunk_kept(a);
  if (n == 0 && (KIND != kDw || a.chunk > 0)) return;  // (dw of no rows at all is 0)
  const Cover<T, KIND, BMT> cv(a, n);
  const int units = cv.mt * cv.nt * cv.slices, per = (units + 7) / 8;
  const int u = (blockIdx.x & 7) * per + (blockIdx.x >> 3);  // an equal contiguous share for each XCD
  if ((int)(blockIdx.x >> 3) >= per || u >= units) return;
  const int r = u / cv.slices, slice = u - r * cv.slices;
  int mt, nt;
  row_tile(r, cv.mt, cv.nt, mt, nt);
  const int row0 = mt * BMT, n0 = nt * BN;
  const int kper = (cv.ktiles + cv.slices - 1) / cv.slices, kbase = slice * kper;
  const int ktiles = max(0, min(kper, cv.ktiles - kbase));

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave / WAVES_N, wn = wave % WAVES_N;
  const int wave_rows = __builtin_amdgcn_readfirstlane(cv.M - row0 - wm * WTM);
  const T* xc = (const T*)a.xc + (int64_t)a.chunk * a.chunk_rows * a.Dp;
  const T* p = (const T*)a.p;
  const T* w = (const T*)a.w;
  typename TP::Acc acc[FM][FN];
  if constexpr (KIND == kLogits)
    TP::run(acc, xc, a.Dp, row0, n, w, a.ldv, n0, a.Vp, kbase, ktiles, cv.K, wave_rows, lds);
  else if constexpr (KIND == kDx)
    TP::run(acc, p, a.Vp, row0, n, w, a.ldv, n0, a.D, kbase, ktiles, cv.K, wave_rows, lds);
  else
    TP::run(acc, xc, a.Dp, row0, a.Dp, p, a.Vp, n0, a.Vp, kbase, ktiles, cv.K, wave_rows, lds);

  // Fragment (i, j): lane l has row l % 32 and columns 8 g + 4 (l / 32) .. +3 for g = 0..3.
  const int rl = lane & 31, ch = 4 * (lane >> 5);
  if constexpr (KIND == kLogits) {
    const int strip = n0 / WTN + wn, first = n0 + wn * WTN;
    uint16_t* tile = reinterpret_cast<uint16_t*>(lds);  // bf16: the exponentials' tile on its way out
    constexpr int LDC = GE::LDC, CV = BN / VEC;
    __syncthreads();  // every fragment read is done
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int row = row0 + wm * WTM + i * 32 + rl;
      float l[FN][16];
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int q = 0; q < 16; ++q) l[j][q] = acc[i][j][q];
      if (n0 + BN > a.V) {  // columns past the vocabulary are no logits
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int q = 0; q < 16; ++q)
            if (first + j * 32 + 8 * (q >> 2) + ch + (q & 3) >= a.V) l[j][q] = -__builtin_inff();
      }
      if (row < n) {
        const int t = a.tgt[a.chunk * a.chunk_rows + row] - first;
        if (t >= 0 && t < WTN && ((t >> 2) & 1) == (lane >> 5)) {
          float at = 0.f;
#pragma unroll
          for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) at = t == j * 32 + 8 * (q >> 2) + ch + (q & 3) ? l[j][q] : at;
          a.target_logit[a.chunk * a.chunk_rows + row] = at;
        }
      }
      float m = l[0][0];
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int q = 0; q < 16; ++q) m = fmaxf(m, l[j][q]);
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      const float m2 = fmaxf(m * kLog2e, -3.0e38f);  // (finite in a strip of -inf, whose exponentials are 0)
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float e[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            e[k] = __builtin_amdgcn_exp2f(__builtin_fmaf(l[j][4 * g + k], kLog2e, -m2));
            s += e[k];
          }
          if (!a.grad) continue;
          if constexpr (sizeof(T) == 2) {
            *reinterpret_cast<uint2*>(tile + (wm * WTM + i * 32 + rl) * LDC + wn * WTN + j * 32 + 8 * g + ch) =
                make_uint2(encode2(e[0], e[1]), encode2(e[2], e[3]));
          } else if (row < n && first + j * 32 + 8 * g + ch < a.Vp) {
            // (fp32: 16 bytes of a row a lane; its tile is larger than LDS)
            *reinterpret_cast<float4*>((float*)a.p + (int64_t)row * a.Vp + first + j * 32 + 8 * g + ch) =
                make_float4(e[0], e[1], e[2], e[3]);
          }
        }
      s += __shfl_xor(s, 32, 64);
      if (row < n && lane < 32 && first < a.V) a.stats[(int64_t)strip * a.chunk_rows + row] = make_float2(m2, s);
    }
    if (!a.grad) return;
    if constexpr (sizeof(T) == 2) {
      __syncthreads();
#pragma unroll 8
      for (int v = tid; v < BMT * CV; v += NT) {
        const int row = row0 + v / CV, col = n0 + v % CV * VEC;
        if (row < n && col < a.Vp) st16((uint16_t*)a.p + (int64_t)row * a.Vp + col, ld16(tile + v / CV * LDC + v % CV * VEC));
      }
    }
  }

  if constexpr (KIND != kLogits) {
    __syncthreads();  // every fragment read is done: the tile goes out through the stages' LDS
    if (cv.slices > 1) {  // a slice's fp32 tile, for lce_reduce_kernel
      float* out = a.parts + (int64_t)u * (BMT * BN);
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<float4*>(out + (wm * WTM + i * 32 + rl) * BN + wn * WTN + j * 32 + 8 * g + ch) =
                make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
      return;
    }
    // dw over several chunks: the sum so far, in the fragments' own order, whole lines a wave
    const float4* sum = nullptr;
    if (KIND == kDw && a.chunk > 0) sum = reinterpret_cast<const float4*>(a.acc) + (int64_t)r * (BMT * BN / 4) + tid;
    auto value = [&](int i, int j, int g) __attribute__((always_inline)) {
      float4 v = make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
      if (KIND == kDw && sum) {
        const float4 x = sum[((i * FN + j) * 4 + g) * NT];
        v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
      }
      return v;
    };
    if (KIND == kDw && a.chunks > 1 && (a.chunk + 1) * (int64_t)a.chunk_rows < kept) {  // more to come
      float4* to = reinterpret_cast<float4*>(a.acc) + (int64_t)r * (BMT * BN / 4) + tid;
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int g = 0; g < 4; ++g) to[((i * FN + j) * 4 + g) * NT] = value(i, j, g);
      return;
    }
    // fp32 bands of RB rows through LDS: whole rows of vectors go out
    constexpr int RB = 128, LDB = BN + 4, CV = BN / VEC;
    static_assert(BMT % RB == 0 && (WTM % RB == 0 || RB % WTM == 0) && RB * LDB * 4 <= LDS_ALLOC, "bands of wave rows");
    float* band = reinterpret_cast<float*>(lds);
    const bool whole = KIND == kDx ? a.D == a.Dp : a.V == a.Vp;
#pragma unroll
    for (int pb = 0; pb < BMT / RB; ++pb) {
      if (wm * WTM / RB == pb) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g)
              *reinterpret_cast<float4*>(band + (wm * WTM - pb * RB + i * 32 + rl) * LDB + wn * WTN + j * 32 + 8 * g + ch) =
                  value(i, j, g);
      }
      __syncthreads();
      for (int v = tid; v < RB * CV; v += NT) {
        const int row = row0 + pb * RB + v / CV, col = n0 + v % CV * VEC;
        const float* src = band + v / CV * LDB + v % CV * VEC;
        if (row < cv.M && col < cv.N) {
          float f[VEC];
#pragma unroll
          for (int k = 0; k < VEC; k += 4) *reinterpret_cast<float4*>(f + k) = *reinterpret_cast<const float4*>(src + k);
          store_grad<T, KIND>(a, row, col, f, whole);
        }
      }
      if (pb + 1 < BMT / RB) __syncthreads();
    }
  }
}

// The slices of a product's tiles added in slice order.
template <typename T, int KIND, int BMT>
__global__ __launch_bounds__(256) void lce_reduce_kernel(LceArgs a) {
  constexpr int BN = Geo<BMT, T>::BN, VEC = kVec<T>, CV = BN / VEC;
  const int kept = *a.kept, n = chunk_kept(a);
  if (n == 0) return;
  const Cover<T, KIND, BMT> cv(a, n);
  if (cv.slices <= 1) return;
  const int r = blockIdx.x / (BMT / kReduceRows), band = blockIdx.x % (BMT / kReduceRows);
  if (r >= cv.mt * cv.nt) return;
  int mt, nt;
  row_tile(r, cv.mt, cv.nt, mt, nt);
  const float* tile = a.parts + (int64_t)r * cv.slices * (BMT * BN);
  const bool whole = KIND == kDx ? a.D == a.Dp : a.V == a.Vp;
  for (int v = threadIdx.x; v < kReduceRows * CV; v += 256) {
    const int tr = band * kReduceRows + v / CV, tc = v % CV * VEC;
    const int row = mt * BMT + tr, col = nt * BN + tc;
    if (row >= cv.M || col >= cv.N) continue;
    float f[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) f[k] = 0.f;
    for (int s = 0; s < cv.slices; ++s) {
      const float* src = tile + (int64_t)s * (BMT * BN) + tr * BN + tc;
#pragma unroll
      for (int k = 0; k < VEC; k += 4) {
        const float4 x = *reinterpret_cast<const float4*>(src + k);
        f[k] += x.x;
        f[k + 1] += x.y;
        f[k + 2] += x.z;
        f[k + 3] += x.w;
      }
    }
    if (KIND == kDw && a.chunks > 1) {  // the sum over the chunks so far, at the tile's place
      float* sum = a.acc + (int64_t)r * (BMT * BN) + tr * BN + tc;
      const bool done = (a.chunk + 1) * (int64_t)a.chunk_rows >= kept;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        if (a.chunk > 0) f[k] += sum[k];
        if (!done) sum[k] = f[k];
      }
      if (!done) continue;
    }
    store_grad<T, KIND>(a, row, col, f, whole);
  }
}

// ---------------------------------------------------------------- the rows' losses and P

// Rows of a block.  The strips' statistics of kRowsB rows are joined by 256 / kRowsB threads a row; then P takes the
// place of the exponentials, P = exp(l - m) * (s exp(m - top) / sum), at the target s (p - 1) from its fp32 logit.
constexpr int kRowsB = 8;
constexpr int kStripsB = 512;  // strips whose factors are in LDS at a time
constexpr int kAheadB = 4;     // vectors of a thread in flight

template <typename T>
__global__ __launch_bounds__(256) void lce_rows_kernel(LceArgs a, int strip) {
  constexpr int VEC = kVec<T>, G = 256 / kRowsB;
  __shared__ float2 part_s[G][kRowsB];
  __shared__ float2 row_s[kRowsB];  // maximum, 1 / sum
  __shared__ float factor_s[kStripsB];
  const int tid = threadIdx.x, n = chunk_kept(a), row0 = blockIdx.x * kRowsB, base = a.chunk * a.chunk_rows;
  if (row0 >= n) return;
  const int strips = (a.V + strip - 1) / strip;
  {
    const int r = tid % kRowsB, g = tid / kRowsB, row = min(row0 + r, n - 1);
    float m = -__builtin_inff(), s = 0.f;
    for (int k = g; k < strips; k += G) {
      const float2 st = a.stats[(int64_t)k * a.chunk_rows + row];
      const float top = fmaxf(m, st.x);
      s = s * __builtin_amdgcn_exp2f(m - top) + st.y * __builtin_amdgcn_exp2f(st.x - top);
      m = top;
    }
    part_s[g][r] = make_float2(m, s);
  }
  __syncthreads();
  if (tid < kRowsB) {
    float m = -__builtin_inff(), s = 0.f;
    for (int g = 0; g < G && g < strips; ++g) {
      const float2 st = part_s[g][tid];
      const float top = fmaxf(m, st.x);
      s = s * __builtin_amdgcn_exp2f(m - top) + st.y * __builtin_amdgcn_exp2f(st.x - top);
      m = top;
    }
    row_s[tid] = make_float2(m, 1.0f / s);
    const int row = row0 + tid;
    if (row < n) {
      // the target's distance from the maximum first: it is small where the loss is
      const float l = kLn2 * (__builtin_amdgcn_logf(s) + __builtin_fmaf(-a.target_logit[base + row], kLog2e, m));
      if (a.reduction == ABACUS_LOSS_ROWS) {
        if (a.loss) a.loss[a.idx[base + row]] = l;
      } else {
        a.row_loss[base + row] = l;
      }
    }
  }
  if (!a.grad) return;
  __syncthreads();
  const int kept = *a.kept;
  for (int r = 0; r < min(kRowsB, n - row0); ++r) {
    const int row = row0 + r;
    const float top = row_s[r].x, inv = row_s[r].y;
    const float s = a.row_grad ? a.row_grad[a.idx[base + row]] : a.reduction == ABACUS_LOSS_MEAN ? 1.0f / (float)kept : 1.0f;
    const int t = a.tgt[base + row];
    T* p = (T*)a.p + (int64_t)row * a.Vp;
    for (int k0 = 0; k0 < strips; k0 += kStripsB) {
      __syncthreads();
      for (int k = tid; k < min(kStripsB, strips - k0); k += 256)
        factor_s[k] = s * inv * __builtin_amdgcn_exp2f(a.stats[(int64_t)(k0 + k) * a.chunk_rows + row].x - top);
      __syncthreads();
      const int end = min(a.Vp, (k0 + kStripsB) * strip);
      for (int c0 = k0 * strip + tid * VEC; c0 < end; c0 += 256 * VEC * kAheadB) {
        Vec16 e[kAheadB];
#pragma unroll
        for (int u = 0; u < kAheadB; ++u) e[u] = ld16(p + min(c0 + u * 256 * VEC, a.Vp - VEC));
#pragma unroll
        for (int u = 0; u < kAheadB; ++u) {
          const int c = c0 + u * 256 * VEC;
          if (c >= end) break;
          const float f = factor_s[c / strip - k0];
          float o[VEC];
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            if constexpr (sizeof(T) == 2) o[k] = f * decode(k & 1 ? e[u].w[k >> 1] >> 16 : e[u].w[k >> 1] & 0xffffu);
            else o[k] = f * bits_f32(e[u].w[k]);
          }
          if (t >= c && t < c + VEC) {
            const float pt = inv * __builtin_amdgcn_exp2f(__builtin_fmaf(a.target_logit[base + row], kLog2e, -top));
#pragma unroll
            for (int k = 0; k < VEC; ++k) o[k] = t == c + k ? s * (pt - 1.0f) : o[k];
          }
          Vec16 out;
          if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int k = 0; k < 4; ++k) out.w[k] = pack_bf16x2(o[2 * k], o[2 * k + 1]);
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) out.w[k] = f32_bits(o[k]);
          }
          st16(p + c, out);
        }
      }
    }
  }
}

// The kept rows' losses added in a fixed order, in fp64.
__global__ __launch_bounds__(1024) void lce_sum_kernel(LceArgs a) {
  __shared__ double sum_s[16];
  const int kept = *a.kept, tid = threadIdx.x;
  double s = 0.0;
  for (int i = tid; i < kept; i += 1024) s += (double)a.row_loss[i];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if ((tid & 63) == 0) sum_s[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < 16; ++i) s += sum_s[i];
    a.loss[0] = (float)(a.reduction == ABACUS_LOSS_MEAN ? s / (double)kept : s);
  }
}

// t *= *g, left alone where *g is 1.
template <typename T>
__global__ __launch_bounds__(256) void scale_kernel(T* __restrict__ t, int64_t n, const float* __restrict__ g) {
  const float f = *g;
  if (f == 1.0f) return;
  constexpr int VEC = kVec<T>;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * VEC; i < n; i += (int64_t)gridDim.x * 256 * VEC) {
    if (i + VEC <= n) {
      Vec16 v = ld16(t + i);
#pragma unroll
      for (int k = 0; k < VEC; ++k) VecTraits<T>::set(v, k, f * VecTraits<T>::get(v, k));
      st16(t + i, v);
    } else {
      for (int64_t k = i; k < n; ++k) t[k] = from_f32<T>(f * to_f32<T>(t[k]));
    }
  }
}

// ---------------------------------------------------------------- host

struct Plan {
  int Dp, Vp, chunk_rows, chunks, strip;
  bool thin[3], pad;  // thin: of each kind's tiles
  int64_t kept, idx, tgt, target_logit, row_loss, xc, w, stats, p, acc, parts, total;
};

template <typename T, int KIND, int BMT>
struct Sizes {
  int64_t tiles;
  int ktiles;
  Sizes(int64_t rows, int64_t D, int64_t V) {
    const int64_t M = KIND == kDw ? D : rows, N = KIND == kDx ? D : V, K = KIND == kLogits ? D : KIND == kDx ? V : rows;
    tiles = (M + BMT - 1) / BMT * ((N + Geo<BMT, T>::BN - 1) / Geo<BMT, T>::BN);
    ktiles = (int)((K + kBKT<T> - 1) / kBKT<T>);
  }
  float us() const { return product_us<T, KIND, BMT>(tiles, ktiles, slices_of<T, KIND, BMT>(tiles, ktiles)); }
  int64_t part_bytes() const {
    return KIND == kLogits ? 0 : std::min<int64_t>(kUnits, tiles * kSlices) * BMT * Geo<BMT, T>::BN * 4;
  }
};

// Whether a product of this many rows takes thin tiles: where they are the faster ones by product_us.
template <typename T, int KIND>
bool thin_of(int64_t rows, int64_t D, int64_t V) {
  return Sizes<T, KIND, THIN>(rows, D, V).us() < Sizes<T, KIND, BM>(rows, D, V).us();
}
template <typename T, int KIND>
int64_t part_bytes(bool thin, int64_t rows, int64_t D, int64_t V) {
  return thin ? Sizes<T, KIND, THIN>(rows, D, V).part_bytes() : Sizes<T, KIND, BM>(rows, D, V).part_bytes();
}

template <typename T>
Plan plan_of(int64_t T_, int64_t D, int64_t V, bool grad) {
  constexpr int VEC = VecTraits<T>::kN;
  Plan q;
  q.Dp = (int)((D + VEC - 1) / VEC * VEC);
  q.Vp = (int)((V + VEC - 1) / VEC * VEC);
  q.pad = V % VEC != 0;
  // a strip is half a tile's columns; with gradients a row of P is in a chunk as a whole
  const int64_t row_bytes = grad ? (int64_t)q.Vp * (int64_t)sizeof(T) : (V + 63) / 64 * 8;
  const int64_t rows = std::min(T_, std::max<int64_t>(BM, kChunkBytes / row_bytes / BM * BM));
  q.chunk_rows = (int)rows;
  q.chunks = (int)((T_ + rows - 1) / rows);
  q.thin[kLogits] = thin_of<T, kLogits>(rows, D, V);
  q.thin[kDx] = thin_of<T, kDx>(rows, D, V);
  q.thin[kDw] = thin_of<T, kDw>(rows, D, V);
  q.strip = q.thin[kLogits] ? Geo<THIN, T>::WTN : Geo<BM, T>::WTN;
  const int64_t strips = (V + q.strip - 1) / q.strip;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  q.kept = take(4);
  q.idx = take(T_ * 4);
  q.tgt = take(T_ * 4);
  q.target_logit = take(T_ * 4);
  q.row_loss = take(T_ * 4);
  q.xc = take(T_ * q.Dp * (int64_t)sizeof(T));
  q.w = take(q.pad ? D * q.Vp * (int64_t)sizeof(T) : 0);
  q.stats = take(strips * rows * 8);
  q.p = take(grad ? rows * row_bytes : 0);
  q.acc = take(grad && q.chunks > 1 ? (D + BM - 1) / BM * BM * ((V + BN - 1) / BN * BN) * 4 : 0);
  q.parts = take(grad ? std::max(part_bytes<T, kDx>(q.thin[kDx], rows, D, V), part_bytes<T, kDw>(q.thin[kDw], rows, D, V)) : 0);
  q.total = at;
  return q;
}

int check_sizes(const char* name, int64_t T, int64_t D, int64_t V, int dtype) {
  ABACUS_CHECK_ARG(dtype == kF32 || dtype == kBF16, "%s: unsupported dtype code %d (0 = fp32, 1 = bf16)", name, dtype);
  ABACUS_CHECK_ARG(T >= 0 && T < (1ll << 30), "%s: %lld rows", name, (long long)T);
  ABACUS_CHECK_ARG(D >= 1 && D < (1ll << 24), "%s: dim %lld", name, (long long)D);
  ABACUS_CHECK_ARG(V >= 1 && V < (1ll << 24), "%s: vocabulary of %lld", name, (long long)V);
  return 0;
}

template <typename T, int KIND, int BMT>
int launch_product(const LceArgs& a, hipStream_t s) {
  const int64_t tiles = Sizes<T, KIND, BMT>(std::min(a.chunk_rows, a.T - a.chunk * a.chunk_rows), a.D, a.V).tiles;
  // a product of fewer rows (or a shorter reduction) may be cut into more slices, up to kUnits units
  int64_t units = KIND == kLogits ? tiles : std::max<int64_t>(tiles, std::min<int64_t>(kUnits, tiles * kSlices));
  units = (units + 7) / 8 * 8;
  ABACUS_CHECK_ARG(units < (1ll << 31), "linear_cross_entropy: %lld tiles", (long long)units);
  const bool ragged = KIND == kDw || (KIND == kLogits ? a.D : a.Vp) % kBKT<T> != 0;
  if (ragged) hipLaunchKernelGGL((lce_product_kernel<T, KIND, BMT, true>), dim3((unsigned)units), dim3(NT), 0, s, a);
  else if constexpr (KIND != kDw) hipLaunchKernelGGL((lce_product_kernel<T, KIND, BMT, false>), dim3((unsigned)units), dim3(NT), 0, s, a);
  ABACUS_CHECK_LAUNCH("linear_cross_entropy product");
  if constexpr (KIND != kLogits) {
    if (KIND == kDx || 2 * tiles <= kUnits) {  // (two slices or more are of at most kUnits / 2 tiles)
      const int64_t cut = std::min<int64_t>(tiles, kUnits / 2);
      hipLaunchKernelGGL((lce_reduce_kernel<T, KIND, BMT>), dim3((unsigned)(cut * (BMT / kReduceRows))), dim3(256), 0, s, a);
      ABACUS_CHECK_LAUNCH("linear_cross_entropy reduce");
    }
  }
  return 0;
}

template <typename T>
int run(LceArgs a, char* ws, int64_t ws_bytes, hipStream_t s) {
  const Plan q = plan_of<T>(a.T, a.D, a.V, a.grad);
  ABACUS_CHECK_ARG(ws != nullptr && ws_bytes >= q.total, "linear_cross_entropy: workspace of %lld bytes, %lld needed",
                   (long long)ws_bytes, (long long)q.total);
  a.Dp = q.Dp;
  a.Vp = q.Vp;
  a.chunk_rows = q.chunk_rows;
  a.kept = (int*)(ws + q.kept);
  a.idx = (int*)(ws + q.idx);
  a.tgt = (int*)(ws + q.tgt);
  a.target_logit = (float*)(ws + q.target_logit);
  a.row_loss = (float*)(ws + q.row_loss);
  a.xc = ws + q.xc;
  a.stats = (float2*)(ws + q.stats);
  a.p = ws + q.p;
  a.acc = (float*)(ws + q.acc);
  a.parts = (float*)(ws + q.parts);
  a.ldv = a.V;
  int rows_per = std::max(4, (a.T + 511) / 512);
  rows_per = std::min(rows_per, 4096);
  hipLaunchKernelGGL(pack_rows_kernel<T>, dim3((a.T + rows_per - 1) / rows_per), dim3(256), rows_per * 4, s, a, rows_per);
  ABACUS_CHECK_LAUNCH("linear_cross_entropy pack");
  if (q.pad) {
    const dim3 grid((unsigned)((q.Vp / VecTraits<T>::kN + 255) / 256), (unsigned)((a.D + kPadRows - 1) / kPadRows));
    hipLaunchKernelGGL(pad_w_kernel<T>, grid, dim3(256), 0, s, (const T*)a.w, a.D, a.V, q.Vp, (T*)(ws + q.w));
    ABACUS_CHECK_LAUNCH("linear_cross_entropy pad");
    a.w = ws + q.w;
    a.ldv = q.Vp;
  }
  a.chunks = q.chunks;
  for (a.chunk = 0; a.chunk < q.chunks; ++a.chunk) {
    if (int rc = q.thin[kLogits] ? launch_product<T, kLogits, THIN>(a, s) : launch_product<T, kLogits, BM>(a, s)) return rc;
    const int rows = std::min(a.chunk_rows, a.T - a.chunk * a.chunk_rows);
    hipLaunchKernelGGL(lce_rows_kernel<T>, dim3((rows + kRowsB - 1) / kRowsB), dim3(256), 0, s, a, q.strip);
    ABACUS_CHECK_LAUNCH("linear_cross_entropy rows");
    if (a.dx) {
      if (int rc = q.thin[kDx] ? launch_product<T, kDx, THIN>(a, s) : launch_product<T, kDx, BM>(a, s)) return rc;
    }
    if (a.dw) {
      if (int rc = q.thin[kDw] ? launch_product<T, kDw, THIN>(a, s) : launch_product<T, kDw, BM>(a, s)) return rc;
    }
  }
  if (a.reduction != ABACUS_LOSS_ROWS && a.loss) {
    hipLaunchKernelGGL(lce_sum_kernel, dim3(1), dim3(1024), 0, s, a);
    ABACUS_CHECK_LAUNCH("linear_cross_entropy sum");
  }
  return 0;
}

}  // namespace
}  // namespace abacus

using namespace abacus;

extern "C" {

int64_t abacus_linear_cross_entropy_ws_bytes(int64_t T, int64_t D, int64_t V, int dtype, int grad) {
  if (T <= 0 || check_sizes("linear_cross_entropy", T, D, V, dtype)) return 0;
  return (dtype == kBF16 ? plan_of<uint16_t>(T, D, V, grad != 0) : plan_of<float>(T, D, V, grad != 0)).total;
}

int abacus_linear_cross_entropy(const void* x_TD, int64_t x_stride, const void* w_DV, const int64_t* targets_T, int64_t T,
                                int64_t D, int64_t V, int64_t ignore_index, int dtype, int reduction,
                                const float* row_grad_T, float* loss, void* dx_TD, void* dw_DV, void* ws,
                                int64_t ws_bytes, void* stream) {
  if (int rc = check_sizes("linear_cross_entropy", T, D, V, dtype)) return rc;
  ABACUS_CHECK_ARG(reduction >= ABACUS_LOSS_ROWS && reduction <= ABACUS_LOSS_MEAN, "linear_cross_entropy: reduction %d", reduction);
  ABACUS_CHECK_ARG(x_stride >= D, "linear_cross_entropy: a row stride of %lld for dim %lld", (long long)x_stride, (long long)D);
  ABACUS_CHECK_ARG((row_grad_T != nullptr) <= (reduction == ABACUS_LOSS_ROWS), "linear_cross_entropy: weights of rows come with each row's loss");
  const bool grad = dx_TD != nullptr || dw_DV != nullptr;
  ABACUS_CHECK_ARG(reduction != ABACUS_LOSS_ROWS || grad == (row_grad_T != nullptr), "linear_cross_entropy: gradients of rows' losses need the rows' weights");
  ABACUS_CHECK_ARG(grad || loss != nullptr, "linear_cross_entropy: nothing to compute");
  if (T == 0) return 0;
  LceArgs a{};
  a.x = x_TD;
  a.x_stride = x_stride;
  a.w = w_DV;
  a.targets = targets_T;
  a.ignore_index = ignore_index;
  a.T = (int)T;
  a.D = (int)D;
  a.V = (int)V;
  a.reduction = reduction;
  a.grad = grad;
  a.row_grad = row_grad_T;
  a.loss = loss;
  a.dx = dx_TD;
  a.dw = dw_DV;
  return dtype == kBF16 ? run<uint16_t>(a, (char*)ws, ws_bytes, (hipStream_t)stream)
                        : run<float>(a, (char*)ws, ws_bytes, (hipStream_t)stream);
}

int abacus_scale_by(void* t, int64_t n, int dtype, const float* g, void* stream) {
  ABACUS_CHECK_ARG(dtype == kF32 || dtype == kBF16, "scale_by: unsupported dtype code %d (0 = fp32, 1 = bf16)", dtype);
  ABACUS_CHECK_ARG(n >= 0, "scale_by: %lld values", (long long)n);
  if (n == 0) return 0;
  const unsigned blocks = (unsigned)std::min<int64_t>((n + 2047) / 2048, 4096);
  if (dtype == kBF16) hipLaunchKernelGGL(scale_kernel<uint16_t>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, (uint16_t*)t, n, g);
  else hipLaunchKernelGGL(scale_kernel<float>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, (float*)t, n, g);
  ABACUS_CHECK_LAUNCH("scale_by");
  return 0;
}

}  // extern "C"
