// Cross-entropy of a linear head, x W against targets, with the gradients of both operands: the logits never in
// memory, the probabilities a piece of the rows at a time.  No counterpart in the reference, whose head and loss are two
// steps (transformer_moe.py:75, trainer.py:77-85).
//
//   l = x W  (fp32),   lse_t = log sum_v exp l_tv,   loss_t = lse_t - l[t, target_t]
//   P_tv = s_t (exp(l_tv - lse_t) - [v = target_t]),   dx = c P W^T,   dw = c x^T P
//
// c is 1 / kept rows (mean), 1 (sum) or the largest finite weight of a row, and s_t 1 or the row's share of that: a factor common
// to all rows stays out of P, whose rounding would be the same in each (a P of -1 / 7852 at every target:
// 0.2% off in bf16) and would not average out.  Rows whose target is ignore_index are left out before
// any product: the kept rows are packed (their count stays on the device) and every launch ends at that count, so a
// batch of prompts costs what its answers cost.
//
// One pass over a chunk of kept rows (all of them while their P takes at most kChunkBytes):
//   1. logits: a tile of x W stays in registers; of each row and strip of columns its maximum m and the sum of
//      exp(l - m) go out, and with gradients exp(l - m) itself, in 16 bits of which 10 are mantissa for bf16
//      operands (it is in [0, 1], so 6 bits of exponent and no sign do; rounded eight times finer than P).
//   2. rows: the strips' (m, sum) joined to lse and the loss; P in place of the exponentials, rounded once to the
//      operands' type, which the matrix instructions take.
//   3. dx and dw: two products on P.  Where their tiles are fewer than the CUs, slices of the reduction in fp32,
//      added in slice order.  Over several chunks dw adds up in fp32.
// So 6 n D V operations of matrix products in all: the logits are not computed again for the gradient.
//
// Up to kFewRows rows are bound by w's bytes instead, and three kernels of their own read or write w and dw once each, at any
// alignment, where the tiles need w's rows at whole vectors: a copy where the vocabulary is not.
//
// 8188 x 1024 x 32000 bf16 takes 1.75 ms (1.42 at the rate of a large product alone), 16384 x 4096 x 65536 22.8 ms, the
// losses of 24 x 2048 x 50257 59 us.
#include <algorithm>
#include <type_traits>

#include "gemm_tiles.h"

namespace abacus {
namespace {

using namespace pipe;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kCUs = 256;
// Of P, or of the strips' statistics where there is no P: 16384 x 4096 x 65536 bf16 in two pieces takes 22.6 ms, as in one
// (2 GiB), in four 23.5, as each adds to dw's fp32 sums.
constexpr int64_t kChunkBytes = 1ll << 30;
constexpr int64_t kChunkRows = 1ll << 26;         // 2^31 threads of the rows' launch, which holds fewer than 2^32
constexpr int kUnits = 512;                       // tiles x slices of a sliced product at most
constexpr int kSlices = 32;
// Rows up to which w streams once for each product, without tiles: 64 x 2048 x 32000 bf16 both ways 145 us, by tiles 159;
// of 50257 columns 249 and, with w's copy, 308; 32 x 512 x 8000 48 and 62.  More rows would need more than a wave's registers.
constexpr int kFewRows = 64;
constexpr int kReduceRows = 4;                    // rows of a tile that a work-group of the adding pass takes

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
  int thin;               // bit k: kind k's tiles are thin
  int reduction;          // ABACUS_LOSS_*
  int grad;               // P is wanted
  int add;                // the launch's last work-group adds the losses
  const float* row_grad;  // weights of the rows, or NULL
  float* loss;
  void* dx;               // NULL: not wanted
  void* dw;
  // workspace
  int* kept;              // the number of kept rows, and
  float* scale;           // the factor of both gradients, and
  int* slices;            // (by Kind) of this chunk's products
  int* idx;               // kept row -> row
  int* tgt;               // kept row -> target (-1: outside the vocabulary)
  float* target_logit;    // of each kept row; NaN until its strip writes it
  float* row_loss;        // of each kept row
  void* xc;               // kept rows of x
  void* xt;               // few rows: x transposed, (D, kFewRows)
  float2* stats;          // (strip, chunk row): maximum, sum
  void* p;                // (chunk rows, Vp)
  float* acc;             // dw over several chunks
  float* parts;           // tiles of a sliced product
};

template <typename T> constexpr int kVec = VecTraits<T>::kN;

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
__host__ __device__ inline bool slices_fit(int64_t tiles, int ktiles, int s) {
  return s == 1 || (s <= kSlices && tiles * s <= kUnits && ktiles >= 4 * s);
}
template <typename T, int KIND, int BMT>
__host__ __device__ inline int slices_of(int64_t tiles, int ktiles) {
  int best = 1;
  if constexpr (KIND != kLogits) {
    float least = product_us<T, KIND, BMT>(tiles, ktiles, 1);
    for (int s = 2; slices_fit(tiles, ktiles, s); ++s) {
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

// What a row's weight is worth to the factor of all rows: a NaN or an infinity nothing, as in that factor it would reach
// every row (its own has it by its share of the factor).
__device__ inline float weight_of(float g) { return fabsf(g) < __builtin_inff() ? fabsf(g) : 0.f; }

// A block takes rows_per rows: it counts the kept rows before them, so that no block waits for another, and copies
// its kept rows to their places; the rows left out get a gradient of 0.  (8192 x 1024 bf16: 23 us, half of them the reading
// of the targets; 16384 x 4096: 83 us, 3.2 TB/s.)
template <typename T>
__global__ __launch_bounds__(256) void pack_rows_kernel(LceArgs a, int rows_per) {
  constexpr int VEC = kVec<T>;
  extern __shared__ int place_s[];  // rows_per
  __shared__ int wave_s[4];
  __shared__ float most_s[4];
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
    if (lane == 0 && row0 + rows == a.T) {
      *a.kept = before;
      a.slices[kDx] = a.slices[kDw] = 1;
      if (a.reduction != ABACUS_LOSS_ROWS) *a.scale = a.reduction == ABACUS_LOSS_MEAN ? 1.0f / (float)before : 1.0f;
    }
  }
  if (a.row_grad && row0 + rows == a.T) {  // (the last work-group's business too)
    float most = 0.f;
    for (int i = tid; i < a.T; i += 256) {
      if (a.targets[i] != a.ignore_index) most = fmaxf(most, weight_of(a.row_grad[i]));
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor(most, off, 64));
    if (lane == 0) most_s[wave] = most;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < 4; ++w) most = fmaxf(most, most_s[w]);
      *a.scale = most == 0.f ? 1.0f : most;
    }
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

// The same for few rows: a work-group takes 64 columns of all of them, and turns them for dw.  (Bound by latency: 24 x 2048
// bf16 4.8 us, with a row a wave at a time 8.4 for 40.)
template <typename T>
__global__ __launch_bounds__(256) void pack_few_kernel(LceArgs a) {
  __shared__ int place_s[kFewRows], kept_s;
  __shared__ T tile_s[kFewRows][66];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = blockIdx.x * 64 + lane;
  if (wave == 0) {
    const int64_t t = lane < a.T ? a.targets[lane] : a.ignore_index;
    const bool kept = lane < a.T && t != a.ignore_index;
    const uint64_t mask = __ballot(kept);
    const int at = __popcll(mask & ((1ull << lane) - 1)), n = __popcll(mask);
    place_s[lane] = kept ? at : -1;
    if (lane == 0) kept_s = n;
    if (blockIdx.x == 0) {
      if (kept) {
        a.idx[at] = lane;
        a.tgt[at] = t >= 0 && t < a.V ? (int)t : -1;
        a.target_logit[at] = __builtin_nanf("");
      } else if (lane < a.T && a.reduction == ABACUS_LOSS_ROWS && a.loss) {
        a.loss[lane] = 0.f;
      }
      float most = a.row_grad && kept ? weight_of(a.row_grad[lane]) : 0.f;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor(most, off, 64));
      if (lane == 0) {
        *a.kept = n;
        *a.scale = a.row_grad ? (most == 0.f ? 1.0f : most) : a.reduction == ABACUS_LOSS_MEAN ? 1.0f / (float)n : 1.0f;
      }
    }
  }
  __syncthreads();
  for (int r0 = wave; r0 < a.T; r0 += 32) {
    T v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = ((const T*)a.x)[(int64_t)min(r0 + 4 * u, a.T - 1) * a.x_stride + min(c, a.D - 1)];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int r = r0 + 4 * u, at = r < a.T ? place_s[r] : -1;
      if (at >= 0 && c < a.Dp) {
        if (c >= a.D) v[u] = from_f32<T>(0.f);
        ((T*)a.xc)[(int64_t)at * a.Dp + c] = v[u];
        tile_s[at][lane] = v[u];
      } else if (r < a.T && at < 0 && a.dx && c < a.D) {
        ((T*)a.dx)[(int64_t)r * a.D + c] = from_f32<T>(0.f);
      }
    }
  }
  if (!a.xt) return;
  __syncthreads();
  for (int d = wave; d < min(64, a.D - (int)blockIdx.x * 64); d += 4)  // a lane a row, zeros past the last
    ((T*)a.xt)[(int64_t)(blockIdx.x * 64 + d) * kFewRows + lane] = lane < kept_s ? tile_s[lane][d] : from_f32<T>(0.f);
}

// w's rows of V values at a pitch of whole vectors, zeros behind them.  A thread takes a column of kPadRows vectors, so
// that as many loads are in flight.  (2048 x 50257 bf16: 81 us, 5.1 TB/s; a vector at a time 110.)
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

// exp(l - m).  The difference comes first: it is never above 0, and as exact as l is, however large the logits are (one
// multiply-add of l log2(e) and m log2(e) would save an instruction and be off by the rounding of the second: above 1 for some m).
__device__ inline float exp_from(float l, float m) { return __builtin_amdgcn_exp2f((l - m) * kLog2e); }
// Finite in a strip of -inf, whose exponentials are 0.
__device__ inline float top_of(float m) { return fmaxf(m, -3.0e38f); }

// acc += A B over a range of k-tiles: the operands' tiles come by DMA into a ring of LDS stages, the matrix
// instructions of one k-step cover the fragment reads of the next, and the last step's the DMA.  begin() starts the first
// stages' DMA (every read of the stages has to be done), run() waits for them and does the rest.
template <typename T, bool A_MC, bool B_NC, int BMT, bool RK>
struct TileProduct {
  using Op = MfmaOp<T, 32>;
  using GE = Geo<BMT, T>;
  static constexpr int FM = GE::FM, FN = GE::FN, WTM = GE::WTM, WTN = GE::WTN, ST = GE::ST, LOADS = GE::LOADS;
  static constexpr int MCC_A = BMT * (int)sizeof(T) / 16, MCC_B = GE::BN * (int)sizeof(T) / 16;
  static constexpr int BKT = kBKT<T>, NFRAG = FM + FN, MF = FM * FN;
  using Acc = typename Op::Acc;
  static_assert(MF >= NFRAG, "one fragment read per MFMA at most");

  DmaStream<T, A_MC, GE::DMA_A, BMT> sa;
  DmaStream<T, B_NC, GE::DMA_B, GE::BN> sb;
  int kbase, ktiles, k_lim;
  char* lds;
  uint32_t lds32, stage;
  int k0, lane, wave_u;

  __device__ __attribute__((always_inline)) inline void prep(int kt) {
    stage = lds32 + (uint32_t)((kt % ST) * GE::STAGE);
    k0 = (kt + kbase) * BKT;
  }
  // instruction n of the LOADS of the k-tile that prep() named
  __device__ __attribute__((always_inline)) inline void dma(int n) {
    if (n < GE::DMA_A) sa.template issue_one<RK>(n, stage, wave_u, k0, k_lim);
    else sb.template issue_one<RK>(n - GE::DMA_A, stage + GE::A_BYTES, wave_u, k0, k_lim);
  }
  // At most the newest `later` k-tiles' loads may still be in flight.
  static __device__ __attribute__((always_inline)) inline void wait_for(int later) {
    if (ST >= 4 && later >= 3) wait_vmcnt<(ST >= 4 ? 3 : 0) * LOADS>();
    else if (ST >= 3 && later >= 2) wait_vmcnt<(ST >= 3 ? 2 : 0) * LOADS>();
    else if (later >= 1) wait_vmcnt<LOADS>();
    else wait_vmcnt<0>();
  }

  __device__ __attribute__((always_inline)) inline void begin(const T* A, int64_t lda, int row0, int a_lim, const T* B, int64_t ldb, int n0,
                                                              int b_lim, int kbase_, int ktiles_, int k_lim_, char* lds_) {
    const int wave = threadIdx.x >> 6;
    lane = threadIdx.x & 63;
    wave_u = __builtin_amdgcn_readfirstlane(wave);
    kbase = kbase_;
    ktiles = ktiles_;
    k_lim = k_lim_;
    lds = lds_;
    lds32 = lds_addr32(lds);
    sa.setup(A, nullptr, lda, row0, a_lim, wave, lane);
    sb.setup(B, nullptr, ldb, n0, b_lim, wave, lane);
#pragma unroll
    for (int p = 0; p < ST; ++p)
      if (p < ktiles) {
        prep(p);
#pragma unroll
        for (int n = 0; n < LOADS; ++n) dma(n);
      }
  }

  // The first k-tile has landed.  stores: vector memory operations that every wave has issued since begin(), at least;
  // they may still be in flight.
  template <int STORES>
  __device__ __attribute__((always_inline)) inline void wait_first() {
    if (ktiles < ST) wait_vmcnt<0>();
    else wait_vmcnt<(STORES + LOADS * (ST - 1) < 63 ? STORES + LOADS * (ST - 1) : 63)>();
  }

  __device__ __attribute__((always_inline)) inline void run(Acc (&acc)[FM][FN], int wave_rows) {
    if (ktiles <= 0) return;
    const int wave = threadIdx.x >> 6, wm = wave / WAVES_N, wn = wave % WAVES_N;
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
          for (int n = m * LOADS / MF; n < (m + 1) * LOADS / MF; ++n) dma(n);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto ktile = [&](auto lfc, int kt, bool next, bool dma_next) __attribute__((always_inline)) {
      const char* st = lds + (kt % ST) * GE::STAGE;
      const char* st_next = lds + ((kt + 1) % ST) * GE::STAGE;
#pragma unroll
      for (int t = 0; t < NSTEP - 1; ++t) kstep(lfc, t & 1, true, st, t + 1, (t + 1) & 1, false);
      wait_for(min(ST - 2, ktiles - 2 - kt));  // k-tile kt + 1 has landed
      __builtin_amdgcn_s_waitcnt(0xc07f);  // this wave's reads of the stage are back: it may be refilled
      __syncthreads();
      if (dma_next) prep(kt + ST);
      __builtin_amdgcn_sched_barrier(0);
      kstep(lfc, (NSTEP - 1) & 1, next, st_next, 0, 0, dma_next);
    };
    __builtin_amdgcn_s_waitcnt(0xc07f);
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

// VEC values to p at any element, as many as the row has left.
template <typename T>
__device__ inline void store_left(T* p, const float* f, int left) {
  if (left >= kVec<T>) {
    u32x4_any v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) v[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
      else v[i] = f32_bits(f[i]);
    }
    *reinterpret_cast<u32x4_any*>(p) = v;
  } else if constexpr (sizeof(T) == 2) {
    st8_any(p, Vec16{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])}, left);
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < left) p[i] = f[i];
  }
}

// VEC finished values of a gradient at (row, col) of dx or dw; whole: rows of it are whole vectors.
template <typename T, int KIND>
__device__ inline void store_grad(const LceArgs& a, float scale, int row, int col, float* f, bool whole) {
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) f[i] *= scale;
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
    store_left<T>(out, f, N - col);
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
    slices = KIND == kLogits ? 1 : a.slices[KIND];
  }
  // slices_of by a wave, a number of slices a lane (over several chunks dw's tiles are cut alike in each, as their
  // sums go from one to the next)
  __device__ inline int cut(const LceArgs& a) const {
    const int kt = KIND == kDw && a.chunks > 1 ? (a.chunk_rows + kBKT<T> - 1) / kBKT<T> : ktiles;
    const int64_t tiles = (int64_t)mt * nt;
    int best = (int)(threadIdx.x & 63) + 1;
    float least = slices_fit(tiles, kt, best) ? product_us<T, KIND, BMT>(tiles, kt, best) : 3.0e38f;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const float us = __shfl_xor(least, off, 64);
      const int s = __shfl_xor(best, off, 64);
      if (us < least || (us == least && s < best)) {
        least = us;
        best = s;
      }
    }
    return best;
  }
};

template <typename TP>
__device__ __attribute__((always_inline)) inline void clear(typename TP::Acc (&acc)[TP::FM][TP::FN]) {
#pragma unroll
  for (int i = 0; i < TP::FM; ++i)
#pragma unroll
    for (int j = 0; j < TP::FN; ++j)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.f;
}

// An accumulator read where it is wanted: left to itself the compiler moves all 256 of a lane out of their registers at
// once, to scratch memory.  (settle() before the first: the matrix instructions' results are there.)
__device__ inline float taken(float v) {
  float r;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(r) : "a"(v));
  return r;
}
__device__ inline void settle() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

__device__ inline float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Statistics and exponentials of a tile of logits.  Fragment (i, j): lane l has row l % 32 and columns
// 8 g + 4 (l / 32) .. +3 for g = 0..3.  Everything goes straight from registers to memory, so that the
// next tile's first DMA can be under way: two lanes of a row trade halves for 16 bytes of bf16 operands each.
// WHOLE: every row and column of the tile is one of the product.
template <typename T, int BMT, typename TP, bool WHOLE, bool GRAD>
__device__ __attribute__((always_inline)) inline void logits_out(const LceArgs& a, typename TP::Acc (&acc)[TP::FM][TP::FN], const int (&tgt)[TP::FM],
                                                                 int row0, int n0, int n) {
  using GE = Geo<BMT, T>;
  constexpr int FM = GE::FM, FN = GE::FN, WTM = GE::WTM, WTN = GE::WTN;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WAVES_N, wn = wave % WAVES_N;
  const int rl = lane & 31, half = lane >> 5, strip = n0 / WTN + wn, first = n0 + wn * WTN;
  settle();
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int row = row0 + wm * WTM + i * 32 + rl;
    const bool here = WHOLE || row < n;
    float l[FN][16];
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int q = 0; q < 16; ++q) l[j][q] = taken(acc[i][j][q]);
    if (!WHOLE && n0 + GE::BN > a.V) {  // columns past the vocabulary are no logits
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int q = 0; q < 16; ++q)
          if (first + j * 32 + 8 * (q >> 2) + 4 * half + (q & 3) >= a.V) l[j][q] = -__builtin_inff();
    }
    const int t = tgt[i] - first;
    if (here && t >= 0 && t < WTN && ((t >> 2) & 1) == half) {
      float at = 0.f;
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int q = 0; q < 16; ++q) at = t == j * 32 + 8 * (q >> 2) + 4 * half + (q & 3) ? l[j][q] : at;
      a.target_logit[a.chunk * a.chunk_rows + row] = at;
    }
    float m[4];  // (four at a time: one chain would wait for itself)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      m[k] = l[0][4 * k];
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int q = 4 * k; q < 4 * k + 4; q += 2) m[k] = max3(m[k], l[j][q], l[j][q + 1]);
    }
    m[0] = fmaxf(max3(m[0], m[1], m[2]), m[3]);
    m[0] = fmaxf(m[0], __shfl_xor(m[0], 32, 64));
    const float top = top_of(m[0]);
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int g = 0; g < 4; g += 2) {
        float e[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          e[k] = exp_from(l[j][4 * g + k], top);
          s[k & 3] += e[k];
        }
        if constexpr (GRAD) {
          const int col = first + j * 32 + 8 * g;
          if constexpr (sizeof(T) == 2) {
            const auto x = __builtin_amdgcn_permlane32_swap(encode2(e[0], e[1]), encode2(e[4], e[5]), false, false);
            const auto y = __builtin_amdgcn_permlane32_swap(encode2(e[2], e[3]), encode2(e[6], e[7]), false, false);
            if (WHOLE || (here && col + 8 * half < a.Vp)) {
              Vec16 v;
              v.w[0] = x[0];
              v.w[1] = y[0];
              v.w[2] = x[1];
              v.w[3] = y[1];
              st16((uint16_t*)a.p + (int64_t)row * a.Vp + col + 8 * half, v);
            }
          } else {
#pragma unroll
            for (int k = 0; k < 2; ++k)
              if (WHOLE || (here && col + 8 * k + 4 * half < a.Vp))
                *reinterpret_cast<float4*>((float*)a.p + (int64_t)row * a.Vp + col + 8 * k + 4 * half) =
                    make_float4(e[4 * k], e[4 * k + 1], e[4 * k + 2], e[4 * k + 3]);
          }
        }
      }
    s[0] = (s[0] + s[1]) + (s[2] + s[3]);
    s[0] += __shfl_xor(s[0], 32, 64);
    if (here && lane < 32 && (WHOLE || first < a.V)) a.stats[(int64_t)strip * a.chunk_rows + row] = make_float2(top, s[0]);
  }
}

// The logits' tiles: a work-group on each CU walks its share of the XCD's tiles, and a tile's first DMA is under way while
// the one before goes through its exponentials.  Bound by the matrix instructions and, in short reductions, by the exponentials
// and their rounding after them (about 8 us a tile of 256 x 256, in which the matrix unit rests): 16384 x 4096 x 65536
// bf16 7.3 ms, 1200 TF/s; 8188 x 1024 x 32000 593 to 655 us, 820 to 900 TF/s (a work-group a tile, its exponentials
// through LDS: 667 where this takes 593); 900 x 512 x 8000 fp32 84 us.
template <typename T, int BMT, bool RK, bool GRAD>
__global__ __launch_bounds__(NT, 1) void lce_logits_kernel(LceArgs a) {
  using GE = Geo<BMT, T>;
  using TP = TileProduct<T, false, true, BMT, RK>;
  __shared__ __attribute__((aligned(1024))) char lds[GE::ST * GE::STAGE];
  const int n = chunk_kept(a);
  if (n == 0) return;
  const Cover<T, kLogits, BMT> cv(a, n);
  const int units = cv.mt * cv.nt, per = (units + 7) / 8, xcd = blockIdx.x & 7, step = gridDim.x >> 3;
  const int end = min(units, (xcd + 1) * per);  // an equal contiguous share for each XCD
  const T* xc = (const T*)a.xc + (int64_t)a.chunk * a.chunk_rows * a.Dp;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WAVES_N;
  TP tp;
  int row0 = 0, n0 = 0;
  auto begin = [&](int u) __attribute__((always_inline)) {
    int mt, nt;
    row_tile(u, cv.mt, cv.nt, mt, nt);
    row0 = mt * BMT;
    n0 = nt * GE::BN;
    tp.begin(xc, a.Dp, row0, n, (const T*)a.w, a.ldv, n0, a.Vp, 0, cv.ktiles, cv.K, lds);
  };
  int u = xcd * per + ((int)blockIdx.x >> 3);
  if (u >= end) return;
  begin(u);
  bool whole = false;  // every lane of the tile before stored all it has
  for (;;) {
    const int row_now = row0, n_now = n0;
    const int wave_rows = __builtin_amdgcn_readfirstlane(n - row_now - wm * GE::WTM);
    int tgt[GE::FM];
#pragma unroll
    for (int i = 0; i < GE::FM; ++i)
      tgt[i] = a.tgt[a.chunk * a.chunk_rows + min(row_now + wm * GE::WTM + i * 32 + (lane & 31), n - 1)];
    typename TP::Acc acc[GE::FM][GE::FN];
    clear<TP>(acc);
    if (whole) tp.template wait_first<GE::FM * GE::FN * 2>();
    else tp.template wait_first<0>();
    tp.run(acc, wave_rows);
    u += step;
    const bool more = u < end;
    if (more) begin(u);  // (the stages were last read before run()'s last barrier)
    const bool inside = row_now + BMT <= n && n_now + GE::BN <= a.V;
    if (inside) logits_out<T, BMT, TP, true, GRAD>(a, acc, tgt, row_now, n_now, n);
    else logits_out<T, BMT, TP, false, GRAD>(a, acc, tgt, row_now, n_now, n);
    if (!more) break;
    whole = GRAD && inside;
  }
}

// A tile, or a slice of its reduction, of dx = P W^T (kDx) or dw = x^T P (kDw) a work-group: bound by the matrix
// instructions, at large sizes by the clock that their power leaves.  8188 x 1024 x 32000 bf16: 468 and 460 us, 1150 and 1170
// TF/s; 16384 x 4096 x 65536: 7.0 and 7.4 ms, 1250 and 1180; 900 x 512 x 8000 fp32, thin tiles: 82 and 79 us.
template <typename T, int KIND, int BMT, bool RK, bool SUMS>
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
  typename TP::Acc acc[FM][FN];
  clear<TP>(acc);
  TP tp;
  if constexpr (KIND == kDx)
    tp.begin(p, a.Vp, row0, n, (const T*)a.w, a.ldv, n0, a.D, kbase, ktiles, a.Vp, lds);
  else
    tp.begin(xc, a.Dp, row0, a.Dp, p, a.Vp, n0, a.Vp, kbase, ktiles, cv.K, lds);
  tp.template wait_first<0>();
  tp.run(acc, wave_rows);

  // Fragment (i, j): lane l has row l % 32 and columns 8 g + 4 (l / 32) .. +3 for g = 0..3.
  const int rl = lane & 31, ch = 4 * (lane >> 5);
  __syncthreads();  // every fragment read is done: the tile goes out through the stages' LDS
  if (cv.slices > 1) {  // a slice's fp32 tile, for lce_reduce_kernel
    float* out = a.parts + (int64_t)u * (BMT * BN);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int row = wm * WTM + i * 32 + rl;
      if (row0 + row >= cv.M) continue;
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<float4*>(out + row * BN + wn * WTN + j * 32 + 8 * g + ch) =
              make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
    }
    return;
  }
  // fp32 bands of RB rows through LDS: whole rows of vectors go out
  constexpr int RB = 128, LDB = BN + 4, CV = BN / VEC;
  static_assert(BMT % RB == 0 && (WTM % RB == 0 || RB % WTM == 0) && RB * LDB * 4 <= LDS_ALLOC, "bands of wave rows");
  float* band = reinterpret_cast<float*>(lds);
  const float scale = kept > 0 ? *a.scale : 1.0f;
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
                make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
    }
    __syncthreads();
    if constexpr (SUMS) {
      // dw over several chunks: the sum so far, a tile's rows one after the other, several of a thread's vectors in flight
      constexpr int U = 4;
      static_assert(RB * CV % (U * NT) == 0, "whole batches");
      const bool last = (a.chunk + 1) * (int64_t)a.chunk_rows >= kept;
      float* sums = a.acc + (int64_t)r * (BMT * BN) + pb * RB * BN;
      for (int v0 = tid; v0 < RB * CV; v0 += U * NT) {
        float4 so_far[U][VEC / 4];
        if (a.chunk > 0) {
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < VEC / 4; ++k) so_far[u][k] = *reinterpret_cast<const float4*>(sums + (v0 + u * NT) * VEC + 4 * k);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int v = v0 + u * NT, row = row0 + pb * RB + v / CV, col = n0 + v % CV * VEC;
          const float* src = band + v / CV * LDB + v % CV * VEC;
          float f[VEC];
#pragma unroll
          for (int k = 0; k < VEC; k += 4) {
            float4 x = *reinterpret_cast<const float4*>(src + k);
            if (a.chunk > 0) x = make_float4(x.x + so_far[u][k / 4].x, x.y + so_far[u][k / 4].y, x.z + so_far[u][k / 4].z, x.w + so_far[u][k / 4].w);
            *reinterpret_cast<float4*>(f + k) = x;
            if (!last) *reinterpret_cast<float4*>(sums + v * VEC + k) = x;
          }
          if (last && row < cv.M && col < cv.N) store_grad<T, KIND>(a, scale, row, col, f, whole);
        }
      }
    } else {
      for (int v = tid; v < RB * CV; v += NT) {
        const int row = row0 + pb * RB + v / CV, col = n0 + v % CV * VEC;
        const float* src = band + v / CV * LDB + v % CV * VEC;
        if (row < cv.M && col < cv.N) {
          float f[VEC];
#pragma unroll
          for (int k = 0; k < VEC; k += 4) *reinterpret_cast<float4*>(f + k) = *reinterpret_cast<const float4*>(src + k);
          store_grad<T, KIND>(a, scale, row, col, f, whole);
        }
      }
    }
    if (pb + 1 < BMT / RB) __syncthreads();
  }
}

// ---------------------------------------------------------------- few rows

// The logits of at most 32 RF rows: w streams once through the CUs, straight into the matrix instructions' registers, at
// any alignment.  A wave takes 32 CW columns (CW neighbouring ones a lane, one of each of CW fragments) and an eighth
// of the reduction, a step of 16 (bf16) or 8 rows of w in turn; the work-group adds the eighths in wave order.  Narrower
// columns where the vocabulary would leave CUs without work.  Bound by w's bytes: 24 x 2048 x 50257 bf16 50 us, 4.1 TB/s
// (55 with an eighth in one run of rows, 57 without by_xcd too, 114 through an aligned copy of w and tiles of 128 rows);
// 40 rows 76 us, as the registers leave one work-group a CU.
constexpr int kFewWaves = 8;

// Block b of n -> the one of its place where each XCD (it runs on XCD b % 8) has neighbouring ones: they share the cache lines
// that their columns' ends lie in.
__device__ inline int by_xcd(int b, int n) {
  const int x = b & 7;
  return x * (n >> 3) + min(x, n & 7) + (b >> 3);
}

// CW values of each of 8 (bf16) or 4 (fp32) rows of w, and the fragments of x beside them: a k-step of 16 or 8.
template <typename T, int CW, int RF>
struct FewStep {
  static constexpr int KL = sizeof(T) == 2 ? 8 : 4;  // k of a lane
  static constexpr int WORDS = CW * (int)sizeof(T) / 4;
  uint32_t b[KL][WORDS];
  Vec16 a[RF];

  // every value in bounds: k0 + 2 KL <= D - 1, and past a row's end the next row's first values (of columns that are no logits)
  __device__ __attribute__((always_inline)) inline void load(const LceArgs& g, const T* const (&x)[RF], int k0, int half, int col) {
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      typedef uint32_t words_any __attribute__((ext_vector_type(WORDS > 1 ? WORDS : 2), aligned(2)));
      typedef uint32_t word_any __attribute__((aligned(2)));
      const T* p = (const T*)g.w + (int64_t)(k0 + KL * half + i) * g.V + col;
      if constexpr (WORDS > 1) {
        const words_any v = *reinterpret_cast<const words_any*>(p);
#pragma unroll
        for (int w = 0; w < WORDS; ++w) b[i][w] = v[w];
      } else {
        b[i][0] = *reinterpret_cast<const word_any*>(p);
      }
    }
#pragma unroll
    for (int r = 0; r < RF; ++r) a[r] = ld16(x[r] + k0 + KL * half);
  }
  // the reduction's end, value by value
  __device__ inline void load_last(const LceArgs& g, const T* const (&x)[RF], int k0, int half, int col) {
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      const int k = k0 + KL * half + i;
      T e[CW];
#pragma unroll
      for (int c = 0; c < CW; ++c)
        e[c] = k < g.D && col + c < g.V ? ((const T*)g.w)[(int64_t)k * g.V + col + c] : from_f32<T>(0.f);
      __builtin_memcpy(b[i], e, sizeof(e));
    }
#pragma unroll
    for (int r = 0; r < RF; ++r) a[r] = k0 + KL * half < g.D ? ld16(x[r] + k0 + KL * half) : zero16();
  }
  __device__ __attribute__((always_inline)) inline void run(f32x16_t (&acc)[RF][CW]) const {
#pragma unroll
    for (int c = 0; c < CW; ++c) {
      if constexpr (sizeof(T) == 2) {
        Vec16 f;  // column c of the 8 rows
#pragma unroll
        for (int w = 0; w < 4; ++w)
          f.w[w] = __builtin_amdgcn_perm(b[2 * w + 1][c >> 1], b[2 * w][c >> 1], c & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int r = 0; r < RF; ++r)
          acc[r][c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a[r]), __builtin_bit_cast(bf16x8_t, f),
                                                              acc[r][c], 0, 0, 0);
      } else {
#pragma unroll
        for (int i = 0; i < KL; ++i)
#pragma unroll
          for (int r = 0; r < RF; ++r)
            acc[r][c] = __builtin_amdgcn_mfma_f32_32x32x2f32(bits_f32(a[r].w[i]), bits_f32(b[i][c]), acc[r][c], 0, 0, 0);
      }
    }
  }
};

template <typename T, int CW, int RF>
__global__ __launch_bounds__(kFewWaves * 64, RF == 1 ? 4 : 2) void lce_few_kernel(LceArgs a) {
  using Step = FewStep<T, CW, RF>;
  constexpr int KS = 2 * Step::KL, COLS = 32 * CW, ROWS = 32 * RF, LDL = COLS + 4;
  __shared__ __attribute__((aligned(16))) float part_s[kFewWaves][64 * 16];
  __shared__ __attribute__((aligned(16))) float logit_s[ROWS * LDL];
  const int n = chunk_kept(a);
  if (n == 0) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
  const int strip = by_xcd(blockIdx.x, gridDim.x);
  const int n0 = strip * COLS, col = min(n0 + (lane & 31) * CW, a.V - 1);
  const T* x[RF];
#pragma unroll
  for (int r = 0; r < RF; ++r)
    x[r] = (const T*)a.xc + ((int64_t)a.chunk * a.chunk_rows + min(32 * r + (lane & 31), n - 1)) * a.Dp;
  f32x16_t acc[RF][CW];
#pragma unroll
  for (int r = 0; r < RF; ++r)
#pragma unroll
    for (int c = 0; c < CW; ++c)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[r][c][q] = 0.f;
  // (whole steps end before w's last row, whose end nothing follows)
  const int whole = max(0, (a.D - 1) / KS), steps = (a.D + KS - 1) / KS;
  // a step of each wave in turn: together they read 128 neighbouring rows of w
  if (wave < whole) {
    Step s0, s1;
    s0.load(a, x, wave * KS, half, col);
    for (int k = wave; k + kFewWaves < whole; k += kFewWaves) {
      s1.load(a, x, (k + kFewWaves) * KS, half, col);
      s0.run(acc);
      s0 = s1;
    }
    s0.run(acc);
  }
  if (wave == kFewWaves - 1) {
    for (int k = whole; k < steps; ++k) {
      Step s;
      s.load_last(a, x, k * KS, half, n0 + (lane & 31) * CW);
      s.run(acc);
    }
  }
  // the waves' sums of a fragment at a time: a lane's 16 values as it has them, added in wave order to the logits' place
#pragma unroll
  for (int f = 0; f < RF * CW; ++f) {
    const int r = f / CW, c = f % CW;
    float* mine = part_s[wave] + lane * 4;
    if (f > 0) __syncthreads();
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<float4*>(mine + g * 256) =
          make_float4(acc[r][c][4 * g], acc[r][c][4 * g + 1], acc[r][c][4 * g + 2], acc[r][c][4 * g + 3]);
    __syncthreads();
#pragma unroll
    for (int v = tid; v < 1024; v += kFewWaves * 64) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) sum += part_s[w][v];
      const int g = v >> 8, l = (v >> 2) & 63, k = v & 3;  // register 4 g + k of lane l
      logit_s[(32 * r + 8 * g + 4 * (l >> 5) + k) * LDL + (l & 31) * CW + c] = sum;
    }
  }
  __syncthreads();
  // a row is LPR lanes': its statistics and exponentials
  constexpr int LPR = kFewWaves * 64 / ROWS, PER = COLS / LPR;
  const int row = tid / LPR, c0 = tid % LPR * PER;
  float l[PER], m = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    l[i] = n0 + c0 + i < a.V ? logit_s[row * LDL + c0 + i] : -__builtin_inff();
    m = fmaxf(m, l[i]);
  }
#pragma unroll
  for (int off = LPR / 2; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
  if (row >= n) return;
  const int at = a.tgt[a.chunk * a.chunk_rows + row] - n0 - c0;
  if (at >= 0 && at < PER) a.target_logit[a.chunk * a.chunk_rows + row] = logit_s[row * LDL + c0 + at];
  const float top = top_of(m);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    l[i] = exp_from(l[i], top);
    s += l[i];
  }
#pragma unroll
  for (int off = LPR / 2; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if (c0 == 0) a.stats[(int64_t)strip * a.chunk_rows + row] = make_float2(top, s);
  if (!a.grad) return;
#pragma unroll
  for (int i = 0; i < PER; i += 2) {
    const int c = n0 + c0 + i;
    if (c >= a.Vp) break;  // (an even number, as c is)
    if constexpr (sizeof(T) == 2) *reinterpret_cast<uint32_t*>((uint16_t*)a.p + (int64_t)row * a.Vp + c) = encode2(l[i], l[i + 1]);
    else *reinterpret_cast<float2*>((float*)a.p + (int64_t)row * a.Vp + c) = make_float2(l[i], l[i + 1]);
  }
}

// dx of few rows: P W^T.  A wave takes 64 of w's rows and a slice of the vocabulary, in groups of 128 bytes of a row: eight
// lanes load a row's at any alignment, and a part of LDS of the wave's own turns them to the matrix instructions' order, a row a
// lane (loaded as those want them, 16 bytes of 64 rows an instruction, rows of 50257 came at 2.5 TB/s).  A work-group
// adds its waves' slices in order and writes them to parts[blockIdx.y] (rows, Dp), which lce_few_sum_kernel adds.
// (24 x 2048 x 32000 bf16: 27 us, 40 x 2048 x 50257 63: 4.9 and 3.3 TB/s, part of w from the memory-side cache, where the
// logits' pass has left it.)
template <typename T, int RF>
__global__ __launch_bounds__(kFewWaves * 64, 2) void lce_few_dx_kernel(LceArgs a) {
  constexpr int VEC = kVec<T>, GROUP = 8 * VEC, PITCH = 9 * 16;  // bytes of a row in LDS
  __shared__ __attribute__((aligned(16))) char stage_s[kFewWaves][64 * PITCH];
  static_assert(sizeof(stage_s) >= kFewWaves * 1024 * 4, "the waves' sums go through the same place");
  const int n = chunk_kept(a);
  if (n == 0) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, d0 = blockIdx.x * 64;
  const T* wr[8];  // row 8 i + lane / 8, chunk lane % 8
#pragma unroll
  for (int i = 0; i < 8; ++i) wr[i] = (const T*)a.w + (int64_t)min(d0 + 8 * i + (lane >> 3), a.D - 1) * a.V;
  const int chunk = (lane & 7) * VEC;
  const T* pr[RF];  // a lane's half of a group is GROUP / 2 neighbouring values
#pragma unroll
  for (int r = 0; r < RF; ++r) pr[r] = (const T*)a.p + (int64_t)min(32 * r + (lane & 31), n - 1) * a.Vp + half * (GROUP / 2);
  f32x16_t acc[RF][2];
#pragma unroll
  for (int r = 0; r < RF; ++r)
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[r][f][q] = 0.f;
  const int whole = a.V / GROUP, all = (a.V + GROUP - 1) / GROUP, waves = gridDim.y * kFewWaves, per = (all + waves - 1) / waves;
  const int from = (blockIdx.y * kFewWaves + wave) * per, to = min(all, from + per);
  Vec16 w[8], p[RF][4];
  auto load = [&](int k) __attribute__((always_inline)) {
    if (k < whole) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const u32x4_any v = *reinterpret_cast<const u32x4_any*>(wr[i] + (int64_t)k * GROUP + chunk);
#pragma unroll
        for (int c = 0; c < 4; ++c) w[i].w[c] = v[c];
      }
    } else {  // the vocabulary's end: zeros past it
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = load_end<T>(wr[i], k * GROUP + chunk, a.V);
    }
#pragma unroll
    for (int r = 0; r < RF; ++r)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int at = k * GROUP + half * (GROUP / 2) + s * VEC;
        p[r][s] = ld16(pr[r] + min(k * GROUP + s * VEC, a.Vp - VEC - half * (GROUP / 2)));
        if (at >= a.Vp) p[r][s] = zero16();
      }
  };
  char* mine = stage_s[wave];
  if (from < to) load(from);
  for (int k = from; k < to; ++k) {
#pragma unroll
    for (int i = 0; i < 8; ++i) st16(mine + (8 * i + (lane >> 3)) * PITCH + (lane & 7) * 16, w[i]);
    Vec16 pn[RF][4];
#pragma unroll
    for (int r = 0; r < RF; ++r)
#pragma unroll
      for (int s = 0; s < 4; ++s) pn[r][s] = p[r][s];
    if (k + 1 < to) load(k + 1);
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const Vec16 b = ld16(mine + (32 * f + (lane & 31)) * PITCH + (half * 4 + s) * 16);
#pragma unroll
        for (int r = 0; r < RF; ++r) MfmaOp<T, 32>::run(acc[r][f], pn[r][s], b);
      }
    __builtin_amdgcn_wave_barrier();
  }
  float* part = reinterpret_cast<float*>(stage_s);  // (wave, 1024)
#pragma unroll
  for (int f = 0; f < 2 * RF; ++f) {
    __syncthreads();
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<float4*>(part + wave * 1024 + g * 256 + lane * 4) = make_float4(
          acc[f >> 1][f & 1][4 * g], acc[f >> 1][f & 1][4 * g + 1], acc[f >> 1][f & 1][4 * g + 2], acc[f >> 1][f & 1][4 * g + 3]);
    __syncthreads();
#pragma unroll
    for (int u = tid; u < 1024; u += kFewWaves * 64) {
      // neighbouring threads neighbouring columns: register 4 g + k of lane l
      const int l = (u & 31) + (u >> 5 & 1) * 32, k = u >> 6 & 3, g = u >> 8;
      float sum = 0.f;
#pragma unroll
      for (int v = 0; v < kFewWaves; ++v) sum += part[v * 1024 + g * 256 + l * 4 + k];
      const int row = 32 * (f >> 1) + 8 * g + 4 * (l >> 5) + k, col = d0 + 32 * (f & 1) + (l & 31);
      if (row < n && col < a.D) a.parts[((int64_t)blockIdx.y * kFewRows + row) * a.Dp + col] = sum;
    }
  }
}

// The kept rows' losses added in a fixed order, in fp64, by the 256 threads of a work-group beside dx's slices' (a launch of its own
// costs 4 to 10 us and the host 3), or alone.
__device__ inline void add_losses(const LceArgs& a) {
  __shared__ double sum_s[4];
  constexpr int U = 8;
  const int kept = *a.kept, tid = threadIdx.x;
  double s = 0.0;
  for (int i = tid; i < kept; i += 256 * U) {
    float l[U];
#pragma unroll
    for (int u = 0; u < U; ++u) l[u] = a.row_loss[min(i + 256 * u, kept - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u) s += i + 256 * u < kept ? (double)l[u] : 0.0;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if ((tid & 63) == 0) sum_s[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) {
    s = ((s + sum_s[1]) + sum_s[2]) + sum_s[3];
    a.loss[0] = (float)(a.reduction == ABACUS_LOSS_MEAN ? s / (double)kept : s);
  }
}
__global__ __launch_bounds__(256) void lce_sum_kernel(LceArgs a) { add_losses(a); }

// dx from the slices of lce_few_dx_kernel: a wave adds a quarter of them in order, and one the quarters.  (Latency: 24 x 1024
// of 32 slices under 6 us, a thread all slices 8.5.)
template <typename T>
__global__ __launch_bounds__(256) void lce_few_sum_kernel(LceArgs a, int slices) {
  constexpr int VEC = kVec<T>;
  __shared__ float part_s[3][VEC][64];
  if (a.add && blockIdx.x + 1 == gridDim.x) {
    add_losses(a);
    return;
  }
  const int n = chunk_kept(a), vecs = a.Dp / VEC, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = blockIdx.x * 64 + lane;
  if (blockIdx.x * 64 >= n * vecs) return;
  const int row = min(i, n * vecs - 1) / vecs, c = min(i, n * vecs - 1) % vecs * VEC;
  const int each = (slices + 3) / 4, last = min(slices, (wave + 1) * each);
  float f[VEC] = {};
  for (int s0 = wave * each; s0 < last; s0 += 4) {
    float4 x[4][VEC / 4];
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int k = 0; k < VEC / 4; ++k)
        x[s][k] = *reinterpret_cast<const float4*>(a.parts + ((int64_t)min(s0 + s, last - 1) * kFewRows + row) * a.Dp + c + 4 * k);
#pragma unroll
    for (int s = 0; s < 4; ++s)
      if (s0 + s < last)
#pragma unroll
        for (int k = 0; k < VEC / 4; ++k) {
          f[4 * k] += x[s][k].x;
          f[4 * k + 1] += x[s][k].y;
          f[4 * k + 2] += x[s][k].z;
          f[4 * k + 3] += x[s][k].w;
        }
  }
  if (wave > 0) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) part_s[wave - 1][k][lane] = f[k];
  }
  __syncthreads();
  if (wave > 0 || i >= n * vecs) return;
#pragma unroll
  for (int w = 0; w < 3; ++w)
#pragma unroll
    for (int k = 0; k < VEC; ++k) f[k] += part_s[w][k][lane];
  const float scale = *a.scale;
#pragma unroll
  for (int k = 0; k < VEC; ++k) f[k] *= scale;
  store_left<T>((T*)a.dx + (int64_t)a.idx[row] * a.D + c, f, a.D - c);
}

// dw of few rows: x^T P, a reduction of kFewRows at most.  P's fragments of 32 CW columns stay in a wave's registers
// while it walks its part of dw's rows; a lane ends up with CW neighbouring columns of a row, so the 512 bytes
// of a row go out at once, at any alignment, without LDS.  ROWS: 32 or 64.  Bound by dw's bytes: 24 x 2048 x 32000 bf16
// 28 us, 4.7 TB/s; 40 x 2048 x 50257 55 us, 3.7 (63 with neighbouring columns on different XCDs: rows of an odd length share
// cache lines there).
template <typename T, int ROWS>
__global__ __launch_bounds__(256) void lce_few_dw_kernel(LceArgs a, int rows_per) {
  constexpr int VEC = kVec<T>, KL = VEC, KS = 2 * KL, STEPS = ROWS / KS;
  constexpr int CW = sizeof(T) == 2 && ROWS == 64 ? 4 : VEC, WORDS = CW * (int)sizeof(T) / 4;
  const int kept = *a.kept, n = chunk_kept(a), lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int at = by_xcd(blockIdx.x + blockIdx.y * gridDim.x, gridDim.x * gridDim.y), band = at / gridDim.x;
  const int n0 = (at - band * gridDim.x) * 32 * CW, col = n0 + (lane & 31) * CW;
  Vec16 b[STEPS][CW];  // fragment of column c: its KL values of the lane's rows
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    uint32_t v[KL][WORDS];
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      const int t = s * KS + KL * half + i;
      typedef uint32_t words __attribute__((ext_vector_type(WORDS)));
      const words x = *reinterpret_cast<const words*>((const T*)a.p + (int64_t)max(0, min(t, n - 1)) * a.Vp + min(col, a.Vp - CW));
#pragma unroll
      for (int w = 0; w < WORDS; ++w) v[i][w] = t < n ? x[w] : 0u;
    }
#pragma unroll
    for (int c = 0; c < CW; ++c)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if constexpr (sizeof(T) == 2)
          b[s][c].w[w] = __builtin_amdgcn_perm(v[2 * w + 1][c >> 1], v[2 * w][c >> 1], c & 1 ? 0x07060302u : 0x05040100u);
        else
          b[s][c].w[w] = v[w][c];
      }
  }
  const float scale = kept > 0 ? *a.scale : 1.0f;
  const int from = (band * 4 + wave) * rows_per, to = min(a.D, from + rows_per);
  for (int d0 = from; d0 < to; d0 += 32) {
    const T* xt = (const T*)a.xt + (int64_t)min(d0 + (lane & 31), a.D - 1) * kFewRows;
    Vec16 x[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) x[s] = ld16(xt + s * KS + KL * half);
    f32x16_t acc[CW];
#pragma unroll
    for (int c = 0; c < CW; ++c)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[c][q] = 0.f;
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int c = 0; c < CW; ++c) MfmaOp<T, 32>::run(acc[c], x[s], b[s][c]);
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      const int d = d0 + 8 * (q >> 2) + 4 * half + (q & 3);
      if (d >= to || col >= a.V) continue;
      T* out = (T*)a.dw + (int64_t)d * a.V + col;
      float f[VEC] = {};
#pragma unroll
      for (int c = 0; c < CW; ++c) f[c] = acc[c][q] * scale;
      if constexpr (CW == VEC) {
        store_left<T>(out, f, a.V - col);
      } else {
        typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
        if (col + CW <= a.V) *reinterpret_cast<u32x2_any*>(out) = u32x2_any{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])};
        else st8_any(out, Vec16{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])}, a.V - col);
      }
    }
  }
}

// The slices of a product's tiles added in slice order, bound by their bytes: of 8192 x 1024 in 32 x 4 tiles 14 us, 18 with the
// losses' sum beside them.
template <typename T, int KIND, int BMT>
__global__ __launch_bounds__(256) void lce_reduce_kernel(LceArgs a) {
  constexpr int BN = Geo<BMT, T>::BN, VEC = kVec<T>, CV = BN / VEC;
  if (KIND == kDx && a.add && blockIdx.x + 1 == gridDim.x) {
    add_losses(a);
    return;
  }
  const int kept = *a.kept, n = chunk_kept(a);
  if (n == 0) return;
  const Cover<T, KIND, BMT> cv(a, n);
  if (cv.slices <= 1) return;
  const int r = blockIdx.x / (BMT / kReduceRows), band = blockIdx.x % (BMT / kReduceRows);
  if (r >= cv.mt * cv.nt) return;
  int mt, nt;
  row_tile(r, cv.mt, cv.nt, mt, nt);
  const float* tile = a.parts + (int64_t)r * cv.slices * (BMT * BN);
  const float scale = *a.scale;
  const bool whole = KIND == kDx ? a.D == a.Dp : a.V == a.Vp;
  for (int v = threadIdx.x; v < kReduceRows * CV; v += 256) {
    const int tr = band * kReduceRows + v / CV, tc = v % CV * VEC;
    const int row = mt * BMT + tr, col = nt * BN + tc;
    if (row >= cv.M || col >= cv.N) continue;
    float f[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) f[k] = 0.f;
    for (int s0 = 0; s0 < cv.slices; s0 += 4) {
      float4 x[4][VEC / 4];
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int k = 0; k < VEC / 4; ++k)
          x[s][k] = *reinterpret_cast<const float4*>(tile + (int64_t)min(s0 + s, cv.slices - 1) * (BMT * BN) + tr * BN + tc + 4 * k);
#pragma unroll
      for (int s = 0; s < 4; ++s)
        if (s0 + s < cv.slices)
#pragma unroll
          for (int k = 0; k < VEC / 4; ++k) {
            f[4 * k] += x[s][k].x;
            f[4 * k + 1] += x[s][k].y;
            f[4 * k + 2] += x[s][k].z;
            f[4 * k + 3] += x[s][k].w;
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
    store_grad<T, KIND>(a, scale, row, col, f, whole);
  }
}

// ---------------------------------------------------------------- the rows' losses and P

// Rows of a block.  The strips' statistics of kRowsB rows are joined by 256 / kRowsB threads a row; then P takes the
// place of the exponentials, P = exp(l - m) * (s exp(m - top) / sum), at the target s (p - 1) from its fp32 logit.
constexpr int kRowsB = 8;
constexpr int kStripsB = 512;  // strips whose factors are in LDS at a time
constexpr int kAheadB = 4;     // vectors of a thread in flight

// A row group's work-groups take seg strips each (grid.y) and, where that leaves CUs without work, every grid.z-th row of it:
// 24 x 16000 bf16 11 us with all 8 rows in turn, under 6 so.  Bound by P's bytes, there and back: 8188 x 32000 bf16 210 us,
// 5.0 TB/s; 1793 x 50257 79 us.
template <typename T>
__global__ __launch_bounds__(256) void lce_rows_kernel(LceArgs a, int strip, int seg) {
  constexpr int VEC = kVec<T>, G = 256 / kRowsB;
  __shared__ float2 part_s[4][kRowsB];
  __shared__ float2 row_s[kRowsB];  // maximum, 1 / sum
  __shared__ float factor_s[kStripsB];
  const int tid = threadIdx.x, n = chunk_kept(a), row0 = blockIdx.x * kRowsB, base = a.chunk * a.chunk_rows;
  if (row0 >= n) return;
  const int strips = (a.V + strip - 1) / strip;
  auto join = [](float& m, float& s, float2 o) {
    const float top = fmaxf(m, o.x);
    s = s * exp_from(m, top) + o.y * exp_from(o.x, top);
    m = top;
  };
  {
    const int r = tid % kRowsB, g = tid / kRowsB, row = min(row0 + r, n - 1);
    float m = -3.0e38f, s = 0.f;  // (no strip's maximum is less)
    for (int k = g; k < strips; k += 4 * G) {
      float2 st[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) st[u] = a.stats[(int64_t)min(k + u * G, strips - 1) * a.chunk_rows + row];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (k + u * G < strips) join(m, s, st[u]);
    }
#pragma unroll
    for (int off = kRowsB; off < 64; off <<= 1) join(m, s, make_float2(__shfl_xor(m, off, 64), __shfl_xor(s, off, 64)));
    if ((tid & 63) < kRowsB) part_s[tid >> 6][r] = make_float2(m, s);
  }
  __syncthreads();
  if (tid < kRowsB) {
    float m = part_s[0][tid].x, s = part_s[0][tid].y;
    for (int w = 1; w < 4; ++w) join(m, s, part_s[w][tid]);
    row_s[tid] = make_float2(m, 1.0f / s);
    const int row = row0 + tid;
    if (row < n && blockIdx.y == 0 && blockIdx.z == 0) {
      // the target's distance from the maximum first: it is small where the loss is
      const float l = __builtin_fmaf(kLn2, __builtin_amdgcn_logf(s), m - a.target_logit[base + row]);
      if (a.reduction == ABACUS_LOSS_ROWS) {
        if (a.loss) a.loss[a.idx[base + row]] = l;
      } else {
        a.row_loss[base + row] = l;
      }
    }
  }
  if (!a.grad) return;
  if (row0 == 0 && blockIdx.y == 0 && blockIdx.z == 0 && !a.xt && tid >= 128) {  // for the products that follow, a wave each
    const int cut = tid < 192 ? (a.thin & 1 << kDx ? Cover<T, kDx, THIN>(a, n).cut(a) : Cover<T, kDx, BM>(a, n).cut(a))
                              : (a.thin & 1 << kDw ? Cover<T, kDw, THIN>(a, n).cut(a) : Cover<T, kDw, BM>(a, n).cut(a));
    if (tid % 64 == 0) a.slices[tid < 192 ? kDx : kDw] = cut;
  }
  __syncthreads();
  const int first = blockIdx.y * seg, last = min(strips, first + seg);
  for (int r = blockIdx.z; r < min(kRowsB, n - row0); r += gridDim.z) {
    const int row = row0 + r;
    const float top = row_s[r].x, inv = row_s[r].y;
    const float s = a.row_grad ? a.row_grad[a.idx[base + row]] / *a.scale : 1.0f;
    const int t = a.tgt[base + row];
    T* p = (T*)a.p + (int64_t)row * a.Vp;
    for (int k0 = first; k0 < last; k0 += kStripsB) {
      __syncthreads();
      for (int k = tid; k < min(kStripsB, last - k0); k += 256)
        factor_s[k] = s * inv * exp_from(a.stats[(int64_t)(k0 + k) * a.chunk_rows + row].x, top);
      __syncthreads();
      const int end = min(a.Vp, min(last, k0 + kStripsB) * strip);
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
            const float pt = inv * exp_from(a.target_logit[base + row], top);
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

// t *= *g (blockIdx.y 1: u), left alone where *g is 1 (a launch, 4 us).
template <typename T>
__global__ __launch_bounds__(256) void scale_kernel(T* __restrict__ t, int64_t n, T* __restrict__ u, int64_t m,
                                                    const float* __restrict__ g) {
  const float f = *g;
  if (f == 1.0f) return;
  if (blockIdx.y) {
    t = u;
    n = m;
  }
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
  int few;            // few rows: columns a lane of their logits; 0: tiles
  int64_t kept, idx, tgt, target_logit, row_loss, xc, xt, w, stats, p, acc, parts, total;
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

int few_slices(int64_t D) { return (int)std::max<int64_t>(1, 2 * kCUs / ((D + 63) / 64)); }

// Columns a lane: as many (registers for two work-groups a CU) as leave work for most CUs.  (24 x 2048 x 32000 bf16: 4 columns
// 250 work-groups, 39 us, 2 columns 500, 44 us.)
template <typename T>
int few_columns(int64_t V) {
  constexpr int least = sizeof(T) == 2 ? 2 : 1;
  int cw = 4;
  while (cw > least && (V + 32 * cw - 1) / (32 * cw) < 180) cw /= 2;
  return cw;
}

template <typename T>
Plan plan_of(int64_t T_, int64_t D, int64_t V, bool grad) {
  constexpr int VEC = VecTraits<T>::kN;
  Plan q;
  q.Dp = (int)((D + VEC - 1) / VEC * VEC);
  q.Vp = (int)((V + VEC - 1) / VEC * VEC);
  // a strip is half a tile's columns; with gradients a row of P is in a chunk as a whole
  const int64_t row_bytes = grad ? (int64_t)q.Vp * (int64_t)sizeof(T) : (V + 31) / 32 * 8;
  const int64_t rows = std::min(T_, std::max<int64_t>(BM, std::min(kChunkBytes / row_bytes, kChunkRows) / BM * BM));
  q.chunk_rows = (int)rows;
  q.chunks = (int)((T_ + rows - 1) / rows);
  q.thin[kLogits] = thin_of<T, kLogits>(rows, D, V);
  q.thin[kDx] = thin_of<T, kDx>(rows, D, V);
  q.thin[kDw] = thin_of<T, kDw>(rows, D, V);
  q.few = T_ <= kFewRows && V >= 64 ? few_columns<T>(V) : 0;
  // (few rows read w at any alignment, and at least 64 of its columns at a time)
  q.pad = V % VEC != 0 && !q.few;
  q.strip = q.few ? 32 * q.few : q.thin[kLogits] ? Geo<THIN, T>::WTN : Geo<BM, T>::WTN;
  const int64_t strips = (V + q.strip - 1) / q.strip;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  q.kept = take(20);
  q.idx = take(T_ * 4);
  q.tgt = take(T_ * 4);
  q.target_logit = take(T_ * 4);
  q.row_loss = take(T_ * 4);
  q.xc = take(T_ * q.Dp * (int64_t)sizeof(T));
  q.w = take(q.pad ? D * q.Vp * (int64_t)sizeof(T) : 0);
  q.xt = take(q.few && grad ? D * kFewRows * (int64_t)sizeof(T) : 0);
  q.stats = take(strips * rows * 8);
  q.p = take(grad ? rows * row_bytes : 0);
  q.acc = take(grad && q.chunks > 1 ? (D + BM - 1) / BM * BM * ((V + BN - 1) / BN * BN) * 4 : 0);
  if (q.few) q.parts = take(grad ? (int64_t)few_slices(D) * kFewRows * q.Dp * 4 : 0);
  else q.parts = take(grad ? std::max(part_bytes<T, kDx>(q.thin[kDx], rows, D, V), part_bytes<T, kDw>(q.thin[kDw], rows, D, V)) : 0);
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

template <typename T, int CW>
int launch_few_columns(const LceArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.V + 32 * CW - 1) / (32 * CW))), block(kFewWaves * 64);
  if (a.T <= 32) hipLaunchKernelGGL((lce_few_kernel<T, CW, 1>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((lce_few_kernel<T, CW, 2>), grid, block, 0, s, a);
  ABACUS_CHECK_LAUNCH("linear_cross_entropy few rows");
  return 0;
}
template <typename T>
int launch_few(const LceArgs& a, int cw, hipStream_t s) {
  if (cw == 4) return launch_few_columns<T, 4>(a, s);
  if (cw == 2) return launch_few_columns<T, 2>(a, s);
  if constexpr (sizeof(T) == 4) return launch_few_columns<T, 1>(a, s);
  return 1;  // (not reached: few_columns gives bf16 two at least)
}

template <typename T>
int launch_few_dx(const LceArgs& a, hipStream_t s) {
  const int slices = few_slices(a.D);
  const dim3 grid((unsigned)((a.D + 63) / 64), (unsigned)slices), block(kFewWaves * 64);
  if (a.T <= 32) hipLaunchKernelGGL((lce_few_dx_kernel<T, 1>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((lce_few_dx_kernel<T, 2>), grid, block, 0, s, a);
  ABACUS_CHECK_LAUNCH("linear_cross_entropy few rows' dx");
  const int64_t vecs = (int64_t)a.T * (a.Dp / VecTraits<T>::kN);
  hipLaunchKernelGGL(lce_few_sum_kernel<T>, dim3((unsigned)((vecs + 63) / 64 + a.add)), dim3(256), 0, s, a, slices);
  ABACUS_CHECK_LAUNCH("linear_cross_entropy few rows' dx sum");
  return 0;
}

template <typename T>
int launch_few_dw(const LceArgs& a, hipStream_t s) {
  const int cols = 32 * (sizeof(T) == 2 && a.T > 32 ? 4 : VecTraits<T>::kN);
  // rows of dw a wave walks: enough waves for every SIMD twice, and P's fragments used as often as that allows
  const int64_t groups = (a.V + cols - 1) / cols;
  int rows_per = 256;
  while (rows_per > 32 && groups * ((a.D + rows_per - 1) / rows_per) < 8 * kCUs) rows_per /= 2;
  const dim3 grid((unsigned)groups, (unsigned)((a.D + 4 * rows_per - 1) / (4 * rows_per)));
  if (a.T <= 32) hipLaunchKernelGGL((lce_few_dw_kernel<T, 32>), grid, dim3(256), 0, s, a, rows_per);
  else hipLaunchKernelGGL((lce_few_dw_kernel<T, 64>), grid, dim3(256), 0, s, a, rows_per);
  ABACUS_CHECK_LAUNCH("linear_cross_entropy few rows' dw");
  return 0;
}

template <typename T, int BMT>
int launch_logits(const LceArgs& a, hipStream_t s) {
  const int64_t tiles = Sizes<T, kLogits, BMT>(std::min(a.chunk_rows, a.T - a.chunk * a.chunk_rows), a.D, a.V).tiles;
  ABACUS_CHECK_ARG(tiles < (1ll << 31) - 8, "linear_cross_entropy: %lld tiles", (long long)tiles);
  const dim3 grid((unsigned)std::min<int64_t>(kCUs, (tiles + 7) / 8 * 8));
#define ABACUS_GO(RK)                                                                                  \
  do {                                                                                                 \
    if (a.grad) hipLaunchKernelGGL((lce_logits_kernel<T, BMT, RK, true>), grid, dim3(NT), 0, s, a);    \
    else hipLaunchKernelGGL((lce_logits_kernel<T, BMT, RK, false>), grid, dim3(NT), 0, s, a);          \
  } while (0)
  if (a.D % kBKT<T> != 0) ABACUS_GO(true);
  else ABACUS_GO(false);
#undef ABACUS_GO
  ABACUS_CHECK_LAUNCH("linear_cross_entropy logits");
  return 0;
}

template <typename T, int KIND, int BMT>
int launch_product(const LceArgs& a, hipStream_t s) {
  const int64_t tiles = Sizes<T, KIND, BMT>(std::min(a.chunk_rows, a.T - a.chunk * a.chunk_rows), a.D, a.V).tiles;
  // a product of fewer rows (or a shorter reduction) may be cut into more slices, up to kUnits units
  const int64_t units = (std::max<int64_t>(tiles, std::min<int64_t>(kUnits, tiles * kSlices)) + 7) / 8 * 8;
  ABACUS_CHECK_ARG(units < (1ll << 31), "linear_cross_entropy: %lld tiles", (long long)units);
  const dim3 grid((unsigned)units);
  if constexpr (KIND == kDw) {
    if (a.chunks > 1) hipLaunchKernelGGL((lce_product_kernel<T, KIND, BMT, true, true>), grid, dim3(NT), 0, s, a);
    else hipLaunchKernelGGL((lce_product_kernel<T, KIND, BMT, true, false>), grid, dim3(NT), 0, s, a);
  } else if (a.Vp % kBKT<T> != 0) {
    hipLaunchKernelGGL((lce_product_kernel<T, KIND, BMT, true, false>), grid, dim3(NT), 0, s, a);
  } else {
    hipLaunchKernelGGL((lce_product_kernel<T, KIND, BMT, false, false>), grid, dim3(NT), 0, s, a);
  }
  ABACUS_CHECK_LAUNCH("linear_cross_entropy product");
  if (KIND == kDx || 2 * tiles <= kUnits) {  // (two slices or more are of at most kUnits / 2 tiles)
    const int64_t cut = std::min<int64_t>(tiles, kUnits / 2);
    hipLaunchKernelGGL((lce_reduce_kernel<T, KIND, BMT>), dim3((unsigned)(cut * (BMT / kReduceRows) + (KIND == kDx ? a.add : 0))), dim3(256), 0, s, a);
    ABACUS_CHECK_LAUNCH("linear_cross_entropy reduce");
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
  a.scale = (float*)(ws + q.kept) + 1;
  a.slices = (int*)(ws + q.kept) + 2;
  a.idx = (int*)(ws + q.idx);
  a.tgt = (int*)(ws + q.tgt);
  a.target_logit = (float*)(ws + q.target_logit);
  a.row_loss = (float*)(ws + q.row_loss);
  a.xc = ws + q.xc;
  a.xt = q.few && a.grad ? ws + q.xt : nullptr;
  a.stats = (float2*)(ws + q.stats);
  a.p = ws + q.p;
  a.acc = (float*)(ws + q.acc);
  a.parts = (float*)(ws + q.parts);
  a.ldv = a.V;
  const int rows_per = std::min(4096, std::max(4, (a.T + 511) / 512));
  if (q.few) hipLaunchKernelGGL(pack_few_kernel<T>, dim3((a.Dp + 63) / 64), dim3(256), 0, s, a);
  else hipLaunchKernelGGL(pack_rows_kernel<T>, dim3((a.T + rows_per - 1) / rows_per), dim3(256), rows_per * 4, s, a, rows_per);
  ABACUS_CHECK_LAUNCH("linear_cross_entropy pack");
  if (q.pad) {
    const dim3 grid((unsigned)((q.Vp / VecTraits<T>::kN + 255) / 256), (unsigned)((a.D + kPadRows - 1) / kPadRows));
    hipLaunchKernelGGL(pad_w_kernel<T>, grid, dim3(256), 0, s, (const T*)a.w, a.D, a.V, q.Vp, (T*)(ws + q.w));
    ABACUS_CHECK_LAUNCH("linear_cross_entropy pad");
    a.w = ws + q.w;
    a.ldv = q.Vp;
  }
  a.chunks = q.chunks;
  a.thin = q.thin[kDx] << kDx | q.thin[kDw] << kDw;
  const bool one_loss = a.reduction != ABACUS_LOSS_ROWS && a.loss;
  for (a.chunk = 0; a.chunk < q.chunks; ++a.chunk) {
    a.add = one_loss && a.dx && a.chunk + 1 == q.chunks;
    if (int rc = q.few ? launch_few<T>(a, q.few, s) : q.thin[kLogits] ? launch_logits<T, THIN>(a, s) : launch_logits<T, BM>(a, s)) return rc;
    const int rows = std::min(a.chunk_rows, a.T - a.chunk * a.chunk_rows);
    // (work-groups enough for every CU twice, of a few strips at least)
    const int groups = (rows + kRowsB - 1) / kRowsB, strips = (a.V + q.strip - 1) / q.strip;
    const int segs = a.grad ? std::max(1, std::min(2 * kCUs / groups, strips / 8)) : 1, seg = (strips + segs - 1) / segs;
    const int pieces = (strips + seg - 1) / seg, turns = a.grad ? std::max(1, std::min(kRowsB, 4 * kCUs / (groups * pieces))) : 1;
    hipLaunchKernelGGL(lce_rows_kernel<T>, dim3(groups, pieces, turns), dim3(256), 0, s, a, q.strip, seg);
    ABACUS_CHECK_LAUNCH("linear_cross_entropy rows");
    if (a.dx) {
      if (int rc = q.few ? launch_few_dx<T>(a, s) : q.thin[kDx] ? launch_product<T, kDx, THIN>(a, s) : launch_product<T, kDx, BM>(a, s)) return rc;
    }
    if (a.dw) {
      if (int rc = q.few ? launch_few_dw<T>(a, s) : q.thin[kDw] ? launch_product<T, kDw, THIN>(a, s) : launch_product<T, kDw, BM>(a, s)) return rc;
    }
  }
  if (one_loss && !a.dx) {
    hipLaunchKernelGGL(lce_sum_kernel, dim3(1), dim3(256), 0, s, a);
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
  ABACUS_CHECK_ARG(T > 0, "linear_cross_entropy: no rows");
  ABACUS_CHECK_ARG(x_TD && w_DV && targets_T, "linear_cross_entropy: null pointer");
  ABACUS_CHECK_ARG(((uintptr_t)w_DV | (uintptr_t)dx_TD | (uintptr_t)dw_DV | (uintptr_t)ws) % 16 == 0,
                   "linear_cross_entropy: w, the gradients and the workspace must be 16-byte aligned");
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

int abacus_capture_id(int64_t* id, void* stream) {
  ABACUS_CHECK_ARG(id != nullptr, "capture_id: no place for the answer");
  hipStreamCaptureStatus status;
  unsigned long long at = 0;
  const hipError_t rc = hipStreamGetCaptureInfo((hipStream_t)stream, &status, &at);
  ABACUS_CHECK_ARG(rc == hipSuccess, "capture_id: %s", hipGetErrorString(rc));
  *id = status == hipStreamCaptureStatusActive ? (int64_t)at : 0;
  return 0;
}

int abacus_scale_by(void* t, int64_t n, void* u, int64_t m, int dtype, const float* g, void* stream) {
  ABACUS_CHECK_ARG(dtype == kF32 || dtype == kBF16, "scale_by: unsupported dtype code %d (0 = fp32, 1 = bf16)", dtype);
  ABACUS_CHECK_ARG(n >= 0 && m >= 0, "scale_by: %lld and %lld values", (long long)n, (long long)m);
  if (n == 0 && m == 0) return 0;
  ABACUS_CHECK_ARG(g && (t || n == 0) && (u || m == 0), "scale_by: null pointer");
  ABACUS_CHECK_ARG(((uintptr_t)t | (uintptr_t)u) % 16 == 0, "scale_by: values must be 16-byte aligned");
  const dim3 grid((unsigned)std::min<int64_t>((std::max(n, m) + 2047) / 2048, 4096), 2);
  if (dtype == kBF16)
    hipLaunchKernelGGL(scale_kernel<uint16_t>, grid, dim3(256), 0, (hipStream_t)stream, (uint16_t*)t, n, (uint16_t*)u, m, g);
  else
    hipLaunchKernelGGL(scale_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, (float*)t, n, (float*)u, m, g);
  ABACUS_CHECK_LAUNCH("scale_by");
  return 0;
}

}  // extern "C"
