// Verification of drafted tokens against the target's probabilities, from given
// random numbers.
//
// p = softmax(target / temperature), q = softmax(draft / temperature), row by row.  The
// draft x after row t is accepted where u0 q(x) < p(x); after the first rejection the
// next token is drawn from max(p - q, 0) by its running sum, with all accepted from the
// last row's p.  So the tokens that come out are distributed as the target's own.
//
// The outcome is integers that a border between two tokens decides, so exponentials and
// sums are in 64 bits: the result is that of the formula unless a random number lies
// within 1e-13 of a border.  Sums run in a fixed order.
//
// Two launches over slices of kSlice logits: every row's slice maxima and sums; then each
// sequence's decision and the slice sums of the mass that its next token is drawn from,
// whose last block to end draws it from the slice that the random number falls into (which
// block that is changes nothing).  Probabilities are never written out: logits are read
// once, and once more for the one row that a token is drawn from.  Temperature 0 takes
// maxima alone.
//
// The first launch is bound by its exponentials: some 20 instructions of 64 bits a logit, 10 us
// of arithmetic for the 576 rows of 32000 bf16 logits that 64 sequences with 4 drafts have,
// beside 6 us of reading; it takes 20 us.  The second is bound by latency (15 us there): what
// it reads depends on what it has read, from the row numbers to the blocks' counts.
#include <algorithm>

#include "paged_rows.h"

namespace abacus {
namespace {

constexpr int kSlice = 8192;  // logits of a block of the first launch
constexpr int kEach = 8, kThreads = 512, kWaves = kThreads / 64;  // of the second: the draw is one block's work
constexpr int kMassSlice = kEach * kThreads;

struct VerifyArgs {
  const void *target, *draft;
  const int64_t* tokens;
  const int* query_start;
  const float* uniforms;
  int T, S, slices, mass_slices;
  int64_t V;
  double to_log2;  // log2(e) / temperature, for logits less their maximum (products first would lose digits)
  bool greedy;
  int32_t* accepted;
  int64_t* next;
  double* sums;   // [2][T][slices]: of exp((x - slice max) / temperature)
  double* mass;   // [S][mass_slices]
  float* tops;    // [2][T][slices]: slice maxima, NaN where there is one
  float* drafted; // [2][T]: the logit of the draft after the row
  int* at;        // [T][slices]: where (greedy)
  int* ended;     // [S]: blocks that are done with the sequence
  int* good;      // [1]: the sequences before the first bad range
};

template <typename T> struct alignas(sizeof(T)) Loose { T v[16 / sizeof(T)]; };  // 16 bytes at any element

// 8 logits of a row from i0 on, and 8 more `step` further each time; -inf past its end.
template <typename T, int Each>
__device__ inline void load_logits(const T* row, int64_t i0, int64_t step, int64_t V, float (&x)[Each]) {
  constexpr int N = 16 / sizeof(T);
  static_assert(Each % 8 == 0, "whole loads");
#pragma unroll
  for (int c = 0; c < Each / N; ++c) {
    const int64_t i = i0 + c * N / 8 * step + c * N % 8;
    if (i + N <= V) {
      const Loose<T> w = *reinterpret_cast<const Loose<T>*>(row + i);
#pragma unroll
      for (int e = 0; e < N; ++e) x[c * N + e] = to_f32(w.v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) x[c * N + e] = i + e < V ? to_f32(row[i + e]) : -__builtin_inff();
    }
  }
}

// maximum that keeps a NaN
__device__ inline float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Over a wave, in a fixed order and without LDS: rows of 16 lanes by DPP, then the four rows.
template <int kCtrl> __device__ inline float moved(float x) {
  return bits_f32((uint32_t)dpp_or_0<kCtrl>((int)f32_bits(x)));
}
template <int kCtrl> __device__ inline double moved(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)dpp_or_0<kCtrl>((int)(uint32_t)u), hi = (uint32_t)dpp_or_0<kCtrl>((int)(u >> 32));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ inline double lane_of(double x, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ inline float wave_max(float x) {
  x = max_nan(x, moved<0x121>(x));  // row_ror:1, 2, 4, 8
  x = max_nan(x, moved<0x122>(x));
  x = max_nan(x, moved<0x124>(x));
  x = max_nan(x, moved<0x128>(x));
  float r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = bits_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_bits(x), 16 * i));
  return max_nan(max_nan(r[0], r[1]), max_nan(r[2], r[3]));
}
__device__ inline double wave_sum64(double x) {
  x += moved<0x121>(x);
  x += moved<0x122>(x);
  x += moved<0x124>(x);
  x += moved<0x128>(x);
  return (lane_of(x, 0) + lane_of(x, 16)) + (lane_of(x, 32) + lane_of(x, 48));
}
// inclusive sums over the lanes; `total` the whole wave's
__device__ inline double wave_scan64(double x, double& total) {
  x += moved<0x111>(x);  // row_shr:1, 2, 4, 8
  x += moved<0x112>(x);
  x += moved<0x114>(x);
  x += moved<0x118>(x);
  const double r0 = lane_of(x, 15), r1 = r0 + lane_of(x, 31), r2 = r1 + lane_of(x, 47);
  const int row = (threadIdx.x & 63) >> 4;
  x += row == 0 ? 0.0 : row == 1 ? r0 : row == 2 ? r1 : r2;
  total = lane_of(x, 63);
  return x;
}

// 2^y for y <= 0 (2^-1000 below that): y = n + f with |f| <= 1/2, and the polynomial of
// degree 9 that is 2^f at the ten Chebyshev nodes, off by at most 1.9e-14 of it and the
// roundings.  n comes from the addition that rounds and goes straight into the exponent's
// bits.  N values step by step, as each step waits for the one before.
template <int N>
__device__ inline void exp2_64(double (&y)[N]) {
  constexpr double kRound = 0x1.8p52;
  constexpr double c[] = {1.0205905413765595e-07, 1.325964524488711e-06, 1.5252672924850737e-05,
                          0.0001540343375125101,  0.0013333558200794592, 0.009618129193934313,
                          0.05550410866465167,    0.2402265069564034,    0.6931471805599462,
                          1.0000000000000135};
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  uint32_t n[N];
  double s[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    y[i] = fmax(y[i], -1000.0);
    const double shifted = y[i] + kRound;
    n[i] = (uint32_t)__builtin_bit_cast(uint64_t, shifted) << 20;  // its low bits
    y[i] -= shifted - kRound;
    s[i] = c[0];
  }
#pragma unroll
  for (int k = 1; k < 10; ++k)
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = fma(s[i], y[i], c[k]);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const u32x2 u = __builtin_bit_cast(u32x2, s[i]);
    y[i] = __builtin_bit_cast(double, u32x2{u[0], u[1] + n[i]});
  }
}
__device__ inline double exp2_64(double y) {
  double x[1] = {y};
  exp2_64(x);
  return x[0];
}

// The rows of sequence s, none from the first bad range on (as paged_rows.h has it).
__device__ inline void rows_of(const VerifyArgs& a, int s, int& first, int& n) {
  const int b = a.query_start[s], e = a.query_start[s + 1];
  const bool in = range_in(b, e, a.T) && s < *a.good; // (with T = 0 nothing has counted them)
  first = in ? b : 0;
  n = in ? e - b : 0;
}

template <int N>
__device__ inline double block_sum(const double (&w)[N]) {
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < N; ++i) s += w[i];
  return s;
}

// One row's slice: its maximum (and, greedy, its place) and sum.  blockIdx: slice, row,
// target or draft.  Threads: 256 with 32 logits each where there are rows enough to fill the
// GPU, 1024 with 8 where there are not.
template <typename T, int Threads>
__global__ __launch_bounds__(Threads) void verify_rows_kernel(VerifyArgs a) {
  constexpr int Each = kSlice / Threads, Waves = Threads / 64;
  __shared__ float top_w[Waves];
  __shared__ int at_w[Waves];
  __shared__ double sum_w[Waves];
  __shared__ int first_bad;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int slice = blockIdx.x, row = blockIdx.y, which = blockIdx.z;
  if (which == 0 && slice == 0 && tid == 0)
    for (int s = row; s < a.S; s += a.T) a.ended[s] = 0;
  const int64_t i0 = (int64_t)slice * kSlice + tid * 8;
  if (tid == 0 && !a.greedy && row + 1 < a.T) {  // read here, where nothing waits for it
    const int64_t x = a.tokens[row + 1];
    if (x >= 0 && x < a.V && x / kSlice == slice)
      a.drafted[which * a.T + row] = to_f32(((const T*)(which ? a.draft : a.target))[row * a.V + x]);
  }
  float x[Each];
  load_logits((const T*)(which ? a.draft : a.target) + row * a.V, i0, 8 * Threads, a.V, x);
  if (which == 1) {  // a sequence's last row has no draft after it (those from the first bad range on do not count)
    uint64_t bad = 0, end = 0;
    for (int s = lane; s - lane < a.S && !(bad | end); s += 64) {
      const int b = s < a.S ? a.query_start[s] : 0, e = s < a.S ? a.query_start[s + 1] : 0;
      bad = __ballot(!range_in(b, e, a.T));
      end = __ballot(e == row + 1);
    }
    if (end && (!bad || __builtin_ctzll(end) < __builtin_ctzll(bad))) return;
  } else if (row == 0 && slice == 0) {  // the sequences before that range, for the second launch
    if (tid == 0) first_bad = a.S;
    __syncthreads();
    int bad = a.S;
    for (int s = tid; s < a.S; s += Threads)
      if (!range_in(a.query_start[s], a.query_start[s + 1], a.T)) bad = min(bad, s);
    if (bad < a.S) atomicMin(&first_bad, bad);
    __syncthreads();
    if (tid == 0) *a.good = first_bad;
  }
  float top = x[0];
#pragma unroll
  for (int e = 1; e < Each; ++e) top = max_nan(top, x[e]);
  const float wave_top = wave_max(top);
  if (lane == 0) top_w[wave] = wave_top;
  if (a.greedy) {
    int at = 0x7fffffff;  // the lowest place that has it
#pragma unroll
    for (int e = Each - 1; e >= 0; --e)
      if (x[e] == wave_top) at = (int)i0 + e / 8 * 8 * Threads + e % 8;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) at = min(at, __shfl_xor(at, off, 64));
    if (lane == 0) at_w[wave] = at;
  }
  __syncthreads();
  top = top_w[0];
#pragma unroll
  for (int w = 1; w < Waves; ++w) top = max_nan(top, top_w[w]);
  const int64_t out = ((int64_t)which * a.T + row) * a.slices + slice;
  if (a.greedy) {
    if (tid == 0) {
      int at = 0x7fffffff;
      for (int w = 0; w < Waves; ++w)
        if (top_w[w] == top) at = min(at, at_w[w]);
      a.tops[out] = top, a.at[out] = at;
    }
    return;
  }
  double sum = 0.0;
  if (top > -__builtin_inff() && top < __builtin_inff()) {
    const double t = (double)top;
#pragma unroll
    for (int e = 0; e < Each; e += 4) {
      if ((int64_t)slice * kSlice + e / 8 * 8 * Threads >= a.V) break;  // (the same for all)
      double y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = ((double)x[e + i] - t) * a.to_log2;
      exp2_64(y);
      sum += (y[0] + y[1]) + (y[2] + y[3]);
    }
  }
  sum = wave_sum64(sum);
  if (lane == 0) sum_w[wave] = sum;
  __syncthreads();
  if (tid == 0) {
    a.tops[out] = top;
    a.sums[out] = block_sum(sum_w);
  }
}

struct RowStat {
  float top;   // NaN, +inf or -inf: no distribution
  double inv;  // 1 / sum of exp((x - top) / temperature)
  __device__ bool fine() const { return top > -__builtin_inff() && top < __builtin_inff(); }
};

// A row's maximum and sum from its slices', by one wave: lane l has slice l, 64 + l, ...
struct RowParts {
  float top;  // the first 64, read ahead
  double sum;
};
__device__ inline RowParts parts_of(const VerifyArgs& a, int which, int row) {
  const int lane = threadIdx.x & 63;
  const int64_t at = ((int64_t)which * a.T + row) * a.slices + lane;
  return lane < a.slices ? RowParts{a.tops[at], a.sums[at]} : RowParts{-__builtin_inff(), 0.0};
}
__device__ inline RowStat row_stat(const VerifyArgs& a, int which, int row, const RowParts& x) {
  const int lane = threadIdx.x & 63;
  const int64_t base = ((int64_t)which * a.T + row) * a.slices;
  float top = x.top;
  for (int i = 64 + lane; i < a.slices; i += 64) top = max_nan(top, a.tops[base + i]);
  RowStat r;
  r.top = wave_max(top);
  double sum = 0.0;
  if (r.fine()) {
    sum = x.sum * exp2_64(((double)x.top - (double)r.top) * a.to_log2);
    for (int i = 64 + lane; i < a.slices; i += 64)
      sum += a.sums[base + i] * exp2_64(((double)a.tops[base + i] - (double)r.top) * a.to_log2);
  }
  r.inv = 1.0 / wave_sum64(sum);
  return r;
}

__device__ inline double prob(const VerifyArgs& a, const RowStat& r, float x) {
  const double e = exp2_64(((double)x - (double)r.top) * a.to_log2);
  return e > 0x1p-999 ? e * r.inv : 0.0;  // (2^-1000 for a logit of -inf)
}

// Of a row's kEach logits at i0: the mass that the next token is drawn from; no
// token of -inf may come out.
template <typename T>
__device__ inline void masses(const VerifyArgs& a, int row, bool residual, int64_t drafted, const RowStat& p,
                              const RowStat& q, int64_t i0, double (&m)[kEach]) {
  float x[kEach], y[kEach];
  load_logits((const T*)a.target + row * a.V, i0, 0, a.V, x);
  if (residual && a.draft) load_logits((const T*)a.draft + row * a.V, i0, 0, a.V, y);
  const double p_top = (double)p.top, q_top = (double)q.top;
#pragma unroll
  for (int e0 = 0; e0 < kEach; e0 += 4) {  // (four at a time, for registers)
    double u[4], d[4] = {};
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = ((double)x[e0 + e] - p_top) * a.to_log2;
    exp2_64(u);
    if (residual && a.draft) {
#pragma unroll
      for (int e = 0; e < 4; ++e) d[e] = ((double)y[e0 + e] - q_top) * a.to_log2;
      exp2_64(d);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      u[e] = u[e] > 0x1p-999 ? u[e] * p.inv : 0.0;
      if (residual) u[e] = fmax(u[e] - (a.draft ? d[e] * q.inv : i0 + e0 + e == drafted ? 1.0 : 0.0), 0.0);
      m[e0 + e] = u[e];
    }
  }
}

constexpr int kKept = 32;  // rows whose maximum and sum a block keeps, of those it decides on

// blockIdx: slice, sequence.  Every block of a sequence decides alike and sums its slice's
// mass; the last to end draws.  (Six waves a SIMD, three blocks a CU: 124 fp32 sequences of
// 32000 logits 41 us with two, 38 with three.)
template <typename T>
__global__ __launch_bounds__(kThreads, 6) void verify_decide_kernel(VerifyArgs a) {
  __shared__ int stop, order;
  __shared__ double sum_w[kWaves];
  __shared__ RowStat kept[2][kKept];
  __shared__ long long token, best[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int slice = blockIdx.x, seq = blockIdx.y;
  int first, n;
  rows_of(a, seq, first, n);
  if (n == 0) {
    if (slice == 0 && tid == 0) {
      a.accepted[seq] = 0;
      a.next[seq] = -1;
    }
    return;
  }
  if (tid == 0) stop = n - 1, token = -1;
  __syncthreads();
  for (int j = wave; j < n; j += kWaves) {
    const int row = first + j;
    const bool draft = j < n - 1;  // (the last row is drawn from, should all be accepted)
    const bool both = draft && a.draft;
    // everything that is read, at once
    const RowParts pp = parts_of(a, 0, row), qp = both ? parts_of(a, 1, row) : pp;
    const int64_t x = draft ? a.tokens[row + 1] : -1;
    const bool known = x >= 0 && x < a.V;
    const float px = a.drafted[row], qx = both ? a.drafted[a.T + row] : 0.f;  // (anything, where it is not known)
    const float u = draft ? a.uniforms[2 * row] : 0.f;
    const RowStat p = row_stat(a, 0, row, pp), q = both ? row_stat(a, 1, row, qp) : p;
    if (j < kKept && lane == 0) kept[0][j] = p, kept[1][j] = q;
    const bool take = p.fine() && q.fine() && known && (double)u * (both ? prob(a, q, qx) : 1.0) < prob(a, p, px);
    if (draft && !take && lane == 0) atomicMin(&stop, j);
  }
  __syncthreads();
  const int j = stop, row = first + j;
  bool residual = j < n - 1;
  RowStat p, q;
  if (j < kKept) {
    p = kept[0][j], q = kept[1][j];
  } else {
    p = row_stat(a, 0, row, parts_of(a, 0, row));
    q = residual && a.draft ? row_stat(a, 1, row, parts_of(a, 1, row)) : p;
  }
  const int64_t drafted = residual ? a.tokens[row + 1] : -1;
  const bool fine = p.fine() && q.fine();
  if (slice == 0 && tid == 0) {
    a.accepted[seq] = j;
    if (!fine) a.next[seq] = -1;
  }
  if (!fine) return;
  double m[kEach], own = 0.0;
  masses<T>(a, row, residual, drafted, p, q, (int64_t)slice * kMassSlice + tid * kEach, m);
#pragma unroll
  for (int e = 0; e < kEach; ++e) own += m[e];
  double sum = wave_sum64(own);
  if (lane == 0) sum_w[wave] = sum;
  __syncthreads();
  double* mass = a.mass + (int64_t)seq * a.mass_slices;
  const bool alone = a.mass_slices == 1;
  // What passes between the blocks does so in agent-scope operations, which do not stop at
  // this XCD's L2; the store has ended before the count goes up.  (A release would write the
  // whole L2 back, once a block.)
  if (tid == 0 && !alone) {
    __hip_atomic_store(mass + slice, block_sum(sum_w), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    order = __hip_atomic_fetch_add(a.ended + seq, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!alone && order != a.mass_slices - 1) return;

  // the draw: the border, the slice whose end passes it first, the token in it
  auto mass_of = [&](int i) {
    return i < a.mass_slices ? __hip_atomic_load(mass + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
  };
  double total = alone ? block_sum(sum_w) : 0.0, before = 0.0;
  for (int s0 = 0; !alone && s0 < a.mass_slices; s0 += 64) {
    double part;
    wave_scan64(mass_of(s0 + lane), part);
    total += part;
  }
  const bool plain = !(total > 0.0);  // no mass is left of p - q: p itself, from its first slice
  if (plain) residual = false, total = 1.0;
  const double border = fmin((double)a.uniforms[2 * row + 1], 1.0 - 0x1p-53) * total;
  int at = 0;
  for (int s0 = 0; !plain && !alone && s0 < a.mass_slices; s0 += 64) {
    double part;
    const double x = mass_of(s0 + lane), upto = wave_scan64(x, part);
    const unsigned long long has = __ballot(s0 + lane < a.mass_slices && before + upto > border);
    const int l = has ? __ffsll(has) - 1 : min(63, a.mass_slices - 1 - s0);
    at = s0 + l;
    if (has || s0 + 64 >= a.mass_slices) {
      before += lane_of(upto - x, l);
      break;
    }
    before += part;
  }
  bool held = !plain;   // whether m are this block's slice's
  long long last = -1;  // the last token with any mass, should rounding leave none past the border
  for (; at < a.mass_slices; ++at) {
    const int64_t i0 = (int64_t)at * kMassSlice + tid * kEach;
    if (!held || at != slice) masses<T>(a, row, residual, drafted, p, q, i0, m);
    held = false;
    own = 0.0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      own += m[e];
      if (m[e] > 0.0) last = i0 + e;
    }
    double part;
    const double upto = wave_scan64(own, part);
    __syncthreads();  // (what was in sum_w is read)
    if (lane == 0) sum_w[wave] = part;
    __syncthreads();
    double run = before + (upto - own);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) run += sum_w[w];
      before += sum_w[w];
    }
    long long mine = -1;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      run += m[e];
      if (mine < 0 && m[e] > 0.0 && run > border) mine = i0 + e;
    }
    const unsigned long long has = __ballot(mine >= 0);  // the lowest lane that has one
    if (has ? lane == __ffsll(has) - 1 : lane == 0) best[wave] = mine;
    __syncthreads();
    if (tid == 0)
      for (int w = 0; w < kWaves && token < 0; ++w) token = best[w];
    __syncthreads();
    if (token >= 0) break;
  }
  if (token < 0) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) last = max(last, __shfl_xor(last, off, 64));
    if (lane == 0) best[wave] = last;
    __syncthreads();
    if (tid == 0)
      for (int w = 0; w < kWaves; ++w) token = max(token, best[w]);
    __syncthreads();
  }
  if (tid == 0) a.next[seq] = token;
}

// Temperature 0, a wave per sequence.
__global__ __launch_bounds__(64) void verify_greedy_kernel(VerifyArgs a) {
  const int lane = threadIdx.x, seq = blockIdx.x;
  int first, n;
  rows_of(a, seq, first, n);
  int j = 0;
  int64_t token = -1;
  for (; j < n; ++j) {
    const int64_t base = (int64_t)(first + j) * a.slices;
    float top = -__builtin_inff();
    int at = 0x7fffffff;
    for (int i = lane; i < a.slices; i += 64) {
      if (a.tops[base + i] > top) at = a.at[base + i];
      top = max_nan(top, a.tops[base + i]);
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const float other = __shfl_xor(top, off, 64);
      const int there = __shfl_xor(at, off, 64);
      at = other > top ? there : other == top ? min(at, there) : at;
      top = max_nan(top, other);
    }
    token = top > -__builtin_inff() && top < __builtin_inff() ? at : -1;
    if (j == n - 1 || token < 0 || token != a.tokens[first + j + 1]) break;
  }
  if (lane == 0) {
    a.accepted[seq] = j < n ? j : 0;
    a.next[seq] = token;
  }
}

inline int64_t slices_of(int64_t V) { return (V + kSlice - 1) / kSlice; }
inline int64_t mass_slices_of(int64_t V) { return (V + kMassSlice - 1) / kMassSlice; }

}  // namespace
}  // namespace abacus

using namespace abacus;

extern "C" int64_t abacus_verify_drafts_ws_bytes(int64_t T, int64_t V, int64_t S) {
  const int64_t n = slices_of(V);
  return (2 * T * n + S * mass_slices_of(V)) * 8 + 2 * T * n * 4 + 2 * T * 4 + T * n * 4 + (S + 1) * 4;
}

extern "C" int abacus_verify_drafts(const void* target_TV, const void* draft_TV, const int64_t* tokens_T,
                                    const int32_t* query_start, const float* uniforms_T2, int64_t T, int64_t V,
                                    int64_t S, int dtype, double temperature, int32_t* accepted_S, int64_t* next_S,
                                    void* ws, int64_t ws_bytes, void* stream) {
  ABACUS_CHECK_ARG(dtype == kF32 || dtype == kBF16, "verify_drafts: dtype code %d", dtype);
  ABACUS_CHECK_ARG(S >= 1 && S <= 65535 && T >= 0 && T <= 65535, "verify_drafts: %lld rows of %lld sequences",
                   (long long)T, (long long)S);
  ABACUS_CHECK_ARG(V >= 1 && V < (1ll << 30), "verify_drafts: a vocabulary of %lld", (long long)V);
  ABACUS_CHECK_ARG(temperature >= 0.0 && temperature < __builtin_inf(), "verify_drafts: temperature %g", temperature);
  ABACUS_CHECK_ARG(query_start && accepted_S && next_S && ws && (T == 0 || (target_TV && tokens_T)),
                   "verify_drafts: null pointer");
  ABACUS_CHECK_ARG(temperature == 0.0 || T == 0 || uniforms_T2, "verify_drafts: no random numbers");
  ABACUS_CHECK_ARG((uintptr_t)ws % 16 == 0 && ws_bytes >= abacus_verify_drafts_ws_bytes(T, V, S),
                   "verify_drafts: workspace of %lld bytes, need %lld", (long long)ws_bytes,
                   (long long)abacus_verify_drafts_ws_bytes(T, V, S));
  const int64_t n = slices_of(V);
  VerifyArgs a;
  a.target = target_TV, a.draft = temperature == 0.0 ? nullptr : draft_TV, a.tokens = tokens_T;
  a.query_start = query_start, a.uniforms = uniforms_T2;
  a.T = (int)T, a.S = (int)S, a.slices = (int)n, a.mass_slices = (int)mass_slices_of(V), a.V = V;
  a.greedy = temperature == 0.0;
  a.to_log2 = a.greedy ? 0.0 : std::min(1.4426950408889634 / temperature, 1e300);  // (0 times infinity)
  a.accepted = accepted_S, a.next = next_S;
  a.sums = (double*)ws;
  a.mass = a.sums + 2 * T * n;
  a.tops = (float*)(a.mass + S * a.mass_slices);
  a.drafted = a.tops + 2 * T * n;
  a.at = (int*)(a.drafted + 2 * T);
  a.ended = a.at + T * n;
  a.good = a.ended + S;
  hipStream_t s = (hipStream_t)stream;
  const dim3 rows((unsigned)n, (unsigned)T, a.draft ? 2 : 1), decide((unsigned)a.mass_slices, (unsigned)S);
  const bool bf = dtype == kBF16;
  if (T > 0) {
    const bool many = n * T * rows.z >= 512;  // two blocks a CU
    if (bf && many) hipLaunchKernelGGL((verify_rows_kernel<uint16_t, 256>), rows, dim3(256), 0, s, a);
    else if (bf) hipLaunchKernelGGL((verify_rows_kernel<uint16_t, 1024>), rows, dim3(1024), 0, s, a);
    else if (many) hipLaunchKernelGGL((verify_rows_kernel<float, 256>), rows, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((verify_rows_kernel<float, 1024>), rows, dim3(1024), 0, s, a);
    ABACUS_CHECK_LAUNCH("verify_drafts (rows)");
  }
  if (a.greedy) {
    hipLaunchKernelGGL(verify_greedy_kernel, dim3((unsigned)S), dim3(64), 0, s, a);
    ABACUS_CHECK_LAUNCH("verify_drafts (greedy)");
    return 0;
  }
  if (bf) hipLaunchKernelGGL(verify_decide_kernel<uint16_t>, decide, dim3(kThreads), 0, s, a);
  else hipLaunchKernelGGL(verify_decide_kernel<float>, decide, dim3(kThreads), 0, s, a);
  ABACUS_CHECK_LAUNCH("verify_drafts (decide)");
  return 0;
}
