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
// Three launches over slices of kSlice logits: every row's slice maxima and sums; each
// sequence's decision and the slice sums of the mass that its next token is drawn from;
// the draw in the slice that the random number falls into.  Probabilities are never
// written out: logits are read once, and once more for the one row that a token is
// drawn from.  Temperature 0 takes maxima alone, and two launches.
#include <algorithm>

#include "paged_rows.h"

namespace abacus {
namespace {

constexpr int kThreads = 256;
constexpr int kEach = 16;                   // logits of a thread
constexpr int kSlice = kThreads * kEach;    // of a block

struct VerifyArgs {
  const void *target, *draft;
  const int64_t* tokens;
  const int* query_start;
  const float* uniforms;
  int T, S, slices;
  int64_t V;
  double inv_t;
  bool greedy;
  int32_t* accepted;
  int64_t* next;
  double* sums;   // [2][T][slices]: of exp((x - slice max) / temperature)
  double* mass;   // [S][slices]
  int2* found;    // [S]: the row drawn from, and whether from p - q (1), from p (0), or nothing (-1)
  float* tops;    // [2][T][slices]: slice maxima, NaN where there is one
  int* at;        // [T][slices]: where (greedy)
};

template <typename T> struct alignas(sizeof(T)) Loose { T v[16 / sizeof(T)]; };  // 16 bytes at any element

// Logits slice * kSlice + tid * kEach ..+15 of a row; -inf past its end.
template <typename T>
__device__ inline void load_logits(const T* row, int64_t i0, int64_t V, float (&x)[kEach]) {
  constexpr int N = 16 / sizeof(T);
#pragma unroll
  for (int c = 0; c < kEach / N; ++c) {
    const int64_t i = i0 + c * N;
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

__device__ inline double wave_sum64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
// maximum that keeps a NaN
__device__ inline float max_nan(float a, float b) { return a != a || b != b ? __builtin_nanf("") : fmaxf(a, b); }

// e^x for x <= 0
__device__ inline double exp64(double x) { return exp(x); }

// The rows of sequence s, clipped to what there is.
__device__ inline void rows_of(const VerifyArgs& a, int s, int& first, int& n) {
  const int b = a.query_start[s], e = a.query_start[s + 1];
  const bool in = b >= 0 && e >= b && e <= a.T;
  first = in ? b : 0;
  n = in ? e - b : 0;
}

// One row's slice: its maximum (and, greedy, its place) and sum.  blockIdx: slice, row, target or draft.
template <typename T>
__global__ __launch_bounds__(kThreads) void verify_rows_kernel(VerifyArgs a) {
  __shared__ float top_w[4];
  __shared__ int at_w[4];
  __shared__ double sum_w[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int slice = blockIdx.x, row = blockIdx.y, which = blockIdx.z;
  const int64_t i0 = (int64_t)slice * kSlice + tid * kEach;
  float x[kEach];
  load_logits((const T*)(which ? a.draft : a.target) + row * a.V, i0, a.V, x);
  float top = -__builtin_inff();
  int at = 0x7fffffff;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    if (x[e] > top) at = (int)i0 + e;
    top = max_nan(top, x[e]);
  }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const float other = __shfl_xor(top, off, 64);
    const int there = __shfl_xor(at, off, 64);
    at = other > top ? there : other == top ? min(at, there) : at;
    top = max_nan(top, other);
  }
  if (lane == 0) top_w[wave] = top, at_w[wave] = at;
  __syncthreads();
  top = top_w[0], at = at_w[0];
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    if (top_w[w] > top) at = at_w[w];
    top = max_nan(top, top_w[w]);
  }
  const int64_t out = ((int64_t)which * a.T + row) * a.slices + slice;
  if (a.greedy) {
    if (tid == 0) a.tops[out] = top, a.at[out] = at;
    return;
  }
  double sum = 0.0;
  if (top > -__builtin_inff() && top < __builtin_inff()) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) sum += exp64(((double)x[e] - (double)top) * a.inv_t);
  }
  sum = wave_sum64(sum);
  if (lane == 0) sum_w[wave] = sum;
  __syncthreads();
  if (tid == 0) {
    a.tops[out] = top;
    a.sums[out] = (sum_w[0] + sum_w[1]) + (sum_w[2] + sum_w[3]);
  }
}

struct RowStat {
  float top;   // NaN, +inf or -inf: no distribution
  double inv;  // 1 / sum of exp((x - top) / temperature)
  __device__ bool fine() const { return top > -__builtin_inff() && top < __builtin_inff(); }
};

// A row's maximum and sum from its slices', by one wave.
__device__ inline RowStat row_stat(const VerifyArgs& a, int which, int row) {
  const int lane = threadIdx.x & 63;
  const int64_t base = ((int64_t)which * a.T + row) * a.slices;
  RowStat r;
  r.top = -__builtin_inff();
  for (int i = lane; i < a.slices; i += 64) r.top = max_nan(r.top, a.tops[base + i]);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) r.top = max_nan(r.top, __shfl_xor(r.top, off, 64));
  double sum = 0.0;
  if (r.fine())
    for (int i = lane; i < a.slices; i += 64)
      sum += a.sums[base + i] * exp64(((double)a.tops[base + i] - (double)r.top) * a.inv_t);
  r.inv = 1.0 / wave_sum64(sum);
  return r;
}

template <typename T>
__device__ inline double prob(const VerifyArgs& a, const T* logits, const RowStat& r, int64_t x) {
  return exp64(((double)to_f32(logits[x]) - (double)r.top) * a.inv_t) * r.inv;
}

// Of a row's 16 logits at i0: the mass that the next token is drawn from.
template <typename T>
__device__ inline void masses(const VerifyArgs& a, int row, bool residual, int64_t drafted, const RowStat& p,
                              const RowStat& q, int64_t i0, double (&m)[kEach]) {
  float x[kEach], y[kEach];
  load_logits((const T*)a.target + row * a.V, i0, a.V, x);
  if (residual && a.draft) load_logits((const T*)a.draft + row * a.V, i0, a.V, y);
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    m[e] = exp64(((double)x[e] - (double)p.top) * a.inv_t) * p.inv;
    if (residual) {
      const double d = a.draft ? exp64(((double)y[e] - (double)q.top) * a.inv_t) * q.inv : (i0 + e == drafted ? 1.0 : 0.0);
      m[e] = fmax(m[e] - d, 0.0);
    }
  }
}

// blockIdx: slice, sequence.  Every block of a sequence decides alike; slice 0's writes it down.
template <typename T>
__global__ __launch_bounds__(kThreads) void verify_decide_kernel(VerifyArgs a) {
  __shared__ int stop;
  __shared__ double sum_w[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int slice = blockIdx.x, seq = blockIdx.y;
  int first, n;
  rows_of(a, seq, first, n);
  if (n == 0) {
    if (slice == 0 && tid == 0) {
      a.accepted[seq] = 0;
      a.next[seq] = -1;
      a.found[seq] = make_int2(0, -1);
    }
    return;
  }
  if (tid == 0) stop = n - 1;
  __syncthreads();
  for (int j = wave; j < n - 1; j += 4) {
    const int row = first + j;
    const int64_t x = a.tokens[row + 1];
    const RowStat p = row_stat(a, 0, row);
    bool take = p.fine() && x >= 0 && x < a.V;
    if (take) {
      double qx = 1.0;
      if (a.draft) {
        const RowStat q = row_stat(a, 1, row);
        take = q.fine();
        if (take) qx = prob(a, (const T*)a.draft + row * a.V, q, x);
      }
      take = take && (double)a.uniforms[2 * row] * qx < prob(a, (const T*)a.target + row * a.V, p, x);
    }
    if (!take && lane == 0) atomicMin(&stop, j);
  }
  __syncthreads();
  const int j = stop, row = first + j;
  const bool residual = j < n - 1;
  const RowStat p = row_stat(a, 0, row);
  RowStat q = p;
  if (residual && a.draft) q = row_stat(a, 1, row);
  const int64_t drafted = residual ? a.tokens[row + 1] : -1;
  const bool fine = p.fine() && q.fine();
  if (slice == 0 && tid == 0) {
    a.accepted[seq] = j;
    a.found[seq] = make_int2(row, fine ? (int)residual : -1);
  }
  if (!fine) return;
  double m[kEach], sum = 0.0;
  masses<T>(a, row, residual, drafted, p, q, (int64_t)slice * kSlice + tid * kEach, m);
#pragma unroll
  for (int e = 0; e < kEach; ++e) sum += m[e];
  sum = wave_sum64(sum);
  if (lane == 0) sum_w[wave] = sum;
  __syncthreads();
  if (tid == 0) a.mass[(int64_t)seq * a.slices + slice] = (sum_w[0] + sum_w[1]) + (sum_w[2] + sum_w[3]);
}

// The draw, one block per sequence.
template <typename T>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(VerifyArgs a) {
  __shared__ double upto_w[4];
  __shared__ int64_t token;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int seq = blockIdx.x;
  const int2 f = a.found[seq];
  if (f.y < 0) {
    if (tid == 0) a.next[seq] = -1;
    return;
  }
  const int row = f.x;
  bool residual = f.y == 1;
  const double* mass = a.mass + (int64_t)seq * a.slices;
  const RowStat p = row_stat(a, 0, row);
  RowStat q = p;
  if (residual && a.draft) q = row_stat(a, 1, row);
  const int64_t drafted = residual ? a.tokens[row + 1] : -1;
  double total = 0.0;
  for (int i = 0; i < a.slices; ++i) total += mass[i];
  bool plain = false;  // no mass is left of p - q: p itself
  if (!(total > 0.0)) {
    plain = true;
    residual = false;
    total = 1.0;
  }
  const double border = fmin((double)a.uniforms[2 * row + 1], 1.0 - 0x1p-53) * total;
  if (tid == 0) token = -1;
  double before = 0.0;
  int slice = 0;
  if (!plain)  // the first slice whose end passes the border
    while (slice < a.slices - 1 && !(before + mass[slice] > border)) before += mass[slice++];
  __syncthreads();
  int64_t last = -1;  // the last token with any mass, should rounding leave none past the border
  for (; slice < a.slices; ++slice) {
    double m[kEach], own = 0.0;
    const int64_t i0 = (int64_t)slice * kSlice + tid * kEach;
    masses<T>(a, row, residual, drafted, p, q, i0, m);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      own += m[e];
      if (m[e] > 0.0) last = i0 + e;
    }
    double upto = own;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const double v = __shfl_up(upto, off, 64);
      if (lane >= off) upto += v;
    }
    if (lane == 63) upto_w[wave] = upto;
    __syncthreads();
    double start = before;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) start += upto_w[w];
      before += upto_w[w];
    }
    double run = start + (upto - own);
    int64_t mine = -1;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      run += m[e];
      if (mine < 0 && m[e] > 0.0 && run > border) mine = i0 + e;
    }
    // the lowest thread that has one
    const unsigned long long has = __ballot(mine >= 0);
    __shared__ int64_t best[4];
    if (lane == 0) best[wave] = -1;
    if (has && lane == __ffsll(has) - 1) best[wave] = mine;
    __syncthreads();
    if (tid == 0)
      for (int w = 0; w < 4 && token < 0; ++w) token = best[w];
    __syncthreads();
    if (token >= 0) break;
  }
  if (token < 0) {
    __shared__ long long ends[kThreads];
    ends[tid] = last;
    __syncthreads();
    if (tid == 0) {
      long long t = -1;
      for (int i = 0; i < kThreads; ++i) t = max(t, ends[i]);
      token = t;
    }
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

}  // namespace
}  // namespace abacus

using namespace abacus;

extern "C" int64_t abacus_verify_drafts_ws_bytes(int64_t T, int64_t V, int64_t S) {
  const int64_t n = slices_of(V);
  return (2 * T * n + S * n) * 8 + S * 8 + 2 * T * n * 4 + T * n * 4;
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
  a.T = (int)T, a.S = (int)S, a.slices = (int)n, a.V = V;
  a.greedy = temperature == 0.0;
  a.inv_t = a.greedy ? 1.0 : 1.0 / temperature;
  a.accepted = accepted_S, a.next = next_S;
  a.sums = (double*)ws;
  a.mass = a.sums + 2 * T * n;
  a.found = (int2*)(a.mass + S * n);
  a.tops = (float*)(a.found + S);
  a.at = (int*)(a.tops + 2 * T * n);
  hipStream_t s = (hipStream_t)stream;
  const dim3 rows((unsigned)n, (unsigned)T, a.draft ? 2 : 1), decide((unsigned)n, (unsigned)S);
  const bool bf = dtype == kBF16;
  if (T > 0) {
    if (bf) hipLaunchKernelGGL(verify_rows_kernel<uint16_t>, rows, dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL(verify_rows_kernel<float>, rows, dim3(kThreads), 0, s, a);
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
  if (bf) hipLaunchKernelGGL(verify_draw_kernel<uint16_t>, dim3((unsigned)S), dim3(kThreads), 0, s, a);
  else hipLaunchKernelGGL(verify_draw_kernel<float>, dim3((unsigned)S), dim3(kThreads), 0, s, a);
  ABACUS_CHECK_LAUNCH("verify_drafts (draw)");
  return 0;
}
