// The paged key/value cache: written (as it is, or quantised to e4m3) and read back.
//
// Key pages are (page, head, slot, dim), value pages (page, head, dim, slot):
// the attention multiplies V^T by P^T, whose operand is 8 consecutive keys of one
// dim, so with the values turned once here, where each is touched once, the
// attention reads them as they lie on every later token.
//
// e4m3: one exponent byte per token and head.  With amax the largest magnitude,
// e = the smallest integer with amax <= 448 * 2^e and byte = e + 127 (e = 0 for
// amax = 0, and never below -110, so that every value a code stands for is a
// normal bf16 number); codes are x * 2^-e rounded to nearest even.  The scale is a
// power of two because it costs a floating-point code no precision, makes what a
// code stands for exact in bf16, and is applied by the conversion instruction.  A
// token's head with an infinity or NaN in its key or its value gets key codes NaN
// and value codes 0: whoever sees the key gets NaN from its score, and nobody else
// anything from 0 * V.
//
// Both kernels are bound by their bytes.  A work-group takes 16 (row, head) pairs
// of one 16-slot group of one sequence, 16 lanes with 8 dims each per pair, so
// that a full group is turned through LDS into whole 16-slot runs; a step's single
// row (one group each) takes its 16 heads at once instead.  8190 bf16 rows of 8 x 128
// are written in 13.7 us (4.9 TB/s in and out, a large copy's rate), a step's 64 rows in
// 4.5 us, which is a launch.
#include <algorithm>

#include "paged_rows.h"

namespace abacus {
namespace {

constexpr int kGroup = 16;   // slots of a group: a divisor of every page size
constexpr int kMaxK = 128;
constexpr uint8_t kNaNCode = 0x7f;

struct Pages {
  void *k, *v;
  uint8_t *k_scale, *v_scale;  // null unless e4m3
  int H, K;
};

// 8 values at p as fp32
template <typename T>
__device__ inline void load8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 2) {
    const Vec16 v = ld16(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = lo_bf16(v.w[i]);
      x[2 * i + 1] = hi_bf16(v.w[i]);
    }
  } else {
    const Vec16 a = ld16(p), b = ld16(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = bits_f32(a.w[i]);
      x[4 + i] = bits_f32(b.w[i]);
    }
  }
}

// 8 values to 8 of T; Stream: past the caches, for what is written once and not read here
template <bool Stream, typename T>
__device__ inline void store8(T* to, const float (&x)[8]) {
  constexpr int N = 8 * sizeof(T) / 16;
  Vec16 w[N];
#pragma unroll
  for (int i = 0; i < 8 * (int)sizeof(T) / 4; ++i) {
    if constexpr (sizeof(T) == 2) w[i / 4].w[i % 4] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
    else w[i / 4].w[i % 4] = f32_bits(x[i]);
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if constexpr (Stream) st16_stream((char*)to + 16 * n, w[n]);
    else st16((char*)to + 16 * n, w[n]);
  }
}

// The exponent byte of a row whose largest magnitude is amax (finite): 448 = 1.75 * 2^8.
__device__ inline int scale_byte(float amax) {
  const uint32_t u = f32_bits(amax);
  const int e = (int)(u >> 23) - 127 - ((u & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return amax == 0.f ? 127 : max(e, -110) + 127;
}

// 8 values to 8 e4m3 codes of 2^(byte - 127) each
__device__ inline uint2 codes8(const float (&x)[8], int byte) {
  const float f = bits_f32((uint32_t)(254 - byte) << 23);  // (byte is 17 to 247)
  uint2 c;
  int w = 0;
  w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * f, x[1] * f, w, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * f, x[3] * f, w, true);
  c.x = (uint32_t)w;
  w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4] * f, x[5] * f, w, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(x[6] * f, x[7] * f, w, true);
  c.y = (uint32_t)w;
  return c;
}

// C: what a slot holds (uint16_t bf16, float, uint8_t e4m3 code); T: what the rows are.
template <typename T, typename C>
__global__ __launch_bounds__(256) void kv_write_kernel(const T* __restrict__ k, const T* __restrict__ v, PagedRows a,
                                                       Pages p) {
  constexpr bool kCodes = sizeof(C) == 1;
  __shared__ __attribute__((aligned(16))) C turned[kGroup][kMaxK + 16 / sizeof(C)];
  const int tid = threadIdx.x, H = p.H, K = p.K;
  int seq, local;
  SeqRows r;
  if (!SeqScan(a).find(blockIdx.x, [](const SeqRows& r) {
        return r.n > 0 && r.len > 0 ? (r.len - 1) / kGroup - max(r.len - r.n, 0) / kGroup + 1 : 0;
      }, seq, local, r))
    return;
  const int g0 = (max(r.len - r.n, 0) / kGroup + local) * kGroup;  // the group's first position
  const int p0 = max(g0, r.len - r.n), p1 = min(g0 + kGroup, r.len), rows = p1 - p0;
  const int pair0 = blockIdx.y * 16;
  if (pair0 >= rows * H) return;
  bool bad;
  const int page = page_of(a, seq, g0, bad);
  if (bad || r.bad) return;
  const int in_page = g0 & ((1 << a.shift) - 1);

  // this thread's pair and 8 dims
  const int pair = pair0 + tid / 16, d0 = (tid % 16) * 8;
  const int head = pair / rows, pos = p0 + pair % rows;
  const bool mine = pair < rows * H && d0 < K;
  const int64_t row = r.first + pos - (r.len - r.n);
  float x[8] = {}, y[8] = {};
  if (mine) {
    load8(k + (row * H + head) * K + d0, x);
    load8(v + (row * H + head) * K + d0, y);
  }
  const int64_t tile = (int64_t)page * H + head;  // (page, head)
  if constexpr (kCodes) {
    float mk = 0.f, mv = 0.f, bad_sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      mk = fmaxf(mk, fabsf(x[i]));
      mv = fmaxf(mv, fabsf(y[i]));
      bad_sum += x[i] * 0.f + y[i] * 0.f;  // 0, or NaN where an infinity or NaN is among them
    }
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) {
      mk = fmaxf(mk, __shfl_xor(mk, off, 64));
      mv = fmaxf(mv, __shfl_xor(mv, off, 64));
      bad_sum += __shfl_xor(bad_sum, off, 64);
    }
    const bool poison = !(bad_sum == 0.f);
    const int bk = poison ? 127 : scale_byte(mk), bv = poison ? 127 : scale_byte(mv);
    uint2 ck = codes8(x, bk), cv = codes8(y, bv);
    if (poison) {
      ck.x = ck.y = kNaNCode * 0x01010101u;
      cv.x = cv.y = 0;
    }
    if (mine) {
      const int64_t slot = (tile << a.shift) + in_page + (pos - g0);
      *reinterpret_cast<uint2*>((uint8_t*)p.k + slot * K + d0) = ck;
      if (d0 == 0) {
        p.k_scale[slot] = (uint8_t)bk;
        p.v_scale[slot] = (uint8_t)bv;
      }
    }
    *reinterpret_cast<uint2*>(&turned[tid / 16][d0]) = cv;
  } else {
    if (mine) store8<false>((C*)p.k + ((tile << a.shift) + in_page + (pos - g0)) * K + d0, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) turned[tid / 16][d0 + i] = from_f32<C>(y[i]);
  }
  __syncthreads();
  // the values, slot by slot of one dim
  if (rows == kGroup) {  // 16 pairs are one head's 16 slots
    for (int i = tid; i < K * 2; i += 256) {
      const int d = i / 2, s0 = (i % 2) * 8;
      C* to = (C*)p.v + ((((int64_t)page * H + pair0 / kGroup) * K + d) << a.shift) + in_page + s0;
      union { C c[8]; uint32_t w[2 * sizeof(C)]; } run;
#pragma unroll
      for (int j = 0; j < 8; ++j) run.c[j] = turned[s0 + j][d];
#pragma unroll
      for (int j = 0; j < (int)(2 * sizeof(C)); j += 2) {
        uint2 w;
        w.x = run.w[j];
        w.y = run.w[j + 1];
        *reinterpret_cast<uint2*>((uint32_t*)to + j) = w;
      }
    }
  } else {
    for (int i = tid; i < 16 * K; i += 256) {
      const int q = i / K, d = i % K, pr = pair0 + q;
      if (pr >= rows * H) break;
      const int off = in_page + p0 - g0 + pr % rows;
      ((C*)p.v)[((((int64_t)page * H + pr / rows) * K + d) << a.shift) + off] = turned[q][d];
    }
  }
}

// 8 held values (codes: times 2^(byte - 127)) as fp32
template <typename C>
__device__ inline void widen8(const C* p, int byte, float (&x)[8]) {
  if constexpr (sizeof(C) == 1) {
    const uint2 c = *reinterpret_cast<const uint2*>(p);
    const float s = bits_f32((uint32_t)byte << 23);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int w = (int)(h ? c.y : c.x);
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
      x[4 * h] = lo[0] * s;
      x[4 * h + 1] = lo[1] * s;
      x[4 * h + 2] = hi[0] * s;
      x[4 * h + 3] = hi[1] * s;
    }
  } else {
    load8(p, x);
  }
}

// 8 values of one position out of 8 rows of V^T, four positions of each at hand (C's of a row in
// n dwords), as fp32.
template <typename C, int N>
__device__ inline void position_of(const uint32_t (&w)[8][N], int pos, int byte, float (&y)[8]) {
  if constexpr (sizeof(C) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = bits_f32(w[i][pos]);
  } else if constexpr (sizeof(C) == 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = pos & 1 ? hi_bf16(w[i][pos / 2]) : lo_bf16(w[i][pos / 2]);
  } else {
    const int sel = 0x0c0c0400 + pos * 0x0101;  // byte pos of two words, side by side
    uint2 c;
    c.x = __builtin_amdgcn_perm(w[1][0], w[0][0], sel) | __builtin_amdgcn_perm(w[3][0], w[2][0], sel) << 16;
    c.y = __builtin_amdgcn_perm(w[5][0], w[4][0], sel) | __builtin_amdgcn_perm(w[7][0], w[6][0], sel) << 16;
    widen8((const C*)&c, byte, y);
  }
}

// Rows (s, l) of out, l < L: position l of sequence s, 0 past its length.  A block takes
// Span groups of one head, all their loads under way at once: 4 where there are blocks enough
// all the same (16 x 4096 e4m3 tokens of 16 x 64: 95 us with 1, 78 us with 4, 4.6 TB/s),
// else 1 (1000 bf16 tokens of 8 x 128: 3.5 us, 6.4 us with 4).
template <class T, int N> __device__ inline T pick_of(const T (&x)[N], int j) {
  if constexpr (N == 1) return x[0];
  const T a = j & 1 ? x[1] : x[0], b = j & 1 ? x[N - 1] : x[N / 2];
  return j & 2 ? b : a;
}
template <typename C, typename T, int Span>
__global__ __launch_bounds__(256) void kv_read_kernel(PagedRows a, Pages p, int64_t L, T* __restrict__ k,
                                                      T* __restrict__ v) {
  static_assert(Span == 1 || Span == 4, "pick_of");
  constexpr int N = (int)sizeof(C);  // dwords of four values
  constexpr int kPitch = 4 * N + 1;  // dwords of a V^T row in LDS: 8 rows apart is 8 or 40 banks
  __shared__ uint32_t turned[Span][kMaxK * kPitch];
  __shared__ uint8_t exponents[Span * kGroup], nan[Span * kGroup];
  const int tid = threadIdx.x, H = p.H, K = p.K, octets = K / 8;
  const int seq = blockIdx.z, head = blockIdx.x, l0 = blockIdx.y * kGroup * Span;
  const int given = a.lengths[seq], most = a.P << a.shift, len = min(max(given, 0), most);
  const int in_page = (1 << a.shift) - 1;
  int64_t tile[Span];  // (page, head) of each group; groups past the length take the first page
  bool bad[Span];
#pragma unroll
  for (int j = 0; j < Span; ++j) {
    const int pos = l0 + j * kGroup;
    tile[j] = (int64_t)page_of(a, seq, pos < len ? pos : 0, bad[j]) * H + head;
    bad[j] |= given > most;
  }
  // V^T into LDS, 16 bytes at a time; of codes the values' exponents and which positions are NaN
  for (int i = tid; i < Span * K * N; i += 256) {
    const int j = i / (K * N), d = i / N % K, c = i % N;
    const Vec16 w = ld16((const C*)p.v + ((pick_of(tile, j) * K + d) << a.shift) + ((l0 + j * kGroup) & in_page) + c * (16 / N));
#pragma unroll
    for (int e = 0; e < 4; ++e) turned[j][d * kPitch + 4 * c + e] = w.w[e];
  }
  if (tid < Span * kGroup) {
    const int j = tid / kGroup, l = l0 + tid;
    const int64_t slot = (pick_of(tile, j) << a.shift) + (l & in_page);
    bool none = pick_of(bad, j);
    if constexpr (N == 1) {
      exponents[tid] = p.v_scale[slot];
      none |= (((const uint8_t*)p.k)[slot * K] & 0x7f) == kNaNCode;
    }
    nan[tid] = none;
  }
  // keys: 8 dims of one position a thread
  for (int i = tid; i < Span * kGroup * octets; i += 256) {
    const int r = i / octets, d0 = i % octets * 8, j = r / kGroup, l = l0 + r;
    if (l >= L) break;
    float x[8] = {};
    if (l < len) {
      const int64_t slot = (pick_of(tile, j) << a.shift) + (l & in_page);
      int byte = 127;
      if constexpr (N == 1) byte = p.k_scale[slot];
      widen8((const C*)p.k + slot * K + d0, byte, x);
      if (pick_of(bad, j))
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __builtin_nanf("");
    }
    store8<true>(k + ((seq * L + l) * H + head) * K + d0, x);
  }
  __syncthreads();
  // values: 8 dims of four positions
  for (int i = tid; i < Span * 4 * octets; i += 256) {
    const int d0 = i % octets * 8, quad = i / octets, j = quad / 4;
    uint32_t w[8][N];
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int n = 0; n < N; ++n) w[e][n] = turned[j][(d0 + e) * kPitch + quad % 4 * N + n];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int at = quad * 4 + r, l = l0 + at;
      if (l >= L) break;
      float y[8] = {};
      if (l < len) {
        position_of<C>(w, r, N == 1 ? exponents[at] : 127, y);
        if (nan[at])
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = __builtin_nanf("");
      }
      store8<true>(v + ((seq * L + l) * H + head) * K + d0, y);
    }
  }
}

template <typename C, typename T>
void launch_read(const PagedRows& a, const Pages& p, int64_t L, void* k, void* v, hipStream_t s) {
  const int64_t groups = (L + kGroup - 1) / kGroup, spans = (groups + 3) / 4;
  if (spans * p.H * a.S >= 2048)
    hipLaunchKernelGGL((kv_read_kernel<C, T, 4>), dim3((unsigned)p.H, (unsigned)spans, (unsigned)a.S), dim3(256), 0, s, a, p,
                       L, (T*)k, (T*)v);
  else
    hipLaunchKernelGGL((kv_read_kernel<C, T, 1>), dim3((unsigned)p.H, (unsigned)groups, (unsigned)a.S), dim3(256), 0, s, a, p,
                       L, (T*)k, (T*)v);
}

// Each row's position in its sequence, 0 for rows of none: a thread a row, by bisection of the
// ranges that count.
__global__ __launch_bounds__(256) void batch_positions_kernel(PagedRows a, int64_t* __restrict__ positions) {
  const int good = good_sequences(a.query_start, a.S, a.T), row = blockIdx.x * 256 + threadIdx.x;
  if (row >= a.T) return;
  int lo = 0, hi = good;  // the first sequence whose range ends behind the row
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.query_start[mid + 1] > row) hi = mid;
    else lo = mid + 1;
  }
  int64_t pos = 0;
  if (lo < good && row >= a.query_start[0]) pos = (int64_t)a.lengths[lo] - a.query_start[lo + 1] + row;
  positions[row] = pos > 0 ? pos : 0;
}

int check_pages(const char* what, const void* k, const void* v, const void* k_scale, const void* v_scale, int dtype,
                int held) {
  ABACUS_CHECK_ARG(dtype == kF32 || dtype == kBF16, "%s: dtype code %d", what, dtype);
  ABACUS_CHECK_ARG(held == dtype || held == ABACUS_E4M3, "%s: a cache of dtype code %d with rows of %d", what, held, dtype);
  ABACUS_CHECK_ARG(k && v && (held != ABACUS_E4M3 || (k_scale && v_scale)), "%s: null pointer", what);
  ABACUS_CHECK_ARG(((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_scale | (uintptr_t)v_scale) % 16 == 0,
                   "%s: pages must be 16-byte aligned", what);
  return 0;
}

}  // namespace
}  // namespace abacus

using namespace abacus;

extern "C" int abacus_batch_positions(const int32_t* query_start, const int32_t* lengths, int64_t S, int64_t T,
                                      int64_t* positions_T, void* stream) {
  ABACUS_CHECK_ARG(S >= 1 && S <= (1 << 20) && T >= 0 && T < (1ll << 24), "batch_positions: %lld rows of %lld sequences",
                   (long long)T, (long long)S);
  ABACUS_CHECK_ARG(query_start && lengths && (T == 0 || positions_T), "batch_positions: null pointer");
  if (T == 0) return 0;
  PagedRows a{nullptr, query_start, lengths, (int)S, 0, (int)T, 0, 0};
  hipLaunchKernelGGL(batch_positions_kernel, dim3((unsigned)((T + 255) / 256)), dim3(256), 0, (hipStream_t)stream, a,
                     positions_T);
  ABACUS_CHECK_LAUNCH("batch_positions");
  return 0;
}

extern "C" int abacus_kv_write(const void* k_THK, const void* v_THK, int64_t T, int64_t H, int64_t K, int dtype,
                               const int32_t* page_table_SP, const int32_t* query_start, const int32_t* lengths,
                               int64_t S, int64_t P, int64_t page_size, int64_t n_pages, int held, void* k_pages,
                               void* v_pages, void* k_scale, void* v_scale, void* stream) {
  if (check_paged_rows("kv_write", page_table_SP, query_start, lengths, S, P, T, page_size, n_pages, H, K)) return 1;
  if (check_pages("kv_write", k_pages, v_pages, k_scale, v_scale, dtype, held)) return 1;
  if (T == 0) return 0;
  ABACUS_CHECK_ARG(k_THK && v_THK && ((uintptr_t)k_THK | (uintptr_t)v_THK) % 16 == 0,
                   "kv_write: k and v must be there, and 16-byte aligned");
  PagedRows a{page_table_SP, query_start, lengths, (int)S, (int)P, (int)T, __builtin_ctzll(page_size), (int)n_pages};
  Pages p{k_pages, v_pages, (uint8_t*)k_scale, (uint8_t*)v_scale, (int)H, (int)K};
  // a sequence's rows touch at most n / 16 groups and the two at their ends
  const int64_t groups = std::min<int64_t>(T, T / kGroup + 2 * S);
  const dim3 grid((unsigned)groups, (unsigned)H);  // 16 pairs a block, at most 16 H in a group
  hipStream_t s = (hipStream_t)stream;
  if (held == ABACUS_E4M3 && dtype == kBF16)
    hipLaunchKernelGGL((kv_write_kernel<uint16_t, uint8_t>), grid, dim3(256), 0, s, (const uint16_t*)k_THK,
                       (const uint16_t*)v_THK, a, p);
  else if (held == ABACUS_E4M3)
    hipLaunchKernelGGL((kv_write_kernel<float, uint8_t>), grid, dim3(256), 0, s, (const float*)k_THK,
                       (const float*)v_THK, a, p);
  else if (dtype == kBF16)
    hipLaunchKernelGGL((kv_write_kernel<uint16_t, uint16_t>), grid, dim3(256), 0, s, (const uint16_t*)k_THK,
                       (const uint16_t*)v_THK, a, p);
  else
    hipLaunchKernelGGL((kv_write_kernel<float, float>), grid, dim3(256), 0, s, (const float*)k_THK,
                       (const float*)v_THK, a, p);
  ABACUS_CHECK_LAUNCH("kv_write");
  return 0;
}

extern "C" int abacus_kv_read(const int32_t* page_table_SP, const int32_t* lengths, int64_t S, int64_t P,
                              int64_t page_size, int64_t n_pages, int64_t H, int64_t K, int held, const void* k_pages,
                              const void* v_pages, const void* k_scale, const void* v_scale, int64_t L, int dtype,
                              void* k_SLHK, void* v_SLHK, void* stream) {
  if (check_paged_rows("kv_read", page_table_SP, lengths, lengths, S, P, 0, page_size, n_pages, H, K)) return 1;
  if (check_pages("kv_read", k_pages, v_pages, k_scale, v_scale, dtype, held)) return 1;
  ABACUS_CHECK_ARG(S <= 65535 && L >= 0 && L <= 65535 * kGroup, "kv_read: %lld sequences of %lld tokens", (long long)S,
                   (long long)L);
  if (L == 0) return 0;
  ABACUS_CHECK_ARG(k_SLHK && v_SLHK && ((uintptr_t)k_SLHK | (uintptr_t)v_SLHK) % 16 == 0,
                   "kv_read: k and v must be there, and 16-byte aligned");
  PagedRows a{page_table_SP, nullptr, lengths, (int)S, (int)P, 0, __builtin_ctzll(page_size), (int)n_pages};
  Pages p{(void*)k_pages, (void*)v_pages, (uint8_t*)k_scale, (uint8_t*)v_scale, (int)H, (int)K};
  hipStream_t s = (hipStream_t)stream;
  if (held == ABACUS_E4M3 && dtype == kBF16) launch_read<uint8_t, uint16_t>(a, p, L, k_SLHK, v_SLHK, s);
  else if (held == ABACUS_E4M3) launch_read<uint8_t, float>(a, p, L, k_SLHK, v_SLHK, s);
  else if (dtype == kBF16) launch_read<uint16_t, uint16_t>(a, p, L, k_SLHK, v_SLHK, s);
  else launch_read<float, float>(a, p, L, k_SLHK, v_SLHK, s);
  ABACUS_CHECK_LAUNCH("kv_read");
  return 0;
}
