// The rows of a call over a paged cache: which sequence a row belongs to, and
// where a position of a sequence lies in the pool.
//
// T rows of S sequences lie one after the other: rows query_start[s] ..
// query_start[s + 1] - 1 are the last n_s positions of sequence s, which has
// lengths[s] tokens in all.  Position p lies in slot p % page_size of page
// table[s][p / page_size].  All of this is device memory that no host check
// has seen, so every value is bounded here: from the first range that runs backwards
// or out of [0, T] on every sequence is without rows (so no two share one, and there
// are at most T in all, which launches and workspaces are sized by), a length past the
// table marks its sequence, a page id outside the pool marks its positions.  Nothing is kept between calls: each wave finds its
// place by a scan over the sequences, one load per 64 of them.
#pragma once

#include "common.h"

namespace abacus {

struct PagedRows {
  const int* table;        // (S, P) page ids
  const int* query_start;  // (S + 1)
  const int* lengths;      // (S)
  int S, P, T;
  int shift;    // log2 of the page size
  int n_pages;  // pages in the pool
};

struct SeqRows {
  int first;  // its first row
  int n;      // rows
  int len;    // tokens, the rows' own included, at most what the table holds
  bool bad;   // the table has no place for that many
};

__device__ inline bool range_in(int first, int end, int T) { return first >= 0 && end >= first && end <= T; }

__device__ inline SeqRows seq_rows(const PagedRows& a, int s, bool& in) {
  SeqRows r;
  const int first = a.query_start[s], end = a.query_start[s + 1], len = a.lengths[s];
  in = range_in(first, end, a.T);
  const int most = a.P << a.shift;
  r.first = in ? first : 0;
  r.n = in ? end - first : 0;
  r.len = min(max(len, 0), most);
  r.bad = len > most;
  return r;
}

// The sequences before the first bad range, by a wave.
__device__ inline int good_sequences(const int* query_start, int S, int T) {
  for (int s0 = 0; s0 < S; s0 += 64) {
    const int s = s0 + (threadIdx.x & 63);
    const uint64_t out = __ballot(s < S && !range_in(query_start[s], query_start[s + 1], T));
    if (out) return s0 + __ffsll((unsigned long long)out) - 1;
  }
  return S;
}

// Sums over a wave without LDS: within rows of 16 lanes by DPP, then over the rows.
template <int kCtrl> __device__ inline int dpp_or_0(int x) {
  return __builtin_amdgcn_update_dpp(0, x, kCtrl, 0xf, 0xf, true);
}
__device__ inline int wave_scan(int x, int& total) {  // inclusive; total: the whole wave's
  x += dpp_or_0<0x111>(x);  // row_shr:1, 2, 4, 8
  x += dpp_or_0<0x112>(x);
  x += dpp_or_0<0x114>(x);
  x += dpp_or_0<0x118>(x);
  const int r0 = __builtin_amdgcn_readlane(x, 15), r1 = __builtin_amdgcn_readlane(x, 31),
            r2 = __builtin_amdgcn_readlane(x, 47), row = (threadIdx.x & 63) >> 4;
  x += (row > 0 ? r0 : 0) + (row > 1 ? r1 : 0) + (row > 2 ? r2 : 0);
  total = __builtin_amdgcn_readlane(x, 63);
  return x;
}
__device__ inline float wave_total(float x) {
  x += bits_f32((uint32_t)dpp_or_0<0x121>((int)f32_bits(x)));  // row_ror:1, 2, 4, 8
  x += bits_f32((uint32_t)dpp_or_0<0x122>((int)f32_bits(x)));
  x += bits_f32((uint32_t)dpp_or_0<0x124>((int)f32_bits(x)));
  x += bits_f32((uint32_t)dpp_or_0<0x128>((int)f32_bits(x)));
  float sum = 0.f;
#pragma unroll
  for (int r = 0; r < 4; ++r) sum += bits_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_bits(x), 16 * r));
  return sum;
}

// The sequences as a wave looks through them: lane l has sequence l, 64 + l, ... ; the
// first 64 are read once.
struct SeqScan {
  const PagedRows& a;
  bool first_ended = false;
  SeqRows first;
  __device__ inline explicit SeqScan(const PagedRows& rows) : a(rows) { first = next(0, first_ended); }
  // sequences s0 .. s0 + 63; `ended`: whether there was a bad range before them, among them
  __device__ inline SeqRows next(int s0, bool& ended) const {
    const int lane = threadIdx.x & 63, s = s0 + lane;
    SeqRows r{0, 0, 0, false};
    bool in = true;
    if (s < a.S) r = seq_rows(a, s, in);
    const uint64_t out = __ballot(!in);
    if (ended || (out & ((1ull << lane) - 1))) r.n = 0;
    ended |= out != 0;
    return r;
  }
  __device__ inline SeqRows at(int s0, bool& ended) const {
    if (s0 > 0) return next(s0, ended);
    ended = first_ended;
    return first;
  }
  // sum of value(sequence) over all
  template <class F>
  __device__ inline float sum(F value) const {
    bool ended;
    float x = value(at(0, ended));
    for (int s0 = 64; s0 < a.S; s0 += 64) x += value(at(s0, ended));
    return wave_total(x);
  }
  // sum of count(sequence) over the sequences before `seq`
  template <class F>
  __device__ inline int before(int seq, F count) const {
    int base = 0;
    bool ended;
    for (int s0 = 0; s0 < a.S; s0 += 64) {
      const int c = count(at(s0, ended));
      int total;
      const int upto = wave_scan(c, total);
      if (seq < s0 + 64) return base + __builtin_amdgcn_readlane(upto - c, seq - s0);
      base += total;
    }
    return base;
  }
  // Sequence and place of unit b where a sequence has count(sequence) units; false past the last.
  template <class F>
  __device__ inline bool find(int b, F count, int& seq, int& local, SeqRows& r) const {
    int base = 0;
    bool ended;
    for (int s0 = 0; s0 < a.S; s0 += 64) {
      const SeqRows mine = at(s0, ended);
      const int c = count(mine);
      int total;
      const int upto = wave_scan(c, total);
      if (b < base + total) {
        const int l = __ffsll((unsigned long long)__ballot(base + upto > b)) - 1;
        seq = s0 + l;
        local = b - base - __builtin_amdgcn_readlane(upto - c, l);
        r.first = __builtin_amdgcn_readlane(mine.first, l);
        r.n = __builtin_amdgcn_readlane(mine.n, l);
        r.len = __builtin_amdgcn_readlane(mine.len, l);
        r.bad = __builtin_amdgcn_readlane((int)mine.bad, l);
        return true;
      }
      base += total;
    }
    return false;
  }
};

// Page of a sequence's position; `bad` is set, and page 0 taken, where there is none.
__device__ inline int page_of(const PagedRows& a, int seq, int pos, bool& bad) {
  const int i = pos >> a.shift;
  const int id = a.table[(int64_t)seq * a.P + min(i, a.P - 1)];
  bad = i >= a.P || (unsigned)id >= (unsigned)a.n_pages;
  return bad ? 0 : id;
}

// Host side: the values that the launch itself is sized by.
inline int check_paged_rows(const char* what, const void* table, const void* query_start, const void* lengths,
                            int64_t S, int64_t P, int64_t T, int64_t page_size, int64_t n_pages, int64_t H,
                            int64_t K) {
  ABACUS_CHECK_ARG(table && query_start && lengths, "%s: null pointer", what);
  ABACUS_CHECK_ARG(S >= 1 && S <= (1 << 20), "%s: %lld sequences", what, (long long)S);
  ABACUS_CHECK_ARG(T >= 0 && T < (1ll << 24), "%s: %lld rows", what, (long long)T);
  ABACUS_CHECK_ARG(page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0,
                   "%s: page size %lld is not a power of two from 16 to 256", what, (long long)page_size);
  ABACUS_CHECK_ARG(P >= 1 && P * page_size < (1ll << 30), "%s: a table of %lld pages", what, (long long)P);
  ABACUS_CHECK_ARG(n_pages >= 1 && n_pages < (1ll << 31), "%s: a pool of %lld pages", what, (long long)n_pages);
  ABACUS_CHECK_ARG(K >= 16 && K <= 128 && K % 16 == 0, "%s: head_dim %lld is not a multiple of 16 up to 128", what,
                   (long long)K);
  ABACUS_CHECK_ARG(H >= 1 && H <= 1024, "%s: %lld heads", what, (long long)H);
  return 0;
}

}  // namespace abacus
