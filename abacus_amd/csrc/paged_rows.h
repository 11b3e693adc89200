// The rows of a call over a paged cache: which sequence a row belongs to, and
// where a position of a sequence lies in the pool.
//
// T rows of S sequences lie one after the other: rows query_start[s] ..
// query_start[s + 1] - 1 are the last n_s positions of sequence s, which has
// lengths[s] tokens in all.  Position p lies in slot p % page_size of page
// table[s][p / page_size].  All of this is device memory that no host check
// has seen, so every value is bounded here: a range of rows outside [0, T] is
// empty, a length past the table marks its sequence, a page id outside the
// pool marks its positions.  Nothing is kept between calls: each wave finds its
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

__device__ inline SeqRows seq_rows(const PagedRows& a, int s) {
  SeqRows r;
  const int first = a.query_start[s], end = a.query_start[s + 1], len = a.lengths[s];
  const bool in = first >= 0 && end >= first && end <= a.T;
  const int most = a.P << a.shift;
  r.first = in ? first : 0;
  r.n = in ? end - first : 0;
  r.len = min(max(len, 0), most);
  r.bad = len > most;
  return r;
}

// Sequence and place of unit b where sequence s has count(s) units, for a whole
// wave; false past the last one.
template <class Count>
__device__ inline bool find_unit(int S, int b, Count count, int& seq, int& local) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int s0 = 0; s0 < S; s0 += 64) {
    const int c = s0 + lane < S ? count(s0 + lane) : 0;
    int upto = c;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int v = __shfl_up(upto, off, 64);
      if (lane >= off) upto += v;
    }
    const int total = __shfl(upto, 63, 64);
    if (b < base + total) {
      const int at = __ffsll((unsigned long long)__ballot(base + upto > b)) - 1;
      seq = __builtin_amdgcn_readfirstlane(s0 + at);
      local = __builtin_amdgcn_readfirstlane(b - base - __shfl(upto - c, at, 64));
      return true;
    }
    base += total;
  }
  return false;
}

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
