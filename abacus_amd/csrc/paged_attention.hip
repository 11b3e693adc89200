// Attention of new tokens over a paged key/value cache.
//
// Row j of a sequence's n new tokens has position len - n + j and sees the keys
// up to it: o = sum_j softmax(scale q . k_j) v_j, query head h with key head h / G.
// One pass over the keys with the running maximum and sum of the softmax in fp32.
//
// How the work is cut over units of rows and pieces of keys is paged_cut.h's.  Sequences with
// few rows, and all fp32 ones, are paged_few.h's; those with many bf16 rows paged_chunk.h's.
// Where a call may have both, one launch has the blocks of both (paged_chunk.hip): a chunk is
// bound by its products and a step by its bytes.  A second launch joins the pieces.
#include <algorithm>

#include "paged_few.h"

namespace abacus {
namespace {

constexpr int kFewPieces = 2048;   // pieces the work of a launch is cut into, about: eight a CU, as sequences differ
constexpr int kOnePieces = 448;    // where a CU holds one work-group: two turns, less the sequences' last pieces
constexpr int kLeast = 4;          // tiles of one at least
constexpr int kFewJoined = 16;     // pieces that a wave joins for several rows at once
// Of the chunk kernel's: two work-groups a CU, less the sequences' last pieces (259 tokens of 16 heads
// over 8, K = 80, over 48042 keys: 219 us with 512, 155).  768 gains 7% where K = 64 and no single
// tokens are there to fill the CUs, and loses 20% beside them.
// Where the units, if they are all alike, would be more pieces than run at once, the last few of
// those would run alone: a finer cut (576 tokens of 64 heads over 8, K = 128, over 7085 keys: 255 us, 215).
constexpr int kChunkPieces = 480, kChunkPlaces = 512, kChunkFiner = 960;

template <typename Q, bool Cd, int KD, bool Full, int QT>
__global__ __launch_bounds__(256, QT == 1 ? (KD <= 64 ? 3 : 2) : (KD <= 64 ? 2 : 1)) void paged_few_kernel(PagedArgs p) {
  __shared__ __attribute__((aligned(16))) FewLds<KD, QT> lds;
  few_block<Q, Cd, KD, Full, QT>(p, blockIdx.x, gridDim.x, lds);
}

// Joins the pieces of the units that were cut, K / 4 lanes to a row of a piece.  blockIdx: unit
// and key head, and the first of the block's rows.  (With one thread for all the pieces of its
// four dims a row of 128 pieces took 100 us, with one wave 19.)
struct JoinLds {
  float top[4], l[4];
  float o[4][128];
};
template <typename Q, int R>
__device__ inline void join_block(const PagedArgs& p, int block, JoinLds& lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, K = p.K, lanes = K / 4;
  const int b = block / p.Hk, kh = block % p.Hk;
  const SeqScan scan(p.a);
  int given;
  const int chunk = piece_tiles<R>(p, scan, given);
  int seq, local;
  SeqRows r;
  if (!scan.find(b, [&](const SeqRows& r) { return units_of<R>(p, r); }, seq, local, r)) return;
  const int split = pieces_of(r, chunk), units = units_of<R>(p, r);
  if (split == 1) return;
  const int before = scan.before(seq, [&](const SeqRows& r) { return units_of<R>(p, r) * pieces_of(r, chunk); });
  const int item = before + (units - 1 - local) * split;
  const int64_t pitch = (int64_t)p.Hk * R * (K + 2);  // between a unit's pieces
  const float* part = p.part + ((int64_t)item * p.Hk + kh) * R * (K + 2);
  const int rows = min(R, r.n * p.G - local * R);
  if (split <= kFewJoined) {  // as many rows at a time as the wave holds, piece by piece
    const int sub = lane / lanes, subs = 64 / lanes, d = lane % lanes * 4;
    for (int m0 = (blockIdx.y * 4 + wave) * subs; m0 < rows; m0 += gridDim.y * 4 * subs) {
      const int m = min(m0 + sub, rows - 1);
      float top = -__builtin_inff(), l = 0.f;
#pragma unroll 4
      for (int i = 0; i < split; ++i) top = fmaxf(top, part[i * pitch + R * K + m]);
      pa_f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int i = 0; i < split; ++i) {
        const float pm = part[i * pitch + R * K + m], pl = part[i * pitch + R * K + R + m];
        const pa_f32x4 x = *reinterpret_cast<const pa_f32x4*>(part + i * pitch + (int64_t)m * K + d);
        const float f = weight_of(pm, pl, top);
        l += f * pl;
        if (f != 0.f) o += f * x;  // (an empty piece weighs nothing)
      }
      if (sub < subs && m0 + sub < rows) store_row4<Q>(p, r, kh, local * R + m, d, o, l);
    }
    return;
  }
  // a row at a time, its pieces dealt out to the waves in runs
  const int sub = lane / lanes, subs = 64 / lanes, d = lane % lanes * 4;
  const int run = (split + 3) / 4, begin = min(wave * run, split), end = min(begin + run, split);
  for (int m = blockIdx.y; m < rows; m += gridDim.y) {
    float top = -__builtin_inff(), l = 0.f;
    for (int i = begin + lane; i < end; i += 64) top = fmaxf(top, part[i * pitch + R * K + m]);
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
    pa_f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = begin; i0 < end; i0 += 64) {
      float f = 0.f;
      if (i0 + lane < end) {
        const float pm = part[(i0 + lane) * pitch + R * K + m], pl = part[(i0 + lane) * pitch + R * K + R + m];
        f = weight_of(pm, pl, top);
        l += f * pl;
      }
      const int n = min(64, end - i0);
      for (int j0 = 0; j0 < n; j0 += 8 * subs) {
        pa_f32x4 x[8];
        float w[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const int j = j0 + c * subs + sub;
          w[c] = __shfl(f, min(j, 63), 64);
          const bool in = j < n && sub < subs;
          if (!in) w[c] = 0.f;
          x[c] = *reinterpret_cast<const pa_f32x4*>(part + (i0 + (in ? j : 0)) * pitch + (int64_t)m * K + d);
        }
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (w[c] != 0.f) o += w[c] * x[c];  // (an empty piece weighs nothing)
      }
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) l += __shfl_xor(l, off, 64);
    pa_f32x4 sum = o;
    for (int j = 1; j < subs; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += __shfl(o[e], (lane + j * lanes) & 63, 64);
    if (sub == 0) *reinterpret_cast<pa_f32x4*>(&lds.o[wave][d]) = sum;
    if (lane == 0) lds.top[wave] = top, lds.l[wave] = l;
    __syncthreads();
    if (threadIdx.x < lanes) {
      float all = lds.top[0];
#pragma unroll
      for (int v = 1; v < 4; ++v) all = fmaxf(all, lds.top[v]);
      l = 0.f, o = pa_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float f = weight_of(lds.top[v], lds.l[v], all);
        l += f * lds.l[v];
        if (f != 0.f) o += f * *reinterpret_cast<const pa_f32x4*>(&lds.o[v][d]);
      }
      store_row4<Q>(p, r, kh, local * R + m, d, o, l);
    }
    __syncthreads();
  }
}

template <typename Q, int R>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs p) {
  __shared__ __attribute__((aligned(16))) JoinLds lds;
  join_block<Q, R>(p, blockIdx.x, lds);
}

// The same for a launch of both kinds.
template <int R>
__global__ __launch_bounds__(256) void paged_join_both_kernel(PagedArgs few, PagedArgs many, int many_blocks) {
  __shared__ __attribute__((aligned(16))) JoinLds lds;
  if ((int)blockIdx.x < many_blocks) join_block<uint16_t, kChunkRows>(many, blockIdx.x, lds);
  else join_block<uint16_t, R>(few, (int)blockIdx.x - many_blocks, lds);
}

// The blocks of one kind, as a launch is sized on the host.
struct Part {
  int R;           // rows of a unit, 0: none of this kind
  int over, upto;  // the sequences they take, by their rows of a key head
  int target, least, full;  // (paged_cut.h)
  int64_t units, items;  // at most
  bool cuts;      // whether a unit can be cut
  int64_t floats(int64_t Hk, int64_t K) const { return cuts ? items * Hk * R * (K + 2) : 0; }
};

// The sequences with at most 16 or 32 rows of a key head, and, where there may be others, those
// that the chunk blocks serve better.
struct Plan {
  Part few, many;
};

Part part_of(int R, int64_t over, int64_t upto, int target, int full, int uncut, int64_t T, int64_t S, int64_t P,
             int64_t page_size, int64_t G, int64_t Hk) {
  Part n;
  n.R = R, n.over = (int)over, n.upto = (int)upto, n.target = target;
  // a sequence of this launch has more than `over` rows; at most R of them are one unit
  const int64_t seqs = std::min(std::min(S, T), T * G / (over + 1) + (over == 0 ? T : 0));
  n.units = upto <= R ? seqs : std::min(T * G, T * G / R + seqs);
  const int64_t tiles = (P * page_size + kTile - 1) / kTile;
  n.cuts = tiles > uncut;  // a launch that can do without the join does
  n.least = n.cuts ? kLeast : uncut;
  n.full = n.cuts ? full : uncut;
  n.items = std::min(n.units * ((tiles + n.least - 1) / n.least), n.units + (target + Hk - 1) / Hk);
  return n;
}

Plan plan_of(int64_t T, int64_t S, int64_t P, int64_t page_size, int64_t G, int64_t Hk, int64_t K, int dtype,
             int held, int64_t max_new) {
  constexpr int64_t kAll = 0x7fffffff;
  const int64_t rows = std::min(T, max_new) * G;
  // a full piece is a quarter of a megabyte, 256 to 1024 keys: what is shorter takes its block's
  // beginning and the join longer than its keys, and pays only where CUs would have nothing (one
  // sequence of 1500 bf16 keys in pieces of 1024 12.6 us, of 256 9.7; 16 sequences of 3000 e4m3
  // keys, 8 heads of 128, in pieces of 1024 23 us, of 256 26; 700 keys uncut 9 us, in two pieces 14)
  const int64_t tile = 2 * kTile * K * (held == ABACUS_E4M3 ? 1 : held == kBF16 ? 2 : 4);
  const int full = (int)std::min<int64_t>(std::max<int64_t>((256 << 10) / tile, kLeast), 16);
  const bool chunks = dtype == kBF16;
  Plan n;
  n.many.R = 0, n.many.cuts = false;
  if (rows <= 32 || !chunks) {
    // a work-group fills a CU's registers: few turns of long pieces, as nothing covers a piece's
    // beginning (20 rows of 16 sequences over 9000 bf16 keys in pieces as the others 120 us, 87 so)
    const bool one = rows > 16 && K > 64;
    n.few = part_of(rows <= 16 ? 16 : 32, 0, kAll, one ? kOnePieces : kFewPieces, one ? 32 : full, full, T, S, P,
                    page_size, G, Hk);
  } else {
    const int few = G <= 16 ? 16 : 32;
    n.few = part_of(few, 0, few, kFewPieces, full, full, T, S, P, page_size, G, Hk);
    // (four tiles: 36 rows of 16 sequences over 3000 keys, K = 128, 54 us at 16, 44 at 4)
    int target = kChunkPieces;
    if (T == S * std::min(T, max_new)) {  // every sequence has a chunk of max_new
      const int64_t units = S * ((rows + kChunkRows - 1) / kChunkRows) * Hk;
      if ((kChunkPieces + units - 1) / units * units > kChunkPlaces) target = kChunkFiner;
    }
    n.many = part_of(kChunkRows, few, kAll, target, kLeast, kLeast, T, S, P, page_size, G, Hk);
  }
  return n;
}

template <typename Q, bool Cd, int QT>
void launch_few(const PagedArgs& p, unsigned blocks, hipStream_t s) {
  const dim3 grid(blocks), threads(256);
  // laid out for 32 dims instead of 64: 48 fp32 rows over 54074 keys 112 us, 63; not for codes, as
  // 16 bytes in each lane group are 64 dims there
  if constexpr (!Cd) {
    if (p.K <= 32) {
      if (p.K == 32) hipLaunchKernelGGL((paged_few_kernel<Q, Cd, 32, true, QT>), grid, threads, 0, s, p);
      else hipLaunchKernelGGL((paged_few_kernel<Q, Cd, 32, false, QT>), grid, threads, 0, s, p);
      return;
    }
  }
  if (p.K == 64) hipLaunchKernelGGL((paged_few_kernel<Q, Cd, 64, true, QT>), grid, threads, 0, s, p);
  else if (p.K == 128) hipLaunchKernelGGL((paged_few_kernel<Q, Cd, 128, true, QT>), grid, threads, 0, s, p);
  else if (p.K < 64) hipLaunchKernelGGL((paged_few_kernel<Q, Cd, 64, false, QT>), grid, threads, 0, s, p);
  else hipLaunchKernelGGL((paged_few_kernel<Q, Cd, 128, false, QT>), grid, threads, 0, s, p);
}

template <typename Q>
int launch(const PagedArgs& p, const Plan& n, bool codes, float* ws, int64_t rows, hipStream_t s) {
  auto args = [&](const Part& part, float* at) {
    PagedArgs a = p;
    a.over = part.over, a.upto = part.upto, a.target = part.target, a.least = part.least, a.full = part.full, a.part = at;
    return a;
  };
  const PagedArgs few = args(n.few, ws);
  const unsigned few_blocks = (unsigned)(n.few.items * p.Hk);
  const unsigned few_units = n.few.cuts ? (unsigned)(n.few.units * p.Hk) : 0;
  // a join block per row where that makes few blocks (a chunk of 128 rows over 243 pieces 52 us
  // with eight rows a block, 30 with one), else per four or more
  auto join_y = [&](int64_t units, int R) {
    const int64_t most = std::min<int64_t>(R, rows), at_once = std::min<int64_t>(most, 16);
    return (unsigned)(units < 128 ? std::max(at_once, std::min(most, 1024 / units)) : (at_once + 3) / 4);
  };
  if constexpr (sizeof(Q) == 2) {
    if (n.many.R > 0) {
      const PagedArgs many = args(n.many, ws + n.few.floats(p.Hk, p.K));
      if (launch_both(few, many, few_blocks, (unsigned)(n.many.items * p.Hk), n.few.R, codes, s)) return 2;
      const unsigned units = n.many.cuts ? (unsigned)(n.many.units * p.Hk) : 0;
      if (units + few_units > 0) {
        const dim3 grid(units + few_units, join_y(units + few_units, kChunkRows));
        if (n.few.R == 16) hipLaunchKernelGGL(paged_join_both_kernel<16>, grid, dim3(256), 0, s, few, many, (int)units);
        else hipLaunchKernelGGL(paged_join_both_kernel<32>, grid, dim3(256), 0, s, few, many, (int)units);
        ABACUS_CHECK_LAUNCH("paged_attention (join)");
      }
      return 0;
    }
  }
  if (n.few.R == 16) codes ? launch_few<Q, true, 1>(few, few_blocks, s) : launch_few<Q, false, 1>(few, few_blocks, s);
  else codes ? launch_few<Q, true, 2>(few, few_blocks, s) : launch_few<Q, false, 2>(few, few_blocks, s);
  ABACUS_CHECK_LAUNCH("paged_attention");
  if (few_units > 0) {
    const dim3 grid(few_units, join_y(few_units, n.few.R));
    if (n.few.R == 16) hipLaunchKernelGGL((paged_join_kernel<Q, 16>), grid, dim3(256), 0, s, few);
    else hipLaunchKernelGGL((paged_join_kernel<Q, 32>), grid, dim3(256), 0, s, few);
    ABACUS_CHECK_LAUNCH("paged_attention (join)");
  }
  return 0;
}

}  // namespace
}  // namespace abacus

using namespace abacus;

extern "C" int64_t abacus_paged_attention_ws_bytes(int64_t T, int64_t H, int64_t Hk, int64_t K, int dtype, int held,
                                                   int64_t S, int64_t P, int64_t page_size, int64_t max_new) {
  if (T < 1 || Hk < 1 || H % Hk != 0) return 0;
  const Plan n = plan_of(T, S, P, page_size, H / Hk, Hk, K, dtype, held, max_new);
  return (n.few.floats(Hk, K) + n.many.floats(Hk, K)) * 4;
}

extern "C" int abacus_paged_attention(const void* q_THK, int64_t T, int64_t H, int64_t Hk, int64_t K, int dtype,
                                      const int32_t* page_table_SP, const int32_t* query_start,
                                      const int32_t* lengths, int64_t S, int64_t P, int64_t page_size,
                                      int64_t n_pages, int held, const void* k_pages, const void* v_pages,
                                      const void* k_scale, const void* v_scale, float scale, int64_t max_new,
                                      int zero_rest, void* o_THK, void* ws, int64_t ws_bytes, void* stream) {
  if (check_paged_rows("paged_attention", page_table_SP, query_start, lengths, S, P, T, page_size, n_pages, Hk, K))
    return 1;
  ABACUS_CHECK_ARG(dtype == kF32 || dtype == kBF16, "paged_attention: dtype code %d", dtype);
  ABACUS_CHECK_ARG(held == dtype || held == ABACUS_E4M3, "paged_attention: a cache of dtype code %d with queries of %d",
                   held, dtype);
  ABACUS_CHECK_ARG(H >= Hk && H % Hk == 0 && H <= 1024, "paged_attention: %lld heads over %lld key heads", (long long)H,
                   (long long)Hk);
  ABACUS_CHECK_ARG(T * H < (1ll << 31), "paged_attention: %lld rows of %lld heads are too many", (long long)T, (long long)H);
  ABACUS_CHECK_ARG(scale > 0.f && scale < __builtin_inff(), "paged_attention: scale %g", (double)scale);
  ABACUS_CHECK_ARG(max_new >= 1, "paged_attention: max_new %lld", (long long)max_new);
  if (T == 0) return 0;
  ABACUS_CHECK_ARG(q_THK && k_pages && v_pages && o_THK && (held != ABACUS_E4M3 || (k_scale && v_scale)),
                   "paged_attention: null pointer");
  ABACUS_CHECK_ARG(((uintptr_t)q_THK | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)k_scale |
                    (uintptr_t)v_scale | (uintptr_t)o_THK | (uintptr_t)ws) % 16 == 0,
                   "paged_attention: tensors must be 16-byte aligned");
  const Plan n = plan_of(T, S, P, page_size, H / Hk, Hk, K, dtype, held, max_new);
  const int64_t need = (n.few.floats(Hk, K) + n.many.floats(Hk, K)) * 4;
  ABACUS_CHECK_ARG(need == 0 || (ws && ws_bytes >= need), "paged_attention: workspace of %lld bytes, need %lld",
                   (long long)ws_bytes, (long long)need);
  // a launch holds fewer than 2^32 threads, 256 to a block
  ABACUS_CHECK_ARG((n.few.items + (n.many.R > 0 ? n.many.items : 0)) * Hk < (1ll << 24),
                   "paged_attention: %lld rows of %lld heads in %lld sequences are too many", (long long)T, (long long)H,
                   (long long)S);
  PagedArgs p;
  p.a = PagedRows{page_table_SP, query_start, lengths, (int)S, (int)P, (int)T, __builtin_ctzll(page_size), (int)n_pages};
  p.q = q_THK, p.k = k_pages, p.v = v_pages;
  p.k_scale = (const uint8_t*)k_scale, p.v_scale = (const uint8_t*)v_scale;
  p.o = o_THK;
  p.H = (int)H, p.Hk = (int)Hk, p.G = (int)(H / Hk), p.K = (int)K;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.zero_rest = zero_rest;
  hipStream_t s = (hipStream_t)stream;
  const bool codes = held == ABACUS_E4M3;
  const int64_t rows = std::min(T, max_new) * (H / Hk);
  return dtype == kBF16 ? launch<uint16_t>(p, n, codes, (float*)ws, rows, s) : launch<float>(p, n, codes, (float*)ws, rows, s);
}
