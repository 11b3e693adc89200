// The embedding of tokens and its gradient.  Reference: abacus/embedding.py:20-23, w[tokens], and its derivative.
//
//   out[t] = scale * w[token_t]                      a negative token counts from the end, as torch's indexing has it
//   dw[v]  = scale * sum over t with token_t = v of dy[t]     in fp32, in a fixed order
//
// Forward: a row is read and written once.  Backward: the tokens are sorted by id without a sort's passes:
//   1. sort: a work-group owns a range of ids.  It reads all tokens, counts its own (a counter for each wave's part of
//      the tokens and id, in LDS) and those of ids before its range, which is where its part of the sorted list
//      starts; a second reading writes the list.  No work-group waits for another and no order is left to chance.
//   2. rows: a wave adds up 64 vectors of the rows of kIds ids in the order of t and writes them, zeros where no token has
//      the id.  Ids with many tokens (more than kHot: padding, a frequent word) would keep one wave busy alone, so their
//      sorted positions are added up in pieces of kPiece by work-groups of the same launch, in fp32;
//   3. join: which a last launch adds, every fourth piece in order and the four sums.
// Bound by bytes, and short calls by the launches: 8192 x 1024 of 32000 bf16 takes 46 us both ways, 23 at a copy's rate;
// 16384 x 2048 of 50257 fp32, a third of the tokens one id, 205 us, 160 at that rate.
#include <algorithm>

#include "common.h"

namespace abacus {
namespace {

// Sorted positions of a piece: 16, 32 and 64 cost the join 51, 25 and 17 us of 16384 x 2048 fp32 with 5500 tokens of one id,
// and the rows' launch, with 2, 4 and 8 ids a wave, 24.0, 23.4 and 32.1 us of 8192 x 1024 of 32000 bf16.
constexpr int kPiece = 32;
constexpr int kHot = kPiece;   // an id with more tokens goes by pieces: a piece then holds parts of two such ids at most
constexpr int kIds = 4;        // of a wave
constexpr int kRowsAhead = 8;  // rows of dy whose loads are in flight together
constexpr int kSortWaves = 16;
constexpr int kSortAhead = 8;  // tokens a lane, likewise
constexpr int kMaxIds = 960;   // of a sorting work-group (its counters under 64 KB)

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

// Its row, or -1: no row of the table.
__device__ inline int row_of(int64_t token, int V) {
  if (token < 0) token += V;
  return token >= 0 && token < V ? (int)token : -1;
}

template <typename T>
__device__ inline void load_any(const T* p, int n, float* f) {
  constexpr int EPV = VecTraits<T>::kN;
  if (n >= EPV) {
    const u32x4_any v = *reinterpret_cast<const u32x4_any*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) {
        f[2 * i] = lo_bf16(v[i]);
        f[2 * i + 1] = hi_bf16(v[i]);
      } else {
        f[i] = bits_f32(v[i]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < EPV; ++i) f[i] = i < n ? to_f32<T>(p[i]) : 0.f;
  }
}

template <typename T>
__device__ inline void store_any(T* p, int n, const float* f) {
  constexpr int EPV = VecTraits<T>::kN;
  if (n >= EPV) {
    u32x4_any v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) v[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
      else v[i] = f32_bits(f[i]);
    }
    *reinterpret_cast<u32x4_any*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < EPV; ++i)
      if (i < n) p[i] = from_f32<T>(f[i]);
  }
}

// A vector of 16 bytes a thread: 8192 x 1024 bf16 7 us, 16384 x 2048 fp32 46 us (5.8 TB/s), 64 x 2048 bf16 2.7 us.
template <typename T>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(const int64_t* __restrict__ tokens, const T* __restrict__ w,
                                                            int64_t n, int vecs, int V, int D, float scale,
                                                            T* __restrict__ out) {
  constexpr int EPV = VecTraits<T>::kN;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / vecs;
    const int c = (int)(i - t * vecs) * EPV, row = row_of(tokens[t], V);
    float f[EPV];
    load_any<T>(w + (int64_t)max(row, 0) * D + c, D - c, f);
#pragma unroll
    for (int k = 0; k < EPV; ++k) f[k] = row < 0 ? __builtin_nanf("") : f[k] * scale;
    store_any<T>(out + t * D + c, D - c, f);
  }
}

// ---------------------------------------------------------------- backward

// start[v] .. start[v + 1] - 1 are the places in `order` of the tokens of id v, in the order of t.  Bound by the work-group
// that owns the most frequent ids, whose tokens of one id take turns: 8192 tokens 12 us, 16384 20, 65536 (20000 of one
// id) 58.  Tables of more ids than 256 work-groups own have the tokens read more often: both ways of 65536 tokens of
// 500000 x 64 bf16 take 190 us, of 300000 of 2000000 x 64 1220, where indexing takes 103 and 385 if no id is frequent, 14000
// and 91000 if half of the tokens are one.  More tokens in flight (16 or 32 a lane) changed nothing, the lanes of one id
// found by bits instead of id by id cost 73.
__global__ __launch_bounds__(kSortWaves * 64) void embedding_sort_kernel(const int64_t* __restrict__ tokens, int T, int V,
                                                                         int ids, int* __restrict__ start,
                                                                         int* __restrict__ order) {
  extern __shared__ int count_s[];  // (kSortWaves, ids)
  __shared__ int wave_s[kSortWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lo = blockIdx.x * ids, mine = min(ids, V - lo);
  for (int i = tid; i < kSortWaves * ids; i += kSortWaves * 64) count_s[i] = 0;
  __syncthreads();
  const int part = ((T + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
  const int t0 = wave * part, t1 = min(T, t0 + part);
  int* count = count_s + wave * ids;
  auto read = [&](int b, int (&v)[kSortAhead]) {  // ids of tokens b .. of this wave, -1 past its part
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u) {
      const int t = b + u * 64 + lane;
      v[u] = t < t1 ? row_of(tokens[t], V) : -1;
    }
  };
  int before = 0;
  for (int b = t0; b < t1; b += 64 * kSortAhead) {
    int v[kSortAhead];
    read(b, v);
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u) {
      before += v[u] >= 0 && v[u] < lo;
      if (v[u] >= lo && v[u] < lo + mine) atomicAdd(&count[v[u] - lo], 1);
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) before += __shfl_xor(before, off, 64);
  if (lane == 0) wave_s[wave] = before;
  __syncthreads();
  before = 0;
  for (int w = 0; w < kSortWaves; ++w) before += wave_s[w];
  __syncthreads();
  // a thread an id: its tokens over the waves, then a scan over the ids
  int own = 0;
  if (tid < mine)
    for (int w = 0; w < kSortWaves; ++w) own += count_s[w * ids + tid];
  int scan = own;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int up = __shfl_up(scan, off, 64);
    if (lane >= off) scan += up;
  }
  if (lane == 63) wave_s[wave] = scan;
  __syncthreads();
  int at = before + scan - own;
  for (int w = 0; w < wave; ++w) at += wave_s[w];
  if (tid < mine) {
    start[lo + tid] = at;
    if (lo + tid == V - 1) start[V] = at + own;
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = count_s[w * ids + tid];
      count_s[w * ids + tid] = at;
      at += c;
    }
  }
  __syncthreads();
  // the same reading again: count[] is now the next free place
  volatile int* next = count;
  for (int b = t0; b < t1; b += 64 * kSortAhead) {
    int ids_[kSortAhead];
    read(b, ids_);
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u) {
      const int v = ids_[u] - lo;
      const bool in = v >= 0 && v < mine;
      uint64_t left = __ballot(in);
      while (left) {  // an id at a time
        const int leader = __ffsll((unsigned long long)left) - 1;
        const int id = __shfl(v, leader, 64);
        const uint64_t same = __ballot(in && v == id);
        const int place = next[id];
        if (in && v == id) order[place + __popcll(same & ((1ull << lane) - 1))] = b + u * 64 + lane;
        if (lane == leader) next[id] = place + __popcll(same);
        left &= ~same;
      }
    }
  }
}

// f = the sum of n rows of dy at column c, in order; row k's number is the k-th lane's `mine` (n at most 64).
template <typename T>
__device__ inline void add_rows(const T* dy, int mine, int n, int D, int c, float* f) {
  constexpr int EPV = VecTraits<T>::kN;
#pragma unroll
  for (int k = 0; k < EPV; ++k) f[k] = 0.f;
  for (int i = 0; i < n; i += kRowsAhead) {
    float g[kRowsAhead][EPV];
#pragma unroll
    for (int u = 0; u < kRowsAhead; ++u) {
      const int t = __builtin_amdgcn_readlane(mine, min(i + u, n - 1));
      load_any<T>(dy + (int64_t)t * D + c, i + u < n ? D - c : 0, g[u]);
    }
#pragma unroll
    for (int u = 0; u < kRowsAhead; ++u)
#pragma unroll
      for (int k = 0; k < EPV; ++k) f[k] += g[u][k];
  }
}

// The hot id whose tokens piece `p` holds at its start (slot 0) or at its end (slot 1), and its places there; false: none.
struct Piece {
  int id, first, last;  // all of the id's places
  int a, b;             // those in the piece
  __device__ inline bool find(const int64_t* tokens, const int* start, const int* order, int V, int p, int slot) {
    const int total = start[V], p0 = p * kPiece, p1 = min(p0 + kPiece, total);
    if (p0 >= p1) return false;
    id = row_of(tokens[order[slot == 0 ? p0 : p1 - 1]], V);
    if (slot == 1 && id == row_of(tokens[order[p0]], V)) return false;
    first = start[id];
    last = start[id + 1];
    a = max(first, p0);
    b = min(last, p1);
    return last - first > kHot;
  }
};

// Work-groups 0 .. 2 pieces - 1: (piece, slot); they note in `joins` which id, if any, a piece is the first of.
// The others: a wave takes kIds ids and 64 vectors of their rows.  (8192 x 1024 of 32000 bf16 23.5 us, of which the table's
// rows are 66 MB written; 16384 x 2048 of 50257 fp32 114 us, 4.8 TB/s; an id a wave and a row at a time 55 and 321.)
template <typename T>
__global__ __launch_bounds__(256) void embedding_rows_kernel(const int64_t* __restrict__ tokens, const T* __restrict__ dy,
                                                             const int* __restrict__ start, const int* __restrict__ order,
                                                             int V, int D, int slabs, float scale, int pieces,
                                                             int* __restrict__ joins, float* __restrict__ parts,
                                                             T* __restrict__ dw) {
  constexpr int EPV = VecTraits<T>::kN;
  const int tid = threadIdx.x, lane = tid & 63;
  if ((int)blockIdx.x < 2 * pieces) {  // (the long ones first)
    Piece pc;
    const int p = blockIdx.x >> 1, slot = blockIdx.x & 1;
    const bool hot = pc.find(tokens, start, order, V, p, slot);
    if (tid == 0) joins[blockIdx.x] = hot && pc.first >= p * kPiece ? pc.id : -1;
    if (!hot) return;
    const int n = pc.b - pc.a, mine = order[pc.a + min(lane, n - 1)];
    for (int c0 = 0; c0 < D; c0 += 256 * EPV) {
      const int c = c0 + tid * EPV;
      float f[EPV];
      add_rows<T>(dy, mine, n, D, c, f);
      float* out = parts + (int64_t)blockIdx.x * D + c;
#pragma unroll
      for (int k = 0; k < EPV; ++k)
        if (c + k < D) out[k] = f[k];
    }
    return;
  }
  const int64_t task = ((int64_t)blockIdx.x - 2 * pieces) * 4 + (tid >> 6);
  const int v0 = (int)(task / slabs) * kIds, c = (int)(task % slabs) * 64 * EPV + lane * EPV;
  if (v0 >= V) return;
  const int bound = start[min(v0 + min(lane, kIds), V)];
  int a[kIds], n[kIds], mine[kIds];
#pragma unroll
  for (int k = 0; k < kIds; ++k) {
    a[k] = __builtin_amdgcn_readlane(bound, k);
    n[k] = __builtin_amdgcn_readlane(bound, k + 1) - a[k];
    mine[k] = lane < n[k] ? order[a[k] + lane] : 0;
  }
#pragma unroll
  for (int k = 0; k < kIds; ++k) {
    if (v0 + k >= V || n[k] > kHot) continue;
    float f[EPV];
    add_rows<T>(dy, mine[k], n[k], D, c, f);
#pragma unroll
    for (int i = 0; i < EPV; ++i) f[i] *= scale;
    store_any<T>(dw + (int64_t)(v0 + k) * D + c, D - c, f);
  }
}

// Hot ids: the pieces' sums in order, 64 columns a work-group whose 4 waves take every 4th piece.  (4 us where few ids are,
// 25 for 172 pieces of 2048 columns: a chain of additions.)
template <typename T>
__global__ __launch_bounds__(256) void embedding_join_kernel(const int* __restrict__ start, const int* __restrict__ joins,
                                                             int V, int D, float scale, const float* __restrict__ parts,
                                                             T* __restrict__ dw) {
  __shared__ float sum_s[4][64];
  const int id = joins[blockIdx.x];
  if (id < 0) return;
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int p = blockIdx.x >> 1, slot = blockIdx.x & 1, n = (start[id + 1] - 1) / kPiece - p + 1;
  for (int c0 = blockIdx.y * 64; c0 < D; c0 += gridDim.y * 64) {
    const int c = min(c0 + l, D - 1);
    float s = 0.f;
#pragma unroll 8
    for (int k = w; k < n; k += 4) s += parts[((int64_t)(p + k) * 2 + (k == 0 ? slot : 0)) * D + c];
    sum_s[w][l] = s;
    __syncthreads();
    if (w == 0 && c0 + l < D) dw[(int64_t)id * D + c] = from_f32<T>((((s + sum_s[1][l]) + sum_s[2][l]) + sum_s[3][l]) * scale);
    __syncthreads();
  }
}

int check(const char* name, int64_t T, int64_t V, int64_t D, int dtype) {
  ABACUS_CHECK_ARG(dtype == kF32 || dtype == kBF16, "%s: unsupported dtype code %d (0 = fp32, 1 = bf16)", name, dtype);
  ABACUS_CHECK_ARG(T >= 0 && T < (1ll << 30), "%s: %lld tokens", name, (long long)T);
  ABACUS_CHECK_ARG(V >= 1 && V < (1ll << 30), "%s: a table of %lld rows", name, (long long)V);
  ABACUS_CHECK_ARG(D >= 1 && D < (1ll << 22), "%s: dim %lld", name, (long long)D);
  return 0;
}

struct Space {
  int64_t start, order, joins, parts, total;
  Space(int64_t T, int64_t V, int64_t D) {
    auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
    start = 0;
    order = up((V + 1) * 4);
    joins = order + up(T * 4);
    const int64_t slots = T > kHot ? (T + kPiece - 1) / kPiece * 2 : 0;
    parts = joins + up(slots * 4);
    total = parts + slots * D * 4;
  }
};

template <typename T>
int backward(const int64_t* tokens, const void* dy, int64_t n, int64_t V, int64_t D, float scale, void* dw, char* ws,
             hipStream_t s) {
  const Space sp(n, V, D);
  int* start = (int*)(ws + sp.start);
  int* order = (int*)(ws + sp.order);
  int* joins = (int*)(ws + sp.joins);
  float* parts = (float*)(ws + sp.parts);
  const int pieces = n > kHot ? (int)((n + kPiece - 1) / kPiece) : 0;
  const int slabs = (int)((D + 64 * VecTraits<T>::kN - 1) / (64 * VecTraits<T>::kN));
  const int64_t tasks = (V + kIds - 1) / kIds * slabs, blocks = 2 * pieces + (tasks + 3) / 4;
  // (a launch has fewer than 2^32 threads a dimension)
  ABACUS_CHECK_ARG(blocks < (1ll << 24), "embedding_bwd: %lld tokens of a table of %lld x %lld", (long long)n, (long long)V,
                   (long long)D);
  const int ids = (int)std::min<int64_t>(kMaxIds, (V + 255) / 256);
  hipLaunchKernelGGL(embedding_sort_kernel, dim3((unsigned)((V + ids - 1) / ids)), dim3(kSortWaves * 64),
                     kSortWaves * ids * 4, s, tokens, (int)n, (int)V, ids, start, order);
  ABACUS_CHECK_LAUNCH("embedding_bwd sort");
  hipLaunchKernelGGL(embedding_rows_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, s, tokens, (const T*)dy, start, order, (int)V,
                     (int)D, slabs, scale, pieces, joins, parts, (T*)dw);
  ABACUS_CHECK_LAUNCH("embedding_bwd rows");
  if (pieces) {
    hipLaunchKernelGGL(embedding_join_kernel<T>, dim3(2 * pieces, (unsigned)std::min<int64_t>((D + 63) / 64, 8)), dim3(256), 0, s,
                       start, joins, (int)V, (int)D, scale, parts, (T*)dw);
    ABACUS_CHECK_LAUNCH("embedding_bwd join");
  }
  return 0;
}

}  // namespace
}  // namespace abacus

using namespace abacus;

extern "C" {

int abacus_embedding_fwd(const int64_t* tokens_T, const void* w_VD, int64_t T, int64_t V, int64_t D, float scale, int dtype,
                         void* out_TD, void* stream) {
  if (int rc = check("embedding_fwd", T, V, D, dtype)) return rc;
  if (T == 0) return 0;
  ABACUS_CHECK_ARG(tokens_T && w_VD && out_TD, "embedding_fwd: null pointer");
  const int epv = dtype == kBF16 ? 8 : 4, vecs = (int)((D + epv - 1) / epv);
  const int64_t n = T * vecs;
  const unsigned blocks = (unsigned)std::min<int64_t>((n + 255) / 256, 1 << 16);
  if (dtype == kBF16)
    hipLaunchKernelGGL(embedding_fwd_kernel<uint16_t>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, tokens_T,
                       (const uint16_t*)w_VD, n, vecs, (int)V, (int)D, scale, (uint16_t*)out_TD);
  else
    hipLaunchKernelGGL(embedding_fwd_kernel<float>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, tokens_T,
                       (const float*)w_VD, n, vecs, (int)V, (int)D, scale, (float*)out_TD);
  ABACUS_CHECK_LAUNCH("embedding_fwd");
  return 0;
}

int64_t abacus_embedding_bwd_ws_bytes(int64_t T, int64_t V, int64_t D) {
  if (T < 0 || V <= 0 || D <= 0) return 0;
  return Space(T, V, D).total;
}

int abacus_embedding_bwd(const int64_t* tokens_T, const void* d_out_TD, int64_t T, int64_t V, int64_t D, float scale,
                         int dtype, void* dw_VD, void* ws, int64_t ws_bytes, void* stream) {
  if (int rc = check("embedding_bwd", T, V, D, dtype)) return rc;
  ABACUS_CHECK_ARG(dw_VD && (T == 0 || (tokens_T && d_out_TD)), "embedding_bwd: null pointer");
  const int64_t need = Space(T, V, D).total;
  ABACUS_CHECK_ARG(ws != nullptr && (uintptr_t)ws % 16 == 0 && ws_bytes >= need,
                   "embedding_bwd: workspace of %lld bytes, %lld needed, 16-byte aligned", (long long)ws_bytes, (long long)need);
  return dtype == kBF16 ? backward<uint16_t>(tokens_T, d_out_TD, T, V, D, scale, dw_VD, (char*)ws, (hipStream_t)stream)
                        : backward<float>(tokens_T, d_out_TD, T, V, D, scale, dw_VD, (char*)ws, (hipStream_t)stream);
}

}  // extern "C"
