// The embedding of tokens and its gradient.  Reference: abacus/embedding.py:20-23, w[tokens], and its derivative.
//
//   out[t] = scale * w[token_t]                      a negative token counts from the end, as torch's indexing has it
//   dw[v]  = scale * sum over t with token_t = v of dy[t]     in fp32, in the order of t
//
// Forward: a row is read and written once.  Backward: the tokens are sorted by id without a sort's passes:
//   1. sort: a work-group owns a range of ids.  It reads all tokens, counts its own (a counter for each wave's part of
//      the tokens and id, in LDS) and those of ids before its range, which is where its part of the sorted list
//      starts; a second reading writes the list.  No work-group waits for another and no order is left to chance.
//   2. rows: a wave adds up a row of dw and writes it, zeros where no token has the id.  Ids with many tokens (kHot
//      and more: padding, a frequent word) would keep one wave busy alone, so their sorted positions are
//      added up in pieces of kPiece by work-groups of the same launch, in fp32;
//   3. join: which a last launch adds in order.
#include <algorithm>

#include "common.h"

namespace abacus {
namespace {

constexpr int kPiece = 64;     // sorted positions of a piece
constexpr int kHot = kPiece;   // an id with more tokens goes by pieces: a piece then holds parts of two such ids at most
constexpr int kSortWaves = 16;
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

// start[v] .. start[v + 1] - 1 are the places in `order` of the tokens of id v, in the order of t.
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
  int before = 0;
  for (int t = t0 + lane; t < t1; t += 64) {
    const int v = row_of(tokens[t], V);
    before += v >= 0 && v < lo;
    if (v >= lo && v < lo + mine) atomicAdd(&count[v - lo], 1);
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
  for (int b = t0; b < t1; b += 64) {
    const int t = b + lane;
    const int v = t < t1 ? row_of(tokens[t], V) - lo : -1;
    const bool in = v >= 0 && v < mine;
    uint64_t left = __ballot(in);
    while (left) {  // an id at a time
      const int leader = __ffsll((unsigned long long)left) - 1;
      const int id = __shfl(v, leader, 64);
      const uint64_t same = __ballot(in && v == id);
      const int place = next[id];
      if (in && v == id) order[place + __popcll(same & ((1ull << lane) - 1))] = t;
      if (lane == leader) next[id] = place + __popcll(same);
      left &= ~same;
    }
  }
}

// Sum of dy's rows order[a] .. order[b - 1] at column c.
template <typename T>
__device__ inline void add_rows(const T* dy, const int* order, int a, int b, int D, int c, float* f) {
  constexpr int EPV = VecTraits<T>::kN;
#pragma unroll
  for (int k = 0; k < EPV; ++k) f[k] = 0.f;
  int i = a;
  for (; i + 4 <= b; i += 4) {
    float g[4][EPV];
#pragma unroll
    for (int u = 0; u < 4; ++u) load_any<T>(dy + (int64_t)order[i + u] * D + c, D - c, g[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int k = 0; k < EPV; ++k) f[k] += g[u][k];
  }
  for (; i < b; ++i) {
    float g[EPV];
    load_any<T>(dy + (int64_t)order[i] * D + c, D - c, g);
#pragma unroll
    for (int k = 0; k < EPV; ++k) f[k] += g[k];
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

template <typename T>
__global__ __launch_bounds__(256) void embedding_rows_kernel(const int64_t* __restrict__ tokens, const T* __restrict__ dy,
                                                             const int* __restrict__ start, const int* __restrict__ order,
                                                             int V, int D, float scale, int pieces,
                                                             float* __restrict__ parts, T* __restrict__ dw) {
  constexpr int EPV = VecTraits<T>::kN;
  const int tid = threadIdx.x, lane = tid & 63;
  if ((int)blockIdx.x < 2 * pieces) {  // (the long ones first)
    Piece pc;
    const int p = blockIdx.x >> 1, slot = blockIdx.x & 1;
    if (!pc.find(tokens, start, order, V, p, slot)) return;
    for (int c = tid * EPV; c < D; c += 256 * EPV) {
      float f[EPV];
      add_rows<T>(dy, order, pc.a, pc.b, D, c, f);
      float* out = parts + (int64_t)blockIdx.x * D + c;
#pragma unroll
      for (int k = 0; k < EPV; ++k)
        if (c + k < D) out[k] = f[k];
    }
    return;
  }
  const int v = ((int)blockIdx.x - 2 * pieces) * 4 + (tid >> 6);
  if (v >= V) return;
  const int a = start[v], b = start[v + 1];
  if (b - a > kHot) return;
  for (int c = lane * EPV; c < D; c += 64 * EPV) {
    float f[EPV];
    add_rows<T>(dy, order, a, b, D, c, f);
#pragma unroll
    for (int k = 0; k < EPV; ++k) f[k] *= scale;
    store_any<T>(dw + (int64_t)v * D + c, D - c, f);
  }
}

// Hot ids: the pieces' sums in order, 64 columns a work-group whose 16 waves take every 16th piece.
template <typename T>
__global__ __launch_bounds__(1024) void embedding_join_kernel(const int64_t* __restrict__ tokens, const int* __restrict__ start,
                                                              const int* __restrict__ order, int V, int D, float scale,
                                                              const float* __restrict__ parts, T* __restrict__ dw) {
  __shared__ float sum_s[16][64];
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, c = blockIdx.y * 64 + l;
  const int p = blockIdx.x >> 1, slot = blockIdx.x & 1;
  Piece pc;
  if (!pc.find(tokens, start, order, V, p, slot) || pc.first < p * kPiece) return;  // (not the piece that it starts in)
  const int n = (pc.last - 1) / kPiece - p + 1;
  float s = 0.f;
  for (int k = w; k < n; k += 16)
    if (c < D) s += parts[((int64_t)(p + k) * 2 + (k == 0 ? slot : 0)) * D + c];
  sum_s[w][l] = s;
  __syncthreads();
  if (w == 0 && c < D) {
    for (int k = 1; k < 16; ++k) s += sum_s[k][l];
    dw[(int64_t)pc.id * D + c] = from_f32<T>(s * scale);
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
  int64_t start, order, parts, total;
  Space(int64_t T, int64_t V, int64_t D) {
    auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
    start = 0;
    order = up((V + 1) * 4);
    parts = order + up(T * 4);
    total = parts + (T > kHot ? (T + kPiece - 1) / kPiece * 2 * D * 4 : 0);
  }
};

template <typename T>
int backward(const int64_t* tokens, const void* dy, int64_t n, int64_t V, int64_t D, float scale, void* dw, char* ws,
             hipStream_t s) {
  const Space sp(n, V, D);
  int* start = (int*)(ws + sp.start);
  int* order = (int*)(ws + sp.order);
  float* parts = (float*)(ws + sp.parts);
  const int ids = (int)std::min<int64_t>(kMaxIds, (V + 255) / 256);
  hipLaunchKernelGGL(embedding_sort_kernel, dim3((unsigned)((V + ids - 1) / ids)), dim3(kSortWaves * 64),
                     kSortWaves * ids * 4, s, tokens, (int)n, (int)V, ids, start, order);
  ABACUS_CHECK_LAUNCH("embedding_bwd sort");
  const int pieces = n > kHot ? (int)((n + kPiece - 1) / kPiece) : 0;
  hipLaunchKernelGGL(embedding_rows_kernel<T>, dim3((unsigned)(2 * pieces + (V + 3) / 4)), dim3(256), 0, s, tokens, (const T*)dy,
                     start, order, (int)V, (int)D, scale, pieces, parts, (T*)dw);
  ABACUS_CHECK_LAUNCH("embedding_bwd rows");
  if (pieces) {
    hipLaunchKernelGGL(embedding_join_kernel<T>, dim3(2 * pieces, (unsigned)((D + 63) / 64)), dim3(1024), 0, s, tokens, start,
                       order, (int)V, (int)D, scale, parts, (T*)dw);
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
  const int64_t need = Space(T, V, D).total;
  ABACUS_CHECK_ARG(ws != nullptr && ws_bytes >= need, "embedding_bwd: workspace of %lld bytes, %lld needed",
                   (long long)ws_bytes, (long long)need);
  return dtype == kBF16 ? backward<uint16_t>(tokens_T, d_out_TD, T, V, D, scale, dw_VD, (char*)ws, (hipStream_t)stream)
                        : backward<float>(tokens_T, d_out_TD, T, V, D, scale, dw_VD, (char*)ws, (hipStream_t)stream);
}

}  // extern "C"
