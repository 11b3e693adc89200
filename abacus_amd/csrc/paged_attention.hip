// Attention of new tokens over a paged key/value cache.
//
// Row j of a sequence's n new tokens has position len - n + j and sees the keys
// up to it: o = sum_j softmax(scale q . k_j) v_j, query head h with key head h / G.
// One pass over the keys with the running maximum and sum of the softmax in fp32.
//
// How the work is cut over units of rows and pieces of keys is paged_cut.h's; sequences with
// many bf16 rows go to paged_chunk.hip's kernel, the others and all fp32 ones to this file's.
//
// In registers (v_mfma_f32_16x16x32_bf16: lane l gives A[l % 16][8 (l / 16) .. +7] and
// B[8 (l / 16) .. +7][l % 16], and holds D[4 (l / 16) + r][l % 16] in register r; the fp32
// product takes one element of each per lane): a wave's tile is four groups of KG keys, as
// many as 16 bytes of values hold (16 codes, 8 bf16, 4 fp32).  S^T = K Q^T takes them in KG / 4
// products t whose row i is key KG (i / 4) + 4 t + i % 4.  Lane l then holds the scores of
// query l % 16 against the KG keys of group l / 16, in their order, and those are, as they
// lie, the operand P^T of O^T = V^T P^T with 16 bytes of a V^T row: neither the scores nor a
// tile of keys or values goes through LDS, and every load of the cache is 16 bytes a lane.
#include <algorithm>
#include <type_traits>

#include "paged_cut.h"

namespace abacus {
namespace {

constexpr int kFewPieces = 2048;   // pieces the work of a launch is cut into, about
constexpr int kWavesOf16 = 4;      // waves of a block of 16 rows
constexpr int kFewJoined = 16;     // pieces that a wave joins for several rows at once
constexpr int kChunkPieces = 512;  // (of the chunk kernel's: two work-groups a CU)

typedef __bf16 pa_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 pa_bf16x2 __attribute__((ext_vector_type(2)));
typedef float pa_f32x4 __attribute__((ext_vector_type(4)));
// 16 bytes of operands.  A vector and not Vec16's four words: of words loaded together and
// masked on a branch the compiler (ROCm 7.2) let some be overwritten before their use.
typedef uint32_t pa_u32x4 __attribute__((ext_vector_type(4)));

// The value of lanes l, l ^ 16, l ^ 32 and l ^ 48, combined (no LDS round trip).
template <class Op>
__device__ inline float over_groups(float x, Op op) {
  uint32_t a = f32_bits(x);
  const auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  a = f32_bits(op(bits_f32(r[0]), bits_f32(r[1])));
  const auto s = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  return op(bits_f32(s[0]), bits_f32(s[1]));
}
__device__ inline float group_max(float x) {
  return over_groups(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ inline float group_sum(float x) {
  return over_groups(x, [](float a, float b) { return a + b; });
}

__device__ inline pa_u32x4 load16(const void* p) { return *reinterpret_cast<const pa_u32x4*>(p); }

__device__ inline void mfma16(pa_f32x4& acc, pa_u32x4 a, pa_u32x4 b) {
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pa_bf16x8, a), __builtin_bit_cast(pa_bf16x8, b), acc,
                                                0, 0, 0);
}
__device__ inline void mfma16_f32(pa_f32x4& acc, float a, float b) {
  acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, acc, 0, 0, 0);
}

// 4 codes (a dword), times s, as fp32
__device__ inline pa_u32x4 codes_f32(uint32_t w, float s) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  pa_u32x4 r;
  r[0] = f32_bits(lo[0] * s);
  r[1] = f32_bits(lo[1] * s);
  r[2] = f32_bits(hi[0] * s);
  r[3] = f32_bits(hi[1] * s);
  return r;
}

// What a part with maximum m and sum l weighs where the largest maximum is `top`: nothing if it
// has seen nothing, and NaN stays.
__device__ inline float weight_of(float m, float l, float top) {
  return m == -__builtin_inff() ? (l == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(m - top);
}

// One wave's tile.  Q: uint16_t (bf16 products) or float (fp32 products); Cd: whether the
// cache holds codes.  KD: the head dim the registers are laid out for, K <= KD the one there
// is (Full: K == KD).
template <typename Q, bool Cd, int KD, bool Full>
struct Tile {
  static constexpr bool kBf = sizeof(Q) == 2;
  static constexpr int kHeld = Cd ? 1 : (int)sizeof(Q);  // bytes of a held value
  static constexpr int KG = 16 / kHeld;                  // dims, or keys, of a 16-byte load
  static constexpr int KT = 4 * KG;                      // keys
  static constexpr int NT = KG / 4;                      // products of scores
  static constexpr int NC = KD / KT;                     // key loads of a lane and product
  static constexpr int NS = KG / (kBf ? 8 : 4) * NC;     // operands of those (8 bf16 or 4 fp32 dims each)
  static constexpr int ND = KD / 16;                     // rows of 16 dims of V^T
  pa_u32x4 k[NT][NC], v[ND];
  pa_u32x4 ks, vs;  // exponent bytes: of the lane's key group's rows, of its value keys

  // dims of key load c in lane group g
  __device__ static inline int dim_of(int c, int g) { return (4 * c + g) * KG; }

  __device__ inline void load_k(const PagedArgs& p, int64_t tile, int off, int lane) {
    const int i = lane & 15, g = lane >> 4, ps = p.a.shift;
    const char* base = (const char*)p.k + (((tile << ps) + off + (i & 3)) * p.K) * kHeld;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int d = dim_of(c, g);
        const bool in = Full || d < p.K;
        k[t][c] = load16(base + (4 * t * p.K + (in ? d : 0)) * kHeld);
        if constexpr (!Full)
          if (!in) k[t][c] = pa_u32x4{0, 0, 0, 0};
      }
    if constexpr (Cd) ks = load16(p.k_scale + (tile << ps) + off);
  }
  __device__ inline void load_v(const PagedArgs& p, int64_t tile, int off, int lane) {
    const int ps = p.a.shift;
    const char* at = (const char*)p.v + (((tile * p.K + (lane & 15)) << ps) + off) * kHeld;
    int64_t step = (int64_t)(16 * kHeld) << ps;
    if constexpr (Full) asm volatile("" : "+s"(step));  // (one address a row of loads, not ND kept)
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) {
      if constexpr (Full) v[dt] = load16(at);
      else v[dt] = load16(at - (dt * 16 + (lane & 15) < p.K ? 0 : (int64_t)((dt * 16 + (lane & 15)) * kHeld) << ps));
      at += step;
    }
    if constexpr (Cd) vs = load16(p.v_scale + (tile << ps) + off);
  }
};

// A block: the rows of one unit and key head against one piece of its keys, the
// tiles dealt out to its waves.
constexpr int few_waves(int QT) { return QT == 1 ? kWavesOf16 : 4; }
template <typename Q, bool Cd, int KD, bool Full, int QT>
__global__ __launch_bounds__(64 * few_waves(QT), QT == 1 ? (KD == 64 ? 3 : 2) : (KD == 64 ? 2 : 1)) void paged_few_kernel(PagedArgs p) {
  using TileT = Tile<Q, Cd, KD, Full>;
  constexpr bool kBf = TileT::kBf;
  constexpr int R = 16 * QT, ND = TileT::ND, NS = TileT::NS, NT = TileT::NT, KG = TileT::KG, KT = TileT::KT;
  constexpr int NW = few_waves(QT), kPitch = KD + 4;  // waves; floats of a row's output in LDS
  __shared__ __attribute__((aligned(16))) float merged[NW][R][kPitch];
  __shared__ float stat_m[NW][R], stat_l[NW][R];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4;
  const int item = blockIdx.x / p.Hk, kh = blockIdx.x % p.Hk, G = p.G, K = p.K;

  // rows of no sequence, read now and cleared last
  const int rest0 = p.zero_rest ? p.a.query_start[0] : 0, rest1 = p.zero_rest ? p.a.query_start[p.a.S] : 0x7fffffff;
  auto clear_rest = [&] {
    const int first = min(max(rest0, 0), p.a.T), end = min(max(rest1, first), p.a.T);
    const int rest = p.a.T - (end - first), items = gridDim.x / p.Hk;
    for (int r = item; r < rest; r += items) {
      Q* row = (Q*)p.o + ((int64_t)(r < first ? r : end + r - first) * p.H + kh * G) * K;
      for (int d = tid; d < G * K; d += 64 * NW) row[d] = from_f32<Q>(0.f);
    }
  };
  Item w;
  if (!find_item<R>(p, item, w)) {
    clear_rest();
    return;
  }
  const SeqRows r = w.r;
  const int seq = w.seq, row0 = w.row0, rows = w.rows, seen = w.seen, least = w.least;
  const int t0 = w.t0 * (kTile / KT), t1 = min(w.t1 * (kTile / KT), (seen + KT - 1) / KT);

  // Q^T operands, and how many keys the lane's rows see
  pa_u32x4 qf[QT][NS];
  int vis[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int m = qt * 16 + i, row = row0 + min(m, rows - 1);
    const int token = row / G, head = kh * G + row % G;
    vis[qt] = m < rows ? max(0, r.len - r.n + token + 1) : 0;
    const Q* at = (const Q*)p.q + ((int64_t)(r.first + token) * p.H + head) * K;
#pragma unroll
    for (int c = 0; c < TileT::NC; ++c)
#pragma unroll
      for (int j = 0; j < NS / TileT::NC; ++j) {
        const int d = TileT::dim_of(c, g) + j * (kBf ? 8 : 4);
        const bool in = Full || d < K;
        pa_u32x4 x = load16(at + (in ? d : 0));
        if (!in) x = pa_u32x4{0, 0, 0, 0};
        qf[qt][c * (NS / TileT::NC) + j] = x;
      }
  }

  pa_f32x4 acc[QT][ND];
  float m_run[QT], l_run[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    m_run[qt] = -__builtin_inff();
    l_run[qt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) acc[qt][dt] = pa_f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // The pages of a tile's four groups of keys: the lane's key rows are in group
  // i / 4, its value keys in group g.  Groups past the last key seen take the first.
  struct Ids { int k, v; };
  struct Place { int64_t k, v; int ko, vo; bool bad; };
  const int in_mask = (1 << p.a.shift) - 1;
  const int* table = p.a.table + (int64_t)seq * p.a.P;
  auto ids_of = [&](int tile) __attribute__((always_inline)) {
    const int pk = tile * KT + (i >> 2) * KG, pv = tile * KT + g * KG;
    return Ids{table[(pk < seen ? pk : 0) >> p.a.shift], table[(pv < seen ? pv : 0) >> p.a.shift]};
  };
  auto place = [&](int tile, Ids id) __attribute__((always_inline)) {
    Place w;
    const int pk = tile * KT + (i >> 2) * KG, pv = tile * KT + g * KG;
    const bool bad_k = (unsigned)id.k >= (unsigned)p.a.n_pages, bad_v = (unsigned)id.v >= (unsigned)p.a.n_pages;
    w.k = (int64_t)(bad_k ? 0 : id.k) * p.Hk + kh;
    w.v = (int64_t)(bad_v ? 0 : id.v) * p.Hk + kh;
    w.ko = pk & in_mask;
    w.vo = pv & in_mask;
    w.bad = bad_v && pv < seen;
    return w;
  };

  TileT x;
  Place here;
  // One tile: scores, running maximum and sum, P V.  Edge: some row does not see some key of
  // it.  `between` runs once the keys are used.
  auto step = [&](int tile, auto edge_t, auto between) __attribute__((always_inline)) {
    constexpr bool edge = decltype(edge_t)::value;
    const int key0 = tile * KT + g * KG;  // the lane's first key
    // scores
    pa_f32x4 s[QT][NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) s[qt][t] = pa_f32x4{0.f, 0.f, 0.f, 0.f};
      const float sc = Cd ? byte_scale(x.ks[t], i & 3) : 1.f;
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        pa_u32x4 kf;
        if constexpr (Cd && kBf) {
          const uint2 a = codes_bf16(x.k[t][n / 2][2 * (n % 2)], sc), b = codes_bf16(x.k[t][n / 2][2 * (n % 2) + 1], sc);
          kf[0] = a.x, kf[1] = a.y, kf[2] = b.x, kf[3] = b.y;
        } else if constexpr (Cd) {
          kf = codes_f32(x.k[t][n / 4][n % 4], sc);
        } else {
          kf = x.k[t][n];
        }
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          if constexpr (kBf) {
            mfma16(s[qt][t], kf, qf[qt][n]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) mfma16_f32(s[qt][t], bits_f32(kf[e]), bits_f32(qf[qt][n][e]));
          }
        }
      }
    }
    between();
    if (__any(here.bad)) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[qt][t][e] = here.bad ? __builtin_nanf("") : s[qt][t][e];
    }
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      if constexpr (edge) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key0 + 4 * t + e >= vis[qt]) s[qt][t][e] = -__builtin_inff();
      }
      float mx = s[qt][0][0];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[qt][t][e]);
      mx = group_max(mx) * p.scale_log2;
      // the maximum moves only when it grows by more than 8 (base 2): probabilities
      // stay below 2^8, and most tiles leave the accumulators alone
      const bool grow = mx > m_run[qt] + 8.f;
      if (__any(grow)) {
        const float m_new = grow ? mx : m_run[qt];
        const float alpha = grow ? __builtin_amdgcn_exp2f(m_run[qt] - m_new) : 1.f;
        l_run[qt] *= alpha;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) acc[qt][dt] *= alpha;
        m_run[qt] = m_new;
      }
      const float m_use = m_run[qt] == -__builtin_inff() ? 0.f : m_run[qt];  // (nothing seen yet)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[qt][t][e], p.scale_log2, -m_use));
          s[qt][t][e] = pr;
          l_run[qt] += pr;
        }
    }
    // Where a row does not look there may be anything, and 0 times an infinity or NaN is
    // NaN.  Slots past the last key seen may hold what was there before: codes and
    // exponents of those are cleared.  In a cache of the rows' own type a key that only
    // some of the rows see may also be infinite or NaN (codes never are).
    [[maybe_unused]] bool poison = false;
    if constexpr (edge) {
      if constexpr (Cd) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int there = min(max(seen - key0 - 4 * t, 0), 4);
          const uint32_t mask = there == 4 ? ~0u : (1u << (8 * there)) - 1u;
          x.vs[t] &= mask;
#pragma unroll
          for (int dt = 0; dt < ND; ++dt) x.v[dt][t] &= mask;
        }
      } else {
        constexpr uint32_t top = kBf ? 0x7f80u : 0x7f800000u;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t w = x.v[dt][e];
            poison |= (w & top) == top;
            if constexpr (kBf) poison |= (w & (top << 16)) == (top << 16);
          }
      }
    }
    if constexpr (edge && !Cd) {
      if (__any(poison)) {  // those values' products one by one, to the rows that see them; 0 in their place below
        for (int key = 0; key < KT && tile * KT + key < seen; ++key) {
          const int from = key / KG * 16;
          const int64_t pool = __shfl(here.v, from, 64);
          const Q* at = (const Q*)p.v + ((pool * K) << p.a.shift) + __shfl(here.vo, from, 64) + key % KG;
          int first_d = g * 4;
          asm volatile("" : "+v"(first_d));  // (nothing of the addresses is kept over the loop)
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) {
            float pr = 0.f;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (key % KG == 4 * t + e) pr = s[qt][t][e];
            pr = __shfl(pr, from + i, 64);
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) {
              __builtin_amdgcn_sched_barrier(0);  // (few registers: the path above wants them)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int d = dt * 16 + first_d + e;
                const float f = to_f32(at[(int64_t)(Full || d < K ? d : 0) << p.a.shift]);
                if (tile * KT + key < vis[qt] && !(fabsf(f) < __builtin_inff())) acc[qt][dt][e] += pr * f;
              }
            }
          }
        }
#pragma unroll
        for (int dt = 0; dt < ND; ++dt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t w = x.v[dt][e];
            if constexpr (kBf) {
              if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
              if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
            } else if ((w & 0x7f800000u) == 0x7f800000u) {
              w = 0;
            }
            x.v[dt][e] = w;
          }
      }
    }
    if constexpr (kBf) {
#pragma unroll
      for (int h = 0; h < KG / 8; ++h) {
        pa_u32x4 pf[QT];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          float w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            w[e] = s[qt][2 * h + e / 4][e % 4];
            if constexpr (Cd) w[e] *= byte_scale(x.vs[2 * h + e / 4], e % 4);  // exact: a power of two
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) pf[qt][e] = pack_bf16x2(w[2 * e], w[2 * e + 1]);
        }
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) {
          pa_u32x4 vf;
          if constexpr (Cd) {
            const uint2 a = codes_bf16(x.v[dt][2 * h], 1.f), b = codes_bf16(x.v[dt][2 * h + 1], 1.f);
            vf[0] = a.x, vf[1] = a.y, vf[2] = b.x, vf[3] = b.y;
          } else {
            vf = x.v[dt];
          }
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) mfma16(acc[qt][dt], vf, pf[qt]);
        }
      }
    } else {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if constexpr (Cd) {
#pragma unroll
          for (int qt = 0; qt < QT; ++qt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[qt][t][e] *= byte_scale(x.vs[t], e);
        }
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) {
          pa_u32x4 vf;
          if constexpr (Cd) vf = codes_f32(x.v[dt][t], 1.f);
          else vf = x.v[dt];
#pragma unroll
          for (int qt = 0; qt < QT; ++qt)
#pragma unroll
            for (int e = 0; e < 4; ++e) mfma16_f32(acc[qt][dt], bits_f32(vf[e]), s[qt][t][e]);
        }
      }
    }
  };

  // (page numbers are read two tiles ahead, as the loads of a tile wait for them)
  int tile = t0 + wave;
  if (tile < t1) {
    Ids then = ids_of(min(tile + NW, t1 - 1));
    here = place(tile, ids_of(tile));
    x.load_k(p, here.k, here.ko, lane);
    x.load_v(p, here.v, here.vo, lane);
    // every row sees all of these: the next tile's keys are on their way while this one's
    // scores are weighed, its values while the next one's scores are formed
    while (tile * KT + KT <= least) {
      const bool more = tile + NW < t1;
      const Place next = place(tile + NW, then);
      then = ids_of(min(tile + 2 * NW, t1 - 1));
      step(tile, std::false_type{}, [&]() __attribute__((always_inline)) {
        if (more) x.load_k(p, next.k, next.ko, lane);
      });
      if (more) x.load_v(p, next.v, next.vo, lane);
      here = next;
      tile += NW;
      if (!more) break;
    }
    // the others, one at a time: their masks cost registers that the loop above would lack
    while (tile < t1) {
      step(tile, std::true_type{}, [] {});
      tile += NW;
      if (tile < t1) {
        here = place(tile, then);
        then = ids_of(min(tile + NW, t1 - 1));
        x.load_k(p, here.k, here.ko, lane);
        x.load_v(p, here.v, here.vo, lane);
      }
    }
  }

  // the waves' parts, joined in their order
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const float l = group_sum(l_run[qt]);
    if (g == 0) {
      stat_m[wave][qt * 16 + i] = m_run[qt];
      stat_l[wave][qt * 16 + i] = l;
    }
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
      *reinterpret_cast<pa_f32x4*>(&merged[wave][qt * 16 + i][dt * 16 + g * 4]) = acc[qt][dt];
  }
  __syncthreads();
  float* part = p.part + (int64_t)blockIdx.x * R * (K + 2);
  for (int e = tid; e < rows * (K / 4); e += 64 * NW) {
    const int m = e / (K / 4), d = e % (K / 4) * 4;
    float top = stat_m[0][m];
#pragma unroll
    for (int v = 1; v < NW; ++v) top = fmaxf(top, stat_m[v][m]);
    float l = 0.f;
    pa_f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NW; ++v) {
      const float f = weight_of(stat_m[v][m], stat_l[v][m], top);
      l += f * stat_l[v][m];
      o += f * *reinterpret_cast<const pa_f32x4*>(&merged[v][m][d]);
    }
    if (w.split > 1) {
      *reinterpret_cast<pa_f32x4*>(part + (int64_t)m * K + d) = o;
      if (d == 0) {
        part[R * K + m] = top;
        part[R * K + R + m] = l;
      }
    } else {
      store_row4<Q>(p, r, kh, row0 + m, d, o, l);
    }
  }
  clear_rest();
}

// Joins the pieces of the units that were cut, K / 4 lanes to a row of a piece.  blockIdx: unit
// and key head, and the first of the block's rows.  (With one thread for all the pieces of its
// four dims a row of 128 pieces took 100 us, with one wave 19.)
template <typename Q, int R>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, K = p.K, lanes = K / 4;
  const int b = blockIdx.x / p.Hk, kh = blockIdx.x % p.Hk;
  const SeqScan scan(p.a);
  const int chunk = piece_tiles<R>(p, scan);
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
  __shared__ float wave_top[4], wave_l[4];
  __shared__ __attribute__((aligned(16))) float wave_o[4][128];
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
    if (sub == 0) *reinterpret_cast<pa_f32x4*>(&wave_o[wave][d]) = sum;
    if (lane == 0) wave_top[wave] = top, wave_l[wave] = l;
    __syncthreads();
    if (threadIdx.x < lanes) {
      float all = wave_top[0];
#pragma unroll
      for (int v = 1; v < 4; ++v) all = fmaxf(all, wave_top[v]);
      l = 0.f, o = pa_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float f = weight_of(wave_top[v], wave_l[v], all);
        l += f * wave_l[v];
        if (f != 0.f) o += f * *reinterpret_cast<const pa_f32x4*>(&wave_o[v][d]);
      }
      store_row4<Q>(p, r, kh, local * R + m, d, o, l);
    }
    __syncthreads();
  }
}

// A launch, as it is sized on the host.
struct Part {
  int R;          // rows of a unit, 0: no launch
  int over, upto; // the sequences it takes, by their rows of a key head
  int target, least;  // pieces, and tiles of one at least
  int64_t units, items;  // at most
  bool cuts;      // whether a unit can be cut
  int64_t floats(int64_t Hk, int64_t K) const { return cuts ? items * Hk * R * (K + 2) : 0; }
};

// A launch of the sequences with at most 16 or 32 rows of a key head, and, where there may be
// others that it serves better, one of paged_chunk.hip's kernel.
struct Plan {
  Part few, many;
};

Part part_of(int R, int64_t over, int64_t upto, int target, int least, int64_t T, int64_t S, int64_t P, int64_t page_size, int64_t G,
             int64_t Hk) {
  Part n;
  n.R = R, n.over = (int)over, n.upto = (int)upto, n.target = target, n.least = least;
  // a sequence of this launch has more than `over` rows; at most R of them are one unit
  const int64_t seqs = std::min(std::min(S, T), T * G / (over + 1) + (over == 0 ? T : 0));
  n.units = upto <= R ? seqs : std::min(T * G, T * G / R + seqs);
  const int64_t tiles = (P * page_size + kTile - 1) / kTile, most = (tiles + least - 1) / least;
  n.cuts = most > 1;
  n.items = std::min(n.units * most, n.units + (target + Hk - 1) / Hk);
  return n;
}

Plan plan_of(int64_t T, int64_t S, int64_t P, int64_t page_size, int64_t G, int64_t Hk, int64_t K, int dtype,
             int held, int64_t max_new) {
  constexpr int64_t kAll = 0x7fffffff;
  const int64_t rows = std::min(T, max_new) * G;
  // a piece of a quarter of a megabyte, 256 to 1024 keys: less and its block's beginning and the
  // join take longer than its keys (700 bf16 tokens in one piece 9 us, in two 14)
  const int64_t tile = 2 * kTile * K * (held == ABACUS_E4M3 ? 1 : held == kBF16 ? 2 : 4);
  const int least = (int)std::min<int64_t>(std::max<int64_t>((256 << 10) / tile, 4), 16);
  const bool chunks = dtype == kBF16;
  Plan n;
  n.many.R = 0, n.many.cuts = false;
  if (rows <= 32 || !chunks) {
    n.few = part_of(rows <= 16 ? 16 : 32, 0, kAll, kFewPieces, least, T, S, P, page_size, G, Hk);
  } else {
    const int few = G <= 16 ? 16 : 32;
    n.few = part_of(few, 0, few, kFewPieces, least, T, S, P, page_size, G, Hk);
    n.many = part_of(kChunkRows, few, kAll, kChunkPieces, 16, T, S, P, page_size, G, Hk);
  }
  return n;
}

template <typename Q, bool Cd, int QT>
void launch_few(const PagedArgs& p, unsigned blocks, hipStream_t s) {
  if (p.K == 64) hipLaunchKernelGGL((paged_few_kernel<Q, Cd, 64, true, QT>), dim3(blocks), dim3(64 * few_waves(QT)), 0, s, p);
  else if (p.K == 128) hipLaunchKernelGGL((paged_few_kernel<Q, Cd, 128, true, QT>), dim3(blocks), dim3(64 * few_waves(QT)), 0, s, p);
  else if (p.K < 64) hipLaunchKernelGGL((paged_few_kernel<Q, Cd, 64, false, QT>), dim3(blocks), dim3(64 * few_waves(QT)), 0, s, p);
  else hipLaunchKernelGGL((paged_few_kernel<Q, Cd, 128, false, QT>), dim3(blocks), dim3(64 * few_waves(QT)), 0, s, p);
}

template <typename Q>
int launch(PagedArgs p, const Plan& n, bool codes, float* ws, int64_t rows, hipStream_t s) {
  auto set = [&](const Part& part, float* at) {
    p.over = part.over, p.upto = part.upto, p.target = part.target, p.least = part.least, p.part = at;
    return (unsigned)(part.items * p.Hk);
  };
  auto join_grid = [&](const Part& part) {
    const int64_t at_once = std::min<int64_t>(std::min<int64_t>(part.R, rows), 16);
    return dim3((unsigned)(part.units * p.Hk), (unsigned)(part.units * p.Hk < 128 ? at_once : (at_once + 3) / 4));
  };
  const unsigned blocks = set(n.few, ws);
  if (n.few.R == 16) codes ? launch_few<Q, true, 1>(p, blocks, s) : launch_few<Q, false, 1>(p, blocks, s);
  else codes ? launch_few<Q, true, 2>(p, blocks, s) : launch_few<Q, false, 2>(p, blocks, s);
  ABACUS_CHECK_LAUNCH("paged_attention");
  if (n.few.cuts) {
    if (n.few.R == 16) hipLaunchKernelGGL((paged_join_kernel<Q, 16>), join_grid(n.few), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((paged_join_kernel<Q, 32>), join_grid(n.few), dim3(256), 0, s, p);
    ABACUS_CHECK_LAUNCH("paged_attention (join)");
  }
  if (n.many.R == 0) return 0;
  p.zero_rest = 0;
  const unsigned chunks = set(n.many, ws + n.few.floats(p.Hk, p.K));
  if (launch_chunk(p, chunks, codes, s)) return 2;
  if (n.many.cuts) {
    hipLaunchKernelGGL((paged_join_kernel<Q, kChunkRows>), join_grid(n.many), dim3(256), 0, s, p);
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
  ABACUS_CHECK_ARG(n.few.items * Hk < (1ll << 31), "paged_attention: %lld rows of %lld heads are too many", (long long)T,
                   (long long)H);
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
