// Attention of few rows over a paged cache (16 or 32 of a key head in a work-group): a step's
// single tokens, drafted ones, and all fp32 rows.  Work and its cut: paged_cut.h.
//
// In registers (v_mfma_f32_16x16x32_bf16: lane l gives A[l % 16][8 (l / 16) .. +7] and
// B[8 (l / 16) .. +7][l % 16], and holds D[4 (l / 16) + r][l % 16] in register r; the fp32
// product takes one element of each per lane): a wave's tile is four groups of KG keys, as
// many as 16 bytes of values hold (16 codes, 8 bf16, 4 fp32).  S^T = K Q^T takes them in KG / 4
// products t whose row i is key KG (i / 4) + 4 t + i % 4.  Lane l then holds the scores of
// query l % 16 against the KG keys of group l / 16, in their order, and those are, as they
// lie, the operand P^T of O^T = V^T P^T with 16 bytes of a V^T row: neither the scores nor a
// tile of keys or values goes through LDS, and every load of the cache is 16 bytes a lane.
//
// Bound by the bytes of the cache.  4 query heads a key head, K = 128: 64 tokens over up to 8192
// e4m3 keys 133 us (5.3 TB/s; the vector unit is busy a quarter of it), 2 over
// 131072 bf16 keys 193 us (5.6 TB/s).  The tiles of a block's piece are dealt out to its four
// waves in turn: runs of tiles a wave took 230 us for the first, eight waves 156.  With more
// than 16 rows the fp32 products weigh as much (97 TF/s of 154 for a chunk of K = 128).
#pragma once

#include <type_traits>

#include "paged_cut.h"

namespace abacus {

typedef __bf16 pa_bf16x8 __attribute__((ext_vector_type(8)));
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

constexpr int kFewWaves = 4;
// The waves' parts of a block's rows.
template <int KD, int QT>
struct FewLds {
  float merged[kFewWaves][16 * QT][KD + 4];
  float stat_m[kFewWaves][16 * QT], stat_l[kFewWaves][16 * QT];
};

// Block `block` of `blocks`: the rows of one unit and key head against one piece of its keys,
// the tiles dealt out to its waves.
template <typename Q, bool Cd, int KD, bool Full, int QT>
__device__ __attribute__((always_inline)) inline void few_block(const PagedArgs& p, int block, int blocks,
                                                                FewLds<KD, QT>& lds) {
  using TileT = Tile<Q, Cd, KD, Full>;
  constexpr bool kBf = TileT::kBf;
  constexpr int R = 16 * QT, ND = TileT::ND, NS = TileT::NS, NT = TileT::NT, KG = TileT::KG, KT = TileT::KT;
  constexpr int NW = kFewWaves;
  auto& merged = lds.merged;
  auto& stat_m = lds.stat_m;
  auto& stat_l = lds.stat_l;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4;
  const int item = block / p.Hk, kh = block % p.Hk, G = p.G, K = p.K;

  Item w;
  // Rows of no sequence, cleared last: those before and behind the rows that the scan gives the
  // sequences, which no block stores.  (The last entry of query_start does not say where those
  // end: it may lie behind a range that runs backwards or past the call's rows.)
  const int start = p.zero_rest ? p.a.query_start[0] : 0;  // read now
  auto clear_rest = [&] {
    if (!p.zero_rest) return;
    const int rest = p.a.T - w.given, items = blocks / p.Hk;
    for (int r = item; r < rest; r += items) {  // (no sequence has a row: any start will do)
      const int at = w.given > 0 && r >= start ? r + w.given : r;
      Q* row = (Q*)p.o + ((int64_t)at * p.H + kh * G) * K;
      for (int d = tid; d < G * K; d += 64 * NW) row[d] = from_f32<Q>(0.f);
    }
  };
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
        pa_u32x4 pf[QT];  // probabilities in bf16, as in paged_chunk.h; fp32 rows keep theirs
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
  float* part = p.part + (int64_t)block * R * (K + 2);
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

}  // namespace abacus
