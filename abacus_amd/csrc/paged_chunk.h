// Attention of a chunk of new tokens over a paged cache: bf16 queries, a cache in bf16 or
// e4m3.  Work and its cut: paged_cut.h.  The tiles are laid out for head dim 64 or 128 (HD);
// another one (K < HD, not Full) leaves their last dims 0, which are cleared once and not
// loaded after.
//
// A work-group has 128 rows (token, query head) of one key head, 32 to a wave, and walks
// its piece's 64-key tiles with a running maximum and sum in fp32.  A tile of K and of V^T
// lies in LDS for the four waves, the next one is under way while it is used: bf16 pages
// by DMA straight into the other stage, codes through registers, where they become bf16 on
// the way (keys times their exponents, which is exact; the values' exponents go to the
// probabilities, as neighbours in a V^T row have different ones).
//
// S^T = K Q^T in v_mfma_f32_32x32x16_bf16, row i of a product being key i with bits 2 and 3
// exchanged: lane l then holds, of query l % 32, the scores against keys 16 c + 8 (l / 32)
// + 0..7 in registers 8 c .. 8 c + 7, which is the operand P^T of O^T = V^T P^T as it lies.
//
// Bound by the products and the exponentials together: two chunks of 2048 tokens over 8192 (32
// heads over 8, K = 128) take 667 us, 930 TF/s, in a long row of calls, the matrix unit busy 0.40
// of the 1.46 million cycles, the vector unit 0.46.  The clock decides: the first 20 calls after a
// pause take 716 to 850 us, calls among others with their join 650 to 720.  K = 64, where the
// products are half as much, 610 TF/s; codes 790.  Two work-groups a CU hide a tile's loads, so two
// stages are enough; the next tile's scores formed under this one's exponentials won nothing
// (705 to 712 against 717 us) and spilled.
#pragma once

#include <type_traits>

#include "attention_tiles.h"
#include "paged_cut.h"

namespace abacus {

constexpr int kChunkStages = 2;

template <int HD>
struct ChunkLds {
  char k[kChunkStages][kTile * HD * 2];
  char v[kChunkStages][HD * kTile * 2];
  float vs[kChunkStages][kTile];  // what the value codes of a key are to be multiplied by
};

// The pages of a tile's four 16-key groups, the same for the whole block.
struct Groups {
  int page[4];
  int bad;  // bit per group that lies in no page
};

__device__ inline Groups groups_of(const PagedArgs& p, int seq, int key0, int seen) {
  Groups g;
  g.bad = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int pos = key0 + 16 * j < seen ? key0 + 16 * j : 0;  // (past the last key seen: any page that exists)
    bool bad;
    g.page[j] = __builtin_amdgcn_readfirstlane(page_of(p.a, seq, pos, bad));
    if (__builtin_amdgcn_readfirstlane(bad)) g.bad |= 1 << j;
  }
  return g;
}

template <class T>
__device__ inline T pick(const T (&x)[4], int j) {
  const T a = j & 1 ? x[1] : x[0], b = j & 1 ? x[3] : x[2];
  return j & 2 ? b : a;
}

// bf16 pages: 16 bytes a lane and instruction, straight into the swizzled tile.
template <int HD, bool Full>
__device__ inline void dma_tile(const PagedArgs& p, int kh, const Groups& g, int key0, char* kt, char* vt) {
  constexpr int CH = HD / 8;  // chunks of a key row
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), ps = p.a.shift;
  const int K = Full ? HD : p.K;
  const int in_page = (1 << ps) - 1;  // group j's slots begin at (key0 + 16 j) & in_page
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) {
    const int at = i * 256 + tid, row = at / CH, j = HD == 128 ? i : 2 * i + (wave >> 1);  // the row's group
    const int64_t slot = (((int64_t)pick(g.page, j) * p.Hk + kh) << ps) + ((key0 + 16 * j) & in_page) + (row & 15);
    const int c = (at % CH) ^ tile_swz<HD>(row);
    if (Full || c * 8 < K) dma16((const uint16_t*)p.k + slot * K + c * 8, kt + (i * 4 + wave) * 1024);
  }
  const int d0 = tid / 8, c = (tid % 8) ^ tile_swz<64>(d0);  // V^T rows d0 + 32 i: the swizzle is the same for all
  const int64_t page = (int64_t)pick(g.page, c >> 1) * p.Hk + kh;
  const uint16_t* from = (const uint16_t*)p.v + ((page * K + d0) << ps) + ((key0 + 8 * c) & in_page);
#pragma unroll
  for (int i = 0; i < HD / 32; ++i)
    if (Full || d0 + 32 * i < K) dma16(from + ((int64_t)(32 * i) << ps), vt + (i * 4 + wave) * 1024);
}

// Codes: loaded while the tile before is used, made bf16 and stored after it.
template <int HD, bool Full>
struct Codes {
  static constexpr int N = HD / 64;  // 16-byte loads of a thread, of keys and of values
  typedef uint32_t U4 __attribute__((ext_vector_type(4)));
  U4 k[N], v[N];
  int ks[N];
  U4 vs;
  __device__ inline void load(const PagedArgs& p, int kh, const Groups& g, int key0) {
    const int tid = threadIdx.x, ps = p.a.shift, in_page = (1 << ps) - 1, K = Full ? HD : p.K;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = (i * 256 + tid) / (HD / 16), c = tid % (HD / 16);
      const int64_t slot = (((int64_t)pick(g.page, row >> 4) * p.Hk + kh) << ps) + ((key0 + row) & in_page);
      k[i] = *reinterpret_cast<const U4*>((const uint8_t*)p.k + slot * K + (Full || c * 16 < K ? c * 16 : 0));
      ks[i] = p.k_scale[slot];
      const int d = (i * 256 + tid) / 4, j = tid & 3;
      const int64_t page = (int64_t)pick(g.page, j) * p.Hk + kh;
      v[i] = *reinterpret_cast<const U4*>((const uint8_t*)p.v + ((page * K + (Full || d < K ? d : 0)) << ps) +
                                           ((key0 + 16 * j) & in_page));
      if (i == 0) vs = *reinterpret_cast<const U4*>(p.v_scale + (page << ps) + ((key0 + 16 * j) & in_page));
    }
  }
  // `left`: keys of the tile that exist (past them there may be anything in V: 0)
  __device__ inline void store(char* kt, char* vt, float* scales, int left, int K) {
    const int tid = threadIdx.x;
    if (left < kTile) {
      const int j = tid & 3;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int there = min(max(left - 16 * j - 4 * e, 0), 4);
        const uint32_t mask = there == 4 ? ~0u : (1u << (8 * there)) - 1u;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i][e] &= mask;
        vs[e] &= mask;
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = (i * 256 + tid) / (HD / 16), c = tid % (HD / 16), d = (i * 256 + tid) / 4, j = tid & 3;
      const float s = bits_f32((uint32_t)ks[i] << 23);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint2 a = codes_bf16(k[i][2 * h], s), b = codes_bf16(k[i][2 * h + 1], s);
        Vec16 w;
        w.w[0] = a.x, w.w[1] = a.y, w.w[2] = b.x, w.w[3] = b.y;
        if (Full || c * 16 < K) *reinterpret_cast<Vec16*>(kt + tile_off<HD>(row, 2 * c + h)) = w;
        const uint2 y = codes_bf16(v[i][2 * h], 1.f), z = codes_bf16(v[i][2 * h + 1], 1.f);
        w.w[0] = y.x, w.w[1] = y.y, w.w[2] = z.x, w.w[3] = z.y;
        if (Full || d < K) *reinterpret_cast<Vec16*>(vt + tile_off<64>(d, 2 * j + h)) = w;
      }
    }
    if (tid < 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<float4*>(scales + 16 * tid + 4 * e) = make_float4(byte_scale(vs[e], 0), byte_scale(vs[e], 1),
                                                                            byte_scale(vs[e], 2), byte_scale(vs[e], 3));
    }
  }
};

__device__ inline bool not_finite(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

// N: 32-key halves of a tile that a wave takes.  With 1 (at most 64 rows) waves 2 and 3 have the
// rows of 0 and 1 and the tiles' other halves, which are joined at the end.
template <bool Cd, int HD, bool Full, int N>
__device__ __attribute__((always_inline)) inline void chunk_rows(const PagedArgs& p, int block, const Item& w,
                                                                 ChunkLds<HD>& lds) {
  constexpr int R = kChunkRows;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int kh = block % p.Hk, G = p.G, K = Full ? HD : p.K;
  const int half = N == 1 ? wave >> 1 : 0;

  // this wave's rows, and the keys that the last of them sees
  const int m0 = (N == 1 ? wave & 1 : wave) * 32, m = m0 + (lane & 31);
  const int row = w.row0 + min(m, w.rows - 1);
  const int token = row / G, head = kh * G + row % G;
  const int vis = m < w.rows ? max(0, w.r.len - w.r.n + token + 1) : 0;
  const int seen = m0 < w.rows ? seen_of(w.r, w.row0 + min(m0 + 31, w.rows - 1), G) : 0;
  const uint16_t* at = (const uint16_t*)p.q + ((int64_t)(w.r.first + token) * p.H + head) * K;
  Vec16 qf[HD / 16];
#pragma unroll
  for (int c = 0; c < HD / 16; ++c) qf[c] = Full || 16 * c < K ? ld16(at + 16 * c + 8 * h) : zero16();

  attn_f32x16 acc[HD / 32];
#pragma unroll
  for (int t = 0; t < HD / 32; ++t) acc[t] = attn_f32x16{};
  float m_run = -__builtin_inff(), l_run = 0.f;
  const int key_row = (lane & 0x13) | (lane & 4) << 1 | (lane & 8) >> 1;  // bits 2 and 3 of l % 32 exchanged

  auto step = [&](const char* kt, const char* vt, const float* scales, int key0, int bad,
                  auto edge_t) __attribute__((always_inline)) {
    constexpr bool edge = decltype(edge_t)::value;
    attn_f32x16 s[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      s[n] = attn_f32x16{};
#pragma unroll
      for (int c = 0; c < HD / 16; ++c)
        mfma32(s[n], *reinterpret_cast<const Vec16*>(kt + tile_off<HD>(32 * (n + half) + key_row, 2 * c + h)), qf[c]);
    }
    if (bad) {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (bad >> (2 * (n + half) + r / 8) & 1) s[n][r] = __builtin_nanf("");
    }
    if constexpr (edge) {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (key0 + 32 * (n + half) + 16 * (r >> 3) + 8 * h + (r & 7) >= vis) s[n][r] = -__builtin_inff();
    }
    float mx = s[0][0];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[n][r]);
    mx = pair_max(mx) * p.scale_log2;
    // the maximum moves only when it grows by more than 8 (base 2)
    const bool grow = mx > m_run + 8.f;
    if (__any(grow)) {
      const float m_new = grow ? mx : m_run;
      const float alpha = grow ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.f;
      l_run *= alpha;
#pragma unroll
      for (int t = 0; t < HD / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] *= alpha;
      m_run = m_new;
    }
    const float m_use = m_run == -__builtin_inff() ? 0.f : m_run;  // (nothing seen yet)
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[n][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][r], p.scale_log2, -m_use));
        l_run += s[n][r];
      }
    // A cache in bf16 may hold infinities and NaN that a row does not see, and 0 times those
    // is NaN: their products one by one, to the rows that see them, and 0 in their place.
    [[maybe_unused]] bool poison = false;
    if constexpr (edge && !Cd) {
      for (int c = 0; c < HD / 8; ++c) {
        const Vec16 x = *reinterpret_cast<const Vec16*>(vt + (c * 64 + lane) * 16);
        for (int e = 0; e < 4; ++e) poison |= not_finite(x.w[e]);
      }
      poison = __any(poison);
      if (poison) {
#pragma unroll 1
        for (int key = 32 * half; key < 32 * (half + N); ++key) {
          float pr = 0.f;
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (32 * (n + half) + 16 * (r >> 3) + (r & 7) == (key & ~8)) pr = s[n][r];
          pr = __shfl(pr, (lane & 31) + 4 * (key & 8), 64);
          int first_d = 4 * h;
          asm volatile("" : "+v"(first_d));  // (nothing of the addresses is kept over the loop)
#pragma unroll
          for (int t = 0; t < HD / 32; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              __builtin_amdgcn_sched_barrier(0);
              const int d = 32 * t + 8 * (r >> 2) + first_d + (r & 3);
              const float f = to_f32(*reinterpret_cast<const uint16_t*>(vt + tile_off<64>(d, key >> 3) + 2 * (key & 7)));
              if (key0 + key < vis && !(fabsf(f) < __builtin_inff())) acc[t][r] += pr * f;
            }
        }
      }
    }
#pragma unroll
    for (int c = 0; c < 2 * N; ++c) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = s[c >> 1][8 * (c & 1) + e];
      if constexpr (Cd) {
        const float4 a = *reinterpret_cast<const float4*>(scales + 16 * (c + 2 * half) + 8 * h);
        const float4 b = *reinterpret_cast<const float4*>(scales + 16 * (c + 2 * half) + 8 * h + 4);
        const float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= f[e];  // exact: powers of two
      }
      // Rounded to bf16 for the product with the values, and summed unrounded: fp32 products run at
      // an eighth of the rate, and o's own rounding is as large (o is 0.0023 off the formula,
      // normwise, where its rounding alone is 0.0017).
      Vec16 pf;
#pragma unroll
      for (int e = 0; e < 4; ++e) pf.w[e] = pack_bf16x2(x[2 * e], x[2 * e + 1]);
#pragma unroll
      for (int t = 0; t < HD / 32; ++t) {
        Vec16 vf = *reinterpret_cast<const Vec16*>(vt + tile_off<64>(32 * t + (lane & 31), 2 * (c + 2 * half) + h));
        if constexpr (edge && !Cd) {
          if (poison) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if ((vf.w[e] & 0x7f80u) == 0x7f80u) vf.w[e] &= 0xffff0000u;
              if ((vf.w[e] & 0x7f800000u) == 0x7f800000u) vf.w[e] &= 0xffffu;
            }
          }
        }
        mfma32(acc[t], vf, pf);
      }
    }
  };

  // The ring: tile t is in stage t % 2; once it has landed everywhere (this thread's wait,
  // then the barrier, after which no wave still reads the other stage) the next is sent.
  if (w.t0 < w.t1) {
    if constexpr (!Full) {
      for (int i = tid; i < (int)sizeof(lds) / 16; i += 256) reinterpret_cast<Vec16*>(&lds)[i] = zero16();
      __syncthreads();
    }
    Groups next = groups_of(p, w.seq, w.t0 * kTile, w.seen);
    int bad = next.bad;
    [[maybe_unused]] Codes<HD, Full> codes;
    if constexpr (Cd) {
      codes.load(p, kh, next, w.t0 * kTile);
      codes.store(lds.k[0], lds.v[0], lds.vs[0], w.seen - w.t0 * kTile, K);
    } else {
      dma_tile<HD, Full>(p, kh, next, w.t0 * kTile, lds.k[0], lds.v[0]);
    }
    if (w.t0 + 1 < w.t1) next = groups_of(p, w.seq, (w.t0 + 1) * kTile, w.seen);
    auto turn = [&](int t, auto edge_t) __attribute__((always_inline)) {
      const int st = (t - w.t0) % kChunkStages, key0 = t * kTile;
      const bool more = t + 1 < w.t1;
      if constexpr (!Cd) wait_vmcnt<0>();
      __syncthreads();
      if (more) {
        if constexpr (Cd) codes.load(p, kh, next, key0 + kTile);
        else dma_tile<HD, Full>(p, kh, next, key0 + kTile, lds.k[st ^ 1], lds.v[st ^ 1]);
      }
      const int next_bad = next.bad;
      if (t + 2 < w.t1) next = groups_of(p, w.seq, key0 + 2 * kTile, w.seen);
      if (!decltype(edge_t)::value || key0 + 32 * half < seen) step(lds.k[st], lds.v[st], lds.vs[st], key0, bad, edge_t);
      if constexpr (Cd) {
        if (more) codes.store(lds.k[st ^ 1], lds.v[st ^ 1], lds.vs[st ^ 1], w.seen - key0 - kTile, K);
      }
      bad = next_bad;
    };
    // the tiles that every row sees whole, then the others (in a loop of their own: their
    // masks cost registers that the first would lack)
    int t = w.t0;
    for (; t < min(w.t1, w.least / kTile); ++t) turn(t, std::false_type{});
    for (; t < w.t1; ++t) turn(t, std::true_type{});
  }
  if constexpr (N == 1) {  // waves 2 and 3 hand over what they have
    constexpr int kAcc = HD / 2;  // of a lane
    static_assert(sizeof(ChunkLds<HD>) >= 2 * (kAcc + 2) * 64 * 4, "two waves' sums");
    float* to = reinterpret_cast<float*>(&lds) + (wave & 1) * (kAcc + 2) * 64 + lane;
    __syncthreads();
    if (wave >= 2) {
#pragma unroll
      for (int i = 0; i < kAcc; ++i) to[i * 64] = acc[i / 16][i % 16];
      to[kAcc * 64] = m_run, to[(kAcc + 1) * 64] = l_run;
    }
    __syncthreads();
    if (wave >= 2) return;
    const float other = to[kAcc * 64], top = fmaxf(m_run, other), from = top == -__builtin_inff() ? 0.f : top;
    const float a = __builtin_amdgcn_exp2f(m_run - from), b = __builtin_amdgcn_exp2f(other - from);
    m_run = top;
    l_run = a * l_run + b * to[(kAcc + 1) * 64];
#pragma unroll
    for (int i = 0; i < kAcc; ++i) acc[i / 16][i % 16] = a * acc[i / 16][i % 16] + b * to[i * 64];
  }
  if (m >= w.rows) return;
  const float l = pair_sum(l_run);
  float* part = p.part + (int64_t)block * R * (K + 2);
#pragma unroll
  for (int t = 0; t < HD / 32; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * t + 8 * g + 4 * h;
      if (!Full && d >= K) continue;
      const float o[4] = {acc[t][4 * g], acc[t][4 * g + 1], acc[t][4 * g + 2], acc[t][4 * g + 3]};
      if (w.split > 1) *reinterpret_cast<float4*>(part + m * K + d) = make_float4(o[0], o[1], o[2], o[3]);
      else store_row4<uint16_t>(p, w.r, kh, row, d, o, l);
    }
  if (w.split > 1 && h == 0) {
    part[R * K + m] = m_run;
    part[R * K + R + m] = l;
  }
}

template <bool Cd, int HD, bool Full>
__device__ __attribute__((always_inline)) inline void chunk_block(const PagedArgs& p, int block, ChunkLds<HD>& lds) {
  Item w;
  if (!find_item<kChunkRows>(p, block / p.Hk, w)) return;
  if (w.rows > kChunkRows / 2) chunk_rows<Cd, HD, Full, 2>(p, block, w, lds);
  else chunk_rows<Cd, HD, Full, 1>(p, block, w, lds);
}

}  // namespace abacus
