// The residual stream between two blocks of the decoder, forward and backward: a block's output, through a norm of its
// own and a gate where it has them, is added to the stream, and the next block's norm is taken of the sum.
//
//   b = y                                  or  post * y * p,  p = 1 / sqrt(mean(y^2) + eps)
//   r = x + scale * gate * b               (rounded to the tensors' type)
//   h = gamma * r * q,  q = 1 / sqrt(mean(r^2) + eps), of r as it is stored
//
//   n = r q, g = dh gamma;   dr' = dr + q (g - n mean(g n)),   dx = dr',   dgamma = sum over rows of dh n
//   db = scale gate dr',     dgate = scale dr' b (summed over rows for a gate a channel)
//   dy = db                  or  p (post db - m mean(post db m)),  m = y p,   dpost = sum over rows of db m
//
// The reference has the plain form as two steps, x + attention (transformer_block.py:98-100) and RMSNorm
// (norm.py:26-31); without post, gate and scale r and h have the bits of those two.  Each way is one pass:
// everything but the outputs' rounding is fp32.
//
// Layout: a lane holds VPL vectors of 16 bytes of a row, which is spread over
//   kEven    lpr lanes of a wave that its vectors divide evenly (the RMSNorm kernels' layout, so the same sums),
//   kWave    the 64 lanes of a wave,
//   kGroup   the waves of a work-group: long rows, whose vectors and sums would crowd a lane's registers.
// Rows may start at any element.  Where a row is not whole vectors the last one ends at the row's end and
// overlaps the one before: its first elements are left out of sums and stores.
// The sums over rows (dgamma, dpost, dgate) are added up by a lane over its rows, over the work-group's waves in
// wave order, and over work-groups by a second kernel in block order: the same bits every run.
// Both ways are bound by bytes: 16384 x 4096 bf16 95 + 121 us (5.6 and 4.4 TB/s), 4095 x 2568 with post and a channel's gate
// 24 + 43, 2048 x 1000 fp32 with a token's gate 9 + 13, 64 x 4096 without gradients 6; the sums over work-groups take 5 to 7.
#include <algorithm>

#include "common.h"

namespace abacus {
namespace {

enum Gate : int { kNoGate = 0, kChannelGate = 1, kTokenGate = 2 };

struct NormArgs {
  const void *x, *y, *gamma, *post, *gate;
  void *r, *h;
  float *rstd, *y_rstd;  // NULL: not kept
  const void *dr, *dh;   // NULL: zeros
  void *dx, *dy, *dgamma, *dpost, *dgate;  // (the last three NULL: not wanted)
  float* partial;        // (blocks, sums, D)
  int64_t rows;
  int D, lpr, gate_kind;
  float scale, eps;
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

template <typename T>
__device__ inline float get(const u32x4& v, int i) {
  if constexpr (sizeof(T) == 2) return i & 1 ? hi_bf16(v[i >> 1]) : lo_bf16(v[i >> 1]);
  else return bits_f32(v[i]);
}
template <typename T>
__device__ inline u32x4 pack(const float* f) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) v[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
    else v[i] = f32_bits(f[i]);
  }
  return v;
}

// Keeps a value in its packed registers: without it the compiler holds on to the unpacked floats of every use.
__device__ inline void hold(u32x4& v) { asm volatile("" : "+v"(v)); }

enum Layout : int { kEven = 0, kWave = 1, kGroup = 2 };

// A lane's vector v: its column, and how many of its first elements are another vector's (EPV and more: all are).
template <typename T, int LAYOUT>
struct Place {
  int col, skip;
  __device__ inline Place(int li, int lanes, int v, int D) {
    constexpr int EPV = VecTraits<T>::kN;
    const int c = (li + v * lanes) * EPV;
    col = LAYOUT == kEven ? c : min(c, D - EPV);
    skip = c - col;
  }
};

// Every load is made, in bounds, whatever the lane holds: loads without branches between them are in flight together.
// What is another vector's or past the row is left out of sums by masking one factor of each term (own()), and is not stored.
template <typename T, int LAYOUT>
__device__ inline u32x4 load_vec(const T* row, const Place<T, LAYOUT>& p) {
  return *reinterpret_cast<const u32x4_any*>(row + p.col);
}
template <typename T, int LAYOUT>
__device__ inline u32x4 own(u32x4 v, const Place<T, LAYOUT>& p) {
  if constexpr (LAYOUT != kEven) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) v[i] &= (2 * i < p.skip ? 0u : 0xffffu) | (2 * i + 1 < p.skip ? 0u : 0xffff0000u);
      else v[i] = i < p.skip ? 0u : v[i];
    }
  }
  return v;
}
template <typename T, int LAYOUT>
__device__ inline void store_vec(T* row, const Place<T, LAYOUT>& p, const u32x4& v) {
  constexpr int EPV = VecTraits<T>::kN;
  if (LAYOUT == kEven || p.skip == 0) {
    *reinterpret_cast<u32x4_any*>(row + p.col) = v;
  } else if (p.skip < EPV) {
#pragma unroll
    for (int i = 1; i < EPV; ++i)
      if (i >= p.skip) row[p.col + i] = from_f32<T>(get<T>(v, i));
  }
}

// A row's sum over its lanes.  kGroup: the work-group's waves in order, through one of two places of sum_s in
// turn (the barrier of the next sum is between this one's reads and the next writes to its place).
template <int LAYOUT>
__device__ inline float row_sum(float v, int lpr, float (*sum_s)[16], int& turn) {
  for (int off = lpr >> 1; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  if constexpr (LAYOUT == kGroup) {
    float* s = sum_s[turn];
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s[0];
    for (int w = 1; w < (int)blockDim.x >> 6; ++w) v += s[w];
  }
  return v;
}

// The rows of a work-group, one after the other: the first, the step, a lane's place in its row.
template <int LAYOUT>
struct Rows {
  int lane, wave, li, sub, lanes, lpr;
  int64_t first, step;
  __device__ inline Rows(int lpr_) {
    lpr = LAYOUT == kEven ? lpr_ : 64;
    lane = threadIdx.x & 63;
    wave = threadIdx.x >> 6;
    lanes = LAYOUT == kGroup ? (int)blockDim.x : lpr;
    li = LAYOUT == kGroup ? (int)threadIdx.x : lane % lpr;
    sub = LAYOUT == kEven ? lane / lpr : 0;
    const int rpw = 64 / lpr;
    first = LAYOUT == kGroup ? (int64_t)blockIdx.x : ((int64_t)blockIdx.x * 4 + wave) * rpw;
    step = LAYOUT == kGroup ? (int64_t)gridDim.x : (int64_t)gridDim.x * 4 * rpw;
  }
};

constexpr int threads_of(int layout) { return layout == kGroup ? 1024 : 256; }

// PLAIN: without post, gate and scale.  A row is read once and stays in packed registers for its sums and stores; other rows'
// waves cover its loads (16384 x 4096 bf16 95 us; unpacked, with fewer waves a CU, 174).
template <typename T, int VPL, int LAYOUT, bool PLAIN>
__global__ __launch_bounds__(threads_of(LAYOUT)) void residual_norm_fwd_kernel(NormArgs a) {
  constexpr int EPV = VecTraits<T>::kN;
  __shared__ float sum_s[2][16];
  int turn = 0;
  const Rows<LAYOUT> at(a.lpr);
  const int D = a.D;
  for (int64_t r0 = at.first; r0 < a.rows; r0 += at.step) {
    const int64_t row = r0 + at.sub;
    const bool act = LAYOUT == kGroup || row < a.rows;
    const int64_t o = min(row, a.rows - 1) * D;  // (lanes past the last row read it again, and write nothing)
    u32x4 x[VPL], y[VPL];
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const Place<T, LAYOUT> c(at.li, at.lanes, v, D);
      x[v] = load_vec((const T*)a.x + o, c);
      y[v] = load_vec((const T*)a.y + o, c);
    }
    float p = 1.0f;
    if (!PLAIN && a.post) {
      float ss = 0.f;
#pragma unroll
      for (int v = 0; v < VPL; ++v) {
        const u32x4 mine = own(y[v], Place<T, LAYOUT>(at.li, at.lanes, v, D));
#pragma unroll
        for (int i = 0; i < EPV; ++i) {
          const float f = get<T>(mine, i);
          ss += f * f;
        }
        hold(y[v]);
      }
      ss = row_sum<LAYOUT>(ss, at.lpr, sum_s, turn);
      p = 1.0f / sqrtf(ss / (float)D + a.eps);
      if (act && at.li == 0 && a.y_rstd) a.y_rstd[row] = p;
    }
    float ss = 0.f;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const Place<T, LAYOUT> c(at.li, at.lanes, v, D);
      float f[EPV];
      if constexpr (PLAIN) {
#pragma unroll
        for (int i = 0; i < EPV; ++i) f[i] = get<T>(x[v], i) + get<T>(y[v], i);
      } else {
#pragma unroll
        for (int i = 0; i < EPV; ++i) f[i] = get<T>(y[v], i);
        if (a.post) {
          const u32x4 post = load_vec((const T*)a.post, c);
#pragma unroll
          for (int i = 0; i < EPV; ++i) f[i] = get<T>(post, i) * (f[i] * p);
        }
        if (a.gate_kind != kNoGate) {
          const u32x4 gate = load_vec((const T*)a.gate + (a.gate_kind == kTokenGate ? o : 0), c);
#pragma unroll
          for (int i = 0; i < EPV; ++i) f[i] *= get<T>(gate, i);
        }
#pragma unroll
        for (int i = 0; i < EPV; ++i) f[i] = get<T>(x[v], i) + f[i] * a.scale;
      }
      x[v] = own(pack<T>(f), c);  // r
#pragma unroll
      for (int i = 0; i < EPV; ++i) {
        const float r = get<T>(x[v], i);
        ss += r * r;
      }
      hold(x[v]);
    }
    ss = row_sum<LAYOUT>(ss, at.lpr, sum_s, turn);
    const float q = 1.0f / sqrtf(ss / (float)D + a.eps);
    if (!act) continue;
    if (at.li == 0 && a.rstd) a.rstd[row] = q;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const Place<T, LAYOUT> c(at.li, at.lanes, v, D);
      const u32x4 gamma = load_vec((const T*)a.gamma, c);
      store_vec((T*)a.r + o, c, x[v]);
      float f[EPV];
#pragma unroll
      for (int i = 0; i < EPV; ++i) f[i] = get<T>(gamma, i) * get<T>(x[v], i) * q;
      store_vec((T*)a.h + o, c, pack<T>(f));
    }
  }
}

// The three tensors of a row that every backward reads; the next row's are loaded before this row's sums.
template <typename T, int VPL, int LAYOUT>
struct RowIn {
  u32x4 r[VPL], dh[VPL], dr[VPL];
  float q;
  __device__ inline void load(const NormArgs& a, int64_t row, int li, int lanes) {
    const bool here = LAYOUT == kGroup || row < a.rows;
    row = min(row, a.rows - 1);
    const int64_t o = row * a.D;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const Place<T, LAYOUT> c(li, lanes, v, a.D);
      r[v] = load_vec((const T*)a.r + o, c);
      dh[v] = dr[v] = u32x4{0, 0, 0, 0};
      if (a.dh) dh[v] = load_vec((const T*)a.dh + o, c);
      if (a.dr) dr[v] = load_vec((const T*)a.dr + o, c);
    }
    q = here ? a.rstd[row] : 0.f;  // (lanes past the last row add nothing to the sums over rows)
  }
};

// sums: of dgamma, dpost and the channel gate's those that are wanted, in that order: a lane's own in registers over all
// its rows.  (16384 x 4096 bf16 121 us; with a row in one wave's registers, which spilled, 169.)
template <typename T, int VPL, int LAYOUT, bool PLAIN>
__global__ __launch_bounds__(threads_of(LAYOUT)) void residual_norm_bwd_kernel(NormArgs a) {
  constexpr int EPV = VecTraits<T>::kN, NE = VPL * EPV, SUMS = PLAIN ? 1 : 3;
  __shared__ float sum_s[2][16];
  __shared__ float red_s[LAYOUT == kGroup ? 1 : 4 * 64 * NE];
  int turn = 0;
  const Rows<LAYOUT> at(a.lpr);
  const int D = a.D;
  float sums[SUMS][NE];
#pragma unroll
  for (int k = 0; k < SUMS; ++k)
#pragma unroll
    for (int i = 0; i < NE; ++i) sums[k][i] = 0.f;
  const bool need_y = !PLAIN && (a.post || a.gate_kind != kNoGate);
  u32x4 gamma[VPL], post[VPL], gate[VPL];
#pragma unroll
  for (int v = 0; v < VPL; ++v) {
    const Place<T, LAYOUT> c(at.li, at.lanes, v, D);
    gamma[v] = own(load_vec((const T*)a.gamma, c), c);
    post[v] = gate[v] = u32x4{0, 0, 0, 0};
    if (!PLAIN && a.post) post[v] = own(load_vec((const T*)a.post, c), c);
    if (!PLAIN && a.gate_kind == kChannelGate) gate[v] = load_vec((const T*)a.gate, c);
  }
  RowIn<T, VPL, LAYOUT> next;
  if (at.first < a.rows) next.load(a, at.first + at.sub, at.li, at.lanes);
  for (int64_t r0 = at.first; r0 < a.rows; r0 += at.step) {
    const int64_t row = r0 + at.sub;
    const bool act = LAYOUT == kGroup || row < a.rows;
    const int64_t o = min(row, a.rows - 1) * D;
    RowIn<T, VPL, LAYOUT> in = next;
    u32x4 y[VPL];
    if constexpr (!PLAIN) {
#pragma unroll
      for (int v = 0; v < VPL; ++v) {
        const Place<T, LAYOUT> c(at.li, at.lanes, v, D);
        y[v] = u32x4{0, 0, 0, 0};
        if (need_y) y[v] = load_vec((const T*)a.y + o, c);
        if (a.gate_kind == kTokenGate) gate[v] = load_vec((const T*)a.gate + o, c);
      }
    }
    const float p = !PLAIN && a.post ? a.y_rstd[min(row, a.rows - 1)] : 1.0f;
    if (r0 + at.step < a.rows) next.load(a, r0 + at.step + at.sub, at.li, at.lanes);
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
#pragma unroll
      for (int i = 0; i < EPV; ++i) {
        const float t = get<T>(in.dh[v], i) * (get<T>(in.r[v], i) * in.q);
        sums[0][v * EPV + i] += t;
        s += get<T>(gamma[v], i) * t;
      }
      hold(in.dh[v]);
      hold(in.r[v]);
      hold(gamma[v]);
    }
    s = row_sum<LAYOUT>(s, at.lpr, sum_s, turn) / (float)D;
    float d[PLAIN ? 1 : NE];
    float t = 0.f;
    const float scale = act ? a.scale : 0.f;  // (likewise)
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const Place<T, LAYOUT> c(at.li, at.lanes, v, D);
      float f[EPV];
#pragma unroll
      for (int i = 0; i < EPV; ++i)
        f[i] = get<T>(in.dr[v], i) +
               in.q * (get<T>(in.dh[v], i) * get<T>(gamma[v], i) - get<T>(in.r[v], i) * in.q * s);
      if (act) store_vec((T*)a.dx + o, c, pack<T>(f));
      if constexpr (!PLAIN) {
        // f becomes db through the gate, then post's
        float dg[EPV];
#pragma unroll
        for (int i = 0; i < EPV; ++i) {
          const int e = v * EPV + i;
          const float m = get<T>(y[v], i) * p;
          f[i] *= scale;
          if (a.gate_kind != kNoGate) {
            dg[i] = f[i] * (a.post ? get<T>(post[v], i) * m : m);
            sums[2][e] += dg[i];
            f[i] *= get<T>(gate[v], i);
          }
          if (a.post) {
            sums[1][e] += f[i] * m;
            f[i] *= get<T>(post[v], i);
          }
          d[e] = f[i];
          t += f[i] * m;
        }
        hold(y[v]);
        hold(post[v]);
        hold(gate[v]);
        if (a.gate_kind == kTokenGate && a.dgate && act) store_vec((T*)a.dgate + o, c, pack<T>(dg));
      }
    }
    if constexpr (!PLAIN) {
      if (a.post) t = row_sum<LAYOUT>(t, at.lpr, sum_s, turn) / (float)D;
      if (act) {
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
          float f[EPV];
#pragma unroll
          for (int i = 0; i < EPV; ++i) {
            const int e = v * EPV + i;
            f[i] = a.post ? p * (d[e] - get<T>(y[v], i) * p * t) : d[e];
          }
          store_vec((T*)a.dy + o, Place<T, LAYOUT>(at.li, at.lanes, v, D), pack<T>(f));
        }
      }
    }
  }
  // the work-group's sums, one row of the partials each
  const bool wanted[3] = {a.dgamma != nullptr, !PLAIN && a.dpost, !PLAIN && a.gate_kind == kChannelGate && a.dgate};
  const int count = (int)wanted[0] + (int)wanted[1] + (int)wanted[2];
  int place = 0;
#pragma unroll
  for (int k = 0; k < SUMS; ++k) {
    if (!wanted[k]) continue;
    float* out = a.partial + ((int64_t)blockIdx.x * count + place++) * D;
    if constexpr (LAYOUT == kGroup) {
#pragma unroll
      for (int v = 0; v < VPL; ++v) {
        const Place<T, LAYOUT> c(at.li, at.lanes, v, D);
#pragma unroll
        for (int i = 0; i < EPV; ++i)
          if (i >= c.skip) out[c.col + i] = sums[k][v * EPV + i];
      }
    } else {
      // by element: a lane's vector v is vector li + v lanes of the row
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        float v = sums[k][i];
        for (int off = at.lpr; off < 64; off <<= 1) v += __shfl_xor(v, off, 64);
        if (at.sub == 0) red_s[(at.wave * 64 + at.li) * NE + i] = v;
      }
      __syncthreads();
      for (int c = threadIdx.x; c < D; c += 256) {
        const int vec = c / EPV, l = vec % at.lanes, v = vec / at.lanes;
        const int e = c - Place<T, LAYOUT>(l, at.lanes, v, D).col;
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) t += red_s[(w * 64 + l) * NE + v * EPV + e];
        out[c] = t;
      }
      __syncthreads();
    }
  }
}

// The work-groups' sums in block order: 64 columns a block, its 16 waves take 16 partial rows of each 256 at a time.
struct SumOut {
  void* out[3];
};
template <typename T>
__global__ __launch_bounds__(1024) void residual_norm_sum_kernel(const float* __restrict__ partial, int blocks, int count,
                                                                 int D, SumOut o) {
  __shared__ float part_s[16][64];
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, c = blockIdx.x * 64 + l;
  float total = 0.f;
  for (int b0 = 0; b0 < blocks; b0 += 256) {
    float v[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      const int b = b0 + 16 * w + u;
      v[u] = c < D && b < blocks ? partial[((int64_t)b * count + blockIdx.y) * D + c] : 0.f;
    }
#pragma unroll
    for (int h = 8; h >= 1; h >>= 1)
#pragma unroll
      for (int u = 0; u < h; ++u) v[u] += v[u + h];
    part_s[w][l] = v[0];
    __syncthreads();
    if (w == 0) {
#pragma unroll
      for (int u = 0; u < 16; ++u) total += part_s[u][l];
    }
    __syncthreads();
  }
  if (w == 0 && c < D) ((T*)o.out[blockIdx.y])[c] = from_f32<T>(total);
}

// ---------------------------------------------------------------- host

// Work-groups of the backward at most, a row of partials each.  Those of two waves may be more: 16384 x 1024 bf16 with post and a
// gate 53 + 9 us by 1280, 68 + 6 by 768; of more waves, more of them only cost the sums (plain 57 to 64 us of 16384 x 1024).
constexpr int kBwdBlocks = 768, kBwdSmallBlocks = 1280;
constexpr int kFwdBlocks = 4096;
// Waves of the backward that a CU holds at once, by its registers: a work-group more would wait for a place and
// then work alone.  (With post and a gate 8, 16 and 24: 56, 43 and 58 us of 4095 x 2568 bf16; plain 16, 24 and 32 alike.)
constexpr int kBwdWavesPlain = 24, kBwdWaves = 16;

struct Shape {
  int layout, lpr, vpl, threads;
  int64_t blocks(int64_t rows, int most) const {
    const int64_t per = layout == kGroup ? 1 : 4 * (64 / lpr);
    return std::max<int64_t>(1, std::min<int64_t>((rows + per - 1) / per, most));
  }
};

// Vectors of a lane in kEven.  Plain forwards have the RMSNorm kernels' (a work-group a row of 4096 bf16 91 us, not 95, but other
// sums); otherwise what a lane's registers hold beside the sums over rows.  With post and a gate, one vector more or less (the
// rows go to kGroup then): forwards of 8192 x 4096 bf16 57 us of one, 69 of eight, of 16384 x 1024 32 of one, 29 of two;
// backwards of 16384 x 1024 bf16 53 of one, 80 of two, of 32768 x 512 fp32 (half the values) 87 of one, 76 of two; plain
// backwards of 16384 x 1024 bf16 34 of one, 27 of two.
constexpr int kPlainFwdVectors = 8, kVectors = 2, kBf16BwdVectors = 1;
int most_vectors(bool bwd, bool plain, int dtype) {
  if (!bwd) return plain ? kPlainFwdVectors : kVectors;
  return plain || dtype != kBF16 ? kVectors : kBf16BwdVectors;
}

// kEven where the RMSNorm kernels take D and a lane would hold at most `most` vectors; else kWave with up to two of them,
// else kGroup with one.
Shape shape_of(int64_t D, int epv, int most) {
  const int64_t nvec = (D + epv - 1) / epv;
  int lpr = 64;
  while (lpr > 1 && nvec % lpr != 0) lpr >>= 1;
  const int64_t each = nvec / lpr;
  if (D % epv == 0 && each <= most && (each & (each - 1)) == 0) return {kEven, lpr, (int)each, 256};
  if (nvec <= 64 * std::min(most, kVectors)) return {kWave, 64, nvec <= 64 ? 1 : 2, 256};
  return {kGroup, 64, 1, (int)((nvec + 63) / 64) * 64};
}

int check(const char* name, int64_t rows, int64_t D, int gate_kind, bool gate, int dtype) {
  ABACUS_CHECK_ARG(dtype == kF32 || dtype == kBF16, "%s: unsupported dtype code %d (0 = fp32, 1 = bf16)", name, dtype);
  ABACUS_CHECK_ARG(rows >= 0, "%s: %lld rows", name, (long long)rows);
  const int least = dtype == kBF16 ? 8 : 4, most = 1024 * least;
  ABACUS_CHECK_ARG(D >= least && D <= most, "%s: dim %lld, %d to %d", name, (long long)D, least, most);
  ABACUS_CHECK_ARG(gate_kind >= kNoGate && gate_kind <= kTokenGate && gate == (gate_kind != kNoGate), "%s: gate kind %d", name,
                   gate_kind);
  return 0;
}

template <typename T, int VPL, int LAYOUT, bool PLAIN, bool BWD>
int launch(const NormArgs& a, const Shape& sh, int64_t blocks, hipStream_t s) {
  if constexpr (BWD)
    hipLaunchKernelGGL((residual_norm_bwd_kernel<T, VPL, LAYOUT, PLAIN>), dim3((unsigned)blocks), dim3(sh.threads), 0, s, a);
  else
    hipLaunchKernelGGL((residual_norm_fwd_kernel<T, VPL, LAYOUT, PLAIN>), dim3((unsigned)blocks), dim3(sh.threads), 0, s, a);
  ABACUS_CHECK_LAUNCH("residual_norm");
  return 0;
}

template <typename T, bool PLAIN, bool BWD>
int by_shape(const NormArgs& a, const Shape& sh, int64_t blocks, hipStream_t s) {
  if (sh.layout == kGroup) return launch<T, 1, kGroup, PLAIN, BWD>(a, sh, blocks, s);
  if (sh.vpl == 1)
    return sh.layout == kWave ? launch<T, 1, kWave, PLAIN, BWD>(a, sh, blocks, s) : launch<T, 1, kEven, PLAIN, BWD>(a, sh, blocks, s);
  if constexpr (!BWD || PLAIN || sizeof(T) == 4) {
    if (sh.vpl == 2)
      return sh.layout == kWave ? launch<T, 2, kWave, PLAIN, BWD>(a, sh, blocks, s) : launch<T, 2, kEven, PLAIN, BWD>(a, sh, blocks, s);
  }
  if constexpr (!BWD && PLAIN)
    return sh.vpl == 4 ? launch<T, 4, kEven, PLAIN, BWD>(a, sh, blocks, s) : launch<T, 8, kEven, PLAIN, BWD>(a, sh, blocks, s);
  return 1;  // (not reached: most_vectors)
}

template <bool BWD>
int dispatch(const NormArgs& a, const Shape& sh, int64_t blocks, int dtype, hipStream_t s) {
  if (!a.post && a.gate_kind == kNoGate && a.scale == 1.0f)
    return dtype == kBF16 ? by_shape<uint16_t, true, BWD>(a, sh, blocks, s) : by_shape<float, true, BWD>(a, sh, blocks, s);
  return dtype == kBF16 ? by_shape<uint16_t, false, BWD>(a, sh, blocks, s) : by_shape<float, false, BWD>(a, sh, blocks, s);
}

int sums_of(bool post, int gate_kind) { return 1 + (post ? 1 : 0) + (gate_kind == kChannelGate ? 1 : 0); }

}  // namespace
}  // namespace abacus

using namespace abacus;

extern "C" {

int abacus_residual_norm_fwd(const void* x, const void* y, const void* gamma, const void* post_gamma, const void* gate,
                             int gate_kind, int64_t rows, int64_t D, float scale, float eps, int dtype, void* r, void* h,
                             float* rstd, float* y_rstd, void* stream) {
  if (int rc = check("residual_norm_fwd", rows, D, gate_kind, gate != nullptr, dtype)) return rc;
  if (rows == 0) return 0;
  ABACUS_CHECK_ARG(x && y && gamma && r && h, "residual_norm_fwd: null pointer");
  NormArgs a{};
  a.x = x;
  a.y = y;
  a.gamma = gamma;
  a.post = post_gamma;
  a.gate = gate;
  a.gate_kind = gate_kind;
  a.rows = rows;
  a.D = (int)D;
  a.scale = scale;
  a.eps = eps;
  a.r = r;
  a.h = h;
  a.rstd = rstd;
  a.y_rstd = y_rstd;
  const bool plain = !post_gamma && gate_kind == kNoGate && scale == 1.0f;
  const Shape sh = shape_of(D, dtype == kBF16 ? 8 : 4, most_vectors(false, plain, dtype));
  a.lpr = sh.lpr;
  return dispatch<false>(a, sh, sh.blocks(rows, kFwdBlocks), dtype, (hipStream_t)stream);
}

int64_t abacus_residual_norm_bwd_ws_bytes(int64_t rows, int64_t D, int post, int gate_kind) {
  if (rows <= 0 || D <= 0) return 0;
  return std::min<int64_t>(kBwdSmallBlocks, rows) * sums_of(post != 0, gate_kind) * D * 4;
}

int abacus_residual_norm_bwd(const void* dr, const void* dh, const void* r, const void* y, const void* gamma,
                             const void* post_gamma, const void* gate, int gate_kind, const float* rstd,
                             const float* y_rstd, int64_t rows, int64_t D, float scale, int dtype, void* dx, void* dy,
                             void* dgamma, void* dpost, void* dgate, void* ws, int64_t ws_bytes, void* stream) {
  if (int rc = check("residual_norm_bwd", rows, D, gate_kind, gate != nullptr, dtype)) return rc;
  ABACUS_CHECK_ARG((post_gamma || !dpost) && (gate || !dgate), "residual_norm_bwd: the post norm's and the gate's gradients come with them");
  ABACUS_CHECK_ARG(rows >= 1, "residual_norm_bwd: no rows");
  ABACUS_CHECK_ARG(r && gamma && dx, "residual_norm_bwd: null pointer");
  const bool plain = !post_gamma && gate_kind == kNoGate && scale == 1.0f;
  ABACUS_CHECK_ARG(plain ? !dy || dy == dx : dy && dy != dx,
                   "residual_norm_bwd: dy is dx's memory or NULL without post_gamma, gate and scale, and its own with one");
  ABACUS_CHECK_ARG(rstd && (!post_gamma || y_rstd) && (y || (!post_gamma && gate_kind == kNoGate)),
                   "residual_norm_bwd: the forward's rstd, and with post_gamma y_rstd, and with it or a gate y");
  const int64_t need = abacus_residual_norm_bwd_ws_bytes(rows, D, post_gamma != nullptr, gate_kind);
  ABACUS_CHECK_ARG(ws != nullptr && (uintptr_t)ws % 16 == 0 && ws_bytes >= need,
                   "residual_norm_bwd: workspace of %lld bytes, %lld needed, 16-byte aligned", (long long)ws_bytes, (long long)need);
  NormArgs a{};
  a.dr = dr;
  a.dh = dh;
  a.r = const_cast<void*>(r);
  a.y = y;
  a.gamma = gamma;
  a.post = post_gamma;
  a.gate = gate;
  a.gate_kind = gate_kind;
  a.rstd = const_cast<float*>(rstd);
  a.y_rstd = const_cast<float*>(y_rstd);
  a.rows = rows;
  a.D = (int)D;
  a.scale = scale;
  a.dx = dx;
  a.dy = dy;
  a.dgamma = dgamma;
  a.dpost = dpost;
  a.dgate = dgate;
  a.partial = (float*)ws;
  const Shape sh = shape_of(D, dtype == kBF16 ? 8 : 4, most_vectors(true, plain, dtype));
  a.lpr = sh.lpr;
  const int at_once = std::max(1, (plain ? kBwdWavesPlain : kBwdWaves) / (sh.threads / 64));
  const int64_t blocks = sh.blocks(rows, std::min(sh.threads <= 128 ? kBwdSmallBlocks : kBwdBlocks, 256 * at_once));
  const hipStream_t s = (hipStream_t)stream;
  if (int rc = dispatch<true>(a, sh, blocks, dtype, s)) return rc;
  SumOut o{};
  int count = 0;
  for (void* sum : {dgamma, dpost, gate_kind == kChannelGate ? dgate : nullptr})
    if (sum) o.out[count++] = sum;
  if (count == 0) return 0;
  const dim3 grid((unsigned)((D + 63) / 64), (unsigned)count);
  if (dtype == kBF16)
    hipLaunchKernelGGL(residual_norm_sum_kernel<uint16_t>, grid, dim3(1024), 0, s, a.partial, (int)blocks, count, (int)D, o);
  else
    hipLaunchKernelGGL(residual_norm_sum_kernel<float>, grid, dim3(1024), 0, s, a.partial, (int)blocks, count, (int)D, o);
  ABACUS_CHECK_LAUNCH("residual_norm_bwd sums");
  return 0;
}

}  // extern "C"
