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
// Layout: a row is spread over lpr lanes of a wave (the RMSNorm kernels' layout, so the same sums), or over a
// work-group of 4 waves where it is longer; a lane holds VPL vectors of 16 bytes.  Rows may start at any element: the last
// vector of a D that is not whole vectors is taken element by element.
// The sums over rows (dgamma, dpost, dgate) are added up by a lane over its rows, over the work-group's waves in
// wave order, and over work-groups by a second kernel in block order: the same bits every run.
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
  void *dx, *dy, *dgate;
  float* partial;        // (blocks, sums, D)
  int64_t rows;
  int D, lpr, gate_kind;
  float scale, eps;
};

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

// The n (at most one vector's) values at p, at any element.
template <typename T>
__device__ inline void load_row(const T* p, int n, float* f) {
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
__device__ inline void store_row(T* p, int n, const float* f) {
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

// A row's sum over its lanes.  WIDE: the work-group's; sum_s is free again after the next barrier.
template <bool WIDE>
__device__ inline float row_sum(float v, int lpr, float* sum_s) {
  for (int off = lpr >> 1; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  if constexpr (WIDE) {
    if ((threadIdx.x & 63) == 0) sum_s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sum_s[0] + sum_s[1] + sum_s[2] + sum_s[3];
    __syncthreads();
  }
  return v;
}

// The rows of a work-group of 4 waves, one after the other: the first, the step, a lane's place in its row.
template <bool WIDE>
struct Rows {
  int lane, wave, li, sub;
  int64_t first, step;
  __device__ inline Rows(int lpr) {
    lane = threadIdx.x & 63;
    wave = threadIdx.x >> 6;
    li = WIDE ? (int)threadIdx.x : lane % lpr;
    sub = WIDE ? 0 : lane / lpr;
    const int rpw = WIDE ? 1 : 64 / lpr;
    first = WIDE ? (int64_t)blockIdx.x : ((int64_t)blockIdx.x * 4 + wave) * rpw;
    step = WIDE ? (int64_t)gridDim.x : (int64_t)gridDim.x * 4 * rpw;
  }
};

template <typename T, int VPL, bool WIDE, bool PLAIN>
__global__ __launch_bounds__(256) void residual_norm_fwd_kernel(NormArgs a) {
  constexpr int EPV = VecTraits<T>::kN, NE = VPL * EPV;
  __shared__ float sum_s[4];
  const Rows<WIDE> at(a.lpr);
  const int lanes = WIDE ? 256 : a.lpr, D = a.D;
  for (int64_t r0 = at.first; r0 < a.rows; r0 += at.step) {
    const int64_t row = r0 + at.sub;
    const bool act = row < a.rows;
    const int64_t o = row * D;
    float x[NE], y[NE];
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const int c = (at.li + v * lanes) * EPV, n = act ? D - c : 0;
      load_row<T>((const T*)a.x + o + c, n, x + v * EPV);
      load_row<T>((const T*)a.y + o + c, n, y + v * EPV);
    }
    if constexpr (!PLAIN) {
      if (a.post) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < NE; ++i) ss += y[i] * y[i];
        ss = row_sum<WIDE>(ss, WIDE ? 64 : a.lpr, sum_s);
        const float p = 1.0f / sqrtf(ss / (float)D + a.eps);
        if (act && at.li == 0 && a.y_rstd) a.y_rstd[row] = p;
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
          const int c = (at.li + v * lanes) * EPV;
          float f[EPV];
          load_row<T>((const T*)a.post + c, D - c, f);
#pragma unroll
          for (int i = 0; i < EPV; ++i) y[v * EPV + i] = f[i] * (y[v * EPV + i] * p);
        }
      }
      if (a.gate_kind != kNoGate) {
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
          const int c = (at.li + v * lanes) * EPV;
          float f[EPV];
          load_row<T>((const T*)a.gate + (a.gate_kind == kTokenGate ? o : 0) + c, act ? D - c : 0, f);
#pragma unroll
          for (int i = 0; i < EPV; ++i) y[v * EPV + i] *= f[i];
        }
      }
#pragma unroll
      for (int i = 0; i < NE; ++i) y[i] *= a.scale;
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      x[i] = round_to<T>(x[i] + y[i]);
      ss += x[i] * x[i];
    }
    ss = row_sum<WIDE>(ss, WIDE ? 64 : a.lpr, sum_s);
    const float q = 1.0f / sqrtf(ss / (float)D + a.eps);
    if (!act) continue;
    if (at.li == 0 && a.rstd) a.rstd[row] = q;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const int c = (at.li + v * lanes) * EPV;
      store_row<T>((T*)a.r + o + c, D - c, x + v * EPV);
      float f[EPV];
      load_row<T>((const T*)a.gamma + c, D - c, f);
#pragma unroll
      for (int i = 0; i < EPV; ++i) f[i] = f[i] * x[v * EPV + i] * q;
      store_row<T>((T*)a.h + o + c, D - c, f);
    }
  }
}

// sums: dgamma, and where they are wanted dpost and the channel gate's, in that order.
template <typename T, int VPL, bool WIDE, bool PLAIN>
__global__ __launch_bounds__(256) void residual_norm_bwd_kernel(NormArgs a) {
  constexpr int EPV = VecTraits<T>::kN, NE = VPL * EPV, SUMS = PLAIN ? 1 : 3;
  __shared__ float sum_s[4];
  __shared__ float red_s[WIDE ? 1 : 4 * 64 * NE];
  const Rows<WIDE> at(a.lpr);
  const int lanes = WIDE ? 256 : a.lpr, D = a.D;
  float sums[SUMS][NE];
#pragma unroll
  for (int k = 0; k < SUMS; ++k)
#pragma unroll
    for (int i = 0; i < NE; ++i) sums[k][i] = 0.f;
  for (int64_t r0 = at.first; r0 < a.rows; r0 += at.step) {
    const int64_t row = r0 + at.sub;
    const bool act = row < a.rows;
    const int64_t o = row * D;
    float g[NE], n[NE], d[NE];  // dh then g; r then n; dr
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const int c = (at.li + v * lanes) * EPV, left = act ? D - c : 0;
      load_row<T>((const T*)a.r + o + c, left, n + v * EPV);
      load_row<T>((const T*)a.dh + o + c, a.dh ? left : 0, g + v * EPV);
      load_row<T>((const T*)a.dr + o + c, a.dr ? left : 0, d + v * EPV);
    }
    const float q = act ? a.rstd[row] : 0.f;
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const int c = (at.li + v * lanes) * EPV;
      float f[EPV];
      load_row<T>((const T*)a.gamma + c, D - c, f);
#pragma unroll
      for (int i = 0; i < EPV; ++i) {
        const int e = v * EPV + i;
        n[e] *= q;
        sums[0][e] += g[e] * n[e];
        g[e] *= f[i];
        s += g[e] * n[e];
      }
    }
    s = row_sum<WIDE>(s, WIDE ? 64 : a.lpr, sum_s) / (float)D;
#pragma unroll
    for (int i = 0; i < NE; ++i) d[i] += q * (g[i] - n[i] * s);
    if (act) {
#pragma unroll
      for (int v = 0; v < VPL; ++v) {
        const int c = (at.li + v * lanes) * EPV;
        store_row<T>((T*)a.dx + o + c, D - c, d + v * EPV);
      }
    }
    if constexpr (!PLAIN) {
      // d becomes db; n the norm of y (or y) and g the branch b
#pragma unroll
      for (int i = 0; i < NE; ++i) d[i] *= a.scale;
      const bool need_y = a.post || a.gate_kind != kNoGate;
      const float p = a.post && act ? a.y_rstd[row] : 1.0f;
#pragma unroll
      for (int v = 0; v < VPL; ++v) {
        const int c = (at.li + v * lanes) * EPV, left = act ? D - c : 0;
        float post[EPV], gate[EPV];
        load_row<T>((const T*)a.y + o + c, need_y ? left : 0, n + v * EPV);
        load_row<T>((const T*)a.post + c, a.post ? D - c : 0, post);
        load_row<T>((const T*)a.gate + (a.gate_kind == kTokenGate ? o : 0) + c, a.gate_kind != kNoGate ? left : 0, gate);
#pragma unroll
        for (int i = 0; i < EPV; ++i) {
          const int e = v * EPV + i;
          n[e] *= p;
          const float b = a.post ? post[i] * n[e] : n[e];
          if (a.gate_kind != kNoGate) {
            const float dg = d[e] * b;
            sums[2][e] += dg;
            d[e] *= gate[i];
            gate[i] = dg;
          }
          if (a.post) {
            sums[1][e] += d[e] * n[e];
            d[e] *= post[i];
          }
        }
        if (a.gate_kind == kTokenGate && act) store_row<T>((T*)a.dgate + o + c, D - c, gate);
      }
      if (a.post) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < NE; ++i) t += d[i] * n[i];
        t = row_sum<WIDE>(t, WIDE ? 64 : a.lpr, sum_s) / (float)D;
#pragma unroll
        for (int i = 0; i < NE; ++i) d[i] = p * (d[i] - n[i] * t);
      }
      if (act && a.dy) {
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
          const int c = (at.li + v * lanes) * EPV;
          store_row<T>((T*)a.dy + o + c, D - c, d + v * EPV);
        }
      }
    }
  }
  // the work-group's sums, one row of the partials each
  const bool wanted[3] = {true, !PLAIN && a.post, !PLAIN && a.gate_kind == kChannelGate};
  int place = 0;
#pragma unroll
  for (int k = 0; k < SUMS; ++k) {
    if (!wanted[k]) continue;
    const int count = 1 + (int)wanted[1] + (int)wanted[2];
    float* out = a.partial + ((int64_t)blockIdx.x * count + place++) * D;
    if constexpr (WIDE) {
#pragma unroll
      for (int v = 0; v < VPL; ++v)
#pragma unroll
        for (int i = 0; i < EPV; ++i) {
          const int c = (at.li + v * lanes) * EPV + i;
          if (c < D) out[c] = sums[k][v * EPV + i];
        }
    } else {
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        float v = sums[k][i];
        for (int off = a.lpr; off < 64; off <<= 1) v += __shfl_xor(v, off, 64);
        if (at.sub == 0) red_s[(at.wave * 64 + at.li) * NE + i] = v;
      }
      __syncthreads();
      for (int c = threadIdx.x; c < D; c += 256) {
        const int vec = c / EPV, l = vec % lanes, v = vec / lanes;
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) t += red_s[(w * 64 + l) * NE + v * EPV + c % EPV];
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

constexpr int kBwdBlocks = 512;  // at most: a row of partials each
constexpr int kFwdBlocks = 4096;

struct Shape {
  int lpr, vpl;
  bool wide;
  int64_t blocks(int64_t rows, int most) const {
    const int64_t per = wide ? 1 : 4 * (64 / lpr);
    return std::max<int64_t>(1, std::min<int64_t>((rows + per - 1) / per, most));
  }
};

// The RMSNorm kernels' lanes where they take D (the largest power of two that divides the row's vectors), or a whole
// wave, up to `most` vectors a lane; else a work-group.
Shape shape_of(int64_t D, int epv, int most) {
  const int64_t nvec = (D + epv - 1) / epv;
  int lpr = 64;
  while (lpr > 1 && nvec % lpr != 0) lpr >>= 1;
  if (D % epv != 0 || nvec / lpr > most) lpr = 64;
  int64_t v = (nvec + lpr - 1) / lpr;
  const bool wide = v > most;
  if (wide) v = (nvec + 255) / 256;
  return {wide ? 64 : lpr, (int)(v <= 1 ? 1 : v <= 2 ? 2 : v <= 4 ? 4 : 8), wide};
}

constexpr int kFwdVectors = 8, kBwdVectors = 2;  // of a lane before a row takes a work-group

int check(const char* name, int64_t rows, int64_t D, int gate_kind, bool gate, int dtype) {
  ABACUS_CHECK_ARG(dtype == kF32 || dtype == kBF16, "%s: unsupported dtype code %d (0 = fp32, 1 = bf16)", name, dtype);
  ABACUS_CHECK_ARG(rows >= 0, "%s: %lld rows", name, (long long)rows);
  const int most = 256 * 8 * (dtype == kBF16 ? 8 : 4);
  ABACUS_CHECK_ARG(D >= 1 && D <= most, "%s: dim %lld, at most %d", name, (long long)D, most);
  ABACUS_CHECK_ARG(gate_kind >= kNoGate && gate_kind <= kTokenGate && gate == (gate_kind != kNoGate), "%s: gate kind %d", name,
                   gate_kind);
  return 0;
}

template <typename T, bool WIDE, bool PLAIN, bool BWD>
int launch(const NormArgs& a, int vpl, int64_t blocks, hipStream_t s) {
#define ABACUS_GO(V)                                                                                               \
  do {                                                                                                             \
    if constexpr (BWD) hipLaunchKernelGGL((residual_norm_bwd_kernel<T, V, WIDE, PLAIN>), dim3((unsigned)blocks), dim3(256), 0, s, a); \
    else hipLaunchKernelGGL((residual_norm_fwd_kernel<T, V, WIDE, PLAIN>), dim3((unsigned)blocks), dim3(256), 0, s, a); \
  } while (0)
  if (vpl == 1) ABACUS_GO(1);
  else if (vpl == 2) ABACUS_GO(2);
  else if constexpr (!BWD || WIDE) {
    if (vpl == 4) ABACUS_GO(4);
    else ABACUS_GO(8);
  }
#undef ABACUS_GO
  ABACUS_CHECK_LAUNCH("residual_norm");
  return 0;
}

template <bool BWD>
int dispatch(const NormArgs& a, const Shape& sh, int64_t blocks, int dtype, hipStream_t s) {
  const bool plain = !a.post && a.gate_kind == kNoGate && a.scale == 1.0f;
#define ABACUS_GO(T)                                                                                  \
  (sh.wide ? (plain ? launch<T, true, true, BWD>(a, sh.vpl, blocks, s) : launch<T, true, false, BWD>(a, sh.vpl, blocks, s)) \
           : (plain ? launch<T, false, true, BWD>(a, sh.vpl, blocks, s) : launch<T, false, false, BWD>(a, sh.vpl, blocks, s)))
  return dtype == kBF16 ? ABACUS_GO(uint16_t) : ABACUS_GO(float);
#undef ABACUS_GO
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
  const Shape sh = shape_of(D, dtype == kBF16 ? 8 : 4, kFwdVectors);
  a.lpr = sh.lpr;
  return dispatch<false>(a, sh, sh.blocks(rows, kFwdBlocks), dtype, (hipStream_t)stream);
}

int64_t abacus_residual_norm_bwd_ws_bytes(int64_t rows, int64_t D, int post, int gate_kind) {
  if (rows <= 0 || D <= 0) return 0;
  return (int64_t)kBwdBlocks * sums_of(post != 0, gate_kind) * D * 4;
}

int abacus_residual_norm_bwd(const void* dr, const void* dh, const void* r, const void* y, const void* gamma,
                             const void* post_gamma, const void* gate, int gate_kind, const float* rstd,
                             const float* y_rstd, int64_t rows, int64_t D, float scale, int dtype, void* dx, void* dy,
                             void* dgamma, void* dpost, void* dgate, void* ws, int64_t ws_bytes, void* stream) {
  if (int rc = check("residual_norm_bwd", rows, D, gate_kind, gate != nullptr, dtype)) return rc;
  ABACUS_CHECK_ARG((post_gamma != nullptr) == (dpost != nullptr) && (gate != nullptr) == (dgate != nullptr),
                   "residual_norm_bwd: the post norm's and the gate's gradients come with them");
  ABACUS_CHECK_ARG(rows >= 1, "residual_norm_bwd: no rows");
  const int64_t need = abacus_residual_norm_bwd_ws_bytes(rows, D, post_gamma != nullptr, gate_kind);
  ABACUS_CHECK_ARG(ws != nullptr && ws_bytes >= need, "residual_norm_bwd: workspace of %lld bytes, %lld needed",
                   (long long)ws_bytes, (long long)need);
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
  a.dgate = dgate;
  a.partial = (float*)ws;
  const Shape sh = shape_of(D, dtype == kBF16 ? 8 : 4, kBwdVectors);
  a.lpr = sh.lpr;
  const int64_t blocks = sh.blocks(rows, kBwdBlocks);
  const hipStream_t s = (hipStream_t)stream;
  if (int rc = dispatch<true>(a, sh, blocks, dtype, s)) return rc;
  SumOut o{{dgamma, dgate, nullptr}};
  if (post_gamma) o.out[1] = dpost, o.out[2] = dgate;
  const int count = sums_of(post_gamma != nullptr, gate_kind);
  const dim3 grid((unsigned)((D + 63) / 64), (unsigned)count);
  if (dtype == kBF16)
    hipLaunchKernelGGL(residual_norm_sum_kernel<uint16_t>, grid, dim3(1024), 0, s, a.partial, (int)blocks, count, (int)D, o);
  else
    hipLaunchKernelGGL(residual_norm_sum_kernel<float>, grid, dim3(1024), 0, s, a.partial, (int)blocks, count, (int)D, o);
  ABACUS_CHECK_LAUNCH("residual_norm_bwd sums");
  return 0;
}

}  // extern "C"
