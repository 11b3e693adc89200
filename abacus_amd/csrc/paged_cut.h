// The work of an attention call over a paged cache, and how it is cut.
//
// Rows r = (token, query head of the group) of one key head are packed, R to a unit; a
// unit's keys are cut into `split` pieces of whole 64-key tiles where there are too few
// units for the GPU, and each piece gives its rows' maximum, sum and unscaled output,
// which a second kernel joins in order.  The piece length is the same for the whole
// launch: its (unit, key head, tile)s spread over kShort pieces of at least `least` tiles
// each, and over up to `target` pieces as long as those have `full` tiles.  The units are
// found from the device's lengths by a scan (paged_rows.h), a launch being sized for the
// most there can be.  Blocks of a kind take the sequences whose rows of a key head number
// more than `over` and at most `upto`.
#pragma once

#include "paged_rows.h"

namespace abacus {

constexpr int kTile = 64;   // keys of a tile

struct PagedArgs {
  PagedRows a;
  const void *q, *k, *v;
  const uint8_t *k_scale, *v_scale;
  void* o;
  float* part;  // (item, key head): R x K outputs, then R maxima, R sums
  int H, Hk, G, K;
  float scale_log2;
  int zero_rest;   // rows of no sequence: 0, or left as they are
  int over, upto;  // rows of a key head that a sequence of these blocks has
  int target, least, full;
};

// Pieces there may be before they have to be full ones: one a CU, as the sequences' last add to them.
constexpr int kShort = 192;

// Units of a sequence for blocks of this kind.
template <int R>
__device__ inline int units_of(const PagedArgs& p, const SeqRows& r) {
  const int rows = r.n * p.G;
  return rows > p.over && rows <= p.upto ? (rows + R - 1) / R : 0;
}

// Tiles of a piece, the same on every wave and in both kernels.  (A sum in floats, taken
// larger by more than they can be off: the launch has room for no more pieces.)
// `given`: the rows that the sequences have, of both kinds (in floats too: at most 2^24).
template <int R>
__device__ inline int piece_tiles(const PagedArgs& p, const SeqScan& scan, int& given) {
  float rows = 0.f;
  const float total = scan.sum([&](const SeqRows& r) {  // tiles of one key head
    rows += (float)r.n;
    return (float)units_of<R>(p, r) * (float)((r.len + kTile - 1) / kTile);
  });
  given = (int)wave_total(rows);
  auto spread = [&](int pieces) {
    return (int)fminf(ceilf(total * 1.001f / (float)((pieces + p.Hk - 1) / p.Hk)), 1e9f);
  };
  return max(max(p.least, spread(p.target)), min(p.full, spread(kShort)));
}

// Pieces of each of a sequence's units.
__device__ inline int pieces_of(const SeqRows& r, int chunk) {
  return max(1, ((r.len + kTile - 1) / kTile + chunk - 1) / chunk);
}

// What a block has: rows row0 .. row0 + rows - 1 of a sequence's n * G against tiles t0 .. t1 - 1.
struct Item {
  SeqRows r;
  int seq, split, row0, rows;
  int seen, least;  // keys that the last, the first of the rows sees
  int t0, t1;
  int given;  // rows that the call's sequences have, one after the other from query_start[0] on
};

__device__ inline int seen_of(const SeqRows& r, int row, int G) { return max(0, r.len - r.n + row / G + 1); }

// The whole block's item, false where there is none (`given` is set all the same).
template <int R>
__device__ inline bool find_item(const PagedArgs& p, int item, Item& w) {
  const SeqScan scan(p.a);
  const int chunk = piece_tiles<R>(p, scan, w.given);
  int local;
  if (!scan.find(item, [&](const SeqRows& r) { return units_of<R>(p, r) * pieces_of(r, chunk); }, w.seq, local, w.r))
    return false;
  w.split = pieces_of(w.r, chunk);
  const int units = units_of<R>(p, w.r);
  const int unit = units - 1 - local / w.split, piece = local % w.split;  // those with the most keys first
  w.row0 = unit * R;
  w.rows = min(R, w.r.n * p.G - w.row0);
  w.seen = seen_of(w.r, w.row0 + w.rows - 1, p.G);
  w.least = seen_of(w.r, w.row0, p.G);
  const int tiles = (w.seen + kTile - 1) / kTile, per = (tiles + w.split - 1) / w.split;
  w.t0 = min(piece * per, tiles);
  w.t1 = min(w.t0 + per, tiles);
  return true;
}

// o of row `row` (of the sequence's n * G), dims d .. d + 3, from the unscaled sums.
template <typename Q, class V4>
__device__ inline void store_row4(const PagedArgs& p, const SeqRows& r, int kh, int row, int d, const V4& o, float l) {
  const int sees = r.len - r.n + row / p.G + 1;
  const float inv = r.bad ? __builtin_nanf("") : 1.f / l;
  Q* to = (Q*)p.o + ((int64_t)(r.first + row / p.G) * p.H + kh * p.G + row % p.G) * p.K + d;
  float x[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) x[n] = sees <= 0 && !r.bad ? 0.f : o[n] * inv;
  if constexpr (sizeof(Q) == 2) {
    uint2 w;
    w.x = pack_bf16x2(x[0], x[1]);
    w.y = pack_bf16x2(x[2], x[3]);
    *reinterpret_cast<uint2*>(to) = w;
  } else {
    *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
  }
}

// 4 codes (a dword), times 2^(exponent of s), as bf16
__device__ inline uint2 codes_bf16(uint32_t w, float s) {
  uint2 r;
  r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false));
  r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true));
  return r;
}
// 2^(byte i of w - 127)
__device__ inline float byte_scale(uint32_t w, int i) { return bits_f32(((w >> (8 * i)) & 0xffu) << 23); }

// Rows of a key head that a chunk block has (paged_chunk.h), and the launch with blocks of both
// kinds (paged_chunk.hip; few_rows: 16 or 32).
constexpr int kChunkRows = 128;
int launch_both(const PagedArgs& few, const PagedArgs& many, unsigned few_blocks, unsigned many_blocks, int few_rows,
                bool codes, hipStream_t s);

}  // namespace abacus
