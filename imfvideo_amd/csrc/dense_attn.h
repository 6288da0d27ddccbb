// Shared pieces of the dense attention kernels (forward and backward), gfx950:
// 32 x 32 x 16 MFMA tiles on 64-channel heads, tiles of 64 rows in LDS.
//
// Operand layout of a 32 x 32 x 16 product, lane l = 32 h + r:
//   A (rows) and B (columns): row / column r, contracted slots 8 h .. 8 h + 7;
//   C: column r, rows 8 g + 4 h + i in register 4 g + i (g, i = 0 .. 3).
// A C tile is therefore the B operand of a product that contracts its rows: step s
// (16 rows) takes registers 8 s .. 8 s + 7, slot j holding row 16 s + 8 (j / 4) + 4 h + j % 4.
// The A operand of that product reads the other matrix transposed from its row-major tile
// in LDS (ds_read_b64_tr_b16), rows in the same order.  Probabilities never leave
// the registers.
//
// LDS tile: 64 rows x 128 bytes, the 16-byte chunk c of row r at chunk c ^ key(r), key(r) the
// bits 1, 2, 3 of r reversed.  The 64 banks serve 256 bytes a cycle: 16 lanes of an operand read
// (one chunk of 16 rows: rows of one parity share 32 banks and have eight different keys) and 32
// lanes of a transposing read (64 bytes of four rows: the rows of one parity differ in the
// key's top bit, so their chunk quads do not meet).  Without conflicts for both; with r & 7 as
// the key both take twice the cycles.  The tiles are loaded straight into LDS (buffer_load ... lds): the
// swizzle is applied to the chunk each lane fetches, and rows past the end of a sequence come
// back as zeros from the buffer's range check, whatever memory holds there.
#pragma once

#include "common.h"

namespace sla2h {

typedef __attribute__((ext_vector_type(16))) float f32x16;

constexpr int kDD = 64;         // head width
constexpr int kRowB = 2 * kDD;  // bytes of a row of a head
constexpr int kTileRows = 64;
constexpr int kTileB = kTileRows * kRowB;

template <typename T16>
__device__ inline f32x16 mfma_32x32x16(u32x4 a, u32x4 b, f32x16 c);
template <>
__device__ inline f32x16 mfma_32x32x16<BF16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ inline f32x16 mfma_32x32x16<F16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ inline f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

__device__ inline void dma16(__amdgpu_buffer_rsrc_t rs, void* dst, int voff, int soff = 0) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)dst, 16,
                                           voff, soff, 0, 0);
}

// Rows [row0, row0 + n) of a (rows, 64) 16-bit matrix with row stride `ld` bytes as
// a buffer resource whose range check ends with the last row; n <= 0: empty.
__device__ inline __amdgpu_buffer_rsrc_t rows_rsrc(const uint16_t* base, int64_t row0, int64_t n,
                                                   int64_t ld) {
  const char* p = reinterpret_cast<const char*>(base) + row0 * ld;
  const int64_t rows = n < kTileRows ? n : kTileRows;
  return make_rsrc(p, n <= 0 ? 0 : (rows - 1) * ld + kRowB);
}

// Byte address (within a tile) of the 16-byte chunk c of row r.
__device__ inline int row_key(int r) {
  return ((r << 1) & 4) | ((r >> 1) & 2) | ((r >> 3) & 1);
}
__device__ inline int chunk_addr(int r, int c) { return r * kRowB + ((c ^ row_key(r)) << 4); }

// Loads eight rows (8 j .. 8 j + 7 of a tile) straight into LDS: lane l brings the chunk of
// row 8 j + l / 8 that belongs at its place.
__device__ inline void dma_rows8(__amdgpu_buffer_rsrc_t rs, unsigned char* tile, int j, int ld,
                                 int l) {
  const int r = 8 * j + (l >> 3);
  dma16(rs, tile + 8 * j * kRowB, r * ld + (((l & 7) ^ row_key(r)) << 4));
}

// A lane's byte offsets in a tile, for the operand reads below: eight registers, everything
// else is an immediate of the read.
struct LaneOff {
  int row[4];     // chunk 2 s + h of row l & 31
  int col[2][2];  // channels 32 mb .. of rows 4 h + .., and of the rows eight further on
  __device__ explicit LaneOff(int l) {
    const int h = l >> 5;
#pragma unroll
    for (int s = 0; s < 4; ++s) row[s] = chunk_addr(l & 31, 2 * s + h);
    const int r = 4 * h + ((l & 15) >> 2), c = 2 * ((l >> 4) & 1) + ((l & 3) >> 1);
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        col[mb][x] = chunk_addr(r + 8 * x, 4 * mb + c) + 8 * (l & 1);
  }
};

// Row operand (A or B) of rows r0 + (l & 31), r0 a multiple of 32: step s contracts channels
// 16 s .. 16 s + 15.
__device__ inline u32x4 row_frag(const unsigned char* tile, int r0, int s, const LaneOff& o) {
  return *reinterpret_cast<const u32x4*>(tile + o.row[s] + r0 * kRowB);
}

// Transposed operand: row = channel 32 mb + (l & 31), contracted over the tile's rows
// r0 .. r0 + 15 (r0 a multiple of 16) in the order of a C tile's registers (see above).
__device__ inline u32x4 col_frag(const unsigned char* tile, int r0, int mb, const LaneOff& o) {
  const u32x2 lo = lds_read_tr16(tile + o.col[mb][0] + r0 * kRowB);
  const u32x2 hi = lds_read_tr16(tile + o.col[mb][1] + r0 * kRowB);
  return u32x4{lo.x, lo.y, hi.x, hi.y};
}

// The B operand of step s from a C tile's registers, rounded to 16 bits.
template <typename T16>
__device__ inline u32x4 pack_step(const f32x16& p, int s) {
  return u32x4{pack_pair<T16>(p[8 * s], p[8 * s + 1]), pack_pair<T16>(p[8 * s + 2], p[8 * s + 3]),
               pack_pair<T16>(p[8 * s + 4], p[8 * s + 5]),
               pack_pair<T16>(p[8 * s + 6], p[8 * s + 7])};
}

// What that rounding lost, rounded to 16 bits itself (hi = pack_step(p, s)).
template <typename T16>
__device__ inline u32x4 lost_step(const f32x16& p, int s, const u32x4& hi) {
  u32x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    y[i] = pack_pair<T16>(p[8 * s + 2 * i] - T16::to_f32((uint16_t)(hi[i] & 0xffff)),
                          p[8 * s + 2 * i + 1] - T16::to_f32((uint16_t)(hi[i] >> 16)));
  return y;
}

__device__ inline float swap32_max(float v) {
  const float2 a = swap32(v);
  return fmaxf(a.x, a.y);
}
__device__ inline float swap32_sum(float v) {
  const float2 a = swap32(v);
  return a.x + a.y;
}

// s_waitcnt vmcnt(n) lgkmcnt(0)
constexpr int wait_vm_lgkm0(int n) { return (n & 15) | ((n >> 4) << 14) | 0x70; }

// Sequence lengths of batch b, clamped into [0, L]; L without an array.
__device__ inline int seq_len(const int32_t* lens, int b, int64_t L) {
  if (!lens) return (int)L;
  const int n = __builtin_amdgcn_readfirstlane(lens[b]);
  return n < 0 ? 0 : (n > L ? (int)L : n);
}

// Sizes that forward and backward take, the same for both: what the forward has answered the
// backward can answer.  Sizes of sequences fit an int with a tile's room, heads of a batch too (the
// launches' own bounds are looked at where their grids are known).
inline bool sizes_ok(int B, int H, int Hkv, int64_t Lq, int64_t Lk) {
  return B > 0 && H > 0 && Hkv > 0 && H % Hkv == 0 && Lq > 0 && Lk > 0 &&
         Lq < ((int64_t)1 << 30) && Lk < ((int64_t)1 << 30) &&
         (int64_t)B * H < ((int64_t)1 << 20) && (H / Hkv) * Lq < ((int64_t)1 << 31);
}

// ---- Softmax in one pass over the keys (forward kernels): see dense_attn.hip.

// Probabilities are held as exp2(S - m + shift); a lane's sum of 16 stays at or below `most`.
// fp16 spends its exponent range on the small ones (2^-24 to 2^15); bf16 has fp32's range.
template <typename T16>
struct Range;
template <>
struct Range<BF16> {
  static constexpr float shift = 0.f, most = 1024.f;
};
template <>
struct Range<F16> {
  static constexpr float shift = 9.f, most = 32768.f;
};
constexpr float kFloor = -1e30f;  // m before the first key (finite: -inf - m stays -inf)

// Largest of a lane's 16 scores.
__device__ inline float lane_max(const f32x16& s) {
  float mx = fmaxf(fmaxf(s[0], s[1]), s[2]);
#pragma unroll
  for (int i = 3; i < 15; i += 2) mx = fmaxf(fmaxf(mx, s[i]), s[i + 1]);
  return fmaxf(mx, s[15]);
}

// Moves the bound of a 32-key x 32-query tile to its maximum and rescales what the old
// bound weighed.
template <int MB>
__device__ inline void raise_bound(float mx, float c, float& m, float& lsum, f32x16 (&acc)[MB]) {
  const float mn = fmaxf(m, swap32_max(mx) * c);
  const float f = fast_exp2(m - mn);
  m = mn;
  lsum *= f;
#pragma unroll
  for (int b = 0; b < MB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[b][i] *= f;
}

// Probabilities of a tile, packed as the operands of the two product steps; their sum.
template <typename T16>
__device__ inline float probabilities(const f32x16& s, float c, float m, u32x4 (&p)[2]) {
  const float off = Range<T16>::shift - m;
  f32x16 e;
#pragma unroll
  for (int i = 0; i < 16; ++i) e[i] = fast_exp2(__builtin_fmaf(s[i], c, off));
#pragma unroll
  for (int t = 0; t < 2; ++t) p[t] = pack_step<T16>(e, t);
  float r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = (e[i] + e[4 + i]) + (e[8 + i] + e[12 + i]);
  return (r[0] + r[1]) + (r[2] + r[3]);
}

// What the rounding of a tile's probabilities lost, packed alike.
template <typename T16>
__device__ inline void lost_halves(const f32x16& s, float c, float m, const u32x4 (&p)[2],
                                   u32x4 (&q)[2]) {
  const float off = Range<T16>::shift - m;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = 8 * t + 2 * i;
      const uint32_t w = p[t][i];
      q[t][i] = pack_pair<T16>(
          fast_exp2(__builtin_fmaf(s[k], c, off)) - T16::to_f32((uint16_t)(w & 0xffff)),
          fast_exp2(__builtin_fmaf(s[k + 1], c, off)) - T16::to_f32((uint16_t)(w >> 16)));
    }
}

// scores of keys at or past a lane's limit -> -inf; lim counts from the tile's first key
__device__ inline void mask_tile(f32x16& s, int lim, int h) {
  const int x = lim - 4 * h;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    s[i] = 8 * (i >> 2) + (i & 3) < x ? s[i] : -__builtin_inff();
}

// Two values as 16 bits, and what the rounding lost as 16 bits again (0 past the type's range).
template <typename T16>
__device__ inline uint32_t round_pair(float x, float y, uint32_t& lost) {
  const uint32_t p = pack_pair<T16>(x, y);
  const float ex = x - T16::to_f32((uint16_t)(p & 0xffff)), ey = y - T16::to_f32((uint16_t)(p >> 16));
  lost = pack_pair<T16>(__builtin_fabsf(ex) < __builtin_inff() ? ex : 0.f,
                        __builtin_fabsf(ey) < __builtin_inff() ? ey : 0.f);
  return p;
}

// Keys that query i sees: [0, limit).
__device__ inline int key_limit(int i, int qlen, int klen, int causal) {
  if (i >= qlen) return 0;
  if (!causal) return klen;
  const int64_t e = (int64_t)i + klen - qlen + 1;
  return e < 0 ? 0 : (e < klen ? (int)e : klen);
}

// Which head and tile a workgroup takes.  Workgroups go to the eight XCDs in turn, each with
// an L2 of its own.
//   even tiles (no mask, no lengths): an XCD takes a run of neighbouring tiles, so that those of
//     a head share the streamed operand in its L2;
//   uneven ones: heads in turn over the XCDs (a multiple of eight heads: each XCD keeps its own),
//     tile by tile, the longest first where the mask orders them (`last`): runs of
//     neighbours would leave the XCDs of short sequences idle (B = 3, H = 8, L = 4,159, causal: forward
//     83 us in runs, 72 so).
struct WorkMap {
  int heads, tiles;  // tiles of a head
  int n;             // heads * tiles
  int even, last;
};
inline WorkMap work_map(int64_t heads, int64_t tiles, bool even, bool last) {
  return WorkMap{(int)heads, (int)tiles, (int)(heads * tiles), even, last};
}
inline unsigned work_grid(const WorkMap& m) { return 8u * ((m.n + 7) / 8); }
__device__ inline bool work_item(const WorkMap& m, int blk, int& head, int& tile) {
  if (m.even) {
    const int i = (blk & 7) * ((m.n + 7) / 8) + (blk >> 3);
    if (i >= m.n) return false;
    head = i / m.tiles;
    tile = i - head * m.tiles;
  } else if (blk >= m.n) {
    return false;
  } else if (m.heads % 8 == 0) {
    const int per = m.heads / 8, i = blk >> 3;
    tile = i / per;
    head = (blk & 7) + 8 * (i - tile * per);
  } else {
    tile = blk / m.heads;
    head = blk - tile * m.heads;
  }
  head = __builtin_amdgcn_readfirstlane(head);
  tile = __builtin_amdgcn_readfirstlane(m.last ? m.tiles - 1 - tile : tile);
  return true;
}

}  // namespace sla2h
