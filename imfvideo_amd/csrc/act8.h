// Activations kept in 8 bits for the backward pass, gfx950: tiles of 64 rows x 64 columns,
//   s = max|x| / 127 + 1e-12 (fp32),  code = round_half_away(x / s),  value = code * s.
// Storage: codes (row tiles, column tiles, 64, 64) int8, a tile's 4 KB row-major and
// contiguous, zero past the edges; scales (row tiles, column tiles) fp32.  A tile that holds
// an infinity or a NaN has a NaN scale: its values come back as NaN, not as numbers that
// were never there.
#pragma once

#include "common.h"

namespace sla2h {

constexpr int kAct = 64;                 // rows and columns of a tile
constexpr int kActBytes = kAct * kAct;   // codes of a tile

// Eight 16-bit elements of a row at column c (columns past F: zero), any 2-byte alignment.
// Whole groups are one 16-byte access; the last one of a row goes element by element, so that
// nothing past the row is touched.
typedef u32x4 __attribute__((aligned(2))) u32x4_2;
__device__ inline u32x4 load_row8(const uint16_t* row, int c, int F) {
  if (c + 8 <= F) return *reinterpret_cast<const u32x4_2*>(row + c);
  u32x4 v{0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (c + e < F) v[e >> 1] |= (uint32_t)row[c + e] << (16 * (e & 1));
  return v;
}
__device__ inline void store_row8(uint16_t* row, int c, int F, u32x4 v) {
  if (c + 8 <= F) {
    *reinterpret_cast<u32x4_2*>(row + c) = v;
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (c + e < F) row[c + e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
}

// |x| bits, two per register: 16-bit magnitudes order as integers (NaN above infinity)
typedef __attribute__((ext_vector_type(2))) uint16_t u16x2;
__device__ inline uint32_t abs_max2(uint32_t a, uint32_t b) {
  const u16x2 x = __builtin_bit_cast(u16x2, a), y = __builtin_bit_cast(u16x2, b & 0x7fff7fffu);
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(x, y));
}

// Largest magnitude of a wave's lanes (infinity for a NaN too), and the scale of a tile.
template <typename T16>
__device__ inline float wave_top_of(uint32_t top2) {
  constexpr uint32_t kInf = T16::kDtype == SLA2H_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
  const uint32_t a = top2 & 0xffffu, b = top2 >> 16;
  const uint32_t m = a > b ? a : b;
  return wave_max(m >= kInf ? __builtin_inff() : T16::to_f32((uint16_t)m));
}
__device__ inline float scale_of_top(float top) {
  return top == __builtin_inff() ? __builtin_nanf("") : top / 127.0f + 1e-12f;
}

// Codes of four elements, packed.  r = fl(1 / s): the product with r is within an ulp of
// the quotient, and one step of the remainder makes it the correctly rounded x / s (Markstein's
// theorem).  A half is added just below 0.5, which rounds halves away from zero and
// nothing under them.
__device__ inline uint32_t code4(float x0, float x1, float x2, float x3, float s, float r) {
  auto code = [&](float x) -> uint32_t {
    const float n0 = x * r;
    const float n = __builtin_fmaf(__builtin_fmaf(-n0, s, x), r, n0);
    return (uint32_t)(int)(n + __builtin_copysignf(0x1.fffffep-2f, n));
  };
  const uint32_t lo = __builtin_amdgcn_perm(code(x1), code(x0), 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(code(x3), code(x2), 0x0c0c0400u);
  return lo | (hi << 16);
}
template <typename T16>
__device__ inline u32x2 codes8(u32x4 v, float s, float r) {
  float x[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = T16::to_f32((uint16_t)(v[e] & 0xffff));
    x[2 * e + 1] = T16::to_f32((uint16_t)(v[e] >> 16));
  }
  return u32x2{code4(x[0], x[1], x[2], x[3], s, r), code4(x[4], x[5], x[6], x[7], s, r)};
}

// byte b of w as a signed number
template <int b>
__device__ inline float code_f32(uint32_t w) {
  return (float)(int8_t)(w >> (8 * b));
}
__device__ inline void values8(u32x2 c, float s, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    x[4 * e] = code_f32<0>(c[e]) * s;
    x[4 * e + 1] = code_f32<1>(c[e]) * s;
    x[4 * e + 2] = code_f32<2>(c[e]) * s;
    x[4 * e + 3] = code_f32<3>(c[e]) * s;
  }
}

}  // namespace sla2h
