// Shared pieces of the differential attention kernels (forward and backward), gfx950: tiles of 32
// rows of a pair of heads, four matrices of 64 channels side by side (key or query heads 2p and
// 2p + 1 of the two maps, value or output heads 2p and 2p + 1: one 128-channel matrix).
#pragma once

#include "dense_attn.h"

namespace sla2h {

constexpr int kUnitRows = 32;
constexpr int kUnitB = kUnitRows * kRowB;  // one matrix's rows: 4 KB
constexpr int kStageB = 4 * kUnitB;        // a stage: 16 KB

// Rows [row0, row0 + n), at most 32, of one 64-channel matrix into its place of a stage, by one wave.
__device__ inline void load_unit(const uint16_t* base, int64_t row0, int64_t n, int64_t ld,
                                 unsigned char* unit, int l) {
  const auto rs = rows_rsrc(base, row0, n < kUnitRows ? n : kUnitRows, ld);
#pragma unroll
  for (int j = 0; j < 4; ++j) dma_rows8(rs, unit, j, (int)ld, l);
}

// The pairs' weights of the second map: fp16, bf16 or fp32 (2), `stride` elements apart (0: one for all).
struct Weights {
  const void* p;
  int dtype;
  int64_t stride;
  __device__ float operator[](int64_t i) const {
    if (dtype == 2) return static_cast<const float*>(p)[i * stride];
    const uint16_t v = static_cast<const uint16_t*>(p)[i * stride];
    return dtype == SLA2H_DTYPE_BF16 ? BF16::to_f32(v) : F16::to_f32(v);
  }
  bool ok() const {
    return p && dtype >= 0 && dtype <= 2 && stride >= 0 &&
           reinterpret_cast<uintptr_t>(p) % (dtype == 2 ? 4 : 2) == 0;
  }
};

inline bool diff_sizes_ok(int B, int H, int Hkv, int64_t Lq, int64_t Lk) {
  return sizes_ok(B, H, Hkv, Lq, Lk) && H % 2 == 0 && Hkv % 2 == 0;
}

}  // namespace sla2h
