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

// What a launch of workgroups, two of which fit on a CU, takes (us on this card, without launching):
// per stage `two` for every full round of 512 and, for the rest, `one` while each has a CU of its own.
// Work of unequal workgroups (share below 1: what is left of all of it on average) has no rounds, but
// takes no less than its longest one, a fifth more for its neighbours.  Ranges of a long axis: `join`
// more per workgroup for its partial sums' way through memory, and the launch that adds them.
struct SplitCost {
  float one, two, join;
  int least;         // stages of a range
  int64_t most = 1280;  // workgroups
  float time(int64_t blocks, int64_t stages, int64_t s, float share) const {
    const int64_t w = blocks * s, n = (stages + s - 1) / s, rest = w % 512;
    const float full = two * (float)w * share / 512.f, longest = 1.2f * one;
    const float stage = share == 1.f
                            ? (float)(w / 512) * two + (rest == 0 ? 0.f : (rest <= 256 ? one : two))
                            : (full > longest ? full : longest);
    return (float)n * stage + (s > 1 ? 3.f + join * (float)w : 0.f);
  }
};
constexpr float kShares[2][2] = {{1.f, 0.7f}, {0.5f, 0.35f}};  // causal, lengths
// The number of ranges that takes least (of many, every eighth part more is tried).
inline int best_split(int64_t blocks, int64_t stages, float share, const SplitCost& c, float& least) {
  int best = 1;
  least = c.time(blocks, stages, 1, share);
  for (int64_t s = 2; blocks * s <= c.most && stages >= s * c.least; s += s < 16 ? 1 : s / 8) {
    const float t = c.time(blocks, stages, s, share);
    if (t < least) least = t, best = (int)s;
  }
  return best;
}

}  // namespace sla2h
