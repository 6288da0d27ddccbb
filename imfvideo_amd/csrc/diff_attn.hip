// Differential attention, forward, gfx950: a pair p of heads (2p, 2p + 1) attends twice with the same
// 128 value channels (value heads 2p and 2p + 1 side by side),
//
//   A_m = softmax(c q_m k_m^T) (m = 1, 2; keys j < k_len, causal: j <= i + k_len - q_len),
//   o = (A_1 - lam_p A_2) v;   a row without a key is 0.
//
// One pass over the keys, each map as in dense_attn.hip: O_m^T += V^T P_m^T with P_m = exp2(S - m)
// in 16 bits, row sums of the fp32 values, a bound m that moves only when a tile outgrows it.  The two
// sums meet at the end, when both normalisers are known: six products of 64 channels per (query,
// key) where a second pass over the scores would make it 2 + 2 + 2 and the exponentials twice.
// A wave belongs to one map: it holds 128 channels of its rows' sums and reads its own keys and all
// values; the waves of the other map sit beside it in the workgroup and hand their result over
// through LDS.  (Both maps in one wave would need both maps' queries and twice the sums for the same rows:
// half the rows per value operand read from LDS.)
#include "diff_attn.h"

#include <initializer_list>

namespace sla2h {

namespace {

// What the rounding of P lost is added by a second product for clips of so many units of keys: their rows'
// few large probabilities make delta_m of the backward, and dA - delta_m, which then nearly cancel (2
// keys: dq and dk six times as far off).  And for clips of a few rows of not many keys, whose few
// roundings do not average out in any sum over the rows (two rows of 146 and 248 keys: o 1.5 times as far
// off as its own rounding, 1.05 so; 17 rows of 1,000 keys or 16 of 1,100: 1.04).  The clip's own lengths
// decide, not those that its batch is padded to.
constexpr int kFewUnits = 4, kFineRows = 16, kFineUnits = 32;
__host__ __device__ inline bool fine_clip(int64_t qlen, int64_t klen) {
  return klen <= kFewUnits * kUnitRows || (qlen <= kFineRows && klen <= kFineUnits * kUnitRows);
}

struct DiffFwdArgs {
  const uint16_t *q, *k, *v;
  Weights lam;       // (P)
  uint16_t* o;       // (B, Lq, H, 64)
  float* maps;       // (B, Lq, P, 2, 128): A_m v, or null
  float* lse;        // (B, H, Lq) or null
  const int32_t *q_lens, *k_lens;
  int64_t qb, qh, ql, kb, kh, kl, vb, vh, vl;  // strides in elements
  int64_t Lq, Lk;
  int P, Pk, rep;  // pairs of query heads, of key heads
  int causal;
  float c;  // scale * log2(e)
  WorkMap map;
  int qtiles;
  float* part;   // [range][map][B * P * Lq][128] unnormalised sums
  float2* ml;    // [range][map][B * P * Lq] (m, l)
  int splits, units;  // few queries: 32-key units of a range
  int64_t nrows;      // B * P * Lq
};

// Element of a row's results: pair bp = b P + p, row i.
__device__ inline uint16_t* out_row(const DiffFwdArgs& a, int64_t bp, int64_t i) {
  const int64_t b = bp / a.P, p = bp - b * a.P;
  return a.o + ((b * a.Lq + i) * a.P + p) * 128;
}

// Workgroup = 4 waves: two query groups of 32 NQ rows x two maps, of one pair.  Stages of 32 keys
// (k of both maps, the 128 value channels) three ahead in four LDS slots, one barrier each.  The
// scores of a wave's first 32 rows are one stage ahead, and the products of its last ones with the values
// one behind: every product has exponentials of other numbers to run under (weave).
// FINE (few rows): what the rounding of P lost by a second product.
template <typename T16, int NQ, bool FINE>
__global__ __launch_bounds__(256, 2) void diff_fwd_kernel(DiffFwdArgs a) {
  __shared__ __align__(16) unsigned char s0[kStageB], s1[kStageB], s2[kStageB], s3[kStageB],
      s4[kStageB];
  int bp, item;
  if (!work_item(a.map, blockIdx.x, bp, item)) return;
  const int qt = item / a.splits, sp = item - qt * a.splits;
  const int b = bp / a.P, p = bp - b * a.P, kp = p / a.rep;
  const int tid = threadIdx.x, l = tid & 63, h = l >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), m = w & 1;
  const LaneOff lo(l);
  const int qlen = seq_len(a.q_lens, b, a.Lq), klen = seq_len(a.k_lens, b, a.Lk);

  const int q0 = qt * (64 * NQ);               // first row of the workgroup
  const int qw = q0 + (w >> 1) * (32 * NQ);    // ... of the wave
  const int qend = min(q0 + 64 * NQ, qlen);
  const int kmax = qend > q0 ? key_limit(qend - 1, qlen, klen, a.causal) : 0;
  const int nunit = (kmax + kUnitRows - 1) / kUnitRows;
  const int per = (nunit + a.splits - 1) / a.splits;
  const int t0 = sp * per, nt = min(nunit, t0 + per);  // this range's stages

  // wave w loads the stage's matrix w: k of map 0, of map 1, the lower and the upper value channels
  const uint16_t* src = w < 2 ? a.k + b * a.kb + (2 * kp + w) * a.kh
                              : a.v + b * a.vb + (2 * kp + w - 2) * a.vh;
  const int64_t ld = (w < 2 ? a.kl : a.vl) * 2;
  auto load = [&](int t, unsigned char* s) __attribute__((always_inline)) {
    const int64_t row = (int64_t)t * kUnitRows;
    load_unit(src, row, (int64_t)klen - row, ld, s + w * kUnitB, l);
  };

  u32x4 qf[NQ][4];
  int lim[NQ];
  {
    const uint16_t* qp = a.q + b * a.qb + (2 * p + m) * a.qh;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int i = qw + 32 * n + (l & 31);
      lim[n] = key_limit(i, qlen, klen, a.causal);
#pragma unroll
      for (int s = 0; s < 4; ++s)
        qf[n][s] = i < qlen ? *reinterpret_cast<const u32x4*>(qp + i * a.ql + 16 * s + 8 * h)
                            : u32x4{0, 0, 0, 0};
    }
  }
  // keys that every query of the wave sees, and that any of them sees
  const int wlast = min(qw + 32 * NQ, qlen) - 1;
  const int wany = wlast >= qw ? key_limit(wlast, qlen, klen, a.causal) : 0;
  const int wall = wlast >= qw ? key_limit(qw, qlen, klen, a.causal) : 0;

  f32x16 acc[NQ][4];
  float mx[NQ], lsum[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
#pragma unroll
    for (int mb = 0; mb < 4; ++mb) acc[n][mb] = zero16();
    mx[n] = kFloor;
    lsum[n] = 0.f;
  }
  f32x16 sc[NQ];
  u32x4 pr[NQ][2], lo_[2];
  auto scores = [&](int n, const unsigned char* s) __attribute__((always_inline)) {
    sc[n] = zero16();
#pragma unroll
    for (int x = 0; x < 4; ++x)
      sc[n] = mfma_32x32x16<T16>(row_frag(s + m * kUnitB, 0, x, lo), qf[n][x], sc[n]);
  };
  auto mask = [&](int n, int base) __attribute__((always_inline)) {
    if (base + kUnitRows > wall) {
      asm volatile("");  // a branch: rare, and 16 selects when speculated
      mask_tile(sc[n], lim[n] - base, h);
    }
  };
  // rows n again under a new bound
  auto again = [&](int n, int base, const unsigned char* cur) __attribute__((always_inline)) {
    const f32x16 ahead = sc[n];  // (NQ = 1: the next stage's)
    scores(n, cur);
    mask(n, base);
    raise_bound(lane_max(sc[n]), a.c, mx[n], lsum[n], acc[n]);
    float r = 0.f;
    if (FINE) {
      const float off = Range<T16>::shift - mx[n];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float x = fast_exp2(__builtin_fmaf(sc[n][2 * k], a.c, off));
        const float y = fast_exp2(__builtin_fmaf(sc[n][2 * k + 1], a.c, off));
        uint32_t word = pack_pair<T16>(x, y);
        asm volatile("" : "+v"(word));
        r += x + y;
        pr[n][k >> 2][k & 3] = word;
        lo_[k >> 2][k & 3] = pack_pair<T16>(x - T16::to_f32((uint16_t)(word & 0xffff)),
                                            y - T16::to_f32((uint16_t)(word >> 16)));
      }
    } else {
      r = probabilities<T16>(sc[n], a.c, mx[n], pr[n]);
    }
    if (NQ == 1) sc[n] = ahead;
    return r;
  };
  auto value = [&](int j, const unsigned char* s) __attribute__((always_inline)) {
    return col_frag(s + (2 + ((j & 3) >> 1)) * kUnitB, 16 * (j >> 2), j & 1, lo);
  };
  auto values = [&](int n, const unsigned char* s) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const u32x4 v = value(j, s);
      acc[n][j & 3] = mfma_32x32x16<T16>(v, pr[n][j >> 2], acc[n][j & 3]);
      if (FINE) acc[n][j & 3] = mfma_32x32x16<T16>(v, lo_[j >> 2], acc[n][j & 3]);
    }
  };
  // Half a stage: rows ns's scores of the keys in `ks`, rows nv's products with the values in `vs`, among
  // rows ne's exponentials; returns their sum.  Twelve products, their LDS operands read two products
  // ahead, each beside a share of the exponentials that covers its 32 cycles.  The order is fixed: left
  // to the compiler the products come first, each behind its operand, and the exponentials after them
  // (7 % more cycles).
  auto weave = [&](auto ns_, const unsigned char* ks, auto nv_, const unsigned char* vs, auto ne_)
      __attribute__((always_inline)) {
    constexpr int ns = decltype(ns_)::value, nv = decltype(nv_)::value, ne = decltype(ne_)::value;
    u32x4 f[3], next[2], lost[2];
    auto operand = [&](int i) __attribute__((always_inline)) {
      return i % 3 == 0 ? row_frag(ks + m * kUnitB, 0, i / 3, lo) : value(i / 3 * 2 + i % 3 - 1, vs);
    };
    const float off = Range<T16>::shift - mx[ne];
    float r[2] = {0.f, 0.f};
    f32x16 z = zero16();
    f[0] = operand(0);
    f[1] = operand(1);
#pragma unroll
    for (int i = 0; i < 12; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      if (i + 2 < 12) f[(i + 2) % 3] = operand(i + 2);
      if (i % 3 == 0) {
        z = mfma_32x32x16<T16>(f[i % 3], qf[ns][i / 3], z);
      } else {
        const int j = i / 3 * 2 + i % 3 - 1;
        acc[nv][j & 3] = mfma_32x32x16<T16>(f[i % 3], pr[nv][j >> 2], acc[nv][j & 3]);
        if (FINE) acc[nv][j & 3] = mfma_32x32x16<T16>(f[i % 3], lo_[j >> 2], acc[nv][j & 3]);
      }
      if (i % 3 < 2) {  // scores 2 k, 2 k + 1
        const int k = i / 3 * 2 + i % 3;
        const float x = fast_exp2(__builtin_fmaf(sc[ne][2 * k], a.c, off));
        const float y = fast_exp2(__builtin_fmaf(sc[ne][2 * k + 1], a.c, off));
        uint32_t word = pack_pair<T16>(x, y);
        r[0] += x;
        r[1] += y;
        asm volatile("" : "+v"(word), "+v"(r[0]), "+v"(r[1]));  // here, not behind the products
        next[k >> 2][k & 3] = word;
        if (FINE) {
          uint32_t rest = pack_pair<T16>(x - T16::to_f32((uint16_t)(word & 0xffff)),
                                         y - T16::to_f32((uint16_t)(word >> 16)));
          asm volatile("" : "+v"(rest));
          lost[k >> 2][k & 3] = rest;
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    sc[ns] = z;
    pr[ne][0] = next[0];
    pr[ne][1] = next[1];
    if (FINE) lo_[0] = lost[0], lo_[1] = lost[1];
    return r[0] + r[1];
  };
  constexpr std::integral_constant<int, 0> first{};
  constexpr std::integral_constant<int, NQ - 1> other{};
  auto stage = [&](int t, const unsigned char* prev, const unsigned char* cur,
                   const unsigned char* nxt, unsigned char* to) __attribute__((always_inline)) {
    // the stages up to t + 1 have landed, stage t - 2 is read
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(4));
    __builtin_amdgcn_s_barrier();
    load(t + 3, to);
    const int base = t * kUnitRows;
    mask(0, base);
    float r = NQ == 2 ? weave(other, cur, other, prev, first) : weave(first, nxt, first, prev, first);
    if (__builtin_amdgcn_ballot_w64(r > Range<T16>::most)) r = again(0, base, cur);
    lsum[0] += r;
    if (NQ == 2) {
      mask(NQ - 1, base);
      r = weave(first, nxt, first, cur, other);
      if (__builtin_amdgcn_ballot_w64(r > Range<T16>::most)) r = again(NQ - 1, base, cur);
      lsum[NQ - 1] += r;
    }
  };
  load(t0, s0);
  load(t0 + 1, s1);
  load(t0 + 2, s2);
  __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(8));
  __builtin_amdgcn_s_barrier();
  scores(0, s0);
#pragma unroll
  for (int n = 0; n < NQ; ++n) pr[n][0] = pr[n][1] = lo_[0] = lo_[1] = u32x4{0, 0, 0, 0};
  // The first stage adds what its own slot holds with probabilities of 0; the other rows of the
  // last stage that the wave has keys in come behind the loop, and then the waits and loads alone.
  const int wn = min(nt, (wany + kUnitRows - 1) / kUnitRows);
  const unsigned char* last = s0;
  auto slot_of = [&](int t) __attribute__((always_inline)) {
    const int x = (t - t0) % 5;
    return x == 0 ? s0 : x == 1 ? s1 : x == 2 ? s2 : x == 3 ? s3 : s4;
  };
  if (NQ == 1 && !FINE && fine_clip(qlen, klen)) {  // a short clip in a padded batch, stage after stage
    for (int t = t0; t < nt; ++t) {
      __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(4));
      __builtin_amdgcn_s_barrier();
      load(t + 3, slot_of(t + 3));
      if (t >= wn) continue;
      const unsigned char* s = slot_of(t);
      scores(0, s);
      mask_tile(sc[0], lim[0] - t * kUnitRows, h);
      raise_bound(lane_max(sc[0]), a.c, mx[0], lsum[0], acc[0]);
      lsum[0] += probabilities<T16>(sc[0], a.c, mx[0], pr[0]);
      lost_halves<T16>(sc[0], a.c, mx[0], pr[0], lo_);
      values(0, s);
      pr[0][0] = lo_[0], pr[0][1] = lo_[1];
      values(0, s);
    }
  } else {
    for (int t = t0; t < wn; t += 5) {
      stage(t, t == t0 ? s0 : s4, s0, s1, s3);
      last = s0;
      if (t + 1 >= wn) break;
      stage(t + 1, s0, s1, s2, s4);
      last = s1;
      if (t + 2 >= wn) break;
      stage(t + 2, s1, s2, s3, s0);
      last = s2;
      if (t + 3 >= wn) break;
      stage(t + 3, s2, s3, s4, s1);
      last = s3;
      if (t + 4 >= wn) break;
      stage(t + 4, s3, s4, s0, s2);
      last = s4;
    }
    values(NQ - 1, last);
    for (int t = max(wn, t0); t < nt; ++t) {
      __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(4));
      __builtin_amdgcn_s_barrier();
      load(t + 3, slot_of(t + 3));
    }
  }
  __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));  // no load into this LDS outlives the workgroup

  float inv[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int i = qw + 32 * n + (l & 31);
    const float ls = swap32_sum(lsum[n]);
    if (a.splits > 1) {
      if (i >= a.Lq) continue;
      const int64_t flat = (sp * 2 + m) * a.nrows + (int64_t)bp * a.Lq + i;
#pragma unroll
      for (int mb = 0; mb < 4; ++mb)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(a.part + flat * 128 + 32 * mb + 8 * g + 4 * h) =
              f32x4{acc[n][mb][4 * g], acc[n][mb][4 * g + 1], acc[n][mb][4 * g + 2],
                    acc[n][mb][4 * g + 3]};
      if (h == 0) a.ml[flat] = make_float2(mx[n], ls);
      continue;
    }
    inv[n] = 1.f / ls;  // a row whose scores are all -inf is NaN
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[n][mb][e] = lim[n] > 0 ? acc[n][mb][e] * inv[n] : 0.f;
    if (i >= a.Lq) continue;
    if (a.maps) {
      float* d = a.maps + ((((int64_t)b * a.Lq + i) * a.P + p) * 2 + m) * 128;
#pragma unroll
      for (int mb = 0; mb < 4; ++mb)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(d + 32 * mb + 8 * g + 4 * h) =
              f32x4{acc[n][mb][4 * g], acc[n][mb][4 * g + 1], acc[n][mb][4 * g + 2],
                    acc[n][mb][4 * g + 3]};
    }
    if (a.lse && h == 0)
      a.lse[((int64_t)b * 2 * a.P + 2 * p + m) * a.Lq + i] =
          lim[n] > 0 ? (mx[n] - Range<T16>::shift + __log2f(ls)) * kLn2 : -__builtin_inff();
  }
  if (a.splits > 1) return;

  // map 1's rows through LDS: 16 KB per 32 rows, quads of channels of all rows beside each other
  __syncthreads();
  auto slot = [&](int n) __attribute__((always_inline)) {
    const int x = (w >> 1) * NQ + n;
    return reinterpret_cast<f32x4*>(x == 0 ? s0 : x == 1 ? s1 : x == 2 ? s2 : s3);
  };
  if (m == 1) {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      f32x4* x = slot(n);
#pragma unroll
      for (int mb = 0; mb < 4; ++mb)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          x[(8 * mb + 2 * g + h) * 32 + (l & 31)] = f32x4{acc[n][mb][4 * g], acc[n][mb][4 * g + 1],
                                                          acc[n][mb][4 * g + 2], acc[n][mb][4 * g + 3]};
    }
  }
  __syncthreads();
  if (m == 1) return;
  const float lam = a.lam[p];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int i = qw + 32 * n + (l & 31);
    if (i >= a.Lq) continue;
    const f32x4* x = slot(n);
    uint16_t* d = out_row(a, bp, i);
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 y = x[(8 * mb + 2 * g + h) * 32 + (l & 31)];
        float z[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          z[e] = lim[n] > 0 ? __builtin_fmaf(-lam, y[e], acc[n][mb][4 * g + e]) : 0.f;
        *reinterpret_cast<u32x2*>(d + 32 * mb + 8 * g + 4 * h) =
            u32x2{pack_pair<T16>(z[0], z[1]), pack_pair<T16>(z[2], z[3])};
      }
  }
}

// Writes eight channels of a finished row: o, and for a backward the maps' rows and log-sum-exps.
template <typename T16>
__device__ inline void finish_row(const DiffFwdArgs& a, int64_t bp, int64_t i, int c0, bool some,
                                  const float (&x)[2][8], const float (&mm)[2],
                                  const float (&ll)[2]) {
  const int64_t b = bp / a.P, p = bp - b * a.P;
  const float lam = a.lam[p];
  float y[2][8];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const float inv = 1.f / ll[m];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[m][e] = some ? x[m][e] * inv : 0.f;
    if (a.maps) {
      float* d = a.maps + (((b * a.Lq + i) * a.P + p) * 2 + m) * 128 + c0;
      *reinterpret_cast<f32x4*>(d) = f32x4{y[m][0], y[m][1], y[m][2], y[m][3]};
      *reinterpret_cast<f32x4*>(d + 4) = f32x4{y[m][4], y[m][5], y[m][6], y[m][7]};
    }
    if (a.lse && c0 == 0)
      a.lse[(b * 2 * a.P + 2 * p + m) * a.Lq + i] =
          some ? (mm[m] - Range<T16>::shift + __log2f(ll[m])) * kLn2 : -__builtin_inff();
  }
  u32x4 z;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    z[e] = some ? pack_pair<T16>(__builtin_fmaf(-lam, y[1][2 * e], y[0][2 * e]),
                                 __builtin_fmaf(-lam, y[1][2 * e + 1], y[0][2 * e + 1]))
                : 0u;
  *reinterpret_cast<u32x4*>(out_row(a, bp, i) + c0) = z;
}

// Few queries of grouped heads, or few keys: workgroup = 32 rows of the `rep` query pairs that share a
// key pair, over one range of keys; its four waves take the 32-key units in turn, both maps of a unit,
// each with an LDS slot of its own (no barrier in the loop), and their sums are joined in LDS.  A wave
// waits for its unit and computes it while the others' units are on their way (eight waves, one
// workgroup per CU: no faster).  The products wait for the loads here, so what the rounding of P lost
// is always added by a second one.
constexpr int W = 4;  // waves
template <typename T16>
__global__ __launch_bounds__(64 * W, 2) void diff_fwd_split_kernel(DiffFwdArgs a) {
  __shared__ __align__(16) unsigned char kv[W][kStageB];
  __shared__ float mls[W][2][2][32];  // wave, map, (m, l)
  const int blk = blockIdx.x / a.splits, sp = blockIdx.x - blk * a.splits;
  const int bk = __builtin_amdgcn_readfirstlane(blk / a.qtiles);
  const int qt = __builtin_amdgcn_readfirstlane(blk - bk * a.qtiles);
  const int b = bk / a.Pk, kp = bk - b * a.Pk;
  const int tid = threadIdx.x, l = tid & 63, h = l >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const LaneOff lo(l);
  const int qlen = seq_len(a.q_lens, b, a.Lq), klen = seq_len(a.k_lens, b, a.Lk);

  // row of the group: pair kp rep + row / Lq, query row % Lq
  // (fewer than 2^31 of them: 32-bit divisions)
  const uint32_t lq = (uint32_t)a.Lq, rows = (uint32_t)a.rep * lq;
  const uint32_t row = (uint32_t)qt * 32 + (l & 31), rq = row / lq;
  const bool live = row < rows;
  const int p = kp * a.rep + (live ? (int)rq : 0);
  const int i = live ? (int)(row - rq * lq) : 0;
  const int lim = live ? key_limit(i, qlen, klen, a.causal) : 0;
  int kmax = lim, kmin = lim;
#pragma unroll
  for (int s = 16; s >= 1; s >>= 1) {
    kmax = max(kmax, __shfl_xor(kmax, s, 64));
    kmin = min(kmin, __shfl_xor(kmin, s, 64));
  }
  kmax = __builtin_amdgcn_readfirstlane(kmax);
  kmin = __builtin_amdgcn_readfirstlane(kmin);

  const int64_t u0 = (int64_t)sp * a.units;
  const int64_t uend = min(u0 + a.units, ((int64_t)kmax + kUnitRows - 1) / kUnitRows);
  auto load = [&](int64_t u) __attribute__((always_inline)) {
    const int64_t n = u < uend ? (int64_t)klen - u * kUnitRows : 0;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      load_unit(a.k + b * a.kb + (2 * kp + x) * a.kh, u * kUnitRows, n, a.kl * 2, kv[w] + x * kUnitB,
                l);
      load_unit(a.v + b * a.vb + (2 * kp + x) * a.vh, u * kUnitRows, n, a.vl * 2,
                kv[w] + (2 + x) * kUnitB, l);
    }
  };
  int64_t u = u0 + w;
  load(u);

  u32x4 qf[2][4];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const uint16_t* qp = a.q + b * a.qb + (2 * p + m) * a.qh + i * a.ql;
#pragma unroll
    for (int s = 0; s < 4; ++s)
      qf[m][s] = lim > 0 ? *reinterpret_cast<const u32x4*>(qp + 16 * s + 8 * h) : u32x4{0, 0, 0, 0};
  }
  f32x16 acc[2][4];
  float mx[2], lsum[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
#pragma unroll
    for (int mb = 0; mb < 4; ++mb) acc[m][mb] = zero16();
    mx[m] = kFloor;
    lsum[m] = 0.f;
  }
  for (; u < uend; u += W) {
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));
    const unsigned char* s = kv[w];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      f32x16 sc = zero16();
#pragma unroll
      for (int x = 0; x < 4; ++x)
        sc = mfma_32x32x16<T16>(row_frag(s + m * kUnitB, 0, x, lo), qf[m][x], sc);
      if (u * kUnitRows + kUnitRows > kmin) mask_tile(sc, (int)(lim - u * kUnitRows), h);
      // the wave's first unit sets the bound of the rows that see a key of it
      u32x4 pr[2], lost[2];
      float r = probabilities<T16>(sc, a.c, mx[m], pr);
      if (__builtin_amdgcn_ballot_w64(r > Range<T16>::most)) {
        raise_bound(lane_max(sc), a.c, mx[m], lsum[m], acc[m]);
        r = probabilities<T16>(sc, a.c, mx[m], pr);
      }
      lsum[m] += r;
      lost_halves<T16>(sc, a.c, mx[m], pr, lost);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) {
          const u32x4 vf = col_frag(s + (2 + (mb >> 1)) * kUnitB, 16 * x, mb & 1, lo);
          acc[m][mb] = mfma_32x32x16<T16>(vf, pr[x], acc[m][mb]);
          acc[m][mb] = mfma_32x32x16<T16>(vf, lost[x], acc[m][mb]);
        }
    }
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));  // the reads of this slot are done
    load(u + W);
  }
  __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));

  // join the waves, map by map: fp32 O^T tiles [channel][row] in the slots' memory
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const float ls = swap32_sum(lsum[m]);
    if (h == 0) {
      mls[w][m][0][l] = mx[m];
      mls[w][m][1][l] = ls;
    }
  }
  // thread: row tid % 32, channels 8 c8 .., 128 / (2 W) groups of them in turn
  const int r = tid & 31;
  // (row r of the tile is lane r's, in every wave)
  const bool mine = live;
  const int64_t op = (int64_t)b * a.P + p, oi = i, flat = op * a.Lq + oi;
  constexpr int NG = 8 / W;  // groups of eight channels of a thread
  float mm[2], ll[2], x[2][NG][8];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    if (m) __syncthreads();
    float* ot = reinterpret_cast<float*>(kv[w]);
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        ot[(32 * mb + 8 * (e >> 2) + 4 * h + (e & 3)) * 32 + (l & 31)] = acc[m][mb][e];
    __syncthreads();
    mm[m] = kFloor;
#pragma unroll
    for (int j = 0; j < W; ++j) mm[m] = fmaxf(mm[m], mls[j][m][0][r]);
    ll[m] = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[m][g][e] = 0.f;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const float f = fast_exp2(mls[j][m][0][r] - mm[m]);
      ll[m] += f * mls[j][m][1][r];
      const float* src = reinterpret_cast<const float*>(kv[j]);
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x[m][g][e] += f * src[((g * 2 * W + (tid >> 5)) * 8 + e) * 32 + r];
    }
  }
  if (!mine) return;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const int c0 = (g * 2 * W + (tid >> 5)) * 8;
    if (a.splits == 1) {
      const float y[2][8] = {{x[0][g][0], x[0][g][1], x[0][g][2], x[0][g][3], x[0][g][4], x[0][g][5],
                              x[0][g][6], x[0][g][7]},
                             {x[1][g][0], x[1][g][1], x[1][g][2], x[1][g][3], x[1][g][4], x[1][g][5],
                              x[1][g][6], x[1][g][7]}};
      finish_row<T16>(a, op, oi, c0, key_limit((int)oi, qlen, klen, a.causal) > 0, y, mm, ll);
      continue;
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float* d = a.part + ((sp * 2 + m) * a.nrows + flat) * 128 + c0;
      *reinterpret_cast<f32x4*>(d) = f32x4{x[m][g][0], x[m][g][1], x[m][g][2], x[m][g][3]};
      *reinterpret_cast<f32x4*>(d + 4) = f32x4{x[m][g][4], x[m][g][5], x[m][g][6], x[m][g][7]};
      if (c0 == 0) a.ml[(sp * 2 + m) * a.nrows + flat] = make_float2(mm[m], ll[m]);
    }
  }
}

// Joins the key ranges of a row, many rows: 16 lanes for each map (eight channels per lane) take the
// ranges one after the other, eight rows per workgroup.
template <typename T16>
__global__ __launch_bounds__(256) void diff_join_rows_kernel(DiffFwdArgs a) {
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int64_t flat = row < a.nrows ? row : a.nrows - 1;
  const int m = (threadIdx.x >> 4) & 1, c0 = (threadIdx.x & 15) * 8;
  float t[2][8], mm[2], ll[2];
  float top = kFloor, sum = 0.f;
  f32x4 x{0.f, 0.f, 0.f, 0.f}, y = x;
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const int64_t at = (s * 2 + m) * a.nrows + flat;
    const float2 ml = a.ml[at];
    const f32x4* src = reinterpret_cast<const f32x4*>(a.part + at * 128 + c0);
    const f32x4 p0 = src[0], p1 = src[1];
    const float mn = fmaxf(top, ml.x), f = fast_exp2(top - mn), g = fast_exp2(ml.x - mn);
    top = mn;
    sum = sum * f + g * ml.y;
    x = x * f + g * p0;
    y = y * f + g * p1;
  }
  // the second map's lanes hand theirs over
  mm[0] = top, ll[0] = sum;
  mm[1] = __shfl_xor(top, 16, 64);
  ll[1] = __shfl_xor(sum, 16, 64);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    t[0][e] = e < 4 ? x[e & 3] : y[e & 3];
    t[1][e] = __shfl_xor(t[0][e], 16, 64);
  }
  if (m || row >= a.nrows) return;
  const int64_t bp = flat / a.Lq, i = flat - bp * a.Lq;
  const int b = (int)(bp / a.P);
  // (the halves of a wave may be of two clips: seq_len would take the first one's)
  auto len = [&](const int32_t* lens, int64_t L) {
    const int n = lens ? lens[b] : (int)L;
    return n < 0 ? 0 : (n > L ? (int)L : n);
  };
  finish_row<T16>(a, bp, i, c0,
                  key_limit((int)i, len(a.q_lens, a.Lq), len(a.k_lens, a.Lk), a.causal) > 0, t, mm, ll);
}

// Few rows and many ranges: a workgroup per row, 64 groups of 16 lanes, 32 for each map, take the
// ranges in turn, and their sums are added in order.
template <typename T16>
__global__ __launch_bounds__(1024) void diff_join_kernel(DiffFwdArgs a) {
  __shared__ float sm[2][32], sl[2][32];
  __shared__ f32x4 sx[2][32][32];
  const int64_t flat = blockIdx.x;
  const int m = threadIdx.x >> 9, grp = (threadIdx.x >> 4) & 31, c0 = (threadIdx.x & 15) * 8;
  const int64_t bp = flat / a.Lq, i = flat - bp * a.Lq;
  const int b = (int)(bp / a.P);
  float mm = kFloor, ll = 0.f;
  f32x4 x{0.f, 0.f, 0.f, 0.f}, y = x;
#pragma unroll 2
  for (int s = grp; s < a.splits; s += 32) {
    const int64_t at = (s * 2 + m) * a.nrows + flat;
    const float2 ml = a.ml[at];
    const f32x4* src = reinterpret_cast<const f32x4*>(a.part + at * 128 + c0);
    const f32x4 p0 = src[0], p1 = src[1];
    const float mn = fmaxf(mm, ml.x), f = fast_exp2(mm - mn), g = fast_exp2(ml.x - mn);
    mm = mn;
    ll = ll * f + g * ml.y;
    x = x * f + g * p0;
    y = y * f + g * p1;
  }
  sx[m][grp][c0 / 4] = x;
  sx[m][grp][c0 / 4 + 1] = y;
  if (c0 == 0) sm[m][grp] = mm, sl[m][grp] = ll;
  __syncthreads();
  if (threadIdx.x >= 64) return;  // one wave: lane j of each half the weight of group j
  const int qlen = seq_len(a.q_lens, b, a.Lq), klen = seq_len(a.k_lens, b, a.Lk);
  const int k0 = threadIdx.x >> 5, j0 = threadIdx.x & 31;
  float top = sm[k0][j0];
#pragma unroll
  for (int s = 16; s >= 1; s >>= 1) top = fmaxf(top, __shfl_xor(top, s, 64));
  const float weight = fast_exp2(sm[k0][j0] - top);
  float all = weight * sl[k0][j0];
#pragma unroll
  for (int s = 16; s >= 1; s >>= 1) all += __shfl_xor(all, s, 64);
  sm[k0][j0] = weight;
  __builtin_amdgcn_wave_barrier();  // (read by this wave alone)
  const float tm[2] = {__shfl(top, 0, 64), __shfl(top, 32, 64)};
  const float tl[2] = {__shfl(all, 0, 64), __shfl(all, 32, 64)};
  if (threadIdx.x >= 16) return;
  float t[2][8];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int e = 0; e < 8; ++e) t[k][e] = 0.f;
#pragma unroll 8
    for (int j = 0; j < 32; ++j) {
      const float f = sm[k][j];
      const f32x4 p0 = sx[k][j][c0 / 4], p1 = sx[k][j][c0 / 4 + 1];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        t[k][e] += f * p0[e];
        t[k][4 + e] += f * p1[e];
      }
    }
  }
  finish_row<T16>(a, bp, i, c0, key_limit((int)i, qlen, klen, a.causal) > 0, t, tm, tl);
}

// The form of a call: query blocks of 128 or 64 rows, over all keys or ranges of them; or the one tile
// of 32 rows of a key pair's group.
struct FwdPlan {
  int nq;  // 2, 1: diff_fwd_kernel<NQ>; 0: diff_fwd_split_kernel
  bool fine;  // nq = 1
  int64_t qtiles, nwork;
  int splits;  // ranges of keys
  int64_t units;  // nq = 0: 32-key units of a range
};

FwdPlan fwd_plan(int B, int H, int Hkv, int64_t Lq, int64_t Lk, bool causal, bool lens) {
  FwdPlan p{};
  const int64_t bp = (int64_t)B * H / 2, bk = (int64_t)B * Hkv / 2, rep = H / Hkv;
  const int64_t units = (Lk + kUnitRows - 1) / kUnitRows;
  const float share = kShares[causal][lens];
  // A group's rows in one tile read their keys once (us, in this form / in query blocks: 64 clips, H = 16,
  // Hkv = 2, 1 query, 2,000 keys 23 / 64; 1 clip, 29,952 keys 18 / 27; 32 clips, 32, 4, 4 queries
  // 27 / 48; in two tiles and more: 8 clips, 16, 2, 16 queries 20 / 18), and so do calls of few keys, with
  // their second product (100 of 100 keys 10 / 8 us without it).
  if (units <= kFewUnits || (rep > 1 && rep * Lq <= 32)) {
    p.qtiles = (rep * Lq + 31) / 32;
    const int64_t blocks = bk * p.qtiles;
    const int64_t s = 512 / blocks, most = units / 8;  // two units per wave and range at least
    p.splits = (int)(s < 1 || most < 1 ? 1 : (s < most ? s : most));
    p.units = (units + p.splits - 1) / p.splits;
    p.splits = (int)((units + p.units - 1) / p.units);
    p.nwork = blocks * p.splits;
    return p;
  }
  // 128 rows (no ranges; not where lengths may leave few keys) or 64, by what a stage takes (SplitCost)
  // with one and two workgroups per CU.  us, 128 / 64, H = 8: 1 clip of 8,192 231 / 208, of 12,000 476 / 479, of 16,384 738 / 809, 4 clips of
  // 2,048, H = 16, 106 / 113; causal 12,000 334 / 244, 24,000 831 / 870.
  const int64_t q2 = (Lq + 127) / 128, q1 = (Lq + 63) / 64;
  const SplitCost c2{0.88f, 1.43f, 0.f, 0};
  SplitCost c1{0.53f, 0.74f, 0.033f, 4};
  if (q1 == 1) {
    // One block of queries reads every key from memory, and 256 workgroups are all that it feeds (us for 2
    // clips, H = 8, 1 query, 29,952 keys and fewer: 192 27, 256 25, 320 to 512 26 to 28, more 30 to 34);
    // its partial sums are few.
    c1.most = 256;
    c1.join *= (float)Lq / 64.f;
  }
  float t1;
  p.splits = best_split(bp * q1, units, share, c1, t1);
  p.nq = !lens && c2.time(bp * q2, units, 1, share) < t1 ? 2 : 1;
  if (p.nq == 2) p.splits = 1;
  p.qtiles = p.nq == 2 ? q2 : q1;
  p.nwork = bp * p.qtiles;
  // (all clips of the call: one body for it.  us without / with the second products, 8 heads, 1 query:
  // 1,000 keys 10.1 / 10.8, 64 clips of 1,000 26.3 / 28.7; of 29,952 keys it would be 19.8 / 21.8)
  p.fine = p.nq == 1 && fine_clip(Lq, Lk);
  return p;
}

}  // namespace

}  // namespace sla2h

using namespace sla2h;

extern "C" size_t sla2h_diff_attn_fwd_workspace_bytes(int B, int H, int Hkv, int64_t Lq,
                                                      int64_t Lk) {
  if (!diff_sizes_ok(B, H, Hkv, Lq, Lk)) return 0;
  size_t most = 0;
  for (int i = 0; i < 4; ++i) {
    const FwdPlan p = fwd_plan(B, H, Hkv, Lq, Lk, i & 1, i & 2);
    const size_t n = p.splits > 1 ? (size_t)p.splits * B * H * Lq * (128 * 4 + 8) : 0;
    most = n > most ? n : most;
  }
  return most;
}

extern "C" int sla2h_diff_attn_fwd(const void* q, const void* k, const void* v, const void* lam,
                                   int lam_dtype, int64_t lam_stride, const int64_t* strides,
                                   const int32_t* q_lens, const int32_t* k_lens, int dtype, int B, int H, int Hkv,
                                   int64_t Lq, int64_t Lk, int causal, float scale,
                                   void* workspace, void* o, float* lse, float* maps,
                                   void* stream) {
  const Weights wts{lam, lam_dtype, lam_stride};
  SLA2H_CHECK_ARG(q && k && v && wts.ok() && strides && o && !lse == !maps);
  SLA2H_CHECK_ARG(dtype == SLA2H_DTYPE_F16 || dtype == SLA2H_DTYPE_BF16);
  SLA2H_CHECK_ARG(diff_sizes_ok(B, H, Hkv, Lq, Lk));
  SLA2H_CHECK_ARG(scale > 0.f && scale < 1e30f);
  SLA2H_CHECK_ARG(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o | (uintptr_t)maps |
                   (uintptr_t)workspace) % 16 == 0);
  SLA2H_CHECK_ARG(((uintptr_t)lse | (uintptr_t)q_lens | (uintptr_t)k_lens) % 4 == 0);
  for (int i = 0; i < 9; ++i) SLA2H_CHECK_ARG(strides[i] >= 0 && strides[i] % 8 == 0);
  // rows apart from each other: the range check of a tile's load tells them by their offset
  for (int i : {2, 5, 8}) SLA2H_CHECK_ARG(strides[i] >= kDD);
  // 32-bit byte offsets within a tile
  SLA2H_CHECK_ARG(strides[5] < ((int64_t)1 << 23) && strides[8] < ((int64_t)1 << 23));
  const bool even = !causal && !q_lens && !k_lens;
  const FwdPlan p = fwd_plan(B, H, Hkv, Lq, Lk, causal != 0, q_lens || k_lens);
  SLA2H_CHECK_ARG(p.splits == 1 || workspace);
  const int64_t nrows = (int64_t)B * (H / 2) * Lq;
  SLA2H_CHECK_ARG(p.nwork * (p.nq ? p.splits : 1) < ((int64_t)1 << 30));
  SLA2H_CHECK_ARG(p.splits == 1 || nrows < ((int64_t)1 << 31));
  DiffFwdArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.lam = wts;
  a.o = static_cast<uint16_t*>(o);
  a.maps = maps;
  a.lse = lse;
  a.q_lens = q_lens;
  a.k_lens = k_lens;
  a.qb = strides[0], a.qh = strides[1], a.ql = strides[2];
  a.kb = strides[3], a.kh = strides[4], a.kl = strides[5];
  a.vb = strides[6], a.vh = strides[7], a.vl = strides[8];
  a.Lq = Lq;
  a.Lk = Lk;
  a.P = H / 2;
  a.Pk = Hkv / 2;
  a.rep = H / Hkv;
  a.causal = causal != 0;
  a.c = scale * kLog2e;
  a.qtiles = (int)p.qtiles;
  a.map = work_map((int64_t)B * a.P, p.qtiles * (p.nq ? p.splits : 1), even, causal);
  a.splits = p.splits;
  a.units = (int)p.units;
  a.nrows = nrows;
  if (p.splits > 1) {
    a.part = static_cast<float*>(workspace);
    a.ml = reinterpret_cast<float2*>(a.part + (int64_t)p.splits * 2 * a.nrows * 128);
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto go = [&](auto tag) -> int {
    using T16 = decltype(tag);
    if (p.nq == 2)
      diff_fwd_kernel<T16, 2, false><<<work_grid(a.map), 256, 0, st>>>(a);
    else if (p.fine)
      diff_fwd_kernel<T16, 1, true><<<work_grid(a.map), 256, 0, st>>>(a);
    else if (p.nq == 1)
      diff_fwd_kernel<T16, 1, false><<<work_grid(a.map), 256, 0, st>>>(a);
    else
      diff_fwd_split_kernel<T16><<<(unsigned)p.nwork, 256, 0, st>>>(a);
    const int err = (int)hipGetLastError();
    if (err || p.splits == 1) return err;
    // (us: 4 rows, 64 ranges 14 / 4; 2,000 rows of 4 pairs, 2 ranges 10 / 40)
    if (a.nrows >= 512 || p.splits <= 8)
      diff_join_rows_kernel<T16><<<(unsigned)((a.nrows + 7) / 8), 256, 0, st>>>(a);
    else
      diff_join_kernel<T16><<<(unsigned)a.nrows, 1024, 0, st>>>(a);
    return (int)hipGetLastError();
  };
  return dtype == SLA2H_DTYPE_BF16 ? go(BF16{}) : go(F16{});
}
