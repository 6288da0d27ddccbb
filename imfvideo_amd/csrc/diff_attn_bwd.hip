// Backward of differential attention, gfx950.  The two maps of a pair are recomputed from the
// rows' log-sum-exps; with the values' 128 channels v and dA = do v^T, delta_m = do . A_m v:
//
//   dS_1 = A_1 (dA - delta_1), dS_2 = -lam A_2 (dA - delta_2),
//   dq_m = scale dS_m k_m,  dk_m = scale dS_m^T q_m,  dv = (A_1 - lam A_2)^T do,
//   dlam = -sum delta_2     (dk, dv summed over the query pairs of a key pair).
//
// Both maps share dA, and the combined map has one product with do: a wave holds both.  The
// launches: the rows' delta; dk and dv with a workgroup per key block (queries streamed through
// LDS); dq with a workgroup per query block (keys streamed) and, in workgroups of its own, the sum of
// dlam; where ranges of an axis are computed apart, their sum.  14 products of 64 channels per (query, key) where one fused pass has 10, but no sum goes through
// atomics or memory: the result does not depend on the order of dispatch.
//
// fp16 operands: maps (down to 1 / length) and dS would fall below fp16's normal range, so the
// exponents take + shift, where 2^shift (1 + |lam|) is at most 2^15, and dA - delta a power of two from
// |dA - delta| <= 2 max|do_i| max|v_j| (row norms, per key pair, times |lam| where that is above
// one), which brings |dS| below 2^15; both are taken out of the fp32 sums again.  bf16 has
// fp32's range and needs neither.
#include "diff_attn.h"

#include <initializer_list>

namespace sla2h {

namespace {

template <typename T16>
struct Scaled {
  static constexpr bool value = false;
};
template <>
struct Scaled<F16> {
  static constexpr bool value = true;
};

// What the rounding of dS to 16 bits lost is added by a second product.  dq (its rounding alone would
// make it 1.5 times as far off as a rounded exact result): in all stages of sequences of at most
// kFineKeys keys or kFineRows queries and of causal waves that see at most kFineRows keys, else in
// every second stage (1.25 times; B = 1, H = 8, L = 29,952: 0.4 ms).  dk, dv: clips of at most
// kFineSums rows per key pair, or of one block of keys, whose few large probabilities round alike in
// row after row; longer sums average the roundings out (dk without them, in units of its own rounding, not
// causal / causal: 130 rows 1.37 / 1.42, 600 1.27 / 1.34, 2,000 1.13 / 1.23, with them 1.00 to 1.04).  A
// clip's own lengths decide, whatever its batch is padded to.  us for the backward of 8 heads without / with
// them: 1,000 tokens 36 / 41, 16 clips of 1,000 176 / 199, eight of 100 to 2,000 250 / 293.
constexpr int kFineKeys = 4096, kFineRows = 512, kFineSums = 2048;
constexpr int kKeyRows = 128;  // keys of a workgroup of dk and dv
__host__ __device__ inline bool fine_clip(int64_t rep, int64_t qlen, int64_t klen) {
  return rep * qlen <= kFineSums || klen <= kKeyRows;
}
constexpr int kNormRows = 64;  // rows of a partial maximum of the norms and of a partial sum of dlam

struct DiffBwdArgs {
  const uint16_t *q, *k, *v, *dout;
  Weights weights;   // (P)
  float* lam;        // (P): the same in fp32, from the first launch
  const float *lse, *maps;
  uint16_t *dq, *dk, *dv;
  void* dlam;        // (P), the weights' type
  const int32_t *q_lens, *k_lens;
  int64_t qb, qh, ql, kb, kh, kl, vb, vh, vl;
  int64_t Lq, Lk;
  int B, P, Pk, rep;
  int causal;
  float c, inv_c, scale;
  float* stat;          // [4][B * P * Lq]: (shift - lse_m log2e) / c, -delta_m
  int64_t nrows;        // B * P * Lq
  float *gmax, *vmax;   // (B, P, nqb), (B, Pk, nkb): largest row norms (fp16)
  float* lsum;          // (B, P, nqb): sums of -delta_2
  int nqb, nkb;
  WorkMap dq_map, kv_map;  // tiles x splits of a query pair, of a key pair
  int dq_splits, kv_splits, dq_blocks, kv_blocks;
  float *dq_part, *dk_part, *dv_part;
};

// Queries [first, qlen) see a key.
__device__ inline int first_query(int qlen, int klen, int causal) {
  if (klen == 0) return qlen;
  return causal && qlen > klen ? qlen - klen : 0;
}

// fp16: the exponents' shift of a key pair's group, with 2^shift (1 + |lam|) <= 2^15 for its weights.
__device__ inline float power_of_two(int e) { return __builtin_bit_cast(float, (127 + e) << 23); }
// e with x < 2^e, in [-100, 100]
__device__ inline int exponent(float x) {
  int e;
  (void)frexpf(x, &e);
  e = e < -100 ? -100 : (e > 100 ? 100 : e);
  return __builtin_amdgcn_readfirstlane(e);
}
__device__ inline float top_weight(const DiffBwdArgs& a, int kp) {
  float ml = 0.f;
  for (int i = threadIdx.x & 63; i < a.rep; i += 64)
    ml = fmaxf(ml, __builtin_fabsf(a.weights[kp * a.rep + i]));
  return wave_max(ml);
}
__device__ inline int weight_shift(float ml) {
  const float most = 1.f + ml;
  return most < 1e30f ? 15 - exponent(most) : 15;  // 2^(e - 1) <= 1 + |lam| < 2^e
}

// delta of 64 rows of a pair (16 lanes per row), the sum of their -delta_2, and for fp16 the
// largest row norm of do; the workgroups behind them take the norms of v.
template <typename T16>
__global__ __launch_bounds__(256) void diff_bwd_prep_kernel(DiffBwdArgs a, int64_t nq) {
  __shared__ float red[2][4];
  const int tid = threadIdx.x, c0 = (tid & 15) * 8;
  const bool is_v = blockIdx.x >= nq;
  const int64_t blk = is_v ? blockIdx.x - nq : blockIdx.x;
  const int nb = is_v ? a.nkb : a.nqb, pairs = is_v ? a.Pk : a.P;
  const int64_t bp = blk / nb;
  const int t = (int)(blk - bp * nb), b = (int)(bp / pairs), p = (int)(bp - (int64_t)b * pairs);
  const int qlen = seq_len(a.q_lens, b, a.Lq), klen = seq_len(a.k_lens, b, a.Lk);
  const int len = is_v ? klen : qlen;
  const int first = is_v ? 0 : first_query(qlen, klen, a.causal);
  if (blockIdx.x == 0)
    for (int i = tid; i < a.P; i += 256) a.lam[i] = a.weights[i];
  float top = 0.f, sum = 0.f;
  const float shift = Scaled<T16>::value && !is_v ? (float)weight_shift(top_weight(a, p / a.rep)) : 0.f;
#pragma unroll
  for (int j = 0; j < kNormRows / 16; ++j) {
    const int64_t i = (int64_t)t * kNormRows + 16 * j + (tid >> 4);
    const bool live = i >= first && i < len;
    float dot[2] = {0.f, 0.f}, nrm = 0.f;
    if (live) {
      const int64_t at = (((int64_t)b * a.Lq + i) * a.P + p) * 128 + c0;
      const u32x4 g = *reinterpret_cast<const u32x4*>(
          is_v ? a.v + b * a.vb + (2 * p + (c0 >> 6)) * a.vh + i * a.vl + (c0 & 63) : a.dout + at);
      f32x4 o[2][2];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          o[m][x] = is_v ? f32x4{0.f, 0.f, 0.f, 0.f}
                         : *reinterpret_cast<const f32x4*>(a.maps + 2 * (at - c0) + m * 128 + c0 + 4 * x);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float gv = T16::to_f32((uint16_t)(g[e >> 1] >> (16 * (e & 1))));
#pragma unroll
        for (int m = 0; m < 2; ++m) dot[m] += gv * o[m][e >> 2][e & 3];
        nrm += gv * gv;
      }
    }
#pragma unroll
    for (int s = 8; s >= 1; s >>= 1) {
      dot[0] += __shfl_xor(dot[0], s, 64);
      dot[1] += __shfl_xor(dot[1], s, 64);
      if (Scaled<T16>::value) nrm += __shfl_xor(nrm, s, 64);
    }
    top = fmaxf(top, nrm);
    if (!is_v && c0 == 0 && i < a.Lq) {
      const int64_t f = bp * a.Lq + i;
#pragma unroll
      for (int m = 0; m < 2; ++m)
        a.stat[m * a.nrows + f] =
            live ? (shift - a.lse[((int64_t)b * 2 * a.P + 2 * p + m) * a.Lq + i] * kLog2e) * a.inv_c
                 : -__builtin_inff();
      a.stat[2 * a.nrows + f] = live ? -dot[0] : 0.f;
      a.stat[3 * a.nrows + f] = live ? -dot[1] : 0.f;
    }
    sum += c0 == 0 ? -dot[1] : 0.f;
  }
  sum += __shfl_xor(sum, 16, 64);
  sum += __shfl_xor(sum, 32, 64);
  if (Scaled<T16>::value) top = wave_max(top);
  if ((tid & 63) == 0) {
    red[0][tid >> 6] = top;
    red[1][tid >> 6] = sum;
  }
  __syncthreads();
  if (tid) return;
  if (Scaled<T16>::value)
    (is_v ? a.vmax : a.gmax)[blk] =
        sqrtf(fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3])));
  if (!is_v) a.lsum[blk] = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
}

// fp16: the power of two m with 2 max|do| max|v| max(1, |lam|) m <= 1 for a key pair's group, and
// what takes the exponents' shift out again.
struct Powers {
  float m, back;
};
__device__ inline Powers powers(const DiffBwdArgs& a, int b, int kp) {
  const int l = threadIdx.x & 63;
  const int64_t ng = (int64_t)a.rep * a.nqb;
  const float* g = a.gmax + ((int64_t)b * a.P + (int64_t)kp * a.rep) * a.nqb;
  const float* v = a.vmax + ((int64_t)b * a.Pk + kp) * a.nkb;
  float mg = 0.f, mv = 0.f;
#pragma unroll 8
  for (int64_t i = l; i < ng; i += 64) mg = fmaxf(mg, g[i]);
#pragma unroll 8
  for (int i = l; i < a.nkb; i += 64) mv = fmaxf(mv, v[i]);
  const float ml = top_weight(a, kp);
  const float bound = 2.f * wave_max(mg) * wave_max(mv) * fmaxf(ml, 1.f);
  return Powers{bound > 0.f && bound < 1e30f ? power_of_two(-exponent(bound)) : 1.f,
                power_of_two(-weight_shift(ml))};
}

// A C tile pair ([channel][row]) of a lane's row: 16-bit, or fp32 parts.
template <typename T16>
__device__ inline void store_row(uint16_t* p, const f32x16 (&x)[2], float f, int h, bool keep) {
#pragma unroll
  for (int mb = 0; mb < 2; ++mb)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const u32x2 y{pack_pair<T16>(x[mb][4 * g] * f, x[mb][4 * g + 1] * f),
                    pack_pair<T16>(x[mb][4 * g + 2] * f, x[mb][4 * g + 3] * f)};
      *reinterpret_cast<u32x2*>(p + 32 * mb + 8 * g + 4 * h) = keep ? y : u32x2{0, 0};
    }
}
__device__ inline void store_part(float* p, const f32x16 (&x)[2], float f, int h, bool keep) {
#pragma unroll
  for (int mb = 0; mb < 2; ++mb)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 y;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = keep ? x[mb][4 * g + i] * f : 0.f;
      *reinterpret_cast<f32x4*>(p + 32 * mb + 8 * g + 4 * h) = y;
    }
}

// dq: workgroup = 4 waves x 32 query rows of a pair; keys of both maps and values in stages of 32
// through four LDS slots, three ahead.  dQ_m^T += K_m^T dS_m^T with dS_m^T straight from the score
// tile's registers.
template <typename T16>
__device__ inline __attribute__((always_inline)) void dq_of(const DiffBwdArgs& a, int blk,
                                                            unsigned char* s0, unsigned char* s1,
                                                            unsigned char* s2, unsigned char* s3) {
  const int tid = threadIdx.x, l = tid & 63, h = l >> 5;
  if (blk >= a.dq_blocks) {  // dlam of a pair: batch by batch, block by block
    const int p = blk - a.dq_blocks;
    float* red = reinterpret_cast<float*>(s0);
    float s = 0.f;
    const int64_t n = (int64_t)a.B * a.nqb;
    for (int64_t i = tid; i < n; i += 256) {
      const int64_t b = i / a.nqb;
      s += a.lsum[(b * a.P + p) * a.nqb + (i - b * a.nqb)];
    }
    red[tid] = s;
    __syncthreads();
    for (int x = 128; x >= 1; x >>= 1) {
      if (tid < x) red[tid] += red[tid + x];
      __syncthreads();
    }
    if (tid) return;
    if (a.weights.dtype == 2)
      static_cast<float*>(a.dlam)[p] = red[0];
    else
      static_cast<uint16_t*>(a.dlam)[p] =
          a.weights.dtype == SLA2H_DTYPE_BF16 ? BF16::from_f32(red[0]) : F16::from_f32(red[0]);
    return;
  }
  int bp, item;
  if (!work_item(a.dq_map, blk, bp, item)) return;
  const int qt = item / a.dq_splits, sp = item - qt * a.dq_splits;
  const int b = bp / a.P, p = bp - b * a.P, kp = p / a.rep;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const LaneOff lo(l);
  const int qlen = seq_len(a.q_lens, b, a.Lq), klen = seq_len(a.k_lens, b, a.Lk);

  const int q0 = qt * 128, qw = q0 + w * 32;
  const int qend = min(q0 + 128, qlen);
  const int kmax = qend > q0 ? key_limit(qend - 1, qlen, klen, a.causal) : 0;
  const int nunit = (kmax + kUnitRows - 1) / kUnitRows;
  const int per = (nunit + a.dq_splits - 1) / a.dq_splits;
  const int t0 = sp * per, nt = min(nunit, t0 + per);

  const uint16_t* src = w < 2 ? a.k + b * a.kb + (2 * kp + w) * a.kh
                              : a.v + b * a.vb + (2 * kp + w - 2) * a.vh;
  const int64_t ld = (w < 2 ? a.kl : a.vl) * 2;
  auto load = [&](int t, unsigned char* s) __attribute__((always_inline)) {
    const int64_t row = (int64_t)t * kUnitRows;
    load_unit(src, row, (int64_t)klen - row, ld, s + w * kUnitB, l);
  };

  Powers pw{1.f, 1.f};
  if (Scaled<T16>::value) pw = powers(a, b, kp);
  const int i = qw + (l & 31);
  const int lim = key_limit(i, qlen, klen, a.causal);
  const bool live = lim > 0;
  const int64_t flat = (int64_t)bp * a.Lq + i;
  float nl[2], nd[2];  // shift - lse_m log2e, -delta_m (times m)
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    nl[m] = live ? a.stat[m * a.nrows + flat] * a.c : -__builtin_inff();
    nd[m] = live ? a.stat[(2 + m) * a.nrows + flat] * pw.m : 0.f;
  }
  u32x4 qf[2][4], gf[2][4];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const uint16_t* qp = a.q + b * a.qb + (2 * p + m) * a.qh + i * a.ql + 8 * h;
    const uint16_t* gp = a.dout + (((int64_t)b * a.Lq + i) * a.P + p) * 128 + 64 * m + 8 * h;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      qf[m][s] = live ? *reinterpret_cast<const u32x4*>(qp + 16 * s) : u32x4{0, 0, 0, 0};
      gf[m][s] = live ? *reinterpret_cast<const u32x4*>(gp + 16 * s) : u32x4{0, 0, 0, 0};
    }
  }
  // keys that any query of the wave sees, and that all of them see
  const int wlast = min(qw + 32, qlen) - 1;
  const int wany = wlast >= qw ? key_limit(wlast, qlen, klen, a.causal) : 0;
  const int wall = wlast >= qw ? key_limit(qw, qlen, klen, a.causal) : 0;
  const bool few = klen <= kFineKeys || wany <= kFineRows || qlen <= kFineRows;

  f32x16 acc[2][2];
#pragma unroll
  for (int m = 0; m < 2; ++m) acc[m][0] = acc[m][1] = zero16();
  auto part = [&](auto masked, bool fine, int base, const unsigned char* s)
      __attribute__((always_inline)) {
    f32x16 sc[2] = {zero16(), zero16()}, dp = zero16();
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      sc[0] = mfma_32x32x16<T16>(row_frag(s, 0, x, lo), qf[0][x], sc[0]);
      dp = mfma_32x32x16<T16>(row_frag(s + 2 * kUnitB, 0, x, lo), gf[0][x], dp);
      sc[1] = mfma_32x32x16<T16>(row_frag(s + kUnitB, 0, x, lo), qf[1][x], sc[1]);
      dp = mfma_32x32x16<T16>(row_frag(s + 3 * kUnitB, 0, x, lo), gf[1][x], dp);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      f32x16 d;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        d[e] = fast_exp2(__builtin_fmaf(sc[m][e], a.c, nl[m])) *
               (Scaled<T16>::value ? __builtin_fmaf(dp[e], pw.m, nd[m]) : dp[e] + nd[m]);
      if (decltype(masked)::value) {
        const int x = lim - base - 4 * h;
#pragma unroll
        for (int e = 0; e < 16; ++e) d[e] = 8 * (e >> 2) + (e & 3) < x ? d[e] : 0.f;
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const u32x4 ds = pack_step<T16>(d, x);
        u32x4 kf[2];
#pragma unroll
        for (int mb = 0; mb < 2; ++mb) {
          kf[mb] = col_frag(s + m * kUnitB, 16 * x, mb, lo);
          acc[m][mb] = mfma_32x32x16<T16>(kf[mb], ds, acc[m][mb]);
        }
        if (fine) {
          const u32x4 lost = lost_step<T16>(d, x, ds);
#pragma unroll
          for (int mb = 0; mb < 2; ++mb)
            acc[m][mb] = mfma_32x32x16<T16>(kf[mb], lost, acc[m][mb]);
        }
      }
    }
  };
  auto stage = [&](int t, bool fine, const unsigned char* cur, unsigned char* to)
      __attribute__((always_inline)) {
    // the stages up to t have landed, stage t - 1 is read
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(8));
    __builtin_amdgcn_s_barrier();
    load(t + 3, to);
    const int base = t * kUnitRows;
    if (base + kUnitRows <= wall)  // a stage that every query of the wave sees: no branch inside
      part(std::false_type{}, fine, base, cur);
    else if (base < wany)
      part(std::true_type{}, true, base, cur);
  };
  load(t0, s0);
  load(t0 + 1, s1);
  load(t0 + 2, s2);
  for (int t = t0; t < nt; t += 4) {
    stage(t, true, s0, s3);
    if (t + 1 >= nt) break;
    stage(t + 1, few, s1, s0);
    if (t + 2 >= nt) break;
    stage(t + 2, true, s2, s1);
    if (t + 3 >= nt) break;
    stage(t + 3, few, s3, s2);
  }
  __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));  // no load into this LDS outlives the workgroup

  if (i >= a.Lq) return;
  const int64_t orow = ((int64_t)b * a.Lq + i) * a.P + p;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    // (the softmax of one key is constant: its dS is the rounding of dA - delta)
    const float f = lim == 1 ? 0.f : (m ? -a.lam[p] : 1.f) * a.scale * pw.back / pw.m;
    if (a.dq_splits == 1)
      store_row<T16>(a.dq + orow * 128 + 64 * m, acc[m], f, h, live);
    else
      store_part(a.dq_part + ((int64_t)sp * a.nrows + orow) * 128 + 64 * m, acc[m], f, h, live);
  }
}

// The value that the lanes' place e of 16 holds, in all lanes of their row of 16.
template <int E>
__device__ inline float row_value(float x) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x150 + E, 0xf, 0xf, true));
}
__device__ inline float row_value_at(float x, int e) {  // e a constant where it is called
  switch (e) {
#define SLA2H_ROW(E) \
  case E:            \
    return row_value<E>(x);
    SLA2H_ROW(0) SLA2H_ROW(1) SLA2H_ROW(2) SLA2H_ROW(3) SLA2H_ROW(4) SLA2H_ROW(5) SLA2H_ROW(6)
    SLA2H_ROW(7) SLA2H_ROW(8) SLA2H_ROW(9) SLA2H_ROW(10) SLA2H_ROW(11) SLA2H_ROW(12) SLA2H_ROW(13)
    SLA2H_ROW(14)
#undef SLA2H_ROW
    default:
      return row_value<15>(x);
  }
}

// dk, dv: workgroup = 4 waves x 32 keys of one key pair; the query rows (both maps' queries, the 128
// channels of do) of the pairs that read it are streamed in stages of 32 rows through two LDS slots, one
// ahead, with their four statistics.  A wave holds 128 channels of dv, 64 of each dk and its keys in
// registers; its values lie in LDS, so that two workgroups fit on a CU and one computes while the other
// waits (with the values in registers, one wave per SIMD: 6.1 ms at B = 1, H = 8, L = 29,952, bf16; eight
// waves in one workgroup: 4.1; this form 3.75, 0.98 PFLOP/s, at the card's power limit).  A row's
// statistic belongs to one register of a score tile in all lanes of a half: a lane reads one value, and
// the add takes it from there (DPP).
template <typename T16, bool CAUSAL, bool FINE>
__device__ inline __attribute__((always_inline)) void dkdv_body(const DiffBwdArgs& a, int blk,
                                                                unsigned char* r0, unsigned char* r1,
                                                                float (*t0_)[64], float (*t1_)[64],
                                                                unsigned char* vt) {
  int bk, item;
  if (!work_item(a.kv_map, blk, bk, item)) return;
  const int ktile = item / a.kv_splits, sp = item - ktile * a.kv_splits;
  const int b = bk / a.Pk, kp = bk - b * a.Pk;
  const int tid = threadIdx.x, l = tid & 63, h = l >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const LaneOff lo(l);
  const int qlen = seq_len(a.q_lens, b, a.Lq), klen = seq_len(a.k_lens, b, a.Lk);

  const int key0 = ktile * kKeyRows, kw = key0 + w * 32;
  // first query that sees a key of the workgroup (causal: i >= j - off)
  const int off = klen - qlen;
  int first = first_query(qlen, klen, a.causal);
  if (CAUSAL) first = max(first, key0 - off);
  const int nq = key0 < klen && first < qlen ? (qlen - first + kUnitRows - 1) / kUnitRows : 0;
  const int total = nq * a.rep;  // (pair, stage)
  const int per = (total + a.kv_splits - 1) / a.kv_splits;
  const int u0 = sp * per, u1 = min(total, u0 + per);

  // this wave's values
#pragma unroll
  for (int m = 0; m < 2; ++m)
    load_unit(a.v + b * a.vb + (2 * kp + m) * a.vh, kw, (int64_t)klen - kw, a.vl * 2,
              vt + (2 * w + m) * kUnitB, l);

  // the stage to load next, and the one to compute (their pair of the group and first row)
  int lu = u0, lp = u0 < u1 ? u0 / nq : 0;
  int lrow = first + (u0 < u1 ? u0 - lp * nq : 0) * kUnitRows;
  int cu = u0, cp = lp, crow = lrow;
  // wave x loads matrix x of the stage and statistic x
  const int x = w;
  auto load = [&](unsigned char* s, float (*st)[64]) __attribute__((always_inline)) {
    const int64_t p = (int64_t)kp * a.rep + lp, n = lu < u1 ? (int64_t)qlen - lrow : 0;
    const uint16_t* src = x < 2 ? a.q + b * a.qb + (2 * p + x) * a.qh
                                : a.dout + ((int64_t)b * a.Lq * a.P + p) * 128 + 64 * (x - 2);
    const int64_t ld = x < 2 ? a.ql * 2 : (int64_t)a.P * 256;
    load_unit(src, lrow, n, ld, s + x * kUnitB, l);
    const auto rt = make_rsrc(a.stat + x * a.nrows + ((int64_t)b * a.P + p) * a.Lq + lrow,
                              n <= 0 ? 0 : (n < kUnitRows ? n : kUnitRows) * 4);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        rt, (__attribute__((address_space(3))) void*)&st[x][0], 4, 4 * l, 0, 0, 0);
    ++lu;
    lrow += kUnitRows;
    if (lrow >= qlen && lu < u1) lrow = first, ++lp;
  };

  Powers pw{1.f, 1.f};
  if (Scaled<T16>::value) pw = powers(a, b, kp);
  u32x4 kf[2][4];
  {
    const int j = kw + (l & 31);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int s = 0; s < 4; ++s)
        kf[m][s] = j < klen ? *reinterpret_cast<const u32x4*>(a.k + b * a.kb + (2 * kp + m) * a.kh +
                                                              j * a.kl + 16 * s + 8 * h)
                            : u32x4{0, 0, 0, 0};
  }
  f32x16 ak[2][2], av[4];
#pragma unroll
  for (int y = 0; y < 2; ++y) ak[0][y] = ak[1][y] = av[y] = av[2 + y] = zero16();
  // The weight of the pair at hand: |lam| goes into the exponent, its sign into the packed dS.  (Loaded
  // where the pair changes only: a load in every stage would wait for the stages on their way.)
  float log_lam = 0.f;
  bool minus = false;
  auto load_weight = [&]() __attribute__((always_inline)) {
    const float lam = a.lam[kp * a.rep + cp];
    log_lam = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(
                                            int, __log2f(__builtin_fabsf(lam)) * a.inv_c)));
    minus = __builtin_amdgcn_readfirstlane(lam < 0.f);
  };
  load_weight();
  // register e of a tile is row 8 (e / 4) + 4 h + e % 4: lane e of each 16 reads it
  const int srow = 8 * ((l & 15) >> 2) + 4 * h + (l & 3);

  // A stage in four runs of products, each in a fixed order with its LDS operands read ahead (by two
  // products, by one where the lost halves need the registers) and a share of the
  // exponentials beside it: S_1 and dA; S_2 under map 1; dk_1 under map 2; dk_2 and dv.
  constexpr int AHEAD = FINE ? 1 : 2;
  auto stage = [&](const unsigned char* s, const float (*st)[64], unsigned char* sl, float (*tl)[64])
      __attribute__((always_inline)) {
    // this stage has landed, the one before is read
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));
    __builtin_amdgcn_s_barrier();
    load(sl, tl);
    if (kw < klen) {
      float sv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) sv[i] = st[i][srow];
      sv[1] += log_lam;
      const float sign = minus ? -1.f : 1.f;
      const uint32_t flip = minus ? 0x80008000u : 0u;
      auto mask = [&](f32x16& x) __attribute__((always_inline)) {
        if (CAUSAL && crow < kw + 31 - off) {
          asm volatile("");
          const int y = kw + (l & 31) - off - crow - 4 * h;
#pragma unroll
          for (int e = 0; e < 16; ++e)
            x[e] = 8 * (e >> 2) + (e & 3) >= y ? x[e] : -__builtin_inff();
        }
      };
      f32x16 dp = zero16(), p[2] = {zero16(), zero16()};
      int vw = w * 2 * kUnitB;
      asm volatile("" : "+s"(vw));  // (four addresses held for the whole loop otherwise)
      {
        u32x4 fa[AHEAD + 1], fb[AHEAD + 1];
        auto operands = [&](int i) __attribute__((always_inline)) {
          const int j = i / 3 * 2 + i % 3 - 1, r = i % (AHEAD + 1);  // j: dA's products
          fa[r] = i % 3 ? row_frag(s + (2 + (j >> 2)) * kUnitB, 0, j & 3, lo)
                        : row_frag(s, 0, i / 3, lo);
          if (i % 3) fb[r] = row_frag(vt + vw + (j >> 2) * kUnitB, 0, j & 3, lo);
        };
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) operands(i);
#pragma unroll
        for (int i = 0; i < 12; ++i) {
          __builtin_amdgcn_sched_barrier(0);
          if (i + AHEAD < 12) operands(i + AHEAD);
          const int r = i % (AHEAD + 1);
          if (i % 3)
            dp = mfma_32x32x16<T16>(fa[r], fb[r], dp);
          else
            p[0] = mfma_32x32x16<T16>(fa[r], kf[0][i / 3], p[0]);
        }
      }
      mask(p[0]);
      u32x4 dd[2][2], dl[2][2], f[2];
      // registers 4 g .. 4 g + 3 of map m: probabilities (times |lam|), dS in 16 bits
      auto elements = [&](int m, int g) __attribute__((always_inline)) {
        float d[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = 4 * g + i;
          const float y = fast_exp2((p[m][e] + row_value_at(sv[m], e)) * a.c);
          d[i] = (Scaled<T16>::value ? y * pw.m : y) * (dp[e] + row_value_at(sv[2 + m], e));
          p[m][e] = y;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t word = pack_pair<T16>(d[2 * i], d[2 * i + 1]);
          asm volatile("" : "+v"(word));  // here, not behind the products
          dd[m][g >> 1][2 * (g & 1) + i] = m ? word ^ flip : word;
          if (FINE) {
            const uint32_t lost = pack_pair<T16>(d[2 * i] - T16::to_f32((uint16_t)(word & 0xffff)),
                                                 d[2 * i + 1] - T16::to_f32((uint16_t)(word >> 16)));
            dl[m][g >> 1][2 * (g & 1) + i] = m ? lost ^ flip : lost;
          }
        }
      };
      __builtin_amdgcn_sched_barrier(0);
      f[0] = row_frag(s + kUnitB, 0, 0, lo);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        __builtin_amdgcn_sched_barrier(0);
        if (g < 3) f[(g + 1) & 1] = row_frag(s + kUnitB, 0, g + 1, lo);
        p[1] = mfma_32x32x16<T16>(f[g & 1], kf[1][g], p[1]);
        elements(0, g);
      }
      mask(p[1]);
      __builtin_amdgcn_sched_barrier(0);
      f[0] = col_frag(s, 0, 0, lo);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        __builtin_amdgcn_sched_barrier(0);
        if (g < 3) f[(g + 1) & 1] = col_frag(s, 16 * ((g + 1) >> 1), (g + 1) & 1, lo);
        ak[0][g & 1] = mfma_32x32x16<T16>(f[g & 1], dd[0][g >> 1], ak[0][g & 1]);
        if (FINE) ak[0][g & 1] = mfma_32x32x16<T16>(f[g & 1], dl[0][g >> 1], ak[0][g & 1]);
        elements(1, g);
      }
      u32x4 pp[2], pl[2], fv[AHEAD + 1];
      auto value = [&](int j) __attribute__((always_inline)) {
        return j < 4 ? col_frag(s + kUnitB, 16 * (j >> 1), j & 1, lo)
                     : col_frag(s + (2 + ((j & 3) >> 1)) * kUnitB, 16 * ((j - 4) >> 2), j & 1, lo);
      };
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) fv[j] = value(j);
#pragma unroll
      for (int j = 0; j < 12; ++j) {
        __builtin_amdgcn_sched_barrier(0);
        if (j + AHEAD < 12) fv[(j + AHEAD) % (AHEAD + 1)] = value(j + AHEAD);
        const int r = j % (AHEAD + 1);
        if (j < 4) {
          ak[1][j & 1] = mfma_32x32x16<T16>(fv[r], dd[1][j >> 1], ak[1][j & 1]);
          if (FINE) ak[1][j & 1] = mfma_32x32x16<T16>(fv[r], dl[1][j >> 1], ak[1][j & 1]);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int e = 4 * j + 2 * i;
            const float x = __builtin_fmaf(-sign, p[1][e], p[0][e]);
            const float y = __builtin_fmaf(-sign, p[1][e + 1], p[0][e + 1]);
            uint32_t word = pack_pair<T16>(x, y);
            asm volatile("" : "+v"(word));
            pp[j >> 1][2 * (j & 1) + i] = word;
            if (FINE)
              pl[j >> 1][2 * (j & 1) + i] =
                  pack_pair<T16>(x - T16::to_f32((uint16_t)(word & 0xffff)),
                                 y - T16::to_f32((uint16_t)(word >> 16)));
          }
        } else {
          const int k = (j - 4) >> 2;
          av[j & 3] = mfma_32x32x16<T16>(fv[r], pp[k], av[j & 3]);
          if (FINE) av[j & 3] = mfma_32x32x16<T16>(fv[r], pl[k], av[j & 3]);
        }
      }
    }
    ++cu;
    crow += kUnitRows;
    if (crow >= qlen && cu < u1) {
      crow = first;
      ++cp;
      load_weight();
    }
  };
  load(r0, t0_);
  for (int u = u0; u < u1; u += 2) {
    stage(r0, t0_, r1, t1_);
    if (u + 1 >= u1) break;
    stage(r1, t1_, r0, t0_);
  }
  __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));

  const int j = kw + (l & 31);
  if (j >= a.Lk) return;
  const bool keep = j < klen;
  const int64_t orow = ((int64_t)b * a.Lk + j) * a.Pk + kp, n = (int64_t)a.B * a.Lk * a.Pk;
  const float fk = klen == 1 ? 0.f : a.scale * pw.back / pw.m;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const f32x16 y[2] = {av[2 * m], av[2 * m + 1]};
    if (a.kv_splits == 1) {
      store_row<T16>(a.dk + orow * 128 + 64 * m, ak[m], m ? -fk : fk, h, keep);
      store_row<T16>(a.dv + orow * 128 + 64 * m, y, pw.back, h, keep);
    } else {
      const int64_t at = (sp * n + orow) * 128 + 64 * m;
      store_part(a.dk_part + at, ak[m], m ? -fk : fk, h, keep);
      store_part(a.dv_part + at, y, pw.back, h, keep);
    }
  }
}

// The launches.  dk and dv with the lost halves in all clips (fine_clip), in none, or in those whose own
// lengths ask for them: both bodies, a workgroup takes one (clips of 4,159, 2,703 and 1,247 tokens, which
// take none, causal: 226 us for 230).
enum { kNone, kAll, kByClip };
template <typename T16, bool CAUSAL, int LOST>
__device__ inline __attribute__((always_inline)) void dkdv_of(const DiffBwdArgs& a, int blk,
                                                              unsigned char* r0, unsigned char* r1,
                                                              float (*t0_)[64], float (*t1_)[64],
                                                              unsigned char* vt) {
  bool fine = LOST == kAll;
  if (LOST == kByClip) {
    int bk, item;
    if (!work_item(a.kv_map, blk, bk, item)) return;
    const int b = bk / a.Pk;
    fine = fine_clip(a.rep, seq_len(a.q_lens, b, a.Lq), seq_len(a.k_lens, b, a.Lk));
  }
  if (fine)
    dkdv_body<T16, CAUSAL, true>(a, blk, r0, r1, t0_, t1_, vt);
  else
    dkdv_body<T16, CAUSAL, false>(a, blk, r0, r1, t0_, t1_, vt);
}

// Calls whose clips all take the lost halves and those whose workgroups are all resident at once: both in
// one launch, side by side (us for the backward of 8 heads, in one / one after the other: 600 tokens 36 /
// 48, 1,000 41 / 54, causal 44 / 52, 2,500 90 / 104; 600 queries of 5,000 keys 58 / 68).  Of others the
// two bodies under one allocation spill 20 registers (29,952 tokens: 7.65 ms, one after the other 7.2).
// Spilled in what is kept: 12 to 47 registers in one launch, 4 to 27 with both bodies of dk and dv, 9 to
// 12 in dq's own; none in dk and dv's without the lost halves.
template <typename T16, bool CAUSAL, int LOST>
__global__ __launch_bounds__(256, 2) void diff_bwd_few_kernel(DiffBwdArgs a) {
  __shared__ __align__(16) unsigned char s0[kStageB], s1[kStageB], v[2 * kStageB];
  __shared__ __align__(16) float t0_[4][64], t1_[4][64];
  const int blk = blockIdx.x;
  if (blk < a.kv_blocks)
    dkdv_of<T16, CAUSAL, LOST>(a, blk, s0, s1, t0_, t1_, v);
  else
    dq_of<T16>(a, blk - a.kv_blocks, s0, s1, v, v + kStageB);
}
template <typename T16, bool CAUSAL, int LOST>
__global__ __launch_bounds__(256, 2) void diff_bwd_dkdv_kernel(DiffBwdArgs a) {
  __shared__ __align__(16) unsigned char s0[kStageB], s1[kStageB], v[2 * kStageB];
  __shared__ __align__(16) float t0_[4][64], t1_[4][64];
  dkdv_of<T16, CAUSAL, LOST>(a, blockIdx.x, s0, s1, t0_, t1_, v);
}
template <typename T16>
__global__ __launch_bounds__(256, 2) void diff_bwd_dq_kernel(DiffBwdArgs a) {
  __shared__ __align__(16) unsigned char s0[kStageB], s1[kStageB], s2[kStageB], s3[kStageB];
  dq_of<T16>(a, blockIdx.x, s0, s1, s2, s3);
}

// Adds the parts of a result in order; blockIdx.y: which.
struct JoinArgs {
  const float* part[3];
  uint16_t* y[3];
  int64_t n[3];
  int splits[3];
};
template <typename T16>
__global__ __launch_bounds__(256) void diff_bwd_join_kernel(JoinArgs a) {
  const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4, n = a.n[blockIdx.y];
  if (e >= n) return;
  const float* part = a.part[blockIdx.y] + e;
  const int splits = a.splits[blockIdx.y];
  f32x4 x{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) x += *reinterpret_cast<const f32x4*>(part + s * n);
  *reinterpret_cast<u32x2*>(a.y[blockIdx.y] + e) =
      u32x2{pack_pair<T16>(x[0], x[1]), pack_pair<T16>(x[2], x[3])};
}

struct BwdPlan {
  int64_t qtiles, dq_nwork, ktiles, kv_nwork;
  int dq_splits, kv_splits;
  int64_t nqb, nkb;
  size_t stats, dq_parts, kv_parts;  // floats (kv_parts: of dk, and as many of dv)
};

BwdPlan bwd_plan(int dtype, int B, int H, int Hkv, int64_t Lq, int64_t Lk, float share) {
  BwdPlan p{};
  const int64_t bp = (int64_t)B * H / 2, bk = (int64_t)B * Hkv / 2, rep = H / Hkv;
  p.qtiles = (Lq + 127) / 128;
  // (us, unsplit / split, B x H x L: 2 x 8 x 2,048 dq 87 / 63, dk and dv 90 / 69; 1 x 8 x 6,000 204 / 164,
  // 230 / 194; causal 1 x 8 x 12,000 417 / 283, 488 / 339)
  float t;
  p.dq_splits = best_split(bp * p.qtiles, (Lk + 31) / 32, share, SplitCost{1.15f, 2.f, 0.033f, 8}, t);
  p.dq_nwork = bp * p.qtiles * p.dq_splits;
  p.ktiles = (Lk + kKeyRows - 1) / kKeyRows;
  p.kv_splits = best_split(bk * p.ktiles, rep * ((Lq + 31) / 32), share,
                           SplitCost{1.2f, 2.1f, 0.066f, 8}, t);
  p.kv_nwork = bk * p.ktiles * p.kv_splits;
  p.nqb = (Lq + kNormRows - 1) / kNormRows;
  p.nkb = (Lk + kNormRows - 1) / kNormRows;
  p.stats = 4 * bp * Lq + bp * p.nqb + (dtype == SLA2H_DTYPE_F16 ? bp * p.nqb + bk * p.nkb : 0);
  p.stats = ((p.stats + 3) & ~(size_t)3) + ((H / 2 + 3) & ~3);  // ... and the weights
  p.dq_parts = p.dq_splits > 1 ? (size_t)p.dq_splits * bp * Lq * 128 : 0;
  p.kv_parts = p.kv_splits > 1 ? (size_t)p.kv_splits * bk * Lk * 128 : 0;
  return p;
}

}  // namespace

}  // namespace sla2h

using namespace sla2h;

extern "C" size_t sla2h_diff_attn_bwd_workspace_bytes(int dtype, int B, int H, int Hkv, int64_t Lq,
                                                      int64_t Lk) {
  if (!diff_sizes_ok(B, H, Hkv, Lq, Lk)) return 0;
  size_t most = 0;
  for (int i = 0; i < 4; ++i) {
    const float share = kShares[i & 1][i >> 1];
    const BwdPlan p = bwd_plan(dtype, B, H, Hkv, Lq, Lk, share);
    const size_t n = p.stats + p.dq_parts + 2 * p.kv_parts;
    most = n > most ? n : most;
  }
  return most * 4;
}

extern "C" int sla2h_diff_attn_bwd(const void* q, const void* k, const void* v, const void* lam,
                                   int lam_dtype, int64_t lam_stride, const void* dout,
                                   const float* lse, const float* maps,
                                   const int64_t* strides, const int32_t* q_lens,
                                   const int32_t* k_lens, int dtype, int B, int H, int Hkv,
                                   int64_t Lq, int64_t Lk, int causal, float scale,
                                   void* workspace, void* dq, void* dk, void* dv, void* dlam,
                                   void* stream) {
  const Weights wts{lam, lam_dtype, lam_stride};
  SLA2H_CHECK_ARG(q && k && v && wts.ok() && dout && lse && maps && strides && workspace && dlam);
  SLA2H_CHECK_ARG(!dk == !dv);
  SLA2H_CHECK_ARG(dtype == SLA2H_DTYPE_F16 || dtype == SLA2H_DTYPE_BF16);
  SLA2H_CHECK_ARG(diff_sizes_ok(B, H, Hkv, Lq, Lk));
  SLA2H_CHECK_ARG(scale > 0.f && scale < 1e30f);
  SLA2H_CHECK_ARG(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)dout | (uintptr_t)maps |
                   (uintptr_t)workspace | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) % 16 == 0);
  SLA2H_CHECK_ARG(((uintptr_t)lse | (uintptr_t)q_lens | (uintptr_t)k_lens) % 4 == 0 &&
                  (uintptr_t)dlam % (lam_dtype == 2 ? 4 : 2) == 0);
  for (int i = 0; i < 9; ++i) SLA2H_CHECK_ARG(strides[i] >= 0 && strides[i] % 8 == 0);
  // rows apart from each other: the range check of a tile's load tells them by their offset; 32-bit
  // byte offsets within a tile
  for (int i : {2, 5, 8}) SLA2H_CHECK_ARG(strides[i] >= kDD && strides[i] < ((int64_t)1 << 23));
  SLA2H_CHECK_ARG((int64_t)H * kDD < ((int64_t)1 << 23));
  const bool even = !causal && !q_lens && !k_lens;
  const BwdPlan p = bwd_plan(dtype, B, H, Hkv, Lq, Lk, kShares[causal != 0][q_lens || k_lens]);
  SLA2H_CHECK_ARG(p.dq_nwork < ((int64_t)1 << 30) && p.kv_nwork < ((int64_t)1 << 30));
  const int64_t bp = (int64_t)B * H / 2, bk = (int64_t)B * Hkv / 2;
  const int64_t pq = bp * p.nqb, pv = dtype == SLA2H_DTYPE_F16 ? bk * p.nkb : 0;
  SLA2H_CHECK_ARG(pq + pv < ((int64_t)1 << 31));
  DiffBwdArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.dout = static_cast<const uint16_t*>(dout);
  a.weights = wts, a.lse = lse, a.maps = maps;
  a.dq = static_cast<uint16_t*>(dq);
  a.dk = static_cast<uint16_t*>(dk);
  a.dv = static_cast<uint16_t*>(dv);
  a.dlam = dlam;
  a.q_lens = q_lens;
  a.k_lens = k_lens;
  a.qb = strides[0], a.qh = strides[1], a.ql = strides[2];
  a.kb = strides[3], a.kh = strides[4], a.kl = strides[5];
  a.vb = strides[6], a.vh = strides[7], a.vl = strides[8];
  a.Lq = Lq;
  a.Lk = Lk;
  a.B = B;
  a.P = H / 2;
  a.Pk = Hkv / 2;
  a.rep = H / Hkv;
  a.causal = causal != 0;
  a.c = scale * kLog2e;
  a.inv_c = 1.f / a.c;
  a.scale = scale;
  a.nrows = bp * Lq;
  a.stat = static_cast<float*>(workspace);
  a.lsum = a.stat + 4 * a.nrows;
  a.gmax = a.lsum + bp * p.nqb;
  a.vmax = a.gmax + bp * p.nqb;
  a.lam = a.stat + p.stats - ((a.P + 3) & ~3);
  a.nqb = (int)p.nqb;
  a.nkb = (int)p.nkb;
  a.dq_part = a.stat + p.stats;
  a.dk_part = a.dq_part + p.dq_parts;
  a.dv_part = a.dk_part + p.kv_parts;
  a.dq_map = work_map(bp, p.qtiles * p.dq_splits, even, causal);
  a.kv_map = work_map(bk, p.ktiles * p.kv_splits, even, false);  // causal: the first keys' are longest
  a.dq_blocks = dq ? (int)work_grid(a.dq_map) : 0;
  a.kv_blocks = dk ? (int)work_grid(a.kv_map) : 0;
  a.dq_splits = p.dq_splits;
  a.kv_splits = p.kv_splits;
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto go = [&](auto tag) -> int {
    using T16 = decltype(tag);
    int err;
    diff_bwd_prep_kernel<T16><<<(unsigned)(pq + pv), 256, 0, st>>>(a, pq);
    if ((err = (int)hipGetLastError())) return err;
    const unsigned nq = (unsigned)(a.dq_blocks + a.P), nk = (unsigned)a.kv_blocks;
    const bool all = fine_clip(a.rep, Lq, Lk);
    // (whether or not both are asked for: a gradient does not depend on the others)
    const bool one = all || work_grid(a.kv_map) + work_grid(a.dq_map) <= 512;
    using std::integral_constant;
    auto launch = [&](auto causal_, auto lost) {
      constexpr bool CAUSAL = decltype(causal_)::value;
      constexpr int LOST = decltype(lost)::value;
      if (one)
        diff_bwd_few_kernel<T16, CAUSAL, LOST><<<nk + nq, 256, 0, st>>>(a);
      else if constexpr (LOST != kAll)
        if (dk) diff_bwd_dkdv_kernel<T16, CAUSAL, LOST><<<nk, 256, 0, st>>>(a);
    };
    auto lost = [&](auto causal_) {
      if (all)
        launch(causal_, integral_constant<int, kAll>{});
      else if (q_lens || k_lens)
        launch(causal_, integral_constant<int, kByClip>{});
      else
        launch(causal_, integral_constant<int, kNone>{});
    };
    if (causal)
      lost(std::true_type{});
    else
      lost(std::false_type{});
    if (!one) {
      if ((err = (int)hipGetLastError())) return err;
      diff_bwd_dq_kernel<T16><<<nq, 256, 0, st>>>(a);
    }
    if ((err = (int)hipGetLastError())) return err;
    JoinArgs j{};
    int joins = 0;
    int64_t most = 0;
    auto join = [&](const float* part, uint16_t* y, int64_t n, int splits) {
      if (!y || splits == 1) return;
      j.part[joins] = part, j.y[joins] = y, j.n[joins] = n, j.splits[joins] = splits;
      most = n > most ? n : most;
      ++joins;
    };
    join(a.dq_part, a.dq, a.nrows * 128, p.dq_splits);
    join(a.dk_part, a.dk, bk * Lk * 128, p.kv_splits);
    join(a.dv_part, a.dv, bk * Lk * 128, p.kv_splits);
    if (joins)
      diff_bwd_join_kernel<T16><<<dim3((unsigned)((most / 4 + 255) / 256), joins), 256, 0, st>>>(j);
    return (int)hipGetLastError();
  };
  return dtype == SLA2H_DTYPE_BF16 ? go(BF16{}) : go(F16{});
}
