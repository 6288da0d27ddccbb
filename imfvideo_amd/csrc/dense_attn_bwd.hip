// Backward of dense softmax attention on 64-channel heads, gfx950.  The probabilities
// are recomputed from the rows' log-sum-exp:
//
//   P_ij = exp(S_ij - lse_i),  delta_i = do_i . o_i,  dP = do v^T,  dS = P (dP - delta),
//   dq = scale dS k,  dk = scale dS^T q,  dv = P^T do   (summed over a key head's queries).
//
// Two kernels: the rows' delta; then dq with a workgroup per query block (keys streamed
// through LDS) beside dk and dv with a workgroup per key block (queries streamed through LDS).
// Seven tile products instead of the five of one fused pass, but no sum goes through
// atomics or memory: the result does not depend on the order of dispatch.
//
// fp16 operands: P (down to 1 / length) and dS would fall below fp16's normal range, so the
// exponent takes + kShift and dP - delta a power of two from the bound
// |dP - delta| <= 2 max|do_i| max|v_j| (row norms, per key head), which brings |dS| below
// 2^kShift; both are taken out of the fp32 sums again.  bf16 has fp32's range and needs
// neither.
#include "dense_attn.h"

#include <initializer_list>

namespace sla2h {

namespace {

template <typename T16>
struct Shift {
  static constexpr bool scaled = false;
  static constexpr float p = 0.f;
};
template <>
struct Shift<F16> {
  static constexpr bool scaled = true;
  static constexpr float p = 15.f;
};

// FINE: add what the rounding of P and dS lost with a second product.  Small sums do not
// average the rounding out, and a small call's time is not its products.  dq: sequences of at
// most kFineKeys keys or kFineRows queries, and causal waves that see at most kFineRows keys; dk
// and dv: workgroups that see at most kFineRows rows, and sequences of at most 32 keys (one wave
// of a workgroup).  bf16, 2-norm of dq's error: 1.7e-3 (its own rounding) to 1.8e-3 instead of
// 2.4e-3 to 2.8e-3.  Backward, us, without : with, H = 8: two clips of 274 tokens 22.3 : 22.5; two of
// 8,192 queries x 77 keys 41.8 : 43.5; L = 2,048 47 : 53, 4,096 127 : 144; causal L = 4,096
// 109 : 122, B = 3 clips of up to 4,159 152 : 159, L = 29,952 2,970 : 3,017.  The instance that asks
// the waves costs padded batches whose sequences are long, too: forward and backward, us, of clips of
// 4,159, 2,703 and 1,247 tokens, H = 8 over 2, 390 : 417, of 29,952 and 18,720 14,000 : 14,400.
constexpr int kFineKeys = 4096, kFineRows = 512;
constexpr int kNormRows = 64;  // rows of a partial maximum of the norms

struct DenseBwdArgs {
  const uint16_t *q, *k, *v, *o, *o_lo, *dout;
  const float* lse;
  uint16_t *dq, *dk, *dv;
  const int32_t *q_lens, *k_lens;
  int64_t qb, qh, ql, kb, kh, kl, vb, vh, vl, ob, oh, ol, gb, gh, gl;
  int64_t dqb, dqh, dql, dkb, dkh, dkl, dvb, dvh, dvl;
  int64_t Lq, Lk;
  int H, Hkv, rep, nbh, nbk;
  int causal;
  float c, inv_c, scale;
  float *nlse, *ndelta;  // (B, H, Lq): -(lse log2e - shift) / c and -delta
  float *gmax, *vmax;    // (B, H, nqb), (B, Hkv, nkb): largest row norms (fp16)
  int nqb, nkb;
  WorkMap dq_map, kv_map;  // tiles x splits of a query head, of a key head
  int kv_blocks;           // workgroups of dk and dv, before those of dq
  int dq_splits, kv_splits;
  float *dq_part, *kv_part;
};

// Queries [first, qlen) see a key.
__device__ inline int first_query(int qlen, int klen, int causal) {
  if (klen == 0) return qlen;
  return causal && qlen > klen ? qlen - klen : 0;
}

// delta of 64 rows of a head (8 lanes per row; HBM-bound: 16 us at B = 1, H = 8, L = 29,952), and
// for fp16 the largest row norm of do; the workgroups behind them take the norms of v.
template <typename T16>
__global__ __launch_bounds__(256) void dense_bwd_prep_kernel(DenseBwdArgs a, int64_t nq) {
  __shared__ float red[4];
  const int tid = threadIdx.x, c0 = (tid & 7) * 8;
  const bool is_v = blockIdx.x >= nq;
  const int64_t blk = is_v ? blockIdx.x - nq : blockIdx.x;
  const int nb = is_v ? a.nkb : a.nqb, heads = is_v ? a.Hkv : a.H;
  const int64_t bh = blk / nb;
  const int t = (int)(blk - bh * nb), b = (int)(bh / heads), hh = (int)(bh - (int64_t)b * heads);
  const int qlen = seq_len(a.q_lens, b, a.Lq), klen = seq_len(a.k_lens, b, a.Lk);
  const int len = is_v ? klen : qlen;
  const int first = is_v ? 0 : first_query(qlen, klen, a.causal);
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < kNormRows / 32; ++j) {
    const int64_t i = (int64_t)t * kNormRows + 32 * j + (tid >> 3);
    float dot = 0.f, nrm = 0.f;
    if (i >= first && i < len) {
      const u32x4 g = *reinterpret_cast<const u32x4*>(
          is_v ? a.v + b * a.vb + hh * a.vh + i * a.vl + c0
               : a.dout + b * a.gb + hh * a.gh + i * a.gl + c0);
      u32x4 o{0, 0, 0, 0}, ol{0, 0, 0, 0};
      if (!is_v) {
        o = *reinterpret_cast<const u32x4*>(a.o + b * a.ob + hh * a.oh + i * a.ol + c0);
        if (a.o_lo)
          ol = *reinterpret_cast<const u32x4*>(
              a.o_lo + (((int64_t)b * a.Lq + i) * a.H + hh) * kDD + c0);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float gv = T16::to_f32((uint16_t)(g[e] >> (16 * x)));
          dot += gv * (T16::to_f32((uint16_t)(o[e] >> (16 * x))) +
                       T16::to_f32((uint16_t)(ol[e] >> (16 * x))));
          nrm += gv * gv;
        }
    }
#pragma unroll
    for (int s = 4; s >= 1; s >>= 1) {
      dot += __shfl_xor(dot, s, 64);
      if (Shift<T16>::scaled) nrm += __shfl_xor(nrm, s, 64);
    }
    top = fmaxf(top, nrm);
    if (!is_v && c0 == 0 && i < a.Lq) {
      const bool live = i >= first && i < len;
      const int64_t f = bh * a.Lq + i;
      a.ndelta[f] = live ? -dot : 0.f;
      a.nlse[f] = live ? (Shift<T16>::p - a.lse[f] * kLog2e) * a.inv_c : -__builtin_inff();
    }
  }
  if (Shift<T16>::scaled) {
    top = wave_max(top);
    if ((tid & 63) == 0) red[tid >> 6] = top;
    __syncthreads();
    if (tid == 0)
      (is_v ? a.vmax : a.gmax)[blk] =
          sqrtf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
  }
}

// fp16: the power of two m with 2 max|do| max|v| m <= 1 for a key head's group.
__device__ inline float ds_scale(const DenseBwdArgs& a, int b, int hk) {
  const int tid = threadIdx.x, l = tid & 63;
  const int64_t ng = (int64_t)a.rep * a.nqb;
  const float* g = a.gmax + ((int64_t)b * a.H + (int64_t)hk * a.rep) * a.nqb;
  const float* v = a.vmax + ((int64_t)b * a.Hkv + hk) * a.nkb;
  float mg = 0.f, mv = 0.f;
#pragma unroll 8
  for (int64_t i = l; i < ng; i += 64) mg = fmaxf(mg, g[i]);
#pragma unroll 8
  for (int i = l; i < a.nkb; i += 64) mv = fmaxf(mv, v[i]);
  const float bound = 2.f * wave_max(mg) * wave_max(mv);
  if (!(bound > 0.f) || !(bound < 1e38f)) return 1.f;
  int e;
  (void)frexpf(bound, &e);  // bound < 2^e
  e = e < -100 ? -100 : e;
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane((127 - e) << 23));
}

// A C tile pair (dO^T-like, [channel][row]) of a lane's row, 16-bit or fp32 parts.
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

// dq: workgroup = 4 waves x 32 query rows; keys and values in tiles of 64 rows through three
// LDS slots.  dQ^T += K^T dS^T with dS^T straight from the score tile's registers.  (64 rows per
// wave halve the LDS reads but spill at two waves per SIMD: the whole backward 6.04 ms against
// 6.11 at B = 1, H = 8, L = 29,952, 2.96 against 2.93 causal.)
template <typename T16, bool FINE>
__device__ __attribute__((always_inline)) inline void dq_rows(
    const DenseBwdArgs& a, int blk, unsigned char* k0, unsigned char* k1, unsigned char* k2,
    unsigned char* v0, unsigned char* v1, unsigned char* v2) {
  int bh, item;
  if (!work_item(a.dq_map, blk, bh, item)) return;
  const int qt = item / a.dq_splits, sp = item - qt * a.dq_splits;
  const int b = bh / a.H, hq = bh - b * a.H, hk = hq / a.rep;
  const int tid = threadIdx.x, l = tid & 63, h = l >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const LaneOff lo(l);
  const int qlen = seq_len(a.q_lens, b, a.Lq), klen = seq_len(a.k_lens, b, a.Lk);

  const int q0 = qt * 128, qw = q0 + w * 32;
  const int qend = min(q0 + 128, qlen);
  auto limit = [&](int i) __attribute__((always_inline)) {
    if (i >= qlen) return 0;
    if (!a.causal) return klen;
    const int64_t e = (int64_t)i + klen - qlen + 1;
    return e < 0 ? 0 : (e < klen ? (int)e : klen);
  };
  const int kmax = qend > q0 ? limit(qend - 1) : 0;
  const int ntile = (kmax + kTileRows - 1) / kTileRows;
  const int per = (ntile + a.dq_splits - 1) / a.dq_splits;
  const int t0 = sp * per, nt = min(ntile, t0 + per);

  const uint16_t* kp = a.k + b * a.kb + hk * a.kh;
  const uint16_t* vp = a.v + b * a.vb + hk * a.vh;
  const int64_t kld = a.kl * 2, vld = a.vl * 2;
  auto load_tile = [&](int t, unsigned char* kt, unsigned char* vt) __attribute__((always_inline)) {
    const int64_t n = (int64_t)klen - (int64_t)t * kTileRows;
    const auto rk = rows_rsrc(kp, (int64_t)t * kTileRows, n, kld);
    const auto rv = rows_rsrc(vp, (int64_t)t * kTileRows, n, vld);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      dma_rows8(rk, kt, 2 * w + i, (int)kld, l);
      dma_rows8(rv, vt, 2 * w + i, (int)vld, l);
    }
  };

  float mul = 1.f;
  if (Shift<T16>::scaled) mul = ds_scale(a, b, hk);
  const int i = qw + (l & 31);
  const int lim = limit(i);
  const bool live = lim > 0;
  // shift - lse log2e, -delta (times mul)
  const float nl = live ? a.nlse[(int64_t)bh * a.Lq + i] * a.c : -__builtin_inff();
  const float nd = live ? a.ndelta[(int64_t)bh * a.Lq + i] * mul : 0.f;
  u32x4 qf[4], gf[4];
  {
    const uint16_t* qp = a.q + b * a.qb + hq * a.qh + i * a.ql + 8 * h;
    const uint16_t* gp = a.dout + b * a.gb + hq * a.gh + i * a.gl + 8 * h;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      qf[s] = live ? *reinterpret_cast<const u32x4*>(qp + 16 * s) : u32x4{0, 0, 0, 0};
      gf[s] = live ? *reinterpret_cast<const u32x4*>(gp + 16 * s) : u32x4{0, 0, 0, 0};
    }
  }
  // keys that any query of the wave sees, and that all of them see
  const int wlast = min(qw + 32, qlen) - 1;
  const int wany = wlast >= qw ? limit(wlast) : 0;
  const int wall = wlast >= qw ? limit(qw) : 0;
  const bool fine = FINE && (klen <= kFineKeys || wany <= kFineRows || qlen <= kFineRows);

  f32x16 acc[2] = {zero16(), zero16()};
  auto part = [&](auto masked, int base, const unsigned char* kt, const unsigned char* vt)
      __attribute__((always_inline)) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      f32x16 sc = zero16(), dp = zero16();
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        sc = mfma_32x32x16<T16>(row_frag(kt, 32 * kb, s, lo), qf[s], sc);
        dp = mfma_32x32x16<T16>(row_frag(vt, 32 * kb, s, lo), gf[s], dp);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float p = fast_exp2(__builtin_fmaf(sc[e], a.c, nl));
        dp[e] = p * (Shift<T16>::scaled ? __builtin_fmaf(dp[e], mul, nd) : dp[e] + nd);
      }
      if (decltype(masked)::value) {
        const int x = lim - base - 32 * kb - 4 * h;
#pragma unroll
        for (int e = 0; e < 16; ++e) dp[e] = 8 * (e >> 2) + (e & 3) < x ? dp[e] : 0.f;
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const u32x4 ds = pack_step<T16>(dp, s);
        u32x4 kf[2];
#pragma unroll
        for (int mb = 0; mb < 2; ++mb) {
          kf[mb] = col_frag(kt, 32 * kb + 16 * s, mb, lo);
          acc[mb] = mfma_32x32x16<T16>(kf[mb], ds, acc[mb]);
        }
        if (FINE && fine) {
          const u32x4 lost = lost_step<T16>(dp, s, ds);
#pragma unroll
          for (int mb = 0; mb < 2; ++mb) acc[mb] = mfma_32x32x16<T16>(kf[mb], lost, acc[mb]);
        }
      }
    }
  };
  // a tile that every query of the wave sees runs without a branch
  auto compute = [&](int t, const unsigned char* kt, const unsigned char* vt)
      __attribute__((always_inline)) {
    const int base = t * kTileRows;
    if (base + kTileRows <= wall)
      part(std::false_type{}, base, kt, vt);
    else if (base < wany)
      part(std::true_type{}, base, kt, vt);
  };

  load_tile(t0, k0, v0);
  load_tile(t0 + 1, k1, v1);
  for (int t = t0; t < nt; t += 3) {
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(4));
    __builtin_amdgcn_s_barrier();  // tile t has landed, tile t - 1 is read
    load_tile(t + 2, k2, v2);
    compute(t, k0, v0);
    if (t + 1 >= nt) break;
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(4));
    __builtin_amdgcn_s_barrier();
    load_tile(t + 3, k0, v0);
    compute(t + 1, k1, v1);
    if (t + 2 >= nt) break;
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(4));
    __builtin_amdgcn_s_barrier();
    load_tile(t + 4, k1, v1);
    compute(t + 2, k2, v2);
  }
  __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));

  if (i >= a.Lq) return;
  // (the softmax of one key is constant: its dS is the rounding of dP - delta)
  const float f = lim == 1             ? 0.f
                  : Shift<T16>::scaled ? a.scale * (1.f / 32768.f) / mul
                                       : a.scale;
  if (a.dq_splits == 1)
    store_row<T16>(a.dq + b * a.dqb + hq * a.dqh + i * a.dql, acc, f, h, live);
  else
    store_part(a.dq_part + (((int64_t)sp * a.nbh + bh) * a.Lq + i) * kDD, acc, f, h, live);
}

// dk, dv: workgroup = 4 waves x 32 keys of one key head; the query rows of the heads that
// read it are streamed through LDS in tiles of 64, three tiles ahead into four slots, with
// their -lse and -delta, which start the accumulators of S and dP.  The step of 32 rows is
// software-pipelined as in the forward: S and dP of the next step run on the matrix cores
// under this step's exponentials.  B = 1, H = 8, L = 29,952, bf16, launched alone: 3.46 ms, 1.06
// PFLOP/s of its four products (dq 2.7 ms, 1.02 of its three), the clock at the power limit;
// 64 keys per wave, which halves the LDS reads but leaves one wave per SIMD: 3.8.
template <typename T16, bool CAUSAL, bool FINE>
__device__ __attribute__((always_inline)) inline void dkdv_rows(
    const DenseBwdArgs& a, int blk, unsigned char* q0_, unsigned char* q1_, unsigned char* q2_,
    unsigned char* q3_, unsigned char* g0_, unsigned char* g1_, unsigned char* g2_,
    unsigned char* g3_, float (*s0_)[64], float (*s1_)[64], float (*s2_)[64], float (*s3_)[64]) {
  int bk, item;
  if (!work_item(a.kv_map, blk, bk, item)) return;
  const int ktile = item / a.kv_splits, sp = item - ktile * a.kv_splits;
  const int b = bk / a.Hkv, hk = bk - b * a.Hkv;
  const int tid = threadIdx.x, l = tid & 63, h = l >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const LaneOff lo(l);
  const int qlen = seq_len(a.q_lens, b, a.Lq), klen = seq_len(a.k_lens, b, a.Lk);

  const int key0 = ktile * 128, kw = key0 + w * 32;
  // first query that sees a key of the workgroup (causal: i >= j - off)
  const int off = klen - qlen;
  int first = first_query(qlen, klen, a.causal);
  if (CAUSAL) first = max(first, key0 - off);
  const int nq = key0 < klen && first < qlen ? (qlen - first + kTileRows - 1) / kTileRows : 0;
  const int total = nq * a.rep;  // (head, query tile) pairs
  const bool fine = FINE && (total <= kFineRows / kTileRows || klen <= 32);
  const int per = (total + a.kv_splits - 1) / a.kv_splits;
  const int u0 = sp * per, u1 = min(total, u0 + per);

  const int64_t qld = a.ql * 2, gld = a.gl * 2;
  // the tile to load next, and the one to compute (their head of the group and first row)
  int lu = u0, lh = u0 < u1 ? u0 / nq : 0;
  int lrow = first + (u0 < u1 ? u0 - lh * nq : 0) * kTileRows, crow = lrow;
  auto load_tile = [&](unsigned char* qt, unsigned char* gt, float (*st)[64])
      __attribute__((always_inline)) {
    const int hq = hk * a.rep + lh;
    const int64_t n = lu < u1 ? (int64_t)qlen - lrow : 0;
    const auto rq = rows_rsrc(a.q + b * a.qb + hq * a.qh, lrow, n, qld);
    const auto rg = rows_rsrc(a.dout + b * a.gb + hq * a.gh, lrow, n, gld);
    const float* stat = (w & 1) ? a.ndelta : a.nlse;
    const auto rs = make_rsrc(stat + ((int64_t)b * a.H + hq) * a.Lq + lrow,
                              n <= 0 ? 0 : (n < 64 ? n : 64) * 4);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      dma_rows8(rq, qt, 2 * w + i, (int)qld, l);
      dma_rows8(rg, gt, 2 * w + i, (int)gld, l);
    }
    // waves 0 and 2 bring -lse, 1 and 3 -delta (the same values twice)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        rs, (__attribute__((address_space(3))) void*)&st[w & 1][0], 4, 4 * l, 0, 0, 0);
    ++lu;
    lrow += kTileRows;
    if (lrow >= qlen && lu < u1) lrow = first, ++lh;
  };

  float mul = 1.f;
  if (Shift<T16>::scaled) mul = ds_scale(a, b, hk);
  u32x4 kf[4], vf[4];
  {
    const int j = kw + (l & 31);
    const bool live = j < klen;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      kf[s] = live ? *reinterpret_cast<const u32x4*>(a.k + b * a.kb + hk * a.kh + j * a.kl +
                                                     16 * s + 8 * h)
                   : u32x4{0, 0, 0, 0};
      vf[s] = live ? *reinterpret_cast<const u32x4*>(a.v + b * a.vb + hk * a.vh + j * a.vl +
                                                     16 * s + 8 * h)
                   : u32x4{0, 0, 0, 0};
    }
  }
  f32x16 ak[2] = {zero16(), zero16()}, av[2] = {zero16(), zero16()};
  f32x16 sc[2], dp[2];

  // S and dP of rows 32 qb .. of a tile
  auto scores = [&](int qb, const unsigned char* qt, const unsigned char* gt, const float (*st)[64])
      __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(&st[0][32 * qb + 8 * g + 4 * h]);
      const f32x4 y = *reinterpret_cast<const f32x4*>(&st[1][32 * qb + 8 * g + 4 * h]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sc[qb][4 * g + i] = x[i];
        dp[qb][4 * g + i] = y[i];
      }
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      sc[qb] = mfma_32x32x16<T16>(row_frag(qt, 32 * qb, s, lo), kf[s], sc[qb]);
      dp[qb] = mfma_32x32x16<T16>(row_frag(gt, 32 * qb, s, lo), vf[s], dp[qb]);
    }
  };
  // the step of rows 32 qb of this tile; the next one's are rows 32 (qb ^ 1) of (qn, gn, sn)
  auto step = [&](int qb, const unsigned char* qt, const unsigned char* gt, const unsigned char* qn,
                  const unsigned char* gn, const float (*sn)[64]) __attribute__((always_inline)) {
    scores(qb ^ 1, qn, gn, sn);
    f32x16 p;
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = fast_exp2(sc[qb][i] * a.c);
    if (CAUSAL && crow + 32 * qb < kw + 31 - off) {
      asm volatile("");
      const int x = kw + (l & 31) - off - crow - 32 * qb - 4 * h;
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] = 8 * (i >> 2) + (i & 3) >= x ? p[i] : 0.f;
    }
    f32x16 d;
#pragma unroll
    for (int i = 0; i < 16; ++i) d[i] = (Shift<T16>::scaled ? p[i] * mul : p[i]) * dp[qb][i];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const u32x4 pp = pack_step<T16>(p, s), dd = pack_step<T16>(d, s);
      u32x4 gf[2], qf[2];
#pragma unroll
      for (int mb = 0; mb < 2; ++mb) {
        gf[mb] = col_frag(gt, 32 * qb + 16 * s, mb, lo);
        av[mb] = mfma_32x32x16<T16>(gf[mb], pp, av[mb]);
        qf[mb] = col_frag(qt, 32 * qb + 16 * s, mb, lo);
        ak[mb] = mfma_32x32x16<T16>(qf[mb], dd, ak[mb]);
      }
      if (FINE && fine) {
        const u32x4 pl = lost_step<T16>(p, s, pp), dl = lost_step<T16>(d, s, dd);
#pragma unroll
        for (int mb = 0; mb < 2; ++mb) {
          av[mb] = mfma_32x32x16<T16>(gf[mb], pl, av[mb]);
          ak[mb] = mfma_32x32x16<T16>(qf[mb], dl, ak[mb]);
        }
      }
    }
  };
  // Tile i of this range lives in slot i % 4; at its top the tiles up to i + 1 have landed
  // and tile i - 1 is read.  Tiles past the last one are empty (zeros).
  auto tile = [&](const unsigned char* qt, const unsigned char* gt, const float (*st)[64],
                  const unsigned char* qn, const unsigned char* gn, const float (*sn)[64],
                  unsigned char* ql, unsigned char* gl, float (*sl)[64])
                  __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(5));
    __builtin_amdgcn_s_barrier();
    load_tile(ql, gl, sl);
    if (kw < klen) {
      step(0, qt, gt, qt, gt, st);
      step(1, qt, gt, qn, gn, sn);
    }
    if (CAUSAL) {
      crow += kTileRows;
      if (crow >= qlen) crow = first;
    }
  };
  load_tile(q0_, g0_, s0_);
  load_tile(q1_, g1_, s1_);
  load_tile(q2_, g2_, s2_);
  __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(10));
  __builtin_amdgcn_s_barrier();
  scores(0, q0_, g0_, s0_);
  for (int u = u0; u < u1; u += 4) {
    tile(q0_, g0_, s0_, q1_, g1_, s1_, q3_, g3_, s3_);
    if (u + 1 >= u1) break;
    tile(q1_, g1_, s1_, q2_, g2_, s2_, q0_, g0_, s0_);
    if (u + 2 >= u1) break;
    tile(q2_, g2_, s2_, q3_, g3_, s3_, q1_, g1_, s1_);
    if (u + 3 >= u1) break;
    tile(q3_, g3_, s3_, q0_, g0_, s0_, q2_, g2_, s2_);
  }
  __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));

  const float fv = Shift<T16>::scaled ? 1.f / 32768.f : 1.f;
  const float fk = klen == 1            ? 0.f
                   : Shift<T16>::scaled ? a.scale * (1.f / 32768.f) / mul
                                        : a.scale;
  const int j = kw + (l & 31);
  if (j >= a.Lk) return;
  const bool keep = j < klen;
  if (a.kv_splits == 1) {
    store_row<T16>(a.dk + b * a.dkb + hk * a.dkh + j * a.dkl, ak, fk, h, keep);
    store_row<T16>(a.dv + b * a.dvb + hk * a.dvh + j * a.dvl, av, fv, h, keep);
  } else {
    float* d = a.kv_part + (((int64_t)sp * a.nbk + bk) * a.Lk + j) * (2 * kDD);
    store_part(d, ak, fk, h, keep);
    store_part(d + kDD, av, fv, h, keep);
  }
}

// Both in one launch, the workgroups of dk and dv first: neither reads what the other writes,
// so the ones fill the places that the others' last round leaves (and a small call waits for
// the longer of the two, not for both).  The price is one register allocation for two bodies:
// without the lost halves (long sequences) 256 VGPRs, one of them spilled with 24 bytes of scratch;
// 206 to 219 and none spilled with them; 59 to 88 SGPRs kept in lanes of VGPRs in all.
template <typename T16, bool CAUSAL, bool FINE>
__global__ __launch_bounds__(256, 2) void dense_bwd_kernel(DenseBwdArgs a) {
  __shared__ __align__(16) unsigned char a0[kTileB], a1[kTileB], a2[kTileB], a3[kTileB];
  __shared__ __align__(16) unsigned char b0[kTileB], b1[kTileB], b2[kTileB], b3[kTileB];
  __shared__ __align__(16) float s0[2][64], s1[2][64], s2[2][64], s3[2][64];
  const int blk = blockIdx.x;
  if (blk < a.kv_blocks)
    dkdv_rows<T16, CAUSAL, FINE>(a, blk, a0, a1, a2, a3, b0, b1, b2, b3, s0, s1, s2, s3);
  else
    dq_rows<T16, FINE>(a, blk - a.kv_blocks, a0, a1, a2, b0, b1, b2);
}

// Adds the parts of a row of W = 64 (dq) or 128 (dk | dv) channels in order.
template <typename T16, int W>
__global__ __launch_bounds__(256) void dense_bwd_join_kernel(const float* __restrict__ part,
                                                             int splits, int64_t nrows, int64_t L,
                                                             int heads, uint16_t* y0, int64_t b0,
                                                             int64_t h0, int64_t l0, uint16_t* y1,
                                                             int64_t b1, int64_t h1, int64_t l1) {
  const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (e >= nrows * W) return;
  const int64_t row = e / W, bh = row / L, i = row - bh * L;
  const int c = (int)(e - row * W);
  const int64_t b = bh / heads, hh = bh - b * heads;
  f32x4 x{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < splits; ++s)
    x += *reinterpret_cast<const f32x4*>(part + (s * nrows + row) * W + c);
  const u32x2 y{pack_pair<T16>(x[0], x[1]), pack_pair<T16>(x[2], x[3])};
  uint16_t* d = W == 64 || c < 64 ? y0 + b * b0 + hh * h0 + i * l0 + c
                                  : y1 + b * b1 + hh * h1 + i * l1 + (c - 64);
  *reinterpret_cast<u32x2*>(d) = y;
}

struct BwdPlan {
  int64_t qtiles, dq_nwork, ktiles, kv_nwork;
  int dq_splits, kv_splits;
  int64_t nqb, nkb;
  size_t stats, dq_parts, kv_parts;  // floats
};

// even: neither causal nor lengths.  Workgroups of uneven length balance by number: twice
// the ranges.  Backward, us, with ranges for 256 (even) or 512 workgroups of each kind against twice
// as many and against half: L = 2,048, H = 8 51 : 67 : 50; B = 3 clips of up to 4,159, H = 8 over 2, causal
// 149 : 182 : 297, not causal 284 : 301 : 310.
BwdPlan bwd_plan(int dtype, int B, int H, int Hkv, int64_t Lq, int64_t Lk, bool even) {
  BwdPlan p{};
  const int64_t bh = (int64_t)B * H, bk = (int64_t)B * Hkv, rep = H / Hkv;
  p.qtiles = (Lq + 127) / 128;
  auto split = [&](int64_t blocks, int64_t tiles) {
    const int64_t want = even ? 256 : 512;
    if (blocks >= want / 2) return 1;
    const int64_t s = (want + blocks - 1) / blocks, most = tiles / 4;
    return (int)(s < most ? s : (most < 1 ? 1 : most));
  };
  p.dq_splits = split(bh * p.qtiles, (Lk + 63) / 64);
  p.dq_nwork = bh * p.qtiles * p.dq_splits;
  p.ktiles = (Lk + 127) / 128;
  p.kv_splits = split(bk * p.ktiles, rep * ((Lq + 63) / 64));
  p.kv_nwork = bk * p.ktiles * p.kv_splits;
  p.nqb = (Lq + kNormRows - 1) / kNormRows;
  p.nkb = (Lk + kNormRows - 1) / kNormRows;
  p.stats = 2 * bh * Lq + (dtype == SLA2H_DTYPE_F16 ? bh * p.nqb + bk * p.nkb : 0);
  p.stats = (p.stats + 3) & ~(size_t)3;
  p.dq_parts = p.dq_splits > 1 ? (size_t)p.dq_splits * bh * Lq * kDD : 0;
  p.kv_parts = p.kv_splits > 1 ? (size_t)p.kv_splits * bk * Lk * 2 * kDD : 0;
  return p;
}

}  // namespace

}  // namespace sla2h

using namespace sla2h;

extern "C" size_t sla2h_dense_attn_bwd_workspace_bytes(int dtype, int B, int H, int Hkv,
                                                       int64_t Lq, int64_t Lk) {
  if (!sizes_ok(B, H, Hkv, Lq, Lk)) return 0;
  size_t most = 0;
  for (bool even : {false, true}) {
    const BwdPlan p = bwd_plan(dtype, B, H, Hkv, Lq, Lk, even);
    const size_t n = p.stats + p.dq_parts + p.kv_parts;
    most = n > most ? n : most;
  }
  return most * 4;
}

extern "C" int sla2h_dense_attn_bwd(const void* q, const void* k, const void* v, const void* o,
                                    const void* o_lo, const void* dout, const float* lse,
                                    const int64_t* strides, const int32_t* q_lens, const int32_t* k_lens, int dtype,
                                    int B, int H, int Hkv, int64_t Lq, int64_t Lk, int causal,
                                    float scale, void* workspace, void* dq, void* dk, void* dv,
                                    void* stream) {
  SLA2H_CHECK_ARG(q && k && v && o && dout && lse && strides && workspace);
  SLA2H_CHECK_ARG((dq || dk) && !dk == !dv);
  SLA2H_CHECK_ARG(dtype == SLA2H_DTYPE_F16 || dtype == SLA2H_DTYPE_BF16);
  SLA2H_CHECK_ARG(sizes_ok(B, H, Hkv, Lq, Lk));
  SLA2H_CHECK_ARG(scale > 0.f && scale < 1e30f);
  SLA2H_CHECK_ARG(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o | (uintptr_t)dout |
                   (uintptr_t)o_lo | (uintptr_t)workspace | (uintptr_t)dq | (uintptr_t)dk |
                   (uintptr_t)dv) % 16 == 0);
  SLA2H_CHECK_ARG(((uintptr_t)lse | (uintptr_t)q_lens | (uintptr_t)k_lens) % 4 == 0);
  for (int i = 0; i < 24; ++i) SLA2H_CHECK_ARG(strides[i] >= 0 && strides[i] % 8 == 0);
  // rows apart from each other: the range check of a tile's load tells them by their offset
  for (int i : {2, 5, 8, 11, 14, 17, 20, 23}) SLA2H_CHECK_ARG(strides[i] >= kDD);
  // 32-bit byte offsets within a tile of 64 rows
  for (int i : {2, 5, 8, 14}) SLA2H_CHECK_ARG(strides[i] < ((int64_t)1 << 23));
  const bool even = !causal && !q_lens && !k_lens;
  const BwdPlan p = bwd_plan(dtype, B, H, Hkv, Lq, Lk, even);
  SLA2H_CHECK_ARG(p.dq_nwork < ((int64_t)1 << 30) && p.kv_nwork < ((int64_t)1 << 30));
  const int64_t bh = (int64_t)B * H, bk = (int64_t)B * Hkv;
  const int64_t pq = bh * p.nqb, pv = dtype == SLA2H_DTYPE_F16 ? bk * p.nkb : 0;
  SLA2H_CHECK_ARG(pq + pv < ((int64_t)1 << 31));
  DenseBwdArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.o = static_cast<const uint16_t*>(o);
  a.o_lo = static_cast<const uint16_t*>(o_lo);
  a.dout = static_cast<const uint16_t*>(dout);
  a.lse = lse;
  a.dq = static_cast<uint16_t*>(dq);
  a.dk = static_cast<uint16_t*>(dk);
  a.dv = static_cast<uint16_t*>(dv);
  a.q_lens = q_lens;
  a.k_lens = k_lens;
  int64_t* dst[24] = {&a.qb,  &a.qh,  &a.ql,  &a.kb,  &a.kh,  &a.kl,  &a.vb,  &a.vh,
                      &a.vl,  &a.ob,  &a.oh,  &a.ol,  &a.gb,  &a.gh,  &a.gl,  &a.dqb,
                      &a.dqh, &a.dql, &a.dkb, &a.dkh, &a.dkl, &a.dvb, &a.dvh, &a.dvl};
  for (int i = 0; i < 24; ++i) *dst[i] = strides[i];
  a.Lq = Lq;
  a.Lk = Lk;
  a.H = H;
  a.Hkv = Hkv;
  a.rep = H / Hkv;
  a.nbh = (int)bh;
  a.nbk = (int)bk;
  a.causal = causal != 0;
  a.c = scale * kLog2e;
  a.inv_c = 1.f / a.c;
  a.scale = scale;
  a.nlse = static_cast<float*>(workspace);
  a.ndelta = a.nlse + bh * Lq;
  a.gmax = a.ndelta + bh * Lq;
  a.vmax = a.gmax + bh * p.nqb;
  a.nqb = (int)p.nqb;
  a.nkb = (int)p.nkb;
  a.dq_part = a.nlse + p.stats;
  a.kv_part = a.dq_part + p.dq_parts;
  a.dq_map = work_map(bh, p.qtiles * p.dq_splits, even, causal);
  a.kv_map = work_map(bk, p.ktiles * p.kv_splits, even, false);  // causal: the first keys' are longest
  a.kv_blocks = dk ? (int)work_grid(a.kv_map) : 0;
  a.dq_splits = p.dq_splits;
  a.kv_splits = p.kv_splits;
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto go = [&](auto tag) -> int {
    using T16 = decltype(tag);
    int err;
    dense_bwd_prep_kernel<T16><<<(unsigned)(pq + pv), 256, 0, st>>>(a, pq);
    if ((err = (int)hipGetLastError())) return err;
    const unsigned grid = a.kv_blocks + (dq ? work_grid(a.dq_map) : 0);
    if (causal)
      dense_bwd_kernel<T16, true, true><<<grid, 256, 0, st>>>(a);
    else if (Lk <= kFineKeys || Lq <= kFineRows || q_lens || k_lens)  // (sequences, not the padding)
      dense_bwd_kernel<T16, false, true><<<grid, 256, 0, st>>>(a);
    else
      dense_bwd_kernel<T16, false, false><<<grid, 256, 0, st>>>(a);
    if ((err = (int)hipGetLastError())) return err;
    if (dq && p.dq_splits > 1) {
      dense_bwd_join_kernel<T16, kDD>
          <<<(unsigned)((bh * Lq * kDD / 4 + 255) / 256), 256, 0, st>>>(
              a.dq_part, p.dq_splits, bh * Lq, Lq, H, a.dq, a.dqb, a.dqh, a.dql, nullptr, 0, 0, 0);
      if ((err = (int)hipGetLastError())) return err;
    }
    if (dk && p.kv_splits > 1)
      dense_bwd_join_kernel<T16, 2 * kDD>
          <<<(unsigned)((bk * Lk * 2 * kDD / 4 + 255) / 256), 256, 0, st>>>(
              a.kv_part, p.kv_splits, bk * Lk, Lk, Hkv, a.dk, a.dkb, a.dkh, a.dkl, a.dv, a.dvb,
              a.dvh, a.dvl);
    return (int)hipGetLastError();
  };
  return dtype == SLA2H_DTYPE_BF16 ? go(BF16{}) : go(F16{});
}
