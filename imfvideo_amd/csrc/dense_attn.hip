// Dense softmax attention on 64-channel heads, forward, gfx950.
//
//   S = c q k^T over the keys j < k_len (causal: j <= i + k_len - q_len),
//   o = softmax(S) v,  lse = log sum exp S;  a row without a key: o = 0, lse = -inf.
//
// One pass over the keys: O^T += V^T P^T with P = exp2(S - m), row sums beside it, m a
// row bound in log2 units, the maximum of the first keys.  It moves only when a tile's sums
// show that its probabilities have outgrown the range set aside for them (a wave-uniform,
// rarely taken branch computes the tile again and rescales the accumulators): the result
// does not depend on m beyond rounding, and the common path computes no maximum.  P is
// rounded to the operands' 16-bit type for the product (an error of half a unit in its last place
// per term, as the inputs themselves carry); row sums add the fp32 values, so that lse, which
// the backward builds on, is exact to fp32.
#include "dense_attn.h"

#include <initializer_list>

namespace sla2h {

namespace {

constexpr int kFineKeys = 512, kFewBlocks = 256;

struct DenseFwdArgs {
  const uint16_t *q, *k, *v;
  uint16_t *o, *lo;  // lo: (B, Lq, H, 64) or null
  float* lse;
  const int32_t *q_lens, *k_lens;
  int64_t qb, qh, ql, kb, kh, kl, vb, vh, vl, ob, oh, ol;  // strides in elements
  int64_t Lq, Lk;
  int H, Hkv, rep;
  int causal;
  float c;  // scale * log2(e)
  WorkMap map;
  int qtiles, nwork;  // split form: query tiles of a key head, workgroups
  // ranges of keys
  float* part;   // [range][B * H * Lq][64] unnormalised sums
  float2* ml;    // [range][B * H * Lq] (m, l)
  int splits, units;  // split form: 32-key units of a range
  int64_t nrows;      // B * H * Lq
};

// Workgroup = 4 waves x (32 NQ) query rows of one head; all waves read the key and value
// tiles of 64 rows from LDS, loaded three tiles ahead into four slots with one barrier per tile.
// The step of 32 keys is software-pipelined: its scores were computed one step earlier, so
// that the score products of the next step, which depend on nothing here, run on the matrix
// cores under this step's exponentials; operands of the step after are read from LDS meanwhile.
// 64 rows per wave at B = 1, H = 8, L = 29,952, bf16: 1.78 ms, 1.03 PFLOP/s (8192^3 matrix product of
// the library on the same card 1.25); MFMA 48 %, VALU 61 % busy, the clock at the power limit.
// FINE: waves whose rows see at most kFineKeys keys add what the rounding of P lost with a
// second product.  delta = dO . O of the backward inherits that rounding, and dS = P (dP - delta)
// shows it where few keys share a row (77 keys: dq and dk 2.6e-3 off against 2.4e-3, of which the
// roundings of dS and of the result are 2.4e-3).  Longer rows keep the one rounding of P (the
// second product would be half as many matrix instructions again): o is then 2.3e-3 off in bf16
// (2-norm; its own rounding alone 1.7e-3).  Without gradients the same, so that both calls
// give the same output.
template <typename T16, int NQ, bool FINE>
__global__ __launch_bounds__(256, 2) void dense_fwd_kernel(DenseFwdArgs a) {
  __shared__ __align__(16) unsigned char k0[kTileB], k1[kTileB], k2[kTileB], k3[kTileB];
  __shared__ __align__(16) unsigned char v0[kTileB], v1[kTileB], v2[kTileB], v3[kTileB];
  int bh, item;
  if (!work_item(a.map, blockIdx.x, bh, item)) return;
  const int qt = item / a.splits, sp = item - qt * a.splits;
  const int b = bh / a.H, hq = bh - b * a.H, hk = hq / a.rep;
  const int tid = threadIdx.x, l = tid & 63, h = l >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const LaneOff lo(l);
  const int qlen = seq_len(a.q_lens, b, a.Lq), klen = seq_len(a.k_lens, b, a.Lk);

  const int q0 = qt * (128 * NQ);           // first row of the workgroup
  const int qw = q0 + w * (32 * NQ);        // ... of the wave
  const int qend = min(q0 + 128 * NQ, qlen);
  const int kmax = qend > q0 ? key_limit(qend - 1, qlen, klen, a.causal) : 0;
  const int ntile = (kmax + kTileRows - 1) / kTileRows;
  const int per = (ntile + a.splits - 1) / a.splits;
  const int t0 = sp * per, nt = min(ntile, t0 + per);  // this range's tiles

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

  u32x4 qf[NQ][4];
  int lim[NQ];
  {
    const uint16_t* qp = a.q + b * a.qb + hq * a.qh;
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

  f32x16 acc[NQ][2];
  float m[NQ], lsum[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    acc[n][0] = zero16();
    acc[n][1] = zero16();
    m[n] = kFloor;
    lsum[n] = 0.f;
  }

  f32x16 sc[2][NQ];
  u32x4 kf[4];
  auto read_k = [&](const unsigned char* kt, int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < 4; ++s) kf[s] = row_frag(kt, 32 * kb, s, lo);
  };
  auto scores = [&](int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < NQ; ++n) sc[kb][n] = zero16();
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int n = 0; n < NQ; ++n) sc[kb][n] = mfma_32x32x16<T16>(kf[s], qf[n][s], sc[kb][n]);
  };
  auto mask = [&](int kb, int base) __attribute__((always_inline)) {
    if (base + 32 > wall) {
      asm volatile("");  // a branch: rare, and 64 selects when speculated
#pragma unroll
      for (int n = 0; n < NQ; ++n) mask_tile(sc[kb][n], lim[n] - base, h);
    }
  };
  auto raise = [&](int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < NQ; ++n)
      raise_bound(lane_max(sc[kb][n]), a.c, m[n], lsum[n], acc[n]);
  };
  // one step: keys 32 kb .. of tile t; rows 32 kb .. of kn are the step after next
  auto step = [&](int t, int kb, const unsigned char* kt, const unsigned char* vt,
                  const unsigned char* kn) __attribute__((always_inline)) {
    const int base = t * kTileRows + 32 * kb;
    u32x4 vf[2][2], p[NQ][2];
    float r[NQ];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int mb = 0; mb < 2; ++mb) vf[s][mb] = col_frag(vt, 32 * kb + 16 * s, mb, lo);
    mask(kb, base);
    scores(kb ^ 1);
    read_k(kn, kb);
#pragma unroll
    for (int n = 0; n < NQ; ++n) r[n] = probabilities<T16>(sc[kb][n], a.c, m[n], p[n]);
    bool over = r[0] > Range<T16>::most;
    if (NQ == 2) over = over || r[NQ - 1] > Range<T16>::most;
    if (__builtin_amdgcn_ballot_w64(over)) {  // the step's scores again, under a new bound
      read_k(kt, kb);
      scores(kb);
      mask(kb, base);
      raise(kb);
#pragma unroll
      for (int n = 0; n < NQ; ++n) r[n] = probabilities<T16>(sc[kb][n], a.c, m[n], p[n]);
      read_k(kn, kb);
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) lsum[n] += r[n];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int n = 0; n < NQ; ++n)
          acc[n][mb] = mfma_32x32x16<T16>(vf[s][mb], p[n][s], acc[n][mb]);
    if (FINE && wany <= kFineKeys) {
      asm volatile("");
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        u32x4 q[2];
        lost_halves<T16>(sc[kb][n], a.c, m[n], p[n], q);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int mb = 0; mb < 2; ++mb)
            acc[n][mb] = mfma_32x32x16<T16>(vf[s][mb], q[s], acc[n][mb]);
      }
    }
  };
  // Tile t0 + i lives in slot i % 4; tiles past the sequence are empty (zeros).  At the top of
  // tile t the tiles up to t + 1 have landed and tile t - 1 is read.
  auto tile = [&](int t, const unsigned char* kt, const unsigned char* vt,
                  const unsigned char* kt1, unsigned char* kl, unsigned char* vl)
      __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(4));
    __builtin_amdgcn_s_barrier();
    load_tile(t + 3, kl, vl);
    if (t * kTileRows >= wany) return;
    step(t, 0, kt, vt, kt1);
    step(t, 1, kt, vt, kt1);
  };
  load_tile(t0, k0, v0);
  load_tile(t0 + 1, k1, v1);
  load_tile(t0 + 2, k2, v2);
  __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(8));
  __builtin_amdgcn_s_barrier();
  read_k(k0, 0);
  scores(0);
  mask(0, t0 * kTileRows);
  raise(0);
  read_k(k0, 1);
  for (int t = t0; t < nt; t += 4) {
    tile(t, k0, v0, k1, k3, v3);
    if (t + 1 >= nt) break;
    tile(t + 1, k1, v1, k2, k0, v0);
    if (t + 2 >= nt) break;
    tile(t + 2, k2, v2, k3, k1, v1);
    if (t + 3 >= nt) break;
    tile(t + 3, k3, v3, k0, k2, v2);
  }
  __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));  // no load into this LDS outlives the workgroup

  uint16_t* op = a.o + b * a.ob + hq * a.oh;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int i = qw + 32 * n + (l & 31);
    if (i >= a.Lq) continue;
    const float ls = swap32_sum(lsum[n]);
    if (a.splits > 1) {
      const int64_t flat = sp * a.nrows + (int64_t)bh * a.Lq + i;
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(a.part + flat * kDD + 32 * mb + 8 * g + 4 * h) =
              f32x4{acc[n][mb][4 * g], acc[n][mb][4 * g + 1], acc[n][mb][4 * g + 2],
                    acc[n][mb][4 * g + 3]};
      if (h == 0) a.ml[flat] = make_float2(m[n], ls);
      continue;
    }
    const float inv = 1.f / ls;  // a row whose scores are all -inf is NaN
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        u32x2 x, y;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t lost;
          x[e] = round_pair<T16>(acc[n][mb][4 * g + 2 * e] * inv,
                                 acc[n][mb][4 * g + 2 * e + 1] * inv, lost);
          y[e] = lost;
        }
        const int c = 32 * mb + 8 * g + 4 * h;
        *reinterpret_cast<u32x2*>(op + i * a.ol + c) = lim[n] > 0 ? x : u32x2{0, 0};
        if (a.lo)
          *reinterpret_cast<u32x2*>(a.lo + (((int64_t)b * a.Lq + i) * a.H + hq) * kDD + c) =
              lim[n] > 0 ? y : u32x2{0, 0};
      }
    if (a.lse && h == 0)
      a.lse[(int64_t)bh * a.Lq + i] =
          lim[n] > 0 ? (m[n] - Range<T16>::shift + __log2f(ls)) * kLn2 : -__builtin_inff();
  }
}

// Few queries: workgroup = 32 rows (of the `rep` query heads that share a key head) over one
// range of keys; its waves take the 32-key units in turn, each with LDS slots of its own (no
// barrier in the loop), and their sums are joined in LDS: one query over 29,952 and 18,720 keys
// of 8 heads (99.7 MB) in 24.5 us, 4.1 TB/s, at best 23.8 (called again and again, so that part of them
// may still be in the last-level cache).  With one range the result is final, else a second kernel
// adds the ranges in order.
// What the rounding of P lost is added over any number of keys where at most kFewBlocks blocks
// of rows leave the matrix cores idle under the loads; us, without : with, H = 8: one query as above 29.2 :
// 30.2 a call, L = 1,024 (256 blocks) 25.3 : 25.8, but L = 1,500 (376) 37 : 40, 2,048 (512) 22 : 26.
template <typename T16, bool FEW>
__global__ __launch_bounds__(256, 2) void dense_fwd_split_kernel(DenseFwdArgs a) {
  constexpr int kUnitB = 32 * kRowB;
  __shared__ __align__(16) unsigned char kv0[4][2 * kUnitB], kv1[4][2 * kUnitB];
  __shared__ float mls[4][2][32];
  const int blk = blockIdx.x / a.splits, sp = blockIdx.x - blk * a.splits;
  const int bk = __builtin_amdgcn_readfirstlane(blk / a.qtiles);
  const int qt = __builtin_amdgcn_readfirstlane(blk - bk * a.qtiles);
  const int b = bk / a.Hkv, hk = bk - b * a.Hkv;
  const int tid = threadIdx.x, l = tid & 63, h = l >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const LaneOff lo(l);
  const int qlen = seq_len(a.q_lens, b, a.Lq), klen = seq_len(a.k_lens, b, a.Lk);

  // row of the group: head hk rep + row / Lq, query row % Lq
  const int64_t row = (int64_t)qt * 32 + (l & 31);
  const bool live = row < (int64_t)a.rep * a.Lq;
  const int hq = hk * a.rep + (live ? (int)(row / a.Lq) : 0);
  const int i = live ? (int)(row % a.Lq) : 0;
  const int lim = live ? key_limit(i, qlen, klen, a.causal) : 0;
  int kmax = lim, kmin = lim;
#pragma unroll
  for (int s = 16; s >= 1; s >>= 1) {
    kmax = max(kmax, __shfl_xor(kmax, s, 64));
    kmin = min(kmin, __shfl_xor(kmin, s, 64));
  }
  kmax = __builtin_amdgcn_readfirstlane(kmax);
  kmin = __builtin_amdgcn_readfirstlane(kmin);

  const uint16_t* kp = a.k + b * a.kb + hk * a.kh;
  const uint16_t* vp = a.v + b * a.vb + hk * a.vh;
  const int64_t kld = a.kl * 2, vld = a.vl * 2;
  const int64_t u0 = (int64_t)sp * a.units;
  const int64_t uend = min(u0 + a.units, ((int64_t)kmax + 31) / 32);
  auto load_unit = [&](int64_t u, unsigned char* kv) __attribute__((always_inline)) {
    const int64_t n = u < uend ? min((int64_t)klen - u * 32, (int64_t)32) : 0;
    const auto rk = rows_rsrc(kp, u * 32, n, kld);
    const auto rv = rows_rsrc(vp, u * 32, n, vld);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      dma_rows8(rk, kv, j, (int)kld, l);
      dma_rows8(rv, kv + kUnitB, j, (int)vld, l);
    }
  };

  u32x4 qf[4];
  {
    const uint16_t* qp = a.q + b * a.qb + hq * a.qh + i * a.ql;
#pragma unroll
    for (int s = 0; s < 4; ++s)
      qf[s] = lim > 0 ? *reinterpret_cast<const u32x4*>(qp + 16 * s + 8 * h) : u32x4{0, 0, 0, 0};
  }
  f32x16 acc[2] = {zero16(), zero16()};
  float m = kFloor, lsum = 0.f;
  const bool fine = FEW || kmax <= kFineKeys;
  auto compute = [&](int64_t u, const unsigned char* kv) __attribute__((always_inline)) {
    f32x16 sc = zero16();
#pragma unroll
    for (int s = 0; s < 4; ++s) sc = mfma_32x32x16<T16>(row_frag(kv, 0, s, lo), qf[s], sc);
    if (u * 32 + 32 > kmin) mask_tile(sc, (int)(lim - u * 32), h);
    // the wave's first unit sets the bound of the rows that see a key of it
    u32x4 p[2];
    float r = probabilities<T16>(sc, a.c, m, p);
    if (__builtin_amdgcn_ballot_w64(r > Range<T16>::most)) {
      raise_bound(lane_max(sc), a.c, m, lsum, acc);
      r = probabilities<T16>(sc, a.c, m, p);
    }
    lsum += r;
    u32x4 q[2];
    if (fine) lost_halves<T16>(sc, a.c, m, p, q);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int mb = 0; mb < 2; ++mb) {
        const u32x4 vf = col_frag(kv + kUnitB, 16 * s, mb, lo);
        acc[mb] = mfma_32x32x16<T16>(vf, p[s], acc[mb]);
        if (fine) acc[mb] = mfma_32x32x16<T16>(vf, q[s], acc[mb]);
      }
  };
  int64_t u = u0 + w;
  load_unit(u, kv0[w]);
  for (; u < uend; u += 8) {
    load_unit(u + 4, kv1[w]);
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(8));
    compute(u, kv0[w]);
    if (u + 4 >= uend) break;
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(8));
    load_unit(u + 8, kv0[w]);
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(8));
    compute(u + 4, kv1[w]);
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(8));
  }
  __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));

  // join the four waves: fp32 O^T tiles [channel][row] in the slots' memory
  lsum = swap32_sum(lsum);
  if (h == 0) {
    mls[w][0][l] = m;
    mls[w][1][l] = lsum;
  }
  float* ot = reinterpret_cast<float*>(w < 2 ? kv0[2 * w] : kv1[2 * (w - 2)]);
  __syncthreads();
#pragma unroll
  for (int mb = 0; mb < 2; ++mb)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      ot[(32 * mb + 8 * (r >> 2) + 4 * h + (r & 3)) * 32 + (l & 31)] = acc[mb][r];
  __syncthreads();
  // thread: row tid % 32, channels 8 (tid / 32) ..
  const int r = tid & 31, c0 = (tid >> 5) * 8;
  float mm = fmaxf(fmaxf(mls[0][0][r], mls[1][0][r]), fmaxf(mls[2][0][r], mls[3][0][r]));
  float f[4], ll = 0.f, x[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[j] = fast_exp2(mls[j][0][r] - mm);
    ll += f[j] * mls[j][1][r];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float* src = reinterpret_cast<const float*>(j < 2 ? kv0[2 * j] : kv1[2 * (j - 2)]);
      x[e] += f[j] * src[(c0 + e) * 32 + r];
    }
  }
  const int64_t orow = (int64_t)qt * 32 + r;
  if (orow >= (int64_t)a.rep * a.Lq) return;
  const int oh = hk * a.rep + (int)(orow / a.Lq), oi = (int)(orow % a.Lq);
  const int64_t flat = ((int64_t)b * a.H + oh) * a.Lq + oi;
  if (a.splits > 1) {
    float* d = a.part + (sp * a.nrows + flat) * kDD + c0;
    *reinterpret_cast<f32x4*>(d) = f32x4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<f32x4*>(d + 4) = f32x4{x[4], x[5], x[6], x[7]};
    if (c0 == 0) a.ml[sp * a.nrows + flat] = make_float2(mm, ll);
    return;
  }
  const bool some = key_limit(oi, qlen, klen, a.causal) > 0;
  const float inv = 1.f / ll;
  u32x4 y, z;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t lost;
    const uint32_t p = round_pair<T16>(x[2 * e] * inv, x[2 * e + 1] * inv, lost);
    y[e] = some ? p : 0u;
    z[e] = some ? lost : 0u;
  }
  *reinterpret_cast<u32x4*>(a.o + b * a.ob + oh * a.oh + oi * a.ol + c0) = y;
  if (a.lo)
    *reinterpret_cast<u32x4*>(a.lo + (((int64_t)b * a.Lq + oi) * a.H + oh) * kDD + c0) = z;
  if (a.lse && c0 == 0)
    a.lse[flat] = some ? (mm - Range<T16>::shift + __log2f(ll)) * kLn2 : -__builtin_inff();
}

// Joins the key ranges of a row: a workgroup's 16 groups of 16 lanes (four channels each) take
// the ranges in turn, and their sums are added in order (the ranges come in the tens
// where rows are few, so that one group alone would wait for one load after the other).
template <typename T16>
__global__ __launch_bounds__(256) void dense_join_kernel(DenseFwdArgs a) {
  __shared__ float sm[16], sl[16];
  __shared__ f32x4 sx[16][16];
  const int64_t flat = blockIdx.x;
  const int grp = threadIdx.x >> 4, c0 = (threadIdx.x & 15) * 4;
  const int64_t bh = flat / a.Lq;
  const int i = (int)(flat - bh * a.Lq), b = (int)(bh / a.H), hq = (int)(bh - (int64_t)b * a.H);
  const int qlen = seq_len(a.q_lens, b, a.Lq), klen = seq_len(a.k_lens, b, a.Lk);
  float mm = kFloor, ll = 0.f;
  f32x4 x{0.f, 0.f, 0.f, 0.f};
  for (int s = grp; s < a.splits; s += 16) {
    const float2 ml = a.ml[s * a.nrows + flat];
    const f32x4 y = *reinterpret_cast<const f32x4*>(a.part + (s * a.nrows + flat) * kDD + c0);
    const float mn = fmaxf(mm, ml.x), f = fast_exp2(mm - mn), g = fast_exp2(ml.x - mn);
    mm = mn;
    ll = ll * f + g * ml.y;
    x = x * f + g * y;
  }
  sx[grp][threadIdx.x & 15] = x;
  if (c0 == 0) sm[grp] = mm, sl[grp] = ll;
  __syncthreads();
  if (grp) return;
#pragma unroll
  for (int j = 0; j < 16; ++j) mm = fmaxf(mm, sm[j]);
  ll = 0.f;
  x = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float f = fast_exp2(sm[j] - mm);
    ll += f * sl[j];
    x += f * sx[j][threadIdx.x & 15];
  }
  const bool some = key_limit(i, qlen, klen, a.causal) > 0;
  const float inv = 1.f / ll;
  u32x2 y, z;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    uint32_t lost;
    const uint32_t p = round_pair<T16>(x[2 * e] * inv, x[2 * e + 1] * inv, lost);
    y[e] = some ? p : 0u;
    z[e] = some ? lost : 0u;
  }
  *reinterpret_cast<u32x2*>(a.o + b * a.ob + hq * a.oh + i * a.ol + c0) = y;
  if (a.lo)
    *reinterpret_cast<u32x2*>(a.lo + (((int64_t)b * a.Lq + i) * a.H + hq) * kDD + c0) = z;
  if (a.lse && c0 == 0)
    a.lse[flat] = some ? (mm - Range<T16>::shift + __log2f(ll)) * kLn2 : -__builtin_inff();
}

// The form of a call: query blocks of 256 or 128 rows, or of 32 rows of a key head's group.
struct FwdPlan {
  int nq;  // 2, 1: dense_fwd_kernel<NQ>; 0: dense_fwd_split_kernel
  int64_t qtiles, nwork;
  int splits;  // ranges of keys
  int64_t units;
  bool few;  // nq = 0: at most kFewBlocks blocks of rows
};

// even: neither causal nor lengths
FwdPlan fwd_plan(int B, int H, int Hkv, int64_t Lq, int64_t Lk, bool even) {
  FwdPlan p{};
  const int64_t bh = (int64_t)B * H;
  p.splits = 1;
  p.qtiles = (Lq + 255) / 256;
  p.nwork = bh * p.qtiles;
  // 64 rows per wave read each operand from LDS half as often, 32 rows make twice as many
  // workgroups.  us, 256 against 128 rows per workgroup: even tiles B = 1, H = 8, L = 29,952
  // (936 workgroups) 1,784 : 2,027, L = 8,192 (256) 153 : 154; causal L = 29,952 889 : 951, L = 8,192
  // 143 : 100; B = 3, L = 4,159 (408) 111 : 83.
  p.nq = 2;
  if (p.nwork >= (even ? 256 : 768)) return p;
  p.nq = 1;
  p.qtiles = (Lq + 127) / 128;
  p.nwork = bh * p.qtiles;
  if (p.nwork >= 256) return p;
  // ... with ranges of keys where blocks of 32 rows would read all keys over and over; us, so and
  // in blocks of 32 rows: 77 queries over 29,952 keys, H = 8, 23 : 39; 300 48 : 91; 2,000, H = 1, 32 : 50; L =
  // 1,500, H = 4 23 : 24; but L = 2,048, H = 8 (128 workgroups) 41 : 19, where the parts weigh more
  if (p.nwork <= 64 && Lq > 48 && Lk >= 1024) {
    const int64_t tiles = (Lk + kTileRows - 1) / kTileRows, most = tiles / 4;
    const int64_t s = (512 + p.nwork - 1) / p.nwork;
    p.splits = (int)(s < most ? s : most);
    return p;
  }
  p.nq = 0;
  p.qtiles = ((H / Hkv) * Lq + 31) / 32;
  const int64_t blocks = (int64_t)B * Hkv * p.qtiles, units = (Lk + 31) / 32;
  p.few = blocks <= kFewBlocks;
  int64_t s = (512 + blocks - 1) / blocks;
  const int64_t most = units / 8;  // two units per wave and range at least
  s = s < most ? s : most;
  p.splits = s < 1 ? 1 : (int)s;
  p.units = (units + p.splits - 1) / p.splits;
  p.splits = (int)((units + p.units - 1) / p.units);
  p.nwork = blocks * p.splits;
  return p;
}

}  // namespace

}  // namespace sla2h

using namespace sla2h;

extern "C" size_t sla2h_dense_attn_fwd_workspace_bytes(int B, int H, int Hkv, int64_t Lq,
                                                       int64_t Lk) {
  if (!sizes_ok(B, H, Hkv, Lq, Lk)) return 0;
  const FwdPlan p = fwd_plan(B, H, Hkv, Lq, Lk, true);  // the split form does not depend on it
  return p.splits > 1 ? (size_t)p.splits * B * H * Lq * (kDD * 4 + 8) : 0;
}

extern "C" int sla2h_dense_attn_fwd(const void* q, const void* k, const void* v,
                                    const int64_t* strides, const int32_t* q_lens,
                                    const int32_t* k_lens, int dtype, int B, int H, int Hkv,
                                    int64_t Lq, int64_t Lk, int causal, float scale,
                                    void* workspace, void* o, float* lse, void* o_lo,
                                    void* stream) {
  SLA2H_CHECK_ARG(q && k && v && strides && o);
  SLA2H_CHECK_ARG(dtype == SLA2H_DTYPE_F16 || dtype == SLA2H_DTYPE_BF16);
  SLA2H_CHECK_ARG(sizes_ok(B, H, Hkv, Lq, Lk));
  SLA2H_CHECK_ARG(scale > 0.f && scale < 1e30f);
  SLA2H_CHECK_ARG(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o |
                   (uintptr_t)o_lo | (uintptr_t)workspace) % 16 == 0);
  SLA2H_CHECK_ARG(((uintptr_t)lse | (uintptr_t)q_lens | (uintptr_t)k_lens) % 4 == 0);
  for (int i = 0; i < 12; ++i) SLA2H_CHECK_ARG(strides[i] >= 0 && strides[i] % 8 == 0);
  // rows apart from each other: the range check of a tile's load tells them by their offset
  for (int i : {2, 5, 8, 11}) SLA2H_CHECK_ARG(strides[i] >= kDD);
  // 32-bit byte offsets within a tile of 64 rows
  SLA2H_CHECK_ARG(strides[5] < ((int64_t)1 << 23) && strides[8] < ((int64_t)1 << 23));
  const bool even = !causal && !q_lens && !k_lens;
  const FwdPlan p = fwd_plan(B, H, Hkv, Lq, Lk, even);
  SLA2H_CHECK_ARG(p.splits == 1 || workspace);
  SLA2H_CHECK_ARG(p.nwork < ((int64_t)1 << 30));
  DenseFwdArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.o = static_cast<uint16_t*>(o);
  a.lo = static_cast<uint16_t*>(o_lo);
  a.lse = lse;
  a.q_lens = q_lens;
  a.k_lens = k_lens;
  a.qb = strides[0], a.qh = strides[1], a.ql = strides[2];
  a.kb = strides[3], a.kh = strides[4], a.kl = strides[5];
  a.vb = strides[6], a.vh = strides[7], a.vl = strides[8];
  a.ob = strides[9], a.oh = strides[10], a.ol = strides[11];
  a.Lq = Lq;
  a.Lk = Lk;
  a.H = H;
  a.Hkv = Hkv;
  a.rep = H / Hkv;
  a.causal = causal != 0;
  a.c = scale * kLog2e;
  a.qtiles = (int)p.qtiles;
  a.nwork = (int)p.nwork;
  a.map = work_map((int64_t)B * H, p.qtiles * (p.nq ? p.splits : 1), even, causal);
  a.splits = p.splits;
  a.units = (int)p.units;
  a.nrows = (int64_t)B * H * Lq;
  if (p.splits > 1) {
    a.part = static_cast<float*>(workspace);
    a.ml = reinterpret_cast<float2*>(a.part + (int64_t)p.splits * a.nrows * kDD);
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto go = [&](auto tag) -> int {
    using T16 = decltype(tag);
    const unsigned grid = work_grid(a.map);
    // (a wave decides by the keys that its rows see: with causal order or lengths any may be few)
    const bool fine = Lk <= kFineKeys || causal || k_lens;
    if (p.nq == 2 && fine)
      dense_fwd_kernel<T16, 2, true><<<grid, 256, 0, st>>>(a);
    else if (p.nq == 2)
      dense_fwd_kernel<T16, 2, false><<<grid, 256, 0, st>>>(a);
    else if (p.nq == 1 && fine)
      dense_fwd_kernel<T16, 1, true><<<grid, 256, 0, st>>>(a);
    else if (p.nq == 1)
      dense_fwd_kernel<T16, 1, false><<<grid, 256, 0, st>>>(a);
    else if (p.few)
      dense_fwd_split_kernel<T16, true><<<a.nwork, 256, 0, st>>>(a);
    else
      dense_fwd_split_kernel<T16, false><<<a.nwork, 256, 0, st>>>(a);
    const int err = (int)hipGetLastError();
    if (err || p.splits == 1) return err;
    dense_join_kernel<T16><<<(unsigned)a.nrows, 256, 0, st>>>(a);
    return (int)hipGetLastError();
  };
  return dtype == SLA2H_DTYPE_BF16 ? go(BF16{}) : go(F16{});
}
