// Orthogonalised updates by Newton-Schulz products, gfx950: for each of n matrices G (R, C)
//
//   X = G / |G|_F (the shorter side as rows: r x m),  A = X X^T,  X <- a X + (b A + c A^2) X
//
// some steps, each with coefficients of its own, back in G's type and layout.  A and b A + c A^2
// are symmetric: the tiles above the diagonal are computed and written twice.
//
// Small singular values grow by a in every step (3.4445^5 = 485 in five), and what rounding adds
// to their directions grows with them: in one 16-bit number per element the result would
// be 1e-2 off.  Every intermediate is therefore a pair of fp16 numbers hi + lo, 22 bits of a value
// scaled by a power of two that keeps lo a normal number (absolute resolution 2^-25 of a unit), and a
// product of two pairs is three products of the matrix cores, hi hi + hi lo + lo hi, summed in fp32:
// lo lo, below 2^-24 of the product, is what fp32 arithmetic rounds off too.  (In A^2 of up to 128 rows,
// where the squares of the diagonal's lo show, it is the fourth: 20 rows 0.7e-6 off otherwise.)  The result
// is as exact as with fp32 products, at three times the 16-bit rate's cost.
#include "dense_attn.h"

#include <initializer_list>

namespace sla2h {

namespace {

// Powers of two that the planes are scaled with: |X| and |A| below 15.99, |b A + c A^2| below 127.9
// (singular values of X stay below 1.3 with the usual coefficients) keep hi, an fp16 number, finite.
constexpr float kScaleX = 4096.f, kScaleB = 512.f;

// A matrix of pairs: rows of blocks of 32 columns, [32 hi | 32 lo] each, 128 bytes: the row of an LDS
// tile, so that one load brings both halves.  Element of the block's first half for column j:
__device__ inline int64_t pair_index(int64_t i, int j, int ld) {
  return i * 2 * ld + 2 * (j & ~31) + (j & 31);
}

struct OrthoArgs {
  const void* g;        // (n, R, C)
  void* out;
  double* sums;         // (n, parts) partial sums of squares
  uint16_t *x, *y;      // (n, rp, mp) pairs: the step's X and the next one
  uint16_t *A, *B;      // (n, rp, rp) pairs
  int64_t n, count;     // matrices, elements of one
  int R, C, r, m, rp, mp, parts;
  bool turn;            // rows of X are G's columns
  bool wide_out;        // eight neighbours of a row of out can be stored at once
  float a, b, c;
};

__device__ inline float load_g(const OrthoArgs& a, int dtype, int64_t i) {
  if (dtype == 2) return static_cast<const float*>(a.g)[i];
  const uint16_t v = static_cast<const uint16_t*>(a.g)[i];
  return dtype == SLA2H_DTYPE_BF16 ? BF16::to_f32(v) : F16::to_f32(v);
}

__device__ inline double wave_sum(double v) {
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) v += __shfl_xor(v, s, 64);
  return v;
}

// Partial sums of squares in double: no overflow of a float's square, and the same sum whatever
// the launch.  Thread by thread over the part (multiples of eight values), then a tree.
__global__ __launch_bounds__(256) void ortho_norm_kernel(OrthoArgs a, int dtype, int aligned) {
  __shared__ double red[4];
  const int64_t mat = blockIdx.x / a.parts;
  const int part = (int)(blockIdx.x - mat * a.parts);
  const int64_t per = ((a.count + a.parts - 1) / a.parts + 7) & ~(int64_t)7;
  const int64_t lo = part * per, hi = lo + per < a.count ? lo + per : a.count;
  double s = 0.0;
#pragma unroll 2
  for (int64_t i = lo + 8 * (int)threadIdx.x; i < hi; i += 2048) {
    float v[8];
    const int64_t at = mat * a.count + i;
    if (aligned && i + 8 <= hi) {
      if (dtype == 2) {
        const f32x4* q = reinterpret_cast<const f32x4*>(static_cast<const float*>(a.g) + at);
        const f32x4 x = q[0], y = q[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = x[e], v[4 + e] = y[e];
      } else {
        const u32x4 x = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.g) + at);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint16_t u = (uint16_t)(x[e >> 1] >> (16 * (e & 1)));
          v[e] = dtype == SLA2H_DTYPE_BF16 ? BF16::to_f32(u) : F16::to_f32(u);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = i + e < hi ? load_g(a, dtype, at + e) : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s += (double)v[e] * (double)v[e];
  }
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) a.sums[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// x plus, or minus, half E of a packed pair of fp16 numbers: one instruction that widens as it reads
template <int E>
__device__ inline float minus_half(float x, uint32_t p) {
  float d;
  if (E)
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d) : "v"(p), "v"(x));
  else
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(d) : "v"(p), "v"(x));
  return d;
}
__device__ inline float pair_at(uint32_t hi, uint32_t lo, int e) {
  float d;
  if (e)
    asm("v_fma_mix_f32 %0, %1, 1.0, %2 op_sel:[1,0,1] op_sel_hi:[1,0,1]" : "=v"(d) : "v"(hi), "v"(lo));
  else
    asm("v_fma_mix_f32 %0, %1, 1.0, %2 op_sel_hi:[1,0,1]" : "=v"(d) : "v"(hi), "v"(lo));
  return d;
}
// hi and lo of two scaled values
__device__ inline void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pack_pair<F16>(x, y);
  lo = pack_pair<F16>(minus_half<0>(x, hi), minus_half<1>(y, hi));
}
__device__ inline void split4(const float (&v)[4], u32x2& hi, u32x2& lo) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    uint32_t a, b;
    split2(v[2 * e], v[2 * e + 1], a, b);
    hi[e] = a;
    lo[e] = b;
  }
}

// X of the first step, zeros up to the padded sizes; a 64 x 64 tile per workgroup, turned through
// LDS where G's columns become rows.
__global__ __launch_bounds__(256) void ortho_split_kernel(OrthoArgs a, int dtype) {
  __shared__ float tile[64][65];
  const int tm = a.mp / 64, tr = a.rp / 64;
  const int64_t mat = blockIdx.x / (tm * tr);
  const int t = (int)(blockIdx.x - mat * (tm * tr)), i0 = t / tm * 64, j0 = t % tm * 64;
  const int q = threadIdx.x & 63, w = threadIdx.x >> 6;
  // G's rows of the tile, 64 lanes side by side; all of them under way before the sum is needed
  const int g0 = a.turn ? j0 : i0, h0 = a.turn ? i0 : j0;
  float g[16];
  uint16_t raw[16];
  const int64_t first = mat * a.count + (int64_t)(g0 + w) * a.C + h0 + q;
  const bool in = h0 + q < a.C;
  if (dtype == 2) {
#pragma unroll
    for (int k = 0; k < 16; ++k)
      g[k] = in && g0 + w + 4 * k < a.R
                 ? static_cast<const float*>(a.g)[first + (int64_t)(4 * k) * a.C] : 0.f;
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k)
      raw[k] = in && g0 + w + 4 * k < a.R
                   ? static_cast<const uint16_t*>(a.g)[first + (int64_t)(4 * k) * a.C] : (uint16_t)0;
#pragma unroll
    for (int k = 0; k < 16; ++k)
      g[k] = dtype == SLA2H_DTYPE_BF16 ? BF16::to_f32(raw[k]) : F16::to_f32(raw[k]);
  }
  const double s = wave_sum(q < a.parts ? a.sums[mat * a.parts + q] : 0.0);  // (at most 64 parts)
  const double inv = s == 0.0 ? 0.0 : (double)kScaleX / sqrt(s);
#pragma unroll
  for (int k = 0; k < 16; ++k) tile[4 * k + w][q] = (float)((double)g[k] * inv);
  __syncthreads();
  uint16_t* x = a.x + mat * 2 * a.rp * a.mp;
  const int c = 4 * (threadIdx.x & 15);
  for (int k = threadIdx.x >> 4; k < 64; k += 16) {
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = a.turn ? tile[c + e][k] : tile[k][c + e];
    u32x2 hi, lo;
    split4(v, hi, lo);
    uint16_t* d = x + pair_index(i0 + k, j0 + c, a.mp);
    *reinterpret_cast<u32x2*>(d) = hi;
    *reinterpret_cast<u32x2*>(d + 32) = lo;
  }
}

// Element (i, j) of the last X (scaled), where G has one, in G's type and layout.
__device__ inline void store_out(const OrthoArgs& a, int dtype, int64_t mat, int i, int j, float v) {
  if (i >= a.r || j >= a.m) return;
  v *= 1.f / kScaleX;
  const int64_t at = mat * a.count + (a.turn ? (int64_t)j * a.C + i : (int64_t)i * a.C + j);
  if (dtype == 2)
    static_cast<float*>(a.out)[at] = v;
  else
    static_cast<uint16_t*>(a.out)[at] =
        dtype == SLA2H_DTYPE_BF16 ? BF16::from_f32(v) : F16::from_f32(v);
}
// Eight neighbours of a row of the result (row u of G, columns c on)
__device__ inline void store_row8(const OrthoArgs& a, int dtype, int64_t mat, int u, int c,
                                  const float (&v)[8]) {
  if (u >= a.R || c >= a.C) return;
  if (!a.wide_out) {  // (a row's end, or an address, off the 16 bytes)
#pragma unroll
    for (int e = 0; e < 8; ++e) store_out(a, dtype, mat, a.turn ? c + e : u, a.turn ? u : c + e, v[e]);
    return;
  }
  const int64_t at = mat * a.count + (int64_t)u * a.C + c;
  if (dtype == 2) {
    f32x4* d = reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + at);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      f32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = v[4 * q + e] * (1.f / kScaleX);
      d[q] = x;
    }
    return;
  }
  u32x4 x;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float p = v[2 * e] * (1.f / kScaleX), q = v[2 * e + 1] * (1.f / kScaleX);
    x[e] = dtype == SLA2H_DTYPE_BF16 ? pack2(BF16::from_f32(p), BF16::from_f32(q))
                                     : pack2(F16::from_f32(p), F16::from_f32(q));
  }
  *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.out) + at) = x;
}

enum { kGram, kGramFew, kPoly, kPolyFew, kStep, kLast };

// Offsets of the transposed operand whose slots follow row_frag's order: rows 8 h + 4 x + 0 .. 3.
// (Channels 32 mb on: four chunks further, a bit of the address that no swizzle carries into.)
struct ColOff {
  int at[2];
  __device__ explicit ColOff(int l) {
    const int h = l >> 5, c = 2 * ((l >> 4) & 1) + ((l & 3) >> 1);
#pragma unroll
    for (int x = 0; x < 2; ++x)
      at[x] = chunk_addr(8 * h + 4 * x + ((l & 15) >> 2), c) + 8 * (l & 1);
  }
};
__device__ inline u32x4 turned_frag(const unsigned char* tile, int s, int mb, const ColOff& o) {
  const u32x2 lo = lds_read_tr16(tile + (o.at[0] ^ (64 * mb)) + 16 * s * kRowB);
  const u32x2 hi = lds_read_tr16(tile + (o.at[1] ^ (64 * mb)) + 16 * s * kRowB);
  return u32x4{lo.x, lo.y, hi.x, hi.y};
}

// One product, T x T tiles, a workgroup of 2 x 2 waves per tile.  A stage contracts 32 channels: T rows
// of 128 bytes, hi and lo, of the operand along the lanes and as much of the other one (kStep: 32 rows
// of T columns, read transposed).  The steps of T = 128: two LDS slots of 32 KB, one stage ahead, two
// workgroups per CU, so that one's first loads and its epilogue run beside the other's products (one
// workgroup with 64 channels a stage: 24 x 512 x 2048, kStep 174 us for 84).  The others: four slots,
// three stages ahead, the operands of half a stage read beside the products of the half before (left to
// the compiler's order: 24 x 512 x 2048, kGram 63 us for 48).  Result element (i, j): j along the
// registers, i along the lanes; it goes through LDS, so that whole rows are stored (from the registers,
// eight bytes to a row: kStep 105 us for 91, kGram 65 for 58).  24 x 512 x 2048: kGram 1.0, kStep 0.92
// PFLOP/s of 16-bit products, with 200 MB read and written beside kStep's.
//   kGram, kGramFew: A = X X^T;  kPoly, kPolyFew (with lo lo): B = b A + c A A^T;  kStep: Y = a X + B X;
//   kLast: that, to G's type
template <int T, int OP>
__global__ __launch_bounds__(256, T == 128 && OP < kStep ? 1 : 2) void ortho_product_kernel(
    OrthoArgs a, int dtype, int work) {
  constexpr bool STEP = OP >= kStep, POLY = OP == kPoly || OP == kPolyFew,
                 GRAM = OP == kGram || OP == kGramFew;
  constexpr int NT = T / 64;      // 32 x 32 tiles of a wave: NT x NT
  constexpr int NU = T / 32;      // 32-row units (4 KB) of an operand's stage
  constexpr int kUnit = 32 * kRowB;
  constexpr bool DEEP = T == 64 || !STEP;  // four slots
  __shared__ __align__(16) unsigned char s0[2 * NU * kUnit], s1[2 * NU * kUnit];
  __shared__ __align__(16) unsigned char s2[DEEP ? 2 * NU * kUnit : 16];
  __shared__ __align__(16) unsigned char s3[DEEP ? 2 * NU * kUnit : 16];
  // neighbouring tiles of a matrix on one XCD
  const int per = (work + 7) / 8, item = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (item >= work) return;
  const int ti = (a.rp + T - 1) / T, tj = STEP ? (a.mp + T - 1) / T : ti;
  const int tiles = STEP ? ti * tj : ti * (ti + 1) / 2;
  const int mat = __builtin_amdgcn_readfirstlane(item / tiles);
  int t = item - mat * tiles, it = 0, jt;
  if (STEP) {
    it = t % ti;
    jt = t / ti;
  } else {  // row it of the upper triangle
    while (t >= ti - it) t -= ti - it, ++it;
    jt = it + t;
  }
  it = __builtin_amdgcn_readfirstlane(it);
  jt = __builtin_amdgcn_readfirstlane(jt);
  const int tid = threadIdx.x, l = tid & 63, h = l >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), wi = w >> 1, wj = w & 1;
  const LaneOff lo(l);
  const ColOff co(l);

  const int64_t px = (int64_t)2 * a.rp * a.mp, pa = (int64_t)2 * a.rp * a.rp;
  const uint16_t* X = a.x + mat * px;
  const uint16_t* A = a.A + mat * pa;
  const uint16_t* P = GRAM ? X : POLY ? A : a.B + mat * pa;  // rows i
  const int ldp = (GRAM ? a.mp : a.rp) * 4, ldx = a.mp * 4;         // bytes
  const int K = GRAM ? a.mp : a.rp;

  // Unit u of a stage: rows 32 u .. of the operand along the lanes, then the other one's; wave w loads
  // rows 8 w .. of each.  Rows past the matrix: zeros; columns past it: what stands there, for results
  // that are not stored; a stage past K: the last one again, for no product.
  const int r = 8 * w + (l >> 3), ch = ((l & 7) ^ row_key(r)) << 4;
  int vi[NU], vj[NU];  // a lane's places in an operand
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    vi[u] = (32 * u + r) * ldp + ch;
    vj[u] = STEP ? r * ldx + 128 * u + ch : vi[u];
  }
  auto rows_of = [&](int t) __attribute__((always_inline)) {
    const int n = a.rp - t * T < T ? a.rp - t * T : T;
    return make_rsrc(reinterpret_cast<const char*>(P) + (int64_t)t * T * ldp, (int64_t)n * ldp);
  };
  const auto ri = rows_of(it), rk = rows_of(STEP ? it : jt);
  auto load = [&](int k0, unsigned char* s, int u0, int u1) __attribute__((always_inline)) {
    const int k = k0 < K ? k0 : K - 32;
    const auto rj = STEP ? make_rsrc(reinterpret_cast<const char*>(X) + (int64_t)k * ldx + 4 * T * jt,
                                     (int64_t)31 * ldx + 4 * (a.mp - T * jt))
                         : rk;
#pragma unroll
    for (int u = u0; u < u1; ++u) {
      dma16(ri, s + u * kUnit + 8 * w * kRowB, vi[u], 4 * k);
      dma16(rj, s + (NU + u) * kUnit + 8 * w * kRowB, vj[u], STEP ? 0 : 4 * k);
    }
  };

  // The epilogue's share of a thread: rows, T / 8 threads each, kPass of them at once.  The matrix that
  // is added is on its way while something else is done (T = 64: from the start).
  constexpr int kRows = 2048 / T, kPass = T == 64 ? 2 : 4;
  const int ld = STEP ? a.mp : a.rp;
  const int ni = a.rp - it * T < T ? a.rp - it * T : T, nj = ld - jt * T < T ? ld - jt * T : T;
  const bool diagonal = !STEP && it == jt, columns = OP == kLast && a.turn;
  const int il = tid / (T / 8), jl = 8 * (tid % (T / 8));
  u32x4 ph[kPass]{}, pl[kPass]{};
  auto fetch = [&](int p0) __attribute__((always_inline)) {
    if (GRAM || p0 * kRows >= ni || jl >= nj) return;
#pragma unroll
    for (int p = 0; p < kPass; ++p) {
      const uint16_t* s = (POLY ? A : X) +
                          pair_index(it * T + il + (p0 + p) * kRows, jt * T + jl, ld);
      ph[p] = *reinterpret_cast<const u32x4*>(s);
      pl[p] = *reinterpret_cast<const u32x4*>(s + 32);
    }
  };
  if (T == 64) fetch(0);

  // hi hi, and the two cross products; of few rows the second halves of the stages apart: half as long a
  // chain of additions (20 rows of 1,500: 1.5 to 1.9 times fp32's error otherwise)
  f32x16 acc[NT][NT], low[NT][NT], acc2[NT][NT], low2[NT][NT];
#pragma unroll
  for (int x = 0; x < NT; ++x)
#pragma unroll
    for (int y = 0; y < NT; ++y)
      acc[x][y] = low[x][y] = acc2[x][y] = low2[x][y] = zero16();
  struct Frags {
    u32x4 i[2][NT], j[2][NT];
  };
  auto read_i = [&](const unsigned char* s, int k, int pl, Frags& f) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < NT; ++x) f.i[pl][x] = row_frag(s + (NT * wi + x) * kUnit, 0, 2 * pl + k, lo);
  };
  auto read_j = [&](const unsigned char* s, int k, int pl, Frags& f) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const unsigned char* u = s + (NU + NT * wj + x) * kUnit;
      f.j[pl][x] = STEP ? turned_frag(u, k, pl, co) : row_frag(u, 0, 2 * pl + k, lo);
    }
  };
  // row x of the wave's tiles
  auto products = [&](const Frags& f, int pj, int pi, int x, f32x16 (&to)[NT][NT])
      __attribute__((always_inline)) {
#pragma unroll
    for (int y = 0; y < NT; ++y) to[x][y] = mfma_32x32x16<F16>(f.j[pj][y], f.i[pi][x], to[x][y]);
  };
  auto compute = [&](const unsigned char* s) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      Frags f;
#pragma unroll
      for (int pl = 0; pl < 2; ++pl) {
        read_i(s, k, pl, f);
        read_j(s, k, pl, f);
      }
#pragma unroll
      for (int x = 0; x < NT; ++x) products(f, 1, 0, x, low);
#pragma unroll
      for (int x = 0; x < NT; ++x) products(f, 0, 0, x, acc);
#pragma unroll
      for (int x = 0; x < NT; ++x) products(f, 0, 1, x, low);
    }
  };
  // The same, while the operands of the next half stage are read and, where k is 1, a stage's loads
  // issued: a wave issues in order, so that what stands between two products takes their time unless
  // it is less than one of them.  The order is fixed for T = 128.  T = 64, whose workgroups run in step,
  // is left to the compiler: with the fixed order its bursts make some cards lower their clock (8 x 512 x
  // 512, one call after another: 238 us for 176; zeros, which draw less, 148 for 154).
  auto half = [&](const Frags& f, const unsigned char* s, int k, Frags& next, int k0,
                  unsigned char* to, f32x16 (&acc)[NT][NT], f32x16 (&low)[NT][NT])
      __attribute__((always_inline)) {
#pragma unroll
    for (int z = 0; z < 3 * NT; ++z) {
      if (z == 0) read_i(s, k, 0, next);
      if (z == NT - 1) read_j(s, k, 1, next);
      if (z == NT) read_j(s, k, 0, next);
      if (z == 2 * NT - 1 + (NT == 1)) read_i(s, k, 1, next);
      if (k && z < NU) load(k0, to, z, z + 1);
      if (T == 128) __builtin_amdgcn_sched_barrier(0);
      if (z < NT)
        products(f, 1, 0, z, low);
      else if (z < 2 * NT)
        products(f, 0, 0, z - NT, acc);
      else
        products(f, 0, 1, z - 2 * NT, low);
      if (OP == kPolyFew && z >= 2 * NT) products(f, 1, 1, z - 2 * NT, low);
      if (T == 128) __builtin_amdgcn_sched_barrier(0);
    }
  };
  // (K is a multiple of 64; a stage's loads: 2 NU per wave)
  if (!DEEP) {
    load(0, s0, 0, NU);
    for (int k0 = 0; k0 < K; k0 += 64) {
      __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));
      __builtin_amdgcn_s_barrier();  // the stage has landed, the one before is read
      load(k0 + 32, s1, 0, NU);
      compute(s0);
      __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));
      __builtin_amdgcn_s_barrier();
      load(k0 + 64, s0, 0, NU);
      compute(s1);
    }
  } else {
    // half a stage ahead: the operands of one half are read while the other's products run; the
    // barrier between the halves: the next stage has landed, and this one is read
    Frags f0, f1;
    auto stage = [&](int k0, const unsigned char* cur, const unsigned char* next, unsigned char* to)
        __attribute__((always_inline)) {
      half(f0, cur, 1, f1, k0 + 96, to, acc, low);
      __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(4 * NU));
      __builtin_amdgcn_s_barrier();
      if (OP == kGramFew)
        half(f1, next, 0, f0, 0, to, acc2, low2);
      else
        half(f1, next, 0, f0, 0, to, acc, low);
    };
    load(0, s0, 0, NU);
    load(32, s1, 0, NU);
    load(64, s2, 0, NU);
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(4 * NU));
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int pl = 0; pl < 2; ++pl) {
      read_i(s0, 0, pl, f0);
      read_j(s0, 0, pl, f0);
    }
    int k0 = 0;
    for (; k0 + 64 < K; k0 += 128) {
      stage(k0, s0, s1, s3);
      stage(k0 + 32, s1, s2, s0);
      stage(k0 + 64, s2, s3, s1);
      stage(k0 + 96, s3, s0, s2);
    }
    if (k0 < K) {
      stage(k0, s0, s1, s3);
      stage(k0 + 32, s1, s2, s0);
    }
  }
  __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));  // no load into this LDS outlives the workgroup
  __builtin_amdgcn_s_barrier();

  // The tile in fp32 in LDS, rows i < T / 2 in s0, the others in s1: from there eight neighbours of a
  // row, or of a column, to a thread.  The 16-byte units of row i are permuted by its number, so
  // that 16 columns x 4 groups of eight rows, too, are read from 64 banks.
  auto unit = [&](int i, int u) __attribute__((always_inline)) {
    return (i & (T / 2 - 1)) * (4 * T) + 16 * (u ^ ((i & 7) ^ (((i >> 3) & 3) << 2)));
  };
  auto one = [&](int i, int j) __attribute__((always_inline)) {
    return reinterpret_cast<float*>((i >= T / 2 ? s1 : s0) + unit(i, j >> 2) + 4 * (j & 3));
  };
  if (T == 128) fetch(0);
#pragma unroll
  for (int x = 0; x < NT; ++x)
#pragma unroll
    for (int y = 0; y < NT; ++y)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          v[e] = acc[x][y][r] + low[x][y][r];
          if (OP == kGramFew) v[e] = (acc[x][y][r] + acc2[x][y][r]) + (low[x][y][r] + low2[x][y][r]);
        }
        const int i = (T / 2) * wi + 32 * x + (l & 31), j = (T / 2) * wj + 32 * y + 8 * g + 4 * h;
        if (!diagonal) {
          *reinterpret_cast<f32x4*>(one(i, j)) = v;
          continue;
        }
        // the elements above the diagonal for both sides: symmetric to the bit
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i <= j + e) {
            *one(i, j + e) = v[e];
            *one(j + e, i) = v[e];
          }
      }
  __syncthreads();
  // v: products' sums; hi, lo: eight neighbours of the matrix that the epilogue adds.  (The fused
  // operations are written out: rows, columns and every T round alike.)
  auto finish = [&](float (&v)[8], const u32x4& hi, const u32x4& lw) __attribute__((always_inline)) {
    const float cb = a.b * (kScaleB / kScaleX), cc = a.c * (kScaleB / (kScaleX * kScaleX));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p = GRAM ? 0.f : pair_at(hi[e >> 1], lw[e >> 1], e & 1);
      v[e] = GRAM   ? v[e] * (1.f / kScaleX)
             : POLY ? __builtin_fmaf(cc, v[e], cb * p)
                           : __builtin_fmaf(a.a, p, (1.f / kScaleB) * v[e]);
    }
  };
  auto store_pairs = [&](uint16_t* d, const float (&v)[8]) __attribute__((always_inline)) {
    u32x4 hi, lw;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t x, y;
      split2(v[2 * e], v[2 * e + 1], x, y);
      hi[e] = x;
      lw[e] = y;
    }
    *reinterpret_cast<u32x4*>(d) = hi;
    *reinterpret_cast<u32x4*>(d + 32) = lw;
  };
  uint16_t* base = GRAM ? a.A + mat * pa : POLY ? a.B + mat * pa : a.y + mat * px;
  if (jl < nj)
    for (int p0 = 0; p0 * kRows < ni; p0 += kPass) {
      float v[kPass][8];
#pragma unroll
      for (int p = 0; p < kPass; ++p) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const f32x4 z = *reinterpret_cast<const f32x4*>(one(il + (p0 + p) * kRows, jl + 4 * q));
#pragma unroll
          for (int e = 0; e < 4; ++e) v[p][4 * q + e] = z[e];
        }
      }
#pragma unroll
      for (int p = 0; p < kPass; ++p) finish(v[p], ph[p], pl[p]);
      fetch(p0 + kPass);
#pragma unroll
      for (int p = 0; p < kPass; ++p) {
        const int i = it * T + il + (p0 + p) * kRows, j = jt * T + jl;
        if (columns) {  // back to its place
#pragma unroll
          for (int q = 0; q < 2; ++q)
            *reinterpret_cast<f32x4*>(one(il + (p0 + p) * kRows, jl + 4 * q)) =
                f32x4{v[p][4 * q], v[p][4 * q + 1], v[p][4 * q + 2], v[p][4 * q + 3]};
        } else if (OP == kLast) {
          store_row8(a, dtype, mat, i, j, v[p]);
        } else {
          store_pairs(base + pair_index(i, j, ld), v[p]);
        }
      }
    }
  if (columns) __syncthreads();
  // columns, eight rows to a thread, 16 columns x 32 rows to a wave: the tile below the diagonal
  // (A is symmetric: the same neighbours), or the result of a G whose columns are X's rows
  if (columns || (!STEP && !diagonal))
    for (int i0 = 0; i0 < ni; i0 += 32)
#pragma unroll
      for (int p = 0; p < T / 64; ++p) {
        const int j0 = 16 * w + 64 * p;
        if (j0 >= nj) continue;
        const int ic = i0 + 8 * (l & 3), jc = j0 + (l >> 2), i = it * T + ic, j = jt * T + jc;
        u32x4 hi{}, lw{};
        if (POLY) {
          const uint16_t* s = A + pair_index(j, i, ld);
          hi = *reinterpret_cast<const u32x4*>(s);
          lw = *reinterpret_cast<const u32x4*>(s + 32);
        }
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = *one(ic + e, jc);
        if (OP == kLast) {
          store_row8(a, dtype, mat, j, i, v);
        } else {
          finish(v, hi, lw);
          store_pairs(base + pair_index(j, i, ld), v);
        }
      }
}

// Small matrices (r <= 64, m <= 512): all steps of a matrix in one workgroup, X (at most 128 KB) and A,
// then b A + c A^2 in its place, in LDS as pairs, in tiles of 64 rows x 32 columns, hi and lo.  (A chain of
// launches waits for first loads, not for products: 64 x 128, five steps, 90 us in fifteen launches.)
// A and its square: waves 0 .. 3 a 32 x 32 tile each, for A beside waves 4 .. 7 that take every second
// block of columns; X: a wave takes whole blocks of columns, and replaces them.
constexpr int kSmallM = 512;
struct NsTable {
  float v[3 * 64];
};
__global__ __launch_bounds__(512, 2) void ortho_small_kernel(OrthoArgs a, int dtype, int steps,
                                                             NsTable table) {
  __shared__ __align__(16) unsigned char xs[kSmallM / 32][kTileB], as[2][kTileB];
  __shared__ double red[8];
  const int64_t mat = blockIdx.x;
  const int tid = threadIdx.x, l = tid & 63, h = l >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), grp = w >> 2, wi = (w >> 1) & 1, wj = w & 1;
  const LaneOff lo(l);
  const ColOff co(l);
  const int nb = a.mp / 32;  // blocks of columns
  // four neighbours of row i: the halves' places in a tile
  auto place = [&](int i, int j) __attribute__((always_inline)) {
    return chunk_addr(i, (j & 31) >> 3) + 2 * (j & 7);
  };
  auto put = [&](unsigned char* tile, int i, int j, const float (&v)[4])
      __attribute__((always_inline)) {
    u32x2 hi, lw;
    split4(v, hi, lw);
    const int at = place(i, j);
    *reinterpret_cast<u32x2*>(tile + at) = hi;
    *reinterpret_cast<u32x2*>(tile + (at ^ 64)) = lw;  // four chunks further
  };

  double s = 0.0;
#pragma unroll 4
  for (int i = tid; i < (int)a.count; i += 512) {
    const double v = load_g(a, dtype, mat * a.count + i);
    s += v * v;
  }
  s = wave_sum(s);
  if (l == 0) red[w] = s;
  __syncthreads();
  s = ((red[0] + red[1]) + (red[2] + red[3])) + ((red[4] + red[5]) + (red[6] + red[7]));
  const double inv = s == 0.0 ? 0.0 : (double)kScaleX / sqrt(s);
  for (int k = tid; k < 64 * 8 * nb; k += 512) {  // neighbouring threads read neighbours in G
    const int i = a.turn ? k & 63 : k / (8 * nb), j = 4 * (a.turn ? k >> 6 : k % (8 * nb));
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t at = mat * a.count + (a.turn ? (int64_t)(j + e) * a.C + i : (int64_t)i * a.C + j + e);
      v[e] = i < a.r && j + e < a.m ? (float)((double)load_g(a, dtype, at) * inv) : 0.f;
    }
    put(xs[j >> 5], i, j, v);
  }
  __syncthreads();

  for (int step = 0; step < steps; ++step) {
    const float ca = table.v[3 * step], cb = table.v[3 * step + 1], cc = table.v[3 * step + 2];
    f32x16 acc = zero16(), low = zero16();
    // rows 32 wj and 32 wi of a block of 32 contracted columns
    auto block = [&](const unsigned char* tile, bool square) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const u32x4 ih = row_frag(tile, 32 * wi, k, lo), il = row_frag(tile, 32 * wi, 2 + k, lo);
        const u32x4 jh = row_frag(tile, 32 * wj, k, lo), jl = row_frag(tile, 32 * wj, 2 + k, lo);
        low = mfma_32x32x16<F16>(jl, ih, low);
        acc = mfma_32x32x16<F16>(jh, ih, acc);
        low = mfma_32x32x16<F16>(jh, il, low);
        if (square) low = mfma_32x32x16<F16>(jl, il, low);
      }
    };
    for (int c = grp; c < nb; c += 2) block(xs[c], false);
    f32x4* join = reinterpret_cast<f32x4*>(as[0]) + (w & 3) * 256 + l;
    if (grp) {
#pragma unroll
      for (int g = 0; g < 4; ++g)
        join[64 * g] = f32x4{acc[4 * g] + low[4 * g], acc[4 * g + 1] + low[4 * g + 1],
                             acc[4 * g + 2] + low[4 * g + 2], acc[4 * g + 3] + low[4 * g + 3]};
    }
    __syncthreads();
    float A[16];
    if (!grp) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 z = join[64 * g];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          A[4 * g + e] = (acc[4 * g + e] + low[4 * g + e] + z[e]) * (1.f / kScaleX);
      }
    }
    __syncthreads();
    const int row = 32 * wi + (l & 31);
    if (!grp) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float v[4] = {A[4 * g], A[4 * g + 1], A[4 * g + 2], A[4 * g + 3]};
        put(as[wj], row, 8 * g + 4 * h, v);
      }
    }
    __syncthreads();
    if (!grp) {
      acc = low = zero16();
      block(as[0], true);
      block(as[1], true);
    }
    __syncthreads();
    if (!grp) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] = cc * (kScaleB / (kScaleX * kScaleX)) * (acc[4 * g + e] + low[4 * g + e]) +
                 cb * (kScaleB / kScaleX) * A[4 * g + e];
        put(as[wj], row, 8 * g + 4 * h, v);
      }
    }
    __syncthreads();
    for (int c = w; c < nb; c += 8) {
      f32x16 y[2], z[2];
      y[0] = y[1] = z[0] = z[1] = zero16();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const u32x4 jh = turned_frag(xs[c], k, 0, co), jl = turned_frag(xs[c], k, 1, co);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const u32x4 ih = row_frag(as[k >> 1], 32 * x, k & 1, lo);
          const u32x4 il = row_frag(as[k >> 1], 32 * x, 2 + (k & 1), lo);
          z[x] = mfma_32x32x16<F16>(jl, ih, z[x]);
          y[x] = mfma_32x32x16<F16>(jh, ih, y[x]);
          z[x] = mfma_32x32x16<F16>(jh, il, z[x]);
        }
      }
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int i = 32 * x + (l & 31), jj = 8 * g + 4 * h, at = place(i, jj);
          const u32x2 p = *reinterpret_cast<const u32x2*>(xs[c] + at);
          const u32x2 q = *reinterpret_cast<const u32x2*>(xs[c] + (at ^ 64));
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[e] = (1.f / kScaleB) * (y[x][4 * g + e] + z[x][4 * g + e]) +
                   ca * pair_at(p[e >> 1], q[e >> 1], e & 1);
          if (step + 1 < steps) {
            put(xs[c], i, jj, v);
            continue;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) store_out(a, dtype, mat, i, 32 * c + jj + e, v[e]);
        }
    }
    __syncthreads();
  }
}

struct OrthoPlan {
  int r, m, rp, mp, parts;
  bool small;     // one launch, no workspace
  size_t sums, x, A;  // bytes of the sums, of X, of A
};
bool ortho_plan(int64_t n, int64_t R, int64_t C, OrthoPlan& p) {
  if (n <= 0 || R <= 0 || C <= 0 || R > 32768 || C > 32768) return false;
  p.r = (int)(R < C ? R : C);
  p.m = (int)(R < C ? C : R);
  p.small = p.r <= 64 && p.m <= kSmallM;
  p.rp = (p.r + 63) & ~63;
  p.mp = (p.m + 63) & ~63;
  // (numbers of workgroups and bytes of all matrices)
  if (n * (p.rp / 64) * (p.mp / 64) >= ((int64_t)1 << 28)) return false;
  const int64_t parts = (R * C + 8191) / 8192;
  p.parts = (int)(parts < 64 ? parts : 64);
  p.sums = ((size_t)n * p.parts * 8 + 255) & ~(size_t)255;
  p.x = (size_t)n * 4 * p.rp * p.mp;
  p.A = (size_t)n * 4 * p.rp * p.rp;
  return true;
}

template <int OP>
int ortho_product(const OrthoArgs& a, int dtype, hipStream_t st) {
  auto tiles = [&](int t) -> int64_t {
    const int64_t ti = (a.rp + t - 1) / t, tj = (a.mp + t - 1) / t;
    return a.n * (OP >= kStep ? ti * tj : ti * (ti + 1) / 2);
  };
  // Tiles of 128 read half the bytes per product, tiles of 64 take half as long to begin and end, and are
  // four times as many.  us, 128 / 64, at the number of tiles of 128 and the length that is contracted:
  // step 224, 512: 22 / 19; 384, 512: 26 / 28; 1024, 256: 37 / 47; 1536, 512: 84 / 101; 256, 1024: 37 / 33;
  // 256, 2048: 64 / 76; Gram and square 240, 512: 19 / 19; 400, 512: 33 / 27; 480, 512: 39 / 35; 72, 2048:
  // 36 / 27; 136, 2048: 40 / 44; 240, 2048: 48 / 53; 528, 4096: 230 / 330.
  const bool deep = (OP == kGram ? a.mp : a.rp) >= 2048;
  constexpr bool few = OP == kGramFew || OP == kPolyFew;
  const bool wide = few ? false
                    : OP >= kStep  ? tiles(128) >= (deep ? 200 : 300)
                                   : deep && tiles(128) >= 130;
  const int64_t work = tiles(wide ? 128 : 64);
  const unsigned grid = 8u * (unsigned)((work + 7) / 8);
  if (wide)
    ortho_product_kernel<few ? 64 : 128, OP><<<grid, 256, 0, st>>>(a, dtype, (int)work);
  else
    ortho_product_kernel<64, OP><<<grid, 256, 0, st>>>(a, dtype, (int)work);
  return (int)hipGetLastError();
}

}  // namespace

}  // namespace sla2h

using namespace sla2h;

extern "C" size_t sla2h_orthogonalize_workspace_bytes(int64_t n, int64_t R, int64_t C) {
  OrthoPlan p;
  if (!ortho_plan(n, R, C, p)) return 0;
  return p.small ? 256 : p.sums + 2 * p.x + 2 * p.A;
}

extern "C" int sla2h_orthogonalize(const void* g, int dtype, int64_t n, int64_t R, int64_t C,
                                   int steps, const float* coeffs, void* workspace, void* out,
                                   void* stream) {
  OrthoPlan p;
  SLA2H_CHECK_ARG(g && out && workspace && coeffs && steps > 0 && steps <= 64);
  SLA2H_CHECK_ARG(dtype >= 0 && dtype <= 2 && ortho_plan(n, R, C, p));
  SLA2H_CHECK_ARG(reinterpret_cast<uintptr_t>(workspace) % 16 == 0);
  OrthoArgs a{};
  char* ws = static_cast<char*>(workspace);
  a.g = g, a.out = out;
  a.sums = reinterpret_cast<double*>(ws);
  a.x = reinterpret_cast<uint16_t*>(ws + p.sums);
  a.y = reinterpret_cast<uint16_t*>(ws + p.sums + p.x);
  a.A = reinterpret_cast<uint16_t*>(ws + p.sums + 2 * p.x);
  a.B = reinterpret_cast<uint16_t*>(ws + p.sums + 2 * p.x + p.A);
  a.n = n, a.count = R * C;
  a.R = (int)R, a.C = (int)C, a.r = p.r, a.m = p.m, a.rp = p.rp, a.mp = p.mp, a.parts = p.parts;
  a.turn = R > C;
  a.wide_out = C % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  int err;
  if (p.small) {
    NsTable t{};
    for (int i = 0; i < 3 * steps; ++i) t.v[i] = coeffs[i];
    ortho_small_kernel<<<(unsigned)n, 512, 0, st>>>(a, dtype, steps, t);
    return (int)hipGetLastError();
  }
  const int size = dtype == 2 ? 4 : 2;
  ortho_norm_kernel<<<(unsigned)(n * p.parts), 256, 0, st>>>(
      a, dtype, reinterpret_cast<uintptr_t>(g) % 16 == 0 && a.count * size % 16 == 0);
  if ((err = (int)hipGetLastError())) return err;
  ortho_split_kernel<<<(unsigned)(n * (p.rp / 64) * (p.mp / 64)), 256, 0, st>>>(a, dtype);
  if ((err = (int)hipGetLastError())) return err;
  for (int s = 0; s < steps; ++s) {
    a.a = coeffs[3 * s], a.b = coeffs[3 * s + 1], a.c = coeffs[3 * s + 2];
    const bool few = a.rp <= 128;
    err = few ? ortho_product<kGramFew>(a, dtype, st) : ortho_product<kGram>(a, dtype, st);
    if (err) return err;
    // (few rows: 8 x 448 x 448 would take 175 us for 150 with the fourth product, and gain nothing)
    err = few ? ortho_product<kPolyFew>(a, dtype, st) : ortho_product<kPoly>(a, dtype, st);
    if (err) return err;
    if ((err = s + 1 < steps ? ortho_product<kStep>(a, dtype, st)
                             : ortho_product<kLast>(a, dtype, st)))
      return err;
    uint16_t* t = a.x;
    a.x = a.y;
    a.y = t;
  }
  return (int)hipGetLastError();
}
