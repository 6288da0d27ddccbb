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
// lo lo, below 2^-24 of the product, is what fp32 arithmetic rounds off too.  The result is as
// exact as with fp32 products (1.1 times their error), at three times the 16-bit rate's cost.
#include "dense_attn.h"

#include <initializer_list>

namespace sla2h {

namespace {

// Powers of two that the planes are scaled with: |X| below 16, |A| below 16, |b A + c A^2| below 128
// (singular values of X stay below 1.3 with the usual coefficients) keep hi finite.
constexpr float kScaleX = 4096.f, kScaleB = 512.f;

struct OrthoArgs {
  const void* g;        // (n, R, C)
  void* out;
  double* sums;         // (n, parts) partial sums of squares
  uint16_t *x, *y;      // (n, 2, rp, mp) hi and lo: the step's X and the next one
  uint16_t *A, *B;      // (n, 2, rp, rp)
  int64_t n, count;     // matrices, elements of one
  int R, C, r, m, rp, mp, parts;
  bool turn;            // rows of X are G's columns
  float a, b, c;
};

__device__ inline float load_g(const OrthoArgs& a, int dtype, int64_t i) {
  if (dtype == 2) return static_cast<const float*>(a.g)[i];
  const uint16_t v = static_cast<const uint16_t*>(a.g)[i];
  return dtype == SLA2H_DTYPE_BF16 ? BF16::to_f32(v) : F16::to_f32(v);
}

// Partial sums of squares in double: no overflow of a float's square, and the same sum whatever
// the launch.  Thread by thread over the part, then a tree.
__global__ __launch_bounds__(256) void ortho_norm_kernel(OrthoArgs a, int dtype) {
  __shared__ double red[256];
  const int64_t mat = blockIdx.x / a.parts;
  const int part = (int)(blockIdx.x - mat * a.parts);
  const int64_t per = (a.count + a.parts - 1) / a.parts;
  const int64_t lo = part * per, hi = lo + per < a.count ? lo + per : a.count;
  double s = 0.0;
#pragma unroll 4
  for (int64_t i = lo + threadIdx.x; i < hi; i += 256) {
    const double v = load_g(a, dtype, mat * a.count + i);
    s += v * v;
  }
  red[threadIdx.x] = s;
  __syncthreads();
  for (int w = 128; w >= 1; w >>= 1) {
    if ((int)threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
    __syncthreads();
  }
  if (threadIdx.x == 0) a.sums[blockIdx.x] = red[0];
}

// hi and lo of a scaled value
__device__ inline uint16_t split_hi(float v, uint16_t& lo) {
  const uint16_t hi = F16::from_f32(v);
  lo = F16::from_f32(v - F16::to_f32(hi));
  return hi;
}
__device__ inline void split4(const float (&v)[4], u32x2& hi, u32x2& lo) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    uint16_t l0, l1;
    const uint16_t h0 = split_hi(v[2 * e], l0), h1 = split_hi(v[2 * e + 1], l1);
    hi[e] = pack2(h0, h1);
    lo[e] = pack2(l0, l1);
  }
}
__device__ inline float pair_at(uint32_t hi, uint32_t lo, int e) {
  return F16::to_f32((uint16_t)(hi >> (16 * e))) + F16::to_f32((uint16_t)(lo >> (16 * e)));
}

// X of the first step, zeros up to the padded sizes; a 64 x 64 tile per workgroup, turned through
// LDS where G's columns become rows.
__global__ __launch_bounds__(256) void ortho_split_kernel(OrthoArgs a, int dtype) {
  __shared__ float tile[64][65];
  const int tm = a.mp / 64, tr = a.rp / 64;
  const int64_t mat = blockIdx.x / (tm * tr);
  const int t = (int)(blockIdx.x - mat * (tm * tr)), i0 = t / tm * 64, j0 = t % tm * 64;
  double s = 0.0;
  for (int p = 0; p < a.parts; ++p) s += a.sums[mat * a.parts + p];
  const double inv = s == 0.0 ? 0.0 : (double)kScaleX / sqrt(s);
  const int q = threadIdx.x & 63, w = threadIdx.x >> 6;
  // G's rows of the tile, 64 lanes side by side
  const int g0 = a.turn ? j0 : i0, h0 = a.turn ? i0 : j0;
#pragma unroll 4
  for (int k = w; k < 64; k += 4) {
    const bool in = g0 + k < a.R && h0 + q < a.C;
    const int64_t at = mat * a.count + (int64_t)(g0 + k) * a.C + h0 + q;
    tile[k][q] = in ? (float)((double)load_g(a, dtype, at) * inv) : 0.f;
  }
  __syncthreads();
  uint16_t* x = a.x + mat * 2 * a.rp * a.mp;
  const int64_t plane = (int64_t)a.rp * a.mp;
  const int c = 4 * (threadIdx.x & 15);
  for (int k = threadIdx.x >> 4; k < 64; k += 16) {
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = a.turn ? tile[c + e][k] : tile[k][c + e];
    u32x2 hi, lo;
    split4(v, hi, lo);
    uint16_t* d = x + (int64_t)(i0 + k) * a.mp + j0 + c;
    *reinterpret_cast<u32x2*>(d) = hi;
    *reinterpret_cast<u32x2*>(d + plane) = lo;
  }
}

enum { kGram, kPoly, kStep, kLast };

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

// One product, T x T tiles, a workgroup of 2 x 2 waves per tile; 64 contracted channels a stage in
// two LDS slots, hi and lo of both operands (T = 128: 64 KB a slot, one workgroup per CU; T = 64: 32
// KB, two).  Result element (i, j): j along the registers, i along the lanes, so that four neighbours
// of a row are stored at once.
//   kGram: A = X X^T;  kPoly: B = b A + c A A^T;  kStep: Y = a X + B X;  kLast: that, to G's type
template <int T, int OP>
__global__ __launch_bounds__(256, T == 128 ? 1 : 2) void ortho_product_kernel(OrthoArgs a,
                                                                              int dtype, int work) {
  constexpr bool STEP = OP >= kStep;
  constexpr int NT = T / 64;  // 64-row units of an operand; 32 x 32 tiles of a wave: NT x NT
  __shared__ __align__(16) unsigned char lds[2][4 * NT][kTileB];
  // neighbouring tiles of a matrix on one XCD
  const int per = (work + 7) / 8, item = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (item >= work) return;
  const int ti = (a.rp + T - 1) / T, tj = STEP ? (a.mp + T - 1) / T : ti;
  const int tiles = STEP ? ti * tj : ti * (ti + 1) / 2;
  const int mat = item / tiles;
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

  const int64_t px = (int64_t)a.rp * a.mp, pa = (int64_t)a.rp * a.rp;
  const uint16_t* X = a.x + mat * 2 * px;
  const uint16_t* A = a.A + mat * 2 * pa;
  const uint16_t* B = a.B + mat * 2 * pa;
  const uint16_t* P = OP == kGram ? X : OP == kPoly ? A : B;  // rows i
  const int ldp = (OP == kGram ? a.mp : a.rp) * 2;
  const int64_t pp = OP == kGram ? px : pa;
  const int K = OP == kGram ? a.mp : a.rp;

  auto load = [&](int k0, unsigned char (*s)[kTileB]) __attribute__((always_inline)) {
#pragma unroll
    for (int pl = 0; pl < 2; ++pl)
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const int i = it * T + 64 * u, j = jt * T + 64 * u;
        const auto ri = rows_rsrc(P + pl * pp + k0, i, k0 < K ? a.rp - i : 0, ldp);
        const auto rj = STEP ? rows_rsrc(X + pl * px + j, k0, j < a.mp ? K - k0 : 0, 2 * a.mp)
                             : rows_rsrc(P + pl * pp + k0, j, k0 < K ? a.rp - j : 0, ldp);
        const int ldj = STEP ? 2 * a.mp : ldp;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          dma_rows8(ri, s[pl * NT + u], 2 * w + q, ldp, l);
          dma_rows8(rj, s[2 * NT + pl * NT + u], 2 * w + q, ldj, l);
        }
      }
  };

  f32x16 acc[NT][NT], low[NT][NT];  // hi hi, and the two cross products
#pragma unroll
  for (int x = 0; x < NT; ++x)
#pragma unroll
    for (int y = 0; y < NT; ++y) acc[x][y] = low[x][y] = zero16();
  const int ui = T == 128 ? wi : 0, uj = T == 128 ? wj : 0;  // this wave's units
  auto compute = [&](const unsigned char (*s)[kTileB]) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      u32x4 fi[2][NT], fj[2][NT];
#pragma unroll
      for (int pl = 0; pl < 2; ++pl)
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          const int r0 = T == 128 ? 32 * x : 32 * wi, c0 = T == 128 ? x : wj;
          fi[pl][x] = row_frag(s[pl * NT + ui], r0, k, lo);
          fj[pl][x] = STEP ? turned_frag(s[2 * NT + pl * NT + uj], k, c0, co)
                           : row_frag(s[2 * NT + pl * NT + uj], 32 * c0, k, lo);
        }
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int y = 0; y < NT; ++y) low[x][y] = mfma_32x32x16<F16>(fj[1][y], fi[0][x], low[x][y]);
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int y = 0; y < NT; ++y) acc[x][y] = mfma_32x32x16<F16>(fj[0][y], fi[0][x], acc[x][y]);
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int y = 0; y < NT; ++y) low[x][y] = mfma_32x32x16<F16>(fj[0][y], fi[1][x], low[x][y]);
    }
  };
  load(0, lds[0]);
  for (int k0 = 0; k0 < K; k0 += 128) {
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));
    __builtin_amdgcn_s_barrier();  // the stage has landed, the one before is read
    load(k0 + 64, lds[1]);
    compute(lds[0]);
    if (k0 + 64 >= K) break;
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));
    __builtin_amdgcn_s_barrier();
    load(k0 + 128, lds[0]);
    compute(lds[1]);
  }
  __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));  // no load into this LDS outlives the workgroup

#pragma unroll
  for (int x = 0; x < NT; ++x)
#pragma unroll
    for (int y = 0; y < NT; ++y)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int i = it * T + (T / 2) * wi + 32 * x + (l & 31);
        const int j = jt * T + (T / 2) * wj + 32 * y + 8 * g + 4 * h;
        if (i >= a.rp || j >= (STEP ? a.mp : a.rp)) continue;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[x][y][4 * g + e] + low[x][y][4 * g + e];
        if (OP == kGram) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] *= 1.f / kScaleX;
        } else if (OP == kPoly) {
          const uint16_t* s = A + (int64_t)i * a.rp + j;
          const u32x2 p = *reinterpret_cast<const u32x2*>(s);
          const u32x2 q = *reinterpret_cast<const u32x2*>(s + pa);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[e] = a.c * (kScaleB / (kScaleX * kScaleX)) * v[e] +
                   a.b * (kScaleB / kScaleX) * pair_at(p[e >> 1], q[e >> 1], e & 1);
        } else {
          const uint16_t* s = X + (int64_t)i * a.mp + j;
          const u32x2 p = *reinterpret_cast<const u32x2*>(s);
          const u32x2 q = *reinterpret_cast<const u32x2*>(s + px);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[e] = (1.f / kScaleB) * v[e] + a.a * pair_at(p[e >> 1], q[e >> 1], e & 1);
        }
        if (OP == kLast) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (i >= a.r || j + e >= a.m) continue;
            const float z = v[e] * (1.f / kScaleX);
            const int64_t at = mat * a.count + (a.turn ? (int64_t)(j + e) * a.C + i
                                                       : (int64_t)i * a.C + j + e);
            if (dtype == 2)
              static_cast<float*>(a.out)[at] = z;
            else
              static_cast<uint16_t*>(a.out)[at] =
                  dtype == SLA2H_DTYPE_BF16 ? BF16::from_f32(z) : F16::from_f32(z);
          }
          continue;
        }
        u32x2 hi, lw;
        split4(v, hi, lw);
        uint16_t* base = OP == kGram ? a.A + mat * 2 * pa : OP == kPoly ? a.B + mat * 2 * pa
                                                                        : a.y + mat * 2 * px;
        const int ld = STEP ? a.mp : a.rp;
        const int64_t plane = STEP ? px : pa;
        uint16_t* d = base + (int64_t)i * ld + j;
        if (STEP || it != jt) {
          *reinterpret_cast<u32x2*>(d) = hi;
          *reinterpret_cast<u32x2*>(d + plane) = lw;
        }
        if (STEP) continue;
        // below the diagonal too (within a tile on it the elements above are the ones kept, so
        // that the matrix is symmetric to the bit, whatever the tiles)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (it == jt && j + e < i) continue;
          const uint16_t x0 = (uint16_t)(hi[e >> 1] >> (16 * (e & 1)));
          const uint16_t x1 = (uint16_t)(lw[e >> 1] >> (16 * (e & 1)));
          uint16_t* d2 = base + (int64_t)(j + e) * ld + i;
          d2[0] = x0;
          d2[plane] = x1;
          if (it == jt) {
            d[e] = x0;
            d[e + plane] = x1;
          }
        }
      }
}

struct OrthoPlan {
  int r, m, rp, mp, parts;
  size_t sums, x, A;  // bytes of the sums, of X, of A
};
bool ortho_plan(int64_t n, int64_t R, int64_t C, OrthoPlan& p) {
  if (n <= 0 || R <= 0 || C <= 0 || R > 32768 || C > 32768) return false;
  p.r = (int)(R < C ? R : C);
  p.m = (int)(R < C ? C : R);
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
  const bool wide = tiles(128) >= 200;
  const int64_t work = tiles(wide ? 128 : 64);
  const unsigned grid = 8u * (unsigned)((work + 7) / 8);
  if (wide)
    ortho_product_kernel<128, OP><<<grid, 256, 0, st>>>(a, dtype, (int)work);
  else
    ortho_product_kernel<64, OP><<<grid, 256, 0, st>>>(a, dtype, (int)work);
  return (int)hipGetLastError();
}

}  // namespace

}  // namespace sla2h

using namespace sla2h;

extern "C" size_t sla2h_orthogonalize_workspace_bytes(int64_t n, int64_t R, int64_t C) {
  OrthoPlan p;
  return ortho_plan(n, R, C, p) ? p.sums + 2 * p.x + 2 * p.A : 0;
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
  hipStream_t st = static_cast<hipStream_t>(stream);
  int err;
  ortho_norm_kernel<<<(unsigned)(n * p.parts), 256, 0, st>>>(a, dtype);
  if ((err = (int)hipGetLastError())) return err;
  ortho_split_kernel<<<(unsigned)(n * (p.rp / 64) * (p.mp / 64)), 256, 0, st>>>(a, dtype);
  if ((err = (int)hipGetLastError())) return err;
  for (int s = 0; s < steps; ++s) {
    a.a = coeffs[3 * s], a.b = coeffs[3 * s + 1], a.c = coeffs[3 * s + 2];
    if ((err = ortho_product<kGram>(a, dtype, st))) return err;
    if ((err = ortho_product<kPoly>(a, dtype, st))) return err;
    if ((err = s + 1 < steps ? ortho_product<kStep>(a, dtype, st)
                             : ortho_product<kLast>(a, dtype, st)))
      return err;
    uint16_t* t = a.x;
    a.x = a.y;
    a.y = t;
  }
  return (int)hipGetLastError();
}
