// Weight gradient of a linear layer, dW = dY^T X over the token rows, gfx950.
//
// Reference semantics: torch autograd of the nn.Linear layers of
// models/imf_dit_video.py:174-187, 422-467 (their fp32 weights' gradients
// under a 16-bit autocast).
//
// The product contracts over the rows (tokens, tens of thousands) and its
// output is small (a weight: 160 x 512 ... 2048 x 512), so one workgroup per
// output tile leaves most of the 256 CUs idle.  The rows are split into ranges
// as well: grid = output tiles x ranges, fp32 partial tiles, then one pass
// that adds the ranges in order (no atomics: the result does not depend on
// the dispatch order).
#include "act8.h"
#include "common.h"

namespace sla2h {

namespace {

constexpr int kWT = 128;             // output tile (rows of dY columns x X columns)
constexpr int kWK = 32;              // token rows per stage: one K = 32 MFMA step
constexpr int kWStages = 4;          // LDS slots; three stages of loads in flight
constexpr int kWHalf = kWK * kWT * 2;  // bytes of one operand's stage: 32 rows x 256 B
constexpr int kWStage = 2 * kWHalf;
// s_waitcnt vmcnt(8): everything but the last two stages' loads (4 per wave each)
constexpr int kWaitVm8 = 0x0F78;

struct WgradArgs {
  const uint16_t* dy;
  const uint16_t* x;
  float* out;  // partial tiles [split][M][N] (the weight gradient itself with one range)
  int64_t ldy, ldx;
  int rows, M, N;
  int tn;        // column tiles of X
  int tiles;     // output tiles
  int per_split;  // rows of a range, a multiple of kWK
  int nwork, per_xcd;
};

// Four fragments (sub-tiles at LDS byte addresses a[t] + slot, K halves 4096
// bytes apart) read transposed, complete on return.  The compiler makes every
// LDS read that it sees wait for all copies into LDS still in flight
// (vmcnt(0)), which would undo the prefetch; reads in an asm block that waits
// for itself depend on the explicit vmcnt count of the loop alone.
__device__ inline void read_frags(const uint32_t (&a)[4], uint32_t slot, u32x4 (&f)[4]) {
  u32x2 q[8];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\t"
      "ds_read_b64_tr_b16 %1, %8 offset:4096\n\t"
      "ds_read_b64_tr_b16 %2, %9\n\t"
      "ds_read_b64_tr_b16 %3, %9 offset:4096\n\t"
      "ds_read_b64_tr_b16 %4, %10\n\t"
      "ds_read_b64_tr_b16 %5, %10 offset:4096\n\t"
      "ds_read_b64_tr_b16 %6, %11\n\t"
      "ds_read_b64_tr_b16 %7, %11 offset:4096\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(q[0]), "=&v"(q[1]), "=&v"(q[2]), "=&v"(q[3]), "=&v"(q[4]), "=&v"(q[5]),
        "=&v"(q[6]), "=&v"(q[7])
      : "v"(a[0] + slot), "v"(a[1] + slot), "v"(a[2] + slot), "v"(a[3] + slot)
      : "memory");
#pragma unroll
  for (int t = 0; t < 4; ++t) f[t] = u32x4{q[2 * t].x, q[2 * t].y, q[2 * t + 1].x, q[2 * t + 1].y};
}
__device__ inline void dma16(__amdgpu_buffer_rsrc_t rs, void* dst, int voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)dst, 16,
                                           voff, 0, 0, 0);
}

// Workgroup = one 128 x 128 tile of dW over one range of rows; wave (wm, wn)
// owns 64 x 64 of it.  Both operands are row-major in the contracted index, so
// each stage's 32 rows x 128 columns of dY and of X go to LDS as they are
// (buffer loads straight into LDS, three stages ahead, one barrier per stage)
// and the MFMA fragments come out transposed (ds_read_b64_tr_b16: a group of
// 16 lanes reads a 4 row x 16 column block per instruction).  A row's 32-byte
// column chunk c sits at chunk c ^ (row & 7), so the 16 rows of one fragment
// read cover all banks evenly.
template <typename T16>
__global__ __launch_bounds__(256, 2) void wgrad_kernel(WgradArgs a) {
  __shared__ __align__(16) unsigned char lds[kWStages * kWStage];
  const int logical = (blockIdx.x & 7) * a.per_xcd + (blockIdx.x >> 3);
  if (logical >= a.nwork) return;
  // ranges outermost: the workgroups of an XCD share a range's rows in its L2
  const int sp = __builtin_amdgcn_readfirstlane(logical / a.tiles);
  const int tile = __builtin_amdgcn_readfirstlane(logical - sp * a.tiles);
  const int m0 = (tile / a.tn) * kWT, n0 = (tile % a.tn) * kWT;
  const int k0 = sp * a.per_split;
  const int k1 = min(a.rows, k0 + a.per_split);
  const int nst = (k1 - k0 + kWK - 1) / kWK;
  const int tid = threadIdx.x;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l = tid & 63, r = l & 15, g = l >> 4;
  const int wm = w >> 1, wn = w & 1;

  // Rows past the last one read as zero (range check), which ends the last
  // range; a column past M or N reads the next row's (or zero) and only ever
  // feeds an output that is not stored.
  const auto ry = make_rsrc(a.dy, ((int64_t)(a.rows - 1) * a.ldy + a.M) * 2);
  const auto rx = make_rsrc(a.x, ((int64_t)(a.rows - 1) * a.ldx + a.N) * 2);
  const int ldy2 = (int)a.ldy * 2, ldx2 = (int)a.ldx * 2;
  // lane l of a load covers row 4 slot + l / 16, LDS chunk (l % 16) / 2
  const int lrow = 4 * w + (l >> 4);
  const int col = ((((l & 15) >> 1) ^ (lrow & 7)) << 5) + (l & 1) * 16;
  int oy = (k0 + lrow) * ldy2 + m0 * 2 + col;
  int ox = (k0 + lrow) * ldx2 + n0 * 2 + col;
  auto load_stage = [&](int slot) {
    unsigned char* p = lds + slot * kWStage + w * 1024;
    dma16(ry, p, oy);
    dma16(ry, p + 4096, oy + 16 * ldy2);
    dma16(rx, p + kWHalf, ox);
    dma16(rx, p + kWHalf + 4096, ox + 16 * ldx2);
    oy += kWK * ldy2;
    ox += kWK * ldx2;
  };

  // fragment reads: row 4 g + r / 4 (and + 16), chunk = 16-column sub-tile
  const int rho = 4 * g + (r >> 2);
  const uint32_t lbase = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
  uint32_t fy[4], fx[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    fy[t] = lbase + rho * 256 + (((4 * wm + t) ^ (rho & 7)) << 5) + (r & 3) * 8;
    fx[t] = lbase + kWHalf + rho * 256 + (((4 * wn + t) ^ (rho & 7)) << 5) + (r & 3) * 8;
  }

  f32x4 acc[4][4];  // [n sub-tile][m sub-tile]: lane holds dW[m = r][n = 4 g + i]
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // Stage s lives in slot s % 4; the stages loaded past the last one hold zeros
  // or the next range's rows and are never used.
  load_stage(0);
  load_stage(1);
  load_stage(2);
  for (int s = 0; s < nst; ++s) {
    __builtin_amdgcn_s_waitcnt(kWaitVm8);  // this wave's part of stage s has landed
    __builtin_amdgcn_s_barrier();          // everyone's has, and stage s - 1 is read
    load_stage((s + 3) & 3);
    u32x4 fm[4], fn[4];
    const uint32_t slot = (s & 3) * kWStage;
    read_frags(fy, slot, fm);
    read_frags(fx, slot, fn);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = mfma_16x16x32<T16>(fn[i], fm[j], acc[i][j]);
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // no load into this workgroup's LDS outlives it

  float* out = a.out + (int64_t)sp * a.M * a.N;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int m = m0 + 64 * wm + 16 * j + r;
    if (m >= a.M) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + 64 * wn + 16 * i + 4 * g;
      if (n < a.N) *reinterpret_cast<f32x4*>(out + (int64_t)m * a.N + n) = acc[i][j];
    }
  }
}

// dW = sum over the ranges in order, four elements per thread
__global__ __launch_bounds__(256) void wgrad_sum_kernel(const f32x4* __restrict__ part, int splits,
                                                       int64_t n4, f32x4* __restrict__ dw) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n4) return;
  f32x4 s = part[i];
#pragma unroll 8
  for (int j = 1; j < splits; ++j) s += part[j * n4 + i];
  dw[i] = s;
}

// --- dW = dY^T X with X in 8 bits (act8.h) -----------------------------------
//
// dW_mn = sum over row tiles t of s_t,n (sum over the tile's rows dY_rm code_rn): the codes are
// whole numbers up to 127 and exact in either 16-bit type, so each product is exact in fp32.
// The tile's 64 are added in fp32, which rounds, and its scale is applied to their sum.  X is
// never rounded to 16 bits again.
struct Wgrad8Args {
  const uint16_t* dy;
  const int8_t* codes;
  const float* scales;
  float* out;  // [range][M][N]
  int64_t rows, ldy;
  int M, N, cb;
  int tn, tiles;
  int64_t per_split;  // row tiles of a range
  int nwork, per_xcd;
};

// A byte offset past every stage's range (64 rows of at most 2^24 bytes) whose group of eight
// elements and the dword behind it are offsets too.
constexpr int kPastEnd = 0x7fffff00;
static_assert(kPastEnd > (kAct << 24) && kPastEnd + 16 + 4 > kPastEnd);

constexpr int kAStage = kAct * kWT * 2;  // bytes of one operand's stage: 64 rows x 256 B

// sixteen codes as 16-bit numbers, exactly
template <typename T16>
__device__ inline void widen16(u32x4 c, u32x4& lo, u32x4& hi) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t a = pack_pair<T16>(code_f32<0>(c[e]), code_f32<1>(c[e]));
    const uint32_t b = pack_pair<T16>(code_f32<2>(c[e]), code_f32<3>(c[e]));
    if (e < 2)
      lo[2 * e] = a, lo[2 * e + 1] = b;
    else
      hi[2 * e - 4] = a, hi[2 * e - 3] = b;
  }
}

// Workgroup = one 128 x 128 tile of dW over one range of row tiles, wave (wm, wn) 64 x 64 of it
// (one code tile wide, so its scale is one number per stage).  A stage is 64 rows in one of two
// LDS slots: dY goes there as it is (DMA: buffer loads straight into LDS, for 16-byte
// aligned rows; else through registers, as aligned dwords funnelled to the row's start), the
// codes are widened on their way, and the fragments are read transposed.  A slot is an array
// of its own: LDS reads of one then need not wait for the loads into the other.  59,904 x 2,048 x 512
// bf16: 160 us, 785 TFLOP/s (MFMA 30 %, VALU 43 % busy, the rest LDS latency at two waves per
// SIMD); rows of 2,730 bytes (29,138 x 1,365 x 512): 72 us, element by element 193.
template <typename T16, bool DMA>
__global__ __launch_bounds__(256, 2) void wgrad8_kernel(Wgrad8Args a) {
  __shared__ __align__(16) unsigned char ly0[kAStage], ly1[kAStage];
  __shared__ __align__(16) unsigned char lx0[kAStage], lx1[kAStage];
  const int logical = (blockIdx.x & 7) * a.per_xcd + (blockIdx.x >> 3);
  if (logical >= a.nwork) return;
  const int sp = __builtin_amdgcn_readfirstlane(logical / a.tiles);
  const int tile = __builtin_amdgcn_readfirstlane(logical - sp * a.tiles);
  const int m0 = (tile / a.tn) * kWT, n0 = (tile % a.tn) * kWT;
  const int64_t rts = (a.rows + kAct - 1) / kAct;
  const int64_t t0 = sp * a.per_split;
  const int nst = (int)(min(rts, t0 + a.per_split) - t0);
  const int tid = threadIdx.x;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l = tid & 63, r = l & 15, g = l >> 4;
  const int wm = w >> 1, wn = w & 1;

  // dY rows of stage s as a buffer from the dword that holds its first element, rows past the
  // last one read as zero; a column past M reads the next row's and only ever feeds an
  // output that is not stored.
  const int64_t ld2 = a.ldy * 2;
  const int odd = (int)((uintptr_t)a.dy & 2);
  auto rows_of = [&](int s) __attribute__((always_inline)) {
    const int64_t row = (t0 + s) * kAct, left = s < nst ? a.rows - row : 0;
    const uintptr_t p = (uintptr_t)a.dy + row * ld2;
    const int64_t n = ((left < kAct ? left : kAct) - 1) * ld2 + a.M * 2 + (p & 2);
    return make_rsrc(reinterpret_cast<const void*>(p & ~(uintptr_t)3),
                     left <= 0 ? 0 : (n + 3) & ~(int64_t)3);
  };
  const int lrow = 4 * w + (l >> 4);
  const int voff = lrow * (int)ld2 + m0 * 2 + ((((l & 15) >> 1) ^ (lrow & 7)) << 5) + (l & 1) * 16;
  auto dma_y = [&](int s, unsigned char* ly) __attribute__((always_inline)) {
    const auto ry = rows_of(s);
#pragma unroll
    for (int k = 0; k < 4; ++k) dma16(ry, ly + w * 1024 + 4096 * k, voff + 16 * k * (int)ld2);
  };
  // thread: row 16 k + tid / 16, eight elements; a stage's first row is an even number of
  // elements past dy's, so its alignment is dy's
  const int yr = tid >> 4;
  auto y_off = [&](int k) { return (16 * k + yr) * (int)ld2 + m0 * 2 + (tid & 15) * 16 + odd; };
  auto load_y = [&](int s, u32x4 (&v)[4], uint32_t (&x)[4]) __attribute__((always_inline)) {
    const auto ry = rows_of(s);
    // the range ends with a whole dword: the row behind the last one may begin in it
    const int64_t left = a.rows - (t0 + s) * kAct;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int o = 16 * k + yr < left ? y_off(k) & ~3 : kPastEnd;
      v[k] = buf_load16(ry, o, 0);
      x[k] = __builtin_amdgcn_raw_buffer_load_b32(ry, o + 16, 0, 0);
    }
  };
  auto put_y = [&](unsigned char* ly, const u32x4 (&v)[4], const uint32_t (&x)[4])
      __attribute__((always_inline)) {
    unsigned char* p = ly + yr * 256 + ((((tid & 15) >> 1) ^ (yr & 7)) << 5) + (tid & 1) * 16;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t sh = y_off(k) & 2;
      *reinterpret_cast<u32x4*>(p + 4096 * k) =
          u32x4{__builtin_amdgcn_alignbyte(v[k][1], v[k][0], sh),
                __builtin_amdgcn_alignbyte(v[k][2], v[k][1], sh),
                __builtin_amdgcn_alignbyte(v[k][3], v[k][2], sh),
                __builtin_amdgcn_alignbyte(x[k], v[k][3], sh)};
    }
  };
  // codes: threads 0 .. 127 the first tile's 4 KB, the others the second's, 16 bytes each twice
  // (zeros past the last tile)
  const int ct = n0 / kAct, xi = tid & 127;
  const int xoff = (tid >> 7) * kActBytes + xi * 16;
  auto load_x = [&](int s, u32x4 (&v)[2]) __attribute__((always_inline)) {
    const auto rx = make_rsrc(a.codes + ((t0 + s) * a.cb + ct) * kActBytes,
                              s < nst ? (a.cb - ct < 2 ? 1 : 2) * kActBytes : 0);
    v[0] = buf_load16(rx, xoff, 0);
    v[1] = buf_load16(rx, xoff + 2048, 0);
  };
  auto put_x = [&](unsigned char* lx, const u32x4 (&v)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int row = (xi >> 2) + 32 * k, c = 4 * (tid >> 7) + (xi & 3);
      u32x4 lo, hi;
      widen16<T16>(v[k], lo, hi);
      u32x4* p = reinterpret_cast<u32x4*>(lx + row * 256 + ((c ^ (row & 7)) << 5));
      p[0] = lo;
      p[1] = hi;
    }
  };
  const int st = n0 / kAct + wn;  // this wave's code tile
  auto scale_of = [&](int s) {
    return s < nst && st < a.cb ? a.scales[(t0 + s) * a.cb + st] : 0.f;
  };

  // fragment reads: row 4 g + r / 4 (and + 16) of each half stage, chunk = 16-column sub-tile
  const int rho = 4 * g + (r >> 2);
  int fy[4], fx[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    fy[t] = rho * 256 + (((4 * wm + t) ^ (rho & 7)) << 5) + (r & 3) * 8;
    fx[t] = rho * 256 + (((4 * wn + t) ^ (rho & 7)) << 5) + (r & 3) * 8;
  }
  auto frag = [&](const unsigned char* p) __attribute__((always_inline)) {
    const u32x2 lo = lds_read_tr16(p), hi = lds_read_tr16(p + 4096);
    return u32x4{lo.x, lo.y, hi.x, hi.y};
  };
  f32x4 acc[4][4];  // [n sub-tile][m sub-tile]: lane holds dW[m = r][n = 4 g + i]
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  u32x4 xv[2], yv[4];
  uint32_t ye[4];
  float sc = scale_of(0);
  // one stage: everything of stage s + 1 moves into the other slot meanwhile
  auto stage = [&](int s, const unsigned char* ly, const unsigned char* lx, unsigned char* ny,
                   unsigned char* nx) __attribute__((always_inline)) {
    // this wave's part of stage s is in LDS, then everyone's, and stage s - 1 is read
    __builtin_amdgcn_s_waitcnt(DMA ? 0x0070 : 0xC07F);
    __builtin_amdgcn_s_barrier();
    u32x4 xn[2];
    load_x(s + 2, xn);
    if (DMA) {
      dma_y(s + 1, ny);
    } else {
      put_y(ny, yv, ye);
      load_y(s + 2, yv, ye);
    }
    const float scn = scale_of(s + 1);
    u32x4 fm[2][4];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) fm[k][j] = frag(ly + 8192 * k + fy[j]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4 fn[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) fn[k] = frag(lx + 8192 * k + fx[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x4 t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 2; ++k) t = mfma_16x16x32<T16>(fn[k], fm[k][j], t);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(sc, t[e], acc[i][j][e]);
      }
    }
    put_x(nx, xv);
    xv[0] = xn[0];
    xv[1] = xn[1];
    sc = scn;
  };
  load_x(0, xv);
  if (DMA) {
    dma_y(0, ly0);
  } else {
    load_y(0, yv, ye);
    put_y(ly0, yv, ye);
    load_y(1, yv, ye);
  }
  put_x(lx0, xv);
  load_x(1, xv);
  for (int s = 0; s < nst; s += 2) {
    stage(s, ly0, lx0, ly1, lx1);
    if (s + 1 >= nst) break;
    stage(s + 1, ly1, lx1, ly0, lx0);
  }
  __builtin_amdgcn_s_waitcnt(0x0070);  // no load into this workgroup's LDS outlives it

  float* out = a.out + (int64_t)sp * a.M * a.N;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int m = m0 + 64 * wm + 16 * j + r;
    if (m >= a.M) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + 64 * wn + 16 * i + 4 * g;
      float* o = out + (int64_t)m * a.N + n;
      if (a.N % 4 == 0) {
        if (n < a.N) *reinterpret_cast<f32x4*>(o) = acc[i][j];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < a.N) o[e] = acc[i][j][e];
      }
    }
  }
}

// the ranges' sum for a weight whose size is no multiple of four
__global__ __launch_bounds__(256) void wgrad_sum1_kernel(const float* __restrict__ part, int splits,
                                                        int64_t n, float* __restrict__ dw) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float s = part[i];
#pragma unroll 8
  for (int j = 1; j < splits; ++j) s += part[j * n + i];
  dw[i] = s;
}

// Ranges of row tiles: about two workgroups per CU, at least four stages each.
int wgrad8_splits(int64_t rows, int M, int N) {
  const int64_t tiles = (int64_t)((M + kWT - 1) / kWT) * ((N + kWT - 1) / kWT);
  int64_t s = 512 / tiles;
  const int64_t most = (rows + kAct - 1) / kAct / 4;
  s = s < most ? s : most;
  return s < 1 ? 1 : (int)s;
}

// Ranges of rows: enough workgroups for two on each of the 256 CUs, and at
// least eight stages per range.
int wgrad_splits(int64_t rows, int M, int N) {
  const int64_t tiles = (int64_t)((M + kWT - 1) / kWT) * ((N + kWT - 1) / kWT);
  int64_t s = 512 / tiles;
  const int64_t most = rows / (8 * kWK);
  s = s < most ? s : most;
  return s < 1 ? 1 : (int)s;
}

}  // namespace

}  // namespace sla2h

using namespace sla2h;

extern "C" size_t sla2h_linear_wgrad_workspace_bytes(int64_t rows, int M, int N) {
  if (rows <= 0 || M <= 0 || N <= 0) return 0;
  const int s = wgrad_splits(rows, M, N);
  return s > 1 ? (size_t)s * M * N * 4 : 0;
}

extern "C" int sla2h_linear_wgrad(const void* dy, int64_t ldy, const void* x, int64_t ldx,
                                  int dtype, int64_t rows, int M, int N, void* workspace,
                                  float* dw, void* stream) {
  SLA2H_CHECK_ARG(dy && x && dw);
  SLA2H_CHECK_ARG(dtype == SLA2H_DTYPE_F16 || dtype == SLA2H_DTYPE_BF16);
  SLA2H_CHECK_ARG(rows > 0 && M > 0 && N > 0 && M % 8 == 0 && N % 8 == 0);
  SLA2H_CHECK_ARG(ldy >= M && ldx >= N && ldy % 8 == 0 && ldx % 8 == 0);
  SLA2H_CHECK_ARG(((uintptr_t)dy | (uintptr_t)x | (uintptr_t)dw | (uintptr_t)workspace) % 16 == 0);
  // 32-bit byte offsets, three stages and a tile of columns past the end included
  const int64_t pad = 4 * kWK + 16;
  SLA2H_CHECK_ARG((rows + pad) * ldy * 2 + 2 * kWT < ((int64_t)1 << 31) &&
                  (rows + pad) * ldx * 2 + 2 * kWT < ((int64_t)1 << 31));
  const int splits = wgrad_splits(rows, M, N);
  SLA2H_CHECK_ARG(splits == 1 || workspace);
  const int tm = (M + kWT - 1) / kWT, tn = (N + kWT - 1) / kWT;
  const int64_t per = ((rows + splits - 1) / splits + kWK - 1) / kWK * kWK;
  const int used = (int)((rows + per - 1) / per);  // ranges that hold a row
  const int64_t nwork = (int64_t)tm * tn * used;
  SLA2H_CHECK_ARG(nwork < ((int64_t)1 << 28));
  hipStream_t st = static_cast<hipStream_t>(stream);
  WgradArgs a;
  a.dy = static_cast<const uint16_t*>(dy);
  a.x = static_cast<const uint16_t*>(x);
  a.out = used > 1 ? static_cast<float*>(workspace) : dw;
  a.ldy = ldy;
  a.ldx = ldx;
  a.rows = (int)rows;
  a.M = M;
  a.N = N;
  a.tn = tn;
  a.tiles = tm * tn;
  a.per_split = (int)per;
  a.nwork = (int)nwork;
  a.per_xcd = (int)((nwork + 7) / 8);
  if (dtype == SLA2H_DTYPE_BF16)
    wgrad_kernel<BF16><<<8 * a.per_xcd, 256, 0, st>>>(a);
  else
    wgrad_kernel<F16><<<8 * a.per_xcd, 256, 0, st>>>(a);
  int err = (int)hipGetLastError();
  if (err || used == 1) return err;
  const int64_t n4 = (int64_t)M * N / 4;
  wgrad_sum_kernel<<<(unsigned)((n4 + 255) / 256), 256, 0, st>>>(
      static_cast<const f32x4*>(workspace), used, n4, reinterpret_cast<f32x4*>(dw));
  return (int)hipGetLastError();
}

extern "C" size_t sla2h_linear_wgrad8_workspace_bytes(int64_t rows, int M, int N) {
  if (rows <= 0 || M <= 0 || N <= 0) return 0;
  const int s = wgrad8_splits(rows, M, N);
  return s > 1 ? (size_t)s * M * N * 4 : 0;
}

extern "C" int sla2h_linear_wgrad8(const void* dy, int64_t ldy, const int8_t* codes,
                                   const float* scales, int dtype, int64_t rows, int M, int N,
                                   void* workspace, float* dw, void* stream) {
  SLA2H_CHECK_ARG(dy && codes && scales && dw);
  SLA2H_CHECK_ARG(dtype == SLA2H_DTYPE_F16 || dtype == SLA2H_DTYPE_BF16);
  SLA2H_CHECK_ARG(rows > 0 && M > 0 && N > 0 && ldy >= M && ldy < ((int64_t)1 << 23));
  SLA2H_CHECK_ARG(((uintptr_t)codes | (uintptr_t)dw | (uintptr_t)workspace) % 16 == 0 &&
                  (uintptr_t)scales % 4 == 0 && (uintptr_t)dy % 2 == 0);
  const int splits = wgrad8_splits(rows, M, N);
  SLA2H_CHECK_ARG(splits == 1 || workspace);
  const int64_t tm = ((int64_t)M + kWT - 1) / kWT, tn = ((int64_t)N + kWT - 1) / kWT;
  const int64_t rts = (rows + kAct - 1) / kAct, per = (rts + splits - 1) / splits;
  const int64_t used = (rts + per - 1) / per;  // ranges that hold a row
  SLA2H_CHECK_ARG(tm * tn * used < ((int64_t)1 << 28) && per < ((int64_t)1 << 30));
  hipStream_t st = static_cast<hipStream_t>(stream);
  Wgrad8Args a;
  a.dy = static_cast<const uint16_t*>(dy);
  a.codes = codes;
  a.scales = scales;
  a.out = used > 1 ? static_cast<float*>(workspace) : dw;
  a.rows = rows;
  a.ldy = ldy;
  a.M = M;
  a.N = N;
  a.cb = (N + kAct - 1) / kAct;
  a.tn = (int)tn;
  a.tiles = (int)(tm * tn);
  a.per_split = per;
  a.nwork = (int)(tm * tn * used);
  a.per_xcd = (a.nwork + 7) / 8;
  const bool dma = (uintptr_t)dy % 16 == 0 && ldy % 8 == 0 && M % 8 == 0;
  const unsigned grid = 8u * a.per_xcd;
  auto go = [&](auto tag) {
    using T16 = decltype(tag);
    if (dma)
      wgrad8_kernel<T16, true><<<grid, 256, 0, st>>>(a);
    else
      wgrad8_kernel<T16, false><<<grid, 256, 0, st>>>(a);
  };
  if (dtype == SLA2H_DTYPE_BF16)
    go(BF16{});
  else
    go(F16{});
  const int err = (int)hipGetLastError();
  if (err || used == 1) return err;
  const int64_t n = (int64_t)M * N;
  if (n % 4 == 0)
    wgrad_sum_kernel<<<(unsigned)((n / 4 + 255) / 256), 256, 0, st>>>(
        static_cast<const f32x4*>(workspace), (int)used, n / 4, reinterpret_cast<f32x4*>(dw));
  else
    wgrad_sum1_kernel<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(
        static_cast<const float*>(workspace), (int)used, n, dw);
  return (int)hipGetLastError();
}
