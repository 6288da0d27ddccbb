// Activations kept in 8 bits between forward and backward, gfx950: packing and
// restoring, and the gate product h = situ(g) sat(u) of the DiT block's MLP whose forward
// leaves 8-bit gate and up behind and whose backward reads them.
//
//   situ(g) = beta tanh(g / beta) sigmoid(g),  sat(u) = lb tanh(u / lb) (u for lb = 0)
//   dg = dh sat(u) situ'(g),  du = dh situ(g) sat'(u)   at the restored g and u.
//
// HBM-bound by design (8 bytes per element each way for the gate, against 10 with 16-bit
// gate and up in the backward): one wave per 64 x 64 tile, so a tile's scale needs no exchange
// through LDS, and all of a wave's loads (8 or 16 KB) are in flight before it computes.
//
// With a = e^(-2|x|), tanh|x| = (1 - a) / (1 + a) and sech^2 x = 4 a / (1 + a)^2: one exp
// gives both without the cancellation of 1 - tanh^2; 1 - a itself cancels for small |x|, where
// two terms of its series take over.
#include "act8.h"

namespace sla2h {

namespace {

struct Tile {
  int64_t row;  // of this lane's first group of eight
  int c;        // its column
  int64_t id;   // tile number
};

// Wave w of the grid takes tile w; lane l holds row 8 i + l / 8, columns 8 (l % 8) .. + 7.
__device__ inline bool my_tile(int64_t ntile, int cb, Tile& t) {
  t.id = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t.id >= ntile) return false;
  const int l = threadIdx.x & 63;
  const int64_t rt = t.id / cb;
  t.row = rt * kAct + (l >> 3);
  t.c = (int)(t.id - rt * cb) * kAct + (l & 7) * 8;
  return true;
}

template <typename T16>
__device__ inline void load_tile(const uint16_t* x, int64_t ld, int64_t rows, int F, const Tile& t,
                                 u32x4 (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = t.row + 8 * i;
    v[i] = r < rows ? load_row8(x + r * ld, t.c, F) : u32x4{0, 0, 0, 0};
  }
}

template <typename T16>
__device__ inline void pack_tile(const u32x4 (&v)[8], const Tile& t, int8_t* codes,
                                 float* scales) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) top = abs_max2(top, v[i][e]);
  const float s = tile_scale<T16>(top), r = 1.0f / s;
  const int l = threadIdx.x & 63;
  u32x2* dst = reinterpret_cast<u32x2*>(codes + t.id * kActBytes) + l;
#pragma unroll
  for (int i = 0; i < 8; ++i) dst[64 * i] = codes8<T16>(v[i], s, r);
  if (l == 0) scales[t.id] = s;
}

template <typename T16>
__global__ __launch_bounds__(256) void act8_pack_kernel(const uint16_t* __restrict__ x, int64_t ld,
                                                        int64_t rows, int F, int cb, int64_t ntile,
                                                        int8_t* __restrict__ codes,
                                                        float* __restrict__ scales) {
  Tile t;
  if (!my_tile(ntile, cb, t)) return;
  u32x4 v[8];
  load_tile<T16>(x, ld, rows, F, t, v);
  pack_tile<T16>(v, t, codes, scales);
}

template <typename T16>
__global__ __launch_bounds__(256) void act8_unpack_kernel(const int8_t* __restrict__ codes,
                                                          const float* __restrict__ scales,
                                                          int64_t rows, int F, int cb,
                                                          int64_t ntile,
                                                          uint16_t* __restrict__ x) {
  Tile t;
  if (!my_tile(ntile, cb, t)) return;
  const float s = scales[t.id];
  const u32x2* src = reinterpret_cast<const u32x2*>(codes + t.id * kActBytes) + (threadIdx.x & 63);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = t.row + 8 * i;
    float y[8];
    values8(src[64 * i], s, y);
    if (r < rows)
      store_row8(x + r * F, t.c, F,
                 u32x4{pack_pair<T16>(y[0], y[1]), pack_pair<T16>(y[2], y[3]),
                       pack_pair<T16>(y[4], y[5]), pack_pair<T16>(y[6], y[7])});
  }
}

// e^(-y) and 1 - e^(-y), y >= 0
__device__ inline float exp_neg(float y, float& one_minus) {
  const float a = fast_exp2(-kLog2e * y);
  const float series = y * __builtin_fmaf(y, __builtin_fmaf(y, 1.f / 6.f, -0.5f), 1.f);
  one_minus = y < 0.03125f ? series : 1.f - a;
  return a;
}
__device__ inline float sign_of(float mag, float s) { return __builtin_copysignf(mag, s); }

struct Gate {
  float beta, two_over_beta, lb, two_over_lb;
};

// situ(g) sat(u): all divisions in one reciprocal
template <bool SAT>
__device__ inline float gate_fwd(float g, float u, const Gate& p) {
  float na, nd = 1.f, den;
  const float a = exp_neg(__builtin_fabsf(g) * p.two_over_beta, na);
  const float b = fast_exp2(-kLog2e * g);  // sigmoid = 1 / (1 + b); inf gives 0
  den = (1.f + a) * (1.f + b);
  float num = p.beta * na;
  if (SAT) {
    const float d = exp_neg(__builtin_fabsf(u) * p.two_over_lb, nd);
    den *= 1.f + d;
    num *= sign_of(p.lb * nd, u);
  } else {
    num *= u;
  }
  return sign_of(1.f, g) * num * __builtin_amdgcn_rcpf(den);
}

template <bool SAT>
__device__ inline void gate_bwd(float dh, float g, float u, const Gate& p, float& dg, float& du,
                                float& h) {
  float na, nd;
  const float a = exp_neg(__builtin_fabsf(g) * p.two_over_beta, na);
  // e^-g, kept finite: sigmoid(-g) = b / (1 + b)
  const float b = fast_exp2(fminf(-kLog2e * g, 126.f));
  const float ra = __builtin_amdgcn_rcpf(1.f + a), rb = __builtin_amdgcn_rcpf(1.f + b);
  const float situ = sign_of(p.beta * na * ra, g) * rb;
  const float slope = rb * (4.f * a * ra * ra) + situ * (b * rb);
  float sat = u, dsat = 1.f;
  if (SAT) {
    const float d = exp_neg(__builtin_fabsf(u) * p.two_over_lb, nd);
    const float rd = __builtin_amdgcn_rcpf(1.f + d);
    sat = sign_of(p.lb * nd * rd, u);
    dsat = 4.f * d * rd * rd;
  }
  dg = dh * sat * slope;
  du = dh * situ * dsat;
  h = situ * sat;
}

template <typename T16, bool SAT>
__global__ __launch_bounds__(256) void situ8_fwd_kernel(
    const uint16_t* __restrict__ G, const uint16_t* __restrict__ U, int64_t sg, int64_t su,
    int64_t rows, int F, int cb, int64_t ntile, Gate p, uint16_t* __restrict__ H,
    int8_t* __restrict__ gc, float* __restrict__ gs, int8_t* __restrict__ uc,
    float* __restrict__ us) {
  Tile t;
  if (!my_tile(ntile, cb, t)) return;
  u32x4 g[8], u[8];
  load_tile<T16>(G, sg, rows, F, t, g);
  load_tile<T16>(U, su, rows, F, t, u);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    u32x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      y[e] = pack_pair<T16>(gate_fwd<SAT>(T16::to_f32((uint16_t)(g[i][e] & 0xffff)),
                                          T16::to_f32((uint16_t)(u[i][e] & 0xffff)), p),
                            gate_fwd<SAT>(T16::to_f32((uint16_t)(g[i][e] >> 16)),
                                          T16::to_f32((uint16_t)(u[i][e] >> 16)), p));
    const int64_t r = t.row + 8 * i;
    if (r < rows) store_row8(H + r * F, t.c, F, y);
  }
  pack_tile<T16>(g, t, gc, gs);
  pack_tile<T16>(u, t, uc, us);
}

template <typename T16, bool SAT, bool WITH_H>
__global__ __launch_bounds__(256) void situ8_bwd_kernel(
    const uint16_t* __restrict__ DH, int64_t sd, const int8_t* __restrict__ gc,
    const float* __restrict__ gs, const int8_t* __restrict__ uc, const float* __restrict__ us,
    int64_t rows, int F, int cb, int64_t ntile, Gate p, int64_t so, uint16_t* __restrict__ DG,
    uint16_t* __restrict__ DU, uint16_t* __restrict__ H) {
  Tile t;
  if (!my_tile(ntile, cb, t)) return;
  const int l = threadIdx.x & 63;
  const u32x2* gp = reinterpret_cast<const u32x2*>(gc + t.id * kActBytes) + l;
  const u32x2* up = reinterpret_cast<const u32x2*>(uc + t.id * kActBytes) + l;
  u32x4 dh[8];
  u32x2 g8[8], u8[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    g8[i] = gp[64 * i];
    u8[i] = up[64 * i];
  }
  load_tile<T16>(DH, sd, rows, F, t, dh);
  const float s1 = gs[t.id], s2 = us[t.id];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float g[8], u[8], dg[8], du[8], h[8];
    values8(g8[i], s1, g);
    values8(u8[i], s2, u);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      gate_bwd<SAT>(T16::to_f32((uint16_t)(dh[i][e >> 1] >> (16 * (e & 1)))), g[e], u[e], p,
                    dg[e], du[e], h[e]);
    const int64_t r = t.row + 8 * i;
    if (r >= rows) continue;
    auto put = [&](uint16_t* y, const float (&x)[8]) {
      store_row8(y + r * so, t.c, F,
                 u32x4{pack_pair<T16>(x[0], x[1]), pack_pair<T16>(x[2], x[3]),
                       pack_pair<T16>(x[4], x[5]), pack_pair<T16>(x[6], x[7])});
    };
    put(DG, dg);
    put(DU, du);
    if (WITH_H) put(H, h);
  }
}

bool plan(int64_t rows, int F, int& cb, int64_t& ntile, unsigned& grid) {
  if (rows <= 0 || F <= 0) return false;
  cb = (F + kAct - 1) / kAct;
  ntile = (rows + kAct - 1) / kAct * cb;
  const int64_t g = (ntile + 3) / 4;
  grid = (unsigned)g;
  return g < ((int64_t)1 << 31);
}

bool code_ok(const void* c, const void* s) { return c && s && (uintptr_t)c % 16 == 0 && (uintptr_t)s % 4 == 0; }
bool half_ok(const void* p) { return p && (uintptr_t)p % 2 == 0; }
bool dtype_ok(int d) { return d == SLA2H_DTYPE_F16 || d == SLA2H_DTYPE_BF16; }

}  // namespace

}  // namespace sla2h

using namespace sla2h;

extern "C" int sla2h_act8_pack(const void* x, int64_t ld, int dtype, int64_t rows, int F,
                               int8_t* codes, float* scales, void* stream) {
  int cb;
  int64_t nt;
  unsigned grid;
  SLA2H_CHECK_ARG(half_ok(x) && code_ok(codes, scales) && dtype_ok(dtype));
  SLA2H_CHECK_ARG(plan(rows, F, cb, nt, grid) && ld >= F);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const uint16_t* xp = static_cast<const uint16_t*>(x);
  if (dtype == SLA2H_DTYPE_BF16)
    act8_pack_kernel<BF16><<<grid, 256, 0, st>>>(xp, ld, rows, F, cb, nt, codes, scales);
  else
    act8_pack_kernel<F16><<<grid, 256, 0, st>>>(xp, ld, rows, F, cb, nt, codes, scales);
  return (int)hipGetLastError();
}

extern "C" int sla2h_act8_unpack(const int8_t* codes, const float* scales, int dtype, int64_t rows,
                                 int F, void* x, void* stream) {
  int cb;
  int64_t nt;
  unsigned grid;
  SLA2H_CHECK_ARG(half_ok(x) && code_ok(codes, scales) && dtype_ok(dtype));
  SLA2H_CHECK_ARG(plan(rows, F, cb, nt, grid));
  hipStream_t st = static_cast<hipStream_t>(stream);
  uint16_t* xp = static_cast<uint16_t*>(x);
  if (dtype == SLA2H_DTYPE_BF16)
    act8_unpack_kernel<BF16><<<grid, 256, 0, st>>>(codes, scales, rows, F, cb, nt, xp);
  else
    act8_unpack_kernel<F16><<<grid, 256, 0, st>>>(codes, scales, rows, F, cb, nt, xp);
  return (int)hipGetLastError();
}

static Gate make_gate(float beta, float lb) {
  return Gate{beta, 2.f / beta, lb, lb > 0.f ? 2.f / lb : 0.f};
}

extern "C" int sla2h_situ8_fwd(const void* gate, const void* up, int dtype, int64_t rows, int F,
                               int64_t sg, int64_t su, float beta, float lb, void* h,
                               int8_t* gate_codes, float* gate_scales, int8_t* up_codes,
                               float* up_scales, void* stream) {
  int cb;
  int64_t nt;
  unsigned grid;
  SLA2H_CHECK_ARG(half_ok(gate) && half_ok(up) && half_ok(h) && dtype_ok(dtype));
  SLA2H_CHECK_ARG(code_ok(gate_codes, gate_scales) && code_ok(up_codes, up_scales));
  SLA2H_CHECK_ARG(plan(rows, F, cb, nt, grid) && sg >= F && su >= F);
  SLA2H_CHECK_ARG(beta > 0.f && beta < 1e30f && lb >= 0.f && lb < 1e30f);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const Gate p = make_gate(beta, lb);
  auto go = [&](auto tag, auto sat) -> int {
    using T16 = decltype(tag);
    situ8_fwd_kernel<T16, decltype(sat)::value><<<grid, 256, 0, st>>>(
        static_cast<const uint16_t*>(gate), static_cast<const uint16_t*>(up), sg, su, rows, F, cb,
        nt, p, static_cast<uint16_t*>(h), gate_codes, gate_scales, up_codes, up_scales);
    return (int)hipGetLastError();
  };
  if (dtype == SLA2H_DTYPE_BF16)
    return lb > 0.f ? go(BF16{}, std::true_type{}) : go(BF16{}, std::false_type{});
  return lb > 0.f ? go(F16{}, std::true_type{}) : go(F16{}, std::false_type{});
}

extern "C" int sla2h_situ8_bwd(const void* dh, int64_t sd, const int8_t* gate_codes,
                               const float* gate_scales, const int8_t* up_codes,
                               const float* up_scales, int dtype, int64_t rows, int F, float beta,
                               float lb, int64_t so, void* dgate, void* dup, void* h,
                               void* stream) {
  int cb;
  int64_t nt;
  unsigned grid;
  SLA2H_CHECK_ARG(half_ok(dh) && half_ok(dgate) && half_ok(dup) && (uintptr_t)h % 2 == 0);
  SLA2H_CHECK_ARG(code_ok(gate_codes, gate_scales) && code_ok(up_codes, up_scales));
  SLA2H_CHECK_ARG(dtype_ok(dtype) && plan(rows, F, cb, nt, grid) && sd >= F && so >= F);
  SLA2H_CHECK_ARG(beta > 0.f && beta < 1e30f && lb >= 0.f && lb < 1e30f);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const Gate p = make_gate(beta, lb);
  auto go = [&](auto tag, auto sat, auto wh) -> int {
    using T16 = decltype(tag);
    situ8_bwd_kernel<T16, decltype(sat)::value, decltype(wh)::value><<<grid, 256, 0, st>>>(
        static_cast<const uint16_t*>(dh), sd, gate_codes, gate_scales, up_codes, up_scales, rows,
        F, cb, nt, p, so, static_cast<uint16_t*>(dgate), static_cast<uint16_t*>(dup),
        static_cast<uint16_t*>(h));
    return (int)hipGetLastError();
  };
  auto pick = [&](auto tag) -> int {
    using Y = std::true_type;
    using N = std::false_type;
    if (lb > 0.f) return h ? go(tag, Y{}, Y{}) : go(tag, Y{}, N{});
    return h ? go(tag, N{}, Y{}) : go(tag, N{}, N{});
  };
  return dtype == SLA2H_DTYPE_BF16 ? pick(BF16{}) : pick(F16{});
}
