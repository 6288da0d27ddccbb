// Activations kept in 8 bits between forward and backward, gfx950: packing and
// restoring, and the gate product h = situ(g) sat(u) of the DiT block's MLP whose forward
// leaves 8-bit gate and up behind and whose backward reads them.
//
//   situ(g) = beta tanh(g / beta) sigmoid(g),  sat(u) = lb tanh(u / lb) (u for lb = 0)
//   dg = dh sat(u) situ'(g),  du = dh situ(g) sat'(u)   at the restored g and u.
//
// HBM-bound by design: 8 bytes per element each way for the gate (10 with 16-bit gate and
// up in the backward).  59,904 x 2,048 bf16: both in 421 to 444 us by card, 4.4 to 4.7 TB/s (copy rate
// 5.2) beside about 75 VALU per element; each alone under the profiler, median (least) of 30: forward
// 242 (223), backward 254 us (233); packing 59,904 x 512 18 us, 5.1 TB/s.
//
// With a = e^(-2|x|), tanh|x| = (1 - a) / (1 + a) and sech^2 x = 4 a / (1 + a)^2: one exp
// gives both without the cancellation of 1 - tanh^2; 1 - a itself cancels for small |x|, where
// two terms of its series take over.
#include "act8.h"

namespace sla2h {

namespace {

// Workgroup = one tile, 16 elements of each operand per thread: thread t holds rows
// t / 8 and 32 + t / 8, columns 8 (t % 8) .. + 7, so a wave's access covers eight rows of 128
// bytes and its codes 512 bytes in a row.  (A wave per tile needs no exchange for the scale, but four
// times the registers, which left two waves per SIMD, and four times the latency of a small
// call: 274 x 1,365 forward 21 us against 9.)
struct Tile {
  int64_t row;  // of this thread's first group of eight
  int c;        // its column
  int64_t id;   // tile number
};

__device__ inline Tile my_tile(int cb) {
  Tile t;
  t.id = blockIdx.x;
  const int64_t rt = t.id / cb;
  t.row = rt * kAct + (threadIdx.x >> 3);
  t.c = (int)(t.id - rt * cb) * kAct + (threadIdx.x & 7) * 8;
  return t;
}

__device__ inline void load_tile(const uint16_t* x, int64_t ld, int64_t rows, int F, const Tile& t,
                                 u32x4 (&v)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t r = t.row + 32 * i;
    v[i] = r < rows ? load_row8(x + r * ld, t.c, F) : u32x4{0, 0, 0, 0};
  }
}

template <typename T16>
__device__ inline uint32_t top_of(const u32x4 (&v)[2]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) top = abs_max2(top, v[i][e]);
  return top;
}

// Scales of N operands' tiles (one barrier).
template <typename T16, int N>
__device__ inline void tile_scales(const u32x4 (*const (&v)[N])[2], float (&s)[N]) {
  __shared__ float wave_top[N][4];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const float f = wave_top_of<T16>(top_of<T16>(*v[n]));
    if ((threadIdx.x & 63) == 0) wave_top[n][threadIdx.x >> 6] = f;
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const float* w = wave_top[n];
    s[n] = scale_of_top(fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3])));
  }
}

template <typename T16>
__device__ inline void store_codes(const u32x4 (&v)[2], float s, const Tile& t, int8_t* codes,
                                   float* scales) {
  const float r = 1.0f / s;
  u32x2* dst = reinterpret_cast<u32x2*>(codes + t.id * kActBytes) + threadIdx.x;
#pragma unroll
  for (int i = 0; i < 2; ++i) dst[256 * i] = codes8<T16>(v[i], s, r);
  if (threadIdx.x == 0) scales[t.id] = s;
}

template <typename T16>
__global__ __launch_bounds__(256) void act8_pack_kernel(const uint16_t* __restrict__ x, int64_t ld,
                                                        int64_t rows, int F, int cb,
                                                        int8_t* __restrict__ codes,
                                                        float* __restrict__ scales) {
  const Tile t = my_tile(cb);
  u32x4 v[2];
  load_tile(x, ld, rows, F, t, v);
  float s[1];
  tile_scales<T16, 1>({&v}, s);
  store_codes<T16>(v, s[0], t, codes, scales);
}

template <typename T16>
__global__ __launch_bounds__(256) void act8_unpack_kernel(const int8_t* __restrict__ codes,
                                                          const float* __restrict__ scales,
                                                          int64_t rows, int F, int cb,
                                                          uint16_t* __restrict__ x) {
  const Tile t = my_tile(cb);
  const float s = scales[t.id];
  const u32x2* src = reinterpret_cast<const u32x2*>(codes + t.id * kActBytes) + threadIdx.x;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t r = t.row + 32 * i;
    float y[8];
    values8(src[256 * i], s, y);
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
    int64_t rows, int F, int cb, Gate p, uint16_t* __restrict__ H, int8_t* __restrict__ gc,
    float* __restrict__ gs, int8_t* __restrict__ uc, float* __restrict__ us) {
  const Tile t = my_tile(cb);
  u32x4 g[2], u[2];
  load_tile(G, sg, rows, F, t, g);
  load_tile(U, su, rows, F, t, u);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    u32x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      y[e] = pack_pair<T16>(gate_fwd<SAT>(T16::to_f32((uint16_t)(g[i][e] & 0xffff)),
                                          T16::to_f32((uint16_t)(u[i][e] & 0xffff)), p),
                            gate_fwd<SAT>(T16::to_f32((uint16_t)(g[i][e] >> 16)),
                                          T16::to_f32((uint16_t)(u[i][e] >> 16)), p));
    const int64_t r = t.row + 32 * i;
    if (r < rows) store_row8(H + r * F, t.c, F, y);
  }
  float s[2];
  tile_scales<T16, 2>({&g, &u}, s);
  store_codes<T16>(g, s[0], t, gc, gs);
  store_codes<T16>(u, s[1], t, uc, us);
}

template <typename T16, bool SAT, bool WITH_H>
__global__ __launch_bounds__(256) void situ8_bwd_kernel(
    const uint16_t* __restrict__ DH, int64_t sd, const int8_t* __restrict__ gc,
    const float* __restrict__ gs, const int8_t* __restrict__ uc, const float* __restrict__ us,
    int64_t rows, int F, int cb, Gate p, int64_t so, uint16_t* __restrict__ DG,
    uint16_t* __restrict__ DU, uint16_t* __restrict__ H) {
  const Tile t = my_tile(cb);
  const u32x2* gp = reinterpret_cast<const u32x2*>(gc + t.id * kActBytes) + threadIdx.x;
  const u32x2* up = reinterpret_cast<const u32x2*>(uc + t.id * kActBytes) + threadIdx.x;
  u32x4 dh[2];
  u32x2 g8[2], u8[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    g8[i] = gp[256 * i];
    u8[i] = up[256 * i];
  }
  load_tile(DH, sd, rows, F, t, dh);
  const float s1 = gs[t.id], s2 = us[t.id];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float g[8], u[8], dg[8], du[8], h[8];
    values8(g8[i], s1, g);
    values8(u8[i], s2, u);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      gate_bwd<SAT>(T16::to_f32((uint16_t)(dh[i][e >> 1] >> (16 * (e & 1)))), g[e], u[e], p,
                    dg[e], du[e], h[e]);
    const int64_t r = t.row + 32 * i;
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
  grid = (unsigned)ntile;
  return ntile < ((int64_t)1 << 31);
}

bool code_ok(const void* c, const void* s) {
  return c && s && (uintptr_t)c % 16 == 0 && (uintptr_t)s % 4 == 0;
}
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
    act8_pack_kernel<BF16><<<grid, 256, 0, st>>>(xp, ld, rows, F, cb, codes, scales);
  else
    act8_pack_kernel<F16><<<grid, 256, 0, st>>>(xp, ld, rows, F, cb, codes, scales);
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
    act8_unpack_kernel<BF16><<<grid, 256, 0, st>>>(codes, scales, rows, F, cb, xp);
  else
    act8_unpack_kernel<F16><<<grid, 256, 0, st>>>(codes, scales, rows, F, cb, xp);
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
        p, static_cast<uint16_t*>(h), gate_codes, gate_scales, up_codes, up_scales);
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
        F, cb, p, so, static_cast<uint16_t*>(dgate), static_cast<uint16_t*>(dup),
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
