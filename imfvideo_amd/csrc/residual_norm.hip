// The residual step between two sublayers, with a norm on both of its sides, gfx950:
//
//   ah = a ra, ra = rsqrt(mean(a^2) + eps);   k_b = scale * w_post * gate_b (gate of clip b)
//   y = x + k_b * ah;   n = w_pre * yh, yh = y ry, ry = rsqrt(mean(y^2) + eps)
//
// and its backward from y and a alone (the two factors ra and ry are a row's sums again):
//
//   dy = dpass + ry (u - yh mean(u yh)), u = w_pre * (dn_0 + dn_1 + dn_2);   dx = dy
//   da = ra (v - ah mean(v ah)), v = dy * k_b
//   dw_pre = sum dn yh;   T_b = sum over clip b of dy ah, of which the gradients of scale, w_post
//   (summed over the clips) and gate_b are products with the other two vectors.
//
// All of it is fp32 arithmetic between one read of each input and one write of each output: bound by
// HBM (2 x 29,952 x 512, bf16, two consumers: forward 368 MB in 66 us, backward 614 MB in 133, 5.6 and
// 4.6 TB/s, where a large copy reaches 4.8).  A row lies in the registers of LPR lanes (a wave's part, or
// a workgroup from 1,025 channels on), eight channels each per step, 16 bytes of a 16-bit row; a group
// of lanes walks rows of one clip, so that k_b, w_pre and, backward, the two column sums stay in
// registers.  The column sums leave a workgroup as one row of partial sums, added in a fixed order by a
// second launch.
#include "common.h"

namespace sla2h {

namespace {

struct F32 {};  // fp32 storage

struct ResNormArgs {
  const float* x;  // the residual stream; backward: y
  const void* a;
  const float *scale, *post, *pre, *gate;  // pre, gate or null
  const float* dy;                         // or null
  const void* dn[3];
  float* y;  // backward: dx
  void* n;   // backward: da
  float* part;
  int64_t L;
  int D, Dp;  // Dp: floats of a partial sum's row
  int chunk;  // rows of a workgroup
  int chunks;  // workgroups of a clip
  float eps, inv_d;
};

// Eight values of a row; VEC: 16-byte accesses of eight neighbours, else values 8 LPR apart
// lanes' width, so that a wave's accesses stay neighbours whatever the alignment.
template <typename T>
__device__ inline void load_vec(const void* p, int64_t i, float (&v)[8]) {
  const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[2 * e] = T::to_f32((uint16_t)(w[e] & 0xffff));
    v[2 * e + 1] = T::to_f32((uint16_t)(w[e] >> 16));
  }
}
template <>
__device__ inline void load_vec<F32>(const void* p, int64_t i, float (&v)[8]) {
  const f32x4* q = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
  const f32x4 lo = q[0], hi = q[1];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = lo[e], v[4 + e] = hi[e];
}
template <typename T>
__device__ inline float load_one(const void* p, int64_t i) {
  return T::to_f32(static_cast<const uint16_t*>(p)[i]);
}
template <>
__device__ inline float load_one<F32>(const void* p, int64_t i) {
  return static_cast<const float*>(p)[i];
}
template <typename T>
__device__ inline void store_vec(void* p, int64_t i, const float (&v)[8]) {
  *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + i) =
      u32x4{pack_pair<T>(v[0], v[1]), pack_pair<T>(v[2], v[3]), pack_pair<T>(v[4], v[5]),
            pack_pair<T>(v[6], v[7])};
}
template <>
__device__ inline void store_vec<F32>(void* p, int64_t i, const float (&v)[8]) {
  f32x4* q = reinterpret_cast<f32x4*>(static_cast<float*>(p) + i);
  q[0] = f32x4{v[0], v[1], v[2], v[3]};
  q[1] = f32x4{v[4], v[5], v[6], v[7]};
}
template <typename T>
__device__ inline void store_one(void* p, int64_t i, float v) {
  static_cast<uint16_t*>(p)[i] = T::from_f32(v);
}
template <>
__device__ inline void store_one<F32>(void* p, int64_t i, float v) {
  static_cast<float*>(p)[i] = v;
}

// A row of D channels over LPR lanes, NC steps of eight channels each.
template <int LPR, int NC, bool VEC>
struct Row {
  int lane, D;
  __device__ int at(int k, int e) const {
    return VEC ? (k * LPR + lane) * 8 + e : (k * 8 + e) * LPR + lane;
  }
  template <typename T>
  __device__ void load(const void* p, int64_t base, float (&v)[NC][8]) const {
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      if (VEC) {
        if (at(k, 0) < D) {
          load_vec<T>(p, base + at(k, 0), v[k]);
          continue;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[k][e] = 0.f;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[k][e] = at(k, e) < D ? load_one<T>(p, base + at(k, e)) : 0.f;
      }
    }
  }
  template <typename T>
  __device__ void store(void* p, int64_t base, const float (&v)[NC][8]) const {
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      if (VEC) {
        if (at(k, 0) < D) store_vec<T>(p, base + at(k, 0), v[k]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (at(k, e) < D) store_one<T>(p, base + at(k, e), v[k][e]);
      }
    }
  }
};

// Sum over a row's LPR lanes, the same bits in each of them.  Rows of 16 lanes rotate (DPP), wider
// ones swap rows; a workgroup's row goes through LDS (`red`: two sets of four, used in turn, so
// that one barrier separates a set's readers from its next writers).
template <int LPR>
__device__ inline float row_sum(float v, float (*red)[4], int& turn) {
  auto ror = [](float x, auto n) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                                         0, __builtin_bit_cast(int, x), 0x120 + decltype(n)::value,
                                         0xf, 0xf, false));
  };
  v += ror(v, std::integral_constant<int, 8>{});
  v += ror(v, std::integral_constant<int, 4>{});
  v += ror(v, std::integral_constant<int, 2>{});
  v += ror(v, std::integral_constant<int, 1>{});
  if (LPR >= 32) {
    const float2 s = swap16(v);
    v = s.x + s.y;
  }
  if (LPR >= 64) {
    const float2 s = swap32(v);
    v = s.x + s.y;
  }
  if (LPR == 256) {
    float* r = red[turn];
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (r[0] + r[1]) + (r[2] + r[3]);
  }
  return v;
}

template <int NC>
__device__ inline float dot(const float (&x)[NC][8], const float (&y)[NC][8]) {
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NC; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) s = __builtin_fmaf(x[k][e], y[k][e], s);
  return s;
}

// k_b of a lane's channels
template <int LPR, int NC, bool VEC>
__device__ inline void load_gain(const ResNormArgs& a, const Row<LPR, NC, VEC>& row, int b,
                                 float (&kb)[NC][8]) {
  float t[NC][8];
  row.template load<F32>(a.scale, 0, kb);
  row.template load<F32>(a.post, 0, t);
#pragma unroll
  for (int k = 0; k < NC; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) kb[k][e] *= t[k][e];
  if (!a.gate) return;
  row.template load<F32>(a.gate, (int64_t)b * a.D, t);
#pragma unroll
  for (int k = 0; k < NC; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) kb[k][e] *= t[k][e];
}

template <typename T, int LPR, int NC, bool VEC>
__global__ __launch_bounds__(256) void residual_norm_fwd_kernel(ResNormArgs a) {
  __shared__ float red[2][4];
  constexpr int G = 256 / LPR;
  const int b = blockIdx.x / a.chunks, r0 = (blockIdx.x - b * a.chunks) * a.chunk;
  const int64_t end = r0 + (int64_t)a.chunk < a.L ? r0 + (int64_t)a.chunk : a.L;
  const Row<LPR, NC, VEC> row{(int)threadIdx.x % LPR, a.D};
  int turn = 0;
  float kb[NC][8], wp[NC][8];
  load_gain(a, row, b, kb);
  if (a.pre) row.template load<F32>(a.pre, 0, wp);
  for (int64_t r = r0 + (int)threadIdx.x / LPR; r < end; r += G) {
    const int64_t base = ((int64_t)b * a.L + r) * a.D;
    float x[NC][8], s[NC][8];
    row.template load<T>(a.a, base, s);
    row.template load<F32>(a.x, base, x);
    const float ra = rsqrtf(row_sum<LPR>(dot(s, s), red, turn) * a.inv_d + a.eps);
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[k][e] = __builtin_fmaf(kb[k][e], s[k][e] * ra, x[k][e]);
    row.template store<F32>(a.y, base, x);
    if (!a.pre) continue;
    const float ry = rsqrtf(row_sum<LPR>(dot(x, x), red, turn) * a.inv_d + a.eps);
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[k][e] = x[k][e] * ry * wp[k][e];
    row.template store<T>(a.n, base, x);
  }
}

template <typename T, int LPR, int NC, bool VEC>
__global__ __launch_bounds__(256) void residual_norm_bwd_kernel(ResNormArgs a) {
  __shared__ float red[2][4];
  __shared__ float cols[LPR == 256 ? 1 : 2][LPR == 256 ? 1 : LPR * NC * 8];
  constexpr int G = 256 / LPR;
  const int b = blockIdx.x / a.chunks, r0 = (blockIdx.x - b * a.chunks) * a.chunk;
  const int64_t end = r0 + (int64_t)a.chunk < a.L ? r0 + (int64_t)a.chunk : a.L;
  const Row<LPR, NC, VEC> row{(int)threadIdx.x % LPR, a.D};
  int turn = 0;
  float kb[NC][8], wp[NC][8], sp[NC][8], st[NC][8];
  load_gain(a, row, b, kb);
  const bool pre = a.pre && a.dn[0];
  if (pre) row.template load<F32>(a.pre, 0, wp);
#pragma unroll
  for (int k = 0; k < NC; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) sp[k][e] = st[k][e] = 0.f;
  for (int64_t r = r0 + (int)threadIdx.x / LPR; r < end; r += G) {
    const int64_t base = ((int64_t)b * a.L + r) * a.D;
    float s[NC][8], d[NC][8];
    row.template load<T>(a.a, base, s);
    if (a.dy) {
      row.template load<F32>(a.dy, base, d);
    } else {
#pragma unroll
      for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) d[k][e] = 0.f;
    }
    if (pre) {
      float y[NC][8], u[NC][8], t[NC][8];
      row.template load<F32>(a.x, base, y);
      row.template load<T>(a.dn[0], base, u);
#pragma unroll
      for (int i = 1; i < 3; ++i) {
        if (!a.dn[i]) break;
        row.template load<T>(a.dn[i], base, t);
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) u[k][e] += t[k][e];
      }
      const float ry = rsqrtf(row_sum<LPR>(dot(y, y), red, turn) * a.inv_d + a.eps);
#pragma unroll
      for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y[k][e] *= ry;
          sp[k][e] = __builtin_fmaf(u[k][e], y[k][e], sp[k][e]);
          u[k][e] *= wp[k][e];
        }
      const float m = row_sum<LPR>(dot(u, y), red, turn) * a.inv_d;
#pragma unroll
      for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) d[k][e] += ry * (u[k][e] - y[k][e] * m);
    }
    row.template store<F32>(a.y, base, d);
    const float ra = rsqrtf(row_sum<LPR>(dot(s, s), red, turn) * a.inv_d + a.eps);
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[k][e] *= ra;
        st[k][e] = __builtin_fmaf(d[k][e], s[k][e], st[k][e]);
        d[k][e] *= kb[k][e];
      }
    const float m = row_sum<LPR>(dot(d, s), red, turn) * a.inv_d;
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) d[k][e] = ra * (d[k][e] - s[k][e] * m);
    row.template store<T>(a.n, base, d);
  }
  // the groups' sums in order, then one row [w_pre's | T] of this workgroup
  float* out = a.part + (int64_t)blockIdx.x * 2 * a.Dp;
  if (G > 1) {
    for (int g = 0; g < G; ++g) {
      if ((int)threadIdx.x / LPR == g) {
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            // (a lane's own places in every group: no order among lanes)
            const int c = (k * 8 + e) * LPR + row.lane;
            cols[0][c] = g ? cols[0][c] + sp[k][e] : sp[k][e];
            cols[LPR == 256 ? 0 : 1][c] = g ? cols[LPR == 256 ? 0 : 1][c] + st[k][e] : st[k][e];
          }
      }
      __syncthreads();
    }
    if ((int)threadIdx.x >= LPR) return;
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = (k * 8 + e) * LPR + row.lane;
        sp[k][e] = cols[0][c];
        st[k][e] = cols[LPR == 256 ? 0 : 1][c];
      }
  }
#pragma unroll
  for (int k = 0; k < NC; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (row.at(k, e) < a.D) {
        out[row.at(k, e)] = sp[k][e];
        out[a.Dp + row.at(k, e)] = st[k][e];
      }
}

// Adds the partial sums of 32 columns: eight quads of columns x 32 groups of workgroups in turn, and
// the groups' sums in order.  blockIdx.y: 0 dw_pre, 1 the gradients that T_b gives, clip after clip in one
// workgroup (1.1 us each: two clips 8 us, 1,024 clips with gates 1.1 ms).
struct ResNormSums {
  const float* part;
  const float *scale, *post, *gate;
  float *dscale, *dpost, *dpre, *dgate;
  int64_t B;
  int chunks, D, Dp;
};
__global__ __launch_bounds__(256) void residual_norm_sums_kernel(ResNormSums a) {
  __shared__ f32x4 part[32][8];
  const int q = threadIdx.x & 7, g = threadIdx.x >> 3;
  const int c = blockIdx.x * 32 + 4 * q;
  const bool is_t = blockIdx.y == 1, live = c < a.Dp;
  if (!is_t && !a.dpre) return;
  auto sum = [&](int64_t first, int64_t n) -> f32x4 {
    f32x4 x{0.f, 0.f, 0.f, 0.f};
    const float* p = a.part + first * 2 * a.Dp + (is_t ? a.Dp : 0) + c;
    if (live) {
#pragma unroll 8
      for (int64_t i = g; i < n; i += 32) x += *reinterpret_cast<const f32x4*>(p + i * 2 * a.Dp);
    }
    part[g][q] = x;
    __syncthreads();
    f32x4 y{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 32; ++i) y += part[i][q];
    __syncthreads();
    return y;
  };
  if (!is_t) {
    const f32x4 y = sum(0, a.B * a.chunks);
    if (g < 4 && c + g < a.D) a.dpre[c + g] = y[g];
    return;
  }
  // thread g < 4: column c + g
  const bool mine = g < 4 && c + g < a.D;
  const float s = mine ? a.scale[c + g] : 0.f, w = mine ? a.post[c + g] : 0.f;
  float all = 0.f;
  for (int64_t b = 0; b < a.B; ++b) {
    const f32x4 y = sum(b * a.chunks, a.chunks);
    const float t = g < 4 ? y[g] : 0.f;
    if (mine && a.gate) {
      all += a.gate[b * a.D + c + g] * t;
      a.dgate[b * a.D + c + g] = t * (s * w);
    } else {
      all += t;
    }
  }
  if (mine) {
    a.dscale[c + g] = all * w;
    a.dpost[c + g] = all * s;
  }
}

// Workgroups of a clip and rows of each.  Two rounds of what the card holds (eight waves per SIMD, four
// backward), whose partial sums are read again.  us at 2 x 29,952 x 512, bf16, by workgroups: forward
// 512 72, 1,024 70, 2,048 69, 4,096 66, 16,384 64; backward with its sums 512 146, 1,024 145, 2,048 143,
// 4,096 146.
struct ResNormPlan {
  int lpr, nc, chunk, chunks;
};
ResNormPlan res_plan(int64_t B, int64_t L, int D, int64_t want) {
  ResNormPlan p{};
  p.lpr = D <= 128 ? 16 : D <= 256 ? 32 : D <= 1024 ? 64 : 256;
  p.nc = (D + 8 * p.lpr - 1) / (8 * p.lpr);
  p.nc = p.nc == 3 ? 4 : p.nc;
  const int64_t g = 256 / p.lpr;
  int64_t rows = (B * L + want - 1) / want;
  rows = (rows + g - 1) / g * g;
  rows = rows < (L + g - 1) / g * g ? rows : (L + g - 1) / g * g;
  p.chunk = (int)rows;
  p.chunks = (int)((L + rows - 1) / rows);
  return p;
}
constexpr int64_t kFwdBlocks = 4096, kBwdBlocks = 2048;

bool res_sizes_ok(int64_t B, int64_t L, int D) {
  return B > 0 && L > 0 && D > 0 && D <= 8192 && B < ((int64_t)1 << 30) && L < ((int64_t)1 << 30) &&
         B * L < ((int64_t)1 << 40) / D;
}

// f(T{}, lanes per row, steps, vector accesses) for a call
template <typename F>
int res_dispatch(int dtype, const ResNormPlan& p, bool vec, F f) {
  auto width = [&](auto t, auto v) -> int {
    using std::integral_constant;
    if (p.lpr == 16) return f(t, integral_constant<int, 16>{}, integral_constant<int, 1>{}, v);
    if (p.lpr == 32) return f(t, integral_constant<int, 32>{}, integral_constant<int, 1>{}, v);
    if (p.lpr == 64 && p.nc == 1)
      return f(t, integral_constant<int, 64>{}, integral_constant<int, 1>{}, v);
    if (p.lpr == 64) return f(t, integral_constant<int, 64>{}, integral_constant<int, 2>{}, v);
    if (p.nc == 1) return f(t, integral_constant<int, 256>{}, integral_constant<int, 1>{}, v);
    if (p.nc == 2) return f(t, integral_constant<int, 256>{}, integral_constant<int, 2>{}, v);
    return f(t, integral_constant<int, 256>{}, integral_constant<int, 4>{}, v);
  };
  auto typed = [&](auto t) -> int {
    return vec ? width(t, std::true_type{}) : width(t, std::false_type{});
  };
  if (dtype == SLA2H_DTYPE_BF16) return typed(BF16{});
  if (dtype == SLA2H_DTYPE_F16) return typed(F16{});
  return typed(F32{});
}

}  // namespace

}  // namespace sla2h

using namespace sla2h;

extern "C" int sla2h_residual_norm_fwd(const float* x, const void* a, int dtype,
                                       const float* scale, const float* post, const float* pre,
                                       const float* gate, int64_t B, int64_t L, int D, float eps,
                                       float* y, void* n, void* stream) {
  SLA2H_CHECK_ARG(x && a && scale && post && y && !pre == !n);
  SLA2H_CHECK_ARG(dtype >= 0 && dtype <= 2 && res_sizes_ok(B, L, D) && eps > 0.f);
  const ResNormPlan p = res_plan(B, L, D, kFwdBlocks);
  const int64_t grid = B * p.chunks;
  SLA2H_CHECK_ARG(grid < ((int64_t)1 << 31));
  ResNormArgs g{};
  g.x = x, g.a = a, g.scale = scale, g.post = post, g.pre = pre, g.gate = gate, g.y = y, g.n = n;
  g.L = L, g.D = D, g.chunk = p.chunk, g.chunks = p.chunks;
  g.eps = eps, g.inv_d = 1.f / (float)D;
  uintptr_t all = 0;
  for (const void* q : {(const void*)x, a, (const void*)scale, (const void*)post, (const void*)pre,
                        (const void*)gate, (const void*)y, (const void*)n})
    all |= reinterpret_cast<uintptr_t>(q);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return res_dispatch(dtype, p, D % 8 == 0 && all % 16 == 0,
                      [&](auto t, auto lpr, auto nc, auto vec) -> int {
                        residual_norm_fwd_kernel<decltype(t), decltype(lpr)::value,
                                                 decltype(nc)::value, decltype(vec)::value>
                            <<<(unsigned)grid, 256, 0, st>>>(g);
                        return (int)hipGetLastError();
                      });
}

extern "C" size_t sla2h_residual_norm_bwd_workspace_bytes(int64_t B, int64_t L, int D) {
  if (!res_sizes_ok(B, L, D)) return 0;
  return (size_t)B * res_plan(B, L, D, kBwdBlocks).chunks * 2 * ((D + 3) & ~3) * 4;
}

extern "C" int sla2h_residual_norm_bwd(const float* y, const void* a, int dtype, const float* scale,
                                       const float* post, const float* pre, const float* gate,
                                       const float* dy, const void* dn0, const void* dn1,
                                       const void* dn2, int64_t B, int64_t L, int D, float eps,
                                       float* dx, void* da, float* dscale, float* dpost,
                                       float* dpre, float* dgate, void* workspace, void* stream) {
  SLA2H_CHECK_ARG(a && scale && post && dx && da && dscale && dpost && workspace);
  SLA2H_CHECK_ARG(!gate == !dgate && (dn0 || !(dn1 || dn2)) && (dn1 || !dn2));
  SLA2H_CHECK_ARG(dn0 ? y && pre && dpre : !dpre);
  SLA2H_CHECK_ARG(dtype >= 0 && dtype <= 2 && res_sizes_ok(B, L, D) && eps > 0.f);
  const ResNormPlan p = res_plan(B, L, D, kBwdBlocks);
  const int64_t grid = B * p.chunks;
  SLA2H_CHECK_ARG(grid < ((int64_t)1 << 31) && reinterpret_cast<uintptr_t>(workspace) % 16 == 0);
  ResNormArgs g{};
  g.x = y, g.a = a, g.scale = scale, g.post = post, g.pre = pre, g.gate = gate, g.dy = dy;
  g.dn[0] = dn0, g.dn[1] = dn1, g.dn[2] = dn2;
  g.y = dx, g.n = da, g.part = static_cast<float*>(workspace);
  g.L = L, g.D = D, g.Dp = (D + 3) & ~3, g.chunk = p.chunk, g.chunks = p.chunks;
  g.eps = eps, g.inv_d = 1.f / (float)D;
  uintptr_t all = 0;
  for (const void* q : {(const void*)y, a, (const void*)scale, (const void*)post, (const void*)pre,
                        (const void*)gate, (const void*)dy, dn0, dn1, dn2, (const void*)dx,
                        (const void*)da})
    all |= reinterpret_cast<uintptr_t>(q);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int err = res_dispatch(dtype, p, D % 8 == 0 && all % 16 == 0,
                               [&](auto t, auto lpr, auto nc, auto vec) -> int {
                                 residual_norm_bwd_kernel<decltype(t), decltype(lpr)::value,
                                                          decltype(nc)::value, decltype(vec)::value>
                                     <<<(unsigned)grid, 256, 0, st>>>(g);
                                 return (int)hipGetLastError();
                               });
  if (err) return err;
  ResNormSums s{};
  s.part = g.part, s.scale = scale, s.post = post, s.gate = gate;
  s.dscale = dscale, s.dpost = dpost, s.dpre = dpre, s.dgate = dgate;
  s.B = B, s.chunks = p.chunks, s.D = D, s.Dp = g.Dp;
  residual_norm_sums_kernel<<<dim3((unsigned)((D + 31) / 32), 2), 256, 0, st>>>(s);
  return (int)hipGetLastError();
}
