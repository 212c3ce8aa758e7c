// Residual addition, RMS norm and e4m3 codes with one f32 scale per 128
// columns of a row, in one pass: what an 8-bit product reads next.
//
//   h = round(x + delta)                     (stored as the new residual)
//   y = h * rsqrt(mean(h^2) + eps) * (1 + w) | * (1 + scale) + shift | h
//   s_g = f32(max(max_g |y|, 2^-60) / 448),  q = rne_e4m3(y / s_g)
//
// The codes are those of the formula without rounding in between: a value
// computed to 32 bits lands on the wrong side of a border between two codes
// for a few elements in a million, and is then off by a whole code, so the
// row sum, the group maximum and the products are held in 64 bits.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace fvb {
namespace n8 {

constexpr int GROUP = 128;              // columns that share a scale
constexpr int VEC = 8;                  // columns of one thread's vector
constexpr int LANES = GROUP / VEC;      // lanes that share a scale
constexpr int MAX_THREADS = 512;
constexpr double E4M3_MAX = 448.0;
constexpr double MIN_AMAX = 0x1p-60;

enum { DELTA_NONE = 0, DELTA_F32 = 1, DELTA_BF16 = 2 };

struct Dev {
  int mode;
  const void* x;
  long long ld_x;
  const void* delta;
  long long ld_delta;
  void* res;
  long long ld_res;
  const bf16* w;
  const float* mod;
  uint8_t* q;
  long long ld_q;
  float* scales;
  long long ld_scales;
  int dim;
  double eps;
  int vec;  // 16-byte rows everywhere: vector loads and stores
};

__device__ __forceinline__ void load8(const float* p, int n, bool vec, float (&v)[8]) {
  if (vec && n == 8) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    const float4 b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? p[j] : 0.f;
  }
}
__device__ __forceinline__ void load8(const bf16* p, int n, bool vec, float (&v)[8]) {
  if (vec && n == 8) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&a);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __bfloat1622float2(h[j]);
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? __bfloat162float(p[j]) : 0.f;
  }
}
__device__ __forceinline__ void store8(float* p, int n, bool vec, const float (&v)[8]) {
  if (vec && n == 8) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = v[j];
  }
}
__device__ __forceinline__ void store8(bf16* p, int n, bool vec, const float (&v)[8]) {
  if (vec && n == 8) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                   pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = __float2bfloat16(v[j]);
  }
}
// the value as the residual stream stores it
__device__ __forceinline__ float as_stored(float v, const float*) { return v; }
__device__ __forceinline__ float as_stored(float v, const bf16*) {
  return __bfloat162float(__float2bfloat16(v));
}

// t = f32(y / s) made safe to round to e4m3: rounding y / s to 32 bits keeps
// its order against every border between two codes, except that it may land
// on the border itself.  There the exact product border * s (5 + 24 bits)
// says on which side y lies, and t moves one step that way; y on the border
// stays there and goes to the even code.
__device__ __forceinline__ float off_border(float t, double y, double s) {
  const uint32_t b = __float_as_uint(t) & 0x7fffffffu;
  bool border;
  if (b >= 0x3c800000u) {  // 2^-6: three mantissa bits above the border's
    border = (b & 0xfffffu) == 0x80000u;
  } else {                 // below it the step is 2^-9
    const float r = __uint_as_float(b) * 1024.f;
    border = r == truncf(r) && (static_cast<int>(r) & 1);
  }
  if (border) {
    const double d = fma(-static_cast<double>(__uint_as_float(b)), s, fabs(y));
    const uint32_t nb = d > 0.0 ? b + 1 : (d < 0.0 ? b - 1 : b);
    t = __uint_as_float((__float_as_uint(t) & 0x80000000u) | nb);
  }
  return t;
}

// One row (or, without a norm, one run of columns of a row) per CTA; thread t
// holds VPT vectors of 8 columns, so 16 neighbouring lanes share a scale.
template <typename TX, int DT, int VPT>
__global__ void __launch_bounds__(MAX_THREADS) norm_fp8_kernel(const Dev p) {
  __shared__ double part[MAX_THREADS / 32];
  const int T = blockDim.x, tid = threadIdx.x, lane = tid & 31;
  const long long row = blockIdx.x;
  const int c0 = (blockIdx.y * VPT * T + tid) * VEC;
  const bool vec = p.vec;
  const TX* x = static_cast<const TX*>(p.x) + row * p.ld_x;
  griddep_wait();
  griddep_launch_dependents();
  float h[VPT][8];
  double ss = 0.0;
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int c = c0 + v * T * VEC;
    const int n = min(max(p.dim - c, 0), VEC);
    load8(x + c, n, vec, h[v]);
    if (DT != DELTA_NONE) {
      float d[8];
      if (DT == DELTA_F32)
        load8(static_cast<const float*>(p.delta) + row * p.ld_delta + c, n, vec, d);
      else
        load8(static_cast<const bf16*>(p.delta) + row * p.ld_delta + c, n, vec, d);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[v][j] = as_stored(h[v][j] + d[j], x);
      store8(static_cast<TX*>(p.res) + row * p.ld_res + c, n, vec, h[v]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double e = h[v][j];
      ss = fma(e, e, ss);
    }
  }
  double rstd = 1.0;
  if (p.mode != FVB_NORM_NONE) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (lane == 0) part[tid >> 5] = ss;
    __syncthreads();
    ss = 0.0;
    for (int i = 0; i < T / 32; ++i) ss += part[i];
    rstd = 1.0 / sqrt(ss / p.dim + p.eps);
  }
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int c = c0 + v * T * VEC;
    const int n = min(max(p.dim - c, 0), VEC);
    double y[8];
    if (p.mode == FVB_NORM_GEMMA_RMS) {
      float w[8];
      load8(p.w + c, n, vec, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = h[v][j] * rstd * (1.0 + w[j]);
    } else if (p.mode == FVB_NORM_ADA_RMS) {
      float s[8], b[8];
      load8(p.mod + c, n, vec, s);
      load8(p.mod + p.dim + c, n, vec, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = h[v][j] * rstd * (1.0 + s[j]) + b[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = h[v][j] * rstd;
    }
    double top = 0.0;  // fmax drops NaN: the others keep their codes
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmax(top, fabs(y[j]));
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1)
      top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float s = static_cast<float>(fmax(top, MIN_AMAX) / E4M3_MAX);
    const double sd = s, inv = 1.0 / sd;
    uint32_t code[2] = {0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float t = off_border(static_cast<float>(y[j] * inv), y[j], sd);
      code[j >> 2] |= static_cast<uint32_t>(
                          __nv_cvt_float_to_fp8(t, __NV_SATFINITE, __NV_E4M3))
                      << (8 * (j & 3));
    }
    if (n <= 0) continue;
    uint8_t* q = p.q + row * p.ld_q + c;
    if (vec && n == 8) {
      *reinterpret_cast<uint2*>(q) = make_uint2(code[0], code[1]);
    } else {
      for (int j = 0; j < n; ++j) q[j] = static_cast<uint8_t>(code[j >> 2] >> (8 * (j & 3)));
    }
    if ((lane & (LANES - 1)) == 0) p.scales[row * p.ld_scales + c / GROUP] = s;
  }
}

}  // namespace n8
}  // namespace fvb
