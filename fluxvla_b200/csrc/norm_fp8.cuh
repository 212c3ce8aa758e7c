// Residual addition, RMS norm and e4m3 codes with one f32 scale per 128
// columns of a row, in one pass: what an 8-bit product reads next.
//
//   h = x + delta                            (stored as the new residual)
//   y = h * rsqrt(mean(h^2) + eps) * (1 + w) | * (1 + scale) + shift | h
//   s_g = f32(max(max_g |y|, 2^-60) / 448),  q = rne_e4m3(y / s_g)
//
// The sum is formed in f32 and rounded to x's type, as (x + delta).to(x.dtype)
// is: for bf16 x and an f32 delta that is two roundings, off by half a step and
// 2^-17 of one at most.  From h on, the codes and scales are those of the formula
// without rounding in between:
// a value computed to 32 bits lands on the wrong side of a border between two
// codes for a few elements in a million, and is then off by a whole code.  All
// of it in 64 bits is bound by the conversions (848 x 16384 bf16 codes: 24 us
// against 6.5 us of memory traffic), so 64 bits are used where they decide:
// the row's sum of squares, the group's largest value, and those vectors of
// which a value, computed to 32 bits with its error bound, has a border inside
// the bound (about one in ten thousand).  Without a norm y is what 32 bits
// hold, and y / s rounded to odd takes their place: 10.5 us on 848 x 16384,
// bound by the issue of instructions.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace fvb {
namespace n8 {

constexpr int GROUP = 128;              // columns that share a scale
constexpr int VEC = 8;                  // columns of one thread's vector
constexpr int LANES = GROUP / VEC;      // lanes that share a scale
constexpr int MAX_THREADS = 512;
// bound of the relative error of a value computed to 32 bits: 6 roundings of
// 2^-24 and the reciprocal of the scale
constexpr float EPS = 0x1p-20f;
constexpr double E4M3_MAX = 448.0;
constexpr double MIN_AMAX = 0x1p-60;

enum { DELTA_NONE = 0, DELTA_F32 = 1, DELTA_BF16 = 2 };
// what is done to a value: nothing, norm * (1 + w), norm * (1 + scale) + shift
enum { CODES = 0, SCALE = 1, SHIFT = 2 };

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
  double eps, inv_dim;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void from_f32(bf16* p, float v) { *p = __float2bfloat16(v); }

__device__ __forceinline__ void load_vec(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  const float4 b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load_vec(const bf16* p, float (&v)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&a);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __bfloat1622float2(h[j]);
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}
__device__ __forceinline__ void store_vec(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store_vec(bf16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                            pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// How a warp's lanes reach their columns c..c+7 of a row, c STRIDE apart from
// lane to lane: with 16-byte accesses where all rows allow them (VECS), else
// with neighbouring lanes on neighbouring columns and an exchange through
// shared memory (lanes on 8 columns each, value by value, took 71 us instead
// of 22 on 4096 x 2047 codes of bf16 + bf16, 49 instead of 36 with an adaRMS
// norm; only the RMS norm without a delta gains nothing, 20.6 and 22.9).  All lanes call.
template <int STRIDE, bool VECS>
struct Columns {
  int dim, lane;
  float* stage;  // [256]

  // column of value lane of the warp's 256; value lane + 32 k is 4 k lanes on
  __device__ __forceinline__ int first(int c) const {
    return c + ((lane >> 3) - lane) * STRIDE + (lane & 7);
  }
  // ALIGNED: the row starts on 16 bytes
  template <bool ALIGNED = VECS, typename T>
  __device__ __forceinline__ void load(const T* row, int c, float (&v)[8]) const {
    if (ALIGNED && c + 8 <= dim) {
      load_vec(row + c, v);
    } else if (ALIGNED) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c + j < dim ? to_f32(row[c + j]) : 0.f;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int at = first(c) + 4 * STRIDE * k;
        v[k] = at < dim ? to_f32(row[at]) : 0.f;
      }
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 8; ++k) stage[lane + 32 * k] = v[k];
      __syncwarp();
      load_vec(stage + lane * 8, v);
    }
  }
  // of a vector that all rows share, aligned or not
  template <typename T>
  __device__ __forceinline__ void load_shared(const T* row, int c, float (&v)[8]) const {
    if (VECS || (reinterpret_cast<uintptr_t>(row) & 15) == 0)
      load<true>(row, c, v);
    else
      load<false>(row, c, v);
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, int c, const float (&v)[8]) const {
    if (VECS && c + 8 <= dim) {
      store_vec(row + c, v);
    } else if (VECS) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < dim) from_f32(row + c + j, v[j]);
    } else {
      __syncwarp();
      store_vec(stage + lane * 8, v);
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int at = first(c) + 4 * STRIDE * k;
        if (at < dim) from_f32(row + at, stage[lane + 32 * k]);
      }
    }
  }
  __device__ __forceinline__ void store_codes(uint8_t* row, int c, uint32_t lo, uint32_t hi) const {
    if (VECS && c + 8 <= dim) {
      *reinterpret_cast<uint2*>(row + c) = make_uint2(lo, hi);
    } else if (VECS) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < dim) row[c + j] = static_cast<uint8_t>((j < 4 ? lo : hi) >> (8 * (j & 3)));
    } else {
      uint8_t* bytes = reinterpret_cast<uint8_t*>(stage);
      __syncwarp();
      *reinterpret_cast<uint2*>(bytes + lane * 8) = make_uint2(lo, hi);
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int at = first(c) + 4 * STRIDE * k;
        if (at < dim) row[at] = bytes[lane + 32 * k];
      }
    }
  }
};

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

// Two 32-bit values to an instruction.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(f32x2 v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// y / s rounded to odd (toward zero, and the last bit set where that was not
// exact), which rounds to e4m3 as y / s itself does (Boldo and Melquiond,
// Emulation of FMA and correctly rounded sums: proved algorithms using rounding
// to odd, IEEE Transactions on Computers 57, 2008); y0, y1 >= 0 that f32
// holds, r = 1 / s within an ulp.  t is the quotient within its last bit, so
// that the remainder y - t s, rounded once, has the sign of the error.
__device__ __forceinline__ void divide_odd(float y0, float y1, float s, float r, float& t0,
                                           float& t1) {
  const f32x2 y = pair(y0, y1), ns = pair(-s, -s), r2 = pair(r, r);
  const f32x2 q = mul2(y, r2), t = fma2(fma2(ns, q, y), r2, q);
  float d0, d1;
  unpair(fma2(ns, t, y), d0, d1);
  unpair(t, t0, t1);
  t0 = __uint_as_float((__float_as_uint(t0) - (d0 < 0.f)) | (d0 != 0.f));
  t1 = __uint_as_float((__float_as_uint(t1) - (d1 < 0.f)) | (d1 != 0.f));
}

__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

__device__ __forceinline__ float rcp(float x) {  // within an ulp
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// largest of the N lanes that share a scale; values not negative
template <int N = LANES>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// One row (or, without a norm, one run of columns of a row) per CTA; thread t
// holds VPT vectors of 8 columns.  With a norm these are T vectors apart and 16
// neighbouring lanes share a scale; without one they are neighbours, and 16 /
// VPT lanes do.
template <typename TX, int DT, int VPT, int KIND, bool VECS>
__global__ void __launch_bounds__(KIND == CODES ? 256 : MAX_THREADS,
                                  KIND != CODES && VPT == 1 && !VECS ? 2 : 0)
    norm_fp8_kernel(const Dev p) {
  constexpr bool NORM = KIND != CODES, ADA = KIND == SHIFT;
  __shared__ double part[MAX_THREADS / 32];
  const int T = blockDim.x, tid = threadIdx.x, lane = tid & 31;
  const long long row = blockIdx.x;
  const int c0 = (blockIdx.y * T + tid) * VEC * (NORM ? 1 : VPT);
  const int step = NORM ? T * VEC : VEC;  // from a thread's vector to its next
  extern __shared__ __align__(16) float stage[];  // 256 a warp, if !VECS
  const Columns<NORM ? VEC : VEC * VPT, VECS> io = {p.dim, lane, stage + (tid >> 5) * 256};
  const TX* x = static_cast<const TX*>(p.x) + row * p.ld_x;
  griddep_wait();
  griddep_launch_dependents();
  float h[VPT][8];
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int c = c0 + v * step;
    io.load(x, c, h[v]);
  }
  if (DT != DELTA_NONE) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int c = c0 + v * step;
      float d[8];
      if (DT == DELTA_F32)
        io.load(static_cast<const float*>(p.delta) + row * p.ld_delta, c, d);
      else
        io.load(static_cast<const bf16*>(p.delta) + row * p.ld_delta, c, d);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[v][j] = as_stored(h[v][j] + d[j], x);
      io.store(static_cast<TX*>(p.res) + row * p.ld_res, c, h[v]);
    }
  }
  if (!NORM) {
    float top = static_cast<float>(MIN_AMAX);  // fmax drops NaN: the others keep their codes
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(h[v][j]));
    // top / 448 rounded to f32, by a multiplication and its remainder
    // (Markstein); infinity stays infinity
    top = group_max<LANES / VPT>(top);
    constexpr float M = static_cast<float>(E4M3_MAX), I = 1.f / M;
    const float q = top * I;
    const float s = top < INFINITY ? fmaf(fmaf(-M, q, top), I, q) : top;
    const float r = rcp(s);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int c = c0 + v * step;
      float t[8];
      if (s < INFINITY) {
#pragma unroll
        for (int j = 0; j < 8; j += 2)
          divide_odd(fabsf(h[v][j]), fabsf(h[v][j + 1]), s, r, t[j], t[j + 1]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = fabsf(h[v][j]) * 0.f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = copysignf(t[j], h[v][j]);
      io.store_codes(p.q + row * p.ld_q, c, codes4(t[0], t[1], t[2], t[3]),
                     codes4(t[4], t[5], t[6], t[7]));
    }
    if ((lane & (LANES / VPT - 1)) == 0 && c0 < p.dim)
      p.scales[row * p.ld_scales + c0 / GROUP] = s;
    return;
  }
  double rstd = 1.0;
  {
    double ss = 0.0;
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double e = h[v][j];
        ss = fma(e, e, ss);
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (lane == 0) part[tid >> 5] = ss;
    __syncthreads();
    ss = 0.0;
    for (int i = 0; i < T / 32; ++i) ss += part[i];
    rstd = rsqrt(fma(ss, p.inv_dim, p.eps));
  }
  const float rf = static_cast<float>(rstd);
  // near the ends of the 32-bit range the bounds do not hold (nor where rf is
  // NaN): such rows are computed in 64 bits throughout, and so are vectors with
  // a weight above 2^40.  Below it no value overflows (a normed one is at most
  // 2^7), and what a normed value loses below 2^-126, at most 2^-150, is no
  // more than 2^-109 after it: nothing to the lowest border, which is 2^-79.
  const bool fine_row = rf >= 0x1p-100f && rf <= 0x1p100f;
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int c = c0 + v * step;
    // y to 32 bits, and what bounds its error: EPS * mag
    float y[8], mag[8], w[8], b[8];
    if (KIND == SCALE) {
      if (p.mode == FVB_NORM_GEMMA_RMS) {
        io.load_shared(p.w, c, w);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = 0.f;
      }
    } else if (ADA) {
      io.load_shared(p.mod, c, w);
      io.load_shared(p.mod + p.dim, c, b);
    }
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const f32x2 one = pair(1.f, 1.f);
      const f32x2 z = mul2(mul2(pair(h[v][j], h[v][j + 1]), pair(rf, rf)),
                           add2(pair(w[j], w[j + 1]), one));
      unpair(z, y[j], y[j + 1]);
      mag[j] = fabsf(y[j]);
      mag[j + 1] = fabsf(y[j + 1]);
      if (ADA) {
        unpair(add2(pair(mag[j], mag[j + 1]), pair(fabsf(b[j]), fabsf(b[j + 1]))), mag[j],
               mag[j + 1]);
        unpair(add2(z, pair(b[j], b[j + 1])), y[j], y[j + 1]);
      }
    }
    bool fine = fine_row;
    if (KIND == SHIFT || p.mode == FVB_NORM_GEMMA_RMS) {
      float most = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(w[j]));
      fine = fine && most <= 0x1p40f;
    }
    auto exact = [&](int j) {
      double r = h[v][j] * rstd * (1.0 + w[j]);
      if (ADA) r += b[j];
      return r;
    };
    // of the values that may be the largest, the largest scale
    float low = 0.f, high = 0.f;  // fmax drops NaN: the others keep their codes
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float a0 = fabsf(y[j]), a1 = fabsf(y[j + 1]);
      if (ADA) {
        const f32x2 a = pair(a0, a1), m = pair(mag[j], mag[j + 1]);
        float t0, t1;
        unpair(fma2(pair(-EPS, -EPS), m, a), t0, t1);
        low = fmaxf(low, fmaxf(t0, t1));
        unpair(fma2(pair(EPS, EPS), m, a), t0, t1);
        high = fmaxf(high, fmaxf(t0, t1));
      } else {
        low = fmaxf(low, fmaxf(a0, a1));
      }
    }
    if (!ADA) {
      high = low * (1.f + EPS);
      low *= 1.f - EPS;
    }
    low = group_max(fine ? low : 0.f);
    float s = static_cast<float>(MIN_AMAX / E4M3_MAX);
    // (low is 0 where shifts cancel all values to within their bounds: then each
    // of them may be the largest; a high of 0 is a value of zero)
    if (!fine || (high >= low && high > 0.f)) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (!fine || fmaf(EPS, mag[j], fabsf(y[j])) >= low)
          s = fmaxf(s, static_cast<float>(fabs(exact(j)) * (1.0 / E4M3_MAX)));
    }
    s = group_max(s);
    // codes of both ends of each value's interval
    const float r = rcp(s), r_lo = ADA ? r : r * (1.f - EPS), r_hi = ADA ? r : r * (1.f + EPS);
    float lo[8], hi[8];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const f32x2 a = pair(y[j], y[j + 1]), m = pair(mag[j], mag[j + 1]);
      const f32x2 below = ADA ? fma2(pair(-EPS, -EPS), m, a) : a;
      const f32x2 above = ADA ? fma2(pair(EPS, EPS), m, a) : a;
      unpair(mul2(below, pair(r_lo, r_lo)), lo[j], lo[j + 1]);
      unpair(mul2(above, pair(r_hi, r_hi)), hi[j], hi[j + 1]);
    }
    uint32_t code[2] = {codes4(lo[0], lo[1], lo[2], lo[3]), codes4(lo[4], lo[5], lo[6], lo[7])};
    if (!fine || code[0] != codes4(hi[0], hi[1], hi[2], hi[3]) ||
        code[1] != codes4(hi[4], hi[5], hi[6], hi[7])) {
      float t[8];
      const double sd = s, inv = 1.0 / sd;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double e = exact(j);
        t[j] = off_border(static_cast<float>(e * inv), e, sd);
      }
      code[0] = codes4(t[0], t[1], t[2], t[3]);
      code[1] = codes4(t[4], t[5], t[6], t[7]);
    }
    io.store_codes(p.q + row * p.ld_q, c, code[0], code[1]);
    if ((lane & (LANES - 1)) == 0 && c < p.dim) p.scales[row * p.ld_scales + c / GROUP] = s;
  }
}

}  // namespace n8
}  // namespace fvb
