// Shared pieces of the linear-layer operators (qrb_linear.cu, qrb_mm.cu,
// qrb_act.cu): element types, activations and their derivatives, the packed
// 8-bit form, and the internal launchers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/qrb200_linear.h"
#include "qrb_common.cuh"

namespace qrb {
// qrb_set_config test hooks of the linear products: "linear_cut" (0 automatic,
// else 1000 * CTAs per tile + tile width: 2256, 2128, 1128 or 1064),
// "linear_splits" (parts of the reduction, 0 automatic) and "linear_rows" (most
// rows of the few-row kernel, -1 automatic).
int linear_cut();
int linear_splits();
int linear_rows();
namespace lin {

using bf16 = __nv_bfloat16;
using f16 = __half;

constexpr int kBlk = 32;         // values that share an exponent in the packed form
constexpr int kNanCode = -128;

// Programmatic dependent launch between the kernels of one call: the earlier one
// lets the later one's blocks start (where an SM has room) once all of its own
// have; the later one sets itself up and then waits for the earlier one's
// results.
__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_for_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
// The attribute of a launch that may start before the one in front of it ends.
inline cudaLaunchAttribute early_start() {
  cudaLaunchAttribute a = {};
  a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a.val.programmaticStreamSerializationAllowed = 1;
  return a;
}

// ---------------------------------------------------------------------------
// element types
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<f16>(f16 v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<bf16>(bf16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ f16 from_f<f16>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ bf16 from_f<bf16>(float v) { return __float2bfloat16_rn(v); }

// Exponent range of the packed form (the step 2^e and 63 * 2^emax are normal
// or exact in the type).
template <typename T>
struct ExpRange {
  static constexpr int lo = -126, hi = 122;
};
template <>
struct ExpRange<f16> {
  static constexpr int lo = -24, hi = 10;
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

// N consecutive elements at p as floats: vector accesses (the caller has
// checked alignment) or, element by element, the first `valid` of them (the
// others read as 0).
template <typename T, int N>
__device__ __forceinline__ void load_n(const T* p, bool vec, int valid, float (&out)[N]) {
  if (vec && valid >= N) {
    constexpr int W = (int)(16 / sizeof(T)) < N ? (int)(16 / sizeof(T)) : N;
#pragma unroll
    for (int c = 0; c < N; c += W) {
      const Vec<T, W> u = *reinterpret_cast<const Vec<T, W>*>(p + c);
#pragma unroll
      for (int i = 0; i < W; ++i) out[c + i] = to_f<T>(u.v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = i < valid ? to_f<T>(p[i]) : 0.f;
  }
}

// Eight elements as they are in memory, and their values.
template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load_raw8(const T* p, bool vec, int valid) {
  Raw8<T> out;
  if (vec && valid >= 8) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) out.w[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
    Vec<T, 8> u;
#pragma unroll
    for (int i = 0; i < 8; ++i) u.v[i] = i < valid ? p[i] : from_f<T>(0.f);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) out.w[i] = reinterpret_cast<const uint4*>(&u)[i];
  }
  return out;
}
template <typename T>
__device__ __forceinline__ void values2(uint32_t w, float& lo, float& hi) {
  if constexpr (__is_same(T, bf16)) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = f.x;
    hi = f.y;
  }
}
template <typename T>
__device__ __forceinline__ uint32_t pair_of(float a, float b) {
  if constexpr (__is_same(T, bf16)) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <typename T>
__device__ __forceinline__ void values8(const Raw8<T>& r, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v[4 * i] = __uint_as_float(r.w[i].x);
      v[4 * i + 1] = __uint_as_float(r.w[i].y);
      v[4 * i + 2] = __uint_as_float(r.w[i].z);
      v[4 * i + 3] = __uint_as_float(r.w[i].w);
    }
  } else {
    values2<T>(r.w[0].x, v[0], v[1]);
    values2<T>(r.w[0].y, v[2], v[3]);
    values2<T>(r.w[0].z, v[4], v[5]);
    values2<T>(r.w[0].w, v[6], v[7]);
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_n(T* p, bool vec, int valid, const float (&in)[N]) {
  if (vec && valid >= N) {
    constexpr int W = (int)(16 / sizeof(T)) < N ? (int)(16 / sizeof(T)) : N;
#pragma unroll
    for (int c = 0; c < N; c += W) {
      Vec<T, W> u;
#pragma unroll
      for (int i = 0; i < W; ++i) u.v[i] = from_f<T>(in[c + i]);
      *reinterpret_cast<Vec<T, W>*>(p + c) = u;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < valid) p[i] = from_f<T>(in[i]);
  }
}

// ---------------------------------------------------------------------------
// activations
// ---------------------------------------------------------------------------
// Two values at a time in packed FP32, with the hardware exponential and
// reciprocal (relative error below 2^-21). Every activation is z / (1 + 2^t)
// with t a polynomial in z: t = -log2(e) z for SILU,
// -log2(e) 2 sqrt(2 / pi) (z + 0.044715 z^3) for GELU_TANH, and for GELU a
// degree-13 odd polynomial fitted here to -log2(e) logit(Phi(z)) so that Phi is
// within 6e-8 (weighted minimax over |z| <= 7; beyond, t keeps its sign and
// grows, so Phi saturates): as close as z / 2 (1 + erf) in FP32. The library's
// expf, erfcf and division keep more of the far tails' relative accuracy but
// cost four times the instructions, and unrolled over a row they no longer fit
// the instruction cache (an FP32 128 x 128 tile's epilogue took 17,000 clocks).
constexpr float kTanhC = 1.5957691216057308f;  // 2 sqrt(2 / pi): tanh(u) = 2 sigmoid(2 u) - 1

// Two FP32 values in one 64-bit register.
using f2 = unsigned long long;
__device__ __forceinline__ f2 f2_of(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ f2 f2_of(float a) { return f2_of(a, a); }
__device__ __forceinline__ void f2_to(f2 v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ f2 ex2_2(f2 x) {
  float a, b;
  f2_to(x, a, b);
  return f2_of(ex2(a), ex2(b));
}
__device__ __forceinline__ f2 rcp_2(f2 x) {
  float a, b, r, q;
  f2_to(x, a, b);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(b));
  return f2_of(r, q);
}

constexpr float kLog2e = 1.4426950408889634f;
// 1 / (1 + 2^t(z)); zz = z^2
template <int ACT>
__device__ __forceinline__ f2 gate2(f2 z, f2 zz) {
  f2 t;
  if constexpr (ACT == QRBL_ACT_SILU) {
    t = mul2(z, f2_of(-kLog2e));
  } else if constexpr (ACT == QRBL_ACT_GELU_TANH) {
    t = mul2(z, fma2(zz, f2_of(-kLog2e * kTanhC * 0.044715f), f2_of(-kLog2e * kTanhC)));
  } else {
    f2 q = f2_of(-kLog2e * 3.51234251e-09f);
    q = fma2(q, zz, f2_of(-kLog2e * -2.64526714e-07f));
    q = fma2(q, zz, f2_of(-kLog2e * 7.92948924e-06f));
    q = fma2(q, zz, f2_of(-kLog2e * -1.10612389e-04f));
    q = fma2(q, zz, f2_of(-kLog2e * -6.51899468e-05f));
    q = fma2(q, zz, f2_of(-kLog2e * 7.26661691e-02f));
    q = fma2(q, zz, f2_of(-kLog2e * 1.59576988f));
    t = mul2(z, q);
  }
  return rcp_2(add2(ex2_2(t), f2_of(1.f)));
}
template <int ACT>
__device__ __forceinline__ f2 act2(f2 z) {
  return mul2(z, gate2<ACT>(z, mul2(z, z)));
}
template <int ACT>
__device__ __forceinline__ f2 act_grad2(f2 z) {
  const f2 zz = mul2(z, z);
  if constexpr (ACT == QRBL_ACT_GELU) {
    // Phi(z) + z g / sqrt(2 pi) with g = exp(-z^2 / 2), which also gives Phi:
    // by Abramowitz and Stegun 7.1.26, with x = |z| / sqrt(2) and
    // t = 1 / (1 + 0.3275911 x), erfc(x) = g (a1 t + .. + a5 t^5) within
    // 1.5e-7. (One exponential and one reciprocal; the polynomial above would
    // need a second exponential for g.)
    const f2 sign = 0x8000000080000000ull;
    const f2 g = ex2_2(mul2(zz, f2_of(-0.5f * kLog2e)));
    const f2 t = rcp_2(fma2(z & ~sign, f2_of(0.3275911f * 0.70710678118654752f), f2_of(1.f)));
    f2 q = fma2(t, f2_of(-0.5f * 1.061405429f), f2_of(0.5f * 1.453152027f));
    q = fma2(q, t, f2_of(-0.5f * 1.421413741f));
    q = fma2(q, t, f2_of(0.5f * 0.284496736f));
    q = fma2(q, t, f2_of(-0.5f * 0.254829592f));
    const f2 half = fma2(mul2(q, t), g, f2_of(0.5f));  // 1 / 2 - erfc(x) / 2 >= 0
    const f2 phi = add2(half | (z & sign), f2_of(0.5f));
    return fma2(mul2(z, f2_of(0.3989422804014327f)), g, phi);
  }
  const f2 s = gate2<ACT>(z, zz);
  const f2 d = fma2(mul2(s, f2_of(-1.f)), s, s);  // s (1 - s)
  if constexpr (ACT == QRBL_ACT_GELU_TANH) {
    float a, b;
    f2_to(zz, a, b);  // capped: the factor stays finite where s (1 - s) is 0
    const f2 cap = f2_of(fminf(a, 1e6f), fminf(b, 1e6f));
    return fma2(mul2(z, d), fma2(cap, f2_of(0.134145f * kTanhC), f2_of(kTanhC)), s);
  }
  return fma2(z, d, s);
}

// v <- act(v), and d <- d act'(z).
template <int ACT, int N>
__device__ __forceinline__ void act_n(float (&v)[N]) {
  if constexpr (ACT == QRBL_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = v[i] <= 0.f ? 0.f : v[i];  // NaN stays NaN
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) f2_to(act2<ACT>(f2_of(v[i], v[i + 1])), v[i], v[i + 1]);
  }
}
template <int ACT>
__device__ __forceinline__ f2 slope2(f2 z) {
  if constexpr (ACT == QRBL_ACT_RELU) {
    float a, b;
    f2_to(z, a, b);
    return f2_of(a > 0.f ? 1.f : (a <= 0.f ? 0.f : a), b > 0.f ? 1.f : (b <= 0.f ? 0.f : b));
  } else {
    return act_grad2<ACT>(z);
  }
}
template <int ACT, int N>
__device__ __forceinline__ void act_grad_n(f2 (&d)[N], const f2 (&z)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) d[i] = mul2(d[i], slope2<ACT>(z[i]));
}
template <int N>
__device__ __forceinline__ void act_by(float (&v)[N], int act) {
  switch (act) {
    case QRBL_ACT_RELU: act_n<QRBL_ACT_RELU>(v); break;
    case QRBL_ACT_GELU: act_n<QRBL_ACT_GELU>(v); break;
    case QRBL_ACT_GELU_TANH: act_n<QRBL_ACT_GELU_TANH>(v); break;
    case QRBL_ACT_SILU: act_n<QRBL_ACT_SILU>(v); break;
    default: break;
  }
}
template <int N>
__device__ __forceinline__ void act_grad_by(f2 (&d)[N], const f2 (&z)[N], int act) {
  switch (act) {
    case QRBL_ACT_RELU: act_grad_n<QRBL_ACT_RELU>(d, z); break;
    case QRBL_ACT_GELU: act_grad_n<QRBL_ACT_GELU>(d, z); break;
    case QRBL_ACT_GELU_TANH: act_grad_n<QRBL_ACT_GELU_TANH>(d, z); break;
    case QRBL_ACT_SILU: act_grad_n<QRBL_ACT_SILU>(d, z); break;
    default: break;
  }
}

// ---------------------------------------------------------------------------
// the packed form
// ---------------------------------------------------------------------------
__device__ __forceinline__ bool finite_f(float x) {
  return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
}

// The smallest e with amax <= 127 * 2^e, clamped to [lo, hi]; amax finite.
// With amax = f * 2^p, 0.5 <= f < 1: e = p - 7, one more where f > 127 / 128.
__device__ __forceinline__ int block_exponent(float amax, int lo, int hi) {
  const uint32_t u = __float_as_uint(amax);
  int e = (int)(u >> 23) - 126 - 7 + ((u & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  e = e < lo ? lo : e;
  return e > hi ? hi : e;
}
__device__ __forceinline__ float pow2f(int e) {  // -126 <= e <= 127
  return __uint_as_float((uint32_t)(e + 127) << 23);
}
// The larger magnitude; NaN if either is.
__device__ __forceinline__ float max_abs_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}
// Whether a block whose largest magnitude is amax (by max_abs_nan) and whose
// exponent is e takes the short path of encode: all values finite, and none
// rounds above its limit.
__device__ __forceinline__ bool plain_block(float amax, int e, int hi) {
  return finite_f(amax) && e < hi;
}
// Codes of N values of a block, x / 2^e rounded to nearest even. Short path:
// x * 2^-e (exact) added to 1.5 * 2^23 in one rounding leaves the integer in
// the sum's low byte. Otherwise Inf and NaN get kNanCode and the rest is held
// to `most`.
template <int N>
__device__ __forceinline__ void encode(const float (&v)[N], int e, bool plain, float most,
                                       uint32_t (&w)[N / 4]) {
  const float scale = pow2f(-e);
  if (plain) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      uint32_t t[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) t[j] = __float_as_uint(fmaf(v[i + j], scale, 12582912.f));
      w[i / 4] = __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040),
                             0x5410);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      uint32_t t[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float q = fminf(fmaxf(rintf(v[i + j] * scale), -most), most);
        t[j] = (uint32_t)(finite_f(v[i + j]) ? (int)q : kNanCode) & 255u;
      }
      w[i / 4] = t[0] | (t[1] << 8) | (t[2] << 16) | (t[3] << 24);
    }
  }
}
// The largest finite magnitude (the short path's amax where all are finite).
template <int N>
__device__ __forceinline__ float finite_amax(const float (&v)[N]) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) a = fmaxf(a, finite_f(v[i]) ? fabsf(v[i]) : 0.f);
  return a;
}
// One code as a value.
__device__ __forceinline__ float value_of(int code, float step) {
  return code == kNanCode ? __uint_as_float(0x7fc00000u) : (float)code * step;
}
// Eight codes of a block with exponent e as values. A byte q + 128 put under the
// exponent of 2^23 is the float 2^23 + 128 + q; one multiply-add takes the offset
// off and scales (exactly: a power of two), as long as the scaled offset does not
// overflow. kNanCode (byte 0 after the flip) and exponents beyond that go the
// long way.
constexpr int kDecodeMost = 104;
__device__ __forceinline__ float code_float(uint32_t flipped, int i) {
  return __uint_as_float(__byte_perm(flipped, 0x4b000000u, 0x7540 + i));
}
__device__ __forceinline__ bool decode_long(uint32_t y0, uint32_t y1, int e) {
  return ((((y0 - 0x01010101u) & ~y0) | ((y1 - 0x01010101u) & ~y1)) & 0x80808080u) != 0 ||
         e > kDecodeMost;
}
__device__ __forceinline__ float decode_one(uint32_t flipped, int i, int e) {
  const int code = (int)((flipped >> (8 * i)) & 255u) - 128;
  return code == kNanCode ? __uint_as_float(0x7fc00000u) : (float)code * pow2f(e);
}
__device__ __forceinline__ void decode8(uint2 q, int e, float (&out)[8]) {
  const uint32_t y0 = q.x ^ 0x80808080u, y1 = q.y ^ 0x80808080u;
  const float step = pow2f(e), off = -8388736.f * step;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    out[i] = fmaf(code_float(y0, i), step, off);
    out[4 + i] = fmaf(code_float(y1, i), step, off);
  }
  if (decode_long(y0, y1, e)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out[i] = decode_one(y0, i, e);
      out[4 + i] = decode_one(y1, i, e);
    }
  }
}
__device__ __forceinline__ void decode8(uint2 q, int e, f2 (&out)[4]) {  // as pairs
  const uint32_t y0 = q.x ^ 0x80808080u, y1 = q.y ^ 0x80808080u;
  const float step = pow2f(e), off = -8388736.f * step;
  const f2 st = f2_of(step), of = f2_of(off);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    out[i] = fma2(f2_of(code_float(y0, 2 * i), code_float(y0, 2 * i + 1)), st, of);
    out[2 + i] = fma2(f2_of(code_float(y1, 2 * i), code_float(y1, 2 * i + 1)), st, of);
  }
  if (decode_long(y0, y1, e)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      out[i] = f2_of(decode_one(y0, 2 * i, e), decode_one(y0, 2 * i + 1, e));
      out[2 + i] = f2_of(decode_one(y1, 2 * i, e), decode_one(y1, 2 * i + 1, e));
    }
  }
}

// An FP32 value as three BF16 parts by truncation: a + b + c == x exactly for
// 2^-110 < |x| < inf (smaller values lose low bits). Inf and NaN stay in a.
__device__ __forceinline__ void split3(float x, bf16& a, bf16& b, bf16& c) {
  if (!finite_f(x)) {
    a = __float2bfloat16_rn(x);
    b = c = __float2bfloat16_rn(0.f);
    return;
  }
  const float h = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
  const float r = x - h;
  const float m = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
  a = __float2bfloat16_rn(h);
  b = __float2bfloat16_rn(m);
  c = __float2bfloat16_rn(r - m);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
inline int elem_size(int dtype) { return dtype == QRBL_F32 ? 4 : 2; }
inline int64_t blocks_of(int64_t cols) { return (cols + kBlk - 1) / kBlk; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// What the product's epilogue reads and writes beside the accumulators.
struct Epilogue {
  void* out = nullptr;
  int64_t ldo = 0;
  const void* bias = nullptr;
  const void* residual = nullptr;
  int64_t ldr = 0;
  void* z = nullptr;
  int64_t ldz = 0;
  int8_t* z_codes = nullptr;
  int8_t* z_exps = nullptr;
  int act = QRBL_ACT_NONE;
  int vec = 0;  // out, residual and z rows are 16-byte aligned
};

// One operand of a product: `rows` x `cols` elements in memory, row stride ld,
// 16-byte aligned rows. FP32 layers: three BF16 planes, `plane` elements apart.
struct Operand {
  const void* p = nullptr;
  int64_t rows = 0, cols = 0, ld = 0, plane = 0;
};

// out [m, n] = A B + epilogue with A [m, k] and B [k, n] given as operands:
//   kForward  A = x [m, k], B = w [n, k] transposed
//   kGradIn   A = dz [m, k], B = w [k, n]
//   kGradW    A = dz [k, m] transposed, B = x [k, n]
enum ProductKind { kForward = 0, kGradIn = 1, kGradW = 2 };

struct ProductSize {
  int64_t m = 0, n = 0, k = 0;
  int epilogue = 0;  // extra work per value: 1 activation, 2 kept z, 4 residual;
                     // 8: chains summed in FP32 (z kept in 8 bits)
};
struct Product {
  int kind = kForward;
  ProductSize size;
  Operand a, b;
  float* part = nullptr;  // splits > 1: part_bytes of workspace
  Epilogue e;
};
// How the products of one launch are cut: tiles of 128 cg x bn on cg CTAs, each
// product's reduction in `splits` parts (their FP32 sums joined by a second
// kernel), the tiles of product `first` first.
struct ProductPlan {
  bool ok = false;
  int cg = 1, bn = 128, first = 0;
  int splits[2] = {1, 1};
  int64_t part_rows[2] = {0, 0}, part_ld[2] = {0, 0};
  size_t part_bytes[2] = {0, 0};
  size_t chain_bytes = 0;  // 16-bit reductions longer than an accumulator chain
};
struct ColSum;
ProductPlan plan_products(int dtype, const ProductSize* sizes, int count);
// chains: the plan's chain_bytes of workspace (null where it has none). sum (may be
// null): column sums finished in the same launch. after_prepare: the launch in front
// of it on the stream is this call's launch_prepare.
int launch_products(int dtype, const Product* products, int count, const ProductPlan& plan,
                    float* chains, const ColSum* sum, bool after_prepare, cudaStream_t s);
// The forward product of few rows (where takes_rows), x and w read in place at any
// alignment.
bool takes_rows(int dtype, int64_t m, int64_t n, int64_t k, bool packed);
int launch_rows(int dtype, const Operand& x, const Operand& w, int64_t m, int64_t n, int64_t k,
                const Epilogue& e, cudaStream_t s);
// out = epilogue(sum of `splits` partial sums), part[s][row][col] with rows
// `rows` and row stride ld (splits may be 0). after_product: the launch in front
// of it on the stream is this call's k_product (or another join after it).
int launch_join(int dtype, const float* part, int splits, int64_t rows, int64_t ld, int64_t m,
                int64_t n, const Epilogue& e, bool after_product, cudaStream_t s);

int launch_pack(int dtype, const void* x, int64_t ld, int64_t rows, int64_t cols, int8_t* codes,
                int8_t* exps, cudaStream_t s);
int launch_unpack(int dtype, const int8_t* codes, const int8_t* exps, int64_t rows, int64_t cols,
                  void* x, int64_t ld, cudaStream_t s);
// What has to be done before a product, in one launch: up to two operands
// staged, and dz = dy act'(z).
// A plain (src) or packed (codes, exps) matrix as a product's operand: copied
// to dst with row stride ldd, FP32 split into three planes `plane` apart.
struct StageArgs {
  const void* src = nullptr;
  int64_t lds = 0;
  const int8_t* codes = nullptr;
  const int8_t* exps = nullptr;
  int64_t rows = 0, cols = 0;
  void* dst = nullptr;
  int64_t ldd = 0, plane = 0;
};
// dz as an operand (dst may be null: only the sums), and the column sums of the
// unrounded dz over each block of colsum_rows(m, n) rows into part [blocks][n]
// (null: none).
int colsum_rows(int64_t m, int64_t n);
struct DzArgs {
  const void* dy = nullptr;
  int64_t lddy = 0;
  const void* z = nullptr;
  int64_t ldz = 0;
  const int8_t* z_codes = nullptr;
  const int8_t* z_exps = nullptr;
  int act = 0;
  int64_t m = 0, n = 0;
  void* dst = nullptr;
  int64_t ldd = 0, plane = 0;
  float* part = nullptr;
};
struct Prepare {
  StageArgs stage[2];
  int stages = 0;
  DzArgs dz;
  bool has_dz = false;
};
int launch_prepare(int dtype, const Prepare& p, cudaStream_t s);
// out[col] = sum of part[block][col]; a product's launch can do it as well
// (ColSum), while its first tiles accumulate.
struct ColSum {
  const float* part = nullptr;
  int64_t blocks = 0, n = 0;
  void* out = nullptr;
  int slices = 1;  // lanes of a warp that share a column, a power of two
};
// A warp takes 32 / slices columns: lane (slice, column) adds every slices-th block's
// sum in order, then the slices are added in a fixed tree, all in 64 bits (there are
// as many sums as a long batch has blocks).
template <typename T>
__device__ __forceinline__ void column_sum(const ColSum& c, int64_t warp, int64_t warps) {
  const int lane = threadIdx.x & 31, wide = 32 / c.slices, slice = lane / wide;
  for (int64_t c0 = warp * wide; c0 < c.n; c0 += warps * wide) {
    const int64_t col = c0 + lane % wide;
    double s = 0;
    if (col < c.n) {
#pragma unroll 16
      for (int64_t b = slice; b < c.blocks; b += c.slices) s += c.part[b * c.n + col];
    }
    for (int o = wide; o < 32; o *= 2) s += __shfl_xor_sync(kFull, s, o);
    if (slice == 0 && col < c.n) reinterpret_cast<T*>(c.out)[col] = from_f<T>((float)s);
  }
}
// As many slices as leave each lane 16 sums, which it loads together, or as fill half
// the card's lanes. Whole backward calls, BF16, k = 64, with one lane a column and so:
// 20,000 x 64 25.0 and 13.6 us, 1,000,000 x 64 565 and 277, 8192 x 1024 21.3 and 16.1.
inline int colsum_slices(int64_t blocks, int64_t n) {
  int s = 1;
  while (s < 32 && blocks > 16 * s && n * s <= 148 * 256) s *= 2;
  return s;
}
int launch_colsum(int dtype, const ColSum& c, cudaStream_t s);

}  // namespace lin
}  // namespace qrb
