// Shared pieces of the linear-layer operators (qrb_linear.cu, qrb_mm.cu,
// qrb_act.cu): element types, activations and their derivatives, the packed
// 8-bit form, and the internal launchers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/qrb200_linear.h"
#include "qrb_common.cuh"

namespace qrb {
namespace lin {

using bf16 = __nv_bfloat16;
using f16 = __half;

constexpr int kBlk = 32;         // values that share an exponent in the packed form
constexpr int kNanCode = -128;

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
// EXACT (FP32 layers): the library functions. Otherwise (results rounded to 8
// or 11 bits): the hardware exponential and reciprocal (relative error below
// 2^-20), and Phi from Abramowitz and Stegun 7.1.26 (absolute error of erf
// below 1.5e-7).
template <bool EXACT>
__device__ __forceinline__ float sigmoid(float v) {
  if constexpr (EXACT) return 1.0f / (1.0f + expf(-v));
  return __fdividef(1.0f, 1.0f + __expf(-v));  // exp overflow: 1 / inf = 0
}

// Phi(z), and exp(-z^2 / 2) for its derivative.
template <bool EXACT>
__device__ __forceinline__ float normal_cdf(float z, float* gauss) {
  const float h = z * 0.70710678118654752f;
  if constexpr (EXACT) {
    *gauss = expf(-h * h);
    return 0.5f * erfcf(-h);
  }
  const float x = fabsf(h);
  const float e = __expf(-x * x);
  const float t = __fdividef(1.0f, fmaf(0.3275911f, x, 1.0f));
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  const float q = 0.5f * p * t * e;  // erfc(x) / 2
  *gauss = e;
  return z >= 0.f ? 1.0f - q : (z < 0.f ? q : z);  // NaN stays NaN
}

constexpr float kTanhC = 1.5957691216057308f;  // 2 sqrt(2 / pi): tanh(u) = 2 sigmoid(2 u) - 1

template <bool EXACT>
__device__ __forceinline__ float act_fn(float z, int act) {
  switch (act) {
    case QRBL_ACT_RELU: return z > 0.f ? z : (z <= 0.f ? 0.f : z);
    case QRBL_ACT_GELU: {
      float g;
      return z * normal_cdf<EXACT>(z, &g);
    }
    case QRBL_ACT_GELU_TANH: return z * sigmoid<EXACT>(kTanhC * fmaf(0.044715f * z * z, z, z));
    case QRBL_ACT_SILU: return z * sigmoid<EXACT>(z);
    default: return z;
  }
}

template <bool EXACT>
__device__ __forceinline__ float act_grad_fn(float z, int act) {
  switch (act) {
    case QRBL_ACT_RELU: return z > 0.f ? 1.f : (z <= 0.f ? 0.f : z);
    case QRBL_ACT_GELU: {
      float g;
      const float p = normal_cdf<EXACT>(z, &g);
      return fmaf(0.3989422804014327f * z, g, p);
    }
    case QRBL_ACT_GELU_TANH: {
      const float z2 = z * z;
      const float s = sigmoid<EXACT>(kTanhC * fmaf(0.044715f * z2, z, z));
      // z s (1 - s) u' with u' = kTanhC (1 + 3 * 0.044715 z^2); s (1 - s) is 0
      // where the sigmoid has saturated, also where u' overflows
      const float d = s * (1.0f - s);
      return d > 0.f ? fmaf(z * d, kTanhC * fmaf(0.134145f, z2, 1.0f), s) : s;
    }
    case QRBL_ACT_SILU: {
      const float s = sigmoid<EXACT>(z);
      const float d = s * (1.0f - s);
      return d > 0.f ? fmaf(z, d, s) : s;
    }
    default: return 1.f;
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
// Four codes as values. A byte q + 128 put under the exponent of 2^23 is the
// float 2^23 + 128 + q; kNanCode (byte 0 after the flip) becomes NaN.
__device__ __forceinline__ void decode4(uint32_t codes, float step, float (&out)[4]) {
  const uint32_t y = codes ^ 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    out[i] = (__uint_as_float(__byte_perm(y, 0x4b000000u, 0x7540 + i)) - 8388736.f) * step;
  if ((y - 0x01010101u) & ~y & 0x80808080u) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (((y >> (8 * i)) & 255u) == 0) out[i] = __uint_as_float(0x7fc00000u);
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
};
ProductPlan plan_products(int dtype, const ProductSize* sizes, int count);
int launch_products(int dtype, const Product* products, int count, const ProductPlan& plan,
                    cudaStream_t s);
// out = epilogue(sum of `splits` partial sums), part[s][row][col] with rows
// `rows` and row stride ld (splits may be 0).
int launch_join(int dtype, const float* part, int splits, int64_t rows, int64_t ld, int64_t m,
                int64_t n, const Epilogue& e, cudaStream_t s);

int launch_pack(int dtype, const void* x, int64_t ld, int64_t rows, int64_t cols, int8_t* codes,
                int8_t* exps, cudaStream_t s);
int launch_unpack(int dtype, const int8_t* codes, const int8_t* exps, int64_t rows, int64_t cols,
                  void* x, int64_t ld, cudaStream_t s);
// A plain (src) or packed (codes, exps) matrix as a product's operand: copied
// to dst with row stride ldd, FP32 split into three planes `plane` apart.
int launch_stage(int dtype, const void* src, int64_t lds, const int8_t* codes, const int8_t* exps,
                 int64_t rows, int64_t cols, void* dst, int64_t ldd, int64_t plane,
                 cudaStream_t s);
// dz = dy act'(z) as an operand (dst may be null: only the sums), and the
// column sums of the unrounded dz over each block of colsum_rows(m, n) rows
// into part [blocks][n] (null: none).
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
int launch_dz(int dtype, const DzArgs& a, cudaStream_t s);
int launch_colsum(int dtype, const float* part, int64_t blocks, int64_t n, void* out,
                  cudaStream_t s);

}  // namespace lin
}  // namespace qrb
