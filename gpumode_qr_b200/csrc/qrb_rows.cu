// The forward product of a few rows (tokens): y = act(x W^T + b) + r with
// m <= kRowsMost rows, bound by reading W once. One launch, no workspace: a CTA
// takes 16 or 32 of W's rows, its eight warps interleave along k and add their
// sums in shared memory in order, then run the epilogue.
//
// 16-bit types: W's rows are the 16-row operand of mma.sync m16n8k16 and eight
// tokens the 8-column one, so both go from global memory straight to registers.
// (tcgen05 takes its operands from shared memory and rows in 128s; at a few
// tokens the product is 1 / 100 of what either unit does while W streams in.)
// The reduction's order is free, so lane (g, t) takes 8 consecutive values at
// 8 t of row g, one 16-byte load, as the fragments of two MMAs; x is read the
// same way. FP32: fused multiply-adds, four rows of W per warp.
#include "qrb_linear.cuh"

namespace qrb {
namespace lin {
namespace {

constexpr int kWarps = 8;
constexpr int kStep = 32;  // reduction values of one warp step

// Eight 16-bit elements, the first `valid` of them where a 16-byte access is
// not possible.
__device__ __forceinline__ uint4 load8(const void* p, bool vec, int valid) {
  if (valid >= 8 && vec) return __ldg(reinterpret_cast<const uint4*>(p));
  const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < valid) w[i / 2] |= (uint32_t)__ldg(q + i) << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                      uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (__is_same(T, bf16))
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The epilogue of one value per lane: lane = column of W's rows (ROWS of them),
// token tok; every lane of the warp calls it.
template <typename T, int ROWS>
__device__ __forceinline__ void finish1(float s, int tok, int64_t col, bool live, int64_t n,
                                        const Epilogue& e) {
  float v[1] = {s};
  if (live && e.bias != nullptr) v[0] += to_f<T>(reinterpret_cast<const T*>(e.bias)[col]);
  if (live && e.z != nullptr)
    reinterpret_cast<T*>(e.z)[(int64_t)tok * e.ldz + col] = from_f<T>(v[0]);
  if constexpr (ROWS == 32) {
    if (e.z_codes != nullptr) {  // a warp is one token's block of 32 columns
      constexpr int lo = ExpRange<T>::lo, hi = ExpRange<T>::hi;
      float f = live && finite_f(v[0]) ? fabsf(v[0]) : 0.f;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) f = fmaxf(f, __shfl_xor_sync(kFull, f, o));
      const int ex = block_exponent(f, lo, hi);
      const float q4[4] = {v[0], 0.f, 0.f, 0.f};
      uint32_t w[1];
      encode(q4, ex, false, ex == hi ? 63.f : 127.f, w);
      if (live) {
        e.z_codes[(int64_t)tok * n + col] = (int8_t)(w[0] & 255u);
        if ((threadIdx.x & 31) == 0)
          e.z_exps[(int64_t)tok * ((n + kBlk - 1) / kBlk) + col / kBlk] = (int8_t)ex;
      }
    }
  }
  if (!live) return;
  float p[2] = {v[0], 0.f};
  act_by(p, e.act);
  if (e.residual != nullptr)
    p[0] += to_f<T>(reinterpret_cast<const T*>(e.residual)[(int64_t)tok * e.ldr + col]);
  reinterpret_cast<T*>(e.out)[(int64_t)tok * e.ldo + col] = from_f<T>(p[0]);
}

// RG groups of 16 rows of W, NT groups of 8 tokens.
template <typename T, int RG, int NT>
__global__ void __launch_bounds__(kWarps * 32)
    k_rows(const T* __restrict__ x, int64_t ldx, const T* __restrict__ w, int64_t ldw, int m,
           int64_t n, int64_t k, int vx, int vw, Epilogue e) {
  constexpr int ROWS = 16 * RG, TOK = 8 * NT, U = NT == 4 ? 2 : 4;
  constexpr int PITCH = ROWS + 4;  // floats of one token's sums
  __shared__ float part[kWarps][TOK][PITCH];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t n0 = (int64_t)blockIdx.x * ROWS;
  float d[RG][NT][4];
#pragma unroll
  for (int r = 0; r < RG; ++r)
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) d[r][c][i] = 0.f;
  for (int64_t kk = warp * kStep; kk < k; kk += kWarps * kStep * U) {
    uint4 a[U][RG][2], b[U][NT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t c = kk + u * kWarps * kStep + t * 8;
      const int have = c >= k ? 0 : (k - c < 8 ? (int)(k - c) : 8);
#pragma unroll
      for (int r = 0; r < RG; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int64_t row = n0 + 16 * r + 8 * h + g;
          a[u][r][h] = load8(w + row * ldw + c, vw, row < n ? have : 0);
        }
#pragma unroll
      for (int q = 0; q < NT; ++q) {
        const int tok = 8 * q + g;
        b[u][q] = load8(x + (int64_t)tok * ldx + c, vx, tok < m ? have : 0);
      }
    }
    // (short chains, added in FP32: the tensor core does not round its adds)
#pragma unroll
    for (int r = 0; r < RG; ++r)
#pragma unroll
      for (int q = 0; q < NT; ++q) {
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < U; ++u) {
          mma16<T>(s, a[u][r][0].x, a[u][r][1].x, a[u][r][0].y, a[u][r][1].y, b[u][q].x,
                   b[u][q].y);
          mma16<T>(s, a[u][r][0].z, a[u][r][1].z, a[u][r][0].w, a[u][r][1].w, b[u][q].z,
                   b[u][q].w);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) d[r][q][i] += s[i];
      }
  }
#pragma unroll
  for (int r = 0; r < RG; ++r)
#pragma unroll
    for (int q = 0; q < NT; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        part[warp][8 * q + 2 * t + (i & 1)][16 * r + g + 8 * (i >> 1)] = d[r][q][i];
  __syncthreads();
  // a warp takes 32 / ROWS tokens at a time
  constexpr int PER = 32 / ROWS;
  const int row = lane % ROWS;
  const int64_t col = n0 + row;
  for (int t0 = warp * PER; t0 < m; t0 += kWarps * PER) {
    const int tok = t0 + lane / ROWS;
    float s = 0.f;
    if (tok < TOK) {
#pragma unroll
      for (int v = 0; v < kWarps; ++v) s += part[v][tok][row];
    }
    finish1<T, ROWS>(s, tok, col, tok < m && col < n, n, e);
  }
}

// FP32: 32 rows of W per CTA, four per warp and pass over k by all 32 lanes.
template <int MT>
__global__ void __launch_bounds__(kWarps * 32)
    k_rows32(const float* __restrict__ x, int64_t ldx, const float* __restrict__ w, int64_t ldw,
             int m, int64_t n, int64_t k, int vx, int vw, Epilogue e) {
  __shared__ float sums[MT][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n0 = (int64_t)blockIdx.x * 32;
  float acc[4][MT];
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int q = 0; q < MT; ++q) acc[r][q] = 0.f;
#pragma unroll 2
  for (int64_t c = lane * 4; c < k; c += 128) {
    const int have = k - c < 4 ? (int)(k - c) : 4;
    float a[4][4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t row = n0 + warp * 4 + r;
      load_n<float, 4>(w + row * ldw + c, vw, row < n ? have : 0, a[r]);
    }
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      float b[4];
      load_n<float, 4>(x + (int64_t)q * ldx + c, vx, q < m ? have : 0, b);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[r][q] = fmaf(a[r][i], b[i], acc[r][q]);
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      float s = acc[r][q];
#pragma unroll
      for (int o = 16; o > 0; o /= 2) s += __shfl_xor_sync(kFull, s, o);
      if (lane == 0) sums[q][warp * 4 + r] = s;
    }
  __syncthreads();
  for (int tok = warp; tok < m; tok += kWarps)
    finish1<float, 32>(sums[tok][lane], tok, n0 + lane, n0 + lane < n, n, e);
}

template <typename T, int RG, int NT>
void run16(const Operand& x, const Operand& w, int64_t m, int64_t n, int64_t k, int vx, int vw,
           const Epilogue& e, cudaStream_t s) {
  const int64_t grid = (n + 16 * RG - 1) / (16 * RG);
  k_rows<T, RG, NT><<<(unsigned)grid, kWarps * 32, 0, s>>>(
      reinterpret_cast<const T*>(x.p), x.ld, reinterpret_cast<const T*>(w.p), w.ld, (int)m, n, k,
      vx, vw, e);
}
template <typename T>
void rows16(const Operand& x, const Operand& w, int64_t m, int64_t n, int64_t k, int vx, int vw,
            const Epilogue& e, cudaStream_t s) {
  const bool wide = e.z_codes != nullptr;  // a packed block is 32 columns
  if (m <= 8)
    wide ? run16<T, 2, 1>(x, w, m, n, k, vx, vw, e, s) : run16<T, 1, 1>(x, w, m, n, k, vx, vw, e, s);
  else if (m <= 16)
    wide ? run16<T, 2, 2>(x, w, m, n, k, vx, vw, e, s) : run16<T, 1, 2>(x, w, m, n, k, vx, vw, e, s);
  else
    wide ? run16<T, 2, 4>(x, w, m, n, k, vx, vw, e, s) : run16<T, 1, 4>(x, w, m, n, k, vx, vw, e, s);
}
template <int MT>
void rows32(const Operand& x, const Operand& w, int64_t m, int64_t n, int64_t k, int vx, int vw,
            const Epilogue& e, cudaStream_t s) {
  k_rows32<MT><<<(unsigned)((n + 31) / 32), kWarps * 32, 0, s>>>(
      reinterpret_cast<const float*>(x.p), x.ld, reinterpret_cast<const float*>(w.p), w.ld, (int)m,
      n, k, vx, vw, e);
}

}  // namespace

int64_t rows_most(int dtype) {
  const int64_t most = dtype == QRBL_F32 ? 8 : 32;
  const int hook = linear_rows();
  return hook < 0 || hook > most ? most : hook;
}

int launch_rows(int dtype, const Operand& x, const Operand& w, int64_t m, int64_t n, int64_t k,
                const Epilogue& e, cudaStream_t s) {
  const int es = elem_size(dtype);
  const int vx = aligned16(x.p) && (m <= 1 || (x.ld * es) % 16 == 0);
  const int vw = aligned16(w.p) && (n <= 1 || (w.ld * es) % 16 == 0);
  switch (dtype) {
    case QRBL_F32:
      if (m <= 1) rows32<1>(x, w, m, n, k, vx, vw, e, s);
      else if (m <= 2) rows32<2>(x, w, m, n, k, vx, vw, e, s);
      else if (m <= 4) rows32<4>(x, w, m, n, k, vx, vw, e, s);
      else rows32<8>(x, w, m, n, k, vx, vw, e, s);
      break;
    case QRBL_F16: rows16<f16>(x, w, m, n, k, vx, vw, e, s); break;
    case QRBL_BF16: rows16<bf16>(x, w, m, n, k, vx, vw, e, s); break;
    default: return QRB_ERR_INVALID_ARG;
  }
  note_launches(1);
  return cudaGetLastError() == cudaSuccess ? QRB_OK : QRB_ERR_LAUNCH;
}

}  // namespace lin
}  // namespace qrb
