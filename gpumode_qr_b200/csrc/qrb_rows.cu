// The forward product of a few rows (tokens): y = act(x W^T + b) + r where
// takes_rows(), bound by reading W once. One launch, no workspace: a
// CTA takes 16 of W's rows (FP32: 8; z kept in 8 bits: 32), its eight warps
// interleave along k and add their sums in shared memory in order, then run the
// epilogue. 1 x 4096 x 4096 BF16: 9.2 us from HBM, 3.6 TB/s (its floor 5.2 us;
// the rest is the launch and two round trips to HBM), FP32 14.8 us, 4.5 TB/s.
//
// 16-bit types: W's rows are the 16-row operand of mma.sync m16n8k16 and eight
// tokens the 8-column one, so both go from global memory straight to registers.
// (tcgen05 takes its operands from shared memory and rows in 128s; at a few
// tokens the product is 1 / 100 of what either unit does while W streams in.)
// The reduction's order is free, so lane (g, t) takes 8 consecutive values at
// 8 t of row g, one 16-byte load, as the fragments of two MMAs; x is read the
// same way. FP32: fused multiply-adds, eight rows of W at a time, two CTAs on an SM;
// more tokens in groups of four or eight over the grid, each of which reads W
// again from L2 (8 x 4096 x 4096: 26.6 us; with five shuffles for each of a warp's 64
// sums and one CTA on an SM 42.8).
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
  if (valid <= 0) return make_uint4(0, 0, 0, 0);
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

// RG groups of 16 rows of W, NT groups of 8 tokens, U steps' loads in flight.
template <typename T, int RG, int NT, int U>
__global__ void __launch_bounds__(kWarps * 32)
    k_rows(const T* __restrict__ x, int64_t ldx, const T* __restrict__ w, int64_t ldw, int m,
           int64_t n, int64_t k, int vx, int vw, Epilogue e) {
  constexpr int ROWS = 16 * RG, TOK = 8 * NT;
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

// FP32: G passes of 8 rows of W per CTA and MT tokens (of blockIdx.y's group); in
// each its eight warps interleave along k, 128 values a step.
template <int MT, int G>
__global__ void __launch_bounds__(kWarps * 32, 2)
    k_rows32(const float* __restrict__ x, int64_t ldx, const float* __restrict__ w, int64_t ldw,
             int m, int64_t n, int64_t k, int vx, int vw, Epilogue e) {
  constexpr int R = 8;
  __shared__ float sums[kWarps][MT][R * G + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n0 = (int64_t)blockIdx.x * R * G;
  const int tok0 = (int)blockIdx.y * MT;
  x += (int64_t)tok0 * ldx;
  m -= tok0;
#pragma unroll 1
  for (int g = 0; g < G; ++g) {
    float acc[R][MT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int q = 0; q < MT; ++q) acc[r][q] = 0.f;
#pragma unroll(MT == 8 ? 1 : 2)
    for (int64_t c = warp * 128 + lane * 4; c < k; c += kWarps * 128) {
      const int have = k - c < 4 ? (int)(k - c) : 4;
      float a[R][4];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int64_t row = n0 + g * R + r;
        load_n<float, 4>(w + row * ldw + c, vw, row < n ? have : 0, a[r]);
      }
#pragma unroll
      for (int q = 0; q < MT; ++q) {
        float b[4];
        load_n<float, 4>(x + (int64_t)q * ldx + c, vx, q < m ? have : 0, b);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[r][q] = fmaf(a[r][i], b[i], acc[r][q]);
      }
    }
    // the warp's sums of each of the R MT accumulators: a step over half the lanes
    // also halves the accumulators a lane still holds, of which it keeps those of
    // its side, so 64 take 62 shuffles instead of 320
    constexpr int N = R * MT;
    float(&v)[N] = *reinterpret_cast<float(*)[N]>(&acc[0][0]);
#pragma unroll
    for (int o = 16, left = N; o > 0; o /= 2) {
      const bool up = (lane & o) != 0;
      if (left > 1) {
        left /= 2;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          if (i >= left) break;
          const float mine = up ? v[i + left] : v[i], other = up ? v[i] : v[i + left];
          v[i] = mine + __shfl_xor_sync(kFull, other, o);
        }
      } else {
        v[0] += __shfl_xor_sync(kFull, v[0], o);
      }
    }
    constexpr int EACH = N > 32 ? N / 32 : 1, SAME = N < 32 ? 32 / N : 1;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const int at = lane / SAME * EACH + j;
      if (lane % SAME == 0) sums[warp][at % MT][g * R + at / MT] = v[j];
    }
  }
  __syncthreads();
  // a warp takes 32 / (R G) tokens at a time
  constexpr int ROWS = R * G, PER = 32 / ROWS;
  const int row = lane % ROWS;
  const int64_t col = n0 + row;
  for (int t0 = warp * PER; t0 < MT; t0 += kWarps * PER) {
    const int tok = t0 + lane / ROWS;
    float s = 0.f;
    if (tok < MT) {
#pragma unroll
      for (int v = 0; v < kWarps; ++v) s += sums[v][tok][row];
    }
    finish1<float, ROWS>(s, tok0 + tok, col, tok < MT && tok < m && col < n, n, e);
  }
}

template <typename T, int RG, int NT, int U>
void run16(const Operand& x, const Operand& w, int64_t m, int64_t n, int64_t k, int vx, int vw,
           const Epilogue& e, cudaStream_t s) {
  const int64_t grid = (n + 16 * RG - 1) / (16 * RG);
  k_rows<T, RG, NT, U><<<(unsigned)grid, kWarps * 32, 0, s>>>(
      reinterpret_cast<const T*>(x.p), x.ld, reinterpret_cast<const T*>(w.p), w.ld, (int)m, n, k,
      vx, vw, e);
}
// Steps in flight: what k has for one warp, at most 8 (one group of tokens), 4 or
// 2: at 1 x 4096 x 4096 8 steps take 9.2 us against 11.0 for 4; at k = 512, where a
// warp has 2 steps, 8 take 5.1 us and 4 take 3.3.
template <typename T, int RG>
void rows16(const Operand& x, const Operand& w, int64_t m, int64_t n, int64_t k, int vx, int vw,
            const Epilogue& e, cudaStream_t s) {
  const int64_t steps = (k + kWarps * kStep - 1) / (kWarps * kStep);
  if (m > 16)
    run16<T, RG, 4, 2>(x, w, m, n, k, vx, vw, e, s);
  else if (m > 8)
    steps > 2 ? run16<T, RG, 2, 4>(x, w, m, n, k, vx, vw, e, s)
              : run16<T, RG, 2, 2>(x, w, m, n, k, vx, vw, e, s);
  else if (steps > 4 && RG == 1)
    run16<T, RG, 1, RG == 1 ? 8 : 4>(x, w, m, n, k, vx, vw, e, s);
  else if (steps > 2)
    run16<T, RG, 1, 4>(x, w, m, n, k, vx, vw, e, s);
  else
    run16<T, RG, 1, 2>(x, w, m, n, k, vx, vw, e, s);
}
// Whether groups of four tokens give no more CTAs than fit (two on each of 148
// SMs): faster than groups of eight then (8 x 1024 x 1024: 3.4 us against 5.0), slower
// where they read W twice as often in more waves (8 x 4096 x 4096: 32.3 against 26.6).
bool at_once(int64_t m, int64_t n, bool wide) {
  const int64_t rows = wide ? 32 : 8;
  return (n + rows - 1) / rows * ((m + 3) / 4) <= 2 * 148;
}
template <int MT>
void rows32(const Operand& x, const Operand& w, int64_t m, int64_t n, int64_t k, int vx, int vw,
            const Epilogue& e, cudaStream_t s) {
  const bool wide = e.z_codes != nullptr;  // a packed block is 32 columns
  const int64_t rows = wide ? 32 : 8;
  const dim3 grid((unsigned)((n + rows - 1) / rows), (unsigned)((m + MT - 1) / MT));
  const float* xp = reinterpret_cast<const float*>(x.p);
  const float* wp = reinterpret_cast<const float*>(w.p);
  if (wide)
    k_rows32<MT, 4><<<grid, kWarps * 32, 0, s>>>(xp, x.ld, wp, w.ld, (int)m, n, k, vx,
                                                           vw, e);
  else
    k_rows32<MT, 1><<<grid, kWarps * 32, 0, s>>>(xp, x.ld, wp, w.ld, (int)m, n, k, vx,
                                                           vw, e);
}

}  // namespace

// 16-bit types: up to 16 rows, 32 where k is short (32 x 4096 x 1024: 5.6 us
// against 8.5 for tiles; 32 x 4096 x 4096: 15.9 against 13.9). FP32: up to 8 rows, and
// more where the groups' estimate, in microseconds, is below the tiles', most of
// which is W's three planes being written and read back (32 x 1024 x 1024: 9.9
// against 13.0, 48: 13.7 against 13.2; 16 x 4096 x 4096: 51.6 against 68.7, 24: 74.5
// against 68.2; 64 x 1024 x 256: 15.3 against 11.5). With z packed a CTA's four passes
// over k follow one another, which few columns do not hide (4 x 64 x 8192: 38.1
// against 16.8).
bool takes_rows(int dtype, int64_t m, int64_t n, int64_t k, bool packed) {
  const int hook = linear_rows();
  if (hook >= 0) return m <= hook;
  if (dtype != QRBL_F32) return m <= (k <= 1024 ? 32 : 16);
  const double tiles = 10.0 + 3.4e-6 * (double)n * (double)k;
  if (m > 128 || (packed && 5.0 + 0.004 * (double)k > tiles)) return false;
  const double groups = (double)((n + 7) / 8 * ((m + 7) / 8));
  return m <= 8 || 1.3 + groups * (0.0128 + 8e-6 * (double)k) < tiles;
}

int launch_rows(int dtype, const Operand& x, const Operand& w, int64_t m, int64_t n, int64_t k,
                const Epilogue& e, cudaStream_t s) {
  const int es = elem_size(dtype);
  const int vx = aligned16(x.p) && (m <= 1 || (x.ld * es) % 16 == 0);
  const int vw = aligned16(w.p) && (n <= 1 || (w.ld * es) % 16 == 0);
  const bool wide = e.z_codes != nullptr;  // a packed block is 32 columns
  switch (dtype) {
    case QRBL_F32:
      if (m <= 1) rows32<1>(x, w, m, n, k, vx, vw, e, s);
      else if (m <= 2) rows32<2>(x, w, m, n, k, vx, vw, e, s);
      else if (m <= 4 || at_once(m, n, wide)) rows32<4>(x, w, m, n, k, vx, vw, e, s);
      else rows32<8>(x, w, m, n, k, vx, vw, e, s);
      break;
    case QRBL_F16:
      wide ? rows16<f16, 2>(x, w, m, n, k, vx, vw, e, s) : rows16<f16, 1>(x, w, m, n, k, vx, vw, e, s);
      break;
    case QRBL_BF16:
      wide ? rows16<bf16, 2>(x, w, m, n, k, vx, vw, e, s)
           : rows16<bf16, 1>(x, w, m, n, k, vx, vw, e, s);
      break;
    default: return QRB_ERR_INVALID_ARG;
  }
  note_launches(1);
  return cudaGetLastError() == cudaSuccess ? QRB_OK : QRB_ERR_LAUNCH;
}

}  // namespace lin
}  // namespace qrb
