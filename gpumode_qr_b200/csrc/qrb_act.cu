// Elementwise and column-sum kernels of the linear-layer operators: the packed
// 8-bit form, operands staged for the products, dz = dy act'(z) with the bias
// gradient's sums, and the join of a product split along its reduction. All
// are bound by HBM: each value is read once and written once, 8 per thread.
#include "qrb_linear.cuh"

namespace qrb {
namespace lin {
namespace {

constexpr int kThreads = 256;
constexpr int kVals = 8;     // values per thread and row

// Threads tx over the columns (8 each), 256 / tx over the rows.
struct Grid2 {
  int tx;
  dim3 grid, block;
};
Grid2 grid2(int64_t rows, int64_t cols, int rows_per_thread, bool* ok) {
  Grid2 g;
  int64_t want = (cols + kVals - 1) / kVals;
  g.tx = 4;  // a 32-value block stays within one warp
  while (g.tx < want && g.tx < kThreads) g.tx *= 2;
  const int64_t per = (int64_t)(kThreads / g.tx) * rows_per_thread;
  const int64_t gx = (rows + per - 1) / per;
  const int64_t gy = (want + g.tx - 1) / g.tx;
  *ok = gx <= 0x7fffffffLL && gy <= 65535;
  g.grid = dim3((unsigned)gx, (unsigned)gy);
  g.block = dim3((unsigned)g.tx, (unsigned)(kThreads / g.tx));
  return g;
}

// Eight codes: one access where they are all there and aligned.
__device__ __forceinline__ uint2 load_codes(const int8_t* p, bool vec, int valid) {
  if (vec && valid >= kVals) return *reinterpret_cast<const uint2*>(p);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < kVals; ++i)
    if (i < valid) w[i / 4] |= (uint32_t)(uint8_t)p[i] << (8 * (i % 4));
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void decode8(uint2 q, float step, float (&out)[kVals]) {
  float lo[4], hi[4];
  decode4(q.x, step, lo);
  decode4(q.y, step, hi);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    out[i] = lo[i];
    out[4 + i] = hi[i];
  }
}

// ---------------------------------------------------------------------------
// pack / unpack
// ---------------------------------------------------------------------------
// Four neighbouring threads hold one block of 32 values; its largest magnitude
// comes from two shuffles. ROWS rows per thread keep that many loads in flight.
template <typename T, int ROWS>
__global__ void __launch_bounds__(kThreads)
    k_pack(const T* __restrict__ x, int64_t ld, int64_t rows, int64_t cols, int64_t nblk,
           int8_t* __restrict__ codes, int8_t* __restrict__ exps, int vin, int vout) {
  const int64_t c = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * kVals;
  const int64_t r0 = (int64_t)blockIdx.x * blockDim.y * ROWS + threadIdx.y;
  constexpr int lo = ExpRange<T>::lo, hi = ExpRange<T>::hi;
  float v[ROWS][kVals];
  const int valid = (int)(cols - c < kVals ? (cols > c ? cols - c : 0) : kVals);
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const int64_t r = r0 + (int64_t)j * blockDim.y;
    load_n<T, kVals>(x + r * ld + c, vin, r < rows ? valid : 0, v[j]);
  }
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const int64_t r = r0 + (int64_t)j * blockDim.y;
    float a = fabsf(v[j][0]);
#pragma unroll
    for (int i = 1; i < kVals; ++i) a = max_abs_nan(a, v[j][i]);
    a = max_abs_nan(a, __shfl_xor_sync(kFull, a, 1));
    a = max_abs_nan(a, __shfl_xor_sync(kFull, a, 2));
    if (__any_sync(kFull, !finite_f(a))) {
      const bool fine = finite_f(a);
      float f = finite_amax(v[j]);
      f = fmaxf(f, __shfl_xor_sync(kFull, f, 1));
      f = fmaxf(f, __shfl_xor_sync(kFull, f, 2));
      if (!fine) {  // Inf or NaN in this block: its exponent from the rest
        const int e = block_exponent(f, lo, hi);
        uint32_t w[2];
        encode(v[j], e, false, e == hi ? 63.f : 127.f, w);
        if (r < rows && valid > 0) {
          int8_t* out = codes + r * cols + c;
#pragma unroll
          for (int i = 0; i < kVals; ++i)
            if (i < valid) out[i] = (int8_t)(w[i / 4] >> (8 * (i % 4)));
          if ((threadIdx.x & 3) == 0) exps[r * nblk + c / kBlk] = (int8_t)e;
        }
        continue;
      }
    }
    const int e = block_exponent(a, lo, hi);
    uint32_t w[2];
    encode(v[j], e, plain_block(a, e, hi), 63.f, w);
    if (r >= rows || valid == 0) continue;
    int8_t* out = codes + r * cols + c;
    if (vout && valid >= kVals) {
      *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int i = 0; i < kVals; ++i)
        if (i < valid) out[i] = (int8_t)(w[i / 4] >> (8 * (i % 4)));
    }
    if ((threadIdx.x & 3) == 0) exps[r * nblk + c / kBlk] = (int8_t)e;
  }
}

// A matrix as a product's operand or as itself. PACKED: from codes and
// exponents. PLANES: three BF16 planes of FP32 values; else type T.
template <typename T, bool PACKED, bool PLANES, int ROWS>
__global__ void __launch_bounds__(kThreads)
    k_stage(const T* __restrict__ x, int64_t ld, const int8_t* __restrict__ codes,
            const int8_t* __restrict__ exps, int64_t rows, int64_t cols, int64_t nblk,
            void* __restrict__ dst, int64_t ldd, int64_t plane, int vin, int vout) {
  const int64_t c = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * kVals;
  const int64_t r0 = (int64_t)blockIdx.x * blockDim.y * ROWS + threadIdx.y;
  if (c >= cols) return;
  const int valid = (int)(cols - c < kVals ? cols - c : kVals);
  float v[ROWS][kVals];
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const int64_t r = r0 + (int64_t)j * blockDim.y;
    if constexpr (PACKED) {
      const uint2 q = load_codes(codes + r * cols + c, vin, r < rows ? valid : 0);
      decode8(q, r < rows ? pow2f(exps[r * nblk + c / kBlk]) : 0.f, v[j]);
    } else {
      load_n<T, kVals>(x + r * ld + c, vin, r < rows ? valid : 0, v[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const int64_t r = r0 + (int64_t)j * blockDim.y;
    if (r >= rows) continue;
    if constexpr (PLANES) {
      bf16* d = reinterpret_cast<bf16*>(dst) + r * ldd + c;
      Vec<bf16, kVals> p[3];
#pragma unroll
      for (int i = 0; i < kVals; ++i) split3(v[j][i], p[0].v[i], p[1].v[i], p[2].v[i]);
#pragma unroll
      for (int k = 0; k < 3; ++k)  // ldd % 8 == 0: the padding may be written
        *reinterpret_cast<Vec<bf16, kVals>*>(d + k * plane) = p[k];
    } else {
      store_n<T, kVals>(reinterpret_cast<T*>(dst) + r * ldd + c, vout, valid, v[j]);
    }
  }
}

// ---------------------------------------------------------------------------
// dz = dy act'(z), and its column sums
// ---------------------------------------------------------------------------
// Warps of 256 columns (8 per lane), 8 warps over the rows; a block takes `rows`
// rows of them, 2 per warp at a time so that their loads are in flight
// together. Each thread sums its rows in order, then the block's warps are
// added in order: the same bits every time. part[blockIdx.x][col].
constexpr int kDzRows = 2;
template <bool EXACT, int ACT>
__device__ __forceinline__ void dz8(float (&d)[kVals], const float (&z)[kVals]) {
#pragma unroll
  for (int i = 0; i < kVals; ++i) d[i] *= act_grad_fn<EXACT>(z[i], ACT);
}
template <typename T, bool PACKED, bool PLANES>
__global__ void __launch_bounds__(kThreads, 3)
    k_dz(DzArgs a, int64_t nblk, int rows, int vdy, int vz, int vdst) {
  __shared__ float sums[8][32 * kVals];
  constexpr bool EXACT = sizeof(T) == 4;
  const int lane = threadIdx.x, warp = threadIdx.y;
  const int64_t c = ((int64_t)blockIdx.y * 32 + lane) * kVals;
  const int64_t rb = (int64_t)blockIdx.x * rows;
  const int64_t rend = rb + rows < a.m ? rb + rows : a.m;
  const int valid = (int)(a.n - c < kVals ? (a.n > c ? a.n - c : 0) : kVals);
  float acc[kVals];
#pragma unroll
  for (int i = 0; i < kVals; ++i) acc[i] = 0.f;
  if (valid > 0) {
    for (int64_t r0 = rb + warp; r0 < rend; r0 += 8 * kDzRows) {
      Raw8<T> g[kDzRows], z[kDzRows];
      uint2 q[kDzRows];
      int e[kDzRows];
#pragma unroll
      for (int j = 0; j < kDzRows; ++j) {
        const int64_t r = r0 + 8 * j;
        const int have = r < rend ? valid : 0;
        g[j] = load_raw8<T>(reinterpret_cast<const T*>(a.dy) + r * a.lddy + c, vdy, have);
        if (a.act != QRBL_ACT_NONE) {
          if constexpr (PACKED) {
            q[j] = load_codes(a.z_codes + r * a.n + c, vz, have);
            e[j] = have > 0 ? a.z_exps[r * nblk + c / kBlk] : 0;
          } else {
            z[j] = load_raw8<T>(reinterpret_cast<const T*>(a.z) + r * a.ldz + c, vz, have);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kDzRows; ++j) {
        const int64_t r = r0 + 8 * j;
        if (r >= rend) break;
        float d[kVals];
        values8<T>(g[j], d);
        if (a.act != QRBL_ACT_NONE) {
          float f[kVals];
          if constexpr (PACKED) {
            decode8(q[j], pow2f(e[j]), f);
          } else {
            values8<T>(z[j], f);
          }
          switch (a.act) {
            case QRBL_ACT_RELU: dz8<EXACT, QRBL_ACT_RELU>(d, f); break;
            case QRBL_ACT_GELU: dz8<EXACT, QRBL_ACT_GELU>(d, f); break;
            case QRBL_ACT_GELU_TANH: dz8<EXACT, QRBL_ACT_GELU_TANH>(d, f); break;
            case QRBL_ACT_SILU: dz8<EXACT, QRBL_ACT_SILU>(d, f); break;
          }
        }
#pragma unroll
        for (int i = 0; i < kVals; ++i) acc[i] += d[i];
        if (a.dst == nullptr) continue;
        if constexpr (PLANES) {
          bf16* out = reinterpret_cast<bf16*>(a.dst) + r * a.ldd + c;
          Vec<bf16, kVals> p[3];
#pragma unroll
          for (int i = 0; i < kVals; ++i) split3(d[i], p[0].v[i], p[1].v[i], p[2].v[i]);
#pragma unroll
          for (int k = 0; k < 3; ++k)
            *reinterpret_cast<Vec<bf16, kVals>*>(out + k * a.plane) = p[k];
        } else {
          store_n<T, kVals>(reinterpret_cast<T*>(a.dst) + r * a.ldd + c, vdst, valid, d);
        }
      }
    }
  }
  if (a.part == nullptr) return;
#pragma unroll
  for (int i = 0; i < kVals; ++i) sums[warp][lane + 32 * i] = acc[i];
  __syncthreads();
  const int t = warp * 32 + lane;  // one column each: lane t / 8, value t % 8
  float s = 0.f;
#pragma unroll
  for (int y = 0; y < 8; ++y) s += sums[y][t / kVals + 32 * (t % kVals)];
  const int64_t col = (int64_t)blockIdx.y * 256 + t;
  if (col < a.n) a.part[(int64_t)blockIdx.x * a.n + col] = s;
}

// out[col] = sum over the blocks of part[block][col]: 32 columns and 8 groups
// of blocks per CTA, the groups added in order.
template <typename T>
__global__ void __launch_bounds__(256)
    k_colsum(const float* __restrict__ part, int64_t blocks, int64_t n, T* __restrict__ out) {
  __shared__ float sums[8][33];
  const int64_t col = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (col < n) {
#pragma unroll 8
    for (int64_t b = threadIdx.y; b < blocks; b += 8) s += part[b * n + col];
  }
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && col < n) {
    float t = 0.f;
#pragma unroll
    for (int y = 0; y < 8; ++y) t += sums[y][threadIdx.x];
    out[col] = from_f<T>(t);
  }
}

// ---------------------------------------------------------------------------
// join: epilogue(sum of the partial products)
// ---------------------------------------------------------------------------
// Four columns per thread, eight neighbouring threads per packed block.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    k_join(const float* __restrict__ part, int splits, int64_t rows, int64_t ld, int64_t m,
           int64_t n, Epilogue e) {
  constexpr bool EXACT = sizeof(T) == 4;
  const int64_t c = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * 4;
  const int64_t r = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const int valid = r < m && c < n ? (int)(n - c < 4 ? n - c : 4) : 0;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (valid > 0) {
    const float* p = part + r * ld + c;  // ld % 4 == 0: the padding is there
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      const float4 u = *reinterpret_cast<const float4*>(p + (int64_t)s * rows * ld);
      v[0] += u.x; v[1] += u.y; v[2] += u.z; v[3] += u.w;
    }
    if (e.bias != nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < valid) v[i] += to_f<T>(reinterpret_cast<const T*>(e.bias)[c + i]);
    }
    if (e.z != nullptr)
      store_n<T, 4>(reinterpret_cast<T*>(e.z) + r * e.ldz + c, e.vec, valid, v);
  }
  if (e.z_codes != nullptr) {  // (the values beyond the row are 0)
    constexpr int lo = ExpRange<T>::lo, hi = ExpRange<T>::hi;
    float f = finite_amax(v), a = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) a = max_abs_nan(a, v[i]);
#pragma unroll
    for (int o = 1; o < 8; o *= 2) {
      f = fmaxf(f, __shfl_xor_sync(kFull, f, o));
      a = max_abs_nan(a, __shfl_xor_sync(kFull, a, o));
    }
    const int ex = block_exponent(f, lo, hi);
    uint32_t w[1];
    encode(v, ex, plain_block(a, ex, hi), ex == hi ? 63.f : 127.f, w);
    if (valid > 0) {
      int8_t* out = e.z_codes + r * n + c;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < valid) out[i] = (int8_t)(w[0] >> (8 * i));
      if ((threadIdx.x & 7) == 0) e.z_exps[r * ((n + kBlk - 1) / kBlk) + c / kBlk] = (int8_t)ex;
    }
  }
  if (valid == 0) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = act_fn<EXACT>(v[i], e.act);
  if (e.residual != nullptr) {
    float q[4];
    load_n<T, 4>(reinterpret_cast<const T*>(e.residual) + r * e.ldr + c, e.vec, valid, q);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += q[i];
  }
  store_n<T, 4>(reinterpret_cast<T*>(e.out) + r * e.ldo + c, e.vec, valid, v);
}

int launched() {
  note_launches(1);
  return cudaGetLastError() == cudaSuccess ? QRB_OK : QRB_ERR_LAUNCH;
}

bool rows_aligned(const void* p, int64_t ld, int elem, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) % bytes) == 0 && (ld * elem) % bytes == 0;
}

template <typename T>
int pack_t(const void* x, int64_t ld, int64_t rows, int64_t cols, int8_t* codes, int8_t* exps,
           cudaStream_t s) {
  constexpr int ROWS = 4;
  bool ok;
  const Grid2 g = grid2(rows, cols, ROWS, &ok);
  if (!ok) return QRB_ERR_UNSUPPORTED;
  k_pack<T, ROWS><<<g.grid, g.block, 0, s>>>(
      reinterpret_cast<const T*>(x), ld, rows, cols, blocks_of(cols), codes, exps,
      rows_aligned(x, ld, sizeof(T), 16), rows_aligned(codes, cols, 1, 8));
  return launched();
}

template <typename T, bool PLANES>
int stage_t(const void* src, int64_t lds, const int8_t* codes, const int8_t* exps, int64_t rows,
            int64_t cols, void* dst, int64_t ldd, int64_t plane, cudaStream_t s) {
  constexpr int ROWS = 4;
  bool ok;
  const Grid2 g = grid2(rows, cols, ROWS, &ok);
  if (!ok) return QRB_ERR_UNSUPPORTED;
  const int vout = rows_aligned(dst, ldd, sizeof(T), 16);
  if (codes != nullptr)
    k_stage<T, true, PLANES, ROWS><<<g.grid, g.block, 0, s>>>(
        nullptr, 0, codes, exps, rows, cols, blocks_of(cols), dst, ldd, plane,
        rows_aligned(codes, cols, 1, 8), vout);
  else
    k_stage<T, false, PLANES, ROWS><<<g.grid, g.block, 0, s>>>(
        reinterpret_cast<const T*>(src), lds, nullptr, nullptr, rows, cols, blocks_of(cols), dst,
        ldd, plane, rows_aligned(src, lds, sizeof(T), 16), vout);
  return launched();
}

template <typename T>
int dz_t(const DzArgs& a, cudaStream_t s) {
  constexpr bool PLANES = sizeof(T) == 4;
  const int rows = colsum_rows(a.m, a.n);
  const int64_t gx = (a.m + rows - 1) / rows, gy = (a.n + 255) / 256;
  if (gx > 0x7fffffffLL || gy > 65535) return QRB_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)gx, (unsigned)gy), block(32, 8);
  const int vdy = rows_aligned(a.dy, a.lddy, sizeof(T), 16);
  const int vdst = rows_aligned(a.dst, a.ldd, sizeof(T), 16);
  if (a.z_codes != nullptr)
    k_dz<T, true, PLANES><<<grid, block, 0, s>>>(a, blocks_of(a.n), rows, vdy,
                                                 rows_aligned(a.z_codes, a.n, 1, 8), vdst);
  else
    k_dz<T, false, PLANES><<<grid, block, 0, s>>>(
        a, blocks_of(a.n), rows, vdy, rows_aligned(a.z, a.ldz, sizeof(T), 16), vdst);
  return launched();
}

template <typename T>
int join_t(const float* part, int splits, int64_t rows, int64_t ld, int64_t m, int64_t n,
           const Epilogue& e, cudaStream_t s) {
  int tx = 8;  // a packed block stays within one warp
  while (tx * 4 < n && tx < kThreads) tx *= 2;
  const int ty = kThreads / tx;
  const int64_t gx = (m + ty - 1) / ty, gy = (n + 4 * tx - 1) / (4 * tx);
  if (gx > 0x7fffffffLL || gy > 65535) return QRB_ERR_UNSUPPORTED;
  k_join<T><<<dim3((unsigned)gx, (unsigned)gy), dim3((unsigned)tx, (unsigned)ty), 0, s>>>(
      part, splits, rows, ld, m, n, e);
  return launched();
}

}  // namespace

#define QRBL_BY_TYPE(dtype, ...)                      \
  switch (dtype) {                                    \
    case QRBL_F32: { using T = float; __VA_ARGS__; }  \
    case QRBL_F16: { using T = f16; __VA_ARGS__; }    \
    case QRBL_BF16: { using T = bf16; __VA_ARGS__; }  \
    default: return QRB_ERR_INVALID_ARG;              \
  }

int launch_pack(int dtype, const void* x, int64_t ld, int64_t rows, int64_t cols, int8_t* codes,
                int8_t* exps, cudaStream_t s) {
  QRBL_BY_TYPE(dtype, return pack_t<T>(x, ld, rows, cols, codes, exps, s));
}

int launch_unpack(int dtype, const int8_t* codes, const int8_t* exps, int64_t rows, int64_t cols,
                  void* x, int64_t ld, cudaStream_t s) {
  QRBL_BY_TYPE(dtype, return (stage_t<T, false>(nullptr, 0, codes, exps, rows, cols, x, ld, 0, s)));
}

int launch_stage(int dtype, const void* src, int64_t lds, const int8_t* codes, const int8_t* exps,
                 int64_t rows, int64_t cols, void* dst, int64_t ldd, int64_t plane,
                 cudaStream_t s) {
  QRBL_BY_TYPE(dtype, return (stage_t<T, sizeof(T) == 4>(src, lds, codes, exps, rows, cols, dst,
                                                         ldd, plane, s)));
}

// 128 rows where that leaves four blocks or more per SM (fewer partial sums to
// write and add), else 32.
int colsum_rows(int64_t m, int64_t n) {
  return ((m + 127) / 128) * ((n + 255) / 256) >= 592 ? 128 : 32;
}

int launch_dz(int dtype, const DzArgs& a, cudaStream_t s) {
  QRBL_BY_TYPE(dtype, return dz_t<T>(a, s));
}

int launch_colsum(int dtype, const float* part, int64_t blocks, int64_t n, void* out,
                  cudaStream_t s) {
  const int64_t gx = (n + 31) / 32;
  QRBL_BY_TYPE(dtype, {
    k_colsum<T><<<(unsigned)gx, dim3(32, 8), 0, s>>>(part, blocks, n, reinterpret_cast<T*>(out));
    return launched();
  });
}

int launch_join(int dtype, const float* part, int splits, int64_t rows, int64_t ld, int64_t m,
                int64_t n, const Epilogue& e, cudaStream_t s) {
  QRBL_BY_TYPE(dtype, return join_t<T>(part, splits, rows, ld, m, n, e, s));
}

}  // namespace lin
}  // namespace qrb
