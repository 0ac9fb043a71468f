// Elementwise and column-sum kernels of the linear-layer operators: the packed
// 8-bit form, operands staged for the products, dz = dy act'(z) with the bias
// gradient's sums, and the join of a product split along its reduction. Each
// value is read once and written once, so HBM bounds them; what keeps them from it
// is instructions per value, hence the byte permutes instead of conversions, the
// packed FP32 arithmetic and 16 values per access. Measured on a B200, 8192 x 4096
// BF16: k_pack 18.6 us (5.4 TB/s), k_unpack 16.7 us (6.0 TB/s), dz with GELU from
// packed z 39 us (4.2 TB/s: 26 instructions a value, among them two of the
// special-function unit, which alone take 15 us), of HBM's 6.5 TB/s. FP32, the same
// size: k_pack 26.1 us (6.4 TB/s), k_unpack 43.5 us (3.9 TB/s).
#include "qrb_linear.cuh"

namespace qrb {
namespace lin {
namespace {

constexpr int kThreads = 256;

bool rows_aligned(const void* p, int64_t ld, int elem, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) % bytes) == 0 && (ld * elem) % bytes == 0;
}

// Threads tx over the columns (V values each), 256 / tx over the rows, `per`
// rows each: blocks over the columns fastest.
struct Cover {
  int tx;            // a power of two, at least one packed block's threads
  int64_t nx;        // blocks along the columns
  int64_t blocks;
};
Cover cover(int64_t rows, int64_t cols, int v, int per) {
  Cover c;
  const int64_t want = (cols + v - 1) / v;
  c.tx = 4;
  while (c.tx < want && c.tx < kThreads) c.tx *= 2;
  c.nx = (want + c.tx - 1) / c.tx;
  const int64_t high = (int64_t)(kThreads / c.tx) * per;
  c.blocks = c.nx * ((rows + high - 1) / high);
  return c;
}

// Eight codes: one access where they are all there and aligned.
__device__ __forceinline__ uint2 load_codes(const int8_t* p, bool vec, int valid) {
  if (vec && valid >= 8) return *reinterpret_cast<const uint2*>(p);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < valid) w[i / 4] |= (uint32_t)(uint8_t)p[i] << (8 * (i % 4));
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ int clip(int64_t left, int most) {
  return left >= most ? most : (left > 0 ? (int)left : 0);
}

// 32 bytes at a 32-byte aligned address in one access.
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]),
               "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
// ---------------------------------------------------------------------------
// pack
// ---------------------------------------------------------------------------
// Two neighbouring threads hold one block of 32 values; its largest magnitude
// comes from one shuffle. ROWS rows per thread keep that many loads in flight
// (8192 x 4096 BF16: 18.6 us, 5.4 TB/s; four rows hold too many registers, 18.9).
template <typename T, int ROWS>
__global__ void __launch_bounds__(kThreads)
    k_pack(const T* __restrict__ x, int64_t ld, int64_t rows, int64_t cols, int64_t nblk,
           int8_t* __restrict__ codes, int8_t* __restrict__ exps, int tx, int64_t nx, int vin,
           int vout) {
  constexpr int lo = ExpRange<T>::lo, hi = ExpRange<T>::hi, V = 16;
  const int64_t by = blockIdx.x / (uint32_t)nx, bx = blockIdx.x % (uint32_t)nx;
  const int ty = kThreads / tx, x0 = threadIdx.x & (tx - 1), y0 = threadIdx.x / tx;
  const int64_t c = (bx * tx + x0) * V;
  const int64_t r0 = by * ty * ROWS + y0;
  const int valid = clip(cols - c, V);
  Raw8<T> raw[ROWS][2];
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const int64_t r = r0 + (int64_t)j * ty;
    const int have = r < rows ? valid : 0;
    const T* p = x + r * ld + c;
    raw[j][0] = load_raw8<T>(p, vin, have);
    raw[j][1] = load_raw8<T>(p + 8, vin, have - 8);
  }
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const int64_t r = r0 + (int64_t)j * ty;
    float v[V];
    values8<T>(raw[j][0], *reinterpret_cast<float(*)[8]>(v));
    values8<T>(raw[j][1], *reinterpret_cast<float(*)[8]>(v + 8));
    float a = fabsf(v[0]);
#pragma unroll
    for (int i = 1; i < V; ++i) a = max_abs_nan(a, v[i]);
    a = max_abs_nan(a, __shfl_xor_sync(kFull, a, 1));
    const bool fine = finite_f(a);
    if (__any_sync(kFull, !fine)) {  // Inf or NaN somewhere: exponents from the rest
      float f = finite_amax(v);
      f = fmaxf(f, __shfl_xor_sync(kFull, f, 1));
      a = f;
    }
    const int e = block_exponent(a, lo, hi);
    uint32_t w[V / 4];
    encode(v, e, fine && e < hi, e == hi ? 63.f : 127.f, w);
    if (r >= rows || valid == 0) continue;
    int8_t* out = codes + r * cols + c;
    if (vout && valid == V) {
      *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < valid) out[i] = (int8_t)(w[i / 4] >> (8 * (i % 4)));
    }
    if ((threadIdx.x & 1) == 0) exps[r * nblk + c / kBlk] = (int8_t)e;
  }
}

// ---------------------------------------------------------------------------
// stage / unpack
// ---------------------------------------------------------------------------
struct StageJob {
  StageArgs a;
  int tx = 4;
  int64_t nx = 1, blocks = 0, nblk = 0;
  int vin = 0, vout = 0;
};
constexpr int stage_rows(int elem) { return elem == 4 ? 2 : 4; }
constexpr int kStageVals = 16;

// A matrix as a product's operand or as itself. PACKED: from codes and
// exponents. PLANES: three BF16 planes of FP32 values; else type T. 16 values of
// each of four rows (FP32: two) per thread, the loads of all in flight together.
template <typename T, bool PACKED, bool PLANES>
__device__ __forceinline__ void stage_block(const StageJob& j, int64_t block) {
  constexpr int V = kStageVals, ROWS = sizeof(T) == 4 ? 2 : 4;
  const StageArgs& a = j.a;
  const int64_t by = (uint32_t)block / (uint32_t)j.nx, bx = (uint32_t)block % (uint32_t)j.nx;
  const int ty = kThreads / j.tx, x0 = threadIdx.x & (j.tx - 1), y0 = threadIdx.x / j.tx;
  const int64_t c = (bx * j.tx + x0) * V;
  if (!j.vin) {  // rows not 16-byte aligned: one row, neighbouring threads at neighbouring values
    const int64_t c0 = bx * j.tx * V + x0;
    const int64_t r = by * ty + y0;
    if (r >= a.rows) return;
    float v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int64_t cc = c0 + (int64_t)k * j.tx;
      if (cc >= a.cols)
        v[k] = 0.f;
      else if constexpr (PACKED)
        v[k] = value_of(a.codes[r * a.cols + cc], pow2f(a.exps[r * j.nblk + cc / kBlk]));
      else
        v[k] = to_f<T>(reinterpret_cast<const T*>(a.src)[r * a.lds + cc]);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int64_t cc = c0 + (int64_t)k * j.tx;
      if (cc >= a.cols) continue;
      if constexpr (PLANES) {
        bf16* d = reinterpret_cast<bf16*>(a.dst) + r * a.ldd + cc;
        split3(v[k], d[0], d[a.plane], d[2 * a.plane]);
      } else {
        reinterpret_cast<T*>(a.dst)[r * a.ldd + cc] = from_f<T>(v[k]);
      }
    }
    return;
  }
  const int64_t r0 = by * ty * ROWS + y0;
  const int valid = clip(a.cols - c, V);
  if (valid == 0) return;
  Raw8<T> raw[ROWS][2];
  uint4 q[ROWS];
  int e[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int64_t r = r0 + (int64_t)i * ty;
    const int have = r < a.rows ? valid : 0;
    if constexpr (PACKED) {
      const int8_t* p = a.codes + r * a.cols + c;
      if (j.vin && have == V) {
        q[i] = *reinterpret_cast<const uint4*>(p);
      } else {
        const uint2 lo = load_codes(p, false, have), hi = load_codes(p + 8, false, have - 8);
        q[i] = make_uint4(lo.x, lo.y, hi.x, hi.y);
      }
      e[i] = have > 0 ? a.exps[r * j.nblk + c / kBlk] : 0;
    } else {
      const T* p = reinterpret_cast<const T*>(a.src) + r * a.lds + c;
      raw[i][0] = load_raw8<T>(p, j.vin, have);
      raw[i][1] = load_raw8<T>(p + 8, j.vin, have - 8);
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int64_t r = r0 + (int64_t)i * ty;
    if (r >= a.rows) return;
    if constexpr (PACKED && sizeof(T) == 2) {
      if (j.vout == 2 && valid == V) {
        uint32_t w[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[8];
          decode8(h == 0 ? make_uint2(q[i].x, q[i].y) : make_uint2(q[i].z, q[i].w), e[i],
                  v);
#pragma unroll
          for (int k = 0; k < 4; ++k) w[4 * h + k] = pair_of<T>(v[2 * k], v[2 * k + 1]);
        }
        store32(reinterpret_cast<T*>(a.dst) + r * a.ldd + c, w);
        continue;
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (valid <= 8 * h) continue;
      float v[8];
      if constexpr (PACKED)
        decode8(h == 0 ? make_uint2(q[i].x, q[i].y) : make_uint2(q[i].z, q[i].w), e[i], v);
      else
        values8<T>(raw[i][h], v);
      if constexpr (PLANES) {
        bf16* d = reinterpret_cast<bf16*>(a.dst) + r * a.ldd + c + 8 * h;
        Vec<bf16, 8> p[3];
#pragma unroll
        for (int k = 0; k < 8; ++k) split3(v[k], p[0].v[k], p[1].v[k], p[2].v[k]);
#pragma unroll
        for (int k = 0; k < 3; ++k)  // ldd % 8 == 0: the padding may be written
          *reinterpret_cast<Vec<bf16, 8>*>(d + k * a.plane) = p[k];
      } else {
        store_n<T, 8>(reinterpret_cast<T*>(a.dst) + r * a.ldd + c + 8 * h, j.vout, valid - 8 * h,
                      v);
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_unpack(StageJob j) {
  stage_block<T, true, false>(j, blockIdx.x);
}

// ---------------------------------------------------------------------------
// dz = dy act'(z), and its column sums
// ---------------------------------------------------------------------------
// dz is rounded to T here: the tensor cores take operands of one 16-bit type, and a
// second one with the remainder would double both products (8192 x 4096 x 4096: 340 us
// more). It puts dx's and dW's relative error from 1.66e-3, the rounding of the result
// alone, to 2.35e-3 in BF16 and from 2.1e-4 to 2.9e-4 in FP16. The bias gradient sums
// dz unrounded; FP32 dz keeps its 24 bits.
// Warps of 256 columns (8 per lane), 8 warps over the rows; a block takes `rows`
// rows of them, 2 (FP32: 1) per warp loaded together. Each thread sums its rows in
// order, then the block's warps are added in order: the same bits every time.
// part[row block][col].
struct DzJob {
  DzArgs a;
  int64_t nx = 1, blocks = 0, nblk = 0;
  int rows = 32, vdy = 0, vz = 0, vdst = 0;
};
// Rows that are not all aligned: one value at a time, lane + 32 i of the
// block's 256 columns, neighbouring lanes at neighbouring values.
template <typename T, bool PACKED, bool PLANES>
__device__ __forceinline__ void dz_rows_any(const DzJob& j, int64_t c0, int64_t rb, int64_t rend,
                                            float (&acc)[8]) {
  const DzArgs& a = j.a;
  for (int64_t r = rb + (threadIdx.x >> 5); r < rend; r += 8) {
    float d[8], f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t c = c0 + (threadIdx.x & 31) + 32 * i;
      const bool in = c < a.n;
      d[i] = in ? to_f<T>(reinterpret_cast<const T*>(a.dy)[r * a.lddy + c]) : 0.f;
      f[i] = 0.f;
      if (a.act != QRBL_ACT_NONE && in) {
        if constexpr (PACKED)
          f[i] = value_of(a.z_codes[r * a.n + c], pow2f(a.z_exps[r * j.nblk + c / kBlk]));
        else
          f[i] = to_f<T>(reinterpret_cast<const T*>(a.z)[r * a.ldz + c]);
      }
    }
    f2 d2[4], f2v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      d2[i] = f2_of(d[2 * i], d[2 * i + 1]);
      f2v[i] = f2_of(f[2 * i], f[2 * i + 1]);
    }
    act_grad_by(d2, f2v, a.act);
#pragma unroll
    for (int i = 0; i < 4; ++i) f2_to(d2[i], d[2 * i], d[2 * i + 1]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t c = c0 + (threadIdx.x & 31) + 32 * i;
      acc[i] += d[i];
      if (a.dst == nullptr || c >= a.n) continue;
      if constexpr (PLANES) {
        bf16* out = reinterpret_cast<bf16*>(a.dst) + r * a.ldd + c;
        split3(d[i], out[0], out[a.plane], out[2 * a.plane]);
      } else {
        reinterpret_cast<T*>(a.dst)[r * a.ldd + c] = from_f<T>(d[i]);
      }
    }
  }
}

template <typename T, bool PACKED, bool PLANES>
__device__ __forceinline__ void dz_block(const DzJob& j, int64_t block, float (*sums)[256]) {
  constexpr int V = 8, D = sizeof(T) == 4 ? 1 : 2;  // rows loaded together
  const DzArgs& a = j.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t by = (uint32_t)block / (uint32_t)j.nx, bx = (uint32_t)block % (uint32_t)j.nx;
  const int64_t c = (bx * 32 + lane) * V;
  const int64_t rb = by * j.rows;
  const int64_t rend = rb + j.rows < a.m ? rb + j.rows : a.m;
  const int valid = clip(a.n - c, V);
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  const bool any = !(j.vdy && (j.vz || a.act == QRBL_ACT_NONE) && (j.vdst || a.dst == nullptr));
  if (any) {
    dz_rows_any<T, PACKED, PLANES>(j, bx * 256, rb, rend, acc);
  } else if (valid > 0) {
    f2 sum[4] = {0, 0, 0, 0};
    // this lane's values of its first row, and the step to the warp's next
    const int64_t r0 = rb + warp;
    const T* pg = reinterpret_cast<const T*>(a.dy) + r0 * a.lddy + c;
    const T* pz = reinterpret_cast<const T*>(a.z) + (PACKED ? 0 : r0 * a.ldz + c);
    const int8_t* pq = a.z_codes + (PACKED ? r0 * a.n + c : 0);
    const int8_t* pe = a.z_exps + (PACKED ? r0 * j.nblk + c / kBlk : 0);
    T* pd = reinterpret_cast<T*>(a.dst);
    if constexpr (PLANES)
      pd = reinterpret_cast<T*>(reinterpret_cast<bf16*>(a.dst) + r0 * a.ldd + c);
    else
      pd += r0 * a.ldd + c;
    const int64_t sg = 8 * a.lddy, sz = 8 * a.ldz, sq = 8 * a.n, se = 8 * j.nblk, sd = 8 * a.ldd;
    for (int left = (int)(rend - r0); left > 0; left -= 8 * D) {
      Raw8<T> g[D], z[D];
      uint2 q[D];
      int e[D];
#pragma unroll
      for (int k = 0; k < D; ++k) {
        const int have = left > 8 * k ? valid : 0;
        g[k] = load_raw8<T>(pg + k * sg, true, have);
        if (a.act != QRBL_ACT_NONE) {
          if constexpr (PACKED) {
            q[k] = load_codes(pq + k * sq, true, have);
            e[k] = have > 0 ? pe[k * se] : 0;
          } else {
            z[k] = load_raw8<T>(pz + k * sz, true, have);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < D; ++k) {
        if (left <= 8 * k) break;
        float f[V];
        f2 d[4];
        values8<T>(g[k], f);
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = f2_of(f[2 * i], f[2 * i + 1]);
        if (a.act != QRBL_ACT_NONE) {
          f2 zv[4];
          if constexpr (PACKED) {
            decode8(q[k], e[k], zv);
          } else {
            values8<T>(z[k], f);
#pragma unroll
            for (int i = 0; i < 4; ++i) zv[i] = f2_of(f[2 * i], f[2 * i + 1]);
          }
          act_grad_by(d, zv, a.act);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = add2(sum[i], d[i]);
        if (a.dst == nullptr) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) f2_to(d[i], f[2 * i], f[2 * i + 1]);
        if constexpr (PLANES) {
          bf16* out = reinterpret_cast<bf16*>(pd) + k * sd;
          Vec<bf16, V> p[3];
#pragma unroll
          for (int i = 0; i < V; ++i) split3(f[i], p[0].v[i], p[1].v[i], p[2].v[i]);
#pragma unroll
          for (int i = 0; i < 3; ++i)
            *reinterpret_cast<Vec<bf16, V>*>(out + i * a.plane) = p[i];
        } else {
          store_n<T, V>(pd + k * sd, true, valid, f);
        }
      }
      pg += D * sg;
      if constexpr (PACKED) {
        pq += D * sq;
        pe += D * se;
      } else {
        pz += D * sz;
      }
      if constexpr (PLANES)
        pd = reinterpret_cast<T*>(reinterpret_cast<bf16*>(pd) + D * sd);
      else
        pd += D * sd;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) f2_to(sum[i], acc[2 * i], acc[2 * i + 1]);
  }
  if (a.part == nullptr) return;
#pragma unroll
  for (int i = 0; i < V; ++i) sums[warp][lane + 32 * i] = acc[i];
  __syncthreads();
  const int t = threadIdx.x;  // one column each: lane t / 8, value t % 8 (any: lane t % 32)
  const int at = any ? t : t / V + 32 * (t % V);
  float s = 0.f;
#pragma unroll
  for (int y = 0; y < 8; ++y) s += sums[y][at];
  const int64_t col = bx * 256 + t;
  if (col < a.n) a.part[by * a.n + col] = s;
}

// One launch for all that comes before a product: the first blocks are dz's,
// then the first and the second staged operand's. (Alternating dz's, which are
// bound by instructions, with the staged operands', which are bound by HBM,
// leaves the long dz blocks to the end: 69 us instead of 57 at 8192 x 4096 GELU
// and packed x; so do dz blocks of 32 rows, 66.)
struct PrepArgs {
  DzJob dz;
  StageJob st[2];
};
template <typename T>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 3 : 4)
    k_prepare(const __grid_constant__ PrepArgs p) {
  constexpr bool PLANES = sizeof(T) == 4;
  __shared__ float sums[8][256];
  let_next_start();
  int64_t b = blockIdx.x;
  if (b < p.dz.blocks) {
    if (p.dz.a.z_codes != nullptr)
      dz_block<T, true, PLANES>(p.dz, b, sums);
    else
      dz_block<T, false, PLANES>(p.dz, b, sums);
    return;
  }
  b -= p.dz.blocks;
  const bool second = b >= p.st[0].blocks;
  const StageJob& j = p.st[second ? 1 : 0];
  if (second) b -= p.st[0].blocks;
  if (j.a.codes != nullptr)
    stage_block<T, true, PLANES>(j, b);
  else
    stage_block<T, false, PLANES>(j, b);
}

// out[col] = sum over the blocks of part[block][col].
template <typename T>
__global__ void __launch_bounds__(128) k_colsum(ColSum c) {
  column_sum<T>(c, (int64_t)blockIdx.x * 4 + threadIdx.x / 32, (int64_t)gridDim.x * 4);
}

// ---------------------------------------------------------------------------
// join: epilogue(sum of the partial products)
// ---------------------------------------------------------------------------
// Four columns per thread, eight neighbouring threads per packed block.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    k_join(const float* __restrict__ part, int splits, int64_t rows, int64_t ld, int64_t m,
           int64_t n, Epilogue e) {
  wait_for_previous();
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
  act_by(v, e.act);
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

template <typename T>
int pack_t(const void* x, int64_t ld, int64_t rows, int64_t cols, int8_t* codes, int8_t* exps,
           cudaStream_t s) {
  constexpr int ROWS = sizeof(T) == 4 ? 1 : 2;
  const Cover g = cover(rows, cols, 16, ROWS);
  if (g.blocks > 0x7fffffffLL) return QRB_ERR_UNSUPPORTED;
  k_pack<T, ROWS><<<(unsigned)g.blocks, kThreads, 0, s>>>(
      reinterpret_cast<const T*>(x), ld, rows, cols, blocks_of(cols), codes, exps, g.tx, g.nx,
      rows_aligned(x, ld, sizeof(T), 16), rows_aligned(codes, cols, 1, 16));
  return launched();
}

StageJob stage_job(int elem, const StageArgs& a) {
  StageJob j;
  j.a = a;
  j.vin = a.codes != nullptr ? rows_aligned(a.codes, a.cols, 1, 16)
                             : rows_aligned(a.src, a.lds, elem, 16);
  const Cover g = cover(a.rows, a.cols, kStageVals, j.vin ? stage_rows(elem) : 1);
  j.tx = g.tx;
  j.nx = g.nx;
  j.blocks = g.blocks;
  j.nblk = blocks_of(a.cols);
  j.vout = rows_aligned(a.dst, a.ldd, elem, 32) ? 2 : rows_aligned(a.dst, a.ldd, elem, 16);
  return j;
}

template <typename T>
int unpack_t(const int8_t* codes, const int8_t* exps, int64_t rows, int64_t cols, void* x,
             int64_t ld, cudaStream_t s) {
  StageArgs a;
  a.codes = codes;
  a.exps = exps;
  a.rows = rows;
  a.cols = cols;
  a.dst = x;
  a.ldd = ld;
  const StageJob j = stage_job(sizeof(T), a);
  if (j.blocks > 0x7fffffffLL) return QRB_ERR_UNSUPPORTED;
  k_unpack<T><<<(unsigned)j.blocks, kThreads, 0, s>>>(j);
  return launched();
}

template <typename T>
int prepare_t(const Prepare& p, cudaStream_t s) {
  PrepArgs a;
  int64_t blocks = 0;
  if (p.has_dz) {
    const DzArgs& d = p.dz;
    a.dz.a = d;
    a.dz.rows = colsum_rows(d.m, d.n);
    a.dz.nx = (d.n + 255) / 256;
    a.dz.blocks = a.dz.nx * ((d.m + a.dz.rows - 1) / a.dz.rows);
    a.dz.nblk = blocks_of(d.n);
    a.dz.vdy = rows_aligned(d.dy, d.lddy, sizeof(T), 16);
    a.dz.vdst = rows_aligned(d.dst, d.ldd, sizeof(T), 16);
    a.dz.vz = d.z_codes != nullptr ? rows_aligned(d.z_codes, d.n, 1, 8)
                                   : rows_aligned(d.z, d.ldz, sizeof(T), 16);
    blocks += a.dz.blocks;
  }
  for (int i = 0; i < p.stages; ++i) {
    a.st[i] = stage_job(sizeof(T), p.stage[i]);
    blocks += a.st[i].blocks;
  }
  if (blocks == 0) return QRB_OK;
  if (blocks > 0x7fffffffLL) return QRB_ERR_UNSUPPORTED;
  k_prepare<T><<<(unsigned)blocks, kThreads, 0, s>>>(a);
  return launched();
}

template <typename T>
int join_t(const float* part, int splits, int64_t rows, int64_t ld, int64_t m, int64_t n,
           const Epilogue& e, bool after_product, cudaStream_t s) {
  int tx = 8;  // a packed block stays within one warp
  while (tx * 4 < n && tx < kThreads) tx *= 2;
  const int ty = kThreads / tx;
  const int64_t gx = (m + ty - 1) / ty, gy = (n + 4 * tx - 1) / (4 * tx);
  if (gx > 0x7fffffffLL || gy > 65535) return QRB_ERR_UNSUPPORTED;
  cudaLaunchConfig_t lc = {};
  cudaLaunchAttribute early = early_start();
  lc.gridDim = dim3((unsigned)gx, (unsigned)gy);
  lc.blockDim = dim3((unsigned)tx, (unsigned)ty);
  lc.stream = s;
  lc.attrs = &early;
  lc.numAttrs = after_product ? 1 : 0;
  if (cudaLaunchKernelEx(&lc, k_join<T>, part, splits, rows, ld, m, n, e) != cudaSuccess) {
    (void)cudaGetLastError();
    return QRB_ERR_LAUNCH;
  }
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
  QRBL_BY_TYPE(dtype, return unpack_t<T>(codes, exps, rows, cols, x, ld, s));
}

int launch_prepare(int dtype, const Prepare& p, cudaStream_t s) {
  QRBL_BY_TYPE(dtype, return prepare_t<T>(p, s));
}

// 128 rows where that leaves four blocks or more per SM (fewer partial sums to
// write and add), 32 where that leaves one, else 8: a row per warp.
int colsum_rows(int64_t m, int64_t n) {
  const int64_t across = (n + 255) / 256;
  if ((m + 127) / 128 * across >= 592) return 128;
  return (m + 31) / 32 * across >= 148 ? 32 : 8;
}

int launch_colsum(int dtype, const ColSum& c, cudaStream_t s) {
  const int64_t gx = (c.n * c.slices + 127) / 128;
  const unsigned grid = (unsigned)(gx < 65535 ? gx : 65535);
  QRBL_BY_TYPE(dtype, {
    k_colsum<T><<<grid, 128, 0, s>>>(c);
    return launched();
  });
}

int launch_join(int dtype, const float* part, int splits, int64_t rows, int64_t ld, int64_t m,
                int64_t n, const Epilogue& e, bool after_product, cudaStream_t s) {
  QRBL_BY_TYPE(dtype, return join_t<T>(part, splits, rows, ld, m, n, e, after_product, s));
}

}  // namespace lin
}  // namespace qrb
