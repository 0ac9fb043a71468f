// The linear layers' matrix product: out [m, n] = epilogue(A B) on the tcgen05
// tensor cores, operands fed by TMA, for the forward product x W^T and the
// backward products dz W and dz^T x.
//
// Tiles of 128 x BN per CTA over a persistent grid of one CTA per SM. Ten
// warps: 0-7 read the accumulators (warp w: TMEM lanes 32 (w & 3) .. + 31, one
// half of the columns by w >> 2) and run the epilogue, 8 loads (one lane
// issues TMA boxes into a ring of stages), 9 issues the MMAs (one lane) and
// owns the TMEM. A stage holds 64 of the reduction's values for both operands
// (128-byte swizzle). An operand whose reduction runs along memory rows is
// K-major; one whose reduction runs across them (w in dz W, both operands of
// dz^T x) is MN-major, so no operand is ever transposed in memory. Two
// accumulator buffers let the epilogue of one tile run beside the MMAs of the
// next.
//
// FP32 operands come as three BF16 planes a0 + a1 + a2 (24 bits). A stage
// holds all three planes of both operands, and the six products a_i b_j with
// i + j <= 2 are formed from it: the main product a0 b0 in one accumulator, the
// five small ones in another. The tensor core does not round to nearest at
// every add, so a chain over the whole reduction would drift: every kChain
// stages (a unit) the two accumulators are read and added to FP32 sums in
// registers.
//
// A reduction split over several CTAs (few tiles, long k) writes FP32 partial
// tiles that k_join adds in order: no atomics, the same bits every time.
//
// Every wait is bounded: a timeout sets a block-wide abort flag and the device
// error flag; the producer then waits (bounded) for its loads in flight, the
// MMA warp for its MMAs, and the TMEM is freed.
#include <mutex>

#include "qrb_linear.cuh"
#include "qrb_tc.cuh"
#include "qrb_tma.cuh"

namespace qrb {
namespace lin {
namespace {

constexpr int BM = 128;       // rows per CTA
constexpr int BK = 64;        // reduction values per stage: 128 bytes
constexpr int kChain = 4;     // FP32: stages per accumulator chain
constexpr int kEpiWarps = 8;
constexpr int kThreads = (kEpiWarps + 2) * 32;
constexpr int kMaxStages = 8;
constexpr uint32_t kSmemMost = 232448;  // 227 KB
constexpr uint32_t ATOM = 64 * 128;     // MN-major box: 64 reduction rows of 128 bytes

// control block at the start of shared memory
constexpr int B_FULL = 0, B_EMPTY = kMaxStages, B_ACCFULL = 2 * kMaxStages,
              B_ACCEMPTY = B_ACCFULL + 2, B_FIN = B_ACCEMPTY + 2, NBAR = B_FIN + 1;
constexpr uint32_t OFF_TMEM = NBAR * 8, OFF_ABORT = OFF_TMEM + 4, CTRL = 1024;
static_assert(OFF_ABORT + 4 <= CTRL, "control block");

template <int BN, typename T>
struct Lay {
  static constexpr int NP = sizeof(T) == 4 ? 3 : 1;  // planes
  static constexpr uint32_t A = BM * 128, B = BN * 128;
  static constexpr uint32_t STAGE = NP * (A + B);
  static constexpr int FIT = (int)((kSmemMost - CTRL - 1024) / STAGE);
  static constexpr int ST = FIT < kMaxStages ? FIT : kMaxStages;
  static constexpr uint32_t SMEM = 1024 + CTRL + ST * STAGE;  // 1024: base alignment
  static constexpr int ACC = NP == 3 ? 2 * BN : BN;  // TMEM columns per buffer
  static constexpr int TMEM = 2 * ACC;
  static_assert(ST >= 2 && TMEM <= 512 && TMEM >= 32, "stage ring and TMEM");
};

struct Args {
  int m, n;
  int mt, nt;       // tiles
  int kb;           // stages of the whole reduction
  int splits;
  int items;        // mt * nt * splits
  int group;        // tile rows that run together (operand reuse in L2)
  float* part;      // splits > 1: partial tiles
  long long part_rows, part_ld;
  Epilogue e;
  int vcodes;       // packed rows are 16-byte aligned
  int* err;
  long long limit;
  int skip_mma;     // test hook: withhold the MMAs, so that the waits run out
};

struct Item {
  int m0, n0, kb0, kb1, split;
};
template <int BN>
__device__ __forceinline__ Item item_of(const Args& a, int item) {
  const int tiles = a.mt * a.nt;
  Item it;
  it.split = item / tiles;
  const int t = item - it.split * tiles;
  const int per = a.group * a.nt;
  const int g = t / per, r = t - g * per;
  const int first = g * a.group;
  const int gm = a.mt - first < a.group ? a.mt - first : a.group;
  it.m0 = (first + r % gm) * BM;
  it.n0 = (r / gm) * BN;
  it.kb0 = (int)((long long)a.kb * it.split / a.splits);
  it.kb1 = (int)((long long)a.kb * (it.split + 1) / a.splits);
  return it;
}

constexpr uint64_t kSw128 = 2;
__device__ __forceinline__ uint64_t desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)((lbo >> 4) & 0x3FFF) << 16) |
         ((uint64_t)((sbo >> 4) & 0x3FFF) << 32) | (1ull << 46) | (kSw128 << 61);
}
// K-major: rows of 128 bytes, 8-row groups 1024 bytes apart; 16 reduction
// values are 32 bytes. MN-major: 64-value atoms ATOM apart, 8-row (reduction)
// groups 1024 bytes apart; 16 reduction rows are 2048 bytes.
template <bool MN>
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr) {
  return MN ? desc(saddr, ATOM, 1024) : desc(saddr, 16, 1024);
}
template <bool MN>
constexpr uint64_t kStep = MN ? 2048 >> 4 : 32 >> 4;

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t id,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(accumulate)
      : "memory");
}

// One operand's tile of one stage.
template <bool MN, int ROWS>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                          int mn0, int kb, int plane) {
  if constexpr (MN) {
#pragma unroll
    for (int j = 0; j < ROWS / 64; ++j)
      tma::load_3d(dst + j * ATOM, map, bar, mn0 + 64 * j, kb * BK, plane);
  } else {
    tma::load_3d(dst, map, bar, kb * BK, mn0, plane);
  }
}

template <typename T, int ACT>
__device__ __forceinline__ void act32(float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = act_fn<sizeof(T) == 4>(v[i], ACT);
}

// The epilogue of 32 consecutive columns of one row (one thread).
template <typename T, bool FWD>
__device__ __forceinline__ void finish32(float (&v)[32], int row, int col, const Args& a) {
  if (row >= a.m || col >= a.n) return;
  const int valid = a.n - col < 32 ? a.n - col : 32;
  const Epilogue& e = a.e;
  if constexpr (FWD) {
    if (e.bias != nullptr) {
      float b[32];
      load_n<T, 32>(reinterpret_cast<const T*>(e.bias) + col, e.vec, valid, b);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] += b[i];
    }
    if (e.z != nullptr)
      store_n<T, 32>(reinterpret_cast<T*>(e.z) + (int64_t)row * e.ldz + col, e.vec, valid, v);
    if (e.z_codes != nullptr) {
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        amax = fmaxf(amax, i < valid && finite_f(v[i]) ? fabsf(v[i]) : 0.f);
      const int ex = block_exponent(amax, ExpRange<T>::lo, ExpRange<T>::hi);
      const float scale = pow2f(-ex), most = ex == ExpRange<T>::hi ? 63.f : 127.f;
      int8_t* out = e.z_codes + (int64_t)row * a.n + col;
      if (a.vcodes && valid == 32) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          w[i] = pack4(code_of(v[4 * i], scale, most), code_of(v[4 * i + 1], scale, most),
                       code_of(v[4 * i + 2], scale, most), code_of(v[4 * i + 3], scale, most));
        reinterpret_cast<uint4*>(out)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<uint4*>(out)[1] = make_uint4(w[4], w[5], w[6], w[7]);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i < valid) out[i] = (int8_t)code_of(v[i], scale, most);
      }
      e.z_exps[(int64_t)row * ((a.n + kBlk - 1) / kBlk) + col / kBlk] = (int8_t)ex;
    }
    switch (e.act) {
      case QRBL_ACT_RELU: act32<T, QRBL_ACT_RELU>(v); break;
      case QRBL_ACT_GELU: act32<T, QRBL_ACT_GELU>(v); break;
      case QRBL_ACT_GELU_TANH: act32<T, QRBL_ACT_GELU_TANH>(v); break;
      case QRBL_ACT_SILU: act32<T, QRBL_ACT_SILU>(v); break;
      default: break;
    }
    if (e.residual != nullptr) {
      float r[32];
      load_n<T, 32>(reinterpret_cast<const T*>(e.residual) + (int64_t)row * e.ldr + col, e.vec,
                    valid, r);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] += r[i];
    }
  }
  store_n<T, 32>(reinterpret_cast<T*>(e.out) + (int64_t)row * e.ldo + col, e.vec, valid, v);
}

// A split product's partial tile (rows and columns padded to whole tiles).
__device__ __forceinline__ void partial32(const float (&v)[32], int row, int col, int split,
                                          const Args& a) {
  float* p = a.part + ((long long)split * a.part_rows + row) * a.part_ld + col;
#pragma unroll
  for (int i = 0; i < 32; i += 4)
    *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
}

template <int BN, bool AMN, bool BMN, typename T, bool FWD>
__global__ void __launch_bounds__(kThreads, 1)
    k_product(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
              const __grid_constant__ Args a) {
  using L = Lay<BN, T>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = tma::smem_addr(smem_raw);
  const uint32_t pad = (1024 - (raw & 1023)) & 1023;
  uint8_t* sm = smem_raw + pad;
  const uint32_t base = raw + pad;
  const uint32_t ring = base + CTRL;
  volatile int* s_abort = reinterpret_cast<volatile int*>(sm + OFF_ABORT);
  auto BAR = [&](int i) { return base + 8u * (uint32_t)i; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::ST; ++s) {
      tma::mbar_init(BAR(B_FULL + s), 1);
      tma::mbar_init(BAR(B_EMPTY + s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      tma::mbar_init(BAR(B_ACCFULL + b), 1);
      tma::mbar_init(BAR(B_ACCEMPTY + b), kEpiWarps);
    }
    tma::mbar_init(BAR(B_FIN), 1);
    tma::mbar_fence_init();
    *s_abort = 0;
  }
  if (warp == kEpiWarps + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     base + OFF_TMEM),
                 "n"(L::TMEM)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + OFF_TMEM);

  if (warp == kEpiWarps) {  // ---- loads ----
    if (lane == 0) {
      tma::prefetch_map(&map_a);
      tma::prefetch_map(&map_b);
      int u = 0;  // stages issued
      for (int item = blockIdx.x; item < a.items && *s_abort == 0; item += gridDim.x) {
        const Item it = item_of<BN>(a, item);
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          const int s = u % L::ST;
          if (u >= L::ST && !tma::mbar_wait_or_abort(BAR(B_EMPTY + s),
                                                     (uint32_t)((u / L::ST - 1) & 1), a.limit,
                                                     s_abort))
            break;
          tma::mbar_expect_tx(BAR(B_FULL + s), L::STAGE);
          const uint32_t st = ring + s * L::STAGE;
#pragma unroll
          for (int p = 0; p < L::NP; ++p)
            load_tile<AMN, BM>(st + p * L::A, &map_a, BAR(B_FULL + s), it.m0, kb, p);
#pragma unroll
          for (int p = 0; p < L::NP; ++p)
            load_tile<BMN, BN>(st + L::NP * L::A + p * L::B, &map_b, BAR(B_FULL + s), it.n0, kb,
                               p);
          ++u;
        }
      }
      if (*s_abort != 0) {  // no load may land after the block has gone
        for (int v = u > L::ST ? u - L::ST : 0; v < u; ++v)
          tma::mbar_wait_bounded(BAR(B_FULL + v % L::ST), (uint32_t)((v / L::ST) & 1), a.limit);
      }
    }
  } else if (warp == kEpiWarps + 1) {  // ---- MMAs ----
    if (lane == 0) {
      constexpr uint32_t fmt = sizeof(T) == 4 || !__is_same(T, f16) ? 1u : 0u;  // BF16 : F16
      constexpr uint32_t id = (1u << 4) | (fmt << 7) | (fmt << 10) | ((AMN ? 1u : 0u) << 15) |
                              ((BMN ? 1u : 0u) << 16) | ((uint32_t)(BN >> 3) << 17) |
                              ((uint32_t)(BM >> 4) << 24);
      int u = 0, unit = 0;
      for (int item = blockIdx.x; item < a.items && *s_abort == 0; item += gridDim.x) {
        const Item it = item_of<BN>(a, item);
        for (int kb = it.kb0; kb < it.kb1 && *s_abort == 0;) {
          const int end = L::NP == 3 && kb + kChain < it.kb1 ? kb + kChain : it.kb1;
          const int buf = unit & 1;
          if (unit >= 2 && !tma::mbar_wait_or_abort(BAR(B_ACCEMPTY + buf),
                                                    (uint32_t)((unit / 2 - 1) & 1), a.limit,
                                                    s_abort))
            break;
          tc::fence_after();
          const uint32_t d = tmem + buf * L::ACC;
          uint32_t more = 0;
          for (; kb < end; ++kb, ++u) {
            const int s = u % L::ST;
            if (!tma::mbar_wait_or_abort(BAR(B_FULL + s), (uint32_t)((u / L::ST) & 1), a.limit,
                                         s_abort))
              break;
            tc::fence_after();
            const uint32_t sa = ring + s * L::STAGE, sb = sa + L::NP * L::A;
            if (a.skip_mma == 0) {
#pragma unroll
              for (int q = 0; q < (L::NP == 3 ? 6 : 1); ++q) {
                // (0, 0) into the main accumulator, then the small products
                constexpr int pi[6] = {0, 0, 1, 1, 0, 2}, pj[6] = {0, 1, 0, 1, 2, 0};
                const uint64_t da = operand_desc<AMN>(sa + pi[q] * L::A);
                const uint64_t db = operand_desc<BMN>(sb + pj[q] * L::B);
                const uint32_t dq = q == 0 ? d : d + BN;
#pragma unroll
                for (int k = 0; k < BK / 16; ++k)
                  mma_f16(dq, da + k * kStep<AMN>, db + k * kStep<BMN>, id,
                          more | (q > 1 || k > 0 ? 1u : 0u));
              }
              more = 1;
              tc::mma_commit(BAR(B_EMPTY + s));
            }
          }
          if (*s_abort != 0) break;
          if (a.skip_mma == 0) tc::mma_commit(BAR(B_ACCFULL + buf));
          ++unit;
        }
      }
      if (*s_abort != 0) tc::drain_mmas(BAR(B_FIN));
    }
  } else {  // ---- epilogue ----
    const int quad = warp & 3, half = warp >> 2;
    constexpr int HC = BN / 2;  // columns of this warp
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    int unit = 0;
    for (int item = blockIdx.x; item < a.items; item += gridDim.x) {
      const Item it = item_of<BN>(a, item);
      const int row = it.m0 + quad * 32 + lane, col = it.n0 + half * HC;
      bool ok = true;
      if constexpr (L::NP == 1) {
        const int buf = unit & 1;
        ok = *s_abort == 0 && tma::mbar_wait_or_abort(BAR(B_ACCFULL + buf),
                                                      (uint32_t)((unit / 2) & 1), a.limit, s_abort);
        ok = __all_sync(kFull, ok);
        if (!ok) break;
        tc::fence_after();
        const uint32_t t = tmem + lanes + buf * L::ACC + half * HC;
#pragma unroll 1
        for (int c = 0; c < HC; c += 32) {
          float v[32];
          tc::tmem_ld32(t + c, v);
          if (c + 32 == HC) {  // the accumulators are read: hand the buffer back
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tma::mbar_arrive(BAR(B_ACCEMPTY + buf));
          }
          if (a.splits > 1)
            partial32(v, row, col + c, it.split, a);
          else
            finish32<T, FWD>(v, row, col + c, a);
        }
        ++unit;
      } else {
        float sum[HC / 32][32];
#pragma unroll
        for (int c = 0; c < HC / 32; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) sum[c][i] = 0.f;
        for (int kb = it.kb0; kb < it.kb1; kb += kChain, ++unit) {
          const int buf = unit & 1;
          ok = *s_abort == 0 &&
               tma::mbar_wait_or_abort(BAR(B_ACCFULL + buf), (uint32_t)((unit / 2) & 1), a.limit,
                                       s_abort);
          ok = __all_sync(kFull, ok);
          if (!ok) break;
          tc::fence_after();
          const uint32_t t = tmem + lanes + buf * L::ACC + half * HC;
#pragma unroll
          for (int c = 0; c < HC / 32; ++c) {
            float v[32], w[32];
            tc::tmem_ld32(t + c * 32, v);
            tc::tmem_ld32(t + BN + c * 32, w);
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[c][i] += v[i] + w[i];
          }
          tc::fence_before();
          __syncwarp();
          if (lane == 0) tma::mbar_arrive(BAR(B_ACCEMPTY + buf));
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < HC / 32; ++c) {
          if (a.splits > 1)
            partial32(sum[c], row, col + c * 32, it.split, a);
          else
            finish32<T, FWD>(sum[c], row, col + c * 32, a);
        }
      }
    }
  }

  __syncwarp();
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (threadIdx.x == 0 && *s_abort != 0) atomicExch(a.err, 1);
  if (warp == kEpiWarps + 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(L::TMEM)
                 : "memory");
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
bool encode16(CUtensorMap* map, const Operand& o, int planes, uint32_t box_rows) {
  PFN_cuTensorMapEncodeTiled_v12000 fn = tma::encoder();
  if (fn == nullptr) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)planes};
  const cuuint64_t row = (cuuint64_t)o.ld * 2;
  const cuuint64_t strides[2] = {row, planes > 1 ? (cuuint64_t)o.plane * 2
                                                 : row * (cuuint64_t)o.rows};
  const cuuint32_t box[3] = {64, box_rows, 1}, es[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(o.p), dims, strides, box,
            es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Device {
  int sms = 0;
  int* err = nullptr;
};
// Per-device facts, looked up once; nullptr where there is no usable device.
const Device* device_info() {
  static Device info[64];
  static std::once_flag once[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  std::call_once(once[dev], [dev] {
    int sms = 0;
    int* err = nullptr;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess &&
        device_error_ptr(&err) == QRB_OK) {
      info[dev].err = err;
      info[dev].sms = sms;
    }
  });
  return info[dev].sms > 0 ? &info[dev] : nullptr;
}

template <int BN, bool AMN, bool BMN, typename T, bool FWD>
int launch_t(const Operand& a, const Operand& b, Args& args, const Device& d, cudaStream_t s) {
  using L = Lay<BN, T>;
  static std::once_flag once[64];
  static bool ready[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return QRB_ERR_DEVICE;
  std::call_once(once[dev], [dev] {
    ready[dev] = cudaFuncSetAttribute(k_product<BN, AMN, BMN, T, FWD>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)L::SMEM) == cudaSuccess;
  });
  if (!ready[dev]) return QRB_ERR_LAUNCH;
  CUtensorMap ma, mb;
  if (!encode16(&ma, a, L::NP, AMN ? BK : BM) || !encode16(&mb, b, L::NP, BMN ? BK : BN))
    return QRB_ERR_UNSUPPORTED;
  const int grid = args.items < d.sms ? args.items : d.sms;
  k_product<BN, AMN, BMN, T, FWD><<<grid, kThreads, L::SMEM, s>>>(ma, mb, args);
  note_launches(1);
  return cudaGetLastError() == cudaSuccess ? QRB_OK : QRB_ERR_LAUNCH;
}

template <int BN, typename T>
int launch_kind(int kind, const Operand& a, const Operand& b, Args& args, const Device& d,
                cudaStream_t s) {
  switch (kind) {
    case kForward: return launch_t<BN, false, false, T, true>(a, b, args, d, s);
    case kGradIn: return launch_t<BN, false, true, T, false>(a, b, args, d, s);
    case kGradW: return launch_t<BN, true, true, T, false>(a, b, args, d, s);
  }
  return QRB_ERR_INVALID_ARG;
}

template <int BN>
int launch_bn(int dtype, int kind, const Operand& a, const Operand& b, Args& args, const Device& d,
              cudaStream_t s) {
  switch (dtype) {
    case QRBL_F32:
      if constexpr (BN <= 128) return launch_kind<BN, float>(kind, a, b, args, d, s);
      return QRB_ERR_INVALID_ARG;
    case QRBL_F16: return launch_kind<BN, f16>(kind, a, b, args, d, s);
    case QRBL_BF16: return launch_kind<BN, bf16>(kind, a, b, args, d, s);
  }
  return QRB_ERR_INVALID_ARG;
}

int64_t tiles_of(int64_t v, int64_t t) { return (v + t - 1) / t; }

}  // namespace

// The cut with the least estimated time, in SM clocks: a stage takes the larger
// of its MMAs (2 BN clocks, six times as many in FP32) and its loads (64 bytes
// a clock); a tile adds a start and an end; a split adds writing and reading
// the partial tiles and the second launch.
ProductPlan plan_product(int dtype, int kind, int64_t m, int64_t n, int64_t k) {
  (void)kind;
  ProductPlan best;
  const Device* d = device_info();
  const int64_t sms = d != nullptr ? d->sms : 148;
  const bool f32 = dtype == QRBL_F32;
  const int64_t kb = tiles_of(k, BK), mt = tiles_of(m, BM);
  double least = 0;
  const int rows = m < BM ? (int)m : BM;
  for (int bn = f32 ? 128 : 256; bn >= 64; bn /= 2) {
    const int64_t tiles = mt * tiles_of(n, bn);
    const double mma = 2.0 * bn * (f32 ? 6 : 1), load = 2.0 * (rows + bn) * (f32 ? 3 : 1);
    const double stage = mma > load ? mma : load;
    for (int s = 1; s <= 16 && s <= kb; ++s) {
      if (s > 1 && tiles * (s - 1) >= sms) break;
      const double waves = (double)tiles_of(tiles * s, sms);
      double t = waves * ((double)tiles_of(kb, s) * stage + 4.0 * bn) + 3000.0;
      if (s > 1) t += 6000.0 + 2.0 * s * (double)m * (double)n * 4.0 / 2500.0;
      if (least == 0 || t < least) {
        least = t;
        best.bn = bn;
        best.splits = s;
      }
    }
  }
  if (best.splits > 1) {
    best.part_rows = mt * BM;
    best.part_ld = tiles_of(n, best.bn) * best.bn;
    best.part_bytes = (size_t)best.splits * best.part_rows * best.part_ld * sizeof(float);
  }
  return best;
}

int launch_product(int dtype, int kind, const Operand& a, const Operand& b, int64_t m, int64_t n,
                   int64_t k, const ProductPlan& plan, float* part, const Epilogue& e,
                   cudaStream_t s) {
  const Device* d = device_info();
  if (d == nullptr) return QRB_ERR_DEVICE;
  Args args = {};
  args.m = (int)m;
  args.n = (int)n;
  const int64_t mt = tiles_of(m, BM), nt = tiles_of(n, plan.bn);
  if (mt * nt * plan.splits > 0x7fffffffLL) return QRB_ERR_UNSUPPORTED;
  args.mt = (int)mt;
  args.nt = (int)nt;
  args.kb = (int)tiles_of(k, BK);
  args.splits = plan.splits;
  args.items = (int)(mt * nt * plan.splits);
  args.group = 8;
  args.part = plan.splits > 1 ? part : nullptr;
  args.part_rows = plan.part_rows;
  args.part_ld = plan.part_ld;
  args.e = e;
  args.vcodes = aligned16(e.z_codes) && n % 16 == 0;
  args.err = d->err;
  args.limit = device_wait_limit();
  args.skip_mma = test_skip_mma() ? 1 : 0;
  int rc = QRB_ERR_INVALID_ARG;
  switch (plan.bn) {
    case 64: rc = launch_bn<64>(dtype, kind, a, b, args, *d, s); break;
    case 128: rc = launch_bn<128>(dtype, kind, a, b, args, *d, s); break;
    case 256: rc = launch_bn<256>(dtype, kind, a, b, args, *d, s); break;
  }
  if (rc != QRB_OK || plan.splits <= 1) return rc;
  return launch_join(dtype, part, plan.splits, plan.part_rows, plan.part_ld, m, n, e, s);
}

}  // namespace lin
}  // namespace qrb
