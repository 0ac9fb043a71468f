// The linear layers' matrix product: out [m, n] = epilogue(A B) on the tcgen05
// tensor cores, operands fed by TMA, for the forward product x W^T and the
// backward products dz W and dz^T x.
//
// Tiles of 128 x BN per CTA, or 256 x BN per pair of CTAs (CG = 2: one MMA over
// both SMs, each holding 128 rows of A and half of B's columns, so a CTA loads
// two thirds of the bytes), over a persistent grid of one CTA per SM. Ten warps:
// 0-7 read the accumulators (warp w: TMEM lanes 32 (w & 3) .. + 31, one half of
// the columns by w >> 2) and run the epilogue, 8 loads (one lane issues TMA
// boxes into a ring of stages), 9 issues the MMAs (one lane, of the pair's first
// CTA) and owns the TMEM. A stage holds 64 of the reduction's values for both
// operands (128-byte swizzle). An operand whose reduction runs along memory rows
// is K-major; one whose reduction runs across them (w in dz W, both operands of
// dz^T x) is MN-major, so no operand is ever transposed in memory. Two
// accumulator buffers let the epilogue of one tile run beside the MMAs of the
// next.
//
// One launch takes one product or two independent ones (dx and dW): each CTA
// or pair runs its share of the longer tiles first, then as many of the shorter
// ones as level the load (Schedule), so only one launch has a tail.
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
// MMA warp for its MMAs, and the TMEM is freed. In a pair each CTA's waits for
// the other are bounded the same way, and both reach the closing cluster
// barrier before either exits.
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
constexpr int kPitch = 33;              // words of a row in a warp's turning buffer
constexpr uint32_t ATOM = 64 * 128;     // MN-major box: 64 reduction rows of 128 bytes

// control block at the start of shared memory
constexpr int B_FULL = 0, B_EMPTY = kMaxStages, B_ACCFULL = 2 * kMaxStages,
              B_ACCEMPTY = B_ACCFULL + 2, B_FIN = B_ACCEMPTY + 2, NBAR = B_FIN + 1;
constexpr uint32_t OFF_TMEM = NBAR * 8, OFF_ABORT = OFF_TMEM + 4, CTRL = 1024;
static_assert(OFF_ABORT + 4 <= CTRL, "control block");

template <int CG, int BN, typename T>
struct Lay {
  static constexpr int NP = sizeof(T) == 4 ? 3 : 1;  // planes
  static constexpr int BROWS = BN / CG;              // B's columns of one CTA
  static constexpr uint32_t A = BM * 128, B = BROWS * 128;
  static constexpr uint32_t STAGE = NP * (A + B);
  // rows that a warp turns at a time (FP32: few, which leaves room for a stage)
  static constexpr int TROWS = NP == 3 ? 8 : 32;
  static constexpr uint32_t TURN = kEpiWarps * TROWS * kPitch * 4;
  static constexpr int FIT = (int)((kSmemMost - CTRL - 1024 - TURN) / STAGE);
  static constexpr int ST = FIT < kMaxStages ? FIT : kMaxStages;
  static constexpr uint32_t SMEM = 1024 + CTRL + ST * STAGE + TURN;  // 1024: base alignment
  static constexpr int ACC = NP == 3 ? 2 * BN : BN;  // TMEM columns per buffer
  static constexpr int TMEM = 2 * ACC;
  static_assert(ST >= 2 && TMEM <= 512 && TMEM >= 32, "stage ring and TMEM");
  static_assert(BROWS % 64 == 0, "MN-major atoms");
};

struct Problem {
  int m, n;
  int mt, nt;       // tiles
  int kb;           // stages of the whole reduction
  int splits;
  int items;        // mt * nt * splits
  int group;        // tile rows that run together (operand reuse in L2)
  int amn, bmn;     // operands are MN-major
  float* part;      // splits > 1: partial tiles
  long long part_rows, part_ld;
  Epilogue e;
};
// Which items a worker (CTA or pair) runs: of problem 0 every workers-th,
// worker by worker; then of problem 1 its count, x or (with one more of
// problem 0: worker < r) y <= x. The first (x - y) rounds have only the
// workers >= r, the later ones all of them.
struct Schedule {
  int workers;
  int q, r;         // problem 0: q items each, one more for the first r workers
  int x, y;
};
struct Args {
  Problem p[2];
  Schedule s;
  ColSum sum;       // column sums to finish beside the products (out null: none)
  int* err;
  long long limit;
  int skip_mma;     // test hook: withhold the MMAs, so that the waits run out
};

struct Item {
  int prob;         // -1: no more
  int m0, n0, kb0, kb1, split;
};
template <int CG, int BN>
__device__ __forceinline__ Item item_of(const Args& a, int worker, int step) {
  const Schedule& s = a.s;
  Item it;
  int item;
  const int own = s.q + (worker < s.r ? 1 : 0);
  if (step < own) {
    it.prob = 0;
    item = step * s.workers + worker;
  } else {
    const int j = step - own, lead = s.x - s.y, late = s.workers - s.r;
    it.prob = j < (worker < s.r ? s.y : s.x) ? 1 : -1;
    if (worker < s.r)
      item = lead * late + j * s.workers + worker;
    else
      item = j < lead ? j * late + (worker - s.r) : lead * late + (j - lead) * s.workers + worker;
    if (it.prob < 0 || item >= a.p[1].items) {
      it.prob = -1;
      return it;
    }
  }
  const Problem& p = a.p[it.prob];
  const int tiles = p.mt * p.nt;
  it.split = item / tiles;
  const int t = item - it.split * tiles;
  const int per = p.group * p.nt;
  const int g = t / per, r = t - g * per;
  const int first = g * p.group;
  const int gm = p.mt - first < p.group ? p.mt - first : p.group;
  it.m0 = (first + r % gm) * (BM * CG);
  it.n0 = (r / gm) * BN;
  it.kb0 = (int)((long long)p.kb * it.split / p.splits);
  it.kb1 = (int)((long long)p.kb * (it.split + 1) / p.splits);
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
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr, bool mn) {
  return desc(saddr, mn ? ATOM : 16, 1024);
}

template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t id,
                                        uint32_t accumulate) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(accumulate)
        : "memory");
}
// An arrival on the barrier (of both CTAs of a pair) once every MMA issued so
// far is done.
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (CG == 1)
    tc::mma_commit(bar);
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(bar),
        "h"((unsigned short)3)
        : "memory");
}
template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t where, uint32_t columns) {
  if constexpr (CG == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t columns) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns)
                 : "memory");
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns)
                 : "memory");
}
// Every thread of the block, or of both blocks of a pair.
template <int CG>
__device__ __forceinline__ void sync_all() {
  if constexpr (CG == 1) {
    __syncthreads();
  } else {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}
// The same shared-memory address in the pair's first CTA.
__device__ __forceinline__ uint32_t in_first_cta(uint32_t addr) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
// Bounded: false on a timeout (which sets *abort) or once *abort is set.
// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t pred;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(pred));
  return pred != 0;
}
// Block-scope acquire, also for what the other CTA of a pair announces: all that
// passes between them is TMA and TMEM traffic, ordered by the barriers
// themselves; a cluster-scope release or acquire would wait for this CTA's
// global stores and drop its L1 (measured: 25,000 clocks per 128 x 256 tile
// with GELU and packing, against 9,000 without).
__device__ __forceinline__ bool wait_or_abort(uint32_t bar, uint32_t parity, long long limit,
                                              volatile int* abort) {
  if (tma::mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  while (!tma::mbar_try(bar, parity)) {
    if (*abort != 0) return false;
    if (clock64() - t0 > limit) {
      *abort = 1;
      return false;
    }
  }
  return true;
}

// The same for a whole warp: every lane gets the same answer.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, long long limit,
                                          volatile int* abort) {
  return __all_sync(kFull, wait_or_abort(bar, parity, limit, abort));
}

template <int CG>
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x,
                                         int y, int z) {
  if constexpr (CG == 1)
    tma::load_3d(dst, map, bar, x, y, z);
  else  // into this CTA's memory, announced on the first CTA's barrier
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        ".cta_group::2 [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
// One operand's tile of one stage.
template <int CG, int ROWS>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, bool mn,
                                          uint32_t bar, int mn0, int kb, int plane) {
  if (mn) {
#pragma unroll
    for (int j = 0; j < ROWS / 64; ++j)
      load_box<CG>(dst + j * ATOM, map, bar, mn0 + 64 * j, kb * BK, plane);
  } else {
    load_box<CG>(dst, map, bar, kb * BK, mn0, plane);
  }
}

// A warp's block of 32 columns of up to eight rows, packed (lane = column).
template <typename T>
__device__ __forceinline__ void pack_rows(const float (&p)[8], int64_t row, int left, bool live,
                                          int col, const Problem& a) {
  constexpr int lo = ExpRange<T>::lo, hi = ExpRange<T>::hi;
  const int lane = threadIdx.x & 31;
  const Epilogue& e = a.e;
  float amax[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) amax[k] = live && finite_f(p[k]) ? fabsf(p[k]) : 0.f;
#pragma unroll
  for (int o = 1; o < 32; o *= 2)
#pragma unroll
    for (int k = 0; k < 8; ++k)
      amax[k] = fmaxf(amax[k], __shfl_xor_sync(kFull, amax[k], o));
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int ex = block_exponent(amax[k], lo, hi);
    const float one[4] = {p[k], 0.f, 0.f, 0.f};
    uint32_t w[1];
    encode(one, ex, finite_f(p[k]) && ex < hi, ex == hi ? 63.f : 127.f, w);
    if (live && k < left) {
      e.z_codes[(row + k) * a.n + col + lane] = (int8_t)(w[0] & 255u);
      if (lane == 0)
        e.z_exps[(row + k) * ((a.n + kBlk - 1) / kBlk) + col / kBlk] = (int8_t)ex;
    }
  }
}

// The epilogue of a warp's 32 x 32 block, rows from row0, columns from col, as
// lane = column: the block (v: lane = row) is turned through shared memory, TROWS
// rows at a time, so that every access is consecutive elements of one row,
// whatever their alignment: blocks that are cut by the matrix's edge or whose
// rows are not 16-byte aligned.
template <typename T, bool FWD, int TROWS>
__device__ __forceinline__ void finish_turned(const float (&v)[32], int row0, int col,
                                              const Problem& a, float* turn) {
  if (row0 >= a.m || col >= a.n) return;
  const int lane = threadIdx.x & 31;
  const int rows = a.m - row0 < 32 ? a.m - row0 : 32;
  const bool live = col + lane < a.n;
  const Epilogue& e = a.e;
  float bias = 0.f;
  if constexpr (FWD) {
    if (e.bias != nullptr && live) bias = to_f<T>(reinterpret_cast<const T*>(e.bias)[col + lane]);
  }
#pragma unroll 1
  for (int base = 0; base < rows; base += TROWS) {
    __syncwarp();
    if (lane >= base && lane < base + TROWS) {
#pragma unroll
      for (int i = 0; i < 32; ++i) turn[(lane - base) * kPitch + i] = v[i];
    }
    __syncwarp();
    const int most = rows - base < TROWS ? rows - base : TROWS;
#pragma unroll 1
    for (int r0 = 0; r0 < most; r0 += 8) {
      const int64_t row0g = row0 + base + r0;
      const int left = most - r0;
      // eight rows' values and residuals together, then eight rows' results
      float p[8], q[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        p[k] = k < left ? turn[(r0 + k) * kPitch + lane] : 0.f;
        q[k] = 0.f;
      }
      if constexpr (FWD) {
        if (e.residual != nullptr) {
          const T* s = reinterpret_cast<const T*>(e.residual) + row0g * e.ldr + col + lane;
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (live && k < left) q[k] = to_f<T>(s[k * e.ldr]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) p[k] += bias;
        if (e.z != nullptr && live) {
          T* z = reinterpret_cast<T*>(e.z) + row0g * e.ldz + col + lane;
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < left) z[k * e.ldz] = from_f<T>(p[k]);
        }
        if (e.z_codes != nullptr) pack_rows<T>(p, row0g, left, live, col, a);
        act_by(p, e.act);
#pragma unroll
        for (int k = 0; k < 8; ++k) p[k] += q[k];
      }
      if (live) {
        T* out = reinterpret_cast<T*>(e.out) + row0g * e.ldo + col + lane;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < left) out[k * e.ldo] = from_f<T>(p[k]);
      }
    }
  }
}

// The same for a whole block of 16-byte aligned rows, as lane = row: each lane's
// 32 columns are whole sectors. 16-bit types: the bias and residual were loaded
// before the accumulators were ready.
template <typename T, bool FWD>
__device__ __forceinline__ void finish32(float (&v)[32], int row, int col, const Problem& a,
                                         const Raw32<T>& bias, const Raw32<T>& res) {
  const Epilogue& e = a.e;
  if constexpr (FWD) {
    if (e.bias != nullptr) add_raw32<T>(v, bias);
    Raw32<T> late;  // (FP32: no registers to hold it earlier)
    if constexpr (sizeof(T) == 4) {
      if (e.residual != nullptr)
        late = load_raw32<T>(reinterpret_cast<const T*>(e.residual) + (int64_t)row * e.ldr + col);
    }
    if (e.z != nullptr)
      store_n<T, 32>(reinterpret_cast<T*>(e.z) + (int64_t)row * e.ldz + col, true, 32, v);
    if (e.z_codes != nullptr) {
      constexpr int lo = ExpRange<T>::lo, hi = ExpRange<T>::hi;
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < 32; ++i) amax = max_abs_nan(amax, v[i]);
      const bool fine = finite_f(amax);
      if (!fine) amax = finite_amax(v);
      const int ex = block_exponent(amax, lo, hi);
      uint32_t w[8];
      encode(v, ex, fine && ex < hi, ex == hi ? 63.f : 127.f, w);
      uint4* out = reinterpret_cast<uint4*>(e.z_codes + (int64_t)row * a.n + col);
      out[0] = make_uint4(w[0], w[1], w[2], w[3]);
      out[1] = make_uint4(w[4], w[5], w[6], w[7]);
      e.z_exps[(int64_t)row * ((a.n + kBlk - 1) / kBlk) + col / kBlk] = (int8_t)ex;
    }
    act_by(v, e.act);
    if (e.residual != nullptr) add_raw32<T>(v, sizeof(T) == 4 ? late : res);
  }
  store_n<T, 32>(reinterpret_cast<T*>(e.out) + (int64_t)row * e.ldo + col, true, 32, v);
}

// A split product's partial tile (rows and columns padded to whole tiles).
__device__ __forceinline__ void partial32(const float (&v)[32], int row, int col, int split,
                                          const Problem& a) {
  float* p = a.part + ((long long)split * a.part_rows + row) * a.part_ld + col;
#pragma unroll
  for (int i = 0; i < 32; i += 4)
    *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
}

template <int CG, int BN, typename T, bool FWD>
__global__ void __launch_bounds__(kThreads, 1)
    k_product(const __grid_constant__ CUtensorMap map_a0, const __grid_constant__ CUtensorMap map_b0,
              const __grid_constant__ CUtensorMap map_a1, const __grid_constant__ CUtensorMap map_b1,
              const __grid_constant__ Args a) {
  using L = Lay<CG, BN, T>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = tma::smem_addr(smem_raw);
  const uint32_t pad = (1024 - (raw & 1023)) & 1023;
  uint8_t* sm = smem_raw + pad;
  const uint32_t base = raw + pad;
  const uint32_t ring = base + CTRL;
  volatile int* s_abort = reinterpret_cast<volatile int*>(sm + OFF_ABORT);
  auto BAR = [&](int i) { return base + 8u * (uint32_t)i; };
  // (the shuffle tells the compiler that a warp's lanes agree: the loading and
  // the issuing warp run whole, in uniform registers, and one elected lane
  // issues; with a lane's own registers each tcgen05.mma took 120 clocks)
  const int warp = __shfl_sync(kFull, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int worker = (int)blockIdx.x / CG, rank = (int)blockIdx.x % CG;

  if (warp == kEpiWarps && lane == 0) {
    tma::prefetch_map(&map_a0);
    tma::prefetch_map(&map_b0);
    if (a.p[1].items > 0) {
      tma::prefetch_map(&map_a1);
      tma::prefetch_map(&map_b1);
    }
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < L::ST; ++s) {
      tma::mbar_init(BAR(B_FULL + s), 1);
      tma::mbar_init(BAR(B_EMPTY + s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      tma::mbar_init(BAR(B_ACCFULL + b), 1);
      tma::mbar_init(BAR(B_ACCEMPTY + b), CG * kEpiWarps);
    }
    tma::mbar_init(BAR(B_FIN), 1);
    tma::mbar_fence_init();
    *s_abort = 0;
  }
  if (warp == kEpiWarps + 1) tmem_alloc<CG>(base + OFF_TMEM, L::TMEM);
  tc::fence_before();
  __syncthreads();
  if constexpr (CG == 2) sync_all<CG>();
  tc::fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + OFF_TMEM);

  if (warp == kEpiWarps) {  // ---- loads ----
    int u = 0;  // stages issued
    bool live = true;
    for (int step = 0; live; ++step) {
      const Item it = item_of<CG, BN>(a, worker, step);
      if (it.prob < 0) break;
      const CUtensorMap* ma = it.prob == 0 ? &map_a0 : &map_a1;
      const CUtensorMap* mb = it.prob == 0 ? &map_b0 : &map_b1;
      const bool amn = a.p[it.prob].amn != 0, bmn = a.p[it.prob].bmn != 0;
      const int am = it.m0 + rank * BM, bn = it.n0 + rank * L::BROWS;
      for (int kb = it.kb0; kb < it.kb1; ++kb) {
        const int s = u % L::ST;
        if (u >= L::ST)
          live = warp_wait(BAR(B_EMPTY + s), (uint32_t)((u / L::ST - 1) & 1), a.limit, s_abort);
        if (!live) break;
        const uint32_t bar = CG == 1 ? BAR(B_FULL + s) : in_first_cta(BAR(B_FULL + s));
        const uint32_t st = ring + s * L::STAGE;
        if (elect_one()) {
          if (rank == 0) tma::mbar_expect_tx(BAR(B_FULL + s), CG * L::STAGE);
#pragma unroll
          for (int p = 0; p < L::NP; ++p)
            load_tile<CG, BM>(st + p * L::A, ma, amn, bar, am, kb, p);
#pragma unroll
          for (int p = 0; p < L::NP; ++p)
            load_tile<CG, L::BROWS>(st + L::NP * L::A + p * L::B, mb, bmn, bar, bn, kb, p);
        }
        __syncwarp();
        ++u;
      }
    }
    if (__any_sync(kFull, *s_abort != 0)) {  // no load may land after the block has gone
      if constexpr (CG == 1) {
        for (int v = u > L::ST ? u - L::ST : 0; v < u; ++v)
          tma::mbar_wait_bounded(BAR(B_FULL + v % L::ST), (uint32_t)((v / L::ST) & 1), a.limit);
      } else {  // announced on one CTA's barrier: a fixed time, far above any load's
        const long long t0 = clock64();
        while (clock64() - t0 < 4000000LL) {
        }
      }
    }
  } else if (warp == kEpiWarps + 1) {  // ---- MMAs ----
    if (rank == 0) {
      constexpr uint32_t fmt = __is_same(T, f16) ? 0u : 1u;  // F16 : BF16
      int u = 0, unit = 0;
      bool live = true;
      for (int step = 0; live; ++step) {
        const Item it = item_of<CG, BN>(a, worker, step);
        if (it.prob < 0) break;
        const bool amn = a.p[it.prob].amn != 0, bmn = a.p[it.prob].bmn != 0;
        const uint32_t id = (1u << 4) | (fmt << 7) | (fmt << 10) | ((amn ? 1u : 0u) << 15) |
                            ((bmn ? 1u : 0u) << 16) | ((uint32_t)(BN >> 3) << 17) |
                            ((uint32_t)((BM * CG) >> 4) << 24);
        const uint64_t ka = amn ? 2048 >> 4 : 32 >> 4, kbs = bmn ? 2048 >> 4 : 32 >> 4;
        const uint64_t da0 = operand_desc(ring, amn);
        const uint64_t db0 = operand_desc(ring + L::NP * L::A, bmn);
        for (int kb = it.kb0; live && kb < it.kb1;) {
          const int end = L::NP == 3 && kb + kChain < it.kb1 ? kb + kChain : it.kb1;
          const int buf = unit & 1;
          if (unit >= 2)
            live = warp_wait(BAR(B_ACCEMPTY + buf), (uint32_t)((unit / 2 - 1) & 1), a.limit,
                             s_abort);
          tc::fence_after();
          const uint32_t d = tmem + buf * L::ACC;
          uint32_t more = 0;
          for (; live && kb < end; ++kb, ++u) {
            const int s = u % L::ST;
            live = warp_wait(BAR(B_FULL + s), (uint32_t)((u / L::ST) & 1), a.limit, s_abort);
            if (!live) break;
            tc::fence_after();
            const uint64_t at = (uint64_t)(s * (int)(L::STAGE >> 4));
            if (a.skip_mma == 0 && elect_one()) {
#pragma unroll
              for (int q = 0; q < (L::NP == 3 ? 6 : 1); ++q) {
                // (0, 0) into the main accumulator, then the small products
                constexpr int pi[6] = {0, 0, 1, 1, 0, 2}, pj[6] = {0, 1, 0, 1, 2, 0};
                const uint64_t da = da0 + at + (uint64_t)(pi[q] * (L::A >> 4));
                const uint64_t db = db0 + at + (uint64_t)(pj[q] * (L::B >> 4));
                const uint32_t dq = q == 0 ? d : d + BN;
#pragma unroll
                for (int k = 0; k < BK / 16; ++k)
                  mma_f16<CG>(dq, da + k * ka, db + k * kbs, id,
                              more | (q > 1 || k > 0 ? 1u : 0u));
              }
              commit<CG>(BAR(B_EMPTY + s));
            }
            __syncwarp();
            more = 1;
          }
          if (!live) break;
          if (a.skip_mma == 0 && elect_one()) commit<CG>(BAR(B_ACCFULL + buf));
          __syncwarp();
          ++unit;
        }
      }
      if (__any_sync(kFull, *s_abort != 0)) {  // no MMA may run on into freed TMEM (a pair: fixed time as above)
        if constexpr (CG == 1) {
          if (elect_one()) tc::drain_mmas(BAR(B_FIN));
        } else {
          const long long t0 = clock64();
          while (clock64() - t0 < 4000000LL) {
          }
        }
      }
    }
  } else {  // ---- epilogue ----
    const int quad = warp & 3, half = warp >> 2;
    constexpr int HC = BN / 2;  // columns of this warp
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    float* turn = reinterpret_cast<float*>(sm + CTRL + L::ST * L::STAGE) + warp * L::TROWS * kPitch;
    int unit = 0;
    auto hand_back = [&](int buf) {  // the accumulators are read
      tc::fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 1)
          tma::mbar_arrive(BAR(B_ACCEMPTY + buf));
        else
          asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(
                           in_first_cta(BAR(B_ACCEMPTY + buf)))
                       : "memory");
      }
    };
    if constexpr (!FWD) {
      if (a.sum.out != nullptr)
        column_sum<T>(a.sum, (int64_t)blockIdx.x * (kEpiWarps * 32) + threadIdx.x,
                      (int64_t)gridDim.x * (kEpiWarps * 32));
    }
    for (int step = 0;; ++step) {
      const Item it = item_of<CG, BN>(a, worker, step);
      if (it.prob < 0) break;
      const Problem& p = a.p[FWD ? 0 : it.prob];
      const int row0 = it.m0 + rank * BM + quad * 32, col = it.n0 + half * HC;
      bool ok = true;
      if constexpr (L::NP == 1) {
        // the bias and residual of a block are loaded while the accumulators
        // (first block) or the block before are worked on
        Raw32<T> bias, res;
        const Epilogue& e = p.e;
        const int row = row0 + lane;
        // whole aligned blocks; all lanes agree except on rows beyond m
        auto whole = [&](int c) { return e.vec != 0 && c + 32 <= p.n; };
        auto ahead = [&](int c) { return FWD && p.splits == 1 && whole(c) && row < p.m; };
        auto load_bias = [&](int c) {
          if (e.bias != nullptr) bias = load_raw32<T>(reinterpret_cast<const T*>(e.bias) + c);
        };
        auto load_res = [&](int c) {
          if (e.residual != nullptr)
            res = load_raw32<T>(reinterpret_cast<const T*>(e.residual) +
                                (int64_t)row * e.ldr + c);
        };
        if (ahead(col)) {
          load_bias(col);
          load_res(col);
        }
        const int buf = unit & 1;
        ok = warp_wait(BAR(B_ACCFULL + buf), (uint32_t)((unit / 2) & 1), a.limit, s_abort);
        if (!ok) break;
        tc::fence_after();
        const uint32_t t = tmem + lanes + buf * L::ACC + half * HC;
#pragma unroll 1
        for (int c = 0; c < HC; c += 32) {
          float v[32];
          tc::tmem_ld32(t + c, v);
          if (c + 32 == HC) hand_back(buf);
          if (p.splits > 1) {
            partial32(v, row, col + c, it.split, p);
          } else if (whole(col + c)) {
            if (row < p.m) finish32<T, FWD>(v, row, col + c, p, bias, res);
          } else {
            finish_turned<T, FWD, L::TROWS>(v, row0, col + c, p, turn);
          }
          if (c + 32 < HC && ahead(col + c + 32)) {
            load_bias(col + c + 32);
            load_res(col + c + 32);
          }
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
          ok = warp_wait(BAR(B_ACCFULL + buf), (uint32_t)((unit / 2) & 1), a.limit, s_abort);
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
          hand_back(buf);
        }
        if (!ok) break;
#pragma unroll 1
        for (int c = 0; c < HC / 32; ++c) {
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = HC == 32 || c == 0 ? sum[0][i] : sum[HC / 32 - 1][i];
          const int at = col + c * 32;
          if (p.splits > 1) {
            partial32(v, row0 + lane, at, it.split, p);
          } else if (p.e.vec != 0 && at + 32 <= p.n) {
            if (row0 + lane < p.m) {
              Raw32<T> bias;
              if (FWD && p.e.bias != nullptr)
                bias = load_raw32<T>(reinterpret_cast<const T*>(p.e.bias) + at);
              finish32<T, FWD>(v, row0 + lane, at, p, bias, bias);
            }
          } else {
            finish_turned<T, FWD, L::TROWS>(v, row0, at, p, turn);
          }
        }
      }
    }
  }

  __syncwarp();
  tc::fence_before();
  __syncthreads();
  if constexpr (CG == 2) sync_all<CG>();
  tc::fence_after();
  if (threadIdx.x == 0 && *s_abort != 0) atomicExch(a.err, 1);
  if (warp == kEpiWarps + 1) tmem_free<CG>(tmem, L::TMEM);
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

// The kernel for both (or one of the) products, or for a forward product.
template <int CG, int BN, typename T, bool FWD>
int launch_t(const Product* const* q, int count, Args& args, const Device& d, cudaStream_t s) {
  using L = Lay<CG, BN, T>;
  static std::once_flag once[64];
  static bool ready[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return QRB_ERR_DEVICE;
  std::call_once(once[dev], [dev] {
    ready[dev] = cudaFuncSetAttribute(k_product<CG, BN, T, FWD>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)L::SMEM) == cudaSuccess;
  });
  if (!ready[dev]) return QRB_ERR_LAUNCH;
  CUtensorMap ma[2], mb[2];
  for (int i = 0; i < count; ++i) {
    if (!encode16(&ma[i], q[i]->a, L::NP, args.p[i].amn ? BK : BM) ||
        !encode16(&mb[i], q[i]->b, L::NP, args.p[i].bmn ? BK : L::BROWS))
      return QRB_ERR_UNSUPPORTED;
  }
  if (count == 1) {
    ma[1] = ma[0];
    mb[1] = mb[0];
  }
  if constexpr (CG == 1) {
    k_product<CG, BN, T, FWD><<<args.s.workers, kThreads, L::SMEM, s>>>(ma[0], mb[0], ma[1], mb[1],
                                                                        args);
  } else {
    cudaLaunchConfig_t lc = {};
    cudaLaunchAttribute la[1];
    la[0].id = cudaLaunchAttributeClusterDimension;
    la[0].val.clusterDim.x = 2;
    la[0].val.clusterDim.y = 1;
    la[0].val.clusterDim.z = 1;
    lc.gridDim = dim3(2 * (unsigned)args.s.workers);
    lc.blockDim = dim3(kThreads);
    lc.dynamicSmemBytes = L::SMEM;
    lc.stream = s;
    lc.attrs = la;
    lc.numAttrs = 1;
    if (cudaLaunchKernelEx(&lc, k_product<CG, BN, T, FWD>, ma[0], mb[0], ma[1], mb[1], args) !=
        cudaSuccess) {
      (void)cudaGetLastError();
      return QRB_ERR_LAUNCH;
    }
  }
  (void)d;
  note_launches(1);
  return cudaGetLastError() == cudaSuccess ? QRB_OK : QRB_ERR_LAUNCH;
}

template <int CG, int BN, typename T>
int launch_dir(bool fwd, const Product* const* q, int count, Args& args, const Device& d,
               cudaStream_t s) {
  return fwd ? launch_t<CG, BN, T, true>(q, count, args, d, s)
             : launch_t<CG, BN, T, false>(q, count, args, d, s);
}

template <typename T>
int launch_type(int cg, int bn, bool fwd, const Product* const* q, int count, Args& args,
                const Device& d, cudaStream_t s) {
  if (cg == 1 && bn == 64) return launch_dir<1, 64, T>(fwd, q, count, args, d, s);
  if (cg == 1 && bn == 128) return launch_dir<1, 128, T>(fwd, q, count, args, d, s);
  if (cg == 2 && bn == 128) return launch_dir<2, 128, T>(fwd, q, count, args, d, s);
  if constexpr (sizeof(T) == 2) {
    if (cg == 2 && bn == 256) return launch_dir<2, 256, T>(fwd, q, count, args, d, s);
  }
  return QRB_ERR_INVALID_ARG;
}

int64_t tiles_of(int64_t v, int64_t t) { return (v + t - 1) / t; }

// The cuts of the kernel: CTAs per tile and tile width.
struct Cut {
  int cg, bn;
};
constexpr Cut kCuts16[] = {{2, 256}, {2, 128}, {1, 128}, {1, 64}};
constexpr Cut kCuts32[] = {{2, 128}, {1, 128}, {1, 64}};

// Estimated SM clocks of one stage of one CTA: the larger of its MMAs (2 BN
// clocks, shared by a pair; six times as many in FP32) and its loads (64 bytes
// a clock; rows beyond a short m are not read).
double stage_clocks(bool f32, Cut c, int64_t m) {
  const double rows = m < BM ? (double)m : BM;
  const double mma = 2.0 * c.bn * (f32 ? 6 : 1);
  const double load = 2.0 * (rows + c.bn / c.cg) * (f32 ? 3 : 1);
  return mma > load ? mma : load;
}
double item_clocks(bool f32, Cut c, int64_t m, int64_t kb) {
  return (double)kb * stage_clocks(f32, c, m) + 500.0;
}

// The schedule of `items[0]` longer and `items[1]` shorter items over `most`
// workers, and its length in the items' clocks.
double make_schedule(const int64_t* items, const double* clocks, int64_t most, Schedule* out) {
  const int64_t all = items[0] + items[1];
  const int64_t g = all < most ? all : most;
  Schedule s = {};
  s.workers = (int)g;
  s.q = (int)(items[0] / g);
  s.r = (int)(items[0] % g);
  double length = (s.q + (s.r > 0 ? 1 : 0)) * clocks[0];
  if (items[1] > 0) {
    // the least x whose level holds every short item; y by what the one more
    // long item leaves of it
    const double ratio = clocks[0] / clocks[1];
    int64_t x = (items[1] - 1) / g;
    for (;; ++x) {
      int64_t y = x - (int64_t)(ratio + 0.5);
      if (y < 0) y = 0;
      if (s.r == 0) y = x;
      if (x * (g - s.r) + y * s.r >= items[1]) {
        s.x = (int)x;
        s.y = (int)y;
        break;
      }
    }
    const double late = s.q * clocks[0] + s.x * clocks[1];
    const double early = s.r > 0 ? (s.q + 1) * clocks[0] + s.y * clocks[1] : 0;
    length = late > early ? late : early;
  }
  *out = s;
  return length;
}

Problem problem_of(int kind, int64_t m, int64_t n, int64_t k, Cut c, int splits) {
  Problem p = {};
  p.m = (int)m;
  p.n = (int)n;
  p.mt = (int)tiles_of(m, BM * c.cg);
  p.nt = (int)tiles_of(n, c.bn);
  p.kb = (int)tiles_of(k, BK);
  p.splits = splits;
  p.items = p.mt * p.nt * splits;
  p.group = c.cg == 2 ? 8 : 16;
  p.amn = kind == kGradW;
  p.bmn = kind != kForward;
  return p;
}

}  // namespace

// The cut with the least estimated time, in SM clocks: the schedule's length, a
// start, and for each split product the writing and reading of its partial
// tiles and its second launch.
static ProductPlan search_plan(int dtype, const ProductSize* sizes, int count) {
  ProductPlan best;
  const Device* d = device_info();
  const int64_t sms = d != nullptr ? d->sms : 148;
  const bool f32 = dtype == QRBL_F32;
  double least = -1;
  const Cut* cuts = f32 ? kCuts32 : kCuts16;
  const int ncuts = f32 ? 3 : 4;
  for (int ci = 0; ci < ncuts; ++ci) {
    const Cut c = cuts[ci];
    const int64_t workers = sms / c.cg;
    int64_t tiles[2] = {0, 0}, kb[2] = {1, 1};
    for (int i = 0; i < count; ++i) {
      tiles[i] = tiles_of(sizes[i].m, BM * c.cg) * tiles_of(sizes[i].n, c.bn);
      kb[i] = tiles_of(sizes[i].k, BK);
      if (tiles[i] > (1 << 26)) return best;  // (refused: 26 bits of tiles)
    }
    for (int s0 = 1; s0 <= 16 && s0 <= kb[0]; ++s0) {
      if (s0 > 1 && tiles[0] * (s0 - 1) >= workers) break;
      for (int s1 = 1; s1 <= (count > 1 ? 16 : 1) && s1 <= kb[1]; ++s1) {
        if (s1 > 1 && tiles[1] * (s1 - 1) >= workers) break;
        const int sp[2] = {s0, s1};
        double len[2] = {0, 0}, t = 3000.0;
        int64_t items[2] = {0, 0};
        for (int i = 0; i < count; ++i) {
          items[i] = tiles[i] * sp[i];
          len[i] = item_clocks(f32, c, sizes[i].m, tiles_of(kb[i], sp[i]));
          if (sp[i] > 1)
            t += 6000.0 + 2.0 * sp[i] * (double)sizes[i].m * (double)sizes[i].n * 4.0 / 2500.0;
        }
        const bool swap = count > 1 && len[1] > len[0];
        const int64_t it[2] = {items[swap ? 1 : 0], count > 1 ? items[swap ? 0 : 1] : 0};
        const double cl[2] = {len[swap ? 1 : 0], count > 1 ? len[swap ? 0 : 1] : 1.0};
        Schedule sc;
        t += make_schedule(it, cl, workers, &sc);
        if (least < 0 || t < least) {
          least = t;
          best.cg = c.cg;
          best.bn = c.bn;
          best.first = swap ? 1 : 0;
          best.splits[0] = s0;
          best.splits[1] = s1;
        }
      }
    }
  }
  for (int i = 0; i < count; ++i) {
    if (best.splits[i] <= 1) continue;
    best.part_rows[i] = tiles_of(sizes[i].m, BM * best.cg) * BM * best.cg;
    best.part_ld[i] = tiles_of(sizes[i].n, best.bn) * best.bn;
    best.part_bytes[i] =
        (size_t)best.splits[i] * best.part_rows[i] * best.part_ld[i] * sizeof(float);
  }
  best.ok = least >= 0;
  return best;
}

// A pure function of its arguments and the device's SM count; the last few
// results are kept per thread, since a call asks twice (its workspace, its
// launch) and a model's layers repeat.
ProductPlan plan_products(int dtype, const ProductSize* sizes, int count) {
  struct Entry {
    int dtype = -1, count = 0, sms = 0;
    ProductSize z[2];
    ProductPlan plan;
  };
  static thread_local Entry kept[64];
  const Device* d = device_info();
  const int sms = d != nullptr ? d->sms : 0;
  uint64_t h = (uint64_t)dtype * 3 + (uint64_t)count;
  for (int i = 0; i < count; ++i)
    h = (h * 1000003u + (uint64_t)sizes[i].m) * 1000003u + (uint64_t)sizes[i].n * 8191u +
        (uint64_t)sizes[i].k;
  Entry& e = kept[(h ^ (h >> 17) ^ (h >> 31)) % 64];
  bool same = e.dtype == dtype && e.count == count && e.sms == sms;
  for (int i = 0; i < count && same; ++i)
    same = e.z[i].m == sizes[i].m && e.z[i].n == sizes[i].n && e.z[i].k == sizes[i].k;
  if (!same) {
    e.dtype = dtype;
    e.count = count;
    e.sms = sms;
    for (int i = 0; i < count; ++i) e.z[i] = sizes[i];
    e.plan = search_plan(dtype, sizes, count);
  }
  return e.plan;
}

int launch_products(int dtype, const Product* products, int count, const ProductPlan& plan,
                    const ColSum* sum, cudaStream_t s) {
  const Device* d = device_info();
  if (d == nullptr) return QRB_ERR_DEVICE;
  if (!plan.ok) return QRB_ERR_UNSUPPORTED;
  const Cut c = {plan.cg, plan.bn};
  const bool f32 = dtype == QRBL_F32;
  Args args = {};
  const Product* q[2] = {nullptr, nullptr};
  int64_t items[2] = {0, 0};
  double clocks[2] = {1.0, 1.0};
  for (int j = 0; j < count; ++j) {
    const int i = count > 1 ? (j == 0 ? plan.first : 1 - plan.first) : 0;  // longer items first
    q[j] = &products[i];
    const ProductSize& z = products[i].size;
    args.p[j] = problem_of(products[i].kind, z.m, z.n, z.k, c, plan.splits[i]);
    args.p[j].part = plan.splits[i] > 1 ? products[i].part : nullptr;
    args.p[j].part_rows = plan.part_rows[i];
    args.p[j].part_ld = plan.part_ld[i];
    args.p[j].e = products[i].e;
    if (products[i].e.z_codes != nullptr)  // packed rows 16-byte aligned too
      args.p[j].e.vec &= aligned16(products[i].e.z_codes) && z.n % 16 == 0;
    items[j] = args.p[j].items;
    clocks[j] = item_clocks(f32, c, z.m, tiles_of(args.p[j].kb, plan.splits[i]));
  }
  make_schedule(items, clocks, d->sms / c.cg, &args.s);
  if (sum != nullptr) args.sum = *sum;
  args.err = d->err;
  args.limit = device_wait_limit();
  args.skip_mma = test_skip_mma() ? 1 : 0;
  const bool fwd = products[0].kind == kForward;
  int rc = QRB_ERR_INVALID_ARG;
  switch (dtype) {
    case QRBL_F32: rc = launch_type<float>(c.cg, c.bn, fwd, q, count, args, *d, s); break;
    case QRBL_F16: rc = launch_type<f16>(c.cg, c.bn, fwd, q, count, args, *d, s); break;
    case QRBL_BF16: rc = launch_type<bf16>(c.cg, c.bn, fwd, q, count, args, *d, s); break;
  }
  for (int i = 0; i < count && rc == QRB_OK; ++i)
    if (plan.splits[i] > 1)
      rc = launch_join(dtype, products[i].part, plan.splits[i], plan.part_rows[i],
                       plan.part_ld[i], products[i].size.m, products[i].size.n, products[i].e, s);
  return rc;
}

}  // namespace lin
}  // namespace qrb
