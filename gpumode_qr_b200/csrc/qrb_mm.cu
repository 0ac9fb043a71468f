// The linear layers' matrix product: out [m, n] = epilogue(A B) on the tcgen05
// tensor cores, operands fed by TMA, for the forward product x W^T and the
// backward products dz W and dz^T x.
//
// Tiles of 128 x BN per CTA, or 256 x BN per pair of CTAs (CG = 2: one MMA over
// both SMs, each holding 128 rows of A and half of B's columns, so a CTA loads
// two thirds of the bytes), over a persistent grid of one CTA per SM. 16 warps (8
// for 64 columns) read the accumulators and run the epilogue (warp w: TMEM lanes
// 32 (w & 3) .. + 31, a quarter of the columns by w >> 2: four warps per scheduler,
// since one's loads, waits and special functions leave most of its issue slots
// empty), one loads (an elected lane issues TMA boxes into a ring of stages), one
// issues the MMAs (of the pair's first CTA) and owns the TMEM. A stage holds 64 of
// the reduction's values for both operands (128-byte swizzle). An operand whose
// reduction runs along memory rows is K-major; one whose reduction runs across them
// (w in dz W, both operands of dz^T x) is MN-major, so no operand is ever
// transposed in memory. Two accumulator buffers let the epilogue of one tile run
// beside the MMAs of the next.
//
// One launch takes one product or two independent ones (dx and dW): each CTA
// or pair runs its share of the longer tiles first, then as many of the shorter
// ones as level the load (Schedule), so only one launch has a tail.
//
// FP32 operands come as three BF16 planes a0 + a1 + a2 (24 bits). A stage
// holds all three planes of both operands, and the six products a_i b_j with
// i + j <= 2 are formed from it: the main product a0 b0 in one accumulator, the
// five small ones in another. The tensor core does not round to nearest at
// every add, so a chain over the whole reduction would drift: every CHAIN
// stages (a unit) the two accumulators are read and added to FP32 sums in
// registers. A 16-bit forward product whose z is kept in 8 bits sums its chains
// the same way (SUM): a code near a border shows the drift (z's relative error
// against exact codes 3.2e-4 -> 1.0e-4 at k = 4096, an FP32 product's 1.2e-4).
// Other 16-bit results are rounded above the drift of a chain of 8192 values:
// each 16 of them cost at most 2^-23 of the sum, so a chain 2^-14, an eighth of
// FP16's half step (measured on a long batch of one sign 5e-5; without an end to
// the chain 1.5e-3 at 262,144 values, three half steps, and growing with them).
// Longer reductions are read out every 8192 values and added in FP32 to this
// warp's part of a buffer in the workspace, beside the next chain's MMAs: their
// 256-column tiles leave no registers for the sums.
//
// A reduction split over several CTAs (few tiles, long k) writes FP32 partial
// tiles that k_join adds in order: no atomics, the same bits every time.
//
// What bounds it, measured on a B200 (single launches):
//  - long reductions: the tensor cores. dW and dx of 8192 x 4096 x 4096 BF16 in one
//    launch 332 us = 1656 TFLOP/s (a library product's burst rate is 1689), the
//    forward product alone 178 us = 1544; back to back the card's power limit takes
//    both to about 1300. 256 x 256 tiles on a pair: a CTA's 128 x 256 would need 96 bytes a
//    clock from L2, more than the 64 an SM gets (719 clocks a stage; a pair 800
//    until its MMAs were issued from uniform registers, now 580).
//  - short reductions (k <= 1024): products and epilogue about equally. 4096 x 4096
//    x 1024 with bias, GELU and a residual 32.5 us, with GELU and packed z 39 (eight
//    epilogue warps instead of 16: 38.5 and 47).
//  - single tiles: 1,500 clocks until the TMEM and the cluster are set up, 2,000 for
//    the first load, then the epilogue: 8 us in all at k <= 512.
//
// Every wait is bounded: a timeout sets a block-wide abort flag and the device
// error flag; the producer then waits (bounded) for its loads in flight, the
// MMA warp for its MMAs, and the TMEM is freed. In a pair each CTA's waits for
// the other are bounded the same way, and both reach the closing cluster
// barrier before either exits; by then each loading warp has seen every stage
// released, so no commit's arrival is still on its way to either.
#include <mutex>

#include "qrb_linear.cuh"
#include "qrb_tc.cuh"
#include "qrb_tma.cuh"

namespace qrb {
namespace lin {
namespace {

constexpr int BM = 128;       // rows per CTA
constexpr int kChainValues = 256;  // sums in registers: reduction values per accumulator chain
constexpr int kLongChain = 8192;   // sums in the workspace: the same
constexpr int kMostEpiWarps = 16;
constexpr int kMaxStages = 8;
constexpr uint32_t kSmemMost = 232448;  // 227 KB
constexpr int kPitch = 33;              // words of a row in a warp's turned block

// control block at the start of shared memory
constexpr int B_FULL = 0, B_EMPTY = kMaxStages, B_ACCFULL = 2 * kMaxStages,
              B_ACCEMPTY = B_ACCFULL + 4, B_FIN = B_ACCEMPTY + 4, B_RES = B_FIN + 1,
              NBAR = B_RES + 2 * kMostEpiWarps;
constexpr uint32_t OFF_TMEM = NBAR * 8, OFF_ABORT = OFF_TMEM + 4, CTRL = 1024;
static_assert(OFF_ABORT + 4 <= CTRL, "control block");

template <int CG, int BN, typename T, bool FWD, bool SUM>
struct Lay {
  static constexpr int NP = sizeof(T) == 4 ? 3 : 1;  // planes
  static constexpr int BK = NP == 3 ? 32 : 64;       // reduction values per stage
  static constexpr uint32_t KROW = BK * 2;           // bytes of a K-major row
  static constexpr uint32_t ATOM = BK * 128;         // MN-major box: BK rows of 128 bytes
  // stages per accumulator chain
  static constexpr int CHAIN = (SUM ? kChainValues : kLongChain) / BK;
  static constexpr int BROWS = BN / CG;              // B's columns of one CTA
  static constexpr uint32_t A = BM * KROW, B = BROWS * KROW;
  static constexpr uint32_t STAGE = NP * (A + B);
  // EW epilogue warps, EW / 4 of them across the columns, HC columns each. Each
  // has HALVES staging buffers for a block of 32 x 32 values (rows of ROWB bytes),
  // from which TMA stores the results (and into which it loads the residual); a
  // split product's FP32 blocks use both as one, unaligned matrices turn their
  // blocks there, TROWS rows at a time.
  static constexpr int EW = BN == 64 ? 8 : 16;
  static constexpr int THREADS = (EW + 2) * 32;
  static constexpr int HC = BN / (EW / 4);
  static constexpr uint32_t ROWB = 32 * sizeof(T);
  static constexpr uint32_t HBUF = 32 * ROWB, WBUF = 4096;
  static constexpr int HALVES = WBUF / HBUF;
  // without a residual or z, two blocks side by side as one box of 128-byte rows
  static constexpr bool PAIRED = !FWD && sizeof(T) == 2 && HC == 64;
  static constexpr int TROWS = 16;
  static constexpr uint32_t TURN = EW * WBUF;
  static constexpr int FIT = (int)((kSmemMost - CTRL - 1024 - TURN) / STAGE);
  static constexpr int ST = FIT < kMaxStages ? FIT : kMaxStages;
  static constexpr uint32_t SMEM = 1024 + CTRL + ST * STAGE + TURN;  // 1024: base alignment
  static_assert(TROWS * kPitch * 4 <= (int)WBUF && HC % 32 == 0, "staging");
  static_assert(A % 1024 == 0 && B % 1024 == 0, "swizzle atoms");
  static constexpr int ACC = NP == 3 ? 2 * BN : BN;  // TMEM columns per buffer
  // accumulator buffers (SUM: as many as fit, so that the MMAs of the next tile's
  // chains run while this tile's epilogue does)
  static constexpr int NACC = SUM && NP == 1 ? 4 : 2;
  static constexpr int TMEM = NACC * ACC;
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
  float* chains;    // sums of long reductions' chains, BM x BN per CTA (null: none is long)
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
  uint32_t t = (uint32_t)item;
  it.split = 0;
  it.kb0 = 0;
  it.kb1 = p.kb;
  if (p.splits > 1) {
    const uint32_t tiles = (uint32_t)(p.mt * p.nt);
    it.split = (int)(t / tiles);
    t -= (uint32_t)it.split * tiles;
    it.kb0 = (int)((long long)p.kb * it.split / p.splits);
    it.kb1 = (int)((long long)p.kb * (it.split + 1) / p.splits);
  }
  const uint32_t per = (uint32_t)(p.group * p.nt);
  const uint32_t g = t / per, r = t - g * per;
  const uint32_t first = g * (uint32_t)p.group;
  const uint32_t left = (uint32_t)p.mt - first;
  const uint32_t gm = left < (uint32_t)p.group ? left : (uint32_t)p.group;
  const uint32_t q = r / gm;
  it.m0 = (int)(first + r - q * gm) * (BM * CG);
  it.n0 = (int)q * BN;
  return it;
}

constexpr uint64_t kSw128 = 2, kSw64 = 4;
__device__ __forceinline__ uint64_t desc(uint32_t saddr, uint32_t lbo, uint32_t sbo,
                                         uint64_t layout) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)((lbo >> 4) & 0x3FFF) << 16) |
         ((uint64_t)((sbo >> 4) & 0x3FFF) << 32) | (1ull << 46) | (layout << 61);
}
// K-major: rows of KROW bytes (128 or 64, swizzled over that width), 8-row
// groups 8 KROW apart; 16 reduction values are 32 bytes. MN-major: 64-value
// atoms (128-byte rows) ATOM apart, 8-row (reduction) groups 1024 bytes apart;
// 16 reduction rows are 2048 bytes.
template <typename L>
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr, bool mn) {
  return mn ? desc(saddr, L::ATOM, 1024, kSw128)
            : desc(saddr, 16, 8 * L::KROW, L::KROW == 128 ? kSw128 : kSw64);
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
// Bounded: false on a timeout (which sets *abort) or once *abort is set.
// Block-scope acquire, also for what the other CTA of a pair announces: all that
// passes between them is TMA and TMEM traffic, ordered by the barriers
// themselves; a cluster-scope release or acquire would wait for this CTA's
// global stores and drop its L1 (4096 x 4096 x 1024 with GELU and packed z:
// 55.6 us against 52.4).
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
template <int CG, typename L, int ROWS>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, bool mn,
                                          uint32_t bar, int mn0, int kb, int plane) {
  if (mn) {
#pragma unroll
    for (int j = 0; j < ROWS / 64; ++j)
      load_box<CG>(dst + j * L::ATOM, map, bar, mn0 + 64 * j, kb * L::BK, plane);
  } else {
    load_box<CG>(dst, map, bar, kb * L::BK, mn0, plane);
  }
}

// Staged blocks: 32 rows (lane = row) of ROWB bytes with TMA's swizzle of that
// width, which also spreads a warp's 16-byte accesses over the banks.
template <uint32_t ROWB>
__device__ __forceinline__ uint32_t staged_at(uint32_t buf, int row, int unit) {
  const int x = ROWB == 128 ? unit ^ (row & 7)
                            : (ROWB == 64 ? unit ^ ((row >> 1) & 3) : unit ^ ((row >> 2) & 1));
  return buf + row * ROWB + x * 16;
}
// The lane's row of a block.
template <typename E, uint32_t ROWB>
__device__ __forceinline__ void stage_write(uint32_t buf, const float (&v)[32], int unit = 0) {
  const int row = threadIdx.x & 31;
  constexpr int PER = 16 / sizeof(E);  // values of 16 bytes
#pragma unroll
  for (int j = 0; j < 32 / PER; ++j) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (sizeof(E) == 4)
        w[k] = __float_as_uint(v[PER * j + k]);
      else
        w[k] = pair_of<E>(v[PER * j + 2 * k], v[PER * j + 2 * k + 1]);
    }
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(
                     staged_at<ROWB>(buf, row, unit + j)),
                 "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                 : "memory");
  }
}
template <typename T, uint32_t ROWB>
__device__ __forceinline__ void stage_add(uint32_t buf, float (&v)[32]) {
  const int row = threadIdx.x & 31;
  constexpr int PER = 16 / sizeof(T);
#pragma unroll
  for (int j = 0; j < 32 / PER; ++j) {
    uint32_t w[4];
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(staged_at<ROWB>(buf, row, j))
                 : "memory");
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (sizeof(T) == 4) {
        v[PER * j + k] += __uint_as_float(w[k]);
      } else {
        float lo, hi;
        values2<T>(w[k], lo, hi);
        v[PER * j + 2 * k] += lo;
        v[PER * j + 2 * k + 1] += hi;
      }
    }
  }
}
__device__ __forceinline__ void store_box(const CUtensorMap* map, uint32_t src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::
                   "l"(reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void load_box2(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x,
                                          int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
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
template <typename T, bool FWD, bool SUM, int TROWS>
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
  // all rows' residuals in flight together
  T res[32];
  if constexpr (FWD) {
    if (e.residual != nullptr) {
      const T* s = reinterpret_cast<const T*>(e.residual) + (int64_t)row0 * e.ldr + col + lane;
#pragma unroll
      for (int k = 0; k < 32; ++k) res[k] = live && k < rows ? s[k * e.ldr] : from_f<T>(0.f);
    }
  }
#pragma unroll
  for (int base = 0; base < 32; base += TROWS) {
    if (base >= rows) break;
    __syncwarp();
    if (lane >= base && lane < base + TROWS) {
#pragma unroll
      for (int i = 0; i < 32; ++i) turn[(lane - base) * kPitch + i] = v[i];
    }
    __syncwarp();
    const int most = rows - base < TROWS ? rows - base : TROWS;
#pragma unroll
    for (int r0 = 0; r0 < TROWS; r0 += 8) {
      if (r0 >= most) break;
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
#pragma unroll
          for (int k = 0; k < 8; ++k) q[k] = to_f<T>(res[base + r0 + k]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) p[k] += bias;
        if (e.z != nullptr && live) {
          T* z = reinterpret_cast<T*>(e.z) + row0g * e.ldz + col + lane;
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < left) z[k * e.ldz] = from_f<T>(p[k]);
        }
        if constexpr (SUM) {
          if (e.z_codes != nullptr) pack_rows<T>(p, row0g, left, live, col, a);
        }
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

// The packed form of the lane's row of a block: codes into the staged block (rows
// of 32 bytes); returns the exponent.
template <typename T>
__device__ __forceinline__ int pack32(uint32_t buf, const float (&v)[32]) {
  constexpr int lo = ExpRange<T>::lo, hi = ExpRange<T>::hi;
  // columns beyond the matrix are 0 (or, beside Inf or NaN, NaN)
  float part[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
  for (int i = 4; i < 32; ++i) part[i & 3] = max_abs_nan(part[i & 3], v[i]);
  float amax = max_abs_nan(max_abs_nan(part[0], part[1]), max_abs_nan(part[2], part[3]));
  const bool fine = finite_f(amax);
  if (!fine) amax = finite_amax(v);
  const int ex = block_exponent(amax, lo, hi);
  uint32_t w[8];
  encode(v, ex, fine && ex < hi, ex == hi ? 63.f : 127.f, w);
#pragma unroll
  for (int j = 0; j < 2; ++j)
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(
                     staged_at<32>(buf, threadIdx.x & 31, j)),
                 "r"(w[4 * j]), "r"(w[4 * j + 1]), "r"(w[4 * j + 2]), "r"(w[4 * j + 3])
                 : "memory");
  return ex;
}

// sum <- sum + the 32 columns at t (first: <- them).
__device__ __forceinline__ void drain(uint32_t t, float (&sum)[32], bool first) {
  float v[32];
  tc::tmem_ld32(t, v);
  if (first) {
#pragma unroll
    for (int i = 0; i < 32; ++i) sum[i] = v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 32; i += 2)
      f2_to(add2(f2_of(sum[i], sum[i + 1]), f2_of(v[i], v[i + 1])), sum[i], sum[i + 1]);
  }
}

// The lane's 32 sums in the workspace, lanes at neighbouring 16 bytes.
__device__ __forceinline__ void keep(float4* p, const float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    p[32 * i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
}
__device__ __forceinline__ void add_kept(const float4* p, float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float4 u = p[32 * i];
    v[4 * i] += u.x;
    v[4 * i + 1] += u.y;
    v[4 * i + 2] += u.z;
    v[4 * i + 3] += u.w;
  }
}

template <int CG, int BN, typename T, bool FWD, bool SUM>
__global__ void __launch_bounds__((Lay<CG, BN, T, FWD, SUM>::THREADS), 1)
    k_product(const __grid_constant__ CUtensorMap map_a0, const __grid_constant__ CUtensorMap map_b0,
              const __grid_constant__ CUtensorMap map_a1, const __grid_constant__ CUtensorMap map_b1,
              const __grid_constant__ CUtensorMap map_o0, const __grid_constant__ CUtensorMap map_o1,
              const __grid_constant__ CUtensorMap map_r, const __grid_constant__ CUtensorMap map_z,
              const __grid_constant__ CUtensorMap map_q,
              const __grid_constant__ Args a) {
  using L = Lay<CG, BN, T, FWD, SUM>;
  constexpr int kEpiWarps = L::EW;
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
  if (threadIdx.x < NBAR) {  // one barrier per thread
    const int i = (int)threadIdx.x;
    const bool acc_empty = i >= B_ACCEMPTY && i < B_FIN;
    tma::mbar_init(BAR(i), acc_empty ? CG * kEpiWarps : 1);
    tma::mbar_fence_init();
    if (i == 0) *s_abort = 0;
  }
  if (warp == kEpiWarps + 1) tmem_alloc<CG>(base + OFF_TMEM, L::TMEM);
  tc::fence_before();
  __syncthreads();
  if constexpr (CG == 2) sync_all<CG>();
  tc::fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + OFF_TMEM);
  let_next_start();     // k_join, of a split product
  wait_for_previous();  // k_prepare, where there is one

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
            load_tile<CG, L, BM>(st + p * L::A, ma, amn, bar, am, kb, p);
#pragma unroll
          for (int p = 0; p < L::NP; ++p)
            load_tile<CG, L, L::BROWS>(st + L::NP * L::A + p * L::B, mb, bmn, bar, bn, kb, p);
        }
        __syncwarp();
        ++u;
      }
    }
    // The last stages' releases are waited for as well: the MMA warp's commits arrive
    // on this CTA's barriers from outside its threads (a pair's second CTA gets them
    // from the first one), and separate commits' arrivals need not land in order, so
    // the accumulators being ready does not say that these are in. None may reach
    // shared memory that this CTA has given back.
    for (int v = u > L::ST ? u - L::ST : 0; live && v < u; ++v)
      live = warp_wait(BAR(B_EMPTY + v % L::ST), (uint32_t)((v / L::ST) & 1), a.limit, s_abort);
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
        const uint64_t da0 = operand_desc<L>(ring, amn);
        const uint64_t db0 = operand_desc<L>(ring + L::NP * L::A, bmn);
        for (int kb = it.kb0; live && kb < it.kb1;) {
          const int end = kb + L::CHAIN < it.kb1 ? kb + L::CHAIN : it.kb1;
          const int buf = unit % L::NACC;
          if (unit >= L::NACC)
            live = warp_wait(BAR(B_ACCEMPTY + buf), (uint32_t)((unit / L::NACC - 1) & 1), a.limit,
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
                for (int k = 0; k < L::BK / 16; ++k)
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
      // no MMA may run on into freed TMEM (a pair: a fixed time, as above)
      if (__any_sync(kFull, *s_abort != 0)) {
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
    const int quad = warp & 3, part_of = warp >> 2;  // rows, columns
    constexpr int HC = L::HC;  // columns of this warp
    constexpr int NH = L::HALVES;
    static_assert(HC == 32 || NH == 2, "a block's staging is free or waited for once");
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t stg = ring + L::ST * L::STAGE + warp * L::WBUF;
    float* turn = reinterpret_cast<float*>(sm + (stg - base));
    int unit = 0;
    uint32_t uses0 = 0, uses1 = 0;  // residual loads issued into each half
    bool live = true;
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
      if (a.sum.out != nullptr)  // over the blocks first: no tile waits long for it
        column_sum<T>(a.sum, (int64_t)warp * gridDim.x + blockIdx.x,
                      (int64_t)gridDim.x * kEpiWarps);
    }
    for (int step = 0; live; ++step) {
      const Item it = item_of<CG, BN>(a, worker, step);
      if (it.prob < 0) break;
      const Problem& p = a.p[FWD ? 0 : it.prob];
      const Epilogue& e = p.e;
      const CUtensorMap* map_o = it.prob == 0 ? &map_o0 : &map_o1;
      const int row0 = it.m0 + rank * BM + quad * 32, col = it.n0 + part_of * HC;
      const bool part = p.splits > 1, inside = row0 < p.m;
      const bool staged = part || e.vec != 0;
      // what is kept of z goes through the first half, y through the second
      const bool plain_z = FWD && !part && staged && e.z != nullptr;
      const bool packed_z = FWD && SUM && !part && staged && e.z_codes != nullptr;
      const bool keep_z = plain_z || packed_z;
      const bool has_res = FWD && !part && staged && e.residual != nullptr;
      // The staging is free once the last tile's stores have read it: awaited here
      // for a residual that is loaded into it, else before its first use.
      auto staging_free = [&]() {
        if (lane == 0) tma::bulk_wait_read_all();
        tma::fence_proxy_async();
        __syncwarp();
      };
      if (has_res) staging_free();
      // residual of block g into its half (z kept: the second; else alternating)
      auto half_of = [&](int g) { return NH == 1 ? 0 : (keep_z ? 1 : (g & 1)); };
      auto load_res = [&](int g) {
        const int h = half_of(g);
        if (lane == 0) {
          const uint32_t bar = BAR(B_RES + 2 * warp + h);
          tma::mbar_expect_tx(bar, L::HBUF);
          load_box2(stg + h * L::HBUF, &map_r, bar, col + 32 * g, row0);
        }
        uses0 += h == 0 ? 1u : 0u;
        uses1 += h == 0 ? 0u : 1u;
      };
      // the bias of the warp's columns: lane l has column l of each block of 32
      float bias[HC / 32];
      if constexpr (FWD) {
#pragma unroll
        for (int i = 0; i < HC / 32; ++i) {
          const int c = col + 32 * i + lane;
          bias[i] = e.bias != nullptr && c < p.n && staged && !part
                        ? to_f<T>(reinterpret_cast<const T*>(e.bias)[c])
                        : 0.f;
        }
      }
      const bool early = has_res && inside && !(NH == 1 && keep_z);
      if (early && col < p.n) load_res(0);
      if (early && !keep_z && NH == 2 && HC > 32 && col + 32 < p.n) load_res(1);

      // One block of 32 columns, c from the warp's first: v holds the sums.
      auto finish = [&](float(&v)[32], int c) {
        const int at = col + c;
        if (c == 0 && !has_res) staging_free();
        const int g = c / 32;
        if (part) {  // (rows and columns padded to whole tiles; one buffer)
          if (g > 0) {
            if (lane == 0) tma::bulk_wait_read_all();
            __syncwarp();
          }
          stage_write<float, 128>(stg, v);
          tma::fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            store_box(map_o, stg, at, (int)(it.split * p.part_rows) + row0);
            tma::bulk_commit();
          }
          return;
        }
        if (at >= p.n || !inside) return;
        if (!staged) {
          finish_turned<T, FWD, SUM, L::TROWS>(v, row0, at, p, turn);
          return;
        }
        if constexpr (L::PAIRED) {
          stage_write<T, 128>(stg, v, 4 * g);
          if (g == 1 || at + 32 >= p.n) {
            tma::fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
              store_box(map_o, stg, col, row0);
              tma::bulk_commit();
            }
          }
          return;
        }
        const uint32_t ybuf = stg + half_of(g) * L::HBUF;
        if (g > 0 && keep_z) {  // (the second and last block) its staging is free
          if (lane == 0) tma::bulk_wait_read_all();
          __syncwarp();
          if (has_res) load_res(g);
        }
        // a kept block of z out of the first half
        auto flush_z = [&](const CUtensorMap* map) {
          tma::fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            store_box(map, stg, at, row0);
            tma::bulk_commit();
            if constexpr (NH == 1) tma::bulk_wait_read_all();
          }
          __syncwarp();
          if (NH == 1 && has_res) load_res(g);
        };
        if constexpr (FWD) {
          if (e.bias != nullptr) {
            float mine = bias[0];
#pragma unroll
            for (int i = 1; i < HC / 32; ++i) mine = c == 32 * i ? bias[i] : mine;
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] += __shfl_sync(kFull, mine, i);
          }
          if (plain_z) {
            stage_write<T, L::ROWB>(stg, v);
            flush_z(&map_z);
          }
          if constexpr (SUM) {  // (one block of 32 columns a warp)
            if (packed_z) {
              const int ex = pack32<T>(stg, v);
              flush_z(&map_q);
              if (row0 + lane < p.m)
                e.z_exps[(int64_t)(row0 + lane) * ((p.n + kBlk - 1) / kBlk) + at / kBlk] =
                    (int8_t)ex;
            }
          }
          act_by(v, e.act);
          if (has_res) {
            const int h = half_of(g);
            const uint32_t uses = h == 0 ? uses0 : uses1;
            live = warp_wait(BAR(B_RES + 2 * warp + h), (uses - 1) & 1, a.limit, s_abort);
            stage_add<T, L::ROWB>(ybuf, v);
          }
        }
        stage_write<T, L::ROWB>(ybuf, v);
        tma::fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          store_box(map_o, ybuf, at, row0);
          tma::bulk_commit();
        }
      };

      if constexpr (!SUM) {
        // this lane's sums of the chains before the last: four columns each 32 apart
        float4* kept = reinterpret_cast<float4*>(a.chains) +
                       ((size_t)blockIdx.x * kEpiWarps + warp) * (HC * 8) + lane;
        int kb = it.kb0;
        do {
          const int buf = unit % L::NACC;
          live = warp_wait(BAR(B_ACCFULL + buf), (uint32_t)((unit / L::NACC) & 1), a.limit,
                           s_abort);
          if (!live) break;
          tc::fence_after();
          const uint32_t t = tmem + lanes + buf * L::ACC + part_of * HC;
          const bool last = kb + L::CHAIN >= it.kb1;
#pragma unroll 1
          for (int c = 0; c < HC; c += 32) {
            float v[32];
            tc::tmem_ld32(t + c, v);
            if (c + 32 == HC) hand_back(buf);
            if (kb > it.kb0) add_kept(kept + 8 * c, v);
            if (last)
              finish(v, c);
            else
              keep(kept + 8 * c, v);
          }
          kb += L::CHAIN;
          ++unit;
        } while (live && kb < it.kb1);
        if (!live) break;
      } else {
        static_assert(!SUM || HC == 32, "one block of sums per warp");
        float sum[32];
        for (int kb = it.kb0; kb < it.kb1; kb += L::CHAIN, ++unit) {
          const int buf = unit % L::NACC;
          live = warp_wait(BAR(B_ACCFULL + buf), (uint32_t)((unit / L::NACC) & 1), a.limit,
                           s_abort);
          if (!live) break;
          tc::fence_after();
          const uint32_t t = tmem + lanes + buf * L::ACC + part_of * HC;
          drain(t, sum, kb == it.kb0);
          if constexpr (L::NP == 3) drain(t + BN, sum, false);
          hand_back(buf);
        }
        if (!live) break;
        finish(sum, 0);
      }
    }
    // no load or store of this warp's may use the staging after the block has gone
    if (lane == 0) {
      if (*s_abort != 0) {
        for (int h = 0; h < 2; ++h) {
          const uint32_t uses = h == 0 ? uses0 : uses1;
          if (uses > 0)
            tma::mbar_wait_bounded(BAR(B_RES + 2 * warp + h), (uses - 1) & 1, a.limit);
        }
      }
      tma::bulk_wait_read_all();
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
// An operand as boxes of `inner` x `rows` elements per plane (inner 64: 128
// bytes and their swizzle, 32: 64).
bool encode_operand(CUtensorMap* map, const Operand& o, int planes, uint32_t inner,
                    uint32_t rows) {
  PFN_cuTensorMapEncodeTiled_v12000 fn = tma::encoder();
  if (fn == nullptr) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)planes};
  const cuuint64_t row = (cuuint64_t)o.ld * 2;
  const cuuint64_t strides[2] = {row, planes > 1 ? (cuuint64_t)o.plane * 2
                                                 : row * (cuuint64_t)o.rows};
  const cuuint32_t box[3] = {inner, rows, 1}, es[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(o.p), dims, strides, box,
            es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            inner == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A row-major matrix as the epilogue's staged blocks: 32 rows of rowb bytes.
bool encode_staged(CUtensorMap* map, const void* p, int elem, int64_t cols, int64_t rows,
                   int64_t ld, uint32_t rowb) {
  PFN_cuTensorMapEncodeTiled_v12000 fn = tma::encoder();
  if (fn == nullptr) return false;
  if (rows <= 1) ld = (cols + 15) / 16 * 16;  // one row: any legal stride
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * (cuuint64_t)elem};
  const cuuint32_t box[2] = {rowb / (uint32_t)elem, 32}, es[2] = {1, 1};
  const CUtensorMapDataType type = elem == 4   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : elem == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                               : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const CUtensorMapSwizzle swizzle = rowb == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                     : rowb == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                  : CU_TENSOR_MAP_SWIZZLE_32B;
  return fn(map, type, 2, const_cast<void*>(p), dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_NONE,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
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
template <int CG, int BN, typename T, bool FWD, bool SUM>
int launch_t(const Product* const* q, int count, Args& args, bool after_prepare, cudaStream_t s) {
  using L = Lay<CG, BN, T, FWD, SUM>;
  static std::once_flag once[64];
  static bool ready[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return QRB_ERR_DEVICE;
  std::call_once(once[dev], [dev] {
    ready[dev] = cudaFuncSetAttribute(k_product<CG, BN, T, FWD, SUM>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)L::SMEM) == cudaSuccess;
  });
  if (!ready[dev]) return QRB_ERR_LAUNCH;
  CUtensorMap ma[2], mb[2], mo[2], mr, mz, mq;
  constexpr int ES = sizeof(T);
  for (int i = 0; i < count; ++i) {
    const Problem& p = args.p[i];
    const Epilogue& e = p.e;
    bool fine = encode_operand(&ma[i], q[i]->a, L::NP, p.amn ? 64 : L::BK, p.amn ? L::BK : BM) &&
                encode_operand(&mb[i], q[i]->b, L::NP, p.bmn ? 64 : L::BK,
                               p.bmn ? L::BK : L::BROWS);
    if (p.splits > 1)
      fine = fine && encode_staged(&mo[i], p.part, 4, p.part_ld, p.part_rows * p.splits,
                                   p.part_ld, 128);
    else if (e.vec)
      fine = fine && encode_staged(&mo[i], e.out, ES, p.n, p.m, e.ldo,
                                   L::PAIRED ? 128 : L::ROWB);
    else
      mo[i] = ma[i];  // (not used)
    if (!fine) return QRB_ERR_UNSUPPORTED;
  }
  if (count == 1) {
    ma[1] = ma[0];
    mb[1] = mb[0];
    mo[1] = mo[0];
  }
  mr = mz = mq = mo[0];
  if (FWD && args.p[0].splits == 1 && args.p[0].e.vec) {
    const Problem& p = args.p[0];
    if ((p.e.residual != nullptr &&
         !encode_staged(&mr, p.e.residual, ES, p.n, p.m, p.e.ldr, L::ROWB)) ||
        (p.e.z != nullptr && !encode_staged(&mz, p.e.z, ES, p.n, p.m, p.e.ldz, L::ROWB)) ||
        (p.e.z_codes != nullptr && !encode_staged(&mq, p.e.z_codes, 1, p.n, p.m, p.n, 32)))
      return QRB_ERR_UNSUPPORTED;
  }
  cudaLaunchConfig_t lc = {};
  cudaLaunchAttribute la[2];
  int attrs = 0;
  if (CG == 2) {
    la[attrs].id = cudaLaunchAttributeClusterDimension;
    la[attrs].val.clusterDim.x = 2;
    la[attrs].val.clusterDim.y = 1;
    la[attrs++].val.clusterDim.z = 1;
  }
  if (after_prepare) la[attrs++] = early_start();
  lc.gridDim = dim3(CG * (unsigned)args.s.workers);
  lc.blockDim = dim3(L::THREADS);
  lc.dynamicSmemBytes = L::SMEM;
  lc.stream = s;
  lc.attrs = la;
  lc.numAttrs = attrs;
  if (cudaLaunchKernelEx(&lc, k_product<CG, BN, T, FWD, SUM>, ma[0], mb[0], ma[1], mb[1], mo[0],
                         mo[1], mr, mz, mq, args) != cudaSuccess) {
    (void)cudaGetLastError();
    return QRB_ERR_LAUNCH;
  }
  note_launches(1);
  return cudaGetLastError() == cudaSuccess ? QRB_OK : QRB_ERR_LAUNCH;
}

template <int CG, int BN, typename T>
int launch_dir(bool fwd, bool sum, const Product* const* q, int count, Args& args, bool after_prepare,
               cudaStream_t s) {
  constexpr bool F32 = sizeof(T) == 4;
  if (!fwd) return launch_t<CG, BN, T, false, F32>(q, count, args, after_prepare, s);
  if constexpr (!F32 && BN <= 128) {
    if (sum) return launch_t<CG, BN, T, true, true>(q, count, args, after_prepare, s);
  }
  return launch_t<CG, BN, T, true, F32>(q, count, args, after_prepare, s);
}

template <typename T>
int launch_type(int cg, int bn, bool fwd, bool sum, const Product* const* q, int count,
                Args& args, bool after_prepare, cudaStream_t s) {
  if (cg == 1 && bn == 64) return launch_dir<1, 64, T>(fwd, sum, q, count, args, after_prepare, s);
  if (cg == 1 && bn == 128) return launch_dir<1, 128, T>(fwd, sum, q, count, args, after_prepare, s);
  if (cg == 2 && bn == 128) return launch_dir<2, 128, T>(fwd, sum, q, count, args, after_prepare, s);
  if constexpr (sizeof(T) == 2) {
    if (cg == 2 && bn == 256) return launch_dir<2, 256, T>(fwd, sum, q, count, args, after_prepare, s);
  }
  return QRB_ERR_INVALID_ARG;
}

int64_t tiles_of(int64_t v, int64_t t) { return (v + t - 1) / t; }

// The cuts of the kernel: CTAs per tile, tile width, and what one stage of one
// tile takes, in microseconds, measured on a B200 over m, n, k = 360 .. 8192.
struct Cut {
  int cg, bn;
  double stage;
};
constexpr Cut kCuts16[] = {{2, 256, 0.33}, {2, 128, 0.25}, {1, 128, 0.25}, {1, 64, 0.20}};
constexpr Cut kCuts32[] = {{2, 128, 0.65}, {1, 128, 0.72}, {1, 64, 0.53}};

// One tile's products and its epilogue (which run beside another tile's), in
// microseconds: a column of results takes 9 ns, 6 more with an activation, 6 with
// z kept, 4 with a residual (FP32 twice that).
struct TileTime {
  double main, epi;
  double longer() const { return main > epi ? main : epi; }
  double shorter() const { return main > epi ? epi : main; }
};
TileTime tile_time(bool f32, const Cut& c, const ProductSize& z, int64_t kb, bool split) {
  const double col = split ? 0.009
                           : 0.009 + ((z.epilogue & 1) ? 0.006 : 0) + ((z.epilogue & 2) ? 0.006 : 0) +
                                 ((z.epilogue & 4) ? 0.004 : 0);
  return {(double)kb * c.stage, c.bn * col * (f32 ? 2 : 1)};
}

// The schedule of `items[0]` longer and `items[1]` shorter items over `most`
// workers, and its length in the items' own times.
double make_schedule(const int64_t* items, const double* each, int64_t most, Schedule* out) {
  const int64_t all = items[0] + items[1];
  const int64_t g = all < most ? all : most;
  Schedule s = {};
  s.workers = (int)g;
  s.q = (int)(items[0] / g);
  s.r = (int)(items[0] % g);
  double length = (s.q + (s.r > 0 ? 1 : 0)) * each[0];
  if (items[1] > 0) {
    // `more` rounds of short items fit beside the one more long item that the
    // first r workers have; the least x and y = x - more (or 0) that hold all
    const int64_t more = (int64_t)(each[0] / each[1] + 0.5), rest = g - s.r;
    int64_t x = (items[1] + rest - 1) / rest, y = 0;
    if (s.r == 0) {
      y = x;
    } else if (x > more) {
      x = (items[1] + more * s.r + g - 1) / g;
      y = x - more;
    }
    s.x = (int)x;
    s.y = (int)y;
    const double late = s.q * each[0] + s.x * each[1];
    const double early = s.r > 0 ? (s.q + 1) * each[0] + s.y * each[1] : 0;
    length = late > early ? late : early;
  }
  *out = s;
  return length;
}

int stage_values(bool f32) {
  return f32 ? Lay<1, 64, float, true, true>::BK : Lay<1, 64, bf16, true, false>::BK;
}

Problem problem_of(int kind, int64_t m, int64_t n, int64_t k, const Cut& c, int bk, int splits) {
  Problem p = {};
  p.m = (int)m;
  p.n = (int)n;
  p.mt = (int)tiles_of(m, BM * c.cg);
  p.nt = (int)tiles_of(n, c.bn);
  p.kb = (int)tiles_of(k, bk);
  p.splits = splits;
  p.items = p.mt * p.nt * splits;
  p.group = c.cg == 2 ? 8 : 16;
  p.amn = kind == kGradW;
  p.bmn = kind != kForward;
  return p;
}

}  // namespace

// The cut with the least estimated time: a start of 4.5 us, the schedule's
// length, the end of the last tile, and for each split product 2.5 us for its
// second launch and its partial sums' way out and back at 5 TB/s.
static ProductPlan search_plan(int dtype, const ProductSize* sizes, int count) {
  ProductPlan best;
  const Device* d = device_info();
  const int64_t sms = d != nullptr ? d->sms : 148;
  const bool f32 = dtype == QRBL_F32;
  double least = -1;
  const Cut* cuts = f32 ? kCuts32 : kCuts16;
  const int ncuts = f32 ? 3 : 4;
  const bool chains = f32 || (sizes[0].epilogue & 8) != 0;
  const int hook_splits = linear_splits();
  const int hook_cut = chains && linear_cut() == 2256 ? 2128 : linear_cut();
  for (int ci = 0; ci < ncuts; ++ci) {
    const Cut c = cuts[ci];
    if (c.bn > 128 && chains) continue;  // no registers for its sums
    if (hook_cut != 0 && hook_cut != 1000 * c.cg + c.bn) continue;
    const int64_t workers = sms / c.cg;
    int64_t tiles[2] = {0, 0}, kb[2] = {1, 1};
    for (int i = 0; i < count; ++i) {
      tiles[i] = tiles_of(sizes[i].m, BM * c.cg) * tiles_of(sizes[i].n, c.bn);
      kb[i] = tiles_of(sizes[i].k, stage_values(f32));
      if (tiles[i] > (1 << 26)) return best;  // (refused: 26 bits of tiles)
    }
    for (int s0 = 1; s0 <= 16 && s0 <= kb[0]; ++s0) {
      if (hook_splits > 0 && s0 != hook_splits && s0 != kb[0]) continue;
      if (hook_splits == 0 && s0 > 1 && tiles[0] * (s0 - 1) >= workers) break;
      for (int s1 = 1; s1 <= (count > 1 ? 16 : 1) && s1 <= kb[1]; ++s1) {
        if (hook_splits > 0 && count > 1 && s1 != hook_splits && s1 != kb[1]) continue;
        if (hook_splits == 0 && s1 > 1 && tiles[1] * (s1 - 1) >= workers) break;
        const int sp[2] = {s0, s1};
        double len[2] = {0, 0}, t = 4.5, end = 0;
        int64_t items[2] = {0, 0};
        for (int i = 0; i < count; ++i) {
          const ProductSize& z = sizes[i];
          const TileTime x = tile_time(f32, c, z, tiles_of(kb[i], sp[i]), sp[i] > 1);
          items[i] = tiles[i] * sp[i];
          len[i] = x.longer();
          if (x.shorter() > end) end = x.shorter();
          if (sp[i] > 1) t += 2.5 + 8.0 * sp[i] * (double)z.m * (double)z.n / 5e6;
        }
        const bool swap = count > 1 && len[1] > len[0];
        const int64_t it[2] = {items[swap ? 1 : 0], count > 1 ? items[swap ? 0 : 1] : 0};
        const double each[2] = {len[swap ? 1 : 0], count > 1 ? len[swap ? 0 : 1] : 1.0};
        Schedule sc;
        t += make_schedule(it, each, workers, &sc) + end;
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
  if (!chains && least >= 0) {
    int64_t items = 0;
    bool some = false;
    for (int i = 0; i < count; ++i) {
      items += tiles_of(sizes[i].m, BM * best.cg) * tiles_of(sizes[i].n, best.bn) * best.splits[i];
      some |= tiles_of(tiles_of(sizes[i].k, stage_values(f32)), best.splits[i]) >
              kLongChain / stage_values(f32);
    }
    const int64_t workers = items < sms / best.cg ? items : sms / best.cg;
    if (some) best.chain_bytes = (size_t)workers * best.cg * BM * best.bn * sizeof(float);
  }
  best.ok = least >= 0;
  return best;
}

// A pure function of its arguments and the device's SM count; the last few
// results are kept per thread, since a call asks twice (its workspace, its
// launch) and a model's layers repeat.
ProductPlan plan_products(int dtype, const ProductSize* sizes, int count) {
  struct Entry {
    int dtype = -1, count = 0, sms = 0, hooks = 0;
    ProductSize z[2];
    ProductPlan plan;
  };
  static thread_local Entry kept[64];
  const Device* d = device_info();
  const int sms = d != nullptr ? d->sms : 0;
  const int hooks = linear_cut() * 32 + linear_splits();
  uint64_t h = (uint64_t)dtype * 3 + (uint64_t)count;
  for (int i = 0; i < count; ++i)
    h = (h * 1000003u + (uint64_t)sizes[i].m) * 1000003u + (uint64_t)sizes[i].n * 8191u +
        (uint64_t)sizes[i].k;
  Entry& e = kept[(h ^ (h >> 17) ^ (h >> 31)) % 64];
  bool same = e.dtype == dtype && e.count == count && e.sms == sms && e.hooks == hooks;
  for (int i = 0; i < count && same; ++i)
    same = e.z[i].m == sizes[i].m && e.z[i].n == sizes[i].n && e.z[i].k == sizes[i].k &&
           e.z[i].epilogue == sizes[i].epilogue;
  if (!same) {
    e.dtype = dtype;
    e.count = count;
    e.sms = sms;
    e.hooks = hooks;
    for (int i = 0; i < count; ++i) e.z[i] = sizes[i];
    e.plan = search_plan(dtype, sizes, count);
  }
  return e.plan;
}

int launch_products(int dtype, const Product* products, int count, const ProductPlan& plan,
                    float* chains, const ColSum* cols, bool after_prepare, cudaStream_t s) {
  const Device* d = device_info();
  if (d == nullptr) return QRB_ERR_DEVICE;
  if (!plan.ok) return QRB_ERR_UNSUPPORTED;
  const bool f32 = dtype == QRBL_F32;
  Cut c = {plan.cg, plan.bn, 1.0};
  for (const Cut& k : kCuts16)
    if (!f32 && k.cg == c.cg && k.bn == c.bn) c = k;
  for (const Cut& k : kCuts32)
    if (f32 && k.cg == c.cg && k.bn == c.bn) c = k;
  Args args = {};
  const Product* q[2] = {nullptr, nullptr};
  int64_t items[2] = {0, 0};
  double each[2] = {1.0, 1.0};
  for (int j = 0; j < count; ++j) {
    const int i = count > 1 ? (j == 0 ? plan.first : 1 - plan.first) : 0;  // longer items first
    q[j] = &products[i];
    const ProductSize& z = products[i].size;
    args.p[j] = problem_of(products[i].kind, z.m, z.n, z.k, c, stage_values(f32), plan.splits[i]);
    args.p[j].part = plan.splits[i] > 1 ? products[i].part : nullptr;
    args.p[j].part_rows = plan.part_rows[i];
    args.p[j].part_ld = plan.part_ld[i];
    args.p[j].e = products[i].e;
    // packed rows 16-byte aligned too (and z not kept both ways: one staging half)
    if (products[i].e.z_codes != nullptr)
      args.p[j].e.vec &= aligned16(products[i].e.z_codes) && z.n % 16 == 0 &&
                         products[i].e.z == nullptr;
    items[j] = args.p[j].items;
    each[j] = tile_time(f32, c, z, tiles_of(args.p[j].kb, plan.splits[i]), plan.splits[i] > 1)
                  .longer();
  }
  make_schedule(items, each, d->sms / c.cg, &args.s);
  if (cols != nullptr) args.sum = *cols;
  args.chains = chains;
  args.err = d->err;
  args.limit = device_wait_limit();
  args.skip_mma = test_skip_mma() ? 1 : 0;
  const bool fwd = products[0].kind == kForward;
  const bool sum = (products[0].size.epilogue & 8) != 0;
  int rc = QRB_ERR_INVALID_ARG;
  switch (dtype) {
    case QRBL_F32: rc = launch_type<float>(c.cg, c.bn, fwd, sum, q, count, args, after_prepare, s); break;
    case QRBL_F16: rc = launch_type<f16>(c.cg, c.bn, fwd, sum, q, count, args, after_prepare, s); break;
    case QRBL_BF16: rc = launch_type<bf16>(c.cg, c.bn, fwd, sum, q, count, args, after_prepare, s); break;
  }
  for (int i = 0; i < count && rc == QRB_OK; ++i)
    if (plan.splits[i] > 1)
      rc = launch_join(dtype, products[i].part, plan.splits[i], plan.part_rows[i],
                       plan.part_ld[i], products[i].size.m, products[i].size.n, products[i].e, true,
                       s);
  return rc;
}

}  // namespace lin
}  // namespace qrb
