// Matrix products C = sum_k A[m][k] B[n][k] of bf16 operands with float32
// accumulators, as a tile for each workgroup with an epilogue of the caller's.
//
// An operand lies in memory by rows of its free index with k contiguous, or by
// rows of k with the free index contiguous (COL); each kind goes to LDS as it
// lies, by LDS-DMA in a ring of stages, and is read from there by one 16-byte
// read a fragment, or two transposing reads.  A float32 operand is
// given as planes of bf16 pieces, and the product as a sum over pairs of planes:
// the same loop goes over k once for each pair.
//
// Lane l's accumulators of tile (i, j) of 16 x 16 are four consecutive m, from
// m_of(i) on, at the one n 16 j + l % 16.
#pragma once
#include "tile.h"

namespace gmdn {
namespace {

struct MMOperand {
  const bf16* p;
  int64_t stride, plane;   // elements between rows, and between planes
  // the last valid free index and (COL) k: what lies behind them reads them again.  Every
  // tile begins within both (a copy's offset from there is not negative).
  int64_t last, k_last;
};
struct MMArgs {
  MMOperand a, b;
  int steps;              // k in stages of BK
  int per;                // stages of a split
  int tiles_m, tiles_n;
  int pairs;
  uint32_t pair_a, pair_b;  // the planes of pair i: four bits from 4 i on
};

template <int TM_, int TN_, int BK_, int STAGES_, int WM_, int WN_>
struct MMShape {
  static constexpr int TM = TM_, TN = TN_, BK = BK_, STAGES = STAGES_, WM = WM_, WN = WN_;
  static constexpr int THREADS = 64 * WM * WN;
  static constexpr int MT = TM / WM / 16, NT = TN / WN / 16;
};

// An operand's tile in LDS: where a thread's copies come from (NOPS of 16 bytes, byte
// offsets from the tile's first element) and go to, and how fragments are read.
// Reads are free of bank conflicts (the bank model in tile.h).
//
// COL, 256 columns: a copy of a wave is 1 KiB, two rows of k.  Rows k and k + 4, which
// no read takes together, are such a pair, and a pair is followed by 32 unused
// bytes: the eight rows that 32 lanes read at once, 32 bytes each, are of eight
// pairs in a row and fall into eight different places of the 256 bytes of banks.
// All addresses are a lane's one base and constants; under an XOR swizzle the
// addresses of 24 fragments were as many registers, and 31 were spilled.
// Others: the XOR swizzles of tile.h.
template <int T, int BK, int THREADS, bool COL, bool PERM>
struct MMPlan {
  static constexpr bool PAIRS = COL && T == 256;
  static constexpr int COLS = COL ? T : BK, PAIR = 2 * T * 2 + 32;
  using L = std::conditional_t<COL, PairSwz<COLS>, RowSwz<COLS>>;
  static constexpr int GPR = COLS / 8, NOPS = T * BK / 8 / THREADS;
  static constexpr int BYTES = PAIRS ? BK / 2 * PAIR : T * BK * 2;
  static_assert(T * BK / 8 % THREADS == 0, "a tile splits evenly over the workgroup");
  // PERM: within 32 rows, row 16 u + 4 G + j of the tile is the operand's 8 G + 4 u + j, so
  // that two tiles hold eight consecutive m of a lane and 32 of its four groups.
  static GMDN_DEV int row_of(int r) { return PERM ? (r & ~31) | ((r & 12) << 1) | ((r & 16) >> 2) | (r & 3) : r; }
  uint32_t off[NOPS];
  GMDN_DEV void init(const MMOperand& o, int64_t first, int64_t k0) {
    const int l = lane_id(), w = wave_id();
#pragma unroll
    for (int i = 0; i < NOPS; ++i) {
      const int p = i * THREADS + w * 64 + l;
      int r = p / GPR, q = (p % GPR) ^ L::xr(p / GPR);
      if constexpr (PAIRS) {
        const int pair = p / 64;
        r = ((pair >> 2) << 3) | (l >> 5) << 2 | (pair & 3);
        q = l & 31;
      }
      if constexpr (COL) {
        const int64_t group = (o.last - first) / 8, k = o.k_last - k0, at = r < k ? r : k;
        off[i] = (uint32_t)((at * o.stride + 8 * (q < group ? q : group)) * 2);
      } else {
        const int64_t left = o.last - first, at = row_of(r);
        off[i] = (uint32_t)(((at < left ? at : left) * o.stride + 8 * q) * 2);
      }
    }
  }
  GMDN_DEV void issue(const bf16* from, uint32_t lds) const {
    // the same for the whole wave, and in scalar registers
    const uint64_t p = (uint64_t)from;
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(p >> 32)), lo = __builtin_amdgcn_readfirstlane((uint32_t)p);
    const bf16* const g = (const bf16*)((uint64_t)hi << 32 | lo);
    constexpr int WAVE = PAIRS ? PAIR : 1024;  // bytes that a wave's copy goes forward
    const uint32_t at = lds + __builtin_amdgcn_readfirstlane(wave_id()) * WAVE;
#pragma unroll
    for (int i = 0; i < NOPS; ++i) lds_dma16_s(g, off[i], at + i * (THREADS / 64) * WAVE);
  }
  // the fragment of 16 free indices from f, k0 .. k0 + 31
  static GMDN_DEV bf16x8 fragment(lds_cptr tile, int f, int k0) {
    const int l = lane_id(), i = l & 15, G = l >> 4;
    if constexpr (PAIRS) {
      const lds_cptr at = tile + (4 * G + (i >> 2)) * PAIR + 8 * (i & 3) + (k0 / 2 * PAIR + 2 * f);
      return cat8(lds_tr16(at), lds_tr16(at + 2 * T));
    } else if constexpr (COL) {
      const int r = k0 + 8 * G + (i >> 2), c = f + 4 * (i & 3);
      return cat8(lds_tr16(tile + swz_off<L>(r, c)), lds_tr16(tile + swz_off<L>(r + 4, c)));
    } else {
      return lds_ld<bf16x8>(tile + swz_off<L>(f + i, k0 + 8 * G));
    }
  }
};

// The tile that a workgroup forms.  Each of the 8 XCDs takes a contiguous range of
// an order that goes through 8 tiles of n for each tile of m, so that the
// workgroups that run on it at one time share their operands in its L2.
struct MMTile {
  int m, n;
};
GMDN_DEV MMTile mm_tile(const MMArgs& a) {
  const int total = a.tiles_m * a.tiles_n, x = blockIdx.x;
  const int per = total / 8, more = total % 8, xcd = x % 8;
  const int id = xcd * per + (xcd < more ? xcd : more) + x / 8;
  const int group = id / (8 * a.tiles_m), in = id % (8 * a.tiles_m);
  const int left = a.tiles_n - 8 * group, width = left < 8 ? left : 8;
  return {in / width, 8 * group + in % width};
}

template <class S, bool ACOL, bool BCOL, bool PERM>
struct MMLds {
  using PA = MMPlan<S::TM, S::BK, S::THREADS, ACOL, PERM>;
  using PB = MMPlan<S::TN, S::BK, S::THREADS, BCOL, false>;
  static constexpr int A_BYTES = PA::BYTES, STAGE = A_BYTES + PB::BYTES, BYTES = S::STAGES * STAGE;
};

// epi(acc, tile, first m and n of the workgroup's tile, the wave's place in it, LDS)
template <class S, bool ACOL, bool BCOL, bool PERM, class Epi>
__global__ void __launch_bounds__(S::THREADS)
mm_kernel(MMArgs a, Epi epi) {
  extern __shared__ __align__(16) char mm_smem[];
  using M = MMLds<S, ACOL, BCOL, PERM>;
  using PA = typename M::PA;
  using PB = typename M::PB;
  constexpr int BK = S::BK, STAGES = S::STAGES, OPS = PA::NOPS + PB::NOPS;
  static_assert(BK == 64, "a stage is two halves");
  const lds_ptr lds = lds_base(mm_smem);
  const uint32_t lds0 = lds_addr(mm_smem);
  const MMTile tile = mm_tile(a);
  const int64_t m0 = (int64_t)tile.m * S::TM, n0 = (int64_t)tile.n * S::TN;
  const int w = __builtin_amdgcn_readfirstlane(wave_id()), wm = w / S::WN, wn = w % S::WN;
  const int first = blockIdx.y * a.per, count = first + a.per < a.steps ? a.per : a.steps - first;
  const int total = a.pairs * count;
  PA pa;
  PB pb;
  pa.init(a.a, m0, 0);
  pb.init(a.b, n0, 0);
  const bf16* const ga = a.a.p + (ACOL ? m0 : m0 * a.a.stride);
  const bf16* const gb = a.b.p + (BCOL ? n0 : n0 * a.b.stride);
  const int64_t step_a = ACOL ? BK * a.a.stride : BK, step_b = BCOL ? BK * a.b.stride : BK;
  int pair = 0, at = first;
  auto issue = [&](int stage) {
    const uint32_t to = lds0 + stage * M::STAGE;
    const bf16* const pga = ga + (a.pair_a >> (4 * pair) & 15) * a.a.plane + at * step_a;
    const bf16* const pgb = gb + (a.pair_b >> (4 * pair) & 15) * a.b.plane + at * step_b;
    const int64_t k0 = (int64_t)at * BK;
    if ((ACOL && k0 + BK - 1 > a.a.k_last) || (BCOL && k0 + BK - 1 > a.b.k_last)) {
      PA ta;
      PB tb;
      ta.init(a.a, m0, k0);
      tb.init(a.b, n0, k0);
      ta.issue(pga, to);
      tb.issue(pgb, to + M::A_BYTES);
    } else {
      pa.issue(pga, to);
      pb.issue(pgb, to + M::A_BYTES);
    }
    if (++at == first + count) {
      at = first;
      ++pair;
    }
  };
  f32x4 acc[S::MT][S::NT];
#pragma unroll
  for (int i = 0; i < S::MT; ++i)
#pragma unroll
    for (int j = 0; j < S::NT; ++j) acc[i][j] = zero4();

  // A stage is two halves of k.  While a half's products run the next half's
  // fragments are read; between the halves of a stage, when all of it is in registers,
  // the workgroup meets: the next stage is there, and this one's place is filled again.
  struct Half {
    bf16x8 a[S::MT], b[S::NT];
  } half[2];
  auto read = [&](Half& h, int stage, int k) {
    const lds_cptr ta = lds + stage * M::STAGE, tb = ta + M::A_BYTES;
#pragma unroll
    for (int j = 0; j < S::NT; ++j) h.b[j] = PB::fragment(tb, (wn * S::NT + j) * 16, k);
#pragma unroll
    for (int i = 0; i < S::MT; ++i) h.a[i] = PA::fragment(ta, (wm * S::MT + i) * 16, k);
  };
  auto multiply = [&](const Half& h) {
#pragma unroll
    for (int i = 0; i < S::MT; ++i)
#pragma unroll
      for (int j = 0; j < S::NT; ++j) acc[i][j] = mfma(h.a[i], h.b[j], acc[i][j]);
  };
  // a share of the products, then one LDS read: left to itself the compiler reads
  // each fragment just before it is used, and waits for it
  auto interleave = [] {
    constexpr int READS = S::MT * (ACOL ? 2 : 1) + S::NT * (BCOL ? 2 : 1), EACH = S::MT * S::NT / READS;
#pragma unroll
    for (int i = 0; i < READS; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, EACH < 1 ? 1 : EACH, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  int issued = 0;
  for (; issued < STAGES && issued < total; ++issued) issue(issued);
  if (issued == STAGES)
    wait_vmem_le<(STAGES - 1) * OPS>();
  else
    wait_vmem();
  asm volatile("s_barrier" ::: "memory");
  read(half[0], 0, 0);
  int stage = 0;
  for (int s = 0; s < total; ++s) {
    const int next = stage + 1 == STAGES ? 0 : stage + 1;
    read(half[1], stage, 32);
    multiply(half[0]);
    interleave();
    // the next stage's copies are the oldest; the last stages have nothing behind them
    if (issued - s - 2 >= STAGES - 2)
      wait_vmem_le<(STAGES - 2) * OPS>();
    else
      wait_vmem();
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (issued < total) {
      issue(stage);
      ++issued;
    }
    __builtin_amdgcn_sched_barrier(0);
    read(half[0], next, 0);  // behind the last stage: a stale one, not used
    multiply(half[1]);
    interleave();
    stage = next;
  }
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  epi(acc, tile, m0, n0, wm, wn, mm_smem);
}

// First of the four m that the accumulators of the workgroup's m tile i hold in
// lane group G, from the workgroup's first.
template <bool PERM>
GMDN_DEV int m_of(int i, int G) {
  return PERM ? (i & ~1) * 16 + 8 * G + 4 * (i & 1) : 16 * i + 4 * G;
}

template <class S, bool ACOL, bool BCOL, bool PERM, class Epi>
bool mm_launch(const MMArgs& a, const Epi& epi, int splits, hipStream_t st) {
  auto* const kern = mm_kernel<S, ACOL, BCOL, PERM, Epi>;
  constexpr int LDS = MMLds<S, ACOL, BCOL, PERM>::BYTES;
  if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess) return false;
  hipLaunchKernelGGL(kern, dim3((unsigned)(a.tiles_m * a.tiles_n), (unsigned)splits), dim3(S::THREADS), LDS, st, a, epi);
  return hipGetLastError() == hipSuccess;
}

}  // namespace
}  // namespace gmdn
