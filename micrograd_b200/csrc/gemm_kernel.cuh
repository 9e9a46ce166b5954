// The FP64 tensor-core GEMM kernel, its tile configurations and its launch.  gemm.cu
// describes the design and instantiates it for the dense products; gemm_ext.cu does so
// for few rows, row pitches, odd row lengths and 8-bit masks.
#pragma once

#include "common.cuh"
#include "gemm.cuh"
#include "tma.cuh"

namespace mg {

constexpr int BK = 16;  // contraction depth of one stage (one 128-byte swizzle row of doubles)
constexpr int kConsumerWarps = 8;
constexpr int kProducerWarps = 4;  // one warp group; only its first lane issues copies
constexpr int kGemmThreads = (kConsumerWarps + kProducerWarps) * 32;  // 384
// Register split between the warp groups (setmaxnreg): 8*32*232 + 4*32*40 <= 64 K.
constexpr int kConsumerRegs = 232, kProducerRegs = 40;

// CTA tile = (8 / WARPS_N) x WARPS_N consumer warps, each owning MT x NT
// sub-tiles of 16 x 8 outputs.
template <int WARPS_N_, int MT_, int NT_, int STAGES_>
struct TileCfg {
  static constexpr int WARPS_N = WARPS_N_, WARPS_M = kConsumerWarps / WARPS_N_;
  static constexpr int MT = MT_, NT = NT_, STAGES = STAGES_;
  static constexpr int BM = WARPS_M * MT * 16, BN = WARPS_N * NT * 8;
  static constexpr int A_BYTES = BM * BK * 8, B_BYTES = BN * BK * 8;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  // full + empty barrier per stage, plus the consumers' meeting point around the tile ticket
  static constexpr int kBarriers = 2 * STAGES + 1;
  static constexpr int SMEM_BYTES =
      STAGES * STAGE_BYTES + 1024 /* alignment slack */ + kBarriers * 8;
  // The ReLU-mask source tile of an output tile, staged through the same ring
  // after the last k-tile: BN/16 boxes of BM rows x 16 columns (128-byte rows).
  static constexpr int MASK_BOXES = BN / 16, MASK_BOX_BYTES = BM * 128;
  static constexpr int MASK_BOXES_PER_STAGE = STAGE_BYTES / MASK_BOX_BYTES;
  static constexpr int MASK_STAGES = (MASK_BOXES + MASK_BOXES_PER_STAGE - 1) / MASK_BOXES_PER_STAGE;
  static_assert(MASK_BOXES_PER_STAGE >= 1 && MASK_STAGES <= STAGES, "mask tile must fit the ring");
  static_assert(MASK_BOX_BYTES % 1024 == 0, "swizzled boxes need 1 KB alignment");
  static_assert(A_BYTES % 1024 == 0 && B_BYTES % 1024 == 0, "swizzled tiles need 1 KB alignment");
  static_assert(BM % 16 == 0 && BN % 16 == 0, "tiles are built from 16-wide TMA boxes");
};
// 128 x 128, six 32 KB stages: compute-bound shapes.
using MainCfg = TileCfg<4, 4, 4, 6>;
// 128 x 32, eight 20 KB stages: outputs at most 32 columns wide (the 10 logits).
// All eight warps split the rows, so the MMAs spread over the four SM
// sub-partitions instead of landing on the one that owns a single warp column.
using SkinnyCfg = TileCfg<1, 1, 4, 8>;
// 128 x 16, eight 18 KB stages: outputs at most 16 columns wide.  Such a problem
// streams its tall operand once and is bound by HBM only if the MMAs on padding
// columns stay below the copy time: at 32 columns the 10-logit layer spent 0.52 us
// of tensor-pipe time per k-tile against 0.37 us of copy time, at 16 it is 0.26.
using Skinny16Cfg = TileCfg<1, 1, 2, 8>;
// 128 x 64, eight 24 KB stages: used when 128 x 128 tiles would leave the last
// wave of CTAs mostly empty (e.g. 512 tiles on 148 SMs).
using HalfCfg = TileCfg<2, 2, 4, 8>;
// 112 x 128, six 30 KB stages: eight warps side by side, each 112 rows x 16
// columns.  For outputs whose row count is a multiple of 112 but not of 128
// (784 = 7 x 112, the MNIST-sized input layer's weight gradient), where 128-row
// tiles would spend an eighth of the machine on padding.
using Rows112Cfg = TileCfg<8, 7, 2, 6>;
// 128 x 112, seven 30 KB stages: the same for column counts (the gradient with
// respect to a 784-wide input): 4 x 2 warps of 32 x 56.
using Cols112Cfg = TileCfg<2, 2, 7, 7>;
// 16, 32 and 64 x 128 (eight warps side by side): outputs of few rows, which stream
// their wide operand once.  With 16 rows the MMAs of a k-tile take 0.26 us and its 18 KB
// 0.41 us at an SM's share of HBM; on 128-row tiles the MMAs alone would take 2.1 us.
using Rows16Cfg = TileCfg<8, 1, 2, 10>;
using Rows32Cfg = TileCfg<8, 2, 2, 10>;
using Rows64Cfg = TileCfg<8, 4, 2, 8>;

struct GemmEpilogue {
  double *D;            // output [M][N]
  const double *aux;    // bias[N] or mask source [M][N]
  double *partial;      // packed partial tiles [slot][BM][BN] of split tiles, or null
  int mode;             // MG_EPI_*
  int accumulate;       // D += instead of D =
  // ANYD instantiations only:
  size_t ldd;                // row pitch of D
  const signed char *mask8;  // ReLU mask source in 8 bits, row pitch ld_mask8 (or null)
  size_t ld_mask8;
  int pairs;                 // D's rows all start on 16-byte boundaries
};

// Fragment pair (k = 2c, 2c+1) of the A operand for the MT row sub-tiles of a
// warp: lo = rows g, hi = rows g + 8 of each 16-row sub-tile.
template <bool KCONTIG, int MT>
__device__ __forceinline__ void load_a_frags(const uint8_t *As, int c, int g, int wm,
                                             double2 (&lo)[MT], double2 (&hi)[MT]) {
  if (KCONTIG) {
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
      const int off = (wm + mt * 16 + g) * 128 + ((c ^ g) << 4);
      lo[mt] = *reinterpret_cast<const double2 *>(As + off);
      hi[mt] = *reinterpret_cast<const double2 *>(As + off + 8 * 128);
    }
  } else {
    const int ka = 2 * c, kb = 2 * c + 1;
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
      const int base = ((wm >> 4) + mt) * 2048;
      const int mlo = g, mhi = g + 8;
      lo[mt].x = *reinterpret_cast<const double *>(
          As + base + ka * 128 + ((((mlo >> 1) ^ (ka & 7))) << 4) + (mlo & 1) * 8);
      lo[mt].y = *reinterpret_cast<const double *>(
          As + base + kb * 128 + ((((mlo >> 1) ^ (kb & 7))) << 4) + (mlo & 1) * 8);
      hi[mt].x = *reinterpret_cast<const double *>(
          As + base + ka * 128 + ((((mhi >> 1) ^ (ka & 7))) << 4) + (mhi & 1) * 8);
      hi[mt].y = *reinterpret_cast<const double *>(
          As + base + kb * 128 + ((((mhi >> 1) ^ (kb & 7))) << 4) + (mhi & 1) * 8);
    }
  }
}

// Fragment pair of the B operand for the NT column sub-tiles of a warp (column g).
template <bool KCONTIG, int NT>
__device__ __forceinline__ void load_b_frags(const uint8_t *Bs, int c, int g, int wn,
                                             double2 (&b)[NT]) {
  if (KCONTIG) {
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int off = (wn + nt * 8 + g) * 128 + ((c ^ g) << 4);
      b[nt] = *reinterpret_cast<const double2 *>(Bs + off);
    }
  } else {
    const int ka = 2 * c, kb = 2 * c + 1;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int nl = wn + nt * 8 + g;
      const int base = (nl >> 4) * 2048, nn = nl & 15;
      b[nt].x = *reinterpret_cast<const double *>(
          Bs + base + ka * 128 + ((((nn >> 1) ^ (ka & 7))) << 4) + (nn & 1) * 8);
      b[nt].y = *reinterpret_cast<const double *>(
          Bs + base + kb * 128 + ((((nn >> 1) ^ (kb & 7))) << 4) + (nn & 1) * 8);
    }
  }
}

// One 16-deep stage of MMAs for a warp.
template <bool A_KCONTIG, bool B_KCONTIG, int SHAPE, int MT, int NT>
__device__ __forceinline__ void compute_stage(double (&acc)[MT][NT][4], const uint8_t *As,
                                              const uint8_t *Bs, int c0, int g, int wm, int wn) {
  if (SHAPE == 3) {
    double2 lo0[MT], hi0[MT], b0[NT], lo1[MT], hi1[MT], b1[NT];
    load_a_frags<A_KCONTIG, MT>(As, c0, g, wm, lo0, hi0);
    load_b_frags<B_KCONTIG, NT>(Bs, c0, g, wn, b0);
    load_a_frags<A_KCONTIG, MT>(As, c0 ^ 1, g, wm, lo1, hi1);
    load_b_frags<B_KCONTIG, NT>(Bs, c0 ^ 1, g, wn, b1);
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        dmma_m16n8k16(acc[mt][nt], lo0[mt].x, hi0[mt].x, lo0[mt].y, hi0[mt].y, lo1[mt].x, hi1[mt].x,
                      lo1[mt].y, hi1[mt].y, b0[nt].x, b0[nt].y, b1[nt].x, b1[nt].y);
      }
  } else {
#pragma unroll
    for (int slab = 0; slab < 2; slab++) {
      double2 lo[MT], hi[MT], b[NT];
      load_a_frags<A_KCONTIG, MT>(As, c0 ^ slab, g, wm, lo, hi);
      load_b_frags<B_KCONTIG, NT>(Bs, c0 ^ slab, g, wn, b);
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            if (SHAPE == 2) {
            dmma_m16n8k8(acc[mt][nt], lo[mt].x, hi[mt].x, lo[mt].y, hi[mt].y, b[nt].x, b[nt].y);
          } else if (SHAPE == 1) {
            dmma_m16n8k4(acc[mt][nt], lo[mt].x, hi[mt].x, b[nt].x);
            dmma_m16n8k4(acc[mt][nt], lo[mt].y, hi[mt].y, b[nt].y);
          } else {
            dmma_m8n8k4(acc[mt][nt][0], acc[mt][nt][1], lo[mt].x, b[nt].x);
            dmma_m8n8k4(acc[mt][nt][2], acc[mt][nt][3], hi[mt].x, b[nt].x);
            dmma_m8n8k4(acc[mt][nt][0], acc[mt][nt][1], lo[mt].y, b[nt].y);
            dmma_m8n8k4(acc[mt][nt][2], acc[mt][nt][3], hi[mt].y, b[nt].y);
          }
        }
    }
  }
}

// Consumer side of the stage ring: wait for a stage, run its MMAs, hand the
// stage back.  `active` is false for a warp whose whole sub-block lies outside
// the matrix (ragged border tiles): it skips the arithmetic but keeps the
// barrier protocol.  Returns false if a bounded wait gave up.
template <bool A_KCONTIG, bool B_KCONTIG, int SHAPE, class Cfg>
__device__ __forceinline__ bool consumer_loop(double (&acc)[Cfg::MT][Cfg::NT][4], const uint8_t *smem,
                                              uint64_t *full_bar, uint64_t *empty_bar, int nkt,
                                              unsigned &ring, volatile int *abort_flag, int c0, int g,
                                              int wm, int wn, int lane, bool active) {
  // `ring` counts stages consumed by this CTA since it started; it runs on across
  // the tiles a persistent CTA processes, so stage index and barrier phase follow.
  for (int it = 0; it < nkt; ++it, ++ring) {
    const unsigned s = ring % Cfg::STAGES;
    if (!mbar_wait_bounded(smem_u32(full_bar + s), (ring / Cfg::STAGES) & 1, abort_flag)) return false;
    const uint8_t *As = smem + s * Cfg::STAGE_BYTES;
    const uint8_t *Bs = As + Cfg::A_BYTES;
    if (active)
      compute_stage<A_KCONTIG, B_KCONTIG, SHAPE, Cfg::MT, Cfg::NT>(acc, As, Bs, c0, g, wm, wn);
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(empty_bar + s));
  }
  return true;
}

// SHAPE: 0 m8n8k4, 1 m16n8k4, 2 m16n8k8, 3 m16n8k16.
// EDGE: the problem has ragged tiles (M or N not a multiple of the tile); only
// then is the per-warp skipping compiled in.
// One unit of work of a launch: an output tile and a range of k-tiles.
struct WorkItem {
  int m0, n0, kt_begin, nkt;
  int slot;  // >= 0: write a packed partial tile into this slot; < 0: final epilogue
  // For a segment of a split tile: the tile's first slot, its segment count and
  // its index (which names the tile's arrival counter).
  int first_slot, count, tile;
};

// One segment of a split contraction, as laid out by the host (32 bytes).
struct SegItem {
  int m0, n0, kt_begin, nkt, slot, first_slot, count, tile;
};

// Work order without a segment table: whole tiles, numbered row-major, so the
// thin bottom border of a ragged problem comes last and its short items fill the
// tail instead of pushing full ones into an extra round.
template <class Cfg>
__device__ __forceinline__ WorkItem decode_work(int id, int tiles_n, int KT,
                                                const SegItem *__restrict__ table) {
  WorkItem w;
  if (table) {
    const int4 a = __ldg(reinterpret_cast<const int4 *>(table + id));
    w.m0 = a.x;
    w.n0 = a.y;
    w.kt_begin = a.z;
    w.nkt = a.w;
    const int4 b = __ldg(reinterpret_cast<const int4 *>(table + id) + 1);
    w.slot = b.x;
    w.first_slot = b.y;
    w.count = b.z;
    w.tile = b.w;
    return w;
  }
  const int tile_m = id / tiles_n, tile_n = id - tile_m * tiles_n;
  w.m0 = tile_m * Cfg::BM;
  w.n0 = tile_n * Cfg::BN;
  w.kt_begin = 0;
  w.nkt = KT;
  w.slot = -1;
  w.first_slot = 0;
  w.count = 0;
  w.tile = id;
  return w;
}

// PERSISTENT: the grid has at most one CTA per SM and CTA b processes work items
// b, b + gridDim.x, ...; the producer runs ahead into the next item while the
// consumers are still in the epilogue of the current one, so the pipeline fill
// of an item is hidden behind the previous item's stores.  Used for short items
// (skinny or shallow problems).  Otherwise every CTA processes exactly one item
// and the hardware scheduler balances the load; the loop below then compiles to
// straight-line code, which keeps the consumer's register budget free of spills.
// MASKED: the epilogue is the ReLU mask and its source tile is staged through the
// ring by the producer (a separate instantiation, so that the other epilogues'
// register allocation is untouched).
// FOLD: launches of a split contraction.  Every segment of a split tile stores its
// packed partial tile and then takes a ticket from the tile's arrival counter;
// the segment that arrives last adds up the tile's partial tiles in slot order
// (= k order, whatever the arrival order: the sum is reproducible) and runs the
// final epilogue itself, so no second kernel is needed and the fold of one tile
// overlaps the other CTAs' MMAs.
// ANYD: the output has a row pitch, rows of odd length or a ReLU mask in 8 bits.
template <bool A_KCONTIG, bool B_KCONTIG, int SHAPE, bool EDGE, class Cfg, bool PERSISTENT, bool MASKED,
          bool FOLD, bool ANYD = false>
__global__ void __launch_bounds__(kGemmThreads, 1)
dmma_gemm_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB,
                 const __grid_constant__ CUtensorMap mapMask, GemmEpilogue ep, int M, int N, int K,
                 int tiles_n, const SegItem *__restrict__ table, int grouped_ab, int total_items,
                 unsigned int *tile_tickets, int *status) {
  static_assert(!(MASKED && ANYD), "no such variant");
  constexpr int BM = Cfg::BM, BN = Cfg::BN, MT = Cfg::MT, NT = Cfg::NT;
  constexpr int kStages = Cfg::STAGES, kStageBytes = Cfg::STAGE_BYTES, kTileBytes = Cfg::A_BYTES;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int abort_flag_s;
  __shared__ int fold_last_s;
  volatile int *abort_flag = &abort_flag_s;

  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~static_cast<uintptr_t>(1023));
  uint64_t *full_bar = reinterpret_cast<uint64_t *>(smem + kStages * kStageBytes);
  uint64_t *empty_bar = full_bar + kStages;
  uint64_t *fold_bar = full_bar + 2 * kStages;  // consumer warps meet here around the tile ticket
  static_assert(2 * kStages + 1 == Cfg::kBarriers, "barrier area and its users out of step");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int KT = (K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    abort_flag_s = 0;
    for (int s = 0; s < kStages; s++) {
      mbar_init(smem_u32(full_bar + s), 1);
      mbar_init(smem_u32(empty_bar + s), kConsumerWarps);
    }
    mbar_init(smem_u32(fold_bar), kConsumerWarps);
    mbar_fence_init();
  }
  __syncthreads();

  if (warp >= kConsumerWarps) {
    // ---------------- producer warp group: one lane drives the TMA ring ----------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProducerRegs));
    if (warp == kConsumerWarps && lane == 0) {
      prefetch_tensormap(&mapA);
      prefetch_tensormap(&mapB);
      if (MASKED) prefetch_tensormap(&mapMask);
      unsigned ring = 0;  // stages issued by this CTA so far
      bool alive = true;
      int id = blockIdx.x;
      do {
        const WorkItem w = decode_work<Cfg>(id, tiles_n, KT, table);
        for (int it = 0; it < w.nkt; ++it, ++ring) {
          const unsigned s = ring % kStages;
          if (ring >= (unsigned)kStages) {
            if (!mbar_wait_bounded(smem_u32(empty_bar + s), ((ring / kStages) - 1) & 1, abort_flag)) {
              alive = false;
              break;
            }
          }
          const uint32_t bar = smem_u32(full_bar + s);
          mbar_arrive_expect_tx(bar, kStageBytes);
          const int k0 = (w.kt_begin + it) * BK;
          const uint32_t a_dst = smem_u32(smem + s * kStageBytes);
          const uint32_t b_dst = a_dst + kTileBytes;
          if (A_KCONTIG) {
            tma_load_2d(a_dst, &mapA, k0, w.m0, bar);
          } else if (grouped_ab & 1) {
            tma_load_3d(a_dst, &mapA, 0, k0, w.m0 >> 4, bar);  // all 16-column groups in one copy
          } else {
            for (int b = 0; b < BM / 16; b++)
              tma_load_2d(a_dst + b * 2048, &mapA, w.m0 + 16 * b, k0, bar);
          }
          if (B_KCONTIG) {
            tma_load_2d(b_dst, &mapB, k0, w.n0, bar);
          } else if (grouped_ab & 2) {
            tma_load_3d(b_dst, &mapB, 0, k0, w.n0 >> 4, bar);
          } else {
            for (int b = 0; b < BN / 16; b++)
              tma_load_2d(b_dst + b * 2048, &mapB, w.n0 + 16 * b, k0, bar);
          }
        }
        // The mask source of this tile follows its operands through the ring: the
        // copies overlap the tile's last MMAs and the epilogue reads shared memory.
        if (MASKED && w.slot < 0 && alive) {
          for (int ms = 0; ms < Cfg::MASK_STAGES; ++ms, ++ring) {
            const unsigned s = ring % kStages;
            if (ring >= (unsigned)kStages) {
              if (!mbar_wait_bounded(smem_u32(empty_bar + s), ((ring / kStages) - 1) & 1, abort_flag)) {
                alive = false;
                break;
              }
            }
            const uint32_t bar = smem_u32(full_bar + s);
            const int first = ms * Cfg::MASK_BOXES_PER_STAGE;
            const int boxes = min(Cfg::MASK_BOXES_PER_STAGE, Cfg::MASK_BOXES - first);
            mbar_arrive_expect_tx(bar, (uint32_t)(boxes * Cfg::MASK_BOX_BYTES));
            const uint32_t dst = smem_u32(smem + s * kStageBytes);
            for (int b = 0; b < boxes; b++)
              tma_load_2d(dst + b * Cfg::MASK_BOX_BYTES, &mapMask, w.n0 + 16 * (first + b), w.m0, bar);
          }
        }
        if (!PERSISTENT) break;
        id += gridDim.x;
      } while (alive && id < total_items);
    }
  } else {
    // ---------------- consumer warp groups ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kConsumerRegs));
    const int g = lane >> 2, t = lane & 3;
    const int wm = (warp / Cfg::WARPS_N) * (MT * 16), wn = (warp % Cfg::WARPS_N) * (NT * 8);
    // 16-byte chunk owned by this thread in the first half-slab; the second
    // half-slab uses chunk ^ 1.
    const int c0 = (t << 1) | (__popc(t) & 1);
    unsigned ring = 0;  // stages consumed by this CTA so far
    unsigned fold_phase = 0;  // uses of fold_bar so far

    int id = blockIdx.x;
    do {
      const WorkItem w = decode_work<Cfg>(id, tiles_n, KT, table);
      const int m0 = w.m0, n0 = w.n0;

      double acc[MT][NT][4];
#pragma unroll
      for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
          for (int r = 0; r < 4; r++) acc[i][j][r] = 0.0;

      // Ragged border tiles: a warp whose whole sub-block lies outside the matrix
      // does no arithmetic.  (Skipping at the granularity of single MMAs was
      // measured to be slower than issuing them: the guards break up the
      // instruction stream.)  Out-of-range rows and columns of a live warp read
      // zeros from the TMA fill and are dropped in the epilogue.
      const bool active = !EDGE || (M > m0 + wm && N > n0 + wn);
      const bool ok = consumer_loop<A_KCONTIG, B_KCONTIG, SHAPE, Cfg>(
          acc, smem, full_bar, empty_bar, w.nkt, ring, abort_flag, c0, g, wm, wn, lane, active);
      if (!ok) break;
      // Mask source staged by the producer: wait for all of its stages (every warp,
      // also an inactive one, keeps the ring's barrier protocol).
      const bool mask_smem = MASKED && w.slot < 0;
      const unsigned mask_ring = ring;
      bool mask_ok = true;
      if (mask_smem) {
        for (int ms = 0; ms < Cfg::MASK_STAGES && mask_ok; ms++) {
          const unsigned r2 = mask_ring + ms;
          mask_ok = mbar_wait_bounded(smem_u32(full_bar + r2 % kStages), (r2 / kStages) & 1, abort_flag);
        }
        if (!mask_ok) break;
      }
      // ---------------- epilogue ----------------
      // A segment of a split tile stores its whole BM x BN accumulator, packed,
      // into its slot of the scratch buffer (rows and columns beyond the matrix
      // hold zeros or are never read).
      bool finalize = w.slot < 0;
      if (w.slot >= 0) {
        if (active) {
          double *slot = ep.partial + (size_t)w.slot * (size_t)(BM * BN);
#pragma unroll
          for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
              for (int nt = 0; nt < NT; nt++)
                *reinterpret_cast<double2 *>(slot + (wm + mt * 16 + g + 8 * h) * BN + wn + nt * 8 + 2 * t) =
                    make_double2(acc[mt][nt][2 * h], acc[mt][nt][2 * h + 1]);
        }
        if (FOLD) {
          // All consumer warps' stores are fenced before one thread takes the
          // tile's ticket; the meeting point is an mbarrier with a bounded wait, so
          // a warp that gave up earlier cannot strand the others.
          __threadfence();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(fold_bar));
          if (!mbar_wait_bounded(smem_u32(fold_bar), fold_phase++ & 1, abort_flag)) break;
          if (warp == 0 && lane == 0) {
            const unsigned prev = atomicAdd(tile_tickets + w.tile, 1u);
            const bool last = prev == (unsigned)w.count - 1u;
            if (last) tile_tickets[w.tile] = 0u;  // ready for the next launch (stream-ordered)
            fold_last_s = last ? 1 : 0;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(fold_bar));
          if (!mbar_wait_bounded(smem_u32(fold_bar), fold_phase++ & 1, abort_flag)) break;
          if (fold_last_s) {
            __threadfence();
            if (active) {
#pragma unroll
              for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                  for (int r = 0; r < 4; r++) acc[i][j][r] = 0.0;
              for (int k = 0; k < w.count; k++) {
                const double *part = ep.partial + (size_t)(w.first_slot + k) * (size_t)(BM * BN);
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                  for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                      const double2 v = __ldcg(reinterpret_cast<const double2 *>(
                          part + (wm + mt * 16 + g + 8 * h) * BN + wn + nt * 8 + 2 * t));
                      acc[mt][nt][2 * h] += v.x;
                      acc[mt][nt][2 * h + 1] += v.y;
                    }
              }
            }
            finalize = true;
          }
        }
      }
      // Final epilogue.  Per 16-row sub-tile: first every global load the epilogue
      // needs (ReLU mask source, old values for accumulation) is issued, then the
      // arithmetic, then the stores.  Interleaving load/store pairs would serialise
      // them (a store may alias the next load as far as the compiler can tell) and
      // turn the epilogue into a chain of exposed memory latencies.
      if (active && finalize) {
      if constexpr (ANYD) {
        const bool use_bias = ep.mode == MG_EPI_BIAS || ep.mode == MG_EPI_BIAS_RELU;
        double2 bias[NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          const int col = n0 + wn + nt * 8 + 2 * t;
          bias[nt] = make_double2(use_bias && col < N ? __ldg(ep.aux + col) : 0.0,
                                  use_bias && col + 1 < N ? __ldg(ep.aux + col + 1) : 0.0);
        }
        // Whole pairs in one access each where every pair of the output (and of the mask)
        // starts on its own boundary, single elements otherwise.
        const bool pairs = ep.pairs && !(N & 1);
        constexpr int EG = (MT * NT <= 8) ? MT : 1;  // as below: small tiles fetch everything first
#pragma unroll
        for (int mt0 = 0; mt0 < MT; mt0 += EG) {
          double2 old[EG][2][NT];
          unsigned short codes[EG][2][NT];
          if (ep.accumulate || ep.mask8) {
#pragma unroll
            for (int e = 0; e < EG; e++) {
#pragma unroll
              for (int h = 0; h < 2; h++) {
                const int row = m0 + wm + (mt0 + e) * 16 + g + 8 * h;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                  const int col = n0 + wn + nt * 8 + 2 * t;
                  const bool in0 = row < M && col < N, in1 = row < M && col + 1 < N;
                  old[e][h][nt] = make_double2(0.0, 0.0);
                  codes[e][h][nt] = 0;
                  if (ep.mask8) {
                    const signed char *m = ep.mask8 + (size_t)row * ep.ld_mask8 + col;
                    if (pairs) {
                      if (in0) codes[e][h][nt] = __ldg(reinterpret_cast<const unsigned short *>(m));
                    } else {
                      if (in0) codes[e][h][nt] = (unsigned char)m[0];
                      if (in1) codes[e][h][nt] |= (unsigned short)((unsigned char)m[1] << 8);
                    }
                  }
                  if (ep.accumulate) {
                    const double *src = ep.D + (size_t)row * ep.ldd + col;
                    if (pairs) {
                      if (in0) old[e][h][nt] = __ldcs(reinterpret_cast<const double2 *>(src));
                    } else {
                      if (in0) old[e][h][nt].x = __ldcs(src);
                      if (in1) old[e][h][nt].y = __ldcs(src + 1);
                    }
                  }
                }
              }
            }
          }
#pragma unroll
          for (int e = 0; e < EG; e++) {
            const int mt = mt0 + e;
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const int row = m0 + wm + mt * 16 + g + 8 * h;
              if (row >= M) continue;
#pragma unroll
              for (int nt = 0; nt < NT; nt++) {
                const int col = n0 + wn + nt * 8 + 2 * t;
                if (col >= N) continue;
                double2 v = make_double2(acc[mt][nt][2 * h] + bias[nt].x, acc[mt][nt][2 * h + 1] + bias[nt].y);
                if (ep.mode == MG_EPI_BIAS_RELU) {
                  v.x = v.x > 0 ? v.x : 0.0;
                  v.y = v.y > 0 ? v.y : 0.0;
                }
                if (ep.mask8) {
                  v.x = v.x * ((signed char)codes[e][h][nt] > 0 ? 1.0 : 0.0);
                  v.y = v.y * ((short)codes[e][h][nt] >= 256 ? 1.0 : 0.0);  // (its high byte > 0)
                }
                if (ep.accumulate) {
                  v.x = old[e][h][nt].x + v.x;
                  v.y = old[e][h][nt].y + v.y;
                }
                double *dst = ep.D + (size_t)row * ep.ldd + col;
                if (ep.pairs && col + 1 < N) {
                  *reinterpret_cast<double2 *>(dst) = v;
                } else {
                  dst[0] = v.x;
                  if (col + 1 < N) dst[1] = v.y;
                }
              }
            }
          }
        }
      } else {
      double *dst = ep.D;
      const bool use_mask = ep.mode == MG_EPI_RELU_MASK;
      const bool use_bias = !MASKED && (ep.mode == MG_EPI_BIAS || ep.mode == MG_EPI_BIAS_RELU);
      const bool use_old = ep.accumulate != 0;
      double2 bias[NT];
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        const int col = n0 + wn + nt * 8 + 2 * t;
        bias[nt] = make_double2(0.0, 0.0);
        if (use_bias && col < N) bias[nt] = make_double2(__ldg(ep.aux + col), __ldg(ep.aux + col + 1));
      }
      // Small accumulators (128 x 64 tiles and narrower) leave room to fetch the
      // mask / old values of the whole tile at once: twice the loads in flight,
      // which is what a one-k-tile problem (the gradient through the 10 logits)
      // lives on.  Larger ones go 16 rows at a time.
      constexpr int EG = (MT * NT <= 8) ? MT : 1;
#pragma unroll
      for (int mt0 = 0; mt0 < MT; mt0 += EG) {
        double2 mask[EG][2][NT], old[EG][2][NT];
        if (use_mask || use_old) {
#pragma unroll
          for (int e = 0; e < EG; e++) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const int row = m0 + wm + (mt0 + e) * 16 + g + 8 * h;
#pragma unroll
              for (int nt = 0; nt < NT; nt++) {
                const int col = n0 + wn + nt * 8 + 2 * t;
                const bool in = row < M && col < N;
                const size_t at = (size_t)row * (size_t)N + (size_t)col;
                if (mask_smem) {
                  // box = 16-column group of the tile, 128-byte rows, 16-byte chunks
                  // XOR-swizzled with the row; out-of-range elements were zero-filled.
                  const int r = row - m0, cc = col - n0, box = cc >> 4, chunk = (cc & 15) >> 1;
                  const unsigned st = (mask_ring + box / Cfg::MASK_BOXES_PER_STAGE) % kStages;
                  mask[e][h][nt] = *reinterpret_cast<const double2 *>(
                      smem + st * kStageBytes + (box % Cfg::MASK_BOXES_PER_STAGE) * Cfg::MASK_BOX_BYTES +
                      r * 128 + ((chunk ^ (r & 7)) << 4));
                } else {
                  mask[e][h][nt] = (use_mask && in)
                                       ? __ldcs(reinterpret_cast<const double2 *>(ep.aux + at))
                                       : make_double2(0.0, 0.0);
                }
                old[e][h][nt] = (use_old && in) ? __ldcs(reinterpret_cast<const double2 *>(ep.D + at))
                                                : make_double2(0.0, 0.0);
              }
            }
          }
        }
#pragma unroll
        for (int e = 0; e < EG; e++) {
          const int mt = mt0 + e;
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const int row = m0 + wm + mt * 16 + g + 8 * h;
            if (row >= M) continue;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              const int col = n0 + wn + nt * 8 + 2 * t;
              if (col >= N) continue;
              const size_t at = (size_t)row * (size_t)N + (size_t)col;
              double2 v = make_double2(acc[mt][nt][2 * h], acc[mt][nt][2 * h + 1]);
              if (use_bias) {
                v.x += bias[nt].x;
                v.y += bias[nt].y;
                if (ep.mode == MG_EPI_BIAS_RELU) {
                  v.x = v.x > 0 ? v.x : 0.0;
                  v.y = v.y > 0 ? v.y : 0.0;
                }
              }
              if (use_mask) {
                v.x = v.x * (mask[e][h][nt].x > 0 ? 1.0 : 0.0);
                v.y = v.y * (mask[e][h][nt].y > 0 ? 1.0 : 0.0);
              }
              if (use_old) {
                v.x = old[e][h][nt].x + v.x;
                v.y = old[e][h][nt].y + v.y;
              }
              *reinterpret_cast<double2 *>(dst + at) = v;
            }
          }
        }
      }
      }  // final epilogue
      }  // active
      if (mask_smem) {
        __syncwarp();
        if (lane == 0)
          for (int ms = 0; ms < Cfg::MASK_STAGES; ms++)
            mbar_arrive(smem_u32(empty_bar + (mask_ring + ms) % kStages));
        ring += Cfg::MASK_STAGES;
      }
      if (!PERSISTENT) break;
      id += gridDim.x;
    } while (id < total_items);
  }

  // A bounded wait gave up somewhere in this CTA: raise the fault word, give the
  // copies still in flight time to land in this CTA's shared memory, then leave.
  if (*abort_flag) {
    if (threadIdx.x == 0) atomicExch(status, 201);
    const long long start = clock64();
    while (clock64() - start < 2000000ll) {
    }
  }
}

struct DmmaLaunch {
  CUtensorMap ma, mb, mmask;
  int mask_tma;  // mmask describes the ReLU-mask source; the producer stages it
  GemmEpilogue ep;
  int M, N, K, tiles_m, tiles_n;
  const SegItem *table;  // segments of a split contraction (device), or null: whole tiles
  unsigned int *tickets;  // arrival counters of the split tiles: fold in the kernel; null: no fold
  int items;             // CTAs' worth of work: segments, or tiles
  int min_nkt;           // shortest item, in k-tiles
  int grouped_ab;  // bit 0 / bit 1: operand A / B uses the grouped 3-D tensor map
};

template <bool AK, bool BK_, int SHAPE, bool EDGE, class Cfg, bool PERSISTENT, bool MASKED, bool FOLD,
          bool ANYD = false>
static int launch_dmma_masked(const DmmaLaunch &L) {
  static bool configured = false;
  auto kernel = dmma_gemm_kernel<AK, BK_, SHAPE, EDGE, Cfg, PERSISTENT, MASKED, FOLD, ANYD>;
  if (!configured) {
    MG_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     Cfg::SMEM_BYTES));
    configured = true;
  }
  Context &c = ctx();
  // Long items (many k-tiles) are left to the hardware scheduler, one item per
  // CTA: it balances them dynamically.  Short items (skinny or shallow problems)
  // run as a persistent grid, where the cross-item prefetch hides the pipeline
  // fill that would otherwise dominate them.
  dim3 grid((unsigned)((PERSISTENT && L.items > c.sm_count) ? c.sm_count : L.items), 1, 1);
  kernel<<<grid, kGemmThreads, Cfg::SMEM_BYTES, c.stream>>>(L.ma, L.mb, L.mmask, L.ep, L.M, L.N, L.K,
                                                             L.tiles_n, L.table, L.grouped_ab,
                                                             L.items, L.tickets, c.kernel_status);
  MG_LAUNCH_CHECK("dmma_gemm");
  return MG_OK;
}

// ---------------------------------------------------------------------------
// Planning (gemm.cu)
// ---------------------------------------------------------------------------
enum TileChoice {
  kTileMain = 0, kTileSkinny = 1, kTileHalf = 2, kTileRows112 = 3, kTileSkinny16 = 4, kTileCols112 = 5,
  kTileRows16 = 6, kTileRows32 = 7, kTileRows64 = 8
};

struct GemmPlan {
  int tile, bm, bn, spans;
};

// Segment table of a split contraction (see gemm.cu).
struct SegTable {
  int tiles_m, tiles_n, KT, bm, bn, spans;  // key
  int items, slots, min_nkt;
  SegItem *dev_items;  // [items], longest first
  unsigned int *dev_tickets;  // [tiles]: arrival counters of the in-kernel fold, zero between launches
  int2 *dev_tiles;            // [tiles]: first slot and segment count of a split tile, (0, 0) of a whole one
  bool recorded;              // a recorded step reads it
};

int choose_spans(int tiles, int KT, int sms);
int seg_table_for(int tiles_m, int tiles_n, int KT, int bm, int bn, int spans, const SegTable **out);

}  // namespace mg
