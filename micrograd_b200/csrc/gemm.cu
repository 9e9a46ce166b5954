// fp64 matrix multiply: forward C = A.B (src/ops/Matmul.cpp:30-38) and the two
// gradient products dA += G.B^T (:44-50) and dB += A^T.G (:52-58).
//
// Main kernel: FP64 tensor-core (DMMA, mma.sync ... f64) tiles fed by TMA.
//   - Eight consumer warps and one producer warp group per CTA (registers re-split
//     with setmaxnreg); a ring of stages filled by cp.async.bulk.tensor and handed
//     over through full/empty mbarriers.  Tile configurations (TileCfg): 128 x 128
//     (2 x 4 warps of 64 x 32) for the compute-bound shapes, 128 x 64 when that
//     fills the last wave of CTAs better or the contraction is a single k-tile,
//     128 x 32 and 128 x 16 for outputs at most that many columns wide, 112 x 128
//     for row counts that are multiples of 112 but not of 128.
//   - Operands land in shared memory in the 128-byte swizzle.  With the k index
//     of a 16-deep slab permuted (the same permutation for A and B, so the sum is
//     unchanged) every fragment load is free of bank conflicts: a thread reads
//     16-byte chunk c = {0,3,5,6}[t] (first half of the slab) or c^1 (second
//     half), i.e. k = 2c and 2c+1, for all three operand layouts:
//        k-contiguous tile  [row][16 k]      : one 16-byte load per fragment pair
//        mn-contiguous tile [16-col group][k][16 cols] : 8-byte loads
//   - The accumulators stay in registers (FP64 MMA has no TMEM form); the
//     epilogue adds the bias, applies ReLU or the ReLU mask, and stores or
//     accumulates 16 bytes per thread per row, all loads before the stores.  The
//     mask source tile of the input-gradient product follows the operands
//     through the TMA ring, so its copy overlaps the tile's last MMAs.
//   - When the output has too few tiles to fill 148 SMs (weight gradients: the
//     contraction runs over the batch), the (tile, k-tile) iteration space is cut
//     into one equal span per SM; a span that crosses a tile boundary becomes two
//     segments.  Every segment is one CTA; segments are issued longest first, so
//     the hardware scheduler pairs each SM's long piece with the complementary
//     short one and all SMs finish together.  A tile covered by several segments
//     is written as packed partial tiles; the segment that finishes last (a
//     ticket per tile) adds them up in k order, whatever the arrival order, and
//     runs the epilogue, so the result is reproducible and no second kernel runs.
//   - Short work items run as a persistent grid (one CTA per SM looping over
//     items, the producer prefetching across items); long ones as one item per
//     CTA under the hardware scheduler.
// Fallback kernel: a plain shared-memory tiled FMA kernel with full bounds
// checks for shapes the TMA path cannot take (odd row lengths, unaligned
// bases) and for tiny problems.
#include "gemm_kernel.cuh"

#include <algorithm>
#include <cstdlib>
#include <type_traits>
#include <vector>

namespace mg {

// ---------------------------------------------------------------------------
// Fallback: D[m,n] (+)= sum_k A(m,k) B(k,n) with arbitrary element strides.
// 64 x 64 x 16 tiles, 256 threads, 4 x 4 outputs per thread, full bounds checks.
// ---------------------------------------------------------------------------
struct StridedOperands {
  const double *A;
  const double *B;
  long long sAm, sAk, sBk, sBn;
};

__global__ void __launch_bounds__(256)
gemm_fallback_kernel(StridedOperands op, GemmEpilogue ep, int M, int N, int K) {
  constexpr int TM = 64, TN = 64, TK = 16;
  __shared__ double As[TK][TM + 1];
  __shared__ double Bs[TK][TN + 1];
  const int tid = threadIdx.x;
  const int m0 = blockIdx.y * TM, n0 = blockIdx.x * TN;
  const int ty = tid / 16, tx = tid % 16;  // thread owns rows ty*4.., cols tx*4..
  double acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[i][j] = 0.0;

  const bool a_k_fast = (op.sAk == 1);
  const bool b_n_fast = (op.sBn == 1);
  for (int k0 = 0; k0 < K; k0 += TK) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int idx = tid + e * 256;  // 0..1023
      int m, k;
      if (a_k_fast) { m = idx / TK; k = idx % TK; } else { m = idx % TM; k = idx / TM; }
      const int gm = m0 + m, gk = k0 + k;
      As[k][m] = (gm < M && gk < K) ? op.A[(long long)gm * op.sAm + (long long)gk * op.sAk] : 0.0;
      int n, kk;
      if (b_n_fast) { n = idx % TN; kk = idx / TN; } else { n = idx / TK; kk = idx % TK; }
      const int gn = n0 + n, gk2 = k0 + kk;
      Bs[kk][n] = (gn < N && gk2 < K) ? op.B[(long long)gk2 * op.sBk + (long long)gn * op.sBn] : 0.0;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < TK; k++) {
      double a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; i++) a[i] = As[k][ty * 4 + i];
#pragma unroll
      for (int j = 0; j < 4; j++) b[j] = Bs[k][tx * 4 + j];
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = fma(a[i], b[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int row = m0 + ty * 4 + i;
    if (row >= M) continue;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int col = n0 + tx * 4 + j;
      if (col >= N) continue;
      const size_t at = (size_t)row * (size_t)N + (size_t)col;
      double v = acc[i][j];
      if (ep.mode == MG_EPI_BIAS || ep.mode == MG_EPI_BIAS_RELU) {
        v += ep.aux[col];
        if (ep.mode == MG_EPI_BIAS_RELU) v = v > 0 ? v : 0.0;
      } else if (ep.mode == MG_EPI_RELU_MASK) {
        v = v * (ep.aux[at] > 0 ? 1.0 : 0.0);
      }
      if (ep.accumulate) v = ep.D[at] + v;
      ep.D[at] = v;
    }
  }
}

// ---------------------------------------------------------------------------
// Host dispatch
// ---------------------------------------------------------------------------
static int g_gemm_path = 0;    // 0 auto, 1 fallback only, 2 tensor-core whenever eligible
static int g_dmma_shape = -1;  // -1: default

static int default_dmma_shape() {
  const char *v = std::getenv("MG_DMMA_SHAPE");
  if (v && *v) {
    int s = std::atoi(v);
    if (s >= 0 && s <= 3) return s;
  }
  return 2;
}

// The staged-mask instantiation exists for the default mma shape and the layout
// of the input-gradient product (both operands k-contiguous), its only user.
template <bool AK, bool BK_, int SHAPE, bool EDGE, class Cfg, bool PERSISTENT>
static int launch_dmma_variant(const DmmaLaunch &L) {
  if constexpr (AK && BK_ && SHAPE == 2) {
    if (L.mask_tma) return launch_dmma_masked<AK, BK_, SHAPE, EDGE, Cfg, PERSISTENT, true, false>(L);
  }
  // The folding instantiation serves split contractions only: they never run
  // persistently and read their mask (if any) with plain loads.
  if constexpr (!PERSISTENT) {
    if (L.tickets) return launch_dmma_masked<AK, BK_, SHAPE, EDGE, Cfg, false, false, true>(L);
  }
  return launch_dmma_masked<AK, BK_, SHAPE, EDGE, Cfg, PERSISTENT, false, false>(L);
}

template <bool AK, bool BK_, int SHAPE, bool EDGE, class Cfg>
static int launch_dmma_kernel(const DmmaLaunch &L) {
  static const int persist_mode = [] {
    const char *v = std::getenv("MG_GEMM_PERSIST");  // diagnostic: 0 never, 1 always
    return v && *v ? std::atoi(v) : -1;
  }();
  // Segments of a split contraction have unequal lengths and rely on the
  // hardware scheduler's longest-first pairing, so they never run persistently.
  bool persistent = !L.table && (L.min_nkt < 32 || Cfg::BN <= 32) && L.items > ctx().sm_count;
  if (persist_mode == 0) persistent = false;
  if (persist_mode == 1 && !L.table && L.items > ctx().sm_count) persistent = true;
  if (persistent) return launch_dmma_variant<AK, BK_, SHAPE, EDGE, Cfg, true>(L);
  return launch_dmma_variant<AK, BK_, SHAPE, EDGE, Cfg, false>(L);
}

// One launch over all tiles; problems with a ragged border use the instantiation
// that can skip out-of-range sub-tiles.
template <bool AK, bool BK_, int SHAPE, class Cfg>
static int launch_tiles(const DmmaLaunch &L) {
  if ((L.M % Cfg::BM) != 0 || (L.N % Cfg::BN) != 0)
    return launch_dmma_kernel<AK, BK_, SHAPE, true, Cfg>(L);
  return launch_dmma_kernel<AK, BK_, SHAPE, false, Cfg>(L);
}

template <bool AK, bool BK_>
static int launch_layout(int shape, int tile, const DmmaLaunch &L) {
  // The narrow and half-width configurations exist for the default mma shape only.
  if (tile == kTileSkinny)
    return launch_dmma_kernel<AK, BK_, 2, true, SkinnyCfg>(L);
  if (tile == kTileSkinny16)
    return launch_dmma_kernel<AK, BK_, 2, true, Skinny16Cfg>(L);
  if (tile == kTileHalf) return launch_tiles<AK, BK_, 2, HalfCfg>(L);
  if (tile == kTileRows112) return launch_tiles<AK, BK_, 2, Rows112Cfg>(L);
  if (tile == kTileCols112) return launch_tiles<AK, BK_, 2, Cols112Cfg>(L);
  switch (shape) {
    case 0: return launch_tiles<AK, BK_, 0, MainCfg>(L);
    case 1: return launch_tiles<AK, BK_, 1, MainCfg>(L);
    case 3: return launch_tiles<AK, BK_, 3, MainCfg>(L);
    default: return launch_tiles<AK, BK_, 2, MainCfg>(L);
  }
}

// Number of equal spans the (tile, k-tile) iteration space of a problem is cut
// into, or 0 to run whole tiles.  Whole tiles are kept when they already fill
// at least 95% of their last wave of CTAs, or when the contraction is too short
// to share; otherwise one span per SM, at least 16 k-tiles long.
int choose_spans(int tiles, int KT, int sms) {
  if (tiles >= 4 * sms || KT < 32) return 0;
  const int waves = (tiles + sms - 1) / sms;
  if ((double)tiles / ((double)waves * sms) >= 0.95) return 0;
  long long spans = (long long)tiles * KT / 16;
  if (spans > sms) spans = sms;
  return spans > 1 ? (int)spans : 0;
}

// Tile configuration and contraction split for a problem.  Candidates are
// costed as (rounds of CTAs) x (work per CTA), with a small handicap for the
// half-width tile (more operand traffic per flop) and for a split contraction
// (its partial tiles are written and folded: ~22.8 (p+1)/K of the GEMM's time
// when p partial tiles are written per output tile).
static GemmPlan choose_plan(int M, int N, int K, int sms, int shape) {
  const int KT = (K + BK - 1) / BK;
  auto tiles_of = [&](int bm, int bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
  if (N <= Skinny16Cfg::BN) {
    return {kTileSkinny16, Skinny16Cfg::BM, Skinny16Cfg::BN,
            choose_spans(tiles_of(Skinny16Cfg::BM, Skinny16Cfg::BN), KT, sms)};
  }
  if (N <= SkinnyCfg::BN) {
    return {kTileSkinny, SkinnyCfg::BM, SkinnyCfg::BN,
            choose_spans(tiles_of(SkinnyCfg::BM, SkinnyCfg::BN), KT, sms)};
  }
  GemmPlan main_plan{kTileMain, MainCfg::BM, MainCfg::BN,
                     choose_spans(tiles_of(MainCfg::BM, MainCfg::BN), KT, sms)};
  static const int forced = [] {
    const char *v = std::getenv("MG_GEMM_TILE");  // diagnostic: "main" or "half"
    if (!v) return -1;
    return v[0] == 'h' ? (int)kTileHalf : (v[0] == 'm' ? (int)kTileMain : -1);
  }();
  if (shape != 2 || forced == kTileMain) return main_plan;
  GemmPlan half_plan{kTileHalf, HalfCfg::BM, HalfCfg::BN,
                     choose_spans(tiles_of(HalfCfg::BM, HalfCfg::BN), KT, sms)};
  if (forced == kTileHalf) return half_plan;
  // One k-tile: the problem is all epilogue (a rank-16 update streamed through
  // HBM); the half-width tile keeps the whole tile's epilogue loads in flight.
  if (KT == 1) return half_plan;
  // Every CTA also pays about 3.3 us of launch, pipeline fill and epilogue that
  // nothing overlaps: 25 800 in the cost's units (bm x bn x k-tiles).
  constexpr double kPerCta = 25800.0;
  auto cost = [&](const GemmPlan &p, double handicap) {
    const int tiles = tiles_of(p.bm, p.bn);
    if (p.spans == 0) {
      const int waves = (tiles + sms - 1) / sms;
      return (double)waves * ((double)p.bm * p.bn * KT * handicap + kPerCta);
    }
    const double per_cta = (double)tiles * KT / p.spans;
    const double segments = (double)tiles / p.spans + 1.0;
    const double partials = std::min(2.0 * p.spans, (double)p.spans + tiles) / tiles;
    double c = (per_cta * p.bm * p.bn * handicap + segments * kPerCta) *
               (1.0 + 22.8 * (partials + 1.0) / (double)K);
    // With more tiles than SMs most segments are whole tiles and the cut ones
    // lose the L2 sharing of a wave that walks k in step: measured 2 % behind
    // the half-width tile where the model calls it even.
    if (tiles >= sms) c *= 1.04;
    return c;
  };
  GemmPlan best = cost(half_plan, 1.04) < cost(main_plan, 1.0) ? half_plan : main_plan;
  double best_cost = best.tile == kTileHalf ? cost(half_plan, 1.04) : cost(main_plan, 1.0);
  if (M % MainCfg::BM != 0 && M % Rows112Cfg::BM == 0) {
    GemmPlan p112{kTileRows112, Rows112Cfg::BM, Rows112Cfg::BN,
                  choose_spans(tiles_of(Rows112Cfg::BM, Rows112Cfg::BN), KT, sms)};
    if (cost(p112, 1.02) < best_cost) {
      best = p112;
      best_cost = cost(p112, 1.02);
    }
  }
  if (N % MainCfg::BN != 0 && N % Cols112Cfg::BN == 0) {
    GemmPlan c112{kTileCols112, Cols112Cfg::BM, Cols112Cfg::BN,
                  choose_spans(tiles_of(Cols112Cfg::BM, Cols112Cfg::BN), KT, sms)};
    if (cost(c112, 1.02) < best_cost) best = c112;
  }
  return best;
}

// ---------------------------------------------------------------------------
// Segment tables of split contractions.  A table depends only on the tile grid,
// the k-tile count and the span count, so it is built once per shape and kept
// on the device: the 256 latest ones, and those that the kernels of a recorded step
// read (their addresses are part of the step) as long as any step exists.
// ---------------------------------------------------------------------------
static std::vector<SegTable> g_seg_tables;
constexpr size_t kMostTables = 256;

static void release_tables(bool recorded_too) {
  std::vector<SegTable> kept;
  for (auto &t : g_seg_tables) {
    if (t.recorded && !recorded_too) {
      kept.push_back(t);
      continue;
    }
    cudaFree(t.dev_items);
    cudaFree(t.dev_tickets);
    cudaFree(t.dev_tiles);
  }
  g_seg_tables.swap(kept);
}

void gemm_release_tables() { release_tables(true); }

// After a kernel fault (a bounded wait gave up) a split tile may be left with a
// partly counted ticket; clear them all so later launches start clean.
void gemm_reset_tickets() {
  for (auto &t : g_seg_tables)
    cudaMemsetAsync(t.dev_tickets, 0, sizeof(unsigned int) * (size_t)(t.tiles_m * t.tiles_n), ctx().stream);
}

// Host-only construction of a segment table: `segs` in issue order (longest
// first), `tile_info[t]` = (first slot, segment count) of every tile covered by
// more than one segment, (0, 0) otherwise.  Slots number the segments of split
// tiles in (tile, k) order, so a tile's partial tiles are consecutive and in k order.
static void build_segments(int tiles_m, int tiles_n, int KT, int bm, int bn, int spans,
                           std::vector<SegItem> &segs, std::vector<int2> &tile_info, int &slots,
                           int &min_nkt) {
  const int tiles = tiles_m * tiles_n;
  const long long units = (long long)tiles * KT;
  segs.clear();
  std::vector<int> per_tile((size_t)tiles, 0);
  for (int j = 0; j < spans; j++) {
    long long u = units * j / spans;
    const long long end = units * (j + 1) / spans;
    while (u < end) {
      const int tile = (int)(u / KT);
      const int kt = (int)(u - (long long)tile * KT);
      const int n = (int)std::min<long long>(end - u, KT - kt);
      SegItem it{};
      it.m0 = (tile / tiles_n) * bm;
      it.n0 = (tile % tiles_n) * bn;
      it.kt_begin = kt;
      it.nkt = n;
      it.slot = tile;  // provisional: the tile index
      segs.push_back(it);
      per_tile[(size_t)tile]++;
      u += n;
    }
  }
  tile_info.assign((size_t)tiles, make_int2(0, 0));
  slots = 0;
  min_nkt = KT;
  for (auto &it : segs) {
    const int tile = it.slot;
    it.tile = tile;
    if (per_tile[(size_t)tile] > 1) {
      if (tile_info[(size_t)tile].y == 0) tile_info[(size_t)tile].x = slots;
      tile_info[(size_t)tile].y++;
      it.slot = slots++;
    } else {
      it.slot = -1;
    }
    min_nkt = std::min(min_nkt, it.nkt);
  }
  for (auto &it : segs) {
    it.first_slot = tile_info[(size_t)it.tile].x;
    it.count = tile_info[(size_t)it.tile].y;
  }
  std::stable_sort(segs.begin(), segs.end(),
                   [](const SegItem &a, const SegItem &b) { return a.nkt > b.nkt; });
}

int seg_table_for(int tiles_m, int tiles_n, int KT, int bm, int bn, int spans,
                         const SegTable **out) {
  for (auto &t : g_seg_tables) {
    if (t.tiles_m == tiles_m && t.tiles_n == tiles_n && t.KT == KT && t.bm == bm && t.bn == bn &&
        t.spans == spans) {
      t.recorded = t.recorded || ctx().capturing;
      *out = &t;
      return MG_OK;
    }
  }
  if (ctx().capturing)
    return fail(MG_ERR_INVALID,
                "a GEMM of a new shape needs its segment table built while a step is being recorded; "
                "run the step once before mg_graph_begin()");
  // A job with ever-changing shapes (e.g. a varying batch) would grow the cache
  // without bound: start over beyond 256 tables (cudaFree waits for the kernels
  // that still read them).
  size_t loose = 0;
  for (const auto &t : g_seg_tables) loose += t.recorded ? 0 : 1;
  if (loose >= kMostTables) release_tables(mg_graph_count() == 0);
  std::vector<SegItem> segs;
  std::vector<int2> tile_info;
  int slots = 0, min_nkt = KT;
  build_segments(tiles_m, tiles_n, KT, bm, bn, spans, segs, tile_info, slots, min_nkt);
  SegTable t{};
  t.tiles_m = tiles_m; t.tiles_n = tiles_n; t.KT = KT; t.bm = bm; t.bn = bn; t.spans = spans;
  t.items = (int)segs.size();
  t.slots = slots;
  t.min_nkt = min_nkt;
  MG_CUDA_TRY(cudaMalloc(&t.dev_items, segs.size() * sizeof(SegItem)));
  MG_CUDA_TRY(cudaMalloc(&t.dev_tickets, tile_info.size() * sizeof(unsigned int)));
  MG_CUDA_TRY(cudaMalloc(&t.dev_tiles, tile_info.size() * sizeof(int2)));
  MG_CUDA_TRY(cudaMemcpy(t.dev_tiles, tile_info.data(), tile_info.size() * sizeof(int2), cudaMemcpyHostToDevice));
  MG_CUDA_TRY(cudaMemset(t.dev_tickets, 0, tile_info.size() * sizeof(unsigned int)));
  MG_CUDA_TRY(cudaMemcpy(t.dev_items, segs.data(), segs.size() * sizeof(SegItem),
                         cudaMemcpyHostToDevice));
  g_seg_tables.push_back(t);
  *out = &g_seg_tables.back();
  return MG_OK;
}

static bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static bool dmma_eligible(const GemmDesc &d) {
  const size_t a_row = d.a_kcontig ? d.K : d.M;
  const size_t b_row = d.b_kcontig ? d.K : d.N;
  if ((a_row | b_row | d.N) & 1) return false;
  if (!aligned16(d.A) || !aligned16(d.B) || !aligned16(d.D)) return false;
  if (d.mode == MG_EPI_RELU_MASK && !aligned16(d.aux)) return false;
  const size_t lim = (size_t)1 << 30;
  if (d.M >= lim || d.N >= lim || d.K >= lim) return false;
  return true;
}

int run_gemm(const GemmDesc &d) {
  if (d.M == 0 || d.N == 0) return MG_OK;
  Context &c = ctx();
  GemmEpilogue ep{};
  ep.D = d.D;
  ep.aux = d.aux;
  ep.partial = nullptr;
  ep.mode = d.mode;
  ep.accumulate = d.accumulate;
  if ((d.mode == MG_EPI_BIAS || d.mode == MG_EPI_BIAS_RELU || d.mode == MG_EPI_RELU_MASK) && !d.aux)
    return fail(MG_ERR_INVALID, "gemm: epilogue %d needs its auxiliary operand", d.mode);
  if (d.K == 0) {
    // Empty contraction: the product is all zeros; only the epilogue remains.
    if (d.accumulate && d.mode == MG_EPI_NONE) return MG_OK;
    if (d.accumulate && d.mode == MG_EPI_RELU_MASK) return MG_OK;
  }

  bool use_dmma = dmma_eligible(d) && d.K > 0;
  if (g_gemm_path == 1) use_dmma = false;
  // Below M.N.K = 512 the plain kernel is used.  The bar used to be 64^3; measured on
  // the launch-bound steps (batch-32 training step: 112.6 -> 97.3 us, recorded 83.9 ->
  // 69.6 us; the per-sample trainer loop: 5.6 k -> 7.6 k samples/s), one CTA of the
  // tensor-core kernel finishes a tiny product in less time than the plain
  // kernel's chain of dependent 16-deep global loads.
  static const size_t min_dmma_volume = [] {
    const char *v = std::getenv("MG_GEMM_MIN_VOLUME");  // diagnostic
    return v && *v ? (size_t)std::atoll(v) : (size_t)512;
  }();
  if (g_gemm_path == 0 && use_dmma && d.M * d.N * d.K < min_dmma_volume) use_dmma = false;

  const int M = (int)d.M, N = (int)d.N, K = (int)d.K;
  if (!use_dmma) {
    if (d.M >= ((size_t)1 << 31) || d.N >= ((size_t)1 << 31) || d.K >= ((size_t)1 << 31))
      return fail(MG_ERR_INVALID, "gemm: dimension too large");
    StridedOperands op;
    op.A = d.A;
    op.B = d.B;
    if (d.a_kcontig) { op.sAm = (long long)d.K; op.sAk = 1; } else { op.sAm = 1; op.sAk = (long long)d.M; }
    if (d.b_kcontig) { op.sBk = 1; op.sBn = (long long)d.K; } else { op.sBk = (long long)d.N; op.sBn = 1; }
    dim3 grid((unsigned)((N + 63) / 64), (unsigned)((M + 63) / 64));
    if (grid.y > 65535) return fail(MG_ERR_INVALID, "gemm fallback: too many row tiles (%u)", grid.y);
    gemm_fallback_kernel<<<grid, 256, 0, c.stream>>>(op, ep, M, N, K);
    MG_LAUNCH_CHECK("gemm_fallback");
    return MG_OK;
  }

  const int shape = g_dmma_shape >= 0 ? g_dmma_shape : default_dmma_shape();
  const GemmPlan plan = choose_plan(M, N, K, c.sm_count, shape);
  const int bm = plan.bm, bn = plan.bn;
  DmmaLaunch L{};
  // Operands whose contiguous axis is m or n arrive as 16-column groups.  When the
  // row length is a multiple of 16 one 3-D copy per stage brings all groups of the
  // tile; otherwise each group is its own 2-D copy.
  L.grouped_ab = 0;
  bool ok_a, ok_b;
  if (d.a_kcontig) {
    ok_a = make_tensor_map_f64(&L.ma, d.A, d.M, d.K, BK, bm);
  } else if (d.M % 16 == 0 && make_tensor_map_f64_grouped(&L.ma, d.A, d.K, d.M, BK, bm / 16)) {
    ok_a = true;
    L.grouped_ab |= 1;
  } else {
    ok_a = make_tensor_map_f64(&L.ma, d.A, d.K, d.M, 16, BK);
  }
  if (d.b_kcontig) {
    ok_b = make_tensor_map_f64(&L.mb, d.B, d.N, d.K, BK, bn);
  } else if (d.N % 16 == 0 && make_tensor_map_f64_grouped(&L.mb, d.B, d.K, d.N, BK, bn / 16)) {
    ok_b = true;
    L.grouped_ab |= 2;
  } else {
    ok_b = make_tensor_map_f64(&L.mb, d.B, d.K, d.N, 16, BK);
  }
  if (!ok_a || !ok_b) return fail(MG_ERR_CUDA, "gemm: cuTensorMapEncodeTiled failed");
  // ReLU-mask source [M][N]: boxes of bm rows x 16 columns.  If the map cannot be
  // built the epilogue reads the mask with plain loads instead.
  L.mmask = L.ma;
  L.mask_tma = (d.mode == MG_EPI_RELU_MASK && d.a_kcontig && d.b_kcontig && shape == 2 &&
                make_tensor_map_f64(&L.mmask, d.aux, d.M, d.N, 16, bm))
                   ? 1 : 0;

  const int tiles_m = (M + bm - 1) / bm, tiles_n = (N + bn - 1) / bn;
  const int KT = (K + BK - 1) / BK;
  const SegTable *table = nullptr;
  if (plan.spans > 0) {
    int rc = seg_table_for(tiles_m, tiles_n, KT, bm, bn, plan.spans, &table);
    if (rc != MG_OK) return rc;
    if (table->slots > 0) {
      rc = ensure_scratch(&c.splitk_scratch, &c.splitk_scratch_elems,
                          (size_t)table->slots * (size_t)bm * (size_t)bn);
      if (rc != MG_OK) return rc;
      ep.partial = c.splitk_scratch;
    }
  }
  L.ep = ep;
  L.M = M; L.N = N; L.K = K;
  L.tiles_m = tiles_m; L.tiles_n = tiles_n;
  L.table = table ? table->dev_items : nullptr;
  // Split tiles are folded inside the kernel by their last-arriving segment.
  const bool fold = table && table->slots > 0;
  L.tickets = fold ? table->dev_tickets : nullptr;
  if (fold) L.mask_tma = 0;
  L.items = table ? table->items : tiles_m * tiles_n;
  L.min_nkt = table ? table->min_nkt : KT;
  int rc;
  if (d.a_kcontig && !d.b_kcontig)
    rc = launch_layout<true, false>(shape, plan.tile, L);
  else if (d.a_kcontig && d.b_kcontig)
    rc = launch_layout<true, true>(shape, plan.tile, L);
  else if (!d.a_kcontig && !d.b_kcontig)
    rc = launch_layout<false, false>(shape, plan.tile, L);
  else
    return fail(MG_ERR_INVALID, "gemm: unsupported operand layout");
  if (rc != MG_OK) return rc;
  return MG_OK;
}

}  // namespace mg

using namespace mg;

extern "C" {

int mg_gemm_plan_describe(size_t M, size_t N, size_t K, int sm_count, int *plan5, int *segments,
                          int max_segments) {
  if (!plan5 || M == 0 || N == 0 || K == 0 || sm_count < 1 || M >= ((size_t)1 << 30) ||
      N >= ((size_t)1 << 30) || K >= ((size_t)1 << 30))
    return fail(MG_ERR_INVALID, "mg_gemm_plan_describe: bad arguments");
  const GemmPlan plan = choose_plan((int)M, (int)N, (int)K, sm_count, 2);
  const int tiles_m = ((int)M + plan.bm - 1) / plan.bm, tiles_n = ((int)N + plan.bn - 1) / plan.bn;
  const int KT = ((int)K + BK - 1) / BK;
  plan5[0] = plan.bm;
  plan5[1] = plan.bn;
  plan5[2] = plan.spans;
  plan5[3] = tiles_m * tiles_n;
  plan5[4] = 0;
  if (plan.spans == 0) return MG_OK;
  std::vector<SegItem> segs;
  std::vector<int2> tile_info;
  int slots = 0, min_nkt = 0;
  build_segments(tiles_m, tiles_n, KT, plan.bm, plan.bn, plan.spans, segs, tile_info, slots, min_nkt);
  plan5[3] = (int)segs.size();
  plan5[4] = slots;
  if (segments) {
    if ((int)segs.size() > max_segments)
      return fail(MG_ERR_INVALID, "mg_gemm_plan_describe: %zu segments, room for %d", segs.size(),
                  max_segments);
    for (size_t i = 0; i < segs.size(); i++) {
      segments[5 * i + 0] = segs[i].m0;
      segments[5 * i + 1] = segs[i].n0;
      segments[5 * i + 2] = segs[i].kt_begin;
      segments[5 * i + 3] = segs[i].nkt;
      segments[5 * i + 4] = segs[i].slot;
    }
  }
  return MG_OK;
}

int mg_gemm_config(int path, int dmma_shape) {
  if (path < 0 || path > 2) return fail(MG_ERR_INVALID, "mg_gemm_config: path must be 0, 1 or 2");
  if (dmma_shape < -1 || dmma_shape > 3)
    return fail(MG_ERR_INVALID, "mg_gemm_config: shape must be -1..3");
  g_gemm_path = path;
  g_dmma_shape = dmma_shape;
  return MG_OK;
}

int mg_gemm_nn(const double *A, const double *B, double *C, size_t M, size_t N, size_t K,
               int accumulate, int epilogue, const double *bias) {
  MG_ENSURE_INIT();
  if (M && N && (!C || (K && (!A || !B)))) return fail(MG_ERR_INVALID, "mg_gemm_nn: null pointer");
  if (epilogue != MG_EPI_NONE && epilogue != MG_EPI_BIAS && epilogue != MG_EPI_BIAS_RELU)
    return fail(MG_ERR_INVALID, "mg_gemm_nn: epilogue %d not valid here", epilogue);
  GemmDesc d{A, B, C, M, N, K, true, false, accumulate, epilogue, bias};
  return run_gemm(d);
}

int mg_gemm_nt(const double *G, const double *B, double *dA, size_t M, size_t N, size_t K,
               int accumulate, int epilogue, const double *mask_src) {
  MG_ENSURE_INIT();
  if (M && K && (!dA || (N && (!G || !B)))) return fail(MG_ERR_INVALID, "mg_gemm_nt: null pointer");
  if (epilogue != MG_EPI_NONE && epilogue != MG_EPI_RELU_MASK)
    return fail(MG_ERR_INVALID, "mg_gemm_nt: epilogue %d not valid here", epilogue);
  // Output [M][K]; contraction over N; G is [M][N] (k-contiguous), B is [K][N]
  // (output-column major, k-contiguous).
  GemmDesc d{G, B, dA, M, K, N, true, true, accumulate, epilogue, mask_src};
  return run_gemm(d);
}

int mg_gemm_tn(const double *A, const double *G, double *dB, size_t M, size_t N, size_t K,
               int accumulate) {
  MG_ENSURE_INIT();
  if (K && N && (!dB || (M && (!A || !G)))) return fail(MG_ERR_INVALID, "mg_gemm_tn: null pointer");
  // Output [K][N]; contraction over M; A is [M][K] (output-row contiguous),
  // G is [M][N] (output-column contiguous).
  GemmDesc d{A, G, dB, K, N, M, false, false, accumulate, MG_EPI_NONE, nullptr};
  return run_gemm(d);
}

}  // extern "C"
