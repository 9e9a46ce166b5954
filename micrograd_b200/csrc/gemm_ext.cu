// The tensor-core GEMM of gemm.cu for callers whose matrices are not dense even rows:
// see run_gemm_ext in gemm.cuh.
#include "gemm_kernel.cuh"

namespace mg {

// One instantiation per tile, contraction split and grid form; all can skip the
// ragged border (EDGE) and write any output (ANYD).
template <bool AK, bool BK_, class Cfg> static int launch_ext(const DmmaLaunch &L) {
  if (L.tickets) return launch_dmma_masked<AK, BK_, 2, true, Cfg, false, false, true, true>(L);
  if (!L.table && (L.min_nkt < 32 || Cfg::BN <= 32) && L.items > ctx().sm_count)
    return launch_dmma_masked<AK, BK_, 2, true, Cfg, true, false, false, true>(L);
  return launch_dmma_masked<AK, BK_, 2, true, Cfg, false, false, false, true>(L);
}

template <bool AK, bool BK_> static int launch_layout_ext(int tile, const DmmaLaunch &L) {
  switch (tile) {
    case kTileSkinny: return launch_ext<AK, BK_, SkinnyCfg>(L);
    case kTileSkinny16: return launch_ext<AK, BK_, Skinny16Cfg>(L);
    case kTileHalf: return launch_ext<AK, BK_, HalfCfg>(L);
    case kTileRows16: return launch_ext<AK, BK_, Rows16Cfg>(L);
    case kTileRows32: return launch_ext<AK, BK_, Rows32Cfg>(L);
    case kTileRows64: return launch_ext<AK, BK_, Rows64Cfg>(L);
    case kTileRows112: return launch_ext<AK, BK_, Rows112Cfg>(L);
    default: return launch_ext<AK, BK_, MainCfg>(L);
  }
}

constexpr int kFoldBySegments = 6;  // split tiles are folded by a kernel of its own from here on

// Tile and split of a problem, by choose_plan's cost (rounds of CTAs x work per CTA plus
// 3.3 us per CTA), with the small tiles among the candidates: problems that leave SMs idle
// on large ones, and those of few rows.  A small tile moves more bytes per flop, from L2
// where the problem is small; the handicaps are the ratio of its copy time at 148 SMs to
// its tensor time.
static GemmPlan plan_ext(int M, int N, int K, int sms) {
  struct Candidate {
    int tile, bm, bn;
    double handicap;
  };
  static const Candidate candidates[] = {
      {kTileMain, 128, 128, 1.0},   {kTileHalf, 128, 64, 1.04},    {kTileRows112, 112, 128, 1.06}, {kTileRows64, 64, 128, 1.06},
      {kTileRows32, 32, 128, 1.3},  {kTileSkinny, 128, 32, 1.3},   {kTileRows16, 16, 128, 1.7},
      {kTileSkinny16, 128, 16, 1.7},
  };
  const int KT = (K + BK - 1) / BK;
  GemmPlan best{};
  double best_cost = 0.0;
  for (const Candidate &c : candidates) {
    const long long tiles = (long long)((M + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn);
    if (tiles >= (1ll << 30)) continue;
    const GemmPlan p{c.tile, c.bm, c.bn, choose_spans((int)tiles, KT, sms)};
    const double kt = (double)c.bm * c.bn * c.handicap, per_cta = 25800.0;
    double cost;
    if (p.spans == 0) {
      cost = (double)((tiles + sms - 1) / sms) * (kt * KT + per_cta);
    } else {
      const double work = (double)tiles * KT / p.spans, segments = (double)tiles / p.spans + 1.0;
      cost = (work * kt + segments * per_cta) * (tiles >= sms ? 1.04 : 1.0);
      // the fold: by all SMs in a launch of its own, or one CTA per tile
      cost += p.spans >= kFoldBySegments * tiles ? 25800.0 : 4000.0 * p.spans / (double)tiles * c.bm * c.bn / 16384.0;
    }
    if (best_cost == 0.0 || cost < best_cost) {
      best = p;
      best_cost = cost;
    }
  }
  return best;
}

// Adds up the partial tiles of split tiles in a fixed order (that of k within an eighth of
// the segments, then the eighths) and runs the epilogue.  The kernel's own fold has one CTA per tile, which is
// right for many tiles; for few it is the longest part: 148 partial tiles of 128 x 64
// take one CTA over 100 us and all SMs 4.
__global__ void __launch_bounds__(256)
fold_tiles_kernel(GemmEpilogue ep, const int2 *__restrict__ tiles, int tiles_n, int bm, int bn, int M, int N) {
  cudaGridDependencySynchronize();
  __shared__ double part[8][33];
  const int2 info = tiles[blockIdx.y];
  if (info.y == 0) return;  // a whole tile: written by the kernel itself
  // 32 elements per CTA; its eight warps take consecutive eighths of the segments.
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int e = blockIdx.x * 32 + lane, r = e / bn, c = e - r * bn;
  const int row = (blockIdx.y / tiles_n) * bm + r, col = (blockIdx.y % tiles_n) * bn + c;
  const bool in = row < M && col < N;
  const size_t slot = (size_t)bm * bn;
  const double *src = ep.partial + info.x * slot + e;
  const int first = info.y * warp / 8, last = info.y * (warp + 1) / 8;
  double v = 0.0;
  if (in) {
#pragma unroll 8
    for (int k = first; k < last; k++) v += __ldcs(src + k * slot);
  }
  part[warp][lane] = v;
  __syncthreads();
  if (warp != 0 || !in) return;
  v = 0.0;
#pragma unroll
  for (int w = 0; w < 8; w++) v += part[w][lane];
  if (ep.mode == MG_EPI_BIAS || ep.mode == MG_EPI_BIAS_RELU) v += __ldg(ep.aux + col);
  if (ep.mode == MG_EPI_BIAS_RELU) v = v > 0 ? v : 0.0;
  if (ep.mask8) v = v * (ep.mask8[(size_t)row * ep.ld_mask8 + col] > 0 ? 1.0 : 0.0);
  double *dst = ep.D + (size_t)row * ep.ldd + col;
  *dst = ep.accumulate ? *dst + v : v;
}

__global__ void __launch_bounds__(256)
copy_rows_kernel(const double *__restrict__ src, size_t rows, size_t cols, size_t src_pitch,
                 double *__restrict__ dst, size_t dst_pitch, const int *__restrict__ labels, size_t classes) {
  // (threads x along the row, y over rows: short rows still fill a warp)
  for (size_t r = (size_t)blockIdx.y * blockDim.y + threadIdx.y; r < rows; r += (size_t)gridDim.y * blockDim.y) {
    const bool live = !labels || (labels[r] >= 0 && (size_t)labels[r] < classes);
    for (size_t c = (size_t)blockIdx.x * blockDim.x + threadIdx.x; c < dst_pitch; c += (size_t)gridDim.x * blockDim.x)
      dst[r * dst_pitch + c] = live && c < cols ? src[r * src_pitch + c] : 0.0;
  }
}

int copy_rows(const double *src, size_t rows, size_t cols, size_t src_pitch, double *dst, size_t dst_pitch,
              const int *labels, size_t classes) {
  if (rows == 0 || dst_pitch == 0) return MG_OK;
  unsigned x = 16;
  while (x < 256 && x < dst_pitch) x *= 2;
  const unsigned y = 256 / x;
  const size_t gx = (dst_pitch + x * 4 - 1) / (x * 4);  // four columns per thread
  size_t gy = (rows + y - 1) / y;
  const size_t cap = (size_t)ctx().sm_count * 32 / (gx < 64 ? gx : 64) + 1;
  if (gy > cap) gy = cap;
  if (gy > 65535) gy = 65535;
  copy_rows_kernel<<<dim3((unsigned)(gx < 64 ? gx : 64), (unsigned)gy), dim3(x, y), 0, ctx().stream>>>(
      src, rows, cols, src_pitch, dst, dst_pitch, labels, classes);
  MG_LAUNCH_CHECK("copy_rows");
  return MG_OK;
}

__global__ void __launch_bounds__(256)
empty_product_kernel(double *D, size_t M, size_t N, size_t ldd, int mode, const double *__restrict__ bias,
                     int accumulate) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < M * N; i += (size_t)gridDim.x * 256) {
    const size_t r = i / N, c = i - r * N;
    double v = mode == MG_EPI_BIAS || mode == MG_EPI_BIAS_RELU ? bias[c] : 0.0;
    if (mode == MG_EPI_BIAS_RELU) v = v > 0 ? v : 0.0;
    D[r * ldd + c] = accumulate ? D[r * ldd + c] + v : v;
  }
}

int run_gemm_ext(const GemmExt &e) {
  const GemmDesc &d = e.d;
  if (d.M == 0 || d.N == 0) return MG_OK;
  const size_t lim = (size_t)1 << 30;
  if (d.M >= lim || d.N >= lim || d.K >= lim) return fail(MG_ERR_INVALID, "gemm: dimension too large");
  const size_t a_row = d.a_kcontig ? d.K : d.M, b_row = d.b_kcontig ? d.K : d.N;
  const size_t lda = e.lda ? e.lda : a_row, ldb = e.ldb ? e.ldb : b_row, ldd = e.ldd ? e.ldd : d.N;
  const bool dense = lda == a_row && ldb == b_row && ldd == d.N && !((a_row | b_row | d.N) & 1) &&
                     !off_16_bytes(d.D);
  if (d.K == 0) {
    // Nothing to sum up (and no tensor map of nothing): the epilogue alone.
    if (d.accumulate && d.mode == MG_EPI_NONE) return MG_OK;
    empty_product_kernel<<<grid_for(d.M * d.N, 256, 16), 256, 0, ctx().stream>>>(d.D, d.M, d.N, ldd, d.mode, d.aux,
                                                                               d.accumulate);
    MG_LAUNCH_CHECK("gemm (empty contraction)");
    return MG_OK;
  }
  Context &c = ctx();
  const int M = (int)d.M, N = (int)d.N, K = (int)d.K;
  const GemmPlan plan = plan_ext(M, N, K, c.sm_count);
  const int tiles_m = (M + plan.bm - 1) / plan.bm, tiles_n = (N + plan.bn - 1) / plan.bn;
  const bool fold_here = plan.spans >= kFoldBySegments * tiles_m * tiles_n;
  // Where a large tile is right and the matrices are dense, gemm.cu's instantiations and
  // its own choice among the large tiles are the faster ones.
  if (!e.mask8 && dense && !fold_here &&
      (plan.tile == kTileMain || plan.tile == kTileHalf || plan.tile == kTileRows112))
    return run_gemm(d);
  if ((lda & 1) || off_16_bytes(d.A) || (ldb & 1) || off_16_bytes(d.B))
    return fail(MG_ERR_INVALID, "gemm: operand rows do not start on 16-byte boundaries");
  DmmaLaunch L{};
  bool ok_a, ok_b;
  if (d.a_kcontig) {
    ok_a = make_tensor_map_f64(&L.ma, d.A, d.M, d.K, BK, plan.bm, lda);
  } else if (lda % 16 == 0 && make_tensor_map_f64_grouped(&L.ma, d.A, d.K, lda, BK, plan.bm / 16)) {
    ok_a = true;
    L.grouped_ab |= 1;
  } else {
    ok_a = make_tensor_map_f64(&L.ma, d.A, d.K, d.M, 16, BK, lda);
  }
  if (d.b_kcontig) {
    ok_b = make_tensor_map_f64(&L.mb, d.B, d.N, d.K, BK, plan.bn, ldb);
  } else if (ldb % 16 == 0 && make_tensor_map_f64_grouped(&L.mb, d.B, d.K, ldb, BK, plan.bn / 16)) {
    ok_b = true;
    L.grouped_ab |= 2;
  } else {
    ok_b = make_tensor_map_f64(&L.mb, d.B, d.K, d.N, 16, BK, ldb);
  }
  if (!ok_a || !ok_b) return fail(MG_ERR_CUDA, "gemm: cuTensorMapEncodeTiled failed");
  L.mmask = L.mb;

  GemmEpilogue ep{};
  ep.D = d.D;
  ep.aux = d.aux;
  ep.mode = d.mode;
  ep.accumulate = d.accumulate;
  ep.ldd = ldd;
  ep.mask8 = e.mask8;
  ep.ld_mask8 = d.N;
  ep.pairs = ldd % 2 == 0 && !off_16_bytes(d.D) && !(reinterpret_cast<uintptr_t>(e.mask8) & 1);
  const int KT = (K + BK - 1) / BK;
  const SegTable *table = nullptr;
  if (plan.spans > 0) {
    int rc = seg_table_for(tiles_m, tiles_n, KT, plan.bm, plan.bn, plan.spans, &table);
    if (rc != MG_OK) return rc;
    if (table->slots > 0) {
      rc = ensure_scratch(&c.splitk_scratch, &c.splitk_scratch_elems,
                          (size_t)table->slots * (size_t)plan.bm * (size_t)plan.bn);
      if (rc != MG_OK) return rc;
      ep.partial = c.splitk_scratch;
    }
  }
  L.ep = ep;
  L.M = M; L.N = N; L.K = K;
  L.tiles_m = tiles_m; L.tiles_n = tiles_n;
  L.table = table ? table->dev_items : nullptr;
  const bool split = table && table->slots > 0;
  L.tickets = split && !fold_here ? table->dev_tickets : nullptr;
  L.items = table ? table->items : tiles_m * tiles_n;
  L.min_nkt = table ? table->min_nkt : KT;
  int rc;
  if (d.a_kcontig && !d.b_kcontig) rc = launch_layout_ext<true, false>(plan.tile, L);
  else if (d.a_kcontig) rc = launch_layout_ext<true, true>(plan.tile, L);
  else rc = launch_layout_ext<false, false>(plan.tile, L);
  if (rc != MG_OK || !split || !fold_here) return rc;
  MG_CUDA_TRY(launch_overlapped(fold_tiles_kernel, dim3((unsigned)(plan.bm * plan.bn / 32), (unsigned)(tiles_m * tiles_n)),
                                dim3(256), ep, table->dev_tiles, tiles_n, plan.bm, plan.bn, M, N));
  MG_LAUNCH_CHECK("gemm fold");
  return MG_OK;
}

}  // namespace mg
