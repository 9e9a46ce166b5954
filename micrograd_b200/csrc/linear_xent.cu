// Softmax cross-entropy of a linear layer over many classes, straight from the
// layer's inputs x[M][K], weights w[K][V] and bias[V]:
//
//   z = x w + bias,  loss = sum_i keep_i (log sum_v exp z_iv - z_{i,label_i}) / denom
//   p = gloss / denom keep (softmax z - onehot)
//   gx += p w^T,  gw += x^T p,  gbias += column sums of p
//
// keep_i is 0 for a row whose label is -1: it adds nothing to any output, whatever
// its values are.  The M x V logits never exist as a whole: a block of rows at a time
// has them in a workspace (kBlockBytes at most, however large M V is), where p
// replaces them before the two gradient products read it.  The gradient therefore
// costs three products, 6 M K V flop; going through the classes in pieces instead,
// with the running maximum and sum of each row, would need the logits a second time:
// 8 M K V flop.  The products run on the FP64 tensor kernel of gemm.cu.
#include "common.cuh"
#include "gemm.cuh"

namespace mg {

// Logits held at a time, and rows (launches over strips of them have 65 535 at most).
constexpr size_t kBlockBytes = (size_t)1 << 30;
constexpr size_t kBlockRows = (size_t)1 << 18;

__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}
__device__ __forceinline__ double warp_total(double v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// The block's softmax in three passes without a barrier in any of them: a warp per 512
// classes of a row leaves their (max, sum of exp); a warp per row joins those; then a
// thread per pair of classes walks down the rows, which turns the logits into p and adds
// up the bias gradient on the way.  24 bytes of traffic and two exponentials per logit:
// 777 x 50 257 takes 236 us with the bias gradient.  Rows held in the registers of a
// cluster of CTAs (16 bytes, one exponential, and a pass of its own for the bias
// gradient) took 304: two CTAs fit an SM, and each waits for its loads, two cluster
// barriers and its stores in turn.
constexpr int kSegment = 512;  // classes per warp: 16 per lane

__global__ void __launch_bounds__(256)
xent_segments_kernel(const double *__restrict__ z, size_t pitch, size_t rows, int V, unsigned segments,
                     double2 *__restrict__ out) {
  cudaGridDependencySynchronize();
  const int lane = threadIdx.x & 31;
  const size_t all = rows * segments;
  for (size_t at = ((size_t)blockIdx.x * 256 + threadIdx.x) >> 5; at < all; at += (size_t)gridDim.x * 8) {
    const size_t row = at / segments;
    const int j0 = (int)(at - row * segments) * kSegment + lane * 4;
    const double *r = z + row * pitch;
    double v[16];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      // (lanes behind the end read the row's first classes: the pitch is a multiple of 16)
      const int j = j0 + 128 * i;
      const double4v q = *reinterpret_cast<const double4v *>(r + (j < V ? j : 0));
      v[4 * i] = j < V ? q.x : -INFINITY;
      v[4 * i + 1] = j + 1 < V ? q.y : -INFINITY;
      v[4 * i + 2] = j + 2 < V ? q.z : -INFINITY;
      v[4 * i + 3] = j + 3 < V ? q.w : -INFINITY;
    }
    double top = v[0];
#pragma unroll
    for (int i = 1; i < 16; i++) top = fmax(top, v[i]);
    top = warp_max(top);
    // (classes without probability add nothing, also where a segment has no others; a
    // NaN is in the sum)
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < 16; i++) sum += v[i] == -INFINITY ? 0.0 : exp(v[i] - top);
    sum = warp_total(sum);
    if (lane == 0) out[at] = make_double2(top, sum);
  }
}

// row_stats[i] = (max, gloss / denom / sum), or (0, 0) for a row that is left out;
// row_loss[i].
__global__ void __launch_bounds__(256)
xent_join_kernel(const double *__restrict__ z, size_t pitch, const double2 *__restrict__ parts, unsigned segments,
                 const int *__restrict__ labels, const double *__restrict__ gloss, size_t rows, int V,
                 double inv_denom, double2 *__restrict__ row_stats, double *__restrict__ row_loss, int *status) {
  cudaGridDependencySynchronize();
  const int lane = threadIdx.x & 31;
  const size_t row = ((size_t)blockIdx.x * 256 + threadIdx.x) >> 5;
  if (row >= rows) return;
  const int label = labels[row];
  const bool keep = label >= 0 && label < V;
  double top = -INFINITY;
  for (unsigned s = lane; s < segments; s += 32) top = fmax(top, parts[row * segments + s].x);
  top = warp_max(top);
  double sum = 0.0;
  for (unsigned s = lane; s < segments; s += 32) {
    const double2 p = parts[row * segments + s];
    sum += p.y * exp(p.x - top);
  }
  sum = warp_total(sum);
  if (lane != 0) return;
  row_loss[row] = keep ? -(z[row * pitch + label] - top - log(sum)) : 0.0;
  row_stats[row] = keep ? make_double2(top, (gloss ? *gloss : 1.0) * inv_denom / sum) : make_double2(0.0, 0.0);
  if (!keep && label != -1) atomicExch(status, 101);  // not a class and not "left out"
}

// z becomes p for 512 classes x `strip` rows per CTA; the classes' sums over these rows
// go to parts[blockIdx.y][pitch] (or are not wanted: null).
constexpr int kApplyRows = 64;  // most rows of a strip

__global__ void __launch_bounds__(256)
xent_apply_kernel(double *__restrict__ z, size_t pitch, size_t rows, int V, const double2 *__restrict__ row_stats,
                  const int *__restrict__ labels, const double *__restrict__ gloss, double inv_denom,
                  double *__restrict__ parts, int strip) {
  cudaGridDependencySynchronize();
  __shared__ double2 stats[kApplyRows];
  __shared__ int label[kApplyRows];
  const size_t r0 = (size_t)blockIdx.y * strip;
  const int count = rows - r0 < (size_t)strip ? (int)(rows - r0) : strip;
  if ((int)threadIdx.x < count) {
    stats[threadIdx.x] = row_stats[r0 + threadIdx.x];
    label[threadIdx.x] = labels[r0 + threadIdx.x];
  }
  __syncthreads();
  const int j = blockIdx.x * 512 + 2 * threadIdx.x;
  if (j >= V) return;  // (the pair may reach into the pitch: what is there is not used)
  const double c = (gloss ? *gloss : 1.0) * inv_denom;
  double *at = z + r0 * pitch + j;
  double s0 = 0.0, s1 = 0.0;
#pragma unroll 4
  for (int r = 0; r < count; r++, at += pitch) {
    const double2 v = __ldcs(reinterpret_cast<const double2 *>(at)), st = stats[r];
    // (scale 0 marks a row that is left out, whatever its logits are; a row whose sum is
    // not finite has a NaN or 0 scale from it and exponentials to match)
    const bool out = label[r] < 0 || label[r] >= V;
    double p0 = out ? 0.0 : exp(v.x - st.x) * st.y, p1 = out ? 0.0 : exp(v.y - st.x) * st.y;
    if (j == label[r]) p0 -= c;
    if (j + 1 == label[r]) p1 -= c;
    s0 += p0;
    s1 += p1;
    *reinterpret_cast<double2 *>(at) = make_double2(p0, p1);
  }
  if (parts) *reinterpret_cast<double2 *>(parts + blockIdx.y * pitch + j) = make_double2(s0, s1);
}

// loss[0] = sum of the rows' losses / denom, one CTA, fixed order.
__global__ void __launch_bounds__(1024)
xent_loss_kernel(const double *__restrict__ row_loss, size_t M, double inv_denom, double *loss) {
  cudaGridDependencySynchronize();
  __shared__ double smem32[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double sum = 0.0;
  for (size_t i = threadIdx.x; i < M; i += 1024) sum += row_loss[i];
  sum = warp_total(sum);
  if (lane == 0) smem32[warp] = sum;
  __syncthreads();
  if (warp != 0) return;
  sum = warp_total(smem32[lane]);
  if (lane == 0) loss[0] = sum * inv_denom;
}

// out[v] (+)= sum over the rows of p[rows][pitch]: a CTA per 64 columns, its warps the
// rows in turn (fixed order).
constexpr int kColWarps = 16;
__global__ void __launch_bounds__(32 * kColWarps)
column_sums_kernel(const double *__restrict__ p, size_t pitch, size_t rows, size_t V, double *out, bool accumulate) {
  cudaGridDependencySynchronize();
  __shared__ double part[kColWarps][64];
  const int lane = threadIdx.x, warp = threadIdx.y;
  const size_t c0 = (size_t)blockIdx.x * 64 + 2 * lane;
  double s0 = 0.0, s1 = 0.0;
  if (c0 < V) {  // (the row's last pair may reach into the pitch, which is a multiple of 16)
#pragma unroll 4
    for (size_t r = warp; r < rows; r += kColWarps) {
      const double2 v = __ldcs(reinterpret_cast<const double2 *>(p + r * pitch + c0));
      s0 += v.x;
      s1 += v.y;
    }
  }
  part[warp][2 * lane] = s0;
  part[warp][2 * lane + 1] = s1;
  __syncthreads();
  const int t = warp * 32 + lane;
  const size_t c = (size_t)blockIdx.x * 64 + t;
  if (t < 64 && c < V) {
    double s = 0.0;
    for (int w = 0; w < kColWarps; w++) s += part[w][t];
    out[c] = accumulate ? out[c] + s : s;
  }
}

static int column_sums(const double *p, size_t pitch, size_t rows, size_t V, double *out, bool accumulate) {
  MG_CUDA_TRY(launch_overlapped(column_sums_kernel, dim3((unsigned)((V + 63) / 64)), dim3(32, kColWarps), p, pitch, rows,
                                V, out, accumulate));
  MG_LAUNCH_CHECK("linear_xent column sums");
  return MG_OK;
}

struct Head {
  const double *x, *w, *bias;
  const int *labels;
  const double *gloss;
  double *loss, *gx, *gw, *gbias;
  size_t M, K, V;
  double denom;
  int flags;
  bool grad;
};

// ---------------------------------------------------------------------------
// Up to four rows (a single one in the per-sample loop), eight for some losses alone: everything is a stream over w, so no
// tile of the tensor kernel is worth filling.  A CTA takes a slab of 64 classes.
//   1. z = x w + bias of the slab, each warp every eighth row of w, and the slab's
//      (max, sum of exp) per row; the CTA that finishes last joins the slabs (in order)
//      to each row's (max, sum) and the loss.
//   2. p of the slab; gw and gbias of its classes, and its share of gx.
//   3. gx: the slabs' shares, in order.
// Left-out rows count as zeros of x and p, whatever x holds.
// ---------------------------------------------------------------------------
constexpr int kFewRows = 4, kFewRowsFwd = 8, kSlab = 64, kFewThreads = 256, kFewWarps = kFewThreads / 32, kFewK = 128;

struct FewRows {
  const double *x, *w, *bias;
  const int *labels;
  const double *gloss;
  double *loss, *gx, *gw, *gbias;
  double *z, *slabs, *at_label, *rows, *shares;  // workspace: [M][Vp], [slabs][M][2], [M], [M][2], [slabs][M][K]
  int M, K, V;
  size_t Vp;
  double inv_denom;
  bool acc_x, acc_w, acc_b, grad;
  unsigned int *ticket;
  int *status;
};

__device__ __forceinline__ bool few_keep(const FewRows &a, int i) {
  return i < a.M && a.labels[i] >= 0 && a.labels[i] < a.V;
}

// w's values of the lane's two classes in the row at src.  Lanes without classes read the
// last ones (a conditional load would be waited for where it meets its default).
template <bool PAIR> __device__ __forceinline__ void few_load(const double *src, int c0, int c1, int V, double &w0, double &w1) {
  if (PAIR) {
    const double2 t = __ldg(reinterpret_cast<const double2 *>(src + (c0 < V ? c0 : V - 2)));
    w0 = t.x;
    w1 = t.y;
  } else {
    w0 = __ldg(src + (c0 < V ? c0 : V - 1));
    w1 = __ldg(src + (c1 < V ? c1 : V - 1));
  }
}

// The lane's two classes of a slab: neighbours where w's rows allow pairs, 32 apart else.
template <bool PAIR> __device__ __forceinline__ int few_class(int lane, int j) {
  return PAIR ? 2 * lane + j : lane + 32 * j;
}

template <int MR, bool PAIR>
__global__ void __launch_bounds__(kFewThreads) few_rows_fwd_kernel(const FewRows a) {
  __shared__ double xs[kFewK][MR];
  __shared__ double sums[kFewWarps][MR][kSlab];
  __shared__ double red[32];
  __shared__ bool is_last;
  cudaGridDependencySynchronize();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, v0 = blockIdx.x * kSlab;
  const int c0 = v0 + few_class<PAIR>(lane, 0), c1 = v0 + few_class<PAIR>(lane, 1);
  // (what the end needs, asked for now)
  const int label = warp < a.M ? a.labels[warp] : -1;
  double bias[2];
#pragma unroll
  for (int j = 0; j < 2; j++) bias[j] = a.bias && v0 + lane + 32 * j < a.V ? __ldg(a.bias + v0 + lane + 32 * j) : 0.0;
  double acc[MR][2];
#pragma unroll
  for (int i = 0; i < MR; i++) acc[i][0] = acc[i][1] = 0.0;
  constexpr int kRowsPerWarp = kFewK / kFewWarps;
  for (int k0 = 0; k0 < a.K; k0 += kFewK) {
    const int ks = a.K - k0 < kFewK ? a.K - k0 : kFewK;
    // All of the warp's rows of w are on their way before x is waited for.
    double w0[kRowsPerWarp], w1[kRowsPerWarp];
#pragma unroll
    for (int r = 0; r < kRowsPerWarp; r++) {
      const int k = warp + r * kFewWarps < ks ? warp + r * kFewWarps : ks - 1;
      few_load<PAIR>(a.w + (size_t)(k0 + k) * a.V, c0, c1, a.V, w0[r], w1[r]);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < kFewK * MR; e += kFewThreads) {
      const int i = e / kFewK, k = e % kFewK;
      xs[k][i] = i < a.M && k < ks ? a.x[(size_t)i * a.K + k0 + k] : 0.0;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRowsPerWarp; r++) {
      if (warp + r * kFewWarps < ks) {
#pragma unroll
        for (int i = 0; i < MR; i++) {
          const double x = xs[warp + r * kFewWarps][i];
          acc[i][0] = fma(x, w0[r], acc[i][0]);
          acc[i][1] = fma(x, w1[r], acc[i][1]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MR; i++) {
    sums[warp][i][few_class<PAIR>(lane, 0)] = acc[i][0];
    sums[warp][i][few_class<PAIR>(lane, 1)] = acc[i][1];
  }
  __syncthreads();
  // A warp per row: its 64 logits, two per lane.
  static_assert(MR <= kFewWarps, "a warp per row");
  if (warp < a.M) {
    const int i = warp;
    double z[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int s = lane + 32 * j, c = v0 + s;
      z[j] = -INFINITY;
      if (c < a.V) {
        double t = 0.0;
#pragma unroll
        for (int w = 0; w < kFewWarps; w++) t += sums[w][i][s];
        t += bias[j];
        z[j] = t;
        if (a.grad) a.z[(size_t)i * a.Vp + c] = t;
        if (c == label) a.at_label[i] = t;
      }
    }
    double top = fmax(z[0], z[1]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, off));
    // (a slab of classes without probability adds nothing; a NaN is in the sum)
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < 2; j++) sum += z[j] == -INFINITY ? 0.0 : exp(z[j] - top);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane == 0) {
      double *out = a.slabs + ((size_t)blockIdx.x * a.M + i) * 2;
      out[0] = top;
      out[1] = sum;
    }
  }
  // (the gradients' kernel may be set up from here on; it waits for this one's end)
  cudaTriggerProgrammaticLaunchCompletion();
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) is_last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!is_last) return;
  __threadfence();
  if (warp < a.M) {
    const int i = warp;
    const bool keep = label >= 0 && label < a.V;
    double top = -INFINITY;
    for (unsigned s = lane; s < gridDim.x; s += 32) top = fmax(top, __ldcg(a.slabs + ((size_t)s * a.M + i) * 2));
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, off));
    double sum = 0.0;
    for (unsigned s = lane; s < gridDim.x; s += 32) {
      const double *p = a.slabs + ((size_t)s * a.M + i) * 2;
      sum += __ldcg(p + 1) * exp(__ldcg(p) - top);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane == 0) {
      a.rows[2 * i] = top;
      a.rows[2 * i + 1] = sum;
      red[i] = keep ? -(__ldcg(a.at_label + i) - top - log(sum)) : 0.0;
      if (!keep && label != -1) atomicExch(a.status, 101);  // not a class and not "left out"
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double loss = 0.0;
    for (int i = 0; i < a.M; i++) loss += red[i];
    a.loss[0] = loss * a.inv_denom;
    *a.ticket = 0u;
  }
}

template <int MR, bool PAIR>
__global__ void __launch_bounds__(kFewThreads) few_rows_bwd_kernel(const FewRows a) {
  constexpr int kPitch = kSlab + 4;  // eight rows x four classes 4 apart fall into different banks
  __shared__ double xs[kSlab][MR];
  __shared__ __align__(16) double ps[kSlab][MR];
  __shared__ double ws[kSlab][kPitch];
  __shared__ bool kept[MR];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, v0 = blockIdx.x * kSlab;
  const int s0 = few_class<PAIR>(lane, 0), s1 = few_class<PAIR>(lane, 1), c0 = v0 + s0, c1 = v0 + s1;
  constexpr int kRowsPerWarp = kSlab / kFewWarps;
  // Rows k0 ... of w (64 at a time), asked for one step ahead.
  double w0[kRowsPerWarp], w1[kRowsPerWarp];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int r = 0; r < kRowsPerWarp; r++) {
      const int k = k0 + warp + r * kFewWarps < a.K ? k0 + warp + r * kFewWarps : a.K - 1;
      few_load<PAIR>(a.w + (size_t)k * a.V, c0, c1, a.V, w0[r], w1[r]);
    }
  };
  constexpr int kXs = (kSlab * MR + kFewThreads - 1) / kFewThreads;
  double x_next[kXs];
  auto fetch_x = [&](int k0) {
#pragma unroll
    for (int r = 0; r < kXs; r++) {
      const int e = threadIdx.x + r * kFewThreads, i = e / kSlab < a.M ? e / kSlab : 0, k = k0 + (e & (kSlab - 1));
      x_next[r] = __ldg(a.x + (size_t)i * a.K + (k < a.K ? k : a.K - 1));
    }
  };
  // The inputs do not depend on the kernel before this one, which may still be running
  // here; everything after the wait may.
  if (a.gx) fetch(0);
  if (a.K) fetch_x(0);
  if (threadIdx.x < MR) kept[threadIdx.x] = few_keep(a, threadIdx.x);
  cudaGridDependencySynchronize();
  __syncthreads();
  const double c = (a.gloss ? *a.gloss : 1.0) * a.inv_denom;
  for (int e = threadIdx.x; e < kSlab * MR; e += kFewThreads) {
    const int i = e / kSlab, s = e - i * kSlab, v = v0 + s;
    double p = 0.0;
    if (v < a.V && kept[i]) {
      const double scale = c / a.rows[2 * i + 1];
      p = exp(a.z[(size_t)i * a.Vp + v] - a.rows[2 * i]);
      p = v == a.labels[i] ? fma(p, scale, -c) : p * scale;
    }
    ps[s][i] = p;
  }
  __syncthreads();
  if (a.gbias && threadIdx.x < kSlab && v0 + (int)threadIdx.x < a.V) {
    double s = 0.0;
    for (int i = 0; i < a.M; i++) s += ps[threadIdx.x][i];
    double *dst = a.gbias + v0 + threadIdx.x;
    *dst = a.acc_b ? *dst + s : s;
  }
  double p0[MR], p1[MR];
#pragma unroll
  for (int i = 0; i < MR; i++) {
    p0[i] = ps[s0][i];
    p1[i] = ps[s1][i];
  }
  cudaTriggerProgrammaticLaunchCompletion();
  for (int k0 = 0; k0 < a.K; k0 += kSlab) {
    const int ks = a.K - k0 < kSlab ? a.K - k0 : kSlab;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kXs; r++) {
      const int e = threadIdx.x + r * kFewThreads, i = e / kSlab, k = e & (kSlab - 1);
      if (i < MR) xs[k][i] = k < ks && kept[i] ? x_next[r] : 0.0;
    }
    if (k0 + kSlab < a.K) fetch_x(k0 + kSlab);
    if (a.gx) {
#pragma unroll
      for (int r = 0; r < kRowsPerWarp; r++) {
        // (classes behind the last one have p = 0, but w there may be anything)
        ws[warp + r * kFewWarps][s0] = c0 < a.V ? w0[r] : 0.0;
        ws[warp + r * kFewWarps][s1] = c1 < a.V ? w1[r] : 0.0;
      }
      if (k0 + kSlab < a.K) fetch(k0 + kSlab);
    }
    __syncthreads();
    if (a.gw) {
#pragma unroll 4
      for (int k = warp; k < ks; k += kFewWarps) {
        double g0 = 0.0, g1 = 0.0;
#pragma unroll
        for (int i = 0; i < MR; i++) {
          g0 = fma(xs[k][i], p0[i], g0);
          g1 = fma(xs[k][i], p1[i], g1);
        }
        double *dst = a.gw + (size_t)(k0 + k) * a.V;
        if (PAIR) {
          if (c0 < a.V) {
            double2 *d = reinterpret_cast<double2 *>(dst + c0);
            if (a.acc_w) {
              const double2 o = *d;
              g0 = o.x + g0;
              g1 = o.y + g1;
            }
            __stcs(d, make_double2(g0, g1));
          }
        } else {
          if (c0 < a.V) dst[c0] = a.acc_w ? dst[c0] + g0 : g0;
          if (c1 < a.V) dst[c1] = a.acc_w ? dst[c1] + g1 : g1;
        }
      }
    }
    if (a.gx) {
      // Four lanes share a row of w, every fourth class each.
      const int k = warp * 8 + (lane >> 2), q = lane & 3;
      double s[MR];
#pragma unroll
      for (int i = 0; i < MR; i++) s[i] = 0.0;
#pragma unroll
      for (int v = 0; v < kSlab; v += 4) {
        const double w = ws[k][v + q];
#pragma unroll
        for (int i = 0; i < MR; i++) s[i] = fma(w, ps[v + q][i], s[i]);
      }
#pragma unroll
      for (int i = 0; i < MR; i++) {
        s[i] += __shfl_xor_sync(0xffffffffu, s[i], 1);
        s[i] += __shfl_xor_sync(0xffffffffu, s[i], 2);
        if ((i & 3) == q && i < a.M && k < ks)
          a.shares[((size_t)blockIdx.x * a.M + i) * a.K + k0 + k] = s[i];
      }
    }
  }
}

// gx[i] (+)= sum over the slabs of shares[slab][i]: 16 entries per CTA, 16 threads each.
__global__ void __launch_bounds__(256)
few_rows_gx_kernel(const double *__restrict__ shares, unsigned slabs, size_t n, double *gx, bool accumulate) {
  __shared__ double part[16][17];
  const int e = threadIdx.x & 15, t = threadIdx.x >> 4;
  const size_t at = (size_t)blockIdx.x * 16 + e;
  cudaGridDependencySynchronize();
  double s = 0.0;
  if (at < n) {
#pragma unroll 8
    for (unsigned k = t; k < slabs; k += 16) s += __ldcs(shares + k * n + at);
  }
  part[t][e] = s;
  __syncthreads();
  if (t == 0 && at < n) {
    s = 0.0;
    for (int k = 0; k < 16; k++) s += part[k][e];
    gx[at] = accumulate ? gx[at] + s : s;
  }
}

template <int MR, bool PAIR> static int launch_few_fwd(const FewRows &a) {
  const unsigned slabs = (unsigned)((a.V + kSlab - 1) / kSlab);
  MG_CUDA_TRY(launch_overlapped(few_rows_fwd_kernel<MR, PAIR>, dim3(slabs), dim3(kFewThreads), a));
  MG_LAUNCH_CHECK("linear_xent (few rows)");
  return MG_OK;
}

template <int MR> static int launch_few(const FewRows &a, bool pair) {
  const unsigned slabs = (unsigned)((a.V + kSlab - 1) / kSlab);
  const int rc = pair ? launch_few_fwd<MR, true>(a) : launch_few_fwd<MR, false>(a);
  if (rc != MG_OK || !a.grad) return rc;
  MG_CUDA_TRY(launch_overlapped(pair ? few_rows_bwd_kernel<MR, true> : few_rows_bwd_kernel<MR, false>, dim3(slabs),
                                dim3(kFewThreads), a));
  MG_LAUNCH_CHECK("linear_xent (few rows, gradients)");
  if (!a.gx) return MG_OK;
  const size_t n = (size_t)a.M * a.K;
  MG_CUDA_TRY(launch_overlapped(few_rows_gx_kernel, dim3((unsigned)((n + 15) / 16)), dim3(256), a.shares, slabs, n,
                                a.gx, a.acc_x));
  MG_LAUNCH_CHECK("linear_xent (few rows, gx)");
  return MG_OK;
}

static int run_few_rows(const Head &h) {
  Context &c = ctx();
  FewRows a{};
  a.x = h.x; a.w = h.w; a.bias = h.bias; a.labels = h.labels; a.gloss = h.gloss; a.loss = h.loss;
  a.gx = h.K ? h.gx : nullptr; a.gw = h.K ? h.gw : nullptr; a.gbias = h.gbias;
  a.M = (int)h.M; a.K = (int)h.K; a.V = (int)h.V;
  a.Vp = pitch16(h.V);
  a.inv_denom = 1.0 / h.denom;
  a.acc_x = !(h.flags & MG_ACC_STORE_A);
  a.acc_w = !(h.flags & MG_ACC_STORE_B);
  a.acc_b = !(h.flags & MG_ACC_STORE_C);
  a.grad = h.grad;
  a.ticket = c.reduce_ticket + 1;
  a.status = c.kernel_status;
  const size_t slabs = (h.V + kSlab - 1) / kSlab;
  double *ws = nullptr;
  const size_t n_z = h.grad ? h.M * a.Vp : 0, n_slabs = slabs * h.M * 2, n_rows = 3 * h.M;
  int rc = mg_alloc(n_z + n_slabs + n_rows + (a.gx ? slabs * h.M * h.K : 0), &ws);
  if (rc != MG_OK) return rc;
  a.z = ws;
  a.slabs = ws + n_z;
  a.at_label = a.slabs + n_slabs;
  a.rows = a.at_label + h.M;
  a.shares = a.rows + 2 * h.M;
  const bool pair = h.V % 2 == 0 && !off_16_bytes(h.w) && !(a.gw && off_16_bytes(a.gw));
  if (h.M == 1) rc = launch_few<1>(a, pair);
  else if (h.M == 2) rc = launch_few<2>(a, pair);
  else if (h.M <= (size_t)kFewRows) rc = launch_few<kFewRows>(a, pair);
  else rc = launch_few_fwd<kFewRowsFwd, false>(a);  // (neighbours cannot be paired there)
  const int freed = mg_free(ws);
  return rc != MG_OK ? rc : freed;
}

static int run_head(const Head &h) {
  if (h.M <= (size_t)kFewRows) return run_few_rows(h);
  const bool copy_w = h.V % 2 != 0 || off_16_bytes(h.w);
  // The loss alone of five to eight rows streams over w too where the tensor kernel would
  // need a copy of it: 5 and 8 rows x 676 x 90 181 143 and 177 us instead of 310, 300 x
  // 5001 13 and 15 instead of 26.  (90 182 classes, without the copy: 119 on the tensor
  // kernel, 142 and 177 here.  Two groups of eight rows lose to the copy at 64 x 30 001.)
  if (!h.grad && copy_w && h.M <= (size_t)kFewRowsFwd) return run_few_rows(h);
  Context &c = ctx();
  // The tensor kernel takes operand rows of an even number of doubles from 16-byte
  // boundaries.  x and w that do not come like that are copied into rows that do (M K
  // or K V elements once, against 2 M K V flop or more); with gradients x is copied in
  // any case, the rows that are left out as zeros: whatever they hold, 0 times it is
  // not 0 in x^T p.
  const size_t Kp = pitch16(h.K), Vp = pitch16(h.V);
  const bool copy_x = h.grad || h.K % 2 != 0 || off_16_bytes(h.x);
  size_t R = kBlockBytes / sizeof(double) / Vp;
  R = R >= 128 ? R / 128 * 128 : R / 16 * 16;  // whole tiles
  if (R < 16) R = 16;
  if (R > kBlockRows) R = kBlockRows;
  if (R > h.M) R = h.M;

  size_t need = 0;
  auto take = [&](bool wanted, size_t n) {
    const size_t at = need;
    if (wanted) need += (n + 31) / 32 * 32;  // 256-byte boundaries
    return at;
  };
  const size_t at_z = take(true, R * Vp), at_loss = take(true, h.M), at_x = take(copy_x, h.M * Kp);
  const size_t at_w = take(copy_w, h.K * Vp);
  const unsigned segments = (unsigned)((h.V + kSegment - 1) / kSegment);
  // Strips of 64 rows, fewer where that would leave SMs without a CTA (at least four: each
  // strip costs a row of sums).
  const size_t wide = (h.V + 511) / 512;
  size_t strip = R * wide / ((size_t)c.sm_count * 2);
  strip = strip > (size_t)kApplyRows ? kApplyRows : (strip < 4 ? 4 : strip);
  const size_t strips = (R + strip - 1) / strip;
  const size_t at_parts = take(true, 2 * R * segments), at_stats = take(true, 2 * R);
  const size_t at_sums = take(h.grad && h.gbias, strips * Vp);
  double *ws = nullptr;
  int rc = mg_alloc(need, &ws);
  if (rc != MG_OK) return rc;

  rc = [&]() -> int {
    const double *x = h.x, *w = h.w;
    const size_t ldx = copy_x ? Kp : h.K, ldw = copy_w ? Vp : h.V;
    int r;
    if (copy_x) {
      if ((r = copy_rows(h.x, h.M, h.K, h.K, ws + at_x, Kp, h.grad ? h.labels : nullptr, h.V)) != MG_OK) return r;
      x = ws + at_x;
    }
    if (copy_w) {
      if ((r = copy_rows(h.w, h.K, h.V, h.V, ws + at_w, Vp)) != MG_OK) return r;
      w = ws + at_w;
    }
    double *z = ws + at_z;
    const double inv = 1.0 / h.denom;
    for (size_t m0 = 0; m0 < h.M; m0 += R) {
      const size_t rows = h.M - m0 < R ? h.M - m0 : R;
      const double *xb = x + m0 * ldx;
      GemmExt fwd{{xb, w, z, rows, h.V, h.K, true, false, 0, h.bias ? MG_EPI_BIAS : MG_EPI_NONE, h.bias}};
      fwd.lda = ldx;
      fwd.ldb = ldw;
      fwd.ldd = Vp;
      if ((r = run_gemm_ext(fwd)) != MG_OK) return r;
      double2 *parts = reinterpret_cast<double2 *>(ws + at_parts), *stats = reinterpret_cast<double2 *>(ws + at_stats);
      const int *labels = h.labels + m0;
      MG_CUDA_TRY(launch_overlapped(xent_segments_kernel, dim3(grid_for(rows * segments * 32, 256, 32)), dim3(256), z, Vp,
                                    rows, (int)h.V, segments, parts));
      MG_LAUNCH_CHECK("linear_xent segments");
      MG_CUDA_TRY(launch_overlapped(xent_join_kernel, dim3((unsigned)((rows * 32 + 255) / 256)), dim3(256), z, Vp, parts,
                                    segments, labels, h.gloss, rows, (int)h.V, inv, stats, ws + at_loss + m0,
                                    c.kernel_status));
      MG_LAUNCH_CHECK("linear_xent join");
      if (!h.grad) continue;
      const unsigned used = (unsigned)((rows + strip - 1) / strip);
      MG_CUDA_TRY(launch_overlapped(xent_apply_kernel, dim3((unsigned)wide, used), dim3(256), z, Vp, rows, (int)h.V, stats,
                                    labels, h.gloss, inv, h.gbias ? ws + at_sums : nullptr, (int)strip));
      MG_LAUNCH_CHECK("linear_xent apply");
      const bool first = m0 == 0;
      if (h.gx) {
        GemmExt e{{z, w, h.gx + m0 * h.K, rows, h.K, h.V, true, true, !(h.flags & MG_ACC_STORE_A), MG_EPI_NONE, nullptr}};
        e.lda = Vp;
        e.ldb = ldw;
        if ((r = run_gemm_ext(e)) != MG_OK) return r;
      }
      if (h.gw) {
        GemmExt e{{xb, z, h.gw, h.K, h.V, rows, false, false, !first || !(h.flags & MG_ACC_STORE_B), MG_EPI_NONE, nullptr}};
        e.lda = ldx;
        e.ldb = Vp;
        if ((r = run_gemm_ext(e)) != MG_OK) return r;
      }
      if (h.gbias) {
        if ((r = column_sums(ws + at_sums, Vp, used, h.V, h.gbias, !first || !(h.flags & MG_ACC_STORE_C))) != MG_OK) return r;
      }
    }
    MG_CUDA_TRY(launch_overlapped(xent_loss_kernel, dim3(1), dim3(1024), ws + at_loss, h.M, inv, h.loss));
    MG_LAUNCH_CHECK("linear_xent loss");
    return MG_OK;
  }();
  const int freed = mg_free(ws);
  return rc != MG_OK ? rc : freed;
}

static int check_head(const char *name, const Head &h) {
  if (!h.loss) return fail(MG_ERR_INVALID, "%s: null output", name);
  const size_t lim = (size_t)1 << 30;
  if (h.M >= lim || h.K >= lim || h.V >= lim) return fail(MG_ERR_INVALID, "%s: dimension too large", name);
  if (h.M && h.V && (!h.labels || (h.K && (!h.x || !h.w))))
    return fail(MG_ERR_INVALID, "%s: null input", name);
  if (!(h.denom > 0.0)) return fail(MG_ERR_INVALID, "%s: denom must be positive", name);
  return MG_OK;
}

}  // namespace mg

using namespace mg;

extern "C" {

int mg_linear_xent_fwd(const double *x, const double *w, const double *bias, const int *labels, double *loss1,
                       size_t M, size_t K, size_t V, double denom) {
  const Head h{x, w, bias, labels, nullptr, loss1, nullptr, nullptr, nullptr, M, K, V, denom, 0, false};
  int rc = check_head("mg_linear_xent_fwd", h);
  if (rc != MG_OK) return rc;
  MG_ENSURE_INIT();
  if (M == 0 || V == 0) return mg_fill(loss1, 0.0, 1);
  return run_head(h);
}

int mg_linear_xent_fwd_bwd(const double *x, const double *w, const double *bias, const int *labels,
                           const double *gloss1, double *loss1, double *gx, double *gw, double *gbias, size_t M,
                           size_t K, size_t V, double denom, int flags) {
  const Head h{x, w, bias, labels, gloss1, loss1, gx, gw, gbias, M, K, V, denom, flags, gx || gw || gbias};
  int rc = check_head("mg_linear_xent_fwd_bwd", h);
  if (rc != MG_OK) return rc;
  MG_ENSURE_INIT();
  if (M == 0 || V == 0) {
    // Nothing to add: destinations that may be stored to hold sums of nothing.
    if (gx && (flags & MG_ACC_STORE_A) && M * K) rc = mg_fill(gx, 0.0, M * K);
    if (rc == MG_OK && gw && (flags & MG_ACC_STORE_B) && K * V) rc = mg_fill(gw, 0.0, K * V);
    if (rc == MG_OK && gbias && (flags & MG_ACC_STORE_C) && V) rc = mg_fill(gbias, 0.0, V);
    return rc != MG_OK ? rc : mg_fill(loss1, 0.0, 1);
  }
  return run_head(h);
}

}  // extern "C"
