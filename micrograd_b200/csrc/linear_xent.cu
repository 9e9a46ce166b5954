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

#include <cooperative_groups.h>

namespace mg {

// Logits held at a time.
constexpr size_t kBlockBytes = (size_t)1 << 30;

__device__ __forceinline__ double block_reduce(double v, bool take_max, double *smem32) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const double o = __shfl_xor_sync(0xffffffffu, v, off);
    v = take_max ? fmax(v, o) : v + o;
  }
  __syncthreads();
  if (lane == 0) smem32[warp] = v;
  __syncthreads();
  const int warps = blockDim.x >> 5;
  v = lane < warps ? smem32[lane] : (take_max ? -INFINITY : 0.0);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const double o = __shfl_xor_sync(0xffffffffu, v, off);
    v = take_max ? fmax(v, o) : v + o;
  }
  return v;
}

// Over the CS CTAs of a row; slot is double-buffered by the two calls a row makes.
template <int CS> __device__ __forceinline__ double row_reduce(double v, bool take_max, double *smem32, double *slot) {
  v = block_reduce(v, take_max, smem32);
  if (CS == 1) return v;
  auto cluster = cooperative_groups::this_cluster();
  if (threadIdx.x == 0) *slot = v;
  cluster.sync();
  double all = take_max ? -INFINITY : 0.0;
#pragma unroll
  for (int r = 0; r < CS; r++) {
    const double o = *cluster.map_shared_rank(slot, r);
    all = take_max ? fmax(all, o) : all + o;
  }
  return all;
}

// A row's loss and, when GRAD, its logits replaced by p.  CS CTAs (a cluster) share a
// row: each keeps its part, a contiguous piece of `piece` classes (a multiple of 4, at
// most kRowsThreads x kRowsValues), in registers, so that a logit is read once, its
// exponential computed once and p written once.  What is between V and the pitch is
// neither used nor written.
constexpr int kRowsThreads = 512, kRowsValues = 16;

template <bool GRAD, int CS>
__global__ void __launch_bounds__(kRowsThreads, 2)
xent_rows_kernel(double *__restrict__ z, const int *__restrict__ labels, const double *__restrict__ gloss,
                 double *__restrict__ row_loss, int V, size_t pitch, int piece, double inv_denom, int *status) {
  __shared__ double smem32[32];
  __shared__ double slot[2];
  const size_t row = blockIdx.x / CS;
  const int rank = CS > 1 ? (int)(blockIdx.x % CS) : 0;
  const int begin = rank * piece, end = begin + piece < V ? begin + piece : V;
  double *r = z + row * pitch;
  const int label = labels[row];
  const bool keep = label >= 0 && label < V;
  if (!keep) {  // (the same in all CTAs of the row)
    if (threadIdx.x == 0 && rank == 0) {
      if (label != -1) atomicExch(status, 101);  // not a class and not "left out"
      row_loss[row] = 0.0;
    }
    if (GRAD)
      for (int j = begin + threadIdx.x; j < end; j += kRowsThreads) r[j] = 0.0;
    return;
  }
  double v[kRowsValues];
  double top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kRowsValues / 4; i++) {
    const int j = begin + (i * kRowsThreads + threadIdx.x) * 4;
    double4v q{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (j < end) q = *reinterpret_cast<const double4v *>(r + j);  // (the pitch is a multiple of 16)
    v[4 * i] = q.x;
    v[4 * i + 1] = j + 1 < end ? q.y : -INFINITY;
    v[4 * i + 2] = j + 2 < end ? q.z : -INFINITY;
    v[4 * i + 3] = j + 3 < end ? q.w : -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < kRowsValues; i++) top = fmax(top, v[i]);
  top = row_reduce<CS>(top, true, smem32, &slot[0]);
  const double at_label = threadIdx.x == 0 && rank == 0 ? r[label] : 0.0;
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < kRowsValues; i++) {
    const int j = begin + ((i >> 2) * kRowsThreads + threadIdx.x) * 4 + (i & 3);
    if (j < end) {
      v[i] = exp(v[i] - top);
      sum += v[i];
    }
  }
  // (p is written only after every CTA of the row has passed this meeting point, so
  // the label's logit has been read)
  sum = row_reduce<CS>(sum, false, smem32, &slot[1]);
  if (threadIdx.x == 0 && rank == 0) row_loss[row] = -(at_label - top - log(sum));
  if (GRAD) {
    const double c = (gloss ? *gloss : 1.0) * inv_denom, scale = c / sum;
#pragma unroll
    for (int i = 0; i < kRowsValues / 4; i++) {
      const int j = begin + (i * kRowsThreads + threadIdx.x) * 4;
      if (j >= end) continue;
      double q[4];
#pragma unroll
      for (int k = 0; k < 4; k++) q[k] = j + k == label ? fma(v[4 * i + k], scale, -c) : v[4 * i + k] * scale;
      if (j + 3 < end) {
        *reinterpret_cast<double4v *>(r + j) = double4v{q[0], q[1], q[2], q[3]};
      } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (j + k < end) r[j + k] = q[k];
      }
    }
  }
  if (CS > 1) cooperative_groups::this_cluster().sync();  // nobody leaves while its slots may be read
}

// The same for rows that eight CTAs cannot hold (over 65 536 classes): the running
// maximum and sum of each thread in one pass, p in a second.
template <bool GRAD>
__global__ void __launch_bounds__(kRowsThreads)
xent_long_rows_kernel(double *__restrict__ z, const int *__restrict__ labels, const double *__restrict__ gloss,
                      double *__restrict__ row_loss, int V, size_t pitch, double inv_denom, int *status) {
  __shared__ double smem32[32];
  double *r = z + (size_t)blockIdx.x * pitch;
  const int label = labels[blockIdx.x];
  const bool keep = label >= 0 && label < V;
  if (!keep) {
    if (threadIdx.x == 0) {
      if (label != -1) atomicExch(status, 101);
      row_loss[blockIdx.x] = 0.0;
    }
    if (GRAD)
      for (int j = threadIdx.x; j < V; j += kRowsThreads) r[j] = 0.0;
    return;
  }
  double own = -INFINITY, sum = 0.0;
  for (int j0 = threadIdx.x; j0 < V; j0 += 8 * kRowsThreads) {
    double v[8], m = own;
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = j0 + k * kRowsThreads < V ? r[j0 + k * kRowsThreads] : -INFINITY;
#pragma unroll
    for (int k = 0; k < 8; k++) m = fmax(m, v[k]);
    if (m > own) {
      sum *= exp(own - m);
      own = m;
    }
    // (own stays -inf while all classes so far have probability 0; a NaN enters the sum)
#pragma unroll
    for (int k = 0; k < 8; k++)
      if (j0 + k * kRowsThreads < V) sum += v[k] == -INFINITY ? 0.0 : exp(v[k] - own);
  }
  const double top = block_reduce(own, true, smem32);
  sum = block_reduce(own == -INFINITY && sum == 0.0 ? 0.0 : sum * exp(own - top), false, smem32);
  if (threadIdx.x == 0) row_loss[blockIdx.x] = -(r[label] - top - log(sum));
  if (GRAD) {
    __syncthreads();
    const double c = (gloss ? *gloss : 1.0) * inv_denom, scale = c / sum;
    for (int j0 = threadIdx.x; j0 < V; j0 += 8 * kRowsThreads) {
      double v[8];
#pragma unroll
      for (int k = 0; k < 8; k++) v[k] = j0 + k * kRowsThreads < V ? r[j0 + k * kRowsThreads] : 0.0;
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const int j = j0 + k * kRowsThreads;
        if (j < V) r[j] = j == label ? fma(exp(v[k] - top), scale, -c) : exp(v[k] - top) * scale;
      }
    }
  }
}

template <bool GRAD, int CS>
static int launch_rows(double *z, const int *labels, const double *gloss, double *row_loss, size_t rows, size_t V,
                       size_t pitch, double inv_denom) {
  Context &c = ctx();
  const size_t piece = ((V + CS - 1) / CS + 3) / 4 * 4;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * CS));
  cfg.blockDim = dim3(kRowsThreads);
  cfg.stream = c.stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CS;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CS > 1 ? 1 : 0;
  MG_CUDA_TRY(cudaLaunchKernelEx(&cfg, xent_rows_kernel<GRAD, CS>, z, labels, gloss, row_loss, (int)V, pitch,
                                 (int)piece, inv_denom, c.kernel_status));
  MG_LAUNCH_CHECK("linear_xent rows");
  return MG_OK;
}

template <bool GRAD>
static int softmax_rows(double *z, const int *labels, const double *gloss, double *row_loss, size_t rows, size_t V,
                        size_t pitch, double inv_denom) {
  Context &c = ctx();
  const size_t room = (size_t)kRowsThreads * kRowsValues;
  if (V > 8 * room) {
    xent_long_rows_kernel<GRAD><<<(unsigned)rows, kRowsThreads, 0, c.stream>>>(z, labels, gloss, row_loss, (int)V,
                                                                             pitch, inv_denom, c.kernel_status);
    MG_LAUNCH_CHECK("linear_xent rows");
    return MG_OK;
  }
  // As few CTAs per row as hold it, more while that leaves SMs without any.
  size_t cs = 1;
  while (cs * (room - 4) < V && cs < 8) cs *= 2;
  while (cs < 8 && rows * cs < (size_t)c.sm_count && V / cs > 2048) cs *= 2;
  if (cs == 1) return launch_rows<GRAD, 1>(z, labels, gloss, row_loss, rows, V, pitch, inv_denom);
  if (cs == 2) return launch_rows<GRAD, 2>(z, labels, gloss, row_loss, rows, V, pitch, inv_denom);
  if (cs == 4) return launch_rows<GRAD, 4>(z, labels, gloss, row_loss, rows, V, pitch, inv_denom);
  return launch_rows<GRAD, 8>(z, labels, gloss, row_loss, rows, V, pitch, inv_denom);
}

// loss[0] = sum of the rows' losses / denom, one CTA, fixed order.
__global__ void __launch_bounds__(1024)
xent_loss_kernel(const double *__restrict__ row_loss, size_t M, double inv_denom, double *loss) {
  __shared__ double smem32[32];
  double sum = 0.0;
  for (size_t i = threadIdx.x; i < M; i += 1024) sum += row_loss[i];
  sum = block_reduce(sum, false, smem32);
  if (threadIdx.x == 0) loss[0] = sum * inv_denom;
}

// out[v] (+)= sum over the rows of p[rows][pitch]: a CTA per 64 columns, its warps the
// rows in turn (fixed order).
constexpr int kColWarps = 16;
__global__ void __launch_bounds__(32 * kColWarps)
column_sums_kernel(const double *__restrict__ p, size_t pitch, size_t rows, size_t V, double *out, bool accumulate) {
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
  column_sums_kernel<<<(unsigned)((V + 63) / 64), dim3(32, kColWarps), 0, ctx().stream>>>(p, pitch, rows, V, out, accumulate);
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

static int run_head(const Head &h) {
  Context &c = ctx();
  // The tensor kernel takes operand rows of an even number of doubles from 16-byte
  // boundaries.  x and w that do not come like that are copied into rows that do (M K
  // or K V elements once, against 2 M K V flop or more); with gradients x is copied in
  // any case, the rows that are left out as zeros: whatever they hold, 0 times it is
  // not 0 in x^T p.
  const size_t Kp = pitch16(h.K), Vp = pitch16(h.V);
  const bool copy_w = h.V % 2 != 0 || off_16_bytes(h.w);
  const bool copy_x = h.grad || h.K % 2 != 0 || off_16_bytes(h.x);
  size_t R = kBlockBytes / sizeof(double) / Vp / 128 * 128;
  if (R < 128) R = 128;
  if (R > h.M) R = h.M;

  size_t need = 0;
  auto take = [&](bool wanted, size_t n) {
    const size_t at = need;
    if (wanted) need += (n + 31) / 32 * 32;  // 256-byte boundaries
    return at;
  };
  const size_t at_z = take(true, R * Vp), at_loss = take(true, h.M), at_x = take(copy_x, h.M * Kp);
  const size_t at_w = take(copy_w, h.K * Vp);
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
      r = h.grad ? softmax_rows<true>(z, h.labels + m0, h.gloss, ws + at_loss + m0, rows, h.V, Vp, inv)
                 : softmax_rows<false>(z, h.labels + m0, h.gloss, ws + at_loss + m0, rows, h.V, Vp, inv);
      if (r != MG_OK) return r;
      const bool first = m0 == 0;
      if (h.grad && h.gx) {
        GemmExt e{{z, w, h.gx + m0 * h.K, rows, h.K, h.V, true, true, !(h.flags & MG_ACC_STORE_A), MG_EPI_NONE, nullptr}};
        e.lda = Vp;
        e.ldb = ldw;
        if ((r = run_gemm_ext(e)) != MG_OK) return r;
      }
      if (h.grad && h.gw) {
        GemmExt e{{xb, z, h.gw, h.K, h.V, rows, false, false, !first || !(h.flags & MG_ACC_STORE_B), MG_EPI_NONE, nullptr}};
        e.lda = ldx;
        e.ldb = Vp;
        if ((r = run_gemm_ext(e)) != MG_OK) return r;
      }
      if (h.grad && h.gbias) {
        if ((r = column_sums(z, Vp, rows, h.V, h.gbias, !first || !(h.flags & MG_ACC_STORE_C))) != MG_OK) return r;
      }
    }
    xent_loss_kernel<<<1, 1024, 0, c.stream>>>(ws + at_loss, h.M, inv, h.loss);
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
