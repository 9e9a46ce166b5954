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

// Logits held at a time.
constexpr size_t kBlockBytes = (size_t)1 << 30;
constexpr int kXentThreads = 256;

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

// A CTA per row of the block: row_loss[i], and the row's logits replaced by p (with
// zeros in the columns from V to pitch) when GRAD.
template <bool GRAD>
__global__ void __launch_bounds__(kXentThreads)
xent_rows_kernel(double *__restrict__ z, const int *__restrict__ labels, const double *__restrict__ gloss,
                 double *__restrict__ row_loss, size_t V, size_t pitch, double inv_denom, int *status) {
  __shared__ double smem32[32];
  double *r = z + (size_t)blockIdx.x * pitch;
  const int label = labels[blockIdx.x];
  const bool keep = label >= 0 && (size_t)label < V;
  if (!keep) {
    if (threadIdx.x == 0) {
      if (label != -1) atomicExch(status, 101);  // not a class and not "left out"
      row_loss[blockIdx.x] = 0.0;
    }
    if (GRAD)
      for (size_t j = threadIdx.x; j < pitch; j += kXentThreads) r[j] = 0.0;
    return;
  }
  double top = -INFINITY;
  for (size_t j = threadIdx.x; j < V; j += kXentThreads) top = fmax(top, r[j]);
  top = block_reduce(top, true, smem32);
  double sum = 0.0;
  for (size_t j = threadIdx.x; j < V; j += kXentThreads) sum += exp(r[j] - top);
  sum = block_reduce(sum, false, smem32);
  if (threadIdx.x == 0) row_loss[blockIdx.x] = -(r[label] - top - log(sum));
  if (GRAD) {
    __syncthreads();
    const double scale = (gloss ? *gloss : 1.0) * inv_denom, unit = 1.0 / sum;
    for (size_t j = threadIdx.x; j < pitch; j += kXentThreads)
      r[j] = j < V ? scale * (exp(r[j] - top) * unit - (j == (size_t)label ? 1.0 : 0.0)) : 0.0;
  }
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
      if (h.grad)
        xent_rows_kernel<true><<<(unsigned)rows, kXentThreads, 0, c.stream>>>(
            z, h.labels + m0, h.gloss, ws + at_loss + m0, h.V, Vp, inv, c.kernel_status);
      else
        xent_rows_kernel<false><<<(unsigned)rows, kXentThreads, 0, c.stream>>>(
            z, h.labels + m0, h.gloss, ws + at_loss + m0, h.V, Vp, inv, c.kernel_status);
      MG_LAUNCH_CHECK("linear_xent rows");
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
