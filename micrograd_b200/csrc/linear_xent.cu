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

// dst[drows][dcols] = src[srows][scols] with zeros around it; where labels are given,
// rows that are left out become zeros too (0 times whatever they hold would not).
__global__ void __launch_bounds__(256)
pad_kernel(const double *__restrict__ src, size_t srows, size_t scols, double *__restrict__ dst, size_t drows,
           size_t dcols, const int *__restrict__ labels, size_t V) {
  for (size_t r = blockIdx.y; r < drows; r += gridDim.y) {
    const bool live = r < srows && (!labels || (labels[r] >= 0 && (size_t)labels[r] < V));
    for (size_t c = (size_t)blockIdx.x * 256 + threadIdx.x; c < dcols; c += (size_t)gridDim.x * 256)
      dst[r * dcols + c] = live && c < scols ? src[r * scols + c] : 0.0;
  }
}

// dst[rows][cols] (+)= the left part of src[rows][pitch].
__global__ void __launch_bounds__(256)
unpad_kernel(const double *__restrict__ src, size_t pitch, double *dst, size_t rows, size_t cols, bool accumulate) {
  for (size_t r = blockIdx.y; r < rows; r += gridDim.y)
    for (size_t c = (size_t)blockIdx.x * 256 + threadIdx.x; c < cols; c += (size_t)gridDim.x * 256) {
      const double v = src[r * pitch + c];
      dst[r * cols + c] = accumulate ? dst[r * cols + c] + v : v;
    }
}

static dim3 grid2d(size_t rows, size_t cols) {
  const size_t gx = (cols + 255) / 256 < 64 ? (cols + 255) / 256 : 64;
  size_t gy = rows < 65535 ? rows : 65535;
  return dim3((unsigned)(gx ? gx : 1), (unsigned)(gy ? gy : 1));
}

static bool odd_address(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }
static size_t even(size_t n) { return (n + 1) / 2 * 2; }

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
  const bool want_gx = h.grad && h.gx, want_gw = h.grad && h.gw, want_gb = h.grad && h.gbias;
  // The tensor kernel takes rows of an even number of doubles from 16-byte
  // boundaries.  What does not come like that is copied into that form: M K + K V
  // elements once, against 2 M K V flop or more.
  const size_t Kp = even(h.K), Vp = even(h.V);
  const bool pad_w = Kp != h.K || Vp != h.V || odd_address(h.w);
  const bool pad_bias = h.bias && (Vp != h.V || odd_address(h.bias));
  const bool pad_gw = want_gw && (Kp != h.K || Vp != h.V || odd_address(h.gw));
  const bool pad_gx = want_gx && (Kp != h.K || odd_address(h.gx));
  const bool pad_gb = want_gb && Vp != h.V;
  const bool pad_x = h.grad || Kp != h.K || odd_address(h.x);
  size_t R = kBlockBytes / sizeof(double) / Vp / 128 * 128;
  if (R < 128) R = 128;
  if (R > h.M) R = h.M;

  size_t need = 0;
  auto take = [&](bool wanted, size_t n) {
    const size_t at = need;
    if (wanted) need += (n + 31) / 32 * 32;  // 256-byte boundaries
    return at;
  };
  const size_t at_z = take(true, R * Vp), at_loss = take(true, h.M), at_x = take(pad_x, h.M * Kp);
  const size_t at_w = take(pad_w, Kp * Vp), at_b = take(pad_bias, Vp), at_gw = take(pad_gw, Kp * Vp);
  const size_t at_gx = take(pad_gx, R * Kp), at_gb = take(pad_gb, Vp);
  double *ws = nullptr;
  int rc = mg_alloc(need, &ws);
  if (rc != MG_OK) return rc;

  rc = [&]() -> int {
    const double *x = h.x, *w = h.w, *bias = h.bias;
    auto pad = [&](const double *src, size_t srows, size_t scols, double *dst, size_t drows, size_t dcols,
                   const int *labels) -> int {
      pad_kernel<<<grid2d(drows, dcols), 256, 0, c.stream>>>(src, srows, scols, dst, drows, dcols, labels, h.V);
      MG_LAUNCH_CHECK("linear_xent pad");
      return MG_OK;
    };
    int r;
    if (pad_x) {
      if ((r = pad(h.x, h.M, h.K, ws + at_x, h.M, Kp, h.grad ? h.labels : nullptr)) != MG_OK) return r;
      x = ws + at_x;
    }
    if (pad_w) {
      if ((r = pad(h.w, h.K, h.V, ws + at_w, Kp, Vp, nullptr)) != MG_OK) return r;
      w = ws + at_w;
    }
    if (pad_bias) {
      if ((r = pad(h.bias, 1, h.V, ws + at_b, 1, Vp, nullptr)) != MG_OK) return r;
      bias = ws + at_b;
    }
    double *z = ws + at_z, *gw = pad_gw ? ws + at_gw : h.gw, *gb = pad_gb ? ws + at_gb : h.gbias;
    const double inv = 1.0 / h.denom;
    for (size_t m0 = 0; m0 < h.M; m0 += R) {
      const size_t rows = h.M - m0 < R ? h.M - m0 : R;
      const double *xb = x + m0 * Kp;
      if ((r = run_gemm({xb, w, z, rows, Vp, Kp, true, false, 0, bias ? MG_EPI_BIAS : MG_EPI_NONE, bias})) != MG_OK)
        return r;
      if (h.grad)
        xent_rows_kernel<true><<<(unsigned)rows, kXentThreads, 0, c.stream>>>(
            z, h.labels + m0, h.gloss, ws + at_loss + m0, h.V, Vp, inv, c.kernel_status);
      else
        xent_rows_kernel<false><<<(unsigned)rows, kXentThreads, 0, c.stream>>>(
            z, h.labels + m0, h.gloss, ws + at_loss + m0, h.V, Vp, inv, c.kernel_status);
      MG_LAUNCH_CHECK("linear_xent rows");
      if (want_gx) {
        const bool acc = !(h.flags & MG_ACC_STORE_A);
        double *dst = pad_gx ? ws + at_gx : h.gx + m0 * h.K;
        if ((r = run_gemm({z, w, dst, rows, Kp, Vp, true, true, pad_gx ? 0 : acc, MG_EPI_NONE, nullptr})) != MG_OK)
          return r;
        if (pad_gx) {
          unpad_kernel<<<grid2d(rows, h.K), 256, 0, c.stream>>>(dst, Kp, h.gx + m0 * h.K, rows, h.K, acc);
          MG_LAUNCH_CHECK("linear_xent gx");
        }
      }
      const bool first = m0 == 0;
      if (want_gw) {
        const bool acc = !first || (!pad_gw && !(h.flags & MG_ACC_STORE_B));
        if ((r = run_gemm({xb, z, gw, Kp, Vp, rows, false, false, acc, MG_EPI_NONE, nullptr})) != MG_OK) return r;
      }
      if (want_gb) {
        const bool acc = !first || (!pad_gb && !(h.flags & MG_ACC_STORE_C));
        if ((r = mg_add_row_bwd(z, nullptr, gb, rows, Vp, acc ? 0 : MG_ACC_STORE_B)) != MG_OK) return r;
      }
    }
    if (pad_gw) {
      unpad_kernel<<<grid2d(h.K, h.V), 256, 0, c.stream>>>(gw, Vp, h.gw, h.K, h.V, !(h.flags & MG_ACC_STORE_B));
      MG_LAUNCH_CHECK("linear_xent gw");
    }
    if (pad_gb) {
      unpad_kernel<<<grid2d(1, h.V), 256, 0, c.stream>>>(gb, Vp, h.gbias, 1, h.V, !(h.flags & MG_ACC_STORE_C));
      MG_LAUNCH_CHECK("linear_xent gbias");
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
