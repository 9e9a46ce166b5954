// Group norm with an activation over channels-last data x[N][P][C]: N samples of P
// positions, C channels in G groups of D = C / G neighbours.  For every (n, g), over
// the E = P D values of the group:
//
//   mean = sum x / E,  var = sum (x - mean)^2 / E,  rstd = 1 / sqrt(var + eps)
//   unit = (x - mean) rstd,  z = unit gamma + beta,  y = act(z)
//
// and, with gz = gy act'(z), u = gz gamma,  m1 = sum u / E,  m2 = sum u unit / E:
//
//   gx = rstd (u - m1 - unit m2),  ggamma = sum_{n,p} gz unit,  gbeta = sum_{n,p} gz
//
// Every sum is taken in a fixed order: nothing here depends on scheduling.
// Variances are never formed as a difference of large numbers: each piece of a
// group is summed around its own mean and pieces are joined by
//   delta = mean_b - mean_a,  mean = mean_a + delta n_b / n,
//   M2 = M2_a + M2_b + delta^2 n_a n_b / n      (Chan, Golub and LeVeque 1979).
#include "common.cuh"

#include <type_traits>

namespace mg {

struct Moments {
  double n, mean, m2;
};

__device__ __forceinline__ Moments join(const Moments &a, const Moments &b) {
  const double n = a.n + b.n;
  if (n == 0.0) return a;
  const double share = b.n / n, delta = b.mean - a.mean;
  return {n, a.mean + delta * share, a.m2 + b.m2 + delta * delta * a.n * share};
}

__device__ __forceinline__ double shfl_sum(double v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// Sum over the CTA, valid in every thread (blockDim.x a multiple of 32).
__device__ __forceinline__ double cta_sum(double v, double *smem32) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = shfl_sum(v);
  __syncthreads();
  if (lane == 0) smem32[warp] = v;
  __syncthreads();
  double t = lane < (int)(blockDim.x >> 5) ? smem32[lane] : 0.0;
  return shfl_sum(t);
}

template <int ACT> __device__ __forceinline__ double act_fwd(double z) {
  if (ACT == MG_ACT_RELU) return z > 0 ? z : 0.0;
  if (ACT == MG_ACT_SILU) return z / (1.0 + exp(-z));
  return z;
}

template <int ACT> __device__ __forceinline__ double act_bwd(double z, double g) {
  if (ACT == MG_ACT_RELU) return z > 0 ? g : g * 0.0;
  if (ACT == MG_ACT_SILU) {
    const double s = 1.0 / (1.0 + exp(-z));
    return g * (s * (1.0 + z * (1.0 - s)));
  }
  return g;
}

struct NormShape {
  size_t N, P;
  int C, G, D;
};

constexpr int kGnThreads = 256;
// Values of a group that one CTA takes in the general form: 64 KB, so that its
// second look at them comes from L2.
constexpr size_t kGnPiece = 8192;

// General form, step 1: moments of one piece of one group.
__global__ void __launch_bounds__(kGnThreads)
gn_moments_kernel(const double *__restrict__ x, NormShape s, size_t piece, double *__restrict__ parts,
                  double eps, double *__restrict__ mean_out, double *__restrict__ rstd_out) {
  __shared__ double smem32[32];
  const size_t ng = blockIdx.x, n = ng / s.G, g = ng - n * s.G;
  const size_t E = s.P * (size_t)s.D;
  const size_t begin = blockIdx.y * piece, end = begin + piece < E ? begin + piece : E;
  const double *base = x + n * s.P * s.C + g * s.D;
  double sum = 0.0;
  for (size_t e = begin + threadIdx.x; e < end; e += kGnThreads) {
    const size_t p = e / s.D, d = e - p * s.D;
    sum += base[p * s.C + d];
  }
  const double count = (double)(end - begin), mean = cta_sum(sum, smem32) / count;
  double m2 = 0.0;
  for (size_t e = begin + threadIdx.x; e < end; e += kGnThreads) {
    const size_t p = e / s.D, d = e - p * s.D;
    const double v = base[p * s.C + d] - mean;
    m2 += v * v;
  }
  m2 = cta_sum(m2, smem32);
  if (threadIdx.x != 0) return;
  if (gridDim.y == 1) {
    mean_out[ng] = mean;
    rstd_out[ng] = 1.0 / sqrt(m2 / count + eps);
  } else {
    double *out = parts + 3 * (ng * gridDim.y + blockIdx.y);
    out[0] = count;
    out[1] = mean;
    out[2] = m2;
  }
}

// Step 2: the pieces of a group joined, a warp per group.
__global__ void __launch_bounds__(kGnThreads)
gn_moments_join_kernel(const double *__restrict__ parts, size_t groups, unsigned pieces, double eps,
                       double *__restrict__ mean_out, double *__restrict__ rstd_out) {
  const int lane = threadIdx.x & 31;
  const size_t ng = ((size_t)blockIdx.x * kGnThreads + threadIdx.x) >> 5;
  if (ng >= groups) return;
  Moments m{0.0, 0.0, 0.0};
  for (unsigned k = lane; k < pieces; k += 32) {
    const double *p = parts + 3 * (ng * pieces + k);
    m = join(m, {p[0], p[1], p[2]});
  }
  for (int off = 16; off > 0; off >>= 1) {
    const Moments o{__shfl_down_sync(0xffffffffu, m.n, off), __shfl_down_sync(0xffffffffu, m.mean, off),
                    __shfl_down_sync(0xffffffffu, m.m2, off)};
    m = join(m, o);
  }
  if (lane == 0) {
    mean_out[ng] = m.mean;
    rstd_out[ng] = 1.0 / sqrt(m.m2 / m.n + eps);
  }
}

// Step 3: normalise.  A thread keeps its channel and walks the rows (n, p).
template <int ACT>
__global__ void __launch_bounds__(kGnThreads)
gn_apply_kernel(const double *__restrict__ x, const double *__restrict__ gamma,
                const double *__restrict__ beta, const double *__restrict__ mean,
                const double *__restrict__ rstd, double *__restrict__ y, NormShape s) {
  const int c = blockIdx.x * 32 + threadIdx.x;
  if (c >= s.C) return;
  const int g = c / s.D;
  const double ga = gamma ? gamma[c] : 1.0, be = beta ? beta[c] : 0.0;
  const size_t rows = s.N * s.P;
  for (size_t r = (size_t)blockIdx.y * blockDim.y + threadIdx.y; r < rows; r += (size_t)gridDim.y * blockDim.y) {
    const size_t ng = r / s.P * s.G + g;
    const double unit = (x[r * s.C + c] - __ldg(mean + ng)) * __ldg(rstd + ng);
    y[r * s.C + c] = act_fwd<ACT>(unit * ga + be);
  }
}

// Backward, step 1: sums of gz and gz unit over one piece of a sample's positions,
// per channel: parts[n][piece][2][C].
template <int ACT>
__global__ void __launch_bounds__(kGnThreads)
gn_bwd_sums_kernel(const double *__restrict__ x, const double *__restrict__ gamma,
                   const double *__restrict__ beta, const double *__restrict__ mean,
                   const double *__restrict__ rstd, const double *__restrict__ gy, NormShape s,
                   unsigned pieces, size_t piece, double *__restrict__ parts) {
  __shared__ double sums[2][8][33];
  const int tx = threadIdx.x, ty = threadIdx.y, c = blockIdx.x * 32 + tx;
  for (size_t unit_id = blockIdx.y; unit_id < s.N * pieces; unit_id += gridDim.y) {
    const size_t n = unit_id / pieces, k = unit_id - n * pieces;
    const size_t end = (k + 1) * piece < s.P ? (k + 1) * piece : s.P;
    double sb = 0.0, sg = 0.0;
    if (c < s.C) {
      const size_t ng = n * s.G + c / s.D;
      const double ga = gamma ? gamma[c] : 1.0, be = beta ? beta[c] : 0.0, mu = mean[ng], rs = rstd[ng];
      for (size_t p = k * piece + ty; p < end; p += 8) {
        const size_t at = (n * s.P + p) * s.C + c;
        const double unit = (x[at] - mu) * rs, gz = act_bwd<ACT>(unit * ga + be, gy[at]);
        sb += gz;
        sg += gz * unit;
      }
    }
    sums[0][ty][tx] = sb;
    sums[1][ty][tx] = sg;
    __syncthreads();
    if (ty < 2 && c < s.C) {
      double t = 0.0;
      for (int j = 0; j < 8; j++) t += sums[ty][j][tx];
      parts[(unit_id * 2 + ty) * s.C + c] = t;
    }
    __syncthreads();
  }
}

// Step 2: m1 and m2 of every group, a warp per group.
__global__ void __launch_bounds__(kGnThreads)
gn_bwd_groups_kernel(const double *__restrict__ parts, const double *__restrict__ gamma, NormShape s,
                     unsigned pieces, double *__restrict__ m12) {
  const int lane = threadIdx.x & 31;
  const size_t ng = ((size_t)blockIdx.x * kGnThreads + threadIdx.x) >> 5;
  if (ng >= s.N * s.G) return;
  const size_t n = ng / s.G;
  const int c0 = (int)(ng - n * s.G) * s.D;
  double m1 = 0.0, m2 = 0.0;
  for (size_t i = lane; i < (size_t)pieces * s.D; i += 32) {
    const size_t k = i / s.D;
    const int c = c0 + (int)(i - k * s.D);
    const double ga = gamma ? gamma[c] : 1.0;
    m1 += ga * parts[((n * pieces + k) * 2) * s.C + c];
    m2 += ga * parts[((n * pieces + k) * 2 + 1) * s.C + c];
  }
  m1 = shfl_sum(m1);
  m2 = shfl_sum(m2);
  if (lane == 0) {
    const double E = (double)s.P * s.D;
    m12[2 * ng] = m1 / E;
    m12[2 * ng + 1] = m2 / E;
  }
}

// Parameter gradients: parts[rows][2][C] summed over the rows, 32 channels per CTA.
__global__ void __launch_bounds__(kGnThreads)
gn_bwd_params_kernel(const double *__restrict__ parts, size_t rows, int C, double *ggamma, double *gbeta,
                     bool acc_gamma, bool acc_beta) {
  __shared__ double sums[2][8][33];
  const int tx = threadIdx.x, ty = threadIdx.y, c = blockIdx.x * 32 + tx;
  double sb = 0.0, sg = 0.0;
  if (c < C) {
    for (size_t r = ty; r < rows; r += 8) {
      sb += parts[(r * 2) * C + c];
      sg += parts[(r * 2 + 1) * C + c];
    }
  }
  sums[0][ty][tx] = sb;
  sums[1][ty][tx] = sg;
  __syncthreads();
  if (ty < 2 && c < C) {
    double t = 0.0;
    for (int j = 0; j < 8; j++) t += sums[ty][j][tx];
    double *dst = ty == 0 ? gbeta : ggamma;
    const bool acc = ty == 0 ? acc_beta : acc_gamma;
    if (dst) dst[c] = acc ? dst[c] + t : t;
  }
}

// Step 3: the input's gradient.
template <int ACT>
__global__ void __launch_bounds__(kGnThreads)
gn_bwd_apply_kernel(const double *__restrict__ x, const double *__restrict__ gamma,
                    const double *__restrict__ beta, const double *__restrict__ mean,
                    const double *__restrict__ rstd, const double *__restrict__ gy,
                    const double *__restrict__ m12, double *gx, bool accumulate, NormShape s) {
  const int c = blockIdx.x * 32 + threadIdx.x;
  if (c >= s.C) return;
  const int g = c / s.D;
  const double ga = gamma ? gamma[c] : 1.0, be = beta ? beta[c] : 0.0;
  const size_t rows = s.N * s.P;
  for (size_t r = (size_t)blockIdx.y * blockDim.y + threadIdx.y; r < rows; r += (size_t)gridDim.y * blockDim.y) {
    const size_t ng = r / s.P * s.G + g, at = r * s.C + c;
    const double rs = __ldg(rstd + ng), unit = (x[at] - __ldg(mean + ng)) * rs;
    const double u = act_bwd<ACT>(unit * ga + be, gy[at]) * ga;
    const double v = rs * (u - __ldg(m12 + 2 * ng) - unit * __ldg(m12 + 2 * ng + 1));
    gx[at] = accumulate ? gx[at] + v : v;
  }
}

// Rows (n, p) dealt out to CTAs of 8 rows x 32 channels, about sixteen CTAs per SM.
static dim3 rows_grid(const NormShape &s, size_t units) {
  const unsigned gx = (unsigned)((s.C + 31) / 32);
  size_t gy = (size_t)ctx().sm_count * 16 / gx;
  if (gy > units) gy = units;
  if (gy < 1) gy = 1;
  if (gy > 65535) gy = 65535;
  return dim3(gx, (unsigned)gy);
}

static int check_shape(const char *name, size_t N, size_t P, size_t C, size_t G, int act, NormShape *s) {
  if (G == 0 || C == 0 || C % G != 0)
    return fail(MG_ERR_INVALID, "%s: %zu channels do not make %zu groups of equal size", name, C, G);
  if (act != MG_ACT_NONE && act != MG_ACT_RELU && act != MG_ACT_SILU)
    return fail(MG_ERR_INVALID, "%s: unknown activation %d", name, act);
  const size_t lim = (size_t)1 << 30;
  if (C >= lim || P >= lim || N >= lim || (N && P > (((size_t)1 << 60) / C) / N))
    return fail(MG_ERR_INVALID, "%s: dimension too large", name);
  // (one CTA per group in the general form's first launch)
  if (N * G >= ((size_t)1 << 31)) return fail(MG_ERR_INVALID, "%s: too many groups (%zu)", name, N * G);
  *s = {N, P, (int)C, (int)G, (int)(C / G)};
  return MG_OK;
}

template <class F> static int by_activation(int act, F &&f) {
  if (act == MG_ACT_RELU) return f(std::integral_constant<int, MG_ACT_RELU>());
  if (act == MG_ACT_SILU) return f(std::integral_constant<int, MG_ACT_SILU>());
  return f(std::integral_constant<int, MG_ACT_NONE>());
}

static int scratch(size_t elems, double **out) {
  Context &c = ctx();
  int rc = ensure_scratch(&c.norm_scratch, &c.norm_scratch_elems, elems);
  *out = c.norm_scratch;
  return rc;
}

static int general_fwd(const double *x, const double *gamma, const double *beta, double *y, double *mean,
                       double *rstd, const NormShape &s, double eps, int act) {
  Context &c = ctx();
  const size_t E = s.P * (size_t)s.D, groups = s.N * s.G;
  size_t pieces = (E + kGnPiece - 1) / kGnPiece;
  if (pieces > 65535) pieces = 65535;
  const size_t piece = (E + pieces - 1) / pieces;
  pieces = (E + piece - 1) / piece;
  double *parts = nullptr;
  if (pieces > 1) {
    int rc = scratch(3 * groups * pieces, &parts);
    if (rc != MG_OK) return rc;
  }
  gn_moments_kernel<<<dim3((unsigned)groups, (unsigned)pieces), kGnThreads, 0, c.stream>>>(
      x, s, piece, parts, eps, mean, rstd);
  MG_LAUNCH_CHECK("group_norm moments");
  if (pieces > 1) {
    gn_moments_join_kernel<<<(unsigned)((groups * 32 + kGnThreads - 1) / kGnThreads), kGnThreads, 0, c.stream>>>(
        parts, groups, (unsigned)pieces, eps, mean, rstd);
    MG_LAUNCH_CHECK("group_norm moments join");
  }
  return by_activation(act, [&](auto a) {
    gn_apply_kernel<decltype(a)::value><<<rows_grid(s, (s.N * s.P + 7) / 8), dim3(32, 8), 0, c.stream>>>(
        x, gamma, beta, mean, rstd, y, s);
    MG_LAUNCH_CHECK("group_norm apply");
    return MG_OK;
  });
}

static int general_bwd(const double *x, const double *gamma, const double *beta, const double *mean,
                       const double *rstd, const double *gy, double *gx, double *ggamma, double *gbeta,
                       const NormShape &s, int act, int flags) {
  Context &c = ctx();
  // A piece of 256 positions costs 16 C bytes of sums for 4096 C bytes of data.
  const size_t piece = 256, pieces = (s.P + piece - 1) / piece, rows = s.N * pieces;
  double *parts = nullptr;
  int rc = scratch(rows * 2 * s.C + 2 * s.N * s.G, &parts);
  if (rc != MG_OK) return rc;
  double *m12 = parts + rows * 2 * s.C;
  rc = by_activation(act, [&](auto a) {
    gn_bwd_sums_kernel<decltype(a)::value><<<rows_grid(s, rows), dim3(32, 8), 0, c.stream>>>(
        x, gamma, beta, mean, rstd, gy, s, (unsigned)pieces, piece, parts);
    MG_LAUNCH_CHECK("group_norm backward sums");
    return MG_OK;
  });
  if (rc != MG_OK) return rc;
  if (ggamma || gbeta) {
    gn_bwd_params_kernel<<<(unsigned)((s.C + 31) / 32), dim3(32, 8), 0, c.stream>>>(
        parts, rows, s.C, ggamma, gbeta, !(flags & MG_ACC_STORE_B), !(flags & MG_ACC_STORE_C));
    MG_LAUNCH_CHECK("group_norm parameter gradients");
  }
  if (!gx) return MG_OK;
  gn_bwd_groups_kernel<<<(unsigned)((s.N * s.G * 32 + kGnThreads - 1) / kGnThreads), kGnThreads, 0, c.stream>>>(
      parts, gamma, s, (unsigned)pieces, m12);
  MG_LAUNCH_CHECK("group_norm backward groups");
  return by_activation(act, [&](auto a) {
    gn_bwd_apply_kernel<decltype(a)::value><<<rows_grid(s, (s.N * s.P + 7) / 8), dim3(32, 8), 0, c.stream>>>(
        x, gamma, beta, mean, rstd, gy, m12, gx, !(flags & MG_ACC_STORE_A), s);
    MG_LAUNCH_CHECK("group_norm backward apply");
    return MG_OK;
  });
}

}  // namespace mg

using namespace mg;

extern "C" {

int mg_group_norm_fwd(const double *x, const double *gamma, const double *beta, double *y, double *mean,
                      double *rstd, size_t N, size_t P, size_t C, size_t G, double eps, int act) {
  NormShape s;
  int rc = check_shape("mg_group_norm_fwd", N, P, C, G, act, &s);
  if (rc != MG_OK) return rc;
  if (!(eps >= 0.0)) return fail(MG_ERR_INVALID, "mg_group_norm_fwd: eps must not be negative");
  if (N && P && (!x || !y || !mean || !rstd)) return fail(MG_ERR_INVALID, "mg_group_norm_fwd: null pointer");
  MG_ENSURE_INIT();
  if (N == 0 || P == 0) return MG_OK;
  return general_fwd(x, gamma, beta, y, mean, rstd, s, eps, act);
}

int mg_group_norm_bwd(const double *x, const double *gamma, const double *beta, const double *mean,
                      const double *rstd, const double *gy, double *gx, double *ggamma, double *gbeta,
                      size_t N, size_t P, size_t C, size_t G, int act, int flags) {
  NormShape s;
  int rc = check_shape("mg_group_norm_bwd", N, P, C, G, act, &s);
  if (rc != MG_OK) return rc;
  if (N && P && (gx || ggamma || gbeta) && (!x || !mean || !rstd || !gy))
    return fail(MG_ERR_INVALID, "mg_group_norm_bwd: null pointer");
  MG_ENSURE_INIT();
  if (!gx && !ggamma && !gbeta) return MG_OK;
  if (N == 0 || P == 0) {
    // No data: a destination that may be stored to holds a sum of nothing.
    if (ggamma && (flags & MG_ACC_STORE_B)) rc = mg_fill(ggamma, 0.0, C);
    if (rc == MG_OK && gbeta && (flags & MG_ACC_STORE_C)) rc = mg_fill(gbeta, 0.0, C);
    return rc;
  }
  return general_bwd(x, gamma, beta, mean, rstd, gy, gx, ggamma, gbeta, s, act, flags);
}

}  // extern "C"
