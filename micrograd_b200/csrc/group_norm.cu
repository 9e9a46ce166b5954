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

#include <cooperative_groups.h>

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

// 1 / (1 + exp(-z)) in about 26 fp64 instructions, against some 45 for the library's exp
// and a division: these kernels have 45 (forward) to 68 (backward) per element.  With
// a = |z| and -a = k ln 2 + r, |r| <= 0.35: exp(-a) = 2^k exp(r), exp(r) by its Taylor
// series to r^13 / 13! (the rest is below 2^-56); then n / (1 + exp(-a)) with n = 1 or
// exp(-a) by one Newton step on the hardware's first guess and one correction of the
// quotient by its remainder.  ln 2 is taken in two parts, its first 40 binary places and
// the rest, so that k times the first (k has ten bits) is exact.
// From |z| = 708 on exp(-a) counts as 0 (2^k would not be a normal number), which takes at
// most 2.4e-305 from a value z or a derivative formed with it.  It has to be 0 and
// nothing that is left over: z may be anything up to the largest number.  z = -infinity
// gives 0, and so NaN times z, as the definition does; NaN stays NaN in z.
__device__ __forceinline__ double sigmoid_onepath(double z) {
  // (compared as integers: the fp64 units have enough to do)
  const bool in = (__double2hiint(z) & 0x7fffffff) < 0x40862000;  // high word of 708.0
  const double a = in ? fabs(z) : 708.0;
  const double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
  const double km = fma(a, -1.4426950408889634, kMagic);  // 1 / ln 2
  const double kd = km - kMagic;
  double r = fma(kd, -0x1.62e42fefa4000p-1, -a);
  r = fma(kd, 0x1.8432a1b0e2634p-43, r);  // (the first places are rounded up)
  double q = 1.0 / 6227020800.0;
  q = fma(q, r, 1.0 / 479001600.0);
  q = fma(q, r, 1.0 / 39916800.0);
  q = fma(q, r, 1.0 / 3628800.0);
  q = fma(q, r, 1.0 / 362880.0);
  q = fma(q, r, 1.0 / 40320.0);
  q = fma(q, r, 1.0 / 5040.0);
  q = fma(q, r, 1.0 / 720.0);
  q = fma(q, r, 1.0 / 120.0);
  q = fma(q, r, 1.0 / 24.0);
  q = fma(q, r, 1.0 / 6.0);
  q = fma(q, r, 0.5);
  const double p = fma(r * r, q, r);  // exp(r) - 1
  const double s = __hiloint2double(in ? (__double2loint(km) + 1023) << 20 : 0, 0);  // 2^k, k in [-1021, 0], or 0
  const double e = fma(s, p, s), d = 1.0 + e, n = __double2hiint(z) < 0 ? e : 1.0;
  double y;
  asm("rcp.approx.ftz.f64 %0, %1;" : "=d"(y) : "d"(d));
  y = fma(y, fma(-d, y, 1.0), y);
  const double t = n * y;
  return fma(fma(-d, t, n), y, t);
}

template <int ACT> __device__ __forceinline__ double act_fwd(double z) {
  if (ACT == MG_ACT_RELU) return z > 0 ? z : (z == z ? 0.0 : z);
  if (ACT == MG_ACT_SILU) return z * sigmoid_onepath(z);
  return z;
}

template <int ACT> __device__ __forceinline__ double act_bwd(double z, double g) {
  if (ACT == MG_ACT_RELU) return z > 0 ? g : g * 0.0;
  if (ACT == MG_ACT_SILU) {
    const double s = sigmoid_onepath(z);
    return g * (s * fma(z, 1.0 - s, 1.0));
  }
  return g;
}

struct NormShape {
  size_t N, P;
  int C, G, D;
};

// ---------------------------------------------------------------------------
// General form: what the one-pass forms below do not take, that is groups beyond the
// shared memory of eight CTAs and rows of more than 512 threads' channels (1024 channels
// a group in the gradients, 2048 forward; 512 where their number is odd).  x is read two
// or three times forward (the second time of a piece from L2), and x and gy twice in the
// gradients: 40 bytes per value.  65 536 x 2048 in one group, SiLU: forward 0.91 ms,
// gradients 1.79, against 0.33 and 0.49 for what has to be moved.
// ---------------------------------------------------------------------------
constexpr int kGnThreads = 256;
// Values of a group that one CTA takes: 64 KB, so that its second look at them comes
// from L2.
constexpr size_t kGnPiece = 8192;

// Forward, step 1: moments of one piece of one group.
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

// Backward, step 1: sums of u and u unit over one piece of one group; with one piece they
// are its m1 and m2.
template <int ACT>
__global__ void __launch_bounds__(kGnThreads)
gn_bwd_groups_kernel(const double *__restrict__ x, const double *__restrict__ gamma,
                     const double *__restrict__ beta, const double *__restrict__ mean,
                     const double *__restrict__ rstd, const double *__restrict__ gy, NormShape s,
                     size_t piece, double *__restrict__ parts, double *__restrict__ m12) {
  __shared__ double smem32[32];
  const size_t ng = blockIdx.x, n = ng / s.G;
  const int c0 = (int)(ng - n * s.G) * s.D;
  const size_t E = s.P * (size_t)s.D;
  const size_t begin = blockIdx.y * piece, end = begin + piece < E ? begin + piece : E;
  const double mu = mean[ng], rs = rstd[ng];
  // Position and channel of the values e, e + kGnThreads, ... without a division for each.
  size_t e = begin + threadIdx.x, at = e / s.D;
  int d = (int)(e - at * s.D);
  at = (n * s.P + at) * s.C + c0;
  const int rows = kGnThreads / s.D, columns = kGnThreads - rows * s.D;
  double s1 = 0.0, s2 = 0.0;
  for (; e < end; e += kGnThreads) {
    const double ga = gamma ? __ldg(gamma + c0 + d) : 1.0, be = beta ? __ldg(beta + c0 + d) : 0.0;
    const double unit = (x[at + d] - mu) * rs, u = act_bwd<ACT>(fma(unit, ga, be), gy[at + d]) * ga;
    s1 += u;
    s2 = fma(u, unit, s2);
    at += (size_t)rows * s.C;
    d += columns;
    if (d >= s.D) {
      d -= s.D;
      at += s.C;
    }
  }
  s1 = cta_sum(s1, smem32);
  s2 = cta_sum(s2, smem32);
  if (threadIdx.x != 0) return;
  double *out = gridDim.y == 1 ? m12 + 2 * ng : parts + 2 * (ng * gridDim.y + blockIdx.y);
  out[0] = gridDim.y == 1 ? s1 / (double)E : s1;
  out[1] = gridDim.y == 1 ? s2 / (double)E : s2;
}

// Step 2: the pieces of a group joined, a warp per group.
__global__ void __launch_bounds__(kGnThreads)
gn_bwd_groups_join_kernel(const double *__restrict__ parts, size_t groups, unsigned pieces, double E,
                          double *__restrict__ m12) {
  const int lane = threadIdx.x & 31;
  const size_t ng = ((size_t)blockIdx.x * kGnThreads + threadIdx.x) >> 5;
  if (ng >= groups) return;
  double s1 = 0.0, s2 = 0.0;
  for (unsigned k = lane; k < pieces; k += 32) {
    s1 += parts[2 * (ng * pieces + k)];
    s2 += parts[2 * (ng * pieces + k) + 1];
  }
  s1 = shfl_sum(s1);
  s2 = shfl_sum(s2);
  if (lane == 0) {
    m12[2 * ng] = s1 / E;
    m12[2 * ng + 1] = s2 / E;
  }
}

// Parameter gradients: parts[rows][2][C] summed over the rows, 32 channels per CTA, a
// warp for every kParamRows-th row.  With gridDim.y > 1 each layer of CTAs takes a range
// of the rows and leaves joined[layer][2][C] for a second launch over the layers.
constexpr int kParamRows = 32;

__global__ void __launch_bounds__(32 * kParamRows)
gn_bwd_params_kernel(const double *__restrict__ parts, size_t rows, int C, double *ggamma, double *gbeta,
                     bool acc_gamma, bool acc_beta, double *__restrict__ joined) {
  cudaGridDependencySynchronize();
  __shared__ double sums[2][kParamRows][33];
  const int tx = threadIdx.x, ty = threadIdx.y, c = blockIdx.x * 32 + tx;
  const size_t begin = rows * blockIdx.y / gridDim.y, end = rows * (blockIdx.y + 1) / gridDim.y;
  double sb = 0.0, sg = 0.0;
  if (c < C) {
#pragma unroll 4
    for (size_t r = begin + ty; r < end; r += kParamRows) {
      sb += parts[(r * 2) * C + c];
      sg += parts[(r * 2 + 1) * C + c];
    }
  }
  sums[0][ty][tx] = sb;
  sums[1][ty][tx] = sg;
  __syncthreads();
  if (ty < 2 && c < C) {
    double t = 0.0;
    for (int j = 0; j < kParamRows; j++) t += sums[ty][j][tx];
    if (joined) {
      joined[((size_t)blockIdx.y * 2 + ty) * C + c] = t;
      return;
    }
    double *dst = ty == 0 ? gbeta : ggamma;
    const bool acc = ty == 0 ? acc_beta : acc_gamma;
    if (dst) dst[c] = acc ? dst[c] + t : t;
  }
}

// Layers that the rows are cut into: a CTA alone takes 0.25 us for 32 rows.
static size_t param_layers(size_t rows) {
  const size_t layers = rows / 128;
  return layers < 2 ? 1 : (layers > 64 ? 64 : layers);
}

// parts has room for param_layers(rows) more rows behind the `rows` it holds.
static int sum_params(double *parts, size_t rows, int C, double *ggamma, double *gbeta, int flags) {
  const bool acc_gamma = !(flags & MG_ACC_STORE_B), acc_beta = !(flags & MG_ACC_STORE_C);
  const unsigned wide = (unsigned)((C + 31) / 32), layers = (unsigned)param_layers(rows);
  if (layers > 1) {
    double *joined = parts + rows * 2 * C;
    MG_CUDA_TRY(launch_overlapped(gn_bwd_params_kernel, dim3(wide, layers), dim3(32, kParamRows), parts, rows, C, nullptr,
                                  nullptr, false, false, joined));
    MG_LAUNCH_CHECK("group_norm parameter gradients");
    parts = joined;
    rows = layers;
  }
  MG_CUDA_TRY(launch_overlapped(gn_bwd_params_kernel, dim3(wide), dim3(32, kParamRows), parts, rows, C, ggamma, gbeta,
                                acc_gamma, acc_beta, nullptr));
  MG_LAUNCH_CHECK("group_norm parameter gradients");
  return MG_OK;
}

// Step 3: the input's gradient (gx may be null), and the sums of gz and gz unit over the
// rows (n, p) that a CTA walks, per channel: parts[blockIdx.y][2][C] (or null).  The sums
// stay in the threads until the end, so that they take no more memory than there are CTAs.
template <int ACT>
__global__ void __launch_bounds__(kGnThreads)
gn_bwd_apply_kernel(const double *__restrict__ x, const double *__restrict__ gamma,
                    const double *__restrict__ beta, const double *__restrict__ mean,
                    const double *__restrict__ rstd, const double *__restrict__ gy,
                    const double *__restrict__ m12, double *gx, bool accumulate, NormShape s,
                    double *__restrict__ parts) {
  __shared__ double sums[2][8][33];
  const int tx = threadIdx.x, ty = threadIdx.y, c = blockIdx.x * 32 + tx;
  double sb = 0.0, sg = 0.0;
  if (c < s.C) {
    const int g = c / s.D;
    const double ga = gamma ? gamma[c] : 1.0, be = beta ? beta[c] : 0.0;
    const size_t rows = s.N * s.P, step = (size_t)gridDim.y * 8, step_n = step / s.P, step_p = step - step_n * s.P;
    size_t r = (size_t)blockIdx.y * 8 + ty, n = r / s.P, p = r - n * s.P;
    for (; r < rows; r += step) {
      const size_t ng = n * s.G + g, at = r * s.C + c;
      const double rs = __ldg(rstd + ng), unit = (x[at] - __ldg(mean + ng)) * rs;
      const double gz = act_bwd<ACT>(fma(unit, ga, be), gy[at]);
      sb += gz;
      sg = fma(gz, unit, sg);
      if (gx) {
        const double v = rs * (gz * ga - __ldg(m12 + 2 * ng) - unit * __ldg(m12 + 2 * ng + 1));
        gx[at] = accumulate ? gx[at] + v : v;
      }
      n += step_n;
      p += step_p;
      if (p >= s.P) {
        p -= s.P;
        n++;
      }
    }
  }
  if (!parts) return;
  sums[0][ty][tx] = sb;
  sums[1][ty][tx] = sg;
  __syncthreads();
  if (ty < 2 && c < s.C) {
    double t = 0.0;
    for (int j = 0; j < 8; j++) t += sums[ty][j][tx];
    parts[((size_t)blockIdx.y * 2 + ty) * s.C + c] = t;
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
  const size_t E = s.P * (size_t)s.D, groups = s.N * s.G;
  size_t pieces = (E + kGnPiece - 1) / kGnPiece;
  if (pieces > 65535) pieces = 65535;
  const size_t piece = (E + pieces - 1) / pieces;
  pieces = (E + piece - 1) / piece;
  const dim3 grid = rows_grid(s, (s.N * s.P + 7) / 8);
  const size_t n_rows = (grid.y + param_layers(grid.y)) * 2 * (size_t)s.C;
  double *parts = nullptr;
  int rc = scratch(n_rows + 2 * groups * (pieces > 1 ? pieces + 1 : 1), &parts);
  if (rc != MG_OK) return rc;
  double *m12 = parts + n_rows, *piece_sums = m12 + 2 * groups;
  if (gx) {
    rc = by_activation(act, [&](auto a) {
      gn_bwd_groups_kernel<decltype(a)::value><<<dim3((unsigned)groups, (unsigned)pieces), kGnThreads, 0, c.stream>>>(
          x, gamma, beta, mean, rstd, gy, s, piece, piece_sums, m12);
      MG_LAUNCH_CHECK("group_norm backward groups");
      return MG_OK;
    });
    if (rc != MG_OK) return rc;
    if (pieces > 1) {
      gn_bwd_groups_join_kernel<<<(unsigned)((groups * 32 + kGnThreads - 1) / kGnThreads), kGnThreads, 0, c.stream>>>(
          piece_sums, groups, (unsigned)pieces, (double)E, m12);
      MG_LAUNCH_CHECK("group_norm backward groups join");
    }
  }
  const bool params = ggamma || gbeta;
  rc = by_activation(act, [&](auto a) {
    gn_bwd_apply_kernel<decltype(a)::value><<<grid, dim3(32, 8), 0, c.stream>>>(
        x, gamma, beta, mean, rstd, gy, m12, gx, !(flags & MG_ACC_STORE_A), s, params ? parts : nullptr);
    MG_LAUNCH_CHECK("group_norm backward apply");
    return MG_OK;
  });
  if (rc != MG_OK || !params) return rc;
  return sum_params(parts, grid.y, s.C, ggamma, gbeta, flags);
}

// ---------------------------------------------------------------------------
// What the two one-pass forms below share.  A thread keeps VEC neighbouring channels
// and takes every TY-th position, so its channels' parameters, and the sums of their
// gradients, stay in registers while it walks the samples n0, n0 + nstep, ...
// ---------------------------------------------------------------------------
struct TeamArgs {
  const double *x, *gamma, *beta, *gy;
  double *mean, *rstd;  // outputs of the forward pass, inputs of the backward pass
  double *out;          // y or gx
  double *parts;        // backward: [nstep * CS][2][C], or null
  size_t N, P, Pc, nstep;
  int C, G, D, Dv, TY, logL;
  double eps, inv_E;
  bool accumulate;
};

template <int VEC> struct Pack {
  double v[VEC];
};
__device__ __forceinline__ Pack<1> load_pack(const Pack<1> *p) { return {{__ldcs(&p->v[0])}}; }
__device__ __forceinline__ Pack<2> load_pack(const Pack<2> *p) {
  const double2 t = __ldcs(reinterpret_cast<const double2 *>(p));
  return {{t.x, t.y}};
}
__device__ __forceinline__ Pack<4> load_pack(const Pack<4> *p) {
  const double4v t = ld_stream_v4(reinterpret_cast<const double4v *>(p));
  return {{t.x, t.y, t.z, t.w}};
}
__device__ __forceinline__ void store_pack(Pack<1> *p, const Pack<1> &t) { __stcs(&p->v[0], t.v[0]); }
__device__ __forceinline__ void store_pack(Pack<2> *p, const Pack<2> &t) {
  __stcs(reinterpret_cast<double2 *>(p), make_double2(t.v[0], t.v[1]));
}
__device__ __forceinline__ void store_pack(Pack<4> *p, const Pack<4> &t) {
  st_stream_v4(reinterpret_cast<double4v *>(p), double4v{t.v[0], t.v[1], t.v[2], t.v[3]});
}

// One value's gradient up to the group's means: unit and gz = gy act'(z).
template <int ACT>
__device__ __forceinline__ double grad_z(double x, double gy, double mean, double rstd, double ga, double be,
                                         double &unit) {
  unit = (x - mean) * rstd;
  return act_bwd<ACT>(fma(unit, ga, be), gy);
}

// Writes the channel sums of the threads that share a channel (tx, all ty) in the order
// of ty: row[c + v] = sum of sum_b, row[C + c + v] = sum of sum_g.  All threads of the
// CTA call it; chan has room for 2 VEC doubles each.
template <int VEC>
__device__ __forceinline__ void write_channel_sums(const double (&sum_b)[VEC], const double (&sum_g)[VEC], double *chan,
                                                   int Dv, int TY, bool writer, double *row, int c, int C) {
  double *mine = chan + 2 * VEC * threadIdx.x;
#pragma unroll
  for (int v = 0; v < VEC; v++) {
    mine[2 * v] = sum_b[v];
    mine[2 * v + 1] = sum_g[v];
  }
  __syncthreads();
  if (!writer) return;
#pragma unroll
  for (int v = 0; v < VEC; v++) {
    double b = 0.0, w = 0.0;
    for (int t = 0; t < TY; t++) {
      b += mine[2 * VEC * (size_t)t * Dv + 2 * v];
      w += mine[2 * VEC * (size_t)t * Dv + 2 * v + 1];
    }
    row[c + v] = b;
    row[C + c + v] = w;
  }
}

// ---------------------------------------------------------------------------
// Warp form, for groups of up to 32 x 8 values: a team of L = 2^logL
// lanes of one warp holds U samples of a group in registers, R positions of each per
// lane.  x (and gy) is read once, y (gx) written once, nothing meets at a barrier.
// ---------------------------------------------------------------------------
constexpr int kWarpFormThreads = 256;

template <int K> __device__ __forceinline__ void lanes_sum(double (&v)[K], int width) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    if (off < width) {
#pragma unroll
      for (int k = 0; k < K; k++) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
    }
}

template <int VEC, int U, int R, int ACT, bool BWD>
__global__ void __launch_bounds__(kWarpFormThreads, BWD ? 2 : 4) gn_warp_kernel(const TeamArgs a) {
  __shared__ double chan[BWD ? 2 * VEC * kWarpFormThreads : 1];
  cudaGridDependencySynchronize();
  const int width = 1 << a.logL, l = threadIdx.x & (width - 1), ty = l / a.Dv, tx = l - ty * a.Dv;
  const size_t team = ((size_t)blockIdx.x * kWarpFormThreads + threadIdx.x) >> a.logL;
  const size_t n0 = team / a.G;
  const int g = (int)(team - n0 * a.G);
  const bool live = n0 < a.nstep && ty < a.TY;
  const int c = g * a.D + tx * VEC;
  // (positions fit an int: a group has at most 32 x 8 values here)
  const int P = (int)a.P;
  const size_t step_n = a.nstep * a.P * a.C, step_p = (size_t)a.TY * a.C;
  size_t at0 = (n0 * a.P + ty) * a.C + c;

  double ga[VEC], be[VEC], sum_b[VEC], sum_g[VEC];
#pragma unroll
  for (int v = 0; v < VEC; v++) {
    ga[v] = a.gamma && live ? __ldg(a.gamma + c + v) : 1.0;
    be[v] = a.beta && live ? __ldg(a.beta + c + v) : 0.0;
    sum_b[v] = sum_g[v] = 0.0;
  }
  // All lanes make the same number of rounds (they shuffle together).
  for (size_t n = n0; n - n0 < a.N; n += a.nstep * U, at0 += step_n * U) {
    Pack<VEC> x[U][R], gy[BWD ? U : 1][BWD ? R : 1];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const bool in = live && n + u * a.nstep < a.N;
#pragma unroll
      for (int i = 0; i < R; i++) {
        const size_t at = at0 + u * step_n + i * step_p;
        if (in && ty + i * a.TY < P) {
          x[u][i] = load_pack(reinterpret_cast<const Pack<VEC> *>(a.x + at));
          if (BWD) gy[u][i] = load_pack(reinterpret_cast<const Pack<VEC> *>(a.gy + at));
        } else {
#pragma unroll
          for (int v = 0; v < VEC; v++) {
            x[u][i].v[v] = 0.0;
            if (BWD) gy[u][i].v[v] = 0.0;
          }
        }
      }
    }
    if constexpr (!BWD) {
      double s[U], mean[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        s[u] = 0.0;
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
          for (int v = 0; v < VEC; v++) s[u] += x[u][i].v[v];
      }
      lanes_sum<U>(s, width);
#pragma unroll
      for (int u = 0; u < U; u++) {
        mean[u] = s[u] * a.inv_E;
        s[u] = 0.0;
#pragma unroll
        for (int i = 0; i < R; i++) {
          if (ty < a.TY && ty + i * a.TY < P) {
#pragma unroll
            for (int v = 0; v < VEC; v++) {
              x[u][i].v[v] -= mean[u];
              s[u] = fma(x[u][i].v[v], x[u][i].v[v], s[u]);
            }
          }
        }
      }
      lanes_sum<U>(s, width);
#pragma unroll
      for (int u = 0; u < U; u++) {
        const size_t nu = n + u * a.nstep;
        if (!(live && nu < a.N)) continue;
        const double rstd = 1.0 / sqrt(fma(s[u], a.inv_E, a.eps));
        if (l == 0) {
          a.mean[nu * a.G + g] = mean[u];
          a.rstd[nu * a.G + g] = rstd;
        }
#pragma unroll
        for (int i = 0; i < R; i++) {
          if (ty + i * a.TY < P) {
            Pack<VEC> y;
#pragma unroll
            for (int v = 0; v < VEC; v++) y.v[v] = act_fwd<ACT>(fma(x[u][i].v[v] * rstd, ga[v], be[v]));
            store_pack(reinterpret_cast<Pack<VEC> *>(a.out + at0 + u * step_n + i * step_p), y);
          }
        }
      }
    } else {
      double s[2 * U], rstd[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const bool in = live && n + u * a.nstep < a.N;
        const size_t ng = (n + u * a.nstep) * a.G + g;
        const double mean = in ? __ldg(a.mean + ng) : 0.0;
        rstd[u] = in ? __ldg(a.rstd + ng) : 0.0;
        double b[VEC], w[VEC];
#pragma unroll
        for (int v = 0; v < VEC; v++) b[v] = w[v] = 0.0;
#pragma unroll
        for (int i = 0; i < R; i++) {
          if (in && ty + i * a.TY < P) {
#pragma unroll
            for (int v = 0; v < VEC; v++) {
              double unit;
              const double gz = grad_z<ACT>(x[u][i].v[v], gy[u][i].v[v], mean, rstd[u], ga[v], be[v], unit);
              b[v] += gz;
              w[v] = fma(gz, unit, w[v]);
              x[u][i].v[v] = unit;
              gy[u][i].v[v] = gz * ga[v];
            }
          }
        }
        s[2 * u] = s[2 * u + 1] = 0.0;
#pragma unroll
        for (int v = 0; v < VEC; v++) {
          sum_b[v] += b[v];
          sum_g[v] += w[v];
          s[2 * u] = fma(b[v], ga[v], s[2 * u]);
          s[2 * u + 1] = fma(w[v], ga[v], s[2 * u + 1]);
        }
      }
      if (!a.out) continue;
      lanes_sum<2 * U>(s, width);
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (!(live && n + u * a.nstep < a.N)) continue;
        const double m1 = s[2 * u] * a.inv_E, m2 = s[2 * u + 1] * a.inv_E;
#pragma unroll
        for (int i = 0; i < R; i++) {
          if (ty + i * a.TY < P) {
            Pack<VEC> *dst = reinterpret_cast<Pack<VEC> *>(a.out + at0 + u * step_n + i * step_p);
            Pack<VEC> r;
#pragma unroll
            for (int v = 0; v < VEC; v++) r.v[v] = rstd[u] * fma(-m2, x[u][i].v[v], gy[u][i].v[v] - m1);
            if (a.accumulate) {
              const Pack<VEC> old = load_pack(dst);
#pragma unroll
              for (int v = 0; v < VEC; v++) r.v[v] = old.v[v] + r.v[v];
            }
            store_pack(dst, r);
          }
        }
      }
    }
  }
  if constexpr (BWD) {
    if (a.parts)
      write_channel_sums<VEC>(sum_b, sum_g, chan, a.Dv, a.TY, live && ty == 0,
                              a.parts + n0 * 2 * (size_t)a.C, c, a.C);
  }
}

// ---------------------------------------------------------------------------
// Tile form, for larger groups: a CTA, or CS of them as a cluster, has all of a group's
// values in shared memory, brought there by asynchronous copies.  Every thread fetches,
// rewrites and reads only its own cells, so the barriers are those of the sums.
// ---------------------------------------------------------------------------
constexpr int kTileThreads = 512;

// A cell of a thread: chunks of 16 bytes (8 with VEC = 1), the threads of the CTA next
// to each other within a chunk, so that no access conflicts.  Addresses are those of
// the shared window (32 bits).
template <int VEC> __device__ __forceinline__ void fetch_cell(uint32_t cell, uint32_t half, const double *src) {
  if (VEC == 1) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(cell), "l"(src) : "memory");
  } else {
#pragma unroll
    for (int h = 0; h < VEC / 2; h++)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(cell + h * half), "l"(src + 2 * h) : "memory");
  }
}
template <int VEC> __device__ __forceinline__ Pack<VEC> get_cell(uint32_t cell, uint32_t half) {
  Pack<VEC> r;
  if constexpr (VEC == 1) {
    asm volatile("ld.shared.f64 %0, [%1];" : "=d"(r.v[0]) : "r"(cell) : "memory");
  } else {
#pragma unroll
    for (int h = 0; h < VEC / 2; h++)
      asm volatile("ld.shared.v2.f64 {%0, %1}, [%2];"
                   : "=d"(r.v[2 * h]), "=d"(r.v[2 * h + 1])
                   : "r"(cell + h * half)
                   : "memory");
  }
  return r;
}
template <int VEC> __device__ __forceinline__ void put_cell(uint32_t cell, uint32_t half, const Pack<VEC> &p) {
  if constexpr (VEC == 1) {
    asm volatile("st.shared.f64 [%0], %1;" ::"r"(cell), "d"(p.v[0]) : "memory");
  } else {
#pragma unroll
    for (int h = 0; h < VEC / 2; h++)
      asm volatile("st.shared.v2.f64 [%0], {%1, %2};" ::"r"(cell + h * half), "d"(p.v[2 * h]), "d"(p.v[2 * h + 1])
                   : "memory");
  }
}

// Sums of K values per thread over the CTA (over the cluster), valid in every thread;
// all of them call it.  `phase` alternates between two buffers, so that one barrier per
// call is enough: a buffer is written again only after the barrier of the call in
// between, which all of its readers have passed.
template <int K, int CS>
__device__ __forceinline__ void tile_sum(double (&v)[K], int phase, double (&red)[2][kTileThreads / 32][K],
                                         double (&slot)[2][K]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  lanes_sum<K>(v, 32);
  if (lane == 0) {
#pragma unroll
    for (int k = 0; k < K; k++) red[phase][warp][k] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; k++) v[k] = lane < warps ? red[phase][lane][k] : 0.0;
  lanes_sum<K>(v, 16);  // (at most 16 warps: lanes 16 to 31 hold zeros)
#pragma unroll
  for (int k = 0; k < K; k++) v[k] = __shfl_sync(0xffffffffu, v[k], 0);
  if (CS > 1) {
    namespace cg = cooperative_groups;
    auto cluster = cg::this_cluster();
    if (threadIdx.x == 0) {
#pragma unroll
      for (int k = 0; k < K; k++) slot[phase][k] = v[k];
    }
    cluster.sync();
    double other[CS][K];
#pragma unroll
    for (int r = 0; r < CS; r++) {
      const double *p = cluster.map_shared_rank(&slot[phase][0], r);
#pragma unroll
      for (int k = 0; k < K; k++) other[r][k] = p[k];
    }
#pragma unroll
    for (int k = 0; k < K; k++) {
      v[k] = 0.0;
#pragma unroll
      for (int r = 0; r < CS; r++) v[k] += other[r][k];
    }
  }
}

template <int VEC, int ACT, bool BWD, int CS>
__global__ void __launch_bounds__(kTileThreads, 2) gn_tile_kernel(const TeamArgs a) {
  constexpr int K = BWD ? 2 : 1;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ double red[2][kTileThreads / 32][K];
  __shared__ double slot[2][K];
  cudaGridDependencySynchronize();
  const int ty = threadIdx.x / a.Dv, tx = threadIdx.x - ty * a.Dv;
  const size_t team = blockIdx.x / CS, n0 = team / a.G;
  const int g = (int)(team - n0 * a.G), rank = CS > 1 ? (int)(blockIdx.x % CS) : 0;
  const int c = g * a.D + tx * VEC;
  const size_t p0 = (size_t)rank * a.Pc, p1 = p0 + a.Pc < a.P ? p0 + a.Pc : a.P;
  // cells of this thread: positions p0 + ty, p0 + ty + TY, ... below p1
  const int cells = ty < a.TY && p0 + ty < p1 ? (int)((p1 - p0 - ty + a.TY - 1) / a.TY) : 0;
  const int most = (int)((a.Pc + a.TY - 1) / a.TY);
  const size_t step_n = a.nstep * a.P * a.C, step_p = (size_t)a.TY * a.C;
  size_t at0 = (n0 * a.P + p0 + ty) * a.C + c;
  const uint32_t pitch = blockDim.x * VEC * 8, half = blockDim.x * 16;
  const uint32_t xs = (uint32_t)__cvta_generic_to_shared(smem) + threadIdx.x * (VEC == 1 ? 8 : 16);
  const uint32_t to_gy = (uint32_t)most * pitch;  // from a cell of x to the one of gy

  double ga[VEC], be[VEC], sum_b[VEC], sum_g[VEC];
#pragma unroll
  for (int v = 0; v < VEC; v++) {
    ga[v] = a.gamma && cells ? __ldg(a.gamma + c + v) : 1.0;
    be[v] = a.beta && cells ? __ldg(a.beta + c + v) : 0.0;
    sum_b[v] = sum_g[v] = 0.0;
  }
  auto fetch_all = [&](size_t at) {
    const double *px = a.x + at, *pg = BWD ? a.gy + at : nullptr;
    uint32_t cell = xs;
    for (int i = 0; i < cells; i++, cell += pitch) {
      fetch_cell<VEC>(cell, half, px);
      px += step_p;
      if (BWD) {
        fetch_cell<VEC>(cell + to_gy, half, pg);
        pg += step_p;
      }
    }
  };
  int phase = 0;
  // (the same samples in the whole cluster)
  if (n0 < a.N) fetch_all(at0);
  for (size_t n = n0; n < a.N; n += a.nstep, at0 += step_n) {
    asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
    // The last pass over a cell asks for the next sample's values in it: they arrive
    // while the other cells, and the other CTAs of the SM, are at work.  (The stores
    // use what was read from the cell, so the read is over when the copy is issued.)
    const bool more = n + a.nstep < a.N;
    const size_t ng = n * a.G + g;
    if constexpr (!BWD) {
      double s[1] = {0.0};
      uint32_t cell = xs;
#pragma unroll 4
      for (int i = 0; i < cells; i++, cell += pitch) {
        const Pack<VEC> x = get_cell<VEC>(cell, half);
#pragma unroll
        for (int v = 0; v < VEC; v++) s[0] += x.v[v];
      }
      tile_sum<1, CS>(s, phase, red, slot);
      phase ^= 1;
      const double mean = s[0] * a.inv_E;
      s[0] = 0.0;
      cell = xs;
#pragma unroll 4
      for (int i = 0; i < cells; i++, cell += pitch) {
        const Pack<VEC> x = get_cell<VEC>(cell, half);
#pragma unroll
        for (int v = 0; v < VEC; v++) s[0] = fma(x.v[v] - mean, x.v[v] - mean, s[0]);
      }
      tile_sum<1, CS>(s, phase, red, slot);
      phase ^= 1;
      const double rstd = 1.0 / sqrt(fma(s[0], a.inv_E, a.eps));
      if (threadIdx.x == 0 && rank == 0) {
        a.mean[ng] = mean;
        a.rstd[ng] = rstd;
      }
      double *py = a.out + at0;
      const double *px = a.x + at0 + step_n;
      cell = xs;
#pragma unroll 2
      for (int i = 0; i < cells; i++, cell += pitch) {
        const Pack<VEC> x = get_cell<VEC>(cell, half);
        Pack<VEC> y;
#pragma unroll
        for (int v = 0; v < VEC; v++) y.v[v] = act_fwd<ACT>(fma((x.v[v] - mean) * rstd, ga[v], be[v]));
        store_pack(reinterpret_cast<Pack<VEC> *>(py), y);
        if (more) fetch_cell<VEC>(cell, half, px);
        py += step_p;
        px += step_p;
      }
    } else {
      const double mean = __ldg(a.mean + ng), rstd = __ldg(a.rstd + ng);
      double b[VEC], w[VEC];
#pragma unroll
      for (int v = 0; v < VEC; v++) b[v] = w[v] = 0.0;
      uint32_t cell = xs;
#pragma unroll 2
      for (int i = 0; i < cells; i++, cell += pitch) {
        const Pack<VEC> x = get_cell<VEC>(cell, half);
        Pack<VEC> gy = get_cell<VEC>(cell + to_gy, half);
#pragma unroll
        for (int v = 0; v < VEC; v++) {
          double unit;
          const double gz = grad_z<ACT>(x.v[v], gy.v[v], mean, rstd, ga[v], be[v], unit);
          b[v] += gz;
          w[v] = fma(gz, unit, w[v]);
          gy.v[v] = gz * ga[v];
        }
        put_cell<VEC>(cell + to_gy, half, gy);
      }
      double s[2] = {0.0, 0.0};
#pragma unroll
      for (int v = 0; v < VEC; v++) {
        sum_b[v] += b[v];
        sum_g[v] += w[v];
        s[0] = fma(b[v], ga[v], s[0]);
        s[1] = fma(w[v], ga[v], s[1]);
      }
      if (!a.out) {  // the parameters' gradients alone
        if (more) fetch_all(at0 + step_n);
        continue;
      }
      tile_sum<2, CS>(s, phase, red, slot);
      phase ^= 1;
      const double m1 = s[0] * a.inv_E, m2 = s[1] * a.inv_E;
      double *py = a.out + at0;
      const double *px = a.x + at0 + step_n, *pg = a.gy + at0 + step_n;
      cell = xs;
#pragma unroll 2
      for (int i = 0; i < cells; i++, cell += pitch) {
        const Pack<VEC> x = get_cell<VEC>(cell, half), u = get_cell<VEC>(cell + to_gy, half);
        Pack<VEC> r;
#pragma unroll
        for (int v = 0; v < VEC; v++) r.v[v] = rstd * fma(-m2, (x.v[v] - mean) * rstd, u.v[v] - m1);
        if (a.accumulate) {
          const Pack<VEC> old = load_pack(reinterpret_cast<const Pack<VEC> *>(py));
#pragma unroll
          for (int v = 0; v < VEC; v++) r.v[v] = old.v[v] + r.v[v];
        }
        store_pack(reinterpret_cast<Pack<VEC> *>(py), r);
        if (more) {
          fetch_cell<VEC>(cell, half, px);
          fetch_cell<VEC>(cell + to_gy, half, pg);
        }
        py += step_p;
        px += step_p;
        pg += step_p;
      }
    }
  }
  if constexpr (BWD) {
    if (a.parts) {
      __syncthreads();  // the cells become the room for the channel sums
      write_channel_sums<VEC>(sum_b, sum_g, reinterpret_cast<double *>(smem), a.Dv, a.TY, ty == 0,
                              a.parts + (n0 * CS + rank) * 2 * (size_t)a.C, c, a.C);
    }
  }
  if (CS > 1) cooperative_groups::this_cluster().sync();  // nobody leaves while its sums may be read
}

// ---------------------------------------------------------------------------
// How a shape is dealt out
// ---------------------------------------------------------------------------
enum NormForm { kFormGeneral, kFormWarp, kFormTile };

struct TeamPlan {
  NormForm form;
  int vec, logL, TY, cs, threads;
  bool small;  // warp form: one position per lane, several samples at a time
  size_t Pc, smem;
};

// Values of x a lane holds in the warp form.  65 536 x 1024 in groups of 64, forward:
// 172 us (6.3 TB/s, the rate of a copy) with 8 and four CTAs per SM; 16 values and two
// CTAs took 1.28 times as long, 4 values backward 1.02 times.
constexpr int kWarpValues = 8;

static int log2_ceil(size_t n) {
  int k = 0;
  while (((size_t)1 << k) < n) k++;
  return k;
}

static TeamPlan plan_norm(const NormShape &s, uintptr_t address_bits, bool bwd) {
  TeamPlan t{};
  t.form = kFormGeneral;
  t.cs = 1;
  t.Pc = s.P;
  t.vec = (s.D % 4 == 0 && (address_bits & 31) == 0) ? 4 : (s.D % 2 == 0 && (address_bits & 15) == 0) ? 2 : 1;
  size_t Dv = s.D / t.vec;
  const size_t slots = kWarpValues / t.vec;
  const size_t lanes = Dv * ((s.P + slots - 1) / slots);
  if (lanes <= 32) {
    t.form = kFormWarp;
    t.logL = log2_ceil(lanes);
    t.TY = (1 << t.logL) / (int)Dv;
    t.small = s.P <= (size_t)t.TY;
    t.threads = kWarpFormThreads;
    return t;
  }
  // Backward, four channels' parameters and sums do not fit the registers that 28 warps
  // per SM leave (128 x 784 x 256 in groups of 8 channels with SiLU: 144 us with 16-byte
  // cells and 512 threads, 4.3 TB/s; 32-byte cells and 256 threads took 1.3 times as long).
  // What holds it there is latency: HBM and the fp64 units are both less than half busy
  // (48 and 42 %), and the 26 warps of an SM wait for loads and for dependent results.
  // Forward, where less is kept, CTAs of 256 threads are better (103 us; 512 threads: 1.15
  // times as long).
  if (bwd && t.vec > 2) t.vec = 2;
  Dv = s.D / t.vec;
  if (Dv > (size_t)kTileThreads) return t;
  size_t max_threads = !bwd && Dv <= 256 ? 256 : kTileThreads;
  // Where there are groups for all SMs several times over: as many CTAs per SM as have
  // their groups in its shared memory, and 1024 threads among them, so that one's copies
  // and sums overlap another's arithmetic (33 x 197 positions, 30 groups of 5 channels,
  // backward, 11.8 us; CTAs of 512 threads took 1.3 times as long).
  if (s.N * s.G >= (size_t)ctx().sm_count * 2) {
    const size_t per_sm = (224 << 10) / (s.P * (size_t)s.D * (bwd ? 16 : 8) + 1024);
    size_t fit = per_sm > 1 ? (1024 / per_sm + 31) / 32 * 32 : max_threads;
    if (fit < 64) fit = 64;
    if (fit < Dv) fit = (Dv + 31) / 32 * 32;
    if (fit < max_threads) max_threads = fit;
  }
  // Two CTAs per SM where the group allows it: one computes while the other copies.
  const size_t half = 112 << 10, whole = 224 << 10;
  for (size_t limit : {half, whole}) {
    for (int cs = 1; cs <= 8; cs *= 2) {
      const size_t Pc = (s.P + cs - 1) / cs;
      if (cs > 1 && (size_t)(cs - 1) * Pc >= s.P) break;
      // As many cells per thread as max_threads make necessary, then as few threads as
      // that many cells need: no cell stays empty but in the last of them.
      const size_t most_ty = max_threads / Dv;
      const size_t cells = (Pc + most_ty - 1) / most_ty, TY = (Pc + cells - 1) / cells;
      const size_t threads = (TY * Dv + 31) / 32 * 32;
      size_t smem = cells * threads * t.vec * 8 * (bwd ? 2 : 1);
      if (bwd && smem < threads * t.vec * 16) smem = threads * t.vec * 16;  // channel sums
      if (smem > limit) continue;
      t.form = kFormTile;
      t.cs = cs;
      t.Pc = Pc;
      t.threads = (int)threads;
      t.TY = (int)TY;
      t.smem = smem;
      return t;
    }
  }
  return t;
}

template <int VEC, int U, int R, int ACT, bool BWD>
static int launch_warp(const TeamArgs &a, const TeamPlan &t) {
  const size_t ctas = ((a.nstep * a.G << t.logL) + kWarpFormThreads - 1) / kWarpFormThreads;
  MG_CUDA_TRY(launch_overlapped(gn_warp_kernel<VEC, U, R, ACT, BWD>, dim3((unsigned)ctas), dim3(kWarpFormThreads), a));
  MG_LAUNCH_CHECK("group_norm (warp form)");
  return MG_OK;
}

// CTAs (clusters) of the tile form that are resident at once: 64 registers per thread,
// 228 KB of shared memory per SM (1 KB of it per CTA).
static size_t resident_ctas(const TeamPlan &t) {
  size_t per_sm = 1024 / (size_t)t.threads;
  const size_t by_smem = (228 << 10) / (t.smem + 2048);
  if (by_smem < per_sm) per_sm = by_smem;
  const size_t resident = (size_t)ctx().sm_count * (per_sm ? per_sm : 1) / t.cs;
  return resident ? resident : 1;
}

// Walkers over the samples of the backward pass in the tile form: waves of the resident
// CTAs times samples per walker, and half a sample for the first one's copies that
// nothing overlaps, should be least.
static size_t tile_walkers(const NormShape &s, const TeamPlan &t) {
  const size_t resident = resident_ctas(t);
  size_t best = 1;
  double least = 0.0;
  for (size_t walk = 1; walk <= s.N; walk++) {  // samples per walker
    const size_t n = (s.N + walk - 1) / walk, waves = (n * s.G + resident - 1) / resident;
    const double cost = (double)waves * ((double)walk + 0.5);
    if (least == 0.0 || cost < least) {
      least = cost;
      best = n;
    }
    if (n * s.G <= resident) break;  // one wave: longer walks only idle CTAs
  }
  return best;
}

template <int VEC, int ACT, bool BWD, int CS>
static int launch_tile(const TeamArgs &a, const TeamPlan &t) {
  auto kernel = gn_tile_kernel<VEC, ACT, BWD, CS>;
  static bool configured = false;
  if (!configured) {
    MG_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 << 10));
    configured = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.nstep * a.G * CS));
  cfg.blockDim = dim3((unsigned)t.threads);
  cfg.dynamicSmemBytes = t.smem;
  cfg.stream = ctx().stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // as launch_overlapped
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CS;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CS > 1 ? 2 : 1;
  MG_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a));
  MG_LAUNCH_CHECK("group_norm (tile form)");
  return MG_OK;
}

template <int VEC, int ACT, bool BWD> static int launch_form(const TeamArgs &a, const TeamPlan &t) {
  constexpr int kR = kWarpValues / VEC, kU = kR < 8 ? kR : 8;
  if (t.form == kFormWarp && t.small) return launch_warp<VEC, kU, 1, ACT, BWD>(a, t);
  if (t.form == kFormWarp) return launch_warp<VEC, 1, kR, ACT, BWD>(a, t);
  if (t.cs == 1) return launch_tile<VEC, ACT, BWD, 1>(a, t);
  if (t.cs == 2) return launch_tile<VEC, ACT, BWD, 2>(a, t);
  if (t.cs == 4) return launch_tile<VEC, ACT, BWD, 4>(a, t);
  return launch_tile<VEC, ACT, BWD, 8>(a, t);
}

template <bool BWD> static int run_form(const TeamArgs &a, const TeamPlan &t, int act) {
  return by_activation(act, [&](auto kind) {
    constexpr int ACT = decltype(kind)::value;
    if (t.vec == 4) return launch_form<4, ACT, BWD>(a, t);
    if (t.vec == 2) return launch_form<2, ACT, BWD>(a, t);
    return launch_form<1, ACT, BWD>(a, t);
  });
}

// Samples a team of the warp form has in its registers at a time.
static size_t samples_at_once(const TeamPlan &t) {
  if (t.form != kFormWarp || !t.small) return 1;
  const int most = kWarpValues / t.vec;
  return most < 8 ? most : 8;
}

static uintptr_t bits_of(const void *a, const void *b, const void *c) {
  return reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c);
}

static int one_pass_fwd(const double *x, const double *gamma, const double *beta, double *y, double *mean,
                        double *rstd, const NormShape &s, double eps, int act, const TeamPlan &t) {
  size_t nstep;
  if (t.form == kFormWarp) {
    // About four rounds per team, for which its parameters are loaded once; fewer where
    // that would leave SMs idle.
    const size_t U = samples_at_once(t), fill = (size_t)ctx().sm_count * 4 * (kWarpFormThreads >> t.logL) / s.G;
    nstep = (s.N + 4 * U - 1) / (4 * U);
    if (nstep < fill) nstep = fill < (s.N + U - 1) / U ? fill : (s.N + U - 1) / U;
  } else {
    // The same for CTAs (128 x 784 x 256 in groups of 8: 103 us; one wave of them took
    // 1.1 times as long).
    nstep = resident_ctas(t) / s.G;
    if (nstep > s.N) nstep = s.N;
    if (nstep < (s.N + 3) / 4) nstep = (s.N + 3) / 4;
  }
  const TeamArgs a{x, gamma, beta, nullptr, mean, rstd, y, nullptr, s.N, s.P, t.Pc, nstep, s.C, s.G, s.D,
                   s.D / t.vec, t.TY, t.logL, eps, 1.0 / ((double)s.P * s.D), false};
  return run_form<false>(a, t, act);
}

static int one_pass_bwd(const double *x, const double *gamma, const double *beta, const double *mean,
                        const double *rstd, const double *gy, double *gx, double *ggamma, double *gbeta,
                        const NormShape &s, int act, int flags, const TeamPlan &t) {
  Context &c = ctx();
  // Each of the nstep walkers over the samples leaves a row of sums per channel, so
  // there are no more of them than keep the SMs busy.
  const size_t U = samples_at_once(t);
  size_t nstep;
  if (t.form == kFormWarp) {
    nstep = (size_t)c.sm_count * 2 * (kWarpFormThreads >> t.logL) / s.G;
    if (nstep < 1) nstep = 1;
    const size_t most = (s.N + U - 1) / U;
    if (nstep > most) nstep = most;
  } else {
    nstep = tile_walkers(s, t);
  }
  const size_t rows = nstep * t.cs;
  double *parts = nullptr;
  if (ggamma || gbeta) {
    int rc = scratch((rows + param_layers(rows)) * 2 * s.C, &parts);
    if (rc != MG_OK) return rc;
  }
  const TeamArgs a{x, gamma, beta, gy, const_cast<double *>(mean), const_cast<double *>(rstd), gx, parts,
                   s.N, s.P, t.Pc, nstep, s.C, s.G, s.D, s.D / t.vec, t.TY, t.logL, 0.0,
                   1.0 / ((double)s.P * s.D), !(flags & MG_ACC_STORE_A)};
  int rc = run_form<true>(a, t, act);
  if (rc != MG_OK || !parts) return rc;
  return sum_params(parts, rows, s.C, ggamma, gbeta, flags);
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
  const TeamPlan t = plan_norm(s, bits_of(x, y, nullptr), false);
  if (t.form != kFormGeneral) return one_pass_fwd(x, gamma, beta, y, mean, rstd, s, eps, act, t);
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
  const TeamPlan t = plan_norm(s, bits_of(x, gy, gx), true);
  if (t.form != kFormGeneral)
    return one_pass_bwd(x, gamma, beta, mean, rstd, gy, gx, ggamma, gbeta, s, act, flags, t);
  return general_bwd(x, gamma, beta, mean, rstd, gy, gx, ggamma, gbeta, s, act, flags);
}

}  // extern "C"
