// Activations kept in 8 bits between the forward and the backward pass.
//
// The columns of a row x[M][N] are cut into blocks of MG_Q8_BLOCK = 64 (the last one
// may be shorter).  With a = max |x| over a block:
//
//   scale = a / 127,  code = rint(x (127 / a)),  and code = sign(x) where that
//   rounds to 0 and x is not 0;  the value kept is code * scale.
//
// So a code is at most half a step from x (up to a whole step where a small value is
// kept away from 0), and sign(code) = sign(x) always: a ReLU mask taken from the
// codes is the mask of the fp64 values, bit for bit.
// (The scale is at most kQ8MaxScale, so that 127 steps of it stay finite.)
// Special blocks: all zeros, or a below 1e-300 (127 / a would overflow): scale 0.  A
// block that holds an infinity or a NaN: scale NaN, so every value reads back as NaN
// instead of as a plausible number; codes are the signs, 0 for a NaN.
#include "common.cuh"
#include "gemm.cuh"

namespace mg {

constexpr int kQ8Threads = 256;
constexpr int kQ8Block = MG_Q8_BLOCK;
constexpr double kQ8MaxScale = 0x1.0204081020407p+1017;  // largest s with 127 s finite
static_assert(kQ8Block == 64, "the kernels deal a block to the lanes of a warp two columns each");

__device__ __forceinline__ double q8_inverse(double top) { return top >= 1e-300 ? 127.0 / top : 0.0; }

__device__ __forceinline__ int q8_code(double x, double inverse) {
  const int q = (int)rint(x * inverse);
  return q != 0 ? q : (x > 0 ? 1 : (x < 0 ? -1 : 0));
}

// A warp per block, lane l the columns l and l + 32.
__global__ void __launch_bounds__(kQ8Threads)
q8_pack_kernel(const double *__restrict__ x, signed char *__restrict__ codes, double *__restrict__ scales,
               size_t M, size_t N, size_t nb) {
  const int lane = threadIdx.x & 31;
  const size_t warps = (size_t)gridDim.x * (kQ8Threads / 32), blocks = M * nb;
  for (size_t b = (size_t)blockIdx.x * (kQ8Threads / 32) + (threadIdx.x >> 5); b < blocks; b += warps) {
    const size_t row = b / nb, c0 = (b - row * nb) * kQ8Block, at = row * N + c0;
    const bool in0 = c0 + lane < N, in1 = c0 + lane + 32 < N;
    const double v0 = in0 ? x[at + lane] : 0.0, v1 = in1 ? x[at + lane + 32] : 0.0;
    // NaN > infinity > every finite number in the order of the bit patterns of |x|.
    unsigned long long m0 = __double_as_longlong(fabs(v0)), m1 = __double_as_longlong(fabs(v1));
    unsigned long long m = m0 > m1 ? m0 : m1;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const unsigned long long o = __shfl_xor_sync(0xffffffffu, m, off);
      m = o > m ? o : m;
    }
    const double top = __longlong_as_double((long long)m);
    const bool finite = m < 0x7ff0000000000000ull;
    const double inverse = finite ? q8_inverse(top) : 0.0;
    if (in0) codes[at + lane] = (signed char)q8_code(finite ? v0 : copysign(v0 == v0 ? 1.0 : 0.0, v0), inverse);
    if (in1) codes[at + lane + 32] = (signed char)q8_code(finite ? v1 : copysign(v1 == v1 ? 1.0 : 0.0, v1), inverse);
    if (lane == 0)
      scales[b] = !finite ? __longlong_as_double(0x7ff8000000000000ll) : inverse > 0.0 ? fmin(top / 127.0, kQ8MaxScale) : 0.0;
  }
}

__global__ void __launch_bounds__(kQ8Threads)
q8_unpack_kernel(const signed char *__restrict__ codes, const double *__restrict__ scales,
                 double *__restrict__ x, size_t M, size_t N, size_t nb) {
  const int lane = threadIdx.x & 31;
  const size_t warps = (size_t)gridDim.x * (kQ8Threads / 32), blocks = M * nb;
  for (size_t b = (size_t)blockIdx.x * (kQ8Threads / 32) + (threadIdx.x >> 5); b < blocks; b += warps) {
    const size_t row = b / nb, c0 = (b - row * nb) * kQ8Block, at = row * N + c0;
    const double scale = scales[b];
    if (c0 + lane < N) x[at + lane] = (double)codes[at + lane] * scale;
    if (c0 + lane + 32 < N) x[at + lane + 32] = (double)codes[at + lane + 32] * scale;
  }
}

// gx (+)= g where the code is positive: the gradient of a ReLU whose input or output
// is kept in 8 bits.
__global__ void __launch_bounds__(kQ8Threads)
q8_relu_bwd_kernel(const signed char *__restrict__ codes, const double *g, double *gx, size_t n,
                   bool accumulate) {
  const size_t stride = (size_t)gridDim.x * kQ8Threads;
  for (size_t i = (size_t)blockIdx.x * kQ8Threads + threadIdx.x; i < n; i += stride) {
    const double v = g[i] * (codes[i] > 0 ? 1.0 : 0.0);
    gx[i] = accumulate ? gx[i] + v : v;
  }
}

static size_t q8_blocks(size_t N) { return (N + kQ8Block - 1) / kQ8Block; }

static int check_q8(const char *name, size_t M, size_t N) {
  if (M >= ((size_t)1 << 40) || N >= ((size_t)1 << 40) || (M && N > ((size_t)1 << 60) / M))
    return fail(MG_ERR_INVALID, "%s: dimension too large", name);
  return MG_OK;
}

}  // namespace mg

using namespace mg;

extern "C" {

int mg_q8_pack(const double *x, signed char *codes, double *scales, size_t M, size_t N) {
  int rc = check_q8("mg_q8_pack", M, N);
  if (rc != MG_OK) return rc;
  if (M && N && (!x || !codes || !scales)) return fail(MG_ERR_INVALID, "mg_q8_pack: null pointer");
  MG_ENSURE_INIT();
  if (M == 0 || N == 0) return MG_OK;
  const size_t nb = q8_blocks(N);
  q8_pack_kernel<<<grid_for(M * nb * 32, kQ8Threads, 64), kQ8Threads, 0, ctx().stream>>>(x, codes, scales, M, N, nb);
  MG_LAUNCH_CHECK("q8_pack");
  return MG_OK;
}

int mg_q8_unpack(const signed char *codes, const double *scales, double *x, size_t M, size_t N) {
  int rc = check_q8("mg_q8_unpack", M, N);
  if (rc != MG_OK) return rc;
  if (M && N && (!x || !codes || !scales)) return fail(MG_ERR_INVALID, "mg_q8_unpack: null pointer");
  MG_ENSURE_INIT();
  if (M == 0 || N == 0) return MG_OK;
  const size_t nb = q8_blocks(N);
  q8_unpack_kernel<<<grid_for(M * nb * 32, kQ8Threads, 64), kQ8Threads, 0, ctx().stream>>>(codes, scales, x, M, N, nb);
  MG_LAUNCH_CHECK("q8_unpack");
  return MG_OK;
}

int mg_relu_bwd_q8(const signed char *codes, const double *g, double *gx, size_t n, int flags) {
  if (n && (!codes || !g || !gx)) return fail(MG_ERR_INVALID, "mg_relu_bwd_q8: null pointer");
  MG_ENSURE_INIT();
  if (n == 0) return MG_OK;
  q8_relu_bwd_kernel<<<grid_for(n, kQ8Threads, 64), kQ8Threads, 0, ctx().stream>>>(codes, g, gx, n,
                                                                                !(flags & MG_ACC_STORE_A));
  MG_LAUNCH_CHECK("relu_bwd_q8");
  return MG_OK;
}

int mg_gemm_tn_q8(const signed char *codes, const double *scales, const double *G, double *dB, size_t M,
                  size_t N, size_t K, int accumulate) {
  int rc = check_q8("mg_gemm_tn_q8", M, K);
  if (rc != MG_OK) return rc;
  if (K && N && (!dB || (M && (!codes || !scales || !G))))
    return fail(MG_ERR_INVALID, "mg_gemm_tn_q8: null pointer");
  MG_ENSURE_INIT();
  if (K == 0 || N == 0) return MG_OK;
  // Output [K][N], contraction over the M rows; the codes are widened inside the kernel.
  GemmExt e{{nullptr, G, dB, K, N, M, false, false, accumulate, MG_EPI_NONE, nullptr}};
  e.codes = codes;
  e.scales = scales;
  if (N % 2 == 0 && !off_16_bytes(G)) return run_gemm_ext(e);
  // Rows of G that the tensor kernel cannot take are copied into rows it can.
  double *g = nullptr;
  e.ldb = pitch16(N);
  rc = mg_alloc(M * e.ldb, &g);
  if (rc != MG_OK) return rc;
  rc = copy_rows(G, M, N, N, g, e.ldb);
  e.d.B = g;
  if (rc == MG_OK) rc = run_gemm_ext(e);
  const int freed = mg_free(g);
  return rc != MG_OK ? rc : freed;
}

int mg_gemm_nt_q8(const double *G, const double *B, double *dA, size_t M, size_t N, size_t K, int accumulate,
                  const signed char *mask_codes) {
  if (M && K && (!dA || !mask_codes || (N && (!G || !B))))
    return fail(MG_ERR_INVALID, "mg_gemm_nt_q8: null pointer");
  MG_ENSURE_INIT();
  if (M == 0 || K == 0) return MG_OK;
  // Output [M][K], contraction over N.
  GemmExt e{{G, B, dA, M, K, N, true, true, accumulate, MG_EPI_NONE, nullptr}};
  e.mask8 = mask_codes;
  if (N % 2 == 0 && !off_16_bytes(G) && !off_16_bytes(B)) return run_gemm_ext(e);
  const size_t pitch = pitch16(N);
  double *room = nullptr;
  int rc = mg_alloc((M + K) * pitch, &room);
  if (rc != MG_OK) return rc;
  rc = copy_rows(G, M, N, N, room, pitch);
  if (rc == MG_OK) rc = copy_rows(B, K, N, N, room + M * pitch, pitch);
  e.d.A = room;
  e.d.B = room + M * pitch;
  e.lda = e.ldb = pitch;
  if (rc == MG_OK) rc = run_gemm_ext(e);
  const int freed = mg_free(room);
  return rc != MG_OK ? rc : freed;
}

}  // extern "C"
