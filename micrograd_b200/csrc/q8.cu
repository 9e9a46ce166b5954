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
static_assert(kQ8Block == 64, "the kernels deal a block to 16 or 32 lanes");

__device__ __forceinline__ double q8_inverse(double top) { return top >= 1e-300 ? 127.0 / top : 0.0; }

// rint(x * inverse), |x * inverse| < 128, as the low word of the sum with 1.5 * 2^52
// (ties to even, like rint); the sign of x where that is 0 and x is not.
__device__ __forceinline__ int q8_code(double x, double inverse) {
  const int q = __double2loint(x * inverse + 6755399441055744.0);
  const int hi = __double2hiint(x), some = (hi << 1) | __double2loint(x);
  return q != 0 || some == 0 ? q : (hi < 0 ? -1 : 1);
}

// Reads and writes of VEC neighbouring values and codes.
template <int VEC> __device__ __forceinline__ void load_values(const double *p, double (&v)[VEC]) {
  if constexpr (VEC == 4) {
    const double4v t = ld_stream_v4(reinterpret_cast<const double4v *>(p));
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
  } else if constexpr (VEC == 2) {
    const double2 t = __ldcs(reinterpret_cast<const double2 *>(p));
    v[0] = t.x; v[1] = t.y;
  } else {
    v[0] = __ldcs(p);
  }
}

// LANES lanes take a block, VEC neighbouring columns each, UN blocks at a time so that
// 64 to 128 bytes per lane are on their way.  A lane of a block's ragged end has no
// column; LANES x VEC = 64.
template <int VEC, int UN, bool FLAT>
__global__ void __launch_bounds__(kQ8Threads)
q8_pack_kernel(const double *__restrict__ x, signed char *__restrict__ codes, double *__restrict__ scales,
               size_t blocks, size_t N, unsigned nb) {
  constexpr int LANES = VEC == 4 ? 16 : 32, PER = 64 / LANES;  // columns per lane
  const int lane = threadIdx.x % LANES;
  const size_t teams = (size_t)gridDim.x * (kQ8Threads / LANES);
  // (all lanes of a warp make the same number of rounds: they shuffle together)
  const size_t first = ((size_t)blockIdx.x * kQ8Threads + threadIdx.x) / LANES, rounds = (blocks + teams * UN - 1) / (teams * UN);
  for (size_t round = 0; round < rounds; round++) {
    double v[UN][PER];
    size_t at[UN];
    int cols[UN];  // columns of this lane
#pragma unroll
    for (int u = 0; u < UN; u++) {
      const size_t b = first + (round * UN + u) * teams;
      cols[u] = 0;
      if (b < blocks) {
        if (FLAT) {
          at[u] = b * 64 + lane * PER;
          cols[u] = PER;
        } else {
          const size_t row = blocks >> 32 ? b / nb : (size_t)((unsigned)b / nb);
          const size_t c = (b - row * nb) * 64 + lane * PER;
          at[u] = row * N + c;
          cols[u] = c < N ? (N - c < PER ? (int)(N - c) : PER) : 0;
        }
      }
#pragma unroll
      for (int k = 0; k < PER; k++) v[u][k] = 0.0;
      if constexpr (VEC == PER) {
        if (cols[u] > 0) load_values<VEC>(x + at[u], v[u]);  // (N is a multiple of VEC)
      } else {
#pragma unroll
        for (int k = 0; k < PER; k++)
          if (k < cols[u]) v[u][k] = __ldcs(x + at[u] + k);
      }
    }
#pragma unroll
    for (int u = 0; u < UN; u++) {
      // NaN > infinity > every finite number in the order of the bit patterns of |x|.
      unsigned long long m = 0;
#pragma unroll
      for (int k = 0; k < PER; k++) {
        const unsigned long long o = (unsigned long long)__double_as_longlong(fabs(v[u][k]));
        m = o > m ? o : m;
      }
#pragma unroll
      for (int off = LANES / 2; off > 0; off >>= 1) {
        const unsigned long long o = __shfl_xor_sync(0xffffffffu, m, off);
        m = o > m ? o : m;
      }
      const double top = __longlong_as_double((long long)m);
      const bool finite = m < 0x7ff0000000000000ull;
      const double inverse = finite ? q8_inverse(top) : 0.0;
      unsigned word = 0;
#pragma unroll
      for (int k = 0; k < PER; k++) {
        double y = v[u][k];
        if (!finite) y = y > 0 ? 1.0 : (y < 0 ? -1.0 : 0.0);
        word |= (unsigned)(q8_code(y, inverse) & 255) << (8 * k);
      }
      if (VEC == PER && cols[u] > 0) {
        if (PER == 4) *reinterpret_cast<unsigned *>(codes + at[u]) = word;
        else *reinterpret_cast<unsigned short *>(codes + at[u]) = (unsigned short)word;
      } else {
#pragma unroll
        for (int k = 0; k < PER; k++)
          if (k < cols[u]) codes[at[u] + k] = (signed char)(word >> (8 * k));
      }
      const size_t b = first + (round * UN + u) * teams;
      if (lane == 0 && b < blocks)
        scales[b] = !finite ? __longlong_as_double(0x7ff8000000000000ll)
                            : inverse > 0.0 ? fmin(top / 127.0, kQ8MaxScale) : 0.0;
    }
  }
}

template <int VEC, int UN, bool FLAT>
__global__ void __launch_bounds__(kQ8Threads)
q8_unpack_kernel(const signed char *__restrict__ codes, const double *__restrict__ scales,
                 double *__restrict__ x, size_t blocks, size_t N, unsigned nb) {
  constexpr int LANES = VEC == 4 ? 16 : 32, PER = 64 / LANES;
  const int lane = threadIdx.x % LANES;
  const size_t teams = (size_t)gridDim.x * (kQ8Threads / LANES);
  for (size_t b0 = ((size_t)blockIdx.x * kQ8Threads + threadIdx.x) / LANES; b0 < blocks; b0 += teams * UN) {
    unsigned word[UN];
    double scale[UN];
    size_t at[UN];
    int cols[UN];
#pragma unroll
    for (int u = 0; u < UN; u++) {
      const size_t b = b0 + u * teams;
      cols[u] = 0;
      word[u] = 0;
      if (b < blocks) {
        if (FLAT) {
          at[u] = b * 64 + lane * PER;
          cols[u] = PER;
        } else {
          const size_t row = blocks >> 32 ? b / nb : (size_t)((unsigned)b / nb);
          const size_t c = (b - row * nb) * 64 + lane * PER;
          at[u] = row * N + c;
          cols[u] = c < N ? (N - c < PER ? (int)(N - c) : PER) : 0;
        }
      }
      if (cols[u] > 0) {
        scale[u] = __ldg(scales + b);
        if constexpr (VEC == PER) {
          if (PER == 4) word[u] = __ldcs(reinterpret_cast<const unsigned *>(codes + at[u]));
          else word[u] = __ldcs(reinterpret_cast<const unsigned short *>(codes + at[u]));
        } else {
#pragma unroll
          for (int k = 0; k < PER; k++)
            if (k < cols[u]) word[u] |= (unsigned)(unsigned char)codes[at[u] + k] << (8 * k);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < UN; u++) {
      if (cols[u] <= 0) continue;
      double v[PER];
#pragma unroll
      for (int k = 0; k < PER; k++) v[k] = (double)(signed char)(word[u] >> (8 * k)) * scale[u];
      if constexpr (VEC == PER && PER == 4) {
        st_stream_v4(reinterpret_cast<double4v *>(x + at[u]), double4v{v[0], v[1], v[2], v[3]});
      } else if constexpr (VEC == PER) {
        __stcs(reinterpret_cast<double2 *>(x + at[u]), make_double2(v[0], v[1]));
      } else {
#pragma unroll
        for (int k = 0; k < PER; k++)
          if (k < cols[u]) x[at[u] + k] = v[k];
      }
    }
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

// Widest access that the row length and both addresses allow.
static int q8_vec(const double *x, const signed char *codes, size_t N) {
  const uintptr_t px = reinterpret_cast<uintptr_t>(x), pc = reinterpret_cast<uintptr_t>(codes);
  if (N % 4 == 0 && px % 32 == 0 && pc % 4 == 0) return 4;
  if (N % 2 == 0 && px % 16 == 0 && pc % 2 == 0) return 2;
  return 1;
}

static size_t q8_blocks(size_t N) { return (N + kQ8Block - 1) / kQ8Block; }

// dst[rows][pitch] = src[rows][cols], zeros behind them (pitch a multiple of 16).
__global__ void __launch_bounds__(256)
q8_copy_rows_kernel(const signed char *__restrict__ src, size_t rows, size_t cols, signed char *__restrict__ dst,
                    size_t pitch) {
  const size_t words = pitch / 4, all = rows * words;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (size_t)gridDim.x * 256) {
    const size_t r = all >> 32 ? i / words : (size_t)((unsigned)i / (unsigned)words), c = (i - r * words) * 4;
    const signed char *p = src + r * cols + c;
    unsigned w = 0;
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (c + k < cols) w |= (unsigned)(unsigned char)p[k] << (8 * k);
    reinterpret_cast<unsigned *>(dst)[i] = w;
  }
}

static int copy_codes_rows(const signed char *src, size_t rows, size_t cols, signed char *dst, size_t pitch) {
  q8_copy_rows_kernel<<<grid_for(rows * pitch / 4, 256, 32), 256, 0, ctx().stream>>>(src, rows, cols, dst, pitch);
  MG_LAUNCH_CHECK("copy of codes");
  return MG_OK;
}

// dA[M][K] (+)= (G[M][N] . B[K][N]^T) * (mask > 0) for N <= 16: nothing but streaming
// the output, 9 bytes per element (17 when accumulating) against 2 N flop.  A thread
// keeps two columns' rows of B in registers and walks down the rows; the rows of G pass
// through shared memory, where a warp reads each value once for its 64 outputs.
// PAIR: the two columns are neighbours (K even, aligned), else TX apart.  The next
// rows of G and of the mask are on their way while a block of rows is computed.
constexpr int kOuterRows = 8;  // rows per thread and block

template <int NN, bool PAIR>
__global__ void __launch_bounds__(256, 2)
q8_outer_kernel(const double *__restrict__ G, const double *__restrict__ B, double *dA,
                const signed char *__restrict__ mask, size_t M, int N, size_t K, bool accumulate) {
  constexpr int kMostTY = 8, kPer = (kOuterRows * kMostTY * NN + 255) / 256;
  __shared__ __align__(16) double gs[2][kOuterRows * kMostTY * NN];
  const int TX = blockDim.x, TY = blockDim.y, tid = threadIdx.y * TX + threadIdx.x;
  const size_t c0 = (size_t)blockIdx.x * 2 * TX + (PAIR ? 2 * threadIdx.x : threadIdx.x), c1 = PAIR ? c0 + 1 : c0 + TX;
  const bool in0 = c0 < K, in1 = c1 < K;
  double b0[NN], b1[NN];
#pragma unroll
  for (int n = 0; n < NN; n++) {
    b0[n] = in0 && n < N ? B[c0 * N + n] : 0.0;
    b1[n] = in1 && n < N ? B[c1 * N + n] : 0.0;
  }
  const int rows = kOuterRows * TY, values = rows * NN;
  const size_t blocks = (M + rows - 1) / rows;
  unsigned short next[kOuterRows];  // a row's two codes
  double g_next[kPer];
  auto read = [&](size_t blk) {
    const size_t m0 = blk * rows;
#pragma unroll
    for (int u = 0; u < kOuterRows; u++) {
      const size_t m = m0 + u * TY + threadIdx.y, at = m * K;
      next[u] = 0;
      if (m < M) {
        if (PAIR) {
          if (in0) next[u] = __ldcs(reinterpret_cast<const unsigned short *>(mask + at + c0));
        } else {
          if (in0) next[u] = (unsigned char)mask[at + c0];
          if (in1) next[u] |= (unsigned short)((unsigned char)mask[at + c1] << 8);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kPer; k++) {
      const int i = tid + 256 * k, r = i / NN, n = i % NN;
      g_next[k] = i < values && m0 + r < M && n < N ? __ldg(G + (m0 + r) * N + n) : 0.0;
    }
  };
  auto hand_over = [&](int buf) {
#pragma unroll
    for (int k = 0; k < kPer; k++)
      if (tid + 256 * k < values) gs[buf][tid + 256 * k] = g_next[k];
  };
  size_t blk = blockIdx.y;
  if (blk < blocks) read(blk);
  hand_over(0);
  int buf = 0;
  for (; blk < blocks; blk += gridDim.y, buf ^= 1) {
    __syncthreads();  // gs[buf] is complete, and nobody reads the other one any more
    unsigned short codes[kOuterRows];
#pragma unroll
    for (int u = 0; u < kOuterRows; u++) codes[u] = next[u];
    if (blk + gridDim.y < blocks) read(blk + gridDim.y);
#pragma unroll
    for (int u = 0; u < kOuterRows; u++) {
      const int r = u * TY + threadIdx.y;
      const size_t m = blk * rows + r;
      if (m >= M) continue;
      const double *g = &gs[buf][r * NN];
      double s0 = 0.0, s1 = 0.0;
#pragma unroll
      for (int n = 0; n < NN; n += 2) {
        const double2 v = *reinterpret_cast<const double2 *>(g + n);
        s0 = fma(v.x, b0[n], s0);
        s1 = fma(v.x, b1[n], s1);
        s0 = fma(v.y, b0[n + 1], s0);
        s1 = fma(v.y, b1[n + 1], s1);
      }
      s0 = s0 * ((signed char)codes[u] > 0 ? 1.0 : 0.0);
      s1 = s1 * ((short)codes[u] >= 256 ? 1.0 : 0.0);  // (its high byte > 0)
      double *dst = dA + m * K;
      if (PAIR) {
        if (!in0) continue;
        if (accumulate) {
          const double2 o = *reinterpret_cast<const double2 *>(dst + c0);
          s0 = o.x + s0;
          s1 = o.y + s1;
        }
        __stcs(reinterpret_cast<double2 *>(dst + c0), make_double2(s0, s1));
      } else {
        if (in0) dst[c0] = accumulate ? dst[c0] + s0 : s0;
        if (in1) dst[c1] = accumulate ? dst[c1] + s1 : s1;
      }
    }
    hand_over(buf ^ 1);
  }
}

static int outer_q8(const double *G, const double *B, double *dA, size_t M, size_t N, size_t K, int accumulate,
                    const signed char *mask) {
  unsigned tx = 32;
  while (tx < 256 && 2 * (size_t)tx < K) tx *= 2;
  const bool pair = K % 2 == 0 && !off_16_bytes(dA) && !(reinterpret_cast<uintptr_t>(mask) & 1);
  const size_t rows = (size_t)kOuterRows * (256 / tx), gx = (K + 2 * tx - 1) / (2 * tx), blocks = (M + rows - 1) / rows;
  size_t gy = (size_t)ctx().sm_count * 16 / gx + 1;
  if (gy > blocks) gy = blocks;
  if (gy > 65535) gy = 65535;
  const dim3 grid((unsigned)gx, (unsigned)gy), block(tx, 256 / tx);
  cudaStream_t stream = ctx().stream;
#define MG_OUTER(NN)                                                                                        \
  (pair ? q8_outer_kernel<NN, true><<<grid, block, 0, stream>>>(G, B, dA, mask, M, (int)N, K, accumulate != 0) \
        : q8_outer_kernel<NN, false><<<grid, block, 0, stream>>>(G, B, dA, mask, M, (int)N, K, accumulate != 0))
  if (N <= 4) MG_OUTER(4);
  else if (N <= 8) MG_OUTER(8);
  else if (N <= 12) MG_OUTER(12);
  else MG_OUTER(16);
#undef MG_OUTER
  MG_LAUNCH_CHECK("gemm_nt_q8 (few columns)");
  return MG_OK;
}

static int check_q8(const char *name, size_t M, size_t N) {
  if (M >= ((size_t)1 << 40) || N >= ((size_t)1 << 36) || (M && N > ((size_t)1 << 60) / M))
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
  const size_t nb = q8_blocks(N), blocks = M * nb;
  cudaStream_t stream = ctx().stream;
  const int vec = q8_vec(x, codes, N);
  const unsigned grid = grid_for(blocks * (vec == 4 ? 16 : 32), kQ8Threads, 64);
  if (vec == 4 && N % 64 == 0)
    q8_pack_kernel<4, 4, true><<<grid, kQ8Threads, 0, stream>>>(x, codes, scales, blocks, N, (unsigned)nb);
  else if (vec == 4)
    q8_pack_kernel<4, 2, false><<<grid, kQ8Threads, 0, stream>>>(x, codes, scales, blocks, N, (unsigned)nb);
  else if (vec == 2)
    q8_pack_kernel<2, 4, false><<<grid, kQ8Threads, 0, stream>>>(x, codes, scales, blocks, N, (unsigned)nb);
  else
    q8_pack_kernel<1, 4, false><<<grid, kQ8Threads, 0, stream>>>(x, codes, scales, blocks, N, (unsigned)nb);
  MG_LAUNCH_CHECK("q8_pack");
  return MG_OK;
}

int mg_q8_unpack(const signed char *codes, const double *scales, double *x, size_t M, size_t N) {
  int rc = check_q8("mg_q8_unpack", M, N);
  if (rc != MG_OK) return rc;
  if (M && N && (!x || !codes || !scales)) return fail(MG_ERR_INVALID, "mg_q8_unpack: null pointer");
  MG_ENSURE_INIT();
  if (M == 0 || N == 0) return MG_OK;
  const size_t nb = q8_blocks(N), blocks = M * nb;
  cudaStream_t stream = ctx().stream;
  const int vec = q8_vec(x, codes, N);
  const unsigned grid = grid_for(blocks * (vec == 4 ? 16 : 32), kQ8Threads, 64);
  if (vec == 4 && N % 64 == 0)
    q8_unpack_kernel<4, 4, true><<<grid, kQ8Threads, 0, stream>>>(codes, scales, x, blocks, N, (unsigned)nb);
  else if (vec == 4)
    q8_unpack_kernel<4, 2, false><<<grid, kQ8Threads, 0, stream>>>(codes, scales, x, blocks, N, (unsigned)nb);
  else if (vec == 2)
    q8_unpack_kernel<2, 4, false><<<grid, kQ8Threads, 0, stream>>>(codes, scales, x, blocks, N, (unsigned)nb);
  else
    q8_unpack_kernel<1, 4, false><<<grid, kQ8Threads, 0, stream>>>(codes, scales, x, blocks, N, (unsigned)nb);
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
  // Rows of codes or of G that it cannot take are copied into rows that it can.
  GemmExt e{{nullptr, G, dB, K, N, M, false, false, accumulate, MG_EPI_NONE, nullptr}};
  e.codes = codes;
  e.scales = scales;
  e.lda = K;
  const bool copy_codes = K % 16 != 0 || off_16_bytes(codes), copy_g = N % 2 != 0 || off_16_bytes(G);
  if (!copy_codes && !copy_g) return run_gemm_ext(e);
  const size_t pitch_c = pitch16(K), pitch_g = pitch16(N);
  const size_t code_room = copy_codes ? (M * pitch_c + 255) / 256 * 32 : 0;  // in doubles
  double *room = nullptr;
  rc = mg_alloc(code_room + (copy_g ? M * pitch_g : 0), &room);
  if (rc != MG_OK) return rc;
  if (copy_codes) {
    signed char *dst = reinterpret_cast<signed char *>(room);
    rc = copy_codes_rows(codes, M, K, dst, pitch_c);
    e.codes = dst;
    e.lda = pitch_c;
  }
  if (rc == MG_OK && copy_g) {
    rc = copy_rows(G, M, N, N, room + code_room, pitch_g);
    e.d.B = room + code_room;
    e.ldb = pitch_g;
  }
  if (rc == MG_OK) rc = run_gemm_ext(e);
  const int freed = mg_free(room);
  return rc != MG_OK ? rc : freed;
}

int mg_gemm_nt_q8(const double *G, const double *B, double *dA, size_t M, size_t N, size_t K, int accumulate,
                  const signed char *mask_codes) {
  if (M && K && (!dA || !mask_codes || (N && (!G || !B))))
    return fail(MG_ERR_INVALID, "mg_gemm_nt_q8: null pointer");
  MG_ENSURE_INIT();
  if (M == 0 || K == 0) return MG_OK;
  if (N > 0 && N <= 16) return outer_q8(G, B, dA, M, N, K, accumulate, mask_codes);
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
