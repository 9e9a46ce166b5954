// Activations kept in 8 bits between the forward and the backward pass.
//
// The columns of a row x[M][N] are cut into blocks of MG_Q8_BLOCK = 64 (the last one
// may be shorter).  With a = max |x| over a block:
//
//   scale = a / 127,  code = rint(x (127 / a)),  and code = sign(x) where that
//   rounds to 0 and x is not 0;  the value kept is code * scale
//
// with each quotient and product rounded to fp64 before it is used.
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
// (ties to even, like rint); the sign of x where that is 0 and x is not.  The product is
// rounded before the sum: one fma would give 63 for 2.5 under a maximum of 5, where
// 2.5 (127 / 5) rounds to 63.5 and so to 64.
__device__ __forceinline__ int q8_code(double x, double inverse) {
  const int q = __double2loint(__dadd_rn(__dmul_rn(x, inverse), 6755399441055744.0));
  const int hi = __double2hiint(x), some = (hi << 1) | __double2loint(x);
  return q != 0 || some == 0 ? q : (hi >> 31) | 1;
}

// Row and block in it of the blocks b, b + step, ... without a division for each.
struct BlockWalk {
  size_t row, row_step;
  unsigned block, block_step, nb;
  __device__ __forceinline__ BlockWalk(size_t b, size_t step, unsigned per_row, bool flat) : nb(per_row) {
    row = flat ? 0 : b / nb;
    block = flat ? 0 : (unsigned)(b - row * nb);
    row_step = flat ? 0 : step / nb;
    block_step = flat ? 0 : (unsigned)(step - row_step * nb);
  }
  __device__ __forceinline__ void next() {
    row += row_step;
    block += block_step;
    if (block >= nb) {
      block -= nb;
      row++;
    }
  }
};

// A warp per block, two columns per lane, UN blocks at a time so that 32 to 64 bytes per
// lane are on their way.  The integer units bound this kernel before HBM does (70 and
// 49 % of their rates at 65 536 x 1024, the fp64 units 19 %), so the
// block's maximum is taken by two warp-wide integer reductions: of the high words of
// |x|, then of the low words under the largest high word (their bit patterns are in the
// order of the values, infinity and NaN above all numbers); and its two quotients are
// taken by one lane, for all UN blocks at once.
// PAIR: the columns are neighbours (even rows, aligned), else 32 apart.  FLAT: rows are
// whole blocks.
// 65 536 x 1024: 134 us with two blocks at a time and six CTAs per SM, 151 with four and
// four, 170 with the maximum by shuffles.
template <bool PAIR, int UN, bool FLAT>
__global__ void __launch_bounds__(kQ8Threads, UN == 2 ? 6 : 4)
q8_pack_kernel(const double *__restrict__ x, signed char *__restrict__ codes, double *__restrict__ scales,
               size_t blocks, size_t N, unsigned nb) {
  cudaGridDependencySynchronize();
  const int lane = threadIdx.x & 31;
  const size_t warps = (size_t)gridDim.x * (kQ8Threads / 32);
  size_t b0 = ((size_t)blockIdx.x * kQ8Threads + threadIdx.x) >> 5;
  BlockWalk walk(b0, warps, nb, FLAT);
  for (; b0 < blocks; b0 += warps * UN) {
    double v0[UN], v1[UN];
    size_t at[UN];
    int cols[UN];  // columns of the block (0: there is no such block)
    // Loads are never conditional (a value merged with a default is waited for at the
    // merge, one after the other): a column that does not exist reads the block's first
    // value, or the array's, and is dropped below.
#pragma unroll
    for (int u = 0; u < UN; u++) {
      const size_t b = b0 + u * warps;
      cols[u] = 0;
      at[u] = 0;
      if (b < blocks) {
        if (FLAT) {
          at[u] = b * 64;
          cols[u] = 64;
        } else {
          const size_t c = (size_t)walk.block * 64;
          at[u] = walk.row * N + c;
          cols[u] = N - c < 64 ? (int)(N - c) : 64;
        }
      }
      if (!FLAT) walk.next();
      if (PAIR) {
        const double2 t = __ldcs(reinterpret_cast<const double2 *>(x + at[u] + (2 * lane < cols[u] ? 2 * lane : 0)));
        v0[u] = t.x;
        v1[u] = t.y;
      } else {
        v0[u] = __ldcs(x + at[u] + (lane < cols[u] ? lane : 0));
        v1[u] = __ldcs(x + at[u] + (lane + 32 < cols[u] ? lane + 32 : 0));
      }
    }
    unsigned top_hi[UN], top_lo[UN];
#pragma unroll
    for (int u = 0; u < UN; u++) {
      // (a dropped column holds a value of the block, so it does not change the maximum)
      const unsigned h0 = __double2hiint(v0[u]) & 0x7fffffff, h1 = __double2hiint(v1[u]) & 0x7fffffff;
      top_hi[u] = __reduce_max_sync(0xffffffffu, h0 > h1 ? h0 : h1);
      const unsigned l0 = h0 == top_hi[u] ? (unsigned)__double2loint(v0[u]) : 0u;
      const unsigned l1 = h1 == top_hi[u] ? (unsigned)__double2loint(v1[u]) : 0u;
      top_lo[u] = __reduce_max_sync(0xffffffffu, l0 > l1 ? l0 : l1);
    }
    unsigned my_hi = top_hi[0], my_lo = top_lo[0];
#pragma unroll
    for (int u = 1; u < UN; u++) {
      my_hi = (lane & (UN - 1)) == u ? top_hi[u] : my_hi;
      my_lo = (lane & (UN - 1)) == u ? top_lo[u] : my_lo;
    }
    const double top = __hiloint2double((int)my_hi, (int)my_lo);
    const double my_inverse = my_hi < 0x7ff00000u ? q8_inverse(top) : 0.0;
    if (lane < UN && b0 + lane * warps < blocks)
      scales[b0 + lane * warps] = my_hi >= 0x7ff00000u ? __longlong_as_double(0x7ff8000000000000ll)
                                  : my_inverse > 0.0   ? fmin(top / 127.0, kQ8MaxScale)
                                                       : 0.0;
#pragma unroll
    for (int u = 0; u < UN; u++) {
      const double inverse = __shfl_sync(0xffffffffu, my_inverse, u);
      double y0 = v0[u], y1 = v1[u];
      if (top_hi[u] >= 0x7ff00000u) {  // (the same in the whole warp) an infinity or a NaN: signs
        y0 = y0 > 0 ? 1.0 : (y0 < 0 ? -1.0 : 0.0);
        y1 = y1 > 0 ? 1.0 : (y1 < 0 ? -1.0 : 0.0);
      }
      const int q0 = q8_code(y0, inverse), q1 = q8_code(y1, inverse);
      signed char *dst = codes + at[u];
      if (PAIR) {
        if (2 * lane < cols[u])
          *reinterpret_cast<unsigned short *>(dst + 2 * lane) = (unsigned short)__byte_perm(q0, q1, 0x0040);
      } else {
        if (lane < cols[u]) dst[lane] = (signed char)q0;
        if (lane + 32 < cols[u]) dst[lane + 32] = (signed char)q1;
      }
    }
  }
}

template <int VEC, int UN, bool FLAT>
__global__ void __launch_bounds__(kQ8Threads)
q8_unpack_kernel(const signed char *__restrict__ codes, const double *__restrict__ scales,
                 double *__restrict__ x, size_t pitch, size_t blocks, size_t N, unsigned nb) {
  cudaGridDependencySynchronize();
  constexpr int LANES = VEC == 4 ? 16 : 32, PER = 64 / LANES;
  const int lane = threadIdx.x % LANES;
  const size_t teams = (size_t)gridDim.x * (kQ8Threads / LANES);
  size_t b0 = ((size_t)blockIdx.x * kQ8Threads + threadIdx.x) / LANES;
  BlockWalk walk(b0, teams, nb, FLAT);
  for (; b0 < blocks; b0 += teams * UN) {
    unsigned word[UN];
    double scale[UN];
    size_t at[UN], to[UN];
    int cols[UN];
#pragma unroll
    for (int u = 0; u < UN; u++) {
      const size_t b = b0 + u * teams;
      cols[u] = 0;
      at[u] = to[u] = 0;
      if (b < blocks) {
        if (FLAT) {
          at[u] = to[u] = b * 64 + lane * PER;
          cols[u] = PER;
        } else {
          const size_t c = (size_t)walk.block * 64 + lane * PER;
          if (c < N) {
            at[u] = walk.row * N + c;
            to[u] = walk.row * pitch + c;
            cols[u] = N - c < PER ? (int)(N - c) : PER;
          }
        }
      }
      if (!FLAT) walk.next();
      scale[u] = __ldg(scales + (b < blocks ? b : 0));
      if constexpr (VEC == PER) {
        if (PER == 4) word[u] = __ldcs(reinterpret_cast<const unsigned *>(codes + at[u]));
        else word[u] = __ldcs(reinterpret_cast<const unsigned short *>(codes + at[u]));
      } else {
        word[u] = 0;
#pragma unroll
        for (int k = 0; k < PER; k++)
          word[u] |= (unsigned)(unsigned char)codes[at[u] + (k < cols[u] ? k : 0)] << (8 * k);
      }
    }
#pragma unroll
    for (int u = 0; u < UN; u++) {
      if (cols[u] <= 0) continue;
      double v[PER];
#pragma unroll
      for (int k = 0; k < PER; k++) v[k] = (double)(signed char)(word[u] >> (8 * k)) * scale[u];
      if constexpr (VEC == PER && PER == 4) {
        st_stream_v4(reinterpret_cast<double4v *>(x + to[u]), double4v{v[0], v[1], v[2], v[3]});
      } else if constexpr (VEC == PER) {
        __stcs(reinterpret_cast<double2 *>(x + to[u]), make_double2(v[0], v[1]));
      } else {
#pragma unroll
        for (int k = 0; k < PER; k++)
          if (k < cols[u]) x[to[u] + k] = v[k];
      }
    }
  }
}

static size_t q8_blocks(size_t N) { return (N + kQ8Block - 1) / kQ8Block; }

// gx (+)= g where the code is positive: the gradient of a ReLU whose input or output
// is kept in 8 bits.  17 bytes per value, 25 when accumulating:
// 65 536 x 1024 in 168 us (6.8 TB/s) and 243 us; one value per thread 208 and 259.
// QUADS: four values per thread, where all three addresses allow it.
template <bool QUADS>
__global__ void __launch_bounds__(kQ8Threads)
q8_relu_bwd_kernel(const signed char *__restrict__ codes, const double *g, double *gx, size_t n,
                   bool accumulate) {
  cudaGridDependencySynchronize();
  const size_t stride = (size_t)gridDim.x * kQ8Threads, first = (size_t)blockIdx.x * kQ8Threads + threadIdx.x;
  const size_t quads = QUADS ? n / 4 : 0;
  for (size_t i = first; i < quads; i += stride) {
    const char4 k = reinterpret_cast<const char4 *>(codes)[i];
    const double4v v = ld_stream_v4(reinterpret_cast<const double4v *>(g) + i);
    double4v *to = reinterpret_cast<double4v *>(gx) + i;
    double4v r = {v.x * (k.x > 0 ? 1.0 : 0.0), v.y * (k.y > 0 ? 1.0 : 0.0), v.z * (k.z > 0 ? 1.0 : 0.0),
                  v.w * (k.w > 0 ? 1.0 : 0.0)};
    if (accumulate) {
      const double4v o = ld_stream_v4(to);
      r = {o.x + r.x, o.y + r.y, o.z + r.z, o.w + r.w};
    }
    st_stream_v4(to, r);
  }
  for (size_t i = 4 * quads + first; i < n; i += stride) {
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


// ---------------------------------------------------------------------------
// Products with few columns (N <= 32): streams of one byte per element for 2 N flop.
// The tensor kernel would need the fp64 form of the codes, 8 bytes each, written and
// read, or spend its tiles on padding.  These keep the narrow operand's values (or the
// sums) of two columns per lane in registers; tiles of codes and the rows of G that go
// with them come through a ring of kRing stages in shared memory by asynchronous copies.
// ---------------------------------------------------------------------------
constexpr int kRing = 3;

__device__ __forceinline__ uint32_t shared_address(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 8 bytes, or zeros.
__device__ __forceinline__ void copy8(void *dst, const void *src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(shared_address(dst)), "l"(src), "r"(in ? 8 : 0)
               : "memory");
}

// Rows m0 .. m0 + rows - 1 of G[M][N] into dst[rows][NN] (its last column is left alone
// where N is odd, rows from M on become zeros), by the CTA's `threads` threads.  Even N
// from a 16-byte boundary: the rows are one run of memory on both sides.
template <int NN>
__device__ __forceinline__ void copy_g(double *dst, const double *__restrict__ G, size_t m0, size_t M, int rows, int N,
                                       int tid, int threads, bool run) {
  const double *src = G + m0 * N;
  if (run) {
    const int in = M > m0 ? (M - m0 < (size_t)rows ? (int)(M - m0) : rows) * N : 0;  // values that exist
    for (int i = 2 * tid; i < rows * NN; i += 2 * threads)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(shared_address(dst + i)),
                   "l"(i < in ? src + i : G), "r"(i < in ? 16 : 0)
                   : "memory");
  } else {
    for (int i = tid; i < rows * N; i += threads) {
      const int r = i / N;
      const bool in = m0 + r < M;
      copy8(dst + r * NN + (i - r * N), in ? src + i : G, in);
    }
  }
}

// How the rows of a matrix of codes can be read: 16 or 4 bytes at a time, or single ones.
enum { kCodes16, kCodes4, kCodes1 };
static int code_access(const signed char *codes, size_t K) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(codes) | K;
  return bits % 16 == 0 ? kCodes16 : (bits % 4 == 0 ? kCodes4 : kCodes1);
}

// The 16 codes from column `col` of row m on into dst (16-byte aligned), zeros outside.
template <int ACCESS>
__device__ __forceinline__ void copy_codes(uint8_t *dst, const signed char *__restrict__ codes, size_t m, size_t M,
                                           size_t col, size_t K) {
  const bool row = m < M;
  const signed char *src = codes + (row ? m * K : 0);
  if (ACCESS == kCodes16) {
    const bool in = row && col < K;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(shared_address(dst)), "l"(in ? src + col : src),
                 "r"(in ? 16 : 0)
                 : "memory");
  } else if (ACCESS == kCodes4) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const bool in = row && col + 4 * k < K;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(shared_address(dst + 4 * k)),
                   "l"(in ? src + col + 4 * k : src), "r"(in ? 4 : 0)
                   : "memory");
    }
  } else {
    unsigned word[4] = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < 16; k++)
      if (row && col + k < K) word[k >> 2] |= (unsigned)(unsigned char)src[col + k] << (8 * (k & 3));
    *reinterpret_cast<uint4 *>(dst) = make_uint4(word[0], word[1], word[2], word[3]);
  }
}

// dA[M][K] (+)= (G[M][N] . B[K][N]^T) * (mask > 0), N <= 16: nothing but streaming the
// output, 9 bytes per element (17 when accumulating).  TX x TY threads take 2 TX columns
// of 8 TY rows at a time.  PAIR: the two columns of a thread are neighbours (K even,
// dA aligned), else TX apart.
// Two CTAs per SM with more than eight columns: 108 us for 65 536 x 1024, ten columns;
// three spill registers, 122 us.
constexpr int outer_ctas(int nn) { return nn <= 8 ? 4 : 2; }
constexpr int kOuterRows = 8;  // rows per thread and tile
constexpr int kOuterCodes = 256 * 2 * kOuterRows;  // codes of a tile

template <int NN, bool PAIR, int ACCESS>
__global__ void __launch_bounds__(256, outer_ctas(NN))
q8_outer_kernel(const double *__restrict__ G, const double *__restrict__ B, double *dA,
                const signed char *__restrict__ mask, size_t M, int N, size_t K, bool accumulate) {
  constexpr int kMostRows = kOuterRows * 8;
  __shared__ __align__(16) double gs[kRing][kMostRows * NN];
  __shared__ __align__(16) uint8_t cs[kRing][kOuterCodes];
  const int TX = blockDim.x, TY = blockDim.y, tid = threadIdx.y * TX + threadIdx.x;
  const int width = 2 * TX, rows = kOuterRows * TY, mine = PAIR ? 2 * threadIdx.x : threadIdx.x, apart = PAIR ? 1 : TX;
  const size_t col0 = (size_t)blockIdx.x * width, c0 = col0 + mine;
  const bool in0 = c0 < K, in1 = c0 + apart < K;
  const size_t tiles = (M + rows - 1) / rows;
  const int chunks = width / 16, my_row = tid / chunks, my_col = (tid - my_row * chunks) * 16;
  if (N < NN)  // (an odd N: the last value of a staged row stays 0)
    for (int i = tid; i < kRing * rows; i += 256) gs[i / rows][(i % rows) * NN + N] = 0.0;
  const bool run = N == NN && (reinterpret_cast<uintptr_t>(G) & 15) == 0;
  auto fetch = [&](size_t tile, int stage) {
    if (tile < tiles) {
      const size_t m0 = tile * rows;
      copy_codes<ACCESS>(&cs[stage][my_row * width + my_col], mask, m0 + my_row, M, col0 + my_col, K);
      copy_g<NN>(gs[stage], G, m0, M, rows, N, tid, 256, run);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  double b0[NN], b1[NN];
#pragma unroll
  for (int n = 0; n < NN; n++) {
    b0[n] = in0 && n < N ? B[c0 * N + n] : 0.0;
    b1[n] = in1 && n < N ? B[(c0 + apart) * N + n] : 0.0;
  }
  size_t tile = blockIdx.y;
#pragma unroll
  for (int s = 0; s < kRing - 1; s++) fetch(tile + s * (size_t)gridDim.y, s);
  const size_t step = (size_t)TY * K;
  int stage = 0;
  for (; tile < tiles; tile += gridDim.y) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
    __syncthreads();  // the stage is complete, and the one before it is read no more
    fetch(tile + (kRing - 1) * (size_t)gridDim.y, stage == 0 ? kRing - 1 : stage - 1);
    const size_t m0 = tile * rows;
    const int left = (int)(M - m0 < (size_t)rows ? M - m0 : rows);
    double *dst = dA + (m0 + threadIdx.y) * K + c0;
    const double *g = &gs[stage][threadIdx.y * NN];
    const uint8_t *code = &cs[stage][threadIdx.y * width + mine];
#pragma unroll 2
    for (int r = threadIdx.y; r < left; r += TY, dst += step, g += TY * NN, code += TY * width) {
      int k0, k1;
      if (PAIR) {
        const short two = *reinterpret_cast<const short *>(code);
        k0 = (signed char)two;
        k1 = two >> 8;
      } else {
        k0 = (signed char)code[0];
        k1 = (signed char)code[apart];
      }
      double s0 = 0.0, s1 = 0.0;
#pragma unroll
      for (int n = 0; n < NN; n += 2) {
        const double2 v = *reinterpret_cast<const double2 *>(g + n);
        s0 = fma(v.x, b0[n], s0);
        s1 = fma(v.x, b1[n], s1);
        s0 = fma(v.y, b0[n + 1], s0);
        s1 = fma(v.y, b1[n + 1], s1);
      }
      s0 = s0 * (k0 > 0 ? 1.0 : 0.0);
      s1 = s1 * (k1 > 0 ? 1.0 : 0.0);
      if (PAIR) {
        if (!in0) continue;
        if (accumulate) {
          const double2 o = *reinterpret_cast<const double2 *>(dst);
          s0 = o.x + s0;
          s1 = o.y + s1;
        }
        __stcs(reinterpret_cast<double2 *>(dst), make_double2(s0, s1));
      } else {
        if (in0) dst[0] = accumulate ? dst[0] + s0 : s0;
        if (in1) dst[apart] = accumulate ? dst[apart] + s1 : s1;
      }
    }
    stage = stage + 1 == kRing ? 0 : stage + 1;
  }
}

template <int NN>
static void launch_outer(dim3 grid, dim3 block, bool pair, int access, const double *G, const double *B, double *dA,
                         const signed char *mask, size_t M, int N, size_t K, bool acc) {
  cudaStream_t s = ctx().stream;
  if (pair && access == kCodes16) q8_outer_kernel<NN, true, kCodes16><<<grid, block, 0, s>>>(G, B, dA, mask, M, N, K, acc);
  else if (pair && access == kCodes4) q8_outer_kernel<NN, true, kCodes4><<<grid, block, 0, s>>>(G, B, dA, mask, M, N, K, acc);
  else if (pair) q8_outer_kernel<NN, true, kCodes1><<<grid, block, 0, s>>>(G, B, dA, mask, M, N, K, acc);
  else q8_outer_kernel<NN, false, kCodes1><<<grid, block, 0, s>>>(G, B, dA, mask, M, N, K, acc);
}

static int outer_q8(const double *G, const double *B, double *dA, size_t M, size_t N, size_t K, int accumulate,
                    const signed char *mask) {
  unsigned tx = 32;
  while (tx < 256 && 2 * (size_t)tx < K) tx *= 2;
  const bool pair = K % 2 == 0 && !off_16_bytes(dA);
  const int access = code_access(mask, K);
  const size_t rows = (size_t)kOuterRows * (256 / tx), gx = (K + 2 * tx - 1) / (2 * tx), tiles = (M + rows - 1) / rows;
  // (one wave: a CTA's start, its rows of B, costs as much as several tiles)
  size_t gy = (size_t)ctx().sm_count * outer_ctas((int)N) / gx;
  if (gy < 1) gy = 1;
  if (gy > tiles) gy = tiles;
  const dim3 grid((unsigned)gx, (unsigned)gy), block(tx, 256 / tx);
  switch ((N + 1) / 2) {
    case 1: launch_outer<2>(grid, block, pair, access, G, B, dA, mask, M, (int)N, K, accumulate != 0); break;
    case 2: launch_outer<4>(grid, block, pair, access, G, B, dA, mask, M, (int)N, K, accumulate != 0); break;
    case 3: launch_outer<6>(grid, block, pair, access, G, B, dA, mask, M, (int)N, K, accumulate != 0); break;
    case 4: launch_outer<8>(grid, block, pair, access, G, B, dA, mask, M, (int)N, K, accumulate != 0); break;
    case 5: launch_outer<10>(grid, block, pair, access, G, B, dA, mask, M, (int)N, K, accumulate != 0); break;
    case 6: launch_outer<12>(grid, block, pair, access, G, B, dA, mask, M, (int)N, K, accumulate != 0); break;
    case 7: launch_outer<14>(grid, block, pair, access, G, B, dA, mask, M, (int)N, K, accumulate != 0); break;
    default: launch_outer<16>(grid, block, pair, access, G, B, dA, mask, M, (int)N, K, accumulate != 0); break;
  }
  MG_LAUNCH_CHECK("gemm_nt_q8 (few columns)");
  return MG_OK;
}

// dB[K][N] (+)= (codes scales)[M][K]^T . G[M][N], N <= 32.  A CTA takes one block of 64
// columns of the codes (so one scale per row) and a piece of the rows; its four warps
// take every fourth row, a lane two columns with their N sums each.  The warps' sums are
// added up in order, the pieces' by a second kernel, in order.  N + 2 fp64 instructions
// per code are 43 us of 65 536 x 1024 x 10 at their rate, of 98: the counters show the
// fp64 units half busy, shared memory at 61 %, 2.1 instructions a cycle from 12 warps per
// SM.  The rest is what a lane does for a row besides its sums (G's values, a scale, two
// codes, their widening), which serves two columns only.
constexpr int kTallThreads = 128, kTallRows = 32;
// CTAs per SM: 65 536 x 1024, ten columns: 98 us with four and all eight rows of a warp
// unrolled, 112 with six and two rows (more warps, but twice the instructions a row).
constexpr int tall_ctas(int nn) { return nn <= 16 ? 4 : 3; }

template <int NN, int ACCESS>
__global__ void __launch_bounds__(kTallThreads, tall_ctas(NN))
q8_tall_kernel(const signed char *__restrict__ codes, const double *__restrict__ scales,
               const double *__restrict__ G, double *__restrict__ parts, size_t M, int N, size_t K, size_t nb,
               size_t piece) {
  // gs is reused for the sums: NN x 64 doubles fit kRing x 32 x NN.
  __shared__ __align__(16) double gs[kRing][kTallRows * NN];
  __shared__ __align__(16) double ss[kRing][kTallRows];
  __shared__ __align__(16) uint8_t cs[kRing][kTallRows * 64];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t col0 = (size_t)blockIdx.x * 64, begin = blockIdx.y * piece, end = begin + piece < M ? begin + piece : M;
  if (N < NN)
    for (int i = threadIdx.x; i < kRing * kTallRows * (NN - N); i += kTallThreads) {
      const int s = i / (kTallRows * (NN - N)), j = i - s * kTallRows * (NN - N);
      gs[s][(j / (NN - N)) * NN + N + j % (NN - N)] = 0.0;
    }
  const bool run = N == NN && (reinterpret_cast<uintptr_t>(G) & 15) == 0;
  auto fetch = [&](size_t m0, int stage) {
    if (m0 < end) {
      const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;
      copy_codes<ACCESS>(&cs[stage][r * 64 + c], codes, m0 + r, end, col0 + c, K);
      if (threadIdx.x < kTallRows) {
        const bool in = m0 + threadIdx.x < end;
        copy8(&ss[stage][threadIdx.x], in ? scales + (m0 + threadIdx.x) * nb + blockIdx.x : scales, in);
      }
      copy_g<NN>(gs[stage], G, m0, end, kTallRows, N, threadIdx.x, kTallThreads, run);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  double a0[NN], a1[NN];
#pragma unroll
  for (int n = 0; n < NN; n++) a0[n] = a1[n] = 0.0;
#pragma unroll
  for (int s = 0; s < kRing - 1; s++) fetch(begin + s * kTallRows, s);
  int stage = 0;
  for (size_t m0 = begin; m0 < end; m0 += kTallRows) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
    __syncthreads();  // the stage is complete, and the one before it is read no more
    fetch(m0 + (kRing - 1) * kTallRows, stage == 0 ? kRing - 1 : stage - 1);
#pragma unroll
    for (int r0 = 0; r0 < kTallRows; r0 += 4) {  // (rows behind the end are zeros)
      const int r = r0 + warp;
      const int two = *reinterpret_cast<const unsigned short *>(&cs[stage][r * 64 + 2 * lane]) ^ 0x8080;
      const double s = ss[stage][r];
      // the byte, its top bit flipped, as the low end of 2^52 + byte + 128
      const double x0 = (__hiloint2double(0x43300000, two & 255) - 4503599627370624.0) * s;
      const double x1 = (__hiloint2double(0x43300000, two >> 8) - 4503599627370624.0) * s;
      const double *g = &gs[stage][r * NN];
#pragma unroll
      for (int n = 0; n < NN; n += 2) {
        const double2 v = *reinterpret_cast<const double2 *>(g + n);
        a0[n] = fma(x0, v.x, a0[n]);
        a1[n] = fma(x1, v.x, a1[n]);
        a0[n + 1] = fma(x0, v.y, a0[n + 1]);
        a1[n + 1] = fma(x1, v.y, a1[n + 1]);
      }
    }
    stage = stage + 1 == kRing ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  double *sums = &gs[0][0];  // [n][column]
  for (int w = 0; w < 4; w++) {
    __syncthreads();
    if (warp == w) {
#pragma unroll
      for (int n = 0; n < NN; n++) {
        double2 *s = reinterpret_cast<double2 *>(sums + n * 64 + 2 * lane);
        const double2 o = w == 0 ? make_double2(0.0, 0.0) : *s;
        *s = make_double2(o.x + a0[n], o.y + a1[n]);
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 64 * N; i += kTallThreads) {
    const int c = i / N, n = i - c * N;
    if (col0 + c < K) parts[(blockIdx.y * K + col0 + c) * N + n] = sums[n * 64 + c];
  }
}

__global__ void __launch_bounds__(256)
q8_tall_join_kernel(const double *__restrict__ parts, size_t pieces, size_t n, double *dB, bool accumulate) {
  cudaGridDependencySynchronize();
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  double s = 0.0;
#pragma unroll 8
  for (size_t k = 0; k < pieces; k++) s += __ldcs(parts + k * n + i);
  dB[i] = accumulate ? dB[i] + s : s;
}

template <int NN>
static int launch_tall(const signed char *codes, const double *scales, const double *G, double *dB, size_t M, size_t N,
                       size_t K, int accumulate) {
  Context &c = ctx();
  const size_t gx = q8_blocks(K);
  // One wave, each CTA with at least four tiles of rows.
  size_t pieces = (size_t)c.sm_count * tall_ctas(NN) / gx;
  if (pieces < 1) pieces = 1;
  const size_t most = (M + 4 * kTallRows - 1) / (4 * kTallRows);
  if (pieces > most) pieces = most;
  const size_t piece = ((M + pieces - 1) / pieces + kTallRows - 1) / kTallRows * kTallRows;
  pieces = (M + piece - 1) / piece;
  double *parts = dB;
  const bool direct = pieces == 1 && !accumulate;
  if (!direct) {
    int rc = mg_alloc(pieces * K * N, &parts);
    if (rc != MG_OK) return rc;
  }
  const dim3 grid((unsigned)gx, (unsigned)pieces);
  const int access = code_access(codes, K);
  if (access == kCodes16)
    q8_tall_kernel<NN, kCodes16><<<grid, kTallThreads, 0, c.stream>>>(codes, scales, G, parts, M, (int)N, K, gx, piece);
  else if (access == kCodes4)
    q8_tall_kernel<NN, kCodes4><<<grid, kTallThreads, 0, c.stream>>>(codes, scales, G, parts, M, (int)N, K, gx, piece);
  else
    q8_tall_kernel<NN, kCodes1><<<grid, kTallThreads, 0, c.stream>>>(codes, scales, G, parts, M, (int)N, K, gx, piece);
  MG_LAUNCH_CHECK("gemm_tn_q8 (few columns)");
  if (direct) return MG_OK;
  MG_CUDA_TRY(launch_overlapped(q8_tall_join_kernel, dim3((unsigned)((K * N + 255) / 256)), dim3(256), parts, pieces, K * N,
                                dB, accumulate != 0));
  MG_LAUNCH_CHECK("gemm_tn_q8 (join)");
  return mg_free(parts);
}

static int tall_q8(const signed char *codes, const double *scales, const double *G, double *dB, size_t M, size_t N,
                   size_t K, int accumulate) {
  if (N <= 2) return launch_tall<2>(codes, scales, G, dB, M, N, K, accumulate);
  if (N <= 4) return launch_tall<4>(codes, scales, G, dB, M, N, K, accumulate);
  if (N <= 6) return launch_tall<6>(codes, scales, G, dB, M, N, K, accumulate);
  if (N <= 8) return launch_tall<8>(codes, scales, G, dB, M, N, K, accumulate);
  if (N <= 10) return launch_tall<10>(codes, scales, G, dB, M, N, K, accumulate);
  if (N <= 12) return launch_tall<12>(codes, scales, G, dB, M, N, K, accumulate);
  if (N <= 16) return launch_tall<16>(codes, scales, G, dB, M, N, K, accumulate);
  if (N <= 24) return launch_tall<24>(codes, scales, G, dB, M, N, K, accumulate);
  return launch_tall<32>(codes, scales, G, dB, M, N, K, accumulate);
}

// x[M][pitch] = the values of codes[M][N]; what is behind the N columns stays as it is.
static int unpack_rows(const signed char *codes, const double *scales, double *x, size_t pitch, size_t M, size_t N) {
  const size_t nb = q8_blocks(N), blocks = M * nb;
  int vec = q8_vec(x, codes, N);
  if (pitch % 4 != 0 && vec == 4) vec = pitch % 2 == 0 ? 2 : 1;
  const unsigned grid = grid_for(blocks * (vec == 4 ? 16 : 32), kQ8Threads, 64);
  if (vec == 4 && N % 64 == 0 && pitch == N)
    MG_CUDA_TRY(launch_overlapped(q8_unpack_kernel<4, 4, true>, dim3(grid), dim3(kQ8Threads), codes, scales, x, pitch, blocks, N, (unsigned)nb));
  else if (vec == 4)
    MG_CUDA_TRY(launch_overlapped(q8_unpack_kernel<4, 2, false>, dim3(grid), dim3(kQ8Threads), codes, scales, x, pitch, blocks, N, (unsigned)nb));
  else if (vec == 2)
    MG_CUDA_TRY(launch_overlapped(q8_unpack_kernel<2, 4, false>, dim3(grid), dim3(kQ8Threads), codes, scales, x, pitch, blocks, N, (unsigned)nb));
  else
    MG_CUDA_TRY(launch_overlapped(q8_unpack_kernel<1, 4, false>, dim3(grid), dim3(kQ8Threads), codes, scales, x, pitch, blocks, N, (unsigned)nb));
  MG_LAUNCH_CHECK("q8_unpack");
  return MG_OK;
}

// fp64 values held at a time for a weight gradient, and for the rows of an input gradient
// that have to be copied.
constexpr size_t kQ8UnpackBytes = (size_t)256 << 20;

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
  const unsigned grid = grid_for(blocks * 32, kQ8Threads, 64), wide = (unsigned)nb;
  const bool pair = q8_vec(x, codes, N) >= 2;
  if (pair && N % 64 == 0)
    MG_CUDA_TRY(launch_overlapped(q8_pack_kernel<true, 2, true>, dim3(grid), dim3(kQ8Threads), x, codes, scales, blocks, N, wide));
  else if (pair)
    MG_CUDA_TRY(launch_overlapped(q8_pack_kernel<true, 4, false>, dim3(grid), dim3(kQ8Threads), x, codes, scales, blocks, N, wide));
  else
    MG_CUDA_TRY(launch_overlapped(q8_pack_kernel<false, 4, false>, dim3(grid), dim3(kQ8Threads), x, codes, scales, blocks, N, wide));
  MG_LAUNCH_CHECK("q8_pack");
  return MG_OK;
}

int mg_q8_unpack(const signed char *codes, const double *scales, double *x, size_t M, size_t N) {
  int rc = check_q8("mg_q8_unpack", M, N);
  if (rc != MG_OK) return rc;
  if (M && N && (!x || !codes || !scales)) return fail(MG_ERR_INVALID, "mg_q8_unpack: null pointer");
  MG_ENSURE_INIT();
  if (M == 0 || N == 0) return MG_OK;
  return unpack_rows(codes, scales, x, N, M, N);
}

int mg_relu_bwd_q8(const signed char *codes, const double *g, double *gx, size_t n, int flags) {
  if (n && (!codes || !g || !gx)) return fail(MG_ERR_INVALID, "mg_relu_bwd_q8: null pointer");
  MG_ENSURE_INIT();
  if (n == 0) return MG_OK;
  const bool quads = ((reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(gx)) & 31) == 0 &&
                     (reinterpret_cast<uintptr_t>(codes) & 3) == 0;
  MG_CUDA_TRY(launch_overlapped(quads ? q8_relu_bwd_kernel<true> : q8_relu_bwd_kernel<false>,
                                dim3(grid_for(quads ? (n + 3) / 4 : n, kQ8Threads, 64)), dim3(kQ8Threads), codes, g, gx, n,
                                !(flags & MG_ACC_STORE_A)));
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
  if (M == 0) return accumulate ? MG_OK : mg_fill(dB, 0.0, K * N);
  if (N <= 32) return tall_q8(codes, scales, G, dB, M, N, K, accumulate);
  // Output [K][N], contraction over the M rows: the tensor kernel on the fp64 form of as
  // many rows at a time as kQ8UnpackBytes hold.  Widening costs 9 bytes of traffic per
  // code against 2 N flop: 2 % of the product at 1024 columns.  (Codes widened by the
  // kernel's own producer warps were slower: the fp64 units, or the warps' latency, then
  // hold up the tensor instructions; 4.32 ms against 4.05 at 65 536 x 1024 x 1024.)
  const size_t pitch = pitch16(K), pitch_g = pitch16(N);
  const bool copy_g = N % 2 != 0 || off_16_bytes(G);
  size_t rows = kQ8UnpackBytes / 8 / (copy_g && pitch_g > pitch ? pitch_g : pitch) / 64 * 64;
  if (rows < 64) rows = 64;
  if (rows > M) rows = M;
  double *room = nullptr;
  rc = mg_alloc(rows * pitch + (copy_g ? rows * pitch_g : 0), &room);
  if (rc != MG_OK) return rc;
  const size_t nb = q8_blocks(K);
  for (size_t m = 0; m < M && rc == MG_OK; m += rows) {
    const size_t part = M - m < rows ? M - m : rows;
    rc = unpack_rows(codes + m * K, scales + m * nb, room, pitch, part, K);
    GemmExt e{{room, G + m * N, dB, K, N, part, false, false, accumulate || m > 0, MG_EPI_NONE, nullptr}};
    e.lda = pitch;
    if (rc == MG_OK && copy_g) {
      e.d.B = room + rows * pitch;
      e.ldb = pitch_g;
      rc = copy_rows(G + m * N, part, N, N, room + rows * pitch, pitch_g);
    }
    if (rc == MG_OK) rc = run_gemm_ext(e);
  }
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
  // Odd rows, or rows off a 16-byte boundary: B is copied once into rows the tensor kernel
  // can take, G in pieces of as many rows as kQ8UnpackBytes hold.
  const size_t pitch = pitch16(N);
  size_t rows = kQ8UnpackBytes / 8 / pitch / 128 * 128;
  if (rows < 128) rows = 128;
  if (rows > M) rows = M;
  double *room = nullptr;
  int rc = mg_alloc((rows + K) * pitch, &room);
  if (rc != MG_OK) return rc;
  rc = copy_rows(B, K, N, N, room + rows * pitch, pitch);
  e.d.A = room;
  e.d.B = room + rows * pitch;
  e.lda = e.ldb = pitch;
  for (size_t m = 0; m < M && rc == MG_OK; m += rows) {
    e.d.M = M - m < rows ? M - m : rows;
    e.d.D = dA + m * K;
    e.mask8 = mask_codes + m * K;
    rc = copy_rows(G + m * N, e.d.M, N, N, room, pitch);
    if (rc == MG_OK) rc = run_gemm_ext(e);
  }
  const int freed = mg_free(room);
  return rc != MG_OK ? rc : freed;
}

}  // extern "C"
