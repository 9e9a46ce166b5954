// What the matrix product dispatcher of gemm.cu offers to the library's other files.
#pragma once

#include "common.cuh"

namespace mg {

struct GemmDesc {
  const double *A;  // a_kcontig ? [M][K] : [K][M]
  const double *B;  // b_kcontig ? [N][K] : [K][N]
  double *D;        // [M][N]
  size_t M, N, K;
  bool a_kcontig, b_kcontig;
  int accumulate, mode;
  const double *aux;
};

// One of the dense products of gemm.cu.
int run_gemm(const GemmDesc &d);

// The same on the tensor-core kernel with what the dense form does not know: row
// pitches (0: dense), any row lengths of the output, few rows, or an output mask in 8
// bits.  A and B may have any extents, but need even row pitches and 16-byte aligned
// bases, and an operand whose contiguous axis is not k must have memory up to a pitch
// that is a multiple of 16 where its row length is none (what it holds there is not
// used).
struct GemmExt {
  GemmDesc d;
  size_t lda = 0, ldb = 0, ldd = 0;
  const signed char *mask8 = nullptr;  // [M][N]: output * (mask8 > 0)
};
int run_gemm_ext(const GemmExt &e);

// dst[rows][dst_pitch] = src[rows][src_pitch], cols of each row; zeros up to dst_pitch.
// Where labels are given, a row whose label is outside [0, classes) becomes zeros.
int copy_rows(const double *src, size_t rows, size_t cols, size_t src_pitch, double *dst, size_t dst_pitch,
              const int *labels = nullptr, size_t classes = 0);

inline size_t pitch16(size_t n) { return (n + 15) / 16 * 16; }
inline bool off_16_bytes(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace mg
