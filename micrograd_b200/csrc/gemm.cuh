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

int run_gemm(const GemmDesc &d);

}  // namespace mg
