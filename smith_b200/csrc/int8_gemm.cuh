// int8_gemm.cuh -- layout of the packed int8 weights and the launches that make codes (int8_rows.cu),
// shared with the product (int8_gemm.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace smith {

// Layout of packed weights [experts][K][N]; the format is described in int8_rows.cu.
struct int8_layout {
  int64_t n_tiles, k_slabs, experts;
  size_t code_bytes, bytes;     // the channels' maxima f32 [experts][n_tiles * 128] start at code_bytes
};
int8_layout int8_weight_layout(int64_t K, int64_t N, int64_t experts);

// Codes and maxima (NaN for a row that is not finite) of `rows` rows of a [rows][K] (pitch lda elements; dtype kDenseF32 / kDenseF16):
// codes [places][K rounded up to 128] and maxima [places]; row r goes to place r, or with `position` to
// the places position[r * fan .. r * fan + fan).  Places outside [0, places) are skipped.
// n_counters words at `counters` are set to 0.
cudaError_t launch_int8_rows(int dtype, const void* a, int64_t rows, int64_t lda, int64_t K, const int* position, int fan,
                             int64_t places, uint8_t* codes, float* maxima, int* counters, int n_counters,
                             cudaStream_t s);

}  // namespace smith
