// What the two forms of the Newton-Schulz steps share (ortho.cu: any size, a
// launch a product; ortho_small.cu: small matrices, one launch).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace h3b {

struct OrthoCall {
  const void* x;
  void* out;
  int dtype;
  int64_t batch, m, n;
  int64_t batch_stride, ld;  // of x; out is contiguous
  int steps;
  float a, b, c, eps;
};

// Whether one cluster of CTAs holds a matrix of these sides in shared memory.
bool ortho_small_fits(int64_t m, int64_t n);
int ortho_small(const OrthoCall& call, cudaStream_t stream);

}  // namespace h3b
