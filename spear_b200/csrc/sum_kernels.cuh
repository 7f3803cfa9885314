// Sums over the rows of a buffer of partial results, in a fixed order.
#pragma once

#include "btp_elem.cuh"

namespace btp_elem {

// out[j] = sum over i of part[i][j], in the order of i within each strand and then of the strands; out in float or T.
// CTA: 32 columns x STRANDS (8 for a few rows, 32 for hundreds).
template <class T, int STRANDS>
__global__ void __launch_bounds__(32 * STRANDS) column_sum_kernel(const float* part, void* out, int parts, long long cols, bool out_f32) {
  __shared__ float s[STRANDS][33];
  const int lane = threadIdx.x & 31, strand = threadIdx.x >> 5;
  const long long j = static_cast<long long>(blockIdx.x) * 32 + lane;
  grid_dependency_wait();
  float a = 0.f;
  if (j < cols)
#pragma unroll 4
    for (int i = strand; i < parts; i += STRANDS) a += part[i * cols + j];
  s[strand][lane] = a;
  __syncthreads();
  if (strand == 0 && j < cols) {
    a = s[0][lane];
#pragma unroll
    for (int i = 1; i < STRANDS; ++i) a += s[i][lane];
    if (out_f32)
      static_cast<float*>(out)[j] = a;
    else
      static_cast<T*>(out)[j] = from_f<T>(a);
  }
}

}  // namespace btp_elem
