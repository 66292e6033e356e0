// The last step of the column sums of layer_norm_backward and linear_backward.
#pragma once
#include "nn_common.h"

namespace mia {
namespace nn {
// Sums over groups of partial[group][i], i < n, in a fixed order, in double; the first `split` go to out0, the
// rest to out1.  32 columns per workgroup, each of its 32 slices every 32nd group.
static __global__ __launch_bounds__(1024) void join_columns_kernel(const float* __restrict__ partial, int groups, int n,
                                                                   float* __restrict__ out0, float* __restrict__ out1,
                                                                   int split) {
  __shared__ double part[32][32];
  const int slice = threadIdx.x >> 5, c = threadIdx.x & 31;
  const int i = blockIdx.x * 32 + c;
  double s[2] = {};
  if (i < n) {
    int g = slice;
    for (; g + 96 < groups; g += 128) {  // four loads in flight
      const float a = partial[(long long)g * n + i], b = partial[(long long)(g + 32) * n + i];
      const float d = partial[(long long)(g + 64) * n + i], e = partial[(long long)(g + 96) * n + i];
      s[0] += (double)a + (double)b;
      s[1] += (double)d + (double)e;
    }
    for (; g < groups; g += 32) s[0] += (double)partial[(long long)g * n + i];
  }
  part[slice][c] = s[0] + s[1];
  __syncthreads();
  if (slice == 0 && i < n) {
    double t = 0.0;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += part[k][c];
    (i < split ? out0[i] : out1[i - split]) = (float)t;
  }
}
}  // namespace nn
}  // namespace mia
