// Arguments shared by the cross-attention gradient kernels.
#pragma once

#include "cross_attention.cuh"

namespace bl {
namespace xa {

struct BackArgs {
  Args a;  // a.out: the forward's output, a.lse: its statistics
  const void *dy, *dout;  // gradient of out; do ([batch][nq][heads][d]; dy itself without a gate)
  const void *dlow;       // bf16 with a gate: do - bf16(do), else null
  float *delta;           // [batch][heads][nq]
  void *dq, *dk, *dv, *dgate, *dbias;  // contiguous; dbias [batch / share][heads][nq][dbias_ld] or null
  int64_t dbias_ld;
};

// The saved reference of a row's scores as the gradient kernels want it: +inf for a query
// without keys (all its p become 0).
__device__ __forceinline__ float row_max(float m) { return m == -INFINITY ? INFINITY : m; }

// cross_attention_backward_tc.cu: each runs its kernel and sets *taken where it covers the call.
int keys_tc(const BackArgs &x, cudaStream_t stream, bool *taken);
int queries_tc(const BackArgs &x, cudaStream_t stream, bool *taken);
int bias_tc(const BackArgs &x, cudaStream_t stream, bool *taken);

}  // namespace xa
}  // namespace bl
