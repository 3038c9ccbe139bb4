// moe.cuh — the router as other kernels' first launch.
#pragma once
#include <cuda_runtime.h>

namespace nvfp4 {
namespace moe {

// nvfp4_moe_route with its checks; its first launch also sets n_clear integers of `clear` to
// zero.
int route_tokens(const void *logits, int dtype, const float *bias, int T, int E, int top_k, int scoring,
                 int renormalize, float scale, float *weights, int *experts, int *rows, int *m_offsets,
                 void *workspace, size_t workspace_bytes, int *clear, int n_clear, void *stream);

}  // namespace moe
}  // namespace nvfp4
