// Internal interface of the grouped router (kq_route.cu) to its C entry points.
#pragma once

#include <cuda_runtime.h>

namespace kq {

struct RouteArgs {
  const void* logits;  // [T, E]
  int dtype, T, E, G, top_groups, group_top, top_k, scoring, norm;  // scoring: 0 softmax, 1 sigmoid
  const float* bias;   // [E] or nullptr
  float scale;
  int* indices;        // [T, top_k]
  float* weights;      // [T, top_k]
  const float* dw;     // [T, top_k]  (gradient only)
  void* dlogits;       // [T, E], or nullptr: the forward pass
  int size, whole, whole_bias;  // set by the launch: experts of a group; a lane's logits, biases are read at once
};
cudaError_t launch_route(RouteArgs a, cudaStream_t st);

}  // namespace kq
