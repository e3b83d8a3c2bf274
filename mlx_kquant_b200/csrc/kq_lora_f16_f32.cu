// The tile kernels of __half rows and float parameters (kq_lora.cuh).
#include "kq_lora.cuh"

namespace kq {
cudaError_t launch_lora_tile_f16_f32(const LoraArgs& a, bool backward, int mt, int cluster, cudaStream_t st) {
  return lora::launch_types<__half, float>(a, backward, mt, cluster, st);
}
}  // namespace kq
