// The tile kernels of bf16 rows and float parameters (kq_lora.cuh).
#include "kq_lora.cuh"

namespace kq {
cudaError_t launch_lora_tile_bf16_f32(const LoraArgs& a, bool backward, int mt, int cluster, cudaStream_t st) {
  return lora::launch_types<lora::bf16, float>(a, backward, mt, cluster, st);
}
}  // namespace kq
