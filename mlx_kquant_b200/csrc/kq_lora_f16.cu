// The tile kernels of __half rows and __half parameters (kq_lora.cuh).
#include "kq_lora.cuh"

namespace kq {
cudaError_t launch_lora_tile_f16(const LoraArgs& a, bool backward, int mt, int cluster, cudaStream_t st) {
  return lora::launch_types<__half, __half>(a, backward, mt, cluster, st);
}
}  // namespace kq
