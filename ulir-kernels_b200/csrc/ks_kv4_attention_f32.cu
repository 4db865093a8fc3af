// ks_kv4_attention_f32.cu -- the attention kernels of ks_kv4_attention.cuh for f32 queries and outputs.

#include "ks_kv4_attention.cuh"

namespace ksb {

cudaError_t launch_kv4_attention_f32(const Kv4AttnArgs &k, cudaStream_t stream, int device) {
  return launch_kv4_attention_typed<float, 2, 2>(k, stream, device);
}

}  // namespace ksb
