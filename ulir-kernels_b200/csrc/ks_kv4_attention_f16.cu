// ks_kv4_attention_f16.cu -- the attention kernels of ks_kv4_attention.cuh for f16 queries and outputs.

#include "ks_kv4_attention.cuh"

namespace ksb {

cudaError_t launch_kv4_attention_f16(const Kv4AttnArgs &k, cudaStream_t stream, int device) {
  return launch_kv4_attention_typed<__half, 1, 2>(k, stream, device);
}

}  // namespace ksb
