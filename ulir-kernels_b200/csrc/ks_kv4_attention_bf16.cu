// ks_kv4_attention_bf16.cu -- the attention kernels of ks_kv4_attention.cuh for bf16 queries and outputs.

#include "ks_kv4_attention.cuh"

namespace ksb {

cudaError_t launch_kv4_attention_bf16(const Kv4AttnArgs &k, cudaStream_t stream, int device) {
  return launch_kv4_attention_typed<__nv_bfloat16, 1, 1>(k, stream, device);
}

}  // namespace ksb
