// ks_kv4.cuh -- the paged 4-bit key/value cache: where a token's codes,
// scales and accumulated weight stand, shared by the kernels that write, read
// and evict (ks_kv4.cu) and those that attend (ks_kv4_attention.cuh).
//
// A pool holds n_pages pages of page_size tokens (a power of two, 16..256),
// each [kv_head][page_size / 16 blocks].  A block is 16 tokens of one head:
//   key codes   16 rows of head_dim / 2 bytes
//   key scales  16 rows of head_dim / group f16
//   value codes, value scales likewise
// in one piece, so that any run of blocks within a page, and a block's keys
// alone, are consecutive bytes, which arrive in shared memory by asynchronous
// 16-byte copies.  Codes are the library's signed int4 (even element in the low half of its byte).
// Within a row the bytes stand in the order in which the lanes of a warp feed
// them to the tensor cores:
//   keys    pair d, d+1 (d even) is byte (d%32/8) * (head_dim/8) + (d/32)*4 + d%8/2
//           (lane t of four takes elements 8t..8t+7 of every 32: head_dim/8
//           bytes in a row, one 16-byte load at head_dim 128)
//   values  pair d, d+1 is byte (d%16/2) * (head_dim/16) + d/16
//           (lane g of eight takes elements 2g, 2g+1 of every 16)
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "ks_internal.h"
#include "ks_ptx.cuh"

namespace ksb {

constexpr int kKv4Block = 16;  // tokens
// Words at the start of a workspace that are 0 between calls of the attention.
constexpr int kKv4Counters = 2048;

__host__ __device__ constexpr int kv4_half_block_bytes(int d, int groups) { return kKv4Block * (d / 2 + 2 * groups); }
__host__ __device__ constexpr int kv4_block_bytes(int d, int groups) { return 2 * kv4_half_block_bytes(d, groups); }

// On streams where launches may overlap, every kernel of the cache waits for
// the kernels before it before it touches memory, and lets the next one be set
// up after that.
__device__ __forceinline__ void kv4_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void kv4_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void kv4_begin() {
  kv4_wait();
  kv4_next();
}

template <typename... A, typename... B>
cudaError_t kv4_launch(void (*kernel)(A...), dim3 grid, int threads, size_t shared, cudaStream_t stream, B... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  if (pdl_enabled(stream)) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, kernel, A(args)...);
}

// A sequence's part of the call: its cached tokens (the new ones among them),
// its first row among the packed new tokens and how many it has.  A
// descriptor that does not fit the call's buffers is reported in status word
// 0 and reads as a sequence without tokens or without rows.
struct Kv4Seq {
  int len, first, n_new;
};

__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4Batch &b, int s, uint32_t *status) {
  Kv4Seq q;
  q.first = b.offsets ? b.offsets[s] : s;
  q.n_new = b.offsets ? b.offsets[s + 1] - q.first : 1;
  q.len = b.lens[s];
  if (q.len < 0 || q.len > b.max_len) {
    set_status(status, kStatusBadScale);
    q.len = 0;
  }
  if (q.first < 0 || q.n_new < 0 || q.first > b.n_tokens || q.n_new > b.n_tokens - q.first) {
    set_status(status, kStatusBadScale);
    q.n_new = 0;
  }
  return q;
}

// The page that holds token `pos` of sequence s, or -1 (reported) when the
// table names none of the pool's.
__device__ __forceinline__ int kv4_page(const Kv4View &c, const int32_t *table, int64_t stride, int s, int pos,
                                        uint32_t *status) {
  const int p = table[s * stride + (pos >> c.page_shift)];
  if ((uint32_t)p < (uint32_t)c.n_pages) return p;
  set_status(status, kStatusBadScale);
  return -1;
}

// Start of the block that holds slot `slot` of a page's head.
__device__ __forceinline__ uint8_t *kv4_block(const Kv4View &c, int page, int head, int slot) {
  return c.pool + page * c.page_bytes + head * c.head_bytes + (int64_t)(slot >> 4) * c.block_bytes;
}

__device__ __forceinline__ float kv4_load(const float *p) { return *p; }
__device__ __forceinline__ float kv4_load(const __half *p) { return __half2float(*p); }
__device__ __forceinline__ float kv4_load(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ void kv4_store(float *p, float v) { *p = v; }
__device__ __forceinline__ void kv4_store(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void kv4_store(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}

template <int BYTES>
__device__ __forceinline__ void lds(const void *p, uint32_t (&w)[BYTES / 4]) {
  if constexpr (BYTES == 16) {
    const uint4 v = *static_cast<const uint4 *>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (BYTES == 8) {
    const uint2 v = *static_cast<const uint2 *>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *static_cast<const uint32_t *>(p);
  }
}

// The NG scales of one token.
template <int NG>
__device__ __forceinline__ void load_scales(const void *p, float (&s)[NG]) {
  const __half *h = static_cast<const __half *>(p);
  if constexpr (NG == 1) {
    s[0] = __half2float(h[0]);
  } else {
    uint32_t w[NG / 2];
    lds<NG * 2>(p, w);
#pragma unroll
    for (int k = 0; k < NG / 2; ++k) {
      const float2 v = unpack_f16(w[k]);
      s[2 * k] = v.x, s[2 * k + 1] = v.y;
    }
  }
}

}  // namespace ksb
