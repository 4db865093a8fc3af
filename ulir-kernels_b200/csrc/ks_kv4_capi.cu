// ks_kv4_capi.cu -- C entry points of the paged 4-bit key/value cache
// (include/ks_b200.h): argument checks, then the launches of ks_kv4.cu and
// ks_kv4_attention.cuh.

#include <cmath>
#include <cstdint>
#include <string>

#include "ks_b200.h"
#include "ks_internal.h"
#include "ks_kv4_attention.cuh"

using namespace ksb;

namespace {

int fail(int code, const char *msg) {
  set_last_error(msg);
  return code;
}

int cuda_fail(cudaError_t e, const char *what) {
  set_last_error(std::string(what) + ": " + cudaGetErrorString(e));
  cudaGetLastError();
  return KS_ERR_DEVICE;
}

constexpr size_t kMost = 0x7FFFFFFF;
constexpr size_t kMaxLen = kMost - 16384;  // positions of 32 tiles ahead are 32-bit
constexpr size_t kPlanSms = 148;  // a B200's; a constant, so that the workspace needs no device to be known

bool misaligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; }

bool shape_supported(size_t page_size, size_t kv_heads, size_t head_dim, size_t group) {
  return page_size >= 16 && page_size <= 256 && !(page_size & (page_size - 1)) && kv_heads > 0 && kv_heads <= 65535 &&
         (head_dim == 64 || head_dim == 128) && (group == 32 || group == 64 || group == 128) && group <= head_dim;
}

// The cache's description in the kernels' terms; KS_OK or an error.
int view_of(const ks_b200_kv4_cache *c, Kv4View *v) {
  if (!c || !c->pool) return fail(KS_ERR_INVALID_ARG, "NULL pointer");
  if (c->n_pages == 0 || c->page_size == 0 || c->kv_heads == 0 || c->head_dim == 0 || c->group_size == 0)
    return fail(KS_ERR_INVALID_ARG, "n_pages, page_size, kv_heads, head_dim and group_size must be > 0");
  if (misaligned(c->pool, 16) || misaligned(c->weights, 4))
    return fail(KS_ERR_INVALID_ARG, "the pool must be 16-byte aligned, the weights 4-byte aligned");
  if (c->n_pages > kMost || !shape_supported(c->page_size, c->kv_heads, c->head_dim, c->group_size))
    return fail(KS_ERR_UNSUPPORTED,
                "the 4-bit cache needs page_size 16, 32, 64, 128 or 256, head_dim 64 or 128, group_size 32, 64 or 128 "
                "and at most head_dim, kv_heads <= 65535");
  v->pool = static_cast<uint8_t *>(c->pool);
  v->weights = c->weights;
  v->groups = (int)(c->head_dim / c->group_size);
  v->head_dim = (int)c->head_dim;
  v->kv_heads = (int)c->kv_heads;
  v->n_pages = (int)c->n_pages;
  v->page_shift = 0;
  while ((size_t)1 << v->page_shift < c->page_size) ++v->page_shift;
  v->block_bytes = kv4_block_bytes(v->head_dim, v->groups);
  v->head_bytes = (int64_t)(c->page_size / kKv4Block) * v->block_bytes;
  v->page_bytes = v->head_bytes * v->kv_heads;
  return KS_OK;
}

// max_len null: what a row of the table holds.
int batch_of(const Kv4View &v, const int32_t *page_table, size_t stride, const int32_t *seq_lens,
             const int32_t *offsets, size_t n_seqs, size_t n_tokens, const size_t *max_len, Kv4Batch *b) {
  if (!page_table || !seq_lens) return fail(KS_ERR_INVALID_ARG, "NULL pointer");
  if (n_seqs == 0 || stride == 0) return fail(KS_ERR_INVALID_ARG, "n_seqs and the table's stride must be > 0");
  if (!offsets && n_tokens != n_seqs)
    return fail(KS_ERR_INVALID_ARG, "without token_offsets there is one token to a sequence");
  if (misaligned(page_table, 4) || misaligned(seq_lens, 4) || misaligned(offsets, 4))
    return fail(KS_ERR_INVALID_ARG, "tables, lengths and offsets must be 4-byte aligned");
  if (n_seqs > 65535 || n_tokens > kMost || stride > kMost)
    return fail(KS_ERR_UNSUPPORTED, "at most 65535 sequences, 2^31 - 1 tokens and table entries");
  const size_t holds = stride << v.page_shift;
  const size_t most = max_len ? *max_len : holds;
  if (most > holds) return fail(KS_ERR_INVALID_ARG, "max_len is more than a row of the page table holds");
  b->table = page_table;
  b->table_stride = (int64_t)stride;
  b->lens = seq_lens;
  b->offsets = offsets;
  b->n_seqs = (int)n_seqs;
  b->n_tokens = (int)n_tokens;
  b->max_len = (int)(most < kMaxLen ? most : kMaxLen);
  return KS_OK;
}

// Rows that are read may lie over each other (strides of 0 broadcast), those that are written may not.
int rows_ok(const void *p, size_t tokens, size_t token_stride, size_t heads, size_t head_stride, size_t head_dim,
            int dtype, bool written) {
  if (!p) return fail(KS_ERR_INVALID_ARG, "NULL pointer");
  if (dtype != KS_B200_DTYPE_F32 && dtype != KS_B200_DTYPE_F16 && dtype != KS_B200_DTYPE_BF16)
    return fail(KS_ERR_INVALID_ARG, "dtype must be KS_B200_DTYPE_F32, _F16 or _BF16");
  if (misaligned(p, dtype == KS_B200_DTYPE_F32 ? 4 : 2)) return fail(KS_ERR_INVALID_ARG, "misaligned tensor");
  if (token_stride > kMost || head_stride > kMost) return fail(KS_ERR_INVALID_ARG, "strides beyond 2^31 - 1 elements");
  if (written && ((tokens > 1 && token_stride < head_dim) || (heads > 1 && head_stride < head_dim)))
    return fail(KS_ERR_INVALID_ARG, "a written tensor's strides must be >= head_dim elements");
  return KS_OK;
}

// How the attention is cut.  Row tiles of 8 while the rows of a key/value head
// fit, else 16; as many CTAs as the GPU holds at once, but no more than there
// can be units of work.
Kv4Plan plan_of(const Kv4View &v, size_t group_heads, size_t n_seqs, size_t max_new, size_t max_len) {
  Kv4Plan p;
  const size_t rows = max_new * group_heads;
  const int nt = rows <= 8 ? 1 : 2;
  p.rows_tile = 8 * nt;
  p.row_tiles = (int)((rows + p.rows_tile - 1) / p.rows_tile);
  const size_t unit = kv4_unit_tokens(nt, v.groups);
  const size_t units = n_seqs * v.kv_heads * p.row_tiles * ((max_len + unit - 1) / unit);
  const size_t ctas = kPlanSms * kv4_ctas_per_sm(nt);
  static_assert(kPlanSms * kv4_ctas_per_sm(1) <= kAttnCtas && 3 * kAttnCtas <= kKv4Counters, "three counters to a CTA");
  p.ctas = (int)(units < ctas ? units : ctas);
  return p;
}

bool attention_sizes_ok(const Kv4View &v, size_t q_heads, size_t n_seqs, size_t max_new, size_t max_len) {
  return q_heads > 0 && q_heads % v.kv_heads == 0 && q_heads <= kMost && n_seqs > 0 && n_seqs <= 65535 && max_new > 0 &&
         max_len > 0 && max_new <= max_len && max_len <= kMaxLen && max_new <= kMost / q_heads &&
         // units of work, a row tile of at least 8 rows and 128 tokens each, are counted in 31 bits
         n_seqs * v.kv_heads <=
             kMost / (max_new * (q_heads / v.kv_heads) / 8 + 1) / (max_len / kv4_unit_tokens(2, 1) + 1 + kItemUnits);
}

// The counters, then two parts of every CTA.
size_t attention_bytes(const Kv4View &v, size_t group_heads, size_t n_seqs, size_t max_new, size_t max_len) {
  const Kv4Plan p = plan_of(v, group_heads, n_seqs, max_new, max_len);
  return 4 * (kKv4Counters + 2 * (size_t)p.ctas * p.rows_tile * (v.head_dim + 2));
}

}  // namespace

extern "C" size_t ks_b200_kv4_page_bytes(size_t page_size, size_t kv_heads, size_t head_dim, size_t group_size) {
  if (!shape_supported(page_size, kv_heads, head_dim, group_size)) return 0;
  return page_size / kKv4Block * kv_heads * kv4_block_bytes((int)head_dim, (int)(head_dim / group_size));
}

namespace {

int rows_call(bool append, const ks_b200_kv4_cache *cache, const int32_t *page_table, size_t page_table_stride,
              const int32_t *seq_lens, const int32_t *token_offsets, size_t n_seqs, size_t n_tokens,
              const size_t *max_len, void *k, size_t k_token_stride, size_t k_head_stride, void *v, size_t v_token_stride,
              size_t v_head_stride, int dtype, uint32_t *status, void *stream) {
  Kv4View view{};
  Kv4Batch b;
  int rc;
  if ((rc = view_of(cache, &view)) != KS_OK) return rc;
  if ((rc = batch_of(view, page_table, page_table_stride, seq_lens, token_offsets, n_seqs, n_tokens, max_len, &b)) !=
      KS_OK)
    return rc;
  if (n_tokens == 0) return KS_OK;
  if (max_len && *max_len == 0) return fail(KS_ERR_INVALID_ARG, "max_len must be > 0");
  if ((rc = rows_ok(k, n_tokens, k_token_stride, cache->kv_heads, k_head_stride, cache->head_dim, dtype, !append)) !=
          KS_OK ||
      (rc = rows_ok(v, n_tokens, v_token_stride, cache->kv_heads, v_head_stride, cache->head_dim, dtype, !append)) !=
          KS_OK)
    return rc;
  const Kv4Rows r{k, v, (int64_t)k_token_stride, (int64_t)k_head_stride, (int64_t)v_token_stride,
                  (int64_t)v_head_stride, dtype};
  const cudaError_t e = append ? launch_kv4_append(view, b, r, status, static_cast<cudaStream_t>(stream))
                               : launch_kv4_read(view, b, r, status, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? KS_OK : cuda_fail(e, "kernel launch");
}

}  // namespace

extern "C" int ks_b200_kv4_append_async(const ks_b200_kv4_cache *cache, const int32_t *page_table,
                                        size_t page_table_stride, const int32_t *seq_lens,
                                        const int32_t *token_offsets, size_t n_seqs, size_t n_tokens, const void *k,
                                        size_t k_token_stride, size_t k_head_stride, const void *v,
                                        size_t v_token_stride, size_t v_head_stride, int dtype, uint32_t *status,
                                        void *stream) {
  return rows_call(true, cache, page_table, page_table_stride, seq_lens, token_offsets, n_seqs, n_tokens, nullptr,
                   const_cast<void *>(k), k_token_stride, k_head_stride, const_cast<void *>(v), v_token_stride,
                   v_head_stride, dtype, status, stream);
}

extern "C" int ks_b200_kv4_append_bounded_async(const ks_b200_kv4_cache *cache, const int32_t *page_table,
                                                size_t page_table_stride, const int32_t *seq_lens,
                                                const int32_t *token_offsets, size_t n_seqs, size_t n_tokens,
                                                size_t max_len, const void *k, size_t k_token_stride,
                                                size_t k_head_stride, const void *v, size_t v_token_stride,
                                                size_t v_head_stride, int dtype, uint32_t *status, void *stream) {
  return rows_call(true, cache, page_table, page_table_stride, seq_lens, token_offsets, n_seqs, n_tokens, &max_len,
                   const_cast<void *>(k), k_token_stride, k_head_stride, const_cast<void *>(v), v_token_stride,
                   v_head_stride, dtype, status, stream);
}

extern "C" int ks_b200_kv4_read_async(const ks_b200_kv4_cache *cache, const int32_t *page_table,
                                      size_t page_table_stride, const int32_t *seq_lens,
                                      const int32_t *token_offsets, size_t n_seqs, size_t n_tokens, void *k,
                                      size_t k_token_stride, size_t k_head_stride, void *v, size_t v_token_stride,
                                      size_t v_head_stride, int dtype, uint32_t *status, void *stream) {
  return rows_call(false, cache, page_table, page_table_stride, seq_lens, token_offsets, n_seqs, n_tokens, nullptr,
                   k, k_token_stride, k_head_stride, v, v_token_stride, v_head_stride, dtype, status, stream);
}

extern "C" int ks_b200_kv4_read_bounded_async(const ks_b200_kv4_cache *cache, const int32_t *page_table,
                                              size_t page_table_stride, const int32_t *seq_lens,
                                              const int32_t *token_offsets, size_t n_seqs, size_t n_tokens,
                                              size_t max_len, void *k, size_t k_token_stride, size_t k_head_stride,
                                              void *v, size_t v_token_stride, size_t v_head_stride, int dtype,
                                              uint32_t *status, void *stream) {
  return rows_call(false, cache, page_table, page_table_stride, seq_lens, token_offsets, n_seqs, n_tokens, &max_len, k,
                   k_token_stride, k_head_stride, v, v_token_stride, v_head_stride, dtype, status, stream);
}

extern "C" size_t ks_b200_kv4_attention_workspace(const ks_b200_kv4_cache *cache, size_t q_heads, size_t n_seqs,
                                                  size_t n_tokens, size_t max_new, size_t max_len) {
  (void)n_tokens;
  if (max_len > kMaxLen) max_len = kMaxLen;  // as the call has it
  Kv4View v{};
  if (view_of(cache, &v) != KS_OK || !attention_sizes_ok(v, q_heads, n_seqs, max_new, max_len)) return 0;
  return attention_bytes(v, q_heads / v.kv_heads, n_seqs, max_new, max_len);
}

extern "C" int ks_b200_kv4_attention_async(const ks_b200_kv4_cache *cache, const int32_t *page_table,
                                           size_t page_table_stride, const int32_t *seq_lens,
                                           const int32_t *token_offsets, size_t n_seqs, size_t n_tokens,
                                           size_t max_new, size_t max_len, const void *q, size_t q_token_stride,
                                           size_t q_head_stride, size_t q_heads, float scale, void *out,
                                           size_t out_token_stride, size_t out_head_stride, int dtype, float *lse,
                                           int accumulate, void *workspace, size_t workspace_bytes, uint32_t *status,
                                           void *stream) {
  Kv4AttnArgs k{};
  int rc;
  if ((rc = view_of(cache, &k.c)) != KS_OK) return rc;
  if (max_new == 0 || max_len == 0 || max_new > max_len)
    return fail(KS_ERR_INVALID_ARG, "max_new and max_len must be > 0, max_new <= max_len");
  if ((rc = batch_of(k.c, page_table, page_table_stride, seq_lens, token_offsets, n_seqs, n_tokens, &max_len, &k.b)) !=
      KS_OK)
    return rc;
  if (q_heads == 0 || q_heads % k.c.kv_heads)
    return fail(KS_ERR_INVALID_ARG, "q_heads must be a positive multiple of kv_heads");
  if (!std::isfinite(scale)) return fail(KS_ERR_INVALID_ARG, "scale must be finite");
  if (n_tokens == 0) return KS_OK;
  if ((rc = rows_ok(q, n_tokens, q_token_stride, q_heads, q_head_stride, cache->head_dim, dtype, false)) != KS_OK ||
      (rc = rows_ok(out, n_tokens, out_token_stride, q_heads, out_head_stride, cache->head_dim, dtype, true)) != KS_OK)
    return rc;
  if (misaligned(lse, 4)) return fail(KS_ERR_INVALID_ARG, "lse must be 4-byte aligned");
  if (accumulate && (!lse || !cache->weights))
    return fail(KS_ERR_INVALID_ARG, "accumulating weights needs cache->weights and lse");
  if (!attention_sizes_ok(k.c, q_heads, n_seqs, max_new, (size_t)k.b.max_len))
    return fail(KS_ERR_UNSUPPORTED, "too many rows or tokens for one call");
  k.group_heads = (int)(q_heads / k.c.kv_heads);
  k.p = plan_of(k.c, k.group_heads, n_seqs, max_new, (size_t)k.b.max_len);
  const size_t need = attention_bytes(k.c, k.group_heads, n_seqs, max_new, (size_t)k.b.max_len);
  if (!workspace || misaligned(workspace, 16) || workspace_bytes < need)
    return fail(KS_ERR_WORKSPACE, "workspace smaller than ks_b200_kv4_attention_workspace, or not 16-byte aligned");
  k.a.q = q;
  k.a.out = out;
  k.a.q_token = (int64_t)q_token_stride;
  k.a.q_head = (int64_t)q_head_stride;
  k.a.out_token = (int64_t)out_token_stride;
  k.a.out_head = (int64_t)out_head_stride;
  k.a.q_heads = (int)q_heads;
  k.a.max_new = (int)max_new;
  k.a.scale = scale;
  k.a.lse = lse;
  k.a.accumulate = accumulate != 0;
  k.a.workspace = workspace;
  k.status = status;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  e = dtype == KS_B200_DTYPE_F32   ? launch_kv4_attention_f32(k, s, device)
      : dtype == KS_B200_DTYPE_F16 ? launch_kv4_attention_f16(k, s, device)
                                   : launch_kv4_attention_bf16(k, s, device);
  return e == cudaSuccess ? KS_OK : cuda_fail(e, "kernel launch");
}

// 0: more lists and weights than any memory holds, or than 64 bits count.
static size_t evict_bytes(const Kv4View &v, size_t n_seqs, size_t max_len, size_t budget) {
  if (n_seqs * v.kv_heads > ((size_t)1 << 58) / (max_len + budget)) return 0;
  return kv4_evict_workspace(v, (int)n_seqs, (int)max_len, (int)budget);
}

extern "C" size_t ks_b200_kv4_evict_workspace(const ks_b200_kv4_cache *cache, size_t n_seqs, size_t max_len,
                                              size_t budget) {
  Kv4View v{};
  if (max_len > kMost) max_len = kMost;  // the call goes by kMaxLen, which is less
  if (view_of(cache, &v) != KS_OK || n_seqs == 0 || n_seqs > 65535 || max_len == 0 || budget == 0 || budget > kMost)
    return 0;
  return evict_bytes(v, n_seqs, max_len, budget);
}

extern "C" int ks_b200_kv4_evict_async(const ks_b200_kv4_cache *cache, const int32_t *page_table,
                                       size_t page_table_stride, const int32_t *seq_lens, size_t n_seqs,
                                       size_t max_len, const int32_t *to_table, size_t to_table_stride,
                                       int32_t *to_lens, size_t budget, size_t recent, int32_t *kept, void *workspace,
                                       size_t workspace_bytes, uint32_t *status, void *stream) {
  Kv4View v{};
  Kv4Batch b;
  int rc;
  if ((rc = view_of(cache, &v)) != KS_OK) return rc;
  if (max_len == 0) return fail(KS_ERR_INVALID_ARG, "max_len must be > 0");
  if ((rc = batch_of(v, page_table, page_table_stride, seq_lens, nullptr, n_seqs, n_seqs, &max_len, &b)) != KS_OK)
    return rc;
  if (!cache->weights) return fail(KS_ERR_INVALID_ARG, "eviction needs cache->weights");
  if (!to_table || !to_lens) return fail(KS_ERR_INVALID_ARG, "NULL pointer");
  if (budget == 0 || recent > budget) return fail(KS_ERR_INVALID_ARG, "budget must be > 0 and recent <= budget");
  if (misaligned(to_table, 4) || misaligned(to_lens, 4) || misaligned(kept, 4))
    return fail(KS_ERR_INVALID_ARG, "tables and lengths must be 4-byte aligned");
  if (budget > kMost || to_table_stride > kMost) return fail(KS_ERR_UNSUPPORTED, "budget beyond 2^31 - 1");
  const size_t most = budget < (size_t)b.max_len ? budget : (size_t)b.max_len;
  if ((to_table_stride << v.page_shift) < most)
    return fail(KS_ERR_INVALID_ARG, "a row of to_table holds fewer tokens than may be kept");
  const size_t need = evict_bytes(v, n_seqs, (size_t)b.max_len, budget);
  if (need == 0) return fail(KS_ERR_UNSUPPORTED, "too many heads, tokens or kept tokens for one call");
  if (!workspace || misaligned(workspace, 16) || workspace_bytes < need)
    return fail(KS_ERR_WORKSPACE, "workspace smaller than ks_b200_kv4_evict_workspace, or not 16-byte aligned");
  const Kv4Evict e{to_table, (int64_t)to_table_stride, to_lens, kept, (int)budget, (int)recent, workspace};
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) return cuda_fail(err, "cudaGetDevice");
  err = launch_kv4_evict(v, b, e, status, static_cast<cudaStream_t>(stream), device);
  return err == cudaSuccess ? KS_OK : cuda_fail(err, "kernel launch");
}
