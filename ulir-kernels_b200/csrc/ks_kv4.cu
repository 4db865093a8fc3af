// ks_kv4.cu -- the paged 4-bit key/value cache: quantising new tokens into it,
// reading tokens back, and evicting by accumulated attention weight.  The
// layout is in ks_kv4.cuh, the attention in ks_kv4_attention.cuh.
//
// Append.  For each group of 32, 64 or 128 elements of one token and head
//   scale = max(max(v, 0) / 7, -min(v, 0) / 8) rounded to f16, kept within the
//           positive finite f16 values (1 if every element is 0)
//   code  = clamp(rne(v / scale), -8, 7)
// the rule of the Q4_0 importer with f16 scales.  Both roundings are decided
// by the exact quotient: the scale's by one division in 64 bits, a code's by
// the sign of v - x * scale where the f32 quotient x falls on a tie.  NaN
// counts as 0 and an infinity as beyond every code; both are reported.

#include "ks_kv4.cuh"

namespace ksb {

namespace {

// The sequence whose rows hold packed row i (-1: none).  32-ary search, the
// whole warp on one i.
__device__ __forceinline__ int kv4_find_seq(const Kv4Batch &b, int i) {
  if (!b.offsets) return i < b.n_seqs ? i : -1;
  if (i < b.offsets[0] || i >= b.offsets[b.n_seqs]) return -1;
  const int lane = threadIdx.x & 31;
  int lo = 0, n = b.n_seqs;
  while (n > 1) {
    const int step = (n + 31) >> 5;
    const int at = lane * step;
    const unsigned le = __ballot_sync(0xffffffffu, at < n && b.offsets[lo + at] <= i);
    const int c = le ? 31 - __clz(le) : 0;
    lo += c * step;
    n = min(step, n - c * step);
  }
  return lo;
}

// Eight elements of one token and head per lane.  keys: lane l of head_dim / 8
// has elements 8l .. 8l + 7, one word of the row's codes.  values: lane l =
// g * (head_dim / 64) + a has elements 16 (4a + k) + 2g + {0, 1}, k = 0..3,
// again one word.
template <int D, bool V>
__device__ __forceinline__ int kv4_element(int l, int k) {  // first element of pair k
  if constexpr (!V) return 8 * l + 2 * k;
  constexpr int A = D / 64;
  return 16 * (4 * (l % A) + k) + 2 * (l / A);
}
template <int D, bool V>
__device__ __forceinline__ int kv4_word(int l) {  // byte of that word in the row
  if constexpr (!V) return (l & 3) * (D / 8) + (l >> 2) * 4;
  return l * 4;
}

template <typename T>
__device__ __forceinline__ void load_pair(const T *p, bool vec, float &a, float &b) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      const float2 v = *reinterpret_cast<const float2 *>(p);
      a = v.x;
      b = v.y;
    } else {
      const uint32_t v = *reinterpret_cast<const uint32_t *>(p);
      const T x = reinterpret_cast<const T *>(&v)[0], y = reinterpret_cast<const T *>(&v)[1];
      a = kv4_load(&x);
      b = kv4_load(&y);
    }
  } else {
    a = kv4_load(p);
    b = kv4_load(p + 1);
  }
}

template <typename T>
__device__ __forceinline__ void store_pair(T *p, bool vec, float a, float b) {
  T x, y;
  kv4_store(&x, a);
  kv4_store(&y, b);
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float2 *>(p) = make_float2(a, b);
    } else {
      T v[2] = {x, y};
      *reinterpret_cast<uint32_t *>(p) = *reinterpret_cast<uint32_t *>(v);
    }
  } else {
    p[0] = x;
    p[1] = y;
  }
}

// max(hi / 7, -lo / 8) in f16: one division and one rounding of the exact
// quotient (a double holds enough bits of it that f16 rounds as from it).
__device__ __forceinline__ __half kv4_scale(float lo, float hi) {
  const double r = fmax((double)hi / 7.0, -(double)lo * 0.125);
  if (r == 0.0) return __float2half_rn(1.0f);
  return __double2half(fmin(fmax(r, 0x1p-24), 65504.0));
}

// clamp(rne(v / s), -8, 7) of the exact quotient, as a nibble.
__device__ __forceinline__ uint32_t kv4_code(float v, float s) {
  const float x = fminf(fmaxf(__fdiv_rn(v, s), -9.0f), 8.0f);
  float q = rintf(x);
  const float low = floorf(x);
  if (x - low == 0.5f) {  // the f32 quotient is a tie: is the exact one beside it?
    const float r = __fmaf_rn(-x, s, v);
    if (r != 0.0f) q = r > 0.0f ? low + 1.0f : low;
  }
  q = fminf(fmaxf(q, -8.0f), 7.0f);
  return (uint32_t)((int)q) & 0xFu;
}

// One CTA per (row of new tokens, keys or values); head_dim / 8 lanes per head.
template <typename T, int D, bool V>
__device__ __forceinline__ void append_rows(const Kv4View &c, const Kv4Batch &b, const T *x, int64_t token_stride,
                                            int64_t head_stride, uint32_t *status) {
  constexpr int L = D / 8, A = D / 64;
  const int i = blockIdx.x, l = threadIdx.x % L;
  const unsigned lanes = (L == 32 ? 0xffffffffu : ((1u << L) - 1u)) << ((threadIdx.x & 31) & ~(L - 1));
  const int seq = kv4_find_seq(b, i);
  if (seq < 0) return;
  const Kv4Seq q = kv4_seq(b, seq, status);
  const int pos = q.len - q.n_new + (i - q.first);
  if (pos < 0 || i - q.first >= q.n_new) {  // more new tokens than the sequence has
    set_status(status, kStatusBadScale);
    return;
  }
  const int page = kv4_page(c, b.table, b.table_stride, seq, pos, status);
  if (page < 0) return;
  const int slot = pos & ((1 << c.page_shift) - 1);
  const int group = D / c.groups;
  for (int head = threadIdx.x / L; head < c.kv_heads; head += blockDim.x / L) {
    const T *src = x + i * token_stride + head * head_stride;
    const bool vec = (reinterpret_cast<uintptr_t>(src) & (2 * sizeof(T) - 1)) == 0;
    float v[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) load_pair(src + kv4_element<D, V>(l, k), vec, v[2 * k], v[2 * k + 1]);
    bool odd = false;
    float hi[2] = {0.0f, 0.0f}, lo[2] = {0.0f, 0.0f};  // of elements 0..3 and 4..7
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      odd |= !isfinite(v[k]);
      if (isnan(v[k])) v[k] = 0.0f;
      hi[k / 4] = fmaxf(hi[k / 4], v[k]);
      lo[k / 4] = fminf(lo[k / 4], v[k]);
    }
    if (odd) set_status(status, kStatusBadScale);
    // over the lanes that share the group
    if (!V || group >= 64) {
      hi[0] = hi[1] = fmaxf(hi[0], hi[1]);
      lo[0] = lo[1] = fminf(lo[0], lo[1]);
    }
    const int first = V ? A : 1, last = V ? 4 * A : group / 16;
    auto share = [&](int o) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        hi[h] = fmaxf(hi[h], __shfl_xor_sync(lanes, hi[h], o));
        lo[h] = fminf(lo[h], __shfl_xor_sync(lanes, lo[h], o));
      }
    };
    for (int o = first; o <= last; o *= 2) share(o);
    if (V && group == 128) share(1);
    const __half s[2] = {kv4_scale(lo[0], hi[0]), kv4_scale(lo[1], hi[1])};
    const float sf[2] = {__half2float(s[0]), __half2float(s[1])};
    uint32_t word = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) word |= kv4_code(v[k], sf[k / 4]) << (4 * k);
    uint8_t *half = kv4_block(c, page, head, slot) + (V ? c.block_bytes / 2 : 0);
    *reinterpret_cast<uint32_t *>(half + (slot & 15) * (D / 2) + kv4_word<D, V>(l)) = word;
    __half *scales = reinterpret_cast<__half *>(half + 8 * D) + (slot & 15) * c.groups;
    if (!V) {
      if (l % (group / 8) == 0) scales[8 * l / group] = s[0];
    } else if (l < A) {
      if (group == 32) scales[2 * l] = s[0], scales[2 * l + 1] = s[1];
      if (group == 64) scales[l] = s[0];
      if (group == 128 && l == 0) scales[0] = s[0];
    }
    if (!V && c.weights && l == 0) c.weights[(((int64_t)page * c.kv_heads + head) << c.page_shift) + slot] = 0.0f;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_append_kernel(Kv4View c, Kv4Batch b, Kv4Rows r, uint32_t *status) {
  if (blockIdx.y == 0)
    append_rows<T, D, false>(c, b, static_cast<const T *>(r.k), r.k_token, r.k_head, status);
  else
    append_rows<T, D, true>(c, b, static_cast<const T *>(r.v), r.v_token, r.v_head, status);
}

template <typename T, int D, bool V>
__device__ __forceinline__ void read_rows(const Kv4View &c, const Kv4Batch &b, T *x, int64_t token_stride,
                                          int64_t head_stride, uint32_t *status) {
  constexpr int L = D / 8;
  const int i = blockIdx.x, l = threadIdx.x % L;
  const int seq = kv4_find_seq(b, i);
  if (seq < 0) return;
  const Kv4Seq q = kv4_seq(b, seq, status);
  const int pos = q.len - q.n_new + (i - q.first);
  if (pos < 0 || i - q.first >= q.n_new) {
    set_status(status, kStatusBadScale);
    return;
  }
  const int page = kv4_page(c, b.table, b.table_stride, seq, pos, status);
  if (page < 0) return;
  const int slot = pos & ((1 << c.page_shift) - 1);
  const int group = D / c.groups;
  for (int head = threadIdx.x / L; head < c.kv_heads; head += blockDim.x / L) {
    const uint8_t *half = kv4_block(c, page, head, slot) + (V ? c.block_bytes / 2 : 0);
    const uint32_t word =
        *reinterpret_cast<const uint32_t *>(half + (slot & 15) * (D / 2) + kv4_word<D, V>(l)) ^ 0x88888888u;
    const __half *scales = reinterpret_cast<const __half *>(half + 8 * D) + (slot & 15) * c.groups;
    T *dst = x + i * token_stride + head * head_stride;
    const bool vec = (reinterpret_cast<uintptr_t>(dst) & (2 * sizeof(T) - 1)) == 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int e = kv4_element<D, V>(l, k);
      const float s = __half2float(scales[e / group]);
      const float lo = (float)((word >> (8 * k)) & 15u) - 8.0f, hi = (float)((word >> (8 * k + 4)) & 15u) - 8.0f;
      store_pair(dst + e, vec, lo * s, hi * s);  // exact in f32
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(Kv4View c, Kv4Batch b, Kv4Rows r, uint32_t *status) {
  if (blockIdx.y == 0)
    read_rows<T, D, false>(c, b, static_cast<T *>(r.k), r.k_token, r.k_head, status);
  else
    read_rows<T, D, true>(c, b, static_cast<T *>(r.v), r.v_token, r.v_head, status);
}

template <bool READ, int D>
cudaError_t launch_rows(const Kv4View &c, const Kv4Batch &b, const Kv4Rows &r, uint32_t *status, cudaStream_t stream) {
  const dim3 grid((unsigned)b.n_tokens, 2);
  const int want = (c.kv_heads * (D / 8) + 31) / 32 * 32, threads = want < 256 ? want : 256;
  auto go = [&](auto zero) {
    using T = decltype(zero);
    if (READ)
      kv4_read_kernel<T, D><<<grid, threads, 0, stream>>>(c, b, r, status);
    else
      kv4_append_kernel<T, D><<<grid, threads, 0, stream>>>(c, b, r, status);
  };
  if (r.dtype == kF32) go(0.0f);
  if (r.dtype == kF16) go(__half());
  if (r.dtype == kBF16) go(__nv_bfloat16());
  return cudaGetLastError();
}

// ------------------------------------------------------------------ eviction
// Of a sequence of len > budget tokens each head keeps the newest `recent` and,
// of the older ones, the budget - recent with the largest accumulated weight,
// the lower position first among equal ones (a NaN weight is below all).  A
// first kernel, one CTA per (sequence, head), finds the smallest weight that
// is kept by four 8-bit passes over the weights as order-preserving integers
// and lists the positions in order; a second moves the tokens.  The first
// writes only the workspace, so to_lens may be the sequences' own lengths.
constexpr int kSelectThreads = 512;

struct EvictWorkspace {
  uint32_t *keys;  // [seq][head][max_len]
  int32_t *list;   // [seq][head][budget]
  int32_t *count;  // [seq]
};

__host__ __device__ inline EvictWorkspace evict_workspace(void *w, int64_t rows, int64_t max_len, int64_t budget) {
  EvictWorkspace e;
  e.keys = static_cast<uint32_t *>(w);
  e.list = reinterpret_cast<int32_t *>(e.keys + rows * max_len);
  e.count = e.list + rows * budget;
  return e;
}

// Larger weights have larger keys; NaN has key 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (isnan(w)) return 0u;
  const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Exclusive sums over the CTA of two counts below 2^16 each, packed.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *total, uint32_t *shared) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t sum = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const uint32_t n = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += n;
  }
  __syncthreads();
  if (lane == 31) shared[warp] = sum;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int k = 0; k < kSelectThreads / 32; ++k) {
    if (k < warp) before += shared[k];
    all += shared[k];
  }
  *total = all;
  return before + sum - v;
}

__global__ void __launch_bounds__(kSelectThreads) kv4_select_kernel(Kv4View c, Kv4Batch b, Kv4Evict e,
                                                                    uint32_t *status) {
  __shared__ uint32_t hist[256], scan[kSelectThreads / 32], found[2];
  const int head = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x;
  int len = b.lens[seq];
  if (len < 0 || len > b.max_len) {
    if (tid == 0) set_status(status, kStatusBadScale);
    len = 0;
  }
  const EvictWorkspace ws =
      evict_workspace(e.workspace, (int64_t)b.n_seqs * c.kv_heads, b.max_len, e.budget);
  const int64_t row = (int64_t)seq * c.kv_heads + head;
  uint32_t *keys = ws.keys + row * b.max_len;
  int32_t *list = ws.list + row * e.budget;
  const int count = min(len, e.budget);
  if (head == 0 && tid == 0) ws.count[seq] = count;
  if (len <= e.budget) {
    for (int i = tid; i < len; i += kSelectThreads) list[i] = i;
    return;
  }
  const int old = len - e.recent, want = e.budget - e.recent;
  for (int i = tid; i < e.recent; i += kSelectThreads) list[want + i] = old + i;
  if (want == 0) return;
  for (int i = tid; i < old; i += kSelectThreads) {
    const int page = kv4_page(c, b.table, b.table_stride, seq, i, status);
    const int slot = i & ((1 << c.page_shift) - 1);
    keys[i] = page < 0 ? 0u : weight_key(c.weights[(((int64_t)page * c.kv_heads + head) << c.page_shift) + slot]);
  }
  // the want-th largest key, byte by byte: `rank` of the keys with this prefix are still wanted
  uint32_t prefix = 0;
  int rank = want;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kSelectThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < old; i += kSelectThreads) {
      const uint32_t k = keys[i];
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid < 32) {  // lane l has bins 255 - 8l .. 248 - 8l
      uint32_t n[8], sum = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += n[k] = hist[255 - 8 * tid - k];
      uint32_t upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const uint32_t m = __shfl_up_sync(0xffffffffu, upto, o);
        if (tid >= o) upto += m;
      }
      uint32_t before = upto - sum;
      if (before < (uint32_t)rank && upto >= (uint32_t)rank) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (before < (uint32_t)rank && before + n[k] >= (uint32_t)rank) {
            found[0] = 255u - 8 * tid - k;
            found[1] = before;
          }
          before += n[k];
        }
      }
    }
    __syncthreads();
    prefix |= found[0] << shift;
    rank -= (int)found[1];
  }
  // `rank` tokens with exactly that key are kept, those of the lowest positions
  constexpr int kEach = 8;
  int above = 0, equal = 0;
  for (int base = 0; base < old; base += kSelectThreads * kEach) {
    uint32_t k[kEach], mine = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = base + tid * kEach + j;
      k[j] = i < old ? keys[i] : 0u;
      if (i < old) mine += k[j] > prefix ? 1u : k[j] == prefix ? 65536u : 0u;
    }
    uint32_t all;
    const uint32_t at = block_scan(mine, &all, scan);
    int a = above + (int)(at & 65535u), q = equal + (int)(at >> 16);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = base + tid * kEach + j;
      if (i >= old) break;
      if (k[j] > prefix) {
        list[a + min(q, rank)] = i;
        ++a;
      } else if (k[j] == prefix) {
        if (q < rank) list[a + q] = i;
        ++q;
      }
    }
    above += (int)(all & 65535u);
    equal += (int)(all >> 16);
  }
}

// Moves tokens, eight lanes each: the codes in 16-byte pieces (head_dim / 32
// of keys and as many of values, a lane each), the scales and the weight by
// three of the lanes.
constexpr int kMoveThreads = 256, kMoveTokens = kMoveThreads / 8;

__global__ void __launch_bounds__(kMoveThreads) kv4_move_kernel(Kv4View c, Kv4Batch b, Kv4Evict e, uint32_t *status) {
  const int head = blockIdx.y, seq = blockIdx.z, l = threadIdx.x & 7;
  const int to = blockIdx.x * kMoveTokens + (threadIdx.x >> 3);
  const EvictWorkspace ws =
      evict_workspace(e.workspace, (int64_t)b.n_seqs * c.kv_heads, b.max_len, e.budget);
  const int count = ws.count[seq];
  if (blockIdx.x == 0 && head == 0 && threadIdx.x == 0) e.to_lens[seq] = count;
  if (to >= count) return;
  const int64_t row = ((int64_t)seq * c.kv_heads + head) * e.budget;
  const int from = ws.list[row + to];
  if (e.kept && l == 0) e.kept[row + to] = from;
  const int src = kv4_page(c, b.table, b.table_stride, seq, from, status);
  const int dst = kv4_page(c, e.to_table, e.to_stride, seq, to, status);
  if (src < 0 || dst < 0) return;
  const int mask = (1 << c.page_shift) - 1, s = from & mask, t = to & mask;
  const uint8_t *sb = kv4_block(c, src, head, s);
  uint8_t *db = kv4_block(c, dst, head, t);
  const int codes = c.head_dim / 2, half = c.block_bytes / 2, pieces = codes / 16;
  if (l < 2 * pieces) {
    const int o = (l < pieces ? 0 : half) + (l % pieces) * 16;
    *reinterpret_cast<uint4 *>(db + o + (t & 15) * codes) =
        *reinterpret_cast<const uint4 *>(sb + o + (s & 15) * codes);
  }
  if (l < 2) {
    const int o = l * half + 16 * codes;
    const __half *ss = reinterpret_cast<const __half *>(sb + o) + (s & 15) * c.groups;
    __half *ds = reinterpret_cast<__half *>(db + o) + (t & 15) * c.groups;
    for (int g = 0; g < c.groups; ++g) ds[g] = ss[g];
  }
  if (l == 2) {
    c.weights[(((int64_t)dst * c.kv_heads + head) << c.page_shift) + t] =
        c.weights[(((int64_t)src * c.kv_heads + head) << c.page_shift) + s];
  }
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4View &c, const Kv4Batch &b, const Kv4Rows &r, uint32_t *status,
                              cudaStream_t stream) {
  return c.head_dim == 128 ? launch_rows<false, 128>(c, b, r, status, stream)
                           : launch_rows<false, 64>(c, b, r, status, stream);
}

cudaError_t launch_kv4_read(const Kv4View &c, const Kv4Batch &b, const Kv4Rows &r, uint32_t *status,
                            cudaStream_t stream) {
  return c.head_dim == 128 ? launch_rows<true, 128>(c, b, r, status, stream)
                           : launch_rows<true, 64>(c, b, r, status, stream);
}

size_t kv4_evict_workspace(const Kv4View &c, int n_seqs, int max_len, int budget) {
  const size_t rows = (size_t)n_seqs * c.kv_heads;
  return (rows * ((size_t)max_len + budget) + n_seqs) * 4;
}

cudaError_t launch_kv4_evict(const Kv4View &c, const Kv4Batch &b, const Kv4Evict &e, uint32_t *status,
                             cudaStream_t stream) {
  kv4_select_kernel<<<dim3((unsigned)c.kv_heads, (unsigned)b.n_seqs), kSelectThreads, 0, stream>>>(c, b, e, status);
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  const int most = e.budget < b.max_len ? e.budget : b.max_len;
  const dim3 grid((unsigned)((most + kMoveTokens - 1) / kMoveTokens), (unsigned)c.kv_heads, (unsigned)b.n_seqs);
  kv4_move_kernel<<<grid, kMoveThreads, 0, stream>>>(c, b, e, status);
  return cudaGetLastError();
}

}  // namespace ksb
