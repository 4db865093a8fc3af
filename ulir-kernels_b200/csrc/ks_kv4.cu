// ks_kv4.cu -- the paged 4-bit key/value cache: quantising new tokens into it,
// reading tokens back, and evicting by accumulated attention weight.  The
// layout is in ks_kv4.cuh, the attention in ks_kv4_attention.cuh.
//
// Append.  For each group of 32, 64 or 128 elements of one token and head
//   scale = max(max(v, 0) / 7, -min(v, 0) / 8) rounded to f16, kept within the
//           positive finite f16 values (1 if every element is 0)
//   code  = clamp(rne(v / scale), -8, 7)
// the rule of the Q4_0 importer with f16 scales.  Both roundings are decided
// by the exact quotient.  NaN counts as 0 and an infinity as beyond every code;
// both are reported.

#include "ks_kv4.cuh"

namespace ksb {

namespace {

// The sequence whose rows hold packed row i (-1: none), by bisection.
__device__ __forceinline__ int kv4_find_seq(const Kv4Batch &b, int i) {
  if (!b.offsets) return i < b.n_seqs ? i : -1;
  if (i < b.offsets[0] || i >= b.offsets[b.n_seqs]) return -1;
  int lo = 0, hi = b.n_seqs;  // offsets[lo] <= i < offsets[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (b.offsets[mid] <= i)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Four threads have one token's keys or values of one head, D / 4 elements
// each, which are D / 8 bytes in a row of the codes and 8 elements of every 32:
//   keys    thread t: elements 32 w + 8 t .. + 7 of each w
//   values  thread t: elements 16 i + 4 t .. + 3 of each i
// Run r of a thread is the consecutive elements that one load or store moves.
template <int D, bool V>
struct Kv4Runs {
  static constexpr int kLength = V ? 4 : 8, kRuns = D / 4 / kLength;
  static __device__ __forceinline__ int first(int t, int r) { return r * 4 * kLength + t * kLength; }
  // Where element e of a thread's D / 4 (in order of the runs) has its nibble among the thread's words.
  static __host__ __device__ constexpr int word(int e) { return V ? (e % 4 / 2) * (D / 64) + e / 4 / 4 : e / 8; }
  static __host__ __device__ constexpr int shift(int e) { return V ? (e / 4 % 4) * 8 + (e % 2) * 4 : (e % 8) * 4; }
};

template <typename T, int N>
__device__ __forceinline__ void load_run(const T *p, bool vec, float *v) {
  constexpr int kBytes = N * sizeof(T);
  if (vec) {
    T x[N];
    if constexpr (kBytes == 8)
      *reinterpret_cast<uint2 *>(x) = *reinterpret_cast<const uint2 *>(p);
    else
#pragma unroll
      for (int k = 0; k < kBytes / 16; ++k)
        reinterpret_cast<uint4 *>(x)[k] = reinterpret_cast<const uint4 *>(p)[k];
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = kv4_load(&x[k]);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = kv4_load(p + k);
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_run(T *p, bool vec, const float *v) {
  constexpr int kBytes = N * sizeof(T);
  T x[N];
#pragma unroll
  for (int k = 0; k < N; ++k) kv4_store(&x[k], v[k]);
  if (vec) {
    if constexpr (kBytes == 8)
      *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(x);
    else
#pragma unroll
      for (int k = 0; k < kBytes / 16; ++k)
        reinterpret_cast<uint4 *>(p)[k] = reinterpret_cast<const uint4 *>(x)[k];
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) p[k] = x[k];
  }
}

template <int BYTES>
__device__ __forceinline__ void copy_words(void *to, const void *from) {
  if constexpr (BYTES == 16)
    *static_cast<uint4 *>(to) = *static_cast<const uint4 *>(from);
  else
    *static_cast<uint2 *>(to) = *static_cast<const uint2 *>(from);
}

// max(hi / 7, -lo / 8) in f16, as rounded from the exact quotient: where the
// f32 quotient stands between two f16 values it may have been rounded there,
// and below 2^-14 f16's steps are wider; the division is then made in 64 bits
// (enough of them that f16 rounds as from the exact quotient).
__device__ __forceinline__ __half kv4_scale(float lo, float hi) {
  const float a = __fdiv_rn(hi, 7.0f), r = fmaxf(a, -lo * 0.125f);
  if (hi == 0.0f && lo == 0.0f) return __float2half_rn(1.0f);
  if (r >= 0x1p-14f && (__float_as_uint(a) & 0x1FFFu) != 0x1000u) return __float2half_rn(fminf(r, 65504.0f));
  const double x = fmax((double)hi / 7.0, -(double)lo * 0.125);
  return __double2half(fmin(fmax(x, 0x1p-24), 65504.0));
}

// clamp(rne(v / s), -8, 7) of the exact quotient, as a nibble in the lowest
// bits of the result; inv = 1 / s.  v * inv is within 2^-20 of v / s, so only
// next to a tie is the quotient itself needed, and where that falls on the tie
// in f32 the sign of v - x * s says on which side it lies.
__device__ __forceinline__ uint32_t kv4_code(float v, float s, float inv) {
  constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23
  float x = fminf(fmaxf(v * inv, -8.0f), 7.0f);
  float y = __fadd_rn(x, kMagic);
  if (fabsf(x - __fsub_rn(y, kMagic)) > 0.5f - 0x1p-14f) {
    x = fminf(fmaxf(__fdiv_rn(v, s), -8.5f), 7.5f);
    float q = rintf(x);
    const float low = floorf(x), r = __fmaf_rn(-x, s, v);
    if (x - low == 0.5f && r != 0.0f) q = r > 0.0f ? low + 1.0f : low;
    y = __fadd_rn(fminf(fmaxf(q, -8.0f), 7.0f), kMagic);
  }
  return __float_as_uint(y) & 15u;
}

constexpr int kRowThreads = 256, kRowTokens = 32;  // tokens of a CTA, at most

struct Kv4Place {
  int page, slot;  // page -1: the row is left out
};

// Where the CTA's rows first .. first + tokens - 1 stand in the cache, one thread each.
__device__ __forceinline__ void find_places(const Kv4View &c, const Kv4Batch &b, int first, int tokens,
                                            Kv4Place *places, uint32_t *status) {
  if ((int)threadIdx.x < tokens) {
    const int i = first + threadIdx.x;
    Kv4Place p{-1, 0};
    const int seq = kv4_find_seq(b, i);
    if (seq >= 0) {
      const Kv4Seq q = kv4_seq(b, seq, status);
      const int pos = q.len - q.n_new + (i - q.first);
      if (pos < 0 || i - q.first >= q.n_new) {  // more new tokens than the sequence has
        set_status(status, kStatusBadScale);
      } else {
        p.page = kv4_page(c, b.table, b.table_stride, seq, pos, status);
        p.slot = pos & ((1 << c.page_shift) - 1);
      }
    }
    places[threadIdx.x] = p;
  }
  __syncthreads();
}

template <typename T, int D, bool V>
__device__ __forceinline__ void append_rows(const Kv4View &c, const Kv4Place *places, int first_row, int tokens,
                                            const T *x, int64_t token_stride, int64_t head_stride, uint32_t *status) {
  using R = Kv4Runs<D, V>;
  constexpr int E = D / 4, G32 = D / 32;  // elements of a thread, groups of 32
  const int group = D / c.groups, t = threadIdx.x & 3;
  const unsigned lanes = 15u << (threadIdx.x & 28);
  bool odd = false;
  for (int i = threadIdx.x >> 2; i < tokens * c.kv_heads; i += kRowThreads / 4) {
    const int token = i / c.kv_heads, head = i - token * c.kv_heads;
    const T *src = x + (int64_t)(first_row + token) * token_stride + head * head_stride;
    const bool vec = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
    float v[E];
#pragma unroll
    for (int r = 0; r < R::kRuns; ++r) load_run<T, R::kLength>(src + R::first(t, r), vec, v + r * R::kLength);
    const Kv4Place p = places[token];
    if (p.page < 0) continue;
    // extremes of the thread's 8 elements of every 32 (e / 8 for both orders), then over the four threads
    float lo[G32], hi[G32];
#pragma unroll
    for (int g = 0; g < G32; ++g) {
      lo[g] = hi[g] = 0.0f;
#pragma unroll
      for (int e = 8 * g; e < 8 * g + 8; ++e) {
        odd |= !isfinite(v[e]);
        v[e] = isnan(v[e]) ? 0.0f : v[e];
        lo[g] = fminf(lo[g], v[e]);
        hi[g] = fmaxf(hi[g], v[e]);
      }
    }
#pragma unroll
    for (int g = 0; g < G32; ++g)
#pragma unroll
      for (int o = 1; o < 4; o *= 2) {
        lo[g] = fminf(lo[g], __shfl_xor_sync(lanes, lo[g], o));
        hi[g] = fmaxf(hi[g], __shfl_xor_sync(lanes, hi[g], o));
      }
    if (group >= 64)
#pragma unroll
      for (int g = 0; g < G32; g += 2) {
        lo[g] = lo[g + 1] = fminf(lo[g], lo[g + 1]);
        hi[g] = hi[g + 1] = fmaxf(hi[g], hi[g + 1]);
      }
    if (group == 128) {
      const float l = fminf(lo[0], lo[G32 - 1]), h = fmaxf(hi[0], hi[G32 - 1]);
#pragma unroll
      for (int g = 0; g < G32; ++g) lo[g] = l, hi[g] = h;
    }
    // thread t makes the scale of group of 32 t, all take it from there
    float l = lo[0], h = hi[0];
#pragma unroll
    for (int g = 1; g < G32; ++g)
      if (t == g) l = lo[g], h = hi[g];
    const __half mine = kv4_scale(l, h);
    const float scale = __half2float(mine), inverse = __fdiv_rn(1.0f, scale);
    uint32_t words[D / 32];
#pragma unroll
    for (int w = 0; w < D / 32; ++w) words[w] = 0;
#pragma unroll
    for (int g = 0; g < G32; ++g) {
      const float s = __shfl_sync(lanes, scale, g, 4), inv = __shfl_sync(lanes, inverse, g, 4);
#pragma unroll
      for (int e = 8 * g; e < 8 * g + 8; ++e) words[R::word(e)] |= kv4_code(v[e], s, inv) << R::shift(e);
    }
    uint8_t *half = kv4_block(c, p.page, head, p.slot) + (V ? c.block_bytes / 2 : 0);
    copy_words<D / 8>(half + (p.slot & 15) * (D / 2) + t * (D / 8), words);
    const int each = group / 32;
    if (t < G32 && t % each == 0)
      reinterpret_cast<__half *>(half + 8 * D)[(p.slot & 15) * c.groups + t / each] = mine;
    if (!V && c.weights && t == 0)
      c.weights[(((int64_t)p.page * c.kv_heads + head) << c.page_shift) + p.slot] = 0.0f;
  }
  if (odd) set_status(status, kStatusBadScale);
}

template <typename T, int D, bool V>
__device__ __forceinline__ void read_rows(const Kv4View &c, const Kv4Place *places, int first_row, int tokens, T *x,
                                          int64_t token_stride, int64_t head_stride) {
  using R = Kv4Runs<D, V>;
  const int group = D / c.groups, t = threadIdx.x & 3;
#pragma unroll 2
  for (int i = threadIdx.x >> 2; i < tokens * c.kv_heads; i += kRowThreads / 4) {
    const int token = i / c.kv_heads, head = i - token * c.kv_heads;
    const Kv4Place p = places[token];
    if (p.page < 0) continue;
    const uint8_t *half = kv4_block(c, p.page, head, p.slot) + (V ? c.block_bytes / 2 : 0);
    uint32_t words[D / 32];
    copy_words<D / 8>(words, half + (p.slot & 15) * (D / 2) + t * (D / 8));
    const __half *scales = reinterpret_cast<const __half *>(half + 8 * D) + (p.slot & 15) * c.groups;
    float s[D / 32];
#pragma unroll
    for (int g = 0; g < D / 32; ++g) s[g] = __half2float(scales[32 * g / group]);
    T *dst = x + (int64_t)(first_row + token) * token_stride + head * head_stride;
    const bool vec = (reinterpret_cast<uintptr_t>(dst) & 15) == 0;
#pragma unroll
    for (int r = 0; r < R::kRuns; ++r) {
      float v[R::kLength];
#pragma unroll
      for (int k = 0; k < R::kLength; ++k) {
        const int e = r * R::kLength + k;
        // the code in the top bits, its sign with it: an exact multiple of 2^28
        const int code = (int)(words[R::word(e)] << (28 - R::shift(e))) >> 28;
        v[k] = (float)code * s[e / 8];  // exact in f32
      }
      store_run<T, R::kLength>(dst + R::first(t, r), vec, v);
    }
  }
}

template <typename T, int D, bool READ>
__global__ void __launch_bounds__(kRowThreads) kv4_rows_kernel(Kv4View c, Kv4Batch b, Kv4Rows r, int cta_tokens,
                                                               uint32_t *status) {
  __shared__ Kv4Place places[kRowTokens];
  const int first = blockIdx.x * cta_tokens, tokens = min(cta_tokens, b.n_tokens - first);
  find_places(c, b, first, tokens, places, status);
  if constexpr (READ) {
    if (blockIdx.y == 0)
      read_rows<T, D, false>(c, places, first, tokens, static_cast<T *>(r.k), r.k_token, r.k_head);
    else
      read_rows<T, D, true>(c, places, first, tokens, static_cast<T *>(r.v), r.v_token, r.v_head);
  } else {
    if (blockIdx.y == 0)
      append_rows<T, D, false>(c, places, first, tokens, static_cast<const T *>(r.k), r.k_token, r.k_head, status);
    else
      append_rows<T, D, true>(c, places, first, tokens, static_cast<const T *>(r.v), r.v_token, r.v_head, status);
  }
}

// Tokens of a CTA: enough for its threads (four to a head) four times over,
// fewer where that would leave SMs without a CTA.
template <bool READ, int D>
cudaError_t launch_rows(const Kv4View &c, const Kv4Batch &b, const Kv4Rows &r, uint32_t *status, cudaStream_t stream) {
  int tokens = 4 * kRowThreads / 4 / c.kv_heads;
  tokens = tokens < 1 ? 1 : tokens > kRowTokens ? kRowTokens : tokens;
  while (tokens > 1 && (b.n_tokens + tokens - 1) / tokens < 148) tokens /= 2;
  const dim3 grid((unsigned)((b.n_tokens + tokens - 1) / tokens), 2);
  auto go = [&](auto zero) {
    using T = decltype(zero);
    kv4_rows_kernel<T, D, READ><<<grid, kRowThreads, 0, stream>>>(c, b, r, tokens, status);
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
