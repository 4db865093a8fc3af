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

#include <atomic>

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

// One 32-bit word of a tensor's elements as f32, and back.
__device__ __forceinline__ void unpack_word(uint32_t w, float *v, const float *) { v[0] = __uint_as_float(w); }
__device__ __forceinline__ void unpack_word(uint32_t w, float *v, const __half *) {
  const float2 f = unpack_f16(w);
  v[0] = f.x, v[1] = f.y;
}
__device__ __forceinline__ void unpack_word(uint32_t w, float *v, const __nv_bfloat16 *) {
  v[0] = __uint_as_float(w << 16), v[1] = __uint_as_float(w & 0xFFFF0000u);
}
__device__ __forceinline__ uint32_t pack_word(const float *v, const float *) { return __float_as_uint(v[0]); }
__device__ __forceinline__ uint32_t pack_word(const float *v, const __half *) { return pack_f16(v[0], v[1]); }
__device__ __forceinline__ uint32_t pack_word(const float *v, const __nv_bfloat16 *) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(v[0], v[1]);
  return *reinterpret_cast<const uint32_t *>(&b);
}

template <typename T, int N, bool VEC>
__device__ __forceinline__ void load_run(const T *p, float *v) {
  constexpr int kWords = N * sizeof(T) / 4, kPer = 4 / sizeof(T);
  if constexpr (VEC) {
    uint32_t w[kWords];
    if constexpr (kWords == 2) {
      const uint2 x = *reinterpret_cast<const uint2 *>(p);
      w[0] = x.x, w[1] = x.y;
    } else {
#pragma unroll
      for (int k = 0; k < kWords; k += 4) {
        const uint4 x = reinterpret_cast<const uint4 *>(p)[k / 4];
        w[k] = x.x, w[k + 1] = x.y, w[k + 2] = x.z, w[k + 3] = x.w;
      }
    }
#pragma unroll
    for (int k = 0; k < kWords; ++k) unpack_word(w[k], v + k * kPer, p);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = kv4_load(p + k);
  }
}

template <typename T, int N, bool VEC>
__device__ __forceinline__ void store_run(T *p, const float *v) {
  constexpr int kWords = N * sizeof(T) / 4, kPer = 4 / sizeof(T);
  if constexpr (VEC) {
    uint32_t w[kWords];
#pragma unroll
    for (int k = 0; k < kWords; ++k) w[k] = pack_word(v + k * kPer, p);
    if constexpr (kWords == 2)
      *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
    else
#pragma unroll
      for (int k = 0; k < kWords; k += 4)
        reinterpret_cast<uint4 *>(p)[k / 4] = make_uint4(w[k], w[k + 1], w[k + 2], w[k + 3]);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) kv4_store(p + k, v[k]);
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

// clamp(rne(v / s), -8, 7) of the exact quotient: where the f32 quotient falls
// on a tie, the sign of v - x * s says on which side the exact one lies.
__device__ __forceinline__ float kv4_code(float v, float s) {
  const float x = fminf(fmaxf(__fdiv_rn(v, s), -8.5f), 7.5f), low = floorf(x), r = __fmaf_rn(-x, s, v);
  float q = rintf(x);
  if (x - low == 0.5f && r != 0.0f) q = r > 0.0f ? low + 1.0f : low;
  return fminf(fmaxf(q, -8.0f), 7.0f);
}

constexpr int kRowThreads = 256, kRowTokens = 256;  // tokens of a CTA, at most

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
  // One CTA looks at every sequence, so that those without a row are reported too: from the last thread down, as the
  // first ones have the lookups of short calls.
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int s = kRowThreads - 1 - (int)threadIdx.x; s < b.n_seqs; s += kRowThreads) kv4_seq(b, s, status);
  __syncthreads();
}

// Of x[0 .. 2N), the lane keeps the extremes of its own and its partner's (lane ^ o) upper or lower N, in x[0 .. N).
template <int N, bool MAX, int SIZE>
__device__ __forceinline__ void hand_over(float (&x)[SIZE], int o, bool upper) {
#pragma unroll
  for (int g = 0; g < N; ++g) {
    const float give = upper ? x[g] : x[g + N], keep = upper ? x[g + N] : x[g];
    const float got = __shfl_xor_sync(0xffffffffu, give, o);
    x[g] = MAX ? fmaxf(keep, got) : fminf(keep, got);
  }
}

// Goes over the rows (token, head) of a CTA, kRowThreads / 4 at a time, without dividing each time.
struct RowWalk {
  int token, head, step_token, step_head, heads;
  __device__ RowWalk(int row, int kv_heads) : heads(kv_heads) {
    token = row / heads;
    head = row - token * heads;
    step_token = kRowThreads / 4 / heads;
    step_head = kRowThreads / 4 - step_token * heads;
  }
  __device__ __forceinline__ void next() {
    token += step_token;
    head += step_head;
    if (head >= heads) {
      head -= heads;
      ++token;
    }
  }
};

template <typename T, int D, int NG, bool V>
__device__ __forceinline__ void append_rows(const Kv4View &c, const Kv4Place *places, int first_row, int tokens,
                                            const T *x, int64_t token_stride, int64_t head_stride, uint32_t *status) {
  using R = Kv4Runs<D, V>;
  constexpr int E = D / 4, G32 = D / 32;  // elements of a thread, groups of 32
  constexpr float kMagic = 12582912.0f;   // 1.5 * 2^23: adding it rounds to an integer, ties to even
  constexpr int group = D / NG;
  const int t = threadIdx.x & 3;
  bool odd = false;
  // whole warps go on while one of their rows is there
  for (RowWalk at(threadIdx.x >> 2, c.kv_heads); __any_sync(0xffffffffu, at.token < tokens); at.next()) {
    const int token = at.token, head = at.head;
    const Kv4Place p = token < tokens ? places[token] : Kv4Place{-1, 0};
    const T *src = x + ((int64_t)first_row + token) * token_stride + head * head_stride;
    float v[E];
    if (p.page < 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = 0.0f;
    } else if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
#pragma unroll
      for (int r = 0; r < R::kRuns; ++r) load_run<T, R::kLength, true>(src + R::first(t, r), v + r * R::kLength);
    } else {
#pragma unroll
      for (int r = 0; r < R::kRuns; ++r) load_run<T, R::kLength, false>(src + R::first(t, r), v + r * R::kLength);
    }
    // extremes of the thread's 8 elements of every 32 (e / 8 for both orders; NaN is passed over)
    float lo[G32], hi[G32], zero = 0.0f;
#pragma unroll
    for (int g = 0; g < G32; ++g) {
      lo[g] = hi[g] = 0.0f;
#pragma unroll
      for (int e = 8 * g; e < 8 * g + 8; ++e) {
        zero = fmaf(v[e], 0.0f, zero);  // NaN if one is not finite
        lo[g] = fminf(lo[g], v[e]);
        hi[g] = fmaxf(hi[g], v[e]);
      }
    }
    // over the four threads: each step hands the other half of the groups to the partner, thread t ends with group of
    // 32 t (t % 2 where there are two), makes the scale of its group and all take it from there
    if constexpr (G32 == 4) {
      hand_over<2, false>(lo, 2, t & 2);
      hand_over<2, true>(hi, 2, t & 2);
    } else {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        lo[g] = fminf(lo[g], __shfl_xor_sync(0xffffffffu, lo[g], 2));
        hi[g] = fmaxf(hi[g], __shfl_xor_sync(0xffffffffu, hi[g], 2));
      }
    }
    hand_over<1, false>(lo, 1, t & 1);
    hand_over<1, true>(hi, 1, t & 1);
    float l = lo[0], h = hi[0];
#pragma unroll
    for (int o = 1; 32 * o < group; o *= 2) {
      l = fminf(l, __shfl_xor_sync(0xffffffffu, l, o));
      h = fmaxf(h, __shfl_xor_sync(0xffffffffu, h, o));
    }
    const __half mine = kv4_scale(l, h);
    const float scale = __half2float(mine), inverse = __fdiv_rn(1.0f, scale);
    // Codes are q = rne(v * (1 / s)) with 1 / s in two parts: the f32 nearest to a quotient that is off by no more than
    // 2^-45, so a quotient on a tie gives the tie.  One beside a tie gives it too only if that is within 2^-24, which is
    // ruled out where v has 11 bits (s has, so they differ by 2^-16 at least); for f32 the remainder v - q * s (exact)
    // then decides.  Held scales (v / s may leave [-8.5, 7.5]) and values that are not finite go through the quotient.
    // A word is q + 8 in base 16, exact in f32 four codes at a time.
    const bool plain = zero == 0.0f;
    odd |= !plain;
    float sums[D / 32][2];
#pragma unroll
    for (int w = 0; w < D / 32; ++w) sums[w][0] = sums[w][1] = 8388608.0f + 34952.0f;  // 2^23 + 0x8888
#pragma unroll
    for (int g = 0; g < G32; ++g) {
      const float s = __shfl_sync(0xffffffffu, scale, g, 4), inv = __shfl_sync(0xffffffffu, inverse, g, 4);
      const float rest = __fmaf_rn(-s, inv, 1.0f) * inv;
      float q[8], off = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = __fmaf_rn(v[8 * g + e], inv, v[8 * g + e] * rest);
        q[e] = __fsub_rn(__fadd_rn(y, kMagic), kMagic);
        if (sizeof(T) == 4) off = fmaxf(off, fabsf(y - q[e]));
      }
      if (!plain || s >= 65504.0f || s < 0x1p-14f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = kv4_code(isnan(v[8 * g + e]) ? 0.0f : v[8 * g + e], s);
      } else if (sizeof(T) == 4 && off >= 0.5f - 0x1p-20f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float r = __fmaf_rn(-q[e], s, v[8 * g + e]), half = 0.5f * s;
          const bool is_odd = __float_as_uint(q[e] + kMagic) & 1u;
          if (fabsf(r) > half || (fabsf(r) == half && is_odd)) q[e] += copysignf(1.0f, r);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int n = R::shift(8 * g + e) / 4;
        constexpr float kBase[4] = {1.0f, 16.0f, 256.0f, 4096.0f};
        float &sum = sums[R::word(8 * g + e)][n / 4];
        sum = fmaf(q[e], kBase[n % 4], sum);
      }
    }
    uint32_t words[D / 32];
#pragma unroll
    for (int w = 0; w < D / 32; ++w)
      words[w] = prmt(__float_as_uint(sums[w][0]), __float_as_uint(sums[w][1]), 0x5410) ^ 0x88888888u;
    if (p.page < 0) continue;
    uint8_t *half = kv4_block(c, p.page, head, p.slot) + (V ? c.block_bytes / 2 : 0);
    copy_words<D / 8>(half + (p.slot & 15) * (D / 2) + t * (D / 8), words);
    constexpr int each = group / 32;
    if (t < G32 && t % each == 0) reinterpret_cast<__half *>(half + 8 * D)[(p.slot & 15) * NG + t / each] = mine;
    if (!V && c.weights && t == 0)
      c.weights[(((int64_t)p.page * c.kv_heads + head) << c.page_shift) + p.slot] = 0.0f;
  }
  if (odd) set_status(status, kStatusBadScale);
}

// The 8 codes of a word, in order of the nibbles.
__device__ __forceinline__ void word_codes(uint32_t w, float (&f)[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    // 1024 + (code + 8), as f16, of nibbles k and k + 4
    const uint32_t u = and_xor(w >> (4 * k), 0x000F000Fu, 0x64086408u);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&u), __floats2half2_rn(1032.0f, 1032.0f));
    const float2 x = __half22float2(h);
    f[k] = x.x;
    f[k + 4] = x.y;
  }
}

template <typename T, int D, int NG, bool V>
__device__ __forceinline__ void read_rows(const Kv4View &c, const Kv4Place *places, int first_row, int tokens, T *x,
                                          int64_t token_stride, int64_t head_stride) {
  using R = Kv4Runs<D, V>;
  const int t = threadIdx.x & 3;
  constexpr int N = 2;  // rows whose loads are under way together
  for (RowWalk at(threadIdx.x >> 2, c.kv_heads); at.token < tokens;) {
    uint32_t words[N][D / 32];
    float s[N][D / 32];
    T *dst[N];
#pragma unroll
    for (int n = 0; n < N; ++n, at.next()) {
      const int token = at.token, head = at.head;
      dst[n] = nullptr;
      if (token >= tokens || places[token].page < 0) continue;
      const Kv4Place p = places[token];
      const uint8_t *half = kv4_block(c, p.page, head, p.slot) + (V ? c.block_bytes / 2 : 0);
      copy_words<D / 8>(words[n], half + (p.slot & 15) * (D / 2) + t * (D / 8));
      float sc[NG];
      load_scales<NG>(half + 8 * D + (p.slot & 15) * 2 * NG, sc);
#pragma unroll
      for (int g = 0; g < D / 32; ++g) s[n][g] = sc[g * NG / (D / 32)];
      dst[n] = x + ((int64_t)first_row + token) * token_stride + head * head_stride;
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (!dst[n]) continue;
      float f[D / 32][8];
#pragma unroll
      for (int w = 0; w < D / 32; ++w) word_codes(words[n][w], f[w]);
      const bool vec = (reinterpret_cast<uintptr_t>(dst[n]) & 15) == 0;
      float v[D / 4];
#pragma unroll
      for (int e = 0; e < D / 4; ++e) v[e] = f[R::word(e)][R::shift(e) / 4] * s[n][e / 8];  // exact in f32
      if (vec) {
#pragma unroll
        for (int r = 0; r < R::kRuns; ++r) store_run<T, R::kLength, true>(dst[n] + R::first(t, r), v + r * R::kLength);
      } else {
#pragma unroll
        for (int r = 0; r < R::kRuns; ++r) store_run<T, R::kLength, false>(dst[n] + R::first(t, r), v + r * R::kLength);
      }
    }
  }
}

// One pass over what is read and written, with nothing shared between tokens:
// four threads to a token's row, so that a warp's 16-byte pieces fill whole
// sectors on both sides, keys and values in CTAs of their own.  19880 tokens,
// 8 heads of 128, bf16, groups of 64: append 30 us (3.4 TB/s; issued in 0.64 of the
// cycles, the largest wait is for a row's loads, of which a thread has one row's
// under way; quotients by a reciprocal, with one branch on alignment to a row, took
// 8 us off), read 21 us (4.9 TB/s, two rows under way); 58000 tokens, f16: read
// 57 us, 5.3 TB/s.
// 64 tokens take 4 us, the latency of the lookup and of one row.
template <typename T, int D, int NG, bool READ>
__global__ void __launch_bounds__(kRowThreads, READ ? 4 : 3) kv4_rows_kernel(Kv4View c, Kv4Batch b, Kv4Rows r,
                                                                              int cta_tokens, uint32_t *status) {
  __shared__ Kv4Place places[kRowTokens];
  const int first = blockIdx.x * cta_tokens, tokens = min(cta_tokens, b.n_tokens - first);
  kv4_begin();
  find_places(c, b, first, tokens, places, status);
  if constexpr (READ) {
    if (blockIdx.y == 0)
      read_rows<T, D, NG, false>(c, places, first, tokens, static_cast<T *>(r.k), r.k_token, r.k_head);
    else
      read_rows<T, D, NG, true>(c, places, first, tokens, static_cast<T *>(r.v), r.v_token, r.v_head);
  } else {
    if (blockIdx.y == 0)
      append_rows<T, D, NG, false>(c, places, first, tokens, static_cast<const T *>(r.k), r.k_token, r.k_head, status);
    else
      append_rows<T, D, NG, true>(c, places, first, tokens, static_cast<const T *>(r.v), r.v_token, r.v_head, status);
  }
}

// Tokens of a CTA: what gives all that the GPU holds at once the same number, so
// that the lookup is done once (19880 tokens: append 29.7 us, read 20.7; with
// CTAs of 32 tokens, one after the other, 30.2 and 22.9; 58000 tokens: read 57
// and 61), in whole turns of its threads (four to a head); fewer where that
// would leave SMs without a CTA.
template <bool READ, int D, int NG>
cudaError_t launch_rows(const Kv4View &c, const Kv4Batch &b, const Kv4Rows &r, uint32_t *status, cudaStream_t stream) {
  constexpr int kSlots = 148 * (READ ? 4 : 3) / 2;  // of keys, and of values
  const int turn = c.kv_heads < kRowThreads / 4 ? kRowThreads / 4 / c.kv_heads : 1;
  const int waves = (b.n_tokens - 1) / (kSlots * kRowTokens) + 1;
  int tokens = (b.n_tokens - 1) / (kSlots * waves) + 1;
  tokens = (tokens + turn - 1) / turn * turn;
  tokens = tokens > kRowTokens ? kRowTokens : tokens;
  auto ctas = [&](int each) { return (unsigned)((b.n_tokens - 1) / each) + 1; };
  while (tokens > 1 && ctas(tokens) < 148) tokens /= 2;
  const dim3 grid(ctas(tokens), 2);
  auto *kernel = r.dtype == kF32   ? kv4_rows_kernel<float, D, NG, READ>
                 : r.dtype == kF16 ? kv4_rows_kernel<__half, D, NG, READ>
                                   : kv4_rows_kernel<__nv_bfloat16, D, NG, READ>;
  return kv4_launch(kernel, grid, kRowThreads, 0, stream, c, b, r, tokens, status);
}

template <bool READ>
cudaError_t launch_rows(const Kv4View &c, const Kv4Batch &b, const Kv4Rows &r, uint32_t *status, cudaStream_t stream) {
  if (c.head_dim == 64)
    return c.groups == 1 ? launch_rows<READ, 64, 1>(c, b, r, status, stream)
                         : launch_rows<READ, 64, 2>(c, b, r, status, stream);
  return c.groups == 1   ? launch_rows<READ, 128, 1>(c, b, r, status, stream)
         : c.groups == 2 ? launch_rows<READ, 128, 2>(c, b, r, status, stream)
                         : launch_rows<READ, 128, 4>(c, b, r, status, stream);
}

// ------------------------------------------------------------------ eviction
// Of a sequence of len > budget tokens each head keeps the newest `recent` and,
// of the older ones, the budget - recent with the largest accumulated weight,
// the lower position first among equal ones (a NaN weight is below all).  A
// first kernel, one CTA per (sequence, head), finds the smallest weight that
// is kept by three passes (11, 11 and 10 bits) over the weights as
// order-preserving integers and lists the positions in order; a second moves the tokens.  The first
// writes only the workspace, so to_lens may be the sequences' own lengths.
// 32 sequences of up to 8192 tokens to 2048, 8 heads of 128, groups of 64: 45
// us, 17 of them the search (each CTA's passes follow one another: latency) and
// 28 the move (130 MB, 4.7 TB/s).  One sequence of 1100: 10 us, latency.
constexpr int kSelectThreads = 1024;
constexpr int kSelectShared = 200 * 1024;  // keys that fit stay in shared memory

// Behind the words that the attention wants to be 0, so that one workspace serves both in turn.
struct EvictWorkspace {
  uint32_t *keys;  // [seq][head][max_len]
  int32_t *list;   // [seq][head][budget]
  int32_t *count;  // [seq]
};

__host__ __device__ inline EvictWorkspace evict_workspace(void *w, int64_t rows, int64_t max_len, int64_t budget) {
  EvictWorkspace e;
  e.keys = static_cast<uint32_t *>(w) + kKv4Counters;
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

// Exclusive sums over the CTA (also of two counts below 2^16 each, packed).
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *total, uint32_t *shared) {
  constexpr int kWarps = kSelectThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto warp_scan = [&](uint32_t x) {
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const uint32_t n = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += n;
    }
    return x;
  };
  const uint32_t sum = warp_scan(v);
  __syncthreads();
  if (lane == 31) shared[warp] = sum;
  __syncthreads();
  if (warp == 0) shared[lane] = warp_scan(lane < kWarps ? shared[lane] : 0u);
  __syncthreads();
  *total = shared[kWarps - 1];
  return (warp ? shared[warp - 1] : 0u) + sum - v;
}

template <bool SHARED>
__global__ void __launch_bounds__(kSelectThreads) kv4_select_kernel(Kv4View c, Kv4Batch b, Kv4Evict e,
                                                                    uint32_t *status) {
  constexpr int kBins = 2048;
  __shared__ uint32_t hist[kBins], scan[32], found[2];
  extern __shared__ uint32_t shared_keys[];
  const int head = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x;
  kv4_begin();
  int len = b.lens[seq];
  if (len < 0 || len > b.max_len) {
    if (tid == 0) set_status(status, kStatusBadScale);
    len = 0;
  }
  const EvictWorkspace ws =
      evict_workspace(e.workspace, (int64_t)b.n_seqs * c.kv_heads, b.max_len, e.budget);
  const int64_t row = (int64_t)seq * c.kv_heads + head;
  uint32_t *keys = SHARED ? shared_keys : ws.keys + row * b.max_len;
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
  for (int i = tid; i < kBins; i += kSelectThreads) hist[i] = 0;
  __syncthreads();
#pragma unroll 4
  for (int i = tid; i < old; i += kSelectThreads) {
    const int page = kv4_page(c, b.table, b.table_stride, seq, i, status);
    const int slot = i & ((1 << c.page_shift) - 1);
    const uint32_t k =
        page < 0 ? 0u : weight_key(c.weights[(((int64_t)page * c.kv_heads + head) << c.page_shift) + slot]);
    keys[i] = k;
    atomicAdd(&hist[k >> 21], 1u);
  }
  // the want-th largest key, digit by digit: `rank` of the keys with this prefix are still wanted
  uint32_t prefix = 0;
  int rank = want;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : kBins;
    if (pass > 0) {
      for (int i = tid; i < bins; i += kSelectThreads) hist[i] = 0;
      __syncthreads();
      const int known = pass == 1 ? 21 : 10;
      for (int i = tid; i < old; i += kSelectThreads) {
        const uint32_t k = keys[i];
        if (k >> known == prefix >> known) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1u);
      }
    }
    __syncthreads();
    // thread t has the bins bins - 1 - 2t and below it, from the largest down
    const int top = bins - 1 - 2 * tid;
    const uint32_t n0 = top >= 0 ? hist[top] : 0u, n1 = top >= 1 ? hist[top - 1] : 0u;
    uint32_t all;
    const uint32_t before = block_scan(n0 + n1, &all, scan);
    if (before < (uint32_t)rank && before + n0 + n1 >= (uint32_t)rank) {
      const bool second = before + n0 < (uint32_t)rank;
      found[0] = (uint32_t)(top - second);
      found[1] = before + (second ? n0 : 0u);
    }
    __syncthreads();
    prefix |= found[0] << shift;
    rank -= (int)found[1];
    __syncthreads();
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

// Moves 128 tokens of a head: a thread each for where they are and go, their
// weight and list entry, then eight lanes to a token for the codes in 16-byte
// pieces (head_dim / 32 of keys and as many of values) and the scales, all of a
// thread's loads before its stores.
constexpr int kMoveThreads = 256, kMoveTokens = 128;

template <int D>
__global__ void __launch_bounds__(kMoveThreads) kv4_move_kernel(Kv4View c, Kv4Batch b, Kv4Evict e, uint32_t *status) {
  __shared__ uint8_t *rows[kMoveTokens][2];  // source and destination: the token's row of key codes
  __shared__ int slots[kMoveTokens];         // their slots in the blocks, 16 * source + destination; -1: none
  const int head = blockIdx.y, seq = blockIdx.z, tid = threadIdx.x, base = blockIdx.x * kMoveTokens;
  const EvictWorkspace ws =
      evict_workspace(e.workspace, (int64_t)b.n_seqs * c.kv_heads, b.max_len, e.budget);
  kv4_begin();
  const int count = ws.count[seq];
  if (blockIdx.x == 0 && head == 0 && tid == 0) e.to_lens[seq] = count;
  if (base >= count) return;
  if (tid < kMoveTokens) {
    int slot = -1;
    const int to = base + tid;
    if (to < count) {
      const int64_t row = ((int64_t)seq * c.kv_heads + head) * e.budget;
      const int from = ws.list[row + to];
      if (e.kept) e.kept[row + to] = from;
      const int src = kv4_page(c, b.table, b.table_stride, seq, from, status);
      const int dst = kv4_page(c, e.to_table, e.to_stride, seq, to, status);
      if (src >= 0 && dst >= 0) {
        const int mask = (1 << c.page_shift) - 1, s = from & mask, t = to & mask;
        rows[tid][0] = kv4_block(c, src, head, s) + (s & 15) * (D / 2);
        rows[tid][1] = kv4_block(c, dst, head, t) + (t & 15) * (D / 2);
        slot = (s & 15) * 16 + (t & 15);
        c.weights[(((int64_t)dst * c.kv_heads + head) << c.page_shift) + t] =
            c.weights[(((int64_t)src * c.kv_heads + head) << c.page_shift) + s];
      }
    }
    slots[tid] = slot;
  }
  __syncthreads();
  constexpr int kPieces = D / 32, kEach = kMoveTokens * 8 / kMoveThreads;
  const int l = tid & 7, half = c.block_bytes / 2, piece = (l < kPieces ? 0 : half) + (l % kPieces) * 16;
  const bool code = l < 2 * kPieces;
  uint4 data[kEach];
  uint2 scale[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = (tid >> 3) + k * (kMoveThreads / 8), slot = slots[i];
    if (slot < 0) continue;
    const uint8_t *src = rows[i][0];
    if (code) data[k] = *reinterpret_cast<const uint4 *>(src + piece);
    if (l < 2) {  // behind the block's 16 rows of codes
      const uint8_t *from = src - (slot >> 4) * (D / 2) + 8 * D + l * half + (slot >> 4) * 2 * c.groups;
      if (c.groups == 4)
        scale[k] = *reinterpret_cast<const uint2 *>(from);
      else if (c.groups == 2)
        scale[k].x = *reinterpret_cast<const uint32_t *>(from);
      else
        scale[k].x = *reinterpret_cast<const uint16_t *>(from);
    }
  }
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = (tid >> 3) + k * (kMoveThreads / 8), slot = slots[i];
    if (slot < 0) continue;
    uint8_t *dst = rows[i][1];
    if (code) *reinterpret_cast<uint4 *>(dst + piece) = data[k];
    if (l < 2) {
      uint8_t *to = dst - (slot & 15) * (D / 2) + 8 * D + l * half + (slot & 15) * 2 * c.groups;
      if (c.groups == 4)
        *reinterpret_cast<uint2 *>(to) = scale[k];
      else if (c.groups == 2)
        *reinterpret_cast<uint32_t *>(to) = scale[k].x;
      else
        *reinterpret_cast<uint16_t *>(to) = (uint16_t)scale[k].x;
    }
  }
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4View &c, const Kv4Batch &b, const Kv4Rows &r, uint32_t *status,
                              cudaStream_t stream) {
  return launch_rows<false>(c, b, r, status, stream);
}

cudaError_t launch_kv4_read(const Kv4View &c, const Kv4Batch &b, const Kv4Rows &r, uint32_t *status,
                            cudaStream_t stream) {
  return launch_rows<true>(c, b, r, status, stream);
}

size_t kv4_evict_workspace(const Kv4View &c, int n_seqs, int max_len, int budget) {
  const size_t rows = (size_t)n_seqs * c.kv_heads;
  return (kKv4Counters + rows * ((size_t)max_len + budget) + n_seqs) * 4;
}

cudaError_t launch_kv4_evict(const Kv4View &c, const Kv4Batch &b, const Kv4Evict &e, uint32_t *status,
                             cudaStream_t stream, int device) {
  static std::atomic<uint64_t> ready{0};  // devices on which the kernel may have that much shared memory
  const uint64_t bit = (uint64_t)1 << (device & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    const cudaError_t err =
        cudaFuncSetAttribute(kv4_select_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSelectShared);
    if (err != cudaSuccess) return err;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  const int64_t bytes = (int64_t)b.max_len * 4;
  const dim3 rows((unsigned)c.kv_heads, (unsigned)b.n_seqs);
  const bool shared = bytes <= kSelectShared;
  cudaError_t err = kv4_launch(shared ? kv4_select_kernel<true> : kv4_select_kernel<false>, rows, kSelectThreads,
                               shared ? (size_t)bytes : 0, stream, c, b, e, status);
  if (err != cudaSuccess) return err;
  const int most = e.budget < b.max_len ? e.budget : b.max_len;
  const dim3 grid((unsigned)((most + kMoveTokens - 1) / kMoveTokens), (unsigned)c.kv_heads, (unsigned)b.n_seqs);
  return kv4_launch(c.head_dim == 128 ? kv4_move_kernel<128> : kv4_move_kernel<64>, grid, kMoveThreads, 0, stream, c, b,
                    e, status);
}

}  // namespace ksb
