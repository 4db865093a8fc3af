// ks_kv4_attention.cuh -- attention over the paged 4-bit key/value cache.
//
// For a query row (new token j, query head) of a sequence with len cached
// tokens, n of them new, and every position t <= len - n + j
//   x_t = scale * q . k_t      out = sum_t e^(x_t - lse) v_t      lse = log sum_t e^(x_t)
// in one pass over the cache, with the running maximum and sum of the softmax.
//
// Tiles.  The rows of one key/value head (its query heads times the new
// tokens) are cut into tiles of 8 NT; a CTA takes one tile and one chunk of
// the tokens, its four warps take turns at tiles of 32 tokens, each through a
// ring of its own in shared memory that bulk copies fill.  Chunks are joined
// by a second kernel from (maximum, sum, unnormalised output) in f32.
//
// Products.  Both run on the tensor cores with the tokens' codes as the A
// operand, made in registers, and the query rows as the 8-wide N side, so that
// a decode step's few rows waste little: S^T = K Q^T (16 tokens x 8 rows,
// K over head_dim) and O^T = V^T P^T (16 elements x 8 rows, K over tokens).
//   keys    a 32-bit word holds 8 codes of a token; masked with 0x000F000F it
//           is, as two f16, the codes (+ 8, by flipping their top bit) times
//           2^-24, with 0x00F000F0 times 2^-20.  The queries carry a factor 16
//           where the codes have 2^-24, and the accumulators start at
//           -8 * sum(q), so a pair costs one logic instruction.
//   values  bytes of two tokens side by side, then 1024 + code - 1032 (or
//           (1024 + 16 code) / 16 - 72): signed, so that nothing has to cancel
//           in a sum over many tokens.
// The scales stay outside the products, in f32: a group's scores are
// multiplied by the token's key scale, the softmax weights by the token's
// value scale (times a power of two, the tile's, that brings them into f16's
// range) once per group.
//
// Precision.  Codes are exact in f16.  For f32 tensors queries (scaled by a
// power of two per row) and weighted probabilities are split into two f16
// parts with a product each, 22 bits; f16 and bf16 queries fit one part, and
// for bf16 results one part of the probabilities (11 bits) is well below the
// result's own rounding.  Sums over tokens leave the tensor core's accumulator
// (which truncates) after 32 tokens and go on in f32 registers.
#pragma once

#include "ks_kv4.cuh"

namespace ksb {

constexpr int kAttnWarps = 4, kAttnThreads = 32 * kAttnWarps;
constexpr int kTileBlocks = 2, kTileTokens = kTileBlocks * kKv4Block;
constexpr int kAttnStages = 3;

// How a call is cut: the same on the host, for the workspace, and in both kernels.
struct Kv4Plan {
  int rows_tile;  // 8 NT
  int row_tiles;  // tiles of a (sequence, key/value head)
  int chunk;      // tokens of a CTA
  int chunks;     // at most, of a tile
};

struct Kv4AttnArgs {
  Kv4View c;
  Kv4Batch b;
  Kv4Attention a;
  Kv4Plan p;
  int group_heads;
  uint32_t *status;
};

// Partial results of a tile's chunk: rows_tile x head_dim f32, then rows_tile maxima and sums.
__device__ __forceinline__ float *kv4_partial(const Kv4AttnArgs &k, int64_t tile, int chunk) {
  return static_cast<float *>(k.a.workspace) +
         (tile * k.p.chunks + chunk) * ((int64_t)k.p.rows_tile * (k.c.head_dim + 2));
}

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

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

// Row g of the products' token side is token kv4_token(g) of the block: any
// order serves, and with 0 1 3 2 4 5 7 6 the 16-byte loads of the keys (two
// rows, 64 bytes apart or an odd multiple of it, to a quarter warp) meet no
// bank twice and those of the values (rows 2t, t = 0..3) at most two times.
__device__ __forceinline__ int kv4_token(int g) { return g ^ ((g >> 1) & 1); }

template <int D, int NG, int NT, int QS>
struct Kv4Smem {
  static constexpr int kBlock = kv4_block_bytes(D, NG);
  static constexpr int kStage = kTileBlocks * kBlock;
  static constexpr int kRing = kAttnWarps * kAttnStages * kStage;
  static constexpr int kMerge = kAttnWarps * 8 * NT * (D + 2) * 4;  // over the ring, once it is drained
  static constexpr int kQ = kRing > kMerge ? kRing : kMerge;        // NT x D/32 x QS fragments of 512 bytes
  static constexpr int kCorr = kQ + NT * (D / 32) * QS * 512;       // NT x NG x 8 f32
  static constexpr int kFactor = kCorr + NT * NG * 8 * 4;           // 8 NT f32
  static constexpr int kLse = kFactor + 8 * NT * 4;                 // 8 NT f32
  static constexpr int kBar = kLse + 8 * NT * 4;                    // mbarriers
  static constexpr int kBytes = kBar + kAttnWarps * kAttnStages * 8;
};

// Reads the tile's query rows into B fragments.  A thread has the 8 elements
// 32w + 8t .. of one row, the ones that lane (row, t) multiplies with the words
// of a token's keys: halves (0, 4) and (2, 6), with the factor 16, and (1, 5)
// and (3, 7).  A row is scaled by the power of two that brings its largest
// element into [2^10, 2^11).
template <typename T, int D, int NG, int NT, int QS>
__device__ __forceinline__ void load_queries(const Kv4AttnArgs &k, const Kv4Seq &q, int head, int row0, int rows,
                                             char *smem) {
  using S = Kv4Smem<D, NG, NT, QS>;
  constexpr int PER = D / 8;  // threads of a row
  constexpr int W = D / 32 / NG;  // words of a group
  const int tid = threadIdx.x;
#pragma unroll
  for (int base = 0; base < 8 * NT * PER; base += kAttnThreads) {
    const int i = base + tid, n = i / PER, w = (i % PER) >> 2, t = i & 3;  // (8 NT PER is a multiple of 64)
    if (8 * NT * PER % kAttnThreads && i >= 8 * NT * PER) break;           // whole warps
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    const int r = row0 + n;
    if (r < rows) {
      const int j = r / k.group_heads, h = head * k.group_heads + r % k.group_heads;
      const T *src = static_cast<const T *>(k.a.q) + (int64_t)(q.first + j) * k.a.q_token + h * k.a.q_head + 32 * w +
                     8 * t;
      if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
        T x[8];
#pragma unroll
        for (int e = 0; e < (int)sizeof(T) / 2; ++e)
          reinterpret_cast<uint4 *>(x)[e] = reinterpret_cast<const uint4 *>(src)[e];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = kv4_load(&x[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = kv4_load(src + e);
      }
    }
    float top = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[e]));
#pragma unroll
    for (int o = 1; o < PER; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int power = top > 0.0f && isfinite(top) ? min(max(10 - ilogbf(top), -100), 120) : 0;
    const float up = ldexpf(1.0f, power);
    uint32_t hi[4], lo[4];  // (0, 4) (1, 5) (2, 6) (3, 7)
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float f = e & 1 ? up : 16.0f * up, a = v[e] * f, b = v[e + 4] * f;
      hi[e] = pack_f16(a, b);
      const float2 h = unpack_f16(hi[e]);
      float2 l = make_float2(0.0f, 0.0f);
      if (QS == 2) {
        lo[e] = pack_f16(a - h.x, b - h.y);
        l = unpack_f16(lo[e]);
      }
      sum += (e & 1 ? 1.0f : 0.0625f) * ((h.x + l.x) + (h.y + l.y));
    }
    const int at = (n & 7) * 4 + t, frag = ((n >> 3) * (D / 32) + w) * QS;
    reinterpret_cast<uint4 *>(smem + S::kQ + frag * 512)[at] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if (QS == 2) reinterpret_cast<uint4 *>(smem + S::kQ + (frag + 1) * 512)[at] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
#pragma unroll
    for (int o = 1; o < 4 * W; o *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (t == 0 && w % W == 0)  // codes + 8 stand for 2^-20 of their value
      reinterpret_cast<float *>(smem + S::kCorr)[((n >> 3) * NG + w / W) * 8 + (n & 7)] = sum * (-8.0f * 0x1p-20f);
    if (w == 0 && t == 0)
      reinterpret_cast<float *>(smem + S::kFactor)[n] =
          (r < rows ? k.a.scale * 1.44269504088896341f : 0.0f) * ldexpf(1.0f, 20 - power);
  }
}

// The scores, times log2(e), of a block's 16 tokens: s[nt][0..3] of (token g,
// row 2t), (g, 2t + 1), (g + 8, 2t), (g + 8, 2t + 1), tokens as kv4_token has them.
template <int D, int NG, int NT, int QS>
__device__ __forceinline__ void block_scores(const char *block, const char *smem, const float (&factor)[NT][2],
                                             float (&s)[NT][4]) {
  using S = Kv4Smem<D, NG, NT, QS>;
  constexpr int W = D / 32 / NG;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, tok = kv4_token(g);
  uint32_t x[D / 32], y[D / 32];
  lds<D / 8>(block + tok * (D / 2) + t * (D / 8), x);
  lds<D / 8>(block + (tok + 8) * (D / 2) + t * (D / 8), y);
  float sx[NG], sy[NG];
  load_scales<NG>(block + 8 * D + tok * 2 * NG, sx);
  load_scales<NG>(block + 8 * D + (tok + 8) * 2 * NG, sy);
#pragma unroll
  for (int gr = 0; gr < NG; ++gr) {
    float acc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float2 c = *reinterpret_cast<const float2 *>(smem + S::kCorr + ((nt * NG + gr) * 8 + 2 * t) * 4);
      acc[nt][0] = acc[nt][2] = c.x;
      acc[nt][1] = acc[nt][3] = c.y;
    }
#pragma unroll
    for (int w = gr * W; w < (gr + 1) * W; ++w) {
      constexpr uint32_t L = 0x000F000Fu, H = 0x00F000F0u, FL = 0x00080008u, FH = 0x00800080u;
      const uint32_t x8 = x[w] >> 8, y8 = y[w] >> 8;
      const uint32_t a[8] = {and_xor(x[w], L, FL), and_xor(y[w], L, FL), and_xor(x[w], H, FH), and_xor(y[w], H, FH),
                             and_xor(x8, L, FL),   and_xor(y8, L, FL),   and_xor(x8, H, FH),   and_xor(y8, H, FH)};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int p = 0; p < QS; ++p) {
          uint32_t q[4];
          lds<16>(smem + S::kQ + ((nt * (D / 32) + w) * QS + p) * 512 + lane * 16, q);
          mma_f16(acc[nt], a[0], a[1], a[2], a[3], q[0], q[1]);
          mma_f16(acc[nt], a[4], a[5], a[6], a[7], q[2], q[3]);
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      s[nt][0] = gr ? fmaf(acc[nt][0], sx[gr], s[nt][0]) : acc[nt][0] * sx[gr];
      s[nt][1] = gr ? fmaf(acc[nt][1], sx[gr], s[nt][1]) : acc[nt][1] * sx[gr];
      s[nt][2] = gr ? fmaf(acc[nt][2], sy[gr], s[nt][2]) : acc[nt][2] * sy[gr];
      s[nt][3] = gr ? fmaf(acc[nt][3], sy[gr], s[nt][3]) : acc[nt][3] * sy[gr];
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[nt][e] *= factor[nt][e & 1];
}

// Start copying the blocks of the tile at token `at` (below `end`) into a
// stage; HALF of a block is its keys.  One lane.
template <int D, int NG, bool KEYS>
__device__ __forceinline__ void fetch_tile(const Kv4AttnArgs &k, int seq, int head, int at, int end, char *stage,
                                           uint64_t *bar) {
  constexpr int B = kv4_block_bytes(D, NG), N = KEYS ? B / 2 : B;
  const int blocks = min(kTileBlocks, (end - at + kKv4Block - 1) / kKv4Block);
  const int mask = (1 << k.c.page_shift) - 1;
  mbar_arrive_expect_tx(bar, (uint32_t)(blocks * N));
  if (!KEYS && k.c.page_shift >= 5) {  // a tile lies within a page
    const int page = max(kv4_page(k.c, k.b.table, k.b.table_stride, seq, at, k.status), 0);
    bulk_g2s(stage, kv4_block(k.c, page, head, at & mask), (uint32_t)(blocks * N), bar);
  } else {
    for (int i = 0; i < blocks; ++i) {
      const int pos = at + i * kKv4Block;
      const int page = max(kv4_page(k.c, k.b.table, k.b.table_stride, seq, pos, k.status), 0);
      bulk_g2s(stage + i * B, kv4_block(k.c, page, head, pos & mask), (uint32_t)N, bar);
    }
  }
}

// WEIGHTS: adds the attention weights of every token to the cache's, given the rows' lse.
template <typename T, int D, int NG, int NT, int QS, int PS, bool WEIGHTS>
__global__ void __launch_bounds__(kAttnThreads, NT == 1 ? 3 : 2) kv4_attention_kernel(const Kv4AttnArgs k) {
  using S = Kv4Smem<D, NG, NT, QS>;
  extern __shared__ __align__(128) char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  // row tiles next to each other, then heads, sequences and, slowest, chunks
  int64_t id = blockIdx.x;
  const int row_tiles = WEIGHTS ? 1 : k.p.row_tiles;
  const int first_tile = (int)(id % row_tiles);
  id /= row_tiles;
  const int head = (int)(id % k.c.kv_heads);
  id /= k.c.kv_heads;
  const int seq = (int)(id % k.b.n_seqs), chunk = (int)(id / k.b.n_seqs);
  const Kv4Seq q = kv4_seq(k.b, seq, k.status);
  if (q.n_new > k.a.max_new && tid == 0) set_status(k.status, kStatusBadScale);
  const int rows = min(q.n_new, k.a.max_new) * k.group_heads;
  const int past = q.len - q.n_new + 1;  // tokens that the first new one sees

  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + S::kBar) + warp * kAttnStages;
  if (lane == 0) {
    for (int s = 0; s < kAttnStages; ++s) mbar_init(&bars[s], 1);
    fence_mbarrier_init();
  }
  __syncwarp();
  char *ring = smem + warp * kAttnStages * S::kStage;
  int fetched = 0, used = 0;  // tiles of this warp, over all row tiles
  bool lost = false;

  for (int tile = first_tile; tile < (WEIGHTS ? k.p.row_tiles : first_tile + 1); ++tile) {
    const int row0 = tile * k.p.rows_tile;
    if (row0 >= rows) break;
    const int last = min(row0 + k.p.rows_tile, rows) - 1;
    const int seen = min(max(past + last / k.group_heads, 0), q.len);  // of the tile's last row
    const int begin = chunk * k.p.chunk, end = min(begin + k.p.chunk, seen);
    if (begin >= seen && (chunk > 0 || WEIGHTS)) {
      if (WEIGHTS) continue;
      break;
    }
    const int tiles = (end - begin + kTileTokens - 1) / kTileTokens;          // <= 0: nothing is seen
    const int mine = tiles > warp ? (tiles - warp + kAttnWarps - 1) / kAttnWarps : 0;
    auto fetch = [&](int i) {
      if (lane == 0) {
        const int stage = fetched % kAttnStages;
        fetch_tile<D, NG, WEIGHTS>(k, seq, head, begin + (warp + i * kAttnWarps) * kTileTokens, end,
                                   ring + stage * S::kStage, &bars[stage]);
      }
      ++fetched;
    };
    for (int i = 0; i < min(mine, kAttnStages); ++i) fetch(i);

    if (WEIGHTS) __syncthreads();  // the previous rows' fragments have been read
    load_queries<T, D, NG, NT, QS>(k, q, head, row0, rows, smem);
    if (WEIGHTS && tid < 8 * NT) {
      const int r = row0 + tid;
      float v = INFINITY;  // no weight for rows that are not there or see nothing
      if (r < rows) {
        const float lse = k.a.lse[(int64_t)(q.first + r / k.group_heads) * k.a.q_heads + head * k.group_heads +
                                  r % k.group_heads];
        if (lse != -INFINITY) v = lse * 1.44269504088896341f;
      }
      reinterpret_cast<float *>(smem + S::kLse)[tid] = v;
    }
    __syncthreads();

    float factor[NT][2], lse2[NT][2];
    int limit[NT][2];  // tokens that rows 2t, 2t + 1 see
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int n = nt * 8 + 2 * t + e, r = row0 + n;
        factor[nt][e] = reinterpret_cast<const float *>(smem + S::kFactor)[n];
        lse2[nt][e] = WEIGHTS ? reinterpret_cast<const float *>(smem + S::kLse)[n] : 0.0f;
        limit[nt][e] = r < rows ? min(past + r / k.group_heads, q.len) : q.len;
      }
    const int all_see = max(past + row0 / k.group_heads, 0);  // no mask below

    float o[NT][WEIGHTS ? 1 : D / 16][4], top[NT][2], sum[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      top[nt][0] = top[nt][1] = -INFINITY;
      sum[nt][0] = sum[nt][1] = 0.0f;
      if constexpr (!WEIGHTS) {
#pragma unroll
        for (int m = 0; m < D / 16; ++m) o[nt][m][0] = o[nt][m][1] = o[nt][m][2] = o[nt][m][3] = 0.0f;
      }
    }

    for (int i = 0; i < mine; ++i) {
      const int stage = used % kAttnStages, at = begin + (warp + i * kAttnWarps) * kTileTokens;
      const char *buf = ring + stage * S::kStage;
      if (!mbar_wait(&bars[stage], (used / kAttnStages) & 1)) {
        set_status(k.status, kStatusTimeout);
        lost = true;
        break;
      }
      ++used;
      const bool whole = at + kTileTokens <= min(all_see, end);
      float p[kTileBlocks][NT][4];
#pragma unroll
      for (int b = 0; b < kTileBlocks; ++b) {
        block_scores<D, NG, NT, QS>(buf + b * S::kBlock, smem, factor, p[b]);
        if (!whole) {
          const int tok = at + b * kKv4Block + kv4_token(g);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (tok + (e >> 1) * 8 >= min(limit[nt][e & 1], end)) p[b][nt][e] = -INFINITY;
        }
      }

      if constexpr (WEIGHTS) {
#pragma unroll
        for (int b = 0; b < kTileBlocks; ++b) {
          float w[2] = {0.0f, 0.0f};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e >> 1] += fast_exp2(p[b][nt][e] - lse2[nt][e & 1]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            w[e] += __shfl_xor_sync(0xffffffffu, w[e], 1);
            w[e] += __shfl_xor_sync(0xffffffffu, w[e], 2);
            const int tok = at + b * kKv4Block + kv4_token(g) + 8 * e;
            if (t == 0 && tok < end) {
              const int page = kv4_page(k.c, k.b.table, k.b.table_stride, seq, tok, k.status);
              if (page >= 0)
                k.c.weights[(((int64_t)page * k.c.kv_heads + head) << k.c.page_shift) +
                            (tok & ((1 << k.c.page_shift) - 1))] += w[e];
            }
          }
        }
      } else {
        // running maximum and sum
        float alpha[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float m = fmaxf(p[0][nt][e], p[0][nt][e + 2]);
#pragma unroll
            for (int b = 1; b < kTileBlocks; ++b) m = fmaxf(m, fmaxf(p[b][nt][e], p[b][nt][e + 2]));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
            m = fmaxf(m, top[nt][e]);
            const float base = m == -INFINITY ? 0.0f : m;  // a row that has seen nothing yet
            alpha[nt][e] = fast_exp2(top[nt][e] - base);
            top[nt][e] = m;
            float add = 0.0f;
#pragma unroll
            for (int b = 0; b < kTileBlocks; ++b) {
              p[b][nt][e] = fast_exp2(p[b][nt][e] - base);
              p[b][nt][e + 2] = fast_exp2(p[b][nt][e + 2] - base);
              add += p[b][nt][e] + p[b][nt][e + 2];
            }
            sum[nt][e] = fmaf(sum[nt][e], alpha[nt][e], add);
          }
        // value scales of this lane's tokens, and the power of two that brings the largest to [2^14, 2^15)
        float sv[kTileBlocks][2][NG], big = 0.0f;
#pragma unroll
        for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int tok = kv4_token(g) + 8 * e;
            load_scales<NG>(buf + b * S::kBlock + S::kBlock / 2 + 8 * D + tok * 2 * NG, sv[b][e]);
            const bool there = at + b * kKv4Block + tok < end;  // what stands behind the last token is not read
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
              sv[b][e][gr] = there ? sv[b][e][gr] : 0.0f;
              big = fmaxf(big, sv[b][e][gr]);
            }
          }
#pragma unroll
        for (int x = 4; x < 32; x *= 2) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, x));
        const uint32_t power = max(__float_as_uint(big) >> 23, 16u);  // biased; f16 scales are normal in f32
        const float up = __uint_as_float((127u + 14u + 127u - power) << 23);
        const float down = __uint_as_float((power - 14u) << 23);

        // value codes: a 32-bit word has this lane's pairs of four 16-element slices
        uint32_t v[kTileBlocks][4][D / 64];
#pragma unroll
        for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            lds<D / 16>(buf + b * S::kBlock + S::kBlock / 2 +
                            (kv4_token(2 * t + (e & 1)) + 8 * (e >> 1)) * (D / 2) + g * (D / 16),
                        v[b][e]);
        uint32_t ph[kTileBlocks][NT][2], pl[kTileBlocks][NT][2];
#pragma unroll
        for (int m = 0; m < D / 16; ++m) {
          constexpr int M = D / 16 / NG;  // slices of a group
          if (m % M == 0) {
#pragma unroll
            for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float f = sv[b][e][m / M] * up;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  const float x0 = p[b][nt][2 * e] * f, x1 = p[b][nt][2 * e + 1] * f;
                  const uint32_t h = pack_f16(x0, x1);
                  ph[b][nt][e] = transpose8x8(h);
                  if (PS == 2) {
                    const float2 r = unpack_f16(h);
                    pl[b][nt][e] = transpose8x8(pack_f16(x0 - r.x, x1 - r.y));
                  }
                }
              }
          }
          float acc[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.0f;
#pragma unroll
          for (int b = 0; b < kTileBlocks; ++b) {
            uint32_t a[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t w = prmt(v[b][2 * e][m / 4], v[b][2 * e + 1][m / 4], (m % 4) | ((4 + m % 4) << 8));
              const uint32_t lo = and_xor(w, 0x000F000Fu, 0x64086408u), hi = and_xor(w, 0x00F000F0u, 0x64806480u);
              const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&lo), __floats2half2_rn(1032.0f, 1032.0f));
              const __half2 y = __hfma2(*reinterpret_cast<const __half2 *>(&hi), __floats2half2_rn(0.0625f, 0.0625f),
                                        __floats2half2_rn(-72.0f, -72.0f));
              a[2 * e] = *reinterpret_cast<const uint32_t *>(&x);
              a[2 * e + 1] = *reinterpret_cast<const uint32_t *>(&y);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_f16(acc[nt], a[0], a[1], a[2], a[3], ph[b][nt][0], ph[b][nt][1]);
              if (PS == 2) mma_f16(acc[nt], a[0], a[1], a[2], a[3], pl[b][nt][0], pl[b][nt][1]);
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][m][e] = fmaf(acc[nt][e], down, o[nt][m][e] * alpha[nt][e & 1]);
        }
      }
      __syncwarp();  // every lane has read the stage
      if (i + kAttnStages < mine) fetch(i + kAttnStages);
    }
    if constexpr (WEIGHTS) {
      if (lost) used = fetched;
      continue;
    } else {
      // join the warps: the ring is drained, each writes its part over it
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int x = 4; x < 32; x *= 2) sum[nt][e] += __shfl_xor_sync(0xffffffffu, sum[nt][e], x);
      __syncthreads();
      constexpr int R = 8 * NT;
      float *part = reinterpret_cast<float *>(smem);  // [warp][row][D], then [warp][2][row]
      float *stat = part + kAttnWarps * R * D;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int n = nt * 8 + 2 * t + e;
#pragma unroll
          for (int m = 0; m < D / 16; ++m)
            *reinterpret_cast<float2 *>(part + (warp * R + n) * D + 16 * m + 2 * g) =
                make_float2(o[nt][m][e], o[nt][m][e + 2]);
          if (g == 0) {
            stat[warp * 2 * R + n] = top[nt][e];
            stat[warp * 2 * R + R + n] = sum[nt][e];
          }
        }
      __syncthreads();
      const int chunks = max((seen + k.p.chunk - 1) / k.p.chunk, 1);
      const int64_t tile_id = ((int64_t)seq * k.c.kv_heads + head) * k.p.row_tiles + tile;
      float *to = kv4_partial(k, tile_id, chunk);
      for (int i = tid; i < R * D; i += kAttnThreads) {
        const int n = i / D, d = i % D, r = row0 + n;
        if (r >= rows) break;
        float m = stat[n];
#pragma unroll
        for (int w = 1; w < kAttnWarps; ++w) m = fmaxf(m, stat[w * 2 * R + n]);
        const float base = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, x = 0.0f;
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) {
          const float f = fast_exp2(stat[w * 2 * R + n] - base);
          l = fmaf(stat[w * 2 * R + R + n], f, l);
          x = fmaf(part[(w * R + n) * D + d], f, x);
        }
        if (chunks > 1) {
          to[i] = x;
          if (d == 0) {
            to[R * D + n] = m;
            to[R * D + R + n] = l;
          }
        } else {
          const int64_t token = q.first + r / k.group_heads;
          const int h = head * k.group_heads + r % k.group_heads;
          kv4_store(static_cast<T *>(k.a.out) + token * k.a.out_token + h * k.a.out_head + d,
                    l > 0.0f || l != l ? x / l : 0.0f);
          if (d == 0 && k.a.lse)
            k.a.lse[token * k.a.q_heads + h] = l > 0.0f || l != l ? (m + log2f(l)) * 0.693147180559945309f : -INFINITY;
        }
      }
    }
  }
}

// Joins the chunks of one query row: a CTA of head_dim threads in each of four
// groups, which take turns at the chunks.
template <typename T, int D>
__global__ void __launch_bounds__(4 * D) kv4_join_kernel(const Kv4AttnArgs k) {
  __shared__ float part[4][D + 1];
  const int d = threadIdx.x % D, way = threadIdx.x / D;
  int64_t id = blockIdx.x;
  const int rows_all = k.p.row_tiles * k.p.rows_tile;
  const int r = (int)(id % rows_all);
  id /= rows_all;
  const int head = (int)(id % k.c.kv_heads), seq = (int)(id / k.c.kv_heads);
  const Kv4Seq q = kv4_seq(k.b, seq, nullptr);
  const int rows = min(q.n_new, k.a.max_new) * k.group_heads;
  if (r >= rows) return;
  const int tile = r / k.p.rows_tile, n = r % k.p.rows_tile, R = k.p.rows_tile;
  const int last = min(tile * R + R, rows) - 1;
  const int seen = min(max(q.len - q.n_new + 1 + last / k.group_heads, 0), q.len);
  const int chunks = (seen + k.p.chunk - 1) / k.p.chunk;
  if (chunks <= 1) return;  // written already
  const int64_t tile_id = ((int64_t)seq * k.c.kv_heads + head) * k.p.row_tiles + tile;
  float m = -INFINITY;
  for (int c = 0; c < chunks; ++c) m = fmaxf(m, kv4_partial(k, tile_id, c)[R * D + n]);
  const float base = m == -INFINITY ? 0.0f : m;
  float x = 0.0f, l = 0.0f;
  for (int c = way; c < chunks; c += 4) {
    const float *p = kv4_partial(k, tile_id, c);
    const float f = fast_exp2(p[R * D + n] - base);
    x = fmaf(p[n * D + d], f, x);
    l = fmaf(p[R * D + R + n], f, l);
  }
  part[way][d] = x;
  if (d == 0) part[way][D] = l;
  __syncthreads();
  if (way) return;
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    x += part[w][d];
    l += part[w][D];
  }
  const int64_t token = q.first + r / k.group_heads;
  const int h = head * k.group_heads + r % k.group_heads;
  kv4_store(static_cast<T *>(k.a.out) + token * k.a.out_token + h * k.a.out_head + d, l > 0.0f || l != l ? x / l : 0.0f);
  if (d == 0 && k.a.lse)
    k.a.lse[token * k.a.q_heads + h] = l > 0.0f || l != l ? (m + log2f(l)) * 0.693147180559945309f : -INFINITY;
}

template <typename T, int D, int NG, int NT, int QS, int PS, bool WEIGHTS>
cudaError_t launch_kv4_attention_pass(const Kv4AttnArgs &k, cudaStream_t stream) {
  const int64_t ctas =
      (int64_t)(WEIGHTS ? 1 : k.p.row_tiles) * k.c.kv_heads * k.b.n_seqs * k.p.chunks;
  if (ctas > 0x7FFFFFFF) return cudaErrorInvalidValue;
  constexpr int bytes = Kv4Smem<D, NG, NT, QS>::kBytes;
  auto *f = kv4_attention_kernel<T, D, NG, NT, QS, PS, WEIGHTS>;
  cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return e;
  f<<<(unsigned)ctas, kAttnThreads, bytes, stream>>>(k);
  return cudaGetLastError();
}

template <typename T, int D, int NG, int NT, int QS, int PS>
cudaError_t launch_kv4_attention_all(const Kv4AttnArgs &k, cudaStream_t stream) {
  cudaError_t e = launch_kv4_attention_pass<T, D, NG, NT, QS, PS, false>(k, stream);
  if (e == cudaSuccess && k.p.chunks > 1) {
    const int64_t ctas = (int64_t)k.p.row_tiles * k.p.rows_tile * k.c.kv_heads * k.b.n_seqs;
    if (ctas > 0x7FFFFFFF) return cudaErrorInvalidValue;
    kv4_join_kernel<T, D><<<(unsigned)ctas, 4 * D, 0, stream>>>(k);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess && k.a.accumulate) e = launch_kv4_attention_pass<T, D, NG, NT, QS, PS, true>(k, stream);
  return e;
}

// One translation unit per type: QS and PS as the precision note says.
template <typename T, int QS, int PS>
cudaError_t launch_kv4_attention_typed(const Kv4AttnArgs &k, cudaStream_t stream) {
  const int key = k.c.head_dim * 100 + k.c.groups * 10 + k.p.rows_tile / 8;
  switch (key) {
#define KS_KV4_CASE(D, NG)                                                   \
  case D * 100 + NG * 10 + 1:                                                \
    return launch_kv4_attention_all<T, D, NG, 1, QS, PS>(k, stream);         \
  case D * 100 + NG * 10 + 2:                                                \
    return launch_kv4_attention_all<T, D, NG, 2, QS, PS>(k, stream);
    KS_KV4_CASE(128, 4)
    KS_KV4_CASE(128, 2)
    KS_KV4_CASE(128, 1)
    KS_KV4_CASE(64, 2)
    KS_KV4_CASE(64, 1)
#undef KS_KV4_CASE
    default:
      return cudaErrorInvalidValue;
  }
}

cudaError_t launch_kv4_attention_f32(const Kv4AttnArgs &k, cudaStream_t stream);
cudaError_t launch_kv4_attention_f16(const Kv4AttnArgs &k, cudaStream_t stream);
cudaError_t launch_kv4_attention_bf16(const Kv4AttnArgs &k, cudaStream_t stream);

}  // namespace ksb
