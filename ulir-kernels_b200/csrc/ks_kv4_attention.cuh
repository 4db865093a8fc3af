// ks_kv4_attention.cuh -- attention over the paged 4-bit key/value cache.
//
// For a query row (new token j, query head) of a sequence with len cached
// tokens, n of them new, and every position t <= len - n + j
//   x_t = scale * q . k_t      out = sum_t e^(x_t - lse) v_t      lse = log sum_t e^(x_t)
// in one pass over the cache, with the running maximum and sum of the softmax.
//
// Work.  The rows of one key/value head (its query heads times the new
// tokens) are cut into tiles of 8 NT; a row tile's tokens, 128 or 256 at a
// time, are the units of work.  All units of the call stand in one line
// (sequence, head, row tile, tokens) and every CTA of a grid that the GPU holds
// at once takes an equal stretch of it, so that sequences of unequal lengths and
// few long ones alike fill the GPU evenly.  An item's beginning counts as three units more,
// about what it costs: 64 sequences of up to 8192 tokens, 8 heads, take 69 us
// (before joins were made shorter 70, and then 98 without).  (Where few items
// give each CTA about one, it gets a part of one
// item.)  Of an item (a row tile and all its tokens) that
// a stretch ends within, each CTA leaves its part (maximum, sum, unnormalised
// output, f32) in the workspace; the last of them to finish joins the parts in
// their order, so results do not depend on which one that is.  Within a CTA
// four warps take turns at tiles of 32 or 64 tokens, each through a ring of its
// own in shared memory that its lanes fill by asynchronous 16-byte copies (one
// bulk copy for each tile, issued by a lane, took the same time).
//
// Products.  Both run on the tensor cores with the tokens' codes as the A
// operand, made in registers, and the query rows as the 8-wide N side, so that
// a decode step's few rows waste little: S^T = K Q^T (16 tokens x 8 rows,
// K over head_dim) and O^T = V^T P^T (16 elements x 8 rows, K over tokens).
//   keys    a 32-bit word holds 8 codes of a token; masked with 0x000F000F it
//           is, as two f16, the codes (+ 8, by flipping their top bit) times
//           2^-24, with 0x00F000F0 times 2^-20.  The queries carry a factor 16
//           where the codes have 2^-24.  The accumulators start at -8 *
//           sum(q), so a pair costs one logic instruction.
//   values  bytes of two tokens side by side, then 1024 + code - 1032 (or
//           (1024 + 16 code) / 16 - 72): signed, so that nothing has to cancel
//           in a sum over many tokens.
// The scales stay outside the products, in f32: a group's scores are
// multiplied by the token's key scale, the softmax weights by the token's
// value scale (times a power of two that brings them into f16's range) once
// per group.  The maximum that the exponentials refer to, and that power of
// two, are only raised when a tile exceeds them (the maximum by 2^4), which a
// vote finds: most tiles need no reduction over lanes and no rescaling.
//
// What bounds it.  No unit is full; a warp's scores, vote, exponentials and value
// products follow one another, and the three warps that a scheduler has (168
// registers to a thread) do not fill each other's waits.  64 sequences of up to
// 8192 tokens, 8 heads, bf16, groups of 64: 37.4 M warp instructions (275 for 16
// tokens of a head, most of them widen codes), 32 us if every scheduler issued one
// a cycle; they are issued in 0.54 of the cycles, the integer pipe is busy in 0.47,
// the tensor cores in 0.25, DRAM in 0.48; 0.92 of a warp is ready in the mean, and
// of a warp's waits the largest is for results of fixed latency.  For an eighth of
// the time an SM has not begun or has no more work (16 sequences of up to 4096,
// f32: for more than a quarter, 0.46 issued).  With few rows the products are not
// what takes the time, which is why these are the warp-wide ones, whose A operand
// is made in registers: a tensor-memory operand would have to be stored there
// first.  444 equal items of 4096 tokens, 128 elements, bf16: 46 us, 5.2 TB/s of
// codes and scales with groups of 128, 57 us, 4.6 TB/s with groups of 32; f16 52 and
// 65, f32 60 and 75 us, 4.0 and 3.5 TB/s.  The copies without the products take 0.8
// of the time.
// A call's beginning (the lengths, the queries) and end (the four warps' sums,
// the join of an item's parts) take 8 us together, which is what short calls
// take.
//
// Precision.  Codes are exact in f16.  For f32 tensors queries (scaled by a
// power of two per row) and weighted probabilities are split into two f16
// parts with a product each, 22 bits.  The accumulators truncate, which over a
// few steps would cost two bits: so the queries' first parts are integers up to
// 2^11, whose sums of up to 128 products stay below 2^24 and are exact, the
// second parts have accumulators of their own, and sums over tokens leave the
// accumulators after a tile and go on in f32 registers.  f16 and bf16 queries
// fit one part, and for bf16 results one part of the probabilities (11 bits) is
// an eighth of the result's own rounding.  Their sums over tokens stay in the
// accumulators for 128 products, a loss of at most 2^-16, and are then added up
// in f32 (kept for a whole item of 524288 tokens, they lost 7e-4, more than half
// a step of f16; adding up after every tile, as for f32, takes 6 % more time at
// 64 sequences of up to 8192, this 1 %).
// A weight (probability times value scale) has its parts' last bit at 2^-24,
// where the largest value scale stands at 2^10: 22 bits for scales down to 2^-11
// of that.  Once a warp meets a smaller one, in any token or group (f16 results:
// 2^-14, bf16: 2^-15), it goes on in a second form of the loop, where the largest
// weight of each tile, row and group is brought to 2^13 and each tile's product is
// added in f32: a result far below values that have next to no weight in it keeps
// its bits (without, it lost all of them from 2^-36 on).  The second form takes 1.2
// times as long with groups of 128, twice as long with groups of 32.  Looking for
// such a scale takes 1 to 3 % (64 sequences of up to 8192, bf16: 68.6 -> 69.4 us;
// 16 of up to 4096, f32: 21.7 -> 22.2).
#pragma once

#include <atomic>
#include <type_traits>

#include "ks_kv4.cuh"

namespace ksb {

constexpr int kAttnWarps = 4, kAttnThreads = 32 * kAttnWarps;
// Blocks of a warp's tile: four where two such tiles of every warp fit shared
// memory and their scores the registers, for fewer waits and votes (64 sequences
// of up to 8192 tokens, bf16, groups of 64: 70 us, 72 with two blocks and four
// CTAs; a sequence of 131071: 40, 42; 8 of 2047 in pages of 32, f16: 21, 19.5, all
// before the joins were made shorter).
__host__ __device__ constexpr int kv4_tile_blocks(int nt, int groups) { return nt == 1 && groups <= 2 ? 4 : 2; }
// Tokens of a unit of work.
__host__ __device__ constexpr int kv4_unit_tokens(int nt, int groups) {
  return kAttnWarps * kv4_tile_blocks(nt, groups) * kKv4Block;
}
// Products after which sums over tokens leave the accumulators (f16 and bf16; each may cost 2^-23 of the sum).
constexpr int kFoldProducts = 128;
constexpr int kJoin = 8;  // parts that are loaded together to be joined
// Of kKv4Counters at the start of the workspace a CTA has three, of the
// item that begins in its stretch (finished groups of parts), of that item's
// first group of parts and of a later group, which begins at this CTA.
constexpr int kAttnCtas = 680;

// How a call is cut: the same on the host, for the workspace, and in the kernel.
struct Kv4Plan {
  int rows_tile;  // 8 NT
  int row_tiles;  // tiles of a (sequence, key/value head), at most
  int ctas;
};

struct Kv4AttnArgs {
  Kv4View c;
  Kv4Batch b;
  Kv4Attention a;
  Kv4Plan p;
  int group_heads;
  uint32_t *status;
};

// CTAs of a pass that an SM holds, bounded by registers: 168 a thread, 255 with
// NT 2.  (Four CTAs of 128 registers, tiles of two blocks, f16 and bf16: the same
// time per item over 148 sequences of 4096 tokens, 4 heads.)  With 128 elements some
// kernels have more than fits and spill: f32 156 bytes a thread (groups of 64, NT 1),
// 148 (groups of 32, NT 2), 28 (groups of 32, NT 1), others and f16 up to 8.
constexpr int kv4_ctas_per_sm(int nt) { return nt == 1 ? 3 : 2; }

// Partial results of CTA c: rows_tile x head_dim f32, then rows_tile maxima
// and sums; slot 0 of an item that an earlier CTA began, slot 1 of one that a
// later CTA ends.
__device__ __forceinline__ float *kv4_partial(const Kv4AttnArgs &k, int cta, int slot) {
  return static_cast<float *>(k.a.workspace) + kKv4Counters +
         ((int64_t)cta * 2 + slot) * (k.p.rows_tile * (k.c.head_dim + 2));
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

// d = a * b + c, the rows' constants of a lane's four accumulators
__device__ __forceinline__ void mma_f16_from(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1, const float4 &c) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, "
      "%12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c.x), "f"(c.y), "f"(c.z), "f"(c.w));
}

__device__ __forceinline__ void copy16_async(void *to, const void *from) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

// Row g of the products' token side is token kv4_token(g) of the block: any
// order serves, and with 0 1 3 2 4 5 7 6 the 16-byte loads of the keys (two
// rows, 64 bytes apart or an odd multiple of it, to a quarter warp) meet no
// bank twice and those of the values (rows 2t, t = 0..3) at most two times.
__device__ __forceinline__ int kv4_token(int g) { return g ^ ((g >> 1) & 1); }

template <int D, int NG, int NT, int QS>
struct Kv4Smem {
  static constexpr int kBlock = kv4_block_bytes(D, NG);
  static constexpr int kTileBlocks = kv4_tile_blocks(NT, NG);
  static constexpr int kStage = kTileBlocks * kBlock;
  static constexpr int kStages = kTileBlocks == 4 ? 2 : 3;
  static constexpr int kRing = kAttnWarps * kStages * kStage;
  static constexpr int kMerge = kAttnWarps * 8 * NT * (D + 2) * 4;  // over the ring, once it is drained
  static constexpr int kQ = kRing > kMerge ? kRing : kMerge;        // NT x D/32 x QS fragments of 512 bytes
  static constexpr int kCorr = kQ + NT * (D / 32) * QS * 512;       // NT x NG x QS x 4 float4
  static constexpr int kFactor = kCorr + NT * NG * QS * 64;        // 8 NT f32
  static constexpr int kLse = kFactor + 8 * NT * 4;                 // 8 NT f32
  static constexpr int kShare = kLse + 8 * NT * 4;                  // 8 words
  static constexpr int kBytes = kShare + 32;
};

// The tile's query rows as B fragments.  A thread has the 8 elements 32w + 8t ..
// of one row (of each 128 / (D / 8) rows), the ones that lane (row, t)
// multiplies with the words of a token's keys: halves (0, 4) and (2, 6), with
// the factor 16, and (1, 5) and (3, 7).  A row is scaled by the power of two
// that brings its largest element into [2^10, 2^11), and has the sign of the
// scale.
template <int D, int NT>
constexpr int kQuerySets = (NT * D + kAttnThreads - 1) / kAttnThreads;  // rows of a thread

template <typename T, int D, int NT>
__device__ __forceinline__ void load_queries(const Kv4AttnArgs &k, const Kv4Seq &q, int head, int row0, int rows,
                                             T (&x)[kQuerySets<D, NT>][8]) {
  constexpr int PER = D / 8;  // threads of a row
#pragma unroll
  for (int set = 0; set < kQuerySets<D, NT>; ++set) {
    const int i = set * kAttnThreads + threadIdx.x, n = i / PER, r = row0 + n;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[set][e] = T(0.0f);
    if (n < 8 * NT && r < rows) {
      const int j = r / k.group_heads, h = head * k.group_heads + r % k.group_heads;
      const T *src = static_cast<const T *>(k.a.q) + (int64_t)(q.first + j) * k.a.q_token + h * k.a.q_head + i % PER * 8;
      if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
#pragma unroll
        for (int e = 0; e < (int)sizeof(T) / 2; ++e)
          reinterpret_cast<uint4 *>(x[set])[e] = reinterpret_cast<const uint4 *>(src)[e];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[set][e] = src[e];
      }
    }
  }
}

template <typename T, int D, int NG, int NT, int QS>
__device__ __forceinline__ void place_queries(const Kv4AttnArgs &k, int row0, int rows,
                                              const T (&x)[kQuerySets<D, NT>][8], char *smem) {
  using S = Kv4Smem<D, NG, NT, QS>;
  constexpr int PER = D / 8;      // threads of a row
  constexpr int W = D / 32 / NG;  // words of a group
  const float sign = k.a.scale < 0.0f ? -1.0f : k.a.scale == 0.0f ? 0.0f : 1.0f;
#pragma unroll
  for (int set = 0; set < kQuerySets<D, NT>; ++set) {
    const int i = set * kAttnThreads + threadIdx.x, n = i / PER, w = (i % PER) >> 2, t = i & 3, r = row0 + n;
    if (8 * NT * PER % kAttnThreads && n >= 8 * NT) break;  // whole warps
    float v[8];
    float top = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = kv4_load(&x[set][e]) * sign;
      top = fmaxf(top, fabsf(v[e]));
    }
#pragma unroll
    for (int o = 1; o < PER; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int power = top > 0.0f && isfinite(top) ? min(max(10 - ilogbf(top), -100), 120) : 0;
    const float up = ldexpf(1.0f, power);
    uint32_t part[QS][4];  // (0, 4) (1, 5) (2, 6) (3, 7)
    float sum[QS];
#pragma unroll
    for (int p = 0; p < QS; ++p) sum[p] = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float a = v[e] * up, b = v[e + 4] * up;
      const float f = e & 1 ? 1.0f : 16.0f;
#pragma unroll
      for (int p = 0; p < QS; ++p) {
        const float x = QS == 2 && p == 0 ? rintf(a) : a, y = QS == 2 && p == 0 ? rintf(b) : b;
        part[p][e] = pack_f16(x * f, y * f);
        const float2 h = unpack_f16(part[p][e]);
        sum[p] += (h.x + h.y) / f;
        a -= x;
        b -= y;
      }
    }
    const int at = (n & 7) * 4 + t, frag = ((n >> 3) * (D / 32) + w) * QS;
#pragma unroll
    for (int p = 0; p < QS; ++p) {
      reinterpret_cast<uint4 *>(smem + S::kQ + (frag + p) * 512)[at] =
          make_uint4(part[p][0], part[p][1], part[p][2], part[p][3]);
#pragma unroll
      for (int o = 1; o < 4 * W; o *= 2) sum[p] += __shfl_xor_sync(0xffffffffu, sum[p], o);
      if (t == 0 && w % W == 0) {  // codes + 8 stand for 2^-20 of their value; rows 2t, 2t + 1, twice
        float *c = reinterpret_cast<float *>(smem + S::kCorr) + (((n >> 3) * NG + w / W) * QS + p) * 16 +
                   (n & 7) / 2 * 4 + (n & 1);
        c[0] = c[2] = sum[p] * (-8.0f * 0x1p-20f);
      }
    }
    if (w == 0 && t == 0)  // not 0: times -inf, that would be NaN
      reinterpret_cast<float *>(smem + S::kFactor)[n] =
          r < rows && sign != 0.0f
              ? fmaxf(fabsf(k.a.scale) * 1.44269504088896341f * ldexpf(1.0f, 20 - power), 0x1p-126f)
              : 1.0f;
  }
}

// 8 codes of a word, + 8, as four f16 pairs (0, 4) (1, 5) (2, 6) (3, 7), times
// 2^-24, 2^-20, 2^-24, 2^-20.
__device__ __forceinline__ void key_pairs(uint32_t x, uint32_t (&a)[4]) {
  constexpr uint32_t L = 0x000F000Fu, H = 0x00F000F0u, FL = 0x00080008u, FH = 0x00800080u;
  const uint32_t x8 = x >> 8;
  a[0] = and_xor(x, L, FL);
  a[1] = and_xor(x, H, FH);
  a[2] = and_xor(x8, L, FL);
  a[3] = and_xor(x8, H, FH);
}

// The scores of two blocks' tokens, without the rows' factors: s[b][nt][0..3] of
// (token g, row 2t), (g, 2t + 1), (g + 8, 2t), (g + 8, 2t + 1) of block b,
// tokens as kv4_token has them.
template <int D, int NG, int NT, int QS>
__device__ __forceinline__ void block_scores(const char *buf, const char *smem, float (*s)[NT][4]) {
  using S = Kv4Smem<D, NG, NT, QS>;
  constexpr int W = D / 32 / NG;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, tok = kv4_token(g);
  uint32_t x[2][2][D / 32];
  float sc[2][2][NG];
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      lds<D / 8>(buf + b * S::kBlock + (tok + 8 * e) * (D / 2) + t * (D / 8), x[b][e]);
      load_scales<NG>(buf + b * S::kBlock + 8 * D + (tok + 8 * e) * 2 * NG, sc[b][e]);
    }
#pragma unroll
  for (int gr = 0; gr < NG; ++gr) {
    float acc[2][NT][QS][4];
    float4 start[NT][QS];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int p = 0; p < QS; ++p)
        start[nt][p] = reinterpret_cast<const float4 *>(smem + S::kCorr)[((nt * NG + gr) * QS + p) * 4 + t];
#pragma unroll
    for (int w = gr * W; w < (gr + 1) * W; ++w) {
      uint32_t q[NT][QS][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int p = 0; p < QS; ++p)
          lds<16>(smem + S::kQ + ((nt * (D / 32) + w) * QS + p) * 512 + lane * 16, q[nt][p]);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        uint32_t u[4], v[4];
        key_pairs(x[b][0][w], u);
        key_pairs(x[b][1][w], v);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int p = 0; p < QS; ++p) {
            if (w == gr * W)
              mma_f16_from(acc[b][nt][p], u[0], v[0], u[1], v[1], q[nt][p][0], q[nt][p][1], start[nt][p]);
            else
              mma_f16(acc[b][nt][p], u[0], v[0], u[1], v[1], q[nt][p][0], q[nt][p][1]);
            mma_f16(acc[b][nt][p], u[2], v[2], u[3], v[3], q[nt][p][2], q[nt][p][3]);
          }
      }
    }
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = QS == 2 ? acc[b][nt][0][e] + acc[b][nt][QS - 1][e] : acc[b][nt][0][e];
          s[b][nt][e] = gr ? fmaf(a, sc[b][e >> 1][gr], s[b][nt][e]) : a * sc[b][e >> 1][gr];
        }
  }
}

// Units of a sequence's work: those of one item, and how many items.  In a
// stretch over several items each begins with kItemUnits more, about the time
// that it takes to finish one item and begin another.
constexpr int kItemUnits = 3;

// (R rows to a row tile, UNIT tokens to a unit: powers of two.)
template <bool WEIGHTS, int R, int UNIT>
struct Kv4Units {
  int per, row_tiles, items;
  __device__ Kv4Units(const Kv4AttnArgs &k, const Kv4Seq &q) {
    const int rows = min(q.n_new, k.a.max_new) * k.group_heads;
    // the weights' pass takes all row tiles of a stretch of tokens together; without tokens it has nothing to do
    row_tiles = rows == 0 ? 0 : WEIGHTS ? 1 : (int)((unsigned)(rows + R - 1) / R);
    items = k.c.kv_heads * row_tiles;
    per = (int)((unsigned)(q.len + UNIT - 1) / UNIT);
    if (!WEIGHTS) per = max(per, 1);
  }
  __device__ int all() const { return (kItemUnits + per) * items; }
};

// Sum over the CTA, and over its threads before this one.
__device__ __forceinline__ int cta_scan(int v, int *total, int *shared) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int sum = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int n = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += n;
  }
  __syncthreads();
  if (lane == 31) shared[warp] = sum;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kAttnWarps; ++w) {
    if (w < warp) before += shared[w];
    all += shared[w];
  }
  *total = all;
  return before + sum - v;
}

// Joins the parts of CTAs first, first + step, .. (count of them) of the item
// that CTA c0 began: outputs x, maxima m and sums l of this thread's four
// elements of a row, I times (row and element by thread as in the kernel).
template <int D, int R, int I>
__device__ __forceinline__ void join_parts(const Kv4AttnArgs &k, int c0, int first, int count, int step,
                                           float4 (&x)[I], float (&m)[I], float (&l)[I]) {
  constexpr int B = I <= 2 ? kJoin : kJoin / 2;  // parts in flight
#pragma unroll
  for (int i = 0; i < I; ++i) {
    x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    m[i] = -INFINITY;
    l[i] = 0.0f;
  }
  for (int at = 0; at < count; at += B) {
    float4 y[I][B];
    float pm[I][B], pl[I][B];
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const int e = threadIdx.x + i * kAttnThreads, n = e / (D / 4), d = e % (D / 4) * 4;
        pm[i][b] = -INFINITY;
        pl[i][b] = 0.0f;
        y[i][b] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (at + b < count) {
          const int c = first + (at + b) * step;
          const float *in = kv4_partial(k, c, c == c0);
          pm[i][b] = __ldcg(in + R * D + n);
          pl[i][b] = __ldcg(in + R * D + R + n);
          y[i][b] = __ldcg(reinterpret_cast<const float4 *>(in + n * D + d));
        }
      }
#pragma unroll
    for (int i = 0; i < I; ++i) {
      float to = m[i];
#pragma unroll
      for (int b = 0; b < B; ++b) to = fmaxf(to, pm[i][b]);
      const float base = to == -INFINITY ? 0.0f : to, f = fast_exp2(m[i] - base);
      m[i] = to;
      l[i] *= f;
      x[i].x *= f, x[i].y *= f, x[i].z *= f, x[i].w *= f;
#pragma unroll
      for (int b = 0; b < B; ++b) {
        const float w = fast_exp2(pm[i][b] - base);
        l[i] = fmaf(pl[i][b], w, l[i]);
        x[i].x = fmaf(y[i][b].x, w, x[i].x);
        x[i].y = fmaf(y[i][b].y, w, x[i].y);
        x[i].z = fmaf(y[i][b].z, w, x[i].z);
        x[i].w = fmaf(y[i][b].w, w, x[i].w);
      }
    }
  }
}

// WEIGHTS: adds the attention weights of every token to the cache's, given the rows' lse.
template <typename T, int D, int NG, int NT, int QS, int PS, bool WEIGHTS>
__global__ void __launch_bounds__(kAttnThreads, kv4_ctas_per_sm(NT)) kv4_attention_kernel(const Kv4AttnArgs k) {
  using S = Kv4Smem<D, NG, NT, QS>;
  constexpr bool kWide = QS == 2;  // sums over tokens in f32 registers
  constexpr int R = 8 * NT, kStages = S::kStages, kTileBlocks = S::kTileBlocks, kTileTokens = kTileBlocks * kKv4Block;
  constexpr bool kFold = !kWide && !WEIGHTS;  // or there after every kFoldTiles tiles
  constexpr int kFoldTiles = kFoldProducts / (kTileBlocks * PS);
  constexpr int kUnitTokens = kv4_unit_tokens(NT, NG);
  using Units = Kv4Units<WEIGHTS, R, kUnitTokens>;
  extern __shared__ __align__(128) char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  int *share = reinterpret_cast<int *>(smem + S::kShare);

  char *ring = smem + warp * kStages * S::kStage;
  // This CTA's stretch of the units (the first `extra` CTAs have one more), and the sequence that it begins in; or,
  // where that takes no more than three units longer, one of the `parts` of one item: a stretch over two items costs
  // some three units' time between them.
  int ctas, first_unit, end_unit, each = 0, extra = 0, seq = k.b.n_seqs, seq_unit = 0, parts = 0, part = 0;
  const int cta = blockIdx.x;
  // The weights' pass reads no more than the first pass did (which waited for what came before it) until it needs lse;
  // every CTA waits once.
  if (!WEIGHTS) kv4_wait();
  auto end = [] {
    if (WEIGHTS) kv4_wait();
  };
  if (k.b.n_seqs <= 32) {  // every warp by itself, a sequence to a lane
    int per = 1, items = 0;
    if (lane < k.b.n_seqs) {
      const Units u(k, kv4_seq(k.b, lane, k.status));
      per = u.per, items = u.items;
    }
    auto scan = [&](int v) {
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int n = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += n;
      }
      return v;
    };
    const int upto_units = scan((kItemUnits + per) * items), total = __shfl_sync(0xffffffffu, upto_units, 31);
    if (total == 0) return end();
    int units = per * items;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) units += __shfl_xor_sync(0xffffffffu, units, o);
    ctas = min((int)gridDim.x, total);
    each = total / ctas, extra = total - each * ctas;
    // the shortest part that gives no more parts than CTAs: lane l counts those of candidate l % 4 in every eighth
    // sequence
    const int shortest = max((units + (int)gridDim.x - 1) / (int)gridDim.x, 1);
    int count = 0;
#pragma unroll
    for (int s = 0; s < 32; s += 8) {
      const int p = __shfl_sync(0xffffffffu, per, s + (lane >> 2)), n = __shfl_sync(0xffffffffu, items, s + (lane >> 2));
      if (s < k.b.n_seqs) count += n * ((p + shortest + (lane & 3) - 1) / (shortest + (lane & 3)));
    }
#pragma unroll
    for (int o = 4; o < 32; o *= 2) count += __shfl_xor_sync(0xffffffffu, count, o);
    const unsigned fits = __ballot_sync(0xffffffffu, lane < 4 && count <= (int)gridDim.x);
    if (fits) {
      const int most = shortest + __ffs(fits) - 1, pieces = (per + most - 1) / most;
      const int upto = scan(items * pieces), before = upto - items * pieces;
      const unsigned here = __ballot_sync(0xffffffffu, cta >= before && cta < upto);
      if (!here) return end();
      seq = __ffs(here) - 1;
      parts = __shfl_sync(0xffffffffu, pieces, seq);
      const int of = __shfl_sync(0xffffffffu, per, seq), at = cta - __shfl_sync(0xffffffffu, before, seq);
      const int item = at / parts;
      part = at - item * parts;
      seq_unit = __shfl_sync(0xffffffffu, upto_units - (kItemUnits + per) * items, seq);
      // even parts, the longer ones first
      const int short_part = of / parts, longer = of - short_part * parts;
      first_unit = seq_unit + item * (kItemUnits + of) + kItemUnits + short_part * part + min(part, longer);
      end_unit = first_unit + short_part + (part < longer);
    } else {
      if (cta >= ctas) return end();
      first_unit = each * cta + min(cta, extra);
      end_unit = first_unit + each + (cta < extra);
      const unsigned here = __ballot_sync(0xffffffffu, first_unit < upto_units);
      seq = __ffs(here) - 1;
      seq_unit = __shfl_sync(0xffffffffu, upto_units - (kItemUnits + per) * items, seq);
    }
  } else {
    int mine = 0, total = 0;
    for (int s = tid; s < k.b.n_seqs; s += kAttnThreads) mine += Units(k, kv4_seq(k.b, s, k.status)).all();
    const int before = cta_scan(mine, &total, share);
    ctas = min((int)gridDim.x, total);
    if (cta >= ctas) return end();
    each = total / ctas, extra = total - each * ctas;
    first_unit = each * cta + min(cta, extra);
    end_unit = first_unit + each + (cta < extra);
    __syncthreads();
    if (k.b.n_seqs <= kAttnThreads) {
      if (first_unit >= before && first_unit < before + mine) {
        share[0] = tid;
        share[1] = before;
      }
      __syncthreads();
      seq = share[0];
      seq_unit = share[1];
    } else {
      int passed = 0;
      for (int base = 0; base < k.b.n_seqs; base += kAttnThreads) {
        const int s = base + tid;
        const int u = s < k.b.n_seqs ? Units(k, kv4_seq(k.b, s, nullptr)).all() : 0;
        int some;
        const int at = passed + cta_scan(u, &some, share);
        if (first_unit >= passed + some) {
          passed += some;
          continue;
        }
        __syncthreads();
        if (first_unit >= at && first_unit < at + u) {
          share[0] = s;
          share[1] = at;
        }
        __syncthreads();
        seq = share[0];
        seq_unit = share[1];
        break;
      }
    }
  }

  for (int unit = first_unit; unit < end_unit && seq < k.b.n_seqs;) {
    const Kv4Seq q = kv4_seq(k.b, seq, nullptr);
    const Units units(k, q);
    if (unit >= seq_unit + units.all()) {
      seq_unit += units.all();
      ++seq;
      continue;
    }
    if (q.n_new > k.a.max_new && tid == 0) set_status(k.status, kStatusBadScale);
    const int rows = min(q.n_new, k.a.max_new) * k.group_heads;
    const int past = q.len - q.n_new + 1;  // tokens that the first new one sees
    // the part of one item that falls into the stretch
    const int with = kItemUnits + units.per, item = (unit - seq_unit) / with, item_unit = seq_unit + item * with;
    const int from = max(unit - item_unit - kItemUnits, 0), upto = min(end_unit - item_unit - kItemUnits, units.per);
    unit = upto > from ? item_unit + kItemUnits + upto : item_unit + with;
    if (upto <= from) continue;  // its work begins in the next stretch, or (weights of no tokens) it has none
    const int head = units.row_tiles == 1 ? item : item / units.row_tiles;
    const int first_tile = item - head * units.row_tiles;
    const int last_tile = WEIGHTS ? (rows - 1) / R : first_tile;

    for (int tile = first_tile; tile <= last_tile; ++tile) {
      const int row0 = tile * R;
      const int seen = min(max(past + (min(row0 + R, rows) - 1) / k.group_heads, 0), q.len);  // of the last row
      const int begin = from * kUnitTokens, end = min(upto * kUnitTokens, seen);
      const int tiles = max((end - begin + kTileTokens - 1) / kTileTokens, 0);
      const int count = (tiles - warp + kAttnWarps - 1) / kAttnWarps;  // this warp's; <= 0: none
      // A lane knows where one of the next 32 of this warp's tiles stands; where that tile is whole and within a page,
      // the same copies fetch it each time.
      constexpr int N = WEIGHTS ? S::kBlock / 2 : S::kBlock;  // of a block: its keys alone, or all
      constexpr int kShift = kTileBlocks == 4 ? 6 : 5;        // a page of 2^kShift tokens holds whole tiles
      int fetched = 0, pages[kTileBlocks];
      char *to = ring + lane * 16;
      const uint8_t *mine_at = nullptr;
      auto fetch = [&]() {
        if (fetched < count) {
          const int at = begin + (warp + fetched * kAttnWarps) * kTileTokens, mask = (1 << k.c.page_shift) - 1;
          if (!(fetched & 31)) {
            const int lane_at = at + lane * kAttnWarps * kTileTokens;
            pages[0] = 0;
            if (lane_at < end) pages[0] = max(kv4_page(k.c, k.b.table, k.b.table_stride, seq, lane_at, k.status), 0);
            mine_at = kv4_block(k.c, pages[0], head, lane_at & mask);
            if (k.c.page_shift < kShift) {
#pragma unroll
              for (int b = 1; b < kTileBlocks; ++b) {
                pages[b] = 0;
                if (lane_at + b * kKv4Block < end)
                  pages[b] =
                      max(kv4_page(k.c, k.b.table, k.b.table_stride, seq, lane_at + b * kKv4Block, k.status), 0);
              }
            }
          }
          const uint8_t *src = reinterpret_cast<const uint8_t *>(
                                   __shfl_sync(0xffffffffu, reinterpret_cast<uintptr_t>(mine_at), fetched & 31)) +
                               lane * 16;
          if (k.c.page_shift >= kShift && at + kTileTokens <= end) {
            constexpr int kPieces = WEIGHTS ? kTileBlocks : 1, kBytes = WEIGHTS ? N : S::kStage;
#pragma unroll
            for (int b = 0; b < kPieces; ++b)
#pragma unroll
              for (int c = 0; c < kBytes; c += 512)
                if (c + 512 <= kBytes || c + lane * 16 < kBytes)
                  copy16_async(to + b * S::kBlock + c, src + b * S::kBlock + c);
          } else {
#pragma unroll
            for (int b = 0; b < kTileBlocks; ++b) {
              if (at + b * kKv4Block >= end) break;
              const uint8_t *from = src + b * S::kBlock;
              if (k.c.page_shift < kShift)
                from = kv4_block(k.c, __shfl_sync(0xffffffffu, pages[b], fetched & 31), head,
                                 (at + b * kKv4Block) & mask) +
                       lane * 16;
#pragma unroll
              for (int c = 0; c < N; c += 512)
                if (c + 512 <= N || c + lane * 16 < N) copy16_async(to + b * S::kBlock + c, from + c);
            }
          }
          to = to + S::kStage == ring + lane * 16 + kStages * S::kStage ? ring + lane * 16 : to + S::kStage;
          ++fetched;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      T queries[kQuerySets<D, NT>][8];
      load_queries<T, D, NT>(k, q, head, row0, rows, queries);  // on their way while the pages are looked up
      for (int i = 0; i < kStages; ++i) fetch();

      if (WEIGHTS) {
        kv4_wait();
        __syncthreads();  // the previous rows' fragments have been read
      }
      place_queries<T, D, NG, NT, QS>(k, row0, rows, queries, smem);
      if (WEIGHTS && tid < R) {
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

      // In powers of two: top, the maximum of rows 2t, 2t + 1 at its last rise (limit: the score, without the row's
      // factor, at which it has to rise again), and base, what the exponentials refer to: top - lift, where 2^lift brings
      // the largest value scale into [2^10, 2^11), so that products with probabilities up to 2^4 stay below f16's
      // largest.  (lse in the weights' pass.)  Outputs and sums are both in units of 2^base.
      float factor[NT][2], base[NT][2], top[NT][2], limit[NT][2], sum[NT][2];
      int sees[NT][2];  // tokens that these rows see
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int n = nt * 8 + 2 * t + e, r = row0 + n;
          factor[nt][e] = reinterpret_cast<const float *>(smem + S::kFactor)[n];
          base[nt][e] = WEIGHTS ? reinterpret_cast<const float *>(smem + S::kLse)[n] : 0.0f;
          top[nt][e] = limit[nt][e] = -INFINITY;
          sum[nt][e] = 0.0f;
          sees[nt][e] = min(r < rows ? min(past + r / k.group_heads, q.len) : q.len, end);
        }
      const int all_see = min(past + row0 / k.group_heads, end);  // no mask below

      float o[NT][WEIGHTS ? 1 : D / 16][4];
      if constexpr (!WEIGHTS) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int m = 0; m < D / 16; ++m) o[nt][m][0] = o[nt][m][1] = o[nt][m][2] = o[nt][m][3] = 0.0f;
      }
      float lift = 0.0f;
      __half2 scale_limit = __floats2half2_rn(0.0f, 0.0f);  // value scales up to this one fit
      // The least value scale so far (a lane's own).  So far below the limit that its weights would lose bits that a result
      // of this type shows, each tile's weights have a power of two of their own (apart) from there on.
      __half2 least = __floats2half2_rn(INFINITY, INFINITY);
      constexpr float kApartFrom = QS == 2 ? 0x1p11f : PS == 2 ? 0x1p14f : 0x1p15f;
      auto too_small = [&] { return !__hbge2(__hmul2(least, __floats2half2_rn(kApartFrom, kApartFrom)), scale_limit); };

      // Sums of the tiles before, in units of 2^folded_base (volatile: in local memory, the registers are taken), and their
      // factor in units of 2^base, which has only risen.
      [[maybe_unused]] volatile float folded[WEIGHTS ? 1 : NT][WEIGHTS ? 1 : D / 16][4], folded_base[WEIGHTS ? 1 : NT][2];
      [[maybe_unused]] auto unfold = [&](int nt, int e) { return fast_exp2(folded_base[nt][e] - base[nt][e]); };
      bool has_folded = false;
      auto fold = [&] {
        if constexpr (!WEIGHTS) {
          const bool first = !has_folded;
          has_folded = true;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float f = first ? 0.0f : unfold(nt, e);
              folded_base[nt][e] = top[nt][e] == -INFINITY ? -INFINITY : base[nt][e];
#pragma unroll
              for (int m = 0; m < D / 16; ++m)
#pragma unroll
                for (int h = e; h < 4; h += 2) {
                  folded[nt][m][h] = first ? o[nt][m][h] : fmaf(folded[nt][m][h], f, o[nt][m][h]);
                  o[nt][m][h] = 0.0f;
                }
            }
        }
      };

      int i = 0, stage_out = 0;  // the tile and its place in the ring
      // Goes over the tile (and is true), or finds that it has to be gone over with weights apart.
      auto go_over = [&](auto weights_apart) {
        [[maybe_unused]] constexpr bool kApart = decltype(weights_apart)::value;
        const int at = begin + (warp + i * kAttnWarps) * kTileTokens;
        char *buf = ring + stage_out * S::kStage;
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        __syncwarp();  // every lane's copies are there
        float p[kTileBlocks][NT][4];
#pragma unroll
        for (int b = 0; b < kTileBlocks; b += 2) block_scores<D, NG, NT, QS>(buf + b * S::kBlock, smem, p + b);
        const bool whole = at + kTileTokens <= all_see;
        if (!whole) {
#pragma unroll
          for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (at + b * kKv4Block + kv4_token(g) + (e >> 1) * 8 >= sees[nt][e & 1]) p[b][nt][e] = -INFINITY;
        }

        if constexpr (WEIGHTS) {
#pragma unroll
          for (int b = 0; b < kTileBlocks; ++b) {
            float w[2] = {0.0f, 0.0f};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e >> 1] += fast_exp2(fmaf(p[b][nt][e], factor[nt][e & 1], -base[nt][e & 1]));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              w[e] += __shfl_xor_sync(0xffffffffu, w[e], 1);
              w[e] += __shfl_xor_sync(0xffffffffu, w[e], 2);
              const int tok = at + b * kKv4Block + kv4_token(g) + 8 * e;
              if (t == 0 && tok < end) {
                const int page = kv4_page(k.c, k.b.table, k.b.table_stride, seq, tok, nullptr);
                if (page >= 0)
                  k.c.weights[(((int64_t)page * k.c.kv_heads + head) << k.c.page_shift) +
                              (tok & ((1 << k.c.page_shift) - 1))] += w[e];
              }
            }
          }
        } else {
          // does a score exceed its row's limit, or a value scale what fits?
          bool rise = false;
          float m[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              m[nt][e] = fmaxf(p[0][nt][e], p[0][nt][e + 2]);
#pragma unroll
              for (int b = 1; b < kTileBlocks; ++b) m[nt][e] = fmaxf(m[nt][e], fmaxf(p[b][nt][e], p[b][nt][e + 2]));
              rise |= m[nt][e] > limit[nt][e];
            }
          if (!whole) {  // what stands behind the last token is not a scale: the tile's first token's in its place
            const __half *first = reinterpret_cast<const __half *>(buf + S::kBlock / 2 + 8 * D);
            for (int x = lane; x < kTileTokens; x += 32)
              if (at + x >= end)
                for (int gr = 0; gr < NG; ++gr)
                  reinterpret_cast<__half *>(buf + (x >> 4) * S::kBlock + S::kBlock / 2 + 8 * D)[(x & 15) * NG + gr] =
                      first[gr];
            __syncwarp();
          }
          __half2 h[kTileBlocks][2][(NG + 1) / 2], big = __floats2half2_rn(0.0f, 0.0f);
#pragma unroll
          for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const char *from = buf + b * S::kBlock + S::kBlock / 2 + 8 * D + (kv4_token(g) + 8 * e) * 2 * NG;
              if constexpr (NG == 1) {
                h[b][e][0] = __half2half2(*reinterpret_cast<const __half *>(from));
              } else {
                uint32_t w[NG / 2];
                lds<NG * 2>(from, w);
#pragma unroll
                for (int x = 0; x < NG / 2; ++x) h[b][e][x] = *reinterpret_cast<const __half2 *>(&w[x]);
              }
#pragma unroll
              for (int x = 0; x < (NG + 1) / 2; ++x) {
                big = __hmax2(big, h[b][e][x]);
                if (!kApart) least = __hmin2(least, h[b][e][x]);
              }
            }
          if (__any_sync(0xffffffffu, rise || !__hble2(big, scale_limit) || (!kApart && too_small()))) {
            float all = fmaxf(__low2float(big), __high2float(big));
#pragma unroll
            for (int x = 4; x < 32; x *= 2) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, x));
            float up = 0.0f;  // of lift
            if (all > __low2float(scale_limit)) {
              const int power = ilogbf(all);
              const float most = ldexpf(2.0f, power) * (1.0f - 0x1p-11f);
              scale_limit = __floats2half2_rn(most, most);
              up = (float)(10 - power) - lift;
              lift += up;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float x = m[nt][e] * factor[nt][e];
#pragma unroll
                for (int y = 4; y < 32; y *= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, y));
                x = fmaxf(x, top[nt][e]);
                // sums and outputs so far are in units of 2^(top - lift)
                const float f = x == -INFINITY ? 1.0f : fast_exp2(top[nt][e] - x + up);
                top[nt][e] = x;
                base[nt][e] = x == -INFINITY ? 0.0f : x - lift;
                limit[nt][e] = x == -INFINITY ? x : (x + 4.0f) / factor[nt][e];
                sum[nt][e] *= f;
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                  if constexpr (kApart) {
                    folded[nt][d][e] = folded[nt][d][e] * f;
                    folded[nt][d][e + 2] = folded[nt][d][e + 2] * f;
                  } else {
                    o[nt][d][e] *= f;
                    o[nt][d][e + 2] *= f;
                  }
                }
              }
            if (!kApart && __any_sync(0xffffffffu, too_small())) return false;
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                p[b][nt][e] = fast_exp2(fmaf(p[b][nt][e], factor[nt][e & 1], -base[nt][e & 1]));
                sum[nt][e & 1] += p[b][nt][e];
              }

          // value codes: a 32-bit word has this lane's pairs of four 16-element slices
          uint32_t v[kTileBlocks][4][D / 64];
#pragma unroll
          for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              lds<D / 16>(buf + b * S::kBlock + S::kBlock / 2 +
                              (kv4_token(2 * t + (e & 1)) + 8 * (e >> 1)) * (D / 2) + g * (D / 16),
                          v[b][e]);
          // the slice m of the 16 elements of a block's tokens, as an A operand
          auto value_slice = [&](int b, int m, uint32_t (&a)[4]) {
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
          };
          // the value scale of group gr, of token g (e = 0) or g + 8 of a block
          auto value_scale = [&](int b, int e, int gr) {
            constexpr int kTwo = NG > 1 ? 2 : 1;
            const __half2 pair = h[b][e][gr / kTwo];
            return gr % kTwo ? __high2float(pair) : __low2float(pair);
          };
          uint32_t ph[kTileBlocks][NT][2], pl[kTileBlocks][NT][2];
          // two tokens' weights as (one or two) f16 parts, rows and tokens exchanged
          auto place_weights = [&](int b, int nt, int e, float x0, float x1) {
            const uint32_t h = pack_f16(x0, x1);
            ph[b][nt][e] = transpose8x8(h);
            if (PS == 2) {
              const float2 r = unpack_f16(h);
              pl[b][nt][e] = transpose8x8(pack_f16(x0 - r.x, x1 - r.y));
            }
          };
          constexpr int M = D / 16 / NG;  // slices of a group
          if constexpr (!kApart) {
#pragma unroll
            for (int m = 0; m < D / 16; ++m) {
              if (m % M == 0) {
#pragma unroll
                for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    const float f = value_scale(b, e, m / M);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                      place_weights(b, nt, e, p[b][nt][2 * e] * f, p[b][nt][2 * e + 1] * f);
                  }
              }
              float acc[NT][4];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[nt][e] = kWide ? 0.0f : o[nt][m][e];
#pragma unroll
              for (int b = 0; b < kTileBlocks; ++b) {
                uint32_t a[4];
                value_slice(b, m, a);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  mma_f16(acc[nt], a[0], a[1], a[2], a[3], ph[b][nt][0], ph[b][nt][1]);
                  if (PS == 2) mma_f16(acc[nt], a[0], a[1], a[2], a[3], pl[b][nt][0], pl[b][nt][1]);
                }
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[nt][m][e] = kWide ? o[nt][m][e] + acc[nt][e] : acc[nt][e];
            }
          } else {
            // the tile's largest weight of a row and group in [2^13, 2^14), one slice and row tile after the other
            float down[2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int m = 0; m < D / 16; ++m) {
                if (m % M == 0) {
                  float up[2];
#pragma unroll
                  for (int r = 0; r < 2; ++r) {
                    float x = 0.0f;
#pragma unroll
                    for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
                      for (int e = 0; e < 2; ++e) x = fmaxf(x, p[b][nt][2 * e + r] * value_scale(b, e, m / M));
#pragma unroll
                    for (int y = 4; y < 32; y *= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, y));
                    const int power = x > 0.0f && isfinite(x) ? min(max(13 - ilogbf(x), -126), 126) : 0;
                    up[r] = ldexpf(1.0f, power);
                    down[r] = ldexpf(1.0f, -power);
                  }
#pragma unroll
                  for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                      const float f = value_scale(b, e, m / M);
                      place_weights(b, nt, e, p[b][nt][2 * e] * f * up[0], p[b][nt][2 * e + 1] * f * up[1]);
                    }
                }
                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int b = 0; b < kTileBlocks; ++b) {
                  uint32_t a[4];
                  value_slice(b, m, a);
                  mma_f16(acc, a[0], a[1], a[2], a[3], ph[b][nt][0], ph[b][nt][1]);
                  if (PS == 2) mma_f16(acc, a[0], a[1], a[2], a[3], pl[b][nt][0], pl[b][nt][1]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) folded[nt][m][e] = fmaf(acc[e], down[e & 1], folded[nt][m][e]);
              }
          }
        }
        return true;
      };
      auto done = [&] {  // with the tile
        __syncwarp();  // every lane has read the stage
        fetch();
        ++i;
        stage_out = stage_out + 1 == kStages ? 0 : stage_out + 1;
      };
      bool together = true;
      while (together && i < count) {
        for (const int turn = kFold ? min(i + kFoldTiles, count) : count; i < turn; done())
          if (!(together = go_over(std::false_type()))) break;
        if (together && i < count) fold();
      }
      if constexpr (!WEIGHTS) {
        if (!together) {
          fold();
          for (; i < count; done()) go_over(std::true_type());
        }
      }
      if constexpr (!WEIGHTS) {
        // The next kernel may be set up: not before, or its CTAs would take the places that the first CTAs to end leave,
        // some SMs more of them than others.
        if (unit >= end_unit) kv4_next();
        if (has_folded) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float f = unfold(nt, e);
#pragma unroll
              for (int m = 0; m < D / 16; ++m)
#pragma unroll
                for (int h = e; h < 4; h += 2)
                  o[nt][m][h] = together ? fmaf(folded[nt][m][h], f, o[nt][m][h]) : folded[nt][m][h];
            }
        }
        // join the warps: the ring is drained, each writes its part over it
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int x = 4; x < 32; x *= 2) sum[nt][e] += __shfl_xor_sync(0xffffffffu, sum[nt][e], x);
        __syncthreads();
        float *outs = reinterpret_cast<float *>(smem);  // [warp][row][D], then [warp][2][row]
        float *stat = outs + kAttnWarps * R * D;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int n = nt * 8 + 2 * t + e;
#pragma unroll
            for (int m = 0; m < D / 16; ++m)
              *reinterpret_cast<float2 *>(outs + (warp * R + n) * D + 16 * m + 2 * g) =
                  make_float2(o[nt][m][e], o[nt][m][e + 2]);
            if (g == 0) {
              stat[warp * 2 * R + n] = top[nt][e] == -INFINITY ? -INFINITY : base[nt][e];
              stat[warp * 2 * R + R + n] = sum[nt][e];
            }
          }
        __syncthreads();
        auto store = [&](int n, int d, float4 x, float m, float l) {
          const int r = row0 + n;
          const int64_t token = q.first + r / k.group_heads;
          const int h = head * k.group_heads + r % k.group_heads;
          const bool some = l > 0.0f || l != l;
          T *to = static_cast<T *>(k.a.out) + token * k.a.out_token + h * k.a.out_head + d;
          const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) kv4_store(to + e, some ? y[e] / l : 0.0f);
          if (d == 0 && k.a.lse)
            k.a.lse[token * k.a.q_heads + h] = some ? (m + log2f(l)) * 0.693147180559945309f : -INFINITY;
        };
        const bool ends = upto == units.per;
        float *out = kv4_partial(k, cta, from == 0);
        for (int i = tid; i < R * D / 4; i += kAttnThreads) {
          const int n = i / (D / 4), d = i % (D / 4) * 4;
          if (row0 + n >= rows) break;
          float m = stat[n];
#pragma unroll
          for (int w = 1; w < kAttnWarps; ++w) m = fmaxf(m, stat[w * 2 * R + n]);
          const float to = m == -INFINITY ? 0.0f : m;
          float l = 0.0f;
          float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
          for (int w = 0; w < kAttnWarps; ++w) {
            const float f = fast_exp2(stat[w * 2 * R + n] - to);
            l = fmaf(stat[w * 2 * R + R + n], f, l);
            const float4 y = *reinterpret_cast<const float4 *>(outs + (w * R + n) * D + d);
            x.x = fmaf(y.x, f, x.x);
            x.y = fmaf(y.y, f, x.y);
            x.z = fmaf(y.z, f, x.z);
            x.w = fmaf(y.w, f, x.w);
          }
          if (from == 0 && ends) {
            store(n, d, x, m, l);
          } else {
            *reinterpret_cast<float4 *>(out + n * D + d) = x;
            if (d == 0) {
              out[R * D + n] = m;
              out[R * D + R + n] = l;
            }
          }
        }
        if (from != 0 || !ends) {
          // the CTAs that the item's first and last unit fall to
          auto cta_of = [&](int u) {
            const int more = extra * (each + 1);
            return u < more ? u / (each + 1) : extra + (u - more) / each;
          };
          const int c0 = parts ? cta - part : cta_of(item_unit + kItemUnits);
          const int count_parts = parts ? parts : cta_of(item_unit + kItemUnits + units.per - 1) - c0 + 1;
          uint32_t *counters = static_cast<uint32_t *>(k.a.workspace);
          // whether this CTA is the last of `of` to arrive; all that the others wrote is then visible
          auto last_of = [&](uint32_t *counter, int of) {
            __syncthreads();
            if (tid == 0) {
              uint32_t before;  // with the barriers around it, for the whole CTA
              asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
              const bool last = before == (uint32_t)of - 1u;
              if (last) *counter = 0;
              share[0] = last;
            }
            __syncthreads();
            return share[0] != 0;
          };
          // few parts at once; more in groups (about as many as each has parts, these a multiple of what is loaded
          // together), whose results take the place of their first parts, and then these
          constexpr int I = R * D / 4 / kAttnThreads;
          float4 x[I];
          float m[I], l[I];
          const int join = (int)ceilf(sqrtf((float)count_parts) / kJoin) * kJoin;
          const int group = (cta - c0) / join, head_cta = c0 + group * join;
          const int in_group = min(join, count_parts - group * join), groups = (count_parts + join - 1) / join;
          bool last = last_of(counters + (group ? 2 : 1) * kAttnCtas + head_cta, in_group);
          if (last) join_parts<D, R, I>(k, c0, head_cta, in_group, 1, x, m, l);
          if (last && groups > 1) {
            float *to = kv4_partial(k, head_cta, head_cta == c0);
            __syncthreads();  // all have read the first part
#pragma unroll
            for (int i = 0; i < I; ++i) {
              const int e = tid + i * kAttnThreads, n = e / (D / 4), d = e % (D / 4) * 4;
              *reinterpret_cast<float4 *>(to + n * D + d) = x[i];
              if (d == 0) {
                to[R * D + n] = m[i];
                to[R * D + R + n] = l[i];
              }
            }
            last = last_of(counters + c0, groups);
            if (last) join_parts<D, R, I>(k, c0, c0, groups, join, x, m, l);
          }
          if (last) {
#pragma unroll
            for (int i = 0; i < I; ++i) {
              const int e = tid + i * kAttnThreads, n = e / (D / 4), d = e % (D / 4) * 4;
              if (row0 + n < rows) store(n, d, x[i], m[i], l[i]);
            }
          }
        }
        __syncthreads();  // the next copies come after these accesses of the ring
      }
    }
  }
  end();
}

template <typename T, int D, int NG, int NT, int QS, int PS, bool WEIGHTS>
cudaError_t launch_kv4_attention_pass(const Kv4AttnArgs &k, cudaStream_t stream, int device) {
  constexpr int bytes = Kv4Smem<D, NG, NT, QS>::kBytes;
  auto *f = kv4_attention_kernel<T, D, NG, NT, QS, PS, WEIGHTS>;
  static std::atomic<uint64_t> ready{0};  // devices on which the kernel may have that much shared memory
  const uint64_t bit = (uint64_t)1 << (device & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  return kv4_launch(f, dim3((unsigned)k.p.ctas), kAttnThreads, bytes, stream, k);
}

template <typename T, int D, int NG, int NT, int QS, int PS>
cudaError_t launch_kv4_attention_all(const Kv4AttnArgs &k, cudaStream_t stream, int device) {
  cudaError_t e = launch_kv4_attention_pass<T, D, NG, NT, QS, PS, false>(k, stream, device);
  if (e == cudaSuccess && k.a.accumulate) e = launch_kv4_attention_pass<T, D, NG, NT, QS, PS, true>(k, stream, device);
  return e;
}

// One translation unit per type: QS and PS as the precision note says.
template <typename T, int QS, int PS>
cudaError_t launch_kv4_attention_typed(const Kv4AttnArgs &k, cudaStream_t stream, int device) {
  const int key = k.c.head_dim * 100 + k.c.groups * 10 + k.p.rows_tile / 8;
  switch (key) {
#define KS_KV4_CASE(D, NG)                                                   \
  case D * 100 + NG * 10 + 1:                                                \
    return launch_kv4_attention_all<T, D, NG, 1, QS, PS>(k, stream, device);         \
  case D * 100 + NG * 10 + 2:                                                \
    return launch_kv4_attention_all<T, D, NG, 2, QS, PS>(k, stream, device);
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

cudaError_t launch_kv4_attention_f32(const Kv4AttnArgs &k, cudaStream_t stream, int device);
cudaError_t launch_kv4_attention_f16(const Kv4AttnArgs &k, cudaStream_t stream, int device);
cudaError_t launch_kv4_attention_bf16(const Kv4AttnArgs &k, cudaStream_t stream, int device);

}  // namespace ksb
