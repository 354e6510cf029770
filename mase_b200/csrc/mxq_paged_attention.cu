// Attention of one new token per sequence over a paged MX key/value cache (mxq_paged_attention):
//   s_j = scaling * <q, k_j>,  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m = max_j s_j.
// One pass over the cache with a running maximum and sum, split over the length and joined.
//
// A warp works on tiles of 16 cached tokens with m16n8k16 tensor-core products, both transposed so that the cache is the
// 16-row operand and the query heads of one key/value head are the 8 columns:
//   S^T[token, head] = K[token, d] Q^T[d, head]          rows = tokens, accumulated over head_dim
//   O^T[d, head]    += V^T[d, token] P^T[token, head]    rows = d, accumulated over the tokens of all tiles
// The order of the summed index of a product is free, and so is the order of the rows of O^T, so a lane's operands are
// pieces of up to 16 contiguous bytes of a row (four lanes share a key row, eight lanes a value row) and nothing is
// transposed in memory; Q^T and the output follow the same permutation.  Tiles reach shared memory by asynchronous copies
// in address order: a kernel of such copies and nothing else moves 6.7 TB/s, one whose lanes copy their own operand pieces 3.9.
//
// Codes become bf16 in registers: sign, exponent and fraction fields are moved to the bf16 positions with masks and
// shifts and the result is multiplied by one power of two (block scale times the difference of the exponent biases).
// Every value of every format has at most 8 significant bits, so this is exact, subnormal codes included.  bf16 queries
// are exact operands too; fp32 queries are split into three bf16 terms.  Probabilities are fp32 and enter the second
// product as two (fp32 queries: three) bf16 terms, 16 (24) significant bits, where the result keeps 8 (24); scores, maxima, sums
// and O^T are fp32.
//
// Bound: HBM in principle (2 g multiply-adds per cached byte of a group of g query heads), in practice the instructions
// that make bf16 of codes: 550 to 600 a tile of 16 x 128 one-byte codes, about 300 of them conversions; issue slots 63 % and the
// logic unit 55 % busy.  Measured (graph replays, join kernel included): sequences of 100001 and 131072 tokens, 8 heads of 128,
// MXINT8: 105 us, 4.7 TB/s (with the copies alone 84 us, 5.8 TB/s); 32 sequences of 1 to 8192, E4M3: 70 us, 4.1 TB/s; bf16 pages,
// 16 sequences of 777 to 2049, 32 heads of 64: 40 us, 4.6 TB/s.

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "mxq.h"
#include "mxq_common.cuh"
#include "mxq_internal.h"
#include "mxq_paged.cuh"

namespace mxq {
namespace paged {

constexpr int kWarps = 4;
constexpr int kTile = 16;                // cached tokens of a warp's tile
constexpr int kUnit = kWarps * kTile;    // tokens that a CTA takes at a time: the grain of the split
constexpr int kRowCost = 2;              // units that a row counts for beyond its tokens, 1 / 2 / 4: 32 sequences of 1 to 8192
                                         // tokens 75 / 70 / 68 us, 64 of 1 to 100 tokens 16.4 / 16.4 / 18.4, 16 of 777 to
                                         // 2049 in bf16 pages 40.3 / 39.8 / 40.6, append and 16 of 100 to 1023 18.5 / 20.5 / 19.8
__host__ __device__ constexpr int finish_threads(int w) { return w > 4 ? 32 * w : 128; }

struct AttnArgs {
  const void *q;
  void *out;
  int64_t q_stride_b, q_stride_h;
  float c_hi, c_lo;  // scaling * log2(e) in two terms
  int group;       // query heads per key/value head
  int q_heads;
  int head_tiles;  // tiles of 8 * NT query heads of a group
  int batch;
  const int32_t *lengths;
  int64_t most;    // tokens that tables (and weights) can hold
  int ctas;        // CTAs of the launch
  float *part_o;   // [ctas, 2, 8 * NT, dim]: unnormalised results of the rows a CTA shares with others
  float2 *part_ml; // [ctas, 2, 8 * NT]: their maximum and sum
  float2 *stats;   // [batch, q_heads] maximum and sum of rows of one CTA, when weights are accumulated
  float *scores;   // [batch, heads, head_tiles, tokens, score_heads] when weights are accumulated
  int64_t score_tokens;
  int score_heads; // heads of a tile that are kept: 2, 4, 8 or 16
  float *weights;
  int64_t weights_width;
  int *status;
};

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// ---- asynchronous copies into a warp's ring --------------------------------------------------------------------------
template <int kBytes>
__device__ __forceinline__ void copy_async(uint8_t *dst, const uint8_t *src) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(src), "n"(kBytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}
// kBytes (2, 4, 8 or 16) bytes of shared memory as words
template <int kBytes>
__device__ __forceinline__ void load_piece(const uint8_t *p, uint32_t *w) {
  if constexpr (kBytes == 16) {
    const uint4 r = *reinterpret_cast<const uint4 *>(p);
    w[0] = r.x, w[1] = r.y, w[2] = r.z, w[3] = r.w;
  } else if constexpr (kBytes == 8) {
    const uint2 r = *reinterpret_cast<const uint2 *>(p);
    w[0] = r.x, w[1] = r.y;
  } else if constexpr (kBytes == 4) {
    w[0] = *reinterpret_cast<const uint32_t *>(p);
  } else {
    w[0] = *reinterpret_cast<const uint16_t *>(p);
  }
}

template <int kFormat, int D>
struct Shape {
  static constexpr int kBits = Format<kFormat>::kBits;
  static constexpr int kRow = D * kBits / 8;                        // bytes of a row
  static constexpr int kKeyPiece = kRow / 4 < 16 ? kRow / 4 : 16;   // a lane's contiguous bytes of a key row
  static constexpr int kKeyPieces = kRow / 4 / kKeyPiece;
  static constexpr int kKeyWords = kKeyPiece / 4;
  static constexpr int kValPiece = kRow / 8 < 16 ? kRow / 8 : 16;   // and of a value row
  static constexpr int kValPieces = kRow / 8 / kValPiece;
  static constexpr int kValWords = (kValPiece + 3) / 4;
  static constexpr int kValElems = kValPiece * 8 / kBits;           // elements of a piece
  static constexpr int kPairs = kBits == 16 ? 1 : (kBits == 8 ? 2 : 4);  // bf16 pairs of a key word
  static constexpr int kScaleRow = kFormat == MXQ_CACHE_BF16 ? 0 : D / 32;  // scale bytes of a row
  // One stage of a warp's ring: the tile's key rows, its value rows, the scale bytes of both.  The rows of a tile are
  // contiguous in their page and are copied in order, 512 bytes an instruction; where they land is permuted in units of
  // 16 (keys) or 32 bytes inside each 128-byte line, so that the lanes' reads (below) hit every bank once.
  static constexpr int kSide = kTile * kRow;
  static constexpr int kScaleBytes = kTile * kScaleRow;
  static constexpr int kStage = 2 * kSide + 2 * kScaleBytes;
  // where byte `byte` of a token's row lies in the stage
  static __device__ __forceinline__ int key_slot(int token, int byte) {
    return token * kRow + byte ^ (kRow >= 128 ? (token & 1) << 6 : 0);
  }
  static __device__ __forceinline__ int value_slot(int token, int byte) {
    return token * kRow + byte ^ (kRow >= 32 ? ((token >> 1) & 3) << 5 : 0);
  }
  // the parts of a slot's permutation that a copy at byte i (a multiple of 512) of the tile adds to that of byte 0
  static __host__ __device__ constexpr int key_turn(int i) { return kRow == 512 ? ((i >> 9) & 1) << 6 : 0; }
  static __host__ __device__ constexpr int value_turn(int i) {
    return kRow == 128 ? ((i >> 8) & 3) << 5 : (kRow == 256 ? ((i >> 9) & 3) << 5 : (kRow == 512 ? ((i >> 10) & 3) << 5 : 0));
  }
  static constexpr int kStages = kRow <= 64 ? 4 : 2;  // three for rows of 128 bytes: 106 us against 105 (100001 + 131072 MXINT8)
};
// element (0 .. D-1) that half `half` of pair i of key word w of piece c of lane t holds
template <int kFormat, int D>
__device__ __forceinline__ int key_element(int c, int w, int i, int half, int t) {
  using S = Shape<kFormat, D>;
  return (c * 4 * S::kKeyPiece + t * S::kKeyPiece + w * 4) * 8 / S::kBits + pair_element<kFormat>(i, half);
}
// element that entry e (0 .. D/8 - 1) of value lane r holds
template <int kFormat, int D>
__device__ __forceinline__ int value_element(int e, int r) {
  using S = Shape<kFormat, D>;
  const int c = e / S::kValElems;
  return (c * 8 + r) * S::kValElems + e % S::kValElems;
}

__device__ __forceinline__ float load_q(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_q(const float *p) { return *p; }
__device__ __forceinline__ float bf16_of(float v) { return __bfloat162float(__float2bfloat16_rn(v)); }

// Scores are kept in units of log2: x_j = scaling * log2(e) * <q, k_j>, and the softmax is 2^(x_j - m) / sum.
// A tile raises the reference m only when a score exceeds it by more than kSlack: probabilities then stay below 2^11.5
// and the rescaling (shuffles, D/4 products) runs a few times per warp instead of once per tile.
constexpr float kSlack = 11.5f;
constexpr float kLowest = -3.0e38f;  // m before the first score: finite, so that no difference is inf - inf

__device__ __forceinline__ float exp2_fast(float x) {  // results below 2^-126 become 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Which tile a warp works on, for the few uses that need to know.
struct Place {
  int b, row, rows, tok;
  __device__ __forceinline__ int64_t score_row(const AttnArgs &a) const {
    return ((int64_t)b * rows + row) * a.score_tokens + tok;
  }
};

template <typename T, int kFormat, int D, int NT>
struct Worker {
  using S = Shape<kFormat, D>;
  int key_at[2], value_at[2];  // where the lane reads: key pieces of even and odd number, value rows 2t and 2t + 1
  static constexpr int kTerms = Elem<T>::kBf16 ? 1 : 3;   // bf16 terms of a query element
  static constexpr int kPTerms = Elem<T>::kBf16 ? 2 : 3;  // and of a probability
  static constexpr int kSteps = D / 16;
  uint32_t q[kTerms][kSteps][NT][2];
  float o[kSteps][NT][4];
  float m[NT][2], l[NT][2];

  __device__ __forceinline__ void setup(int lane) {
    const int t = lane & 3, r = lane >> 2;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      key_at[x] = S::key_slot(r, x * 64 + t * S::kKeyPiece);
      value_at[x] = S::value_slot(2 * t + x, r * S::kValPiece);
    }
  }
  __device__ __forceinline__ void load_query(const T *qrow, int64_t stride_h, int heads, int lane) {
    const int t = lane & 3, head = lane >> 2;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const bool live = n * 8 + head < heads;
      const T *row = qrow + (int64_t)(n * 8 + head) * stride_h;
#pragma unroll
      for (int p = 0; p < kSteps * 2; ++p) {  // pair p of this lane's key pieces
        const int w = p / S::kPairs, c = w / S::kKeyWords;
        float v[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          v[h] = live ? load_q(row + key_element<kFormat, D>(c, w % S::kKeyWords, p % S::kPairs, h, t)) : 0.f;
#pragma unroll
        for (int x = 0; x < kTerms; ++x) {
          q[x][p / 2][n][p & 1] = pack_bf16x2(v[0], v[1]);
          v[0] -= bf16_of(v[0]), v[1] -= bf16_of(v[1]);
        }
      }
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int h = 0; h < 2; ++h) m[n][h] = kLowest, l[n][h] = 0.f;
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][n][i] = 0.f;
    }
  }

  // x - m in units of log2; fp32 queries take the factor scaling * log2(e) with 48 bits (an infinite score only the first term:
  // the second one may be zero or of the other sign)
  static __device__ __forceinline__ float score(float s, float c_hi, float c_lo, float m) {
    const float x = fmaf(s, c_hi, -m);
    return Elem<T>::kBf16 || fabsf(x) == INFINITY ? x : fmaf(s, c_lo, x);
  }

  // One tile from a stage of the ring; `live` tokens of it exist.
  template <bool kRare>
  __device__ __forceinline__ void tile(const uint8_t *stage, int live, int bits, const AttnArgs &a, const Place &at, int lane) {
    const float c_hi = a.c_hi, c_lo = a.c_lo;
    const int t = lane & 3, r = lane >> 2;
    const int offset = raw_offset<kFormat>(bits);
    // Two chains of products, even and odd steps, and for fp32 queries one of their lower terms: the tensor cores cut off what
    // lies below the last bit of the larger summand, which the small terms would only multiply.
    float s[NT][4], s_odd[NT][4], s_low[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = s_odd[n][i] = s_low[n][i] = 0.f;
#pragma unroll
    for (int c = 0; c < S::kKeyPieces; ++c) {
      uint32_t pairs[2][S::kKeyWords * S::kPairs];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t f = 0, rest = 0, kk[S::kKeyWords];
        if constexpr (kFormat != MXQ_CACHE_BF16) {
          const uint32_t b = stage[2 * S::kSide + (r + 8 * h) * S::kScaleRow +
                                   (((c * 4 + t) * S::kKeyPiece * 8 / S::kBits) >> 5)];
          f = kRare ? rare_factor<kFormat>(b, offset) * 0x00010001u : b * 0x00800080u + (uint32_t)offset * 0x00800080u;
          if (kRare) rest = rare_rest<kFormat>(b, offset) * 0x00010001u;
        }
        load_piece<S::kKeyPiece>(stage + key_at[c & 1] + h * 8 * S::kRow + (c >> 1) * 128, kk);
#pragma unroll
        for (int w = 0; w < S::kKeyWords; ++w) key_word<kFormat, kRare>(kk[w], f, rest, &pairs[h][w * S::kPairs]);
      }
      constexpr int kStepsHere = S::kKeyWords * S::kPairs / 2;
#pragma unroll
      for (int k = 0; k < kStepsHere; ++k) {
        const uint32_t rows[4] = {pairs[0][2 * k], pairs[1][2 * k], pairs[0][2 * k + 1], pairs[1][2 * k + 1]};
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int z = kTerms - 1; z >= 0; --z)
            mma(z > 0 ? s_low[n] : ((c * kStepsHere + k) & 1 ? s_odd[n] : s[n]), rows, q[z][c * kStepsHere + k][n][0],
                q[z][c * kStepsHere + k][n][1]);
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float high = s[n][i] + s_odd[n][i];  // of the first terms
        // an infinite key has this score; the lower terms, zero or of the other sign, would make it NaN
        s[n][i] = kTerms == 1 || fabsf(high) == INFINITY ? high : s[n][i] + (s_odd[n][i] + s_low[n][i]);
      }
    // rows: tokens r (entries 0, 1) and r + 8 (2, 3); columns: heads 2t, 2t + 1
    float x[NT][4], top = kLowest;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[n][i] = score(s[n][i], c_hi, c_lo, m[n][i & 1]);
    if (live < kTile) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (r + 8 * (i >> 1) >= live) x[n][i] = -INFINITY;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, x[n][i]);
    if (a.scores != nullptr) {
      float *scores = a.scores + at.score_row(a) * a.score_heads;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (r + 8 * h < live && n * 8 + 2 * t < a.score_heads)
            *reinterpret_cast<float2 *>(scores + (r + 8 * h) * a.score_heads + n * 8 + 2 * t) =
                make_float2(score(s[n][2 * h], c_hi, c_lo, 0.f), score(s[n][2 * h + 1], c_hi, c_lo, 0.f));
    }
    if (__any_sync(0xFFFFFFFFu, top > kSlack)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float y[2], high = m[n][h];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            y[i] = r + 8 * i < live ? score(s[n][2 * i + h], c_hi, c_lo, 0.f) : -INFINITY;
            high = fmaxf(high, y[i]);
          }
#pragma unroll
          for (int z = 4; z < 32; z <<= 1) high = fmaxf(high, __shfl_xor_sync(0xFFFFFFFFu, high, z));
          const float f = exp2_fast(m[n][h] - high);
          m[n][h] = high, l[n][h] *= f;
#pragma unroll
          for (int i = 0; i < 2; ++i)
            x[n][2 * i + h] = r + 8 * i < live ? score(s[n][2 * i + h], c_hi, c_lo, high) : -INFINITY;
#pragma unroll
          for (int j = 0; j < kSteps; ++j) o[j][n][h] *= f, o[j][n][2 + h] *= f;
        }
    }
    uint32_t pb[kPTerms][NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = exp2_fast(x[n][i]);
        l[n][i & 1] += p[i];
      }
#pragma unroll
      for (int z = 0; z < kPTerms; ++z)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t pair = pack_bf16x2(p[2 * h], p[2 * h + 1]);
          pb[z][n][h] = transpose8x8(pair);
          if (z + 1 < kPTerms)
            p[2 * h] -= __uint_as_float(pair << 16), p[2 * h + 1] -= __uint_as_float(pair & 0xFFFF0000u);
        }
    }
#pragma unroll
    for (int c = 0; c < S::kValPieces; ++c) {
      uint32_t f[2] = {0, 0}, rest[2] = {0, 0}, vv[4][S::kValWords];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        load_piece<S::kValPiece>(stage + S::kSide + value_at[i & 1] + 8 * (i >> 1) * S::kRow + c * 128, vv[i]);
      }
      if constexpr (kFormat != MXQ_CACHE_BF16) {
        uint32_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          b[i] = stage[2 * S::kSide + S::kScaleBytes + (2 * t + (i & 1) + 8 * (i >> 1)) * S::kScaleRow +
                       (((c * 8 + r) * S::kValPiece * 8 / S::kBits) >> 5)];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (kRare) {
            f[h] = rare_factor<kFormat>(b[2 * h], offset) | rare_factor<kFormat>(b[2 * h + 1], offset) << 16;
            rest[h] = rare_rest<kFormat>(b[2 * h], offset) | rare_rest<kFormat>(b[2 * h + 1], offset) << 16;
          } else {
            f[h] = b[2 * h] * 128u + (b[2 * h + 1] * (128u << 16) + (uint32_t)offset * 0x00800080u);
          }
          // a token behind the last one has factor 0: whatever its slot holds, it adds nothing
          if (live < kTile) {
            if (2 * t + 8 * h >= live) f[h] = 0;
            else if (2 * t + 8 * h + 1 >= live) f[h] &= 0xFFFFu;
          }
        }
      }
      constexpr int kPerWord = 32 / S::kBits;
#pragma unroll
      for (int w = 0; w < S::kValWords; ++w) {
        uint32_t e[2][kPerWord];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t v0 = vv[2 * h][w], v1 = vv[2 * h + 1][w];
          if constexpr (kFormat == MXQ_CACHE_BF16) {
            if (2 * t + 8 * h >= live) v0 = 0;
            if (2 * t + 8 * h + 1 >= live) v1 = 0;
          }
          value_words<kFormat, kRare>(v0, v1, f[h], rest[h], e[h]);
        }
        constexpr int kHere = S::kValElems < kPerWord ? S::kValElems : kPerWord;
#pragma unroll
        for (int k = 0; k < kHere; k += 2) {
          const int j = (c * S::kValElems + w * kPerWord + k) / 2;
          const uint32_t rows[4] = {e[0][k], e[0][k + 1], e[1][k], e[1][k + 1]};
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if constexpr (Elem<T>::kBf16) {
#pragma unroll
              for (int z = kPTerms - 1; z >= 0; --z) mma(o[j][n], rows, pb[z][n][0], pb[z][n][1]);
            } else {  // a tile's sum by itself, added with rounding: no cut-off at the size of O^T, tile after tile
              float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int z = kPTerms - 1; z >= 0; --z) mma(part, rows, pb[z][n][0], pb[z][n][1]);
#pragma unroll
              for (int i = 0; i < 4; ++i) o[j][n][i] += part[i];
            }
          }
        }
      }
    }
  }
};

// ---- split ---------------------------------------------------------------------------------------------------------------
// The rows of a launch are (sequence, key/value head, head tile), each a run of units of kUnit tokens (at least one) and
// kRowCost empty units, which stand for what beginning and ending a row costs.  The units of all rows in order are divided
// evenly between the CTAs, whatever the lengths are: with total = q * ctas + r, CTA i takes q or (i < r) q + 1 of them.
// A row inside one CTA is finished there; of a row that several CTAs share each leaves an unnormalised part with its
// maximum and sum, and the finish kernel joins them in the order of the CTAs.  A CTA shares at most its first and its
// last row, so there are two part slots per CTA.
struct Split {
  int64_t q, r;
  __device__ __forceinline__ Split(int64_t total, int64_t ctas) {
    if (total <= UINT32_MAX)
      q = (uint32_t)total / (uint32_t)ctas, r = (uint32_t)total % (uint32_t)ctas;
    else
      q = total / ctas, r = total % ctas;
  }
  __device__ __forceinline__ int64_t start(int64_t i) const { return i * q + min(i, r); }
  __device__ __forceinline__ int64_t cta_of(int64_t u) const {  // the CTA that takes unit u
    const int64_t longer = r * (q + 1), n = u < longer ? u : u - longer, d = u < longer ? q + 1 : q;
    return (u < longer ? 0 : r) + (n <= UINT32_MAX && d <= UINT32_MAX ? (uint32_t)n / (uint32_t)d : n / d);
  }
};
__device__ __forceinline__ int length_of(const AttnArgs &a, int b) { return clamp_length(a.lengths[b], a.most, a.status); }
__device__ __forceinline__ int work_of_length(int n) { return max(1, (n + kUnit - 1) / kUnit); }
__device__ __forceinline__ int units_of_length(int n) { return work_of_length(n) + kRowCost; }
__device__ __forceinline__ int warp_sum(int v) {
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, x);
  return v;
}
// units (of one row each) of the sequences first .. end - 1; called by whole warps
__device__ __forceinline__ int64_t units_between(const AttnArgs &a, int first, int end, int lane) {
  int64_t sum = 0;
  for (int b0 = first; b0 < end; b0 += 32)
    sum += warp_sum(b0 + lane < end ? units_of_length(length_of(a, b0 + lane)) : 0);
  return sum;
}
// the sequence that holds unit `target` of the concatenated sequences, and the units before it
__device__ __forceinline__ int sequence_at(const AttnArgs &a, int64_t target, int lane, int64_t &before) {
  int64_t base = 0;
  for (int b0 = 0;; b0 += 32) {
    const int n = b0 + lane < a.batch ? units_of_length(length_of(a, b0 + lane)) : 0;
    int s = n;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const int y = __shfl_up_sync(0xFFFFFFFFu, s, x);
      if (lane >= x) s += y;
    }
    const uint32_t past = __ballot_sync(0xFFFFFFFFu, base + s > target);
    if (past != 0 || b0 + 32 >= a.batch) {
      const int k = past != 0 ? __ffs(past) - 1 : 0;
      before = base + __shfl_sync(0xFFFFFFFFu, s - n, k);
      return min(b0 + k, a.batch - 1);
    }
    base += __shfl_sync(0xFFFFFFFFu, s, 31);
  }
}

// Place of a unit in the rows.
struct Cursor {
  int b, row, unit, units, length;
  // to the next unit; `more`: there is one
  __device__ __forceinline__ void advance(const AttnArgs &a, int rows, bool more) {
    if (++unit < units) return;
    unit = 0;
    if (++row < rows) return;
    row = 0;
    if (more) length = length_of(a, ++b), units = units_of_length(length);
  }
};

template <int kFormat, int D, int NT>
struct Smem {
  static constexpr int kRing = kWarps * Shape<kFormat, D>::kStages * Shape<kFormat, D>::kStage;
  static constexpr int kJoin = kWarps * 8 * NT * (D + 2) * 4;
  static constexpr int kTotal = kRing + kJoin;
};

// Any of the four scale bytes outside of the plain range of factors?
template <int kFormat>
__device__ __forceinline__ bool any_rare(uint32_t w, int bits) {
  const uint32_t low = w & 0x7F7F7F7Fu;
  if constexpr (kFormat == MXQ_CACHE_INT8) {
    const uint32_t small = ~((low + (uint32_t)(128 - bits) * 0x01010101u) | w);  // byte < bits
    return ((small | ((low + 0x01010101u) & w)) & 0x80808080u) != 0;             // or byte == 255
  } else {
    const uint32_t limit = 254 - raw_offset<kFormat>(0);  // 128 .. 142: rare above it
    return ((low + (255u - limit) * 0x01010101u) & w & 0x80808080u) != 0;
  }
}

// Three CTAs per SM where the registers would allow two: 105 us on 100001 + 131072 MXINT8 tokens; two 119; four spill, 111.
template <typename T, int kFormat, int D, int NT>
__global__ void __launch_bounds__(kWarps * 32, Elem<T>::kBf16 && D == 128 && NT == 1 ? 3 : 1)
attention_kernel(const Cache c, const Table table, const AttnArgs a) {
  using S = Shape<kFormat, D>;
  constexpr int kHeads = 8 * NT;
  extern __shared__ __align__(128) uint8_t smem[];
  float *sm_o = reinterpret_cast<float *>(smem + Smem<kFormat, D, NT>::kRing);  // [kWarps][kHeads * D / 32][32]
  float *sm_m = sm_o + kWarps * kHeads * D, *sm_l = sm_m + kWarps * kHeads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = lane & 3, r = lane >> 2;
  uint8_t *ring = smem + warp * (S::kStages * S::kStage);

  wait_for_previous();
  const int rows = c.heads * a.head_tiles;
  const int64_t total = units_between(a, 0, a.batch, lane) * rows;
  const int64_t ctas = min((int64_t)a.ctas, total);
  if (blockIdx.x >= ctas) return;
  const Split split(total, ctas);
  const int64_t begin = split.start(blockIdx.x);
  const int todo = (int)(split.start(blockIdx.x + 1) - begin);  // the host bounds the units of a launch
  Cursor here;  // the unit being worked on
  {
    int64_t before;
    const int64_t target = total <= UINT32_MAX ? (uint32_t)begin / (uint32_t)rows : begin / rows;
    here.b = sequence_at(a, target, lane, before);
    here.length = length_of(a, here.b), here.units = units_of_length(here.length);
    const int64_t in_seq = begin - before * rows;
    here.row = (int)(in_seq <= UINT32_MAX ? (uint32_t)in_seq / (uint32_t)here.units : in_seq / here.units);
    here.unit = (int)(in_seq - (int64_t)here.row * here.units);
  }

  // Where the warp's tiles lie is worked out for 32 units at a time, one per lane: `place` is the offset of the
  // lane's tile (of the batch of units in use) from the start of the pages in units of 16 bytes, `entry` and `entry_off` are the page table
  // entry and the offset inside the page for the batch after it, whose loads have 32 units of time to arrive.
  Cursor ahead = here;  // first unit of the batch that is looked up next
  int looked_up = 0;    // units looked up
  int entry = 0;
  uint32_t entry_off = 0;
  uint32_t place = 0;
  constexpr uint32_t kNoTile = 0xFFFFFFFFu;
  const uint32_t page_bytes = (uint32_t)(c.heads << c.page_log2) * S::kRow;  // below 2^32: at most 32767 heads
  auto look_up = [&]() {
    Cursor mine = ahead;
    int64_t pos = (int64_t)mine.row * mine.units + mine.unit + lane;  // place in the units of all rows of the sequence
    const bool any = looked_up + lane < todo;
    while (any && pos >= (int64_t)rows * mine.units) {
      pos -= (int64_t)rows * mine.units;
      mine.length = length_of(a, ++mine.b), mine.units = units_of_length(mine.length);
    }
    if (any) {
      mine.row = (int)(pos <= UINT32_MAX ? (uint32_t)pos / (uint32_t)mine.units : pos / mine.units);
      mine.unit = (int)(pos - (int64_t)mine.row * mine.units);
    }
    const int tok = mine.unit * kUnit + warp * kTile;
    entry_off = kNoTile;
    if (any && tok < mine.length) {
      entry = table.entries[mine.b * table.stride + (tok >> c.page_log2)];
      const int head = a.head_tiles == 1 ? mine.row : mine.row / a.head_tiles;
      entry_off = (uint32_t)((head << c.page_log2) + (tok & ((1 << c.page_log2) - 1))) * S::kRow;
    }
    looked_up += 32;
    if (looked_up < todo) {  // every lane had a unit: go on behind the last one
      ahead.b = __shfl_sync(0xFFFFFFFFu, mine.b, 31), ahead.row = __shfl_sync(0xFFFFFFFFu, mine.row, 31);
      ahead.unit = __shfl_sync(0xFFFFFFFFu, mine.unit, 31), ahead.units = __shfl_sync(0xFFFFFFFFu, mine.units, 31);
      ahead.length = __shfl_sync(0xFFFFFFFFu, mine.length, 31);
      ahead.advance(a, rows, true);
    }
  };
  auto settle = [&]() {
    place = kNoTile;
    if (entry_off != kNoTile) {
      if (entry < 0 || entry >= c.pages)
        report(a.status);
      else
        place = (uint32_t)(((uint64_t)(uint32_t)entry * page_bytes + entry_off) >> 4);  // the host bounds it
    }
  };
  const int key_to = S::key_slot(lane * 16 / S::kRow, lane * 16 % S::kRow);
  const int value_to = S::value_slot(lane * 16 / S::kRow, lane * 16 % S::kRow);
  const uint8_t *k_base = c.codes[0] + lane * 16, *v_base = c.codes[1] + lane * 16;
  // scale bytes: 4 to a lane, first those of the key rows, then those of the value rows (head_dim 256: one after the other)
  constexpr int kScaleWords = 4 * S::kScaleRow;  // of one side
  const bool value_scales = kScaleWords < 32 && lane >= kScaleWords;
  const uint8_t *s_base = (value_scales ? c.scales[1] : c.scales[0]) + (lane - (value_scales ? kScaleWords : 0)) * 4;
  const int64_t to_value_scales = c.scales[1] - c.scales[0];
  auto copy_scales = [&](uint8_t *dst, const uint8_t *sp) {
    if constexpr (kScaleWords == 32) {
      copy_async<4>(dst + lane * 4, sp), copy_async<4>(dst + S::kScaleBytes + lane * 4, sp + to_value_scales);
    } else {
      if (lane < 2 * kScaleWords) copy_async<4>(dst + lane * 4, sp);
    }
  };
  uint32_t absent = 0;  // bit s: the tile in stage s does not exist
  auto issue = [&](int unit, int stage) {  // copies the warp's tile of a unit of the batch in use
    const uint32_t off = __shfl_sync(0xFFFFFFFFu, place, unit & 31);
    if (off != kNoTile) {
      absent &= ~(1u << stage);
      uint8_t *dst = ring + stage * S::kStage;
      const uint8_t *kp = k_base + (uint64_t)off * 16, *vp = v_base + (uint64_t)off * 16;
#pragma unroll
      for (int i = 0; i < S::kSide; i += 512)
        if (S::kSide % 512 == 0 || lane * 16 < S::kSide) {
          copy_async<16>(dst + i + (key_to ^ S::key_turn(i)), kp + i);
          copy_async<16>(dst + S::kSide + i + (value_to ^ S::value_turn(i)), vp + i);
        }
      if constexpr (kFormat != MXQ_CACHE_BF16) {
        constexpr int kScalesPer16 = 16 * 8 / S::kBits;  // elements of 16 code bytes; one scale byte for 32
        const uint8_t *sp = s_base + (kScalesPer16 == 32 ? (uint64_t)off : (uint64_t)(off >> 1));
        copy_scales(dst + 2 * S::kSide, sp);
      }
    } else {
      absent |= 1u << stage;
    }
    copy_commit();
  };

  look_up();
  settle();
  if (looked_up < todo) look_up();
#pragma unroll
  for (int k = 0; k < S::kStages - 1; ++k) {
    if (k < todo)
      issue(k, k);
    else
      copy_commit();
  }

  auto tile_of_head = [&](const Cursor &at, int &first_head, int &heads) {
    const int head = a.head_tiles == 1 ? at.row : at.row / a.head_tiles, ht = at.row - head * a.head_tiles;
    first_head = head * a.group + ht * kHeads, heads = min(a.group - ht * kHeads, kHeads);
  };
  Worker<T, kFormat, D, NT> w;
  int first_head, heads;
  auto load_query = [&](const Cursor &at, int first, int n) {
    w.load_query(static_cast<const T *>(a.q) + at.b * a.q_stride_b + first * a.q_stride_h, a.q_stride_h, n, lane);
  };
  w.setup(lane);
  w.clear();
  tile_of_head(here, first_head, heads);
  load_query(here, first_head, heads);
  int from = 0, from_unit = here.unit;  // where the CTA's part of the row begins: in its own units, in the row's
  bool joined = false;
  for (int i = 0, stage = 0; i < todo; ++i) {
    copy_wait<S::kStages - 2>();
    __syncwarp();  // the scale bytes were copied by other lanes; and all lanes are done with the stage before this one
    const int fill = i + S::kStages - 1;
    if (fill < todo) {
      if ((fill & 31) == 0) {
        settle();
        if (looked_up < todo) look_up();
      }
      issue(fill, stage == 0 ? S::kStages - 1 : stage - 1);
    } else {
      copy_commit();
    }
    const int work = here.units - kRowCost;
    const int tok = here.unit * kUnit + warp * kTile;
    const int live = here.length - tok;
    if ((absent >> stage) & 1u) {  // behind the end, or the page does not exist: its tokens are left out
      if (a.scores != nullptr) {
        float *sc = a.scores + Place{here.b, here.row, rows, tok}.score_row(a) * a.score_heads;
        for (int j = lane; j < min(live, kTile) * a.score_heads; j += 32) sc[j] = -INFINITY;
      }
    } else {
      const uint8_t *st = ring + stage * S::kStage;
      bool rare = false;
      if constexpr (kFormat != MXQ_CACHE_BF16) {
#pragma unroll
        for (int j = 0; j < 8 * S::kScaleRow; j += 32)
          if (8 * S::kScaleRow % 32 == 0 || j + lane < 8 * S::kScaleRow)
            rare |= any_rare<kFormat>(reinterpret_cast<const uint32_t *>(st + 2 * S::kSide)[j + lane], c.bits);
        rare = __any_sync(0xFFFFFFFFu, rare);
      }
      if (kFormat != MXQ_CACHE_BF16 && rare)
        w.template tile<true>(st, live, c.bits, a, Place{here.b, here.row, rows, tok}, lane);
      else
        w.template tile<false>(st, live, c.bits, a, Place{here.b, here.row, rows, tok}, lane);
    }
    stage = stage == S::kStages - 1 ? 0 : stage + 1;
    if (i + 1 == todo) let_next_start();
    if (here.unit + 1 < work && i + 1 < todo) {
      ++here.unit;
      continue;
    }
    const bool ends = here.unit < work;  // the CTA's part of the row ends here (otherwise an empty unit)
    const int slot = from > 0, b_now = here.b, head_now = first_head, heads_now = heads;
    const bool whole = from_unit == 0 && here.unit + 1 == work;
    here.advance(a, rows, i + 1 < todo);
    if (here.unit == 0) {  // the next row's queries are on their way while this row is joined
      from = i + 1, from_unit = 0;
      if (i + 1 < todo) tile_of_head(here, first_head, heads), load_query(here, first_head, heads);
    }
    if (!ends) continue;

    // Join the warps.  Every lane holds heads 2t, 2t + 1 of each tile (entry & 1) at two rows of O^T (entry >> 1) for each
    // of D / 16 steps; sums run over the lanes of equal t.
    if (joined) __syncthreads();  // the previous join has been read
    joined = true;
    constexpr int kEntries = NT * D / 4;  // of a lane: [n][h][2 j + row]
    float *mine = sm_o + warp * kEntries * 32 + lane;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float l = w.l[n][h];
#pragma unroll
        for (int y = 4; y < 32; y <<= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, y);
        const int hh = warp * kHeads + n * 8 + 2 * t + h;
        if (r == 0) sm_m[hh] = w.m[n][h], sm_l[hh] = l;
#pragma unroll
        for (int e = 0; e < D / 8; ++e) mine[((n * 2 + h) * (D / 8) + e) * 32] = w.o[e >> 1][n][2 * (e & 1) + h];
      }
    }
    w.clear();
    __syncthreads();
    // a warp takes a quarter of the entries of its lanes' heads: 8 or fewer neighbouring elements of a head
    constexpr int kQuarter = kEntries / kWarps;
    const int e0 = warp * kQuarter, h = (e0 / (D / 8) / 2) * 8 + 2 * t + ((e0 / (D / 8)) & 1);
    if (h < heads_now) {
      float top = sm_m[h], f[kWarps], sum = 0.f;
#pragma unroll
      for (int k = 1; k < kWarps; ++k) top = fmaxf(top, sm_m[k * kHeads + h]);
#pragma unroll
      for (int k = 0; k < kWarps; ++k) f[k] = exp2f(sm_m[k * kHeads + h] - top), sum += f[k] * sm_l[k * kHeads + h];
      const int64_t head_row = (int64_t)b_now * a.q_heads + head_now + h;
      const int64_t part = ((int64_t)blockIdx.x * 2 + slot) * kHeads + h;
#pragma unroll
      for (int e = 0; e < kQuarter; ++e) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) v += f[k] * sm_o[(k * kEntries + e0 + e) * 32 + lane];
        const int d = value_element<kFormat, D>((e0 + e) % (D / 8), r);
        if (whole)
          store_scalar(static_cast<T *>(a.out) + head_row * D + d, sum == 0.f ? 0.f : v / sum);
        else
          a.part_o[part * D + d] = v;
      }
      if (r == 0 && e0 % (D / 8) == 0) {
        if (!whole)
          a.part_ml[part] = make_float2(top, sum);
        else if (a.stats != nullptr)
          a.stats[head_row] = make_float2(top, sum);
      }
    }
  }
}

// Joins the parts of the rows that CTAs share, and adds the softmax weights of every token to the caller's statistics:
//   weights[b, head, j] += sum over the group of exp(s_j - m) / l.
// Without weights bound by latency: 8 to 9 us by itself, of which the launch during the attention kernel hides some.  With them,
// 8 sequences of 3000 to 8192 tokens, 8 x 4 heads of 128, E4M3: 18 us for 12 MB, behind an attention kernel that takes 28 us
// with the scores written and 26 without; the two calls take 43 and 33 us.
// grid: (x, heads, batch): the x CTAs take the heads of the group in turn, W warps a head, and their threads the tokens.
// Before the wait only what the attention kernel does not write is read: its CTAs let this kernel start after their own
// wait, so everything before it in the stream has finished.
template <typename T, int W>
__global__ void __launch_bounds__(finish_threads(W))
finish_kernel(const AttnArgs a, int heads, int tile_heads, int dim) {
  constexpr int kThreads = finish_threads(W), kAtOnce = kThreads / 32 / W;  // heads of the group at a time
  __shared__ float4 sums[W > 1 ? kThreads : 1];
  extern __shared__ float2 stats[];  // [group] pairs of maximum and 1 / sum
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = blockIdx.y, b = blockIdx.z;
  const int rows = heads * a.head_tiles;
  const int64_t before = units_between(a, 0, b, lane);
  const int length = length_of(a, b), n = units_of_length(length);
  const int64_t total = (before + n + units_between(a, b + 1, a.batch, lane)) * rows;
  const Split split(total, min((int64_t)a.ctas, total));

  // CTAs first .. last hold the parts of head g's row; part of CTA c in its slot 0 or 1
  auto locate = [&](int g, int &first, int &last, bool &late) {
    const int64_t u0 = before * rows + (int64_t)(head * a.head_tiles + g / tile_heads) * n;
    first = (int)split.cta_of(u0), last = (int)split.cta_of(u0 + n - kRowCost - 1);
    late = split.start(first) < u0;  // the row is not the first one of its first CTA
  };
  auto part_of = [&](int c, int first, bool late, int g) {
    return (int64_t)(c * 2 + (c == first && late ? 1 : 0)) * tile_heads + g % tile_heads;
  };
  // maximum and sum of head g, by a whole warp
  auto join = [&](int g, int first, int last, bool late) {
    if (first == last) return a.stats != nullptr ? a.stats[(int64_t)b * a.q_heads + head * a.group + g] : make_float2(0.f, 0.f);
    float top = kLowest, sum = 0.f;
#pragma unroll 8
    for (int c = first + lane; c <= last; c += 32) {  // running maximum and sum: one pass over the parts
      const float2 p = a.part_ml[part_of(c, first, late, g)];
      const float high = fmaxf(top, p.x);
      sum = sum * exp2f(top - high) + p.y * exp2f(p.x - high), top = high;
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) {
      const float t2 = __shfl_xor_sync(0xFFFFFFFFu, top, x), s2 = __shfl_xor_sync(0xFFFFFFFFu, sum, x);
      const float high = fmaxf(top, t2);
      sum = sum * exp2f(top - high) + s2 * exp2f(t2 - high), top = high;
    }
    return make_float2(top, sum);
  };
  int first, last;
  bool late;
  const int sub = warp % W, g_first = blockIdx.x * kAtOnce + warp / W;
  locate(min(g_first, a.group - 1), first, last, late);
  wait_for_previous();

  // A part is dim / 4 vectors: lanes beyond that take further parts, to be added up at the end.
  const int vecs = dim >> 2, at_once = vecs < 32 ? 32 / vecs : 1;
  for (int g0 = blockIdx.x * kAtOnce; g0 < a.group; g0 += gridDim.x * kAtOnce) {
    const int g = g0 + warp / W;
    const bool there = g < a.group;
    if (there && g != g_first) locate(g, first, last, late);
    const bool parts = there && first != last;  // otherwise finished by its CTA
    const float2 st = parts ? join(g, first, last, late) : make_float2(0.f, 0.f);
    for (int v0 = 0; v0 < vecs; v0 += 32) {  // more than once for head_dim 256
      const int vec = v0 + (vecs < 32 ? lane & (vecs - 1) : lane);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (parts) {
#pragma unroll 8
        for (int c = first + sub * at_once + (vecs < 32 ? lane / vecs : 0); c <= last; c += W * at_once) {
          const int64_t part = part_of(c, first, late, g);
          const float f = exp2f(a.part_ml[part].x - st.x);
          const float4 o = reinterpret_cast<const float4 *>(a.part_o + part * dim)[vec];
          v.x += f * o.x, v.y += f * o.y, v.z += f * o.z, v.w += f * o.w;
        }
      }
      if constexpr (W > 1) {
        if (v0 > 0 || g0 > blockIdx.x * kAtOnce) __syncthreads();  // the sums before have been read
        sums[tid] = v;
        __syncthreads();
        if (sub == 0) {
#pragma unroll
          for (int k = 1; k < W; ++k) {
            const float4 o = sums[tid + 32 * k];
            v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
          }
        }
      }
      for (int x = 16; x >= vecs; x >>= 1) {
        v.x += __shfl_xor_sync(0xFFFFFFFFu, v.x, x), v.y += __shfl_xor_sync(0xFFFFFFFFu, v.y, x);
        v.z += __shfl_xor_sync(0xFFFFFFFFu, v.z, x), v.w += __shfl_xor_sync(0xFFFFFFFFu, v.w, x);
      }
      if (parts && sub == 0 && (vecs >= 32 || lane < vecs)) {
        const float r[4] = {v.x / st.y, v.y / st.y, v.z / st.y, v.w / st.y};
        const float none[4] = {0.f, 0.f, 0.f, 0.f};
        T *out = static_cast<T *>(a.out) + ((int64_t)b * a.q_heads + head * a.group + g) * dim + 4 * vec;
        if (st.y == 0.f)
          store_vals(out, 0, none);
        else
          store_vals(out, 0, r);
      }
    }
  }
  if (a.weights == nullptr) return;
  for (int g = warp; g < a.group; g += kThreads / 32) {
    locate(g, first, last, late);
    const float2 st = join(g, first, last, late);
    if (lane == 0) stats[g] = make_float2(st.x, st.y == 0.f ? 0.f : 1.f / st.y);
  }
  __syncthreads();
  const float *scores = a.scores + ((int64_t)b * rows + head * a.head_tiles) * a.score_tokens * a.score_heads;
  float *weights = a.weights + ((int64_t)b * heads + head) * a.weights_width;
  for (int j = blockIdx.x * kThreads + tid; j < length; j += gridDim.x * kThreads) {
    float sum = 0.f;
    for (int g = 0; g < a.group; g += 2) {  // two heads of a tile lie together
      const int ht = g / tile_heads;
      const float2 s = *reinterpret_cast<const float2 *>(scores + ((int64_t)ht * a.score_tokens + j) * a.score_heads + (g - ht * tile_heads));
      sum += exp2f(s.x - stats[g].x) * stats[g].y;
      if (g + 1 < a.group) sum += exp2f(s.y - stats[g + 1].x) * stats[g + 1].y;
    }
    weights[j] += sum;
  }
}

// Query heads in tiles of 8, or of 16 for bf16 queries of more than 8 heads a group and head_dim <= 128 (larger ones do
// not fit the registers): 16 heads a group over 8 x 8192 E4M3 tokens of 8 heads of 128 take 55 us in one tile, 67 us in two.
static int tiles_per_row(int dtype, int dim, int64_t group) { return dtype == MXQ_BF16 && group > 8 && dim <= 128 ? 2 : 1; }
constexpr int kMostPerSm = 8;  // CTAs of the attention kernel on one SM, at most

static int64_t units_of_launch(int64_t batch, int64_t rows, int64_t tokens) {
  return batch * rows * ((tokens + kUnit - 1) / kUnit + kRowCost);
}
// Heads of a tile whose scores are kept for the weights: all of them, or the group's rounded up to a power of two.
static int score_heads(int nt, int64_t group) {
  int n = 2;
  while (n < group && n < 8 * nt) n *= 2;
  return n;
}
struct Workspace {
  int64_t ml, o, stats, scores, total;  // byte offsets
};
static Workspace workspace_of(int nt, int64_t batch, int64_t heads, int64_t q_heads, int dim, int64_t tokens, bool weights,
                              int64_t &most_ctas) {
  const int64_t head_tiles = (q_heads / heads + 8 * nt - 1) / (8 * nt);
  const int64_t units = units_of_launch(batch, heads * head_tiles, tokens);
  most_ctas = (int64_t)gemm::sm_count() * kMostPerSm;
  if (units < most_ctas) most_ctas = units;
  auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
  const bool parts = tokens > kUnit;
  Workspace w;
  w.ml = 0;
  w.o = parts ? up(most_ctas * 2 * 8 * nt * (int64_t)sizeof(float2)) : 0;
  w.stats = w.o + (parts ? up(most_ctas * 2 * 8 * nt * dim * 4) : 0);
  w.scores = w.stats + (weights ? up(batch * q_heads * (int64_t)sizeof(float2)) : 0);
  w.total = w.scores + (weights ? batch * heads * head_tiles * tokens * score_heads(nt, q_heads / heads) * 4 : 0);
  return w;
}

template <typename T, int kFormat, int D, int NT>
static int launch_one(const Cache &c, const Table &t, AttnArgs &a, int64_t most_ctas, cudaStream_t st) {
  constexpr int kSmem = Smem<kFormat, D, NT>::kTotal;
  auto kernel = attention_kernel<T, kFormat, D, NT>;
  static std::atomic<int> known[64];  // CTAs per SM on each device, once the kernel has been set up there
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return MXQ_ERR_LAUNCH;
  int per_sm = known[device & 63].load(std::memory_order_relaxed);
  if (per_sm == 0) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kWarps * 32, kSmem) != cudaSuccess || per_sm < 1) {
      cudaGetLastError();
      return MXQ_ERR_LAUNCH;
    }
    known[device & 63].store(per_sm, std::memory_order_relaxed);
  }
  int64_t ctas = (int64_t)gemm::sm_count() * (per_sm < kMostPerSm ? per_sm : kMostPerSm);
  if (ctas > most_ctas) ctas = most_ctas;
  a.ctas = (int)ctas;
  return launch_chained(kernel, dim3((unsigned)ctas), kWarps * 32, kSmem, st, 1, c, t, a);
}
template <typename T, int kFormat, int D>
static int launch_dim(const Cache &c, const Table &t, AttnArgs &a, int nt, int64_t most_ctas, cudaStream_t st) {
  if constexpr (Elem<T>::kBf16 && D <= 128) {
    if (nt == 2) return launch_one<T, kFormat, D, 2>(c, t, a, most_ctas, st);
  }
  return launch_one<T, kFormat, D, 1>(c, t, a, most_ctas, st);
}
template <typename T>
static int launch_attention(int format, int dim, const Cache &c, const Table &t, AttnArgs &a, int nt, int64_t most_ctas,
                            cudaStream_t st) {
#define CALL(f)                                                                      \
  if (format == f) {                                                                 \
    if (dim == 32) return launch_dim<T, f, 32>(c, t, a, nt, most_ctas, st);          \
    if (dim == 64) return launch_dim<T, f, 64>(c, t, a, nt, most_ctas, st);          \
    if (dim == 128) return launch_dim<T, f, 128>(c, t, a, nt, most_ctas, st);        \
    if (dim == 256) return launch_dim<T, f, 256>(c, t, a, nt, most_ctas, st);        \
  }
  MXQ_PAGED_FORMATS(CALL)
#undef CALL
  return MXQ_ERR_FORMAT;
}

}  // namespace paged
}  // namespace mxq

using namespace mxq;
using namespace mxq::paged;

// Checks shared by the size query and the call; `group` comes back.
static int check_attention(const mxq_paged_cache *cache, int64_t batch, int64_t q_heads, int64_t table_width, int page_log2,
                           int64_t &group) {
  if (batch < 0 || batch > 65535 || q_heads < 1 || q_heads > 65535 || q_heads % cache->heads) return MXQ_ERR_SHAPE;
  if (table_width < 1 || table_width > (kMostTokens >> page_log2)) return MXQ_ERR_SHAPE;
  group = q_heads / cache->heads;
  return group <= 4096 ? MXQ_OK : MXQ_ERR_SHAPE;  // the statistics of a group fit shared memory
}

extern "C" {

int64_t mxq_paged_attention_workspace_bytes(const mxq_paged_cache *cache, int64_t batch, int64_t q_heads,
                                            int64_t table_width, int with_weights) {
  Cache c;
  int rc = read_cache(cache, c);
  if (rc != MXQ_OK) return rc;
  int64_t group;
  if ((rc = check_attention(cache, batch, q_heads, table_width, c.page_log2, group)) != MXQ_OK) return rc;
  if (batch == 0) return 0;
  const int64_t tokens = table_width << c.page_log2;
  int64_t most = 0;
  for (int dtype : {MXQ_F32, MXQ_BF16}) {
    int64_t ctas;
    const int nt = tiles_per_row(dtype, cache->head_dim, group);
    const int64_t n = workspace_of(nt, batch, c.heads, q_heads, cache->head_dim, tokens, with_weights != 0, ctas).total;
    if (n > most) most = n;
  }
  return most;
}

int mxq_paged_attention(const mxq_paged_cache *cache, const void *q, void *out, int dtype, int64_t batch, int64_t q_heads,
                        int64_t q_stride_b, int64_t q_stride_h, float scaling, const int32_t *page_table,
                        int64_t table_width, int64_t table_stride, const int32_t *lengths, float *weights,
                        int64_t weights_width, void *workspace, int64_t workspace_bytes, int *status, void *stream) {
  Cache c;
  int rc = read_cache(cache, c);
  if (rc != MXQ_OK) return rc;
  if (dtype != MXQ_F32 && dtype != MXQ_BF16) return MXQ_ERR_DTYPE;
  if (batch == 0) return MXQ_OK;
  if ((rc = read_table(page_table, table_width, table_stride, batch, c.page_log2)) != MXQ_OK) return rc;
  int64_t group;
  if ((rc = check_attention(cache, batch, q_heads, table_width, c.page_log2, group)) != MXQ_OK) return rc;
  if (!q || !out || !lengths) return MXQ_ERR_NULL;
  if (!aligned(out, 16)) return MXQ_ERR_ALIGN;
  if (weights && weights_width < 1) return MXQ_ERR_SHAPE;
  const int dim = cache->head_dim;
  const int64_t tokens = table_width << c.page_log2;
  if (c.pages > MXQ_CACHE_SIDE_BYTES / (((int64_t)c.heads << c.page_log2) * row_bytes_of(cache->format, dim)))
    return MXQ_ERR_SHAPE;  // tiles are addressed by 32-bit multiples of 16 bytes
  const int nt = tiles_per_row(dtype, dim, group);
  int64_t most_ctas;
  const Workspace w = workspace_of(nt, batch, c.heads, q_heads, dim, tokens, weights != nullptr, most_ctas);
  // a CTA counts its units in 32 bits: with one CTA on each SM it has at most this many
  if (units_of_launch(batch, c.heads * ((group + 8 * nt - 1) / (8 * nt)), tokens) / gemm::sm_count() >= INT32_MAX)
    return MXQ_ERR_SHAPE;
  if (w.total > 0) {
    if (!workspace) return MXQ_ERR_NULL;
    if (!aligned(workspace, 16)) return MXQ_ERR_ALIGN;
    if (workspace_bytes < w.total) return MXQ_ERR_SHAPE;
  }
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  AttnArgs a;
  a.q = q, a.out = out, a.q_stride_b = q_stride_b, a.q_stride_h = q_stride_h;
  const double factor = (double)scaling * 1.4426950408889634074;
  a.c_hi = (float)factor, a.c_lo = (float)(factor - a.c_hi);
  a.group = (int)group, a.q_heads = (int)q_heads, a.head_tiles = (int)((group + 8 * nt - 1) / (8 * nt));
  a.batch = (int)batch, a.lengths = lengths;
  a.most = weights && weights_width < tokens ? weights_width : tokens;
  const bool parts = tokens > kUnit;  // otherwise every row is one unit and finished by its CTA
  a.part_ml = parts ? reinterpret_cast<float2 *>(ws + w.ml) : nullptr;
  a.part_o = parts ? reinterpret_cast<float *>(ws + w.o) : nullptr;
  a.stats = weights ? reinterpret_cast<float2 *>(ws + w.stats) : nullptr;
  a.scores = weights ? reinterpret_cast<float *>(ws + w.scores) : nullptr;
  a.score_tokens = tokens, a.score_heads = score_heads(nt, group);
  a.weights = weights, a.weights_width = weights_width, a.status = status;
  const Table t{page_table, table_stride, table_width};
  cudaStream_t st = (cudaStream_t)stream;
  rc = dtype == MXQ_BF16 ? launch_attention<__nv_bfloat16>(cache->format, dim, c, t, a, nt, most_ctas, st)
                         : launch_attention<float>(cache->format, dim, c, t, a, nt, most_ctas, st);
  if (rc != MXQ_OK || (!parts && !weights)) return rc;
  // Warps for a head: one where rows are shared by few CTAs (64 sequences, 512 rows: 80 us against 88 with four), four or
  // sixteen where they are shared by many (one row of 40000 tokens in 444 parts: 23 us with sixteen, 33 with four, 94 with
  // one; 16 rows of 28 parts: 104 us with four, 109 with one).
  const int64_t per_row = a.ctas / (batch * c.heads * a.head_tiles);
  const int w_head = per_row >= 64 ? 16 : (per_row >= 8 ? 4 : 1), threads = finish_threads(w_head);
  const int64_t at_once = threads / 32 / w_head;
  int64_t x = (group + at_once - 1) / at_once;
  if (weights) {  // enough CTAs for the tokens, and no more than the GPU holds at once
    const int64_t need = (tokens + threads - 1) / threads;
    const int64_t cap = ((int64_t)gemm::sm_count() * (2048 / threads) + c.heads * batch - 1) / (c.heads * batch);
    const int64_t most = need < cap ? need : cap;
    x = most > x ? most : x;
  }
  const dim3 grid((unsigned)x, (unsigned)c.heads, (unsigned)batch);
  const size_t smem = weights ? group * sizeof(float2) : 0;
#define CALL(T)                                                                                                   \
  return w_head == 16  ? launch_chained(finish_kernel<T, 16>, grid, threads, smem, st, 1, a, c.heads, 8 * nt, dim) \
         : w_head == 4 ? launch_chained(finish_kernel<T, 4>, grid, threads, smem, st, 1, a, c.heads, 8 * nt, dim)  \
                       : launch_chained(finish_kernel<T, 1>, grid, threads, smem, st, 1, a, c.heads, 8 * nt, dim);
  if (dtype == MXQ_BF16) CALL(__nv_bfloat16)
  CALL(float)
#undef CALL
}

}  // extern "C"
