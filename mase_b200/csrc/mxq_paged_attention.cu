// Attention of one new token per sequence over a paged MX key/value cache (mxq_paged_attention):
//   s_j = scaling * <q, k_j>,  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m = max_j s_j.
// One pass over the cache with a running maximum and sum, split over the length and joined.
//
// A warp works on tiles of 16 cached tokens with m16n8k16 tensor-core products, both transposed so that the cache is the
// 16-row operand and the query heads of one key/value head are the 8 columns:
//   S^T[token, head] = K[token, d] Q^T[d, head]          rows = tokens, accumulated over head_dim
//   O^T[d, head]    += V^T[d, token] P^T[token, head]    rows = d, accumulated over the tokens of all tiles
// The order of the summed index of a product is free, and so is the order of the rows of O^T, so every lane loads its
// operands straight from the pages in pieces of up to 16 contiguous bytes (four lanes share a key row, eight lanes a value
// row) and no transposition of the cache goes through shared memory; Q^T and the output follow the same permutation.
//
// Codes become bf16 in registers: sign, exponent and fraction fields are moved to the bf16 positions with masks and
// shifts and the result is multiplied by one power of two (block scale times the difference of the exponent biases).
// Every value of every format has at most 8 significant bits, so this is exact, subnormal codes included.  bf16 queries
// are exact operands too; fp32 queries are split into three bf16 terms.  Probabilities are fp32 and enter the second
// product as two (fp32 queries: three) bf16 terms, 16 (24) significant bits; scores, maxima, sums and O^T are fp32.

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "mxq.h"
#include "mxq_common.cuh"
#include "mxq_internal.h"
#include "mxq_paged.cuh"

namespace mxq {
namespace paged {

constexpr int kWarps = 4;
constexpr int kTile = 16;
constexpr int kJoinThreads = 128;

struct AttnArgs {
  const void *q;
  void *out;
  int64_t q_stride_b, q_stride_h;
  float scaling;
  int group;     // query heads per key/value head
  int q_heads;
  int head_tiles;
  const int32_t *lengths;
  int64_t most;  // tokens that tables (and weights) can hold
  int chunk, chunks;
  float *part_o;   // [batch, q_heads, chunks, dim]
  float2 *part_ml; // [batch, q_heads, chunks]: maximum and sum
  float *scores;   // [batch, heads, head_tiles, tokens, 8 * NT] when weights are accumulated
  int64_t score_tokens;
  float *weights;
  int64_t weights_width;
  int *status;
};

// ---- codes to bf16 ---------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// exponent offset of the raw bf16 pattern of a code: value = raw * 2^offset * 2^(scale - 127)
template <int kFormat>
__device__ __forceinline__ int raw_offset(int bits) {
  if constexpr (kFormat == MXQ_CACHE_INT8)
    return 1 - bits;
  else if constexpr (kFormat == MXQ_CACHE_BF16)
    return 0;
  else
    return 127 - ((1 << (Format<kFormat>::E - 1)) - 1);
}
// bf16 pattern of 2^x, x >= -133 (0 below); x above 127 saturates
__device__ __forceinline__ uint32_t pow2_bf16(int x) {
  if (x > 127) x = 127;
  return x >= -126 ? (uint32_t)(x + 127) << 7 : (x >= -133 ? 1u << (x + 133) : 0u);
}
// The multiplier of a block; kBig: the part of the exponent above 127 goes into `rest`.
template <int kFormat>
__device__ __forceinline__ int block_exponent(uint32_t scale, int bits) {
  if (kFormat == MXQ_CACHE_INT8 && scale == 255) return 128;  // 2^128: the reference multiplies zeros by inf
  return (int)scale - 127 + raw_offset<kFormat>(bits);
}
template <int kFormat>
__device__ __forceinline__ uint32_t block_factor(int x) {
  if (kFormat == MXQ_CACHE_INT8 && x == 128) return 0x7F80u;
  return pow2_bf16(x);
}

// Two codes, one in the upper byte of each half of x (what is in the lower bytes does not matter) -> raw bf16 pair.
template <int kFormat>
__device__ __forceinline__ uint32_t raw_upper(uint32_t x) {
  if constexpr (kFormat == MXQ_CACHE_E4M3) return ((x >> 4) & 0x07F007F0u) | (x & 0x80008000u);
  if constexpr (kFormat == MXQ_CACHE_E5M2) return ((x >> 3) & 0x0FE00FE0u) | (x & 0x80008000u);
  return 0;
}
// Two int8, one in the lower byte of each half -> bf16 pair: 128 + (u & 127) minus 128 or 256 by the sign bit.
__device__ __forceinline__ uint32_t int8_lower(uint32_t x) {
  return sub2((x & 0x007F007Fu) | 0x43004300u, (x & 0x00800080u) | 0x43004300u);
}
// Nibble i (0..3) of each half -> raw bf16 pair of E2M1.
template <int i>
__device__ __forceinline__ uint32_t raw_nibble(uint32_t x) {
  if constexpr (i == 0) return ((x << 12) & 0x80008000u) | ((x << 6) & 0x01C001C0u);
  if constexpr (i == 1) return ((x << 8) & 0x80008000u) | ((x << 2) & 0x01C001C0u);
  if constexpr (i == 2) return ((x << 4) & 0x80008000u) | ((x >> 2) & 0x01C001C0u);
  return (x & 0x80008000u) | ((x >> 6) & 0x01C001C0u);
}

template <bool kBig>
__device__ __forceinline__ uint32_t scaled(uint32_t raw, uint32_t f, uint32_t rest) {
  raw = mul2(raw, f);
  return kBig ? mul2(raw, rest) : raw;
}

// One word of a key row -> bf16 pairs.  Pair i of the word holds these elements (relative to the word's first one):
//   16 bit: (0, 1);  8 bit: (i, i + 2);  4 bit: (i, i + 4)
template <int kFormat, bool kBig>
__device__ __forceinline__ void key_word(uint32_t w, uint32_t f, uint32_t rest, uint32_t *out) {
  if constexpr (kFormat == MXQ_CACHE_BF16) {
    out[0] = w;
  } else if constexpr (kFormat == MXQ_CACHE_INT8) {
    out[0] = scaled<kBig>(int8_lower(w), f, rest), out[1] = scaled<kBig>(int8_lower(w >> 8), f, rest);
  } else if constexpr (Format<kFormat>::kBits == 8) {
    out[0] = scaled<kBig>(raw_upper<kFormat>(w << 8), f, rest), out[1] = scaled<kBig>(raw_upper<kFormat>(w), f, rest);
  } else {
    out[0] = scaled<kBig>(raw_nibble<0>(w), f, rest), out[1] = scaled<kBig>(raw_nibble<1>(w), f, rest);
    out[2] = scaled<kBig>(raw_nibble<2>(w), f, rest), out[3] = scaled<kBig>(raw_nibble<3>(w), f, rest);
  }
}
// The same word of two value rows -> pairs (row a, row b) of its elements 0, 1, 2, ...
template <int kFormat, bool kBig>
__device__ __forceinline__ void value_words(uint32_t a, uint32_t b, uint32_t f, uint32_t rest, uint32_t *out) {
  if constexpr (kFormat == MXQ_CACHE_BF16) {
    out[0] = __byte_perm(a, b, 0x5410), out[1] = __byte_perm(a, b, 0x7632);
  } else if constexpr (kFormat == MXQ_CACHE_INT8) {
    out[0] = scaled<kBig>(int8_lower(__byte_perm(a, b, 0x4400)), f, rest);
    out[1] = scaled<kBig>(int8_lower(__byte_perm(a, b, 0x5511)), f, rest);
    out[2] = scaled<kBig>(int8_lower(__byte_perm(a, b, 0x6622)), f, rest);
    out[3] = scaled<kBig>(int8_lower(__byte_perm(a, b, 0x7733)), f, rest);
  } else if constexpr (Format<kFormat>::kBits == 8) {
    out[0] = scaled<kBig>(raw_upper<kFormat>(__byte_perm(a, b, 0x4400)), f, rest);
    out[1] = scaled<kBig>(raw_upper<kFormat>(__byte_perm(a, b, 0x5511)), f, rest);
    out[2] = scaled<kBig>(raw_upper<kFormat>(__byte_perm(a, b, 0x6622)), f, rest);
    out[3] = scaled<kBig>(raw_upper<kFormat>(__byte_perm(a, b, 0x7733)), f, rest);
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t x = __byte_perm(a, b, h ? 0x7632 : 0x5410);
      out[4 * h + 0] = scaled<kBig>(raw_nibble<0>(x), f, rest), out[4 * h + 1] = scaled<kBig>(raw_nibble<1>(x), f, rest);
      out[4 * h + 2] = scaled<kBig>(raw_nibble<2>(x), f, rest), out[4 * h + 3] = scaled<kBig>(raw_nibble<3>(x), f, rest);
    }
  }
}

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

// kBytes (2, 4, 8 or 16) contiguous bytes as words
template <int kBytes>
__device__ __forceinline__ void load_piece(const uint8_t *p, uint32_t *w) {
  if constexpr (kBytes == 16) {
    const uint4 r = __ldcs(reinterpret_cast<const uint4 *>(p));
    w[0] = r.x, w[1] = r.y, w[2] = r.z, w[3] = r.w;
  } else if constexpr (kBytes == 8) {
    const uint2 r = __ldcs(reinterpret_cast<const uint2 *>(p));
    w[0] = r.x, w[1] = r.y;
  } else if constexpr (kBytes == 4) {
    w[0] = __ldcs(reinterpret_cast<const uint32_t *>(p));
  } else {
    w[0] = __ldcs(reinterpret_cast<const unsigned short *>(p));
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
};
// element (0 .. D-1) that half `half` of pair i of key word w of piece c of lane t holds
template <int kFormat, int D>
__device__ __forceinline__ int key_element(int c, int w, int i, int half, int t) {
  using S = Shape<kFormat, D>;
  const int first = (c * 4 * S::kKeyPiece + t * S::kKeyPiece + w * 4) * 8 / S::kBits;
  return first + (S::kBits == 16 ? half : (S::kBits == 8 ? i + 2 * half : i + 4 * half));
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

constexpr float kLog2e = 1.4426950408889634f;
// A tile raises the running maximum only when a score exceeds it by more than this: probabilities then stay below
// e^8 and the rescaling (shuffles, D/4 products) runs a few times per warp instead of once per tile.
constexpr float kSlack = 8.f;

template <typename T, int kFormat, int D, int NT>
struct Worker {
  using S = Shape<kFormat, D>;
  static constexpr int kTerms = Elem<T>::kBf16 ? 1 : 3;   // bf16 terms of a query element
  static constexpr int kPTerms = Elem<T>::kBf16 ? 2 : 3;  // and of a probability
  static constexpr int kSteps = D / 16;
  uint32_t q[kTerms][kSteps][NT][2];
  float o[kSteps][NT][4];
  float m[NT][2], l[NT][2];

  __device__ __forceinline__ void start(const T *qrow, int64_t stride_h, int heads, int lane) {
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
#pragma unroll
      for (int h = 0; h < 2; ++h) m[n][h] = -INFINITY, l[n][h] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < kSteps; ++j)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][n][i] = 0.f;
  }

  // kk: key words of tokens r and r + 8; vv: value words of tokens 2t, 2t + 1, 2t + 8, 2t + 9; fk, fv: their exponents
  template <bool kBig>
  __device__ __forceinline__ void tile(const uint32_t (&kk)[2][S::kKeyPieces][S::kKeyWords],
                                       const uint32_t (&vv)[4][S::kValPieces][S::kValWords],
                                       const int (&xk)[2][S::kKeyPieces], const int (&xv)[4][S::kValPieces], int live,
                                       float scaling, float *scores, int lane) {
    const int t = lane & 3, r = lane >> 2;
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int c = 0; c < S::kKeyPieces; ++c) {
      uint32_t pairs[2][S::kKeyWords * S::kPairs];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t f = 0, rest = 0;
        if constexpr (kFormat != MXQ_CACHE_BF16) {
          f = block_factor<kFormat>(xk[h][c]) * 0x00010001u;
          if (kBig) rest = pow2_bf16(max(xk[h][c] - 127, 0)) * 0x00010001u;
        }
#pragma unroll
        for (int w = 0; w < S::kKeyWords; ++w) key_word<kFormat, kBig>(kk[h][c][w], f, rest, &pairs[h][w * S::kPairs]);
      }
      constexpr int kStepsHere = S::kKeyWords * S::kPairs / 2;
#pragma unroll
      for (int k = 0; k < kStepsHere; ++k) {
        const uint32_t a[4] = {pairs[0][2 * k], pairs[1][2 * k], pairs[0][2 * k + 1], pairs[1][2 * k + 1]};
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = kTerms - 1; x >= 0; --x)
            mma(s[n], a, q[x][c * kStepsHere + k][n][0], q[x][c * kStepsHere + k][n][1]);
      }
    }
    // rows: tokens r (entries 0, 1) and r + 8 (2, 3); columns: heads 2t, 2t + 1
    bool raise = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[n][i] = r + 8 * (i >> 1) < live ? s[n][i] * scaling : -INFINITY;
        raise |= s[n][i] > m[n][i & 1] + kSlack;
      }
    if (scores != nullptr) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (r + 8 * h < live)
            *reinterpret_cast<float2 *>(scores + (int64_t)(r + 8 * h) * (8 * NT) + n * 8 + 2 * t) =
                make_float2(s[n][2 * h], s[n][2 * h + 1]);
    }
    if (__any_sync(0xFFFFFFFFu, raise)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float top = fmaxf(s[n][h], s[n][2 + h]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
          top = fmaxf(top, m[n][h]);
          const float f = top == m[n][h] ? 1.f : exp2f((m[n][h] - top) * kLog2e);
          m[n][h] = top, l[n][h] *= f;
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
        p[i] = s[n][i] == -INFINITY ? 0.f : exp2f((s[n][i] - m[n][i & 1]) * kLog2e);
        l[n][i & 1] += p[i];
      }
#pragma unroll
      for (int x = 0; x < kPTerms; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          pb[x][n][h] = transpose8x8(pack_bf16x2(p[2 * h], p[2 * h + 1]));
          p[2 * h] -= bf16_of(p[2 * h]), p[2 * h + 1] -= bf16_of(p[2 * h + 1]);
        }
    }
#pragma unroll
    for (int c = 0; c < S::kValPieces; ++c) {
      uint32_t f[2] = {0, 0}, rest[2] = {0, 0};
      if constexpr (kFormat != MXQ_CACHE_BF16) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // a token behind the last one has factor 0: whatever its slot holds, it adds nothing
          const uint32_t a = 2 * t + 8 * h < live ? block_factor<kFormat>(xv[2 * h][c]) : 0u;
          const uint32_t b = 2 * t + 8 * h + 1 < live ? block_factor<kFormat>(xv[2 * h + 1][c]) : 0u;
          f[h] = a | (b << 16);
          if (kBig)
            rest[h] = pow2_bf16(max(xv[2 * h][c] - 127, 0)) | (pow2_bf16(max(xv[2 * h + 1][c] - 127, 0)) << 16);
        }
      }
      constexpr int kPerWord = 32 / S::kBits;
#pragma unroll
      for (int w = 0; w < S::kValWords; ++w) {
        uint32_t e[2][kPerWord];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t a = vv[2 * h][c][w], b = vv[2 * h + 1][c][w];
          if constexpr (kFormat == MXQ_CACHE_BF16) {
            if (2 * t + 8 * h >= live) a = 0;
            if (2 * t + 8 * h + 1 >= live) b = 0;
          }
          value_words<kFormat, kBig>(a, b, f[h], rest[h], e[h]);
        }
        constexpr int kHere = S::kValElems < kPerWord ? S::kValElems : kPerWord;
#pragma unroll
        for (int k = 0; k < kHere; k += 2) {
          const int j = (c * S::kValElems + w * kPerWord + k) / 2;
          const uint32_t a[4] = {e[0][k], e[0][k + 1], e[1][k], e[1][k + 1]};
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int x = kPTerms - 1; x >= 0; --x) mma(o[j][n], a, pb[x][n][0], pb[x][n][1]);
        }
      }
    }
  }
};

// grid: (chunks, heads * head tiles, batch); the CTA's warps take the chunk's tiles in turn.
template <typename T, int kFormat, int D, int NT>
__global__ void __launch_bounds__(kWarps * 32)
attention_kernel(const Cache c, const Table table, const AttnArgs a) {
  using S = Shape<kFormat, D>;
  __shared__ float sm_o[kWarps][NT * 8][D];
  __shared__ float sm_m[kWarps][NT * 8], sm_l[kWarps][NT * 8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = lane & 3, r = lane >> 2;
  const int head = blockIdx.y / a.head_tiles, ht = blockIdx.y - head * a.head_tiles;
  const int64_t b = blockIdx.z;
  const int length = clamp_length(a.lengths[b], a.most, a.status);
  const int begin = blockIdx.x * a.chunk, end = min(begin + a.chunk, length);
  if (begin >= end && !(blockIdx.x == 0 && a.chunks == 1)) return;
  const int first_head = head * a.group + ht * (8 * NT);
  const int heads = min(a.group - ht * (8 * NT), 8 * NT);

  Worker<T, kFormat, D, NT> w;
  w.start(static_cast<const T *>(a.q) + b * a.q_stride_b + first_head * a.q_stride_h, a.q_stride_h, heads, lane);
  float *scores = a.scores == nullptr
                      ? nullptr
                      : a.scores + (((b * c.heads + head) * a.head_tiles + ht) * a.score_tokens) * (8 * NT);
  const int in_page = (1 << c.page_log2) - 1;
  for (int tok = begin + warp * kTile; tok < end; tok += kWarps * kTile) {
    const int live = end - tok;
    const int64_t first = page_row(c, table, b, head, tok, a.status);
    if (first < 0) {  // the page does not exist: its tokens are left out
      if (scores != nullptr)
        for (int i = lane; i < min(live, kTile) * 8 * NT; i += 32) scores[(int64_t)tok * (8 * NT) + i] = -INFINITY;
      continue;
    }
    const int64_t row = first + (tok & in_page);
    uint32_t kk[2][S::kKeyPieces][S::kKeyWords], vv[4][S::kValPieces][S::kValWords];
    int xk[2][S::kKeyPieces], xv[4][S::kValPieces];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint8_t *p = c.codes[0] + (row + r + 8 * h) * S::kRow + t * S::kKeyPiece;
#pragma unroll
      for (int k = 0; k < S::kKeyPieces; ++k) load_piece<S::kKeyPiece>(p + k * 4 * S::kKeyPiece, kk[h][k]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t *p = c.codes[1] + (row + 2 * t + (i & 1) + 8 * (i >> 1)) * S::kRow + r * S::kValPiece;
#pragma unroll
      for (int k = 0; k < S::kValPieces; ++k) load_piece<S::kValPiece>(p + k * 8 * S::kValPiece, vv[i][k]);
    }
    bool big = false;
    if constexpr (kFormat != MXQ_CACHE_BF16) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t *p = c.scales[0] + (row + r + 8 * h) * (D / 32);
#pragma unroll
        for (int k = 0; k < S::kKeyPieces; ++k)
          xk[h][k] = block_exponent<kFormat>(p[((k * 4 + t) * S::kKeyPiece * 8 / S::kBits) >> 5], c.bits);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t *p = c.scales[1] + (row + 2 * t + (i & 1) + 8 * (i >> 1)) * (D / 32);
#pragma unroll
        for (int k = 0; k < S::kValPieces; ++k)
          xv[i][k] = block_exponent<kFormat>(p[((k * 8 + r) * S::kValPiece * 8 / S::kBits) >> 5], c.bits);
      }
      if constexpr (kFormat != MXQ_CACHE_INT8) {
#pragma unroll
        for (int k = 0; k < S::kKeyPieces; ++k) big |= xk[0][k] > 127 || xk[1][k] > 127;
#pragma unroll
        for (int k = 0; k < S::kValPieces; ++k)
          big |= xv[0][k] > 127 || xv[1][k] > 127 || xv[2][k] > 127 || xv[3][k] > 127;
        big = __any_sync(0xFFFFFFFFu, big);
      }
    }
    float *sc = scores == nullptr ? nullptr : scores + (int64_t)tok * (8 * NT);
    if (kFormat != MXQ_CACHE_BF16 && kFormat != MXQ_CACHE_INT8 && big)
      w.template tile<true>(kk, vv, xk, xv, live, a.scaling, sc, lane);
    else
      w.template tile<false>(kk, vv, xk, xv, live, a.scaling, sc, lane);
  }

  // join the warps: every lane holds heads 2t, 2t + 1 of each tile; sums run over the lanes of equal t
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float l = w.l[n][h];
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, x);
      if (r == 0) sm_m[warp][n * 8 + 2 * t + h] = w.m[n][h], sm_l[warp][n * 8 + 2 * t + h] = l;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        sm_o[warp][n * 8 + 2 * t + h][value_element<kFormat, D>(2 * j, r)] = w.o[j][n][h];
        sm_o[warp][n * 8 + 2 * t + h][value_element<kFormat, D>(2 * j + 1, r)] = w.o[j][n][2 + h];
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * D; i += kWarps * 32) {
    const int h = i / D, d = i - h * D;
    float top = sm_m[0][h];
#pragma unroll
    for (int k = 1; k < kWarps; ++k) top = fmaxf(top, sm_m[k][h]);
    float sum = 0.f, v = 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
      const float f = sm_m[k][h] == -INFINITY ? 0.f : exp2f((sm_m[k][h] - top) * kLog2e);
      sum += f * sm_l[k][h], v += f * sm_o[k][h][d];
    }
    const int64_t head_row = b * a.q_heads + first_head + h;
    if (a.part_o == nullptr) {
      store_scalar(static_cast<T *>(a.out) + head_row * D + d, sum > 0.f ? v / sum : (sum == 0.f ? 0.f : sum));
    } else {
      const int64_t part = head_row * a.chunks + blockIdx.x;
      a.part_o[part * D + d] = v;
      if (d == 0) a.part_ml[part] = make_float2(top, sum);
    }
  }
}

// Maximum and sum over a head's chunks; every thread of a warp gets them.
__device__ __forceinline__ float2 join_stats(const float2 *ml, int n, int lane) {
  float top = -INFINITY;
  for (int k = lane; k < n; k += 32) top = fmaxf(top, ml[k].x);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
  float sum = 0.f;
  for (int k = lane; k < n; k += 32) sum += ml[k].x == -INFINITY ? ml[k].y : ml[k].y * exp2f((ml[k].x - top) * kLog2e);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, x);
  return make_float2(top, sum);
}

// grid: (query heads, batch); threads over head_dim
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const AttnArgs a, int dim) {
  const int head = blockIdx.x;
  const int64_t b = blockIdx.y, row = b * a.q_heads + head;
  const int length = clamp_length(a.lengths[b], a.most, a.status);
  const int n = (length + a.chunk - 1) / a.chunk;
  const float2 *ml = a.part_ml + row * a.chunks;
  const float2 st = join_stats(ml, n, threadIdx.x & 31);
  for (int d = threadIdx.x; d < dim; d += kJoinThreads) {
    float v = 0.f;
    for (int k = 0; k < n; ++k) {
      const float f = ml[k].x == -INFINITY ? 0.f : exp2f((ml[k].x - st.x) * kLog2e);
      v += f * a.part_o[(row * a.chunks + k) * dim + d];
    }
    store_scalar(static_cast<T *>(a.out) + row * dim + d, st.y > 0.f ? v / st.y : (st.y == 0.f ? 0.f : st.y));
  }
}

// weights[b, head, j] += sum over the group of exp(s_j - m) / l.  grid: (token chunks, heads, batch)
__global__ void __launch_bounds__(kJoinThreads) weights_kernel(const AttnArgs a, int heads, int tile_heads) {
  extern __shared__ float2 stats[];  // [group]: maximum, 1 / sum
  const int head = blockIdx.y, lane = threadIdx.x & 31;
  const int64_t b = blockIdx.z;
  const int length = clamp_length(a.lengths[b], a.most, a.status);
  const int n = (length + a.chunk - 1) / a.chunk;
  for (int g = threadIdx.x >> 5; g < a.group; g += kJoinThreads / 32) {
    const float2 st = join_stats(a.part_ml + (b * a.q_heads + head * a.group + g) * a.chunks, n, lane);
    if (lane == 0) stats[g] = make_float2(st.x, st.y == 0.f ? 0.f : 1.f / st.y);
  }
  __syncthreads();
  for (int j = blockIdx.x * kJoinThreads + threadIdx.x; j < length; j += gridDim.x * kJoinThreads) {
    float sum = 0.f;
    for (int g = 0; g < a.group; ++g) {
      const int ht = g / tile_heads;
      const float s = a.scores[(((b * heads + head) * a.head_tiles + ht) * a.score_tokens + j) * tile_heads + g % tile_heads];
      sum += s == -INFINITY ? 0.f : exp2f((s - stats[g].x) * kLog2e) * stats[g].y;
    }
    a.weights[(b * heads + head) * a.weights_width + j] += sum;
  }
}

// How a call is split: query heads in tiles of 8 (16 for bf16 queries of more than 8 heads a group and head_dim <= 128),
// the length in chunks so that the launch has about two CTAs' worth of work for each of the four a SM holds.
struct Plan {
  int nt, head_tiles, chunk, chunks;
};
static Plan plan_of(int dtype, int dim, int64_t group, int64_t heads, int64_t batch, int64_t tokens) {
  Plan p;
  p.nt = dtype == MXQ_BF16 && group > 8 && dim <= 128 ? 2 : 1;
  p.head_tiles = (int)((group + 8 * p.nt - 1) / (8 * p.nt));
  const int64_t rows = heads * p.head_tiles * batch;
  int64_t chunk = (tokens * rows + gemm::sm_count() * 8 - 1) / (gemm::sm_count() * 8);
  chunk = (chunk + 63) / 64 * 64;
  if (chunk < 64) chunk = 64;
  p.chunk = (int)chunk;
  p.chunks = (int)((tokens + chunk - 1) / chunk);
  return p;
}
struct Workspace {
  int64_t ml, o, scores, total;  // byte offsets
};
static Workspace workspace_of(const Plan &p, int64_t batch, int64_t heads, int64_t q_heads, int dim, int64_t tokens,
                              bool weights) {
  Workspace w;
  auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
  const bool parts = p.chunks > 1 || weights;
  w.ml = 0;
  w.o = parts ? up(batch * q_heads * p.chunks * (int64_t)sizeof(float2)) : 0;
  w.scores = w.o + (parts ? up(batch * q_heads * p.chunks * (int64_t)dim * 4) : 0);
  w.total = w.scores + (weights ? batch * heads * p.head_tiles * tokens * (8 * p.nt) * 4 : 0);
  return w;
}

template <typename T, int kFormat, int D>
static void launch_attention(const Cache &c, const Table &t, const AttnArgs &a, const Plan &p, int64_t batch,
                             cudaStream_t st) {
  const dim3 grid((unsigned)p.chunks, (unsigned)(c.heads * p.head_tiles), (unsigned)batch);
  if constexpr (Elem<T>::kBf16 && D <= 128) {
    if (p.nt == 2) {
      attention_kernel<T, kFormat, D, 2><<<grid, kWarps * 32, 0, st>>>(c, t, a);
      return;
    }
  }
  attention_kernel<T, kFormat, D, 1><<<grid, kWarps * 32, 0, st>>>(c, t, a);
}
template <typename T>
static void launch_attention(int format, int dim, const Cache &c, const Table &t, const AttnArgs &a, const Plan &p,
                             int64_t batch, cudaStream_t st) {
#define CALL(f)                                                              \
  if (format == f) {                                                         \
    if (dim == 32) launch_attention<T, f, 32>(c, t, a, p, batch, st);        \
    if (dim == 64) launch_attention<T, f, 64>(c, t, a, p, batch, st);        \
    if (dim == 128) launch_attention<T, f, 128>(c, t, a, p, batch, st);      \
    if (dim == 256) launch_attention<T, f, 256>(c, t, a, p, batch, st);      \
  }
  MXQ_PAGED_FORMATS(CALL)
#undef CALL
}

}  // namespace paged
}  // namespace mxq

using namespace mxq;
using namespace mxq::paged;

// Checks shared by the size query and the call; `group` comes back.
static int check_attention(const mxq_paged_cache *cache, int64_t batch, int64_t q_heads, int64_t table_width, int page_log2,
                           int64_t &group) {
  if (batch < 0 || batch > 65535 || q_heads < 1 || q_heads > 65535 || q_heads % cache->heads) return MXQ_ERR_SHAPE;
  if (table_width < 1 || table_width > (INT32_MAX >> page_log2)) return MXQ_ERR_SHAPE;
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
    const Plan p = plan_of(dtype, cache->head_dim, group, c.heads, batch, tokens);
    const int64_t n = workspace_of(p, batch, c.heads, q_heads, cache->head_dim, tokens, with_weights != 0).total;
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
  if (weights && weights_width < 1) return MXQ_ERR_SHAPE;
  const int dim = cache->head_dim;
  const int64_t tokens = table_width << c.page_log2;
  const Plan p = plan_of(dtype, dim, group, c.heads, batch, tokens);
  if ((int64_t)c.heads * p.head_tiles > 65535) return MXQ_ERR_SHAPE;
  const Workspace w = workspace_of(p, batch, c.heads, q_heads, dim, tokens, weights != nullptr);
  if (w.total > 0) {
    if (!workspace) return MXQ_ERR_NULL;
    if (!aligned(workspace, 16)) return MXQ_ERR_ALIGN;
    if (workspace_bytes < w.total) return MXQ_ERR_SHAPE;
  }
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  AttnArgs a;
  a.q = q, a.out = out, a.q_stride_b = q_stride_b, a.q_stride_h = q_stride_h, a.scaling = scaling;
  a.group = (int)group, a.q_heads = (int)q_heads, a.head_tiles = p.head_tiles;
  a.lengths = lengths;
  a.most = weights && weights_width < tokens ? weights_width : tokens;
  a.chunk = p.chunk, a.chunks = p.chunks;
  const bool parts = p.chunks > 1 || weights != nullptr;
  a.part_ml = parts ? reinterpret_cast<float2 *>(ws + w.ml) : nullptr;
  a.part_o = parts ? reinterpret_cast<float *>(ws + w.o) : nullptr;
  a.scores = weights ? reinterpret_cast<float *>(ws + w.scores) : nullptr;
  a.score_tokens = tokens;
  a.weights = weights, a.weights_width = weights_width, a.status = status;
  const Table t{page_table, table_stride, table_width};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == MXQ_BF16)
    launch_attention<__nv_bfloat16>(cache->format, dim, c, t, a, p, batch, st);
  else
    launch_attention<float>(cache->format, dim, c, t, a, p, batch, st);
  if (cudaGetLastError() != cudaSuccess) return MXQ_ERR_LAUNCH;
  if (!parts) return MXQ_OK;
  const dim3 join_grid((unsigned)q_heads, (unsigned)batch);
  if (dtype == MXQ_BF16)
    join_kernel<__nv_bfloat16><<<join_grid, kJoinThreads, 0, st>>>(a, dim);
  else
    join_kernel<float><<<join_grid, kJoinThreads, 0, st>>>(a, dim);
  if (cudaGetLastError() != cudaSuccess) return MXQ_ERR_LAUNCH;
  if (weights) {
    int64_t x = (tokens + kJoinThreads - 1) / kJoinThreads;
    const int64_t cap = ((int64_t)gemm::sm_count() * 16 + c.heads * batch - 1) / (c.heads * batch);
    if (x > cap) x = cap;
    weights_kernel<<<dim3((unsigned)x, (unsigned)c.heads, (unsigned)batch), kJoinThreads, group * sizeof(float2), st>>>(
        a, c.heads, 8 * p.nt);
    if (cudaGetLastError() != cudaSuccess) return MXQ_ERR_LAUNCH;
  }
  return MXQ_OK;
}

}  // extern "C"
