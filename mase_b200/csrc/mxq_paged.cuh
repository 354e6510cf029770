// What the kernels of the paged key/value cache share: the cache's geometry, page lookup, and the row formats.
#pragma once

#include "mxq_common.cuh"

namespace mxq {
namespace paged {

constexpr int kMostTokens = 1 << 30;  // of a page table: token counts and what lies a few units behind fit 32 bits
constexpr int kStatusBadPage = 8;  // a page table entry or a length points outside of the cache

// Geometry of one cache; sides: 0 = keys, 1 = values.
struct Cache {
  uint8_t *codes[2];
  uint8_t *scales[2];
  int64_t pages;
  int heads, page_log2;
  int bits;  // MXINT mantissa bits
};
struct Table {
  const int32_t *entries;
  int64_t stride, width;
};

inline int log2_of(int v) {
  int k = 0;
  while ((1 << k) < v) ++k;
  return k;
}
inline bool aligned(const void *p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

inline int row_bytes_of(int format, int dim) {
  return format == MXQ_CACHE_BF16 ? 2 * dim : (format == MXQ_CACHE_E2M1X2 ? dim / 2 : dim);
}

// Checks a caller's cache description and fills the kernels' one in.
inline int read_cache(const mxq_paged_cache *c, Cache &out) {
  if (!c || !c->key || !c->value) return MXQ_ERR_NULL;
  if (c->format < MXQ_CACHE_BF16 || c->format > MXQ_CACHE_INT8) return MXQ_ERR_FORMAT;
  if (c->format == MXQ_CACHE_INT8 && (c->bits < 2 || c->bits > 8)) return MXQ_ERR_FORMAT;
  if (c->format != MXQ_CACHE_BF16 && (!c->key_scales || !c->value_scales)) return MXQ_ERR_NULL;
  if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return MXQ_ERR_UNSUPPORTED;
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1))) return MXQ_ERR_UNSUPPORTED;
  if (c->heads < 1 || c->heads > 32767 || c->pages < 0 || c->pages > INT32_MAX) return MXQ_ERR_SHAPE;
  if (!aligned(c->key, 16) || !aligned(c->value, 16) || !aligned(c->key_scales, 16) || !aligned(c->value_scales, 16))
    return MXQ_ERR_ALIGN;
  out.codes[0] = static_cast<uint8_t *>(c->key), out.codes[1] = static_cast<uint8_t *>(c->value);
  out.scales[0] = c->key_scales, out.scales[1] = c->value_scales;
  out.pages = c->pages, out.heads = c->heads, out.page_log2 = log2_of(c->page_size), out.bits = c->bits;
  return MXQ_OK;
}
inline int read_table(const int32_t *table, int64_t width, int64_t stride, int64_t batch, int page_log2) {
  if (!table) return MXQ_ERR_NULL;
  if (width < 1 || stride < 0 || (batch > 1 && stride < width)) return MXQ_ERR_SHAPE;
  if (batch < 0 || batch > 65535 || width > (kMostTokens >> page_log2)) return MXQ_ERR_SHAPE;
  return MXQ_OK;
}

__device__ __forceinline__ void report(int *status) {
  if (status != nullptr) *status = kStatusBadPage;
}
// A sequence's length clamped to what its table (and statistics) can hold.
__device__ __forceinline__ int clamp_length(int length, int64_t most, int *status) {
  if (length < 0 || length > most) {
    report(status);
    return length < 0 ? 0 : (int)most;
  }
  return length;
}
// First row (in units of rows of the whole cache) of the page that holds `slot` of sequence b for `head`; -1 when the
// table names no page of the cache.
__device__ __forceinline__ int64_t page_row(const Cache &c, const Table &t, int64_t b, int head, int slot, int *status) {
  const int page = t.entries[b * t.stride + (slot >> c.page_log2)];
  if (page < 0 || page >= c.pages) {
    report(status);
    return -1;
  }
  return ((int64_t)page * c.heads + head) << c.page_log2;
}

// ---- row formats -----------------------------------------------------------------------------------------------------
template <int kFormat>
struct Format;
template <>
struct Format<MXQ_CACHE_BF16> {
  static constexpr int kBits = 16, E = 0, F = 0;
};
template <>
struct Format<MXQ_CACHE_E4M3> {
  static constexpr int kBits = 8, E = 4, F = 3;
};
template <>
struct Format<MXQ_CACHE_E5M2> {
  static constexpr int kBits = 8, E = 5, F = 2;
};
template <>
struct Format<MXQ_CACHE_E2M1X2> {
  static constexpr int kBits = 4, E = 2, F = 1;
};
template <>
struct Format<MXQ_CACHE_INT8> {
  static constexpr int kBits = 8, E = 0, F = 0;
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
// The raw bf16 pattern of a code stands for raw = value * 2^-offset in units of the block scale, so a block's factor is
// 2^(scale - 127 + offset), in bf16 the exponent field scale + offset.  That field is out of [1, 254] for MXFP blocks with
// a scale far above one and for MXINT blocks at either end: those tiles take a second factor (kRare).
template <int kFormat>
__device__ __forceinline__ int raw_offset(int bits) {
  if constexpr (kFormat == MXQ_CACHE_INT8)
    return 1 - bits;
  else if constexpr (kFormat == MXQ_CACHE_BF16)
    return 0;
  else
    return 127 - ((1 << (Format<kFormat>::E - 1)) - 1);
}
template <int kFormat>
__device__ __forceinline__ bool rare_scale(uint32_t scale, int offset) {
  if constexpr (kFormat == MXQ_CACHE_INT8)
    return (int)scale + offset < 1 || scale == 255u;
  else
    return (int)scale + offset > 254;
}
// first factor of a rare block (bf16 pattern): the field clamped to 254; for MXINT also subnormal powers, and infinity
// for scale byte 255 (the reference multiplies the zero mantissas of such a block by 2^128)
template <int kFormat>
__device__ __forceinline__ uint32_t rare_factor(uint32_t scale, int offset) {
  const int field = (int)scale + offset;
  if constexpr (kFormat == MXQ_CACHE_INT8) {
    if (scale == 255u) return 0x7F80u;
    return field >= 1 ? (uint32_t)field << 7 : (field > -7 ? 1u << (field + 6) : 0u);
  }
  return (uint32_t)min(field, 254) << 7;
}
template <int kFormat>
__device__ __forceinline__ uint32_t rare_rest(uint32_t scale, int offset) {
  return (uint32_t)(127 + max((int)scale + offset - 254, 0)) << 7;
}

template <bool kRare>
__device__ __forceinline__ uint32_t scaled(uint32_t raw, uint32_t f, uint32_t rest) {
  raw = mul2(raw, f);
  return kRare ? mul2(raw, rest) : raw;
}

__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {  // one instruction
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(x), "r"(mask), "r"(bits));
  return d;
}
// 8-bit codes of bytes 0 and 2 (even) or 1 and 3 (odd) of a word -> raw bf16 pair: the sign to bit 15, exponent and
// fraction fields down to the bf16 fraction boundary.  Shifts to the left run beside the half-rate logic unit.
template <int kFormat>
__device__ __forceinline__ uint32_t raw_even(uint32_t w) {
  if constexpr (kFormat == MXQ_CACHE_E4M3)
    return and_or(w << 8, 0x80008000u, (w << 4) & 0x07F007F0u);
  else
    return and_or(w << 8, 0x80008000u, (w << 5) & 0x0FE00FE0u);
}
template <int kFormat>
__device__ __forceinline__ uint32_t raw_odd(uint32_t w) {
  if constexpr (kFormat == MXQ_CACHE_E4M3)
    return and_or(w, 0x80008000u, (w >> 4) & 0x07F007F0u);
  else
    return and_or(w, 0x80008000u, (w >> 3) & 0x0FE00FE0u);
}
// E2M1 codes of nibble i of each half -> raw bf16 pair
template <int i>
__device__ __forceinline__ uint32_t raw_nibble(uint32_t w) {
  if constexpr (i == 0) return and_or(w << 12, 0x80008000u, (w << 6) & 0x01C001C0u);
  if constexpr (i == 1) return and_or(w << 8, 0x80008000u, (w << 2) & 0x01C001C0u);
  if constexpr (i == 2) return and_or(w << 4, 0x80008000u, (w >> 2) & 0x01C001C0u);
  return and_or(w, 0x80008000u, (w >> 6) & 0x01C001C0u);
}
// Two int8, one in the lower byte of each half -> bf16 pair: 128 + (u & 127) minus 128 or 256 by the sign bit.
__device__ __forceinline__ uint32_t int8_lower(uint32_t x) {
  return sub2(and_or(x, 0x007F007Fu, 0x43004300u), and_or(x, 0x00800080u, 0x43004300u));
}

// One word of a key row -> bf16 pairs.  Halves of pair i of the word are these elements, from the word's first one:
//   16 bit: 0, 1;  8 bit: i, i + 2;  4 bit: i, i + 4
template <int kFormat>
__device__ __forceinline__ int pair_element(int i, int half) {
  return kFormat == MXQ_CACHE_BF16 ? half : i + half * (16 / Format<kFormat>::kBits);
}
template <int kFormat, bool kRare>
__device__ __forceinline__ void key_word(uint32_t w, uint32_t f, uint32_t rest, uint32_t *out) {
  if constexpr (kFormat == MXQ_CACHE_BF16) {
    out[0] = w;
  } else if constexpr (kFormat == MXQ_CACHE_INT8) {
    out[0] = scaled<kRare>(int8_lower(w), f, rest), out[1] = scaled<kRare>(int8_lower(w >> 8), f, rest);
  } else if constexpr (Format<kFormat>::kBits == 8) {
    out[0] = scaled<kRare>(raw_even<kFormat>(w), f, rest), out[1] = scaled<kRare>(raw_odd<kFormat>(w), f, rest);
  } else {
    out[0] = scaled<kRare>(raw_nibble<0>(w), f, rest), out[1] = scaled<kRare>(raw_nibble<1>(w), f, rest);
    out[2] = scaled<kRare>(raw_nibble<2>(w), f, rest), out[3] = scaled<kRare>(raw_nibble<3>(w), f, rest);
  }
}
// The same word of two value rows -> pairs (row a, row b) of its elements 0, 1, 2, ...
template <int kFormat, bool kRare>
__device__ __forceinline__ void value_words(uint32_t a, uint32_t b, uint32_t f, uint32_t rest, uint32_t *out) {
  constexpr int kHalf = 16 / Format<kFormat>::kBits;  // elements of half a word
  // halves of the two words side by side: the key's pairs of such a word are the wanted ones
  key_word<kFormat, kRare>(__byte_perm(a, b, 0x5410), f, rest, out);
  key_word<kFormat, kRare>(__byte_perm(a, b, 0x7632), f, rest, out + kHalf);
}

// ---- launches --------------------------------------------------------------------------------------------------------
// The kernels are launched with programmatic stream serialization: a kernel's CTAs may be set up while the kernel before
// it drains, and wait here, before they read or write anything, until it has finished.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... P, typename... V>
static int launch_chained(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, int cluster, V &&...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid, cfg.blockDim = dim3((unsigned)threads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = cluster > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kernel, P(args)...) != cudaSuccess) {
    cudaGetLastError();
    return MXQ_ERR_LAUNCH;
  }
  return MXQ_OK;
}

#define MXQ_PAGED_FORMATS(CALL)                                                                             \
  CALL(MXQ_CACHE_BF16) CALL(MXQ_CACHE_E4M3) CALL(MXQ_CACHE_E5M2) CALL(MXQ_CACHE_E2M1X2) CALL(MXQ_CACHE_INT8)

}  // namespace paged
}  // namespace mxq
