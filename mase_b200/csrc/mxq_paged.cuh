// What the kernels of the paged key/value cache share: the cache's geometry, page lookup, and the row formats.
#pragma once

#include "mxq_common.cuh"

namespace mxq {
namespace paged {

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
  if (batch < 0 || batch > 65535 || width > (INT32_MAX >> page_log2)) return MXQ_ERR_SHAPE;
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
// Four 8-bit codes -> upper and lower bytes of their raw bf16 patterns: sign, then exponent and fraction fields moved down
// to the bf16 fraction boundary.
template <int kFormat>
__device__ __forceinline__ void split_bytes(uint32_t w, uint32_t &hi, uint32_t &lo) {
  if constexpr (kFormat == MXQ_CACHE_E4M3) {
    hi = and_or(w, 0x80808080u, (w >> 4) & 0x07070707u), lo = (w << 4) & 0xF0F0F0F0u;
  } else {
    hi = and_or(w, 0x80808080u, (w >> 3) & 0x0F0F0F0Fu), lo = (w << 5) & 0xE0E0E0E0u;
  }
}
// Eight E2M1 codes -> the same bytes of the even (0, 2, 4, 6) and odd (1, 3, 5, 7) ones.
__device__ __forceinline__ void split_nibbles(uint32_t w, uint32_t &hi_even, uint32_t &lo_even, uint32_t &hi_odd,
                                              uint32_t &lo_odd) {
  hi_even = and_or(w << 4, 0x80808080u, (w >> 2) & 0x01010101u), lo_even = (w << 6) & 0xC0C0C0C0u;
  hi_odd = and_or(w, 0x80808080u, (w >> 6) & 0x01010101u), lo_odd = (w << 2) & 0xC0C0C0C0u;
}
// Two int8, one in the lower byte of each half -> bf16 pair: 128 + (u & 127) minus 128 or 256 by the sign bit.
__device__ __forceinline__ uint32_t int8_lower(uint32_t x) {
  return sub2(and_or(x, 0x007F007Fu, 0x43004300u), and_or(x, 0x00800080u, 0x43004300u));
}

// One word of a key row -> bf16 pairs.  Halves of pair i of the word are these elements, from the word's first one:
//   16 bit: 0, 1;  E4M3 / E5M2: 2 i, 2 i + 1;  int8: i, i + 2;  E2M1: 4 (i & 1) + (i >> 1) and that + 2
template <int kFormat>
__device__ __forceinline__ int pair_element(int i, int half) {
  if (kFormat == MXQ_CACHE_INT8) return i + 2 * half;
  if (kFormat == MXQ_CACHE_E2M1X2) return 4 * (i & 1) + (i >> 1) + 2 * half;
  return 2 * i + half;
}
template <int kFormat, bool kRare>
__device__ __forceinline__ void key_word(uint32_t w, uint32_t f, uint32_t rest, uint32_t *out) {
  if constexpr (kFormat == MXQ_CACHE_BF16) {
    out[0] = w;
  } else if constexpr (kFormat == MXQ_CACHE_INT8) {
    out[0] = scaled<kRare>(int8_lower(w), f, rest), out[1] = scaled<kRare>(int8_lower(w >> 8), f, rest);
  } else if constexpr (Format<kFormat>::kBits == 8) {
    uint32_t hi, lo;
    split_bytes<kFormat>(w, hi, lo);
    out[0] = scaled<kRare>(__byte_perm(lo, hi, 0x5140), f, rest), out[1] = scaled<kRare>(__byte_perm(lo, hi, 0x7362), f, rest);
  } else {
    uint32_t he, le, ho, lo;
    split_nibbles(w, he, le, ho, lo);
    out[0] = scaled<kRare>(__byte_perm(le, he, 0x5140), f, rest), out[1] = scaled<kRare>(__byte_perm(le, he, 0x7362), f, rest);
    out[2] = scaled<kRare>(__byte_perm(lo, ho, 0x5140), f, rest), out[3] = scaled<kRare>(__byte_perm(lo, ho, 0x7362), f, rest);
  }
}
// The same word of two value rows -> pairs (row a, row b) of its elements 0, 1, 2, ...
template <int kFormat, bool kRare>
__device__ __forceinline__ void value_words(uint32_t a, uint32_t b, uint32_t f, uint32_t rest, uint32_t *out) {
  if constexpr (kFormat == MXQ_CACHE_BF16) {
    out[0] = __byte_perm(a, b, 0x5410), out[1] = __byte_perm(a, b, 0x7632);
  } else if constexpr (kFormat == MXQ_CACHE_INT8) {
    out[0] = scaled<kRare>(int8_lower(__byte_perm(a, b, 0x4400)), f, rest);
    out[1] = scaled<kRare>(int8_lower(__byte_perm(a, b, 0x5511)), f, rest);
    out[2] = scaled<kRare>(int8_lower(__byte_perm(a, b, 0x6622)), f, rest);
    out[3] = scaled<kRare>(int8_lower(__byte_perm(a, b, 0x7733)), f, rest);
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t x = __byte_perm(a, b, h ? 0x7362 : 0x5140);  // bytes a, b, a, b of neighbouring positions
      if constexpr (Format<kFormat>::kBits == 8) {
        uint32_t hi, lo;
        split_bytes<kFormat>(x, hi, lo);
        out[2 * h] = scaled<kRare>(__byte_perm(lo, hi, 0x5140), f, rest);
        out[2 * h + 1] = scaled<kRare>(__byte_perm(lo, hi, 0x7362), f, rest);
      } else {
        uint32_t he, le, ho, lo;
        split_nibbles(x, he, le, ho, lo);
        out[4 * h] = scaled<kRare>(__byte_perm(le, he, 0x5140), f, rest);
        out[4 * h + 1] = scaled<kRare>(__byte_perm(lo, ho, 0x5140), f, rest);
        out[4 * h + 2] = scaled<kRare>(__byte_perm(le, he, 0x7362), f, rest);
        out[4 * h + 3] = scaled<kRare>(__byte_perm(lo, ho, 0x7362), f, rest);
      }
    }
  }
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
