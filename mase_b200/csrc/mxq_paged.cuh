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

#define MXQ_PAGED_FORMATS(CALL)                                                                             \
  CALL(MXQ_CACHE_BF16) CALL(MXQ_CACHE_E4M3) CALL(MXQ_CACHE_E5M2) CALL(MXQ_CACHE_E2M1X2) CALL(MXQ_CACHE_INT8)

}  // namespace paged
}  // namespace mxq
