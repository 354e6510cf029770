// Paged key/value cache in MX formats: writing new rows (mxq_paged_append), reading rows back (mxq_paged_gather) and
// evicting the tokens with the least accumulated attention weight (mxq_paged_evict).

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "mxq.h"
#include "mxq_common.cuh"
#include "mxq_internal.h"
#include "mxq_pack.cuh"
#include "mxq_paged.cuh"

namespace mxq {
namespace paged {

constexpr int kThreads = 256;

// ---- append ----------------------------------------------------------------------------------------------------------
// Two neighbouring lanes share a block of 32 elements, 16 each; the codes and the shared exponent are those of the plain
// quantizers (the bf16 routines are the ones behind mxq_mxfp_extract / mxq_mxint_extract).  Bound by the logic unit
// (about 18 instructions an element) with reads and page lookups in flight under it: 4 x 2048 tokens x 8 heads of 128, bf16
// to E4M3: 19 us, and 12 us for the read-back of what is cached then (105 MB in both, 28 us in a row).
struct AppendArgs {
  const void *src[2];
  int64_t stride_b[2], stride_h[2], stride_t[2];
  const int32_t *lengths, *counts, *next_position;
  int32_t *positions;
  int64_t positions_width;
  int64_t tokens;
  int *status;
};

__device__ __forceinline__ void load16(const float *p, float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 r = reinterpret_cast<const float4 *>(p)[i];
    v[4 * i] = r.x, v[4 * i + 1] = r.y, v[4 * i + 2] = r.z, v[4 * i + 3] = r.w;
  }
}
__device__ __forceinline__ uint4 bytes_of(const uint32_t (&c)[16]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = (c[4 * i] & 0xFFu) | (c[4 * i + 1] & 0xFFu) << 8 | (c[4 * i + 2] & 0xFFu) << 16 | c[4 * i + 3] << 24;
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// MXFP codes of 16 elements by the element codec, with the block maximum over the neighbouring lane's half too; returns the
// scale byte.
template <int kFormat>
__device__ __forceinline__ int encode_elements(const float (&v)[16], const Log2Tab &tab, uint32_t (&code)[16]) {
  using Fmt = Format<kFormat>;
  uint32_t amax = 0;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const uint32_t a = __float_as_uint(v[k]) & 0x7FFFFFFFu;
    amax = max(amax, (a >> 23) == 0 ? 0u : a);
  }
  amax = group_max(amax, 2);
  const MxfpBlock b = mxfp_block(amax, Fmt::E, tab);
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const uint32_t r = __float_as_uint(v[k]);
    code[k] = mxfp_encode(((r & 0x7FFFFFFFu) >> 23) == 0 ? 0u : r, b.sh, Fmt::E, Fmt::F);
  }
  return b.scale;
}

// Half a block of 32 elements: loaded, and turned into codes (one per byte) and the block's scale byte together with the
// neighbouring lane's half.  Every lane of the warp calls encode().
template <typename T>
struct Half;
template <>
struct Half<__nv_bfloat16> {
  uint4 lo, hi;
  __device__ __forceinline__ void clear() { lo = hi = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void load(const __nv_bfloat16 *p) {
    lo = ld_stream(reinterpret_cast<const uint4 *>(p)), hi = ld_stream(reinterpret_cast<const uint4 *>(p) + 1);
  }
  __device__ __forceinline__ void store_bf16(uint4 *d) const { d[0] = lo, d[1] = hi; }
  template <int kFormat>
  __device__ __forceinline__ uint4 encode(int bits, const Log2Tab &tab, int &scale) const {
    if constexpr (kFormat == MXQ_CACHE_INT8) {
      return mxint_codes_bf16(lo, hi, tab, bits, scale);
    } else if constexpr (Format<kFormat>::kBits == 4) {
      // with the four exponents of E2M1 nearly every block has subnormal codes, which the other routine patches one by one:
      // 16 heads x 4096 tokens of 128 with the read-back 55 us, 58 with it (E4M3 27)
      float v[16];
      uint32_t b[8], code[16];
      unpack(lo, b);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = __uint_as_float(b[k]);
      unpack(hi, b);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[8 + k] = __uint_as_float(b[k]);
      scale = encode_elements<kFormat>(v, tab, code);
      return bytes_of(code);
    } else
      return codes_bf16<Format<kFormat>::E, Format<kFormat>::F>(lo, hi, tab, scale);
  }
};
template <>
struct Half<float> {
  float v[16];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = 0.f;
  }
  __device__ __forceinline__ void load(const float *p) { load16(p, v); }
  __device__ __forceinline__ void store_bf16(uint4 *d) const {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      d[k] = make_uint4(pack_bf16x2(v[8 * k], v[8 * k + 1]), pack_bf16x2(v[8 * k + 2], v[8 * k + 3]),
                        pack_bf16x2(v[8 * k + 4], v[8 * k + 5]), pack_bf16x2(v[8 * k + 6], v[8 * k + 7]));
  }
  template <int kFormat>
  __device__ __forceinline__ uint4 encode(int bits, const Log2Tab &tab, int &scale) const {
    uint32_t code[16];
    if constexpr (kFormat == MXQ_CACHE_INT8) {
      float amax = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) amax = fmaxf(amax, fabsf(v[k]));
      amax = group_max(amax, 2);
      const MxintBlock b = mxint_block<false>(amax, bits, tab);
      scale = b.scale;
#pragma unroll
      for (int k = 0; k < 16; ++k) code[k] = (uint32_t)(int)mxint_mant(v[k], b);
    } else {
      scale = encode_elements<kFormat>(v, tab, code);
    }
    return bytes_of(code);
  }
};

// grid: (chunks of the units of one (sequence, head), heads * 2 sides, batch); a unit is half a block of one token, and a
// thread has two in flight: the reads of the rows and of the page table do not depend on one another.
template <typename T, int kFormat>
__global__ void __launch_bounds__(kThreads, Elem<T>::kBf16 ? 4 : 2)
append_kernel(const Cache c, const Table table, const AppendArgs a, int dim_log2, const __grid_constant__ Log2Tab tab) {
  using Fmt = Format<kFormat>;
  constexpr int kAtOnce = 2;
  wait_for_previous();
  let_next_start();
  const int side = blockIdx.y & 1, head = blockIdx.y >> 1, dim = 1 << dim_log2;
  const int64_t b = blockIdx.z;
  const int units_log2 = dim_log2 - 4;  // 2, 4, 8 or 16 units a token: a pair of lanes never straddles two rows
  const int64_t most = table.width << c.page_log2;
  const int length = clamp_length(a.lengths[b], most, a.status);
  int64_t count = a.counts != nullptr ? a.counts[b] : a.tokens;
  if (count < 0 || count > a.tokens || length + count > most) {
    report(a.status);
    count = count < 0 ? 0 : min(min(count, a.tokens), most - length);
  }
  const int64_t stride_t = side ? a.stride_t[1] : a.stride_t[0];
  const T *src = static_cast<const T *>(side ? a.src[1] : a.src[0]) + b * (side ? a.stride_b[1] : a.stride_b[0]) +
                 head * (side ? a.stride_h[1] : a.stride_h[0]);
  uint8_t *codes = side ? c.codes[1] : c.codes[0], *scales = side ? c.scales[1] : c.scales[0];
  const int total = (int)count << units_log2;  // at most 2^26 tokens of 16 units
  const int step = gridDim.x * (kThreads * kAtOnce);
  for (int base = blockIdx.x * (kThreads * kAtOnce); base < total; base += step) {
    int64_t row[kAtOnce];
    Half<T> raw[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int i = base + k * kThreads + threadIdx.x, t = i >> units_log2, u = i & ((1 << units_log2) - 1);
      row[k] = -1;
      raw[k].clear();
      if (i < total) {
        raw[k].load(src + t * stride_t + u * 16);
        const int slot = length + t;
        row[k] = page_row(c, table, b, head, slot, a.status);
        if (row[k] >= 0) row[k] += slot & ((1 << c.page_log2) - 1);
        if (side == 0 && u == 0 && a.positions != nullptr) {
          if (slot < a.positions_width)
            a.positions[(b * c.heads + head) * a.positions_width + slot] =
                (a.next_position != nullptr ? a.next_position[b] : length) + t;
          else
            report(a.status);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int u = (base + k * kThreads + threadIdx.x) & ((1 << units_log2) - 1);
      if constexpr (kFormat == MXQ_CACHE_BF16) {
        if (row[k] >= 0) raw[k].store_bf16(reinterpret_cast<uint4 *>(codes + row[k] * (dim * 2) + u * 32));
      } else {
        int scale;
        const uint4 code = raw[k].template encode<kFormat>(c.bits, tab, scale);
        if (row[k] >= 0) {
          if constexpr (Fmt::kBits == 4) {
            uint32_t w[4] = {code.x, code.y, code.z, code.w};
#pragma unroll
            for (int x = 0; x < 4; ++x) w[x] |= w[x] >> 4;  // bytes 0 and 2 now hold two codes each
            *reinterpret_cast<uint2 *>(codes + row[k] * (dim / 2) + u * 8) =
                make_uint2(__byte_perm(w[0], w[1], 0x6420), __byte_perm(w[2], w[3], 0x6420));
          } else {
            *reinterpret_cast<uint4 *>(codes + row[k] * dim + u * 16) = code;
          }
          if ((u & 1) == 0) scales[row[k] * (dim >> 5) + (u >> 1)] = (uint8_t)scale;
        }
      }
    }
  }
}

// ---- gather ----------------------------------------------------------------------------------------------------------
// 32 bytes, aligned to 32
__device__ __forceinline__ void store32(void *p, const uint32_t (&w)[8]) {
  asm volatile("st.global.cs.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// 16 elements of a block as 8 bf16 pairs in order.  The values are codes times a power of two: exact in bf16 unless the
// block's scale lies at an end of the range (kRare), where the second factor or the rounding to subnormals takes part.
template <int kFormat, bool kRare>
__device__ __forceinline__ void decode16(const uint8_t *p, uint32_t scale, int bits, uint32_t (&out)[8]) {
  if constexpr (kFormat == MXQ_CACHE_BF16) {
    const uint4 lo = ld_stream(reinterpret_cast<const uint4 *>(p)), hi = ld_stream(reinterpret_cast<const uint4 *>(p) + 1);
    out[0] = lo.x, out[1] = lo.y, out[2] = lo.z, out[3] = lo.w, out[4] = hi.x, out[5] = hi.y, out[6] = hi.z, out[7] = hi.w;
  } else {
    const int offset = raw_offset<kFormat>(bits);
    const uint32_t f = kRare ? rare_factor<kFormat>(scale, offset) * 0x00010001u : (uint32_t)((int)scale + offset) * 0x00800080u;
    const uint32_t rest = kRare ? rare_rest<kFormat>(scale, offset) * 0x00010001u : 0u;
    uint32_t e[8];
    if constexpr (Format<kFormat>::kBits == 4) {
      const uint2 r = __ldcs(reinterpret_cast<const uint2 *>(p));
      key_word<kFormat, kRare>(r.x, f, rest, e), key_word<kFormat, kRare>(r.y, f, rest, e + 4);
#pragma unroll
      for (int k = 0; k < 8; k += 4) {  // (0, 4) (1, 5) (2, 6) (3, 7) -> (0, 1) (2, 3) (4, 5) (6, 7)
        out[k] = __byte_perm(e[k], e[k + 1], 0x5410), out[k + 1] = __byte_perm(e[k + 2], e[k + 3], 0x5410);
        out[k + 2] = __byte_perm(e[k], e[k + 1], 0x7632), out[k + 3] = __byte_perm(e[k + 2], e[k + 3], 0x7632);
      }
    } else {
      const uint4 r = ld_stream(reinterpret_cast<const uint4 *>(p));
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {  // (0, 2) (1, 3) -> (0, 1) (2, 3)
        key_word<kFormat, kRare>(w[k], f, rest, e);
        out[2 * k] = __byte_perm(e[0], e[1], 0x5410), out[2 * k + 1] = __byte_perm(e[0], e[1], 0x7632);
      }
    }
  }
}
// The same in fp32, from the element codecs: for scales at which a product may be below the range of bf16.
template <int kFormat>
__device__ __forceinline__ void decode16_wide(const uint8_t *p, int scale, int bits, float (&v)[16]) {
  using Fmt = Format<kFormat>;
  const float sf = kFormat == MXQ_CACHE_INT8 ? (scale == 255 ? INFINITY : pow2f(scale - 127 - (bits - 1))) : pow2f(scale - 127);
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const uint32_t code = Fmt::kBits == 4 ? (p[k >> 1] >> (4 * (k & 1))) & 15u : p[k];
    v[k] = (kFormat == MXQ_CACHE_INT8 ? (float)(int8_t)code : mxfp_decode(code, Fmt::E, Fmt::F)) * sf;
  }
}

// Bound by HBM: one unit reads 8, 16 or 32 bytes of codes and writes 32 (bf16) or 64 bytes.
// grid: (chunks of the units of one (sequence, head), heads * 2 sides, batch); a unit is 16 elements of one token.
template <typename T, int kFormat>
__global__ void __launch_bounds__(kThreads)
gather_kernel(const Cache c, const Table table, const int32_t *lengths, T *key, T *value, int64_t tokens, int dim_log2,
              int *status) {
  using Fmt = Format<kFormat>;
  wait_for_previous();
  let_next_start();
  const int side = blockIdx.y & 1, head = blockIdx.y >> 1, dim = 1 << dim_log2;
  const int64_t b = blockIdx.z;
  const int units_log2 = dim_log2 - 4;
  const int length = clamp_length(lengths[b], table.width << c.page_log2, status);
  const uint8_t *codes = side ? c.codes[1] : c.codes[0], *scales = side ? c.scales[1] : c.scales[0];
  T *dst = (side ? value : key) + (b * c.heads + head) * tokens * dim;
  const int total = (int)tokens << units_log2;  // at most 2^26 tokens of 16 units
#pragma unroll 2
  for (int i = blockIdx.x * kThreads + threadIdx.x; i < total; i += gridDim.x * kThreads) {
    const int t = i >> units_log2, u = i & ((1 << units_log2) - 1);
    int64_t row = -1;
    if (t < length) row = page_row(c, table, b, head, t, status);
    uint32_t w[8] = {};
    T *to = dst + (int64_t)t * dim + u * 16;
    if (row >= 0) {
      row += t & ((1 << c.page_log2) - 1);
      const uint8_t *p = codes + row * (dim * Fmt::kBits / 8) + u * (2 * Fmt::kBits);
      uint32_t scale = 0;
      if constexpr (kFormat != MXQ_CACHE_BF16) scale = scales[row * (dim >> 5) + (u >> 1)];
      if constexpr (kFormat != MXQ_CACHE_BF16) {
        if (!Elem<T>::kBf16 && scale < 16) {
          float v[16];
          decode16_wide<kFormat>(p, (int)scale, c.bits, v);
#pragma unroll
          for (int k = 0; k < 16; ++k) store_scalar(to + k, v[k]);
          continue;
        }
      }
      if (kFormat != MXQ_CACHE_BF16 && rare_scale<kFormat>(scale, raw_offset<kFormat>(c.bits)))
        decode16<kFormat, true>(p, scale, c.bits, w);
      else
        decode16<kFormat, false>(p, scale, c.bits, w);
    }
    if constexpr (Elem<T>::kBf16) {
      store32(to, w);
    } else {
      uint32_t lo[8], hi[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        lo[2 * k] = w[k] << 16, lo[2 * k + 1] = w[k] & 0xFFFF0000u;
        hi[2 * k] = w[k + 4] << 16, hi[2 * k + 1] = w[k + 4] & 0xFFFF0000u;
      }
      store32(to, lo), store32(to + 8, hi);
    }
  }
}

// ---- evict -----------------------------------------------------------------------------------------------------------
// Selection: a cluster of 1 to 8 CTAs per (sequence, head), each with a contiguous part of the slots.  The weights become
// 32-bit keys whose unsigned order is the order of preference; three passes over 11 + 11 + 10 bits of the keys (a
// histogram in each CTA's shared memory, added up over the cluster) find the key of the last token kept, and every warp
// then walks a contiguous part of the slots, four neighbours a lane, so that ranks follow the slot order.  Keys live in
// shared memory when they fit and are read again from L2 otherwise.  Bound by the chain of barriers and scans, not by its
// 16 bytes a slot: 64 rows of 12000 to 16384 slots take 20 us, 8 rows of 1500 slots 8; with the moves behind it 68 and 12 us.
constexpr int kSelectThreads = 512;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kBins = 2048;
constexpr int kSlotsPerCta = 2048;  // rows of more slots are shared by a cluster
constexpr int kKeysInShared = 48 * 1024;

struct EvictArgs {
  const int32_t *lengths;
  const float *weights;
  const int32_t *positions, *next_position;
  int64_t width;
  int keep, recent, max_moves;
  int32_t *new_lengths, *new_positions;
  float *new_weights;
  int32_t *from, *to, *moves;  // workspace: [rows, max_moves] twice, [rows]
  int *status;
};

__device__ __forceinline__ uint32_t key_of(float w) {
  if (isnan(w)) return 0u;
  const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

namespace cg = cooperative_groups;

__device__ __forceinline__ int warp_total(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
__device__ __forceinline__ int warp_scan(int v) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xFFFFFFFFu, v, o);
    if ((int)(threadIdx.x & 31) >= o) v += x;
  }
  return v;
}
// exclusive prefix sum over the CTA's warps of a per-warp value held by every lane; `total` = the sum
__device__ __forceinline__ int scan_warps(int v, int *scratch, int &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  int s = lane < kSelectWarps ? scratch[lane] : 0;
#pragma unroll
  for (int o = 1; o < kSelectWarps; o <<= 1) {
    const int n = __shfl_up_sync(0xFFFFFFFFu, s, o);
    if (lane >= o) s += n;
  }
  total = __shfl_sync(0xFFFFFFFFu, s, kSelectWarps - 1);
  const int before = __shfl_sync(0xFFFFFFFFu, s, warp == 0 ? 0 : warp - 1);
  return warp == 0 ? 0 : before;
}

// grid: (heads * cluster, batch)
__global__ void __launch_bounds__(kSelectThreads)
evict_select_kernel(const Cache c, int64_t table_tokens, const EvictArgs a) {
  extern __shared__ __align__(16) uint32_t keys[];
  __shared__ __align__(16) int hist[3][kBins];  // one per pass: the CTAs of a cluster read each other's without a second barrier
  __shared__ int scratch[kSelectWarps];
  __shared__ int found[2];   // bin of the last kept key, keys in bins above it
  __shared__ int counts[3];  // of this CTA's part: keys equal to the last one, holes, movers
  cg::cluster_group cluster = cg::this_cluster();
  const int size = cluster.num_blocks(), rank = cluster.block_rank();
  wait_for_previous();
  let_next_start();
  const int head = blockIdx.x / size, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t b = blockIdx.y;
  const int64_t row = b * c.heads + head;
  const int n = clamp_length(a.lengths[b], min(table_tokens, a.width), a.status);
  const int m = min(n, a.keep);
  const float *w = a.weights + row * a.width;
  const int32_t *p = a.positions != nullptr ? a.positions + row * a.width : nullptr;
  float *nw = a.new_weights + row * a.width;
  int32_t *np = a.new_positions + row * a.width;
  if (head == 0 && rank == 0 && tid == 0) a.new_lengths[b] = m;
  for (int64_t j = m + rank * kSelectThreads + tid; j < a.width; j += size * kSelectThreads) nw[j] = 0.f, np[j] = -1;
  // this CTA's part of the slots, whole warps of it each
  const int begin = (int)min((int64_t)rank * ((n + size - 1) / size), (int64_t)n);
  const int end = min(begin + (n + size - 1) / size, n);
  if (n <= a.keep) {  // the same for every CTA of the cluster
    for (int j = begin + tid; j < end; j += kSelectThreads) nw[j] = w[j], np[j] = p != nullptr ? p[j] : j;
    if (rank == 0 && tid == 0) a.moves[row] = 0;
    return;
  }
  const int64_t first_safe = (int64_t)(p != nullptr && a.next_position != nullptr ? a.next_position[b] : n) - a.recent;
  const int mine = end - begin;
  const bool shared_keys = mine <= kKeysInShared;
  auto make_key = [&](float x, int pos) { return pos >= first_safe ? 0xFFFFFFFFu : key_of(x); };
  // keys of the four slots from begin + l on (l a multiple of 4); what lies behind the part is not used
  auto load4 = [&](int l, uint32_t (&k)[4]) {
    if (shared_keys) {
      const uint4 v = *reinterpret_cast<const uint4 *>(keys + l);
      k[0] = v.x, k[1] = v.y, k[2] = v.z, k[3] = v.w;
    } else {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int j = min(begin + l + x, end - 1);
        k[x] = make_key(w[j], p != nullptr ? p[j] : j);
      }
    }
  };
  for (int k = tid; k < 3 * kBins; k += kSelectThreads) (&hist[0][0])[k] = 0;
  __syncthreads();
  // every slot below `keep` starts out with its own statistics; the move kernel overwrites those that are filled anew
  constexpr int kBatch = 8;  // reads in flight
  for (int j0 = begin + tid; j0 < end; j0 += kSelectThreads * kBatch) {
    float x[kBatch];
    int pos[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int j = j0 + k * kSelectThreads;
      x[k] = j < end ? w[j] : 0.f, pos[k] = j < end && p != nullptr ? p[j] : j;
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int j = j0 + k * kSelectThreads;
      if (j < end) {
        if (j < m) nw[j] = x[k], np[j] = pos[k];
        const uint32_t key = make_key(x[k], pos[k]);
        if (shared_keys) keys[j - begin] = key;
        atomicAdd(&hist[0][key >> 21], 1);
      }
    }
  }

  uint32_t prefix = 0;  // the digits found so far, in place
  int need = m;         // how many of the keys that share the prefix are kept
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
    const int bins = pass == 2 ? 1024 : 2048;
    const uint32_t above = pass == 1 ? 0xFFE00000u : 0xFFFFFC00u;
    __syncthreads();
    if (pass > 0) {
      for (int l = 4 * tid; l < mine; l += 4 * kSelectThreads) {
        uint32_t k[4];
        load4(l, k);
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if ((k[x] & above) == prefix && l + x < mine) atomicAdd(&hist[pass][(k[x] >> shift) & (bins - 1)], 1);
      }
    }
    if (size > 1)
      cluster.sync();
    else
      __syncthreads();
    // thread t owns kOwn bins from bins - 1 - kOwn * t down: the running sum goes from the largest key down
    constexpr int kOwn = kBins / kSelectThreads;
    static_assert(kOwn == 4, "a thread reads its bins as one vector");
    int cnt[kOwn] = {}, s = 0;
    const int low = bins - kOwn - kOwn * tid;
    if (low >= 0)
#pragma unroll 4
      for (int r = 0; r < size; ++r) {
        const int4 h = *reinterpret_cast<const int4 *>(size > 1 ? cluster.map_shared_rank(&hist[pass][low], r) : &hist[pass][low]);
        cnt[0] += h.w, cnt[1] += h.z, cnt[2] += h.y, cnt[3] += h.x;
      }
    s = cnt[0] + cnt[1] + cnt[2] + cnt[3];
    int run = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xFFFFFFFFu, run, o);
      if (lane >= o) run += x;
    }
    int total;
    int base = scan_warps(__shfl_sync(0xFFFFFFFFu, run, 31), scratch, total) + run - s;
#pragma unroll
    for (int x = 0; x < kOwn; ++x) {
      if (base < need && base + cnt[x] >= need) found[0] = low + kOwn - 1 - x, found[1] = base;
      base += cnt[x];
    }
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    need -= found[1];
  }
  const uint32_t last = prefix;  // tokens above it are kept, and the first `need` equal to it

  // Count, for every warp's part of the slots: keys above the last one and equal to it, below and from `keep` on.
  const int part = (mine + kSelectWarps * 128 - 1) / (kSelectWarps * 128) * 128;
  const int first = min(warp * part, mine), stop = min(first + part, mine);
  const int edge = max(0, min(m - begin, mine));  // slots of this CTA before it lie below `keep`
  int more_low = 0, more_high = 0, tie_low = 0, tie_high = 0;
  for (int l = first + 4 * lane; l < stop; l += 128) {
    uint32_t k[4];
    load4(l, k);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const bool in = l + x < stop, low = l + x < edge;
      more_low += in && low && k[x] > last, more_high += in && !low && k[x] > last;
      tie_low += in && low && k[x] == last, tie_high += in && !low && k[x] == last;
    }
  }
  more_low = warp_total(more_low), more_high = warp_total(more_high);
  tie_low = warp_total(tie_low), tie_high = warp_total(tie_high);
  // sum over the CTAs before this one of one of their counts, by a whole warp
  auto before = [&](int which) { return warp_total(lane < rank ? *cluster.map_shared_rank(&counts[which], lane) : 0); };
  int total;
  int seen = scan_warps(tie_low + tie_high, scratch, total);  // ties before the warp's part
  if (size > 1) {
    if (tid == 0) counts[0] = total;
    cluster.sync();
    seen += before(0);
  }
  const int kept_ties = max(0, min(need - seen, tie_low + tie_high)), kept_low = min(kept_ties, tie_low);
  const int n_low = max(0, min(edge, stop) - first);
  int n_holes, n_movers;
  int hole_at = scan_warps(n_low - more_low - kept_low, scratch, n_holes);
  int mover_at = scan_warps(more_high + kept_ties - kept_low, scratch, n_movers);
  if (size > 1) {
    if (tid == 0) counts[1] = n_holes, counts[2] = n_movers;
    cluster.sync();
    const int holes_before = before(1);
    hole_at += holes_before, mover_at += before(2);
    if (rank == size - 1 && tid == 0) a.moves[row] = holes_before + n_holes;
  } else if (tid == 0) {
    a.moves[row] = n_holes;
  }
  int32_t *from = a.from + row * a.max_moves, *to = a.to + row * a.max_moves;
  for (int l0 = first; l0 < stop; l0 += 128) {  // the warp takes 128 slots at a time, four neighbours a lane
    const int l = l0 + 4 * lane;
    uint32_t k[4] = {};
    if (l < stop) load4(l, k);
    int ties = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x) ties += l + x < stop && k[x] == last;
    int rank_of_tie = seen;
    if (__any_sync(0xFFFFFFFFu, ties != 0)) {
      const int upto = warp_scan(ties);
      rank_of_tie += upto - ties, seen += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
    uint32_t holes = 0, movers = 0;  // bit x: slot l + x
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const bool in = l + x < stop, tie = in && k[x] == last;
      const bool kept = in && (k[x] > last || (tie && rank_of_tie < need));
      rank_of_tie += tie;
      holes |= (uint32_t)(in && !kept && l + x < edge) << x, movers |= (uint32_t)(kept && l + x >= edge) << x;
    }
    const int both = __popc(holes) | __popc(movers) << 16;
    const int upto = warp_scan(both), all = __shfl_sync(0xFFFFFFFFu, upto, 31);
    int h = hole_at + ((upto - both) & 0xFFFF), v = mover_at + ((upto - both) >> 16);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if ((holes >> x) & 1u) to[h++] = begin + l + x;
      if ((movers >> x) & 1u) from[v++] = begin + l + x;
    }
    hole_at += all & 0xFFFF, mover_at += all >> 16;
  }
  if (size > 1) cluster.sync();  // no CTA leaves while another may still read its counts
}

// A warp takes `per_warp` moves at a time (up to 32): each lane looks one of them up (slots, pages) and moves its
// statistics, then the warp copies the key and value rows of all of them, 16 bytes a lane with four copies in flight.
// Sources lie at or above `keep`, destinations below it, so moves never overlap.  Bound by HBM and the latency of rows in
// random places: 226,000 moves of two 256-byte rows, in and out, in 41 us (5.6 TB/s).  The whole eviction then takes 69 us; 102
// with eight copies in flight, 91 with seven CTAs an SM (more spills than the 28 bytes of six), 76 with four.  The same on E4M3
// pages, whose scale bytes are moved one by one: 56 us for a floor of 21; E2M1 49 us for 12.
__global__ void __launch_bounds__(kThreads, 6)
evict_move_kernel(const Cache c, const Table table, const EvictArgs a, int row_bytes_log2, int scale_bytes, int per_warp) {
  wait_for_previous();
  let_next_start();
  const int head = blockIdx.y, lane = threadIdx.x & 31;
  const int64_t b = blockIdx.z;
  const int64_t row = b * c.heads + head;
  const int n = a.moves[row];
  const int in_page = (1 << c.page_log2) - 1;
  const int32_t *from = a.from + row * a.max_moves, *to = a.to + row * a.max_moves;
  const int pieces_log2 = row_bytes_log2 - 4, pieces = 1 << pieces_log2;  // of 16 bytes
  const int stride = gridDim.x * (kThreads / 32) * per_warp;
  for (int i0 = (blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * per_warp; i0 < n; i0 += stride) {
    int64_t sr = -1, dr = -1;
    if (lane < per_warp && i0 + lane < n) {
      const int s = from[i0 + lane], d = to[i0 + lane];
      a.new_weights[row * a.width + d] = a.weights[row * a.width + s];
      a.new_positions[row * a.width + d] = a.positions != nullptr ? a.positions[row * a.width + s] : s;
      sr = page_row(c, table, b, head, s, a.status), dr = page_row(c, table, b, head, d, a.status);
      if (sr < 0 || dr < 0)
        sr = dr = -1;
      else
        sr += s & in_page, dr += d & in_page;
    }
    const int live = min(n - i0, per_warp);
    // 16-byte pieces of the moves in order: [move][side][piece]
    const int total = live << (pieces_log2 + 1);
    for (int k0 = 0; k0 < total; k0 += 128) {
      uint4 v[4];
      uint8_t *dst[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int k = k0 + x * 32 + lane, move = min(k >> (pieces_log2 + 1), 31);
        const int64_t ms = __shfl_sync(0xFFFFFFFFu, sr, move), md = __shfl_sync(0xFFFFFFFFu, dr, move);
        uint8_t *side = (k >> pieces_log2) & 1 ? c.codes[1] : c.codes[0];
        const int at = (k & (pieces - 1)) * 16;
        dst[x] = nullptr;
        if (k < total && ms >= 0) {
          v[x] = ld_stream(reinterpret_cast<const uint4 *>(side + (ms << row_bytes_log2) + at));
          dst[x] = side + (md << row_bytes_log2) + at;
        }
      }
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (dst[x] != nullptr) *reinterpret_cast<uint4 *>(dst[x]) = v[x];
    }
    if (sr >= 0)
      for (int k = 0; k < scale_bytes; ++k) {
        c.scales[0][dr * scale_bytes + k] = c.scales[0][sr * scale_bytes + k];
        c.scales[1][dr * scale_bytes + k] = c.scales[1][sr * scale_bytes + k];
      }
  }
}

// CTAs along x so that the whole grid holds about `per_sm` CTAs per SM, and no more than the work needs.
static unsigned grid_x(int64_t need, int64_t yz, int per_sm) {
  int64_t most = (int64_t)gemm::sm_count() * per_sm / yz;
  if (most < 1) most = 1;
  if (need < 1) need = 1;
  const int64_t rounds = (need + most - 1) / most;  // of every CTA, the same for all
  return (unsigned)((need + rounds - 1) / rounds);
}

}  // namespace paged
}  // namespace mxq

using namespace mxq;
using namespace mxq::paged;

extern "C" {

int mxq_paged_cache_size(void) { return (int)sizeof(mxq_paged_cache); }

int mxq_paged_append(const mxq_paged_cache *cache, const void *key, const void *value, int dtype, int64_t batch,
                     int64_t tokens, int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_t, int64_t v_stride_b,
                     int64_t v_stride_h, int64_t v_stride_t, const int32_t *page_table, int64_t table_width,
                     int64_t table_stride, const int32_t *lengths, const int32_t *counts, int32_t *positions,
                     int64_t positions_width, const int32_t *next_position, const uint8_t *log2_tab_host, int *status,
                     void *stream) {
  Cache c;
  int rc = read_cache(cache, c);
  if (rc != MXQ_OK) return rc;
  if (dtype != MXQ_F32 && dtype != MXQ_BF16) return MXQ_ERR_DTYPE;
  if (batch < 0 || tokens < 0 || tokens > (1 << 26)) return MXQ_ERR_SHAPE;
  if (batch == 0 || tokens == 0) return MXQ_OK;
  if ((rc = read_table(page_table, table_width, table_stride, batch, c.page_log2)) != MXQ_OK) return rc;
  if (!key || !value || !lengths || (!log2_tab_host && cache->format != MXQ_CACHE_BF16)) return MXQ_ERR_NULL;
  if (positions && positions_width < 1) return MXQ_ERR_SHAPE;
  const int64_t need = dtype == MXQ_BF16 ? 8 : 4;  // elements per 16 bytes
  if (!aligned(key, 16) || !aligned(value, 16) ||
      (k_stride_b | k_stride_h | k_stride_t | v_stride_b | v_stride_h | v_stride_t) % need)
    return MXQ_ERR_ALIGN;
  AppendArgs a;
  a.src[0] = key, a.src[1] = value;
  a.stride_b[0] = k_stride_b, a.stride_h[0] = k_stride_h, a.stride_t[0] = k_stride_t;
  a.stride_b[1] = v_stride_b, a.stride_h[1] = v_stride_h, a.stride_t[1] = v_stride_t;
  a.lengths = lengths, a.counts = counts, a.next_position = next_position;
  a.positions = positions, a.positions_width = positions_width, a.tokens = tokens, a.status = status;
  Log2Tab tab;
  for (int i = 0; i < 256; ++i) tab.t[i] = log2_tab_host ? log2_tab_host[i] : 0;
  const Table t{page_table, table_stride, table_width};
  const int dim = cache->head_dim;
  const int64_t yz = (int64_t)c.heads * 2 * batch;
  const dim3 grid(grid_x((tokens * (dim / 16) + 2 * kThreads - 1) / (2 * kThreads), yz, 8), c.heads * 2, (unsigned)batch);
  cudaStream_t st = (cudaStream_t)stream;
#define CALL(f)                                                                                                            \
  if (cache->format == f)                                                                                                  \
    return dtype == MXQ_BF16                                                                                               \
               ? launch_chained(append_kernel<__nv_bfloat16, f>, grid, kThreads, 0, st, 1, c, t, a, log2_of(dim), tab)        \
               : launch_chained(append_kernel<float, f>, grid, kThreads, 0, st, 1, c, t, a, log2_of(dim), tab);
  MXQ_PAGED_FORMATS(CALL)
#undef CALL
  return MXQ_ERR_FORMAT;
}

int mxq_paged_gather(const mxq_paged_cache *cache, void *key, void *value, int dtype, int64_t batch, int64_t max_tokens,
                     const int32_t *page_table, int64_t table_width, int64_t table_stride, const int32_t *lengths,
                     int *status, void *stream) {
  Cache c;
  int rc = read_cache(cache, c);
  if (rc != MXQ_OK) return rc;
  if (dtype != MXQ_F32 && dtype != MXQ_BF16) return MXQ_ERR_DTYPE;
  if (batch < 0 || max_tokens < 0 || max_tokens > (1 << 26)) return MXQ_ERR_SHAPE;
  if (batch == 0 || max_tokens == 0) return MXQ_OK;
  if ((rc = read_table(page_table, table_width, table_stride, batch, c.page_log2)) != MXQ_OK) return rc;
  if (!key || !value || !lengths) return MXQ_ERR_NULL;
  if (!aligned(key, 32) || !aligned(value, 32)) return MXQ_ERR_ALIGN;
  const Table t{page_table, table_stride, table_width};
  const int dim = cache->head_dim;
  const int64_t yz = (int64_t)c.heads * 2 * batch;
  const dim3 grid(grid_x((max_tokens * (dim / 16) + kThreads - 1) / kThreads, yz, 16), c.heads * 2, (unsigned)batch);
  cudaStream_t st = (cudaStream_t)stream;
#define CALL(f)                                                                                                             \
  if (cache->format == f)                                                                                                   \
    return dtype == MXQ_BF16 ? launch_chained(gather_kernel<__nv_bfloat16, f>, grid, kThreads, 0, st, 1, c, t, lengths,        \
                                              (__nv_bfloat16 *)key, (__nv_bfloat16 *)value, max_tokens, log2_of(dim), status) \
                             : launch_chained(gather_kernel<float, f>, grid, kThreads, 0, st, 1, c, t, lengths, (float *)key,  \
                                              (float *)value, max_tokens, log2_of(dim), status);
  MXQ_PAGED_FORMATS(CALL)
#undef CALL
  return MXQ_ERR_FORMAT;
}

static int64_t max_moves_of(int64_t width, int64_t keep) {
  const int64_t behind = width > keep ? width - keep : 0;
  return keep < behind ? keep : behind;
}

int64_t mxq_paged_evict_workspace_bytes(const mxq_paged_cache *cache, int64_t batch, int64_t width, int64_t keep) {
  if (!cache || batch < 0 || width < 1 || keep < 1) return MXQ_ERR_SHAPE;
  return batch * cache->heads * (2 * max_moves_of(width, keep) + 1) * 4;
}

int mxq_paged_evict(const mxq_paged_cache *cache, int64_t batch, const int32_t *page_table, int64_t table_width,
                    int64_t table_stride, const int32_t *lengths, const float *weights, const int32_t *positions,
                    const int32_t *next_position, int64_t width, int64_t keep, int64_t recent, int32_t *new_lengths,
                    float *new_weights, int32_t *new_positions, void *workspace, int64_t workspace_bytes, int *status,
                    void *stream) {
  Cache c;
  int rc = read_cache(cache, c);
  if (rc != MXQ_OK) return rc;
  if (batch < 0 || width < 1 || width > INT32_MAX || keep < 1 || keep > INT32_MAX || recent < 0 || recent > keep)
    return MXQ_ERR_SHAPE;
  if (batch == 0) return MXQ_OK;
  if ((rc = read_table(page_table, table_width, table_stride, batch, c.page_log2)) != MXQ_OK) return rc;
  if (!lengths || !weights || !new_lengths || !new_weights || !new_positions || !workspace) return MXQ_ERR_NULL;
  if (!aligned(workspace, 16)) return MXQ_ERR_ALIGN;
  if (workspace_bytes < mxq_paged_evict_workspace_bytes(cache, batch, width, keep)) return MXQ_ERR_SHAPE;
  const int64_t rows = batch * c.heads, most = max_moves_of(width, keep);
  EvictArgs a;
  a.lengths = lengths, a.weights = weights, a.positions = positions, a.next_position = next_position;
  a.width = width, a.keep = (int)keep, a.recent = (int)recent, a.max_moves = (int)most;
  a.new_lengths = new_lengths, a.new_weights = new_weights, a.new_positions = new_positions;
  a.moves = static_cast<int32_t *>(workspace), a.from = a.moves + rows, a.to = a.from + rows * most;
  a.status = status;
  const Table t{page_table, table_stride, table_width};
  cudaStream_t st = (cudaStream_t)stream;
  // Clusters of up to 8 CTAs share a long row's slots as long as there are fewer CTAs than SMs: 64 rows of 16384 slots 77 us
  // with clusters of 4, 81 without (whole eviction), one such row 20.5 and 24.9; 8 rows of 1500 slots 14.4 us when shared by 2,
  // 12.4 when not.
  int cluster = 1;
  while (cluster < 8 && width / cluster > kSlotsPerCta && rows * cluster < gemm::sm_count()) cluster *= 2;
  static std::atomic<bool> set_up[64];  // the kernel's shared memory limit has been raised on this device
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return MXQ_ERR_LAUNCH;
  if (!set_up[device & 63].load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kKeysInShared * 4) !=
        cudaSuccess) {
      cudaGetLastError();
      return MXQ_ERR_LAUNCH;
    }
    set_up[device & 63].store(true, std::memory_order_relaxed);
  }
  const int64_t part = (width + cluster - 1) / cluster;
  const int64_t n_keys = part < kKeysInShared ? (part + 3) / 4 * 4 : kKeysInShared;
  rc = launch_chained(evict_select_kernel, dim3((unsigned)(c.heads * cluster), (unsigned)batch), kSelectThreads,
                      (size_t)n_keys * 4, st, cluster, c, table_width << c.page_log2, a);
  if (rc != MXQ_OK || most == 0) return rc;
  const int row_bytes = row_bytes_of(cache->format, cache->head_dim);
  const int scale_bytes = cache->format == MXQ_CACHE_BF16 ? 0 : cache->head_dim / 32;
  // Moves a warp looks up at once: 8 (8 x 12000 to 16384 slots halved: 69 us; with 32, 75), or 4 so that there is work for four
  // warps on every SM (8 rows of 300 slots halved: 10.3 us; with 8, 11.7).
  int per_warp = 8;
  while (per_warp > 4 && rows * most < (int64_t)gemm::sm_count() * 4 * per_warp) per_warp /= 2;
  const int64_t per_cta = kThreads / 32 * per_warp;
  const dim3 grid(grid_x((most + per_cta - 1) / per_cta, rows, 6), (unsigned)c.heads, (unsigned)batch);
  return launch_chained(evict_move_kernel, grid, kThreads, 0, st, 1, c, t, a, log2_of(row_bytes), scale_bytes, per_warp);
}

}  // extern "C"
