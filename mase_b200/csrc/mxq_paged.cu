// Paged key/value cache in MX formats: writing new rows (mxq_paged_append), reading rows back (mxq_paged_gather) and
// evicting the tokens with the least accumulated attention weight (mxq_paged_evict).

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
// quantizers (the bf16 routines are the ones behind mxq_mxfp_extract / mxq_mxint_extract).
struct AppendArgs {
  const void *src[2];
  int64_t stride_b[2], stride_h[2], stride_t[2];
  const int32_t *lengths, *counts, *next_position;
  int32_t *positions;
  int64_t positions_width;
  int64_t tokens;
  int *status;
};

__device__ __forceinline__ void load16(const __nv_bfloat16 *p, float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint4 r = reinterpret_cast<const uint4 *>(p)[i];
    uint32_t b[8];
    unpack(r, b);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[8 * i + k] = __uint_as_float(b[k]);
  }
}
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

// Codes of this lane's 16 elements (one per byte) and the block's scale byte.  Every lane of the warp calls it.
template <typename T, int kFormat>
__device__ __forceinline__ uint4 encode16(const T *p, bool live, int bits, const Log2Tab &tab, int &scale) {
  using Fmt = Format<kFormat>;
  if constexpr (Elem<T>::kBf16) {
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const uint4 lo = live ? reinterpret_cast<const uint4 *>(p)[0] : zero;
    const uint4 hi = live ? reinterpret_cast<const uint4 *>(p)[1] : zero;
    if constexpr (kFormat == MXQ_CACHE_INT8)
      return mxint_codes_bf16(lo, hi, tab, bits, scale);
    else
      return codes_bf16<Fmt::E, Fmt::F>(lo, hi, tab, scale);
  } else {
    float v[16] = {};
    if (live) load16(p, v);
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
      uint32_t amax = 0;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const uint32_t a = __float_as_uint(v[k]) & 0x7FFFFFFFu;
        amax = max(amax, (a >> 23) == 0 ? 0u : a);
      }
      amax = group_max(amax, 2);
      const MxfpBlock b = mxfp_block(amax, Fmt::E, tab);
      scale = b.scale;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const uint32_t r = __float_as_uint(v[k]);
        code[k] = mxfp_encode(((r & 0x7FFFFFFFu) >> 23) == 0 ? 0u : r, b.sh, Fmt::E, Fmt::F);
      }
    }
    return bytes_of(code);
  }
}

// grid: (chunks of the units of one (sequence, head), heads * 2 sides, batch); a unit is half a block of one token.
template <typename T, int kFormat>
__global__ void __launch_bounds__(kThreads)
append_kernel(const Cache c, const Table table, const AppendArgs a, int dim, const __grid_constant__ Log2Tab tab) {
  using Fmt = Format<kFormat>;
  const int side = blockIdx.y & 1, head = blockIdx.y >> 1;
  const int64_t b = blockIdx.z;
  const int units = dim >> 4;  // 2, 4, 8 or 16: a pair of lanes never straddles two rows
  const int64_t most = table.width << c.page_log2;
  const int length = clamp_length(a.lengths[b], most, a.status);
  int64_t count = a.counts != nullptr ? a.counts[b] : a.tokens;
  if (count < 0 || count > a.tokens || length + count > most) {
    report(a.status);
    count = count < 0 ? 0 : min(min(count, a.tokens), most - length);
  }
  const T *src = static_cast<const T *>(a.src[side]) + b * a.stride_b[side] + head * a.stride_h[side];
  const int64_t total = count * units;
  const int64_t step = (int64_t)gridDim.x * kThreads;
  for (int64_t base = (int64_t)blockIdx.x * kThreads; base < total; base += step) {
    const int64_t i = base + threadIdx.x;
    const bool live = i < total;
    const int64_t t = live ? i / units : 0;
    const int u = (int)(i - t * units);
    int64_t row = -1;
    int slot = 0;
    if (live) {
      slot = length + (int)t;
      row = page_row(c, table, b, head, slot, a.status);
      if (row >= 0) row += slot & ((1 << c.page_log2) - 1);
    }
    const T *p = src + t * a.stride_t[side] + u * 16;
    if constexpr (kFormat == MXQ_CACHE_BF16) {
      if (row >= 0) {
        uint4 *d = reinterpret_cast<uint4 *>(c.codes[side] + row * (dim * 2) + u * 32);
        if constexpr (Elem<T>::kBf16) {
          d[0] = reinterpret_cast<const uint4 *>(p)[0], d[1] = reinterpret_cast<const uint4 *>(p)[1];
        } else {
          float v[16];
          load16(p, v);
#pragma unroll
          for (int k = 0; k < 2; ++k)
            d[k] = make_uint4(pack_bf16x2(v[8 * k], v[8 * k + 1]), pack_bf16x2(v[8 * k + 2], v[8 * k + 3]),
                              pack_bf16x2(v[8 * k + 4], v[8 * k + 5]), pack_bf16x2(v[8 * k + 6], v[8 * k + 7]));
        }
      }
    } else {
      int scale;
      const uint4 code = encode16<T, kFormat>(p, live, c.bits, tab, scale);
      if (row >= 0) {
        if constexpr (Fmt::kBits == 4) {
          uint32_t w[4] = {code.x, code.y, code.z, code.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] |= w[k] >> 4;  // bytes 0 and 2 now hold two codes each
          *reinterpret_cast<uint2 *>(c.codes[side] + row * (dim / 2) + u * 8) =
              make_uint2(__byte_perm(w[0], w[1], 0x6420), __byte_perm(w[2], w[3], 0x6420));
        } else {
          *reinterpret_cast<uint4 *>(c.codes[side] + row * dim + u * 16) = code;
        }
        if ((u & 1) == 0) c.scales[side][row * (dim >> 5) + (u >> 1)] = (uint8_t)scale;
      }
    }
    if (side == 0 && u == 0 && live && a.positions != nullptr) {
      if (slot < a.positions_width)
        a.positions[(b * c.heads + head) * a.positions_width + slot] =
            (a.next_position != nullptr ? a.next_position[b] : length) + (int)t;
      else
        report(a.status);
    }
  }
}

// ---- gather ----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void store16(__nv_bfloat16 *p, const float (&v)[16]) {
#pragma unroll
  for (int k = 0; k < 2; ++k)
    st_stream(reinterpret_cast<uint4 *>(p) + k,
              make_uint4(pack_bf16x2(v[8 * k], v[8 * k + 1]), pack_bf16x2(v[8 * k + 2], v[8 * k + 3]),
                         pack_bf16x2(v[8 * k + 4], v[8 * k + 5]), pack_bf16x2(v[8 * k + 6], v[8 * k + 7])));
}
__device__ __forceinline__ void store16(float *p, const float (&v)[16]) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    st_stream(reinterpret_cast<uint4 *>(p) + k,
              make_uint4(__float_as_uint(v[4 * k]), __float_as_uint(v[4 * k + 1]), __float_as_uint(v[4 * k + 2]),
                         __float_as_uint(v[4 * k + 3])));
}

// 16 elements from `p` (codes) with the block's scale byte.
template <int kFormat>
__device__ __forceinline__ void decode16(const uint8_t *p, int scale, int bits, float (&v)[16]) {
  using Fmt = Format<kFormat>;
  if constexpr (kFormat == MXQ_CACHE_BF16) {
    load16(reinterpret_cast<const __nv_bfloat16 *>(p), v);
  } else if constexpr (Fmt::kBits == 4) {
    const uint2 r = *reinterpret_cast<const uint2 *>(p);
    const float sf = pow2f(scale - 127);
#pragma unroll
    for (int k = 0; k < 16; ++k)
      v[k] = mxfp_decode(((k < 8 ? r.x : r.y) >> (4 * (k & 7))) & 15u, Fmt::E, Fmt::F) * sf;
  } else {
    const uint4 r = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    const float sf = kFormat == MXQ_CACHE_INT8 ? (scale == 255 ? INFINITY : pow2f(scale - 127 - (bits - 1)))
                                               : pow2f(scale - 127);
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const uint32_t code = (w[k >> 2] >> (8 * (k & 3))) & 0xFFu;
      v[k] = (kFormat == MXQ_CACHE_INT8 ? (float)(int8_t)code : mxfp_decode(code, Fmt::E, Fmt::F)) * sf;
    }
  }
}

// grid: (chunks of the units of one (sequence, head), heads * 2 sides, batch); a unit is 16 elements of one token.
template <typename T, int kFormat>
__global__ void __launch_bounds__(kThreads)
gather_kernel(const Cache c, const Table table, const int32_t *lengths, T *key, T *value, int64_t tokens, int dim,
              int *status) {
  using Fmt = Format<kFormat>;
  const int side = blockIdx.y & 1, head = blockIdx.y >> 1;
  const int64_t b = blockIdx.z;
  const int units = dim >> 4;
  const int length = clamp_length(lengths[b], table.width << c.page_log2, status);
  T *dst = (side ? value : key) + (b * c.heads + head) * tokens * dim;
  const int64_t total = tokens * units;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
    const int64_t t = i / units;
    const int u = (int)(i - t * units);
    float v[16] = {};
    if (t < length) {
      int64_t row = page_row(c, table, b, head, (int)t, status);
      if (row >= 0) {
        row += t & ((1 << c.page_log2) - 1);
        int scale = 0;
        if constexpr (kFormat != MXQ_CACHE_BF16) scale = c.scales[side][row * (dim >> 5) + (u >> 1)];
        decode16<kFormat>(c.codes[side] + row * (dim * Fmt::kBits / 8) + u * (2 * Fmt::kBits), scale, c.bits, v);
      }
    }
    store16(dst + t * dim + u * 16, v);
  }
}

// ---- evict -----------------------------------------------------------------------------------------------------------
// Selection: one CTA per (sequence, head).  The weights become 32-bit keys whose unsigned order is the order of
// preference; three passes over 11 + 11 + 10 bits of the keys (a histogram in shared memory each) find the key of the
// last token kept, and every warp then walks a contiguous part of the slots with ballots, so that ranks follow the slot
// order.  Keys live in shared memory when they fit and are read again from L2 otherwise.
constexpr int kSelectThreads = 1024;
constexpr int kBins = 2048;
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

// exclusive prefix sum over the CTA's 32 warps of a per-warp value held by every lane; `total` = the sum
__device__ __forceinline__ int scan_warps(int v, int *scratch, int &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  int s = scratch[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xFFFFFFFFu, s, o);
    if (lane >= o) s += n;
  }
  total = __shfl_sync(0xFFFFFFFFu, s, 31);
  const int before = __shfl_sync(0xFFFFFFFFu, s, warp == 0 ? 0 : warp - 1);
  return warp == 0 ? 0 : before;
}

__global__ void __launch_bounds__(kSelectThreads)
evict_select_kernel(const Cache c, int64_t table_tokens, const EvictArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ int hist[kBins];
  __shared__ int scratch[32];
  __shared__ int found[2];  // bin of the last kept key, keys in bins above it
  const int head = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t b = blockIdx.y;
  const int64_t row = b * c.heads + head;
  const int n = clamp_length(a.lengths[b], min(table_tokens, a.width), a.status);
  const int m = min(n, a.keep);
  const float *w = a.weights + row * a.width;
  const int32_t *p = a.positions != nullptr ? a.positions + row * a.width : nullptr;
  float *nw = a.new_weights + row * a.width;
  int32_t *np = a.new_positions + row * a.width;
  if (head == 0 && tid == 0) a.new_lengths[b] = m;
  for (int64_t j = m + tid; j < a.width; j += kSelectThreads) nw[j] = 0.f, np[j] = -1;
  if (n <= a.keep) {
    for (int j = tid; j < n; j += kSelectThreads) nw[j] = w[j], np[j] = p != nullptr ? p[j] : j;
    if (tid == 0) a.moves[row] = 0;
    return;
  }
  const int64_t first_safe = (int64_t)(p != nullptr && a.next_position != nullptr ? a.next_position[b] : n) - a.recent;
  const bool shared_keys = n <= kKeysInShared;
  auto make_key = [&](int j) {
    const int64_t pos = p != nullptr ? p[j] : j;
    return pos >= first_safe ? 0xFFFFFFFFu : key_of(w[j]);
  };
  auto key_at = [&](int j) { return shared_keys ? keys[j] : make_key(j); };
  if (shared_keys)
    for (int j = tid; j < n; j += kSelectThreads) keys[j] = make_key(j);

  uint32_t prefix = 0;  // the digits found so far, in place
  int need = m;         // how many of the keys that share the prefix are kept
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
    const int bins = pass == 2 ? 1024 : 2048;
    const uint32_t above = pass == 0 ? 0u : (pass == 1 ? 0xFFE00000u : 0xFFFFFC00u);
    __syncthreads();
    for (int k = tid; k < kBins; k += kSelectThreads) hist[k] = 0;
    __syncthreads();
    for (int j = tid; j < n; j += kSelectThreads) {
      const uint32_t k = key_at(j);
      if ((k & above) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1);
    }
    __syncthreads();
    // thread t owns bins bins - 1 - 2t and bins - 2 - 2t: the running sum goes from the largest key down
    const int hi = bins - 1 - 2 * tid, lo = hi - 1;
    const int ch = hi >= 0 ? hist[hi] : 0, cl = lo >= 0 ? hist[lo] : 0;
    int s = ch + cl;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xFFFFFFFFu, s, o);
      if (lane >= o) s += x;
    }
    int total;
    const int base = scan_warps(__shfl_sync(0xFFFFFFFFu, s, 31), scratch, total) + s - ch - cl;
    if (base < need && base + ch >= need) found[0] = hi, found[1] = base;
    if (base + ch < need && base + ch + cl >= need) found[0] = lo, found[1] = base + ch;
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    need -= found[1];
  }
  const uint32_t last = prefix;  // tokens above it are kept, and the first `need` equal to it

  const int part = ((n + 1023) / 1024) * 32;  // slots of one warp
  const int begin = min(warp * part, n), end = min(begin + part, n);
  int ties = 0, total;
  for (int j0 = begin; j0 < end; j0 += 32)
    ties += __popc(__ballot_sync(0xFFFFFFFFu, j0 + lane < end && key_at(min(j0 + lane, n - 1)) == last));
  const int ties_before = scan_warps(ties, scratch, total);
  const uint32_t below = (1u << lane) - 1u;
  int holes = 0, movers = 0, seen = ties_before;
  auto classify = [&](int j, bool in, bool &kept) {
    const uint32_t k = in ? key_at(j) : 0u;
    const uint32_t tie = __ballot_sync(0xFFFFFFFFu, in && k == last);
    kept = in && (k > last || (k == last && seen + __popc(tie & below) < need));
    seen += __popc(tie);
  };
  for (int j0 = begin; j0 < end; j0 += 32) {
    const int j = j0 + lane;
    bool kept;
    classify(j, j < end, kept);
    holes += __popc(__ballot_sync(0xFFFFFFFFu, j < end && j < m && !kept));
    movers += __popc(__ballot_sync(0xFFFFFFFFu, kept && j >= m));
  }
  int n_moves;
  int hole_at = scan_warps(holes, scratch, n_moves);
  int mover_at = scan_warps(movers, scratch, n_moves);
  int32_t *from = a.from + row * a.max_moves, *to = a.to + row * a.max_moves;
  seen = ties_before;
  for (int j0 = begin; j0 < end; j0 += 32) {
    const int j = j0 + lane;
    bool kept;
    classify(j, j < end, kept);
    const bool hole = j < end && j < m && !kept, mover = kept && j >= m;
    const uint32_t hb = __ballot_sync(0xFFFFFFFFu, hole), mb = __ballot_sync(0xFFFFFFFFu, mover);
    if (hole) to[hole_at + __popc(hb & below)] = j;
    if (mover) from[mover_at + __popc(mb & below)] = j;
    if (kept && j < m) nw[j] = w[j], np[j] = p != nullptr ? p[j] : j;
    hole_at += __popc(hb), mover_at += __popc(mb);
  }
  __syncthreads();  // the lists are complete for the whole CTA
  for (int i = tid; i < n_moves; i += kSelectThreads) {
    const int s = from[i], d = to[i];
    nw[d] = w[s], np[d] = p != nullptr ? p[s] : s;
  }
  if (tid == 0) a.moves[row] = n_moves;
}

// One warp per moved token: its key and value rows in 16-byte pieces, then the scale bytes.  Sources lie at or above
// `keep`, destinations below it, so moves never overlap.
__global__ void __launch_bounds__(kThreads)
evict_move_kernel(const Cache c, const Table table, const int32_t *from, const int32_t *to, const int32_t *moves,
                  int max_moves, int row_bytes, int scale_bytes, int *status) {
  const int head = blockIdx.y, lane = threadIdx.x & 31;
  const int64_t b = blockIdx.z;
  const int64_t row = b * c.heads + head;
  const int n = moves[row];
  const int in_page = (1 << c.page_log2) - 1;
  const int pieces = row_bytes >> 4;
  for (int i = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); i < n; i += gridDim.x * (kThreads / 32)) {
    const int s = from[row * max_moves + i], d = to[row * max_moves + i];
    int64_t sr = page_row(c, table, b, head, s, status), dr = page_row(c, table, b, head, d, status);
    if (sr < 0 || dr < 0) continue;
    sr += s & in_page, dr += d & in_page;
    for (int k = lane; k < 2 * pieces; k += 32) {
      const int side = k >= pieces, at = side ? k - pieces : k;
      reinterpret_cast<uint4 *>(c.codes[side] + dr * row_bytes)[at] =
          reinterpret_cast<const uint4 *>(c.codes[side] + sr * row_bytes)[at];
    }
    if (lane < 2 * scale_bytes) {
      const int side = lane >= scale_bytes, at = side ? lane - scale_bytes : lane;
      c.scales[side][dr * scale_bytes + at] = c.scales[side][sr * scale_bytes + at];
    }
  }
}

static int launched() { return cudaGetLastError() == cudaSuccess ? MXQ_OK : MXQ_ERR_LAUNCH; }

// CTAs along x so that the whole grid holds about `per_sm` CTAs per SM, and no more than the work needs.
static unsigned grid_x(int64_t need, int64_t yz, int per_sm) {
  int64_t most = ((int64_t)gemm::sm_count() * per_sm + yz - 1) / yz;
  if (most < 1) most = 1;
  if (need < 1) need = 1;
  return (unsigned)(need < most ? need : most);
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
  if (batch < 0 || tokens < 0 || tokens > INT32_MAX) return MXQ_ERR_SHAPE;
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
  const dim3 grid(grid_x((tokens * (dim / 16) + kThreads - 1) / kThreads, yz, 16), c.heads * 2, (unsigned)batch);
  cudaStream_t st = (cudaStream_t)stream;
#define CALL(f)                                                                               \
  if (cache->format == f) {                                                                   \
    if (dtype == MXQ_BF16)                                                                    \
      append_kernel<__nv_bfloat16, f><<<grid, kThreads, 0, st>>>(c, t, a, dim, tab);          \
    else                                                                                      \
      append_kernel<float, f><<<grid, kThreads, 0, st>>>(c, t, a, dim, tab);                  \
  }
  MXQ_PAGED_FORMATS(CALL)
#undef CALL
  return launched();
}

int mxq_paged_gather(const mxq_paged_cache *cache, void *key, void *value, int dtype, int64_t batch, int64_t max_tokens,
                     const int32_t *page_table, int64_t table_width, int64_t table_stride, const int32_t *lengths,
                     int *status, void *stream) {
  Cache c;
  int rc = read_cache(cache, c);
  if (rc != MXQ_OK) return rc;
  if (dtype != MXQ_F32 && dtype != MXQ_BF16) return MXQ_ERR_DTYPE;
  if (batch < 0 || max_tokens < 0 || max_tokens > INT32_MAX) return MXQ_ERR_SHAPE;
  if (batch == 0 || max_tokens == 0) return MXQ_OK;
  if ((rc = read_table(page_table, table_width, table_stride, batch, c.page_log2)) != MXQ_OK) return rc;
  if (!key || !value || !lengths) return MXQ_ERR_NULL;
  if (!aligned(key, 16) || !aligned(value, 16)) return MXQ_ERR_ALIGN;
  const Table t{page_table, table_stride, table_width};
  const int dim = cache->head_dim;
  const int64_t yz = (int64_t)c.heads * 2 * batch;
  const dim3 grid(grid_x((max_tokens * (dim / 16) + kThreads - 1) / kThreads, yz, 16), c.heads * 2, (unsigned)batch);
  cudaStream_t st = (cudaStream_t)stream;
#define CALL(f)                                                                                                    \
  if (cache->format == f) {                                                                                        \
    if (dtype == MXQ_BF16)                                                                                         \
      gather_kernel<__nv_bfloat16, f><<<grid, kThreads, 0, st>>>(c, t, lengths, (__nv_bfloat16 *)key,               \
                                                                 (__nv_bfloat16 *)value, max_tokens, dim, status); \
    else                                                                                                           \
      gather_kernel<float, f><<<grid, kThreads, 0, st>>>(c, t, lengths, (float *)key, (float *)value, max_tokens,   \
                                                         dim, status);                                             \
  }
  MXQ_PAGED_FORMATS(CALL)
#undef CALL
  return launched();
}

static int64_t max_moves_of(int64_t width, int64_t keep) {
  const int64_t behind = width > keep ? width - keep : 0;
  return keep < behind ? keep : behind;
}

int64_t mxq_paged_evict_workspace_bytes(const mxq_paged_cache *cache, int64_t batch, int64_t width, int64_t keep) {
  if (!cache || batch < 0 || width < 0 || keep < 1) return MXQ_ERR_SHAPE;
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
  if (batch < 0 || width < 0 || width > INT32_MAX || keep < 1 || keep > INT32_MAX || recent < 0 || recent > keep)
    return MXQ_ERR_SHAPE;
  if (batch == 0 || width == 0) return MXQ_OK;
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
  const int64_t n_keys = width < kKeysInShared ? width : kKeysInShared;
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
  evict_select_kernel<<<dim3((unsigned)c.heads, (unsigned)batch), kSelectThreads, (size_t)n_keys * 4, st>>>(
      c, table_width << c.page_log2, a);
  if ((rc = launched()) != MXQ_OK || most == 0) return rc;
  const int row_bytes = row_bytes_of(cache->format, cache->head_dim);
  const int scale_bytes = cache->format == MXQ_CACHE_BF16 ? 0 : cache->head_dim / 32;
  const dim3 grid(grid_x((most + kThreads / 32 - 1) / (kThreads / 32), rows, 16), (unsigned)c.heads, (unsigned)batch);
  evict_move_kernel<<<grid, kThreads, 0, st>>>(c, t, a.from, a.to, a.moves, a.max_moves, row_bytes, scale_bytes, status);
  return launched();
}

}  // extern "C"
