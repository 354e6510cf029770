"""Paged key/value cache in MX formats and the attention of one new token over it.

The reference quantizes what it caches as dense tensors (`kv_cache_mxfp` / `kv_cache_mxint`,
chop/nn/quantized/functional/kvcache.py:8-43) and keeps the fake-quantized values at full width.  Here the cache holds the
codes and shared exponents (1.03 bytes per element for 8-bit formats, 0.53 for MXFP4, bf16 without quantization) in pages
that sequences share out between them, and a decoding step reads those:

    cache = PagedKVCache(num_pages, num_kv_heads, head_dim, page_size=64, fmt="mxfp", config=kv_cache_config, device="cuda")
    paged_kv_append(cache, key, value, page_table, lengths)          # quantize new rows into the pages
    out = paged_attention(cache, query, page_table, lengths, scaling)  # one new token per sequence
    key, value = paged_kv_gather(cache, page_table, lengths, max_length)  # dense tensors, for the attention of a prompt
    lengths, weights, positions = paged_kv_evict(cache, page_table, lengths, weights, keep, recent)

Sequence b's token i lives in slot i % page_size of page page_table[b, i // page_size].  Page tables (int32 [batch, width];
entries that no token needs may hold anything) and lengths (int32 [batch]) are device tensors which only the kernels look
at, so calls can be captured into a CUDA graph and follow later changes of their contents.  A needed entry that names no
page of the cache, or a length that does not fit its table, is reported by `mase_b200.gemm.check_status()`; nothing
outside of the cache is read or written.

`PagedKVState` bundles the caches of a model's layers with their page table and lengths; the attention blocks of
`mase_b200.attention` take it as `past_key_value`.
"""

from __future__ import annotations

import ctypes

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib
from . import gemm
from .gemm import _status, check_status
from .quantizers import _DT, _ceil_tab_ptr, _floor_tab_ptr, _on_device, _require_cuda, _stream

_BINDING = None


def _binding():
    """The compiled torch binding when it is built and has the cache's entries, else False (see mase_b200.gemm._ext)."""
    global _BINDING
    if _BINDING is None:
        ext = gemm._ext()
        _BINDING = ext if ext and hasattr(ext, "paged_attention") else False
    return _BINDING


def _check_every_call(cache) -> None:
    if gemm._CHECK_EVERY_CALL:
        check_status(cache.device)


_MXFP_FORMATS = {(4, 3): _lib.CACHE_E4M3, (5, 2): _lib.CACHE_E5M2, (2, 1): _lib.CACHE_E2M1X2}
_HEAD_DIMS, _PAGE_SIZES = (32, 64, 128, 256), (16, 32, 64, 128, 256)


def _format_of(fmt: str | None, config: dict | None) -> tuple[int, int]:
    """(MXQ_CACHE_* code, mantissa bits) of a `kv_cache` configuration of the quantized attention blocks."""
    if fmt is None or (config or {}).get("bypass", False):
        return _lib.CACHE_BF16, 0
    if fmt not in ("mxfp", "mxint"):
        raise ValueError(f"fmt is None, 'mxfp' or 'mxint', not {fmt!r}")
    if config is None:
        raise ValueError(f"a cache with fmt={fmt!r} needs the quantizer's config")
    if config["data_in_block_size"] != 32:
        raise NotImplementedError("paged caches are provided for blocks of 32 elements")
    if fmt == "mxint":
        bits = config["data_in_width"]
        if not 2 <= bits <= 8:
            raise NotImplementedError("mxint: element_bits must be between 2 and 8")
        return _lib.CACHE_INT8, bits
    ef = (config["data_in_exponent_width"], config["data_in_frac_width"])
    if ef not in _MXFP_FORMATS:
        raise NotImplementedError(f"paged caches are provided for MXFP elements {sorted(_MXFP_FORMATS)}, not {ef}")
    return _MXFP_FORMATS[ef], 0


def _row_bytes(code: int, head_dim: int) -> int:
    return {_lib.CACHE_BF16: 2 * head_dim, _lib.CACHE_E2M1X2: head_dim // 2}.get(code, head_dim)


class PagedKVCache:
    """The pages of one attention layer.

    key, value                [num_pages, num_kv_heads, page_size, row]: uint8 codes -- one MXFP code or int8 mantissa per
                              byte, two E2M1 codes per byte (element 2i in the low nibble) -- or bf16 values (fmt None)
    key_scales, value_scales  uint8 [num_pages, num_kv_heads, page_size, head_dim // 32], None for fmt None

    `fmt` / `config` are those of the attention blocks' `kv_cache` entry: "mxfp" with data_in_exponent_width /
    data_in_frac_width (4, 3), (5, 2) or (2, 1); "mxint" with data_in_width 2..8; blocks of 32.  head_dim 32, 64, 128 or
    256, page_size 16, 32, 64, 128 or 256.  The four tensors may be written in place but not exchanged."""

    def __init__(self, num_pages: int, num_kv_heads: int, head_dim: int, page_size: int = 64, fmt: str | None = None,
                 config: dict | None = None, device=None):
        code, _ = _format_of(fmt, config)
        self._check_sizes(num_pages, num_kv_heads, head_dim, page_size)
        shape = (num_pages, num_kv_heads, page_size)
        dt, row = (torch.bfloat16, head_dim) if code == _lib.CACHE_BF16 else (torch.uint8, _row_bytes(code, head_dim))
        pages = [torch.zeros((*shape, row), dtype=dt, device=device) for _ in range(2)]
        scales = [None, None] if code == _lib.CACHE_BF16 else \
            [torch.zeros((*shape, head_dim // 32), dtype=torch.uint8, device=device) for _ in range(2)]
        self._take(*pages, *scales, fmt, config)

    @classmethod
    def from_pages(cls, key: Tensor, value: Tensor, key_scales: Tensor | None, value_scales: Tensor | None,
                   fmt: str | None = None, config: dict | None = None) -> "PagedKVCache":
        """A cache on pages that exist already (the tensors are kept, not copied)."""
        self = cls.__new__(cls)
        self._take(key, value, key_scales, value_scales, fmt, config)
        return self

    @staticmethod
    def _check_sizes(num_pages, heads, head_dim, page_size):
        if head_dim not in _HEAD_DIMS:
            raise NotImplementedError(f"paged caches are provided for head_dim in {_HEAD_DIMS}, not {head_dim}")
        if page_size not in _PAGE_SIZES:
            raise NotImplementedError(f"paged caches are provided for page_size in {_PAGE_SIZES}, not {page_size}")
        if num_pages < 1 or heads < 1:
            raise ValueError("a paged cache has at least one page and one key/value head")

    def _take(self, key, value, key_scales, value_scales, fmt, config):
        code, bits = _format_of(fmt, config)
        if key.dim() != 4 or key.shape != value.shape:
            raise ValueError("key and value pages are [num_pages, num_kv_heads, page_size, row] of the same shape")
        want = torch.bfloat16 if code == _lib.CACHE_BF16 else torch.uint8
        tensors = [key, value]
        row = key.shape[3]
        dim = row * 2 if code == _lib.CACHE_E2M1X2 else row
        self._check_sizes(key.shape[0], key.shape[1], dim, key.shape[2])
        if code == _lib.CACHE_BF16:
            if key_scales is not None or value_scales is not None:
                raise ValueError("a cache without quantization has no scales")
        else:
            for s in (key_scales, value_scales):
                if s is None or s.dtype != torch.uint8 or tuple(s.shape) != (*key.shape[:3], dim // 32):
                    raise ValueError("scales are uint8 [num_pages, num_kv_heads, page_size, head_dim // 32]")
            tensors += [key_scales, value_scales]
        for t in tensors[:2]:
            if t.dtype != want:
                raise NotImplementedError(f"pages of this format are {want}, not {t.dtype}")
        for t in tensors:
            _require_cuda(t, "PagedKVCache")
            if not t.is_contiguous() or t.data_ptr() % 16 or t.device != key.device:
                raise ValueError("pages and scales are contiguous, 16-byte aligned and on one device")
        self.fmt, self.config = (None, None) if code == _lib.CACHE_BF16 else (fmt, dict(config))
        self._tensors = key, value, key_scales, value_scales  # kept for as long as _desc points at them
        self.num_pages, self.num_kv_heads, self.page_size = key.shape[:3]
        self.head_dim, self.device, self._index = dim, key.device, key.device.index
        self._code, self._bits = code, bits
        ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        self._desc = _lib.PagedCache(ptr(key), ptr(value), ptr(key_scales), ptr(value_scales), self.num_pages, code, bits,
                                     self.num_kv_heads, dim, self.page_size, 0)
        self._addr = ctypes.addressof(self._desc)
        _status(self.device)  # made here, not during a capture

    # The pages cannot be exchanged: the calls go by the addresses taken above.  `from_pages` makes a cache of other tensors.
    key = property(lambda self: self._tensors[0])
    value = property(lambda self: self._tensors[1])
    key_scales = property(lambda self: self._tensors[2])
    value_scales = property(lambda self: self._tensors[3])

    def _log2_tab(self, dtype: torch.dtype):
        if self._code == _lib.CACHE_BF16:
            return 0
        if dtype not in _DT:
            return 0
        return _ceil_tab_ptr(dtype) if self._code == _lib.CACHE_INT8 else _floor_tab_ptr()


def _no_autograd(what: str, *tensors: Tensor | None) -> None:
    """Raises when one of the tensors carries a gradient or, in forward mode, a tangent: the calls would drop it."""
    for t in tensors:
        if t is not None and ((t.requires_grad and torch.is_grad_enabled()) or forward_ad.unpack_dual(t).tangent is not None):
            raise NotImplementedError(f"{what} has no derivative: call it under torch.no_grad() on tensors without a tangent")


def _check_table(cache: PagedKVCache, page_table: Tensor, lengths: Tensor) -> int:
    """Checks a page table [batch, width] and the lengths [batch]; returns the batch size."""
    if page_table.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise NotImplementedError("page_table and lengths are int32")
    if page_table.dim() != 2 or lengths.dim() != 1 or page_table.shape[0] != lengths.shape[0]:
        raise ValueError("page_table is [batch, width] and lengths [batch]")
    if page_table.shape[1] < 1 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError("page_table has at least one column and contiguous rows")
    if page_table.shape[0] > 1 and page_table.stride(0) < page_table.shape[1]:
        raise ValueError("the rows of page_table may not overlap")
    if lengths.stride(0) != 1 and lengths.shape[0] > 1:
        raise ValueError("lengths is contiguous")
    if page_table.device != cache.device or lengths.device != cache.device:
        raise RuntimeError("page_table and lengths are on the cache's device")
    return page_table.shape[0]


def _check_int32(t: Tensor, name: str, shape: tuple, cache: PagedKVCache) -> None:
    if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != cache.device:
        raise ValueError(f"{name} is a contiguous int32 tensor of shape {shape} on the cache's device")


def _check_stats(t: Tensor, name: str, dtype: torch.dtype, batch: int, cache: PagedKVCache, width: int | None = None):
    if t.dtype != dtype:
        raise NotImplementedError(f"{name} is {dtype}, not {t.dtype}")
    if t.dim() != 3 or t.shape[:2] != (batch, cache.num_kv_heads) or t.shape[2] < 1 or not t.is_contiguous() \
            or t.device != cache.device or (width is not None and t.shape[2] != width):
        raise ValueError(f"{name} is a contiguous tensor [batch, num_kv_heads, width] on the cache's device")


def _rows_of(x: Tensor, dtype: torch.dtype) -> Tensor:
    """x with a contiguous last dimension and every row on a 16-byte boundary (a copy where it is not so)."""
    need = 16 // x.element_size()
    if x.stride(-1) == 1 and x.data_ptr() % 16 == 0 and \
            all(s % need == 0 for s, n in zip(x.stride()[:-1], x.shape[:-1]) if n > 1):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _step(x: Tensor, d: int) -> int:
    """Stride of dimension d; 0 where it has one entry (its stride may be anything there)."""
    return x.stride(d) if x.shape[d] > 1 else 0


def paged_kv_append(cache: PagedKVCache, key: Tensor, value: Tensor, page_table: Tensor, lengths: Tensor,
                    counts: Tensor | None = None, positions: Tensor | None = None,
                    next_position: Tensor | None = None) -> None:
    """Quantize key / value [batch, num_kv_heads, tokens, head_dim] (fp32 or bf16, any strides) into the pages: token t of
    sequence b goes to slot lengths[b] + t.  `counts` (int32 [batch]): only the first counts[b] tokens of sequence b exist
    (a padded batch).  Codes and shared exponents are those of `mxfp_quantizer` / `mxint_quantizer` along head_dim.
    `lengths` is not changed: add the new tokens to it once every layer has them.  The pages that are written belong to one
    sequence of the batch each.  Rows are finite: no code stands for an infinity or NaN, and what a block of 32 with one in
    it holds means nothing (other blocks are not touched by it).

    `positions` (int32 [batch, num_kv_heads, width]) is the record of token positions that `paged_kv_evict` keeps: the
    entries of the new slots become next_position[b] + t (int32 [batch]; default: lengths[b] + t)."""
    ext = _binding()
    if ext and ext.paged_append(cache._addr, cache._index, key, value, page_table, lengths, counts, positions, next_position,
                                cache._log2_tab(key.dtype), _status(cache.device)):
        return _check_every_call(cache)
    _require_cuda(key, "paged_kv_append")
    _require_cuda(value, "paged_kv_append")
    if key.dtype not in _DT or value.dtype != key.dtype:
        raise NotImplementedError(f"paged_kv_append: dtypes {key.dtype} / {value.dtype} are not supported "
                                  "(float32 and bfloat16 are, the same for both)")
    _no_autograd("paged_kv_append", key, value)
    batch = _check_table(cache, page_table, lengths)
    if key.dim() != 4 or key.shape != value.shape or key.shape[0] != batch or key.shape[1] != cache.num_kv_heads \
            or key.shape[3] != cache.head_dim:
        raise ValueError(f"key and value are [{batch}, {cache.num_kv_heads}, tokens, {cache.head_dim}]")
    if key.device != cache.device or value.device != cache.device:
        raise RuntimeError("key and value are on the cache's device")
    if counts is not None:
        _check_int32(counts, "counts", (batch,), cache)
    if positions is not None:
        _check_stats(positions, "positions", torch.int32, batch, cache)
    if next_position is not None:
        if positions is None:
            raise ValueError("next_position goes with positions")
        _check_int32(next_position, "next_position", (batch,), cache)
    if key.numel() == 0:
        return
    k, v = _rows_of(key, key.dtype), _rows_of(value, value.dtype)
    with _on_device(key):
        rc = _lib.lib().mxq_paged_append(
            cache._addr, k.data_ptr(), v.data_ptr(), _DT[key.dtype], batch, key.shape[2], _step(k, 0), _step(k, 1),
            _step(k, 2), _step(v, 0), _step(v, 1), _step(v, 2), page_table.data_ptr(), page_table.shape[1],
            page_table.stride(0), lengths.data_ptr(), 0 if counts is None else counts.data_ptr(),
            0 if positions is None else positions.data_ptr(), 0 if positions is None else positions.shape[2],
            0 if next_position is None else next_position.data_ptr(), cache._log2_tab(key.dtype),
            _status(cache.device).data_ptr(), _stream(key))
    _lib.check(rc, "mxq_paged_append")
    _check_every_call(cache)


def paged_kv_gather(cache: PagedKVCache, page_table: Tensor, lengths: Tensor, max_length: int,
                    dtype: torch.dtype = torch.bfloat16) -> tuple[Tensor, Tensor]:
    """The cached rows as dense tensors (key, value), each [batch, num_kv_heads, max_length, head_dim] of `dtype`: what
    `kv_cache_mxfp` / `kv_cache_mxint` made of the rows that went in, except that MXINT mantissas hold no negative zero.
    Rows from lengths[b] on are zeros; tokens from max_length on are left out."""
    ext = _binding()
    if ext and (got := ext.paged_gather(cache._addr, cache._index, page_table, lengths, max_length, dtype,
                                        _status(cache.device))) is not None:
        _check_every_call(cache)
        return got
    if dtype not in _DT:
        raise NotImplementedError(f"paged_kv_gather: dtype {dtype} is not supported (float32 and bfloat16 are)")
    batch = _check_table(cache, page_table, lengths)
    if max_length < 0:
        raise ValueError("max_length is not negative")
    shape = (batch, cache.num_kv_heads, max_length, cache.head_dim)
    key, value = (torch.empty(shape, dtype=dtype, device=cache.device) for _ in range(2))
    if key.numel() == 0:
        return key, value
    with _on_device(key):
        rc = _lib.lib().mxq_paged_gather(cache._addr, key.data_ptr(), value.data_ptr(), _DT[dtype], batch, max_length,
                                         page_table.data_ptr(), page_table.shape[1], page_table.stride(0),
                                         lengths.data_ptr(), _status(cache.device).data_ptr(), _stream(key))
    _lib.check(rc, "mxq_paged_gather")
    _check_every_call(cache)
    return key, value


def paged_attention(cache: PagedKVCache, query: Tensor, page_table: Tensor, lengths: Tensor, scaling: float | None = None,
                    weights: Tensor | None = None) -> Tensor:
    """softmax(scaling * query key^T) value over each sequence's cached tokens, for one new token per sequence.

    query [batch, heads, 1, head_dim] (or [batch, heads, head_dim]), fp32 or bf16; heads is a multiple of the cache's
    num_kv_heads, query heads h * group .. h * group + group - 1 read key/value head h (what `repeat_kv` lays out).
    `lengths` counts the new token when it has been appended.  scaling: default head_dim ** -0.5.  The result has the
    query's shape and dtype; a sequence of length 0 gives zeros.  Softmax and sums in fp32.  Queries and values are finite
    (an infinite value makes its element of the result NaN); a key whose score is -inf has weight 0.

    `weights` (fp32 [batch, num_kv_heads, width], width at least the largest length) accumulates in place: the softmax
    weight of every cached token, summed over the query heads of its key/value head, is added to its entry.  The call then
    takes a workspace of 4 bytes a query head (a group's rounded up to a power of two) and slot of the narrower of page
    table and `weights`, whatever the lengths are: give neither more columns than the sequences may need."""
    if scaling is None:
        scaling = cache.head_dim ** -0.5
    ext = _binding()
    if ext and (out := ext.paged_attention(cache._addr, cache._index, query, page_table, lengths, scaling, weights,
                                           _status(cache.device))) is not None:
        _check_every_call(cache)
        return out
    _require_cuda(query, "paged_attention")
    if query.dtype not in _DT:
        raise NotImplementedError(f"paged_attention: dtype {query.dtype} is not supported (float32 and bfloat16 are)")
    _no_autograd("paged_attention", query, weights)
    batch = _check_table(cache, page_table, lengths)
    if query.dim() == 4:
        if query.shape[2] != 1:
            raise ValueError("paged_attention takes one new token per sequence: query is [batch, heads, 1, head_dim]")
        q = query[:, :, 0]
    else:
        q = query
    if q.dim() != 3 or q.shape[0] != batch or q.shape[2] != cache.head_dim or q.shape[1] < 1 \
            or q.shape[1] % cache.num_kv_heads:
        raise ValueError(f"query is [{batch}, heads, 1, {cache.head_dim}] with heads a multiple of {cache.num_kv_heads}")
    if query.device != cache.device:
        raise RuntimeError("query is on the cache's device")
    if weights is not None:
        _check_stats(weights, "weights", torch.float32, batch, cache)
    out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    if batch == 0:
        return out
    if q.stride(2) != 1:
        q = q.contiguous()
    lib = _lib.lib()
    heads, width = q.shape[1], page_table.shape[1]
    if weights is not None:  # the workspace holds scores for every slot of the table: none behind the statistics
        width = min(width, -(-weights.shape[2] // cache.page_size))
    n_ws = int(lib.mxq_paged_attention_workspace_bytes(cache._addr, batch, heads, width, 0 if weights is None else 1))
    if n_ws < 0:
        _lib.check(n_ws, "mxq_paged_attention_workspace_bytes")
    with _on_device(query):
        ws = torch.empty((n_ws,), dtype=torch.uint8, device=query.device)
        rc = lib.mxq_paged_attention(
            cache._addr, q.data_ptr(), out.data_ptr(), _DT[q.dtype], batch, heads, q.stride(0), q.stride(1),
            float(scaling), page_table.data_ptr(), width,
            page_table.stride(0), lengths.data_ptr(), 0 if weights is None else weights.data_ptr(),
            0 if weights is None else weights.shape[2], ws.data_ptr(), n_ws, _status(cache.device).data_ptr(),
            _stream(query))
    _lib.check(rc, "mxq_paged_attention")
    _check_every_call(cache)
    return out


def paged_kv_evict(cache: PagedKVCache, page_table: Tensor, lengths: Tensor, weights: Tensor, keep: int, recent: int = 0,
                   positions: Tensor | None = None,
                   next_position: Tensor | None = None) -> tuple[Tensor, Tensor, Tensor]:
    """Shrink every sequence of more than `keep` tokens to `keep`, per key/value head, in place: kept are the tokens of the
    last `recent` positions (position >= next_position[b] - recent) and then those with the largest accumulated weight
    (`weights` of `paged_attention`), the lowest slot first among equals; NaN ranks below every number.  Rows that stay
    are not touched: the i-th free slot below `keep` takes the i-th kept token from `keep` on, so heads may hold different
    tokens in the same slot, and slots are in no order of age afterwards.

    positions (int32, shape of `weights`) records the position of the token in every slot, next_position (int32 [batch])
    the position the next token will have: give both back to `paged_kv_append` and later evictions.  Without `positions`
    nothing has been evicted yet and slot i holds position i; next_position then is `lengths`.

    Returns (lengths, weights, positions) of the shrunken sequences as new tensors; entries behind the new length are 0
    and -1.  The pages behind ceil(length / page_size) are free.  Rows move inside a sequence's pages: none of them may be
    shared with another sequence."""
    ext = _binding()
    if ext and (got := ext.paged_evict(cache._addr, cache._index, page_table, lengths, weights, keep, recent, positions,
                                       next_position, _status(cache.device))) is not None:
        _check_every_call(cache)
        return got
    _require_cuda(weights, "paged_kv_evict")
    _no_autograd("paged_kv_evict", weights)
    batch = _check_table(cache, page_table, lengths)
    _check_stats(weights, "weights", torch.float32, batch, cache)
    width = weights.shape[2]
    if keep < 1 or recent < 0 or recent > keep:
        raise ValueError("paged_kv_evict: keep is at least 1 and recent between 0 and keep")
    if positions is not None:
        _check_stats(positions, "positions", torch.int32, batch, cache, width)
        if next_position is None:
            raise ValueError("positions goes with next_position")
        _check_int32(next_position, "next_position", (batch,), cache)
    elif next_position is not None:
        raise ValueError("next_position goes with positions")
    new_lengths = torch.empty_like(lengths)
    new_weights, new_positions = torch.empty_like(weights), torch.empty(weights.shape, dtype=torch.int32, device=cache.device)
    if batch == 0:
        return new_lengths, new_weights, new_positions
    lib = _lib.lib()
    keep = min(keep, 2**31 - 1)
    n_ws = int(lib.mxq_paged_evict_workspace_bytes(cache._addr, batch, width, keep))
    with _on_device(weights):
        ws = torch.empty((n_ws,), dtype=torch.uint8, device=cache.device)
        rc = lib.mxq_paged_evict(cache._addr, batch, page_table.data_ptr(), page_table.shape[1], page_table.stride(0),
                                 lengths.data_ptr(), weights.data_ptr(), 0 if positions is None else positions.data_ptr(),
                                 0 if next_position is None else next_position.data_ptr(), width, keep, recent,
                                 new_lengths.data_ptr(), new_weights.data_ptr(), new_positions.data_ptr(), ws.data_ptr(),
                                 n_ws, _status(cache.device).data_ptr(), _stream(weights))
    _lib.check(rc, "mxq_paged_evict")
    _check_every_call(cache)
    return new_lengths, new_weights, new_positions


class PagedKVState:
    """The paged caches of a model's attention layers, with the page table, the lengths and (`track=True`) the statistics
    that eviction needs.  The attention blocks of `mase_b200.attention` take it as `past_key_value`:

        state = PagedKVState([PagedKVCache(...) for _ in layers], page_table)
        block(hidden, (cos, sin), mask, past_key_value=state)   # every layer, layer_idx names its cache
        state.advance(tokens)                                   # once per forward, when all layers have run

    A block writes its new keys and values into the pages.  A single new token per sequence then attends over the pages
    (`paged_attention`) when the block asks for nothing that needs the dense probabilities: no attention_mask, and softmax
    and probabilities not quantized (`bypass` of "softmax" and "av_matmul").  Everything else, prompts above all, reads the
    cached rows back as dense tensors.

    counts (int32 [batch] or None): how many of the forward's tokens each sequence has (a right-padded batch); set it before
    the forward, `advance` uses it and clears it.  max_length is the host's bound on the lengths (default: their
    maximum now): dense tensors are that long, plus the new tokens, and a mask has to be at least that wide.  `advance` adds
    the padded number of tokens to it; `refresh()` makes it the largest length again, which the room check does by itself
    before it refuses, and every forward on dense tensors once `advance` or `evict` has been captured into a graph.  A
    captured forward on dense tensors has them as long as they were at its capture: a replay with longer sequences is
    reported by `check_status()`.  `lengths`, `next_position` and the tensors of `weights` and `positions` are updated in
    place.  There is no backward pass: run the model under torch.no_grad() or torch.inference_mode()."""

    def __init__(self, caches: list[PagedKVCache], page_table: Tensor, lengths: Tensor | None = None,
                 max_length: int | None = None, track: bool = False):
        if not caches:
            raise ValueError("PagedKVState needs the cache of at least one layer")
        first = caches[0]
        for c in caches:
            if (c.num_kv_heads, c.page_size, c.device) != (first.num_kv_heads, first.page_size, first.device):
                raise ValueError("the layers' caches have the same heads and page size and are on one device")
        self.caches, self.page_table = list(caches), page_table
        if lengths is None:
            lengths, max_length = torch.zeros(page_table.shape[0], dtype=torch.int32, device=first.device), max_length or 0
        batch = _check_table(first, page_table, lengths)
        self.lengths, self.max_length, self.counts = lengths, max_length, None
        self._replayed = False  # a captured graph moves the lengths: max_length may be anything by the next forward
        if max_length is None:
            self.refresh()
        self.capacity = page_table.shape[1] * first.page_size
        self.next_position = lengths.clone()  # positions count evicted tokens too
        self._slots = torch.arange(self.capacity, dtype=torch.int32, device=first.device)
        self._slots[:1] = -1  # the first row is hidden from nobody: a softmax needs one
        self.weights = self.positions = None
        if track:
            shape = (batch, first.num_kv_heads, self.capacity)
            slots = torch.arange(self.capacity, dtype=torch.int32, device=first.device).expand(shape)
            self.weights = [torch.zeros(shape, dtype=torch.float32, device=first.device) for _ in caches]
            self.positions = [slots.contiguous() for _ in caches]

    def check_format(self, layer_idx: int, fmt: str | None, config: dict | None) -> None:
        """Raises unless the layer's cache has the format that a block's `kv_cache` entry asks for."""
        c = self.caches[layer_idx]
        if (c._code, c._bits) != _format_of(fmt, config):
            raise ValueError(f"layer {layer_idx}: the block's kv_cache configuration is not the format of its paged cache")

    def _capturing(self) -> bool:
        if not self.lengths.is_cuda:
            return False
        with _on_device(self.lengths):
            return torch.cuda.is_current_stream_capturing()

    def refresh(self) -> None:
        """Set max_length to the largest length now.  Reads the lengths back: not while a graph is captured."""
        if self._capturing():
            raise RuntimeError("PagedKVState.refresh reads the lengths back: call it before the capture")
        self.max_length = int(self.lengths.max()) if self.lengths.numel() else 0

    def _check_room(self, tokens: int) -> None:
        if self.max_length + tokens <= self.capacity:
            return
        if not self._capturing():  # the bound counts padded tokens too: look at the lengths before refusing
            self.refresh()
            after = self.lengths + (tokens if self.counts is None else self.counts)
            if after.numel() == 0 or int(after.max()) <= self.capacity:
                return
        raise ValueError(f"{self.max_length} + {tokens} tokens do not fit a page table of {self.capacity}"
                         + (" (refresh() before the capture goes by the lengths)" if self._capturing() else ""))

    def lengths_after(self, tokens: int) -> Tensor:
        """The lengths once the forward's tokens are cached.  Added up by every call: a sum that is kept would not be part
        of a captured graph, and replays of one change the lengths behind the host's back."""
        self._check_room(tokens)
        return self.lengths + (tokens if self.counts is None else self.counts)

    def append(self, key: Tensor, value: Tensor, layer_idx: int) -> None:
        self._check_room(key.shape[2])
        tracked = {} if self.positions is None else {"positions": self.positions[layer_idx],
                                                     "next_position": self.next_position}
        paged_kv_append(self.caches[layer_idx], key, value, self.page_table, self.lengths, self.counts, **tracked)

    def update(self, key: Tensor, value: Tensor, layer_idx: int, cache_kwargs=None) -> tuple[Tensor, Tensor]:
        """Write new keys and values and return all cached ones as dense tensors (the call of a key/value cache)."""
        if self._replayed and not self._capturing():
            self.refresh()
        self.append(key, value, layer_idx)
        cache, tokens = self.caches[layer_idx], key.shape[2]
        keys, after = self.max_length + tokens, self.lengths_after(tokens)
        # a length that the dense tensors do not cover (a graph replayed beyond what it was captured for) is reported
        _status(cache.device).masked_fill_((after > keys).any(), 8)
        return paged_kv_gather(cache, self.page_table, after, keys, key.dtype)

    def attend(self, query: Tensor, layer_idx: int, scaling: float | None = None) -> Tensor:
        """`paged_attention` of the token that has just been appended; accumulates its weights when tracking.  The query of
        a sequence that has no new token (`counts` 0) is padding: it adds nothing to the statistics, and when tracking its
        result is zeros."""
        lengths, weights = self.lengths_after(1), None if self.weights is None else self.weights[layer_idx]
        if weights is not None and self.counts is not None:
            lengths = lengths.masked_fill(self.counts <= 0, 0)
        return paged_attention(self.caches[layer_idx], query, self.page_table, lengths, scaling, weights)

    def _absent(self, tokens: int, keys: int) -> Tensor:
        """[batch, 1, 1, keys]: the dense row is behind the sequence's tokens, and not its first one."""
        slots = self._slots[:keys]
        if keys > self.capacity:  # padded tokens
            slots = torch.cat([slots, torch.arange(self.capacity, keys, dtype=torch.int32, device=slots.device)])
        return slots >= self.lengths_after(tokens)[:, None, None, None]

    def hide_absent(self, mask: Tensor | None, tokens: int, keys: int, dtype: torch.dtype) -> Tensor:
        """An additive mask for the scores [batch, heads, tokens, keys] over the dense tensors of `update`: `mask` with the
        lowest value of its type at the rows that are behind a sequence's tokens (zeros in the dense tensors, which would
        take their share of the softmax).  A sequence without tokens keeps its first row, and gets its zeros as a result."""
        absent = self._absent(tokens, keys)  # [batch, 1, 1, keys]
        if mask is None:
            mask = absent.to(dtype).mul(torch.finfo(dtype).min)
            return mask if tokens == 1 else mask.expand(-1, -1, tokens, -1).contiguous()
        if not mask.is_floating_point():
            mask = mask.to(dtype)
        return mask[:, :, :, :keys].masked_fill(absent, torch.finfo(mask.dtype).min)

    def accumulate(self, probabilities: Tensor, layer_idx: int) -> None:
        """Add dense softmax weights [batch, heads, tokens, keys] of the forward's tokens (before dropout and the quantizer
        of the probabilities, as `attend` counts them) to the statistics of the tokens that each sequence has."""
        if self.weights is None:
            return
        b, h, t, n = probabilities.shape
        heads = self.caches[layer_idx].num_kv_heads
        p = probabilities.detach().float().masked_fill(self._absent(t, n), 0.0)
        if self.counts is not None:  # rows of padding count for nothing
            padding = torch.arange(t, device=p.device) >= self.counts[:, None]
            p = p.masked_fill(padding[:, None, :, None], 0.0)
        p = p.view(b, heads, h // heads, t, n).sum((2, 3))
        self.weights[layer_idx][:, :, :n] += p[:, :, : self.capacity]  # padding may make the dense tensors longer than that

    def advance(self, tokens: int) -> None:
        """The forward's tokens are now cached in every layer."""
        self._check_room(tokens)
        new = tokens if self.counts is None else self.counts
        self.lengths.add_(new)
        self.next_position.add_(new)
        self.max_length += tokens
        self.counts = None
        self._replayed |= self._capturing()

    def evict(self, keep: int, recent: int = 0) -> None:
        """`paged_kv_evict` in every layer; needs `track=True`."""
        if self.weights is None:
            raise RuntimeError("eviction needs the statistics of a PagedKVState with track=True")
        for i, cache in enumerate(self.caches):
            lengths, weights, positions = paged_kv_evict(
                cache, self.page_table, self.lengths, self.weights[i], keep, recent, self.positions[i], self.next_position)
            self.weights[i].copy_(weights)  # in place: captured steps hold on to these tensors
            self.positions[i].copy_(positions)
        self.lengths.copy_(lengths)
        self.max_length = min(self.max_length, keep)
        self._replayed |= self._capturing()
