"""Paged key/value cache without a GPU: refusals before any launch, in Python and at the C entry points."""

import ctypes

import pytest
import torch

import mase_b200 as mb
from mase_b200 import _lib, build

CFG = {"data_in_block_size": 32, "data_in_exponent_width": 4, "data_in_frac_width": 3}


@pytest.fixture(scope="module")
def library():
    build.build()
    return _lib.lib()


def desc(**changes):
    fields = dict(key=256, value=256, key_scales=256, value_scales=256, pages=4, format=_lib.CACHE_E4M3, bits=0, heads=2,
                  head_dim=64, page_size=16, reserved=0)
    fields.update(changes)
    return _lib.PagedCache(**fields)


def test_struct_matches_the_library(library):
    assert library.mxq_paged_cache_size() == ctypes.sizeof(_lib.PagedCache) == 64


def test_cpu_tensors_and_unknown_formats_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        mb.PagedKVCache(4, 2, 64, 16, "mxfp", CFG, "cpu")
    for kwargs in ({"head_dim": 80}, {"page_size": 8}, {"config": dict(CFG, data_in_exponent_width=3, data_in_frac_width=2)},
                   {"config": dict(CFG, data_in_block_size=64)}, {"fmt": "mxint", "config": {"data_in_block_size": 32, "data_in_width": 9}}):
        with pytest.raises(NotImplementedError):
            mb.PagedKVCache(**{**dict(num_pages=4, num_kv_heads=2, head_dim=64, page_size=16, fmt="mxfp", config=CFG), **kwargs})
    for kwargs in ({"fmt": "int4"}, {"config": None}, {"num_pages": 0}, {"num_kv_heads": 0}):
        with pytest.raises(ValueError):
            mb.PagedKVCache(**{**dict(num_pages=4, num_kv_heads=2, head_dim=64, page_size=16, fmt="mxfp", config=CFG), **kwargs})


@pytest.mark.parametrize("changes,code", [
    ({"key": 0}, -5), ({"value_scales": 0}, -5), ({"format": 5}, -3), ({"format": -1}, -3),
    ({"format": _lib.CACHE_INT8, "bits": 9}, -3), ({"head_dim": 96}, -7), ({"page_size": 8}, -7), ({"page_size": 48}, -7),
    ({"page_size": 512}, -7), ({"heads": 0}, -2), ({"heads": 70000}, -2), ({"pages": -1}, -2), ({"pages": 2 ** 31}, -2),
    ({"key": 264}, -4), ({"key_scales": 260}, -4)])
def test_bad_caches_are_refused_at_every_entry_point(library, changes, code):
    c = ctypes.addressof(d := desc(**changes))
    tab = (ctypes.c_uint8 * 256)()
    assert library.mxq_paged_append(c, 256, 256, 1, 1, 1, 0, 0, 0, 0, 0, 0, 256, 1, 1, 256, None, None, 0, None, tab, None, None) == code
    assert library.mxq_paged_gather(c, 256, 256, 1, 1, 1, 256, 1, 1, 256, None, None) == code
    assert library.mxq_paged_attention(c, 256, 256, 1, 1, 2, 64, 64, 1.0, 256, 1, 1, 256, None, 0, 256, 1 << 30, None, None) == code
    assert library.mxq_paged_evict(c, 1, 256, 1, 1, 256, 256, None, None, 16, 4, 0, 256, 256, 256, 256, 1 << 20, None, None) == code
    assert library.mxq_paged_attention_workspace_bytes(c, 1, 2, 1, 0) == code
    del d


def test_bad_arguments_are_refused(library):
    c = ctypes.addressof(d := desc())
    tab = (ctypes.c_uint8 * 256)()

    def append(key=256, value=256, dtype=1, batch=1, tokens=1, strides=(0, 0, 0, 0, 0, 0), table=256, width=1, stride=1,
               lengths=256, positions=None, pwidth=0, tab=tab):
        return library.mxq_paged_append(c, key, value, dtype, batch, tokens, *strides, table, width, stride, lengths, None,
                                        positions, pwidth, None, tab, None, None)

    assert append(batch=0) == 0 and append(tokens=0) == 0
    assert append(dtype=2) == -1 and append(batch=-1) == -2 and append(tokens=-1) == -2 and append(batch=70000) == -2
    assert append(key=None) == -5 and append(lengths=None) == -5 and append(table=None) == -5 and append(tab=None) == -5
    assert append(key=264) == -4 and append(strides=(4, 0, 0, 0, 0, 0)) == -4
    assert append(width=0) == -2 and append(batch=2, width=4, stride=3) == -2 and append(width=2 ** 28) == -2
    assert append(positions=256, pwidth=0) == -2

    def attention(q=256, out=256, dtype=1, batch=1, heads=2, table=256, width=1, stride=1, lengths=256, weights=None, ww=0,
                  ws=256, n_ws=1 << 30):
        return library.mxq_paged_attention(c, q, out, dtype, batch, heads, 64, 64, 1.0, table, width, stride, lengths, weights,
                                           ww, ws, n_ws, None, None)

    assert attention(batch=0) == 0
    assert attention(dtype=3) == -1 and attention(heads=3) == -2 and attention(heads=0) == -2 and attention(batch=-1) == -2
    assert attention(q=None) == -5 and attention(lengths=None) == -5 and attention(table=None) == -5
    assert attention(weights=256, ww=0) == -2
    assert attention(width=64, ws=None) == -5 and attention(width=64, ws=264) == -4 and attention(width=64, n_ws=64) == -2
    big = desc(pages=2 ** 31 - 1, heads=32767, head_dim=256, page_size=256, format=_lib.CACHE_BF16)
    assert library.mxq_paged_attention(ctypes.addressof(big), 256, 256, 1, 1, 32767, 64, 64, 1.0, 256, 1, 1, 256, None, 0, 256,
                                       1 << 40, None, None) == -2  # keys of more than 64 GiB
    need = library.mxq_paged_attention_workspace_bytes
    assert need(c, 1, 2, 64, 0) > 0 and need(c, 1, 2, 64, 1) > need(c, 1, 2, 64, 0) and need(c, 1, 3, 64, 0) == -2
    assert need(c, 0, 2, 64, 0) == 0

    def evict(batch=1, table=256, lengths=256, weights=256, width=32, keep=4, recent=0, out=256, ws=256, n_ws=1 << 20):
        return library.mxq_paged_evict(c, batch, table, 2, 2, lengths, weights, None, None, width, keep, recent, out, out, out,
                                       ws, n_ws, None, None)

    assert evict(batch=0) == 0 and evict(width=0) == -2
    assert evict(keep=0) == -2 and evict(recent=5) == -2 and evict(recent=-1) == -2 and evict(n_ws=8) == -2
    assert evict(weights=None) == -5 and evict(ws=None) == -5 and evict(ws=260) == -4 and evict(table=None) == -5
    assert library.mxq_paged_evict_workspace_bytes(c, 3, 32, 4) == 3 * 2 * 9 * 4
    assert library.mxq_paged_evict_workspace_bytes(c, 3, 32, 0) == -2

    gather = lambda dtype=1, tokens=1, key=256: library.mxq_paged_gather(c, key, 256, dtype, 1, tokens, 256, 1, 1, 256, None, None)  # noqa: E731
    assert gather(tokens=0) == 0 and gather(dtype=9) == -1 and gather(tokens=-1) == -2 and gather(key=None) == -5 and gather(key=8) == -4
    del d
