"""Paged MX key/value cache on the GPU: append / gather against the CPU oracle bit for bit, single-token attention against
a plain implementation in 64 bits, eviction against a plain selection, and all of them together.

Bounds of the attention tests.  With A = sum_j p_j |v_j| and B = max_j scaling * sum_d |q_d k_jd| (both in 64 bits):
  * scores are sums of head_dim exact products in at most head_dim / 16 accumulation steps (times three for the split fp32
    queries), each of which may drop 2**-22 of the partial sums' magnitude, plus the rounding of the scaling: the error of
    a score is at most gamma * B, gamma = (3 * head_dim / 16 + 4) * 2**-22;
  * a probability's relative error is at most twice that plus exp2 and its argument (|s - m| <= 2 B, relative 2**-23 each,
    and 2 ulp of the function: 2**-21), and the same again for the sum;
  * probabilities enter the second product with 16 significant bits (bf16 queries: 2**-16) or 24 (2**-23);
  * the result is rounded once: half a step of its type."""

import math

import pytest
import torch

import mase_b200 as mb
from conftest import assert_bits_equal
from mase_b200 import _lib, gemm
from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

CONFIGS = {
    "none": (None, None),
    "e4m3": ("mxfp", {"data_in_block_size": 32, "data_in_exponent_width": 4, "data_in_frac_width": 3}),
    "e5m2": ("mxfp", {"data_in_block_size": 32, "data_in_exponent_width": 5, "data_in_frac_width": 2}),
    "e2m1": ("mxfp", {"data_in_block_size": 32, "data_in_exponent_width": 2, "data_in_frac_width": 1}),
    "int8": ("mxint", {"data_in_block_size": 32, "data_in_width": 8}),
    "int5": ("mxint", {"data_in_block_size": 32, "data_in_width": 5}),
}


def fake(x, name):
    """What the cache holds of x, by the oracle (CPU)."""
    fmt, cfg = CONFIGS[name]
    if fmt is None:
        return x.bfloat16()
    if fmt == "mxfp":
        return O.mxfp_fake(x, 32, cfg["data_in_exponent_width"], cfg["data_in_frac_width"])
    return O.mxint_fake(x, 32, cfg["data_in_width"])


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def make_cache(name, heads, dim, page, tokens, spare=2, seed=0, fill=0xFF):
    """A cache with room for sequences of `tokens` (list), shuffled pages and garbage in every slot; and its table."""
    fmt, cfg = CONFIGS[name]
    need = [-(-n // page) for n in tokens]
    pages = sum(need) + spare
    cache = mb.PagedKVCache(pages, heads, dim, page, fmt, cfg, DEV)
    for t in (cache.key, cache.value, cache.key_scales, cache.value_scales):
        if t is not None:
            t.view(torch.uint8).fill_(fill)  # NaN for bf16, the top code and scale byte 255 for the quantized formats
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(tokens), max(1, max(need))), -1, dtype=torch.int32)
    for i, k in enumerate(need):
        table[i, :k] = torch.tensor([order.pop() for _ in range(k)], dtype=torch.int32)
    return cache, table.to(DEV)


def rows(*shape, seed, dtype, spread=0.6):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    return (x * torch.exp(spread * torch.randn(shape[-1], generator=g))).to(dtype)


def fill(cache, table, lens, name, seed, dtype=torch.bfloat16, scale=1.0):
    """Random keys and values for every cached token; returns their cached values, float64 [batch, heads, most, dim]."""
    heads, dim, most = cache.num_kv_heads, cache.head_dim, max(max(lens), 1)
    k = rows(len(lens), heads, most, dim, seed=seed, dtype=dtype) * scale
    v = rows(len(lens), heads, most, dim, seed=seed + 1, dtype=dtype) * scale
    mb.paged_kv_append(cache, k.to(DEV), v.to(DEV), table, i32([0] * len(lens)), counts=i32(lens))
    return fake(k, name).double(), fake(v, name).double()


def plain_attention(q, k, v, lens, scaling):
    """(out, weights, A, B) in 64 bits; q [batch, heads, dim], k, v [batch, kv_heads, most, dim]."""
    n, hq, dim = q.shape
    hkv, most = k.shape[1], k.shape[2]
    g = hq // hkv
    qg = q.double().view(n, hkv, g, dim)
    out, a, bound = torch.zeros(n, hkv, g, dim).double(), torch.zeros(n, hkv, g, dim).double(), torch.zeros(n, hkv, g, 1).double()
    w = torch.zeros(n, hkv, most).double()
    for b, length in enumerate(lens):
        if length == 0:
            continue
        kb, vb = k[b, :, :length], v[b, :, :length]
        p = torch.softmax(qg[b] @ kb.transpose(1, 2) * scaling, -1)
        out[b], a[b], w[b, :, :length] = p @ vb, p @ vb.abs(), p.sum(1)
        bound[b] = (qg[b].abs() @ kb.abs().transpose(1, 2)).amax(-1, keepdim=True) * abs(scaling)
    return out.view(n, hq, dim), w, a.view(n, hq, dim), bound.view(n, hq, 1)


def weight_error(bound, dim):
    gamma = (3 * dim / 16 + 4) * 2.0 ** -22
    return 2 * (2 * gamma * bound + 2 * bound * 2.0 ** -22 + 2.0 ** -20)


def check_attention(out, q, k, v, lens, scaling):
    ref, w, a, bound = plain_attention(q, k, v, lens, scaling)
    bf = out.dtype == torch.bfloat16
    tol = a * (weight_error(bound, q.shape[-1]) + (2.0 ** -16 if bf else 2.0 ** -22)) + \
        ref.abs() * torch.finfo(out.dtype).eps / 2 + 1e-37
    err = (out.double().cpu().view_as(ref) - ref).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    return w, bound


# ---- append and gather -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name", list(CONFIGS))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,page,heads", [(32, 16, 3), (64, 32, 1), (128, 64, 2), (256, 128, 2)])
def test_append_then_gather_equals_the_oracle(name, dtype, dim, page, heads):
    before, new = [0, 5, page, 2 * page - 1], [37, 1, 0, page + 2]
    after = [a + b for a, b in zip(before, new)]
    cache, table = make_cache(name, heads, dim, page, after, seed=dim)
    old_k, old_v = fill(cache, table, before, name, seed=1, dtype=dtype)
    untouched = [t.clone() for t in (cache.key, cache.value, cache.key_scales, cache.value_scales) if t is not None]
    # as a projection leaves them: [batch, tokens, heads, dim] seen as [batch, heads, tokens, dim]
    k, v = (rows(4, max(new), heads, dim, seed=s, dtype=dtype).transpose(1, 2) for s in (3, 4))
    k[0, :, 1, :32] = 0.0
    k[3, 0, 0, :32] *= 2.0 ** -20
    mb.paged_kv_append(cache, k.to(DEV), v.to(DEV), table, i32(before), counts=i32(new))
    got_k, got_v = mb.paged_kv_gather(cache, table, i32(after), max(after) + 3, dtype)
    gemm.check_status()
    for got, old, x in ((got_k, old_k, k), (got_v, old_v, v)):
        x = fake(x.contiguous(), name).to(dtype)
        for b in range(4):
            want = torch.cat([old[b, :, : before[b]].to(dtype), x[b, :, : new[b]],
                              torch.zeros(heads, got.shape[2] - after[b], dim, dtype=dtype)], dim=1)
            assert_bits_equal(got[b], want, f"{name} sequence {b}", signed_zero=False)
    # nothing but the new rows changed
    written = torch.zeros(cache.key.shape[0], page, dtype=torch.bool)
    for b in range(4):
        for i in range(before[b], after[b]):
            written[table[b, i // page].item(), i % page] = True
    for t, u in zip([t for t in (cache.key, cache.value, cache.key_scales, cache.value_scales) if t is not None], untouched):
        same = (t.view(torch.uint8) == u.view(torch.uint8)).all(-1).all(1).cpu()
        assert bool(same[~written].all())


@pytest.mark.parametrize("name", ["e4m3", "e5m2", "e2m1", "int8", "int5"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gather_at_the_ends_of_the_range(name, dtype):
    """Blocks of every magnitude a float has, from subnormal results to the largest finite ones."""
    n = 250
    cache, table = make_cache(name, 1, 32, 16, [n])
    x = rows(1, 1, n, 32, seed=7, dtype=torch.float32, spread=1.0)
    x = x / x.abs().amax(-1, keepdim=True) * torch.exp2(torch.arange(n).float() - 124)[None, None, :, None]
    x = x.to(dtype)
    mb.paged_kv_append(cache, x.to(DEV), x.to(DEV), table, i32([0]))
    for got in mb.paged_kv_gather(cache, table, i32([n]), n, dtype):
        assert_bits_equal(got, fake(x, name), name, signed_zero=False)


@pytest.mark.parametrize("name", ["e4m3", "e5m2", "int8", "int5"])
def test_codes_are_those_of_the_plain_quantizers(name):
    cache, table = make_cache(name, 2, 64, 16, [16], spare=0)
    x = rows(1, 2, 16, 64, seed=9, dtype=torch.bfloat16).to(DEV)
    mb.paged_kv_append(cache, x, -x, table, i32([0]))
    fmt, cfg = CONFIGS[name]
    for side, y in ((0, x), (1, -x)):
        if fmt == "mxfp":
            meta = mb.MXFPMeta(32, 8, cfg["data_in_exponent_width"], cfg["data_in_frac_width"], True, "rn")
            scales, codes = mb.extract_mxfp_components(y, meta)
        else:
            scales, codes = mb.mxint_codes(y, 32, cfg["data_in_width"])
        page = (cache.key, cache.value)[side][table[0, 0]], (cache.key_scales, cache.value_scales)[side][table[0, 0]]
        assert torch.equal(page[0].reshape(-1), codes.view(torch.uint8).reshape(-1))
        assert torch.equal(page[1].reshape(-1), scales.reshape(-1))


def test_positions_are_recorded():
    cache, table = make_cache("int8", 2, 32, 16, [20, 9])
    pos = torch.full((2, 2, 24), -7, dtype=torch.int32, device=DEV)
    x = rows(2, 2, 4, 32, seed=1, dtype=torch.float32).to(DEV)
    mb.paged_kv_append(cache, x, x, table, i32([16, 5]), counts=i32([4, 3]), positions=pos)
    assert pos[0, :, 16:20].tolist() == [[16, 17, 18, 19]] * 2 and pos[1, :, 5:8].tolist() == [[5, 6, 7]] * 2
    mb.paged_kv_append(cache, x, x, table, i32([10, 0]), counts=i32([2, 1]), positions=pos, next_position=i32([100, 3]))
    assert pos[0, :, 10:12].tolist() == [[100, 101]] * 2 and pos[1, :, 0].tolist() == [3, 3]
    assert int((pos == -7).sum()) == 2 * (24 - 6) + 2 * (24 - 4)
    gemm.check_status()


# ---- attention -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name", list(CONFIGS))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,page,heads,group", [(32, 16, 2, 1), (64, 16, 1, 5), (128, 64, 2, 4), (128, 32, 1, 19),
                                                  (256, 128, 1, 8), (64, 256, 3, 16)])
def test_attention_against_64_bits(name, dtype, dim, page, heads, group):
    lens = [0, 1, 15, 16, 17, 64, 65, 203]
    cache, table = make_cache(name, heads, dim, page, lens, seed=3)
    k, v = fill(cache, table, lens, name, seed=11)
    # strided queries: heads inside a wider row
    q = rows(len(lens), heads * group, 2, dim, seed=12, dtype=dtype)[:, :, :1]
    out = mb.paged_attention(cache, q.to(DEV), table, i32(lens), dim ** -0.5)
    gemm.check_status()
    assert out.shape == q.shape and out.dtype == dtype and bool((out[0] == 0).all())
    check_attention(out[:, :, 0], q[:, :, 0], k, v, lens, dim ** -0.5)


@pytest.mark.parametrize("name,group,dtype", [("e4m3", 4, torch.bfloat16), ("e5m2", 2, torch.bfloat16), ("int8", 19, torch.bfloat16),
                                              ("e4m3", 11, torch.float32), ("int8", 1, torch.float32), ("none", 8, torch.bfloat16),
                                              ("e2m1", 12, torch.bfloat16)])
def test_attention_split_over_the_length(name, group, dtype):
    """Lengths that end anywhere in the split, a table that is much wider than most sequences, accumulated weights."""
    lens = [9001, 1, 4096, 0, 2500]
    cache, table = make_cache(name, 2, 64, 64, lens, seed=5)
    k, v = fill(cache, table, lens, name, seed=21)
    q = rows(len(lens), 2 * group, 64, seed=22, dtype=dtype)
    out = mb.paged_attention(cache, q.to(DEV), table, i32(lens))
    w, bound = check_attention(out, q, k, v, lens, 0.125)
    start = torch.rand(len(lens), 2, 9100, device=DEV)
    acc = start.clone()
    again = mb.paged_attention(cache, q.to(DEV), table, i32(lens), weights=acc)
    assert_bits_equal(again, out, "with weights")
    gemm.check_status()
    grown = (acc - start).double().cpu()[:, :, :9001]
    tol = w * weight_error(bound, 64).view(len(lens), 2, -1).amax(-1, keepdim=True) + 2.0 ** -23
    assert bool(((grown - w).abs() <= tol).all())
    for b, length in enumerate(lens):
        assert torch.equal(acc[b, :, length:], start[b, :, length:])  # entries behind the sequence stay
    for b in range(len(lens)):  # repeatable, whatever else is in the batch
        one = mb.paged_attention(cache, q[b : b + 1].to(DEV), table[b : b + 1], i32(lens[b : b + 1]))
        check_attention(one, q[b : b + 1], k[b : b + 1], v[b : b + 1], lens[b : b + 1], 0.125)
    assert_bits_equal(mb.paged_attention(cache, q.to(DEV), table, i32(lens)), out, "second call")


@pytest.mark.parametrize("batch,longest,group", [(300, 40, 2), (70, 700, 1), (1000, 3, 16)])
def test_many_short_sequences(batch, longest, group):
    """More sequences than one warp looks at, rows that begin and end inside every CTA, rows of single tokens."""
    g = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, longest + 1, (batch,), generator=g).tolist()
    cache, table = make_cache("int8", 3, 32, 16, lens, seed=6)
    k, v = fill(cache, table, lens, "int8", seed=23)
    q = rows(batch, 3 * group, 32, seed=24, dtype=torch.bfloat16)
    acc = torch.zeros(batch, 3, longest, device=DEV)
    out = mb.paged_attention(cache, q.to(DEV), table, i32(lens), weights=acc)
    gemm.check_status()
    w, bound = check_attention(out, q, k, v, lens, 32 ** -0.5)
    tol = w * weight_error(bound, 32).view(batch, 3, -1).amax(-1, keepdim=True) + 2.0 ** -23
    most = w.shape[2]
    assert bool(((acc.double().cpu()[:, :, :most] - w).abs() <= tol).all()) and bool((acc[:, :, most:] == 0).all())


@pytest.mark.parametrize("name", ["e4m3", "e5m2", "e2m1", "int8", "none"])
@pytest.mark.parametrize("scale", [2.0 ** 40, 2.0 ** 100, 2.0 ** -60, 2.0 ** -100])
def test_attention_at_the_ends_of_the_range(name, scale):
    """Block scales far from one (the part of the exponent above 2**127 takes a second multiplication)."""
    lens = [70, 33]
    cache, table = make_cache(name, 1, 64, 16, lens)
    k, v = fill(cache, table, lens, name, seed=31, scale=scale)
    q = (rows(2, 4, 64, seed=32, dtype=torch.bfloat16).float() / scale).bfloat16()
    out = mb.paged_attention(cache, q.to(DEV), table, i32(lens))
    check_attention(out, q, k, v, lens, 0.125)


def test_scores_that_grow_and_fall_along_the_sequence():
    """The running maximum is raised late, in steps larger and smaller than its slack, and in some heads only."""
    n, dim = 600, 64
    cache, table = make_cache("none", 1, dim, 32, [n])
    k = torch.zeros(1, 1, n, dim)
    k[0, 0, :, 0] = torch.linspace(-40, 60, n)
    k[0, 0, :, 1] = 30 * torch.sin(torch.arange(n) / 7.0)
    k, v = k.bfloat16(), rows(1, 1, n, dim, seed=41, dtype=torch.bfloat16)
    mb.paged_kv_append(cache, k.to(DEV), v.to(DEV), table, i32([0]))
    q = torch.zeros(1, 4, dim)
    q[0, 0, 0], q[0, 1, 0], q[0, 2, 1], q[0, 3, 1] = 1, -1, 1, 0.01
    out = mb.paged_attention(cache, q.bfloat16().to(DEV), table, i32([n]), 1.0)
    check_attention(out, q.bfloat16(), k.double(), v.double(), [n], 1.0)


def test_offsets_beyond_32_bits():
    """The pages of a sequence at the end of a cache of more than 2**32 bytes a side."""
    dim, page, heads = 256, 256, 8
    pages = (2 ** 32) // (dim * 2 * page * heads) + 3
    fmt_none = mb.PagedKVCache(pages, heads, dim, page, None, None, DEV)
    table = i32([[pages - 1, 0, pages - 2]])
    n = 2 * page + 100
    k, v = (rows(1, heads, n, dim, seed=s, dtype=torch.bfloat16) for s in (51, 52))
    mb.paged_kv_append(fmt_none, k.to(DEV), v.to(DEV), table, i32([0]))
    got, _ = mb.paged_kv_gather(fmt_none, table, i32([n]), n)
    assert_bits_equal(got, k, "gathered")
    q = rows(1, heads, dim, seed=53, dtype=torch.bfloat16)
    check_attention(mb.paged_attention(fmt_none, q.to(DEV), table, i32([n])), q, k.double(), v.double(), [n], 1 / 16)
    lens, _, pos = mb.paged_kv_evict(fmt_none, table, i32([n]), torch.rand(1, heads, n, device=DEV), 300, 30)
    got, _ = mb.paged_kv_gather(fmt_none, table, lens, 300)
    for h in range(heads):
        assert torch.equal(got[0, h].cpu(), k[0, h][pos[0, h, :300].cpu().long()])


# ---- tables and lengths that point outside ---------------------------------------------------------------------------
def test_bad_pages_and_lengths_are_reported_and_left_out():
    lens = [40, 40, 40]
    cache, table = make_cache("e4m3", 2, 64, 16, lens, fill=0)
    k, v = fill(cache, table, lens, "e4m3", seed=61)
    q = rows(3, 4, 64, seed=62, dtype=torch.bfloat16)
    gemm.check_status()
    bad = table.clone()
    bad[1, 1] = cache.num_pages  # one past the end
    bad[2, 0] = -5
    out = mb.paged_attention(cache, q.to(DEV), bad, i32(lens))
    with pytest.raises(_lib.MxqError, match="paged cache"):
        gemm.check_status()
    gemm.check_status()  # reported once
    keep1, keep2 = [*range(16), *range(32, 40)], [*range(16, 40)]
    check_attention(out[:1], q[:1], k[:1], v[:1], [40], 0.125)
    check_attention(out[1:2], q[1:2], k[1:2, :, keep1], v[1:2, :, keep1], [24], 0.125)
    check_attention(out[2:], q[2:], k[2:, :, keep2], v[2:, :, keep2], [24], 0.125)
    w = torch.zeros(3, 2, 48, device=DEV)
    mb.paged_attention(cache, q.to(DEV), bad, i32(lens), weights=w)
    assert bool((w[1, :, 16:32] == 0).all()) and bool((w[2, :, :16] == 0).all())
    assert torch.allclose(w.sum(-1), torch.full((3, 2), 2.0, device=DEV), atol=1e-5)
    gk, _ = mb.paged_kv_gather(cache, bad, i32(lens), 40)
    assert bool((gk[1, :, 16:32] == 0).all()) and torch.equal(gk[1, :, 32:].double().cpu(), k[1, :, 32:40])
    before = [t.clone() for t in (cache.key, cache.value, cache.key_scales, cache.value_scales)]
    x = rows(3, 2, 4, 64, seed=63, dtype=torch.bfloat16).to(DEV)
    mb.paged_kv_append(cache, x, x, torch.full_like(table, -1), i32([3, 20, 45]))
    mb.paged_kv_evict(cache, torch.full_like(table, 10 ** 6), i32(lens), torch.rand(3, 2, 48, device=DEV), 20)
    for t, u in zip((cache.key, cache.value, cache.key_scales, cache.value_scales), before):
        assert torch.equal(t, u)
    with pytest.raises(_lib.MxqError, match="paged cache"):
        gemm.check_status()
    # lengths the table cannot hold, negative ones
    out = mb.paged_attention(cache, q.to(DEV), table, i32([40, 10 ** 9, -3]))
    with pytest.raises(_lib.MxqError, match="paged cache"):
        gemm.check_status()
    check_attention(out[:1], q[:1], k[:1], v[:1], [40], 0.125)
    assert bool((out[2] == 0).all())
    mb.paged_kv_append(cache, x, x, table, i32([47, 2 ** 31 - 1, -1]))  # only slot 47 of sequence 0 exists
    with pytest.raises(_lib.MxqError, match="paged cache"):
        gemm.check_status()
    gk, _ = mb.paged_kv_gather(cache, table, i32([48, 40, 40]), 48)
    assert torch.equal(gk[0, :, 47].double().cpu(), fake(x[0, :, 0].cpu(), "e4m3").double())
    assert torch.equal(gk[0, :, :40].double().cpu(), k[0])


# ---- eviction --------------------------------------------------------------------------------------------------------
def plain_evict(w, pos, length, nxt, keep, recent):
    """Source slot of every new slot of one (sequence, head)."""
    m = min(length, keep)
    if length <= keep:
        return list(range(m))
    rank = []
    for j in range(length):
        x = float(w[j])
        rank.append((0 if pos[j] >= nxt - recent else 1, 1 if math.isnan(x) else 0, 0.0 if math.isnan(x) else -x, j))
    kept = sorted(r[3] for r in sorted(rank)[:m])
    movers = iter(j for j in kept if j >= m)
    stay = {j for j in kept if j < m}
    return [j if j in stay else next(movers) for j in range(m)]


@pytest.mark.parametrize("name,dim,page", [("none", 32, 16), ("e4m3", 128, 64), ("e2m1", 32, 16), ("int8", 64, 32),
                                           ("e5m2", 256, 16)])
@pytest.mark.parametrize("keep,recent,positions", [(1, 0, False), (40, 40, True), (64, 10, True), (64, 10, False), (200, 0, True)])
def test_eviction(name, dim, page, keep, recent, positions):
    lens, heads, width = [150, 64, 65, 0, 97, 1], 2, 160
    cache, table = make_cache(name, heads, dim, page, lens, seed=71)
    fill(cache, table, lens, name, seed=72)
    g = torch.Generator().manual_seed(73)
    w = torch.randint(0, 12, (6, heads, width), generator=g).float() / 4  # many equal weights
    w[0, 0, 3], w[0, 0, 90], w[0, 1, 20:60] = math.nan, math.nan, -1.0
    w[4, 0, 5], w[4, 1, :] = -0.0, 0.0
    pos = torch.arange(width, dtype=torch.int32).expand(6, heads, width).contiguous()
    nxt = list(lens)
    if positions:
        pos = torch.stack([torch.randperm(width, generator=g) for _ in range(6 * heads)]).view(6, heads, width).int()
        nxt = [width] * 6
    before = mb.paged_kv_gather(cache, table, i32(lens), 150, torch.float32)
    raw = [t.clone() for t in (cache.key, cache.value, cache.key_scales, cache.value_scales) if t is not None]
    w_in, pos_in = w.to(DEV), pos.to(DEV)
    got = mb.paged_kv_evict(cache, table, i32(lens), w_in, keep, recent, **({"positions": pos_in, "next_position": i32(nxt)}
                                                                            if positions else {}))
    gemm.check_status()
    new_lens, new_w, new_pos = (t.cpu() for t in got)
    assert new_lens.tolist() == [min(n, keep) for n in lens]
    after = mb.paged_kv_gather(cache, table, got[0], 150, torch.float32)
    for b, length in enumerate(lens):
        m = min(length, keep)
        for h in range(heads):
            src = plain_evict(w[b, h].tolist(), pos[b, h].tolist(), length, nxt[b], keep, recent)
            assert_bits_equal(new_w[b, h], torch.cat([w[b, h][src], torch.zeros(width - m)]), "weights")
            assert new_pos[b, h].tolist() == pos[b, h][src].tolist() + [-1] * (width - m)
            for x, y in zip(before, after):
                assert torch.equal(x[b, h].cpu()[src], y[b, h, :m].cpu()), (b, h)
    assert_bits_equal(w_in, w, "input weights") if not w.isnan().any() else None
    assert torch.equal(pos_in.cpu(), pos)
    # the rows from the new length on, and pages of nobody, are as they were
    free = torch.ones(cache.num_pages, page, dtype=torch.bool)
    for b in range(6):
        for i in range(min(lens[b], keep)):
            free[table[b, i // page].item(), i % page] = False
    for t, u in zip([t for t in (cache.key, cache.value, cache.key_scales, cache.value_scales) if t is not None], raw):
        assert bool((t.view(torch.uint8) == u.view(torch.uint8)).all(-1).all(1).cpu()[free].all())


@pytest.mark.parametrize("heads,n", [(1, 60000), (8, 9000), (150, 50000)])
def test_eviction_of_long_rows(heads, n):
    """Rows shared by a cluster of CTAs, and rows of more slots than one CTA keeps keys of on chip."""
    keep, page = n // 3, 256
    cache, table = make_cache("none", heads, 32, page, [n], spare=0)
    x = rows(1, heads, n, 32, seed=81, dtype=torch.bfloat16)
    mb.paged_kv_append(cache, x.to(DEV), x.to(DEV), table, i32([0]))
    w = torch.rand(1, heads, n, generator=torch.Generator().manual_seed(82)).mul(5000).floor()
    lens, new_w, pos = mb.paged_kv_evict(cache, table, i32([n]), w.to(DEV), keep, 500)
    got, _ = mb.paged_kv_gather(cache, table, lens, keep)
    gemm.check_status()
    for h in {0, heads // 2, heads - 1}:
        src = plain_evict(w[0, h].tolist(), list(range(n)), n, n, keep, 500)
        assert pos[0, h, :keep].tolist() == src and torch.equal(new_w[0, h, :keep].cpu(), w[0, h][src])
        assert torch.equal(got[0, h].cpu(), x[0, h][src])
    assert bool((pos[..., keep:] == -1).all()) and bool((new_w[..., keep:] == 0).all())


# ---- together --------------------------------------------------------------------------------------------------------
class Model:
    """Dense bookkeeping of what a cache holds, sequence by sequence and head by head."""

    def __init__(self, n, heads, dim):
        self.k = [[torch.zeros(0, dim).double() for _ in range(heads)] for _ in range(n)]
        self.v = [[torch.zeros(0, dim).double() for _ in range(heads)] for _ in range(n)]


@pytest.mark.parametrize("name", ["e4m3", "int8"])
def test_prompt_steps_and_eviction_together(name):
    n, heads, group, dim, page, budget = 3, 2, 3, 64, 16, 48
    prompt = [30, 47, 9]
    cache, table = make_cache(name, heads, dim, page, [budget + 16] * n, seed=91)
    width = budget + 16
    weights = torch.zeros(n, heads, width, device=DEV)
    positions = torch.full((n, heads, width), -1, dtype=torch.int32, device=DEV)
    k, v = (rows(n, heads, max(prompt), dim, seed=s, dtype=torch.bfloat16) for s in (92, 93))
    mb.paged_kv_append(cache, k.to(DEV), v.to(DEV), table, i32([0] * n), counts=i32(prompt), positions=positions)
    dense = [[[fake(x[b, h, : prompt[b]], name).double() for h in range(heads)] for b in range(n)] for x in (k, v)]
    seen, lengths = i32(prompt), i32(prompt)
    acc = [[torch.zeros(prompt[b]).double() for _ in range(heads)] for b in range(n)]
    for step in range(30):
        nk, nv = (rows(n, heads, 1, dim, seed=100 + 2 * step + s, dtype=torch.bfloat16) for s in (0, 1))
        mb.paged_kv_append(cache, nk.to(DEV), nv.to(DEV), table, lengths, positions=positions, next_position=seen)
        lengths, seen = lengths + 1, seen + 1
        q = rows(n, heads * group, dim, seed=200 + step, dtype=torch.bfloat16)
        out = mb.paged_attention(cache, q.to(DEV), table, lengths, weights=weights)
        for b in range(n):
            for h in range(heads):
                for side, x in ((0, nk), (1, nv)):
                    dense[side][b][h] = torch.cat([dense[side][b][h], fake(x[b, h], name).double()])
                kk, vv = dense[0][b][h][None, None], dense[1][b][h][None, None]
                qq = q[b, h * group : (h + 1) * group][None]
                w, _ = check_attention(out[b, h * group : (h + 1) * group][None], qq, kk, vv, [kk.shape[2]], dim ** -0.5)
                acc[b][h] = torch.cat([acc[b][h], torch.zeros(1).double()]) + w[0, 0]
        if int(lengths.max()) > budget + 7:
            old_pos = positions.clone()
            lengths, new_weights, positions = mb.paged_kv_evict(cache, table, lengths, weights, budget, 8, positions, seen)
            for b in range(n):
                for h in range(heads):
                    length = len(acc[b][h])
                    at = {p: i for i, p in enumerate(old_pos[b, h, :length].tolist())}
                    src = [at[p] for p in positions[b, h, : int(lengths[b])].tolist()]
                    assert src == plain_evict(weights[b, h].tolist(), old_pos[b, h].tolist(), length, int(seen[b]), budget, 8)
                    acc[b][h] = acc[b][h][src]
                    for side in (0, 1):
                        dense[side][b][h] = dense[side][b][h][src]
            weights = new_weights
        for b in range(n):
            for h in range(heads):
                assert torch.allclose(weights[b, h, : len(acc[b][h])].double().cpu(), acc[b][h], rtol=1e-4, atol=1e-5)
    gemm.check_status()


def test_steps_without_a_pause():
    """Kernels are set up while their predecessors drain: every call still sees what the calls before it wrote, torch's
    in-place additions to the lengths among them."""
    n, heads, dim, steps = 3, 2, 64, 60
    cache, table = make_cache("e4m3", heads, dim, 16, [steps + 5] * n, seed=15)
    start = [0, 5, 2]
    k0, v0 = fill(cache, table, start, "e4m3", seed=16)
    new = [[rows(n, heads, 1, dim, seed=300 + 2 * i + s, dtype=torch.bfloat16) for s in (0, 1)] for i in range(steps)]
    qs = [rows(n, heads * 4, dim, seed=500 + i, dtype=torch.bfloat16) for i in range(steps)]
    on_gpu = [[t.to(DEV) for t in pair] + [q.to(DEV)] for pair, q in zip(new, qs)]
    lengths, outs = i32(start), []
    torch.cuda.synchronize()
    for key, value, q in on_gpu:
        mb.paged_kv_append(cache, key, value, table, lengths)
        lengths.add_(1)
        outs.append(mb.paged_attention(cache, q, table, lengths))
    gemm.check_status()
    dense = [[torch.cat([x[b, :, : start[b]]] + [fake(p[s][b], "e4m3").double() for p in new], 1) for b in range(n)]
             for s, x in ((0, k0), (1, v0))]
    for i in range(steps):
        for b in range(n):
            m = start[b] + i + 1
            check_attention(outs[i][b : b + 1], qs[i][b : b + 1], dense[0][b][None, :, :m], dense[1][b][None, :, :m], [m], 0.125)


def test_two_streams_at_once():
    """The same cache read by calls on two streams at the same time: workspaces are their own."""
    lens = [5000, 300]
    cache, table = make_cache("int8", 4, 128, 64, lens, seed=17)
    k, v = fill(cache, table, lens, "int8", seed=18)
    qs = [rows(2, 16, 128, seed=19 + i, dtype=torch.bfloat16) for i in range(2)]
    on_gpu, lengths = [q.to(DEV) for q in qs], i32(lens)
    alone = [mb.paged_attention(cache, q, table, lengths) for q in on_gpu]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(mb.paged_attention(cache, on_gpu[i], table, lengths))
    torch.cuda.synchronize()
    gemm.check_status()
    for i in range(2):
        check_attention(alone[i], qs[i], k, v, lens, 128 ** -0.5)
        for out in got[i]:
            assert torch.equal(out, alone[i])


def test_captured_eviction():
    """Eviction and read-back in a graph follow the weights and lengths of each replay."""
    cache, table = make_cache("e4m3", 2, 64, 16, [100, 90], seed=25)
    fill(cache, table, [100, 90], "e4m3", seed=26)
    kept = [t.clone() for t in (cache.key, cache.value, cache.key_scales, cache.value_scales)]
    w, lengths = torch.rand(2, 2, 112, device=DEV), i32([100, 90])
    mb.paged_kv_evict(cache, table, lengths, w, 30, 5)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        lens, new_w, pos = mb.paged_kv_evict(cache, table, lengths, w, 30, 5)
        k, _ = mb.paged_kv_gather(cache, table, lens, 30)
    for seed, n in ((1, [100, 90]), (2, [64, 20]), (3, [31, 90])):
        results = []
        for how in (g.replay, None):
            for t, u in zip((cache.key, cache.value, cache.key_scales, cache.value_scales), kept):
                t.copy_(u)
            w.copy_(torch.rand(2, 2, 112, generator=torch.Generator().manual_seed(seed)))
            lengths.copy_(i32(n))
            if how is not None:
                how()
                results.append([t.clone() for t in (lens, new_w, pos, k)])
            else:
                a = mb.paged_kv_evict(cache, table, lengths, w, 30, 5)
                results.append([*a, mb.paged_kv_gather(cache, table, a[0], 30)[0]])
        for x, y in zip(*results):
            assert torch.equal(x, y)
    gemm.check_status()


def test_captured_steps_follow_their_tensors_and_share_nothing():
    """Two graphs of the same step on different inputs, replayed in turn on another stream with changed lengths."""
    n, heads, dim, page = 2, 2, 64, 16
    tokens = 400
    cache, table = make_cache("e4m3", heads, dim, page, [tokens] * n, seed=95)
    k, v = fill(cache, table, [tokens] * n, "e4m3", seed=96)
    graphs = []
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for i in range(2):
            lens = i32([100 + i, 7])
            q = rows(n, 4, dim, seed=97 + i, dtype=torch.bfloat16).to(DEV)
            new = rows(n, heads, 1, dim, seed=99 + i, dtype=torch.bfloat16).to(DEV)
            acc = torch.zeros(n, heads, tokens, device=DEV)
            mb.paged_attention(cache, q, table, lens, weights=acc)
            g = torch.cuda.CUDAGraph()
            acc.zero_()
            with torch.cuda.graph(g, stream=stream):
                mb.paged_kv_append(cache, new, new, table, lens)
                lens += 1
                out = mb.paged_attention(cache, q, table, lens, weights=acc)
            graphs.append((g, lens, q, new, acc, out))
        for lens0 in ([50, 399], [1, 200]):
            for g, lens, q, new, acc, out in graphs:
                lens.copy_(i32(lens0))
                acc.zero_()
            for g, *_ in graphs:
                g.replay()
            stream.synchronize()
            # both graphs write the same slot; the second one's token is there now, the first attended to its own
            for i, (g, lens, q, new, acc, out) in enumerate(graphs):
                kk, vv = k.clone(), v.clone()
                for b in range(n):
                    kk[b, :, lens0[b]] = vv[b, :, lens0[b]] = fake(new[b, :, 0].cpu(), "e4m3").double()
                now = [x + 1 for x in lens0]
                assert lens.tolist() == now
                w, _ = check_attention(out, q.cpu(), kk, vv, now, 0.125)
                assert torch.allclose(acc.sum(-1), torch.full((n, heads), 2.0, device=DEV), atol=1e-5)
            for b in range(n):
                k[b, :, lens0[b]] = v[b, :, lens0[b]] = fake(graphs[1][3][b, :, 0].cpu(), "e4m3").double()
    gemm.check_status()


class ListCache:
    """The part of a dense key/value cache the attention block uses."""

    def __init__(self):
        self.k, self.v = {}, {}

    def update(self, k, v, layer_idx, cache_kwargs=None):
        self.k[layer_idx] = k if layer_idx not in self.k else torch.cat([self.k[layer_idx], k], dim=-2)
        self.v[layer_idx] = v if layer_idx not in self.v else torch.cat([self.v[layer_idx], v], dim=-2)
        return self.k[layer_idx], self.v[layer_idx]


def blocks(name, dtype, bypass, layers=2, seed=5):
    """Attention blocks of hidden 128, 8 heads of 32 over 2 key/value heads; `bypass`: softmax and probabilities plain."""
    fmt, cfg = CONFIGS[name]
    mini = {"data_in_exponent_width": 5, "data_in_frac_width": 10}
    q = {"rope": mini, "qk_matmul": cfg or {"bypass": True}, "kv_cache": cfg or {"bypass": True},
         "softmax": {"bypass": True} if bypass else mini, "av_matmul": {"bypass": True} if bypass else cfg}
    cls = mb.AttentionMXInt if fmt == "mxint" else mb.AttentionMXFP
    torch.manual_seed(seed)
    made = [cls(None, i, q, hidden_size=128, num_heads=8, num_kv_heads=2, head_dim=32, dtype=dtype) for i in range(layers)]
    return [m.to(DEV).eval() for m in made]


def rope(start, n, batch, dtype):
    pos = torch.as_tensor(start).view(-1, 1) + torch.arange(n)
    ang = pos[..., None] * (1.0 / 10000 ** (torch.arange(0, 32, 2) / 32))
    ang = torch.cat([ang, ang], -1).expand(batch, n, 32)
    return ang.cos().to(dtype).to(DEV), ang.sin().to(dtype).to(DEV)


def causal(n, past, batch, dtype):
    m = torch.full((n, past + n), torch.finfo(dtype).min).triu(past + 1).to(dtype)
    return m.expand(batch, 1, n, past + n).contiguous().to(DEV)


@pytest.mark.parametrize("name,dtype,bypass", [("e4m3", torch.float32, True), ("e4m3", torch.bfloat16, True),
                                               ("int8", torch.float32, True), ("none", torch.bfloat16, True),
                                               ("e4m3", torch.float32, False), ("e2m1", torch.float32, True)])
def test_attention_blocks_on_a_paged_cache(name, dtype, bypass):
    """A prompt, its continuation as a second chunk, and single tokens through two blocks: the same outputs as with a dense
    cache of fake-quantized keys and values.  fp32: both sides round only in fp32, over at most 96 keys; the tensor-core
    products and the softmax are each good to about 2**-18 of the largest value.  bf16: the dense side rounds scores and
    probabilities to bf16 (2**-8 of a score of magnitude up to 8 moves a probability by 3 %, weights that sum to one)."""
    batch, heads, page, width = 2, 2, 16, 6
    fmt, cfg = CONFIGS[name]
    layers = blocks(name, dtype, bypass)
    caches = [mb.PagedKVCache(batch * width + 1, heads, 32, page, fmt, cfg, DEV) for _ in layers]
    table = torch.randperm(batch * width, generator=torch.Generator().manual_seed(1)).view(batch, width).int().to(DEV)
    state, dense = mb.PagedKVState(caches, table, track=True), ListCache()
    # quantized probabilities come in blocks of 32 keys, in the dense block as well
    sizes, past = [33, 32, 1, 1, 1] if bypass else [32, 64], 0
    with torch.no_grad():
        for i, n in enumerate(sizes):
            h1 = h2 = rows(batch, n, 128, seed=40 + i, dtype=dtype, spread=0.1).to(DEV)
            cs = rope(past, n, batch, dtype)
            mask = causal(n, past, batch, dtype)
            for layer in layers:
                # the last step of the paged side runs with a mask, that is on dense tensors
                o1, p1 = layer(h1, cs, mask if n > 1 or i == 4 else None, past_key_value=state)
                o2, p2 = layer(h2, cs, mask, past_key_value=dense)
                assert (p1 is None) == (n == 1 and i < 4 and bypass)
                tol = 2e-4 if dtype == torch.float32 else 4e-2
                if not bypass:
                    tol = 2e-2  # a probability that lands on the other side of a rounding border
                err = float((o1.float() - o2.float()).abs().max() / o2.float().abs().max())
                assert err <= tol, (name, i, err)
                h1, h2 = o1, o2
                if dtype == torch.bfloat16 or not bypass:
                    h1 = h2  # compare layer by layer, not what errors grow into
            state.advance(n)
            past += n
    gemm.check_status()
    assert state.lengths.tolist() == [past, past] == state.next_position.tolist()
    for w in state.weights:  # one unit of weight for every query of every head of a group
        assert torch.allclose(w.sum(-1), torch.full((batch, heads), 4.0 * past, device=DEV), rtol=3e-2 if dtype == torch.bfloat16 or not bypass else 1e-5)
    state.evict(40, 8)
    assert state.lengths.tolist() == [40, 40] and state.max_length == 40
    for w, pos in zip(state.weights, state.positions):
        assert bool((w[..., 40:] == 0).all()) and bool((pos[..., 40:] == -1).all())
        for x in pos[..., :40].reshape(-1, 40).tolist():
            assert len(set(x)) == 40 and set(range(past - 8, past)) <= set(x)
    if not bypass:
        return
    with torch.no_grad():
        h = rows(batch, 1, 128, seed=60, dtype=dtype).to(DEV)
        for layer in layers:
            out, _ = layer(h, rope(past, 1, batch, dtype), None, past_key_value=state)
        state.advance(1)
    assert bool(torch.isfinite(out).all()) and state.lengths.tolist() == [41, 41]
    assert state.positions[0][:, :, 40].unique().tolist() == [past]
    gemm.check_status()


def test_padded_prompts_and_refusals_of_the_state():
    layers = blocks("int8", torch.float32, True, layers=1)
    fmt, cfg = CONFIGS["int8"]
    cache = mb.PagedKVCache(9, 2, 32, 16, fmt, cfg, DEV)
    table = torch.arange(8, dtype=torch.int32, device=DEV).view(2, 4)
    state = mb.PagedKVState([cache], table, track=True)
    h = rows(2, 20, 128, seed=3, dtype=torch.float32, spread=0.1).to(DEV)
    with torch.no_grad():
        state.counts = i32([20, 13])
        layers[0](h, rope(0, 20, 2, torch.float32), causal(20, 0, 2, torch.float32), past_key_value=state)
        state.advance(20)
        assert state.lengths.tolist() == [20, 13] and state.max_length == 20 and state.counts is None
        assert torch.allclose(state.weights[0].sum(-1).cpu(), torch.tensor([[80.0, 80.0], [52.0, 52.0]]), rtol=1e-5)
        step = rows(2, 1, 128, seed=4, dtype=torch.float32, spread=0.1).to(DEV)
        out, _ = layers[0](step, rope([20, 13], 1, 2, torch.float32), None, past_key_value=state)
        # the shorter sequence by itself
        alone = mb.PagedKVState([mb.PagedKVCache(9, 2, 32, 16, fmt, cfg, DEV)], table[1:])
        layers[0](h[1:, :13], rope(0, 13, 1, torch.float32), causal(13, 0, 1, torch.float32), past_key_value=alone)
        alone.advance(13)
        one, _ = layers[0](step[1:], rope(13, 1, 1, torch.float32), None, past_key_value=alone)
    assert float((out[1:] - one).abs().max() / one.abs().max()) <= 1e-5
    with pytest.raises(RuntimeError, match="track"):
        alone.evict(4)
    with pytest.raises(ValueError, match="fit"):
        state.lengths_after(60)
    with pytest.raises(ValueError, match="format"):
        blocks("e4m3", torch.float32, True, layers=1)[0](step, rope(20, 1, 2, torch.float32), None, past_key_value=state)
    with pytest.raises(ValueError):
        mb.PagedKVState([], table)
    with pytest.raises(ValueError):
        mb.PagedKVState([cache, mb.PagedKVCache(9, 2, 32, 32, fmt, cfg, DEV)], table)
    gemm.check_status()


def test_calls_without_the_compiled_binding(monkeypatch):
    """The same C calls through ctypes, arguments that need a copy among them."""
    from mase_b200 import kv_cache

    got = []
    for binding in (kv_cache._binding(), False):
        monkeypatch.setattr(kv_cache, "_BINDING", binding)
        cache, table = make_cache("e4m3", 2, 64, 16, [40, 33], fill=0)
        x = rows(2, 2, 40, 66, seed=3, dtype=torch.bfloat16).to(DEV)
        k, v = x[..., 1:65], x[..., 2:].transpose(2, 3).contiguous().transpose(2, 3)  # unaligned rows, strided elements
        positions = torch.zeros(2, 2, 48, dtype=torch.int32, device=DEV)
        mb.paged_kv_append(cache, k, v, table, i32([0, 0]), counts=i32([40, 33]), positions=positions, next_position=i32([5, 0]))
        w = torch.zeros(2, 2, 48, device=DEV)
        q = rows(2, 4, 64, 2, seed=4, dtype=torch.float32).to(DEV)[..., 0]
        out = mb.paged_attention(cache, q, table, i32([40, 33]), weights=w)
        gathered = mb.paged_kv_gather(cache, table, i32([40, 33]), 41, torch.float32)
        evicted = mb.paged_kv_evict(cache, table, i32([40, 33]), w, 20, 4, positions, i32([45, 33]))
        got.append([positions, w, out, *gathered, *evicted, cache.key, cache.value, cache.key_scales, cache.value_scales])
        assert torch.equal(gathered[0][0, :, :40].cpu(), fake(k[0].cpu().contiguous(), "e4m3").float())
    gemm.check_status()
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_refusals():
    cfg = CONFIGS["e4m3"][1]
    cache, table = make_cache("e4m3", 2, 64, 16, [16, 16])
    lens = i32([3, 4])
    q = torch.zeros(2, 4, 1, 64, device=DEV, dtype=torch.bfloat16)
    kv = torch.zeros(2, 2, 1, 64, device=DEV, dtype=torch.bfloat16)
    w = torch.zeros(2, 2, 16, device=DEV)
    for bad in (q.half(), q.double()):
        with pytest.raises(NotImplementedError):
            mb.paged_attention(cache, bad, table, lens)
        with pytest.raises(NotImplementedError):
            mb.paged_kv_append(cache, bad[:, :2], bad[:, :2], table, lens)
    with pytest.raises(NotImplementedError):
        mb.paged_kv_append(cache, kv, kv.float(), table, lens)
    with pytest.raises(NotImplementedError):
        mb.paged_kv_append(cache, kv.float().requires_grad_(), kv.float(), table, lens)
    for bad in (q[:, :3], q[:1], q[..., :32], q.expand(2, 4, 2, 64), q[:, :0]):
        with pytest.raises(ValueError):
            mb.paged_attention(cache, bad, table, lens)
    with pytest.raises(NotImplementedError):
        mb.paged_attention(cache, q.float().requires_grad_(), table, lens)
    with pytest.raises(NotImplementedError):
        mb.paged_attention(cache, q, table.long(), lens)
    with pytest.raises(ValueError):
        mb.paged_attention(cache, q, table[0], lens)
    with pytest.raises(ValueError):
        mb.paged_attention(cache, q, table[:1].expand(2, -1), lens)
    with pytest.raises(RuntimeError):
        mb.paged_attention(cache, q, table.cpu(), lens)
    with pytest.raises(RuntimeError):
        mb.paged_attention(cache, q.cpu(), table, lens)
    with pytest.raises(ValueError):
        mb.paged_attention(cache, q, table, lens, weights=w[:, :1])
    with pytest.raises(NotImplementedError):
        mb.paged_attention(cache, q, table, lens, weights=w.double())
    for bad in (kv[:, :1], kv[..., :32], kv[:1]):
        with pytest.raises(ValueError):
            mb.paged_kv_append(cache, bad, bad, table, lens)
    with pytest.raises(ValueError):
        mb.paged_kv_append(cache, kv, kv, table, lens, counts=lens.long())
    with pytest.raises(ValueError):
        mb.paged_kv_append(cache, kv, kv, table, lens, next_position=lens)
    for keep, recent in ((0, 0), (4, 5), (4, -1)):
        with pytest.raises(ValueError):
            mb.paged_kv_evict(cache, table, lens, w, keep, recent)
    with pytest.raises(ValueError):
        mb.paged_kv_evict(cache, table, lens, w, 4, 1, positions=w.int())
    with pytest.raises(ValueError):
        mb.paged_kv_gather(cache, table, lens, -1)
    with pytest.raises(NotImplementedError):
        mb.paged_kv_gather(cache, table, lens, 4, torch.float16)
    for kwargs in ({"head_dim": 96}, {"page_size": 24}, {"config": dict(cfg, data_in_exponent_width=2, data_in_frac_width=3)},
                   {"config": dict(cfg, data_in_block_size=16)}):
        with pytest.raises(NotImplementedError):
            mb.PagedKVCache(**{**dict(num_pages=4, num_kv_heads=2, head_dim=64, page_size=16, fmt="mxfp", config=cfg, device=DEV),
                               **kwargs})
    with pytest.raises(ValueError):
        mb.PagedKVCache.from_pages(cache.key, cache.value, None, cache.value_scales, "mxfp", cfg)
    with pytest.raises(ValueError):
        mb.PagedKVCache.from_pages(cache.key, cache.value[:1], cache.key_scales, cache.value_scales, "mxfp", cfg)
    # nothing to do is not an error
    assert mb.paged_attention(cache, q[:0], table[:0], lens[:0]).shape == (0, 4, 1, 64)
    mb.paged_kv_append(cache, kv[:, :, :0], kv[:, :, :0], table, lens)
    assert mb.paged_kv_gather(cache, table, lens, 0)[0].shape == (2, 2, 0, 64)
    gemm.check_status()
