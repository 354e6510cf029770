"""The ends of what the paged cache's rows can hold: signs of zeros, the last binades, infinities and NaN."""

import pytest
import torch

import mase_b200 as mb
from conftest import assert_bits_equal
from mase_b200 import gemm
from test_kv_cache_gpu import CONFIGS, DEV, check_attention, fake, fill, i32, make_cache, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,group", [(32, 1), (128, 4), (128, 12), (256, 2)])
def test_a_key_of_minus_infinity_has_no_weight(dtype, dim, group):
    """Keys with an infinite element in bf16 pages: the token as if it were not there, with queries of one bf16 term and of
    three, whose lower terms may be zero or of either sign."""
    lens, at = [5, 200, 1], [3, 130, 0]
    cache, table = make_cache("none", 2, dim, 32, lens, seed=1)
    k, v = fill(cache, table, lens, "none", seed=2)
    page, slot = [table[b, j // 32].item() for b, j in enumerate(at)], [j % 32 for j in at]
    for b in range(3):
        cache.key[page[b], :, slot[b], 7] = -float("inf")
    q = rows(3, 2 * group, dim, seed=4, dtype=dtype)
    q[..., 7] = q[..., 7].abs() + 0.5
    q[1, ..., 7] = 1.5  # one bf16 term: the others are zero
    w = torch.zeros(3, 2, 200, device=DEV)
    out = mb.paged_attention(cache, q.to(DEV), table, i32(lens), weights=w)
    gemm.check_status()
    for b, j in enumerate(at):
        rest = [i for i in range(lens[b]) if i != j]
        check_attention(out[b : b + 1], q[b : b + 1], k[b : b + 1, :, rest], v[b : b + 1, :, rest], [len(rest)], dim ** -0.5)
        assert bool((w[b, :, j] == 0).all()) and bool(torch.isfinite(w[b]).all())


@pytest.mark.parametrize("name", list(CONFIGS))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_and_signs_over_the_whole_range(name, dtype):
    """Blocks of every magnitude a float has, the subnormal and the last two binades included: the oracle's values, for
    MXFP and bf16 pages with the signs of zeros; int8 mantissas hold no negative zero."""
    n = 278  # largest elements 2**-151 .. 2**126 and 2**127 (1 - 2**-8)
    x = rows(1, 1, n + 1, 32, seed=7, dtype=torch.float32, spread=1.0).double()
    x = x / x.abs().amax(-1, keepdim=True)
    x = x * torch.cat([torch.exp2(torch.arange(n).double() - 151), torch.tensor([2.0 ** 127 * (2 - 2.0 ** -7)])])[None, None, :, None]
    x = x.float().to(dtype)
    x[..., 3], x[..., 4] = 0.0, -0.0
    assert bool(torch.isfinite(x).all()) and float(x.abs().max()) > 2.0 ** 127
    cache, table = make_cache(name, 1, 32, 16, [n + 1])
    mb.paged_kv_append(cache, x.to(DEV), -x.to(DEV), table, i32([0]))
    got = mb.paged_kv_gather(cache, table, i32([n + 1]), n + 1, dtype)
    gemm.check_status()
    for y, want in zip(got, (x, -x)):
        assert_bits_equal(y, fake(want, name).to(dtype), name, signed_zero=not name.startswith("int"))


@pytest.mark.parametrize("name", ["e4m3", "e5m2", "e2m1", "int8", "int5"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_infinities_and_nan_stay_in_their_blocks(name, dtype, bad):
    """No format has a code for them: what their block of 32 holds means nothing (with an infinity, what the plain
    quantizer makes of the block), every other block is as without them."""
    x = rows(2, 2, 40, 64, seed=9, dtype=dtype)
    spoiled = x.clone()
    spoiled[:, :, ::3, 5], spoiled[1, 1, 7, 40] = bad, bad
    blocks = torch.isfinite(spoiled.float()).view(2, 2, 40, 2, 32).all(-1, keepdim=True).expand(2, 2, 40, 2, 32).reshape(x.shape)
    cache, table = make_cache(name, 2, 64, 16, [40, 40])
    mb.paged_kv_append(cache, spoiled.to(DEV), spoiled.to(DEV), table, i32([0, 0]))
    got = mb.paged_kv_gather(cache, table, i32([40, 40]), 40, dtype)
    gemm.check_status()
    want, (fmt, cfg) = fake(x, name), CONFIGS[name]
    for y in got:
        assert_bits_equal(y.cpu()[blocks], want[blocks], name, signed_zero=fmt == "mxfp")
    if bad == bad:
        plain = mb.mxfp_quantizer(spoiled.to(DEV), 32, cfg["data_in_exponent_width"], cfg["data_in_frac_width"]) if fmt == "mxfp" \
            else mb.mxint_quantizer(spoiled.to(DEV), 32, cfg["data_in_width"])
        assert_bits_equal(got[0], plain, name, signed_zero=fmt == "mxfp")


@pytest.mark.parametrize("keep,positions", [(1, False), (40, True), (64, False), (200, True)])
def test_eviction_leaves_its_inputs_alone(keep, positions):
    """Weights (NaN among them), positions, lengths and page table keep every bit."""
    lens, width = [150, 64, 65, 0, 97, 1], 160
    cache, table = make_cache("e4m3", 2, 64, 32, lens, seed=71)
    fill(cache, table, lens, "e4m3", seed=72)
    g = torch.Generator().manual_seed(73)
    w = torch.randn(6, 2, width, generator=g)
    w[0, 0, 3], w[0, 0, 90], w[0, 1, 20:60], w[4, 1, :] = float("nan"), float("nan"), -0.0, 0.0
    pos = torch.stack([torch.randperm(width, generator=g) for _ in range(12)]).view(6, 2, width).int()
    inputs = [w.to(DEV), pos.to(DEV), i32(lens), table, i32([width] * 6)]
    before = [t.clone() for t in inputs]
    mb.paged_kv_evict(cache, table, inputs[2], inputs[0], keep, 0, **({"positions": inputs[1], "next_position": inputs[4]} if positions else {}))
    gemm.check_status()
    for a, b in zip(inputs, before):
        assert torch.equal(a.view(torch.int32), b.view(torch.int32))
