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
