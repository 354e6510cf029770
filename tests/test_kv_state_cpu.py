"""The bookkeeping of `PagedKVState` without a GPU: lengths, room, masks and statistics on CPU tensors."""

from types import SimpleNamespace

import pytest
import torch

import mase_b200 as mb


def i32(v):
    return torch.tensor(v, dtype=torch.int32)


def make_state(batch=2, width=4, page=16, heads=2, lengths=None, track=True, layers=1, **more):
    """A state over caches of which only the sizes are looked at."""
    caches = [SimpleNamespace(num_kv_heads=heads, page_size=page, device=torch.device("cpu")) for _ in range(layers)]
    table = torch.arange(batch * width, dtype=torch.int32).view(batch, width)
    return mb.PagedKVState(caches, table, None if lengths is None else i32(lengths), track=track, **more)


def test_statistics_take_no_weight_behind_a_sequence():
    state = make_state(lengths=[5, 2])
    p = torch.full((2, 4, 1, 6), 1 / 6)  # a softmax that nothing was hidden from: 6 dense rows for lengths 6 and 3
    state.accumulate(p, 0)
    assert torch.equal(state.weights[0][0, :, :6], torch.full((2, 6), 2 / 6))
    assert torch.equal(state.weights[0][1, :, :3], torch.full((2, 3), 2 / 6)) and float(state.weights[0][1, :, 3:].abs().max()) == 0.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_absent_rows_are_hidden(dtype):
    state = make_state(batch=3, lengths=[5, 2, 0])
    low = torch.finfo(dtype).min
    state.counts = i32([1, 1, 0])
    got = state.hide_absent(None, 1, 6, dtype)
    assert got.dtype == dtype and got.shape == (3, 1, 1, 6)
    want = torch.zeros(3, 6, dtype=dtype)
    want[1, 3:], want[2, 1:] = low, low  # a sequence without tokens keeps one row, of zeros
    assert torch.equal(got[:, 0, 0], want)
    # a caller's mask stays as it is where there are tokens, and may be wider and shared by the batch
    mask = torch.randn(1, 1, 1, 9).to(dtype)
    got = state.hide_absent(mask, 1, 6, dtype)
    assert got.dtype == dtype and torch.equal(got[:, 0, 0], torch.where(want == low, want, mask[0, 0, :, :6].expand(3, 6)))
    with pytest.raises(RuntimeError):
        state.hide_absent(mask[..., :4], 1, 6, dtype)
