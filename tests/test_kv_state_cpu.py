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


@pytest.mark.parametrize("made,counted", [(True, True), (True, False), (False, True)])
def test_inference_mode(made, counted):
    """Tensors made under inference mode have no version counter; a state and its counts may be such tensors."""
    with torch.inference_mode(made):
        state = make_state(lengths=[5, 2])
    with torch.inference_mode(counted):
        counts = i32([1, 0])
    with torch.inference_mode():
        assert state.lengths_after(1).tolist() == [6, 3]
        state.counts = counts
        assert state.lengths_after(1).tolist() == [6, 2]
        state.accumulate(torch.full((2, 4, 1, 6), 0.25), 0)
        state.advance(1)
        assert state.lengths.tolist() == [6, 2] == state.next_position.tolist() and state.max_length == 6


def test_lengths_that_change_behind_the_hosts_back():
    """What a replayed graph does to the lengths leaves no trace on the host."""
    state = make_state(lengths=[5, 2])
    assert state.lengths_after(1).tolist() == [6, 3]
    state.lengths.data.add_(4)  # does not count as a new version
    assert state.lengths_after(1).tolist() == [10, 7]


def test_eviction_keeps_the_statistics_tensors(monkeypatch):
    """A captured step writes the tensors it was captured with: eviction leaves its results there."""
    from mase_b200 import kv_cache

    def evict(cache, table, lengths, weights, keep, recent, positions, next_position):
        return lengths.clamp(max=keep), weights.flip(-1), positions.flip(-1)

    monkeypatch.setattr(kv_cache, "paged_kv_evict", evict)
    state = make_state(lengths=[9, 2], layers=2)
    for w in state.weights:
        w.copy_(torch.rand_like(w))
    held = list(state.weights) + list(state.positions)
    want = [t.flip(-1) for t in held]
    state.evict(5)
    assert all(a is b for a, b in zip(held, state.weights + state.positions))
    assert all(torch.equal(a, b) for a, b in zip(held, want))
    assert state.lengths.tolist() == [5, 2] and state.max_length == 5


@pytest.mark.parametrize("track", [True, False])
def test_a_sequence_without_a_new_token_adds_no_weight(monkeypatch, track):
    from mase_b200 import kv_cache

    seen = []
    monkeypatch.setattr(kv_cache, "paged_attention", lambda cache, query, table, lengths, scaling, weights: seen.append((lengths, weights)))
    state = make_state(lengths=[5, 2], track=track)
    state.attend(None, 0)
    state.counts = i32([0, 1])
    state.attend(None, 0)
    assert [n.tolist() for n, _ in seen] == [[6, 3], [0, 3] if track else [5, 3]]
    assert all(n.dtype == torch.int32 and w is (state.weights[0] if track else None) for n, w in seen)


def test_room_goes_by_the_lengths_not_by_the_padding():
    state = make_state()  # room for 64 tokens
    for counts in ([30, 0], [0, 30]):
        state.counts = i32(counts)
        assert state.lengths_after(30).tolist() == [sum(x) for x in zip(state.lengths.tolist(), counts)]
        state.advance(30)
    assert state.lengths.tolist() == [30, 30] and state.max_length == 60
    assert state.lengths_after(10).tolist() == [40, 40] and state.max_length == 30
    state.advance(10)
    state.counts = i32([24, 3])  # 30 padded tokens, of which the first sequence has 24
    assert state.lengths_after(30).tolist() == [64, 43]
    p = torch.full((2, 4, 30, 70), 1 / 70)  # dense tensors of 40 + 30 rows
    state.accumulate(p, 0)
    assert torch.allclose(state.weights[0].sum(-1), torch.tensor([[48 * 64 / 70] * 2, [6 * 43 / 70] * 2]))
    state.advance(30)
    assert state.lengths.tolist() == [64, 43]
    with pytest.raises(ValueError, match="fit"):
        state.lengths_after(1)
    state.counts = i32([0, 1])
    assert state.lengths_after(1).tolist() == [64, 44]
    state.counts = None
    state.refresh()
    assert state.max_length == 64


def test_a_state_of_no_sequences():
    state = make_state(batch=0, lengths=[])
    assert state.max_length == 0 and state.lengths_after(3).tolist() == []


def test_the_status_word_can_be_cleared_under_any_mode(monkeypatch):
    """A status word made by a first call under inference mode is cleared and reported outside of it."""
    from mase_b200 import _lib, gemm

    monkeypatch.setattr(gemm, "_STATUS", {})
    with torch.inference_mode():
        status = gemm._status(torch.device("cpu"))
    status.fill_(8)
    with pytest.raises(_lib.MxqError, match="paged cache"):
        gemm.check_status()
    assert int(status) == 0
    gemm.check_status()


def test_the_bound_after_captured_steps(monkeypatch):
    """A captured advance or eviction runs on the host once, and on the lengths with every replay: the dense length of the
    next forward goes by the lengths."""
    from mase_b200 import gemm, kv_cache

    asked = []
    monkeypatch.setattr(gemm, "_STATUS", {})
    monkeypatch.setattr(kv_cache, "paged_kv_append", lambda *a, **k: None)
    monkeypatch.setattr(kv_cache, "paged_kv_gather", lambda cache, table, after, keys, dtype: asked.append((after.tolist(), keys)))
    monkeypatch.setattr(kv_cache, "paged_kv_evict", lambda c, t, n, w, keep, recent, p, x: (n.clamp(max=keep), w, p))
    row = torch.zeros(2, 2, 3, 8)
    for step in (lambda s: s.advance(1), lambda s: s.evict(4)):
        state = make_state(lengths=[9, 5])
        state.update(row, row, 0)
        with monkeypatch.context() as m:
            m.setattr(state, "_capturing", lambda: True)
            before = state.lengths.clone()
            step(state)
            state.lengths.copy_(before)  # a capture executes nothing
            state.update(row, row, 0)  # and cannot look at the lengths
        bound = state.max_length
        state.lengths.copy_(i32([20, 11]))  # replays
        state.update(row, row, 0)
        assert asked == [([12, 8], 12), ([12, 8], bound + 3), ([23, 14], 23)] and state.max_length == 20
        asked.clear()
        gemm._STATUS.clear()


def test_lengths_beyond_the_dense_tensors_are_reported(monkeypatch):
    from mase_b200 import _lib, gemm, kv_cache

    monkeypatch.setattr(gemm, "_STATUS", {})
    monkeypatch.setattr(kv_cache, "paged_kv_append", lambda *a, **k: None)
    monkeypatch.setattr(kv_cache, "paged_kv_gather", lambda *a: None)
    row = torch.zeros(2, 2, 3, 8)
    state = make_state(lengths=[9, 5])
    state.update(row, row, 0)
    gemm.check_status()
    state.lengths.data.add_(1)
    state.update(row, row, 0)
    with pytest.raises(_lib.MxqError, match="paged cache"):
        gemm.check_status()


def test_the_pages_of_a_cache_cannot_be_exchanged():
    """The calls go by the tensors' addresses, so a cache keeps the tensors it was made with."""
    cache = mb.PagedKVCache.__new__(mb.PagedKVCache)
    cache._tensors = tuple(torch.zeros(1) for _ in range(4))
    for i, name in enumerate(("key", "value", "key_scales", "value_scales")):
        assert getattr(cache, name) is cache._tensors[i]
        with pytest.raises(AttributeError):
            setattr(cache, name, torch.zeros(1))
        with pytest.raises(AttributeError):
            delattr(cache, name)


def test_derivatives_are_refused():
    from torch.autograd import forward_ad

    from mase_b200.kv_cache import _no_autograd

    x = torch.zeros(3)
    _no_autograd("call", x, None)
    with pytest.raises(NotImplementedError, match="call has no derivative"):
        _no_autograd("call", x, torch.zeros(3, requires_grad=True))
    with torch.no_grad():
        _no_autograd("call", torch.zeros(3, requires_grad=True))
    with forward_ad.dual_level():
        _no_autograd("call", x)
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(NotImplementedError, match="call has no derivative"):
                _no_autograd("call", forward_ad.make_dual(x, x))


def test_page_tables_of_one_column_have_no_column_stride():
    from mase_b200.kv_cache import _check_table

    cache = SimpleNamespace(device=torch.device("cpu"))
    wide = torch.zeros(3, 8, dtype=torch.int32)
    assert _check_table(cache, wide[:, ::8], i32([1, 2, 3])) == 3 and wide[:, ::8].stride(1) == 8
    assert _check_table(cache, wide[:1, ::8].t(), i32([1])) == 1
    with pytest.raises(ValueError, match="contiguous rows"):
        _check_table(cache, wide[:, ::2], i32([1, 2, 3]))


def test_a_capture_cannot_look_at_the_lengths(monkeypatch):
    state = make_state(lengths=[9, 5])
    state.max_length = 60  # padding
    with monkeypatch.context() as m:
        m.setattr(state, "_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="before the capture"):
            state.refresh()
        with pytest.raises(ValueError, match="do not fit.*before the capture"):
            state.lengths_after(5)
    assert state.lengths_after(5).tolist() == [14, 10] and state.max_length == 9
