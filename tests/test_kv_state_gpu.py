"""`PagedKVState` through the attention blocks on the GPU: ragged batches without masks, captured steps, inference mode."""

import pytest
import torch

import mase_b200 as mb
from mase_b200 import gemm
from test_kv_cache_gpu import CONFIGS, DEV, blocks, causal, i32, rope, rows

pytestmark = pytest.mark.gpu


def make_state(name, batch, width=6, layers=1, track=True, page=16):
    fmt, cfg = CONFIGS[name]
    caches = [mb.PagedKVCache(batch * width + 1, 2, 32, page, fmt, cfg, DEV) for _ in range(layers)]
    table = torch.randperm(batch * width, generator=torch.Generator().manual_seed(1)).view(batch, width).int().to(DEV)
    return mb.PagedKVState(caches, table, track=track)


def softmax_quantized(block, av):
    """The block with its softmax input quantized, and its probabilities if `av`."""
    block.softmax_bypass = False
    block.softmax_config = {"data_in_exponent_width": 5, "data_in_frac_width": 10}
    block.av_bypass = not av
    return block


@pytest.mark.parametrize("mask", [None, "zeros"])
@pytest.mark.parametrize("name,lens,av", [("e4m3", [20, 13, 0], False), ("int8", [63, 31], True)])
def test_dense_steps_of_a_ragged_batch_without_a_mask(name, lens, av, mask):
    """One new token per sequence through a block that needs the dense tensors: each sequence as by itself, whatever rows
    of zeros the others' length leaves behind it.  Both sides round scores to 11 bits (a score of magnitude up to 8 moves
    by 2**-8, a weight by 2**-7 of itself) and, for `av`, probabilities to 8: 2e-2 of the largest output; an unmasked
    row of zeros would take 1/64 of the weight, and there are 7 to 32 of them."""
    layer = softmax_quantized(blocks(name, torch.float32, True, layers=1)[0], av)
    if av:
        layer.av_config = CONFIGS[name][1]
    n, most = len(lens), max(lens)
    state = make_state(name, n)
    k, v = (rows(n, 2, most, 32, seed=s, dtype=torch.float32).to(DEV) for s in (1, 2))
    step = rows(n, 1, 128, seed=4, dtype=torch.float32, spread=0.1).to(DEV)
    with torch.no_grad():
        state.counts = i32(lens)
        state.append(k, v, 0)
        state.advance(most)
        m = None if mask is None else torch.zeros(1, 1, 1, most + 1, device=DEV)
        out, p = layer(step, rope(lens, 1, n, torch.float32), m, past_key_value=state)
        assert p.shape[-1] == most + 1
        for b, length in enumerate(lens):
            alone = make_state(name, 1)
            if length:
                alone.append(k[b : b + 1, :, :length], v[b : b + 1, :, :length], 0)
                alone.advance(length)
            one, p1 = layer(step[b : b + 1], rope(length, 1, 1, torch.float32), None, past_key_value=alone)
            assert p1.shape[-1] == length + 1
            assert float((out[b] - one[0]).abs().max() / one.abs().max()) <= 2e-2, (b, length)
            w = state.weights[0][b]
            assert bool((w[:, length + 1 :] == 0).all())
            assert torch.allclose(w, alone.weights[0][0], rtol=0.1, atol=2e-2)
    gemm.check_status()


@pytest.mark.parametrize("advance", [True, False])
def test_captured_steps_follow_the_lengths(advance):
    """Single tokens captured after a warm-up that did not advance: every replay attends to what is cached by then, the
    lengths moved by the graph itself or between the replays."""
    layers = blocks("e4m3", torch.float32, True, layers=2)
    states = [make_state("e4m3", 2, layers=2) for _ in range(2)]
    prompt = rows(2, 20, 128, seed=2, dtype=torch.float32, spread=0.1).to(DEV)
    steps = [rows(2, 1, 128, seed=10 + i, dtype=torch.float32, spread=0.1).to(DEV) for i in range(5)]
    ropes = [rope([20 + i, 13 + i], 1, 2, torch.float32) for i in range(5)]
    outs = [[], []]
    with torch.no_grad():
        for state in states:
            state.counts = i32([20, 13])
            for layer in layers:
                layer(prompt, rope(0, 20, 2, torch.float32), causal(20, 0, 2, torch.float32), past_key_value=state)
            state.advance(20)
        for i in range(5):  # the eager side
            h = steps[i]
            for layer in layers:
                h, _ = layer(h, ropes[i], None, past_key_value=states[0])
            states[0].advance(1)
            outs[0].append(h)
        state, x, cs = states[1], steps[0].clone(), [t.clone() for t in ropes[0]]
        saved = [[t.clone() for t in group] for group in (state.weights, state.positions)]

        def forward():
            h = x
            for layer in layers:
                h, _ = layer(h, cs, None, past_key_value=state)
            return h

        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            forward()  # warm-up
            for group, old in zip((state.weights, state.positions), saved):
                for t, u in zip(group, old):
                    t.copy_(u)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                out = forward()
                if advance:
                    state.advance(1)
            for i in range(5):
                x.copy_(steps[i])
                for t, u in zip(cs, ropes[i]):
                    t.copy_(u)
                g.replay()
                if not advance:
                    state.advance(1)
                outs[1].append(out.clone())
        stream.synchronize()
    assert states[0].lengths.tolist() == [25, 18] == states[1].lengths.tolist()
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    for a, b in zip(states[0].weights + states[0].positions, states[1].weights + states[1].positions):
        assert torch.equal(a, b)
    gemm.check_status()


def test_steps_under_inference_mode():
    layer = blocks("e4m3", torch.float32, True, layers=1)[0]
    prompt = rows(2, 20, 128, seed=2, dtype=torch.float32, spread=0.1).to(DEV)
    step = rows(2, 1, 128, seed=3, dtype=torch.float32, spread=0.1).to(DEV)
    got = []
    for mode in (torch.inference_mode, torch.no_grad):
        with mode():
            s = make_state("e4m3", 2)
            s.counts = i32([20, 13])
            layer(prompt, rope(0, 20, 2, torch.float32), causal(20, 0, 2, torch.float32), past_key_value=s)
            s.advance(20)
            for i in range(2):
                out, _ = layer(step, rope([20 + i, 13 + i], 1, 2, torch.float32), None, past_key_value=s)
                s.advance(1)
            s.evict(12, 4)
            got.append([out, s.lengths, *s.weights, *s.positions])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    gemm.check_status()


def test_captured_steps_and_eviction():
    """A captured tracked step, replayed before and after evictions (one eager, one captured): the statistics that the
    evictions go by are the ones that the replays add to."""
    layer = blocks("e4m3", torch.float32, True, layers=1)[0]
    prompt = rows(2, 20, 128, seed=2, dtype=torch.float32, spread=0.1).to(DEV)
    steps = [rows(2, 1, 128, seed=10 + i, dtype=torch.float32, spread=0.1).to(DEV) for i in range(9)]
    ropes = [rope([20 + i, 13 + i], 1, 2, torch.float32) for i in range(9)]
    results = []
    with torch.no_grad():
        for captured in (False, True):
            state, x, cs = make_state("e4m3", 2), steps[0].clone(), [t.clone() for t in ropes[0]]
            state.counts = i32([20, 13])
            layer(prompt, rope(0, 20, 2, torch.float32), causal(20, 0, 2, torch.float32), past_key_value=state)
            state.advance(20)

            def forward():
                out, _ = layer(x, cs, None, past_key_value=state)
                state.advance(1)
                return out

            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                if captured:
                    parts = [state.lengths, state.next_position, *state.weights, *state.positions]
                    saved = [t.clone() for t in parts]
                    forward(), state.evict(12, 4)  # warm-up
                    for t, u in zip(parts, saved):
                        t.copy_(u)
                    c = state.caches[0]
                    layer(prompt, rope(0, 20, 2, torch.float32), causal(20, 0, 2, torch.float32),
                          past_key_value=(again := mb.PagedKVState([c], state.page_table)))  # the rows that moved, put back
                    assert again.max_length == 0
                    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
                    with torch.cuda.graph(graphs[0], stream=stream):
                        out = forward()
                    with torch.cuda.graph(graphs[1], stream=stream):
                        state.evict(12, 4)
                outs = []
                for i in range(9):
                    x.copy_(steps[i])
                    for t, u in zip(cs, ropes[i]):
                        t.copy_(u)
                    if captured:
                        graphs[0].replay()
                    else:
                        out = forward()
                    outs.append(out.clone())
                    if i == 3:
                        state.evict(16, 4)
                    if i == 6:
                        graphs[1].replay() if captured else state.evict(12, 4)
            stream.synchronize()
            results.append(outs + [state.lengths, state.next_position, *state.weights, *state.positions])
    assert state.lengths.tolist() == [14, 14]
    for a, b in zip(*results):
        assert torch.equal(a, b)
    gemm.check_status()


def test_tracked_step_with_an_idle_sequence():
    """counts 0 in a step on the pages and in one on dense tensors: neither touches the idle sequence's statistics, and the
    other's are those of the step alone."""
    for quantized in (False, True):
        layer = blocks("e4m3", torch.float32, True, layers=1)[0]
        if quantized:
            softmax_quantized(layer, False)
        state = make_state("e4m3", 2)
        prompt = rows(2, 20, 128, seed=2, dtype=torch.float32, spread=0.1).to(DEV)
        step = rows(2, 1, 128, seed=3, dtype=torch.float32, spread=0.1).to(DEV)
        with torch.no_grad():
            state.counts = i32([20, 13])
            layer(prompt, rope(0, 20, 2, torch.float32), causal(20, 0, 2, torch.float32), past_key_value=state)
            state.advance(20)
            before = state.weights[0].clone()
            state.counts = i32([1, 0])
            layer(step, rope([20, 13], 1, 2, torch.float32), None, past_key_value=state)
            state.advance(1)
        assert state.lengths.tolist() == [21, 13] == state.next_position.tolist()
        assert torch.equal(state.weights[0][1], before[1])
        assert torch.allclose((state.weights[0][0] - before[0]).sum(-1).cpu(), torch.full((2,), 4.0), rtol=1e-4)
    gemm.check_status()


def test_padded_chunks_fill_the_pages():
    """Chunks whose padding reaches behind the page table, prompts one sequence after the other: as the sequence alone.
    Projections of 60 and of 25 rows may round differently in fp32, which can move a code of one key or value by a step,
    2**-6 of the largest element of its block, and with a weight of 1/25 or more for a value: 5e-3 of the largest output
    leaves room for ten of those; a chunk that is cut off or misplaced changes it by its own size."""
    layer = blocks("int8", torch.float32, True, layers=1)[0]
    state, alone = make_state("int8", 2, width=4), make_state("int8", 1, width=4)
    parts = [rows(2, n, 128, seed=20 + i, dtype=torch.float32, spread=0.1).to(DEV) for i, n in enumerate((30, 30, 30))]
    with torch.no_grad():
        for i, (counts, start) in enumerate((([0, 30], [0, 0]), ([30, 0], [0, 30]), ([34 - 4, 25], [30, 30]))):
            state.counts = i32(counts)
            keys = state.max_length + 30
            mask = torch.stack([causal(30, s, 1, torch.float32)[0] if s + 30 == keys else torch.nn.functional.pad(
                causal(30, s, 1, torch.float32)[0], (0, keys - s - 30), value=torch.finfo(torch.float32).min) for s in start])
            out, _ = layer(parts[i], rope(start, 30, 2, torch.float32), mask, past_key_value=state)
            state.advance(30)
        assert state.lengths.tolist() == [60, 55] and state.max_length == 60
        for i, n in ((0, 30), (2, 25)):
            one, _ = layer(parts[i][1:, :n], rope(30 * (i > 0), n, 1, torch.float32), causal(n, 30 * (i > 0), 1, torch.float32),
                           past_key_value=alone)
            alone.advance(n)
        assert float((out[1, :25] - one[0]).abs().max() / one.abs().max()) <= 5e-3
        with pytest.raises(ValueError, match="fit"):
            layer(parts[0], rope(60, 30, 2, torch.float32), None, past_key_value=state)
    gemm.check_status()


def test_a_chunk_after_replayed_steps():
    """Captured single tokens, replayed, then a prompt chunk on dense tensors: as with steps that were not captured."""
    layer = blocks("e4m3", torch.float32, True, layers=1)[0]
    prompt = rows(2, 20, 128, seed=2, dtype=torch.float32, spread=0.1).to(DEV)
    step = rows(2, 1, 128, seed=3, dtype=torch.float32, spread=0.1).to(DEV)
    chunk = rows(2, 7, 128, seed=4, dtype=torch.float32, spread=0.1).to(DEV)
    cs, outs = rope(20, 1, 2, torch.float32), []
    with torch.no_grad():
        for captured in (False, True):
            state = make_state("e4m3", 2)
            layer(prompt, rope(0, 20, 2, torch.float32), causal(20, 0, 2, torch.float32), past_key_value=state)
            state.advance(20)

            def forward():
                layer(step, cs, None, past_key_value=state)
                state.advance(1)

            if captured:
                stream = torch.cuda.Stream()
                stream.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(stream):
                    forward()
                    g = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(g, stream=stream):
                        forward()
                    for _ in range(4):
                        g.replay()
                stream.synchronize()
                state.refresh()
            else:
                for _ in range(5):
                    forward()
            assert state.max_length == 25
            outs.append(layer(chunk, rope(25, 7, 2, torch.float32), causal(7, 25, 2, torch.float32), past_key_value=state)[0])
            state.advance(7)
            if captured:
                g.replay()
                outs.append(layer(chunk, rope(33, 7, 2, torch.float32), causal(7, 33, 2, torch.float32), past_key_value=state)[1])
                assert outs.pop().shape[-1] == 40
    assert torch.equal(*outs)
    gemm.check_status()


def test_masks_that_the_fused_softmax_does_not_take():
    """A mask with fewer columns than there are keys (a view whose memory goes on behind them), on another device, or with
    rows that share memory is left to the separate operations, which broadcast or refuse it."""
    from mase_b200 import functional as F

    scores = torch.randn(1, 4, 3, 64, device=DEV)
    wide = torch.randn(1, 1, 3, 96, device=DEV)
    fused = lambda mask: F.attention_softmax(scores, 0.5, mask, None, None, None, None)  # noqa: E731
    assert fused(wide[..., :40]) is None and fused(wide[..., :1]) is None and fused(wide[..., :64].cpu()) is None
    assert fused(wide[:, :, :1, :64].expand(1, 1, 3, 64)) is None
    assert torch.allclose(fused(wide), torch.softmax(scores * 0.5 + wide[..., :64], -1), atol=1e-6)
    layer = blocks("e4m3", torch.float32, True, layers=1)[0]
    h = rows(1, 32, 128, seed=2, dtype=torch.float32, spread=0.1).to(DEV)
    m = torch.randn(1, 1, 1, 32, device=DEV)
    with torch.no_grad():
        for bad in (causal(32, 0, 1, torch.float32)[..., :20], causal(32, 0, 1, torch.float32).cpu()):
            with pytest.raises(RuntimeError):
                layer(h, rope(0, 32, 1, torch.float32), bad)
        cs = rope(0, 32, 1, torch.float32)
        a, b = (layer(h, cs, x)[0] for x in (m.expand(1, 1, 32, 32), m.expand(1, 1, 32, 32).contiguous()))
    assert torch.allclose(a, b, atol=1e-5 * float(b.abs().max()))


def test_derivatives_are_refused_by_the_calls():
    from torch.autograd import forward_ad

    state = make_state("e4m3", 2)
    cache, table, lens = state.caches[0], state.page_table, i32([3, 4])
    q, kv, w = torch.zeros(2, 4, 1, 32, device=DEV), torch.zeros(2, 2, 1, 32, device=DEV), torch.zeros(2, 2, 16, device=DEV)
    calls = [lambda f: mb.paged_attention(cache, f(q), table, lens), lambda f: mb.paged_attention(cache, q, table, lens, weights=f(w)),
             lambda f: mb.paged_kv_append(cache, f(kv), kv, table, lens), lambda f: mb.paged_kv_append(cache, kv, f(kv), table, lens),
             lambda f: mb.paged_kv_evict(cache, table, lens, f(w), 2)]
    with forward_ad.dual_level():
        for call in calls:
            call(lambda t: t)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="no derivative"):
                call(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))
    for call in calls:
        with pytest.raises(NotImplementedError, match="no derivative"):
            call(lambda t: t.clone().requires_grad_())
        with torch.no_grad():
            call(lambda t: t.clone().requires_grad_())
    gemm.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dropout", [0.0, 0.5])
def test_statistics_are_those_of_the_plain_softmax(dropout, dtype):
    """Dense forwards count the softmax weights, one unit a query, not what the quantizer of the probabilities (here four
    bits) or dropout makes of them; and tracking changes no output.  The softmax is fp32; a bf16 weight is off by at most
    2**-9 of itself on one side, so is their sum."""
    layer = softmax_quantized(blocks("e4m3", dtype, True, layers=1)[0], True)
    layer.av_config = CONFIGS["e2m1"][1]
    layer.attention_dropout = dropout
    layer.train(dropout > 0)
    h = rows(2, 64, 128, seed=2, dtype=dtype, spread=0.1).to(DEV)
    outs = []
    for track in (True, False):
        state = make_state("e4m3", 2, track=track)
        with torch.no_grad():
            torch.manual_seed(5)
            outs.append(layer(h, rope(0, 64, 2, dtype), causal(64, 0, 2, dtype), past_key_value=state))
        if track:
            got = state.weights[0][:, :, :64].sum(-1)
            rel = 1e-5 if dtype == torch.float32 else 2.0 ** -9
            assert bool(((got / 256 - 1).abs() <= rel + 1e-5).all()), got
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    assert not torch.allclose(outs[0][1].float().sum(-1), torch.ones((), device=DEV), rtol=1e-2)  # the quantizer shows
    gemm.check_status()


@pytest.mark.parametrize("binding", [True, False])
def test_the_workspace_of_a_tracked_step_follows_the_statistics(monkeypatch, binding):
    """A page table far wider than the statistics: the same results and a workspace for the statistics' slots only; lengths
    behind them are reported as before."""
    from mase_b200 import _lib, kv_cache

    if not binding:
        monkeypatch.setattr(kv_cache, "_BINDING", False)
    fmt, cfg = CONFIGS["e4m3"]
    cache = mb.PagedKVCache(13, 2, 64, 16, fmt, cfg, DEV)
    table = torch.full((3, 40000), -1, dtype=torch.int32)
    table[:, :4] = torch.arange(12).view(3, 4)
    table = table.to(DEV)
    k = rows(3, 2, 50, 64, seed=1, dtype=torch.bfloat16).to(DEV)
    mb.paged_kv_append(cache, k, k, table, i32([0, 0, 0]))
    q, lens = rows(3, 8, 64, seed=2, dtype=torch.bfloat16).to(DEV), i32([50, 0, 33])
    want_w = torch.zeros(3, 2, 50, device=DEV)
    want = mb.paged_attention(cache, q, table[:, :4].contiguous(), lens, weights=want_w)
    w = torch.zeros(3, 2, 50, device=DEV)
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = mb.paged_attention(cache, q, table, lens, weights=w)
    assert torch.cuda.max_memory_allocated() - before < 8 << 20  # 3 x 40000 x 16 slots of 8 heads of scores: 61 MB
    assert torch.equal(got, want) and torch.equal(w, want_w)
    gemm.check_status()
    mb.paged_attention(cache, q, table, i32([51, 0, 33]), weights=w)
    with pytest.raises(_lib.MxqError, match="paged cache"):
        gemm.check_status()


def test_page_table_of_one_strided_column():
    fmt, cfg = CONFIGS["int8"]
    cache = mb.PagedKVCache(3, 2, 64, 16, fmt, cfg, DEV)
    table = torch.full((3, 8), -1, dtype=torch.int32, device=DEV)
    table[:, 0] = i32([2, 0, 1])
    k, lens = rows(3, 2, 9, 64, seed=1, dtype=torch.bfloat16).to(DEV), i32([9, 0, 4])
    q, got = rows(3, 8, 64, seed=2, dtype=torch.bfloat16).to(DEV), []
    for t in (table[:, ::8], table[:, :1].contiguous()):
        mb.paged_kv_append(cache, k, k, t, i32([0, 0, 0]))
        got.append([mb.paged_attention(cache, q, t, lens), *mb.paged_kv_gather(cache, t, lens, 9)])
    gemm.check_status()
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_dense_steps(dtype):
    """Steps that need the dense tensors, captured with a bound that leaves room for the replays: as eager steps on tensors
    of the same length.  A replay beyond them is reported."""
    from mase_b200 import _lib

    layer = softmax_quantized(blocks("e4m3", dtype, True, layers=1)[0], False)
    prompt = rows(3, 20, 128, seed=2, dtype=dtype, spread=0.1).to(DEV)
    steps = [rows(3, 1, 128, seed=10 + i, dtype=dtype, spread=0.1).to(DEV) for i in range(4)]
    ropes = [rope([20 + i, 13 + i, 4], 1, 3, dtype) for i in range(4)]
    results = []
    with torch.no_grad():
        for captured in (False, True):
            state = make_state("e4m3", 3)
            state.counts = i32([20, 13, 4])
            layer(prompt, rope(0, 20, 3, dtype), causal(20, 0, 3, dtype), past_key_value=state)
            state.advance(20)
            x, cs, counts = steps[0].clone(), [t.clone() for t in ropes[0]], i32([1, 1, 0])

            def forward():
                state.counts = counts
                out, p = layer(x, cs, None, past_key_value=state)
                state.advance(1)
                return out, p

            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                parts = [state.lengths, state.next_position, *state.weights, *state.positions]
                saved = [t.clone() for t in parts]
                state.max_length = 23
                forward()  # warm-up
                for t, u in zip(parts, saved):
                    t.copy_(u)
                state.max_length = 23
                if captured:
                    g = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(g, stream=stream):
                        out, p = forward()
                outs = []
                for i in range(4):
                    x.copy_(steps[i])
                    for t, u in zip(cs, ropes[i]):
                        t.copy_(u)
                    if captured:
                        g.replay()
                    else:
                        state.max_length = 23
                        out, p = forward()
                    assert p.shape[-1] == 24
                    outs += [out.clone(), p.clone()]
            stream.synchronize()
            gemm.check_status()
            assert state.lengths.tolist() == [24, 17, 4]
            results.append(outs + [*state.weights, *state.positions])
        for a, b in zip(*results):
            assert torch.equal(a, b)
        with torch.cuda.stream(stream):
            g.replay()
        stream.synchronize()
        with pytest.raises(_lib.MxqError, match="paged cache"):
            gemm.check_status()
