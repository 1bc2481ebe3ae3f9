"""Recurrent layers and beam search as they are used together: chosen blocks behind a reordering, selection, reordering and a recurrent
layer's step in one captured graph, a module's parameters, copies, two calls at once."""
import numpy as np
import pytest
import torch

import kvhip
from tests.test_gpu_beams import moved, rows_of, write
from tests.test_gpu_gated_delta import conv_inputs, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_blocks_are_chosen_by_the_rows_that_a_sequence_has_become(dtype):
    """Bounds of blocks, whole and unfinished, move with their rows."""
    gen = torch.Generator(device="cuda").manual_seed(1)

    def new(n):
        return (torch.randn(4, 2, n, 128, generator=gen, device="cuda").to(dtype) for _ in range(2))

    order = torch.tensor([2, 2, 0, 1], dtype=torch.int32)
    cache, plain = kvhip.BlockScaledKVCache(), kvhip.BlockScaledKVCache()
    for n in (700, 1, 90, 1, 1):
        k, v = new(n)
        write(cache, k, v)
        write(plain, k, v)
    cache.reorder(order.cuda())
    for step in range(70):  # (over a block's end)
        q = torch.randn(4, 8, 1, 128, generator=gen, device="cuda").to(dtype)
        want, got = plain.select_blocks(q, 5), cache.select_blocks(moved(q, order), 5)
        assert torch.equal(got, moved(want, order)), step
        k, v = new(1)
        a = plain.update_attend_blocks(q, k, v, 0.1, 5)[0]
        b = cache.update_attend_blocks(moved(q, order), moved(k, order), moved(v, order), 0.1, 5)[0]
        assert torch.equal(b, moved(a, order)), step


@pytest.mark.parametrize("n", [1, 40])
def test_selection_reordering_and_a_recurrent_step_in_one_graph(n):
    """What has no position on the host can be replayed: every replay is the eager calls'."""
    rng = np.random.default_rng(n)
    gen = torch.Generator(device="cuda").manual_seed(2)
    B, K, V = 2, 3, 5000
    dtype = torch.bfloat16
    x, state = make(rng, B * K, n, 2, 4, 128, 128, dtype)
    y, w, bias, window = conv_inputs(rng, B * K, n, 1024, 4, dtype)
    logits, scores = torch.randn(B, K, V, generator=gen, device="cuda"), torch.zeros(B, K, device="cuda")
    k, v = (torch.randn(B * K, 2, 300, 64, generator=gen, device="cuda").to(dtype) for _ in range(2))

    def step(kv, cache):
        rows, tokens, best = kvhip.beam_select(logits, scores)
        kv.reorder(rows.flatten(), shared=100)
        cache.reorder(rows.flatten())
        return rows, tokens, best, kvhip.causal_convolution(y, w, cache, bias=bias), kvhip.gated_delta_update(**x, cache=cache)

    def caches():
        kv, cache = kvhip.KVCacheSimple(), kvhip.GatedDeltaCache()
        kv.update(k, v, fetch=False)
        cache.window, cache.delta_state = window, state
        return kv, cache

    eager, captured = caches(), caches()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*captured)
    for replay in range(5):
        graph.replay()
        torch.cuda.synchronize()
        want = step(*eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), replay
        assert all(torch.equal(a, b) for i in (0, 1) for a, b in zip(rows_of(captured[i]), rows_of(eager[i]))), replay
        logits.normal_(generator=gen)
        y.normal_(generator=gen)
        torch.cuda.synchronize()


@pytest.mark.parametrize("kept", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 70])
def test_a_modules_parameters(n, kept):
    """Parameters, which require gradients, in any type that a checkpoint has: what their values give."""
    rng = np.random.default_rng(n)
    dtype = torch.bfloat16
    x, state = make(rng, 2, n, 2, 4, 64, 64, dtype)
    y, w, bias, window = conv_inputs(rng, 2, n, 512, 4, dtype)
    x["a_log"], x["dt_bias"] = x["a_log"].to(kept), x["dt_bias"].to(kept)
    results = []
    for own in (lambda t: t, torch.nn.Parameter):
        cache = kvhip.GatedDeltaCache()
        cache.window, cache.delta_state = window, state
        out = kvhip.causal_convolution(y, own(w), cache, bias=own(bias))
        given = dict(x, a_log=own(x["a_log"]), dt_bias=own(x["dt_bias"]))
        results.append((out, kvhip.gated_delta_update(**given, cache=cache), cache.window, cache.delta_state))
    assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(*results))


def test_two_streams_at_once():
    """Two layers' calls side by side, each with a workspace of its own."""
    rng = np.random.default_rng(3)
    x, state = make(rng, 4, 700, 4, 8, 128, 128, torch.bfloat16)
    gen = torch.Generator(device="cuda").manual_seed(4)
    logits, scores = torch.randn(4, 8, 100000, generator=gen, device="cuda").bfloat16(), -100 - torch.rand(4, 8, generator=gen, device="cuda")

    def calls():
        cache = kvhip.GatedDeltaCache()
        cache.delta_state = state
        return [*(kvhip.gated_delta_update(**x, cache=cache) for _ in range(3)), cache.delta_state, *kvhip.beam_select(logits, scores, 16)]

    want = calls()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for _ in range(3):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                results.append(calls())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in results for a, b in zip(r, want))
