"""Beam search's selection against its definition in float64, reordered caches against the same moves on dense arrays, and both in
a run of steps.

A score is a float32 rounding of float64 arithmetic on a float32 sum of at most 2^18 exponentials: each is off by at most
|x - M| + 4 units of 2^-24 (the product with log2 e, the exponential), and partial sums of at most 64 terms to a thread, 8 to a
wavefront's step and the segments in float64 add 80 more, so that the logarithm is off by less than 200 units for |x - M| < 100 wherever an
exponential still counts."""
import numpy as np
import pytest
import torch

import kvhip
from oracle import beams as OB

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
UNIT = 2.0 ** -24


def check_select(logits, scores, count, done=None, pad_token=0):
    got = kvhip.beam_select(logits, scores, count, done, pad_token)
    want = OB.beam_select(logits.float().cpu().numpy(), None if scores is None else scores.cpu().numpy(), count,
                          None if done is None else done.cpu().numpy(), pad_token)
    rows, tokens, best = (t.cpu().numpy() for t in got)
    assert rows.dtype == np.int32 and tokens.dtype == np.int32 and best.dtype == np.float32
    assert np.array_equal(rows, want[0]) and np.array_equal(tokens, want[1])
    fine = np.isfinite(want[2])
    best, score = best.astype(np.float64), want[2]
    assert np.array_equal(np.isneginf(best), np.isneginf(score))
    assert (np.abs(best[fine] - score[fine]) <= 200 * UNIT + UNIT * np.abs(score[fine])).all()
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B, K, V, count", [(1, 1, 1, 1), (1, 1, 5, 3), (2, 4, 1000, 4), (1, 4, 32000, 8), (3, 5, 2049, 10), (2, 8, 50001, 16), (1, 64, 300, 64),
                                            (5, 3, 16383, 3), (40, 16, 4099, 16), (1, 2, 151936, 64)])
def test_select(dtype, B, K, V, count):
    gen = torch.Generator(device="cuda").manual_seed(V)
    x = (2.5 * torch.randn(B, K, V, generator=gen, device="cuda")).to(dtype)
    scores = -20 * torch.rand(B, K, generator=gen, device="cuda")
    check_select(x, scores, count)
    check_select(x, None, count)
    check_select(x, scores, count, torch.rand(B, K, generator=gen, device="cuda") < 0.4, V - 1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_values(dtype):
    """Rows of one value, of two, of few: the lower beam and the lower token, whatever the order of anything."""
    for V in (100, 5000, 40000):
        x = torch.zeros(2, 3, V, dtype=dtype, device="cuda")
        check_select(x, None, 7)
        check_select(x, torch.tensor([[0.0, 0.0, 0.0], [-1.0, 0.0, -1.0]], device="cuda"), 64)
        x[:, :, V // 2:] = 1.0
        check_select(x, None, 20)
        x = torch.randint(0, 3, (2, 3, V), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype)
        check_select(x, torch.zeros(2, 3, device="cuda"), 33)
        x = -x
        x[0, 0, :10] = 0.0
        x[0, 0, 3:5] = -0.0
        check_select(x, None, 5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_vocabularies(dtype):
    """Grammars leave a few tokens, one, or none; beams that are dead, or no numbers."""
    inf, nan = float("inf"), float("nan")
    gen = torch.Generator(device="cuda").manual_seed(2)
    for V in (50, 9000, 70001):
        x = torch.full((4, 4, V), -inf, dtype=dtype, device="cuda")
        for b in range(4):
            for k in range(4):
                n = [0, 1, 3, 40][(b + k) % 4]
                at = torch.randperm(V, generator=gen, device="cuda")[:n]
                x[b, k, at] = torch.randn(n, generator=gen, device="cuda").to(dtype)
        scores = torch.tensor([[0.0, -1.0, -2.0, -3.0], [0.0, -inf, -inf, -inf], [nan, -1.0, -inf, -2.0], [-inf] * 4], device="cuda")
        check_select(x, scores, 6)
        x[0, 1] = torch.finfo(dtype).min
        x[1, 2] = nan
        x[1, 0, 5:] = nan
        x[2, 1, 7] = inf
        x[2, 3, 2:4] = inf
        x[3, 0] = torch.finfo(dtype).max
        check_select(x, scores, 6)
        check_select(x, None, 30, torch.tensor([[True] * 4, [False, True, False, False], [False] * 4, [True, False, False, True]], device="cuda"), 3)


def test_fewer_candidates_than_asked_for():
    x = torch.randn(2, 2, 3, device="cuda")
    check_select(x, None, 10)
    rows, tokens, best = check_select(x, torch.tensor([[0.0, -1.0], [0.5, 0.25]], device="cuda"), 4, torch.ones(2, 2, dtype=torch.bool, device="cuda"), 1)
    assert rows.tolist() == [[0, 1, -1, -1], [2, 3, -1, -1]] and tokens.tolist() == [[1, 1, -1, -1]] * 2 and torch.isneginf(best[:, 2:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_rows_of_a_wider_array(dtype, shift):
    """Logits of a padded vocabulary, from any element on: what stands behind the vocabulary is never seen."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    whole = torch.full((2, 3, 5104), 1e4, dtype=dtype, device="cuda")
    part = whole[..., shift:shift + 5003]
    part.copy_(torch.randn(2, 3, 5003, generator=gen, device="cuda"))
    check_select(part, torch.zeros(2, 3, device="cuda"), 6)
    check_select(part.transpose(0, 1), None, 4)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_lie_apart_and_rows_that_are_one(dtype):
    """One beam to a batch row out of wider rows, rows that several beams share, and a prompt's one row as every beam's."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    whole = torch.randn(6, 1, 2100, generator=gen, device="cuda").to(dtype)
    for part in (whole[..., :2003], whole[:, :, 3:1900], whole[::2, :, :700], whole[:1].expand(5, 1, 2100), whole[:1].expand(1, 4, 2100),
                 whole.expand(6, 3, 2100)):
        B, K = part.shape[:2]
        scores = -torch.arange(B * K, device="cuda", dtype=torch.float32).reshape(B, K)
        check_select(part, scores, 3)
        check_select(part, scores, 3, torch.zeros(B, K, dtype=torch.bool, device="cuda"))
        check_select(part, None, 2)


def test_many_rows_and_offsets_beyond_32_bits():
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.empty(140, 64, 262144, dtype=torch.bfloat16, device="cuda")
    x.normal_(generator=gen)
    x[139, 63, 262143] = 50.0
    scores = torch.zeros(140, 64, device="cuda")
    rows, tokens, best = kvhip.beam_select(x, scores, 4)
    assert rows[139, 0] == 140 * 64 - 1 and tokens[139, 0] == 262143
    a = kvhip.beam_select(x[137:], scores[137:], 4)
    assert torch.equal(a[0] + 137 * 64, rows[137:]) and torch.equal(a[1], tokens[137:])


def test_select_in_a_graph_and_on_another_stream():
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, scores = torch.randn(4, 4, 30000, generator=gen, device="cuda"), torch.zeros(4, 4, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = kvhip.beam_select(x, scores)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # (two graphs, each with scratch of its own)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = kvhip.beam_select(x, scores)
        graphs.append((g, outs))
    for _ in range(3):
        for g, outs in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for _, outs in graphs for a, b in zip(outs, want))
        x.add_(torch.randn(4, 4, 30000, generator=gen, device="cuda"))
        want = check_select(x, scores, 4)


# ---- reordered caches -------------------------------------------------------------------------------------------------
def orders(B, rng):
    yield torch.arange(B, dtype=torch.int32)
    yield torch.zeros(B, dtype=torch.int32)
    yield torch.arange(B - 1, -1, -1, dtype=torch.int32)
    yield torch.from_numpy(rng.integers(0, B, B).astype(np.int32))
    yield torch.from_numpy(rng.permutation(B).astype(np.int64))
    odd = torch.from_numpy(rng.integers(0, B, B).astype(np.int32))
    odd[0], odd[-1] = -1, B
    yield odd


def moved(t, order):
    """What an array becomes: entries outside the batch leave their row."""
    at = torch.arange(t.shape[0])
    order = order.long()
    return t[torch.where((order >= 0) & (order < t.shape[0]), order, at).to(t.device)]


def kinds():
    yield "simple", lambda: kvhip.KVCacheSimple(), DTYPES
    yield "rotating", lambda: kvhip.RotatingKVCache(200, keep=4), DTYPES
    for bits in (2, 3, 4, 5, 6, 8):
        yield f"quantized {bits}", lambda bits=bits: kvhip.QuantizedKVCache(32, bits), DTYPES[:2]
    yield "block-scaled", lambda: kvhip.BlockScaledKVCache(), DTYPES[:2]


def write(cache, k, v):
    if isinstance(cache, kvhip.QuantizedKVCache):
        cache.update_quantized(k, v, fetch=False)
    else:
        cache.update(k, v, fetch=False)


def rows_of(cache):
    return [t.clone() for t in cache.state]


@pytest.mark.parametrize("name, dtype", [(n, d) for n, _, ds in kinds() for d in ds])
@pytest.mark.parametrize("B, H, Dk, Dv", [(3, 2, 64, 64), (8, 1, 128, 128), (5, 2, 96, 64), (1, 1, 64, 64)])
def test_reordered_caches(name, dtype, B, H, Dk, Dv):
    """Every kind, behind prompts and tokens: rows, and what attention and later tokens make of them."""
    make = dict((n, m) for n, m, _ in kinds())[name]
    rng = np.random.default_rng(B)
    gen = torch.Generator(device="cuda").manual_seed(B)

    def new(n):
        return torch.randn(B, H, n, Dk, generator=gen, device="cuda").to(dtype), torch.randn(B, H, n, Dv, generator=gen, device="cuda").to(dtype)

    for order in orders(B, rng):
        cache, plain = make(), make()
        for n in (70, 1, 140, 1, 1, 60):
            k, v = new(n)
            write(cache, k, v)
            write(plain, k, v)
        before = rows_of(cache)
        cache.reorder(order.cuda())
        for a, b in zip(rows_of(cache), before):
            assert torch.equal(a, moved(b, order)), name
        q = torch.randn(B, 2 * H, 1, Dk, generator=gen, device="cuda").to(dtype)
        want = plain.attend(q, 0.1)
        at = order.long()
        back = torch.arange(B)
        at = torch.where((at >= 0) & (at < B), at, back)
        # a row's attention under its parent's query is the parent's, bit for bit
        assert torch.equal(cache.attend(moved(q, order), 0.1), want[at.cuda()])
        k, v = new(3)
        write(cache, moved(k, order), moved(v, order))
        write(plain, k, v)
        for a, b in zip(rows_of(cache), rows_of(plain)):
            assert torch.equal(a, moved(b, order)), name


@pytest.mark.parametrize("kind", ["simple", "quantized", "block-scaled"])
def test_shared_positions_do_not_move(kind):
    """Beams of one prompt: the tiles that lie in it are left alone (here they differ, so that it shows), the others move whole."""
    B, H, D, n = 4, 2, 64, 300
    make = dict((name.split()[0], m) for name, m, _ in kinds())[kind]
    gen = torch.Generator(device="cuda").manual_seed(0)
    order = torch.tensor([2, 2, 0, 1], dtype=torch.int32)
    for shared in (0, 1, 63, 64, 100, 256, 299, 300, 320, 10 ** 9):
        cache = make()
        write(cache, *(torch.randn(B, H, n, D, generator=gen, device="cuda").half() for _ in range(2)))
        before = rows_of(cache)
        cache.reorder(order.cuda(), shared=shared)
        first = min(shared // 64 * 64, n)
        if shared >= n:
            first = n
        if kind == "block-scaled":
            first = min(first, 256)  # (rows that are not in whole blocks always move)
        for a, b in zip(rows_of(cache), before):
            if kind == "block-scaled" and shared >= 256:
                # the block in front of the unfinished one is held as codes, which stay; rows as they came move
                assert torch.equal(a[:, :, :256], b[:, :, :256]) and torch.equal(a[:, :, 256:], moved(b, order)[:, :, 256:])
                continue
            assert torch.equal(a[:, :, :first], b[:, :, :first])
            assert torch.equal(a[:, :, first:], moved(b, order)[:, :, first:])


def test_reorder_behind_a_trim_and_before_more_rows():
    """Rows that a trim took off do not come back, and what is written later is where it belongs."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    for name, make, dtypes in kinds():
        if name == "rotating":
            continue
        cache, plain = make(), make()
        k, v = (torch.randn(3, 2, 200, 64, generator=gen, device="cuda").to(dtypes[0]) for _ in range(2))
        for c in (cache, plain):
            write(c, k, v)
            c.trim(37)
        order = torch.tensor([1, 2, 2], dtype=torch.int32)
        cache.reorder(order.cuda())
        k, v = (torch.randn(3, 2, 90, 64, generator=gen, device="cuda").to(dtypes[0]) for _ in range(2))
        write(cache, moved(k, order), moved(v, order))
        write(plain, k, v)
        assert cache.offset == plain.offset == 253
        for a, b in zip(rows_of(cache), rows_of(plain)):
            assert torch.equal(a, moved(b, order)), name


def test_rotating_cache_that_has_wrapped_and_staged_rounds():
    gen = torch.Generator(device="cuda").manual_seed(2)
    cache = kvhip.RotatingKVCache(64, keep=4)
    for n in (50,) + (1,) * 40 + (7, 1):
        cache.update(*(torch.randn(3, 1, n, 64, generator=gen, device="cuda").half() for _ in range(2)), fetch=False)
    order = torch.tensor([1, 0, 0], dtype=torch.int32)
    before = rows_of(cache)
    cache.reorder(order.cuda(), shared=40)
    assert all(torch.equal(a, moved(b, order)) for a, b in zip(rows_of(cache), before))
    staged = kvhip.RotatingStagedKVCache(cache)
    with pytest.raises(kvhip.KVHipError):
        cache.reorder(order.cuda())
    staged.commit(0)
    cache.reorder(order.cuda())


def test_many_rows_and_a_long_cache():
    """As many rows as a workgroup holds, one more refused; and cells 5 GB behind the first."""
    for B in (257, 2048):
        gen = torch.Generator(device="cuda").manual_seed(B)
        cache = kvhip.KVCacheSimple()
        cache.update(*(torch.randn(B, 1, 5, 64, generator=gen, device="cuda").half() for _ in range(2)), fetch=False)
        order = torch.randint(0, B, (B,), generator=gen, device="cuda")
        before = rows_of(cache)
        cache.reorder(order)
        assert all(torch.equal(a, moved(b, order.cpu())) for a, b in zip(rows_of(cache), before))
    cache = kvhip.KVCacheSimple()
    cache.update(*(torch.zeros(2049, 1, 1, 64, device="cuda").half() for _ in range(2)), fetch=False)
    with pytest.raises(kvhip.KVHipError):
        cache.reorder(torch.zeros(2049, dtype=torch.int32, device="cuda"))
    cache = kvhip.KVCacheSimple()
    cache.reserve(2, 64, 256, 256, torch.bfloat16, 70000)
    k = torch.randn(2, 64, 70000, 256, device="cuda", dtype=torch.bfloat16)
    cache.update(k, k, fetch=False)
    cache.reorder(torch.tensor([1, 0], device="cuda"))
    a, b = cache.fetch()
    assert torch.equal(a, k.flip(0)) and torch.equal(b, k.flip(0))


def test_reorder_refusals():
    cache = kvhip.KVCacheSimple()
    cache.reorder(torch.zeros(3, dtype=torch.int32, device="cuda"))  # (holds nothing)
    k = torch.zeros(3, 1, 4, 64, device="cuda").half()
    cache.update(k, k, fetch=False)
    for bad in (torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(3, device="cuda"), torch.zeros(3, dtype=torch.int32),
                torch.zeros(3, 1, dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError):
            cache.reorder(bad)
    with pytest.raises(kvhip.KVHipError):
        cache.reorder(torch.zeros(3, dtype=torch.int32, device="cuda"), shared=-1)
    state = kvhip.GatedDeltaCache()
    state.reorder(torch.zeros(3, dtype=torch.int32, device="cuda"))
    state.delta_state = torch.zeros(3, 1, 4, 4, device="cuda")
    with pytest.raises(ValueError):
        state.reorder(torch.zeros(4, dtype=torch.int32, device="cuda"))
    state.window = torch.zeros(2, 3, 4, device="cuda")
    with pytest.raises(ValueError):
        state.reorder(torch.zeros(3, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, width", [(4, 1), (3, 5), (7, 24), (2, 4096), (33, 1000)])
def test_reordered_recurrent_states(dtype, rows, width):
    """Dense arrays of any row size (1 to 16 bytes to a unit), out of one call."""
    rng = np.random.default_rng(rows)
    gen = torch.Generator(device="cuda").manual_seed(rows)
    for order in orders(rows, rng):
        cache = kvhip.GatedDeltaCache(2)
        cache.window = torch.randn(rows, 1, width, generator=gen, device="cuda").to(dtype)
        cache.delta_state = torch.randn(rows, 1, 3, width, generator=gen, device="cuda")
        before = rows_of(cache)
        cache.reorder(order.cuda())
        assert all(torch.equal(a, moved(b, order)) for a, b in zip(rows_of(cache), before))


def test_entries_beyond_32_bits_leave_a_row_its_own():
    order = torch.tensor([2 ** 32 + 1, -2 ** 40, 2 ** 31], device="cuda")
    cache = kvhip.GatedDeltaCache()
    cache.delta_state = torch.randn(3, 1, 2, 8, device="cuda")
    simple = kvhip.KVCacheSimple()
    write(simple, *(torch.randn(3, 2, 5, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    for c in (cache, simple):
        before = rows_of(c)
        c.reorder(order, shared=2)
        assert all(torch.equal(a, b) for a, b in zip(rows_of(c), before))


def test_reorder_in_a_graph():
    gen = torch.Generator(device="cuda").manual_seed(6)
    cache, twin = kvhip.KVCacheSimple(), kvhip.KVCacheSimple()
    k, v = (torch.randn(6, 2, 400, 128, generator=gen, device="cuda").half() for _ in range(2))
    for c in (cache, twin):
        c.update(k, v, fetch=False)
    order = torch.tensor([1, 1, 0, 5, 3, 3], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.reorder(order, shared=70)
    for _ in range(4):
        graph.replay()
        twin.reorder(order, shared=70)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(rows_of(cache), rows_of(twin)))
        order.copy_(torch.randint(0, 6, (6,), generator=gen, device="cuda"))
        torch.cuda.synchronize()


@pytest.mark.parametrize("quantized", [False, True])
def test_beam_search_over_a_hybrid_model(quantized):
    """Whole steps of a two-layer toy -- attention over a KV cache, gated delta over its state -- under beam search, against running every
    hypothesis again from its first token without a cache that moves."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    B, K, V, H, D, steps, P = 2, 3, 211, 2, 64, 6, 70
    rows = B * K

    def r(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    embed, read = r(V, H * D).half(), (r(H * D, V) * 0.05).half()
    w = r(3 * H * D, 4) * 0.3
    a_log, bias = torch.zeros(H, device="cuda"), torch.zeros(H, device="cuda") - 2

    def layers(tokens, kv, state):
        """Logits of the last token of each row: tokens [rows, n]."""
        n = tokens.shape[1]
        x = embed[tokens]
        heads = x.unflatten(-1, (H, D)).transpose(1, 2).contiguous()
        attended = kvhip.attention_with_cache_update(heads, heads, heads, kv, D ** -0.5, kvhip.create_attention_mask(n, kv))
        mixed = kvhip.causal_convolution(torch.cat([x, x, x], -1).float(), w, state)
        q, k, v = (t.unflatten(-1, (H, D)) for t in mixed.split(H * D, -1))
        gate = x.unflatten(-1, (H, D)).float().mean(-1)
        out = kvhip.gated_delta_update(q, k, v, gate, gate, a_log, bias, state)
        return ((attended.transpose(1, 2).float() + out).flatten(2)[:, -1] @ read.float()).half().unflatten(0, (B, K))

    def caches():
        return (kvhip.QuantizedKVCache(64, 8) if quantized else kvhip.KVCacheSimple()), kvhip.GatedDeltaCache()

    prompt = torch.randint(0, V, (B, P), generator=gen, device="cuda").repeat_interleave(K, 0)
    kv, state = caches()
    scores = torch.tensor([0.0] + [-float("inf")] * (K - 1), device="cuda").repeat(B, 1)
    logits = layers(prompt, kv, state)
    texts = prompt
    for step in range(steps):
        order, tokens, scores = kvhip.beam_select(logits, scores)
        order = order.flatten()
        kv.reorder(order, shared=P)
        state.reorder(order)
        texts = torch.cat([texts[order.long()], tokens.reshape(rows, 1).long()], 1)
        logits = layers(tokens.reshape(rows, 1).long(), kv, state)
        fresh_kv, fresh = caches()
        layers(texts[:, :P], fresh_kv, fresh)
        for i in range(P, texts.shape[1]):
            want = layers(texts[:, i:i + 1], fresh_kv, fresh)
        assert torch.equal(logits, want), step
        assert torch.equal(state.delta_state, fresh.delta_state) and torch.equal(state.window, fresh.window)
