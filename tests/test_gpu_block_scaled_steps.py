"""Single tokens into a block-scaled cache that the attention kernel writes, whichever kernel takes the call."""
import ctypes as C

import numpy as np
import pytest
import torch

import kvhip
from kvhip import _lib as L
from oracle import block_scaled as O
from test_gpu_block_scaled import causal, check, check_rows, exact_and_bound, fill, pair
from util import NAME, randn

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sizes", [(128, 128), (192, 128), (256, 256), (64, 64), (96, 96)])
@pytest.mark.parametrize("heads", [33, 48, 64])
def test_steps_of_many_heads_to_a_kv_head(dtype, sizes, heads):
    """More query heads to a kv head than a wavefront's tiles hold: the row is written all the same.  Tokens before, on and behind
    a block's end, and one behind a trim."""
    rng = np.random.default_rng(heads + sizes[0])
    make = pair(dtype, rng, 2, 1, sizes)
    cache, oracle = kvhip.BlockScaledKVCache(), O.BlockScaledCache(NAME[dtype])
    fill(cache, oracle, make, [61])
    scale = sizes[0] ** -0.5
    for n in (1, 1, 1, 1, -1, 1, 1):
        if n < 0:
            cache.trim(1)
            oracle.trim(1)
            continue
        (k, kd), (v, vd) = make(1)
        q, qd = randn(rng, (2, heads, 1, sizes[0]), dtype)
        got = cache.update_attend(qd, kd, vd, scale)
        oracle.update(k, v)
        check(got, *exact_and_bound(q, oracle, scale, causal(oracle.offset, 1, [0, 0])))
        check_rows(cache, oracle)


def test_a_choice_for_a_cache_made_from_a_handle():
    """Its kv heads are known to the library alone: no array of lists can be made for them here."""
    (_, k), (_, v) = pair(BF16, np.random.default_rng(1), 2, 4)(200)
    owner = kvhip.BlockScaledKVCache()
    owner.update(k, v, fetch=False)
    other = kvhip.BlockScaledKVCache(handle=owner._h)
    try:
        with pytest.raises(ValueError):
            other.select_blocks(torch.zeros(2, 8, 1, 128, dtype=BF16, device="cuda"), 3)
        with pytest.raises(ValueError):
            other.attend_blocks(torch.zeros(2, 8, 1, 128, dtype=BF16, device="cuda"), torch.zeros(2, 4, 1, 3, dtype=torch.int32, device="cuda"), 0.1)
    finally:
        other._h = None


# ---- rotary positions ---------------------------------------------------------------------------------------------
def heads_of(gen, dtype, n, sizes, heads, B=2):
    hq, h = heads
    return [torch.randn(B, x, n, d, generator=gen, device="cuda").to(dtype) for x, d in ((hq, sizes[0]), (h, sizes[0]), (h, sizes[1]))]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sizes,dims", [((64, 64), 64), ((96, 96), 64), ((192, 128), 64), ((256, 256), 128), ((50, 36), 20), ((112, 72), 112)])
@pytest.mark.parametrize("traditional", [False, True])
def test_rotary_calls_equal_rotated_arrays(dtype, sizes, dims, traditional):
    gen = torch.Generator(device="cuda").manual_seed(dims)
    rope = kvhip.RoPE(dims, traditional=traditional)
    a, b, c = (kvhip.BlockScaledKVCache() for _ in range(3))
    for n in (70, 1, 1, 60, 300, 1):
        q, k, v = heads_of(gen, dtype, n, sizes, (4, 2))
        mask = kvhip.create_attention_mask(n, a)
        at = None if n != 60 else torch.tensor([3, 900], device="cuda")
        got = kvhip.attention_with_rope_and_cache_update(rope, q, k, v, a, 0.1, mask, batch_offsets=at)
        qr, kr = (kvhip.apply_rotary_position(rope, x, b if at is None else at) for x in (q, k))
        assert torch.equal(got, b.update_attend(qr, kr, v, 0.1, mask))
        c.update_rope(rope, k, v, at)
        assert torch.equal(got, c.attend(qr, 0.1, mask))
    for other in (b, c):
        for x, y in zip(a.fetch(), other.fetch()):
            assert torch.equal(x, y)


@pytest.mark.parametrize("sizes,heads", [((128, 128), (8, 2)), ((64, 64), (3, 3)), ((50, 36), (4, 1))])
@pytest.mark.parametrize("n", [1, 4, 70])
@pytest.mark.parametrize("warm", [False, True])
@pytest.mark.parametrize("form", ["one", "apart"])
def test_captured_rotary_calls(sizes, heads, n, warm, form):
    """Also the first rotary call of a cache: what turns finds room without an allocation of the cache's.  Replay after replay."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    rope = kvhip.RoPE(sizes[0])
    cache, other = kvhip.BlockScaledKVCache(), kvhip.BlockScaledKVCache()
    _, k, v = heads_of(gen, BF16, 300, sizes, heads)
    q, k1, v1 = heads_of(gen, BF16, n, sizes, heads)
    for c in (cache, other):
        c.update(k, v, fetch=False)
        c.update_attend(q, k1, v1, 0.1, kvhip.create_attention_mask(n, c))  # (pages and attention scratch are there)
        c.trim(n)

    def step(c):
        mask = kvhip.create_attention_mask(n, c)
        if form == "one":
            return kvhip.attention_with_rope_and_cache_update(rope, q, k1, v1, c, 0.1, mask)
        turned = kvhip.apply_rotary_position(rope, q, c)
        c.update_rope(rope, k1, v1)
        return c.attend(turned, 0.1, mask)

    if warm:
        step(cache)
        cache.trim(n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(cache)
    for _ in range(3):
        for dst, src in zip((q, k1, v1), heads_of(gen, BF16, n, sizes, heads)):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, step(other))
        for a, b in zip(cache.fetch(), other.fetch()):
            assert torch.equal(a, b)
        other.trim(n)


def test_a_captured_rotary_call_without_room_does_nothing():
    """Through the C entries: refused before anything is written or allocated, and the capture goes on."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    rope = kvhip.RoPE(128)
    cache = kvhip.BlockScaledKVCache()
    _, k, v = heads_of(gen, BF16, 100, (128, 128), (8, 2))
    cache.update(k, v, fetch=False)
    q, k, v = heads_of(gen, BF16, 1, (128, 128), (8, 2))
    want = cache.attend(q, 0.1)
    r, keep = rope.to_c()
    lib, mask, out = kvhip.load(), kvhip.MaskMode.none().to_c(2, 8, 1)[0], torch.empty_like(q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s = torch.cuda.current_stream().cuda_stream
        for room in (None, q.data_ptr()):
            status = lib.kvhip_cache_update_attend_rope(cache._h, C.byref(r), None, q.data_ptr(), k.data_ptr(), v.data_ptr(), 2, 8, 2, 1, 128, 128, L.BF16,
                                                        0.1, C.byref(mask), room, out.data_ptr(), s)
            assert status == L.ERR_UNSUPPORTED
        status = lib.kvhip_cache_update_rope(cache._h, C.byref(r), None, k.data_ptr(), v.data_ptr(), 2, 2, 1, 128, 128, L.BF16, s)
        assert status == L.ERR_UNSUPPORTED and cache.offset == 100
        cache.attend(q, 0.1, out=out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    # with room, also the queries' own place, which is a buffer's business outside a capture
    other = cache.copy()
    turned = kvhip.apply_rotary_position(rope, q, cache)
    own = q.clone()
    assert lib.kvhip_cache_update_attend_rope(cache._h, C.byref(r), None, own.data_ptr(), k.data_ptr(), v.data_ptr(), 2, 8, 2, 1, 128, 128, L.BF16,
                                              0.1, C.byref(mask), own.data_ptr(), out.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    other.update_rope(rope, k, v)
    assert torch.equal(out, other.attend(turned, 0.1))
    assert lib.kvhip_cache_update_attend_rope(cache._h, C.byref(r), None, q.data_ptr(), k.data_ptr(), v.data_ptr(), 2, 7, 2, 1, 128, 128, L.BF16,
                                              0.1, C.byref(mask), None, out.data_ptr(), None) == -2
    assert cache.offset == 101


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n", [64, 65, 128, 129, 161, 300])
@pytest.mark.parametrize("heads,pads", [((4, 4), (0, 0)), ((2, 2), (70, 300)), ((2, 1), (0, 11))])
def test_prompt_chunks_of_keys_of_192(dtype, n, heads, pads):
    """Either kernel, and the rows at which one takes over from the other."""
    rng = np.random.default_rng(n)
    cache, oracle = kvhip.BlockScaledKVCache(), O.BlockScaledCache(NAME[dtype])
    fill(cache, oracle, pair(dtype, rng, 2, heads[1], (192, 128)), [730])
    q, qd = randn(rng, (2, heads[0], n, 192), dtype)
    mask = kvhip.MaskMode.window_mask(730 - n, 0, left_pad=torch.tensor(pads, device="cuda"))
    check(cache.attend(qd, 0.07, mask), *exact_and_bound(q, oracle, 0.07, causal(730, n, pads)))


@pytest.mark.parametrize("sizes", [(128, 128), (50, 36)])
@pytest.mark.parametrize("n", [1, 3])
def test_a_step_over_blocks_without_memory_has_done_nothing(sizes, n):
    """Scratch that would have to grow while a stream is being captured: the call fails before it counts its rows in, and made
    again outside it is what it would have been."""
    hip = C.CDLL("libamdhip64.so")
    gen = torch.Generator(device="cuda").manual_seed(2)
    _, k, v = heads_of(gen, BF16, 20000, sizes, (8, 2))
    cache, other = kvhip.BlockScaledKVCache(), kvhip.BlockScaledKVCache()
    cache.reserve(2, 2, sizes[0], sizes[1], BF16, 21000)
    for c in (cache, other):
        c.update(k, v, fetch=False)
    q, k, v = heads_of(gen, BF16, n, sizes, (8, 2))
    out, blocks = torch.empty(2, 8, n, sizes[1], dtype=BF16, device="cuda"), torch.empty(2, 2, n, 40, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), C.c_void_p()
    assert hip.hipStreamBeginCapture(C.c_void_p(stream.cuda_stream), 0) == 0
    status = kvhip.load().kvhip_cache_update_attend_blocks(cache._h, q.data_ptr(), k.data_ptr(), v.data_ptr(), 2, 8, 2, n, sizes[0], sizes[1], L.BF16, 0.1,
                                                           40, 1, 2, None, blocks.data_ptr(), out.data_ptr(), stream.cuda_stream)
    hip.hipStreamEndCapture(C.c_void_p(stream.cuda_stream), C.byref(graph))
    hip.hipGetLastError()
    if status == 0:  # (memory of freed caches was at hand: a captured call like any other, not replayed)
        cache.trim(n)
    assert cache.offset == 20000
    got, chosen = cache.update_attend_blocks(q, k, v, 0.1, 40, 1, 2)
    want, same = other.update_attend_blocks(q, k, v, 0.1, 40, 1, 2)
    assert torch.equal(got, want) and torch.equal(chosen, same)
    for a, b in zip(cache.fetch(), other.fetch()):
        assert torch.equal(a, b)


# ---- scores far from zero -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sizes", [(64, 64), (128, 128), (256, 256)])
@pytest.mark.parametrize("n", [1, 4, 100])
@pytest.mark.parametrize("scale", [0.37, 1.7, 3.1, -5.3])
def test_scores_beyond_24_bits(dtype, sizes, n, scale):
    """Scores whose units are beyond float32's: the keys that score highest, all alike, share the weight, and no other has any.
    A query is one channel of 2^12 to 2^15, a key the same channel of 2^11 or 2^12; scores are exact."""
    rng = np.random.default_rng(n)
    dk, dv = sizes
    T = 300
    size = np.where(rng.random((2, 2, T)) < 0.1, 4096.0, 2048.0)
    size[:, :, 0] = 4096.0
    if scale < 0:
        size = 6144.0 - size
    k = np.zeros((2, 2, T, dk), np.float32)
    k[..., 3] = size
    v, vd = randn(rng, (2, 2, T, dv), dtype)
    q = np.zeros((2, 8, n, dk), np.float32)
    q[..., 3] = 2.0 ** rng.integers(12, 16, (2, 8, n)) * rng.choice([1.0, 1.5, 1.75], (2, 8, n))
    cache = kvhip.BlockScaledKVCache()
    kd, qd = (torch.from_numpy(x).to(dtype).cuda() for x in (k, q))
    cache.update(kd, vd, fetch=False)
    held, value = (x.double().cpu().numpy() for x in cache.fetch())
    assert np.array_equal(held, k)
    keep = np.arange(T) <= np.arange(T - n, T)[:, None]
    best = 4096.0 if scale > 0 else 2048.0
    weight = (keep & (size == best)[:, :, None]).astype(np.float64)
    weight /= weight.sum(-1, keepdims=True)
    want = np.repeat(weight @ value, 4, 1)
    # the weights' and the output's half steps, and the sums over at most 300 of them
    u = torch.finfo(dtype).eps / 2
    bound = u * np.abs(want) + (2 * u + 2 * T * 2.0 ** -24) * np.repeat(weight @ np.abs(value), 4, 1) + 1e-30
    check(cache.attend(qd, scale, kvhip.MaskMode.causal()), want, bound)
    blocks = torch.arange(5, dtype=torch.int32, device="cuda").expand(2, 2, n, 5).contiguous()
    check(cache.attend_blocks(qd, blocks, scale), want, bound)
    array = torch.from_numpy(keep).cuda().expand(2, 1, n, T)
    check(cache.attend(qd, scale, kvhip.MaskMode.from_array(array)), want, bound)
