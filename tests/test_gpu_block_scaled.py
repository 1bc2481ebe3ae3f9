"""The block-scaled cache, attention over it and over chosen blocks, against oracle/block_scaled.py in float64."""
import numpy as np
import pytest
import torch

import kvhip
from kvhip import _lib as L
from oracle import block_scaled as O
from util import NAME, np32, randn

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
INF, NAN = float("inf"), float("nan")
# (key size, value size): those that the kernels are built for, and others that are stored padded
SIZES = [(64, 64), (96, 96), (128, 128), (256, 256), (192, 128), (80, 80), (50, 36), (112, 72)]


def pair(dtype, rng, B=2, H=2, sizes=(128, 128)):
    return lambda n: tuple(randn(rng, (B, H, n, d), dtype, 2.0) for d in sizes)


def fill(cache, oracle, make, lengths):
    for n in lengths:
        (k, kd), (v, vd) = make(n)
        cache.update(kd, vd, fetch=False)
        oracle.update(k, v)


def check_rows(cache, oracle):
    assert cache.offset == cache.presented_length == oracle.offset
    for got, want in zip(cache.fetch(), (oracle.keys, oracle.values)):
        assert np.array_equal(np32(got).astype(np.float64), want, equal_nan=True)


# ---- write and read back ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("lengths", [[1], [63, 1], [64], [65], [5, 190, 64, 1], [130, 126]])
def test_rows_are_read_back_by_the_definition(dtype, sizes, lengths):
    rng = np.random.default_rng(sum(lengths) + sizes[0])
    cache, oracle = kvhip.BlockScaledKVCache(), O.BlockScaledCache(NAME[dtype])
    fill(cache, oracle, pair(dtype, rng, sizes=sizes), lengths)
    check_rows(cache, oracle)


def test_rows_do_not_depend_on_how_many_came_together():
    make = pair(BF16, np.random.default_rng(3))
    (_, k), (_, v) = make(300)
    one, many = kvhip.BlockScaledKVCache(), kvhip.BlockScaledKVCache()
    one.update(k, v, fetch=False)
    at = 0
    for n in [1, 2, 60, 1, 1, 100, 64, 7, 63, 1]:
        many.update(k[:, :, at:at + n], v[:, :, at:at + n], fetch=False)
        at += n
    assert at == 300
    for a, b in zip(one.fetch(), many.fetch()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_edges_of_the_codes(dtype):
    """Zeros, the steps at 448 and at powers of two, ties, the type's largest and smallest values, infinities and NaN."""
    x = np.zeros((1, 1, 8 * 64, 64), np.float32)
    blocks = x[0, 0].reshape(8, 64, 64)
    top = float(torch.finfo(dtype).max)
    blocks[1, :, :8] = [448, 1, -1, 0.0625, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, -448]
    blocks[2, 3, :6] = [225, 232, 17, 19, 21, -17]                  # ties of four bits, both ways
    blocks[3, 5, :4] = [top, -top, 1.0, top / 2]
    blocks[4, :, :3] = float(torch.finfo(dtype).tiny) * 2.0 ** (-8 if dtype == F16 else -5)
    blocks[4, 0, :1] = float(torch.finfo(dtype).tiny)
    blocks[5, 7, :5] = [INF, -INF, NAN, 3.0, -5.0]
    blocks[6] = NAN
    blocks[7, 0, 0], blocks[7, 1, 1] = 1.75, 1.7578125              # the scale's step
    k = torch.from_numpy(x).to(dtype)
    cache, oracle = kvhip.BlockScaledKVCache(), O.BlockScaledCache(NAME[dtype])
    cache.update(k.cuda(), k.flip(3).contiguous().cuda(), fetch=False)
    oracle.update(k.double().numpy(), k.flip(3).double().numpy())
    check_rows(cache, oracle)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sizes", [(64, 64), (192, 128), (50, 36)])
@pytest.mark.parametrize("lengths,cut", [([200], 3), ([200], 72), ([200], 8), ([200], 136), ([128], 1), ([128], 128), ([70, 70], 100)])
def test_trimmed_rows_are_written_again(dtype, sizes, lengths, cut):
    rng = np.random.default_rng(cut)
    make = pair(dtype, rng, sizes=sizes)
    cache, oracle = kvhip.BlockScaledKVCache(), O.BlockScaledCache(NAME[dtype])
    fill(cache, oracle, make, lengths)
    assert cache.trim(cut) == cut
    oracle.trim(cut)
    if oracle.offset:
        check_rows(cache, oracle)
    for n in (1, 2, 61, 70):
        fill(cache, oracle, make, [n])
        check_rows(cache, oracle)


def test_values_read_back_are_stored_the_same():
    """Also those of a block whose scale shrinks because its largest value rounded down to 224 scales."""
    for dtype in (F16, BF16):
        gen = torch.Generator(device="cuda").manual_seed(7)
        k = (torch.randn(2, 2, 640, 64, generator=gen, device="cuda") * 10).to(dtype)
        k[0, 0, :64] = k[0, 0, :64].clamp(-1, 1)
        k[0, 0, 5, 5] = 228.0 / 128
        cache = kvhip.BlockScaledKVCache()
        a, b = cache.update(k, -k)
        again = kvhip.BlockScaledKVCache()
        c, d = again.update(a, b)
        assert torch.equal(a, c) and torch.equal(b, d)


def test_state_copy_and_trim():
    make = pair(BF16, np.random.default_rng(11), sizes=(112, 72))
    cache, oracle = kvhip.BlockScaledKVCache(), O.BlockScaledCache("bfloat16")
    assert cache.state == [] and cache.meta_state == [""] and cache.is_trimmable
    fill(cache, oracle, make, [150])
    other = cache.copy()
    restored = kvhip.BlockScaledKVCache()
    restored.state, restored.meta_state = cache.state, [""]
    for c in (other, restored):
        check_rows(c, oracle)
    cache.trim(100)
    fill(cache, O.BlockScaledCache("bfloat16"), make, [3])
    check_rows(other, oracle)  # (a copy of its own)
    fill(other, oracle, make, [60])
    check_rows(other, oracle)
    assert other.trim(-5) == 0 and other.trim(1000) == 210 and other.offset == 0
    with pytest.raises(kvhip.KVHipError):
        other.offset = 10
    fresh = O.BlockScaledCache("bfloat16")
    fill(other, fresh, make, [66])
    check_rows(other, fresh)


@pytest.mark.parametrize("step", [100, 257])
def test_growth_over_many_allocations(step):
    """Pages from a few allocations are found by the kernels' arguments, from more by the page table: the same rows either way."""
    make = pair(BF16, np.random.default_rng(step), sizes=(64, 64))
    cache, oracle = kvhip.BlockScaledKVCache(), O.BlockScaledCache("bfloat16")
    rng = np.random.default_rng(0)
    for i in range(4200 // step):
        fill(cache, oracle, make, [step])
        if i % 4 == 3:
            check_rows(cache, oracle)
            q, qd = randn(rng, (2, 4, 3, 64), BF16)
            T = oracle.offset
            check(cache.attend(qd, 0.1, kvhip.MaskMode.causal()), *exact_and_bound(q, oracle, 0.1, causal(T, 3, [0, 0])))
            blocks = cache.select_blocks(qd, 5)
            assert np.array_equal(blocks.cpu().numpy(), O.select(q, oracle, 5, 1, 1, [0, 0]))
            check(cache.attend_blocks(qd, blocks, 0.1), *exact_and_bound(q, oracle, 0.1, O.listed_keep(blocks.cpu().numpy(), T, [0, 0])))
    one = cache.copy()
    check_rows(one, oracle)


def test_emptied_caches():
    make = pair(F16, np.random.default_rng(8))
    cache = kvhip.BlockScaledKVCache()
    fill(cache, O.BlockScaledCache("float16"), make, [70])
    assert cache.trim(70) == 70
    other, restored = cache.copy(), kvhip.BlockScaledKVCache()
    assert all(a.shape[2] == 0 for a in cache.state) and all(a.shape[2] == 0 for a in cache.fetch())
    restored.state = cache.state
    for c in (cache, other, restored):
        assert c.offset == 0
        with pytest.raises(kvhip.KVHipError):
            c.attend(torch.zeros(2, 4, 1, 128, dtype=F16, device="cuda"), 0.1)
        with pytest.raises(kvhip.KVHipError):
            c.select_blocks(torch.zeros(2, 4, 1, 128, dtype=F16, device="cuda"), 1)
        fresh = O.BlockScaledCache("float16")
        fill(c, fresh, make, [1, 64])
        check_rows(c, fresh)


def test_saved_as_full_precision(tmp_path):
    """A prompt-cache file holds the rows as they are read back, under the class that the reference knows."""
    make = pair(BF16, np.random.default_rng(5))
    cache, oracle = kvhip.BlockScaledKVCache(), O.BlockScaledCache("bfloat16")
    fill(cache, oracle, make, [100])
    kvhip.save_prompt_cache(tmp_path / "c.safetensors", [cache], {"a": "b"})
    (loaded,), meta = kvhip.load_prompt_cache(tmp_path / "c.safetensors")
    assert type(loaded) is kvhip.KVCacheSimple and meta == {"a": "b"}
    for a, b in zip(loaded.state, cache.state):
        assert torch.equal(a, b)


# ---- attention ------------------------------------------------------------------------------------------------------
def exact_and_bound(q, oracle, scale, weight, add=None):
    """Attention in float64 over the rows that the cache holds, and how far the kernel's result may lie from it.

    weight [B, 1 or Hkv or Hq, L, T]: how often a key counts.  The kernel's errors, each by its own bound (u: half a step):
      - a score's float32 sum of D products (exact each: 8 and 4 bits) and its scaling: (D + 2) 2^-24 sum |q k| scale, and the
        exponent's argument and value: 2^-22 (|s - max| + 1); both relative to the weight, so e = their sum
      - a weight rounded to the cache's type: u of that type, relative
      - the sums over T keys and the joining of parts: (T + 64) 2^-24, relative to sum w |v|
      - the output's rounding: u of the type.
    So |error| <= u |o| + (u + 2 e + 2 (T + 64) 2^-24) sum w |v|  (e twice and the sums twice: numerator and denominator)."""
    B, Hq, n, D = q.shape
    k, v = oracle.keys, oracle.values
    Hkv, T = k.shape[1], k.shape[2]
    G = Hq // Hkv
    q = q.astype(np.float64)
    out, bound = np.zeros((B, Hq, n, v.shape[3])), np.zeros((B, Hq, n, v.shape[3]))
    u = (2.0 ** -11 if oracle.dtype == "float16" else 2.0 ** -8)
    for b in range(B):
        for hq in range(Hq):
            h = hq // G
            w = weight[b, {1: 0, Hkv: h}.get(weight.shape[1], hq)]
            s = q[b, hq] @ k[b, h].T * scale
            size = np.abs(q[b, hq]) @ np.abs(k[b, h]).T * abs(scale)
            if add is not None:
                s = s + add[b, hq]
                size = size + np.where(np.isfinite(add[b, hq]), np.abs(add[b, hq]), 0.0)
            s = np.where(w > 0, s, -np.inf)
            top = s.max(-1, keepdims=True)
            top = np.where(np.isfinite(top), top, 0.0)
            p = np.exp(s - top) * w
            total = p.sum(-1, keepdims=True)
            p = p / np.where(total > 0, total, 1.0)
            far = np.where(p > 0, top - s, 0.0)
            e = (D + 2) * 2.0 ** -24 * size + 2.0 ** -22 * (far + 1)
            vv = np.nan_to_num(v[b, h]) if np.isnan(v[b, h]).any() else v[b, h]
            out[b, hq] = p @ vv
            bound[b, hq] = u * np.abs(out[b, hq]) + (u + 2 * (T + 64) * 2.0 ** -24) * (p @ np.abs(vv)) + 2 * (p * e) @ np.abs(vv) + 1e-30
            bound[b, hq] += 2 * (p * e).sum(-1, keepdims=True) * (p @ np.abs(vv))
    return out, bound


def check(got, want, bound):
    got = np32(got).astype(np.float64)
    assert np.isfinite(got).all()
    worst = (np.abs(got - want) / bound).max()
    assert worst <= 1.0, f"{worst:.3g} times the bound"


def causal(T, n, pads, window=0):
    pos, col = np.arange(T - n, T)[:, None], np.arange(T)[None]
    keep = np.stack([(col <= pos) & (col >= p) & (col > pos - window if window else True) for p in pads])
    return keep[:, None].astype(np.float64)


# (query heads, kv heads, key size, value size)
LAYOUTS = [(8, 2, 128, 128), (6, 2, 64, 64), (4, 4, 96, 96), (14, 2, 256, 256), (4, 4, 192, 128), (4, 2, 50, 36)]


def held(dtype, T, layout, seed=0, B=2, rows=None):
    rng = np.random.default_rng(seed + T)
    cache, oracle = kvhip.BlockScaledKVCache(), O.BlockScaledCache(NAME[dtype])
    hq, h, dk, dv = layout
    fill(cache, oracle, pair(dtype, rng, B, h, (dk, dv)), rows or [T])
    return cache, oracle, lambda n: randn(rng, (B, hq, n, dk), dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("T,n", [(1, 1), (2, 1), (63, 1), (64, 1), (65, 1), (700, 1), (3000, 1), (2, 2), (66, 3), (300, 5), (64, 20),
                                 (200, 40), (1000, 67), (5000, 9)])
def test_attention_with_causal_masks(dtype, layout, T, n):
    cache, oracle, queries = held(dtype, T, layout)
    q, qd = queries(n)
    scale = layout[2] ** -0.5
    got = cache.attend(qd, scale, kvhip.MaskMode.causal() if n > 1 else None)
    assert kvhip.load().kvhip_last_attend_kernel() == 7
    check(got, *exact_and_bound(q, oracle, scale, causal(T, n, [0, 0])))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layout", LAYOUTS[:4])
@pytest.mark.parametrize("T,n,pads,window", [(500, 1, (0, 499), 0), (500, 3, (130, 498), 0), (500, 3, (500, 7), 0), (700, 40, (0, 690), 0),
                                             (700, 1, (0, 0), 100), (700, 40, (3, 200), 65), (300, 130, (64, 128), 0), (90, 90, (0, 90), 1)])
def test_attention_of_padded_batches_and_windows(dtype, layout, T, n, pads, window):
    cache, oracle, queries = held(dtype, T, layout, seed=1)
    q, qd = queries(n)
    scale = layout[2] ** -0.5
    mask = kvhip.MaskMode.window_mask(T - n, window, left_pad=torch.tensor(pads, device="cuda"))
    got = cache.attend(qd, scale, mask)
    check(got, *exact_and_bound(q, oracle, scale, causal(T, n, pads, window)))


@pytest.mark.parametrize("layout", [LAYOUTS[0], LAYOUTS[3]])
@pytest.mark.parametrize("n", [1, 3, 50])
def test_attention_with_lengths(layout, n):
    """Sequences that end before the cache does, one of them before its first key."""
    cache, oracle, queries = held(BF16, 400, layout, seed=6, B=3)
    rng = np.random.default_rng(n)
    q, qd = randn(rng, (3, layout[0], n, layout[2]), BF16)
    lengths = (400, 130, 0)
    mask = kvhip.MaskMode.window_mask(400 - n, 0, lengths=torch.tensor(lengths, device="cuda"))
    keep = causal(400, n, [0, 0, 0])
    for b, m in enumerate(lengths):
        keep[b, :, :, m:] = 0
    got = cache.attend(qd, 0.1, mask)
    check(got, *exact_and_bound(q, oracle, 0.1, keep))
    assert (got[2] == 0).all()


@pytest.mark.parametrize("scale", [-0.1, 0.0, 3.0])
@pytest.mark.parametrize("n", [1, 40])
def test_scales_of_any_sign(scale, n):
    cache, oracle, queries = held(BF16, 300, LAYOUTS[0], seed=7)
    q, qd = queries(n)
    check(cache.attend(qd, scale, kvhip.MaskMode.causal()), *exact_and_bound(q, oracle, scale, causal(300, n, [0, 0])))
    blocks = cache.select_blocks(qd, 5)
    want = O.listed_keep(blocks.cpu().numpy(), 300, [0, 0])
    check(cache.attend_blocks(qd, blocks, scale), *exact_and_bound(q, oracle, scale, want))


def test_arrays_that_start_anywhere():
    """Keys, values, queries and outputs aligned as their elements are."""
    gen = torch.Generator(device="cuda").manual_seed(2)

    def at(shape, off):
        n = int(np.prod(shape))
        flat = torch.randn(n + off, generator=gen, device="cuda").to(BF16)
        return flat[off:].view(shape)

    k, v, q = at((2, 2, 130, 128), 1), at((2, 2, 130, 128), 3), at((2, 8, 40, 128), 5)
    out = torch.zeros(2 * 8 * 40 * 128 + 1, dtype=BF16, device="cuda")[1:].view(2, 8, 40, 128)
    a, b = kvhip.BlockScaledKVCache(), kvhip.BlockScaledKVCache()
    a.update(k, v, fetch=False)
    b.update(k.clone(), v.clone(), fetch=False)
    for x, y in zip(a.fetch(), b.fetch()):
        assert torch.equal(x, y)
    a.attend(q, 0.1, kvhip.MaskMode.causal(), out=out)
    assert torch.equal(out, b.attend(q.clone(), 0.1, kvhip.MaskMode.causal()))
    chosen = a.select_blocks(q, 2)
    assert torch.equal(chosen, b.select_blocks(q.clone(), 2))
    one = at((2, 8, 1, 128), 7)
    k1, v1 = at((2, 2, 1, 128), 1), at((2, 2, 1, 128), 1)
    assert torch.equal(a.update_attend(one, k1, v1, 0.1), b.update_attend(one.clone(), k1.clone(), v1.clone(), 0.1))


def test_speculative_rounds_write_through_and_trim():
    """An append-only leaf of a round: drafts are written, the rejected ones trimmed, and accepted ones as if alone."""
    make = pair(BF16, np.random.default_rng(12))
    cache, oracle = kvhip.BlockScaledKVCache(), O.BlockScaledCache("bfloat16")
    fill(cache, oracle, make, [61])
    for accepted in (2, 0, 4, 1):
        drafts = [make(1) for _ in range(4)]
        for (k, kd), (v, vd) in drafts:
            cache.update(kd, vd, fetch=False)
            oracle.update(k, v)
        assert cache.trim(4 - accepted) == 4 - accepted
        if accepted < 4:
            oracle.trim(4 - accepted)
    check_rows(cache, oracle)
    assert kvhip.can_trim_prompt_cache([cache]) and cache.is_trimmable_after(1000)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layout", [LAYOUTS[0], LAYOUTS[3], LAYOUTS[5]])
@pytest.mark.parametrize("T,n", [(70, 1), (300, 3), (513, 20)])
@pytest.mark.parametrize("kind", ["bool", "f32", "own", "lowest", "empty"])
def test_attention_with_array_masks(dtype, layout, T, n, kind):
    cache, oracle, queries = held(dtype, T, layout, seed=2)
    q, qd = queries(n)
    B, hq = q.shape[:2]
    scale = layout[2] ** -0.5
    gen = torch.Generator(device="cuda").manual_seed(T + n)
    keep = torch.rand(B, hq if kind == "bool" else 1, n, T, generator=gen, device="cuda") < 0.6
    keep[..., 0] = True
    add = None
    if kind == "empty":
        keep[0, :, 0] = False
        keep[1, :, n - 1, 5:] = False
    if kind in ("bool", "empty"):
        mask = keep
    else:
        t = {"f32": torch.float32, "own": dtype, "lowest": dtype}[kind]
        mask = torch.randn(B, 1, n, T, generator=gen, device="cuda").to(t)
        if kind == "lowest":
            mask = torch.where(keep, mask, torch.full_like(mask, torch.finfo(t).min))
            mask[0, 0, 0] = torch.finfo(t).min  # (equal weights: the score is lost beside it)
        else:
            mask = torch.where(keep, mask, torch.full_like(mask, -INF))
            mask[1, 0, n - 1, 3:] = -INF
            keep[1, 0, n - 1, 3:] = False
        add = np.broadcast_to(mask.double().cpu().numpy(), (B, hq, n, T))
    weight = np.broadcast_to(keep.double().cpu().numpy(), (B, hq, n, T))
    if kind == "lowest":
        weight = np.ones((B, hq, n, T))
    got = cache.attend(qd, scale, kvhip.MaskMode.from_array(mask))
    if kind == "lowest":
        # what float32 leaves of a score beside the lowest value
        h = np.repeat(oracle.keys, hq // layout[1], axis=1)
        s = (np.einsum("bhld,bhtd->bhlt", q.astype(np.float64), h) * scale).astype(np.float32) + add.astype(np.float32)
        want, bound = exact_and_bound(q * 0, oracle, scale, weight, s.astype(np.float64))
        e = (layout[2] + 6) * 2.0 ** -24 * np.einsum("bhld,bhtd->bhlt", np.abs(q.astype(np.float64)), np.abs(h)).max() * scale
        ones = np.repeat(np.abs(oracle.values), hq // layout[1], axis=1).max(2, keepdims=True)
        far = 2.0 ** -22 * (np.where(s > -1e30, np.abs(s), 0).max() + 1)
        _, plain = exact_and_bound(q * 0, oracle, scale, weight, np.where(add > -1e4, s, -INF).astype(np.float64))
        row = (add > -1e4).any(-1, keepdims=True)
        check(got, want, np.where(row, plain, bound * 0 + 2.0 ** -7 * ones) + 4 * (e + far) * ones)
        return
    check(got, *exact_and_bound(q, oracle, scale, weight, add))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,n", [(75, 1), (140, 4), (400, 30), (256, 70)])
def test_values_that_are_no_numbers_in_masked_places(dtype, T, n):
    """NaN and infinities in paddings, in later tokens of the chunk and in rows trimmed away reach no row that does not see
    them, and every row that does."""
    layout = LAYOUTS[0]
    rng = np.random.default_rng(T)
    make = pair(dtype, rng, 2, 2, (128, 128))
    cache, oracle = kvhip.BlockScaledKVCache(), O.BlockScaledCache(NAME[dtype])
    (k, kd), (v, vd) = make(T + 9)
    bad = {(0, 3): NAN, (0, 10): INF, (1, 2): -INF, (0, T - 1): NAN}
    for (b, t), x in bad.items():
        v[b, 0, t, 5], vd[b, 0, t, 5] = x, x
    for x in (k, v, kd, vd):
        x[:, :, T:] = NAN if x is k or x is v or x is kd else INF
    k[0, 1, 3, 2], kd[0, 1, 3, 2] = NAN, NAN
    cache.update(kd, vd, fetch=False)
    oracle.update(k, v)
    cache.trim(9)
    oracle.trim(9)
    q, qd = randn(rng, (2, 8, n, 128), dtype)
    scale = 128 ** -0.5
    pads = (11, 3)
    got = cache.attend(qd, scale, kvhip.MaskMode.window_mask(T - n, 0, left_pad=torch.tensor(pads, device="cuda")))
    oracle.keys = np.nan_to_num(oracle.keys)
    want, bound = exact_and_bound(q, oracle, scale, causal(T, n, pads))
    seen = torch.zeros_like(got, dtype=torch.bool)
    seen[0, :4, n - 1, 5] = True  # (the last token of the first sequence, kv head 0, sees the NaN at T - 1)
    assert torch.isnan(got[seen]).all()
    check(got.masked_fill(seen, 0), np.where(seen.cpu().numpy(), 0, want), bound)
    # without the paddings every row of kv head 0 sees them, and kv head 1 of the first sequence has a key that is none
    got = cache.attend(qd, scale, kvhip.MaskMode.causal())
    assert torch.isnan(got[0, :4, :, 5]).all() and torch.isnan(got[1, :4, :, 5]).all() and torch.isnan(got[0, 4:]).all()
    assert torch.isfinite(got[1, 4:]).all() and torch.isfinite(got[:, :4, :n - 1, 6:]).all()


@pytest.mark.parametrize("dtype,layout", [(F16, LAYOUTS[0]), (BF16, LAYOUTS[1]), (BF16, LAYOUTS[5])])
def test_a_conversation(dtype, layout):
    """A prompt, tokens one by one over block ends, a rejected draft, a chunk, as the functions of the framework run them:
    each call against the oracle, and the same as update and attention apart."""
    hq, h, dk, dv = layout
    rng = np.random.default_rng(21)
    make = pair(dtype, rng, 2, h, (dk, dv))
    cache, apart, oracle = kvhip.BlockScaledKVCache(), kvhip.BlockScaledKVCache(), O.BlockScaledCache(NAME[dtype])
    scale = dk ** -0.5
    for n in [100] + [1] * 30 + [4, -3] + [1] * 3 + [90, -40] + [1] * 20:
        if n < 0:
            assert kvhip.trim_prompt_cache([cache, apart], -n) == -n
            oracle.trim(-n)
            continue
        (k, kd), (v, vd) = make(n)
        q, qd = randn(rng, (2, hq, n, dk), dtype)
        got = kvhip.attention_with_cache_update(qd, kd, vd, cache, scale, kvhip.create_attention_mask(n, cache))
        mask = kvhip.create_attention_mask(n, apart)
        apart.update(kd, vd, fetch=False)
        assert torch.equal(got, apart.attend(qd, scale, mask))
        oracle.update(k, v)
        check(got, *exact_and_bound(q, oracle, scale, causal(oracle.offset, n, [0, 0])))
    check_rows(cache, oracle)


def test_rotary_steps():
    """Keys turned on their way in are what kvhip_rope_apply makes of them."""
    rng = np.random.default_rng(4)
    rope = kvhip.RoPE(128, base=10000.0)
    a, b = kvhip.BlockScaledKVCache(), kvhip.BlockScaledKVCache()
    make = pair(BF16, rng)
    for n in (70, 1, 1, 60, 1):
        (_, k), (_, v) = make(n)
        _, q = randn(rng, (2, 8, n, 128), BF16)
        mask = kvhip.create_attention_mask(n, a)
        got = kvhip.attention_with_rope_and_cache_update(rope, q, k, v, a, 0.1, mask)
        qr, kr = (kvhip.apply_rotary_position(rope, x, b) for x in (q, k))
        assert torch.equal(got, b.update_attend(qr, kr, v, 0.1, mask))
    for x, y in zip(a.fetch(), b.fetch()):
        assert torch.equal(x, y)


def test_static_scratch_and_streams():
    cache, oracle, queries = held(BF16, 2500, LAYOUTS[0])
    q, qd = queries(3)
    want = cache.attend(qd, 0.1, kvhip.MaskMode.causal())
    got = cache.attend(qd, 0.1, kvhip.MaskMode.causal(), static_scratch=True)
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = cache.attend(qd, 0.1, kvhip.MaskMode.causal())
    side.synchronize()
    assert torch.equal(got, want)
    q, qd = queries(1100)  # partials that would not fit: fewer parts
    check(cache.attend(qd, 0.1, kvhip.MaskMode.causal(), static_scratch=True), *exact_and_bound(q, oracle, 0.1, causal(2500, 1100, [0, 0])))


def close_to_float64(got, q, k, v, scale, keep):
    """`got` [..., n, Dv] of one kv head against float64 over its rows as read back, within what the roundings allow: the output's
    and the weights' half steps, relative to the output and to the weights' sum over |v|, and as much again for the sums."""
    s = (q.double() @ k.double().T * scale).masked_fill(~keep, -INF)
    p = torch.softmax(s, -1)
    want, size = p @ v.double(), p @ v.double().abs()
    u = torch.finfo(got.dtype).eps / 2
    assert ((got.double() - want).abs() <= u * want.abs() + 2 * u * size).all()


@pytest.mark.parametrize("B,H,G,D,T,n", [(32, 8, 1, 64, 38500, 1), (8, 8, 4, 128, 20100, 64), (16, 16, 8, 64, 17000, 4)])
def test_walks_of_many_blocks(B, H, G, D, T, n):
    """More than 64 blocks to a wavefront: their addresses are looked up in turns."""
    gen = torch.Generator(device="cuda").manual_seed(T)
    cache = kvhip.BlockScaledKVCache()
    cache.reserve(B, H, D, D, BF16, T)
    for at in range(0, T, 4096):
        m = min(4096, T - at)
        k, v = (torch.randn(B, H, m, D, generator=gen, device="cuda").to(BF16) for _ in range(2))
        cache.update(k, v, fetch=False)
    q = torch.randn(B, H * G, n, D, generator=gen, device="cuda").to(BF16)
    out = cache.attend(q, 0.2, kvhip.MaskMode.causal())
    k, v = cache.fetch()
    keep = torch.arange(T, device="cuda") <= torch.arange(T - n, T, device="cuda")[:, None]
    for b, h in ((0, 0), (B - 1, H - 1), (B // 2, 3)):
        close_to_float64(out[b, h * G:(h + 1) * G].flatten(0, 1), q[b, h * G:(h + 1) * G].flatten(0, 1), k[b, h], v[b, h], 0.2, keep.repeat(G, 1))


def test_offsets_beyond_32_bits():
    """Codes of keys past 4 GiB: rows at the far end, whole and listed, against a cache of nothing else."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    step, D = 1 << 20, 256
    k, v = (torch.randn(1, 1, step, D, generator=gen, device="cuda").to(BF16) for _ in range(2))
    cache, near = kvhip.BlockScaledKVCache(), kvhip.BlockScaledKVCache()
    cache.reserve(1, 1, D, D, BF16, 17 * step)
    for _ in range(16):
        cache.update(k, v, fetch=False)
    last = [x[:, :, :5000] * 0.5 for x in (k, v)]
    cache.update(*last, fetch=False)
    near.update(*last, fetch=False)
    T = 16 * step + 5000
    assert cache.offset == T and T * D > 1 << 32
    q = torch.randn(1, 4, 20, D, generator=gen, device="cuda").to(BF16)
    keep = torch.arange(5000, device="cuda") <= torch.arange(4980, 5000, device="cuda")[:, None]
    nk, nv = (x[0, 0] for x in near.fetch())
    far = torch.tensor([T - 5000], device="cuda")
    out = cache.attend(q, 0.1, kvhip.MaskMode.window_mask(T - 20, 0, left_pad=far))
    close_to_float64(out[0].flatten(0, 1), q[0].flatten(0, 1), nk, nv, 0.1, keep.repeat(4, 1))
    blocks = torch.arange((T - 5000) // 64, (T + 63) // 64, dtype=torch.int32, device="cuda").expand(1, 1, 20, -1).contiguous()
    out = cache.attend_blocks(q, blocks, 0.1, far)
    close_to_float64(out[0].flatten(0, 1), q[0].flatten(0, 1), nk, nv, 0.1, keep.repeat(4, 1))
    del cache


# ---- choosing blocks ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layout", LAYOUTS + [(5, 5, 64, 64), (40, 2, 128, 128), (3, 1, 96, 96)])
@pytest.mark.parametrize("T,n,count,first,recent,pads", [(1, 1, 3, 1, 1, (0, 0)), (64, 1, 2, 0, 1, (0, 0)), (1000, 1, 5, 1, 2, (0, 300)),
                                                        (1000, 3, 16, 0, 1, (999, 1000)), (1003, 7, 3, 1, 1, (64, 130)),
                                                        (1920, 1, 20, 2, 3, (0, 63)), (650, 70, 4, 0, 2, (0, 640))])
def test_blocks_are_chosen_by_the_definition(dtype, layout, T, n, count, first, recent, pads):
    cache, oracle, queries = held(dtype, T, layout, seed=3)
    q, qd = queries(n)
    got = cache.select_blocks(qd, count, first, recent, torch.tensor(pads, device="cuda"))
    assert np.array_equal(got.cpu().numpy(), O.select(q, oracle, count, first, recent, pads))


@pytest.mark.parametrize("T,n", [(1300, 1), (1300, 9), (12000, 1)])
@pytest.mark.parametrize("keys_at,queries_at", [(126, 126), (-100, -100), (126, -120), (-60, 100), (40, 100)])
def test_bounds_beyond_float32(T, n, keys_at, queries_at):
    """Blocks of sizes from 2^(keys_at - 24) on against queries about 2^queries_at: bounds beyond what a float holds, either side."""
    rng = np.random.default_rng(T + n)
    size = 2.0 ** np.repeat(keys_at - rng.integers(0, 25, (2, 2, (T + 63) // 64, 1)), 64, 2)[:, :, :T]

    def drawn(x):
        t = torch.from_numpy(x).to(BF16)
        return t.double().numpy(), t.cuda()

    k, kd = drawn(rng.uniform(-1, 1, (2, 2, T, 128)) * size)
    q, qd = drawn(rng.uniform(-1, 1, (2, 8, n, 128)) * 2.0 ** queries_at)
    cache, oracle = kvhip.BlockScaledKVCache(), O.BlockScaledCache("bfloat16")
    cache.update(kd, kd, fetch=False)
    oracle.update(k, k)
    got = cache.select_blocks(qd, 9, 0, 1)
    assert np.array_equal(got.cpu().numpy(), O.select(q, oracle, 9, 0, 1, (0, 0)))


@pytest.mark.parametrize("layout", [(8, 2, 128, 128), (40, 1, 64, 64), (3, 1, 96, 96), (2, 1, 256, 256), (70, 1, 50, 36)])
@pytest.mark.parametrize("n,count,first,recent,pads", [(1, 40, 1, 2, (0, 0)), (1, 3, 1, 2, (5000, 0)), (3, 17, 0, 1, (100, 17100)), (19, 300, 3, 4, (0, 64))])
def test_blocks_of_long_caches(layout, n, count, first, recent, pads):
    """More blocks than one workgroup takes in: bounds and choice in launches of their own."""
    cache, oracle, queries = held(BF16, 17100, layout, seed=4)
    q, qd = queries(n)
    got = cache.select_blocks(qd, count, first, recent, torch.tensor(pads, device="cuda"))
    assert np.array_equal(got.cpu().numpy(), O.select(q, oracle, count, first, recent, pads))


@pytest.mark.parametrize("H,G,T,n,count", [(1, 4, 1_200_000, 1, 50), (1, 4, 66_000, 2100, 33), (2, 16, 140_000, 3, 64)])
def test_blocks_of_very_long_caches(H, G, T, n, count):
    """Keys of the choice beyond 64 KiB of LDS, in either form of the launch."""
    gen = torch.Generator(device="cuda").manual_seed(T)
    keys = torch.randn(1, H, T, 64, generator=gen, device="cuda").to(F16)
    cache = kvhip.BlockScaledKVCache()
    cache.update(keys, keys, fetch=False)
    q = torch.randn(1, H * G, n, 64, generator=gen, device="cuda").to(F16)
    got = cache.select_blocks(q, count, 1, 2)
    whole = T // 64
    x = keys[0, :, :whole * 64].double().unflatten(1, (whole, 64))
    read = cache.fetch()[0][0, :, :whole * 64].double().unflatten(1, (whole, 64))
    m, e = torch.frexp(x.abs().amax((2, 3)))
    two_to = lambda n: ((n.long() + 1023) << 52).view(torch.float64)  # noqa: E731 (exactly)
    unit = two_to(e - 9 + (m > 0.875).to(e.dtype) + 2)
    units = torch.round(read / unit[..., None, None])
    hi, lo = units.amax(2), units.amin(2)
    rows = q[0].double().unflatten(0, (H, G))
    m, f = torch.frexp(rows.abs().amax(-1))
    grid = two_to(f - 7 + (m > 127 / 128).to(f.dtype))[..., None]
    whole_q = torch.round(rows / grid)
    at = torch.arange(T - n, T, device="cuda")[:, None] // 64
    index = torch.arange((T + 63) // 64, device="cuda")
    for h in range(H):
        bound = ((whole_q[h].clamp(min=0) @ hi[h].T + whole_q[h].clamp(max=0) @ lo[h].T) * grid[h] * unit[h]).amax(0)
        rank = torch.full((n, len(index)), -INF, dtype=torch.float64, device="cuda")
        rank[:, :whole] = bound
        rank = rank.masked_fill((index < 1) | (index > at - 2), INF).masked_fill(index > at, -INF)
        want = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :count].sort(-1).values
        off = (got[0, h].long() != want).any(-1).nonzero()
        assert len(off) == 0, f"{len(off)} tokens, the first {int(off[0])}: {got[0, h, off[0]].tolist()} for {want[off[0]].tolist()}"


def test_equal_bounds_of_long_caches():
    one = torch.ones(1, 1, 64, 64, device="cuda").to(BF16)
    k = one.repeat(1, 1, 400, 1)
    k[:, :, 64 * 333:64 * 334] *= 2
    cache = kvhip.BlockScaledKVCache()
    cache.update(k, k, fetch=False)
    got = cache.select_blocks(one[:, :, :1], 300, 0, 1)[0, 0, 0].cpu()
    assert (got == torch.tensor(list(range(298)) + [333, 399])).all()
    assert (cache.select_blocks(0 * one[:, :, :1], 300, 0, 1)[0, 0, 0].cpu() == torch.tensor(list(range(299)) + [399])).all()


def test_equal_bounds_take_the_lower_block():
    gen = torch.Generator(device="cuda").manual_seed(1)
    one = torch.randn(1, 2, 64, 64, generator=gen, device="cuda").to(BF16)
    k = one.repeat(1, 1, 40, 1)
    k[:, :, 64 * 17:64 * 18] *= 2
    cache = kvhip.BlockScaledKVCache()
    cache.update(k, k, fetch=False)
    q = torch.randn(1, 8, 1, 64, generator=gen, device="cuda").to(BF16)
    got = cache.select_blocks(q, 7, 0, 1)
    assert (got[0, :, 0].cpu() == torch.tensor([0, 1, 2, 3, 4, 17, 39])).all()
    assert (cache.select_blocks(q * 0, 4, 0, 1)[0, :, 0].cpu() == torch.tensor([0, 1, 2, 39])).all()
    assert (cache.select_blocks(q * NAN, 4, 0, 1)[0, :, 0].cpu() == torch.tensor([0, 1, 2, 39])).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layout", LAYOUTS + [(40, 2, 128, 128)])
@pytest.mark.parametrize("T,n,count,pads", [(1, 1, 1, (0, 0)), (900, 1, 6, (0, 200)), (900, 1, 40, (0, 899)), (901, 5, 7, (901, 70)), (640, 40, 3, (0, 0))])
def test_attention_over_chosen_blocks(dtype, layout, T, n, count, pads):
    hq, h, dk, dv = layout
    rng = np.random.default_rng(T)
    make = pair(dtype, rng, 2, h, (dk, dv))
    cache, oracle = kvhip.BlockScaledKVCache(), O.BlockScaledCache(NAME[dtype])
    if T > n:
        fill(cache, oracle, make, [T - n])
    (k, kd), (v, vd) = make(n)
    q, qd = randn(rng, (2, hq, n, dk), dtype)
    pad = torch.tensor(pads, device="cuda")
    scale = dk ** -0.5
    got, blocks = cache.update_attend_blocks(qd, kd, vd, scale, count, first=0, recent=1, left_pad=pad)
    assert kvhip.load().kvhip_last_attend_kernel() == 8
    oracle.update(k, v)
    want = O.select(q, oracle, count, 0, 1, pads)
    assert np.array_equal(blocks.cpu().numpy(), want)
    check(got, *exact_and_bound(q, oracle, scale, O.listed_keep(want, T, pads)))
    assert torch.equal(cache.attend_blocks(qd, blocks, scale, pad), got)
    assert torch.equal(cache.select_blocks(qd, count, 0, 1, pad), blocks)
    check_rows(cache, oracle)


@pytest.mark.parametrize("layout", LAYOUTS + [(40, 2, 128, 128)])
@pytest.mark.parametrize("T,n,count,first,recent,pads", [(9000, 1, 20, 1, 2, (0, 0)), (9001, 3, 7, 0, 1, (8999, 300)), (12000, 1, 64, 2, 3, (11999, 64)),
                                                        (9000, 2, 200, 1, 1, (0, 0)), (30000, 1, 1100, 1, 1, (0, 9000))])
def test_steps_that_choose_their_blocks(layout, T, n, count, first, recent, pads):
    """One call on a long cache -- the attention makes the choice itself where that is the shorter -- against the choice and the
    attention apart, and against float64."""
    hq, h, dk, dv = layout
    rng = np.random.default_rng(T)
    gen = torch.Generator(device="cuda").manual_seed(T)
    k, v = (torch.randn(2, h, T - n, d, generator=gen, device="cuda").to(BF16) for d in (dk, dv))
    cache = kvhip.BlockScaledKVCache()
    cache.update(k, v, fetch=False)
    apart = cache.copy()
    q, k, v = (torch.randn(2, x, n, d, generator=gen, device="cuda").to(BF16) for x, d in ((hq, dk), (h, dk), (h, dv)))
    pad = torch.tensor(pads, device="cuda")
    scale = dk ** -0.5
    got, blocks = cache.update_attend_blocks(q, k, v, scale, count, first, recent, pad)
    apart.update(k, v, fetch=False)
    assert torch.equal(blocks, apart.select_blocks(q, count, first, recent, pad))
    assert torch.equal(got, apart.attend_blocks(q, blocks, scale, pad))
    keys, values = cache.fetch()
    weight = torch.from_numpy(O.listed_keep(blocks[:, :1].cpu().numpy(), T, pads)).cuda()
    G = hq // h
    for b in range(2):
        for t in range(n):
            keep = weight[b, 0, t] > 0
            if keep.any():
                close_to_float64(got[b, :G, t], q[b, :G, t], keys[b, 0], values[b, 0], scale, keep[None])
            else:
                assert (got[b, :G, t] == 0).all()


@pytest.mark.parametrize("n", [1, 4])
def test_blocks_listed_again_count_again(n):
    """Behind a lower entry a block counts anew, the unfinished one too, whichever wavefront meets it."""
    cache, oracle, queries = held(BF16, 700, LAYOUTS[0])
    q, qd = queries(n)
    for entries in ([10, 3, 10], [10, -1, 10, -1, 10, -1, 10, -1, 10, 3, 4, 10], [4, 10] * 150 + [-1, 2], [10, 0, 10, 0, 0, 10, 10, 5, 5]):
        blocks = torch.tensor(entries, dtype=torch.int32, device="cuda").expand(2, 2, n, -1).contiguous()
        got = cache.attend_blocks(qd, blocks, 0.1)
        check(got, *exact_and_bound(q, oracle, 0.1, O.listed_keep(blocks.cpu().numpy(), 700, (0, 0))))


def test_lists_of_any_content():
    """Entries outside what the token sees, repeated and descending ones are passed over; nothing listed: zeros."""
    cache, oracle, queries = held(BF16, 700, LAYOUTS[0])
    q, qd = queries(4)
    lists = [[-1, -1, -1, -1, -1], [10, 10, 10, 10, 10], [3, 2, 5, 1, 0], [-7, 4, 2 ** 31 - 1, 11, 12]]
    blocks = torch.tensor(lists, dtype=torch.int32, device="cuda").expand(2, 2, 4, 5).contiguous()
    blocks[1, 1, 0] = torch.tensor([0, 4, 6, 8, 10])
    pads = (0, 75)
    got = cache.attend_blocks(qd, blocks, 0.1, torch.tensor(pads, device="cuda"))
    check(got, *exact_and_bound(q, oracle, 0.1, O.listed_keep(blocks.cpu().numpy(), 700, pads)))
    assert (got[0, :, 0] == 0).all()


def test_every_block_listed_is_the_whole_attention():
    cache, oracle, queries = held(F16, 1000, LAYOUTS[0])
    q, qd = queries(9)
    out = kvhip.sparse_attention_with_cache_update
    blocks = cache.select_blocks(qd, 16)
    check(cache.attend_blocks(qd, blocks, 0.1), *exact_and_bound(q, oracle, 0.1, causal(1000, 9, [0, 0])))
    (k, kd), (v, vd) = pair(F16, np.random.default_rng(0))(1)
    oracle.update(k, v)
    check(out(qd[:, :, :1].contiguous(), kd, vd, cache, 0.1, 16), *exact_and_bound(q[:, :, :1], oracle, 0.1, causal(1001, 1, [0, 0])))


def test_captured_steps_replay():
    """A captured step (the choice, both attentions) replayed with eager work in between."""
    cache, oracle, queries = held(BF16, 5000, LAYOUTS[0])
    _, q = queries(1)
    out = torch.empty(2, 8, 1, 128, dtype=BF16, device="cuda")
    cache.attend(q, 0.1, out=out)
    chosen = cache.attend_blocks(q, cache.select_blocks(q, 9), 0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        blocks = cache.select_blocks(q, 9)
        sparse = cache.attend_blocks(q, blocks, 0.1)
        cache.attend(q, 0.1, out=out)
    for i in range(4):
        fresh = torch.randn(2, 8, 1, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)).to(BF16)
        q.copy_(fresh)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got, got_sparse = out.clone(), sparse.clone()
        assert torch.equal(got, cache.attend(fresh, 0.1))
        assert torch.equal(got_sparse, cache.attend_blocks(fresh, cache.select_blocks(fresh, 9), 0.1))
    assert torch.isfinite(chosen).all()


@pytest.mark.parametrize("held_rows", [9000, 9023])
def test_captured_steps_that_write(held_rows):
    """A captured step writes its row and attends, replay after replay: the last inputs' row is what the cache holds.  The second
    length ends its block with the row (63 rows of it held before), which is a launch of its own."""
    cache, oracle, queries = held(BF16, held_rows, LAYOUTS[0], seed=9)
    other = cache.copy()
    gen = torch.Generator(device="cuda").manual_seed(3)

    def fresh():
        return [torch.randn(2, h, 1, 128, generator=gen, device="cuda").to(BF16) for h in (8, 2, 2)]

    q, k, v = fresh()
    for sparse in (False, True):
        def step(c):
            if sparse:
                return c.update_attend_blocks(q, k, v, 0.1, 20)
            return c.update_attend(q, k, v, 0.1)

        step(cache)  # (scratch is there from here on)
        cache.trim(1)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(cache)
        for _ in range(3):
            for dst, src in zip((q, k, v), fresh()):
                dst.copy_(src)
            graph.replay()
            torch.cuda.synchronize()
            want = step(other)
            for a, b in zip(got if sparse else [got], want if sparse else [want]):
                assert torch.equal(a, b)
            for a, b in zip(cache.fetch(), other.fetch()):
                assert torch.equal(a, b)
            other.trim(1)
        cache.trim(1)


# ---- refusals -------------------------------------------------------------------------------------------------------
def test_a_refused_first_call_leaves_the_cache_open():
    cache = kvhip.BlockScaledKVCache()
    q, k = (torch.randn(1, h, 1, 128, device="cuda").to(BF16) for h in (4, 2))
    for bad in ({"count": 0}, {"count": 2, "first": 2}, {"count": 2, "first": -1}):
        with pytest.raises(kvhip.KVHipError):
            cache.update_attend_blocks(q, k, k, 0.1, **bad)
    assert cache.offset == 0
    q, k = (torch.randn(3, h, 2, 64, device="cuda").to(F16) for h in (6, 3))
    cache.update_attend_blocks(q, k, k, 0.1, 2)
    assert cache.offset == 2 and torch.equal(cache.fetch()[0], k)


def test_refusals():
    cache, oracle, queries = held(BF16, 200, LAYOUTS[0])
    _, q = queries(2)
    blocks = cache.select_blocks(q, 3)

    def refused(status, call, *args, **kw):
        with pytest.raises(kvhip.KVHipError) as e:
            call(*args, **kw)
        assert e.value.status == status

    k = torch.zeros(2, 2, 1, 128, dtype=BF16, device="cuda")
    refused(-2, cache.select_blocks, q, 0)
    assert kvhip.load().kvhip_cache_attend_blocks(cache._h, q.data_ptr(), 2, 8, 2, 128, 0.1, blocks.data_ptr(), (1 << 20) + 1, None, q.data_ptr(), None) == -2
    refused(-2, cache.select_blocks, q, 3, first=3, recent=1)
    refused(-2, cache.select_blocks, q, 3, first=-1)
    refused(-2, cache.select_blocks, q, 3, recent=0)
    refused(-2, cache.select_blocks, q[:, :7].contiguous(), 3)
    refused(-2, cache.select_blocks, queries(201)[1], 3)
    refused(-2, cache.attend_blocks, queries(201)[1], blocks[:, :, :1].expand(2, 2, 201, 3).contiguous(), 0.1)
    refused(-3, kvhip.BlockScaledKVCache().update, k.float(), k.float())
    refused(-3, kvhip.BlockScaledKVCache().update, k.repeat(1, 1, 1, 3), k)
    refused(-4, kvhip.BlockScaledKVCache().select_blocks, q, 3)
    refused(-2, cache.update_attend_blocks, q[:, :, :1].contiguous(), k, k, 0.1, 2, first=2)
    refused(-2, cache.update, k[:1], k[:1])
    assert cache.offset == 200
    with pytest.raises(ValueError):
        cache.attend_blocks(q, blocks.long(), 0.1)
    with pytest.raises(ValueError):
        cache.attend_blocks(q, blocks[:, :1], 0.1)
    with pytest.raises(ValueError):
        cache.select_blocks(q, 3, left_pad=torch.zeros(3, device="cuda"))
    with pytest.raises(ValueError):
        cache.update_attend_blocks(q, k, k, 0.1, 3)
    with pytest.raises(TypeError):
        cache.select_blocks(q.half(), 3)
    with pytest.raises(TypeError):
        cache.to_quantized()
    lib, simple = kvhip.load(), kvhip.KVCacheSimple()
    simple.update(k, k, fetch=False)
    assert lib.kvhip_cache_select_blocks(simple._h, q.data_ptr(), 2, 8, 1, 128, 3, 1, 1, None, blocks.data_ptr(), None) == L.OK - 2
    check_rows(cache, oracle)
