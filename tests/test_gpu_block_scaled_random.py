"""Block-scaled caches at drawn head layouts, lengths and masks: whole attention and attention over chosen and listed blocks."""
import numpy as np
import pytest
import torch

import kvhip
from oracle import block_scaled as O
from test_gpu_block_scaled import causal, check, check_rows, exact_and_bound, fill, pair
from util import NAME, randn

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def drawn(rng):
    sizes = [(64, 64), (96, 96), (128, 128), (256, 256), (192, 128), (80, 80), (50, 36), (33, 200), (1, 1), (8, 130), (191, 128)]
    dk, dv = sizes[rng.integers(len(sizes))]
    h = int(rng.integers(1, 4))
    G = int(rng.choice([1, 2, 3, 4, 5, 7, 8, 15, 16, 17, 32, 33, 40, 71]))
    B = int(rng.integers(1, 4))
    T = int(np.exp(rng.uniform(0, np.log(1500))))
    n = int(min(T, np.exp(rng.uniform(0, np.log(60))) if rng.random() < 0.7 else 1))
    return B, h, G, dk, dv, max(T, 1), max(n, 1)


@pytest.mark.parametrize("seed", range(40))
def test_drawn_calls(seed):
    rng = np.random.default_rng(1000 + seed)
    dtype = (F16, BF16)[seed % 2]
    B, h, G, dk, dv, T, n = drawn(rng)
    cache, oracle = kvhip.BlockScaledKVCache(), O.BlockScaledCache(NAME[dtype])
    make = pair(dtype, rng, B, h, (dk, dv))
    lengths = []
    while sum(lengths) < T - n:
        lengths.append(int(rng.integers(1, T - n - sum(lengths) + 1)))
    fill(cache, oracle, make, lengths)
    (k, kd), (v, vd) = make(n)
    q, qd = randn(rng, (B, h * G, n, dk), dtype)
    scale = float(rng.choice([dk ** -0.5, -0.05, 0.3]))
    pads = [int(rng.integers(0, T + 1)) if rng.random() < 0.5 else 0 for _ in range(B)]
    window = int(rng.integers(1, T + 1)) if rng.random() < 0.3 else 0
    if n == 1 and rng.random() < 0.6:
        got = cache.update_attend(qd, kd, vd, scale)
        oracle.update(k, v)
        check(got, *exact_and_bound(q, oracle, scale, np.ones((B, 1, 1, T))))
    else:
        mask = kvhip.MaskMode.window_mask(T - n, window, left_pad=torch.tensor(pads, device="cuda"))
        got = cache.update_attend(qd, kd, vd, scale, mask)
        oracle.update(k, v)
        check(got, *exact_and_bound(q, oracle, scale, causal(T, n, pads, window)))
    check_rows(cache, oracle)
    check(cache.attend(qd, scale, kvhip.MaskMode.causal()), *exact_and_bound(q, oracle, scale, causal(T, n, [0] * B)))
    keep = torch.from_numpy(rng.random((B, h * G if rng.random() < 0.5 else 1, n, T)) < 0.5)
    weight = np.broadcast_to(keep.double().numpy(), (B, h * G, n, T))
    check(cache.attend(qd, scale, kvhip.MaskMode.from_array(keep.cuda())), *exact_and_bound(q, oracle, scale, weight))
    count = int(rng.integers(1, (T + 63) // 64 + 3))
    first = int(rng.integers(0, count))
    recent = int(rng.integers(1, count - first + 1))
    pad = torch.tensor(pads, device="cuda")
    blocks = cache.select_blocks(qd, count, first, recent, pad)
    assert np.array_equal(blocks.cpu().numpy(), O.select(q, oracle, count, first, recent, pads))
    check(cache.attend_blocks(qd, blocks, scale, pad), *exact_and_bound(q, oracle, scale, O.listed_keep(blocks.cpu().numpy(), T, pads)))
    any_list = rng.integers(-1, (T + 63) // 64 + 1, (B, h, n, 7)).astype(np.int32)
    got = cache.attend_blocks(qd, torch.from_numpy(any_list).cuda(), scale, pad)
    check(got, *exact_and_bound(q, oracle, scale, O.listed_keep(any_list, T, pads)))
    # the same rows once more through the call that chooses as it goes
    assert cache.trim(n) == n
    oracle.trim(n)
    got, chosen = cache.update_attend_blocks(qd, kd, vd, scale, count, first, recent, pad)
    oracle.update(k, v)
    assert torch.equal(chosen, blocks)
    check(got, *exact_and_bound(q, oracle, scale, O.listed_keep(blocks.cpu().numpy(), T, pads)))
    check_rows(cache, oracle)


@pytest.mark.parametrize("n", [5, 40, 200])
def test_more_queries_than_keys(n):
    """Tokens in front of the first key see nothing: zeros."""
    rng = np.random.default_rng(n)
    cache, oracle = kvhip.BlockScaledKVCache(), O.BlockScaledCache("bfloat16")
    fill(cache, oracle, pair(BF16, rng), [70])
    q, qd = randn(rng, (2, 8, n + 66, 128), BF16)
    keep = (np.arange(70)[None] <= np.arange(70 - (n + 66), 70)[:, None]).astype(np.float64)[None, None].repeat(2, 0)
    got = cache.attend(qd, 0.1, kvhip.MaskMode.causal())
    check(got, *exact_and_bound(q, oracle, 0.1, keep))
