"""Block-scaled attention where keys and values are no numbers: they reach every query row that sees them and no other, for each
head size the kernels are built for and each kind of mask."""
import numpy as np
import pytest
import torch

import kvhip
from oracle import block_scaled as O
from test_gpu_block_scaled import causal, exact_and_bound, pair
from util import NAME, np32, randn

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
INF, NAN = float("inf"), float("nan")


def spoiled(dtype, T, layout, gone=9, per_head=5):
    """A cache of T rows, some of whose elements are no numbers, behind which `gone` rows of nothing else were taken off."""
    rng = np.random.default_rng(T + layout[2])
    hq, h, dk, dv = layout
    cache, oracle = kvhip.BlockScaledKVCache(), O.BlockScaledCache(NAME[dtype])
    (k, kd), (v, vd) = pair(dtype, rng, 2, h, (dk, dv))(T + gone)
    for x, xd, d in ((k, kd, dk), (v, vd, dv)):
        for b in range(2):
            for i in range(h):
                if x is k and i % 2:
                    continue  # (a head whose keys are numbers: its rows stay readable)
                for t in [*rng.integers(0, T, per_head), T - 1]:
                    at = (b, i, int(t), int(rng.integers(d)))
                    x[at] = xd[at] = float(rng.choice([NAN, INF, -INF]))
        x[:, :, T:] = NAN
        xd[:, :, T:] = NAN
    cache.update(kd, vd, fetch=False)
    oracle.update(k, v)
    cache.trim(gone)
    oracle.trim(gone)
    return cache, oracle, lambda n: randn(rng, (2, hq, n, dk), dtype)


def check_spoiled(got, q, oracle, scale, weight, add=None):
    B, Hq, n, _ = q.shape
    G = Hq // oracle.keys.shape[1]
    weight = np.broadcast_to(weight, (B, weight.shape[1], n, weight.shape[3]))
    w = np.stack([weight[:, {1: 0, Hq // G: x // G}.get(weight.shape[1], x)] for x in range(Hq)], 1) > 0  # [B, Hq, n, T]
    bad_key = np.repeat(np.isnan(oracle.keys).any(-1), G, 1)[:, :, None]
    bad_value = np.repeat(np.isnan(oracle.values), G, 1).astype(np.float64)
    want_nan = (w & bad_key).any(-1)[..., None] | (w.astype(np.float64) @ bad_value > 0)
    got = np32(got).astype(np.float64)
    assert want_nan.any() and not want_nan.all()
    assert np.array_equal(np.isnan(got), want_nan)
    numbers = O.BlockScaledCache(oracle.dtype)
    numbers.keys, numbers.values = np.nan_to_num(oracle.keys), np.nan_to_num(oracle.values)
    want, bound = exact_and_bound(q, numbers, scale, weight, add)
    error = np.where(want_nan, 0.0, np.abs(got - want)) / bound
    assert np.isfinite(got[~want_nan]).all() and error.max() <= 1.0, error.max()


SPOILED = [(64, 64, 6, 2), (96, 96, 4, 4), (192, 128, 4, 2), (256, 256, 6, 2), (50, 36, 4, 2), (128, 128, 8, 2)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sizes", SPOILED)
@pytest.mark.parametrize("T,n,pads,window", [(75, 1, (11, 3), 0), (140, 4, (0, 70), 0), (400, 30, (64, 5), 100), (330, 140, (3, 200), 0), (192, 1, (0, 191), 0)])
def test_masks_of_indices(dtype, sizes, T, n, pads, window):
    dk, dv, hq, h = sizes
    cache, oracle, queries = spoiled(dtype, T, (hq, h, dk, dv))
    q, qd = queries(n)
    mask = kvhip.MaskMode.window_mask(T - n, window, left_pad=torch.tensor(pads, device="cuda"))
    check_spoiled(cache.attend(qd, dk ** -0.5, mask), q, oracle, dk ** -0.5, causal(T, n, pads, window))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sizes", SPOILED)
@pytest.mark.parametrize("T,n", [(75, 1), (140, 4), (300, 30)])
@pytest.mark.parametrize("kind", ["bool", "added"])
def test_array_masks(dtype, sizes, T, n, kind):
    dk, dv, hq, h = sizes
    cache, oracle, queries = spoiled(dtype, T, (hq, h, dk, dv))
    q, qd = queries(n)
    gen = torch.Generator(device="cuda").manual_seed(T)
    keep = torch.rand(2, hq, n, T, generator=gen, device="cuda") < 0.1
    keep[0, 0, 0] = False
    mask, add = keep, None
    if kind == "added":
        mask = torch.randn(2, hq, n, T, generator=gen, device="cuda").masked_fill(~keep, -INF)
        add = mask.double().cpu().numpy()
    got = cache.attend(qd, dk ** -0.5, kvhip.MaskMode.from_array(mask))
    check_spoiled(got, q, oracle, dk ** -0.5, keep.double().cpu().numpy(), add)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sizes", SPOILED)
@pytest.mark.parametrize("T,n,count,pads", [(700, 1, 3, (0, 200)), (701, 5, 4, (70, 640)), (2100, 2, 9, (0, 0)), (690, 30, 2, (0, 650))])
def test_listed_blocks(dtype, sizes, T, n, count, pads):
    dk, dv, hq, h = sizes
    cache, oracle, queries = spoiled(dtype, T, (hq, h, dk, dv))
    q, qd = queries(n)
    rng = np.random.default_rng(count)
    blocks = np.full((2, h, n, count), -1, np.int32)
    for at in np.ndindex(2, h, n):
        some = np.sort(rng.choice((T + 63) // 64, count, replace=False))
        blocks[at] = some
    weight = O.listed_keep(blocks, T, pads)
    pad = torch.tensor(pads, device="cuda")
    check_spoiled(cache.attend_blocks(qd, torch.from_numpy(blocks).cuda(), dk ** -0.5, pad), q, oracle, dk ** -0.5, weight)
    # a choice among keys that are no numbers: their elements have no say
    assert np.array_equal(cache.select_blocks(qd, count, 0, 1, pad).cpu().numpy(), O.select(q, oracle, count, 0, 1, pads))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sizes", SPOILED)
def test_steps_that_write_what_is_no_number(dtype, sizes):
    """A token's own key and value, written by the attention kernel: infinities are NaN from the same call on."""
    dk, dv, hq, h = sizes
    rng = np.random.default_rng(dk)
    make = pair(dtype, rng, 2, h, (dk, dv))
    cache, oracle = kvhip.BlockScaledKVCache(), O.BlockScaledCache(NAME[dtype])
    (k, kd), (v, vd) = make(62)
    cache.update(kd, vd, fetch=False)
    oracle.update(k, v)
    for i in range(4):
        (k, kd), (v, vd) = make(1)
        k[1, h - 1, 0, dk - 1], v[0, 0, 0, dv - 1 - i] = (INF, -INF, NAN, INF)[i], (NAN, INF, INF, -INF)[i]
        kd, vd = (torch.from_numpy(x).to(dtype).cuda() for x in (k, v))
        q, qd = randn(rng, (2, hq, 1, dk), dtype)
        got = cache.update_attend(qd, kd, vd, 0.1)
        oracle.update(k, v)
        check_spoiled(got, q, oracle, 0.1, causal(oracle.offset, 1, (0, 0)))
        for x, y in zip(cache.fetch(), (oracle.keys, oracle.values)):
            assert np.array_equal(np32(x).astype(np.float64), y, equal_nan=True)
