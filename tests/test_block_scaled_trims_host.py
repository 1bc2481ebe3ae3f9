"""The oracle of block-scaled caches where rows are taken off again: what is left of a block is as it came."""
import numpy as np
import pytest
import torch

from oracle import block_scaled as O


def rows(rng, n, dtype, size):
    x = torch.from_numpy(rng.standard_normal((1, 2, n, 8)) * size).to(getattr(torch, dtype))
    return x.double().numpy()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("held", [61, 62, 63, 126])
def test_rejected_drafts_leave_no_trace(dtype, held):
    rng = np.random.default_rng(held)
    cache, alone = O.BlockScaledCache(dtype), O.BlockScaledCache(dtype)
    first = rows(rng, held, dtype, 0.01)
    for c in (cache, alone):
        c.update(first, first)
    for accepted in (1, 0, 3, 2, 0, 3):
        draft = rows(rng, 4, dtype, 1000.0)
        draft[:, :, :accepted] = rows(rng, accepted, dtype, 0.01)
        cache.update(draft, draft)
        cache.trim(4 - accepted)
        if accepted:
            alone.update(draft[:, :, :accepted], draft[:, :, :accepted])
        assert cache.offset == alone.offset
        assert np.array_equal(cache.keys, alone.keys) and np.array_equal(cache.values, alone.values)


def test_a_call_taken_back():
    rng = np.random.default_rng(1)
    cache = O.BlockScaledCache("bfloat16")
    first = rows(rng, 100, "bfloat16", 0.01)
    cache.update(first, first)
    before = cache.keys.copy()
    for n in (300, 28, 64, 1):
        more = rows(rng, n, "bfloat16", 100.0)
        cache.update(more, more)
        cache.trim(n)
        assert np.array_equal(cache.keys, before)
