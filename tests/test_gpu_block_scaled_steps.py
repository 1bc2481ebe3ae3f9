"""Single tokens into a block-scaled cache that the attention kernel writes, whichever kernel takes the call."""
import numpy as np
import pytest
import torch

import kvhip
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
