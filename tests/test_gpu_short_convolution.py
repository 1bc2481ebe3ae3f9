"""How far a token of the short convolution reaches: W - 1 tokens on and no further, wherever tiles and calls are cut."""
import numpy as np
import pytest
import torch

import kvhip
from tests.test_gpu_gated_delta import DTYPES, conv_inputs

pytestmark = pytest.mark.gpu


def run(x, w, bias, window, cuts):
    cache = kvhip.GatedDeltaCache(w.shape[1])
    cache.window = window
    edges = [0, *cuts, x.shape[1]]
    return torch.cat([cache.convolve(x[:, a:b], w, bias) for a, b in zip(edges, edges[1:])], 1), cache.window


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [40, 7])
@pytest.mark.parametrize("W", range(1, 9))
def test_what_is_no_number_reaches_no_further_than_the_taps(dtype, c, W):
    rng = np.random.default_rng(W)
    n = 100
    x, w, bias, window = conv_inputs(rng, 2, n, c, W, dtype)
    fine, kept = run(x, w, bias, window, [])
    for at, value in ((0, float("nan")), (5, float("inf")), (29, float("nan")), (31, float("-inf")), (32, float("nan")), (95, float("inf")), (99, float("nan"))):
        y = x.clone()
        y[0, at, 3] = value
        reach = min(at + W, n)  # of tokens at .. at + W - 1
        for cuts in ([], [at] if at else [1], [at + 1] if at + 1 < n else [50], [3, 4, 40]):
            got, new = run(y, w, bias, window, cuts)
            assert torch.equal(got[1], fine[1]) and torch.equal(new[1], kept[1])
            assert torch.equal(got[0, :, [i for i in range(c) if i != 3]], fine[0, :, [i for i in range(c) if i != 3]])
            assert torch.equal(got[0, :at, 3], fine[0, :at, 3]) and torch.equal(got[0, reach:, 3], fine[0, reach:, 3]), (at, cuts)
            assert not torch.isfinite(got[0, at:reach, 3].float()).all()
    if W > 1:  # the window's oldest row is the first tap of the first token alone
        start = window.clone()
        start[0, 0, 3] = float("nan")
        for cuts in ([], [1], [2, 33]):
            got, _ = run(x, w, bias, start, cuts)
            assert torch.isnan(got[0, 0, 3]) and torch.equal(got[0, 1:], fine[0, 1:]) and torch.equal(got[1], fine[1])
