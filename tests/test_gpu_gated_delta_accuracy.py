"""Accuracy of the gated delta rule where the bounds of a worst case say little.

A 16-bit output is a float32 value y, rounded once: with o the definition's value, |out - o| <= |y - o| + half a step of the type at the larger of
both.  What |out - o| has beyond that half step is therefore no more than |y - o|, which is held to what states are held to: errors
that add up at random stay below 4e-6 of the 2-norm."""
import numpy as np
import pytest
import torch

import kvhip
from oracle import recurrent as R
from tests.test_gpu_gated_delta import DTYPES, LAYOUTS, expect, f64, make

pytestmark = pytest.mark.gpu


def half_steps(out, o, dtype):
    """Half the distance of `dtype`'s neighbouring values where `out` and `o` lie."""
    info = torch.finfo(dtype)
    size = np.maximum(np.maximum(np.abs(out), np.abs(o)), info.tiny)
    return 2.0 ** np.floor(np.log2(size)) * info.eps / 2


def beyond_rounding(out, o, dtype):
    got = f64(out)
    return np.maximum(np.abs(got - o) - (half_steps(got, o, dtype) if dtype != torch.float32 else 0.0), 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("n", [1, 5, 40, 200])
def test_outputs_are_rounded_once(dtype, layout, n):
    rng = np.random.default_rng(200 + n)
    x, state = make(rng, 2, n, *layout, dtype)
    cache = kvhip.GatedDeltaCache()
    cache.delta_state = state
    out = kvhip.gated_delta_update(**x, cache=cache)
    o, s, _ = expect(x, state)
    assert np.linalg.norm(f64(cache.delta_state) - s) <= 4e-6 * np.linalg.norm(s)
    assert np.linalg.norm(beyond_rounding(out, o, dtype)) <= 4e-6 * np.linalg.norm(o)


@pytest.mark.parametrize("dtype", DTYPES[:2])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("n", [20, 100, 200])
def test_what_memory_held_before_is_nothing_to_a_prompt(dtype, layout, n):
    """Workspace and registers are of no content: matrix instructions work on whole registers whatever lanes are masked, and what they
    work on has to have been written."""
    rng = np.random.default_rng(300 + n)
    x, state = make(rng, 2, n, *layout, dtype)
    results = []
    for junk in (float("nan"), float("inf"), 0.0):
        held = [torch.full((size,), junk, device="cuda") for size in (500, 8192, 13000, 16384, 60000, 200000)]
        cache = kvhip.GatedDeltaCache()
        cache.delta_state = state
        del held
        results.append((kvhip.gated_delta_update(**x, cache=cache), cache.delta_state))
    assert all(torch.equal(a, b) for r in results[1:] for a, b in zip(r, results[0]))
    o, s, _ = expect(x, state)
    assert np.linalg.norm(f64(results[0][1]) - s) <= 4e-6 * np.linalg.norm(s)
    assert np.linalg.norm(beyond_rounding(results[0][0], o, dtype)) <= 4e-6 * np.linalg.norm(o)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e3, 1e5, 1e6, 1e7, 6e7])
@pytest.mark.parametrize("n, first, fade", [(64, 20, 24), (64, 3, 3), (150, 75, 80), (20, 5, 6)])
def test_values_that_are_forgotten_cost_the_others_nothing(dtype, size, n, first, fade):
    """Values of up to 6e7 times the others (float16 goes no further) that a chunk's decays wipe out: what stays keeps its accuracy, and so do
    the outputs behind them."""
    rng = np.random.default_rng(8)
    x, state = make(rng, 2, n, 1, 2, 128, 32, dtype, gate_dtype=torch.float32)
    low = min(1.0, 1e4 / size)
    x["v"] = (x["v"].float() * low).to(dtype)
    x["v"][:, :first] = (x["v"][:, :first].float() * size).to(dtype)
    a = torch.full((2, n, 2), -0.01, device="cuda")
    a[:, fade:fade + 8] = -8.0  # (e^-64 of what was there is left)
    given = dict(x, a=a, b=torch.sigmoid(x["b"]), a_log=None, dt_bias=None)
    assert torch.isfinite(x["v"].float()).all()
    cache = kvhip.GatedDeltaCache()
    cache.delta_state = state * low
    out = kvhip.gated_delta_update(**given, cache=cache)
    o, s, _ = R.gated_delta(*(f64(given[k]) for k in ("q", "k", "v", "a", "b")), None, None, f64(state * low))
    assert np.linalg.norm(f64(cache.delta_state) - s) <= 4e-6 * np.linalg.norm(s)
    behind = slice(fade + 8, n)
    assert np.linalg.norm(beyond_rounding(out, o, dtype)[:, behind]) <= 4e-6 * np.linalg.norm(o[:, behind])
