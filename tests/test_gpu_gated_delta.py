"""The gated delta rule and the short convolution against their definitions in float64.

Bounds.  Delta rule, keys of norm at most one and rates at most one: a step is a contraction of the state, so that what one token's
arithmetic adds is never enlarged by a later one and errors add up over tokens.  With M the largest row norm of a state (or element
of v) that is met, a token adds: two products of Dk terms, each off by at most (Dk / 8 + 3 + 4) half units of float32 of M
(eight lanes' chains, three permutes, the norms' roots and quotients), the decay (its exponent is off by a few
units of itself: x e^-x <= 0.37, so at most four units), the update and the sums.  96 units of 2^-24 M a token hold all of it
for Dk <= 256.  Operands of the matrix cores are split into two parts of 11 bits: the state, what is added to it, the triangular system and
its right side are each off by at most two units of the largest in their row or column, eight units a token, where the sums over 32 terms
at a time are off by less than the chains of Dk / 8.  The output is rounded once: half a step of its type.
Convolution: at most 8 products and sums of terms no larger than sum |w e| = A, then x sigmoid(x), whose slope is below 1.1: 16 units of A, and
the output's rounding.
"""
import numpy as np
import pytest
import torch

import ctypes as C

import kvhip
from kvhip import _lib as L
from oracle import recurrent as R
from tests.util import np32

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
UNIT = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(rng, B, n, Hk, Hv, Dk, Dv, dtype, gate_dtype=None):
    def t(*shape, scale=1.0, kind=dtype):
        return torch.from_numpy((rng.standard_normal(shape) * scale).astype(np.float32)).to(kind).cuda()

    x = {"q": t(B, n, Hk, Dk), "k": t(B, n, Hk, Dk), "v": t(B, n, Hv, Dv), "a": t(B, n, Hv, kind=gate_dtype or dtype),
         "b": t(B, n, Hv, kind=gate_dtype or dtype), "a_log": t(Hv, kind=torch.float32), "dt_bias": t(Hv, kind=torch.float32) - 3.0}
    return x, t(B, Hv, Dv, Dk, scale=0.2, kind=torch.float32)


def f64(t):
    return None if t is None else t.double().cpu().numpy()


def expect(x, state, **given):
    names = {k: v.cpu().numpy() if isinstance(v, torch.Tensor) else v for k, v in given.items()}
    return R.gated_delta(*(f64(x[k]) for k in ("q", "k", "v", "a", "b")), f64(x["a_log"]), f64(x["dt_bias"]), f64(state), **names)


def check(out, new, want, n, dtype, scale=1.0):
    o, s, largest = want
    bound = 96 * UNIT * (n + 2) * largest
    got, state = out.double().cpu().numpy(), new.double().cpu().numpy()
    assert np.isfinite(got).all() and np.isfinite(state).all()
    assert (np.abs(state - s) <= bound).all(), float(np.abs(state - s).max() / bound)
    room = bound * scale + half_step(dtype) * (np.abs(o) + bound * scale) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert (np.abs(got - o) <= room).all(), float((np.abs(got - o) / room).max())
    # errors that add up at random stay far below: within 4e-6 of the state's 2-norm
    assert np.linalg.norm(state - s) <= 4e-6 * np.linalg.norm(s) + 1e-30


LAYOUTS = [(2, 4, 128, 128), (1, 1, 64, 64), (1, 2, 256, 64), (1, 3, 96, 80)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("n", [1, 2, 5, 16])
def test_steps(dtype, layout, n):
    rng = np.random.default_rng(n)
    x, state = make(rng, 3, n, *layout, dtype)
    cache = kvhip.GatedDeltaCache()
    cache.delta_state = state
    out = kvhip.gated_delta_update(**x, cache=cache)
    check(out, cache.delta_state, expect(x, state), n, dtype, scale=layout[2] ** -0.5)
    assert cache.offset == n and out.shape == x["v"].shape and out.dtype == dtype


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("n", [17, 33, 63, 64, 65, 128, 200])
def test_prompts(dtype, layout, n):
    rng = np.random.default_rng(100 + n)
    x, state = make(rng, 2, n, *layout, dtype)
    cache = kvhip.GatedDeltaCache()
    cache.delta_state = state
    out = kvhip.gated_delta_update(**x, cache=cache)
    check(out, cache.delta_state, expect(x, state), n, dtype, scale=layout[2] ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_without_a_state(dtype):
    rng = np.random.default_rng(3)
    x, _ = make(rng, 2, 130, 2, 4, 128, 128, dtype)
    cache = kvhip.GatedDeltaCache()
    out = kvhip.gated_delta_update(**x, cache=cache)
    check(out, cache.delta_state, expect(x, None), 130, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Dk, Dv", [(5, 7), (30, 33), (100, 16), (130, 130), (256, 512), (16, 1), (1, 3)])
@pytest.mark.parametrize("n", [1, 70])
def test_odd_sizes(dtype, Dk, Dv, n):
    rng = np.random.default_rng(Dk)
    x, state = make(rng, 2, n, 1, 2, Dk, Dv, dtype)
    cache = kvhip.GatedDeltaCache()
    cache.delta_state = state
    out = kvhip.gated_delta_update(**x, cache=cache)
    check(out, cache.delta_state, expect(x, state), n, dtype, scale=Dk ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [3, 150])
def test_padded_batches(dtype, n):
    """Tokens that are not there: what stands in their place is never used, and a sequence may have none."""
    rng = np.random.default_rng(n)
    B = 7
    x, state = make(rng, B, n, 2, 4, 128, 64, dtype)
    pad = torch.tensor([0, 1, n, 0, n // 2, n + 5, -2], dtype=torch.int32)
    ends = torch.tensor([n, n - 1, n, 0, n // 2 + 1, n, n + 9], dtype=torch.int32)
    want = expect(x, state, left_pad=pad, lengths=ends)
    for i in range(B):
        first, end = R.span(i, n, pad.numpy(), ends.numpy())
        for name in ("q", "k", "v", "a", "b"):
            x[name][i, :first] = float("nan")
            x[name][i, end:] = float("inf")
    cache = kvhip.GatedDeltaCache()
    cache.delta_state = state
    out = kvhip.gated_delta_update(**x, cache=cache, left_pad=pad, lengths=ends.long())
    check(out, cache.delta_state, want, n, dtype)
    for i in range(B):
        first, end = R.span(i, n, pad.numpy(), ends.numpy())
        assert not out[i, :first].any() and not out[i, end:].any()
        if first == end:
            assert torch.equal(cache.delta_state[i], state[i])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompts_beyond_one_stretch_of_the_workspace(dtype):
    """Prompts that are laid out in two stretches, with sequences that end in the first, begin in the second, or have no token."""
    rng = np.random.default_rng(3)
    B, H, n = 32, 32, 400
    x, state = make(rng, B, n, H, H, 8, 4, dtype)
    sizes = dict(B=B, Hk=H, Hv=H, Dk=8, Dv=4, dtype={torch.float16: L.F16, torch.bfloat16: L.BF16}[dtype], gate_dtype=L.F32)
    need = [L.load().kvhip_gated_delta_workspace(C.byref(L.GatedDelta(L=m, **sizes))) for m in (n, 2 * n)]
    assert need[0] == need[1]
    pad = torch.from_numpy(rng.integers(0, 70, B).astype(np.int32))
    ends = torch.from_numpy(rng.integers(300, n + 1, B).astype(np.int32))
    pad[3], ends[4], ends[5], pad[6] = 333, 100, 0, n
    cache = kvhip.GatedDeltaCache()
    cache.delta_state = state
    out = kvhip.gated_delta_update(**x, cache=cache, left_pad=pad, lengths=ends)
    check(out, cache.delta_state, expect(x, state, left_pad=pad, lengths=ends), n, dtype)
    assert not out[5].any() and torch.equal(cache.delta_state[5], state[5]) and torch.equal(cache.delta_state[6], state[6])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [3, 150])
def test_what_is_no_number_stays_in_its_sequence(dtype, n):
    rng = np.random.default_rng(n)
    x, state = make(rng, 4, n, 2, 4, 64, 48, dtype)
    cache = kvhip.GatedDeltaCache()
    cache.delta_state = state
    fine = kvhip.gated_delta_update(**x, cache=cache)
    at = n - 2
    x["k"][0, at, 1, 5] = float("inf")
    x["a"][1, at, 2] = float("nan")
    x["v"][2, at, 3, 7] = float("nan")
    other = kvhip.GatedDeltaCache()
    other.delta_state = state
    out = kvhip.gated_delta_update(**x, cache=other)
    assert torch.equal(out[3], fine[3]) and torch.equal(other.delta_state[3], cache.delta_state[3])
    for b, head, rows in ((0, (2, 3), slice(None)), (1, (2,), slice(None)), (2, (3,), slice(7, 8))):
        for h in range(4):
            if h not in head:
                assert torch.equal(out[b, :, h], fine[b, :, h]) and torch.equal(other.delta_state[b, h], cache.delta_state[b, h])
        for h in head:
            assert not torch.isfinite(other.delta_state[b, h, rows]).all() and torch.isnan(out[b, at:, h, rows]).any()
    assert torch.isnan(other.delta_state[1, 2]).all() and torch.isnan(out[1, at:, 2]).all()
    still = [c for c in range(48) if c != 7]
    assert torch.equal(out[2, :, 3, still], fine[2, :, 3, still]) and torch.equal(other.delta_state[2, 3, still], cache.delta_state[2, 3, still])


@pytest.mark.parametrize("n", [1, 40])
def test_gates_of_other_types(n):
    """Gates in float32 beside 16-bit rows, their parameters in any type, with no bias, and the same by either way into the library."""
    rng = np.random.default_rng(n)
    dtype = torch.bfloat16
    x, state = make(rng, 2, n, 2, 4, 64, 64, dtype, gate_dtype=torch.float32)
    x["a_log"], x["dt_bias"] = x["a_log"].to(dtype), x["dt_bias"].to(dtype)
    plain = dict(x, a_log=x["a_log"].float(), dt_bias=x["dt_bias"].float())
    results = []
    for given in (x, plain, dict(plain, left_pad=torch.zeros(2, dtype=torch.int64))):
        cache = kvhip.GatedDeltaCache()
        cache.delta_state = state
        out = kvhip.gated_delta_update(**given, cache=cache)
        check(out, cache.delta_state, expect(plain, state), n, dtype)
        results.append((out, cache.delta_state))
    assert all(torch.equal(a, b) for r in results[1:] for a, b in zip(r, results[0]))
    none = dict(plain, dt_bias=torch.zeros(4, device="cuda"))
    cache = kvhip.GatedDeltaCache()
    cache.delta_state = state
    out = kvhip.gated_delta_update(**dict(none, dt_bias=None), cache=cache)
    check(out, cache.delta_state, expect(none, state), n, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_small_values_behind_large_ones_that_fade(dtype):
    """What a chunk adds to the state is laid out by a bound that large values in front raise: a state that is a thousandth of them
    loses nothing."""
    rng = np.random.default_rng(8)
    n = 64
    x, state = make(rng, 2, n, 1, 2, 128, 32, dtype, gate_dtype=torch.float32)
    x["v"][:, :20] *= 1000
    x["a"] = torch.full((2, n, 2), -0.01, device="cuda")
    x["a"][:, 24:32] = -3.0  # (e^-24 of what was there is left)
    x["b"] = torch.sigmoid(x["b"])
    given = dict(x, a_log=None, dt_bias=None)
    cache = kvhip.GatedDeltaCache()
    cache.delta_state = state
    out = kvhip.gated_delta_update(**given, cache=cache)
    want = R.gated_delta(*(f64(x[k]) for k in ("q", "k", "v", "a", "b")), None, None, f64(state))
    new = cache.delta_state.double().cpu().numpy()
    assert np.linalg.norm(new - want[1]) <= 4e-6 * np.linalg.norm(want[1]) and torch.isfinite(out.float()).all()


@pytest.mark.parametrize("n", [4, 96])
def test_parts_of_one_array(n):
    """Queries, keys and values as the convolution hands them on, side by side; gates side by side; from an odd element on."""
    rng = np.random.default_rng(n)
    dtype = torch.bfloat16
    x, state = make(rng, 2, n, 2, 4, 64, 64, dtype)
    for shift in (0, 1, 4):
        whole = torch.full((2, n, 3 + 4 * 64 + 4 * 64 + 9), 7.0, dtype=dtype, device="cuda")
        gates = torch.full((2, n, 13), 7.0, dtype=dtype, device="cuda")
        y = dict(x)
        at = shift
        for name, heads in (("q", 2), ("k", 2), ("v", 4)):
            part = whole[..., at:at + heads * 64].unflatten(-1, (heads, 64))
            part.copy_(x[name])
            y[name] = part
            at += heads * 64
        y["a"], y["b"] = gates[..., shift:shift + 4], gates[..., shift + 4:shift + 8]
        y["a"].copy_(x["a"])
        y["b"].copy_(x["b"])
        cache = kvhip.GatedDeltaCache()
        cache.delta_state = state
        out = kvhip.gated_delta_update(**y, cache=cache)
        check(out, cache.delta_state, expect(x, state), n, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [2, 100])
def test_gates_given_and_no_norms(dtype, n):
    """a the decays' logarithms, b the rates, both float32; queries and keys as they come (keys of norm below one)."""
    rng = np.random.default_rng(n)
    x, state = make(rng, 2, n, 1, 2, 128, 128, dtype, gate_dtype=torch.float32)
    x["k"] = (x["k"].float() * 0.08).to(dtype)
    x["k"] = (x["k"].float() / x["k"].float().norm(dim=-1, keepdim=True).clamp(min=1.0)).to(dtype)
    x["a"], x["b"] = -x["a"].abs(), torch.sigmoid(x["b"])
    x["a"][:, ::3] = 0.0
    x["b"][:, 1::4] = 0.0
    x["a_log"] = x["dt_bias"] = None
    cache = kvhip.GatedDeltaCache()
    cache.delta_state = state
    out = kvhip.gated_delta_update(**x, cache=cache, scale=0.25, norm_eps=0.0)
    top = float(np.sqrt((f64(x["q"]) ** 2).sum(-1)).max())
    check(out, cache.delta_state, expect(x, state, scale=0.25, norm_eps=0.0), n, dtype, scale=0.25 * top)


@pytest.mark.parametrize("dtype", DTYPES)
def test_decays_from_none_to_all(dtype):
    """Decays of e^-1000 (a text begins anew) among decays of nothing: what is summed up over a chunk must not lose the small ones."""
    rng = np.random.default_rng(5)
    n = 192
    x, state = make(rng, 1, n, 1, 3, 128, 128, dtype, gate_dtype=torch.float32)
    a = -np.abs(rng.standard_normal((1, n, 3))) * 1e-3
    a[:, 5], a[:, 64], a[:, 100, 1], a[:, 150, 2] = -1000.0, -300.0, -88.0, -1e30
    a[:, 20:40, 0] = 0.0
    x["a"], x["b"] = torch.from_numpy(a.astype(np.float32)).cuda(), torch.sigmoid(x["b"])
    x["a_log"] = x["dt_bias"] = None
    cache = kvhip.GatedDeltaCache()
    cache.delta_state = state
    out = kvhip.gated_delta_update(**x, cache=cache)
    check(out, cache.delta_state, expect(x, state), n, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_key_again_and_again(dtype):
    """The same key for a whole prompt, at full rate and without decay: the chunk's system is as far from the identity as it gets."""
    rng = np.random.default_rng(6)
    n = 150
    x, state = make(rng, 1, n, 1, 1, 64, 64, dtype, gate_dtype=torch.float32)
    x["k"][:] = x["k"][:, :1].clone()
    x["a"], x["b"] = torch.zeros_like(x["a"]), torch.ones_like(x["b"])
    x["a_log"] = x["dt_bias"] = None
    cache = kvhip.GatedDeltaCache()
    cache.delta_state = state
    out = kvhip.gated_delta_update(**x, cache=cache)
    check(out, cache.delta_state, expect(x, state), n, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e4, 1e-4])
def test_values_of_other_sizes(dtype, size):
    """States of any size: nothing between is held in fewer bits' range.  Zero queries and keys among them."""
    rng = np.random.default_rng(7)
    n = 100
    x, state = make(rng, 1, n, 1, 2, 128, 64, dtype)
    x["v"] = (x["v"].float() * size).to(dtype)
    state = state * size
    x["k"][:, 11] = 0.0
    x["q"][:, 70] = 0.0
    cache = kvhip.GatedDeltaCache()
    cache.delta_state = state
    out = kvhip.gated_delta_update(**x, cache=cache)
    check(out, cache.delta_state, expect(x, state), n, dtype)


@pytest.mark.parametrize("n", [3, 100])
@pytest.mark.parametrize("size", [2.0 ** 118, 2.0 ** -110])
def test_values_at_the_ends_of_the_range(n, size):
    """bfloat16 has float32's range, and so has what a prompt is made of."""
    rng = np.random.default_rng(9)
    x, state = make(rng, 2, n, 1, 2, 128, 64, torch.bfloat16)
    x["v"] = x["v"] * size
    state = state * size
    cache = kvhip.GatedDeltaCache()
    cache.delta_state = state
    out = kvhip.gated_delta_update(**x, cache=cache)
    check(out, cache.delta_state, expect(x, state), n, torch.bfloat16)


def test_calls_join():
    """A prompt, a draft and tokens give what they give in one call, within the bound of both; a copy is what it was."""
    rng = np.random.default_rng(8)
    x, _ = make(rng, 2, 140, 2, 4, 128, 128, torch.bfloat16)
    cache = kvhip.GatedDeltaCache()
    outs, at = [], 0
    for n in (70, 1, 5, 1, 63):
        part = {k: v[:, at:at + n] if v.dim() > 1 else v for k, v in x.items()}
        outs.append(kvhip.gated_delta_update(**part, cache=cache))
        at += n
        if at == 71:
            kept = cache.copy()
    check(torch.cat(outs, 1), cache.delta_state, expect(x, None), 140, torch.bfloat16)
    assert cache.offset == 140 and kept.offset == 71
    again = [kvhip.gated_delta_update(**{k: v[:, a:b] if v.dim() > 1 else v for k, v in x.items()}, cache=kept) for a, b in ((71, 76), (76, 77), (77, 140))]
    assert torch.equal(torch.cat(again, 1), torch.cat(outs[2:], 1)) and torch.equal(kept.delta_state, cache.delta_state)


@pytest.mark.parametrize("n", [4, 100])
def test_state_kept_for_a_rejected_draft(n):
    """state_in and state_out apart: the old one stays."""
    rng = np.random.default_rng(9)
    x, state = make(rng, 2, n, 1, 2, 64, 64, torch.float16)
    cache = kvhip.GatedDeltaCache()
    cache.delta_state = state
    want = kvhip.gated_delta_update(**x, cache=cache)
    old, new, out = state.clone(), torch.full_like(state, 3.0), torch.empty_like(want)
    a = L.GatedDelta(q=x["q"].data_ptr(), k=x["k"].data_ptr(), v=x["v"].data_ptr(), a=x["a"].data_ptr(), b=x["b"].data_ptr(), a_log=x["a_log"].data_ptr(),
                     dt_bias=x["dt_bias"].data_ptr(), state_in=old.data_ptr(), state_out=new.data_ptr(), out=out.data_ptr(), B=2, L=n, Hk=1, Hv=2, Dk=64,
                     Dv=64, dtype=L.F16, gate_dtype=L.F16, scale=64 ** -0.5, norm_eps=1e-6)
    for name in ("q", "k", "v", "a", "b"):
        setattr(a, name + "_stride_b", x[name].stride(0))
        setattr(a, name + "_stride_l", x[name].stride(1))
    lib = kvhip.load()
    need = lib.kvhip_gated_delta_workspace(C.byref(a))
    scratch = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    assert lib.kvhip_gated_delta(C.byref(a), scratch.data_ptr() if need else None, need, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out, want) and torch.equal(new, cache.delta_state) and torch.equal(old, state)


@pytest.mark.parametrize("n", [1, 130])
def test_on_a_stream_of_its_own_and_in_a_graph(n):
    rng = np.random.default_rng(10)
    x, state = make(rng, 2, n, 2, 4, 128, 128, torch.bfloat16)
    w = torch.randn(512, 4, device="cuda").bfloat16()
    y = torch.randn(2, n, 512, device="cuda").bfloat16()

    def step(cache):
        return kvhip.causal_convolution(y, w, cache), kvhip.gated_delta_update(**x, cache=cache)

    eager, captured = kvhip.GatedDeltaCache(), kvhip.GatedDeltaCache()
    for c in (eager, captured):
        c.delta_state, c.window = state, y[:, :1].expand(-1, 3, -1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step(eager)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(captured)
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, first))
        assert torch.equal(captured.delta_state, eager.delta_state) and torch.equal(captured.window, eager.window)
        first = step(eager)
        torch.cuda.synchronize()


def test_offsets_beyond_32_bits():
    """Tokens 2^27 elements apart: the last one begins 5 GB behind the first."""
    rng = np.random.default_rng(11)
    x, state = make(rng, 1, 20, 1, 1, 64, 64, torch.bfloat16)
    far = torch.empty(19 * 2 ** 27 + 256, dtype=torch.bfloat16, device="cuda")
    y = dict(x)
    for i, name in enumerate(("q", "k", "v")):
        y[name] = far[64 * i:].as_strided((1, 20, 1, 64), (0, 2 ** 27, 64, 1), 64 * i)
        y[name].copy_(x[name])
    cache = kvhip.GatedDeltaCache()
    cache.delta_state = state
    out = kvhip.gated_delta_update(**y, cache=cache)
    check(out, cache.delta_state, expect(x, state), 20, torch.bfloat16)


def test_empty_calls():
    cache = kvhip.GatedDeltaCache()
    x, _ = make(np.random.default_rng(0), 1, 0, 1, 1, 64, 64, torch.bfloat16)
    assert kvhip.gated_delta_update(**x, cache=cache).shape == (1, 0, 1, 64)
    assert cache.convolve(torch.empty(2, 0, 8, device="cuda"), torch.empty(8, 4, device="cuda")).shape == (2, 0, 8)
    assert cache.state == [] and cache.offset == 0


# ---- the short convolution --------------------------------------------------------------------------------------------
def conv_inputs(rng, B, n, c, W, dtype):
    def t(*shape):
        return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dtype).cuda()
    return t(B, n, c), t(c, W), t(c), t(B, W - 1, c)


def check_conv(y, cache, x, w, bias, window, dtype, silu=True, **given):
    names = {k: v.cpu().numpy() for k, v in given.items()}
    want, new = R.short_convolution(f64(x), f64(w), f64(bias), f64(window), silu, **names)
    size, _ = R.short_convolution(np.abs(f64(x)), np.abs(f64(w)), None if bias is None else np.abs(f64(bias)),
                                  None if window is None else np.abs(f64(window)), False, **names)
    room = 16 * UNIT * size + half_step(dtype) * (np.abs(want) + 16 * UNIT * size) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    got = y.double().cpu().numpy()
    assert (np.abs(got - want) <= room).all(), float((np.abs(got - want) / np.maximum(room, 1e-300)).max())
    assert np.array_equal(f64(cache.window), new)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 3, 4, 31, 32, 33, 65, 100])
@pytest.mark.parametrize("c, W", [(64, 4), (24, 4), (1000, 4), (7, 4), (64, 2), (16, 1), (40, 7), (64, 8), (3, 3)])
def test_convolution(dtype, n, c, W):
    rng = np.random.default_rng(n)
    x, w, bias, window = conv_inputs(rng, 2, n, c, W, dtype)
    for b, start, silu in ((None, None, True), (bias, window, True), (bias, window, False)):
        cache = kvhip.GatedDeltaCache(W)
        cache.window = start
        y = kvhip.causal_convolution(x, w, cache, bias=b, silu=silu)
        check_conv(y, cache, x, w, b, start, dtype, silu)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [2, 37, 70])
@pytest.mark.parametrize("W", [4, 6])
def test_convolution_of_padded_batches(dtype, n, W):
    rng = np.random.default_rng(n)
    B = 8
    x, w, bias, window = conv_inputs(rng, B, n, 48, W, dtype)
    pad = torch.tensor([0, 1, n, 0, n // 2, n + 5, -2, max(0, n - 3)], dtype=torch.int32)
    ends = torch.tensor([n, n - 1, n, 0, n // 2 + 1, n, n + 9, n], dtype=torch.int32)
    clean = x.clone()
    for i in range(B):
        first, end = R.span(i, n, pad.numpy(), ends.numpy())
        clean[i, :first] = 0
        clean[i, end:] = 0
        x[i, :first] = float("nan")
        x[i, end:] = float("inf")
    cache = kvhip.GatedDeltaCache(W)
    cache.window = window
    y = kvhip.causal_convolution(x, w, cache, bias=bias, left_pad=pad, lengths=ends)
    check_conv(y, cache, clean, w, bias, window, dtype, left_pad=pad, lengths=ends)


@pytest.mark.parametrize("dtype", DTYPES)
def test_convolution_of_parts_and_calls_that_join(dtype):
    rng = np.random.default_rng(4)
    x, w, bias, window = conv_inputs(rng, 2, 90, 40, 4, dtype)
    whole = torch.empty(2, 90, 61, dtype=dtype, device="cuda")
    for shift in (0, 5, 8):
        part = whole[..., shift:shift + 40]
        part.copy_(x)
        cache = kvhip.GatedDeltaCache(4)
        cache.window = window
        y = torch.cat([cache.convolve(part[:, a:b], w, bias) for a, b in ((0, 1), (1, 3), (3, 50), (50, 90))], 1)
        check_conv(y, cache, x, w, bias, window, dtype)


@pytest.mark.parametrize("n", [1, 40])
def test_convolution_with_weights_that_lie_otherwise(n):
    """Weights of another layer's layout, a strided bias and a column of a wider batch give what dense ones give, by either way in."""
    rng = np.random.default_rng(n)
    dtype = torch.bfloat16
    x, w, bias, window = conv_inputs(rng, 3, n, 24, 4, dtype)
    taps, wide = w.t().contiguous().t(), torch.stack([bias, bias], -1)[:, 0]
    part = torch.stack([x, x], 1)[:, 1]
    results = []
    for given in (dict(x=x, weight=w, bias=bias), dict(x=x, weight=taps, bias=wide), dict(x=part, weight=w, bias=bias),
                  dict(x=x, weight=w, bias=bias, left_pad=torch.zeros(3, dtype=torch.int32))):
        cache = kvhip.GatedDeltaCache(4)
        cache.window = window
        y = kvhip.causal_convolution(cache=cache, **given)
        check_conv(y, cache, x, w, bias, window, dtype)
        results.append((y, cache.window))
    assert all(torch.equal(a, b) for r in results[1:] for a, b in zip(r, results[0]))
    with pytest.raises(ValueError):
        cache.convolve(x, w[:, :3])
    with pytest.raises(ValueError):
        cache.convolve(x[:2], w)
    with pytest.raises(ValueError):
        cache.convolve(x, w, bias.float())


def test_a_layers_calls_together():
    """Convolution, its parts as queries, keys and values, the delta rule: a prompt and two tokens, as a layer makes them."""
    rng = np.random.default_rng(12)
    B, Hk, Hv, D = 2, 2, 4, 64
    c = (2 * Hk + Hv) * D
    x, w, _, _ = conv_inputs(rng, B, 75, c, 4, torch.float32)
    gates, _ = make(rng, B, 75, Hk, Hv, D, D, torch.float32)
    cache = kvhip.GatedDeltaCache()
    outs = []
    for a, b in ((0, 73), (73, 74), (74, 75)):
        q, k, v = kvhip.causal_convolution(x[:, a:b], w, cache).split([Hk * D, Hk * D, Hv * D], -1)
        outs.append(kvhip.gated_delta_update(q.unflatten(-1, (Hk, D)), k.unflatten(-1, (Hk, D)), v.unflatten(-1, (Hv, D)), gates["a"][:, a:b],
                                             gates["b"][:, a:b], gates["a_log"], gates["dt_bias"], cache))
    y, window = R.short_convolution(f64(x), f64(w))
    q, k, v = np.split(y, [Hk * D, 2 * Hk * D], -1)
    parts = [t.reshape(B, 75, -1, D) for t in (q, k, v)]
    o, s, largest = R.gated_delta(*parts, f64(gates["a"]), f64(gates["b"]), f64(gates["a_log"]), f64(gates["dt_bias"]))
    # (the convolution's float32 rounding, through norms of vectors that are at least 1 long and a contraction, adds no more than the rule's own)
    bound = 2 * 96 * UNIT * 77 * largest
    assert (np.abs(f64(torch.cat(outs, 1)) - o) <= bound).all() and (np.abs(f64(cache.delta_state) - s) <= bound).all()
    assert np.array_equal(f64(cache.window), window)
