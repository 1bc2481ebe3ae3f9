"""Refusals of the recurrent layers' operators, of beam selection and of reordering: nothing reaches a device.  And the oracle
against what can be said without it."""
import ctypes as C

import numpy as np
import pytest
import torch

import kvhip
from kvhip import _lib as L
from kvhip import recurrent
from oracle import recurrent as R
from oracle import beams as OB

P = C.c_void_p(4096)  # stands for device memory that a refused call never touches


def delta(**given):
    x = L.GatedDelta(q=4096, k=4096, v=4096, a=4096, b=4096, state_out=4096, out=4096, B=1, L=4, Hk=2, Hv=4, Dk=64, Dv=64, dtype=L.BF16,
                     gate_dtype=L.BF16, scale=1.0, norm_eps=1e-6)
    for name in ("q", "k", "v", "a", "b"):
        setattr(x, name + "_stride_b", 1024)
        setattr(x, name + "_stride_l", 256)
    for name, value in given.items():
        setattr(x, name, value)
    return x


INVALID, UNSUPPORTED = -2, -3


@pytest.mark.parametrize("given, status", [
    (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(state_out=None), INVALID), (dict(b=None), INVALID), (dict(B=0), INVALID),
    (dict(L=0), INVALID), (dict(Dv=-1), INVALID), (dict(Hv=5), INVALID), (dict(dtype=L.U32), INVALID), (dict(gate_dtype=9), INVALID),
    (dict(norm_eps=-1.0), INVALID), (dict(norm_eps=float("nan")), INVALID), (dict(k_stride_l=-1), INVALID), (dict(Dk=257), UNSUPPORTED),
    (dict(B=65536), UNSUPPORTED), (dict(L=2 ** 25), UNSUPPORTED)])
def test_gated_delta_refuses(given, status):
    lib = kvhip.load()
    assert lib.kvhip_gated_delta(C.byref(delta(**given)), P, 1 << 40, None) == status
    assert lib.kvhip_last_error_message()


@pytest.mark.parametrize("workspace, less, status", [(None, 0, INVALID), (P, 1, INVALID), (C.c_void_p(4104), 0, INVALID)])
def test_prompts_refuse_a_workspace_that_is_none(workspace, less, status):
    lib = kvhip.load()
    x = delta(L=64)
    need = lib.kvhip_gated_delta_workspace(C.byref(x))
    assert need > 0
    assert lib.kvhip_gated_delta(C.byref(x), workspace, need - less, None) == status


def test_workspaces_go_by_sizes_alone():
    """No array has to be there to ask; single tokens and float32 need none; long prompts are laid out a stretch at a time."""
    lib = kvhip.load()

    def need(**given):
        return lib.kvhip_gated_delta_workspace(C.byref(delta(**given)))

    assert need(L=64, q=None, k=None, v=None, a=None, b=None, state_out=None, out=None) == need(L=64) > 0
    assert need(L=1) == need(L=4) == need(L=5000, dtype=L.F32) == need(L=64, Dk=300) == 0
    assert need(L=65) > need(L=64) and need(L=2 ** 20, B=8, Hk=16, Hv=32, Dk=128, Dv=128) < 2 ** 30


def test_gated_delta_refuses_nothing():
    lib = kvhip.load()
    assert lib.kvhip_gated_delta(None, None, 0, None) == INVALID
    assert lib.kvhip_gated_delta_workspace(None) == 0


@pytest.mark.parametrize("given, status", [
    (dict(x=None), INVALID), (dict(weight=None), INVALID), (dict(out=None), INVALID), (dict(window_out=None), INVALID), (dict(B=0), INVALID),
    (dict(L=-3), INVALID), (dict(W=0), INVALID), (dict(dtype=L.BOOL), INVALID), (dict(W=9), UNSUPPORTED), (dict(L=2 ** 21), UNSUPPORTED)])
def test_short_convolution_refuses(given, status):
    a = dict(x=P, sb=64, sl=8, weight=P, bias=None, B=1, L=8, C=8, W=4, dtype=L.F16, silu=1, pad=None, ends=None, window_in=None, window_out=P, out=P)
    a.update(given)
    assert kvhip.load().kvhip_short_convolution(*a.values(), None) == status


@pytest.mark.parametrize("given, status", [
    (dict(logits=None), INVALID), (dict(rows=None), INVALID), (dict(groups=0), INVALID), (dict(count=0), INVALID), (dict(dtype=3), INVALID),
    (dict(stride=-1), INVALID), (dict(beams=65), UNSUPPORTED), (dict(count=65), UNSUPPORTED), (dict(groups=40000), UNSUPPORTED),
    (dict(vocabulary=2 ** 24 + 1), UNSUPPORTED), (dict(done=P, pad=-1), INVALID), (dict(done=P, pad=1000), INVALID), (dict(bytes=15), INVALID),
    (dict(workspace=C.c_void_p(4100)), INVALID), (dict(workspace=None), INVALID)])
def test_beam_select_refuses(given, status):
    a = dict(logits=P, stride=1000, groups=2, beams=4, vocabulary=1000, dtype=L.BF16, scores=P, done=None, count=4, pad=0, rows=P, tokens=P, best=P,
             workspace=P, bytes=1 << 30)
    a.update(given)
    lib = kvhip.load()
    assert lib.kvhip_beam_select(*a.values(), None) == status
    if status == UNSUPPORTED:
        assert lib.kvhip_beam_select_workspace(a["groups"], a["beams"], a["vocabulary"], a["dtype"], a["count"]) == 0


def test_beam_workspace_grows_with_the_call():
    lib = kvhip.load()
    sizes = [lib.kvhip_beam_select_workspace(b, k, v, L.F32, c) for b, k, v, c in [(1, 1, 1, 1), (1, 4, 32000, 4), (8, 4, 32000, 4), (8, 4, 32000, 64)]]
    assert 0 < sizes[0] < sizes[1] < sizes[2] < sizes[3]


def test_reorder_refuses():
    lib = kvhip.load()
    at, sizes = (C.c_void_p * 9)(*[4096] * 9), (C.c_size_t * 9)(*[64] * 9)
    assert lib.kvhip_reorder_rows(1, at, sizes, 4, None, None) == INVALID
    assert lib.kvhip_reorder_rows(1, at, sizes, 0, P, None) == INVALID
    assert lib.kvhip_reorder_rows(-1, at, sizes, 4, P, None) == INVALID
    assert lib.kvhip_reorder_rows(9, at, sizes, 4, P, None) == UNSUPPORTED
    assert lib.kvhip_reorder_rows(1, at, sizes, 2049, P, None) == UNSUPPORTED
    at[0] = None
    assert lib.kvhip_reorder_rows(1, at, sizes, 4, P, None) == INVALID
    h = C.c_void_p()
    assert lib.kvhip_cache_create(C.byref(L.Config(kind=L.KIND_SIMPLE)), C.byref(h)) == 0
    assert lib.kvhip_cache_reorder(None, P, 0, None) == INVALID
    assert lib.kvhip_cache_reorder(h, None, 0, None) == INVALID
    assert lib.kvhip_cache_reorder(h, P, -1, None) == INVALID
    assert lib.kvhip_cache_reorder(h, P, 0, None) == 0  # (nothing is held yet)
    lib.kvhip_cache_free(h)


def test_cache_refuses_arrays_that_do_not_go_together():
    cache = kvhip.GatedDeltaCache(4)
    with pytest.raises(ValueError):
        kvhip.GatedDeltaCache(9)
    with pytest.raises(ValueError):
        cache.window = torch.zeros(2, 4, 8)
    with pytest.raises(ValueError):
        cache.delta_state = torch.zeros(2, 4, 8, 8, dtype=torch.float16)
    with pytest.raises(ValueError):
        cache.delta_state = torch.zeros(2, 4, 8, 8)  # (not on the device)
    with pytest.raises(ValueError):
        cache.state = [torch.zeros(2, 3, 8), torch.zeros(2, 3, 8)]
    x = torch.zeros(2, 5, 8)
    with pytest.raises(ValueError):
        cache.convolve(x, torch.zeros(8, 3))
    with pytest.raises(ValueError):
        cache.convolve(x, torch.zeros(8, 4), bias=torch.zeros(7))
    with pytest.raises(ValueError):
        cache.convolve(x, torch.zeros(8, 4), left_pad=torch.zeros(3))
    with pytest.raises(ValueError):
        cache.convolve(x, torch.zeros(8, 4))
    q, v, a = torch.zeros(2, 5, 2, 8), torch.zeros(2, 5, 4, 8), torch.zeros(2, 5, 4)
    with pytest.raises(ValueError):
        cache.update(q, q[:, :4], v, a, a)
    with pytest.raises(TypeError):
        cache.update(q, q.half(), v, a, a)
    with pytest.raises(ValueError):
        cache.update(q, q, v, a[..., :3], a)
    with pytest.raises(ValueError):
        cache.update(q, q, v, a, a, a_log=torch.zeros(3))
    with pytest.raises(ValueError):
        cache.update(q, q, v, a, a, dt_bias=torch.zeros(4))
    with pytest.raises(ValueError):
        cache.update(q, q, v, a, a)
    assert cache.offset == 0 and cache.state == [] and not cache.is_trimmable and cache.trim(3) == 0
    assert cache.meta_state == ["4", "0"]
    with pytest.raises(ValueError):
        cache.meta_state = ["3", "0"]
    with pytest.raises(ValueError):
        recurrent._per_sequence(torch.zeros(2), 2, "lengths")
    assert recurrent._int32(torch.tensor([2 ** 40, -2 ** 40, 7])).tolist() == [2 ** 31 - 1, -2 ** 31, 7]
    with pytest.raises(ValueError):
        kvhip.beam_select(torch.zeros(2, 5))
    with pytest.raises(ValueError):
        kvhip.beam_select(torch.zeros(2, 5, 7), scores=torch.zeros(2, 4))
    with pytest.raises(ValueError):
        kvhip.beam_select(torch.zeros(2, 5, 7), done=torch.zeros(2, 5))
    with pytest.raises(ValueError):
        kvhip.beam_select(torch.zeros(2, 5, 7))


def test_a_hybrid_models_caches_where_all_have_to_go_back():
    """A recurrent state cannot go back: rounds and trims refuse the list and touch nothing, its file format too."""
    caches = [kvhip.GatedDeltaCache(), kvhip.GatedDeltaCache(2)]
    assert kvhip.KVCacheStorage(caches).begin_round(4) is None
    assert not kvhip.can_trim_prompt_cache(caches) and kvhip.trim_prompt_cache(caches, 3) == 0
    with pytest.raises((ValueError, TypeError)):
        kvhip.save_prompt_cache("/nonexistent/file.safetensors", caches)


def test_oracle_state_is_what_was_written():
    """Orthonormal keys, rate one, no decay: the state returns each value for its key, and a key's second value takes the first's place."""
    rng = np.random.default_rng(0)
    k = np.eye(4)[None, :, None]
    v = rng.standard_normal((1, 4, 1, 3))
    out, s, _ = R.gated_delta(k, k, v, np.zeros((1, 4, 1)), np.ones((1, 4, 1)), scale=1.0, norm_eps=0.0)
    assert np.allclose(out, v) and np.allclose(s[0, 0] @ np.eye(4), v[0, :, 0].T)
    out, s, _ = R.gated_delta(k[:, :1], k[:, :1], 2 * v[:, :1], np.full((1, 1, 1), np.log(0.5)), np.ones((1, 1, 1)), state=s, scale=1.0, norm_eps=0.0)
    assert np.allclose(out[0, 0], 2 * v[0, 0]) and np.allclose(s[0, 0][:, 1:], 0.5 * v[0, 1:, 0].T)


def test_oracle_calls_join():
    rng = np.random.default_rng(1)
    q, k, v = rng.standard_normal((2, 7, 1, 4)), rng.standard_normal((2, 7, 1, 4)), rng.standard_normal((2, 7, 2, 3))
    a, b, log = rng.standard_normal((2, 7, 2)), rng.standard_normal((2, 7, 2)), np.zeros(2)
    whole, s, _ = R.gated_delta(q, k, v, a, b, log)
    first, t, _ = R.gated_delta(*(x[:, :3] for x in (q, k, v, a, b)), log)
    second, t, _ = R.gated_delta(*(x[:, 3:] for x in (q, k, v, a, b)), log, state=t)
    assert np.allclose(np.concatenate([first, second], 1), whole) and np.allclose(s, t)
    x, w = rng.standard_normal((2, 7, 5)), rng.standard_normal((5, 4))
    whole, e = R.short_convolution(x, w)
    first, f = R.short_convolution(x[:, :2], w)
    second, f = R.short_convolution(x[:, 2:], w, window=f)
    assert np.allclose(np.concatenate([first, second], 1), whole) and np.allclose(e, f)


def test_oracle_selection():
    x = np.array([[[0.0, 1.0, 1.0], [5.0, -np.inf, np.nan]]])
    rows, tokens, best = OB.beam_select(x, np.array([[0.0, -1.0]]), 4)
    assert tokens.tolist() == [[1, 2, 0, 0]] and rows.tolist() == [[0, 0, 1, 0]]
    assert np.allclose(best[0, 2], -1.0)
    rows, tokens, best = OB.beam_select(x, np.array([[-3.0, -0.5]]), 2, done=np.array([[False, True]]), pad_token=2)
    assert rows.tolist() == [[1, 0]] and tokens.tolist() == [[2, 1]] and best[0, 0] == -0.5
