"""What the block-scaled cache refuses and answers without a device, and its oracle's own arithmetic."""
import ctypes as C

import numpy as np
import pytest
import torch

import kvhip
from kvhip import _lib as L
from oracle import block_scaled as O


def make(kind=L.KIND_BLOCK_SCALED):
    lib, h = kvhip.load(), C.c_void_p()
    assert lib.kvhip_cache_create(C.byref(L.Config(kind=kind)), C.byref(h)) == 0
    return lib, h


def test_an_empty_cache():
    lib, h = make()
    assert lib.kvhip_cache_offset(h) == 0 and lib.kvhip_cache_trim(h, 5) == 0 and lib.kvhip_cache_trim(h, -5) == 0
    assert lib.kvhip_cache_group_size(h) == 64 and lib.kvhip_cache_bits(h) == 8
    assert lib.kvhip_cache_is_trimmable(h, 10) == 1 and lib.kvhip_cache_state_count(h) == 0 and lib.kvhip_cache_meta_count(h) == 1
    assert lib.kvhip_cache_set_offset(h, 1) == -4 and lib.kvhip_cache_set_offset(h, 0) == 0
    assert lib.kvhip_cache_fetch(h, None, None, None) == -4
    lib.kvhip_cache_free(h)
    assert lib.kvhip_cache_create(C.byref(L.Config(kind=4)), C.byref(C.c_void_p())) == -2


def test_refused_before_anything_is_touched():
    lib, h = make()
    p = C.c_void_p(16)
    for args, status in [((2, 2, 1, 128, 128, L.F32), -3), ((2, 2, 1, 257, 128, L.F16), -3), ((2, 2, 1, 128, 300, L.BF16), -3),
                         ((2, 2, 0, 128, 128, L.F16), -2), ((0, 2, 1, 128, 128, L.F16), -2), ((2, 2, 1, 128, 128, L.U32), -2),
                         ((300, 300, 1, 64, 64, L.F16), -3)]:
        assert lib.kvhip_cache_update(h, p, p, *args, None) == status
    assert lib.kvhip_cache_select_blocks(h, p, 1, 1, 1, 64, 1, 0, 1, None, p, None) == -4
    assert lib.kvhip_cache_attend_blocks(h, p, 1, 1, 1, 64, 1.0, p, 1, None, p, None) == -4
    assert lib.kvhip_cache_attend(h, p, 1, 1, 1, 64, 1.0, None, p, None) == -4
    assert lib.kvhip_cache_select_blocks(h, None, 1, 1, 1, 64, 1, 0, 1, None, p, None) == -2
    assert lib.kvhip_cache_update_attend_blocks(h, p, p, p, 1, 3, 2, 1, 64, 64, L.F16, 1.0, 1, 0, 1, None, p, p, None) == -2
    assert lib.kvhip_cache_offset(h) == 0
    lib.kvhip_cache_free(h)
    lib, h = make(L.KIND_SIMPLE)
    for call in (lambda: lib.kvhip_cache_select_blocks(h, p, 1, 1, 1, 64, 1, 0, 1, None, p, None),
                 lambda: lib.kvhip_cache_attend_blocks(h, p, 1, 1, 1, 64, 1.0, p, 1, None, p, None),
                 lambda: lib.kvhip_cache_update_attend_blocks(h, p, p, p, 1, 1, 1, 1, 64, 64, L.F16, 1.0, 1, 0, 1, None, p, p, None)):
        assert call() == -2
    lib.kvhip_cache_free(h)


def test_oracle_codes_are_e4m3():
    """The oracle's rounding against torch's float8_e4m3fn casts, and every code against itself."""
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    codes = codes[np.isfinite(codes)]
    assert np.array_equal(O.e4m3(codes), codes)
    x = np.random.default_rng(0).uniform(-448, 448, 20000) * 2.0 ** np.random.default_rng(1).integers(-20, 1, 20000)
    x = np.concatenate([x, (codes[:-1] + codes[1:]) / 2])
    x = torch.from_numpy(x).float()
    assert np.array_equal(O.e4m3(x.double().numpy()), x.to(torch.float8_e4m3fn).double().numpy())


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_oracle_blocks_are_stored_the_same_twice(dtype):
    rng = np.random.default_rng(2)
    for scale in (1e-6, 1.0, 700.0):
        x = torch.from_numpy(rng.standard_normal((64, 64)) * scale).to(getattr(torch, dtype)).double().numpy()
        codes, e = O.code_block(x, dtype)
        once = codes * 2.0 ** e
        assert np.abs(codes).max() <= 448 and (np.abs(x).max() == 0 or np.abs(codes).max() >= 224)
        assert np.array_equal(torch.from_numpy(once).to(getattr(torch, dtype)).double().numpy(), once)
        codes, e = O.code_block(once, dtype)
        assert np.array_equal(codes * 2.0 ** e, once)
