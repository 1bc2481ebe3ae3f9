"""Which way a call of the gated delta rule goes: a workspace is asked for where it goes through chunks."""
import ctypes as C

import pytest

import kvhip
from kvhip import _lib as L


def chunks(tokens, B, Hv, Dk, dtype):
    x = L.GatedDelta(B=B, L=tokens, Hk=Hv, Hv=Hv, Dk=Dk, Dv=Dk, dtype=dtype, gate_dtype=L.F32)
    return kvhip.load().kvhip_gated_delta_workspace(C.byref(x)) > 0


@pytest.mark.parametrize("dtype", [L.F16, L.BF16])
@pytest.mark.parametrize("B, Hv, Dk, tokens", [(1, 32, 128, 10), (2, 16, 64, 10), (1, 33, 128, 14), (4, 32, 96, 14), (8, 32, 128, 20), (64, 32, 128, 20),
                                               (2, 4, 256, 7), (4, 8, 192, 11), (64, 4, 256, 14)])
def test_single_tokens_up_to_where_chunks_are_faster(dtype, B, Hv, Dk, tokens):
    assert not any(chunks(n, B, Hv, Dk, dtype) for n in range(1, tokens + 1))
    assert all(chunks(n, B, Hv, Dk, dtype) for n in (tokens + 1, 64, 1000))
    assert not chunks(1000, B, Hv, Dk, L.F32)
