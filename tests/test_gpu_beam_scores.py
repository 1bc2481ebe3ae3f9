"""Selection where bounds have little to tell candidates apart by: accumulated scores far from zero and close together, logits far from
zero, as many candidates as are allowed, equal ones by the thousand."""
import pytest
import torch

import kvhip
from tests.test_gpu_beams import DTYPES, check_select

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("own", [-100.0, -300.0, -1e4])
@pytest.mark.parametrize("B, K, V, count", [(3, 8, 30011, 8), (2, 16, 20000, 32), (1, 16, 70001, 64), (1, 64, 9001, 64), (9, 4, 9000, 4)])
def test_beams_a_few_nats_apart(dtype, own, B, K, V, count):
    gen = torch.Generator(device="cuda").manual_seed(V)
    x = (2.5 * torch.randn(B, K, V, generator=gen, device="cuda")).to(dtype)
    scores = own - 3 * torch.rand(B, K, generator=gen, device="cuda")
    check_select(x, scores, count)
    check_select(x, scores, count, torch.rand(B, K, generator=gen, device="cuda") < 0.3, 7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift", [1000.0, -1000.0, 30000.0])
@pytest.mark.parametrize("B, K, V, count", [(2, 4, 40000, 4), (1, 3, 20011, 64)])
def test_shifted_logits(dtype, shift, B, K, V, count):
    """A row's logits all shifted by the same: what they score does not change but by their rounding."""
    gen = torch.Generator(device="cuda").manual_seed(V)
    x = (2.5 * torch.randn(B, K, V, generator=gen, device="cuda") + shift).to(dtype)
    check_select(x, -5 * torch.rand(B, K, generator=gen, device="cuda"), count)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count", [1, 33, 64])
def test_equal_candidates_by_the_thousand(dtype, count):
    """Beams whose candidates are all alike, or all but a few: nothing but the order of beams and tokens is left to choose by."""
    for K, V in ((64, 700), (64, 33000), (7, 20001)):
        x = torch.zeros(1, K, V, dtype=dtype, device="cuda")
        check_select(x, None, count)
        check_select(x, torch.full((1, K), -200.0, device="cuda"), count)
        x[0, :, V - 3] = 0.5
        x[0, K - 1, 5] = 0.5
        check_select(x, torch.full((1, K), -200.0, device="cuda"), count)
        x[:] = -float("inf")
        x[0, 2, ::3] = 1.0
        check_select(x, torch.zeros(1, K, device="cuda"), count)
    x = torch.randint(0, 2, (2, 64, 3000), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(dtype)
    check_select(x, torch.randint(-3, 0, (2, 64), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").float(), count)


def test_many_candidates_in_a_graph():
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, scores = torch.randn(2, 16, 40000, generator=gen, device="cuda").bfloat16(), -100 - torch.rand(2, 16, generator=gen, device="cuda")
    kvhip.beam_select(x, scores, 64)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = kvhip.beam_select(x, scores, 64)
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, check_select(x, scores, 64)))
        x.copy_(torch.randn(2, 16, 40000, generator=gen, device="cuda"))
        torch.cuda.synchronize()
