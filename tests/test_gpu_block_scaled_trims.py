"""Rows taken off a block-scaled cache again: what is left is as if the others had never been written."""
import numpy as np
import pytest
import torch

import kvhip
from oracle import block_scaled as O
from test_gpu_block_scaled import causal, check, check_rows, exact_and_bound, pair
from util import NAME, randn

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
SIZES = [(128, 128), (96, 96), (192, 128), (50, 36)]


class Pair:
    """Two caches: one that has drafts written and rejected, and one that only ever has the rows that stay."""

    def __init__(self, dtype, sizes, seed, B=2, H=2):
        self.dtype, self.sizes, self.shape = dtype, sizes, (B, H)
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.cache, self.alone = kvhip.BlockScaledKVCache(), kvhip.BlockScaledKVCache()

    def rows(self, n, size=1.0):
        return [(torch.randn(*self.shape, n, d, generator=self.gen, device="cuda") * size).to(self.dtype) for d in self.sizes]

    def both(self, n, size=1.0):
        k, v = self.rows(n, size)
        for c in (self.cache, self.alone):
            c.update(k, v, fetch=False)

    def same(self, heads=4):
        """The rows, the attention over them and the blocks chosen among them."""
        assert self.cache.offset == self.cache.presented_length == self.alone.offset
        if self.cache.offset == 0:
            return
        for a, b in zip(self.cache.fetch(), self.alone.fetch()):
            assert torch.equal(a, b)
        q = torch.randn(self.shape[0], heads, 1, self.sizes[0], generator=self.gen, device="cuda").to(self.dtype)
        assert torch.equal(self.cache.attend(q, 0.1), self.alone.attend(q, 0.1))
        count = max(1, self.cache.offset // 128)
        assert torch.equal(self.cache.select_blocks(q, count, 0, 1), self.alone.select_blocks(q, count, 0, 1))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("held", [61, 62, 63, 64, 190])
@pytest.mark.parametrize("size", [1e-3, 1.0, 1000.0])
@pytest.mark.parametrize("one_by_one", [False, True])
def test_rejected_drafts_leave_no_trace(dtype, sizes, held, size, one_by_one):
    """Four drafts, of them 0 to 3 accepted, round after round over block ends: drafts much larger and much smaller than the rows
    before them, in one call or token by token."""
    p = Pair(dtype, sizes, held)
    p.both(held, 0.01)
    p.same()
    for accepted in (1, 0, 3, 2, 0, 3, 3, 1):
        k, v = p.rows(4, size)
        k[:, :, :accepted] *= 0.01 / size  # (what stays is like the rows before it)
        v[:, :, :accepted] *= 0.01 / size
        if one_by_one:
            for i in range(4):
                p.cache.update(k[:, :, i:i + 1], v[:, :, i:i + 1], fetch=False)
        else:
            p.cache.update(k, v, fetch=False)
        assert p.cache.trim(4 - accepted) == 4 - accepted
        if accepted:
            p.alone.update(k[:, :, :accepted], v[:, :, :accepted], fetch=False)
        p.same()
    p.both(60, 0.01)
    p.same()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("held,new", [(1000, 300), (40, 64), (63, 130), (100, 28), (1, 63), (127, 1), (64, 200), (130, 1000)])
def test_a_call_taken_back_and_made_again(dtype, sizes, held, new):
    p = Pair(dtype, sizes, held + new)
    p.both(held, 0.01)
    for size in (100.0, 1e-3, 1.0):
        k, v = p.rows(new, size)
        p.cache.update(k, v, fetch=False)
        assert p.cache.trim(new) == new
        p.same()
    p.both(new)
    p.same()
    p.both(70)
    p.same()


@pytest.mark.parametrize("lengths,cut", [([200], 30), ([200], 71), ([128], 1), ([128], 63), ([70, 70], 70), ([70, 70], 12), ([64, 64, 1], 60),
                                         ([10, 300], 300), ([100] + [1] * 40, 50), ([300, 20, 2], 60)])
def test_back_into_the_block_finished_last(lengths, cut):
    """Rows of the last block that was finished are still there as they came, also where one call brought the whole block."""
    p = Pair(BF16, (128, 128), cut)
    total, made = sum(lengths), 0
    left = total - cut
    for n in lengths:
        k, v = p.rows(n, 0.01 if made < left else 50.0)
        if made < left < made + n:
            k[:, :, left - made:] *= 5000
            v[:, :, left - made:] *= 5000
        p.cache.update(k, v, fetch=False)
        stay = min(n, max(left - made, 0))
        if stay:
            p.alone.update(k[:, :, :stay], v[:, :, :stay], fetch=False)
        made += n
    for _ in range(cut // 2):
        assert p.cache.trim(1) == 1
    p.cache.offset = left
    p.same()
    other, p.cache = p.cache, p.cache.copy()
    p.same()
    for n in (1, 2, 61, 70):
        k, v = p.rows(n)
        for c in (p.cache, p.alone, other):
            c.update(k, v, fetch=False)
        p.same()
        for a, b in zip(other.fetch(), p.alone.fetch()):
            assert torch.equal(a, b)


def test_steps_behind_a_rejected_draft():
    """The attention kernel writes its token into the block that a trim opened again."""
    p = Pair(F16, (128, 128), 5)
    p.both(60, 0.01)
    for _ in range(20):
        p.cache.update(*p.rows(6, 300.0), fetch=False)
        assert p.cache.trim(6) == 6
        k, v = p.rows(1)
        q = torch.randn(2, 8, 1, 128, generator=p.gen, device="cuda").to(F16)
        assert torch.equal(p.cache.update_attend(q, k, v, 0.1), p.alone.update_attend(q, k, v, 0.1))
        p.same()


@pytest.mark.parametrize("held_rows", [63, 62, 9023])
def test_captured_drafts_replay_and_are_rejected(held_rows):
    """A captured update that finishes a block, replayed with other rows each time: the last one's are what the cache holds,
    and behind a trim the rows before them are as they came."""
    p = Pair(BF16, (128, 128), held_rows)
    p.both(held_rows, 0.01)
    k, v = p.rows(3)
    p.cache.update(k, v, fetch=False)  # (pages are there from here on)
    p.cache.trim(3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.cache.update(k, v, fetch=False)
    for size in (1.0, 1000.0, 1e-3):
        for dst, src in zip((k, v), p.rows(3, size)):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        p.alone.update(k, v, fetch=False)
        p.same()
        p.alone.trim(3)
    p.cache.trim(3)
    p.same()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("seed", range(6))
def test_random_schedules(dtype, seed):
    """Calls of any length and trims to anywhere -- also into blocks of which only codes are left -- against the oracle, rows, whole
    attention and chosen blocks."""
    rng = np.random.default_rng(100 + seed)
    sizes = [(64, 64), (50, 36), (192, 128)][seed % 3]
    make = pair(dtype, rng, 1, 2, sizes)
    cache, oracle = kvhip.BlockScaledKVCache(), O.BlockScaledCache(NAME[dtype])
    for i in range(40):
        if oracle.offset and rng.random() < 0.45:
            cut = int(rng.choice([1, 3, 64, rng.integers(1, oracle.offset + 1)]))
            cut = min(cut, oracle.offset)
            assert cache.trim(cut) == cut
            oracle.trim(cut)
        else:
            n = int(rng.choice([1, 1, 4, 63, 64, rng.integers(1, 300)]))
            (k, kd), (v, vd) = make(n)
            if rng.random() < 0.3:
                k, v, kd, vd = (x * 64 for x in (k, v, kd, vd))
            cache.update(kd, vd, fetch=False)
            oracle.update(k, v)
        if oracle.offset == 0:
            continue
        check_rows(cache, oracle)
        q, qd = randn(rng, (1, 4, 1, sizes[0]), dtype, 0.1)
        check(cache.attend(qd, 0.1), *exact_and_bound(q, oracle, 0.1, causal(oracle.offset, 1, [0])))
        blocks = cache.select_blocks(qd, 3, 0, 1)
        assert np.array_equal(blocks.cpu().numpy(), O.select(q, oracle, 3, 0, 1, [0]))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_choices_of_copies_and_of_caches_filled_from_a_state(dtype):
    """A copy chooses as its source does.  A cache filled from a state holds the same values and chooses by what it was filled with: blocks
    whose largest element was rounded down have half the scale there."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    k = torch.randn(1, 2, 64 * 40, 64, generator=gen, device="cuda")
    k[..., 7] *= 8
    top = k.unflatten(2, (40, 64)).abs().amax((3, 4), keepdim=True)
    k = (k.unflatten(2, (40, 64)) * (228.0 / 128 / top)).flatten(2, 3).to(dtype)  # (every block's largest: 228 of 2^-7)
    cache, filled = kvhip.BlockScaledKVCache(), kvhip.BlockScaledKVCache()
    cache.update(k, k, fetch=False)
    copy = cache.copy()
    filled.state = cache.state
    first, again = O.BlockScaledCache(NAME[dtype]), O.BlockScaledCache(NAME[dtype])
    first.update(*[k.double().cpu().numpy()] * 2)
    again.update(first.keys, first.values)
    scales = [[c.codes[0, 0, i][1] for i in range(40)] for c in (first, again)]
    assert all(a == b + 1 for a, b in zip(*scales))
    for c in (copy, filled):
        for a, b in zip(c.fetch(), cache.fetch()):
            assert torch.equal(a, b)
    q = torch.randn(1, 4, 9, 64, generator=gen, device="cuda").to(dtype)
    qn = q.double().cpu().numpy()
    got = cache.select_blocks(q, 6, 0, 1)
    assert torch.equal(got, copy.select_blocks(q, 6, 0, 1))
    assert np.array_equal(got.cpu().numpy(), O.select(qn, first, 6, 0, 1, [0]))
    assert np.array_equal(filled.select_blocks(q, 6, 0, 1).cpu().numpy(), O.select(qn, again, 6, 0, 1, [0]))
