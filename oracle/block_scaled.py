"""The block-scaled cache and attention over chosen blocks in float64 numpy: test infrastructure only.

Written from the definition in include/kvhip.h; there is no counterpart in the reference, so nothing here is pinned to it.
Arrays are [B, Hkv, T, D] of numbers that the cache's dtype holds ("float16" or "bfloat16").
"""
import numpy as np

BLOCK = 64
LARGEST = {"float16": 61440.0, "bfloat16": 1.875 * 2.0 ** 127}


def exponent(a, limit, least=None):
    """The least integer e with a 2^-e <= limit; 0 for a = 0."""
    if a == 0:
        return 0
    e = int(np.floor(np.log2(a / limit))) - 1
    while a > limit * 2.0 ** e:
        e += 1
    return e if least is None else max(e, least)


def e4m3(x):
    """Nearest e4m3 number, ties to even, of numbers up to 448."""
    size = np.floor(np.log2(np.maximum(np.abs(np.where(np.isnan(x), 1.0, x)), 2.0 ** -6)))
    step = 2.0 ** (size - 3)
    return np.rint(x / step) * step


def code_block(x, dtype):
    """[64, D] -> (codes as numbers, exponent)."""
    x = np.where(np.isinf(x), np.nan, np.clip(x, -LARGEST[dtype], LARGEST[dtype]))
    a = float(np.max(np.where(np.isnan(x), 0.0, np.abs(x))))
    e = exponent(a, 448.0, -100)
    return e4m3(x * 2.0 ** -e), e


class BlockScaledCache:
    """Rows as they are read back, block by block.  Of some blocks the rows are kept as they came: of the unfinished one, the one in
    front of it and the one that was unfinished before the last update."""

    def __init__(self, dtype):
        self.dtype, self.keys, self.values, self.coded = dtype, None, None, 0
        self.codes = {}  # (b, h, block) -> (codes of the keys, exponent)
        self.kept = {}   # block -> (its first rows' keys, values)

    @property
    def offset(self):
        return 0 if self.keys is None else self.keys.shape[2]

    def trim(self, n):
        left = self.offset - n
        block, rows = left // BLOCK, left % BLOCK
        arrays = [x[:, :, :left] for x in (self.keys, self.values)]
        if rows and block in self.kept and self.kept[block][0].shape[2] >= rows:
            arrays = [np.concatenate([x[:, :, :left - rows], raw[:, :, :rows]], 2) for x, raw in zip(arrays, self.kept[block])]
            self.coded = min(self.coded, block)
        elif not rows:
            self.coded = min(self.coded, block)
        self.keys, self.values = arrays

    def update(self, keys, values):
        before = self.offset
        begun = before // BLOCK
        unfinished = before % BLOCK > 0 and self.coded == begun
        new = [np.where(np.isinf(x), np.nan, np.asarray(x, dtype=np.float64)) for x in (keys, values)]
        rows = [n if h is None else np.concatenate([h, n], 2) for h, n in zip((self.keys, self.values), new)]
        self.coded = rows[0].shape[2] // BLOCK

        def raw(block, end):
            return [x[:, :, block * BLOCK:end].copy() for x in rows]

        kept = {self.coded - 1: self.kept[self.coded - 1]} if self.coded == begun and self.coded - 1 in self.kept else {}
        if unfinished:
            kept[begun] = raw(begun, before)
        if self.coded > begun:
            kept[self.coded - 1] = raw(self.coded - 1, self.coded * BLOCK)
        if rows[0].shape[2] % BLOCK:
            kept[self.coded] = raw(self.coded, rows[0].shape[2])
        self.kept = kept
        for which, x in enumerate(rows):
            for b in range(x.shape[0]):
                for h in range(x.shape[1]):
                    for c in range(begun, self.coded):
                        codes, e = code_block(x[b, h, c * BLOCK:(c + 1) * BLOCK], self.dtype)
                        x[b, h, c * BLOCK:(c + 1) * BLOCK] = codes * 2.0 ** e
                        if which == 0:
                            self.codes[b, h, c] = codes, e
        self.keys, self.values = rows


def bounds(queries, cache):
    """[B, Hkv, L, coded] bounds of each token on each whole block."""
    B, Hq, L, D = queries.shape
    Hkv = cache.keys.shape[1]
    G = Hq // Hkv
    out = np.full((B, Hkv, L, cache.coded), -np.inf)
    for b in range(B):
        for h in range(Hkv):
            ends = []
            for c in range(cache.coded):
                codes, e = cache.codes[b, h, c]
                units = np.rint(codes / 4)
                some = ~np.isnan(units).all(0)
                hi, lo = np.zeros(units.shape[1]), np.zeros(units.shape[1])
                hi[some], lo[some] = np.nanmax(units[:, some], 0), np.nanmin(units[:, some], 0)
                ends.append((hi, lo, 2.0 ** (e + 2)))
            for q in range(G):
                for t in range(L):
                    x = np.nan_to_num(queries[b, h * G + q, t].astype(np.float64), nan=0.0, posinf=0.0, neginf=0.0)
                    f = exponent(float(np.abs(x).max()), 127.0)
                    i = np.rint(x * 2.0 ** -f)
                    for c, (hi, lo, unit) in enumerate(ends):
                        out[b, h, t, c] = max(out[b, h, t, c], np.maximum(i * hi, i * lo).sum() * unit * 2.0 ** f)
    return out


def select(queries, cache, count, first, recent, pads):
    B, Hq, L, D = queries.shape
    bound = bounds(queries, cache)
    T, Hkv = cache.offset, cache.keys.shape[1]
    out = np.full((B, Hkv, L, count), -1, dtype=np.int32)
    for b in range(B):
        for t in range(L):
            p = T - L + t
            if p < pads[b]:
                continue
            lead, last = pads[b] // BLOCK, p // BLOCK
            for h in range(Hkv):
                rest = [c for c in range(lead, last + 1) if not (c < lead + first or c > last - recent)]
                chosen = [c for c in range(lead, last + 1) if c not in rest]
                chosen += sorted(rest, key=lambda c: (-bound[b, h, t, c], c))[:count - len(chosen)]
                out[b, h, t, :len(chosen)] = sorted(chosen)
    return out


def listed_keep(blocks, T, pads):
    """Which keys [B, Hkv, L, T] the tokens of a list [B, Hkv, L, count] attend over, as often as each is listed."""
    B, Hkv, L, count = blocks.shape
    keep = np.zeros((B, Hkv, L, T))
    for b in range(B):
        for h in range(Hkv):
            for t in range(L):
                p, before = T - L + t, None
                for c in blocks[b, h, t]:
                    lo, hi = max(int(c) * BLOCK, pads[b]), min(int(c) * BLOCK + BLOCK - 1, p)
                    if c >= pads[b] // BLOCK and lo <= hi and (before is None or c > before):
                        keep[b, h, t, lo:hi + 1] += 1
                    before = int(c)
    return keep
