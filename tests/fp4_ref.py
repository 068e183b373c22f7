"""The 4-bit block cache in numpy, 64 bits: what the header says, element by element."""
import numpy as np

import fp8_ref

BLOCK, GROUP = 64, 32
EMIN, EMAX = -40, 40
TOP = 6.0 * 2.0 ** EMAX
POS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
NUMBERS = np.concatenate([POS, -POS])  # of the sixteen codes


def code_of(y):
    """The code of the nearest E2M1 number, ties to the even code, past 6 that of 6."""
    a = np.minimum(np.abs(y), 6.0)
    hi = np.clip(np.searchsorted(POS, a), 0, 7)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - POS[lo], POS[hi] - a
    pick = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))
    pick = np.where(POS[hi] == a, hi, pick)
    return (pick + np.where(np.signbit(y), 8, 0)).astype(np.uint8)


def exponents(amax):
    e = np.full(amax.shape, EMIN)
    for k in range(EMIN, EMAX):
        e = np.where(amax > 6.0 * 2.0 ** k, k + 1, e)
    return e


def place(p):
    """Of position p's exponent in its plane of 64."""
    return p // 4 % 4 * 16 + p // 16 * 4 + p % 4


class RefCache(fp8_ref.RefCache):
    """Codes [2][layers][blocks][heads][64][hd], biased exponents [...][64][hd / 32], weights
    [layers][blocks][heads][64]. Places and attention are the 8-bit cache's."""

    def __init__(self, hd, layers, heads, n_blocks):
        self.hd, self.heads, self.n_blocks = hd, heads, n_blocks
        self.codes = np.zeros((2, layers, n_blocks, heads, BLOCK, hd), np.uint8)
        self.exps = np.full((2, layers, n_blocks, heads, BLOCK, hd // GROUP), 127 + EMIN, np.uint8)
        self.weight = np.zeros((layers, n_blocks, heads, BLOCK))

    def write(self, layer, table, lens, row, n_rows, k, v):
        for i, r, b, at, pos in self.places(table, lens, row, n_rows):
            if b < 0:
                continue
            for side, x in enumerate((k, v)):
                if x is None:
                    continue
                y = np.asarray(x[r], np.float64)
                y = np.clip(np.where(np.isnan(y), 0.0, y), -TOP, TOP).reshape(self.heads, -1, GROUP)
                e = exponents(np.abs(y).max(-1))
                if at == 0:  # the block starts anew
                    self.exps[side, layer, b] = 127 + EMIN
                self.codes[side, layer, b, :, at] = code_of(y * 2.0 ** -e[..., None]).reshape(self.heads, -1)
                self.exps[side, layer, b, :, at] = e + 127
            if k is not None:
                self.weight[layer, b, :, at] = 0.0

    def stored(self, side, layer, b):
        """[heads, 64, hd]"""
        e = np.repeat(self.exps[side, layer, b].astype(np.float64) - 127, GROUP, -1)
        return NUMBERS[self.codes[side, layer, b]] * 2.0 ** e

    def values(self, side, layer, b):
        """What attention sees of them: multiples of 2^-24 of the block's largest scale."""
        e = np.repeat(self.exps[side, layer, b].astype(np.float64) - 127, GROUP, -1)
        top = e.max((1, 2), keepdims=True)
        return np.round(NUMBERS[self.codes[side, layer, b]] * 2.0 ** (e - top + 24)) * 2.0 ** (top - 24)

    def code_bytes(self, side):
        """The device's bytes: [layers, blocks, heads, 32 * hd]."""
        c = self.codes[side]
        two = c[..., 0::2] | c[..., 1::2] << 4
        two = two.reshape(c.shape[:4] + (self.hd // 8, 4))
        return np.moveaxis(two, 4, 3).reshape(c.shape[:3] + (-1,))

    def exp_bytes(self, side):
        """[layers, blocks, heads, 2 * hd]"""
        e = np.moveaxis(self.exps[side], 4, 3)
        out = np.empty_like(e)
        out[..., place(np.arange(BLOCK))] = e
        return out.reshape(e.shape[:3] + (-1,))

    def weigh(self, layer, table, lens, row, n_rows, q, scale, window, lse):
        """Adds to the weights; how far a kernel's sums may be off, from its arithmetic.

        A score (a dot of hd products, summed in fp32 in some order) is off by at most (hd + 4) 2^-24 of
        sum |q| |k|, with a split fp32 query 2^-22 more; the difference to lse is rounded once, and once
        more times log2 e (its own constant too): 3 2^-24 of it; the exponential 2^-22. A column's weight is off by
        that; n columns are summed in fp32 in some order, n 2^-24, and added to the weight, 2^-24 of what
        comes out. What is below 2^-126 may count as nothing."""
        tol = np.zeros_like(self.weight)
        n_q = q.shape[1]
        group = n_q // self.heads
        split = 2.0 ** -22 if q.dtype == np.float32 else 0.0
        q = q.astype(np.float64)
        for i in range(len(lens)):
            r0, r1 = (row[i], row[i + 1]) if row is not None else (i, i + 1)
            for j, b in enumerate(table[i]):
                if not (0 <= b < self.n_blocks and j * BLOCK < lens[i]):
                    continue
                K = self.values(0, layer, b)
                pos = np.arange(BLOCK) + j * BLOCK
                for r in range(r0, r1):
                    p = lens[i] - r1 + r
                    see = pos <= p
                    if window > 0:
                        see &= pos > p - window
                    for n in range(n_q):
                        if not np.isfinite(lse[r, n]) or not np.isfinite(q[r, n]).all():
                            continue
                        h = n // group
                        d = K[h] @ q[r, n] * scale - lse[r, n]
                        steep = np.abs(K[h]) @ np.abs(q[r, n]) * abs(scale)
                        add = np.where(see, np.exp(d), 0.0)
                        self.weight[layer, b, h] += add
                        off = steep * ((self.hd + 4) * 2.0 ** -24 + split) + np.abs(d) * 3 * 2.0 ** -24 + 2.0 ** -22
                        tol[layer, b, h] += add * (1.01 * off + (r1 - r0) * group * 2.0 ** -24) + see * 2.0 ** -126
        return tol + (tol > 0) * np.abs(self.weight) * 2.0 ** -23

    def evict(self, layer, table, lens, keep, first, recent):
        kept = np.full((len(lens), self.heads, keep), -1, np.int64)
        for i, n in enumerate(lens):
            if n <= keep:
                kept[i, :, :max(n, 0)] = np.arange(max(n, 0))
                continue
            used = (n + BLOCK - 1) // BLOCK
            if used > len(table[i]) or any(not 0 <= b < self.n_blocks for b in table[i][:used]):
                continue
            b = np.array(table[i])[:used]
            for h in range(self.heads):
                w = self.weight[layer, b, h].reshape(-1)[:n]
                inner = np.arange(first, n - recent)
                # by weight, then by position; NaN behind all
                order = sorted(inner, key=lambda p: (np.isnan(w[p]), -w[p] if w[p] == w[p] else 0.0, p))
                stay = sorted(list(range(first)) + order[:keep - first - recent] + list(range(n - recent, n)))
                kept[i, h] = stay
                src = np.array(stay)
                dst = np.arange(keep)
                for x in (self.codes, self.exps):
                    x[:, layer, b[dst // BLOCK], h, dst % BLOCK] = x[:, layer, b[src // BLOCK], h, src % BLOCK].copy()
                self.weight[layer, b[dst // BLOCK], h, dst % BLOCK] = w[src]
                if keep % BLOCK:
                    self.exps[:, layer, b[keep // BLOCK], h, keep % BLOCK:] = 127 + EMIN
        return kept
