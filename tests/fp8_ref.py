"""The 8-bit block cache in numpy, 64 bits: what the header says, element by element."""
import numpy as np

BLOCK = 64
EMIN, EMAX = -40, 40
TOP = 448.0 * 2.0 ** EMAX


def numbers():
    """The E4M3 number of each byte (the two NaN bytes as NaN)."""
    out = np.empty(256)
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        v = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out[b] = np.nan if b & 127 == 127 else -v if b & 128 else v
    return out


NUMBERS = numbers()
_POS = NUMBERS[:127]


def code_of(y):
    """The byte of the nearest E4M3 number, ties to the even byte, past 448 that of 448."""
    a = np.minimum(np.abs(y), 448.0)
    hi = np.clip(np.searchsorted(_POS, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - _POS[lo], _POS[hi] - a
    pick = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))
    pick = np.where(_POS[hi] == a, hi, pick)
    return (pick + np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def least_exponent(amax):
    e = EMIN
    while e < EMAX and amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def k_order(hd):
    """[64, hd] byte offsets of K's (position, channel) in a tile."""
    t, d = np.arange(BLOCK)[:, None], np.arange(hd)[None, :]
    return (((t // 32) * (hd // 32) + d // 32) * 64 + (d // 8) % 4 * 16 + t % 16) * 16 + (t // 16) % 2 * 8 + d % 8


def v_order(hd):
    t, d = np.arange(BLOCK)[:, None], np.arange(hd)[None, :]
    return ((d // 16) * 64 + (t // 4) % 4 * 16 + d % 16) * 16 + (t // 16) * 4 + t % 4


class RefCache:
    """Codes [2][layers][blocks][heads][64][hd] in natural order, exponents [2][...][heads]."""

    def __init__(self, hd, layers, heads, n_blocks):
        self.hd, self.heads, self.n_blocks = hd, heads, n_blocks
        self.codes = np.zeros((2, layers, n_blocks, heads, BLOCK, hd), np.uint8)
        self.exps = np.full((2, layers, n_blocks, heads), 127 + EMIN, np.uint8)

    def places(self, table, lens, row, n_rows):
        """(row, block or -1, position in it, position) of every row that a sequence has."""
        for i in range(len(lens)):
            r0, r1 = (row[i], row[i + 1]) if row is not None else (i, i + 1)
            for r in range(r0, r1):
                pos = lens[i] - r1 + r
                j = pos // BLOCK
                b = table[i][j] if 0 <= j < len(table[i]) else -1
                yield i, r, b if 0 <= b < self.n_blocks else -1, pos % BLOCK, pos

    def write(self, layer, table, lens, row, n_rows, k, v):
        groups = {}
        for i, r, b, at, pos in self.places(table, lens, row, n_rows):
            if b >= 0:
                groups.setdefault((i, b), []).append((r, at))
        for (_, b), rows in groups.items():
            lo = min(at for _, at in rows)
            idx, ats = [r for r, _ in rows], [at for _, at in rows]
            for side, x in enumerate((k, v)):
                if x is None:
                    continue
                for h in range(self.heads):
                    y = np.asarray(x[idx, h], np.float64)
                    y = np.clip(np.where(np.isnan(y), 0.0, y), -TOP, TOP)
                    e, old = least_exponent(np.abs(y).max()), int(self.exps[side, layer, b, h]) - 127
                    tile = self.codes[side, layer, b, h]
                    if lo > 0:
                        e = max(e, old)
                        if e > old:
                            tile[:lo] = code_of(NUMBERS[tile[:lo]] * 2.0 ** (old - e))
                    tile[ats] = code_of(y * 2.0 ** -e)
                    self.exps[side, layer, b, h] = e + 127

    def values(self, side, layer, b):
        """[heads, 64, hd]"""
        e = self.exps[side, layer, b].astype(np.float64) - 127
        return NUMBERS[self.codes[side, layer, b]] * 2.0 ** e[:, None, None]

    def tiles(self, side):
        """The device's bytes: [layers, blocks, heads, 64 * hd]."""
        order = (k_order if side == 0 else v_order)(self.hd).reshape(-1)
        c = self.codes[side]
        out = np.empty(c.shape[:3] + (BLOCK * self.hd,), np.uint8)
        out[..., order] = c.reshape(c.shape[:3] + (-1,))
        return out

    def attend(self, layer, table, lens, row, n_rows, q, scale, window):
        """out [n_rows, n_q, hd], lse [n_rows, n_q], and the sums that bound a kernel's errors:
        reach (the weights' mean of |v| in [0], its plain sum in [1]) and steep (the largest
        kq_scale * sum |q| |k| seen)."""
        n_q = q.shape[1]
        group = n_q // self.heads
        out = np.full((n_rows, n_q, self.hd), np.nan)
        lse = np.full((n_rows, n_q), np.nan)
        reach = np.zeros((2, n_rows, n_q, self.hd))
        steep = np.zeros((n_rows, n_q))
        for i in range(len(lens)):
            r0, r1 = (row[i], row[i + 1]) if row is not None else (i, i + 1)
            here = [(j, b) for j, b in enumerate(table[i]) if 0 <= b < self.n_blocks and j * BLOCK < lens[i]]
            pos = np.concatenate([np.arange(BLOCK) + j * BLOCK for j, _ in here]) if here else np.zeros(0, int)
            K = np.concatenate([self.values(0, layer, b) for _, b in here], 1) if here else None
            V = np.concatenate([self.values(1, layer, b) for _, b in here], 1) if here else None
            for r in range(r0, r1):
                p = lens[i] - r1 + r
                see = (pos <= p) & (pos < lens[i])
                if window > 0:
                    see &= pos > p - window
                if not see.any():
                    out[r], lse[r] = 0.0, -np.inf
                    continue
                for h in range(self.heads):
                    qs = q[r, h * group:(h + 1) * group].astype(np.float64)
                    s = qs @ K[h][see].T * scale
                    m = s.max(-1, keepdims=True)
                    w = np.exp(s - m)
                    t = w.sum(-1, keepdims=True)
                    sl = slice(h * group, (h + 1) * group)
                    out[r, sl] = w / t @ V[h][see]
                    reach[0, r, sl] = w / t @ np.abs(V[h][see])
                    reach[1, r, sl] = np.abs(V[h][see]).sum(0)
                    lse[r, sl] = (m + np.log(t))[:, 0]
                    steep[r, sl] = (np.abs(qs) @ np.abs(K[h][see]).T).max(-1) * abs(scale)
        return out, lse, reach, steep


def bounds(dtype, hd, seen, out, reach, steep):
    """How far a kernel's out and lse may be off, from its arithmetic.

    A score (a dot of hd products, summed in fp32 in some order) is off by at most
    (hd + 4) 2^-24 of sum |q| |k| (the four: two scale products, the difference to the maximum
    and log2 e's own rounding), and with a split fp32 query 2^-22 more. Its weight: that, and
    2^-22 for the exponential and the running rescale. Sums of `seen` weights in fp32: seen 2^-24, a rescale
    for every 64. The product with V takes the weights rounded to fp16, 2^-11 (fp32: split, 2^-22),
    and those of the smallest as if they were 2^-18 of the largest (fp16 numbers are normal down to
    2^-14 and count from 2^12 at the largest, from 2^4 in a block whose V scale is 2^8 below
    another's; split ones count from 2^14: 2^-28), and the result is rounded once to its type."""
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    score = steep * ((hd + 4) * 2.0 ** -24 + (2.0 ** -22 if dtype == "f32" else 0.0))
    sums = (seen + seen / 16 + 64) * 2.0 ** -24 + 2.0 ** -22
    lse = score + sums + 2.0 ** -22
    w = 2 * (score + sums) + (2.0 ** -21 if dtype == "f32" else 2.0 ** -11)
    least = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}[dtype]
    reach = reach[0] + (2.0 ** -28 if dtype == "f32" else 2.0 ** -18) * reach[1]
    return w[..., None] * reach + half * np.abs(out) + least, lse
