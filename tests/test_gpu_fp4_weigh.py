"""Attention weights of the 4-bit block cache where keys, queries and scales are far apart, where calls have
more to do than one round of blocks of threads, and where rows are not finite, against numpy in 64 bits
(fp4_ref's bounds)."""
import math

import numpy as np
import pytest
import torch

from fp4_pair import Pair, copy
from test_gpu_fp4_cache import fill_device
from test_gpu_fp8_cache import TORCH, queries, tables

pytestmark = pytest.mark.gpu


def set_exponents(P, side, e):
    P.ref.exps[side] = e
    copy((P.dev.c.d_k_exp, P.dev.c.d_v_exp)[side], torch.from_numpy(np.ascontiguousarray(P.ref.exp_bytes(side))).cuda())


# ---- the keys are those that attention sees ----

@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
def test_weigh_beside_an_infinite_key(hd, dtype, pad):
    """An infinite entry is held as 6 * 2^40: beside it attention sees nothing of the block's other keys, and
    the weights add up to what its softmax does."""
    rng = np.random.default_rng(hd)
    P = Pair(hd, 2, 6)
    P.batch([[4, 2, 0]], [150], [0, 150])
    k = P.rows(rng, "f32")
    k[20, 0, 5], k[75, 1, hd - 1], k[149, 0, 0] = -math.inf, math.inf, math.inf
    P.write("f32", k, P.rows(rng, "f32"))
    P.batch(P.table, [150], [0, 40])
    q = queries(rng, P, 8, dtype)
    q[..., 5], q[..., hd - 1], q[..., 0] = 0, 0, 0  # so that the scores of these keys are no larger than others'
    added = P.check_weigh(dtype, q, 0.4, pad=pad)
    assert abs(added.sum() - 8 * 40) < 1e-2


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
def test_weigh_of_scales_far_apart(hd, dtype):
    """Scales from 2^-20 to 2^-30 of a block's largest: rounded at 2^-24 of it, and scores that show the last bit."""
    rng = np.random.default_rng(hd + 1)
    P = Pair(hd, 1, 8)
    P.batch(tables(rng, [400], 8), [400], [0, 70])
    fill_device(rng, P)
    top = 127 + rng.integers(-3, 4, P.ref.exps[0].shape[:2] + (1, 1, 1))
    e = top - rng.integers(20, 31, P.ref.exps[0].shape)
    e[..., 0] = top[..., 0]  # the first 32 channels, which no query has
    set_exponents(P, 0, e)
    for n_q in (4, 1):
        q = torch.from_numpy(rng.standard_normal((70, n_q, hd))).to(TORCH[dtype])
        q[..., :32] = 0
        P.check_weigh(dtype, q, 2.0 ** 21)
    diff = np.abs(P.ref.stored(0, 0, 0) - P.ref.values(0, 0, 0))
    assert diff.max() > 0  # (what attention sees is not what the codes say)


# ---- queries and kq_scale of any size ----

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("qe,ke", [(-118, 0), (-118, 20), (-60, 0), (-60, 20), (-60, -20), (60, 0), (60, 20), (60, -20),
                                   (120, 0), (120, -20)])
def test_weigh_of_queries_of_any_size(qe, ke, dtype):
    """Scores near 1 from queries of 2^qe, keys of 2^ke and the kq_scale that makes up for them."""
    se = -qe - ke - 2
    rng = np.random.default_rng(qe + 200 + ke)
    for hd in (64, 128):
        P = Pair(hd, 1, 6)
        P.batch(tables(rng, [300], 6), [300], [0, 30])
        fill_device(rng, P)
        set_exponents(P, 0, (P.ref.exps[0].astype(int) + ke).astype(np.uint8))
        for n_q in (4, 1):
            q = torch.from_numpy(rng.standard_normal((30, n_q, hd)).clip(-3, 3)).to(TORCH[dtype])
            P.check_weigh(dtype, q * 2.0 ** qe, 2.0 ** se)
            P.check_weigh(dtype, q * 2.0 ** qe, -(2.0 ** se), window=70)


def test_weigh_of_the_largest_queries():
    """bf16 queries next to the largest number, against keys next to theirs: sums that stay within a float."""
    rng = np.random.default_rng(5)
    for hd in (64, 256):
        P = Pair(hd, 1, 4)
        P.batch(tables(rng, [200], 4), [200], [0, 20])
        fill_device(rng, P)
        P.ref.codes[0] = rng.choice([7, 15], P.ref.codes[0].shape)  # 6 and -6
        copy(P.dev.c.d_k_codes, torch.from_numpy(np.ascontiguousarray(P.ref.code_bytes(0))).cuda())
        set_exponents(P, 0, np.full_like(P.ref.exps[0], 127))
        q = torch.full((20, 2, hd), torch.finfo(torch.bfloat16).max, dtype=torch.bfloat16)
        q[:, 1] *= torch.from_numpy(rng.choice([-1.0, 1.0], (20, hd))).bfloat16()
        P.check_weigh("bf16", q, 2.0 ** -133)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_weigh_of_large_scores_beside_each_other(dtype):
    """Scores past 2^12 with many positions within a few units of the largest: channel 0 lifts all of a row's
    scores, the others tell them apart. Both are whole numbers times ln 2, exact in fp32."""
    rng = np.random.default_rng(8)
    P = Pair(64, 1, 6)
    P.batch(tables(rng, [320], 6), [320], [0, 320])
    k = np.zeros((320, 1, 64))
    k[:, 0, 0] = 6.0
    k[:, 0, 32:36] = rng.integers(-1, 2, (320, 4))
    P.write("f32", torch.from_numpy(k).float(), torch.from_numpy(k).float())
    P.batch(P.table, [320], [0, 50])
    q = np.zeros((50, 4, 64))
    q[..., 0] = rng.integers(128, 240, (50, 4)) * 8
    q[..., 32:36] = 1.0
    added = P.check_weigh(dtype, torch.from_numpy(q).to(TORCH[dtype]), float(np.float32(math.log(2))))
    assert abs(added.sum() - 200) < 1.0 and (added > 0).sum() > 100


# ---- more items than the grid has blocks of threads ----

def weigh64(P, q, scale, lse, window):
    """fp4_ref.RefCache.weigh, a sequence at a time."""
    w, tol = np.zeros_like(P.ref.weight), np.zeros_like(P.ref.weight)
    group = q.shape[1] // P.heads
    split = 2.0 ** -22 if q.dtype == torch.float32 else 0.0
    x = q.double().numpy()
    for i, n in enumerate(P.lens):
        r0, r1 = P.row[i], P.row[i + 1]
        p = n - r1 + np.arange(r0, r1)
        for j, b in enumerate(P.table[i]):
            if not 0 <= b < P.n_blocks or j * 64 >= n or r1 == r0:
                continue
            K, pos = P.ref.values(0, 0, b), j * 64 + np.arange(64)
            see = pos[None] <= p[:, None]
            if window:
                see &= pos[None] > p[:, None] - window
            for h in range(P.heads):
                qh, lh = x[r0:r1, h * group:(h + 1) * group], lse[r0:r1, h * group:(h + 1) * group, None]
                fine = (np.isfinite(lh) & np.isfinite(qh).all(-1, keepdims=True) & see[:, None]).astype(bool)
                qh, lh = np.where(np.isfinite(qh), qh, 0.0), np.where(np.isfinite(lh), lh, 0.0)
                d, steep = qh @ K[h].T * scale - lh, np.abs(qh) @ np.abs(K[h]).T * abs(scale)
                add = np.where(fine, np.exp(np.where(fine, d, 0.0)), 0.0)
                off = steep * ((P.hd + 4) * 2.0 ** -24 + split) + np.abs(d) * 3 * 2.0 ** -24 + 2.0 ** -22
                w[0, b, h] += add.sum((0, 1))
                tol[0, b, h] += (add * (1.01 * off + (r1 - r0) * group * 2.0 ** -24) + fine * 2.0 ** -126).sum((0, 1))
    return w, tol


def check64(P, dtype, q, scale, window=0, pad=0, shift=0, lse=None):
    if lse is None:
        _, lse = P.attend(dtype, q, scale, window)
    before = P.weights()
    P.weigh(dtype, q, scale, lse, window, pad=pad, shift=shift)
    want, tol = weigh64(P, q, float(np.float32(scale)), np.asarray(lse, np.float64), window)
    tol += (tol > 0) * np.abs(before + want) * 2.0 ** -23
    d = np.abs(P.weights() - before - want)
    assert (d <= tol).all(), (float((d - tol).max()), float(d.max()))


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype,pad", [("f32", 1), ("f16", 0), ("bf16", 0), ("bf16", 4)])
def test_weigh_second_items(hd, dtype, pad):
    """32 heads leave 32 blocks of threads a head; these sequences have 60 items, of one, two and three
    stages of columns, some of blocks that the table lacks, so that each block of threads goes on to others."""
    rng = np.random.default_rng(hd + pad)
    lens = [1290 - 37 * i for i in range(20)]
    rows = [(i * 29) % 13 for i in range(20)]
    rows[3], rows[4], rows[11], rows[17] = 150, 290, 129, 64
    P = Pair(hd, 32, 330)
    table = tables(rng, lens, 330)
    table[4][2], table[9][0], table[19][-1] = -1, 9999, -7
    P.batch(table, lens, np.concatenate([[0], np.cumsum(rows)]).tolist(), sum(rows) + 3)
    fill_device(rng, P)
    q = queries(rng, P, 32, dtype)
    check64(P, dtype, q, 0.1, window=0 if hd > 96 else 700, pad=pad)


# ---- rows that are not finite ----

@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype,pad,shift", [("f32", 0, 0), ("f32", 3, 1), ("f16", 0, 0), ("f16", 4, 4), ("f16", 3, 1),
                                             ("bf16", 0, 0), ("bf16", 5, 0)])
def test_weigh_passes_over_what_is_not_finite_in_every_form(hd, dtype, pad, shift):
    rng = np.random.default_rng(hd)
    for heads, lens, rows in ((2, [300, 200], [20, 20]), (32, [700] * 5, [9, 0, 30, 1, 5])):
        P = Pair(hd, heads, 64)
        P.batch(tables(rng, lens, 64), lens, np.concatenate([[0], np.cumsum(rows)]).tolist())
        fill_device(rng, P)
        q = queries(rng, P, 2 * heads, dtype)
        _, lse = P.attend(dtype, q, 0.2)
        for r, n, d, x in ((5, 1, 3, math.nan), (31, 0, 0, math.inf), (32, 1, hd - 1, -math.inf), (8, 2 * heads - 1, 32, math.nan),
                           (8, 2 * heads - 2, hd - 1, math.inf)):
            q[r, n, d] = x
        q[33, 3, 1], q[33, 3, 2] = math.inf, -math.inf
        lse[7, 2], lse[8, 0], lse[9, 3] = np.nan, np.inf, -np.inf
        check64(P, dtype, q, 0.2, pad=pad, shift=shift, lse=lse)
        assert np.isfinite(P.weights()).all()


# ---- rows at any address ----

@pytest.mark.parametrize("hd", [64, 96, 128, 256])
def test_weigh_of_rows_at_any_address(hd):
    """float32 rows at every multiple of their element's size: the same bits."""
    rng = np.random.default_rng(hd)
    P = Pair(hd, 2, 12)
    P.batch(tables(rng, [300, 200], 12), [300, 200], [0, 40, 45])
    fill_device(rng, P)
    q = queries(rng, P, 8, "f32")
    _, lse = P.attend("f32", q, 0.1)
    got = []
    for shift, pad in ((0, 0), (4, 0), (4, 4), (2, 6), (1, 0), (0, 1), (3, 5)):
        P.set_weights(np.zeros(P.ref.weight.shape))
        P.weigh("f32", q, 0.1, lse, pad=pad, shift=shift)
        got.append(P.weights())
    assert all(np.array_equal(x, got[0]) for x in got[1:])


# ---- how exact a weight is ----

@pytest.mark.parametrize("dtype,pad", [("f32", 0), ("f16", 0), ("bf16", 0), ("bf16", 3)])
@pytest.mark.parametrize("scale", [0.125, 0.1, -0.3, 0.7071])
def test_weigh_to_the_last_bits(scale, dtype, pad):
    """Scores near 60 that are whole numbers times kq_scale, exact in fp32: what is left is the exponential of the
    difference to lse. In powers of two that difference e is rounded once, 2^-24 |e|, and kq_scale log2 e's own rounding counts
    on it alone, 2^-24 |e| more; the exponential and the factor that takes up what kq_scale, lse and log2 e lose in 32 bits are
    within 2^-22 each, their product and the sum 2^-23."""
    rng = np.random.default_rng(int(abs(scale) * 1000))
    P = Pair(64, 2, 24)
    lens = [130, 64, 200, 77, 150, 99]
    table = tables(rng, lens, 24)
    top = round(60 / abs(scale))
    k = np.zeros((sum(lens), 2, 64))
    k[..., 0] = 6.0 if scale > 0 else -6.0
    k[..., 32:40] = rng.integers(0, 2, k[..., 32:40].shape)
    P.batch(table, lens, np.concatenate([[0], np.cumsum(lens)]).tolist())
    P.write("f32", torch.from_numpy(k).float(), torch.from_numpy(k).float())
    P.batch(table, lens)
    q = np.zeros((len(lens), 2, 64))
    q[..., 0] = (top + rng.integers(-8, 9, q.shape[:2])) // 6
    q[..., 32:40] = rng.integers(-2, 3, q[..., 32:40].shape)
    q = torch.from_numpy(q).to(TORCH[dtype])
    _, lse = P.attend(dtype, q, scale)
    assert (np.abs(lse) > 45).all()
    P.weigh(dtype, q, scale, lse, pad=pad)
    got, s = P.weights()[0], float(np.float32(scale))
    for i, n in enumerate(lens):
        for h in range(2):
            K = np.concatenate([P.ref.stored(0, 0, b)[h] for b in table[i]])[:n]
            w = np.exp(K @ q[i, h].double().numpy() * s - lse[i, h])
            have = np.concatenate([got[b, h] for b in table[i]])[:n]
            off = np.abs(np.log2(w)) * 2.0 ** -23 * math.log(2) + 2 * 2.0 ** -22 + 2.0 ** -23
            assert (np.abs(have - w) <= off * w).all(), float((np.abs(have / w - 1) / off).max())
