"""The 8-bit block cache's attention over the range of scores that its calls accept, against the
numpy form in 64 bits.

With kq_scale the float nearest to ln 2 a score counts in powers of two, so that scores which are
whole numbers are exact in the kernels (fp32 holds every product and sum below: each is a multiple of
the last bit that a float of its size has) and exact in the numpy form with ln 2 itself. What is then
left of fp8_ref.bounds is its part that does not come from the scores."""
import math

import numpy as np
import pytest
import torch

import fp8_ref as R
from test_gpu_fp8_cache import TORCH, Pair

pytestmark = pytest.mark.gpu

LN2 = float(np.float32(math.log(2)))
assert np.float32(LN2) * np.float32(1.4426950408889634) == 1.0  # the factor of the kernels' exponents
KE = 8  # K's values count in 2^KE, so that fp16 queries reach large scores

# M * 2^(E - 7) is the smallest of the large scores, with M in [128, 240): fp32 counts in 2^(E - 23) there
TOPS = [(131, 19), (128, 20), (160, 25), (200, 25), (176, 26), (160, 27), (150, 29)]


def step_of(E):
    """Distance of the scores: a float's last bit there, at least 1 (a weight half as large)."""
    return max(2.0 ** (E - 23), 1.0)


def check(P, dtype, q, window=0):
    """P.check_attend for scores that are exact."""
    out, lse = P.attend(dtype, q, LN2, window)
    want, wlse, reach, steep = P.ref.attend(0, P.table, P.lens, P.row, P.n_rows, q.double().numpy(), math.log(2), window)
    tol, ltol = R.bounds(dtype, P.hd, max(P.lens), want, reach, 0 * steep)
    assert np.isfinite(out).all() and np.isfinite(lse).all(), "a finite row came out infinite or NaN"
    d, dl = np.abs(out - want), np.abs(lse - wlse)
    assert (d <= tol).all(), (float((d - tol).max()), float(d.max()))
    assert (dl <= ltol + 2.0 ** -23 * np.abs(wlse)).all(), float((dl - 2.0 ** -23 * np.abs(wlse)).max())


def fill(P, rng, length, grade, large=lambda block: np.full(block.shape, 256.0)):
    """K: channel 0 makes a score large (by block), channel 1 grades it; V: strength by block."""
    block = np.arange(length) // 64
    k = np.zeros((length, 1, P.hd))
    k[:, 0, 0], k[:, 0, 1] = large(block), grade(block, np.arange(length))
    v = rng.standard_normal((length, 1, P.hd)) * 2.0 ** ((block * 5) % 13 - 6.0)[:, None, None]
    P.batch([rng.permutation(P.n_blocks).tolist()], [length], [0, length])
    P.write("f32", torch.from_numpy(k * 2.0 ** KE).float(), torch.from_numpy(v).float())


def large_queries(n, n_q, hd, M, E, sign, dtype):
    """Row r, head h: score (M + (r + h) % 14) 2^(E - 7) of channel 0's 256, one step for each of channel 1's 1."""
    q = np.zeros((n, n_q, hd))
    rh = np.arange(n)[:, None] + np.arange(n_q)[None]
    q[..., 0] = sign * (M + rh % 14) * 2.0 ** (E - 7 - 8 - KE)
    q[..., 1] = step_of(E) * 2.0 ** -KE
    t = torch.from_numpy(q).to(TORCH[dtype])
    assert (t.double().numpy() == q).all()
    return t


GRADES = {"within": lambda block, t: (t * 7) % 4 + (t % 64 == 17), "rising": lambda block, t: np.minimum(block // 4, 15)}


@pytest.mark.parametrize("length", [300, 2560])  # 2560: in shares, joined
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("M,E", TOPS)
def test_large_scores(M, E, sign, length):
    """The kernel for few rows: one row, a few, and more than 16 columns a wave."""
    rng = np.random.default_rng(E)
    for hd, grade in ((64, "within"), (256, "rising")):
        P = Pair(hd, 1, (length + 63) // 64)
        fill(P, rng, length, GRADES[grade])
        for dtype in ("f16", "bf16", "f32"):
            for row, n_q in ((None, 3), ([0, 4], 3), ([0, 9], 4)):
                P.batch(P.table, [length], row)
                check(P, dtype, large_queries(P.n_rows, n_q, hd, M, E, sign, dtype))


@pytest.mark.parametrize("length", [300, 2560])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("M,E", TOPS)
def test_large_scores_of_many_columns(M, E, sign, length):
    """The kernel for many rows, its waves of 32 columns and of 16."""
    rng = np.random.default_rng(E)
    for hd in (64, 256):
        P = Pair(hd, 1, (length + 63) // 64)
        fill(P, rng, length, GRADES["within"])
        for dtype in ("bf16", "f32"):
            n = {(64, "bf16"): 129, (64, "f32"): 65}.get((hd, dtype), 65)  # 8256 columns, else 4160
            P.batch(P.table, [length], [0, n])
            check(P, dtype, large_queries(n, 64, hd, M, E, sign, dtype))


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("M,E", TOPS)
def test_large_scores_in_rising_shares(M, E, sign):
    """The shares of the kernel for many rows have maxima of their own, a step or more apart."""
    rng = np.random.default_rng(E)
    for hd in (64, 256):
        P = Pair(hd, 1, 40)
        fill(P, rng, 2560, GRADES["rising"])
        P.batch(P.table, [2560], [0, 129 if hd == 64 else 65])
        for dtype in ("f16", "bf16", "f32"):
            check(P, dtype, large_queries(P.n_rows, 64, hd, M, E, sign, dtype))


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("M,E", [(128, 20), (160, 25), (160, 27)])
def test_scores_small_then_large(M, E, sign):
    """Blocks without channel 0 among blocks with it: the maximum jumps up, or from far below 0 to near it."""
    rng = np.random.default_rng(E)
    for hd in (64, 128):
        P = Pair(hd, 1, 12)
        fill(P, rng, 700, GRADES["within"], lambda block: np.where(np.isin(block, (0, 1, 5, 8)), 0.0, 256.0))
        for dtype in ("bf16", "f32"):
            for row, n_q in ((None, 3), ([0, 9], 4), ([0, 600], 16)):
                for window in (0, 100):
                    P.batch(P.table, [700], row)
                    check(P, dtype, large_queries(P.n_rows, n_q, hd, M, E, sign, dtype), window)


def test_scales_whose_product_is_past_a_float():
    """Finite scores from factors whose scales multiply to more, or whose kq_scale does with log2 e."""
    rng = np.random.default_rng(3)
    k = torch.from_numpy(rng.standard_normal((300, 1, 64))).float()
    k[:, 0, 0] = 0.0
    v = torch.from_numpy(rng.standard_normal((300, 1, 64))).float()
    for ke in (45, -27, -40):
        P = Pair(64, 1, 6)
        P.batch([[3, 0, 1, 2, 5]], [300], [0, 300])
        P.write("f32", k * 2.0 ** ke, v)
        for dtype in ("f32", "bf16"):
            for row, n_q in ((None, 3), ([0, 9], 4), ([0, 300], 32)):
                P.batch(P.table, [300], row)
                q = torch.from_numpy(rng.standard_normal((P.n_rows, n_q, 64))).to(TORCH[dtype])
                first = torch.zeros_like(q)
                first[..., 0] = 2.0 ** 126  # meets zeros alone
                P.check_attend(dtype, q * 0.0, 3.2e38)
                P.check_attend(dtype, first, 0.125)
                P.check_attend(dtype, first, -(2.0 ** 120))
                if ke == -27:  # scores near 1
                    P.check_attend(dtype, q * 2.0 ** -101, 3.2e38)
                    P.check_attend(dtype, q * 2.0 ** 122, 2.0 ** -96)
                if ke == -40:  # scores near 2^104
                    P.check_attend(dtype, q * 2.0 ** 110, 2.0 ** 34)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_neighbours_of_infinite_and_large_queries(dtype):
    """Rows beside one whose query is infinite, or whose scores are past 2^25, are bit for bit what they
    are beside an ordinary one (few rows; one sequence, so that the shares are the same)."""
    rng = np.random.default_rng(12)
    for hd, length in ((64, 300), (256, 2560)):
        P = Pair(hd, 1, (length + 63) // 64)
        P.fill(rng, [list(range(P.n_blocks))], [length], "f32", 0.3)
        for row, n_q in ((None, 4), ([0, 9], 4)):
            P.batch(P.table, [length], row)
            q = torch.from_numpy(rng.standard_normal((P.n_rows, n_q, hd))).to(TORCH[dtype])
            good = P.check_attend(dtype, q, 0.11)
            for much in (float("inf"), -float("inf"), 3e4):  # past 2^25 at the larger scale
                scale = 0.11 if math.isinf(much) else 2.0 ** 11
                bad = q * (0.11 / scale) if scale != 0.11 else q.clone()
                want = good if scale == 0.11 else P.attend(dtype, bad, scale)
                bad[0, 1] = 0.0
                bad[0, 1, 5] = much
                got = P.attend(dtype, bad, scale)
                others = np.ones(q.shape[:2], bool)
                others[0, 1] = False
                assert np.array_equal(got[0][others], want[0][others]), much
                assert np.array_equal(got[1][others], want[1][others]), much
                if math.isinf(much):
                    assert not np.isfinite(got[0][0, 1]).any()
