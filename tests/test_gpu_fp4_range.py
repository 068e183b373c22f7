"""The 4-bit block cache's attention with scores of any size, and with more sequences than a wave has lanes, against
numpy in 64 bits.

As for the 8-bit cache kq_scale is the float nearest to ln 2 and scores are whole numbers, exact in fp32 and in the
numpy form. What makes a score large and what grades it lie in groups of 32 channels of their own, each with its scale."""
import numpy as np
import pytest
import torch

from fp4_pair import Pair
from test_gpu_fp4_cache import fill_device
from test_gpu_fp8_cache import TORCH, queries, tables
from test_gpu_fp8_range import GRADES, KE, TOPS, check, step_of

pytestmark = pytest.mark.gpu


def fill(P, rng, length, grade, large=lambda block: np.full(block.shape, 256.0)):
    """K: channel 0 makes a score large (by block), channel 32 grades it; V: strength by block."""
    block = np.arange(length) // 64
    k = np.zeros((length, 1, P.hd))
    k[:, 0, 0], k[:, 0, 32] = large(block), grade(block, np.arange(length))
    v = rng.standard_normal((length, 1, P.hd)) * 2.0 ** ((block * 5) % 13 - 6.0)[:, None, None]
    P.batch([rng.permutation(P.n_blocks).tolist()], [length], [0, length])
    P.write("f32", torch.from_numpy(k * 2.0 ** KE).float(), torch.from_numpy(v).float())


def large_queries(n, n_q, hd, M, E, sign, dtype):
    """Row r, head h: score (M + (r + h) % 14) 2^(E - 7) of channel 0's 256, one step for each of channel 32's 1."""
    q = np.zeros((n, n_q, hd))
    rh = np.arange(n)[:, None] + np.arange(n_q)[None]
    q[..., 0] = sign * (M + rh % 14) * 2.0 ** (E - 7 - 8 - KE)
    q[..., 32] = step_of(E) * 2.0 ** -KE
    t = torch.from_numpy(q).to(TORCH[dtype])
    assert (t.double().numpy() == q).all()
    return t


SOME = [TOPS[i] for i in (0, 3, 6)]  # past 2^18, where a float counts in 4, and in 64


@pytest.mark.parametrize("length", [300, 2560])  # 2560: in shares, joined
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("M,E", SOME)
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


@pytest.mark.parametrize("grade,length", [("within", 300), ("rising", 2560)])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("M,E", SOME)
def test_large_scores_of_many_columns(M, E, sign, grade, length):
    """The kernel for many rows, its waves of 32 columns and of 16."""
    rng = np.random.default_rng(E)
    for hd in (64, 256):
        P = Pair(hd, 1, (length + 63) // 64)
        fill(P, rng, length, GRADES[grade])
        for dtype in ("bf16", "f32"):
            P.batch(P.table, [length], [0, {(64, "bf16"): 129}.get((hd, dtype), 65)])  # 8256 columns, else 4160
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


@pytest.mark.parametrize("n_seq", [65, 130])
@pytest.mark.parametrize("hd,dtype", [(64, "f16"), (96, "bf16"), (128, "f32"), (256, "bf16")])
def test_two_shares_a_cu_of_many_sequences(n_seq, hd, dtype):
    """Past 64 sequences, and a group for each CU, shares come in the sequences' order: long ones among short and empty
    ones, first, last and in each wave's worth of them; one row of each, and few."""
    rng = np.random.default_rng(n_seq)
    P = Pair(hd, 8, 64 + 3 * n_seq)
    lens = [(0, 1, 64, 65, 130)[i % 5] for i in range(n_seq)]
    lens[0], lens[63], lens[64], lens[-1] = 700, 1500, 900, 600
    table = tables(rng, lens, P.n_blocks)
    P.batch(table, lens)
    fill_device(rng, P)
    a = P.check_attend(dtype, queries(rng, P, 16, dtype), 0.1)
    assert np.isfinite(a[0]).all()
    rows = [min(n, 2) for n in lens]
    P.batch(table, lens, np.concatenate([[0], np.cumsum(rows)]).tolist(), sum(rows) + 1)
    q = queries(rng, P, 32, dtype)
    a, b = P.check_attend(dtype, q, 0.1), P.attend(dtype, q, 0.1)
    assert all(np.array_equal(x, y) for x, y in zip(a, b)), "the order of arrival shows"
