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
