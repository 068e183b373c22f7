"""Attention weights kept beside the 4-bit block cache's positions, and eviction by them, against
numpy in 64 bits (weights within bounds derived from the arithmetic, kept positions and what is
moved exactly)."""
import math

import numpy as np
import pytest
import torch

import sp_hip as S
from fp4_pair import Pair
from test_gpu_fp4_cache import fill_device
from test_gpu_fp8_cache import LENS, cur, queries, tables

pytestmark = pytest.mark.gpu


# ---- weigh ----

@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window", [0, 100])
def test_weigh_steps(hd, dtype, window):
    rng = np.random.default_rng(hd)
    P = Pair(hd, 2, 40, layers=2)
    table = tables(rng, LENS, 40, extra=1)
    P.fill(rng, table, LENS, "f32", 0.5, layer=1)
    P.batch(table, LENS)
    P.set_weights(rng.random(P.ref.weight.shape) * 0.1)
    added = P.check_weigh(dtype, queries(rng, P, 8, dtype), 1 / math.sqrt(hd), window, layer=1)
    # softmax weights: each KV head's four query heads give every sequence 4 in all
    live = sum(n > 0 for n in LENS)
    assert abs(added.sum() - 8 * live) < 1e-3 and (added[0] == 0).all()
    P.check_weigh(dtype, queries(rng, P, 2, dtype), -0.3, window, layer=1, pad=5, shift=1)
    P.check_weigh(dtype, queries(rng, P, 6, dtype), 0.0, window, layer=1, pad=4)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_weigh_rows(hd, dtype):
    rng = np.random.default_rng(hd + 7)
    P = Pair(hd, 2, 40)
    lens = [1, 0, 63, 64, 65, 1100, 129, 3]
    table = tables(rng, lens, 40, extra=1)
    P.batch(table, lens)
    fill_device(rng, P)
    news = [1, 0, 20, 10, 0, 37, 29, 7]  # the last: more rows than positions
    row = np.concatenate([[0], np.cumsum(news)]).tolist()
    for n_q, scale, window, kw in ((8, 1 / math.sqrt(hd), 0, {}), (2, -0.3, 77, dict(pad=3, shift=1)),
                                   (6, 0.2, 0, dict(pad=8))):
        P.batch(table, lens, row, row[-1] + 3)
        P.check_weigh(dtype, queries(rng, P, n_q, dtype), scale, window, **kw)


@pytest.mark.parametrize("group", [1, 3, 16, 17, 70])
def test_weigh_groups(group):
    rng = np.random.default_rng(group)
    P = Pair(64, 3, 30)
    lens = [5, 400, 64, 0, 777]
    P.batch(tables(rng, lens, 30), lens)
    fill_device(rng, P)
    for dtype in ("bf16", "f32"):
        P.check_weigh(dtype, queries(rng, P, 3 * group, dtype), 0.1)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype,pad", [("f32", 0), ("f16", 0), ("bf16", 0), ("bf16", 3)])
def test_weigh_more_columns_than_a_stage(hd, dtype, pad):
    rng = np.random.default_rng(hd + pad)
    P = Pair(hd, 2, 24)
    lens = [150, 1000]
    P.fill(rng, tables(rng, lens, 24), lens, dtype)
    P.batch(P.table, lens, [0, 150, 251], 255)
    P.check_weigh(dtype, queries(rng, P, 10, dtype), 0.1, pad=pad)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_weigh_with_every_cu(hd, dtype):
    """Tables so wide that no columns are shared out."""
    rng = np.random.default_rng(hd)
    P = Pair(hd, 32, 8)
    lens = [300, 70]
    table = [list(t) + [-1] * (70 - len(t)) for t in tables(rng, lens, 8)]
    P.fill(rng, table, lens, dtype)
    P.batch(table, lens, [0, 45, 46], 47)
    P.check_weigh(dtype, queries(rng, P, 96, dtype), 0.1)


def test_weigh_many_sequences_and_holes():
    rng = np.random.default_rng(3)
    P = Pair(64, 1, 320)
    lens = [1 + (i * 29) % 130 for i in range(130)]
    lens[97] = 4000
    table = tables(rng, lens, 320)
    table[97][5], table[97][20], table[3][0] = -1, 9999, -5
    P.batch(table, lens)
    fill_device(rng, P)
    P.check_weigh("f16", queries(rng, P, 8, "f16"), 0.2)
    P.check_weigh("f16", queries(rng, P, 2, "f16"), 0.2, window=700)


def test_weigh_passes_over_what_is_not_finite():
    rng = np.random.default_rng(4)
    P = Pair(128, 2, 12)
    P.batch(tables(rng, [300, 200], 12), [300, 200], [0, 20, 40])
    fill_device(rng, P)
    q = queries(rng, P, 4, "bf16")
    _, lse = P.attend("bf16", q, 0.2)
    q[5, 1, 3], q[31, 0, 0], q[32, 1, 127] = float("nan"), float("inf"), -float("inf")
    lse[7, 2], lse[8, 0], lse[9, 3] = np.nan, np.inf, -np.inf
    P.check_weigh("bf16", q, 0.2, lse=lse)
    assert np.isfinite(P.weights()).all()


def test_weigh_of_sequences_that_share_blocks():
    rng = np.random.default_rng(5)
    P = Pair(64, 1, 12)
    P.batch([[0, 1, 2], [0, 1, 3], [0, 0, 0]], [150, 140, 192])
    fill_device(rng, P)
    P.check_weigh("f32", queries(rng, P, 4, "f32"), 0.1)


def test_weigh_large_scores():
    """Scores of 2^20 beside each other: the difference to lse is what counts."""
    rng = np.random.default_rng(6)
    P = Pair(64, 1, 4)
    P.batch([[0, 1, 2]], [130])
    fill_device(rng, P)
    for dtype in ("bf16", "f32"):
        P.check_weigh(dtype, (queries(rng, P, 4, dtype) * 2.0 ** 6).to(queries(rng, P, 1, dtype).dtype), 4.0)


# ---- evict ----

@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("keep,first,recent", [(1, 0, 0), (1, 1, 0), (63, 4, 20), (64, 0, 64), (100, 0, 0),
                                               (128, 100, 28), (200, 3, 17), (700, 1, 1)])
def test_evict(hd, keep, first, recent):
    rng = np.random.default_rng(keep)
    P = Pair(hd, 3, 60, layers=2)
    lens = [700, 1, 0, 64, 65, 699, 128, 201, keep, keep + 1]
    P.batch(tables(rng, lens, 60), lens)
    fill_device(rng, P)
    P.set_weights(np.exp(2 * rng.standard_normal(P.ref.weight.shape)))
    P.check_evict(keep, first, recent, layer=1)


@pytest.mark.parametrize("kind", ["equal", "few", "nan", "signs", "tiny"])
def test_evict_ties_and_odd_weights(kind):
    rng = np.random.default_rng(1)
    P = Pair(64, 2, 60)
    lens = [1500, 900, 64]
    P.batch(tables(rng, lens, 60), lens)
    fill_device(rng, P)
    w = rng.random(P.ref.weight.shape)
    if kind == "equal":
        w[:] = 0.25
    if kind == "few":  # few values, each many times; also neighbours in their last bit
        w = np.float32(1.0) + rng.integers(0, 4, w.shape) * 2.0 ** -23
    if kind == "nan":
        w[rng.random(w.shape) < 0.7] = np.nan
    if kind == "signs":
        w = rng.choice([0.0, -0.0, -1.0, 1.0, -np.inf, np.inf, 1e-45, -1e-45], w.shape)
    if kind == "tiny":
        w *= 1e-43
    P.set_weights(w)
    P.check_evict(333, 4, 29)


def test_evict_long_and_ragged():
    rng = np.random.default_rng(2)
    P = Pair(64, 2, 700)
    lens = [20000, 8193, 3000, 4097, 4100]
    P.batch(tables(rng, lens, 700), lens)
    fill_device(rng, P)
    P.set_weights(np.exp(2 * rng.standard_normal(P.ref.weight.shape)))
    P.check_evict(4097, 4, 512)
    P.batch(P.table, [min(n, 4097) for n in lens])
    P.check_evict(2100, 0, 0)


@pytest.mark.parametrize("longest", [3000, 20000, 40000])
@pytest.mark.parametrize("kind", ["spread", "few", "equal", "crowded"])
def test_evict_by_length(longest, kind):
    """Table rows of each length that the selection tells apart; values that are all different, that are few, one,
    or neighbours in their last bits."""
    rng = np.random.default_rng(longest)
    P = Pair(64, 1, 1300)
    lens = [longest, longest * 4 // 5 + 1, 64, longest // 4 + 200]
    P.batch(tables(rng, lens, 1300), lens)
    fill_device(rng, P)
    shape = P.ref.weight.shape
    P.set_weights({"spread": lambda: np.exp(2 * rng.standard_normal(shape)),
                   "few": lambda: rng.integers(0, 5, shape) / 4.0,
                   "equal": lambda: np.full(shape, 0.5),
                   "crowded": lambda: np.float32(1.0) + rng.integers(0, 4096, shape) * 2.0 ** -23}[kind]())
    P.check_evict(longest // 4 + 11, 4, 300)


def test_evict_keeps_nothing_by_weight():
    """All that stays is first or recent; and a few to choose from."""
    rng = np.random.default_rng(12)
    P = Pair(96, 2, 30)
    lens = [600, 300, 201]
    P.batch(tables(rng, lens, 30), lens)
    fill_device(rng, P)
    P.set_weights(rng.random(P.ref.weight.shape))
    P.check_evict(200, 60, 140)
    P.batch(P.table, [min(n, 200) for n in lens])
    P.check_evict(100, 0, 1)


def test_evict_many_sequences():
    """More than one round of places in each of many blocks of threads."""
    rng = np.random.default_rng(13)
    P = Pair(64, 8, 460)
    lens = [1600 - 7 * i for i in range(17)]
    P.batch(tables(rng, lens, 460), lens)
    fill_device(rng, P)
    P.set_weights(rng.random(P.ref.weight.shape))
    P.check_evict(1500, 4, 100)


def test_evict_leaves_incomplete_sequences():
    rng = np.random.default_rng(3)
    P = Pair(128, 2, 30)
    table = [[0, 1, 2, 3], [4, -1, 5, 6], [7, 8, 30, 9], [10, 11], [12, 13, 14, -1]]
    P.batch(table, [256, 256, 200, 300, 192])  # a missing block, one past the pool, a length past the table
    fill_device(rng, P)
    P.set_weights(rng.random(P.ref.weight.shape))
    kept = P.check_evict(100, 2, 10)
    assert (kept[1:4] == -1).all() and (kept[[0, 4]] >= 0).all()


def test_evict_most_and_least():
    """One row less, and all but one."""
    rng = np.random.default_rng(4)
    P = Pair(64, 1, 20)
    P.batch(tables(rng, [1200], 20), [1200])
    fill_device(rng, P)
    P.set_weights(rng.random(P.ref.weight.shape))
    P.check_evict(1199, 0, 0)
    P.batch(P.table, [1199])
    P.check_evict(1, 0, 0)


# ---- together ----

@pytest.mark.parametrize("hd,dtype", [(128, "bf16"), (64, "f16"), (256, "f32"), (96, "bf16")])
def test_a_chat_within_a_budget(hd, dtype):
    """A prompt is written and attended, its last rows weigh it, it is cut to a budget; steps follow that are
    written, attended and weighed, and cut again when a block has filled up."""
    rng = np.random.default_rng(hd)
    H, n_q, budget = 2, 6, 150
    P = Pair(hd, H, 20)
    lens = [400, 90]
    table = tables(rng, [n + 70 for n in lens], 20)
    P.fill(rng, table, lens, dtype, 0.5)
    q = queries(rng, P, n_q, dtype)
    P.check_attend(dtype, q, 0.1)
    P.batch(table, lens, [0, 32, 64])  # the last 32 rows of each
    P.check_weigh(dtype, queries(rng, P, n_q, dtype), 0.1)
    P.ref.weight = P.weights()
    for turn in range(6):
        P.batch(table, lens)
        if turn % 3 == 0:
            P.check_evict(budget, 4, 32)
            lens = [min(n, budget) for n in lens]
        lens = [n + 1 for n in lens]
        P.batch(table, lens)
        P.write(dtype, P.rows(rng, dtype), P.rows(rng, dtype))
        q = queries(rng, P, n_q, dtype)
        _, lse = P.check_attend(dtype, q, 0.1)
        P.check_weigh(dtype, q, 0.1, lse=lse)
        P.ref.weight = P.weights()
        P.check_memory()


def test_captured_eviction_follows_lengths():
    rng = np.random.default_rng(9)
    P = Pair(64, 2, 40)
    lens = [700, 300]
    table = tables(rng, [800, 600], 40)
    P.batch(table, [0, 0])
    fill_device(rng, P)
    kept = torch.zeros((2, 2, 200), dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        S.check(S.lib().sp_hip_fp4_evict(P.dev.ref, 0, P.b.ref, 200, 4, 40, kept.data_ptr(),
                                         torch.cuda.current_stream().cuda_stream), "evict")
    for turn in range(4):
        P.set_lens(lens)
        P.set_weights(rng.random(P.ref.weight.shape))
        g.replay()
        torch.cuda.synchronize()
        want = P.ref.evict(0, P.table, lens, 200, 4, 40)
        np.testing.assert_array_equal(kept.cpu().numpy(), want)
        P.check_memory()
        lens = [200 + 37 * (turn + 1), 100 + 70 * (turn + 1)]


def test_captured_weigh_adds_at_each_replay():
    rng = np.random.default_rng(10)
    H, n_q = 2, 8
    P = Pair(128, H, 20)
    lens = [400, 130]
    P.fill(rng, tables(rng, [500, 300], 20), lens, "bf16")
    P.batch(P.table, lens)
    q = queries(rng, P, n_q, "bf16")
    qt = q.cuda()
    out = torch.zeros_like(qt)
    lse = torch.zeros((2, n_q), dtype=torch.float32, device="cuda")
    L = S.lib()
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        s = torch.cuda.current_stream().cuda_stream
        S.check(L.sp_hip_fp4_attn_decode(P.dev.ref, 0, P.b.ref, qt.data_ptr(), n_q * 128, n_q, S.DTYPE_BF16, 0.1, 0,
                                         out.data_ptr(), n_q * 128, lse.data_ptr(), s), "decode")
        S.check(L.sp_hip_fp4_weigh(P.dev.ref, 0, P.b.ref, qt.data_ptr(), n_q * 128, n_q, S.DTYPE_BF16, 0.1, 0,
                                   lse.data_ptr(), s), "weigh")
    for turn in range(4):
        P.set_lens(lens)
        before = P.weights()
        g.replay()
        torch.cuda.synchronize()
        P.ref.weight = before.copy()
        tol = P.ref.weigh(0, P.table, lens, None, 2, q.double().numpy(), float(np.float32(0.1)), 0,
                          lse.double().cpu().numpy())
        assert (np.abs(P.weights() - P.ref.weight) <= tol).all()
        lens = [n - 60 for n in lens]
        torch.full((64, 1024), 3.0, device="cuda").sum()
        torch.cuda.synchronize()
