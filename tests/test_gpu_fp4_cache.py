"""The 4-bit block cache on the GPU against its numpy form in 64 bits: codes and scales
exactly, attention within the bounds of the 8-bit cache's arithmetic (fp8_ref.bounds: codes times
their scales are exact in both)."""
import math

import numpy as np
import pytest
import torch

import fp4_ref as R
import sp_hip as S
from fp4_pair import Pair
from gpu_util import d2h
from test_gpu_fp8_cache import CODE, ESIZE, LENS, TORCH, cur, queries, tables

pytestmark = pytest.mark.gpu


# ---- write and read ----

@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_write_then_appends(hd, dtype):
    rng = np.random.default_rng(hd)
    P = Pair(hd, 3, 24, layers=2)
    P.set_weights(rng.random(P.ref.weight.shape))
    lens = [1, 64, 65, 200, 131]
    table = tables(rng, [n + 130 for n in lens], 24)
    P.fill(rng, table, lens, dtype)
    P.check_memory()
    for step, news in enumerate(([1, 1, 1, 1, 1], [3, 0, 70, 64, 2], [1, 5, 0, 0, 63])):
        lens = [n + m for n, m in zip(lens, news)]
        P.batch(table, lens, np.concatenate([[0], np.cumsum(news)]).tolist(), sum(news) + step)
        for side in range(2):
            k = P.rows(rng, dtype, 2.0) if side == 0 else None
            v = P.rows(rng, dtype, 2.0) if side == 1 else None
            P.write(dtype, k, v, layer=1, pad=step * 4, shift=(0, 0, 1)[step])
        P.check_memory()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_every_border(dtype):
    """Each number, the borders between two and what is next to them, at three scales, and each
    border of a scale."""
    P = Pair(64, 1, 2)
    mid = (R.POS[:-1] + R.POS[1:]) / 2
    eps = torch.finfo(TORCH[dtype]).eps
    around = np.concatenate([R.POS, mid, mid * (1 + eps), mid * (1 - eps / 2)])
    around = np.concatenate([around, -around])[:60]
    x = np.zeros((64, 1, 64))
    for r in range(64):
        x[r, 0, :31] = np.roll(around, r)[:31] * 2.0 ** (r % 3 - 1)
        x[r, 0, 31] = 6.0 * 2.0 ** (r % 3 - 1)
        x[r, 0, 32:63] = np.roll(around, 31 + r)[:31]
        x[r, 0, 63] = 6.0 * (1 + eps * (r % 2))  # next to a border of the scale
    P.batch([[1]], [64], [0, 64])
    P.write(dtype, torch.from_numpy(x).to(TORCH[dtype]), torch.from_numpy(-x).to(TORCH[dtype]))
    P.check_memory()


def test_extremes_are_finite():
    P = Pair(64, 1, 4)
    P.batch([[0, 1, 2]], [130], [0, 130])
    k = torch.zeros(130, 1, 64)
    k[0, 0, 0], k[1, 0, 1], k[2, 0, 2] = float("nan"), float("inf"), -float("inf")
    k[3, 0, 3] = 1.0
    k[70, 0, 5] = 1e-30           # below what the least scale holds
    k[71, 0, 5] = 2.0 ** -149
    k[129, 0, 7] = 3e38
    v = torch.full((130, 1, 64), 2.0 ** -45)
    v[5] = float("nan")
    P.write("f32", k, v)
    P.check_memory()


def test_a_shorter_sequence_goes_on_and_a_block_starts_anew():
    rng = np.random.default_rng(5)
    P = Pair(128, 2, 8)
    table = [[3, 4], [5, 6], [1, 2]]
    P.fill(rng, table, [100, 64, 90])
    for lens, news in (([70, 65, 60], [5, 1, 1]), ([66, 64, 3], [2, 64, 3]), ([65, 1, 65], [1, 1, 65])):
        P.batch(table, lens, np.concatenate([[0], np.cumsum(news)]).tolist())
        P.write("f16", P.rows(rng, "f16", 2.0), P.rows(rng, "f16", 2.0))
        P.check_memory()


def test_absent_positions_are_passed_over():
    rng = np.random.default_rng(9)
    P = Pair(128, 2, 6)
    # blocks past the pool, negative entries, a length past the table, rows before position 0
    P.batch([[0, 6, 1], [-1, 2, 7], [3, 4, 5], [-7, 1 << 30, 3]], [192, 130, 300, 5], [0, 192, 322, 522, 530], 541)
    P.write("bf16", P.rows(rng, "bf16"), P.rows(rng, "bf16"))
    P.check_memory()
    out = [torch.full((541, 2, 128), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    S.check(S.lib().sp_hip_fp4_read(P.dev.ref, 0, P.b.ref, out[0].data_ptr(), out[1].data_ptr(), 256, S.DTYPE_BF16,
                                    cur()), "read")
    torch.cuda.synchronize()
    for side in range(2):
        want = np.full((541, 2, 128), 7.0)
        for _, r, b, at, _ in P.ref.places(P.table, P.lens, P.row, 541):
            want[r] = P.ref.stored(side, 0, b)[:, at] if b >= 0 else 0.0
        np.testing.assert_array_equal(out[side].cpu().double().numpy(),
                                      torch.from_numpy(want).bfloat16().double().numpy())


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_read(hd, dtype):
    rng = np.random.default_rng(hd + 1)
    P = Pair(hd, 3, 16, layers=2)
    lens = [1, 64, 127, 300]
    P.fill(rng, tables(rng, lens, 16), lens, "f32", 0.5, layer=1)
    for news, pad, shift in (([1, 1, 1, 1], 0, 0), (lens, 8, 0), ([1, 30, 64, 299], 3, 1), ([1, 17, 15, 80], 4, 0)):
        row = None if max(news) == 1 else np.concatenate([[0], np.cumsum(news)]).tolist()
        P.batch(P.table, lens, row)
        width = 3 * hd
        got = [torch.full((shift + P.n_rows * (width + pad),), 7.0, dtype=TORCH[dtype], device="cuda")
               for _ in range(2)]
        p = [t.data_ptr() + shift * ESIZE[dtype] for t in got]
        S.check(S.lib().sp_hip_fp4_read(P.dev.ref, 1, P.b.ref, p[0], p[1], width + pad, CODE[dtype], cur()), "read")
        torch.cuda.synchronize()
        for side, t in enumerate(got):
            t = t.cpu()
            assert (t[:shift] == 7.0).all()
            t = t[shift:].view(P.n_rows, width + pad)
            assert (t[:, width:] == 7.0).all()
            want = np.stack([P.ref.stored(side, 1, b)[:, at] for _, _, b, at, _ in
                             P.ref.places(P.table, P.lens, P.row, P.n_rows)])
            want = torch.from_numpy(want).to(TORCH[dtype])  # the numbers are exact in fp32: one rounding
            assert torch.equal(t[:, :width].reshape(want.shape), want)


def test_many_sequences_and_empty_ones():
    """More sequences than a wave has lanes, some without rows, rows behind the last."""
    rng = np.random.default_rng(3)
    P = Pair(64, 1, 300)
    news = [(i * 7) % 5 if i % 3 else 0 for i in range(150)]
    lens = [n + (i * 13) % 90 for i, n in enumerate(news)]
    table = tables(rng, lens, 300)
    P.batch(table, lens, np.concatenate([[0], np.cumsum(news)]).tolist(), sum(news) + 7)
    P.write("f32", P.rows(rng, "f32"), P.rows(rng, "f32"))
    P.check_memory()
    P.check_attend("f32", queries(rng, P, 2, "f32"), 0.125)


# ---- attention: few rows ----

@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window", [0, 100])
def test_decode(hd, dtype, window):
    rng = np.random.default_rng(hd)
    P = Pair(hd, 2, 40, layers=2)
    table = tables(rng, LENS, 40, extra=1)
    P.fill(rng, table, LENS, "f32", 0.5, layer=1)
    P.batch(table, LENS)
    P.check_attend(dtype, queries(rng, P, 8, dtype), 1 / math.sqrt(hd), window, layer=1)
    P.check_attend(dtype, queries(rng, P, 2, dtype), -0.3, window, layer=1, pad=5, shift=1)
    P.check_attend(dtype, queries(rng, P, 2, dtype), 0.0, window, layer=1, pad=4)


@pytest.mark.parametrize("group", [1, 3, 15, 16, 17, 40])
def test_decode_groups(group):
    rng = np.random.default_rng(group)
    P = Pair(128, 3, 30)
    lens = [5, 400, 64, 0, 777]
    P.fill(rng, tables(rng, lens, 30), lens)
    P.batch(P.table, lens)
    for dtype in ("bf16", "f32"):
        P.check_attend(dtype, queries(rng, P, 3 * group, dtype), 0.1)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window", [0, 77])
def test_prefill(hd, dtype, window):
    rng = np.random.default_rng(hd + 7)
    P = Pair(hd, 2, 40, layers=2)
    lens = [1, 0, 63, 64, 65, 500, 129, 3]
    table = tables(rng, lens, 40, extra=1)
    P.fill(rng, table, lens, "f32", 0.5, layer=1)
    news = [1, 0, 63, 10, 0, 137, 129, 7]  # the last: more rows than positions
    row = np.concatenate([[0], np.cumsum(news)]).tolist()
    for n_q, scale, kw in ((8, 1 / math.sqrt(hd), {}), (2, -0.3, dict(pad=3, shift=1)), (6, 0.2, dict(pad=8))):
        P.batch(table, lens, row, row[-1] + 3)
        P.check_attend(dtype, queries(rng, P, n_q, dtype), scale, window, layer=1, **kw)


@pytest.mark.parametrize("new,length", [(1, 20000), (6, 20001), (300, 9000), (1, 131072)])
def test_long_sequences(new, length):
    """Work split over many shares of one sequence."""
    rng = np.random.default_rng(new)
    P = Pair(64, 1, (length + 63) // 64 + 2)
    P.batch(tables(rng, [length], P.n_blocks), [length], [0, length])
    fill_device(rng, P)
    P.batch(P.table, [length], None if new == 1 else [0, new])
    for dtype in ("bf16", "f32"):
        P.check_attend(dtype, queries(rng, P, 4, dtype), 0.2)
    P.check_attend("f16", queries(rng, P, 4, "f16"), 0.2, window=5000)
    q = queries(rng, P, 4, "f32")
    a, b = P.attend("f32", q, 0.2), P.attend("f32", q, 0.2)
    assert all(np.array_equal(x, y) for x, y in zip(a, b)), "the order of arrival shows"


def fill_device(rng, P, layer=0):
    """Every block with codes and exponents of its own, set on both sides (the numpy form's write
    goes row by row)."""
    from fp4_pair import copy
    for side, (codes, exps) in enumerate(((P.dev.c.d_k_codes, P.dev.c.d_k_exp), (P.dev.c.d_v_codes, P.dev.c.d_v_exp))):
        P.ref.codes[side] = rng.integers(0, 16, P.ref.codes[side].shape)
        P.ref.exps[side] = rng.integers(121, 128, P.ref.exps[side].shape)
        for to, x in ((codes, P.ref.code_bytes(side)), (exps, P.ref.exp_bytes(side))):
            copy(to, torch.from_numpy(np.ascontiguousarray(x)).cuda())


# ---- attention: many rows ----

@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window", [0, 77])
def test_many_columns(hd, dtype, window):
    """Column groups of the kernel for many rows: whole, partly filled, and with none to do."""
    rng = np.random.default_rng(hd + 3)
    P = Pair(hd, 2, 40)
    lens, news = [0, 500, 400], [0, 300, 130]
    P.batch(tables(rng, lens, 40, extra=1), lens, [0, 0, 300, 430], 433)
    fill_device(rng, P)
    for group, scale, kw in ((10, 1 / math.sqrt(hd), {}), (11, -0.2, dict(pad=3, shift=1))):
        P.check_attend(dtype, queries(rng, P, 2 * group, dtype), scale, window, **kw)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_columns_shared_out(hd, dtype):
    """Few column groups over many cache blocks: shares, joined; more blocks than are looked up at once."""
    rng = np.random.default_rng(hd)
    P = Pair(hd, 1, 210)
    P.batch(tables(rng, [13000], 210), [13000], [0, 130])
    fill_device(rng, P)
    P.check_attend(dtype, queries(rng, P, 64, dtype), 0.1)


def test_many_columns_over_many_blocks():
    """A share of more than 64 cache blocks: exponents looked up a second time."""
    rng = np.random.default_rng(8)
    P = Pair(64, 16, 75)
    P.batch(tables(rng, [4700], 75), [4700], [0, 260])
    fill_device(rng, P)
    P.check_attend("bf16", queries(rng, P, 256, "bf16")[:, :256], 0.1)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_a_chunk_behind_a_long_table(hd, dtype):
    """Fewer rows than the table's length makes worth sharing a conversion: short and empty sequences among them."""
    rng = np.random.default_rng(hd)
    P = Pair(hd, 16, 16)
    lens, news = [300, 40, 0, 65], [33, 32, 0, 40]
    table = [list(t) + [-1] * (100 - len(t)) for t in tables(rng, lens, 16)]
    P.fill(rng, table, lens, dtype)
    P.batch(table, lens, np.concatenate([[0], np.cumsum(news)]).tolist(), sum(news) + 2)
    P.check_attend(dtype, queries(rng, P, 64, dtype), 0.1, window=0)


@pytest.mark.parametrize("hd,dtype", [(128, "bf16"), (256, "f32")])
def test_a_chunk_behind_a_long_cache(hd, dtype):
    rng = np.random.default_rng(hd)
    P = Pair(hd, 2, 110)
    P.fill(rng, tables(rng, [6500], 110), [6500], dtype)
    P.batch(P.table, [6500], [0, 70])
    P.check_attend(dtype, queries(rng, P, 64, dtype), 0.1)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_more_column_groups_than_cus(hd, dtype):
    rng = np.random.default_rng(hd)
    P = Pair(hd, 32, 64)
    lens = [1, 64, 700, 65, 0, 130, 300, 20, 513]
    table = tables(rng, [n + 3 for n in lens], 64)
    P.fill(rng, table, lens, dtype)
    P.batch(table, lens)
    P.check_attend(dtype, queries(rng, P, 96, dtype), 0.1)
    lens = [n + 3 for n in lens]
    P.batch(table, lens, [3 * i for i in range(len(lens) + 1)])
    P.write(dtype, P.rows(rng, dtype), P.rows(rng, dtype))
    P.check_attend(dtype, queries(rng, P, 192, dtype), 0.1)


@pytest.mark.parametrize("n_seq", [12, 20, 63])
@pytest.mark.parametrize("hd,dtype", [(64, "f16"), (128, "f32"), (256, "bf16")])
def test_unequal_lengths_past_the_cus(n_seq, hd, dtype):
    """The longest first: some empty, several alike, and few rows of each besides."""
    rng = np.random.default_rng(n_seq)
    H = 32 if n_seq < 60 else 8
    P = Pair(hd, H, 240)
    lens = [(0, 1, 64, 65, 130)[i % 5] for i in range(n_seq)]
    lens[n_seq // 2], lens[-1], lens[3] = 2300, 1200, 1200
    if n_seq > 60:
        lens = [min(n, 65) if i % 2 else n for i, n in enumerate(lens)]
        lens[1] = 2300
    table = tables(rng, lens, 240)
    P.fill(rng, table, lens, dtype)
    P.batch(table, lens)
    P.check_attend(dtype, queries(rng, P, H * (4 if H == 8 else 1), dtype), 0.1)
    rows = [min(n, 2) for n in lens]
    P.batch(table, lens, np.concatenate([[0], np.cumsum(rows)]).tolist(), sum(rows) + 1)
    P.check_attend(dtype, queries(rng, P, H * 3, dtype), 0.1)


def test_tables_with_holes():
    rng = np.random.default_rng(1)
    for hd in (64, 128, 256):
        P = Pair(hd, 2, 30)
        table = [[3, -1, 5, 6, 7, 30], [8, 9, 10], [-1, -1], [11, 12, 99, 13]]
        lens = [384, 500, 100, 250]
        P.batch(table, lens)
        fill_device(rng, P)
        for dtype in ("bf16", "f32"):
            P.batch(table, lens)
            P.check_attend(dtype, queries(rng, P, 4, dtype), 0.2)
            P.batch(table, lens, [0, 150, 152, 160, 300])
            P.check_attend(dtype, queries(rng, P, 64, dtype), 0.2, window=200)


@pytest.mark.parametrize("rows", [1, 130])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_scales_far_apart(rows, dtype):
    """Blocks whose scales are octaves apart, positions and groups of channels whose scales are: what
    lies below 2^-25 of a block's largest is not seen, everything else is."""
    rng = np.random.default_rng(2)
    for hd in (64, 128, 256):
        P = Pair(hd, 1, 12)
        P.batch(tables(rng, [700], 12), [700], [0, rows])
        fill_device(rng, P)
        from fp4_pair import copy
        for side, exps in enumerate((P.dev.c.d_k_exp, P.dev.c.d_v_exp)):
            e = P.ref.exps[side]
            base = 127 + rng.integers(-12, 13 if side else 1, e.shape[:2] + (1, 1, 1))  # of a block
            P.ref.exps[side] = base - rng.integers(0, 30, e.shape) * (rng.random(e.shape) < 0.3)
            copy(exps, torch.from_numpy(np.ascontiguousarray(P.ref.exp_bytes(side))).cuda())
        P.check_attend(dtype, queries(rng, P, 70, dtype), 0.05)
    top = 2.0 ** (P.ref.exps[1].max((3, 4), keepdims=True)[..., 0, 0][0, 0, 0].astype(float) - 127)
    assert np.abs(P.ref.stored(1, 0, 0) - P.ref.values(1, 0, 0)).max() <= 2.0 ** -25 * top


def test_masked_places_hold_nothing_that_shows():
    """A block used before, with the largest numbers there are: what lies behind the rows of the
    sequence that has it now neither shows nor costs it precision."""
    rng = np.random.default_rng(6)
    for hd in (64, 96, 128, 256):
        P = Pair(hd, 2, 4)
        P.batch([[1, 2]], [128], [0, 128])
        big = torch.full((128, 2, hd), float("inf"))
        P.write("f32", big, -big)
        P.batch([[1, 2]], [70], [0, 70])
        P.write("f32", P.rows(rng, "f32"), P.rows(rng, "f32"))
        P.check_memory()
        P.batch([[1, 2]], [70])
        P.check_attend("f32", queries(rng, P, 4, "f32"), 0.2)
        P.batch([[1, 2]], [70], [0, 69])
        P.check_attend("f32", queries(rng, P, 130, "f32"), 0.2)
        P.check_attend("bf16", queries(rng, P, 130, "bf16"), 0.2)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_not_finite_queries_stay_in_their_rows(hd):
    rng = np.random.default_rng(hd)
    P = Pair(hd, 2, 12)
    P.batch(tables(rng, [300, 200], 12), [300, 200], [0, 130, 260], 260)
    fill_device(rng, P)
    for heads in (4, 40):
        q = queries(rng, P, heads, "bf16")
        q[5, 1, 3], q[131, 0, 0] = float("nan"), float("inf")
        out, lse = P.attend("bf16", q, 0.2)
        q0 = q.clone()
        q0[5, 1], q0[131, 0] = 0, 0
        want, wlse, reach, steep = P.ref.attend(0, P.table, P.lens, P.row, P.n_rows, q0.double().numpy(), 0.2, 0)
        tol, _ = __import__("fp8_ref").bounds("bf16", hd, 300, want, reach, steep)
        good = np.ones(out.shape[:2], bool)
        good[5, 1] = good[131, 0] = False
        assert (np.abs(out - want)[good] <= tol[good]).all()
        assert np.isnan(out[5, 1]).all()


def test_blocks_past_4_gib():
    """A pool whose codes pass 32 bits of bytes: rows written, read and attended at its end."""
    rng = np.random.default_rng(11)
    n = 140000  # 4 heads of 256: 32 KB of codes a block and side
    P = S.Fp4Cache(S.config(256, 1, 4), n, cur())
    small = Pair(256, 4, 4)
    tab = [[0, 3], [1, 2]]
    far = [[0, n - 1], [n - 2, 137001]]
    small.batch(tab, [100, 90], [0, 100, 190])
    k, v = small.rows(rng, "bf16"), small.rows(rng, "bf16")
    small.write("bf16", k, v)
    t = torch.tensor(far, dtype=torch.int32, device="cuda")
    b = S.Fp4Batch(2, 2, t.data_ptr(), small.keep[1].data_ptr(), small.keep[2].data_ptr(), 190)
    kd, vd = k.cuda(), v.cuda()
    S.check(S.lib().sp_hip_fp4_write(P.ref, 0, b.ref, kd.data_ptr(), vd.data_ptr(), 1024, S.DTYPE_BF16, cur()), "write")
    q = queries(rng, small, 8, "bf16").cuda()
    outs = []
    for cache, bb in ((P, b), (small.dev, small.b)):
        out = torch.empty_like(q)
        lse = torch.empty((190, 8), device="cuda")
        S.check(S.lib().sp_hip_fp4_attn_prefill(cache.ref, 0, bb.ref, q.data_ptr(), 2048, 8, S.DTYPE_BF16, 0.1, 0,
                                                out.data_ptr(), 2048, lse.data_ptr(), cur()), "attend")
        back = torch.empty_like(kd)
        S.check(S.lib().sp_hip_fp4_read(cache.ref, 0, bb.ref, back.data_ptr(), None, 1024, S.DTYPE_BF16, cur()), "read")
        S.check(S.lib().sp_hip_fp4_weigh(cache.ref, 0, bb.ref, q.data_ptr(), 2048, 8, S.DTYPE_BF16, 0.1, 0,
                                         lse.data_ptr(), cur()), "weigh")
        kept = torch.empty((2, 4, 70), dtype=torch.int32, device="cuda")
        S.check(S.lib().sp_hip_fp4_evict(cache.ref, 0, bb.ref, 70, 2, 8, kept.data_ptr(), cur()), "evict")
        lens = torch.tensor([70, 70], dtype=torch.int32, device="cuda")
        short = S.Fp4Batch(2, 2, (t if cache is P else small.keep[0]).data_ptr(), lens.data_ptr())
        after = torch.empty((2, 8, 256), dtype=torch.bfloat16, device="cuda")
        S.check(S.lib().sp_hip_fp4_attn_decode(cache.ref, 0, short.ref, q.data_ptr(), 2048, 8, S.DTYPE_BF16, 0.1, 0,
                                               after.data_ptr(), 2048, None, cur()), "attend")
        torch.cuda.synchronize()
        outs.append((out, lse, back, kept, after))
    for x, y in zip(*outs):
        assert torch.equal(x, y)
    P.free()


# ---- streams and graphs ----

def test_captured_steps_follow_lengths_and_tables():
    """A step captured once: rows written, attended and weighed, with lengths and blocks of each
    replay, beside eager calls between the replays."""
    rng = np.random.default_rng(21)
    hd, H, n_q = 128, 2, 8
    P = Pair(hd, H, 40)
    lens = [100, 61, 0]
    table = tables(rng, [n + 200 for n in lens], 40)
    P.fill(rng, table, lens)
    P.batch(table, lens)
    k, v = (torch.zeros((3, H, hd), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q = torch.zeros((3, n_q, hd), dtype=torch.bfloat16, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros((3, n_q), device="cuda")
    L = S.lib()

    def step(stream):
        a = (P.dev.ref, 0, P.b.ref)
        S.check(L.sp_hip_fp4_write(*a, k.data_ptr(), v.data_ptr(), H * hd, S.DTYPE_BF16, stream), "write")
        S.check(L.sp_hip_fp4_attn_decode(*a, q.data_ptr(), n_q * hd, n_q, S.DTYPE_BF16, 0.1, 0, out.data_ptr(),
                                         n_q * hd, lse.data_ptr(), stream), "attend")
        S.check(L.sp_hip_fp4_weigh(*a, q.data_ptr(), n_q * hd, n_q, S.DTYPE_BF16, 0.1, 0, lse.data_ptr(), stream),
                "weigh")

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    P.set_lens([0, 0, 0])  # nothing to do while it is captured
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        step(torch.cuda.current_stream().cuda_stream)
    for turn in range(4):
        lens = [n + 1 for n in lens]
        P.set_lens(lens)
        kr, vr = P.rows(rng, "bf16"), P.rows(rng, "bf16")
        qr = queries(rng, P, n_q, "bf16")
        k.copy_(kr), v.copy_(vr), q.copy_(qr)
        torch.cuda.synchronize()
        before = P.weights()
        g.replay()
        torch.cuda.synchronize()
        P.ref.write(0, P.table, lens, None, 3, kr.double().numpy(), vr.double().numpy())
        P.check_memory(weights=False)
        got = out.double().cpu().numpy()
        eager, elng = P.check_attend("bf16", qr, 0.1)
        assert np.array_equal(got, eager) and np.array_equal(lse.double().cpu().numpy(), elng)
        added = P.weights()
        P.ref.weight = before
        P.ref.write(0, P.table, lens, None, 3, kr.double().numpy(), vr.double().numpy())
        tol = P.ref.weigh(0, P.table, lens, None, 3, qr.double().numpy(), float(np.float32(0.1)), 0, elng)
        assert (np.abs(added - P.ref.weight) <= tol).all()


def test_without_a_stream_and_on_another():
    rng = np.random.default_rng(22)
    P = Pair(128, 2, 20)
    P.fill(rng, tables(rng, [500, 300], 20), [500, 300])
    P.batch(P.table, [500, 300])
    q = queries(rng, P, 8, "f16")
    a = P.attend("f16", q, 0.1)
    b = P.attend("f16", q, 0.1, stream=0)
    s = torch.cuda.Stream()
    c = P.attend("f16", q, 0.1, stream=s.cuda_stream)
    for x in (b, c):
        assert np.array_equal(a[0], x[0]) and np.array_equal(a[1], x[1])


def test_a_prompt_beside_a_decode_step():
    """One of each kind of attention call under way on two streams."""
    rng = np.random.default_rng(23)
    P = Pair(128, 4, 150)
    lens = [5000, 4000]
    P.batch(tables(rng, lens, 150), lens, [0, 40, 80])
    fill_device(rng, P)
    q = queries(rng, P, 32, "bf16").cuda()
    two = S.Fp4Batch(2, P.b.c.table_stride, P.keep[0].data_ptr(), P.keep[1].data_ptr())
    s = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for streams in ((s[0], s[0]), (s[0], s[1])):
        got = [torch.zeros((80, 32, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(5):
            S.check(S.lib().sp_hip_fp4_attn_prefill(P.dev.ref, 0, P.b.ref, q.data_ptr(), 4096, 32, S.DTYPE_BF16, 0.1, 0,
                                                    got[0].data_ptr(), 4096, None, streams[0].cuda_stream), "prefill")
            S.check(S.lib().sp_hip_fp4_attn_decode(P.dev.ref, 0, two.ref, q.data_ptr(), 4096, 32, S.DTYPE_BF16, 0.1, 0,
                                                   got[1].data_ptr(), 4096, None, streams[1].cuda_stream), "decode")
        torch.cuda.synchronize()
        outs.append(got)
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def test_init_reports_what_it_cannot_have():
    c = S.SpHipFp4Cache()
    import ctypes as C
    cfg = S.config(256, 64, 64)
    assert S.lib().sp_hip_fp4_cache_init(C.byref(c), C.byref(cfg), 1 << 21, None) == -1
    assert "memory" in S.last_error() and not c.priv
