"""The 8-bit block cache on the GPU against its numpy form in 64 bits: codes and scales
exactly, attention within bounds derived from its arithmetic (fp8_ref.bounds)."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import fp8_ref as R
import sp_hip as S
from gpu_util import d2h

pytestmark = pytest.mark.gpu

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": S.DTYPE_F32, "f16": S.DTYPE_F16, "bf16": S.DTYPE_BF16}
ESIZE = {"f32": 4, "f16": 2, "bf16": 2}


def cur():
    return torch.cuda.current_stream().cuda_stream


class Pair:
    """A device cache, its numpy form, and one batch description for both."""

    def __init__(self, hd, heads, n_blocks, layers=1):
        self.hd, self.heads, self.n_blocks, self.layers = hd, heads, n_blocks, layers
        self.dev = S.Fp8Cache(S.config(hd, layers, heads), n_blocks, cur())
        self.ref = R.RefCache(hd, layers, heads, n_blocks)

    def batch(self, table, lens, row=None, n_rows=None):
        stride = max(1, max((len(t) for t in table), default=1))
        self.table = [list(t) + [-1] * (stride - len(t)) for t in table]
        self.lens, self.row = list(lens), row
        self.n_rows = n_rows if n_rows is not None else (row[-1] if row is not None else len(lens))
        self.keep = [torch.tensor(x, dtype=torch.int32, device="cuda")
                     for x in (self.table, self.lens, row if row is not None else [0])]
        self.b = S.Fp8Batch(len(lens), stride, self.keep[0].data_ptr(), self.keep[1].data_ptr(),
                            self.keep[2].data_ptr() if row is not None else 0, self.n_rows)
        return self.b

    def batch_of(self, lens, row):
        """Another batch over the same table; the arrays of earlier ones stay."""
        self.kept = getattr(self, "kept", []) + [self.keep]
        self.batch(self.table, lens, row)
        return self

    def set_lens(self, lens):
        self.lens = list(lens)
        self.keep[1].copy_(torch.tensor(lens, dtype=torch.int32))

    def rows(self, rng, dtype, spread=1.0):
        x = rng.standard_normal((self.n_rows, self.heads, self.hd)) * np.exp(spread * rng.standard_normal(
            (self.n_rows, self.heads, 1)))
        return torch.from_numpy(x).to(TORCH[dtype])

    def write(self, dtype, k, v, layer=0, pad=0, shift=0):
        """k, v: torch rows on the host or None; pad: spare elements between rows; shift: elements
        in front (an address that no vector load takes)."""
        width = self.heads * self.hd
        dev = []
        for x in (k, v):
            if x is None:
                dev.append(None)
                continue
            t = torch.full((shift + self.n_rows * (width + pad),), float("nan"), dtype=TORCH[dtype])
            t[shift:].view(self.n_rows, width + pad)[:, :width] = x.reshape(self.n_rows, width)
            dev.append(t.cuda())
        ptr = [t.data_ptr() + shift * ESIZE[dtype] if t is not None else None for t in dev]
        S.check(S.lib().sp_hip_fp8_write(self.dev.ref, layer, self.b.ref, ptr[0], ptr[1], width + pad, CODE[dtype],
                                         cur()), "write")
        self.ref.write(layer, self.table, self.lens, self.row, self.n_rows,
                       *[x.double().numpy() if x is not None else None for x in (k, v)])
        torch.cuda.synchronize()

    def check_memory(self):
        c = self.dev.c
        n = self.layers * self.n_blocks * self.heads
        for side, (codes, exps) in enumerate(((c.d_k_codes, c.d_k_exp), (c.d_v_codes, c.d_v_exp))):
            got = d2h(codes, n * 64 * self.hd).reshape(self.layers, self.n_blocks, self.heads, -1)
            want = self.ref.tiles(side)
            np.testing.assert_array_equal(d2h(exps, n).reshape(self.ref.exps[side].shape), self.ref.exps[side])
            np.testing.assert_array_equal(np.where(got == 128, 0, got), np.where(want == 128, 0, want))

    def fill(self, rng, table, lens, dtype="f32", spread=1.0, layer=0):
        """Write whole sequences."""
        row = np.concatenate([[0], np.cumsum(lens)]).tolist()
        self.batch(table, lens, row)
        self.write(dtype, self.rows(rng, dtype, spread), self.rows(rng, dtype, spread), layer)

    def attend(self, dtype, q, scale, window=0, layer=0, pad=0, shift=0, stream=None, want_lse=True):
        n_q = q.shape[1]
        width = n_q * self.hd
        qt = torch.full((shift + self.n_rows * (width + pad),), float("nan"), dtype=TORCH[dtype])
        qt[shift:].view(self.n_rows, width + pad)[:, :width] = q.reshape(self.n_rows, width)
        qt = qt.cuda()
        out = torch.full((shift + self.n_rows * (width + pad),), 77.0, dtype=TORCH[dtype], device="cuda")
        lse = torch.full((self.n_rows, n_q), 77.0, dtype=torch.float32, device="cuda")
        L = S.lib()
        call = L.sp_hip_fp8_attn_prefill if self.row is not None else L.sp_hip_fp8_attn_decode
        torch.cuda.synchronize()
        S.check(call(self.dev.ref, layer, self.b.ref, qt.data_ptr() + shift * ESIZE[dtype], width + pad, n_q,
                     CODE[dtype], scale, window, out.data_ptr() + shift * ESIZE[dtype], width + pad,
                     lse.data_ptr() if want_lse else None, stream if stream is not None else cur()), "attend")
        torch.cuda.synchronize()
        o = out.cpu()
        rows = o[shift:].view(self.n_rows, width + pad)
        assert (o[:shift] == 77.0).all() and (rows[:, width:] == 77.0).all(), "written between the rows"
        return rows[:, :width].reshape(self.n_rows, n_q, self.hd).double().numpy(), lse.double().cpu().numpy()

    def check_attend(self, dtype, q, scale, window=0, layer=0, pad=0, shift=0, stream=None):
        out, lse = self.attend(dtype, q, scale, window, layer, pad, shift, stream)
        want, wlse, reach, steep = self.ref.attend(layer, self.table, self.lens, self.row, self.n_rows,
                                                   q.double().numpy(), scale, window)
        mine = ~np.isnan(wlse)
        assert (out[~mine] == 77.0).all() and (lse[~mine] == 77.0).all(), "a row of no sequence was written"
        tol, ltol = R.bounds(dtype, self.hd, max(self.lens + [1]), want, reach, steep)
        empty = np.isneginf(wlse)
        assert (out[empty] == 0).all() and np.isneginf(lse[empty]).all()
        live = mine & ~empty
        d, dl = np.abs(out[live] - want[live]), np.abs(lse[live] - wlse[live])
        assert (d <= tol[live]).all(), (float((d - tol[live]).max()), float(d.max()))
        assert (dl <= ltol[live] + 2.0 ** -23 * np.abs(wlse[live])).all(), float(dl.max())
        return out, lse


def queries(rng, pair, n_q, dtype):
    return torch.from_numpy(rng.standard_normal((pair.n_rows, n_q, pair.hd)) *
                            np.exp(rng.standard_normal((pair.n_rows, n_q, 1)))).to(TORCH[dtype])


def tables(rng, lens, n_blocks, extra=0):
    order = rng.permutation(n_blocks).tolist()
    out = []
    for n in lens:
        m = (n + 63) // 64 + extra
        out.append(order[:m])
        order = order[m:]
    return out


# ---- write and read ----

@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_write_then_appends(hd, dtype):
    rng = np.random.default_rng(hd)
    P = Pair(hd, 3, 24, layers=2)
    lens = [1, 64, 65, 200, 131]
    table = tables(rng, [n + 130 for n in lens], 24)
    P.fill(rng, table, lens, dtype)
    P.check_memory()
    # rows appended inside blocks, some strong enough to raise the scale by several octaves
    for step, news in enumerate(([1, 1, 1, 1, 1], [3, 0, 70, 64, 2], [1, 5, 0, 0, 63])):
        lens = [n + m for n, m in zip(lens, news)]
        P.batch(table, lens, np.concatenate([[0], np.cumsum(news)]).tolist(), sum(news) + step)
        for side in range(2):
            k = P.rows(rng, dtype, 2.0) if side == 0 else None
            v = P.rows(rng, dtype, 2.0) if side == 1 else None
            P.write(dtype, k, v, layer=1, pad=step * 4, shift=(0, 0, 1)[step])
        P.check_memory()


def test_one_row_each_and_rewriting():
    rng = np.random.default_rng(5)
    P = Pair(128, 2, 8)
    P.batch([[3], [5], [1]], [1, 1, 1])
    P.write("f16", P.rows(rng, "f16"), P.rows(rng, "f16"))
    P.check_memory()
    for n in (2, 3):  # strengths 2^12 apart: codes go subnormal and vanish
        P.batch([[3], [5], [1]], [n, n, n])
        P.write("f16", P.rows(rng, "f16") * 2.0 ** (5 * (n - 1)), P.rows(rng, "f16") * 2.0 ** -n)
        P.check_memory()
    P.batch([[3], [5], [1]], [2, 1, 3])  # a shorter sequence goes on from there; a fresh one starts anew
    P.write("f16", P.rows(rng, "f16"), P.rows(rng, "f16"))
    P.check_memory()


def test_extremes_are_finite():
    P = Pair(64, 1, 4)
    P.batch([[0, 1, 2]], [130], [0, 130])
    k = torch.zeros(130, 1, 64)
    k[0, 0, 0], k[1, 0, 1], k[2, 0, 2] = float("nan"), float("inf"), -float("inf")
    k[3, 0, 3] = 1.0
    k[70, 0, 5] = 1e-30           # below what the least scale holds
    k[129, 0, 7] = 3e38
    v = torch.full((130, 1, 64), 2.0 ** -45)
    v[5] = float("nan")
    P.write("f32", k, v)
    P.check_memory()
    got = d2h(P.dev.c.d_k_codes, 4 * 64 * 64)
    assert not np.any((got & 127) == 127)


def test_absent_positions_are_passed_over():
    rng = np.random.default_rng(9)
    P = Pair(128, 2, 6)
    # blocks past the pool, negative entries, a length past the table, rows before position 0
    P.batch([[0, 6, 1], [-1, 2, 7], [3, 4, 5], [-7, 1 << 30, 3]], [192, 130, 300, 5], [0, 192, 322, 522, 530], 541)
    k, v = P.rows(rng, "bf16"), P.rows(rng, "bf16")
    P.write("bf16", k, v)
    P.check_memory()
    out = [torch.full((541, 2, 128), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    S.check(S.lib().sp_hip_fp8_read(P.dev.ref, 0, P.b.ref, out[0].data_ptr(), out[1].data_ptr(), 256, S.DTYPE_BF16,
                                    cur()), "read")
    torch.cuda.synchronize()
    for side in range(2):
        want = np.full((541, 2, 128), 7.0)
        for _, r, b, at, _ in P.ref.places(P.table, P.lens, P.row, 541):
            want[r] = P.ref.values(side, 0, b)[:, at] if b >= 0 else 0.0
        np.testing.assert_array_equal(out[side].cpu().double().numpy(),
                                      torch.from_numpy(want).bfloat16().double().numpy())


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_read(hd, dtype):
    rng = np.random.default_rng(hd + 1)
    P = Pair(hd, 3, 16, layers=2)
    lens = [1, 64, 127, 300]
    P.fill(rng, tables(rng, lens, 16), lens, "f32", 0.5, layer=1)
    for news, pad, shift in (([1, 1, 1, 1], 0, 0), (lens, 8, 0), ([1, 30, 64, 299], 3, 1)):
        row = None if max(news) == 1 else np.concatenate([[0], np.cumsum(news)]).tolist()
        P.batch(P.table, lens, row)
        width = 3 * hd
        got = []
        for _ in range(2):
            t = torch.full((shift + P.n_rows * (width + pad),), 7.0, dtype=TORCH[dtype], device="cuda")
            got.append(t)
        p = [t.data_ptr() + shift * ESIZE[dtype] for t in got]
        S.check(S.lib().sp_hip_fp8_read(P.dev.ref, 1, P.b.ref, p[0], p[1], width + pad, CODE[dtype], cur()), "read")
        torch.cuda.synchronize()
        for side, t in enumerate(got):
            t = t.cpu()
            assert (t[:shift] == 7.0).all()
            t = t[shift:].view(P.n_rows, width + pad)
            assert (t[:, width:] == 7.0).all()
            want = np.stack([P.ref.values(side, 1, b)[:, at] for _, _, b, at, _ in
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
    q = queries(rng, P, 2, "f32")
    P.check_attend("f32", q, 0.125)


def test_many_sequences_one_long():
    """Shares of a long sequence found behind more sequences than a wave has lanes."""
    rng = np.random.default_rng(13)
    P = Pair(64, 2, 330)
    lens = [1 + (i * 29) % 130 for i in range(130)]
    lens[97] = 5000
    table = tables(rng, lens, 330)
    P.fill(rng, table, lens)
    P.batch(table, lens)
    P.check_attend("f16", queries(rng, P, 8, "f16"), 0.2)
    news = [min(n, 1 + i % 7) for i, n in enumerate(lens)]
    P.batch(table, lens, np.concatenate([[0], np.cumsum(news)]).tolist(), sum(news) + 1)
    P.check_attend("f32", queries(rng, P, 4, "f32"), 0.2, window=3000)


def test_many_sequences_of_many_rows():
    rng = np.random.default_rng(14)
    lens = [40 + (i * 31) % 60 for i in range(70)]
    lens[68] = 1900
    P = Pair(64, 1, 190)
    table = tables(rng, lens, 190)
    P.fill(rng, table, lens)
    P.batch(table, lens, [33 * i for i in range(71)])
    for dtype in ("bf16", "f32"):
        P.check_attend(dtype, queries(rng, P, 4, dtype), 0.2)


def test_lengths_past_everything():
    """Lengths at the end of an int: the table's positions are all seen, the rows' own are not there."""
    rng = np.random.default_rng(15)
    P = Pair(64, 1, 6)
    P.fill(rng, [[0, 1], [2, 3, 4]], [128, 192])
    P.batch([[0, 1, -1], [2, 3, 4]], [128, 192])
    q = queries(rng, P, 2, "f32")
    want = P.attend("f32", q, 0.2)
    for row in (None, [0, 1, 2]):
        P.batch([[0, 1, -1], [2, 3, 4]], [2 ** 31 - 1, 2 ** 30 + 7], row)
        before = d2h(P.dev.c.d_k_codes, 6 * 64 * 64).copy()
        k = torch.ones(2, 1, 64, device="cuda")
        S.check(S.lib().sp_hip_fp8_write(P.dev.ref, 0, P.b.ref, k.data_ptr(), k.data_ptr(), 64, S.DTYPE_F32, cur()), "w")
        assert np.array_equal(before, d2h(P.dev.c.d_k_codes, 6 * 64 * 64))
        got = P.attend("f32", q, 0.2)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_rows_array_out_of_order_touches_nothing_else():
    """An array of rows that does not ascend: within the call's rows and blocks whatever it holds."""
    rng = np.random.default_rng(4)
    P = Pair(64, 1, 8)
    P.fill(rng, [[0, 1], [2, 3]], [100, 90])
    P.batch([[0, 1], [2, 3]], [100, 90], [0, 50, 20], 20)
    P.row = [0, 9, 20]  # (unused)
    S.check(S.lib().sp_hip_fp8_write(P.dev.ref, 0, P.b.ref, torch.zeros(20 * 64, device="cuda").data_ptr(), None, 64,
                                     S.DTYPE_F32, cur()), "write")
    q = torch.zeros(20 * 64, device="cuda")
    out = torch.zeros(20 * 64 + 64, device="cuda")
    P.keep.append(torch.tensor([-5, 60, -3], dtype=torch.int32, device="cuda"))
    b = S.Fp8Batch(2, 2, P.keep[0].data_ptr(), P.keep[1].data_ptr(), P.keep[-1].data_ptr(), 20)
    S.check(S.lib().sp_hip_fp8_attn_prefill(P.dev.ref, 0, b.ref, q.data_ptr(), 64, 1, S.DTYPE_F32, 1.0, 0,
                                            out.data_ptr(), 64, None, cur()), "attend")
    torch.cuda.synchronize()
    assert (out[20 * 64:] == 0).all()
    # and the next call finds its workspace as it should be
    P.batch([[4, 5], [2, 3]], [128, 90])
    P.fill(rng, [[4, 5], [2, 3]], [128, 90])
    P.batch([[4, 5], [2, 3]], [128, 90])
    P.ref.codes[:, 0, [0, 1]] = 0
    P.check_attend("f32", queries(rng, P, 2, "f32"), 0.2)


# ---- attention ----

LENS = [1, 0, 63, 64, 65, 700, 129]


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


@pytest.mark.parametrize("group", [1, 3, 7, 15, 16, 17, 40])
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


@pytest.mark.parametrize("group", [1, 2, 5, 16, 33])
@pytest.mark.parametrize("new", [2, 17, 128])
def test_prefill_groups(group, new):
    rng = np.random.default_rng(group)
    P = Pair(64, 2, 30)
    lens = [new, 700, 333]
    P.fill(rng, tables(rng, lens, 30), lens)
    news = [new, new, 1]
    P.batch(P.table, lens, [0, new, 2 * new, 2 * new + 1])
    for dtype in ("f16", "f32"):
        P.check_attend(dtype, queries(rng, P, 2 * group, dtype), 0.2)


@pytest.mark.parametrize("new,length", [(1, 20000), (6, 20001), (300, 9000), (1, 131072), (257, 30000)])
def test_long_sequences(new, length):
    """Work split over many shares of one sequence."""
    rng = np.random.default_rng(new)
    P = Pair(64, 1, (length + 63) // 64 + 2)
    P.fill(rng, tables(rng, [length], P.n_blocks), [length])
    P.batch(P.table, [length], None if new == 1 else [0, new])
    for dtype in ("bf16", "f32"):
        a = P.check_attend(dtype, queries(rng, P, 4, dtype), 0.2)
    P.check_attend("f16", queries(rng, P, 4, "f16"), 0.2, window=5000)
    q = queries(rng, P, 4, "f32")
    a, b = P.attend("f32", q, 0.2), P.attend("f32", q, 0.2)
    assert all(np.array_equal(x, y) for x, y in zip(a, b)), "the order of arrival shows"


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_many_rows_shared_out(hd, dtype):
    """Column groups of many rows whose cache blocks are divided over blocks of threads, beside
    sequences that are not: one row, no rows, rows at the start."""
    rng = np.random.default_rng(hd)
    P = Pair(hd, 2, 80)
    lens = [2500, 40, 700, 0]
    news = [150, 1, 0, 0] if hd < 256 else [149, 3, 0, 0]
    P.fill(rng, tables(rng, lens, 80, extra=1), lens, "f32", 0.5)
    row = np.concatenate([[0], np.cumsum(news)]).tolist()
    for group, scale, window, pad in ((8, 1 / math.sqrt(hd), 0, 0), (9, -0.2, 1500, 8), (8, 0.0, 0, 1)):
        P.batch(P.table, lens, row, row[-1] + 2)
        P.check_attend(dtype, queries(rng, P, 2 * group, dtype), scale, window, pad=pad)


def test_tables_with_holes():
    rng = np.random.default_rng(12)
    P = Pair(128, 2, 12)
    lens = [640, 300]
    P.fill(rng, tables(rng, lens, 12, extra=-1), [576, 256])
    t = [list(x) for x in P.table]
    t[0] = t[0][:9] + [-1]
    t[0][3], t[0][8] = -1, 99
    t[1] = [12, -5, 1 << 30, t[1][2]] + [-1]
    P.batch(t, lens)
    P.check_attend("f32", queries(rng, P, 8, "f32"), 0.1)
    P.batch(t, lens, [0, 130, 133])
    P.check_attend("f16", queries(rng, P, 8, "f16"), 0.1, window=150)
    P.batch(t, lens, [0, 500, 790])  # many rows
    for dtype, window in (("f16", 150), ("bf16", 0), ("f32", 333)):
        P.check_attend(dtype, queries(rng, P, 8, dtype), 0.1, window=window)
    P.batch([[-1, -1], [-1, 12]], [128, 100])  # nothing to see at all
    P.check_attend("f16", queries(rng, P, 8, "f16"), 0.1)


@pytest.mark.parametrize("kind", ["v", "k", "q"])
def test_scales_far_apart(kind):
    """Blocks whose scales are up to 2^70 apart, and weak blocks that carry all the weight."""
    rng = np.random.default_rng(2)
    P = Pair(64, 1, 10)
    P.batch([[0, 1, 2, 3, 4, 5]], [384], [0, 384])
    k, v = P.rows(rng, "f32", 0.0), P.rows(rng, "f32", 0.0)
    k *= 0.1
    for j, e in enumerate((30, -35, 0, 35, -30, 4)):
        (v if kind == "v" else k)[64 * j:64 * j + 64] *= 2.0 ** (e if kind == "v" else e / 8 - 4)
    if kind == "v":
        k[64:128] += 1.0  # the weakest values are seen best by a positive query
    P.write("f32", k, v)
    q = torch.from_numpy(np.abs(rng.standard_normal((384, 2, 64))))
    scale = 0.5
    if kind == "q":
        q = q / q.abs().amax(-1, keepdim=True) * 2.0 ** 60
        scale = 2.0 ** -58
    for dtype in ("f32", "bf16"):
        P.check_attend(dtype, q.to(TORCH[dtype]), scale)
        P.check_attend(dtype, torch.cat([q, q, q], 1).to(TORCH[dtype]), scale)  # many rows
        P.batch([[0, 1, 2, 3, 4, 5]], [384])
        P.check_attend(dtype, q[:1].to(TORCH[dtype]), scale)
        P.batch([[0, 1, 2, 3, 4, 5]], [384], [0, 384])


def test_masked_places_hold_nothing_that_shows():
    """What lies behind a sequence's length, before its window or in another sequence's rows
    of the call: NaN and infinity were written there."""
    rng = np.random.default_rng(8)
    P = Pair(128, 1, 6)
    P.batch([[2, 4, 1]], [192], [0, 192])
    k, v = P.rows(rng, "f32", 0.3), P.rows(rng, "f32", 0.3)
    for x in (k, v):
        x[:20] = float("inf")
        x[20:30] = float("nan")
        x[150:] = 3e38
    P.write("f32", k, v)
    P.batch([[2, 4, 1]], [140], [0, 100])
    for n_q in (4, 12):
        P.check_attend("bf16", queries(rng, P, n_q, "bf16"), 0.1, window=90)
    P.batch([[2, 4, 1]], [150])
    P.check_attend("f32", queries(rng, P, 4, "f32"), 0.1, window=64)


def test_not_finite_queries_stay_in_their_rows():
    rng = np.random.default_rng(8)
    P = Pair(64, 2, 8)
    P.fill(rng, tables(rng, [200, 130], 8), [200, 130])
    for row, n_q in ((None, 4), ([0, 70, 100], 4), ([0, 200, 330], 8)):
        P.batch(P.table, [200, 130], row)
        q = queries(rng, P, n_q, "f32")
        good = P.attend("f32", q, 0.1)
        bad = q.clone()
        bad[1, 1, 3] = float("nan")
        bad[0, 2, 5] = float("inf")
        got = P.attend("f32", bad, 0.1)
        same = np.ones(q.shape[:2], bool)
        same[1, 1] = same[0, 2] = False
        assert np.array_equal(got[0][same], good[0][same]) and np.array_equal(got[1][same], good[1][same])
        assert np.isnan(got[0][1, 1]).all() and np.isnan(got[1][1, 1])
        assert not np.isfinite(got[0][0, 2]).any()


def test_blocks_past_4_gib():
    """Codes of one side in more than 2^32 bytes."""
    rng = np.random.default_rng(6)
    P = Pair.__new__(Pair)
    hd, H, n = 256, 8, 33000  # 128 KiB a block and side
    P.hd, P.heads, P.layers, P.n_blocks = hd, H, 1, n
    P.dev = S.Fp8Cache(S.config(hd, 1, H), n, cur())
    few = R.RefCache(hd, 1, H, 4)  # the blocks that the test uses, renumbered
    far = [32999, 3, 32768, 32767]
    rngk = rng.standard_normal((240, H, hd)).astype(np.float32)
    P.batch([far], [240], [0, 240])
    k, v = torch.from_numpy(rngk), torch.from_numpy(rngk[::-1].copy())
    kd, vd = k.cuda(), v.cuda()
    S.check(S.lib().sp_hip_fp8_write(P.dev.ref, 0, P.b.ref, kd.data_ptr(), vd.data_ptr(), H * hd, S.DTYPE_F32, cur()),
            "write")
    few.write(0, [[0, 1, 2, 3]], [240], [0, 240], 240, k.double().numpy(), v.double().numpy())
    got = [torch.empty(240, H, hd, device="cuda") for _ in range(2)]
    S.check(S.lib().sp_hip_fp8_read(P.dev.ref, 0, P.b.ref, got[0].data_ptr(), got[1].data_ptr(), H * hd, S.DTYPE_F32,
                                    cur()), "read")
    torch.cuda.synchronize()
    for side in range(2):
        want = np.concatenate([few.values(side, 0, b) for b in range(4)], 1)[:, :240].transpose(1, 0, 2)
        np.testing.assert_array_equal(got[side].cpu().double().numpy(), want)
    P.batch([far], [240], [0, 9])
    q = queries(rng, P, 16, "bf16")
    out, lse = P.attend("bf16", q, 1 / 16)
    want, wlse, reach, steep = few.attend(0, [[0, 1, 2, 3]], [240], [0, 9], 9, q.double().numpy(), 1 / 16, 0)
    tol, ltol = R.bounds("bf16", hd, 240, want, reach, steep)
    assert (np.abs(out - want) <= tol).all() and (np.abs(lse - wlse) <= ltol + 2.0 ** -23 * np.abs(wlse)).all()
    P.dev.free()


# ---- rows enough for the kernel that takes a block over many columns (columns of all KV heads) ----

@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window", [0, 77])
def test_many_columns(hd, dtype, window):
    rng = np.random.default_rng(hd + 9)
    P = Pair(hd, 4, 20)
    lens, news = [1, 0, 500, 129, 65, 63], [1, 0, 437, 64, 0, 70]  # the last: more rows than positions
    P.fill(rng, tables(rng, lens, 20, extra=1), lens, "f32", 0.5)
    row = np.concatenate([[0], np.cumsum(news)]).tolist()
    for group, scale, kw in ((6, 1 / math.sqrt(hd), {}), (7, -0.3, dict(pad=3, shift=1)), (6, 0.0, dict(pad=8))):
        P.batch(P.table, lens, row, row[-1] + 3)
        P.check_attend(dtype, queries(rng, P, 4 * group, dtype), scale, window, **kw)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_many_columns_shared_out(hd, dtype):
    rng = np.random.default_rng(hd + 1)
    P = Pair(hd, 2, 80)
    lens, news = [2500, 40, 700, 0], [450, 1, 0, 0]
    P.fill(rng, tables(rng, lens, 80, extra=1), lens, "f32", 0.5)
    row = np.concatenate([[0], np.cumsum(news)]).tolist()
    for window, pad in ((0, 0), (1500, 1)):
        P.batch(P.table, lens, row, row[-1] + 2)
        q = queries(rng, P, 28, dtype)
        a = P.check_attend(dtype, q, 1 / math.sqrt(hd), window, pad=pad)
    b = P.attend(dtype, q, 1 / math.sqrt(hd), window, pad=pad)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_many_columns_of_many_sequences():
    rng = np.random.default_rng(14)
    lens = [40 + (i * 31) % 60 for i in range(70)]
    lens[68] = 1900
    P = Pair(64, 4, 190)
    table = tables(rng, lens, 190)
    P.fill(rng, table, lens)
    P.batch(table, lens, [33 * i for i in range(71)])
    for dtype in ("bf16", "f32"):
        P.check_attend(dtype, queries(rng, P, 16, dtype), 0.2)


@pytest.mark.parametrize("hd", [128, 256])
def test_many_columns_over_holes(hd):
    rng = np.random.default_rng(12)
    P = Pair(hd, 8, 12)
    lens = [640, 300]
    P.fill(rng, tables(rng, lens, 12, extra=-1), [576, 256])
    t = [list(x) for x in P.table]
    t[0] = t[0][:9] + [-1]
    t[0][3], t[0][8] = -1, 99
    t[1] = [12, -5, 1 << 30, t[1][2]] + [-1]
    P.batch(t, lens, [0, 500, 790])
    for dtype, window in (("f16", 150), ("bf16", 0), ("f32", 333)):
        P.check_attend(dtype, queries(rng, P, 16, dtype), 0.1, window=window)
    P.batch([[-1, -1], [-1, 12]], [500, 400], [0, 500, 900])  # nothing to see at all
    P.check_attend("f16", queries(rng, P, 16, "f16"), 0.1)


@pytest.mark.parametrize("kind", ["v", "k", "q"])
def test_many_columns_scales_far_apart(kind):
    rng = np.random.default_rng(2)
    for hd in (64, 128):
        P = Pair(hd, 1, 10)
        P.batch([[0, 1, 2, 3, 4, 5]], [384], [0, 384])
        k, v = P.rows(rng, "f32", 0.0), P.rows(rng, "f32", 0.0)
        k *= 0.1
        for j, e in enumerate((30, -35, 0, 35, -30, 4)):
            (v if kind == "v" else k)[64 * j:64 * j + 64] *= 2.0 ** (e if kind == "v" else e / 8 - 4)
        if kind == "v":
            k[64:128] += 1.0
        P.write("f32", k, v)
        q = torch.from_numpy(np.abs(rng.standard_normal((384, 32, hd))))
        scale = 0.5 * 64 / hd
        if kind == "q":
            q = q / q.abs().amax(-1, keepdim=True) * 2.0 ** 60
            scale *= 2.0 ** -57
        for dtype in ("f32", "bf16"):
            P.check_attend(dtype, q.to(TORCH[dtype]), scale)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_many_columns_not_finite(hd):
    """Queries that are not finite stay in their rows, what was written as such in masked places
    does not show."""
    rng = np.random.default_rng(8)
    P = Pair(hd, 4, 8)
    row = [0, 200, 330]
    P.batch(tables(rng, [250, 130], 8), [250, 130], [0, 250, 380])
    k, v = P.rows(rng, "f32", 0.3), P.rows(rng, "f32", 0.3)
    for x in (k, v):
        x[:20], x[20:30], x[240:250] = float("inf"), float("nan"), 3e38
    P.write("f32", k, v)
    P.batch(P.table, [240, 130], row)
    for dtype in ("f32", "bf16"):
        q = queries(rng, P, 40, dtype)
        good = P.check_attend(dtype, q, 0.1, window=10)
        bad = q.clone()
        bad[1, 1, 3] = float("nan")
        bad[0, 2, 5] = float("inf")
        got = P.attend(dtype, bad, 0.1, window=10)
        same = np.ones(q.shape[:2], bool)
        same[1, 1] = same[0, 2] = False
        assert np.array_equal(got[0][same], good[0][same]) and np.array_equal(got[1][same], good[1][same])
        assert np.isnan(got[0][1, 1]).all() and np.isnan(got[1][1, 1])
        assert not np.isfinite(got[0][0, 2]).any()


def test_captured_chunk_of_many_columns():
    """One graph of a chunk's attention, its shares joined by a second launch, replayed over more
    of a sequence that is there already."""
    rng = np.random.default_rng(34)
    P = Pair(64, 2, 80)
    table = tables(rng, [4000], 80)
    new, n_q = 130, 96
    P.fill(rng, table, [4000])
    P.batch(table, [1500], [0, new])
    q = queries(rng, P, n_q, "bf16").cuda()
    out, lse = torch.zeros_like(q), torch.zeros(new, n_q, device="cuda")

    def step(stream):
        S.check(S.lib().sp_hip_fp8_attn_prefill(P.dev.ref, 0, P.b.ref, q.data_ptr(), n_q * 64, n_q, S.DTYPE_BF16, 0.125,
                                                0, out.data_ptr(), n_q * 64, lse.data_ptr(), stream), "a")

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(cur())
    for length in (1630, 200, 3900):
        P.set_lens([length])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = P.check_attend("bf16", q.cpu(), 0.125)
        assert np.array_equal(out.double().cpu().numpy(), eager[0])
        assert np.array_equal(lse.double().cpu().numpy(), eager[1])


# ---- as a server uses them ----

def test_a_prompt_then_steps_then_proposals():
    """Two layers: a prompt in chunks, decode steps, then proposed tokens of which some are taken
    back, each attending over what the calls before it wrote."""
    rng = np.random.default_rng(21)
    P = Pair(128, 2, 40, layers=2)
    table = tables(rng, [500, 300, 260], 40, extra=1)
    lens = [0, 0, 0]
    for news in ([100, 33, 64], [150, 200, 1], [1, 1, 1], [1, 1, 1], [5, 5, 5], [-3, -1, -5], [1, 1, 1], [70, 1, 3]):
        lens = [n + m for n, m in zip(lens, news)]
        if min(news) < 0:
            continue  # taken back
        row = None if max(news) == 1 else np.concatenate([[0], np.cumsum(news)]).tolist()
        P.batch(table, lens, row)
        for layer in range(2):
            P.write("bf16", P.rows(rng, "bf16", 0.5), P.rows(rng, "bf16", 0.5), layer)
            P.check_attend("bf16", queries(rng, P, 8, "bf16"), 0.09, layer=layer)
        P.check_memory()


def test_captured_step_follows_lengths_and_tables():
    """One graph of a write and an attention call, replayed as the sequences grow; the cache's
    other calls run between replays."""
    rng = np.random.default_rng(31)
    P = Pair(128, 2, 48)
    lens = [1000, 70, 3]
    table = tables(rng, [1100, 200, 100], 48)
    P.fill(rng, table, lens)
    P.batch(table, lens)
    k, v = (torch.zeros(3, 2, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    q = torch.zeros(3, 8, 128, dtype=torch.float16, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros(3, 8, device="cuda")
    L = S.lib()

    def step(stream):
        S.check(L.sp_hip_fp8_write(P.dev.ref, 0, P.b.ref, k.data_ptr(), v.data_ptr(), 256, S.DTYPE_F16, stream), "w")
        S.check(L.sp_hip_fp8_attn_decode(P.dev.ref, 0, P.b.ref, q.data_ptr(), 1024, 8, S.DTYPE_F16, 0.1, 0,
                                         out.data_ptr(), 1024, lse.data_ptr(), stream), "a")

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(side.cuda_stream)
    torch.cuda.synchronize()
    # the call above wrote zeros at the newest positions, in the numpy form too
    P.ref.write(0, P.table, P.lens, None, 3, *[np.zeros((3, 2, 128))] * 2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(cur())
    for n in range(4):
        lens = [x + (63 if n == 2 and i == 1 else 1) for i, x in enumerate(lens)]
        P.set_lens(lens)
        rows = [P.rows(rng, "f16") for _ in range(2)]
        qs = queries(rng, P, 8, "f16")
        k.copy_(rows[0]), v.copy_(rows[1]), q.copy_(qs)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        P.ref.write(0, P.table, lens, None, 3, *[x.double().numpy() for x in rows])
        P.check_memory()
        got = out.double().cpu().numpy(), lse.double().cpu().numpy()
        eager = P.check_attend("f16", qs, 0.1)
        assert np.array_equal(got[0], eager[0]) and np.array_equal(got[1], eager[1])


def test_captured_chunk_follows_lengths():
    """One graph of a chunk's write and attention, its shares joined by a second launch, replayed as
    the sequence grows."""
    rng = np.random.default_rng(33)
    P = Pair(64, 2, 80)
    table = tables(rng, [4000], 80)
    new, n_q = 130, 16
    P.fill(rng, table, [1500])
    P.batch(table, [1500], [0, new])
    k, v = (torch.zeros(new, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q = torch.zeros(new, n_q, 64, dtype=torch.bfloat16, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros(new, n_q, device="cuda")
    L = S.lib()

    def step(stream):
        S.check(L.sp_hip_fp8_write(P.dev.ref, 0, P.b.ref, k.data_ptr(), v.data_ptr(), 128, S.DTYPE_BF16, stream), "w")
        S.check(L.sp_hip_fp8_attn_prefill(P.dev.ref, 0, P.b.ref, q.data_ptr(), n_q * 64, n_q, S.DTYPE_BF16, 0.125, 0,
                                          out.data_ptr(), n_q * 64, lse.data_ptr(), stream), "a")

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(cur())
    for length in (1630, 1760, 3900):
        P.set_lens([length])
        rows = [P.rows(rng, "bf16") for _ in range(2)]
        qs = queries(rng, P, n_q, "bf16")
        k.copy_(rows[0]), v.copy_(rows[1]), q.copy_(qs)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        P.ref.write(0, P.table, P.lens, P.row, new, *[x.double().numpy() for x in rows])
        P.check_memory()
        eager = P.check_attend("bf16", qs, 0.125)
        assert np.array_equal(out.double().cpu().numpy(), eager[0])
        assert np.array_equal(lse.double().cpu().numpy(), eager[1])


def test_another_stream_and_two_caches():
    rng = np.random.default_rng(41)
    A, B = Pair(128, 2, 40), Pair(64, 4, 40)
    for P in (A, B):
        P.fill(rng, tables(rng, [1500, 600], 40), [1500, 600])
        P.batch(P.table, [1500, 600])
    streams = [torch.cuda.Stream() for _ in range(2)]
    qs = [queries(rng, A, 8, "f16").cuda(), queries(rng, B, 8, "f16").cuda()]
    outs = [torch.zeros_like(x) for x in qs]
    want = [P.attend("f16", q.cpu(), 0.1)[0] for P, q in zip((A, B), qs)]
    torch.cuda.synchronize()
    for _ in range(5):
        for P, s, q, o in zip((A, B), streams, qs, outs):
            S.check(S.lib().sp_hip_fp8_attn_decode(P.dev.ref, 0, P.b.ref, q.data_ptr(), 8 * P.hd, 8, S.DTYPE_F16, 0.1,
                                                   0, o.data_ptr(), 8 * P.hd, None, s.cuda_stream), "a")
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert np.array_equal(o.double().cpu().numpy(), w)


def test_without_a_stream_the_caches_own_is_used():
    rng = np.random.default_rng(43)
    P = Pair(64, 1, 8)
    own = torch.cuda.Stream()
    P.dev = S.Fp8Cache(S.config(64, 1, 1), 8, own.cuda_stream)
    P.batch([[1, 2]], [100], [0, 100])
    k = P.rows(rng, "f32").cuda()
    torch.cuda.synchronize()
    S.check(S.lib().sp_hip_fp8_write(P.dev.ref, 0, P.b.ref, k.data_ptr(), None, 64, S.DTYPE_F32, None), "write")
    back = torch.zeros_like(k)
    torch.cuda.synchronize()
    S.check(S.lib().sp_hip_fp8_read(P.dev.ref, 0, P.b.ref, back.data_ptr(), None, 64, S.DTYPE_F32, None), "read")
    own.synchronize()
    P.ref.write(0, P.table, [100], [0, 100], 100, k.double().cpu().numpy(), None)
    want = np.concatenate([P.ref.values(0, 0, b) for b in (1, 2)], 1)[:, :100].transpose(1, 0, 2)
    np.testing.assert_array_equal(back.double().cpu().numpy(), want)


def test_init_reports_what_it_cannot_have():
    c = S.SpHipFp8Cache()
    cfg = S.config(128, 64, 64)
    assert S.lib().sp_hip_fp8_cache_init(C.byref(c), C.byref(cfg), 1 << 14, None) == -1  # 512 GiB a side
    assert "memory" in S.last_error() and not c.priv and not c.d_k_codes
    torch.zeros(4, device="cuda").add_(1)  # the failure is not left for the next user of the device
    torch.cuda.synchronize()
    assert S.lib().sp_hip_fp8_cache_init(C.byref(c), C.byref(S.config(128, 1, 1)), 4, None) == 0
    S.lib().sp_hip_fp8_cache_free(C.byref(c))


def test_a_prompt_beside_a_decode_step():
    """A prefill and a decode call on one cache at once, on two streams, both with shares to join."""
    rng = np.random.default_rng(47)
    P = Pair(128, 2, 300)
    lens = [9000, 8000]
    P.fill(rng, tables(rng, lens, 300), lens)
    q1, q2 = queries(rng, P.batch_of(lens, [0, 300, 300]), 8, "f16"), None
    a = P.b
    q2 = queries(rng, P.batch_of(lens, None), 8, "f16")
    b = P.b
    first = [t.cuda() for t in (q1, q2)]
    outs = [torch.zeros_like(t) for t in first]
    L, want = S.lib(), []
    streams = [torch.cuda.Stream() for _ in range(2)]

    def call(i, stream):
        f, batch = (L.sp_hip_fp8_attn_prefill, a) if i == 0 else (L.sp_hip_fp8_attn_decode, b)
        S.check(f(P.dev.ref, 0, batch.ref, first[i].data_ptr(), 1024, 8, S.DTYPE_F16, 0.1, 0, outs[i].data_ptr(), 1024,
                  None, stream), "attend")
    torch.cuda.synchronize()
    for i in range(2):
        call(i, cur())
        torch.cuda.synchronize()
        want.append(outs[i].clone())
    for _ in range(6):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            call(i, streams[i].cuda_stream)
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
