"""The 8-bit block cache's attention where its kernels take a path that small calls do not: more cache
blocks than a wave looks up at once, row arrays that do not ascend in calls whose shares are joined,
and the kernel for many rows beside a decode call."""
import math

import numpy as np
import pytest
import torch

import fp8_ref as R
import sp_hip as S
from gpu_util import d2h
from test_gpu_fp8_cache import CODE, TORCH, Pair, cur, queries, tables

pytestmark = pytest.mark.gpu


def for_many_rows(hd, dtype, columns, heads):
    """The launch's choice for one sequence: the kernel for many rows (columns: rows * n_q / heads)."""
    two = hd != 256 and dtype != "f32"
    return columns * heads >= 256 * 16 * (2 if two else 1) + (hd != 256)


def attend64(q, K, V, scale, seen):
    """q [n, hd], K and V [length, hd], seen [n, length]: out, lse and the sums of fp8_ref.bounds, in
    torch's 64 bits on the GPU, some rows at a time."""
    q, K, V = (torch.as_tensor(x, dtype=torch.float64, device="cuda") for x in (q, K, V))
    parts = []
    for i in range(0, q.shape[0], 1024):
        x, hide = q[i:i + 1024], ~seen(i, min(i + 1024, q.shape[0]))
        s = (x @ K.T).mul_(scale).masked_fill_(hide, -math.inf)
        lse = torch.logsumexp(s, -1)
        w = s.sub_(lse[:, None]).exp_()
        steep = (x.abs() @ K.abs().T).masked_fill_(hide, 0.0).amax(-1) * abs(scale)
        parts.append((w @ V, lse, w @ V.abs(), (~hide).double() @ V.abs(), steep))
    out, lse, reach, plain, steep = (torch.cat(x).cpu().numpy() for x in zip(*parts))
    return out, lse, np.stack([reach, plain]), steep


def close(dtype, hd, seen, got, want):
    out, lse = got
    wout, wlse, reach, steep = want
    tol, ltol = R.bounds(dtype, hd, seen, wout, reach, steep)
    d, dl = np.abs(out - wout), np.abs(lse - wlse)
    assert (d <= tol).all(), (float((d - tol).max()), float(d.max()))
    assert (dl <= ltol + 2.0 ** -23 * np.abs(wlse)).all(), float(dl.max())


def all_values(P, holes=()):
    """K and V of a one-head cache's first sequence, and which positions there are."""
    here = np.repeat([j not in holes for j in range(len(P.table[0]))], 64)
    kv = [np.concatenate([P.ref.values(side, 0, b)[0] if b >= 0 else np.zeros((64, P.hd)) for b in P.table[0]])
          for side in range(2)]
    return kv[0], kv[1], torch.from_numpy(here).cuda()


# 256 sequences of one head are a share each. A wave of eight looks 64 of its blocks up at once: 512 a
# share; one of four (head_dim 256) 256.
@pytest.mark.parametrize("hd,dtype,n_q,length", [(64, "bf16", 3, 33000), (64, "f16", 20, 33000), (96, "f32", 2, 33000),
                                                 (256, "bf16", 2, 16500)])
def test_more_blocks_a_wave_than_it_looks_up_at_once(hd, dtype, n_q, length):
    rng = np.random.default_rng(hd)
    n, longest = 256, length + 999
    P = Pair(hd, 1, (longest + 63) // 64)
    P.fill(rng, tables(rng, [longest], P.n_blocks), [longest], "f32", 0.5)
    row, last = list(P.table[0]), len(P.table[0]) - 1
    holes = (5, last - 10)  # the second is past the first 512 (256)
    for j in holes:
        row[j] = -1 if j == 5 else P.n_blocks
    lens = [length + (i * 37) % 1000 for i in range(n)]
    P.batch([row] * n, lens)
    q = queries(rng, P, n_q, dtype)
    got = P.attend(dtype, q, 0.7 / math.sqrt(hd))
    P.table = [[b if 0 <= b < P.n_blocks else -1 for b in row]]
    K, V, here = all_values(P, holes)
    at, end = torch.arange(K.shape[0], device="cuda"), torch.tensor(lens, device="cuda").repeat_interleave(n_q)
    want = attend64(q.double().numpy().reshape(-1, hd), K, V, 0.7 / math.sqrt(hd),
                    lambda a, b: (at[None] < end[a:b, None]) & here[None])
    close(dtype, hd, longest, (got[0].reshape(-1, hd), got[1].reshape(-1)), want)


# 33 column groups (of 256 columns, or 128 in waves of 16) over 516 blocks: 7 shares each of 74, and
# a block of threads looks 64 of them up at once.
@pytest.mark.parametrize("hd,dtype,new,n_q", [(64, "bf16", 128, 66), (128, "f16", 128, 66), (128, "f32", 65, 64),
                                              (256, "bf16", 65, 64)])
def test_more_blocks_a_share_than_are_looked_up_at_once(hd, dtype, new, n_q):
    assert for_many_rows(hd, dtype, new * n_q, 1)
    rng = np.random.default_rng(hd)
    length = 33000
    P = Pair(hd, 1, (length + 63) // 64)
    P.fill(rng, tables(rng, [length], P.n_blocks), [length], "f32", 0.5)
    row = list(P.table[0])
    holes = (70, 400)  # the first behind a share's first 64
    for j in holes:
        row[j] = -1
    P.batch([row], [length], [0, new])
    q = queries(rng, P, n_q, dtype)
    got = P.attend(dtype, q, 0.7 / math.sqrt(hd))
    K, V, here = all_values(P, holes)
    at = torch.arange(K.shape[0], device="cuda")
    pos = torch.arange(length - new, length, device="cuda").repeat_interleave(n_q)
    want = attend64(q.double().numpy().reshape(-1, hd), K, V, 0.7 / math.sqrt(hd),
                    lambda a, b: (at[None] <= pos[a:b, None]) & here[None])
    close(dtype, hd, length, (got[0].reshape(-1, hd), got[1].reshape(-1)), want)


class Rows:
    """A prefill call over P's batch with a row array of its own, its outputs marked before."""

    def __init__(self, P, rng, lens, row, n_rows, n_q, dtype):
        self.P, self.n_q, self.dtype = P, n_q, dtype
        P.batch(P.table, lens, row, n_rows)
        self.keep = list(P.keep)
        self.b, self.n_rows = P.b, n_rows
        self.q = queries(rng, P, n_q, dtype).cuda()

    def run(self, row=None):
        P, width = self.P, self.n_q * self.P.hd
        out = torch.full((self.n_rows + 1, self.n_q, P.hd), 77.0, dtype=TORCH[self.dtype], device="cuda")
        lse = torch.full((self.n_rows + 1, self.n_q), 77.0, device="cuda")
        b = self.b
        if row is not None:
            t = torch.tensor(row, dtype=torch.int32, device="cuda")
            self.keep.append(t)
            b = S.Fp8Batch(self.b.c.n_seq, self.b.c.table_stride, self.keep[0].data_ptr(), self.keep[1].data_ptr(),
                           t.data_ptr(), self.n_rows)
        S.check(S.lib().sp_hip_fp8_attn_prefill(P.dev.ref, 0, b.ref, self.q.data_ptr(), width, self.n_q, CODE[self.dtype],
                                                0.125, 0, out.data_ptr(), width, lse.data_ptr(), cur()), "attend")
        torch.cuda.synchronize()
        return out.cpu(), lse.cpu()


# sequences' lengths, new rows of each, n_q: shares joined by the last to arrive (few columns) or by a
# second launch; the last set has more sequences than a wave has lanes
BAD_ROWS = {
    "few": ([4000, 2600], [5, 4], 4, [[0, 9, 4], [-5, 4, 9], [0, 5, 10], [1 << 30, 5, 9], [0, -(1 << 31), 9]]),
    "few, one sequence": ([4000], [9], 4, [[-1, 9], [9, 3], [0, 10], [-9, -1]]),
    "few, many sequences": ([3000] + [70] * 79, [2] * 80, 4, [[2 * i for i in range(75)] + [100] + [2 * i for i in range(76, 81)]]),
    "many": ([2600, 1900], [80, 60], 64, [[0, 140, 80], [-5, 80, 140], [0, 80, 141]]),
    "many, one sequence": ([2600], [140], 64, [[-1, 140], [140, 3], [0, 141]]),
}


@pytest.mark.parametrize("kind", list(BAD_ROWS))
def test_attention_over_rows_out_of_order_does_nothing(kind):
    lens, news, n_q, bad = BAD_ROWS[kind]
    rng = np.random.default_rng(4)
    P = Pair(64, 1, sum((n + 63) // 64 for n in lens))
    table = tables(rng, lens, P.n_blocks)
    P.fill(rng, table, lens, "f32", 0.5)
    row = [sum(news[:i]) for i in range(len(news) + 1)]
    assert for_many_rows(64, "bf16", row[-1] * n_q, 1) == kind.startswith("many")
    call = Rows(P, rng, lens, row, row[-1], n_q, "bf16")
    good = call.run()
    assert (good[0][-1] == 77).all() and (good[1][-1] == 77).all() and not (good[1][:-1] == 77).any()
    for r in bad:
        out, lse = call.run(r)
        assert (out == 77).all() and (lse == 77).all(), r
        again = call.run()  # the workspace and its counters are as they were
        assert torch.equal(again[0], good[0]) and torch.equal(again[1], good[1]), r
    P.batch(table, lens, row)
    P.check_attend("bf16", call.q.cpu(), 0.125)


def test_copies_with_rows_out_of_order_keep_to_their_rows_and_blocks():
    rng = np.random.default_rng(6)
    P = Pair(64, 2, 12)
    P.fill(rng, [[0, 1], [2, 3], [8, 9, 10]], [100, 90, 192])
    table, lens, n = [[0, 1], [2, 3]], [100, 90], 20
    others = [b for b in range(12) if b > 3]
    before = [d2h(p, 12 * 2 * 64 * 64).reshape(12, -1).copy() for p in (P.dev.c.d_k_codes, P.dev.c.d_v_codes)]
    scales = [d2h(p, 12 * 2).reshape(12, -1).copy() for p in (P.dev.c.d_k_exp, P.dev.c.d_v_exp)]
    for row in ([0, 50, 20], [-5, 60, -3], [15, 3, 20], [1 << 30, -(1 << 31), 20]):
        P.batch(table, lens, row, n)
        src = torch.full((n + 1, 2, 64), 3.0, device="cuda")
        src[n] = float("nan")
        back = torch.full((n + 1, 2, 64), 7.0, device="cuda")
        for v in (None, src.data_ptr()):
            S.check(S.lib().sp_hip_fp8_write(P.dev.ref, 0, P.b.ref, src.data_ptr(), v, 128, S.DTYPE_F32, cur()), "write")
        S.check(S.lib().sp_hip_fp8_read(P.dev.ref, 0, P.b.ref, back.data_ptr(), None, 128, S.DTYPE_F32, cur()), "read")
        torch.cuda.synchronize()
        assert (back[n] == 7.0).all()
        for side, (codes, exps) in enumerate(((P.dev.c.d_k_codes, P.dev.c.d_k_exp), (P.dev.c.d_v_codes, P.dev.c.d_v_exp))):
            assert np.array_equal(d2h(codes, 12 * 2 * 64 * 64).reshape(12, -1)[others], before[side][others])
            assert np.array_equal(d2h(exps, 12 * 2).reshape(12, -1)[others], scales[side][others])


def test_many_rows_beside_a_decode_step():
    """A prefill call whose shares a second launch joins and a decode call whose last share joins
    them, on one cache at once."""
    rng = np.random.default_rng(48)
    P = Pair(128, 2, 300)
    lens, new, n_q = [9000, 8000], 300, 32
    assert for_many_rows(128, "f16", new * n_q // 2, 2)
    P.fill(rng, tables(rng, lens, 300), lens)
    q, batches = [], []
    for row in ([0, new, new], None):
        q.append(queries(rng, P.batch_of(lens, row), n_q, "f16").cuda())
        batches.append(P.b)
    outs = [torch.zeros_like(t) for t in q]
    lses = [torch.zeros(t.shape[:2], device="cuda") for t in q]
    L, streams = S.lib(), [torch.cuda.Stream() for _ in range(2)]

    def call(i, stream):
        f = (L.sp_hip_fp8_attn_prefill, L.sp_hip_fp8_attn_decode)[i]
        S.check(f(P.dev.ref, 0, batches[i].ref, q[i].data_ptr(), n_q * 128, n_q, S.DTYPE_F16, 0.05, 0,
                  outs[i].data_ptr(), n_q * 128, lses[i].data_ptr(), stream), "attend")
    torch.cuda.synchronize()
    want = []
    for i in range(2):
        call(i, cur())
        torch.cuda.synchronize()
        want.append((outs[i].clone(), lses[i].clone()))
    assert not any((o == 0).all() for o, _ in want)
    for turn in range(6):
        for t in outs + lses:
            t.zero_()
        torch.cuda.synchronize()
        for i in ((0, 1), (1, 0))[turn % 2]:
            call(i, streams[i].cuda_stream)
        torch.cuda.synchronize()
        for i, (o, l) in enumerate(want):
            assert torch.equal(outs[i], o) and torch.equal(lses[i], l)
