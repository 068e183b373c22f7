"""A 4-bit block cache on the device beside its numpy form."""
import numpy as np
import torch

import fp4_ref as R
import sp_hip as S
from gpu_util import d2h
from test_gpu_fp8_cache import CODE, ESIZE, TORCH, Pair as Fp8Pair, cur


class Pair(Fp8Pair):
    """The 8-bit cache's pair (batches, rows, attention's check) over the 4-bit cache's calls."""

    def __init__(self, hd, heads, n_blocks, layers=1):
        self.hd, self.heads, self.n_blocks, self.layers = hd, heads, n_blocks, layers
        self.dev = S.Fp4Cache(S.config(hd, layers, heads), n_blocks, cur())
        self.ref = R.RefCache(hd, layers, heads, n_blocks)

    def on_device(self, x, width, dtype, pad, shift):
        t = torch.full((shift + self.n_rows * (width + pad),), float("nan"), dtype=TORCH[dtype])
        t[shift:].view(self.n_rows, width + pad)[:, :width] = x.reshape(self.n_rows, width)
        return t.cuda()

    def write(self, dtype, k, v, layer=0, pad=0, shift=0):
        width = self.heads * self.hd
        dev = [self.on_device(x, width, dtype, pad, shift) if x is not None else None for x in (k, v)]
        ptr = [t.data_ptr() + shift * ESIZE[dtype] if t is not None else None for t in dev]
        S.check(S.lib().sp_hip_fp4_write(self.dev.ref, layer, self.b.ref, ptr[0], ptr[1], width + pad, CODE[dtype],
                                         cur()), "write")
        self.ref.write(layer, self.table, self.lens, self.row, self.n_rows,
                       *[x.double().numpy() if x is not None else None for x in (k, v)])
        torch.cuda.synchronize()

    def weights(self):
        n = self.layers * self.n_blocks * self.heads * 64 * 4
        return d2h(self.dev.c.d_weight, n).view(np.float32).reshape(self.ref.weight.shape).astype(np.float64)

    def set_weights(self, w):
        """w: as the reference's, rounded to fp32 for both."""
        w = w.astype(np.float32)
        self.ref.weight = w.astype(np.float64)
        t = torch.from_numpy(np.ascontiguousarray(w)).cuda()
        torch.cuda.synchronize()
        copy(self.dev.c.d_weight, t)

    def check_memory(self, weights=True):
        c = self.dev.c
        n = self.layers * self.n_blocks * self.heads
        for side, (codes, exps) in enumerate(((c.d_k_codes, c.d_k_exp), (c.d_v_codes, c.d_v_exp))):
            want = self.ref.code_bytes(side)
            np.testing.assert_array_equal(d2h(codes, n * 32 * self.hd).reshape(want.shape), want)
            want = self.ref.exp_bytes(side)
            np.testing.assert_array_equal(d2h(exps, n * 2 * self.hd).reshape(want.shape), want)
        if weights:
            np.testing.assert_array_equal(self.weights(), self.ref.weight)

    def attend(self, dtype, q, scale, window=0, layer=0, pad=0, shift=0, stream=None, want_lse=True):
        n_q = q.shape[1]
        width = n_q * self.hd
        qt = self.on_device(q, width, dtype, pad, shift)
        out = torch.full((shift + self.n_rows * (width + pad),), 77.0, dtype=TORCH[dtype], device="cuda")
        lse = torch.full((self.n_rows, n_q), 77.0, dtype=torch.float32, device="cuda")
        L = S.lib()
        call = L.sp_hip_fp4_attn_prefill if self.row is not None else L.sp_hip_fp4_attn_decode
        torch.cuda.synchronize()
        S.check(call(self.dev.ref, layer, self.b.ref, qt.data_ptr() + shift * ESIZE[dtype], width + pad, n_q,
                     CODE[dtype], scale, window, out.data_ptr() + shift * ESIZE[dtype], width + pad,
                     lse.data_ptr() if want_lse else None, stream if stream is not None else cur()), "attend")
        torch.cuda.synchronize()
        o = out.cpu()
        rows = o[shift:].view(self.n_rows, width + pad)
        assert (o[:shift] == 77.0).all() and (rows[:, width:] == 77.0).all(), "written between the rows"
        return rows[:, :width].reshape(self.n_rows, n_q, self.hd).double().numpy(), lse.double().cpu().numpy()

    def weigh(self, dtype, q, scale, lse, window=0, layer=0, pad=0, shift=0):
        n_q = q.shape[1]
        qt = self.on_device(q, n_q * self.hd, dtype, pad, shift)
        lt = torch.from_numpy(np.ascontiguousarray(lse, np.float32)).cuda()
        S.check(S.lib().sp_hip_fp4_weigh(self.dev.ref, layer, self.b.ref, qt.data_ptr() + shift * ESIZE[dtype],
                                         n_q * self.hd + pad, n_q, CODE[dtype], scale, window, lt.data_ptr(), cur()),
                "weigh")
        torch.cuda.synchronize()

    def check_weigh(self, dtype, q, scale, window=0, layer=0, pad=0, shift=0, lse=None):
        """The call's own lse if there is none."""
        if lse is None:
            _, lse = self.attend(dtype, q, scale, window, layer)
        before = self.weights()
        self.weigh(dtype, q, scale, lse, window, layer, pad, shift)
        self.ref.weight = before.copy()
        x = q.numpy() if dtype == "f32" else q.double().numpy()
        tol = self.ref.weigh(layer, self.table, self.lens, self.row, self.n_rows, x, float(np.float32(scale)), window,
                             np.asarray(lse, np.float64))
        got = self.weights()
        d = np.abs(got - self.ref.weight)
        assert (d <= tol).all(), (float((d - tol).max()), float(d.max()))
        return got - before

    def check_evict(self, keep, first, recent, layer=0, guard=5):
        kept = torch.full((len(self.lens) * self.heads * keep + guard,), -77, dtype=torch.int32, device="cuda")
        S.check(S.lib().sp_hip_fp4_evict(self.dev.ref, layer, self.b.ref, keep, first, recent, kept.data_ptr(), cur()),
                "evict")
        torch.cuda.synchronize()
        kept = kept.cpu().numpy()
        assert (kept[len(kept) - guard:] == -77).all()
        want = self.ref.evict(layer, self.table, self.lens, keep, first, recent)
        np.testing.assert_array_equal(kept[:len(kept) - guard].reshape(want.shape), want)
        self.check_memory(weights=False)
        np.testing.assert_array_equal(np.nan_to_num(self.weights(), nan=-5.0), np.nan_to_num(self.ref.weight, nan=-5.0))
        return want


def copy(to, tensor):
    """A contiguous device tensor's bytes to a device address."""
    import ctypes as C
    hip = C.CDLL("libamdhip64.so")
    hip.hipMemcpy.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int]
    assert hip.hipMemcpy(to, tensor.data_ptr(), tensor.numel() * tensor.element_size(), 3) == 0
    torch.cuda.synchronize()
