"""Sequences of the 4-bit block cache whose tables have holes, beside another stream that writes blocks which are
not theirs."""
import numpy as np
import pytest
import torch

import sp_hip as S
from fp4_pair import Pair
from test_gpu_fp4_cache import fill_device
from test_gpu_fp8_cache import CODE, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 6, 300])  # the kernel for few rows, one and several, and the one for many
def test_a_hole_shows_nothing_of_the_first_block(rows, hd, dtype):
    """Block 0 is written anew all the time, with scales of 2^-40 and of 2^40 in turn: what is read of it in a hole's
    place, codes and scales at different times, adds nothing, and not NaN either."""
    rng = np.random.default_rng(hd + rows)
    P = Pair(hd, 2, 30)
    hole = [3, -1, 5, 6, 30, 7, 8, -1]
    P.batch([hole, [9, 10, -5, 11, 12]], [512, 300], None if rows == 1 else [0, rows, 2 * rows])
    fill_device(rng, P)
    q = queries(rng, P, 32, dtype)
    want, wlse = P.check_attend(dtype, q, 0.1)
    qt = q.cuda()
    out = [torch.empty_like(qt) for _ in range(40)]
    lse = torch.empty((P.n_rows, 32), device="cuda")
    first = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    full, row = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([64], [0, 64]))
    b = S.Fp4Batch(1, 1, first.data_ptr(), full.data_ptr(), row.data_ptr(), 64)
    kv = [torch.full((64, 2, hd), x, device="cuda") for x in (2.0 ** -50, 6.0 * 2.0 ** 40)]
    A, B = torch.cuda.Stream(), torch.cuda.Stream()
    L = S.lib()
    call = L.sp_hip_fp4_attn_prefill if rows > 1 else L.sp_hip_fp4_attn_decode
    torch.cuda.synchronize()
    for o in out:
        for k in range(6):
            x = kv[k % 2].data_ptr()
            S.check(L.sp_hip_fp4_write(P.dev.ref, 0, b.ref, x, x, 2 * hd, S.DTYPE_F32, B.cuda_stream), "write")
        S.check(call(P.dev.ref, 0, P.b.ref, qt.data_ptr(), 32 * hd, 32, CODE[dtype], 0.1, 0, o.data_ptr(), 32 * hd,
                     lse.data_ptr(), A.cuda_stream), "attend")
    torch.cuda.synchronize()
    for o in out:
        assert np.array_equal(o.double().cpu().numpy(), want)
    assert np.array_equal(lse.double().cpu().numpy(), wlse)
