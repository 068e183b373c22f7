"""Batches of the 8-bit block cache that would take more threads than a launch counts are refused."""
import ctypes as C

import pytest

import sp_hip as S
from test_fp8_args import attend, batch, cache, write  # noqa: F401  (cache: the fixture)


@pytest.mark.parametrize("name", ["sp_hip_fp8_write", "sp_hip_fp8_read"])
@pytest.mark.parametrize("kw", [dict(n_seq=1 << 23), dict(n_seq=(1 << 23) - 1, row=1 << 20, n_rows=1 << 23),
                                dict(n_seq=1, row=1 << 20, n_rows=1 << 30)])
def test_copies_of_too_many_sequences_or_rows(cache, name, kw):  # noqa: F811
    assert write(cache, b=batch(**kw), name=name) == -1
    assert "too many" in S.last_error()


@pytest.mark.gpu
def test_attention_of_too_many_sequences():
    """Refused by the launch's host code: nothing runs, the arrays are not read."""
    c = S.Fp8Cache(S.config(64, 1, 1), 4)
    n = 1 << 24
    for name, b in (("sp_hip_fp8_attn_decode", batch(n)), ("sp_hip_fp8_attn_prefill", batch(n, row=1 << 20, n_rows=n))):
        assert attend(c.c, b=b, n_q=1, q_stride=64, out_stride=64, name=name) == -1
        assert "invalid" in S.last_error()
