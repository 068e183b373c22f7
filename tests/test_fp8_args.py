"""The 8-bit block cache's refusals: what the host can see is refused before anything is
launched, with a reason (no GPU: a cache whose memory is never touched)."""
import ctypes as C

import numpy as np
import pytest

import fp8_ref as R
import sp_hip as S


@pytest.fixture
def cache():
    c = S.SpHipFp8Cache()
    S.lib().sp_config_init(C.byref(c.config), 128, 2, 4)
    c.n_blocks = 16
    c.d_k_codes = c.d_v_codes = c.d_k_exp = c.d_v_exp = 1 << 20
    priv = C.create_string_buffer(256)  # device 0
    c.priv = C.addressof(priv)
    yield c
    c.priv = None


def batch(n_seq=3, stride=4, table=1 << 20, lens=1 << 20, row=0, n_rows=None):
    return S.Fp8Batch(n_seq, stride, table, lens, row, n_rows)


def write(c, layer=0, b=None, k=4096, v=4096, stride=512, dtype=S.DTYPE_F16, name="sp_hip_fp8_write"):
    return getattr(S.lib(), name)(C.byref(c) if c is not None else None, layer, (b or batch()).ref, k, v, stride,
                                  dtype, None)


def attend(c, layer=0, b=None, q=4096, q_stride=1024, n_q=8, dtype=S.DTYPE_F16, scale=0.1, window=0, out=4096,
           out_stride=1024, lse=None, name="sp_hip_fp8_attn_prefill"):
    return getattr(S.lib(), name)(C.byref(c) if c is not None else None, layer, (b or batch()).ref, q, q_stride, n_q,
                                  dtype, scale, window, out, out_stride, lse, None)


BAD_BATCHES = [dict(n_seq=-1, n_rows=-1), dict(n_rows=4), dict(table=0), dict(lens=0), dict(stride=0),
               dict(stride=(1 << 24) + 1), dict(row=1 << 20, n_rows=-2), dict(row=(1 << 20) + 2, n_rows=3),
               dict(table=(1 << 20) + 1), dict(row=1 << 20, n_rows=(1 << 30) + 1)]


@pytest.mark.parametrize("name", ["sp_hip_fp8_write", "sp_hip_fp8_read"])
@pytest.mark.parametrize("bad", [dict(layer=-1), dict(layer=2), dict(stride=511), dict(stride=1 << 40), dict(dtype=3),
                                 dict(dtype=-1), dict(k=4097), dict(v=4095)])
def test_copies_refuse(cache, name, bad):
    assert write(cache, name=name, **bad) == -1
    assert S.last_error().startswith(name[7:])


@pytest.mark.parametrize("bad", BAD_BATCHES)
def test_batches_refused(cache, bad):
    assert write(cache, b=batch(**bad)) == -1
    assert write(cache, b=batch(**bad), name="sp_hip_fp8_read") == -1
    assert attend(cache, b=batch(**bad)) == -1
    assert attend(cache, b=batch(**bad), name="sp_hip_fp8_attn_decode") == -1


@pytest.mark.parametrize("name", ["sp_hip_fp8_attn_prefill", "sp_hip_fp8_attn_decode"])
@pytest.mark.parametrize("bad", [dict(layer=2), dict(n_q=0), dict(n_q=-4), dict(n_q=6), dict(dtype=7),
                                 dict(q_stride=1023), dict(out_stride=1023), dict(scale=float("inf")),
                                 dict(scale=float("nan")), dict(window=-1), dict(q=4097), dict(out=4097),
                                 dict(lse=4098), dict(q=0), dict(out=0), dict(n_q=1 << 24, q_stride=1 << 32,
                                                                              out_stride=1 << 32)])
def test_attention_refuses(cache, name, bad):
    assert attend(cache, name=name, **bad) == -1
    assert S.last_error().startswith(name[7:])


def test_no_cache_and_no_batch(cache):
    L = S.lib()
    assert write(None) == -1 and attend(None) == -1
    empty = S.SpHipFp8Cache()
    assert write(empty) == -1 and attend(empty) == -1
    assert L.sp_hip_fp8_write(C.byref(cache), 0, None, 4096, 4096, 512, S.DTYPE_F16, None) == -1
    assert L.sp_hip_fp8_attn_decode(C.byref(cache), 0, None, 4096, 1024, 8, 1, 0.1, 0, 4096, 1024, None, None) == -1
    L.sp_hip_fp8_cache_free(None)
    L.sp_hip_fp8_cache_free(C.byref(empty))


def test_decode_takes_one_row_per_sequence(cache):
    assert attend(cache, b=batch(row=1 << 20, n_rows=3), name="sp_hip_fp8_attn_decode") == -1
    assert "d_row" in S.last_error()


def test_nothing_to_do_is_done(cache):
    none = batch(n_seq=0, n_rows=0, table=0, lens=0, stride=0)
    assert write(cache, b=none) == 0 and attend(cache, b=none, q=0, out=0) == 0
    assert write(cache, k=0, v=0) == 0
    assert attend(cache, b=batch(row=1 << 20, n_rows=0), q=0, out=0) == 0


@pytest.mark.parametrize("hd,layers,heads,blocks", [(100, 1, 1, 4), (0, 1, 1, 4), (512, 1, 1, 4), (128, 0, 1, 4),
                                                    (128, 1, 0, 4), (128, 1, 65536, 4), (128, 1, 1, 0),
                                                    (128, 1, 1, -3), (256, 1 << 20, 1 << 15, 1 << 30)])
def test_init_refuses(hd, layers, heads, blocks):
    cfg = S.SpConfig()
    S.lib().sp_config_init(C.byref(cfg), hd, layers, heads)
    cfg.head_dim, cfg.n_layers, cfg.n_heads_kv = hd, layers, heads
    c = S.SpHipFp8Cache()
    assert S.lib().sp_hip_fp8_cache_init(C.byref(c), C.byref(cfg), blocks, None) == -1
    assert S.last_error().startswith("fp8_cache_init") and not c.priv
    assert S.lib().sp_hip_fp8_cache_init(None, C.byref(cfg), blocks, None) == -1
    assert S.lib().sp_hip_fp8_cache_init(C.byref(c), None, 4, None) == -1


# ---- the plain form itself ----

def test_reference_numbers():
    assert R.NUMBERS[0x7E] == 448.0 and R.NUMBERS[1] == 2.0 ** -9 and R.NUMBERS[0x08] == 2.0 ** -6
    codes = np.arange(127)
    assert np.array_equal(R.code_of(R.NUMBERS[codes]), codes)
    mid = (R.NUMBERS[codes[:-1]] + R.NUMBERS[codes[1:]]) / 2
    assert np.array_equal(R.code_of(mid), codes[:-1] + codes[:-1] % 2)  # ties to even
    assert R.code_of(np.array([1e9, -1e9, -0.0])).tolist() == [0x7E, 0xFE, 0x80]


@pytest.mark.parametrize("amax,e", [(0.0, -40), (448.0, 0), (448.1, 1), (1.75, -8), (1.7500002, -7), (1.0, -8),
                                    (65504.0, 8), (2.0 ** -80, -40), (448.0 * 2.0 ** 40, 40)])
def test_reference_exponent(amax, e):
    assert R.least_exponent(amax) == e


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
def test_orders_are_permutations(hd):
    for order in (R.k_order(hd), R.v_order(hd)):
        assert np.array_equal(np.sort(order.reshape(-1)), np.arange(64 * hd))
