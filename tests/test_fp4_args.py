"""The 4-bit block cache's refusals: what the host can see is refused before anything is
launched, with a reason (no GPU: a cache whose memory is never touched)."""
import ctypes as C
import subprocess

import numpy as np
import pytest

import fp4_ref as R
import sp_hip as S
from test_fp8_args import BAD_BATCHES, attend as attend8, batch, write as write8


@pytest.fixture
def cache():
    c = S.SpHipFp4Cache()
    S.lib().sp_config_init(C.byref(c.config), 128, 2, 4)
    c.n_blocks = 16
    c.d_k_codes = c.d_v_codes = c.d_k_exp = c.d_v_exp = c.d_weight = 1 << 20
    priv = C.create_string_buffer(256)  # device 0
    c.priv = C.addressof(priv)
    yield c
    c.priv = None


def write(c, name="sp_hip_fp4_write", **kw):
    return write8(c, name=name, **kw)


def attend(c, name="sp_hip_fp4_attn_prefill", **kw):
    return attend8(c, name=name, **kw)


def weigh(c, layer=0, b=None, q=4096, q_stride=1024, n_q=8, dtype=S.DTYPE_F16, scale=0.1, window=0, lse=4096):
    return S.lib().sp_hip_fp4_weigh(C.byref(c) if c is not None else None, layer, (b or batch()).ref, q, q_stride, n_q,
                                    dtype, scale, window, lse, None)


def evict(c, layer=0, b=None, keep=100, first=4, recent=20, kept=4096):
    return S.lib().sp_hip_fp4_evict(C.byref(c) if c is not None else None, layer, (b or batch()).ref, keep, first,
                                    recent, kept, None)


@pytest.mark.parametrize("name", ["sp_hip_fp4_write", "sp_hip_fp4_read"])
@pytest.mark.parametrize("bad", [dict(layer=-1), dict(layer=2), dict(stride=511), dict(stride=1 << 40), dict(dtype=3),
                                 dict(dtype=-1), dict(k=4097), dict(v=4095), dict(b=batch(n_seq=1 << 23))])
def test_copies_refuse(cache, name, bad):
    assert write(cache, name=name, **bad) == -1
    assert S.last_error().startswith(name[7:])


@pytest.mark.parametrize("bad", BAD_BATCHES)
def test_batches_refused(cache, bad):
    assert write(cache, b=batch(**bad)) == -1
    assert write(cache, b=batch(**bad), name="sp_hip_fp4_read") == -1
    assert attend(cache, b=batch(**bad)) == -1
    assert attend(cache, b=batch(**bad), name="sp_hip_fp4_attn_decode") == -1
    assert weigh(cache, b=batch(**bad)) == -1
    assert evict(cache, b=batch(**bad)) == -1


QUERIES = [dict(layer=2), dict(n_q=0), dict(n_q=-4), dict(n_q=6), dict(dtype=7), dict(q_stride=1023),
           dict(scale=float("inf")), dict(scale=float("nan")), dict(window=-1), dict(q=4097), dict(lse=4098), dict(q=0)]


@pytest.mark.parametrize("name", ["sp_hip_fp4_attn_prefill", "sp_hip_fp4_attn_decode"])
@pytest.mark.parametrize("bad", QUERIES + [dict(out_stride=1023), dict(out=4097), dict(out=0),
                                           dict(n_q=1 << 24, q_stride=1 << 32, out_stride=1 << 32)])
def test_attention_refuses(cache, name, bad):
    assert attend(cache, name=name, **bad) == -1
    assert S.last_error().startswith(name[7:])


@pytest.mark.parametrize("bad", QUERIES + [dict(lse=0), dict(n_q=1 << 24, q_stride=1 << 32)])
def test_weigh_refuses(cache, bad):
    assert weigh(cache, **bad) == -1
    assert S.last_error().startswith("fp4_weigh")


@pytest.mark.parametrize("bad", [dict(layer=-1), dict(layer=2), dict(keep=0), dict(keep=-5), dict(first=-1),
                                 dict(recent=-1), dict(first=90), dict(recent=97), dict(first=101, recent=0),
                                 dict(first=(1 << 31) - 1, recent=1), dict(keep=(1 << 30) + 1), dict(kept=0),
                                 dict(kept=4098), dict(b=batch(n_seq=1 << 20))])
def test_evict_refuses(cache, bad):
    assert evict(cache, **bad) == -1
    assert S.last_error().startswith("fp4_evict")


def test_no_cache_and_no_batch(cache):
    L = S.lib()
    empty = S.SpHipFp4Cache()
    for c in (None, empty):
        assert write(c) == -1 and attend(c) == -1 and weigh(c) == -1 and evict(c) == -1
    assert L.sp_hip_fp4_write(C.byref(cache), 0, None, 4096, 4096, 512, S.DTYPE_F16, None) == -1
    assert L.sp_hip_fp4_attn_decode(C.byref(cache), 0, None, 4096, 1024, 8, 1, 0.1, 0, 4096, 1024, None, None) == -1
    assert L.sp_hip_fp4_weigh(C.byref(cache), 0, None, 4096, 1024, 8, 1, 0.1, 0, 4096, None) == -1
    assert L.sp_hip_fp4_evict(C.byref(cache), 0, None, 8, 0, 0, 4096, None) == -1
    L.sp_hip_fp4_cache_free(None)
    L.sp_hip_fp4_cache_free(C.byref(empty))


def test_decode_takes_one_row_per_sequence(cache):
    assert attend(cache, b=batch(row=1 << 20, n_rows=3), name="sp_hip_fp4_attn_decode") == -1
    assert "d_row" in S.last_error()


def test_nothing_to_do_is_done(cache):
    none = batch(n_seq=0, n_rows=0, table=0, lens=0, stride=0)
    assert write(cache, b=none) == 0 and attend(cache, b=none, q=0, out=0) == 0
    assert weigh(cache, b=none, q=0, lse=0) == 0 and evict(cache, b=none, kept=0) == 0
    assert write(cache, k=0, v=0) == 0
    assert attend(cache, b=batch(row=1 << 20, n_rows=0), q=0, out=0) == 0
    assert weigh(cache, b=batch(row=1 << 20, n_rows=0), q=0, lse=0) == 0


@pytest.mark.parametrize("hd,layers,heads,blocks", [(100, 1, 1, 4), (0, 1, 1, 4), (512, 1, 1, 4), (128, 0, 1, 4),
                                                    (128, 1, 0, 4), (128, 1, 65536, 4), (128, 1, 1, 0),
                                                    (128, 1, 1, -3), (256, 1 << 20, 1 << 15, 1 << 30)])
def test_init_refuses(hd, layers, heads, blocks):
    cfg = S.SpConfig()
    S.lib().sp_config_init(C.byref(cfg), hd, layers, heads)
    cfg.head_dim, cfg.n_layers, cfg.n_heads_kv = hd, layers, heads
    c = S.SpHipFp4Cache()
    assert S.lib().sp_hip_fp4_cache_init(C.byref(c), C.byref(cfg), blocks, None) == -1
    assert S.last_error().startswith("fp4_cache_init") and not c.priv
    assert S.lib().sp_hip_fp4_cache_init(None, C.byref(cfg), blocks, None) == -1
    assert S.lib().sp_hip_fp4_cache_init(C.byref(c), None, 4, None) == -1


# ---- the plain form itself ----

def test_reference_codes():
    assert np.array_equal(R.code_of(R.POS), np.arange(8))
    mid = (R.POS[:-1] + R.POS[1:]) / 2
    assert R.code_of(mid).tolist() == [0, 2, 2, 4, 4, 6, 6]  # ties to the even code
    assert R.code_of(np.nextafter(mid, 9)).tolist() == [1, 2, 3, 4, 5, 6, 7]
    assert R.code_of(np.nextafter(mid, 0)).tolist() == [0, 1, 2, 3, 4, 5, 6]
    assert R.code_of(np.array([1e9, -1e9, -0.0, -0.3])).tolist() == [7, 15, 8, 9]


@pytest.mark.parametrize("amax,e", [(0.0, -40), (6.0, 0), (6.0000001, 1), (1.5, -2), (1.5000002, -1), (1.0, -2),
                                    (65504.0, 14), (2.0 ** -80, -40), (6.0 * 2.0 ** 40, 40)])
def test_reference_exponent(amax, e):
    assert R.exponents(np.array([amax]))[0] == e


def test_exponents_places_are_a_permutation():
    assert sorted(R.place(np.arange(64)).tolist()) == list(range(64))


def test_reference_eviction():
    c = R.RefCache(64, 1, 1, 2)
    c.weight[0, :, 0] = np.arange(128).reshape(2, 64)[::-1] % 7  # ties
    c.codes[0, 0, :, 0] = (np.arange(128) % 16).reshape(2, 64, 1)
    kept = c.evict(0, [[1, 0]], [100], 40, 3, 5)[0, 0]
    w = np.concatenate([np.arange(64) % 7, (64 + np.arange(36)) % 7])
    inner = [p for p in kept if 3 <= p < 95]
    assert kept[:3].tolist() == [0, 1, 2] and kept[-5:].tolist() == list(range(95, 100)) and len(inner) == 32
    low = min(w[p] for p in inner)
    gone = [p for p in range(3, 95) if p not in inner]
    assert max(w[p] for p in gone) <= low
    assert max(p for p in inner if w[p] == low) < min([p for p in gone if w[p] == low], default=999)
    assert c.codes[0, 0, 1, 0, 4, 0] == kept[4] % 16


@pytest.mark.parametrize("compiler,ext", [("gcc", "c"), ("g++", "cpp")])
def test_the_header_stands_alone(tmp_path, compiler, ext):
    f = tmp_path / f"t.{ext}"
    f.write_text('#include "sp_hip_fp4.h"\nint main(void){sp_hip_fp4_cache_t c; sp_hip_fp4_cache_free(&c); return SP_FP4_BLOCK;}\n')
    r = subprocess.run([compiler, "-fsyntax-only", "-Wall", "-Werror", "-I", S.INCLUDE_DIR, str(f)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
