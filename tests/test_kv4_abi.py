"""The 4-bit cache's and the sampler's C entry points reject bad arguments before
any launch (no GPU needed)."""
import ctypes
import math

import pytest

import _dip_hip as K


@pytest.fixture(scope="module")
def p():
    buf = (ctypes.c_uint8 * 64)()
    addr = ctypes.addressof(buf)
    yield addr + (-addr % 16)
    del buf


def _write(p, k=1, v=1, strides=(256, 128, 256, 128), kc=1, start=0, tokens=4, nkv=2, hd=128,
           max_len=64, off=0):
    return K.lib.dip_kv4_write(p + off if k else None, p if v else None, *strides, p if kc else None,
                               p, p, start, tokens, nkv, hd, max_len, None)


def test_write(p):
    assert _write(p, hd=64) == -4
    assert _write(p, kc=0) == -1
    assert _write(p, k=0) == -1 and _write(p, v=0) == -1
    assert _write(p, max_len=65) == -2 and _write(p, max_len=0) == -2
    assert _write(p, max_len=1 << 31) == -2
    assert _write(p, nkv=0) == -2 and _write(p, nkv=5000) == -2
    assert _write(p, start=-1) == -2 and _write(p, start=61) == -2
    assert _write(p, start=1 << 62, tokens=1 << 62) == -2
    assert _write(p, tokens=-1) == -2
    assert _write(p, strides=(-2, 128, 256, 128)) == -2
    assert _write(p, strides=(257, 128, 256, 128)) == -3
    assert _write(p, off=2) == -3
    assert _write(p, k=0, v=0, tokens=0) == 0


def test_read(p):
    L = K.lib
    assert L.dip_kv4_read(p, p, p, p, p, 0, 4, 2, 64, 64, None) == -4
    assert L.dip_kv4_read(p, p, None, p, p, 0, 4, 2, 128, 64, None) == -1
    assert L.dip_kv4_read(p, p, p, None, p, 0, 4, 2, 128, 64, None) == -1
    assert L.dip_kv4_read(p, p, p, p, p, 61, 4, 2, 128, 64, None) == -2
    assert L.dip_kv4_read(p + 8, p, p, p, p, 0, 4, 2, 128, 64, None) == -3
    assert L.dip_kv4_read(p, p, p, p + 8, p, 0, 4, 2, 128, 64, None) == -3
    assert L.dip_kv4_read(p, p, p, None, None, 64, 0, 2, 128, 64, None) == 0


def test_launches_of_two_to_the_32_threads(p):
    """HIP takes none of these: refused as too large, not passed on."""
    L = K.lib
    big = 1 << 30
    assert _write(p, nkv=8, max_len=big, tokens=1 << 26) == -2
    assert L.dip_kv4_read(p, p, p, p, p, 0, big, 1, 128, big, None) == -2
    assert L.dip_qk_norm_rope_kv4_rows(p, p, p, p, p, 0, p, p, p, p, 1 << 23, 64, 8, 128, big, 1e-6,
                                       None) == -2
    assert L.dip_sample(p, 2, 1 << 22, 5000, 5000, p, 1.0, 0, 1.0, 0.0, p, p, p, 1 << 62,
                        None) == -2
    n = L.dip_kv4_prompt_attention_workspace_size(big, 0, 64, 8, 128)
    assert L.dip_kv4_prompt_attention(p, p, p, p, 0, p, big, 64, 8, 128, big, 0.1, p, n, None) == -2


def test_norm_rope(p):
    L = K.lib
    one = lambda pos=1, hd=128, ml=64, eps=1e-6, nh=4: L.dip_qk_norm_rope_kv4(
        p, p, p, p, p, p if pos else None, p, p, p, p, nh, 2, hd, ml, eps, None)
    assert one(pos=0) == -1 and one(hd=96) == -4 and one(ml=33) == -2 and one(nh=0) == -2
    assert one(eps=-1.0) == -6 and one(eps=math.nan) == -6
    rows = lambda start=0, tokens=4, q=1: L.dip_qk_norm_rope_kv4_rows(
        p, p, p, p, p, start, p if q else None, p, p, p, tokens, 4, 2, 128, 64, 1e-6, None)
    assert rows(start=-1) == -2 and rows(start=61) == -2 and rows(tokens=-1) == -2
    assert rows(q=0) == -1 and rows(tokens=0) == 0


def test_attention(p):
    L = K.lib
    ws = L.dip_kv4_decode_attention_workspace_size(64, 8, 128, 32768)
    assert ws > 0 and L.dip_kv4_decode_attention_workspace_size(63, 8, 128, 32768) == 0
    dec = lambda nh=64, nkv=8, hd=128, ml=32768, w=p, n=ws, pos=p, q=p: \
        L.dip_kv4_decode_attention(q, p, p, p, pos, p, nh, nkv, hd, ml, 0.1, w, n, None)
    assert dec(pos=None) == -1 and dec(q=None) == -1 and dec(hd=64) == -4
    assert dec(nh=63) == -2 and dec(nh=8192) == -2 and dec(ml=100) == -2
    assert dec(w=None) == -5 and dec(n=ws - 1) == -5 and dec(w=p + 8) == -3 and dec(q=p + 2) == -3
    ws = L.dip_kv4_prompt_attention_workspace_size(5, 20000, 32, 8, 128)
    assert ws > 0
    pro = lambda start=20000, tokens=5, w=p, n=ws, nh=32: L.dip_kv4_prompt_attention(
        p, p, p, p, start, p, tokens, nh, 8, 128, 32768, 0.1, w, n, None)
    assert pro(start=-1) == -2 and pro(start=32764) == -2 and pro(tokens=-1) == -2
    assert pro(nh=33) == -2 and pro(w=None) == -5 and pro(n=ws - 1) == -5
    assert pro(tokens=0) == 0


def test_sample(p):
    L = K.lib

    def call(dtype=0, rows=2, vocab=8, stride=8, t=1.0, k=0, tp=1.0, mp=0.0, logits=p, u=p, tok=p):
        return L.dip_sample(logits, dtype, rows, vocab, stride, u, t, k, tp, mp, tok, p, p, 1 << 30,
                            None)
    assert call(dtype=3) == -4
    assert call(rows=-1) == -2 and call(vocab=0) == -2 and call(stride=-1) == -2
    for bad in (dict(t=-1.0), dict(t=math.nan), dict(t=math.inf), dict(k=-1), dict(tp=0.0),
                dict(tp=1.5), dict(tp=math.nan), dict(mp=-0.1), dict(mp=1.1), dict(mp=math.nan)):
        assert call(**bad) == -6, bad
    assert call(logits=None) == -1 and call(u=None) == -1 and call(tok=None) == -1
    assert call(logits=p + 1) == -3
    assert call(rows=0, logits=None) == 0


@pytest.mark.parametrize("args", [dict(temperature=-1), dict(temperature=math.inf), dict(top_k=-2),
                                  dict(top_k=1.5), dict(top_p=0), dict(top_p=1.01),
                                  dict(min_p=2), dict(min_p=math.nan)])
def test_sampling_settings(args):
    ok = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    K.check_sampling(**ok)
    with pytest.raises(RuntimeError):
        K.check_sampling(**{**ok, **args})


@pytest.mark.parametrize("temperature", [math.nan, 1.1e300, -1e-300])
def test_sampling_temperature_is_the_librarys(p, temperature):
    """check_sampling refuses what the library does: generate asks it before it runs the
    prompt."""
    assert K.lib.dip_sample(p, 0, 1, 8, 8, p, temperature, 0, 1.0, 0.0, p, p, p, 1 << 30,
                            None) == -6
    with pytest.raises(RuntimeError):
        K.check_sampling(temperature, 0, 1.0, 0.0)
    K.check_sampling(1e300, 0, 1.0, 0.0)


@pytest.mark.parametrize("top_k", [math.inf, math.nan])
def test_sampling_refuses_a_top_k_without_end(top_k):
    with pytest.raises(RuntimeError):
        K.check_sampling(1.0, top_k, 1.0, 0.0)
