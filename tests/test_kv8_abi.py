"""The paged 8-bit cache's entry points reject bad arguments before any launch (no GPU
needed)."""
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


def _write(p, k=1, v=1, ks=(1024, 256, 128), vs=(1024, 256, 128), kc=1, pages=8, table=1, width=2,
           pos=1, seqs=2, tokens=4, nkv=2, hd=128, off=0, poff=0):
    return K.lib.dip_kv8_write(p + off if k else None, p if v else None, *ks, *vs,
                               p if kc else None, p, p, pages, p if table else None, width,
                               p + poff if pos else None, seqs, tokens, nkv, hd, None)


def test_write(p):
    assert _write(p, hd=64) == -4
    assert _write(p, kc=0) == -1 and _write(p, k=0) == -1 and _write(p, v=0) == -1
    assert _write(p, table=0) == -1 and _write(p, pos=0) == -1
    for bad in (dict(pages=0), dict(pages=1 << 29), dict(width=0), dict(width=1 << 25),
                dict(seqs=-1), dict(seqs=1 << 25), dict(tokens=-1), dict(tokens=1 << 31),
                dict(nkv=0), dict(nkv=5000), dict(ks=(-2, 256, 128))):
        assert _write(p, **bad) == -2, bad
    for bad in (dict(ks=(1024, 257, 128)), dict(vs=(1, 256, 128)), dict(off=2), dict(poff=4)):
        assert _write(p, **bad) == -3, bad
    assert _write(p, k=0, v=0, tokens=0) == 0 and _write(p, k=0, v=0, seqs=0, table=0) == 0


def test_read(p):
    L = K.lib
    call = lambda pages=8, table=p, width=2, pos=p, k=p, v=p, seqs=2, tokens=4, nkv=2, hd=128, \
        kc=p: L.dip_kv8_read(kc, p, p, pages, table, width, pos, k, v, seqs, tokens, nkv, hd, None)
    assert call(hd=64) == -4 and call(kc=None) == -1 and call(table=None) == -1
    assert call(k=None) == -1 and call(pos=None) == -1
    assert call(tokens=-1) == -2 and call(seqs=-1) == -2 and call(nkv=0) == -2
    assert call(k=p + 8) == -3 and call(kc=p + 8) == -3 and call(pos=p + 4) == -3
    assert call(table=p + 2) == -3
    assert call(k=None, v=None, tokens=0) == 0


def test_norm_rope(p):
    L = K.lib
    call = lambda qkv=p, rows=64, pos=p, q=p, pages=8, table=p, width=2, seqs=2, tokens=4, nh=4, \
        nkv=2, hd=128, eps=1e-6: L.dip_qk_norm_rope_kv8(qkv, p, p, p, p, rows, pos, q, p, p, p,
                                                        pages, table, width, seqs, tokens, nh, nkv,
                                                        hd, eps, None)
    assert call(hd=96) == -4
    assert call(pos=None) == -1 and call(q=None) == -1 and call(table=None) == -1
    assert call(nh=0) == -2 and call(nh=5000) == -2 and call(rows=0) == -2
    assert call(tokens=-1) == -2 and call(width=0) == -2
    assert call(eps=-1.0) == -6 and call(eps=math.nan) == -6
    assert call(q=p + 8) == -3 and call(qkv=p + 2) == -3
    assert call(tokens=0, qkv=None) == 0 and call(seqs=0, q=None) == 0


def test_attention(p):
    L = K.lib
    size = L.dip_kv8_decode_attention_workspace_size
    ws = size(4, 1, 64, 8, 128, 500)
    assert ws > 0
    for bad in ((4, 1, 63, 8, 128, 500), (0, 1, 64, 8, 128, 500), (4, 1, 64, 8, 64, 500),
                (4, 1, 64, 8, 128, 0), (4, 0, 64, 8, 128, 500)):
        assert size(*bad) == 0
    dec = lambda q=p, pages=8, table=p, width=500, pos=p, out=p, seqs=4, tokens=1, nh=64, nkv=8, \
        hd=128, w=p, n=ws: L.dip_kv8_decode_attention(q, p, p, p, pages, table, width, pos, out,
                                                      seqs, tokens, nh, nkv, hd, 0.1, w, n, None)
    assert dec(pos=None) == -1 and dec(q=None) == -1 and dec(out=None) == -1 and dec(hd=64) == -4
    assert dec(table=None) == -1
    assert dec(nh=63) == -2 and dec(nh=8192) == -2 and dec(width=0) == -2 and dec(tokens=-1) == -2
    assert dec(w=None) == -5 and dec(n=ws - 1) == -5 and dec(w=p + 8) == -3 and dec(q=p + 2) == -3
    assert dec(pos=p + 4) == -3
    assert dec(tokens=0, q=None) == 0 and dec(seqs=0, q=None) == 0
    size = L.dip_kv8_prompt_attention_workspace_size
    ws = size(5, 20000, 32, 8, 128)
    assert ws > 0 and size(0, 0, 32, 8, 128) == 0 and size(5, -1, 32, 8, 128) == 0
    pro = lambda start=20000, tokens=5, w=p, n=ws, nh=32, width=400, q=p, hd=128, table=p: \
        L.dip_kv8_prompt_attention(q, p, p, p, 8, table, width, start, p, tokens, nh, 8, hd, 0.1,
                                   w, n, None)
    assert pro(start=-1) == -2 and pro(start=25596) == -2 and pro(tokens=-1) == -2
    assert pro(start=1 << 62) == -2
    assert pro(nh=33) == -2 and pro(w=None) == -5 and pro(n=ws - 1) == -5 and pro(hd=32) == -4
    assert pro(q=None) == -1 and pro(table=None) == -1 and pro(w=p + 4) == -3
    assert pro(tokens=0, q=None) == 0


def test_launches_of_two_to_the_32_threads(p):
    """HIP takes none of these: refused as too large, not passed on."""
    L = K.lib
    big = 1 << 30
    assert _write(p, nkv=4096, width=1 << 24, tokens=big) == -2
    assert _write(p, seqs=1 << 24, nkv=8) == -2
    assert L.dip_kv8_read(p, p, p, 8, p, 1 << 24, p, p, p, 1, big, 4096, 128, None) == -2
    assert L.dip_qk_norm_rope_kv8(p, p, p, p, p, big, p, p, p, p, p, 8, p, 1 << 24, 1, 1 << 23, 64,
                                  8, 128, 1e-6, None) == -2
    n = 1 << 62
    assert L.dip_kv8_decode_attention(p, p, p, p, 8, p, 1 << 24, p, p, 1 << 20, 1, 64, 8, 128, 0.1,
                                      p, n, None) == -2
    assert L.dip_kv8_prompt_attention(p, p, p, p, 8, p, 1 << 24, 0, p, big, 64, 8, 128, 0.1, p, n,
                                      None) == -2


def test_calls_on_host_tensors_are_refused():
    import torch
    with pytest.raises(RuntimeError):
        K.kv8_cache(2, 4, device="cpu")
    with pytest.raises(RuntimeError):
        K.kv8_cache(0, 4)
    with pytest.raises(RuntimeError):
        K.kv8_read("cache", torch.zeros(1, 1), torch.zeros(1), 1)
