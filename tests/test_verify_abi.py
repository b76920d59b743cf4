"""dip_verify rejects bad arguments before any launch (no GPU needed)."""
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


def _call(p, logits=1, dtype=0, seqs=2, tokens=3, vocab=8, stride=8, drafted=1, draft=1, dstride=8,
          u=1, t=1.0, k=0, tp=1.0, mp=0.0, out=1, acc=1, ws=1, n=1 << 30, off=0, doff=0, woff=0):
    return K.lib.dip_verify(p + off if logits else None, dtype, seqs, tokens, vocab, stride,
                            p if drafted else None, p + doff if draft else None, dstride,
                            p if u else None, t, k, tp, mp, p if out else None, p if acc else None,
                            p + woff if ws else None, n, None)


def test_verify(p):
    assert _call(p, dtype=3) == -4
    for bad in (dict(seqs=-1), dict(seqs=1 << 23), dict(tokens=-1), dict(tokens=1 << 21),
                dict(vocab=0), dict(vocab=(1 << 30) + 1), dict(stride=-1), dict(dstride=-1),
                dict(seqs=1 << 21, tokens=1)):
        assert _call(p, **bad) == -2, bad
    for bad in (dict(t=-1.0), dict(t=math.nan), dict(t=math.inf), dict(k=-1), dict(tp=0.0),
                dict(tp=1.5), dict(tp=math.nan), dict(mp=-0.1), dict(mp=1.1), dict(mp=math.nan)):
        assert _call(p, **bad) == -6, bad
    for name in ("logits", "drafted", "u", "out", "acc"):
        assert _call(p, **{name: 0}) == -1, name
    size = K.lib.dip_verify_workspace_size
    assert 0 < size(2, 3, 8, 0) < size(2, 3, 8, 1)
    assert size(0, 3, 8, 0) == 0 and size(2, -1, 8, 0) == 0 and size(2, 3, 0, 0) == 0
    assert _call(p, ws=0) == -5 and _call(p, n=size(2, 3, 8, 1) - 1) == -5
    assert _call(p, off=1) == -3 and _call(p, doff=1) == -3 and _call(p, woff=8) == -3
    assert _call(p, seqs=0, logits=0) == 0


def test_the_workspace_of_long_rows_has_room_for_their_slices():
    size = K.lib.dip_verify_workspace_size
    # a row's list of 4096 words, and a histogram of 1024 for each of its slices
    assert size(1, 0, 151936, 0) > 4096 * 8 + 149 * 1024 * 8
    assert size(4, 4, 151936, 1) > 36 * (4096 * 8 + 1024 * 8)


def test_host_tensors_are_refused():
    import torch
    with pytest.raises(RuntimeError):
        K.verify(torch.zeros(1, 2, 8), torch.zeros(1, 1, dtype=torch.int64), torch.zeros(1, 2))
