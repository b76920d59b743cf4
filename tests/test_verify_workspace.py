"""The workspace that dip_verify asks for is never above what dip_verify_workspace_size
gives for the call's sizes, greedy calls that hand over the draft's logits included (no
GPU needed: a misaligned workspace ends the call behind the check of its size)."""
import ctypes

import pytest
import torch

import _dip_hip as K

SIZE, WORKSPACE, ALIGN = K.lib.dip_verify_workspace_size, -5, -3


@pytest.fixture(scope="module")
def p():
    buf = (ctypes.c_uint8 * 64)()
    addr = ctypes.addressof(buf)
    yield addr + (-addr % 16)
    del buf


def _call(p, seqs, tokens, vocab, n, dtype=0, t=1.0, k=0, tp=1.0, mp=0.0, draft=True):
    return K.lib.dip_verify(p, dtype, seqs, tokens, vocab, vocab, p, p if draft else None, vocab, p,
                            t, k, tp, mp, p, p, p + 8, n, None)


# rows * slices lies on both sides of 2048, where rows are cut more coarsely; rows that a
# workgroup holds and rows in slices
VOCABS = (1, 8, 1024, 2049, 3000, 4000, 4096, 5003, 6143, 8000, 8188, 16380, 32003, 151936, 700001)


@pytest.mark.parametrize("vocab", VOCABS)
def test_the_drafts_logits_never_ask_for_less(vocab):
    for tokens in range(9):
        for seqs in list(range(1, 65)) + list(range(70, 600, 7)) + [1024, 2047, 4096]:
            assert SIZE(seqs, tokens, vocab, 1) >= SIZE(seqs, tokens, vocab, 0), (seqs, tokens)


@pytest.mark.parametrize("seqs,tokens,vocab", [(128, 1, 8000), (86, 1, 8188), (300, 2, 3000),
                                               (599, 8, 4096), (2, 3, 8), (16, 5, 151936)])
@pytest.mark.parametrize("how", [dict(t=0.0), dict(k=1), dict(), dict(k=20), dict(tp=0.9)])
def test_that_much_is_enough(p, seqs, tokens, vocab, how):
    for draft in (False, True):
        n = SIZE(seqs, tokens, vocab, int(draft))
        for dtype in range(3):
            assert _call(p, seqs, tokens, vocab, n, dtype=dtype, draft=draft, **how) == ALIGN
        assert _call(p, seqs, tokens, vocab, 0, draft=draft, **how) == WORKSPACE


@pytest.mark.gpu
@pytest.mark.parametrize("how", [dict(temperature=0.0), dict(top_k=1), dict(top_k=20)])
def test_many_short_rows_with_the_drafts_logits(how):
    from test_gpu_verify import _check, _inputs
    print(f"verify 128x1 of 8000, {how}", flush=True)
    x, d, u, y = _inputs(128, 1, 8000, torch.bfloat16, 5)
    _check(x, d, u, y, **how)
