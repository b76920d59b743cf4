"""GPU: queries of tokens whose page the table lacks inside its width stay as they were,
as their keys and values do; those of the tokens before and behind are written."""
import pytest
import torch

from test_gpu_kv8 import _gen, _pos

pytestmark = pytest.mark.gpu

MARK = 7.0


def _call(qkv, q, cache, table, pos, heads):
    import _dip_hip as K
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    tab = torch.ones(512, 128, dtype=torch.bfloat16, device="cuda")
    K.qk_norm_rope_kv8(qkv, w, w, tab, tab, pos, q, cache, table, heads, cache.n_kv_heads, 1e-6)


@pytest.mark.parametrize("missing", [-1, 9, -(1 << 31), (1 << 31) - 1])
@pytest.mark.parametrize("heads,nkv", [(2, 1), (5, 1), (64, 8)])
def test_a_page_missing_in_the_middle(heads, nkv, missing):
    import _dip_hip as K
    print(f"page {missing}, {heads} / {nkv} heads", flush=True)
    n = 140  # from 30 on: pages 0, 1 and 2
    qkv = torch.randn(2, n, (heads + 2 * nkv) * 128, device="cuda",
                      generator=_gen(heads)).to(torch.bfloat16)
    table = torch.tensor([[4, missing, 2], [0, 1, 3]], dtype=torch.int32, device="cuda")
    full = torch.tensor([[4, 5, 2], [0, 1, 3]], dtype=torch.int32, device="cuda")
    out = []
    for t in (table, full):
        cache = K.kv8_cache(nkv, 9)
        q = torch.full((2, n, heads * 128), MARK, dtype=torch.bfloat16, device="cuda")
        _call(qkv, q, cache, t, _pos(30, 7), heads)
        out.append((q, cache))
    (q, cache), (want, whole) = out
    gone = slice(64 - 30, 128 - 30)
    assert bool((q[0, gone] == MARK).all())
    assert torch.equal(q[0, :gone.start], want[0, :gone.start])
    assert torch.equal(q[0, gone.stop:], want[0, gone.stop:]) and torch.equal(q[1], want[1])
    assert not bool((want == MARK).flatten(0, 1).all(-1).any())
    for x, y in zip(cache, whole):
        y = y.clone()
        y[5] = 0  # the page that the other table has
        assert torch.equal(x, y)


@pytest.mark.parametrize("tokens", [1, 3])
def test_one_sequence_of_many_has_no_page(tokens):
    import _dip_hip as K
    qkv = torch.randn(3, tokens, 6 * 128, device="cuda", generator=_gen(3)).to(torch.bfloat16)
    table = torch.tensor([[1, 2], [-1, 0], [5, 3]], dtype=torch.int32, device="cuda")
    cache = K.kv8_cache(1, 5)
    q = torch.full((3, tokens, 4 * 128), MARK, dtype=torch.bfloat16, device="cuda")
    _call(qkv, q, cache, table, _pos(20, 63, 5), 4)
    assert not bool((q[0] == MARK).all(-1).any()) and bool((q[2] == MARK).all())
    assert bool((q[1, 0] == MARK).all())  # of page -1; the next is row 0 of page 0
    assert not bool((q[1, 1:] == MARK).all(-1).any())
