"""GPU: the 8-bit cache's attention with negative and zero scales, by each route, long
prompts in splits, shared pages, and sizes of nothing."""
import math

import pytest
import torch

from kv4_util import attention
from kv8_util import PAGE, attention_bound
from test_gpu_kv8 import _check, _filled, _gen, _kv, _pos

pytestmark = pytest.mark.gpu

SCALE = 1 / math.sqrt(128)


@pytest.mark.parametrize("scale", [-SCALE, 0.0, -2.5])
@pytest.mark.parametrize("tokens", [1, 5, 20, 40])
def test_scales_of_every_sign(tokens, scale):
    import _dip_hip as K
    print(f"kv8 attention tokens={tokens} scale={scale}", flush=True)
    g = _gen(tokens)
    nh, nkv, lengths = 16, 2, [300, 1300]
    cache, table, values = _filled(g, lengths, nkv)
    # (scores of 2.5 times products of 128 stay below 2^6 with queries this small)
    q = (0.1 * torch.randn(2, tokens, nh * 128, device="cuda", generator=g)).to(torch.bfloat16)
    out = K.kv8_decode_attention(q, cache, table, _pos(*[n - tokens for n in lengths]), None, scale)
    _check(out, q, values, lengths, tokens, nh, scale)
    for i, n in enumerate(lengths):
        one = K.kv8_prompt_attention(q[i], cache, table[i], n - tokens, None, scale)
        _check(one[None], q[i:i + 1], values[i:i + 1], [n], tokens, nh, scale)


@pytest.mark.parametrize("tokens,start,nh,nkv", [(40, 5000, 16, 1), (300, 6001, 4, 2),
                                                 (129, 4000, 2, 1)])
def test_prompts_behind_many_rows(tokens, start, nh, nkv):
    import _dip_hip as K
    print(f"kv8 prompt tokens={tokens} start={start} heads={nh}/{nkv}", flush=True)
    g = _gen(start)
    cache, table, values = _filled(g, [start + tokens], nkv)
    q = torch.randn(tokens, nh * 128, device="cuda", generator=g).to(torch.bfloat16)
    out = K.kv8_prompt_attention(q, cache, table[0], start, None, SCALE)
    (k, v), some = values[0], sorted({0, 1, tokens // 2, tokens - 2, tokens - 1})
    want, size = attention(q[some].view(len(some), nh, 128), k, v, [start + t + 1 for t in some],
                           SCALE)
    err = (out[some].view(len(some), nh, 128).double().cpu() - want).abs()
    assert bool((err <= attention_bound(want, size)).all()), float(err.max())


def test_sequences_that_share_pages():
    """A common beginning, in the tables of several sequences at once."""
    import _dip_hip as K
    g = _gen(8)
    cache = K.kv8_cache(2, 8)
    table = torch.tensor([[5, 1, 2], [5, 1, 7], [5, 0, 5]], dtype=torch.int32, device="cuda")
    K.kv8_write(*_kv(g, 1, 512, 2), cache, torch.arange(8, dtype=torch.int32, device="cuda")[None],
                _pos(0))
    q = torch.randn(3, 2, 8 * 128, device="cuda", generator=g).to(torch.bfloat16)
    pos = _pos(170, 130, 128)
    out = K.kv8_decode_attention(q, cache, table, pos, None, SCALE)
    for i in range(3):
        k, v = (x[0].double().cpu() for x in K.kv8_read(cache, table[i:i + 1], _pos(0), 3 * PAGE))
        n = int(pos[i]) + 2
        _check(out[i:i + 1], q[i:i + 1], [(k[:n], v[:n])], [n], 2, 8)


def test_sizes_of_nothing():
    import _dip_hip as K
    cache, cuda = K.kv8_cache(2, 2), dict(device="cuda")
    before = [t.clone() for t in cache]
    table = torch.zeros(1, 2, dtype=torch.int32, **cuda)
    bf16 = dict(dtype=torch.bfloat16, **cuda)
    none = torch.empty(1, 0, 2, 128, **bf16)
    K.kv8_write(none, none, cache, table, _pos(0))
    assert K.kv8_read(cache, table, _pos(0), 0)[0].shape == (1, 0, 2, 128)
    assert K.kv8_decode_attention(torch.empty(1, 0, 512, **bf16), cache, table, _pos(0), None,
                                  SCALE).shape == (1, 0, 512)
    assert K.kv8_prompt_attention(torch.empty(0, 512, **bf16), cache, table[0], 0, None,
                                  SCALE).shape == (0, 512)
    w, tab = torch.ones(128, **bf16), torch.ones(9, 128, **bf16)
    q = torch.empty(1, 0, 512, **bf16)
    assert K.qk_norm_rope_kv8(torch.empty(1, 0, 1024, **bf16), w, w, tab, tab, _pos(0), q, cache,
                              table, 4, 2, 1e-6) is q
    no = torch.zeros(0, 2, dtype=torch.int32, **cuda)
    pos = torch.zeros(0, dtype=torch.int64, **cuda)
    assert K.kv8_decode_attention(torch.empty(0, 1, 512, **bf16), cache, no, pos, None,
                                  SCALE).shape == (0, 1, 512)
    K.kv8_write(torch.empty(0, 3, 2, 128, **bf16), torch.empty(0, 3, 2, 128, **bf16), cache, no, pos)
    assert K.kv8_read(cache, no, pos, 3)[0].shape == (0, 3, 2, 128)
    t, a = K.verify(torch.empty(0, 3, 50, **bf16), torch.empty(0, 2, dtype=torch.int64, **cuda),
                    torch.empty(0, 3, **cuda))
    assert t.shape == (0, 3) and a.shape == (0,)
    t, a = K.verify(torch.arange(50, **cuda).view(1, 1, 50).bfloat16() * 100,
                    torch.empty(1, 0, dtype=torch.int64, **cuda), torch.full((1, 1), 0.5, **cuda),
                    torch.empty(1, 0, 50, **bf16))
    assert t.tolist() == [[49]] and a.tolist() == [0]
    assert all(torch.equal(x, y) for x, y in zip(cache, before))
